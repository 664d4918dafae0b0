// Attention of drafted tokens (a tree per sequence; one token is plain
// decoding) over a paged key/value cache, with gpt-oss's sinks and sliding
// window (transformers models/gpt_oss/modeling_gpt_oss.py, GptOssAttention and
// eager_attention_forward).
//
// The T * Hq/Hkv rows that share a kv head are taken together, so a key is read
// once for all of them.  One pass over the keys with the running maximum m and
// sum z of the softmax (base 2): with x_j = scale log2(e) q . k_j,
//   m' = max(m, max_j x_j);  z' = z 2^(m-m') + sum_j 2^(x_j-m');
//   O' = O 2^(m-m') + sum_j 2^(x_j-m') v_j,     out = O / (z + 2^(sink-m)).
// Partial (m, z, O) of key ranges join by the same rule, in a fixed order.  A maximum
// passes over NaN, a sum does not: a part has nothing to add where z is 0, not where m
// is -inf, which a part whose every score is NaN has too.
//
// Statistics, sums and O are 32 bits.  The weights are rounded to bf16 for the product
// with V, whose values are bf16 (both operands of it have one type): off by 2^-8 of each
// weight at most, which adds to the output's own rounding.  Against 64 bits, relative
// to the whole output: 16-token trees over 131072 keys 2.3e-3, one token over 500 keys
// 1.9e-3, where weights of 32 bits and the same last rounding give 1.7e-3.
// It is a product of matrices: a value of infinity or NaN in a slot that some row of
// the kv head may attend reaches the other rows as 0 times itself.
//
// Work split: the keys of every (sequence, kv head, row tile) are cut into
// units; the units of all items, in item order, are cut into equal contiguous
// ranges, one per CTA, from the lengths on the device (no host read, no idle
// SMs for ragged batches or single sequences).  An item inside one range is
// finished there; the pieces of the others go to the workspace and a second
// launch (programmatic, so that its start overlaps) joins them.
#include <type_traits>

#include "bs_paged.cuh"
#include "bs_ring.cuh"

namespace bs {

int paged_cache(const char* fn, const bs_kv_cache* c, int64_t extra, bool need_v, PagedCache* o) {
  BS_ARG(c->k && (c->v || !need_v) && c->page_table && c->lens, "%s: null pointer in the cache", fn);
  BS_ARG(c->pages > 0 && c->page_size > 0 && c->heads > 0 && c->table_width > 0 && c->batch >= 0, "%s: bad cache sizes", fn);
  BS_ARG(c->dim > 0 && c->dim <= 128 && c->dim % 8 == 0, "%s: the head size must be a multiple of 8 up to 128", fn);
  // (slots and their sums with a tile stay below 2^31)
  BS_ARG(c->pages < INT32_MAX && c->page_size < INT32_MAX && c->heads <= 65535 && c->batch < (1 << 24) &&
             c->table_width * c->page_size < INT32_MAX - (1 << 16) && c->table_stride >= 0,
         "%s: cache sizes too large", fn);
  BS_ARG(extra >= 0 && extra <= c->table_width * c->page_size, "%s: more drafted tokens than slots in a table row", fn);
  BS_ALIGNED16(c->k, "the key cache");
  BS_ALIGNED16(c->v, "the value cache");
  const int64_t strides[6] = {c->k_stride_page, c->k_stride_slot, c->k_stride_head,
                              c->v_stride_page, c->v_stride_slot, c->v_stride_head};
  for (int i = 0; i < (need_v ? 6 : 3); ++i)
    BS_REQUIRE(strides[i] % 8 == 0, BS_ERR_MISALIGNED, "%s: cache strides must be multiples of 8 elements", fn);
  o->k = static_cast<__nv_bfloat16*>(c->k);
  o->v = static_cast<__nv_bfloat16*>(c->v);
  o->kp = c->k_stride_page, o->ks = c->k_stride_slot, o->kh = c->k_stride_head;
  o->vp = c->v_stride_page, o->vs = c->v_stride_slot, o->vh = c->v_stride_head;
  o->table = c->page_table;
  o->table_stride = c->table_stride;
  o->lens = c->lens;
  o->pages = (int)c->pages;
  o->heads = (int)c->heads;
  o->dim = (int)c->dim;
  o->capacity = (int)(c->table_width * c->page_size);
  o->div.size = (int)c->page_size;
  o->div.shift = -1;
  for (int s = 0; s < 31; ++s)
    if ((1ll << s) == c->page_size) o->div.shift = s;
  o->status = device_status_ptr();
  return BS_OK;
}

int cache_box_rows(const bs_kv_cache* c, int most) {
  int r = 1;
  while (r < most && c->page_size % (2 * r) == 0) r *= 2;
  return r;
}

int cache_maps(const bs_kv_cache* c, int rows, bool need_v, CacheMaps* o) {
  const uint64_t dims[4] = {(uint64_t)c->dim, (uint64_t)c->heads, (uint64_t)c->page_size, (uint64_t)c->pages};
  const uint32_t box[4] = {64, 1, (uint32_t)rows, 1};
  // a dimension of one element may have any stride in the caller's tensor
  auto bytes = [](int64_t stride, int64_t n) { return n > 1 ? (uint64_t)stride * 2 : (uint64_t)16; };
  const uint64_t ks[3] = {bytes(c->k_stride_head, c->heads), bytes(c->k_stride_slot, c->page_size), bytes(c->k_stride_page, c->pages)};
  BS_TRY(make_map_4d(&o->k, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, c->k, dims, ks, box, CU_TENSOR_MAP_SWIZZLE_128B));
  if (!need_v) return BS_OK;
  const uint64_t vs[3] = {bytes(c->v_stride_head, c->heads), bytes(c->v_stride_slot, c->page_size), bytes(c->v_stride_page, c->pages)};
  return make_map_4d(&o->v, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, c->v, dims, vs, box, CU_TENSOR_MAP_SWIZZLE_128B);
}

namespace {

constexpr int kMaxDrafts = 256;
// Where no more than so many keys are in reach an item is not cut, and there is one
// launch.  The reach is known on the host: the window, or the width of the page table
// (lengths are on the device), so a table for longer sequences has its items cut however
// short they are.  Uncut / cut, us, tables of the very length and for 131072 slots, 8 kv
// heads, one token: 256 x 300 keys 49 / 54, 64 x 450 24 / 22, 8 x 450 12.2 / 12.5,
// 1 x 450 12.1 / 11.3 on the device, where the second launch costs the host 1.8 more
// (19.7 / 21.5 a call); 900 keys 16.7 / 10.5; 64 x 450 with a window of 128 18.1 / 21.5.
constexpr int kWholeKeys = 512;
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;

struct TreeArgs : SplitArgs {
  const __nv_bfloat16* q;
  int64_t qb, qt, qh;
  const uint8_t* mask;
  int64_t mask_b;
  const float* sinks;
  float scale2;  // scale * log2(e)
  int G, R;
  __nv_bfloat16* out;
  float* lse;
  float4* part_o;   // [2 * grid][dim / 4][tile rows]: rows adjacent, as the writers' threads are
  float2* part_ml;  // [2 * grid][tile rows]
};

// ---------------------------------------------------------------- few rows
// Row tiles of MT * 16 rows on mma.sync, four warps per CTA, each streaming its
// own units of kU keys into its own ring (no barrier between warps) and holding
// its own (m, z, O); they meet at the end of an item.  HBM-bound for long items: of each
// warp's ring all stages but the one that is worked on are in flight, 96 KB per SM in
// three CTAs of two stages, 128 KB in two of three.  64 sequences of up to 8192 keys, 64 / 8
// heads of 64: 92 us, 5.9 TB/s (90% of the measured copy rate); heads of 128: 176 to 180 us,
// 6.0 TB/s; heads of 80 and 96, which are worked on as 128: 162 us.  2 x 131072 keys: 90 us
// where a head's slots lie together in a page, 113 us where heads are interleaved
// (128 bytes in every KB).  Short items are bound by the chain of an item's start, units
// and end, some 8000 cycles, which a third CTA hides better than a third stage of the
// rings (256 ragged sequences to 1000 keys: 68.8 us, 88 with two CTAs); heads of 128
// would spill with three (133 us, 126 with two).
// kTma: a unit is fetched by a few TMA boxes (pages of a multiple of 8 slots); else
// by 16-byte asynchronous copies, whose address arithmetic and issue are most of
// the kernel's instructions then (pages of 12 slots: 119 us for the 64 sequences, 250 with
// heads of 128).
template <int DP>
struct RowsCfg {
  static constexpr int kU = DP == 64 ? 32 : 16;
  static constexpr int kStages = DP == 64 ? 2 : 3;
  static constexpr int kTile = kU * DP * 2;           // bytes of a K (or V) unit
  static constexpr int kWarpBytes = 2 * kTile * kStages;
};
template <int DP, int MT>
struct RowsSmem {
  static constexpr int kRows = 16 * MT;
  static constexpr int merge = 4 * RowsCfg<DP>::kWarpBytes;
  static constexpr int kBufs = MT * DP == 64 ? 2 : 1;          // warps whose O is passed at once
  static constexpr int ml = merge + kBufs * kRows * DP * 4;    // [4 warps][rows] float2
  static constexpr int bits = ml + 4 * kRows * 8;              // [rows][8] words
  static constexpr int thr = bits + kRows * (kMaxDrafts / 32) * 4;
  static constexpr int q = merge;                              // the item's Q, until its fragments are read
  static constexpr int sums = (thr + kRows * 4 + 15) / 16 * 16;
  static constexpr int bars = sums + 64;                       // [4 warps][kStages]
  static constexpr int total = bars + 4 * RowsCfg<DP>::kStages * 8 + 1024;
};
static_assert(3 * (RowsSmem<64, 1>::total + 1024) <= 228 * 1024, "three CTAs per SM");

// CTAs of an SM.
constexpr int rows_ctas(int rows, int64_t dim) { return rows == 16 && dim <= 64 ? 3 : 2; }

template <int DP, int MT, bool kTma>
__global__ void __launch_bounds__(128, rows_ctas(16 * MT, DP)) tree_rows_kernel(const __grid_constant__ TreeArgs a,
                                                           const __grid_constant__ CacheMaps maps) {
  using Cfg = RowsCfg<DP>;
  using Sm = RowsSmem<DP, MT>;
  constexpr int kU = Cfg::kU, KS = DP / 16, NT = kU / 8, kRows = 16 * MT, kWords = kMaxDrafts / 32;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
  __shared__ int abort_flag;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  float* merge = reinterpret_cast<float*>(smem + Sm::merge);
  float2* ml = reinterpret_cast<float2*>(smem + Sm::ml);
  uint32_t* bits = reinterpret_cast<uint32_t*>(smem + Sm::bits);
  int* thr = reinterpret_cast<int*>(smem + Sm::thr);
  const uint32_t base = ptx::smem_addr(smem) + warp * Cfg::kWarpBytes;
  const uint32_t bar = ptx::smem_addr(smem) + Sm::bars + warp * Cfg::kStages * 8;
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");

  if constexpr (kTma) {
    if (threadIdx.x == 0) abort_flag = 0;
    if (lane == 0) {
      for (int s = 0; s < Cfg::kStages; ++s) ptx::mbar_init(bar + 8 * s, 1);
      ptx::fence_mbar_init();
    }
  } else if (a.c.dim < DP) {
    // columns dim..DP are zeros that no copy touches
    for (int i = threadIdx.x; i < 4 * Cfg::kWarpBytes / 16; i += 128)
      reinterpret_cast<uint4*>(smem)[i] = make_uint4(0, 0, 0, 0);
  }
  __syncthreads();
  const Range r = locate<kU>(a, blockIdx.x, gridDim.x, reinterpret_cast<int64_t*>(smem + Sm::sums));
  Walk lw, cw;
  if (r.p0 >= r.p1 || !walk_begin<kU>(a, r, lw)) return;
  cw = lw;

  // ---- loading.  Lane g holds the page and row of the next unit's g-th box (or,
  // without TMA, slot); pages are looked up one unit ahead.
  const int box = kTma ? min(a.box, kU) : 1, boxes = kU / box;
  lw.u = lw.start + warp;
  bool more = true;
  Ring<Cfg::kStages> ring;
  int next_page = 0, next_row = -1;  // row < 0: no key there
  auto find = [&]() {
    while (more && lw.u >= lw.end) {
      more = walk_next<kU>(a, lw);
      lw.u = lw.start + warp;
    }
    next_row = -1;
    if (!more || lane >= boxes) return;
    const int slot = lw.k.lo + lw.u * kU + lane * box;
    if (kTma ? slot < lw.k.hi : holds_key(a, lw.b, lw.k, slot)) {
      int p;
      a.c.div.split(slot, p, next_row);
      next_page = __ldg(a.c.table + lw.b * a.c.table_stride + p);
    }
  };
  auto load = [&](int stage) {
    if (more) {
      const uint32_t kd = base + stage * 2 * Cfg::kTile, vd = kd + Cfg::kTile;
      if (next_row >= 0 && (unsigned)next_page >= (unsigned)a.c.pages) {
        if (!kTma || box_in_use(a, lw.b, lw.k.n, lw.k.lo + lw.u * kU + lane * box)) {
          record_status(a.c.status, BS_ERR_CAPACITY);
          next_page = next_page < 0 ? 0 : a.c.pages - 1;
        } else {
          next_row = -1;
        }
      }
      if constexpr (kTma) {
        if (lane == 0) ptx::mbar_arrive_expect_tx(bar + 8 * stage, 2 * Cfg::kTile);
        __syncwarp();
        if (lane < boxes) {
          // a box behind the last slot lies outside the descriptor's pages: zeros
          const int page = next_row >= 0 ? next_page : a.c.pages, row = max(next_row, 0);
#pragma unroll
          for (int x = 0; x < DP / 64; ++x) {
            const uint32_t at = x * (kU * 128) + lane * box * 128;
            ptx::tma_load_4d(kd + at, &maps.k, bar + 8 * stage, x * 64, lw.h, row, page);
            ptx::tma_load_4d(vd + at, &maps.v, bar + 8 * stage, x * 64, lw.h, row, page);
          }
        }
      } else {
        constexpr int kLanesRow = DP / 8;  // lanes that copy one row
        const int c = lane % kLanesRow;
        const __nv_bfloat16* kb = a.c.k + lw.h * a.c.kh + c * 8;
        const __nv_bfloat16* vb = a.c.v + lw.h * a.c.vh + c * 8;
        const bool col = c * 8 < a.c.dim;
#pragma unroll
        for (int i = 0; i < kU * kLanesRow / 32; ++i) {
          const int row = lane / kLanesRow + i * (32 / kLanesRow);
          const int p = __shfl_sync(0xffffffffu, next_page, row);
          const int x = __shfl_sync(0xffffffffu, next_row, row);
          if (col) {
            const uint32_t at = mma::tile_at<kU>(row, c);
            const bool on = x >= 0;
            mma::cp_async_16_or_zero(kd + at, on ? kb + p * a.c.kp + x * a.c.ks : kb, on);
            mma::cp_async_16_or_zero(vd + at, on ? vb + p * a.c.vp + x * a.c.vs : vb, on);
          }
        }
      }
      lw.u += 4;
      find();
    }
    if constexpr (!kTma) ptx::cp_async_commit();
  };
  find();
#pragma unroll
  for (int s = 0; s < Cfg::kStages - 1; ++s) {
    ring.place(more);
    load(s);
  }

  // ---- what an item starts with, asked for while the item before it is worked on: its Q,
  // and the positions and masks of the first row of bits of each warp
  constexpr int kChunks = DP / 8, kQ = kRows * kChunks / 128;
  const int words = (a.T + 31) / 32;
  uint4 next_q[kQ];
  int next_pt = -1, next_pu = -1;
  uint8_t next_may = 0;
  auto ask = [&](const Walk& w) {
    const int row0 = w.tile * kRows, rows = min(kRows, a.R - row0);
#pragma unroll
    for (int i = 0; i < kQ; ++i) {
      const int x = threadIdx.x + i * 128, row = row0 + min(x / kChunks, rows - 1), t = row / a.G, g = row - t * a.G;
      next_q[i] = __ldg(reinterpret_cast<const uint4*>(a.q + w.b * a.qb + t * a.qt + (int64_t)(w.h * a.G + g) * a.qh +
                                                       min(x % kChunks * 8, a.c.dim - 8)));
    }
    const int tl = min(warp / words, (row0 + rows - 1) / a.G - row0 / a.G), t = row0 / a.G + tl;
    const int uc = min((warp - warp / words * words) * 32 + lane, a.T - 1);
    const int32_t* pos = a.pos + (int64_t)w.b * a.T;
    next_pt = __ldg(pos + t), next_pu = __ldg(pos + uc);
    if (a.mask) next_may = __ldg(a.mask + w.b * a.mask_b + (int64_t)t * a.T + uc);
  };
  ask(cw);

  // ---- pieces
  while (true) {
    const int row0 = cw.tile * kRows, rows = min(kRows, a.R - row0);
    const int t0 = row0 / a.G, toks = (row0 + rows - 1) / a.G - t0 + 1;
#pragma unroll
    for (int i = 0; i < kQ; ++i) {
      const int x = threadIdx.x + i * 128, r = x / kChunks, c = x % kChunks;
      const bool on = r < rows && c * 8 < a.c.dim;
      *reinterpret_cast<uint4*>(smem + Sm::q + mma::tile_at<kRows>(r, c)) = on ? next_q[i] : make_uint4(0, 0, 0, 0);
    }
    // masks of the tile's tokens over the drafts, and each one's window
    if (a.window || cw.k.lo + cw.end * kU > cw.k.n) {
      const int32_t* pos = a.pos + (int64_t)cw.b * a.T;
      for (int i = warp; i < toks * words; i += 4) {
        const int tl = i / words, w = i - tl * words, t = t0 + tl, u = w * 32 + lane;
        int pt = next_pt, pu = next_pu;
        uint8_t may = next_may;
        if (i >= 4) {
          const int uc = min(u, a.T - 1);
          pt = __ldg(pos + t), pu = __ldg(pos + uc);
          if (a.mask) may = __ldg(a.mask + cw.b * a.mask_b + (int64_t)t * a.T + uc);
        }
        const int below = a.window ? max(pt, cw.k.n) - a.window : -1;
        const uint32_t m = __ballot_sync(0xffffffffu, u < a.T && (a.mask ? may != 0 : u <= t) && pt >= 0 && pu >= 0 &&
                                                          (!a.window || pu > below));
        if (lane == 0) {
          bits[tl * kWords + w] = m;
          if (w == 0) thr[tl] = pt >= 0 ? below : INT_MAX;
        }
      }
    }
    // (what the rows' ends need is loaded meanwhile)
    int tl[MT][2], pt[MT][2];
    float sink[MT][2];
    int64_t at[MT][2];
#pragma unroll
    for (int mt = 0; mt < MT; ++mt)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int row = row0 + min(mt * 16 + lane / 4 + e * 8, rows - 1), t = row / a.G, h = cw.h * a.G + row - t * a.G;
        tl[mt][e] = t - t0;
        at[mt][e] = ((int64_t)cw.b * a.T + t) * a.Hkv * a.G + h;
        pt[mt][e] = __ldg(a.pos + (int64_t)cw.b * a.T + t);
        sink[mt][e] = a.sinks ? __ldg(a.sinks + h) : -INFINITY;
      }
    __syncthreads();
    uint32_t qf[MT][KS][4];
#pragma unroll
    for (int mt = 0; mt < MT; ++mt)
#pragma unroll
      for (int k = 0; k < KS; ++k)
        mma::ldsm_x4(ptx::smem_addr(smem) + Sm::q + mma::tile_at<kRows>(mt * 16 + (lane & 15), 2 * k + (lane >> 4)), qf[mt][k]);
    Walk nw = cw;
    const bool again = walk_next<kU>(a, nw);
    if (again) ask(nw);

    float m[MT][2], z[MT][2], o[MT][DP / 8][4];
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
      m[mt][0] = m[mt][1] = -INFINITY;
      z[mt][0] = z[mt][1] = 0.f;
#pragma unroll
      for (int d = 0; d < DP / 8; ++d) o[mt][d][0] = o[mt][d][1] = o[mt][d][2] = o[mt][d][3] = 0.f;
    }
    for (int u = cw.start + warp; u < cw.end; u += 4) {
      const uint32_t kt = base + ring.stage * 2 * Cfg::kTile, vt = kt + Cfg::kTile;
      const int slot0 = cw.k.lo + u * kU;
      if constexpr (kTma) {
        // (a wait that ran out is reported at the end)
        more = ring.take([&](int s, int parity, bool again) {
          volatile int gone = 0;
          return warp_wait(bar + 8 * s, parity, again ? &gone : &abort_flag);
        }) && more;
        if (slot0 < cw.k.low || slot0 + kU > cw.k.n) {
          // a box brings all its slots: those that hold no key become zeros in V
          if (lane < kU && !holds_key(a, cw.b, cw.k, slot0 + lane)) {
            uint8_t* v = smem + (vt - ptx::smem_addr(smem)) + lane * 128;
#pragma unroll
            for (int i = 0; i < DP / 8; ++i)
              *reinterpret_cast<uint4*>(v + (i >> 3) * (kU * 128) + (i & 7) * 16) = make_uint4(0, 0, 0, 0);
          }
          ptx::fence_proxy_async_smem();
        }
      } else {
        ptx::cp_async_wait<Cfg::kStages - 2>();
      }
      __syncwarp();
      load(ring.place(more));
      ring.next();

      float s[MT][NT][4];
#pragma unroll
      for (int mt = 0; mt < MT; ++mt)
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) s[mt][nt][0] = s[mt][nt][1] = s[mt][nt][2] = s[mt][nt][3] = 0.f;
#pragma unroll
      for (int k = 0; k < KS; ++k)
#pragma unroll
        for (int np = 0; np < NT / 2; ++np) {
          uint32_t f[4];
          mma::ldsm_x4(kt + mma::tile_at<kU>(np * 16 + (lane >> 4) * 8 + (lane & 7), 2 * k + ((lane >> 3) & 1)), f);
#pragma unroll
          for (int mt = 0; mt < MT; ++mt) {
            mma::bf16_16816(s[mt][2 * np], qf[mt][k], f[0], f[1]);
            mma::bf16_16816(s[mt][2 * np + 1], qf[mt][k], f[2], f[3]);
          }
        }
      const bool edge = slot0 + kU > cw.k.n || a.window;
#pragma unroll
      for (int mt = 0; mt < MT; ++mt) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            float x = s[mt][nt][e] * a.scale2;
            if (edge) {
              const int key = slot0 + nt * 8 + (lane & 3) * 2 + (e & 1), at = tl[mt][e >> 1], d = key - cw.k.n;
              const bool see = d < 0 ? key > thr[at] : d < a.T && (bits[at * kWords + (d >> 5)] >> (d & 31) & 1);
              x = see ? x : -INFINITY;
            }
            s[mt][nt][e] = x;
          }
        uint32_t p[NT][2];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          float mx = m[mt][e];
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) mx = fmaxf(mx, fmaxf(s[mt][nt][2 * e], s[mt][nt][2 * e + 1]));
          mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
          mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
          const float ref = mx == -INFINITY ? 0.f : mx;
          const float f = mma::exp2_fast(m[mt][e] - ref);
          m[mt][e] = mx;
          float sum = 0.f;
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
            const float y0 = mma::exp2_fast(s[mt][nt][2 * e] - ref);
            const float y1 = mma::exp2_fast(s[mt][nt][2 * e + 1] - ref);
            sum += y0 + y1;
            p[nt][e] = pack_bf16x2(y0, y1);  // (the choice of bf16: at the top)
          }
          z[mt][e] = z[mt][e] * f + sum;
          if (__any_sync(0xffffffffu, f != 1.f)) {
#pragma unroll
            for (int d = 0; d < DP / 8; ++d) {
              o[mt][d][2 * e] *= f;
              o[mt][d][2 * e + 1] *= f;
            }
          }
        }
#pragma unroll
        for (int j = 0; j < kU / 16; ++j) {
          const uint32_t pf[4] = {p[2 * j][0], p[2 * j][1], p[2 * j + 1][0], p[2 * j + 1][1]};
#pragma unroll
          for (int dp = 0; dp < DP / 16; ++dp) {
            uint32_t f[4];
            mma::ldsm_x4_trans(vt + mma::tile_at<kU>(j * 16 + ((lane >> 3) & 1) * 8 + (lane & 7), 2 * dp + (lane >> 4)), f);
            mma::bf16_16816(o[mt][2 * dp], pf, f[0], f[1]);
            mma::bf16_16816(o[mt][2 * dp + 1], pf, f[2], f[3]);
          }
        }
      }
    }

    // ---- the warps' parts meet: common maximum, then O of warps 2, 3 to 0, 1 and of 1 to 0
    const bool whole = cw.whole();
    const int64_t slot = 2 * (int64_t)blockIdx.x + (cw.start == 0 ? 1 : 0);
    const int dim = a.c.dim;
#pragma unroll
    for (int mt = 0; mt < MT; ++mt)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        sink[mt][e] *= kLog2e;
        z[mt][e] += __shfl_xor_sync(0xffffffffu, z[mt][e], 1);
        z[mt][e] += __shfl_xor_sync(0xffffffffu, z[mt][e], 2);
        if ((lane & 3) == 0) ml[warp * kRows + mt * 16 + lane / 4 + e * 8] = make_float2(m[mt][e], z[mt][e]);
      }
    __syncthreads();
#pragma unroll
    for (int mt = 0; mt < MT; ++mt)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int row = mt * 16 + lane / 4 + e * 8;
        float mx = -INFINITY, zz = 0.f;
#pragma unroll
        for (int w = 0; w < 4; ++w) mx = fmaxf(mx, ml[w * kRows + row].x);
#pragma unroll
        for (int w = 0; w < 4; ++w) {
          const float2 v = ml[w * kRows + row];
          zz += v.y != 0.f ? v.y * mma::exp2_fast(v.x - mx) : 0.f;
        }
        const float f = mx == -INFINITY ? 0.f : mma::exp2_fast(m[mt][e] - mx);
#pragma unroll
        for (int d = 0; d < DP / 8; ++d) {
          o[mt][d][2 * e] *= f;
          o[mt][d][2 * e + 1] *= f;
        }
        m[mt][e] = mx;
        z[mt][e] = zz;
      }
    // two buffers: 2, 3 -> 0, 1, then 1 -> 0; one (where two would cost the second CTA of an SM): 3, 2, 1 -> 0
#pragma unroll 1
    for (int step = Sm::kBufs == 2 ? 2 : 3; step; step = Sm::kBufs == 2 ? step / 2 : step - 1) {
      const int to = warp - step, n = Sm::kBufs == 2 ? step : 1;
      if (to >= 0 && to < n) {
#pragma unroll
        for (int mt = 0; mt < MT; ++mt)
#pragma unroll
          for (int d = 0; d < DP / 8; ++d)
            *reinterpret_cast<float4*>(merge + (((to * MT + mt) * (DP / 8) + d) * 32 + lane) * 4) =
                make_float4(o[mt][d][0], o[mt][d][1], o[mt][d][2], o[mt][d][3]);
      }
      __syncthreads();
      if (warp < n) {
#pragma unroll
        for (int mt = 0; mt < MT; ++mt)
#pragma unroll
          for (int d = 0; d < DP / 8; ++d) {
            const float4 v = *reinterpret_cast<const float4*>(merge + (((warp * MT + mt) * (DP / 8) + d) * 32 + lane) * 4);
            o[mt][d][0] += v.x;
            o[mt][d][1] += v.y;
            o[mt][d][2] += v.z;
            o[mt][d][3] += v.w;
          }
      }
      __syncthreads();
    }
    if (warp == 0) {
#pragma unroll
      for (int mt = 0; mt < MT; ++mt)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int row = mt * 16 + lane / 4 + e * 8;
          if (row >= rows) continue;
          const float mx = m[mt][e];
          if (!whole) {
#pragma unroll
            for (int d = 0; d < DP / 8; ++d)
              if (d * 8 < dim)
                *reinterpret_cast<float2*>(reinterpret_cast<float*>(
                    a.part_o + (slot * (dim / 4) + 2 * d + ((lane & 3) >> 1)) * kRows + row) + (lane & 1) * 2) =
                    make_float2(o[mt][d][2 * e], o[mt][d][2 * e + 1]);
            if ((lane & 3) == 0) a.part_ml[slot * kRows + row] = make_float2(mx, z[mt][e]);
            continue;
          }
          const float top = fmaxf(mx, sink[mt][e]);
          const float ref = top == -INFINITY ? 0.f : top;
          const float f = mx == -INFINITY ? 0.f : mma::exp2_fast(mx - ref);
          const float den = z[mt][e] * f + (a.sinks ? mma::exp2_fast(sink[mt][e] - ref) : 0.f);
          const float g = pt[mt][e] >= 0 && z[mt][e] != 0.f ? f / den : 0.f;
#pragma unroll
          for (int d = 0; d < DP / 8; ++d)
            if (d * 8 < dim)
              *reinterpret_cast<uint32_t*>(a.out + at[mt][e] * dim + d * 8 + (lane & 3) * 2) =
                  g == 0.f ? 0u : pack_bf16x2(o[mt][d][2 * e] * g, o[mt][d][2 * e + 1] * g);
          if ((lane & 3) == 0 && a.lse) a.lse[at[mt][e]] = pt[mt][e] >= 0 ? ref * kLn2 + logf(den) : -INFINITY;
        }
    }
    if (!again) break;
    cw = nw;
    __syncthreads();
  }
  if constexpr (kTma) {
    if (lane == 0 && *(volatile int*)&abort_flag) record_status(a.c.status, BS_ERR_TIMEOUT);
  } else {
    ptx::cp_async_wait_all();
  }
}

// ---------------------------------------------------------------- many rows
// Row tiles of 128 on tcgen05: S = Q K^T (128 x 64 per half tile of keys, both
// operands in shared memory) into tensor memory, the weights P = 2^(x - m) back
// into the same columns as bf16, O += P V with P as the tensor-memory operand and
// V as it lies in the cache (keys along K, the head contiguous).
//
// Two pipelines per CTA.  With more than 128 rows to a kv head (kPair) they take two
// row tiles and share every K and V tile; with fewer they take alternate tiles of
// keys for the same rows, and both accumulators are read at the end of an item (same
// lanes of tensor memory).  A pipeline has two (heads of 128) or three (heads of 64)
// half tiles of S in tensor memory, so that products run ahead of the softmax; two
// groups of four softmax warps, a thread per row, that take its half tiles in turn;
// and a warp each that issues S and PV products.  One warp fetches K and V by TMA
// boxes of a page's slots into a ring of tiles.
//
// The groups of a pipeline settle a row's reference m half tile by half tile, in
// turn, through shared memory.  It only moves when a row's scores exceed it by 2^8:
// P stays far below the bf16 range, sums are fp32, and O is rarely rescaled.
//
// What bounds it: the softmax warps' issue slots and the special-function unit (16
// exponentials per clock and SM).  Steps that paid, 2 x 131072 keys, 16 drafts, heads
// of 64 (128 rows) / 8 x 16384 keys, 64 drafts, heads of 128, us: 16-byte
// copies 257 / 257; TMA boxes 170 / 246; products issued from a converged warp 136 /
// 202; half tiles of S ahead 125 / 156; starts of items counted in the split - / 110;
// two softmax groups and two issuing warps per pipeline 125 / 85; registers moved to
// the softmax warps, no spills 107 / 80.  82 and 37 us are the floors.
template <int DP>
struct TilesCfg {
  static constexpr int kSlot = 128 * DP * 2;             // a K or V tile, [DP / 64] panels of 128 rows x 128 bytes
  static constexpr int kSlots = DP == 64 ? 10 : 4;
  // tensor memory of pipeline p: S half tiles at p * kSCol, 64 columns each; O at kOCol + p * DP
  static constexpr int kBufs = DP == 64 ? 3 : 2;
  static constexpr uint32_t kSCol = 64 * kBufs, kOCol = 2 * kSCol;
  static constexpr int q = kSlots * kSlot;               // two Q tiles
  static constexpr int bits = q + 2 * kSlot;             // [512 threads][8 words]
  static constexpr int ml = bits + 512 * 32;             // [4 groups][128] float2
  static constexpr int mref = ml + 4 * 128 * 8;          // [2 pipelines][128] float
  static constexpr int bars = mref + 2 * 128 * 4;
  static constexpr int total = bars + 512 + 1024;        // barriers; alignment of the base
};
constexpr int kTileThreads = 768;  // 16 softmax warps, loader, four issuing warps, three idle
// Registers of a thread: 80 at launch; the softmax warps want more, and the other
// eight warps give it (512 * 96 + 256 * 48 = 768 * 80).
constexpr int kSoftmaxRegs = 96, kOtherRegs = 48;
constexpr float kRescale = 8.f;
// One pair of exponentials in so many runs on the FMA pipe.  2 x 131072 keys, 16
// drafts, heads of 64: 1/16 114.3 us, 1/8 115.4, 1/4 117.3; 8 x 16384 keys, 64
// drafts, heads of 128: 90.2, 90.5, 90.6.
constexpr int kPolyOf = 16;

// A K x N operand whose N extent is contiguous (64 values = 128 bytes per row
// of K, 128B-swizzled): 8-row groups 1024 bytes apart, 64-value panels `panel`.
__device__ __forceinline__ uint64_t sdesc_nmajor_sw128(uint32_t saddr, uint32_t panel) {
  return (uint64_t)((saddr & 0x3FFFFu) >> 4) | ((uint64_t)(panel >> 4) << 16) | ((uint64_t)(1024 >> 4) << 32) |
         (1ull << 46) | (2ull << 61);
}
// Bits of a 256-bit row starting at bit `at` (which may lie outside).
__device__ __forceinline__ uint32_t bits_from(const uint32_t* row, int at) {
  const int w = at >> 5, s = at & 31;
  const uint32_t lo = (unsigned)w < 8u ? row[w] : 0u;
  const uint32_t hi = (unsigned)(w + 1) < 8u ? row[w + 1] : 0u;
  return __funnelshift_r(lo, hi, s);
}
// Bits [a, b) of a word, a and b clamped to 0..32.
__device__ __forceinline__ uint32_t bit_range(int a, int b) {
  a = min(max(a, 0), 32);
  b = min(max(b, 0), 32);
  const uint32_t below_b = b == 32 ? 0xffffffffu : (1u << b) - 1u;
  const uint32_t below_a = a == 32 ? 0xffffffffu : (1u << a) - 1u;
  return below_b & ~below_a;
}

// Which drafts the rows of a warp's tokens may attend: a row of 256 bits (its
// first ceil(T / 32) words) written by the lane of each row to `row`.  Lanes hold
// consecutive rows, `tok` and its position `pt`; every lane calls.  The mask bytes
// of kBatch tokens and two words are loaded at once.
template <int kBatch>
__device__ __forceinline__ void draft_bits(const TreeArgs& a, int b, int n, int tok, int pt, uint32_t* row) {
  const int lane = threadIdx.x & 31;
  const int t0 = __shfl_sync(0xffffffffu, tok, 0), t1 = __reduce_max_sync(0xffffffffu, tok);
  const uint8_t* mask = a.mask ? a.mask + b * a.mask_b : nullptr;
#pragma unroll 1
  for (int i = 0; i < kMaxDrafts / 32; i += 2) {
    if (i * 32 >= a.T) {
      row[i] = row[i + 1] = 0;
      continue;
    }
    int u[2], pu[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      u[h] = (i + h) * 32 + lane;
      pu[h] = __ldg(a.pos + (int64_t)b * a.T + min(u[h], a.T - 1));
      if (u[h] >= a.T) pu[h] = -1;
    }
#pragma unroll 1
    for (int x = t0; x <= t1; x += kBatch) {
      uint32_t on[kBatch][2];
      if (mask) {  // loads without a condition, so that all are in flight together
#pragma unroll
        for (int j = 0; j < kBatch; ++j)
#pragma unroll
          for (int h = 0; h < 2; ++h) on[j][h] = __ldg(mask + (int64_t)min(x + j, t1) * a.T + min(u[h], a.T - 1));
      } else {
#pragma unroll
        for (int j = 0; j < kBatch; ++j)
#pragma unroll
          for (int h = 0; h < 2; ++h) on[j][h] = u[h] <= min(x + j, t1);
      }
#pragma unroll
      for (int j = 0; j < kBatch; ++j) {
        const int t = min(x + j, t1);
        const int px = __shfl_sync(0xffffffffu, pt, __ffs(__ballot_sync(0xffffffffu, tok == t)) - 1);
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const uint32_t v =
              __ballot_sync(0xffffffffu, on[j][h] && pu[h] >= 0 && px >= 0 && (!a.window || pu[h] > max(px, n) - a.window));
          if (tok == t) row[i + h] = v;
        }
      }
    }
  }
}

template <int DP, bool kPair>
__global__ void __launch_bounds__(kTileThreads, 1) tree_tiles_kernel(const __grid_constant__ TreeArgs a,
                                                                     const __grid_constant__ CacheMaps maps) {
  using Cfg = TilesCfg<DP>;
  constexpr int kU = 128, kRows = kPair ? 256 : 128;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
  __shared__ int64_t sums[6];
  __shared__ uint32_t tmem_at;
  __shared__ int abort_flag;
  __shared__ Range range;
  volatile int* abort = &abort_flag;
  const int tid = threadIdx.x, lane = tid & 31, warp = __shfl_sync(0xffffffffu, tid >> 5, 0);
  const uint32_t sbase = ptx::smem_addr(smem);
  const uint32_t bar = sbase + Cfg::bars;
  auto full = [&](int s) { return bar + 8 * s; };
  auto empty = [&](int s) { return bar + 8 * (Cfg::kSlots + s); };
  constexpr int kB = 16 * Cfg::kSlots;
  auto sfull = [&](int p, int buf) { return bar + kB + 24 * p + 8 * buf; };
  auto pready = [&](int p, int buf) { return bar + kB + 48 + 24 * p + 8 * buf; };
  auto pvdone = [&](int p, int buf) { return bar + kB + 96 + 24 * p + 8 * buf; };
  auto qfull = [&](int p) { return bar + kB + 144 + 8 * p; };
  auto odone = [&](int p) { return bar + kB + 160 + 8 * p; };
  auto meet = [&](int p) { return bar + kB + 176 + 8 * p; };
  auto drain = [&](int i) { return bar + kB + 192 + 8 * i; };
  auto turn = [&](int p, int w, int half) { return bar + kB + 224 + 64 * p + 16 * w + 8 * half; };
  static_assert(kB + 352 <= 512, "barriers");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");

  if (tid < 128) {
    const Range r = locate<kU>(a, blockIdx.x, gridDim.x, sums);
    if (tid == 0) range = r;
  } else if (warp == 18) {
    ptx::tmem_alloc(ptx::smem_addr(&tmem_at), 512);
    ptx::tmem_relinquish();
  } else if (tid == 128) {
    abort_flag = 0;
    for (int i = 0; i < Cfg::kSlots; ++i) {
      ptx::mbar_init(full(i), 1);
      ptx::mbar_init(empty(i), kPair ? 2 : 1);
    }
    for (int p = 0; p < 2; ++p) {
      for (int i = 0; i < Cfg::kBufs; ++i) {
        ptx::mbar_init(sfull(p, i), 1);
        ptx::mbar_init(pready(p, i), 128);
        ptx::mbar_init(pvdone(p, i), 1);
      }
      ptx::mbar_init(qfull(p), 256);
      ptx::mbar_init(meet(p), kPair ? 256 : 512);
      for (int w = 0; w < 4; ++w)
        for (int half = 0; half < 2; ++half) ptx::mbar_init(turn(p, w, half), 1);
      ptx::mbar_init(odone(p), 1);      // the last product of a piece
      ptx::mbar_init(drain(p), 1);
      ptx::mbar_init(drain(2 + p), 1);
    }
    ptx::fence_mbar_init();
  }
  __syncwarp();
  ptx::tc_fence_before();
  __syncthreads();
  ptx::tc_fence_after();
  const Range r = range;
  const uint32_t tmem = 0;  // all columns: they start at 0
  bool ok = true;

  if (r.p0 < r.p1) {
    int base = 0;  // tiles of the pieces before this one
    if (warp == 16) {
      // ------------------------------------------------ loader: lane g fetches the g-th box of a tile
      asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kOtherRegs));
      Walk w;
      bool more = walk_begin<kU>(a, r, w);
      const int boxes = kU / a.box;
      int page = 0, row = -1, i = more ? w.start : 0, s = 0;
      auto find = [&]() {
        row = -1;
        const int slot = w.k.lo + i * kU + lane * a.box;
        if (lane < boxes && slot < w.k.hi) {
          int p;
          a.c.div.split(slot, p, row);
          page = __ldg(a.c.table + w.b * a.c.table_stride + p);
        }
      };
      if (more) find();
      while (more && ok) {
        if (row >= 0 && (unsigned)page >= (unsigned)a.c.pages) {
          if (box_in_use(a, w.b, w.k.n, w.k.lo + i * kU + lane * a.box)) {
            record_status(a.c.status, BS_ERR_CAPACITY);
            page = page < 0 ? 0 : a.c.pages - 1;
          } else {
            row = -1;
          }
        }
        // a box behind the last slot lies outside the descriptor's pages: zeros
        const int y = w.h, x = row >= 0 ? page : a.c.pages, z = max(row, 0);
        if (++i == w.end) {
          more = walk_next<kU>(a, w);
          i = w.start;
        }
        if (more) find();  // while the copies below are issued
        for (int kv = 0; kv < 2 && ok; ++kv, ++s) {
          const int at = s % Cfg::kSlots;
          if (s >= Cfg::kSlots) ok = warp_wait(empty(at), (s / Cfg::kSlots - 1) & 1, abort);
          if (!ok) break;
          if (lane == 0) ptx::mbar_arrive_expect_tx(full(at), Cfg::kSlot);
          __syncwarp();
          if (lane < boxes) {
#pragma unroll
            for (int c = 0; c < DP / 64; ++c)
              ptx::tma_load_4d(sbase + at * Cfg::kSlot + c * 16384 + lane * a.box * 128, kv ? &maps.v : &maps.k, full(at),
                               c * 64, y, z, x);
          }
        }
      }
      // copies in flight end before the CTA's memory is given back, whichever warp gave up
      volatile int gone = 0;
      for (int k = max(0, s - Cfg::kSlots); k < s; ++k) ptx::mbar_wait(full(k % Cfg::kSlots), (k / Cfg::kSlots) & 1, &gone);
    } else if (warp >= 17 && warp < 21) {
      // ------------------------------------------------ MMA issue: S and PV of each pipeline have a
      // warp each.  One thread gets about one product or commit out per 95 cycles whatever its
      // size (32 to 64 cycles of the tensor pipe here), so four threads issue.  The whole warp
      // walks the loops and one elected thread issues.
      asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kOtherRegs));
      const int p = (warp - 17) & 1;
      constexpr int step = kPair ? 1 : 2;
      const int first = kPair ? 0 : p;
      constexpr int kBufs = Cfg::kBufs;
      const uint32_t s_col = p * Cfg::kSCol, o_col = Cfg::kOCol + p * DP;
      const bool elected = ptx::elect_one();
      Walk w;
      bool more = walk_begin<kU>(a, r, w);
      int halves = 0, pieces = 0, tiles = 0;  // half tiles and pieces of this pipeline, tiles of the CTA so far
      if (warp < 19) {
        constexpr uint32_t idesc = (1u << 4) | (1u << 7) | (1u << 10) | ((64u >> 3) << 17) | ((128u >> 4) << 24);
        const uint64_t qd = ptx::sdesc_kmajor_sw128(sbase + Cfg::q + p * Cfg::kSlot), kd0 = ptx::sdesc_kmajor_sw128(sbase);
        while (more && ok) {
          const int n = w.end - w.start, total = first < n ? 2 * ((n - first + step - 1) / step) : 0;
          if (total) {
            ok = warp_wait(qfull(p), pieces & 1, abort);
            ++pieces;
          }
          for (int h = 0; h < total && ok; ++h, ++halves) {
            const uint32_t ks = 2 * (tiles + first + (h >> 1) * step), ka = ks % Cfg::kSlots;
            if (!(h & 1)) ok = warp_wait(full(ka), (ks / Cfg::kSlots) & 1, abort);
            // the product that last read the weights in these columns has ended
            const uint32_t buf = (uint32_t)halves % kBufs, use = (uint32_t)halves / kBufs;
            if (use) ok = ok && warp_wait(pvdone(p, buf), (use - 1) & 1, abort);
            if (!ok) break;
            ptx::tc_fence_after();
            if (elected) {
              const uint64_t kd = kd0 + ka * (Cfg::kSlot >> 4) + (h & 1) * (8192 >> 4);
#pragma unroll
              for (int k = 0; k < DP / 16; ++k) {
                const uint32_t off = ((k >> 2) * 16384 + (k & 3) * 32) >> 4;
                ptx::mma_ss_bf16(s_col + buf * 64, qd + off, kd + off, idesc, k > 0);
              }
              ptx::tc_commit(sfull(p, buf));
              if (h & 1) ptx::tc_commit(empty(ka));
            }
            __syncwarp();
          }
          tiles += n;
          more = walk_next<kU>(a, w);
        }
      } else {
        constexpr uint32_t idesc = (1u << 4) | (1u << 7) | (1u << 10) | (1u << 16) /* B with N contiguous */ |
                                   (((uint32_t)DP >> 3) << 17) | ((128u >> 4) << 24);
        const uint64_t vd0 = sdesc_nmajor_sw128(sbase, 16384);
        while (more && ok) {
          const int n = w.end - w.start, total = first < n ? 2 * ((n - first + step - 1) / step) : 0;
          for (int h = 0; h < total && ok; ++h, ++halves) {
            const uint32_t vs = 2 * (tiles + first + (h >> 1) * step) + 1, va = vs % Cfg::kSlots;
            const uint32_t buf = (uint32_t)halves % kBufs, use = (uint32_t)halves / kBufs;
            ok = warp_wait(pready(p, buf), use & 1, abort);
            ok = ok && warp_wait(full(va), (vs / Cfg::kSlots) & 1, abort);
            if (!ok) break;
            ptx::tc_fence_after();
            if (elected) {
              const uint64_t vd = vd0 + va * (Cfg::kSlot >> 4) + (h & 1) * (8192 >> 4);
#pragma unroll
              for (int k = 0; k < 4; ++k)
                ptx::mma_ts_bf16(o_col, s_col + buf * 64 + k * 8, vd + k * 128, idesc, h > 0 || k > 0);
              ptx::tc_commit(pvdone(p, buf));
              if (h + 1 == total) ptx::tc_commit(odone(p));
              if (h & 1) ptx::tc_commit(empty(va));
            }
            __syncwarp();
          }
          tiles += n;
          more = walk_next<kU>(a, w);
        }
      }
      // products in flight end before tensor memory is given back, whichever warp gave up
      if (elected) {
        volatile int gone = 0;
        ptx::tc_commit(drain(warp - 17));
        ptx::mbar_wait(drain(warp - 17), 0, &gone);
      }
      __syncwarp();
    } else if (warp < 16) {
      // ------------------------------------------------ softmax, a thread per row; group `hp` of
      // pipeline p takes its even or odd half tiles
      asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kSoftmaxRegs));
      Walk w;
      bool more = walk_begin<kU>(a, r, w);
      const int p = warp >> 3, hp = (warp >> 2) & 1, t = tid & 127;
      const uint32_t lanes = (uint32_t)(warp & 3) << 21;  // lane offset in a tensor-memory address
      constexpr int kBufs = Cfg::kBufs;
      uint32_t* bits = reinterpret_cast<uint32_t*>(smem + Cfg::bits) + tid * 8;
      float2* ml = reinterpret_cast<float2*>(smem + Cfg::ml) + t;
      float* mref = reinterpret_cast<float*>(smem + Cfg::mref) + p * 128 + t;
      const uint32_t my_turn = turn(p, warp & 3, hp), other_turn = turn(p, warp & 3, hp ^ 1);
      constexpr int step = kPair ? 1 : 2;
      const int first = kPair ? 0 : p;
      int halves = 0, pieces = 0, meets = 0;  // half tiles and pieces of this pipeline so far
      int turns = 0;                          // references that this warp has settled
      while (more && ok) {
        const int n = w.end - w.start;
        const int row0 = w.tile * kRows + (kPair ? p * 128 : 0);
        const int rows = min(128, a.R - row0);  // may be negative: the second tile of a pair is empty
        const bool mine = t < rows, warp_on = (warp & 3) * 32 < rows;
        const int tok = mine ? (row0 + t) / a.G : 0, g = mine ? row0 + t - tok * a.G : 0;
        const int hq = w.h * a.G + g;
        const int pt = mine ? a.pos[(int64_t)w.b * a.T + tok] : -1;
        int below = -1;  // keys up to here are outside the row's window (a row not in use is zeroed at the end)
        float m = -INFINITY, z = 0.f;  // z of this group's halves, relative to the reference m that it last saw
        if (first < n) {
          // half of the row of Q, and which keys the row may attend; the loads of both are in flight together
          uint8_t* qs = smem + Cfg::q + p * Cfg::kSlot;
          constexpr int kMine = DP / 16;
          const int c0 = hp * kMine;
          const __nv_bfloat16* q = a.q + w.b * a.qb + tok * a.qt + (int64_t)hq * a.qh;
          uint4 v[kMine];
#pragma unroll
          for (int c = 0; c < kMine; ++c) v[c] = __ldg(reinterpret_cast<const uint4*>(q + min((c0 + c) * 8, a.c.dim - 8)));
          if (a.window) below = max(pt, w.k.n) - a.window;
          if (warp_on && w.k.lo + w.end * kU > w.k.n) draft_bits<8>(a, w.b, w.k.n, tok, pt, bits);
#pragma unroll
          for (int c = 0; c < kMine; ++c)
            *reinterpret_cast<uint4*>(qs + mma::tile_at<128>(t, c0 + c)) =
                mine && (c0 + c) * 8 < a.c.dim ? v[c] : make_uint4(0, 0, 0, 0);
          ptx::fence_proxy_async_smem();
          __syncwarp();
          ptx::mbar_arrive(qfull(p));
          const int total = 2 * ((n - first + step - 1) / step);
          for (int h = hp; h < total && ok; h += 2) {
            const int i = first + (h >> 1) * step, done = halves + h;
            const int tile0 = w.k.lo + (w.start + i) * kU, key0 = tile0 + hp * 64;
            const uint32_t buf = (uint32_t)done % kBufs, use = (uint32_t)done / kBufs;
            const uint32_t s_col = tmem + lanes + p * Cfg::kSCol + buf * 64;
            ok = warp_wait(sfull(p, buf), use & 1, abort);
            if (!ok) break;
            ptx::tc_fence_after();
            if (warp_on) {
              const bool slow = key0 + 64 > w.k.n || a.window || a.scale2 < 0.f;
              const float mul = slow ? 1.f : a.scale2;
              float s[32];
              // 32 columns of S (read again for the weights: tensor memory is nearer than
              // the registers that holding all would take)
              auto fetch = [&](int c) {
                ptx::tmem_ld_32x32b_x32(s_col + c * 32, reinterpret_cast<uint32_t*>(s));
                ptx::tmem_wait_ld();
                if (slow) {
                  const int k0 = key0 + c * 32;
                  const uint32_t see = bit_range(below + 1 - k0, w.k.n - k0) | bits_from(bits, k0 - w.k.n);
#pragma unroll
                  for (int e = 0; e < 32; ++e) s[e] = see >> e & 1 ? s[e] * a.scale2 : -INFINITY;
                }
              };
              float mx = -INFINITY;
#pragma unroll
              for (int c = 0; c < 2; ++c) {
                fetch(c);
                float top[8];
#pragma unroll
                for (int e = 0; e < 8; ++e) top[e] = fmaxf(mma::max3(s[e], s[e + 8], s[e + 16]), s[e + 24]);
                mx = fmaxf(mx, mma::max3(mma::max3(top[0], top[1], top[2]), mma::max3(top[3], top[4], top[5]),
                                         fmaxf(top[6], top[7])));
              }
              mx *= mul;
              // the groups of a pipeline settle the row's reference half tile by half tile, in turn
              float ref = -INFINITY;
              if (h > 0) {
                ok = warp_wait(other_turn, (turns + hp + 1) & 1, abort);
                if (!ok) break;
                ref = *mref;
              }
              const bool move = mx > ref + kRescale || (ref == -INFINITY && mx > -INFINITY);
              const float f = move ? mma::exp2_fast(ref - mx) : 1.f;  // 0 from -inf
              if (move) ref = mx;
              if (move || h == 0) *mref = ref;
              __syncwarp();
              if (lane == 0) ptx::mbar_arrive(my_turn);
              ++turns;
              if (h > 0 && __any_sync(0xffffffffu, move)) {
                const uint32_t last = done - 1;  // the product before this one
                ok = warp_wait(pvdone(p, last % kBufs), (last / kBufs) & 1, abort);
                if (!ok) break;
                ptx::tc_fence_after();
                const uint32_t o_col = tmem + lanes + Cfg::kOCol + p * DP;
#pragma unroll 1
                for (int c = 0; c < DP / 16; ++c) {
                  uint32_t o[16];
                  ptx::tmem_ld_32x32b_x16(o_col + c * 16, o);
                  ptx::tmem_wait_ld();
#pragma unroll
                  for (int e = 0; e < 16; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * f);
                  ptx::tmem_st_32x32b_x16(o_col + c * 16, o);
                }
              }
              if (ref != m) {
                z *= mma::exp2_fast(m - ref);  // z is 0 where m is -inf
                m = ref;
              }
              ref = ref == -INFINITY ? 0.f : ref;
              float2 sum[2] = {};
#pragma unroll
              for (int c = 0; c < 2; ++c) {
                fetch(c);
                uint32_t pk[16];
#pragma unroll
                for (int e = 0; e < 16; ++e) {
                  float2 x = mma::fma2(make_float2(s[2 * e], s[2 * e + 1]), mul, -ref);
                  if (e % kPolyOf == kPolyOf - 1) {
                    x = mma::exp2_poly(x);
                  } else {
                    x.x = mma::exp2_fast(x.x);
                    x.y = mma::exp2_fast(x.y);
                  }
                  sum[e & 1] = mma::add2(sum[e & 1], x);
                  pk[e] = pack_bf16x2(x.x, x.y);  // (the choice of bf16: at the top)
                }
                ptx::tmem_st_32x32b_x16(s_col + c * 16, pk);
              }
              sum[0] = mma::add2(sum[0], sum[1]);
              z += sum[0].x + sum[0].y;
            }
            if (hp == 0 && (tile0 < w.k.low || tile0 + kU > w.k.n)) {
              // the tile's boxes bring all their slots: those that hold no key become zeros in V
              const int vs = 2 * (base + i) + 1, va = vs % Cfg::kSlots;
              ok = warp_wait(full(va), (vs / Cfg::kSlots) & 1, abort);
              if (!ok) break;
              if (!holds_key(a, w.b, w.k, tile0 + t)) {
                uint8_t* row = smem + va * Cfg::kSlot + t * 128;
#pragma unroll
                for (int c = 0; c < DP / 8; ++c)
                  *reinterpret_cast<uint4*>(row + (c >> 3) * 16384 + (c & 7) * 16) = make_uint4(0, 0, 0, 0);
              }
              ptx::fence_proxy_async_smem();
              __syncwarp();
            }
            if (warp_on) ptx::tmem_wait_st();
            ptx::tc_fence_before();
            ptx::mbar_arrive(pready(p, buf));
          }
          halves += total;
        }
        if (!ok) break;
        // ---- end of the piece: read the accumulators
        if (first < n) {
          ok = warp_wait(odone(p), pieces & 1, abort);
          ++pieces;
        }
        if (!ok) break;
        // the groups' sums: of this pipeline, or of both where they hold the same rows
        ml[(2 * p + hp) * 128] = make_float2(m, z);
        ptx::tc_fence_before();
        ptx::mbar_arrive(meet(kPair ? p : 0));
        ok = warp_wait(meet(kPair ? p : 0), meets & 1, abort);
        if (!ok) break;
        ++meets;
        ptx::tc_fence_after();
        auto both = [&](int x) {
          const float2 u = ml[2 * x * 128], v = ml[(2 * x + 1) * 128];
          const float top = fmaxf(u.x, v.x);
          const float zz = (u.y == 0.f ? 0.f : u.y * mma::exp2_fast(u.x - top)) +
                           (v.y == 0.f ? 0.f : v.y * mma::exp2_fast(v.x - top));
          return make_float2(top, zz);
        };
        float f0 = 1.f, f1 = 0.f;
        if (kPair) {
          const float2 u = both(p);
          m = u.x, z = u.y;
        } else {
          const float2 u = both(0), v = both(1);
          m = fmaxf(u.x, v.x);
          f0 = u.x == -INFINITY ? 0.f : mma::exp2_fast(u.x - m);
          f1 = v.x == -INFINITY ? 0.f : mma::exp2_fast(v.x - m);
          z = u.y * f0 + v.y * f1;
        }
        const bool whole = w.whole();
        const int64_t slot = 2 * (int64_t)blockIdx.x + (w.start == 0 ? 1 : 0);
        const int dim = a.c.dim, row = (kPair ? p * 128 : 0) + t;
        const int64_t at = ((int64_t)w.b * a.T + tok) * a.Hkv * a.G + hq;
        const bool speaks = mine && hp == 0 && (kPair || p == 0);  // for the row
        float scale_o = 1.f;
        if (whole && mine) {
          const bool used = pt >= 0;
          const float sink = a.sinks ? a.sinks[hq] * kLog2e : -INFINITY;
          const float top = fmaxf(m, sink);
          const float ref = top == -INFINITY ? 0.f : top;
          const float f = m == -INFINITY ? 0.f : mma::exp2_fast(m - ref);
          const float den = z * f + (a.sinks ? mma::exp2_fast(sink - ref) : 0.f);
          scale_o = used && z != 0.f ? f / den : 0.f;
          if (a.lse && speaks) a.lse[at] = used ? ref * kLn2 + logf(den) : -INFINITY;
        }
        if (!whole && speaks) a.part_ml[slot * kRows + row] = make_float2(m, z);
        if (warp_on) {
          // columns of this group: half of its tile's, or a quarter of the shared tile's.
          // bf16 rows go through this thread's part of Q (no longer read) to be stored in lines.
          constexpr int kCols = kPair ? DP / 2 : DP / 4;
          const int c0 = kPair ? hp * kCols : (2 * p + hp) * kCols;
          uint8_t* stage = smem + Cfg::q + p * Cfg::kSlot;
          const int chunk0 = hp * (DP / 16);
#pragma unroll 1
          for (int c = 0; c < kCols; c += 16) {
            float x[16], y[16];
            ptx::tmem_ld_32x32b_x16(tmem + lanes + Cfg::kOCol + (kPair ? p * DP : 0) + c0 + c, reinterpret_cast<uint32_t*>(x));
            if (!kPair) ptx::tmem_ld_32x32b_x16(tmem + lanes + Cfg::kOCol + DP + c0 + c, reinterpret_cast<uint32_t*>(y));
            ptx::tmem_wait_ld();
#pragma unroll
            for (int e = 0; e < 16; ++e) {
              x[e] = f0 == 0.f ? 0.f : x[e] * f0;
              if (!kPair && f1 != 0.f) x[e] += y[e] * f1;
            }
            if (whole) {
#pragma unroll
              for (int j = 0; j < 2; ++j) {
                uint32_t pk[4];
#pragma unroll
                for (int e = 0; e < 4; ++e)
                  pk[e] = scale_o == 0.f ? 0u : pack_bf16x2(x[j * 8 + 2 * e] * scale_o, x[j * 8 + 2 * e + 1] * scale_o);
                *reinterpret_cast<uint4*>(stage + mma::tile_at<128>(t, chunk0 + c / 8 + j)) =
                    make_uint4(pk[0], pk[1], pk[2], pk[3]);
              }
            } else if (mine) {
#pragma unroll
              for (int j = 0; j < 4; ++j)
                if (c0 + c + j * 4 < dim)
                  a.part_o[(slot * (dim / 4) + (c0 + c) / 4 + j) * kRows + row] =
                      make_float4(x[j * 4], x[j * 4 + 1], x[j * 4 + 2], x[j * 4 + 3]);
            }
            __syncwarp();
          }
          if (whole) {
            constexpr int kChunks = kCols / 8, kAtOnce = 32 / kChunks;
#pragma unroll 2
            for (int j = 0; j < 32 / kAtOnce; ++j) {
              const int x = j * kAtOnce + lane / kChunks, chunk = lane % kChunks;
              const int64_t to = __shfl_sync(0xffffffffu, at, x);
              const bool on = __shfl_sync(0xffffffffu, (int)mine, x);
              const uint4 v = *reinterpret_cast<const uint4*>(stage + mma::tile_at<128>((warp & 3) * 32 + x, chunk0 + chunk));
              if (on && c0 + chunk * 8 < dim) *reinterpret_cast<uint4*>(a.out + to * dim + c0 + chunk * 8) = v;
            }
            __syncwarp();
          }
        }
        ptx::tc_fence_before();
        if (!kPair) {
          // the other pipeline's accumulator has been read before it is written again (a pair's
          // is only read by the two groups whose next Q its next product waits for)
          ptx::mbar_arrive(meet(0));
          ok = warp_wait(meet(0), meets & 1, abort);
          if (!ok) break;
          ++meets;
        }
        base += n;
        more = walk_next<kU>(a, w);
      }
      if (!ok) ptx::tmem_wait_st();
    } else {
      asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kOtherRegs));
    }
  }
  __syncwarp();
  if (!ok && lane == 0) record_status(a.c.status, BS_ERR_TIMEOUT);
  ptx::tc_fence_before();
  __syncthreads();
  if (warp == 18) {
    ptx::tc_fence_after();
    ptx::tmem_dealloc(tmem_at, 512);
  }
}

// Joins the pieces of the items that several CTAs share; a block takes kJoinRows rows
// and some groups of four columns of an item.  kSplit neighbouring lanes take every
// kSplit-th piece of one row and group (a fixed order of the sums, so equal results on
// every run).  Bound by latency: a lane asks for its pieces' maxima and outputs at once.
// One sequence of 8192 / 131072 keys, 8 kv heads, 37 pieces to an item: with the kernel
// before it 22.0 / 65 us where one lane took all pieces after their maxima, 13.0 / 54 so.
constexpr int kJoinRows = 8;
template <int kSplit>
struct JoinCfg {
  static constexpr int kCols = kSplit == 1 ? 16 : 8, kThreads = kJoinRows * kSplit * kCols;
};
template <int kU, int kRows, int kSplit>
__global__ void __launch_bounds__(JoinCfg<kSplit>::kThreads) tree_join_kernel(const __grid_constant__ TreeArgs a, int grid) {
  constexpr int kThreads = JoinCfg<kSplit>::kThreads, kWarps = kThreads / 32;
  __shared__ int64_t sums[2][kWarps];
  const int per = a.Hkv * a.tiles, tid = threadIdx.x;
  const int b = blockIdx.x / per, item = blockIdx.x - b * per;
  const int h = item / a.tiles, tile = item - h * a.tiles;
  // units before this sequence, and in all (the lengths are inputs of the first
  // launch too, so nothing of this waits for it)
  int64_t before = 0, total = 0;
  for (int i = tid; i < a.B; i += kThreads) {
    const int64_t w = units_of<kU>(a, i) * per;
    total += w;
    if (i < b) before += w;
  }
#pragma unroll
  for (int o = 16; o; o >>= 1) {
    before += __shfl_xor_sync(0xffffffffu, before, o);
    total += __shfl_xor_sync(0xffffffffu, total, o);
  }
  if ((tid & 31) == 0) sums[0][tid / 32] = before, sums[1][tid / 32] = total;
  __syncthreads();
  before = total = 0;
#pragma unroll
  for (int i = 0; i < kWarps; ++i) before += sums[0][i], total += sums[1][i];
  const int64_t units = units_of<kU>(a, b);
  const int64_t chunk = chunk_of(a, total, grid);
  const int64_t s = before + item * units, e = s + units;
  const int c0 = (int)((s + a.setup) / chunk), c1 = (int)((e - 1) / chunk);
  const int dim = a.c.dim, row0 = tile * kRows, rows = min(kRows, a.R - row0);
  const int row = blockIdx.y * kJoinRows + tid % kJoinRows, mine = min(row, rows - 1);
  const int part = tid / kJoinRows % kSplit, c = blockIdx.z * JoinCfg<kSplit>::kCols + tid / (kJoinRows * kSplit);
  const int t = (row0 + mine) / a.G, hq = h * a.G + row0 + mine - t * a.G;
  const bool used = c0 != c1 && a.pos[(int64_t)b * a.T + t] >= 0;
  const float sink = c0 != c1 && a.sinks ? a.sinks[hq] * kLog2e : -INFINITY;
  // every thread waits, so that this launch does not end before the first
  asm volatile("griddepcontrol.wait;" ::: "memory");
  if (c0 == c1) return;
  constexpr int kAhead = kSplit == 1 ? 4 : 10;
  const int col = min(c, dim / 4 - 1);
  auto slot = [&](int x) { return 2 * (int64_t)x + (x == c0); };
  float m = -INFINITY, z = 0.f;  // of this lane's pieces, and v relative to m
  float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int x = c0 + part; x <= c1; x += kAhead * kSplit) {
    float2 mz[kAhead];
    float4 p[kAhead];
#pragma unroll
    for (int j = 0; j < kAhead; ++j) {
      const int64_t at = slot(min(x + j * kSplit, c1));
      mz[j] = a.part_ml[at * kRows + mine];
      p[j] = a.part_o[(at * (dim / 4) + col) * kRows + mine];
    }
    float top = m;
#pragma unroll
    for (int j = 0; j < kAhead; ++j)
      if (x + j * kSplit <= c1) top = fmaxf(top, mz[j].x);
    const float ref = top == -INFINITY ? 0.f : top;
    const float f = mma::exp2_fast(m - ref);
    z *= f, v.x *= f, v.y *= f, v.z *= f, v.w *= f;
    m = top;
#pragma unroll
    for (int j = 0; j < kAhead; ++j) {
      if (x + j * kSplit > c1 || mz[j].y == 0.f) continue;
      const float g = mma::exp2_fast(mz[j].x - ref);
      z += mz[j].y * g, v.x += p[j].x * g, v.y += p[j].y * g, v.z += p[j].z * g, v.w += p[j].w * g;
    }
  }
  float mx = m;
#pragma unroll
  for (int o = kJoinRows; o < kJoinRows * kSplit; o <<= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
  const float top = fmaxf(mx, sink);
  const float ref = top == -INFINITY ? 0.f : top;
  const float f = m == -INFINITY ? 0.f : mma::exp2_fast(m - ref);
  z *= f, v.x *= f, v.y *= f, v.z *= f, v.w *= f;
#pragma unroll
  for (int o = kJoinRows; o < kJoinRows * kSplit; o <<= 1) {
    z += __shfl_xor_sync(0xffffffffu, z, o);
    v.x += __shfl_xor_sync(0xffffffffu, v.x, o);
    v.y += __shfl_xor_sync(0xffffffffu, v.y, o);
    v.z += __shfl_xor_sync(0xffffffffu, v.z, o);
    v.w += __shfl_xor_sync(0xffffffffu, v.w, o);
  }
  if (part || row >= rows || c >= dim / 4) return;
  const float den = z + (a.sinks ? mma::exp2_fast(sink - ref) : 0.f);
  uint2 w = make_uint2(0u, 0u);
  if (used && z != 0.f) w = make_uint2(pack_bf16x2(v.x / den, v.y / den), pack_bf16x2(v.z / den, v.w / den));
  const int64_t at = ((int64_t)b * a.T + t) * a.Hkv * a.G + hq;
  *reinterpret_cast<uint2*>(a.out + at * dim + c * 4) = w;
  if (c == 0 && a.lse) a.lse[at] = used ? ref * kLn2 + logf(den) : -INFINITY;
}

// Rows of a tile: 16 run on the kernel of few rows, 128 and 256 (a pair of tiles) on
// tcgen05, which needs TMA boxes; without them tiles of 32 (heads up to 64) serve all.
// 24 or 32 rows, heads of 64, in tiles of 32 on mma.sync and of 128 on tcgen05, us:
// 2 x 131072 keys 136 / 99, 8 x 8192 47 / 38, 64 ragged to 8192 162 / 131.  Where no more
// than kShortKeys are in reach, two tiles of 16 that read the keys twice end sooner: of
// 16 and of 128, 256 x 300 keys 91 / 125, 256 ragged to 1000 135 / 165, 64 x 600 38 / 47,
// 1 x 1000 11.5 / 13.1, 64 x 1000 55 / 56, but 64 x 2000 91 / 80.  (The reach is the page
// table's: behind one of 131072 slots 256 x 300 keys take 139, 64 x 900 60 instead of 53.)
// Without boxes and over heads of 64 the tiles stay at 16 rows (of 255 registers they take
// 241) and read the keys once for each: 64 rows of 128 over 4 x 8192 keys 130 us, 41 with boxes.
// The workspace is sized without the page size and the reach, for the largest.
constexpr int64_t kShortKeys = 1024;
int tile_rows(int64_t R, int64_t D, bool tma, int64_t reach) {
  if (R <= 16 || (!tma && D > 64) || (R <= 32 && D <= 64 && reach <= kShortKeys)) return 16;
  if (!tma) return 32;
  return R <= 128 ? 128 : 256;
}

template <int kU, int kRows, int kSplit>
int launch_join(const TreeArgs& a, int grid, cudaStream_t st) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(a.B * a.Hkv * a.tiles), (unsigned)cdiv(std::min(kRows, a.R), kJoinRows),
                     (unsigned)cdiv(a.c.dim / 4, JoinCfg<kSplit>::kCols));
  cfg.blockDim = dim3(JoinCfg<kSplit>::kThreads);
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  BS_CUDA(cudaLaunchKernelEx(&cfg, tree_join_kernel<kU, kRows, kSplit>, a, grid));
  return BS_OK;
}
template <int kU, int kRows>
int launch_join(const TreeArgs& a, int grid, cudaStream_t st) {
  if (a.fixed) return BS_OK;  // no item is cut
  // four lanes to a row's pieces where an item has more than four of them, about, unless
  // the blocks fill the GPU anyway (4 x 32768 keys, 32 tokens of 32 / 8 heads of 128: 118 us
  // with four lanes, 107 with one)
  const int64_t items = (int64_t)a.B * a.Hkv * a.tiles;
  const int64_t blocks = items * cdiv(std::min(kRows, a.R), kJoinRows) * cdiv(a.c.dim / 4, JoinCfg<1>::kCols);
  return grid > 4 * items && blocks <= 2 * sm_count() ? launch_join<kU, kRows, 4>(a, grid, st)
                                                       : launch_join<kU, kRows, 1>(a, grid, st);
}

template <int DP, int MT, bool kTma>
int launch_rows(TreeArgs& a, const CacheMaps& maps, int grid, cudaStream_t st) {
  constexpr int smem = RowsSmem<DP, MT>::total;
  static bool set[64] = {};
  int dev = 0;
  BS_CUDA(cudaGetDevice(&dev));
  if (dev >= 64 || !set[dev]) {
    BS_CUDA(cudaFuncSetAttribute(tree_rows_kernel<DP, MT, kTma>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
    if (dev < 64) set[dev] = true;
  }
  tree_rows_kernel<DP, MT, kTma><<<grid, 128, smem, st>>>(a, maps);
  BS_LAUNCHED();
  return launch_join<RowsCfg<DP>::kU, 16 * MT>(a, grid, st);
}

int grid_for(int rows, int64_t D) { return rows <= 32 ? rows_ctas(rows, D) * sm_count() : sm_count(); }

template <int DP, bool kPair>
int launch_tiles(TreeArgs& a, const CacheMaps& maps, int grid, cudaStream_t st) {
  constexpr int smem = TilesCfg<DP>::total;
  static bool set[64] = {};
  int dev = 0;
  BS_CUDA(cudaGetDevice(&dev));
  if (dev >= 64 || !set[dev]) {
    BS_CUDA(cudaFuncSetAttribute(tree_tiles_kernel<DP, kPair>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
    if (dev < 64) set[dev] = true;
  }
  tree_tiles_kernel<DP, kPair><<<grid, kTileThreads, smem, st>>>(a, maps);
  BS_LAUNCHED();
  return launch_join<128, kPair ? 256 : 128>(a, grid, st);
}

}  // namespace
}  // namespace bs

extern "C" size_t bs_tree_attention_workspace_bytes(int64_t B, int64_t T, int64_t Hq, int64_t Hkv, int64_t D) {
  using namespace bs;
  if (B <= 0 || T <= 0 || Hq <= 0 || Hkv <= 0 || D <= 0) return 0;
  int64_t most = 0;
  for (bool tma : {false, true})
    for (int64_t reach : {kShortKeys, kShortKeys + 1}) {
      const int rows = tile_rows(T * (Hq / Hkv), D, tma, reach);
      most = std::max(most, 2 * (int64_t)grid_for(rows, D) * rows * (D * 4 + 8));
    }
  return align_up((size_t)most, 256);
}

extern "C" int bs_tree_attention(const bs_heads* q, const bs_kv_cache* cache, int64_t T, int64_t Hq,
                                 const int32_t* positions, const void* mask, int64_t mask_stride_b,
                                 const float* sinks, int64_t window, float scale, void* out, float* lse,
                                 void* workspace, size_t workspace_bytes, void* stream) {
  using namespace bs;
  const char* fn = "bs_tree_attention";
  BS_ARG(q && cache, "%s: null pointer", fn);
  if (cache->batch == 0) return BS_OK;
  BS_ARG(q->ptr && positions && out, "%s: null pointer", fn);
  BS_ARG(T >= 1 && T <= kMaxDrafts, "%s: 1 to %d drafted tokens per sequence", fn, kMaxDrafts);
  TreeArgs a = {};
  BS_TRY(paged_cache(fn, cache, T, true, &a.c));
  BS_ARG(Hq > 0 && Hq % cache->heads == 0 && Hq <= 65535, "%s: query heads must be a multiple of the cache's heads", fn);
  BS_ARG(window >= 0, "%s: window must not be negative", fn);
  BS_ARG(mask_stride_b >= 0, "%s: negative mask stride", fn);
  BS_ALIGNED16(q->ptr, "q");
  BS_ALIGNED16(out, "out");
  BS_REQUIRE(q->stride_b % 8 == 0 && q->stride_t % 8 == 0 && q->stride_h % 8 == 0, BS_ERR_MISALIGNED,
             "%s: q strides must be multiples of 8 elements", fn);
  const int64_t D = cache->dim;
  const size_t need = bs_tree_attention_workspace_bytes(cache->batch, T, Hq, cache->heads, D);
  BS_REQUIRE(workspace && workspace_bytes >= need, BS_ERR_CAPACITY, "%s: workspace of %zu bytes, %zu needed", fn,
             workspace_bytes, need);
  BS_ALIGNED16(workspace, "workspace");
  a.q = static_cast<const __nv_bfloat16*>(q->ptr);
  a.qb = q->stride_b, a.qt = q->stride_t, a.qh = q->stride_h;
  a.pos = positions;
  a.mask = static_cast<const uint8_t*>(mask);
  a.mask_b = mask_stride_b;
  a.sinks = sinks;
  a.scale2 = scale * kLog2e;
  a.window = (int)std::min<int64_t>(window, 1 << 30);
  a.T = (int)T;
  a.Hkv = (int)cache->heads;
  a.G = (int)(Hq / cache->heads);
  a.R = a.T * a.G;
  a.B = (int)cache->batch;
  a.box = cache_box_rows(cache, 128);
  const bool tma = a.box >= 8;
  const int64_t reach = a.window ? std::min<int64_t>((int64_t)a.window - 1 + a.T + a.box - 1, a.c.capacity) : a.c.capacity;
  const int rows = tile_rows(a.R, D, tma, reach);
  a.tiles = (int)cdiv(a.R, (int64_t)rows);
  BS_ARG((int64_t)a.B * a.Hkv * a.tiles < INT32_MAX, "%s: sizes too large", fn);
  a.out = static_cast<__nv_bfloat16*>(out);
  a.lse = lse;
  const int grid = grid_for(rows, D);
  a.part_o = static_cast<float4*>(workspace);
  a.part_ml = reinterpret_cast<float2*>(a.part_o + (int64_t)2 * grid * rows * (D / 4));
  a.min_chunk = rows <= 32 ? 8 : 2;  // 4 / 6 / 8 units: 13.8 / 13.4 / 12.6 us at 1 x 8192 keys, the same elsewhere
  a.setup = rows <= 32 ? 16 : 8;
  // short ranges of keys (a window, a small cache): whole items to the CTAs, and no second launch
  const int unit = rows > 32 ? 128 : D <= 64 ? RowsCfg<64>::kU : RowsCfg<128>::kU;
  if (reach <= kWholeKeys) a.fixed = (int)cdiv(reach, (int64_t)unit);
  BS_TRY(check_device());
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  CacheMaps maps = {};
  if (tma) {
    if (rows <= 32) a.box = std::min(a.box, D <= 64 ? RowsCfg<64>::kU : RowsCfg<128>::kU);
    BS_TRY(cache_maps(cache, a.box, true, &maps));
  } else {
    a.box = 1;
  }
  if (rows == 128) return D <= 64 ? launch_tiles<64, false>(a, maps, grid, st) : launch_tiles<128, false>(a, maps, grid, st);
  if (rows == 256) return D <= 64 ? launch_tiles<64, true>(a, maps, grid, st) : launch_tiles<128, true>(a, maps, grid, st);
  if (D > 64) return tma ? launch_rows<128, 1, true>(a, maps, grid, st) : launch_rows<128, 1, false>(a, maps, grid, st);
  if (rows == 32) return launch_rows<64, 2, false>(a, maps, grid, st);
  return tma ? launch_rows<64, 1, true>(a, maps, grid, st) : launch_rows<64, 1, false>(a, maps, grid, st);
}
