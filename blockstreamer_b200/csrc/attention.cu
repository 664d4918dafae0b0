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
// Partial (m, z, O) of key ranges join by the same rule, in a fixed order.
//
// Work split: the keys of every (sequence, kv head, row tile) are cut into
// units; the units of all items, in item order, are cut into equal contiguous
// ranges, one per CTA, from the lengths on the device (no host read, no idle
// SMs for ragged batches or single sequences).  An item inside one range is
// finished there; the pieces of the others go to the workspace and a second
// launch (programmatic, so that its start overlaps) joins them.
#include "bs_paged.cuh"

namespace bs {

int paged_cache(const char* fn, const bs_kv_cache* c, int64_t extra, bool need_v, PagedCache* o) {
  BS_ARG(c->k && (c->v || !need_v) && c->page_table && c->lens, "%s: null pointer in the cache", fn);
  BS_ARG(c->pages > 0 && c->page_size > 0 && c->heads > 0 && c->table_width > 0 && c->batch >= 0, "%s: bad cache sizes", fn);
  BS_ARG(c->dim > 0 && c->dim <= 128 && c->dim % 8 == 0, "%s: the head size must be a multiple of 8 up to 128", fn);
  BS_ARG(c->pages < INT32_MAX && c->page_size < INT32_MAX && c->heads <= 65535 && c->batch < (1 << 24) &&
             c->table_width * c->page_size < INT32_MAX && c->table_stride >= 0,
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

namespace {

constexpr int kMaxDrafts = 256;
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;

struct TreeArgs {
  const __nv_bfloat16* q;
  int64_t qb, qt, qh;
  PagedCache c;
  const int32_t* pos;
  const uint8_t* mask;
  int64_t mask_b;
  const float* sinks;
  float scale2;  // scale * log2(e)
  int window, T, G, R, tiles, Hkv, B;
  __nv_bfloat16* out;
  float* lse;
  float* part_o;    // [2 * grid][tile rows][dim]
  float2* part_ml;  // [2 * grid][tile rows]
  int min_chunk;
};

// The key range of a sequence: [lo, n + T), n committed.
struct Keys {
  int n, lo, hi;
};
__device__ __forceinline__ Keys keys_of(const TreeArgs& a, int b) {
  Keys k;
  k.n = a.c.len(b, a.T);
  k.hi = k.n + a.T;
  k.lo = a.window ? max(0, k.n - a.window + 1) : 0;
  return k;
}

// Where the work of CTA `cta` of `grid` lies, units of kU keys: its range
// [p0, p1) and the first item in it.  Every thread of a 128-thread CTA calls.
struct Range {
  int64_t p0, p1, chunk;
  int b;           // sequence of unit p0
  int64_t before;  // units of the sequences before b
};
template <int kU>
__device__ __forceinline__ int64_t units_of(const TreeArgs& a, int b) {
  const Keys k = keys_of(a, b);
  return (k.hi - k.lo + kU - 1) / kU;
}
template <int kU>
__device__ Range locate(const TreeArgs& a, int cta, int grid, int64_t* sums /* smem [6] */) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t per = (int64_t)a.Hkv * a.tiles;
  int64_t total = 0;
  for (int b = threadIdx.x; b < a.B; b += 128) total += units_of<kU>(a, b) * per;
#pragma unroll
  for (int o = 16; o; o >>= 1) total += __shfl_xor_sync(0xffffffffu, total, o);
  if (lane == 0) sums[warp] = total;
  __syncthreads();
  total = sums[0] + sums[1] + sums[2] + sums[3];
  Range r;
  r.chunk = max((int64_t)a.min_chunk, (total + grid - 1) / grid);
  r.p0 = min(total, cta * r.chunk);
  r.p1 = min(total, r.p0 + r.chunk);
  r.b = 0;
  r.before = 0;
  if (r.p0 >= r.p1) return r;
  // the sequence that holds unit p0: a scan of the sequences' units, 128 at a time
  int64_t run = 0;
  for (int base = 0; base < a.B && run <= r.p0; base += 128) {
    const int b = base + threadIdx.x;
    const int64_t w = b < a.B ? units_of<kU>(a, b) * per : 0;
    int64_t incl = w;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int64_t v = __shfl_up_sync(0xffffffffu, incl, o);
      if (lane >= o) incl += v;
    }
    __syncthreads();
    if (lane == 31) sums[warp] = incl;
    __syncthreads();
    int64_t start = run + incl - w;
    for (int i = 0; i < warp; ++i) start += sums[i];
    run += sums[0] + sums[1] + sums[2] + sums[3];
    if (w > 0 && start <= r.p0 && r.p0 < start + w) sums[4] = b, sums[5] = start;
  }
  __syncthreads();
  r.b = (int)sums[4];
  r.before = sums[5];
  return r;
}

// ---------------------------------------------------------------- few rows
// Row tiles of MT * 16 rows on mma.sync, four warps per CTA, each streaming its
// own units of kU keys (16-byte asynchronous copies, kStages units per warp, no
// barrier between warps) and holding its own (m, z, O); they meet at the end of
// an item.  HBM-bound: 148 SMs x 2 CTAs x 4 warps keep ~190 KB per SM in flight.
template <int DP>
struct RowsCfg {
  static constexpr int kU = DP <= 64 ? 32 : 16;
  static constexpr int kStages = DP == 96 || DP == 32 ? 4 : 3;
  static constexpr int kTile = kU * DP * 2;           // bytes of a K (or V) unit
  static constexpr int kWarpBytes = 2 * kTile * kStages;
};
template <int DP, int MT>
struct RowsSmem {
  static constexpr int kRows = 16 * MT;
  static constexpr int stages = 0;
  static constexpr int merge = 4 * RowsCfg<DP>::kWarpBytes;
  static constexpr int ml = merge + kRows * DP * 4;            // [4 warps][rows] float2
  static constexpr int bits = ml + 4 * kRows * 8;              // [rows][8] words
  static constexpr int thr = bits + kRows * (kMaxDrafts / 32) * 4;
  static constexpr int sums = (thr + kRows * 4 + 15) / 16 * 16;
  static constexpr int total = sums + 64;
};

// The units of a CTA's range as one warp meets them (it takes every fourth
// unit of each item's piece).
struct Walk {
  int b, h, tile;
  Keys k;
  int u, end;      // next unit of this warp; end of the piece, in units of the item
  int64_t pos;     // global index of the piece's first unit
  int start;       // first unit of the piece
  int units;       // units of the item
};
template <int kU>
__device__ __forceinline__ void walk_piece(const TreeArgs& a, Walk& w, int64_t pos, int64_t p1, int first) {
  w.units = (w.k.hi - w.k.lo + kU - 1) / kU;
  w.pos = pos;
  w.start = first;
  w.end = (int)min((int64_t)w.units, first + (p1 - pos));
}
template <int kU>
__device__ __forceinline__ void walk_begin(const TreeArgs& a, const Range& r, Walk& w) {
  w.b = r.b;
  w.k = keys_of(a, r.b);
  const int units = (w.k.hi - w.k.lo + kU - 1) / kU;
  const int64_t rel = r.p0 - r.before;
  const int item = (int)(rel / units);
  w.h = item / a.tiles;
  w.tile = item - w.h * a.tiles;
  walk_piece<kU>(a, w, r.p0, r.p1, (int)(rel - (int64_t)item * units));
}
// The next piece of the range; false at its end.
template <int kU>
__device__ __forceinline__ bool walk_next(const TreeArgs& a, int64_t p1, Walk& w) {
  const int64_t pos = w.pos + (w.end - w.start);
  if (pos >= p1) return false;
  if (++w.tile == a.tiles) {
    w.tile = 0;
    if (++w.h == a.Hkv) {
      w.h = 0;
      ++w.b;
      w.k = keys_of(a, w.b);
    }
  }
  walk_piece<kU>(a, w, pos, p1, 0);
  return true;
}

template <int DP, int MT>
__global__ void __launch_bounds__(128, 2) tree_rows_kernel(const __grid_constant__ TreeArgs a) {
  using Cfg = RowsCfg<DP>;
  using Sm = RowsSmem<DP, MT>;
  constexpr int kU = Cfg::kU, KS = DP / 16, NT = kU / 8, kRows = 16 * MT, kWords = kMaxDrafts / 32;
  extern __shared__ __align__(1024) uint8_t smem[];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  float* merge = reinterpret_cast<float*>(smem + Sm::merge);
  float2* ml = reinterpret_cast<float2*>(smem + Sm::ml);
  uint32_t* bits = reinterpret_cast<uint32_t*>(smem + Sm::bits);
  int* thr = reinterpret_cast<int*>(smem + Sm::thr);
  const uint32_t base = ptx::smem_addr(smem) + warp * Cfg::kWarpBytes;
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");

  // columns dim..DP are zeros that no copy touches
  if (a.c.dim < DP) {
    for (int i = threadIdx.x; i < 4 * Cfg::kWarpBytes / 16; i += 128)
      reinterpret_cast<uint4*>(smem)[i] = make_uint4(0, 0, 0, 0);
    __syncthreads();
  }
  const Range r = locate<kU>(a, blockIdx.x, gridDim.x, reinterpret_cast<int64_t*>(smem + Sm::sums));
  if (r.p0 >= r.p1) return;

  // ---- loading: lane l < kU holds where row l of the next unit lies
  Walk lw;
  walk_begin<kU>(a, r, lw);
  lw.u = lw.start + warp;
  bool more = true;
  int next_page = 0, next_row = -1;  // row < 0: zeros
  auto find = [&]() {
    while (more && lw.u >= lw.end) {
      more = walk_next<kU>(a, r.p1, lw);
      lw.u = lw.start + warp;
    }
    next_row = -1;
    if (!more || lane >= kU) return;
    const int slot = lw.k.lo + lw.u * kU + lane;
    bool on = slot < lw.k.hi;
    if (on && slot >= lw.k.n) on = a.pos[(int64_t)lw.b * a.T + slot - lw.k.n] >= 0;
    if (on) {
      int p;
      a.c.div.split(slot, p, next_row);
      next_page = a.c.page_of(lw.b, p);
    }
  };
  constexpr int kLanesRow = DP <= 64 ? 8 : 16;  // lanes that copy one row
  auto load = [&](int stage) {
    if (more) {
      const uint32_t kd = base + stage * 2 * Cfg::kTile, vd = kd + Cfg::kTile;
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
          const uint32_t at = mma::tile_at<DP>(row, c);
          const bool on = x >= 0;
          mma::cp_async_16_or_zero(kd + at, on ? kb + p * a.c.kp + x * a.c.ks : kb, on);
          mma::cp_async_16_or_zero(vd + at, on ? vb + p * a.c.vp + x * a.c.vs : vb, on);
        }
      }
      lw.u += 4;
      find();
    }
    ptx::cp_async_commit();
  };
  find();
#pragma unroll
  for (int s = 0; s < Cfg::kStages - 1; ++s) load(s);

  // ---- pieces
  Walk cw;
  walk_begin<kU>(a, r, cw);
  int stage = 0;
  while (true) {
    const int row0 = cw.tile * kRows, rows = min(kRows, a.R - row0);
    const int t0 = row0 / a.G, toks = (row0 + rows - 1) / a.G - t0 + 1;
    // masks of the tile's tokens over the drafts, and each one's window
    {
      const int words = (a.T + 31) / 32;
      const int32_t* pos = a.pos + (int64_t)cw.b * a.T;
      for (int i = warp; i < toks * words; i += 4) {
        const int tl = i / words, w = i - tl * words, t = t0 + tl, u = w * 32 + lane;
        const int pt = pos[t];
        const int below = a.window ? max(pt, cw.k.n) - a.window : -1;
        bool on = false;
        if (pt >= 0 && u < a.T) {
          const int pu = pos[u];
          on = pu >= 0 && (!a.window || pu > below) &&
               (a.mask ? a.mask[cw.b * a.mask_b + (int64_t)t * a.T + u] != 0 : u <= t);
        }
        const uint32_t m = __ballot_sync(0xffffffffu, on);
        if (lane == 0) {
          bits[tl * kWords + w] = m;
          if (w == 0) thr[tl] = pt >= 0 ? below : INT_MAX;
        }
      }
    }
    uint32_t qf[MT][KS][4];
#pragma unroll
    for (int mt = 0; mt < MT; ++mt)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int row = mt * 16 + lane / 4 + e * 8;
        const bool on = row < rows;
        const int t = on ? (row0 + row) / a.G : 0, g = on ? row0 + row - t * a.G : 0;
        const __nv_bfloat16* q = a.q + cw.b * a.qb + t * a.qt + (int64_t)(cw.h * a.G + g) * a.qh + (lane & 3) * 2;
#pragma unroll
        for (int k = 0; k < KS; ++k)
#pragma unroll
          for (int half = 0; half < 2; ++half) {
            const int col = k * 16 + half * 8;
            qf[mt][k][e + 2 * half] =
                on && col < a.c.dim ? __ldg(reinterpret_cast<const uint32_t*>(q + col)) : 0u;
          }
      }
    int tl[MT][2];
#pragma unroll
    for (int mt = 0; mt < MT; ++mt)
#pragma unroll
      for (int e = 0; e < 2; ++e)
        tl[mt][e] = (row0 + min(mt * 16 + lane / 4 + e * 8, rows - 1)) / a.G - t0;
    __syncthreads();

    float m[MT][2], z[MT][2], o[MT][DP / 8][4];
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
      m[mt][0] = m[mt][1] = -INFINITY;
      z[mt][0] = z[mt][1] = 0.f;
#pragma unroll
      for (int d = 0; d < DP / 8; ++d) o[mt][d][0] = o[mt][d][1] = o[mt][d][2] = o[mt][d][3] = 0.f;
    }
    for (int u = cw.start + warp; u < cw.end; u += 4) {
      ptx::cp_async_wait<Cfg::kStages - 2>();
      __syncwarp();
      const uint32_t kt = base + stage * 2 * Cfg::kTile, vt = kt + Cfg::kTile;
      load((stage + Cfg::kStages - 1) % Cfg::kStages);
      stage = stage + 1 == Cfg::kStages ? 0 : stage + 1;

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
          mma::ldsm_x4(kt + mma::tile_at<DP>(np * 16 + (lane >> 4) * 8 + (lane & 7), 2 * k + ((lane >> 3) & 1)), f);
#pragma unroll
          for (int mt = 0; mt < MT; ++mt) {
            mma::bf16_16816(s[mt][2 * np], qf[mt][k], f[0], f[1]);
            mma::bf16_16816(s[mt][2 * np + 1], qf[mt][k], f[2], f[3]);
          }
        }
      const int slot0 = cw.k.lo + u * kU;
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
            p[nt][e] = pack_bf16x2(y0, y1);
          }
          z[mt][e] = z[mt][e] * f + sum;
#pragma unroll
          for (int d = 0; d < DP / 8; ++d) {
            o[mt][d][2 * e] *= f;
            o[mt][d][2 * e + 1] *= f;
          }
        }
#pragma unroll
        for (int j = 0; j < kU / 16; ++j) {
          const uint32_t pf[4] = {p[2 * j][0], p[2 * j][1], p[2 * j + 1][0], p[2 * j + 1][1]};
#pragma unroll
          for (int dp = 0; dp < DP / 16; ++dp) {
            uint32_t f[4];
            mma::ldsm_x4_trans(vt + mma::tile_at<DP>(j * 16 + ((lane >> 3) & 1) * 8 + (lane & 7), 2 * dp + (lane >> 4)), f);
            mma::bf16_16816(o[mt][2 * dp], pf, f[0], f[1]);
            mma::bf16_16816(o[mt][2 * dp + 1], pf, f[2], f[3]);
          }
        }
      }
    }

    // ---- the warps' parts meet: common maximum, then their O in warp order
#pragma unroll
    for (int mt = 0; mt < MT; ++mt)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
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
        float mx = -INFINITY;
        for (int w = 0; w < 4; ++w) mx = fmaxf(mx, ml[w * kRows + row].x);
        const float f = mx == -INFINITY ? 0.f : mma::exp2_fast(m[mt][e] - mx);
#pragma unroll
        for (int d = 0; d < DP / 8; ++d) {
          o[mt][d][2 * e] *= f;
          o[mt][d][2 * e + 1] *= f;
        }
      }
    for (int w = 0; w < 4; ++w) {
      if (warp == w) {
#pragma unroll
        for (int mt = 0; mt < MT; ++mt)
#pragma unroll
          for (int e = 0; e < 2; ++e)
#pragma unroll
            for (int d = 0; d < DP / 8; ++d) {
              float2* at = reinterpret_cast<float2*>(merge + (mt * 16 + lane / 4 + e * 8) * DP + d * 8 + (lane & 3) * 2);
              float2 v = w ? *at : make_float2(0.f, 0.f);
              v.x += o[mt][d][2 * e];
              v.y += o[mt][d][2 * e + 1];
              *at = v;
            }
      }
      __syncthreads();
    }
    const bool whole = cw.start == 0 && cw.end == cw.units;
    const int64_t slot = 2 * (int64_t)blockIdx.x + (cw.start == 0 ? 1 : 0);
    const int dim = a.c.dim;
    for (int i = threadIdx.x; i < rows * (dim / 8); i += 128) {
      const int row = i / (dim / 8), c = i - row * (dim / 8);
      float mx = -INFINITY, zz = 0.f;
      for (int w = 0; w < 4; ++w) mx = fmaxf(mx, ml[w * kRows + row].x);
      for (int w = 0; w < 4; ++w) {
        const float2 v = ml[w * kRows + row];
        if (v.x > -INFINITY) zz += v.y * mma::exp2_fast(v.x - mx);
      }
      const float4 v0 = *reinterpret_cast<const float4*>(merge + row * DP + c * 8);
      const float4 v1 = *reinterpret_cast<const float4*>(merge + row * DP + c * 8 + 4);
      if (!whole) {
        float* po = a.part_o + (slot * kRows + row) * dim + c * 8;
        *reinterpret_cast<float4*>(po) = v0;
        *reinterpret_cast<float4*>(po + 4) = v1;
        if (c == 0) a.part_ml[slot * kRows + row] = make_float2(mx, zz);
        continue;
      }
      const int t = (row0 + row) / a.G, h = cw.h * a.G + row0 + row - t * a.G;
      const int64_t at = ((int64_t)cw.b * a.T + t) * a.Hkv * a.G + h;
      const bool used = a.pos[(int64_t)cw.b * a.T + t] >= 0;
      float sink = a.sinks ? a.sinks[h] * kLog2e : -INFINITY;
      const float top = fmaxf(mx, sink);
      const float ref = top == -INFINITY ? 0.f : top;
      const float f = mx == -INFINITY ? 0.f : mma::exp2_fast(mx - ref);
      const float den = zz * f + (a.sinks ? mma::exp2_fast(sink - ref) : 0.f);
      const float g = used && mx > -INFINITY ? f / den : 0.f;
      uint4 w;
      w.x = pack_bf16x2(g == 0.f ? 0.f : v0.x * g, g == 0.f ? 0.f : v0.y * g);
      w.y = pack_bf16x2(g == 0.f ? 0.f : v0.z * g, g == 0.f ? 0.f : v0.w * g);
      w.z = pack_bf16x2(g == 0.f ? 0.f : v1.x * g, g == 0.f ? 0.f : v1.y * g);
      w.w = pack_bf16x2(g == 0.f ? 0.f : v1.z * g, g == 0.f ? 0.f : v1.w * g);
      *reinterpret_cast<uint4*>(a.out + at * dim + c * 8) = w;
      if (c == 0 && a.lse) a.lse[at] = used ? ref * kLn2 + logf(den) : -INFINITY;
    }
    if (!walk_next<kU>(a, r.p1, cw)) break;
    __syncthreads();
  }
  ptx::cp_async_wait_all();
}

// Joins the pieces of the items that several CTAs share, in CTA order.
template <int kU, int kRows>
__global__ void __launch_bounds__(128) tree_join_kernel(const __grid_constant__ TreeArgs a, int grid) {
  __shared__ int64_t sums[8];
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int per = a.Hkv * a.tiles;
  const int b = blockIdx.x / per, item = blockIdx.x - b * per;
  const int h = item / a.tiles, tile = item - h * a.tiles;
  // units before this sequence, and in all
  int64_t before = 0, total = 0;
  for (int i = threadIdx.x; i < a.B; i += 128) {
    const Keys k = keys_of(a, i);
    const int64_t w = (int64_t)((k.hi - k.lo + kU - 1) / kU) * per;
    total += w;
    if (i < b) before += w;
  }
#pragma unroll
  for (int o = 16; o; o >>= 1) {
    before += __shfl_xor_sync(0xffffffffu, before, o);
    total += __shfl_xor_sync(0xffffffffu, total, o);
  }
  if ((threadIdx.x & 31) == 0) sums[threadIdx.x / 32] = before, sums[4 + threadIdx.x / 32] = total;
  __syncthreads();
  before = sums[0] + sums[1] + sums[2] + sums[3];
  total = sums[4] + sums[5] + sums[6] + sums[7];
  const Keys k = keys_of(a, b);
  const int64_t units = (k.hi - k.lo + kU - 1) / kU;
  const int64_t chunk = max((int64_t)a.min_chunk, (total + grid - 1) / grid);
  const int64_t s = before + item * units, e = s + units;
  const int c0 = (int)(s / chunk), c1 = (int)((e - 1) / chunk);
  if (c0 == c1) return;
  const int dim = a.c.dim, row0 = tile * kRows, rows = min(kRows, a.R - row0);
  for (int i = threadIdx.x; i < rows * (dim / 4); i += 128) {
    const int row = i / (dim / 4), c = i - row * (dim / 4);
    float mx = -INFINITY;
    for (int x = c0; x <= c1; ++x) mx = fmaxf(mx, a.part_ml[(2 * (int64_t)x + (x == c0)) * kRows + row].x);
    const int t = (row0 + row) / a.G, hq = h * a.G + row0 + row - t * a.G;
    const bool used = a.pos[(int64_t)b * a.T + t] >= 0;
    const float sink = a.sinks ? a.sinks[hq] * kLog2e : -INFINITY;
    const float top = fmaxf(mx, sink);
    const float ref = top == -INFINITY ? 0.f : top;
    float den = a.sinks ? mma::exp2_fast(sink - ref) : 0.f;
    float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int x = c0; x <= c1; ++x) {
      const int64_t at = (2 * (int64_t)x + (x == c0)) * kRows + row;
      const float2 mz = a.part_ml[at];
      if (mz.x == -INFINITY) continue;
      const float f = mma::exp2_fast(mz.x - ref);
      den += mz.y * f;
      const float4 p = *reinterpret_cast<const float4*>(a.part_o + at * dim + c * 4);
      v.x += p.x * f;
      v.y += p.y * f;
      v.z += p.z * f;
      v.w += p.w * f;
    }
    const int64_t at = ((int64_t)b * a.T + t) * a.Hkv * a.G + hq;
    const bool any = used && mx > -INFINITY;
    uint2 w = make_uint2(0u, 0u);
    if (any) w = make_uint2(pack_bf16x2(v.x / den, v.y / den), pack_bf16x2(v.z / den, v.w / den));
    *reinterpret_cast<uint2*>(a.out + at * dim + c * 4) = w;
    if (c == 0 && a.lse) a.lse[at] = used ? ref * kLn2 + logf(den) : -INFINITY;
  }
}

int tile_rows(int64_t R, int64_t D) { return R <= 16 || D > 64 ? 16 : 32; }

template <int DP, int MT>
int launch_rows(TreeArgs& a, int grid, cudaStream_t st) {
  constexpr int smem = RowsSmem<DP, MT>::total;
  static bool set[64] = {};
  int dev = 0;
  BS_CUDA(cudaGetDevice(&dev));
  if (dev >= 64 || !set[dev]) {
    BS_CUDA(cudaFuncSetAttribute(tree_rows_kernel<DP, MT>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
    if (dev < 64) set[dev] = true;
  }
  tree_rows_kernel<DP, MT><<<grid, 128, smem, st>>>(a);
  BS_LAUNCHED();
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(a.B * a.Hkv * a.tiles));
  cfg.blockDim = dim3(128);
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  BS_CUDA(cudaLaunchKernelEx(&cfg, tree_join_kernel<RowsCfg<DP>::kU, 16 * MT>, a, grid));
  return BS_OK;
}

int grid_for(int64_t) { return 2 * sm_count(); }

}  // namespace
}  // namespace bs

extern "C" size_t bs_tree_attention_workspace_bytes(int64_t B, int64_t T, int64_t Hq, int64_t Hkv, int64_t D) {
  using namespace bs;
  if (B <= 0 || T <= 0 || Hq <= 0 || Hkv <= 0 || D <= 0) return 0;
  const int64_t rows = tile_rows(T * (Hq / Hkv), D);
  return align_up((size_t)(2 * (int64_t)grid_for(D) * rows * (D * 4 + 8)), 256);
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
  const int rows = tile_rows(a.R, D);
  a.tiles = (int)cdiv(a.R, (int64_t)rows);
  BS_ARG((int64_t)a.B * a.Hkv * a.tiles < INT32_MAX, "%s: sizes too large", fn);
  a.out = static_cast<__nv_bfloat16*>(out);
  a.lse = lse;
  const int grid = grid_for(D);
  a.part_o = static_cast<float*>(workspace);
  a.part_ml = reinterpret_cast<float2*>(a.part_o + (int64_t)2 * grid * rows * D);
  a.min_chunk = 4;
  BS_TRY(check_device());
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  if (D <= 32) return rows == 16 ? launch_rows<32, 1>(a, grid, st) : launch_rows<32, 2>(a, grid, st);
  if (D <= 64) return rows == 16 ? launch_rows<64, 1>(a, grid, st) : launch_rows<64, 2>(a, grid, st);
  if (D <= 96) return launch_rows<96, 1>(a, grid, st);
  return launch_rows<128, 1>(a, grid, st);
}
