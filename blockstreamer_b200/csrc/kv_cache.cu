// Upkeep of the paged key/value cache between decoding steps: the accepted
// drafts moved together, the attention weight that each cached key received
// added to its score, and the keys of lowest score evicted.
#include <type_traits>

#include "bs_paged.cuh"
#include "bs_ring.cuh"

namespace bs {
namespace {

constexpr float kLog2e = 1.4426950408889634f;

// ---------------------------------------------------------------- commit
// One CTA per (sequence, kv head): all accepted rows are read before any is
// written (slot n + i may itself be the source of an earlier row).  Bound by the
// launch and one round trip: 5 of 16 drafts, 8 heads of 64: 2.7 us for one sequence,
// 3.2 for 64.
__global__ void __launch_bounds__(256) tree_commit_kernel(const __grid_constant__ PagedCache c, int T,
                                                          const int32_t* __restrict__ accepted, int A) {
  extern __shared__ __align__(16) uint4 rows[];
  __shared__ int count, bad;
  const int b = blockIdx.x / c.heads, h = blockIdx.x - b * c.heads;
  const int32_t* acc = accepted + (int64_t)b * A;
  if (threadIdx.x == 0) count = 0, bad = 0;
  __syncthreads();
  for (int i = threadIdx.x; i < A; i += blockDim.x) {
    const int u = acc[i];
    if (u < 0) continue;
    atomicMax(&count, i + 1);
    if (u >= T || (i > 0 && acc[i - 1] >= u) || (i > 0 && acc[i - 1] < 0)) bad = 1;
  }
  __syncthreads();
  if (bad) {
    if (threadIdx.x == 0) record_status(c.status, BS_ERR_INVALID_ARGUMENT);
    return;
  }
  // nothing is written through a clamped index: a sequence whose length is bad stays as it is,
  // and so does a slot that its own or its source's page would leave the pool for
  const int n = c.lens[b], per = c.dim / 8, items = 2 * count * per;
  if (n < 0 || n > c.capacity - T) {
    if (threadIdx.x == 0) record_status(c.status, BS_ERR_CAPACITY);
    return;
  }
  auto at = [&](int i, int row) -> __nv_bfloat16* {
    const int col = i % per * 8, v = i / per & 1;
    int page, in;
    c.div.split(n + row, page, in);
    const int p = __ldg(c.table + b * c.table_stride + page);
    if ((unsigned)p >= (unsigned)c.pages) {
      record_status(c.status, BS_ERR_CAPACITY);
      return nullptr;
    }
    return v ? c.v + p * c.vp + in * c.vs + h * c.vh + col : c.k + p * c.kp + in * c.ks + h * c.kh + col;
  };
  uint32_t found = 0;  // which of the thread's pieces were read (32 at most: 2 * 256 rows of 128 by 256 threads)
  for (int i = threadIdx.x, j = 0; i < items; i += blockDim.x, ++j) {
    const __nv_bfloat16* from = at(i, acc[i / (2 * per)]);
    if (from) rows[i] = *reinterpret_cast<const uint4*>(from), found |= 1u << j;
  }
  __syncthreads();
  for (int i = threadIdx.x, j = 0; i < items; i += blockDim.x, ++j) {
    if (acc[i / (2 * per)] == i / (2 * per) || !(found >> j & 1)) continue;
    if (__nv_bfloat16* to = at(i, i / (2 * per))) *reinterpret_cast<uint4*>(to) = rows[i];
  }
}

// ---------------------------------------------------------------- scores
// K is the 16-row operand of the tensor-core product and the accepted rows its
// columns, so that a key's sum over the rows stays in one lane group: no atomics,
// one store per slot.  HBM-bound: 2 dim + 8 bytes per slot and kv head (32 sequences,
// 149 MB: 32 us, 4.7 TB/s, of which about 5 are the launch, the search for the CTA's
// range and the first keys' way; 537 MB of 2 x 131072 keys: 90 us, 6.0 TB/s).  The
// slots of all (sequence, kv head) items are cut into equal ranges, one per CTA;
// each warp streams its own units of 32 or 64 keys through its own ring (TMA boxes where
// the pages allow, else 16-byte copies), the rows' queries are in shared memory.
struct ScoreArgs : SplitArgs {  // T: accepted entries; slots lens + i belong to them
  const __nv_bfloat16* q;
  int64_t qb, qt, qh;
  const float* lse;
  const int32_t* accepted;
  const float* scores;
  float* out;
  float scale2;
  int tokens, i0, rows, G, Hq, capacity;  // this launch: accepted entries i0 .. i0 + rows / G
};

template <int DP>
struct ScoreCfg {
  static constexpr int kU = DP == 64 ? 64 : 32;
  static constexpr int kStages = 3;
  static constexpr int kTile = kU * DP * 2;
  static constexpr int kWarpBytes = kTile * kStages;
  static constexpr int bars = 4 * kWarpBytes;            // [4 warps][kStages]
  static constexpr int sums = bars + 4 * kStages * 8;
  static constexpr int q = (sums + 64 + 127) / 128 * 128;  // [rows] q, [rows] float2
  static int smem(int rows) { return q + rows * (DP * 2 + 8) + 1024; }
};

// Whether a slot from `slot` on has a row that sees it.  Asked where its page lies outside
// the pool: the page table may hold anything behind the accepted tokens.
__device__ __forceinline__ bool seen_from(const ScoreArgs& a, int b, int n, int slot) {
  bool any = slot < n;
#pragma unroll 1
  for (int i = max(slot - n, 0); i < a.T && !any; ++i)
    any = !a.accepted || (unsigned)__ldg(a.accepted + (int64_t)b * a.T + i) < (unsigned)a.tokens;
  return any;
}

// Behind an item's last unit scores are only copied: an equal share of the whole array
// for the one warp of each CTA that does it.
template <int kU>
__device__ __forceinline__ void copy_rest(const ScoreArgs& a, int lane) {
  if (a.out == a.scores) return;
  const int64_t all = (int64_t)a.B * a.Hkv * a.capacity, share = (all + gridDim.x - 1) / gridDim.x;
  const int64_t end = min(all, (blockIdx.x + 1) * share);
  int64_t from = blockIdx.x * share;
  int item = (int)(from / a.capacity);
  for (; from < end; ++item) {
    const int64_t first = (int64_t)item * a.capacity, to = min(end, first + a.capacity);
    const int n = a.c.len(item / a.Hkv, a.T) + a.T;
    const int64_t begin = max(from, first + min(a.capacity, (n + kU - 1) / kU * kU));
    for (int64_t i = begin + lane; i < to; i += 16 * 32) {
      float v[16];
#pragma unroll
      for (int j = 0; j < 16; ++j) v[j] = a.scores[min(i + j * 32, all - 1)];
#pragma unroll
      for (int j = 0; j < 16; ++j)
        if (i + j * 32 < to) a.out[i + j * 32] = v[j];
    }
    from = to;
  }
}

constexpr int kScoreThreads = 160;  // four warps of keys, and one that copies

template <int DP, bool kTma>
__global__ void __launch_bounds__(kScoreThreads, 2) kv_scores_kernel(const __grid_constant__ ScoreArgs a,
                                                        const __grid_constant__ CacheMaps maps) {
  using Cfg = ScoreCfg<DP>;
  constexpr int kU = Cfg::kU, KS = DP / 16, MT = kU / 16, kMine = kU / 32;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
  __shared__ int abort_flag;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int rows8 = (a.rows + 7) / 8 * 8;
  const uint32_t base = ptx::smem_addr(smem) + warp * Cfg::kWarpBytes;
  const uint32_t bar = ptx::smem_addr(smem) + Cfg::bars + warp * Cfg::kStages * 8;
  uint8_t* qs = smem + Cfg::q;
  float2* info = reinterpret_cast<float2*>(qs + rows8 * DP * 2);  // (lse log2(e), last slot seen)
  auto qat = [&](int r, int c) { return (uint32_t)((c >> 3) * (rows8 * 128) + r * 128 + (((c & 7) ^ (r & 7)) << 4)); };

  if constexpr (kTma) {
    if (threadIdx.x == 0) abort_flag = 0;
    if (lane == 0 && warp < 4) {
      for (int s = 0; s < Cfg::kStages; ++s) ptx::mbar_init(bar + 8 * s, 1);
      ptx::fence_mbar_init();
    }
  } else if (a.c.dim < DP) {
    for (int i = threadIdx.x; i < 4 * Cfg::kWarpBytes / 16; i += kScoreThreads)
      reinterpret_cast<uint4*>(smem)[i] = make_uint4(0, 0, 0, 0);
  }
  __syncthreads();
  if (warp == 4) {
    copy_rest<kU>(a, lane);
    return;
  }
  const Range r = locate<kU>(a, blockIdx.x, gridDim.x, reinterpret_cast<int64_t*>(smem + Cfg::sums));
  Walk lw, cw;
  bool more = r.p0 < r.p1 && walk_begin<kU>(a, r, lw);
  const bool any = more;
  cw = lw;

  // ---- loading: lane g holds where the next unit's g-th box (or slot) lies
  const int box = kTma ? a.box : 1, boxes = kU / box;
  if (any) lw.u = lw.start + warp;
  Ring<Cfg::kStages> ring;
  int next_page[kMine] = {}, next_row[kMine];  // row < 0: no key there
  auto find = [&]() {
    while (more && lw.u >= lw.end) {
      more = walk_next<kU>(a, lw);
      lw.u = lw.start + warp;
    }
#pragma unroll
    for (int e = 0; e < kMine; ++e) {
      next_row[e] = -1;
      const int g = lane + 32 * e, slot = lw.u * kU + g * box;
      if (more && g < boxes && slot < lw.k.hi) {
        int p;
        a.c.div.split(slot, p, next_row[e]);
        next_page[e] = __ldg(a.c.table + lw.b * a.c.table_stride + p);
      }
    }
  };
  auto load = [&](int stage) {
    if (more) {
      const uint32_t kd = base + stage * Cfg::kTile;
#pragma unroll
      for (int e = 0; e < kMine; ++e)
        if (next_row[e] >= 0 && (unsigned)next_page[e] >= (unsigned)a.c.pages) {
          if (seen_from(a, lw.b, lw.k.n, lw.u * kU + (lane + 32 * e) * box)) {
            record_status(a.c.status, BS_ERR_CAPACITY);
            next_page[e] = next_page[e] < 0 ? 0 : a.c.pages - 1;
          } else {
            next_row[e] = -1;
          }
        }
      if constexpr (kTma) {  // at most kU / 8 <= 32 boxes: the first of a lane's places
        if (lane == 0) ptx::mbar_arrive_expect_tx(bar + 8 * stage, Cfg::kTile);
        __syncwarp();
        if (lane < boxes) {
          // a box behind the last slot lies outside the descriptor's pages: zeros
          const int page = next_row[0] >= 0 ? next_page[0] : a.c.pages, row = max(next_row[0], 0);
#pragma unroll
          for (int x = 0; x < DP / 64; ++x)
            ptx::tma_load_4d(kd + x * (kU * 128) + lane * box * 128, &maps.k, bar + 8 * stage, x * 64, lw.h, row, page);
        }
      } else {
        constexpr int kLanesRow = DP / 8;
        const int c = lane % kLanesRow;
        const __nv_bfloat16* kb = a.c.k + lw.h * a.c.kh + c * 8;
#pragma unroll
        for (int i = 0; i < kU * kLanesRow / 32; ++i) {
          const int row = lane / kLanesRow + i * (32 / kLanesRow);
          const int e = i * (32 / kLanesRow) / 32;  // the same for all lanes
          const int p = __shfl_sync(0xffffffffu, next_page[e], row & 31), x = __shfl_sync(0xffffffffu, next_row[e], row & 31);
          if (c * 8 < a.c.dim)
            mma::cp_async_16_or_zero(kd + mma::tile_at<kU>(row, c), x >= 0 ? kb + p * a.c.kp + x * a.c.ks : kb, x >= 0);
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
  const uint32_t qaddr = ptx::smem_addr(qs);
  const int mine = lane / 4 + (lane & 3) * 8;  // the slots of a unit that this lane stores: mine, mine + 32

  while (any) {
    const int64_t row0 = ((int64_t)cw.b * a.Hkv + cw.h) * a.capacity;
    // the scores to add to are asked for one unit ahead
    const int top = a.out != a.scores ? a.capacity : min(a.capacity, cw.k.hi);
    float next[kMine];
    auto ask = [&](int u) {
#pragma unroll
      for (int e = 0; e < kMine; ++e) next[e] = __ldg(a.scores + row0 + min(u * kU + mine + 32 * e, a.capacity - 1));
    };
    ask(cw.start + warp);
    // the token of row r, or -1: the loads below do not wait for one another
    auto token = [&](int r) -> int {
      const int e = a.i0 + min(r, a.rows - 1) / a.G, u = a.accepted ? __ldg(a.accepted + (int64_t)cw.b * a.T + e) : e;
      return r < a.rows && (unsigned)u < (unsigned)a.tokens ? u : -1;
    };
#pragma unroll 4
    for (int i = threadIdx.x; i < rows8 * (DP / 8); i += 128) {
      const int r = i / (DP / 8), c = i - r * (DP / 8), u = token(r), hq = cw.h * a.G + r % a.G;
      const bool on = u >= 0 && c * 8 < a.c.dim;
      mma::cp_async_16_or_zero(qaddr + qat(r, c), on ? a.q + cw.b * a.qb + u * a.qt + hq * a.qh + c * 8 : a.q, on);
    }
    for (int r = threadIdx.x; r < rows8; r += 128) {
      const int u = token(r), hq = cw.h * a.G + r % a.G;
      const float l = u >= 0 ? a.lse[((int64_t)cw.b * a.tokens + u) * a.Hq + hq] : -INFINITY;
      info[r] = l != -INFINITY ? make_float2(l * kLog2e, __int_as_float(cw.k.n + a.i0 + r / a.G))
                               : make_float2(INFINITY, __int_as_float(-1));
    }
    ptx::cp_async_commit();
    ptx::cp_async_wait_all();
    sync128();
    for (int u = cw.start + warp; u < cw.end; u += 4) {
      const int slot0 = u * kU;
      float before[kMine];
#pragma unroll
      for (int e = 0; e < kMine; ++e) before[e] = next[e];
      ask(u + 4);
      const uint32_t kt = base + ring.stage * Cfg::kTile;
      if constexpr (kTma)
        // (a wait that ran out is reported at the end)
        more = ring.take([&](int s, int parity, bool again) {
          volatile int gone = 0;
          return warp_wait(bar + 8 * s, parity, again ? &gone : &abort_flag);
        }) && more;
      else
        ptx::cp_async_wait<Cfg::kStages - 2>();
      __syncwarp();
      load(ring.place(more));
      ring.next();
      uint32_t kf[MT][KS][4];
#pragma unroll
      for (int mt = 0; mt < MT; ++mt)
#pragma unroll
        for (int k = 0; k < KS; ++k)
          mma::ldsm_x4(kt + mma::tile_at<kU>(mt * 16 + (lane & 15), 2 * k + (lane >> 4)), kf[mt][k]);
      float sum[2 * MT] = {};  // slots slot0 + lane / 4 + 8 i
      // eight rows at a time, or twice eight whose chains of products run side by side
      auto add_rows = [&](int r, auto blocks) {
        constexpr int N = decltype(blocks)::value;
        float s[N][MT][4] = {};
#pragma unroll
        for (int k = 0; k < KS; k += 2) {
          uint32_t f[N][4];
#pragma unroll
          for (int x = 0; x < N; ++x) mma::ldsm_x4(qaddr + qat(r + 8 * x + (lane & 7), 2 * k + (lane >> 3)), f[x]);
#pragma unroll
          for (int half = 0; half < 4; half += 2)
#pragma unroll
            for (int x = 0; x < N; ++x)
#pragma unroll
              for (int mt = 0; mt < MT; ++mt) mma::bf16_16816(s[x][mt], kf[mt][k + half / 2], f[x][half], f[x][half + 1]);
        }
#pragma unroll
        for (int x = 0; x < N; ++x) {
          const float2 f0 = info[r + 8 * x + (lane & 3) * 2], f1 = info[r + 8 * x + (lane & 3) * 2 + 1];
#pragma unroll
          for (int mt = 0; mt < MT; ++mt)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const float2 f = e & 1 ? f1 : f0;
              const int key = slot0 + mt * 16 + lane / 4 + (e >> 1) * 8;
              const float p = mma::exp2_fast(s[x][mt][e] * a.scale2 - f.x);
              sum[mt * 2 + (e >> 1)] += key <= __float_as_int(f.y) ? p : 0.f;
            }
        }
      };
      int r = 0;
      for (; r + 16 <= rows8; r += 16) add_rows(r, std::integral_constant<int, 2>());
      if (r < rows8) add_rows(r, std::integral_constant<int, 1>());
#pragma unroll
      for (int i = 0; i < 2 * MT; ++i) {
        sum[i] += __shfl_xor_sync(0xffffffffu, sum[i], 1);
        sum[i] += __shfl_xor_sync(0xffffffffu, sum[i], 2);
      }
      const int sel = lane & 3;
#pragma unroll
      for (int e = 0; e < kMine; ++e) {
        const float* t = sum + 4 * e;
        const float add = sel == 0 ? t[0] : sel == 1 ? t[1] : sel == 2 ? t[2] : t[3];
        if (slot0 + mine + 32 * e < top) a.out[row0 + slot0 + mine + 32 * e] = before[e] + add;
      }
    }
    if (!walk_next<kU>(a, cw)) break;
    sync128();
  }
  if constexpr (kTma) {
    if (lane == 0 && *(volatile int*)&abort_flag) record_status(a.c.status, BS_ERR_TIMEOUT);
  } else {
    ptx::cp_async_wait_all();
  }
}

// ---------------------------------------------------------------- scores, many rows
// Tiles of 128 keys against up to 256 rows: S = K Q^T is one tcgen05 product per 16
// values of the head, K the 128-row operand, so that a thread of the epilogue holds one
// key and adds up its weights over the rows alone.  Four groups of four warps take the
// tiles in turn, a quarter of tensor memory each.
//
// HBM-bound up to about 64 rows (dim 128: 537 MB of 2 x 131072 keys in 89 us, 6.0 TB/s),
// then by the exponentials, 16 a clock and SM (128 rows, dim 64: 268 million in 85 us, 70%
// of that; 121 us with two groups, 89 with the comparison at every weight, 101 with a
// quarter of the exponentials on the FMA pipe).  More than 128 rows take several launches.
constexpr int kScoreGroups = 4;       // of four warps that each take a tile
constexpr int kScoreWarps = 4 * kScoreGroups;
constexpr int kScoreTileThreads = 32 * (kScoreWarps + 3);  // and loader, issuer, copier
constexpr int kScoreRows = 128;       // of a launch

template <int DP>
struct ScoreTilesCfg {
  static constexpr int kSlot = 128 * DP * 2;
  static constexpr int kSlots = DP == 64 ? 8 : 4;
  static constexpr int q = kSlots * kSlot;               // [rows16] x DP, panels of 64 values
  static constexpr int info = q + kScoreRows * DP * 2;   // [rows] -lse log2(e), [rows] last slot seen
  static constexpr int bars = info + kScoreRows * 8;
  static constexpr int total = bars + 512 + 1024;
};

template <int DP>
__global__ void __launch_bounds__(kScoreTileThreads, 1) kv_scores_tiles_kernel(const __grid_constant__ ScoreArgs a,
                                                                               const __grid_constant__ CacheMaps maps) {
  using Cfg = ScoreTilesCfg<DP>;
  constexpr int kU = 128;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
  __shared__ int64_t sums[6];
  __shared__ uint32_t tmem_at;
  __shared__ int abort_flag;
  __shared__ Range range;
  __shared__ __align__(8) uint8_t all_on[kScoreRows / 16];  // whether 16 rows all count
  volatile int* abort = &abort_flag;
  const int tid = threadIdx.x, lane = tid & 31, warp = __shfl_sync(0xffffffffu, tid >> 5, 0);
  const uint32_t sbase = ptx::smem_addr(smem), bar = sbase + Cfg::bars;
  auto full = [&](int s) { return bar + 8 * s; };
  auto empty = [&](int s) { return bar + 64 + 8 * s; };
  auto sfull = [&](int b) { return bar + 128 + 8 * b; };
  auto sempty = [&](int b) { return bar + 160 + 8 * b; };
  const uint32_t qfull = bar + 192, meet = bar + 200, drain = bar + 208;
  const int rows16 = (a.rows + 15) / 16 * 16;
  constexpr int bufs = 4, stride = 512 / bufs;  // of S in tensor memory

  if (tid < 128) {
    const Range r = locate<kU>(a, blockIdx.x, gridDim.x, sums);
    if (tid == 0) range = r;
  } else if (warp == kScoreWarps + 1) {
    ptx::tmem_alloc(ptx::smem_addr(&tmem_at), 512);
    ptx::tmem_relinquish();
  } else if (tid == 128) {
    abort_flag = 0;
    for (int i = 0; i < Cfg::kSlots; ++i) {
      ptx::mbar_init(full(i), 1);
      ptx::mbar_init(empty(i), 1);
    }
    for (int i = 0; i < 4; ++i) {
      ptx::mbar_init(sfull(i), 1);
      ptx::mbar_init(sempty(i), 4);
    }
    ptx::mbar_init(qfull, 32 * kScoreWarps);
    ptx::mbar_init(meet, 32 * kScoreWarps);
    ptx::mbar_init(drain, 1);
    ptx::fence_mbar_init();
  }
  __syncwarp();
  ptx::tc_fence_before();
  __syncthreads();
  ptx::tc_fence_after();
  const Range r = range;
  bool ok = true;

  if (warp == kScoreWarps + 2) {
    copy_rest<kU>(a, lane);
  } else if (r.p0 < r.p1) {
    Walk w;
    bool more = walk_begin<kU>(a, r, w);
    int tiles = 0;  // of the pieces before this one
    if (warp == kScoreWarps) {
      // ------------------------------------------------ loader: lane g fetches the g-th box of a tile
      const int boxes = kU / a.box;
      int page = 0, row = -1, i = more ? w.start : 0, s = 0;
      auto find = [&]() {
        row = -1;
        const int slot = i * kU + lane * a.box;
        if (lane < boxes && slot < w.k.hi) {
          int p;
          a.c.div.split(slot, p, row);
          page = __ldg(a.c.table + w.b * a.c.table_stride + p);
        }
      };
      if (more) find();
      for (; more; ++s) {
        if (row >= 0 && (unsigned)page >= (unsigned)a.c.pages) {
          if (seen_from(a, w.b, w.k.n, i * kU + lane * a.box)) {
            record_status(a.c.status, BS_ERR_CAPACITY);
            page = page < 0 ? 0 : a.c.pages - 1;
          } else {
            row = -1;
          }
        }
        // a box behind the last slot lies outside the descriptor's pages: zeros
        const int y = w.h, x = row >= 0 ? page : a.c.pages, z = max(row, 0), at = s % Cfg::kSlots;
        if (++i == w.end) {
          more = walk_next<kU>(a, w);
          i = w.start;
        }
        if (more) find();
        if (s >= Cfg::kSlots) ok = warp_wait(empty(at), (s / Cfg::kSlots - 1) & 1, abort);
        if (!ok) break;
        if (lane == 0) ptx::mbar_arrive_expect_tx(full(at), Cfg::kSlot);
        __syncwarp();
        if (lane < boxes) {
#pragma unroll
          for (int c = 0; c < DP / 64; ++c)
            ptx::tma_load_4d(sbase + at * Cfg::kSlot + c * 16384 + lane * a.box * 128, &maps.k, full(at), c * 64, y, z, x);
        }
      }
      // copies in flight end before the CTA's memory is given back, whichever warp gave up
      volatile int gone = 0;
      for (int k = max(0, s - Cfg::kSlots); k < s; ++k) ptx::mbar_wait(full(k % Cfg::kSlots), (k / Cfg::kSlots) & 1, &gone);
    } else if (warp == kScoreWarps + 1) {
      // ------------------------------------------------ MMA issue, by one elected thread
      const uint32_t idesc = ptx::idesc_bf16_f32(128, rows16);
      const uint64_t qd = ptx::sdesc_kmajor_sw128(sbase + Cfg::q), kd0 = ptx::sdesc_kmajor_sw128(sbase);
      const uint32_t qpanel = rows16 * 128;
      const bool elected = ptx::elect_one();
      for (int pieces = 0; more && ok; ++pieces) {
        const int n = w.end - w.start;
        ok = warp_wait(qfull, pieces & 1, abort);
        for (int t = tiles; t < tiles + n && ok; ++t) {
          const int at = t % Cfg::kSlots, buf = t & (bufs - 1), use = t / bufs;
          ok = warp_wait(full(at), (t / Cfg::kSlots) & 1, abort);
          if (use) ok = ok && warp_wait(sempty(buf), (use - 1) & 1, abort);
          if (!ok) break;
          ptx::tc_fence_after();
          if (elected) {
            const uint64_t kd = kd0 + at * (Cfg::kSlot >> 4);
#pragma unroll
            for (int k = 0; k < DP / 16; ++k)
              ptx::mma_ss_bf16(buf * stride, kd + (((k >> 2) * 16384 + (k & 3) * 32) >> 4),
                               qd + (((k >> 2) * qpanel + (k & 3) * 32) >> 4), idesc, k > 0);
            ptx::tc_commit(empty(at));
            ptx::tc_commit(sfull(buf));
          }
          __syncwarp();
        }
        tiles += n;
        more = walk_next<kU>(a, w);
      }
      // products in flight end before tensor memory is given back, whichever warp gave up
      if (elected) {
        volatile int gone = 0;
        ptx::tc_commit(drain);
        ptx::mbar_wait(drain, 0, &gone);
      }
      __syncwarp();
    } else {
      // ------------------------------------------------ a thread per key
      const float2 scale = make_float2(a.scale2, a.scale2);
      const int group = warp >> 2, key0 = (warp & 3) * 32 + lane;
      const uint32_t lanes = (uint32_t)(warp & 3) << 21;  // lane offset in a tensor-memory address
      uint8_t* qs = smem + Cfg::q;
      float* shift = reinterpret_cast<float*>(smem + Cfg::info);
      int* last = reinterpret_cast<int*>(shift + kScoreRows);
      for (int pieces = 0; more && ok; ++pieces) {
        const int n = w.end - w.start;
        const int64_t row0 = ((int64_t)w.b * a.Hkv + w.h) * a.capacity;
        const int top = a.out != a.scores ? a.capacity : min(a.capacity, w.k.hi);
        auto ask = [&](int i) { return __ldg(a.scores + row0 + min(i * kU + key0, a.capacity - 1)); };
        int i = w.start + ((group - tiles) & (kScoreGroups - 1));  // this group's first tile
        float next = ask(i);
        if (pieces) {  // the rows of the piece before are no longer read
          ptx::mbar_arrive(meet);
          ok = warp_wait(meet, (pieces - 1) & 1, abort);
          if (!ok) break;
        }
        auto token = [&](int x) -> int {
          const int e = a.i0 + min(x, a.rows - 1) / a.G, u = a.accepted ? __ldg(a.accepted + (int64_t)w.b * a.T + e) : e;
          return x < a.rows && (unsigned)u < (unsigned)a.tokens ? u : -1;
        };
#pragma unroll 4
        for (int j = tid; j < rows16 * (DP / 8); j += 32 * kScoreWarps) {
          const int x = j / (DP / 8), c = j - x * (DP / 8), u = token(x), hq = w.h * a.G + x % a.G;
          const bool on = u >= 0 && c * 8 < a.c.dim;
          mma::cp_async_16_or_zero(ptx::smem_addr(qs) + (c >> 3) * (rows16 * 128) + x * 128 + (((c & 7) ^ (x & 7)) << 4),
                                   on ? a.q + w.b * a.qb + u * a.qt + hq * a.qh + c * 8 : a.q, on);
        }
        if (tid < kScoreRows) {
          const int u = token(tid), hq = w.h * a.G + tid % a.G;
          const float l = u >= 0 ? a.lse[((int64_t)w.b * a.tokens + u) * a.Hq + hq] : -INFINITY;
          const bool on = l != -INFINITY;
          shift[tid] = on ? -l * kLog2e : -INFINITY;
          last[tid] = on ? w.k.n + a.i0 + tid / a.G : -1;
          const uint32_t rows_on = __ballot_sync(0xffffffffu, on);
          if (lane == 0) all_on[2 * warp] = (rows_on & 0xffffu) == 0xffffu, all_on[2 * warp + 1] = rows_on >> 16 == 0xffffu;
        }
        ptx::cp_async_commit();
        ptx::cp_async_wait_all();
        ptx::fence_proxy_async_smem();
        ptx::mbar_arrive(qfull);
        ok = warp_wait(qfull, pieces & 1, abort);
        const uint64_t plain = *reinterpret_cast<const uint64_t*>(all_on);
        for (; i < w.end && ok; i += kScoreGroups) {
          const int t = tiles + i - w.start, buf = t & (bufs - 1), key = i * kU + key0;
          const float before = next;
          next = ask(i + kScoreGroups);
          ok = warp_wait(sfull(buf), (t / bufs) & 1, abort);
          if (!ok) break;
          ptx::tc_fence_after();
          const uint32_t col = buf * stride + lanes;
          uint32_t v[2][16];
          float2 sum = make_float2(0.f, 0.f);
          // every row sees keys up to n + i0; a row that does not count, or does not see the
          // key, is left out rather than multiplied by zero
          const bool seen = i * kU + kU - 1 <= w.k.n + a.i0;
          auto add = [&](const uint32_t* s, int c) {
            if (seen && (plain >> (c / 2) & 1)) {
#pragma unroll
              for (int e = 0; e < 16; e += 4) {
                const float4 f = *reinterpret_cast<const float4*>(shift + c + e);
                const float2 x0 = mma::fma2(make_float2(__uint_as_float(s[e]), __uint_as_float(s[e + 1])), scale,
                                            make_float2(f.x, f.y));
                const float2 x1 = mma::fma2(make_float2(__uint_as_float(s[e + 2]), __uint_as_float(s[e + 3])), scale,
                                            make_float2(f.z, f.w));
                sum = mma::add2(sum, make_float2(mma::exp2_fast(x0.x), mma::exp2_fast(x0.y)));
                sum = mma::add2(sum, make_float2(mma::exp2_fast(x1.x), mma::exp2_fast(x1.y)));
              }
            } else {
#pragma unroll
              for (int e = 0; e < 16; ++e) {
                const float p = mma::exp2_fast(fmaf(__uint_as_float(s[e]), a.scale2, shift[c + e]));
                sum.x += key <= last[c + e] ? p : 0.f;
              }
            }
          };
          ptx::tmem_ld_32x32b_x16(col, v[0]);
          int c = 0;
          for (; c + 32 <= rows16; c += 32) {
            ptx::tmem_wait_ld();
            ptx::tmem_ld_32x32b_x16(col + c + 16, v[1]);
            add(v[0], c);
            ptx::tmem_wait_ld();
            if (c + 32 < rows16) ptx::tmem_ld_32x32b_x16(col + c + 32, v[0]);
            add(v[1], c + 16);
          }
          ptx::tmem_wait_ld();
          if (c < rows16) add(v[0], c);
          ptx::tc_fence_before();
          __syncwarp();
          if (lane == 0) ptx::mbar_arrive(sempty(buf));
          if (key < top) a.out[row0 + key] = before + (sum.x + sum.y);
        }
        tiles += n;
        more = walk_next<kU>(a, w);
      }
    }
  }
  __syncwarp();
  if (!ok && lane == 0) record_status(a.c.status, BS_ERR_TIMEOUT);
  ptx::tc_fence_before();
  __syncthreads();
  if (warp == kScoreWarps + 1) {
    ptx::tc_fence_after();
    ptx::tmem_dealloc(tmem_at, 512);
  }
}

template <int DP>
int scores_tiles_launch(ScoreArgs a, const CacheMaps& maps, cudaStream_t st) {
  using Cfg = ScoreTilesCfg<DP>;
  static bool set[64] = {};
  int dev = 0;
  BS_CUDA(cudaGetDevice(&dev));
  if (dev >= 64 || !set[dev]) {
    BS_CUDA(cudaFuncSetAttribute(kv_scores_tiles_kernel<DP>, cudaFuncAttributeMaxDynamicSharedMemorySize, Cfg::total));
    if (dev < 64) set[dev] = true;
  }
  const int step = kScoreRows / a.G;
  for (a.i0 = 0; a.i0 < a.T; a.i0 += step) {
    a.rows = std::min(step, a.T - a.i0) * a.G;
    kv_scores_tiles_kernel<DP><<<sm_count(), kScoreTileThreads, Cfg::total, st>>>(a, maps);
    BS_LAUNCHED();
    a.scores = a.out;
  }
  return BS_OK;
}

template <int DP, bool kTma>
int scores_launch(ScoreArgs a, const CacheMaps& maps, cudaStream_t st) {
  using Cfg = ScoreCfg<DP>;
  static bool set[64] = {};
  int dev = 0;
  BS_CUDA(cudaGetDevice(&dev));
  constexpr int kMost = 200 * 1024;
  if (dev >= 64 || !set[dev]) {
    BS_CUDA(cudaFuncSetAttribute(kv_scores_kernel<DP, kTma>, cudaFuncAttributeMaxDynamicSharedMemorySize, kMost));
    if (dev < 64) set[dev] = true;
  }
  // as many accepted entries at a time as their queries fit beside the keys
  const int step = std::max(1, (kMost - Cfg::smem(0)) / (DP * 2 + 8) / 8 * 8 / a.G);
  for (a.i0 = 0; a.i0 < a.T; a.i0 += step) {
    a.rows = std::min(step, a.T - a.i0) * a.G;
    const int smem = Cfg::smem((a.rows + 7) / 8 * 8);
    const int grid = sm_count() * (smem <= 113 * 1024 ? 2 : 1);
    kv_scores_kernel<DP, kTma><<<grid, kScoreThreads, smem, st>>>(a, maps);
    BS_LAUNCHED();
    a.scores = a.out;
  }
  return BS_OK;
}

// ---------------------------------------------------------------- eviction
// Selection: one cluster per (sequence, kv head), each CTA a contiguous range
// of its slots, whose scores it holds in shared memory as unsigned keys of the
// same order.  A radix selection over digits of 11, 11 and 10 bits (histograms
// joined through distributed shared memory) finds the key of the last kept slot
// and how many slots of that very key are kept; a scan then writes the kept
// slots in order.  Protected slots get the highest key, NaN the lowest; slots behind the
// scores' width count as 0, what an untouched key has, so that no slot is lost there.
struct EvictArgs {
  PagedCache c;
  const float* scores;
  const int32_t* out_table;
  int32_t* kept;
  int32_t* out_lens;
  float* out_scores;
  int capacity, budget, first, last, out_width, out_capacity, held;  // scores' width; held: keys a CTA has room for
  int vec;    // scores of a (sequence, kv head) start on 16 bytes
  int chunk;  // rows a CTA of the move takes
};

__device__ __forceinline__ uint32_t score_key(float x) {
  if (x != x) return 0u;
  const uint32_t u = __float_as_uint(x + 0.f);  // -0 becomes +0
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}

constexpr int kMoveRows = 256;
constexpr int kSel = 512;         // threads of a selection CTA
constexpr int kBins = 4 * kSel;   // of an 11-bit digit

__device__ __forceinline__ uint32_t dsmem_u32(uint32_t addr, uint32_t rank) {
  uint32_t v;
  asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(ptx::mapa(addr, rank)) : "memory");
  return v;
}
__device__ __forceinline__ uint4 dsmem_u4(uint32_t addr, uint32_t rank) {
  uint4 v;
  asm volatile("ld.shared::cluster.v4.u32 {%0, %1, %2, %3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(ptx::mapa(addr, rank)) : "memory");
  return v;
}

// kFits: shared memory holds the CTA's keys (and those of the first digit once more);
// longer ranges are read again for every digit.
template <int kCluster, bool kFits>
__global__ void __launch_bounds__(kSel) kv_select_kernel(const __grid_constant__ EvictArgs a) {
  extern __shared__ __align__(16) uint32_t held[];
  __shared__ __align__(16) uint32_t hist[2][kBins];
  __shared__ uint32_t found[2], totals[2], warps[2][kSel / 32];
  const int rank = blockIdx.x % kCluster, item = blockIdx.x / kCluster;
  const int b = item / a.c.heads;
  const int n = a.c.len(b, 0);
  const int want = min(n, min(a.budget, a.out_capacity));
  const float* scores = a.scores + (int64_t)item * a.capacity;
  // this CTA's slots [s0, s0 + mine)
  const int per = ((n + kCluster - 1) / kCluster + 3) / 4 * 4;
  const int s0 = min(n, rank * per), mine = min(n, s0 + per) - s0;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  // each warp takes a contiguous run of slots [w0, w1), 128 at a time: four neighbours a lane
  const int run = ((mine + kSel / 32 - 1) / (kSel / 32) + 127) / 128 * 128;
  const int w0 = min(mine, warp * run), w1 = min(mine, w0 + run), steps = (w1 - w0 + 127) / 128;
  auto key_of = [&](int s, float x) -> uint32_t {
    return s < a.first || s >= n - a.last ? 0xffffffffu : score_key(s < a.capacity ? x : 0.f);
  };
  auto load4 = [&](int i) -> float4 {  // scores of four slots, some perhaps behind the last
    const int s = s0 + i, top = a.capacity - 1;
    if (a.vec) return __ldg(reinterpret_cast<const float4*>(scores + min(s, top - 3)));
    return make_float4(__ldg(scores + min(s, top)), __ldg(scores + min(s + 1, top)), __ldg(scores + min(s + 2, top)),
                       __ldg(scores + min(s + 3, top)));
  };
  auto keys4 = [&](int i, float4 x) -> uint4 {
    return make_uint4(key_of(s0 + i, x.x), key_of(s0 + i + 1, x.y), key_of(s0 + i + 2, x.z), key_of(s0 + i + 3, x.w));
  };
  // counts a lane's four keys by their first digit
  auto count4 = [&](int there, const uint32_t* k) {
    const uint32_t d = __shfl_sync(0xffffffffu, k[0] >> 21, 0);
    const bool one = there >= 4 && k[0] >> 21 == d && k[1] >> 21 == d && k[2] >> 21 == d && k[3] >> 21 == d;
    if (__all_sync(0xffffffffu, one)) {  // untouched scores and protected slots: 128 of one digit
      if (lane == 0) atomicAdd(&hist[0][d], 128u);
      return;
    }
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (e < there) atomicAdd(&hist[0][k[e] >> 21], 1u);
  };
  *reinterpret_cast<uint4*>(hist[0] + 4 * threadIdx.x) = make_uint4(0, 0, 0, 0);
  __syncthreads();
  if (kFits) {
    for (int j = 0; j < steps; j += 4) {
      float4 x[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) x[e] = load4(w0 + (j + e) * 128 + lane * 4);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int i = w0 + (j + e) * 128 + lane * 4;
        if (j + e < steps) {
          const uint4 v = keys4(i, x[e]);
          *reinterpret_cast<uint4*>(held + i) = v;
          const uint32_t k[4] = {v.x, v.y, v.z, v.w};
          if (want < n) count4(w1 - i, k);
        }
      }
    }
  }
  // f(first of the lane's four slots, how many of them there are, their keys) for every
  // step of the warp; a lane sees only what it wrote
  auto walk = [&](auto&& f) {
    constexpr int kAtOnce = kFits ? 1 : 4;
#pragma unroll 1
    for (int j = 0; j < steps; j += kAtOnce) {
      const int i = w0 + j * 128 + lane * 4;
      uint4 v[kAtOnce];
      if constexpr (kFits) {
        v[0] = *reinterpret_cast<const uint4*>(held + i);
      } else {
        float4 x[kAtOnce];
#pragma unroll
        for (int e = 0; e < kAtOnce; ++e) x[e] = load4(i + e * 128);
#pragma unroll
        for (int e = 0; e < kAtOnce; ++e) v[e] = keys4(i + e * 128, x[e]);
      }
#pragma unroll
      for (int e = 0; e < kAtOnce; ++e) {
        const uint32_t k[4] = {v[e].x, v[e].y, v[e].z, v[e].w};
        if (j + e < steps) f(s0 + i + e * 128, w1 - i - e * 128, k);
      }
    }
  };

  const uint32_t below = (1u << lane) - 1u;
  uint32_t* match = held + a.held;
  int matches = 0;
  uint32_t gt = 0, eq = 0;  // this lane's keys above the chosen one, and equal to it
  uint32_t prefix = 0, mask = 0;
  int need = want;  // slots still to choose among those whose key matches prefix
  if (want < n) {
    for (int pass = 0; pass < 3; ++pass) {
      const int shift = pass == 0 ? 21 : pass == 1 ? 10 : 0;
      const uint32_t digit = pass == 2 ? 0x3ffu : 0x7ffu;
      uint32_t* hs = hist[pass & 1];
      if (pass) {
        *reinterpret_cast<uint4*>(hs + 4 * threadIdx.x) = make_uint4(0, 0, 0, 0);
        __syncthreads();
      }
      if (pass == 0) {
        if (!kFits) walk([&](int slot, int there, const uint32_t* k) { count4(there, k); });
      } else if (!kFits) {
        walk([&](int slot, int there, const uint32_t* k) {
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (e < there && (k[e] & mask) == prefix) atomicAdd(&hs[k[e] >> shift & digit], 1u);
        });
      } else if (pass == 1) {
        // the keys of the first digit, put together by each warp; those above it are counted
        walk([&](int slot, int there, const uint32_t* k) {
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const bool on = e < there && (k[e] & mask) == prefix;
            const uint32_t m = __ballot_sync(0xffffffffu, on);
            gt += e < there && (k[e] & mask) > prefix;
            if (on) {
              match[w0 + matches + __popc(m & below)] = k[e];
              atomicAdd(&hs[k[e] >> shift & digit], 1u);
            }
            matches += __popc(m);
          }
        });
        __syncwarp();
      } else {
        for (int j = lane; j < matches; j += 32) {
          const uint32_t k = match[w0 + j];
          if ((k & mask) == prefix) atomicAdd(&hs[k & digit], 1u);
        }
      }
      ptx::cluster_sync();
      // every CTA finds the digit whose bin holds the need-th highest key: a thread to
      // four bins from the top, a scan, and the one thread whose bin it is
      uint4 bin = make_uint4(0, 0, 0, 0);
#pragma unroll
      for (int r = 0; r < kCluster; ++r) {
        const uint4 v = dsmem_u4(ptx::smem_addr(hs + kBins - 4 - 4 * threadIdx.x), r);
        bin.x += v.x, bin.y += v.y, bin.z += v.z, bin.w += v.w;
      }
      const uint32_t sum = bin.x + bin.y + bin.z + bin.w;
      uint32_t incl = sum;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const uint32_t v = __shfl_up_sync(0xffffffffu, incl, o);
        if (lane >= o) incl += v;
      }
      if (lane == 31) warps[0][warp] = incl;
      __syncthreads();
      uint32_t above = incl - sum;
#pragma unroll
      for (int w = 0; w < kSel / 32; ++w) above += w < warp ? warps[0][w] : 0u;
      if (above < (uint32_t)need && (uint32_t)need <= above + sum) {
        uint32_t d = kBins - 1 - 4 * threadIdx.x, left = need - above, in = bin.w;
        if (left > in) left -= in, in = bin.z, --d;
        if (left > in) left -= in, in = bin.y, --d;
        if (left > in) left -= in, --d;
        found[0] = d, found[1] = left;
      }
      __syncthreads();
      prefix |= found[0] << shift;
      mask |= digit << shift;
      need = found[1];
      // the other histogram is next: its readers passed the last cluster_sync
    }
  }
  // key == prefix: the first `need` in slot order are kept; key > prefix: all
  const bool all = want == n;
  if (!all && kFits) {
    for (int j = lane; j < matches; j += 32) {
      const uint32_t k = match[w0 + j];
      gt += k > prefix, eq += k == prefix;
    }
  } else if (!all) {
    walk([&](int slot, int there, const uint32_t* k) {
#pragma unroll
      for (int e = 0; e < 4; ++e) gt += e < there && k[e] > prefix, eq += e < there && k[e] == prefix;
    });
  }
  gt = all ? w1 - w0 : __reduce_add_sync(0xffffffffu, gt);
  eq = __reduce_add_sync(0xffffffffu, eq);
  __syncthreads();
  if (lane == 0) warps[0][warp] = gt, warps[1][warp] = eq;
  __syncthreads();
  uint32_t bg = 0, be = 0, tg = 0, te = 0;
#pragma unroll
  for (int w = 0; w < kSel / 32; ++w) {
    const uint32_t u = warps[0][w], v = warps[1][w];
    if (w < warp) bg += u, be += v;
    tg += u, te += v;
  }
  if (threadIdx.x == 0) totals[0] = tg, totals[1] = te;
  ptx::cluster_sync();
  for (int r = 0; r < rank; ++r) {
    bg += dsmem_u32(ptx::smem_addr(&totals[0]), r);
    be += dsmem_u32(ptx::smem_addr(&totals[1]), r);
  }
  // nobody leaves while its shared memory may be read: the wait stands at the end
  asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
  int32_t* kept = a.kept + (int64_t)item * a.budget;
  float* out = a.out_scores + (int64_t)item * a.out_capacity;
  walk([&](int slot, int there, const uint32_t* k) {
    uint32_t count = 0;  // of keys above, and equal ones in the upper half
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (e < there) count += all || k[e] > prefix ? 1u : k[e] == prefix ? 0x10000u : 0u;
    uint32_t incl = count;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const uint32_t v = __shfl_up_sync(0xffffffffu, incl, o);
      if (lane >= o) incl += v;
    }
    uint32_t g = bg + (incl - count & 0xffffu), q = be + (incl - count >> 16);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const bool more = e < there && (all || k[e] > prefix), same = e < there && !all && k[e] == prefix;
      if (more || (same && q < (uint32_t)need)) {
        const uint32_t at = g + min(q, (uint32_t)need);
        kept[at] = slot + e;
        // the key gives the score back, but for protected slots and NaN
        out[at] = k[e] != 0xffffffffu && k[e] != 0u ? __uint_as_float(k[e] & 0x80000000u ? k[e] ^ 0x80000000u : ~k[e])
                  : slot + e < a.capacity           ? scores[slot + e]
                                                    : 0.f;
      }
      g += more, q += same;
    }
    const uint32_t total = __shfl_sync(0xffffffffu, incl, 31);
    bg += total & 0xffffu, be += total >> 16;
  });
  // behind the kept slots: -1 and zero scores
  for (int i = want + rank * kSel + threadIdx.x; i < a.budget; i += kCluster * kSel) kept[i] = -1;
  for (int i = want + rank * kSel + threadIdx.x; i < a.out_capacity; i += kCluster * kSel) out[i] = 0.f;
  if (threadIdx.x == 0 && rank == 0 && item % a.c.heads == 0) {
    a.out_lens[b] = want;
    if (want < min(n, a.budget)) record_status(a.c.status, BS_ERR_CAPACITY);
  }
  asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}

constexpr int kHeldMost = 24 * 1024;  // keys
static_assert(kHeldMost * 8 + sizeof(uint32_t) * 2 * kBins + 1024 <= 227 * 1024, "shared memory of a CTA");

template <int kCluster, bool kFits>
int select_launch(EvictArgs a, int items, cudaStream_t st) {
  static bool set[64] = {};
  int dev = 0;
  BS_CUDA(cudaGetDevice(&dev));
  if (kFits && (dev >= 64 || !set[dev])) {
    BS_CUDA(cudaFuncSetAttribute(kv_select_kernel<kCluster, kFits>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                 kHeldMost * 8));
    if (dev < 64) set[dev] = true;
  }
  const int per = (int)cdiv((int64_t)a.c.capacity, (int64_t)kCluster);
  a.held = kFits ? (int)((per + 3) / 4 * 4 + 127) / 128 * 128 : 0;
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[1];
  cfg.gridDim = dim3((unsigned)items * kCluster);
  cfg.blockDim = dim3(kSel);
  cfg.dynamicSmemBytes = (size_t)a.held * 8;
  cfg.stream = st;
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = kCluster;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  BS_CUDA(cudaLaunchKernelEx(&cfg, kv_select_kernel<kCluster, kFits>, a));
  return BS_OK;
}

template <int kCluster>
int select_of(const EvictArgs& a, int items, cudaStream_t st) {
  return cdiv((int64_t)a.c.capacity, (int64_t)kCluster) <= kHeldMost - 128 ? select_launch<kCluster, true>(a, items, st)
                                                                       : select_launch<kCluster, false>(a, items, st);
}

// Copies the kept rows: a CTA looks up where its rows come from and go to, a row to a
// thread, and then copies them, dim / 8 lanes to a row.  Neighbouring CTAs take the
// heads of the same rows, which lie side by side in caches of interleaved heads.
// HBM-bound: 8 dim bytes a kept row and head.  64 heads of 8192 kept rows, dim 64 (268 MB):
// 50 us, 5.3 TB/s, where a plain copy reaches 6.6; lookups by every lane for its own four
// rows took 60 us.  CTAs of 128 / 256 / 512 / 1024 rows: 83 / 81 / 85 / 93 us with the
// selection, heads apart instead of neighbours 82.5.  Started early, while the selection
// runs, its waiting CTAs slowed that by 5 us, so it starts when the selection ends.
__global__ void __launch_bounds__(256) kv_move_kernel(const __grid_constant__ EvictArgs a) {
  __shared__ int4 place[kMoveRows];  // page and slot in it, of the source and of the copy
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int lanes = a.c.dim <= 64 ? 8 : 16;
  const int c = threadIdx.x % lanes, at_once = 256 / lanes;
  const int b = blockIdx.y, chunk = blockIdx.x / a.c.heads, h = blockIdx.x - chunk * a.c.heads;
  const int i0 = chunk * a.chunk, rows = min(a.chunk, min(a.budget, a.out_capacity) - i0);
  const int32_t* kept = a.kept + ((int64_t)b * a.c.heads + h) * a.budget;
  for (int r = threadIdx.x; r < rows; r += 256) {
    const int s = kept[i0 + r];
    int4 at = make_int4(0, 0, -1, 0);
    if (s >= 0) {
      int page, opage;
      a.c.div.split(s, page, at.y);
      a.c.div.split(i0 + r, opage, at.w);
      at.x = a.c.page_of(b, page);
      at.z = a.out_table[(int64_t)b * a.out_width + opage];
      if ((unsigned)at.z >= (unsigned)a.c.pages) {
        record_status(a.c.status, BS_ERR_CAPACITY);
        at.z = -1;
      }
    }
    place[r] = at;
  }
  __syncthreads();
  if (c * 8 >= a.c.dim) return;
  __nv_bfloat16* k = a.c.k + h * a.c.kh + c * 8;
  __nv_bfloat16* v = a.c.v + h * a.c.vh + c * 8;
  for (int r0 = threadIdx.x / lanes; r0 < rows; r0 += 4 * at_once) {
    uint4 kv[4], vv[4];
    int4 at[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int r = r0 + j * at_once;
      at[j] = r < rows ? place[r] : make_int4(0, 0, -1, 0);
      if (at[j].z < 0) continue;
      kv[j] = *reinterpret_cast<const uint4*>(k + at[j].x * a.c.kp + at[j].y * a.c.ks);
      vv[j] = *reinterpret_cast<const uint4*>(v + at[j].x * a.c.vp + at[j].y * a.c.vs);
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if (at[j].z < 0) continue;
      *reinterpret_cast<uint4*>(k + at[j].z * a.c.kp + at[j].w * a.c.ks) = kv[j];
      *reinterpret_cast<uint4*>(v + at[j].z * a.c.vp + at[j].w * a.c.vs) = vv[j];
    }
  }
}

}  // namespace
}  // namespace bs

extern "C" int bs_tree_commit(const bs_kv_cache* cache, int64_t T, const int32_t* accepted, int64_t A, void* stream) {
  using namespace bs;
  const char* fn = "bs_tree_commit";
  BS_ARG(cache, "%s: null cache", fn);
  if (cache->batch == 0 || A == 0) return BS_OK;
  BS_ARG(accepted, "%s: null pointer", fn);
  BS_ARG(T >= 1 && A >= 0 && A <= 256 && A <= T, "%s: at most 256 accepted of T drafted tokens", fn);
  PagedCache c;
  BS_TRY(paged_cache(fn, cache, T, true, &c));
  BS_ARG(cache->batch * cache->heads < INT32_MAX, "%s: sizes too large", fn);
  BS_TRY(check_device());
  const int smem = (int)(A * cache->dim * 4);
  static bool set[64] = {};
  int dev = 0;
  BS_CUDA(cudaGetDevice(&dev));
  if (smem > 48 * 1024 && (dev >= 64 || !set[dev])) {
    BS_CUDA(cudaFuncSetAttribute(tree_commit_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 256 * 128 * 4));
    if (dev < 64) set[dev] = true;
  }
  tree_commit_kernel<<<(unsigned)(cache->batch * cache->heads), 256, smem, reinterpret_cast<cudaStream_t>(stream)>>>(
      c, (int)T, accepted, (int)A);
  BS_LAUNCHED();
  return BS_OK;
}

extern "C" int bs_kv_scores_add(const bs_heads* q, const bs_kv_cache* cache, int64_t T, int64_t Hq, const float* lse,
                                const int32_t* accepted, int64_t A, float scale, const float* scores,
                                float* scores_out, int64_t capacity, void* stream) {
  using namespace bs;
  const char* fn = "bs_kv_scores_add";
  BS_ARG(q && cache, "%s: null pointer", fn);
  if (cache->batch == 0) return BS_OK;
  BS_ARG(q->ptr && lse && scores && scores_out, "%s: null pointer", fn);
  BS_ARG(T >= 1 && A >= 1 && T < (1 << 20) && A <= T, "%s: 1 to T accepted of T tokens", fn);
  BS_ARG(accepted || A == T, "%s: without a list every token is accepted", fn);
  ScoreArgs a = {};
  BS_TRY(paged_cache(fn, cache, A, false, &a.c));
  BS_ARG(Hq > 0 && Hq % cache->heads == 0 && Hq <= 65535, "%s: query heads must be a multiple of the cache's heads", fn);
  BS_ARG(capacity > 0 && capacity <= a.c.capacity, "%s: scores for more slots than the page table has", fn);
  BS_ARG(cache->batch * cache->heads < INT32_MAX, "%s: sizes too large", fn);
  BS_ALIGNED16(q->ptr, "q");
  BS_REQUIRE(q->stride_b % 8 == 0 && q->stride_t % 8 == 0 && q->stride_h % 8 == 0, BS_ERR_MISALIGNED,
             "%s: q strides must be multiples of 8 elements", fn);
  a.G = (int)(Hq / cache->heads);
  BS_ARG(a.G <= 128, "%s: more than 128 query heads to a kv head", fn);
  a.q = static_cast<const __nv_bfloat16*>(q->ptr);
  a.qb = q->stride_b, a.qt = q->stride_t, a.qh = q->stride_h;
  a.lse = lse;
  a.accepted = accepted;
  a.scores = scores;
  a.out = scores_out;
  a.scale2 = scale * kLog2e;
  a.tokens = (int)T, a.Hq = (int)Hq, a.capacity = (int)capacity;
  a.B = (int)cache->batch, a.Hkv = (int)cache->heads, a.tiles = 1;
  a.T = (int)A;
  BS_TRY(check_device());
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  const int64_t D = cache->dim;
  CacheMaps maps = {};
  // Up to so many rows the products of 16 keys at a time are no slower, and units of 32 or
  // 64 keys share ragged lengths better.  In us, those and tiles of 128 keys: dim 64, 32
  // sequences of 5000 keys, 8 heads: 8 rows 34.0 / 37.2, 24 rows 38.5 / 38.9, 32 rows 42.8 /
  // 38.1, 128 rows 149 / 61; ragged to 8192 keys, 8 rows 32 / 42.  Dim 128, 2 sequences of
  // 131072 keys: 8 rows 89.7 / 89.2, 16 rows 91.1 / 88.6, 32 rows 102 / 88.8, 128 rows 368 / 99.
  // Pages without boxes stay on the former, with 16-byte copies: 514 us for those 128 rows, and
  // 132 for 64 rows of 64 over 2 x 131072 keys where boxes take 57.
  const int few = D <= 64 ? 24 : 16;
  a.box = cache_box_rows(cache, 128);
  if (a.box >= 8 && A * a.G > few) {
    a.setup = 3;  // 1 / 2 / 3 / 4 / 5: 14.7 / 13.4 / 11.1 / 10.9 / 11.2 us at 12 items of 30011 keys, 56 rows
    a.min_chunk = 2;
    BS_TRY(cache_maps(cache, a.box, false, &maps));
    return D <= 64 ? scores_tiles_launch<64>(a, maps, st) : scores_tiles_launch<128>(a, maps, st);
  }
  a.setup = 8;  // 4 / 6 / 8: 38.9 / 34.0 / 32.0 us at 256 ragged items of 8192 keys, 8 rows; 16.8 / 15.2 / 15.8 at 12
  a.min_chunk = 4;
  a.box = cache_box_rows(cache, D <= 64 ? ScoreCfg<64>::kU : ScoreCfg<128>::kU);
  if (a.box >= 8) {
    BS_TRY(cache_maps(cache, a.box, false, &maps));
    return D <= 64 ? scores_launch<64, true>(a, maps, st) : scores_launch<128, true>(a, maps, st);
  }
  a.box = 1;
  return D <= 64 ? scores_launch<64, false>(a, maps, st) : scores_launch<128, false>(a, maps, st);
}

extern "C" int bs_kv_evict(const bs_kv_cache* cache, const float* scores, int64_t capacity, int64_t budget,
                           int64_t keep_first, int64_t keep_last, const int32_t* out_page_table, int64_t out_width,
                           int32_t* kept, int32_t* out_lens, float* out_scores, void* stream) {
  using namespace bs;
  const char* fn = "bs_kv_evict";
  BS_ARG(cache, "%s: null cache", fn);
  if (cache->batch == 0) return BS_OK;
  BS_ARG(scores && out_page_table && kept && out_lens && out_scores, "%s: null pointer", fn);
  EvictArgs a = {};
  BS_TRY(paged_cache(fn, cache, 0, true, &a.c));
  BS_ARG(capacity > 0 && capacity <= a.c.capacity, "%s: scores for more slots than the page table has", fn);
  BS_ARG(budget > 0 && budget < INT32_MAX && keep_first >= 0 && keep_last >= 0 && keep_first + keep_last <= budget,
         "%s: keep_first + keep_last must not exceed the (positive) budget", fn);
  BS_ARG(out_width > 0 && out_width * cache->page_size < INT32_MAX, "%s: bad width of the output page table", fn);
  BS_ARG(std::min(budget, capacity) <= out_width * cache->page_size, "%s: the output pages do not hold the budget", fn);
  BS_ARG(cache->batch * cache->heads <= 65535, "%s: more than 65535 (sequence, kv head) pairs", fn);
  a.scores = scores;
  a.out_table = out_page_table;
  a.kept = kept;
  a.out_lens = out_lens;
  a.out_scores = out_scores;
  a.capacity = (int)capacity, a.budget = (int)budget, a.first = (int)keep_first, a.last = (int)keep_last;
  a.out_width = (int)out_width, a.out_capacity = (int)(out_width * cache->page_size);
  BS_TRY(check_device());
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  a.vec = capacity % 4 == 0 && reinterpret_cast<uintptr_t>(scores) % 16 == 0;
  const int items = (int)(cache->batch * cache->heads);
  // CTAs per (sequence, kv head): 4096 scores each, as long as all clusters run at once and
  // leave each CTA its own SM.  With 1 / 2 / 4 / 8 of them, in us with the move:
  //     8 items of 8192 scores 16.4 / 14.3 / 14.6 / 18.8, of 32768 57 / 24 / 20 / 22, of 131072 211 / 94 / 58 / 37;
  //    64 items of 4096 19.8 / 18.9 / 24 / 61, of 32768 105 / 69 / 71 / 106, of 131072 300 / 178 / 169 / 222;
  //   256 items of 8192 108 / 115 / 137 / 283.
  int cluster = 1;
  while (cluster < 8 && cluster * 4096 < a.c.capacity && items * cluster * 2 <= sm_count()) cluster *= 2;
  BS_TRY(cluster == 1 ? select_of<1>(a, items, st) : cluster == 2 ? select_of<2>(a, items, st)
         : cluster == 4 ? select_of<4>(a, items, st) : select_of<8>(a, items, st));
  const int64_t rows = std::min<int64_t>(budget, std::min(a.c.capacity, a.out_capacity));
  a.chunk = kMoveRows;
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[1];
  cfg.gridDim = dim3((unsigned)(cdiv(rows, (int64_t)a.chunk) * cache->heads), (unsigned)cache->batch);
  cfg.blockDim = dim3(256);
  cfg.stream = st;
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  BS_CUDA(cudaLaunchKernelEx(&cfg, kv_move_kernel, a));
  return BS_OK;
}
