// Upkeep of the paged key/value cache between decoding steps: the accepted
// drafts moved together, the attention weight that each cached key received
// added to its score, and the keys of lowest score evicted.
#include "bs_paged.cuh"

namespace bs {
namespace {

constexpr float kLog2e = 1.4426950408889634f;

// ---------------------------------------------------------------- commit
// One CTA per (sequence, kv head): all accepted rows are read before any is
// written (slot n + i may itself be the source of an earlier row).
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
  const int n = c.len(b, T), per = c.dim / 8, items = 2 * count * per;
  auto at = [&](int i, int row) -> __nv_bfloat16* {
    const int col = i % per * 8, v = i / per & 1;
    int page, in;
    c.div.split(n + row, page, in);
    const int64_t p = c.page_of(b, page);
    return v ? c.v + p * c.vp + in * c.vs + h * c.vh + col : c.k + p * c.kp + in * c.ks + h * c.kh + col;
  };
  for (int i = threadIdx.x; i < items; i += blockDim.x)
    rows[i] = *reinterpret_cast<const uint4*>(at(i, acc[i / (2 * per)]));
  __syncthreads();
  for (int i = threadIdx.x; i < items; i += blockDim.x)
    if (acc[i / (2 * per)] != i / (2 * per)) *reinterpret_cast<uint4*>(at(i, i / (2 * per))) = rows[i];
}

// ---------------------------------------------------------------- scores
// K is the 16-row operand of the tensor-core product and the accepted rows its
// columns, so that a key's sum over the rows stays in one lane group: no atomics,
// one store per slot.  HBM-bound: 2 dim + 8 bytes per slot and kv head.  The
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

template <int DP, bool kTma>
__global__ void __launch_bounds__(128) kv_scores_kernel(const __grid_constant__ ScoreArgs a,
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
    if (lane == 0) {
      for (int s = 0; s < Cfg::kStages; ++s) ptx::mbar_init(bar + 8 * s, 1);
      ptx::fence_mbar_init();
    }
  } else if (a.c.dim < DP) {
    for (int i = threadIdx.x; i < 4 * Cfg::kWarpBytes / 16; i += 128)
      reinterpret_cast<uint4*>(smem)[i] = make_uint4(0, 0, 0, 0);
  }
  __syncthreads();
  const Range r = locate<kU>(a, blockIdx.x, gridDim.x, reinterpret_cast<int64_t*>(smem + Cfg::sums));
  Walk lw, cw;
  bool more = r.p0 < r.p1 && walk_begin<kU>(a, r, lw);
  const bool any = more;
  cw = lw;

  // ---- loading: lane g holds where the next unit's g-th box (or slot) lies
  const int box = kTma ? a.box : 1, boxes = kU / box;
  if (any) lw.u = lw.start + warp;
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
          record_status(a.c.status, BS_ERR_CAPACITY);
          next_page[e] = next_page[e] < 0 ? 0 : a.c.pages - 1;
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
  for (int s = 0; s < Cfg::kStages - 1; ++s) load(s);
  int stage = 0, phase = 0;
  const uint32_t qaddr = ptx::smem_addr(qs);
  const int mine = lane / 4 + (lane & 3) * 8;  // the slots of a unit that this lane stores: mine, mine + 32

  // ---- behind an item's last unit scores are only copied: an equal share of the
  // whole array for each CTA, while the first keys are on their way
  if (a.out != a.scores) {
    const int64_t all = (int64_t)a.B * a.Hkv * a.capacity, share = (all + gridDim.x - 1) / gridDim.x;
    const int64_t end = min(all, (blockIdx.x + 1) * share);
    for (int64_t from = blockIdx.x * share; from < end;) {
      const int64_t item = from / a.capacity, first = item * a.capacity;
      const int64_t to = min(end, first + a.capacity);
      const int n = a.c.len(item / a.Hkv, a.T) + a.T;
      const int64_t begin = max(from, first + min(a.capacity, (n + kU - 1) / kU * kU));
      for (int64_t i = begin + threadIdx.x; i < to; i += 16 * 128) {
        float v[16];
#pragma unroll
        for (int j = 0; j < 16; ++j) v[j] = a.scores[min(i + j * 128, all - 1)];
#pragma unroll
        for (int j = 0; j < 16; ++j)
          if (i + j * 128 < to) a.out[i + j * 128] = v[j];
      }
      from = to;
    }
  }

  while (any) {
    const int64_t row0 = ((int64_t)cw.b * a.Hkv + cw.h) * a.capacity;
    for (int i = threadIdx.x; i < rows8 * (DP / 8); i += 128) {
      const int r = i / (DP / 8), c = i - r * (DP / 8), e = a.i0 + r / a.G;
      uint4 v = make_uint4(0, 0, 0, 0);
      float2 f = make_float2(INFINITY, __int_as_float(-1));
      if (r < a.rows) {
        const int u = a.accepted ? a.accepted[(int64_t)cw.b * a.T + e] : e;
        if ((unsigned)u < (unsigned)a.tokens) {
          const int hq = cw.h * a.G + r % a.G;
          if (c * 8 < a.c.dim)
            v = __ldg(reinterpret_cast<const uint4*>(a.q + cw.b * a.qb + u * a.qt + hq * a.qh + c * 8));
          const float l = a.lse[((int64_t)cw.b * a.tokens + u) * a.Hq + hq];
          if (l != -INFINITY) f = make_float2(l * kLog2e, __int_as_float(cw.k.n + e));
        }
      }
      *reinterpret_cast<uint4*>(qs + qat(r, c)) = v;
      if (c == 0) info[r] = f;
    }
    __syncthreads();
    // the scores to add to are asked for one unit ahead
    const int top = a.out != a.scores ? a.capacity : min(a.capacity, cw.k.hi);
    float next[kMine];
    auto ask = [&](int u) {
#pragma unroll
      for (int e = 0; e < kMine; ++e) next[e] = __ldg(a.scores + row0 + min(u * kU + mine + 32 * e, a.capacity - 1));
    };
    ask(cw.start + warp);
    for (int u = cw.start + warp; u < cw.end; u += 4) {
      const int slot0 = u * kU;
      float before[kMine];
#pragma unroll
      for (int e = 0; e < kMine; ++e) before[e] = next[e];
      ask(u + 4);
      const uint32_t kt = base + stage * Cfg::kTile;
      if constexpr (kTma)
        ptx::mbar_wait(bar + 8 * stage, phase, &abort_flag);  // a wait that ran out is reported at the end
      else
        ptx::cp_async_wait<Cfg::kStages - 2>();
      __syncwarp();
      load((stage + Cfg::kStages - 1) % Cfg::kStages);
      if (++stage == Cfg::kStages) stage = 0, phase ^= 1;
      uint32_t kf[MT][KS][4];
#pragma unroll
      for (int mt = 0; mt < MT; ++mt)
#pragma unroll
        for (int k = 0; k < KS; ++k)
          mma::ldsm_x4(kt + mma::tile_at<kU>(mt * 16 + (lane & 15), 2 * k + (lane >> 4)), kf[mt][k]);
      float sum[2 * MT] = {};  // slots slot0 + lane / 4 + 8 i
      for (int r = 0; r < rows8; r += 8) {
        float s[MT][4] = {};
#pragma unroll
        for (int k = 0; k < KS; k += 2) {
          uint32_t f[4];
          mma::ldsm_x4(qaddr + qat(r + (lane & 7), 2 * k + (lane >> 3)), f);
#pragma unroll
          for (int mt = 0; mt < MT; ++mt) {
            mma::bf16_16816(s[mt], kf[mt][k], f[0], f[1]);
            mma::bf16_16816(s[mt], kf[mt][k + 1], f[2], f[3]);
          }
        }
        const float2 f0 = info[r + (lane & 3) * 2], f1 = info[r + (lane & 3) * 2 + 1];
#pragma unroll
        for (int mt = 0; mt < MT; ++mt)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float2 f = e & 1 ? f1 : f0;
            const int key = slot0 + mt * 16 + lane / 4 + (e >> 1) * 8;
            const float p = mma::exp2_fast(s[mt][e] * a.scale2 - f.x);
            sum[mt * 2 + (e >> 1)] += key <= __float_as_int(f.y) ? p : 0.f;
          }
      }
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
    __syncthreads();
  }
  if constexpr (kTma) {
    if (*(volatile int*)&abort_flag) {
      if (lane == 0) record_status(a.c.status, BS_ERR_TIMEOUT);
      // copies in flight end before the CTA's memory is given back
      volatile int gone = 0;
      for (int s = 0; s < Cfg::kStages; ++s) ptx::mbar_wait(bar + 8 * s, phase ^ 1, &gone);
    }
  } else {
    ptx::cp_async_wait_all();
  }
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
    kv_scores_kernel<DP, kTma><<<grid, 128, smem, st>>>(a, maps);
    BS_LAUNCHED();
    a.scores = a.out;
  }
  return BS_OK;
}

// ---------------------------------------------------------------- eviction
// Selection: one cluster per (sequence, kv head), each CTA a contiguous range
// of its slots, whose scores it holds in shared memory as unsigned keys of the
// same order.  A radix selection over four 8-bit digits (histograms joined
// through distributed shared memory) finds the key of the last kept slot and
// how many slots of that very key are kept; a scan then writes the kept slots
// in order.  Protected slots get the highest key, NaN the lowest.
struct EvictArgs {
  PagedCache c;
  const float* scores;
  const int32_t* out_table;
  int32_t* kept;
  int32_t* out_lens;
  float* out_scores;
  int capacity, budget, first, last, out_width, out_capacity, held;  // held: keys a CTA has room for
};

__device__ __forceinline__ uint32_t score_key(float x) {
  if (x != x) return 0u;
  const uint32_t u = __float_as_uint(x + 0.f);  // -0 becomes +0
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}

constexpr int kSel = 512;  // threads of a selection CTA

__device__ __forceinline__ uint32_t dsmem_u32(uint32_t addr, uint32_t rank) {
  uint32_t v;
  asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(ptx::mapa(addr, rank)) : "memory");
  return v;
}

__global__ void __launch_bounds__(kSel) kv_select_kernel(const __grid_constant__ EvictArgs a, int cluster) {
  extern __shared__ __align__(16) uint32_t held[];
  __shared__ uint32_t hist[2][256];
  __shared__ uint32_t found[2], totals[2], warps[2][kSel / 32];
  const int rank = blockIdx.x % cluster, item = blockIdx.x / cluster;
  const int b = item / a.c.heads;
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const int n = min(a.c.len(b, 0), a.capacity);
  const int want = min(n, a.budget);
  const float* scores = a.scores + (int64_t)item * a.capacity;
  // this CTA's slots [s0, s1)
  const int per = ((n + cluster - 1) / cluster + 3) / 4 * 4;
  const int s0 = min(n, rank * per), s1 = min(n, s0 + per), mine = s1 - s0;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  // each warp takes a contiguous run of slots, 32 at a time
  const int run = ((mine + kSel / 32 - 1) / (kSel / 32) + 31) / 32 * 32;
  const int w0 = min(mine, warp * run), steps = (min(mine, w0 + run) - w0 + 31) / 32;
  const bool fits = per <= a.held;
  auto key_of = [&](int s, float x) -> uint32_t { return s < a.first || s >= n - a.last ? 0xffffffffu : score_key(x); };
  if (fits) {
    // eight loads of a lane in flight; the loops stay short, since each is run once
    // and its instructions come from memory too
    for (int j = 0; j < steps; j += 8) {
      float x[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) x[e] = __ldg(scores + min(s0 + w0 + (j + e) * 32 + lane, a.capacity - 1));
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const int i = w0 + (j + e) * 32 + lane;
        if (j + e < steps) held[i] = key_of(s0 + i, x[e]);
      }
    }
    __syncwarp();
  }
  // f(slot of this lane or -1, its key) for every step of the warp
  auto walk = [&](auto&& f) {
    const int last = min(mine, w0 + run);
#pragma unroll 4
    for (int j = 0; j < steps; ++j) {
      const int i = w0 + j * 32 + lane, c = min(i, last - 1);
      const uint32_t k = fits ? held[c] : key_of(s0 + c, scores[s0 + c]);
      f(i < last ? s0 + i : -1, i < last ? k : 0u);
    }
  };

  const uint32_t below = (1u << lane) - 1u;
  uint32_t* match = held + a.held;
  int matches = 0;
  uint32_t gt = 0, eq = 0;  // this warp's keys above the chosen one, and equal to it
  uint32_t prefix = 0, mask = 0;
  int need = want;  // slots still to choose among those whose key matches prefix
  if (want < n) {
    for (int pass = 0; pass < 4; ++pass) {
      const int shift = 24 - 8 * pass;
      uint32_t* hs = hist[pass & 1];
      for (int i = threadIdx.x; i < 256; i += kSel) hs[i] = 0;
      __syncthreads();
      if (pass == 0) {
        // sign and exponent: few digits, so a warp counts equal ones together
        walk([&](int slot, uint32_t k) {
          const uint32_t same = __match_any_sync(0xffffffffu, slot >= 0 ? k >> 24 : 256u);
          if (slot >= 0 && lane == __ffs(same) - 1) atomicAdd(&hs[k >> 24], (uint32_t)__popc(same));
        });
      } else if (fits) {
        // the keys that still match, put together by each warp after the first digit;
        // those above it are counted on the way
        if (pass == 1) {
          walk([&](int slot, uint32_t k) {
            const bool on = slot >= 0 && (k & mask) == prefix;
            const uint32_t m = __ballot_sync(0xffffffffu, on);
            gt += __popc(__ballot_sync(0xffffffffu, slot >= 0 && (k & mask) > prefix));
            if (on) match[w0 + matches + __popc(m & below)] = k;
            matches += __popc(m);
          });
          __syncwarp();
        }
        const uint32_t digit = shift == 16 ? 0u : 255u << (shift + 8);  // the last digit found
        for (int j = 0; j < matches; j += 32) {
          const uint32_t k = match[w0 + min(j + lane, matches - 1)];
          const bool on = j + lane < matches, now = on && (k & mask) == prefix;
          // among keys that matched before the last digit, those above it
          if (pass > 1)
            gt += __popc(__ballot_sync(0xffffffffu, on && ((k ^ prefix) & (mask & ~digit)) == 0 && (k & digit) > (prefix & digit)));
          if (now) atomicAdd(&hs[k >> shift & 255], 1u);
        }
      } else {
        walk([&](int slot, uint32_t k) {
          if (slot >= 0 && (k & mask) == prefix) atomicAdd(&hs[k >> shift & 255], 1u);
        });
      }
      ptx::cluster_sync();
      // every CTA finds the digit whose bin holds the need-th highest key: a thread
      // per bin from the top, a scan, and the one thread whose bin it is
      uint32_t bin = 0;
      if (threadIdx.x < 256)
        for (int r = 0; r < cluster; ++r) bin += dsmem_u32(ptx::smem_addr(&hs[255 - threadIdx.x]), r);
      uint32_t incl = bin;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const uint32_t v = __shfl_up_sync(0xffffffffu, incl, o);
        if (lane >= o) incl += v;
      }
      if (lane == 31 && warp < 8) warps[0][warp] = incl;
      __syncthreads();
      if (threadIdx.x < 256) {
        uint32_t above = incl - bin;
        for (int w = 0; w < warp; ++w) above += warps[0][w];
        if (above < (uint32_t)need && (uint32_t)need <= above + bin) found[0] = 255 - threadIdx.x, found[1] = need - above;
      }
      __syncthreads();
      prefix |= found[0] << shift;
      mask |= 255u << shift;
      need = found[1];
      // the other histogram is next: its readers passed the last cluster_sync
    }
  }
  // key == prefix: the first `need` in slot order are kept; key > prefix: all
  const bool all = want == n;
  if (all) {
    gt = max(0, min(mine, w0 + run) - w0);
  } else if (fits) {
    for (int j = 0; j < matches; j += 32) {
      const uint32_t k = match[w0 + min(j + lane, matches - 1)];
      const bool near = j + lane < matches && ((k ^ prefix) & 0xffffff00u) == 0;  // all but the last digit
      gt += __popc(__ballot_sync(0xffffffffu, near && k > prefix));
      eq += __popc(__ballot_sync(0xffffffffu, near && k == prefix));
    }
  } else {
    walk([&](int slot, uint32_t k) {
      gt += __popc(__ballot_sync(0xffffffffu, slot >= 0 && k > prefix));
      eq += __popc(__ballot_sync(0xffffffffu, slot >= 0 && k == prefix));
    });
  }
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
  int32_t* kept = a.kept + (int64_t)item * a.budget;
  float* out = a.out_scores + (int64_t)item * a.out_capacity;
  walk([&](int slot, uint32_t k) {
    const bool more = slot >= 0 && (all || k > prefix), same = slot >= 0 && !all && k == prefix;
    const uint32_t mg = __ballot_sync(0xffffffffu, more), me = __ballot_sync(0xffffffffu, same);
    const uint32_t eq0 = be + __popc(me & below);
    if (more || (same && eq0 < (uint32_t)need)) {
      const uint32_t at = bg + __popc(mg & below) + min(eq0, (uint32_t)need);
      kept[at] = slot;
      // the key gives the score back, but for protected slots and NaN
      if (at < (uint32_t)a.out_capacity)
        out[at] = k == 0xffffffffu || k == 0u ? scores[slot] : __uint_as_float(k & 0x80000000u ? k ^ 0x80000000u : ~k);
    }
    bg += __popc(mg);
    be += __popc(me);
  });
  // behind the kept slots: -1 and zero scores
  for (int i = want + rank * kSel + threadIdx.x; i < a.budget; i += cluster * kSel) kept[i] = -1;
  for (int i = want + rank * kSel + threadIdx.x; i < a.out_capacity; i += cluster * kSel) out[i] = 0.f;
  if (threadIdx.x == 0 && rank == 0 && item % a.c.heads == 0) {
    a.out_lens[b] = want;
    if (want > a.out_capacity) record_status(a.c.status, BS_ERR_CAPACITY);
  }
  ptx::cluster_sync();  // nobody leaves while its shared memory may be read
}

// Copies the kept rows: kLanes lanes per row, four rows of each in flight.
__global__ void __launch_bounds__(256) kv_move_kernel(const __grid_constant__ EvictArgs a) {
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int lanes = a.c.dim <= 64 ? 8 : 16;
  const int c = threadIdx.x % lanes, at_once = 256 / lanes;
  const int b = blockIdx.y / a.c.heads, h = blockIdx.y - b * a.c.heads;
  const int rows = min(a.budget, a.out_capacity);
  const int32_t* kept = a.kept + (int64_t)blockIdx.y * a.budget;
  const bool col = c * 8 < a.c.dim;
  uint4 kv[4], vv[4];
  int64_t dk[4], dv[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int i = blockIdx.x * at_once * 4 + j * at_once + threadIdx.x / lanes;
    const int s = i < rows ? kept[i] : -1;
    dk[j] = -1;
    if (s < 0 || !col) continue;
    int page, row, opage, orow;
    a.c.div.split(s, page, row);
    a.c.div.split(i, opage, orow);
    const int64_t p = a.c.page_of(b, page), q = a.out_table[(int64_t)b * a.out_width + opage];
    if ((uint64_t)q >= (uint64_t)a.c.pages) {
      record_status(a.c.status, BS_ERR_CAPACITY);
      continue;
    }
    kv[j] = *reinterpret_cast<const uint4*>(a.c.k + p * a.c.kp + row * a.c.ks + h * a.c.kh + c * 8);
    vv[j] = *reinterpret_cast<const uint4*>(a.c.v + p * a.c.vp + row * a.c.vs + h * a.c.vh + c * 8);
    dk[j] = q * a.c.kp + orow * a.c.ks + h * a.c.kh + c * 8;
    dv[j] = q * a.c.vp + orow * a.c.vs + h * a.c.vh + c * 8;
  }
#pragma unroll
  for (int j = 0; j < 4; ++j)
    if (dk[j] >= 0) {
      *reinterpret_cast<uint4*>(a.c.k + dk[j]) = kv[j];
      *reinterpret_cast<uint4*>(a.c.v + dv[j]) = vv[j];
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
  a.setup = 8;
  a.min_chunk = 4;
  BS_TRY(check_device());
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  const int64_t D = cache->dim;
  CacheMaps maps = {};
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
  // CTAs per (sequence, kv head): 8192 scores each, up to eight CTAs
  int cluster = 1;
  while (cluster < 8 && (int64_t)cluster * 8192 < capacity) cluster *= 2;
  const int64_t per = cdiv(cdiv(capacity, (int64_t)cluster), (int64_t)4) * 4;
  constexpr int kHeldMost = 24 * 1024;  // keys, twice; longer ranges are read again for every digit
  a.held = (int)(std::min<int64_t>(per, kHeldMost) + 31) / 32 * 32;
  static bool set[64] = {};
  int dev = 0;
  BS_CUDA(cudaGetDevice(&dev));
  if (dev >= 64 || !set[dev]) {
    BS_CUDA(cudaFuncSetAttribute(kv_select_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kHeldMost * 8));
    if (dev < 64) set[dev] = true;
  }
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[1];
  const unsigned items = (unsigned)(cache->batch * cache->heads);
  cfg.gridDim = dim3(items * cluster);
  cfg.blockDim = dim3(kSel);
  cfg.dynamicSmemBytes = (size_t)a.held * 8;
  cfg.stream = st;
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = cluster;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  BS_CUDA(cudaLaunchKernelEx(&cfg, kv_select_kernel, a, cluster));
  const int rows = 4 * 256 / (cache->dim <= 64 ? 8 : 16);
  cfg.gridDim = dim3((unsigned)cdiv(std::min<int64_t>(budget, std::min<int64_t>(capacity, a.out_capacity)), (int64_t)rows), items);
  cfg.blockDim = dim3(256);
  cfg.dynamicSmemBytes = 0;
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  BS_CUDA(cudaLaunchKernelEx(&cfg, kv_move_kernel, a));
  return BS_OK;
}
