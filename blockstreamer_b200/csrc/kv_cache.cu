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
// One CTA per kKeys slots of a (sequence, kv head).  K is the 16-row operand of
// the tensor-core product, the accepted rows its columns, so that a key's sum
// over the rows stays in one lane group; no atomics, one store per slot.
// HBM-bound: 2 dim + 8 bytes per slot and kv head.  All K of the CTA is asked for
// at once (TMA boxes where pages allow, else 16-byte copies), then the queries.
struct ScoreArgs {
  PagedCache c;
  const __nv_bfloat16* q;
  int64_t qb, qt, qh;
  const float* lse;
  const int32_t* accepted;
  const float* scores;
  float* out;
  float scale2;
  int T, A, i0, rows, G, Hq, capacity, box;  // accepted entries i0 .. i0 + rows / G
};

template <int DP>
struct ScoreCfg {
  static constexpr int kUnits = DP == 64 ? 4 : 2;   // units of 32 keys per warp
  static constexpr int kKeys = 4 * 32 * kUnits;
  static constexpr int kTile = 32 * DP * 2;
  static constexpr int q = 4 * kUnits * kTile;      // then [rows] q, [rows] float2, barriers
  static int smem(int rows) { return q + rows * (DP * 2 + 8) + 4 * kUnits * 8 + 1024; }
};

template <int DP, bool kTma>
__global__ void __launch_bounds__(128) kv_scores_kernel(const __grid_constant__ ScoreArgs a,
                                                        const __grid_constant__ CacheMaps maps) {
  using Cfg = ScoreCfg<DP>;
  constexpr int KS = DP / 16, kLanesRow = DP / 8, kUnits = Cfg::kUnits;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
  __shared__ int abort_flag;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int b = blockIdx.y / a.c.heads, h = blockIdx.y - b * a.c.heads;
  const int n = a.c.len(b, a.A);
  const int rows8 = (a.rows + 7) / 8 * 8;
  const uint32_t kbase = ptx::smem_addr(smem) + warp * kUnits * Cfg::kTile;
  uint8_t* qs = smem + Cfg::q;
  float2* info = reinterpret_cast<float2*>(qs + rows8 * DP * 2);  // (lse log2(e), last slot seen)
  const uint32_t bar = ptx::smem_addr(info + rows8) + warp * kUnits * 8;
  const int first = blockIdx.x * Cfg::kKeys + warp * 32 * kUnits;
  const int top = min(a.capacity, n + a.A);
  auto qat = [&](int r, int c) { return (uint32_t)((c >> 3) * (rows8 * 128) + r * 128 + (((c & 7) ^ (r & 7)) << 4)); };

  // the scores to add to: slot of lane in each unit
  const int mine = lane / 4 + (lane & 3) * 8;
  const int64_t base = (int64_t)blockIdx.y * a.capacity;
  float before[kUnits];
#pragma unroll
  for (int u = 0; u < kUnits; ++u) {
    const int slot = first + u * 32 + mine;
    before[u] = slot < a.capacity ? a.scores[base + slot] : 0.f;
  }
  if (blockIdx.x * Cfg::kKeys < top) {
    if constexpr (kTma) {
      const int boxes = 32 / a.box, u = lane / boxes, x = lane - u * boxes;
      const int slot = first + u * 32 + x * a.box;
      const bool on = u < kUnits && first + u * 32 < top;
      int page = a.c.pages, row = 0;  // a box behind the last slot lies outside the descriptor's pages: zeros
      if (on && slot < top) {
        int p;
        a.c.div.split(slot, p, row);
        page = a.c.page_of(b, p);
      }
      if (threadIdx.x == 0) abort_flag = 0;
      if (lane < kUnits) ptx::mbar_init(bar + 8 * lane, 1);
      ptx::fence_mbar_init();
      __syncwarp();
      if (lane < kUnits && first + lane * 32 < top) ptx::mbar_arrive_expect_tx(bar + 8 * lane, Cfg::kTile);
      __syncwarp();
      if (on) {
#pragma unroll
        for (int c = 0; c < DP / 64; ++c)
          ptx::tma_load_4d(kbase + u * Cfg::kTile + c * 4096 + x * a.box * 128, &maps.k, bar + 8 * u, c * 64, h, row, page);
      }
    } else {
      if (a.c.dim < DP) {
        for (int i = threadIdx.x; i < Cfg::q / 16; i += 128) reinterpret_cast<uint4*>(smem)[i] = make_uint4(0, 0, 0, 0);
        __syncthreads();
      }
#pragma unroll
      for (int u = 0; u < kUnits; ++u) {
        const int slot = first + u * 32 + lane;
        int page = 0, row = -1;
        if (slot < top) {
          int p;
          a.c.div.split(slot, p, row);
          page = a.c.page_of(b, p);
        }
        const int c = lane % kLanesRow;
        const __nv_bfloat16* kb = a.c.k + h * a.c.kh + c * 8;
#pragma unroll
        for (int i = 0; i < kLanesRow; ++i) {
          const int r = lane / kLanesRow + i * (32 / kLanesRow);
          const int p = __shfl_sync(0xffffffffu, page, r), x = __shfl_sync(0xffffffffu, row, r);
          if (c * 8 < a.c.dim)
            mma::cp_async_16_or_zero(kbase + u * Cfg::kTile + mma::tile_at<32>(r, c),
                                     x >= 0 ? kb + p * a.c.kp + x * a.c.ks : kb, x >= 0);
        }
      }
    }
    for (int i = threadIdx.x; i < rows8 * (DP / 8); i += 128) {
      const int r = i / (DP / 8), c = i - r * (DP / 8), e = a.i0 + r / a.G;
      uint4 v = make_uint4(0, 0, 0, 0);
      float2 f = make_float2(INFINITY, __int_as_float(-1));
      if (r < a.rows) {
        const int u = a.accepted ? a.accepted[(int64_t)b * a.A + e] : e;
        if ((unsigned)u < (unsigned)a.T) {
          const int hq = h * a.G + r % a.G;
          if (c * 8 < a.c.dim)
            v = __ldg(reinterpret_cast<const uint4*>(a.q + b * a.qb + u * a.qt + hq * a.qh + c * 8));
          const float l = a.lse[((int64_t)b * a.T + u) * a.Hq + hq];
          if (l != -INFINITY) f = make_float2(l * kLog2e, __int_as_float(n + e));
        }
      }
      *reinterpret_cast<uint4*>(qs + qat(r, c)) = v;
      if (c == 0) info[r] = f;
    }
    if constexpr (!kTma) ptx::cp_async_wait_all();
    __syncthreads();
  }
  const uint32_t qaddr = ptx::smem_addr(qs);
#pragma unroll
  for (int u = 0; u < kUnits; ++u) {
    const int slot0 = first + u * 32;
    float sum[4] = {0.f, 0.f, 0.f, 0.f};  // slots slot0 + lane / 4 + 8 i
    if (slot0 < top) {
      if constexpr (kTma) {
        ptx::mbar_wait(bar + 8 * u, 0, &abort_flag);  // a wait that ran out is reported at the end
        __syncwarp();
      }
      uint32_t kf[2][KS][4];
#pragma unroll
      for (int mt = 0; mt < 2; ++mt)
#pragma unroll
        for (int k = 0; k < KS; ++k)
          mma::ldsm_x4(kbase + u * Cfg::kTile + mma::tile_at<32>(mt * 16 + (lane & 15), 2 * k + (lane >> 4)), kf[mt][k]);
      for (int r = 0; r < rows8; r += 8) {
        float s[2][4] = {};
#pragma unroll
        for (int k = 0; k < KS; k += 2) {
          uint32_t f[4];
          mma::ldsm_x4(qaddr + qat(r + (lane & 7), 2 * k + (lane >> 3)), f);
#pragma unroll
          for (int mt = 0; mt < 2; ++mt) {
            mma::bf16_16816(s[mt], kf[mt][k], f[0], f[1]);
            mma::bf16_16816(s[mt], kf[mt][k + 1], f[2], f[3]);
          }
        }
        const float2 f0 = info[r + (lane & 3) * 2], f1 = info[r + (lane & 3) * 2 + 1];
#pragma unroll
        for (int mt = 0; mt < 2; ++mt)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float2 f = e & 1 ? f1 : f0;
            const int slot = slot0 + mt * 16 + lane / 4 + (e >> 1) * 8;
            const float p = mma::exp2_fast(s[mt][e] * a.scale2 - f.x);
            sum[mt * 2 + (e >> 1)] += slot <= __float_as_int(f.y) ? p : 0.f;
          }
      }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      sum[i] += __shfl_xor_sync(0xffffffffu, sum[i], 1);
      sum[i] += __shfl_xor_sync(0xffffffffu, sum[i], 2);
    }
    const int sel = lane & 3, slot = slot0 + mine;
    const float add = sel == 0 ? sum[0] : sel == 1 ? sum[1] : sel == 2 ? sum[2] : sum[3];
    if (slot < a.capacity && (slot < top || a.out != a.scores)) a.out[base + slot] = before[u] + add;
  }
  if constexpr (kTma) {
    if (first < top && *(volatile int*)&abort_flag) {
      if (lane == 0) record_status(a.c.status, BS_ERR_TIMEOUT);
      // copies in flight end before the CTA's memory is given back
      volatile int gone = 0;
      for (int u = 0; u < kUnits && first + u * 32 < top; ++u) ptx::mbar_wait(bar + 8 * u, 0, &gone);
    }
  }
}

template <int DP, bool kTma>
int scores_launch(ScoreArgs a, const CacheMaps& maps, int64_t Hkv, int64_t B, cudaStream_t st) {
  using Cfg = ScoreCfg<DP>;
  static bool set[64] = {};
  int dev = 0;
  BS_CUDA(cudaGetDevice(&dev));
  constexpr int kMost = 128 * 1024;
  if (dev >= 64 || !set[dev]) {
    BS_CUDA(cudaFuncSetAttribute(kv_scores_kernel<DP, kTma>, cudaFuncAttributeMaxDynamicSharedMemorySize, kMost));
    if (dev < 64) set[dev] = true;
  }
  // as many accepted entries at a time as their queries fit beside the keys
  const int step = std::max(1, (kMost - Cfg::smem(0)) / (DP * 2 + 8) / 8 * 8 / a.G);
  const dim3 grid((unsigned)cdiv(a.capacity, (int64_t)Cfg::kKeys), (unsigned)(B * Hkv));
  for (a.i0 = 0; a.i0 < a.A; a.i0 += step) {
    a.rows = std::min(step, a.A - a.i0) * a.G;
    kv_scores_kernel<DP, kTma><<<grid, 128, Cfg::smem((a.rows + 7) / 8 * 8), st>>>(a, maps);
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
  // this CTA's slots [s0, s1), a multiple of 4 each
  const int per = ((n + cluster - 1) / cluster + 3) / 4 * 4;
  const int s0 = min(n, rank * per), s1 = min(n, s0 + per), mine = s1 - s0;
  const bool fits = per <= a.held;
  auto key_at = [&](int i) -> uint32_t {
    const int s = s0 + i;
    return s < a.first || s >= n - a.last ? 0xffffffffu : score_key(scores[s]);
  };
  auto key = [&](int i) -> uint32_t { return fits ? held[i] : key_at(i); };
  if (fits)
    for (int i = threadIdx.x; i < mine; i += kSel) held[i] = key_at(i);

  uint32_t prefix = 0, mask = 0;
  int need = want;  // slots still to choose among those whose key matches prefix
  if (want < n) {
    for (int pass = 0; pass < 4; ++pass) {
      const int shift = 24 - 8 * pass;
      uint32_t* hs = hist[pass & 1];
      for (int i = threadIdx.x; i < 256; i += kSel) hs[i] = 0;
      __syncthreads();
      for (int i = threadIdx.x; i < mine; i += kSel) {
        const uint32_t k = key(i);
        if ((k & mask) == prefix) atomicAdd(&hs[k >> shift & 255], 1u);
      }
      ptx::cluster_sync();
      // the digit whose bin holds the need-th highest key: warp 0, eight bins a lane from the top
      if (threadIdx.x < 32) {
        uint32_t bin[8], sum = 0;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const int d = 255 - (threadIdx.x * 8 + j);
          uint32_t v = 0;
          for (int r = 0; r < cluster; ++r) v += dsmem_u32(ptx::smem_addr(&hs[d]), r);
          bin[j] = v;
          sum += v;
        }
        uint32_t incl = sum;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const uint32_t v = __shfl_up_sync(0xffffffffu, incl, o);
          if ((int)threadIdx.x >= o) incl += v;
        }
        uint32_t above = incl - sum;
        if (above < (uint32_t)need && (uint32_t)need <= incl) {
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            if (above < (uint32_t)need && (uint32_t)need <= above + bin[j]) {
              found[0] = 255 - (threadIdx.x * 8 + j);
              found[1] = need - above;
            }
            above += bin[j];
          }
        }
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
  const int run = (mine + kSel - 1) / kSel;
  const int i0 = min(mine, (int)threadIdx.x * run), i1 = min(mine, i0 + run);
  uint32_t gt = 0, eq = 0;
  for (int i = i0; i < i1; ++i) {
    const uint32_t k = all ? 0u : key(i);
    gt += all || k > prefix;
    eq += !all && k == prefix;
  }
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  uint32_t ig = gt, ie = eq;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const uint32_t x = __shfl_up_sync(0xffffffffu, ig, o), y = __shfl_up_sync(0xffffffffu, ie, o);
    if (lane >= o) ig += x, ie += y;
  }
  if (lane == 31) warps[0][warp] = ig, warps[1][warp] = ie;
  __syncthreads();
  if (threadIdx.x == 0) {
    uint32_t x = 0, y = 0;
    for (int w = 0; w < kSel / 32; ++w) {
      const uint32_t u = warps[0][w], v = warps[1][w];
      warps[0][w] = x, warps[1][w] = y;
      x += u, y += v;
    }
    totals[0] = x, totals[1] = y;
  }
  ptx::cluster_sync();
  uint32_t bg = warps[0][warp] + ig - gt, be = warps[1][warp] + ie - eq;
  for (int r = 0; r < rank; ++r) {
    bg += dsmem_u32(ptx::smem_addr(&totals[0]), r);
    be += dsmem_u32(ptx::smem_addr(&totals[1]), r);
  }
  int32_t* kept = a.kept + (int64_t)item * a.budget;
  float* out = a.out_scores + (int64_t)item * a.out_capacity;
  for (int i = i0; i < i1; ++i) {
    const uint32_t k = all ? 0u : key(i);
    const bool more = all || k > prefix, same = !all && k == prefix;
    if (more || (same && be < (uint32_t)need)) {
      const uint32_t at = bg + min(be, (uint32_t)need);
      kept[at] = s0 + i;
      if (at < (uint32_t)a.out_capacity) out[at] = scores[s0 + i];
    }
    bg += more;
    be += same;
  }
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
  BS_ARG(cache->batch * cache->heads <= 65535, "%s: more than 65535 (sequence, kv head) pairs", fn);
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
  a.T = (int)T, a.A = (int)A, a.Hq = (int)Hq, a.capacity = (int)capacity;
  BS_TRY(check_device());
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  const int64_t D = cache->dim;
  CacheMaps maps = {};
  a.box = cache_box_rows(cache, 32);
  if (a.box >= 8) {
    BS_TRY(cache_maps(cache, a.box, false, &maps));
    return D <= 64 ? scores_launch<64, true>(a, maps, cache->heads, cache->batch, st)
                   : scores_launch<128, true>(a, maps, cache->heads, cache->batch, st);
  }
  return D <= 64 ? scores_launch<64, false>(a, maps, cache->heads, cache->batch, st)
                 : scores_launch<128, false>(a, maps, cache->heads, cache->batch, st);
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
  // CTAs per (sequence, kv head): about 8192 scores each, up to eight
  int cluster = 1;
  while (cluster < 8 && (int64_t)cluster * 8192 < capacity) cluster *= 2;
  const int64_t per = cdiv(cdiv(capacity, (int64_t)cluster), (int64_t)4) * 4;
  constexpr int kHeldMost = 48 * 1024;  // keys; longer ranges are read again for every digit
  a.held = (int)std::min<int64_t>(per, kHeldMost);
  static bool set[64] = {};
  int dev = 0;
  BS_CUDA(cudaGetDevice(&dev));
  if (dev >= 64 || !set[dev]) {
    BS_CUDA(cudaFuncSetAttribute(kv_select_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kHeldMost * 4));
    if (dev < 64) set[dev] = true;
  }
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[1];
  const unsigned items = (unsigned)(cache->batch * cache->heads);
  cfg.gridDim = dim3(items * cluster);
  cfg.blockDim = dim3(kSel);
  cfg.dynamicSmemBytes = (size_t)a.held * 4;
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
