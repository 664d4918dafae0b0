// Rotary positions (transformers models/gpt_oss/modeling_gpt_oss.py,
// _apply_rotary_emb): the first `rot` values of every head turned pairwise by
// the angle whose cosine and sine are table[position][pair],
//   (a, b) -> (a c - b s, b c + a s),
// the gradient being the same turn with -s, and the serving form, which also
// puts the turned key and the value into their slots of the paged cache.
//
// HBM-bound: each value is read and written once (one table row of rot * 4
// bytes per token beside the heads' Hq + Hk rows).  A group of threads takes one
// token, each thread the same 16-byte column of several heads, so that a
// thread's cosines and sines are loaded once per token; the loads of three heads
// are in flight together (8192 tokens, 64 + 8 heads of 64: 36 us one after the
// other, 28.4 us so, 5.4 TB/s or 82% of the measured copy rate).  Where a half's start or
// a row is off the 16 bytes an access takes one value (two of neighbouring pairs): rot 40 of
// heads of 80 in halves 118 us, 36.5 in neighbouring pairs, for a floor of 29.
#include "bs_paged.cuh"

namespace bs {
namespace {

template <typename T>
struct HeadsOf {
  T* p;
  int64_t b, t, h;
  __device__ __forceinline__ T* at(int64_t bi, int64_t ti, int hi) const { return p + bi * b + ti * t + hi * h; }
};

template <typename T>
struct RopeArgs {
  HeadsOf<const T> q, k, v;
  HeadsOf<T> qo, ko;
  const float* table;
  const void* pos;
  int64_t max_pos, tokens;  // tokens = B * T
  int T_, Hq, Hk, D, rot, pos64, group;
  float sign;
  int* status;
  PagedCache cache;  // append only
};

// V values of type T: one 16-byte access, or single values.
template <typename T, int V>
struct Chunk {
  T x[V];
  __device__ __forceinline__ void load(const T* p) {
    if constexpr (V * sizeof(T) == 16) {
      *reinterpret_cast<uint4*>(x) = __ldg(reinterpret_cast<const uint4*>(p));
    } else {
#pragma unroll
      for (int i = 0; i < V; ++i) x[i] = p[i];
    }
  }
  __device__ __forceinline__ void store(T* p) const {
    if constexpr (V * sizeof(T) == 16) {
      *reinterpret_cast<uint4*>(p) = *reinterpret_cast<const uint4*>(x);
    } else {
#pragma unroll
      for (int i = 0; i < V; ++i) p[i] = x[i];
    }
  }
  __device__ __forceinline__ void zero() {
#pragma unroll
    for (int i = 0; i < V; ++i) x[i] = T(0.f);
  }
};
__device__ __forceinline__ float val(float x) { return x; }
__device__ __forceinline__ float val(__nv_bfloat16 x) { return __bfloat162float(x); }
template <typename T>
__device__ __forceinline__ T rounded(float x);
template <>
__device__ __forceinline__ float rounded<float>(float x) { return x; }
template <>
__device__ __forceinline__ __nv_bfloat16 rounded<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }

// V: values of an access; INTER: pairs are neighbours, else rot/2 apart.
// A head is cut into units: pair units (two chunks rot/2 apart, or one chunk of
// neighbouring pairs) and, beyond rot, copied chunks.
template <typename T, int V, bool INTER, bool APPEND>
__global__ void __launch_bounds__(128) rope_kernel(const __grid_constant__ RopeArgs<T> a) {
  constexpr int kPairs = INTER ? V / 2 : V, kBatch = 3;
  const int turned = INTER ? a.rot / V : a.rot / 2 / V;
  const int units = turned + (a.D - a.rot) / V;
  const int wide = min(units, a.group);
  const int heads_at_once = a.group / wide;
  const int lane = threadIdx.x % a.group;
  const int u0 = lane % wide, h0 = lane / wide;
  for (int64_t n = (int64_t)blockIdx.x * (blockDim.x / a.group) + threadIdx.x / a.group; n < a.tokens;
       n += (int64_t)gridDim.x * (blockDim.x / a.group)) {
    const int64_t b = n / a.T_, t = n - b * a.T_;
    const int64_t pos = a.pos64 ? static_cast<const int64_t*>(a.pos)[n] : static_cast<const int32_t*>(a.pos)[n];
    const bool used = pos >= 0 && pos < a.max_pos;
    if (pos >= a.max_pos && lane == 0) record_status(a.status, BS_ERR_INVALID_ARGUMENT);
    // where the token's key and value go in the cache
    bool write = false;
    int64_t koff = 0, voff = 0;
    if constexpr (APPEND) {
      // (the length decides, not the slot: a bad one drops all rows of its sequence)
      const int len = a.cache.lens[b];
      write = used && len >= 0 && len <= a.cache.capacity - a.T_;
      int page, row;
      a.cache.div.split(write ? len + (int)t : 0, page, row);
      int p = write ? __ldg(a.cache.table + b * a.cache.table_stride + page) : 0;
      write = write && (unsigned)p < (unsigned)a.cache.pages;
      if (used && !write && lane == 0) record_status(a.status, BS_ERR_CAPACITY);
      koff = p * a.cache.kp + row * a.cache.ks;
      voff = p * a.cache.vp + row * a.cache.vs;
    }
    for (int u = h0 < heads_at_once ? u0 : units; u < units; u += wide) {
      const bool turn = u < turned;
      const int c = turn ? u * V : a.rot + (u - turned) * V;
      float cs[2 * kPairs];
      if (turn && used) {
        const float* row = a.table + pos * a.rot + u * 2 * kPairs;
        if constexpr (kPairs % 2 == 0) {
#pragma unroll
          for (int i = 0; i < kPairs / 2; ++i)
            reinterpret_cast<float4*>(cs)[i] = __ldg(reinterpret_cast<const float4*>(row) + i);
        } else {
#pragma unroll
          for (int i = 0; i < kPairs; ++i) cs[2 * i] = row[2 * i], cs[2 * i + 1] = row[2 * i + 1];
        }
#pragma unroll
        for (int i = 0; i < kPairs; ++i) cs[2 * i + 1] *= a.sign;
      }
      // kBatch heads at a time: their loads are in flight together
      for (int hb = h0; hb < a.Hq + a.Hk; hb += kBatch * heads_at_once) {
        Chunk<T, V> x[kBatch], y[INTER ? 1 : kBatch];
        const bool two = turn && !INTER;
#pragma unroll
        for (int j = 0; j < kBatch; ++j) {
          const int h = min(hb + j * heads_at_once, a.Hq + a.Hk - 1);
          const T* src = (h < a.Hq ? a.q.at(b, t, h) : a.k.at(b, t, h - a.Hq)) + c;
          x[j].load(src);
          if constexpr (!INTER) y[j].load(two ? src + a.rot / 2 : src);
        }
#pragma unroll
        for (int j = 0; j < kBatch; ++j) {
          const int h = hb + j * heads_at_once;
          if (h >= a.Hq + a.Hk) continue;
          const bool isq = h < a.Hq;
          T* dst;
          if constexpr (APPEND) {
            if (!isq && !write) continue;
            dst = isq ? a.qo.at(b, t, h)
                      : reinterpret_cast<T*>(a.cache.k) + koff + (int64_t)(h - a.Hq) * a.cache.kh;
          } else {
            dst = isq ? a.qo.at(b, t, h) : a.ko.at(b, t, h - a.Hq);
          }
          Chunk<T, V>& u0 = x[j];
          Chunk<T, V>& u1 = y[INTER ? 0 : j];
          if (!used) {
            u0.zero();
            if (two) u1.zero();
          } else if (turn) {
#pragma unroll
            for (int i = 0; i < kPairs; ++i) {
              const float p = val(INTER ? u0.x[2 * i] : u0.x[i]);
              const float r = val(INTER ? u0.x[2 * i + 1] : u1.x[i]);
              const T e = rounded<T>(p * cs[2 * i] - r * cs[2 * i + 1]);
              const T f = rounded<T>(r * cs[2 * i] + p * cs[2 * i + 1]);
              if constexpr (INTER)
                u0.x[2 * i] = e, u0.x[2 * i + 1] = f;
              else
                u0.x[i] = e, u1.x[i] = f;
            }
          }
          u0.store(dst + c);
          if (two) u1.store(dst + c + a.rot / 2);
        }
      }
    }
    if constexpr (APPEND) {
      if (write) {
        const int per = a.D / V;
        for (int i = lane; i < a.Hk * per; i += a.group) {
          const int h = i / per, c = (i - h * per) * V;
          Chunk<T, V> x;
          x.load(a.v.at(b, t, h) + c);
          x.store(reinterpret_cast<T*>(a.cache.v) + voff + (int64_t)h * a.cache.vh + c);
        }
      }
    }
  }
}

template <typename T>
bool vector_ok(const bs_heads* h, int64_t Hn) {
  const int64_t v = 16 / sizeof(T);
  return !h->ptr || ((reinterpret_cast<uintptr_t>(h->ptr) & 15) == 0 && h->stride_b % v == 0 &&
                     h->stride_t % v == 0 && (Hn <= 1 || h->stride_h % v == 0));
}

template <typename T>
HeadsOf<T> heads(const bs_heads* h) {
  return {static_cast<T*>(h->ptr), h->stride_b, h->stride_t, h->stride_h};
}
template <typename T>
HeadsOf<const T> heads_in(const bs_heads* h) {
  return {static_cast<const T*>(h->ptr), h->stride_b, h->stride_t, h->stride_h};
}

template <typename T, bool APPEND>
int rope_launch(RopeArgs<T>& a, bool vec, int interleaved, cudaStream_t st) {
  constexpr int V = 16 / sizeof(T);
  vec = vec && a.D % V == 0 && (interleaved ? a.rot % V == 0 : (a.rot / 2) % V == 0);
  // One warp per token keeps every thread's cosines and sines for all heads;
  // with fewer tokens than fill the SMs a whole block takes a token, so that
  // the latency of a few loads, not of a loop over heads, is what is left.
  a.group = a.tokens >= (int64_t)sm_count() * 16 ? 32 : 128;
  const int64_t blocks = cdiv(a.tokens, (int64_t)(128 / a.group));
  const unsigned grid = (unsigned)std::min<int64_t>(blocks, (int64_t)sm_count() * 64);
  if (vec)
    interleaved ? rope_kernel<T, V, true, APPEND><<<grid, 128, 0, st>>>(a)
                : rope_kernel<T, V, false, APPEND><<<grid, 128, 0, st>>>(a);
  else
    interleaved ? rope_kernel<T, 2, true, APPEND><<<grid, 128, 0, st>>>(a)
                : rope_kernel<T, 1, false, APPEND><<<grid, 128, 0, st>>>(a);
  BS_LAUNCHED();
  return BS_OK;
}

template <typename T>
void fill(RopeArgs<T>& a, const bs_heads* q, const bs_heads* k, const bs_heads* qo, int64_t B, int64_t T_,
          int64_t Hq, int64_t Hk, int64_t D, const float* table, int64_t max_pos, int64_t rot, const void* pos,
          int pos_dtype) {
  a = RopeArgs<T>{};
  a.q = heads_in<T>(q);
  if (k) a.k = heads_in<T>(k);
  a.qo = heads<T>(qo);
  a.table = table;
  a.pos = pos;
  a.max_pos = max_pos;
  a.tokens = B * T_;
  a.T_ = (int)T_;
  a.Hq = (int)Hq;
  a.Hk = (int)Hk;
  a.D = (int)D;
  a.rot = (int)rot;
  a.pos64 = pos_dtype == BS_I64;
  a.sign = 1.f;
  a.status = device_status_ptr();
}

int check_rope(const char* fn, const bs_heads* q, const bs_heads* q_out, int64_t B, int64_t T, int64_t Hq,
               int64_t Hk, int64_t D, const float* table, int64_t max_pos, int64_t rot, const void* positions,
               int pos_dtype) {
  BS_ARG(q && q_out && q->ptr && q_out->ptr && table && positions, "%s: null pointer", fn);
  BS_ARG(B > 0 && T > 0 && Hq > 0 && Hk >= 0 && D > 0 && max_pos > 0, "%s: bad sizes", fn);
  BS_ARG(T < INT32_MAX && Hq + Hk < (1 << 20) && D <= (1 << 16) && max_pos < INT32_MAX, "%s: sizes too large", fn);
  BS_ARG(rot > 0 && rot <= D && rot % 2 == 0 && D % 2 == 0,
         "%s: rot must be even, positive and at most the (even) head size", fn);
  BS_ARG(pos_dtype == BS_I32 || pos_dtype == BS_I64, "%s: positions must be int32 or int64", fn);
  BS_ALIGNED16(table, "table");
  return BS_OK;
}

template <typename T>
int rope_typed(const bs_heads* q, const bs_heads* k, const bs_heads* qo, const bs_heads* ko, int64_t B, int64_t T_,
               int64_t Hq, int64_t Hk, int64_t D, const float* table, int64_t max_pos, int64_t rot,
               const void* positions, int pos_dtype, int interleaved, int inverse, cudaStream_t st) {
  RopeArgs<T> a;
  fill<T>(a, q, Hk ? k : nullptr, qo, B, T_, Hq, Hk, D, table, max_pos, rot, positions, pos_dtype);
  if (Hk) a.ko = heads<T>(ko);
  a.sign = inverse ? -1.f : 1.f;
  const bool vec = vector_ok<T>(q, Hq) && vector_ok<T>(qo, Hq) && (!Hk || (vector_ok<T>(k, Hk) && vector_ok<T>(ko, Hk)));
  return rope_launch<T, false>(a, vec, interleaved, st);
}

}  // namespace
}  // namespace bs

extern "C" int bs_rope(const bs_heads* q, const bs_heads* k, const bs_heads* q_out, const bs_heads* k_out, int dtype,
                       int64_t B, int64_t T, int64_t Hq, int64_t Hk, int64_t D, const float* table, int64_t max_pos,
                       int64_t rot, const void* positions, int pos_dtype, int interleaved, int inverse,
                       void* stream) {
  using namespace bs;
  if (B == 0 || T == 0) return BS_OK;
  if (!k || !k->ptr) Hk = 0;
  BS_TRY(check_rope("bs_rope", q, q_out, B, T, Hq, Hk, D, table, max_pos, rot, positions, pos_dtype));
  BS_ARG(!Hk || (k_out && k_out->ptr), "bs_rope: null k_out");
  BS_ARG(dtype == BS_BF16 || dtype == BS_F32, "bs_rope: dtype must be bf16 or f32");
  BS_TRY(check_device());
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  if (dtype == BS_F32)
    return rope_typed<float>(q, k, q_out, k_out, B, T, Hq, Hk, D, table, max_pos, rot, positions, pos_dtype,
                             interleaved, inverse, st);
  return rope_typed<__nv_bfloat16>(q, k, q_out, k_out, B, T, Hq, Hk, D, table, max_pos, rot, positions, pos_dtype,
                                   interleaved, inverse, st);
}

extern "C" int bs_rope_append(const bs_heads* q, const bs_heads* k, const bs_heads* v, const bs_heads* q_out,
                              const bs_kv_cache* cache, int64_t T, int64_t Hq, const float* table, int64_t max_pos,
                              int64_t rot, const void* positions, int pos_dtype, int interleaved, void* stream) {
  using namespace bs;
  typedef __nv_bfloat16 E;
  BS_ARG(cache, "bs_rope_append: null cache");
  if (cache->batch == 0 || T == 0) return BS_OK;
  BS_ARG(k && v && k->ptr && v->ptr, "bs_rope_append: null pointer");
  BS_TRY(check_rope("bs_rope_append", q, q_out, cache->batch, T, Hq, cache->heads, cache->dim, table, max_pos, rot,
                    positions, pos_dtype));
  RopeArgs<E> a;
  fill<E>(a, q, k, q_out, cache->batch, T, Hq, cache->heads, cache->dim, table, max_pos, rot, positions, pos_dtype);
  a.v = heads_in<E>(v);
  BS_TRY(paged_cache("bs_rope_append", cache, T, true, &a.cache));
  BS_TRY(check_device());
  const bool vec = vector_ok<E>(q, Hq) && vector_ok<E>(q_out, Hq) && vector_ok<E>(k, cache->heads) &&
                   vector_ok<E>(v, cache->heads);
  return rope_launch<E, true>(a, vec, interleaved, reinterpret_cast<cudaStream_t>(stream));
}
