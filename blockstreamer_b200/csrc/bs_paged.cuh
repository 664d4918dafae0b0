// The paged key/value cache as the attention kernels see it, and the warp-level
// tensor-core pieces they share.
#pragma once

#include "bs_common.cuh"
#include "bs_ptx.cuh"

namespace bs {

// Division by a page size: shift when it is a power of two, else a 32-bit
// divide (slots are below 2^31).
struct PageDiv {
  int size, shift;  // shift < 0: not a power of two
  __device__ __forceinline__ void split(int slot, int& page, int& row) const {
    page = shift >= 0 ? slot >> shift : slot / size;
    row = slot - page * size;
  }
};

struct PagedCache {
  __nv_bfloat16* k;
  __nv_bfloat16* v;
  int64_t kp, ks, kh, vp, vs, vh;  // strides in elements: page, slot, head
  const int32_t* table;
  int64_t table_stride;
  const int32_t* lens;
  int pages, heads, dim, capacity;  // capacity: slots of a sequence's table row
  PageDiv div;
  int* status;

  // Committed length of sequence b, clamped so that `extra` slots follow it.
  __device__ __forceinline__ int len(int b, int extra) const {
    const int n = lens[b];
    const int top = capacity - extra;
    if (n < 0 || n > top) {
      record_status(status, BS_ERR_CAPACITY);
      return n < 0 ? 0 : top;
    }
    return n;
  }
  // Page of a slot below capacity, clamped into the pool.
  __device__ __forceinline__ int page_of(int b, int index) const {
    const int p = __ldg(table + b * table_stride + index);
    if ((unsigned)p >= (unsigned)pages) {
      record_status(status, BS_ERR_CAPACITY);
      return p < 0 ? 0 : pages - 1;
    }
    return p;
  }
};

// Checks a bs_kv_cache and fills the kernels' form of it (attention.cu).
int paged_cache(const char* fn, const bs_kv_cache* c, int64_t extra, bool need_v, PagedCache* out);

// TMA descriptors of K and V (attention.cu): boxes of `rows` slots of one page
// and head by 64 values, 128B-swizzled.  `rows` is the largest power of two that
// divides the page size, at most `most`; below 8 (one swizzle atom) there is no
// such box and the kernels copy 16 bytes at a time.
struct CacheMaps {
  CUtensorMap k, v;
};
int cache_box_rows(const bs_kv_cache* c, int most);
int cache_maps(const bs_kv_cache* c, int rows, bool need_v, CacheMaps* out);

// What the split of a call's keys over CTAs goes by: items are (sequence, kv
// head, row tile), in that order.
struct SplitArgs {
  PagedCache c;
  const int32_t* pos;    // positions of the drafted tokens [B, T] (attention only)
  int B, Hkv, tiles;
  int T;                 // slots behind the committed ones
  int window;
  int box;               // slots of a TMA box, or 1
  int setup;             // what starting an item costs, in units: it is counted as so many more
  int min_chunk;         // units of a CTA at least
  int fixed;             // not 0: every item counts as so many units and no CTA's range cuts one
};

// The keys of a sequence: n committed; slots [low, hi) may be attended; units
// start at lo, low rounded down to where a TMA box may start.
struct Keys {
  int n, low, lo, hi;
};
__device__ __forceinline__ Keys keys_of(const SplitArgs& a, int b) {
  Keys k;
  k.n = a.c.len(b, a.T);
  k.hi = k.n + a.T;
  k.low = a.window ? max(0, k.n - a.window + 1) : 0;
  k.lo = k.low & -a.box;
  return k;
}
// Whether a slot holds a key that some row may attend (others may hold anything).
__device__ __forceinline__ bool holds_key(const SplitArgs& a, int b, const Keys& k, int slot) {
  return slot >= k.low && (slot < k.n || (slot < k.hi && __ldg(a.pos + (int64_t)b * a.T + slot - k.n) >= 0));
}
// Whether the box from `slot` on holds a committed key or a draft in use.  Asked where its
// page lies outside the pool: the page table may hold anything behind the last one.
__device__ __forceinline__ bool box_in_use(const SplitArgs& a, int b, int n, int slot) {
  bool used = slot < n;
  const int end = min(slot - n + a.box, a.T);
#pragma unroll 1
  for (int u = slot - n; u < end && !used; ++u) used = __ldg(a.pos + (int64_t)b * a.T + u) >= 0;
  return used;
}

// Where the work of CTA `cta` of `grid` lies: its range [p0, p1) of the units of
// all items, item by item, and the sequence that holds unit p0.  An item has
// `setup` units that stand for its start (Q, masks, epilogue), then one for each
// kU keys.  The CTA's first 128 threads call.
struct Range {
  int64_t p0, p1, chunk;
  int b;           // sequence of unit p0
  int64_t before;  // units of the sequences before b
};
template <int kU>
__device__ __forceinline__ int64_t units_of(const SplitArgs& a, int b) {
  if (a.fixed) return a.fixed;
  const Keys k = keys_of(a, b);
  return a.setup + (k.hi - k.lo + kU - 1) / kU;
}
__device__ __forceinline__ int64_t chunk_of(const SplitArgs& a, int64_t total, int grid) {
  const int64_t chunk = max((int64_t)a.min_chunk, (total + grid - 1) / grid);
  return a.fixed ? (chunk + a.fixed - 1) / a.fixed * a.fixed : chunk;
}
// A whole warp waits; false when the wait of some lane ran out.
__device__ __forceinline__ bool warp_wait(uint32_t bar, uint32_t parity, volatile int* abort) {
  return __all_sync(0xffffffffu, ptx::mbar_wait(bar, parity, abort));
}
__device__ __forceinline__ void sync128() { asm volatile("bar.sync 1, 128;" ::: "memory"); }
template <int kU>
__device__ Range locate(const SplitArgs& a, int cta, int grid, int64_t* sums /* smem [6] */) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t per = (int64_t)a.Hkv * a.tiles;
  Range r = {};
  int64_t total = 0;
  if (a.B > 128) {
    for (int b = threadIdx.x; b < a.B; b += 128) total += units_of<kU>(a, b) * per;
#pragma unroll
    for (int o = 16; o; o >>= 1) total += __shfl_xor_sync(0xffffffffu, total, o);
    if (lane == 0) sums[warp] = total;
    sync128();
    total = sums[0] + sums[1] + sums[2] + sums[3];
  }
  // a scan of the sequences' units, 128 at a time (one step gives the total too)
  int64_t run = 0;
  for (int base = 0; base < a.B; base += 128) {
    const int b = base + threadIdx.x;
    const int64_t w = b < a.B ? units_of<kU>(a, b) * per : 0;
    int64_t incl = w;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int64_t v = __shfl_up_sync(0xffffffffu, incl, o);
      if (lane >= o) incl += v;
    }
    sync128();
    if (lane == 31) sums[warp] = incl;
    sync128();
    int64_t start = run + incl - w;
    for (int i = 0; i < warp; ++i) start += sums[i];
    run += sums[0] + sums[1] + sums[2] + sums[3];
    if (base == 0) {
      if (a.B <= 128) total = run;
      r.chunk = chunk_of(a, total, grid);
      r.p0 = min(total, cta * r.chunk);
      r.p1 = min(total, r.p0 + r.chunk);
      if (r.p0 >= r.p1) return r;
    }
    if (w > 0 && start <= r.p0 && r.p0 < start + w) sums[4] = b, sums[5] = start;
    if (run > r.p0) break;
  }
  sync128();
  r.b = (int)sums[4];
  r.before = sums[5];
  return r;
}

// The pieces of a CTA's range, one per item that it touches; pieces without keys
// are passed over.
struct Walk {
  int b, h, tile;
  Keys k;
  int u;               // the caller's next unit
  int start, end;      // units of keys of this piece
  int units;           // units of keys of the item
  int len;             // of the piece, with the units that stand for the start
  int64_t left;        // of the range, this piece included
  __device__ __forceinline__ bool whole() const { return start == 0 && end == units; }
};
template <int kU>
__device__ __forceinline__ bool walk_piece(const SplitArgs& a, Walk& w, int first) {
  w.units = (w.k.hi - w.k.lo + kU - 1) / kU;
  const int lead = a.fixed ? a.fixed - w.units : a.setup;
  w.len = (int)min((int64_t)(w.units + lead - first), w.left);
  w.start = max(0, first - lead);
  w.end = max(0, first + w.len - lead);
  return w.end > w.start;
}
// The next piece of the range; false at its end.
template <int kU>
__device__ __forceinline__ bool walk_next(const SplitArgs& a, Walk& w) {
  while (true) {
    w.left -= w.len;
    if (w.left <= 0) return false;
    if (++w.tile == a.tiles) {
      w.tile = 0;
      if (++w.h == a.Hkv) {
        w.h = 0;
        ++w.b;
        w.k = keys_of(a, w.b);
      }
    }
    if (walk_piece<kU>(a, w, 0)) return true;
  }
}
template <int kU>
__device__ __forceinline__ bool walk_begin(const SplitArgs& a, const Range& r, Walk& w) {
  w.b = r.b;
  w.k = keys_of(a, r.b);
  const int64_t units = units_of<kU>(a, r.b);
  const int64_t rel = r.p0 - r.before;
  const int item = (int)(rel / units);
  w.h = item / a.tiles;
  w.tile = item - w.h * a.tiles;
  w.left = r.p1 - r.p0;
  return walk_piece<kU>(a, w, (int)(rel - item * units)) || walk_next<kU>(a, w);
}

namespace mma {

__device__ __forceinline__ void ldsm_x4(uint32_t addr, uint32_t r[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ void ldsm_x4_trans(uint32_t addr, uint32_t r[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
// d[16 x 8] += a[16 x 16] b[16 x 8], bf16 in, f32 accumulate.
__device__ __forceinline__ void bf16_16816(float d[4], const uint32_t a[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
      "{%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float max3(float a, float b, float c) {
  float y;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(y) : "f"(a), "f"(b), "f"(c));
  return y;
}
// a * b + c and a + b on two values at once.
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  float2 r;
  asm("{\n\t.reg .b64 x, y, z;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\tmov.b64 z, {%6, %7};\n\t"
      "fma.rn.f32x2 x, x, y, z;\n\tmov.b64 {%0, %1}, x;\n\t}"
      : "=f"(r.x), "=f"(r.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
  return r;
}
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float c) { return fma2(a, b, make_float2(c, c)); }
__device__ __forceinline__ float2 fma2(float2 a, float b, float c) { return fma2(a, make_float2(b, b), c); }
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
  float2 r;
  asm("{\n\t.reg .b64 x, y;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\t"
      "add.rn.f32x2 x, x, y;\n\tmov.b64 {%0, %1}, x;\n\t}"
      : "=f"(r.x), "=f"(r.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return r;
}
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
  float2 r;
  asm("{\n\t.reg .b64 x, y;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\t"
      "mul.rn.f32x2 x, x, y;\n\tmov.b64 {%0, %1}, x;\n\t}"
      : "=f"(r.x), "=f"(r.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return r;
}
// The larger, NaN where either is.
__device__ __forceinline__ float max_nan(float a, float b) {
  float y;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(y) : "f"(a), "f"(b));
  return y;
}
// 2^x on the FMA pipe for x up to 126: x = n + f with n the nearest integer, a quartic
// for 2^f on [-1/2, 1/2] fitted here to the least largest relative error (2.6e-6), times
// 2^n, whose bits are the low ones of the rounding sum moved to the exponent.  As with
// ex2.approx.ftz, what lies below the normal numbers is 0 (n of -127 has the exponent
// bits 0, so a masked score of -inf has no weight at all) and NaN gives NaN.
// The special-function unit gives 16 exponentials per clock and SM; a share of them
// computed here shortens a softmax step, and the weights are rounded to bf16.
__device__ __forceinline__ float2 exp2_poly(float2 x) {
  x.x = max_nan(x.x, -127.f);
  x.y = max_nan(x.y, -127.f);
  constexpr float kRound = 12582912.f + 127.f;  // 1.5 * 2^23 and the exponent's bias
  const float2 t = add2(x, make_float2(kRound, kRound));
  const float2 n = add2(t, make_float2(-kRound, -kRound));
  const float2 f = add2(x, make_float2(-n.x, -n.y));
  float2 y = fma2(f, make_float2(0.009570102207362652f, 0.009570102207362652f), 0.05591785907745361f);
  y = fma2(y, f, 0.240247443318367f);
  y = fma2(y, f, 0.6931217908859253f);
  y = fma2(y, f, 0.9999992847442627f);
  return mul2(y, make_float2(__uint_as_float(__float_as_uint(t.x) << 23), __uint_as_float(__float_as_uint(t.y) << 23)));
}
// 16-byte asynchronous copy; zero bytes are read and zeros written when !on.
__device__ __forceinline__ void cp_async_16_or_zero(uint32_t dst, const void* src, bool on) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(on ? 16 : 0)
               : "memory");
}

// Byte offset of 16-byte chunk `c` of row `r` in a tile of kR rows: panels of 64
// values (128 bytes a row), chunks permuted within the row by the row's low three
// bits.  It is the layout of a 128B-swizzled TMA box and of the tensor-core
// descriptors, and leaves ldmatrix without bank conflicts.
template <int kR>
__device__ __forceinline__ uint32_t tile_at(int r, int c) {
  return (uint32_t)((c >> 3) * (kR * 128) + r * 128 + (((c & 7) ^ (r & 7)) << 4));
}

}  // namespace mma
}  // namespace bs
