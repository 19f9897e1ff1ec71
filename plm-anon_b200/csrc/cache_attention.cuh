// Device helpers of the kernels of attention over a paged cache: masks, the base-2 softmax's functions, the join of
// partial results.
#pragma once

#include <type_traits>

#include "cache.cuh"
#include "cache_attention.h"

namespace plm {

constexpr int kUnreachable = 1 << 30;  // no key's index: block tables hold less than 2^30 tokens
constexpr float kLazy = 15.f;          // log2 of how far a weight may pass 1 before its row's maximum is raised: f16 holds it
constexpr float kUsual = 45.f;         // log2 of scales between whose keys weights of 2^-30 of the largest are floats
constexpr float kLeastScale = 7.888609052210118e-31f;  // 2^-100: smaller value scales count as this

// 2^x by the special-function unit (relative error 2^-22; -inf gives +0, NaN stays).
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// log2 of a normal number by the special-function unit (absolute error 2^-22): exact for powers of two.
__device__ __forceinline__ float lg2(float x) {
  float y;
  asm("lg2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// 1 / x of a normal number (1 ulp).
__device__ __forceinline__ float rcp(float x) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// In e4m3 pages the scales s of two values may lie so far apart that the weight w = 2^(score + log2 s - m) of one is no
// float, although its share w / s of the sum l is as large as the other one's: a block of zeros (s = 2^-100) beside values
// of 10^11. That share, 2^(score - m), from x = score + log2 s - m and log2 s:
__device__ __forceinline__ float small_share(float x, float log_v) {
  constexpr float kLift = 50.f;
  return ex2(x - log_v + kLift) * 8.881784197001252e-16f;  // 2^-50
}
// 2^x as a factor of partial results: of l by its root twice, as l 2^x may be a float where 2^x is none.
struct Keep {
  float root;
  __device__ __forceinline__ explicit Keep(float x) : root(ex2(0.5f * x)) {}
  __device__ __forceinline__ float o() const { return root * root; }
  __device__ __forceinline__ float l(float l) const { return l * root * root; }
};
// Two floats rounded to the 16-bit type M, `lo` in the low half.
template <typename M>
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
  uint32_t out;
  if constexpr (std::is_same<M, __nv_bfloat16>::value)
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(out) : "f"(hi), "f"(lo));
  else
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(out) : "f"(hi), "f"(lo));
  return out;
}
// Pairs of floats in one instruction.
struct f32x2 {
  uint64_t v;
};
__device__ __forceinline__ f32x2 pair(float lo, float hi) {
  f32x2 r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r.v) : "f"(lo), "f"(hi));
  return r;
}
__device__ __forceinline__ void unpair(f32x2 x, float& lo, float& hi) {
  asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(x.v));
}
__device__ __forceinline__ f32x2 fma2(f32x2 a, f32x2 b, f32x2 c) {
  f32x2 r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r.v) : "l"(a.v), "l"(b.v), "l"(c.v));
  return r;
}
__device__ __forceinline__ f32x2 mul2(f32x2 a, f32x2 b) {
  f32x2 r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
  return r;
}
__device__ __forceinline__ f32x2 add2(f32x2 a, f32x2 b) {
  f32x2 r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
  return r;
}
// 4-byte asynchronous copy; `valid` false zero-fills.
__device__ __forceinline__ void cp_async_4(void* smem_dst, const void* src, bool valid) {
  const int size = valid ? 4 : 0;
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(smem_u32(smem_dst)), "l"(src), "r"(size) : "memory");
}

// The power of two that queries of a bf16 row are divided by to become f16, 2^e: the row's largest magnitude (`top`, as
// bf16 bits) comes into [2^14, 2^15), so all 8 bits of every element down to 2^-30 of it are kept. 0 for rows of zeros
// or of non-finite numbers.
__device__ __forceinline__ int query_exponent(uint32_t top) {
  if (top == 0 || top >= 0x7f80u) return 0;
  return max(int(top >> 7) - 127 - 14, -126);
}
__device__ __forceinline__ float power_of_two_f32(int e) { return __uint_as_float(uint32_t(127 + e) << 23); }

// Whether element `at` of a word of e4m3 codes (4) or of the model dtype (2) is no finite number.
template <typename T, bool E4M3>
__device__ __forceinline__ bool non_finite(uint32_t word, int at) {
  if (E4M3) return ((word >> (8 * at)) & 0x7fu) == 0x7fu;
  const uint32_t bits = std::is_same<T, __nv_bfloat16>::value ? 0x7f80u : 0x7c00u;
  return ((word >> (16 * at)) & bits) == bits;
}
template <typename T, bool E4M3>
__device__ __forceinline__ float element_f32(uint32_t word, int at) {
  if (E4M3) {
    const uint32_t h = e4m3x2_to_f16x2(uint16_t((word >> (8 * at)) & 0xffu));
    return __low2float(*reinterpret_cast<const __half2*>(&h));
  }
  const uint16_t x = uint16_t(word >> (16 * at));
  return to_f32<T>(*reinterpret_cast<const T*>(&x));
}

// What one row sees: keys [first, last], keys below the sinks up to `last`, and its own block.
struct RowMask {
  int first, last, own_first, own_last;
  __device__ __forceinline__ bool sees(int kv, int sinks) const {
    return (kv <= last && (kv >= first || kv < sinks)) || (kv >= own_first && kv <= own_last);
  }
};
__device__ __forceinline__ RowMask no_row() { return {kUnreachable, -1, kUnreachable, -1}; }

// Row j of the sequence.
__device__ __forceinline__ RowMask row_mask(const CacheAttnArgs& a, const SeqRange& r, int j) {
  int64_t depth = j, own = kUnreachable;
  if (a.depth != nullptr) {
    depth = a.depth[r.start + j];
    own = a.own_start[r.start + j];
  }
  const bool in_own = own <= j;
  const int64_t pos = r.context + depth + (in_own ? j - own : 0);
  RowMask m;
  m.last = int(min(r.context + depth, r.context + r.n - 1));
  m.first = a.window > 0 ? int(min(max(pos - a.window + 1, int64_t(0)), int64_t(kUnreachable))) : 0;
  m.own_first = in_own ? int(max(r.context + own, int64_t(0))) : kUnreachable;
  m.own_last = int(r.context) + j;
  return m;
}

// What rows j0..j1 of a sequence see together: keys [lo, end) and those below `sinks`; every row sees all of
// [full_lo, full_end). In chunks of `kChunk` keys: first the sinks', then those of [lo, end).
struct TileKeys {
  int lo, end, full_lo, full_end, sinks, sink_chunks, skip, chunks;
  template <int kChunk>
  __device__ __forceinline__ void count() {
    sink_chunks = min((sinks + kChunk - 1) / kChunk, lo / kChunk);
    skip = (lo / kChunk - sink_chunks) * kChunk;  // keys between the sinks' chunks and the others
    chunks = sink_chunks + max((end + kChunk - 1) / kChunk - lo / kChunk, 0);
  }
  template <int kChunk>
  __device__ __forceinline__ int key(int chunk) const {
    return chunk * kChunk + (chunk < sink_chunks ? 0 : skip);
  }
  __device__ __forceinline__ bool needed(int kv) const { return kv < end && (kv >= lo || kv < sinks); }
  __device__ __forceinline__ bool all_needed(int kv, int n) const { return kv + n <= end && (kv >= lo || kv + n <= sinks); }
  __device__ __forceinline__ bool all_seen(int kv, int n) const {
    return kv + n <= full_end && (kv >= full_lo || kv + n <= sinks);
  }
};

__device__ __forceinline__ TileKeys causal_keys(const CacheAttnArgs& a, const SeqRange& r, int j0, int j1) {
  TileKeys t;
  const int context = int(r.context);
  t.lo = a.window > 0 ? max(0, context + j0 - a.window + 1) : 0;
  t.full_lo = a.window > 0 ? max(0, context + j1 - a.window + 1) : 0;
  t.full_end = context + j0 + 1;
  t.end = context + j1 + 1;
  t.sinks = min(a.sinks, t.lo);
  return t;
}

// One more row, masked by depth and own_start (starting from lo and full_end kUnreachable, full_lo 0).
__device__ __forceinline__ void widen(TileKeys& t, const RowMask& m) {
  t.lo = min(t.lo, min(m.first, m.own_first));
  t.full_lo = max(t.full_lo, m.first);
  t.full_end = min(t.full_end, m.last + 1);
}

// N neighbouring elements of packed row i (row i / group, query head i % group of the kv head) of a sequence that starts
// at row0, divided by the row's sum.
template <typename T, int N>
__device__ __forceinline__ void store_row(const CacheAttnArgs& a, int row0, int i, int head, int hd, int d,
                                          const float (&sum)[N], float total) {
  const float inv = total == 0.f ? 0.f : 1.f / total;
  T* dst = static_cast<T*>(a.out) + (row0 + i / a.group) * a.out_stride + (head * a.group + i % a.group) * hd + d;
#pragma unroll
  for (int e = 0; e < N; e += 2) reinterpret_cast<uint32_t*>(dst)[e / 2] = pack2<T>(sum[e] * inv, sum[e + 1] * inv);
}

// Adds up the parts of a row in order and stores it: one warp. part(i) is part i's floats, its O row `at` floats in and
// its (m, l) at `ml`. The maxima first, all at once, so that the parts' rows are on their way together.
template <int HD, typename T, typename Part>
__device__ __forceinline__ void join_row(const CacheAttnArgs& a, int count, Part part, int at, int ml, int row0, int i,
                                         int head) {
  const int lane = threadIdx.x & 31;
  constexpr int N = HD / 32;
  float top = -INFINITY;
  for (int x = lane; x < count; x += 32) top = fmaxf(top, part(x)[ml]);
  top = warp_max(top);
  const float from = top == -INFINITY ? 0.f : top;
  float sum[N] = {}, total = 0.f;
  for (int base = 0; base < count; base += 32) {
    float2 mine = make_float2(-INFINITY, 0.f);
    if (base + lane < count) mine = *reinterpret_cast<const float2*>(part(base + lane) + ml);
    const Keep keep(mine.x - from);
    const float f = keep.o();
    const int here = min(32, count - base);
#pragma unroll 8
    for (int x = 0; x < here; ++x) {
      const float* src = part(base + x) + at + lane * N;
      float v[N];
      if constexpr (N == 4) *reinterpret_cast<float4*>(v) = *reinterpret_cast<const float4*>(src);
      else *reinterpret_cast<float2*>(v) = *reinterpret_cast<const float2*>(src);
      const float w = __shfl_sync(0xffffffffu, f, x);
#pragma unroll
      for (int e = 0; e < N; ++e) sum[e] = fmaf(w, v[e], sum[e]);
    }
    total += warp_sum(keep.l(mine.y));
  }
  store_row<T>(a, row0, i, head, HD, lane * N, sum, total);
}

}  // namespace plm
