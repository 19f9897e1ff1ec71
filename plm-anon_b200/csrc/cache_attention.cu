// Attention over a paged cache of several sequences, 16-bit or e4m3 pages, causal or under the round mask, with or
// without a sliding window and sinks.
//
// A CTA takes up to 8 NR packed rows of one kv head of one sequence (packed row i is row i / group, query head i % group
// of the kv head) and a share of the keys; its warps take turns at chunks of 16 keys. Everything is transposed, keys and
// head elements on the M side of mma.m16n8k16, packed rows on the N side:
//     S^T[16 keys, rows] = K Q^T,      O^T[d, rows] += V^T P^T,
// so 8 rows fill an instruction and a K or V element is brought into its fragment once for all rows. A product's inner
// index may be permuted if both operands are, and an output's index if the store undoes it: thread (gq, tq) =
// (lane / 4, lane % 4) takes a quarter of the elements of keys gq and gq + 8 as its part of K, and an eighth of the
// elements of keys 2 tq, 2 tq + 1, 2 tq + 8, 2 tq + 9 as its part of V, both in whole vectors of shared memory.
// P^T changes sides through movmatrix. Every warp has a ring of its own that 16-byte asynchronous copies keep full, so
// the warps of a CTA meet only at the end, where their partial results are joined, and those of a cluster's CTAs.
//
// The softmax is online in base 2 with a lazy maximum: a row's m is raised (and O, l rescaled) only when a score passes
// it by more than 2^8, so most chunks take one vote and no cross-lane maximum; weights stay below 2^8.
//
// e4m3 pages: codes become f16 exactly, and their scales never touch a 16-bit number. A key's scale multiplies its
// scores. A value's scale s enters through w = 2^(score + log2 s - m): O += w code and l += w / s, out = O / l, so that
// m follows the largest term of the sum, w <= 2^8 whatever the scales are, and rounding w to f16 (2^-11) is relative to
// that term. Queries in bf16 become f16 after their row was divided by a power of two that puts its maximum in
// [2^14, 2^15): all 8 bits of every element down to 2^-30 of the row's maximum.
// 16-bit pages: products in the model dtype, w rounded to it, as in round_attention_kernel.
//
// Masks. Keys that no row of the CTA sees are not loaded (their registers are zero, so stale slots, or pages that were
// given away, are never read). Where rows differ in what they see, a masked score is -inf, its weight 0; 0 times a
// non-finite value would still be NaN, so such chunks are searched for non-finite values, which are added to the rows
// that see them by hand and replaced by 0.
#include <type_traits>

#include "cache.cuh"
#include "cache_attention.h"

namespace plm {
namespace {

constexpr int kWarps = 8;
constexpr int kThreads = 32 * kWarps;
constexpr int kChunk = 16;          // keys
constexpr int kMaxSplits = 8;       // CTAs of a portable cluster
constexpr int kUnreachable = 1 << 30;
constexpr float kLazy = 8.f;        // log2 of how far a weight may pass 1
constexpr int kStages = 3;          // chunks of a warp's ring

template <typename M>
__device__ __forceinline__ void mma_16816(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                          uint32_t b0, uint32_t b1) {
  if constexpr (std::is_same<M, __nv_bfloat16>::value) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  } else {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  }
}
// 2^x by the special-function unit (relative error ~2^-22; -inf gives +0, NaN stays).
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ uint32_t transpose_8x8(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}
template <typename M>
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
  const M l = from_f32<M>(lo), h = from_f32<M>(hi);
  return uint32_t(*reinterpret_cast<const uint16_t*>(&l)) | (uint32_t(*reinterpret_cast<const uint16_t*>(&h)) << 16);
}

// A chunk of 16 keys in shared memory: K rows, then V rows, then (e4m3) the 16 key scales and the 16 value scales. Rows
// are vectors of 16 bytes, vector c of row `key` at c ^ swizzle(key), so that the eight threads of a load's phase (two
// neighbouring gq, four tq) meet eight different groups of banks both in K (rows gq) and in V (rows 2 tq + const).
template <int HD, bool E4M3>
struct Chunk {
  static constexpr int ES = E4M3 ? 1 : 2;
  static constexpr int VECS = HD * ES / 16;  // vectors of a row
  static constexpr int PLANE = kChunk * HD * ES;
  static constexpr int BYTES = 2 * PLANE + (E4M3 ? 2 * kChunk * 4 : 0);
  static constexpr int KW = HD / 4 * ES / 4;  // words a thread holds of a key
  static constexpr int VW = HD / 8 * ES / 4;  // and of a value
  static __device__ __forceinline__ int swizzle(int key) {
    if (!E4M3) return ((key & 1) << 2) | ((key >> 1) & 3);
    return VECS == 8 ? key & 7 : (key >> 1) & 3;
  }
  static __device__ __forceinline__ int at(int key, int vec) { return key * (HD * ES) + ((vec ^ swizzle(key)) << 4); }
  // Vector i of thread tq's part of a key, and the first of the 16 / ES elements in it.
  static __device__ __forceinline__ int k_vec(int tq, int i) { return E4M3 ? tq * VECS / 4 + i : tq + 4 * i; }
  // Thread gq's element 2 t of its part of a value.
  static __device__ __forceinline__ int v_vec(int gq, int i) {
    if (E4M3) return VECS == 8 ? gq : gq >> 1;
    return (((gq & 1) << 2) | (gq >> 1)) + 8 * i;
  }
  static __device__ __forceinline__ int v_element(int gq, int t) {
    return E4M3 ? gq * (HD / 8) + 2 * t : v_vec(gq, t / 4) * 8 + (t % 4) * 2;
  }
  static __device__ __forceinline__ void read_key(uint32_t (&r)[KW], const uint8_t* plane, int key, int tq) {
#pragma unroll
    for (int i = 0; i < KW / 4; ++i) {
      const uint4 x = *reinterpret_cast<const uint4*>(plane + at(key, k_vec(tq, i)));
      r[4 * i] = x.x;
      r[4 * i + 1] = x.y;
      r[4 * i + 2] = x.z;
      r[4 * i + 3] = x.w;
    }
  }
  static __device__ __forceinline__ void read_value(uint32_t (&r)[VW], const uint8_t* plane, int key, int gq) {
    if constexpr (VW == 2) {
      const uint2 x = *reinterpret_cast<const uint2*>(plane + at(key, v_vec(gq, 0)) + (gq & 1) * 8);
      r[0] = x.x;
      r[1] = x.y;
    } else {
#pragma unroll
      for (int i = 0; i < VW / 4; ++i) {
        const uint4 x = *reinterpret_cast<const uint4*>(plane + at(key, v_vec(gq, i)));
        r[4 * i] = x.x;
        r[4 * i + 1] = x.y;
        r[4 * i + 2] = x.z;
        r[4 * i + 3] = x.w;
      }
    }
  }
};

// 4-byte asynchronous copy; `valid` false zero-fills.
__device__ __forceinline__ void cp_async_4(void* smem_dst, const void* src, bool valid) {
  const int size = valid ? 4 : 0;
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(smem_u32(smem_dst)), "l"(src), "r"(size) : "memory");
}

// What one packed row sees, as logical indices below 2^30: [first, last] and below `sinks`, and the own block.
struct RowMask {
  int first, last, own_first, own_last;
  __device__ __forceinline__ bool sees(int kv, int sinks) const {
    return (kv <= last && (kv >= first || kv < sinks)) || (kv >= own_first && kv <= own_last);
  }
};

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

// The rings, and after the loop the warps' partial results in their place.
template <int HD, bool E4M3, int NR>
constexpr int decode_smem_bytes() {
  constexpr int ring = kWarps * kStages * Chunk<HD, E4M3>::BYTES;
  constexpr int partial = kWarps * 8 * NR * HD * 4;
  return ring > partial ? ring : partial;
}

template <int HD, typename T, bool E4M3, int NR>
__global__ void __launch_bounds__(kThreads, E4M3 && NR == 1 ? 2 : 1) decode_attention_kernel(const CacheAttnArgs a) {
  using M = typename std::conditional<E4M3, __half, T>::type;  // type of the products
  using C = Chunk<HD, E4M3>;
  constexpr int ES = C::ES, KW = C::KW, VW = C::VW;
  constexpr int KS = HD / 16;           // steps of S over the head elements, and M tiles of O^T
  constexpr int ROWS = 8 * NR;
  extern __shared__ __align__(128) uint8_t smem[];
  float(*po)[ROWS][HD] = reinterpret_cast<float(*)[ROWS][HD]>(smem);  // [kWarps], after the loop
  __shared__ float pm[kWarps][ROWS], pl[kWarps][ROWS];
  __shared__ float cm[ROWS], cl[ROWS];  // the CTA's own maxima and sums, for the cluster

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int gq = lane >> 2, tq = lane & 3;
  const int split = blockIdx.x, seq = blockIdx.z;
  const int head = blockIdx.y % a.c.kv_heads, tile = blockIdx.y / a.c.kv_heads;
  grid_dependency_wait();
  allow_dependents();
  const SeqRange r = sequence_range(a.s, seq, a.err);
  const int i0 = tile * ROWS, rows = min(ROWS, r.n * a.group - i0);
  if (rows <= 0) return;  // the whole cluster alike

  // ---- what the CTA's rows see: keys [lo, end) and below `sinks`; all rows see every key of [full_lo, full_end)
  const int context = int(r.context);
  const int j0 = i0 / a.group, j1 = (i0 + rows - 1) / a.group;
  int lo, end, full_lo, full_end;
  if (a.depth == nullptr) {
    lo = a.window > 0 ? max(0, context + j0 - a.window + 1) : 0;
    full_lo = a.window > 0 ? max(0, context + j1 - a.window + 1) : 0;
    full_end = context + j0 + 1;
    end = context + j1 + 1;
  } else {
    int lowest = kUnreachable, highest = 0, shortest = kUnreachable;
    for (int j = j0 + lane; j <= j1; j += 32) {
      const RowMask m = row_mask(a, r, j);
      lowest = min(lowest, min(m.first, m.own_first));
      highest = max(highest, m.first);
      shortest = min(shortest, m.last + 1);
    }
    lo = max(0, __reduce_min_sync(0xffffffffu, lowest));
    full_lo = max(0, __reduce_max_sync(0xffffffffu, highest));
    full_end = __reduce_min_sync(0xffffffffu, shortest);
    end = context + r.n;
  }
  const int sinks = min(a.sinks, lo);  // keys below it are visible although they lie below lo
  const int sink_chunks = min((sinks + kChunk - 1) / kChunk, lo / kChunk);
  const int chunks = sink_chunks + (end + kChunk - 1) / kChunk - lo / kChunk;
  const int c_begin = int(int64_t(split) * chunks / a.splits), c_end = int(int64_t(split + 1) * chunks / a.splits);
  auto chunk_key = [&](int c) { return (c < sink_chunks ? c : lo / kChunk + c - sink_chunks) * kChunk; };

  // ---- queries: B fragments of S^T, row 8 nr + gq, the elements that thread tq has of a key
  uint32_t qf[NR][2 * KS];
  float q_scale[NR][2];  // of rows 8 nr + 2 tq and the next one
#pragma unroll
  for (int nr = 0; nr < NR; ++nr) {
    const int i = i0 + nr * 8 + gq;
    const bool live = nr * 8 + gq < rows;
#pragma unroll
    for (int w = 0; w < 2 * KS; ++w) qf[nr][w] = 0;
    if (live) {
      const T* src = static_cast<const T*>(a.q) + (r.start + i / a.group) * a.q_stride +
                     (head * a.group + i % a.group) * HD;
#pragma unroll
      for (int w = 0; w < 2 * KS; w += 4) {
        const uint4 v = *reinterpret_cast<const uint4*>(src + (E4M3 ? tq * (HD / 4) + 2 * w : C::k_vec(tq, w / 4) * 8));
        qf[nr][w] = v.x;
        qf[nr][w + 1] = v.y;
        qf[nr][w + 2] = v.z;
        qf[nr][w + 3] = v.w;
      }
    }
    float scale = 1.f;
    if constexpr (E4M3 && std::is_same<T, __nv_bfloat16>::value) {
      uint32_t top = 0;  // the row's largest magnitude, as bits
#pragma unroll
      for (int w = 0; w < 2 * KS; ++w) top = max(top, max(qf[nr][w] & 0x7fffu, (qf[nr][w] >> 16) & 0x7fffu));
      top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
      top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
      // exponent of the divisor: maximum in [2^14, 2^15); rows of zeros, of tiny and of non-finite numbers are bounded
      int e = int(top >> 7) - 127 - 14;
      if (top == 0 || top >= 0x7f80u) e = 0;
      e = max(e, -126);
      const float up = __uint_as_float(uint32_t(127 - min(e, 126)) << 23);  // 2^-e
      scale = __uint_as_float(uint32_t(127 + min(e, 126)) << 23);
#pragma unroll
      for (int w = 0; w < 2 * KS; ++w)
        qf[nr][w] = pack2<__half>(__uint_as_float(qf[nr][w] << 16) * up, __uint_as_float(qf[nr][w] & 0xffff0000u) * up);
    }
    // scale of row 8 nr + x sits in lanes 4 x .. 4 x + 3
    q_scale[nr][0] = __shfl_sync(0xffffffffu, scale, (2 * tq) * 4) * a.scale_log2;
    q_scale[nr][1] = __shfl_sync(0xffffffffu, scale, (2 * tq + 1) * 4) * a.scale_log2;
  }
  RowMask mask[NR][2];
#pragma unroll
  for (int nr = 0; nr < NR; ++nr) {
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      const int i = nr * 8 + 2 * tq + x;
      mask[nr][x] = {kUnreachable, -1, kUnreachable, -1};
      if (i < rows) mask[nr][x] = row_mask(a, r, (i0 + i) / a.group);
    }
  }

  const uint8_t* kp = static_cast<const uint8_t*>(a.c.k);
  const uint8_t* vp = static_cast<const uint8_t*>(a.c.v);
  const int32_t* table = a.s.tables + seq * a.s.table_stride;
  const int page_mask = a.c.page_size - 1;
  // Physical page of key (lane % 16) of the chunk at kv0, or -1 where nothing is to be loaded.
  auto pages_of = [&](int kv0) {
    const int kv = kv0 + (lane & 15);
    if (kv >= end || (kv < lo && kv >= sinks)) return -1;
    const int page = table[kv >> a.c.page_shift];
    if (page >= 0 && page < a.c.num_pages) return page;
    record_error(a.err, kErrBadIndex);
    return -1;
  };
  uint8_t* ring = smem + warp * kStages * C::BYTES;
  // Chunk at kv0 into a stage of the warp's ring; what is not to be loaded becomes zeros.
  auto issue = [&](int stage, int kv0, int pages) {
    uint8_t* dst = ring + stage * C::BYTES;
    constexpr int PER_PASS = 32 / C::VECS;  // rows
    const int vec = lane % C::VECS;
#pragma unroll
    for (int p = 0; p < kChunk / PER_PASS; ++p) {
      const int key = p * PER_PASS + lane / C::VECS;
      const int page = __shfl_sync(0xffffffffu, pages, key);
      const bool valid = page >= 0;
      const size_t row = (size_t(valid ? page : 0) * a.c.kv_heads + head) * a.c.page_size + ((kv0 + key) & page_mask);
      const size_t from = row * (HD * ES) + vec * 16;
      cp_async_16(dst + C::at(key, vec), kp + from, valid);
      cp_async_16(dst + C::PLANE + C::at(key, vec), vp + from, valid);
    }
    if constexpr (E4M3) {  // lanes 0..15 the keys' scales, lanes 16..31 the values'
      const bool valid = pages >= 0;
      const int slot = (kv0 + (lane & 15)) & page_mask;
      const size_t block = (size_t(valid ? pages : 0) * a.c.kv_heads + head) * (a.c.page_size >> a.c.block_shift) +
                           (slot >> a.c.block_shift);
      cp_async_4(dst + 2 * C::PLANE + lane * 4, (lane < 16 ? a.c.k_scale : a.c.v_scale) + block, valid);
    }
  };

  float o[KS][NR][4];
  float m[NR][2], l[NR][2];
#pragma unroll
  for (int nr = 0; nr < NR; ++nr) {
    m[nr][0] = m[nr][1] = -INFINITY;
    l[nr][0] = l[nr][1] = 0.f;
#pragma unroll
    for (int t = 0; t < KS; ++t) o[t][nr][0] = o[t][nr][1] = o[t][nr][2] = o[t][nr][3] = 0.f;
  }
  // One group of copies a chunk, empty ones included; kStages - 1 ahead of the chunk in work.
  const int c_first = c_begin + warp;
  int pages = -1;
#pragma unroll
  for (int i = 0; i < kStages - 1; ++i) {
    const int c = c_first + i * kWarps;
    if (c < c_end) issue(i, chunk_key(c), pages_of(chunk_key(c)));
    cp_async_commit();
  }
  if (c_first + (kStages - 1) * kWarps < c_end) pages = pages_of(chunk_key(c_first + (kStages - 1) * kWarps));

  int stage = 0;
  for (int c = c_first; c < c_end; c += kWarps) {
    const int kv0 = chunk_key(c);
    cp_async_wait<kStages - 2>();
    __syncwarp();  // the chunk is there for every lane, and every lane is done with the one before it
    const int c_next = c + (kStages - 1) * kWarps;
    if (c_next < c_end) issue(stage == 0 ? kStages - 1 : stage - 1, chunk_key(c_next), pages);
    cp_async_commit();
    if (c_next + kWarps < c_end) pages = pages_of(chunk_key(c_next + kWarps));
    const uint8_t* chunk = ring + stage * C::BYTES;
    stage = stage + 1 == kStages ? 0 : stage + 1;
    uint32_t k[2][KW];
    C::read_key(k[0], chunk, gq, tq);
    C::read_key(k[1], chunk, gq + 8, tq);
    // ---- S^T = K Q^T, even and odd steps apart
    float s[NR][4], s_odd[NR][4];
#pragma unroll
    for (int nr = 0; nr < NR; ++nr)
#pragma unroll
      for (int e = 0; e < 4; ++e) s[nr][e] = s_odd[nr][e] = 0.f;
#pragma unroll
    for (int t = 0; t < KS; ++t) {
      uint32_t f[4];
      if constexpr (E4M3) {
        f[0] = e4m3x2_to_f16x2(uint16_t(k[0][t]));
        f[1] = e4m3x2_to_f16x2(uint16_t(k[1][t]));
        f[2] = e4m3x2_to_f16x2(uint16_t(k[0][t] >> 16));
        f[3] = e4m3x2_to_f16x2(uint16_t(k[1][t] >> 16));
      } else {
        f[0] = k[0][2 * t];
        f[1] = k[1][2 * t];
        f[2] = k[0][2 * t + 1];
        f[3] = k[1][2 * t + 1];
      }
#pragma unroll
      for (int nr = 0; nr < NR; ++nr)
        mma_16816<M>(t & 1 ? s_odd[nr] : s[nr], f[0], f[1], f[2], f[3], qf[nr][2 * t], qf[nr][2 * t + 1]);
    }
    uint32_t v[4][VW];
#pragma unroll
    for (int x = 0; x < 4; ++x) C::read_value(v[x], chunk + C::PLANE, 2 * tq + (x & 1) + (x >> 1) * 8, gq);
    // ---- scores in units of log2, masks
    float log_v[2], inv_v[2], k_scale[2];
    if constexpr (E4M3) {
      const float* scales = reinterpret_cast<const float*>(chunk + 2 * C::PLANE);
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        k_scale[x] = scales[gq + 8 * x];
        const float vs = fmaxf(scales[16 + gq + 8 * x], 7.888609052210118e-31f);  // 2^-100
        log_v[x] = log2f(vs);
        inv_v[x] = 1.f / vs;
      }
    }
    const bool full = (kv0 >= full_lo || kv0 + kChunk <= sinks) && kv0 + kChunk <= full_end;
    bool raise = false;
#pragma unroll
    for (int nr = 0; nr < NR; ++nr) {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        float x = s[nr][e] + s_odd[nr][e];
        if constexpr (E4M3) x = fmaf(x, k_scale[e >> 1] * q_scale[nr][e & 1], log_v[e >> 1]);
        else x *= q_scale[nr][e & 1];
        if (!full && !mask[nr][e & 1].sees(kv0 + gq + 8 * (e >> 1), a.sinks)) x = -INFINITY;
        s[nr][e] = x;
        raise |= x > m[nr][e & 1] + kLazy;
      }
    }
    if (__any_sync(0xffffffffu, raise)) {
#pragma unroll
      for (int nr = 0; nr < NR; ++nr) {
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          float top = fmaxf(s[nr][x], s[nr][x + 2]);
          top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 4));
          top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 8));
          top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 16));
          top = fmaxf(top, m[nr][x]);
          const float keep = ex2(m[nr][x] - (top == -INFINITY ? 0.f : top));
          m[nr][x] = top;
          l[nr][x] *= keep;
#pragma unroll
          for (int t = 0; t < KS; ++t) {
            o[t][nr][x] *= keep;
            o[t][nr][x + 2] *= keep;
          }
        }
      }
    }
    uint32_t p[NR][2];
#pragma unroll
    for (int nr = 0; nr < NR; ++nr) {
      float w[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float from = m[nr][e & 1] == -INFINITY ? 0.f : m[nr][e & 1];
        w[e] = ex2(s[nr][e] - from);
        l[nr][e & 1] += E4M3 ? w[e] * inv_v[e >> 1] : w[e];
      }
      p[nr][0] = transpose_8x8(pack2<M>(w[0], w[1]));
      p[nr][1] = transpose_8x8(pack2<M>(w[2], w[3]));
    }
    // ---- values that are no numbers, where not every row sees every key
    if (!full && j1 > j0) {
      auto odd = [&](uint32_t word, int at) {  // is element `at` of the word non-finite
        if (E4M3) return ((word >> (8 * at)) & 0x7fu) == 0x7fu;
        const uint32_t bits = std::is_same<T, __nv_bfloat16>::value ? 0x7f80u : 0x7c00u;
        return ((word >> (16 * at)) & bits) == bits;
      };
      constexpr int PER = 4 / ES;  // elements of a word
      bool any = false;
#pragma unroll
      for (int x = 0; x < 4; ++x)
#pragma unroll
        for (int w = 0; w < VW; ++w)
#pragma unroll
          for (int at = 0; at < PER; ++at) any |= odd(v[x][w], at);
      if (__any_sync(0xffffffffu, any)) {
#pragma unroll
        for (int x = 0; x < 4; ++x) {
#pragma unroll 1
          for (int owner = 0; owner < 4; ++owner) {  // the key of thread (gq, owner)
            const int kv = kv0 + 2 * owner + (x & 1) + (x >> 1) * 8;
#pragma unroll
            for (int w = 0; w < VW; ++w) {
              const uint32_t word = __shfl_sync(0xffffffffu, v[x][w], (lane & ~3) + owner);
#pragma unroll
              for (int at = 0; at < PER; ++at) {
                const int d = w * PER + at;  // of the thread's d/8 elements: M tile d / 2, row gq + 8 (d % 2)
                if (!odd(word, at)) continue;
                float value;
                if (E4M3) value = NAN;
                else if (std::is_same<T, __nv_bfloat16>::value) value = __uint_as_float((word >> (16 * at)) << 16);
                else value = __half2float(__ushort_as_half(uint16_t(word >> (16 * at))));
#pragma unroll
                for (int nr = 0; nr < NR; ++nr)
#pragma unroll
                  for (int y = 0; y < 2; ++y)
                    if (mask[nr][y].sees(kv, a.sinks)) o[d / 2][nr][y + 2 * (d & 1)] += value;
              }
            }
          }
#pragma unroll
          for (int w = 0; w < VW; ++w)
#pragma unroll
            for (int at = 0; at < PER; ++at)
              if (odd(v[x][w], at)) v[x][w] &= ~((E4M3 ? 0xffu : 0xffffu) << ((E4M3 ? 8 : 16) * at));
        }
      }
    }
    // ---- O^T += V^T P^T
#pragma unroll
    for (int t = 0; t < KS; ++t) {
      uint32_t f[4];
      if constexpr (E4M3) {
        const uint32_t sel = t & 1 ? 0x7362 : 0x5140;
        const uint32_t x = __byte_perm(v[0][t >> 1], v[1][t >> 1], sel), y = __byte_perm(v[2][t >> 1], v[3][t >> 1], sel);
        f[0] = e4m3x2_to_f16x2(uint16_t(x));
        f[1] = e4m3x2_to_f16x2(uint16_t(x >> 16));
        f[2] = e4m3x2_to_f16x2(uint16_t(y));
        f[3] = e4m3x2_to_f16x2(uint16_t(y >> 16));
      } else {
        f[0] = __byte_perm(v[0][t], v[1][t], 0x5410);
        f[1] = __byte_perm(v[0][t], v[1][t], 0x7632);
        f[2] = __byte_perm(v[2][t], v[3][t], 0x5410);
        f[3] = __byte_perm(v[2][t], v[3][t], 0x7632);
      }
#pragma unroll
      for (int nr = 0; nr < NR; ++nr) mma_16816<M>(o[t][nr], f[0], f[1], f[2], f[3], p[nr][0], p[nr][1]);
    }
  }
  cp_async_wait<0>();
  __syncthreads();  // the rings make room for the partial results

  // ---- the warps' partial results: row 8 nr + 2 tq + x, two neighbouring elements from every M tile
#pragma unroll
  for (int nr = 0; nr < NR; ++nr) {
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      float sum = l[nr][x];
      sum += __shfl_xor_sync(0xffffffffu, sum, 4);
      sum += __shfl_xor_sync(0xffffffffu, sum, 8);
      sum += __shfl_xor_sync(0xffffffffu, sum, 16);
      const int row = nr * 8 + 2 * tq + x;
      if (gq == 0) {
        pm[warp][row] = m[nr][x];
        pl[warp][row] = sum;
      }
#pragma unroll
      for (int t = 0; t < KS; ++t)
        *reinterpret_cast<float2*>(&po[warp][row][C::v_element(gq, t)]) = make_float2(o[t][nr][x], o[t][nr][x + 2]);
    }
  }
  __syncthreads();
  // ---- joined over the warps, then over the cluster, in order
  constexpr int Q4 = HD / 4;
  auto store = [&](int row, int at, float4 sum, float total) {
    const float inv = total == 0.f ? 0.f : 1.f / total;
    const int i = i0 + row;
    T* dst = static_cast<T*>(a.out) + (r.start + i / a.group) * a.out_stride + (head * a.group + i % a.group) * HD + at;
    *reinterpret_cast<uint2*>(dst) = make_uint2(pack2<T>(sum.x * inv, sum.y * inv), pack2<T>(sum.z * inv, sum.w * inv));
  };
  for (int item = tid; item < rows * Q4; item += kThreads) {
    const int row = item / Q4, at = (item % Q4) * 4;
    float top = -INFINITY;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) top = fmaxf(top, pm[w][row]);
    const float from = top == -INFINITY ? 0.f : top;
    float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
    float total = 0.f;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      const float f = ex2(pm[w][row] - from);
      const float4 x = *reinterpret_cast<const float4*>(&po[w][row][at]);
      sum.x += f * x.x;
      sum.y += f * x.y;
      sum.z += f * x.z;
      sum.w += f * x.w;
      total += f * pl[w][row];
    }
    if (a.splits == 1) {
      store(row, at, sum, total);
    } else {
      *reinterpret_cast<float4*>(&po[0][row][at]) = sum;
      if (at == 0) {
        cm[row] = top;
        cl[row] = total;
      }
    }
  }
  if (a.splits == 1) return;
  cluster_sync();
  for (int item = int(cluster_rank()) * kThreads + tid; item < rows * Q4; item += a.splits * kThreads) {
    const int row = item / Q4, at = (item % Q4) * 4;
    float ms[kMaxSplits], ls[kMaxSplits];
    float4 xs[kMaxSplits];
    float top = -INFINITY;
#pragma unroll
    for (int i = 0; i < kMaxSplits; ++i) {
      ms[i] = -INFINITY;
      ls[i] = 0.f;
      xs[i] = make_float4(0.f, 0.f, 0.f, 0.f);
      if (i < a.splits) {
        ms[i] = ld_dsmem_f32(cluster_map(&cm[row], i));
        ls[i] = ld_dsmem_f32(cluster_map(&cl[row], i));
        xs[i] = ld_dsmem_f32x4(cluster_map(&po[0][row][at], i));
        top = fmaxf(top, ms[i]);
      }
    }
    const float from = top == -INFINITY ? 0.f : top;
    float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
    float total = 0.f;
#pragma unroll
    for (int i = 0; i < kMaxSplits; ++i) {
      const float f = ex2(ms[i] - from);
      sum.x += f * xs[i].x;
      sum.y += f * xs[i].y;
      sum.z += f * xs[i].z;
      sum.w += f * xs[i].w;
      total += f * ls[i];
    }
    store(row, at, sum, total);
  }
  cluster_sync();  // a peer's memory stays until everyone has read it
}

template <int HD, typename T, bool E4M3, int NR>
int decode_launch(CacheAttnArgs a, int64_t max_keys, int num_sms, cudaStream_t stream) {
  const int tiles = int((int64_t(a.s.max_rows) * a.group + 8 * NR - 1) / (8 * NR));
  const int64_t ctas = int64_t(tiles) * a.c.kv_heads * a.s.n_seqs;
  const int64_t keys = a.window > 0 ? std::min<int64_t>(max_keys, int64_t(a.window) + a.sinks + a.s.max_rows) : max_keys;
  int splits = 1;
  while (splits < kMaxSplits && ctas * splits < 6 * num_sms && splits * 2 * kWarps * kChunk * 2 <= keys) splits *= 2;
  a.splits = splits;
  auto kernel = decode_attention_kernel<HD, T, E4M3, NR>;
  constexpr int SMEM = decode_smem_bytes<HD, E4M3, NR>();
  const int st = raise_smem_limit(reinterpret_cast<const void*>(kernel), SMEM, "decode_attention_kernel: shared memory");
  if (st != PLM_OK) return st;
  const dim3 grid(splits, unsigned(tiles * a.c.kv_heads), unsigned(a.s.n_seqs));
  return check_cuda(launch_cluster(kernel, grid, dim3(kThreads), SMEM, stream, true, splits, 1, a), "decode_attention_kernel");
}

template <int HD, typename T>
int attention_launch(const CacheAttnArgs& a, int kind, int64_t max_keys, int num_sms, cudaStream_t stream) {
  const bool wide = int64_t(a.s.max_rows) * a.group > 8;
  if (kind == PLM_CACHE_E4M3)
    return wide ? decode_launch<HD, T, true, 2>(a, max_keys, num_sms, stream)
                : decode_launch<HD, T, true, 1>(a, max_keys, num_sms, stream);
  return wide ? decode_launch<HD, T, false, 2>(a, max_keys, num_sms, stream)
              : decode_launch<HD, T, false, 1>(a, max_keys, num_sms, stream);
}

}  // namespace
}  // namespace plm

using namespace plm;

namespace {

// Validates a call and fills the argument block.
int attention_arguments(plm_ctx* ctx, const plm_cache_attention_desc* d, CacheAttnArgs* out, int64_t* max_keys) {
  if (ctx == nullptr || d == nullptr) return fail(PLM_ERR_INVALID, "plm_cache_attention: null argument");
  CacheAttnArgs& a = *out;
  a = {};
  int st = cache_arguments("plm_cache_attention", d->cache, d->seqs, d->dtype, d->rows, &a.c, &a.s);
  if (st != PLM_OK) return st;
  const int hd = d->cache.head_dim;
  if (d->num_heads < 1 || d->num_heads > 4096 || d->num_heads % d->cache.num_kv_heads != 0)
    return fail(PLM_ERR_INVALID, "plm_cache_attention: %d heads over %d kv heads", d->num_heads, d->cache.num_kv_heads);
  const int64_t width = int64_t(d->num_heads) * hd;
  if (!d->q || !d->out || !aligned16(d->q) || !aligned16(d->out) || d->q_stride < width || d->out_stride < width ||
      d->q_stride % 8 != 0 || d->out_stride % 8 != 0)
    return fail(PLM_ERR_INVALID, "plm_cache_attention: q and out need 16-byte aligned rows of at least %lld elements",
                (long long)width);
  if (d->window < 0 || d->sinks < 0)
    return fail(PLM_ERR_INVALID, "plm_cache_attention: window %d, sinks %d", d->window, d->sinks);
  if ((d->depth == nullptr) != (d->own_start == nullptr))
    return fail(PLM_ERR_INVALID, "plm_cache_attention: depth and own_start go together");
  if (!(d->scale >= 0.f && d->scale < INFINITY))
    return fail(PLM_ERR_INVALID, "plm_cache_attention: scale %g", double(d->scale));
  if (int64_t(d->rows) * d->num_heads >= (int64_t(1) << 31))
    return fail(PLM_ERR_UNSUPPORTED, "plm_cache_attention: %d rows of %d heads in one call", d->rows, d->num_heads);
  a.q = d->q;
  a.q_stride = d->q_stride;
  a.out = d->out;
  a.out_stride = d->out_stride;
  a.heads = d->num_heads;
  a.group = d->num_heads / d->cache.num_kv_heads;
  const double scale = d->scale > 0.f ? double(d->scale) : 1.0 / sqrt(double(hd));
  a.scale_log2 = float(1.4426950408889634 * scale);
  a.window = d->window;
  a.sinks = d->sinks;
  a.depth = d->depth;
  a.own_start = d->own_start;
  a.workspace = d->workspace;
  a.err = ctx->err;
  a.s.max_rows = std::min(a.s.max_rows, a.s.rows);  // a larger bound only widens the grid
  *max_keys = d->seqs.max_keys > 0 ? std::min(d->seqs.max_keys, a.s.max_tokens) : a.s.max_tokens;
  return PLM_OK;
}

size_t workspace_bytes(const plm_ctx* ctx, const plm_cache_attention_desc* d, const CacheAttnArgs& a, int64_t max_keys) {
  return decode_takes(a) ? decode_workspace(a, d->cache.kind, d->cache.head_dim, max_keys, ctx->num_sms) : 0;
}

}  // namespace

extern "C" int plm_cache_attention_workspace(plm_ctx* ctx, const plm_cache_attention_desc* d, int64_t* bytes) {
  CacheAttnArgs a;
  int64_t max_keys = 0;
  if (bytes == nullptr) return fail(PLM_ERR_INVALID, "plm_cache_attention_workspace: null argument");
  const int st = attention_arguments(ctx, d, &a, &max_keys);
  if (st != PLM_OK) return st;
  *bytes = int64_t(workspace_bytes(ctx, d, a, max_keys));
  return PLM_OK;
}

extern "C" int plm_cache_attention(plm_ctx* ctx, const plm_cache_attention_desc* d, void* stream) {
  CacheAttnArgs a;
  int64_t max_keys = 0;
  const int st = attention_arguments(ctx, d, &a, &max_keys);
  if (st != PLM_OK) return st;
  const int64_t needs = int64_t(workspace_bytes(ctx, d, a, max_keys));
  if (needs > 0 && (d->workspace == nullptr || !aligned16(d->workspace) || d->workspace_bytes < needs))
    return fail(PLM_ERR_INVALID, "plm_cache_attention: a 16-byte aligned workspace of %lld bytes is needed (%lld given)",
                (long long)needs, (long long)(d->workspace ? d->workspace_bytes : 0));
  DeviceScope scope(ctx->device);
  if (scope.status() != PLM_OK) return scope.status();
  cudaStream_t on = static_cast<cudaStream_t>(stream);
  const int hd = d->cache.head_dim;
  if (decode_takes(a)) return decode_attention(a, d->cache.kind, d->dtype, hd, max_keys, ctx->num_sms, on);
  if (d->dtype == PLM_F16)
    return hd == 128 ? attention_launch<128, __half>(a, d->cache.kind, max_keys, ctx->num_sms, on)
                     : attention_launch<64, __half>(a, d->cache.kind, max_keys, ctx->num_sms, on);
  return hd == 128 ? attention_launch<128, __nv_bfloat16>(a, d->cache.kind, max_keys, ctx->num_sms, on)
                   : attention_launch<64, __nv_bfloat16>(a, d->cache.kind, max_keys, ctx->num_sms, on);
}
