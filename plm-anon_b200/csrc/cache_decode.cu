// Attention over a paged cache for sequences of few rows (at most 16 packed rows: rows times query heads per kv head).
// Every key and value is read once, 2 d bytes of e4m3 codes or 4 d of 16-bit numbers.
//
// What bounds it: with e4m3 pages the instructions that bring 16 keys through a warp, 434 (75 of them turn codes into
// f16), two a clock on an SM whose schedulers are busy half of the time with 16 warps; with 16-bit pages (355) they are
// busy a quarter of the time with 8 warps, 12 gain 1.5 %, and start, tail and join are what is left around the bytes.
// Measured, head_dim 128, both launches: one token at 32768 e4m3 keys, 16 kv heads, 35.1 us (3.83 TB/s); one token of each
// of 61 sequences, 2 to 8191 e4m3 keys, 32 heads over 8, 122 us (4.1 TB/s); of 8 sequences behind windows of 4096 16-bit
// keys, 32 heads over 8, 29.9 us (4.5 TB/s). One token at 1024 keys takes 10 us, all latency: few chunks to a warp, and
// join_kernel is a second launch.
//
// All chunks of 16 keys of all (sequence, kv head) tiles form one list, and the workers, the CTAs that fit on the GPU at
// once, get equal shares of it, so uneven lengths and few heads keep every SM busy. The host sizes the grid by its bound on
// the keys; where the sequences have fewer chunks than that makes workers, the first ones get a chunk each and the others
// none. A tile that a worker has to itself goes to the output; the parts of one that several hold go to the workspace, and
// join_kernel, launched behind, adds them up in the workers' order. (Clusters that share a tile through distributed shared
// memory leave SMs idle: 16 tiles x 8 CTAs, one to an SM, do not all find a place at once on 148 SMs in GPCs of at most 20.)
//
// Within a worker the warps take turns at the chunks. Everything is transposed, keys and head elements on the M side of
// mma.m16n8k16, packed rows on the N side:
//     S^T[16 keys, rows] = K Q^T,      O^T[d, rows] += V^T P^T,
// so 8 rows fill an instruction and a K or V element is brought into its fragment once for all rows. A product's inner
// index may be permuted if both operands are, and an output's index if the store undoes it: thread (gq, tq) =
// (lane / 4, lane % 4) takes a quarter of the elements of keys gq and gq + 8 as its part of K, and an eighth of the
// elements of keys 2 tq, 2 tq + 1, 2 tq + 8, 2 tq + 9 as its part of V, both in whole vectors of shared memory.
// P^T changes sides through movmatrix. Every warp keeps a ring of its own full with 16-byte asynchronous copies, so the
// warps meet only at a tile's end.
//
// The softmax is online in base 2 with a lazy maximum: a row's m is raised (and O, l rescaled) only when a score passes
// it by more than 2^15, so most chunks take one vote and no cross-lane maximum; weights stay below 2^15.
//
// e4m3 pages: codes become f16 exactly, and their scales never touch a 16-bit number. A key's scale multiplies its
// scores. A value's scale s enters through w = 2^(score + log2 s - m): O += w code and l += w / s, out = O / l, so that
// m follows the largest term of the sum, w <= 2^15 whatever the scales are, and rounding w to f16 (2^-11) is relative to
// that term. A weight that is too small for a float still counts in l (small_share). Queries in bf16 become f16 exactly
// but for elements below 2^-30 of their row's largest (query_exponent).
// 16-bit pages: products in the model dtype, w rounded to it, as in round_attention_kernel.
//
// Masks. Keys that no row of the tile sees are not loaded (their places are zeroed, so stale slots, or pages that were
// given away, are never read). Where rows differ in what they see, a masked score is -inf, its weight 0; 0 times a
// non-finite value would still be NaN, so such chunks are searched for non-finite values, which are added to the rows
// that see them by hand and replaced by 0.
#include "cache_attention.cuh"

namespace plm {
namespace {

constexpr int kWarps = 8;
constexpr int kThreads = 32 * kWarps;
constexpr int kChunk = 16;      // keys
constexpr int kStages = 3;      // chunks of a warp's ring
constexpr int kMaxSeqs = 1024;  // of a launch that shares its chunks out evenly

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
__device__ __forceinline__ uint32_t transpose_8x8(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
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
  // Vector i of thread tq's part of a key.
  static __device__ __forceinline__ int k_vec(int tq, int i) { return E4M3 ? tq * VECS / 4 + i : tq + 4 * i; }
  // Vector i of thread gq's part of a value (with rows of four vectors, half of one).
  static __device__ __forceinline__ int v_vec(int gq, int i) {
    if (E4M3) return VECS == 8 ? gq : gq >> 1;
    return (((gq & 1) << 2) | (gq >> 1)) + 8 * i;
  }
  // The head element that is number 2 t of thread gq's part of a value.
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

// The rings, and after a tile's loop the warps' partial results in their place.
template <int HD, bool E4M3, int NR>
constexpr int decode_smem_bytes() {
  constexpr int ring = kWarps * kStages * Chunk<HD, E4M3>::BYTES;
  constexpr int partial = kWarps * 8 * NR * HD * 4;
  return ring > partial ? ring : partial;
}

// The workspace: for every worker the tile it begins and others go on with, then two partial results for every worker,
// slot 2 w for a tile that an earlier worker began, slot 2 w + 1 for one that it begins itself.
struct SplitTile {
  int count;       // workers that hold a part of it, from this one on; 0: there is none
  int row0, rows;  // the sequence's first row; packed rows
  int head;
};
constexpr size_t split_tile_bytes(int workers) { return (size_t(workers) * sizeof(SplitTile) + 127) & ~size_t(127); }
template <int ROWS, int HD>
constexpr size_t partial_floats() {
  return size_t(ROWS) * (HD + 2);  // O, then (m, l) of every row
}

__device__ __forceinline__ TileKeys few_rows_keys(const CacheAttnArgs& a, const SeqRange& r) {
  TileKeys t = causal_keys(a, r, 0, r.n - 1);
  if (a.depth != nullptr) {
    t.end = int(r.context) + r.n;
    t.lo = t.full_end = kUnreachable;
    t.full_lo = 0;
    for (int j = 0; j < r.n; ++j) widen(t, row_mask(a, r, j));
    t.lo = min(t.lo, t.end);
    t.sinks = min(a.sinks, t.lo);
  }
  t.count<kChunk>();
  t.chunks = max(t.chunks, 1);  // rows that see no key have a chunk to themselves all the same, of zeros, and give zeros
  return t;
}

// EVEN: the workers share all chunks out; otherwise (more than kMaxSeqs sequences) a CTA has a tile to itself.
template <int HD, typename T, bool E4M3, int NR, bool EVEN>
__global__ void __launch_bounds__(kThreads, E4M3 && NR == 1 ? 2 : 1) decode_attention_kernel(const CacheAttnArgs a) {
  using M = typename std::conditional<E4M3, __half, T>::type;  // type of the products
  using C = Chunk<HD, E4M3>;
  constexpr int ES = C::ES, KW = C::KW, VW = C::VW;
  constexpr int KS = HD / 16;  // steps of S over the head elements, and M tiles of O^T
  constexpr int ROWS = 8 * NR;
  constexpr int PER_PASS = 32 / C::VECS;  // rows that the lanes of a warp copy together
  extern __shared__ __align__(128) uint8_t smem[];
  float(*po)[ROWS][HD] = reinterpret_cast<float(*)[ROWS][HD]>(smem);  // [kWarps], after the loop
  __shared__ float pm[kWarps][ROWS], pl[kWarps][ROWS];
  __shared__ int64_t upto[EVEN ? kMaxSeqs : 1];  // chunks of one kv head of the sequences up to and with this one

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int gq = lane >> 2, tq = lane & 3;
  const int worker = blockIdx.x, workers = gridDim.x;
  grid_dependency_wait();
  allow_dependents();

  // ---- this worker's share [at, at_end) of all chunks, in the order of sequences, kv heads and keys
  int64_t all = 0, at = 0, at_end = 1;
  int sharers = 1;  // workers that get a share: no more than there are chunks, as all that hold a part of a tile write one
  if constexpr (EVEN) {
    for (int i = tid; i < a.s.n_seqs; i += kThreads) {
      const SeqRange r = sequence_range(a.s, i, a.err);
      upto[i] = r.n > 0 ? few_rows_keys(a, r).chunks : 0;
    }
    __syncthreads();
    if (warp == 0) {
      int64_t before = 0;
      for (int base = 0; base < a.s.n_seqs; base += 32) {
        int64_t x = base + lane < a.s.n_seqs ? upto[base + lane] : 0;
#pragma unroll
        for (int off = 1; off < 32; off <<= 1) {
          const int64_t y = __shfl_up_sync(0xffffffffu, x, off);
          if (lane >= off) x += y;
        }
        x += before;
        if (base + lane < a.s.n_seqs) upto[base + lane] = x;
        before = __shfl_sync(0xffffffffu, x, 31);
      }
    }
    __syncthreads();
    all = upto[a.s.n_seqs - 1] * a.c.kv_heads;
    sharers = int(min(int64_t(workers), all));
    at = worker < sharers ? all * worker / sharers : 0;
    at_end = worker < sharers ? all * (worker + 1) / sharers : 0;
  }
  SplitTile* const split_tiles = reinterpret_cast<SplitTile*>(a.workspace);
  float* const partials = reinterpret_cast<float*>(static_cast<uint8_t*>(a.workspace) + split_tile_bytes(workers));
  bool begun = false;  // a tile that the next worker goes on with

  while (at < at_end) {
    // ---- the tile and this worker's chunks [c_begin, c_end) of it
    int seq, head, c_begin = 0;
    if constexpr (EVEN) {
      int below = -1;  // upto[below] * kv_heads <= at < upto[seq] * kv_heads
      seq = a.s.n_seqs - 1;
      while (seq - below > 1) {
        const int mid = (below + seq) >> 1;
        if (upto[mid] * a.c.kv_heads <= at) below = mid;
        else seq = mid;
      }
      const int64_t before = seq > 0 ? upto[seq - 1] : 0, in_seq = at - before * a.c.kv_heads;
      head = int(in_seq / (upto[seq] - before));
      c_begin = int(in_seq % (upto[seq] - before));
    } else {
      seq = blockIdx.x / a.c.kv_heads;
      head = blockIdx.x % a.c.kv_heads;
    }
    const SeqRange r = sequence_range(a.s, seq, EVEN ? nullptr : a.err);
    if (r.n == 0) return;  // a tile to itself, and nothing in it
    const TileKeys t = few_rows_keys(a, r);
    const int rows = r.n * a.group;
    const int c_end = EVEN ? int(min(int64_t(t.chunks), c_begin + (at_end - at))) : t.chunks;

    // ---- queries: B fragments of S^T, row 8 nr + gq, the elements that thread tq has of a key
    uint32_t qf[NR][2 * KS];
    float q_scale[NR][2];  // of rows 8 nr + 2 tq and the next one
#pragma unroll
    for (int nr = 0; nr < NR; ++nr) {
      const int i = nr * 8 + gq;
#pragma unroll
      for (int w = 0; w < 2 * KS; ++w) qf[nr][w] = 0;
      if (i < rows) {
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
      float scale = a.scale_log2;
      if constexpr (E4M3 && std::is_same<T, __nv_bfloat16>::value) {
        uint32_t top = 0;  // the row's largest magnitude, as bits
#pragma unroll
        for (int w = 0; w < 2 * KS; ++w) top = max(top, max(qf[nr][w] & 0x7fffu, (qf[nr][w] >> 16) & 0x7fffu));
        top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
        top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
        const int e = query_exponent(top);
        const float up = power_of_two_f32(-e);
        scale *= power_of_two_f32(e);
#pragma unroll
        for (int w = 0; w < 2 * KS; ++w)
          qf[nr][w] = pack2<__half>(__uint_as_float(qf[nr][w] << 16) * up, __uint_as_float(qf[nr][w] & 0xffff0000u) * up);
      }
      // the scale of row 8 nr + x sits in lanes 4 x .. 4 x + 3
      q_scale[nr][0] = __shfl_sync(0xffffffffu, scale, (2 * tq) * 4);
      q_scale[nr][1] = __shfl_sync(0xffffffffu, scale, (2 * tq + 1) * 4);
    }
    RowMask mask[NR][2];
#pragma unroll
    for (int nr = 0; nr < NR; ++nr) {
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        const int i = nr * 8 + 2 * tq + x;
        mask[nr][x] = i < rows ? row_mask(a, r, i / a.group) : no_row();
      }
    }

    // ---- the warp's ring
    const int32_t* table = a.s.tables + seq * a.s.table_stride;
    const int page_mask = a.c.page_size - 1;
    const size_t page_bytes = size_t(a.c.kv_heads) * a.c.page_size * (HD * ES);
    const int vec = lane % C::VECS;
    const uint8_t* const k_lane =
        static_cast<const uint8_t*>(a.c.k) + (size_t(head) * a.c.page_size + lane / C::VECS) * (HD * ES) + vec * 16;
    const ptrdiff_t to_v = static_cast<const uint8_t*>(a.c.v) - static_cast<const uint8_t*>(a.c.k);
    const int page_scales = a.c.page_size >> a.c.block_shift;
    const float* const scale_lane = lane < 16 ? a.c.k_scale : a.c.v_scale;
    uint8_t* const ring = smem + warp * kStages * C::BYTES;
    // Physical page of key (lane % 16) of the chunk at kv0, or -1 where nothing is to be loaded.
    auto pages_of = [&](int kv0) {
      const int kv = kv0 + (lane & 15);
      if (!t.needed(kv)) return -1;
      const int page = table[kv >> a.c.page_shift];
      if (unsigned(page) < unsigned(a.c.num_pages)) return page;
      record_error(a.err, kErrBadIndex);
      return -1;
    };
    // Chunk at kv0 into a stage of the ring; what is not to be loaded becomes zeros.
    auto issue = [&](int stage, int kv0, int pages) {
      uint8_t* dst = ring + stage * C::BYTES;
      if (a.c.page_size >= kChunk && pages >= 0 && t.all_needed(kv0, kChunk)) {  // the lanes agree: one page
        const uint8_t* from = k_lane + size_t(pages) * page_bytes + (kv0 & page_mask) * (HD * ES);
#pragma unroll
        for (int p = 0; p < kChunk / PER_PASS; ++p) {
          const int key = p * PER_PASS + lane / C::VECS;
          cp_async_16(dst + C::at(key, vec), from + p * PER_PASS * (HD * ES), true);
          cp_async_16(dst + C::PLANE + C::at(key, vec), from + p * PER_PASS * (HD * ES) + to_v, true);
        }
      } else {
#pragma unroll 1
        for (int p = 0; p < kChunk / PER_PASS; ++p) {
          const int key = p * PER_PASS + lane / C::VECS;
          const int page = __shfl_sync(0xffffffffu, pages, key);
          const bool valid = page >= 0;
          const uint8_t* from = static_cast<const uint8_t*>(a.c.k) + size_t(valid ? page : 0) * page_bytes +
                                (size_t(head) * a.c.page_size + ((kv0 + key) & page_mask)) * (HD * ES) + vec * 16;
          cp_async_16(dst + C::at(key, vec), from, valid);
          cp_async_16(dst + C::PLANE + C::at(key, vec), from + to_v, valid);
        }
      }
      if constexpr (E4M3) {  // lanes 0..15 the keys' scales, lanes 16..31 the values'
        const bool valid = pages >= 0;
        const int block = ((kv0 + (lane & 15)) & page_mask) >> a.c.block_shift;
        cp_async_4(dst + 2 * C::PLANE + lane * 4,
                   scale_lane + (size_t(valid ? pages : 0) * a.c.kv_heads + head) * page_scales + block, valid);
      }
    };

    float o[KS][NR][4];
    float m[NR][2], l[NR][2];
#pragma unroll
    for (int nr = 0; nr < NR; ++nr) {
      m[nr][0] = m[nr][1] = -INFINITY;
      l[nr][0] = l[nr][1] = 0.f;
#pragma unroll
      for (int s = 0; s < KS; ++s) o[s][nr][0] = o[s][nr][1] = o[s][nr][2] = o[s][nr][3] = 0.f;
    }
    // One group of copies a chunk, empty ones included; kStages - 1 chunks ahead of the one in work.
    const int c_first = c_begin + warp;
#pragma unroll
    for (int i = 0; i < kStages - 1; ++i) {
      const int kv0 = t.key<kChunk>(c_first + i * kWarps);
      if (c_first + i * kWarps < c_end) issue(i, kv0, pages_of(kv0));
      cp_async_commit();
    }
    int pages = -1;
    if (c_first + (kStages - 1) * kWarps < c_end) pages = pages_of(t.key<kChunk>(c_first + (kStages - 1) * kWarps));

    bool apart = false;  // scales were met with which a weight may be too small for a float
    int stage = 0;
    for (int c = c_first; c < c_end; c += kWarps) {
      const int kv0 = t.key<kChunk>(c);
      cp_async_wait<kStages - 2>();
      __syncwarp();  // the chunk is there for every lane, and every lane is done with the one before it
      const int c_next = c + (kStages - 1) * kWarps;
      if (c_next < c_end) issue(stage == 0 ? kStages - 1 : stage - 1, t.key<kChunk>(c_next), pages);
      cp_async_commit();
      if (c_next + kWarps < c_end) pages = pages_of(t.key<kChunk>(c_next + kWarps));
      const uint8_t* chunk = ring + stage * C::BYTES;
      stage = stage + 1 == kStages ? 0 : stage + 1;
      // ---- S^T = K Q^T, even and odd steps apart
      uint32_t k[2][KW];
      C::read_key(k[0], chunk, gq, tq);
      C::read_key(k[1], chunk, gq + 8, tq);
      float s[NR][4], s_odd[NR][4];
#pragma unroll
      for (int nr = 0; nr < NR; ++nr)
#pragma unroll
        for (int e = 0; e < 4; ++e) s[nr][e] = s_odd[nr][e] = 0.f;
#pragma unroll
      for (int x = 0; x < KS; ++x) {
        uint32_t f[4];
        if constexpr (E4M3) {
          f[0] = e4m3x2_to_f16x2(uint16_t(k[0][x]));
          f[1] = e4m3x2_to_f16x2(uint16_t(k[1][x]));
          f[2] = e4m3x2_to_f16x2(uint16_t(k[0][x] >> 16));
          f[3] = e4m3x2_to_f16x2(uint16_t(k[1][x] >> 16));
        } else {
          f[0] = k[0][2 * x];
          f[1] = k[1][2 * x];
          f[2] = k[0][2 * x + 1];
          f[3] = k[1][2 * x + 1];
        }
#pragma unroll
        for (int nr = 0; nr < NR; ++nr)
          mma_16816<M>(x & 1 ? s_odd[nr] : s[nr], f[0], f[1], f[2], f[3], qf[nr][2 * x], qf[nr][2 * x + 1]);
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
          const float vs = fmaxf(scales[16 + gq + 8 * x], kLeastScale);
          log_v[x] = lg2(vs);
          inv_v[x] = rcp(vs);
        }
      }
      const bool full = t.all_seen(kv0, kChunk);
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
      if (__any_sync(0xffffffffu, raise || (E4M3 && (apart || fabsf(log_v[0]) > kUsual || fabsf(log_v[1]) > kUsual)))) {
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
              const Keep keep(m[nr][x] - (top == -INFINITY ? 0.f : top));
              m[nr][x] = top;
              l[nr][x] = keep.l(l[nr][x]);
#pragma unroll
              for (int y = 0; y < KS; ++y) {
                o[y][nr][x] *= keep.o();
                o[y][nr][x + 2] *= keep.o();
              }
            }
          }
        }
        if constexpr (E4M3) {
#pragma unroll
          for (int nr = 0; nr < NR; ++nr)
#pragma unroll
            for (int e = 0; e < 4; ++e) apart |= s[nr][e] > -INFINITY && fabsf(log_v[e >> 1]) > kUsual;
          apart = __any_sync(0xffffffffu, apart);
          if (apart) {
#pragma unroll
            for (int nr = 0; nr < NR; ++nr) {
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                const float x = s[nr][e] - (m[nr][e & 1] == -INFINITY ? 0.f : m[nr][e & 1]);
                if (ex2(x) == 0.f) l[nr][e & 1] += small_share(x, log_v[e >> 1]);
              }
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
      // ---- values that are no numbers, where not every row sees every key (a causal sequence's only row sees all that are
      // loaded; under depth even that one may not)
      if (!full && (r.n > 1 || a.depth != nullptr)) {
        constexpr int PER = 4 / ES;  // elements of a word
        bool any = false;
#pragma unroll
        for (int x = 0; x < 4; ++x)
#pragma unroll
          for (int w = 0; w < VW; ++w)
#pragma unroll
            for (int y = 0; y < PER; ++y) any |= non_finite<T, E4M3>(v[x][w], y);
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
                for (int y = 0; y < PER; ++y) {
                  const int d = w * PER + y;  // of the thread's d/8 elements: M tile d / 2, row gq + 8 (d % 2)
                  if (!non_finite<T, E4M3>(word, y)) continue;
                  const float value = element_f32<T, E4M3>(word, y);
#pragma unroll
                  for (int nr = 0; nr < NR; ++nr)
#pragma unroll
                    for (int z = 0; z < 2; ++z)
                      if (mask[nr][z].sees(kv, a.sinks)) o[d / 2][nr][z + 2 * (d & 1)] += value;
                }
              }
            }
#pragma unroll
            for (int w = 0; w < VW; ++w)
#pragma unroll
              for (int y = 0; y < PER; ++y)
                if (non_finite<T, E4M3>(v[x][w], y)) v[x][w] &= ~((E4M3 ? 0xffu : 0xffffu) << ((E4M3 ? 8 : 16) * y));
          }
        }
      }
      // ---- O^T += V^T P^T
#pragma unroll
      for (int y = 0; y < KS; ++y) {
        uint32_t f[4];
        if constexpr (E4M3) {
          const uint32_t sel = y & 1 ? 0x7362 : 0x5140;
          const uint32_t lo2 = __byte_perm(v[0][y >> 1], v[1][y >> 1], sel), hi2 = __byte_perm(v[2][y >> 1], v[3][y >> 1], sel);
          f[0] = e4m3x2_to_f16x2(uint16_t(lo2));
          f[1] = e4m3x2_to_f16x2(uint16_t(lo2 >> 16));
          f[2] = e4m3x2_to_f16x2(uint16_t(hi2));
          f[3] = e4m3x2_to_f16x2(uint16_t(hi2 >> 16));
        } else {
          f[0] = __byte_perm(v[0][y], v[1][y], 0x5410);
          f[1] = __byte_perm(v[0][y], v[1][y], 0x7632);
          f[2] = __byte_perm(v[2][y], v[3][y], 0x5410);
          f[3] = __byte_perm(v[2][y], v[3][y], 0x7632);
        }
#pragma unroll
        for (int nr = 0; nr < NR; ++nr) mma_16816<M>(o[y][nr], f[0], f[1], f[2], f[3], p[nr][0], p[nr][1]);
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
        if (row < rows) {
#pragma unroll
          for (int y = 0; y < KS; ++y)
            *reinterpret_cast<float2*>(&po[warp][row][C::v_element(gq, y)]) = make_float2(o[y][nr][x], o[y][nr][x + 2]);
        }
      }
    }
    __syncthreads();
    // ---- joined over the warps in order: the output, or a part for join_kernel
    constexpr int Q4 = HD / 4;
    const bool complete = c_begin == 0 && c_end == t.chunks;
    float* const part = partials + size_t(2 * worker + (c_begin == 0 ? 1 : 0)) * partial_floats<ROWS, HD>();
    for (int item = tid; item < rows * Q4; item += kThreads) {
      const int row = item / Q4, d = (item % Q4) * 4;
      float top = -INFINITY;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) top = fmaxf(top, pm[w][row]);
      const float from = top == -INFINITY ? 0.f : top;
      float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
      float total = 0.f;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) {
        const Keep keep(pm[w][row] - from);
        const float f = keep.o();
        const float4 x = *reinterpret_cast<const float4*>(&po[w][row][d]);
        sum.x += f * x.x;
        sum.y += f * x.y;
        sum.z += f * x.z;
        sum.w += f * x.w;
        total += keep.l(pl[w][row]);
      }
      if (complete) {
        const float x[4] = {sum.x, sum.y, sum.z, sum.w};
        store_row<T>(a, r.start, row, head, HD, d, x, total);
      } else {
        *reinterpret_cast<float4*>(part + row * HD + d) = sum;
        if (d == 0) *reinterpret_cast<float2*>(part + ROWS * HD + 2 * row) = make_float2(top, total);
      }
    }
    if (EVEN && !complete && c_begin == 0) {
      begun = true;
      // its last chunk belongs to the largest worker w with all w / sharers <= that chunk's index
      const int64_t last = at + t.chunks - 1;
      if (tid == 0)
        split_tiles[worker] = {int(((last + 1) * sharers - 1) / all) - worker + 1, r.start, rows, head};
    }
    if (!EVEN) return;
    at += c_end - c_begin;
    __syncthreads();  // the partial results make room for the next tile's rings
  }
  if (EVEN && !begun && tid == 0) split_tiles[worker].count = 0;
}

// Joins the tiles that several workers hold parts of, a CTA for each worker that began one, a warp to a row.
template <int HD, typename T, int ROWS>
__global__ void __launch_bounds__(32 * ROWS) join_kernel(const CacheAttnArgs a) {
  grid_dependency_wait();
  allow_dependents();
  const int worker = blockIdx.x, workers = gridDim.x, row = threadIdx.x >> 5;
  const SplitTile t = static_cast<const SplitTile*>(a.workspace)[worker];
  if (t.count == 0 || row >= t.rows) return;
  const float* partials = reinterpret_cast<const float*>(static_cast<const uint8_t*>(a.workspace) + split_tile_bytes(workers));
  join_row<HD, T>(
      a, t.count, [&](int i) { return partials + size_t(2 * (worker + i) + (i == 0 ? 1 : 0)) * partial_floats<ROWS, HD>(); },
      row * HD, ROWS * HD + 2 * row, t.row0, row, t.head);
}

bool one_row_tile(const CacheAttnArgs& a) { return int64_t(a.s.max_rows) * a.group <= 8; }

// Workers of an even launch: the CTAs that are resident at once, or fewer where each would get less than two chunks a
// warp. Where that takes little away, as many to every tile: tiles of one length then begin with a worker, which has one
// tile to fetch queries for and to join. That gains 6 to 9 % with sequences of one length and loses 2 to 8 % with ragged
// ones, whose lengths the host does not know. 32 heads over 8, as many to every tile against all resident CTAs: 8
// windows of 4096 16-bit keys 29.5 us, 32.0; 8 sequences of 8191 e4m3 keys 35.4, 38.6 (16-bit 47.8, 50.6); 8 of 2000 to 8191
// 30.1, 28.9 (35.4, 34.2); 16 of 2 to 8191 67.6, 66.2 (74.6, 73.2); 2 of 101 and 32761 55.6, 51.3 (57.2, 57.8).
int decode_workers(const CacheAttnArgs& a, int kind, int64_t max_keys, int num_sms) {
  const int64_t keys = a.window > 0 ? std::min<int64_t>(max_keys, int64_t(a.window) + a.sinks + a.s.max_rows) : max_keys;
  const int64_t tiles = int64_t(a.s.n_seqs) * a.c.kv_heads, chunks = tiles * ((keys + kChunk - 1) / kChunk);
  const int64_t resident = num_sms * (kind == PLM_CACHE_E4M3 && one_row_tile(a) ? 2 : 1);
  const int64_t workers = std::max<int64_t>(1, std::min<int64_t>(resident, chunks / (2 * kWarps)));
  const int64_t whole = workers / tiles * tiles;
  return int(whole * 100 >= workers * 85 ? whole : workers);
}

template <int HD, typename T, bool E4M3, int NR>
int launch_decode(const CacheAttnArgs& a, int workers, cudaStream_t stream) {
  constexpr int SMEM = decode_smem_bytes<HD, E4M3, NR>();
  const bool even = a.s.n_seqs <= kMaxSeqs;
  auto kernel = even ? decode_attention_kernel<HD, T, E4M3, NR, true> : decode_attention_kernel<HD, T, E4M3, NR, false>;
  const int st = raise_smem_limit(reinterpret_cast<const void*>(kernel), SMEM, "decode_attention_kernel: shared memory");
  if (st != PLM_OK) return st;
  const unsigned ctas = even ? unsigned(workers) : unsigned(a.s.n_seqs) * unsigned(a.c.kv_heads);
  const int done = check_cuda(launch(kernel, dim3(ctas), dim3(kThreads), SMEM, stream, true, a), "decode_attention_kernel");
  if (done != PLM_OK || !even || workers == 1) return done;
  return check_cuda(launch(join_kernel<HD, T, 8 * NR>, dim3(ctas), dim3(32 * 8 * NR), 0, stream, true, a), "join_kernel");
}

template <int HD, typename T>
int launch_decode(const CacheAttnArgs& a, int kind, int workers, cudaStream_t stream) {
  if (kind == PLM_CACHE_E4M3)
    return one_row_tile(a) ? launch_decode<HD, T, true, 1>(a, workers, stream) : launch_decode<HD, T, true, 2>(a, workers, stream);
  return one_row_tile(a) ? launch_decode<HD, T, false, 1>(a, workers, stream) : launch_decode<HD, T, false, 2>(a, workers, stream);
}

}  // namespace

bool decode_takes(const CacheAttnArgs& a) { return int64_t(a.s.max_rows) * a.group <= 16; }

size_t decode_workspace(const CacheAttnArgs& a, int kind, int head_dim, int64_t max_keys, int num_sms) {
  if (a.s.n_seqs > kMaxSeqs) return 0;
  const int workers = decode_workers(a, kind, max_keys, num_sms);
  const size_t rows = one_row_tile(a) ? 8 : 16;
  return split_tile_bytes(workers) + 2 * size_t(workers) * rows * (head_dim + 2) * sizeof(float);
}

int decode_attention(const CacheAttnArgs& a, int kind, int dtype, int head_dim, int64_t max_keys, int num_sms,
                     cudaStream_t stream) {
  const int workers = decode_workers(a, kind, max_keys, num_sms);
  if (dtype == PLM_F16)
    return head_dim == 128 ? launch_decode<128, __half>(a, kind, workers, stream)
                           : launch_decode<64, __half>(a, kind, workers, stream);
  return head_dim == 128 ? launch_decode<128, __nv_bfloat16>(a, kind, workers, stream)
                         : launch_decode<64, __nv_bfloat16>(a, kind, workers, stream);
}

}  // namespace plm
