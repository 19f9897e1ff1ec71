// Append to a paged cache: rotate queries and keys, write keys and values into the pages of several sequences, in the
// model dtype or as e4m3 codes with a power-of-two scale per block of tokens and head.
//
// A thread works on 16 elements of a head: 8 of the first half and the 8 they are rotated with, so every access is a
// 16-byte vector (8 bytes for codes). The product of two 16-bit numbers is exact in fp32, so each rotated value is the
// exact one rounded to fp32 once, and then once to its storage type, whatever the compiler contracts. Powers of two
// as scales make dividing by them exact, and so is bringing a code from an older to a larger scale unless it becomes
// subnormal.
//
// What bounds it: HBM with long prompts, the launch with few rows. Measured: 7 prompts, 21 thousand rows, 32
// heads over 8 of 128, 16-bit pages 91 us (5.7 TB/s of rows read and written, rotated queries included), e4m3 pages 118
// us (4.0 TB/s: a block's rows are all loaded before its scale is known and its codes can go out, so a CTA's loads and
// stores alternate); one row, or 56, 2.5 us inside a graph.
#include <type_traits>

#include "cache.cuh"

namespace plm {
namespace {

constexpr int kAppendThreads = 128;
constexpr int kMaxScaleBlock = 64;
constexpr int kMinExponent = -100;  // scales stay normal floats, and so do their reciprocals

struct AppendArgs {
  CachePages c;
  CacheSeqs s;
  const void *q, *k, *v;
  int64_t q_stride, k_stride, v_stride, q_out_stride;
  void* q_out;
  const void* cos_sin;
  const int32_t* positions;
  int heads;
  int max_pos;
  int kv_units;  // e4m3: blocks of the grid that append keys and values; the rest rotate queries
  int* err;
};

// Code `at` of a word of four.
__device__ __forceinline__ float code_f32(uint32_t word, int at) {
  const uint32_t h = e4m3x2_to_f16x2(uint16_t((word >> (8 * at)) & 0xffu));
  return __low2float(*reinterpret_cast<const __half2*>(&h));
}
// Four values times `factor` as codes.
__device__ __forceinline__ uint32_t pack_codes(const float* x, float factor) {
  return uint32_t(f32x2_to_e4m3x2(x[0] * factor, x[1] * factor)) |
         uint32_t(f32x2_to_e4m3x2(x[2] * factor, x[3] * factor)) << 16;
}

// 8 elements of the model dtype as floats.
template <typename T>
__device__ __forceinline__ void load8(const T* p, float (&x)[8]) {
  const uint4 v = *reinterpret_cast<const uint4*>(p);
#pragma unroll
  for (int e = 0; e < 8; ++e) x[e] = to_f32<T>(reinterpret_cast<const T*>(&v)[e]);
}
template <typename T>
__device__ __forceinline__ void store8(T* p, const float (&x)[8]) {
  uint4 v;
#pragma unroll
  for (int e = 0; e < 8; ++e) reinterpret_cast<T*>(&v)[e] = from_f32<T>(x[e]);
  *reinterpret_cast<uint4*>(p) = v;
}

// Whether the table has the row's position, *pos (0 where it has not: that is recorded, and the row is left out).
__device__ __forceinline__ bool row_position(const AppendArgs& a, int row, int64_t logical, int64_t* pos) {
  *pos = 0;
  if (a.cos_sin == nullptr) return true;
  const int64_t given = a.positions != nullptr ? a.positions[row] : logical;
  const bool there = given >= 0 && given < a.max_pos;
  if (there) *pos = given;
  else record_error(a.err, kErrBadIndex);
  return there;
}

// Rotates (a, b) = elements [8 chunk, + 8) of both halves of a head at position `pos`.
template <int HD, typename T>
__device__ __forceinline__ void rotate(const AppendArgs& a, int64_t pos, int chunk, float (&lo)[8], float (&hi)[8]) {
  if (a.cos_sin == nullptr) return;
  const T* cs = static_cast<const T*>(a.cos_sin) + size_t(pos) * HD + chunk * 8;
  float c[8], s[8];
  load8<T>(cs, c);
  load8<T>(cs + HD / 2, s);
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const float x = lo[e], y = hi[e];
    lo[e] = x * c[e] - y * s[e];
    hi[e] = y * c[e] + x * s[e];
  }
}

// One thread's share of row `row`, slot `slot` (query heads, then key heads, then value heads): 16-bit storage.
template <int HD, typename T>
__device__ __forceinline__ void append_16bit(const AppendArgs& a, int row, int slot, int chunk) {
  const int seq = sequence_of_row(a.s, row);
  if (seq < 0) return;
  const SeqRange r = sequence_range(a.s, seq, a.err);
  if (r.n == 0) return;
  const int64_t logical = r.context + row - r.start;
  const int q_heads = a.q != nullptr ? a.heads : 0;
  float lo[8], hi[8];
  if (slot < q_heads) {
    const T* src = static_cast<const T*>(a.q) + row * a.q_stride + slot * HD + chunk * 8;
    load8<T>(src, lo);
    load8<T>(src + HD / 2, hi);
    int64_t pos;
    if (!row_position(a, row, logical, &pos)) return;
    rotate<HD, T>(a, pos, chunk, lo, hi);
    T* dst = static_cast<T*>(a.q_out) + row * a.q_out_stride + slot * HD + chunk * 8;
    store8<T>(dst, lo);
    store8<T>(dst + HD / 2, hi);
    return;
  }
  const int page = physical_page(a.s, a.c, seq, logical >> a.c.page_shift, a.err);
  if (page < 0) return;
  slot -= q_heads;
  const bool key = slot < a.c.kv_heads;
  const int head = key ? slot : slot - a.c.kv_heads;
  const T* src = (key ? static_cast<const T*>(a.k) + row * a.k_stride : static_cast<const T*>(a.v) + row * a.v_stride) +
                 head * HD + chunk * 8;
  T* dst = static_cast<T*>(key ? a.c.k : a.c.v) +
           ((size_t(page) * a.c.kv_heads + head) * a.c.page_size + size_t(logical & (a.c.page_size - 1))) * HD + chunk * 8;
  load8<T>(src, lo);
  load8<T>(src + HD / 2, hi);
  int64_t pos;
  if (!row_position(a, row, logical, &pos)) return;
  if (key) rotate<HD, T>(a, pos, chunk, lo, hi);
  store8<T>(dst, lo);
  store8<T>(dst + HD / 2, hi);
}

template <int HD, typename T>
__global__ void __launch_bounds__(kAppendThreads) append_rows_kernel(const AppendArgs a) {
  grid_dependency_wait();
  allow_dependents();
  constexpr int CH = HD / 16;
  const int slots = (a.q != nullptr ? a.heads : 0) + 2 * a.c.kv_heads;
  const int64_t item = int64_t(blockIdx.x) * kAppendThreads + threadIdx.x;
  const int64_t head_row = item / CH;
  if (head_row >= int64_t(a.s.rows) * slots) return;
  append_16bit<HD, T>(a, int(head_row / slots), int(head_row % slots), int(item % CH));
}

// ceil(log2(amax / 448)), at least kMinExponent: 448 = 1.75 * 2^8, so with amax = f * 2^x it is x - 8 where
// f <= 1.75 and x - 7 above.
__device__ __forceinline__ int scale_exponent(float amax) {
  const uint32_t bits = __float_as_uint(amax);
  const int x = int(bits >> 23) - 127;
  const int e = x - 8 + ((bits & 0x7fffffu) > 0x600000u ? 1 : 0);
  return max(e, kMinExponent);
}

__device__ __forceinline__ float exp2_int(int e) { return __uint_as_float(uint32_t(e + 127) << 23); }

// The sequence and block of token-block `unit` of the call (blocks in sequence order). Returns the sequence, or -1 past
// the last block; one warp.
__device__ __forceinline__ int locate_block(const CacheSeqs& s, int unit, int block_shift, SeqRange* range,
                                            int64_t* block, int* err) {
  const int lane = threadIdx.x & 31;
  int before = 0;
  for (int base = 0; base < s.n_seqs; base += 32) {
    SeqRange r = {0, 0, 0};
    int count = 0;
    if (base + lane < s.n_seqs) {
      r = sequence_range(s, base + lane, err);
      if (r.n > 0) count = int(((r.context + r.n - 1) >> block_shift) - (r.context >> block_shift)) + 1;
    }
    int upto = count;
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) {
      const int other = __shfl_up_sync(0xffffffffu, upto, off);
      if (lane >= off) upto += other;
    }
    upto += before;
    const uint32_t past = __ballot_sync(0xffffffffu, upto > unit);
    if (past != 0) {
      const int owner = __ffs(past) - 1;
      range->start = __shfl_sync(0xffffffffu, r.start, owner);
      range->n = __shfl_sync(0xffffffffu, r.n, owner);
      range->context = __shfl_sync(0xffffffffu, r.context, owner);
      const int first = __shfl_sync(0xffffffffu, upto - count, owner);
      *block = (range->context >> block_shift) + (unit - first);
      return base + owner;
    }
    before = __shfl_sync(0xffffffffu, upto, 31);
  }
  return -1;
}

// e4m3 pages: a CTA per (block of tokens, kv head) that the call's rows fall into, half of it for K and half for V. Each
// half holds the block's new values in registers (PASSES times as many tokens as it covers at once), agrees on their
// maximum, and writes scale and codes; the rest of the grid rotates queries. Bound by HBM for long prompts; what has to
// follow what (sequence, rows and page, old scale, codes) is kept to one load each.
template <int HD, typename T, int PASSES>
__global__ void __launch_bounds__(2 * kAppendThreads) append_e4m3_kernel(const AppendArgs a) {
  constexpr int CH = HD / 16;
  constexpr int TOK = kAppendThreads / CH;  // tokens a pass over the block covers
  __shared__ float warp_amax[2 * kAppendThreads / 32];
  grid_dependency_wait();
  allow_dependents();
  if (int(blockIdx.x) >= a.kv_units) {
    const int64_t item = int64_t(int(blockIdx.x) - a.kv_units) * 2 * kAppendThreads + threadIdx.x;
    const int64_t head_row = item / CH;
    if (head_row < int64_t(a.s.rows) * a.heads)
      append_16bit<HD, T>(a, int(head_row / a.heads), int(head_row % a.heads), int(item % CH));
    return;
  }
  const bool key = threadIdx.x < kAppendThreads;
  const int tid = threadIdx.x % kAppendThreads, chunk = tid % CH;
  const int head = int(blockIdx.x) % a.c.kv_heads;
  SeqRange r;
  int64_t block;
  const int seq = locate_block(a.s, int(blockIdx.x) / a.c.kv_heads, a.c.block_shift, &r, &block, a.err);
  if (seq < 0) return;
  const int size = 1 << a.c.block_shift;
  const int64_t first = block << a.c.block_shift;
  const int begin = int(max(r.context - first, int64_t(0)));  // the block's tokens before this call
  const int end = int(min(r.context + r.n - first, int64_t(size)));
  const T* src = static_cast<const T*>(key ? a.k : a.v) + head * HD + chunk * 8;
  const int64_t stride = key ? a.k_stride : a.v_stride;

  float lo[PASSES][8], hi[PASSES][8];
#pragma unroll
  for (int p = 0; p < PASSES; ++p) {
    const int token = tid / CH + p * TOK;
    if (token < begin || token >= end) continue;
    const int64_t row = r.start + first + token - r.context;
    load8<T>(src + row * stride, lo[p]);
    load8<T>(src + row * stride + HD / 2, hi[p]);
  }
  const int page = physical_page(a.s, a.c, seq, first >> a.c.page_shift, a.err);
  float amax = -1.f;  // of the tokens that have a position; below 0: there is none
  uint32_t there = 0;  // those of this thread, by pass
#pragma unroll
  for (int p = 0; p < PASSES; ++p) {
    const int token = tid / CH + p * TOK;
    if (token < begin || token >= end) continue;
    int64_t pos;
    const bool counts = row_position(a, int(r.start + first + token - r.context), first + token, &pos);
    if (key) rotate<HD, T>(a, pos, chunk, lo[p], hi[p]);
    if (!counts) continue;
    there |= 1u << p;
    amax = fmaxf(amax, 0.f);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float x = fabsf(lo[p][e]), y = fabsf(hi[p][e]);
      if (x < INFINITY) amax = fmaxf(amax, x);  // false for infinities and NaN
      if (y < INFINITY) amax = fmaxf(amax, y);
    }
  }
  if (page < 0) return;  // the whole CTA
  const size_t head_page = size_t(page) * a.c.kv_heads + head;
  const int slot0 = int(first & (a.c.page_size - 1));
  uint8_t* codes = static_cast<uint8_t*>(key ? a.c.k : a.c.v) + (head_page * a.c.page_size + slot0) * HD + chunk * 8;
  float* scale = (key ? a.c.k_scale : a.c.v_scale) + head_page * (a.c.page_size >> a.c.block_shift) +
                 (slot0 >> a.c.block_shift);
  const float old = begin > 0 ? *scale : 0.f;
  amax = warp_max(amax);
  if ((tid & 31) == 0) warp_amax[threadIdx.x >> 5] = amax;
  __syncthreads();  // also: every thread has read the old scale
#pragma unroll
  for (int w = 0; w < kAppendThreads / 32; ++w) amax = fmaxf(amax, warp_amax[(key ? 0 : kAppendThreads / 32) + w]);
  if (amax < 0.f) return;  // nothing to append: the block stays as it is
  const float now = fmaxf(exp2_int(scale_exponent(amax)), old);
  const float inverse = 1.f / now;
  if (tid == 0) *scale = now;
#pragma unroll
  for (int p = 0; p < PASSES; ++p) {
    const int token = tid / CH + p * TOK;
    if (token >= end) continue;
    uint2* at_lo = reinterpret_cast<uint2*>(codes + token * HD);
    uint2* at_hi = reinterpret_cast<uint2*>(codes + token * HD + HD / 2);
    float factor = inverse;
    if (token < begin) {
      if (now == old) continue;
      const uint2 was[2] = {*at_lo, *at_hi};
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        lo[p][e] = code_f32(e < 4 ? was[0].x : was[0].y, e & 3);
        hi[p][e] = code_f32(e < 4 ? was[1].x : was[1].y, e & 3);
      }
      factor = old * inverse;
    } else if (!(there >> p & 1)) {
      continue;
    }
    uint32_t out[4];
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      out[e] = pack_codes(lo[p] + 4 * e, factor);
      out[2 + e] = pack_codes(hi[p] + 4 * e, factor);
    }
    *at_lo = make_uint2(out[0], out[1]);
    *at_hi = make_uint2(out[2], out[3]);
  }
}

template <int HD, typename T>
int append_launch(AppendArgs a, int kind, cudaStream_t stream) {
  constexpr int CH = HD / 16;
  const int q_heads = a.q != nullptr ? a.heads : 0;
  if (kind == PLM_CACHE_MODEL) {
    const int64_t items = int64_t(a.s.rows) * (q_heads + 2 * a.c.kv_heads) * CH;
    const int64_t blocks = (items + kAppendThreads - 1) / kAppendThreads;
    return check_cuda(launch(append_rows_kernel<HD, T>, dim3(unsigned(blocks)), dim3(kAppendThreads), 0, stream, true, a),
                      "append_rows_kernel");
  }
  // A sequence's rows touch at most rows blocks, and at most two more than its full ones.
  const int64_t blocks = std::min<int64_t>(a.s.rows, (a.s.rows >> a.c.block_shift) + 2 * int64_t(a.s.n_seqs));
  const int64_t units = blocks * a.c.kv_heads;
  constexpr int THREADS = 2 * kAppendThreads;
  const int64_t q_blocks = (int64_t(a.s.rows) * q_heads * CH + THREADS - 1) / THREADS;
  a.kv_units = int(units);
  constexpr int TOK = kAppendThreads / CH;
  const int size = 1 << a.c.block_shift;
  auto kernel = size <= TOK ? append_e4m3_kernel<HD, T, 1>
                            : size <= 2 * TOK ? append_e4m3_kernel<HD, T, 2> : append_e4m3_kernel<HD, T, kMaxScaleBlock / TOK>;
  return check_cuda(launch(kernel, dim3(unsigned(units + q_blocks)), dim3(THREADS), 0, stream, true, a),
                    "append_e4m3_kernel");
}

bool power_of_two(int x) { return x > 0 && (x & (x - 1)) == 0; }

}  // namespace

int cache_arguments(const char* what, const plm_paged_cache& c, const plm_sequences& s, int dtype, int rows,
                    CachePages* pages, CacheSeqs* seqs) {
  if (dtype != PLM_BF16 && dtype != PLM_F16) return fail(PLM_ERR_INVALID, "%s: dtype %d", what, dtype);
  if (c.kind != PLM_CACHE_MODEL && c.kind != PLM_CACHE_E4M3) return fail(PLM_ERR_INVALID, "%s: cache kind %d", what, c.kind);
  if (c.head_dim != 64 && c.head_dim != 128)
    return fail(PLM_ERR_UNSUPPORTED, "%s: head_dim %d (64 or 128)", what, c.head_dim);
  if (!power_of_two(c.page_size) || c.page_size > 4096)
    return fail(PLM_ERR_UNSUPPORTED, "%s: page size %d (a power of two, at most 4096)", what, c.page_size);
  if (c.num_pages < 1 || c.num_kv_heads < 1 || c.num_kv_heads > 1024)
    return fail(PLM_ERR_INVALID, "%s: %d pages of %d kv heads", what, c.num_pages, c.num_kv_heads);
  if (!c.k || !c.v || !aligned16(c.k) || !aligned16(c.v))
    return fail(PLM_ERR_INVALID, "%s: the cache's pages are missing or not 16-byte aligned", what);
  if (c.kind == PLM_CACHE_E4M3) {
    if (!c.k_scale || !c.v_scale) return fail(PLM_ERR_INVALID, "%s: an e4m3 cache needs its scales", what);
    if (!power_of_two(c.scale_block) || c.scale_block > c.page_size || c.scale_block > kMaxScaleBlock)
      return fail(PLM_ERR_UNSUPPORTED, "%s: %d tokens to a scale (a power of two, at most the page size %d and %d)", what,
                  c.scale_block, c.page_size, kMaxScaleBlock);
  }
  if (s.n_seqs < 1 || s.n_seqs > 65535) return fail(PLM_ERR_INVALID, "%s: %d sequences", what, s.n_seqs);
  if (rows < 1 || rows > (1 << 24) || s.max_rows < 1)
    return fail(PLM_ERR_INVALID, "%s: %d rows, at most %d to a sequence", what, rows, s.max_rows);
  if (!s.row_start || !s.context || !s.block_tables) return fail(PLM_ERR_INVALID, "%s: null operand", what);
  if (s.max_pages < 1 || s.table_stride < s.max_pages || int64_t(s.max_pages) * c.page_size >= (int64_t(1) << 30))
    return fail(PLM_ERR_INVALID, "%s: block tables of %d pages, %lld apart", what, s.max_pages, (long long)s.table_stride);
  pages->k = c.k;
  pages->v = c.v;
  pages->k_scale = c.k_scale;
  pages->v_scale = c.v_scale;
  pages->block_shift = c.kind == PLM_CACHE_E4M3 ? __builtin_ctz(unsigned(c.scale_block)) : 0;
  pages->page_shift = __builtin_ctz(unsigned(c.page_size));
  pages->page_size = c.page_size;
  pages->num_pages = c.num_pages;
  pages->kv_heads = c.num_kv_heads;
  seqs->row_start = s.row_start;
  seqs->context = s.context;
  seqs->tables = s.block_tables;
  seqs->table_stride = s.table_stride;
  seqs->max_tokens = int64_t(s.max_pages) * c.page_size;
  seqs->n_seqs = s.n_seqs;
  seqs->max_rows = s.max_rows;
  seqs->rows = rows;
  return PLM_OK;
}

}  // namespace plm

using namespace plm;

extern "C" int plm_cache_append(plm_ctx* ctx, const plm_cache_append_desc* d, void* stream) {
  if (ctx == nullptr || d == nullptr) return fail(PLM_ERR_INVALID, "plm_cache_append: null argument");
  AppendArgs a = {};
  int st = cache_arguments("plm_cache_append", d->cache, d->seqs, d->dtype, d->rows, &a.c, &a.s);
  if (st != PLM_OK) return st;
  const int hd = d->cache.head_dim;
  const int64_t kv_width = int64_t(d->cache.num_kv_heads) * hd, q_width = int64_t(d->num_heads) * hd;
  if (!d->k || !d->v || !aligned16(d->k) || !aligned16(d->v) || d->k_stride < kv_width || d->v_stride < kv_width ||
      d->k_stride % 8 != 0 || d->v_stride % 8 != 0)
    return fail(PLM_ERR_INVALID, "plm_cache_append: k and v need 16-byte aligned rows of at least %lld elements",
                (long long)kv_width);
  if (d->q != nullptr &&
      (d->num_heads < 1 || d->num_heads > 4096 || !d->q_out || !aligned16(d->q) || !aligned16(d->q_out) ||
       d->q_stride < q_width || d->q_out_stride < q_width || d->q_stride % 8 != 0 || d->q_out_stride % 8 != 0))
    return fail(PLM_ERR_INVALID, "plm_cache_append: q and q_out need 16-byte aligned rows of %d heads", d->num_heads);
  if (d->cos_sin != nullptr && (!aligned16(d->cos_sin) || d->max_pos < 1))
    return fail(PLM_ERR_INVALID, "plm_cache_append: cos_sin must be 16-byte aligned, with max_pos rows");
  const int64_t lanes = int64_t(d->rows) * ((d->q ? d->num_heads : 0) + 2 * int64_t(d->cache.num_kv_heads));
  if (lanes >= (int64_t(1) << 31)) return fail(PLM_ERR_UNSUPPORTED, "plm_cache_append: %lld heads in one call", (long long)lanes);
  a.q = d->q;
  a.k = d->k;
  a.v = d->v;
  a.q_stride = d->q_stride;
  a.k_stride = d->k_stride;
  a.v_stride = d->v_stride;
  a.q_out = d->q_out;
  a.q_out_stride = d->q_out_stride;
  a.cos_sin = d->cos_sin;
  a.positions = d->positions;
  a.heads = d->num_heads;
  a.max_pos = d->max_pos;
  a.err = ctx->err;
  DeviceScope scope(ctx->device);
  if (scope.status() != PLM_OK) return scope.status();
  cudaStream_t on = static_cast<cudaStream_t>(stream);
  if (d->dtype == PLM_F16)
    return hd == 128 ? append_launch<128, __half>(a, d->cache.kind, on) : append_launch<64, __half>(a, d->cache.kind, on);
  return hd == 128 ? append_launch<128, __nv_bfloat16>(a, d->cache.kind, on)
                   : append_launch<64, __nv_bfloat16>(a, d->cache.kind, on);
}
