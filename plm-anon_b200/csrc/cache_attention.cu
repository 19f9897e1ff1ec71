// Attention over a paged cache of several sequences, 16-bit or e4m3 pages, causal or under the round mask, with or
// without a sliding window and sinks: one warp per (row, head), a key at a time.
#include "cache.cuh"

namespace plm {
namespace {

constexpr int kAttnWarps = 4;

struct CacheAttnArgs {
  CachePages c;
  CacheSeqs s;
  const void* q;
  int64_t q_stride;
  void* out;
  int64_t out_stride;
  int heads, group;
  float scale_log2;  // score scale in units of log2
  int window, sinks;
  const int32_t *depth, *own_start;
  int* err;
};

template <int HD, typename T, bool E4M3>
__device__ __forceinline__ void load_row(const void* plane, size_t at, float scale, int lane, float (&x)[HD / 32]) {
#pragma unroll
  for (int e = 0; e < HD / 32; ++e) {
    const size_t i = at + lane + e * 32;
    if (E4M3) {
      const uint32_t h = e4m3x2_to_f16x2(static_cast<const uint8_t*>(plane)[i]);
      x[e] = __low2float(*reinterpret_cast<const __half2*>(&h)) * scale;
    } else {
      x[e] = to_f32<T>(static_cast<const T*>(plane)[i]);
    }
  }
}

template <int HD, typename T, bool E4M3>
__global__ void __launch_bounds__(32 * kAttnWarps) attention_rows_kernel(const CacheAttnArgs a) {
  grid_dependency_wait();
  allow_dependents();
  const int warp = blockIdx.x * kAttnWarps + (threadIdx.x >> 5), lane = threadIdx.x & 31;
  const int row = warp / a.heads, head = warp % a.heads;
  if (row >= a.s.rows) return;
  const int seq = sequence_of_row(a.s, row);
  if (seq < 0) return;
  const SeqRange r = sequence_range(a.s, seq, a.err);
  if (r.n == 0) return;
  const int j = row - r.start;
  const int depth = a.depth != nullptr ? a.depth[row] : j;
  const int own = a.depth != nullptr ? a.own_start[row] : (1 << 30);
  const int64_t pos = r.context + depth + (own <= j ? j - own : 0);
  float q[HD / 32], o[HD / 32];
#pragma unroll
  for (int e = 0; e < HD / 32; ++e) {
    q[e] = to_f32<T>(static_cast<const T*>(a.q)[row * a.q_stride + head * HD + lane + e * 32]);
    o[e] = 0.f;
  }
  float m = -INFINITY, l = 0.f;
  const int kv_head = head / a.group;
  for (int64_t kv = 0; kv < r.context + r.n; ++kv) {
    const int64_t rel = kv - r.context;
    const bool visible = (rel <= depth && (a.window == 0 || kv < a.sinks || kv > pos - a.window)) ||
                         (rel >= own && rel <= j);
    if (!visible) continue;
    const int page = physical_page(a.s, a.c, seq, kv >> a.c.page_shift, lane == 0 ? a.err : nullptr);
    const bool valid = page >= 0;
    const size_t head_page = size_t(valid ? page : 0) * a.c.kv_heads + kv_head;
    const int slot = int(kv & (a.c.page_size - 1));
    const size_t at = (head_page * a.c.page_size + slot) * HD;
    const size_t block = head_page * (a.c.page_size >> a.c.block_shift) + (slot >> a.c.block_shift);
    float x[HD / 32];
    load_row<HD, T, E4M3>(a.c.k, at, E4M3 ? a.c.k_scale[block] : 1.f, lane, x);
    float dot = 0.f;
#pragma unroll
    for (int e = 0; e < HD / 32; ++e) dot += q[e] * (valid ? x[e] : 0.f);
    const float score = warp_sum(dot) * a.scale_log2;
    const float top = fmaxf(m, score), from = top == -INFINITY ? 0.f : top;
    const float keep = exp2f(m - from), w = exp2f(score - from);
    m = top;
    l = l * keep + w;
    load_row<HD, T, E4M3>(a.c.v, at, E4M3 ? a.c.v_scale[block] : 1.f, lane, x);
#pragma unroll
    for (int e = 0; e < HD / 32; ++e) o[e] = o[e] * keep + w * (valid ? x[e] : 0.f);
  }
  const float inverse = 1.f / l;
#pragma unroll
  for (int e = 0; e < HD / 32; ++e)
    static_cast<T*>(a.out)[row * a.out_stride + head * HD + lane + e * 32] = from_f32<T>(l == 0.f ? 0.f : o[e] * inverse);
}

template <int HD, typename T>
int attention_launch_kind(const CacheAttnArgs& a, int kind, cudaStream_t stream) {
  const int64_t warps = int64_t(a.s.rows) * a.heads;
  const dim3 grid(unsigned((warps + kAttnWarps - 1) / kAttnWarps));
  auto kernel = kind == PLM_CACHE_E4M3 ? attention_rows_kernel<HD, T, true> : attention_rows_kernel<HD, T, false>;
  return check_cuda(launch(kernel, grid, dim3(32 * kAttnWarps), 0, stream, true, a), "attention_rows_kernel");
}

}  // namespace
}  // namespace plm

using namespace plm;

extern "C" int plm_cache_attention(plm_ctx* ctx, const plm_cache_attention_desc* d, void* stream) {
  if (ctx == nullptr || d == nullptr) return fail(PLM_ERR_INVALID, "plm_cache_attention: null argument");
  CacheAttnArgs a = {};
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
  a.err = ctx->err;
  DeviceScope scope(ctx->device);
  if (scope.status() != PLM_OK) return scope.status();
  cudaStream_t on = static_cast<cudaStream_t>(stream);
  if (d->dtype == PLM_F16)
    return hd == 128 ? attention_launch_kind<128, __half>(a, d->cache.kind, on)
                     : attention_launch_kind<64, __half>(a, d->cache.kind, on);
  return hd == 128 ? attention_launch_kind<128, __nv_bfloat16>(a, d->cache.kind, on)
                   : attention_launch_kind<64, __nv_bfloat16>(a, d->cache.kind, on);
}
