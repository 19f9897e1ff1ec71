// plm_cache_attention: argument checks, workspace and choice of the kernel. Sequences of at most 16 packed rows (rows
// times query heads per kv head) are bound by reading the cache and go to cache_decode.cu; longer ones go to the tensor
// cores' 128-row tiles in cache_prefill.cu, and take a call's short ones along.
#include <algorithm>
#include <cmath>

#include "cache_attention.h"

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
  if (int64_t(d->rows) * d->num_heads >= (int64_t(1) << 30))
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
  return decode_takes(a) ? decode_workspace(a, d->cache.kind, d->cache.head_dim, max_keys, ctx->num_sms)
                         : prefill_workspace(a, d->cache.head_dim, max_keys, ctx->num_sms);
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
  return prefill_attention(a, d->cache.kind, d->dtype, hd, max_keys, ctx->num_sms, on);
}
