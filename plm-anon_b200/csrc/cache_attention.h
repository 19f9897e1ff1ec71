// Argument block of attention over a paged cache, shared by its kernels (cache_attention.cu, cache_prefill.cu).
#pragma once

#include "cache.h"

namespace plm {

struct CacheAttnArgs {
  CachePages c;
  CacheSeqs s;
  const void* q;
  int64_t q_stride;
  void* out;
  int64_t out_stride;
  int heads, group;  // group: query heads of a kv head
  float scale_log2;  // of the scores, in units of log2
  int window, sinks;
  const int32_t *depth, *own_start;
  int splits;        // CTAs that share a unit's keys (cache_prefill.cu)
  void* workspace;
  int* err;
};

// Sequences of at most 16 packed rows (cache_decode.cu): whether all of a call's are, the bytes of workspace the call
// needs, and the launch.
bool decode_takes(const CacheAttnArgs& a);
size_t decode_workspace(const CacheAttnArgs& a, int kind, int head_dim, int64_t max_keys, int num_sms);
int decode_attention(const CacheAttnArgs& a, int kind, int dtype, int head_dim, int64_t max_keys, int num_sms,
                     cudaStream_t stream);
// All others (cache_prefill.cu).
size_t prefill_workspace(const CacheAttnArgs& a, int head_dim, int64_t max_keys, int num_sms);
int prefill_attention(const CacheAttnArgs& a, int kind, int dtype, int head_dim, int64_t max_keys, int num_sms,
                      cudaStream_t stream);

}  // namespace plm
