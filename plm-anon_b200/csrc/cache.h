// Argument blocks of the paged-cache operators over several sequences (cache_append.cu, cache_attention.cu), and the
// host checks they share.
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

#include "../../include/plm_native.h"
#include "runtime.h"

namespace plm {

// plm_paged_cache with its powers of two as shifts.
struct CachePages {
  void *k, *v;
  float *k_scale, *v_scale;
  int block_shift;    // log2 of the tokens that share a scale (e4m3)
  int page_shift;
  int page_size;
  int num_pages;
  int kv_heads;
};

struct CacheSeqs {
  const int32_t* row_start;
  const int64_t* context;
  const int32_t* tables;
  int64_t table_stride;
  int64_t max_tokens;  // max_pages * page_size: the longest sequence a block table can hold
  int n_seqs;
  int max_rows;
  int rows;            // rows of the call's buffers
};

// One sequence of a call as the device arrays give it; n = 0 where they are empty or contradict the host's bounds (the
// latter is recorded).
struct SeqRange {
  int start, n;
  int64_t context;
};

// Validates what plm_cache_append and plm_cache_attention share and fills the argument blocks.
int cache_arguments(const char* what, const plm_paged_cache& c, const plm_sequences& s, int dtype, int rows,
                    CachePages* pages, CacheSeqs* seqs);

// The context's device for the duration of a call, whatever device the caller has current.
class DeviceScope {
 public:
  explicit DeviceScope(int device) {
    status_ = check_cuda(cudaGetDevice(&before_), "cudaGetDevice");
    if (status_ == PLM_OK && before_ != device) {
      status_ = check_cuda(cudaSetDevice(device), "cudaSetDevice");
      switched_ = status_ == PLM_OK;
    }
  }
  ~DeviceScope() {
    if (switched_) cudaSetDevice(before_);
  }
  int status() const { return status_; }

 private:
  int before_ = 0, status_ = PLM_OK;
  bool switched_ = false;
};

inline bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

}  // namespace plm
