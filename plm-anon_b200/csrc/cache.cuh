// Device helpers of the paged-cache operators.
#pragma once

#include <cuda_fp8.h>

#include "cache.h"
#include "common.cuh"

namespace plm {

__device__ __forceinline__ SeqRange sequence_range(const CacheSeqs& s, int i, int* err) {
  const int lo = s.row_start[i], hi = s.row_start[i + 1];
  const int64_t context = s.context[i];
  SeqRange r = {lo, hi - lo, context};
  // Of any context, 2^63 - 1 included: context + r.n could pass 64 bits.
  if (lo < 0 || hi < lo || hi > s.rows || r.n > s.max_rows || context < 0 || context > s.max_tokens - r.n) {
    record_error(err, kErrBadIndex);
    r.n = 0;
  }
  return r;
}

// The sequence that holds row r of the call's buffers, or -1: the last one that starts at or before r.
__device__ __forceinline__ int sequence_of_row(const CacheSeqs& s, int r) {
  int lo = 0, hi = s.n_seqs;  // row_start[lo] <= r < row_start[hi], once checked
  if (r < s.row_start[0] || r >= s.row_start[s.n_seqs]) return -1;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (s.row_start[mid] <= r) lo = mid;
    else hi = mid;
  }
  return lo;
}

// Physical page of logical page lp of sequence i, or -1 (recorded) where the table has none.
__device__ __forceinline__ int physical_page(const CacheSeqs& s, const CachePages& c, int i, int64_t lp, int* err) {
  const int page = s.tables[i * s.table_stride + lp];
  if (page >= 0 && page < c.num_pages) return page;
  record_error(err, kErrBadIndex);
  return -1;
}

// Two e4m3 codes (low byte first) as f16x2, exactly.
__device__ __forceinline__ uint32_t e4m3x2_to_f16x2(uint16_t codes) {
  uint32_t out;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(out) : "h"(codes));
  return out;
}
// Two floats rounded to e4m3, `lo` in the low byte; beyond +-448 saturates, NaN stays NaN.
__device__ __forceinline__ uint16_t f32x2_to_e4m3x2(float lo, float hi) {
  uint16_t out;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(out) : "f"(hi), "f"(lo));
  return out;
}

}  // namespace plm
