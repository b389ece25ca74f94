// The paged KV cache's layout and conversions, shared by its kernels.
#pragma once

#include <hip/hip_runtime.h>

#include <stdio.h>

#include "ckv_device.h"
#include "ckv_error.h"

namespace ckv {

// Rows of sequence b that are committed; a cursor out of its range must not lead a kernel out of the table.
__host__ __device__ inline int paged_capacity(const ckv_paged_cache& c) { return c.table_pages * c.page_size; }
__device__ inline int paged_log2(const ckv_paged_cache& c) { return __builtin_ctz((unsigned)c.page_size); }
__device__ inline int paged_length(const ckv_paged_cache& c, int b) {
  return min(max(gload_i32(c.lengths + b), 0), paged_capacity(c));
}
__device__ inline int step_count(const int32_t* counts, int tokens, int b) {
  return counts ? min(max(gload_i32(counts + b), 0), tokens) : tokens;
}
// A drafted token's depth: any number from 0 on, in any order of the tokens; below 2^30, so positions stay in 31 bits.
__device__ inline int draft_depth(const int32_t* depths, int64_t at) { return min(max(gload_i32(depths + at), 0), (1 << 30) - 1); }

// Two values rounded to the cache's type (to nearest even).
template <int DT>
__device__ inline uint32_t pack_store(float lo, float hi) {
  if constexpr (DT == CKV_BF16) {
    return pack_bf16x2_hw(lo, hi);
  } else {
    typedef float f32x2_t __attribute__((ext_vector_type(2)));
    typedef _Float16 f16x2_t __attribute__((ext_vector_type(2)));
    const f32x2_t v = {lo, hi};
    return __builtin_bit_cast(uint32_t, __builtin_convertvector(v, f16x2_t));
  }
}

// The two 16-bit values of a word.
template <int DT>
__device__ inline float low_value(uint32_t w) {
  if constexpr (DT == CKV_BF16) return ckv_u2f(w << 16);
  else return (float)__builtin_bit_cast(_Float16, (uint16_t)(w & 0xffffu));
}
template <int DT>
__device__ inline float high_value(uint32_t w) {
  if constexpr (DT == CKV_BF16) return ckv_u2f(w & 0xffff0000u);
  else return (float)__builtin_bit_cast(_Float16, (uint16_t)(w >> 16));
}

// Host: checks of a cache handed to a C entry; 0 or an error code.
int validate_paged_cache(const ckv_paged_cache* c, const char* what);
int check_paged_rows(const ckv_quant_rows* rows, int dtype, const char* what);
int paged_error(int code, const char* what, const char* why);
int paged_launched(const char* what);

}  // namespace ckv
