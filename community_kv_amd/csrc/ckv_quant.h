// The 8-bit KV cache's layout and conversions, shared by its kernels.
#pragma once

#include "ckv_device.h"
#include "ckv_error.h"

namespace ckv {

constexpr int QMIN_EXP = -64;  // smallest exponent of a block scale: every scale and its reciprocal is a normal number

// Addresses of one (sequence, head) of a cache.  Rows are counted in 64 bits:
// a cache may hold more than 2^32 bytes.
struct QuantHead {
  uint8_t *key_codes, *value_codes;
  float *key_scales, *value_scales;
  int32_t* positions;
  float* weights;  // null: none
  __device__ uint8_t* codes(int tensor) const { return tensor ? value_codes : key_codes; }
  __device__ float* scales(int tensor) const { return tensor ? value_scales : key_scales; }
};

__device__ inline QuantHead quant_head(const ckv_quant_cache& c, int b, int h) {
  const int64_t head = (int64_t)b * c.kv_heads + h;
  const int64_t row0 = head * c.capacity;
  const int64_t blk0 = head * (c.capacity / c.block);
  QuantHead q;
  q.key_codes = reinterpret_cast<uint8_t*>(c.key_codes) + row0 * D;
  q.value_codes = reinterpret_cast<uint8_t*>(c.value_codes) + row0 * D;
  q.key_scales = c.key_scales + blk0;
  q.value_scales = c.value_scales + blk0;
  q.positions = c.positions + row0;
  q.weights = c.weights ? c.weights + row0 : nullptr;
  return q;
}

// Rows in use of sequence b; a cursor out of its range must not lead a kernel out of the cache.
__device__ inline int quant_length(const ckv_quant_cache& c, int b) { return min(max(c.cursors[b], 0), c.capacity); }

// 2^e, the smallest with amax <= 448 * 2^e and e >= QMIN_EXP (448 = 1.75 * 2^8;
// amax is finite and >= 0, so its bits order like its value).
__device__ inline float block_scale(float amax) {
  const uint32_t bits = ckv_f2u(amax);
  int e = (int)(bits >> 23) - 127 - 8;
  if ((bits & 0x7fffffu) > 0x600000u) e += 1;
  return ckv_u2f((uint32_t)(max(e, QMIN_EXP) + 127) << 23);
}

__device__ inline bool finite_f32(float x) { return (ckv_f2u(x) & 0x7f800000u) != 0x7f800000u; }

// |x| where x is finite, else 0: what counts for a block's scale.
__device__ inline float finite_abs(float x) { return finite_f32(x) ? fabsf(x) : 0.0f; }

// 1 / s of a power of two in [2^-126, 2^126] (exact).
__device__ inline float inverse_scale(float s) { return ckv_u2f((254u << 23) - ckv_f2u(s)); }

// Four values of at most 448, or not finite, to E4M3 codes: round to nearest
// even; what is not finite becomes NaN.
__device__ inline uint32_t encode4(float a, float b, float c, float d) {
  const float nan = __builtin_nanf("");
  a = finite_f32(a) ? a : nan;
  b = finite_f32(b) ? b : nan;
  c = finite_f32(c) ? c : nan;
  d = finite_f32(d) ? d : nan;
  int w = 0;
  w = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, w, false);
  w = __builtin_amdgcn_cvt_pk_fp8_f32(c, d, w, true);
  return (uint32_t)w;
}

__device__ inline void decode4(uint32_t w, float* out) {
  typedef float f32x2_t __attribute__((ext_vector_type(2)));
  const f32x2_t lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, false);
  const f32x2_t hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, true);
  out[0] = lo[0];
  out[1] = lo[1];
  out[2] = hi[0];
  out[3] = hi[1];
}

// Largest of x over a workgroup of 256 threads (every thread gets it).
__device__ inline float block_max256(float x, float* scratch) {
  x = wave_max(x);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) scratch[threadIdx.x >> 6] = x;
  __syncthreads();
  return fmaxf(fmaxf(scratch[0], scratch[1]), fmaxf(scratch[2], scratch[3]));
}

// Host: checks of a cache handed to a C entry; 0 or an error code.
int validate_quant_cache(const ckv_quant_cache* c, const char* what);

}  // namespace ckv
