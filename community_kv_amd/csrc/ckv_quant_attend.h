// Arguments and small pieces that the kernels of attention over the 8-bit KV
// cache share.
#pragma once

#include <hip/hip_runtime.h>

#include <stdio.h>

#include "ckv_quant.h"
#include "ckv_tile.h"

namespace ckv {

constexpr int PART_UNIT = 128;  // the parts that cache rows are split into are multiples of this
constexpr int RANGE_TILE = 64;  // rows of one entry of `ranges`
constexpr float LN2 = 0.6931471805599453f;
constexpr float RESCALE = 8.0f;  // log2: how far scores may exceed the running maximum before it moves

struct QuantAttendArgs {
  ckv_quant_cache cache;
  ckv_quant_rows query;
  const int32_t* counts;
  void* out;
  float* lse;
  float* part_max;   // [batch][kv_heads][row_pad][splits], log2
  float* part_sum;
  float* part_acc;   // [batch][kv_heads][splits][row_pad][128]
  float2* stats;     // [batch][kv_heads][row_pad]: log2 maximum and 1 / sum (0, 0 without a row), or null
  int2* ranges;      // [batch][kv_heads][tiles]: least and largest position of every RANGE_TILE rows, or null
  float* sums;       // [shares][batch][kv_heads][capacity] received weights, or null
  float scale_log2;  // softmax_scale * log2 e
  int32_t tokens, group, rows, row_pad, window, splits;
  uint32_t group_magic;  // ceil(2^32 / group), 0 for a group of one
};

// Two E4M3 codes in the low / high half of `w` as bf16 (exact).
template <bool HIGH>
__device__ inline uint32_t codes_to_bf16(uint32_t w) {
  typedef __bf16 bf16x2_t __attribute__((ext_vector_type(2)));
  return __builtin_bit_cast(uint32_t, (bf16x2_t)__builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.0f, HIGH));
}

__device__ inline uint4 codes8_to_bf16(uint32_t lo, uint32_t hi) {
  return uint4{codes_to_bf16<false>(lo), codes_to_bf16<true>(lo), codes_to_bf16<false>(hi), codes_to_bf16<true>(hi)};
}

constexpr int pieces(int dt) { return dt == CKV_BF16 ? 1 : dt == CKV_F16 ? 2 : 3; }

// x as a sum of NP bf16 values (each the nearest to what is left).
template <int NP>
__device__ inline void split_pair(float a, float b, uint32_t* out, int stride) {
#pragma unroll
  for (int p = 0; p < NP; ++p) {
    const uint32_t w = pack_bf16x2_hw(a, b);
    out[p * stride] = w;
    a -= ckv_u2f(w << 16);
    b -= ckv_u2f(w & 0xffff0000u);
  }
}

template <int DT>
__device__ inline void load_query8(const void* base, int64_t index, float* out) {
  if constexpr (DT == CKV_F16) {
    const uint4 raw = gload16(reinterpret_cast<const uint16_t*>(base) + index);
    const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      out[2 * i] = (float)__builtin_bit_cast(_Float16, (uint16_t)(w[i] & 0xffffu));
      out[2 * i + 1] = (float)__builtin_bit_cast(_Float16, (uint16_t)(w[i] >> 16));
    }
  } else {
    load8<DT>(base, index, out);
  }
}

template <int DT>
__device__ inline void store_out(void* base, int64_t index, float v) {
  if constexpr (DT == CKV_BF16) reinterpret_cast<uint16_t*>(base)[index] = ckv_f32_to_bf16_bits(v);
  else if constexpr (DT == CKV_F16) reinterpret_cast<_Float16*>(base)[index] = (_Float16)v;
  else reinterpret_cast<float*>(base)[index] = v;
}

__device__ inline int new_count(const QuantAttendArgs& a, int b) {
  return a.counts ? min(max(a.counts[b], 0), a.tokens) : a.tokens;
}

// The rows [lo, hi) of part `split`: equal parts of whole units.
__host__ __device__ inline int part_rows(int n, int splits) {
  return ((n + splits - 1) / splits + PART_UNIT - 1) / PART_UNIT * PART_UNIT;
}

// row / group without a division: exact while row * group < 2^32 (rows are below 2^22, groups at most 16).
__device__ inline int token_of(const QuantAttendArgs& a, int row) {
  return a.group_magic ? (int)__umulhi((uint32_t)row, a.group_magic) : row;
}

// Positions that query row `row` may see: [lo, hi].
__device__ inline void query_range(const QuantAttendArgs& a, int row, int count, int seen, int* lo, int* hi) {
  const int t = token_of(a, row);
  const bool ok = row < a.rows && t < count;
  const int at = seen - count + t;
  *hi = ok ? at : -1;
  *lo = a.window > 0 && at >= a.window ? at - a.window + 1 : 0;  // no position is negative
}

// Where query row `row` of KV head h goes: index of its first output element
// and of its lse.
__device__ inline void output_index(const QuantAttendArgs& a, int b, int h, int row, int64_t* out, int64_t* lse) {
  const int t = token_of(a, row), g = row - t * a.group;
  const int64_t hq = (int64_t)h * a.group + g, heads = (int64_t)a.cache.kv_heads * a.group;
  *out = (((int64_t)b * a.tokens + t) * heads + hq) * D;
  *lse = ((int64_t)b * heads + hq) * a.tokens + t;
}

// More query rows than this a head go to the many-row kernels.
constexpr int FEW_ROWS = 64;

// Host-side launchers of the many-row kernels (ckv_quant_rows.hip).
int launch_many_rows(const QuantAttendArgs& a, int dtype, hipStream_t stream);
int launch_many_rows_weights(const QuantAttendArgs& a, int dtype, hipStream_t stream);
int many_row_block(int dtype);  // query rows of one workgroup
int many_row_shares(const ckv_quant_cache* c, int rows);  // workgroups that share a cache row's queries

}  // namespace ckv
