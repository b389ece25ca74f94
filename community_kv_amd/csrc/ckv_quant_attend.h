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
  float* part_max;   // [kv_heads][row_pad][parts], log2
  float* part_sum;
  float* part_acc;   // [kv_heads][parts][row_pad][128]
  float2* stats;     // [batch][kv_heads][row_pad]: log2 maximum and 1 / sum (0, 0 without a row), or null
  int2* ranges;      // [batch][kv_heads][tiles]: least and largest position of every RANGE_TILE rows, or null
  float* scores;     // [batch][kv_heads][rows][capacity] masked scores, log2, or null
  float* sums;       // [shares][batch][kv_heads][capacity] received weights, or null
  float scale_log2;  // softmax_scale * log2 e
  int32_t tokens, group, rows, row_pad, window, parts;
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

// The cache rows of all sequences in `parts` parts of nearly equal size, so that
// every workgroup of a ragged batch has the same work: the least part size, in
// whole units, with which the sequences' parts, max(1, ceil(n / size)) each, are
// at most `parts` together.  The rows of the batch over parts is below it and
// those over parts - batch above, between which it is searched for where they
// are more than 15 % apart (8 sequences of 2,048 rows, 32/8 heads, in a graph: 13.6
// us, with the upper one 14.5; 24 f32 query rows over 5 sequences of 10k to 20k
// rows: 137 and 144; 8 sequences of 8k to 16k rows, 14 % apart: 54.1 either way) and
// there are up to 64 sequences.  With as many parts as sequences each sequence is
// one part.
// Every wave works this out for itself.
struct Part {
  int sequence;    // -1: none
  int index;       // within the sequence
  int first;       // number of the sequence's first part
  int count;       // the sequence's parts
  int rows;        // rows of a part
};

__device__ inline int wave_sum_i32(int v) {
  v += (int)xor_u32<1>((uint32_t)v);
  v += (int)xor_u32<2>((uint32_t)v);
  v += (int)xor_u32<4>((uint32_t)v);
  v += (int)xor_u32<8>((uint32_t)v);
  v += (int)xor_u32<16>((uint32_t)v);
  return __builtin_amdgcn_readfirstlane(v + (int)xor_u32<32>((uint32_t)v));
}

// (No overflow: 2^31 units of codes would be 2^46 bytes.)
__device__ inline int part_size(const ckv_quant_cache& c, int parts) {
  if (parts <= c.batch) return 0x7fffff80;
  const int lane = threadIdx.x & 63;
  int mine = 0, units = 0;
  for (int b0 = 0; b0 < c.batch; b0 += 64) {
    mine = b0 + lane < c.batch ? (quant_length(c, b0 + lane) + PART_UNIT - 1) / PART_UNIT : 0;
    units += mine;
  }
  units = max(wave_sum_i32(units), 1);
  uint32_t least = ((uint32_t)units + parts - 1) / (uint32_t)parts;
  if (c.batch > 1) {
    uint32_t most = ((uint32_t)units + parts - c.batch - 1) / (uint32_t)(parts - c.batch);
    const bool search = c.batch <= 64 && 20 * most > 23 * least;
    while (search && least < most) {
      const uint32_t half = (least + most) / 2;
      if (wave_sum_i32(lane < c.batch ? max((int)(((uint32_t)mine + half - 1) / half), 1) : 0) <= parts) most = half;
      else least = half + 1;
    }
    least = most;
  }
  return (int)least * PART_UNIT;
}

__device__ inline int parts_of_sequence(int n, int size) { return n > size ? (n - 1) / size + 1 : 1; }

// Part number `part` (wanted < 0), or sequence `wanted`'s first part.
__device__ inline Part find_part(const ckv_quant_cache& c, int parts, int part, int wanted) {
  const int size = part_size(c, parts);
  if (parts <= c.batch) {
    const int b = wanted < 0 ? part : wanted;
    return Part{b, 0, b, 1, size};
  }
  const int lane = threadIdx.x & 63;
  int before = 0;
  for (int b0 = 0; b0 < c.batch; b0 += 64) {
    const int mine = b0 + lane < c.batch ? parts_of_sequence(quant_length(c, b0 + lane), size) : 0;
    const int end = before + wave_inclusive_scan(mine);  // parts up to and with this lane's sequence
    const uint64_t hit = wanted < 0 ? __ballot(mine > 0 && part < end) : __ballot(b0 + lane == wanted);
    if (hit) {
      const int at = __ffsll((unsigned long long)hit) - 1;
      const int count = __builtin_amdgcn_readlane(mine, at), first = __builtin_amdgcn_readlane(end, at) - count;
      return Part{b0 + at, part - first, first, count, size};
    }
    before = __builtin_amdgcn_readlane(end, 63);
  }
  return Part{-1, 0, 0, 0, size};
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

// Positions that any of the query rows [first, first + rows) sees: [lo, hi].
__device__ inline void rows_range(const QuantAttendArgs& a, int first, int rows, int count, int seen, int* lo, int* hi) {
  const int t0 = token_of(a, first), t1 = min(token_of(a, min(first + rows, a.rows) - 1), count - 1);
  *lo = 0;
  *hi = -1;
  if (t0 > t1) return;
  int unused;
  query_range(a, t0 * a.group, count, seen, lo, &unused);
  query_range(a, t1 * a.group, count, seen, &unused, hi);
}

// Where query row `row` of KV head h goes: index of its first output element
// and of its lse.
__device__ inline void output_index(const QuantAttendArgs& a, int b, int h, int row, int64_t* out, int64_t* lse) {
  const int t = token_of(a, row), g = row - t * a.group;
  const int64_t hq = (int64_t)h * a.group + g, heads = (int64_t)a.cache.kv_heads * a.group;
  *out = (((int64_t)b * a.tokens + t) * heads + hq) * D;
  *lse = ((int64_t)b * heads + hq) * a.tokens + t;
}

// Which query rows of a head go to the many-row kernels (128 or 256 of them a
// workgroup): the few-row kernel takes 16 a workgroup and reads the cache for each
// 16, but starts sooner.  It has all calls of up to 32 rows (bf16; 64 with two or
// three pieces, whose many-row kernel is slower), and those whose cache rows, over
// all heads and blocks of 16 query rows, are at most FEW_WORK; with received
// weights only up to 128 query rows, beyond which their own kernels decide.
// 32/8 heads, in a graph, full caches, few and many, us: 1 sequence of 1,000 rows,
// bf16, 128 query rows 15.1 and 22.0, 512 rows 27.3 and 30.2; 4,000 rows: 22.4 and
// 36.4, 53.2 and 42.0; 16,000 rows, 64 query rows 31.1 and 40.6, 128 rows 49.1 and
// 42.3; 8 sequences of 16,000 rows: 32 query rows 93 and 143, 64 rows 165 and 147
// (f32: 192 and 261).  With weights, 1,000 rows: 128 query rows 29.4 and 32.6, 512
// rows 66 and 42.  The host knows the capacity alone: 36 query rows over 1,000 rows
// take 12.0 us in a cache of up to 16,384 rows, 19.6 in one of 40,960.
constexpr int64_t FEW_WORK = 720000;
inline bool many_rows(const ckv_quant_cache* c, int rows, int dtype, bool accumulate) {
  if (rows <= (dtype == CKV_BF16 ? 32 : 64)) return false;
  if (accumulate && rows > 128) return true;
  return (int64_t)c->batch * c->kv_heads * ((rows + 15) / 16) * c->capacity > FEW_WORK;
}

// Host-side launchers of the many-row kernels (ckv_quant_rows.hip).
int launch_many_rows(const QuantAttendArgs& a, int dtype, hipStream_t stream);
int launch_many_rows_weights(const QuantAttendArgs& a, int dtype, hipStream_t stream);
int many_row_block(int dtype);  // query rows of one workgroup
int many_row_shares(const ckv_quant_cache* c, int rows);  // workgroups that share a cache row's queries

}  // namespace ckv
