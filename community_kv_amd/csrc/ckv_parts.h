// Cache rows of a ragged batch in parts of nearly equal size, for attention
// kernels that split the rows.
#pragma once

#include "ckv_device.h"

namespace ckv {

constexpr int PART_UNIT = 128;  // the parts that cache rows are split into are multiples of this

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
  int whole;       // earlier sequences that are one part
};

__device__ inline int wave_sum_i32(int v) {
  v += (int)xor_u32<1>((uint32_t)v);
  v += (int)xor_u32<2>((uint32_t)v);
  v += (int)xor_u32<4>((uint32_t)v);
  v += (int)xor_u32<8>((uint32_t)v);
  v += (int)xor_u32<16>((uint32_t)v);
  return __builtin_amdgcn_readfirstlane(v + (int)xor_u32<32>((uint32_t)v));
}

// (The rows of a batch are below 2^38, one sequence's at most 2^30.)
template <class Lengths>
__device__ inline int part_size(const Lengths& c, int parts) {
  if (parts <= c.batch()) return 0x7fffff80;
  const int lane = threadIdx.x & 63;
  int mine = 0, units = 0;
  for (int b0 = 0; b0 < c.batch(); b0 += 64) {
    mine = b0 + lane < c.batch() ? (c(b0 + lane) + PART_UNIT - 1) / PART_UNIT : 0;
    units += mine;
  }
  units = max(wave_sum_i32(units), 1);
  uint32_t least = ((uint32_t)units + parts - 1) / (uint32_t)parts;
  if (c.batch() > 1) {
    uint32_t most = ((uint32_t)units + parts - c.batch() - 1) / (uint32_t)(parts - c.batch());
    const bool search = c.batch() <= 64 && 20 * most > 23 * least;
    while (search && least < most) {
      const uint32_t half = (least + most) / 2;
      if (wave_sum_i32(lane < c.batch() ? max((int)(((uint32_t)mine + half - 1) / half), 1) : 0) <= parts) most = half;
      else least = half + 1;
    }
    least = most;
  }
  return (int)min(least, (uint32_t)(0x40000000 / PART_UNIT)) * PART_UNIT;
}

__device__ inline int parts_of_sequence(int n, int size) { return n > size ? (n - 1) / size + 1 : 1; }

// Part number `part` (wanted < 0), or sequence `wanted`'s first part.
template <class Lengths>
__device__ inline Part find_part(const Lengths& c, int parts, int part, int wanted) {
  const int size = part_size(c, parts);
  if (parts <= c.batch()) {
    const int b = wanted < 0 ? part : wanted;
    return Part{b, 0, b, 1, size, b};
  }
  const int lane = threadIdx.x & 63;
  int before = 0, whole = 0;
  for (int b0 = 0; b0 < c.batch(); b0 += 64) {
    const int mine = b0 + lane < c.batch() ? parts_of_sequence(c(b0 + lane), size) : 0;
    const int end = before + wave_inclusive_scan(mine);  // parts up to and with this lane's sequence
    const uint64_t hit = wanted < 0 ? __ballot(mine > 0 && part < end) : __ballot(b0 + lane == wanted);
    const uint64_t single = __ballot(mine == 1);
    if (hit) {
      const int at = __ffsll((unsigned long long)hit) - 1;
      const int count = __builtin_amdgcn_readlane(mine, at), first = __builtin_amdgcn_readlane(end, at) - count;
      return Part{b0 + at, part - first, first, count, size, whole + (int)__popcll(single & ((1ull << at) - 1))};
    }
    before = __builtin_amdgcn_readlane(end, 63);
    whole += __popcll(single);
  }
  return Part{-1, 0, 0, 0, size, 0};
}

}  // namespace ckv
