// Arguments and small pieces that the kernels of attention over the paged KV
// cache share.
#pragma once

#include "ckv_paged.h"
#include "ckv_parts.h"

namespace ckv {

constexpr float PAGED_LN2 = 0.6931471805599453f;
constexpr float PAGED_RESCALE = 8.0f;  // log2: how far scores may exceed the running maximum before it moves

// Running maxima are kept of the products q . k, without the scale, and an exponent is (q . k - maximum) times the
// scale: the difference first, which is exact where it matters, so the largest score's exponent is the 0 that it is.
// Scaled first, a product of M log2 units is off by 2^-24 M, and from 2^25 on probabilities leave the types' range.

// Probabilities are kept 2^bias times as large: at most 2^(8 + 7) fits fp16, and
// ones below 2^-14 of the maximum, of which a long context has many, keep their
// bits down to 2^-21 (2^-31 in steps).  bf16 has the exponents without it.
template <int DT>
constexpr float prob_bias() { return DT == CKV_F16 ? 7.0f : 0.0f; }

struct PagedAttendArgs {
  ckv_paged_cache cache;   // pages of this layer
  ckv_quant_rows query;
  const int32_t* counts;
  const int32_t* depths;   // null: a chain
  const uint64_t* masks;
  void* out;
  float* lse;
  float* part_max;         // [kv_heads][row_pad][slots], unscaled
  float* part_sum;
  float* part_acc;         // [kv_heads][slots][row_pad][128]
  int2* part_of;           // [batch]: the slot of a sequence's first part, and the number of parts
  float scale_log2;        // softmax_scale * log2 e
  float grow_by;           // PAGED_RESCALE / scale_log2
  int32_t tokens, group, rows, row_pad, window, parts, slots, words, page_log2;
  uint32_t group_magic;    // ceil(2^32 / group), 0 for a group of one
};

// A sequence's rows in use: committed ones and the step's, as far as there is room; none without a new token.
struct PagedStep {
  int start, count, total;
  __device__ PagedStep(const PagedAttendArgs& a, int b)
      : start(paged_length(a.cache, b)), count(step_count(a.counts, a.tokens, b)) {
    total = count ? min(start + count, paged_capacity(a.cache)) : 0;
  }
  // First row that any of the step's tokens may see, down to a whole part unit.
  __device__ int first(const PagedAttendArgs& a) const {
    return a.window > 0 ? max(start - a.window + 1, 0) & -PART_UNIT : 0;
  }
};

// The rows that a batch's parts are made of (see Part).
struct PagedRows {
  const PagedAttendArgs& a;
  __device__ int batch() const { return a.cache.batch; }
  __device__ int operator()(int b) const {
    const PagedStep s(a, b);
    return max(s.total - s.first(a), 0);
  }
};

// Where a part leaves its results for the join: -1, nowhere, where the sequence has no other.  With `extra` parts more than
// sequences at most `extra` are cut, into 2 `extra` parts together.
__device__ inline int part_slot(const Part& part) { return part.count > 1 ? part.first - part.whole + part.index : -1; }
inline int part_slots(int parts, int batch) { return min(parts, 2 * (parts - batch)); }

// The parts of a sequence, told to the join by its first one.
__device__ inline void tell_parts(const PagedAttendArgs& a, const Part& part) {
  if (a.parts > a.cache.batch && part.index == 0 && blockIdx.x % a.cache.kv_heads == 0 && blockIdx.y == 0 && threadIdx.x == 0)
    a.part_of[part.sequence] = int2{part_slot(part), part.count};
}

// row / group without a division: exact while row * group < 2^32 (rows are below 2^22, groups at most 16).
__device__ inline int paged_token(const PagedAttendArgs& a, int row) {
  return a.group_magic ? (int)__umulhi((uint32_t)row, a.group_magic) : row;
}

__device__ inline void paged_output_index(const PagedAttendArgs& a, int b, int h, int row, int64_t* out, int64_t* lse) {
  const int t = paged_token(a, row), g = row - t * a.group;
  const int64_t hq = (int64_t)h * a.group + g, heads = (int64_t)a.cache.kv_heads * a.group;
  *out = (((int64_t)b * a.tokens + t) * heads + hq) * D;
  *lse = ((int64_t)b * heads + hq) * a.tokens + t;
}

// Index of a query row's first element.
__device__ inline int64_t paged_query_index(const PagedAttendArgs& a, int b, int h, int row) {
  const int t = paged_token(a, row), g = row - t * a.group;
  return (int64_t)b * a.query.batch_stride + (int64_t)(h * a.group + g) * a.query.head_stride +
         (int64_t)t * a.query.token_stride;
}

// Pages of one (sequence, head): a page number, checked, and where its rows lie.
struct PagedHead {
  const uint16_t *keys, *values;
  const int32_t* table;
  uint32_t page_elems;  // of all heads: at most 2^30
  int pages, page_log2;
  __device__ PagedHead(const PagedAttendArgs& a, int b, int h)
      : keys(reinterpret_cast<const uint16_t*>(a.cache.key_pages) + ((int64_t)h << a.page_log2) * D),
        values(reinterpret_cast<const uint16_t*>(a.cache.value_pages) + ((int64_t)h << a.page_log2) * D),
        table(a.cache.page_table + (int64_t)b * a.cache.table_pages),
        page_elems(((uint32_t)a.cache.kv_heads << a.page_log2) * D), pages(a.cache.pages), page_log2(a.page_log2) {}
  __device__ int page(int row) const { return gload_i32(table + (row >> page_log2)); }
  // The same for a row that is the same in the whole wave: a scalar load (the table does not change during a call).
  __device__ int uniform_page(int row) const {
    typedef const __attribute__((address_space(4))) int32_t* constant_i32_ptr;
    return *(constant_i32_ptr)(uintptr_t)(table + (row >> page_log2));
  }
  __device__ bool good(int page) const { return (uint32_t)page < (uint32_t)pages; }
  // Element offset of a row; of some row where the page is none.
  __device__ int64_t at(int page, int row) const {
    return (int64_t)((uint64_t)(good(page) ? (uint32_t)page : 0u) * page_elems) + (row & ((1 << page_log2) - 1)) * D;
  }
};

// What one query row sees: positions from lo on in rows up to hi, and of a tree's rows (start and on) those of its mask,
// whose first word is kept (trees of up to 64 tokens have no other).  A committed row's position is its number, a draft
// row's goes by its depth alone, which may be less or more than its place in the draft.
struct Sight {
  int lo, hi, token;
  bool live;
  uint64_t kin0;
  Sight() = default;
  __device__ Sight(const PagedAttendArgs& a, const PagedStep& s, int b, int row) {
    token = min(paged_token(a, row), a.tokens - 1);
    live = row < a.rows && token < s.count;
    int position = s.start + token;
    kin0 = 0;
    if (a.masks) {
      const int64_t at = (int64_t)b * a.tokens + token;
      kin0 = a.masks[at * a.words];
      position = s.start + draft_depth(a.depths, at);
    }
    lo = a.window > 0 ? max(position - a.window + 1, 0) : 0;
    hi = min(a.masks ? s.total : s.start + token + 1, s.total) - 1;
    if (!live) hi = -1;
  }
  // Bit i: row `first` + i is seen, i below 64 (or as many as the caller reads).
  __device__ uint64_t rows(const PagedAttendArgs& a, const PagedStep& s, int b, int first) const {
    const int low = max((a.masks ? min(lo, s.start) : lo) - first, 0), high = min(hi - first, 63);
    if (high < low || low > 63) return 0;
    uint64_t seen = (~0ull >> (63 - high)) & (~0ull << low);
    if (a.masks && first + 63 >= s.start) {
      const int j = first - s.start;  // the draft's token in the first row
      uint64_t kin;
      if (j < 0) {
        kin = (kin0 << -j) | (~0ull >> (64 + j));  // -64 < j: rows before the draft are all there
      } else {
        const int w = j >> 6, shift = j & 63;
        kin = w == 0 ? kin0 >> shift : 0;
        if (a.words > 1) {
          const uint64_t* mask = a.masks + ((int64_t)b * a.tokens + token) * a.words;
          if (w && w < a.words) kin = mask[w] >> shift;
          if (shift && w + 1 < a.words) kin |= mask[w + 1] << (64 - shift);
        }
      }
      seen &= kin;
      if (lo > s.start) {  // draft rows out of the window
        uint64_t drafted = seen & (j < 0 ? ~0ull << -j : ~0ull);
        while (drafted) {
          const int i = __ffsll((unsigned long long)drafted) - 1;
          drafted &= drafted - 1;
          if (s.start + draft_depth(a.depths, (int64_t)b * a.tokens + j + i) < lo) seen &= ~(1ull << i);
        }
      }
    }
    return seen;
  }
};

// The natural log of a sum of probabilities 2^bias times as large, relative to the maximum m.
template <int DT>
__device__ inline float paged_lse(const PagedAttendArgs& a, float m, float sum) {
  return sum == 0.0f ? NEG_INF : (m * a.scale_log2 + (__log2f(sum) - prob_bias<DT>())) * PAGED_LN2;
}

// The first position that all of a wave's queries see in a window over a tree.
template <int N>
__device__ inline int wave_newest_lo(const Sight (&sight)[N]) {
  int most = 0;
#pragma unroll
  for (int r = 0; r < N; ++r) most = max(most, sight[r].live ? sight[r].lo : 0);
  most = max(most, (int)xor_u32<1>((uint32_t)most));
  most = max(most, (int)xor_u32<2>((uint32_t)most));
  most = max(most, (int)xor_u32<4>((uint32_t)most));
  most = max(most, (int)xor_u32<8>((uint32_t)most));
  most = max(most, (int)xor_u32<16>((uint32_t)most));
  return __builtin_amdgcn_readfirstlane(max(most, (int)xor_u32<32>((uint32_t)most)));
}

// Does a word hold a value that is not finite?
template <int DT>
__device__ inline bool has_special(uint32_t w) {
  constexpr uint32_t EXP = DT == CKV_BF16 ? 0x7f80u : 0x7c00u;
  return (w & EXP) == EXP || (w & (EXP << 16)) == EXP << 16;
}
// The word with its values that are not finite as zeros.
template <int DT>
__device__ inline uint32_t without_special(uint32_t w) {
  constexpr uint32_t EXP = DT == CKV_BF16 ? 0x7f80u : 0x7c00u;
  if ((w & EXP) == EXP) w &= 0xffff0000u;
  if ((w & (EXP << 16)) == EXP << 16) w &= 0xffffu;
  return w;
}
// The value of a half word where it is not finite, else 0.
template <int DT>
__device__ inline float special_value(uint32_t half_word) {
  constexpr uint32_t EXP = DT == CKV_BF16 ? 0x7f80u : 0x7c00u;
  return (half_word & EXP) == EXP ? low_value<DT>(half_word) : 0.0f;
}

template <int DT>
__device__ inline void store_value(void* base, int64_t index, float v) {
  if constexpr (DT == CKV_BF16) reinterpret_cast<uint16_t*>(base)[index] = ckv_f32_to_bf16_bits(v);
  else reinterpret_cast<_Float16*>(base)[index] = (_Float16)v;
}

// Host: the launcher of the many-row kernel (ckv_paged_rows.hip).
int paged_row_block(int rows);  // query rows of one workgroup
int launch_paged_rows(const PagedAttendArgs& a, hipStream_t stream);

}  // namespace ckv
