// Attention of many query rows (prompts, pieces of prompts, large trees) over
// the paged KV cache (gfx950).
//
// A workgroup of W waves takes 32 W packed query rows of a KV head (row = token *
// group + query head).  Tiles of 64 (or 32) cache rows come from memory into
// registers two tiles ahead, page by page, and are stored to LDS for the next
// tile.  Each wave computes S^T = K Q^T with the 32 x 32 x 16 matrix instructions,
// which leaves one query row in a lane (lane % 32) and 16 of 32 cache rows in each
// half of the wave, so the softmax is per-lane work; O^T = V^T P^T takes the same
// layout, with V^T by transposing LDS reads.  A tile that not every query of a wave
// sees whole is masked by a bit a row and lane.
//
// Bound by the matrix cores together with the softmax beside them: 2,048 queries
// over 32k rows (32/8 heads, bf16) take 971 to 1,015 us from card to card, 1,050 to
// 1,097 TFLOP/s, where a library product of 16,384^3 reaches 1,373 on the faster card.
// The products alone took 787 us and the softmax alone 615 before the last two steps;
// what the one does not hide of the other is the rest.  The matrix cores are busy 60 %
// of the cycles at the 1.75 to 1.85 GHz that the card keeps under this load.  8 trees of 64
// tokens over 4k to 16k rows each: 109 to 119 us, 2.7 to 3.0 TB/s; there each workgroup
// walks some 38 tiles of its own, 2 us each, and its first rows, its outputs and the
// join take a quarter of the time.
//
// Measured and not taken, for the 2,048 queries: matrix and vector work interleaved
// in every wave in place of the groups' turns (1,147 us); copies from memory into LDS
// past the registers, four stages deep (1,004 against 982; trees 130 against 121);
// row addresses on the vector ALUs (1,005); 64 query rows a wave at one wave a SIMD
// (spills).
#include <hip/hip_runtime.h>

#include "ckv_paged_attend.h"
#include "ckv_tile.h"

namespace {
using namespace ckv;

typedef float f32x16_t __attribute__((ext_vector_type(16)));

constexpr int K_STRIDE = D + 8;      // 17 chunks of 16 bytes: b128 reads of 16 lanes hit distinct banks
constexpr int V_STRIDE = D + 32;     // 20 chunks: transposed b64 reads hit distinct banks
constexpr int O_STRIDE = 64 + 4;     // floats of a row of 64 output dims: b128 writes of 16 rows hit distinct banks

template <int DT>
__device__ inline f32x16_t mfma32(uint4 a, uint4 b, f32x16_t c) {
  if constexpr (DT == CKV_BF16) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8_t, a), __builtin_bit_cast(bf16x8_t, b), c, 0, 0, 0);
  } else {
    typedef _Float16 f16x8_t __attribute__((ext_vector_type(8)));
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8_t, a), __builtin_bit_cast(f16x8_t, b), c, 0, 0, 0);
  }
}

// Largest of three without the moves that quiet a NaN first; a NaN operand is passed over.  The compiler keeps its own
// reads of a matrix product far enough behind it, but does not see those in inline assembly: `behind`, an unused operand,
// is the result of a read that it does see, of the products that these maxima are of.
__device__ inline float max3(float x, float y, float z, float behind) {
  float r;
  asm("v_max3_f32 %0, %1, %2, %3" : "=v"(r) : "v"(x), "v"(y), "v"(z), "v"(behind));
  return r;
}

// A thread's share of a tile of KEYS cache rows: piece i is 8 dims from 8 (tid % 16) on of local row
// tid / 16 + 4 W i.  A wave's four rows of a piece share a page, so pages and the addresses of their rows are the
// scalar unit's work: the vector ALUs have the softmax, and no time to spare.
template <int W, int KEYS>
struct TilePieces {
  static constexpr int C = KEYS / (4 * W);
  uint4 w[C];
};
template <int W, int KEYS>
struct TilePages {
  int32_t page[TilePieces<W, KEYS>::C];
};

template <int W, int KEYS>
__device__ inline void load_pages(const PagedHead& q, int wave, int tile, int last, TilePages<W, KEYS>& p) {
#pragma unroll
  for (int i = 0; i < TilePieces<W, KEYS>::C; ++i) p.page[i] = q.uniform_page(min(tile * KEYS + 4 * wave + i * 4 * W, last));
}

// Rows past the last one are read as they are in its page, and masked.
template <int W, int KEYS>
__device__ inline void load_tile(const PagedHead& q, const uint16_t* base, int wave, int tile, const TilePages<W, KEYS>& p,
                                 TilePieces<W, KEYS>& t) {
#pragma unroll
  for (int i = 0; i < TilePieces<W, KEYS>::C; ++i) {
    const uint16_t* row = base + q.at(p.page[i], tile * KEYS + 4 * wave + i * 4 * W);
    t.w[i] = gload16(row + (uint32_t)(((threadIdx.x & 63) >> 4) * D + 8 * (threadIdx.x & 15)));
  }
}

template <int W, int KEYS>
__device__ inline void store_tile(const TilePieces<W, KEYS>& t, uint16_t* tile, int stride) {
#pragma unroll
  for (int i = 0; i < TilePieces<W, KEYS>::C; ++i)
    *reinterpret_cast<uint4*>(tile + ((threadIdx.x >> 4) + i * 4 * W) * stride + 8 * (threadIdx.x & 15)) = t.w[i];
}

template <int KEYS>
struct TilesLds {
  alignas(16) uint16_t k[2][KEYS * K_STRIDE];
  alignas(16) uint16_t v[2][KEYS * V_STRIDE];
  int special[2];  // the tile, where its values held infinity or NaN that was staged as zero
  int newest_lo[8];  // of each wave's queries, with a window over a tree
};

// LDS of a workgroup: the tiles, or the output rows on their way out.
template <int W, int KEYS>
constexpr size_t rows_lds_bytes() {
  const size_t out = W * 32 * O_STRIDE * sizeof(float);
  return out > sizeof(TilesLds<KEYS>) ? out : sizeof(TilesLds<KEYS>);
}

// Rows that some of the query rows `first` to `first + rows` see, and those that all of them see (but for all_lo of a
// tree, where it goes by the depths).
__device__ inline void ranges_of(const PagedAttendArgs& a, const PagedStep& step, int first, int rows, int* some_lo,
                                 int* some_hi, int* all_lo, int* all_hi) {
  const int t0 = paged_token(a, first), t1 = min(paged_token(a, min(first + rows, a.rows) - 1), step.count - 1);
  const int last = step.total - 1;
  *some_lo = *all_lo = 0;
  *some_hi = -1;
  *all_hi = 0x7ffffffe;  // without a query nothing is masked: the rows are dropped at the end
  if (first >= a.rows || t0 > t1) return;
  *some_hi = min(step.start + (a.masks ? step.count - 1 : t1), last);
  *all_hi = min(a.masks ? step.start - 1 : step.start + t0, last);
  if (a.window > 0) {
    *some_lo = max(step.start + (a.masks ? 0 : t0) - a.window + 1, 0);
    if (!a.masks) *all_lo = max(step.start + t1 - a.window + 1, 0);
  }
}

// Zeros in place of the values that are not finite; whether there were any.
template <int DT, int W, int KEYS>
__device__ inline bool drop_special(TilePieces<W, KEYS>& t) {
  bool found = false;
#pragma unroll
  for (int i = 0; i < TilePieces<W, KEYS>::C; ++i) {
    uint4& w = t.w[i];
    found |= has_special<DT>(w.x) || has_special<DT>(w.y) || has_special<DT>(w.z) || has_special<DT>(w.w);
    w = uint4{without_special<DT>(w.x), without_special<DT>(w.y), without_special<DT>(w.z), without_special<DT>(w.w)};
  }
  return found;
}

// Results of 32 query rows from `row0` on, one a lane of each half: m the maximum of its unscaled scores, l the lane's
// share of the sum, o the outputs (o[i][v]: dim 32 i + 8 (v / 4) + 4 half + v % 4).  They go out through `out_s`, LDS of
// the wave alone, 64 dims at a time, so that whole lines are written: from the accumulators a store would touch 32 lines.
template <int DT>
__device__ inline void write_rows(const PagedAttendArgs& a, int b, int h, int slot, int row0, bool live, float m,
                                  float l, const f32x16_t* o, float* out_s) {
  const int lane = threadIdx.x & 63, half = lane >> 5, row = row0 + (lane & 31);
  const bool joined = slot >= 0;
  const float sum = live ? add_xor32(l) : 0.0f;
  const bool none = joined ? !live : sum == 0.0f;
  const float inv = sum == 0.0f ? 0.0f : 1.0f / sum, factor = joined ? 1.0f : inv;
#pragma unroll
  for (int dims = 0; dims < 2; ++dims) {
    asm volatile("" ::: "memory");
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const f32x16_t& x = o[2 * dims + (i >> 2)];
      const int g = i & 3;
      *reinterpret_cast<float4*>(&out_s[(lane & 31) * O_STRIDE + 32 * (i >> 2) + 8 * g + 4 * half]) =
          none ? float4{0.0f, 0.0f, 0.0f, 0.0f}
               : float4{x[4 * g] * factor, x[4 * g + 1] * factor, x[4 * g + 2] * factor, x[4 * g + 3] * factor};
    }
    asm volatile("" ::: "memory");  // a wave's own LDS operations stay in order
    if (joined) {
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const int local = 4 * j + (lane >> 4), r = row0 + local, dim = 64 * dims + 4 * (lane & 15);
        const float4 x = *reinterpret_cast<const float4*>(&out_s[local * O_STRIDE + 4 * (lane & 15)]);
        if (r < a.rows)
          *reinterpret_cast<float4*>(a.part_acc + (((int64_t)h * a.slots + slot) * a.row_pad + r) * D + dim) = x;
      }
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int local = 8 * j + (lane >> 3), r = row0 + local, dim = 64 * dims + 8 * (lane & 7);
        const float* from = &out_s[local * O_STRIDE + 8 * (lane & 7)];
        const float4 x = *reinterpret_cast<const float4*>(from), y = *reinterpret_cast<const float4*>(from + 4);
        if (r >= a.rows) continue;
        int64_t at_out, at_lse;
        paged_output_index(a, b, h, r, &at_out, &at_lse);
        *reinterpret_cast<uint4*>(reinterpret_cast<uint16_t*>(a.out) + at_out + dim) =
            uint4{pack_store<DT>(x.x, x.y), pack_store<DT>(x.z, x.w), pack_store<DT>(y.x, y.y), pack_store<DT>(y.z, y.w)};
      }
    }
  }
  if (half != 0 || row >= a.rows) return;
  if (joined) {
    a.part_max[((int64_t)h * a.row_pad + row) * a.slots + slot] = live ? m : NEG_INF;
    a.part_sum[((int64_t)h * a.row_pad + row) * a.slots + slot] = sum;
    return;
  }
  int64_t at_out, at_lse;
  paged_output_index(a, b, h, row, &at_out, &at_lse);
  a.lse[at_lse] = paged_lse<DT>(a, m, sum);
}

template <int DT, int W, int KEYS>
__global__ __launch_bounds__(64 * W, 2) void paged_rows_kernel(const PagedAttendArgs a) {
  extern __shared__ __align__(16) unsigned char lds_raw[];
  constexpr int NI = KEYS / 32;  // blocks of 32 cache rows a tile
  TilesLds<KEYS>& lds = *reinterpret_cast<TilesLds<KEYS>*>(lds_raw);
  const ckv_paged_cache& c = a.cache;
  // workgroups that follow one another go to different XCDs: one head's to one, where they share its L2
  const int h = blockIdx.x, number = blockIdx.z;
  // the blocks of the newest rows see the most: they go first
  const int block0 = (int)(gridDim.y - 1 - blockIdx.y) * 32 * W;
  const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63, half = lane >> 5;
  const Part part = find_part(PagedRows{a}, a.parts, number, -1);
  const int b = part.sequence;
  if (b < 0) return;
  tell_parts(a, part);
  const int slot = part_slot(part);
  const PagedStep step(a, b);
  const PagedHead q(a, b, h);
  const int row = block0 + 32 * wave + (lane & 31);
  const Sight see(a, step, b, row);
  const int last = step.total - 1;

  int walk_lo, walk_hi, group_lo, group_hi, wave_lo, wave_hi, unused;
  ranges_of(a, step, block0, 32 * W, &walk_lo, &walk_hi, &group_lo, &group_hi);
  ranges_of(a, step, block0 + 32 * wave, 32, &unused, &unused, &wave_lo, &wave_hi);
  // tiles of this part that are walked (its first row opens one)
  const int lo_row = step.first(a) + part.index * part.rows;
  const int hi_row = (int)min((int64_t)lo_row + part.rows, (int64_t)walk_hi + 1);
  const int first_tile = max(lo_row, walk_lo) / KEYS, end_tile = (hi_row + KEYS - 1) / KEYS;
  int left = walk_hi < 0 ? 0 : max(end_tile - first_tile, 0);

  // a page number that is none: every tile is then masked, page by page
  bool bad = false;
  if (left > 0) {
    const int low = first_tile * KEYS >> a.page_log2, high = min(end_tile * KEYS - 1, last) >> a.page_log2;
    for (int p = low + tid; p <= high; p += 64 * W) bad |= !q.good(gload_i32(q.table + p));
  }

  uint4 qreg[8];
  {
    const int64_t base = paged_query_index(a, b, h, min(row, a.rows - 1));
#pragma unroll
    for (int s = 0; s < 8; ++s)
      qreg[s] = gload16(reinterpret_cast<const uint16_t*>(a.query.data) + base + 16 * s + 8 * half);
  }

  const float sl2 = a.scale_log2;
  float m = NEG_INF;  // running maximum of the unscaled scores, shared by a row's two lanes
  float l = 0.0f;     // this lane's share of the sum
  // Of the maximum, as it last moved: the score that moves it, and the exponents, (score - base) * sl2 - mc.  The rounding
  // of the scaled maximum mc is a factor of all of a query's probabilities, 2^-14 away from one at most up to EXACT log2
  // units, and it saves a subtraction a score (base is 0).  Beyond, mc is 0, and differences are taken before they are
  // scaled.
  constexpr float EXACT = 1024.0f;
  float limit = NEG_INF, base = 0.0f, mc = -prob_bias<DT>();
  bool any_far = false;  // in the wave
  // S^T of a tile: accumulator i holds cache rows 32 i + 8 (v / 4) + 4 half + v % 4 of the lane's query
  f32x16_t o[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) o[i] = f32x16_t{};

  auto is_masked = [&](int tile, int all_lo, int all_hi) __attribute__((always_inline)) {
    return bad || tile * KEYS < all_lo || tile * KEYS + KEYS - 1 > all_hi;
  };
  // Which rows of a tile this lane's query sees, a bit each
  auto seen_rows = [&](int tile) {
    uint64_t seen = see.rows(a, step, b, tile * KEYS);
    if (bad) {
#pragma unroll
      for (int g = 0; g < KEYS / 16; ++g)
        if (!q.good(q.page(min(tile * KEYS + 16 * g, last)))) seen &= ~(0xffffull << (16 * g));
    }
    return seen;
  };
  TilePieces<W, KEYS> kc, vc;
  // Before a tile's values go to LDS: where some query does not see some row, values that are not finite become zeros
  // (a masked row's zero probability times infinity or NaN would spread it) and are added afterwards.
  auto prepare_values = [&](int tile, int stage) __attribute__((always_inline)) {
    if (!is_masked(tile, group_lo, group_hi)) return;
    asm volatile("");
    if (drop_special<DT>(vc)) lds.special[stage] = tile;
  };

  // Two groups of four waves, one of each on a SIMD, take turns: while one has
  // the matrix cores (M_i: O += V P of its tile i and the scores of tile i + 1) the
  // other has the vector ALUs (V_i: the softmax of its tile), and a barrier changes
  // them over.  The first group does V_i in slot 2 i and M_i in slot 2 i + 1, the
  // second each a slot later.  M_i reads X_i = {values of tile i, keys of tile
  // i + 1} from LDS and between its products stores X_(i + 1), which takes the
  // place of X_(i - 1), last read in slot 2 i.  One group alone (four waves) does
  // V_i, M_i and a barrier.  Past the last tile the pipeline stages that tile
  // again, unused.
  constexpr bool TURNS = W == 8;
  const bool second = TURNS && wave >= 4;
  const int last_tile = end_tile - 1;
  int t0 = first_tile;
  TilePages<W, KEYS> ahead;  // of tile i + 2, from V_i on of tile i + 3, whose keys are loaded in M_i
  int stage = 0;  // X_i has its values in v[i & 1], its keys in k[(i + 1) & 1]
  f32x16_t sc[NI];
  if (tid < 2) lds.special[tid] = -1;
  const bool tree_window = a.masks && a.window > 0;
  if (tree_window) {
    const Sight mine[1] = {see};
    wave_lo = wave_newest_lo(mine);
    if (lane == 0) lds.newest_lo[wave] = wave_lo;
  }
  TilePages<W, KEYS> p0, p1;
  const int t1 = min(t0 + 1, last_tile), t2 = min(t0 + 2, last_tile);
  if (left > 0) {
    load_pages<W, KEYS>(q, wave, t0, last, p0);
    load_pages<W, KEYS>(q, wave, t1, last, p1);
    load_pages<W, KEYS>(q, wave, t2, last, ahead);
    load_tile<W, KEYS>(q, q.keys, wave, t0, p0, kc);
    load_tile<W, KEYS>(q, q.values, wave, t0, p0, vc);
  }
  bad = __syncthreads_or(bad);  // with the first rows on their way
  if (tree_window) {
#pragma unroll
    for (int w = 0; w < W; ++w) group_lo = max(group_lo, __builtin_amdgcn_readfirstlane(lds.newest_lo[w]));
  }
  if (left > 0) {
    store_tile<W, KEYS>(kc, lds.k[0], K_STRIDE);
    load_tile<W, KEYS>(q, q.keys, wave, t1, p1, kc);
    prepare_values(t0, 0);
    store_tile<W, KEYS>(vc, lds.v[0], V_STRIDE);
    store_tile<W, KEYS>(kc, lds.k[1], K_STRIDE);
    load_tile<W, KEYS>(q, q.values, wave, t1, p1, vc);
    load_tile<W, KEYS>(q, q.keys, wave, t2, ahead, kc);
    __syncthreads();
#pragma unroll
    for (int k = 0; k < 8 * NI; ++k) {
      const int i = k % NI, x = k / NI;
      const uint4 kf = *reinterpret_cast<const uint4*>(&lds.k[0][(32 * i + (lane & 31)) * K_STRIDE + 16 * x + 8 * half]);
      sc[i] = mfma32<DT>(kf, qreg[x], x == 0 ? f32x16_t{} : sc[i]);
    }
    __syncthreads();  // k[0] is free
    if (second) __syncthreads();
  }

  uint32_t pb[NI][8];
  while (left > 0) {
    // ---- V_i: the vector ALUs ----
    const TilePages<W, KEYS> vpages = ahead;  // of tile i + 2, whose values are loaded in M_i
    load_pages<W, KEYS>(q, wave, min(t0 + 3, last_tile), last, ahead);  // by scalar loads: away from the LDS reads of M_i
    if (is_masked(t0, wave_lo, wave_hi)) {
      asm volatile("");  // a branch, not selects on every tile
      const uint64_t seen = seen_rows(t0) >> (4 * half);
#pragma unroll
      for (int i = 0; i < NI; ++i) {
        const uint32_t bits = (uint32_t)(seen >> (32 * i));
#pragma unroll
        for (int v = 0; v < 16; ++v) sc[i][v] = bits >> (8 * (v >> 2) + (v & 3)) & 1u ? sc[i][v] : NEG_INF;
      }
    }
    const float read = __builtin_amdgcn_fmed3f(sc[0][15], sc[NI - 1][15], 0.0f);
    float tops[2 * NI];
#pragma unroll
    for (int x = 0; x < 2 * NI; ++x) {
      const f32x16_t& v = sc[x >> 1];
      const int e = 8 * (x & 1);
      tops[x] = max3(max3(v[e], v[e + 1], v[e + 2], read), max3(v[e + 3], v[e + 4], v[e + 5], read),
                     max3(v[e + 6], v[e + 7], v[e + 7], read), read);
    }
    float all = tops[0];
#pragma unroll
    for (int x = 1; x < 2 * NI; ++x) all = max3(all, tops[x], tops[x], read);
    const float top = max_xor32(all);
    if (__ballot(top > limit) != 0) {
      const float t = top > limit ? top : m;  // a query's own scores alone decide
      const float f = m == t ? 1.0f : __builtin_amdgcn_exp2f((m - t) * sl2);
      m = t;
      l *= f;
#pragma unroll
      for (int i = 0; i < 4; ++i) o[i] *= f;
      mc = m == NEG_INF ? 0.0f : m * sl2;
      const bool far = !(fabsf(mc) <= EXACT);
      base = far ? m : 0.0f;  // the scores of the wave's other queries stay as they are
      mc = (far ? 0.0f : mc) - prob_bias<DT>();
      limit = far ? m : m + a.grow_by;  // far from 0 the sum is rounded by more than a probability may exceed its type
      any_far = __ballot(far) != 0;
    }
    if (any_far) {
      asm volatile("");
#pragma unroll
      for (int i = 0; i < NI; ++i) {
#pragma unroll
        for (int v = 0; v < 16; ++v) sc[i][v] -= base;
      }
    }
    float sums[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int i = 0; i < NI; ++i) {
#pragma unroll
      for (int v = 0; v < 16; v += 2) {
        const float p0 = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[i][v], sl2, -mc));
        const float p1 = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[i][v + 1], sl2, -mc));
        sums[v & 2] += p0;
        sums[(v & 2) + 1] += p1;
        pb[i][v >> 1] = pack_store<DT>(p0, p1);
        // in this slot: the compiler moves the exponentials behind the barrier otherwise
        if (TURNS) asm volatile("" : "+v"(pb[i][v >> 1]));
      }
    }
    l += (sums[0] + sums[1]) + (sums[2] + sums[3]);
    if (TURNS) asm volatile("" : "+v"(l));  // and the sums
    if (TURNS) __syncthreads();
    // ---- M_i: the matrix cores, and the staging of X_(i + 1) between the products ----
    if (TURNS) __builtin_amdgcn_s_setprio(1);
    const int t1 = min(t0 + 1, last_tile), t2 = min(t0 + 2, last_tile), t3 = min(t0 + 3, last_tile);
    // Operands from LDS are read AHEAD products before they are used: first those of
    // values (rows 16 (k / 4) of the tile, dims 32 (k % 4)), then as many of keys.
    constexpr int HALF = 8 * NI;
    const uint16_t* v_at = lds.v[stage] + (4 * half + ((lane & 15) >> 2)) * V_STRIDE + 16 * ((lane >> 4) & 1) +
                           4 * (lane & 3);
    const uint16_t* k_at = lds.k[stage ^ 1] + (lane & 31) * K_STRIDE + 8 * half;
    auto operand = [&](int k) __attribute__((always_inline)) {
      if (k < HALF) {
        const uint16_t* p = v_at + 16 * (k >> 2) * V_STRIDE + 32 * (k & 3);
        const uint2 x = lds_read_tr16(p), y = lds_read_tr16(p + 8 * V_STRIDE);
        return uint4{x.x, x.y, y.x, y.y};
      }
      return *reinterpret_cast<const uint4*>(k_at + 32 * ((k - HALF) % NI) * K_STRIDE + 16 * ((k - HALF) / NI));
    };
    constexpr int AHEAD = 3;  // 2,048 queries over 32k rows, one card: 1,004 us with 2, 1,003 with 3, 1,006 with 4, 1,016 with 6
    uint4 op[AHEAD];
#pragma unroll
    for (int k = 0; k < AHEAD; ++k) op[k] = operand(k);
    prepare_values(t1, stage ^ 1);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int k = 0; k < 2 * HALF; ++k) {
      const uint4 now = op[k % AHEAD];
      if (k < HALF) {
        const int i = k >> 3, vb = 4 * ((k >> 2) & 1), db = k & 3;
        o[db] = mfma32<DT>(now, uint4{pb[i][vb], pb[i][vb + 1], pb[i][vb + 2], pb[i][vb + 3]}, o[db]);
      } else {
        const int i = (k - HALF) % NI, x = (k - HALF) / NI;
        sc[i] = mfma32<DT>(now, qreg[x], x == 0 ? f32x16_t{} : sc[i]);
      }
      if (k + AHEAD < 2 * HALF) op[k % AHEAD] = operand(k + AHEAD);
      if (k == 2 * NI) store_tile<W, KEYS>(vc, lds.v[stage ^ 1], V_STRIDE);
      if (k == 5 * NI) store_tile<W, KEYS>(kc, lds.k[stage], K_STRIDE);
      if (k == 7 * NI) load_tile<W, KEYS>(q, q.values, wave, t2, vpages, vc);
      if (k == 9 * NI) load_tile<W, KEYS>(q, q.keys, wave, t3, ahead, kc);
      __builtin_amdgcn_sched_barrier(0);
    }
    if (TURNS) __builtin_amdgcn_s_setprio(0);
    if (is_masked(t0, group_lo, group_hi) && lds.special[stage] == t0) {
      asm volatile("");
      // values that were staged as zeros, added for the queries that see their row
      const uint64_t seen = seen_rows(t0);
#pragma nounroll
      for (int r = 0; r < KEYS; ++r) {
        const int at = t0 * KEYS + r;
        if (at > last) break;
        const uint16_t* value = q.values + q.at(q.page(at), at) + 4 * half;
        const bool sees = seen >> r & 1;
#pragma unroll
        for (int db = 0; db < 4; ++db) {
#pragma unroll
          for (int g = 0; g < 4; ++g) {
            const uint2 w = *reinterpret_cast<const uint2*>(value + 32 * db + 8 * g);
            if (!sees) continue;
            o[db][4 * g] += special_value<DT>(w.x & 0xffffu);
            o[db][4 * g + 1] += special_value<DT>(w.x >> 16);
            o[db][4 * g + 2] += special_value<DT>(w.y & 0xffffu);
            o[db][4 * g + 3] += special_value<DT>(w.y >> 16);
          }
        }
      }
    }
    __syncthreads();
    stage ^= 1;
    t0 = t1;
    --left;
    if (TURNS && !second && left == 0) __syncthreads();  // the second group's last slot
  }

  write_rows<DT>(a, b, h, slot, block0 + 32 * wave, see.live, m, l, o,
                 reinterpret_cast<float*>(lds_raw) + wave * 32 * O_STRIDE);
}

// Dynamic LDS of a kernel, set once a device; setting it twice does no harm.
template <class Kernel>
int launch_tiles(Kernel kernel, bool* ready, int rows, int threads, size_t lds, const PagedAttendArgs& a, hipStream_t s) {
  int device = 0;
  if (hipGetDevice(&device) != hipSuccess || device < 0 || device >= 64 || !ready[device]) {
    const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize,
                                             (int)lds);
    if (e != hipSuccess) {
      (void)hipGetLastError();
      return paged_error(CKV_E_LAUNCH, "ckv_paged_attention", hipGetErrorString(e));
    }
    if (device >= 0 && device < 64) ready[device] = true;
  }
  const dim3 grid(a.cache.kv_heads, (a.rows + rows - 1) / rows, a.parts);
  kernel<<<grid, threads, lds, s>>>(a);
  return paged_launched("ckv_paged_attention");
}

template <int DT>
int launch_rows(const PagedAttendArgs& a, hipStream_t s) {
  static bool small[64] = {}, large[64] = {};
  if (paged_row_block(a.rows) == 128)
    return launch_tiles(paged_rows_kernel<DT, 4, 32>, small, 128, 256, rows_lds_bytes<4, 32>(), a, s);
  return launch_tiles(paged_rows_kernel<DT, 8, 64>, large, 256, 512, rows_lds_bytes<8, 64>(), a, s);
}

}  // namespace

namespace ckv {

// 256 rows share what is read, 128 leave fewer of a small call's rows empty: 128 query rows of 8 sequences over 8k rows
// take 71 us with 128 and 81 with 256; 192 query rows of 4 sequences (16/2 heads) over 32k rows 63 and 53.
int paged_row_block(int rows) { return rows <= 128 ? 128 : 256; }

int launch_paged_rows(const PagedAttendArgs& a, hipStream_t stream) {
  return a.cache.dtype == CKV_BF16 ? launch_rows<CKV_BF16>(a, stream) : launch_rows<CKV_F16>(a, stream);
}

}  // namespace ckv
