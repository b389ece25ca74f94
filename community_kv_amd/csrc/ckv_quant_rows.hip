// Attention of many query rows (prompts and pieces of prompts) over the 8-bit
// KV cache, and the weight that every cache row received from them (gfx950).
//
// attend_rows_kernel: a workgroup of W waves takes 32 W packed query rows of a
// KV head (row = token * group + query head).  Tiles of 64 cache rows are
// converted once for the whole workgroup: codes come from memory into registers
// two tiles ahead, become bf16 with the block's power of two folded in (one
// v_cvt_scalef32_pk_bf16_fp8 a pair, exact), and are stored to LDS for the
// next tile.  Each wave computes S^T = K Q^T with v_mfma_f32_32x32x16_bf16, which
// leaves one query row in a lane (lane % 32) and 16 of 32 cache rows in each half of
// the wave, so the softmax is per-lane work; O^T = V^T P^T takes the same layout,
// with V^T by transposing LDS reads.  (P in one bf16 piece for bf16 queries, two for
// fp16, three for f32, as in the few-row kernel; its row sums before that rounding.)
//
// Tiles that no query of the workgroup sees are skipped by their least and
// largest position, which range_kernel writes beforehand; rows may stand in
// any order.
#include <hip/hip_runtime.h>

#include "ckv_quant_attend.h"

namespace {
using namespace ckv;

typedef float f32x16_t __attribute__((ext_vector_type(16)));

constexpr int KEYS = RANGE_TILE;     // cache rows of an LDS tile
constexpr int K_STRIDE = D + 8;      // 17 chunks of 16 bytes: b128 reads of 16 lanes hit distinct banks
constexpr int V_STRIDE = D + 32;     // 20 chunks: transposed b64 reads hit distinct banks
constexpr int K_TILE = KEYS * K_STRIDE;
constexpr int V_TILE = KEYS * V_STRIDE;

int launched(const char* what) {
  const hipError_t e = hipGetLastError();
  if (e == hipSuccess) return CKV_OK;
  static thread_local char message[160];
  snprintf(message, sizeof(message), "%s: %s", what, hipGetErrorString(e));
  return ckv_internal::set_error(CKV_E_LAUNCH, message);
}

__device__ inline f32x16_t mfma32(uint4 a, uint4 b, f32x16_t c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8_t, a), __builtin_bit_cast(bf16x8_t, b), c,
                                                 0, 0, 0);
}

// Largest of three without the moves that quiet a NaN first; a NaN operand is
// passed over.
__device__ inline float max3(float x, float y, float z) {
  float r;
  asm("v_max3_f32 %0, %1, %2, %3" : "=v"(r) : "v"(x), "v"(y), "v"(z));
  return r;
}

// Two codes as bf16 times the power of two in `scale`'s exponent (exact).
template <bool HIGH>
__device__ inline uint32_t scaled_codes(uint32_t w, float scale) {
  typedef __bf16 bf16x2_t __attribute__((ext_vector_type(2)));
  return __builtin_bit_cast(uint32_t, (bf16x2_t)__builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, scale, HIGH));
}

__device__ inline uint4 scaled_codes8(uint32_t lo, uint32_t hi, float scale) {
  return uint4{scaled_codes<false>(lo, scale), scaled_codes<true>(lo, scale), scaled_codes<false>(hi, scale),
               scaled_codes<true>(hi, scale)};
}

// Which positions a query sees: p is one where (uint32_t)(p - lo) <= span.  No
// position is negative or 2^31 - 1, so a query that sees none has lo -2, span 0.
struct Seen {
  int lo;
  uint32_t span;
  __device__ Seen(int low, int high) : lo(high < low ? -2 : low), span(high < low ? 0u : (uint32_t)(high - low)) {}
  // x, or -inf where position p is not seen.  One block of two instructions:
  // apart, the compiler collects the 32 compares of a tile first and spills them.
  __device__ void mask(float& x, int p) const {
    asm("v_cmp_gt_u32 vcc, %1, %2\n\tv_cndmask_b32 %0, %0, %3, vcc"
        : "+v"(x)
        : "v"((uint32_t)(p - lo)), "v"(span), "v"(NEG_INF)
        : "vcc");
  }
};

// Least and largest position of every 64 rows in use.
__global__ __launch_bounds__(256) void range_kernel(const QuantAttendArgs a) {
  const ckv_quant_cache& c = a.cache;
  const int h = blockIdx.y, b = blockIdx.z, lane = threadIdx.x & 63;
  const int n = quant_length(c, b);
  const int64_t tile = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (tile * KEYS >= n) return;
  const int64_t row = tile * KEYS + lane;
  const int32_t p = quant_head(c, b, h).positions[min(row, (int64_t)n - 1)];
  const int top = wave_max_i32(p), low = -wave_max_i32(-p);
  const int64_t tiles = (c.capacity + KEYS - 1) / KEYS;
  if (lane == 0) a.ranges[((int64_t)b * c.kv_heads + h) * tiles + tile] = int2{low, top};
}

struct TileRef {
  int tile, lo, hi;  // -1: none; its least and largest position
};

// Goes over the tiles of [first, last) that hold a position in [lo, hi], in
// order; every wave of a workgroup sees the same.
struct TileWalk {
  const int2* ranges;
  int base, last, lo, hi;
  uint64_t bits;
  int2 mine;
  __device__ TileWalk(const int2* r, int first, int end, int low, int high)
      : ranges(r), base(first - 64), last(end), lo(low), hi(high), bits(0) {}
  __device__ TileRef next() {
    while (bits == 0) {
      base += 64;
      if (base >= last) return TileRef{-1, 0, 0};
      const int t = base + (int)(threadIdx.x & 63);
      bool need = false;
      if (t < last) {
        mine = ranges[t];
        need = mine.x <= hi && mine.y >= lo;
      }
      bits = __ballot(need);
    }
    const int i = __ffsll((unsigned long long)bits) - 1;
    bits &= bits - 1;
    return TileRef{base + i, __builtin_amdgcn_readlane(mine.x, i), __builtin_amdgcn_readlane(mine.y, i)};
  }
};

// A thread's share of a tile's codes: piece i is 16 codes of local row
// tid / 8 + 8 W i, from 16 (tid % 8) on, with its block's scale.
template <int W>
struct TileCodes {
  static constexpr int C = 8 / W;
  uint4 w[C];
  float scale[C];
};

template <int W>
__device__ inline void load_codes(const uint8_t* codes, const float* scales, int tile, int n, int block_log2,
                                  TileCodes<W>& t) {
  const int first = tile * KEYS;
  const int last = min(n - 1 - first, KEYS - 1);  // rows past the last one repeat it
  const uint8_t* base = codes + (int64_t)first * D;
  const float* scale = scales + (first >> block_log2);
#pragma unroll
  for (int i = 0; i < TileCodes<W>::C; ++i) {
    const int local = min((int)(threadIdx.x >> 3) + i * 8 * W, last);
    t.w[i] = gload16(base + local * D + 16 * (threadIdx.x & 7));
    t.scale[i] = gload_f32(scale + (local >> block_log2));  // a tile's first row opens a block, or halves one of 128
  }
}

template <int W>
__device__ inline void store_codes(const TileCodes<W>& t, uint16_t* tile, int stride) {
#pragma unroll
  for (int i = 0; i < TileCodes<W>::C; ++i) {
    uint4* p = reinterpret_cast<uint4*>(tile + ((threadIdx.x >> 3) + i * 8 * W) * stride + 16 * (threadIdx.x & 7));
    p[0] = scaled_codes8(t.w[i].x, t.w[i].y, t.scale[i]);
    p[1] = scaled_codes8(t.w[i].z, t.w[i].w, t.scale[i]);
  }
}

// Zeros in place of NaN codes; whether there were any.
__device__ inline bool drop_nan_codes(uint32_t& w) {
  const uint32_t is = ((w & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u;
  w &= ~((is >> 7) * 0xffu);
  return is != 0;
}

constexpr int O_STRIDE = 64 + 4;     // floats of a row of 64 output dims: b128 writes of 16 rows hit distinct banks

struct RowsLds {
  alignas(16) uint16_t k[2][K_TILE];
  alignas(16) uint16_t v[2][V_TILE];
  alignas(16) int32_t pos[2][KEYS];
  int nan[2];  // the tile, where its values held a NaN code that was staged as zero
};

static_assert(8 * 32 * O_STRIDE * sizeof(float) <= sizeof(RowsLds), "eight waves' output fits");

template <int DT, int W>
__global__ __launch_bounds__(64 * W) void attend_rows_kernel(const QuantAttendArgs a) {
  constexpr int NP = pieces(DT);
  extern __shared__ __align__(16) unsigned char lds_raw[];
  RowsLds& lds = *reinterpret_cast<RowsLds*>(lds_raw);
  const ckv_quant_cache& c = a.cache;
  // workgroups that follow one another go to different XCDs: one head's to one, where they share its L2
  const int h = blockIdx.x, number = blockIdx.z;
  // the blocks of the newest rows see the most: they go first
  const int block0 = (int)(gridDim.y - 1 - blockIdx.y) * 32 * W;
  const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63, half = lane >> 5;
  const Part part = find_part(c, a.parts, number, -1);
  const int b = part.sequence;
  if (b < 0) return;
  const int64_t bh = (int64_t)b * c.kv_heads + h;
  const int n = quant_length(c, b), seen = c.cursors[c.batch + b], count = new_count(a, b);
  const int lo_row = part.index * part.rows, hi_row = (int)min((int64_t)lo_row + part.rows, (int64_t)n);
  const QuantHead q = quant_head(c, b, h);
  const int block_log2 = 31 - __clz(c.block);
  const int row = block0 + 32 * wave + (lane & 31);
  int lo, hi;
  query_range(a, row, count, seen, &lo, &hi);
  const Seen see(lo, hi);
  // Positions that the queries t0 .. t1 see: some of them [some_lo, some_hi], all of them [all_lo, all_hi].
  auto ranges_of = [&](int first, int rows, int* some_lo, int* some_hi, int* all_lo, int* all_hi) {
    const int t0 = token_of(a, first), t1 = min(token_of(a, min(first + rows, a.rows) - 1), count - 1);
    *some_lo = *all_lo = 0;
    *some_hi = -1;
    *all_hi = 0x7ffffffe;  // without a query nothing is masked: the rows are dropped at the end
    if (t0 > t1) return;
    query_range(a, t0 * a.group, count, seen, some_lo, all_hi);
    query_range(a, t1 * a.group, count, seen, all_lo, some_hi);
  };
  int walk_lo, walk_hi, group_lo, group_hi, wave_lo, wave_hi, unused;
  ranges_of(block0, 32 * W, &walk_lo, &walk_hi, &group_lo, &group_hi);
  ranges_of(block0 + 32 * wave, 32, &unused, &unused, &wave_lo, &wave_hi);

  uint4 qreg[NP][8];
  {
    const int qrow = min(row, a.rows - 1);
    const int t = token_of(a, qrow), g = qrow - t * a.group;
    const int64_t base = (int64_t)b * a.query.batch_stride + (int64_t)(h * a.group + g) * a.query.head_stride +
                         (int64_t)t * a.query.token_stride;
#pragma unroll
    for (int s = 0; s < 8; ++s) {
      if constexpr (DT == CKV_BF16) {
        qreg[0][s] = gload16(reinterpret_cast<const uint16_t*>(a.query.data) + base + 16 * s + 8 * half);
      } else {
        float v[8];
        load_query8<DT>(a.query.data, base + 16 * s + 8 * half, v);
        uint32_t w[NP * 4];
#pragma unroll
        for (int i = 0; i < 4; ++i) split_pair<NP>(v[2 * i], v[2 * i + 1], w + i, 4);
#pragma unroll
        for (int p = 0; p < NP; ++p) qreg[p][s] = uint4{w[4 * p], w[4 * p + 1], w[4 * p + 2], w[4 * p + 3]};
      }
    }
  }

  const float sl2 = a.scale_log2;
  const float grow_by = RESCALE / sl2;
  float m = NEG_INF;  // running maximum of the unscaled scores, shared by a row's two lanes
  float l = 0.0f;     // this lane's share of the sum
  // S^T of a tile: accumulator i holds cache rows 32 i + 8 (v / 4) + 4 half + v % 4 of the lane's query
  f32x16_t o[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) o[i] = f32x16_t{};

  auto is_masked = [&](const TileRef& t, int all_lo, int all_hi) __attribute__((always_inline)) {
    return t.lo < all_lo || t.hi > all_hi || (t.tile + 1) * KEYS > n;
  };
  TileCodes<W> kc, vc;
  // Before a tile's values go to LDS: where some query does not see some row, NaN
  // codes become zeros (a masked row's zero probability times NaN would spread it)
  // and are made up for afterwards, and the positions are staged.
  auto prepare_values = [&](const TileRef& t, int stage) __attribute__((always_inline)) {
    if (!is_masked(t, group_lo, group_hi)) return;
    asm volatile("");
    bool nan = false;
#pragma unroll
    for (int i = 0; i < TileCodes<W>::C; ++i) {
      nan |= drop_nan_codes(vc.w[i].x);
      nan |= drop_nan_codes(vc.w[i].y);
      nan |= drop_nan_codes(vc.w[i].z);
      nan |= drop_nan_codes(vc.w[i].w);
    }
    if (nan) lds.nan[stage] = t.tile;
    if (tid < KEYS) {
      const int r = t.tile * KEYS + tid;
      lds.pos[stage][tid] = r < n ? gload_i32(q.positions + r) : 0x7fffffff;
    }
  };
  auto load_keys = [&](const TileRef& t) __attribute__((always_inline)) {
    load_codes<W>(q.key_codes, q.key_scales, t.tile, n, block_log2, kc);
  };
  auto load_values = [&](const TileRef& t) __attribute__((always_inline)) {
    load_codes<W>(q.value_codes, q.value_scales, t.tile, n, block_log2, vc);
  };

  // Two groups of four waves, one of each on a SIMD, take turns: while one has
  // the matrix cores (M_i: O += V P of its tile i and the scores of tile i + 1) the
  // other has the vector ALUs (V_i: the softmax of its tile), and a barrier changes
  // them over.  The first group does V_i in slot 2 i and M_i in slot 2 i + 1, the
  // second each a slot later.  M_i reads X_i = {values of tile i, keys of tile
  // i + 1} from LDS and between its products stores X_(i + 1), which takes the
  // place of X_(i - 1), last read in slot 2 i.  (The positions that masks need
  // are staged by the first group, a slot before it needs them.)  One group alone
  // (four waves) does V_i, M_i and a barrier.  Past the last tile the pipeline
  // stages that tile again, unused.  2,048 queries over 32k rows (32/8 heads,
  // bf16): 1.00 to 1.06 ms, 1,010 to 1,070 TFLOP/s; without turns 1.03 to 1.12.
  // What is left is the matrix cores' own rate: with neither staging nor
  // exponentials the loop takes 0.92 ms, and a large library product runs at
  // 1,300 TFLOP/s on this card.
  constexpr bool TURNS = W == 8;
  const bool second = TURNS && wave >= 4;
  const int64_t tiles = (c.capacity + KEYS - 1) / KEYS;
  TileWalk walk(a.ranges + bh * tiles, lo_row / KEYS, (int)(((int64_t)hi_row + KEYS - 1) / KEYS), walk_lo, walk_hi);
  int left = 0;  // of t0, t1, t2, t3: tiles that there are
  auto advance = [&](const TileRef& after) __attribute__((always_inline)) {
    const TileRef t = walk.next();
    if (t.tile < 0) return after;
    ++left;
    return t;
  };
  TileRef t0 = advance(TileRef{-1, 0, 0});
  TileRef t1 = advance(t0), t2 = advance(t1);
  int stage = 0;  // X_i has its values in v[i & 1], its keys in k[(i + 1) & 1]
  f32x16_t sc[2];
  if (tid < 2) lds.nan[tid] = -1;
  __syncthreads();
  if (left > 0) {
    load_keys(t0);
    store_codes<W>(kc, lds.k[0], K_STRIDE);
    load_values(t0);
    load_keys(t1);
    prepare_values(t0, 0);
    store_codes<W>(vc, lds.v[0], V_STRIDE);
    store_codes<W>(kc, lds.k[1], K_STRIDE);
    load_values(t1);
    load_keys(t2);
    __syncthreads();
#pragma unroll
    for (int k = 0; k < 16; ++k) {
      const int i = k & 1, x = k >> 1;
      const uint4 kf = *reinterpret_cast<const uint4*>(&lds.k[0][(32 * i + (lane & 31)) * K_STRIDE + 16 * x + 8 * half]);
#pragma unroll
      for (int p = 0; p < NP; ++p) sc[i] = mfma32(kf, qreg[p][x], x == 0 && p == 0 ? f32x16_t{} : sc[i]);
    }
    __syncthreads();  // k[0] is free
    if (second) __syncthreads();
  }

  uint32_t pb[NP][2][8];
  while (left > 0) {
    // ---- V_i: the vector ALUs ----
    if (is_masked(t0, wave_lo, wave_hi)) {
      asm volatile("");  // a branch, not selects on every tile
#pragma unroll
      for (int i = 0; i < 2; ++i) {
#pragma unroll
        for (int g = 0; g < 4; ++g) {
          const int4 p = *reinterpret_cast<const int4*>(&lds.pos[stage][32 * i + 8 * g + 4 * half]);
          const int at[4] = {p.x, p.y, p.z, p.w};
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            float x = sc[i][4 * g + e];
            see.mask(x, at[e]);
            sc[i][4 * g + e] = x;
          }
        }
      }
    }
    float tops[4];
#pragma unroll
    for (int x = 0; x < 4; ++x) {
      const f32x16_t& v = sc[x >> 1];
      const int e = 8 * (x & 1);
      tops[x] = max3(max3(v[e], v[e + 1], v[e + 2]), max3(v[e + 3], v[e + 4], v[e + 5]), max3(v[e + 6], v[e + 7], v[e + 7]));
    }
    const float top = max_xor32(max3(max3(tops[0], tops[1], tops[2]), tops[3], tops[3]));
    if (__ballot(top > m + grow_by) != 0) {
      const float t = top > m + grow_by ? top : m;  // a query's own scores alone decide
      const float f = m == t ? 1.0f : __builtin_amdgcn_exp2f((m - t) * sl2);
      m = t;
      l *= f;
#pragma unroll
      for (int i = 0; i < 4; ++i) o[i] *= f;
    }
    const float mc = m == NEG_INF ? 0.0f : m * sl2;
    float sums[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int i = 0; i < 2; ++i) {
#pragma unroll
      for (int v = 0; v < 16; v += 2) {
        const float p0 = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[i][v], sl2, -mc));
        const float p1 = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[i][v + 1], sl2, -mc));
        sums[v & 2] += p0;
        sums[(v & 2) + 1] += p1;
        split_pair<NP>(p0, p1, &pb[0][i][v >> 1], 16);
        // in this slot: the compiler moves the exponentials behind the barrier otherwise
#pragma unroll
        for (int p = 0; TURNS && p < NP; ++p) asm volatile("" : "+v"(pb[p][i][v >> 1]));
      }
    }
    l += (sums[0] + sums[1]) + (sums[2] + sums[3]);
    if (TURNS) __syncthreads();
    // ---- M_i: the matrix cores, and the staging of X_(i + 1) between the products ----
    if (TURNS) __builtin_amdgcn_s_setprio(1);
    const TileRef t3 = advance(t2);
    // Operands from LDS are read AHEAD products before they are used: 16 of
    // values (rows 16 (k / 4) of the tile, dims 32 (k % 4)), then 16 of keys.
    const uint16_t* v_at = lds.v[stage] + (4 * half + ((lane & 15) >> 2)) * V_STRIDE + 16 * ((lane >> 4) & 1) +
                           4 * (lane & 3);
    const uint16_t* k_at = lds.k[stage ^ 1] + (lane & 31) * K_STRIDE + 8 * half;
    auto operand = [&](int k) __attribute__((always_inline)) {
      if (k < 16) {
        const uint16_t* p = v_at + 16 * (k >> 2) * V_STRIDE + 32 * (k & 3);
        const uint2 x = lds_read_tr16(p), y = lds_read_tr16(p + 8 * V_STRIDE);
        return uint4{x.x, x.y, y.x, y.y};
      }
      return *reinterpret_cast<const uint4*>(k_at + 32 * (k & 1) * K_STRIDE + 16 * ((k - 16) >> 1));
    };
    constexpr int AHEAD = 6;
    uint4 op[AHEAD];
#pragma unroll
    for (int k = 0; k < AHEAD; ++k) op[k] = operand(k);
    prepare_values(t1, stage ^ 1);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int k = 0; k < 32; ++k) {
      const uint4 now = op[k % AHEAD];
      if (k < 16) {
        const int i = k >> 3, vb = 4 * ((k >> 2) & 1), db = k & 3;
#pragma unroll
        for (int p = 0; p < NP; ++p)
          o[db] = mfma32(now, uint4{pb[p][i][vb], pb[p][i][vb + 1], pb[p][i][vb + 2], pb[p][i][vb + 3]}, o[db]);
      } else {
        const int i = k & 1, x = (k - 16) >> 1;
#pragma unroll
        for (int p = 0; p < NP; ++p) sc[i] = mfma32(now, qreg[p][x], k < 18 && p == 0 ? f32x16_t{} : sc[i]);
      }
      if (k + AHEAD < 32) op[k % AHEAD] = operand(k + AHEAD);
      if (k == 4) store_codes<W>(vc, lds.v[stage ^ 1], V_STRIDE);
      if (k == 10) store_codes<W>(kc, lds.k[stage], K_STRIDE);
      if (k == 14) load_values(t2);
      if (k == 18) load_keys(t3);
      __builtin_amdgcn_sched_barrier(0);
    }
    if (TURNS) __builtin_amdgcn_s_setprio(0);
    if (is_masked(t0, group_lo, group_hi) && lds.nan[stage] == t0.tile) {
      asm volatile("");
      // NaN codes that were staged as zeros: NaN where a query sees their row
#pragma nounroll
      for (int r = 0; r < KEYS; ++r) {
        if (t0.tile * KEYS + r >= n) break;
        const bool sees = (uint32_t)(lds.pos[stage][r] - see.lo) <= see.span;
        const uint8_t* code = q.value_codes + (int64_t)(t0.tile * KEYS + r) * D + 4 * half;
#pragma unroll
        for (int db = 0; db < 4; ++db) {
#pragma unroll
          for (int g = 0; g < 4; ++g) {
            const uint32_t w = *reinterpret_cast<const uint32_t*>(code + 32 * db + 8 * g);
#pragma unroll
            for (int e = 0; e < 4; ++e)
              if (sees && ((w >> (8 * e)) & 0x7fu) == 0x7fu) o[db][4 * g + e] = __builtin_nanf("");
          }
        }
      }
    }
    __syncthreads();
    stage ^= 1;
    t0 = t1;
    t1 = t2;
    t2 = t3;
    --left;
    if (TURNS && !second && left == 0) __syncthreads();  // the second group's last slot
  }

  // The wave's rows go out through LDS (free by now), 64 dims at a time, so that
  // whole lines are written: from the accumulators a store would touch 32 lines.
  const float sum = hi < 0 ? 0.0f : add_xor32(l);
  const float top = m == NEG_INF ? 0.0f : m * sl2;
  const bool joined = part.count > 1, none = joined ? hi < 0 : sum == 0.0f;
  const float inv = sum == 0.0f ? 0.0f : 1.0f / sum, factor = joined ? 1.0f : inv;
  float* out_s = reinterpret_cast<float*>(lds_raw) + wave * 32 * O_STRIDE;
  const int wave0 = block0 + 32 * wave;
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
    if (joined || DT == CKV_F32) {
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const int local = 4 * j + (lane >> 4), r = wave0 + local, dim = 64 * dims + 4 * (lane & 15);
        const float4 x = *reinterpret_cast<const float4*>(&out_s[local * O_STRIDE + 4 * (lane & 15)]);
        if (r >= a.rows) continue;
        if (joined) {
          *reinterpret_cast<float4*>(a.part_acc + (((int64_t)h * a.parts + number) * a.row_pad + r) * D + dim) = x;
        } else {
          int64_t at_out, at_lse;
          output_index(a, b, h, r, &at_out, &at_lse);
          *reinterpret_cast<float4*>(reinterpret_cast<float*>(a.out) + at_out + dim) = x;
        }
      }
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int local = 8 * j + (lane >> 3), r = wave0 + local, dim = 64 * dims + 8 * (lane & 7);
        const float* from = &out_s[local * O_STRIDE + 8 * (lane & 7)];
        const float4 x = *reinterpret_cast<const float4*>(from), y = *reinterpret_cast<const float4*>(from + 4);
        const float v[8] = {x.x, x.y, x.z, x.w, y.x, y.y, y.z, y.w};
        uint32_t w[4];
#pragma unroll
        for (int e = 0; e < 4; ++e)
          w[e] = DT == CKV_BF16 ? pack_bf16x2_hw(v[2 * e], v[2 * e + 1])
                                : (uint32_t)f16_bits_hw(v[2 * e]) | ((uint32_t)f16_bits_hw(v[2 * e + 1]) << 16);
        if (r >= a.rows) continue;
        int64_t at_out, at_lse;
        output_index(a, b, h, r, &at_out, &at_lse);
        *reinterpret_cast<uint4*>(reinterpret_cast<uint16_t*>(a.out) + at_out + dim) = uint4{w[0], w[1], w[2], w[3]};
      }
    }
  }
  if (half != 0 || row >= a.rows) return;
  if (joined) {
    a.part_max[((int64_t)h * a.row_pad + row) * a.parts + number] = m == NEG_INF || hi < 0 ? NEG_INF : top;
    a.part_sum[((int64_t)h * a.row_pad + row) * a.parts + number] = sum;
    return;
  }
  int64_t at_out, at_lse;
  output_index(a, b, h, row, &at_out, &at_lse);
  a.lse[at_lse] = sum == 0.0f ? NEG_INF : (top + __log2f(sum)) * LN2;
  if (a.stats) a.stats[(int64_t)bh * a.row_pad + row] = float2{top, inv};
}

template <int DT>
constexpr int rows_waves() { return DT == CKV_BF16 ? 8 : 4; }

template <int DT>
int launch_rows(const QuantAttendArgs& a, hipStream_t s) {
  constexpr int W = rows_waves<DT>();
  const ckv_quant_cache& c = a.cache;
  const int64_t tiles = (c.capacity + KEYS - 1) / KEYS;
  range_kernel<<<dim3((uint32_t)((tiles + 3) / 4), c.kv_heads, c.batch), 256, 0, s>>>(a);
  int rc = launched("ckv_quant_attention");
  if (rc) return rc;
  auto kernel = attend_rows_kernel<DT, W>;
  static bool ready[64] = {};  // one flag a device; setting it twice does no harm
  int device = 0;
  if (hipGetDevice(&device) != hipSuccess || device < 0 || device >= 64 || !ready[device]) {
    const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(kernel),
                                             hipFuncAttributeMaxDynamicSharedMemorySize, (int)sizeof(RowsLds));
    if (e != hipSuccess) {
      (void)hipGetLastError();
      return ckv_internal::set_error(CKV_E_LAUNCH, hipGetErrorString(e));
    }
    if (device >= 0 && device < 64) ready[device] = true;
  }
  const dim3 grid(c.kv_heads, (a.rows + 32 * W - 1) / (32 * W), a.parts);
  kernel<<<grid, 64 * W, sizeof(RowsLds), s>>>(a);
  return launched("ckv_quant_attention");
}

// Received weight.  A wave keeps 32 cache rows as A operands in registers; the
// workgroup's eight waves (256 cache rows) go over the query rows, 64 a step,
// staged in LDS a step ahead.  With the scores' layout as above a lane adds up
// what its cache rows got from the queries lane % 32; the lanes are added once
// at the end.  The steps are shared out over `shares` workgroups a block of cache
// rows, which leave sums of their own for weights_add_kernel: one owner a sum
// and a fixed order, no atomics.  Four small waves a SIMD overlap one's products
// with another's exponentials: the counters show the matrix cores busy half of
// the time and the vector ALUs 70 %.  2,048 queries over 32k rows (32/8 heads)
// take 582 us; interleaving the two within a wave, half a step apart, took 612,
// waves of 64 rows, two a SIMD, 10 % more.
constexpr int WT_WAVES = 8;
constexpr int WT_ROWS = 64;   // query rows of a step
constexpr int WT_KEYS = WT_WAVES * 32;

template <int NP>
struct WeightsLds {
  alignas(16) uint16_t q[2][NP][WT_ROWS * K_STRIDE];
  float2 stats[2][WT_ROWS];
  alignas(16) int32_t pos[WT_KEYS];
};

template <int DT>
__global__ __launch_bounds__(64 * WT_WAVES, DT == CKV_F32 ? 2 : 4) void rows_weights_kernel(const QuantAttendArgs a,
                                                                                          const int shares) {
  constexpr int NP = pieces(DT);
  __shared__ __align__(16) WeightsLds<NP> lds;
  const ckv_quant_cache& c = a.cache;
  // (head, share, block): the blocks of the oldest rows meet the most queries and go first
  const uint32_t heads = (uint32_t)c.batch * c.kv_heads, rest = blockIdx.x / heads;
  const int bh = (int)(blockIdx.x - rest * heads), share = (int)(rest % (uint32_t)shares);
  const int b = bh / c.kv_heads, h = bh % c.kv_heads;
  const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63;
  const int half = lane >> 5;
  const int n = quant_length(c, b), seen = c.cursors[c.batch + b], count = new_count(a, b);
  const int64_t first_row = (int64_t)(rest / (uint32_t)shares) * WT_KEYS;
  if (first_row >= n) return;
  const int64_t tiles = (c.capacity + KEYS - 1) / KEYS;
  const int live_tiles = (n + KEYS - 1) / KEYS, tile0 = (int)(first_row / KEYS);
  const QuantHead q = quant_head(c, b, h);
  const int block_log2 = 31 - __clz(c.block);
  const int row0 = (int)first_row + 32 * wave;
  const bool full = row0 + 32 <= n;
  // least and largest position of the tile that this wave's rows lie in, and of the workgroup's
  int2 range{0x7fffffff, -1}, all{0x7fffffff, -1};
#pragma unroll
  for (int t = 0; t < WT_KEYS / KEYS; ++t) {
    if (tile0 + t >= live_tiles) break;
    const int2 r = a.ranges[(int64_t)bh * tiles + tile0 + t];
    if (t == wave >> 1) range = r;
    all.x = min(all.x, r.x);
    all.y = max(all.y, r.y);
  }
  if (tid < WT_KEYS) {
    const int64_t r = first_row + tid;
    lds.pos[tid] = r < n ? gload_i32(q.positions + r) : 0x7fffffff;  // nobody sees rows past the last
  }
  uint4 kop[8];
  {
    const int r = min(row0 + (lane & 31), n - 1);
    const float scale = gload_f32(q.key_scales + (r >> block_log2));
#pragma unroll
    for (int s = 0; s < 8; ++s) {
      const uint2 w = *reinterpret_cast<const uint2*>(q.key_codes + (int64_t)r * D + 16 * s + 8 * half);
      kop[s] = scaled_codes8(w.x, w.y, scale);
    }
  }
  // steps whose queries t see any of the rows: seen - count + t >= least position, and > largest - window
  const int steps = (a.rows + WT_ROWS - 1) / WT_ROWS;
  const int64_t first_at = (int64_t)seen - count;
  const int64_t t_lo = max((int64_t)all.x - first_at, (int64_t)0);
  int64_t t_hi = (int64_t)count - 1;
  if (a.window > 0) t_hi = min(t_hi, (int64_t)all.y + a.window - 1 - first_at);
  const int step_lo = (int)min(t_lo * a.group / WT_ROWS, (int64_t)steps);
  const int step_hi = t_hi < 0 ? 0 : (int)min((t_hi * a.group + a.group - 1) / WT_ROWS + 1, (int64_t)steps);
  const float sl2 = a.scale_log2;
  const float2* stats = a.stats + (int64_t)bh * a.row_pad;
  // a thread stages 16 dims of query row tid / 8 of a step, as they are in memory
  const int qd = 16 * (tid & 7), qr = tid >> 3;
  constexpr int RAW = DT == CKV_F32 ? 4 : 2;  // 16-byte pieces
  uint4 raw[RAW];
  float2 next_st{0.0f, 0.0f};
  auto load = [&](int step) __attribute__((always_inline)) {
    const int row = min(step * WT_ROWS + qr, a.rows - 1);
    const int t = token_of(a, row), g = row - t * a.group;
    const int64_t base = (int64_t)b * a.query.batch_stride + (int64_t)(h * a.group + g) * a.query.head_stride +
                         (int64_t)t * a.query.token_stride + qd;
    const char* from = reinterpret_cast<const char*>(a.query.data) + base * (DT == CKV_F32 ? 4 : 2);
#pragma unroll
    for (int i = 0; i < RAW; ++i) raw[i] = gload16(from + 16 * i);
    if (tid < WT_ROWS) {
      const int r = step * WT_ROWS + tid;
      next_st = r < a.rows ? stats[r] : float2{0.0f, 0.0f};
    }
  };
  auto store = [&](int stage) __attribute__((always_inline)) {
    uint4* to = reinterpret_cast<uint4*>(&lds.q[stage][0][qr * K_STRIDE + qd]);
    if constexpr (DT == CKV_BF16) {
      to[0] = raw[0];
      to[1] = raw[1];
    } else {
      uint32_t w[NP * 8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const uint32_t* r = reinterpret_cast<const uint32_t*>(&raw[0]);
        float lo, hi;
        if constexpr (DT == CKV_F16) {
          lo = (float)__builtin_bit_cast(_Float16, (uint16_t)(r[i] & 0xffffu));
          hi = (float)__builtin_bit_cast(_Float16, (uint16_t)(r[i] >> 16));
        } else {
          lo = ckv_u2f(r[2 * i]);
          hi = ckv_u2f(r[2 * i + 1]);
        }
        split_pair<NP>(lo, hi, w + i, 8);
      }
#pragma unroll
      for (int p = 0; p < NP; ++p) {
        uint4* piece = to + p * (WT_ROWS * K_STRIDE / 8);
        piece[0] = uint4{w[8 * p], w[8 * p + 1], w[8 * p + 2], w[8 * p + 3]};
        piece[1] = uint4{w[8 * p + 4], w[8 * p + 5], w[8 * p + 6], w[8 * p + 7]};
      }
    }
    if (tid < WT_ROWS) lds.stats[stage][tid] = next_st;
  };
  f32x16_t got = {};
  int stage = 0;
  const int first = step_lo + share;
  if (first < step_hi) {
    load(first);
    store(0);
  }
  __syncthreads();
  for (int step = first; step < step_hi; step += shares) {
    load(min(step + shares, step_hi - 1));
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      const int qrow = 32 * x + (lane & 31);
      f32x16_t acc = {};
#pragma unroll
      for (int s = 0; s < 8; ++s) {
#pragma unroll
        for (int p = 0; p < NP; ++p)
          acc = mfma32(kop[s], *reinterpret_cast<const uint4*>(&lds.q[stage][p][qrow * K_STRIDE + 16 * s + 8 * half]),
                       acc);
      }
      float2 st = lds.stats[stage][qrow];
      // the 32 query rows together first, on the scalar unit: all there and all seeing all of the wave's rows
      const int row = step * WT_ROWS + 32 * x, last = row + 31;
      bool clear = full && last < a.rows;
      if (clear) {
        const int t0 = token_of(a, row), t1 = token_of(a, last);
        int lo, hi, unused;
        query_range(a, t0 * a.group, count, seen, &unused, &hi);
        query_range(a, t1 * a.group, count, seen, &lo, &unused);
        clear = t1 < count && range.x >= lo && range.y <= hi;
      }
      if (!clear) {
        asm volatile("");
        int lo, hi;
        query_range(a, step * WT_ROWS + qrow, count, seen, &lo, &hi);
        const Seen see(lo, hi);
#pragma unroll
        for (int g = 0; g < 4; ++g) {
          const int4 p = *reinterpret_cast<const int4*>(&lds.pos[32 * wave + 8 * g + 4 * half]);
          const int at[4] = {p.x, p.y, p.z, p.w};
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            float y = acc[4 * g + e];
            see.mask(y, at[e]);
            acc[4 * g + e] = y;
          }
        }
        if (st.y != st.y) {
          // The query is NaN (by its own values, a key's or an infinite score), and so is what the rows that it sees
          // get; below, a masked row's zero times NaN would be NaN too.
#pragma unroll
          for (int v = 0; v < 16; ++v) {
            const int p = lds.pos[32 * wave + 8 * (v >> 2) + 4 * half + (v & 3)];
            if ((uint32_t)(p - see.lo) <= see.span) got[v] = st.y;
          }
          st = float2{0.0f, 0.0f};
        }
      }
#pragma unroll
      for (int v = 0; v < 16; ++v) {
        const float p = __builtin_amdgcn_exp2f(__builtin_fmaf(acc[v], sl2, -st.x));
        got[v] = __builtin_fmaf(p, st.y, got[v]);
      }
    }
    store(stage ^ 1);
    __syncthreads();
    stage ^= 1;
  }
  // lane 4 g + e of each half writes its row 8 g + 4 half + e
  float sum = 0.0f;
#pragma unroll
  for (int v = 0; v < 16; ++v) {
    float x = got[v];
    x = add_xor_f32<1>(x);
    x = add_xor_f32<2>(x);
    x = add_xor_f32<4>(x);
    x = x + xor_f32<8>(x);
    x = add_xor16(x);
    sum = (lane & 15) == v ? x : sum;
  }
  const int v = lane & 15;
  const int r = row0 + 8 * (v >> 2) + 4 * half + (v & 3);
  if ((lane & 16) == 0 && r < n) {
    if (shares == 1) q.weights[r] += sum;
    else a.sums[((int64_t)share * heads + bh) * c.capacity + r] = sum;
  }
}

__global__ __launch_bounds__(256) void weights_add_kernel(const QuantAttendArgs a, const int shares) {
  const ckv_quant_cache& c = a.cache;
  const int bh = blockIdx.x, b = bh / c.kv_heads, h = bh % c.kv_heads;
  const int64_t r = (int64_t)blockIdx.y * 256 + threadIdx.x;
  if (r >= quant_length(c, b)) return;
  float x = 0.0f;
  for (int s = 0; s < shares; ++s) x += a.sums[((int64_t)s * gridDim.x + bh) * c.capacity + r];
  quant_head(c, b, h).weights[r] += x;
}

template <int DT>
int launch_weights(const QuantAttendArgs& a, hipStream_t s) {
  const ckv_quant_cache& c = a.cache;
  const int64_t blocks = ((int64_t)c.capacity + WT_KEYS - 1) / WT_KEYS;
  const int shares = many_row_shares(&c, a.rows);
  const int64_t grid = blocks * c.batch * c.kv_heads * shares;
  if (grid > 0x7fffffff) return ckv_internal::set_error(CKV_E_LIMIT, "ckv_quant_attention: cache too large");
  rows_weights_kernel<DT><<<(uint32_t)grid, 64 * WT_WAVES, 0, s>>>(a, shares);
  int rc = launched("ckv_quant_attention");
  if (!rc && shares > 1) {
    weights_add_kernel<<<dim3(c.batch * c.kv_heads, (uint32_t)((c.capacity + 255) / 256)), 256, 0, s>>>(a, shares);
    rc = launched("ckv_quant_attention");
  }
  return rc;
}

}  // namespace

namespace ckv {

int many_row_block(int dtype) { return 32 * (dtype == CKV_BF16 ? rows_waves<CKV_BF16>() : rows_waves<CKV_F32>()); }

// Four workgroups a compute unit, which even out what is left over at the end (4,095
// queries of a prompt: the whole call 243 us, with two 254, with eight 247; the old
// rows' blocks last instead of first 262).
int many_row_shares(const ckv_quant_cache* c, int rows) {
  const int64_t blocks = ((int64_t)c->capacity + WT_KEYS - 1) / WT_KEYS * c->batch * c->kv_heads;
  const int64_t steps = (rows + WT_ROWS - 1) / WT_ROWS;
  const int64_t want = (1024 + blocks - 1) / blocks;
  return (int)(want < 1 ? 1 : want > 32 ? (steps < 32 ? steps : 32) : want > steps ? steps : want);
}

int launch_many_rows(const QuantAttendArgs& a, int dtype, hipStream_t stream) {
  if (dtype == CKV_BF16) return launch_rows<CKV_BF16>(a, stream);
  if (dtype == CKV_F16) return launch_rows<CKV_F16>(a, stream);
  return launch_rows<CKV_F32>(a, stream);
}

int launch_many_rows_weights(const QuantAttendArgs& a, int dtype, hipStream_t stream) {
  if (dtype == CKV_BF16) return launch_weights<CKV_BF16>(a, stream);
  if (dtype == CKV_F16) return launch_weights<CKV_F16>(a, stream);
  return launch_weights<CKV_F32>(a, stream);
}

}  // namespace ckv
