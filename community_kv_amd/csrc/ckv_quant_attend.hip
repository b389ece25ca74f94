// Attention over the 8-bit KV cache (gfx950).
//
//   s_j = softmax_scale * s^K_j * (q . c^K_j),  out = sum_j e^{s_j - lse} s^V_j c^V_j
//
// E4M3 codes have four significant bits, so they are exact in bf16, and the
// products run on v_mfma_f32_16x16x32_bf16 with the codes themselves; block
// scales multiply the scores and the probabilities, in 32 bits.  Queries and
// scaled probabilities are split into as many bf16 pieces as their type has
// significant bits (bf16 queries 1, fp16 2, f32 3), each piece a product of its
// own into the same 32-bit accumulator.  The one piece of bf16 rounds a probability
// by up to 2^-8 of it, where the sums and received weights keep 32 bits: against 64
// bits, relative to the outputs' norm, 1.7e-3 for single queries and 1.9e-3 for
// 2,048 over 32k rows, where rounding the exact output alone gives 1.6e-3; a second
// piece would be another product.
//
// A head's query rows are packed as token * group + query head, so that one
// read of a key or value serves the whole group.
#include <hip/hip_runtime.h>

#include "ckv_quant_attend.h"

namespace {
using namespace ckv;

constexpr int STEP = 32;  // cache rows a wave takes at a time
constexpr int WAVES = 4;
constexpr int FEW_WORKGROUPS = 512;  // workgroups that split the cache rows: two a compute unit, all at once
constexpr int MAX_PARTS = FEW_WORKGROUPS;  // of one sequence
static_assert(PART_UNIT % (WAVES * STEP) == 0, "parts are whole rounds of the waves");

int fail(int code, const char* message) { return ckv_internal::set_error(code, message); }

int launched(const char* what) {
  const hipError_t e = hipGetLastError();
  if (e == hipSuccess) return CKV_OK;
  static thread_local char message[160];
  snprintf(message, sizeof(message), "%s: %s", what, hipGetErrorString(e));
  return fail(CKV_E_LAUNCH, message);
}

// The 16 query rows from `row0` as B operands of the four 32-dim steps: lane
// (L, c) = (lane / 16, lane % 16) holds row c, dims dim_of(step, L) .. + 7 --
// 16 neighbouring dims a lane for steps 0, 1 and for 2, 3, so that a cache row's
// codes are read 16 bytes a lane, 64 contiguous bytes for the four lane groups.
__device__ inline int dim_of(int s, int L) { return 64 * (s >> 1) + 16 * L + 8 * (s & 1); }

template <int DT>
struct QueryTile {
  uint4 piece[pieces(DT)][4];
};

template <int DT>
__device__ inline void load_query_tile(const QuantAttendArgs& a, int b, int h, int row0, QueryTile<DT>& q) {
  constexpr int NP = pieces(DT);
  const int L = (threadIdx.x & 63) >> 4;
  const int row = row0 + (threadIdx.x & 15);
  const bool ok = row < a.rows;
  const int t = ok ? token_of(a, row) : 0, g = ok ? row - t * a.group : 0;
  const int64_t base = (int64_t)b * a.query.batch_stride + (int64_t)(h * a.group + g) * a.query.head_stride +
                       (int64_t)t * a.query.token_stride;
#pragma unroll
  for (int s = 0; s < 4; ++s) {
    float v[8];
    load_query8<DT>(a.query.data, base + dim_of(s, L), v);
    uint32_t w[NP * 4];
#pragma unroll
    for (int i = 0; i < 4; ++i) split_pair<NP>(ok ? v[2 * i] : 0.0f, ok ? v[2 * i + 1] : 0.0f, w + i, 4);
#pragma unroll
    for (int p = 0; p < NP; ++p) q.piece[p][s] = uint4{w[4 * p], w[4 * p + 1], w[4 * p + 2], w[4 * p + 3]};
  }
}

// One step's rows of a head: keys as A operands (row m of MFMA block j is cache
// row 8 (m / 4) + 4 j + m % 4 of the step, so that an accumulator lane holds the
// eight rows 8 L .. 8 L + 7, just what the P operand of the value product
// takes), values 8 dims a lane of the rows 8 L + u.
struct StepCodes {
  uint4 k[2][2];
  uint2 v[8];
  float ks, vs;
  int4 pos[2];  // positions of the rows 8 L .. 8 L + 7, where masks need them
};

__device__ inline int step_row(int j, int m) { return 8 * (m >> 2) + 4 * j + (m & 3); }

template <bool WITH_V = true>
__device__ inline void load_step(const QuantHead& q, int t0, int last, int block_log2, bool positions, StepCodes& s) {
  const int lane = threadIdx.x & 63, L = lane >> 4, c = lane & 15;
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    const uint8_t* p = q.key_codes + (int64_t)min(t0 + step_row(j, c), last) * D + 16 * L;
    s.k[j][0] = gload16(p);
    s.k[j][1] = gload16(p + 64);
  }
  const int blk = min(t0 + 8 * L, last) >> block_log2;
  s.ks = gload_f32(q.key_scales + blk);
  if (positions) {
    // eight rows at once: the capacity is a multiple of 16
    const int32_t* p = q.positions + (min(t0 + 8 * L, last) & ~7);
    s.pos[0] = __builtin_bit_cast(int4, gload16(p));
    s.pos[1] = __builtin_bit_cast(int4, gload16(p + 4));
  }
  if constexpr (WITH_V) {
#pragma unroll
    for (int u = 0; u < 8; ++u) {
      typedef unsigned int u32x2_t __attribute__((ext_vector_type(2)));
      typedef const __attribute__((address_space(1))) u32x2_t* global_u32x2_ptr;
      const u32x2_t w = *(global_u32x2_ptr)(q.value_codes + (int64_t)min(t0 + 8 * L + u, last) * D + 8 * c);
      s.v[u] = uint2{w[0], w[1]};
    }
    s.vs = gload_f32(q.value_scales + blk);
  }
}

// Scores of a step in log2 units: sc[4 j + i] = row 8 L + 4 j + i against query
// row c; rows past n and positions outside [lo, hi] are -inf.
template <int DT>
__device__ inline void step_scores(const StepCodes& s, const QueryTile<DT>& q, float scale_log2, float* sc) {
  constexpr int NP = pieces(DT);
  const float f = s.ks * scale_log2;
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    f32x4_t acc = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int st = 0; st < 4; ++st) {
      const uint4 w = s.k[j][st >> 1];
      const uint4 op = (st & 1) ? codes8_to_bf16(w.z, w.w) : codes8_to_bf16(w.x, w.y);
#pragma unroll
      for (int p = 0; p < NP; ++p) acc = mfma_bf16(op, q.piece[p][st], acc);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) sc[4 * j + i] = acc[i] * f;
  }
}

// Masks the scores of the step from t0 on: n rows in use; by_position: only
// positions in [lo, hi] are seen, otherwise all rows in use are.
__device__ inline void mask_step(const StepCodes& s, bool by_position, int t0, int n, int lo, int hi, float* sc) {
  const int L = (threadIdx.x & 63) >> 4;
  const int p[8] = {s.pos[0].x, s.pos[0].y, s.pos[0].z, s.pos[0].w, s.pos[1].x, s.pos[1].y, s.pos[1].z, s.pos[1].w};
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const bool ok = t0 + 8 * L + i < n && (!by_position || (p[i] >= lo && p[i] <= hi));
    sc[i] = ok ? sc[i] : NEG_INF;
  }
}

// B operands of the value product: for dims 8 c + d, the rows 8 L + u.
__device__ inline void value_operands(const uint2* v, uint4* op) {
#pragma unroll
  for (int half = 0; half < 2; ++half) {
#pragma unroll
    for (int pair = 0; pair < 2; ++pair) {  // dims 4 half + 2 pair, + 1
      uint32_t w[4];
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const uint32_t a = half ? v[2 * u].y : v[2 * u].x, b = half ? v[2 * u + 1].y : v[2 * u + 1].x;
        // bytes (row 2u, row 2u + 1) of the first dim, then of the second
        w[u] = __builtin_amdgcn_perm(b, a, pair ? 0x07030602u : 0x05010400u);
      }
      op[4 * half + 2 * pair] = uint4{codes_to_bf16<false>(w[0]), codes_to_bf16<false>(w[1]),
                                      codes_to_bf16<false>(w[2]), codes_to_bf16<false>(w[3])};
      op[4 * half + 2 * pair + 1] = uint4{codes_to_bf16<true>(w[0]), codes_to_bf16<true>(w[1]),
                                          codes_to_bf16<true>(w[2]), codes_to_bf16<true>(w[3])};
    }
  }
}

__device__ inline bool has_nan_code(uint32_t w) {
  // a byte is NaN where its low seven bits are all ones
  return (((w & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u) != 0;
}

__device__ inline uint32_t without_nan_codes(uint32_t w) {
  const uint32_t is = ((w & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u;  // 0x80 in every NaN byte
  const uint32_t all = (is >> 7) * 0xffu;
  return w & ~all;
}

// The running softmax of 16 query rows over the steps of one wave.  m: log2
// maximum of query row c, the same on the four lane groups; l: sum over this
// lane's rows alone; o: accumulators, element i of block nb is query row
// 4 L + i, dim 8 c + nb.
struct Running {
  float m, l;
  f32x4_t o[8];
};

// Adds a step to a row tile's running softmax.  fix_nan: the step has masked
// rows and NaN among its values, which `vop` holds as zeros (a product with a
// masked row's zero probability would spread them) and `v` as they are.
template <int DT>
__device__ inline void add_step(const float* sc, float vs, const uint4* vop, bool fix_nan, const uint2* v, Running& r) {
  constexpr int NP = pieces(DT);
  float top = sc[0];
#pragma unroll
  for (int i = 1; i < 8; ++i) top = fmaxf(top, sc[i]);
  if (__ballot(top > r.m + RESCALE) != 0) {
    float t = fmaxf(top, xor_f32<16>(top));
    t = fmaxf(t, xor_f32<32>(t));
    t = t > r.m + RESCALE ? t : r.m;  // a query's own scores alone decide
    const float corr = r.m == t ? 1.0f : __builtin_amdgcn_exp2f(r.m - t);
    const int L = (threadIdx.x & 63) >> 4;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float f = __shfl(corr, 4 * L + i, 64);
#pragma unroll
      for (int nb = 0; nb < 8; ++nb) r.o[nb][i] *= f;
    }
    r.l *= corr;
    r.m = t;
  }
  const float m = r.m == NEG_INF ? 0.0f : r.m;
  float p[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    p[i] = __builtin_amdgcn_exp2f(sc[i] - m);
    r.l += p[i];
  }
  uint32_t w[NP * 4];
#pragma unroll
  for (int i = 0; i < 4; ++i) split_pair<NP>(p[2 * i] * vs, p[2 * i + 1] * vs, w + i, 4);
#pragma unroll
  for (int q = 0; q < NP; ++q) {
    const uint4 aop = {w[4 * q], w[4 * q + 1], w[4 * q + 2], w[4 * q + 3]};
#pragma unroll
    for (int nb = 0; nb < 8; ++nb) r.o[nb] = mfma_bf16(aop, vop[nb], r.o[nb]);
  }
  if (fix_nan) {
    // values of this step hold NaN, which were taken as zeros above: what is
    // NaN is a query that sees such a row, in that dim
    uint32_t one[4];
#pragma unroll
    for (int i = 0; i < 4; ++i)
      one[i] = (sc[2 * i] == NEG_INF ? 0u : 0x3f80u) | (sc[2 * i + 1] == NEG_INF ? 0u : 0x3f800000u);
    const uint4 aop = {one[0], one[1], one[2], one[3]};
#pragma unroll
    for (int nb = 0; nb < 8; ++nb) {
      uint32_t is[4];
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const uint32_t lo = (nb < 4 ? v[2 * u].x : v[2 * u].y) >> (8 * (nb & 3));
        const uint32_t hi = (nb < 4 ? v[2 * u + 1].x : v[2 * u + 1].y) >> (8 * (nb & 3));
        is[u] = ((lo & 0x7fu) == 0x7fu ? 0x3f80u : 0u) | ((hi & 0x7fu) == 0x7fu ? 0x3f800000u : 0u);
      }
      const f32x4_t hits = mfma_bf16(aop, uint4{is[0], is[1], is[2], is[3]}, f32x4_t{0.0f, 0.0f, 0.0f, 0.0f});
#pragma unroll
      for (int i = 0; i < 4; ++i) r.o[nb][i] = hits[i] > 0.0f ? __builtin_nanf("") : r.o[nb][i];
    }
  }
}

// Received weight from the scores that the split kernel left (at most 16 query
// rows a head): a thread adds up the four cache rows from r on over the query rows.
// Writing and reading 4 bytes a row and query costs less than the keys again.  A
// whole call, 2 sequences of 16,000 rows, 32 heads over 8: 4 query rows a head 27.4
// us from kept scores and 36.4 with them computed again (weights_kernel), 16 rows
// 35.9 and 44.0; 2,000 rows: 16.3 and 18.1, 21.2 and 21.2.  With more query rows
// the kept scores would outgrow the cache itself (64 rows: 256 bytes a cache row).
__device__ inline void add_scores(const QuantAttendArgs& a, int b, int h, int64_t r) {
  const ckv_quant_cache& c = a.cache;
  const int n = quant_length(c, b);
  if (r >= n) return;
  const int64_t bh = (int64_t)b * c.kv_heads + h;
  const QuantHead q = quant_head(c, b, h);
  if (a.window > 0) {  // scores were written only of steps with a row in sight
    int lo, hi;
    rows_range(a, 0, a.rows, new_count(a, b), c.cursors[c.batch + b], &lo, &hi);
    const int4 p = __builtin_bit_cast(int4, gload16(q.positions + r));
    const bool need = (p.x >= lo && p.x <= hi) || (r + 1 < n && p.y >= lo && p.y <= hi) ||
                      (r + 2 < n && p.z >= lo && p.z <= hi) || (r + 3 < n && p.w >= lo && p.w <= hi);
    if (!need) return;
  }
  const float* from = a.scores + bh * a.rows * c.capacity + r;
  const float2* stats = a.stats + bh * a.row_pad;
  float got[4] = {};
  bool nan = false;
#pragma unroll 4
  for (int row = 0; row < a.rows; ++row) {
    const float4 s = *reinterpret_cast<const float4*>(from + (int64_t)row * c.capacity);
    const float2 st = stats[row];
    const float v[4] = {s.x, s.y, s.z, s.w};
    nan |= st.y != st.y;
#pragma unroll
    for (int i = 0; i < 4; ++i) got[i] += v[i] == NEG_INF ? 0.0f : __builtin_amdgcn_exp2f(v[i] - st.x) * st.y;
  }
  if (nan) {  // a NaN query makes what it sees NaN, scores of minus infinity too, which masked rows have as well
    const int4 p = __builtin_bit_cast(int4, gload16(q.positions + r));
    const int at[4] = {p.x, p.y, p.z, p.w};
    const int count = new_count(a, b), seen = c.cursors[c.batch + b];
    for (int row = 0; row < a.rows; ++row) {
      const float share = stats[row].y;
      if (share == share) continue;
      int lo, hi;
      query_range(a, row, count, seen, &lo, &hi);
#pragma unroll
      for (int i = 0; i < 4; ++i) got[i] = at[i] >= lo && at[i] <= hi ? share : got[i];
    }
  }
  float* to = q.weights + r;
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if (r + i < n) to[i] += got[i];
}

// Goes over this wave's steps of a part.  Without a window: the part's rows, STEP
// of every WAVES * STEP.  With one most rows are out of every query's sight, and
// those in it mostly stand together: a part is then every count-th unit of
// WAVES * STEP rows, so that all parts have some of them, and a wave looks at the
// positions of its STEP rows of eight units at once (four a lane) and passes over
// steps that nobody sees.  Eight sequences of 16k-131k rows in order, window 4,096,
// in a graph: 34 us, where reading every row takes 312; of rows in any order, 256.
struct StepWalk {
  int t0, end;       // first row of the step; rows end before `end`
  int unit, stride;  // with a window
  int lo, hi;        // positions that the workgroup's queries see
  uint64_t bits;     // steps to come of the eight units from `unit` on, eight bits each
  __device__ StepWalk(const QuantAttendArgs& a, const Part& part, int n, int wave, int row0, int count, int seen)
      : end(n), lo(0), hi(0), bits(0) {
    if (a.window == 0) {
      end = (int)min((int64_t)part.index * part.rows + part.rows, (int64_t)n);
      t0 = part.index * part.rows + (wave - WAVES) * STEP;
    } else {
      rows_range(a, row0, 16, count, seen, &lo, &hi);
      stride = part.count;
      unit = part.index - 8 * stride;
    }
  }
  __device__ bool next(const QuantAttendArgs& a, const QuantHead& q, int wave) {
    if (a.window == 0) {
      t0 += WAVES * STEP;
      return t0 < end;
    }
    const int lane = threadIdx.x & 63;
    while (bits == 0) {
      unit += 8 * stride;  // at most 2^23 + 2^12 units
      if (unit * (WAVES * STEP) >= end) return false;
      const int row = (unit + (lane >> 3) * stride) * (WAVES * STEP) + wave * STEP + 4 * (lane & 7);
      bool need = false;
      if (row < end) {
        const int4 p = __builtin_bit_cast(int4, gload16(q.positions + row));
        need = (p.x >= lo && p.x <= hi) || (row + 1 < end && p.y >= lo && p.y <= hi) ||
               (row + 2 < end && p.z >= lo && p.z <= hi) || (row + 3 < end && p.w >= lo && p.w <= hi);
      }
      bits = __ballot(need);
    }
    const int k = (__ffsll((unsigned long long)bits) - 1) >> 3;
    bits &= ~(0xffull << (8 * k));
    t0 = (unit + k * stride) * (WAVES * STEP) + wave * STEP;
    return true;
  }
};

// One workgroup of four waves takes a part of the cache rows of a (sequence,
// head) for 16 query rows; its waves take steps in turn and join in LDS.
// Bound by memory: eight sequences of 16k-131k rows (32/8 heads, one query,
// bf16) read 1.69 GB in 283 us, 6.0 TB/s.  512 workgroups, all resident, two
// waves a SIMD: 1,024 and 2,048 workgroups take 3 and 8 % longer there and 9 and
// 20 % at one sequence of 131k; three waves a SIMD (168 registers) the same or
// longer, reading a step ahead into a second set of registers the same.
// SUMS: every sequence is one part and the scores are kept, so that the workgroup
// adds up the received weights itself and no launch has to (8 sequences of 300 rows
// 11.6 us, with a launch 12.5; 64 of 600 21.9 and 23.8).
template <int DT, bool SUMS>
__global__ __launch_bounds__(64 * WAVES, 2) void attend_split_kernel(const QuantAttendArgs a) {
  __shared__ float m_s[WAVES][16];
  __shared__ float l_s[WAVES][16];
  __shared__ float o_s[WAVES][16 * D];
  const ckv_quant_cache& c = a.cache;
  const int h = blockIdx.x % c.kv_heads, number = blockIdx.x / c.kv_heads, row0 = 16 * blockIdx.y;
  const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int lane = tid & 63, L = lane >> 4, col = lane & 15;
  const Part part = find_part(QuantLengths{c}, a.parts, number, -1);
  const int b = part.sequence;
  if (b < 0) return;  // the join knows how many parts there are
  const int n = quant_length(c, b), seen = c.cursors[c.batch + b], count = new_count(a, b);
  const QuantHead q = quant_head(c, b, h);
  const int block_log2 = 31 - __clz(c.block);
  QueryTile<DT> query;
  Running run;
  int lo, hi;
  load_query_tile<DT>(a, b, h, row0, query);
  query_range(a, row0 + col, count, seen, &lo, &hi);
  run.m = NEG_INF;
  run.l = 0.0f;
#pragma unroll
  for (int nb = 0; nb < 8; ++nb) run.o[nb] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
  // with one new token and no window every row in use is at or before it
  const bool by_position = a.window > 0 || a.tokens > 1 || count < a.tokens;
  StepCodes cur;
  StepWalk walk(a, part, n, wave, row0, count, seen);
  while (walk.next(a, q, wave)) {
    const int t0 = walk.t0;
    load_step(q, t0, n - 1, block_log2, by_position, cur);
    const bool tail = t0 + STEP > n;
    bool fix_nan = false;
    uint2 raw[8];
    if (tail || by_position) {
#pragma unroll
      for (int u = 0; u < 8; ++u) raw[u] = cur.v[u];
      bool nan = false;
#pragma unroll
      for (int u = 0; u < 8; ++u) nan = nan || has_nan_code(raw[u].x) || has_nan_code(raw[u].y);
      fix_nan = __ballot(nan) != 0;
      if (fix_nan) {
#pragma unroll
        for (int u = 0; u < 8; ++u) cur.v[u] = uint2{without_nan_codes(raw[u].x), without_nan_codes(raw[u].y)};
      }
    }
    uint4 vop[8];
    value_operands(cur.v, vop);
    float sc[8];
    step_scores<DT>(cur, query, a.scale_log2, sc);
    if (tail || by_position) mask_step(cur, by_position, t0, n, lo, hi, sc);
    if (a.scores && col < a.rows && t0 + 8 * L < n) {
      float4* p = reinterpret_cast<float4*>(
          a.scores + (((int64_t)b * c.kv_heads + h) * a.rows + col) * c.capacity + t0 + 8 * L);
      p[0] = float4{sc[0], sc[1], sc[2], sc[3]};
      p[1] = float4{sc[4], sc[5], sc[6], sc[7]};
    }
    add_step<DT>(sc, cur.vs, vop, fix_nan, raw, run);
  }
  // join the waves
  {
    float l = add_xor16(run.l);
    l = add_xor32(l);
    __syncthreads();
    if (L == 0) {
      m_s[wave][col] = run.m;
      l_s[wave][col] = l;
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      float4* p = reinterpret_cast<float4*>(&o_s[wave][(4 * L + i) * D + 8 * col]);
      p[0] = float4{run.o[0][i], run.o[1][i], run.o[2][i], run.o[3][i]};
      p[1] = float4{run.o[4][i], run.o[5][i], run.o[6][i], run.o[7][i]};
    }
    __syncthreads();
    for (int x = tid; x < 16 * D; x += 64 * WAVES) {
      const int i = x >> 7, d = x & (D - 1), row = row0 + i;
      if (row >= a.rows) continue;
      float m = m_s[0][i];
#pragma unroll
      for (int w = 1; w < WAVES; ++w) m = fmaxf(m, m_s[w][i]);
      const float at = m == NEG_INF ? 0.0f : m;
      float sum = 0.0f, acc = 0.0f;
#pragma unroll
      for (int w = 0; w < WAVES; ++w) {
        // a wave without a row has zeros and a maximum of -inf
        const float f = __builtin_amdgcn_exp2f(m_s[w][i] - at);
        sum += l_s[w][i] * f;
        acc += o_s[w][x] * f;
      }
      const int64_t bh = (int64_t)b * c.kv_heads + h;
      if (part.count == 1) {
        int64_t at_out, at_lse;
        output_index(a, b, h, row, &at_out, &at_lse);
        store_out<DT>(a.out, at_out + d, sum == 0.0f ? 0.0f : acc / sum);
        if (d == 0) {
          a.lse[at_lse] = sum == 0.0f ? NEG_INF : (m + __log2f(sum)) * LN2;
          if (a.stats) a.stats[bh * a.row_pad + row] = float2{at, sum == 0.0f ? 0.0f : 1.0f / sum};
        }
      } else {
        a.part_acc[(((int64_t)h * a.parts + number) * a.row_pad + row) * D + d] = acc;
        if (d == 0) {
          a.part_max[((int64_t)h * a.row_pad + row) * a.parts + number] = m;
          a.part_sum[((int64_t)h * a.row_pad + row) * a.parts + number] = sum;
        }
      }
    }
  }
  if constexpr (SUMS) {
    __syncthreads();  // the scores and statistics are written
    for (int64_t r = 4 * tid; r < n; r += 4 * 64 * WAVES) add_scores(a, b, h, r);
  }
}

// Joins the parts of one query row: a workgroup of 256 threads, a part each for
// the maximum and the sum, then four dims and every eighth part each.
constexpr int JOIN_THREADS = 256;

template <int DT>
__global__ __launch_bounds__(JOIN_THREADS) void attend_join_kernel(const QuantAttendArgs a) {
  __shared__ float factor[MAX_PARTS];
  __shared__ float scratch[4];
  __shared__ float4 acc_s[JOIN_THREADS];
  const ckv_quant_cache& c = a.cache;
  const int row = blockIdx.x, h = blockIdx.y, b = blockIdx.z, tid = threadIdx.x;
  const Part part = find_part(QuantLengths{c}, a.parts, 0, b);
  if (part.count == 1) return;  // written already
  const float* pm = a.part_max + ((int64_t)h * a.row_pad + row) * a.parts + part.first;
  const float* pl = a.part_sum + ((int64_t)h * a.row_pad + row) * a.parts + part.first;
  float m = NEG_INF;
  for (int s = tid; s < part.count; s += JOIN_THREADS) m = fmaxf(m, pm[s]);
  m = block_max256(m, scratch);
  const float at = m == NEG_INF ? 0.0f : m;
  float sum = 0.0f;
  for (int s = tid; s < part.count; s += JOIN_THREADS) {
    const float f = __builtin_amdgcn_exp2f(pm[s] - at);
    factor[s] = f;
    sum += pl[s] * f;
  }
  sum = wave_sum_tree(sum);
  __syncthreads();  // scratch is read
  if ((tid & 63) == 0) scratch[tid >> 6] = sum;
  __syncthreads();
  sum = (scratch[0] + scratch[1]) + (scratch[2] + scratch[3]);
  const int dim = 4 * (tid & 31);
  float4 acc{0.0f, 0.0f, 0.0f, 0.0f};
  const float* pa = a.part_acc + (((int64_t)h * a.parts + part.first) * a.row_pad + row) * D + dim;
#pragma unroll 4
  for (int s = tid >> 5; s < part.count; s += JOIN_THREADS / 32) {
    const float4 x = *reinterpret_cast<const float4*>(pa + (int64_t)s * a.row_pad * D);
    const float f = factor[s];
    acc.x += x.x * f;
    acc.y += x.y * f;
    acc.z += x.z * f;
    acc.w += x.w * f;
  }
  acc_s[tid] = acc;
  __syncthreads();
  int64_t at_out, at_lse;
  output_index(a, b, h, row, &at_out, &at_lse);
  if (tid < D) {
    float x = 0.0f;
#pragma unroll
    for (int g = 0; g < JOIN_THREADS / 32; ++g) x += reinterpret_cast<const float*>(acc_s)[g * D + tid];
    store_out<DT>(a.out, at_out + tid, sum == 0.0f ? 0.0f : x / sum);
  }
  if (tid == 0) {
    a.lse[at_lse] = sum == 0.0f ? NEG_INF : (m + __log2f(sum)) * LN2;
    if (a.stats)
      a.stats[((int64_t)b * c.kv_heads + h) * a.row_pad + row] = float2{at, sum == 0.0f ? 0.0f : 1.0f / sum};
  }
}

// The same for many query rows, of few parts mostly: a wave a row, two dims a lane
// (702 queries over 4,201 rows, 28 heads, in 3 parts: the whole call 75 us, with a
// workgroup a row 94).
template <int DT>
__global__ __launch_bounds__(256) void attend_join_rows_kernel(const QuantAttendArgs a) {
  const ckv_quant_cache& c = a.cache;
  const int row = 4 * blockIdx.x + (threadIdx.x >> 6), h = blockIdx.y, b = blockIdx.z, lane = threadIdx.x & 63;
  if (row >= a.rows) return;
  const Part part = find_part(QuantLengths{c}, a.parts, 0, b);
  if (part.count == 1) return;
  const int64_t first = ((int64_t)h * a.row_pad + row) * a.parts + part.first;
  float m = NEG_INF;
  for (int s = lane; s < part.count; s += 64) m = fmaxf(m, a.part_max[first + s]);
  m = wave_max(m);
  const float at = m == NEG_INF ? 0.0f : m;
  const float* pa = a.part_acc + (((int64_t)h * a.parts + part.first) * a.row_pad + row) * D + 2 * lane;
  float sum = 0.0f;
  float2 acc{0.0f, 0.0f};
  for (int s0 = 0; s0 < part.count; s0 += 64) {
    const int left = min(part.count - s0, 64);
    float f = 0.0f, share = 0.0f;
    if (lane < left) {
      f = __builtin_amdgcn_exp2f(a.part_max[first + s0 + lane] - at);
      share = a.part_sum[first + s0 + lane] * f;
    }
    sum += wave_sum_tree(share);
#pragma unroll 4
    for (int s = 0; s < left; ++s) {
      const float2 x = *reinterpret_cast<const float2*>(pa + (int64_t)(s0 + s) * a.row_pad * D);
      const float of = ckv_u2f((uint32_t)__builtin_amdgcn_readlane((int)ckv_f2u(f), s));
      acc.x += x.x * of;
      acc.y += x.y * of;
    }
  }
  int64_t at_out, at_lse;
  output_index(a, b, h, row, &at_out, &at_lse);
  store_out<DT>(a.out, at_out + 2 * lane, sum == 0.0f ? 0.0f : acc.x / sum);
  store_out<DT>(a.out, at_out + 2 * lane + 1, sum == 0.0f ? 0.0f : acc.y / sum);
  if (lane == 0) {
    a.lse[at_lse] = sum == 0.0f ? NEG_INF : (m + __log2f(sum)) * LN2;
    if (a.stats)
      a.stats[((int64_t)b * c.kv_heads + h) * a.row_pad + row] = float2{at, sum == 0.0f ? 0.0f : 1.0f / sum};
  }
}

constexpr int SUM_THREADS = 64;
__global__ __launch_bounds__(SUM_THREADS) void weights_of_scores_kernel(const QuantAttendArgs a) {
  add_scores(a, blockIdx.z, blockIdx.y, 4 * ((int64_t)blockIdx.x * SUM_THREADS + threadIdx.x));
}

// Received weight: a wave owns 32 cache rows of a (sequence, head), goes over
// all query rows with the scores computed again, and adds up what each row got
// (no atomics: one owner a row, a fixed order).
template <int DT>
__global__ __launch_bounds__(64 * WAVES) void weights_kernel(const QuantAttendArgs a) {
  const ckv_quant_cache& c = a.cache;
  const int h = blockIdx.y, b = blockIdx.z, wave = threadIdx.x >> 6;
  const int lane = threadIdx.x & 63, L = lane >> 4, col = lane & 15;
  const int n = quant_length(c, b), seen = c.cursors[c.batch + b], count = new_count(a, b);
  const int64_t first = ((int64_t)blockIdx.x * WAVES + wave) * STEP;
  if (first >= n) return;
  const int t0 = (int)first;
  const QuantHead q = quant_head(c, b, h);
  if (a.window > 0) {
    int low, high;
    rows_range(a, 0, a.rows, count, seen, &low, &high);
    const int p = q.positions[min(t0 + (lane & 31), n - 1)];
    if (__ballot(p >= low && p <= high) == 0) return;
  }
  const bool by_position = a.window > 0 || a.tokens > 1 || count < a.tokens;
  StepCodes s;
  load_step<false>(q, t0, n - 1, 31 - __clz(c.block), by_position, s);
  const float2* stats = a.stats + ((int64_t)b * c.kv_heads + h) * a.row_pad;
  float got[8] = {};
  for (int row0 = 0; row0 < a.rows; row0 += 16) {
    QueryTile<DT> query;
    load_query_tile<DT>(a, b, h, row0, query);
    int lo, hi;
    query_range(a, row0 + col, count, seen, &lo, &hi);
    const float2 st = row0 + col < a.rows ? stats[row0 + col] : float2{0.0f, 0.0f};
    float sc[8];
    step_scores<DT>(s, query, a.scale_log2, sc);
    mask_step(s, by_position, t0, n, lo, hi, sc);
    if (st.y != st.y) {  // as in add_scores
      float seen_rows[8] = {};
      mask_step(s, by_position, t0, n, lo, hi, seen_rows);
#pragma unroll
      for (int i = 0; i < 8; ++i) got[i] = seen_rows[i] == NEG_INF ? got[i] : st.y;
      continue;
    }
#pragma unroll
    for (int i = 0; i < 8; ++i)
      got[i] += sc[i] == NEG_INF ? 0.0f : __builtin_amdgcn_exp2f(sc[i] - st.x) * st.y;
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    float x = got[i];
    x = add_xor_f32<1>(x);
    x = add_xor_f32<2>(x);
    x = add_xor_f32<4>(x);
    x = x + xor_f32<8>(x);
    const int row = t0 + 8 * L + i;
    if (col == 0 && row < n) q.weights[row] += x;
  }
}

// Parts that the cache rows of the batch are split into: enough workgroups to
// fill the chip (`workgroups`), no more than there are units.  A few units are
// left in one part, which needs no join.  2 sequences, 32/8 heads, bf16, in a graph,
// one part and several, us: up to 400 rows in 4 units 8.3 and 10.4 with 4 query
// rows, 12.5 and 12.2 with 16, 12.7 and 16.9 with 128; 640 rows in 7 units 8.6 and
// 10.0, 14.7 and 12.3, 15.1 and 18.2; 1,000 rows in 8 units 11.6 and 10.7, 19.7 and
// 12.3, 20.2 and 19.2.  (Units of the capacity: a larger cache has parts, one sequence of
// 1,000 rows 10.2 in any.)  With about as many (sequence, head, 16 query rows) as
// workgroups every sequence is one part.  Even batches lose nothing by that, but one long
// sequence among short ones then runs on one workgroup a head: 64 sequences of 8 heads,
// one of 131,072 rows and the rest of 1,000, take 1,060 us, 32 sequences 60.
constexpr int ONE_PART_UNITS = 6;

int parts_for(const ckv_quant_cache* c, int64_t row_blocks, bool many) {
  const int64_t workgroups = many ? 256 : FEW_WORKGROUPS;
  const int64_t units = ((int64_t)c->capacity + PART_UNIT - 1) / PART_UNIT;
  const int64_t want = workgroups / ((int64_t)c->kv_heads * row_blocks);
  // many rows in fewer than two parts a sequence cost more in joins than they even out
  // (8 prompts of 234 tokens, 28 heads over 4: whole 23 us, in 9 parts 44)
  if (want < (many ? 2 * c->batch : c->batch + 1) || units <= (many ? 1 : ONE_PART_UNITS)) return c->batch;
  return (int)(want < c->batch * units ? want : c->batch * units);
}

constexpr int64_t MAX_ROWS = 1 << 21;  // query rows of a head: the grids' second dimension holds their blocks

struct AttendLayout {
  int parts, row_pad;
  bool many, keep_scores;
  size_t stats, ranges, scores, sums, max, sum, acc, bytes;
  AttendLayout(const ckv_quant_cache* c, int rows, int dtype, bool accumulate) {
    row_pad = (rows + 15) / 16 * 16;
    many = many_rows(c, rows, dtype, accumulate);
    const int64_t block = many ? many_row_block(dtype) : 16;
    parts = parts_for(c, (rows + block - 1) / block, many);
    keep_scores = accumulate && rows <= 16;
    const size_t heads = (size_t)c->batch * c->kv_heads;
    size_t at = 0;
    auto take = [&](size_t bytes) {
      const size_t here = at;
      at += (bytes + 15) & ~(size_t)15;
      return here;
    };
    stats = take(accumulate ? heads * row_pad * sizeof(float2) : 0);
    ranges = take(many ? heads * ((c->capacity + RANGE_TILE - 1) / RANGE_TILE) * sizeof(int2) : 0);
    const int shares = many && accumulate ? many_row_shares(c, rows) : 1;
    sums = take(shares > 1 ? heads * c->capacity * shares * sizeof(float) : 0);
    scores = take(keep_scores ? heads * rows * c->capacity * sizeof(float) : 0);
    const size_t each = parts > c->batch ? (size_t)c->kv_heads * row_pad * parts * sizeof(float) : 0;
    max = take(each);
    sum = take(each);
    acc = take(each * D);
    bytes = at;
  }
};

template <int DT>
int launch_attend(const QuantAttendArgs& a, bool many, bool accumulate, hipStream_t s) {
  int rc;
  if (many) {
    rc = launch_many_rows(a, DT, s);
  } else {
    const dim3 grid(a.parts * a.cache.kv_heads, (a.rows + 15) / 16);
    if (a.scores && a.parts == a.cache.batch) attend_split_kernel<DT, true><<<grid, 64 * WAVES, 0, s>>>(a);
    else attend_split_kernel<DT, false><<<grid, 64 * WAVES, 0, s>>>(a);
    rc = launched("ckv_quant_attention");
  }
  if (!rc && a.parts > a.cache.batch) {
    if (many) attend_join_rows_kernel<DT><<<dim3((a.rows + 3) / 4, a.cache.kv_heads, a.cache.batch), 256, 0, s>>>(a);
    else attend_join_kernel<DT><<<dim3(a.rows, a.cache.kv_heads, a.cache.batch), JOIN_THREADS, 0, s>>>(a);
    rc = launched("ckv_quant_attention");
  }
  if (!rc && accumulate) {
    if (many) return launch_many_rows_weights(a, DT, s);
    if (a.scores) {
      if (a.parts == a.cache.batch) return rc;  // added by the attention itself
      const dim3 grid((a.cache.capacity + 4 * SUM_THREADS - 1) / (4 * SUM_THREADS), a.cache.kv_heads, a.cache.batch);
      weights_of_scores_kernel<<<grid, SUM_THREADS, 0, s>>>(a);
      return launched("ckv_quant_attention");
    }
    const dim3 grid((a.cache.capacity + WAVES * STEP - 1) / (WAVES * STEP), a.cache.kv_heads, a.cache.batch);
    weights_kernel<DT><<<grid, 64 * WAVES, 0, s>>>(a);
    rc = launched("ckv_quant_attention");
  }
  return rc;
}

}  // namespace

extern "C" size_t ckv_quant_attention_workspace_bytes(const ckv_quant_cache* cache, int32_t query_heads,
                                                      int32_t tokens, int32_t dtype, int32_t accumulate) {
  if (!cache || cache->batch <= 0 || cache->kv_heads <= 0 || cache->capacity <= 0 || tokens <= 0 ||
      query_heads <= 0 || query_heads % cache->kv_heads)
    return 0;
  const int64_t rows = (int64_t)tokens * (query_heads / cache->kv_heads);
  if (rows > MAX_ROWS) return 0;
  return AttendLayout(cache, (int)rows, dtype, accumulate != 0).bytes;
}

extern "C" int ckv_quant_attention(const ckv_quant_cache* cache, const ckv_quant_rows* query, int32_t query_heads,
                                   int32_t tokens, const int32_t* counts, int32_t dtype, float softmax_scale,
                                   int32_t window, int32_t accumulate, void* out, float* lse, void* workspace,
                                   void* stream) {
  int rc = validate_quant_cache(cache, "ckv_quant_attention");
  if (rc) return rc;
  if (dtype != CKV_BF16 && dtype != CKV_F16 && dtype != CKV_F32)
    return fail(CKV_E_INVALID, "ckv_quant_attention: dtype must be bf16, fp16 or f32");
  if (!query || !query->data || !out || !lse) return fail(CKV_E_INVALID, "ckv_quant_attention: null argument");
  if (query_heads <= 0 || query_heads % cache->kv_heads)
    return fail(CKV_E_INVALID, "ckv_quant_attention: query heads must be a multiple of the cache's heads");
  const int group = query_heads / cache->kv_heads;
  if (group > CKV_MAX_GROUP) return fail(CKV_E_LIMIT, "ckv_quant_attention: group size exceeds 16");
  if (tokens <= 0 || window < 0) return fail(CKV_E_INVALID, "ckv_quant_attention: tokens must be positive, window not negative");
  if ((int64_t)tokens * group > MAX_ROWS)
    return fail(CKV_E_LIMIT, "ckv_quant_attention: more than 2^21 query rows a head");
  if (!(softmax_scale > 0.0f) || softmax_scale > 1e30f)
    return fail(CKV_E_INVALID, "ckv_quant_attention: softmax_scale must be positive");
  const int unit = dtype == CKV_F32 ? 4 : 8;
  if (((uintptr_t)query->data & 15) || query->batch_stride % unit || query->head_stride % unit ||
      query->token_stride % unit)
    return fail(CKV_E_INVALID, "ckv_quant_attention: query rows must be 16-byte aligned");
  if (accumulate && !cache->weights) return fail(CKV_E_INVALID, "ckv_quant_attention: the cache keeps no weights");
  if ((int64_t)cache->batch * cache->kv_heads > 65535)
    return fail(CKV_E_LIMIT, "ckv_quant_attention: more than 65535 heads over the batch");
  const AttendLayout lay(cache, tokens * group, dtype, accumulate != 0);
  if (lay.bytes && (!workspace || ((uintptr_t)workspace & 15)))
    return fail(CKV_E_INVALID, "ckv_quant_attention: workspace");
  char* ws = reinterpret_cast<char*>(workspace);
  QuantAttendArgs a{};
  a.cache = *cache;
  a.query = *query;
  a.counts = counts;
  a.out = out;
  a.lse = lse;
  a.part_max = reinterpret_cast<float*>(ws + lay.max);
  a.part_sum = reinterpret_cast<float*>(ws + lay.sum);
  a.part_acc = reinterpret_cast<float*>(ws + lay.acc);
  a.stats = accumulate ? reinterpret_cast<float2*>(ws + lay.stats) : nullptr;
  a.ranges = lay.many ? reinterpret_cast<int2*>(ws + lay.ranges) : nullptr;
  a.scores = lay.keep_scores ? reinterpret_cast<float*>(ws + lay.scores) : nullptr;
  a.sums = reinterpret_cast<float*>(ws + lay.sums);
  a.scale_log2 = (float)((double)softmax_scale * 1.4426950408889634);
  a.tokens = tokens;
  a.group = group;
  a.group_magic = group > 1 ? (uint32_t)(((1ull << 32) + group - 1) / group) : 0u;
  a.rows = tokens * group;
  a.row_pad = lay.row_pad;
  a.window = window;
  a.parts = lay.parts;
  const hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  if (dtype == CKV_BF16) return launch_attend<CKV_BF16>(a, lay.many, accumulate != 0, s);
  if (dtype == CKV_F16) return launch_attend<CKV_F16>(a, lay.many, accumulate != 0, s);
  return launch_attend<CKV_F32>(a, lay.many, accumulate != 0, s);
}
