// Attention of a step's tokens over the paged KV cache (gfx950).
//
//   s_r = softmax_scale * (q . k_r),  out = sum_r e^{s_r - lse} v_r,
//
// r over the committed rows and the step's tokens that the query sees.  The
// products run on the matrix cores in the cache's own type with 32-bit sums.
// Maxima, sums and outputs are kept in 32 bits; a probability enters the value
// product rounded to the cache's type (by up to 2^-8 or 2^-11 of it, where the
// sums keep it whole), the same rounding that the result itself gets at the end.
//
// A head's query rows are packed as token * group + query head, so that one
// read of a key or value serves the whole group and all tokens of a tree.
#include <hip/hip_runtime.h>

#include "ckv_paged_attend.h"
#include "ckv_tile.h"

namespace {
using namespace ckv;

constexpr int STEP = 32;  // cache rows a wave takes at a time
constexpr int WAVES = 4;
static_assert(PART_UNIT == WAVES * STEP, "parts are whole rounds of the waves");

template <int DT>
__device__ inline f32x4_t mfma16(uint4 a, uint4 b, f32x4_t c) {
  if constexpr (DT == CKV_BF16) {
    return mfma_bf16(a, b, c);
  } else {
    typedef _Float16 f16x8_t __attribute__((ext_vector_type(8)));
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8_t, a), __builtin_bit_cast(f16x8_t, b), c, 0, 0, 0);
  }
}

// One step's rows of a head, straight from memory into operands: keys as A
// operands (row m of MFMA block j is cache row 8 (m / 4) + 4 j + m % 4 of the
// step, so that an accumulator lane holds the eight rows 8 L .. 8 L + 7, just
// what the P operand of the value product takes), values 8 dims a lane of the
// rows 8 L + u.  Eight rows that stand together share a page.
struct StepRows {
  uint4 k[2][4];
  uint4 v[8];
};

struct StepPages {
  int k, v;  // of this lane's rows
};

__device__ inline StepPages step_pages(const PagedHead& q, int t0, int last) {
  const int lane = threadIdx.x & 63;
  return StepPages{q.page(min(t0 + 8 * ((lane & 15) >> 2), last)), q.page(min(t0 + 8 * (lane >> 4), last))};
}

// Rows past the last one are read as they are in its page, and masked.
__device__ inline void load_step(const PagedHead& q, int t0, const StepPages& pages, StepRows& s) {
  const int lane = threadIdx.x & 63, L = lane >> 4, c = lane & 15;
  const uint16_t* k = q.keys + q.at(pages.k, t0 + 8 * (c >> 2) + (c & 3)) + 8 * L;
#pragma unroll
  for (int j = 0; j < 2; ++j) {
#pragma unroll
    for (int x = 0; x < 4; ++x) s.k[j][x] = gload16(k + 4 * j * D + 32 * x);
  }
  const uint16_t* v = q.values + q.at(pages.v, t0 + 8 * L) + 8 * c;
#pragma unroll
  for (int u = 0; u < 8; ++u) s.v[u] = gload16(v + u * D);
}

__device__ inline uint32_t word_of(const uint4& w, int i) { return i == 0 ? w.x : i == 1 ? w.y : i == 2 ? w.z : w.w; }

// B operands of the value product: for dims 8 c + d, the rows 8 L + u (an 8 x 8
// transposition within the lane).
__device__ inline void value_operands(const uint4* v, uint4* op) {
#pragma unroll
  for (int pair = 0; pair < 4; ++pair) {
    uint32_t lo[4], hi[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const uint32_t a = word_of(v[2 * u], pair), b = word_of(v[2 * u + 1], pair);
      lo[u] = __builtin_amdgcn_perm(b, a, 0x05040100u);
      hi[u] = __builtin_amdgcn_perm(b, a, 0x07060302u);
    }
    op[2 * pair] = uint4{lo[0], lo[1], lo[2], lo[3]};
    op[2 * pair + 1] = uint4{hi[0], hi[1], hi[2], hi[3]};
  }
}

// The running softmax of 16 query rows over the steps of one wave.  m: unscaled
// maximum of query row c, the same on the four lane groups; l: sum over this
// lane's rows alone; o: accumulators, element i of block nb is query row
// 4 L + i, dim 8 c + nb.
struct Running {
  float m, l;
  f32x4_t o[8];
};

template <int DT>
__device__ inline void add_step(const PagedAttendArgs& a, const float* sc, const uint4* vop, Running& r) {
  float top = sc[0];
#pragma unroll
  for (int i = 1; i < 8; ++i) top = fmaxf(top, sc[i]);
  if (__ballot(top - r.m > a.grow_by) != 0) {
    float t = fmaxf(top, xor_f32<16>(top));
    t = fmaxf(t, xor_f32<32>(t));
    t = t - r.m > a.grow_by ? t : r.m;  // a query's own scores alone decide
    const float corr = r.m == t ? 1.0f : __builtin_amdgcn_exp2f((r.m - t) * a.scale_log2);
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
    p[i] = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[i] - m, a.scale_log2, prob_bias<DT>()));
    r.l += p[i];
  }
  const uint4 aop = {pack_store<DT>(p[0], p[1]), pack_store<DT>(p[2], p[3]), pack_store<DT>(p[4], p[5]),
                     pack_store<DT>(p[6], p[7])};
#pragma unroll
  for (int nb = 0; nb < 8; ++nb) r.o[nb] = mfma16<DT>(aop, vop[nb], r.o[nb]);
}

// One workgroup of four waves takes a part of the cache rows of a (sequence,
// head) for 16 RT query rows; its waves take steps in turn and join in LDS.
// Keys and values go from memory into operands without LDS: each is used by one
// wave alone.  Bound by memory on long caches: a token over 8 sequences of up to
// 131k rows, 32/8 heads, in 418 us, 5.8 TB/s, where reading alone reaches 6.1;
// by latency on short ones (one sequence of 300 rows: 7.3 us).  Two tiles of
// query rows share what is read; four spill.
template <int DT, int RT>
__global__ __launch_bounds__(64 * WAVES, 2) void paged_split_kernel(const PagedAttendArgs a) {
  __shared__ float m_s[WAVES][16];
  __shared__ float l_s[WAVES][16];
  __shared__ float o_s[WAVES][16 * D];
  const ckv_paged_cache& c = a.cache;
  const int h = blockIdx.x % c.kv_heads, number = blockIdx.x / c.kv_heads, row0 = 16 * RT * blockIdx.y;
  const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int lane = tid & 63, L = lane >> 4, col = lane & 15;
  const Part part = find_part(PagedRows{a}, a.parts, number, -1);
  const int b = part.sequence;
  if (b < 0) return;  // the join knows how many parts there are
  tell_parts(a, part);
  const int slot = part_slot(part);
  const PagedStep step(a, b);
  const PagedHead q(a, b, h);
  // tokens of this workgroup's rows, and the rows that all and that any of them see
  const int first_token = paged_token(a, row0);
  const int last_token = min(paged_token(a, min(row0 + 16 * RT, a.rows) - 1), step.count - 1);
  int begin = step.first(a) + part.index * part.rows;
  int end = (int)min((int64_t)begin + part.rows, (int64_t)step.total);
  int clear_hi = step.start - 1, clear_lo = 0;
  if (!a.masks) {
    clear_hi = step.start + first_token;
    end = min(end, step.start + last_token + 1);
    if (a.window > 0) begin = max(begin, max(step.start + first_token - a.window + 1, 0) & -PART_UNIT);
  }
  if (a.window > 0 && !a.masks) clear_lo = step.start + last_token - a.window + 1;
  if (first_token >= step.count) end = begin;
  clear_hi = min(clear_hi, step.total - 1);

  uint4 query[RT][4];
  Running run[RT];
#pragma unroll
  for (int r = 0; r < RT; ++r) {
    const int64_t from = paged_query_index(a, b, h, min(row0 + 16 * r + col, a.rows - 1));
#pragma unroll
    for (int x = 0; x < 4; ++x)
      query[r][x] = gload16(reinterpret_cast<const uint16_t*>(a.query.data) + from + 32 * x + 8 * L);
    run[r].m = NEG_INF;
    run[r].l = 0.0f;
#pragma unroll
    for (int nb = 0; nb < 8; ++nb) run[r].o[nb] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
  }
  Sight sight[RT];
#pragma unroll
  for (int r = 0; r < RT; ++r) sight[r] = Sight(a, step, b, row0 + 16 * r + col);
  if (a.window > 0 && a.masks) clear_lo = wave_newest_lo(sight);
  const int last = step.total - 1;
  auto add = [&](StepRows& rows, const StepPages& pages, int t0) __attribute__((always_inline)) {
    const bool bad = __ballot(!q.good(pages.k) || !q.good(pages.v)) != 0;
    const bool good_rows = q.good(pages.v);
    const bool masked = bad || t0 < clear_lo || t0 + STEP - 1 > clear_hi;
    bool special = false;
    if (masked) {  // a masked row's zero probability times infinity or NaN would spread it
      bool found = false;
#pragma unroll
      for (int u = 0; u < 8; ++u) {
#pragma unroll
        for (int i = 0; i < 4; ++i) found |= has_special<DT>(word_of(rows.v[u], i));
      }
      special = __ballot(found) != 0;
      if (special) {
#pragma unroll
        for (int u = 0; u < 8; ++u)
          rows.v[u] = uint4{without_special<DT>(rows.v[u].x), without_special<DT>(rows.v[u].y),
                            without_special<DT>(rows.v[u].z), without_special<DT>(rows.v[u].w)};
      }
    }
    uint4 vop[8];
    value_operands(rows.v, vop);
    uint32_t seen[RT];
#pragma unroll
    for (int r = 0; r < RT; ++r) {
      float sc[8];
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        f32x4_t acc = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int x = 0; x < 4; ++x) acc = mfma16<DT>(rows.k[j][x], query[r][x], acc);
#pragma unroll
        for (int i = 0; i < 4; ++i) sc[4 * j + i] = acc[i];
      }
      if (masked) {
        seen[r] = good_rows ? (uint32_t)sight[r].rows(a, step, b, t0 + 8 * L) & 0xffu : 0u;
#pragma unroll
        for (int i = 0; i < 8; ++i) sc[i] = (seen[r] >> i) & 1 ? sc[i] : NEG_INF;
      }
      add_step<DT>(a, sc, vop, run[r]);
    }
    if (special) {
      // values that were taken as zeros above, added for the queries that see their row
#pragma nounroll
      for (int g = 0; g < 4; ++g) {
        const int page = q.page(min(t0 + 8 * g, last));
        const uint16_t* from = q.values + q.at(page, t0 + 8 * g) + 8 * col;
#pragma nounroll
        for (int u = 0; u < 8; ++u) {
          const uint4 w = gload16(from + u * D);
          float x[8];
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            x[2 * i] = special_value<DT>(word_of(w, i) & 0xffffu);
            x[2 * i + 1] = special_value<DT>(word_of(w, i) >> 16);
          }
#pragma unroll
          for (int r = 0; r < RT; ++r) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const uint32_t sees = (uint32_t)__shfl((int)seen[r], 16 * g + 4 * L + i, 64) >> u & 1u;
#pragma unroll
              for (int nb = 0; nb < 8; ++nb) run[r].o[nb][i] += sees ? x[nb] : 0.0f;
            }
          }
        }
      }
    }
  };
  // A step's pages are read a step ahead.  (Reading its rows ahead too, into a second set of registers, changes nothing:
  // two waves a SIMD have enough in flight.)
  constexpr int STRIDE = WAVES * STEP;
  int t0 = begin + wave * STEP;
  StepPages pages{0, 0};
  if (t0 < end) pages = step_pages(q, t0, last);
  for (; t0 < end; t0 += STRIDE) {
    StepRows rows;
    load_step(q, t0, pages, rows);
    const StepPages of = pages;
    if (t0 + STRIDE < end) pages = step_pages(q, t0 + STRIDE, last);
    add(rows, of, t0);
  }
  // join the waves, 16 query rows at a time
#pragma unroll
  for (int r = 0; r < RT; ++r) {
    const int at0 = row0 + 16 * r;
    float l = add_xor16(run[r].l);
    l = add_xor32(l);
    __syncthreads();
    if (L == 0) {
      m_s[wave][col] = run[r].m;
      l_s[wave][col] = l;
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      float4* p = reinterpret_cast<float4*>(&o_s[wave][(4 * L + i) * D + 8 * col]);
      p[0] = float4{run[r].o[0][i], run[r].o[1][i], run[r].o[2][i], run[r].o[3][i]};
      p[1] = float4{run[r].o[4][i], run[r].o[5][i], run[r].o[6][i], run[r].o[7][i]};
    }
    __syncthreads();
    // 16 threads a query row, eight dims each
    const int i = tid >> 4, d = 8 * (tid & 15), row = at0 + i;
    if (row >= a.rows) continue;
    float m = m_s[0][i];
#pragma unroll
    for (int w = 1; w < WAVES; ++w) m = fmaxf(m, m_s[w][i]);
    const float at = m == NEG_INF ? 0.0f : m;
    float sum = 0.0f, acc[8] = {};
#pragma unroll
    for (int w = 0; w < WAVES; ++w) {
      // a wave without a row has zeros and a maximum of -inf
      const float f = __builtin_amdgcn_exp2f((m_s[w][i] - at) * a.scale_log2);
      const float4 x = *reinterpret_cast<const float4*>(&o_s[w][i * D + d]), y = *reinterpret_cast<const float4*>(&o_s[w][i * D + d + 4]);
      sum += l_s[w][i] * f;
      const float v[8] = {x.x, x.y, x.z, x.w, y.x, y.y, y.z, y.w};
#pragma unroll
      for (int e = 0; e < 8; ++e) acc[e] += v[e] * f;
    }
    if (paged_token(a, row) >= step.count) {  // no token
      m = NEG_INF;
      sum = 0.0f;
#pragma unroll
      for (int e = 0; e < 8; ++e) acc[e] = 0.0f;
    }
    if (slot < 0) {
      int64_t at_out, at_lse;
      paged_output_index(a, b, h, row, &at_out, &at_lse);
      const float scale = sum == 0.0f ? 0.0f : 1.0f / sum;
#pragma unroll
      for (int e = 0; e < 8; ++e) acc[e] = sum == 0.0f ? 0.0f : acc[e] * scale;
      *reinterpret_cast<uint4*>(reinterpret_cast<uint16_t*>(a.out) + at_out + d) =
          uint4{pack_store<DT>(acc[0], acc[1]), pack_store<DT>(acc[2], acc[3]), pack_store<DT>(acc[4], acc[5]),
                pack_store<DT>(acc[6], acc[7])};
      if (d == 0) a.lse[at_lse] = paged_lse<DT>(a, m, sum);
    } else {
      float4* to = reinterpret_cast<float4*>(a.part_acc + (((int64_t)h * a.slots + slot) * a.row_pad + row) * D + d);
      to[0] = float4{acc[0], acc[1], acc[2], acc[3]};
      to[1] = float4{acc[4], acc[5], acc[6], acc[7]};
      if (d == 0) {
        a.part_max[((int64_t)h * a.row_pad + row) * a.slots + slot] = m;
        a.part_sum[((int64_t)h * a.row_pad + row) * a.slots + slot] = sum;
      }
    }
  }
}

// Joins the parts of one query row: a workgroup of 256 threads, four dims and
// every eighth part each.  Heads run along the grid's first dimension as they do
// in the kernels that wrote the parts, so where their number is a multiple of
// eight an XCD reads what its own compute units wrote (one sequence, 512 queries
// over 2k rows: 39.4 us against 42.0 for the call with rows first).
constexpr int JOIN_THREADS = 256;
constexpr int MAX_PARTS = 512;  // of one sequence

template <int DT>
__global__ __launch_bounds__(JOIN_THREADS) void paged_join_kernel(const PagedAttendArgs a) {
  __shared__ float factor[MAX_PARTS];
  __shared__ float scratch[4];
  __shared__ float4 acc_s[JOIN_THREADS];
  const int h = blockIdx.x, row = blockIdx.y, b = blockIdx.z, tid = threadIdx.x;
  const int2 part = a.part_of[b];  // the first one's slot and their number
  if (part.y == 1) return;  // written already
  const int64_t first = ((int64_t)h * a.row_pad + row) * a.slots + part.x;
  const float *pm = a.part_max + first, *pl = a.part_sum + first;
  float m = NEG_INF;
  for (int s = tid & 63; s < part.y; s += 64) m = fmaxf(m, pm[s]);
  m = wave_max(m);  // every wave for itself
  const float at = m == NEG_INF ? 0.0f : m;
  float sum = 0.0f;
  for (int s = tid; s < part.y; s += JOIN_THREADS) {
    const float f = __builtin_amdgcn_exp2f((pm[s] - at) * a.scale_log2);
    factor[s] = f;
    sum += pl[s] * f;
  }
  sum = wave_sum_tree(sum);
  if ((tid & 63) == 0) scratch[tid >> 6] = sum;
  __syncthreads();
  sum = (scratch[0] + scratch[1]) + (scratch[2] + scratch[3]);
  const int dim = 4 * (tid & 31);
  float4 acc{0.0f, 0.0f, 0.0f, 0.0f};
  const float* pa = a.part_acc + (((int64_t)h * a.slots + part.x) * a.row_pad + row) * D + dim;
#pragma unroll 4
  for (int s = tid >> 5; s < part.y; s += JOIN_THREADS / 32) {
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
  paged_output_index(a, b, h, row, &at_out, &at_lse);
  if (tid < D) {
    float x = 0.0f;
#pragma unroll
    for (int g = 0; g < JOIN_THREADS / 32; ++g) x += reinterpret_cast<const float*>(acc_s)[g * D + tid];
    store_value<DT>(a.out, at_out + tid, sum == 0.0f ? 0.0f : x / sum);
  }
  if (tid == 0) a.lse[at_lse] = paged_lse<DT>(a, m, sum);
}

// The same for many query rows, of few parts mostly: half a wave a row, four dims a lane; the first parts' outputs are
// read along with their maxima.
template <int DT>
__global__ __launch_bounds__(JOIN_THREADS) void paged_join_rows_kernel(const PagedAttendArgs a) {
  constexpr int TOGETHER = 4;  // parts in flight
  const int h = blockIdx.x, row = (JOIN_THREADS / 32) * blockIdx.y + (threadIdx.x >> 5), b = blockIdx.z, lane = threadIdx.x & 31;
  if (row >= a.rows) return;
  const int2 part = a.part_of[b];
  if (part.y == 1) return;
  const int64_t first = ((int64_t)h * a.row_pad + row) * a.slots + part.x;
  const float *pm = a.part_max + first, *pl = a.part_sum + first;
  const float* pa = a.part_acc + (((int64_t)h * a.slots + part.x) * a.row_pad + row) * D + 4 * lane;
  const int64_t stride = (int64_t)a.row_pad * D;
  float m = NEG_INF, sum = 0.0f;
  float4 acc{0.0f, 0.0f, 0.0f, 0.0f};
  for (int s0 = 0; s0 < part.y; s0 += TOGETHER) {
    float ms[TOGETHER], ls[TOGETHER];
    float4 xs[TOGETHER];
    const int left = part.y - s0;
#pragma unroll
    for (int i = 0; i < TOGETHER; ++i) {
      const int s = s0 + min(i, left - 1);
      xs[i] = *reinterpret_cast<const float4*>(pa + s * stride);
      ms[i] = pm[s];
      ls[i] = pl[s];
    }
    float top = m;
#pragma unroll
    for (int i = 0; i < TOGETHER; ++i) top = fmaxf(top, ms[i]);
    const float at = top == NEG_INF ? 0.0f : top, before = __builtin_amdgcn_exp2f((m - at) * a.scale_log2);
    m = top;
    sum *= before;
    acc = float4{acc.x * before, acc.y * before, acc.z * before, acc.w * before};
#pragma unroll
    for (int i = 0; i < TOGETHER; ++i) {
      if (i >= left) break;
      const float f = __builtin_amdgcn_exp2f((ms[i] - at) * a.scale_log2);
      sum += ls[i] * f;
      acc.x += xs[i].x * f;
      acc.y += xs[i].y * f;
      acc.z += xs[i].z * f;
      acc.w += xs[i].w * f;
    }
  }
  int64_t at_out, at_lse;
  paged_output_index(a, b, h, row, &at_out, &at_lse);
  const float scale = sum == 0.0f ? 0.0f : 1.0f / sum;
  const float4 x = sum == 0.0f ? float4{0.0f, 0.0f, 0.0f, 0.0f} : float4{acc.x * scale, acc.y * scale, acc.z * scale, acc.w * scale};
  *reinterpret_cast<uint2*>(reinterpret_cast<uint16_t*>(a.out) + at_out + 4 * lane) =
      uint2{pack_store<DT>(x.x, x.y), pack_store<DT>(x.z, x.w)};
  if (lane == 0) a.lse[at_lse] = paged_lse<DT>(a, m, sum);
}

constexpr int64_t MAX_ROWS = 1 << 21;  // query rows of a head: the grids' second dimension holds their blocks

// Which kernel, by the call's work: cache rows times blocks of 16 query rows, over all heads and sequences.  Times of the
// attention alone, one tile | two tiles | many rows, on heads of 32/8 unless said:
//   136k (8/8 heads, 128 tokens, 2k rows)              15.7 | 17.5 | 20.4 us
//   256k (64 query rows, 8k cache rows)                20.4 | 18.5 | 22.0
//   544k (512 query rows, 2k cache rows)               27.8 | 24.3 | 30.2
//   848k (4 sequences, 512 query rows, 700 cache rows)  38.3 | 27.4 | 30.2
//   1,032k (256 query rows, 8k cache rows)             50.0 | 36.0 | 29.3
// Up to 16 query rows one tile holds all, and up to 32 two do: the many-row kernel's tile would be empty mostly (8
// sequences, 32 query rows, 32k cache rows: 194 us against 214).
constexpr int64_t FEW_WORK = 850000, ONE_TILE_WORK = 200000;

// Workgroups that parts are cut for.  A workgroup a compute unit, for parts cost a join (two tiles, 32 query rows, one
// sequence of 32k: 31.5 us against 33.2 with two, 39.9 with four); two where a wave hides another's waits: one tile over
// long caches (8 sequences of 32k: 191 us against 200; of 8k, below the limit: 57 against 54) and the many-row kernel of
// 128 rows, of which two fit a compute unit (72 us against 74; 256 rows: 105 against 93).
constexpr int64_t LONG_WORK = 700000;

// How a call is laid out: which kernel, how many parts, and the workspace.
struct PagedLayout {
  int parts, slots, row_pad, tiles;  // tiles of 16 query rows a workgroup of the few-row kernel, 0: the many-row kernel
  bool wide_join;
  size_t max, sum, acc, of, bytes;
  PagedLayout(const ckv_paged_cache* c, int tokens, int group, int window) {
    const int rows = tokens * group;
    row_pad = (rows + 15) / 16 * 16;
    int64_t most = (int64_t)c->table_pages * c->page_size;  // rows that a sequence's tokens may see
    if (window > 0 && (int64_t)window + tokens + 2 * PART_UNIT < most) most = (int64_t)window + tokens + 2 * PART_UNIT;
    const int64_t work = (int64_t)c->batch * c->kv_heads * (row_pad / 16) * most;
    tiles = rows <= 16 || work <= ONE_TILE_WORK ? 1 : rows <= 32 || work <= FEW_WORK ? 2 : 0;
    const int64_t block = tiles ? 16 * tiles : paged_row_block(rows);
    const int64_t blocks = (rows + block - 1) / block;
    const int64_t units = (most + PART_UNIT - 1) / PART_UNIT;
    const int64_t workgroups = (tiles == 1 && work > LONG_WORK) || (!tiles && block == 128) ? 512 : 256;
    const int64_t want = workgroups / (c->kv_heads * blocks);
    // A sequence stays whole where a join costs more than it saves: up to 512 rows for a token or two (380 rows: 8.3 us
    // whole, 9.0 cut; 640: 9.9, 8.7), 768 for a small tree (640 rows: 13.5, 13.8; 890: 15.8, 12.8), 128 for many rows (250
    // rows, 8 sequences: 16 us, 25; 380, one sequence: 16.6, 14.4).
    if (units <= (!tiles ? 1 : rows <= 16 ? 4 : 6)) parts = c->batch;
    else if (want >= (tiles ? c->batch + 1 : 2 * c->batch)) parts = (int)(want < c->batch * units ? want : c->batch * units);
    // A batch that fills the chip with whole sequences gets half as many parts again, so that one long sequence among short
    // ones is cut all the same (equal ones stay whole).  64 sequences, 32/8 heads, a token each: 1,396 us -> 164 with one of
    // 131k rows among ones of 1,000, 512 -> 458 with 1k to 16k rows, for 181 -> 188 with 4,000 rows in each; 24 trees of 64
    // tokens: 379 -> 310 with 1k to 16k rows, 257 either way with 8,000.
    else parts = c->batch + (want >= 2 && units > 32 ? (int)(want < c->batch / 2 ? want : c->batch / 2) : 0);
    // A workgroup a query row joins faster than half a wave a row that reads the parts in turn where the parts are many
    // and the rows few.  Rows of all heads and sequences, parts of a sequence, half waves | workgroups, in us of the whole
    // call: 384, 5: 77.1 | 76.4;  128, 32: 27 | 18;  2,048, 32: 39 | 30;  4,096, 16: 40.5 | 38.6;  5,120, 13: 42 | 43;
    // 8,192, 8: 55 | 60.
    wide_join = parts > 4 * c->batch && (int64_t)rows * c->kv_heads * c->batch <= 4096;
    size_t at = 0;
    auto take = [&](size_t size) {
      const size_t here = at;
      at += (size + 15) & ~(size_t)15;
      return here;
    };
    slots = part_slots(parts, c->batch);
    const size_t each = (size_t)c->kv_heads * row_pad * slots * sizeof(float);
    max = take(each);
    sum = take(each);
    acc = take(each * D);
    of = take(each ? c->batch * sizeof(int2) : 0);
    bytes = at;
  }
};

template <int DT>
int launch_few(const PagedAttendArgs& a, int tiles, hipStream_t s) {
  const dim3 grid(a.parts * a.cache.kv_heads, (a.rows + 16 * tiles - 1) / (16 * tiles));
  if (tiles == 1) paged_split_kernel<DT, 1><<<grid, 64 * WAVES, 0, s>>>(a);
  else paged_split_kernel<DT, 2><<<grid, 64 * WAVES, 0, s>>>(a);
  return paged_launched("ckv_paged_attention");
}

template <int DT>
int launch_attend(const PagedAttendArgs& a, const PagedLayout& lay, hipStream_t s) {
  const int rc = lay.tiles ? launch_few<DT>(a, lay.tiles, s) : launch_paged_rows(a, s);
  if (rc || a.parts == a.cache.batch) return rc;
  if (lay.wide_join) paged_join_kernel<DT><<<dim3(a.cache.kv_heads, a.rows, a.cache.batch), JOIN_THREADS, 0, s>>>(a);
  else paged_join_rows_kernel<DT><<<dim3(a.cache.kv_heads, (a.rows + 7) / 8, a.cache.batch), JOIN_THREADS, 0, s>>>(a);
  return paged_launched("ckv_paged_attention");
}

}  // namespace

extern "C" size_t ckv_paged_attention_workspace_bytes(const ckv_paged_cache* cache, int32_t query_heads, int32_t tokens,
                                                      int32_t window) {
  if (validate_paged_cache(cache, "ckv_paged_attention") || tokens <= 0 || query_heads <= 0 ||
      query_heads % cache->kv_heads || window < 0)
    return 0;
  const int64_t group = query_heads / cache->kv_heads;
  if (tokens * group > MAX_ROWS) return 0;
  return PagedLayout(cache, tokens, (int)group, window).bytes;
}

extern "C" int ckv_paged_attention(const ckv_paged_cache* cache, const ckv_paged_attention_args* args, void* stream) {
  const char* what = "ckv_paged_attention";
  int rc = validate_paged_cache(cache, what);
  if (rc) return rc;
  if (!args) return paged_error(CKV_E_INVALID, what, "null argument");
  const int layer = args->layer, query_heads = args->query_heads, tokens = args->tokens, window = args->window;
  const ckv_draft_tree* tree = args->tree;
  if (layer < 0 || layer >= cache->layers) return paged_error(CKV_E_INVALID, what, "no such layer");
  if (!args->out || ((uintptr_t)args->out & 15) || !args->lse) return paged_error(CKV_E_INVALID, what, "null argument");
  rc = check_paged_rows(&args->query, cache->dtype, what);
  if (rc) return rc;
  if (query_heads <= 0 || query_heads % cache->kv_heads)
    return paged_error(CKV_E_INVALID, what, "query heads must be a multiple of the cache's heads");
  const int group = query_heads / cache->kv_heads;
  if (group > CKV_MAX_GROUP) return paged_error(CKV_E_LIMIT, what, "group size exceeds 16");
  if (tokens <= 0 || window < 0) return paged_error(CKV_E_INVALID, what, "tokens must be positive, window not negative");
  if ((int64_t)tokens * group > MAX_ROWS) return paged_error(CKV_E_LIMIT, what, "more than 2^21 query rows a head");
  if (tree && (!tree->depths || !tree->masks)) return paged_error(CKV_E_INVALID, what, "null argument");
  if (tree && tokens > CKV_MAX_DRAFT) return paged_error(CKV_E_LIMIT, what, "a tree of more than 512 tokens");
  // below, the step that a running maximum makes would not be a number in 32 bits
  if (!(args->softmax_scale >= 0.99e-30f) || args->softmax_scale > 1.01e30f)
    return paged_error(CKV_E_INVALID, what, "softmax_scale must be between 1e-30 and 1e30");
  const PagedLayout lay(cache, tokens, group, window);
  if (lay.bytes && (!args->workspace || ((uintptr_t)args->workspace & 15))) return paged_error(CKV_E_INVALID, what, "workspace");
  char* ws = reinterpret_cast<char*>(args->workspace);
  PagedAttendArgs a{};
  a.cache = *cache;
  const size_t layer_bytes = (size_t)cache->pages * cache->kv_heads * cache->page_size * D * 2;
  a.cache.key_pages = reinterpret_cast<char*>(cache->key_pages) + layer * layer_bytes;
  a.cache.value_pages = reinterpret_cast<char*>(cache->value_pages) + layer * layer_bytes;
  a.query = args->query;
  a.counts = args->counts;
  a.depths = tree ? tree->depths : nullptr;
  a.masks = tree ? tree->masks : nullptr;
  a.out = args->out;
  a.lse = args->lse;
  a.part_max = reinterpret_cast<float*>(ws + lay.max);
  a.part_sum = reinterpret_cast<float*>(ws + lay.sum);
  a.part_acc = reinterpret_cast<float*>(ws + lay.acc);
  a.part_of = reinterpret_cast<int2*>(ws + lay.of);
  a.scale_log2 = (float)((double)args->softmax_scale * 1.4426950408889634);
  a.grow_by = (float)((double)PAGED_RESCALE / (double)a.scale_log2);
  a.tokens = tokens;
  a.group = group;
  a.group_magic = group > 1 ? (uint32_t)(((1ull << 32) + group - 1) / group) : 0u;
  a.rows = tokens * group;
  a.row_pad = lay.row_pad;
  a.window = window;
  a.parts = lay.parts;
  a.slots = lay.slots;
  a.words = (tokens + 63) / 64;
  a.page_log2 = 31 - __builtin_clz((unsigned)cache->page_size);
  const hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  if (cache->dtype == CKV_BF16) return launch_attend<CKV_BF16>(a, lay, s);
  return launch_attend<CKV_F16>(a, lay, s);
}
