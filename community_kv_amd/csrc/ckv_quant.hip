// Writing into the 8-bit KV cache, and eviction from it (gfx950).
//
// append_kernel: a workgroup of 256 threads owns one block of rows of one
// sequence, head and tensor (key or value): 16 threads a row, 8 values each.
// It reads its new rows once into registers, takes the block's largest
// magnitude, settles the scale, and writes codes of 8 bytes a thread (a row of
// 128 bytes by 16 neighbouring threads).  Earlier rows of the block are touched
// only when the scale grows.  The last workgroup of a sequence moves its
// cursors: every workgroup has read them by then.
#include <hip/hip_runtime.h>

#include <stdio.h>

#include "ckv_quant.h"

namespace ckv {

int validate_quant_cache(const ckv_quant_cache* c, const char* what) {
  static thread_local char message[160];
  auto fail = [&](int code, const char* why) {
    snprintf(message, sizeof(message), "%s: %s", what, why);
    return ckv_internal::set_error(code, message);
  };
  if (!c || !c->key_codes || !c->value_codes || !c->key_scales || !c->value_scales || !c->positions || !c->cursors ||
      !c->counters)
    return fail(CKV_E_INVALID, "null argument");
  if (c->batch <= 0 || c->kv_heads <= 0 || c->capacity <= 0)
    return fail(CKV_E_INVALID, "batch, kv_heads and capacity must be positive");
  if (c->block != 16 && c->block != 32 && c->block != 64 && c->block != 128)
    return fail(CKV_E_INVALID, "block must be 16, 32, 64 or 128");
  if (c->capacity % c->block) return fail(CKV_E_INVALID, "capacity must be a multiple of block");
  if (c->capacity > (1 << 30)) return fail(CKV_E_LIMIT, "capacity above 2^30 rows");
  if (c->batch > 32767 || c->kv_heads > 32767) return fail(CKV_E_LIMIT, "batch or kv_heads above 32767");
  if (((uintptr_t)c->key_codes | (uintptr_t)c->value_codes) & 15)
    return fail(CKV_E_INVALID, "codes must be 16-byte aligned");
  return CKV_OK;
}

}  // namespace ckv

namespace {
using namespace ckv;

constexpr int THREADS = 256;

int fail(int code, const char* message) { return ckv_internal::set_error(code, message); }

int launched(const char* what) {
  const hipError_t e = hipGetLastError();
  if (e == hipSuccess) return CKV_OK;
  static thread_local char message[160];
  snprintf(message, sizeof(message), "%s: %s", what, hipGetErrorString(e));
  return fail(CKV_E_LAUNCH, message);
}

template <int DT>
__device__ inline void load_new8(const void* base, int64_t index, float* out) {
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

// Multiplies the codes of the block's rows [row0, row0 + rows) by `ratio`.
__device__ inline void rescale_rows(uint8_t* codes, int64_t row0, int rows, float ratio) {
  const int col = (threadIdx.x & 15) * 8;
  for (int r = threadIdx.x >> 4; r < rows; r += THREADS / 16) {
    uint2* p = reinterpret_cast<uint2*>(codes + (row0 + r) * D + col);
    const uint2 w = *p;
    float v[8];
    decode4(w.x, v);
    decode4(w.y, v + 4);
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] *= ratio;
    *p = uint2{encode4(v[0], v[1], v[2], v[3]), encode4(v[4], v[5], v[6], v[7])};
  }
}

struct AppendArgs {
  ckv_quant_cache cache;
  ckv_quant_rows key, value;
  const int32_t* counts;
  int32_t tokens;
};

template <int DT, int SWEEPS>
__global__ __launch_bounds__(THREADS) void append_kernel(const AppendArgs a) {
  constexpr int BLOCK = 16 * SWEEPS;
  __shared__ float scratch[4];
  const ckv_quant_cache& c = a.cache;
  const int b = blockIdx.z >> 1, tensor = blockIdx.z & 1, h = blockIdx.y;
  const int start = quant_length(c, b), seen = c.cursors[c.batch + b];
  const int count = a.counts ? min(max(a.counts[b], 0), a.tokens) : a.tokens;
  const int end = (int)min((int64_t)start + count, (int64_t)c.capacity);
  const int64_t blk = start / BLOCK + (int64_t)blockIdx.x;
  const int64_t row0 = blk * BLOCK;
  const int lo = (int)max((int64_t)start, row0), hi = (int)min((int64_t)end, row0 + BLOCK);
  if (lo < hi && row0 < c.capacity) {
    const QuantHead q = quant_head(c, b, h);
    const ckv_quant_rows in = tensor ? a.value : a.key;
    const int64_t base = (int64_t)b * in.batch_stride + (int64_t)h * in.head_stride;
    const int tid = threadIdx.x, col = (tid & 15) * 8;
    float v[SWEEPS][8];
    float amax = 0.0f;
#pragma unroll
    for (int s = 0; s < SWEEPS; ++s) {
      const int row = (int)row0 + 16 * s + (tid >> 4);
      if (row >= lo && row < hi) load_new8<DT>(in.data, base + (int64_t)(row - start) * in.token_stride + col, v[s]);
    }
#pragma unroll
    for (int s = 0; s < SWEEPS; ++s) {
      const int row = (int)row0 + 16 * s + (tid >> 4);
      if (row >= lo && row < hi) {
#pragma unroll
        for (int i = 0; i < 8; ++i) amax = fmaxf(amax, finite_abs(v[s][i]));
      }
    }
    amax = block_max256(amax, scratch);
    const float old = row0 < start ? q.scales(tensor)[blk] : 0.0f;
    const float scale = fmaxf(old, block_scale(amax));
    const float inv = inverse_scale(scale);
#pragma unroll
    for (int s = 0; s < SWEEPS; ++s) {
      const int row = (int)row0 + 16 * s + (tid >> 4);
      if (row >= lo && row < hi) {
        float y[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) y[i] = v[s][i] * inv;
        *reinterpret_cast<uint2*>(q.codes(tensor) + (int64_t)row * D + col) =
            uint2{encode4(y[0], y[1], y[2], y[3]), encode4(y[4], y[5], y[6], y[7])};
      }
    }
    if (row0 < start && scale != old) rescale_rows(q.codes(tensor), row0, start - (int)row0, old * inv);
    if (tensor == 0) {
      for (int row = lo + tid; row < hi; row += THREADS) {
        q.positions[row] = seen + (row - start);
        if (q.weights) q.weights[row] = 0.0f;
      }
    }
    __syncthreads();  // every wave has read the old scale
    if (tid == 0 && scale != old) q.scales(tensor)[blk] = scale;
  } else {
    __syncthreads();
  }
  // Two counters in a row, so that a long prompt's workgroups do not all meet
  // at one address.
  if (threadIdx.x == 0) {
    uint32_t* head = c.counters + (int64_t)b * (c.kv_heads + 1) + h;
    uint32_t* sequence = c.counters + (int64_t)b * (c.kv_heads + 1) + c.kv_heads;
    if (atomicAdd(head, 1u) == 2 * gridDim.x - 1) {
      st_agent_u32(head, 0u);
      if (atomicAdd(sequence, 1u) == (uint32_t)c.kv_heads - 1) {
        st_agent_u32(sequence, 0u);
        c.cursors[b] = end;
        c.cursors[c.batch + b] = seen + (end - start);
        if ((int64_t)start + count > c.capacity) c.cursors[2 * c.batch + b] = 1;
      }
    }
  }
}

template <int DT>
int launch_append(const AppendArgs& a, hipStream_t stream) {
  const int block = a.cache.block;
  // a count of `tokens` rows from any start touches at most this many blocks
  const int64_t blocks = min((int64_t)(a.tokens - 1) / block + 2, (int64_t)a.cache.capacity / block);
  const dim3 grid((uint32_t)blocks, a.cache.kv_heads, 2 * a.cache.batch);
  if (block == 16) append_kernel<DT, 1><<<grid, THREADS, 0, stream>>>(a);
  else if (block == 32) append_kernel<DT, 2><<<grid, THREADS, 0, stream>>>(a);
  else if (block == 64) append_kernel<DT, 4><<<grid, THREADS, 0, stream>>>(a);
  else append_kernel<DT, 8><<<grid, THREADS, 0, stream>>>(a);
  return launched("ckv_quant_append");
}

// ---------------------------------------------------------------------------
// Eviction
// ---------------------------------------------------------------------------

// Workspace of one (sequence, head), in 32-bit words: two saved scales of the
// block that holds row `keep`, then the row count before, then the keys of
// every row, the kept rows from `keep` on (ascending), and for every 32 rows
// below `keep` the mask of freed rows and their number before.
struct EvictLayout {
  int64_t keys, movers, holes, base, words;
  __host__ __device__ EvictLayout(int64_t capacity, int64_t keep) {
    const int64_t groups = (keep + 31) / 32;
    keys = 4;
    movers = keys + capacity;
    holes = movers + keep;
    base = holes + groups;
    words = (base + groups + 3) & ~(int64_t)3;
  }
};

struct EvictArgs {
  ckv_quant_cache from, to;
  uint32_t* workspace;
  int32_t keep, num_sink, recent;
};

// Eviction order as an unsigned number: protected rows above NaN above the
// weights by value (-0 and 0 alike).
__device__ inline uint32_t evict_key(float w, bool is_protected) {
  if (is_protected) return 0xffffffffu;
  if (w != w) return 0xfffffffeu;
  return ordered_f32(w + 0.0f);
}

constexpr int SEL_THREADS = 1024;
constexpr int SEL_WAVES = SEL_THREADS / 64;

// Exclusive scan of x over the workgroup, and its total.
__device__ inline int scan1024(int x, int* total, int* scratch) {
  const int incl = wave_inclusive_scan(x);
  const int wave = threadIdx.x >> 6;
  __syncthreads();
  if ((threadIdx.x & 63) == 63) scratch[wave] = incl;
  __syncthreads();
  int before = 0, sum = 0;
#pragma unroll
  for (int w = 0; w < SEL_WAVES; ++w) {
    const int v = scratch[w];
    if (w < wave) before += v;
    sum += v;
  }
  *total = sum;
  return before + incl - x;
}

// One workgroup a (sequence, head): the keys once, then the `keep`-th largest
// by four passes over their bytes, then one pass in row order that takes ties
// by the lower row and lists the freed rows below `keep` and the kept ones above.
__global__ __launch_bounds__(SEL_THREADS) void evict_select_kernel(const EvictArgs a) {
  __shared__ int hist[256];
  __shared__ int scratch[SEL_WAVES];
  __shared__ int found[2];
  const ckv_quant_cache& c = a.from;
  const int h = blockIdx.x, b = blockIdx.y, tid = threadIdx.x;
  const int n = quant_length(c, b), seen = c.cursors[c.batch + b];
  const QuantHead q = quant_head(c, b, h);
  const EvictLayout lay(c.capacity, a.keep);
  uint32_t* ws = a.workspace + ((int64_t)b * c.kv_heads + h) * lay.words;
  if (tid == 0) {
    const int64_t blk = a.keep / c.block;
    const bool inside = a.keep < c.capacity;
    ws[0] = inside ? __float_as_uint(q.key_scales[blk]) : 0u;
    ws[1] = inside ? __float_as_uint(q.value_scales[blk]) : 0u;
    ws[2] = (uint32_t)n;
  }
  if (n <= a.keep) return;
  uint32_t* keys = ws + lay.keys;
  const int64_t newest = (int64_t)seen - a.recent;
  for (int i = tid; i < n; i += SEL_THREADS) {
    const int p = q.positions[i];
    keys[i] = evict_key(q.weights[i], p < a.num_sink || p >= newest);
  }
  __syncthreads();
  uint32_t prefix = 0, mask = 0;
  int target = a.keep;  // how many of the rows that match the prefix are kept
  for (int shift = 24; shift >= 0; shift -= 8) {
    if (tid < 256) hist[tid] = 0;
    __syncthreads();
    for (int i = tid; i < n; i += SEL_THREADS) {
      const uint32_t k = keys[i];
      if ((k & mask) == prefix) atomicAdd(&hist[(k >> shift) & 255u], 1);
    }
    __syncthreads();
    if (tid < 64) find_threshold_bin(hist, target, &found[0], &found[1]);
    __syncthreads();
    prefix |= (uint32_t)found[0] << shift;
    mask |= 255u << shift;
    target -= found[1];
    __syncthreads();
  }
  // in row order: `ties` of the rows at the threshold so far, `above` kept rows from keep on, `freed` rows below it
  uint32_t* movers = ws + lay.movers;
  uint32_t* holes = ws + lay.holes;
  uint32_t* base = ws + lay.base;
  int ties = 0, above = 0, freed = 0;
  for (int64_t i0 = 0; i0 < n; i0 += SEL_THREADS) {
    const int64_t i = i0 + tid;
    const uint32_t k = i < n ? keys[i] : 0u;
    const bool tie = i < n && k == prefix;
    int total;
    const int rank = scan1024(tie, &total, scratch);
    const bool kept = i < n && (k > prefix || (tie && ties + rank < target));
    ties += total;
    const bool hole = i < a.keep && !kept;
    const bool mover = i >= a.keep && kept;
    const int at = scan1024((mover ? 1 << 16 : 0) | (hole ? 1 : 0), &total, scratch);
    if (mover) movers[above + (at >> 16)] = (uint32_t)i;
    const uint64_t ballot = __ballot(hole);
    if ((tid & 31) == 0 && i < a.keep) {
      holes[i >> 5] = (uint32_t)(ballot >> (tid & 32));
      base[i >> 5] = (uint32_t)(freed + (at & 0xffff));
    }
    above += total >> 16;
    freed += total & 0xffff;
  }
}

// A workgroup writes one block of rows of the result: rows that stay (copied
// only when the result is another cache) and rows moved in from `keep` on.  No
// row is both read as a source and written: sources are at or past `keep`.
template <int SWEEPS>
__global__ __launch_bounds__(THREADS) void evict_move_kernel(const EvictArgs a, const bool in_place) {
  constexpr int BLOCK = 16 * SWEEPS;
  __shared__ float scratch[4];
  const ckv_quant_cache& c = a.from;
  const int b = blockIdx.z >> 1, tensor = blockIdx.z & 1, h = blockIdx.y, tid = threadIdx.x;
  const EvictLayout lay(c.capacity, a.keep);
  const uint32_t* ws = a.workspace + ((int64_t)b * c.kv_heads + h) * lay.words;
  const int n = (int)ws[2];
  const int left = min(n, a.keep);
  if (blockIdx.x == 0 && h == 0 && tensor == 0 && tid == 0) {
    // the selection read the cursors; nothing of this launch does, but from a cache that stays as it is
    if (!in_place) {
      a.to.cursors[a.to.batch + b] = c.cursors[c.batch + b];
      a.to.cursors[2 * a.to.batch + b] = c.cursors[2 * c.batch + b];
    }
    a.to.cursors[b] = left;
  }
  const bool moves = n > a.keep;
  const int row0 = blockIdx.x * BLOCK;
  if (row0 >= left || (in_place && !moves)) return;
  const QuantHead src = quant_head(c, b, h), dst = quant_head(a.to, b, h);
  const int col = (tid & 15) * 8;
  const uint32_t* movers = ws + lay.movers;
  // the row that each of this thread's rows takes its content from (-1: none)
  int from[SWEEPS];
  bool hole[SWEEPS];
  bool any = false;
#pragma unroll
  for (int s = 0; s < SWEEPS; ++s) {
    const int row = row0 + 16 * s + (tid >> 4);
    from[s] = row < left ? row : -1;
    hole[s] = false;
    if (moves && row < left) {
      const uint32_t m = ws[lay.holes + (row >> 5)];
      if ((m >> (row & 31)) & 1u) {
        hole[s] = true;
        any = true;
        from[s] = (int)movers[ws[lay.base + (row >> 5)] + __popc(m & ((1u << (row & 31)) - 1u))];
      }
    }
  }
  any = __syncthreads_or(any);
  if (in_place && !any) return;
  uint2 w[SWEEPS];
  float scale_of[SWEEPS];
  const int straddle = a.keep / BLOCK;
#pragma unroll
  for (int s = 0; s < SWEEPS; ++s) {
    w[s] = uint2{0u, 0u};
    scale_of[s] = 1.0f;
    if (from[s] >= 0 && (hole[s] || !in_place)) {
      w[s] = *reinterpret_cast<const uint2*>(src.codes(tensor) + (int64_t)from[s] * D + col);
      // in place, the block around row `keep` is a target too: its scale was saved
      scale_of[s] = in_place && from[s] / BLOCK == straddle ? __uint_as_float(ws[tensor])
                                                           : src.scales(tensor)[from[s] / BLOCK];
    }
  }
  const int blk = row0 / BLOCK;
  const float old = in_place && blk == straddle ? __uint_as_float(ws[tensor]) : src.scales(tensor)[blk];
  float amax = 0.0f;
#pragma unroll
  for (int s = 0; s < SWEEPS; ++s) {
    if (hole[s]) {
      float v[8];
      decode4(w[s].x, v);
      decode4(w[s].y, v + 4);
#pragma unroll
      for (int i = 0; i < 8; ++i) amax = fmaxf(amax, finite_abs(v[i] * scale_of[s]));
    }
  }
  amax = block_max256(amax, scratch);
  const float scale = any ? fmaxf(old, block_scale(amax)) : old;
  const float inv = inverse_scale(scale);
  const float ratio = old * inv;
#pragma unroll
  for (int s = 0; s < SWEEPS; ++s) {
    const int row = row0 + 16 * s + (tid >> 4);
    if (from[s] < 0) continue;
    uint2* p = reinterpret_cast<uint2*>(dst.codes(tensor) + (int64_t)row * D + col);
    if (!hole[s] && scale == old) {
      if (!in_place) *p = w[s];
      continue;
    }
    if (!hole[s] && in_place) w[s] = *p;
    float v[8];
    decode4(w[s].x, v);
    decode4(w[s].y, v + 4);
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] *= hole[s] ? scale_of[s] * inv : ratio;
    *p = uint2{encode4(v[0], v[1], v[2], v[3]), encode4(v[4], v[5], v[6], v[7])};
  }
  if (tensor == 0 && (tid & 15) == 0) {
#pragma unroll
    for (int s = 0; s < SWEEPS; ++s) {
      const int row = row0 + 16 * s + (tid >> 4);
      if (from[s] < 0 || (in_place && !hole[s])) continue;
      dst.positions[row] = src.positions[from[s]];
      if (dst.weights) dst.weights[row] = src.weights[from[s]];
    }
  }
  __syncthreads();  // every wave has read the old scale
  if (tid == 0 && (!in_place || scale != old)) dst.scales(tensor)[blk] = scale;
}

int check_rows(const ckv_quant_rows* r, int dtype, const char* what) {
  static thread_local char message[160];
  const int unit = dtype == CKV_F32 ? 4 : 8;
  if (!r || !r->data) {
    snprintf(message, sizeof(message), "%s: null argument", what);
    return fail(CKV_E_INVALID, message);
  }
  if (((uintptr_t)r->data & 15) || r->batch_stride % unit || r->head_stride % unit || r->token_stride % unit) {
    snprintf(message, sizeof(message), "%s: rows must be 16-byte aligned", what);
    return fail(CKV_E_INVALID, message);
  }
  return CKV_OK;
}

}  // namespace

extern "C" int ckv_quant_append(const ckv_quant_cache* cache, const ckv_quant_rows* key, const ckv_quant_rows* value,
                                int32_t tokens, const int32_t* counts, int32_t dtype, void* stream) {
  int rc = validate_quant_cache(cache, "ckv_quant_append");
  if (rc) return rc;
  if (dtype != CKV_BF16 && dtype != CKV_F16 && dtype != CKV_F32)
    return fail(CKV_E_INVALID, "ckv_quant_append: dtype must be bf16, fp16 or f32");
  if (tokens <= 0) return fail(CKV_E_INVALID, "ckv_quant_append: tokens must be positive");
  rc = check_rows(key, dtype, "ckv_quant_append");
  if (!rc) rc = check_rows(value, dtype, "ckv_quant_append");
  if (rc) return rc;
  const AppendArgs a{*cache, *key, *value, counts, tokens};
  const hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  if (dtype == CKV_BF16) return launch_append<CKV_BF16>(a, s);
  if (dtype == CKV_F16) return launch_append<CKV_F16>(a, s);
  return launch_append<CKV_F32>(a, s);
}

extern "C" size_t ckv_quant_evict_workspace_bytes(const ckv_quant_cache* cache, int32_t keep) {
  if (!cache || cache->batch <= 0 || cache->kv_heads <= 0 || cache->capacity <= 0 || keep <= 0) return 0;
  const int64_t most = keep < cache->capacity ? keep : cache->capacity;
  return (size_t)cache->batch * cache->kv_heads * EvictLayout(cache->capacity, most).words * sizeof(uint32_t);
}

extern "C" int ckv_quant_evict(const ckv_quant_cache* cache, const ckv_quant_cache* into, int32_t keep,
                               int32_t num_sink, int32_t recent, void* workspace, void* stream) {
  int rc = validate_quant_cache(cache, "ckv_quant_evict");
  if (!rc && into) rc = validate_quant_cache(into, "ckv_quant_evict: into");
  if (rc) return rc;
  if (!cache->weights) return fail(CKV_E_INVALID, "ckv_quant_evict: the cache keeps no weights");
  if (keep <= 0 || num_sink < 0 || recent < 0 || (int64_t)num_sink + recent > keep)
    return fail(CKV_E_INVALID, "ckv_quant_evict: keep must be positive and hold num_sink + recent rows");
  if (!workspace || ((uintptr_t)workspace & 15)) return fail(CKV_E_INVALID, "ckv_quant_evict: workspace");
  const int32_t most = keep < cache->capacity ? keep : cache->capacity;
  if (into) {
    if (into->batch != cache->batch || into->kv_heads != cache->kv_heads || into->block != cache->block)
      return fail(CKV_E_INVALID, "ckv_quant_evict: into must have the cache's batch, heads and block");
    if (into->capacity < most) return fail(CKV_E_INVALID, "ckv_quant_evict: into holds fewer rows than keep");
    if (into->key_codes == cache->key_codes || into->value_codes == cache->value_codes ||
        into->cursors == cache->cursors)
      return fail(CKV_E_INVALID, "ckv_quant_evict: into must be another cache");
  } else if (keep >= cache->capacity) {
    return CKV_OK;  // no sequence can hold more
  }
  const EvictArgs a{*cache, into ? *into : *cache, reinterpret_cast<uint32_t*>(workspace), most, num_sink, recent};
  const hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  evict_select_kernel<<<dim3(cache->kv_heads, cache->batch), SEL_THREADS, 0, s>>>(a);
  rc = launched("ckv_quant_evict");
  if (rc) return rc;
  const dim3 grid((most + cache->block - 1) / cache->block, cache->kv_heads, 2 * cache->batch);
  const bool in_place = !into;
  if (cache->block == 16) evict_move_kernel<1><<<grid, THREADS, 0, s>>>(a, in_place);
  else if (cache->block == 32) evict_move_kernel<2><<<grid, THREADS, 0, s>>>(a, in_place);
  else if (cache->block == 64) evict_move_kernel<4><<<grid, THREADS, 0, s>>>(a, in_place);
  else evict_move_kernel<8><<<grid, THREADS, 0, s>>>(a, in_place);
  return launched("ckv_quant_evict");
}
