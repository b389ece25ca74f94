// Writing into the 8-bit KV cache, and eviction from it (gfx950).
//
// append_kernel: a workgroup of 512 threads owns one block of rows of one
// sequence and head, keys in its first half and values in its second: 16
// threads a row, 8 values each.  It reads its new rows once into registers,
// takes the block's largest magnitude, settles the scale, and writes codes of 8
// bytes a thread (a row of 128 bytes by 16 neighbouring threads).  Earlier rows
// of the block are touched only when the scale grows.
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
  if (((uintptr_t)c->key_codes | (uintptr_t)c->value_codes | (uintptr_t)c->positions | (uintptr_t)c->weights) & 15)
    return fail(CKV_E_INVALID, "codes, positions and weights must be 16-byte aligned");
  return CKV_OK;
}

}  // namespace ckv

namespace {
using namespace ckv;

constexpr int THREADS = 256;
constexpr int COUNTER_STRIDE = CKV_QUANT_COUNTERS;  // words between two sequences' counters: a cache line each

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
  const int tid = threadIdx.x & (THREADS - 1), col = (tid & 15) * 8;
  for (int r = tid >> 4; r < rows; r += THREADS / 16) {
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

// The cursors of a sequence move when every workgroup has read them.  With few
// workgroups a sequence (`ticket`) the last to finish moves them; the tickets of
// many queue at one address (12 ns each), and advance_kernel behind the append is
// quicker.  Both in a graph, 8 heads in blocks of 64: one token of 8 sequences 5.4 us
// with tickets and 6.2 with advance_kernel; of one sequence, 449 tokens (64
// workgroups) 7.5 and 7.9, 960 tokens (128) 8.1 and 8.0, 4,096 (520) 14.4 and 10.8,
// 32,768 into an empty cache 61 and 41.
__device__ inline void advance(const ckv_quant_cache& c, int b, int start, int seen, int count) {
  const int end = (int)min((int64_t)start + count, (int64_t)c.capacity);
  c.cursors[b] = end;
  c.cursors[c.batch + b] = seen + (end - start);
  if ((int64_t)start + count > c.capacity) c.cursors[2 * c.batch + b] = 1;
}

__device__ inline int append_count(const AppendArgs& a, int b) {
  return a.counts ? min(max(a.counts[b], 0), a.tokens) : a.tokens;
}

template <int DT, int SWEEPS>
__global__ __launch_bounds__(2 * THREADS) void append_kernel(const AppendArgs a, const bool ticket) {
  constexpr int BLOCK = 16 * SWEEPS;
  __shared__ float scratch[2][4];
  const ckv_quant_cache& c = a.cache;
  const int b = blockIdx.z, h = blockIdx.y, tensor = __builtin_amdgcn_readfirstlane(threadIdx.x >> 8);
  const int tid = threadIdx.x & (THREADS - 1);
  const int start = quant_length(c, b), seen = c.cursors[c.batch + b];
  const int count = append_count(a, b);
  const int end = (int)min((int64_t)start + count, (int64_t)c.capacity);
  const int64_t blk = start / BLOCK + (int64_t)blockIdx.x;
  const int64_t row0 = blk * BLOCK;
  const int lo = (int)max((int64_t)start, row0), hi = (int)min((int64_t)end, row0 + BLOCK);
  if (lo < hi) {  // the same for the whole workgroup
    const QuantHead q = quant_head(c, b, h);
    const ckv_quant_rows in = tensor ? a.value : a.key;
    const int64_t base = (int64_t)b * in.batch_stride + (int64_t)h * in.head_stride;
    const int col = (tid & 15) * 8;
    float v[SWEEPS][8];
    const float old = row0 < start ? q.scales(tensor)[blk] : 0.0f;
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
    wait_vm();  // the old scale has arrived before another wave may write the new one
    amax = wave_max(amax);
    if ((tid & 63) == 0) scratch[tensor][tid >> 6] = amax;
    __syncthreads();
    amax = fmaxf(fmaxf(scratch[tensor][0], scratch[tensor][1]), fmaxf(scratch[tensor][2], scratch[tensor][3]));
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
    if (tid == 0 && scale != old) q.scales(tensor)[blk] = scale;
  }
  if (!ticket) return;
  __syncthreads();  // every wave has read the cursors
  if (threadIdx.x == 0) {
    uint32_t* counter = c.counters + (int64_t)b * COUNTER_STRIDE;
    if (atomicAdd(counter, 1u) == gridDim.x * gridDim.y - 1) {
      st_agent_u32(counter, 0u);
      advance(c, b, start, seen, count);
    }
  }
}

__global__ __launch_bounds__(THREADS) void advance_kernel(const AppendArgs a) {
  const ckv_quant_cache& c = a.cache;
  const int b = blockIdx.x * THREADS + threadIdx.x;
  if (b < c.batch) advance(c, b, quant_length(c, b), c.cursors[c.batch + b], append_count(a, b));
}

template <int DT>
int launch_append(const AppendArgs& a, hipStream_t stream) {
  const int block = a.cache.block;
  // tokens rows from any start touch at most this many blocks
  const int64_t blocks = min((int64_t)(a.tokens + block - 2) / block + 1, (int64_t)a.cache.capacity / block);
  const dim3 grid((uint32_t)blocks, a.cache.kv_heads, a.cache.batch);
  const bool ticket = blocks * a.cache.kv_heads <= 64;
  if (block == 16) append_kernel<DT, 1><<<grid, 2 * THREADS, 0, stream>>>(a, ticket);
  else if (block == 32) append_kernel<DT, 2><<<grid, 2 * THREADS, 0, stream>>>(a, ticket);
  else if (block == 64) append_kernel<DT, 4><<<grid, 2 * THREADS, 0, stream>>>(a, ticket);
  else append_kernel<DT, 8><<<grid, 2 * THREADS, 0, stream>>>(a, ticket);
  int rc = launched("ckv_quant_append");
  if (!rc && !ticket) {
    advance_kernel<<<(a.cache.batch + THREADS - 1) / THREADS, THREADS, 0, stream>>>(a);
    rc = launched("ckv_quant_append");
  }
  return rc;
}

// ---------------------------------------------------------------------------
// Eviction
// ---------------------------------------------------------------------------

// Rows of one workgroup of the selection by several workgroups.
// (131k to 16k rows, 16 heads, in a graph: 60.0 us; 256 threads of 16 keys 63.6, of 8
// 61.9, of 4 65.3.)
constexpr int CHUNK_THREADS = 512;
constexpr int CHUNK_KEYS = 8;  // keys of a thread
constexpr int CHUNK = CHUNK_THREADS * CHUNK_KEYS;
// The keys' digits: 11, 11 and 10 bits.
constexpr int DIGITS = 3;
__host__ __device__ constexpr int digit_shift(int d) { return d == 0 ? 21 : d == 1 ? 10 : 0; }
__host__ __device__ constexpr int digit_bins(int d) { return d == 2 ? 1024 : 2048; }
__host__ __device__ constexpr int digit_bin0(int d) { return 2048 * d; }
constexpr int ALL_BINS = 2048 + 2048 + 1024;

// Workspace of one (sequence, head), in 32-bit words: two saved scales of the
// block that holds row `keep`, the row count before, then what the digits found
// so far (prefix and rows wanted of it, a pair a digit), the digits' histograms,
// four counts a chunk, the keys of every row, the kept rows from `keep` on
// (ascending), and for every 32 rows below `keep` the mask of freed rows and
// their number before.
struct EvictLayout {
  int64_t found, hist, counts, keys, movers, holes, base, words;
  __host__ __device__ EvictLayout(int64_t capacity, int64_t keep) {
    const int64_t groups = (keep + 31) / 32, chunks = (capacity + CHUNK - 1) / CHUNK;
    found = 4;
    hist = found + 2 * DIGITS + 2;
    counts = hist + ALL_BINS;
    keys = counts + 4 * chunks;
    movers = keys + capacity;
    holes = movers + ((keep + 3) & ~(int64_t)3);
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

// One workgroup a (sequence, head) selects where its threads hold all keys, and
// several where they do not.  A whole eviction of 8 heads, half the rows kept, in a
// graph: capacity 1,000 13.6 us with 256 threads of 8 keys, 14.4 with 1,024 (their
// barriers), 25.2 with several workgroups (the launches); 8,000 17.2 with 1,024
// threads of 8 keys, 28.8; 12,000 23.9 with 1,024 of 16, 32.3; 16,300 27.8, 34.8;
// 32,000 48.9 with 32 keys a thread, 40.2.
constexpr int SELECT_FEW = 256, SELECT_MANY = 1024;
constexpr int KEYS_FEW = 8, KEYS_MANY = 16;

// Exclusive scan of x over a workgroup of T threads, and its total.
template <int T>
__device__ inline int block_scan(int x, int* total, int* scratch) {
  const int incl = wave_inclusive_scan(x);
  const int wave = threadIdx.x >> 6;
  __syncthreads();
  if ((threadIdx.x & 63) == 63) scratch[wave] = incl;
  __syncthreads();
  int before = 0, sum = 0;
#pragma unroll
  for (int w = 0; w < T / 64; ++w) {
    const int v = scratch[w];
    if (w < wave) before += v;
    sum += v;
  }
  *total = sum;
  return before + incl - x;
}

// Adds this lane's bin (where `in`) to the histogram in LDS, a whole wave at once
// where its lanes agree (equal weights are common).
__device__ inline void count_bin(int* hist, bool in, uint32_t bin) {
  const uint64_t lanes = __ballot(in);
  if (lanes == 0) return;
  const int leader = __ffsll((unsigned long long)lanes) - 1;
  const uint32_t first = (uint32_t)__builtin_amdgcn_readlane((int)bin, leader);
  if (__ballot(in && bin != first) == 0) {
    if ((int)(threadIdx.x & 63) == leader) atomicAdd(&hist[first], __popcll(lanes));
  } else if (in) {
    atomicAdd(&hist[bin], 1);
  }
}

// The bin where the rows counted from the highest bin reach `target`, and how
// many are still wanted of that bin.  Every thread of the workgroup of T; scratch
// holds T / 64 + 2 words.
template <int T>
__device__ inline void find_digit(const int* hist, int bins, int target, int* scratch, int* bin, int* left) {
  constexpr int MOST = 2048 / T;
  const int each = bins / T, top = bins - 1 - (int)threadIdx.x * each;
  int mine[MOST], sum = 0;
#pragma unroll
  for (int i = 0; i < MOST; ++i) {
    mine[i] = i < each ? hist[top - i] : 0;
    sum += mine[i];
  }
  int total;
  int before = block_scan<T>(sum, &total, scratch);
  if (before < target && before + sum >= target) {
#pragma unroll
    for (int i = 0; i < MOST; ++i) {
      if (before < target && before + mine[i] >= target) {
        scratch[T / 64] = top - i;
        scratch[T / 64 + 1] = target - before;
      }
      before += mine[i];
    }
  }
  __syncthreads();
  *bin = scratch[T / 64];
  *left = scratch[T / 64 + 1];
}

// Which of this thread's K rows from `first` on are kept: those above `key`, and
// of those that equal it the first `ties` of all, `rank` of which come before.
template <int K>
__device__ inline uint32_t kept_rows(const uint32_t* k, int64_t first, int n, uint32_t key, int ties, int rank) {
  uint32_t kept = 0;
#pragma unroll
  for (int i = 0; i < K; ++i) {
    const bool in = first + i < n, tie = in && k[i] == key;
    if (in && (k[i] > key || (tie && rank < ties))) kept |= 1u << i;
    rank += tie;
  }
  return kept;
}

__device__ inline uint32_t low_rows(int64_t first, int keep, int rows) {
  return (uint32_t)((1ull << (int)min(max((int64_t)keep - first, (int64_t)0), (int64_t)rows)) - 1ull);  // rows <= 32
}

// Writes this thread's lists: `kept` of K rows from `first` on, `before` packs the
// freed rows below `keep` (low half) and the kept ones from it on before them in the
// workgroup, freed0 and moved0 those before the workgroup.
template <int K>
__device__ inline void write_lists(uint32_t* ws, const EvictLayout& lay, int64_t first, int keep, uint32_t kept,
                                   int before, int freed0, int moved0) {
  const uint32_t low = low_rows(first, keep, K);
  int moved = moved0 + (before >> 16);
  for (uint32_t m = kept & ~low; m; m &= m - 1) ws[lay.movers + moved++] = (uint32_t)(first + __ffs((int)m) - 1);
  // 32 / K threads' rows make a word of the mask
  uint32_t holes = (~kept & low) << (first & 31);
#pragma unroll
  for (int o = 1; o < 32 / K; o <<= 1) holes |= (uint32_t)__shfl_xor((int)holes, o);
  if ((first & 31) == 0 && first < keep) {
    ws[lay.holes + (first >> 5)] = holes;
    ws[lay.base + (first >> 5)] = (uint32_t)(freed0 + (before & 0xffff));
  }
}

// Loads this thread's keys from the weights and positions, four rows at once (the
// capacity is a multiple of 16).
template <int K>
__device__ inline void make_keys(const EvictArgs& a, const QuantHead& q, int64_t first, int n, int seen, uint32_t* k) {
  const int64_t newest = (int64_t)seen - a.recent;
#pragma unroll
  for (int i = 0; i < K; i += 4) {
    if (first + i < n) {
      const float4 w = *reinterpret_cast<const float4*>(q.weights + first + i);
      const int4 p = *reinterpret_cast<const int4*>(q.positions + first + i);
      k[i] = evict_key(w.x, p.x < a.num_sink || p.x >= newest);
      k[i + 1] = evict_key(w.y, p.y < a.num_sink || p.y >= newest);
      k[i + 2] = evict_key(w.z, p.z < a.num_sink || p.z >= newest);
      k[i + 3] = evict_key(w.w, p.w < a.num_sink || p.w >= newest);
    } else {
      k[i] = k[i + 1] = k[i + 2] = k[i + 3] = 0;
    }
  }
}

__device__ inline void write_header(const EvictArgs& a, const QuantHead& q, uint32_t* ws, int n) {
  const int64_t blk = a.keep / a.from.block;
  const bool inside = a.keep < a.from.capacity;
  ws[0] = inside ? __float_as_uint(q.key_scales[blk]) : 0u;
  ws[1] = inside ? __float_as_uint(q.value_scales[blk]) : 0u;
  ws[2] = (uint32_t)n;
}

// One workgroup a (sequence, head), a thread's KEYS rows in order in
// registers: the `keep`-th largest by its three digits from the highest, then two
// scans in row order, for the ties (taken by the lower row) and for the lists of
// freed rows below `keep` and kept ones from it on.
template <int T, int KEYS>
__global__ __launch_bounds__(T) void evict_select_kernel(const EvictArgs a) {
  __shared__ int hist[2048];
  __shared__ int scratch[T / 64 + 2];
  const ckv_quant_cache& c = a.from;
  const int h = blockIdx.x, b = blockIdx.y, tid = threadIdx.x;
  const int n = quant_length(c, b), seen = c.cursors[c.batch + b];
  const QuantHead q = quant_head(c, b, h);
  const EvictLayout lay(c.capacity, a.keep);
  uint32_t* ws = a.workspace + ((int64_t)b * c.kv_heads + h) * lay.words;
  if (tid == 0) write_header(a, q, ws, n);
  if (n <= a.keep) return;
  uint32_t k[KEYS];
  const int first = tid * KEYS;
  make_keys<KEYS>(a, q, first, n, seen, k);
  uint32_t prefix = 0;
  int target = a.keep;  // how many of the rows that match the prefix are kept
#pragma unroll
  for (int d = 0; d < DIGITS; ++d) {
    const int bins = digit_bins(d), shift = digit_shift(d);
    for (int i = tid; i < bins; i += T) hist[i] = 0;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < KEYS; ++i) {
      const bool in = first + i < n && (d == 0 || (k[i] >> digit_shift(d - 1)) == (prefix >> digit_shift(d - 1)));
      count_bin(hist, in, (k[i] >> shift) & (bins - 1));
    }
    __syncthreads();
    int bin;
    find_digit<T>(hist, bins, target, scratch, &bin, &target);
    prefix |= (uint32_t)bin << shift;
  }
  int equal = 0, total;
#pragma unroll
  for (int i = 0; i < KEYS; ++i) equal += first + i < n && k[i] == prefix;
  const int rank = block_scan<T>(equal, &total, scratch);
  const uint32_t kept = kept_rows<KEYS>(k, first, n, prefix, target, rank);
  const uint32_t low = low_rows(first, a.keep, KEYS);
  const int before = block_scan<T>(__popc(~kept & low) | (__popc(kept & ~low) << 16), &total, scratch);
  write_lists<KEYS>(ws, lay, first, a.keep, kept, before, 0, 0);
}

// The same by several workgroups a (sequence, head), for long sequences, in
// launches that follow one another: keys and the histogram of their first digit;
// the second digit's and the third's among the rows that match so far; counts of
// kept and tied rows a chunk, below row `keep` and from it on; the lists, each
// chunk behind those before it.
struct ChunkPlace {
  uint32_t* ws;
  int n, seen;
  int64_t first;  // row of this thread's first key
};

__device__ inline bool chunk_place(const EvictArgs& a, const EvictLayout& lay, ChunkPlace* p) {
  const ckv_quant_cache& c = a.from;
  const int b = blockIdx.z, h = blockIdx.y;
  p->ws = a.workspace + ((int64_t)b * c.kv_heads + h) * lay.words;
  p->n = quant_length(c, b);
  p->seen = c.cursors[c.batch + b];
  p->first = (int64_t)blockIdx.x * CHUNK + (int64_t)threadIdx.x * CHUNK_KEYS;
  return p->n > a.keep && (int64_t)blockIdx.x * CHUNK < p->n;
}

__device__ inline void load_keys(const uint32_t* keys, uint32_t* k) {
#pragma unroll
  for (int i = 0; i < CHUNK_KEYS / 4; ++i) {
    const uint4 w = gload16(keys + 4 * i);
    k[4 * i] = w.x;
    k[4 * i + 1] = w.y;
    k[4 * i + 2] = w.z;
    k[4 * i + 3] = w.w;
  }
}

__global__ __launch_bounds__(256) void evict_clear_kernel(const EvictArgs a) {
  const EvictLayout lay(a.from.capacity, a.keep);
  uint32_t* hist = a.workspace + (int64_t)blockIdx.x * lay.words + lay.hist;
  for (int i = threadIdx.x; i < ALL_BINS; i += 256) hist[i] = 0;
}

template <int DIGIT>
__global__ __launch_bounds__(CHUNK_THREADS) void evict_digit_kernel(const EvictArgs a) {
  constexpr int BINS = digit_bins(DIGIT), SHIFT = digit_shift(DIGIT);
  __shared__ int hist[BINS];
  __shared__ int scratch[CHUNK_THREADS / 64 + 2];
  const EvictLayout lay(a.from.capacity, a.keep);
  ChunkPlace at;
  const bool work = chunk_place(a, lay, &at);
  const QuantHead q = quant_head(a.from, blockIdx.z, blockIdx.y);
  if (DIGIT == 0 && blockIdx.x == 0 && threadIdx.x == 0) write_header(a, q, at.ws, at.n);
  if (!work) return;
  uint32_t prefix = 0;
  if constexpr (DIGIT > 0) {
    // the digit before, from its histogram
    const uint32_t* found = at.ws + lay.found + 2 * (DIGIT - 1);
    const uint32_t known = DIGIT > 1 ? found[-2] : 0u;
    const int target = DIGIT > 1 ? (int)found[-1] : a.keep;
    int bin, left;
    find_digit<CHUNK_THREADS>(reinterpret_cast<const int*>(at.ws) + lay.hist + digit_bin0(DIGIT - 1),
                              digit_bins(DIGIT - 1), target, scratch, &bin, &left);
    prefix = known | ((uint32_t)bin << digit_shift(DIGIT - 1));
    if (blockIdx.x == 0 && threadIdx.x == 0) {  // for the launches to come
      at.ws[lay.found + 2 * (DIGIT - 1)] = prefix;
      at.ws[lay.found + 2 * (DIGIT - 1) + 1] = (uint32_t)left;
    }
  }
  for (int i = threadIdx.x; i < BINS; i += CHUNK_THREADS) hist[i] = 0;
  __syncthreads();
  uint32_t k[CHUNK_KEYS];
  uint32_t* keys = at.ws + lay.keys + at.first;
  if constexpr (DIGIT == 0) {
    make_keys<CHUNK_KEYS>(a, q, at.first, at.n, at.seen, k);
#pragma unroll
    for (int i = 0; i < CHUNK_KEYS; i += 4) {
      if (at.first + i < at.n) *reinterpret_cast<uint4*>(keys + i) = uint4{k[i], k[i + 1], k[i + 2], k[i + 3]};
    }
  } else if (at.first < at.n) {
    load_keys(keys, k);
  }
#pragma unroll
  for (int i = 0; i < CHUNK_KEYS; ++i) {
    const bool in = at.first + i < at.n && (DIGIT == 0 || (k[i] >> digit_shift(DIGIT - 1)) == (prefix >> digit_shift(DIGIT - 1)));
    count_bin(hist, in, in ? (k[i] >> SHIFT) & (BINS - 1) : 0u);
  }
  __syncthreads();
  uint32_t* all = at.ws + lay.hist + digit_bin0(DIGIT);
  for (int i = threadIdx.x; i < BINS; i += CHUNK_THREADS) {
    const int x = hist[i];
    if (x) atomicAdd(&all[i], (uint32_t)x);
  }
}

// The threshold key and how many of the rows that equal it are kept.
__device__ inline void threshold(const EvictArgs& a, const EvictLayout& lay, const uint32_t* ws, int* scratch,
                                 uint32_t* key, int* ties) {
  const uint32_t* found = ws + lay.found + 2 * (DIGITS - 2);
  int bin;
  find_digit<CHUNK_THREADS>(reinterpret_cast<const int*>(ws) + lay.hist + digit_bin0(DIGITS - 1),
                            digit_bins(DIGITS - 1), (int)found[1], scratch, &bin, ties);
  *key = found[0] | (uint32_t)bin;
}

__global__ __launch_bounds__(CHUNK_THREADS) void evict_count_kernel(const EvictArgs a) {
  __shared__ int scratch[CHUNK_THREADS / 64 + 2];
  const EvictLayout lay(a.from.capacity, a.keep);
  ChunkPlace at;
  if (!chunk_place(a, lay, &at)) return;
  uint32_t key;
  int ties;
  threshold(a, lay, at.ws, scratch, &key, &ties);
  uint32_t k[CHUNK_KEYS];
  int above[2] = {0, 0}, equal[2] = {0, 0};  // below row `keep`, from it on
  if (at.first < at.n) {
    load_keys(at.ws + lay.keys + at.first, k);
#pragma unroll
    for (int i = 0; i < CHUNK_KEYS; ++i) {
      const bool in = at.first + i < at.n, high = at.first + i >= a.keep;
      above[0] += in && !high && k[i] > key;
      above[1] += in && high && k[i] > key;
      equal[0] += in && !high && k[i] == key;
      equal[1] += in && high && k[i] == key;
    }
  }
  int low, high;
  block_scan<CHUNK_THREADS>(above[0] | (equal[0] << 16), &low, scratch);
  block_scan<CHUNK_THREADS>(above[1] | (equal[1] << 16), &high, scratch);
  if (threadIdx.x == 0) {
    uint32_t* counts = at.ws + lay.counts + 4 * blockIdx.x;
    counts[0] = (uint32_t)low & 0xffffu;
    counts[1] = (uint32_t)low >> 16;
    counts[2] = (uint32_t)high & 0xffffu;
    counts[3] = (uint32_t)high >> 16;
  }
}

__global__ __launch_bounds__(CHUNK_THREADS) void evict_list_kernel(const EvictArgs a) {
  __shared__ int scratch[CHUNK_THREADS / 64 + 2];
  const EvictLayout lay(a.from.capacity, a.keep);
  ChunkPlace at;
  if (!chunk_place(a, lay, &at)) return;
  uint32_t key;
  int ties;
  threshold(a, lay, at.ws, scratch, &key, &ties);
  // of the chunks before, one a thread: tied rows, kept rows from `keep` on, kept rows below it
  int tied = 0, moved = 0, kept_low = 0;
  for (int c0 = 0; c0 < (int)blockIdx.x; c0 += CHUNK_THREADS) {
    const int c = c0 + (int)threadIdx.x;
    uint4 n{0u, 0u, 0u, 0u};
    if (c < (int)blockIdx.x) n = *reinterpret_cast<const uint4*>(at.ws + lay.counts + 4 * (int64_t)c);
    int sum_tied, sum_moved, sum_kept;
    const int earlier = tied + block_scan<CHUNK_THREADS>((int)(n.y + n.w), &sum_tied, scratch);
    const int take_low = min(max(ties - earlier, 0), (int)n.y);
    const int take_high = min(max(ties - earlier - (int)n.y, 0), (int)n.w);
    block_scan<CHUNK_THREADS>((int)n.z + take_high, &sum_moved, scratch);
    block_scan<CHUNK_THREADS>((int)n.x + take_low, &sum_kept, scratch);
    tied += sum_tied;
    moved += sum_moved;
    kept_low += sum_kept;
  }
  const int64_t chunk0 = (int64_t)blockIdx.x * CHUNK;
  const int freed = (int)min(chunk0, (int64_t)a.keep) - kept_low;
  uint32_t k[CHUNK_KEYS];
#pragma unroll
  for (int i = 0; i < CHUNK_KEYS; ++i) k[i] = 0;
  if (at.first < at.n) load_keys(at.ws + lay.keys + at.first, k);
  int equal = 0, total;
#pragma unroll
  for (int i = 0; i < CHUNK_KEYS; ++i) equal += at.first + i < at.n && k[i] == key;
  const int rank = tied + block_scan<CHUNK_THREADS>(equal, &total, scratch);
  const uint32_t kept = kept_rows<CHUNK_KEYS>(k, at.first, at.n, key, ties, rank);
  const uint32_t low = low_rows(at.first, a.keep, CHUNK_KEYS);
  const int before =
      block_scan<CHUNK_THREADS>(__popc(~kept & low) | (__popc(kept & ~low) << 16), &total, scratch);
  write_lists<CHUNK_KEYS>(at.ws, lay, at.first, a.keep, kept, before, freed, moved);
}

// A workgroup of 256 threads writes one block of rows of the result, keys in its
// first half and values in its second, 16 codes a thread: rows that stay (copied
// only when the result is another cache) and rows moved in from `keep` on.  No
// row is both read as a source and written: sources are at or past `keep`.
template <int SWEEPS>
__global__ __launch_bounds__(THREADS) void evict_move_kernel(const EvictArgs a, const bool in_place) {
  constexpr int BLOCK = 16 * SWEEPS;
  __shared__ float scratch[4];
  const ckv_quant_cache& c = a.from;
  const int b = blockIdx.z, h = blockIdx.y, tensor = __builtin_amdgcn_readfirstlane(threadIdx.x >> 7);
  const int tid = threadIdx.x & 127;
  const EvictLayout lay(c.capacity, a.keep);
  const uint32_t* ws = a.workspace + ((int64_t)b * c.kv_heads + h) * lay.words;
  const int n = (int)ws[2];
  const int left = min(n, a.keep);
  if (blockIdx.x == 0 && h == 0 && threadIdx.x == 0) {
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
  // freed rows of this block and their number before, a word for 32 rows (a block of 16 takes half of one)
  constexpr int WORDS = (BLOCK + 31) / 32;
  uint32_t mask[WORDS], base[WORDS];
  uint32_t any = 0;
#pragma unroll
  for (int w = 0; w < WORDS; ++w) {
    const int word = (row0 >> 5) + w;
    const bool in = moves && 32 * word < left;
    mask[w] = in ? ws[lay.holes + word] : 0u;
    base[w] = in ? ws[lay.base + word] : 0u;
    any |= BLOCK < 32 ? (mask[w] >> (row0 & 31)) & 0xffffu : mask[w];
  }
  if (in_place && !any) return;
  const QuantHead src = quant_head(c, b, h), dst = quant_head(a.to, b, h);
  const uint32_t* movers = ws + lay.movers;
  const int col = (tid & 7) * 16;
  // the row that each of this thread's rows takes its content from (-1: none)
  int from[SWEEPS];
  bool hole[SWEEPS];
#pragma unroll
  for (int s = 0; s < SWEEPS; ++s) {
    const int row = row0 + 16 * s + (tid >> 3);
    const uint32_t m = mask[s >> 1];
    hole[s] = row < left && ((m >> (row & 31)) & 1u);
    from[s] = row >= left ? -1 : hole[s] ? (int)movers[base[s >> 1] + __popc(m & ((1u << (row & 31)) - 1u))] : row;
  }
  uint4 w[SWEEPS];
  float scale_of[SWEEPS];
  const int straddle = a.keep / BLOCK, blk = row0 / BLOCK;
  // in place, the block around row `keep` is a source and a target: its scale was saved
  auto scale_at = [&](int block) {
    return in_place && block == straddle ? __uint_as_float(ws[tensor]) : gload_f32(src.scales(tensor) + block);
  };
#pragma unroll
  for (int s = 0; s < SWEEPS; ++s) {
    w[s] = uint4{0u, 0u, 0u, 0u};
    scale_of[s] = 1.0f;
    if (from[s] >= 0 && (hole[s] || !in_place)) {
      w[s] = gload16(src.codes(tensor) + (int64_t)from[s] * D + col);
      scale_of[s] = scale_at(from[s] / BLOCK);
    }
  }
  const float old = scale_at(blk);
  float amax = 0.0f;
#pragma unroll
  for (int s = 0; s < SWEEPS; ++s) {
    if (hole[s]) {
      float v[16];
      decode4(w[s].x, v);
      decode4(w[s].y, v + 4);
      decode4(w[s].z, v + 8);
      decode4(w[s].w, v + 12);
#pragma unroll
      for (int i = 0; i < 16; ++i) amax = fmaxf(amax, finite_abs(v[i] * scale_of[s]));
    }
  }
  wait_vm();  // the old scale has arrived before another wave may write the new one
  amax = wave_max(amax);
  if ((tid & 63) == 0) scratch[threadIdx.x >> 6] = amax;
  __syncthreads();
  amax = fmaxf(scratch[2 * tensor], scratch[2 * tensor + 1]);
  const float scale = any ? fmaxf(old, block_scale(amax)) : old;
  const float inv = inverse_scale(scale), ratio = old * inv;
#pragma unroll
  for (int s = 0; s < SWEEPS; ++s) {
    const int row = row0 + 16 * s + (tid >> 3);
    if (from[s] < 0) continue;
    uint4* p = reinterpret_cast<uint4*>(dst.codes(tensor) + (int64_t)row * D + col);
    const float factor = hole[s] ? scale_of[s] * inv : ratio;
    if (factor == 1.0f) {  // the codes as they are
      if (hole[s] || !in_place) *p = w[s];
      continue;
    }
    if (!hole[s] && in_place) w[s] = *p;
    uint32_t x[4] = {w[s].x, w[s].y, w[s].z, w[s].w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      float v[4];
      decode4(x[i], v);
      x[i] = encode4(v[0] * factor, v[1] * factor, v[2] * factor, v[3] * factor);
    }
    *p = uint4{x[0], x[1], x[2], x[3]};
  }
  if (tensor == 0 && (tid & 7) == 0) {
#pragma unroll
    for (int s = 0; s < SWEEPS; ++s) {
      const int row = row0 + 16 * s + (tid >> 3);
      if (from[s] < 0 || (in_place && !hole[s])) continue;
      dst.positions[row] = src.positions[from[s]];
      if (dst.weights) dst.weights[row] = src.weights[from[s]];
    }
  }
  if (tid == 0 && (!in_place || scale != old)) dst.scales(tensor)[blk] = scale;
}

// Whether two caches share any of the memory that an eviction reads or writes.
bool overlap(const ckv_quant_cache& x, const ckv_quant_cache& y) {
  struct Spans {
    uintptr_t at[7], end[7];
    explicit Spans(const ckv_quant_cache& c) {
      const uintptr_t rows = (uintptr_t)c.batch * c.kv_heads * c.capacity, scales = rows / c.block * sizeof(float);
      const void* first[7] = {c.key_codes, c.value_codes, c.key_scales, c.value_scales, c.positions, c.weights, c.cursors};
      const uintptr_t bytes[7] = {rows * D, rows * D, scales, scales, rows * 4, c.weights ? rows * 4 : 0,
                                  (uintptr_t)c.batch * 12};
      for (int i = 0; i < 7; ++i) end[i] = (at[i] = (uintptr_t)first[i]) + bytes[i];
    }
  };
  const Spans a(x), b(y);
  for (int i = 0; i < 7; ++i)
    for (int j = 0; j < 7; ++j)
      if (a.at[i] < b.end[j] && b.at[j] < a.end[i]) return true;
  return false;
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
    if (overlap(*cache, *into)) return fail(CKV_E_INVALID, "ckv_quant_evict: into must be another cache, with no memory of this one");
  } else if (keep >= cache->capacity) {
    return CKV_OK;  // no sequence can hold more
  }
  const EvictArgs a{*cache, into ? *into : *cache, reinterpret_cast<uint32_t*>(workspace), most, num_sink, recent};
  const hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  const dim3 heads(cache->kv_heads, cache->batch);
  if (cache->capacity <= SELECT_FEW * KEYS_FEW) {
    evict_select_kernel<SELECT_FEW, KEYS_FEW><<<heads, SELECT_FEW, 0, s>>>(a);
  } else if (cache->capacity <= SELECT_MANY * KEYS_FEW) {
    evict_select_kernel<SELECT_MANY, KEYS_FEW><<<heads, SELECT_MANY, 0, s>>>(a);
  } else if (cache->capacity <= SELECT_MANY * KEYS_MANY) {
    evict_select_kernel<SELECT_MANY, KEYS_MANY><<<heads, SELECT_MANY, 0, s>>>(a);
  } else {
    const dim3 chunks((cache->capacity + CHUNK - 1) / CHUNK, cache->kv_heads, cache->batch);
    evict_clear_kernel<<<cache->batch * cache->kv_heads, 256, 0, s>>>(a);
    evict_digit_kernel<0><<<chunks, CHUNK_THREADS, 0, s>>>(a);
    evict_digit_kernel<1><<<chunks, CHUNK_THREADS, 0, s>>>(a);
    evict_digit_kernel<2><<<chunks, CHUNK_THREADS, 0, s>>>(a);
    evict_count_kernel<<<chunks, CHUNK_THREADS, 0, s>>>(a);
    evict_list_kernel<<<chunks, CHUNK_THREADS, 0, s>>>(a);
  }
  rc = launched("ckv_quant_evict");
  if (rc) return rc;
  const dim3 grid((most + cache->block - 1) / cache->block, cache->kv_heads, cache->batch);
  const bool in_place = !into;
  if (cache->block == 16) evict_move_kernel<1><<<grid, THREADS, 0, s>>>(a, in_place);
  else if (cache->block == 32) evict_move_kernel<2><<<grid, THREADS, 0, s>>>(a, in_place);
  else if (cache->block == 64) evict_move_kernel<4><<<grid, THREADS, 0, s>>>(a, in_place);
  else evict_move_kernel<8><<<grid, THREADS, 0, s>>>(a, in_place);
  return launched("ckv_quant_evict");
}
