// Paged KV cache: the plan of drafted trees, writing a step's rows with the
// position rotation on the way, and committing them (gfx950).
#include <hip/hip_runtime.h>

#include "ckv_paged.h"

namespace ckv {

int paged_error(int code, const char* what, const char* why) {
  static thread_local char message[160];
  snprintf(message, sizeof(message), "%s: %s", what, why);
  return ckv_internal::set_error(code, message);
}

int paged_launched(const char* what) {
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? CKV_OK : paged_error(CKV_E_LAUNCH, what, hipGetErrorString(e));
}

int validate_paged_cache(const ckv_paged_cache* c, const char* what) {
  if (!c || !c->key_pages || !c->value_pages || !c->page_table || !c->lengths || !c->overflow || !c->counters)
    return paged_error(CKV_E_INVALID, what, "null argument");
  if (c->layers <= 0 || c->pages <= 0 || c->kv_heads <= 0 || c->table_pages <= 0 || c->batch <= 0)
    return paged_error(CKV_E_INVALID, what, "layers, pages, kv_heads, table_pages and batch must be positive");
  if (c->page_size < 16 || c->page_size > 256 || (c->page_size & (c->page_size - 1)))
    return paged_error(CKV_E_INVALID, what, "page_size must be 16, 32, 64, 128 or 256");
  if (c->dtype != CKV_BF16 && c->dtype != CKV_F16) return paged_error(CKV_E_INVALID, what, "the cache must be bf16 or fp16");
  if ((int64_t)c->table_pages * c->page_size > (1 << 30)) return paged_error(CKV_E_LIMIT, what, "more than 2^30 rows a sequence");
  if (c->batch > 32767 || c->kv_heads > 32767 || (int64_t)c->batch * c->kv_heads > 65535)
    return paged_error(CKV_E_LIMIT, what, "more than 65535 heads over the batch");
  if ((int64_t)c->batch * c->table_pages * c->page_size >= ((int64_t)1 << 37))
    return paged_error(CKV_E_LIMIT, what, "more than 2^37 rows over the batch");
  if (((uintptr_t)c->key_pages | (uintptr_t)c->value_pages) & 15)
    return paged_error(CKV_E_INVALID, what, "pages must be 16-byte aligned");
  return CKV_OK;
}

int check_paged_rows(const ckv_quant_rows* r, int dtype, const char* what) {
  const int unit = dtype == CKV_F32 ? 4 : 8;
  if (!r || !r->data) return paged_error(CKV_E_INVALID, what, "null argument");
  if (((uintptr_t)r->data & 15) || r->batch_stride % unit || r->head_stride % unit || r->token_stride % unit)
    return paged_error(CKV_E_INVALID, what, "rows must be 16-byte aligned");
  return CKV_OK;
}

}  // namespace ckv

namespace {
using namespace ckv;

constexpr int THREADS = 256;
constexpr int MAX_WORDS = CKV_MAX_DRAFT / 64;

// ---------------------------------------------------------------------------
// Plan of drafted trees
// ---------------------------------------------------------------------------
// A workgroup a sequence, a thread a token, a wave a word of the masks.  In its wave each token starts with its own bit
// and jumps to its parent; a round adds the bits of the token jumped to and doubles the jump, so at most six rounds of
// shuffles reach every ancestor of the wave, and the token before the wave's that the chain goes on to.  After one
// barrier each token follows these to the earlier waves, a word a hop, up to seven.  Bound by latency: 64 trees of up to
// 500 tokens take 5.0 us, 8 of 64 tokens 2.1.  (Doubling over the whole sequence, nine rounds of LDS between barriers with
// every word of the masks: 10.6 and 2.7.)
__global__ __launch_bounds__(CKV_MAX_DRAFT) void tree_plan_kernel(const int32_t* __restrict__ parents,
                                                                  const int32_t* __restrict__ counts, int tokens,
                                                                  int32_t* __restrict__ depths,
                                                                  uint64_t* __restrict__ masks, int32_t* kept) {
  __shared__ uint64_t own_s[CKV_MAX_DRAFT];  // a token's bits in its own word
  __shared__ int before_s[CKV_MAX_DRAFT];    // its last ancestor before that word, or -1
  const int b = blockIdx.x, t = threadIdx.x, lane = t & 63, words = (tokens + 63) >> 6;
  const int count = step_count(counts, tokens, b);
  if (kept && t == 0) kept[b] = count;
  int parent = -1;
  if (t < count) {
    const int p = parents[(int64_t)b * tokens + t];
    parent = p >= 0 && p < t ? p : -1;
  }
  const bool inside = parent >= t - lane;  // in the same wave
  int jump = inside ? parent & 63 : -1, before = inside ? -1 : parent;
  uint64_t own = t < count ? 1ull << lane : 0ull;
  while (__ballot(jump >= 0) != 0) {
    const int from = jump >= 0 ? jump : lane;
    own |= (uint64_t)__shfl((unsigned long long)own, from, 64);
    before = __shfl(before, from, 64);
    const int next = __shfl(jump, from, 64);
    if (jump >= 0) jump = next;
  }
  own_s[t] = own;
  before_s[t] = before;
  __syncthreads();
  uint64_t mine[MAX_WORDS];
#pragma unroll
  for (int w = MAX_WORDS - 1; w >= 0; --w) {
    mine[w] = w == t >> 6 ? own : 0ull;
    if (before >= 0 && before >> 6 == w) {
      mine[w] = own_s[before];
      before = before_s[before];
    }
  }
  if (t >= tokens) return;
  int kin = 0;
#pragma unroll
  for (int w = 0; w < MAX_WORDS; ++w) {
    if (w < words) {
      masks[((int64_t)b * tokens + t) * words + w] = mine[w];
      kin += __popcll(mine[w]);
    }
  }
  depths[(int64_t)b * tokens + t] = max(kin - 1, 0);
}

// ---------------------------------------------------------------------------
// Writing a step's rows
// ---------------------------------------------------------------------------
struct AppendArgs {
  ckv_paged_cache cache;
  ckv_quant_rows key, value, query;
  ckv_rotary rotary;  // dim 0: none
  const int32_t* counts;
  const int32_t* depths;
  void* query_out;
  int64_t layer_offset;  // elements before this layer's pages
  int32_t tokens, query_heads, shares;  // a token's rows are shared out, eight a wave
};

// Eight values as 32 bits (the loads alone; a later use waits for them).
template <int DT>
struct Eight {
  uint4 raw[DT == CKV_F32 ? 2 : 1];
  __device__ void load(const void* base, int64_t index) {
    if constexpr (DT == CKV_F32) {
      raw[0] = gload16(reinterpret_cast<const float*>(base) + index);
      raw[1] = gload16(reinterpret_cast<const float*>(base) + index + 4);
    } else {
      raw[0] = gload16(reinterpret_cast<const uint16_t*>(base) + index);
    }
  }
  __device__ void values(float* out) const {
    if constexpr (DT == CKV_F32) {
      const uint32_t w[8] = {raw[0].x, raw[0].y, raw[0].z, raw[0].w, raw[1].x, raw[1].y, raw[1].z, raw[1].w};
#pragma unroll
      for (int i = 0; i < 8; ++i) out[i] = ckv_u2f(w[i]);
    } else {
      const uint32_t w[4] = {raw[0].x, raw[0].y, raw[0].z, raw[0].w};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        out[2 * i] = low_value<DT>(w[i]);
        out[2 * i + 1] = high_value<DT>(w[i]);
      }
    }
  }
};

template <int DT>
__device__ inline uint4 pack8(const float* v) {
  return uint4{pack_store<DT>(v[0], v[1]), pack_store<DT>(v[2], v[3]), pack_store<DT>(v[4], v[5]),
               pack_store<DT>(v[6], v[7])};
}

// A wave takes eight of a token's rows (keys, queries, values of all heads): eight lanes a row, two pieces of eight dims
// a lane, which pair up under the rotation.  Bound by memory: 32,768 tokens of 32/8 heads take 140 us, 5.8 TB/s (a large
// copy reaches 4.8).  A wave that takes more rows of its token reads the angles once for them, but they come from cache
// anyway and it has less in flight: 152 us against 145 with a quarter of the waves; 4,096 tokens 19.1 against 18.4.
template <int IN, int STORE>
__global__ __launch_bounds__(THREADS) void append_kernel(const AppendArgs a) {
  const ckv_paged_cache& c = a.cache;
  const int b = blockIdx.y, lane = threadIdx.x & 63, group = lane >> 3, x = lane & 7;
  const int number = __builtin_amdgcn_readfirstlane(blockIdx.x * (THREADS / 64) + (threadIdx.x >> 6));
  const int t = number / a.shares, share = number - t * a.shares;
  if (t >= a.tokens) return;
  const int start = paged_length(c, b), count = step_count(a.counts, a.tokens, b);
  const bool live = t < count;
  const int heads = c.kv_heads, turned = heads + a.query_heads, rows = turned + heads;
  const int half = a.rotary.dim >> 1, pairs = half >> 3;  // pieces of eight dims that are turned, two by two
  // this lane's two pieces of a row: partners under the rotation, or two of the dims that stay
  const int first = x < pairs ? (a.rotary.interleaved ? 2 * x : x) : 2 * x;
  const int second = x < pairs ? (a.rotary.interleaved ? 2 * x + 1 : x + pairs) : 2 * x + 1;
  const int r = 8 * share + group;
  const bool is_query = r >= heads && r < turned;
  const int head = r < heads ? r : is_query ? r - heads : r - turned;
  const ckv_quant_rows& from = r < heads ? a.key : is_query ? a.query : a.value;
  Eight<IN> piece[2];
  if (live && r < rows) {  // before the page is known: its latency and the angles' pass meanwhile
    const int64_t base = (int64_t)b * from.batch_stride + (int64_t)head * from.head_stride + (int64_t)t * from.token_stride;
    piece[0].load(from.data, base + 8 * first);
    piece[1].load(from.data, base + 8 * second);
  }
  float cosine[8], sine[8];
  int64_t to = -1;  // this token's row in head 0
  if (live) {
    const int row = start + t;
    int page = -1;
    if (row < paged_capacity(c)) page = gload_i32(c.page_table + (int64_t)b * c.table_pages + (row >> paged_log2(c)));
    if (x < pairs && 8 * share < turned) {
      const int depth = a.depths ? draft_depth(a.depths, (int64_t)b * a.tokens + t) : t;
      const int64_t at = (int64_t)min(start + depth, a.rotary.positions - 1) * half + 8 * x;
      Eight<CKV_F32> table[2];
      table[0].load(a.rotary.cosines, at);
      table[1].load(a.rotary.sines, at);
      table[0].values(cosine);
      table[1].values(sine);
    }
    if ((uint32_t)page < (uint32_t)c.pages)
      to = a.layer_offset + ((int64_t)page * heads * c.page_size + (row & (c.page_size - 1))) * D;
    else if (share == 0 && lane == 0)
      c.overflow[b] = 1;
  }
  if (r >= rows || (!is_query && to < 0)) return;
  uint16_t* out;
  if (is_query)
    out = reinterpret_cast<uint16_t*>(a.query_out) + (((int64_t)b * a.tokens + t) * a.query_heads + head) * D;
  else
    out = reinterpret_cast<uint16_t*>(r < heads ? c.key_pages : c.value_pages) + to + (int64_t)head * c.page_size * D;
  if (!live) {  // a query past the count
    *reinterpret_cast<uint4*>(out + 8 * first) = uint4{0, 0, 0, 0};
    *reinterpret_cast<uint4*>(out + 8 * second) = uint4{0, 0, 0, 0};
    return;
  }
  if (IN == STORE && (r >= turned || x >= pairs)) {
    *reinterpret_cast<uint4*>(out + 8 * first) = piece[0].raw[0];
    *reinterpret_cast<uint4*>(out + 8 * second) = piece[1].raw[0];
    return;
  }
  float u[8], v[8];
  piece[0].values(u);
  piece[1].values(v);
  if (r < turned && x < pairs) {
    if (a.rotary.interleaved) {
      // the two pieces hold the pairs 8 x .. 8 x + 7, four each
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float p = u[2 * i], q = u[2 * i + 1], s = v[2 * i], w = v[2 * i + 1];
        u[2 * i] = __builtin_fmaf(p, cosine[i], -(q * sine[i]));
        u[2 * i + 1] = __builtin_fmaf(q, cosine[i], p * sine[i]);
        v[2 * i] = __builtin_fmaf(s, cosine[4 + i], -(w * sine[4 + i]));
        v[2 * i + 1] = __builtin_fmaf(w, cosine[4 + i], s * sine[4 + i]);
      }
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float p = u[i], q = v[i];
        u[i] = __builtin_fmaf(p, cosine[i], -(q * sine[i]));
        v[i] = __builtin_fmaf(q, cosine[i], p * sine[i]);
      }
    }
  }
  *reinterpret_cast<uint4*>(out + 8 * first) = pack8<STORE>(u);
  *reinterpret_cast<uint4*>(out + 8 * second) = pack8<STORE>(v);
}

template <int IN>
int launch_append(AppendArgs& a, hipStream_t s) {
  a.shares = (2 * a.cache.kv_heads + a.query_heads + 7) / 8;
  const int64_t blocks = ((int64_t)a.tokens * a.shares + THREADS / 64 - 1) / (THREADS / 64);
  if (blocks * THREADS > 0xffffffffll) return paged_error(CKV_E_LIMIT, "ckv_paged_append", "too many tokens");
  const dim3 grid((uint32_t)blocks, a.cache.batch);
  if (a.cache.dtype == CKV_BF16) append_kernel<IN, CKV_BF16><<<grid, THREADS, 0, s>>>(a);
  else append_kernel<IN, CKV_F16><<<grid, THREADS, 0, s>>>(a);
  return paged_launched("ckv_paged_append");
}

// ---------------------------------------------------------------------------
// Committing a step
// ---------------------------------------------------------------------------
struct CommitArgs {
  ckv_paged_cache cache;
  const int32_t* counts;
  const int32_t* path;
  int32_t tokens, path_tokens;
};

// Tokens of sequence b to commit, as far as there are so many.
__device__ inline int commit_count(const CommitArgs& a, int b) { return a.counts ? max(gload_i32(a.counts + b), 0) : a.tokens; }

// Entries of sequence b's path that count: up to the first that does not ascend or lies past the table's rows (`room`).
__device__ inline int path_length(const CommitArgs& a, int b, int room) {
  const int lane = threadIdx.x & 63, count = min(commit_count(a, b), a.path_tokens);
  const int32_t* path = a.path + (int64_t)b * a.path_tokens;
  for (int j0 = 0; j0 < count; j0 += 64) {
    const int j = j0 + lane;
    bool bad = false;
    if (j < count) {
      const int p = path[j];
      bad = p >= room || p <= (j ? path[j - 1] : -1);
    }
    const uint64_t hit = __ballot(bad);
    if (hit) return j0 + __ffsll((unsigned long long)hit) - 1;
  }
  return count;
}

constexpr int COUNTER_STRIDE = CKV_QUANT_COUNTERS;  // words between two sequences' counters: a cache line each (in one: 11.7 us)
constexpr int MOVE_LOADS = 4;  // of four rows each
// Workgroups of a sequence, each of which takes a ticket of its counter.  More move more at once, and queue at it: 36
// layers of 8 sequences take 16.7 us with 8, 10.3 with 16, 7.5 with 32, 6.9 with 64, 7.2 with 128.
constexpr int MOVE_WORKGROUPS = 64;

// A wave takes (layer, head, keys or values) of a sequence in turn: 16 lanes a row, 16 rows at a time.  The entries ascend, so
// entry j's source is row j or a later one and no later entry reads what an earlier one wrote; within a batch every
// load is issued before the first store.  Rows whose page is none stay where they are.  Bound by latency, a chain of
// cursor, path, pages, rows: 6.7 us for paths of up to 7 tokens in 36 layers of 8 sequences, 4.5 for 4 layers of one
// (moving in one launch and advancing in another: 2 us more on the host).
__global__ __launch_bounds__(THREADS) void move_kernel(const CommitArgs a) {
  const ckv_paged_cache& c = a.cache;
  const int b = blockIdx.y, lane = threadIdx.x & 63;
  const int start = paged_length(c, b), size = path_length(a, b, paged_capacity(c) - start);
  // every wave has read the length: the last workgroup to come here writes the new one
  __syncthreads();
  if (threadIdx.x == 0 && atomicAdd(c.counters + b * COUNTER_STRIDE, 1u) == gridDim.x - 1) {
    c.counters[b * COUNTER_STRIDE] = 0;
    c.lengths[b] = start + size;
  }
  const int64_t head_rows = (int64_t)c.kv_heads * c.page_size;
  const int32_t* table = c.page_table + (int64_t)b * c.table_pages;
  const int32_t* path = a.path + (int64_t)b * a.path_tokens;
  const int planes = 2 * c.layers * c.kv_heads;
  for (int number = blockIdx.x * (THREADS / 64) + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6); number < planes;
       number += gridDim.x * (THREADS / 64)) {
    const int head = number % c.kv_heads, plane = number / c.kv_heads, layer = plane >> 1;
    uint16_t* pages = reinterpret_cast<uint16_t*>(plane & 1 ? c.value_pages : c.key_pages) +
                      ((int64_t)layer * c.pages * head_rows + (int64_t)head * c.page_size) * D + 8 * (lane & 15);
    for (int j0 = 0; j0 < size; j0 += 4 * MOVE_LOADS) {
      uint4 w[MOVE_LOADS];
      int64_t to[MOVE_LOADS];
#pragma unroll
      for (int i = 0; i < MOVE_LOADS; ++i) {
        const int j = j0 + 4 * i + (lane >> 4);
        to[i] = -1;
        if (j >= size || path[j] == j) continue;
        const int source = start + path[j], row = start + j;
        const int from_page = gload_i32(table + (source >> paged_log2(c))), page = gload_i32(table + (row >> paged_log2(c)));
        if ((uint32_t)from_page >= (uint32_t)c.pages || (uint32_t)page >= (uint32_t)c.pages) continue;
        w[i] = gload16(pages + (from_page * head_rows + (source & (c.page_size - 1))) * D);
        to[i] = (page * head_rows + (row & (c.page_size - 1))) * D;
      }
#pragma unroll
      for (int i = 0; i < MOVE_LOADS; ++i)
        if (to[i] >= 0) *reinterpret_cast<uint4*>(pages + to[i]) = w[i];
    }
  }
}

// Without a path: a wave a sequence.
__global__ __launch_bounds__(64) void advance_kernel(const CommitArgs a) {
  const ckv_paged_cache& c = a.cache;
  const int b = blockIdx.x, start = paged_length(c, b);
  if (threadIdx.x == 0) c.lengths[b] = start + min(commit_count(a, b), paged_capacity(c) - start);
}

}  // namespace

extern "C" int ckv_draft_tree_plan_counts(const int32_t* parents, const int32_t* counts, int32_t batch, int32_t tokens,
                                          int32_t* depths, uint64_t* masks, int32_t* counts_out, void* stream) {
  const char* what = "ckv_draft_tree_plan";
  if (!parents || !depths || !masks) return paged_error(CKV_E_INVALID, what, "null argument");
  if (batch <= 0 || tokens <= 0) return paged_error(CKV_E_INVALID, what, "batch and tokens must be positive");
  if (tokens > CKV_MAX_DRAFT) return paged_error(CKV_E_LIMIT, what, "more than 512 tokens");
  tree_plan_kernel<<<batch, (tokens + 63) / 64 * 64, 0, reinterpret_cast<hipStream_t>(stream)>>>(parents, counts, tokens,
                                                                                                 depths, masks, counts_out);
  return paged_launched(what);
}

extern "C" int ckv_draft_tree_plan(const int32_t* parents, const int32_t* counts, int32_t batch, int32_t tokens,
                                   int32_t* depths, uint64_t* masks, void* stream) {
  return ckv_draft_tree_plan_counts(parents, counts, batch, tokens, depths, masks, nullptr, stream);
}

extern "C" int ckv_paged_append(const ckv_paged_cache* cache, const ckv_paged_append_args* args, void* stream) {
  const char* what = "ckv_paged_append";
  int rc = validate_paged_cache(cache, what);
  if (rc) return rc;
  if (!args) return paged_error(CKV_E_INVALID, what, "null argument");
  const ckv_rotary* rotary = args->rotary;
  const bool query = args->query.data != nullptr;
  if (args->layer < 0 || args->layer >= cache->layers) return paged_error(CKV_E_INVALID, what, "no such layer");
  if (args->dtype != CKV_BF16 && args->dtype != CKV_F16 && args->dtype != CKV_F32)
    return paged_error(CKV_E_INVALID, what, "dtype must be bf16, fp16 or f32");
  if (args->tokens <= 0) return paged_error(CKV_E_INVALID, what, "tokens must be positive");
  rc = check_paged_rows(&args->key, args->dtype, what);
  if (!rc) rc = check_paged_rows(&args->value, args->dtype, what);
  if (!rc && query) rc = check_paged_rows(&args->query, args->dtype, what);
  if (rc) return rc;
  if (query && (!args->query_out || ((uintptr_t)args->query_out & 15) || !rotary || args->query_heads <= 0 ||
                args->query_heads > (1 << 20)))
    return paged_error(CKV_E_INVALID, what, "a query needs its output, its heads and the rotation");
  if (rotary) {
    if (!rotary->cosines || !rotary->sines || (((uintptr_t)rotary->cosines | (uintptr_t)rotary->sines) & 15))
      return paged_error(CKV_E_INVALID, what, "rotation tables must be 16-byte aligned");
    if (rotary->dim < 16 || rotary->dim > D || rotary->dim % 16)
      return paged_error(CKV_E_INVALID, what, "rotated dims must be a multiple of 16, at most 128");
    if (rotary->positions < paged_capacity(*cache))
      return paged_error(CKV_E_INVALID, what, "the rotation tables hold fewer positions than a sequence's rows");
  }
  AppendArgs a{};
  a.cache = *cache;
  a.key = args->key;
  a.value = args->value;
  a.query = args->query;
  if (rotary) a.rotary = *rotary;
  a.counts = args->counts;
  a.depths = args->depths;
  a.query_out = args->query_out;
  a.layer_offset = (int64_t)args->layer * cache->pages * cache->kv_heads * cache->page_size * D;
  a.tokens = args->tokens;
  a.query_heads = query ? args->query_heads : 0;
  const hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  if (args->dtype == CKV_BF16) return launch_append<CKV_BF16>(a, s);
  if (args->dtype == CKV_F16) return launch_append<CKV_F16>(a, s);
  return launch_append<CKV_F32>(a, s);
}

extern "C" int ckv_paged_commit(const ckv_paged_cache* cache, int32_t tokens, const int32_t* counts, const int32_t* path,
                                int32_t path_tokens, void* stream) {
  const char* what = "ckv_paged_commit";
  const int rc = validate_paged_cache(cache, what);
  if (rc) return rc;
  if (tokens < 0) return paged_error(CKV_E_INVALID, what, "tokens must not be negative");
  if (path && path_tokens <= 0) return paged_error(CKV_E_INVALID, what, "an empty path");
  if (path && path_tokens > CKV_MAX_DRAFT) return paged_error(CKV_E_LIMIT, what, "a path of more than 512 tokens");
  const CommitArgs a{*cache, counts, path, tokens, path_tokens};
  const hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  if (path) {
    const int64_t waves = 2 * (int64_t)cache->layers * cache->kv_heads, blocks = (waves + THREADS / 64 - 1) / (THREADS / 64);
    if (waves > 0x3fffffff) return paged_error(CKV_E_LIMIT, what, "too many layers");
    move_kernel<<<dim3((uint32_t)(blocks < MOVE_WORKGROUPS ? blocks : MOVE_WORKGROUPS), cache->batch), THREADS, 0, s>>>(a);
    return paged_launched(what);
  }
  advance_kernel<<<cache->batch, 64, 0, s>>>(a);
  return paged_launched(what);
}
