// The paged key/value cache of a serving step: the plan that gives every new
// token its position and slot (smx_paged_plan), and the pass that normalises,
// rotates and stores the new heads (smx_paged_write).
#include "launch.hpp"

namespace smx {
namespace {

// ---------------------------------------------------------------------------
// Plan
// ---------------------------------------------------------------------------

struct PlanArgs {
  const int32_t* context;
  const int32_t* fresh;
  int32_t* tables;
  int64_t table_stride;
  const int32_t* free_pages;
  int32_t *starts, *rows, *known, *positions, *status, *pages;
  int64_t* slots;
  int32_t requests, width, page_shift, num_pages, tokens, max_new, max_context, free_count;
};

// Inclusive sum of x over the workgroup's threads; *total: the whole sum. Both fit 32 bits: 1024
// lengths of at most SMX_PAGED_MAX_TOKENS + 1, or the pages of requests whose rows lie within the step.
// Two barriers; `waves` holds one partial sum per wave.
__device__ int32_t block_scan(int32_t x, int32_t* waves, int32_t* total) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, count = blockDim.x >> 6;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const int32_t y = __shfl_up(x, d);
    if (lane >= d) x += y;
  }
  if (lane == 63) waves[wave] = x;
  __syncthreads();
  int32_t before = 0, all = 0;
  for (int w = 0; w < count; ++w) {
    const int32_t s = waves[w];
    if (w < wave) before += s;
    all += s;
  }
  __syncthreads();
  *total = all;
  return x + before;
}

// Whether entries first .. last of a request's table, for the lanes of a wave with `wanted`, are all pages of the
// cache. A lane looks at its own request's entries where they are few; the long lists of a prompt are
// looked through by the whole wave, one request after another. All lanes take part.
__device__ bool pages_there(const PlanArgs& p, bool wanted, const int32_t* table, int32_t first, int32_t last) {
  constexpr int32_t kOwn = 4;
  bool there = true;
  const bool few = last - first < kOwn;
  if (wanted && few)
    for (int32_t i = first; i <= last; ++i) there &= (uint32_t)table[i] < (uint32_t)p.num_pages;
  for (uint64_t left = __ballot(wanted && !few); left; left &= left - 1) {
    const int who = __builtin_ctzll(left), lane = threadIdx.x & 63;
    const auto* const theirs = (const int32_t*)__shfl((int64_t)(uintptr_t)table, who);
    const int32_t from = __shfl(first, who), to = __shfl(last, who);
    bool all = true;
#pragma unroll 4
    for (int32_t i = from + lane; i <= to; i += 64) all &= (uint32_t)theirs[i] < (uint32_t)p.num_pages;
    if (!__all(all) && lane == who) there = false;
  }
  return there;
}

// Every workgroup scans the requests for itself (a few thousand integers, in
// cache after the first) and lays out its own tokens, so that one launch does
// without a second one behind it: with c the context, n the new tokens and P
// the page size, request b's rows start at the sum of the n before it, and it
// needs ceil((c + n) / P) - ceil(c / P) new pages, taken from the free list in
// request order. LDS: [requests + 1] row starts, then [requests] offsets into the
// free list (-1: not admitted). What bounds it is latency: one load of
// the lengths, two scans, one dependent load per token: 4.4 us at 16 requests,
// 11.7 us at 2048 (13.0 with 64-bit scans).
__global__ __launch_bounds__(1024) void paged_plan(PlanArgs p) {
  extern __shared__ int32_t plan_lds[];
  __shared__ int32_t waves[16], most[32];
  int32_t* const start_of = plan_lds;
  int32_t* const pages_of = plan_lds + p.requests + 1;
  const bool first = blockIdx.x == 0;
  const int32_t mask = (1 << p.page_shift) - 1;
  const int64_t limit = (int64_t)p.tokens + 1;

  int64_t row_base = 0, page_base = 0, used = 0, needed = 0;
  for (int32_t at = 0; at < p.requests; at += blockDim.x) {
    const int32_t b = at + (int32_t)threadIdx.x;
    const bool here = b < p.requests;
    const int64_t c = here ? p.context[b] : 0, given = here ? p.fresh[b] : 0;
    // A length beyond the step's tokens counts as one more than they are, so
    // that the sums stay small and everything behind it is out of rows.
    const int64_t n = min(max(given, (int64_t)0), limit);
    int32_t total;
    const int64_t upto = block_scan((int32_t)n, waves, &total);
    const int64_t start = row_base + upto - n;
    row_base += total;
    int32_t status = SMX_PAGED_OK;
    if (c < 0 || given < 0 || given > p.max_new || c + given > p.max_context) {
      status = SMX_PAGED_BAD_LENGTH;
    } else if (n > 0 && start + n > p.tokens) {
      status = SMX_PAGED_OUT_OF_ROWS;
    }
    // The new tokens' pages that have to be there: that which the context ends in, which the first one joins, and
    // without a free list all of them.
    const bool joins = status == SMX_PAGED_OK && n > 0 && ((c & mask) || !p.free_pages);
    const int32_t page0 = (int32_t)(c >> p.page_shift);
    const int32_t page1 = joins && !p.free_pages ? (int32_t)((c + n - 1) >> p.page_shift) : page0;
    if (!pages_there(p, joins, p.tables + b * p.table_stride, page0, page1)) status = SMX_PAGED_BAD_PAGE;
    const int64_t held = (c + mask) >> p.page_shift;
    const int64_t need =
        here && p.free_pages && status == SMX_PAGED_OK && n > 0 ? ((c + n + mask) >> p.page_shift) - held : 0;
    const int64_t pages = page_base + block_scan((int32_t)need, waves, &total);
    page_base += total;
    if (need > 0 && pages > p.free_count) status = SMX_PAGED_OUT_OF_PAGES;
    if (status == SMX_PAGED_OK) {
      if (need > 0) used = pages;
      if (here) needed = pages;
    }
    if (!here) continue;
    start_of[b] = (int32_t)min(start, (int64_t)INT32_MAX);
    pages_of[b] = status == SMX_PAGED_OK ? (int32_t)(pages - need) : -1;
    if (first) {
      p.starts[b] = start_of[b];
      p.status[b] = status;
      p.rows[b] = status == SMX_PAGED_OK ? (int32_t)n : 0;
      p.known[b] = status == SMX_PAGED_OK ? (int32_t)c : 0;
    }
  }
  if (threadIdx.x == 0) {
    start_of[p.requests] = (int32_t)min(row_base, (int64_t)INT32_MAX);
    if (first) p.starts[p.requests] = start_of[p.requests];
  }
  if (first) {
    // the free pages taken, and those needed up to the last admitted request: inclusive sums
    // of the demand, which grow from request to request
    int32_t taken = (int32_t)used, asked = (int32_t)needed;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) taken = max(taken, __shfl_xor(taken, d)), asked = max(asked, __shfl_xor(asked, d));
    if ((threadIdx.x & 63) == 0) most[threadIdx.x >> 6] = taken, most[16 + (threadIdx.x >> 6)] = asked;
    __syncthreads();
    if (threadIdx.x == 0) {
      for (int w = 1; w < (int)(blockDim.x >> 6); ++w) taken = max(taken, most[w]), asked = max(asked, most[16 + w]);
      p.pages[0] = taken;
      p.pages[1] = asked;
    }
  }
  __syncthreads();

  for (int64_t r = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; r < p.tokens; r += (int64_t)gridDim.x * blockDim.x) {
    // the last request that starts at or before row r
    int32_t low = 0, high = p.requests;
    while (high - low > 1) {
      const int32_t mid = (low + high) >> 1;
      if (start_of[mid] <= r) low = mid; else high = mid;
    }
    const int32_t place = (int32_t)r - start_of[low];
    int32_t position = -1;
    int64_t slot = -1;
    if (r < start_of[low + 1] && pages_of[low] >= 0) {
      const int32_t c = p.context[low];
      position = c + place;
      const int32_t index = position >> p.page_shift;
      const int32_t held = (int32_t)(((int64_t)c + mask) >> p.page_shift);
      int32_t* const entry = p.tables + low * p.table_stride + index;
      int32_t page;
      if (p.free_pages && index >= held) {
        page = p.free_pages[pages_of[low] + index - held];
        if (!(position & mask)) *entry = page;  // one token, the page's first, fills the entry in
      } else {
        page = *entry;
      }
      if ((uint32_t)page < (uint32_t)p.num_pages)
        slot = ((int64_t)page << p.page_shift) + (position & mask);
    }
    p.positions[r] = position;
    p.slots[r] = slot;
  }
}

// ---------------------------------------------------------------------------
// Write
// ---------------------------------------------------------------------------

struct WriteArgs {
  const uint16_t *q, *k, *v;
  int64_t q_token, q_head, k_token, k_head, v_token, v_head;  // strides in elements
  uint16_t *k_cache, *v_cache;
  int64_t page_stride, slot_stride, head_stride;
  const int32_t* positions;
  const int64_t* slots;
  const void *cos, *sin, *q_scale, *k_scale;
  int64_t rope_stride;
  int32_t rope_rows, dtypes;
  float eps;
  uint16_t* out;  // [tokens, heads, head_dim]
  int32_t tokens, heads, kv_heads, page_shift;
  int64_t slot_count;
};

__device__ __forceinline__ F8 load8f(const void* p, int f32, int64_t at) {
  if (!f32) return unpack8(*reinterpret_cast<const u32x4*>(reinterpret_cast<const uint16_t*>(p) + at));
  const f32x4* const x = reinterpret_cast<const f32x4*>(reinterpret_cast<const float*>(p) + at);
  F8 r;
#pragma unroll
  for (int i = 0; i < 4; ++i) r.v[i] = x[0][i], r.v[4 + i] = x[1][i];
  return r;
}

// One head row per D / 16 lanes: lane l holds columns 8 l .. 8 l + 7 of the
// first half (a) and of the second (b), so that a rotation pairs values of one
// lane: a' = a cos - b sin, b' = b cos + a sin. The norm is x / sqrt(mean x^2 + eps)
// * scale. All of it in FP32, rounded to bf16 once at the store. Bound by memory: each
// head is read once and written once (tables and scales come from cache): 8192 tokens of 80 heads 66 us,
// 5.1 TB/s; 16 tokens 4 us.
template <int D>
__global__ __launch_bounds__(256) void paged_write(WriteArgs w) {
  constexpr int kLanes = D / 16, kHeads = 256 / kLanes;
  const int lane = threadIdx.x % kLanes;
  const int32_t q_heads = w.out ? w.heads : 0, per_token = q_heads + 2 * w.kv_heads;
  const int64_t item = (int64_t)blockIdx.x * kHeads + threadIdx.x / kLanes;
  const int64_t token = item / per_token;
  if (token >= w.tokens) return;  // whole head rows: uniform over a head's lanes
  const int32_t head = (int32_t)(item - token * per_token);
  const int32_t position = w.positions[token];
  const bool is_q = head < q_heads, is_k = !is_q && head < q_heads + w.kv_heads;
  const int32_t kv = is_q ? 0 : is_k ? head - q_heads : head - q_heads - w.kv_heads;

  uint16_t* to;
  if (is_q) {
    to = w.out + (token * w.heads + head) * D;
    if (position < 0) {  // no request's row: zero
      const u32x4 zero = {0, 0, 0, 0};
      *reinterpret_cast<u32x4*>(to + 8 * lane) = zero;
      *reinterpret_cast<u32x4*>(to + D / 2 + 8 * lane) = zero;
      return;
    }
  } else {
    const int64_t slot = w.slots[token];
    if (slot < 0 || slot >= w.slot_count) return;
    to = (is_k ? w.k_cache : w.v_cache) + (slot >> w.page_shift) * w.page_stride +
         (slot & ((1 << w.page_shift) - 1)) * w.slot_stride + kv * w.head_stride;
  }
  const uint16_t* const from = is_q   ? w.q + token * w.q_token + head * w.q_head
                               : is_k ? w.k + token * w.k_token + kv * w.k_head
                                      : w.v + token * w.v_token + kv * w.v_head;
  u32x4 a_bits = *reinterpret_cast<const u32x4*>(from + 8 * lane);
  u32x4 b_bits = *reinterpret_cast<const u32x4*>(from + D / 2 + 8 * lane);
  const void* const scale = is_q ? w.q_scale : is_k ? w.k_scale : nullptr;
  const bool rotate = w.cos && (is_q || is_k);
  if (scale || rotate) {
    F8 a = unpack8(a_bits), b = unpack8(b_bits);
    if (scale) {
      float sum = 0.f;
#pragma unroll
      for (int i = 0; i < 8; ++i) sum += a.v[i] * a.v[i] + b.v[i] * b.v[i];
#pragma unroll
      for (int d = 1; d < kLanes; d <<= 1) sum += __shfl_xor(sum, d);
      const float r = 1.0f / sqrtf(sum * (1.0f / D) + w.eps);
      const int f32 = w.dtypes & (is_q ? SMX_PAGED_Q_SCALE_F32 : SMX_PAGED_K_SCALE_F32);
      const F8 sa = load8f(scale, f32, 8 * lane), sb = load8f(scale, f32, D / 2 + 8 * lane);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        a.v[i] = a.v[i] * r * sa.v[i];
        b.v[i] = b.v[i] * r * sb.v[i];
      }
    }
    if (rotate) {
      const int64_t at = (int64_t)min(max(position, 0), w.rope_rows - 1) * w.rope_stride + 8 * lane;
      const int f32 = w.dtypes & SMX_PAGED_ROPE_F32;
      const F8 cs = load8f(w.cos, f32, at), sn = load8f(w.sin, f32, at);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float x = a.v[i], y = b.v[i];
        a.v[i] = x * cs.v[i] - y * sn.v[i];
        b.v[i] = y * cs.v[i] + x * sn.v[i];
      }
    }
    a_bits = pack8(a);
    b_bits = pack8(b);
  }
  *reinterpret_cast<u32x4*>(to + 8 * lane) = a_bits;
  *reinterpret_cast<u32x4*>(to + D / 2 + 8 * lane) = b_bits;
}

bool aligned16(const void* p) { return ((uintptr_t)p & 15) == 0; }

}  // namespace

int paged_layout(const smx_paged_cache* c) {
  if (!c || !c->k || !c->v) return fail(SMX_ERR_INVALID, "null cache");
  if (c->num_pages <= 0 || c->kv_heads <= 0 || c->kv_heads > 65535)
    return fail(SMX_ERR_INVALID, "the cache needs pages and 1 to 65535 heads (num_pages=%d, kv_heads=%d)",
                c->num_pages, c->kv_heads);
  if (c->page_size < 8 || c->page_size > 4096 || (c->page_size & (c->page_size - 1)))
    return fail(SMX_ERR_INVALID, "page_size must be a power of two from 8 to 4096, got %d", c->page_size);
  if (c->head_dim != 64 && c->head_dim != 128)
    return fail(SMX_ERR_UNSUPPORTED, "head_dim must be 64 or 128, got %d", c->head_dim);
  if ((int64_t)c->num_pages * c->page_size > INT32_MAX) return fail(SMX_ERR_UNSUPPORTED, "too many slots");
  if (!aligned16(c->k) || !aligned16(c->v) || c->page_stride % 8 || c->slot_stride % 8 || c->head_stride % 8)
    return fail(SMX_ERR_INVALID, "cache rows must be 16-byte aligned");
  if (c->slot_stride < c->head_dim || c->slot_stride > (1 << 26) || c->page_stride < c->head_dim ||
      c->head_stride < c->head_dim)
    return fail(SMX_ERR_INVALID, "cache strides must be at least head_dim and its slots at most 2^26 elements apart");
  if (c->page_stride > INT32_MAX || c->head_stride > INT32_MAX)
    return fail(SMX_ERR_UNSUPPORTED, "pages and heads may be at most 2^31 - 1 elements apart");
  return SMX_OK;
}

}  // namespace smx

using namespace smx;

extern "C" {

int smx_paged_plan(int32_t requests, int32_t width, int32_t page_size, int32_t num_pages, int32_t tokens,
                   int32_t max_new, int32_t max_context, const int32_t* context_lens, const int32_t* new_lens,
                   int32_t* block_tables, int64_t table_stride, const int32_t* free_pages, int32_t free_count,
                   int32_t* starts, int32_t* rows, int32_t* context, int32_t* positions, int64_t* slots,
                   int32_t* status, int32_t* pages, void* stream) {
  smx::fail(SMX_OK, "%s", "");
  if (requests <= 0 || requests > SMX_PAGED_MAX_REQUESTS)
    return fail(SMX_ERR_INVALID, "a plan takes 1 to %d requests, got %d", SMX_PAGED_MAX_REQUESTS, requests);
  if (tokens <= 0 || tokens > SMX_PAGED_MAX_TOKENS)
    return fail(SMX_ERR_INVALID, "a plan takes 1 to %d tokens, got %d", SMX_PAGED_MAX_TOKENS, tokens);
  if (page_size < 8 || page_size > 4096 || (page_size & (page_size - 1)))
    return fail(SMX_ERR_INVALID, "page_size must be a power of two from 8 to 4096, got %d", page_size);
  if (width <= 0 || num_pages <= 0 || (int64_t)num_pages * page_size > INT32_MAX)
    return fail(SMX_ERR_INVALID, "empty or too large table or cache (width=%d, num_pages=%d)", width, num_pages);
  if (table_stride < width) return fail(SMX_ERR_INVALID, "table_stride must be at least the table's width");
  if (max_new < 0 || max_context < 0 || (int64_t)max_context > (int64_t)width * page_size ||
      max_context > SMX_PAGED_MAX_CONTEXT)
    return fail(SMX_ERR_INVALID, "max_new=%d, max_context=%d: the block tables hold %lld tokens a request, at most %d count",
                max_new, max_context, (long long)width * page_size, SMX_PAGED_MAX_CONTEXT);
  if (free_count < 0 || (free_count > 0 && !free_pages)) return fail(SMX_ERR_INVALID, "free_count without a list");
  if (!context_lens || !new_lens || !block_tables || !starts || !rows || !context || !positions || !slots ||
      !status || !pages)
    return fail(SMX_ERR_INVALID, "null pointer");
  if (free_pages) {
    // entries are filled in while other workgroups read the lists
    const struct {
      const void* list;
      int64_t count;
    } lists[] = {{context_lens, requests}, {new_lens, requests}, {free_pages, free_count}};
    for (const auto& l : lists)
      if (list_meets_table(l.list, l.count, block_tables, requests, width, table_stride, 4))
        return fail(SMX_ERR_INVALID, "block_tables must share no memory with the lengths and free_pages");
  }
  PlanArgs p{context_lens, new_lens, block_tables, table_stride, free_pages, starts, rows, context, positions,
             status, pages, slots, requests, width, __builtin_ctz(page_size), num_pages, tokens, max_new,
             max_context, free_count};
  // Small steps in four waves (their barriers are cheaper), others in sixteen;
  // at least 1024 tokens a workgroup, so that few repeat the scan.
  const int threads = requests <= 256 && tokens <= 256 ? 256 : 1024;
  const int blocks = (int)min((int64_t)256, ((int64_t)tokens + 1023) / 1024);
  const int lds = (2 * requests + 1) * 4;
  if (lds > 48 * 1024) {
    hipError_t e = hipFuncSetAttribute((const void*)paged_plan, hipFuncAttributeMaxDynamicSharedMemorySize, lds);
    if (e != hipSuccess) return fail(SMX_ERR_LAUNCH, "hipFuncSetAttribute: %s", hipGetErrorString(e));
  }
  hipLaunchKernelGGL(paged_plan, dim3((unsigned)blocks), dim3(threads), lds, (hipStream_t)stream, p);
  return check_launch();
}

int smx_paged_write(const smx_paged_cache* cache, int32_t tokens, const int32_t* positions, const int64_t* slots,
                    const smx_heads* q, const smx_heads* k, const smx_heads* v, const void* rope_cos,
                    const void* rope_sin, int32_t rope_rows, int64_t rope_stride, const void* q_scale,
                    const void* k_scale, int32_t dtypes, float eps, void* q_out, void* stream) {
  smx::fail(SMX_OK, "%s", "");
  if (int rc = paged_layout(cache)) return rc;
  if (tokens <= 0 || tokens > SMX_PAGED_MAX_TOKENS)
    return fail(SMX_ERR_INVALID, "1 to %d tokens, got %d", SMX_PAGED_MAX_TOKENS, tokens);
  if (!positions || !slots || !k || !v || !k->data || !v->data) return fail(SMX_ERR_INVALID, "null pointer");
  const bool has_q = q && q->data;
  if (has_q != (q_out != nullptr)) return fail(SMX_ERR_INVALID, "q and q_out go together");
  if (k->heads != cache->kv_heads || v->heads != cache->kv_heads)
    return fail(SMX_ERR_INVALID, "k and v must have the cache's %d heads", cache->kv_heads);
  if (has_q && (q->heads <= 0 || q->heads > 65535)) return fail(SMX_ERR_INVALID, "1 to 65535 query heads");
  for (const smx_heads* x : {has_q ? q : k, k, v})
    if (!aligned16(x->data) || x->token_stride % 8 || x->head_stride % 8 || x->token_stride < 0 || x->head_stride < 0)
      return fail(SMX_ERR_INVALID, "head rows must be 16-byte aligned");
  if (!aligned16(q_out) || !aligned16(rope_cos) || !aligned16(rope_sin) || !aligned16(q_scale) || !aligned16(k_scale))
    return fail(SMX_ERR_INVALID, "q_out, RoPE tables and scales must be 16-byte aligned");
  if ((rope_cos == nullptr) != (rope_sin == nullptr)) return fail(SMX_ERR_INVALID, "rope_cos and rope_sin go together");
  if (rope_cos && (rope_rows <= 0 || rope_stride < cache->head_dim / 2 || rope_stride % 8))
    return fail(SMX_ERR_INVALID, "RoPE tables need rows of head_dim / 2 values, 16-byte aligned");
  if (q_scale && !has_q) return fail(SMX_ERR_INVALID, "q_scale without q");
  if (dtypes & ~(SMX_PAGED_Q_SCALE_F32 | SMX_PAGED_K_SCALE_F32 | SMX_PAGED_ROPE_F32))
    return fail(SMX_ERR_INVALID, "unknown dtype bits 0x%x", dtypes);
  if (!(eps >= 0.f)) return fail(SMX_ERR_INVALID, "eps must not be negative");
  // Heads are stored while others are loaded: no stored row may be another's, nor one that is read.
  const Runs keys = cache_runs(*cache, cache->k), values = cache_runs(*cache, cache->v);
  if (!lie_apart(keys)) return fail(SMX_ERR_INVALID, "the cache holds rows that lie on each other");
  if (meet(keys, values)) return fail(SMX_ERR_INVALID, "keys and values must share no memory of the cache");
  smx_heads result = has_q ? *q : *k;
  result.data = q_out, result.head_stride = cache->head_dim, result.token_stride = (int64_t)result.heads * cache->head_dim;
  const Runs to = head_runs(result, tokens, cache->head_dim);
  for (const smx_heads* x : {has_q ? q : k, k, v}) {
    const Runs from = head_runs(*x, tokens, cache->head_dim);
    if (meet(from, keys) || meet(from, values)) return fail(SMX_ERR_INVALID, "the heads must share no memory with the cache");
    if (has_q && meet(from, to) && !(x == q && same_runs(from, to)))
      return fail(SMX_ERR_INVALID, "q_out must be the queries themselves or share no memory with the heads");
  }
  if (has_q && (meet(to, keys) || meet(to, values))) return fail(SMX_ERR_INVALID, "q_out must share no memory with the cache");
  WriteArgs w{};
  if (has_q) w.q = (const uint16_t*)q->data, w.q_token = q->token_stride, w.q_head = q->head_stride, w.heads = q->heads;
  w.k = (const uint16_t*)k->data, w.k_token = k->token_stride, w.k_head = k->head_stride;
  w.v = (const uint16_t*)v->data, w.v_token = v->token_stride, w.v_head = v->head_stride;
  w.k_cache = (uint16_t*)cache->k, w.v_cache = (uint16_t*)cache->v;
  w.page_stride = cache->page_stride, w.slot_stride = cache->slot_stride, w.head_stride = cache->head_stride;
  w.positions = positions, w.slots = slots;
  w.cos = rope_cos, w.sin = rope_sin, w.q_scale = q_scale, w.k_scale = k_scale;
  w.rope_stride = rope_stride, w.rope_rows = rope_rows, w.dtypes = dtypes, w.eps = eps;
  w.out = (uint16_t*)q_out;
  w.tokens = tokens, w.kv_heads = cache->kv_heads, w.page_shift = __builtin_ctz(cache->page_size);
  w.slot_count = (int64_t)cache->num_pages * cache->page_size;
  const int64_t items = (int64_t)tokens * (w.heads + 2 * w.kv_heads);
  const int per_block = 256 / (cache->head_dim / 16);
  const int64_t blocks = (items + per_block - 1) / per_block;
  if (blocks > INT32_MAX) return fail(SMX_ERR_UNSUPPORTED, "too many heads");
  auto kern = cache->head_dim == 128 ? paged_write<128> : paged_write<64>;
  hipLaunchKernelGGL(kern, dim3((unsigned)blocks), dim3(256), 0, (hipStream_t)stream, w);
  return check_launch();
}

}  // extern "C"
