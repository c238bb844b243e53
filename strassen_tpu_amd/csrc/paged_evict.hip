// Eviction from a paged cache by the attention weight that keys have received (smx_paged_evict).
//
// Of the n tokens of a request, each key/value head keeps `keep`: the last `recent`, and of the m older ones the
// need = keep - recent with the largest weights (ties: the lowest index). Survivors with an index below need stay
// where they are. The places of the evicted ones there are as many as the survivors behind, and the j-th of
// the one takes the j-th of the other; the recent ones move to need .. keep - 1 in order. That is the least that can be
// moved with the cache left without gaps, and no row is moved twice: of 131,000 tokens cut to 32,768 a
// head moves 24,800.
//
// evict_select (a workgroup per head and request) finds the need-th largest weight: weights as integers in their order,
// a histogram over 2048 equal parts of their range, the part that holds it, and so on until its keys fit in LDS,
// where they are compared with each other. evict_move then moves the rows.
#include "launch.hpp"

namespace smx {
namespace {

struct EvictArgs {
  uint16_t *k, *v;
  int64_t page_stride, slot_stride, head_stride;
  float* weights;  // [pages, kv_heads, page_size]
  const int32_t *context, *tables, *keep_lens;
  int64_t table_stride;
  int32_t* lens;
  int32_t requests, kv_heads, head_dim, page_shift, num_pages, keep, recent, max_context, moves, movers, tails;
  struct Found* found;  // [requests * kv_heads]
  int32_t* lists;       // [requests * kv_heads][2][moves]: slots to fill, slots to take from
};

// What evict_select leaves for evict_move: rows of the lists, those of them whose source lies among the places of the recent
// ones, and the recent ones: from index `from` to `to`.
struct Found {
  int32_t count, early, recent, from, to, unused[3];
};

constexpr int kSelectThreads = 1024, kSelectWaves = 16, kBins = 2048, kNear = 512, kQuads = 8;

// Weights in the order of their values; NaN above everything, -0 as 0.
__device__ __forceinline__ uint32_t order_of(float x) {
  const uint32_t bits = __float_as_uint(x + 0.f);
  if (x != x) return ~0u;
  return bits & 0x80000000u ? ~bits : bits | 0x80000000u;
}

__device__ __forceinline__ int wave_sum(int x) {
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) x += __shfl_xor(x, d);
  return x;
}

// Inclusive sum over a wave's lanes.
__device__ __forceinline__ int lane_scan(int x) {
  const int lane = threadIdx.x & 63;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const int y = __shfl_up(x, d);
    if (lane >= d) x += y;
  }
  return x;
}

__global__ __launch_bounds__(kSelectThreads) void evict_select(EvictArgs p) {
  const int head = blockIdx.x, request = blockIdx.y, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  Found* const found = p.found + (int64_t)request * p.kv_heads + head;
  __shared__ int bins[kBins], waves[kSelectWaves][8], bad, near_count;
  __shared__ uint32_t near[kNear], low_key, high_key, edge_key;
  __shared__ int edge_ties, early, picked[2];
  const int32_t n = p.context[request], given = p.keep_lens ? p.keep_lens[request] : p.keep;
  const int32_t* const table = p.tables + request * p.table_stride;
  const int32_t mask = (1 << p.page_shift) - 1;
  if (threadIdx.x == 0) bad = near_count = early = 0, low_key = ~0u, high_key = 0;
  __syncthreads();
  bool whole = n <= given || n > p.max_context || given < 0;
  if (!whole)  // every page of the request has to be there (uniform bounds)
    for (int i = threadIdx.x; i <= (n - 1) >> p.page_shift; i += kSelectThreads)
      if ((uint32_t)table[i] >= (uint32_t)p.num_pages) bad = 1;
  __syncthreads();
  whole = whole || bad;
  if (head == 0 && threadIdx.x == 0) p.lens[request] = whole ? n : given;
  if (whole) {
    if (threadIdx.x == 0) *found = Found{};
    return;
  }
  const int recent = min(p.recent, given), need = given - recent, m = n - recent;

  // A wave's indices lie one behind the other, four to a lane.
  const int each = (m + kSelectWaves * 256 - 1) / (kSelectWaves * 256), begin = wave * each * 256;
  const bool held = each <= kQuads;  // all weights stay in registers
  uint32_t keys[kQuads][4];
  // the slot of index i (of four from a multiple of 4 on: the same page)
  auto slot_of = [&](int i) __attribute__((always_inline)) { return (table[i >> p.page_shift] << p.page_shift) + (i & mask); };
  auto load = [&](int i, uint32_t (&key)[4]) __attribute__((always_inline)) {
    const int at = begin + i * 256 + 4 * lane;
    f32x4 w = {0.f, 0.f, 0.f, 0.f};
    if (at < m)
      w = *reinterpret_cast<const f32x4*>(p.weights + (((int64_t)table[at >> p.page_shift] * p.kv_heads + head) << p.page_shift) +
                                          (at & mask));
#pragma unroll
    for (int j = 0; j < 4; ++j) key[j] = order_of(w[j]);
  };
  if (held) {
#pragma unroll
    for (int i = 0; i < kQuads; ++i)
      if (i < each) load(i, keys[i]);
  }
  // f(key, index) of every weight
  auto over = [&](auto f) __attribute__((always_inline)) {
    if (held) {
#pragma unroll
      for (int i = 0; i < kQuads; ++i)
        if (i < each)
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const int at = begin + i * 256 + 4 * lane + j;
            if (at < m) f(keys[i][j], at);
          }
    } else {
      for (int i = 0; i < each; ++i) {
        uint32_t key[4];
        load(i, key);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int at = begin + i * 256 + 4 * lane + j;
          if (at < m) f(key[j], at);
        }
      }
    }
  };

  uint32_t edge = ~0u;  // survivors: keys above it, and `ties` of those equal to it
  int ties = 0;
  if (need > 0) {
    uint32_t low = ~0u, high = 0;
    over([&](uint32_t key, int) { low = min(low, key), high = max(high, key); });
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) low = min(low, (uint32_t)__shfl_xor((int)low, d)), high = max(high, (uint32_t)__shfl_xor((int)high, d));
    if (lane == 0) atomicMin(&low_key, low), atomicMax(&high_key, high);
    __syncthreads();
    low = low_key, high = high_key;
    int wanted = need;
    for (;;) {  // the range shrinks by a factor of 2048 each time, or the loop ends
      const uint32_t range = high - low;
      if (!range) {
        edge = low, ties = wanted;
        break;
      }
      const int shift = max(0, 32 - (int)__builtin_clz(range) - 11);
      for (int i = threadIdx.x; i < kBins; i += kSelectThreads) bins[i] = 0;
      __syncthreads();
      over([&](uint32_t key, int) {
        if (key >= low && key <= high) atomicAdd(&bins[(key - low) >> shift], 1);
      });
      __syncthreads();
      // sums from the highest part down: thread t holds parts 2 t' and 2 t' + 1, t' = 1023 - t
      const int pair = kSelectThreads - 1 - (int)threadIdx.x, upper = bins[2 * pair + 1], lower = bins[2 * pair];
      int sum = lane_scan(upper + lower);
      if (lane == 63) waves[wave][0] = sum;
      __syncthreads();
      for (int w = 0; w < wave; ++w) sum += waves[w][0];
      const int above = sum - upper - lower;
      if (above < wanted && wanted <= sum) {
        const bool first = wanted <= above + upper;
        picked[0] = 2 * pair + first, picked[1] = wanted - above - (first ? 0 : upper);
      }
      __syncthreads();
      const int part = picked[0], count = bins[part];
      wanted = picked[1];
      low += (uint32_t)part << shift;
      high = low + min(high - low, (1u << shift) - 1);
      __syncthreads();
      if (!shift) {
        edge = low, ties = wanted;
        break;
      }
      if (count > kNear) continue;
      over([&](uint32_t key, int) {
        if (key >= low && key <= high) near[atomicAdd(&near_count, 1)] = key;
      });
      __syncthreads();
      if ((int)threadIdx.x < count) {
        const uint32_t mine = near[threadIdx.x];
        int larger = 0, equal = 0;
        for (int i = 0; i < count; ++i) larger += near[i] > mine, equal += near[i] == mine;
        if (larger < wanted && wanted <= larger + equal) edge_key = mine, edge_ties = wanted - larger;
      }
      __syncthreads();
      edge = edge_key, ties = edge_ties;
      break;
    }
  }

  // Places to fill and survivors behind them, in index order: a wave counts its own first. Of the equal keys
  // the first `ties` survive.
  int count[4] = {0, 0, 0, 0};  // evicted for certain below need, equal there, survivors behind, equal there
  over([&](uint32_t key, int at) {
    const bool front = at < need;
    count[0] += front && key < edge, count[1] += front && key == edge;
    count[2] += !front && key > edge, count[3] += !front && key == edge;
  });
#pragma unroll
  for (int c = 0; c < 4; ++c) count[c] = wave_sum(count[c]);
  __syncthreads();
  if (lane == 0)
#pragma unroll
    for (int c = 0; c < 4; ++c) waves[wave][c] = count[c];
  __syncthreads();
  // equal keys, places and survivors before this wave; survivors in all
  int seen = 0, to = 0, from = 0, all = 0, equals = 0, places_before = 0;
  for (int w = 0; w < kSelectWaves; ++w) {
    if (w == wave) seen = equals, to = places_before, from = all;
    const int front = waves[w][1], back = waves[w][3];  // (its front part comes before its back part)
    const int kept_front = min(front, max(0, ties - equals)), kept_back = min(back, max(0, ties - equals - front));
    places_before += waves[w][0] + front - kept_front, all += waves[w][2] + kept_back, equals += front + back;
  }

  int32_t* const fill = p.lists + ((int64_t)request * p.kv_heads + head) * 2 * p.moves;
  int32_t* const take = fill + p.moves;
  int mine_early = 0;
  auto emit = [&](const uint32_t (&key)[4], int at) __attribute__((always_inline)) {
    // equal keys of the lanes before
    int equal = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) equal += at + j < m && key[j] == edge;
    const int equal_upto = lane_scan(equal);
    int rank = seen + equal_upto - equal, places = 0, sources = 0;
    bool place[4], source[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const bool inside = at + j < m, tie = inside && key[j] == edge;
      const bool stays = inside && (key[j] > edge || (tie && rank < ties));
      rank += tie;
      place[j] = inside && at + j < need && !stays, source[j] = stays && at + j >= need;
      places += place[j], sources += source[j];
    }
    const int places_upto = lane_scan(places), sources_upto = lane_scan(sources);
    int next_place = to + places_upto - places, next_source = from + sources_upto - sources;
    if (places || sources) {
      const int slot = (table[at >> p.page_shift] << p.page_shift) + (at & mask);  // four of one page
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        if (place[j]) fill[next_place++] = slot + j;
        if (source[j]) take[next_source++] = slot + j, mine_early += at + j < given;
      }
    }
    seen += __shfl(equal_upto, 63), to += __shfl(places_upto, 63), from += __shfl(sources_upto, 63);
  };
  if (held) {
#pragma unroll
    for (int i = 0; i < kQuads; ++i)
      if (i < each) emit(keys[i], begin + i * 256 + 4 * lane);
  } else {
    for (int i = 0; i < each; ++i) {
      uint32_t key[4];
      load(i, key);
      emit(key, begin + i * 256 + 4 * lane);
    }
  }
  mine_early = wave_sum(mine_early);
  if (lane == 0) atomicAdd(&early, mine_early);
  __syncthreads();
  if (threadIdx.x == 0) *found = Found{all, early, recent, m, need, {0, 0, 0}};
}

constexpr int kMoveThreads = 256, kAhead = 4;

__device__ __forceinline__ uint16_t* row_at(const EvictArgs& p, uint16_t* cache, int slot, int head) {
  return cache + (int64_t)(slot >> p.page_shift) * p.page_stride + (int64_t)(slot & ((1 << p.page_shift) - 1)) * p.slot_stride +
         (int64_t)head * p.head_stride;
}

__device__ __forceinline__ float* weight_at(const EvictArgs& p, int slot, int head) {
  return p.weights + ((((int64_t)(slot >> p.page_shift) * p.kv_heads + head) << p.page_shift) + (slot & ((1 << p.page_shift) - 1)));
}

// The rows on a head's lists, and its recent ones. The first p.tails workgroups of a head and request take the recent rows, each
// a share of a row's columns: first the survivors out of the places where those go, then the recent ones from the
// front on, all of a block read before any of it is written, since their old and new places may overlap. The other
// workgroups share the rest of the lists. No other two rows meet: bound by memory.
template <int D>
__global__ __launch_bounds__(kMoveThreads) void evict_move(EvictArgs p) {
  constexpr int kChunks = D / 8;  // of 16 bytes in a row of keys, and as many of values
  const int pair = blockIdx.x, head = pair % p.kv_heads, request = pair / p.kv_heads;
  const Found f = p.found[pair];
  const int32_t* const fill = p.lists + (int64_t)pair * 2 * p.moves;
  const int32_t* const take = fill + p.moves;
  const bool tail = (int)blockIdx.y < p.tails;
  const int share = tail ? 2 * kChunks / p.tails : 2 * kChunks, rows = kMoveThreads / share;
  const int chunk = (tail ? blockIdx.y * share : 0) + threadIdx.x % share, row = threadIdx.x / share;
  uint16_t* const cache = (chunk < kChunks ? p.k : p.v) + chunk % kChunks * 8;

  auto listed = [&](int first, int last, int step) __attribute__((always_inline)) {
    for (int j = first; j < last; j += step) {
      u32x4 value[kAhead];
#pragma unroll
      for (int u = 0; u < kAhead; ++u)
        if (j + u * rows < last) value[u] = *reinterpret_cast<const u32x4*>(row_at(p, cache, take[j + u * rows], head));
#pragma unroll
      for (int u = 0; u < kAhead; ++u)
        if (j + u * rows < last) *reinterpret_cast<u32x4*>(row_at(p, cache, fill[j + u * rows], head)) = value[u];
    }
  };
  if (!tail) {
    const int block = blockIdx.y - p.tails;
    listed(f.early + block * rows * kAhead + row, f.count, p.movers * rows * kAhead);
    for (int j = f.early + block * kMoveThreads + (int)threadIdx.x; j < f.count; j += p.movers * kMoveThreads)
      *weight_at(p, fill[j], head) = *weight_at(p, take[j], head);
    return;
  }
  if (!f.recent) return;  // (then no survivor lies among their places)
  listed(row, f.early, rows * kAhead);
  if (blockIdx.y == 0)
    for (int j = threadIdx.x; j < f.early; j += kMoveThreads) *weight_at(p, fill[j], head) = *weight_at(p, take[j], head);
  const int32_t* const table = p.tables + (int64_t)request * p.table_stride;
  auto slot_of = [&](int i) { return (table[i >> p.page_shift] << p.page_shift) + (i & ((1 << p.page_shift) - 1)); };
  for (int i = 0; i < f.recent; i += rows * kAhead) {
    u32x4 value[kAhead];
    float weight = 0.f;
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      const int at = i + u * rows + row;
      if (at < f.recent) value[u] = *reinterpret_cast<const u32x4*>(row_at(p, cache, slot_of(f.from + at), head));
    }
    const int at_weight = i + (int)threadIdx.x;
    const bool weighs = blockIdx.y == 0 && (int)threadIdx.x < rows * kAhead && at_weight < f.recent;
    if (weighs) weight = *weight_at(p, slot_of(f.from + at_weight), head);
    // every wave's loads (and, the first time, those of the survivors) are done
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      const int at = i + u * rows + row;
      if (at < f.recent) *reinterpret_cast<u32x4*>(row_at(p, cache, slot_of(f.to + at), head)) = value[u];
    }
    if (weighs) *weight_at(p, slot_of(f.to + at_weight), head) = weight;
  }
}

// Rows of a head that can move: as many as are evicted, and no more than are kept.
int moves_of(int keep, bool given, int max_context) {
  return max(1, given ? max_context / 2 : min(keep, max(0, max_context - keep)));
}

}  // namespace
}  // namespace smx

using namespace smx;

extern "C" {

int smx_paged_evict_workspace_bytes(int32_t requests, int32_t kv_heads, int32_t keep, int32_t max_context, int64_t* bytes) {
  smx::fail(SMX_OK, "%s", "");
  if (!bytes) return fail(SMX_ERR_INVALID, "null pointer");
  if (requests <= 0 || requests > SMX_PAGED_MAX_REQUESTS || kv_heads <= 0 || kv_heads > 65535)
    return fail(SMX_ERR_INVALID, "1 to %d requests and 1 to 65535 heads (requests=%d, kv_heads=%d)",
                SMX_PAGED_MAX_REQUESTS, requests, kv_heads);
  if (max_context < 0 || max_context > SMX_PAGED_MAX_CONTEXT)
    return fail(SMX_ERR_INVALID, "max_context must be 0 to %d, got %d", SMX_PAGED_MAX_CONTEXT, max_context);
  // keep < 0: a length for each request
  *bytes = (int64_t)requests * kv_heads * (sizeof(Found) + 8 * (int64_t)moves_of(keep, keep < 0, max_context));
  return SMX_OK;
}

int smx_paged_evict(const smx_paged_cache* cache, float* key_weights, int32_t requests, int32_t width, const int32_t* context_lens,
                    const int32_t* block_tables, int64_t table_stride, const int32_t* keep_lens, int32_t keep, int32_t recent,
                    int32_t max_context, int32_t* lens, void* workspace, int64_t workspace_bytes, void* stream) {
  int64_t need = 0;
  if (int rc = paged_layout(cache)) return rc;
  if (keep_lens) keep = -1;
  else if (keep < 0) return fail(SMX_ERR_INVALID, "keep must not be negative, got %d", keep);
  if (int rc = smx_paged_evict_workspace_bytes(requests, cache->kv_heads, keep, max_context, &need)) return rc;
  if (!key_weights || !context_lens || !block_tables || !lens) return fail(SMX_ERR_INVALID, "null pointer");
  if ((uintptr_t)key_weights % 16) return fail(SMX_ERR_INVALID, "key_weights must be 16-byte aligned");
  if (recent < 0) return fail(SMX_ERR_INVALID, "recent must not be negative, got %d", recent);
  if (width <= 0 || table_stride < width) return fail(SMX_ERR_INVALID, "table_stride must be at least the table's width");
  if ((int64_t)max_context > (int64_t)width * cache->page_size)
    return fail(SMX_ERR_INVALID, "max_context=%d: the block tables hold %lld tokens a request", max_context,
                (long long)width * cache->page_size);
  if (!workspace || (uintptr_t)workspace % 16 || workspace_bytes < need)
    return fail(SMX_ERR_INVALID, "the call needs a 16-byte aligned workspace of %lld bytes", (long long)need);
  const Runs keys = cache_runs(*cache, cache->k), values = cache_runs(*cache, cache->v);
  if (!lie_apart(keys)) return fail(SMX_ERR_INVALID, "the cache holds rows that lie on each other");
  if (meet(keys, values)) return fail(SMX_ERR_INVALID, "keys and values must share no memory of the cache");
  const Runs all{key_weights, 2 * (int64_t)cache->num_pages * cache->kv_heads * cache->page_size, {{1, 0}, {1, 0}, {1, 0}}};
  if (meet(all, keys) || meet(all, values)) return fail(SMX_ERR_INVALID, "key_weights must share no memory with the cache");
  EvictArgs p{};
  p.k = (uint16_t*)cache->k, p.v = (uint16_t*)cache->v;
  p.page_stride = cache->page_stride, p.slot_stride = cache->slot_stride, p.head_stride = cache->head_stride;
  p.weights = key_weights, p.context = context_lens, p.tables = block_tables, p.keep_lens = keep_lens;
  p.table_stride = table_stride, p.lens = lens, p.requests = requests, p.kv_heads = cache->kv_heads;
  p.head_dim = cache->head_dim, p.page_shift = __builtin_ctz(cache->page_size), p.num_pages = cache->num_pages;
  p.keep = keep, p.recent = recent, p.max_context = max_context, p.moves = moves_of(keep, keep < 0, max_context);
  const int pairs = requests * cache->kv_heads;
  p.found = (Found*)workspace;
  p.lists = (int32_t*)(p.found + pairs);
  hipLaunchKernelGGL(evict_select, dim3((unsigned)cache->kv_heads, (unsigned)requests), dim3(kSelectThreads), 0,
                     (hipStream_t)stream, p);
  if (int rc = check_launch()) return rc;
  // Workgroups of a head and request: enough to fill the chip, of 64 rows at least.
  p.tails = cache->head_dim / 32;
  p.movers = min((p.moves + 63) / 64, max(1, 8192 / pairs));
  hipLaunchKernelGGL(cache->head_dim == 128 ? evict_move<128> : evict_move<64>, dim3((unsigned)pairs, (unsigned)(p.tails + p.movers)),
                     dim3(kMoveThreads), 0, (hipStream_t)stream, p);
  return check_launch();
}

}  // extern "C"
