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
// a histogram of their leading 11 bits, the part that holds it, and so on until its keys fit in LDS,
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

constexpr int kBins = 2048, kNear = 256, kQuads = 8;

// Weights in the order of their values; NaN above everything, -0 as 0.
__device__ __forceinline__ uint32_t order_of(float x) {
  const uint32_t bits = __float_as_uint(x + 0.f);
  if (x != x) return ~0u;
  return bits & 0x80000000u ? ~bits : bits | 0x80000000u;
}

// x of the lanes that kControl names, in the rows of 16 lanes that kRows names; zero where there are none.
template <int kControl, int kRows>
__device__ __forceinline__ int moved(int x) {
  return __builtin_amdgcn_update_dpp(0, x, kControl, kRows, 15, false);
}

// Inclusive sum over a wave's lanes: within rows of 16 lanes, then a row's last value to the next row, and the
// lower half's to the upper.
__device__ __forceinline__ int lane_scan(int x) {
  x += moved<0x111, 15>(x);
  x += moved<0x112, 15>(x);
  x += moved<0x114, 15>(x);
  x += moved<0x118, 15>(x);
  x += moved<0x142, 10>(x);
  x += moved<0x143, 12>(x);
  return x;
}

// kThreads * 4 * kQuads weights are held in registers, more are read once for each look at them.
template <int kThreads>
__global__ __launch_bounds__(kThreads) void evict_select(EvictArgs p) {
  constexpr int kWaves = kThreads / 64;
  const int head = blockIdx.x, request = blockIdx.y, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  Found* const found = p.found + (int64_t)request * p.kv_heads + head;
  __shared__ int bins[kBins], scans[kWaves], counts[kWaves][4], bad, near_count, early, picked[3];
  __shared__ __attribute__((aligned(16))) uint32_t near[kNear];
  __shared__ uint32_t edge_key, lows[kWaves], highs[kWaves];
  __shared__ int edge_ties, near_at[kNear];
  const int32_t n = p.context[request], given = p.keep_lens ? p.keep_lens[request] : p.keep;
  const int32_t* const table = p.tables + request * p.table_stride;
  const int32_t mask = (1 << p.page_shift) - 1;
  if (n <= given || n > p.max_context || given < 0) {  // uniform
    if (threadIdx.x == 0) {
      *found = Found{};
      if (head == 0) p.lens[request] = n;
    }
    return;
  }
  if (threadIdx.x == 0) bad = near_count = early = 0;
  for (int i = threadIdx.x; i < kBins; i += kThreads) bins[i] = 0;
  if (threadIdx.x < kNear) near[threadIdx.x] = 0;  // below every key
  const int recent = min(p.recent, given), need = given - recent, m = n - recent;

  // A wave's indices lie one behind the other, four to a lane, in batches of kQuads times 256.
  const int each = (m + kWaves * 256 - 1) / (kWaves * 256), begin = wave * each * 256;
  const bool held = each <= kQuads;
  uint32_t keys[kQuads][4];
  bool missing = false;
  auto load = [&](int first) __attribute__((always_inline)) {
    f32x4 w[kQuads];
    int entry[kQuads];
#pragma unroll
    for (int i = 0; i < kQuads; ++i) {
      const int at = begin + (first + i) * 256 + 4 * lane;
      entry[i] = first + i < each && at < m ? table[at >> p.page_shift] : 0;
      missing |= (uint32_t)entry[i] >= (uint32_t)p.num_pages;
      if ((uint32_t)entry[i] >= (uint32_t)p.num_pages) entry[i] = 0;
    }
#pragma unroll
    for (int i = 0; i < kQuads; ++i) {
      const int at = begin + (first + i) * 256 + 4 * lane;
      if (first + i < each && at < m)
        w[i] = *reinterpret_cast<const f32x4*>(p.weights + (((int64_t)entry[i] * p.kv_heads + head) << p.page_shift) + (at & mask));
    }
#pragma unroll
    for (int i = 0; i < kQuads; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) keys[i][j] = order_of(w[i][j]);
  };
  // f(four keys, index of the first) over the wave's indices, in their order; f is called by all lanes
  auto over = [&](auto f) __attribute__((always_inline)) {
    for (int first = 0; first < each; first += kQuads) {
      if (!held) load(first);
#pragma unroll
      for (int i = 0; i < kQuads; ++i)
        if (first + i < each) f(keys[i], begin + (first + i) * 256 + 4 * lane);
    }
  };

  // The range of the weights (of the first batch, where they are more): parts of equal size of the values that
  // are there hold few weights each, and the histogram's additions meet rarely.
  load(0);
  uint32_t low = ~0u, high = 0;
#pragma unroll
  for (int i = 0; i < kQuads; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (i < each && begin + i * 256 + 4 * lane + j < m) low = min(low, keys[i][j]), high = max(high, keys[i][j]);
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) low = min(low, (uint32_t)__shfl_xor((int)low, d)), high = max(high, (uint32_t)__shfl_xor((int)high, d));
  if (lane == 0) lows[wave] = low, highs[wave] = high;
  // every page of the request has to be there, the recent tokens' too
  for (int i = (m >> p.page_shift) + (int)threadIdx.x; i <= (n - 1) >> p.page_shift; i += kThreads)
    missing |= (uint32_t)table[i] >= (uint32_t)p.num_pages;
  __syncthreads();
  for (int w = 0; w < kWaves; ++w) low = min(low, lows[w]), high = max(high, highs[w]);

  // The need-th largest lies between `least` and `most`, the `ties`-th largest of the keys there. (Without need nothing
  // survives: none of the largest keys.)
  uint32_t least = ~0u, most = ~0u;
  int ties = 0;
  if (need > 0) {
    // Keys below `low` count to the first part of the histogram, those above `high` to the last.
    int wanted = need;
    least = 0;
    for (;;) {
      const int shift = max(0, 32 - (high > low ? (int)__builtin_clz(high - low) : 32) - 11);
      over([&](const uint32_t (&key)[4], int at) __attribute__((always_inline)) {
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (at + j < m && key[j] >= least && key[j] <= most)
            atomicAdd(&bins[key[j] <= low ? 0 : min((key[j] - low) >> shift, (uint32_t)kBins - 1)], 1);
      });
      __syncthreads();
      // The part that holds it: sums from the highest one down, kEach parts a thread.
      constexpr int kEach = kBins / kThreads;
      const int top = kBins - 1 - (int)threadIdx.x * kEach;
      int own[kEach], sum = 0;
#pragma unroll
      for (int i = 0; i < kEach; ++i) own[i] = bins[top - i], sum += own[i];
      const int all = sum;
      sum = lane_scan(sum);
      if (lane == 63) scans[wave] = sum;
      __syncthreads();
      for (int w = 0; w < wave; ++w) sum += scans[w];
      int above = sum - all;
#pragma unroll
      for (int i = 0; i < kEach; ++i) {
        if (above < wanted && wanted <= above + own[i]) picked[0] = top - i, picked[1] = wanted - above, picked[2] = own[i];
        above += own[i];
        bins[top - i] = 0;
      }
      __syncthreads();
      const int part = picked[0], count = picked[2];
      wanted = picked[1];
      const uint64_t first = low + ((uint64_t)part << shift);
      if (part) least = (uint32_t)first;
      if (part < kBins - 1) most = (uint32_t)min((uint64_t)most, first + ((uint64_t)1 << shift) - 1);
      low = least, high = most;
      if (least == most || count <= kNear) break;  // else another look, at this part alone
    }
    ties = wanted;
  }
  if (missing) bad = 1;

  // Places to fill and survivors behind them, in index order: a wave counts its own first. Keys of the part found are
  // compared with each other, unless they are equal.
  const bool apart = least < most;
  int count[4] = {0, 0, 0, 0};  // below need: of keys below the part, in it; behind: above it, in it
  over([&](const uint32_t (&key)[4], int at) __attribute__((always_inline)) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const bool inside = at + j < m, front = at + j < need, in = inside && key[j] >= least && key[j] <= most;
      count[0] += inside && front && key[j] < least, count[1] += in && front;
      count[2] += inside && !front && key[j] > most, count[3] += in && !front;
      if (in && apart) {
        const int place = atomicAdd(&near_count, 1);
        if (place < kNear) near[place] = key[j], near_at[place] = at + j;  // (always, while nobody changes the weights)
      }
    }
  });
#pragma unroll
  for (int c = 0; c < 4; ++c) {
    const int sum = lane_scan(count[c]);
    if (lane == 63) counts[wave][c] = apart && (c & 1) ? 0 : sum;
  }
  __syncthreads();
  if (head == 0 && threadIdx.x == 0) p.lens[request] = bad ? n : given;
  if (bad) {  // uniform
    if (threadIdx.x == 0) *found = Found{};
    return;
  }
  // Survivors: keys above the edge, and the first `ties` of those equal to it.
  uint32_t edge = most;
  if (apart) {
    const int near_all = min(near_count, kNear);
    const uint32_t mine = (int)threadIdx.x < near_all ? near[threadIdx.x] : 0;
    if (mine) {
      int larger = 0, equal = 0;
      for (int x = 0; x < near_all; x += 4) {
        const u32x4 other = *reinterpret_cast<const u32x4*>(near + x);
#pragma unroll
        for (int j = 0; j < 4; ++j) larger += other[j] > mine, equal += other[j] == mine;
      }
      if (larger < ties && ties <= larger + equal) edge_key = mine, edge_ties = ties - larger;
    }
    __syncthreads();
    edge = edge_key, ties = edge_ties;
    if (mine) {
      const int at = near_at[threadIdx.x], of = at / (each * 256);
      if (mine == edge) atomicAdd(&counts[of][at < need ? 1 : 3], 1);
      else if (mine < edge && at < need) atomicAdd(&counts[of][0], 1);
      else if (mine > edge && at >= need) atomicAdd(&counts[of][2], 1);
    }
    __syncthreads();
  }
  // equal keys, places and survivors before this wave; survivors in all
  int seen = 0, to = 0, from = 0, all = 0, equals = 0, places_before = 0;
  for (int w = 0; w < kWaves; ++w) {
    if (w == wave) seen = equals, to = places_before, from = all;
    const int front = counts[w][1], back = counts[w][3];  // (its front part comes before its back part)
    const int kept_front = min(front, max(0, ties - equals)), kept_back = min(back, max(0, ties - equals - front));
    places_before += counts[w][0] + front - kept_front, all += counts[w][2] + kept_back, equals += front + back;
  }

  int32_t* const fill = p.lists + ((int64_t)request * p.kv_heads + head) * 2 * p.moves;
  int32_t* const take = fill + p.moves;
  int mine_early = 0;
  over([&](const uint32_t (&key)[4], int at) __attribute__((always_inline)) {
    // equal keys of the lanes before
    int equal = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) equal += at + j < m && key[j] == edge;
    int equal_upto = 0;
    if (__any(equal)) equal_upto = lane_scan(equal);  // (few batches hold any)
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
    // both sums in one: 256 at most
    const int both = lane_scan(places | sources << 16), places_upto = both & 0xffff, sources_upto = both >> 16;
    int next_place = to + places_upto - places, next_source = from + sources_upto - sources;
    if (places || sources) {
      const int slot = (table[at >> p.page_shift] << p.page_shift) + (at & mask);  // four of one page
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        if (place[j] && next_place < p.moves) fill[next_place++] = slot + j;
        if (source[j] && next_source < p.moves) take[next_source++] = slot + j, mine_early += at + j < given;
      }
    }
    seen += __shfl(equal_upto, 63), to += __shfl(places_upto, 63), from += __shfl(sources_upto, 63);
  });
  mine_early = lane_scan(mine_early);
  if (lane == 63) atomicAdd(&early, mine_early);
  __syncthreads();
  if (threadIdx.x == 0) *found = Found{min(all, p.moves), early, recent, m, need, {0, 0, 0}};
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
  // Four waves where they hold the longest context, else sixteen.
  const bool few = max_context <= 256 * 4 * kQuads;
  hipLaunchKernelGGL(few ? evict_select<256> : evict_select<1024>, dim3((unsigned)cache->kv_heads, (unsigned)requests),
                     dim3(few ? 256 : 1024), 0, (hipStream_t)stream, p);
  if (int rc = check_launch()) return rc;
  // Workgroups of a head and request: enough to fill the chip, of 64 rows at least.
  p.tails = cache->head_dim / 32;
  p.movers = min((p.moves + 63) / 64, max(1, 8192 / pairs));
  hipLaunchKernelGGL(cache->head_dim == 128 ? evict_move<128> : evict_move<64>, dim3((unsigned)pairs, (unsigned)(p.tails + p.movers)),
                     dim3(kMoveThreads), 0, (hipStream_t)stream, p);
  return check_launch();
}

}  // extern "C"
