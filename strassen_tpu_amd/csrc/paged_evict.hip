// Eviction from a paged cache by the attention weight that keys have received (smx_paged_evict).
//
// Of the n tokens of a request, each key/value head keeps `keep`: the last `recent`, and of the m older ones the
// need = keep - recent with the largest weights (ties: the lowest index). Survivors with an index below need stay
// where they are. The places of the evicted ones there are as many as the survivors behind, and the j-th of
// the one takes the j-th of the other: of those kept for their weight no fewer can move if there are to be no gaps. The recent ones
// all move, to need .. keep - 1, since they stay in their order. No row is moved twice: of 131,000 tokens cut to 32,768, 512
// of them the last, a head moves 24,800.
//
// evict_select (a workgroup per head and request) finds the need-th largest weight: weights as integers in their order,
// a histogram of equal parts of their range, the part that holds it, and so on until its keys fit in LDS,
// where they are compared with each other. Where contexts are long and heads few, the same is done in parts by several workgroups a
// head (evict_histogram, evict_collect, evict_list). evict_move then moves the rows.
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
  // of long contexts, in `parts` parts of a head and request
  int32_t parts;
  struct Looked* looked;          // [requests * kv_heads]
  struct Candidate* candidates;   // [requests * kv_heads][kCrowd]
  int32_t *bad, *counts;          // [requests * kv_heads][parts], [..][parts][waves][4]
  uint16_t* histograms;           // [requests * kv_heads][parts][kBins]
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

// What a request is cut to.
struct Cut {
  int32_t n, given, recent, need, m;  // its tokens, those kept, the recent among them, the others; the older tokens

  // Whether anything is to be cut.
  __device__ __forceinline__ bool of(const EvictArgs& p, int request) {
    n = p.context[request], given = p.keep_lens ? p.keep_lens[request] : p.keep;
    recent = min(p.recent, given), need = given - recent, m = n - recent;
    return n > given && n <= p.max_context && given >= 0;
  }
};

typedef uint32_t Keys[kQuads][4];

// The keys of indices begin + 256 i + 4 lane .. + 3, i < count, below m. Entries that are no page of the cache are told in
// `missing` and read as page 0.
__device__ __forceinline__ void load_keys(const EvictArgs& p, const int32_t* table, int head, int begin, int count, int m, Keys& keys,
                                          bool& missing) {
  const int lane = threadIdx.x & 63, mask = (1 << p.page_shift) - 1;
  f32x4 w[kQuads];
  int entry[kQuads];
#pragma unroll
  for (int i = 0; i < kQuads; ++i) {
    const int at = begin + i * 256 + 4 * lane;
    entry[i] = i < count && at < m ? table[at >> p.page_shift] : 0;
    missing |= (uint32_t)entry[i] >= (uint32_t)p.num_pages;
    if ((uint32_t)entry[i] >= (uint32_t)p.num_pages) entry[i] = 0;
  }
#pragma unroll
  for (int i = 0; i < kQuads; ++i) {
    const int at = begin + i * 256 + 4 * lane;
    if (i < count && at < m)
      w[i] = *reinterpret_cast<const f32x4*>(p.weights + (((int64_t)entry[i] * p.kv_heads + head) << p.page_shift) + (at & mask));
  }
#pragma unroll
  for (int i = 0; i < kQuads; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) keys[i][j] = order_of(w[i][j]);
}

// The range of the workgroup's keys (two barriers apart from each other's use of `ends`: one within).
template <int kWaves>
__device__ __forceinline__ void range_of(uint32_t& low, uint32_t& high, uint32_t (&ends)[2][kWaves]) {
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) low = min(low, (uint32_t)__shfl_xor((int)low, d)), high = max(high, (uint32_t)__shfl_xor((int)high, d));
  if ((threadIdx.x & 63) == 0) ends[0][threadIdx.x >> 6] = low, ends[1][threadIdx.x >> 6] = high;
  __syncthreads();
  for (int w = 0; w < kWaves; ++w) low = min(low, ends[0][w]), high = max(high, ends[1][w]);
}

// A histogram over the keys from low to high: those below low, low itself (weights of which many are zero end here),
// and equal parts of the others, the last with those above high. Parts of the values that are there hold few keys each, so that
// additions meet rarely (leading bits alone, of which most weights share some: 66 us for 8100 keys
// of 512 heads, and 23 of equal parts in the same state of the rest; 21 now).
struct Look {
  int bins[kBins], scans[16], picked[3];

  __device__ __forceinline__ void clear() {
    for (int i = threadIdx.x; i < kBins; i += blockDim.x) bins[i] = 0;
    if (threadIdx.x < 3) picked[threadIdx.x] = 0;
  }
};

__device__ __forceinline__ int shift_of(uint32_t low, uint32_t high) {
  const uint32_t range = high > low ? high - low : 0;
  const int shift = max(0, 32 - (range ? (int)__builtin_clz(range) : 32) - 11);
  return shift + (range >> shift > kBins - 2);
}

__device__ __forceinline__ int part_of(uint32_t key, uint32_t low, int shift) {
  return key <= low ? key == low : (int)min(((key - low - 1) >> shift) + 2, (uint32_t)kBins - 1);
}

// The wanted-th largest key of those from least to most, of a filled histogram: its part's ends (also as the next
// histogram's), the rank within the part, and how many keys are there. The histogram is cleared.
template <int kThreads>
__device__ __forceinline__ int pick(Look& look, uint32_t& low, uint32_t& high, uint32_t& least, uint32_t& most, int& wanted) {
  constexpr int kEach = kBins / kThreads;
  const int shift = shift_of(low, high), lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  // sums from the highest part down, kEach parts a thread
  const int top = kBins - 1 - (int)threadIdx.x * kEach;
  __syncthreads();
  int own[kEach], sum = 0;
#pragma unroll
  for (int i = 0; i < kEach; ++i) own[i] = look.bins[top - i], sum += own[i];
  const int all = sum;
  sum = lane_scan(sum);
  if (lane == 63) look.scans[wave] = sum;
  __syncthreads();
  for (int w = 0; w < wave; ++w) sum += look.scans[w];
  int above = sum - all;
#pragma unroll
  for (int i = 0; i < kEach; ++i) {
    if (above < wanted && wanted <= above + own[i]) look.picked[0] = top - i, look.picked[1] = wanted - above, look.picked[2] = own[i];
    above += own[i];
    look.bins[top - i] = 0;
  }
  __syncthreads();
  const int part = look.picked[0], count = look.picked[2];
  wanted = look.picked[1];
  if (part == 0) most = low ? low - 1 : 0;
  else if (part == 1) least = most = low;
  else {
    const uint64_t first = (uint64_t)low + 1 + ((uint64_t)(part - 2) << shift);
    least = (uint32_t)first;
    if (part < kBins - 1) most = (uint32_t)min((uint64_t)most, first + ((uint64_t)1 << shift) - 1);
  }
  low = least, high = most;
  return count;
}

// Few keys, compared with each other.
struct Near {
  __attribute__((aligned(16))) uint32_t key[kNear];
  uint32_t edge;
  int at[kNear], count, ties;

  __device__ __forceinline__ void clear() {
    if (threadIdx.x < kNear) key[threadIdx.x] = 0;  // below every key
    if (threadIdx.x == 0) count = 0;
  }
  __device__ __forceinline__ void add(uint32_t k, int index) {
    const int place = atomicAdd(&count, 1);
    if (place < kNear) key[place] = k, at[place] = index;  // (always, while nobody changes the weights)
  }
  // The wanted-th largest, and its rank among those equal to it.
  __device__ __forceinline__ uint32_t resolve(int* wanted) {
    const int all = min(count, kNear);
    const uint32_t mine = (int)threadIdx.x < all ? key[threadIdx.x] : 0;
    if (mine) {
      int larger = 0, equal = 0;
#pragma unroll 4
      for (int x = 0; x < all; x += 4) {
        const u32x4 other = *reinterpret_cast<const u32x4*>(key + x);
#pragma unroll
        for (int j = 0; j < 4; ++j) larger += other[j] > mine, equal += other[j] == mine;
      }
      if (larger < *wanted && *wanted <= larger + equal) edge = mine, ties = *wanted - larger;
    }
    __syncthreads();
    *wanted = ties;
    return edge;
  }
};

// Puts the places to fill and the survivors behind them on the lists, four indices a lane. seen, to and from: equal keys,
// places and survivors before these (uniform). Returns how many of the lane's survivors lie before `given`.
__device__ __forceinline__ int list_four(const EvictArgs& p, const int32_t* table, const Cut& c, uint32_t edge, int ties, int32_t* fill,
                                         int32_t* take, const uint32_t (&key)[4], int at, int& seen, int& to, int& from) {
  // equal keys of the lanes before
  int equal = 0;
#pragma unroll
  for (int j = 0; j < 4; ++j) equal += at + j < c.m && key[j] == edge;
  int equal_upto = 0;
  if (__any(equal)) equal_upto = lane_scan(equal);  // (few hold any)
  int rank = seen + equal_upto - equal, places = 0, sources = 0, early = 0;
  bool place[4], source[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const bool inside = at + j < c.m, tie = inside && key[j] == edge;
    const bool stays = inside && (key[j] > edge || (tie && rank < ties));
    rank += tie;
    place[j] = inside && at + j < c.need && !stays, source[j] = stays && at + j >= c.need;
    places += place[j], sources += source[j];
  }
  // both sums in one: 256 at most
  const int both = lane_scan(places | sources << 16);
  int next_place = to + (both & 0xffff) - places, next_source = from + (both >> 16) - sources;
  if (places || sources) {
    const int slot = (table[at >> p.page_shift] << p.page_shift) + (at & ((1 << p.page_shift) - 1));  // four of one page
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if (place[j] && next_place < p.moves) fill[next_place++] = slot + j;
      if (source[j] && next_source < p.moves) take[next_source++] = slot + j, early += at + j < c.given;
    }
  }
  seen += __builtin_amdgcn_readlane(equal_upto, 63);
  const int sums = __builtin_amdgcn_readlane(both, 63);
  to += sums & 0xffff, from += sums >> 16;
  return early;
}

__device__ __forceinline__ int32_t* lists_of(const EvictArgs& p, int64_t pair) { return p.lists + pair * 2 * p.moves; }

// The whole of one head and request by one workgroup. kThreads * 4 * kQuads weights are held in registers, more are read
// once for each look at them.
template <int kThreads>
__device__ void select_whole(const EvictArgs& p, const Cut& c, int head, int request, Look& look, Near& near) {
  constexpr int kWaves = kThreads / 64;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t pair = (int64_t)request * p.kv_heads + head;
  __shared__ int counts[kWaves][4], bad, early;
  __shared__ uint32_t ends[2][kWaves];
  const int32_t* const table = p.tables + request * p.table_stride;
  if (threadIdx.x == 0) bad = early = 0;
  near.clear();
  look.clear();

  // A wave's indices lie one behind the other, four to a lane, in batches of kQuads times 256.
  const int each = (c.m + kWaves * 256 - 1) / (kWaves * 256), begin = wave * each * 256;
  const bool held = each <= kQuads;
  Keys keys;
  bool missing = false;
  // f(four keys, index of the first) over the wave's indices, in their order; f is called by all lanes
  auto over = [&](auto f) __attribute__((always_inline)) {
    for (int first = 0; first < each; first += kQuads) {
      if (!held) load_keys(p, table, head, begin + first * 256, each - first, c.m, keys, missing);
#pragma unroll
      for (int i = 0; i < kQuads; ++i)
        if (first + i < each) f(keys[i], begin + (first + i) * 256 + 4 * lane);
    }
  };
  // the range of the weights (of the first batch, where they are more)
  load_keys(p, table, head, begin, each, c.m, keys, missing);
  uint32_t low = ~0u, high = 0;
#pragma unroll
  for (int i = 0; i < kQuads; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (i < each && begin + i * 256 + 4 * lane + j < c.m) low = min(low, keys[i][j]), high = max(high, keys[i][j]);
  // every page of the request has to be there, the recent tokens' too
  for (int i = (c.m >> p.page_shift) + (int)threadIdx.x; i <= (c.n - 1) >> p.page_shift; i += kThreads)
    missing |= (uint32_t)table[i] >= (uint32_t)p.num_pages;
  range_of<kWaves>(low, high, ends);

  // The need-th largest lies between `least` and `most`, the `ties`-th largest of the keys there. (Without need nothing
  // survives: none of the largest keys.)
  uint32_t least = ~0u, most = ~0u;
  int ties = 0;
  if (c.need > 0) {
    ties = c.need, least = 0;
    int count;
    do {
      const int shift = shift_of(low, high);
      over([&](const uint32_t (&key)[4], int at) __attribute__((always_inline)) {
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (at + j < c.m && key[j] >= least && key[j] <= most) atomicAdd(&look.bins[part_of(key[j], low, shift)], 1);
      });
      count = pick<kThreads>(look, low, high, least, most, ties);
    } while (least < most && count > kNear);  // another look, at the part alone
  }

  // Places to fill and survivors behind them, in index order: a wave counts its own first. Keys of the part found are
  // compared with each other, unless they are equal.
  const bool apart = least < most;
  int count[4] = {0, 0, 0, 0};  // below need: of keys below the part, in it; behind: above it, in it
  over([&](const uint32_t (&key)[4], int at) __attribute__((always_inline)) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const bool inside = at + j < c.m, front = at + j < c.need, in = inside && key[j] >= least && key[j] <= most;
      count[0] += inside && front && key[j] < least, count[1] += in && front;
      count[2] += inside && !front && key[j] > most, count[3] += in && !front;
      if (in && apart) near.add(key[j], at + j);
    }
  });
  // (now at the latest every page has been looked at: without need there was no look, and keys that are not held were read in
  // this pass for the first time)
  if (missing) bad = 1;
#pragma unroll
  for (int x = 0; x < 4; ++x) {
    const int sum = lane_scan(count[x]);
    if (lane == 63) counts[wave][x] = apart && (x & 1) ? 0 : sum;
  }
  __syncthreads();
  if (head == 0 && threadIdx.x == 0) p.lens[request] = bad ? c.n : c.given;
  if (bad) {  // uniform
    if (threadIdx.x == 0) p.found[pair] = Found{};
    return;
  }
  // Survivors: keys above the edge, and the first `ties` of those equal to it.
  uint32_t edge = most;
  if (apart) {
    edge = near.resolve(&ties);
    if ((int)threadIdx.x < min(near.count, kNear)) {
      const uint32_t mine = near.key[threadIdx.x];
      const int at = near.at[threadIdx.x], of = at / (each * 256);
      if (mine == edge) atomicAdd(&counts[of][at < c.need ? 1 : 3], 1);
      else if (mine < edge && at < c.need) atomicAdd(&counts[of][0], 1);
      else if (mine > edge && at >= c.need) atomicAdd(&counts[of][2], 1);
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
  int32_t* const fill = lists_of(p, pair);
  int mine_early = 0;
  over([&](const uint32_t (&key)[4], int at) __attribute__((always_inline)) {
    mine_early += list_four(p, table, c, edge, ties, fill, fill + p.moves, key, at, seen, to, from);
  });
  mine_early = lane_scan(mine_early);
  if (lane == 63) atomicAdd(&early, mine_early);
  __syncthreads();
  if (threadIdx.x == 0) p.found[pair] = Found{min(all, p.moves), early, c.recent, c.m, c.need, {0, 0, 0}};
}

template <int kThreads>
__global__ __launch_bounds__(kThreads) void evict_select(EvictArgs p) {
  __shared__ Look look;
  __shared__ Near near;
  const int head = blockIdx.x, request = blockIdx.y;
  Cut c;
  if (c.of(p, request)) return select_whole<kThreads>(p, c, head, request, look, near);  // uniform
  if (threadIdx.x == 0) {
    p.found[(int64_t)request * p.kv_heads + head] = Found{};
    if (head == 0) p.lens[request] = c.n;
  }
}

// Long contexts: the older tokens in parts of 8192, a workgroup each, in three launches, for which one workgroup took 128 us for
// 32 heads of 131,000 tokens (in parts 40). evict_histogram counts each part's weights over the range that a thousand of them
// have, evict_collect finds the part of the range that holds the edge and collects its keys, evict_list finds
// the edge among them and puts each part's places and survivors on the lists.
constexpr int kPart = 8192, kPartThreads = 256, kPartWaves = 4, kCrowd = 4096, kMostParts = 64;

// What the three launches leave for each other, of a head and request.
struct Looked {
  uint32_t low, high, least, most;
  // mode 0: nothing is cut, 1: parts, 2: too many keys at the edge, one workgroup does it all (weights all within 2^-12 of each
  // other but for a thousandth far above: four contexts of 131,000 cut to 32,768 634 us, by one workgroup of sixteen waves 437)
  int32_t ties, crowd, mode, unused;
};
struct Candidate {
  uint32_t key;
  int32_t at;
};

__device__ __forceinline__ int parts_of(const Cut& c) { return (c.m + kPart - 1) / kPart; }

__global__ __launch_bounds__(kPartThreads) void evict_histogram(EvictArgs p) {
  const int head = blockIdx.x, request = blockIdx.y, part = blockIdx.z, wave = threadIdx.x >> 6;
  const int64_t pair = (int64_t)request * p.kv_heads + head;
  Looked* const looked = p.looked + pair;
  Cut c;
  if (!c.of(p, request)) {  // uniform
    if (threadIdx.x == 0 && part == 0) {
      looked->mode = 0;
      p.found[pair] = Found{};
      if (head == 0) p.lens[request] = c.n;
    }
    return;
  }
  if (part >= max(1, parts_of(c))) return;
  __shared__ int bins[kBins], bad;
  __shared__ uint32_t ends[2][kPartWaves];
  for (int i = threadIdx.x; i < kBins; i += kPartThreads) bins[i] = 0;
  if (threadIdx.x == 0) bad = 0;
  const int32_t* const table = p.tables + request * p.table_stride;
  bool missing = false;
  Keys keys;
  uint32_t low = ~0u, high = 0;
  // Four weights a thread, evenly apart over all older tokens: what keys receive falls with their index, so that the first of them
  // alone have a range above the others (weights of log(n / j), four contexts of 131,000 cut to 4096: 62 us; from the range of
  // the first thousand 293, since more keys lie below it than are collected).
  const int four = 4 * (int)((int64_t)threadIdx.x * ((c.m + 3) / 4) / kPartThreads);  // below m
  load_keys(p, table, head, four - 4 * (int)(threadIdx.x & 63), 1, c.m, keys, missing);
#pragma unroll
  for (int j = 0; j < 4; ++j)
    if (four + j < c.m) low = min(low, keys[0][j]), high = max(high, keys[0][j]);
  const int begin = part * kPart + wave * (kPart / kPartWaves);
  load_keys(p, table, head, begin, kQuads, c.m, keys, missing);
  if (part == 0)
    for (int i = (c.m >> p.page_shift) + (int)threadIdx.x; i <= (c.n - 1) >> p.page_shift; i += kPartThreads)
      missing |= (uint32_t)table[i] >= (uint32_t)p.num_pages;
  range_of<kPartWaves>(low, high, ends);
  if (missing) bad = 1;
  const int shift = shift_of(low, high);
#pragma unroll
  for (int i = 0; i < kQuads; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (begin + i * 256 + 4 * (int)(threadIdx.x & 63) + j < c.m) atomicAdd(&bins[part_of(keys[i][j], low, shift)], 1);
  __syncthreads();
  u32x4 eight;
#pragma unroll
  for (int j = 0; j < 4; ++j) eight[j] = (uint32_t)bins[8 * threadIdx.x + 2 * j] | (uint32_t)bins[8 * threadIdx.x + 2 * j + 1] << 16;
  reinterpret_cast<u32x4*>(p.histograms)[(pair * p.parts + part) * kPartThreads + threadIdx.x] = eight;
  if (threadIdx.x == 0) {
    p.bad[pair * p.parts + part] = bad;
    if (part == 0) looked->low = low, looked->high = high, looked->crowd = 0, p.found[pair].early = 0;
  }
}

__global__ __launch_bounds__(kPartThreads) void evict_collect(EvictArgs p) {
  const int head = blockIdx.x, request = blockIdx.y, part = blockIdx.z, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t pair = (int64_t)request * p.kv_heads + head;
  Looked* const looked = p.looked + pair;
  Cut c;
  if (!c.of(p, request)) return;
  const int parts = max(1, parts_of(c));
  if (part >= parts) return;
  __shared__ Look look;
  __shared__ Candidate candidates[kCrowd];
  __shared__ int count, base;
  if (threadIdx.x == 0) count = 0;
  if (threadIdx.x < 3) look.picked[threadIdx.x] = 0;
  const int32_t* const table = p.tables + request * p.table_stride;
  const int begin = part * kPart + wave * (kPart / kPartWaves);
  Keys keys;
  bool missing = false;
  load_keys(p, table, head, begin, kQuads, c.m, keys, missing);
  uint32_t low = looked->low, high = looked->high, least = ~0u, most = ~0u;
  int ties = 0, crowd = 0;
  const bool bad = __syncthreads_or((int)threadIdx.x < parts && p.bad[pair * p.parts + threadIdx.x]);
  if (c.need > 0 && !bad) {  // uniform
    int sums[8] = {0, 0, 0, 0, 0, 0, 0, 0};
    const u32x4* const from = reinterpret_cast<const u32x4*>(p.histograms) + pair * p.parts * kPartThreads + threadIdx.x;
#pragma unroll 4
    for (int x = 0; x < parts; ++x) {
      const u32x4 eight = from[x * kPartThreads];
#pragma unroll
      for (int j = 0; j < 4; ++j) sums[2 * j] += eight[j] & 0xffff, sums[2 * j + 1] += eight[j] >> 16;
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) look.bins[8 * threadIdx.x + j] = sums[j];
    ties = c.need, least = 0;
    crowd = pick<kPartThreads>(look, low, high, least, most, ties);
  }
  const int mode = bad ? 0 : least < most && crowd > kCrowd ? 2 : 1;
  if (threadIdx.x == 0 && part == 0) {
    looked->least = least, looked->most = most, looked->ties = ties, looked->mode = mode;
    if (bad) p.found[pair] = Found{};
    if (head == 0) p.lens[request] = bad ? c.n : c.given;
  }
  if (mode != 1) return;
  // The wave's keys that are evicted or survive for certain, and those of the part found.
  int certain[2] = {0, 0};
#pragma unroll
  for (int i = 0; i < kQuads; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int at = begin + i * 256 + 4 * lane + j;
      const uint32_t key = keys[i][j];
      if (at >= c.m) continue;
      certain[0] += at < c.need && key < least, certain[1] += at >= c.need && key > most;
      if (c.need > 0 && key >= least && key <= most && least < most) {
        const int place = atomicAdd(&count, 1);
        if (place < kCrowd) candidates[place] = Candidate{key, at};
      }
    }
  if (least == most) {
    // all of the part found are equal: counted in place of candidates
    int equal[2] = {0, 0};
#pragma unroll
    for (int i = 0; i < kQuads; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int at = begin + i * 256 + 4 * lane + j;
        if (at < c.m && keys[i][j] == least) ++equal[at >= c.need];
      }
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      const int sum = lane_scan(equal[x]);
      if (lane == 63) p.counts[((pair * p.parts + part) * kPartWaves + wave) * 4 + 2 + x] = sum;
    }
  }
#pragma unroll
  for (int x = 0; x < 2; ++x) {
    const int sum = lane_scan(certain[x]);
    if (lane == 63) p.counts[((pair * p.parts + part) * kPartWaves + wave) * 4 + x] = sum;
  }
  __syncthreads();
  const int mine = min(count, kCrowd);
  if (threadIdx.x == 0 && mine) base = atomicAdd(&looked->crowd, mine);  // (their order does not matter)
  __syncthreads();
  for (int i = threadIdx.x; i < mine; i += kPartThreads)
    if (base + i < kCrowd) p.candidates[pair * kCrowd + base + i] = candidates[i];
}

__global__ __launch_bounds__(kPartThreads) void evict_list(EvictArgs p) {
  const int head = blockIdx.x, request = blockIdx.y, part = blockIdx.z, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t pair = (int64_t)request * p.kv_heads + head;
  __shared__ Look look;
  __shared__ Near near;
  __shared__ int early;
  Cut c;
  if (!c.of(p, request)) return;
  const int parts = max(1, parts_of(c));
  const Looked looked = p.looked[pair];
  if (part >= parts || looked.mode == 0) return;
  if (looked.mode == 2) {
    if (part == 0) select_whole<kPartThreads>(p, c, head, request, look, near);
    return;
  }
  const int32_t* const table = p.tables + request * p.table_stride;
  const int begin = part * kPart + wave * (kPart / kPartWaves);
  Keys keys;
  bool missing = false;
  load_keys(p, table, head, begin, kQuads, c.m, keys, missing);
  near.clear();
  look.clear();
  if (threadIdx.x == 0) early = 0;
  __syncthreads();
  // The edge, among the candidates (every workgroup finds it for itself).
  constexpr int kEach = kCrowd / kPartThreads;
  uint32_t least = looked.least, most = looked.most, edge = most;
  int ties = looked.ties;
  const bool apart = least < most;
  const int crowd = apart ? min(looked.crowd, kCrowd) : 0;
  Candidate mine[kEach];
#pragma unroll
  for (int i = 0; i < kEach; ++i) {  // (mostly few of these are there)
    const int at = i * kPartThreads + (int)threadIdx.x;
    mine[i] = at < crowd ? p.candidates[pair * kCrowd + at] : Candidate{0, 0};
  }
  if (apart) {
    uint32_t low = least, high = most;
    int count = crowd;
    while (least < most && count > kNear) {
      const int shift = shift_of(low, high);
#pragma unroll
      for (int i = 0; i < kEach; ++i)
        if (mine[i].key >= least && mine[i].key <= most && mine[i].key) atomicAdd(&look.bins[part_of(mine[i].key, low, shift)], 1);
      count = pick<kPartThreads>(look, low, high, least, most, ties);
    }
    edge = most;
    if (least < most) {
#pragma unroll
      for (int i = 0; i < kEach; ++i)
        if (mine[i].key && mine[i].key >= least && mine[i].key <= most) near.add(mine[i].key, mine[i].at);
      __syncthreads();
      edge = near.resolve(&ties);
    }
  }
  // Before the wave's indices: places for certain, survivors for certain, and of the keys equal to the edge those below
  // need, and all.
  typedef int32_t i32x4 __attribute__((ext_vector_type(4)));
  const i32x4* const counts = reinterpret_cast<const i32x4*>(p.counts) + pair * p.parts * kPartWaves;
  const Candidate* const candidates = p.candidates + pair * kCrowd;
  int before[4] = {0, 0, 0, 0};
#pragma unroll 4
  for (int w = lane; w < part * kPartWaves + wave; w += 64) {
    const i32x4 of = counts[w];
    before[0] += of[0], before[1] += of[1];
    if (!apart) before[2] += of[2], before[3] += of[2] + of[3];
  }
#pragma unroll 4
  for (int i = lane; i < crowd; i += 64) {
    const Candidate x = candidates[i];
    const bool in = x.at < begin, front = x.at < c.need;
    before[0] += in && x.key < edge && front, before[1] += in && x.key > edge && !front;
    before[2] += in && x.key == edge && front, before[3] += in && x.key == edge;
  }
#pragma unroll
  for (int x = 0; x < 4; ++x) before[x] = __builtin_amdgcn_readlane(lane_scan(before[x]), 63);
  int seen = before[3], to = before[0] + before[2] - min(ties, before[2]), mine_early = 0;
  int from = before[1] + min(ties, before[3]) - min(ties, before[2]);
  int32_t* const fill = lists_of(p, pair);
#pragma unroll
  for (int i = 0; i < kQuads; ++i)
    mine_early += list_four(p, table, c, edge, ties, fill, fill + p.moves, keys[i], begin + i * 256 + 4 * lane, seen, to, from);
  mine_early = lane_scan(mine_early);
  if (lane == 63) atomicAdd(&early, mine_early);
  __syncthreads();
  if (threadIdx.x == 0) {
    Found* const found = p.found + pair;
    if (early) atomicAdd(&found->early, early);
    if (part == 0) found->recent = c.recent, found->from = c.m, found->to = c.need;
  }
  if (part == parts - 1 && threadIdx.x == kPartThreads - 1) p.found[pair].count = min(from, p.moves);  // behind the last wave: all
}

constexpr int kMoveThreads = 256, kAhead = 4;

__device__ __forceinline__ uint16_t* row_at(const EvictArgs& p, uint16_t* cache, int slot, int head) {
  return cache + (int64_t)(slot >> p.page_shift) * p.page_stride + (int64_t)(slot & ((1 << p.page_shift) - 1)) * p.slot_stride +
         (int64_t)head * p.head_stride;
}

__device__ __forceinline__ float* weight_at(const EvictArgs& p, int slot, int head) {
  return p.weights + ((((int64_t)(slot >> p.page_shift) * p.kv_heads + head) << p.page_shift) + (slot & ((1 << p.page_shift) - 1)));
}

// kOnce: as values that are not wanted again soon.
template <bool kOnce>
__device__ __forceinline__ u32x4 load_row(const uint16_t* from) {
  const u32x4* const at = reinterpret_cast<const u32x4*>(from);
  return kOnce ? __builtin_nontemporal_load(at) : *at;
}
template <bool kOnce>
__device__ __forceinline__ void store_row(uint16_t* to, u32x4 x) {
  u32x4* const at = reinterpret_cast<u32x4*>(to);
  if constexpr (kOnce) __builtin_nontemporal_store(x, at); else *at = x;
}

// The rows on a head's lists, and its recent ones. The first p.tails workgroups of a head and request take the recent rows, each
// a share of a row's columns: first the survivors out of the places where those go, then the recent ones from the
// front on, all of a block read before any of it is written, since their old and new places may overlap. The other
// workgroups share the rest of the lists. No other two rows meet: bound by memory.
template <int D, bool kOnce>
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
        if (j + u * rows < last) value[u] = load_row<kOnce>(row_at(p, cache, take[j + u * rows], head));
#pragma unroll
      for (int u = 0; u < kAhead; ++u)
        if (j + u * rows < last) store_row<kOnce>(row_at(p, cache, fill[j + u * rows], head), value[u]);
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
      if (at < f.recent) value[u] = load_row<kOnce>(row_at(p, cache, slot_of(f.from + at), head));
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
      if (at < f.recent) store_row<kOnce>(row_at(p, cache, slot_of(f.to + at), head), value[u]);
    }
    if (weighs) *weight_at(p, slot_of(f.to + at_weight), head) = weight;
  }
}

// Rows of a head that can move: as many as are evicted, and no more than are kept.
int moves_of(int keep, bool given, int max_context) {
  return max(1, given ? max_context / 2 : min(keep, max(0, max_context - keep)));
}

// Parts of the longest context where it is long and the heads are few; 0: one workgroup a head and request. Selection
// takes in its kernels, of one workgroup and of parts: 30 and 31 us for 8 heads of 32,000 tokens, which sixteen waves hold in
// registers, 128 and 40 for 32 heads of 131,000, 145 and 114 for 128 of them, and 452 and 44 for 8 of 500,000.
int parts_of(int64_t pairs, int max_context) {
  const int64_t parts = ((int64_t)max_context + kPart - 1) / kPart;
  return max_context > 1024 * 4 * kQuads && parts <= kMostParts && pairs <= 128 ? (int)parts : 0;
}

// Where the workspace's pieces lie, behind each other; the last is its size.
struct Pieces {
  int64_t found, looked, candidates, bad, counts, histograms, lists, end;
  Pieces(int64_t pairs, int parts, int moves) {
    auto next = [](int64_t from, int64_t bytes) { return from + (bytes + 15) / 16 * 16; };
    found = 0;
    looked = next(found, pairs * sizeof(Found));
    candidates = next(looked, parts ? pairs * sizeof(Looked) : 0);
    bad = next(candidates, parts ? pairs * kCrowd * sizeof(Candidate) : 0);
    counts = next(bad, pairs * parts * 4);
    histograms = next(counts, pairs * parts * kPartWaves * 16);
    lists = next(histograms, pairs * parts * kBins * 2);
    end = next(lists, pairs * moves * 8);
  }
};

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
  *bytes = Pieces((int64_t)requests * kv_heads, parts_of((int64_t)requests * kv_heads, max_context), moves_of(keep, keep < 0, max_context)).end;
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
  // lens are written while other workgroups read the lengths
  const auto list = [](const void* at, int64_t entries) { return Runs{at, 2 * entries, {{1, 0}, {1, 0}, {1, 0}}}; };
  if (meet(list(lens, requests), list(context_lens, requests)) || (keep_lens && meet(list(lens, requests), list(keep_lens, requests))) ||
      meet(list(lens, requests), list(block_tables, (requests - 1) * table_stride + width)))
    return fail(SMX_ERR_INVALID, "lens must share no memory with context_lens, keep_lens and block_tables");
  // rows and weights are moved while others look up where theirs lie
  for (const Runs& moved : {keys, values, all})
    if (meet(moved, list(lens, requests)) || meet(moved, list(context_lens, requests)) ||
        (keep_lens && meet(moved, list(keep_lens, requests))) || meet(moved, list(block_tables, (requests - 1) * table_stride + width)))
      return fail(SMX_ERR_INVALID, "the cache and key_weights must share no memory with the lengths and block_tables");
  EvictArgs p{};
  p.k = (uint16_t*)cache->k, p.v = (uint16_t*)cache->v;
  p.page_stride = cache->page_stride, p.slot_stride = cache->slot_stride, p.head_stride = cache->head_stride;
  p.weights = key_weights, p.context = context_lens, p.tables = block_tables, p.keep_lens = keep_lens;
  p.table_stride = table_stride, p.lens = lens, p.requests = requests, p.kv_heads = cache->kv_heads;
  p.head_dim = cache->head_dim, p.page_shift = __builtin_ctz(cache->page_size), p.num_pages = cache->num_pages;
  p.keep = keep, p.recent = recent, p.max_context = max_context, p.moves = moves_of(keep, keep < 0, max_context);
  const int pairs = requests * cache->kv_heads;
  p.parts = parts_of(pairs, max_context);
  const Pieces at(pairs, p.parts, p.moves);
  char* const base = (char*)workspace;
  p.found = (Found*)(base + at.found), p.looked = (Looked*)(base + at.looked), p.candidates = (Candidate*)(base + at.candidates);
  p.bad = (int32_t*)(base + at.bad), p.counts = (int32_t*)(base + at.counts), p.histograms = (uint16_t*)(base + at.histograms);
  p.lists = (int32_t*)(base + at.lists);
  const dim3 heads((unsigned)cache->kv_heads, (unsigned)requests, (unsigned)max(1, p.parts));
  if (p.parts) {
    for (auto kern : {evict_histogram, evict_collect, evict_list}) {
      hipLaunchKernelGGL(kern, heads, dim3(kPartThreads), 0, (hipStream_t)stream, p);
      if (int rc = check_launch()) return rc;
    }
  } else {
    // four waves where they hold the longest context, else sixteen
    const bool few = max_context <= kPart;
    hipLaunchKernelGGL(few ? evict_select<256> : evict_select<1024>, heads, dim3(few ? 256 : 1024), 0, (hipStream_t)stream, p);
    if (int rc = check_launch()) return rc;
  }
  // Workgroups of a head and request: of 64 rows at least, and so many that they even out (64 requests, weights copied back
  // before each: 133 us; 135 of half as many, 142 of a quarter).
  p.tails = cache->head_dim / 32;
  p.movers = min((p.moves + 63) / 64, max(1, 16384 / pairs));
  // Rows that do not fit into the caches anyway pass them by: four prompts of 131,000 216 us (else 227), 64 requests 133 (138), 47 of
  // which 100 MB may move 59.6 (63.0); but 45 requests with 20 MB 26.0 (23.0), 31 with 14 MB 23.0 (21.0).
  const bool once = (int64_t)pairs * (p.moves + min(recent, max_context)) * 4 * p.head_dim > (64 << 20);
  auto move = cache->head_dim == 128 ? (once ? evict_move<128, true> : evict_move<128, false>)
                                     : (once ? evict_move<64, true> : evict_move<64, false>);
  hipLaunchKernelGGL(move, dim3((unsigned)pairs, (unsigned)(p.tails + p.movers)), dim3(kMoveThreads), 0, (hipStream_t)stream, p);
  return check_launch();
}

}  // extern "C"
