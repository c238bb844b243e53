// The attention weight that cached keys receive (smx_paged_key_weights), summed over a step's rows and the query heads
// of a key/value head.
//
// Mathematics. w_j += sum over the rows i that see key j, and the heads of j's group, of
// e^(scale q_i . k_j - lse_i), lse_i = log sum_j e^(scale q_i . k_j) of the step's attention. A step's own keys start
// from zero. Exponentials are powers of two (scale and lse carry log2 e); scores, exponentials and sums are FP32. Values
// are not read, and with lse at hand no maximum runs along: a score is one multiply-add, one
// exponential and one addition.
//
// Matrix products (v_mfma_f32_32x32x16_bf16): S = Q K^T with the keys across the lanes, so that the sum over rows
// adds up a lane's own registers, and one exchange of the wave's halves at the end.
//
// Work. Keys stay in registers while rows go by. The rows of a request are its tokens' heads of one group, one behind the
// other, in steps of 32; an item is a tile of keys with the steps that see any of it. The steps of all items are cut into equal
// spans, one a workgroup, and the sums of items that a span's end cuts are added up by key_weights_join, in their
// order: repeated calls give the same bits.
#include "launch.hpp"
#include "paged_spans.hpp"

namespace smx {
namespace {

struct WeightArgs {
  const uint16_t *q, *k;
  int64_t q_token, q_head, page_stride, slot_stride, head_stride;
  const int32_t* tables;
  int64_t table_stride;
  const int32_t *starts, *rows, *context;
  const float* lse;
  float* weights;  // [pages, kv_heads, page_size]
  int32_t requests, group, kv_heads, page_shift, num_pages, window, min_span;
  uint32_t per_group;    // 2^16 / group, upwards
  float scale;           // times log2 e
  double per_workgroup;  // 1 / workgroups
  float* partial;
  struct WeightRecord* records;
};

// An item that worker w begins and `others` more finish (0: none).
struct WeightRecord {
  int32_t others, worker, head, request, tile, unused[3];
};

constexpr float kLog2E = 1.44269504088896341f;

// n / d downwards, d > 0.
__device__ __forceinline__ int64_t floor_div(int64_t n, int64_t d) { return n >= 0 ? n / d : -((-n + d - 1) / d); }

// The key tiles of one request, of kTile keys, and the steps of kStepRows rows that see each. An item (one of them) counts kItem
// units before its steps, for its start and end.
constexpr int kBlocks = 3, kWave = 32 * kBlocks, kTile = 4 * kWave, kStepRows = 32, kItem = 3;
struct KeyTiles {
  int32_t context, fresh, group, window, first, tiles;

  __device__ KeyTiles(const WeightArgs& p, int32_t context_, int32_t fresh_)
      : context(context_), fresh(fresh_), group(p.group), window(p.window) {
    first = window ? max(0, context - window + 1) / kTile : 0;
    tiles = (context + fresh + kTile - 1) / kTile - first;
  }
  __device__ static KeyTiles uniform(const WeightArgs& p, int32_t context_, int32_t fresh_) {
    KeyTiles r(p, context_, fresh_);
    r.first = __builtin_amdgcn_readfirstlane(r.first), r.tiles = __builtin_amdgcn_readfirstlane(r.tiles);
    return r;
  }
  // Steps of tile t (counted from the first): those of the tokens at its keys or behind them, in the window of any.
  __device__ int begin(int t) const {
    const int64_t token = max(0, (first + t) * kTile - context);
    return (int)(token * group / kStepRows);
  }
  __device__ int end(int t) const {
    int64_t token = fresh;
    if (window) token = min(token, (int64_t)(first + t) * kTile + kTile - 1 - context + window);
    return (int)((token * group + kStepRows - 1) / kStepRows);
  }
  __device__ int count(int t) const { return end(t) - begin(t); }
  // Units of the tiles before t. kTile is a multiple of kStepRows, so that both ends step by a whole number.
  __device__ int64_t before(int t) const {
    const int64_t a = first, b = first + t, g = group, each = g * (kTile / kStepRows);
    const int64_t all = (g * fresh + kStepRows - 1) / kStepRows;
    int64_t sum = (int64_t)t * kItem + (b - a) * all;
    const auto range = [](int64_t from, int64_t to) { return (from + to - 1) * (to - from) / 2; };  // from + .. + (to - 1)
    if (window) {  // tiles whose last token in sight is not the request's last
      const int64_t last = (int64_t)kTile - 1 - context + window;  // of tile s: s kTile + last
      const int64_t upto = min(b, max(a, -floor_div(last - fresh, kTile)));
      if (upto > a)
        sum += each * range(a, upto) + (upto - a) * (-floor_div(-last * g, kStepRows)) - (upto - a) * all;
    }
    const int64_t from = max(a, (int64_t)context / kTile + 1);  // tiles whose first key is a new one
    if (b > from) sum -= each * range(from, b) + (b - from) * floor_div(-(int64_t)context * g, kStepRows);
    return sum;
  }
  __device__ int64_t all() const { return fresh > 0 ? before(tiles) : 0; }
};

// The keys of one 32-key block of a wave: lane l holds key l % 32, values 16 t + 8 (l / 32) .. of step t.
template <int D>
struct Keys {
  bf16x8 k[D / 16];
};

// Of key `key` of a request: its page (clamped into the cache) and whether it is there.
__device__ __forceinline__ bool find_key(const WeightArgs& p, const int32_t* table, int key, int length, int* page) {
  const int entry = table[min(key, length - 1) >> p.page_shift];
  const bool held = (uint32_t)entry < (uint32_t)p.num_pages;
  *page = held ? entry : 0;
  return held && key < length;
}

template <int D>
__device__ __forceinline__ void load_keys(const WeightArgs& p, Keys<D>& to, int page, int key, int head) {
  const uint16_t* const from = p.k + (int64_t)page * p.page_stride + (int64_t)(key & ((1 << p.page_shift) - 1)) * p.slot_stride +
                               (int64_t)head * p.head_stride + 8 * ((threadIdx.x >> 5) & 1);
#pragma unroll
  for (int t = 0; t < D / 16; ++t) to.k[t] = __builtin_bit_cast(bf16x8, *reinterpret_cast<const u32x4*>(from + 16 * t));
}

__device__ __forceinline__ float* weight_of(const WeightArgs& p, int page, int key, int head) {
  return p.weights + ((((int64_t)page * p.kv_heads + head) << p.page_shift) + (key & ((1 << p.page_shift) - 1)));
}

// Register e of half h holds row 8 (e / 4) + 4 h + e % 4 of a step.
__device__ __forceinline__ int row_of_register(int e, int half) { return 8 * (e >> 2) + 4 * half + (e & 3); }

// Sixteen or four bytes a lane from memory into LDS, lane l's at `to` + its size times l. kOnce: nothing reads them again soon,
// and they need not push out of the caches what is written there.
template <bool kOnce = false>
__device__ __forceinline__ void dma16(const void* from, void* to) {
  __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)(uintptr_t)from,
                                   (__attribute__((address_space(3))) void*)to, 16, 0, kOnce ? 2 : 0);
}
__device__ __forceinline__ void dma4(const void* from, void* to) {
  __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)(uintptr_t)from,
                                   (__attribute__((address_space(3))) void*)to, 4, 0, 0);
}

// Many rows: a workgroup of four waves holds 384 keys, 96 a wave, and its rows pass through LDS, 32 a step, fetched
// three steps ahead. Bound by the matrix instructions, the vector work beside them and the power that both draw: 2048 rows of
// 64 heads on 16384 keys, 0.58 TFLOP, take 600 us (970 TFLOP/s; with each wave's own reads of the rows from memory 888) at a
// clock that falls to 2.0 GHz; 485 where all values are zero. More blocks of keys or a deeper pipeline in a wave did not
// shorten it.
template <int D, bool kWhole>
__global__ __launch_bounds__(256, 2) void key_weights_many(WeightArgs p) {
  constexpr int kRow = 2 * D, kChunks = D / 8, kLoads = kStepRows * kChunks / 256, kRing = 4;
  // (LDS of a size that the launch says: behind arrays that the compiler knows it waits for every DMA before a read)
  extern __shared__ __attribute__((aligned(1024))) uint8_t lds[];
  constexpr int kStep = kStepRows * kRow;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), half = lane >> 5;
  WeightRecord* const record = p.records + blockIdx.x;
  if (threadIdx.x == 0) record->others = 0;
  Span s;
  if (!find_span<KeyTiles, 4>(p, &s)) return;
  const int64_t heads = (int64_t)p.group * p.kv_heads;
  const int step_tokens = kStepRows / p.group, step_heads = kStepRows - step_tokens * p.group;

  while (s.left > 0) {
    const KeyTiles r = KeyTiles::uniform(p, s.context, s.fresh);
    const int tile_count = r.count(s.tile);
    const int units = (int)min((int64_t)(tile_count + kItem - s.skip), s.left), rest = tile_count + kItem - s.skip - units;
    const int before = max(0, s.skip - kItem), upto = max(0, s.skip + units - kItem);
    const int from = r.begin(s.tile) + before, count = upto - before;
    if (count > 0) {
      const int length = s.context + s.fresh, key0 = (r.first + s.tile) * kTile + kWave * wave;
      const int32_t* const table = p.tables + s.request * p.table_stride;
      const int64_t start = scalar_at(p.starts, s.request);
      const int rows = s.fresh * p.group;
      // The rows that see a key are consecutive: of the tokens at it and behind it, less than a window from it.
      auto first_row = [&](int key) __attribute__((always_inline)) { return max(0, key - s.context) * p.group; };
      auto last_row = [&](int key) __attribute__((always_inline)) {
        return p.window ? max(0, min(s.fresh, key - s.context + p.window)) * p.group : rows;
      };
      Keys<D> k[kBlocks];
#pragma unroll
      for (int x = 0; x < kBlocks; ++x) {
        const int key = key0 + 32 * x + (lane & 31);
        int page;
        find_key(p, table, key, length, &page);
        load_keys<D>(p, k[x], page, min(key, length - 1), s.head);
      }
      const int all_from = first_row(key0 + kWave - 1), all_upto = last_row(key0);  // rows that see all of the wave's keys
      // The rows of the next step to be fetched: chunks of 16 bytes, and a row's lse, from the first row's token on (the host
      // made sure that a step's queries lie within 2^32 bytes). Rows behind the last are fetched as that one, and count for
      // nothing. In steps of whole tokens (kWhole) a lane keeps its place in them and in the last one.
      const int last_step = (rows - 1) / kStepRows;
      int fetched = min(from, last_step);
      const int token0 = (uint32_t)(fetched * kStepRows) / (uint32_t)p.group;
      int head0 = fetched * kStepRows - token0 * p.group;  // of the step's first row
      const uint8_t* q_from = reinterpret_cast<const uint8_t*>(p.q + (start + token0) * p.q_token + (int64_t)s.head * p.group * p.q_head);
      const uint8_t* lse_from = reinterpret_cast<const uint8_t*>(p.lse + (start + token0) * heads + s.head * p.group);
      // bytes to the lane's row of DMA i (kLoads: the lse), none behind row `most` of the step
      auto place = [&](int i, int most) __attribute__((always_inline)) -> uint32_t {
        const uint32_t in = i < kLoads ? ((kLoads * wave + i) * 64 + lane) / kChunks : lane & 31;
        const uint32_t row = head0 + min(in, (uint32_t)most);               // below 32 + 128: exact
        const uint32_t token = row * p.per_group >> 16, head = row - token * p.group;
        if (i == kLoads) return 4 * (token * (uint32_t)heads + head);
        return 2 * (token * (uint32_t)p.q_token + head * (uint32_t)p.q_head) + 16 * (lane % kChunks ^ (in & (kChunks - 1)));
      };
      uint32_t at[kLoads + 1], at_last[kLoads + 1];
      if constexpr (kWhole)
#pragma unroll
        for (int i = 0; i <= kLoads; ++i) at[i] = place(i, kStepRows - 1), at_last[i] = place(i, rows - 1 - last_step * kStepRows);
      auto fetch = [&](int i) __attribute__((always_inline)) {
        const int buffer = i & (kRing - 1);
        uint8_t* const to = lds + buffer * kStep + kLoads * 1024 * wave;
        const bool last = fetched >= last_step;  // uniform
#pragma unroll
        for (int x = 0; x < kLoads; ++x)
          dma16(q_from + (!kWhole ? place(x, rows - 1 - fetched * kStepRows) : last ? at_last[x] : at[x]), to + 1024 * x);
        dma4(lse_from + (!kWhole ? place(kLoads, rows - 1 - fetched * kStepRows) : last ? at_last[kLoads] : at[kLoads]),
             lds + kRing * kStep + 256 * (kRing * wave + buffer));  // a wave's own: each row's lse, twice
        const int heads_on = head0 + step_heads, wraps = heads_on >= p.group;  // on to the next step, if there is one
        fetched += last ? 0 : 1;
        if constexpr (!kWhole) head0 = last ? head0 : heads_on - (wraps ? p.group : 0);
        const int64_t tokens = last ? 0 : step_tokens + (kWhole ? 0 : wraps);
        q_from += 2 * tokens * p.q_token, lse_from += 4 * tokens * heads;
      };
      float total[kBlocks];
#pragma unroll
      for (int x = 0; x < kBlocks; ++x) total[x] = 0.f;
      // Weights of a block's scores, added up.
      auto weigh = [&](f32x16& score, const f32x4 (&lse)[4], int x) __attribute__((always_inline)) {
#pragma unroll
        for (int e = 0; e < 16; ++e)
          score[e] = __builtin_amdgcn_exp2f(__builtin_fmaf(score[e], p.scale, lse[e >> 2][e & 3]));
        float part[2] = {score[0], score[1]};
#pragma unroll
        for (int e = 2; e < 16; ++e) part[e & 1] += score[e];
        total[x] += part[0] + part[1];
      };
      // The same of rows some of which do not see some of the keys.
      auto weigh_some = [&](f32x16& score, const f32x4 (&lse)[4], int x, int row0) __attribute__((always_inline)) {
        float sum = 0.f;
        const int key = key0 + 32 * x + (lane & 31), first = first_row(key) - row0 - 4 * half, last = last_row(key) - row0 - 4 * half;
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          const int row = row_of_register(e, 0);  // (less row0 + 4 half, as the bounds)
          const float w = __builtin_amdgcn_exp2f(__builtin_fmaf(score[e], p.scale, lse[e >> 2][e & 3]));
          sum += row >= first && row < last ? w : 0.f;
        }
        total[x] += sum;
      };
      bf16x8 q[D / 16];
      f32x16 score[2];
      auto slot_of = [&](int i) { return i & (kRing - 1); };
      auto lse_slot = [&](int i) { return reinterpret_cast<float*>(lds + kRing * kStep + 256 * (kRing * wave + slot_of(i))); };
      auto read_row = [&](int i, int t) __attribute__((always_inline)) {
        q[t] = __builtin_bit_cast(bf16x8, *reinterpret_cast<const u32x4*>(lds + slot_of(i) * kStep + (lane & 31) * kRow +
                                                                         16 * ((2 * t + half) ^ (lane & (kChunks - 1)))));
      };
      auto read_lse = [&](int i, f32x4 (&lse)[4]) __attribute__((always_inline)) {
#pragma unroll
        for (int e = 0; e < 4; ++e) lse[e] = *reinterpret_cast<const f32x4*>(lse_slot(i) + 8 * e + 4 * half);
      };
      auto multiply = [&](f32x16& score, int x, int next) __attribute__((always_inline)) {
#pragma unroll
        for (int e = 0; e < 16; ++e) score[e] = 0.f;
#pragma unroll
        for (int t = 0; t < D / 16; ++t) {
          score = __builtin_amdgcn_mfma_f32_32x32x16_bf16(q[t], k[x].k[t], score, 0, 0, 0);
          if (next) read_row(next, t);
        }
      };
      // all but the fetches of `steps` steps, of every wave
      auto arrived = [&](auto steps) __attribute__((always_inline)) {
        asm volatile("s_waitcnt vmcnt(%0)\n\ts_barrier" ::"i"(decltype(steps)::value * (kLoads + 1)) : "memory");
      };
      // the next step's rows are there, and every wave has read this one's
      auto next_step = [&](int i) __attribute__((always_inline)) {
        __builtin_amdgcn_sched_barrier(0);
        arrived(std::integral_constant<int, kRing - 2>());
        fetch(i + kRing);
        __builtin_amdgcn_sched_barrier(0);
      };
      // A step some of whose rows do not see some of the keys.
      auto some = [&](int i) __attribute__((always_inline)) {
        f32x4 lse[4];
        read_lse(i, lse);
#pragma unroll
        for (int e = 0; e < 4; ++e) lse[e] *= -kLog2E;
#pragma unroll
        for (int x = 0; x < kBlocks; ++x) {
          multiply(score[0], x, 0);
          weigh_some(score[0], lse, x, (from + i) * kStepRows);
        }
        next_step(i);
#pragma unroll
        for (int t = 0; t < D / 16; ++t) read_row(i + 1, t);
      };
      // A step whose rows see all keys. A block's products run beside the weights of the block before: a matrix instruction,
      // then as much vector work as the matrix core takes for it. The next step's rows are read beside the last
      // block's. `before`: lse (times -log2 e) of the step before, `now` of this one, by way of LDS: a lane's row
      // is scaled by one instruction, and then read as the registers need it. kFirst: where the first block's scores go.
      float mine = 0.f;
      auto all = [&](auto kFirst, int i, const f32x4 (&before)[4], f32x4 (&now)[4]) __attribute__((always_inline)) {
        lse_slot(i)[lane] = mine * -kLog2E;
        read_lse(i, now);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int x = 0; x < kBlocks; ++x) {
          const int to = (decltype(kFirst)::value + x) & 1;
          const bool ends = x == kBlocks - 1;
          if (ends) next_step(i);
          multiply(score[to], x, ends ? i + 1 : 0);
          if (ends) mine = lse_slot(i + 1)[lane];
          weigh(score[to ^ 1], x ? now : before, x ? x - 1 : kBlocks - 1);
#pragma unroll
          for (int t = 0; t < D / 16; ++t) {
            __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);            // a matrix instruction
            __builtin_amdgcn_sched_group_barrier(0x002, 4 * 128 / D, 0);  // vector ones
            __builtin_amdgcn_sched_group_barrier(0x400, 2 * 128 / D, 0);  // exponentials
            if (ends) __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);  // a read of LDS
          }
          __builtin_amdgcn_sched_barrier(0);
        }
      };
      // the item before: its rows are read, its fetches have arrived
      asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
#pragma unroll
      for (int i = 0; i < kRing; ++i) fetch(i);
      arrived(std::integral_constant<int, kRing - 1>());
#pragma unroll
      for (int t = 0; t < D / 16; ++t) read_row(0, t);
      // (uniform) the steps whose rows see all of the wave's keys lie between others
      const int all_begin = min(count, max(0, (all_from + kStepRows - 1) / kStepRows - from));
      const int all_end = min(count, max(all_begin, all_upto / kStepRows - from));
      int i = 0;
#pragma unroll 1
      for (; i < all_begin; ++i) some(i);
      if (i < all_end) {
        constexpr std::integral_constant<int, 0> kEven{};
        constexpr std::integral_constant<int, kBlocks & 1> kOdd{};
        f32x4 lse[2][4];
        // nothing is left of a step before: scores of -inf, whose weights are zero
#pragma unroll
        for (int e = 0; e < 16; ++e) score[1][e] = -INFINITY, lse[0][e >> 2][e & 3] = 0.f;
        mine = lse_slot(i)[lane];
#pragma unroll 1
        for (; i + 1 < all_end; i += 2) all(kEven, i, lse[0], lse[1]), all(kOdd, i + 1, lse[1], lse[0]);
        if (i < all_end) {
          all(kEven, i, lse[0], lse[1]), ++i;
          weigh(score[(kBlocks - 1) & 1], lse[1], kBlocks - 1);
        } else {
          weigh(score[1], lse[0], kBlocks - 1);
        }
      }
#pragma unroll 1
      for (; i < count; ++i) some(i);
      const int begins = before == 0;
      float* const part = p.partial + (2 * (int64_t)s.worker + begins) * kTile + kWave * wave;
#pragma unroll
      for (int x = 0; x < kBlocks; ++x) {
        total[x] += other_half(total[x]);
        if (half) continue;  // (both halves hold the sum)
        const int key = key0 + 32 * x + lane;
        int page;
        if (count < tile_count) {
          part[32 * x + lane] = total[x];
        } else if (find_key(p, table, key, length, &page)) {
          float* const to = weight_of(p, page, key, s.head);
          *to = (key < s.context ? *to : 0.f) + total[x];
        }
      }
      if (count < tile_count && begins && threadIdx.x == 0) {
        record->worker = s.worker, record->head = s.head, record->request = s.request, record->tile = s.tile;
        record->others = (int)quotient(rest + s.each - 1, s.each);
      }
    }
    s.left -= units;
    if (s.left <= 0) break;
    next_item(p, &s, r.tiles);
  }
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // no DMA outlives the workgroup
}

// Adds up the sums of an item that several workgroups share: a thread per key.
__global__ __launch_bounds__(kTile) void key_weights_join(WeightArgs p) {
  const WeightRecord record = p.records[blockIdx.x];
  if (record.others <= 0) return;
  const int context = p.context[record.request], fresh = p.rows[record.request];
  const KeyTiles r(p, context, fresh);
  const int key = (r.first + record.tile) * kTile + (int)threadIdx.x;
  int page;
  const bool held = find_key(p, p.tables + record.request * p.table_stride, key, context + fresh, &page);
  if (!held) return;
  float* const to = weight_of(p, page, key, record.head);
  float sum = 0.f;
#pragma unroll 4
  for (int i = 0; i <= record.others; ++i)
    sum += p.partial[(2 * (int64_t)(record.worker + i) + (i == 0)) * kTile + threadIdx.x];
  *to = (key < context ? *to : 0.f) + sum;
}

// A request of few rows is one item: its tiles of 32 keys.
struct FewTiles {
  static constexpr int kKeys = 32;
  int32_t context, fresh, first, tiles, steps;

  __device__ FewTiles(const WeightArgs& p, int32_t context_, int32_t fresh_) : context(context_), fresh(fresh_), tiles(1) {
    first = p.window ? max(0, context - p.window + 1) / kKeys : 0;
    steps = (context + fresh + kKeys - 1) / kKeys - first;
  }
  __device__ static FewTiles uniform(const WeightArgs& p, int32_t context_, int32_t fresh_) {
    FewTiles r(p, context_, fresh_);
    r.first = __builtin_amdgcn_readfirstlane(r.first), r.steps = __builtin_amdgcn_readfirstlane(r.steps);
    return r;
  }
  __device__ int64_t before(int t) const { return t ? all() : 0; }
  __device__ int64_t all() const { return fresh > 0 ? steps + 1 : 0; }  // one for its start
};

// Few rows (at most 32 of a request, decoding): a wave holds them and its keys go by, 32 at a time, through two tiles in
// LDS, one on its way while the other is weighed. Keys are loaded as such that are read once, so that the weights written wait
// in the caches for more of their kind. Bound by memory: 64 requests of 64 heads on 4200 keys on average, 550 MB, take 108 us
// (5.1 TB/s; keys loaded like any others 118), four on 131,000, 1.1 GB, 202 us (5.5 TB/s; 222).
template <int D>
__global__ __launch_bounds__(64) void key_weights_few(WeightArgs p) {
  constexpr int kRow = 2 * D, kChunks = D / 8, kDmaRows = 64 / kChunks, kDmas = 32 / kDmaRows, kRing = 2;
  constexpr int kSlot = 32 * kRow + 256;  // a tile's keys, and its weights before the step (twice)
  extern __shared__ __attribute__((aligned(1024))) uint8_t lds[];
  const int lane = threadIdx.x, half = lane >> 5;
  Span s;
  if (!find_span<FewTiles, 1>(p, &s)) return;
  // The lane's part of eight rows of a page, of a tile's even and odd groups of them: DMA i of a group brings kDmaRows rows.
  uint32_t at[2][8 / kDmaRows];
#pragma unroll
  for (int g = 0; g < 2; ++g)
#pragma unroll
    for (int i = 0; i < 8 / kDmaRows; ++i) {
      const int row = i * kDmaRows + lane / kChunks;
      at[g][i] = (uint32_t)row * (uint32_t)p.slot_stride * 2 + 16 * (lane % kChunks ^ ((8 * g + row) & (kChunks - 1)));
    }
  while (s.left > 0) {
    const FewTiles r = FewTiles::uniform(p, s.context, s.fresh);
    const int units = (int)min((int64_t)(r.steps + 1 - s.skip), s.left);
    const int before = max(0, s.skip - 1), count = max(0, s.skip + units - 1) - before;
    if (count > 0) {
      const int length = s.context + s.fresh, rows = min(s.fresh * p.group, kStepRows);
      const int32_t* const table = p.tables + s.request * p.table_stride;
      const int64_t start = scalar_at(p.starts, s.request);
      const int row = min(lane & 31, rows - 1), token = row / p.group, head = s.head * p.group + row - token * p.group;
      const uint16_t* const from = p.q + (start + token) * p.q_token + (int64_t)head * p.q_head + 8 * half;
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // the item before: its last fetches and stores
      bf16x8 q[D / 16];
#pragma unroll
      for (int t = 0; t < D / 16; ++t) q[t] = __builtin_bit_cast(bf16x8, *reinterpret_cast<const u32x4*>(from + 16 * t));
      const float mine = lane < rows ? p.lse[(start + token) * ((int64_t)p.group * p.kv_heads) + head] * kLog2E : INFINITY;
      float lse[16];
#pragma unroll
      for (int e = 0; e < 16; ++e) lse[e] = __shfl(mine, row_of_register(e, half));
      const int low = s.context, high = s.context + s.fresh - 1;
      const int key_first = (r.first + before) * FewTiles::kKeys, last_page = (length - 1) >> p.page_shift;
      // Lane l holds entry l of 64 table entries, and of the 64 behind them; no tile's pages lie in both.
      int first_page = key_first >> p.page_shift;
      auto entries_of = [&](int page) __attribute__((always_inline)) { return table[min(page + lane, last_page)]; };
      int entries = entries_of(first_page), more = entries_of(first_page + 64);
      // Starts a tile's fetches; the lane's key's page. Tiles past the item's last are fetched as that one again, so that the
      // number of fetches in flight stays the same.
      auto fetch = [&](int i) __attribute__((always_inline)) {
        const int key0 = key_first + min(i, count - 1) * FewTiles::kKeys;
        uint8_t* const to = lds + (i & (kRing - 1)) * kSlot;
        if ((key0 >> p.page_shift) - first_page >= 64) {  // uniform
          first_page += 64;
          entries = more, more = entries_of(first_page + 64);
        }
#pragma unroll
        for (int g = 0; g < 4; ++g) {
          const int key = key0 + 8 * g, entry = __builtin_amdgcn_readlane(entries, (key >> p.page_shift) - first_page);
          const int64_t page = (uint32_t)entry < (uint32_t)p.num_pages ? entry : 0;
          const uint8_t* const base = reinterpret_cast<const uint8_t*>(
              p.k + page * p.page_stride + (int64_t)(key & ((1 << p.page_shift) - 1)) * p.slot_stride + (int64_t)s.head * p.head_stride);
#pragma unroll
          for (int x = 0; x < 8 / kDmaRows; ++x) dma16<true>(base + at[g & 1][x], to + (g * 8 + x * kDmaRows) * kRow);
        }
        const int key = key0 + (lane & 31), entry = __shfl(entries, (key >> p.page_shift) - first_page);
        dma4(weight_of(p, (uint32_t)entry < (uint32_t)p.num_pages ? entry : 0, key, s.head), to + 32 * kRow);
        return entry;
      };
      auto add = [&](int i, int entry) __attribute__((always_inline)) {
        const int key0 = key_first + i * FewTiles::kKeys, key = key0 + (lane & 31);
        const uint8_t* const tile = lds + (i & (kRing - 1)) * kSlot;
        bf16x8 k[D / 16];
#pragma unroll
        for (int t = 0; t < D / 16; ++t)
          k[t] = __builtin_bit_cast(bf16x8, *reinterpret_cast<const u32x4*>(tile + (lane & 31) * kRow + 16 * ((2 * t + half) ^ (lane & (kChunks - 1)))));
        const float old = *reinterpret_cast<const float*>(tile + 32 * kRow + 4 * lane);
        f32x16 score;
#pragma unroll
        for (int e = 0; e < 16; ++e) score[e] = 0.f;
#pragma unroll
        for (int t = 0; t < D / 16; ++t) score = __builtin_amdgcn_mfma_f32_32x32x16_bf16(q[t], k[t], score, 0, 0, 0);
        const bool masked = key0 + FewTiles::kKeys - 1 > low || (p.window && key0 <= high - p.window);
        float sum = 0.f;
#pragma unroll
        for (int e = 0; e < 16; e += 4)
          if (2 * e < rows) {  // (uniform: registers of rows that are there)
#pragma unroll
            for (int j = e; j < e + 4; ++j) {
              float w = __builtin_amdgcn_exp2f(__builtin_fmaf(score[j], p.scale, -lse[j]));
              if (masked) {
                const int place = s.context + __shfl(token, row_of_register(j, half));
                w = key <= place && (!p.window || key > place - p.window) ? w : 0.f;
              }
              sum += w;
            }
          }
        sum += other_half(sum);
        if (!half && key < length && (uint32_t)entry < (uint32_t)p.num_pages)
          *weight_of(p, entry, key, s.head) = (key < s.context ? old : 0.f) + sum;
      };
      int entry[kRing];  // of this tile and those on their way
#pragma unroll
      for (int i = 0; i < kRing - 1; ++i) entry[i] = fetch(i);
      for (int i = 0; i < count; ++i) {
        // all but the fetches of the tiles behind this one
        asm volatile("s_waitcnt vmcnt(%0)" ::"i"((kRing - 2) * (kDmas + 1)) : "memory");
        __builtin_amdgcn_sched_barrier(0);
        entry[kRing - 1] = fetch(i + kRing - 1);
        __builtin_amdgcn_sched_barrier(0);
        add(i, entry[0]);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int x = 0; x + 1 < kRing; ++x) entry[x] = entry[x + 1];
      }
    }
    s.left -= units;
    if (s.left <= 0) break;
    next_item(p, &s, r.tiles);
  }
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // no DMA outlives the wave
}

// Workgroups of a launch, a multiple of the 8 XCDs. Of few rows as many as a CU holds, by their LDS (17 KB at head_dim 128,
// of which nine would fit but not even out). With rings of four tiles and half as many waves 64 requests took 120 us in place of
// 118, 18 requests of head_dim 64 37 in place of 35 (both before keys were loaded as read once). Of many rows
// twice as many: a CU serves the workgroup that came first before the other, so that the last ones run alone
// (2048 rows of 64 heads on 16384 keys: 672 us with as many as fit, 604 with twice as many, 605 with four times).
int few_workgroups(int cus, int head_dim) { return ((head_dim == 128 ? 8 : 16) * cus + 7) / 8 * 8; }
int many_workgroups(int cus) { return (4 * cus + 7) / 8 * 8; }

int64_t workspace_of(int cus) { return many_workgroups(cus) * (int64_t)(sizeof(WeightRecord) + 2 * 4 * kTile); }

template <int D>
int launch_weights(const WeightArgs& p, bool few, unsigned blocks, hipStream_t stream) {
  auto many = kStepRows % p.group == 0 ? key_weights_many<D, true> : key_weights_many<D, false>;
  hipLaunchKernelGGL(few ? key_weights_few<D> : many, dim3(blocks), dim3(few ? 64 : 256),
                     few ? 2 * (32 * 2 * D + 256) : 4 * (kStepRows * 2 * D + 4 * 256), stream, p);
  if (int rc = check_launch()) return rc;
  if (few) return SMX_OK;
  hipLaunchKernelGGL(key_weights_join, dim3(blocks), dim3(kTile), 0, stream, p);
  return check_launch();
}

}  // namespace
}  // namespace smx

using namespace smx;

extern "C" {

int smx_paged_key_weights_workspace_bytes(int64_t* bytes) {
  smx::fail(SMX_OK, "%s", "");
  if (!bytes) return fail(SMX_ERR_INVALID, "null pointer");
  int cus = 0;
  if (int rc = device_cus(&cus)) return rc;
  *bytes = workspace_of(cus);
  return SMX_OK;
}

int smx_paged_key_weights(const smx_paged_cache* cache, const smx_paged_step* step, const smx_heads* q, const float* lse,
                          float scale, int32_t window, float* key_weights, void* workspace, int64_t workspace_bytes,
                          void* stream) {
  smx::fail(SMX_OK, "%s", "");
  if (int rc = paged_layout(cache)) return rc;
  if (!step || !step->block_tables || !step->starts || !step->rows || !step->context || !q || !q->data || !lse || !key_weights)
    return fail(SMX_ERR_INVALID, "null pointer");
  if (step->requests <= 0 || step->requests > SMX_PAGED_MAX_REQUESTS || step->tokens <= 0 ||
      step->tokens > SMX_PAGED_MAX_TOKENS || step->max_new < 0 || step->table_stride <= 0)
    return fail(SMX_ERR_INVALID, "a step has 1 to %d requests and 1 to %d tokens (requests=%d, tokens=%d)",
                SMX_PAGED_MAX_REQUESTS, SMX_PAGED_MAX_TOKENS, step->requests, step->tokens);
  if (q->heads <= 0 || q->heads % cache->kv_heads || q->heads / cache->kv_heads > 128)
    return fail(SMX_ERR_INVALID, "%d query heads are not 1 to 128 for each of %d key/value heads", q->heads, cache->kv_heads);
  if ((uintptr_t)q->data % 16 || q->token_stride % 8 || q->head_stride % 8 || q->token_stride < 0 || q->head_stride < 0)
    return fail(SMX_ERR_INVALID, "head rows must be 16-byte aligned");
  // (offsets within a step's rows are of 32 bits)
  const int64_t group = q->heads / cache->kv_heads, tokens = kStepRows / group + 2;
  if (q->token_stride > INT32_MAX / tokens || q->head_stride > INT32_MAX / group ||
      tokens * q->token_stride + group * q->head_stride + cache->head_dim > INT32_MAX)
    return fail(SMX_ERR_UNSUPPORTED, "the query heads of %d rows must lie within 2^32 bytes", kStepRows);
  if ((uintptr_t)lse % 4 || (uintptr_t)key_weights % 16) return fail(SMX_ERR_INVALID, "misaligned lse or key_weights");
  const Runs to{key_weights, 2 * (int64_t)cache->num_pages * cache->kv_heads * cache->page_size, {{1, 0}, {1, 0}, {1, 0}}};
  const Runs sums{lse, 2 * (int64_t)step->tokens * q->heads, {{1, 0}, {1, 0}, {1, 0}}};
  if (meet(to, cache_runs(*cache, cache->k)) || meet(to, head_runs(*q, step->tokens, cache->head_dim)) || meet(to, sums))
    return fail(SMX_ERR_INVALID, "key_weights must share no memory with the keys, the queries and lse");
  // (a workgroup's lengths and tables are read while others store)
  if (meets_step(key_weights, 2 * to.width, *step)) return fail(SMX_ERR_INVALID, "key_weights must share no memory with the step's lists");
  if (!(scale > 0.f) || !(scale * kLog2E < INFINITY))
    return fail(SMX_ERR_INVALID, "scale must be positive and finite, also times log2 e");
  if (window < 0) return fail(SMX_ERR_INVALID, "window must not be negative (0: none)");
  int cus = 0;
  if (int rc = device_cus(&cus)) return rc;
  if (!workspace || (uintptr_t)workspace % 16 || workspace_bytes < workspace_of(cus))
    return fail(SMX_ERR_INVALID, "the call needs a 16-byte aligned workspace of %lld bytes", (long long)workspace_of(cus));
  WeightArgs p{};
  p.q = (const uint16_t*)q->data, p.q_token = q->token_stride, p.q_head = q->head_stride;
  p.k = (const uint16_t*)cache->k;
  p.page_stride = cache->page_stride, p.slot_stride = cache->slot_stride, p.head_stride = cache->head_stride;
  p.tables = step->block_tables, p.table_stride = step->table_stride;
  p.starts = step->starts, p.rows = step->rows, p.context = step->context;
  p.lse = lse, p.weights = key_weights;
  p.requests = step->requests, p.kv_heads = cache->kv_heads, p.group = q->heads / cache->kv_heads;
  p.page_shift = __builtin_ctz(cache->page_size), p.num_pages = cache->num_pages;
  p.window = window < SMX_PAGED_MAX_CONTEXT ? window : 0;  // wider than any request: none
  const bool few = (int64_t)max(1, step->max_new) * p.group <= kStepRows;
  const int blocks = few ? few_workgroups(cus, cache->head_dim) : many_workgroups(cus);
  // Small steps are spread over more workgroups than have whole items: 14 requests of up to 22 tokens take 12.5 us, with spans
  // of kItem + 4 units 15.6; 3 of up to 465 21.5, with kItem - 1 27.5.
  p.min_span = few ? 1 : kItem + 1;
  p.scale = scale * kLog2E;
  p.per_group = (65535 + p.group) / p.group;
  p.per_workgroup = 1. / blocks;
  p.records = (WeightRecord*)workspace;
  p.partial = (float*)((char*)workspace + blocks * sizeof(WeightRecord));
  return cache->head_dim == 128 ? launch_weights<128>(p, few, (unsigned)blocks, (hipStream_t)stream)
                                : launch_weights<64>(p, few, (unsigned)blocks, (hipStream_t)stream);
}

}  // extern "C"
