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

// The key tiles of one request, of kTile keys, and the steps of 32 rows that see each. An item (one of them) counts kItem
// units before its steps, for its start and end.
constexpr int kTile = 256, kStepRows = 32, kItem = 3;
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

// Many rows: a workgroup of four waves holds 256 keys, 64 a wave, and its rows pass through LDS, 32 at a time.
template <int D>
__global__ __launch_bounds__(256, 2) void key_weights_many(WeightArgs p) {
  constexpr int kRow = 2 * D, kChunks = D / 8, kLoads = kStepRows * kChunks / 256;
  __shared__ __attribute__((aligned(1024))) uint8_t q_tiles[2][kStepRows * kRow];
  __shared__ __attribute__((aligned(16))) float sums[2][kStepRows];
  __shared__ __attribute__((aligned(16))) int32_t places[2][kStepRows];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), half = lane >> 5;
  WeightRecord* const record = p.records + blockIdx.x;
  if (threadIdx.x == 0) record->others = 0;
  Span s;
  if (!find_span<KeyTiles, 4>(p, &s)) return;

  while (s.left > 0) {
    const KeyTiles r = KeyTiles::uniform(p, s.context, s.fresh);
    const int tile_count = r.count(s.tile);
    const int units = (int)min((int64_t)(tile_count + kItem - s.skip), s.left), rest = tile_count + kItem - s.skip - units;
    const int before = max(0, s.skip - kItem), upto = max(0, s.skip + units - kItem);
    const int from = r.begin(s.tile) + before, count = upto - before;
    if (count > 0) {
      const int length = s.context + s.fresh, key0 = (r.first + s.tile) * kTile + 64 * wave;
      const int32_t* const table = p.tables + s.request * p.table_stride;
      const int64_t start = scalar_at(p.starts, s.request);
      const int rows = s.fresh * p.group;
      Keys<D> k[2];
      int page[2];
      bool held[2];
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        const int key = min(key0 + 32 * x + (lane & 31), length - 1);
        held[x] = find_key(p, table, key0 + 32 * x + (lane & 31), length, &page[x]);
        load_keys<D>(p, k[x], page[x], key, s.head);
      }
      // The thread's part of a step's rows: chunks of 16 bytes, and (the first 32) a row's sum and place.
      u32x4 chunk[kLoads];
      float sum = 0.f;
      int32_t place = 0;
      auto load_rows = [&](int step) __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < kLoads; ++i) {
          const int at = threadIdx.x + 256 * i, row = min(step * kStepRows + at / kChunks, rows - 1);
          const int token = (uint32_t)row / (uint32_t)p.group, head = row - token * p.group;
          chunk[i] = *reinterpret_cast<const u32x4*>(p.q + (start + token) * p.q_token +
                                                     (int64_t)(s.head * p.group + head) * p.q_head + at % kChunks * 8);
        }
        if (threadIdx.x < kStepRows) {
          const int at = step * kStepRows + (int)threadIdx.x, row = min(at, rows - 1);
          const int token = (uint32_t)row / (uint32_t)p.group, head = row - token * p.group;
          const float lse = p.lse[(start + token) * ((int64_t)p.group * p.kv_heads) + s.head * p.group + head];
          sum = at < rows ? lse * kLog2E : INFINITY;
          place = s.context + token;
        }
      };
      auto store_rows = [&](int buffer) __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < kLoads; ++i) {
          const int at = threadIdx.x + 256 * i, row = at / kChunks, c = at % kChunks;
          *reinterpret_cast<u32x4*>(q_tiles[buffer] + row * kRow + 16 * (c ^ (row & (kChunks - 1)))) = chunk[i];
        }
        if (threadIdx.x < kStepRows) sums[buffer][threadIdx.x] = sum, places[buffer][threadIdx.x] = place;
      };
      float total[2] = {0.f, 0.f};
      __syncthreads();  // the item before has read its rows
      load_rows(from);
      store_rows(0);
      for (int i = 0; i < count; ++i) {
        const int buffer = i & 1;
        __syncthreads();
        if (i + 1 < count) load_rows(from + i + 1);
        bf16x8 q[D / 16];
#pragma unroll
        for (int t = 0; t < D / 16; ++t)
          q[t] = __builtin_bit_cast(bf16x8, *reinterpret_cast<const u32x4*>(q_tiles[buffer] + (lane & 31) * kRow +
                                                                           16 * ((2 * t + half) ^ (lane & (kChunks - 1)))));
        f32x4 lse[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) lse[e] = *reinterpret_cast<const f32x4*>(&sums[buffer][8 * e + 4 * half]);
        f32x16 score[2];
#pragma unroll
        for (int x = 0; x < 2; ++x)
#pragma unroll
          for (int e = 0; e < 16; ++e) score[x][e] = 0.f;
#pragma unroll
        for (int t = 0; t < D / 16; ++t)
#pragma unroll
          for (int x = 0; x < 2; ++x) score[x] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(q[t], k[x].k[t], score[x], 0, 0, 0);
#pragma unroll
        for (int x = 0; x < 2; ++x)
#pragma unroll
          for (int e = 0; e < 16; ++e)
            score[x][e] = __builtin_amdgcn_exp2f(__builtin_fmaf(score[x][e], p.scale, -lse[e >> 2][e & 3]));
        const int low = places[buffer][0], high = places[buffer][kStepRows - 1];
        if (key0 + 63 > low || (p.window && key0 <= high - p.window)) {
#pragma unroll
          for (int x = 0; x < 2; ++x) {
            const int key = key0 + 32 * x + (lane & 31);
#pragma unroll
            for (int e = 0; e < 16; ++e) {
              const int at = places[buffer][row_of_register(e, half)];
              score[x][e] = key <= at && (!p.window || key > at - p.window) ? score[x][e] : 0.f;
            }
          }
        }
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          float part[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int e = 0; e < 16; ++e) part[e & 3] += score[x][e];
          total[x] += (part[0] + part[1]) + (part[2] + part[3]);
        }
        if (i + 1 < count) store_rows(buffer ^ 1);
      }
#pragma unroll
      for (int x = 0; x < 2; ++x) total[x] += other_half(total[x]);
      const float mine = half ? total[1] : total[0];
      const bool here = half ? held[1] : held[0];
      if (count == tile_count) {
        const int key = key0 + lane;
        if (here) {
          float* const to = weight_of(p, half ? page[1] : page[0], key, s.head);
          *to = (key < s.context ? *to : 0.f) + mine;
        }
      } else {
        const int begins = before == 0;
        p.partial[(2 * (int64_t)s.worker + begins) * kTile + 64 * wave + lane] = mine;
        if (begins && threadIdx.x == 0) {
          record->worker = s.worker, record->head = s.head, record->request = s.request, record->tile = s.tile;
          record->others = (int)quotient(rest + s.each - 1, s.each);
        }
      }
    }
    s.left -= units;
    if (s.left <= 0) break;
    next_item(p, &s, r.tiles);
  }
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

// Few rows (at most 32 of a request, decoding): a wave holds them and its keys go by, 32 at a time, straight from memory into
// registers. Bound by memory.
template <int D>
__global__ __launch_bounds__(64) void key_weights_few(WeightArgs p) {
  const int lane = threadIdx.x, half = lane >> 5;
  Span s;
  if (!find_span<FewTiles, 1>(p, &s)) return;
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
      bf16x8 q[D / 16];
#pragma unroll
      for (int t = 0; t < D / 16; ++t) q[t] = __builtin_bit_cast(bf16x8, *reinterpret_cast<const u32x4*>(from + 16 * t));
      const float mine = lane < rows ? p.lse[(start + token) * ((int64_t)p.group * p.kv_heads) + head] * kLog2E : INFINITY;
      float lse[16];
      int32_t places[16];
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        lse[e] = __shfl(mine, row_of_register(e, half));
        places[e] = s.context + __shfl(token, row_of_register(e, half));
      }
      const int low = s.context, high = s.context + s.fresh - 1;
      const int key_first = (r.first + before) * FewTiles::kKeys;
      struct Ahead {
        Keys<D> k;
        int page;
        bool held;
        float weight;
      };
      auto fetch = [&](int i, Ahead& a) __attribute__((always_inline)) {
        const int key = key_first + i * FewTiles::kKeys + (lane & 31), at = min(key, length - 1);
        a.held = find_key(p, table, key, length, &a.page);
        load_keys<D>(p, a.k, a.page, at, s.head);
        a.weight = *weight_of(p, a.page, at, s.head);
      };
      auto add = [&](int i, const Ahead& a) __attribute__((always_inline)) {
        const int key0 = key_first + i * FewTiles::kKeys, key = key0 + (lane & 31);
        f32x16 score;
#pragma unroll
        for (int e = 0; e < 16; ++e) score[e] = 0.f;
#pragma unroll
        for (int t = 0; t < D / 16; ++t) score = __builtin_amdgcn_mfma_f32_32x32x16_bf16(q[t], a.k.k[t], score, 0, 0, 0);
        const bool masked = key0 + FewTiles::kKeys - 1 > low || (p.window && key0 <= high - p.window);
        float sum = 0.f;
#pragma unroll
        for (int e = 0; e < 16; e += 4)
          if (2 * e < rows) {  // (uniform: registers of rows that are there)
#pragma unroll
            for (int j = e; j < e + 4; ++j) {
              float w = __builtin_amdgcn_exp2f(__builtin_fmaf(score[j], p.scale, -lse[j]));
              if (masked) w = key <= places[j] && (!p.window || key > places[j] - p.window) ? w : 0.f;
              sum += w;
            }
          }
        sum += other_half(sum);
        if (!half && a.held) *weight_of(p, a.page, key, s.head) = (key < s.context ? a.weight : 0.f) + sum;
      };
      Ahead a, b;
      fetch(0, a);
      for (int i = 0; i < count; i += 2) {
        if (i + 1 < count) fetch(i + 1, b);
        add(i, a);
        if (i + 2 < count) fetch(i + 2, a);
        if (i + 1 < count) add(i + 1, b);
      }
    }
    s.left -= units;
    if (s.left <= 0) break;
    next_item(p, &s, r.tiles);
  }
}

// Workgroups of a launch, a multiple of the 8 XCDs: as many as a CU holds.
int workgroups(int cus, bool few) { return ((few ? 8 : 2) * cus + 7) / 8 * 8; }

int64_t workspace_of(int cus) { return workgroups(cus, false) * (int64_t)(sizeof(WeightRecord) + 2 * 4 * kTile); }

template <int D>
int launch_weights(const WeightArgs& p, bool few, unsigned blocks, hipStream_t stream) {
  hipLaunchKernelGGL(few ? key_weights_few<D> : key_weights_many<D>, dim3(blocks), dim3(few ? 64 : 256), 0, stream, p);
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
  if ((uintptr_t)lse % 4 || (uintptr_t)key_weights % 16) return fail(SMX_ERR_INVALID, "misaligned lse or key_weights");
  const Runs to{key_weights, 2 * (int64_t)cache->num_pages * cache->kv_heads * cache->page_size, {{1, 0}, {1, 0}, {1, 0}}};
  const Runs sums{lse, 2 * (int64_t)step->tokens * q->heads, {{1, 0}, {1, 0}, {1, 0}}};
  if (meet(to, cache_runs(*cache, cache->k)) || meet(to, head_runs(*q, step->tokens, cache->head_dim)) || meet(to, sums))
    return fail(SMX_ERR_INVALID, "key_weights must share no memory with the keys, the queries and lse");
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
  const int blocks = workgroups(cus, few);
  p.min_span = few ? 2 : kItem + 4;
  p.scale = scale * kLog2E;
  p.per_workgroup = 1. / blocks;
  p.records = (WeightRecord*)workspace;
  p.partial = (float*)((char*)workspace + blocks * sizeof(WeightRecord));
  return cache->head_dim == 128 ? launch_weights<128>(p, few, (unsigned)blocks, (hipStream_t)stream)
                                : launch_weights<64>(p, few, (unsigned)blocks, (hipStream_t)stream);
}

}  // extern "C"
