// Attention of new tokens over a paged key/value cache (smx_paged_attention):
// requests of ragged lengths, grouped query heads, causal, optionally within a
// sliding window.
//
// Mathematics. For a request with c tokens before the step and n new ones, new
// token i stands at position p = c + i and sees the keys j with p - window < j <= p.
// out_i = sum_j e^(s_j - m) v_j / sum_j e^(s_j - m), s_j = scale q_i . k_j,
// m = max_j s_j, in one pass over the keys with a running maximum and sum (FP32). The
// exponentials are powers of two (scale carries log2 e) and are rounded to bf16 for the
// product with the values; their sum is taken before that rounding.
//
// Rows. The g query heads of a key/value head share its keys: a tile holds
// whole tokens, row r of it being token r / g, head r % g.
//
// Matrix products (v_mfma_f32_32x32x16_bf16, both transposed): S^T = K Q^T gives
// lane l the scores of row l % 32, so that maxima and sums need one exchange
// between lanes l and l ^ 32; O^T = V^T P^T takes P^T as the scores' own registers:
// the sum over keys may run in any order, and the order in which the lanes hold the
// scores (register i of half h: key 8 (i / 4) + 4 h + i % 4) is the one in which the
// transposing LDS reads hand out V^T.
//
// Work. The key tiles of all (key/value head, request, row tile) items, one behind
// the other, are cut into equal spans, one per workgroup: decode steps and long
// prompts, alone or mixed, fill the chip alike. An item cut by a span's end leaves
// partial sums in the workspace that paged_join adds up. Counts of tiles have closed
// forms, so every workgroup finds its span by itself, from the lengths on the device.
#include <cfloat>

#include "kernel_packed.hpp"
#include "launch.hpp"
#include "paged_spans.hpp"

namespace smx {

namespace {

typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));

struct AttentionArgs {
  const uint16_t* q;
  uint16_t* out;
  int64_t q_token, q_head, out_token, out_head;
  const uint16_t *k, *v;
  int64_t page_stride, slot_stride, head_stride;
  const int32_t* tables;
  int64_t table_stride;
  const int32_t *starts, *rows, *context, *positions;
  int32_t requests, tokens, group, kv_heads, page_shift, num_pages, window, tile_tokens, zero_rows, min_span;
  float scale;      // times log2 e
  float per_group;       // 1 / group
  double per_workgroup;  // 1 / workgroups
  float* partial;
  int32_t* records;
  float* lse;  // [tokens, heads] or null: the logarithm of each row's sum of exponentials
};

// What paged_join needs to know of an item that workgroup w begins and others
// finish: its place and the number of those others (0: no such item).
struct Record {
  int32_t others, worker, head, request, tile, unused[3];
};

// a / b for a < 2^24, by the reciprocal (the integer division is ten times as long).
__device__ __forceinline__ uint32_t small_quotient(uint32_t a, uint32_t b) {
  uint32_t q = (uint32_t)((float)a * __builtin_amdgcn_rcpf((float)b));
  if (q * b > a) --q;
  if ((q + 1) * b <= a) ++q;
  return q;
}

// sum_{i < n} floor((a i + b) / kM), for 0 <= a, b and n a + b < 2^32 once a, b < kM, a power of two.
template <int kM>
__device__ __forceinline__ int64_t floor_sum(uint32_t n, uint32_t a, uint32_t b) {
  int64_t sum = (int64_t)n * (n - 1) / 2 * (a / kM) + (int64_t)n * (b / kM);
  a %= kM, b %= kM;
  uint32_t m = kM, top = a * n + b;
  // the steps of the Euclidean algorithm on (m, a), with a, b < m <= kM
  while (top >= m) {
    const uint32_t old = m, times = top / m;
    n = times, b = top - times * m;
    m = a, a = old;
    uint32_t q = small_quotient(a, m);
    sum += (int64_t)n * (n - 1) / 2 * q, a -= q * m;
    q = small_quotient(b, m);
    sum += (int64_t)n * q, b -= q * m;
    top = a * n + b;
  }
  return sum;
}

// The row tiles of one request and the key tiles (of kKeys keys) that each sees. An item (one of
// them) counts kItem units of work before its key tiles, for its start and end: queries to load,
// the first keys to wait for, the result to store.
template <int kKeys, int kItem>
struct Request {
  int32_t context, fresh, per_tile, window, tiles;

  __device__ Request(const AttentionArgs& p, int32_t context_, int32_t fresh_)
      : context(context_), fresh(fresh_), per_tile(p.tile_tokens), window(p.window) {
    tiles = (fresh + per_tile - 1) / per_tile;
  }
  // The request that a whole wave works on: its lengths in scalar registers, on which the
  // page buffers' descriptors depend.
  __device__ static Request uniform(const AttentionArgs& p, int32_t context_, int32_t fresh_) {
    Request r(p, context_, fresh_);
    r.tiles = __builtin_amdgcn_readfirstlane(r.tiles);
    return r;
  }
  __device__ int first(int t) const {
    return window ? max(0, context + t * per_tile - window + 1) / kKeys : 0;
  }
  __device__ int last(int t) const { return (context + min(fresh, (t + 1) * per_tile) + kKeys - 1) / kKeys; }
  __device__ int count(int t) const { return last(t) - first(t); }
  // Units of the row tiles before t < tiles.
  __device__ int64_t before(int t) const {
    if (!t) return 0;
    int64_t sum = (int64_t)t * kItem + floor_sum<kKeys>(t, per_tile, context + per_tile + kKeys - 1);
    if (window) {
      const int x = context - window + 1;  // first(s) = max(0, x + s per_tile) / kKeys
      const int skip = x >= 0 ? 0 : (-x + per_tile - 1) / per_tile;
      if (skip < t) sum -= floor_sum<kKeys>(t - skip, per_tile, x + skip * per_tile);
    }
    return sum;
  }
  __device__ int64_t all() const { return fresh > 0 ? before(tiles - 1) + kItem + count(tiles - 1) : 0; }
};

// The span's part of one item: its first step (key tile), its steps and units.
template <int kKeys, int kItem>
struct Part {
  Request<kKeys, kItem> r;
  int head, request, tile;
  int from, count, tile_count;  // steps of the part, and of the whole item
  int units, rest;              // of the part; of the item behind it
  int begins;                   // 1: no span before has steps of the item

  __device__ __forceinline__ Part(const AttentionArgs& p, const Span& s)
      : r(Request<kKeys, kItem>::uniform(p, s.context, s.fresh)), head(s.head), request(s.request), tile(s.tile) {
    tile_count = r.count(tile);
    units = (int)min((int64_t)(tile_count + kItem - s.skip), s.left);
    rest = tile_count + kItem - s.skip - units;
    const int before = max(0, s.skip - kItem), upto = max(0, s.skip + units - kItem);
    from = r.first(tile) + before, count = upto - before, begins = __builtin_amdgcn_readfirstlane(before == 0);
  }
};

// Row r of a tile belongs to its token r / group; exact for rows below 2^12.
__device__ __forceinline__ int row_token(int row, const AttentionArgs& p) {
  return (int)(((float)row + 0.5f) * p.per_group);
}

// Rows that belong to no request are zeroed behind the work.
template <int D, int kThreads>
__device__ __forceinline__ void clear_rows(const AttentionArgs& p) {
  if (!p.zero_rows) return;
  const int chunks = p.group * p.kv_heads * (D / 8);
  for (int64_t row = blockIdx.x; row < p.tokens; row += gridDim.x)
    if (p.positions[row] < 0)
      for (int c = threadIdx.x; c < chunks; c += kThreads)
        *reinterpret_cast<u32x4*>(p.out + row * p.out_token + c / (D / 8) * p.out_head + c % (D / 8) * 8) =
            u32x4{0, 0, 0, 0};
}

// LDS tiles of keys and values: rows of D bf16. Keys are stored with their 16-byte
// chunks, values with their 32-byte pairs of chunks, XORed with bits of the row, so
// that neither reads (a wave's 32 rows of one chunk; the transposing reads' 4 rows of one pair)
// fall on the same banks. The DMA stores lane l's 16 bytes at 16 l, so the
// lane fetches the chunk that belongs there.
template <int D>
struct Tile {
  static constexpr int kRow = 2 * D, kChunks = D / 8, kDmaRows = 64 / kChunks;  // rows per DMA
  __device__ static int key_chunk(int chunk, int row) { return chunk ^ (row & (kChunks - 1)); }
  __device__ static int value_chunk(int chunk, int row) {
    return chunk ^ (2 * ((D == 128 ? row : row >> 1) & (kChunks / 2 - 1)));
  }
};

// Lane offsets, within eight rows of a page, of the DMAs that bring kRows rows of keys
// and of values into LDS: row and chunk.
template <int D, int kRows>
struct Lanes {
  using T = Tile<D>;
  static constexpr int kDmas = kRows / T::kDmaRows, kPer8 = 8 / T::kDmaRows;
  uint32_t key[kDmas], value[kDmas];

  __device__ explicit Lanes(int64_t slot_stride) {
    const int in = (threadIdx.x & 63) / T::kChunks, chunk = (threadIdx.x & 63) % T::kChunks;
#pragma unroll
    for (int i = 0; i < kDmas; ++i) {
      const int row = i * T::kDmaRows + in;  // the wave's first row is a multiple of 16
      const uint32_t at = (uint32_t)(i % kPer8 * T::kDmaRows + in) * (uint32_t)slot_stride * 2;
      key[i] = at + 16 * T::key_chunk(chunk, row);
      value[i] = at + 16 * T::value_chunk(chunk, row);
    }
  }

  // The DMAs of the eight rows of group g, whose first lies at byte `from` of the cache.
  __device__ __forceinline__ void fetch_group(const AttentionArgs& p, int g, int64_t from, uint32_t bytes, uint8_t* keys,
                                              uint8_t* values) const {
    const auto from_k = packed::panel_rsrc(reinterpret_cast<const uint8_t*>(p.k) + from, bytes);
    const auto from_v = packed::panel_rsrc(reinterpret_cast<const uint8_t*>(p.v) + from, bytes);
#pragma unroll
    for (int i = g * kPer8; i < (g + 1) * kPer8; ++i) {
      packed::dma_frag(from_k, key[i], 0, keys + i * T::kDmaRows * T::kRow);
      packed::dma_frag(from_v, value[i], 0, values + i * T::kDmaRows * T::kRow);
    }
  }

  // Starts the DMAs of rows key0 .. key0 + kRows - 1 of a head to LDS. A page holds whole
  // groups of eight rows: each group is one buffer, whose rows behind `length`, and
  // all of whose rows if its page is not in the cache, read as zeros. Lane
  // lane0 + r of `pages` holds row r's page.
  // kByLane: every lane works out its row's address, and a group reads its lane's. That is a third of
  // the instructions, for a wave alone on its SIMD (1000 keys, one row: 13.4 us, else 14.4); where waves share
  // it, scalar instructions run beside the others' vector ones (8192 rows: 1220 us, by lane 1275).
  template <bool kByLane>
  __device__ __forceinline__ void fetch(const AttentionArgs& p, int head, int key0, int length, int pages, int lane0,
                                        uint8_t* keys, uint8_t* values) const {
    if constexpr (kByLane) {
      const int row = key0 - lane0 + (int)(threadIdx.x & 63);
      const bool held = (uint32_t)pages < (uint32_t)p.num_pages;
      const uint64_t at = 2 * ((uint64_t)(uint32_t)(held ? pages : 0) * (uint32_t)p.page_stride +
                               (uint64_t)(uint32_t)(row & ((1 << p.page_shift) - 1)) * (uint32_t)p.slot_stride +
                               (uint64_t)(uint32_t)head * (uint32_t)p.head_stride);
      const uint32_t bytes = held ? (uint32_t)max(0, min(8, length - row)) * (uint32_t)p.slot_stride * 2 : 0u;
#pragma unroll
      for (int g = 0; g < kRows / 8; ++g)
        fetch_group(p, g, lane_value((int64_t)at, lane0 + 8 * g), __builtin_amdgcn_readlane((int)bytes, lane0 + 8 * g), keys, values);
    } else {
#pragma unroll
      for (int g = 0; g < kRows / 8; ++g) {
        const int first = key0 + 8 * g, page = __builtin_amdgcn_readlane(pages, lane0 + 8 * g);
        const bool held = (uint32_t)page < (uint32_t)p.num_pages;
        const int64_t at = (int64_t)(held ? page : 0) * p.page_stride + (int64_t)(first & ((1 << p.page_shift) - 1)) * p.slot_stride +
                           head * p.head_stride;
        // (the clamp is a vector instruction; the descriptor has to be scalar, or every lane's
        // is compared in a loop around the DMA)
        const int rows = __builtin_amdgcn_readfirstlane(held ? max(0, min(8, length - first)) : 0);
        fetch_group(p, g, 2 * at, (uint32_t)rows * (uint32_t)p.slot_stride * 2, keys, values);
      }
    }
  }
};

// V^T fragments of 32 keys (two MFMA steps): for each block of 32 columns, lane l's 8 values of
// column l % 32 by two transposing LDS reads (4 keys each; lane group l / 16 reads 4
// rows of 16 columns). `at`: LDS address of the block's first read. Written as one asm
// block with its wait: before the builtin of this read the compiler waits for every
// DMA in flight, the next step's too.
template <int D, int kOffset>
__device__ __forceinline__ void read_values(bf16x8 (&v)[2][D / 32], const uint32_t (&at)[D / 32]) {
  constexpr int kRow = 2 * D;
  u32x2 r[2][D / 32][2];
  if constexpr (D == 128) {
    asm volatile(
        "ds_read_b64_tr_b16 %0, %16 offset:%20\n\t"
        "ds_read_b64_tr_b16 %1, %16 offset:%21\n\t"
        "ds_read_b64_tr_b16 %2, %17 offset:%20\n\t"
        "ds_read_b64_tr_b16 %3, %17 offset:%21\n\t"
        "ds_read_b64_tr_b16 %4, %18 offset:%20\n\t"
        "ds_read_b64_tr_b16 %5, %18 offset:%21\n\t"
        "ds_read_b64_tr_b16 %6, %19 offset:%20\n\t"
        "ds_read_b64_tr_b16 %7, %19 offset:%21\n\t"
        "ds_read_b64_tr_b16 %8, %16 offset:%22\n\t"
        "ds_read_b64_tr_b16 %9, %16 offset:%23\n\t"
        "ds_read_b64_tr_b16 %10, %17 offset:%22\n\t"
        "ds_read_b64_tr_b16 %11, %17 offset:%23\n\t"
        "ds_read_b64_tr_b16 %12, %18 offset:%22\n\t"
        "ds_read_b64_tr_b16 %13, %18 offset:%23\n\t"
        "ds_read_b64_tr_b16 %14, %19 offset:%22\n\t"
        "ds_read_b64_tr_b16 %15, %19 offset:%23\n\t"
        "s_waitcnt lgkmcnt(0)"
        : "=&v"(r[0][0][0]), "=&v"(r[0][0][1]), "=&v"(r[0][1][0]), "=&v"(r[0][1][1]), "=&v"(r[0][2][0]),
          "=&v"(r[0][2][1]), "=&v"(r[0][3][0]), "=&v"(r[0][3][1]), "=&v"(r[1][0][0]), "=&v"(r[1][0][1]),
          "=&v"(r[1][1][0]), "=&v"(r[1][1][1]), "=&v"(r[1][2][0]), "=&v"(r[1][2][1]), "=&v"(r[1][3][0]),
          "=&v"(r[1][3][1])
        : "v"(at[0]), "v"(at[1]), "v"(at[2]), "v"(at[3]), "n"(kOffset), "n"(kOffset + 8 * kRow), "n"(kOffset + 16 * kRow),
          "n"(kOffset + 24 * kRow)
        : "memory");
  } else {
    asm volatile(
        "ds_read_b64_tr_b16 %0, %8 offset:%10\n\t"
        "ds_read_b64_tr_b16 %1, %8 offset:%11\n\t"
        "ds_read_b64_tr_b16 %2, %9 offset:%10\n\t"
        "ds_read_b64_tr_b16 %3, %9 offset:%11\n\t"
        "ds_read_b64_tr_b16 %4, %8 offset:%12\n\t"
        "ds_read_b64_tr_b16 %5, %8 offset:%13\n\t"
        "ds_read_b64_tr_b16 %6, %9 offset:%12\n\t"
        "ds_read_b64_tr_b16 %7, %9 offset:%13\n\t"
        "s_waitcnt lgkmcnt(0)"
        : "=&v"(r[0][0][0]), "=&v"(r[0][0][1]), "=&v"(r[0][1][0]), "=&v"(r[0][1][1]), "=&v"(r[1][0][0]),
          "=&v"(r[1][0][1]), "=&v"(r[1][1][0]), "=&v"(r[1][1][1])
        : "v"(at[0]), "v"(at[1]), "n"(kOffset), "n"(kOffset + 8 * kRow), "n"(kOffset + 16 * kRow), "n"(kOffset + 24 * kRow)
        : "memory");
  }
#pragma unroll
  for (int t = 0; t < 2; ++t)
#pragma unroll
    for (int x = 0; x < D / 32; ++x)
      v[t][x] = __builtin_bit_cast(bf16x8, u32x4{r[t][x][0][0], r[t][x][0][1], r[t][x][1][0], r[t][x][1][1]});
}

__device__ __forceinline__ uint32_t lds_address(const uint8_t* p) {
  return (uint32_t)(uintptr_t)(__attribute__((address_space(3))) const uint8_t*)p;
}

// Running softmax and output of a wave's 32 rows: lane l holds row l % 32; register e
// of block x is column 32 x + 8 (e / 4) + 4 (l / 32) + e % 4 of the output.
template <int D>
struct Rows {
  f32x16 o[D / 32];
  float top, sum;  // the reference maximum (scores times scale; -inf: no key was seen); this lane's share of the sum

  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int x = 0; x < D / 32; ++x)
#pragma unroll
      for (int e = 0; e < 16; ++e) o[x][e] = 0.f;
    top = -INFINITY, sum = 0.f;
  }
};

typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));

// Whether a step's values hold an infinity or a NaN, in any lane.
template <int kBlocks, int kColumns>
__device__ __forceinline__ bool any_not_finite(const bf16x8 (&v)[kBlocks][2][kColumns]) {
  u16x2 most = {0, 0};
#pragma unroll
  for (int b = 0; b < kBlocks; ++b)
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int x = 0; x < kColumns; ++x) {
        const u32x4 words = __builtin_bit_cast(u32x4, v[b][h][x]);
#pragma unroll
        for (int i = 0; i < 4; ++i)
          most = __builtin_elementwise_max(most, __builtin_bit_cast(u16x2, words[i] & 0x7fff7fffu));
      }
  return __any(max(most[0], most[1]) >= 0x7f80);
}

// A step that masks keys and whose values are not all finite: a product alone would give 0 * inf = NaN
// to the rows that do not see them. Every +inf and NaN (sign 0), every -inf and NaN (sign 1) that a row
// sees, however small its weight, adds a product beyond FP32's range to its column, which is that infinity
// (both: NaN), and the values themselves become zero. The row sees the step's keys after `oldest` up to `newest`
// (both less 4 half) whose bit in `held` (shifted so too) is set.
template <int D, int kBlocks>
__device__ __forceinline__ void add_not_finite(f32x16 (&o)[D / 32], bf16x8 (&v)[kBlocks][2][D / 32], int oldest, int newest,
                                               uint64_t held) {
  // two values a register; 0 or 1 for no and yes (asm: constants loaded here, not held by the whole kernel)
  uint32_t weight = 0x4380u, ones = 0x10001u, largest[2] = {0x7f7f7f7fu, 0xff7fff7fu};
  asm volatile("" : "+s"(weight), "+s"(ones), "+s"(largest[0]), "+s"(largest[1]));
  const uint32_t finite = largest[0];
  const u16x2 one = __builtin_bit_cast(u16x2, ones), most = __builtin_bit_cast(u16x2, finite);
#pragma unroll
  for (int t = 0; t < 2 * kBlocks; ++t) {
    u32x4 large;  // 2^8 for every key that the row sees
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      large[i] = 0;
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const int e = 8 * (t % 2) + 2 * i + j, key = 32 * (t / 2) + 8 * (e >> 2) + (e & 3);
        large[i] |= key <= newest && key > oldest && ((held >> key) & 1) ? weight << 16 * j : 0;
      }
    }
#pragma unroll
    for (int x = 0; x < D / 32; ++x) {
      u32x4 words = __builtin_bit_cast(u32x4, v[t / 2][t % 2][x]), bad;
#pragma unroll
      for (int sign = 0; sign < 2; ++sign) {
        asm volatile("" : "+v"(words));  // nothing shared with any_not_finite and between signs, for want of registers
        const uint32_t value = largest[sign];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          // (copied before it is reinterpreted: a bit cast of a vector's element takes its first)
          const uint32_t two = words[i], sizes = two & 0x7fff7fffu;
          const u16x2 beyond = __builtin_elementwise_sub_sat(__builtin_bit_cast(u16x2, sizes), most);  // 1: inf, more: NaN
          u16x2 side = __builtin_bit_cast(u16x2, two) >> (uint16_t)15;
          if (!sign) side = one - side;
          const u16x2 hit = __builtin_elementwise_min(beyond >> (uint16_t)1 | side, one) * __builtin_elementwise_min(beyond, one);
          bad[i] = __builtin_bit_cast(uint32_t, hit * __builtin_bit_cast(u16x2, value));
        }
        o[x] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, bad), __builtin_bit_cast(bf16x8, large),
                                                       o[x], 0, 0, 0);
        __builtin_amdgcn_sched_barrier(0);
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        uint32_t two = words[i];
        asm volatile("" : "+v"(two));
        const uint32_t sizes = two & 0x7fff7fffu;
        const u16x2 beyond = __builtin_elementwise_sub_sat(__builtin_bit_cast(u16x2, sizes), most);
        words[i] = __builtin_bit_cast(uint32_t, __builtin_bit_cast(u16x2, two) * (one - __builtin_elementwise_min(beyond, one)));
      }
      v[t / 2][t % 2][x] = __builtin_bit_cast(bf16x8, words);
      __builtin_amdgcn_sched_barrier(0);
    }
  }
}

// One step: the wave's 32 rows against 32 kBlocks keys in LDS. The maximum that the exponentials are taken against
// moves only once it is exceeded by 2^8, so that most steps rescale nothing; sums
// stay below 2^8 times their number of keys.
template <int D, int kBlocks>
__device__ __forceinline__ void attend(Rows<D>& r, const bf16x8 (&q)[D / 16], const uint8_t* keys, const uint8_t* values,
                                       float scale, bool masked, int rel, int window, uint64_t held) {
  using T = Tile<D>;
  const int lane = threadIdx.x & 63, half = lane >> 5;
  f32x16 s[kBlocks];
#pragma unroll
  for (int x = 0; x < kBlocks; ++x)
#pragma unroll
    for (int e = 0; e < 16; ++e) s[x][e] = 0.f;
  // All of the step's keys on their way before the first MFMA (one at a time they cost its latency each).
  bf16x8 k[D / 16][kBlocks];
#pragma unroll
  for (int t = 0; t < D / 16; ++t)
#pragma unroll
    for (int x = 0; x < kBlocks; ++x)
      k[t][x] = packed::ld_frag(keys + (32 * x + (lane & 31)) * T::kRow + 16 * T::key_chunk(2 * t + half, lane & 31));
  __builtin_amdgcn_sched_barrier(0);
#pragma unroll
  for (int t = 0; t < D / 16; ++t)
#pragma unroll
    for (int x = 0; x < kBlocks; ++x) s[x] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(k[t][x], q[t], s[x], 0, 0, 0);
  __builtin_amdgcn_sched_barrier(0);
  // The values too, behind the MFMAs: lane group lane / 16 reads rows 4 half .. + 3 of 16
  // columns; the lane's row and piece there.
  const int row = 4 * half + ((lane & 15) >> 2), piece = lane & 3, side = (lane >> 4) & 1;
  uint32_t at[D / 32];
#pragma unroll
  for (int x = 0; x < D / 32; ++x)
    at[x] = lds_address(values) + row * T::kRow + 16 * T::value_chunk(2 * (2 * x + side), row) + 8 * piece;
  bf16x8 v[kBlocks][2][D / 32];
  read_values<D, 0>(v[0], at);
  if constexpr (kBlocks == 2) read_values<D, 32 * T::kRow>(v[kBlocks - 1], at);
  float lowest = -FLT_MAX;
  if (masked) {
    // key - first key of the step = 32 x + 8 (e / 4) + 4 half + e % 4; `rel` is the
    // row's position less the step's first key
    const int mine = rel - 4 * half;
#pragma unroll
    for (int x = 0; x < kBlocks; ++x)
#pragma unroll
      for (int e = 0; e < 16; ++e) s[x][e] = 32 * x + 8 * (e >> 2) + (e & 3) <= mine ? s[x][e] : -INFINITY;
    if (window || held != (kBlocks == 2 ? ~0ull : 0xffffffffull)) {
      const int oldest = window ? mine - window : -(1 << 30);
      const uint64_t bits = held >> (4 * half);
#pragma unroll
      for (int x = 0; x < kBlocks; ++x)
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          const int key = 32 * x + 8 * (e >> 2) + (e & 3);
          s[x][e] = key > oldest && ((bits >> key) & 1) ? s[x][e] : -INFINITY;
        }
    }
    // the bits of the keys that the row sees
    const int newest = min(rel, 32 * kBlocks - 1), before = window ? min(rel - window, 63) : -1;
    uint64_t sees = newest >= 0 ? held & ~0ull >> (63 - newest) : 0;
    if (before >= 0) sees &= ~(~0ull >> (63 - before));
    if (!sees) lowest = -INFINITY;
  }
  float top = s[0][0];
#pragma unroll
  for (int x = 0; x < kBlocks; ++x)
#pragma unroll
    for (int e = 0; e < 16; ++e) top = fmaxf(top, s[x][e]);
  // (a maximum of -inf is left to rows that see no key)
  top = fmaxf(fmaxf(top, other_half(top)) * scale, lowest);
  if (__any(top > r.top + 8.f)) {
    const float next = fmaxf(r.top, top);
    const float factor = next == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(r.top - next);
    r.top = next;
    r.sum *= factor;
#pragma unroll
    for (int x = 0; x < D / 32; ++x)
#pragma unroll
      for (int e = 0; e < 16; ++e) r.o[x][e] *= factor;
  }
  const float base = r.top == -INFINITY ? 0.f : r.top;
  bf16x8 w[2 * kBlocks];
#pragma unroll
  for (int x = 0; x < kBlocks; ++x) {
#pragma unroll
    for (int e = 0; e < 16; ++e) {
      s[x][e] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[x][e], scale, -base));
      r.sum += s[x][e];
    }
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      u32x4 b;
#pragma unroll
      for (int i = 0; i < 4; ++i) b[i] = pack_bf16(s[x][8 * h + 2 * i], s[x][8 * h + 2 * i + 1]);
      w[2 * x + h] = __builtin_bit_cast(bf16x8, b);
    }
  }
  if (masked && any_not_finite(v))
    add_not_finite<D, kBlocks>(r.o, v, window ? rel - 4 * half - window : -(1 << 30), rel - 4 * half, held >> (4 * half));
#pragma unroll
  for (int t = 0; t < 2 * kBlocks; ++t)
#pragma unroll
    for (int x = 0; x < D / 32; ++x)
      r.o[x] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(v[t / 2][t % 2][x], w[t], r.o[x], 0, 0, 0);
}

// A tile's output or partial sums. kWaves row groups of 32 in a tile. Partial layout per
// worker and slot: D / 8 chunks of [256] float4, then [256] tops and [256] sums.
template <int D>
constexpr int kPartialFloats = 256 * (D / 2 + 2);
// The same of paged_attend_few: [32][D] values, [32] tops, [32] sums.
template <int D>
constexpr int kFewPartialFloats = 32 * (D + 2);

// One block of 32 columns of 32 rows to memory, `to` the lane's row there: lane l of half h holds columns
// 8 (e / 4) + 4 h ..; two lanes exchange halves so that each stores 16 bytes.
__device__ __forceinline__ void store_block(uint16_t* to, const f32x16& o, float inverse, bool valid, int half) {
#pragma unroll
  for (int e = 0; e < 16; e += 8) {
    // columns 4 h .. of groups e / 4 (mine if half 0) and e / 4 + 1 (mine if half 1)
    const uint32_t a0 = pack_bf16(o[e] * inverse, o[e + 1] * inverse);
    const uint32_t a1 = pack_bf16(o[e + 2] * inverse, o[e + 3] * inverse);
    const uint32_t b0 = pack_bf16(o[e + 4] * inverse, o[e + 5] * inverse);
    const uint32_t b1 = pack_bf16(o[e + 6] * inverse, o[e + 7] * inverse);
    // swap: a's upper half with b's lower half
    const auto r0 = __builtin_amdgcn_permlane32_swap(a0, b0, false, false);
    const auto r1 = __builtin_amdgcn_permlane32_swap(a1, b1, false, false);
    const u32x4 v = {r0[0], r1[0], r0[1], r1[1]};
    if (valid) *reinterpret_cast<u32x4*>(to + 8 * ((e >> 2) + half)) = v;
  }
}

template <int D>
__device__ __forceinline__ void store_rows(const AttentionArgs& p, const f32x16 (&o)[D / 32], float inverse, bool valid,
                                           int64_t token, int head) {
  int thread = threadIdx.x;
  asm volatile("" : "+v"(thread));  // (offsets are made here, not held by the whole kernel)
  uint16_t* const to = p.out + token * p.out_token + head * p.out_head;
#pragma unroll
  for (int x = 0; x < D / 32; ++x) store_block(to + 32 * x, o[x], inverse, valid, thread >> 5 & 1);
}

// What a row's values are multiplied with. Its largest weight is 1, so that a sum is zero only without one: a row
// that sees no key (its maximum is still -inf) is zero, and one all of whose scores are -inf is NaN.
__device__ __forceinline__ float inverse_of(float sum, float top) {
  return sum > 0.f ? 1.f / sum : sum == 0.f && top > -INFINITY ? NAN : sum;
}

// The logarithm of a row's sum of exponentials; -inf where there is none.
__device__ __forceinline__ void store_lse(const AttentionArgs& p, int64_t token, int head, float top, float sum) {
  constexpr float kLn2 = 0.693147180559945309f;
  p.lse[token * ((int64_t)p.group * p.kv_heads) + head] = sum > 0.f || sum != sum ? (top + __builtin_amdgcn_logf(sum)) * kLn2 : -INFINITY;
}

// 128 rows a tile (four waves of 32), 64 keys a step, keys and values double buffered. 2048 tokens of 64 heads on
// 16384 cached ones: 1.30 ms, 0.90 PFLOP/s. Matrix cores, vector units and LDS are each busy 41 to 44% of the time
// (one workgroup a CU: 2.0 ms): two waves a SIMD do not cover each other's way from a step's keys to
// its output, and registers and LDS hold no third. Without the exponentials 9% less, without the
// values' reads nothing. Scores of the next step beside the weights of this one, in the same wave: 1.50 ms (247
// registers); the next step's first keys read before its DMAs are started: 64 registers too many.
template <int D>
__global__ __launch_bounds__(256, 2) void paged_attend(AttentionArgs p) {
  using T = Tile<D>;
  constexpr int kKeys = 64, kItem = 3;
  extern __shared__ __attribute__((aligned(1024))) uint8_t lds[];
  constexpr int kTileBytes = kKeys * T::kRow;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), half = lane >> 5;

  Record* const record = reinterpret_cast<Record*>(p.records) + blockIdx.x;
  if (threadIdx.x == 0) record->others = 0;
  Span s;
  if (!find_span<Request<kKeys, kItem>, 4>(p, &s)) return clear_rows<D, 256>(p);

  const Lanes<D, 16> lanes(p.slot_stride);

  using Part = Part<kKeys, kItem>;
  // lane l's page of a step: that of its key 64 step + l
  auto pages_of = [&](const Part& w, int step) __attribute__((always_inline)) {
    const int key = min(step * kKeys + lane, w.r.context + w.r.fresh - 1);
    return p.tables[w.request * p.table_stride + (key >> p.page_shift)];
  };
  auto fetch = [&](const Part& w, int step, int pages, int buffer) __attribute__((always_inline)) {
    uint8_t* const to = lds + buffer * 2 * kTileBytes + 16 * wave * T::kRow;
    lanes.template fetch<false>(p, w.head, step * kKeys + 16 * wave, w.r.context + w.r.fresh, pages, 16 * wave, to, to + kTileBytes);
  };
  auto held_of = [&](int pages) __attribute__((always_inline)) { return __ballot((uint32_t)pages < (uint32_t)p.num_pages); };
  // this lane's row of an item: its token within the request and its query head
  auto row_of = [&](const Part& w, int* local, int* head) __attribute__((always_inline)) {
    const int rows = min(w.r.per_tile, w.r.fresh - w.tile * w.r.per_tile) * p.group;
    int thread = threadIdx.x;
    asm volatile("" : "+v"(thread));  // (made here, not held by the whole kernel)
    const int row = min((thread >> 1 & ~31) + (thread & 31), rows - 1), token = row_token(row, p);
    *local = w.tile * w.r.per_tile + token, *head = w.head * p.group + row - token * p.group;
    return rows;
  };
  bf16x8 q[D / 16];
  auto load_q = [&](const Part& w) __attribute__((always_inline)) {
    int local, head;
    row_of(w, &local, &head);
    const int64_t token = scalar_at(p.starts, w.request) + local;
    int thread = threadIdx.x;
    asm volatile("" : "+v"(thread));  // (the offset is made here, not held by the whole kernel)
    const uint16_t* const from = p.q + token * p.q_token + head * p.q_head + 8 * (thread >> 5 & 1);
#pragma unroll
    for (int t = 0; t < D / 16; ++t) q[t] = __builtin_bit_cast(bf16x8, *reinterpret_cast<const u32x4*>(from + 16 * t));
  };

  // One stream of steps over all parts: while a step is computed the next one's DMAs are on
  // their way, whichever part it belongs to, and the pages of the one after that are looked up.
  // A part may end before its first step (all of its units lie before them): it is passed over.
  auto next_part = [&]() __attribute__((always_inline)) {
    Part w(p, s);
    while (!w.count && s.left > w.units) {
      s.left -= w.units;
      next_item(p, &s, w.r.tiles);
      w = Part(p, s);
    }
    return w;
  };
  Part part = next_part(), next = part;
  if (part.count) {
    int pages = pages_of(part, part.from);
    uint64_t held = held_of(pages);
    load_q(part);
    fetch(part, part.from, pages, 0);
    if (part.count > 1) pages = pages_of(part, part.from + 1);
    int buffer = 0;
    for (;;) {
      int local, head;
      const int tile_rows = row_of(part, &local, &head);
      const int position = part.r.context + local;
      // positions of the wave's first and last row
      const int low = __builtin_amdgcn_readfirstlane(position), high = __builtin_amdgcn_readlane(position, 31);
      const bool active = 32 * wave < tile_rows;  // rows of its own
      int more = __builtin_amdgcn_readfirstlane(s.left > part.units);  // another part follows
      Rows<D> o;
      o.clear();
      for (int i = 0; i < part.count; ++i) {
        const int step = part.from + i;
        packed::stage_barrier<0>();
        const uint64_t now = held;
        const bool ends = i + 1 == part.count;
        if (more && (ends ? part.count == 1 : i + 2 == part.count)) {
          s.left -= part.units;
          next_item(p, &s, part.r.tiles);
          next = next_part();
          more = __builtin_amdgcn_readfirstlane(next.count > 0);
          if (more && ends) pages = pages_of(next, next.from);
        }
        if (!ends) {
          held = held_of(pages);
          fetch(part, step + 1, pages, buffer ^ 1);
          if (i + 2 < part.count)
            pages = pages_of(part, step + 2);
          else if (more)
            pages = pages_of(next, next.from);
        } else if (more) {
          held = held_of(pages);
          fetch(next, next.from, pages, buffer ^ 1);
          if (next.count > 1) pages = pages_of(next, next.from + 1);
        }
        const int key0 = step * kKeys;
        if (active && key0 <= high && (!p.window || key0 + kKeys - 1 > low - p.window)) {
          const bool masked = key0 + kKeys - 1 > low || (p.window && key0 <= high - p.window) || now != ~0ull;
          const uint8_t* const at = lds + buffer * 2 * kTileBytes;
          attend<D, 2>(o, q, at, at + kTileBytes, p.scale, masked, position - key0, p.window, now);
        }
        buffer ^= 1;
        // one set of registers for the output whether the step was the wave's or not (else it is copied)
#pragma unroll
        for (int x = 0; x < D / 32; ++x) asm volatile("" : "+v"(o.o[x]));
      }
      if (more) load_q(next);

      const float sum = o.sum + other_half(o.sum);
      if (part.count == part.tile_count) {
        const int64_t token = scalar_at(p.starts, part.request) + local;
        store_rows<D>(p, o.o, inverse_of(sum, o.top), 32 * wave + (lane & 31) < tile_rows, token, head);
        if (p.lse && !half && 32 * wave + (lane & 31) < tile_rows) store_lse(p, token, head, o.top, sum);
      } else {
        float* const to = p.partial + (2 * (int64_t)s.worker + part.begins) * kPartialFloats<D>;
        int thread = threadIdx.x;
        asm volatile("" : "+v"(thread));  // (nor are these addresses)
#pragma unroll
        for (int x = 0; x < D / 32; ++x)
#pragma unroll
          for (int e = 0; e < 4; ++e)
            reinterpret_cast<f32x4*>(to)[(4 * x + e) * 256 + thread] =
                f32x4{o.o[x][4 * e], o.o[x][4 * e + 1], o.o[x][4 * e + 2], o.o[x][4 * e + 3]};
        to[256 * (D / 2) + thread] = o.top;
        to[256 * (D / 2 + 1) + thread] = sum;
        if (part.begins && threadIdx.x == 0) {
          record->worker = s.worker, record->head = part.head, record->request = part.request, record->tile = part.tile;
          // the item goes on in the spans behind this one
          int64_t each = s.each;
          asm volatile("" : "+s"(each));  // (its floating-point form is made here, not held by the whole kernel)
          record->others = (int)quotient(part.rest + each - 1, each);
        }
      }
      if (!more) break;
      part = next;
    }
  }
  clear_rows<D, 256>(p);
}

// Steps of few rows (decoding): a workgroup is one wave with 32 rows a tile, which streams 32
// keys a step through its own two buffers, so that no barrier joins it to others and
// four of them (32 KB of LDS each at head_dim 128) keep up to 128 KB of a CU's reads in
// flight. Rows are few: what bounds it is the cache's bytes: 64 requests, 260,000 cached tokens of 4 KB, 197 us
// and 7 in paged_join_few (5.2 TB/s); four of 131,000 tokens 367 and 9 (5.7). Short caches are
// bound by latency: 1000 tokens 9 us, of which 1.6 pass until the span is found, 1.4 until the first
// loads are on their way, 1.2 in a step.
template <int D>
__global__ __launch_bounds__(64) void paged_attend_few(AttentionArgs p) {
  using T = Tile<D>;
  constexpr int kKeys = 32, kItem = 1, kDmas = kKeys / T::kDmaRows, kTileBytes = kKeys * T::kRow;
  extern __shared__ __attribute__((aligned(1024))) uint8_t lds[];
  const int lane = threadIdx.x, half = lane >> 5;

  Record* const record = reinterpret_cast<Record*>(p.records) + blockIdx.x;
  if (lane == 0) record->others = 0;
  Span s;
  if (!find_span<Request<kKeys, kItem>, 1>(p, &s)) return clear_rows<D, 64>(p);

  const Lanes<D, kKeys> lanes(p.slot_stride);

  while (s.left > 0) {
    const Part<kKeys, kItem> part(p, s);
    const auto& r = part.r;
    const int count = part.count, from = part.from;
    if (!count) {  // all of its units lie before its first step
      s.left -= part.units;
      if (s.left <= 0) break;
      next_item(p, &s, r.tiles);
      continue;
    }
    const int tile_rows = min(r.per_tile, r.fresh - part.tile * r.per_tile) * p.group;
    const int row = min(lane & 31, tile_rows - 1), in = row_token(row, p);
    const int local = part.tile * r.per_tile + in, head = part.head * p.group + row - in * p.group;
    const int64_t token = scalar_at(p.starts, part.request) + local;
    const int position = r.context + local, length = r.context + r.fresh;
    const int low = __builtin_amdgcn_readfirstlane(position), high = __builtin_amdgcn_readlane(position, 31);
    const bool valid = (lane & 31) < tile_rows;
    const int32_t* const table = p.tables + part.request * p.table_stride;

    // lane l's page of a step: that of its key l % 32 of the step
    auto pages_of = [&](int step) __attribute__((always_inline)) {
      return table[min(step * kKeys + (lane & 31), length - 1) >> p.page_shift];
    };
    // Steps past the item's last are fetched as no rows (zeros, no reads), so that the
    // number of operations in flight stays the same.
    auto fetch = [&](int i, int pages) __attribute__((always_inline)) {
      uint8_t* const to = lds + (i & 1) * 2 * kTileBytes;
      lanes.template fetch<true>(p, s.head, (from + i) * kKeys, i < count ? length : 0, pages, 0, to, to + kTileBytes);
    };
    int pages = pages_of(from), next = pages_of(from + 1);
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // the item before: its last fetches and stores
    bf16x8 q[D / 16];
    const uint16_t* const q_row = p.q + token * p.q_token + head * p.q_head + 8 * half;
#pragma unroll
    for (int t = 0; t < D / 16; ++t) q[t] = __builtin_bit_cast(bf16x8, *reinterpret_cast<const u32x4*>(q_row + 16 * t));
    uint32_t held = (uint32_t)__ballot((uint32_t)pages < (uint32_t)p.num_pages);
    // The loop's waits count operations: none of those behind the first fetch may be moved before its end.
    auto in_order = []() __attribute__((always_inline)) {
      asm volatile("" ::: "memory");
      __builtin_amdgcn_sched_barrier(0);
    };
    fetch(0, pages);
    in_order();
    int after = pages_of(from + 2);
    uint32_t next_held = (uint32_t)__ballot((uint32_t)next < (uint32_t)p.num_pages);
    fetch(1, next);
    in_order();

    Rows<D> o;
    o.clear();
    for (int i = 0; i < count; ++i) {
      // all but the page list and the DMAs of the step behind this one
      asm volatile("s_waitcnt vmcnt(%0)" ::"i"(2 * kDmas + 1) : "memory");
      const int key0 = (from + i) * kKeys;
      const bool masked = key0 + kKeys - 1 > low || (p.window && key0 <= high - p.window) || held != ~0u;
      const uint8_t* const at = lds + (i & 1) * 2 * kTileBytes;
      attend<D, 1>(o, q, at, at + kTileBytes, p.scale, masked, position - key0, p.window, held);
      held = next_held;
      next_held = (uint32_t)__ballot((uint32_t)after < (uint32_t)p.num_pages);
      const int now = after;
      after = pages_of(from + i + 3);
      fetch(i + 2, now);
    }

    const float sum = o.sum + other_half(o.sum);
    if (count == part.tile_count) {
      store_rows<D>(p, o.o, inverse_of(sum, o.top), valid, token, head);
      if (p.lse && valid && !half) store_lse(p, token, head, o.top, sum);
    } else {
      float* const to = p.partial + (2 * (int64_t)s.worker + part.begins) * kFewPartialFloats<D>;
      if (valid) {
#pragma unroll
        for (int x = 0; x < D / 32; ++x)
#pragma unroll
          for (int e = 0; e < 4; ++e)
            *reinterpret_cast<f32x4*>(to + row * D + 32 * x + 8 * e + 4 * half) =
                f32x4{o.o[x][4 * e], o.o[x][4 * e + 1], o.o[x][4 * e + 2], o.o[x][4 * e + 3]};
        if (!half) {
          to[32 * D + row] = o.top;
          to[32 * D + 32 + row] = sum;
        }
      }
      if (part.begins && lane == 0) {
        record->worker = s.worker, record->head = part.head, record->request = part.request, record->tile = part.tile;
        record->others = (int)quotient(part.rest + s.each - 1, s.each);
      }
    }
    s.left -= part.units;
    if (s.left <= 0) break;
    next_item(p, &s, r.tiles);
  }
  // no DMA outlives the wave
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  clear_rows<D, 64>(p);
}

// Adds up the partial sums of paged_attend_few: a workgroup per record, a thread per
// row and four columns; threads that are left divide the partial sums among them. Each
// keeps a running maximum, and the parts meet in LDS.
template <int D>
__global__ __launch_bounds__(1024) void paged_join_few(AttentionArgs p) {
  const Record record = reinterpret_cast<const Record*>(p.records)[blockIdx.x];
  if (record.others <= 0) return;
  __shared__ f32x4 values[1024];
  __shared__ float tops[1024], totals[1024];
  const int fresh = p.rows[record.request];
  const int rows = min(p.tile_tokens, fresh - record.tile * p.tile_tokens) * p.group;
  const int items = rows * (D / 4), parts = 1024 / items;  // rows <= 32: at least one part
  const int part = (int)threadIdx.x / items, item = (int)threadIdx.x - part * items;
  const int row = item / (D / 4), column = item % (D / 4) * 4;
  const float* const base = p.partial + 2 * (int64_t)record.worker * kFewPartialFloats<D>;
  constexpr int64_t kWorker = 2 * (int64_t)kFewPartialFloats<D>;
  float top = -INFINITY, total = 0.f;
  f32x4 value = {0.f, 0.f, 0.f, 0.f};
  if (part < parts)
#pragma unroll 4
    for (int i = part; i <= record.others; i += parts) {
      const float* const from = base + i * kWorker + (i == 0 ? kFewPartialFloats<D> : 0);
      const float mine = from[32 * D + row], sum = from[32 * D + 32 + row];
      const f32x4 v = *reinterpret_cast<const f32x4*>(from + row * D + column);
      const float next = fmaxf(top, mine), ref = next == -INFINITY ? 0.f : next;
      const float keep = __builtin_amdgcn_exp2f(top - ref), add = __builtin_amdgcn_exp2f(mine - ref);
      top = next;
      total = total * keep + sum * add;
#pragma unroll
      for (int j = 0; j < 4; ++j) value[j] = value[j] * keep + v[j] * add;
    }
  values[threadIdx.x] = value, tops[threadIdx.x] = top, totals[threadIdx.x] = total;
  __syncthreads();
  if (part) return;
  for (int i = 1; i < parts; ++i) {
    const int at = i * items + item;
    const float next = fmaxf(top, tops[at]), ref = next == -INFINITY ? 0.f : next;
    const float keep = __builtin_amdgcn_exp2f(top - ref), add = __builtin_amdgcn_exp2f(tops[at] - ref);
    top = next;
    total = total * keep + totals[at] * add;
#pragma unroll
    for (int j = 0; j < 4; ++j) value[j] = value[j] * keep + values[at][j] * add;
  }
  const float inverse = inverse_of(total, top);
  const int64_t token = p.starts[record.request] + record.tile * p.tile_tokens + row / p.group;
  *reinterpret_cast<uint2*>(p.out + token * p.out_token + (record.head * p.group + row % p.group) * p.out_head + column) =
      make_uint2(pack_bf16(value[0] * inverse, value[1] * inverse), pack_bf16(value[2] * inverse, value[3] * inverse));
  if (p.lse && !column) store_lse(p, token, record.head * p.group + row % p.group, top, total);
}

constexpr int kJoinThreads = 256;

// Adds up the partial sums of the items that spans cut, four parts at a time: D / 32 workgroups per
// record, 256 threads in the layout that paged_attend wrote them in for each block of 32 columns. 200 rows of
// four heads on 3000 keys, 14 items of about eleven parts: 25.0 us with the attention before it (one workgroup
// with all threads: 28.4; one of 256 threads, part by part: 43).
template <int D>
__global__ __launch_bounds__(kJoinThreads) void paged_join(AttentionArgs p) {
  const Record record = reinterpret_cast<const Record*>(p.records)[blockIdx.x];
  if (record.others <= 0) return;
  const int thread = threadIdx.x, x = blockIdx.y, lane = thread & 63, wave = thread >> 6;
  f32x16 o;
#pragma unroll
  for (int e = 0; e < 16; ++e) o[e] = 0.f;
  float top = -INFINITY, sum = 0.f;
#pragma unroll 4
  for (int i = 0; i <= record.others; ++i) {
    const float* const from = p.partial + (2 * (int64_t)(record.worker + i) + (i == 0)) * kPartialFloats<D>;
    const float mine = from[256 * (D / 2) + thread], part = from[256 * (D / 2 + 1) + thread];
    f32x4 v[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = reinterpret_cast<const f32x4*>(from)[(4 * x + e) * 256 + thread];
    const float next = fmaxf(top, mine), ref = next == -INFINITY ? 0.f : next;
    const float keep = __builtin_amdgcn_exp2f(top - ref), add = __builtin_amdgcn_exp2f(mine - ref);
    top = next;
    sum = sum * keep + part * add;
#pragma unroll
    for (int e = 0; e < 16; ++e) o[e] = o[e] * keep + v[e >> 2][e & 3] * add;
  }
  const int fresh = p.rows[record.request];
  const int tile_rows = min(p.tile_tokens, fresh - record.tile * p.tile_tokens) * p.group;
  const int at = 32 * wave + (lane & 31), row = min(at, tile_rows - 1);
  const int64_t token = p.starts[record.request] + record.tile * p.tile_tokens + row / p.group;
  store_block(p.out + token * p.out_token + (record.head * p.group + row % p.group) * p.out_head + 32 * x, o,
              inverse_of(sum, top), at < tile_rows, lane >> 5);
  if (p.lse && x == 0 && lane < 32 && at < tile_rows) store_lse(p, token, record.head * p.group + row % p.group, top, sum);
}

// Workgroups of a launch, a multiple of the 8 XCDs: as many as a CU holds (two of paged_attend, by its
// LDS; four of paged_attend_few, by its registers).
int workgroups(int cus, bool few) { return ((few ? 4 : 2) * cus + 7) / 8 * 8; }

constexpr int64_t kRecordBytes = sizeof(Record);

int64_t workspace_of(int cus, int head_dim) {
  const int64_t many = kRecordBytes + 2 * 4 * 256 * (int64_t)(head_dim / 2 + 2);
  const int64_t few = kRecordBytes + 2 * 4 * 32 * (int64_t)(head_dim + 2);
  return max(workgroups(cus, false) * many, workgroups(cus, true) * few);
}

// Requests whose new rows fill one tile of 32 at most take the kernel for few rows: its waves
// share no work, so a tile of four times the rows reads the cache four times less. A step without new rows
// counts as one row a request: a tile holds a token at least.
bool few_rows(int64_t max_new, int group) { return (max_new > 1 ? max_new : 1) * group <= 32; }

template <int D>
int launch_attention(AttentionArgs& p, bool few, unsigned blocks, hipStream_t stream) {
  auto kern = few ? paged_attend_few<D> : paged_attend<D>;
  const int lds = (few ? 4 * 32 : 4 * 64) * 2 * D;
  if (lds > 48 * 1024) {
    hipError_t e = hipFuncSetAttribute((const void*)kern, hipFuncAttributeMaxDynamicSharedMemorySize, lds);
    if (e != hipSuccess) return fail(SMX_ERR_LAUNCH, "hipFuncSetAttribute: %s", hipGetErrorString(e));
  }
  hipLaunchKernelGGL(kern, dim3(blocks), dim3(few ? 64 : 256), lds, stream, p);
  if (int rc = check_launch()) return rc;
  hipLaunchKernelGGL(few ? paged_join_few<D> : paged_join<D>, dim3(blocks, few ? 1 : D / 32),
                     dim3(few ? 1024 : kJoinThreads), 0, stream, p);
  return check_launch();
}

}  // namespace
}  // namespace smx

using namespace smx;

extern "C" {

int smx_paged_attention_workspace_bytes(int32_t head_dim, int64_t* bytes) {
  smx::fail(SMX_OK, "%s", "");
  if (!bytes) return fail(SMX_ERR_INVALID, "null pointer");
  if (head_dim != 64 && head_dim != 128) return fail(SMX_ERR_UNSUPPORTED, "head_dim must be 64 or 128, got %d", head_dim);
  int cus = 0;
  if (int rc = device_cus(&cus)) return rc;
  *bytes = workspace_of(cus, head_dim);
  return SMX_OK;
}

int smx_paged_attention(const smx_paged_cache* cache, const smx_paged_step* step, const smx_heads* q,
                        const smx_heads* out, float scale, int32_t window, int32_t zero_rows, void* workspace,
                        int64_t workspace_bytes, void* stream) {
  return smx_paged_attention_lse(cache, step, q, out, scale, window, zero_rows, nullptr, workspace, workspace_bytes, stream);
}

int smx_paged_attention_lse(const smx_paged_cache* cache, const smx_paged_step* step, const smx_heads* q,
                            const smx_heads* out, float scale, int32_t window, int32_t zero_rows, float* lse,
                            void* workspace, int64_t workspace_bytes, void* stream) {
  smx::fail(SMX_OK, "%s", "");
  if (int rc = paged_layout(cache)) return rc;
  if (!step || !step->block_tables || !step->starts || !step->rows || !step->context || !step->positions || !q ||
      !q->data || !out || !out->data)
    return fail(SMX_ERR_INVALID, "null pointer");
  if (step->requests <= 0 || step->requests > SMX_PAGED_MAX_REQUESTS || step->tokens <= 0 ||
      step->tokens > SMX_PAGED_MAX_TOKENS || step->max_new < 0 || step->table_stride <= 0)
    return fail(SMX_ERR_INVALID, "a step has 1 to %d requests and 1 to %d tokens (requests=%d, tokens=%d)",
                SMX_PAGED_MAX_REQUESTS, SMX_PAGED_MAX_TOKENS, step->requests, step->tokens);
  if (q->heads <= 0 || q->heads % cache->kv_heads || q->heads / cache->kv_heads > 128)
    return fail(SMX_ERR_INVALID, "%d query heads are not 1 to 128 for each of %d key/value heads", q->heads,
                cache->kv_heads);
  if (out->heads != q->heads) return fail(SMX_ERR_INVALID, "out must have the %d query heads", q->heads);
  for (const smx_heads* x : {q, out})
    if ((uintptr_t)x->data % 16 || x->token_stride % 8 || x->head_stride % 8 || x->token_stride < 0 ||
        x->head_stride < 0)
      return fail(SMX_ERR_INVALID, "head rows must be 16-byte aligned");
  // A workgroup stores its rows while others load theirs: no row of out may be another's, nor a query of
  // another row, nor a key or value.
  const Runs from = head_runs(*q, step->tokens, cache->head_dim), to = head_runs(*out, step->tokens, cache->head_dim);
  if (!lie_apart(to)) return fail(SMX_ERR_INVALID, "out holds rows that lie on each other");
  if (!same_runs(from, to) && meet(from, to))
    return fail(SMX_ERR_INVALID, "out must be the queries themselves or share no memory with them");
  for (const void* x : {cache->k, cache->v})
    if (meet(cache_runs(*cache, x), to)) return fail(SMX_ERR_INVALID, "out must share no memory with the cache");
  if (lse) {
    const Runs sums{lse, 2 * (int64_t)step->tokens * q->heads, {{1, 0}, {1, 0}, {1, 0}}};  // (in units of 2 bytes)
    if ((uintptr_t)lse % 4 || meet(sums, from) || meet(sums, to) || meet(sums, cache_runs(*cache, cache->k)) ||
        meet(sums, cache_runs(*cache, cache->v)))
      return fail(SMX_ERR_INVALID, "lse must be aligned and share no memory with the queries, out or the cache");
    if (meets_step(lse, 2 * sums.width, *step)) return fail(SMX_ERR_INVALID, "lse must share no memory with the step's lists");
  }
  constexpr float kLog2E = 1.44269504088896341f;  // (the kernels' exponentials are powers of two)
  if (!(scale > 0.f) || !(scale * kLog2E < INFINITY))
    return fail(SMX_ERR_INVALID, "scale must be positive and finite, also times log2 e");
  if (window < 0) return fail(SMX_ERR_INVALID, "window must not be negative (0: none)");
  int cus = 0;
  if (int rc = device_cus(&cus)) return rc;
  const int64_t need = workspace_of(cus, cache->head_dim);
  if (!workspace || (uintptr_t)workspace % 16 || workspace_bytes < need)
    return fail(SMX_ERR_INVALID, "the call needs a 16-byte aligned workspace of %lld bytes", (long long)need);
  AttentionArgs p{};
  p.q = (const uint16_t*)q->data, p.q_token = q->token_stride, p.q_head = q->head_stride;
  p.out = (uint16_t*)out->data, p.out_token = out->token_stride, p.out_head = out->head_stride;
  p.k = (const uint16_t*)cache->k, p.v = (const uint16_t*)cache->v;
  p.page_stride = cache->page_stride, p.slot_stride = cache->slot_stride, p.head_stride = cache->head_stride;
  p.tables = step->block_tables, p.table_stride = step->table_stride;
  p.starts = step->starts, p.rows = step->rows, p.context = step->context, p.positions = step->positions;
  p.requests = step->requests, p.tokens = step->tokens;
  p.kv_heads = cache->kv_heads, p.group = q->heads / cache->kv_heads;
  p.page_shift = __builtin_ctz(cache->page_size), p.num_pages = cache->num_pages;
  p.window = window < SMX_PAGED_MAX_CONTEXT ? window : 0;  // wider than any request: none
  p.zero_rows = zero_rows;
  const bool few = few_rows(step->max_new, p.group);
  const int blocks = workgroups(cus, few);
  p.tile_tokens = (few ? 32 : 128) / p.group;
  // Units of a span at least, so that few partial sums are joined: an item's start and one step of 32 keys (one row on
  // 1000 keys 12.4 us; with two steps 13.1, three 15.4), two of 64 (two requests of 60 rows on 1000: 25.4; one
  // 27.4, three 26.0).
  p.min_span = few ? 2 : 5;
  p.scale = scale * kLog2E;
  p.per_group = 1.f / p.group;
  p.per_workgroup = 1. / blocks;
  p.records = (int32_t*)workspace;
  p.partial = (float*)((char*)workspace + blocks * kRecordBytes);
  p.lse = lse;
  return cache->head_dim == 128 ? launch_attention<128>(p, few, blocks, (hipStream_t)stream)
                                : launch_attention<64>(p, few, blocks, (hipStream_t)stream);
}

}  // extern "C"
