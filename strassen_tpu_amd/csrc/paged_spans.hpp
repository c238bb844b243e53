// Equal spans of work over a paged cache: the steps of all (key/value head, request, tile) items, one behind
// the other, cut into one span per workgroup. Counts of steps have closed forms, so that every workgroup finds its span
// by itself, from the lengths on the device.
#pragma once

#include "common.hpp"

namespace smx {
namespace {

// A plan's lengths, read through the scalar cache where the index is a wave's.
__device__ __forceinline__ int32_t scalar_at(const int32_t* p, int i) {
  return ((const __attribute__((address_space(4))) int32_t*)(uintptr_t)p)[i];
}

// A workgroup's span of the units, and the item in which it begins.
struct Span {
  int64_t left;         // units to do
  int64_t each;         // units of a span
  int64_t begin;        // of this one, over all key/value heads
  int32_t worker;       // which span this is
  int32_t head, request, tile, skip;  // skip: units of that item that lie in spans before
  int32_t context, fresh;             // of that request
};

__device__ __forceinline__ int64_t lane_value(int64_t x, int lane) {
  return (int64_t)(uint32_t)__builtin_amdgcn_readlane((int)x, lane) |
         (int64_t)__builtin_amdgcn_readlane((int)(x >> 32), lane) << 32;
}

// a / b for 0 <= a, 0 < b and a quotient below 2^19, of which the reciprocal of b misses less
// than one (the integer division is ten times as long).
__device__ __forceinline__ int64_t quotient(int64_t a, int64_t b) {
  int64_t q = (int64_t)((float)a * __builtin_amdgcn_rcpf((float)b));
  if (q * b > a) --q;
  if ((q + 1) * b <= a) ++q;
  return q;
}

// x of the lanes that kControl names, zero where there are none.
template <int kControl, int kRows>
__device__ __forceinline__ int64_t moved(int64_t x) {
  const uint32_t low = __builtin_amdgcn_update_dpp(0, (int)x, kControl, kRows, 15, false);
  const uint32_t high = __builtin_amdgcn_update_dpp(0, (int)(x >> 32), kControl, kRows, 15, false);
  return (int64_t)((uint64_t)high << 32 | low);
}

// Inclusive sum of x over a wave's lanes: within rows of 16 lanes, then a row's last value
// to the next row, and the lower half's to the upper.
__device__ __forceinline__ int64_t wave_scan(int64_t x) {
  x += moved<0x111, 15>(x);
  x += moved<0x112, 15>(x);
  x += moved<0x114, 15>(x);
  x += moved<0x118, 15>(x);
  x += moved<0x142, 10>(x);
  x += moved<0x143, 12>(x);
  return x;
}

// Finds the workgroup's span (kWaves waves, uniform result). Consecutive spans lie
// on one XCD, whose L2 then serves one key/value head's pages at a time.
template <class Request, int kWaves, class Args>
__device__ bool find_span(const Args& p, Span* s) {
  constexpr int kThreads = 64 * kWaves;
  __shared__ int64_t waves[kWaves], found_rest;
  __shared__ int32_t found[3];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  // Inclusive sum over the workgroup of this thread's request among kThreads of them.
  int64_t mine = 0, upto = 0;
  int32_t context = 0, fresh = 0;
  auto scan = [&](int first) -> int64_t {
    const int b = first + (int)threadIdx.x;
    const bool here = b < p.requests;
    context = here ? p.context[b] : 0, fresh = here ? p.rows[b] : 0;
    mine = Request(p, context, fresh).all();
    upto = wave_scan(mine);
    if constexpr (kWaves == 1) return lane_value(upto, 63);
    __syncthreads();
    if (lane == 63) waves[wave] = upto;
    __syncthreads();
    int64_t all = 0;
    for (int w = 0; w < kWaves; ++w) {
      if (w < wave) upto += waves[w];
      all += waves[w];
    }
    return lane_value(all, 0);
  };
  int64_t total = 0;
  for (int first = 0; first < p.requests; first += kThreads) total += scan(first);
  const int64_t everything = total * p.kv_heads;
  int64_t each = (int64_t)((double)everything * p.per_workgroup);  // (at most one short)
  while (each * gridDim.x < everything) ++each;
  s->each = max((int64_t)p.min_span, each);
  const int64_t spans = quotient(everything + s->each - 1, s->each), per_xcd = (spans + 7) / 8;
  s->worker = (int)((blockIdx.x & 7) * per_xcd + (blockIdx.x >> 3));
  if ((blockIdx.x >> 3) >= per_xcd || s->worker >= spans) return false;
  s->begin = (int64_t)s->worker * s->each;
  s->left = min(s->each, everything - s->begin);
  s->head = __builtin_amdgcn_readfirstlane((int)quotient(s->begin, total));
  const int64_t at = s->begin - (int64_t)s->head * total;

  int64_t base = 0, rest = 0;
  for (int first = 0; first < p.requests; first += kThreads) {
    // (the sums of a single round are still there)
    const int64_t all = p.requests <= kThreads ? total : scan(first);
    const bool here = at >= base + upto - mine && at < base + upto;
    if constexpr (kWaves > 1) {
      if (here) {
        found[0] = first + (int)threadIdx.x, found[1] = context, found[2] = fresh;
        found_rest = at - (base + upto - mine);
      }
    } else if (const uint64_t who = __ballot(here)) {
      const int l = __builtin_ctzll(who);
      s->request = first + l;
      s->context = __builtin_amdgcn_readlane(context, l), s->fresh = __builtin_amdgcn_readlane(fresh, l);
      rest = at - (base + lane_value(upto - mine, l));
    }
    base += all;
    if (at < base) break;  // uniform
  }
  if constexpr (kWaves > 1) {
    __syncthreads();
    s->request = __builtin_amdgcn_readfirstlane(found[0]);
    s->context = __builtin_amdgcn_readfirstlane(found[1]), s->fresh = __builtin_amdgcn_readfirstlane(found[2]);
    rest = lane_value(found_rest, 0);
  }
  const auto r = Request::uniform(p, s->context, s->fresh);
  // The last tile with before(tile) <= rest: a lane each for 64 of them, evenly apart (500 rows
  // on 100 keys: 32.8 us, one after another 34.6).
  int low = 0, high = r.tiles;
  int64_t skipped = 0;  // before(low)
  while (high - low > 1) {
    const int width = (high - low + 63) >> 6, tile = low + lane * width;
    const int64_t sum = r.before(min(tile, high - 1));
    const int last = 63 - __builtin_clzll(__ballot(tile < high && sum <= rest));
    skipped = lane_value(sum, last);
    low += last * width, high = min(high, low + width);
  }
  s->tile = __builtin_amdgcn_readfirstlane(low);
  s->skip = __builtin_amdgcn_readfirstlane((int)(rest - skipped));
  return true;
}

// On to the next item with rows.
template <class Args>
__device__ __forceinline__ void next_item(const Args& p, Span* s, int tiles) {
  s->skip = 0;
  if (++s->tile < tiles) return;
  s->tile = 0;
  do {
    if (++s->request == p.requests) s->request = 0, ++s->head;
    s->fresh = scalar_at(p.rows, s->request);
  } while (s->fresh <= 0);
  s->context = scalar_at(p.context, s->request);
}

__device__ __forceinline__ float other_half(float x) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return (threadIdx.x & 32) ? __uint_as_float(r[0]) : __uint_as_float(r[1]);
}

}  // namespace
}  // namespace smx
