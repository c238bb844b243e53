// Verification of drafted tokens (smx_verify_drafts): which of them the target distribution accepts,
// and the token that follows, drawn from given random numbers.
//
// Mathematics. Draft i of a request, x, drawn from q_i, is accepted if u_i q_i(x) < p_i(x). The first that is not is
// replaced by a token drawn from max(p_i - q_i, 0); behind an accepted last one a token is drawn from the last
// row's p. A draw takes the first token whose running sum exceeds v times the whole sum. Products and
// sums are in 64 bits: a sum of 150,000 values in FP32 is off by more than many of them, and the token would depend
// on the order of the additions.
//
// Work. One row of p and one of q a request, whatever the number of drafts: verify_sums cuts the row in slices, a workgroup
// each, verify_draw finds the slice that the draw falls in and looks through that slice alone.
#include "launch.hpp"

namespace smx {
namespace {

struct VerifyArgs {
  const void *target, *draft;  // [rows, vocab] probabilities
  int64_t target_row, draft_row;
  const void* tokens;
  const int32_t *starts, *rows, *positions;
  const float *accept, *sample;
  void* out;
  int32_t* counts;
  int32_t* accepted;  // [requests]
  double* sums;       // [requests][slices][2]: of what is drawn from, and of p alone
  int32_t requests, count, vocab, slice, slices, flags;
};

constexpr int kVerifyThreads = 256, kSlice = 4096, kMostSlices = 1024;

// Probabilities that are no positive finite numbers count as zero.
__device__ __forceinline__ float probability(float x) { return x > 0.f && x < INFINITY ? x : 0.f; }

template <bool kBf16>
__device__ __forceinline__ float value_at(const void* p, int64_t at) {
  return probability(kBf16 ? bf16_to_f32(((const uint16_t*)p)[at]) : ((const float*)p)[at]);
}

__device__ __forceinline__ int64_t token_at(const VerifyArgs& p, int64_t row) {
  return p.flags & SMX_VERIFY_TOKENS_I64 ? ((const int64_t*)p.tokens)[row] : ((const int32_t*)p.tokens)[row];
}

// How many of the request's drafts are accepted; every wave finds out for itself.
template <bool kBf16>
__device__ int accepted_of(const VerifyArgs& p, int64_t start, int drafts) {
  for (int first = 0; first < drafts; first += 64) {
    const int i = first + (threadIdx.x & 63);
    bool refused = false;
    if (i < drafts) {
      const int64_t row = start + i, token = token_at(p, row + 1);
      double mine = 0., theirs = 0.;
      if (token >= 0 && token < p.vocab) {
        mine = value_at<kBf16>(p.target, row * p.target_row + token);
        theirs = p.draft ? value_at<kBf16>(p.draft, row * p.draft_row + token) : 1.f;
      }
      refused = !(mine > 0. && (double)p.accept[row] * theirs < mine);
    }
    if (const uint64_t who = __ballot(refused)) return first + __builtin_ctzll(who);
  }
  return drafts;
}

// What a request draws from: value(i) of token i, and p(i).
template <bool kBf16>
struct Row {
  const void *target, *draft;
  int64_t at, draft_at;
  int64_t left_out;  // a token whose value is zero: a refused one that had no distribution
  bool whole;

  __device__ Row(const VerifyArgs& p, int64_t start, int drafts, int accepted)
      : target(p.target), draft(accepted < drafts ? p.draft : nullptr), at((start + accepted) * p.target_row),
        draft_at((start + accepted) * p.draft_row), left_out(-1) {
    if (accepted < drafts && !p.draft) left_out = token_at(p, start + accepted + 1);
  }
  __device__ double both(int i, double* p) const {
    const float mine = value_at<kBf16>(target, at + i);
    *p = mine;
    if (draft) return max((double)mine - (double)value_at<kBf16>(draft, draft_at + i), 0.);
    return i == left_out ? 0. : (double)mine;
  }
  // Of a row whose max(p - q, 0) is all zero, p itself.
  __device__ double value(int i, bool plain) const {
    double p;
    const double rest = both(i, &p);
    return plain ? p : rest;
  }
};

__device__ __forceinline__ double wave_sum(double x) {
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) x += __shfl_xor(x, d);
  return x;
}

template <bool kBf16>
__global__ __launch_bounds__(kVerifyThreads) void verify_sums(VerifyArgs p) {
  const int request = blockIdx.y, fresh = p.rows[request];
  if (fresh <= 0) return;
  const int64_t start = p.starts[request];
  const int accepted = accepted_of<kBf16>(p, start, fresh - 1);
  if (blockIdx.x == 0 && threadIdx.x == 0) p.accepted[request] = accepted;
  const Row<kBf16> row(p, start, fresh - 1, accepted);
  const int from = blockIdx.x * p.slice, to = min(p.vocab, from + p.slice);
  double rest = 0., whole = 0.;
#pragma unroll 8
  for (int i = from + (int)threadIdx.x; i < to; i += kVerifyThreads) {
    double mine;
    rest += row.both(i, &mine);
    whole += mine;
  }
  __shared__ double parts[2][kVerifyThreads / 64];
  rest = wave_sum(rest), whole = wave_sum(whole);
  if ((threadIdx.x & 63) == 0) parts[0][threadIdx.x >> 6] = rest, parts[1][threadIdx.x >> 6] = whole;
  __syncthreads();
  if (threadIdx.x < 2) {
    double sum = 0.;
    for (int w = 0; w < kVerifyThreads / 64; ++w) sum += parts[threadIdx.x][w];
    p.sums[((int64_t)request * p.slices + blockIdx.x) * 2 + threadIdx.x] = sum;
  }
}

// Inclusive sum over the workgroup's threads.
__device__ double block_scan(double x, double* waves) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const double y = __shfl_up(x, d);
    if (lane >= d) x += y;
  }
  __syncthreads();
  if (lane == 63) waves[wave] = x;
  __syncthreads();
  for (int w = 0; w < wave; ++w) x += waves[w];
  return x;
}

template <bool kBf16>
__global__ __launch_bounds__(kVerifyThreads) void verify_draw(VerifyArgs p) {
  const int request = blockIdx.x, fresh = p.rows[request];
  // rows of no request
  for (int64_t r = (int64_t)request * kVerifyThreads + threadIdx.x; r < p.count; r += (int64_t)gridDim.x * kVerifyThreads)
    if (p.positions[r] < 0) {
      if (p.flags & SMX_VERIFY_TOKENS_I64) ((int64_t*)p.out)[r] = -1; else ((int32_t*)p.out)[r] = -1;
    }
  if (fresh <= 0) {
    if (threadIdx.x == 0) p.counts[request] = 0;
    return;
  }
  __shared__ double waves[kVerifyThreads / 64], base;
  __shared__ int chosen, token, last;
  if (threadIdx.x == 0) chosen = token = INT32_MAX, last = -1;
  const int64_t start = p.starts[request];
  const int accepted = p.accepted[request];
  const double* const sums = p.sums + (int64_t)request * p.slices * 2;
  // a thread's slices, one behind the other
  constexpr int kEach = kMostSlices / kVerifyThreads;
  double mine[2][kEach], total[2];
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    double sum = 0.;
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
      const int s = (int)threadIdx.x * kEach + i;
      mine[k][i] = s < p.slices ? sums[2 * s + k] : 0.;
      sum += mine[k][i];
    }
    total[k] = sum;
  }
  const double upto_rest = block_scan(total[0], waves), upto_whole = block_scan(total[1], waves);
  __shared__ double all[2];
  if (threadIdx.x == kVerifyThreads - 1) all[0] = upto_rest, all[1] = upto_whole;
  __syncthreads();
  const bool plain = !(all[0] > 0.);
  const double goal = (double)p.sample[request] * (plain ? all[1] : all[0]);
  double before = (plain ? upto_whole : upto_rest) - (plain ? total[1] : total[0]);
  // the first slice whose running sum passes the goal, or (by rounding, or a number that is not below 1)
  // the last one that holds anything
#pragma unroll
  for (int i = 0; i < kEach; ++i) {
    const int s = (int)threadIdx.x * kEach + i;
    const double part = plain ? mine[1][i] : mine[0][i];
    if (part > 0.) {
      if (before + part > goal) atomicMin(&chosen, s);
      atomicMax(&last, s);
    }
    before += part;
  }
  __syncthreads();
  const bool beyond = chosen == INT32_MAX;
  const int slice = beyond ? last : chosen;
  if (slice >= 0) {
    if (slice / kEach == (int)threadIdx.x) {
      double b = (plain ? upto_whole : upto_rest) - (plain ? total[1] : total[0]);
#pragma unroll
      for (int i = 0; i < kEach; ++i)
        if (i < slice % kEach) b += plain ? mine[1][i] : mine[0][i];
      base = b;
    }
    __syncthreads();
    if (threadIdx.x == 0) last = -1;
    const Row<kBf16> row(p, start, fresh - 1, accepted);
    const int from = slice * p.slice, to = min(p.vocab, from + p.slice), each = p.slice / kVerifyThreads;
    const int first = from + (int)threadIdx.x * each, end = min(to, first + each);
    double sum = 0.;
#pragma unroll 4
    for (int i = first; i < end; ++i) sum += row.value(i, plain);
    const double upto = base + block_scan(sum, waves);
    double running = upto - sum;
    // a thread's tokens: the first whose running sum passes the goal, and the last with any
    if (sum > 0.) {
      int hit = INT32_MAX, most = -1;
      for (int i = first; i < end; ++i) {
        const double v = row.value(i, plain);
        running += v;
        if (v > 0.) {
          most = i;
          if (running > goal && hit == INT32_MAX) hit = i;
        }
      }
      if (!beyond && hit != INT32_MAX) atomicMin(&token, hit);
      atomicMax(&last, most);
    }
    __syncthreads();
  }
  const int drawn = slice < 0 ? -1 : token != INT32_MAX ? token : last;
  for (int i = threadIdx.x; i < fresh; i += kVerifyThreads) {
    const int64_t value = i < accepted ? token_at(p, start + i + 1) : i == accepted ? drawn : -1;
    if (p.flags & SMX_VERIFY_TOKENS_I64) ((int64_t*)p.out)[start + i] = value; else ((int32_t*)p.out)[start + i] = (int32_t)value;
  }
  if (threadIdx.x == 0) p.counts[request] = accepted + 1;
}

// Tokens of a slice, a multiple of the workgroup's threads.
int slice_of(int vocab) {
  const int64_t least = ((int64_t)vocab + kMostSlices - 1) / kMostSlices;
  return (int)max((int64_t)kSlice, (least + kVerifyThreads - 1) / kVerifyThreads * kVerifyThreads);
}
int slices_of(int vocab) { return (int)(((int64_t)vocab + slice_of(vocab) - 1) / slice_of(vocab)); }

}  // namespace
}  // namespace smx

using namespace smx;

extern "C" {

int smx_verify_workspace_bytes(int32_t requests, int32_t vocab, int64_t* bytes) {
  smx::fail(SMX_OK, "%s", "");
  if (!bytes) return fail(SMX_ERR_INVALID, "null pointer");
  if (requests <= 0 || requests > SMX_PAGED_MAX_REQUESTS || vocab <= 0 || vocab > SMX_VERIFY_MAX_VOCAB)
    return fail(SMX_ERR_INVALID, "1 to %d requests and 1 to %d tokens in the vocabulary (requests=%d, vocab=%d)",
                SMX_PAGED_MAX_REQUESTS, SMX_VERIFY_MAX_VOCAB, requests, vocab);
  *bytes = (int64_t)requests * (slices_of(vocab) * 16 + 8);
  return SMX_OK;
}

int smx_verify_drafts(const smx_paged_step* step, int32_t vocab, const void* target, int64_t target_row, const void* draft,
                      int64_t draft_row, const void* tokens, const float* accept, const float* sample, int32_t flags, void* out,
                      int32_t* counts, void* workspace, int64_t workspace_bytes, void* stream) {
  int64_t need = 0;
  if (!step) return fail(SMX_ERR_INVALID, "null pointer");
  if (int rc = smx_verify_workspace_bytes(step->requests, vocab, &need)) return rc;
  if (!step->starts || !step->rows || !step->positions || !target || !tokens || !accept || !sample || !out || !counts)
    return fail(SMX_ERR_INVALID, "null pointer");
  if (step->tokens <= 0 || step->tokens > SMX_PAGED_MAX_TOKENS)
    return fail(SMX_ERR_INVALID, "1 to %d tokens, got %d", SMX_PAGED_MAX_TOKENS, step->tokens);
  if (flags & ~(SMX_VERIFY_BF16 | SMX_VERIFY_TOKENS_I64)) return fail(SMX_ERR_INVALID, "unknown flags 0x%x", flags);
  if ((step->tokens > 1 && target_row < vocab) || (draft && step->tokens > 1 && draft_row < vocab))
    return fail(SMX_ERR_INVALID, "rows must be at least vocab=%d apart", vocab);
  const int size = flags & SMX_VERIFY_BF16 ? 2 : 4;
  if ((uintptr_t)target % size || (uintptr_t)draft % size || (uintptr_t)tokens % (flags & SMX_VERIFY_TOKENS_I64 ? 8 : 4) ||
      (uintptr_t)out % (flags & SMX_VERIFY_TOKENS_I64 ? 8 : 4))
    return fail(SMX_ERR_INVALID, "misaligned probabilities or tokens");
  if (!workspace || (uintptr_t)workspace % 16 || workspace_bytes < need)
    return fail(SMX_ERR_INVALID, "the call needs a 16-byte aligned workspace of %lld bytes", (long long)need);
  VerifyArgs p{};
  p.target = target, p.draft = draft, p.target_row = target_row, p.draft_row = draft_row, p.tokens = tokens;
  p.starts = step->starts, p.rows = step->rows, p.positions = step->positions, p.accept = accept, p.sample = sample;
  p.out = out, p.counts = counts, p.requests = step->requests, p.count = step->tokens, p.vocab = vocab, p.flags = flags;
  p.slice = slice_of(vocab), p.slices = slices_of(vocab);
  p.sums = (double*)workspace;
  p.accepted = (int32_t*)(p.sums + 2 * (int64_t)p.requests * p.slices);
  const bool bf16 = flags & SMX_VERIFY_BF16;
  hipLaunchKernelGGL(bf16 ? verify_sums<true> : verify_sums<false>, dim3((unsigned)p.slices, (unsigned)p.requests),
                     dim3(kVerifyThreads), 0, (hipStream_t)stream, p);
  if (int rc = check_launch()) return rc;
  hipLaunchKernelGGL(bf16 ? verify_draw<true> : verify_draw<false>, dim3((unsigned)p.requests), dim3(kVerifyThreads), 0,
                     (hipStream_t)stream, p);
  return check_launch();
}

}  // extern "C"
