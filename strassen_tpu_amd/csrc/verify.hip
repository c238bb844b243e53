// Verification of drafted tokens (smx_verify_drafts): which of them the target distribution accepts,
// and the token that follows, drawn from given random numbers.
//
// Mathematics. Draft i of a request, x, drawn from q_i, is accepted if u_i q_i(x) < p_i(x). The first that is not is
// replaced by a token drawn from max(p_i - q_i, 0); behind an accepted last one a token is drawn from the last
// row's p. A draw takes the first token whose running sum exceeds v times the whole sum. Products and
// sums are in 64 bits: a sum of 150,000 values in FP32 is off by more than many of them, and the token would depend
// on the order of the additions (which is another one where a request is shared out, below).
//
// Work. One row of p and one of q a request, whatever the number of drafts: verify_sums cuts the row in slices, a workgroup
// each, verify_draw finds the slice that the draw falls in and looks through that slice alone. Where requests fill the chip or
// the vocabulary is small verify_whole does both in one launch. Bound by memory where requests
// are many: 64 requests with drafts on 151,936 tokens, 78 MB of FP32, take 22 us, 17 of them the sums (4.7 TB/s); one
// request takes 9.5 us, 8 of them in two launches that wait for a chain of lengths, tokens, their probabilities and the row.
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

constexpr int kVerifyThreads = 256;

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

// Four values of a row, of any alignment.
typedef f32x4 f32x4_loose __attribute__((aligned(4)));
typedef uint16_t u16x4 __attribute__((ext_vector_type(4)));
typedef u16x4 u16x4_loose __attribute__((aligned(2)));

// What a request draws from: max(p - q, 0) of the row whose draft was refused, or p.
template <bool kBf16>
struct Row {
  const void *target, *draft;
  int64_t at, draft_at;
  int64_t left_out;  // a token whose value is zero: a refused one that had no distribution

  __device__ Row(const VerifyArgs& p, int64_t start, int drafts, int accepted)
      : target(p.target), draft(accepted < drafts ? p.draft : nullptr), at((start + accepted) * p.target_row),
        draft_at((start + accepted) * p.draft_row), left_out(-1) {
    if (accepted < drafts && !p.draft) left_out = token_at(p, start + accepted + 1);
  }
  // Values i .. i + 3 of the row at `from`, zeros from `end` on.
  __device__ __forceinline__ static f32x4 four(const void* p, int64_t from, int i, int end) {
    f32x4 x = {0.f, 0.f, 0.f, 0.f};
    if (i + 4 <= end) {
      if constexpr (kBf16) {
        const u16x4 v = *reinterpret_cast<const u16x4_loose*>((const uint16_t*)p + from + i);
#pragma unroll
        for (int j = 0; j < 4; ++j) x[j] = bf16_to_f32(v[j]);
      } else {
        x = *reinterpret_cast<const f32x4_loose*>((const float*)p + from + i);
      }
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (i + j < end) x[j] = kBf16 ? bf16_to_f32(((const uint16_t*)p)[from + i + j]) : ((const float*)p)[from + i + j];
    }
    return x;
  }
  struct Four {
    f32x4 p, q;
  };
  __device__ __forceinline__ Four load(int i, int end) const {
    Four f;
    f.p = four(target, at, i, end);
    f.q = draft ? four(draft, draft_at, i, end) : f32x4{0.f, 0.f, 0.f, 0.f};
    return f;
  }
  // Value j of those from i on; `plain`: p itself, for a row whose max(p - q, 0) is all zero.
  __device__ __forceinline__ double value(const Four& f, int i, int j, bool plain) const {
    const double p = probability(f.p[j]);
    if (plain) return p;
    if (draft) return max(p - (double)probability(f.q[j]), 0.);
    return i + j == left_out ? 0. : p;
  }
  // The sums of a share of the tokens from .. to - 1: thread `mine` of kThreads.
  template <int kThreads>
  __device__ __forceinline__ void add(int from, int to, int mine, double& rest, double& whole) const {
#pragma unroll 4
    for (int i = from + 4 * mine; i < to; i += 4 * kThreads) {
      const auto f = load(i, to);
#pragma unroll
      for (int j = 0; j < 4; ++j) rest += value(f, i, j, false), whole += value(f, i, j, true);
    }
  }
};

// Sum over a wave's lanes, in every lane.
__device__ __forceinline__ double wave_sum(double x) {
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) x += __shfl_xor(x, d);
  return x;
}

// Inclusive sum over a wave's lanes.
__device__ __forceinline__ double lane_scan(double x) {
  const int lane = threadIdx.x & 63;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const double y = __shfl_up(x, d);
    if (lane >= d) x += y;
  }
  return x;
}

template <bool kBf16>
__global__ __launch_bounds__(kVerifyThreads) void verify_sums(VerifyArgs p) {
  const int request = blockIdx.y, fresh = p.rows[request];
  const int64_t start = p.starts[request];
  if (fresh <= 0) return;
  const int accepted = accepted_of<kBf16>(p, start, fresh - 1);
  if (blockIdx.x == 0 && threadIdx.x == 0) p.accepted[request] = accepted;
  const Row<kBf16> row(p, start, fresh - 1, accepted);
  const int from = blockIdx.x * p.slice;
  double rest = 0., whole = 0.;
  row.template add<kVerifyThreads>(from, min(p.vocab, from + p.slice), threadIdx.x, rest, whole);
  constexpr int kWaves = kVerifyThreads / 64;
  __shared__ double parts[2][kWaves];
  rest = wave_sum(rest), whole = wave_sum(whole);
  if ((threadIdx.x & 63) == 0) parts[0][threadIdx.x >> 6] = rest, parts[1][threadIdx.x >> 6] = whole;
  __syncthreads();
  if (threadIdx.x < 2) {
    double sum = 0.;
    for (int w = 0; w < kWaves; ++w) sum += parts[threadIdx.x][w];
    p.sums[((int64_t)request * p.slices + blockIdx.x) * 2 + threadIdx.x] = sum;
  }
}

__device__ __forceinline__ void emit(const VerifyArgs& p, int64_t row, int64_t token) {
  if (p.flags & SMX_VERIFY_TOKENS_I64) ((int64_t*)p.out)[row] = token; else ((int32_t*)p.out)[row] = (int32_t)token;
}

// Rows of no request, shared out over all workgroups.
template <int kThreads>
__device__ __forceinline__ void emit_others(const VerifyArgs& p, int request) {
  for (int64_t r = (int64_t)request * kThreads + threadIdx.x; r < p.count; r += (int64_t)p.requests * kThreads)
    if (p.positions[r] < 0) emit(p, r, -1);
}

// A request's token, drawn by its slices' sums (at most 64, one a lane: of what is drawn from, and of p alone), and all that it
// emits.
template <bool kBf16, int kThreads>
__device__ __forceinline__ void draw(const VerifyArgs& p, int request, int64_t start, int fresh, int accepted,
                                     const Row<kBf16>& row, double sample, double mine_rest, double mine_whole) {
  constexpr int kWaves = kThreads / 64, kRun = 4 * kThreads;  // tokens that the workgroup loads at once
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  // Every wave finds the slice.
  const bool plain = !__any(mine_rest > 0.);
  const double mine = plain ? mine_whole : mine_rest, upto = lane_scan(mine);
  const double goal = sample * __shfl(upto, 63);
  // the first whose running sum passes the goal, or (by rounding, or a number that is not below 1) the last one that
  // holds anything
  const uint64_t any = __ballot(mine > 0.), over = __ballot(mine > 0. && upto > goal);
  if (!any) {
    for (int i = threadIdx.x; i < fresh; i += kThreads) emit(p, start + i, i < accepted ? token_at(p, start + i + 1) : -1);
    if (threadIdx.x == 0) p.counts[request] = accepted + 1;
    return;
  }
  const int slice = over ? __builtin_ctzll(over) : 63 - __builtin_clzll(any);
  double base = __shfl(upto - mine, slice);
  const int from = slice * p.slice, to = min(p.vocab, from + p.slice);

  __shared__ double waves[2][kWaves];
  __shared__ int first_of[kWaves], last_of[kWaves];
  int hit = -1, most = -1, buffer = 0;  // the thread's first token past the goal, and its last of any probability
  // A run of the slice after another, four tokens a thread; the next one's are on their way.
  auto f = row.load(from + 4 * (int)threadIdx.x, to);
  for (int run = from; run < to; run += kRun, buffer ^= 1) {
    const int i = run + 4 * (int)threadIdx.x;
    const auto now = f;
    f = row.load(i + kRun, to);
    double value[4], sum = 0.;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      value[j] = row.value(now, i, j, plain), sum += value[j];
      if (value[j] > 0.) most = i + j;
    }
    const double scanned = lane_scan(sum);
    if (lane == 63) waves[buffer][wave] = scanned;
    __syncthreads();
    double running = base + scanned - sum;
    for (int w = 0; w < kWaves; ++w) {
      if (w < wave) running += waves[buffer][w];
      base += waves[buffer][w];
    }
    if (over && base > goal) {  // uniform: here
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        running += value[j];
        if (value[j] > 0. && running > goal && hit < 0) hit = i + j;
      }
      break;
    }
  }
  // The first token past the goal; where sums in another order leave none, the last of any probability.
  const uint64_t hits = __ballot(hit >= 0);  // (of one run, whose tokens are in the threads' order)
  const int wave_hit = hits ? __shfl(hit, __builtin_ctzll(hits)) : -1;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) most = max(most, __shfl_xor(most, d));
  if (lane == 0) first_of[wave] = wave_hit, last_of[wave] = most;
  __syncthreads();
  int drawn = -1, last = -1;
  for (int w = 0; w < kWaves; ++w) {
    if (drawn < 0) drawn = first_of[w];
    last = max(last, last_of[w]);
  }
  if (drawn < 0) drawn = last;
  for (int i = threadIdx.x; i < fresh; i += kThreads)
    emit(p, start + i, i < accepted ? token_at(p, start + i + 1) : i == accepted ? drawn : -1);
  if (threadIdx.x == 0) p.counts[request] = accepted + 1;
}

template <bool kBf16>
__global__ __launch_bounds__(kVerifyThreads) void verify_draw(VerifyArgs p) {
  // (all that does not wait for anything else is read at once; accepted and sums are none of a request without rows)
  const int request = blockIdx.x, lane = threadIdx.x & 63;
  const double* const sums = p.sums + (int64_t)request * p.slices * 2;
  const int fresh = p.rows[request], accepted = p.accepted[request];
  const int64_t start = p.starts[request];
  const double sample = p.sample[request];
  const double rest = lane < p.slices ? sums[2 * lane] : 0., whole = lane < p.slices ? sums[2 * lane + 1] : 0.;
  if (fresh > 0)
    draw<kBf16, kVerifyThreads>(p, request, start, fresh, accepted, Row<kBf16>(p, start, fresh - 1, accepted), sample, rest, whole);
  else if (threadIdx.x == 0)
    p.counts[request] = 0;
  emit_others<kVerifyThreads>(p, request);
}

// The whole of a request by one workgroup, a slice a wave.
template <bool kBf16, int kThreads>
__global__ __launch_bounds__(kThreads) void verify_whole(VerifyArgs p) {
  constexpr int kWaves = kThreads / 64;
  const int request = blockIdx.x, fresh = p.rows[request], lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t start = p.starts[request];
  const double sample = p.sample[request];
  if (fresh > 0) {
    const int accepted = accepted_of<kBf16>(p, start, fresh - 1);
    const Row<kBf16> row(p, start, fresh - 1, accepted);
    __shared__ double sums[2][kWaves];
    double rest = 0., whole = 0.;
    const int from = wave * p.slice;
    row.template add<64>(from, min(p.vocab, from + p.slice), lane, rest, whole);
    rest = wave_sum(rest), whole = wave_sum(whole);
    if (lane == 0) sums[0][wave] = rest, sums[1][wave] = whole;
    __syncthreads();
    draw<kBf16, kThreads>(p, request, start, fresh, accepted, row, sample, lane < kWaves ? sums[0][lane] : 0.,
                          lane < kWaves ? sums[1][lane] : 0.);
  } else if (threadIdx.x == 0) {
    p.counts[request] = 0;
  }
  emit_others<kThreads>(p, request);
}

// Threads of a workgroup that takes the whole of a request, which saves a launch and the second chain of loads; 0: the request is
// shared out. In us, shared out, of 1024 threads and of 512 (bf16, two drafts looked up):
//             8 requests         128                200                256                400
//   2453    9.9  8.7  7.4    10.1  9.1  7.7     10.2  9.3  7.7    10.3  9.1  7.8     11.0 14.9  9.0
//   8000    9.6  9.1 10.6    10.3  9.4 10.1     10.8  9.5 10.2    10.9  9.5 10.0     14.2 16.1 12.2
//  32001    9.6 13.4 15.3    14.8 15.6 17.7     18.6 15.8 20.1    21.3 16.0 20.0     27.5 28.6 21.7
// 151936     11   28   43      30   35   60       38   35   61      47   40   69       77   80   79
int whole_threads(int vocab, int requests) {
  constexpr int kCus = 256;
  if (requests > 2 * kCus) return 0;  // (a second round: 600 requests of 32,001 tokens 37, shared out 32)
  if (vocab <= 4096) return 512;
  if (requests > kCus) return vocab <= 65536 ? 512 : 0;
  return vocab <= 8192 || requests >= 192 ? 1024 : 0;
}

// Tokens of a slice, a multiple of the workgroup's loads: at most 64 slices, of 2048 tokens at least, and no more
// than fill the chip with workgroups twice (64 requests 23.3 us, once 24.7; 100 of 32,001 tokens 14.8 either way).
int slice_of(int vocab, int requests) {
  if (const int waves = whole_threads(vocab, requests) / 64) return (vocab + 4 * waves - 1) / (4 * waves) * 4;
  constexpr int kRun = 4 * kVerifyThreads;
  const int64_t slices = max(1, min(64, 4096 / requests)), least = ((int64_t)vocab + slices - 1) / slices;
  return (int)max((int64_t)2048, (least + kRun - 1) / kRun * kRun);
}
int slices_of(int vocab, int requests) {
  const int slice = slice_of(vocab, requests);
  return (int)(((int64_t)vocab + slice - 1) / slice);
}

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
  *bytes = (int64_t)requests * (slices_of(vocab, requests) * 16 + 8);
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
      (uintptr_t)out % (flags & SMX_VERIFY_TOKENS_I64 ? 8 : 4) || (uintptr_t)accept % 4 || (uintptr_t)sample % 4 || (uintptr_t)counts % 4)
    return fail(SMX_ERR_INVALID, "misaligned probabilities, tokens, random numbers or counts");
  if (!workspace || (uintptr_t)workspace % 16 || workspace_bytes < need)
    return fail(SMX_ERR_INVALID, "the call needs a 16-byte aligned workspace of %lld bytes", (long long)need);
  // a request's tokens and count are stored while others read theirs
  const auto list = [](const void* at, int64_t count, int bytes) { return Runs{at, count * (bytes / 2), {{1, 0}, {1, 0}, {1, 0}}}; };
  const auto rows_of = [&](const void* at, int64_t row) {
    return Runs{at, (int64_t)vocab * (size / 2), {{step->tokens, row * (size / 2)}, {1, 0}, {1, 0}}};
  };
  const int64_t rows = step->tokens, requests = step->requests;
  const int token = flags & SMX_VERIFY_TOKENS_I64 ? 8 : 4;
  const Runs stored[] = {list(out, rows, token), list(counts, requests, 4)};
  if (meet(stored[0], list(tokens, rows, token))) return fail(SMX_ERR_INVALID, "out and tokens must share no memory");
  if (meet(stored[0], stored[1])) return fail(SMX_ERR_INVALID, "out and counts must share no memory");
  // (of the step, starts, rows and positions; the rest of it need not be there)
  const Runs read[] = {list(tokens, rows, token), list(accept, rows, 4), list(sample, requests, 4), list(step->starts, requests, 4),
                       list(step->rows, requests, 4), list(step->positions, rows, 4), rows_of(target, target_row)};
  for (const Runs& to : stored) {
    bool meets = draft && meet(to, rows_of(draft, draft_row));
    for (const Runs& from : read) meets = meets || meet(to, from);
    if (meets) return fail(SMX_ERR_INVALID, "out and counts must share no memory with what the call reads");
  }
  VerifyArgs p{};
  p.target = target, p.draft = draft, p.target_row = target_row, p.draft_row = draft_row, p.tokens = tokens;
  p.starts = step->starts, p.rows = step->rows, p.positions = step->positions, p.accept = accept, p.sample = sample;
  p.out = out, p.counts = counts, p.requests = step->requests, p.count = step->tokens, p.vocab = vocab, p.flags = flags;
  p.slice = slice_of(vocab, p.requests), p.slices = slices_of(vocab, p.requests);
  p.sums = (double*)workspace;
  p.accepted = (int32_t*)(p.sums + 2 * (int64_t)p.requests * p.slices);
  const bool bf16 = flags & SMX_VERIFY_BF16;
  if (const int threads = whole_threads(vocab, p.requests)) {
    auto kern = threads == 512 ? (bf16 ? verify_whole<true, 512> : verify_whole<false, 512>)
                               : (bf16 ? verify_whole<true, 1024> : verify_whole<false, 1024>);
    hipLaunchKernelGGL(kern, dim3((unsigned)p.requests), dim3((unsigned)threads), 0, (hipStream_t)stream, p);
    return check_launch();
  }
  hipLaunchKernelGGL(bf16 ? verify_sums<true> : verify_sums<false>, dim3((unsigned)p.slices, (unsigned)p.requests),
                     dim3(kVerifyThreads), 0, (hipStream_t)stream, p);
  if (int rc = check_launch()) return rc;
  hipLaunchKernelGGL(bf16 ? verify_draw<true> : verify_draw<false>, dim3((unsigned)p.requests), dim3(kVerifyThreads), 0,
                     (hipStream_t)stream, p);
  return check_launch();
}

}  // extern "C"
