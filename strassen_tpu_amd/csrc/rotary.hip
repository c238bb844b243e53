// Rotary positions (smx_rotary): pairs of a head's values turned by an angle that grows with the row's
// position, the head RMS-normalised before if asked.
//
// Mathematics. Pair i of a head at position p turns by p f_i: (a, b) -> A (a cos - b sin, b cos + a sin), (a, b) the
// values (i, i + half) or (2 i, 2 i + 1) of the head's first 2 half, the values behind them as they are. The
// norm is x / sqrt(mean x^2 + eps) w over the whole head. FP32 throughout, one rounding at the store.
//
// Angles. p f_i in FP32 is off by a hundredth of a radian at a position of 10^5, so turns p f_i / (2 pi) are formed in
// 64 bits, less whole quarters, and the rest, at most an eighth of a turn, is exact to FP32's last bit. All heads
// of a row share its angles: a workgroup works them out once, in LDS.
#include "launch.hpp"

namespace smx {
namespace {

struct RotaryArgs {
  const void *x, *positions, *frequencies, *norm;
  void* out;
  int64_t x_token, x_head, out_token, out_head;
  int32_t tokens, heads, dim, half, flags, zero_rows, per_block, heads_each;
  float amplitude, eps;
};

constexpr int kMaxDim = 1024;

// The positions of the workgroup's rows, and the factors of each one's pairs: LDS [rows][half] cos, then sin.
__device__ __forceinline__ void turns(const RotaryArgs& p, int64_t row0, int rows, float* cos, float* sin) {
  for (int i = threadIdx.x; i < rows * p.half; i += blockDim.x) {
    const int row = i / p.half, pair = i - row * p.half;
    const int64_t at = row0 + row;
    const double position = p.flags & SMX_ROTARY_POSITIONS_I64 ? (double)((const int64_t*)p.positions)[at]
                                                               : (double)((const int32_t*)p.positions)[at];
    const double f = p.flags & SMX_ROTARY_FREQUENCIES_F32 ? (double)((const float*)p.frequencies)[pair]
                                                          : ((const double*)p.frequencies)[pair];
    const double turn = position * f * 0.15915494309189533577;  // 1 / (2 pi)
    const double quarters = rint(turn * 4);
    const float rest = (float)(turn - quarters * 0.25);
    // which quarter: quarters mod 4, in 64 bits (a float's turn may pass 2^31)
    const int quarter = (int)(quarters - 4 * floor(quarters * 0.25));
    float s, c;
    sincospif(2 * rest, &s, &c);
    const float a = quarter & 1 ? s : c, b = quarter & 1 ? c : s;
    cos[i] = p.amplitude * (quarter == 1 || quarter == 2 ? -a : a);
    sin[i] = p.amplitude * (quarter >= 2 ? -b : b);
  }
  __syncthreads();
}

__device__ __forceinline__ bool covered(const RotaryArgs& p, int64_t row) {
  return p.flags & SMX_ROTARY_POSITIONS_I64 ? ((const int64_t*)p.positions)[row] >= 0
                                            : ((const int32_t*)p.positions)[row] >= 0;
}

// Sixteen bytes of a head.
template <bool kF32>
struct Run {
  static constexpr int kValues = kF32 ? 4 : 8;
  float v[kValues];

  template <bool kFrom32, bool kOnce = false>
  __device__ __forceinline__ void load(const void* p, int64_t at) {
    if constexpr (kFrom32) {
#pragma unroll
      for (int j = 0; j < kValues / 4; ++j) {
        const f32x4* const from = reinterpret_cast<const f32x4*>((const float*)p + at) + j;
        const f32x4 x = kOnce ? __builtin_nontemporal_load(from) : *from;
#pragma unroll
        for (int i = 0; i < 4; ++i) v[4 * j + i] = x[i];
      }
    } else {
      typedef uint32_t Words __attribute__((ext_vector_type(kValues / 2)));
      const Words* const from = reinterpret_cast<const Words*>((const uint16_t*)p + at);
      const Words x = kOnce ? __builtin_nontemporal_load(from) : *from;
#pragma unroll
      for (int i = 0; i < kValues / 2; ++i) v[2 * i] = lo_f32(x[i]), v[2 * i + 1] = hi_f32(x[i]);
    }
  }
  __device__ __forceinline__ void store(void* p, int64_t at) const {
    if constexpr (kF32) {
      *reinterpret_cast<f32x4*>((float*)p + at) = f32x4{v[0], v[1], v[2], v[3]};
    } else {
      F8 x;
#pragma unroll
      for (int i = 0; i < 8; ++i) x.v[i] = v[i];
      *reinterpret_cast<u32x4*>((uint16_t*)p + at) = pack8(x);
    }
  }
};

// Heads whose values fall into aligned runs of 16 bytes: a lane takes two of them, half of the turned (or of the other)
// values apart, so that a wave's loads are consecutive, and goes from head to head with the next one's on their way (the
// first one's while the angles are worked out). Bound by memory: 302 MB of bf16 in 54 us, 5.5 TB/s, 123 MB of float32 in 24 us,
// 5.2 TB/s (with the runs of a lane next to each other and no loads ahead 32).
template <bool kF32, bool kInterleaved, bool kNorm, bool kOnce>
__global__ __launch_bounds__(256) void rotary_runs(RotaryArgs p) {
  constexpr int kValues = Run<kF32>::kValues;
  extern __shared__ __attribute__((aligned(16))) float rotary_lds[];
  const int64_t row0 = (int64_t)blockIdx.x * p.per_block;
  const int rows = (int)min((int64_t)p.per_block, p.tokens - row0);
  float* const cos = rotary_lds;
  float* const sin = cos + p.per_block * p.half;

  const int turning = p.half / kValues, others = p.dim / kValues - 2 * turning;  // lanes, runs
  const int lanes = turning + (others + 1) / 2, slots = 256 / lanes;
  const int slot = (int)threadIdx.x / lanes, lane = (int)threadIdx.x - slot * lanes;
  const bool turned = lane < turning;
  const int first = turned ? kValues * lane : 2 * p.half + kValues * (lane - turning);
  const int second = first + (turned ? p.half : kValues * ((others + 1) / 2));
  const bool two = second < p.dim;
  const int head0 = blockIdx.y * p.heads_each, heads = min(p.heads_each, p.heads - head0);
  int row = 0, head = slot;
  auto settle = [&] {
    while (head >= heads) head -= heads, ++row;
  };
  settle();
  if (slot >= slots) row = rows;  // (with a norm 256 is a multiple of lanes)
  Run<kF32> wa, wb, a, b;
  auto load = [&] {
    if (row >= rows) return;
    const int64_t from = (row0 + row) * p.x_token + (head0 + head) * p.x_head;
    a.template load<kF32, kOnce>(p.x, from + first);
    if (two) b.template load<kF32, kOnce>(p.x, from + second);
  };
#pragma unroll
  for (int i = 0; i < kValues; ++i) a.v[i] = b.v[i] = 0.f;
  load();
  if constexpr (kNorm) {
    if (p.flags & SMX_ROTARY_NORM_F32) {
      wa.template load<true>(p.norm, first), wb.template load<true>(p.norm, second);
    } else {
      wa.template load<false>(p.norm, first), wb.template load<false>(p.norm, second);
    }
  }
  turns(p, row0, rows, cos, sin);

  while (row < rows) {
    const int64_t token = row0 + row;
    const int64_t to = token * p.out_token + (head0 + head) * p.out_head;
    const int angles = row * p.half;
    Run<kF32> x = a, y = b;
    head += slots;
    settle();
    load();
    if (covered(p, token)) {
      if constexpr (kNorm) {
        float sum = 0.f;
#pragma unroll
        for (int i = 0; i < kValues; ++i) sum += x.v[i] * x.v[i] + y.v[i] * y.v[i];
        for (int d = 1; d < lanes; d <<= 1) sum += __shfl_xor(sum, d);  // a head's lanes stay together in the loop
        const float r = 1.0f / sqrtf(sum / p.dim + p.eps);
#pragma unroll
        for (int i = 0; i < kValues; ++i) x.v[i] = x.v[i] * r * wa.v[i], y.v[i] = y.v[i] * r * wb.v[i];
      }
      if (turned) {
        auto turn = [&](float& u, float& v, int pair) {
          const float c = cos[angles + pair], s = sin[angles + pair], before = u;
          u = before * c - v * s;
          v = v * c + before * s;
        };
        if constexpr (kInterleaved) {
#pragma unroll
          for (int i = 0; i < kValues / 2; ++i) {
            turn(x.v[2 * i], x.v[2 * i + 1], first / 2 + i);
            turn(y.v[2 * i], y.v[2 * i + 1], second / 2 + i);
          }
        } else {
#pragma unroll
          for (int i = 0; i < kValues; ++i) turn(x.v[i], y.v[i], first + i);
        }
      }
    } else {
      if (!p.zero_rows) continue;
#pragma unroll
      for (int i = 0; i < kValues; ++i) x.v[i] = y.v[i] = 0.f;
    }
    x.store(p.out, to + first);
    if (two) y.store(p.out, to + second);
  }
}

// Any other head (outside aligned runs of 16 bytes, or normalised and not a power of two of them wide): a wave takes a head, value by
// value, a workgroup a token. Bound by its instructions and accesses of 2 bytes, not by memory: 8192 tokens of 72 heads of 80
// bf16 values, 40 of them rotated (189 MB), take 132 us, 1.4 TB/s, behind a norm 233, where rotary_runs takes 41 for the same
// heads rotated whole; 4096 tokens of 32 heads 26 us (10), 16 tokens 7.2.
template <bool kF32>
__global__ __launch_bounds__(256) void rotary_values(RotaryArgs p) {
  extern __shared__ __attribute__((aligned(16))) float rotary_lds[];
  const int64_t token = blockIdx.x;
  float* const cos = rotary_lds;
  float* const sin = cos + p.half;
  turns(p, token, 1, cos, sin);
  const int lane = threadIdx.x & 63;
  const bool here = covered(p, token), wide = p.flags & SMX_ROTARY_INTERLEAVED;
  if (!here && !p.zero_rows) return;
  auto load = [&](int64_t at) { return kF32 ? ((const float*)p.x)[at] : bf16_to_f32(((const uint16_t*)p.x)[at]); };
  auto store = [&](int64_t at, float v) {
    if (kF32)
      ((float*)p.out)[at] = v;
    else
      ((uint16_t*)p.out)[at] = f32_to_bf16(v);
  };
  for (int head = threadIdx.x >> 6; head < p.heads; head += 4) {
    const int64_t from = token * p.x_token + head * p.x_head, to = token * p.out_token + head * p.out_head;
    float r = 1.f;
    if (p.norm && here) {
      float sum = 0.f;
      for (int i = lane; i < p.dim; i += 64) {
        const float v = load(from + i);
        sum += v * v;
      }
#pragma unroll
      for (int d = 1; d < 64; d <<= 1) sum += __shfl_xor(sum, d);
      r = 1.0f / sqrtf(sum / p.dim + p.eps);
    }
    auto value = [&](int i) {
      if (!here) return 0.f;
      const float v = load(from + i);
      if (!p.norm) return v;
      return v * r * (p.flags & SMX_ROTARY_NORM_F32 ? ((const float*)p.norm)[i] : bf16_to_f32(((const uint16_t*)p.norm)[i]));
    };
    for (int i = lane; i < p.half; i += 64) {
      const int a = wide ? 2 * i : i, b = wide ? 2 * i + 1 : i + p.half;
      const float u = value(a), v = value(b);
      store(to + a, here ? u * cos[i] - v * sin[i] : 0.f);
      store(to + b, here ? v * cos[i] + u * sin[i] : 0.f);
    }
    for (int i = 2 * p.half + lane; i < p.dim; i += 64) store(to + i, value(i));
  }
}

template <bool kF32, bool kInterleaved>
auto runs_kernel(bool norm, bool once) {
  return norm ? (once ? rotary_runs<kF32, kInterleaved, true, true> : rotary_runs<kF32, kInterleaved, true, false>)
              : (once ? rotary_runs<kF32, kInterleaved, false, true> : rotary_runs<kF32, kInterleaved, false, false>);
}

// Overlap checks count in two-byte units.
Runs runs_of(const smx_heads& x, int64_t tokens, int64_t dim, int units) {
  smx_heads y = x;
  y.token_stride *= units, y.head_stride *= units;
  return head_runs(y, tokens, dim * units);
}

}  // namespace
}  // namespace smx

using namespace smx;

extern "C" {

int smx_rotary(int32_t tokens, int32_t head_dim, int32_t rotary_dim, const smx_heads* x, const smx_heads* out,
               const void* positions, const void* frequencies, const void* norm, int32_t flags, float amplitude,
               float eps, int32_t zero_rows, void* stream) {
  smx::fail(SMX_OK, "%s", "");
  if (!x || !x->data || !out || !out->data || !positions || !frequencies) return fail(SMX_ERR_INVALID, "null pointer");
  if (tokens <= 0 || tokens > SMX_PAGED_MAX_TOKENS)
    return fail(SMX_ERR_INVALID, "1 to %d tokens, got %d", SMX_PAGED_MAX_TOKENS, tokens);
  if (x->heads <= 0 || x->heads > 65535 || out->heads != x->heads)
    return fail(SMX_ERR_INVALID, "1 to 65535 heads, as many out of the call as in (%d, %d)", x->heads, out->heads);
  if (head_dim < 2 || head_dim > kMaxDim) return fail(SMX_ERR_UNSUPPORTED, "head_dim must be 2 to %d, got %d", kMaxDim, head_dim);
  if (rotary_dim < 2 || rotary_dim > head_dim || rotary_dim % 2)
    return fail(SMX_ERR_INVALID, "an even number of values, at most head_dim=%d, are rotated, got %d", head_dim, rotary_dim);
  constexpr int32_t kFlags = SMX_ROTARY_F32 | SMX_ROTARY_NORM_F32 | SMX_ROTARY_FREQUENCIES_F32 | SMX_ROTARY_POSITIONS_I64 |
                             SMX_ROTARY_INTERLEAVED;
  if (flags & ~kFlags) return fail(SMX_ERR_INVALID, "unknown flags 0x%x", flags);
  if (!(amplitude >= -3e38f && amplitude <= 3e38f)) return fail(SMX_ERR_INVALID, "amplitude must be finite");
  if (!(eps >= 0.f)) return fail(SMX_ERR_INVALID, "eps must not be negative");
  const int size = flags & SMX_ROTARY_F32 ? 4 : 2;
  for (const smx_heads* h : {x, out})
    if ((uintptr_t)h->data % size || h->token_stride < 0 || h->head_stride < 0)
      return fail(SMX_ERR_INVALID, "misaligned heads or negative strides");
  const auto misaligned = [](const void* q, int bytes) { return (uintptr_t)q % bytes != 0; };
  if (misaligned(positions, flags & SMX_ROTARY_POSITIONS_I64 ? 8 : 4) ||
      misaligned(frequencies, flags & SMX_ROTARY_FREQUENCIES_F32 ? 4 : 8) || misaligned(norm, flags & SMX_ROTARY_NORM_F32 ? 4 : 2))
    return fail(SMX_ERR_INVALID, "misaligned positions, frequencies or norm");
  // Heads are stored while others are loaded.
  const Runs from = runs_of(*x, tokens, head_dim, size / 2), to = runs_of(*out, tokens, head_dim, size / 2);
  if (!lie_apart(to)) return fail(SMX_ERR_INVALID, "out holds rows that lie on each other");
  if (!same_runs(from, to) && meet(from, to))
    return fail(SMX_ERR_INVALID, "out must be x itself or share no memory with it");
  // ... and read beside positions, frequencies and norm, by every workgroup for itself.
  const auto list = [](const void* at, int64_t count, int bytes) { return Runs{at, count * (bytes / 2), {{1, 0}, {1, 0}, {1, 0}}}; };
  if (meet(to, list(positions, tokens, flags & SMX_ROTARY_POSITIONS_I64 ? 8 : 4)) ||
      meet(to, list(frequencies, rotary_dim / 2, flags & SMX_ROTARY_FREQUENCIES_F32 ? 4 : 8)) ||
      (norm && meet(to, list(norm, head_dim, flags & SMX_ROTARY_NORM_F32 ? 4 : 2))))
    return fail(SMX_ERR_INVALID, "out must share no memory with positions, frequencies and norm");
  RotaryArgs p{};
  p.x = x->data, p.out = out->data, p.positions = positions, p.frequencies = frequencies, p.norm = norm;
  p.x_token = x->token_stride, p.x_head = x->head_stride, p.out_token = out->token_stride, p.out_head = out->head_stride;
  p.tokens = tokens, p.heads = x->heads, p.dim = head_dim, p.half = rotary_dim / 2, p.flags = flags;
  p.zero_rows = zero_rows, p.amplitude = amplitude, p.eps = eps;
  const int run = 16 / size;  // values of 16 bytes
  bool aligned = p.half % run == 0 && head_dim % run == 0 && !misaligned(norm, 16);
  for (const smx_heads* h : {x, out}) aligned = aligned && !misaligned(h->data, 16) && h->token_stride % run == 0 && h->head_stride % run == 0;
  // a norm's sum goes over the lanes of a head, a power of two of them in a wave
  if (norm) aligned = aligned && head_dim >= 2 * run && head_dim <= 128 * run && !(head_dim & (head_dim - 1));
  if (!aligned) {
    p.per_block = 1;
    hipLaunchKernelGGL(flags & SMX_ROTARY_F32 ? rotary_values<true> : rotary_values<false>, dim3((unsigned)tokens), dim3(256),
                       2 * p.half * 4, (hipStream_t)stream, p);
    return check_launch();
  }
  // Rows of a workgroup: several where enough workgroups remain to fill the chip (72 heads of 128, three sets of them in turn; one,
  // two and four rows: 14.2, 14.3 and 14.0 us for 2045 tokens, 53, 52 and 51 for 8192).
  p.per_block = tokens >= 4096 ? 4 : tokens >= 1536 ? 2 : 1;
  const unsigned blocks = (unsigned)((tokens + p.per_block - 1) / p.per_block);
  // Of few tokens a row's heads are shared out, as many to a workgroup as it takes at once (72 heads of 128 without a norm; shared
  // and not, in the kernel: 4.0 and 5.3 us for 16 tokens, 5.7 and 6.4 for 400, 9.7 and 9.0 for 1000).
  const int turning = p.half / run, lanes = turning + (head_dim / run - 2 * turning + 1) / 2;
  p.heads_each = blocks <= 512 ? min(p.heads, max(1, 256 / lanes)) : p.heads;
  const int lds = 2 * p.per_block * p.half * 4;
  // Heads that do not fit into the caches (256 MB) together with the result leave them to the result, which is read next: 302 MB in
  // calls one behind another 54 us (else 65), 270 MB 47 (58); but 80 MB, which fit, 24 (21).
  const bool once = x->data != out->data && 2 * (int64_t)size * tokens * p.heads * head_dim > (int64_t)200 << 20;
  const bool wide = flags & SMX_ROTARY_INTERLEAVED;
  auto kern = flags & SMX_ROTARY_F32 ? (wide ? runs_kernel<true, true>(norm, once) : runs_kernel<true, false>(norm, once))
                                     : (wide ? runs_kernel<false, true>(norm, once) : runs_kernel<false, false>(norm, once));
  hipLaunchKernelGGL(kern, dim3(blocks, (unsigned)((p.heads + p.heads_each - 1) / p.heads_each)), dim3(256), lds, (hipStream_t)stream, p);
  return check_launch();
}

}  // extern "C"
