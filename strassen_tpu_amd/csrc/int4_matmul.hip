// Products of few rows with 4-bit weights (smx_int4_matmul): y = x W with
// W[k, n] = (code[k, n] - zero[k / group, n]) scale[k / group, n], and the fused
// epilogues of the other products.
//
// Mathematics. A code q placed at bits 3 .. 6 of the bf16 pattern of 16.0 is the bf16
// number 16 + q, exactly, so a weight becomes an MFMA operand with half a shift and
// half an and-or. Per group
//   sum_k x_k (q_k - z) = sum_k x_k (16 + q_k) - (16 + z) sum_k x_k,
// whose second term starts the accumulator (sum_k x_k is one more MFMA, against
// ones, shared by all columns of the wave), and the group's scale multiplies the
// FP32 sum: no product is rounded before the end.
//
// Layout. Columns in tiles of 16, K in tiles of 128: one tile is 1 KB, lane l
// of a wave reads its 16 bytes as the MFMA's A operand wants them (column l % 16; word s:
// the 8 codes of k = 32 s + 8 (l / 16) .. + 7). With smx_int4's "swiglu" layout
// tiles alternate between gate and up columns. Beside them one word a group and column: the
// bf16 scale above, -(16 + zero) in bf16 below.
//
// Bound by the weight's bytes from HBM: a wave holds kDepth K tiles of kCols column
// tiles in flight, and the waves of a workgroup take K tiles in turn, so that a projection of few
// columns fills the chip too. Their sums meet in LDS, in wave order.
#include "kernel_packed.hpp"
#include "launch.hpp"

namespace smx {
namespace {

struct Int4Args {
  const uint16_t* x;
  int64_t ldx;
  const u32x4* codes;
  const u32x4* scales;  // [column tiles][groups of K][4 x 4 columns]
  uint16_t* out;
  int64_t ldo;
  const void* extra;  // residual [m, n] or bias [n]
  int64_t lde;
  int32_t m, n, k, k_tiles, epilogue, extra_f32;
};

__device__ __forceinline__ bf16x8 widen(uint32_t w) {
  constexpr uint32_t kMask = 0x00780078, kSixteen = 0x41804180;
  const u32x4 v = {((w << 3) & kMask) | kSixteen, ((w >> 1) & kMask) | kSixteen, ((w >> 5) & kMask) | kSixteen,
                   ((w >> 9) & kMask) | kSixteen};
  return __builtin_bit_cast(bf16x8, v);
}

// One value of the epilogue's operand.
__device__ __forceinline__ float extra_at(const Int4Args& p, int64_t row, int32_t col) {
  const int64_t at = p.epilogue == SMX_EPI_BIAS_ADD ? col : row * p.lde + col;
  return p.extra_f32 ? reinterpret_cast<const float*>(p.extra)[at]
                     : bf16_to_f32(reinterpret_cast<const uint16_t*>(p.extra)[at]);
}

__device__ __forceinline__ f32x4 add4(f32x4 a, f32x4 b) { return f32x4{a[0] + b[0], a[1] + b[1], a[2] + b[2], a[3] + b[3]}; }

// kRows row tiles of 16, kCols column tiles, kWaves waves that divide K, kGroups
// scale groups in a K tile of 128.
template <int kRows, int kCols, int kWaves, int kGroups>
__global__ __launch_bounds__(kWaves * 64) void int4_matmul(Int4Args p) {
  constexpr int kSteps = 4 / kGroups;  // MFMA steps of 32 in a group
  extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), quad = lane >> 4;
  const int64_t tile0 = (int64_t)blockIdx.x * kCols;
  const int row0 = blockIdx.y * (16 * kRows);

  const uint16_t* x_row[kRows];
#pragma unroll
  for (int r = 0; r < kRows; ++r) x_row[r] = p.x + min(row0 + 16 * r + (lane & 15), p.m - 1) * p.ldx + 8 * quad;

  struct Stage {
    u32x4 codes[kCols], scales[kCols][kGroups];
  };
  struct Rows {
    u32x4 x[kRows][4];
  };
  auto load = [&](Stage& s, int kt) __attribute__((always_inline)) {
#pragma unroll
    for (int c = 0; c < kCols; ++c) {
      s.codes[c] = __builtin_nontemporal_load(p.codes + ((tile0 + c) * p.k_tiles + kt) * 64 + lane);
#pragma unroll
      for (int g = 0; g < kGroups; ++g)
        s.scales[c][g] = p.scales[((tile0 + c) * p.k_tiles + kt) * (4 * kGroups) + 4 * g + quad];
    }
  };
  auto load_rows = [&](Rows& s, int kt) __attribute__((always_inline)) {
    const bool whole = (kt + 1) * 128 <= p.k;
#pragma unroll
    for (int r = 0; r < kRows; ++r)
#pragma unroll
      for (int t = 0; t < 4; ++t)
        s.x[r][t] = whole || kt * 128 + 32 * t < p.k
                        ? *reinterpret_cast<const u32x4*>(x_row[r] + (int64_t)kt * 128 + 32 * t)
                        : u32x4{0, 0, 0, 0};
  };

  f32x4 acc[kCols][kRows];
#pragma unroll
  for (int c = 0; c < kCols; ++c)
#pragma unroll
    for (int r = 0; r < kRows; ++r) acc[c][r] = f32x4{0.f, 0.f, 0.f, 0.f};
  const bf16x8 ones = __builtin_bit_cast(bf16x8, u32x4{0x3f803f80, 0x3f803f80, 0x3f803f80, 0x3f803f80});

  auto multiply = [&](const Stage& s, const Rows& x) __attribute__((always_inline)) {
#pragma unroll
    for (int g = 0; g < kGroups; ++g) {
      f32x4 sum[kRows];
#pragma unroll
      for (int r = 0; r < kRows; ++r) {
        sum[r] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int t = 0; t < kSteps; ++t)
          sum[r] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(
              ones, __builtin_bit_cast(bf16x8, x.x[r][g * kSteps + t]), sum[r], 0, 0, 0);
      }
#pragma unroll
      for (int c = 0; c < kCols; ++c) {
        f32x4 part[kRows];
#pragma unroll
        for (int r = 0; r < kRows; ++r)
#pragma unroll
          for (int i = 0; i < 4; ++i) part[r][i] = lo_f32(s.scales[c][g][i]) * sum[r][i];
#pragma unroll
        for (int t = 0; t < kSteps; ++t) {
          const bf16x8 a = widen(s.codes[c][g * kSteps + t]);
#pragma unroll
          for (int r = 0; r < kRows; ++r)
            part[r] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(
                a, __builtin_bit_cast(bf16x8, x.x[r][g * kSteps + t]), part[r], 0, 0, 0);
        }
#pragma unroll
        for (int r = 0; r < kRows; ++r)
#pragma unroll
          for (int i = 0; i < 4; ++i) acc[c][r][i] = __builtin_fmaf(hi_f32(s.scales[c][g][i]), part[r][i], acc[c][r][i]);
      }
    }
  };

  // Two stages: the next K tile's codes are on their way while one is multiplied
  // (with one row tile its rows of x too; more of them would not leave the registers for
  // it). Past the last tile the last is read again, unused.
  constexpr bool kAhead = kRows == 1;
  Stage a, b;
  Rows xa, xb;
  const int last = p.k_tiles - 1;
  if (wave <= last) {
    load(a, wave);
    if (kAhead) load_rows(xa, wave);
    for (int kt = wave; kt <= last; kt += 2 * kWaves) {
      if (!kAhead) load_rows(xa, kt);
      load(b, min(kt + kWaves, last));
      if (kAhead) load_rows(xb, min(kt + kWaves, last));
      multiply(a, xa);
      if (kt + kWaves > last) break;
      if (!kAhead) load_rows(xb, kt + kWaves);
      load(a, min(kt + 2 * kWaves, last));
      if (kAhead) load_rows(xa, min(kt + 2 * kWaves, last));
      multiply(b, xb);
    }
  }

  // The waves' sums, lane l of tile (c, r) holding columns 4 (l / 16) .. + 3 of row l % 16.
  f32x4* const sums = reinterpret_cast<f32x4*>(lds);
  constexpr int kItems = kCols * kRows * 64;
#pragma unroll
  for (int c = 0; c < kCols; ++c)
#pragma unroll
    for (int r = 0; r < kRows; ++r) sums[wave * kItems + (c * kRows + r) * 64 + lane] = acc[c][r];
  __syncthreads();
  auto total = [&](int item) {
    f32x4 s = sums[item];
#pragma unroll
    for (int w = 1; w < kWaves; ++w) s = add4(s, sums[w * kItems + item]);
    return s;
  };
  const bool gated = p.epilogue == SMX_EPI_SWIGLU;
  for (int item = threadIdx.x; item < (gated ? kItems / 2 : kItems); item += kWaves * 64) {
    const int in = item & 63, r = (item >> 6) % kRows, c = (item >> 6) / kRows;
    const int row = row0 + 16 * r + (in & 15);
    f32x4 y;
    int64_t col;
    if (gated) {
      const f32x4 gate = total((2 * c * kRows + r) * 64 + in), up = total(((2 * c + 1) * kRows + r) * 64 + in);
#pragma unroll
      for (int i = 0; i < 4; ++i) y[i] = gate[i] / (1.f + __expf(-gate[i])) * up[i];
      col = (tile0 / 2 + c) * 16 + 4 * (in >> 4);
    } else {
      y = total((c * kRows + r) * 64 + in);
      col = (tile0 + c) * 16 + 4 * (in >> 4);
    }
    if (row >= p.m || col >= p.n) continue;
    const int count = (int)min((int64_t)4, p.n - col);
    if (p.extra)
      for (int i = 0; i < count; ++i) y[i] += extra_at(p, row, (int32_t)col + i);
    uint16_t* const to = p.out + row * p.ldo + col;
    if (count == 4 && p.ldo % 4 == 0) {
      *reinterpret_cast<uint2*>(to) = make_uint2(pack_bf16(y[0], y[1]), pack_bf16(y[2], y[3]));
    } else {
      for (int i = 0; i < count; ++i) to[i] = f32_to_bf16(y[i]);
    }
  }
}

template <int kRows, int kCols, int kWaves, int kGroups>
int launch_shape(const Int4Args& p, int64_t column_tiles, hipStream_t stream) {
  constexpr int lds = kWaves * kCols * kRows * 1024;
  auto kern = int4_matmul<kRows, kCols, kWaves, kGroups>;
  hipError_t e = hipFuncSetAttribute((const void*)kern, hipFuncAttributeMaxDynamicSharedMemorySize, lds);
  if (e != hipSuccess) return fail(SMX_ERR_LAUNCH, "hipFuncSetAttribute: %s", hipGetErrorString(e));
  const unsigned rows = (unsigned)((p.m + 16 * kRows - 1) / (16 * kRows));
  hipLaunchKernelGGL(kern, dim3((unsigned)(column_tiles / kCols), rows), dim3(kWaves * 64), lds, stream, p);
  return check_launch();
}

template <int kGroups>
int launch_int4(const Int4Args& p, int64_t column_tiles, hipStream_t s) {
  if (p.m <= 16) return launch_shape<1, 2, 8, kGroups>(p, column_tiles, s);
  if (p.m <= 32) return launch_shape<2, 2, 8, kGroups>(p, column_tiles, s);
  return launch_shape<4, 2, 8, kGroups>(p, column_tiles, s);
}

}  // namespace
}  // namespace smx

using namespace smx;

extern "C" int smx_int4_matmul(const smx_int4_weight* w, int64_t m, const void* x, int64_t ldx, int32_t epilogue,
                               const void* extra, int64_t lde, int32_t extra_f32, void* out, int64_t ldo,
                               void* stream) {
  smx::fail(SMX_OK, "%s", "");
  if (!w || !w->codes || !w->scales || !x || !out) return fail(SMX_ERR_INVALID, "null pointer");
  if (m <= 0 || m > SMX_PAGED_MAX_TOKENS) return fail(SMX_ERR_INVALID, "1 to %d rows, got %lld", SMX_PAGED_MAX_TOKENS, (long long)m);
  if (w->k <= 0 || w->k > (1 << 24) || w->n <= 0 || w->n > (1 << 24) || w->k % 32)
    return fail(SMX_ERR_INVALID, "k must be a multiple of 32, k and n at most 2^24 (k=%lld, n=%lld)", (long long)w->k,
                (long long)w->n);
  if (w->group != 32 && w->group != 64 && w->group != 128)
    return fail(SMX_ERR_INVALID, "group must be 32, 64 or 128, got %d", w->group);
  const bool gated = epilogue == SMX_EPI_SWIGLU;
  if (epilogue != SMX_EPI_NONE && !gated && epilogue != SMX_EPI_RESIDUAL_ADD && epilogue != SMX_EPI_BIAS_ADD)
    return fail(SMX_ERR_UNSUPPORTED, "epilogue %d is not one of the 4-bit product's", epilogue);
  if (gated != (w->swiglu != 0)) return fail(SMX_ERR_INVALID, "the weight's layout is not that of the epilogue");
  if (gated && w->n % 2) return fail(SMX_ERR_INVALID, "[gate | up] has an even width, got %lld", (long long)w->n);
  const bool takes = epilogue == SMX_EPI_RESIDUAL_ADD || epilogue == SMX_EPI_BIAS_ADD;
  if (takes != (extra != nullptr)) return fail(SMX_ERR_INVALID, "residual or bias go with their epilogue");
  const int64_t n = gated ? w->n / 2 : w->n;
  if (ldx < w->k || ldx % 8 || (uintptr_t)x % 16) return fail(SMX_ERR_INVALID, "x rows must be 16-byte aligned, >= k");
  if (ldo < n || (uintptr_t)out % 8) return fail(SMX_ERR_INVALID, "out rows must hold n values, 8-byte aligned");
  if (epilogue == SMX_EPI_RESIDUAL_ADD && lde < n) return fail(SMX_ERR_INVALID, "residual rows must hold n values");
  if ((uintptr_t)w->codes % 16 || (uintptr_t)w->scales % 16)
    return fail(SMX_ERR_INVALID, "codes and scales must be 16-byte aligned");
  Int4Args p{};
  p.x = (const uint16_t*)x, p.ldx = ldx;
  p.codes = (const u32x4*)w->codes, p.scales = (const u32x4*)w->scales;
  p.out = (uint16_t*)out, p.ldo = ldo, p.extra = extra, p.lde = lde, p.extra_f32 = extra_f32;
  p.m = (int32_t)m, p.n = (int32_t)n, p.k = (int32_t)w->k, p.k_tiles = (int32_t)((w->k + 127) / 128);
  p.epilogue = epilogue;
  // column tiles, whole pairs of them (the layout pads with columns of scale 0)
  const int64_t column_tiles = gated ? 2 * ((n + 15) / 16) : 2 * ((n + 31) / 32);
  if (w->group == 128) return launch_int4<1>(p, column_tiles, (hipStream_t)stream);
  if (w->group == 64) return launch_int4<2>(p, column_tiles, (hipStream_t)stream);
  return launch_int4<4>(p, column_tiles, (hipStream_t)stream);
}
