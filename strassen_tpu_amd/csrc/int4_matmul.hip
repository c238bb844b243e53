// Products of few rows with 4-bit weights (smx_int4_matmul): y = x W with
// W[k, n] = (code[k, n] - zero[k / group, n]) scale[k / group, n], and the fused
// epilogues of the other products.
//
// Mathematics. A code q placed at bits 3 .. 6 of the bf16 pattern of 16.0 is the bf16
// number 16 + q, exactly, so a weight becomes an MFMA operand with half a shift and
// half an and-or. Per group
//   sum_k x_k (q_k - z) = sum_k x_k (16 + q_k) - (16 + z) sum_k x_k,
// whose second sum is one more MFMA, against ones, shared by all columns of the wave, and
// the group's scale multiplies the FP32 sum of both: no product is rounded before the end. (Both sums
// stay below 128 * 31 |x| < 2^127 for |x| up to 2^115; larger values may overflow.) Without zero
// points (z = 8) that MFMA is against -24 and the products start from its result (61 rows of a 5120 x
// 8192 weight in groups of 32: 18.8 us, with the multiply-adds 20.6).
//
// Layout. Columns in tiles of 16, K in tiles of 128: one tile is 1 KB, lane l
// of a wave reads its 16 bytes as the MFMA's A operand wants them (column l % 16; word s:
// the 8 codes of k = 32 s + 8 (l / 16) .. + 7). With smx_int4's "swiglu" layout
// tiles alternate between gate and up columns. Beside them one word a group and column: the
// bf16 scale above, -(16 + zero) in bf16 below.
//
// Two kernels, both bound by the weight's bytes from HBM where rows are few. int4_few keeps all rows of
// x in LDS where they fit and divides K among the waves of a workgroup; int4_tiled streams x through LDS
// in stages that four waves side by side share, and divides K among workgroups, whose FP32
// sums int4_join adds up. Direct loads of x instead would cost the address units as much per
// 16 rows as four column tiles of codes (gate|up of 16 rows: 49 us, 29 without them).
#include "kernel_packed.hpp"
#include "launch.hpp"

namespace smx {
namespace {

struct Int4Args {
  const uint16_t* x;
  int64_t ldx;
  const u32x4* codes;
  const uint32_t* scales;  // [column tiles][K tiles][16 columns][groups of the K tile]
  uint16_t* out;
  int64_t ldo;
  const void* extra;  // residual [m, n] or bias [n]
  int64_t lde;
  int32_t m, n, k, k_tiles, tiles, epilogue, extra_f32;
  int32_t share;   // K tiles of a workgroup of int4_tiled
  float* partial;  // [shares][m][16 tiles] FP32 sums, if there are several
};

// Eight codes to bf16: pair i at bits 4 i + 3 .. + 6 and 4 i + 19 .. + 22 (the last wraps
// around), moved to bits 3 and 19 and joined with 16.0 by one v_and_or_b32. That instruction
// takes no literals: the constants come in registers.
struct Widen {
  uint32_t mask = 0x00780078, sixteen = 0x41804180;
  __device__ __forceinline__ Widen() { asm("" : "+s"(mask), "+v"(sixteen)); }
  __device__ __forceinline__ bf16x8 operator()(uint32_t w) const {
    const u32x4 v = {(w & mask) | sixteen, ((w >> 4) & mask) | sixteen, ((w >> 8) & mask) | sixteen,
                     (__builtin_amdgcn_alignbit(w, w, 12) & mask) | sixteen};
    return __builtin_bit_cast(bf16x8, v);
  }
};

// One value of the epilogue's operand.
__device__ __forceinline__ float extra_at(const Int4Args& p, int64_t row, int32_t col) {
  const int64_t at = p.epilogue == SMX_EPI_BIAS_ADD ? col : row * p.lde + col;
  return p.extra_f32 ? reinterpret_cast<const float*>(p.extra)[at]
                     : bf16_to_f32(reinterpret_cast<const uint16_t*>(p.extra)[at]);
}

// The value of lane kLane of each row of 16 lanes.
template <int kLane>
__device__ __forceinline__ float row_lane(float x) {
  const int v = __builtin_bit_cast(int, x);
  return __builtin_bit_cast(float, __builtin_amdgcn_mov_dpp(v, 0x150 + kLane, 15, 15, true));
}

// The four columns of a quad, of group kGroup.
template <int kGroups, int kGroup>
__device__ __forceinline__ f32x4 quad_columns(float x) {
  return f32x4{row_lane<kGroup>(x), row_lane<kGroups + kGroup>(x), row_lane<2 * kGroups + kGroup>(x),
               row_lane<3 * kGroups + kGroup>(x)};
}

// One K tile's codes and scales of a wave's kCols column tiles.
template <int kCols>
struct Codes {
  u32x4 codes[kCols];
  uint32_t scales[kCols];  // lane j of a quad's 16: column j / kGroups % 4, group j % kGroups
};

// A wave's column tiles as buffers that end with their last K tile: later ones load
// zeros, without memory traffic. Offsets past the end are cut to the end itself, so that no
// sum of offsets wraps.
template <int kCols, int kGroups>
struct Columns {
  __amdgpu_buffer_rsrc_t codes[kCols], scales[kCols];
  uint32_t code_at, scale_at;
  int k_tiles;

  __device__ __forceinline__ Columns(const Int4Args& p, int64_t tile0) : k_tiles(p.k_tiles) {
    const int lane = threadIdx.x & 63;
    const uint32_t code_bytes = (uint32_t)p.k_tiles * 1024, scale_bytes = (uint32_t)p.k_tiles * (64 * kGroups);
#pragma unroll
    for (int c = 0; c < kCols; ++c) {
      const int64_t tile = tile0 + c < p.tiles ? tile0 + c : 0;
      const bool here = tile0 + c < p.tiles;
      codes[c] = packed::panel_rsrc(reinterpret_cast<const uint8_t*>(p.codes) + tile * code_bytes, here ? code_bytes : 0);
      scales[c] = packed::panel_rsrc(reinterpret_cast<const uint8_t*>(p.scales) + tile * scale_bytes, here ? scale_bytes : 0);
    }
    code_at = lane * 16;
    scale_at = ((lane >> 4) * 4 * kGroups + (lane & (4 * kGroups - 1))) * 4;
  }

  __device__ __forceinline__ void load(Codes<kCols>& s, int at) const {
    const int kt = min(at, k_tiles);
#pragma unroll
    for (int c = 0; c < kCols; ++c) {
      s.codes[c] = __builtin_amdgcn_raw_buffer_load_b128(codes[c], code_at, kt * 1024, 2);  // 2: non-temporal
      s.scales[c] = __builtin_amdgcn_raw_buffer_load_b32(scales[c], scale_at, kt * (64 * kGroups), 2);
    }
  }
};

// acc += one K tile. x[r][t]: 16 rows of step t (32 of k) as the MFMA's B operand, lane l
// holding row l % 16, k = 8 (l / 16) .. + 7; acc[c][r]: lane l's columns 4 (l / 16) .. + 3 of row l % 16.
template <int kRows, int kCols, int kGroups, bool kZeros>
__device__ __forceinline__ void multiply(f32x4 (&acc)[kCols][kRows], const Codes<kCols>& s, const u32x4 (&x)[kRows][4],
                                         const Widen& widen) {
  constexpr int kSteps = 4 / kGroups;  // MFMA steps of 32 in a group
  // sum: of x against ones, or without zero points against -24 = -(16 + 8), from which the products start
  constexpr uint32_t kOnes = kZeros ? 0x3f803f80 : 0xc1c0c1c0;
  const bf16x8 ones = __builtin_bit_cast(bf16x8, u32x4{kOnes, kOnes, kOnes, kOnes});
  auto group = [&](auto index) __attribute__((always_inline)) {
    constexpr int g = decltype(index)::value;
    f32x4 sum[kRows];
#pragma unroll
    for (int r = 0; r < kRows; ++r) {
      sum[r] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int t = 0; t < kSteps; ++t)
        sum[r] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(ones, __builtin_bit_cast(bf16x8, x[r][g * kSteps + t]), sum[r], 0, 0, 0);
    }
#pragma unroll
    for (int c = 0; c < kCols; ++c) {
      f32x4 part[kRows];
#pragma unroll
      for (int r = 0; r < kRows; ++r) part[r] = kZeros ? f32x4{0.f, 0.f, 0.f, 0.f} : sum[r];
#pragma unroll
      for (int t = 0; t < kSteps; ++t) {
        const bf16x8 a = widen(s.codes[c][g * kSteps + t]);
#pragma unroll
        for (int r = 0; r < kRows; ++r)
          part[r] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, __builtin_bit_cast(bf16x8, x[r][g * kSteps + t]), part[r], 0, 0, 0);
      }
      const f32x4 scale = quad_columns<kGroups, g>(hi_f32(s.scales[c]));
      if constexpr (kZeros) {
        const f32x4 zero = quad_columns<kGroups, g>(lo_f32(s.scales[c]));
#pragma unroll
        for (int r = 0; r < kRows; ++r)
#pragma unroll
          for (int i = 0; i < 4; ++i) part[r][i] = __builtin_fmaf(zero[i], sum[r][i], part[r][i]);
      }
#pragma unroll
      for (int r = 0; r < kRows; ++r)
#pragma unroll
        for (int i = 0; i < 4; ++i) acc[c][r][i] = __builtin_fmaf(scale[i], part[r][i], acc[c][r][i]);
    }
  };
  group(std::integral_constant<int, 0>{});
  if constexpr (kGroups > 1) group(std::integral_constant<int, 1>{});
  if constexpr (kGroups > 2) {
    group(std::integral_constant<int, 2>{});
    group(std::integral_constant<int, 3>{});
  }
}

__device__ __forceinline__ f32x4 gate4(f32x4 gate, f32x4 up) {
  f32x4 y;
#pragma unroll
  for (int i = 0; i < 4; ++i) y[i] = gate[i] / (1.f + __expf(-gate[i])) * up[i];
  return y;
}

// The epilogue's operand, and columns col .. col + 3 of one output row.
__device__ __forceinline__ void finish4(const Int4Args& p, int64_t row, int64_t col, f32x4 y) {
  if (row >= p.m || col >= p.n) return;
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

// Up to 16 rows: kWaves waves take the K tiles of kCols column tiles in turn, and their sums meet
// in LDS in wave order. kStaged: all of x goes to LDS first ([rows][k tiles of 128, padded by
// 16 bytes]), where a wave's 16 lanes of a quad read the same row's bytes at once. Else a wave
// loads its K tile's rows itself, one tile ahead.
template <int kCols, int kWaves, bool kStaged, int kGroups, bool kZeros>
__global__ __launch_bounds__(kWaves * 64) void int4_few(Int4Args p) {
  extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
  const int lane = threadIdx.x & 63, quad = lane >> 4, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t tile0 = (int64_t)blockIdx.x * kCols;
  const Columns<kCols, kGroups> columns(p, tile0);
  const Widen widen;
  f32x4 acc[kCols][1];
#pragma unroll
  for (int c = 0; c < kCols; ++c) acc[c][0] = f32x4{0.f, 0.f, 0.f, 0.f};
  Codes<kCols> s[2];
  columns.load(s[0], wave);
  columns.load(s[1], wave + kWaves);

  const uint32_t row_bytes = p.k_tiles * 256 + 16;
  if constexpr (kStaged) {
    for (int r = 0; r < p.m; ++r)
      for (uint32_t at = threadIdx.x * 16; at < (uint32_t)p.k_tiles * 256; at += kWaves * 64 * 16)
        *reinterpret_cast<u32x4*>(lds + r * row_bytes + at) =
            at < (uint32_t)p.k * 2 ? *reinterpret_cast<const u32x4*>(p.x + r * p.ldx + at / 2) : u32x4{0, 0, 0, 0};
    __syncthreads();
  }
  const uint8_t* const mine = lds + min(lane & 15, p.m - 1) * row_bytes + 16 * quad;
  // rows behind m, and k behind the last, lie behind the buffer's end: zeros, without memory traffic
  const uint32_t x_bytes = (uint32_t)(((p.m - 1) * p.ldx + p.k) * 2);
  const auto x_rsrc = packed::panel_rsrc(reinterpret_cast<const uint8_t*>(p.x), x_bytes);
  const uint32_t x_at = (lane & 15) < p.m ? (uint32_t)((lane & 15) * p.ldx + 8 * quad) * 2 : ~0u;
  auto rows_of = [&](u32x4 (&x)[1][4], int kt) __attribute__((always_inline)) {
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      if constexpr (kStaged)
        x[0][t] = *reinterpret_cast<const u32x4*>(mine + kt * 256 + 64 * t);
      else
        x[0][t] = __builtin_amdgcn_raw_buffer_load_b128(x_rsrc, x_at,
                                                        kt * 128 + 32 * t < p.k ? (uint32_t)(kt * 256 + 64 * t) : x_bytes, 0);
    }
  };
  u32x4 x[2][1][4];
  if (!kStaged) rows_of(x[0], wave);
  for (int kt = wave; kt < p.k_tiles; kt += 2 * kWaves) {
#pragma unroll
    for (int d = 0; d < 2; ++d) {
      const int at = kt + d * kWaves;
      if (at >= p.k_tiles) break;
      if (kStaged) rows_of(x[0], at); else rows_of(x[d ^ 1], at + kWaves);
      multiply<1, kCols, kGroups, kZeros>(acc, s[d], x[kStaged ? 0 : d], widen);
      columns.load(s[d], at + 2 * kWaves);
      __builtin_amdgcn_sched_barrier(0);
    }
  }

  __syncthreads();
  f32x4* const sums = reinterpret_cast<f32x4*>(lds);
#pragma unroll
  for (int c = 0; c < kCols; ++c) sums[(wave * kCols + c) * 64 + lane] = acc[c][0];
  __syncthreads();
  auto total = [&](int c, int in) {
    f32x4 y = sums[c * 64 + in];
#pragma unroll
    for (int w = 1; w < kWaves; ++w) {
      const f32x4 v = sums[(w * kCols + c) * 64 + in];
#pragma unroll
      for (int i = 0; i < 4; ++i) y[i] += v[i];
    }
    return y;
  };
  if (kCols == 2 && p.epilogue == SMX_EPI_SWIGLU) {
    if (threadIdx.x < 64) finish4(p, lane & 15, tile0 * 8 + 4 * quad, gate4(total(0, lane), total(kCols - 1, lane)));
  } else if (threadIdx.x < kCols * 64) {
    finish4(p, lane & 15, (tile0 + wave) * 16 + 4 * quad, total(wave, lane));
  }
}

// Any number of rows, 16 kRows of them a workgroup of 128 columns: four waves side by side, of two
// column tiles each, times kWays that take the K tiles of a stage, one each. All share the stage's
// rows of x in LDS (brought by DMA, kRing stages around); a row's 16-byte chunks are XORed with
// its low bits, so that 8 rows of one chunk lie on different banks. Codes go to registers. A K
// tile is a chain of MFMAs and vector work that fills a quarter to half of a SIMD, which the
// ways overlap; two of them leave room for two workgroups a CU (16 rows of a 5120 x
// 51200 weight: 32.0 us, with four ways 34.7; 61 rows: 57, with one way 81). blockIdx: columns, shares
// of K, row blocks.
template <int kRows>
struct Ring {
  static constexpr int kWays = 2, kRing = kRows == 1 ? 4 : 3;
  static constexpr int kThreads = 256 * kWays, kTileBytes = kRows * 4096, kStage = kWays * kTileBytes;
  static constexpr int kDmas = kRows;      // a wave's for one stage, of 1 KB
  static constexpr int kLoads = 4 + kDmas;  // and its codes and scales
  static constexpr int kLds = kRing * kStage > kWays * 8 * kRows * 1024 ? kRing * kStage : kWays * 8 * kRows * 1024;
};

template <int kRows, int kGroups, bool kZeros>
__global__ __launch_bounds__(Ring<kRows>::kThreads) void int4_tiled(Int4Args p) {
  using R = Ring<kRows>;
  constexpr int kWays = R::kWays, kRing = R::kRing;
  extern __shared__ __attribute__((aligned(1024))) uint8_t lds[];
  const int lane = threadIdx.x & 63, quad = lane >> 4, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int side = wave % 4, way = wave / 4;
  const int64_t group0 = (int64_t)blockIdx.x * 8, tile0 = group0 + side * 2;
  const int row0 = blockIdx.z * (16 * kRows), rows = min(16 * kRows, p.m - row0);
  const int first = blockIdx.y * p.share, last = min(first + p.share, p.k_tiles);  // K tiles
  const Columns<2, kGroups> columns(p, tile0);
  const Widen widen;

  // A DMA brings four rows of a K tile; rows behind m lie behind the buffer's end
  const uint32_t x_bytes = (uint32_t)(((rows - 1) * p.ldx + p.k) * 2);
  const auto x_rsrc = packed::panel_rsrc(reinterpret_cast<const uint8_t*>(p.x + row0 * p.ldx), x_bytes);
  uint32_t x_at[R::kDmas];
  int x_chunk[R::kDmas];
#pragma unroll
  for (int d = 0; d < R::kDmas; ++d) {
    const int row = ((wave * R::kDmas + d) * 4 + (lane >> 4)) % (16 * kRows);
    x_chunk[d] = (lane & 15) ^ (row & 15);
    x_at[d] = row < rows ? (uint32_t)(row * p.ldx) * 2 + 16 * x_chunk[d] : ~0u;
  }
  Codes<2> s[kRing];
  // K tiles behind the share's last are loaded as those behind the weight's: as zeros, without
  // memory traffic.
  auto load = [&](Codes<2>& codes, int slot, int stage) __attribute__((always_inline)) {
    const int begin = first + stage * kWays;
    columns.load(codes, begin + way < last ? begin + way : p.k_tiles);
#pragma unroll
    for (int d = 0; d < R::kDmas; ++d) {
      const int from = (wave * R::kDmas + d) * 4, in = begin + from / (16 * kRows), tile = in < last ? in : p.k_tiles;
      const uint32_t at = tile * 128 + 8 * x_chunk[d] < p.k ? x_at[d] : ~0u;  // k behind the last: nothing is read
      packed::dma_frag(x_rsrc, at, min((uint32_t)tile * 256, x_bytes), lds + slot * R::kStage + from * 256);
    }
  };

  f32x4 acc[2][kRows];
#pragma unroll
  for (int c = 0; c < 2; ++c)
#pragma unroll
    for (int r = 0; r < kRows; ++r) acc[c][r] = f32x4{0.f, 0.f, 0.f, 0.f};
  uint32_t at[4];
#pragma unroll
  for (int t = 0; t < 4; ++t) at[t] = way * R::kTileBytes + (lane & 15) * 256 + 16 * ((4 * t + quad) ^ (lane & 15));

  const int stages = (last - first + kWays - 1) / kWays;
#pragma unroll
  for (int d = 0; d < kRing - 1; ++d) {
    load(s[d], d, d);
    // the waits below count operations: none of a stage may be moved behind the next one's
    asm volatile("" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
  }
  for (int i = 0; i < stages; i += kRing) {
#pragma unroll
    for (int d = 0; d < kRing; ++d) {
      if (i + d >= stages) break;
      // This stage's loads are done, kRing - 2 stages' are on their way; then everybody's, and the
      // stage before has been multiplied: its slot is free.
      asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"i"((kRing - 2) * R::kLoads) : "memory");
      constexpr int kFree = kRing - 1;
      load(s[(d + kFree) % kRing], (d + kFree) % kRing, i + d + kFree);
      u32x4 x[kRows][4];
#pragma unroll
      for (int r = 0; r < kRows; ++r)
#pragma unroll
        for (int t = 0; t < 4; ++t) x[r][t] = *reinterpret_cast<const u32x4*>(lds + d * R::kStage + r * 4096 + at[t]);
      multiply<kRows, 2, kGroups, kZeros>(acc, s[d], x, widen);
    }
  }
  // The ways' sums meet in LDS (no DMA is left in flight), [way][side][column tile][row tile].
  asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
  f32x4* const sums = reinterpret_cast<f32x4*>(lds);
#pragma unroll
  for (int c = 0; c < 2; ++c)
#pragma unroll
    for (int r = 0; r < kRows; ++r) sums[((wave * 2 + c) * kRows + r) * 64 + lane] = acc[c][r];
  __syncthreads();
  auto total = [&](int c, int r) {  // column tile c of the workgroup's eight
    f32x4 y = sums[(c * kRows + r) * 64 + lane];
#pragma unroll
    for (int w = 1; w < kWays; ++w) {
      const f32x4 v = sums[((w * 8 + c) * kRows + r) * 64 + lane];
#pragma unroll
      for (int i = 0; i < 4; ++i) y[i] += v[i];
    }
    return y;
  };
  // a wave each for pairs of column tiles
  for (int item = wave; item < 4 * kRows; item += 4 * kWays) {
    const int r = item % kRows, c = item / kRows * 2;
    const int64_t row = row0 + 16 * r + (lane & 15), tile = group0 + c;
    if (gridDim.y > 1) {
      if (row < p.m && tile < p.tiles) {
        float* const to = p.partial + (((int64_t)blockIdx.y * p.m + row) * p.tiles + tile) * 16 + 4 * quad;
        *reinterpret_cast<f32x4*>(to) = total(c, r);
        *reinterpret_cast<f32x4*>(to + 16) = total(c + 1, r);
      }
    } else if (p.epilogue == SMX_EPI_SWIGLU) {
      finish4(p, row, tile * 8 + 4 * quad, gate4(total(c, r), total(c + 1, r)));
    } else {
      finish4(p, row, tile * 16 + 4 * quad, total(c, r));
      finish4(p, row, tile * 16 + 16 + 4 * quad, total(c + 1, r));
    }
  }
}

// Sums the shares' FP32 sums in share order and finishes the rows: one thread a row and
// four columns.
__global__ __launch_bounds__(256) void int4_join(Int4Args p, int shares) {
  const bool gated = p.epilogue == SMX_EPI_SWIGLU;
  const int64_t quads = (int64_t)p.tiles * (gated ? 2 : 4), item = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int64_t row = item / quads;
  if (row >= p.m) return;
  const int64_t quad = item - row * quads, tile = gated ? quad / 4 * 2 : quad / 4;
  const float* const from = p.partial + (row * p.tiles + tile) * 16 + quad % 4 * 4;
  const int64_t stride = (int64_t)p.m * p.tiles * 16;
  auto total = [&](const float* at) {
    f32x4 y = *reinterpret_cast<const f32x4*>(at);
#pragma unroll 4
    for (int s = 1; s < shares; ++s) {
      const f32x4 v = *reinterpret_cast<const f32x4*>(at + s * stride);
#pragma unroll
      for (int i = 0; i < 4; ++i) y[i] += v[i];
    }
    return y;
  };
  finish4(p, row, quad * 4, gated ? gate4(total(from), total(from + 16)) : total(from));
}

// How a product runs: int4_few (waves > 0; its column tiles and whether it stages x), or
// int4_tiled with its row tiles and shares of K.
struct Int4Plan {
  int waves, cols, staged, rows, shares, share;
};

// Times are of a pass among others with weights from HBM, of 128-groups with zero points, in us.
Int4Plan int4_plan(int64_t m, int64_t k_tiles, int64_t tiles, bool gated, int cus) {
  Int4Plan plan{};
  const int64_t x_bytes = m * (k_tiles * 256 + 16);
  if (m <= 16) {
    // x in LDS: with room for two workgroups a CU, or for one where more would find no columns
    if (x_bytes <= 64 * 1024 || (x_bytes <= 144 * 1024 && tiles <= 4 * cus)) {
      plan.staged = 1;
      // Two column tiles share a wave's sums over x (25600 x 5120: 17.2, one tile 18.6); one
      // fills the chip better where columns or K are few (5120 x 1024: 4.3, two tiles 5.9). Eight waves where
      // columns abound (5120 x 51200: 29.4, sixteen 36.3).
      plan.waves = tiles > 8 * cus ? 8 : 16;
      plan.cols = gated || k_tiles > 64 || tiles > 4 * cus ? 2 : 1;
      return plan;
    }
    // Short K and no more columns than that: each wave its own x (16 rows, 5120 x 8192: 9.6,
    // int4_tiled 11.8; but 25600 x 5120: 31 and 21.2)
    if (k_tiles <= 64 && tiles <= 4 * cus) {
      plan.waves = 8, plan.cols = 2;
      return plan;
    }
  }
  // 64 rows a workgroup read and widen the weight once for all of them (61 rows, 5120 x 51200: 57, with
  // 32 rows 70); small weights have the workgroups rather (5120 x 8192: 17.5 and 15.8).
  plan.rows = m <= 16 ? 1 : m <= 32 || tiles * k_tiles <= 128 * cus ? 2 : 4;
  const int64_t blocks = (tiles + 7) / 8 * ((m + 16 * plan.rows - 1) / (16 * plan.rows));
  // K in shares of whole stages, up to a workgroup a CU (more only make more sums to join); a
  // weight of four stages is not worth the second launch
  const int64_t stage = 2, stages = (k_tiles + stage - 1) / stage;
  const int64_t shares = stages <= 4 ? 1 : max((int64_t)1, min(cus / blocks, stages));
  const int64_t each = (stages + shares - 1) / shares;
  plan.share = (int)(each * stage);
  plan.shares = (int)((stages + each - 1) / each);
  return plan;
}

int64_t int4_workspace(const Int4Plan& plan, int64_t m, int64_t tiles) {
  return plan.waves || plan.shares == 1 ? 0 : plan.shares * m * tiles * 64;
}

template <class K>
int launch_int4_kernel(K kern, dim3 grid, int threads, int lds, const Int4Args& p, hipStream_t stream) {
  if (lds > 48 * 1024) {
    hipError_t e = hipFuncSetAttribute((const void*)kern, hipFuncAttributeMaxDynamicSharedMemorySize, lds);
    if (e != hipSuccess) return fail(SMX_ERR_LAUNCH, "hipFuncSetAttribute: %s", hipGetErrorString(e));
  }
  hipLaunchKernelGGL(kern, grid, dim3(threads), lds, stream, p);
  return check_launch();
}

template <int kGroups, bool kZeros>
int launch_int4(const Int4Plan& plan, Int4Args p, hipStream_t s) {
  if (plan.waves) {
    const int lds = max(plan.staged ? (int)(p.m * (p.k_tiles * 256 + 16)) : 0, plan.waves * plan.cols * 1024);
    const dim3 grid((unsigned)((p.tiles + plan.cols - 1) / plan.cols));
    if (!plan.staged) return launch_int4_kernel(int4_few<2, 8, false, kGroups, kZeros>, grid, 512, lds, p, s);
    if (plan.cols == 1) return launch_int4_kernel(int4_few<1, 16, true, kGroups, kZeros>, grid, 1024, lds, p, s);
    if (plan.waves == 16) return launch_int4_kernel(int4_few<2, 16, true, kGroups, kZeros>, grid, 1024, lds, p, s);
    return launch_int4_kernel(int4_few<2, 8, true, kGroups, kZeros>, grid, 512, lds, p, s);
  }
  p.share = plan.share;
  const dim3 grid((unsigned)((p.tiles + 7) / 8), (unsigned)plan.shares, (unsigned)((p.m + 16 * plan.rows - 1) / (16 * plan.rows)));
  auto kern = plan.rows == 1 ? int4_tiled<1, kGroups, kZeros> : plan.rows == 2 ? int4_tiled<2, kGroups, kZeros> : int4_tiled<4, kGroups, kZeros>;
  const int lds = plan.rows == 1 ? Ring<1>::kLds : plan.rows == 2 ? Ring<2>::kLds : Ring<4>::kLds;
  if (int rc = launch_int4_kernel(kern, grid, 512, lds, p, s)) return rc;
  if (plan.shares == 1) return SMX_OK;
  const int64_t items = (int64_t)p.m * p.tiles * (p.epilogue == SMX_EPI_SWIGLU ? 2 : 4);
  hipLaunchKernelGGL(int4_join, dim3((unsigned)((items + 255) / 256)), dim3(256), 0, s, p, plan.shares);
  return check_launch();
}

template <int kGroups>
int launch_zeros(const Int4Plan& plan, const Int4Args& p, bool zeros, hipStream_t s) {
  return zeros ? launch_int4<kGroups, true>(plan, p, s) : launch_int4<kGroups, false>(plan, p, s);
}

int int4_check(const smx_int4_weight* w, int64_t m) {
  if (!w || !w->codes || !w->scales) return fail(SMX_ERR_INVALID, "null pointer");
  if (m <= 0 || m > SMX_PAGED_MAX_TOKENS) return fail(SMX_ERR_INVALID, "1 to %d rows, got %lld", SMX_PAGED_MAX_TOKENS, (long long)m);
  if (w->k <= 0 || w->k > (1 << 22) || w->n <= 0 || w->n > (1 << 24) || w->k % 32)
    return fail(SMX_ERR_INVALID, "k must be a multiple of 32 up to 2^22, n at most 2^24 (k=%lld, n=%lld)", (long long)w->k,
                (long long)w->n);
  if (w->group != 32 && w->group != 64 && w->group != 128)
    return fail(SMX_ERR_INVALID, "group must be 32, 64 or 128, got %d", w->group);
  if (w->swiglu && w->n % 2) return fail(SMX_ERR_INVALID, "[gate | up] has an even width, got %lld", (long long)w->n);
  if ((uintptr_t)w->codes % 16 || (uintptr_t)w->scales % 16)
    return fail(SMX_ERR_INVALID, "codes and scales must be 16-byte aligned");
  return SMX_OK;
}

// Column tiles, whole pairs of them (the layout pads with columns of scale 0).
int64_t int4_tiles(const smx_int4_weight* w) { return w->swiglu ? 2 * ((w->n / 2 + 15) / 16) : 2 * ((w->n + 31) / 32); }

}  // namespace
}  // namespace smx

using namespace smx;

extern "C" {

int smx_int4_workspace_bytes(const smx_int4_weight* w, int64_t m, int64_t* bytes) {
  smx::fail(SMX_OK, "%s", "");
  if (!bytes) return fail(SMX_ERR_INVALID, "null pointer");
  if (int rc = int4_check(w, m)) return rc;
  int cus = 0;
  if (int rc = device_cus(&cus)) return rc;
  const int64_t tiles = int4_tiles(w);
  *bytes = int4_workspace(int4_plan(m, (w->k + 127) / 128, tiles, w->swiglu, cus), m, tiles);
  return SMX_OK;
}

int smx_int4_matmul(const smx_int4_weight* w, int64_t m, const void* x, int64_t ldx, int32_t epilogue, const void* extra,
                    int64_t lde, int32_t extra_f32, void* out, int64_t ldo, void* workspace, int64_t workspace_bytes,
                    void* stream) {
  smx::fail(SMX_OK, "%s", "");
  if (!x || !out) return fail(SMX_ERR_INVALID, "null pointer");
  if (int rc = int4_check(w, m)) return rc;
  const bool gated = epilogue == SMX_EPI_SWIGLU;
  if (epilogue != SMX_EPI_NONE && !gated && epilogue != SMX_EPI_RESIDUAL_ADD && epilogue != SMX_EPI_BIAS_ADD)
    return fail(SMX_ERR_UNSUPPORTED, "epilogue %d is not one of the 4-bit product's", epilogue);
  if (gated != (w->swiglu != 0)) return fail(SMX_ERR_INVALID, "the weight's layout is not that of the epilogue");
  const bool takes = epilogue == SMX_EPI_RESIDUAL_ADD || epilogue == SMX_EPI_BIAS_ADD;
  if (takes != (extra != nullptr)) return fail(SMX_ERR_INVALID, "residual or bias go with their epilogue");
  const int64_t n = gated ? w->n / 2 : w->n;
  // 64 rows of x are one buffer, whose offsets have 32 bits
  if (ldx < w->k || ldx % 8 || ldx > (1 << 24) || (uintptr_t)x % 16)
    return fail(SMX_ERR_INVALID, "x rows must be 16-byte aligned, k to 2^24 elements apart");
  if (ldo < n || (uintptr_t)out % 8) return fail(SMX_ERR_INVALID, "out rows must hold n values, 8-byte aligned");
  if (epilogue == SMX_EPI_RESIDUAL_ADD && lde < n) return fail(SMX_ERR_INVALID, "residual rows must hold n values");
  Int4Args p{};
  p.x = (const uint16_t*)x, p.ldx = ldx;
  p.codes = (const u32x4*)w->codes, p.scales = (const uint32_t*)w->scales;
  p.out = (uint16_t*)out, p.ldo = ldo, p.extra = extra, p.lde = lde, p.extra_f32 = extra_f32;
  p.m = (int32_t)m, p.n = (int32_t)n, p.k = (int32_t)w->k, p.k_tiles = (int32_t)((w->k + 127) / 128);
  p.tiles = (int32_t)int4_tiles(w);
  p.epilogue = epilogue;
  int cus = 0;
  if (int rc = device_cus(&cus)) return rc;
  const Int4Plan plan = int4_plan(m, p.k_tiles, p.tiles, gated, cus);
  const int64_t need = int4_workspace(plan, m, p.tiles);
  if (need && (!workspace || (uintptr_t)workspace % 16 || workspace_bytes < need))
    return fail(SMX_ERR_INVALID, "the call needs a 16-byte aligned workspace of %lld bytes", (long long)need);
  p.partial = (float*)workspace;
  if (w->group == 128) return launch_zeros<1>(plan, p, w->zeros, (hipStream_t)stream);
  if (w->group == 64) return launch_zeros<2>(plan, p, w->zeros, (hipStream_t)stream);
  return launch_zeros<4>(plan, p, w->zeros, (hipStream_t)stream);
}

}  // extern "C"
