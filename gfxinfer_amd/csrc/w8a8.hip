// Products in 8-bit integers with one scale per token and one per output channel, for any
// number of tokens, and the quantizer of their rows.
//
//   s = max |x| * fl32(1 / 127),  c = rint(x / s)              (a row: a token, or a channel)
//   y[t][n] = float(sum_k a[t][k] w[n][k]) * (sa[t] * sw[n])
//
// The integer sum is exact (columns < 2^17, codes >= -128: below 2^31), so K may be divided
// among waves and workgroups in any way without changing a bit of y.  Codes stay row-major:
// a lane's 16 bytes of the v_mfma_i32_16x16x64_i8 operand are contiguous in a row.
// Channels are the A operand and tokens the B operand, so a lane ends up with four
// neighbouring channels of one token.
#include <algorithm>
#include <cmath>
#include <string>

#include "common.hpp"

namespace gfx950 {
namespace {

using i32x4 = int __attribute__((ext_vector_type(4)));
using u32x4 = unsigned __attribute__((ext_vector_type(4)));
using f32x4 = float __attribute__((ext_vector_type(4)));
using h16x4 = _Float16 __attribute__((ext_vector_type(4)));
using h16x8 = _Float16 __attribute__((ext_vector_type(8)));
using lds_void = __attribute__((address_space(3))) void;
using global_void = __attribute__((address_space(1))) void;

// ---- quantizer -------------------------------------------------------------------------

// Eight values of a row in fp32 (exact for all three types).
template <int Type>
__device__ __forceinline__ void load8(const void* input, std::size_t at, float (&x)[8]) {
  if constexpr (Type == GFXI_F32) {
    const f32x4* p = reinterpret_cast<const f32x4*>(static_cast<const float*>(input) + at);
    const f32x4 a = p[0], b = p[1];
#pragma unroll
    for (unsigned e = 0; e < 4; ++e) {
      x[e] = a[e];
      x[4 + e] = b[e];
    }
  } else if constexpr (Type == GFXI_F16) {
    const h16x8 a = *reinterpret_cast<const h16x8*>(static_cast<const _Float16*>(input) + at);
#pragma unroll
    for (unsigned e = 0; e < 8; ++e) x[e] = static_cast<float>(a[e]);
  } else {
    const u32x4 a = *reinterpret_cast<const u32x4*>(static_cast<const uint16_t*>(input) + at);
#pragma unroll
    for (unsigned e = 0; e < 4; ++e) {
      x[2 * e] = __uint_as_float(a[e] << 16);
      x[2 * e + 1] = __uint_as_float(a[e] & 0xffff0000u);
    }
  }
}

// rint of the exact quotient: where the rounded quotient is a half, the sign of the remainder
// says on which side of it the exact one lies (zero: on it, and ties go to even).
__device__ __forceinline__ int code_of(float x, float scale) {
  const float q = x / scale;
  float c = rintf(q);
  if (fabsf(q - truncf(q)) == 0.5F) {
    const float rest = fmaf(-q, scale, x);
    if (rest > 0.0F) c = ceilf(q);
    if (rest < 0.0F) c = floorf(q);
  }
  return static_cast<int>(fminf(fmaxf(c, -127.0F), 127.0F));
}

constexpr unsigned kQuantThreads = 256, kQuantWaves = kQuantThreads / 64;
constexpr unsigned kQuantUnits = 8;  // of eight values a thread keeps: rows up to 16384 are read once

// A workgroup a row.  A row that holds an infinity or a NaN gets a NaN scale and zero codes,
// so every product with it is NaN; a row of zeros the smallest normal scale.
template <int Type>
__global__ __launch_bounds__(kQuantThreads) void quantize_rows_kernel(const void* __restrict__ input, std::size_t stride,
                                                                      uint32_t columns, int8_t* __restrict__ codes,
                                                                      float* __restrict__ scales) {
  __shared__ float partial[kQuantWaves];
  const std::size_t row = blockIdx.x;
  const uint32_t units = columns / 8;
  float x[kQuantUnits][8];
  float top = 0.0F;
  bool finite = true;
  auto measure = [&](const float (&v)[8]) __attribute__((always_inline)) {
#pragma unroll
    for (unsigned e = 0; e < 8; ++e) {
      finite &= fabsf(v[e]) < INFINITY;
      top = fmaxf(top, fabsf(v[e]));
    }
  };
#pragma unroll
  for (unsigned u = 0; u < kQuantUnits; ++u) {
    const uint32_t unit = threadIdx.x + u * kQuantThreads;
    if (unit < units) load8<Type>(input, row * stride + 8 * unit, x[u]);
  }
#pragma unroll
  for (unsigned u = 0; u < kQuantUnits; ++u) {
    if (threadIdx.x + u * kQuantThreads < units) measure(x[u]);
  }
  for (uint32_t unit = threadIdx.x + kQuantUnits * kQuantThreads; unit < units; unit += kQuantThreads) {
    float v[8];
    load8<Type>(input, row * stride + 8 * unit, v);
    measure(v);
  }
  top = wave_max(__all(finite) ? top : INFINITY);
  if ((threadIdx.x & 63u) == 0) partial[threadIdx.x >> 6] = top;
  __syncthreads();
#pragma unroll
  for (unsigned w = 0; w < kQuantWaves; ++w) top = fmaxf(top, partial[w]);
  const bool broken = top == INFINITY;
  const float scale = broken ? __builtin_nanf("") : fmaxf(top * (1.0F / 127.0F), 0x1p-126F);
  if (threadIdx.x == 0) scales[row] = scale;
  auto store = [&](const float (&v)[8], uint32_t unit) __attribute__((always_inline)) {
    uint64_t packed = 0;
    if (!broken) {
#pragma unroll
      for (unsigned e = 0; e < 8; ++e) packed |= static_cast<uint64_t>(static_cast<uint8_t>(code_of(v[e], scale))) << 8 * e;
    }
    *reinterpret_cast<uint64_t*>(codes + row * columns + 8 * unit) = packed;
  };
#pragma unroll
  for (unsigned u = 0; u < kQuantUnits; ++u) {
    const uint32_t unit = threadIdx.x + u * kQuantThreads;
    if (unit < units) store(x[u], unit);
  }
  for (uint32_t unit = threadIdx.x + kQuantUnits * kQuantThreads; unit < units; unit += kQuantThreads) {
    float v[8];
    load8<Type>(input, row * stride + 8 * unit, v);
    store(v, unit);
  }
}

// ---- product ---------------------------------------------------------------------------

struct ProductArgs {
  const int8_t* weights;  // [rows][columns]
  const float* weight_scales;
  const int8_t* codes;  // [tokens][columns]
  const float* scales;
  void* output;  // [tokens][rows]
  int32_t* partial;  // [splits][tokens][rows] where K is divided among workgroups
  uint32_t rows, columns, tokens, splits;
  uint32_t half;  // output type
};

// Channels row .. row + 3 of a token.
__device__ __forceinline__ void write_output(const ProductArgs& a, uint32_t token, uint32_t row, const i32x4& sum) {
  if (token >= a.tokens || row >= a.rows) return;
  const float scale = a.scales[token];
  const std::size_t at = static_cast<std::size_t>(token) * a.rows + row;
  float y[4];
#pragma unroll
  for (unsigned e = 0; e < 4; ++e) {
    y[e] = static_cast<float>(sum[e]) * (scale * a.weight_scales[min(row + e, a.rows - 1)]);
  }
  if (a.rows % 4 == 0) {
    if (a.half != 0) {
      h16x4 h;
#pragma unroll
      for (unsigned e = 0; e < 4; ++e) h[e] = static_cast<_Float16>(y[e]);
      *reinterpret_cast<h16x4*>(static_cast<_Float16*>(a.output) + at) = h;
    } else {
      *reinterpret_cast<f32x4*>(static_cast<float*>(a.output) + at) = f32x4{y[0], y[1], y[2], y[3]};
    }
    return;
  }
#pragma unroll
  for (unsigned e = 0; e < 4; ++e) {
    if (row + e >= a.rows) return;
    if (a.half != 0) static_cast<_Float16*>(a.output)[at + e] = static_cast<_Float16>(y[e]);
    else static_cast<float*>(a.output)[at + e] = y[e];
  }
}

// Few tokens: the weights are streamed once, straight into registers.  A workgroup holds
// 16 R channels and 16 T tokens; its waves divide K and add their sums in LDS.
template <unsigned T, unsigned R, unsigned Waves, unsigned Steps>
__global__ __launch_bounds__(Waves * 64) void w8a8_few_kernel(ProductArgs a) {
  __shared__ i32x4 sums[Waves][R * T][64];
  const unsigned lane = threadIdx.x & 63u, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const unsigned n = lane & 15u, q = lane >> 4;
  const uint32_t first = blockIdx.x * 16 * R;
  const int8_t* w[R];
  const int8_t* x[T];
#pragma unroll
  for (unsigned r = 0; r < R; ++r) w[r] = a.weights + static_cast<std::size_t>(min(first + 16 * r + n, a.rows - 1)) * a.columns + 16 * q;
#pragma unroll
  for (unsigned t = 0; t < T; ++t) x[t] = a.codes + static_cast<std::size_t>(min(16 * t + n, a.tokens - 1)) * a.columns + 16 * q;
  const uint32_t steps = (a.columns + 63) / 64, per = (steps + Waves - 1) / Waves;
  const uint32_t from = wave * per, to = min(from + per, steps);
  i32x4 acc[R][T] = {};
  i32x4 wv[2][Steps][R], xv[2][Steps][T];
  auto load = [&](uint32_t step, unsigned b) __attribute__((always_inline)) {
#pragma unroll
    for (unsigned s = 0; s < Steps; ++s) {
      const uint32_t k = (step + s) * 64;
      const bool there = step + s < to && k + 16 * q < a.columns;
#pragma unroll
      for (unsigned r = 0; r < R; ++r) {
        wv[b][s][r] = i32x4{0, 0, 0, 0};
        if (there) wv[b][s][r] = __builtin_nontemporal_load(reinterpret_cast<const i32x4*>(w[r] + k));
      }
#pragma unroll
      for (unsigned t = 0; t < T; ++t) {
        xv[b][s][t] = i32x4{0, 0, 0, 0};
        if (there) xv[b][s][t] = *reinterpret_cast<const i32x4*>(x[t] + k);
      }
    }
  };
  auto multiply = [&](unsigned b) __attribute__((always_inline)) {
#pragma unroll
    for (unsigned s = 0; s < Steps; ++s) {
#pragma unroll
      for (unsigned r = 0; r < R; ++r) {
#pragma unroll
        for (unsigned t = 0; t < T; ++t) {
          acc[r][t] = __builtin_amdgcn_mfma_i32_16x16x64_i8(wv[b][s][r], xv[b][s][t], acc[r][t], 0, 0, 0);
        }
      }
    }
  };
  if (from < to) load(from, 0);
  for (uint32_t step = from; step < to; step += 2 * Steps) {
    if (step + Steps < to) load(step + Steps, 1);
    multiply(0);
    if (step + Steps < to) {
      if (step + 2 * Steps < to) load(step + 2 * Steps, 0);
      multiply(1);
    }
  }
#pragma unroll
  for (unsigned r = 0; r < R; ++r) {
#pragma unroll
    for (unsigned t = 0; t < T; ++t) sums[wave][r * T + t][lane] = acc[r][t];
  }
  __syncthreads();
  for (unsigned i = wave; i < R * T; i += Waves) {
    i32x4 total = sums[0][i][lane];
#pragma unroll
    for (unsigned v = 1; v < Waves; ++v) total += sums[v][i][lane];
    write_output(a, 16 * (i % T) + n, first + 16 * (i / T) + 4 * q, total);
  }
}

// Many tokens: tiles of BN channels and BM tokens, K in stages of 128 bytes that go straight
// from memory into LDS, one ahead of the products.
//
// A stage's row is 128 bytes, eight pieces of 16; piece c of row r lies in slot c ^ (r % 8)
// (the address a lane loads from is permuted, since loads into LDS fill it lane after lane),
// so the rows of an operand fall on different banks.
constexpr unsigned kStage = 128;

template <unsigned BN, unsigned BM, unsigned WN, unsigned WM>
__global__ __launch_bounds__(WN * WM * 64, 2) void w8a8_tile_kernel(ProductArgs a, uint32_t row_tiles, uint32_t token_tiles) {
  constexpr unsigned kWaves = WN * WM;
  constexpr unsigned R = BN / WN / 16, T = BM / WM / 16;   // 16 x 16 tiles of a wave
  constexpr unsigned kLoads = (BN + BM) * kStage / 16 / (kWaves * 64);
  static_assert(BN * kStage / 16 % (kWaves * 64) == 0 && BM * kStage / 16 % (kWaves * 64) == 0);
  __shared__ __align__(1024) int8_t stage0[(BN + BM) * kStage];
  __shared__ __align__(1024) int8_t stage1[(BN + BM) * kStage];
  const unsigned lane = threadIdx.x & 63u, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const unsigned n = lane & 15u, q = lane >> 4;
  // Consecutive workgroups go to the eight XCDs in turn: each XCD takes a run of the tiles, in
  // columns of all token tiles, so that weights are read into one L2.
  const uint32_t tiles = row_tiles * token_tiles, all = tiles * a.splits;
  uint32_t id = blockIdx.x;
  {
    const uint32_t per = all / 8, rest = all % 8, xcd = id % 8, at = id / 8;
    id = xcd * per + min(xcd, rest) + at;
  }
  const uint32_t split = id / tiles, tile = id - split * tiles;
  const uint32_t row0 = tile / token_tiles * BN, token0 = tile % token_tiles * BM;
  const uint32_t stages = (a.columns + kStage - 1) / kStage, per_split = (stages + a.splits - 1) / a.splits;
  const uint32_t from = split * per_split, to = min(from + per_split, stages);

  // Load u of a wave covers 8 rows (lane / 8) of eight pieces each.
  const int8_t* source[kLoads];
  const unsigned piece = (lane & 7u) ^ (lane >> 3);
#pragma unroll
  for (unsigned u = 0; u < kLoads; ++u) {
    const unsigned r = 8 * (wave + kWaves * u) + lane / 8;
    source[u] = r < BN ? a.weights + static_cast<std::size_t>(min(row0 + r, a.rows - 1)) * a.columns
                       : a.codes + static_cast<std::size_t>(min(token0 + r - BN, a.tokens - 1)) * a.columns;
  }
  auto load = [&](int8_t* stage, uint32_t s) __attribute__((always_inline)) {
    const uint32_t k = s * kStage + 16 * piece;
    const uint32_t at = min(k, a.columns - 16);  // past the row: anything of it, see below
#pragma unroll
    for (unsigned u = 0; u < kLoads; ++u) {
      __builtin_amdgcn_global_load_lds((global_void*)(source[u] + at), (lds_void*)(stage + 8 * (wave + kWaves * u) * kStage), 16, 0, 0);
    }
  };
  i32x4 acc[R][T] = {};
  const unsigned wrow = wave / WM * (BN / WN), trow = BN + wave % WM * (BM / WM);
  auto multiply = [&](const int8_t* stage) __attribute__((always_inline)) {
#pragma unroll
    for (unsigned k = 0; k < 2; ++k) {
      const unsigned slot = 16 * ((4 * k + q) ^ (n & 7u));
      i32x4 w[R], x[T];
#pragma unroll
      for (unsigned r = 0; r < R; ++r) w[r] = *reinterpret_cast<const i32x4*>(stage + (wrow + 16 * r + n) * kStage + slot);
#pragma unroll
      for (unsigned t = 0; t < T; ++t) x[t] = *reinterpret_cast<const i32x4*>(stage + (trow + 16 * t + n) * kStage + slot);
#pragma unroll
      for (unsigned r = 0; r < R; ++r) {
#pragma unroll
        for (unsigned t = 0; t < T; ++t) acc[r][t] = __builtin_amdgcn_mfma_i32_16x16x64_i8(w[r], x[t], acc[r][t], 0, 0, 0);
      }
    }
  };
  // The tokens' pieces past the end of a row become zeros, each by the lane that loaded it.
  auto clear_tail = [&](int8_t* stage) __attribute__((always_inline)) {
#pragma unroll
    for (unsigned u = 0; u < kLoads; ++u) {
      const unsigned r = 8 * (wave + kWaves * u);
      if (r >= BN && (stages - 1) * kStage + 16 * piece >= a.columns) {
        *reinterpret_cast<i32x4*>(stage + r * kStage + 16 * lane) = i32x4{0, 0, 0, 0};
      }
    }
  };
  const bool ragged = a.columns % kStage != 0;
  if (from < to) load(stage0, from);
  for (uint32_t s = from; s < to; s += 2) {
    __builtin_amdgcn_s_waitcnt(0x0f70);  // loads into LDS have arrived
    if (ragged && s + 1 == stages) clear_tail(stage0);
    __syncthreads();
    if (s + 1 < to) load(stage1, s + 1);
    multiply(stage0);
    if (s + 1 < to) {
      __builtin_amdgcn_s_waitcnt(0x0f70);
      if (ragged && s + 2 == stages) clear_tail(stage1);
      __syncthreads();
      if (s + 2 < to) load(stage0, s + 2);
      multiply(stage1);
    }
  }
#pragma unroll
  for (unsigned t = 0; t < T; ++t) {
#pragma unroll
    for (unsigned r = 0; r < R; ++r) {
      const uint32_t token = token0 + (trow - BN) + 16 * t + n, row = row0 + wrow + 16 * r + 4 * q;
      if (a.splits == 1) {
        write_output(a, token, row, acc[r][t]);
      } else if (token < a.tokens) {
        int32_t* plane = a.partial + (static_cast<std::size_t>(split) * a.tokens + token) * a.rows;
        if (a.rows % 4 == 0) {
          if (row < a.rows) *reinterpret_cast<i32x4*>(plane + row) = acc[r][t];
        } else {
#pragma unroll
          for (unsigned e = 0; e < 4; ++e) {
            if (row + e < a.rows) plane[row + e] = acc[r][t][e];
          }
        }
      }
    }
  }
}

// Adds the planes of a divided K.
__global__ __launch_bounds__(256) void w8a8_join_kernel(ProductArgs a) {
  const uint32_t quads = (a.rows + 3) / 4;
  const std::size_t i = static_cast<std::size_t>(blockIdx.x) * 256 + threadIdx.x;
  const uint32_t token = static_cast<uint32_t>(i / quads), row = 4 * static_cast<uint32_t>(i % quads);
  if (token >= a.tokens) return;
  i32x4 sum = {0, 0, 0, 0};
  const std::size_t plane = static_cast<std::size_t>(a.tokens) * a.rows;
  const int32_t* at = a.partial + static_cast<std::size_t>(token) * a.rows + row;
  for (uint32_t s = 0; s < a.splits; ++s, at += plane) {
    if (a.rows % 4 == 0) {
      sum += *reinterpret_cast<const i32x4*>(at);
    } else {
#pragma unroll
      for (unsigned e = 0; e < 4; ++e) sum[e] += row + e < a.rows ? at[e] : 0;
    }
  }
  write_output(a, token, row, sum);
}

constexpr uint32_t kFewTokens = 64;

struct ProductShape {
  uint32_t tile;  // channels and tokens of a tile; 0: the kernel for few tokens
  uint32_t row_tiles, token_tiles, splits;
};

ProductShape product_shape(std::size_t rows, std::size_t columns, std::size_t tokens) {
  ProductShape s{};
  s.splits = 1;
  if (tokens <= kFewTokens) return s;
  auto tiles = [&](uint32_t size) { return ((rows + size - 1) / size) * ((tokens + size - 1) / size); };
  s.tile = tiles(256) >= kComputeUnits ? 256 : 128;
  s.row_tiles = static_cast<uint32_t>((rows + s.tile - 1) / s.tile);
  s.token_tiles = static_cast<uint32_t>((tokens + s.tile - 1) / s.tile);
  if (s.tile == 128) {
    const std::size_t places = 2 * kComputeUnits, stages = (columns + kStage - 1) / kStage;
    const std::size_t want = std::max<std::size_t>(1, places / tiles(128));
    s.splits = static_cast<uint32_t>(std::max<std::size_t>(1, std::min(want, stages / 8)));
    // Every split has a stage to do.
    const std::size_t per = (stages + s.splits - 1) / s.splits;
    s.splits = static_cast<uint32_t>((stages + per - 1) / per);
  }
  return s;
}

std::size_t product_workspace(std::size_t rows, std::size_t columns, std::size_t tokens) {
  const ProductShape s = product_shape(rows, columns, tokens);
  return s.splits > 1 ? s.splits * rows * tokens * sizeof(int32_t) : 0;
}

bool product_sizes(std::size_t rows, std::size_t columns, std::size_t tokens) {
  return rows != 0 && rows <= (1u << 24) && tokens != 0 && tokens <= (1u << 24) && columns != 0 && columns % 16 == 0 &&
         columns < (1u << 17);
}

bool aligned(const void* p, std::size_t bytes) { return p != nullptr && reinterpret_cast<uintptr_t>(p) % bytes == 0; }

template <unsigned T, unsigned R, unsigned Waves, unsigned Steps>
void launch_few(const ProductArgs& a, hipStream_t stream) {
  hipLaunchKernelGGL((w8a8_few_kernel<T, R, Waves, Steps>), dim3((a.rows + 16 * R - 1) / (16 * R)), dim3(Waves * 64), 0, stream, a);
}

}  // namespace
}  // namespace gfx950

using namespace gfx950;

extern "C" int32_t gfxinfer_launch_quantize_rows_i8(const void* input, int32_t input_type, size_t rows, size_t columns,
                                                    size_t row_stride, int8_t* codes, float* scales, void* stream) {
  return guarded([&] {
    if (input_type != GFXI_F16 && input_type != GFXI_F32 && input_type != GFXI_BF16) {
      return fail(GFXI_UNSUPPORTED, "row quantizer: input type is fp16, fp32 or bf16");
    }
    if (!product_sizes(1, columns, rows) || row_stride < columns || row_stride % 8 != 0 || row_stride > (1ull << 40)) {
      return fail(GFXI_INVALID_ARGUMENT, "row quantizer: 1..2^24 rows of a multiple of 16 columns below 2^17, 8 | stride >= columns");
    }
    if (!aligned(input, 16) || !aligned(codes, 16) || !aligned(scales, 4)) {
      return fail(GFXI_INVALID_ARGUMENT, "row quantizer: input and codes are 16-byte aligned, scales are set");
    }
    const dim3 grid(static_cast<unsigned>(rows)), block(kQuantThreads);
    const hipStream_t st = static_cast<hipStream_t>(stream);
    const uint32_t n = static_cast<uint32_t>(columns);
    if (input_type == GFXI_F16) hipLaunchKernelGGL(quantize_rows_kernel<GFXI_F16>, grid, block, 0, st, input, row_stride, n, codes, scales);
    else if (input_type == GFXI_F32) hipLaunchKernelGGL(quantize_rows_kernel<GFXI_F32>, grid, block, 0, st, input, row_stride, n, codes, scales);
    else hipLaunchKernelGGL(quantize_rows_kernel<GFXI_BF16>, grid, block, 0, st, input, row_stride, n, codes, scales);
    return launch_status("row quantizer launch failed");
  });
}

extern "C" size_t gfxinfer_w8a8_gemm_workspace_bytes(size_t rows, size_t columns, size_t tokens) {
  return product_sizes(rows, columns, tokens) ? product_workspace(rows, columns, tokens) : 0;
}

extern "C" int32_t gfxinfer_launch_w8a8_gemm(const int8_t* weights, const float* weight_scales, const int8_t* codes,
                                             const float* scales, void* output, int32_t output_type, size_t rows,
                                             size_t columns, size_t tokens, void* workspace, size_t workspace_bytes,
                                             void* stream) {
  return guarded([&] {
    if (output_type != GFXI_F16 && output_type != GFXI_F32) return fail(GFXI_UNSUPPORTED, "8-bit product: output type is fp16 or fp32");
    if (!product_sizes(rows, columns, tokens)) {
      return fail(GFXI_INVALID_ARGUMENT, "8-bit product: 1..2^24 rows and tokens, columns a multiple of 16 below 2^17");
    }
    if (!aligned(weights, 16) || !aligned(codes, 16) || !aligned(weight_scales, 4) || !aligned(scales, 4) || !aligned(output, 16)) {
      return fail(GFXI_INVALID_ARGUMENT, "8-bit product: codes and output are 16-byte aligned, scales are set");
    }
    const ProductShape s = product_shape(rows, columns, tokens);
    if (const std::size_t need = product_workspace(rows, columns, tokens);
        need != 0 && (!aligned(workspace, 16) || workspace_bytes < need)) {
      return fail(GFXI_INVALID_ARGUMENT, "8-bit product: workspace is null, not 16-byte aligned or too small");
    }
    const uint64_t groups = static_cast<uint64_t>(s.row_tiles) * s.token_tiles * s.splits;
    if (groups > (1u << 30) || (s.splits > 1 && static_cast<uint64_t>(rows) * tokens > (1ull << 38))) {
      return fail(GFXI_INVALID_ARGUMENT, "8-bit product: too large for one launch");
    }
    const ProductArgs a{weights, weight_scales, codes, scales, output, static_cast<int32_t*>(workspace),
                        static_cast<uint32_t>(rows), static_cast<uint32_t>(columns), static_cast<uint32_t>(tokens), s.splits,
                        output_type == GFXI_F16 ? 1u : 0u};
    const hipStream_t st = static_cast<hipStream_t>(stream);
    if (s.tile == 0) {
      if (tokens <= 16) launch_few<1, 1, 8, 4>(a, st);
      else if (tokens <= 32) launch_few<2, 2, 8, 2>(a, st);
      else launch_few<4, 2, 8, 2>(a, st);
      return launch_status("8-bit product launch failed");
    }
    const dim3 grid(static_cast<unsigned>(groups));
    if (s.tile == 256) hipLaunchKernelGGL((w8a8_tile_kernel<256, 256, 2, 4>), grid, dim3(512), 0, st, a, s.row_tiles, s.token_tiles);
    else hipLaunchKernelGGL((w8a8_tile_kernel<128, 128, 2, 2>), grid, dim3(256), 0, st, a, s.row_tiles, s.token_tiles);
    if (const int32_t status = launch_status("8-bit product launch failed"); status != GFXI_OK || s.splits == 1) return status;
    const std::size_t quads = (rows + 3) / 4 * tokens;
    hipLaunchKernelGGL(w8a8_join_kernel, dim3(static_cast<unsigned>((quads + 255) / 256)), dim3(256), 0, st, a);
    return launch_status("8-bit product join launch failed");
  });
}
