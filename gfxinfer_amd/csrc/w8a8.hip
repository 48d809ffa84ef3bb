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
//
// What bounds it: with few tokens the weights' bytes (5120 x 5120, one token: 6.9 us, 3.8 TB/s; 17408 x
// 5120, 37 tokens: 25 us, 3.6 TB/s), with many the matrix instructions and the waits between their stages
// (17408 x 5120, 4096 tokens: 393 us, 1.86 POP/s, where a large library product of one size reaches 2.25;
// the matrix units are busy 43 % of the time at about 2.0 GHz, LDS reads have no bank conflicts).
#include <algorithm>
#include <cmath>
#include <string>

#include "common.hpp"

namespace gfx950 {
namespace {

using i32x4 = int __attribute__((ext_vector_type(4)));
using i32x16 = int __attribute__((ext_vector_type(16)));
using u32x4 = unsigned __attribute__((ext_vector_type(4)));
using f32x4 = float __attribute__((ext_vector_type(4)));
using h16x4 = _Float16 __attribute__((ext_vector_type(4)));
using h16x8 = _Float16 __attribute__((ext_vector_type(8)));
using lds_void = __attribute__((address_space(3))) void;

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
__device__ __forceinline__ float exact_code(float x, float scale) {
  const float q = x / scale;
  float c = rintf(q);
  if (fabsf(q - truncf(q)) == 0.5F) {
    const float rest = fmaf(-q, scale, x);
    if (rest > 0.0F) c = ceilf(q);
    if (rest < 0.0F) c = floorf(q);
  }
  return c;
}

// Four codes.  x times the reciprocal is within 2^-16 of the quotient (two roundings of numbers below
// 127.1), so only where it lies that close to a half the quotient is needed: one code in 30000.
__device__ __forceinline__ uint32_t four_codes(const float (&x)[8], unsigned first, float scale, float inverse) {
  float c[4];
  bool close = false;
#pragma unroll
  for (unsigned e = 0; e < 4; ++e) {
    const float q = x[first + e] * inverse;
    c[e] = rintf(q);
    close |= fabsf(q - c[e]) > 0.5F - 0x1p-15F;
  }
  if (close) {
#pragma unroll
    for (unsigned e = 0; e < 4; ++e) c[e] = exact_code(x[first + e], scale);
  }
  uint32_t packed = 0;
#pragma unroll
  for (unsigned e = 0; e < 4; ++e) {
    packed |= (static_cast<uint32_t>(static_cast<int>(__builtin_amdgcn_fmed3f(c[e], -127.0F, 127.0F))) & 0xffu) << 8 * e;
  }
  return packed;
}

constexpr unsigned kQuantUnits = 4;  // of eight values a thread keeps
constexpr unsigned kGridRows = 1u << 20;  // along x: a launch holds less than 2^32 threads in one dimension

// A workgroup a row, read once and kept in registers: bytes, 4096 rows of 5120 in fp16 15 us (4.1 TB/s), one
// row 3.3 us, the time of a launch and three dependent steps.  A row that holds an infinity or a NaN gets a NaN scale and zero codes,
// so every product with it is NaN; a row of zeros the smallest normal scale.
template <int Type, unsigned Threads>
__global__ __launch_bounds__(Threads) void quantize_rows_kernel(const void* __restrict__ input, std::size_t stride, uint32_t rows,
                                                                uint32_t columns, int8_t* __restrict__ codes,
                                                                float* __restrict__ scales) {
  __shared__ float partial[Threads / 64];
  const std::size_t row = blockIdx.y * kGridRows + blockIdx.x;
  if (row >= rows) return;
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
    const uint32_t unit = threadIdx.x + u * Threads;
    if (unit < units) load8<Type>(input, row * stride + 8 * unit, x[u]);
  }
#pragma unroll
  for (unsigned u = 0; u < kQuantUnits; ++u) {
    if (threadIdx.x + u * Threads < units) measure(x[u]);
  }
  for (uint32_t unit = threadIdx.x + kQuantUnits * Threads; unit < units; unit += Threads) {
    float v[8];
    load8<Type>(input, row * stride + 8 * unit, v);
    measure(v);
  }
  top = wave_max(__all(finite) ? top : INFINITY);
  if ((threadIdx.x & 63u) == 0) partial[threadIdx.x >> 6] = top;
  __syncthreads();
#pragma unroll
  for (unsigned w = 0; w < Threads / 64; ++w) top = fmaxf(top, partial[w]);
  const bool broken = top == INFINITY;
  const float scale = broken ? __builtin_nanf("") : fmaxf(top * (1.0F / 127.0F), 0x1p-126F);
  const float inverse = 1.0F / scale;
  if (threadIdx.x == 0) scales[row] = scale;
  auto store = [&](const float (&v)[8], uint32_t unit) __attribute__((always_inline)) {
    uint2 packed = {0, 0};
    if (!broken) packed = uint2{four_codes(v, 0, scale, inverse), four_codes(v, 4, scale, inverse)};
    *reinterpret_cast<uint2*>(codes + row * columns + 8 * unit) = packed;
  };
#pragma unroll
  for (unsigned u = 0; u < kQuantUnits; ++u) {
    const uint32_t unit = threadIdx.x + u * Threads;
    if (unit < units) store(x[u], unit);
  }
  for (uint32_t unit = threadIdx.x + kQuantUnits * Threads; unit < units; unit += Threads) {
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

// Operand tiles (16 rows, 128 bytes of K) first and second of a stage in LDS, both 64-byte steps of
// each, complete when they return.  (The compiler would let reads of its own wait for the later stages'
// loads into LDS, which it cannot tell from this one's.)
__device__ __forceinline__ void read_pair(unsigned first, unsigned second, i32x4 (&x)[2], i32x4 (&y)[2]) {
  asm volatile(
      "ds_read_b128 %0, %4\n\tds_read_b128 %1, %5\n\tds_read_b128 %2, %6\n\tds_read_b128 %3, %7\n\ts_waitcnt lgkmcnt(0)"
      : "=&v"(x[0]), "=&v"(x[1]), "=&v"(y[0]), "=&v"(y[1])
      : "v"(first), "v"(first ^ 64u), "v"(second), "v"(second ^ 64u)
      : "memory");
}

// At most Loads of the wave's loads are on their way.
template <unsigned Loads>
__device__ __forceinline__ void wait_loads() {
  static_assert(Loads < 64);
  __builtin_amdgcn_s_waitcnt((Loads & 15u) | (Loads >> 4) << 14 | 0xfu << 8 | 7u << 4);
  asm volatile("" ::: "memory");
}

// All of the wave's LDS accesses are complete.
__device__ __forceinline__ void wait_reads() { asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory"); }

// Few tokens: the weights are streamed once.  A workgroup holds 16 R channels and 16 T tokens; its
// waves divide K, each with a ring of Depth stages of 128 bytes in LDS for itself, and add their sums
// at the end.  Loads cover whole lines of memory, eight rows of 128 bytes each: straight into the
// registers of an operand they would be sixteen rows of 64 (17408 x 5120, one token: 29 % longer).
// Piece c of row r lies in slot c ^ (r / 2 % 8), see below.
template <unsigned T, unsigned R, unsigned Waves, unsigned Depth>
__global__ __launch_bounds__(Waves * 64) void w8a8_few_kernel(ProductArgs a) {
  constexpr unsigned kTiles = R + T, kStageBytes = kTiles * 2048;
  constexpr unsigned kSums = R * T * 1024;
  __shared__ __align__(1024) int8_t ring[Waves * (Depth * kStageBytes > kSums ? Depth * kStageBytes : kSums)];
  const unsigned lane = threadIdx.x & 63u, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const unsigned n = lane & 15u, q = lane >> 4;
  const uint32_t first = blockIdx.x * 16 * R;
  int8_t* mine = ring + wave * (Depth * kStageBytes);
  const auto weights = __builtin_amdgcn_make_buffer_rsrc(const_cast<int8_t*>(a.weights) + static_cast<std::size_t>(first) * a.columns, 0,
                                                         static_cast<int>(min(16 * R, a.rows - first) * a.columns), 0x20000);
  const auto codes = __builtin_amdgcn_make_buffer_rsrc(const_cast<int8_t*>(a.codes), 0, static_cast<int>(min(16 * T, a.tokens) * a.columns), 0x20000);
  // Load u covers rows 8 u .. of the channels, then of the tokens; rows past the last one load that one.
  const unsigned piece[2] = {(lane & 7u) ^ (lane >> 4), (lane & 7u) ^ (4 + (lane >> 4))};  // of even and odd loads
  uint32_t source[2 * kTiles];
#pragma unroll
  for (unsigned u = 0; u < 2 * kTiles; ++u) {
    const unsigned r = 8 * u + lane / 8;
    source[u] = (u < 2 * R ? min(r, a.rows - first - 1) : min(r - 16 * R, a.tokens - 1)) * a.columns;
  }
  const uint32_t stages = (a.columns + 127) / 128, per = (stages + Waves - 1) / Waves;
  const uint32_t from = wave * per, to = min(from + per, stages);
  auto load = [&](uint32_t s, unsigned slot) __attribute__((always_inline)) {
    // Past the row: anything of it, see below.
    uint32_t at[2];
#pragma unroll
    for (unsigned e = 0; e < 2; ++e) at[e] = min(s * 128 + 16 * piece[e], a.columns - 16);
#pragma unroll
    for (unsigned u = 0; u < 2 * kTiles; ++u) {
      __builtin_amdgcn_raw_ptr_buffer_load_lds(u < 2 * R ? weights : codes, (lds_void*)(mine + slot * kStageBytes + u * 1024), 16,
                                               static_cast<int>(source[u] + at[u % 2]), 0, 0, 0);
    }
  };
  i32x4 acc[R][T] = {};
#pragma unroll
  for (unsigned d = 0; d + 1 < Depth; ++d) {
    if (from + d < to) load(from + d, d);
  }
  const unsigned place = static_cast<unsigned>(reinterpret_cast<uintptr_t>((lds_void*)mine)) + n * 128 + 16 * (q ^ (n >> 1));
  unsigned slot = 0;
#pragma unroll 1
  for (uint32_t s = from; s < to; ++s) {
    // This stage has arrived when only the later ones are on their way.
    if (s + Depth - 1 <= to) wait_loads<(Depth - 2) * 2 * kTiles>();
    else wait_loads<0>();
    if (s + 1 == stages && a.columns % 128 != 0) {
      // The tokens' pieces past the end of a row become zeros, each by the lane that loaded it.
#pragma unroll
      for (unsigned u = 2 * R; u < 2 * kTiles; ++u) {
        if (s * 128 + 16 * piece[u % 2] >= a.columns) *reinterpret_cast<i32x4*>(mine + slot * kStageBytes + u * 1024 + 16 * lane) = i32x4{0, 0, 0, 0};
      }
      wait_reads();
    }
    // The stage before this one has been read: its slot takes the next loads.
    const unsigned before = slot == 0 ? Depth - 1 : slot - 1;
    if (s + Depth - 1 < to) load(s + Depth - 1, before);
    const unsigned at = place + slot * kStageBytes;
    i32x4 w[R + R % 2][2], x[T + T % 2][2];
    // Pairs of tiles: channels, then tokens (an odd one is read twice).
#pragma unroll
    for (unsigned r = 0; r < R; r += 2) read_pair(at + r * 2048, at + (r + 1 < R ? r + 1 : r) * 2048, w[r], w[r + 1]);
#pragma unroll
    for (unsigned t = 0; t < T; t += 2) read_pair(at + (R + t) * 2048, at + (R + (t + 1 < T ? t + 1 : t)) * 2048, x[t], x[t + 1]);
#pragma unroll
    for (unsigned k = 0; k < 2; ++k) {
#pragma unroll
      for (unsigned r = 0; r < R; ++r) {
#pragma unroll
        for (unsigned t = 0; t < T; ++t) acc[r][t] = __builtin_amdgcn_mfma_i32_16x16x64_i8(w[r][k], x[t][k], acc[r][t], 0, 0, 0);
      }
    }
    slot = slot + 1 == Depth ? 0 : slot + 1;
  }
  __syncthreads();  // the rings are done with
  i32x4* sums = reinterpret_cast<i32x4*>(ring);  // [waves][R T][64]
#pragma unroll
  for (unsigned r = 0; r < R; ++r) {
#pragma unroll
    for (unsigned t = 0; t < T; ++t) sums[(wave * R * T + r * T + t) * 64 + lane] = acc[r][t];
  }
  __syncthreads();
  for (unsigned i = wave; i < R * T; i += Waves) {
    i32x4 total = sums[i * 64 + lane];
#pragma unroll
    for (unsigned v = 1; v < Waves; ++v) total += sums[(v * R * T + i) * 64 + lane];
    write_output(a, 16 * (i % T) + n, first + 16 * (i / T) + 4 * q, total);
  }
}

// Many tokens: tiles of BN channels and BM tokens, K in stages of 128 bytes that go straight
// from memory into LDS, Depth - 1 ahead of the products (v_mfma_i32_32x32x32_i8).  Two stages ahead instead
// of one: 5120 x 17408 and 509 tokens 65 us, not 77; the tiles of 256 x 256 have room in LDS for one ahead.
//
// A stage's row is 128 bytes, eight pieces of 16; piece c of row r lies in slot c ^ (r / 2 % 8)
// (the address a lane loads from is permuted, since loads into LDS fill it lane after lane),
// so sixteen rows of an operand, two of which lie side by side in the banks, fall on different ones.
constexpr unsigned kStage = 128;
constexpr unsigned kGroup = 8;  // token tiles that run beside each other

template <unsigned BN, unsigned BM, unsigned WN, unsigned WM, unsigned Depth>
__global__ __launch_bounds__(WN * WM * 64, 2) void w8a8_tile_kernel(ProductArgs a, uint32_t first_row, uint32_t row_tiles, uint32_t token_tiles) {
  constexpr unsigned kWaves = WN * WM;
  constexpr unsigned R = BN / WN / 32, T = BM / WM / 32;   // 32 x 32 tiles of a wave
  constexpr unsigned kLoads = (BN + BM) * kStage / 16 / (kWaves * 64);
  static_assert(BN * kStage / 16 % (kWaves * 64) == 0 && BM * kStage / 16 % (kWaves * 64) == 0);
  // (Arrays of their own, so that the compiler can tell one stage's reads from another's loads.)
  constexpr unsigned kBytes = (BN + BM) * kStage;
  __shared__ __align__(1024) int8_t stage0[kBytes];
  __shared__ __align__(1024) int8_t stage1[kBytes];
  __shared__ __align__(1024) int8_t stage2[Depth > 2 ? kBytes : 16];
  __shared__ __align__(1024) int8_t stage3[Depth > 3 ? kBytes : 16];
  int8_t* const ring[4] = {stage0, stage1, stage2, stage3};
  const unsigned lane = threadIdx.x & 63u, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const unsigned n = lane & 31u, h = lane >> 5;
  // Consecutive workgroups go to the eight XCDs in turn: each XCD takes a run of the tiles, in groups of
  // eight token tiles by all row tiles, so that the 32 tiles it works on at once share their operands
  // through its L2.
  const uint32_t tiles = row_tiles * token_tiles, all = tiles * a.splits;
  uint32_t id = blockIdx.x;
  {
    const uint32_t per = all / 8, rest = all % 8, xcd = id % 8, at = id / 8;
    id = xcd * per + min(xcd, rest) + at;
  }
  const uint32_t split = id / tiles, tile = id - split * tiles;
  const uint32_t group = tile / (kGroup * row_tiles), in_group = tile - group * kGroup * row_tiles;
  const uint32_t wide = min(kGroup, token_tiles - group * kGroup);
  const uint32_t row0 = first_row + in_group / wide * BN, token0 = (group * kGroup + in_group % wide) * BM;
  const uint32_t stages = (a.columns + kStage - 1) / kStage, per_split = (stages + a.splits - 1) / a.splits;
  const uint32_t from = split * per_split, to = min(from + per_split, stages);

  // Load u of a wave covers 8 rows (lane / 8) of eight pieces each; rows past the last one load that one.
  const auto weights = __builtin_amdgcn_make_buffer_rsrc(const_cast<int8_t*>(a.weights) + static_cast<std::size_t>(row0) * a.columns, 0,
                                                         static_cast<int>(min(BN, a.rows - row0) * a.columns), 0x20000);
  const auto codes = __builtin_amdgcn_make_buffer_rsrc(const_cast<int8_t*>(a.codes) + static_cast<std::size_t>(token0) * a.columns, 0,
                                                       static_cast<int>(min(BM, a.tokens - token0) * a.columns), 0x20000);
  uint32_t source[kLoads];
  static_assert(kWaves % 2 == 0);  // loads of a wave are all of even or all of odd groups of eight rows
  const unsigned piece = (lane & 7u) ^ (4 * (wave & 1u) + (lane >> 4));
#pragma unroll
  for (unsigned u = 0; u < kLoads; ++u) {
    const unsigned r = 8 * (wave + kWaves * u) + lane / 8;
    source[u] = (r < BN ? min(r, a.rows - row0 - 1) : min(r - BN, a.tokens - token0 - 1)) * a.columns;
  }
  auto load = [&](int8_t* stage, uint32_t s) __attribute__((always_inline)) {
    const uint32_t at = min(s * kStage + 16 * piece, a.columns - 16);  // past the row: anything of it, see below
#pragma unroll
    for (unsigned u = 0; u < kLoads; ++u) {
      const unsigned r = 8 * (wave + kWaves * u);
      __builtin_amdgcn_raw_ptr_buffer_load_lds(r < BN ? weights : codes, (lds_void*)(stage + r * kStage), 16, static_cast<int>(source[u] + at), 0, 0, 0);
    }
  };
  i32x16 acc[R][T] = {};
  const unsigned wrow = wave / WM * (BN / WN), trow = BN + wave % WM * (BM / WM);
  const unsigned place = n * kStage + 16 * (h ^ (n >> 1 & 7u));  // step k is at the place ^ 32 k
  auto multiply = [&](const int8_t* stage) __attribute__((always_inline)) {
#pragma unroll
    for (unsigned k = 0; k < kStage / 32; ++k) {
      i32x4 w[R], x[T];
#pragma unroll
      for (unsigned t = 0; t < T; ++t) x[t] = *reinterpret_cast<const i32x4*>(stage + (trow + 32 * t) * kStage + (place ^ 32 * k));
#pragma unroll
      for (unsigned r = 0; r < R; ++r) w[r] = *reinterpret_cast<const i32x4*>(stage + (wrow + 32 * r) * kStage + (place ^ 32 * k));
#pragma unroll
      for (unsigned r = 0; r < R; ++r) {
#pragma unroll
        for (unsigned t = 0; t < T; ++t) acc[r][t] = __builtin_amdgcn_mfma_i32_32x32x32_i8(w[r], x[t], acc[r][t], 0, 0, 0);
      }
    }
    // Operands are read two ahead of a step's products.
    constexpr unsigned kReads = kStage / 32 * (R + T), kAhead = R + T + 2;
    __builtin_amdgcn_sched_group_barrier(0x100, kAhead, 0);
#pragma unroll
    for (unsigned e = 0; e < kReads - kAhead; ++e) {
      __builtin_amdgcn_sched_group_barrier(0x8, 1, 0);
      __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
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
  // Stages past the last one load that one again: with no branch around the loads the compiler can count
  // them, too.
#pragma unroll
  for (unsigned d = 0; d + 1 < Depth; ++d) load(ring[d], min(from + d, to - 1));
  auto turn = [&](uint32_t s, unsigned d) __attribute__((always_inline)) {
    // This stage has arrived when only the later ones are on their way.
    wait_loads<(Depth - 2) * kLoads>();
    if (ragged && s + 1 == stages) clear_tail(ring[d]);
    wait_reads();
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    // Every wave has read the stage before this one: its place takes the next loads.
    load(ring[(d + Depth - 1) % Depth], min(s + Depth - 1, to - 1));
    multiply(ring[d]);
  };
  uint32_t s = from;
#pragma unroll 1
  for (; s + Depth <= to; s += Depth) {
#pragma unroll
    for (unsigned d = 0; d < Depth; ++d) turn(s + d, d);
  }
#pragma unroll
  for (unsigned d = 0; d + 1 < Depth; ++d) {
    if (s + d < to) turn(s + d, d);
  }
  // The loads of no stage write into this workgroup's LDS, so it stays until they have.
  wait_loads<0>();
#pragma unroll
  for (unsigned t = 0; t < T; ++t) {
#pragma unroll
    for (unsigned r = 0; r < R; ++r) {
#pragma unroll
      for (unsigned e = 0; e < 16; e += 4) {
        const uint32_t token = token0 + (trow - BN) + 32 * t + n, row = row0 + wrow + 32 * r + 2 * e + 4 * h;
        const i32x4 sum = {acc[r][t][e], acc[r][t][e + 1], acc[r][t][e + 2], acc[r][t][e + 3]};
        if (a.splits == 1) {
          write_output(a, token, row, sum);
        } else if (token < a.tokens) {
          int32_t* plane = a.partial + (static_cast<std::size_t>(split) * a.tokens + token) * a.rows;
          if (a.rows % 4 == 0) {
            if (row < a.rows) *reinterpret_cast<i32x4*>(plane + row) = sum;
          } else {
#pragma unroll
            for (unsigned c = 0; c < 4; ++c) {
              if (row + c < a.rows) plane[row + c] = sum[c];
            }
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

// Up to 64 tokens of small matrices, up to 48 of large ones, up to 8 where there are so few channels that their workgroups
// leave CUs without work over a long K: 5120 x 5120 and 64 tokens 10.1 us, in tiles 11.8; 34816 x 5120 61.6 and 56.9, with
// 40 tokens 52.2 and 54.5; 5120 x 17408 with 16 tokens 27.0 and 25.2, with 40 31.5 and 27.6.
bool few_tokens(std::size_t rows, std::size_t columns, std::size_t tokens) {
  if (rows * columns < (1u << 26)) return tokens <= 64;
  return tokens <= (rows < 32 * kComputeUnits ? 8 : 48);
}

struct ProductShape {
  uint32_t main_tiles;  // of 256 channels, which run first
  uint32_t tile_rows;  // channels of a tile, see below; 0: the kernel for few tokens
  uint32_t row_tiles, token_tiles, splits;
};

// The tile shapes, with the time in nanoseconds that a round of their workgroups takes by itself and for each
// stage of 128 columns, fitted to what 900 products of 65 to 4096 tokens and 1024 to 34816 rows took.
struct TileShape {
  uint32_t rows, tokens, places;
  double round, stage;
};
constexpr TileShape kTileShapes[] = {
    {64, 64, 2 * kComputeUnits, 600, 370},
    {128, 128, kComputeUnits, 2700, 470},
    {256, 128, kComputeUnits, 4500, 620},
};
// Joining splits takes 8.5 us and 1.34 ps for each sum.
constexpr double kJoinTime = 8500, kJoinSum = 0.00134;
constexpr uint32_t kMaxSplits = 8;
constexpr std::size_t kMainTile = 256;

// The shape and the number of splits that take the shortest time: the rounds that the chip needs for the
// workgroups times the time of one. Against the best of all on the same 78 sizes the choice costs 2.3 % on
// average and 16 % at worst. 5120 x 5120 and 160 tokens: 12.6 us in tiles of 64, 18.4 of 128, 28 of 256; 17408 x 5120 and 1024
// tokens: 197, 162 and 127; 5120 x 17408 and 320 tokens: 48 in four splits of 256, 55 in three, 75 in tiles of 64 without.
ProductShape best_shape(std::size_t rows, std::size_t columns, std::size_t tokens, uint32_t most_splits) {
  ProductShape s{};
  const std::size_t stages = (columns + kStage - 1) / kStage;
  double best = 0;
  for (const TileShape& t : kTileShapes) {
    const std::size_t row_tiles = (rows + t.rows - 1) / t.rows, token_tiles = (tokens + t.tokens - 1) / t.tokens;
    for (uint32_t want = 1; want <= std::min<std::size_t>(most_splits, stages); ++want) {
      // Every split has a stage to do.
      const std::size_t per = (stages + want - 1) / want, splits = (stages + per - 1) / per;
      const std::size_t rounds = (row_tiles * token_tiles * splits + t.places - 1) / t.places;
      double time = static_cast<double>(rounds) * (t.round + static_cast<double>(per) * t.stage);
      if (splits > 1) time += kJoinTime + kJoinSum * static_cast<double>(splits * rows * tokens);
      if (s.tile_rows != 0 && time >= best) continue;
      best = time;
      s = {0, t.rows, static_cast<uint32_t>(row_tiles), static_cast<uint32_t>(token_tiles), static_cast<uint32_t>(splits)};
    }
  }
  return s;
}

// Tiles of 256 x 256 take the least time for their size, but a last round of few of them takes as long as a full
// one, and so does a tile with few tokens.  So where they pad the tokens no further than tiles of 128 would, they take the channels
// that make whole rounds, and the others follow in the shape that is best for them.  17408 x 5120 with 4096 tokens: 393 us, in one
// launch of 256 x 128 9 % more; 34816 x 5120 with 509 tokens 120, not 151; 5120 x 5120 with 8192 tokens 234, not 247.  With more
// padding (34816 x 5120 and 300 tokens) it took 111 us and one launch 97; where more than half a round is left it is about even
// (27392 x 5120 with 1024 tokens 199 and 203, 34816 x 5120 with 768 200 and 186).
ProductShape product_shape(std::size_t rows, std::size_t columns, std::size_t tokens) {
  ProductShape s{};
  s.splits = 1;
  if (few_tokens(rows, columns, tokens)) return s;
  const std::size_t wide = (tokens + kMainTile - 1) / kMainTile, rounds = wide * (rows / kMainTile) / kComputeUnits;
  const std::size_t first = rounds * kComputeUnits / wide;
  if (first == 0 || (tokens + 127) / 128 % 2 != 0) return best_shape(rows, columns, tokens, kMaxSplits);
  if (first * kMainTile < rows) s = best_shape(rows - first * kMainTile, columns, tokens, 1);
  s.main_tiles = static_cast<uint32_t>(first);
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

template <unsigned T, unsigned R, unsigned Waves, unsigned Depth>
void launch_few(const ProductArgs& a, hipStream_t stream) {
  hipLaunchKernelGGL((w8a8_few_kernel<T, R, Waves, Depth>), dim3((a.rows + 16 * R - 1) / (16 * R)), dim3(Waves * 64), 0, stream, a);
}

// Rows up to 8192 values fit the registers of four waves, up to 32768 those of sixteen; longer ones are read twice.
template <int Type>
void launch_quantize(const void* input, std::size_t rows, std::size_t stride, uint32_t columns, int8_t* codes, float* scales,
                     hipStream_t stream) {
  const uint32_t n = static_cast<uint32_t>(rows);
  const dim3 grid(std::min(n, kGridRows), (n + kGridRows - 1) / kGridRows);
  if (columns <= 256 * 8 * kQuantUnits) {
    hipLaunchKernelGGL((quantize_rows_kernel<Type, 256>), grid, dim3(256), 0, stream, input, stride, n, columns, codes, scales);
  } else {
    hipLaunchKernelGGL((quantize_rows_kernel<Type, 1024>), grid, dim3(1024), 0, stream, input, stride, n, columns, codes, scales);
  }
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
    const hipStream_t st = static_cast<hipStream_t>(stream);
    const uint32_t n = static_cast<uint32_t>(columns);
    if (input_type == GFXI_F16) launch_quantize<GFXI_F16>(input, rows, row_stride, n, codes, scales, st);
    else if (input_type == GFXI_F32) launch_quantize<GFXI_F32>(input, rows, row_stride, n, codes, scales, st);
    else launch_quantize<GFXI_BF16>(input, rows, row_stride, n, codes, scales, st);
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
    const uint64_t main_groups = static_cast<uint64_t>(s.main_tiles) * ((tokens + kMainTile - 1) / kMainTile);
    // Of the launches' up to 512 threads a workgroup, or a thread for four sums.
    const std::size_t quads = (rows + 3) / 4 * tokens;
    if (groups >= (1u << 23) || main_groups >= (1u << 23) || (s.splits > 1 && quads > 0xffffff00u)) {
      return fail(GFXI_INVALID_ARGUMENT, "8-bit product: too large for one launch");
    }
    const ProductArgs a{weights, weight_scales, codes, scales, output, static_cast<int32_t*>(workspace),
                        static_cast<uint32_t>(rows), static_cast<uint32_t>(columns), static_cast<uint32_t>(tokens), s.splits,
                        output_type == GFXI_F16 ? 1u : 0u};
    const hipStream_t st = static_cast<hipStream_t>(stream);
    if (few_tokens(rows, columns, tokens)) {
      // (With few tokens the weights' rows are all that a workgroup reads, with more its tokens' are worth reading for 32 of
      // them: 17408 x 5120 19.5 us for one token with 16 channels a workgroup, 21.7 with 32; 16 tokens 23.2 and 21.8.)
      if (tokens <= 4) launch_few<1, 1, 4, 3>(a, st);
      else if (tokens <= 16) launch_few<1, 2, 4, 3>(a, st);
      else if (tokens <= 32) launch_few<2, 2, 4, 3>(a, st);
      else if (tokens <= 48) launch_few<3, 2, 4, 3>(a, st);
      else launch_few<4, 2, 4, 3>(a, st);
      return launch_status("8-bit product launch failed");
    }
    uint32_t first_row = 0;
    if (s.main_tiles != 0) {
      const uint32_t token_tiles = static_cast<uint32_t>((tokens + kMainTile - 1) / kMainTile);
      hipLaunchKernelGGL((w8a8_tile_kernel<256, 256, 2, 4, 2>), dim3(s.main_tiles * token_tiles), dim3(512), 0, st, a, 0u, s.main_tiles, token_tiles);
      if (const int32_t status = launch_status("8-bit product launch failed"); status != GFXI_OK || s.tile_rows == 0) return status;
      first_row = s.main_tiles * kMainTile;
    }
    const dim3 grid(static_cast<unsigned>(groups));
    if (s.tile_rows == 64) hipLaunchKernelGGL((w8a8_tile_kernel<64, 64, 2, 2, 4>), grid, dim3(256), 0, st, a, first_row, s.row_tiles, s.token_tiles);
    else if (s.tile_rows == 128) hipLaunchKernelGGL((w8a8_tile_kernel<128, 128, 2, 4, 4>), grid, dim3(512), 0, st, a, first_row, s.row_tiles, s.token_tiles);
    else hipLaunchKernelGGL((w8a8_tile_kernel<256, 128, 4, 2, 3>), grid, dim3(512), 0, st, a, first_row, s.row_tiles, s.token_tiles);
    if (const int32_t status = launch_status("8-bit product launch failed"); status != GFXI_OK || s.splits == 1) return status;
    hipLaunchKernelGGL(w8a8_join_kernel, dim3(static_cast<unsigned>((quads + 255) / 256)), dim3(256), 0, st, a);
    return launch_status("8-bit product join launch failed");
  });
}
