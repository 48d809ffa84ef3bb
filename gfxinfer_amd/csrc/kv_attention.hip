// Gated GQA decode attention over the pages of a K/V cache, for a batch of sequences
// that share a prefix: the prefix is read once for all of them.
//
// Row (i, t, h), token t of the i-th listed sequence at query head h, attends to the first
// length_i + t + 1 positions:  o = softmax(q . K / sqrt(D)) . V * sigmoid(gate).  The rows of
// all sequences are one tall matrix against the prefix (positions below `shared`, read
// through the first sequence's table) and one small matrix per sequence against its own
// positions.  Both are the same work item: a tile of rows, a KV head and a range of positions.
// Each writes (maximum, sum, unnormalized output) and a second launch merges a row's items
// and applies the gate.
//
// Inside an item the four waves take every fourth block of 32 positions and merge at the end:
// a wave meets each K and V row once, for all the rows of the tile, and no barrier stands
// in its loop.  Scores are computed transposed, S^T = K Q^T, so that a lane holds one
// row's scores: the running maximum takes two lane exchanges, the sum none, and the
// weights are already the B operand of O^T = V^T P^T when the positions of a block are
// numbered as the score tiles leave them (k slot 8 b + e is position 4 b + e of the first
// tile for e < 4 and 4 b + e - 4 of the second otherwise).  K comes from memory as the A
// operand; V goes through LDS, whose transposing reads turn rows of V into columns.
#include <algorithm>
#include <cmath>

#include "kv_pages.hpp"

namespace gfx950 {
namespace {

using h8 = _Float16 __attribute__((ext_vector_type(8)));
using f4 = float __attribute__((ext_vector_type(4)));
using u32x4 = unsigned __attribute__((ext_vector_type(4)));
using s16x4 = short __attribute__((ext_vector_type(4)));
using s16x8 = short __attribute__((ext_vector_type(8)));
using lds_s16x4 = __attribute__((address_space(3))) s16x4;

constexpr unsigned kWaves = 4;
constexpr unsigned kBlock = 32;           // positions of one step of a wave
constexpr unsigned kMinBlocks = 2 * kWaves;  // blocks a split is worth at least
constexpr float kLog2E = 1.4426950408889634F;

struct PagedAttnArgs {
  KvPages pages;
  SequenceList list;
  const __half* query;   // [count][tokens][q_heads][D]
  const float* gate;     // [count][tokens][q_heads][2 D] or null
  __half* output;        // [count][tokens][q_heads][D]
  float* partial_o;      // [rows][splits][D]
  float* partial_ml;     // [rows][splits][2]: maximum (of score * log2 e), sum
  uint32_t layer, tokens, q_heads, kv_heads, shared;
  uint32_t prefix_splits, own_splits;   // splits = their sum
  uint32_t prefix_tiles, own_tiles;     // row tiles of a KV head over all sequences / of one sequence
  uint32_t prefix_groups;               // workgroups of the prefix, before those of the sequences
  float scale;                          // log2(e) / sqrt(D)
};

// `blocks` blocks over at most `splits` splits: blocks per split, and the splits in use.
__device__ __forceinline__ uint32_t split_length(uint32_t blocks, uint32_t splits) {
  return max(kMinBlocks, (blocks + splits - 1) / splits);
}
__device__ __forceinline__ uint32_t splits_used(uint32_t blocks, uint32_t splits) {
  const uint32_t per = split_length(blocks, splits);
  return (blocks + per - 1) / per;
}
// Positions the batch's prefix covers: what the first sequence has of them.
__device__ __forceinline__ uint32_t prefix_length(const PagedAttnArgs& a) {
  return min(a.shared, a.pages.lengths[a.list.slot[0]]);
}
// A sequence's own positions run from the tile of 16 that holds the prefix's end.
__device__ __forceinline__ uint32_t own_blocks(uint32_t shared, uint32_t end) {
  return end > shared ? (end - (shared & ~15u) + kBlock - 1) / kBlock : 0u;
}

// Consecutive workgroups go to the eight XCDs in turn; the row tiles of one K/V range get
// numbers eight apart, so that they read it through the same L2.
__host__ __device__ inline uint32_t spread_groups(uint32_t ranges, uint32_t tiles) { return (ranges + 7) / 8 * 8 * tiles; }
__device__ __forceinline__ void unspread(uint32_t id, uint32_t tiles, uint32_t& range, uint32_t& tile) {
  const uint32_t eighth = id / 8;
  tile = eighth % tiles;
  range = eighth / tiles * 8 + id % 8;
}

__device__ __forceinline__ float max_over_quarters(float v) {
  v = fmaxf(v, __shfl_xor(v, 16));
  return fmaxf(v, __shfl_xor(v, 32));
}
__device__ __forceinline__ float sum_over_quarters(float v) {
  v += __shfl_xor(v, 16);
  return v + __shfl_xor(v, 32);
}

template <unsigned D>
constexpr unsigned kPitch = D + 16;  // halves per V row in LDS: rows of a transposing read fall on different banks

template <unsigned D, unsigned NQ>
constexpr std::size_t shared_bytes() {
  const std::size_t values = kWaves * kBlock * kPitch<D> * 2;
  const std::size_t merge = (kWaves - 1) * (D / 64) * NQ * 64 * 16 + kWaves * 16 * NQ * 8;
  return values > merge ? values : merge;
}

// One work item: rows first .. first + 16 NQ - 1 (of `rows`; row = (i * tokens + t) * group + g
// with i counted from `base`), KV head hk, positions [lo, hi) in blocks first_block ..
// last_block - 1 from position `start`, pages of sequence `slot`, result into split `split`.
template <unsigned D, unsigned NQ>
__device__ __forceinline__ void attend(const PagedAttnArgs& a, uint32_t base, uint32_t first, uint32_t rows, uint32_t hk,
                                       uint32_t slot, uint32_t start, uint32_t first_block, uint32_t last_block,
                                       uint32_t lo, uint32_t hi, uint32_t split, char* smem) {
  constexpr unsigned kSteps = D / 32;       // K-steps of the scores
  constexpr unsigned kTiles = D / 16;       // output tiles of 16 dims
  constexpr unsigned kLoads = kBlock * D / 8 / 64;  // 16-byte pieces of a block's V rows per lane
  const unsigned lane = threadIdx.x & 63u, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const unsigned n = lane & 15u, kb = lane >> 4;
  const uint32_t group = a.q_heads / a.kv_heads;
  const KvPages& pg = a.pages;
  const uint32_t in_page = (1u << pg.page_shift) - 1;

  // The lane's row of each row tile: its query as B operand, and the positions it sees.
  h8 q[NQ][kSteps];
  uint32_t visible[NQ], out_row[NQ];
  uint32_t least = 0xffffffffu;
#pragma unroll
  for (unsigned j = 0; j < NQ; ++j) {
    const uint32_t row = first + 16 * j + n;
    visible[j] = 0;
    out_row[j] = 0xffffffffu;
#pragma unroll
    for (unsigned s = 0; s < kSteps; ++s) q[j][s] = h8{};
    if (row < rows) {
      const uint32_t it = row / group, g = row - it * group, i = it / a.tokens, t = it - i * a.tokens;
      out_row[j] = ((base + i) * a.tokens + t) * a.q_heads + hk * group + g;
      visible[j] = min(pg.lengths[a.list.slot[base + i]] + t + 1, hi);
      const __half* src = a.query + static_cast<std::size_t>(out_row[j]) * D + 8 * kb;
#pragma unroll
      for (unsigned s = 0; s < kSteps; ++s) q[j][s] = *reinterpret_cast<const h8*>(src + 32 * s);
      least = min(least, visible[j]);
    }
  }
#pragma unroll
  for (unsigned d = 1; d < 16; d <<= 1) least = min(least, static_cast<uint32_t>(__shfl_xor(static_cast<int>(least), d)));
  least = __builtin_amdgcn_readfirstlane(least);

  const std::size_t plane = static_cast<std::size_t>(a.layer) * pg.page_count << pg.page_shift;
  const __half* keys = pg.key + plane * pg.row + hk * D;
  const __half* values = pg.value + plane * pg.row + hk * D;
  _Float16* vs = reinterpret_cast<_Float16*>(smem) + wave * kBlock * kPitch<D>;

  h8 kr[2][kSteps];
  u32x4 vr[kLoads];
  int32_t page[2];
  auto find_pages = [&](uint32_t at, int32_t (&out)[2]) __attribute__((always_inline)) {
#pragma unroll
    for (unsigned t = 0; t < 2; ++t) {
      out[t] = at + 16 * t < hi ? table_page(pg, slot, (at + 16 * t) >> pg.page_shift) : -1;
      out[t] = __builtin_amdgcn_readfirstlane(out[t]);
    }
  };
  // Missing tiles load page 0 of the pool (always there); their scores and values are masked.
  auto load_k = [&](uint32_t at, const int32_t (&p)[2]) __attribute__((always_inline)) {
#pragma unroll
    for (unsigned t = 0; t < 2; ++t) {
      const std::size_t row = (static_cast<std::size_t>(max(p[t], 0)) << pg.page_shift) + ((at + 16 * t + n) & in_page);
      const __half* src = keys + row * pg.row + 8 * kb;
#pragma unroll
      for (unsigned s = 0; s < kSteps; ++s) kr[t][s] = *reinterpret_cast<const h8*>(src + 32 * s);
    }
  };
  auto load_v = [&](uint32_t at, const int32_t (&p)[2]) __attribute__((always_inline)) {
#pragma unroll
    for (unsigned u = 0; u < kLoads; ++u) {
      const unsigned piece = lane + 64 * u, r = piece / (D / 8), c = piece % (D / 8);
      const std::size_t row = (static_cast<std::size_t>(max(p[u / (kLoads / 2)], 0)) << pg.page_shift) + ((at + r) & in_page);
      vr[u] = *reinterpret_cast<const u32x4*>(values + row * pg.row + 8 * c);
    }
  };

  f4 o[NQ][kTiles];
  float m[NQ], l[NQ];
#pragma unroll
  for (unsigned j = 0; j < NQ; ++j) {
    m[j] = -INFINITY;
    l[j] = 0.0F;
#pragma unroll
    for (unsigned d = 0; d < kTiles; ++d) o[j][d] = f4{0, 0, 0, 0};
  }

  uint32_t block = first_block + wave;
  if (block < last_block) {
    find_pages(start + block * kBlock, page);
    load_k(start + block * kBlock, page);
    load_v(start + block * kBlock, page);
  }
  for (; block < last_block; block += kWaves) {
    const uint32_t at = start + block * kBlock, next = at + kWaves * kBlock;
    const bool more = block + kWaves < last_block;
    int32_t next_page[2] = {-1, -1};
    if (more) find_pages(next, next_page);
    const bool edge = at < lo || at + kBlock > least || page[0] < 0 || page[1] < 0;
    // Scores of 32 positions, the lane's row in the columns.
    f4 s[NQ][2];
#pragma unroll
    for (unsigned j = 0; j < NQ; ++j) {
#pragma unroll
      for (unsigned t = 0; t < 2; ++t) s[j][t] = f4{0, 0, 0, 0};
    }
#pragma unroll
    for (unsigned st = 0; st < kSteps; ++st) {
#pragma unroll
      for (unsigned t = 0; t < 2; ++t) {
#pragma unroll
        for (unsigned j = 0; j < NQ; ++j) s[j][t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kr[t][st], q[j][st], s[j][t], 0, 0, 0);
      }
    }
    if (more) load_k(next, next_page);
    // Values into LDS as they lie in memory; rows no one sees become zeros (what a page
    // holds past a sequence's end may be anything, and 0 * NaN would be NaN).
    bool strange = false;  // an infinity or NaN among the values of an edge block
#pragma unroll
    for (unsigned u = 0; u < kLoads; ++u) {
      const unsigned piece = lane + 64 * u, r = piece / (D / 8), c = piece % (D / 8);
      if (edge) {
        if (at + r < lo || at + r >= hi || page[u / (kLoads / 2)] < 0) vr[u] = u32x4{0, 0, 0, 0};
#pragma unroll
        for (unsigned e = 0; e < 4; ++e) {
          strange |= (vr[u][e] & 0x7c00u) == 0x7c00u || (vr[u][e] & 0x7c000000u) == 0x7c000000u;
        }
      }
      *reinterpret_cast<u32x4*>(vs + r * kPitch<D> + 8 * c) = vr[u];
    }
    if (more) load_v(next, next_page);
    // Running maximum.  The stored maximum moves only when a row's grows by more than 8
    // (a factor of 256): weights stay below 2^8 and most blocks skip the rescaling.
    bool grown = false;
    float top[NQ];
#pragma unroll
    for (unsigned j = 0; j < NQ; ++j) {
      float best = -INFINITY;
#pragma unroll
      for (unsigned t = 0; t < 2; ++t) {
#pragma unroll
        for (unsigned r = 0; r < 4; ++r) {
          float x = s[j][t][r] * a.scale;
          if (edge) {
            const uint32_t position = at + 16 * t + 4 * kb + r;
            if (position < lo || position >= visible[j] || page[t] < 0) x = -INFINITY;
          }
          s[j][t][r] = x;
          best = fmaxf(best, x);
        }
      }
      top[j] = max_over_quarters(best);
      grown |= top[j] > m[j] + 8.0F;
    }
    if (__any(grown)) {
#pragma unroll
      for (unsigned j = 0; j < NQ; ++j) {
        const float next_m = fmaxf(m[j], top[j]);
        const float factor = next_m == -INFINITY ? 1.0F : __builtin_amdgcn_exp2f(m[j] - next_m);
        m[j] = next_m;
        l[j] *= factor;
#pragma unroll
        for (unsigned d = 0; d < kTiles; ++d) o[j][d] *= factor;
      }
    }
    // Weights as an fp16 pair p = hi + lo: two products carry about 22 bits of p, so the
    // output keeps the accuracy of an fp32 product.
    h8 hi_p[NQ], lo_p[NQ];
#pragma unroll
    for (unsigned j = 0; j < NQ; ++j) {
      const float floor = m[j] == -INFINITY ? 0.0F : m[j];
#pragma unroll
      for (unsigned t = 0; t < 2; ++t) {
#pragma unroll
        for (unsigned r = 0; r < 4; ++r) {
          const float p = __builtin_amdgcn_exp2f(s[j][t][r] - floor);
          s[j][t][r] = p;
          l[j] += p;
          const _Float16 h = static_cast<_Float16>(p);
          hi_p[j][4 * t + r] = h;
          lo_p[j][4 * t + r] = static_cast<_Float16>(p - static_cast<float>(h));
        }
      }
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
    if (edge && __any(strange)) {
      // A row must not meet the infinities and NaNs of positions it does not see: products
      // one by one, in fp32, for the positions it does.
#pragma unroll 1
      for (unsigned p = 0; p < kBlock; ++p) {
        const unsigned t = p / 16, owner = ((p % 16) / 4) * 16 + n, r = p % 4;
#pragma unroll
        for (unsigned j = 0; j < NQ; ++j) {
          float w = 0.0F;
#pragma unroll
          for (unsigned e = 0; e < 8; ++e) {
            const float v = __shfl(s[j][e / 4][e % 4], owner);
            if (e == 4 * t + r) w = v;
          }
          const bool seen = at + p >= lo && at + p < visible[j];
#pragma unroll
          for (unsigned d = 0; d < kTiles; ++d) {
#pragma unroll
            for (unsigned e = 0; e < 4; ++e) {
              const float v = static_cast<float>(vs[p * kPitch<D> + 16 * d + 4 * kb + e]);
              if (seen) o[j][d][e] += w * v;
            }
          }
        }
      }
    } else {
#pragma unroll
      for (unsigned d = 0; d < kTiles; ++d) {
        const _Float16* src = vs + (4 * kb + (n >> 2)) * kPitch<D> + 16 * d + 4 * (n & 3u);
        const s16x4 a0 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(src));
        const s16x4 a1 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(src + 16 * kPitch<D>));
        const h8 v = __builtin_bit_cast(h8, __builtin_shufflevector(a0, a1, 0, 1, 2, 3, 4, 5, 6, 7));
#pragma unroll
        for (unsigned j = 0; j < NQ; ++j) {
          o[j][d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v, lo_p[j], o[j][d], 0, 0, 0);
          o[j][d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v, hi_p[j], o[j][d], 0, 0, 0);
        }
      }
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
    page[0] = next_page[0];
    page[1] = next_page[1];
  }

  // Merge the four waves: a common maximum per row, then each wave sums one quarter of
  // the output dims (a lane holds the same row and dims in every wave).
  __syncthreads();  // the V rows are no longer needed
  f4* quarter = reinterpret_cast<f4*>(smem);                                              // [3][D / 64 * NQ][64]
  float2* ml = reinterpret_cast<float2*>(smem + (kWaves - 1) * (D / 64) * NQ * 64 * 16);  // [4][16 NQ]
#pragma unroll
  for (unsigned j = 0; j < NQ; ++j) {
    l[j] = sum_over_quarters(l[j]);
    if (l[j] != l[j] && m[j] == -INFINITY) m[j] = 0.0F;  // only NaN scores: the row is NaN, not empty
    if (kb == 0) ml[wave * 16 * NQ + 16 * j + n] = float2{m[j], l[j]};
  }
  __syncthreads();
  float best[NQ], total[NQ];
#pragma unroll
  for (unsigned j = 0; j < NQ; ++j) {
    best[j] = -INFINITY;
    total[j] = 0.0F;
#pragma unroll
    for (unsigned w = 0; w < kWaves; ++w) best[j] = fmaxf(best[j], ml[w * 16 * NQ + 16 * j + n].x);
#pragma unroll
    for (unsigned w = 0; w < kWaves; ++w) {
      const float2 v = ml[w * 16 * NQ + 16 * j + n];
      if (v.x != -INFINITY) total[j] += v.y * __builtin_amdgcn_exp2f(v.x - best[j]);
    }
    const float factor = m[j] == -INFINITY ? 0.0F : __builtin_amdgcn_exp2f(m[j] - best[j]);
#pragma unroll
    for (unsigned d = 0; d < kTiles; ++d) {
      if (m[j] != -INFINITY) o[j][d] *= factor;
    }
  }
  const uint32_t splits = a.prefix_splits + a.own_splits;
  constexpr unsigned kQuarter = D / 64;
#pragma unroll
  for (unsigned c = 0; c < kWaves; ++c) {
    if (wave != c) {
      const unsigned place = wave < c ? wave : wave - 1;
#pragma unroll
      for (unsigned d = 0; d < kQuarter; ++d) {
#pragma unroll
        for (unsigned j = 0; j < NQ; ++j) quarter[(place * kQuarter * NQ + d * NQ + j) * 64 + lane] = o[j][c * kQuarter + d];
      }
    }
    __syncthreads();
    if (wave == c) {
#pragma unroll
      for (unsigned j = 0; j < NQ; ++j) {
        if (out_row[j] != 0xffffffffu) {
          const std::size_t at = static_cast<std::size_t>(out_row[j]) * splits + split;
#pragma unroll
          for (unsigned d = 0; d < kQuarter; ++d) {
            f4 v = o[j][c * kQuarter + d];
#pragma unroll
            for (unsigned w = 0; w < kWaves - 1; ++w) v += quarter[(w * kQuarter * NQ + d * NQ + j) * 64 + lane];
            *reinterpret_cast<f4*>(a.partial_o + at * D + 16 * (c * kQuarter + d) + 4 * kb) = v;
          }
          if (c == 0 && kb == 0) *reinterpret_cast<float2*>(a.partial_ml + 2 * at) = float2{best[j], total[j]};
        }
      }
    }
    __syncthreads();
  }
}

template <unsigned D, unsigned NQP, unsigned NQS>
__global__ __launch_bounds__(kWaves * 64) void paged_attention_kernel(PagedAttnArgs a) {
  constexpr std::size_t kBytes = std::max(shared_bytes<D, NQP>(), shared_bytes<D, NQS>());
  __shared__ __align__(16) char smem[kBytes];
  const uint32_t shared = prefix_length(a);
  const uint32_t group = a.q_heads / a.kv_heads, count = a.list.count;
  uint32_t range, tile;
  if (blockIdx.x < a.prefix_groups) {
    unspread(blockIdx.x, a.prefix_tiles, range, tile);
    const uint32_t split = range / a.kv_heads, hk = range - split * a.kv_heads;
    const uint32_t blocks = (shared + kBlock - 1) / kBlock, per = split_length(blocks, a.prefix_splits);
    const uint32_t from = split * per;
    if (split >= a.prefix_splits || from >= blocks) return;
    const uint32_t to = min(from + per, blocks);
    attend<D, NQP>(a, 0, tile * 16 * NQP, count * a.tokens * group, hk, a.list.slot[0], 0, from, to, 0, shared, split, smem);
    return;
  }
  unspread(blockIdx.x - a.prefix_groups, a.own_tiles, range, tile);
  const uint32_t hk = range % a.kv_heads, is = range / a.kv_heads, split = is / count, i = is - split * count;
  if (split >= a.own_splits) return;
  const uint32_t slot = a.list.slot[i], end = a.pages.lengths[slot] + a.tokens;
  const uint32_t blocks = own_blocks(shared, end), per = split_length(blocks, a.own_splits), from = split * per;
  if (from >= blocks) return;
  const uint32_t to = min(from + per, blocks);
  attend<D, NQS>(a, i, tile * 16 * NQS, a.tokens * group, hk, slot, shared & ~15u, from, to, shared, end,
                 a.prefix_splits + split, smem);
}

// Merges a row's items and applies the gate: one wave per (row, 128 dims), two dims a lane.
template <unsigned D>
__global__ __launch_bounds__(256) void paged_combine_kernel(PagedAttnArgs a) {
  constexpr unsigned kGroups = D / 128;
  const uint32_t linear = blockIdx.x * 4u + (threadIdx.x >> 6);
  const uint32_t rows = a.list.count * a.tokens * a.q_heads;
  if (linear >= rows * kGroups) return;
  const unsigned lane = threadIdx.x & 63u;
  const uint32_t row = linear / kGroups, part = linear - row * kGroups;
  const uint32_t i = row / (a.tokens * a.q_heads);
  const unsigned d = 128 * part + 2 * lane;
  float2 g = {0.0F, 0.0F};
  if (a.gate != nullptr) g = *reinterpret_cast<const float2*>(a.gate + static_cast<std::size_t>(row) * 2 * D + D + d);
  const uint32_t shared = prefix_length(a), end = a.pages.lengths[a.list.slot[i]] + a.tokens;
  const uint32_t prefix = a.prefix_splits != 0 ? splits_used((shared + kBlock - 1) / kBlock, a.prefix_splits) : 0u;
  const uint32_t own = splits_used(own_blocks(shared, end), a.own_splits);
  const std::size_t first = static_cast<std::size_t>(row) * (a.prefix_splits + a.own_splits);
  float best = -INFINITY;
  auto at = [&](uint32_t s) { return first + (s < prefix ? s : a.prefix_splits + (s - prefix)); };
  for (uint32_t s = 0; s < prefix + own; ++s) best = fmaxf(best, a.partial_ml[2 * at(s)]);
  float total = 0.0F, o0 = 0.0F, o1 = 0.0F;
  for (uint32_t s = 0; s < prefix + own; ++s) {
    const float2 ml = *reinterpret_cast<const float2*>(a.partial_ml + 2 * at(s));
    if (ml.x == -INFINITY) continue;
    const float w = __builtin_amdgcn_exp2f(ml.x - best);
    const float2 v = *reinterpret_cast<const float2*>(a.partial_o + at(s) * D + d);
    total = fmaf(ml.y, w, total);
    o0 = fmaf(v.x, w, o0);
    o1 = fmaf(v.y, w, o1);
  }
  float y0 = 0.0F, y1 = 0.0F;
  if (best != -INFINITY) {
    y0 = o0 / total;
    y1 = o1 / total;
  }
  if (a.gate != nullptr) {
    y0 *= 1.0F / (1.0F + expf(-g.x));
    y1 *= 1.0F / (1.0F + expf(-g.y));
  }
  __half* out = a.output + static_cast<std::size_t>(row) * D + d;
  *reinterpret_cast<__half2*>(out) = __halves2half2(to_half(y0), to_half(y1));
}

// Row tiles per wave: as few as hold the rows, at most 4 (2 at head size 256, whose rows
// take twice the registers).
unsigned row_tiles(uint32_t rows, uint32_t head_size) {
  const unsigned tiles = (rows + 15) / 16;
  if (tiles <= 1) return 1;
  return tiles == 2 || head_size == 256 ? 2 : 4;
}

struct Shape {
  unsigned prefix_nq, own_nq;
  uint32_t prefix_tiles, own_tiles, prefix_splits, own_splits;
  std::size_t rows;
};

// Workgroups that fill the GPU.
constexpr uint32_t kWantedGroups = 2 * kComputeUnits;

Shape shape_of(const KvPages& p, uint32_t kv_heads, uint32_t head_size, uint32_t count, uint32_t tokens, uint32_t q_heads,
               uint32_t shared) {
  Shape s{};
  const uint32_t group = q_heads / kv_heads;
  s.rows = static_cast<std::size_t>(count) * tokens * q_heads;
  auto splits = [](uint32_t ranges, uint64_t positions) {
    const uint64_t most = std::max<uint64_t>(1, (positions + kBlock - 1) / kBlock / kMinBlocks);
    return static_cast<uint32_t>(std::min<uint64_t>(most, std::max(1u, kWantedGroups / ranges)));
  };
  const uint32_t all = count * tokens * group, one = tokens * group;
  s.prefix_nq = shared != 0 ? row_tiles(all, head_size) : 1;
  s.own_nq = row_tiles(one, head_size);
  s.prefix_tiles = (all + 16 * s.prefix_nq - 1) / (16 * s.prefix_nq);
  s.own_tiles = (one + 16 * s.own_nq - 1) / (16 * s.own_nq);
  s.prefix_splits = shared != 0 ? splits(s.prefix_tiles * kv_heads, shared) : 0;
  const uint64_t capacity = static_cast<uint64_t>(p.stride) << p.page_shift;
  s.own_splits = splits(s.own_tiles * kv_heads * count, capacity > shared ? capacity - shared : 1);
  return s;
}

std::size_t partial_bytes(const Shape& s, uint32_t head_size) {
  return s.rows * (s.prefix_splits + s.own_splits) * (head_size + 2) * sizeof(float);
}

int32_t read_batch(const gfxinfer_kv_pages* pages, uint32_t count, uint32_t tokens, uint32_t q_heads, size_t shared, KvPages& p) {
  if (const int32_t s = read_pages(pages, p); s != GFXI_OK) return s;
  if (count == 0 || count > kMaxListed || tokens == 0 || tokens > 32 || q_heads == 0 || q_heads > 1024 ||
      q_heads % pages->kv_heads != 0 || shared > static_cast<uint64_t>(p.stride) << p.page_shift) {
    return fail(GFXI_INVALID_ARGUMENT, "invalid paged attention arguments (1..512 sequences, 1..32 tokens, query heads a "
                                       "multiple of the KV heads, a shared prefix within the table)");
  }
  return GFXI_OK;
}

template <unsigned D, unsigned NQP, unsigned NQS>
void launch(const PagedAttnArgs& a, dim3 grid, hipStream_t stream) {
  hipLaunchKernelGGL((paged_attention_kernel<D, NQP, NQS>), grid, dim3(kWaves * 64), 0, stream, a);
}

template <unsigned D, unsigned NQP>
void launch_own(unsigned own, const PagedAttnArgs& a, dim3 grid, hipStream_t stream) {
  if (own == 1) return launch<D, NQP, 1>(a, grid, stream);
  if (own == 2) return launch<D, NQP, 2>(a, grid, stream);
  if constexpr (D == 128) launch<D, NQP, 4>(a, grid, stream);
}

}  // namespace
}  // namespace gfx950

using namespace gfx950;

extern "C" size_t gfxinfer_kv_pages_attention_workspace_bytes(const gfxinfer_kv_pages* pages, uint32_t count, uint32_t tokens,
                                                              uint32_t q_heads, size_t shared_tokens) {
  size_t bytes = 0;
  guarded([&] {
    KvPages p;
    const int32_t s = read_batch(pages, count, tokens, q_heads, shared_tokens, p);
    if (s == GFXI_OK) {
      bytes = partial_bytes(shape_of(p, pages->kv_heads, pages->head_size, count, tokens, q_heads,
                                     static_cast<uint32_t>(shared_tokens)), pages->head_size);
    }
    return s;
  });
  return bytes;
}

extern "C" int32_t gfxinfer_launch_kv_pages_gated_attention(const gfxinfer_kv_pages* pages, uint32_t layer, const uint16_t* query,
                                                            const float* gate, uint16_t* output, const uint32_t* sequences,
                                                            uint32_t count, uint32_t tokens, uint32_t q_heads,
                                                            size_t shared_tokens, float* workspace, size_t workspace_bytes,
                                                            void* stream) {
  return guarded([&] {
    PagedAttnArgs a{};
    if (const int32_t s = read_batch(pages, count, tokens, q_heads, shared_tokens, a.pages); s != GFXI_OK) return s;
    if (const int32_t s = read_sequences(a.pages, sequences, count, false, a.list); s != GFXI_OK) return s;
    if (layer >= a.pages.layers || query == nullptr || output == nullptr || !aligned16(query) ||
        (reinterpret_cast<uintptr_t>(output) & 3u) != 0 || (reinterpret_cast<uintptr_t>(gate) & 7u) != 0) {
      return fail(GFXI_INVALID_ARGUMENT, "paged attention needs a layer of the cache and aligned rows (query 16 bytes, gate 8, "
                                         "output 4)");
    }
    const uint32_t head_size = pages->head_size, kv_heads = pages->kv_heads;
    const Shape shape = shape_of(a.pages, kv_heads, head_size, count, tokens, q_heads, static_cast<uint32_t>(shared_tokens));
    if (workspace == nullptr || !aligned16(workspace) || workspace_bytes < partial_bytes(shape, head_size)) {
      return fail(GFXI_INVALID_ARGUMENT, "paged attention workspace is null, not 16-byte aligned or too small");
    }
    a.query = reinterpret_cast<const __half*>(query);
    a.gate = gate;
    a.output = reinterpret_cast<__half*>(output);
    a.partial_o = workspace;
    a.partial_ml = workspace + shape.rows * (shape.prefix_splits + shape.own_splits) * head_size;
    a.layer = layer;
    a.tokens = tokens;
    a.q_heads = q_heads;
    a.kv_heads = kv_heads;
    a.shared = static_cast<uint32_t>(shared_tokens);
    a.prefix_splits = shape.prefix_splits;
    a.own_splits = shape.own_splits;
    a.prefix_tiles = shape.prefix_tiles;
    a.own_tiles = shape.own_tiles;
    a.prefix_groups = spread_groups(shape.prefix_splits * kv_heads, shape.prefix_tiles);
    a.scale = kLog2E / std::sqrt(static_cast<float>(head_size));
    const uint64_t groups = a.prefix_groups + static_cast<uint64_t>(spread_groups(shape.own_splits * count * kv_heads, shape.own_tiles));
    if (groups > (1u << 23)) return fail(GFXI_INVALID_ARGUMENT, "paged attention over too many rows for one launch");
    const dim3 grid(static_cast<unsigned>(groups));
    const hipStream_t st = static_cast<hipStream_t>(stream);
    if (head_size == 128) {
      if (shape.prefix_nq == 1) launch_own<128, 1>(shape.own_nq, a, grid, st);
      else if (shape.prefix_nq == 2) launch_own<128, 2>(shape.own_nq, a, grid, st);
      else launch_own<128, 4>(shape.own_nq, a, grid, st);
    } else {
      if (shape.prefix_nq == 1) launch_own<256, 1>(shape.own_nq, a, grid, st);
      else launch_own<256, 2>(shape.own_nq, a, grid, st);
    }
    if (const int32_t s = launch_status("paged attention launch failed"); s != GFXI_OK) return s;
    const dim3 combine(static_cast<unsigned>((shape.rows * (head_size / 128) + 3) / 4));
    if (head_size == 128) hipLaunchKernelGGL(paged_combine_kernel<128>, combine, dim3(256), 0, st, a);
    else hipLaunchKernelGGL(paged_combine_kernel<256>, combine, dim3(256), 0, st, a);
    return launch_status("paged attention combine launch failed");
  });
}
