// Gated GQA attention of ragged chunks of new tokens over the pages of a K/V cache.
//
// Row (t, g) of a listed sequence and a KV head, new token t at query head g of the head's
// group, attends to the first length + t + 1 positions:
//     o = softmax(q . K / sqrt(D)) . V * sigmoid(gate),   L = log(sum exp(q . K / sqrt(D)))
// The rows of a sequence and KV head are one tall matrix, in tiles of 128: a workgroup takes a tile
// and a range of positions, each of its four waves 32 of the rows, and a K / V row staged in LDS
// serves them all.  A second launch joins the ranges of a tile.  (Equal shares of all work, one a
// workgroup and cut anywhere, took 16 % longer: 2048 tokens on 30000.  Workgroups that
// go over the same positions of a head at the same time read them through one L2, those shares
// did not.)
//
// Scores are computed transposed, S^T = K Q^T (v_mfma_f32_32x32x16_f16), so that a lane holds
// half of one row's scores, the running maximum takes one lane exchange, and the weights are
// already the B operand of O^T = V^T P^T when the positions of a step are numbered as the score
// tiles leave them (k slot 8 h + e is position 4 h + e % 4 + 8 (e / 4), h the lane's half).  V
// passes through LDS, whose transposing reads turn rows of V into columns.
//
// The scores of a tile of positions are computed beside the exponentials of the tile before it:
// the exponentials alone take a wave's vector unit nearly as long as both products take the
// matrix unit.
//
// 2048 tokens on 30000, 40 x 8 x 128: 1355 us, 960 TFLOP/s (a large fp16 product: 1.28 PFLOP/s; other cards up to 1445 us); the
// matrix units are busy 48 % of the time, waits take 23 % of the waves'.  24 x 4 x 256: 1850 to 1910 us, 830 TFLOP/s: the outputs of
// 32 rows leave room for one wave a SIMD, and nothing covers its waits.  31 sequences that decode on 200 .. 4090 and a chunk
// of 509: 78 us, 3.6 TB/s.  Eight that decode on up to 600: 14.7 us, two launches of dependent reads.
#include <algorithm>
#include <array>
#include <cmath>
#include <numeric>
#include <type_traits>
#include <vector>

#include "kv_attention.hpp"
#include "kv_weights.hpp"

namespace gfx950 {
namespace {

using f16v = float __attribute__((ext_vector_type(16)));
using h4 = _Float16 __attribute__((ext_vector_type(4)));
using lds_s16x4 = __attribute__((address_space(3))) s16x4;

constexpr unsigned kWaves = 4;
constexpr float kLn2 = 0.6931471805599453F;

constexpr unsigned kRows = kWaves * 32;    // of a row tile
template <unsigned D>
constexpr unsigned kTile = 8192 / D;        // positions of a step: 16 KB of K and of V; two of each in LDS
// Workgroups a CU holds: at head size 256 the outputs and queries of 32 rows alone are 192 of the 256
// registers that two waves of a SIMD would have each.
template <unsigned D>
constexpr unsigned kResident = D == 128 ? 2 : 1;

// A row's weights are 2^(score - m + kLift), scores in units of log2.  m is a maximum of the row so far that moves up
// once it is passed by kRise, so weights stay below 2^15.  Tiles of more than 32 rows carry a weight as one fp16
// number: 11 bits, half the size of the output's own rounding.  A second product for 22 bits takes 40 % longer (2048 tokens on
// 30000 2025 us, on the same card 1445).  Tiles of at most 32 rows wait for memory and carry pairs.
//
// fp16 rounds weights below 2^kSmall by 2^-25 and drops those below that.  Beside peaks whose values are near zero they
// may be all that carries the output (26 nats below a peak, 42 % of 4096 of them was lost).  So a row is open until
// its weights below 2^kPeak sum up to n kMean, n the positions beside one that it sees: then less than 2^-10 of their sum is
// lost where they spread by 3 nats, nothing where they spread by one, and 2^-7 were one weight the sum and all others just too
// small.  (Or until all its weights sum up to kMany: then 16 positions or more are peaks.)  Steps look for that
// until a row has kAmple times as much.  Where small weights were met and the row is open to the end, two more passes
// over the range take what lies below the peaks, with a maximum of its own, and the peaks.
//
// (Products of their own for small weights where they are met took 5 to 17 % of all calls' time by their presence alone,
// as a branch between the products of a step.  A call takes as long as its slowest tile, so what one tile goes over again
// shows: 2048 tokens on 30000 with scores that spread by 3 nats 1590 us, not 1530; by 6 nats 3600, not 1490.)
constexpr float kLift = 11.0F, kRise = 4.0F, kSmall = -14.0F, kPeak = 8.0F, kMean = 0x1p-18F, kMany = 0x1p19F, kAmple = 256.0F;

constexpr float kWritten = -1.0F;  // in the place of range 0's sum: the row is complete, nothing to join

struct ChunkAttnArgs {
  KvPages pages;
  ChunkList list;
  uint32_t first_tile[kMaxChunks];  // of the listed sequences' row tiles
  uint32_t tiles;
  uint32_t whole;        // tiles and KV heads that run first and are not divided, see partial_row
  uint32_t tile_rows;    // most rows of a divided tile
  const __half* query;   // [rows][q_heads][D]
  const float* gate;     // [rows][q_heads][2 D] or null
  __half* output;        // [rows][q_heads][D]
  float* log_sums;       // [rows][q_heads] or null
  float* partial_o;      // [partial rows][ranges][D], where positions are divided
  float* partial_ml;     // [partial rows][ranges][2]: maximum (-inf: the row has nothing there), sum
  uint32_t layer, q_heads, kv_heads, group, ranges;
  float scale;           // log2(e) / sqrt(D)
};

// Where a row's parts are.  If all tiles are divided: by its place in the output, [rows][q_heads].  Otherwise by the
// divided tile (and KV head) that it is in, [divided][tile_rows], so that they take no room for the whole ones (2048 tokens
// of 40 x 8 x 128: 32 MB, by their place 163; 32800 tokens 4 MB, not 2.6 GB).
__device__ __forceinline__ uint32_t partial_row(const ChunkAttnArgs& a, uint32_t item, uint32_t row_of_tile, uint32_t out_row) {
  return a.whole == 0 ? out_row : (item - a.whole) * a.tile_rows + row_of_tile;
}

// Steps a range holds at least, if there is more than one.
constexpr uint32_t kLeastSteps = 2;

// The listed sequence of a row tile, and the steps of a range: ranges are of equal length for all
// sequences, the longest one with new tokens is divided into as many as the launch allows and the others into as few
// as hold them.  The list and the lengths take one round of loads each, a lane a sequence; the first pages of the
// sequence's table come beside its length.
struct Listed {
  uint32_t slot, length, first_row, tokens, first_tile, per;
};
template <unsigned D>
__device__ __forceinline__ Listed find_listed(const ChunkAttnArgs& a, uint32_t row_tile, PageWindow& window) {
  const unsigned lane = threadIdx.x & 63u;
  Listed found{};
  uint32_t most = 0;
  for (uint32_t from = 0; from < a.list.count; from += 64) {
    const uint32_t i = min(from + lane, a.list.count - 1);
    const uint32_t slot = a.list.slot[i], row = a.list.first[i], tokens = a.list.first[i + 1] - row;
    const uint32_t tile = a.first_tile[i], next_tile = tile + (tokens * a.group + kRows - 1) / kRows;
    const uint32_t committed = a.pages.lengths[slot];
    const uint64_t here = __ballot(from + lane < a.list.count && tile <= row_tile && row_tile < next_tile);
    const int at = here != 0 ? __ffsll(static_cast<unsigned long long>(here)) - 1 : 0;
    auto take = [&](uint32_t x) { return static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(x), at)); };
    if (here != 0) window.start(a.pages, take(slot), 0);
    const uint32_t length = min(committed, a.pages.stride << a.pages.page_shift);
    most = max(most, tokens != 0 ? length + tokens : 0);
    if (here != 0) found = Listed{take(slot), take(length), take(row), take(tokens), take(tile), 0};
  }
#pragma unroll
  for (unsigned d = 1; d < 64; d <<= 1) most = max(most, static_cast<uint32_t>(__shfl_xor(static_cast<int>(most), d)));
  const uint32_t steps = (__builtin_amdgcn_readfirstlane(most) + kTile<D> - 1) / kTile<D>;
  found.per = a.ranges == 1 ? 0xffffffffu : max(kLeastSteps, (steps + a.ranges - 1) / a.ranges);
  return found;
}

__device__ __forceinline__ float max_over_halves(float v) {
  const unsigned u = __float_as_uint(v);
  const auto p = __builtin_amdgcn_permlane32_swap(u, u, false, false);
  return __builtin_elementwise_maximum(__uint_as_float(p[0]), __uint_as_float(p[1]));
}
__device__ __forceinline__ float sum_over_halves(float v) {
  const unsigned u = __float_as_uint(v);
  const auto p = __builtin_amdgcn_permlane32_swap(u, u, false, false);
  return __uint_as_float(p[0]) + __uint_as_float(p[1]);
}

// What a row has found of weights beside its peaks.
struct Found {
  float others;  // the sum of weights below 2^kPeak as far as it was looked for
  float small;   // 1: small weights were met on the way
};
__device__ __forceinline__ Found& found_at(Found& found) { return found; }
__device__ __forceinline__ Found& found_at(Found* found) { return *found; }

// A row's maximum, and whether its small weights may matter.  Place: Found, or Found* in LDS where registers, scalar ones
// too, are all taken.  (The compiler lets a read of LDS wait for all loads into LDS that are on their way: it takes
// tiles of few rows 1 to 3 % of their time.)
template <typename Place>
struct Peaks {
  float m;
  Place found;
  bool looks;  // a row of the wave looks for more

  __device__ __forceinline__ void clear() {
    m = -INFINITY;
    found_at(found) = Found{0.0F, 0.0F};
    looks = false;
  }
  __device__ __forceinline__ bool moves(float top) const { return __any(!(top <= m + kRise)) || looks; }
  // Whether a row has `share` times what it needs.  all: the sum of its weights; positions: what it sees in all steps, one at
  // least.
  __device__ __forceinline__ bool has(float share, float others, float all, uint32_t positions) const {
    return m == -INFINITY || others >= kMean * share * static_cast<float>(positions - 1) || all >= kMany;
  }
  // A step that moves: the raw scores s(0) .. s(N - 1) of a lane's half of its row, the largest of the row, `top`, and the
  // lane's sum of weights before this step.  Returns the factor of the sums so far.
  template <bool Look, unsigned N, typename Score>
  __device__ __forceinline__ float move(Score s, float scale, float top, uint32_t positions, float before) {
    const float next = top <= m + kRise ? m : top;
    // From nothing to something: there is nothing to scale yet.
    const float factor = next == m || m == -INFINITY ? 1.0F : rescale_factor(m, next);
    if constexpr (Look) {
      Found now = found_at(found);
      const float all = sum_over_halves(before) * factor;
      // After a rise by so much none of the weights so far is a peak.
      now.others = m != -INFINITY && next - m >= kLift + kRise - kPeak ? all : now.others * factor;
      m = next;
      looks = !__all(has(kAmple, now.others, all, positions));
      if (looks) {
        float here = 0.0F;
        bool small = false;
#pragma unroll
        for (unsigned e = 0; e < N; ++e) {
          const float x = fmaf(s(e), scale, kLift - m);
          here += x < kPeak ? __builtin_amdgcn_exp2f(x) : 0.0F;
          small |= x < kSmall && x > -INFINITY;
        }
        now.others += sum_over_halves(here);
        if (small) now.small = 1.0F;
        looks = !__all(has(kAmple, now.others, all, positions));
      }
      found_at(found) = now;
    }
    m = next;
    return factor;
  }
  // Rows that do not have enough where small weights were met, a bit a lane.
  __device__ __forceinline__ uint64_t open(float all, uint32_t positions) {
    const Found now = found_at(found);
    const uint64_t small = __ballot(now.small != 0.0F);
    return (small | small >> 32 | small << 32) & ~__ballot(has(1.0F, now.others, sum_over_halves(all), positions));
  }
};

// The scores that a careful pass takes, of a lane's row: above x, up to y.  In LDS.
struct Limits {
  float2* scores;
  // All, but for the rows `taken`: those below their peaks.
  __device__ __forceinline__ void below_peaks(float m, uint64_t taken) const {
    scores[threadIdx.x] = float2{-INFINITY, (taken >> (threadIdx.x & 63u) & 1u) != 0 ? m - kLift + kPeak : INFINITY};
  }
  // The peaks; none of the other rows, which are complete.
  __device__ __forceinline__ void peaks() const { scores[threadIdx.x] = float2{scores[threadIdx.x].y, INFINITY}; }
};

// V rows in LDS: piece c of row r lies in slot c ^ 4 (r % 4), so that the four rows of 64 bytes that half
// a wave reads at once (a transposing read of 32 columns) fall on different banks.
__device__ __forceinline__ unsigned value_slot4(unsigned piece, unsigned row) { return piece ^ 4 * (row & 3u); }

// What the waves of a workgroup need of a range of positions of one row tile.
struct Range {
  uint32_t slot, end, from, to, hk;  // steps [from, to)
  uint32_t least;                    // positions that all rows see
};

// Where a lane's part of the first output tile of 16 V rows lies in LDS, in bytes; output tile d is at
// the place ^ 64 d (see the attention kernel).
template <unsigned D>
__device__ __forceinline__ unsigned value_place_of(unsigned lane) {
  const unsigned i16 = lane & 15u, vrow = 4 * (lane >> 5) + (i16 >> 2);
  return vrow * (2 * D) + 16 * value_slot4(2 * (lane >> 4 & 1u) + ((i16 & 3u) >> 1), vrow) + 8 * (i16 & 1u);
}

// Output tiles first .. first + 3 of 16 V rows in LDS, complete when they return.  (The compiler would let
// reads of its own wait for the next block's loads into LDS, which it cannot tell from this block's.)
template <unsigned D, unsigned Rows>
__device__ __forceinline__ void read_tiles(unsigned place, unsigned first, h8 (&v)[4]) {
  s16x4 x[8];
  asm volatile(
      "ds_read_b64_tr_b16 %0, %8 offset:%12\n\tds_read_b64_tr_b16 %1, %8 offset:%13\n\t"
      "ds_read_b64_tr_b16 %2, %9 offset:%12\n\tds_read_b64_tr_b16 %3, %9 offset:%13\n\t"
      "ds_read_b64_tr_b16 %4, %10 offset:%12\n\tds_read_b64_tr_b16 %5, %10 offset:%13\n\t"
      "ds_read_b64_tr_b16 %6, %11 offset:%12\n\tds_read_b64_tr_b16 %7, %11 offset:%13\n\t"
      "s_waitcnt lgkmcnt(0)"
      : "=&v"(x[0]), "=&v"(x[1]), "=&v"(x[2]), "=&v"(x[3]), "=&v"(x[4]), "=&v"(x[5]), "=&v"(x[6]), "=&v"(x[7])
      : "v"(place ^ 64 * first), "v"(place ^ 64 * (first + 1)), "v"(place ^ 64 * (first + 2)), "v"(place ^ 64 * (first + 3)),
        "n"(Rows * 2 * D), "n"((Rows + 8) * 2 * D)
      : "memory");
#pragma unroll
  for (unsigned d = 0; d < 4; ++d) {
    v[d] = __builtin_bit_cast(h8, __builtin_shufflevector(x[2 * d], x[2 * d + 1], 0, 1, 2, 3, 4, 5, 6, 7));
  }
}

// A tile of at most 32 rows, as a decoding sequence has: all waves take the same rows and divide the
// positions, blocks of 32 in turn.  K goes straight into registers, V through a part of LDS of the
// wave's own, both a block ahead and without a barrier.  The waves' results meet in LDS at the end;
// wave w leaves with output tiles w, w + 4 .. of all 32 rows in o[0], o[1] .., and with the rows'
// maxima and sums.
template <unsigned D>
__device__ __forceinline__ void attend_few(const ChunkAttnArgs& a, const Range& w, const h8 (&q)[D / 16], uint32_t visible,
                                           _Float16* (&lds)[kWaves], const Limits& limit, PageWindow& window, f16v (&o)[D / 32], float& m, float& l) {
  constexpr unsigned kBlock = 32, kLoadRows = 512 / D, kLoads = kBlock / kLoadRows;
  const unsigned lane = threadIdx.x & 63u, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const unsigned n = lane & 31u, h = lane >> 5;
  const KvPages& pg = a.pages;
  const uint32_t in_page = (1u << pg.page_shift) - 1, row_bytes = 2 * pg.row;
  const std::size_t layer_row = (static_cast<std::size_t>(a.layer) * pg.page_count << pg.page_shift) * pg.row + w.hk * D;
  const __half* keys = pg.key + layer_row;
  const __half* values = pg.value + layer_row;
  _Float16* vs = wave == 0 ? lds[0] : wave == 1 ? lds[1] : wave == 2 ? lds[2] : lds[3];  // two blocks
  const uint32_t load_row = lane / (D / 8);
  const uint32_t value_part = load_row * row_bytes + 16 * value_slot4(lane % (D / 8), load_row);
  const unsigned value_place = lds_address(vs) + value_place_of<D>(lane);
  const uint32_t first = w.from * kTile<D> / kBlock + wave, last = min(w.to * kTile<D>, w.end + kBlock - 1) / kBlock;
  h8 k[D / 16];
  int32_t page[2];  // of the block's halves, -1: none; these load from page 0 of the pool (always there)
  // Block b's K rows into k, its V rows into the part `to`.
  auto load = [&](uint32_t b, unsigned to) __attribute__((always_inline)) {
    const uint32_t at = b * kBlock;
#pragma unroll
    for (unsigned e = 0; e < 2; ++e) page[e] = at + 16 * e < w.end ? window.find(pg, w.slot, (at + 16 * e) >> pg.page_shift) : -1;
    const uint32_t p = static_cast<uint32_t>(max(n < 16 ? page[0] : page[1], 0));
    const __half* row = keys + ((static_cast<std::size_t>(p) << pg.page_shift) + ((at + n) & in_page)) * pg.row + 8 * h;
#pragma unroll
    for (unsigned st = 0; st < D / 16; ++st) k[st] = *reinterpret_cast<const h8*>(row + 16 * st);
#pragma unroll
    for (unsigned u = 0; u < kLoads; ++u) {
      const unsigned row0 = kLoadRows * u, e = row0 / 16;
      const std::size_t base = ((static_cast<std::size_t>(max(page[e], 0)) << pg.page_shift) + ((at + 16 * e) & in_page)) * pg.row;
      const auto rows16 = __builtin_amdgcn_make_buffer_rsrc(const_cast<__half*>(values + base), 0, static_cast<int>(15 * row_bytes + 2 * D), 0x20000);
      __builtin_amdgcn_raw_ptr_buffer_load_lds(rows16, (lds_void*)(vs + (to * kBlock + row0) * D), 16, static_cast<int>(value_part ^ 64 * (row0 & 3u)),
                                               static_cast<int>((row0 & 15u) * row_bytes), 0, 0);
    }
  };
  Peaks<Found> row{-INFINITY, Found{0.0F, 0.0F}, false};
  // A weight is high + low, both rounded to nearest: off by 2^-23 of itself, or by 2^-25 if that is more.
  auto rest_of = [](float x, _Float16 high) __attribute__((always_inline)) { return static_cast<_Float16>(x - static_cast<float>(high)); };
  // What a row sees of the wave's blocks: whole ones, and one in part.
  const uint32_t cut = visible / kBlock, whole = cut > first ? (min(cut, last) - first + kWaves - 1) / kWaves * kBlock : 0;
  const uint32_t positions = max(1u, whole + (cut < last && cut % kWaves == first % kWaves ? visible % kBlock : 0));
  // Passes: the first one; a careful one, without the peaks of rows whose small weights may matter; those peaks.
  bool careful = false, apart = false, strange;
  row.clear();
  l = 0.0F;
#pragma unroll
  for (unsigned d = 0; d < D / 32; ++d) o[d] = f16v{};
#pragma unroll 1
  for (;;) {
    if (first < last) load(first, 0);
    unsigned in = 0;
#pragma unroll 1
    for (uint32_t b = first; b < last; b += kWaves, in ^= 1) {
      const uint32_t at = b * kBlock;
      const bool gone = page[0] < 0, upper_gone = page[1] < 0;  // of the halves
      f16v s = {};
#pragma unroll
      for (unsigned st = 0; st < D / 16; ++st) s = __builtin_amdgcn_mfma_f32_32x32x16_f16(k[st], q[st], s, 0, 0, 0);
      const bool more = b + kWaves < last;
      if (more) load(b + kWaves, in ^ 1);
      if (at + kBlock > w.least || gone || upper_gone) {
#pragma unroll
        for (unsigned r = 0; r < 16; ++r) {
          if (at + 8 * (r / 4) + 4 * h + r % 4 >= visible || (r < 8 ? gone : upper_gone)) s[r] = -INFINITY;
        }
      }
      if (careful) {
        const float2 limits = limit.scores[threadIdx.x];
#pragma unroll
        for (unsigned r = 0; r < 16; ++r) {
          if (s[r] * a.scale <= limits.x || s[r] * a.scale > limits.y) s[r] = -INFINITY;  // (not NaN)
        }
      }
      float best = s[0];
#pragma unroll
      for (unsigned r = 1; r < 16; ++r) best = __builtin_elementwise_maximum(best, s[r]);
      const float top = max_over_halves(best) * a.scale;
      if (row.moves(top)) {
        const float factor = row.move<true, 16>([&](unsigned e) { return s[e]; }, a.scale, top, positions, l);
        l *= factor;
        if (__any(factor != 1.0F)) {
#pragma unroll
          for (unsigned d = 0; d < D / 32; ++d) {
#pragma unroll
            for (unsigned r = 0; r < 16; ++r) o[d][r] *= factor;
          }
        }
      }
      const float floor = row.m == -INFINITY ? 0.0F : row.m - kLift;
      h8 high[2], low[2];
#pragma unroll
      for (unsigned r = 0; r < 16; ++r) {
        const float x = __builtin_amdgcn_exp2f(fmaf(s[r], a.scale, -floor));
        l += x;
        high[r / 8][r % 8] = static_cast<_Float16>(x);
        low[r / 8][r % 8] = rest_of(x, high[r / 8][r % 8]);
      }
      // The block's V rows are there when only the next block's loads are on their way.
      if (more) wait_loads<D / 16 + kLoads>();
      else wait_loads<0>();
      bool odd = false;
      if (careful || at + kBlock > w.end || gone || upper_gone) {  // as in the attention kernel
#pragma unroll 1
        for (unsigned u = 0; u < kLoads; ++u) {
          const unsigned row0 = kLoadRows * u;
          u32x4* piece = reinterpret_cast<u32x4*>(vs + (in * kBlock + row0) * D) + lane;
          if (at + row0 + load_row >= w.end || (row0 < 16 ? gone : upper_gone)) *piece = u32x4{0, 0, 0, 0};
          if (careful) odd |= take_strange(piece);
        }
        wait_loads<63>();
      }
      const unsigned place = value_place + in * (kBlock * 2 * D);
#pragma unroll
      for (unsigned d = 0; d < D / 32; d += 4) {
        h8 v[4];
        auto add = [&](unsigned half) __attribute__((always_inline)) {
#pragma unroll
          for (unsigned e = 0; e < 4; ++e) o[d + e] = __builtin_amdgcn_mfma_f32_32x32x16_f16(v[e], low[half], o[d + e], 0, 0, 0);
#pragma unroll
          for (unsigned e = 0; e < 4; ++e) o[d + e] = __builtin_amdgcn_mfma_f32_32x32x16_f16(v[e], high[half], o[d + e], 0, 0, 0);
        };
        read_tiles<D, 0>(place, d, v);
        add(0);
        read_tiles<D, 16>(place, d, v);
        add(1);
      }
      if (__any(odd)) {
        // The rows that see an infinity or NaN among the values get it, whatever the weight.
#pragma unroll 1
        for (unsigned x = 0; x < kBlock; ++x) {
          const int32_t one = at + x < w.end ? table_page(pg, w.slot, (at + x) >> pg.page_shift) : -1;
          if (one < 0) continue;
          const __half* v = values + ((static_cast<std::size_t>(one) << pg.page_shift) + ((at + x) & in_page)) * pg.row;
#pragma unroll
          for (unsigned d = 0; d < D / 32; ++d) {
#pragma unroll
            for (unsigned r = 0; r < 16; ++r) {
              const float y = __half2float(v[32 * d + 8 * (r / 4) + 4 * h + r % 4]);
              if (!(fabsf(y) < INFINITY) && at + x < visible) o[d][r] += y;
              asm volatile("" ::: "memory");
            }
          }
        }
      }
    }
    strange = false;
#pragma unroll
    for (unsigned d = 0; d < D / 32; ++d) {
#pragma unroll
      for (unsigned r = 0; r < 16; ++r) strange |= !(fabsf(o[d][r]) < INFINITY);
    }
    if (!careful) {
      const uint64_t taken = row.open(l, positions);
      if (!__any(strange) && taken == 0) break;
      careful = true;
      apart = taken != 0;
      limit.below_peaks(row.m, taken);
      row.clear();
      l = 0.0F;
#pragma unroll
      for (unsigned d = 0; d < D / 32; ++d) o[d] = f16v{};
    } else if (apart) {
      apart = false;
      limit.peaks();  // added to what is there
    } else {
      break;
    }
  }
  l = sum_over_halves(l);
  m = row.m;
  if ((m == -INFINITY && (l != l || (careful && strange))) || m != m) m = 0.0F;
  // The waves' results, four output tiles at a time.
  float2* ml = reinterpret_cast<float2*>(lds[0]);  // [waves][32], once V is no longer needed
  __syncthreads();
  if (h == 0) ml[wave * 32 + n] = float2{m, l};
  __syncthreads();
  float2 part[kWaves];
  float all = -INFINITY, total = 0.0F, factor[kWaves];
#pragma unroll
  for (unsigned v = 0; v < kWaves; ++v) {
    part[v] = ml[v * 32 + n];
    all = fmaxf(all, part[v].x);
  }
#pragma unroll
  for (unsigned v = 0; v < kWaves; ++v) {
    factor[v] = part[v].x == -INFINITY ? 0.0F : rescale_factor(part[v].x, all);
    if (part[v].x != -INFINITY) total += part[v].y * factor[v];
  }
  m = all;
  l = total;
  f16v sum[D / 128];
#pragma unroll
  for (unsigned g = 0; g < D / 128; ++g) {
    __syncthreads();
    f4* mine = reinterpret_cast<f4*>(vs);
#pragma unroll
    for (unsigned d = 0; d < 4; ++d) {
#pragma unroll
      for (unsigned e = 0; e < 4; ++e) mine[(4 * d + e) * 64 + lane] = f4{o[4 * g + d][4 * e], o[4 * g + d][4 * e + 1], o[4 * g + d][4 * e + 2], o[4 * g + d][4 * e + 3]};
    }
    __syncthreads();
    sum[g] = f16v{};
#pragma unroll
    for (unsigned v = 0; v < kWaves; ++v) {
      const f4* other = reinterpret_cast<const f4*>(lds[v]);
#pragma unroll
      for (unsigned e = 0; e < 4; ++e) {
        const f4 x = other[(4 * wave + e) * 64 + lane];
#pragma unroll
        for (unsigned c = 0; c < 4; ++c) {
          if (factor[v] != 0.0F) sum[g][4 * e + c] += x[c] * factor[v];
        }
      }
    }
  }
#pragma unroll
  for (unsigned g = 0; g < D / 128; ++g) o[g] = sum[g];
}

// Output tiles of a row: a range's part, or, where one range holds all positions, the row itself with
// the gate applied.  o[i] is output tile first + i * step; joined: the join goes over the row.
template <unsigned D, unsigned N>
__device__ __forceinline__ void write_row(const ChunkAttnArgs& a, uint32_t out_row, uint32_t part_row, uint32_t range, bool whole,
                                          bool joined, const f16v* o, unsigned first, unsigned step, float m, float l, bool sums) {
  const unsigned h = (threadIdx.x & 63u) >> 5;
  const std::size_t at = static_cast<std::size_t>(part_row) * a.ranges + range;
  if (!whole) {
#pragma unroll
    for (unsigned i = 0; i < N; ++i) {
#pragma unroll
      for (unsigned r = 0; r < 16; r += 4) {
        *reinterpret_cast<f4*>(a.partial_o + at * D + 32 * (first + i * step) + 2 * r + 4 * h) = f4{o[i][r], o[i][r + 1], o[i][r + 2], o[i][r + 3]};
      }
    }
    if (sums) *reinterpret_cast<float2*>(a.partial_ml + 2 * at) = float2{m, l};
    return;
  }
  const bool empty = m == -INFINITY;
  const float inverse = empty ? 0.0F : 1.0F / l;
#pragma unroll
  for (unsigned i = 0; i < N; ++i) {
#pragma unroll
    for (unsigned r = 0; r < 16; r += 4) {
      const unsigned at = 32 * (first + i * step) + 2 * r + 4 * h;
      f4 y;
#pragma unroll
      for (unsigned e = 0; e < 4; ++e) y[e] = empty ? 0.0F : o[i][r + e] * inverse;
      if (a.gate != nullptr) {
        const f4 gate = *reinterpret_cast<const f4*>(a.gate + static_cast<std::size_t>(out_row) * 2 * D + D + at);
#pragma unroll
        for (unsigned e = 0; e < 4; ++e) y[e] *= 1.0F / (1.0F + expf(-gate[e]));
      }
      h4 out;
#pragma unroll
      for (unsigned e = 0; e < 4; ++e) out[e] = static_cast<_Float16>(y[e]);
      *reinterpret_cast<h4*>(a.output + static_cast<std::size_t>(out_row) * D + at) = out;
    }
  }
  if (sums && joined) *reinterpret_cast<float2*>(a.partial_ml + 2 * at) = float2{0.0F, kWritten};
  if (sums && a.log_sums != nullptr) a.log_sums[out_row] = empty ? -INFINITY : (m - kLift) * kLn2 + logf(l);
}

// Sixteen-position parts of a tile: their pages, -1 where there is none.
template <unsigned D>
struct TilePages {
  int32_t page[kTile<D> / 16];
  uint32_t missing;
};

template <unsigned D>
__global__ __launch_bounds__(kWaves * 64, kResident<D>) void chunk_attention_kernel(ChunkAttnArgs a) {
  constexpr unsigned T = kTile<D>, kSub = T / 32, kSteps = T / 16;
  constexpr unsigned kLoadRows = 512 / D;                   // rows a load of a wave covers
  constexpr unsigned kLoads = T / kLoadRows / kWaves;       // of K, and of V, per tile and wave
  // Two tiles of K and of V; with few rows two blocks of V of a wave each.
  constexpr unsigned kPart = T * D > 2 * 32 * D ? T * D : 2 * 32 * D;
  __shared__ __align__(1024) _Float16 k0[kPart];
  __shared__ __align__(1024) _Float16 k1[kPart];
  __shared__ __align__(1024) _Float16 v0[kPart];
  __shared__ __align__(1024) _Float16 v1[kPart];
  __shared__ Found found[kWaves * 64];
  __shared__ float2 taken_scores[kWaves * 64];
  __shared__ uint32_t again[kWaves];       // the wave's rows met an infinity or NaN
  __shared__ uint32_t strange_tiles[32];   // bit x % 1024: a tile x holds infinities or NaNs among its values
  const Limits limit{taken_scores};
  const unsigned lane = threadIdx.x & 63u, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const unsigned n = lane & 31u, h = lane >> 5;
  const KvPages& pg = a.pages;
  // KV heads vary fastest: with eight of them each XCD reads one.  Then row tiles, so that those that
  // read the same positions run together; late tokens, which see most, first.
  // The first range of all tiles, then the others of those that are divided.
  const uint32_t items = a.tiles * a.kv_heads;
  uint32_t item = blockIdx.x, range = 0;
  if (item >= items) {
    const uint32_t divided = items - a.whole;
    range = 1 + (item - items) / divided;
    item = a.whole + (item - items) % divided;
  }
  const uint32_t hk = item % a.kv_heads, row_tile = a.tiles - 1 - item / a.kv_heads;
  const bool joined = a.ranges > 1 && item >= a.whole;
  PageWindow window;
  const Listed listed = find_listed<D>(a, row_tile, window);
  const uint32_t slot = listed.slot, first_row = listed.first_row, tokens = listed.tokens, length = listed.length;
  const uint32_t rows = tokens * a.group, tile_row = (row_tile - listed.first_tile) * kRows;
  // The tile's last row sees this many positions; what lies behind the sequence's end is not read.
  const uint32_t last_row = min(rows, tile_row + kRows) - 1;
  const uint32_t end = length + tokens, steps = (length + last_row / a.group + T) / T;
  // As few ranges as hold them, of equal length.
  const uint32_t used = joined ? (steps - 1) / listed.per + 1 : 1, per = (steps + used - 1) / used;
  const uint32_t from = range * per, to = min(from + per, steps);
  if (from >= steps) {
    const uint32_t row = tile_row + threadIdx.x;
    if (threadIdx.x < kRows && row < rows) {
      const uint32_t out_row = (first_row + row / a.group) * a.q_heads + hk * a.group + row % a.group;
      const std::size_t at = static_cast<std::size_t>(partial_row(a, item, threadIdx.x, out_row)) * a.ranges + range;
      *reinterpret_cast<float2*>(a.partial_ml + 2 * at) = float2{-INFINITY, 0.0F};
    }
    return;
  }

  // With few rows all waves take the same ones and divide the positions.
  const bool few = min(rows, tile_row + kRows) - tile_row <= 32;
  const uint32_t wave_row = few ? tile_row : tile_row + wave * 32, row = wave_row + n;
  const bool works = wave_row < rows;                        // the wave has a row
  const uint32_t least_visible = length + wave_row / a.group + 1;
  const uint32_t visible = row < rows ? length + row / a.group + 1 : 0;
  // Where the lane's row goes, [rows][q_heads], below 2^30.
  const uint32_t out_row = row < rows ? (first_row + row / a.group) * a.q_heads + hk * a.group + row % a.group : 0xffffffffu;
  h8 q[D / 16];
#pragma unroll
  for (unsigned st = 0; st < D / 16; ++st) {
    q[st] = h8{};
    if (row < rows) q[st] = *reinterpret_cast<const h8*>(a.query + static_cast<std::size_t>(out_row) * D + 16 * st + 8 * h);
    if constexpr (D == 256) asm volatile("" : "+a"(q[st]));
  }
  f16v o[D / 32];
  float m, l;
  if (few) {
    _Float16* lds[kWaves] = {k0, k1, v0, v1};
    // (Few rows are left to the join even if one range holds them: its waves divide the gate among more
    // lanes, eight decoding sequences a tenth less.)
    attend_few<D>(a, Range{slot, end, from, to, hk, least_visible}, q, visible, lds, limit, window, o, m, l);
    if (out_row != 0xffffffffu) write_row<D, D / 128>(a, out_row, partial_row(a, item, n, out_row), range, !joined, joined, o, wave, 4, m, l, wave == 0 && h == 0);
    return;
  }
  const std::size_t layer_row = (static_cast<std::size_t>(a.layer) * pg.page_count << pg.page_shift) * pg.row + hk * D;
  const __half* keys = pg.key + layer_row;
  const __half* values = pg.value + layer_row;
  const uint32_t in_page = (1u << pg.page_shift) - 1;
  f16v s[kSub], s_next[kSub];
  Peaks<Found*> peaks{-INFINITY, found + threadIdx.x, false};
  auto find_pages = [&](uint32_t x) __attribute__((always_inline)) {
    TilePages<D> p;
    p.missing = 0;
#pragma unroll
    for (unsigned e = 0; e < T / 16; ++e) {
      const uint32_t at = x * T + 16 * e;
      p.page[e] = at < end ? window.find(pg, slot, at >> pg.page_shift) : -1;
      if (p.page[e] < 0) p.missing |= 1u << e;
    }
    return p;
  };
  // Where the lane's piece of a load lies in memory, in bytes from the first of the load's rows: the rows of
  // load u of a wave are 16 or 8 u and its own, so the order of their pieces (by the row in sixteen for K,
  // in four for V) is that of u % 2.
  const uint32_t load_row = lane / (D / 8), row_bytes = 2 * pg.row;
  uint32_t key_part[2], value_part;
#pragma unroll
  for (unsigned e = 0; e < 2; ++e) {
    key_part[e] = load_row * row_bytes + 16 * key_slot(lane % (D / 8), kLoadRows * (wave + kWaves * e) + load_row);
  }
  value_part = load_row * row_bytes + 16 * value_slot4(lane % (D / 8), kLoadRows * wave + load_row);
  // Rows of a tile into LDS, through buffer descriptors of the parts' sixteen rows (after flat loads into LDS
  // the compiler lets every read of LDS wait for all reads before it).  Parts without a page load from page 0
  // of the pool (always there), and so do those past the end.
  auto load = [&](_Float16* to_lds, const __half* pool, bool key, uint32_t x, const TilePages<D>& p) __attribute__((always_inline)) {
#pragma unroll
    for (unsigned u = 0; u < kLoads; ++u) {
      const unsigned row0 = kLoadRows * (wave + kWaves * u), e = kLoadRows * kWaves * u / 16;
      const std::size_t base = ((static_cast<std::size_t>(max(p.page[e], 0)) << pg.page_shift) + ((x * T + 16 * e) & in_page)) * pg.row;
      const auto rows16 = __builtin_amdgcn_make_buffer_rsrc(const_cast<__half*>(pool + base), 0, static_cast<int>(15 * row_bytes + 2 * D), 0x20000);
      __builtin_amdgcn_raw_ptr_buffer_load_lds(rows16, (lds_void*)(to_lds + row0 * D), 16, static_cast<int>(key ? key_part[D == 128 ? 0 : u % 2] : value_part),
                                               static_cast<int>((row0 & 15u) * row_bytes), 0, 0);
    }
  };

  // Where the lane's part of the first score operand of 32 K rows, and of the first output tile of
  // 16 V rows, lies in bytes.  Operand s is at the place ^ 32 s, output tile d at the place ^ 64 d:
  // the slots of a row are permuted by exclusive or, and rows start at multiples of their size.
  const unsigned key_place = n * (2 * D) + 16 * key_slot(h, n), value_place = value_place_of<D>(lane);

  // What a page holds past a sequence's end, and what a missing one would, may be anything, and 0 * NaN
  // is NaN: the wave's own V rows of such positions become zeros.  A careful pass also takes out
  // infinities and NaNs, and marks the tile.
  auto repair = [&](_Float16* vs, uint32_t x, uint32_t missing, bool careful) __attribute__((always_inline)) {
    bool strange = false;
#pragma unroll 1
    for (unsigned u = 0; u < kLoads; ++u) {
      const unsigned row0 = kLoadRows * (wave + kWaves * u);
      u32x4* piece = reinterpret_cast<u32x4*>(vs + row0 * D) + lane;
      if (x * T + row0 + load_row >= end || (missing >> row0 / 16 & 1u) != 0) *piece = u32x4{0, 0, 0, 0};
      if (careful) strange |= take_strange(piece);
    }
    if (strange) atomicOr(&strange_tiles[x / 32 % 32], 1u << x % 32);
    wait_loads<63>();
  };
  // The rows that see an infinity or NaN among the values get it, whatever the weight: no weight is
  // exactly zero.
  auto add_strange = [&](uint32_t x) {
#pragma unroll 1
    for (unsigned p = 0; p < T; ++p) {
      const uint32_t position = x * T + p;
      const int32_t page = position < end ? table_page(pg, slot, position >> pg.page_shift) : -1;
      if (page < 0) continue;
      const __half* v = values + ((static_cast<std::size_t>(page) << pg.page_shift) + (position & in_page)) * pg.row;
#pragma unroll
      for (unsigned d = 0; d < D / 32; ++d) {
#pragma unroll
        for (unsigned r = 0; r < 16; ++r) {
          const float y = __half2float(v[32 * d + 8 * (r / 4) + 4 * h + r % 4]);
          if (!(fabsf(y) < INFINITY) && position < visible) o[d][r] += y;
        }
      }
    }
  };
  // Raw products of the rows with a tile of K rows.
  auto score = [&](const _Float16* ks, f16v (&out)[kSub]) __attribute__((always_inline)) {
    const char* kb = reinterpret_cast<const char*>(ks);
#pragma unroll
    for (unsigned u = 0; u < kSub; ++u) out[u] = f16v{};
#pragma unroll
    for (unsigned st = 0; st < D / 16; ++st) {
#pragma unroll
      for (unsigned u = 0; u < kSub; ++u) {
        const h8 k = *reinterpret_cast<const h8*>(kb + (key_place ^ 32 * st) + u * 64 * D);
        out[u] = __builtin_amdgcn_mfma_f32_32x32x16_f16(k, q[st], out[u], 0, 0, 0);
      }
    }
  };
  // The outputs and queries belong into the accumulation registers: left to itself the compiler counts them
  // among the others and reads every operand right before its product (4 prompts of 300 on 1500..6000:
  // 7 % more), or moves all of them there and back where maxima might move (12 % more).
  auto keep_outputs = [&]() __attribute__((always_inline)) {
    if constexpr (D == 256) {
#pragma unroll
      for (unsigned d = 0; d < D / 32; ++d) asm volatile("" : "+a"(o[d]));
    }
  };
  // Scores of a tile are ready: hides what a row does not see, and moves the maxima.
  auto positions = [&] { return max(min(visible, to * T), from * T + 1) - from * T; };
  auto settle = [&](f16v (&sc)[kSub], uint32_t x, uint32_t missing, auto careful) __attribute__((always_inline)) {
    if (x * T + T > least_visible || missing != 0) {
#pragma unroll
      for (unsigned u = 0; u < kSub; ++u) {
#pragma unroll
        for (unsigned r = 0; r < 16; ++r) {
          const unsigned p = 32 * u + 8 * (r / 4) + 4 * h + r % 4;
          if (x * T + p >= visible || (missing >> (2 * u + r / 8) & 1u) != 0) sc[u][r] = -INFINITY;
        }
      }
    }
    if constexpr (careful) {
      const float2 limits = taken_scores[threadIdx.x];
#pragma unroll
      for (unsigned e = 0; e < 16 * kSub; ++e) {
        const float score = sc[e / 16][e % 16] * a.scale;
        if (score <= limits.x || score > limits.y) sc[e / 16][e % 16] = -INFINITY;  // (not NaN)
      }
    }
    // (A NaN score makes the maximum NaN and the row's result with it, as it has to.)
    float best = sc[0][0];
#pragma unroll
    for (unsigned e = 1; e < 16 * kSub; ++e) best = __builtin_elementwise_maximum(best, sc[e / 16][e % 16]);
    const float top = max_over_halves(best) * a.scale;
    keep_outputs();
    if (peaks.moves(top)) {
      const float factor = peaks.move<!careful.value, 16 * kSub>([&](unsigned e) { return sc[e / 16][e % 16]; }, a.scale, top,
                                                 positions(), l);
      if (__any(factor != 1.0F)) {
        l *= factor;
#pragma unroll
        for (unsigned d = 0; d < D / 32; ++d) {
#pragma unroll
          for (unsigned r = 0; r < 16; ++r) o[d][r] *= factor;
        }
      }
      keep_outputs();
    }
    keep_outputs();
  };
  // The weights of the tile in s and the scores of the next one, then the values of this one.
  auto step = [&](const _Float16* next_ks, const _Float16* vs) __attribute__((always_inline)) {
    h8 p[kSteps];
    keep_outputs();
    score(next_ks, s_next);
    const float floor = peaks.m == -INFINITY ? 0.0F : peaks.m - kLift;
    float sum[4] = {l, 0.0F, 0.0F, 0.0F};
#pragma unroll
    for (unsigned j = 0; j < kSteps; ++j) {
#pragma unroll
      for (unsigned e = 0; e < 8; ++e) {
        const float w = __builtin_amdgcn_exp2f(fmaf(s[j / 2][8 * (j % 2) + e], a.scale, -floor));
        sum[e % 4] += w;
        p[j][e] = static_cast<_Float16>(w);
      }
    }
    l = (sum[0] + sum[1]) + (sum[2] + sum[3]);
    char* vb = const_cast<char*>(reinterpret_cast<const char*>(vs));
#pragma unroll
    for (unsigned j = 0; j < kSteps; ++j) {
#pragma unroll
      for (unsigned d = 0; d < D / 32; ++d) {
        s16x4 y[2];
#pragma unroll
        for (unsigned e = 0; e < 2; ++e) {
          y[e] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(vb + (value_place ^ 64 * d) + (16 * j + 8 * e) * 2 * D));
        }
        const h8 v = __builtin_bit_cast(h8, __builtin_shufflevector(y[0], y[1], 0, 1, 2, 3, 4, 5, 6, 7));
        o[d] = __builtin_amdgcn_mfma_f32_32x32x16_f16(v, p[j], o[d], 0, 0, 0);
      }
    }
    // The order of all this: operands are read eight ahead of the products, and exponentials go
    // between the products of the next tile's scores.
    constexpr unsigned kScores = kSub * D / 16, kAhead = 8;
    __builtin_amdgcn_sched_group_barrier(0x100, kAhead, 0);
#pragma unroll
    for (unsigned e = 0; e < kScores; ++e) {
      __builtin_amdgcn_sched_group_barrier(0x8, 1, 0);
      __builtin_amdgcn_sched_group_barrier(0x400, 16 * kSub / kScores, 0);
      __builtin_amdgcn_sched_group_barrier(0x2, 3 * 16 * kSub / kScores, 0);
      __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
    }
#pragma unroll
    for (unsigned e = 0; e < kSteps * D / 32; ++e) {
      __builtin_amdgcn_sched_group_barrier(0x8, 1, 0);
      __builtin_amdgcn_sched_group_barrier(0x100, 2, 0);
    }
#pragma unroll
    for (unsigned u = 0; u < kSub; ++u) {
      s[u] = s_next[u];
      if constexpr (D == 256) asm volatile("" : "+v"(s[u]));  // for the vector unit
    }
  };

  // Tile x's V rows and tile x + 1's K rows are read while x + 1's V rows and x + 2's K rows are on their way,
  // each into the place that was read last before the barrier.
  auto clear = [&] {
    peaks.clear();
    l = 0.0F;
#pragma unroll
    for (unsigned d = 0; d < D / 32; ++d) o[d] = f16v{};
  };
  bool odd = false;  // infinities and NaNs among the values are looked for
  auto pass = [&](auto careful, uint32_t from) __attribute__((always_inline)) {
    TilePages<D> now = find_pages(from), next = now;
    if (careful && threadIdx.x < 32) strange_tiles[threadIdx.x] = 0;
    __syncthreads();  // the tile before this one is done with
    load(k0, keys, true, from, now);
    wait_loads<0>();
    __syncthreads();
    load(v0, values, false, from, now);
    if (from + 1 < to) {
      next = find_pages(from + 1);
      load(k1, keys, true, from + 1, next);
    }
    if (works) {
      score(k0, s);
      settle(s, from, now.missing, careful);
    }
    auto turn = [&](uint32_t x, _Float16* k_free, const _Float16* k_next, _Float16* v_now, _Float16* v_free) __attribute__((always_inline)) {
      wait_loads<0>();
      if ((careful && odd) || now.missing != 0 || (x + 1) * T > end) repair(v_now, x, now.missing, careful && odd);
      __syncthreads();
      now = next;
      if (x + 1 < to) load(v_free, values, false, x + 1, next);
      if (x + 2 < to) {
        next = find_pages(x + 2);
        load(k_free, keys, true, x + 2, next);
      }
      if (works) {
        step(k_next, v_now);
        if (x + 1 < to) settle(s, x + 1, now.missing, careful);
      }
    };
#pragma unroll 1
    for (uint32_t x = from; x < to; x += 2) {
      turn(x, k0, k1, v0, v1);
      if (x + 1 < to) turn(x + 1, k1, k0, v1, v0);
    }
  };
  // Whether an output is an infinity or NaN: finite values at weights below 2^15 make none.
  auto is_strange = [&]() __attribute__((always_inline)) {
    bool strange = false;
#pragma unroll
    for (unsigned d = 0; d < D / 32; ++d) {
#pragma unroll
      for (unsigned r = 0; r < 16; ++r) strange |= !(fabsf(o[d][r]) < INFINITY);
    }
    return strange;
  };

  clear();
  pass(std::false_type{}, from);
  bool strange = is_strange();
  // Careful passes follow in the rare case that an output of the first is an infinity or NaN, or that a row's small weights
  // may matter.
  const uint64_t taken = peaks.open(l, positions());
  const uint32_t mine = (__any(strange) ? 1u : 0u) | (taken != 0 ? 2u : 0u);
  if (lane == 0) again[wave] = mine;
  __syncthreads();
  uint32_t any = 0;
  for (unsigned w = 0; w < kWaves; ++w) any |= again[w];
  any = __builtin_amdgcn_readfirstlane(any);
  const bool careful = any != 0;
  if (__builtin_expect(careful, 0)) {
    // Everything but the peaks of such rows, then those peaks.
    odd = (any & 1u) != 0;
    limit.below_peaks(peaks.m, taken);
    clear();
#pragma unroll 1
    for (bool apart = any >= 2;; apart = false) {
      pass(std::true_type{}, fresh_number(from));  // (what follows from it is not kept from one pass for the next)
      if (!apart) break;
      limit.peaks();  // added to what is there
    }
    for (uint32_t x = from; x < to; ++x) {
      if ((__builtin_amdgcn_readfirstlane(strange_tiles[x / 32 % 32]) >> x % 32 & 1u) != 0) add_strange(x);
    }
    strange = is_strange();
  }
  l = sum_over_halves(l);
  m = peaks.m;
  // Only NaN scores, and strange values at scores of -infinity, make a NaN row rather than an empty one.
  if ((m == -INFINITY && (l != l || (careful && strange))) || m != m) m = 0.0F;
  if (out_row != 0xffffffffu) write_row<D, D / 32>(a, out_row, partial_row(a, item, wave * 32 + n, out_row), range, used == 1, joined, o, 0, 1, m, l, h == 0);
}

constexpr uint32_t kJoinRows = 4096;

// Joins the ranges of a row and applies the gate: a wave per row and query head, D / 64 dims a lane.
// Lane r holds range r's maximum and sum; the outputs of the first two ranges are loaded beside them.  `rows` partial rows;
// ByTile: those of the divided tiles.
template <unsigned D, bool ByTile>
__global__ __launch_bounds__(256) void chunk_join_kernel(ChunkAttnArgs a, uint32_t rows) {
  constexpr unsigned J = D / 64;
  using vec = float __attribute__((ext_vector_type(J)));
  using hvec = _Float16 __attribute__((ext_vector_type(J)));
  const unsigned lane = threadIdx.x & 63u;
  const uint32_t part_row = __builtin_amdgcn_readfirstlane(blockIdx.x * 4u + (threadIdx.x >> 6));
  if (part_row >= rows) return;
  uint32_t row = part_row;
  if constexpr (ByTile) {
    const uint32_t item = a.whole + part_row / a.tile_rows, row_of_tile = part_row % a.tile_rows;
    const uint32_t row_tile = a.tiles - 1 - item / a.kv_heads, hk = item % a.kv_heads;
    uint32_t of_sequence = 0xffffffffu, first_row = 0;  // a lane a sequence, one of which has the tile
    for (uint32_t from = 0; from < a.list.count; from += 64) {
      const uint32_t i = min(from + lane, a.list.count - 1), heads = (a.list.first[i + 1] - a.list.first[i]) * a.group;
      const uint32_t here = (row_tile - a.first_tile[i]) * kRows + row_of_tile;
      const uint64_t found = __ballot(from + lane < a.list.count && row_tile >= a.first_tile[i] && here < heads);
      if (found == 0) continue;
      const int at = __ffsll(static_cast<unsigned long long>(found)) - 1;
      of_sequence = static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(here), at));
      first_row = static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(a.list.first[i]), at));
    }
    if (of_sequence == 0xffffffffu) return;  // behind the rows of a sequence's last tile
    row = (first_row + of_sequence / a.group) * a.q_heads + hk * a.group + of_sequence % a.group;
  }
  const std::size_t base = static_cast<std::size_t>(part_row) * a.ranges;
  const float* parts = a.partial_o + base * D + J * lane;
  // Many rows: complete ones are not worth the loads that cover the look.
  if ((ByTile || rows > kJoinRows) && __builtin_amdgcn_readfirstlane(__float_as_int(a.partial_ml[2 * base + 1])) == __float_as_int(kWritten)) return;
  vec g = {};
  if (a.gate != nullptr) g = *reinterpret_cast<const vec*>(a.gate + static_cast<std::size_t>(row) * 2 * D + D + J * lane);
  const vec first[2] = {*reinterpret_cast<const vec*>(parts), *reinterpret_cast<const vec*>(parts + D)};
  float best = -INFINITY, sum = 0.0F;
  vec y = {};
  for (uint32_t from = 0; from < a.ranges; from += 64) {
    const uint32_t here = min(64u, a.ranges - from);
    float2 x = {-INFINITY, 0.0F};
    if (lane < here) x = *reinterpret_cast<const float2*>(a.partial_ml + 2 * (base + from + lane));
    if (from == 0 && lane_value(x.y, 0) == kWritten) return;
    const float next = fmaxf(best, wave_max(x.x));
    if (next == -INFINITY) continue;
    const float w = x.x == -INFINITY ? 0.0F : rescale_factor(x.x, next);
    if (best != -INFINITY) {
      const float keep = rescale_factor(best, next);
      sum *= keep;
      y *= keep;
    }
    best = next;
    sum += wave_sum(w == 0.0F ? 0.0F : x.y * w);
    for (uint64_t left = __ballot(w != 0.0F); left != 0;) {
      constexpr unsigned kBatch = 4;
      vec v[kBatch];
      float wv[kBatch];
#pragma unroll
      for (unsigned e = 0; e < kBatch; ++e) {
        const int r = left != 0 ? __ffsll(static_cast<unsigned long long>(left)) - 1 : -1;
        wv[e] = r < 0 ? 0.0F : lane_value(w, r);
        left &= left - 1;
        if (r < 0) v[e] = vec{};
        else if (from + r < 2) v[e] = r == 0 ? first[0] : first[1];
        else v[e] = *reinterpret_cast<const vec*>(parts + static_cast<std::size_t>(from + r) * D);
      }
#pragma unroll
      for (unsigned e = 0; e < kBatch; ++e) y += v[e] * wv[e];
    }
  }
  const bool empty = best == -INFINITY;
  hvec out;
#pragma unroll
  for (unsigned j = 0; j < J; ++j) {
    float z = empty ? 0.0F : y[j] / sum;
    if (a.gate != nullptr) z *= 1.0F / (1.0F + expf(-g[j]));
    out[j] = static_cast<_Float16>(z);
  }
  *reinterpret_cast<hvec*>(a.output + static_cast<std::size_t>(row) * D + J * lane) = out;
  if (a.log_sums != nullptr && lane == 0) a.log_sums[row] = empty ? -INFINITY : (best - kLift) * kLn2 + logf(sum);
}

// ---- the weight that each position receives ---------------------------------------------

// A listed sequence, all that one load of the arguments has to bring.
struct WeightItem {
  uint32_t slot, first_row, tokens;
};
struct WeightArgs {
  KvPages pages;
  KvWeights weights;
  const __half* query;
  const float* log_sums;
  float* partial;  // [sequences with many rows][kv_heads * parts][capacity]
  uint32_t layer, q_heads, kv_heads, group, parts;
  uint32_t columns;  // workgroups along the positions
  float scale;
  WeightItem item[kMaxChunks];  // of the launch's sequences: those with more than kFewRows rows, or the others
};

// Sums of N registers over the 32 lanes of a half: at each exchange a lane keeps the registers whose
// number has its own bit, so that register r of lane n ends as the whole sum of number n % N.
template <unsigned N, unsigned Distance = 1>
__device__ __forceinline__ float sum_lanes(const float (&sum)[N]) {
  const bool odd = (threadIdx.x & Distance) != 0;
  float half[N > 1 ? N / 2 : 1];
  if constexpr (N == 1) {
    half[0] = sum[0] + __shfl_xor(sum[0], Distance);  // fewer registers than lanes
  } else {
#pragma unroll
    for (unsigned r = 0; r < N / 2; ++r) half[r] = (odd ? sum[2 * r + 1] : sum[2 * r]) + __shfl_xor(odd ? sum[2 * r] : sum[2 * r + 1], Distance);
  }
  if constexpr (Distance == 16) return half[0];
  else return sum_lanes<(N > 1 ? N / 2 : 1), 2 * Distance>(half);
}

// The K row of a position on its page (-1: none), or one that is always there.
__device__ __forceinline__ const __half* key_row(const WeightArgs& a, int32_t page, uint32_t position) {
  const KvPages& pg = a.pages;
  const std::size_t row = (static_cast<std::size_t>(max(page, 0)) << pg.page_shift) + (page < 0 ? 0 : position & ((1u << pg.page_shift) - 1));
  return pg.key + ((static_cast<std::size_t>(a.layer) * pg.page_count << pg.page_shift) + row) * pg.row;
}

static_assert(sizeof(WeightArgs) <= 4096);  // arguments of a launch

constexpr uint32_t kFewRows = 32;  // of a sequence and KV head

// Sequences of at most 32 rows, as a decoding one has: a workgroup takes 32 positions and all KV
// heads, a wave every fourth one, and adds the sum over all of them.  A position's row holds the heads side by side, so
// a workgroup reads whole rows, and one launch does (sixteen on up to 4090, 24 x 4 x 256: 15.7 us, 4.0 TB/s; with
// a sum for each KV head and a second launch 24.6).
template <unsigned D>
__global__ __launch_bounds__(256) void few_weight_kernel(WeightArgs a) {
  __shared__ float parts[4][32];
  const unsigned lane = threadIdx.x & 63u, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const unsigned n = lane & 31u, h = lane >> 5;
  const KvPages& pg = a.pages;
  const WeightItem item = a.item[blockIdx.y];
  const uint32_t slot = item.slot, first_row = item.first_row, tokens = item.tokens, rows = tokens * a.group;
  const uint32_t capacity = pg.stride << pg.page_shift, t = min(n, rows - 1) / a.group;
  const std::size_t out_row = (static_cast<std::size_t>(first_row) + t) * a.q_heads + (min(n, rows - 1) - t * a.group);
  float* weights = a.weights.weight + static_cast<std::size_t>(slot) * capacity;
  const uint32_t length = committed(pg, slot), end = min(length + tokens, capacity);
  // (Pages and weights are not asked for before the length is there: half of the workgroups have no
  // positions, 7 % more.)
  for (uint32_t at = blockIdx.x * 32; at < end; at += gridDim.x * 32) {
    const int32_t page = table_page(pg, slot, (at + n) >> pg.page_shift);
    const bool there = at + n < end && page >= 0;
    const __half* keys = key_row(a, there ? page : -1, at + n) + 8 * h;
    float sum[16] = {};
    for (uint32_t hk = wave; hk < a.kv_heads; hk += 4) {
      const std::size_t row = out_row + hk * a.group;
      h8 k[D / 16], q[D / 16];
#pragma unroll
      for (unsigned s = 0; s < D / 16; ++s) k[s] = *reinterpret_cast<const h8*>(keys + hk * D + 16 * s);
#pragma unroll
      for (unsigned s = 0; s < D / 16; ++s) q[s] = *reinterpret_cast<const h8*>(a.query + row * D + 16 * s + 8 * h);
      const float level = a.log_sums[row] * kLog2E;
      const uint32_t visible = n < rows && level > -INFINITY ? length + t + 1 : 0;  // not of a row that sees nothing, or a NaN
      f16v s = f16v{};
#pragma unroll
      for (unsigned st = 0; st < D / 16; ++st) s = __builtin_amdgcn_mfma_f32_32x32x16_f16(k[st], q[st], s, 0, 0, 0);
#pragma unroll
      for (unsigned r = 0; r < 16; ++r) {
        const float w = __builtin_amdgcn_exp2f(fmaf(s[r], a.scale, -level));
        sum[r] += at + 8 * (r / 4) + 4 * h + r % 4 < visible ? w : 0.0F;
      }
    }
    const float mine = sum_lanes(sum);
    // Lane n has the sum of register n % 16: position 8 (r / 4) + 4 h + r % 4.
    if (n < 16) parts[wave][8 * (n / 4) + 4 * h + n % 4] = mine;
    __syncthreads();
    if (threadIdx.x < 32 && there) {
      float total = 0.0F;
#pragma unroll
      for (unsigned v = 0; v < 4; ++v) total += parts[v][threadIdx.x];
      weights[at + threadIdx.x] += total;
    }
    __syncthreads();
  }
}

constexpr unsigned kWeightPositions = 256;  // of a workgroup: 64 a wave
constexpr unsigned kWeightRows = 32;        // rows of a step
// Workgroups a CU holds.
template <unsigned D>
constexpr unsigned kWeightResident = D == 128 ? 2 : 1;
constexpr unsigned kWeightRing = 4;         // steps in LDS: one is read, two are on their way

// Rows of a step on their way to LDS, and the log sums of its lane's row: each lane walks from a row to
// the one 32 further on without dividing.
struct RowWalk {
  uint32_t head;    // the row's query head of the group
  uint32_t offset;  // from the step's first token, in units of the caller
  __device__ __forceinline__ void start(uint32_t row, uint32_t token, uint32_t group, uint32_t token_step, uint32_t head_step) {
    const uint32_t t = row / group;
    head = row - t * group;
    offset = (t - token) * token_step + head * head_step;
  }
  // `by` = 32 % group; `wrapped`: the step's first token moved on by 32 / group + 1 tokens, not 32 / group.
  __device__ __forceinline__ void step(uint32_t by, bool wrapped, uint32_t group, uint32_t token_step, uint32_t head_step) {
    head += by;
    offset += by * head_step - (wrapped ? token_step : 0);
    const bool over = head >= group;
    head -= over ? group : 0;
    offset += over ? token_step - group * head_step : 0;
  }
};

// A wave holds 64 positions of K as the A operand.  The rows of a KV head pass through LDS, 32 at a time,
// three steps ahead, and serve all waves; the exponentials of a step, each added to the lane's sum of
// its position, go between the next step's products.  64 positions a wave, not 32: a step's operands are read
// from LDS by every wave, which at 32 takes as long as its products.  2048 tokens on 8000: 40 x 8 x 128 225 us, 842
// TFLOP/s, the matrix units busy 47 % of the time, the vector unit 36 %; 24 x 4 x 256 322 us, 706 TFLOP/s.
template <unsigned D>
__global__ __launch_bounds__(256, kWeightResident<D>) void weight_kernel(WeightArgs a) {
  constexpr unsigned P = kWeightPositions / 4 / 32;
  constexpr unsigned kLoadRows = 512 / D, kLoads = kWeightRows / kLoadRows / 4;
  // (Arrays of their own, so that the compiler can tell one step's reads from another's loads.)
  __shared__ __align__(1024) _Float16 step0[kWeightRows * D], step1[kWeightRows * D], step2[kWeightRows * D], step3[kWeightRows * D];
  _Float16* const ring[kWeightRing] = {step0, step1, step2, step3};
  const unsigned lane = threadIdx.x & 63u, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const unsigned n = lane & 31u, h = lane >> 5;
  const KvPages& pg = a.pages;
  const uint32_t hk = blockIdx.x % a.kv_heads, part = blockIdx.x / a.kv_heads % a.parts;
  const uint32_t column = blockIdx.x / a.kv_heads / a.parts;
  const WeightItem item = a.item[blockIdx.y];
  const uint32_t slot = item.slot, first_row = item.first_row, tokens = item.tokens, rows = tokens * a.group;
  const uint32_t all = (rows + kWeightRows - 1) / kWeightRows;
  const uint32_t length = committed(pg, slot), end = min(length + tokens, pg.stride << pg.page_shift);
  const uint32_t per = (all + a.parts - 1) / a.parts, to = min(part * per + per, all);
  const uint32_t token_bytes = a.q_heads * D * 2;
  const std::size_t plane = (static_cast<std::size_t>(blockIdx.y) * a.kv_heads + hk) * a.parts + part;
  float* sums = a.partial + plane * (static_cast<std::size_t>(pg.stride) << pg.page_shift);
  for (uint32_t at = column * kWeightPositions; at < end; at += a.columns * kWeightPositions) {
    const uint32_t mine = at + 32 * P * wave;
    // The step of token x's first row, of all those of a part at most.
    auto step_of = [&](uint32_t x) { return static_cast<uint32_t>(min(static_cast<uint64_t>(x) * a.group / kWeightRows, static_cast<uint64_t>(to))); };
    // Rows of tokens before length + t = at see nothing of these positions, those from seen on all of them.
    const uint32_t from = max(part * per, at > length ? step_of(at - length) : 0u);
    const uint32_t sees = min(at + kWeightPositions, end), seen = sees > length + 1 ? step_of(sees - length - 1 + (kWeightRows - 1) / a.group + 1) : 0;
    float sum[16 * P] = {};
    h8 k[P][D / 16];
    if (from < to) {
#pragma unroll
      for (unsigned p = 0; p < P; ++p) {
        const uint32_t position = mine + 32 * p + n;
        const int32_t page = position < end ? table_page(pg, slot, position >> pg.page_shift) : -1;
        const __half* row = key_row(a, page, position) + hk * D + 8 * h;
#pragma unroll
        for (unsigned st = 0; st < D / 16; ++st) k[p][st] = *reinterpret_cast<const h8*>(row + 16 * st);
      }
    }
    if constexpr (D == 256) {
      // (K in accumulation registers, which leaves the others to the scores and sums.)
#pragma unroll
      for (unsigned p = 0; p < P; ++p) {
#pragma unroll
        for (unsigned st = 0; st < D / 16; ++st) asm volatile("" : "+a"(k[p][st]));
      }
    }
    // Steps [first, last).  Without `masked` every row of them sees every position; false: a row among them
    // has a log sum that is not a number to subtract.
    auto pass = [&](auto masked, uint32_t first, uint32_t last) __attribute__((always_inline)) {
      if (first >= last) return true;
      // The step whose rows are loaded next, its first row's token and head, and the lanes' rows.
      uint32_t ahead = first, token = first * kWeightRows / a.group, head = first * kWeightRows - token * a.group;
      RowWalk walk[kLoads], sum_walk;
#pragma unroll
      for (unsigned u = 0; u < kLoads; ++u) {
        walk[u].start(first * kWeightRows + (wave + 4 * u) * kLoadRows + lane / (D / 8), token, a.group, token_bytes, 2 * D);
      }
      sum_walk.start(first * kWeightRows + n, token, a.group, a.q_heads * 4, 4);
      // Where the lanes' parts of the step are (rows past the last one load that one).
      uint32_t there, part_at[kLoads], level_at;  // rows from the step's first one on; bytes
      const uint32_t load_row = wave * kLoadRows + lane / (D / 8);
      auto place_part = [&](unsigned u) __attribute__((always_inline)) {
        part_at[u] = min(walk[u].offset, (there - 1) * (2 * D)) + 16 * key_slot(lane % (D / 8), load_row + 4 * u * kLoadRows);
      };
      auto place_level = [&] { level_at = min(sum_walk.offset, there * 4 - 4); };
      auto count = [&] { there = min(kWeightRows, tokens - 1 - token) * a.q_heads + a.group; };
      auto load = [&](_Float16* step, float& level) __attribute__((always_inline)) {
        const std::size_t row = (static_cast<std::size_t>(first_row) + token) * a.q_heads + hk * a.group;
        const auto queries = __builtin_amdgcn_make_buffer_rsrc(const_cast<__half*>(a.query + row * D), 0, static_cast<int>(there * (2 * D)), 0x20000);
        const auto levels = __builtin_amdgcn_make_buffer_rsrc(const_cast<float*>(a.log_sums + row), 0, static_cast<int>(there * 4), 0x20000);
        level = __uint_as_float(__builtin_amdgcn_raw_buffer_load_b32(levels, static_cast<int>(level_at), 0, 0));
#pragma unroll
        for (unsigned u = 0; u < kLoads; ++u) {
          __builtin_amdgcn_raw_ptr_buffer_load_lds(queries, (lds_void*)(step + (wave + 4 * u) * kLoadRows * D), 16, static_cast<int>(part_at[u]), 0, 0, 0);
        }
      };
      // On to the next step, in kLoads + 2 pieces of work.
      uint32_t by = 0;
      bool wrapped = false;
      auto advance = [&](unsigned piece) __attribute__((always_inline)) {
        if (piece == 0) {
          const bool more = ++ahead < last;
          by = more ? kWeightRows % a.group : 0;
          head += by;
          wrapped = head >= a.group;
          head -= wrapped ? a.group : 0;
          token += (more ? kWeightRows / a.group : 0) + (wrapped ? 1 : 0);
          count();
        } else if (piece <= kLoads) {
          walk[piece - 1].step(by, wrapped, a.group, token_bytes, 2 * D);
          place_part(piece - 1);
        } else {
          sum_walk.step(by, wrapped, a.group, a.q_heads * 4, 4);
          place_level();
        }
      };
      count();
#pragma unroll
      for (unsigned u = 0; u < kLoads; ++u) place_part(u);
      place_level();
      f16v s[2][P] = {};
      float level[kWeightRing] = {};
      bool plain = true;
      // A piece of the step's rows: the B operand of product st.
      auto read = [&](unsigned d, unsigned place, unsigned st) __attribute__((always_inline)) {
        return *reinterpret_cast<const h8*>(reinterpret_cast<const char*>(ring[d]) + (place ^ 32 * st));
      };
      // What rows n of s[d % 2] give to positions 4 h + [first, last) in the accumulators' order.
      auto add = [&](unsigned d, float level, unsigned first, unsigned last) __attribute__((always_inline)) {
#pragma unroll
        for (unsigned e = first; e < last; ++e) sum[e] += __builtin_amdgcn_exp2f(fmaf(s[d % 2][e / 16][e % 16], a.scale, -level));
      };
      auto add_masked = [&](uint32_t x, unsigned d, float level) __attribute__((always_inline)) {
        const uint32_t row = x * kWeightRows + n;
        const uint32_t base = mine + 4 * h, end_row = length + row / a.group + 1;
        const uint32_t visible = row < rows && level > -INFINITY && end_row > base ? end_row - base : 0;  // not of a row that sees nothing, or a NaN
#pragma unroll
        for (unsigned p = 0; p < P; ++p) {
#pragma unroll
          for (unsigned r = 0; r < 16; ++r) {
            const float w = __builtin_amdgcn_exp2f(fmaf(s[d % 2][p][r], a.scale, -level));
            sum[16 * p + r] += 32 * p + 8 * (r / 4) + r % 4 < visible ? w : 0.0F;
          }
        }
      };
#pragma unroll
      for (unsigned d = 0; d + 1 < kWeightRing; ++d) {
        load(ring[d], level[d]);
        asm volatile("" ::: "memory");  // in this order: the waits below count them
#pragma unroll
        for (unsigned e = 0; e < kLoads + 2; ++e) advance(e);
      }
      auto turn = [&](uint32_t x, unsigned d) __attribute__((always_inline)) {
        // This step has arrived when only the later ones are on their way.
        wait_loads<2 * (kLoads + 1)>();
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
        const unsigned before = (d + kWeightRing - 1) % kWeightRing;
        // Nothing yet before the first step: exponentials of zeros less infinity.
        const float old = x == first ? INFINITY : level[before] * kLog2E;
        if constexpr (!masked.value) plain &= x == first || fabsf(old) < INFINITY;
        // (Computed anew for each step: 32 addresses of 4 steps would take the registers of as many operands.)
        unsigned place = n * (2 * D) + 16 * key_slot(h, n);
        asm volatile("" : "+v"(place));
        constexpr unsigned kSteps = D / 16, kAhead = 3, kEach = 16 * P / kSteps;
        h8 q[kAhead + 1];
#pragma unroll
        for (unsigned st = 0; st < kAhead; ++st) q[st] = read(d, place, st);
        __builtin_amdgcn_sched_barrier(0);
        // Every wave has read the step before this one: its place takes the next loads.
        load(ring[before], level[before]);
        // Products, reads three ahead of them and the last step's exponentials, in this order.
#pragma unroll
        for (unsigned st = 0; st < kSteps; ++st) {
          __builtin_amdgcn_sched_barrier(0);
          if (st + kAhead < kSteps) q[(st + kAhead) % (kAhead + 1)] = read(d, place, st + kAhead);
#pragma unroll
          for (unsigned p = 0; p < P; ++p) s[d % 2][p] = __builtin_amdgcn_mfma_f32_32x32x16_f16(k[p][st], q[st % (kAhead + 1)], st == 0 ? f16v{} : s[d % 2][p], 0, 0, 0);
          if constexpr (!masked.value) add(d + 1, old, kEach * st, kEach * st + kEach);
          if (st < kLoads + 2) advance(st);
        }
        __builtin_amdgcn_sched_barrier(0);
        if constexpr (masked.value) add_masked(x, d, level[d] * kLog2E);
        if constexpr (D == 256) {
          // (In the registers that the vector unit reads.)
#pragma unroll
          for (unsigned p = 0; p < P; ++p) asm volatile("" : "+v"(s[d % 2][p]));
        }
        // (In this turn: left to itself the compiler moves all turns' exponentials behind the last one's products.)
#pragma unroll
        for (unsigned r = 0; r < 16 * P; ++r) asm volatile("" : "+v"(sum[r]));
      };
      uint32_t x = first;
#pragma unroll 1
      for (; x + kWeightRing <= last; x += kWeightRing) {
#pragma unroll
        for (unsigned d = 0; d < kWeightRing; ++d) turn(x + d, d);
      }
#pragma unroll
      for (unsigned d = 0; d < kWeightRing; ++d) {
        if (x + d < last) {
          turn(x + d, d);
        } else if (!masked.value && x + d == last) {
          const float old = level[(d + kWeightRing - 1) % kWeightRing] * kLog2E;
          plain &= fabsf(old) < INFINITY;
          add(d + 1, old, 0, 16 * P);
        }
      }
      // No load writes into LDS when the next rows, or another workgroup's, come there.
      wait_loads<0>();
      __syncthreads();
      return plain;
    };
    // The steps without a mask, and those before and behind them; all with masks where that did not do.
    uint32_t low = max(from, min(seen, to)), high = max(low, min(to, rows / kWeightRows));
    if (__syncthreads_or(!pass(std::false_type{}, low, high))) {
#pragma unroll
      for (unsigned r = 0; r < 16 * P; ++r) sum[r] = 0.0F;
      low = high = to;
    }
#pragma unroll 1
    for (unsigned e = 0; e < 2; ++e) pass(std::true_type{}, e == 0 ? from : high, e == 0 ? low : to);
    // Lane n has the sum of register n of the 32: position 32 (r / 16) + 8 (r / 4 % 4) + 4 h + r % 4.
    const float total = sum_lanes(sum);
    const uint32_t position = mine + 32 * (n / 16) + 8 * (n / 4 % 4) + 4 * h + n % 4;
    if (position < end) sums[position] = total;
  }
}

// Adds the planes of the KV heads and row parts, in their order, to what the positions have: a lane a
// position, a wave a quarter of the planes.
__global__ __launch_bounds__(256) void weight_join_kernel(WeightArgs a) {
  __shared__ float parts[4][64];
  const KvPages& pg = a.pages;
  const unsigned lane = threadIdx.x & 63u, wave = threadIdx.x >> 6;
  const uint32_t slot = a.item[blockIdx.y].slot, tokens = a.item[blockIdx.y].tokens;
  const uint32_t capacity = pg.stride << pg.page_shift, end = min(committed(pg, slot) + tokens, capacity);
  const uint32_t planes = a.kv_heads * a.parts, quarter = (planes + 3) / 4;
  for (uint32_t at = blockIdx.x * 64; at < end; at += gridDim.x * 64) {
    const uint32_t p = at + lane;
    const float* source = a.partial + static_cast<std::size_t>(blockIdx.y) * planes * capacity + min(p, end - 1);
    float sum = 0.0F;
#pragma unroll 8
    for (uint32_t x = wave * quarter; x < min(wave * quarter + quarter, planes); ++x) sum += source[static_cast<std::size_t>(x) * capacity];
    parts[wave][lane] = sum;
    __syncthreads();
    if (wave == 0 && p < end && table_page(pg, slot, p >> pg.page_shift) >= 0) {
      a.weights.weight[static_cast<std::size_t>(slot) * capacity + p] += parts[0][lane] + parts[1][lane] + parts[2][lane] + parts[3][lane];
    }
    __syncthreads();
  }
}

// ---- host side ---------------------------------------------------------------------------

int32_t read_heads(const gfxinfer_kv_pages* pages, uint32_t q_heads) {
  if (q_heads == 0 || q_heads > 1024 || q_heads % pages->kv_heads != 0) {
    return fail(GFXI_INVALID_ARGUMENT, "query heads are 1..1024 and a multiple of the cache's KV heads");
  }
  return GFXI_OK;
}

struct ChunkShape {
  uint32_t tiles, ranges, whole, tile_rows;
};

// Row tiles, and the ranges that the longest sequence's positions are divided into: one and a half workgroups
// for each place (two at head size 256), as far as full tables hold so many.  Where there are tiles for all places, those that
// make whole rounds are not divided, and the rest only as far as it fills one more round: parts cost a trip through memory
// (2048 tokens on 30000 in 640 tiles: all of them in two ranges take 3 % longer; 3000 on 8000 at head size 256: 919 us, undivided 20 %
// longer).
// Not so if sequences decode, each tile of as many positions as its sequence has and few rows' parts: 64 on 200 .. 4090 128 us,
// undivided 139, of 400 .. 600 beside one of 30000 225 and 387, without that one 37 and 31.
constexpr uint64_t kMostOfRest = 4;
ChunkShape chunk_shape(const KvPages& p, const ChunkList& list, uint32_t q_heads, uint32_t kv_heads, uint32_t head_size,
                       uint32_t* first_tile) {
  ChunkShape s{};
  const uint32_t group = q_heads / kv_heads;
  // Tiles run from the last to the first: sequences with few new tokens get the last ones.  (31 that decode and a
  // chunk behind them in the list: in the list's order, with the chunk's tiles first, 6 % longer.)
  std::array<uint16_t, kMaxChunks> order;
  std::iota(order.begin(), order.begin() + list.count, uint16_t{0});
  auto tokens = [&](uint32_t i) { return list.first[i + 1] - list.first[i]; };
  std::stable_sort(order.begin(), order.begin() + list.count, [&](uint32_t a, uint32_t b) { return tokens(a) > tokens(b); });
  for (uint32_t e = 0; e < list.count; ++e) {
    first_tile[order[e]] = s.tiles;
    s.tiles += (tokens(order[e]) * group + kRows - 1) / kRows;
  }
  s.tile_rows = std::min(kRows, tokens(order[0]) * group);
  const uint64_t capacity = static_cast<uint64_t>(p.stride) << p.page_shift, items = static_cast<uint64_t>(s.tiles) * kv_heads;
  const uint64_t places = (head_size == 128 ? kResident<128> : kResident<256>) * kComputeUnits;
  const uint64_t most = std::max<uint64_t>(1, capacity / ((head_size == 128 ? kTile<128> : kTile<256>) * kLeastSteps));
  if (items < places || s.tile_rows <= 32) {
    s.ranges = static_cast<uint32_t>(std::clamp<uint64_t>((places * (head_size == 128 ? 3 : 4) / 2 + items - 1) / items, 1, most));
  } else {
    s.whole = static_cast<uint32_t>(items / places * places);
    const uint64_t rest = items - s.whole;
    s.ranges = rest == 0 ? 1 : static_cast<uint32_t>(std::min({places / rest, most, kMostOfRest}));
  }
  return s;
}

// Rows with parts, see partial_row: at most kRows for each place.  (Below 2^18, so a launch holds a wave for each, and below
// 2^24 workgroups for the items, of which there are at most 2^30 / kRows and one for each sequence and KV head.)
uint32_t partial_rows(const ChunkShape& s, const ChunkList& list, uint32_t q_heads, uint32_t kv_heads) {
  if (s.ranges == 1) return 0;
  return s.whole == 0 ? list.first[kMaxChunks] * q_heads : (s.tiles * kv_heads - s.whole) * s.tile_rows;
}

std::size_t chunk_bytes(const ChunkShape& s, const ChunkList& list, uint32_t q_heads, uint32_t kv_heads, uint32_t head_size) {
  return static_cast<std::size_t>(partial_rows(s, list, q_heads, kv_heads)) * s.ranges * (head_size + 2) * sizeof(float);
}

// How the rows of the long chunks are divided: workgroups along the positions, and parts of the rows.
struct WeightShape {
  uint32_t columns, parts;
  uint32_t few, many;  // sequences of 1 .. kFewRows rows, of more
};

WeightShape weight_shape(const KvPages& p, const ChunkList& list, uint32_t q_heads, uint32_t kv_heads) {
  WeightShape s{};
  const uint64_t capacity = static_cast<uint64_t>(p.stride) << p.page_shift;
  s.columns = static_cast<uint32_t>(std::min<uint64_t>((capacity + kWeightPositions - 1) / kWeightPositions, 1024));
  uint32_t most = 0;
  for (uint32_t i = 0; i < list.count; ++i) {
    const uint32_t tokens = list.first[i + 1] - list.first[i];
    most = std::max(most, tokens);
    const bool many = static_cast<uint64_t>(tokens) * (q_heads / kv_heads) > kFewRows;
    s.few += !many && tokens != 0;
    s.many += many;
  }
  s.parts = 1;
  if (s.many == 0) return s;
  const uint64_t blocks = (static_cast<uint64_t>(most) * (q_heads / kv_heads) + kWeightRows - 1) / kWeightRows;
  const uint64_t items = static_cast<uint64_t>(s.columns) * kv_heads * s.many;
  s.parts = static_cast<uint32_t>(std::clamp<uint64_t>(6 * kComputeUnits / items, 1, std::max<uint64_t>(1, blocks / 8)));
  return s;
}

// (At least a little, also where nothing is divided: a workspace is always given.)
std::size_t weight_bytes(const KvPages& p, uint32_t kv_heads, const WeightShape& s) {
  if (s.many == 0) return 16;
  return static_cast<std::size_t>(s.many) * kv_heads * s.parts * (static_cast<std::size_t>(p.stride) << p.page_shift) * sizeof(float);
}

}  // namespace
}  // namespace gfx950

using namespace gfx950;

extern "C" size_t gfxinfer_kv_pages_chunk_attention_workspace_bytes(const gfxinfer_kv_pages* pages, const uint32_t* tokens,
                                                                    uint32_t count, uint32_t q_heads) {
  size_t bytes = 0;
  guarded([&] {
    ChunkAttnArgs a{};
    if (const int32_t s = read_pages(pages, a.pages); s != GFXI_OK) return s;
    if (const int32_t s = read_heads(pages, q_heads); s != GFXI_OK) return s;
    // The slots do not matter here: every entry names the first one.
    const std::vector<uint32_t> any(std::min(count, kMaxChunks + 1), 0u);
    if (const int32_t s = read_chunks(a.pages, any.data(), tokens, count, false, a.list); s != GFXI_OK) return s;
    const ChunkShape shape = chunk_shape(a.pages, a.list, q_heads, pages->kv_heads, pages->head_size, a.first_tile);
    bytes = chunk_bytes(shape, a.list, q_heads, pages->kv_heads, pages->head_size);
    return GFXI_OK;
  });
  return bytes;
}

extern "C" int32_t gfxinfer_launch_kv_pages_chunk_attention(const gfxinfer_kv_pages* pages, uint32_t layer, const uint16_t* query,
                                                            const float* gate, uint16_t* output, float* log_sums,
                                                            const uint32_t* sequences, const uint32_t* tokens, uint32_t count,
                                                            uint32_t q_heads, float* workspace, size_t workspace_bytes,
                                                            void* stream) {
  return guarded([&] {
    ChunkAttnArgs a{};
    if (const int32_t s = read_pages(pages, a.pages); s != GFXI_OK) return s;
    if (const int32_t s = read_heads(pages, q_heads); s != GFXI_OK) return s;
    if (const int32_t s = read_chunks(a.pages, sequences, tokens, count, false, a.list); s != GFXI_OK) return s;
    if (layer >= a.pages.layers || query == nullptr || output == nullptr || !aligned16(query) || !aligned16(gate) ||
        (reinterpret_cast<uintptr_t>(output) & 7u) != 0 || (reinterpret_cast<uintptr_t>(log_sums) & 3u) != 0) {
      return fail(GFXI_INVALID_ARGUMENT, "chunk attention needs a layer of the cache and aligned rows (query and gate 16 bytes, "
                                         "output 8)");
    }
    const uint32_t head_size = pages->head_size, kv_heads = pages->kv_heads;
    const ChunkShape shape = chunk_shape(a.pages, a.list, q_heads, kv_heads, head_size, a.first_tile);
    const std::size_t need = chunk_bytes(shape, a.list, q_heads, kv_heads, head_size);
    if (need != 0 && (workspace == nullptr || !aligned16(workspace) || workspace_bytes < need)) {
      return fail(GFXI_INVALID_ARGUMENT, "chunk attention workspace is null, not 16-byte aligned or too small");
    }
    const uint32_t items = shape.tiles * kv_heads, rows = partial_rows(shape, a.list, q_heads, kv_heads);
    a.query = reinterpret_cast<const __half*>(query);
    a.gate = gate;
    a.output = reinterpret_cast<__half*>(output);
    a.log_sums = log_sums;
    if (need != 0) {
      a.partial_o = workspace;
      a.partial_ml = a.partial_o + static_cast<std::size_t>(rows) * shape.ranges * head_size;
    }
    a.layer = layer;
    a.q_heads = q_heads;
    a.kv_heads = kv_heads;
    a.group = q_heads / kv_heads;
    a.ranges = shape.ranges;
    a.tiles = shape.tiles;
    a.whole = shape.whole;
    a.tile_rows = shape.tile_rows;
    a.scale = kLog2E / std::sqrt(static_cast<float>(head_size));
    const hipStream_t st = static_cast<hipStream_t>(stream);
    const dim3 grid(items + (items - shape.whole) * (shape.ranges - 1)), block(kWaves * 64), join((rows + 3) / 4);
    if (head_size == 128) hipLaunchKernelGGL(chunk_attention_kernel<128>, grid, block, 0, st, a);
    else hipLaunchKernelGGL(chunk_attention_kernel<256>, grid, block, 0, st, a);
    if (const int32_t s = launch_status("chunk attention launch failed"); s != GFXI_OK || a.ranges == 1) return s;
    if (shape.whole == 0) {
      if (head_size == 128) hipLaunchKernelGGL((chunk_join_kernel<128, false>), join, dim3(256), 0, st, a, rows);
      else hipLaunchKernelGGL((chunk_join_kernel<256, false>), join, dim3(256), 0, st, a, rows);
    } else {
      if (head_size == 128) hipLaunchKernelGGL((chunk_join_kernel<128, true>), join, dim3(256), 0, st, a, rows);
      else hipLaunchKernelGGL((chunk_join_kernel<256, true>), join, dim3(256), 0, st, a, rows);
    }
    return launch_status("chunk attention join launch failed");
  });
}

extern "C" size_t gfxinfer_kv_weights_workspace_bytes(const gfxinfer_kv_pages* pages, const uint32_t* tokens, uint32_t count,
                                                      uint32_t q_heads) {
  size_t bytes = 0;
  guarded([&] {
    KvPages p;
    ChunkList list;
    if (const int32_t s = read_pages(pages, p); s != GFXI_OK) return s;
    if (const int32_t s = read_heads(pages, q_heads); s != GFXI_OK) return s;
    const std::vector<uint32_t> any(std::min(count, kMaxChunks + 1), 0u);
    if (const int32_t s = read_chunks(p, any.data(), tokens, count, false, list); s != GFXI_OK) return s;
    bytes = weight_bytes(p, pages->kv_heads, weight_shape(p, list, q_heads, pages->kv_heads));
    return GFXI_OK;
  });
  return bytes;
}

extern "C" int32_t gfxinfer_launch_kv_weights_add(const gfxinfer_kv_pages* pages, const gfxinfer_kv_weights* weights,
                                                  uint32_t layer, const uint16_t* query, const float* log_sums,
                                                  const uint32_t* sequences, const uint32_t* tokens, uint32_t count,
                                                  uint32_t q_heads, void* workspace, size_t workspace_bytes, void* stream) {
  return guarded([&] {
    WeightArgs a{};
    if (const int32_t s = read_pages(pages, a.pages); s != GFXI_OK) return s;
    if (const int32_t s = read_weights(weights, a.weights); s != GFXI_OK) return s;
    if (const int32_t s = read_heads(pages, q_heads); s != GFXI_OK) return s;
    ChunkList list;
    if (const int32_t s = read_chunks(a.pages, sequences, tokens, count, true, list); s != GFXI_OK) return s;
    if (layer >= a.pages.layers || query == nullptr || log_sums == nullptr || !aligned16(query) ||
        (reinterpret_cast<uintptr_t>(log_sums) & 3u) != 0) {
      return fail(GFXI_INVALID_ARGUMENT, "weights need a layer of the cache, 16-byte aligned queries and their log sums");
    }
    a.kv_heads = pages->kv_heads;
    const WeightShape shape = weight_shape(a.pages, list, q_heads, a.kv_heads);
    a.parts = shape.parts;
    a.columns = shape.columns;
    if (workspace == nullptr || !aligned16(workspace) || workspace_bytes < weight_bytes(a.pages, a.kv_heads, shape)) {
      return fail(GFXI_INVALID_ARGUMENT, "K/V weights workspace is null, not 16-byte aligned or too small");
    }
    a.query = reinterpret_cast<const __half*>(query);
    a.log_sums = log_sums;
    a.partial = static_cast<float*>(workspace);
    a.layer = layer;
    a.q_heads = q_heads;
    a.group = q_heads / a.kv_heads;
    a.scale = kLog2E / std::sqrt(static_cast<float>(pages->head_size));
    const hipStream_t st = static_cast<hipStream_t>(stream);
    const uint64_t capacity = static_cast<uint64_t>(a.pages.stride) << a.pages.page_shift;
    // A launch's sequences in the order of the list; only then is the place of one known without another load.
    auto list_items = [&](bool few) {
      for (uint32_t i = 0, at = 0; i < count; ++i) {
        const WeightItem item{list.slot[i], list.first[i], list.first[i + 1] - list.first[i]};
        const bool few_rows = static_cast<uint64_t>(item.tokens) * a.group <= kFewRows;
        if (few_rows == few && item.tokens != 0) a.item[at++] = item;
      }
    };
    if (shape.few != 0) {
      list_items(true);
      const dim3 grid(static_cast<unsigned>(std::min<uint64_t>((capacity + 31) / 32, 1024)), shape.few);
      if (pages->head_size == 128) hipLaunchKernelGGL(few_weight_kernel<128>, grid, dim3(256), 0, st, a);
      else hipLaunchKernelGGL(few_weight_kernel<256>, grid, dim3(256), 0, st, a);
      if (const int32_t s = launch_status("K/V weights launch failed"); s != GFXI_OK) return s;
    }
    if (shape.many == 0) return GFXI_OK;
    list_items(false);
    const dim3 grid(a.columns * a.kv_heads * a.parts, shape.many);
    if (pages->head_size == 128) hipLaunchKernelGGL(weight_kernel<128>, grid, dim3(256), 0, st, a);
    else hipLaunchKernelGGL(weight_kernel<256>, grid, dim3(256), 0, st, a);
    if (const int32_t s = launch_status("K/V weights launch failed"); s != GFXI_OK) return s;
    hipLaunchKernelGGL(weight_join_kernel, dim3(static_cast<unsigned>(std::min<uint64_t>((capacity + 63) / 64, 1024)), shape.many),
                       dim3(256), 0, st, a);
    return launch_status("K/V weights join launch failed");
  });
}
