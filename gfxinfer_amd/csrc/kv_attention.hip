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
// Scores are computed transposed, S^T = K Q^T, so that a lane holds one row's scores: the
// running maximum takes two lane exchanges, the sum none, and the weights are already the
// B operand of O^T = V^T P^T when the positions of a block are numbered as the score tiles
// leave them (k slot 8 b + e is position 4 b + e of the first tile for e < 4 and 4 b + e - 4
// of the second otherwise).  V passes through LDS, whose transposing reads turn rows of V
// into columns.
//
// Two ways to share an item among the eight waves of a workgroup:
//  - few rows (attend_positions): four waves take turns at blocks of 32 positions, each with its
//    own K and V block in LDS and no barrier in the loop, and merge at the end.
//  - many rows (attend_rows): each wave takes 16 of up to 128 rows, and a K / V row staged in
//    LDS serves them all.
// Both load into LDS directly, without registers, and fill the same places on a CU, so one
// launch holds the prefix's items and the sequences' own, whichever way each goes (two launches
// of two kernels took 6 us more).
//
// What bounds it: with few rows the reads of the cache (64 sequences of 100..900 own positions,
// 8 x 128: 134 MB in 33 us, 4.1 TB/s).  With many, three things that overlap only in part, since
// the waves of a workgroup reach them together: 64 sequences on 32768 shared positions (320 rows
// of a KV head, 480 TFLOP/s, 720 with the second product of the weights) take 91 us, of which
// the matrix units of the fullest SIMDs are busy 45 %, their vector units 53 % and the LDS reads
// take about as much; in copies that leave one out they take 79 us without the second product,
// 81 us without the softmax and 90 us with an eighth of the reads of V.
#include <algorithm>
#include <cmath>

#include "kv_pages.hpp"

namespace gfx950 {
namespace {

using h8 = _Float16 __attribute__((ext_vector_type(8)));
using f4 = float __attribute__((ext_vector_type(4)));
using h2 = _Float16 __attribute__((ext_vector_type(2)));
using f2 = float __attribute__((ext_vector_type(2)));
using u32x4 = unsigned __attribute__((ext_vector_type(4)));
using s16x4 = short __attribute__((ext_vector_type(4)));
using lds_void = __attribute__((address_space(3))) void;
using global_void = __attribute__((address_space(1))) void;

constexpr unsigned kBlock = 32;  // positions: a step of a wave by positions, half of one by rows
constexpr float kLog2E = 1.4426950408889634F;

// The factor between sums with maxima `from` and `to`, from <= to nearly always.  Never zero, so
// that a NaN or an infinity of either reaches the result however far its scores lie below the
// others (2^-126 of a finite sum is nothing beside theirs).
__device__ __forceinline__ float rescale_factor(float from, float to) {
  return fmaxf(__builtin_amdgcn_exp2f(from - to), 0x1p-126F);
}

// A row's weights are 2^(score - m + kLift), scores in units of log2.  The stored maximum m follows
// the maxima of the blocks of positions, downwards too, once one leaves [m - kFall, m + kRise], but
// stays within kSpan of its highest value so that the sums fit fp32.  The largest weight of every
// block so lies between 2^-1 and 2^15, near the top of fp16, and 2^-25, half of fp16's last place,
// is at least 2^24 below it.  (At most 2^8, cut off at 2^-24 and never raised again, the weights
// beside a score 16 nats above 600 others lost 16 % of their sum.)
constexpr float kLift = 11.0F, kRise = 4.0F, kFall = 12.0F, kSpan = 32.0F;
// In a block that moves m, weights below 2^kSmall are multiplied on their own, times kSmallScale
// (down to 2^-49, 41 nats below m), if no weight of the row lies between 2^kBetween and the peak's:
// one that does carries more of the output than the others lose.  Scores that spread by 6 nats have
// one in nearly every block (64 sequences on 32768: 130 us, 168 without this condition, 118 where
// scores spread by 1).
constexpr float kSmall = -9.0F, kBetween = -4.0F, kPeak = 8.0F, kSmallScale = 0x1p24F;

constexpr unsigned kWaves = 8;     // of a workgroup; by rows: 128 rows
constexpr unsigned kPosWaves = 4;  // of them, those that divide positions: a block of K and of V each in LDS
// Workgroups a CU holds: 64 KB of LDS and 128 registers at head size 128, 128 KB and 256 at 256.
constexpr unsigned resident(unsigned head_size) { return head_size == 256 ? 1u : 2u; }
// Blocks a split of the prefix, and of a sequence's own positions, is worth at least.  With 8 of
// the prefix, 8 verify blocks on 2000 positions at head size 256 take 31 us, not 27 (with 2, 32
// sequences on 4000 35 us, not 27); with 8 of its own, one sequence of 4000 15.0 us, not 13.1
// (with 2, 14.1).
constexpr uint32_t kPrefixBlocks = 4, kOwnBlocks = 4;

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

// Positions of a tile of attend_rows (16 KB of K and of V at head size 128, 32 KB at 256), and the
// tiles its LDS ring holds.  A wave takes a tile's positions as one step: with 32 a step, more
// maxima and longer waits, 64 sequences on 32768 positions took 118 us, not 115, and at head size
// 256 32 rows of one sequence on 16000 57 us, not 54.
constexpr unsigned kTile = 64, kRing = 2;

// `blocks` blocks over at most `splits` splits of at least `least`: blocks per split (whole
// tiles), and the splits in use.
__device__ __forceinline__ uint32_t split_length(uint32_t blocks, uint32_t splits, uint32_t least) {
  constexpr uint32_t kUnit = kTile / kBlock;
  return max(least, ((blocks + splits - 1) / splits + kUnit - 1) / kUnit * kUnit);
}
__device__ __forceinline__ uint32_t splits_used(uint32_t blocks, uint32_t splits, uint32_t least) {
  const uint32_t per = split_length(blocks, splits, least);
  return (blocks + per - 1) / per;
}
// Committed positions of a slot; a damaged length does not lead far past the table.
__device__ __forceinline__ uint32_t committed(const KvPages& p, uint32_t slot) {
  return min(static_cast<uint32_t>(__builtin_amdgcn_readfirstlane(p.lengths[slot])), p.stride << p.page_shift);
}
// Positions the batch's prefix covers: what the first sequence has of them.
__device__ __forceinline__ uint32_t prefix_length(const PagedAttnArgs& a) {
  return min(a.shared, committed(a.pages, listed_slot(a.list, 0)));
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

// Over the four lanes (one per 16-lane row) that hold a row's scores.
__device__ __forceinline__ float max_over_quarters(float v) {
  const unsigned u = __float_as_uint(v);
  const auto p = __builtin_amdgcn_permlane16_swap(u, u, false, false);
  const unsigned w = __float_as_uint(__builtin_elementwise_maximum(__uint_as_float(p[0]), __uint_as_float(p[1])));
  const auto q = __builtin_amdgcn_permlane32_swap(w, w, false, false);
  return __builtin_elementwise_maximum(__uint_as_float(q[0]), __uint_as_float(q[1]));
}
__device__ __forceinline__ float sum_over_quarters(float v) {
  const unsigned u = __float_as_uint(v);
  const auto p = __builtin_amdgcn_permlane16_swap(u, u, false, false);
  const unsigned w = __float_as_uint(__uint_as_float(p[0]) + __uint_as_float(p[1]));
  const auto q = __builtin_amdgcn_permlane32_swap(w, w, false, false);
  return __uint_as_float(q[0]) + __uint_as_float(q[1]);
}

// Waits until at most Loads of the wave's loads from memory are on their way, and for all of
// its LDS accesses.
template <unsigned Loads>
__device__ __forceinline__ void wait_loads() {
  static_assert(Loads < 64);
  __builtin_amdgcn_s_waitcnt((Loads & 15u) | (Loads >> 4) << 14 | 7u << 4);
  asm volatile("" ::: "memory");
}

// K and V rows in LDS have no padding (loads into LDS fill it lane after lane); instead the
// 16-byte pieces of a row are permuted, by the address each lane loads from: piece c of K row
// r lies in slot c ^ (r % 16), of V row r in slot c ^ 2 (r % 8).  The rows of a score operand
// and of a transposing read then fall on different banks.
__device__ __forceinline__ unsigned key_slot(unsigned piece, unsigned row) { return piece ^ (row & 15u); }
__device__ __forceinline__ unsigned value_slot(unsigned piece, unsigned row) { return piece ^ 2 * (row & 7u); }

// A load of a wave into LDS covers 512 / D rows: where the lane's piece lies in memory, in
// elements from the first of them, if that is row 0 of a tile.  From row r on (a multiple of
// the rows of a load) it is at this ^ 8 (r % 16) for K and ^ 16 (r % 8) for V: rows start at
// multiples of D elements.
template <unsigned D>
__device__ __forceinline__ uint32_t key_piece(unsigned lane, uint32_t row_elements) {
  const unsigned r = lane / (D / 8);
  return r * row_elements + 8 * key_slot(lane % (D / 8), r);
}
template <unsigned D>
__device__ __forceinline__ uint32_t value_piece(unsigned lane, uint32_t row_elements) {
  const unsigned r = lane / (D / 8);
  return r * row_elements + 8 * value_slot(lane % (D / 8), r);
}

// Where the lane's part of the first score operand of 16 K rows, and of the first output tile
// of 16 V rows, lies in bytes from the rows.  Operand s is at the address ^ 64 s, output tile
// d at the address ^ 32 d: the slots of a row are permuted by exclusive or, and rows start at
// multiples of their size.
template <unsigned D>
__device__ __forceinline__ unsigned key_place() {
  const unsigned lane = threadIdx.x & 63u, n = lane & 15u;
  return n * (D * 2) + 16 * key_slot(lane >> 4, n);
}
template <unsigned D>
__device__ __forceinline__ unsigned value_place() {
  const unsigned lane = threadIdx.x & 63u, n = lane & 15u, row = 4 * (lane >> 4) + (n >> 2);
  return row * (D * 2) + 16 * value_slot((n & 3u) >> 1, row) + 8 * (n & 1u);
}
__device__ __forceinline__ unsigned lds_address(const _Float16* p) {
  return static_cast<unsigned>(reinterpret_cast<uintptr_t>((lds_void*)(p)));
}

// Reads from LDS that are complete when they return.  The compiler lets its own reads wait
// for every load into LDS that is on its way, since it cannot tell the places apart; the
// callers have waited for these rows, so the reads are written out with their own wait.
//
// Score operands first .. first + 3 of 32 K rows (k[0]: the first 16 rows).
template <unsigned D>
__device__ __forceinline__ void read_keys(unsigned place, unsigned first, h8 (&k)[2][4]) {
  asm volatile(
      "ds_read_b128 %0, %8\n\tds_read_b128 %4, %8 offset:%12\n\t"
      "ds_read_b128 %1, %9\n\tds_read_b128 %5, %9 offset:%12\n\t"
      "ds_read_b128 %2, %10\n\tds_read_b128 %6, %10 offset:%12\n\t"
      "ds_read_b128 %3, %11\n\tds_read_b128 %7, %11 offset:%12\n\t"
      "s_waitcnt lgkmcnt(0)"
      : "=&v"(k[0][0]), "=&v"(k[0][1]), "=&v"(k[0][2]), "=&v"(k[0][3]), "=&v"(k[1][0]), "=&v"(k[1][1]), "=&v"(k[1][2]), "=&v"(k[1][3])
      : "v"(place ^ 64 * first), "v"(place ^ 64 * (first + 1)), "v"(place ^ 64 * (first + 2)), "v"(place ^ 64 * (first + 3)),
        "n"(16 * D * 2)
      : "memory");
}
// Output tiles first .. first + 3 of 32 V rows.
template <unsigned D>
__device__ __forceinline__ void read_values(unsigned place, unsigned first, h8 (&v)[4]) {
  s16x4 a[8];
  asm volatile(
      "ds_read_b64_tr_b16 %0, %8\n\tds_read_b64_tr_b16 %1, %8 offset:%12\n\t"
      "ds_read_b64_tr_b16 %2, %9\n\tds_read_b64_tr_b16 %3, %9 offset:%12\n\t"
      "ds_read_b64_tr_b16 %4, %10\n\tds_read_b64_tr_b16 %5, %10 offset:%12\n\t"
      "ds_read_b64_tr_b16 %6, %11\n\tds_read_b64_tr_b16 %7, %11 offset:%12\n\t"
      "s_waitcnt lgkmcnt(0)"
      : "=&v"(a[0]), "=&v"(a[1]), "=&v"(a[2]), "=&v"(a[3]), "=&v"(a[4]), "=&v"(a[5]), "=&v"(a[6]), "=&v"(a[7])
      : "v"(place ^ 32 * first), "v"(place ^ 32 * (first + 1)), "v"(place ^ 32 * (first + 2)), "v"(place ^ 32 * (first + 3)),
        "n"(16 * D * 2)
      : "memory");
#pragma unroll
  for (unsigned u = 0; u < 4; ++u) {
    v[u] = __builtin_bit_cast(h8, __builtin_shufflevector(a[2 * u], a[2 * u + 1], 0, 1, 2, 3, 4, 5, 6, 7));
  }
}

// The lane's number, made anew: what is computed from it inside a loop is not kept in
// registers around the loop, where 128 of them do not suffice.
__device__ __forceinline__ unsigned fresh_lane() {
  unsigned lane;
  asm volatile("v_mbcnt_lo_u32_b32 %0, -1, 0\n\tv_mbcnt_hi_u32_b32 %0, -1, %0" : "=v"(lane));
  return lane;
}

// The same for a number that is equal in all lanes.
__device__ __forceinline__ uint32_t fresh_number(uint32_t x) {
  asm volatile("" : "+s"(x));
  return x;
}

// Sixteen rows of a wave: lane column n's row is the query q (B operand), sees the positions
// below `visible`, and its result goes to row out_row (none: 0xffffffff).
template <unsigned D>
struct Rows {
  h8 q[D / 32];
  uint32_t visible, out_row;
  uint32_t least;  // of visible over the rows
  f4 o[D / 16];
  float m, l;  // m in units of log2; l of the lane's own positions
  float peak;  // the highest m so far

  // Rows first + n of `rows`; row = (i * tokens + t) * group + g, i counted from `base`.  Own:
  // the rows are one sequence's, with hi - tokens committed positions.
  template <bool Own>
  __device__ __forceinline__ void load(const PagedAttnArgs& a, uint32_t base, uint32_t first, uint32_t rows, uint32_t hk,
                                       uint32_t hi) {
    const unsigned lane = threadIdx.x & 63u, kb = lane >> 4;
    const uint32_t group = a.q_heads / a.kv_heads, row = first + (lane & 15u);
    visible = 0;
    out_row = 0xffffffffu;
#pragma unroll
    for (unsigned s = 0; s < D / 32; ++s) q[s] = h8{};
    if (row < rows) {
      const uint32_t it = row / group, g = row - it * group, i = Own ? 0u : it / a.tokens, t = it - i * a.tokens;
      out_row = ((base + i) * a.tokens + t) * a.q_heads + hk * group + g;
      const __half* src = a.query + static_cast<std::size_t>(out_row) * D + 8 * kb;
#pragma unroll
      for (unsigned s = 0; s < D / 32; ++s) q[s] = *reinterpret_cast<const h8*>(src + 32 * s);
      visible = Own ? hi - a.tokens + t + 1 : min(min(a.pages.lengths[a.list.slot[base + i]], hi) + t + 1, hi);
    }
    // Own: the first row sees least.  Prefix: every row sees all of it unless the caller's
    // prefix is longer than a sequence, and then every block is treated as an edge.
    if (Own) least = first < rows ? hi - a.tokens + first / group + 1 : 0xffffffffu;
    else least = __all(row >= rows || visible == hi) ? hi : 0u;
  }

  // The queries have arrived here: a wait for them inside a loop would wait for the loop's
  // own loads too.
  __device__ __forceinline__ void settle() {
#pragma unroll
    for (unsigned s = 0; s < D / 32; ++s) asm volatile("" : "+v"(q[s]));
  }

  __device__ __forceinline__ void clear() {
    m = peak = -INFINITY;
    l = 0.0F;
#pragma unroll
    for (unsigned d = 0; d < D / 16; ++d) o[d] = f4{0, 0, 0, 0};
  }

  // Whether an output is an infinity or NaN: weights reach 2^15, 2^47 after m fell, so only such
  // values (or NaN scores) can make one.
  __device__ __forceinline__ bool strange() const {
    bool found = false;
#pragma unroll
    for (unsigned d = 0; d < D / 16; ++d) {
#pragma unroll
      for (unsigned e = 0; e < 4; ++e) found |= !(fabsf(o[d][e]) < INFINITY);
    }
    return found;
  }

  // The raw products of the rows with a block of 32 positions (K rows in LDS, see read_keys).
  __device__ __forceinline__ void score(unsigned place, f4& s0, f4& s1) const {
    s0 = s1 = f4{0, 0, 0, 0};
#pragma unroll
    for (unsigned st = 0; st < D / 32; st += 4) {
      h8 k[2][4];
      read_keys<D>(place, st, k);
#pragma unroll
      for (unsigned u = 0; u < 4; ++u) {
        s0 = __builtin_amdgcn_mfma_f32_16x16x32_f16(k[0][u], q[st + u], s0, 0, 0, 0);
        s1 = __builtin_amdgcn_mfma_f32_16x16x32_f16(k[1][u], q[st + u], s1, 0, 0, 0);
      }
    }
  }

  // p = high + low, both rounded to nearest: off by 2^-23 p, or by 2^-25 if that is more.
  static __device__ __forceinline__ void halves(float p0, float p1, h8& high, h8& low, unsigned at) {
    const h2 h = __builtin_convertvector((f2{p0, p1}), h2);
    const h2 rest = __builtin_convertvector((f2{p0 - static_cast<float>(h[0]), p1 - static_cast<float>(h[1])}), h2);
#pragma unroll
    for (unsigned e = 0; e < 2; ++e) {
      high[at + e] = h[e];
      low[at + e] = rest[e];
    }
  }

  // Takes the small weights of rows with a peak alone out of the scores s of a block and adds their
  // products.  The outputs are scaled for that and back: powers of two, so nothing is rounded, and
  // no registers.
  template <unsigned T>
  __device__ __forceinline__ void add_small(f4 (&s)[T], float scale, unsigned value_at, bool alone) {
#pragma unroll
    for (unsigned d = 0; d < D / 16; ++d) o[d] *= kSmallScale;
#pragma unroll
    for (unsigned b = 0; b < T / 2; ++b) {
      h8 high, low;
#pragma unroll
      for (unsigned e = 0; e < 8; e += 2) {
        float p[2];
#pragma unroll
        for (unsigned u = 0; u < 2; ++u) {
          const float x = fmaf(s[2 * b + e / 4][e % 4 + u], scale, kLift - m);
          const bool here = alone && x < kSmall;
          p[u] = here ? __builtin_amdgcn_exp2f(x) : 0.0F;
          if (here) s[2 * b + e / 4][e % 4 + u] = -INFINITY;
          l += p[u];
          p[u] *= kSmallScale;
        }
        halves(p[0], p[1], high, low, e);
      }
#pragma unroll
      for (unsigned d = 0; d < D / 16; d += 4) {
        h8 v[4];
        read_values<D>(value_at + b * kBlock * D * 2, d, v);
        add(v, d, high, low);
      }
    }
#pragma unroll
    for (unsigned d = 0; d < D / 16; ++d) o[d] *= 1.0F / kSmallScale;
  }

  // The weights of T tiles of 16 positions from `at`: s the scores (raw products), the weights
  // afterwards.  An edge block holds positions that some row does not see (below lo, past its
  // end, or in a tile of 16 whose page is missing: bit t of `missing`).
  //
  // The weights go out as fp16 pairs, which keeps the accuracy of an fp32 product unless a peak
  // lies far above the others of its block and the others carry the output (the peak's value is
  // near zero): then add_small takes the others.  ready() returns when the block's V rows
  // are in LDS at value_at, zeros where no row sees them.
  template <unsigned T, typename Ready>
  __device__ __forceinline__ void weigh(f4 (&s)[T], unsigned lane, float scale, bool edge, uint32_t at, uint32_t lo,
                                        unsigned missing, unsigned value_at, Ready ready, h8 (&high)[T / 2],
                                        h8 (&low)[T / 2]) {
    if (edge) {
      const unsigned kb = lane >> 4;
#pragma unroll
      for (unsigned t = 0; t < T; ++t) {
#pragma unroll
        for (unsigned r = 0; r < 4; ++r) {
          const uint32_t position = at + 16 * t + 4 * kb + r;
          if (position < lo || position >= visible || (missing >> t & 1u) != 0) s[t][r] = -INFINITY;
        }
      }
    }
    // (A NaN score makes the maximum NaN and the row's result with it, as it has to.)
    float best = s[0][0];
#pragma unroll
    for (unsigned r = 1; r < 4 * T; ++r) best = __builtin_elementwise_maximum(best, s[r / 4][r % 4]);
    const float top = max_over_quarters(best) * scale;
    // Most blocks skip this.  m moves only for the rows that need it, so that a row's result does
    // not depend on the scores of the others.
    if (__any(fabsf(top - (m - 0.5F * (kFall - kRise))) > 0.5F * (kFall + kRise))) {
      const float target = fmaxf(top, peak - kSpan);
      const float next_m = top > m + kRise ? top : top != -INFINITY && target < m - kFall ? target : m;
      const float factor = next_m == m ? 1.0F : rescale_factor(m, next_m);
      m = next_m;
      peak = fmaxf(peak, m);
      l *= factor;
#pragma unroll
      for (unsigned d = 0; d < D / 16; ++d) o[d] *= factor;
      float least_score = s[0][0];
#pragma unroll
      for (unsigned e = 1; e < 4 * T; ++e) least_score = __builtin_elementwise_minimum(least_score, s[e / 4][e % 4]);
      if (edge) {  // of the positions that are seen
        least_score = INFINITY;
#pragma unroll
        for (unsigned e = 0; e < 4 * T; ++e) {
          const float x = s[e / 4][e % 4];
          least_score = __builtin_elementwise_minimum(least_score, x == -INFINITY ? INFINITY : x);
        }
      }
      const bool small = factor != 1.0F && fmaf(least_score, scale, kLift - m) < kSmall;
      if (__builtin_expect(__any(small), 0)) {
        bool between = false;
#pragma unroll
        for (unsigned e = 0; e < 4 * T; ++e) {
          const float x = fmaf(s[e / 4][e % 4], scale, kLift - m);
          between |= x >= kBetween && x < kPeak;
        }
        uint64_t rows = __ballot(between);
        rows |= rows >> 32 | rows << 32;  // a row's four lanes
        rows |= rows >> 16 | rows << 48;
        const bool alone = factor != 1.0F && (rows >> lane & 1u) == 0;
        if (__any(alone && small)) {
          ready();
          add_small(s, scale, value_at, alone);
        }
      }
    }
    const float floor = m == -INFINITY ? 0.0F : m - kLift;
#pragma unroll
    for (unsigned t = 0; t < T; ++t) {
#pragma unroll
      for (unsigned r = 0; r < 4; r += 2) {
        const float p0 = __builtin_amdgcn_exp2f(fmaf(s[t][r], scale, -floor));
        const float p1 = __builtin_amdgcn_exp2f(fmaf(s[t][r + 1], scale, -floor));
        s[t][r] = p0;
        s[t][r + 1] = p1;
        l += p0;
        l += p1;
        halves(p0, p1, high[t / 2], low[t / 2], t % 2 * 4 + r);
      }
    }
  }

  // Output tiles first .. first + 3.
  __device__ __forceinline__ void add(const h8 (&v)[4], unsigned first, const h8& high, const h8& low) {
#pragma unroll
    for (unsigned u = 0; u < 4; ++u) o[first + u] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v[u], low, o[first + u], 0, 0, 0);
#pragma unroll
    for (unsigned u = 0; u < 4; ++u) o[first + u] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v[u], high, o[first + u], 0, 0, 0);
  }

  // In a careful pass the infinities and NaNs among the values of `count` positions are zeros in
  // LDS, since a row must not meet those of positions it does not see; here the rows that see them
  // get them, one by one from the pages, whatever the weight: no weight is exactly zero.
  __device__ __forceinline__ void add_strange(unsigned count, const KvPages& pages, const __half* values, uint32_t slot,
                                              uint32_t at, uint32_t lo, uint32_t hi) {
    const unsigned kb = fresh_lane() >> 4;
#pragma unroll 1
    for (unsigned p = 0; p < count; ++p) {
      const uint32_t position = at + p;
      const int32_t page = position < lo || position >= hi ? -1 : table_page(pages, slot, position >> pages.page_shift);
      if (page < 0) continue;
      const __half* row = values + ((static_cast<std::size_t>(page) << pages.page_shift) +
                                    (position & ((1u << pages.page_shift) - 1))) * pages.row;
#pragma unroll
      for (unsigned d = 0; d < D / 16; ++d) {
#pragma unroll
        for (unsigned e = 0; e < 4; ++e) {
          const float x = __half2float(row[16 * d + 4 * kb + e]);
          if (!(fabsf(x) < INFINITY) && position < visible) o[d][e] += x;
        }
      }
    }
    // Nothing is on its way when the ordinary blocks go on.
    wait_loads<0>();
  }

  // The row sums, complete.  Only NaN scores, and strange values at scores of -infinity, make a NaN
  // row rather than an empty one.
  __device__ __forceinline__ void finish(bool careful) {
    l = sum_over_quarters(l);
    if (m == -INFINITY && (l != l || (careful && strange()))) m = 0.0F;
  }
};

// Eight values in LDS: infinities and NaNs become zeros.  Whether there were any.
__device__ __forceinline__ bool take_strange(u32x4* at) {
  u32x4 v = *at;
  bool strange = false;
#pragma unroll
  for (unsigned e = 0; e < 4; ++e) {
    const bool low = (v[e] & 0x7c00u) == 0x7c00u, high = (v[e] & 0x7c000000u) == 0x7c000000u;
    strange |= low || high;
    v[e] &= (low ? 0xffff0000u : 0xffffffffu) & (high ? 0xffffu : 0xffffffffu);
  }
  if (strange) *at = v;
  return strange;
}

// A sequence's table row, 64 columns at a time in the lanes of a wave: a block's page is a
// lane read, not a load on the way to the block's addresses.
struct PageWindow {
  uint32_t first;
  int32_t entry;
  __device__ __forceinline__ void start(const KvPages& pages, uint32_t slot, uint32_t column) {
    first = column;
    entry = table_page(pages, slot, column + (threadIdx.x & 63u));
  }
  __device__ __forceinline__ int32_t find(const KvPages& pages, uint32_t slot, uint32_t column) {
    if (column - first >= 64u) start(pages, slot, column);  // uniform: columns only grow
    return __builtin_amdgcn_readlane(entry, column - first);
  }
};

// The K or V rows of a KV head of the launch's layer.
__device__ __forceinline__ const __half* head_rows(const PagedAttnArgs& a, const __half* pool, uint32_t hk, unsigned d) {
  return pool + (static_cast<std::size_t>(a.layer) * a.pages.page_count << a.pages.page_shift) * a.pages.row + hk * d;
}

// One work item: rows first .. (see Rows::load), KV head hk, positions [lo, hi) in blocks
// first_block .. last_block - 1 from position `start` (a multiple of 16), pages of sequence
// `slot`, result into split `split`.
struct Item {
  uint32_t base, first, rows, hk, slot, start, first_block, last_block, lo, hi, split;
  bool own;
};

// Whether x holds in any lane of the workgroup.  flags: a word per wave, used once.  (__syncthreads_or
// keeps the thread's number in a register for it: spilled before the loop, its store is one that
// the first loads wait for; 200 sequences of 250..500 positions took 81 us, not 75.)
__device__ __forceinline__ bool in_any_wave(bool x, unsigned wave, uint32_t* flags) {
  const bool mine = __any(x);
  if (fresh_lane() == 0) flags[wave] = mine ? 1u : 0u;
  __syncthreads();
  uint32_t found = 0;
#pragma unroll
  for (unsigned v = 0; v < kWaves; ++v) found |= flags[v];
  return __builtin_amdgcn_readfirstlane(found) != 0;
}

// Tiles of K and V rows and their marks (attend_rows); the waves' flags follow.
template <unsigned D>
constexpr std::size_t rows_bytes() {
  return kRing * (kTile * D * 2 * 2 + 4 * kWaves);
}

// Sixteen rows; the waves divide the positions.
template <unsigned D>
__device__ __forceinline__ void attend_positions(const PagedAttnArgs& a, const Item& w, char* smem) {
  constexpr unsigned kTiles = D / 16;
  constexpr unsigned kLoads = kBlock * D / 8 / 64;   // of a block's K rows, and of its V rows, per lane
  constexpr unsigned kLoadRows = 64 / (D / 8);       // rows one of them covers
  const unsigned wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const KvPages& pg = a.pages;
  const uint32_t in_page = (1u << pg.page_shift) - 1;
  PageWindow window;
  window.start(pg, w.slot, (w.start + min(w.first_block + wave, w.last_block - 1) * kBlock) >> pg.page_shift);
  uint32_t* flags = reinterpret_cast<uint32_t*>(smem + rows_bytes<D>());
  Rows<D> rows;
  if (w.own) rows.template load<true>(a, w.base, w.first, w.rows, w.hk, w.hi);
  else rows.template load<false>(a, w.base, w.first, w.rows, w.hk, w.hi);
  const __half* keys = head_rows(a, pg.key, w.hk, D);
  const __half* values = head_rows(a, pg.value, w.hk, D);
  _Float16* ks = reinterpret_cast<_Float16*>(smem) + wave * 2 * kBlock * D;
  _Float16* vs = ks + kBlock * D;
  const unsigned key_at = lds_address(ks) + key_place<D>(), value_at = lds_address(vs) + value_place<D>();

  int32_t page[2];
  auto find_pages = [&](uint32_t at, int32_t (&out)[2]) __attribute__((always_inline)) {
#pragma unroll
    for (unsigned t = 0; t < 2; ++t) out[t] = at + 16 * t < w.hi ? window.find(pg, w.slot, (at + 16 * t) >> pg.page_shift) : -1;
  };
  // Missing tiles load page 0 of the pool (always there); their scores and values are masked.
  auto tile_row = [&](uint32_t at, unsigned t, const int32_t (&p)[2]) __attribute__((always_inline)) {
    return (static_cast<std::size_t>(max(p[t], 0)) << pg.page_shift) + ((at + 16 * t) & in_page);
  };
  auto load_k = [&](uint32_t at, const int32_t (&p)[2]) __attribute__((always_inline)) {
    const uint32_t key_part = key_piece<D>(fresh_lane(), pg.row);
#pragma unroll
    for (unsigned u = 0; u < kLoads; ++u) {
      const unsigned t = u / (kLoads / 2), r = kLoadRows * (u % (kLoads / 2));
      __builtin_amdgcn_global_load_lds((global_void*)(keys + (tile_row(at, t, p) + r) * pg.row + (key_part ^ 8 * r)),
                                       (lds_void*)(ks + kLoadRows * u * D), 16, 0, 0);
    }
  };
  auto load_v = [&](uint32_t at, const int32_t (&p)[2]) __attribute__((always_inline)) {
    const uint32_t value_part = value_piece<D>(fresh_lane(), pg.row);
#pragma unroll
    for (unsigned u = 0; u < kLoads; ++u) {
      const unsigned t = u / (kLoads / 2), r = kLoadRows * (u % (kLoads / 2));
      __builtin_amdgcn_global_load_lds((global_void*)(values + (tile_row(at, t, p) + r) * pg.row + (value_part ^ 16 * (r & 7u))),
                                       (lds_void*)(vs + kLoadRows * u * D), 16, 0, 0);
    }
  };

  // A second, careful pass follows in the rare case that an output of the first is an
  // infinity or NaN: values are then looked at before they are used.
  bool careful = false;
  for (;; careful = true) {
    rows.clear();
    if (careful) window.first = 0xffffffc0u;  // 64 before column 0
    uint32_t block = fresh_number(wave < kPosWaves ? w.first_block + wave : w.last_block);
    if (block < w.last_block) {
      find_pages(w.start + block * kBlock, page);
      load_k(w.start + block * kBlock, page);
      load_v(w.start + block * kBlock, page);
    }
    rows.settle();
#pragma unroll 1
    for (; block < w.last_block; block += kPosWaves) {
      const uint32_t at = w.start + block * kBlock;
      const unsigned fresh = fresh_lane();
      const bool edge = at < w.lo || at + kBlock > rows.least || page[0] < 0 || page[1] < 0;
      const unsigned missing = (page[0] < 0 ? 1u : 0u) | (page[1] < 0 ? 2u : 0u);
      // The K rows are there when only their V rows are on their way.
      wait_loads<kLoads>();
      f4 s[2];
      rows.score(key_at, s[0], s[1]);
      const bool more = block + kPosWaves < w.last_block;
      if (more) {
        find_pages(at + kPosWaves * kBlock, page);
        load_k(at + kPosWaves * kBlock, page);
      }
      // The V rows are there when only the next K rows are on their way.  Rows no one sees become
      // zeros (what a page holds past a sequence's end may be anything, and 0 * NaN would be NaN);
      // nearly always those from the end on.
      bool strange = false;
      auto ready = [&]() __attribute__((always_inline)) {
        if (more) wait_loads<kLoads>();
        else wait_loads<0>();
        if (edge || careful) {
          const unsigned fresh = fresh_lane();
          const bool end_only = !careful && missing == 0 && at >= w.lo;
#pragma unroll 1
          for (unsigned u = end_only ? (w.hi - at) / kLoadRows : 0; u < kLoads; ++u) {
            const unsigned t = u / (kLoads / 2), r = kLoadRows * u + fresh / (D / 8);
            u32x4* piece = reinterpret_cast<u32x4*>(vs + kLoadRows * u * D) + fresh;
            if (at + r < w.lo || at + r >= w.hi || (missing >> t & 1u) != 0) *piece = u32x4{0, 0, 0, 0};
            if (careful) strange |= take_strange(piece);
          }
          wait_loads<63>();
        }
      };
      h8 high[1], low[1];
      rows.weigh(s, fresh, a.scale, edge, at, w.lo, missing, value_at, ready, high, low);
      ready();
      if (careful && __any(strange)) rows.add_strange(kBlock, pg, values, w.slot, at, w.lo, w.hi);
#pragma unroll
      for (unsigned d = 0; d < kTiles; d += 4) {
        h8 v[4];
        read_values<D>(value_at, d, v);
        rows.add(v, d, high[0], low[0]);
      }
      if (more) load_v(at + kPosWaves * kBlock, page);
    }
    if (careful || !in_any_wave(rows.strange(), wave, flags)) break;
  }

  // Merge the waves (a lane holds the same row and dims in every wave): all maxima and
  // outputs through LDS, then each wave sums its share of the output tiles in wave order.
  __syncthreads();  // the K and V rows are no longer needed
  const unsigned late = fresh_lane(), n = late & 15u, kb = late >> 4;
  f4* outputs = reinterpret_cast<f4*>(smem);                                 // [waves][D / 16][64]
  float2* ml = reinterpret_cast<float2*>(smem + kPosWaves * kTiles * 64 * 16);  // [waves][16]
  rows.finish(careful);
  if (wave < kPosWaves) {
    if (kb == 0) ml[wave * 16 + n] = float2{rows.m, rows.l};
#pragma unroll
    for (unsigned d = 0; d < kTiles; ++d) outputs[(wave * kTiles + d) * 64 + late] = rows.o[d];
  }
  __syncthreads();
  float best = -INFINITY, total = 0.0F, factor[kPosWaves];
#pragma unroll
  for (unsigned v = 0; v < kPosWaves; ++v) best = fmaxf(best, ml[v * 16 + n].x);
#pragma unroll
  for (unsigned v = 0; v < kPosWaves; ++v) {
    const float2 x = ml[v * 16 + n];
    factor[v] = x.x == -INFINITY ? 0.0F : rescale_factor(x.x, best);
    if (x.x != -INFINITY) total += x.y * factor[v];
  }
  if (rows.out_row == 0xffffffffu) return;
  const std::size_t at = static_cast<std::size_t>(rows.out_row) * (a.prefix_splits + a.own_splits) + w.split;
#pragma unroll
  for (unsigned u = 0; u < kTiles / kWaves; ++u) {
    const unsigned d = wave * (kTiles / kWaves) + u;
    f4 sum = {0, 0, 0, 0};
#pragma unroll
    for (unsigned v = 0; v < kPosWaves; ++v) {
      const f4 x = outputs[(v * kTiles + d) * 64 + late];
      if (factor[v] != 0.0F) sum += x * factor[v];
    }
    *reinterpret_cast<f4*>(a.partial_o + at * D + 16 * d + 4 * kb) = sum;
  }
  if (wave == 0 && kb == 0) *reinterpret_cast<float2*>(a.partial_ml + 2 * at) = float2{best, total};
}

// A barrier that orders LDS accesses and leaves loads from memory into LDS on their way
// (__syncthreads would wait for them).
__device__ __forceinline__ void lds_barrier() {
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}

// Up to 128 rows, 16 a wave; each K / V row is loaded into LDS once for all of them, tiles
// ahead, with one barrier a tile.
template <unsigned D>
__device__ __forceinline__ void attend_rows(const PagedAttnArgs& a, const Item& w, char* smem) {
  constexpr unsigned R = kRing, T = kTile;
  constexpr unsigned kLoads = T * D / 8 / (kWaves * 64);  // of K, and of V, per tile and lane
  constexpr unsigned kLoadRows = 64 / (D / 8);            // rows a load of a wave covers
  const unsigned lane = threadIdx.x & 63u, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const KvPages& pg = a.pages;
  const uint32_t in_page = (1u << pg.page_shift) - 1;
  const __half* keys = head_rows(a, pg.key, w.hk, D);
  const __half* values = head_rows(a, pg.value, w.hk, D);
  _Float16* kring = reinterpret_cast<_Float16*>(smem);            // [ring][tile][D]
  _Float16* vring = kring + R * T * D;                            // [ring][tile][D]
  uint32_t* marks = reinterpret_cast<uint32_t*>(vring + R * T * D);  // [ring][waves]
  const unsigned key_at = lds_address(kring) + key_place<D>(), value_at = lds_address(vring) + value_place<D>();
  const uint32_t last = w.start + w.last_block * kBlock;
  const uint32_t end = min(last, w.hi);

  PageWindow window;
  window.start(pg, w.slot, (w.start + w.first_block * kBlock) >> pg.page_shift);
  bool lost = false;  // a page was missing
  // Load u of a wave covers rows kLoadRows * (wave + 8 u) .. of the tile, all of one part of
  // 16 positions.  Parts without a page load from page 0 (always there) and are dealt with
  // in the careful pass; tiles past the item are not asked for.
  auto part_page = [&](unsigned u, uint32_t at) __attribute__((always_inline)) {
    const uint32_t part = at + (kLoadRows * (wave + kWaves * u) & ~15u);
    return part < end ? window.find(pg, w.slot, part >> pg.page_shift) : 0;
  };
  auto load = [&](unsigned slot, uint32_t at) __attribute__((always_inline)) {
    const unsigned fresh = D == 128 ? fresh_lane() : lane;
    const uint32_t key_part = key_piece<D>(fresh, pg.row), value_part = value_piece<D>(fresh, pg.row);
#pragma unroll
    for (unsigned u = 0; u < kLoads; ++u) {
      const unsigned row0 = kLoadRows * (wave + kWaves * u);
      const int32_t page = part_page(u, at);
      lost |= page < 0;
      const std::size_t base = ((static_cast<std::size_t>(max(page, 0)) << pg.page_shift) + ((at + row0) & in_page)) * pg.row;
      __builtin_amdgcn_global_load_lds((global_void*)(keys + base + (key_part ^ 8 * (row0 & 15u))),
                                       (lds_void*)(kring + (slot * T + row0) * D), 16, 0, 0);
      __builtin_amdgcn_global_load_lds((global_void*)(values + base + (value_part ^ 16 * (row0 & 7u))),
                                       (lds_void*)(vring + (slot * T + row0) * D), 16, 0, 0);
    }
  };
  // The wave's own pieces of a tile, once they have arrived: V rows no one sees become zeros
  // (see attend_positions); a careful pass also takes out infinities and NaNs, and notes them
  // (bit 8) and the missing parts (bit t) for all waves.
  auto repair = [&](unsigned slot, uint32_t at, bool careful) __attribute__((always_inline)) {
    const unsigned lane = fresh_lane();
    uint32_t mark = 0;
    bool strange = false;
#pragma unroll
    for (unsigned u = 0; u < kLoads; ++u) {
      const unsigned row0 = kLoadRows * (wave + kWaves * u), r = row0 + lane / (D / 8);
      bool gone = at + r < w.lo || at + r >= w.hi;
      if (careful && part_page(u, at) < 0) {
        gone = true;
        mark |= 1u << (row0 / 16);
      }
      u32x4* piece = reinterpret_cast<u32x4*>(vring + (slot * T + row0) * D) + lane;
      if (gone) *piece = u32x4{0, 0, 0, 0};
      if (careful) strange |= take_strange(piece);
    }
    if (__any(strange)) mark |= 0x100u;
    if (careful && lane == 0) marks[slot * kWaves + wave] = mark;
  };

  Rows<D> rows;
  uint32_t* flags = reinterpret_cast<uint32_t*>(smem + rows_bytes<D>());
  const uint32_t first = w.first + wave * 16;
  if (w.own) rows.template load<true>(a, w.base, first, w.rows, w.hk, w.hi);
  else rows.template load<false>(a, w.base, first, w.rows, w.hk, w.hi);
  const bool works = first < w.rows;
  // A second, careful pass follows in the rare case that an output of the first is an
  // infinity or NaN, or a page was missing: values and pages are then looked at.
  bool careful = false;
  for (;; careful = true) {
    rows.clear();
    if (careful) window.first = 0xffffffc0u;  // 64 before column 0
    const uint32_t begin = fresh_number(w.start + w.first_block * kBlock);
#pragma unroll
    for (unsigned i = 0; i + 1 < R; ++i) {
      if (begin + i * T < last) load(i, begin + i * T);
    }
    rows.settle();
    unsigned slot = 0;
#pragma unroll 1
    for (uint32_t at = begin; at < last; at += T) {
      // This tile has arrived when only the loads of the R - 2 after it are on their way.
      if (at + (R - 2) * T < last) wait_loads<(R - 2) * 2 * kLoads>();
      else wait_loads<0>();
      if (careful || at < w.lo || at + T > w.hi) {
        repair(slot, at, careful);
        wait_loads<63>();
      }
      lds_barrier();
      // Every wave is past the tile before this one: its slot takes the next loads.
      if (at + (R - 1) * T < last) load((slot + R - 1) % R, at + (R - 1) * T);
      if (works) {
        uint32_t mark = 0;
        if (careful) {
          for (unsigned v = 0; v < kWaves; ++v) mark |= marks[slot * kWaves + v];
          mark = __builtin_amdgcn_readfirstlane(mark);
        }
        const unsigned rows_at = slot * T * D * 2, fresh = fresh_lane();
        f4 s[T / 16];
#pragma unroll
        for (unsigned b = 0; b < T / kBlock; ++b) rows.score(key_at + rows_at + b * kBlock * D * 2, s[2 * b], s[2 * b + 1]);
        const bool edge = at < w.lo || at + T > rows.least || (mark & 0xffu) != 0;
        h8 high[T / kBlock], low[T / kBlock];
        rows.weigh(s, fresh, a.scale, edge, at, w.lo, mark, value_at + rows_at, [] {}, high, low);
        if ((mark & 0x100u) != 0) rows.add_strange(T, pg, values, w.slot, at, w.lo, w.hi);
#pragma unroll
        for (unsigned b = 0; b < T / kBlock; ++b) {
#pragma unroll
          for (unsigned d = 0; d < D / 16; d += 4) {
            h8 v[4];
            read_values<D>(value_at + rows_at + b * kBlock * D * 2, d, v);
            rows.add(v, d, high[b], low[b]);
          }
        }
      }
      slot = (slot + 1) % R;
    }
    if (careful || !in_any_wave((works && rows.strange()) || lost, wave, flags)) break;
  }
  if (!works) return;
  rows.finish(careful);
  const unsigned late = fresh_lane();
  if (rows.out_row == 0xffffffffu) return;
  const std::size_t to = static_cast<std::size_t>(rows.out_row) * (a.prefix_splits + a.own_splits) + w.split;
#pragma unroll
  for (unsigned d = 0; d < D / 16; ++d) *reinterpret_cast<f4*>(a.partial_o + to * D + 16 * d + 4 * (late >> 4)) = rows.o[d];
  if (late < 16) *reinterpret_cast<float2*>(a.partial_ml + 2 * to) = float2{rows.m, rows.l};
}

// Whether the waves share an item's rows or its positions.  By positions, every 16 rows read
// the range again, but four waves work where one or two of eight would.  Microseconds of a call
// by rows and by positions: 8 heads of 128, 25 rows on a prefix of 2000 12.3 and 11.7, of 16000
// both 24.3, 50 rows 13.8 and 12.8, 26.4 and 27.1; 8 sequences of 3900 own positions, 5 rows 27.9
// and 27.1, 20 rows 30.0 and 31.6, 40 rows 32 and 45.  4 heads of 256, 30 rows on 2000 16.9 and
// 15.1, on 16000 32.6 and 29.0, 60 rows 19.6 and 17.5, 35.4 and 35.6; 8 sequences of 3900, 6 rows
// 33.1 and 28.6, 24 rows 35.4 and 33.0, 48 rows 39 and 51.
__host__ __device__ constexpr bool by_rows(uint32_t rows, uint32_t head_size, bool own) {
  return rows > (own && head_size == 128 ? 16u : 32u);
}
// Tiles of rows: of 16, or as few of up to 128 as hold them, evenly filled (10 x 16 rows as 5 + 5,
// not 8 + 2: 160 rows on 16000 positions 42 -> 40 us, on 4 x 256 61 -> 58 us).
__host__ __device__ constexpr uint32_t row_tiles(uint32_t rows, uint32_t head_size, bool own) {
  return by_rows(rows, head_size, own) ? (rows + 16 * kWaves - 1) / (16 * kWaves) : (rows + 15) / 16;
}
__host__ __device__ constexpr uint32_t tile_rows(uint32_t rows, uint32_t tiles) { return ((rows + 15) / 16 + tiles - 1) / tiles * 16; }

// Work items: the prefix's come before the sequences' own.
template <unsigned D>
__global__ __launch_bounds__(kWaves * 64, resident(D) * kWaves / 4) void paged_attention_kernel(PagedAttnArgs a) {
  __shared__ __align__(1024) char smem[rows_bytes<D>() + 4 * kWaves];
  const uint32_t shared = prefix_length(a), id = blockIdx.x;
  const uint32_t group = a.q_heads / a.kv_heads, count = a.list.count;
  uint32_t range, tile;
  Item item;
  bool few;
  if (id < a.prefix_groups) {
    unspread(id, a.prefix_tiles, range, tile);
    const uint32_t split = range / a.kv_heads, hk = range - split * a.kv_heads;
    const uint32_t blocks = (shared + kBlock - 1) / kBlock, per = split_length(blocks, a.prefix_splits, kPrefixBlocks);
    const uint32_t from = split * per;
    if (split >= a.prefix_splits || from >= blocks) return;
    const uint32_t rows = count * a.tokens * group, per_tile = tile_rows(rows, a.prefix_tiles);
    few = !by_rows(rows, D, false);
    item = Item{0, tile * per_tile, min(rows, (tile + 1) * per_tile), hk, listed_slot(a.list, 0), 0, from,
                min(from + per, blocks), 0, shared, split, false};
  } else {
    unspread(id - a.prefix_groups, a.own_tiles, range, tile);
    const uint32_t hk = range % a.kv_heads, is = range / a.kv_heads, split = is / count, i = is - split * count;
    if (split >= a.own_splits) return;
    const uint32_t slot = listed_slot(a.list, i), end = committed(a.pages, slot) + a.tokens;
    const uint32_t blocks = own_blocks(shared, end), per = split_length(blocks, a.own_splits, kOwnBlocks), from = split * per;
    if (from >= blocks) return;
    const uint32_t rows = a.tokens * group, per_tile = tile_rows(rows, a.own_tiles);
    few = !by_rows(rows, D, true);
    item = Item{i, tile * per_tile, min(rows, (tile + 1) * per_tile), hk, slot, shared & ~15u, from,
                min(from + per, blocks), shared, end, a.prefix_splits + split, true};
  }
  if (few) attend_positions<D>(a, item, smem);
  else attend_rows<D>(a, item, smem);
}

// Merges a row's items and applies the gate: one wave per (row, 128 dims), two dims a lane.
// Lane s holds item s's maximum and sum, so its weight is computed once; the outputs are
// loaded kBatch at a time ahead of their use (issued before the maxima are known, or 16 at a
// time, they were no faster: the registers leave fewer waves).  Bound by its chain of lengths,
// maxima and outputs: 1280 rows of up to 18 items 5.4 us, 2560 of 22 8.2 us.
template <unsigned D>
__global__ __launch_bounds__(256) void paged_combine_kernel(PagedAttnArgs a) {
  constexpr unsigned kGroups = D / 128, kBatch = 8;
  const uint32_t linear = blockIdx.x * 4u + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const uint32_t rows = a.list.count * a.tokens * a.q_heads;
  if (linear >= rows * kGroups) return;
  const unsigned lane = threadIdx.x & 63u;
  const uint32_t row = linear / kGroups, part = linear - row * kGroups;
  const uint32_t i = row / (a.tokens * a.q_heads);
  const unsigned d = 128 * part + 2 * lane;
  float2 g = {0.0F, 0.0F};
  if (a.gate != nullptr) g = *reinterpret_cast<const float2*>(a.gate + static_cast<std::size_t>(row) * 2 * D + D + d);
  const uint32_t shared = prefix_length(a), end = committed(a.pages, listed_slot(a.list, i)) + a.tokens;
  const uint32_t prefix = a.prefix_splits != 0 ? splits_used((shared + kBlock - 1) / kBlock, a.prefix_splits, kPrefixBlocks) : 0u;
  const uint32_t items = prefix + splits_used(own_blocks(shared, end), a.own_splits, kOwnBlocks);
  const uint32_t skipped = a.prefix_splits - prefix;  // unused between the prefix's items and the own ones
  const std::size_t first = static_cast<std::size_t>(row) * (a.prefix_splits + a.own_splits);
  const float* ml = a.partial_ml + 2 * first;
  const float* outputs = a.partial_o + first * D + d;
  float best = -INFINITY, total = 0.0F, o0 = 0.0F, o1 = 0.0F;
  for (uint32_t from = 0; from < items; from += 64) {
    const uint32_t s = from + lane;
    const float2 x = s < items ? *reinterpret_cast<const float2*>(ml + 2 * (s < prefix ? s : s + skipped)) : float2{-INFINITY, 0.0F};
    const float next = fmaxf(best, wave_max(x.x));
    if (next == -INFINITY) continue;
    const float keep = best == -INFINITY ? 0.0F : rescale_factor(best, next);
    best = next;
    const float w = x.x == -INFINITY ? 0.0F : rescale_factor(x.x, best);
    total = total * keep + wave_sum(w == 0.0F ? 0.0F : x.y * w);
    o0 *= keep;
    o1 *= keep;
    const uint32_t here = min(64u, items - from);
    for (uint32_t k0 = 0; k0 < here; k0 += kBatch) {
      float2 v[kBatch];
#pragma unroll
      for (unsigned k = 0; k < kBatch; ++k) {
        const uint32_t at = from + min(k0 + k, here - 1);
        v[k] = *reinterpret_cast<const float2*>(outputs + static_cast<std::size_t>(at < prefix ? at : at + skipped) * D);
      }
#pragma unroll
      for (unsigned k = 0; k < kBatch; ++k) {
        const float wk = k0 + k < here ? lane_value(w, k0 + k < here ? k0 + k : 0) : 0.0F;
        if (wk != 0.0F) {  // uniform; also past the last item
          o0 = fmaf(v[k].x, wk, o0);
          o1 = fmaf(v[k].y, wk, o1);
        }
      }
    }
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

struct Shape {
  uint32_t prefix_tiles, own_tiles, prefix_splits, own_splits;
  std::size_t rows;
};

Shape shape_of(const KvPages& p, uint32_t kv_heads, uint32_t head_size, uint32_t count, uint32_t tokens, uint32_t q_heads,
               uint32_t shared) {
  Shape s{};
  const uint32_t group = q_heads / kv_heads;
  s.rows = static_cast<std::size_t>(count) * tokens * q_heads;
  const uint32_t all = count * tokens * group, one = tokens * group;
  s.prefix_tiles = row_tiles(all, head_size, false);
  s.own_tiles = row_tiles(one, head_size, true);
  // Workgroups for the places of an XCD, all row tiles of a range on one (see spread_groups).
  auto splits = [](uint32_t workgroups, uint32_t tiles, uint32_t ranges) { return std::max(1u, workgroups / 8 / tiles * 8 / ranges); };
  // The prefix: a workgroup for every CU, of four blocks or more.  At head size 128 a CU holds a
  // second one, which is left to the own positions until the pieces pass 48 blocks (64 sequences
  // with few own positions: on 8192 with one a CU 38 us, with two 41; on 16384 59 and 58, on
  // 32768 105 and 97, on 65536 194 and 170; on 32768 with 100..900 own positions 119 and 122).
  // At 256 there is no second place, so the own positions have up to a quarter of the GPU left
  // (none: 10 sequences on 16000 35.5 us, not 29.7, 32 rows of one 53.7 us, not 45.6; up to half:
  // 25 sequences 57.5 us, not 49.1).
  const uint32_t blocks = (shared + kBlock - 1) / kBlock;
  if (shared != 0) {
    const uint32_t left = head_size == 256 ? std::min(count * kv_heads * s.own_tiles, kComputeUnits / 4) : 0u;
    uint32_t most = splits(kComputeUnits - left, s.prefix_tiles, kv_heads);
    if (blocks / most > 48) most = splits(kComputeUnits * resident(head_size) - left, s.prefix_tiles, kv_heads);
    s.prefix_splits = std::max(1u, std::min(most, (blocks + kPrefixBlocks - 1) / kPrefixBlocks));
  }
  // Own positions: a workgroup for every place, if all sequences fill their tables.
  const uint64_t capacity = (static_cast<uint64_t>(p.stride) << p.page_shift) - shared;
  s.own_splits = static_cast<uint32_t>(std::clamp<uint64_t>(capacity / (kBlock * kOwnBlocks), 1,
                                                            splits(kComputeUnits * resident(head_size), s.own_tiles, kv_heads * count)));
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
    const hipStream_t st = static_cast<hipStream_t>(stream);
    const uint32_t all = static_cast<uint32_t>(groups);
    const dim3 block(kWaves * 64);
    if (head_size == 128) hipLaunchKernelGGL(paged_attention_kernel<128>, dim3(all), block, 0, st, a);
    else hipLaunchKernelGGL(paged_attention_kernel<256>, dim3(all), block, 0, st, a);
    if (const int32_t s = launch_status("paged attention launch failed"); s != GFXI_OK) return s;
    const dim3 combine(static_cast<unsigned>((shape.rows * (head_size / 128) + 3) / 4));
    if (head_size == 128) hipLaunchKernelGGL(paged_combine_kernel<128>, combine, dim3(256), 0, st, a);
    else hipLaunchKernelGGL(paged_combine_kernel<256>, combine, dim3(256), 0, st, a);
    return launch_status("paged attention combine launch failed");
  });
}
