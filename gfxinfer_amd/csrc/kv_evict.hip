// A K/V cache within a budget: what each cached row has been worth, and the eviction of the
// rows that were worth least.
//
// Attention does not depend on the order of a sequence's committed rows, so nothing is shifted:
// the kept rows past the budget move into the holes that dropped rows leave before it, at most
// as many rows as are dropped.  Sources lie past the budget and targets before it, so the
// moves of a call are independent.  The rows' positions in the text move beside them.
//
// Three launches: a workgroup per sequence chooses (select_kernel), one workgroup gives out
// pages for private copies (grant_kernel), and a grid that fills the GPU moves rows and
// commits (move_kernel).
//
// Few sequences in small tables are chosen and granted by one workgroup (select_grant_kernel).
//
// Four sequences that lose a row each take 10.8 + 4.5 us, chains of dependent steps in one workgroup;
// eight that lose 512 rows of 16 layers 9.8 + 5.2 + 98 us, the moves' 418 MB at 4.3 TB/s.
#include <algorithm>
#include <string>
#include <type_traits>

#include "kv_weights.hpp"

namespace gfx950 {
namespace {

using u32x4 = unsigned __attribute__((ext_vector_type(4)));

constexpr unsigned kGrantThreads = 1024;

// The workspace: a header per sequence, then its moves and its copies, then the bits of kept
// rows.  All offsets by the host's sizes alone.
struct EvictHeader {
  uint32_t moves;    // rows to move (0: the sequence stays as it is)
  uint32_t copies;   // pages to copy
  uint32_t length;   // before; 0: nothing to do
  uint32_t failed;   // of the first header: the call fails
};
struct RowMove {
  int32_t page;          // of the source, -1: none
  uint32_t row, target;  // row in its page; the target's row of the sequence
  uint32_t source;       // row of the sequence
};
struct PageCopy {
  uint32_t column;
  int32_t from, to;
  uint32_t unused;
};

struct EvictArgs {
  KvPages pages;
  KvWeights weights;
  SequenceList list;
  EvictHeader* headers;   // [count]
  RowMove* moves;         // [count][most_moves]
  PageCopy* copies;       // [count][most_copies]
  uint32_t* kept;         // [count][kept_words]: bit r % 32 of word r / 32, rows before the budget
  uint32_t most_moves, most_copies, kept_words;
  uint32_t budget, first, recent;
  int32_t* status;
};

__host__ __device__ __forceinline__ uint32_t capacity_of(const KvPages& p) { return p.stride << p.page_shift; }

// Order of weights as unsigned numbers; NaN above all, the zeros equal.
__device__ __forceinline__ uint32_t order_of(float w) {
  if (w != w) return 0xffffffffu;
  const uint32_t u = __float_as_uint(w + 0.0F);
  return (u & 0x80000000u) != 0 ? ~u : u | 0x80000000u;
}

// Sum over the lanes up to this one: within rows of 16, then the rows before (no trips through LDS).
__device__ __forceinline__ uint32_t scan_lanes(uint32_t v) {
  auto from = [](uint32_t x, auto control, auto rows) __attribute__((always_inline)) {
    return static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(x), control.value, rows.value, 0xf, false));
  };
  using Shift1 = std::integral_constant<int, 0x111>;
  using Shift2 = std::integral_constant<int, 0x112>;
  using Shift4 = std::integral_constant<int, 0x114>;
  using Shift8 = std::integral_constant<int, 0x118>;
  using Last15 = std::integral_constant<int, 0x142>;  // a row's last lane to the next row
  using Last31 = std::integral_constant<int, 0x143>;  // lane 31 to the upper rows
  using All = std::integral_constant<int, 0xf>;
  v += from(v, Shift1{}, All{});
  v += from(v, Shift2{}, All{});
  v += from(v, Shift4{}, All{});
  v += from(v, Shift8{}, All{});
  v += from(v, Last15{}, std::integral_constant<int, 0xa>{});
  v += from(v, Last31{}, std::integral_constant<int, 0xc>{});
  return v;
}

// Of the threads of so many waves; with several such groups in a workgroup each has its own partial sums.
template <unsigned Waves>
__device__ __forceinline__ uint32_t scan_waves(uint32_t v, uint32_t* partial, uint32_t& total) {
  const unsigned lane = threadIdx.x & 63u, wave = (threadIdx.x >> 6) % Waves;
  const uint32_t sum = scan_lanes(v);
  if (lane == 63u) partial[wave] = sum;
  __syncthreads();
  uint32_t before = 0;
  total = 0;
#pragma unroll
  for (unsigned w = 0; w < Waves; ++w) {
    const uint32_t part = partial[w];
    if (w < wave) before += part;
    total += part;
  }
  __syncthreads();
  return before + sum - v;
}

constexpr unsigned kSelectKeys = 4;  // of a thread
constexpr unsigned kSmallThreads = 256;
constexpr unsigned kSmallSequences = kGrantThreads / kSmallThreads;

// Numbers of the lanes' flags among those of a block of rows, of keys e * threads + thread in this order: the
// flags before a lane's own.  counts has room for each wave's of each key; one barrier.
template <unsigned Waves>
__device__ __forceinline__ void rank_flags(const bool (&flag)[kSelectKeys], uint32_t* counts, uint32_t (&rank)[kSelectKeys], uint32_t& total) {
  static_assert(kSelectKeys * Waves <= 64);
  const unsigned lane = threadIdx.x & 63u, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) % Waves;
#pragma unroll
  for (unsigned e = 0; e < kSelectKeys; ++e) {
    const uint64_t bits = __ballot(flag[e]);
    rank[e] = static_cast<uint32_t>(__popcll(bits & ((1ull << lane) - 1)));
    if (lane == 0) counts[e * Waves + wave] = static_cast<uint32_t>(__popcll(bits));
  }
  __syncthreads();
  const uint32_t mine = lane < kSelectKeys * Waves ? counts[lane] : 0;
  const uint32_t upto = scan_lanes(mine);
#pragma unroll
  for (unsigned e = 0; e < kSelectKeys; ++e) rank[e] += __builtin_amdgcn_readlane(upto - mine, e * Waves + wave);
  total = __builtin_amdgcn_readlane(upto, 63);
}

// Chooses the rows of one sequence: the number of rows that stay for their position, then the
// key of the last row that fits (a radix select over 8 bits a pass, largest first, until a digit's
// rows all stay), then in row order which rows stay, and the lists of holes and movers.  Up to four rows a thread lie in
// registers all the while; each pass has one barrier, its own counts and every wave looks for the digit.
//
// A group of threads a sequence; several groups of a workgroup go through the same barriers, those
// without a sequence or with nothing to drop among them (Groups: then four rows a thread are all).
constexpr unsigned kCopies = 4;  // of the counts, one for every fourth wave: the first digits of many weights are the same
template <unsigned Threads>
struct SelectShared {
  uint32_t histogram[4][kCopies][256];
  uint32_t partial[Threads / 64];
  uint32_t counts[3][64];
};

template <unsigned Threads, bool Groups>
__device__ __forceinline__ void select_rows(const EvictArgs& a, uint32_t listed, SelectShared<Threads>& lds, uint32_t (*open)[kSmallSequences]) {
  constexpr unsigned kWaves = Threads / 64;
  constexpr uint32_t kRows = Threads * kSelectKeys;
  const unsigned tid = threadIdx.x % Threads, lane = tid & 63u, wave = tid >> 6;
  auto& histogram = lds.histogram;
  auto& partial = lds.partial;
  auto& counts = lds.counts;
  const KvPages& pg = a.pages;
  const uint32_t i = Groups ? min(listed, a.list.count - 1) : listed, slot = listed_slot(a.list, i);
  const uint32_t capacity = capacity_of(pg), length = min(pg.lengths[slot], capacity), dropped = a.weights.dropped[slot];
  const std::size_t base = static_cast<std::size_t>(slot) * capacity;
  const float* weight = a.weights.weight + base;
  const int32_t* position = a.weights.position + base;
  float w[kSelectKeys];
  int32_t p[kSelectKeys];
  auto fetch = [&](uint32_t from) __attribute__((always_inline)) {
#pragma unroll
    for (unsigned e = 0; e < kSelectKeys; ++e) {
      const uint32_t row = min(from + e * Threads + tid, capacity - 1);
      w[e] = weight[row];
      p[e] = position[row];
    }
  };
  // All that the choice reads is asked for before the length is there.
  fetch(0);
  // (A budget may be any number: no more columns than the table's are gone through.)
  const uint32_t columns = min(pages_for(a.budget, pg.page_shift), pg.stride), page_tokens = 1u << pg.page_shift;
  const int32_t first_page = tid < columns ? table_page(pg, slot, tid) : -1;
  const uint32_t first_holders = first_page >= 0 ? pg.references[first_page] : 0;
  const bool over = length > a.budget && i == listed;
  if (!over) {
    if (tid == 0 && i == listed) a.headers[i] = EvictHeader{0, 0, 0, 0};
    if constexpr (!Groups) return;
  }
  const uint32_t n = over ? length : 0;
  const int64_t last = static_cast<int64_t>(n) + dropped - a.recent;  // positions from here on stay
  uint32_t key[kSelectKeys] = {};
  bool fixed[kSelectKeys] = {}, there[kSelectKeys] = {};
  auto take = [&](uint32_t from) __attribute__((always_inline)) {
#pragma unroll
    for (unsigned e = 0; e < kSelectKeys; ++e) {
      there[e] = from + e * Threads + tid < n;
      key[e] = order_of(w[e]);
      fixed[e] = there[e] && (p[e] < static_cast<int64_t>(a.first) || p[e] >= last);
    }
  };
  auto load = [&](uint32_t from) __attribute__((always_inline)) {
    fetch(from);
    take(from);
  };
  if constexpr (Threads == kSmallThreads) __builtin_assume(n <= kRows);  // the table holds no more
  const bool resident = n <= kRows;
  for (uint32_t x = tid; x < 4 * kCopies * 256; x += Threads) (&histogram[0][0][0])[x] = 0;
  uint32_t mine = 0;
#pragma unroll 1
  for (uint32_t from = 0; from < n; from += kRows) {
    if (from != 0) fetch(from);
    take(from);
#pragma unroll
    for (unsigned e = 0; e < kSelectKeys; ++e) mine += fixed[e] ? 1u : 0u;
  }
  uint32_t protected_rows;
  scan_waves<kWaves>(mine, partial, protected_rows);
  // At most first + recent <= budget where positions are distinct, as begin makes them.
  const bool crowded = protected_rows > a.budget;  // damaged positions: then none is protected
  uint32_t wanted = crowded ? a.budget : a.budget - protected_rows, prefix = 0, high = 0;
  const bool none = wanted == 0;
  bool exact = none || !over;  // all rows of this prefix stay, later digits do not matter
#pragma unroll 1
  for (int shift = 24; shift >= 0 && (Groups || !exact); shift -= 8) {
    uint32_t (&own)[256] = histogram[shift / 8][wave % kCopies];
#pragma unroll 1
    for (uint32_t from = 0; from < n; from += kRows) {
      if (!resident) load(from);
#pragma unroll
      for (unsigned e = 0; e < kSelectKeys; ++e) {
        if ((!Groups || !exact) && there[e] && (key[e] & high) == prefix && (crowded || !fixed[e])) atomicAdd(&own[key[e] >> shift & 255u], 1u);
      }
    }
    if (Groups && tid == 0) open[shift / 8][listed] = exact ? 0 : 1;
    __syncthreads();
    if constexpr (Groups) {
      uint32_t any = 0;
#pragma unroll
      for (unsigned g = 0; g < kSmallSequences; ++g) any |= open[shift / 8][g];
      if (__builtin_amdgcn_readfirstlane(any) == 0) break;
      if (exact) continue;
    }
    // The digit in which the wanted-th largest lies: sums from the top, four digits a lane.
    uint32_t four[4] = {}, sum = 0;
#pragma unroll
    for (unsigned c = 0; c < kCopies; ++c) {
      const u32x4 x = *reinterpret_cast<const u32x4*>(&histogram[shift / 8][c][252u - 4 * lane]);
#pragma unroll
      for (unsigned e = 0; e < 4; ++e) four[e] += x[3 - e];
    }
#pragma unroll
    for (unsigned e = 0; e < 4; ++e) sum += four[e];
    const uint32_t upto = scan_lanes(sum);
    uint32_t before = upto - sum, digit = 0, rest = 0;
    bool found = false, all = false;
#pragma unroll
    for (unsigned e = 0; e < 4; ++e) {
      if (before < wanted && wanted <= before + four[e]) {
        found = true;
        digit = 255u - (4 * lane + e);
        rest = wanted - before;
        all = rest == four[e];
      }
      before += four[e];
    }
    // (One lane finds it: there are more rows than wanted.)
    const int at = __ffsll(static_cast<unsigned long long>(__ballot(found))) - 1;
    prefix |= static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(digit), at)) << shift;
    wanted = static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(rest), at));
    exact = __builtin_amdgcn_readlane(all ? 1 : 0, at) != 0;
    high |= 255u << shift;
  }
  // Rows above the prefix stay, and the first `wanted` of those at it.
  uint32_t* kept_bits = a.kept + static_cast<std::size_t>(i) * a.kept_words;
  RowMove* moves = a.moves + static_cast<std::size_t>(i) * a.most_moves;
  uint32_t ties = 0, holes = 0, movers = 0;
#pragma unroll 1
  for (uint32_t from = 0; from < (Groups ? 1 : n); from += kRows) {
    if (!resident) load(from);
    bool stays[kSelectKeys], tie[kSelectKeys];
#pragma unroll
    for (unsigned e = 0; e < kSelectKeys; ++e) {
      const bool stands = there[e] && !crowded && fixed[e];
      stays[e] = stands || (there[e] && !none && (key[e] & high) > prefix);
      tie[e] = there[e] && !stands && !none && (key[e] & high) == prefix;
    }
    uint32_t rank[kSelectKeys], total;
    rank_flags<kWaves>(tie, counts[0], rank, total);
    bool hole[kSelectKeys], mover[kSelectKeys];
#pragma unroll
    for (unsigned e = 0; e < kSelectKeys; ++e) {
      const uint32_t first = from + e * Threads + 64 * wave, row = first + lane;  // 32 | first
      stays[e] |= tie[e] && ties + rank[e] < wanted;
      hole[e] = over && row < a.budget && !stays[e];
      mover[e] = row >= a.budget && stays[e];
      const uint64_t bits = __ballot(stays[e] && row < a.budget);
      if (over && lane == 0 && first / 32 < a.kept_words) kept_bits[first / 32] = static_cast<uint32_t>(bits);
      if (over && lane == 32 && first / 32 + 1 < a.kept_words) kept_bits[first / 32 + 1] = static_cast<uint32_t>(bits >> 32);
    }
    ties += total;
    rank_flags<kWaves>(hole, counts[1], rank, total);
#pragma unroll
    for (unsigned e = 0; e < kSelectKeys; ++e) {
      if (hole[e] && holes + rank[e] < a.most_moves) moves[holes + rank[e]].target = from + e * Threads + tid;
    }
    holes += total;
    rank_flags<kWaves>(mover, counts[2], rank, total);
#pragma unroll
    for (unsigned e = 0; e < kSelectKeys; ++e) {
      const uint32_t row = from + e * Threads + tid;
      if (mover[e] && movers + rank[e] < a.most_moves) {
        RowMove& move = moves[movers + rank[e]];
        move.page = table_page(pg, slot, row >> pg.page_shift);
        move.row = row & ((1u << pg.page_shift) - 1);
        move.source = row;
      }
    }
    movers += total;
  }
  __threadfence_block();
  __syncthreads();
  // Pages with a hole that other sequences hold too.
  PageCopy* copies = a.copies + static_cast<std::size_t>(i) * a.most_copies;
  uint32_t found = 0;
#pragma unroll 1
  for (uint32_t from = 0; from < columns; from += Threads) {
    const uint32_t column = from + tid;
    int32_t page = -1;
    bool copy = false;
    if (over && column < columns) {
      page = from == 0 ? first_page : table_page(pg, slot, column);
      if (page >= 0 && (from == 0 ? first_holders : pg.references[page]) > 1) {
        // A row of the page before the budget whose bit is off.
        const uint32_t begin = column << pg.page_shift, end = min(begin + page_tokens, a.budget);
        for (uint32_t r = begin; r < end; r += 32) {  // begin is a multiple of 16
          const uint32_t word = kept_bits[r / 32], low = r % 32, count = min(end - r, 32u - low);
          const uint32_t wanted_bits = (count == 32 ? 0xffffffffu : (1u << count) - 1u) << low;
          copy |= (word & wanted_bits) != wanted_bits;
          if (low != 0) r -= low;
        }
      }
    }
    uint32_t total;
    const uint32_t at = found + scan_waves<kWaves>(copy ? 1u : 0u, partial, total);
    if (copy) copies[at] = PageCopy{column, page, -1, 0};
    found += total;
  }
  if (tid == 0 && over) a.headers[i] = EvictHeader{min(holes, movers), found, n, 0};
}

template <unsigned Threads>
__global__ __launch_bounds__(Threads) void select_kernel(EvictArgs a) {
  __shared__ SelectShared<Threads> lds;
  select_rows<Threads, false>(a, blockIdx.x, lds, nullptr);
}

// One workgroup gives every copy a free page, lowest first, sequence by sequence, or fails the
// call as a whole (false); then it renames the pages.
struct GrantShared {
  uint32_t partial[kGrantThreads / 64];
  uint32_t start[kMaxListed + 1];
};
__device__ __forceinline__ bool grant_pages(const EvictArgs& a, GrantShared& lds) {
  auto& partial = lds.partial;
  auto& start = lds.start;
  const unsigned tid = threadIdx.x;
  const KvPages& pg = a.pages;
  uint32_t total;
  const uint32_t before = scan_waves<kGrantThreads / 64>(tid < a.list.count ? a.headers[tid].copies : 0u, partial, total);
  if (tid < a.list.count) start[tid] = before;
  if (tid == 0) start[a.list.count] = total;
  __syncthreads();
  if (total == 0) {
    if (tid == 0) *a.status = 0;
    return true;
  }
  // Twice over the counts: is there enough, then who gets what.
  uint32_t available = 0;
  for (uint32_t from = 0; from < pg.page_count && available < total; from += kGrantThreads) {
    uint32_t found;
    scan_waves<kGrantThreads / 64>(from + tid < pg.page_count && pg.references[from + tid] == 0 ? 1u : 0u, partial, found);
    available += found;
  }
  if (tid == 0) {
    *a.status = available < total ? 1 : 0;
    if (available < total) a.headers[0].failed = 1;
  }
  if (available < total) return false;
  uint32_t given = 0;
  for (uint32_t from = 0; from < pg.page_count && given < total; from += kGrantThreads) {
    const uint32_t page = from + tid;
    const bool free = page < pg.page_count && pg.references[page] == 0;
    uint32_t found;
    const uint32_t rank = given + scan_waves<kGrantThreads / 64>(free ? 1u : 0u, partial, found);
    if (free && rank < total) {
      uint32_t low = 0, high = a.list.count;  // the last sequence whose start is <= rank
      while (high - low > 1) {
        const uint32_t mid = (low + high) / 2;
        if (start[mid] <= rank) low = mid;
        else high = mid;
      }
      PageCopy& copy = a.copies[static_cast<std::size_t>(low) * a.most_copies + rank - start[low]];
      copy.to = static_cast<int32_t>(page);
      pg.references[page] = 1;
      pg.table[static_cast<std::size_t>(listed_slot(a.list, low)) * pg.stride + copy.column] = static_cast<int32_t>(page);
    }
    given += found;
  }
  // The holders' shares of the old pages, once no page is looked for any more: one that all of
  // them leave is free for the next call, not for this one.
  __syncthreads();
  for (uint32_t i = 0; i < a.list.count; ++i) {
    for (uint32_t c = tid; c < start[i + 1] - start[i]; c += kGrantThreads) {
      atomicSub(&pg.references[a.copies[static_cast<std::size_t>(i) * a.most_copies + c].from], 1u);
    }
  }
  return true;
}

__global__ __launch_bounds__(kGrantThreads) void grant_kernel(EvictArgs a) {
  __shared__ GrantShared lds;
  grant_pages(a, lds);
}

// Both for up to four sequences whose tables hold at most 1024 rows, a launch less, which is the host's time: four
// sequences, a row each, with all calls of the step take 32.7 us, not 36.4.  On the GPU it is the slower one, 10.7 us for 6.8 and
// 2.0: replayed from a graph the step takes 27.2 us, not 25.9.

__global__ __launch_bounds__(kGrantThreads) void select_grant_kernel(EvictArgs a) {
  __shared__ SelectShared<kSmallThreads> chosen[kSmallSequences];
  __shared__ GrantShared granted;
  __shared__ uint32_t open[4][kSmallSequences];  // whether a pass has anything to do for a group
  const unsigned group = threadIdx.x / kSmallThreads;
  select_rows<kSmallThreads, true>(a, group, chosen[group], open);
  __threadfence_block();
  __syncthreads();
  grant_pages(a, granted);
}

constexpr unsigned kMoveThreads = 256, kMoveWorkgroups = 2048;

// Moves rows of all layers, K and V, a wave a row and plane at a time; then commits.  Sources
// were looked up before pages were renamed, targets are looked up now.
__global__ __launch_bounds__(kMoveThreads) void move_kernel(EvictArgs a) {
  const KvPages& pg = a.pages;
  if (a.headers[0].failed != 0) return;
  const uint32_t s = blockIdx.y, slot = listed_slot(a.list, s);
  const EvictHeader header = a.headers[s];
  if (header.length == 0) return;
  const unsigned lane = threadIdx.x & 63u;
  const uint32_t wave = __builtin_amdgcn_readfirstlane(blockIdx.x * (kMoveThreads / 64) + (threadIdx.x >> 6));
  const uint32_t waves = gridDim.x * (kMoveThreads / 64);
  const uint32_t page_tokens = 1u << pg.page_shift, units = pg.row / 8, planes = 2 * pg.layers;
  const RowMove* moves = a.moves + static_cast<std::size_t>(s) * a.most_moves;
  const PageCopy* copies = a.copies + static_cast<std::size_t>(s) * a.most_copies;
  const uint32_t* kept = a.kept + static_cast<std::size_t>(s) * a.kept_words;
  const uint64_t rows = header.moves + static_cast<uint64_t>(header.copies) * page_tokens;
  auto copy_row = [&](uint32_t plane, int32_t from, uint32_t from_row, int32_t to, uint32_t to_row) __attribute__((always_inline)) {
    u32x4* pool = reinterpret_cast<u32x4*>(plane < pg.layers ? pg.key : pg.value);
    const std::size_t layer = static_cast<std::size_t>(plane < pg.layers ? plane : plane - pg.layers) * pg.page_count;
    const u32x4* source = pool + (((layer + from) << pg.page_shift) + from_row) * units;
    u32x4* target = pool + (((layer + to) << pg.page_shift) + to_row) * units;
    for (uint32_t u = lane; u < units; u += 64) target[u] = source[u];
  };
  for (uint64_t item = wave; item < rows * planes; item += waves) {
    const uint32_t plane = static_cast<uint32_t>(item % planes);
    const uint64_t row = item / planes;
    if (row < header.moves) {
      const RowMove m = moves[row];
      const int32_t to = table_page(pg, slot, m.target >> pg.page_shift);
      if (m.page >= 0 && to >= 0) copy_row(plane, m.page, m.row, to, m.target & (page_tokens - 1));
    } else {
      const uint32_t at = static_cast<uint32_t>(row - header.moves);
      const PageCopy c = copies[at >> pg.page_shift];
      const uint32_t r = at & (page_tokens - 1), j = (c.column << pg.page_shift) + r;
      if (j < a.budget && (kept[j / 32] >> j % 32 & 1u) != 0) copy_row(plane, c.from, r, c.to, r);
    }
  }
  // The commit: no part of this launch reads what it writes.
  const uint32_t thread = blockIdx.x * kMoveThreads + threadIdx.x, threads = gridDim.x * kMoveThreads;
  const std::size_t base = static_cast<std::size_t>(slot) * capacity_of(pg);
  for (uint32_t m = thread; m < header.moves; m += threads) {
    const RowMove move = moves[m];
    a.weights.weight[base + move.target] = a.weights.weight[base + move.source];
    a.weights.position[base + move.target] = a.weights.position[base + move.source];
  }
  for (uint32_t column = pages_for(a.budget, pg.page_shift) + thread; column < pg.stride; column += threads) {
    const int32_t page = table_page(pg, slot, column);
    if (page >= 0) atomicSub(&pg.references[page], 1u);
    pg.table[static_cast<std::size_t>(slot) * pg.stride + column] = -1;
  }
  if (thread == 0) {
    a.weights.dropped[slot] += header.length - a.budget;
    pg.lengths[slot] = a.budget;
  }
}

__global__ __launch_bounds__(256) void begin_kernel(KvPages p, KvWeights w, ChunkList list) {
  const uint32_t i = blockIdx.y, slot = listed_slot(list, i), tokens = list.first[i + 1] - list.first[i];
  const uint32_t t = blockIdx.x * 256 + threadIdx.x, capacity = capacity_of(p), length = min(p.lengths[slot], capacity);
  // Every workgroup of an empty sequence takes 0, whether the first one has written it or not.
  const uint32_t dropped = length == 0 ? 0u : w.dropped[slot];
  if (t == 0 && length == 0) w.dropped[slot] = 0;
  if (t >= tokens || t >= capacity - length) return;
  const std::size_t at = static_cast<std::size_t>(slot) * capacity + length + t;
  w.weight[at] = 0.0F;
  w.position[at] = static_cast<int32_t>(length + t + dropped);
}

// Most rows that a sequence can lose and move, pages it can copy, and words of its bits.
struct EvictSizes {
  std::size_t moves, copies, words, bytes;
};
EvictSizes evict_sizes(const KvPages& p, uint32_t count, uint32_t budget) {
  const uint64_t capacity = static_cast<uint64_t>(p.stride) << p.page_shift;
  EvictSizes s{};
  s.moves = budget < capacity ? std::min<uint64_t>(budget, capacity - budget) : 0;
  s.copies = std::min<uint64_t>(p.stride, (budget + (1ull << p.page_shift) - 1) >> p.page_shift);
  s.words = (std::min<uint64_t>(budget, capacity) + 127) / 128 * 4;
  s.bytes = count * (sizeof(EvictHeader) + s.moves * sizeof(RowMove) + s.copies * sizeof(PageCopy) + s.words * 4);
  return s;
}

}  // namespace

int32_t read_chunks(const KvPages& pages, const uint32_t* sequences, const uint32_t* tokens, uint32_t count, bool distinct,
                    ChunkList& out) {
  if (tokens == nullptr || count == 0 || count > kMaxChunks || (sequences == nullptr && count > pages.sequences)) {
    return fail(GFXI_INVALID_ARGUMENT, "a chunk call names 1.." + std::to_string(kMaxChunks) + " sequences of the cache and their tokens");
  }
  SequenceList list;
  if (const int32_t s = read_sequences(pages, sequences, count, distinct, list); s != GFXI_OK) return s;
  out = ChunkList{};
  out.count = count;
  uint64_t rows = 0;
  for (uint32_t i = 0; i < count; ++i) {
    out.slot[i] = list.slot[i];
    out.first[i] = static_cast<uint32_t>(rows);
    rows += tokens[i];
    if (rows > kMaxRows) return fail(GFXI_INVALID_ARGUMENT, "a chunk call has at most 2^20 rows");
  }
  if (rows == 0) return fail(GFXI_INVALID_ARGUMENT, "a chunk call has at least one token");
  for (uint32_t i = count; i <= kMaxChunks; ++i) out.first[i] = static_cast<uint32_t>(rows);
  return GFXI_OK;
}

int32_t read_weights(const gfxinfer_kv_weights* weights, KvWeights& out) {
  if (weights == nullptr || weights->weight == nullptr || weights->position == nullptr || weights->dropped == nullptr) {
    return fail(GFXI_INVALID_ARGUMENT, "K/V weights: weight, position and dropped must be set");
  }
  out = KvWeights{weights->weight, weights->position, weights->dropped};
  return GFXI_OK;
}

}  // namespace gfx950

using namespace gfx950;

extern "C" int32_t gfxinfer_launch_kv_weights_begin(const gfxinfer_kv_pages* pages, const gfxinfer_kv_weights* weights,
                                                    const uint32_t* sequences, const uint32_t* tokens, uint32_t count,
                                                    void* stream) {
  return guarded([&] {
    KvPages p;
    KvWeights w;
    ChunkList list;
    if (const int32_t s = read_pages(pages, p); s != GFXI_OK) return s;
    if (const int32_t s = read_weights(weights, w); s != GFXI_OK) return s;
    if (const int32_t s = read_chunks(p, sequences, tokens, count, true, list); s != GFXI_OK) return s;
    const uint32_t most = *std::max_element(tokens, tokens + count);
    hipLaunchKernelGGL(begin_kernel, dim3((most + 255) / 256, count), dim3(256), 0, static_cast<hipStream_t>(stream), p, w, list);
    return launch_status("K/V weights launch failed");
  });
}

extern "C" size_t gfxinfer_kv_pages_evict_workspace_bytes(const gfxinfer_kv_pages* pages, uint32_t count, uint32_t budget) {
  size_t bytes = 0;
  guarded([&] {
    KvPages p;
    const int32_t s = read_pages(pages, p);
    if (s == GFXI_OK && count != 0 && count <= kMaxListed && budget != 0) bytes = evict_sizes(p, count, budget).bytes;
    return s;
  });
  return bytes;
}

extern "C" int32_t gfxinfer_launch_kv_pages_evict(const gfxinfer_kv_pages* pages, const gfxinfer_kv_weights* weights,
                                                  const uint32_t* sequences, uint32_t count, uint32_t budget, uint32_t first,
                                                  uint32_t recent, int32_t* status, void* workspace, size_t workspace_bytes,
                                                  void* stream) {
  return guarded([&] {
    EvictArgs a{};
    if (const int32_t s = read_pages(pages, a.pages); s != GFXI_OK) return s;
    if (const int32_t s = read_weights(weights, a.weights); s != GFXI_OK) return s;
    if (const int32_t s = read_sequences(a.pages, sequences, count, true, a.list); s != GFXI_OK) return s;
    if (budget == 0 || static_cast<uint64_t>(first) + recent > budget || status == nullptr) {
      return fail(GFXI_INVALID_ARGUMENT, "eviction needs a budget of at least first + recent rows and 1, and a status word");
    }
    const EvictSizes sizes = evict_sizes(a.pages, count, budget);
    if (workspace == nullptr || !aligned16(workspace) || workspace_bytes < sizes.bytes) {
      return fail(GFXI_INVALID_ARGUMENT, "eviction workspace is null, not 16-byte aligned or too small");
    }
    a.headers = static_cast<EvictHeader*>(workspace);
    a.moves = reinterpret_cast<RowMove*>(a.headers + count);
    a.copies = reinterpret_cast<PageCopy*>(a.moves + count * sizes.moves);
    a.kept = reinterpret_cast<uint32_t*>(a.copies + count * sizes.copies);
    a.most_moves = static_cast<uint32_t>(sizes.moves);
    a.most_copies = static_cast<uint32_t>(sizes.copies);
    a.kept_words = static_cast<uint32_t>(sizes.words);
    a.budget = budget;
    a.first = first;
    a.recent = recent;
    a.status = status;
    const hipStream_t st = static_cast<hipStream_t>(stream);
    // A wave's instructions are what the choice takes its time with, and sixteen waves share a CU's four vector
    // units: tables of few rows take four (501 rows: three quarters of the time with sixteen).
    const bool small = capacity_of(a.pages) <= kSmallThreads * kSelectKeys;
    if (small && count <= kSmallSequences) {
      hipLaunchKernelGGL(select_grant_kernel, dim3(1), dim3(kGrantThreads), 0, st, a);
    } else {
      if (small) hipLaunchKernelGGL(select_kernel<kSmallThreads>, dim3(count), dim3(kSmallThreads), 0, st, a);
      else hipLaunchKernelGGL(select_kernel<1024>, dim3(count), dim3(1024), 0, st, a);
      if (const int32_t s = launch_status("K/V eviction launch failed"); s != GFXI_OK) return s;
      hipLaunchKernelGGL(grant_kernel, dim3(1), dim3(kGrantThreads), 0, st, a);
    }
    if (const int32_t s = launch_status("K/V eviction launch failed"); s != GFXI_OK) return s;
    hipLaunchKernelGGL(move_kernel, dim3(std::max(1u, kMoveWorkgroups / count), count), dim3(kMoveThreads), 0, st, a);
    return launch_status("K/V eviction launch failed");
  });
}
