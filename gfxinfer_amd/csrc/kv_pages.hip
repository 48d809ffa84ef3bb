// Pages of a K/V cache for sequences that share prefixes: fork, reserve (allocation and
// the private copy of a shared tail page), append, advance, free, copy and compact.
//
// The state is three small integer arrays beside the two pools: a table of pages per
// sequence, the committed tokens of each sequence, and how many table entries name each
// page.  A page is free exactly when its count is zero, so there is no free list that
// could disagree with the tables.  Allocation always takes the lowest free pages in a
// fixed order and every count changes by integer atomics, so the state after a call
// does not depend on how its workgroups were scheduled.
//
// The launchers know the sequences they are asked about (host lists) but not their
// lengths (device), so a whole decode step can be recorded into a graph.
#include <algorithm>
#include <string>

#include "kv_pages.hpp"

namespace gfx950 {
namespace {

using u32x4 = unsigned __attribute__((ext_vector_type(4)));
using f32x4 = float __attribute__((ext_vector_type(4)));
using h16x8 = _Float16 __attribute__((ext_vector_type(8)));

// One page copy of a plan: the first `rows` token rows of page `from`, all layers, K and V.
struct Move {
  uint32_t from, to, rows, unused;
};
// A plan in the workspace: the header, then the moves, then (compact) the page map.
struct Plan {
  uint32_t moves;
  uint32_t live;
  uint32_t unused[2];
  Move move[1];
};
std::size_t plan_moves(uint32_t page_count) { return std::max<std::size_t>(kMaxListed, (page_count + 1u) / 2u); }
std::size_t plan_bytes(uint32_t page_count) {
  return 16 + sizeof(Move) * plan_moves(page_count) + sizeof(uint32_t) * static_cast<std::size_t>(page_count);
}
__host__ __device__ inline uint32_t* plan_map(Plan* plan, std::size_t moves) {
  return reinterpret_cast<uint32_t*>(reinterpret_cast<char*>(plan) + 16 + sizeof(Move) * moves);
}

constexpr unsigned kPlanThreads = 1024;
constexpr unsigned kPagesPerThread = 32;  // one bit mask
constexpr unsigned kPagesPerRound = kPlanThreads * kPagesPerThread;

// Exclusive sum over the workgroup in thread order; `total` in every thread.  partial
// holds one word per wave; the call ends with a barrier, so it can be used again.
__device__ __forceinline__ uint32_t block_scan(uint32_t v, uint32_t* partial, uint32_t& total) {
  const unsigned lane = threadIdx.x & 63u, wave = threadIdx.x >> 6;
  uint32_t sum = v;
#pragma unroll
  for (unsigned d = 1; d < 64; d <<= 1) {
    const uint32_t o = __shfl_up(sum, d);
    if (lane >= d) sum += o;
  }
  if (lane == 63u) partial[wave] = sum;
  __syncthreads();
  uint32_t before = 0;
  total = 0;
#pragma unroll
  for (unsigned w = 0; w < kPlanThreads / 64; ++w) {
    const uint32_t part = partial[w];
    if (w < wave) before += part;
    total += part;
  }
  __syncthreads();
  return before + sum - v;
}

// Bit i set: page first + i has references (pages past the pool count as used).
__device__ __forceinline__ uint32_t used_mask(const KvPages& p, uint32_t first) {
  uint32_t mask = 0;
  if (first + kPagesPerThread <= p.page_count) {
    u32x4 v[kPagesPerThread / 4];
#pragma unroll
    for (unsigned i = 0; i < kPagesPerThread / 4; ++i) {
      v[i] = *reinterpret_cast<const u32x4*>(p.references + first + 4 * i);
    }
#pragma unroll
    for (unsigned i = 0; i < kPagesPerThread; ++i) mask |= (v[i / 4][i % 4] != 0u ? 1u : 0u) << i;
  } else if (first < p.page_count) {
    uint32_t v[kPagesPerThread];
#pragma unroll
    for (unsigned i = 0; i < kPagesPerThread; ++i) v[i] = p.references[min(first + i, p.page_count - 1)];
#pragma unroll
    for (unsigned i = 0; i < kPagesPerThread; ++i) mask |= (first + i >= p.page_count || v[i] != 0u ? 1u : 0u) << i;
  } else {
    mask = 0xffffffffu;
  }
  return mask;
}

// One workgroup plans a reserve: how many pages each sequence lacks, whether its partly
// filled tail page is shared, which free pages it gets (sequence by sequence in list
// order, a tail copy before new pages, lowest free pages first), and the copies to do.
// All sequences get their pages or none does.  Bound by its chain of look-ups and scans, not
// by bytes: 7.6 us for 3 sequences, 12 us for 63.
__global__ __launch_bounds__(kPlanThreads) void reserve_kernel(KvPages p, SequenceList list, uint32_t tokens,
                                                               int32_t* __restrict__ status, Plan* plan) {
  __shared__ uint32_t length[kMaxListed], tail[kMaxListed], first[kMaxListed], need[kMaxListed], have[kMaxListed];
  __shared__ uint32_t offset[kMaxListed], copy_rank[kMaxListed];
  __shared__ uint32_t partial[kPlanThreads / 64];
  __shared__ uint32_t taken[kPlanThreads];  // pages of one window of ranks
  __shared__ uint32_t bad;
  const unsigned tid = threadIdx.x;
  constexpr uint32_t kNone = 0xffffffffu;
  // The first round's counts are on their way while the sequences are looked up.
  uint32_t mask = used_mask(p, tid * kPagesPerThread);
  if (tid == 0) bad = 0;
  __syncthreads();
  const bool mine = tid < list.count;
  const uint32_t page_tokens = 1u << p.page_shift;
  if (mine) {
    const uint32_t slot = list.slot[tid], len = p.lengths[slot];
    const uint64_t end = static_cast<uint64_t>(len) + tokens;
    const bool fits = end <= static_cast<uint64_t>(p.stride) << p.page_shift;
    if (!fits) bad = 1;
    length[tid] = len;
    first[tid] = pages_for(len, p.page_shift);
    need[tid] = fits ? pages_for(end, p.page_shift) : 0;
    have[tid] = 0;
    const int32_t page = fits && (len & (page_tokens - 1)) != 0 ? table_page(p, slot, len >> p.page_shift) : -1;
    tail[tid] = page < 0 ? kNone : static_cast<uint32_t>(page);
  }
  __syncthreads();
  if (bad != 0) {  // a sequence would pass its table row
    if (tid == 0) {
      *status = 1;
      plan->moves = 0;
    }
    return;
  }
  // Columns a call can ask for past a sequence's committed pages.
  const uint32_t width = pages_for(tokens, p.page_shift) + 1;
  for (uint32_t i = tid; i < list.count * width; i += kPlanThreads) {
    const uint32_t s = i / width, column = first[s] + (i - s * width);
    if (column < need[s] && table_page(p, list.slot[s], column) >= 0) atomicAdd(&have[s], 1u);
  }
  __syncthreads();
  uint32_t amount = 0, copied = 0;
  if (mine) {
    const uint32_t start = first[tid] + have[tid];
    amount = need[tid] > start ? need[tid] - start : 0;
    if (tail[tid] != kNone) {
      const uint32_t holders = p.references[tail[tid]];
      uint32_t requests = 0;
      bool later = false;
      const uint32_t mine_tail = tail[tid];
#pragma unroll 8
      for (uint32_t j = 0; j < list.count; ++j) {
        const bool same = tail[j] == mine_tail;
        requests += same ? 1u : 0u;
        later |= same && j > tid;
      }
      copied = holders > 1 && (requests < holders || later) ? 1u : 0u;
    }
    amount += copied;
    have[tid] = start;
  }
  uint32_t total, copies;
  const uint32_t before = block_scan(amount, partial, total);
  const uint32_t rank = block_scan(copied, partial, copies);
  if (mine) {
    offset[tid] = before;
    copy_rank[tid] = copied != 0 ? rank : kNone;
  }
  if (total == 0) {  // an ordinary decode step: every page is there and private
    if (tid == 0) {
      *status = 0;
      plan->moves = 0;
    }
    return;
  }
  uint32_t available = 0, rounds = 0;
  for (uint32_t base = 0; base < p.page_count && available < total; base += kPagesPerRound, ++rounds) {
    if (base != 0) mask = used_mask(p, base + tid * kPagesPerThread);
    uint32_t found;
    block_scan(kPagesPerThread - __popc(mask), partial, found);
    available += found;
  }
  if (tid == 0) {
    *status = available < total ? 1 : 0;
    plan->moves = available < total ? 0u : copies;
  }
  if (available < total) return;
  uint32_t done = 0;  // ranks given out in earlier rounds
  for (uint32_t round = 0; round < rounds; ++round) {
    const uint32_t base = round * kPagesPerRound + tid * kPagesPerThread;
    if (rounds > 1) {
      // Pages given out in an earlier round lie below this one, so the mask is as it was.
      mask = used_mask(p, base);
    }
    uint32_t found;
    const uint32_t mine_before = block_scan(kPagesPerThread - __popc(mask), partial, found);
    const uint32_t limit = min(found, total - done);
    for (uint32_t window = 0; window < limit; window += kPlanThreads) {
      uint32_t r = mine_before;
      for (uint32_t free = ~mask; free != 0; free &= free - 1, ++r) {
        if (r >= window && r < window + kPlanThreads && r < limit) taken[r - window] = base + __ffs(free) - 1;
      }
      __syncthreads();
      if (window + tid < limit) {
        const uint32_t page = taken[tid], global = done + window + tid;
        uint32_t low = 0, high = list.count;  // the last sequence whose offset is <= global
        while (high - low > 1) {
          const uint32_t mid = (low + high) / 2;
          if (offset[mid] <= global) low = mid;
          else high = mid;
        }
        const uint32_t slot = list.slot[low], k = global - offset[low];
        const std::size_t row = static_cast<std::size_t>(slot) * p.stride;
        const uint32_t copy = copy_rank[low];
        p.references[page] = 1;
        if (copy != kNone && k == 0) {
          p.table[row + (length[low] >> p.page_shift)] = static_cast<int32_t>(page);
          atomicSub(&p.references[tail[low]], 1u);
          plan->move[copy] = Move{tail[low], page, length[low] & (page_tokens - 1), 0};
        } else {
          p.table[row + have[low] + k - (copy != kNone ? 1u : 0u)] = static_cast<int32_t>(page);
        }
      }
      __syncthreads();
    }
    done += limit;
  }
}

struct PagePairs {
  uint32_t count;
  uint32_t from[256], to[256];
};

constexpr unsigned kCopyThreads = 256;
constexpr unsigned kCopyLoads = 8;  // 16-byte loads a lane keeps in flight
constexpr unsigned kCopyWorkgroups = 2048;

// Carries out page copies, 32 KB pieces over a grid that fills the GPU whatever the plan
// holds (an empty plan costs one load per workgroup: 2 us).  Sources and destinations of one
// plan are different pages, so the order does not matter.  Bound by memory: 32 pages of 4 MB
// (16 layers, K and V) 268 MB read and written in 46.6 us, 5.8 TB/s.
template <bool Listed>
__global__ __launch_bounds__(kCopyThreads) void copy_pages_kernel(KvPages p, const Plan* __restrict__ plan,
                                                                  PagePairs pairs) {
  const uint32_t moves = Listed ? pairs.count : plan->moves;
  if (moves == 0) return;
  const uint32_t units = p.row / 8;  // 16-byte units of a token row
  constexpr uint32_t kPiece = kCopyThreads * kCopyLoads;
  const uint32_t page_units = units << p.page_shift, pieces = (page_units + kPiece - 1) / kPiece;
  const uint64_t items = static_cast<uint64_t>(moves) * 2 * p.layers * pieces;
  for (uint64_t item = blockIdx.x; item < items; item += gridDim.x) {
    const uint32_t piece = static_cast<uint32_t>(item % pieces);
    const uint64_t rest = item / pieces;
    const uint32_t plane = static_cast<uint32_t>(rest % (2 * p.layers)), m = static_cast<uint32_t>(rest / (2 * p.layers));
    const Move move = Listed ? Move{pairs.from[m], pairs.to[m], 1u << p.page_shift, 0} : plan->move[m];
    const uint32_t limit = move.rows * units;
    u32x4* pool = reinterpret_cast<u32x4*>(plane < p.layers ? p.key : p.value);
    const std::size_t layer = static_cast<std::size_t>(plane % p.layers) * p.page_count;
    const u32x4* from = pool + (layer + move.from) * page_units;
    u32x4* to = pool + (layer + move.to) * page_units;
    const uint32_t at = piece * kPiece + threadIdx.x;
    u32x4 v[kCopyLoads];
#pragma unroll
    for (unsigned i = 0; i < kCopyLoads; ++i) {
      if (at + i * kCopyThreads < limit) v[i] = from[at + i * kCopyThreads];
    }
#pragma unroll
    for (unsigned i = 0; i < kCopyLoads; ++i) {
      if (at + i * kCopyThreads < limit) to[at + i * kCopyThreads] = v[i];
    }
  }
}

__global__ __launch_bounds__(256) void reset_kernel(KvPages p) {
  const std::size_t i = static_cast<std::size_t>(blockIdx.x) * 256 + threadIdx.x;
  if (i < static_cast<std::size_t>(p.sequences) * p.stride) p.table[i] = -1;
  if (i < p.sequences) p.lengths[i] = 0;
  if (i < p.page_count) p.references[i] = 0;
}

// Each thread owns one column of one child: what the child held there is given back and
// the parent's page of a committed position taken instead.  Bound by its look-ups, not by
// bytes: 3 children of 32 pages 2.0 us, 63 of 61 pages 3.4 us.
__global__ __launch_bounds__(256) void fork_kernel(KvPages p, uint32_t parent, SequenceList children) {
  const uint32_t column = blockIdx.x * 256 + threadIdx.x, child = listed_slot(children, blockIdx.y);
  if (column >= p.stride) return;
  const uint32_t len = p.lengths[parent];
  const int32_t before = table_page(p, child, column);
  const int32_t after = column < pages_for(len, p.page_shift) ? table_page(p, parent, column) : -1;
  if (before != after) {
    if (before >= 0) atomicSub(&p.references[before], 1u);
    if (after >= 0) atomicAdd(&p.references[after], 1u);
  }
  p.table[static_cast<std::size_t>(child) * p.stride + column] = after;
  if (column == 0) p.lengths[child] = len;
}

struct KeepList {
  uint32_t tokens[kMaxListed];
};

// min(min(len, keep), keep) = min(len, keep): a workgroup that reads the new length of a
// sequence computes the same columns as one that reads the old.  2.0..2.4 us, look-ups.
__global__ __launch_bounds__(256) void free_kernel(KvPages p, SequenceList list, KeepList keep) {
  const uint32_t column = blockIdx.x * 256 + threadIdx.x, slot = listed_slot(list, blockIdx.y);
  if (column >= p.stride) return;
  const uint32_t len = min(p.lengths[slot], keep.tokens[blockIdx.y]);
  if (column >= pages_for(len, p.page_shift)) {
    const int32_t page = table_page(p, slot, column);
    if (page >= 0) atomicSub(&p.references[page], 1u);
    p.table[static_cast<std::size_t>(slot) * p.stride + column] = -1;
  }
  if (column == 0) p.lengths[slot] = len;
}

// One thread a sequence, one load and one store: 1.4 us.
__global__ __launch_bounds__(kMaxListed) void advance_kernel(KvPages p, SequenceList list, uint32_t tokens,
                                                             const uint32_t* __restrict__ counts) {
  if (threadIdx.x >= list.count) return;
  const uint32_t slot = list.slot[threadIdx.x];
  const uint32_t n = counts != nullptr ? min(counts[threadIdx.x], tokens) : tokens;
  const uint64_t end = static_cast<uint64_t>(p.lengths[slot]) + n, most = static_cast<uint64_t>(p.stride) << p.page_shift;
  p.lengths[slot] = static_cast<uint32_t>(min(end, most));
}

// K (fp16) and V (fp32 -> fp16, one rounding) rows of one layer; a lane carries eight
// elements (16 + 32 bytes in, 16 + 16 out), on their way while it looks its page up.
// 2000 tokens of 1024 elements: 20.5 MB in 7.6 us, two dependent look-ups before the stores.
__global__ __launch_bounds__(256) void append_kernel(KvPages p, SequenceList list, uint32_t layer, uint32_t tokens,
                                                     const __half* __restrict__ key, const float* __restrict__ value) {
  const uint32_t units = p.row / 8, i = blockIdx.x * 256 + threadIdx.x, s = blockIdx.y;
  if (i >= tokens * units) return;
  const std::size_t source = static_cast<std::size_t>(s) * tokens * units + i;
  const u32x4 k = reinterpret_cast<const u32x4*>(key)[source];
  const f32x4 v0 = reinterpret_cast<const f32x4*>(value)[2 * source], v1 = reinterpret_cast<const f32x4*>(value)[2 * source + 1];
  const uint32_t slot = listed_slot(list, s), t = i / units, unit = i - t * units;
  const uint64_t position = static_cast<uint64_t>(p.lengths[slot]) + t;
  if (position >> p.page_shift >= p.stride) return;
  const int32_t page = table_page(p, slot, static_cast<uint32_t>(position >> p.page_shift));
  // Shared pages are not written: without a reserve since the last fork, two
  // sequences would write the same rows, in no order.
  if (page < 0 || p.references[page] > 1u) return;
  h16x8 v;
#pragma unroll
  for (unsigned e = 0; e < 4; ++e) {
    v[e] = static_cast<_Float16>(v0[e]);
    v[4 + e] = static_cast<_Float16>(v1[e]);
  }
  const std::size_t row = ((static_cast<std::size_t>(layer) * p.page_count + page) << p.page_shift) +
                          (position & ((1u << p.page_shift) - 1));
  reinterpret_cast<u32x4*>(p.key)[row * units + unit] = k;
  reinterpret_cast<h16x8*>(p.value)[row * units + unit] = v;
}

// One workgroup plans a compaction: with `live` used pages, the used pages at or past
// `live` move, in order, to the free pages before it, in order (there are as many).  Bound by
// two passes of scans over the reference counts: 5.5 us (some hundred pages) to 7.8 us.
__global__ __launch_bounds__(kPlanThreads) void compact_kernel(KvPages p, Plan* plan, uint32_t* map,
                                                               uint32_t* __restrict__ live_pages) {
  __shared__ uint32_t partial[kPlanThreads / 64];
  const unsigned tid = threadIdx.x;
  uint32_t live = 0;
  for (uint32_t base = 0; base < p.page_count; base += kPagesPerRound) {
    const uint32_t first = base + tid * kPagesPerThread;
    // Pages past the pool read as used: not counted.
    const uint32_t there = first >= p.page_count ? 0u : min(kPagesPerThread, p.page_count - first);
    const uint32_t mask = used_mask(p, first) & (there == kPagesPerThread ? 0xffffffffu : (1u << there) - 1u);
    uint32_t found;
    block_scan(__popc(mask), partial, found);
    live += found;
  }
  uint32_t holes = 0, movers = 0;
  for (uint32_t base = 0; base < p.page_count; base += kPagesPerRound) {
    const uint32_t first = base + tid * kPagesPerThread;
    const uint32_t there = first >= p.page_count ? 0u : min(kPagesPerThread, p.page_count - first);
    const uint32_t exists = there == kPagesPerThread ? 0xffffffffu : (1u << there) - 1u;
    const uint32_t below = first >= live ? 0u : live - first >= kPagesPerThread ? 0xffffffffu : (1u << (live - first)) - 1u;
    const uint32_t used = used_mask(p, first);
    const uint32_t hole = ~used & below, mover = used & exists & ~below;
    uint32_t total;  // holes in the low half, movers in the high half: at most 2^15 each per round
    uint32_t before = block_scan(static_cast<uint32_t>(__popc(hole)) | static_cast<uint32_t>(__popc(mover)) << 16,
                                 partial, total);
    uint32_t r = holes + (before & 0xffffu);
    for (uint32_t bits = hole; bits != 0; bits &= bits - 1) plan->move[r++].to = first + __ffs(bits) - 1;
    r = movers + (before >> 16);
    for (uint32_t bits = mover; bits != 0; bits &= bits - 1) {
      plan->move[r].from = first + __ffs(bits) - 1;
      plan->move[r++].rows = 1u << p.page_shift;
    }
    holes += total & 0xffffu;
    movers += total >> 16;
  }
  __threadfence_block();
  __syncthreads();
  for (uint32_t m = tid; m < movers; m += kPlanThreads) {
    const uint32_t from = plan->move[m].from, to = plan->move[m].to;
    map[from] = to;
    p.references[to] = p.references[from];
    p.references[from] = 0;
  }
  if (tid == 0) {
    plan->moves = movers;
    plan->live = live;
    if (live_pages != nullptr) *live_pages = live;
  }
}

// Renames the moved pages in every table entry (a moved page may have several holders): 1.6 us
// for 21 sequences, 4.7 us for 61.
__global__ __launch_bounds__(256) void rewrite_table_kernel(KvPages p, const Plan* __restrict__ plan,
                                                            const uint32_t* __restrict__ map) {
  if (plan->moves == 0) return;
  const uint32_t live = plan->live;
  const std::size_t entries = static_cast<std::size_t>(p.sequences) * p.stride;
  for (std::size_t i = static_cast<std::size_t>(blockIdx.x) * 256 + threadIdx.x; i < entries;
       i += static_cast<std::size_t>(gridDim.x) * 256) {
    const int32_t page = p.table[i];
    if (page >= 0 && static_cast<uint32_t>(page) >= live && static_cast<uint32_t>(page) < p.page_count) {
      p.table[i] = static_cast<int32_t>(map[page]);
    }
  }
}

int32_t copy_plan(const KvPages& p, const Plan* plan, hipStream_t stream) {
  hipLaunchKernelGGL(copy_pages_kernel<false>, dim3(kCopyWorkgroups), dim3(kCopyThreads), 0, stream, p, plan, PagePairs{});
  return launch_status("page copy launch failed");
}

int32_t read_workspace(const KvPages& p, void* workspace, size_t bytes) {
  if (workspace == nullptr || !aligned16(workspace) || bytes < plan_bytes(p.page_count)) {
    return fail(GFXI_INVALID_ARGUMENT, "K/V page workspace is null, not 16-byte aligned or too small");
  }
  return GFXI_OK;
}

}  // namespace

int32_t read_pages(const gfxinfer_kv_pages* pages, KvPages& out) {
  if (pages == nullptr) return fail(GFXI_INVALID_ARGUMENT, "K/V pages are null");
  const gfxinfer_kv_pages& g = *pages;
  if (g.key_pages == nullptr || g.value_pages == nullptr || g.page_table == nullptr || g.lengths == nullptr ||
      g.references == nullptr || !aligned16(g.key_pages) || !aligned16(g.value_pages) || !aligned16(g.references)) {
    return fail(GFXI_INVALID_ARGUMENT, "K/V page pools and state must be set; pools and references 16-byte aligned");
  }
  if (g.layers == 0 || g.layers > 4096 || g.page_count == 0 || g.page_count > (1u << 24) || g.page_tokens < 16 ||
      g.page_tokens > 4096 || (g.page_tokens & (g.page_tokens - 1)) != 0 || g.kv_heads == 0 || g.kv_heads > 1024 ||
      (g.head_size != 128 && g.head_size != 256) || g.sequences == 0 || g.sequences > kMaxSequences ||
      g.table_stride == 0 || g.table_stride > (1u << 20) ||
      static_cast<uint64_t>(g.table_stride) * g.page_tokens > (1ull << 31) ||
      static_cast<uint64_t>(g.table_stride) * g.sequences > (1ull << 31)) {
    return fail(GFXI_INVALID_ARGUMENT,
                "invalid K/V page sizes (pages of 16..4096 tokens, a power of two; head size 128 or 256; at most 2^24 "
                "pages, 65536 sequences, 2^31 tokens per sequence and 2^31 table entries)");
  }
  out.key = reinterpret_cast<__half*>(g.key_pages);
  out.value = reinterpret_cast<__half*>(g.value_pages);
  out.table = g.page_table;
  out.lengths = g.lengths;
  out.references = g.references;
  out.layers = g.layers;
  out.page_count = g.page_count;
  out.page_shift = static_cast<uint32_t>(__builtin_ctz(g.page_tokens));
  out.row = g.kv_heads * g.head_size;
  out.sequences = g.sequences;
  out.stride = g.table_stride;
  return GFXI_OK;
}

int32_t read_sequences(const KvPages& pages, const uint32_t* sequences, uint32_t count, bool distinct,
                       SequenceList& out) {
  if (count == 0 || count > kMaxListed || (sequences == nullptr && count > pages.sequences)) {
    return fail(GFXI_INVALID_ARGUMENT, "a call names 1.." + std::to_string(kMaxListed) + " sequences of the cache");
  }
  out.count = count;
  std::bitset<kMaxSequences> seen;
  for (uint32_t i = 0; i < count; ++i) {
    const uint32_t slot = sequences != nullptr ? sequences[i] : i;
    if (slot >= pages.sequences) {
      return fail(GFXI_INVALID_ARGUMENT, "sequence " + std::to_string(slot) + " is not in the cache");
    }
    if (distinct && sequences != nullptr) {
      if (seen[slot]) return fail(GFXI_INVALID_ARGUMENT, "sequence " + std::to_string(slot) + " is named twice");
      seen[slot] = true;
    }
    out.slot[i] = static_cast<uint16_t>(slot);
  }
  return GFXI_OK;
}

}  // namespace gfx950

using namespace gfx950;

extern "C" size_t gfxinfer_kv_pages_workspace_bytes(const gfxinfer_kv_pages* pages) {
  KvPages p;
  size_t bytes = 0;
  guarded([&] {
    const int32_t s = read_pages(pages, p);
    if (s == GFXI_OK) bytes = plan_bytes(p.page_count);
    return s;
  });
  return bytes;
}

extern "C" int32_t gfxinfer_launch_kv_pages_reset(const gfxinfer_kv_pages* pages, void* stream) {
  return guarded([&] {
    KvPages p;
    if (const int32_t s = read_pages(pages, p); s != GFXI_OK) return s;
    const std::size_t n = std::max<std::size_t>(static_cast<std::size_t>(p.sequences) * p.stride,
                                                std::max(p.sequences, p.page_count));
    hipLaunchKernelGGL(reset_kernel, dim3(static_cast<unsigned>((n + 255) / 256)), dim3(256), 0,
                       static_cast<hipStream_t>(stream), p);
    return launch_status("K/V page reset launch failed");
  });
}

extern "C" int32_t gfxinfer_launch_kv_pages_fork(const gfxinfer_kv_pages* pages, uint32_t parent,
                                                 const uint32_t* children, uint32_t count, void* stream) {
  return guarded([&] {
    KvPages p;
    SequenceList list;
    if (const int32_t s = read_pages(pages, p); s != GFXI_OK) return s;
    if (children == nullptr || parent >= p.sequences) {
      return fail(GFXI_INVALID_ARGUMENT, "fork needs a parent of the cache and a list of children");
    }
    if (const int32_t s = read_sequences(p, children, count, true, list); s != GFXI_OK) return s;
    for (uint32_t i = 0; i < count; ++i) {
      if (list.slot[i] == parent) return fail(GFXI_INVALID_ARGUMENT, "a sequence cannot be forked onto itself");
    }
    hipLaunchKernelGGL(fork_kernel, dim3((p.stride + 255) / 256, count), dim3(256), 0, static_cast<hipStream_t>(stream),
                       p, parent, list);
    return launch_status("K/V page fork launch failed");
  });
}

extern "C" int32_t gfxinfer_launch_kv_pages_free(const gfxinfer_kv_pages* pages, const uint32_t* sequences,
                                                 const uint32_t* keep_tokens, uint32_t count, void* stream) {
  return guarded([&] {
    KvPages p;
    SequenceList list;
    if (const int32_t s = read_pages(pages, p); s != GFXI_OK) return s;
    if (const int32_t s = read_sequences(p, sequences, count, true, list); s != GFXI_OK) return s;
    KeepList keep{};
    for (uint32_t i = 0; i < count && keep_tokens != nullptr; ++i) keep.tokens[i] = keep_tokens[i];
    hipLaunchKernelGGL(free_kernel, dim3((p.stride + 255) / 256, count), dim3(256), 0, static_cast<hipStream_t>(stream),
                       p, list, keep);
    return launch_status("K/V page free launch failed");
  });
}

extern "C" int32_t gfxinfer_launch_kv_pages_reserve(const gfxinfer_kv_pages* pages, const uint32_t* sequences,
                                                    uint32_t count, uint32_t tokens, int32_t* status, void* workspace,
                                                    size_t workspace_bytes, void* stream) {
  return guarded([&] {
    KvPages p;
    SequenceList list;
    if (const int32_t s = read_pages(pages, p); s != GFXI_OK) return s;
    if (const int32_t s = read_sequences(p, sequences, count, true, list); s != GFXI_OK) return s;
    if (tokens == 0 || tokens > (1u << 24) || status == nullptr) {
      return fail(GFXI_INVALID_ARGUMENT, "reserve needs 1..2^24 tokens and a status word");
    }
    if (const int32_t s = read_workspace(p, workspace, workspace_bytes); s != GFXI_OK) return s;
    Plan* plan = static_cast<Plan*>(workspace);
    hipLaunchKernelGGL(reserve_kernel, dim3(1), dim3(kPlanThreads), 0, static_cast<hipStream_t>(stream), p, list, tokens,
                       status, plan);
    if (const int32_t s = launch_status("K/V page reserve launch failed"); s != GFXI_OK) return s;
    return copy_plan(p, plan, static_cast<hipStream_t>(stream));
  });
}

extern "C" int32_t gfxinfer_launch_kv_pages_append(const gfxinfer_kv_pages* pages, uint32_t layer, const uint16_t* key,
                                                   const float* value, const uint32_t* sequences, uint32_t count,
                                                   uint32_t tokens, void* stream) {
  return guarded([&] {
    KvPages p;
    SequenceList list;
    if (const int32_t s = read_pages(pages, p); s != GFXI_OK) return s;
    if (const int32_t s = read_sequences(p, sequences, count, true, list); s != GFXI_OK) return s;
    if (layer >= p.layers || key == nullptr || value == nullptr || !aligned16(key) || !aligned16(value) || tokens == 0) {
      return fail(GFXI_INVALID_ARGUMENT, "append needs a layer of the cache, at least one token and 16-byte aligned rows");
    }
    const uint64_t lanes = static_cast<uint64_t>(count) * tokens * (p.row / 8);
    if (lanes > (1ull << 31)) return fail(GFXI_INVALID_ARGUMENT, "append of too many tokens");
    hipLaunchKernelGGL(append_kernel, dim3(static_cast<unsigned>((lanes / count + 255) / 256), count), dim3(256), 0,
                       static_cast<hipStream_t>(stream), p, list, layer, tokens, reinterpret_cast<const __half*>(key),
                       value);
    return launch_status("K/V page append launch failed");
  });
}

extern "C" int32_t gfxinfer_launch_kv_pages_advance(const gfxinfer_kv_pages* pages, const uint32_t* sequences,
                                                    uint32_t count, uint32_t tokens, const uint32_t* token_counts,
                                                    void* stream) {
  return guarded([&] {
    KvPages p;
    SequenceList list;
    if (const int32_t s = read_pages(pages, p); s != GFXI_OK) return s;
    if (const int32_t s = read_sequences(p, sequences, count, true, list); s != GFXI_OK) return s;
    hipLaunchKernelGGL(advance_kernel, dim3(1), dim3(kMaxListed), 0, static_cast<hipStream_t>(stream), p, list, tokens,
                       token_counts);
    return launch_status("K/V page advance launch failed");
  });
}

extern "C" int32_t gfxinfer_launch_kv_pages_copy(const gfxinfer_kv_pages* pages, const uint32_t* sources,
                                                 const uint32_t* destinations, uint32_t count, void* stream) {
  return guarded([&] {
    KvPages p;
    if (const int32_t s = read_pages(pages, p); s != GFXI_OK) return s;
    PagePairs pairs{};
    if (sources == nullptr || destinations == nullptr || count == 0 || count > std::size(pairs.from)) {
      return fail(GFXI_INVALID_ARGUMENT, "a page copy names 1..256 pairs of pages");
    }
    pairs.count = count;
    for (uint32_t i = 0; i < count; ++i) {
      if (sources[i] >= p.page_count || destinations[i] >= p.page_count) {
        return fail(GFXI_INVALID_ARGUMENT, "a page to copy is not in the pool");
      }
      for (uint32_t j = 0; j < count; ++j) {
        if (sources[j] == destinations[i] || (j < i && destinations[j] == destinations[i])) {
          return fail(GFXI_INVALID_ARGUMENT, "page " + std::to_string(destinations[i]) +
                                                 " is a destination twice or also a source of the same call");
        }
      }
      pairs.from[i] = sources[i];
      pairs.to[i] = destinations[i];
    }
    hipLaunchKernelGGL(copy_pages_kernel<true>, dim3(kCopyWorkgroups), dim3(kCopyThreads), 0,
                       static_cast<hipStream_t>(stream), p, nullptr, pairs);
    return launch_status("page copy launch failed");
  });
}

extern "C" int32_t gfxinfer_launch_kv_pages_compact(const gfxinfer_kv_pages* pages, uint32_t* live_pages, void* workspace,
                                                    size_t workspace_bytes, void* stream) {
  return guarded([&] {
    KvPages p;
    if (const int32_t s = read_pages(pages, p); s != GFXI_OK) return s;
    if (const int32_t s = read_workspace(p, workspace, workspace_bytes); s != GFXI_OK) return s;
    Plan* plan = static_cast<Plan*>(workspace);
    uint32_t* map = plan_map(plan, plan_moves(p.page_count));
    const hipStream_t st = static_cast<hipStream_t>(stream);
    hipLaunchKernelGGL(compact_kernel, dim3(1), dim3(kPlanThreads), 0, st, p, plan, map, live_pages);
    if (const int32_t s = launch_status("K/V page compaction launch failed"); s != GFXI_OK) return s;
    if (const int32_t s = copy_plan(p, plan, st); s != GFXI_OK) return s;
    const std::size_t entries = static_cast<std::size_t>(p.sequences) * p.stride;
    hipLaunchKernelGGL(rewrite_table_kernel, dim3(static_cast<unsigned>(std::min<std::size_t>((entries + 255) / 256, 2048))),
                       dim3(256), 0, st, p, plan, map);
    return launch_status("K/V page table launch failed");
  });
}
