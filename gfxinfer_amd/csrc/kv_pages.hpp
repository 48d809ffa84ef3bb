// The paged K/V cache as the kernels take it, and the host lists of sequences that its
// launchers pass as kernel arguments.
#pragma once

#include <bitset>

#include "common.hpp"

namespace gfx950 {

// Sequences one call names: their slots travel as kernel arguments (1 KB of the 4 KB a
// launch can carry), so a captured call replays with the list it was recorded with.
constexpr uint32_t kMaxListed = 512;
constexpr uint32_t kMaxSequences = 65536;

struct SequenceList {
  uint32_t count;
  alignas(4) uint16_t slot[kMaxListed];
};

// gfxinfer_kv_pages with the sizes the kernels index by.
struct KvPages {
  __half* key;      // [layers][page_count][page_tokens][row]
  __half* value;
  int32_t* table;   // [sequences][stride]
  uint32_t* lengths;
  uint32_t* references;
  uint32_t layers, page_count, page_shift, row, sequences, stride;  // row = kv_heads * head_size halves
};

__device__ __forceinline__ uint32_t pages_for(uint64_t tokens, uint32_t shift) {
  return static_cast<uint32_t>((tokens + (1u << shift) - 1) >> shift);
}

// The i-th listed slot (i the same in all lanes) through the scalar cache, which has no
// 16-bit loads.
__device__ __forceinline__ uint32_t listed_slot(const SequenceList& list, uint32_t i) {
  const uint32_t pair = reinterpret_cast<const uint32_t*>(list.slot)[i / 2];
  return i % 2 != 0 ? pair >> 16 : pair & 0xffffu;
}

// The page of a sequence's table entry, or -1: entries that name no page of the pool are
// treated like missing ones everywhere, so that a damaged table cannot reach outside it.
__device__ __forceinline__ int32_t table_page(const KvPages& p, uint32_t slot, uint32_t column) {
  if (column >= p.stride) return -1;
  const int32_t page = p.table[static_cast<std::size_t>(slot) * p.stride + column];
  return page >= 0 && static_cast<uint32_t>(page) < p.page_count ? page : -1;
}

inline bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

// Checks the description; returns GFXI_OK and fills `out`, or the status to return.
int32_t read_pages(const gfxinfer_kv_pages* pages, KvPages& out);
// Copies a host list of sequences (NULL: 0..count-1) into `out`; `distinct` refuses a
// sequence named twice (calls that write a sequence's state).
int32_t read_sequences(const KvPages& pages, const uint32_t* sequences, uint32_t count, bool distinct,
                       SequenceList& out);

}  // namespace gfx950
