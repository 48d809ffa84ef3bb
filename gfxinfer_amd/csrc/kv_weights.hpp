// What the calls of a cache within a budget share: host lists of sequences with their own
// numbers of new tokens, and the weights beside the pages.
#pragma once

#include "kv_pages.hpp"

namespace gfx950 {

// Sequences of a chunk call: slots, and where their packed rows begin (first[count]: the end).
// 1.5 KB of the 4 KB a launch can carry.
constexpr uint32_t kMaxChunks = 256, kMaxRows = 1u << 20;

struct ChunkList {
  uint32_t count;
  alignas(4) uint16_t slot[kMaxChunks];
  uint32_t first[kMaxChunks + 1];
};

__device__ __forceinline__ uint32_t listed_slot(const ChunkList& list, uint32_t i) {
  const uint32_t pair = reinterpret_cast<const uint32_t*>(list.slot)[i / 2];
  return i % 2 != 0 ? pair >> 16 : pair & 0xffffu;
}

struct KvWeights {
  float* weight;      // [sequences][capacity]
  int32_t* position;  // [sequences][capacity]
  uint32_t* dropped;  // [sequences]
};

// Checks the lists (sequences NULL: 0..count-1) and fills `out`, or returns the status.
int32_t read_chunks(const KvPages& pages, const uint32_t* sequences, const uint32_t* tokens, uint32_t count, bool distinct,
                    ChunkList& out);
int32_t read_weights(const gfxinfer_kv_weights* weights, KvWeights& out);

}  // namespace gfx950
