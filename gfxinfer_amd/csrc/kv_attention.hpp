// Device parts that the attentions over K/V pages share: loads into LDS and their waits, the
// order of K and V rows there, page look-ups, infinities and NaNs among the values.
#pragma once

#include "kv_pages.hpp"

namespace gfx950 {

using h8 = _Float16 __attribute__((ext_vector_type(8)));
using f4 = float __attribute__((ext_vector_type(4)));
using h2 = _Float16 __attribute__((ext_vector_type(2)));
using f2 = float __attribute__((ext_vector_type(2)));
using u32x4 = unsigned __attribute__((ext_vector_type(4)));
using s16x4 = short __attribute__((ext_vector_type(4)));
using lds_void = __attribute__((address_space(3))) void;
using global_void = __attribute__((address_space(1))) void;

constexpr float kLog2E = 1.4426950408889634F;

// The factor between sums with maxima `from` and `to`, from <= to nearly always.  Never zero, so
// that a NaN or an infinity of either reaches the result however far its scores lie below the
// others (2^-126 of a finite sum is nothing beside theirs).
__device__ __forceinline__ float rescale_factor(float from, float to) {
  return fmaxf(__builtin_amdgcn_exp2f(from - to), 0x1p-126F);
}

// Committed positions of a slot; a damaged length does not lead far past the table.
__device__ __forceinline__ uint32_t committed(const KvPages& p, uint32_t slot) {
  return min(static_cast<uint32_t>(__builtin_amdgcn_readfirstlane(p.lengths[slot])), p.stride << p.page_shift);
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

__device__ __forceinline__ unsigned lds_address(const _Float16* p) {
  return static_cast<unsigned>(reinterpret_cast<uintptr_t>((lds_void*)(p)));
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

// A barrier that orders LDS accesses and leaves loads from memory into LDS on their way
// (__syncthreads would wait for them).
__device__ __forceinline__ void lds_barrier() {
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}

}  // namespace gfx950
