// Rules on logits before the greedy pick: repetition, presence and frequency penalties
// over a row's token history, sparse biases and grammar masks, with the argmax of the
// result in the same pass.
//
// For row b and token v, with c = how often v occurs in the generated part of the
// history and r = whether it occurs anywhere in it:
//     x = r ? (x > 0 ? x / repetition : x * repetition) : x
//     x = x - frequency * c, then x - presence if c > 0
//     x = x + bias(v)           (the last entry that names v)
//     x = allowed(v) ? x : -inf
// in fp32, each operation rounded once.
//
// A workgroup takes a slice of the vocabulary.  It keeps one counter word per token of the
// slice in LDS, fills them from the whole history (integer LDS atomics, so the order of the
// lanes does not matter) and then passes over its logits once.  No per-row count array in
// memory has to be cleared, filled and read back; the price is that every slice of a row
// reads the row's history, which stays in L2.  What bounds it is the pass over the logits:
// 256 rows x 151936 move 319 MB in 73.5 us (4.3 TB/s, reads and writes).
#include <algorithm>

#include "common.hpp"

namespace gfx950 {
namespace {

using u32x4 = unsigned __attribute__((ext_vector_type(4)));
using f32x4 = float __attribute__((ext_vector_type(4)));

// Counter word of a token: bits 0..18 its count among the generated tokens, bit 19 set if
// the prompt holds it, bits 20..31 one more than the index of its last bias entry.
constexpr unsigned kPromptBit = 1u << 19;
constexpr unsigned kSeenMask = (1u << 20) - 1;
constexpr unsigned kBiasShift = 20;
constexpr uint32_t kMaxHistory = (1u << 19) - 1;
constexpr uint32_t kMaxBias = (1u << 12) - 1;

constexpr unsigned kThreads = 256;
// History tokens a lane has on their way at once (256 rows x 151936 with 2000-token histories:
// 8 of them 73.7 us, 4 of them 77 us in more rounds, 16 of them 90 us with fewer waves).
constexpr unsigned kHistoryLoads = 8;

struct RulesArgs {
  gfxinfer_logit_rules rules;
  const float* logits;
  float* output;
  unsigned long long* keys;
  std::size_t row_stride, output_stride;
  uint32_t vocabulary, slices;
};

// Larger values have larger keys, equal values (0 and -0 alike) the lower token the larger
// key; 0 for what never wins (NaN, -inf).
__device__ __forceinline__ unsigned long long logit_key(float x, uint32_t token) {
  if (!(x > -INFINITY)) return 0ull;
  const unsigned bits = __float_as_uint(x + 0.0F);
  const unsigned ordered = (bits & 0x80000000u) != 0 ? ~bits : bits | 0x80000000u;
  return (static_cast<unsigned long long>(ordered) << 32) | (0xffffffffu - token);
}

// A lane takes kSlice / kThreads tokens: with Vec in groups of four consecutive ones (16-byte
// loads and stores), otherwise kThreads apart.  Its logits are loaded before the history is
// counted, so that one memory latency covers both.
template <unsigned kSlice, bool Vec>
__global__ __launch_bounds__(kThreads) void logit_rules_kernel(RulesArgs a) {
  constexpr unsigned kItems = kSlice / kThreads;
  __shared__ __align__(16) unsigned counter[kSlice];
  __shared__ unsigned long long partial[kThreads / 64];
  const gfxinfer_logit_rules& r = a.rules;
  const unsigned tid = threadIdx.x;
  const uint32_t b = blockIdx.x / a.slices, slice = blockIdx.x - b * a.slices;
  const uint32_t v0 = slice * kSlice, count = min(kSlice, a.vocabulary - v0);
  auto place = [&](unsigned k) __attribute__((always_inline)) {  // of the lane's k-th token in the slice
    return Vec ? 4 * (tid + kThreads * (k / 4)) + k % 4 : tid + kThreads * k;
  };

  const float* in = a.logits + b * a.row_stride + v0;
  float x[kItems];
#pragma unroll
  for (unsigned k = 0; k < kItems; k += 4) {
    if (Vec && place(k) + 3 < count) {
      const f32x4 v = *reinterpret_cast<const f32x4*>(in + place(k));
#pragma unroll
      for (unsigned e = 0; e < 4; ++e) x[k + e] = v[e];
    } else {
#pragma unroll
      for (unsigned e = 0; e < 4; ++e) x[k + e] = place(k + e) < count ? in[place(k + e)] : -INFINITY;
    }
  }

  const uint32_t* history = nullptr;
  uint32_t length = 0, prompt = 0;
  if (r.history != nullptr) {
    const int32_t row = r.history_rows != nullptr ? r.history_rows[b] : static_cast<int32_t>(b);
    if (row >= 0 && static_cast<uint32_t>(row) < r.history_row_count) {
      history = r.history + static_cast<std::size_t>(row) * r.history_stride;
      length = min(r.history_lengths[b], r.history_stride);
      prompt = r.prompt_lengths != nullptr ? r.prompt_lengths[b] : 0u;
    }
  }
  uint32_t biases = 0;
  if (r.bias_tokens != nullptr) biases = r.bias_counts != nullptr ? min(r.bias_counts[b], r.bias_stride) : r.bias_stride;
  const uint32_t* allowed = nullptr;
  if (r.allowed != nullptr) {
    const int32_t row = r.allowed_rows != nullptr ? r.allowed_rows[b] : static_cast<int32_t>(b);
    if (row >= 0 && static_cast<uint32_t>(row) < r.allowed_row_count) {
      allowed = r.allowed + static_cast<std::size_t>(row) * r.allowed_stride;
    }
  }
  // The mask words of the lane's tokens (one for each group of four with Vec).
  constexpr unsigned kWordStep = Vec ? 4 : 1;
  uint32_t words[kItems / kWordStep];
#pragma unroll
  for (unsigned k = 0; k < kItems; k += kWordStep) {
    words[k / kWordStep] = allowed != nullptr && place(k) < count ? allowed[(v0 + place(k)) / 32] : 0xffffffffu;
  }
  const bool counted = length != 0 || biases != 0;
  if (counted) {
    for (uint32_t i = 4 * tid; i < kSlice; i += 4 * kThreads) *reinterpret_cast<u32x4*>(counter + i) = u32x4{0, 0, 0, 0};
    __syncthreads();
    for (uint32_t base = tid; base < length; base += kThreads * kHistoryLoads) {
      uint32_t u[kHistoryLoads];
#pragma unroll
      for (unsigned k = 0; k < kHistoryLoads; ++k) {
        const uint32_t i = base + k * kThreads;
        u[k] = history[min(i, length - 1)];
      }
#pragma unroll
      for (unsigned k = 0; k < kHistoryLoads; ++k) {
        const uint32_t i = base + k * kThreads;
        if (i < length && u[k] - v0 < count) {  // wraps for tokens before the slice
          if (i < prompt) atomicOr(&counter[u[k] - v0], kPromptBit);
          else atomicAdd(&counter[u[k] - v0], 1u);
        }
      }
    }
    __syncthreads();
    // The low bits no longer change, so the largest word of a token is its last entry's.
    const uint32_t* tokens = r.bias_tokens + static_cast<std::size_t>(b) * r.bias_stride;
    for (uint32_t i = tid; i < biases; i += kThreads) {
      const uint32_t u = tokens[i] - v0;
      if (u < count) atomicMax(&counter[u], (counter[u] & kSeenMask) | (i + 1) << kBiasShift);
    }
    __syncthreads();
  }
  const float repetition = r.repetition != nullptr ? r.repetition[b] : 1.0F;
  const float presence = r.presence != nullptr ? r.presence[b] : 0.0F;
  const float frequency = r.frequency != nullptr ? r.frequency[b] : 0.0F;
  const float* values = r.bias_values + static_cast<std::size_t>(b) * r.bias_stride;
  unsigned long long best = 0ull;
#pragma unroll
  for (unsigned k = 0; k < kItems; ++k) {
    const uint32_t i = place(k);
    if (counted && i < count) {
      const unsigned word = counter[i];
      if (word != 0) {
        float y = x[k];
        if ((word & kSeenMask) != 0) {
          y = y > 0.0F ? y / repetition : y * repetition;
          const unsigned c = word & (kPromptBit - 1);
          if (c != 0) {
            y = y - frequency * static_cast<float>(c);
            y = y - presence;
          }
        }
        if (word >> kBiasShift != 0) y = y + values[(word >> kBiasShift) - 1];
        x[k] = y;
      }
    }
    if ((words[k / kWordStep] >> ((v0 + i) % 32) & 1u) == 0) x[k] = -INFINITY;
    const unsigned long long key = logit_key(x[k], v0 + i);
    if (i < count) best = key > best ? key : best;
  }
  if (a.output != nullptr) {
    float* out = a.output + b * a.output_stride + v0;
#pragma unroll
    for (unsigned k = 0; k < kItems; k += 4) {
      if (Vec && place(k) + 3 < count) {
        *reinterpret_cast<f32x4*>(out + place(k)) = f32x4{x[k], x[k + 1], x[k + 2], x[k + 3]};
      } else {
#pragma unroll
        for (unsigned e = 0; e < 4; ++e) {
          if (place(k + e) < count) out[place(k + e)] = x[k + e];
        }
      }
    }
  }
  if (a.keys == nullptr) return;
  best = wave_max_key(best);
  if ((tid & 63u) == 0) partial[tid >> 6] = best;
  __syncthreads();
  if (tid == 0) {
    for (unsigned w = 1; w < kThreads / 64; ++w) best = partial[w] > best ? partial[w] : best;
    a.keys[blockIdx.x] = best;
  }
}

// The largest of a row's slice keys: a second launch, one load chain (2.6 us for 75 keys a row,
// 4.6 us for 38 keys of 256 rows).
__global__ __launch_bounds__(kThreads) void rule_tokens_kernel(const unsigned long long* __restrict__ keys,
                                                               uint32_t slices, uint32_t* __restrict__ tokens) {
  __shared__ unsigned long long partial[kThreads / 64];
  const unsigned long long best = block_max_key(keys + static_cast<std::size_t>(blockIdx.x) * slices, slices, partial);
  if (threadIdx.x == 0) tokens[blockIdx.x] = argmax_key_row(best);
}

// Tokens of a slice: small ones while the rows do not fill the GPU, large ones where that
// leaves four workgroups a CU, since every slice reads its row's history (256 rows x 151936
// with 2000-token histories: 73.5 us with large slices, 79 us with small ones; 32 rows x
// 248077 with 4000: 19.8 and 21.0 us.  8192 tokens: 95 us, their registers leave too few
// waves).
constexpr unsigned kSmall = 2048, kLarge = 4096;
unsigned slice_of(std::size_t vocabulary, uint32_t batch) {
  return (vocabulary + kLarge - 1) / kLarge * batch >= 4 * kComputeUnits ? kLarge : kSmall;
}
uint32_t slice_count(std::size_t vocabulary, uint32_t batch) {
  const unsigned slice = slice_of(vocabulary, batch);
  return static_cast<uint32_t>((vocabulary + slice - 1) / slice);
}

bool sized(std::size_t vocabulary, uint32_t batch) {
  return vocabulary != 0 && vocabulary <= (1u << 24) && batch != 0 && batch <= 65535;
}

}  // namespace
}  // namespace gfx950

using namespace gfx950;

extern "C" size_t gfxinfer_logit_rules_workspace_bytes(size_t vocabulary_size, uint32_t batch) {
  return sized(vocabulary_size, batch) ? static_cast<std::size_t>(batch) * slice_count(vocabulary_size, batch) * 8 : 0;
}

extern "C" int32_t gfxinfer_launch_logit_rules(const float* logits, size_t row_stride, size_t vocabulary_size, uint32_t batch,
                                               const gfxinfer_logit_rules* rules, float* output, size_t output_stride,
                                               uint32_t* tokens, void* workspace, size_t workspace_bytes, void* stream) {
  return guarded([&] {
    if (logits == nullptr || rules == nullptr || (output == nullptr && tokens == nullptr) || !sized(vocabulary_size, batch) ||
        row_stride < vocabulary_size || (output != nullptr && output_stride < vocabulary_size)) {
      return fail(GFXI_INVALID_ARGUMENT, "invalid logit rule arguments (1..2^24 tokens, 1..65535 rows, strides that hold a "
                                         "row, an output or tokens)");
    }
    if (output == logits && output_stride != row_stride) {
      return fail(GFXI_INVALID_ARGUMENT, "logit rules in place keep the row stride");
    }
    const gfxinfer_logit_rules& r = *rules;
    if (r.history != nullptr && (r.history_lengths == nullptr || r.history_stride == 0 || r.history_stride > kMaxHistory ||
                                 (r.history_rows == nullptr && r.history_row_count < batch))) {
      return fail(GFXI_INVALID_ARGUMENT, "a token history needs lengths, 1..524287 tokens a row and a row for every logits row");
    }
    if ((r.bias_tokens == nullptr) != (r.bias_values == nullptr) ||
        (r.bias_tokens != nullptr && (r.bias_stride == 0 || r.bias_stride > kMaxBias))) {
      return fail(GFXI_INVALID_ARGUMENT, "biases need tokens and values, 1..4095 a row");
    }
    if (r.allowed != nullptr && (r.allowed_stride < (vocabulary_size + 31) / 32 ||
                                 (r.allowed_rows == nullptr && r.allowed_row_count < batch))) {
      return fail(GFXI_INVALID_ARGUMENT, "a mask needs a bit for every token and a row for every logits row");
    }
    if (tokens != nullptr && (workspace == nullptr || (reinterpret_cast<uintptr_t>(workspace) & 7u) != 0 ||
                              workspace_bytes < gfxinfer_logit_rules_workspace_bytes(vocabulary_size, batch))) {
      return fail(GFXI_INVALID_ARGUMENT, "logit rule workspace is null, not 8-byte aligned or too small");
    }
    const uint32_t slices = slice_count(vocabulary_size, batch);
    if (static_cast<uint64_t>(slices) * batch >= (1u << 23)) {
      return fail(GFXI_INVALID_ARGUMENT, "logit rules over too many rows for one launch");
    }
    RulesArgs a{};
    a.rules = r;
    a.logits = logits;
    a.output = output;
    a.keys = tokens != nullptr ? static_cast<unsigned long long*>(workspace) : nullptr;
    a.row_stride = row_stride;
    a.output_stride = output_stride;
    a.vocabulary = static_cast<uint32_t>(vocabulary_size);
    a.slices = slices;
    const hipStream_t st = static_cast<hipStream_t>(stream);
    const auto whole = [](const float* p, size_t stride) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0 && stride % 4 == 0; };
    const bool vec = whole(logits, row_stride) && (output == nullptr || whole(output, output_stride));
    const dim3 grid(slices * batch), block(kThreads);
    if (slice_of(vocabulary_size, batch) == kLarge) {
      if (vec) hipLaunchKernelGGL((logit_rules_kernel<kLarge, true>), grid, block, 0, st, a);
      else hipLaunchKernelGGL((logit_rules_kernel<kLarge, false>), grid, block, 0, st, a);
    } else if (vec) {
      hipLaunchKernelGGL((logit_rules_kernel<kSmall, true>), grid, block, 0, st, a);
    } else {
      hipLaunchKernelGGL((logit_rules_kernel<kSmall, false>), grid, block, 0, st, a);
    }
    if (const int32_t s = launch_status("logit rules launch failed"); s != GFXI_OK || tokens == nullptr) return s;
    hipLaunchKernelGGL(rule_tokens_kernel, dim3(batch), dim3(kThreads), 0, st, a.keys, slices, tokens);
    return launch_status("logit rule argmax launch failed");
  });
}
