// What the kernels of prompt_attention.hip and prompt_attention_mfma.hip are launched with.
#pragma once

#include <math.h>

#include "prompt_spans.h"

namespace lq {

constexpr int PROMPT_ATTENTION_MAX_D = 256;

struct PromptAttention {
  View q, k, v, out;  // strides of (batch row, row, head, dim)
  Spans spans;
  int Hkv, nrep, D;
  float scale;  // log2(e) times the caller's
  uint32_t q_and, q_xor;  // on pairs of 16-bit query values: the scale's sign, and zeros for scale 0
};

constexpr int PROMPT_ATTENTION_WAVES = 4;  // of a workgroup, 32 rows each

// The prompt and part of it (rows x query heads of a KV head) of workgroup t of a KV head.
__device__ __forceinline__ bool find_part(const PromptAttention& p, int t, Span& out) {
  constexpr int ROWS = 32 * PROMPT_ATTENTION_WAVES;
  const int nrep = p.nrep;
  return find_span<true>(
      p.spans, t, [=](int len, bool) { return (len * nrep + ROWS - 1) / ROWS; },
      [=](int begin, int i) { return begin * nrep / ROWS + i; }, out);
}

// In a workgroup's second run the weights are this much smaller, so that no sum of 2^30 values, each weighed 2^8
// at most, leaves fp32 where the result does not. What is a power of two rounds alike, down to weights of 2^-86.
constexpr float PROMPT_ATTENTION_DOWN = 0x1p-40f;

// The 16-bit kernel (prompt_attention_mfma.hip): whether the tensors are in its form, and its launch,
// whose scale is positive.
bool prompt_attention_mfma_fits(const lq_tensor* q, const lq_tensor* k, const lq_tensor* v,
                                const lq_tensor* out);
int launch_prompt_attention_mfma(const PromptAttention& p, int dtype, int64_t parts, hipStream_t st);

}  // namespace lq
