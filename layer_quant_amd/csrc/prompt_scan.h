// What the kernels of prompt_scan.hip and prompt_scan_mfma.hip are launched with.
#pragma once

#include <math.h>

#include "prompt_spans.h"

namespace lq {

constexpr int PROMPT_SCAN_MAX_N = 256;

struct PromptScan {
  View x, B, C, z, out;  // strides of (batch row, row, head or group, index)
  View dt;               // strides of (batch row, row, head)
  View A, D, bias;       // strides of (head)
  View initial, states;  // strides of (prompt, head, p, n)
  Spans spans;
  int H, P, N, ratio;  // ratio: heads per group
  int segment;         // rows of a segment
  int slots;           // of the workspace
  int softplus;
  float dt_min, dt_max;
  float* slot_state;  // [slots][H][P][N]: the state behind a segment that others of its prompt follow
  float* slot_log;    // [slots][H]: log2 of the decay over it
};

// The matrix kernel (prompt_scan_mfma.hip): whether the call is in its form, and the launch of `parts`
// segments.
bool prompt_scan_mfma_fits(const lq_tensor* x, const lq_tensor* B, const lq_tensor* C,
                           const lq_tensor* z, const lq_tensor* initial, const lq_tensor* states,
                           const lq_tensor* out);
void launch_prompt_scan_mfma(const PromptScan& p, bool followed, int64_t parts, hipStream_t st);

// Segments of a prompt (an empty one has one, which hands its state on), and those that others follow.
__device__ __forceinline__ int segments_of(const PromptScan& p, int len, bool gap) {
  return max((len + p.segment - 1) / p.segment, gap ? 0 : 1);
}
__device__ __forceinline__ int followed_segments_of(const PromptScan& p, int len, bool gap) {
  return gap ? 0 : segments_of(p, len, gap) - 1;
}

// log(1 + e^x) with its small values as exact as its large ones
__device__ __forceinline__ float scan_softplus(float x) {
  return fmaxf(x, 0.f) + log1pf(expf(-fabsf(x)));
}

// A NaN step stays one (fminf and fmaxf drop it).
__device__ __forceinline__ float scan_step(const PromptScan& p, float dt, float bias) {
  dt += bias;
  if (p.softplus) dt = scan_softplus(dt);
  return dt < p.dt_min ? p.dt_min : dt > p.dt_max ? p.dt_max : dt;
}

__device__ __forceinline__ float scan_silu(float z) { return z / (1.f + __expf(-z)); }

}  // namespace lq
