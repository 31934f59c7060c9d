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
  int slots_by_rows;   // slot_of's
  int softplus;
  float dt_min, dt_max;
  float* slot_state;  // [slots][H][P][N]: the state in front of each segment of a prompt that has several
  float* slot_log;    // [slots][H]: log2 of the decay over the segment in front of it
  float* steps;       // the matrix kernel's decays and steps, [4][H][rows]
  int64_t rows;       // in all
};

// The matrix kernel (prompt_scan_mfma.hip): whether a geometry, and a call, is in its form, the bytes of
// its steps, and the launches of the steps of `chunks` chunks of 64 rows and of `parts` segments (adds:
// find_segment's).
bool prompt_scan_mfma_geometry(int dtype, int64_t heads, int64_t head_dim, int64_t dstate);
bool prompt_scan_mfma_fits(const lq_tensor* x, const lq_tensor* B, const lq_tensor* C,
                           const lq_tensor* z, const lq_tensor* initial, const lq_tensor* states,
                           const lq_tensor* out);
size_t prompt_scan_mfma_workspace(int64_t rows, int64_t heads);
void launch_prompt_scan_steps(const PromptScan& p, int64_t chunks, hipStream_t st);
void launch_prompt_scan_mfma(const PromptScan& p, bool adds, int64_t parts, hipStream_t st);

// Segments of a prompt (an empty one has one, which hands its state on), and its slots: one for each of
// several segments. With many prompts the first slot of one (find_span's first_slot) is floor(begin / segment) +
// its number, or with many of a segment or less, which need none, floor(2 begin / segment): 2 len / segment whole
// ones are ceil(len / segment) or more where len > segment.
__device__ __forceinline__ int segments_of(const PromptScan& p, int len, bool gap) {
  return max((len + p.segment - 1) / p.segment, gap ? 0 : 1);
}
__device__ __forceinline__ int slots_of_prompt(const PromptScan& p, int len) {
  const int n = segments_of(p, len, false);
  return n < 2 ? 0 : n;
}
__device__ __forceinline__ int slot_of(const PromptScan& p, int begin, int i) {
  return p.slots_by_rows ? 2 * begin / p.segment : begin / p.segment + i;
}

// The segment of a workgroup. ADDS: what each segment but the last of a prompt adds by itself (t: the slot
// of the segment, which goes to the next one), else all segments.
struct Segment {
  Span span;
  int slot;    // its own: the state in front of it
  bool several;
  bool valid;
};
template <bool ADDS>
__device__ __forceinline__ Segment find_segment(const PromptScan& p, int t) {
  Segment s;
  const auto slots = [&](int len) { return slots_of_prompt(p, len); };
  const auto first_slot = [&](int begin, int i) { return slot_of(p, begin, i); };
  if (ADDS) {
    s.valid = find_span<false>(
        p.spans, t, [&](int len, bool) { return slots(len); }, first_slot, slots, first_slot, s.span);
  } else {
    s.valid = find_span<true>(
        p.spans, t, [&](int len, bool gap) { return segments_of(p, len, gap); },
        [&](int begin, int i) { return begin / p.segment + i; }, slots, first_slot, s.span);
  }
  if (!s.valid || s.span.gap) return s;
  const int n = segments_of(p, s.span.len, false);
  s.several = n > 1;
  s.slot = s.span.slots + s.span.part;
  // the last one adds to nothing; starts out of order can ask for more slots than there are
  if (ADDS ? s.span.part == n - 1 || s.slot + 1 >= p.slots : s.several && s.slot >= p.slots) s.valid = false;
  return s;
}

// log(1 + e^x), its small values as exact as its large ones: with u = e^-|x| and s = u / (2 + u) <= 1/3,
// log(1 + u) = 2 (s + s^3 / 3 + s^5 / 5 + ...), the terms behind s^15 below 2^-28 of it.
__device__ __forceinline__ float scan_softplus(float x) {
  const float u = expf(-fabsf(x)), s = u * __builtin_amdgcn_rcpf(2.f + u), s2 = s * s;
  float r = 1.f / 15;
  r = fmaf(r, s2, 1.f / 13);
  r = fmaf(r, s2, 1.f / 11);
  r = fmaf(r, s2, 1.f / 9);
  r = fmaf(r, s2, 1.f / 7);
  r = fmaf(r, s2, 1.f / 5);
  r = fmaf(r, s2, 1.f / 3);
  r = fmaf(r, s2, 1.f);
  return fmaxf(x, 0.f) + 2.f * s * r;
}

// A NaN step stays one (fminf and fmaxf drop it).
__device__ __forceinline__ float scan_step(const PromptScan& p, float dt, float bias) {
  dt += bias;
  if (p.softplus) dt = scan_softplus(dt);
  return dt < p.dt_min ? p.dt_min : dt > p.dt_max ? p.dt_max : dt;
}

__device__ __forceinline__ float scan_silu(float z) { return z * __builtin_amdgcn_rcpf(1.f + __expf(-z)); }

}  // namespace lq
