// Prompts packed one behind another: which prompt, and which part of it, a workgroup has.
//
// starts [S + 1] lies on the device, so the host knows the number of rows and of prompts and no length:
// a launch has a workgroup for as many parts as such prompts can have at most, and each finds its own
// from the starts, 64 prompts at a time. Rows in front of the first start and behind the last are spans
// of their own (the first and the last one), so that every row belongs to one.
#pragma once

#include "lq_common.h"

namespace lq {

struct Spans {
  const void* starts;  // int32 or int64; nullptr: S spans of `rows` rows each (a batch)
  int is64;
  int S;
  int rows;  // rows in all, or of each batch row
};

struct Span {
  int index;  // prompt, or batch row
  int begin;  // first row (0 in a batch)
  int len;
  int part;    // the part of this span
  int before;  // slots of the spans in front of this one
  bool gap;    // rows of no prompt
};

// Starts are taken as they come, but never outside [0, rows].
__device__ __forceinline__ int span_bound(const Spans& s, int i) {
  if (i <= 0) return 0;
  if (i > s.S + 1) return s.rows;
  const int64_t v = s.is64 ? ((const int64_t*)s.starts)[i - 1] : ((const int32_t*)s.starts)[i - 1];
  return (int)(v < 0 ? 0 : v > s.rows ? s.rows : v);
}

__device__ __forceinline__ int wave_prefix_sum(int v, int lane) {
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const int up = __shfl_up(v, o, 64);
    if (lane >= o) v += up;
  }
  return v;
}

// The span and part behind t parts; false where there are not so many. parts(len, gap) gives a span's
// number, slots(len, gap) another one that is summed. Every lane of a wave calls it with the same t.
template <class F, class G>
__device__ __forceinline__ bool find_span(const Spans& s, int t, F&& parts, G&& slots, Span& out) {
  if (s.starts == nullptr) {
    const int n = parts(s.rows, false);
    if (n == 0 || t >= n * s.S) return false;
    out.index = t / n;
    out.part = t - out.index * n;
    out.begin = 0;
    out.len = s.rows;
    out.before = out.index * slots(s.rows, false);
    out.gap = false;
    return true;
  }
  const int lane = (int)(threadIdx.x & 63);
  int run = 0, behind = 0;
  for (int base = 0; base < s.S + 2; base += 64) {
    const int i = base + lane;
    int begin = 0, len = 0;
    if (i < s.S + 2) {
      begin = span_bound(s, i);
      len = max(span_bound(s, i + 1) - begin, 0);
    }
    const bool gap = i == 0 || i >= s.S + 1;
    const int n = parts(len, gap);
    const int upto = wave_prefix_sum(n, lane);
    const int own_slots = slots(len, gap), later = wave_prefix_sum(own_slots, lane);
    const uint64_t have = __ballot(t < run + upto);
    if (have != 0) {
      const int l = __builtin_ctzll(have);
      out.index = base + l - 1;
      out.begin = __builtin_amdgcn_readlane(begin, l);
      out.len = __builtin_amdgcn_readlane(len, l);
      const int own = __builtin_amdgcn_readlane(n, l);
      out.part = t - (run + __builtin_amdgcn_readlane(upto, l) - own);
      out.gap = out.index < 0 || out.index >= s.S;
      out.before = behind + __builtin_amdgcn_readlane(later, l) - __builtin_amdgcn_readlane(own_slots, l);
      return true;
    }
    run += __builtin_amdgcn_readlane(upto, 63);
    behind += __builtin_amdgcn_readlane(later, 63);
  }
  return false;
}

template <class F>
__device__ __forceinline__ bool find_span(const Spans& s, int t, F&& parts, Span& out) {
  return find_span(s, t, parts, [](int, bool) { return 0; }, out);
}

// host: validates `starts` (NULL, or int32/int64 [S + 1]) against packed rows
int make_spans(const lq_tensor* starts, int64_t batch, int64_t rows, Spans& out);

}  // namespace lq
