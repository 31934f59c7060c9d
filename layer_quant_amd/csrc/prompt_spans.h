// Prompts packed one behind another: which prompt, and which part of it, a workgroup has.
//
// starts [S + 1] lies on the device, so the host knows the number of rows and of prompts and no length:
// a launch has a workgroup for as many parts as such prompts can have at most, and each finds its own
// from the starts. Span i, of the rows b to e, begins at part floor(b / rows of a part) + i: a number that
// grows by as many parts as the span can have, as floor(e / n) + 1 - floor(b / n) >= ceil((e - b) / n), and
// that needs no other span's length. So a workgroup searches the starts, 64 at a time in a wave's lanes: one
// round for up to 64 spans, four for 2^24. (A sum of the parts of all spans in front took a round per 64
// spans in every workgroup.) Rows in front of the first start and behind the last are spans of their own
// (the first and the last one), so that every row belongs to one.
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
  int part;  // the part of this span
  bool gap;  // rows of no prompt
};

// Starts are taken as they come, but never outside [0, rows].
__device__ __forceinline__ int span_bound(const Spans& s, int i) {
  if (i <= 0) return 0;
  if (i > s.S + 1) return s.rows;
  const int64_t v = s.is64 ? ((const int64_t*)s.starts)[i - 1] : ((const int32_t*)s.starts)[i - 1];
  return (int)(v < 0 ? 0 : v > s.rows ? s.rows : v);
}

// The span and part of workgroup t; false where it has none. parts(len, gap): the parts of a span;
// first(begin, i): the workgroup of its first one, i the span's number. GAPS: the rows of no prompt are spans,
// too. Every lane of a wave calls it with the same t. Starts out of order give any span, and a part of it.
template <bool GAPS, class F, class G>
__device__ __forceinline__ bool find_span(const Spans& s, int t, F&& parts, G&& first, Span& out) {
  if (s.starts == nullptr) {
    const int n = parts(s.rows, false);
    if (n == 0 || t >= n * s.S) return false;
    out.index = t / n;
    out.part = t - out.index * n;
    out.begin = 0;
    out.len = s.rows;
    out.gap = false;
    return true;
  }
  const int lane = (int)(threadIdx.x & 63), before = GAPS ? 0 : 1;
  int at = 0, n = GAPS ? s.S + 2 : s.S;  // the span is one of n from `at` on
  while (n > 0) {
    const int step = (n + 63) >> 6, i = at + lane * step;
    int begin = 0, end = 0;
    bool reached = false;
    if (lane * step < n) {
      begin = span_bound(s, i + before);
      end = span_bound(s, i + before + 1);
      reached = first(begin, i) <= t;
    }
    const uint64_t not_yet = ~__ballot(reached);
    const int k = (not_yet == 0 ? 64 : __builtin_ctzll(not_yet)) - 1;
    if (k < 0) return false;
    at += k * step;
    if (step > 1) {
      n = min(step, n - k * step);
      continue;
    }
    out.index = at - 1 + before;
    out.begin = __builtin_amdgcn_readlane(begin, k);
    out.len = max(__builtin_amdgcn_readlane(end, k) - out.begin, 0);
    out.part = t - first(out.begin, at);
    out.gap = out.index < 0 || out.index >= s.S;
    return out.part >= 0 && out.part < parts(out.len, out.gap);
  }
  return false;
}

// host: validates `starts` (NULL, or int32/int64 [S + 1]) against packed rows
int make_spans(const lq_tensor* starts, int64_t batch, int64_t rows, Spans& out);

}  // namespace lq
