// Prompts packed one behind another: which prompt, and which part of it, a workgroup has.
//
// starts [S + 1] lies on the device, so the host knows the number of rows and of prompts and no length:
// a launch has a workgroup for as many parts as such prompts can have at most, and each finds its own
// from the starts. Rows in front of the first start and behind the last are spans of their own (the first
// and the last one), so that every row belongs to one.
//
// Up to 512 spans, every workgroup sums the parts of the spans in front of its own, 64 at a time in a wave's
// lanes. Of more, span i, of the rows b to e, begins at part floor(b / rows of a part) + i: a number that grows
// by as many parts as the span can have, as floor(e / n) + 1 - floor(b / n) >= ceil((e - b) / n), and that needs
// no other span's length. So a workgroup searches the starts, 64 at a time: two rounds for 4096 spans, four for
// 2^24. (4000 prompts of 10 rows, attention of 32 heads: 2300 us by sums, 471 by the search; 600 of 64 rows 285 and
// 203.) The search leaves gaps between the spans' parts, workgroups that end at once. Where there are fewer than
// the GPU takes at a time they are dealt out in turn, gaps and all, and some CUs get more work than others: 4
// prompts of 512 rows, the recurrence of 128 heads 59 us against 50, 200 of 64 rows and 8 heads 72 against 49.
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
  int part;   // the part of this span
  int slots;  // of the spans in front of this one
  bool gap;   // rows of no prompt
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

// find_span's by the sums over the spans in front.
template <bool GAPS, class P, class S>
__device__ __forceinline__ bool walk_spans(const Spans& s, int t, P&& parts, S&& slots, Span& out) {
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
    const int n = i >= s.S + 2 || (gap && !GAPS) ? 0 : parts(len, gap), own_slots = gap ? 0 : slots(len);
    const int upto = wave_prefix_sum(n, lane), slots_upto = wave_prefix_sum(own_slots, lane);
    const uint64_t have = __ballot(t < run + upto);
    if (have != 0) {
      const int l = __builtin_ctzll(have);
      out.index = base + l - 1;
      out.begin = __builtin_amdgcn_readlane(begin, l);
      out.len = __builtin_amdgcn_readlane(len, l);
      out.part = t - run - __builtin_amdgcn_readlane(upto - n, l);
      out.slots = behind + __builtin_amdgcn_readlane(slots_upto - own_slots, l);
      out.gap = out.index < 0 || out.index >= s.S;
      return true;
    }
    run += __builtin_amdgcn_readlane(upto, 63);
    behind += __builtin_amdgcn_readlane(slots_upto, 63);
  }
  return false;
}

// The span and part of workgroup t; false where it has none. parts(len, gap): the parts of a span;
// first(begin, i): an upper bound of the parts of the i spans in front, as above. slots and first_slot: the same
// of another number, of prompts alone. GAPS: the rows of no prompt are spans, too. Every lane of a wave calls
// it with the same t. Starts out of order give any span, and a part of it.
template <bool GAPS, class P, class F, class S, class G>
__device__ __forceinline__ bool find_span(const Spans& s, int t, P&& parts, F&& first, S&& slots, G&& first_slot,
                                          Span& out) {
  if (s.starts == nullptr) {
    const int n = parts(s.rows, false);
    if (n == 0 || t >= n * s.S) return false;
    out.index = t / n;
    out.part = t - out.index * n;
    out.slots = out.index * slots(s.rows);
    out.begin = 0;
    out.len = s.rows;
    out.gap = false;
    return true;
  }
  if (s.S + 2 <= 512) return walk_spans<GAPS>(s, t, parts, slots, out);
  const int lane = (int)(threadIdx.x & 63);
  const int before = GAPS ? 0 : 1;
  int at = 0, n = GAPS ? s.S + 2 : s.S;  // the span is one of n from `at` on
  for (;;) {
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
    out.slots = first_slot(out.begin, out.index);
    out.gap = out.index < 0 || out.index >= s.S;
    return out.part >= 0 && out.part < parts(out.len, out.gap);
  }
}

template <bool GAPS, class P, class F>
__device__ __forceinline__ bool find_span(const Spans& s, int t, P&& parts, F&& first, Span& out) {
  return find_span<GAPS>(s, t, parts, first, [](int) { return 0; }, [](int, int) { return 0; }, out);
}

// host: validates `starts` (NULL, or int32/int64 [S + 1]) against packed rows
int make_spans(const lq_tensor* starts, int64_t batch, int64_t rows, Spans& out);

}  // namespace lq
