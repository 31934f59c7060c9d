// Log-probabilities of given tokens, the entropy of each row and its likeliest tokens (no reference
// counterpart; beam_select.hip selects over beams and vocabulary by the same log-softmax):
//
//   lse = log sum_v exp(l_v),  logprob = l_token - lse,  entropy = lse - sum_v p_v l_v
//
// One pass over the logits. A thread takes 32 logits at a time, in 16-byte loads (rows that begin off that
// alignment: from the aligned address in front of them), and keeps m = max l, s = sum 2^z and
// t = sum 2^z z, z = l log2(e) - m log2(e), of its own: nothing is exchanged before the row's end. Every z is
// made from the rounded m log2(e) by one fused multiply-add, the given token's too, so that its rounding falls
// out of logprob and entropy. From |m| = 2^29 on, where that rounding would reach 32 and more, other logits are 32
// or more below m: z is a power of two times l - m there, and their weights, right or not, are 2^-64 and less
// of the largest one's. fp32 sums: a thread adds 8 terms in a row four times over, then the threads in a tree.
// The likeliest tokens: the k-th largest of a wave's 64 lane maxima is a limit that k logits reach, and the
// largest of the waves' limits is the workgroup's. The logits that reach it are few (tens of 8192 random
// ones for k = 8) and go to the wave's list; a full list is cut to its k largest, by ballots, bit by bit from
// the highest in which its keys differ, and that raises the limit. At the end the lists are put in order by
// rank, up to 64 keys as they are, more behind one such cut.
//
// Which form: with 512 rows or more, or 32761 logits or less, a workgroup per row writes the results (256
// threads, or 1024 where one sweep of theirs covers the row); else each 8192 logits are a workgroup's, and
// a wave per row joins the parts, a second launch. One workgroup of 1024 threads over several sweeps instead of
// the parts: 37 rows of 50257 fp32 logits 17.8 us against 16.5.
//
// What it measured (MI355X, us per call, kernel time in brackets): 2048 rows of 131072 bf16 logits 97 (95-96, 5.5
// TB/s: a device copy's rate), with 8 or 32 tokens each 147-150; 64 rows, 8 tokens 16.6 (11.2-11.7 + 5.0);
// 37 rows of 50257 fp32, 20 tokens 17.1 (11-11.6 + 6.4); one row of 32000, 5 tokens 12.2 (10.7; the host's part is
// 12). The small ones are bound by the latency of their dependent steps: load, limit, list, order. Rows whose limit
// holds few logits back, 8 tokens each: all but ten masked 47 (64 rows) and 184 (2048), equal logits 66 and 1380.
//
// Order: the larger logit first, of equal ones (and of 0 and -0) the lower token. -inf logits have no
// part in the sums. A row with a NaN or an infinity, or with -inf alone, has no distribution: NaN.
#include <math.h>

#include "lq_common.h"

namespace lq {
namespace {

constexpr int VPT = 32;                   // logits of a thread and sweep
constexpr int NARROW = 256, WIDE = 1024;  // threads of a workgroup
constexpr int MAX_TOP = 32;
constexpr int LIST = 256;  // entries of a wave's list, 4 per lane
constexpr float LOG2E = 1.44269504088896340736f, LN2 = 0.69314718055994530942f;

struct Sums {
  float m, s, t;
};

// z = l factor - base of a maximum m.
struct Scale {
  float factor, base;
};
__device__ __forceinline__ Scale scale_of(float m) {
  const float factor = fabsf(m) < 0x1p29f ? LOG2E : fabsf(m) < 0x1p100f ? 2.f : 1.f;
  return {factor, m == -INFINITY ? 0.f : m * factor};
}

struct LogprobParams {
  View logits;  // strides of (batch row, row, token)
  View tokens;  // strides of (batch row, row)
  float *logprobs, *entropy, *top_logprobs;
  int64_t* top_tokens;
  int rows, parts, top, len;  // len: rows of a batch row
  int part;                   // logits of a part
  int64_t V;
  Sums* sums;      // [rows][parts]
  uint64_t* keys;  // [rows][parts][top]; 0: none
};

// Larger for the logit that comes first: its bits in order, then the lower token. Never 0.
__device__ __forceinline__ uint32_t order_of(float l) {
  const uint32_t u = __float_as_uint(l + 0.f);
  return (u >> 31) ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float logit_of(uint32_t order) {
  return __uint_as_float((order >> 31) ? order & 0x7fffffffu : ~order);
}

__device__ __forceinline__ int count(uint64_t ballot) { return __builtin_popcountll(ballot); }
__device__ __forceinline__ int below(uint64_t ballot) {
  return __builtin_amdgcn_mbcnt_hi((uint32_t)(ballot >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)ballot, 0));
}

// op over the wave's lanes: rotations within rows of 16, then the four rows.
template <class F>
__device__ __forceinline__ uint32_t wave_fold(uint32_t v, F op) {
  v = op(v, __builtin_amdgcn_update_dpp(0, v, 0x128, 0xf, 0xf, false));
  v = op(v, __builtin_amdgcn_update_dpp(0, v, 0x124, 0xf, 0xf, false));
  v = op(v, __builtin_amdgcn_update_dpp(0, v, 0x122, 0xf, 0xf, false));
  v = op(v, __builtin_amdgcn_update_dpp(0, v, 0x121, 0xf, 0xf, false));
  return op(op(__builtin_amdgcn_readlane(v, 0), __builtin_amdgcn_readlane(v, 16)),
            op(__builtin_amdgcn_readlane(v, 32), __builtin_amdgcn_readlane(v, 48)));
}

// A word that `need` or more of the wave's 64 E words (0: none) reach, and of those that many do the largest
// or one that exactly `need` reach; 0 where there are fewer. Bit by bit from the highest in which the
// words differ.
template <int E>
__device__ __forceinline__ uint32_t kth_word(const uint32_t (&v)[E], int need) {
  uint32_t some = 0, every = ~0u;
  int words = 0;
#pragma unroll
  for (int e = 0; e < E; ++e) {
    some |= v[e];
    every &= v[e] == 0 ? ~0u : v[e];
    words += count(__ballot(v[e] != 0));
  }
  if (words < need) return 0;
  some = wave_fold(some, [](uint32_t x, uint32_t y) { return x | y; });
  uint32_t w = wave_fold(every, [](uint32_t x, uint32_t y) { return x & y; });
  uint32_t differ = some & ~w;
#pragma unroll 1
  while (differ != 0) {
    const uint32_t bit = 0x80000000u >> __builtin_clz(differ);
    differ ^= bit;
    int c = 0;
#pragma unroll
    for (int e = 0; e < E; ++e) c += count(__ballot(v[e] >= (w | bit)));
    if (c >= need) w |= bit;
    if (c == need) break;
  }
  return w;
}

// The wave's 64 E keys (0: none) reduced to the `top` largest: whether each is one of them.
template <int E>
__device__ __forceinline__ uint32_t select_top(const uint32_t (&hi)[E], const uint32_t (&lo)[E], int top) {
  const uint32_t w = kth_word(hi, top);
  uint32_t in = 0;
  int reach = 0, more = 0;
#pragma unroll
  for (int e = 0; e < E; ++e) {
    reach += count(__ballot(hi[e] >= w && hi[e] != 0));
    more += count(__ballot(hi[e] > w));
    in |= (uint32_t)(hi[e] >= w && hi[e] != 0) << e;
  }
  if (reach <= top) return in;
  // too many of equal logits: of those, the ones with the lowest tokens
  uint32_t tie[E];
#pragma unroll
  for (int e = 0; e < E; ++e) tie[e] = hi[e] == w ? lo[e] : 0;
  const uint32_t last = kth_word(tie, top - more);
#pragma unroll
  for (int e = 0; e < E; ++e) {
    if (hi[e] == w && lo[e] < last) in &= ~(1u << e);
  }
  return in;
}

// Orders a wave's reads of its list behind the other lanes' writes.
__device__ __forceinline__ void wave_fence() { __builtin_amdgcn_fence(__ATOMIC_SEQ_CST, "wavefront"); }

// Cuts a wave's list of n keys to its `top` largest; returns how many there are.
__device__ __forceinline__ int cut_list(uint2* list, int n, int top, int lane) {
  wave_fence();
  if (n <= top) return n;
  uint32_t hi[LIST / 64], lo[LIST / 64];
#pragma unroll
  for (int e = 0; e < LIST / 64; ++e) {
    const uint2 k = 64 * e + lane < n ? list[64 * e + lane] : make_uint2(0, 0);
    hi[e] = k.y;
    lo[e] = k.x;
  }
  const uint32_t in = select_top(hi, lo, top);
  int at = 0;
#pragma unroll
  for (int e = 0; e < LIST / 64; ++e) {
    const uint64_t some = __ballot((in >> e) & 1);
    if ((in >> e) & 1) list[at + below(some)] = make_uint2(lo[e], hi[e]);
    at += count(some);
  }
  wave_fence();
  return at;
}

// The `top` largest of a list of n <= 64 E keys, one per lane and in order: lane k has the k-th (0: none).
template <int E>
__device__ __forceinline__ uint64_t sort_list(uint2* list, int n, int top, int lane) {
  wave_fence();
  if (n > 64) {
    uint32_t hi[E], lo[E];
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const uint2 k = 64 * e + lane < n ? list[64 * e + lane] : make_uint2(0, 0);
      hi[e] = k.y;
      lo[e] = k.x;
    }
    // the equal ones at the end may stay, as long as a lane is there for each
    const uint32_t w = kth_word(hi, top);
    uint32_t in = 0;
    int reach = 0;
#pragma unroll
    for (int e = 0; e < E; ++e) {
      reach += count(__ballot(hi[e] >= w));
      in |= (uint32_t)(hi[e] >= w) << e;
    }
    if (reach > 64) in = select_top(hi, lo, top);
    n = 0;
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const uint64_t some = __ballot((in >> e) & 1);
      if ((in >> e) & 1) list[n + below(some)] = make_uint2(lo[e], hi[e]);
      n += count(some);
    }
    wave_fence();
  }
  const uint2 k = lane < n ? list[lane] : make_uint2(0, 0);
  int rank = 0;
#pragma unroll 1
  for (int i = 0; i < n; ++i) {
    const uint32_t lo = __builtin_amdgcn_readlane(k.x, i), hi = __builtin_amdgcn_readlane(k.y, i);
    rank += hi > k.y || (hi == k.y && lo > k.x);
  }
  wave_fence();
  if (lane < n && rank < 64) list[rank] = k;
  wave_fence();
  const uint2 sorted = lane < min(n, top) ? list[lane] : make_uint2(0, 0);
  return ((uint64_t)sorted.y << 32) | sorted.x;
}

// Sums over another maximum: z' = z + d. (Where a factor is not log2(e) another maximum is 32 or more
// away, and what has it nothing beside the larger one.)
__device__ __forceinline__ Sums moved(Sums v, float to) {
  const Scale from = scale_of(v.m), next = scale_of(to);
  const bool near = from.factor == LOG2E && next.factor == LOG2E;
  const float d = v.m == to ? 0.f : near ? fmaxf(from.base - next.base, -200.f) : -200.f;
  const float w = __builtin_amdgcn_exp2f(d);
  return {to, w * v.s, w * fmaf(d, v.s, v.t)};
}
__device__ __forceinline__ Sums wave_sums(Sums v) {
  v = moved(v, group_max<64>(v.m));
  v.s = group_sum<64>(v.s);
  v.t = group_sum<64>(v.t);
  return v;
}

__device__ __forceinline__ int64_t row_at(const LogprobParams& p, int row) {
  const int b = row / p.len;
  return b * p.logits.s[0] + (row - b * p.len) * p.logits.s[1];
}

// A row's results from its sums and, in one wave's registers, its `top` largest keys (lane k: the k-th).
__device__ __forceinline__ void put_row(const LogprobParams& p, int row, Sums v, uint64_t key, int lane) {
  const Scale scale = scale_of(v.m);
  const float log2s = __builtin_amdgcn_logf(v.s);
  const bool known = v.s > 0.f && v.s < INFINITY && v.m < INFINITY;
  const float nan = __builtin_nanf("");
  const auto logprob_of = [&](float l) {
    const float z = fmaf(l, scale.factor, -scale.base);
    // (far below the maximum z can leave fp32 where l - m does not)
    if (scale.factor != LOG2E || z < -0x1p100f) return (l - v.m) - log2s * LN2;
    return (z - log2s) * LN2;
  };
  if (lane == 0) {
    const int b = row / p.len;
    const int64_t token = ((const int64_t*)p.tokens.data)[b * p.tokens.s[0] + (row - b * p.len) * p.tokens.s[1]];
    float lp = 0.f;
    if (token >= 0 && token < p.V) {
      const float l = load_float(p.logits.data, p.logits.dtype, row_at(p, row) + token * p.logits.s[2]);
      lp = known ? logprob_of(l) : nan;
    }
    p.logprobs[row] = lp;
    if (p.entropy != nullptr) p.entropy[row] = known ? LN2 * (log2s - v.t / v.s) : nan;
  }
  if (lane < p.top) {
    // (a row that is not known can hold logits that are not numbers, and its order is not one)
    const int64_t at = (int64_t)row * p.top + lane;
    p.top_logprobs[at] = known ? logprob_of(logit_of((uint32_t)(key >> 32))) : nan;
    p.top_tokens[at] = known ? (int64_t)(0xffffffffu - (uint32_t)key) : lane;
  }
}

// The 32 logits of a thread's sweep from logit `from` on (a multiple of a load's behind the row's aligned
// beginning), -inf outside [lo, hi). Element i of load j is logit from + j * THREADS * W + tid * W + i.
template <int DTYPE, int THREADS, bool ROWS>
__device__ __forceinline__ void load_logits(const LogprobParams& p, int64_t row, int64_t from, int64_t lo,
                                            int64_t hi, int tid, float (&x)[VPT]) {
  constexpr int W = DTYPE == LQ_F32 ? 4 : 8, SIZE = DTYPE == LQ_F32 ? 4 : 2;
  uint4 raw[VPT / W];
#pragma unroll
  for (int j = 0; j < VPT / W; ++j) {
    const int64_t at = from + (int64_t)j * THREADS * W + tid * W;
    if (ROWS) {
      raw[j] = make_uint4(0, 0, 0, 0);
      if (at + W > lo && at < hi) raw[j] = *(const uint4*)((const char*)p.logits.data + (row + at) * SIZE);
    } else {
#pragma unroll
      for (int i = 0; i < W; ++i) {
        x[j * W + i] = at + i >= lo && at + i < hi
                           ? load_float(p.logits.data, DTYPE, row + (at + i) * p.logits.s[2])
                           : -INFINITY;
      }
    }
  }
  if (!ROWS) return;
#pragma unroll
  for (int j = 0; j < VPT / W; ++j) {
    const uint32_t w[4] = {raw[j].x, raw[j].y, raw[j].z, raw[j].w};
#pragma unroll
    for (int i = 0; i < W; ++i) {
      x[j * W + i] = SIZE == 4 ? __uint_as_float(w[i & 3]) : word_elem(w[i >> 1], (i & 1) * 16, DTYPE);
    }
    const int64_t at = from + (int64_t)j * THREADS * W + tid * W;
    if (at < lo || at + W > hi) {
#pragma unroll
      for (int i = 0; i < W; ++i) {
        if (at + i < lo || at + i >= hi) x[j * W + i] = -INFINITY;
      }
    }
  }
}

// A row, or a part of it. ROWS: its logits lie one behind another.
template <int DTYPE, int THREADS, bool ROWS>
__global__ __launch_bounds__(THREADS) void logprob_kernel(LogprobParams p) {
  constexpr int WAVES = THREADS / 64, SWEEP = THREADS * VPT;
  constexpr int W = DTYPE == LQ_F32 ? 4 : 8, SIZE = DTYPE == LQ_F32 ? 4 : 2;
  __shared__ Sums sums[WAVES];
  __shared__ uint2 lists[WAVES][LIST];
  __shared__ uint2 joined[512];
  __shared__ int counts[WAVES];
  __shared__ uint32_t reached;  // the order of a logit that `top` logits of a wave reach
  const int row = blockIdx.x / p.parts, part = blockIdx.x % p.parts;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int64_t base = row_at(p, row);
  // parts lie between aligned addresses, the first one's at or in front of the row's beginning
  const int skew = ROWS ? (int)(((uintptr_t)p.logits.data + (uintptr_t)(base * SIZE)) & 15) / SIZE : 0;
  int64_t from = (int64_t)part * p.part - skew;
  const int64_t lo = max(from, (int64_t)0), hi = min(p.V, from + p.part);
  Sums v = {-INFINITY, 0.f, 0.f};
  float limit = -INFINITY;  // `top` logits of the part reach it
  int listed = 0;
  uint2* list = lists[wave];
  if (p.top > 0) {
    if (tid == 0) reached = 0;
    __syncthreads();
  }
  for (int sweep = 0; from < hi; ++sweep, from += SWEEP) {
    float x[VPT];
    load_logits<DTYPE, THREADS, ROWS>(p, base, from, lo, hi, tid, x);
    float most[4] = {x[0], x[1], x[2], x[3]};
#pragma unroll
    for (int i = 4; i < VPT; ++i) most[i & 3] = fmaxf(most[i & 3], x[i]);
    const float top_l = fmaxf(fmaxf(most[0], most[1]), fmaxf(most[2], most[3]));
    v = moved(v, fmaxf(v.m, top_l));
    const Scale scale = scale_of(v.m);
    float s[4] = {0.f, 0.f, 0.f, 0.f}, t[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      const float z = fmaf(x[i], scale.factor, -scale.base);
      const float e = __builtin_amdgcn_exp2f(z);  // NaN stays; 0 for -inf
      s[i & 3] += e;
      t[i & 3] = fmaf(e, fmaxf(z, -200.f), t[i & 3]);
    }
    v.s += (s[0] + s[1]) + (s[2] + s[3]);
    v.t += (t[0] + t[1]) + (t[2] + t[3]);
    if (p.top == 0) continue;
    if (sweep == 0) {
      const uint32_t word[1] = {order_of(top_l)}, w = kth_word(word, p.top);
      if (lane == 0) atomicMax(&reached, w);
      __syncthreads();
    }
    const uint32_t w = *(volatile uint32_t*)&reached;
    // (a NaN maximum is no limit)
    limit = w > order_of(INFINITY) || w < order_of(-INFINITY) ? -INFINITY : fmaxf(limit, logit_of(w));
    uint32_t hits = 0;
#pragma unroll
    for (int i = 0; i < VPT; ++i) hits |= x[i] >= limit ? 1u << i : 0u;
    // (the few that reach the limit are read again: registers have no index)
    while (uint64_t some = __ballot(hits != 0)) {
      const int i = __builtin_ctz(hits | 0x80000000u);
      const int64_t at = from + (int64_t)(i / W) * SWEEP / (VPT / W) + tid * W + i % W;
      const bool in = hits != 0 && at >= lo && at < hi;
      hits &= hits - 1;
      some = __ballot(in);
      if (listed + count(some) > LIST) {
        listed = cut_list(list, listed, p.top, lane);
        // the smallest that is left is the new limit: `top` logits reach it
        uint32_t least[1] = {lane < listed ? ~list[lane].y : 0};
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) least[0] = max(least[0], (uint32_t)__shfl_xor(least[0], o, 64));
        if (lane == 0) atomicMax(&reached, ~least[0]);
        limit = fmaxf(limit, logit_of(~least[0]));
      }
      if (in) {
        const float l = load_float(p.logits.data, DTYPE, base + at * p.logits.s[2]);
        list[listed + below(some)] = make_uint2(0xffffffffu - (uint32_t)at, order_of(l));
      }
      listed += count(some);
    }
  }
  v = wave_sums(v);
  // the lists together: 512 keys at most
  constexpr int E = 8, MOST = 64 * E / WAVES;
  if (listed > MOST) listed = cut_list(list, listed, p.top, lane);
  if (lane == 0) {
    sums[wave] = v;
    counts[wave] = listed;
  }
  __syncthreads();
  if (wave != 0) return;
  v = wave_sums(lane < WAVES ? sums[lane] : Sums{-INFINITY, 0.f, 0.f});
  uint64_t key = 0;
  if (p.top > 0) {
    int n = counts[0];
    for (int w = 1; w < WAVES; ++w) {
      const int own = counts[w];
      for (int i = lane; i < own; i += 64) joined[n + i] = lists[w][i];
      n += own;
    }
    for (int i = lane; i < counts[0]; i += 64) joined[i] = lists[0][i];
    key = sort_list<E>(joined, n, p.top, lane);
  }
  if (p.parts == 1) return put_row(p, row, v, key, lane);
  const int64_t slot = (int64_t)row * p.parts + part;
  if (lane == 0) p.sums[slot] = v;
  if (lane < p.top) p.keys[slot * p.top + lane] = key;
}

// The parts of a row, one wave per row.
__global__ __launch_bounds__(64) void logprob_join_kernel(LogprobParams p) {
  __shared__ uint2 list[LIST];
  const int row = blockIdx.x, lane = threadIdx.x;
  const Sums* sums = p.sums + (int64_t)row * p.parts;
  Sums v = {-INFINITY, 0.f, 0.f};
  for (int i = lane; i < p.parts; i += 64) {
    const float to = fmaxf(v.m, sums[i].m);
    const Sums a = moved(v, to), b = moved(sums[i], to);
    v = {to, a.s + b.s, a.t + b.t};
  }
  v = wave_sums(v);
  const uint64_t* keys = p.keys + (int64_t)row * p.parts * p.top;
  const int n = p.parts * p.top;
  int listed = 0;
  for (int i = 0; i < n; i += 64) {
    if (listed + 64 > LIST) listed = cut_list(list, listed, p.top, lane);
    const uint64_t k = i + lane < n ? keys[i + lane] : 0;
    const uint64_t some = __ballot(k != 0);
    if (k != 0) list[listed + below(some)] = make_uint2((uint32_t)k, (uint32_t)(k >> 32));
    listed += count(some);
  }
  put_row(p, row, v, p.top > 0 ? sort_list<LIST / 64>(list, listed, p.top, lane) : 0, lane);
}

// Threads of a workgroup and logits of a part (the whole row: one launch). skew: logits between an aligned
// address and a row's beginning, at most.
struct Plan {
  int threads;
  int64_t part, parts;
};
constexpr int MAX_SKEW = 7;
Plan plan_of(int64_t rows, int64_t vocab, int skew) {
  if (rows >= 512) return {NARROW, vocab + MAX_SKEW, 1};
  if (vocab <= WIDE * VPT - MAX_SKEW) return {WIDE, vocab + MAX_SKEW, 1};  // one sweep
  const int64_t part = NARROW * VPT;
  return {NARROW, part, (vocab + skew + part - 1) / part};
}

template <int DTYPE>
void launch_logprobs(const LogprobParams& p, int threads, bool in_a_row, hipStream_t st) {
  const dim3 grid((unsigned)p.rows * (unsigned)p.parts), block(threads);
  if (threads == WIDE) {
    if (in_a_row) hipLaunchKernelGGL((logprob_kernel<DTYPE, WIDE, true>), grid, block, 0, st, p);
    else hipLaunchKernelGGL((logprob_kernel<DTYPE, WIDE, false>), grid, block, 0, st, p);
  } else {
    if (in_a_row) hipLaunchKernelGGL((logprob_kernel<DTYPE, NARROW, true>), grid, block, 0, st, p);
    else hipLaunchKernelGGL((logprob_kernel<DTYPE, NARROW, false>), grid, block, 0, st, p);
  }
}

size_t align256(size_t n) { return (n + 255) & ~(size_t)255; }

}  // namespace
}  // namespace lq

using namespace lq;

extern "C" size_t lq_token_logprobs_workspace(int64_t rows, int64_t vocab, int top) {
  if (rows <= 0 || vocab <= 0 || top < 0 || top > MAX_TOP || vocab > INT32_MAX / 2) return 0;
  const Plan plan = plan_of(rows, vocab, MAX_SKEW);
  if (plan.parts == 1) return 0;
  const size_t parts = (size_t)rows * (size_t)plan.parts;
  return align256(parts * sizeof(Sums)) + parts * (size_t)top * 8;
}

extern "C" int lq_token_logprobs(const lq_tensor* logits, const lq_tensor* tokens,
                                 const lq_tensor* logprobs, const lq_tensor* entropy,
                                 const lq_tensor* top_logprobs, const lq_tensor* top_tokens,
                                 void* workspace, size_t workspace_bytes, void* stream) {
  int rc;
  const int nd = logits != nullptr && logits->ndim == 3 ? 3 : 2;
  if ((rc = check_tensor_or_empty(logits, "logits", nd, true)) != LQ_OK) return rc;
  if ((rc = check_tensor_or_empty(tokens, "tokens", nd - 1, false, LQ_I64)) != LQ_OK) return rc;
  if ((rc = check_tensor_or_empty(logprobs, "logprobs", nd - 1, false, LQ_F32)) != LQ_OK) return rc;
  if (entropy != nullptr && (rc = check_tensor_or_empty(entropy, "entropy", nd - 1, false, LQ_F32)) != LQ_OK) return rc;
  if ((top_logprobs == nullptr) != (top_tokens == nullptr)) {
    return fail(LQ_ERR_INVALID_ARG, "top_logprobs and top_tokens: both or neither");
  }
  const int64_t batch = nd == 3 ? logits->shape[0] : 1, len = logits->shape[nd - 2];
  const int64_t rows = batch * len, V = logits->shape[nd - 1];
  for (int i = 0; i < nd - 1; ++i) {
    if (tokens->shape[i] != logits->shape[i]) {
      return fail(LQ_ERR_INVALID_ARG, "tokens must have a value for each row of the logits");
    }
  }
  int64_t top = 0;
  if (top_logprobs != nullptr) {
    if ((rc = check_tensor_or_empty(top_logprobs, "top_logprobs", nd, false, LQ_F32)) != LQ_OK) return rc;
    if ((rc = check_tensor_or_empty(top_tokens, "top_tokens", nd, false, LQ_I64)) != LQ_OK) return rc;
    top = top_logprobs->shape[nd - 1];
  }
  const lq_tensor* outs[4] = {logprobs, entropy, top_logprobs, top_tokens};
  for (const lq_tensor* t : outs) {
    if (t == nullptr) continue;
    bool flat = true;
    int64_t step = 1;
    for (int i = t->ndim - 1; i >= 0; --i) {
      const int64_t want = i < nd - 1 ? logits->shape[i] : top;
      flat = flat && t->shape[i] == want && (want < 2 || rows < 1 || t->stride[i] == step);
      step *= want;
    }
    if (!flat) {
      return fail(LQ_ERR_INVALID_ARG, "the outputs must be contiguous and have a value for each row");
    }
  }
  if (rows == 0) return LQ_OK;
  if (V < 1 || top > V) {
    return fail(LQ_ERR_INVALID_ARG, "%lld likeliest of a vocabulary of %lld asked for", (long long)top,
                (long long)V);
  }
  const int size = dtype_size(logits->dtype);
  const bool in_a_row = V == 1 || logits->stride[nd - 1] == 1;
  bool aligned = ((uintptr_t)logits->data & 15) == 0;
  for (int i = 0; i < nd - 1; ++i) {
    aligned = aligned && (logits->shape[i] < 2 || logits->stride[i] * size % 16 == 0);
  }
  const Plan plan = plan_of(rows, V, in_a_row && !aligned ? MAX_SKEW : 0);
  if (top > MAX_TOP) {
    return fail(LQ_ERR_UNSUPPORTED, "top %lld unsupported (<= %d)", (long long)top, MAX_TOP);
  }
  if (V > INT32_MAX / 2 || rows > INT32_MAX || rows * plan.parts >= ((int64_t)1 << 32) / plan.threads) {
    return fail(LQ_ERR_UNSUPPORTED, "%lld rows of %lld logits exceed the launch limits",
                (long long)rows, (long long)V);
  }
  const size_t need = lq_token_logprobs_workspace(rows, V, (int)top);
  if (need > 0 && (workspace == nullptr || workspace_bytes < need)) {
    return fail(LQ_ERR_WORKSPACE, "workspace of %zu bytes needed, %zu given", need,
                workspace == nullptr ? (size_t)0 : workspace_bytes);
  }
  if (need > 0 && ((uintptr_t)workspace & 255) != 0) {
    return fail(LQ_ERR_WORKSPACE, "workspace must be 256-byte aligned");
  }
  LogprobParams p{};
  p.logits = make_view(logits);
  p.tokens = make_view(tokens);
  if (nd == 2) {
    p.logits.s[2] = p.logits.s[1];
    p.logits.s[1] = p.logits.s[0];
    p.tokens.s[1] = p.tokens.s[0];
  }
  p.logprobs = (float*)logprobs->data;
  if (entropy != nullptr) p.entropy = (float*)entropy->data;
  if (top > 0) {
    p.top_logprobs = (float*)top_logprobs->data;
    p.top_tokens = (int64_t*)top_tokens->data;
  }
  p.rows = (int)rows;
  p.len = (int)len;
  p.parts = (int)plan.parts;
  p.part = (int)plan.part;
  p.top = (int)top;
  p.V = V;
  p.sums = (Sums*)workspace;
  p.keys = (uint64_t*)((char*)workspace + align256((size_t)(rows * plan.parts) * sizeof(Sums)));
  const hipStream_t st = (hipStream_t)stream;
  if (logits->dtype == LQ_BF16) launch_logprobs<LQ_BF16>(p, plan.threads, in_a_row, st);
  else if (logits->dtype == LQ_F16) launch_logprobs<LQ_F16>(p, plan.threads, in_a_row, st);
  else launch_logprobs<LQ_F32>(p, plan.threads, in_a_row, st);
  if ((rc = check_launch("lq_token_logprobs")) != LQ_OK || plan.parts == 1) return rc;
  hipLaunchKernelGGL(logprob_join_kernel, dim3((unsigned)rows), dim3(64), 0, st, p);
  return check_launch("lq_token_logprobs (join)");
}
