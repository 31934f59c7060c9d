// Beam selection: the `num` best continuations of each prompt's N beams over a vocabulary of V tokens.
//
// The total of beam n and token t is score[n] + logit[n][t] - lse[n], lse[n] the log-sum-exp of the
// beam's logits. Within a beam the order of the totals is the order of the logits, so that one pass over
// the logits gives both.
//
// select_part_kernel: a workgroup of 4 waves takes a part of one beam's row, up to 64 logits per lane, all
// loaded at once and kept in registers as they are. A pass over them makes the lanes' maxima and sums;
// the num-th largest of the 256 maxima is a threshold that num logits reach, and few others (about 34
// for 32, of 16384 random ones). A second pass over the registers collects those in lists, which
// are cut down to their num largest, ties by the lower token. The num-th largest of the values in a
// wave's registers is found bit by bit with ballots (kth_word), with no exchange between lanes. Lists that
// overflow (many equal logits, sorted ones) are cut on the way, which raises the threshold. The part
// leaves (max, sum), its num largest logits and a bound that they all reach.
//
// select_final_kernel: one workgroup per prompt makes lse[n] and the totals in 64 bits. num candidates
// reach the largest of the parts' bounds; those that do (a few hundred) are reduced, wave by wave, to
// the num best, which one wave sorts and writes out, by rank or by place.
//
// The sums of exponentials are fp32 and off by less than 2^-18, which is their logarithms' error: at most
// 24 additions in a row (lane 8, wave 6, workgroup 3, parts 7), 7 exponentials (the term's own and its
// rescales, one step of fp32 each) and their 6 products, 2^-24 each, and the roundings of the exponents,
// 2^-24 of the distance to the maximum, which weighted with the terms is 17 * 2^-24 at 2^24 tokens.
// A whole beam has its lse's error, so that totals of one beam keep their order; those of two beams can
// change places where they are closer than that.
//
// What it measured (MI355X, kernel trace, parts + final): 256 rows of 131072 bf16 logits (67 MB), 32 of
// each of 16 prompts, 19.2 + 10.4 us; 64 rows, 8 of each of 8 prompts, 9.8 + 6.6; 15 rows of 50257 fp32
// 6.6 + 6.6; 4 rows of 32000 6.2 + 5.7. The largest is bound by the VALU (about 13 instructions per logit,
// of which the exponential takes two issue slots), the others by the latency of two launches and of
// their loads. Tried: one block reduction per selected token (1301 us for the largest); lists per run with a
// rising threshold (57 us); the list code inside the 64 unrolled comparisons (part kernel 46.8 us: the
// instruction cache; 23.0 with it outside).
#include <math.h>

#include <algorithm>

#include "lq_common.h"

namespace lq {
namespace {

constexpr int MAX_BEAMS = LQ_BEAM_SELECT_MAX_BEAMS;
constexpr int MAX_NUM = LQ_BEAM_SELECT_MAX_NUM;
constexpr int WAVES = 4;            // waves of a part's workgroup
constexpr int THREADS = 64 * WAVES;
constexpr int PER = 16;             // logits per lane and run
constexpr int RUN = 64 * PER;       // logits per wave and run
constexpr int LIST = 256;           // entries of a wave's candidate list (4 per lane)
constexpr int FINAL_LIST = 1024;    // entries of a prompt's candidate list

struct PartResult {
  float m, s;      // log2e times the maximum, and the sum of 2^(x log2e - m)
  uint32_t bound;  // order of a logit that num of the part's reach; 0: there are fewer
  uint32_t share;  // the same for ceil(num / parts) of them, the part's share of num
};

struct SelectParams {
  View logits;          // strides of (prompt, beam, token)
  const float* scores;  // strides of (prompt, beam)
  int64_t ss[2];
  const uint8_t* finished;  // NULL, or strides of (prompt, beam)
  int64_t fs[2];
  float* out_score;     // [P, num] each
  int64_t* out_beam;
  int64_t* out_token;
  int64_t os[3][2];
  int64_t pad;
  int P, N, num, slots;
  int64_t V;
  int parts, cap;       // parts of a row, places for a part's candidates
  int share;            // ceil(num / parts)
  PartResult* ws_part;  // [rows][parts]
  uint64_t* ws_key;     // [rows][parts][cap]: order of the logit, then of the token; 0: none
  uint32_t inv_cap, inv_parts;  // ceil(2^32 / cap) and .. / parts (0 for 1), for quotients by them
};

constexpr float LOG2E_F = 1.44269504f;
constexpr uint32_t ORDER_NONE = 0x007fffffu;  // order_bits(-inf): words below it are no numbers
constexpr float LOWEST = -3.0e38f;  // stands for the maximum where there is no logit above -inf

// An unsigned integer in the order of the floats (-0 counts as 0).
__device__ __forceinline__ uint32_t order_bits(float x) {
  const uint32_t u = __float_as_uint(x + 0.0f);
  return u ^ ((u >> 31) != 0 ? 0xffffffffu : 0x80000000u);
}

__device__ __forceinline__ float from_order_bits(uint32_t k) {
  return __uint_as_float(k ^ ((k >> 31) != 0 ? 0x80000000u : 0xffffffffu));
}

// Larger is better: the logit, then the lower token. Never 0.
__device__ __forceinline__ uint64_t make_key(float x, uint32_t token) {
  return ((uint64_t)order_bits(x) << 32) | (0xffffffffu - token);
}

__device__ __forceinline__ int count(uint64_t ballot) { return __builtin_popcountll(ballot); }

// The lanes below this one that are set in a ballot.
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

template <int E>
__device__ __forceinline__ int count_from(const uint32_t (&v)[E], uint32_t w) {
  int c = 0;
#pragma unroll
  for (int e = 0; e < E; ++e) c += count(__ballot(v[e] >= w));
  return c;
}

// The need-th largest of the wave's 64 E words (0: none; more than `need` others): a word w that exactly
// `need` of them reach (exact), or else the need-th largest itself, which more reach. Found from the
// highest bit in which the words differ down, by counting those that reach the next guess; a guess that
// leaves the right number ends the search, after 8 to 12 counts for most inputs.
template <int E>
__device__ __forceinline__ uint32_t kth_word(const uint32_t (&v)[E], int need, bool& exact) {
  uint32_t some = 0, every = ~0u;
#pragma unroll
  for (int e = 0; e < E; ++e) {
    some |= v[e];
    every &= v[e] == 0 ? ~0u : v[e];
  }
  some = wave_fold(some, [](uint32_t a, uint32_t b) { return a | b; });
  uint32_t w = wave_fold(every, [](uint32_t a, uint32_t b) { return a & b; });
  uint32_t differ = some & ~w;
  while (differ != 0) {
    const uint32_t bit = 0x80000000u >> __builtin_clz(differ);
    differ ^= bit;
    const int c = count_from<E>(v, w | bit);
    if (c == need) {
      exact = true;
      return w | bit;
    }
    w = c > need ? w | bit : w;
  }
  exact = false;
  return w;
}

// Marks in take[e] the `need` largest of the entries in the running, by one word of their keys (larger
// first, 0: not in the running); where ties go on, v[e] keeps the tied ones' and `need` what is left.
template <int E>
__device__ __forceinline__ void narrow(uint32_t (&v)[E], bool (&take)[E], int& need) {
  const int have = count_from<E>(v, 1);
  if (need >= have) {
#pragma unroll
    for (int e = 0; e < E; ++e) take[e] = take[e] || v[e] != 0;
    need = 0;
    return;
  }
  bool exact;
  const uint32_t w = kth_word<E>(v, need, exact);
  int taken = 0;
#pragma unroll
  for (int e = 0; e < E; ++e) {
    const bool t = v[e] > w || (exact && v[e] == w);
    taken += count(__ballot(t));
    take[e] = take[e] || t;
    v[e] = v[e] == w ? v[e] : 0;
  }
  need -= taken;
}

// take[e]: whether key[e] is among the wave's k largest (all distinct; 0 is no entry).
template <int E>
__device__ __forceinline__ void take_keys(const uint64_t (&key)[E], int k, bool (&take)[E]) {
  uint32_t v[E];
#pragma unroll
  for (int e = 0; e < E; ++e) {
    take[e] = false;
    v[e] = (uint32_t)(key[e] >> 32);
  }
  int need = k;
  narrow<E>(v, take, need);
  if (need == 0) return;
#pragma unroll
  for (int e = 0; e < E; ++e) v[e] = v[e] != 0 ? (uint32_t)key[e] : 0;
  narrow<E>(v, take, need);
}

// The wave's list cut down to its k largest entries; the threshold rises to the smallest of them where
// there are k.
__device__ __forceinline__ void cut_list(uint64_t* list, int& n, int k, uint64_t& bar, float& barf) {
  const int lane = threadIdx.x & 63;
  uint64_t key[4];
  bool take[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) key[e] = 64 * e + lane < n ? list[64 * e + lane] : 0;
  __builtin_amdgcn_wave_barrier();
  take_keys<4>(key, k, take);
  n = 0;
  uint32_t low = ~0u;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const uint64_t b = __ballot(take[e]);
    if (take[e]) {
      list[n + below(b)] = key[e];
      low = min(low, (uint32_t)(key[e] >> 32));
    }
    n += count(b);
  }
  __builtin_amdgcn_wave_barrier();
  if (n >= k) {
    low = wave_fold(low, [](uint32_t a, uint32_t b) { return min(a, b); });
    uint32_t token = ~0u;  // of the entries with the smallest logit, the one with the highest token
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      if (take[e] && (uint32_t)(key[e] >> 32) == low) token = min(token, (uint32_t)key[e]);
    }
    token = wave_fold(token, [](uint32_t a, uint32_t b) { return min(a, b); });
    const uint64_t key_low = (uint64_t)low << 32 | token;
    if (key_low > bar) {
      bar = key_low;
      barf = from_order_bits(low);
    }
  }
}

// The 16 logits of a lane in a run, as they are in memory.
template <int DT>
struct Raw {
  static constexpr int SIZE = DT == LQ_F32 ? 4 : 2;
  static constexpr int N = 16 / SIZE;  // logits of 16 bytes
  static constexpr int WORDS = PER * SIZE / 4;
  uint32_t w[WORDS];

  __device__ __forceinline__ float operator[](int i) const {
    if constexpr (DT == LQ_F32) return __uint_as_float(w[i]);
    else return word_elem(w[i / 2], 16 * (i % 2), DT);
  }
};

// 16 bytes at any address: the order of a row's sums must not depend on where the row starts, so that
// beams with equal logits get equal totals (a row of an odd vocabulary starts at any multiple of 2 bytes).
struct __attribute__((packed, aligned(2))) Unaligned16 {
  uint32_t v[4];
};

// DENSE: the logits of a row are contiguous and loaded 16 bytes per lane, but for the row's last run.
// Otherwise, and there, one element at a time. Wave w takes runs w, w + 4, .. of the part's 4 R.
template <int DT, bool DENSE, int R>
__global__ __launch_bounds__(THREADS) void select_part_kernel(SelectParams p) {
  __shared__ uint64_t lists[WAVES][LIST];
  __shared__ uint32_t maxima[THREADS];
  __shared__ uint32_t threshold[2];  // order of a logit that num (the share of num) of the part's reach
  __shared__ int counts[WAVES];
  __shared__ float wave_m[WAVES], wave_s[WAVES];
  constexpr int VN = Raw<DT>::N;
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  const int64_t row = blockIdx.y;
  const int64_t prompt = row / p.N, beam = row - prompt * p.N;
  if (p.finished != nullptr && p.finished[prompt * p.fs[0] + beam * p.fs[1]] != 0) return;
  const int64_t base = prompt * p.logits.s[0] + beam * p.logits.s[1];
  const char* first = (const char*)p.logits.data + base * Raw<DT>::SIZE;
  const uint32_t V = (uint32_t)p.V;
  const int k = p.num;
  uint64_t* list = lists[wave];

  // first token of run r of the wave, and token of the lane's logit i in it
  auto start_of = [&](int r) -> uint32_t { return (blockIdx.x * (WAVES * R) + r * WAVES + wave) * RUN; };
  auto token = [&](uint32_t start, int i) -> uint32_t {
    return DENSE ? start + ((i / VN) * 64 + lane) * VN + i % VN : start + i * 64 + lane;
  };

  Raw<DT> x[R];
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const uint32_t start = start_of(r);
    if (DENSE && start + RUN <= V) {
      const Unaligned16* at = (const Unaligned16*)(first + (int64_t)start * Raw<DT>::SIZE) + lane;
#pragma unroll
      for (int j = 0; j < PER / VN; ++j) {
#pragma unroll
        for (int u = 0; u < 4; ++u) x[r].w[4 * j + u] = at[64 * j].v[u];
      }
    } else {
      // tokens past the row as -inf
      constexpr uint32_t NONE = DT == LQ_F32 ? 0xff800000u : DT == LQ_BF16 ? 0xff80u : 0xfc00u;
#pragma unroll
      for (int u = 0; u < Raw<DT>::WORDS; ++u) x[r].w[u] = 0;
      if (start < V) {
#pragma unroll
        for (int i = 0; i < PER; ++i) {
          const uint32_t t = token(start, i);
          const int64_t at = base + (int64_t)t * p.logits.s[2];
          uint32_t bits = NONE;
          if constexpr (DT == LQ_F32) {
            if (t < V) bits = ((const uint32_t*)p.logits.data)[at];
            x[r].w[i] = bits;
          } else {
            if (t < V) bits = ((const uint16_t*)p.logits.data)[at];
            x[r].w[i / 2] |= bits << (16 * (i % 2));
          }
        }
      } else {
#pragma unroll
        for (int u = 0; u < Raw<DT>::WORDS; ++u) x[r].w[u] = DT == LQ_F32 ? NONE : NONE | NONE << 16;
      }
    }
  }

  // the lane's maximum and sum, S = sum 2^(x log2e - c) with c = log2e times the maximum so far. The
  // product is exact inside the multiply-add, so that the terms near the maximum are off by the
  // exponential alone; log2e's own rounding drops out when the logarithm is divided by it again, but for
  // 1e-8 times the entropy.
  float mx = -INFINITY, run_max[R], c = LOWEST, sl = 0.0f;
#pragma unroll
  for (int r = 0; r < R; ++r) {
    run_max[r] = x[r][0];
#pragma unroll
    for (int i = 1; i < PER; ++i) run_max[r] = fmaxf(run_max[r], x[r][i]);
    mx = fmaxf(mx, run_max[r]);
    const float c2 = fmaxf(c, run_max[r] * LOG2E_F);
    if (r > 0) sl *= __builtin_amdgcn_exp2f(c - c2);
    c = c2;
    float four[4] = {0.0f, 0.0f, 0.0f, 0.0f};  // (short chains of additions)
#pragma unroll
    for (int i = 0; i < PER; ++i) four[i % 4] += __builtin_amdgcn_exp2f(fmaf(x[r][i], LOG2E_F, -c));
    sl += (four[0] + four[1]) + (four[2] + four[3]);
    // the logits stay as they were loaded: unpacked for the second pass too, they took twice the registers
#pragma unroll
    for (int u = 0; u < Raw<DT>::WORDS; ++u) asm volatile("" : "+v"(x[r].w[u]));
  }
  maxima[threadIdx.x] = token(start_of(0), 0) < V ? order_bits(mx) : 0;  // 0: a lane without a token
  const float wm = group_max<64>(c);
  const float ws = group_sum<64>(sl * __builtin_amdgcn_exp2f(c - wm));
  if (lane == 0) {
    wave_m[wave] = wm;
    wave_s[wave] = ws;
  }
  __syncthreads();

  // the threshold: only keys above bar are taken, whose logits reach barf
  if (wave < 2) {
    uint32_t v[WAVES];
#pragma unroll
    for (int w = 0; w < WAVES; ++w) v[w] = maxima[64 * w + lane];
    const int need = wave == 0 ? k : p.share;
    const int have = count_from<WAVES>(v, 1);
    bool exact;
    uint32_t w = 0;
    if (have > need) {
      w = kth_word<WAVES>(v, need, exact);
    } else if (have == need) {
      uint32_t low = ~0u;
#pragma unroll
      for (int i = 0; i < WAVES; ++i) low = v[i] != 0 ? min(low, v[i]) : low;
      w = wave_fold(low, [](uint32_t a, uint32_t b) { return min(a, b); });
    }
    if (lane == 0) threshold[wave] = w;
  }
  __syncthreads();
  const uint32_t bound = __builtin_amdgcn_readfirstlane(threshold[0]);
  uint64_t bar = 0;
  float barf = -INFINITY;
  if (bound != 0) {
    bar = ((uint64_t)bound << 32) - 1;
    barf = from_order_bits(bound);
  }
  int n = 0;  // entries of the wave's list
  if (bound != 0) {
#pragma unroll
    for (int r = 0; r < R; ++r) {
      if (__ballot(run_max[r] >= barf) == 0) continue;
#pragma unroll
      for (int i = 0; i < PER; ++i) {
        const uint64_t b = __ballot(x[r][i] >= barf);
        if (b == 0) continue;
        const int at = n + below(b);
        if (x[r][i] >= barf && at < LIST) list[at] = make_key(x[r][i], token(start_of(r), i));
        n += count(b);
      }
    }
  }
  // no threshold, more logits at it than the list holds, or the row's end among them (its places past
  // the last token are -inf): once more, the list cut where it is full
  if (bound == 0 || n > LIST || barf == -INFINITY) {
    n = 0;
    for (int r = 0; r < R; ++r) {
      Raw<DT> y = x[0];
#pragma unroll
      for (int q = 1; q < R; ++q) {
#pragma unroll
        for (int u = 0; u < Raw<DT>::WORDS; ++u) y.w[u] = q == r ? x[q].w[u] : y.w[u];
      }
      uint32_t hits = 0;
#pragma unroll
      for (int i = 0; i < PER; ++i) hits |= y[i] >= barf ? 1u << i : 0u;
      // one per lane at a time
      while (__ballot(hits != 0) != 0) {
        const bool more = hits != 0;
        const int i = more ? __builtin_ctz(hits) : 0;
        hits &= hits - 1;  // (0 stays 0)
        uint32_t w = y.w[0];
#pragma unroll
        for (int u = 1; u < Raw<DT>::WORDS; ++u) w = i * Raw<DT>::SIZE / 4 == u ? y.w[u] : w;
        const float xi = DT == LQ_F32 ? __uint_as_float(w) : word_elem(w, 16 * (i & 1), DT);
        const uint32_t t = token(start_of(r), i);
        const uint64_t key = make_key(xi, t);
        bool ok = more && xi >= barf && t < V && key > bar;
        uint64_t b = __ballot(ok);
        if (n + count(b) > LIST) {
          cut_list(list, n, k, bar, barf);
          ok = ok && key > bar;
          b = __ballot(ok);
        }
        if (ok) list[n + below(b)] = key;
        n += count(b);
      }
    }
  }
  __builtin_amdgcn_wave_barrier();
  if (n > 64) cut_list(list, n, k, bar, barf);
  if (lane == 0) counts[wave] = n;
  __syncthreads();
  if (wave != 0) return;

  const int64_t slot = row * p.parts + blockIdx.x;
  float M = wave_m[0], S = 0.0f;
#pragma unroll
  for (int w = 1; w < WAVES; ++w) M = fmaxf(M, wave_m[w]);
#pragma unroll
  for (int w = 0; w < WAVES; ++w) {
    S += wave_s[w] * __builtin_amdgcn_exp2f(wave_m[w] - M);
  }
  // the part's candidates: the lists as they are where they fit (num of them reach the bound, the final
  // workgroup looks at the others' totals anyway), else the num largest
  uint64_t key[WAVES];
  bool take[WAVES];
  int have = 0;
#pragma unroll
  for (int w = 0; w < WAVES; ++w) {
    have += counts[w];
    key[w] = lane < counts[w] ? lists[w][lane] : 0;
    take[w] = key[w] != 0;
  }
  if (have > p.cap) take_keys<WAVES>(key, k, take);
  int total = 0;
  uint32_t low = ~0u;
#pragma unroll
  for (int w = 0; w < WAVES; ++w) {
    const uint64_t b = __ballot(take[w]);
    if (take[w]) {
      p.ws_key[slot * p.cap + total + below(b)] = key[w];
      low = min(low, (uint32_t)(key[w] >> 32));
    }
    total += count(b);
  }
  for (int i = total + lane; i < p.cap; i += 64) p.ws_key[slot * p.cap + i] = 0;
  if (have > p.cap) low = wave_fold(low, [](uint32_t a, uint32_t b) { return min(a, b); });
  else low = bound;
  if (lane == 0) {
    p.ws_part[slot] = PartResult{M, S, total >= k ? low : 0, threshold[1]};
  }
}

// A candidate of a prompt: its total and flat index n * V + token. Larger totals first, then the lower
// index.
struct Candidate {
  double total;
  uint32_t index;
};

__device__ __forceinline__ uint64_t order_bits64(double x) {
  const uint64_t u = (uint64_t)__double_as_longlong(x + 0.0);
  return u ^ ((u >> 63) != 0 ? ~(uint64_t)0 : (uint64_t)1 << 63);
}

// take[e]: whether candidate c[e] (where on[e]) is among the wave's k best. The first 32 bits of a total
// settle nearly every selection.
__device__ __forceinline__ void take_candidates(const Candidate (&c)[4], const bool (&on)[4], int k,
                                                bool (&take)[4]) {
  uint32_t v[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    take[e] = false;
    v[e] = on[e] ? (uint32_t)(order_bits64(c[e].total) >> 32) : 0;
  }
  int need = k;
  narrow<4>(v, take, need);
  if (need == 0) return;
  // (words are compared above 0: the other 32 bits go in two steps, 31 of them and the last)
#pragma unroll
  for (int e = 0; e < 4; ++e) v[e] = v[e] != 0 ? (uint32_t)order_bits64(c[e].total) >> 1 | 0x80000000u : 0;
  narrow<4>(v, take, need);
  if (need == 0) return;
#pragma unroll
  for (int e = 0; e < 4; ++e) v[e] = v[e] != 0 ? ((uint32_t)order_bits64(c[e].total) & 1u) + 1 : 0;
  narrow<4>(v, take, need);
  if (need == 0) return;
#pragma unroll
  for (int e = 0; e < 4; ++e) v[e] = v[e] != 0 ? ~c[e].index : 0;
  narrow<4>(v, take, need);
}

// FW waves per prompt. Everything that does not depend on the sums is loaded first.
template <int FW>
__global__ __launch_bounds__(64 * FW) void select_final_kernel(SelectParams p) {
  __shared__ double base[MAX_BEAMS];   // score - lse; -inf: no candidate above -inf
  __shared__ bool alone[MAX_BEAMS];    // a finished beam
  __shared__ double c_total[FINAL_LIST], d_total[4 * MAX_NUM];
  __shared__ uint32_t c_index[FINAL_LIST], d_index[4 * MAX_NUM];
  __shared__ uint32_t bound_bits;
  __shared__ uint32_t shares[MAX_BEAMS], least[MAX_BEAMS];
  __shared__ int c_count, d_count, has_apart;
  __shared__ int ranks[256], first_of[MAX_BEAMS];
  __shared__ double r_total[MAX_NUM];
  __shared__ uint32_t r_index[MAX_NUM];
  const int64_t prompt = blockIdx.x;
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  const int k = p.num;
  const uint32_t V = (uint32_t)p.V;
  const uint32_t slots = (uint32_t)p.N * p.parts;  // of the prompt
  const uint32_t all = slots * p.cap;
  const PartResult* parts = p.ws_part + prompt * slots;
  const uint64_t* keys = p.ws_key + prompt * slots * p.cap;
  if (threadIdx.x == 0) {
    c_count = d_count = has_apart = 0;
    bound_bits = 0;
  }
  if (threadIdx.x < 256) ranks[threadIdx.x] = 0;
  if (threadIdx.x < MAX_BEAMS) first_of[threadIdx.x] = MAX_NUM;
  // BATCH candidates per thread at a time, the first ones before the sums are made
  constexpr int BATCH = 8;
  uint64_t batch[BATCH];
  auto load_batch = [&](uint32_t from) {
#pragma unroll
    for (int i = 0; i < BATCH; ++i) {
      const uint32_t at = from + i * 64 * FW + threadIdx.x;
      batch[i] = at < all ? keys[at] : 0;
    }
  };
  load_batch(0);
  PartResult first_part = {};
  if (threadIdx.x < slots) first_part = parts[threadIdx.x];

  for (int n = wave; n < p.N; n += FW) {
    // the lane's first part is loaded beside the flag and the score
    PartResult r = {LOWEST, 0.0f, 0, ~0u};
    if (lane < p.parts) r = parts[n * p.parts + lane];
    const float score = p.scores[prompt * p.ss[0] + n * p.ss[1]];
    const bool fin = p.finished != nullptr && p.finished[prompt * p.fs[0] + n * p.fs[1]] != 0;
    double b = score;
    if (!fin) {
      // the largest of the parts' maxima, then their sums
      float m = r.m;
      uint32_t share = r.share;
      for (int i = lane + 64; i < p.parts; i += 64) {
        const PartResult& q = parts[n * p.parts + i];
        share = min(share, q.share);
        m = fmaxf(m, q.m);
      }
      const float M = group_max<64>(m);
      double of_lane = r.s * exp2f(r.m - M);
      for (int i = lane + 64; i < p.parts; i += 64) {
        const PartResult& q = parts[n * p.parts + i];
        of_lane += q.s * exp2f(q.m - M);
      }
      const float s = group_sum<64>((float)of_lane);
      share = wave_fold(share, [](uint32_t a, uint32_t b) { return min(a, b); });
      if (lane == 0) shares[n] = share;
      b = (double)score - ((double)M + log2((double)s)) / (double)LOG2E_F;
    }
    if (lane == 0) {
      alone[n] = fin;
      base[n] = fabs(b) < INFINITY ? b : -INFINITY;
    }
  }
  __syncthreads();

  auto beam_of = [&](uint32_t slot) -> uint32_t {
    return p.inv_parts != 0 ? __umulhi(slot, p.inv_parts) : slot;
  };
  // At least k totals reach the largest of the parts' bounds, and the largest over the beams of the
  // smallest of its parts' share bounds (as the order of an fp32 number, a step below the rounded total).
  uint32_t most = 0;
  for (uint32_t i = threadIdx.x; i < slots; i += 64 * FW) {
    const uint32_t n = beam_of(i);
    uint32_t w = i == threadIdx.x ? first_part.bound : parts[i].bound;
    if (i == n * p.parts) w = max(w, shares[n]);
    if (!alone[n] && base[n] != -INFINITY && w != 0) {
      const uint32_t o = order_bits((float)(base[n] + (double)from_order_bits(w)));
      most = max(most, o > ORDER_NONE ? o - 1 : o);
    }
  }
  most = wave_fold(most, [](uint32_t a, uint32_t b) { return max(a, b); });
  if (lane == 0) atomicMax(&bound_bits, most);
  __syncthreads();
  const double bound = bound_bits == 0 ? -INFINITY : (double)from_order_bits(bound_bits);
  // the order of a logit below those of beam n that reach it (the difference rounded to fp32, two steps
  // down)
  for (int n = threadIdx.x; n < p.N; n += 64 * FW) {
    const bool apart = alone[n] || base[n] == -INFINITY;
    const uint32_t w = order_bits((float)(bound - base[n]));
    least[n] = apart ? ~0u : bound == -INFINITY || w <= 2 ? 1u : w - 2;
    if (apart) has_apart = 1;
  }
  __syncthreads();

  auto place = [&](uint32_t at, uint32_t& n, uint32_t& i) -> bool {  // place i of beam n's first part
    const uint32_t slot = __umulhi(at, p.inv_cap);
    n = beam_of(slot);
    i = at - slot * p.cap;
    return slot == n * p.parts;
  };
  // the candidate with its key; whether it reaches the bound
  auto candidate = [&](uint32_t n, uint64_t key, Candidate& c) -> bool {
    c.total = base[n] + (double)from_order_bits((uint32_t)(key >> 32));
    c.index = n * V + (0xffffffffu - (uint32_t)key);
    return c.total >= bound;
  };
  // the i-th candidate of a beam without logits: a finished beam's own score, where it has one, at the pad
  // token, then the lowest tokens at -inf
  auto apart_candidate = [&](uint32_t n, uint32_t i, Candidate& c) -> bool {
    if (i >= (uint32_t)k || i >= V) return false;
    uint32_t token = i;
    c.total = -INFINITY;
    if (alone[n] && base[n] != -INFINITY) {
      token = i == 0 ? (uint32_t)p.pad : (i <= (uint32_t)p.pad ? i - 1 : i);
      if (i == 0) c.total = base[n];
    }
    c.index = n * V + token;
    return c.total >= bound;
  };
  auto any_candidate = [&](uint32_t at, Candidate& c) -> bool {
    uint32_t n, i;
    c = Candidate{-INFINITY, 0};
    if (at >= all) return false;
    const bool lead = place(at, n, i);
    if (least[n] == ~0u) return lead && apart_candidate(n, i, c);
    const uint64_t key = keys[at];
    return (uint32_t)(key >> 32) >= least[n] && candidate(n, key, c);
  };
  auto append = [&](bool yes, const Candidate& v, double* totals, uint32_t* indexes, int& at, int room) {
    const uint64_t b = __ballot(yes);
    if (b == 0) return;
    int first = 0;
    if (lane == 0) first = atomicAdd(&at, count(b));
    first = __builtin_amdgcn_readfirstlane(first) + below(b);
    if (yes && first < room) {
      totals[first] = v.total;
      indexes[first] = v.index;
    }
  };

  // the candidates that reach the bound, in one list
  Candidate c[4];
  bool on[4], take[4];
  for (uint32_t from = 0; from < all; from += BATCH * 64 * FW) {
    if (from > 0) load_batch(from);
#pragma unroll
    for (int i = 0; i < BATCH; ++i) {
      const uint32_t at = from + i * 64 * FW + threadIdx.x;
      if (at - lane >= all) break;
      const uint32_t n = beam_of(__umulhi(min(at, all - 1), p.inv_cap));
      const bool maybe = (uint32_t)(batch[i] >> 32) >= least[n];  // (0 past the end and where there is none)
      if (__ballot(maybe) == 0) continue;
      append(maybe && candidate(n, batch[i], c[0]), c[0], c_total, c_index, c_count, FINAL_LIST);
    }
  }
  if (has_apart) {
    for (uint32_t at = threadIdx.x; at - lane < (uint32_t)(p.N * k); at += 64 * FW) {
      const uint32_t n = at / (uint32_t)k;
      const bool yes = at < (uint32_t)(p.N * k) && least[n] == ~0u && apart_candidate(n, at - n * k, c[0]);
      append(yes, c[0], c_total, c_index, c_count, FINAL_LIST);
    }
  }
  __syncthreads();
  if (c_count > FINAL_LIST) {
    // too many (most of them equal): each wave's k best of its own, 192 new ones at a time beside the
    // best so far (c[0]), and the waves' in the list
    __syncthreads();
    if (threadIdx.x == 0) c_count = 0;
    double* own_total = &c_total[wave * MAX_NUM];
    uint32_t* own_index = &c_index[wave * MAX_NUM];
    c[0] = Candidate{-INFINITY, 0};
    on[0] = false;
    for (uint32_t slice = wave * 192; slice < all; slice += FW * 192) {
      bool any = false;
#pragma unroll
      for (int e = 1; e < 4; ++e) {
        const uint32_t at = slice + 64 * (e - 1) + lane;
        on[e] = any_candidate(at, c[e]);
        any = any || on[e];
      }
      if (__ballot(any) == 0) continue;
      take_candidates(c, on, k, take);
      int total = 0;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const uint64_t b = __ballot(take[e]);
        if (take[e]) {
          own_total[total + below(b)] = c[e].total;
          own_index[total + below(b)] = c[e].index;
        }
        total += count(b);
      }
      __builtin_amdgcn_wave_barrier();
      on[0] = lane < total;
      if (on[0]) c[0] = Candidate{own_total[lane], own_index[lane]};
      __builtin_amdgcn_wave_barrier();
    }
    __syncthreads();
    append(on[0], c[0], c_total, c_index, c_count, FINAL_LIST);
    __syncthreads();
  }
  // more than 256 entries are reduced, 256 per wave, to a list of k entries per wave
  int entries = c_count;
  const double* totals = c_total;
  const uint32_t* indexes = c_index;
  if (entries > 256) {
    if (256 * wave < entries) {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int i = 256 * wave + 64 * e + lane;
        on[e] = i < entries;
        c[e] = on[e] ? Candidate{c_total[i], c_index[i]} : Candidate{-INFINITY, 0};
      }
      take_candidates(c, on, k, take);
#pragma unroll
      for (int e = 0; e < 4; ++e) append(take[e], c[e], d_total, d_index, d_count, 4 * MAX_NUM);
    }
    __syncthreads();
    entries = d_count;
    totals = d_total;
    indexes = d_index;
  }
  // their ranks: thread t counts for entry t % 256 the better ones of a stretch
  {
    const int i = threadIdx.x & 255;
    const int stretch = (entries + FW / 4 - 1) / (FW / 4);
    const int j0 = (threadIdx.x >> 8) * stretch, j1 = min(entries, j0 + stretch);
    const double total = i < entries ? totals[i] : -INFINITY;
    const uint32_t index = i < entries ? indexes[i] : 0xffffffffu;
    int better = 0;
    if ((i & ~63) < entries) {  // (uniform per wave)
#pragma unroll 4
      for (int j = j0; j < j1; ++j) {
        const double t = totals[j];
        better += t > total || (t == total && indexes[j] < index) ? 1 : 0;
      }
      if (i < entries) atomicAdd(&ranks[i], better);
    }
  }
  __syncthreads();
  if (threadIdx.x < entries && ranks[threadIdx.x] < k) {
    const int r = ranks[threadIdx.x];
    r_total[r] = totals[threadIdx.x];
    r_index[r] = indexes[threadIdx.x];
  }
  __syncthreads();
  if (wave != 0) return;

  // the k chosen ones in order, one per lane (num <= N * V: there are k)
  const bool chosen = lane < k;
  const uint32_t index = chosen ? r_index[lane] : 0;
  const int beam = (int)(index / V);
  int at = lane;
  if (p.slots) {
    // a beam's best continuation keeps the beam's place, the others take the free places in order
    if (chosen) atomicMin(&first_of[beam], lane);
    __builtin_amdgcn_wave_barrier();
    const bool best = chosen && first_of[beam] == lane;
    uint64_t free = __ballot(lane < p.N && first_of[lane] == MAX_NUM);
    const int before = below(__ballot(chosen && !best));
    for (int j = 0; j < before; ++j) free &= free - 1;
    at = best ? beam : __builtin_ctzll(free | (uint64_t)1 << 63);
  }
  if (chosen) {
    p.out_score[prompt * p.os[0][0] + at * p.os[0][1]] = (float)r_total[lane];
    p.out_beam[prompt * p.os[1][0] + at * p.os[1][1]] = beam;
    p.out_token[prompt * p.os[2][0] + at * p.os[2][1]] = index - (uint32_t)beam * V;
  }
}

// Runs per wave of a part: 4 (64 logits per lane), or fewer where that leaves under two workgroups per CU.
int plan_runs(int64_t rows, int64_t V) {
  const int64_t runs = rows * ((V + RUN - 1) / RUN);
  for (int r = 4; r > 1; r /= 2) {
    if (runs / (WAVES * r) >= 2 * (int64_t)device_cus()) return r;
  }
  return 1;
}

// Places for a part's candidates: room for the few beside the num largest that usually reach its bound.
int cap_of(int num) { return num + num / 2 + 8; }

int parts_of(int64_t V, int runs) { return (int)((V + RUN * WAVES * runs - 1) / (RUN * WAVES * runs)); }

template <int DT, bool DENSE>
void launch_runs(const SelectParams& p, int runs, dim3 grid, hipStream_t st) {
  if (runs == 4) hipLaunchKernelGGL((select_part_kernel<DT, DENSE, 4>), grid, dim3(THREADS), 0, st, p);
  else if (runs == 2) hipLaunchKernelGGL((select_part_kernel<DT, DENSE, 2>), grid, dim3(THREADS), 0, st, p);
  else hipLaunchKernelGGL((select_part_kernel<DT, DENSE, 1>), grid, dim3(THREADS), 0, st, p);
}

template <int DT>
void launch_part(const SelectParams& p, int runs, dim3 grid, hipStream_t st) {
  if (p.logits.s[2] == 1) launch_runs<DT, true>(p, runs, grid, st);
  else launch_runs<DT, false>(p, runs, grid, st);
}

size_t align256(size_t n) { return (n + 255) / 256 * 256; }

}  // namespace
}  // namespace lq

using namespace lq;

extern "C" size_t lq_beam_select_workspace(int64_t prompts, int64_t beams, int64_t vocab, int num) {
  if (prompts <= 0 || beams <= 0 || vocab <= 0 || num <= 0) return 0;
  const int64_t rows = prompts * beams;
  const size_t slots = (size_t)rows * (size_t)parts_of(vocab, plan_runs(rows, vocab));
  return align256(slots * sizeof(PartResult)) + slots * (size_t)cap_of(num) * 8;
}

extern "C" int lq_beam_select(const lq_tensor* logits, const lq_tensor* scores,
                              const lq_tensor* finished, const lq_tensor* out_scores,
                              const lq_tensor* out_beams, const lq_tensor* out_tokens,
                              int64_t pad_token, int keep_slots, void* workspace,
                              size_t workspace_bytes, void* stream) {
  int rc;
  const int ldim = logits != nullptr && logits->ndim == 2 ? 2 : 3;
  if ((rc = check_tensor(logits, "logits", ldim, true)) != LQ_OK) return rc;
  if ((rc = check_tensor(scores, "scores", 2, false, LQ_F32)) != LQ_OK) return rc;
  if (finished != nullptr && (rc = check_tensor(finished, "finished", 2, false, LQ_U8)) != LQ_OK) {
    return rc;
  }
  if ((rc = check_tensor(out_scores, "out_scores", 2, false, LQ_F32)) != LQ_OK) return rc;
  if ((rc = check_tensor(out_beams, "out_beams", 2, false, LQ_I64)) != LQ_OK) return rc;
  if ((rc = check_tensor(out_tokens, "out_tokens", 2, false, LQ_I64)) != LQ_OK) return rc;
  const int64_t P = scores->shape[0], N = scores->shape[1], V = logits->shape[ldim - 1];
  const int64_t num = out_scores->shape[1];
  if (ldim == 2 ? logits->shape[0] != P * N : logits->shape[0] != P || logits->shape[1] != N) {
    return fail(LQ_ERR_INVALID_ARG, "logits must be [%lld, %lld, V] or [%lld, V]", (long long)P,
                (long long)N, (long long)(P * N));
  }
  const lq_tensor* rows[2] = {scores, finished};
  for (const lq_tensor* t : rows) {
    if (t != nullptr && (t->shape[0] != P || t->shape[1] != N)) {
      return fail(LQ_ERR_INVALID_ARG, "scores and finished must be [%lld, %lld]", (long long)P,
                  (long long)N);
    }
  }
  const lq_tensor* outs[3] = {out_scores, out_beams, out_tokens};
  for (const lq_tensor* t : outs) {
    if (t->shape[0] != P || t->shape[1] != num) {
      return fail(LQ_ERR_INVALID_ARG, "the outputs must be [%lld, %lld]", (long long)P,
                  (long long)num);
    }
  }
  if (N > MAX_BEAMS || num > MAX_NUM) {
    return fail(LQ_ERR_UNSUPPORTED, "%lld beams, %lld to select unsupported (<= %d, <= %d)",
                (long long)N, (long long)num, MAX_BEAMS, MAX_NUM);
  }
  if (V > (int64_t)LQ_BEAM_SELECT_MAX_VOCAB || P * N > 65535) {
    return fail(LQ_ERR_UNSUPPORTED, "vocabulary of %lld, %lld rows exceed the launch limits",
                (long long)V, (long long)(P * N));
  }
  if (P == 0 || num == 0) return LQ_OK;
  if (num > N * V) {
    return fail(LQ_ERR_INVALID_ARG, "%lld of %lld continuations asked for", (long long)num,
                (long long)(N * V));
  }
  if (keep_slots && num != N) {
    return fail(LQ_ERR_INVALID_ARG, "keep_slots needs as many continuations (%lld) as beams (%lld)",
                (long long)num, (long long)N);
  }
  if (finished != nullptr && (pad_token < 0 || pad_token >= V)) {
    return fail(LQ_ERR_INVALID_ARG, "pad_token=%lld outside the vocabulary of %lld",
                (long long)pad_token, (long long)V);
  }
  const size_t need = lq_beam_select_workspace(P, N, V, (int)num);
  if (workspace == nullptr || workspace_bytes < need) {
    return fail(LQ_ERR_WORKSPACE, "workspace of %zu bytes needed, %zu given", need,
                workspace == nullptr ? (size_t)0 : workspace_bytes);
  }
  if (((uintptr_t)workspace & 255) != 0) {
    return fail(LQ_ERR_WORKSPACE, "workspace must be 256-byte aligned");
  }

  SelectParams p{};
  p.logits = make_view(logits);
  if (ldim == 2) {
    p.logits.s[2] = logits->stride[1];
    p.logits.s[1] = logits->stride[0];
    p.logits.s[0] = logits->stride[0] * N;
  }
  p.scores = (const float*)scores->data;
  for (int i = 0; i < 2; ++i) {
    p.ss[i] = scores->stride[i];
    p.fs[i] = finished == nullptr ? 0 : finished->stride[i];
    for (int j = 0; j < 3; ++j) p.os[j][i] = outs[j]->stride[i];
  }
  p.finished = finished == nullptr ? nullptr : (const uint8_t*)finished->data;
  p.out_score = (float*)out_scores->data;
  p.out_beam = (int64_t*)out_beams->data;
  p.out_token = (int64_t*)out_tokens->data;
  p.pad = pad_token;
  p.P = (int)P;
  p.N = (int)N;
  p.num = (int)num;
  p.slots = keep_slots;
  p.V = V;
  const int runs = plan_runs(P * N, V);
  p.parts = parts_of(V, runs);
  const size_t slots = (size_t)(P * N) * (size_t)p.parts;
  char* ws = (char*)workspace;
  p.cap = cap_of((int)num);
  p.share = (int)((num + p.parts - 1) / p.parts);
  p.inv_cap = (uint32_t)((((uint64_t)1 << 32) + p.cap - 1) / p.cap);
  p.inv_parts = p.parts == 1 ? 0 : (uint32_t)((((uint64_t)1 << 32) + p.parts - 1) / p.parts);
  p.ws_part = (PartResult*)ws;
  p.ws_key = (uint64_t*)(ws + align256(slots * sizeof(PartResult)));
  const hipStream_t st = (hipStream_t)stream;
  const dim3 grid((unsigned)p.parts, (unsigned)(P * N));
  if (p.logits.dtype == LQ_BF16) launch_part<LQ_BF16>(p, runs, grid, st);
  else if (p.logits.dtype == LQ_F16) launch_part<LQ_F16>(p, runs, grid, st);
  else launch_part<LQ_F32>(p, runs, grid, st);
  if ((rc = check_launch("lq_beam_select")) != LQ_OK) return rc;
  // four waves for up to three rounds of candidates, sixteen above
  if (N * p.parts * p.cap <= 3 * 256) {
    hipLaunchKernelGGL(select_final_kernel<4>, dim3((unsigned)P), dim3(256), 0, st, p);
  } else {
    hipLaunchKernelGGL(select_final_kernel<16>, dim3((unsigned)P), dim3(1024), 0, st, p);
  }
  return check_launch("lq_beam_select (final)");
}
