// Beam selection: the `num` best continuations of each prompt's N beams over a vocabulary of V tokens.
//
// The total of beam n and token t is score[n] + logit[n][t] - lse[n], lse[n] the log-sum-exp of the
// beam's logits. Within a beam the order of the totals is the order of the logits, so that one pass over
// the logits gives both.
//
// select_part_kernel: a workgroup of 4 waves takes a part of one beam's row in runs of 1024 logits per
// wave (16 per lane). Each lane keeps a running maximum and the sum of e^(x - maximum); each wave keeps a
// list of the logits above a threshold that only rises: the num-th largest of the lanes' maxima where
// at least that many lanes pass it (num logits are then at least as large), and the num-th largest of the
// list where the list is full. The num-th largest of the values in a wave's registers is found bit by
// bit with ballots (kth_word), with no exchange between lanes. The part leaves (max, sum) and its num
// largest logits, ties by the lower token.
//
// select_final_kernel: one workgroup per prompt makes lse[n] and the totals of the parts' candidates in
// 64 bits (their order then goes wrong only where totals are closer than the sums' rounding, about
// 1e-7), reduces them 256 per wave to num per wave until one wave holds them, sorts those and writes
// them out, by rank or by place.
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
constexpr int FINAL_WAVES = 16;     // waves of a prompt's workgroup
constexpr int FINAL_MAX = 256 * FINAL_WAVES;  // candidates of a prompt
static_assert(MAX_BEAMS * MAX_NUM <= FINAL_MAX, "one part per beam always fits");

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
  int parts, runs;      // parts of a row, runs of a part
  float* ws_m;          // [rows][parts]
  float* ws_s;
  uint64_t* ws_key;     // [rows][parts][num]: order of the logit, then of the token; 0: none
};

constexpr float LOG2E_F = 1.44269504f;

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

template <int DT>
struct Vec {
  static constexpr int N = DT == LQ_F32 ? 4 : 8;  // logits of 16 bytes
  static constexpr int LOADS = PER / N;
  uint4 raw[LOADS];
};

template <int DT>
__device__ __forceinline__ void unpack(const Vec<DT>& v, float (&x)[PER]) {
#pragma unroll
  for (int j = 0; j < Vec<DT>::LOADS; ++j) {
    const uint32_t w[4] = {v.raw[j].x, v.raw[j].y, v.raw[j].z, v.raw[j].w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (DT == LQ_F32) {
        x[4 * j + i] = __uint_as_float(w[i]);
      } else {
        x[8 * j + 2 * i] = word_elem(w[i], 0, DT);
        x[8 * j + 2 * i + 1] = word_elem(w[i], 16, DT);
      }
    }
  }
}

// 16 bytes at any address: the order of a row's sums must not depend on where the row starts, so that
// beams with equal logits get equal totals (a row of an odd vocabulary starts at any multiple of 2 bytes).
struct __attribute__((packed, aligned(2))) Unaligned16 {
  uint4 v;
};

// DENSE: the logits of a row are contiguous and loaded 16 bytes per lane, but for the row's last run.
// Otherwise, and there, one element at a time.
template <int DT, bool DENSE>
__global__ __launch_bounds__(THREADS) void select_part_kernel(SelectParams p) {
  __shared__ uint64_t lists[WAVES][LIST];
  __shared__ int counts[WAVES];
  __shared__ float wave_m[WAVES], wave_s[WAVES];
  constexpr int VN = Vec<DT>::N;
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  const int64_t row = blockIdx.y;
  const int64_t prompt = row / p.N, beam = row - prompt * p.N;
  if (p.finished != nullptr && p.finished[prompt * p.fs[0] + beam * p.fs[1]] != 0) return;
  const int64_t base = prompt * p.logits.s[0] + beam * p.logits.s[1];
  const char* first = (const char*)p.logits.data + base * (DT == LQ_F32 ? 4 : 2);
  const int r0 = blockIdx.x * p.runs;
  const int nruns = (int)min((int64_t)p.runs, (p.V + RUN - 1) / RUN - r0);
  const int k = p.num;
  uint64_t* list = lists[wave];

  // token of the lane's logit i of the run from token `start` on
  auto token = [&](uint32_t start, int i) -> uint32_t {
    return DENSE ? start + ((i / VN) * 64 + lane) * VN + i % VN : start + i * 64 + lane;
  };
  auto load = [&](int r, Vec<DT>& v) {
    const int64_t start = (int64_t)(r0 + r) * RUN;
    if constexpr (DENSE) {
      if (r >= nruns || start + RUN > p.V) return;
      const Unaligned16* at = (const Unaligned16*)(first + start * (DT == LQ_F32 ? 4 : 2)) + lane;
#pragma unroll
      for (int j = 0; j < Vec<DT>::LOADS; ++j) v.raw[j] = at[64 * j].v;
    }
  };

  float ml = -INFINITY, sl = 0.0f;  // the lane's maximum and sum
  int n = 0;                        // entries of the list
  uint64_t bar = 0;                 // only larger keys are taken, whose logits reach barf
  float barf = -INFINITY;
  Vec<DT> next;
  load(wave, next);
  for (int r = wave; r < nruns; r += WAVES) {
    const uint32_t start = (uint32_t)(r0 + r) * RUN;
    float x[PER];
    uint32_t valid = 0xffffu;
    if (DENSE && (int64_t)start + RUN <= p.V) {
      unpack<DT>(next, x);
      load(r + WAVES, next);
    } else {
      valid = 0;
#pragma unroll
      for (int i = 0; i < PER; ++i) {
        const uint32_t t = token(start, i);
        x[i] = -INFINITY;
        if (t < (uint32_t)p.V) {
          x[i] = load_float(p.logits.data, DT, base + (int64_t)t * p.logits.s[2]);
          valid |= 1u << i;
        }
      }
    }
    float mx = x[0];
#pragma unroll
    for (int i = 1; i < PER; ++i) mx = fmaxf(mx, x[i]);
    if (mx > ml) {
      sl *= __builtin_amdgcn_exp2f((ml - mx) * LOG2E_F);
      ml = mx;
    }
    const float m0 = ml == -INFINITY ? 0.0f : ml;
#pragma unroll
    for (int i = 0; i < PER; ++i) sl += __builtin_amdgcn_exp2f((x[i] - m0) * LOG2E_F);

    const uint64_t lanes = __ballot(mx >= barf);
    if (lanes == 0) continue;
    if (count(lanes) >= k) {
      // k lanes' largest logits at least reach it: the k-th largest of those is a threshold
      uint32_t v[1] = {valid != 0 ? order_bits(mx) : 0};
      const int have = count(__ballot(v[0] != 0));
      if (have >= k) {
        bool exact = false;
        uint32_t w = 0;
        if (have == k) {
          w = wave_fold(v[0] != 0 ? v[0] : ~0u, [](uint32_t a, uint32_t b) { return min(a, b); });
        } else {
          w = kth_word<1>(v, k, exact);
        }
        uint64_t low = (uint64_t)w << 32;
        if (!exact && count_from<1>(v, w) > k + 8) {
          // many lanes tie (banned or equal logits): of those the ones with the lowest tokens count
          uint32_t t = 0;
#pragma unroll
          for (int i = PER - 1; i >= 0; --i) {
            if (x[i] == mx && (valid >> i & 1) != 0) t = 0xffffffffu - token(start, i);
          }
          const int need = k - count(__ballot(v[0] > w));
          v[0] = v[0] == w ? t : 0;
          low |= kth_word<1>(v, need, exact);
        }
        if (low != 0 && low - 1 > bar) {
          bar = low - 1;
          barf = from_order_bits(w);
        }
      }
    }
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      if (__ballot(x[i] >= barf) == 0) continue;
      const uint64_t key = make_key(x[i], token(start, i));
      bool ok = x[i] >= barf && (valid >> i & 1) != 0 && key > bar;
      uint64_t b = __ballot(ok);
      if (n + count(b) > LIST) {
        cut_list(list, n, k, bar, barf);
        ok = ok && key > bar;
        b = __ballot(ok);
      }
      if (ok) list[n + below(b)] = key;
      n += count(b);
    }
    __builtin_amdgcn_wave_barrier();
  }
  if (n > k) cut_list(list, n, k, bar, barf);

  const float wm = group_max<64>(ml);
  const float ws = group_sum<64>(sl * (ml == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f((ml - wm) * LOG2E_F)));
  if (lane == 0) {
    counts[wave] = n;
    wave_m[wave] = wm;
    wave_s[wave] = ws;
  }
  __syncthreads();
  if (wave != 0) return;
  const int64_t slot = row * p.parts + blockIdx.x;
  float M = wave_m[0], S = 0.0f;
#pragma unroll
  for (int w = 1; w < WAVES; ++w) M = fmaxf(M, wave_m[w]);
#pragma unroll
  for (int w = 0; w < WAVES; ++w) {
    S += wave_s[w] * (wave_m[w] == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f((wave_m[w] - M) * LOG2E_F));
  }
  uint64_t key[WAVES];
  bool take[WAVES];
#pragma unroll
  for (int w = 0; w < WAVES; ++w) key[w] = lane < counts[w] ? lists[w][lane] : 0;
  __builtin_amdgcn_wave_barrier();
  take_keys<WAVES>(key, k, take);
  int total = 0;
#pragma unroll
  for (int w = 0; w < WAVES; ++w) {
    const uint64_t b = __ballot(take[w]);
    if (take[w]) list[total + below(b)] = key[w];
    total += count(b);
  }
  __builtin_amdgcn_wave_barrier();
  if (lane == 0) {
    p.ws_m[slot] = M;
    p.ws_s[slot] = S;
  }
  if (lane < k) p.ws_key[slot * k + lane] = lane < total ? list[lane] : 0;
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
  // (the low words are compared above 0: their lowest bit is set aside and does not decide)
#pragma unroll
  for (int e = 0; e < 4; ++e) v[e] = v[e] != 0 ? (uint32_t)order_bits64(c[e].total) | 1u : 0;
  narrow<4>(v, take, need);
  if (need == 0) return;
#pragma unroll
  for (int e = 0; e < 4; ++e) v[e] = v[e] != 0 ? ~c[e].index : 0;
  narrow<4>(v, take, need);
}

__global__ __launch_bounds__(64 * FINAL_WAVES) void select_final_kernel(SelectParams p) {
  __shared__ double base[MAX_BEAMS];   // score - lse; -inf: no candidate above -inf
  __shared__ bool alone[MAX_BEAMS];    // a finished beam
  __shared__ double c_total[2][FINAL_WAVES * MAX_NUM];
  __shared__ uint32_t c_index[2][FINAL_WAVES * MAX_NUM];
  __shared__ int c_count[2][FINAL_WAVES];
  const int64_t prompt = blockIdx.x;
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  const int k = p.num;
  for (int n = wave; n < p.N; n += FINAL_WAVES) {
    const int64_t row = prompt * p.N + n;
    const bool fin = p.finished != nullptr && p.finished[prompt * p.fs[0] + n * p.fs[1]] != 0;
    const float score = p.scores[prompt * p.ss[0] + n * p.ss[1]];
    double b = score;
    if (!fin) {
      float m = -INFINITY;
      for (int c = lane; c < p.parts; c += 64) m = fmaxf(m, p.ws_m[row * p.parts + c]);
      m = group_max<64>(m);
      double s = 0.0;
      for (int c = lane; c < p.parts; c += 64) {
        const float mc = p.ws_m[row * p.parts + c], sc = p.ws_s[row * p.parts + c];
        s += (double)(sc * (mc == -INFINITY ? 0.0f : exp2f((mc - m) * LOG2E_F)));
      }
#pragma unroll
      for (int o = 32; o > 0; o >>= 1) s += __shfl_xor(s, o, 64);
      b = (double)score - ((double)m + log(s));
    }
    if (lane == 0) {
      alone[n] = fin;
      base[n] = fabs(b) < INFINITY ? b : -INFINITY;
    }
  }
  __syncthreads();

  // first level: candidates from the parts' lists, 256 per wave
  const int per_row = p.parts * k;
  const int all = p.N * per_row;  // <= FINAL_MAX
  const uint32_t V = (uint32_t)p.V;
  Candidate c[4];
  bool on[4], take[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const int at = 256 * wave + 64 * e + lane;
    c[e] = Candidate{-INFINITY, 0};
    on[e] = false;
    if (at < all) {
      const int n = at / per_row;
      const int j = at - n * per_row;
      if (alone[n] || base[n] == -INFINITY) {
        // a finished beam's own score at the pad token, then the lowest tokens at -inf
        on[e] = j < k && (uint32_t)j < V;
        uint32_t token = j;
        if (alone[n]) {
          token = j == 0 ? (uint32_t)p.pad : ((uint32_t)j <= (uint32_t)p.pad ? j - 1 : j);
          if (j == 0) c[e].total = base[n];
        }
        c[e].index = n * V + token;
      } else {
        const uint64_t key = p.ws_key[(prompt * p.N + n) * per_row + j];
        on[e] = key != 0;
        c[e].total = base[n] + (double)from_order_bits((uint32_t)(key >> 32));
        c[e].index = n * V + (0xffffffffu - (uint32_t)key);
      }
    }
  }
  int level = 0;
  int waves = (all + 255) / 256;  // waves with candidates
  while (true) {
    if (wave < waves) {
      take_candidates(c, on, k, take);
      int total = 0;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const uint64_t b = __ballot(take[e]);
        if (take[e]) {
          c_total[level & 1][wave * k + total + below(b)] = c[e].total;
          c_index[level & 1][wave * k + total + below(b)] = c[e].index;
        }
        total += count(b);
      }
      if (lane == 0) c_count[level & 1][wave] = total;
    }
    __syncthreads();
    if (waves == 1) break;
    // next level: the waves' k places, 256 per wave
    const int places = waves * k;
    waves = (places + 255) / 256;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int at = 256 * wave + 64 * e + lane;
      on[e] = at < places && at % k < c_count[level & 1][at / k];
      c[e] = on[e] ? Candidate{c_total[level & 1][at], c_index[level & 1][at]} : Candidate{-INFINITY, 0};
    }
    ++level;
  }
  if (wave != 0) return;

  // the k chosen ones (there are k: num <= N * V), one per lane, by rank
  const double total = lane < k ? c_total[level & 1][lane] : -INFINITY;
  const uint32_t index = lane < k ? c_index[level & 1][lane] : 0xffffffffu;
  int rank = 0;
  for (int j = 0; j < k; ++j) {
    const double t = c_total[level & 1][j];
    const uint32_t i = c_index[level & 1][j];
    rank += t > total || (t == total && i < index) ? 1 : 0;
  }
  const int beam = (int)(index / V);
  int at = rank;
  if (p.slots) {
    // a beam's best continuation keeps the beam's place, the others take the free places in order
    uint64_t used = 0;
    bool best = lane < k;
    for (int j = 0; j < k; ++j) {
      const int b = __builtin_amdgcn_readlane(beam, j);
      const int r = __builtin_amdgcn_readlane(rank, j);
      used |= (uint64_t)1 << b;
      best = best && !(b == beam && r < rank);
    }
    int before = 0;  // other continuations of a better rank that have no place of their own
    const uint64_t bests = __ballot(best);
    for (int j = 0; j < k; ++j) {
      const int r = __builtin_amdgcn_readlane(rank, j);
      before += (bests >> j & 1) == 0 && r < rank ? 1 : 0;
    }
    uint64_t free = ~used;
    if (!best) {
      for (int j = 0; j < before; ++j) free &= free - 1;
    }
    at = best ? beam : __builtin_ctzll(free);
  }
  if (lane < k) {
    p.out_score[prompt * p.os[0][0] + at * p.os[0][1]] = (float)total;
    p.out_beam[prompt * p.os[1][0] + at * p.os[1][1]] = beam;
    p.out_token[prompt * p.os[2][0] + at * p.os[2][1]] = index - (uint32_t)beam * V;
  }
}

// Parts of a row: of whole rounds of 4 runs, about 2048 workgroups in all, as far as the prompt's
// candidates still fit the final workgroup.
struct SelectPlan {
  int parts, runs;
};

SelectPlan plan_select(int64_t P, int64_t N, int64_t V, int num) {
  const int64_t runs = (V + RUN - 1) / RUN;
  const int64_t most = std::max<int64_t>(1, FINAL_MAX / (N * num));
  const int64_t want = std::min(most, std::max<int64_t>(1, (2048 + P * N - 1) / (P * N)));
  int64_t per = (runs + want - 1) / want;
  per = (per + WAVES - 1) / WAVES * WAVES;
  return SelectPlan{(int)((runs + per - 1) / per), (int)per};
}

template <int DT>
void launch_part(const SelectParams& p, dim3 grid, hipStream_t st) {
  if (p.logits.s[2] == 1) {
    hipLaunchKernelGGL((select_part_kernel<DT, true>), grid, dim3(THREADS), 0, st, p);
  } else {
    hipLaunchKernelGGL((select_part_kernel<DT, false>), grid, dim3(THREADS), 0, st, p);
  }
}

size_t align256(size_t n) { return (n + 255) / 256 * 256; }

}  // namespace
}  // namespace lq

using namespace lq;

extern "C" size_t lq_beam_select_workspace(int64_t prompts, int64_t beams, int64_t vocab, int num) {
  if (prompts <= 0 || beams <= 0 || vocab <= 0 || num <= 0) return 0;
  const size_t slots = (size_t)(prompts * beams) * (size_t)plan_select(prompts, beams, vocab, num).parts;
  return 2 * align256(slots * 4) + slots * (size_t)num * 8;
}

extern "C" int lq_beam_select(const lq_tensor* logits, const lq_tensor* scores,
                              const lq_tensor* finished, const lq_tensor* out_scores,
                              const lq_tensor* out_beams, const lq_tensor* out_tokens,
                              int64_t pad_token, int keep_slots, void* workspace,
                              size_t workspace_bytes, void* stream) {
  int rc;
  if ((rc = check_tensor(logits, "logits", 3, true)) != LQ_OK) return rc;
  if ((rc = check_tensor(scores, "scores", 2, false, LQ_F32)) != LQ_OK) return rc;
  if (finished != nullptr && (rc = check_tensor(finished, "finished", 2, false, LQ_U8)) != LQ_OK) {
    return rc;
  }
  if ((rc = check_tensor(out_scores, "out_scores", 2, false, LQ_F32)) != LQ_OK) return rc;
  if ((rc = check_tensor(out_beams, "out_beams", 2, false, LQ_I64)) != LQ_OK) return rc;
  if ((rc = check_tensor(out_tokens, "out_tokens", 2, false, LQ_I64)) != LQ_OK) return rc;
  const int64_t P = logits->shape[0], N = logits->shape[1], V = logits->shape[2];
  const int64_t num = out_scores->shape[1];
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
  const SelectPlan plan = plan_select(P, N, V, (int)num);
  p.parts = plan.parts;
  p.runs = plan.runs;
  const size_t slots = (size_t)(P * N) * (size_t)p.parts;
  char* ws = (char*)workspace;
  p.ws_m = (float*)ws;
  p.ws_s = (float*)(ws + align256(slots * 4));
  p.ws_key = (uint64_t*)(ws + 2 * align256(slots * 4));
  const hipStream_t st = (hipStream_t)stream;
  const dim3 grid((unsigned)p.parts, (unsigned)(P * N));
  if (p.logits.dtype == LQ_BF16) launch_part<LQ_BF16>(p, grid, st);
  else if (p.logits.dtype == LQ_F16) launch_part<LQ_F16>(p, grid, st);
  else launch_part<LQ_F32>(p, grid, st);
  if ((rc = check_launch("lq_beam_select")) != LQ_OK) return rc;
  hipLaunchKernelGGL(select_final_kernel, dim3((unsigned)P), dim3(64 * FINAL_WAVES), 0, st, p);
  return check_launch("lq_beam_select (final)");
}
