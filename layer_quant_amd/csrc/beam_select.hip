// Beam selection: the `num` best continuations of each prompt's N beams over a vocabulary of V tokens.
//
// The total of beam n and token t is score[n] + logit[n][t] - lse[n], lse[n] the log-sum-exp of the
// beam's logits. Within a beam the order of the totals is the order of the logits, so that the logits
// are read once: each workgroup takes a chunk of one beam's row and leaves the chunk's maximum m,
// sum_t 2^((x_t - m) log2 e) and its `num` largest logits (ties by the lower token); a second kernel,
// one workgroup per prompt, makes lse[n] = M + log(sum_c s_c e^(m_c - M)) and the totals in 64 bits
// (their order then goes wrong only where totals are closer than the sums' rounding, about 1e-7) and
// takes the best `num` of the chunks' candidates.
#include <math.h>

#include <algorithm>

#include "lq_common.h"

namespace lq {
namespace {

constexpr int MAX_BEAMS = LQ_BEAM_SELECT_MAX_BEAMS;
constexpr int MAX_NUM = LQ_BEAM_SELECT_MAX_NUM;
constexpr int THREADS = 256;
constexpr int PER = 16;                 // logits per thread
constexpr int CHUNK = THREADS * PER;    // logits per workgroup

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
  int chunks;
  float* ws_m;          // [rows][chunks]
  float* ws_s;
  uint64_t* ws_key;     // [rows][chunks][num]: order of the logit, then of the token
};

// An unsigned integer in the order of the floats; a NaN is below every number.
__device__ __forceinline__ uint32_t order_bits(float x) {
  if (x != x) return 0u;
  const uint32_t u = __float_as_uint(x + 0.0f);  // -0 counts as 0
  return u ^ ((u >> 31) != 0 ? 0xffffffffu : 0x80000000u);
}

__device__ __forceinline__ float from_order_bits(uint32_t k) {
  return __uint_as_float(k ^ ((k >> 31) != 0 ? 0x80000000u : 0xffffffffu));
}

// Larger is better: the logit, then the lower token.
__device__ __forceinline__ uint64_t make_key(float x, uint32_t token) {
  return ((uint64_t)order_bits(x) << 32) | (0xffffffffu - token);
}

__device__ __forceinline__ uint64_t wave_max_u64(uint64_t v) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) {
    const uint64_t w = __shfl_xor((unsigned long long)v, o, 64);
    v = w > v ? w : v;
  }
  return v;
}

__device__ __forceinline__ uint64_t block_max_u64(uint64_t v, uint64_t* red) {
  v = wave_max_u64(v);
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
  __syncthreads();
  uint64_t r = red[0];
#pragma unroll
  for (int i = 1; i < THREADS / 64; ++i) r = red[i] > r ? red[i] : r;
  __syncthreads();
  return r;
}

__global__ __launch_bounds__(THREADS) void select_chunk_kernel(SelectParams p) {
  __shared__ uint64_t red[THREADS / 64];
  __shared__ float fred[THREADS / 64];
  const int64_t row = blockIdx.y;
  const int64_t prompt = row / p.N, beam = row - prompt * p.N;
  if (p.finished != nullptr && p.finished[prompt * p.fs[0] + beam * p.fs[1]] != 0) return;
  const int64_t base = prompt * p.logits.s[0] + beam * p.logits.s[1];
  const int64_t t0 = (int64_t)blockIdx.x * CHUNK;
  float x[PER];
  uint64_t key[PER];
  float m = -INFINITY;
  bool nan = false;
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const int64_t t = t0 + i * THREADS + threadIdx.x;
    x[i] = t < p.V ? load_float(p.logits.data, p.logits.dtype, base + t * p.logits.s[2]) : -INFINITY;
    key[i] = t < p.V ? make_key(x[i], (uint32_t)t) : 0;
    nan = nan || x[i] != x[i];
    m = fmaxf(m, x[i]);
  }
  const float wm = group_max<64>(m);
  if ((threadIdx.x & 63) == 0) fred[threadIdx.x >> 6] = wm;
  __syncthreads();
  m = fmaxf(fmaxf(fred[0], fred[1]), fmaxf(fred[2], fred[3]));
  __syncthreads();
  float s = 0.0f;
  if (m != -INFINITY) {
#pragma unroll
    for (int i = 0; i < PER; ++i) s += __builtin_amdgcn_exp2f((x[i] - m) * 1.44269504f);
  }
  if (nan) s = NAN;
  s = group_sum<64>(s);
  if ((threadIdx.x & 63) == 0) fred[threadIdx.x >> 6] = s;
  __syncthreads();
  const int64_t slot = row * p.chunks + blockIdx.x;
  if (threadIdx.x == 0) {
    p.ws_m[slot] = m;
    p.ws_s[slot] = fred[0] + fred[1] + fred[2] + fred[3];
  }
  uint64_t last = ~(uint64_t)0;
  for (int k = 0; k < p.num; ++k) {
    uint64_t best = 0;
#pragma unroll
    for (int i = 0; i < PER; ++i) best = key[i] < last && key[i] > best ? key[i] : best;
    last = block_max_u64(best, red);
    if (threadIdx.x == 0) p.ws_key[slot * p.num + k] = last;  // 0: no further token
  }
}

// (total, flat index) of a candidate: larger totals first, then the lower index.
__device__ __forceinline__ bool better(double a, int64_t ia, double b, int64_t ib) {
  return a > b || (a == b && ia < ib);
}

__global__ __launch_bounds__(THREADS) void select_final_kernel(SelectParams p) {
  __shared__ double base[MAX_BEAMS];   // score - lse; -inf: no candidate above -inf
  __shared__ bool alone[MAX_BEAMS];    // a finished beam
  __shared__ double s_t[THREADS / 64];
  __shared__ int64_t s_i[THREADS / 64];
  __shared__ float o_score[MAX_NUM];
  __shared__ int o_beam[MAX_NUM];
  __shared__ int64_t o_token[MAX_NUM];
  __shared__ int place[MAX_NUM];
  const int64_t prompt = blockIdx.x;
  const int tid = threadIdx.x;
  for (int n = tid; n < p.N; n += THREADS) {
    const int64_t row = prompt * p.N + n;
    const bool fin = p.finished != nullptr && p.finished[prompt * p.fs[0] + n * p.fs[1]] != 0;
    const float score = p.scores[prompt * p.ss[0] + n * p.ss[1]];
    double b = score;
    if (!fin) {
      float m = -INFINITY;
      for (int c = 0; c < p.chunks; ++c) m = fmaxf(m, p.ws_m[row * p.chunks + c]);
      double s = 0.0;
      for (int c = 0; c < p.chunks; ++c) {
        const float mc = p.ws_m[row * p.chunks + c];
        if (mc != -INFINITY || p.ws_s[row * p.chunks + c] != 0.0f) {
          s += (double)p.ws_s[row * p.chunks + c] * exp((double)mc - (double)m);
        }
      }
      b = (double)score - ((double)m + log(s));
    }
    alone[n] = fin;
    base[n] = fabs(b) < INFINITY ? b : -INFINITY;
  }
  __syncthreads();

  const int per_row = p.chunks * p.num;
  const int64_t all = (int64_t)p.N * per_row;
  // candidate c as (total, flat index n * V + token); false when there is none
  auto candidate = [&](int64_t c, double& t, int64_t& idx) -> bool {
    const int n = (int)(c / per_row);
    const int j = (int)(c - (int64_t)n * per_row);
    if (alone[n] || base[n] == -INFINITY) {
      // a finished beam's own score at the pad token, then the lowest tokens at -inf
      if (j >= p.num || j >= p.V) return false;
      int64_t token = j;
      t = -INFINITY;
      if (alone[n]) {
        token = j == 0 ? p.pad : (j <= p.pad ? j - 1 : j);
        if (j == 0) t = base[n];
      }
      idx = n * p.V + token;
      return true;
    }
    const uint64_t key = p.ws_key[(prompt * p.N + n) * per_row + j];
    if (key == 0) return false;
    t = base[n] + (double)from_order_bits((uint32_t)(key >> 32));
    idx = n * p.V + (0xffffffffu - (uint32_t)key);
    return true;
  };

  double lt = INFINITY;
  int64_t li = -1;  // the last one taken
  for (int k = 0; k < p.num; ++k) {
    double bt = -INFINITY;
    int64_t bi = INT64_MAX;
    for (int64_t c = tid; c < all; c += THREADS) {
      double t;
      int64_t idx;
      if (!candidate(c, t, idx)) continue;
      if (better(lt, li, t, idx) && better(t, idx, bt, bi)) {
        bt = t;
        bi = idx;
      }
    }
    for (int o = 32; o > 0; o >>= 1) {
      const double t = __shfl_xor(bt, o, 64);
      const int64_t i = __shfl_xor((long long)bi, o, 64);
      if (better(t, i, bt, bi)) {
        bt = t;
        bi = i;
      }
    }
    if ((tid & 63) == 0) {
      s_t[tid >> 6] = bt;
      s_i[tid >> 6] = bi;
    }
    __syncthreads();
    for (int w = 0; w < THREADS / 64; ++w) {
      if (better(s_t[w], s_i[w], bt, bi)) {
        bt = s_t[w];
        bi = s_i[w];
      }
    }
    __syncthreads();
    lt = bt;
    li = bi;
    if (tid == 0) {
      o_score[k] = (float)bt;
      o_beam[k] = (int)(bi / p.V);
      o_token[k] = bi % p.V;
      place[k] = k;
    }
  }
  __syncthreads();
  if (p.slots && tid == 0) {
    // a beam's best continuation keeps the beam's place, the others take the free places in order
    uint64_t used = 0, kept = 0;
    for (int k = 0; k < p.num; ++k) used |= (uint64_t)1 << o_beam[k];
    uint64_t free = ~used;
    for (int k = 0; k < p.num; ++k) {
      const uint64_t bit = (uint64_t)1 << o_beam[k];
      if ((kept & bit) == 0) {
        kept |= bit;
        place[k] = o_beam[k];
      } else {
        place[k] = __builtin_ctzll(free);
        free &= free - 1;
      }
    }
  }
  __syncthreads();
  for (int k = tid; k < p.num; k += THREADS) {
    const int at = place[k];
    p.out_score[prompt * p.os[0][0] + at * p.os[0][1]] = o_score[k];
    p.out_beam[prompt * p.os[1][0] + at * p.os[1][1]] = o_beam[k];
    p.out_token[prompt * p.os[2][0] + at * p.os[2][1]] = o_token[k];
  }
}

int chunks_of(int64_t V) { return (int)((V + CHUNK - 1) / CHUNK); }

size_t align256(size_t n) { return (n + 255) / 256 * 256; }

}  // namespace
}  // namespace lq

using namespace lq;

extern "C" size_t lq_beam_select_workspace(int64_t prompts, int64_t beams, int64_t vocab, int num) {
  if (prompts <= 0 || beams <= 0 || vocab <= 0 || num <= 0) return 0;
  const size_t slots = (size_t)(prompts * beams) * (size_t)chunks_of(vocab);
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
  p.chunks = chunks_of(V);
  const size_t slots = (size_t)(P * N) * (size_t)p.chunks;
  char* ws = (char*)workspace;
  p.ws_m = (float*)ws;
  p.ws_s = (float*)(ws + align256(slots * 4));
  p.ws_key = (uint64_t*)(ws + 2 * align256(slots * 4));
  const hipStream_t st = (hipStream_t)stream;
  hipLaunchKernelGGL(select_chunk_kernel, dim3((unsigned)p.chunks, (unsigned)(P * N)), dim3(THREADS),
                     0, st, p);
  if ((rc = check_launch("lq_beam_select")) != LQ_OK) return rc;
  hipLaunchKernelGGL(select_final_kernel, dim3((unsigned)P), dim3(THREADS), 0, st, p);
  return check_launch("lq_beam_select (final)");
}
