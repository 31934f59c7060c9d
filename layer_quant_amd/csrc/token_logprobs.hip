// Log-probabilities of given tokens, the entropy of each row and its likeliest tokens (no reference
// counterpart; beam_select.hip selects over beams and vocabulary by the same log-softmax):
//
//   lse = log sum_v exp(l_v),  logprob = l_token - lse,  entropy = lse - sum_v p_v l_v
//
// One pass over the logits. A workgroup takes a part of a row into registers, 32 logits per thread, and
// leaves m = max l log2(e), s = sum 2^z and t = sum 2^z z with z = l log2(e) - m, and its `top` largest
// logits; the row's workgroup then joins the parts. fp32 sums. Every z is made from the rounded m by one
// fused multiply-add, the given token's too, so that m's rounding falls out of logprob and entropy.
//
// Order: the larger logit first, of equal ones (and of 0 and -0) the lower token. -inf logits have no
// part in the sums. A row with a NaN or an infinity, or with -inf alone, has no distribution: NaN.
#include <math.h>

#include "lq_common.h"

namespace lq {
namespace {

constexpr int THREADS = 256;
constexpr int VPT = 32;               // logits per thread
constexpr int PART = THREADS * VPT;   // logits of a part
constexpr int MAX_TOP = 32;
constexpr float LOG2E = 1.44269504088896340736f, LN2 = 0.69314718055994530942f;

struct LogprobParams {
  View logits;  // strides of (batch row, row, token)
  View tokens;  // strides of (batch row, row)
  float *logprobs, *entropy, *top_logprobs;
  int64_t* top_tokens;
  int rows, parts, top, len;  // len: rows of a batch row
  int64_t V;
  float* stats;    // [rows][parts][4]: m, s, t
  uint64_t* keys;  // [rows][parts][top]
};

// Larger for the logit that comes first: its bits in order, then the lower token. 0: none.
__device__ __forceinline__ uint64_t key_of(float l, uint32_t token) {
  const uint32_t u = __float_as_uint(l + 0.f);
  const uint32_t up = (u >> 31) ? ~u : u | 0x80000000u;
  return ((uint64_t)up << 32) | (0xffffffffu - token);
}
__device__ __forceinline__ float logit_of(uint64_t key) {
  const uint32_t up = (uint32_t)(key >> 32);
  return __uint_as_float((up >> 31) ? up & 0x7fffffffu : ~up);
}

__device__ __forceinline__ int64_t row_at(const LogprobParams& p, int row) {
  const int b = row / p.len;
  return b * p.logits.s[0] + (row - b * p.len) * p.logits.s[1];
}

__device__ __forceinline__ uint64_t wave_max(uint64_t v) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) {
    const uint32_t lo = __shfl_xor((uint32_t)v, o, 64), hi = __shfl_xor((uint32_t)(v >> 32), o, 64);
    const uint64_t w = ((uint64_t)hi << 32) | lo;
    v = w > v ? w : v;
  }
  return v;
}

template <int DTYPE>
__global__ __launch_bounds__(THREADS) void logprob_part_kernel(LogprobParams p) {
  __shared__ float red[3][THREADS / 64];
  __shared__ uint64_t best[THREADS / 64];
  const int row = blockIdx.x / p.parts, part = blockIdx.x % p.parts;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int64_t base = row_at(p, row);
  const int64_t first = (int64_t)part * PART + tid;
  float l[VPT];
#pragma unroll
  for (int i = 0; i < VPT; ++i) {
    const int64_t v = first + (int64_t)i * THREADS;
    l[i] = v < p.V ? load_float(p.logits.data, DTYPE, base + v * p.logits.s[2]) : -INFINITY;
  }
  float m = -INFINITY;
#pragma unroll
  for (int i = 0; i < VPT; ++i) m = fmaxf(m, l[i]);
  m = group_max<64>(m);
  if (lane == 0) red[0][wave] = m;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < THREADS / 64; ++w) m = fmaxf(m, red[0][w]);
  // a part of -inf alone has s = 0
  m *= LOG2E;
  const float mz = m == -INFINITY ? 0.f : m;
  float s = 0.f, t = 0.f;
#pragma unroll
  for (int i = 0; i < VPT; ++i) {
    const float z = fmaf(l[i], LOG2E, -mz);
    const float e = __builtin_amdgcn_exp2f(z);  // NaN stays; 0 for -inf
    s += e;
    t = fmaf(e, fmaxf(z, -200.f), t);
  }
  s = group_sum<64>(s);
  t = group_sum<64>(t);
  __syncthreads();
  if (lane == 0) {
    red[1][wave] = s;
    red[2][wave] = t;
  }
  __syncthreads();
  if (tid == 0) {
    float* to = p.stats + ((int64_t)row * p.parts + part) * 4;
    s = t = 0.f;
    for (int w = 0; w < THREADS / 64; ++w) {
      s += red[1][w];
      t += red[2][w];
    }
    to[0] = m;
    to[1] = s;
    to[2] = t;
  }
  uint64_t last = ~0ull;
  for (int k = 0; k < p.top; ++k) {
    uint64_t b = 0;
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      const int64_t v = first + (int64_t)i * THREADS;
      if (v >= p.V) continue;
      const uint64_t key = key_of(l[i], (uint32_t)v);
      if (key < last && key > b) b = key;
    }
    b = wave_max(b);
    __syncthreads();
    if (lane == 0) best[wave] = b;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < THREADS / 64; ++w) b = best[w] > b ? best[w] : b;
    last = b;
    if (tid == 0) p.keys[((int64_t)row * p.parts + part) * p.top + k] = b;
  }
}

// One wave per row.
__global__ __launch_bounds__(64) void logprob_final_kernel(LogprobParams p) {
  const int row = blockIdx.x, lane = threadIdx.x;
  const float* st = p.stats + (int64_t)row * p.parts * 4;
  float m = -INFINITY;
  for (int i = lane; i < p.parts; i += 64) m = fmaxf(m, st[4 * i]);
  m = group_max<64>(m);
  const float mz = m == -INFINITY ? 0.f : m;
  float s = 0.f, t = 0.f;
  for (int i = lane; i < p.parts; i += 64) {
    const float d = fmaxf(st[4 * i] - mz, -200.f);
    const float w = __builtin_amdgcn_exp2f(d);
    s = fmaf(w, st[4 * i + 1], s);
    t = fmaf(w, fmaf(d, st[4 * i + 1], st[4 * i + 2]), t);
  }
  s = group_sum<64>(s);
  t = group_sum<64>(t);
  const float log2s = __log2f(s);
  const bool known = s > 0.f && s < INFINITY && m < INFINITY;
  const float nan = __builtin_nanf("");
  if (lane == 0) {
    const int b = row / p.len;
    const int64_t token = ((const int64_t*)p.tokens.data)[b * p.tokens.s[0] + (row - b * p.len) * p.tokens.s[1]];
    float lp = 0.f;
    if (token >= 0 && token < p.V) {
      const float l = load_float(p.logits.data, p.logits.dtype, row_at(p, row) + token * p.logits.s[2]);
      lp = known ? (fmaf(l, LOG2E, -mz) - log2s) * LN2 : nan;
    }
    p.logprobs[row] = lp;
    if (p.entropy != nullptr) p.entropy[row] = known ? LN2 * (log2s - t / s) : nan;
  }
  const uint64_t* keys = p.keys + (int64_t)row * p.parts * p.top;
  uint64_t last = ~0ull;
  for (int k = 0; k < p.top; ++k) {
    uint64_t b = 0;
    for (int i = lane; i < p.parts * p.top; i += 64) {
      const uint64_t key = keys[i];
      if (key < last && key > b) b = key;
    }
    b = wave_max(b);
    last = b;
    if (lane == 0) {
      const int64_t at = (int64_t)row * p.top + k;
      p.top_logprobs[at] = known ? (fmaf(logit_of(b), LOG2E, -mz) - log2s) * LN2 : nan;
      p.top_tokens[at] = known ? (int64_t)(0xffffffffu - (uint32_t)b) : k;
    }
  }
}

size_t align256(size_t n) { return (n + 255) & ~(size_t)255; }

}  // namespace
}  // namespace lq

using namespace lq;

extern "C" size_t lq_token_logprobs_workspace(int64_t rows, int64_t vocab, int top) {
  if (rows <= 0 || vocab <= 0 || top < 0) return 0;
  const size_t parts = (size_t)rows * (size_t)((vocab + PART - 1) / PART);
  return align256(parts * 16) + parts * (size_t)top * 8;
}

extern "C" int lq_token_logprobs(const lq_tensor* logits, const lq_tensor* tokens,
                                 const lq_tensor* logprobs, const lq_tensor* entropy,
                                 const lq_tensor* top_logprobs, const lq_tensor* top_tokens,
                                 void* workspace, size_t workspace_bytes, void* stream) {
  int rc;
  const int nd = logits != nullptr && logits->ndim == 3 ? 3 : 2;
  if ((rc = check_tensor_or_empty(logits, "logits", nd, true)) != LQ_OK) return rc;
  if ((rc = check_tensor_or_empty(tokens, "tokens", nd - 1, false, LQ_I64)) != LQ_OK) return rc;
  if ((rc = check_tensor_or_empty(logprobs, "logprobs", 1, false, LQ_F32)) != LQ_OK) return rc;
  if (entropy != nullptr && (rc = check_tensor_or_empty(entropy, "entropy", 1, false, LQ_F32)) != LQ_OK) return rc;
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
    if ((rc = check_tensor_or_empty(top_logprobs, "top_logprobs", 2, false, LQ_F32)) != LQ_OK) return rc;
    if ((rc = check_tensor_or_empty(top_tokens, "top_tokens", 2, false, LQ_I64)) != LQ_OK) return rc;
    top = top_logprobs->shape[1];
  }
  const lq_tensor* outs[4] = {logprobs, entropy, top_logprobs, top_tokens};
  for (const lq_tensor* t : outs) {
    if (t == nullptr) continue;
    const bool flat = t->ndim == 1 ? t->stride[0] == 1 || rows < 2
                                   : (t->stride[1] == 1 || top < 2) && (t->stride[0] == top || rows < 2);
    if (t->shape[0] != rows || (t->ndim == 2 && t->shape[1] != top) || !flat) {
      return fail(LQ_ERR_INVALID_ARG, "the outputs must be contiguous and have %lld rows", (long long)rows);
    }
  }
  if (rows == 0) return LQ_OK;
  if (V < 1 || top > V) {
    return fail(LQ_ERR_INVALID_ARG, "%lld likeliest of a vocabulary of %lld asked for", (long long)top,
                (long long)V);
  }
  const int64_t parts = (V + PART - 1) / PART;
  if (top > MAX_TOP) {
    return fail(LQ_ERR_UNSUPPORTED, "top %lld unsupported (<= %d)", (long long)top, MAX_TOP);
  }
  if (V > INT32_MAX || rows > INT32_MAX || rows * parts >= ((int64_t)1 << 32) / THREADS) {
    return fail(LQ_ERR_UNSUPPORTED, "%lld rows of %lld logits exceed the launch limits",
                (long long)rows, (long long)V);
  }
  const size_t need = lq_token_logprobs_workspace(rows, V, (int)top);
  if (workspace == nullptr || workspace_bytes < need) {
    return fail(LQ_ERR_WORKSPACE, "workspace of %zu bytes needed, %zu given", need,
                workspace == nullptr ? (size_t)0 : workspace_bytes);
  }
  if (((uintptr_t)workspace & 255) != 0) {
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
  p.parts = (int)parts;
  p.top = (int)top;
  p.V = V;
  p.stats = (float*)workspace;
  p.keys = (uint64_t*)((char*)workspace + align256((size_t)(rows * parts) * 16));
  const hipStream_t st = (hipStream_t)stream;
  const dim3 grid((unsigned)(rows * parts)), block(THREADS);
  if (logits->dtype == LQ_BF16) hipLaunchKernelGGL(logprob_part_kernel<LQ_BF16>, grid, block, 0, st, p);
  else if (logits->dtype == LQ_F16) hipLaunchKernelGGL(logprob_part_kernel<LQ_F16>, grid, block, 0, st, p);
  else hipLaunchKernelGGL(logprob_part_kernel<LQ_F32>, grid, block, 0, st, p);
  if ((rc = check_launch("lq_token_logprobs")) != LQ_OK) return rc;
  hipLaunchKernelGGL(logprob_final_kernel, dim3((unsigned)rows), dim3(64), 0, st, p);
  return check_launch("lq_token_logprobs (final)");
}
