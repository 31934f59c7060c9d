// Causal attention of whole prompts over their own keys, grouped query heads, prompts packed one behind
// another or a batch of equal lengths (no reference counterpart: its forward hands prompts to a library
// attention on repeated K and V, hybrid_quant/int4_8b_attention.py:693-714):
//
//   o_t = sum_{s <= t} softmax_s(scale * q_t . k_s) v_s     over the rows s of t's own prompt
//
// prompt_attention_f32: any float dtype and strides, head_dim <= 256, fp32 products and sums on
// v_mfma_f32_32x32x2_f32. It is the kernel of fp32 inputs and of layouts that the 16-bit kernel
// (prompt_attention_mfma.hip) does not take. Three fp32 prompts up to 1001 rows, 32 query and 8 KV heads:
// 231 us, 72 TFLOP/s, half of the rate of a large fp32 library product (153). With loads one value at a time,
// waited for before each tile, it was 608.
//
// A prompt's rows of a KV head are its positions times the n_rep query heads, head by head within a
// position, so that a workgroup's 128 rows (32 per wave) are as few positions as possible: little lies
// beyond the diagonal, and a prompt of a few tokens still fills a wave. Scores are made transposed,
// S^T[key][row] = K Q^T: a lane then holds the scores of one row, its softmax needs one exchange with
// the lane 32 away, and the register that holds p of a key is by itself the B operand of
// O^T[dim][row] += V^T P^T.
//
// A workgroup with an infinity among its sums, which may be of large values alone, runs its rows again with
// smaller weights (PROMPT_ATTENTION_DOWN).
#include "prompt_attention.h"

namespace lq {
namespace {

constexpr int KT = 32;    // keys per tile
constexpr int ROWS = 32;  // rows per wave
constexpr int NW = PROMPT_ATTENTION_WAVES;

typedef float f32x16_t __attribute__((ext_vector_type(16)));

template <int DP>
struct alignas(16) TileF32 {
  float k[KT][DP + 4];  // rows 4 banks apart: 16 lanes' 16-byte reads of 16 rows hit all 64 banks
  float v[KT][DP + 8];  // rows 4 apart are 32 banks apart: two half-waves read different banks
};

__device__ __forceinline__ bool finite(float x) {
  return (__float_as_uint(x) & 0x7f800000u) != 0x7f800000u;
}

// A span's rows of a workgroup; whether they have to run again, DOWN.
// VEC: fp32 k and v in 16-byte aligned rows of a multiple of 4 dims. Their tiles come in 16-byte loads, a
// tile ahead.
template <int DP, bool VEC, bool DOWN>
__device__ __forceinline__ bool attend(const PromptAttention& p, const Span& sp, int hk, int tid,
                                       TileF32<DP>& tile) {
  const int nrep = p.nrep, lane = tid & 63, wave = tid >> 6, col = lane & 31, hi = lane >> 5;
  const int nrows = sp.len * nrep;
  // the last tile of a prompt has the most keys: it goes first
  const int tiles = (nrows + NW * ROWS - 1) / (NW * ROWS);
  const int first = (tiles - 1 - sp.part) * NW * ROWS;
  const int r = first + wave * ROWS + col;
  const int pos = min(r, nrows - 1) / nrep;
  const int head = hk * nrep + min(r, nrows - 1) % nrep;
  const int64_t row = sp.begin + pos;
  const int64_t lead = p.spans.starts == nullptr ? sp.index : 0;
  const int64_t out_at = lead * p.out.s[0] + row * p.out.s[1] + head * p.out.s[2];
  if (!DOWN && sp.gap) {
    if (r < nrows) {
      for (int d = hi; d < p.D; d += 2) store_float(p.out.data, p.out.dtype, out_at + d * p.out.s[3], 0.f);
    }
    return false;
  }

  // query values of dims 8 j + 4 hi .. + 3, in the order in which the K rows are read
  float q[DP / 2];
  {
    const int64_t at = lead * p.q.s[0] + row * p.q.s[1] + head * p.q.s[2];
#pragma unroll
    for (int i = 0; i < DP / 2; ++i) {
      const int d = 8 * (i >> 2) + 4 * hi + (i & 3);
      q[i] = d < p.D ? load_float(p.q.data, p.q.dtype, at + d * p.q.s[3]) * p.scale : 0.f;
    }
  }
  f32x16_t o[DP / 32];
#pragma unroll
  for (int i = 0; i < DP / 32; ++i) o[i] = f32x16_t{};
  float m = -INFINITY, l = 0.f;
  const int64_t k_at = lead * p.k.s[0] + sp.begin * p.k.s[1] + hk * p.k.s[2];
  const int64_t v_at = lead * p.v.s[0] + sp.begin * p.v.s[1] + hk * p.v.s[2];
  constexpr int LOADS = KT * DP / 4 / (64 * NW);  // 16-byte loads of a thread and tile
  float4 kn[VEC ? LOADS : 1], vn[VEC ? LOADS : 1];
  auto load_tile = [&](int kb) {
#pragma unroll
    for (int j = 0; j < (VEC ? LOADS : 0); ++j) {
      const int i = j * 64 * NW + tid, key = i / (DP / 4), d = i % (DP / 4) * 4;
      const bool in = kb + key < sp.len && d < p.D;
      kn[j] = vn[j] = make_float4(0.f, 0.f, 0.f, 0.f);
      if (in) kn[j] = *(const float4*)((const float*)p.k.data + k_at + (int64_t)(kb + key) * p.k.s[1] + d);
      if (in) vn[j] = *(const float4*)((const float*)p.v.data + v_at + (int64_t)(kb + key) * p.v.s[1] + d);
    }
  };
  load_tile(0);
  const int pos_first = first / nrep;
  const int pos_last = min(first + NW * ROWS - 1, nrows - 1) / nrep;
  for (int kb = 0; kb <= pos_last; kb += KT) {
    const bool diagonal = kb + KT - 1 > pos_first;  // holds keys that some row must not see
    __syncthreads();
    int bad = 0;
    if (VEC) {
#pragma unroll
      for (int j = 0; j < LOADS; ++j) {
        const int i = j * 64 * NW + tid, key = i / (DP / 4), d = i % (DP / 4) * 4;
        *(float4*)&tile.k[key][d] = kn[j];
        *(float4*)&tile.v[key][d] = vn[j];
        bad |= !finite(vn[j].x) || !finite(vn[j].y) || !finite(vn[j].z) || !finite(vn[j].w);
      }
      if (kb + KT <= pos_last) load_tile(kb + KT);
    }
    for (int i = tid; i < (VEC ? 0 : KT * DP); i += 64 * NW) {
      const int key = i / DP, d = i % DP;
      float kv = 0.f, vv = 0.f;
      if (kb + key < sp.len && d < p.D) {
        kv = load_float(p.k.data, p.k.dtype, k_at + (int64_t)(kb + key) * p.k.s[1] + d * p.k.s[3]);
        vv = load_float(p.v.data, p.v.dtype, v_at + (int64_t)(kb + key) * p.v.s[1] + d * p.v.s[3]);
      }
      tile.k[key][d] = kv;
      tile.v[key][d] = vv;
      bad |= !finite(vv);
    }
    if (diagonal) {
      bad = __syncthreads_or(bad);
    } else {
      __syncthreads();
      bad = 0;
    }
    if (bad) {
      // A masked key has p = 0, but 0 * inf is not 0. What is not finite goes to the rows that see it
      // here, and leaves the tile.
      for (int key = 0; key < KT; ++key) {
        if (kb + key > pos) continue;
#pragma unroll
        for (int i = 0; i < DP / 2; ++i) {
          const float v = tile.v[key][32 * (i >> 4) + 8 * ((i >> 2) & 3) + 4 * hi + (i & 3)];
          if (!finite(v)) o[i >> 4][i & 15] += v;
        }
      }
      __syncthreads();
      for (int i = tid; i < KT * DP; i += 64 * NW) {
        float& v = tile.v[i / DP][i % DP];
        if (!finite(v)) v = 0.f;
      }
      __syncthreads();
    }
    f32x16_t s = {};
#pragma unroll
    for (int j = 0; j < DP / 8; ++j) {
      const float4 kv = *(const float4*)&tile.k[col][8 * j + 4 * hi];
      s = __builtin_amdgcn_mfma_f32_32x32x2f32(kv.x, q[4 * j], s, 0, 0, 0);
      s = __builtin_amdgcn_mfma_f32_32x32x2f32(kv.y, q[4 * j + 1], s, 0, 0, 0);
      s = __builtin_amdgcn_mfma_f32_32x32x2f32(kv.z, q[4 * j + 2], s, 0, 0, 0);
      s = __builtin_amdgcn_mfma_f32_32x32x2f32(kv.w, q[4 * j + 3], s, 0, 0, 0);
    }
    float top = m;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      if (kb + 8 * (i >> 2) + 4 * hi + (i & 3) > pos) s[i] = -INFINITY;
      top = fmaxf(top, s[i]);
    }
    top = fmaxf(top, __shfl_xor(top, 32, 64));
    const float base = top == -INFINITY ? 0.f : top;  // all keys so far at -inf: their p is 0
    float keep = __builtin_amdgcn_exp2f(m - base);
    m = top;
    l *= keep;
    if (__any(keep == 0.f)) {  // the infinities, this tile's among them, stay
#pragma unroll
      for (int i = 0; i < DP / 2; ++i) {
        const float x = o[i >> 4][i & 15];
        o[i >> 4][i & 15] = keep == 0.f && finite(x) ? 0.f : x;
      }
      keep = keep == 0.f ? 1.f : keep;
    }
    // (by itself: many small terms, each rounded beside a large l, would be off together)
    float sum = 0.f;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      s[i] = __builtin_amdgcn_exp2f(s[i] - base);
      sum += s[i];
    }
    l += sum;
    if (DOWN) s *= PROMPT_ATTENTION_DOWN;
#pragma unroll
    for (int b = 0; b < DP / 32; ++b) {
      o[b] *= keep;
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const float v = tile.v[8 * (i >> 2) + 4 * hi + (i & 3)][32 * b + col];
        o[b] = __builtin_amdgcn_mfma_f32_32x32x2f32(v, s[i], o[b], 0, 0, 0);
      }
    }
  }
  if (!DOWN) {
    float most = 0.f;
#pragma unroll
    for (int i = 0; i < DP / 2; ++i) most = fmaxf(most, fabsf(o[i >> 4][i & 15]));
    if (__syncthreads_or(most == INFINITY)) return true;
  }
  l += __shfl_xor(l, 32, 64);
  const float inv = (DOWN ? 1.f / PROMPT_ATTENTION_DOWN : 1.f) / l;
  if (r >= nrows) return false;
  int dim = 4 * hi;
  asm volatile("" : "+v"(dim));  // (else the addresses of all stores in registers, through the loop)
#pragma unroll
  for (int b = 0; b < DP / 32; ++b) {
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const int d = 32 * b + 8 * (i >> 2) + dim + (i & 3);
      if (d < p.D) store_float(p.out.data, p.out.dtype, out_at + d * p.out.s[3], o[b][i] * inv);
    }
  }
  return false;
}

template <int DP, bool VEC>
__global__ __launch_bounds__(64 * NW, DP <= 128 ? 2 : 1) void prompt_attention_f32(PromptAttention p) {
  __shared__ TileF32<DP> tile;
  int hk = blockIdx.x % p.Hkv, tid = threadIdx.x;
  Span sp;
  if (!find_part(p, blockIdx.x / p.Hkv, sp)) return;
  if (!attend<DP, VEC, false>(p, sp, hk, tid, tile)) return;
  // Again, from values hidden from the compiler: it would keep what the first run made of them in registers
  // for the second one, through the loop.
  asm volatile("" : "+s"(sp.index), "+s"(sp.begin), "+s"(sp.len), "+s"(sp.part), "+s"(hk), "+v"(tid));
  attend<DP, VEC, true>(p, sp, hk, tid, tile);
}

template <bool VEC>
void launch_f32(const PromptAttention& p, dim3 grid, hipStream_t st) {
  const dim3 block(64 * NW);
  if (p.D <= 64) hipLaunchKernelGGL((prompt_attention_f32<64, VEC>), grid, block, 0, st, p);
  else if (p.D <= 128) hipLaunchKernelGGL((prompt_attention_f32<128, VEC>), grid, block, 0, st, p);
  else hipLaunchKernelGGL((prompt_attention_f32<256, VEC>), grid, block, 0, st, p);
}

}  // namespace

int make_spans(const lq_tensor* starts, int64_t batch, int64_t rows, Spans& out) {
  if (rows > INT32_MAX / 2 || batch > INT32_MAX / 2) {
    return fail(LQ_ERR_UNSUPPORTED, "%lld rows of %lld prompts exceed the launch limits",
                (long long)rows, (long long)batch);
  }
  out = Spans{nullptr, 0, (int)batch, (int)rows};
  if (starts == nullptr) return LQ_OK;
  int rc;
  if ((rc = check_tensor(starts, "starts", 1, false)) != LQ_OK) return rc;
  if (starts->dtype != LQ_I32 && starts->dtype != LQ_I64) {
    return fail(LQ_ERR_INVALID_ARG, "starts: dtype code %d is not int32/int64", starts->dtype);
  }
  if (starts->shape[0] < 1 || (starts->shape[0] > 1 && starts->stride[0] != 1)) {
    return fail(LQ_ERR_INVALID_ARG, "starts must be contiguous and hold at least one value");
  }
  if (starts->shape[0] > (1 << 24)) {
    return fail(LQ_ERR_UNSUPPORTED, "%lld prompts exceed the launch limits",
                (long long)(starts->shape[0] - 1));
  }
  out.starts = starts->data;
  out.is64 = starts->dtype == LQ_I64;
  out.S = (int)(starts->shape[0] - 1);
  return LQ_OK;
}

}  // namespace lq

using namespace lq;

extern "C" int lq_prompt_attention(const lq_tensor* q, const lq_tensor* k, const lq_tensor* v,
                                   const lq_tensor* starts, const lq_tensor* out, float scale,
                                   void* stream) {
  int rc;
  const int nd = starts != nullptr ? 3 : 4;
  if ((rc = check_tensor_or_empty(q, "q", nd, true)) != LQ_OK) return rc;
  if ((rc = check_tensor_or_empty(k, "k", nd, true, q->dtype)) != LQ_OK) return rc;
  if ((rc = check_tensor_or_empty(v, "v", nd, true, q->dtype)) != LQ_OK) return rc;
  if ((rc = check_tensor_or_empty(out, "out", nd, true, q->dtype)) != LQ_OK) return rc;
  const int64_t batch = nd == 4 ? q->shape[0] : 1, rows = q->shape[nd - 3];
  const int64_t Hq = q->shape[nd - 2], Hkv = k->shape[nd - 2], D = q->shape[nd - 1];
  for (int i = 0; i < nd; ++i) {
    if (out->shape[i] != q->shape[i]) return fail(LQ_ERR_INVALID_ARG, "out must have q's shape");
    if (v->shape[i] != k->shape[i]) return fail(LQ_ERR_INVALID_ARG, "v must have k's shape");
    if (i != nd - 2 && k->shape[i] != q->shape[i]) {
      return fail(LQ_ERR_INVALID_ARG, "k must have q's rows and head_dim");
    }
  }
  PromptAttention p{};
  if ((rc = make_spans(starts, batch, rows, p.spans)) != LQ_OK) return rc;
  if (Hkv < 1 || Hq < 1 || Hq % Hkv != 0) {
    return fail(LQ_ERR_INVALID_ARG, "%lld query heads over %lld KV heads", (long long)Hq,
                (long long)Hkv);
  }
  if (D < 1 || D > PROMPT_ATTENTION_MAX_D) {
    return fail(LQ_ERR_UNSUPPORTED, "head_dim %lld unsupported (<= %d)", (long long)D,
                PROMPT_ATTENTION_MAX_D);
  }
  const float scale2 = scale * 1.44269504088896340736f;  // of exponents of 2
  if (!(scale2 - scale2 == 0.f)) return fail(LQ_ERR_INVALID_ARG, "scale must be finite, and so scale log2(e)");
  if (batch == 0 || rows == 0) return LQ_OK;
  const int64_t nrep = Hq / Hkv;
  if (rows * nrep > INT32_MAX / 2) {
    return fail(LQ_ERR_UNSUPPORTED, "%lld rows of %lld heads exceed the launch limits",
                (long long)rows, (long long)Hq);
  }
  if (overlaps_itself(*out) || overlap(*out, *k) || overlap(*out, *v) ||
      (overlap(*out, *q) && !same_elements(*out, *q)) || (starts != nullptr && overlap(*out, *starts))) {
    return fail(LQ_ERR_INVALID_ARG, "out overlaps itself, k, v, starts, or q without being q");
  }
  const lq_tensor* ts[4] = {q, k, v, out};
  View* vs[4] = {&p.q, &p.k, &p.v, &p.out};
  for (int i = 0; i < 4; ++i) {
    *vs[i] = make_view(ts[i]);
    for (int j = 3; j > 3 - nd; --j) vs[i]->s[j] = ts[i]->stride[j - (4 - nd)];
    if (nd == 3) vs[i]->s[0] = 0;
  }
  p.Hkv = (int)Hkv;
  p.nrep = (int)nrep;
  p.D = (int)D;
  p.scale = scale2;
  // parts of 128 rows; packed prompts (and the rows of none in front and behind) have one more each
  const int64_t part = NW * ROWS;
  const int64_t parts = starts == nullptr ? batch * ((rows * nrep + part - 1) / part)
                                          : rows * nrep / part + p.spans.S + 2;
  if (parts * Hkv >= ((int64_t)1 << 32) / (64 * NW) || parts > INT32_MAX / 2) {
    return fail(LQ_ERR_UNSUPPORTED, "%lld parts of %lld KV heads exceed the launch limits",
                (long long)parts, (long long)Hkv);
  }
  const hipStream_t st = (hipStream_t)stream;
  const bool mfma = !diag(LQ_DIAG_PROMPT_FORCE_GENERIC) && prompt_attention_mfma_fits(q, k, v, out);
  if (!mfma && diag(LQ_DIAG_PROMPT_REQUIRE_MFMA)) {
    return fail(LQ_ERR_INVALID_ARG, "the layout takes the general kernel");
  }
  if (mfma) {
    p.q_and = scale == 0.f ? 0 : ~0u;
    p.q_xor = scale < 0.f ? 0x80008000u : 0;
    p.scale = scale == 0.f ? 1.f : fabsf(p.scale);
    return launch_prompt_attention_mfma(p, q->dtype, parts, st);
  }
  const dim3 grid((unsigned)(parts * Hkv));
  bool in_rows = q->dtype == LQ_F32 && D % 4 == 0;
  const lq_tensor* kv[2] = {k, v};
  for (const lq_tensor* t : kv) {
    in_rows = in_rows && t->stride[nd - 1] == 1 && ((uintptr_t)t->data & 15) == 0;
    for (int i = 0; i < nd - 1; ++i) in_rows = in_rows && (t->shape[i] < 2 || t->stride[i] % 4 == 0);
  }
  if (in_rows) launch_f32<true>(p, grid, st);
  else launch_f32<false>(p, grid, st);
  return check_launch("lq_prompt_attention");
}
