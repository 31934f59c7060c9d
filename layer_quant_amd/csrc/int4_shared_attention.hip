// q_len = 1 GQA decode attention of rows that share a prefix: row b = prompt * N + member attends to
// the INT4 cache rows of its prompt (one copy for the prompt's N rows) and then to its own.
//
// Scores and masks are those of lq_int4_decode_attention over the two caches in sequence:
// s_j = (q . k_j) * log2(e)/sqrt(D) (+ mask_j), exp2-domain online softmax, fp32 sums; keys at or
// beyond the mask's length get -inf, and so do masked keys whatever their scores and scales hold. The
// prefix and the own rows are split over workgroups; every split leaves (m, l, acc[D]) of each of its
// query rows in the workspace and the decode attention's merge joins them.
//
//   * shared_mfma_kernel (int4_shared_attention_mfma.hip): head_dim 128, group 32/64/128, 16-bit
//     queries; packs the new token itself.
//   * shared_generic_kernel: any even group dividing any head_dim <= 512, any query type; one wave per
//     (row, query head, split), fp32 VALU throughout, behind shared_pack_kernel. It shares nothing of a
//     prompt's rows: fp32 queries, ctx 4001, group 32, 2 prompts x 8 members 696 us, 16 x 1 843, 2 x 1 128.
#include <math.h>

#include "int4_quant.h"
#include "int4_shared_attention.h"

namespace lq {
namespace {

constexpr int GEN_MAX_D = 512;

// The key's additive mask in exp2 units; -inf for a masked key.
__device__ __forceinline__ float mask_bias(const SharedParams& p, int64_t b, int64_t key) {
  if (p.mask == nullptr) return 0.0f;
  if (key >= p.mask_len) return -INFINITY;
  const int64_t i = b * p.mask_sb + key * p.mask_sk;
  if (p.mask_keep) return ((const int64_t*)p.mask)[i] != 0 ? 0.0f : -INFINITY;
  return ((const float*)p.mask)[i];
}

__global__ __launch_bounds__(64) void shared_generic_kernel(SharedParams p) {
  __shared__ float q_s[GEN_MAX_D];
  __shared__ float p_s[64];
  const int lane = threadIdx.x;
  const int bh = blockIdx.x;
  const int split = blockIdx.y;
  const int b = bh / p.Hq;
  const int qh = bh - b * p.Hq;
  const int kvh = qh / p.nrep;
  const bool is_own = split >= p.nsp;
  const CacheView& c = is_own ? p.own : p.prefix;
  const int64_t row = is_own ? b : b / p.N;
  const int64_t t0 = is_own ? (int64_t)(split - p.nsp) * p.chunk_o : (int64_t)split * p.chunk_p;
  const int64_t t1 = is_own ? min(p.own_len, t0 + p.chunk_o) : min(p.prefix_len, t0 + p.chunk_p);
  const int64_t key0 = is_own ? p.prefix_len : 0;  // the mask's key of cache row 0
  const int D = p.D;
  const int g = p.g;

  for (int d = lane; d < D; d += 64) {
    q_s[d] = load_float(p.q.data, p.q.dtype, b * p.q.s[0] + qh * p.q.s[1] + d * p.q.s[2]);
  }
  __syncthreads();

  const uint8_t* kbase = c.kp + row * c.kps[0] + kvh * c.kps[1];
  const uint8_t* vbase = c.vp + row * c.vps[0] + kvh * c.vps[1];
  const float* ksbase = c.ks + row * c.kss[0] + kvh * c.kss[1];
  const float* vsbase = c.vs + row * c.vss[0] + kvh * c.vss[1];
  const int groups = D / g;

  float m = -INFINITY;
  float l = 0.0f;
  float acc[GEN_MAX_D / 64];
#pragma unroll
  for (int i = 0; i < GEN_MAX_D / 64; ++i) acc[i] = 0.0f;

  for (int64_t start = t0; start < t1; start += 64) {
    const int64_t n = start + lane;
    float s = -INFINITY;
    const float bias = n < t1 ? mask_bias(p, b, key0 + n) : -INFINITY;
    if (bias != -INFINITY) {
      const uint8_t* kr = kbase + n * c.kps[2];
      const float* ksr = ksbase + n * c.kss[2];
      float tot = 0.0f;
      for (int gi = 0; gi < groups; ++gi) {
        float part = 0.0f;
        for (int d = gi * g; d < (gi + 1) * g; d += 2) {
          const int byte = kr[(d >> 1) * c.kps[3]];
          int lo = byte & 15;
          int hi = (byte >> 4) & 15;
          lo = lo >= 8 ? lo - 16 : lo;
          hi = hi >= 8 ? hi - 16 : hi;
          part += q_s[d] * (float)lo + q_s[d + 1] * (float)hi;
        }
        tot += part * ksr[gi * c.kss[3]];
      }
      s = tot * p.scale_sm + bias;
    }
    const float m_new = fmaxf(m, group_max<64>(s));
    const float alpha = (m_new == -INFINITY) ? 1.0f : exp2f(m - m_new);
    const float pn = (s == -INFINITY) ? 0.0f : exp2f(s - m_new);
    l = l * alpha + group_sum<64>(pn);
    p_s[lane] = pn;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < GEN_MAX_D / 64; ++i) acc[i] *= alpha;
    const int cnt = (int)min((int64_t)64, t1 - start);
    for (int j = 0; j < cnt; ++j) {
      const float pj = p_s[j];
      if (pj == 0.0f) continue;  // a masked key's scales may hold anything
      const uint8_t* vr = vbase + (start + j) * c.vps[2];
      const float* vsr = vsbase + (start + j) * c.vss[2];
#pragma unroll
      for (int i = 0; i < GEN_MAX_D / 64; ++i) {
        const int d = lane + 64 * i;
        if (d < D) {
          const int byte = vr[(d >> 1) * c.vps[3]];
          int nib = (d & 1) ? ((byte >> 4) & 15) : (byte & 15);
          nib = nib >= 8 ? nib - 16 : nib;
          acc[i] += pj * ((float)nib * vsr[(d / g) * c.vss[3]]);
        }
      }
    }
    __syncthreads();
    m = m_new;
  }

  const int ns = p.nsp + p.nso;
  if (ns == 1) {
#pragma unroll
    for (int i = 0; i < GEN_MAX_D / 64; ++i) {
      const int d = lane + 64 * i;
      if (d < D) {
        store_float(p.out.data, p.out.dtype, b * p.out.s[0] + qh * p.out.s[1] + d * p.out.s[2],
                    acc[i] / l);
      }
    }
    return;
  }
  const int64_t slot = (int64_t)bh * ns + split;
  if (lane == 0) {
    p.ws_m[slot] = m;
    p.ws_l[slot] = l;
  }
#pragma unroll
  for (int i = 0; i < GEN_MAX_D / 64; ++i) {
    const int d = lane + 64 * i;
    if (d < D) p.ws_acc[slot * D + d] = acc[i];
  }
}

// The new token's K and V rows into own row own_len - 1: one wave per (row, KV head, K or V, group).
__global__ __launch_bounds__(64) void shared_pack_kernel(SharedParams p) {
  const int lane = threadIdx.x;
  const int kvh = blockIdx.x % p.Hkv;
  const int b = blockIdx.x / p.Hkv;
  const int gi = blockIdx.y;
  const bool is_v = blockIdx.z != 0;
  const View& x = is_v ? p.vnew : p.knew;
  const int64_t at = b * x.s[0] + kvh * x.s[1];
  const int64_t row = p.own_len - 1;
  float amax = 0.0f;
  for (int d = gi * p.g + lane; d < (gi + 1) * p.g; d += 64) {
    amax = fmaxf(amax, fabsf(load_float(x.data, x.dtype, at + d * x.s[2])));
  }
  const float scale = token_scale(group_max<64>(amax));
  const int64_t* ps = is_v ? p.own.vps : p.own.kps;
  const int64_t* ss = is_v ? p.own.vss : p.own.kss;
  uint8_t* packed = const_cast<uint8_t*>(is_v ? p.own.vp : p.own.kp) + b * ps[0] + kvh * ps[1] + row * ps[2];
  for (int j = lane; j < p.g / 2; j += 64) {
    const int d = gi * p.g + 2 * j;
    const float x0 = load_float(x.data, x.dtype, at + d * x.s[2]);
    const float x1 = load_float(x.data, x.dtype, at + (d + 1) * x.s[2]);
    packed[(d >> 1) * ps[3]] = (uint8_t)(token_level(x0, scale) | token_level(x1, scale) << 4);
  }
  if (lane == 0) {
    const_cast<float*>(is_v ? p.own.vs : p.own.ks)[b * ss[0] + kvh * ss[1] + row * ss[2] + gi * ss[3]] = scale;
  }
}

// About 2048 waves in flight, at least 64 keys per split, the splits shared out by length.
SharedPlan plan_generic(int64_t B, int64_t Hq, int64_t prefix_len, int64_t own_len) {
  const int64_t rows = std::max<int64_t>(1, B * Hq);
  const int64_t want = std::min<int64_t>((2048 + rows - 1) / rows, 1024);
  const int64_t total = prefix_len + own_len;
  return SharedPlan{split_of(prefix_len, (want * prefix_len + total - 1) / std::max<int64_t>(total, 1), 64),
                    split_of(own_len, (want * own_len + total - 1) / std::max<int64_t>(total, 1), 64)};
}

size_t align256(size_t n) { return (n + 255) / 256 * 256; }

size_t partial_bytes(int64_t B, int64_t Hq, int64_t D, const SharedPlan& plan) {
  const int ns = plan.prefix.nsplit + plan.own.nsplit;
  if (ns <= 1) return 0;
  const size_t slots = (size_t)(B * Hq) * (size_t)ns;
  return 2 * align256(slots * 4) + slots * (size_t)D * 4;
}

// Checks one INT4 cache against rows x Hkv x D and fills its view; *cap gets its capacity.
int check_cache(const lq_tensor* kp, const lq_tensor* vp, const lq_tensor* ks, const lq_tensor* vs,
                const char* name, int64_t rows, int64_t Hkv, int64_t D, int g, int64_t* cap,
                CacheView& c) {
  int rc;
  const lq_tensor* packed[2] = {kp, vp};
  const lq_tensor* scales[2] = {ks, vs};
  for (int i = 0; i < 2; ++i) {
    if ((rc = check_tensor(packed[i], name, 4, false, LQ_U8)) != LQ_OK) return rc;
    if ((rc = check_tensor(scales[i], name, 4, false, LQ_F32)) != LQ_OK) return rc;
  }
  *cap = kp->shape[2];
  for (int i = 0; i < 2; ++i) {
    const lq_tensor *t = packed[i], *s = scales[i];
    if (t->shape[0] != rows || t->shape[1] != Hkv || t->shape[2] != *cap || t->shape[3] != D / 2) {
      return fail(LQ_ERR_INVALID_ARG, "%s: packed caches must be [%lld, %lld, %lld, %lld]", name,
                  (long long)rows, (long long)Hkv, (long long)*cap, (long long)(D / 2));
    }
    if (s->shape[0] != rows || s->shape[1] != Hkv || s->shape[2] != *cap || s->shape[3] != D / g) {
      return fail(LQ_ERR_INVALID_ARG, "%s: scale caches must be [%lld, %lld, %lld, %lld]", name,
                  (long long)rows, (long long)Hkv, (long long)*cap, (long long)(D / g));
    }
  }
  c.kp = (const uint8_t*)kp->data;
  c.vp = (const uint8_t*)vp->data;
  c.ks = (const float*)ks->data;
  c.vs = (const float*)vs->data;
  for (int i = 0; i < 4; ++i) {
    c.kps[i] = kp->stride[i];
    c.vps[i] = vp->stride[i];
    c.kss[i] = ks->stride[i];
    c.vss[i] = vs->stride[i];
  }
  return LQ_OK;
}

}  // namespace
}  // namespace lq

using namespace lq;

extern "C" size_t lq_int4_shared_decode_attention_workspace(int64_t prompts, int64_t members,
                                                            int64_t n_q_heads, int64_t n_kv_heads,
                                                            int64_t head_dim, int64_t prefix_len,
                                                            int64_t seq_len, int group_size) {
  if (prompts <= 0 || members <= 0 || n_q_heads <= 0 || n_kv_heads <= 0 || head_dim <= 0 ||
      prefix_len < 0 || seq_len < 1 || seq_len < prefix_len || group_size <= 0) {
    return 0;
  }
  const int64_t B = prompts * members;
  size_t need = partial_bytes(B, n_q_heads, head_dim,
                              plan_generic(B, n_q_heads, prefix_len, seq_len - prefix_len));
  if (shared_fast_shape_ok(head_dim, group_size) && n_q_heads % n_kv_heads == 0) {
    need = std::max(need, partial_bytes(B, n_q_heads, head_dim,
                                        plan_shared_fast(prompts, members, n_kv_heads,
                                                         n_q_heads / n_kv_heads, prefix_len,
                                                         seq_len - prefix_len)));
  }
  return need;
}

extern "C" int lq_int4_shared_decode_attention(
    const lq_tensor* q, const lq_tensor* k_new, const lq_tensor* v_new,
    const lq_tensor* prefix_k_packed, const lq_tensor* prefix_v_packed,
    const lq_tensor* prefix_k_scale, const lq_tensor* prefix_v_scale, const lq_tensor* k_packed,
    const lq_tensor* v_packed, const lq_tensor* k_scale, const lq_tensor* v_scale,
    const lq_tensor* mask, const lq_tensor* out, int64_t prefix_len, int64_t seq_len,
    int num_key_value_groups, int group_size, void* workspace, size_t workspace_bytes,
    void* stream) {
  int rc;
  if (q == nullptr) return fail(LQ_ERR_INVALID_ARG, "q: descriptor is NULL");
  const int qdim = q->ndim;
  if (qdim != 3 && qdim != 4) {
    return fail(LQ_ERR_INVALID_ARG, "q: expected [B, Hq, 1, D] or [B, Hq, D], got %d dims", qdim);
  }
  if ((rc = check_tensor(q, "q", qdim, true)) != LQ_OK) return rc;
  if (qdim == 4 && q->shape[2] != 1) {
    return fail(LQ_ERR_INVALID_ARG, "Fused INT4 decode attention expects q_len=1, got %lld",
                (long long)q->shape[2]);
  }
  if ((rc = check_tensor(out, "out", 3, true)) != LQ_OK) return rc;
  if ((k_new == nullptr) != (v_new == nullptr)) {
    return fail(LQ_ERR_INVALID_ARG, "k_new and v_new: both or neither");
  }
  const int64_t B = q->shape[0], Hq = q->shape[1], D = q->shape[qdim - 1];
  if (group_size <= 0 || group_size % 2 != 0 || D % group_size != 0) {
    return fail(LQ_ERR_INVALID_ARG, "head_dim=%lld must be divisible by an even group_size=%d",
                (long long)D, group_size);
  }
  if (D > GEN_MAX_D || D % 2 != 0 || D < 2) {
    return fail(LQ_ERR_UNSUPPORTED, "head_dim=%lld unsupported (even, 2 to %d)", (long long)D,
                GEN_MAX_D);
  }
  if (num_key_value_groups <= 0 || Hq % num_key_value_groups != 0) {
    return fail(LQ_ERR_INVALID_ARG, "n_q_heads=%lld is no multiple of groups=%d", (long long)Hq,
                num_key_value_groups);
  }
  if ((rc = check_tensor(prefix_k_packed, "prefix", 4, false, LQ_U8)) != LQ_OK) return rc;
  const int64_t P = prefix_k_packed->shape[0];
  const int64_t Hkv = Hq / num_key_value_groups;
  if (P < 1 ? B != 0 : B % P != 0) {
    return fail(LQ_ERR_INVALID_ARG, "%lld rows do not share out over %lld prompts", (long long)B,
                (long long)P);
  }
  SharedParams p{};
  int64_t prefix_cap = 0, own_cap = 0;
  if ((rc = check_cache(prefix_k_packed, prefix_v_packed, prefix_k_scale, prefix_v_scale, "prefix", P,
                        Hkv, D, group_size, &prefix_cap, p.prefix)) != LQ_OK ||
      (rc = check_cache(k_packed, v_packed, k_scale, v_scale, "own cache", B, Hkv, D, group_size,
                        &own_cap, p.own)) != LQ_OK) {
    return rc;
  }
  if (out->shape[0] != B || out->shape[1] != Hq || out->shape[2] != D) {
    return fail(LQ_ERR_INVALID_ARG, "out must be [%lld, %lld, %lld]", (long long)B, (long long)Hq,
                (long long)D);
  }
  if (prefix_len < 0 || prefix_len > prefix_cap) {
    return fail(LQ_ERR_INVALID_ARG, "prefix_len=%lld outside [0, capacity=%lld]",
                (long long)prefix_len, (long long)prefix_cap);
  }
  if (seq_len < 1 || seq_len < prefix_len || seq_len - prefix_len > own_cap) {
    return fail(LQ_ERR_INVALID_ARG,
                "seq_len=%lld outside [max(1, prefix_len=%lld), prefix_len + capacity=%lld]",
                (long long)seq_len, (long long)prefix_len, (long long)own_cap);
  }
  const int64_t own_len = seq_len - prefix_len;
  const bool keep = mask != nullptr && mask->dtype == LQ_I64;
  if (mask != nullptr) {
    rc = keep ? check_tensor(mask, "keep", 2, false, LQ_I64)
              : check_tensor(mask, "mask", 4, false, LQ_F32);
    if (rc != LQ_OK) return rc;
    if (mask->shape[0] != B) {
      return fail(LQ_ERR_INVALID_ARG, "mask batch %lld != %lld", (long long)mask->shape[0],
                  (long long)B);
    }
  }
  if (k_new != nullptr) {
    if (own_len < 1) {
      return fail(LQ_ERR_INVALID_ARG, "seq_len=%lld leaves the new token no row behind prefix_len=%lld",
                  (long long)seq_len, (long long)prefix_len);
    }
    // the token tensors as lq_int4_pack_kv_pair checks them, one token into the last own row
    if ((rc = pack_pair_at(k_new, v_new, k_packed, v_packed, k_scale, v_scale, own_len - 1,
                           group_size, false, nullptr, "")) != LQ_OK) {
      return rc;
    }
    if (k_new->shape[2] != 1 || v_new->shape[2] != 1) {
      return fail(LQ_ERR_INVALID_ARG, "k_new and v_new must hold one token ([B, Hkv, 1, D])");
    }
  }
  if (B == 0 || Hq == 0) return LQ_OK;
  if (B * Hq * 64 >= (int64_t)1 << 32) {  // threads of the generic kernel's launch
    return fail(LQ_ERR_UNSUPPORTED, "%lld rows x %lld heads exceed the launch limits", (long long)B,
                (long long)Hq);
  }

  auto row_view = [](const lq_tensor* t, int last) {
    return View{t->data, t->dtype, {t->stride[0], t->stride[1], t->stride[last], 0}};
  };
  p.q = row_view(q, qdim - 1);
  p.out = row_view(out, 2);
  if (mask != nullptr) {
    const int last = mask->ndim - 1;
    p.mask = mask->data;
    p.mask_keep = keep;
    p.mask_sb = mask->stride[0];
    p.mask_sk = mask->stride[last];
    p.mask_len = mask->shape[last];
  }
  p.P = (int)P;
  p.N = (int)(B / P);
  p.B = (int)B;
  p.Hq = (int)Hq;
  p.Hkv = (int)Hkv;
  p.D = (int)D;
  p.g = group_size;
  p.nrep = num_key_value_groups;
  p.prefix_len = prefix_len;
  p.own_len = own_len;
  p.scale_sm = (float)(1.4426950408889634 / sqrt((double)D));

  const bool fast = shared_fast_ok(p);
  if (!fast && diag(LQ_DIAG_ATTN_REQUIRE_FAST)) {  // tests: the call must take the MFMA kernel
    return fail(LQ_ERR_INVALID_ARG,
                "LQ_ATTN_REQUIRE_FAST is set and this call takes the generic kernel");
  }
  if (k_new != nullptr) {
    p.knew = row_view(k_new, 3);
    p.vnew = row_view(v_new, 3);
    p.pack = 1;
  }
  const SharedPlan plan = fast ? plan_shared_fast(P, B / P, Hkv, num_key_value_groups, prefix_len, own_len)
                               : plan_generic(B, Hq, prefix_len, own_len);
  p.nsp = plan.prefix.nsplit;
  p.nso = plan.own.nsplit;
  p.chunk_p = plan.prefix.chunk;
  p.chunk_o = plan.own.chunk;
  const size_t need = partial_bytes(B, Hq, D, plan);
  const int ns = p.nsp + p.nso;
  if (need > 0) {
    if (workspace == nullptr || workspace_bytes < need) {
      return fail(LQ_ERR_WORKSPACE, "workspace of %zu bytes needed, %zu given", need,
                  workspace == nullptr ? (size_t)0 : workspace_bytes);
    }
    if (((uintptr_t)workspace & 255) != 0) {
      return fail(LQ_ERR_WORKSPACE, "workspace must be 256-byte aligned");
    }
    const size_t slots = (size_t)(B * Hq) * (size_t)ns;
    p.ws_m = (float*)workspace;
    p.ws_l = (float*)((char*)workspace + align256(slots * 4));
    p.ws_acc = (float*)((char*)workspace + 2 * align256(slots * 4));
  }
  const hipStream_t st = (hipStream_t)stream;
  if (fast) {
    if ((rc = launch_shared_fast(p, st)) != LQ_OK) return rc;
  } else {
    if (p.pack) {
      hipLaunchKernelGGL(shared_pack_kernel, dim3((unsigned)(B * Hkv), (unsigned)(D / group_size), 2),
                         dim3(64), 0, st, p);
      if ((rc = check_launch("lq_int4_shared_decode_attention (pack)")) != LQ_OK) return rc;
    }
    hipLaunchKernelGGL(shared_generic_kernel, dim3((unsigned)(B * Hq), (unsigned)ns), dim3(64), 0, st, p);
    if ((rc = check_launch("lq_int4_shared_decode_attention")) != LQ_OK) return rc;
  }
  if (ns > 1) {
    AttnParams a{};
    a.ws_m = p.ws_m;
    a.ws_l = p.ws_l;
    a.ws_acc = p.ws_acc;
    a.out = p.out;
    a.B = p.B;
    a.Hq = p.Hq;
    a.D = p.D;
    a.nsplit = ns;
    launch_merge(a, st);
    return check_launch("lq_int4_shared_decode_attention (merge)");
  }
  return LQ_OK;
}
