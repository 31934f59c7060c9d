// Shared declarations of the shared-prefix decode attention's kernels.
#pragma once

#include "int4_attention.h"

namespace lq {

// One INT4 cache: packed nibbles and fp32 group scales [rows, Hkv, cap, D/2 or D/g].
struct CacheView {
  const uint8_t* kp;
  const uint8_t* vp;
  const float* ks;
  const float* vs;
  int64_t kps[4], vps[4], kss[4], vss[4];
};

struct SharedParams {
  View q;    // strides of (b, h, d); row b = prompt * N + member
  View out;  // strides of (b, h, d)
  CacheView prefix;  // row = prompt
  CacheView own;     // row = b
  // NULL, an fp32 bias [B, 1, 1, Lm] (batch and key strides used), or (mask_keep) an int64 keep-mask
  // [B, Lm] whose zeros count as -inf; key j of it is prefix row j, then own row j - prefix_len
  const void* mask;
  int64_t mask_sb, mask_sk, mask_len;
  bool mask_keep;
  float* ws_m;  // partials of the prefix splits, then of the own splits, of every (b, h)
  float* ws_l;
  float* ws_acc;
  int P, N, B, Hq, Hkv, D, g, nrep;
  int64_t prefix_len, own_len;
  int nsp, nso;               // splits of the prefix and of the own rows
  int64_t chunk_p, chunk_o;   // keys per split
  float scale_sm;             // log2(e) / sqrt(D)
  // the new token's K and V rows [B, Hkv, D] (strides of b, h, d), packed into own row own_len - 1
  View knew, vnew;
  int pack;
  // MFMA path
  int q_rows;               // query rows contiguous and 16-byte aligned
  int col_tiles;            // 16-row column tiles of a prefix unit's wave
  int rb_prefix, rb_own;    // row blocks of a prefix and of an own unit
  uint32_t prefix_blocks;   // workgroups of the prefix units
  uint32_t own_units;       // own units, times splits
  int own_waves;            // waves per own unit
};

// Splits of the two key ranges.
struct SharedPlan {
  SplitPlan prefix, own;
};

// `len` keys in about `want` splits of whole `step`s.
inline SplitPlan split_of(int64_t len, int64_t want, int64_t step) {
  SplitPlan s{0, step};
  if (len == 0) return s;
  want = std::max<int64_t>(1, std::min(want, (len + step - 1) / step));
  s.chunk = ((len + want - 1) / want + step - 1) / step * step;
  s.nsplit = (int)((len + s.chunk - 1) / s.chunk);
  return s;
}

// The new token's scale: absmax * fl(1/7), the product rounded once, at least 1e-8. It is within one
// unit in the last place of int4_quantize_pair's quotient and equal to what int4_quant_dequant's
// division by 7 gives on the GPU.
__device__ __forceinline__ float token_scale(float amax) {
  return fmaxf(amax * (1.0f / 7.0f), 1.0e-8f);
}

// Level of x under that scale, as 4 bits: IEEE quotient, round half to even, [-8, 7].
__device__ __forceinline__ uint32_t token_level(float x, float scale) {
  return (uint32_t)min(max((int)rintf(x / scale), -8), 7) & 15u;
}

// MFMA path (int4_shared_attention_mfma.hip)
bool shared_fast_shape_ok(int64_t head_dim, int group_size);
bool shared_fast_ok(const SharedParams& p);
SharedPlan plan_shared_fast(int64_t P, int64_t N, int64_t Hkv, int64_t nrep, int64_t prefix_len,
                            int64_t own_len);
int launch_shared_fast(SharedParams p, hipStream_t stream);

}  // namespace lq
