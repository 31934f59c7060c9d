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
};

}  // namespace lq
