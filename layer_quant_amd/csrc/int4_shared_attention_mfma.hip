// MFMA path of the shared-prefix decode attention (head_dim 128, group 32/64/128, bf16 or fp16
// queries, contiguous cache rows).
//
// One workgroup = 4 waves on one unit and key split. A prefix unit is (prompt, KV head, block of 16 QT
// query rows), its query rows the prompt's members x the heads of the KV head; an own unit is (row, KV
// head), its query rows the heads alone. Each wave takes every fourth 32-key tile of the split, on its
// own: a ring of 3 tiles in LDS filled by loads that write LDS directly, no barrier in the key loop.
// At the end the 4 partial softmax states are joined through LDS, and the split's (m, l, acc) goes to
// the workspace (or, where it is the only split, out).
//
// Products use v_mfma_f32_16x16x32_f16 and _bf16, D[16x16] += A[16x32] * B[32x16] (lane l holds A row l%16
// and B column l%16, each with K slots 8*(l/16) .. +7, and D rows 4*(l/16) .. +3 of column l%16):
//   S^T[key][query] per group m: A = K rows as exact fp16 integers, B = Q^T scaled by a power of two
//     per query row so that its largest value lies in [2^14, 2^15) (16-bit queries are then exact in
//     fp16, products exact, sums fp32); the groups' partial sums are scaled by the fp32 key scales and
//     added in fp32.
//   O^T[dim][query]: A = V^T as exact bf16 values n / 16, B = P'_m[key][query] = 2^(s - M) * vscale[key][m],
//     M the lazily moved running maximum of the row's scores. P' is formed in fp32 and split into bf16
//     terms, each the rounding of what the terms before it leave: two for bf16 outputs (off by 2^-16
//     relative at most, 2^-8 of the output's own rounding), three for others (all 24 bits). A term has
//     the exponent range of fp32, so that a key's share keeps its precision whatever the other keys'
//     scales and weights are.
//
// What bounds it (MI355X, kernel trace, group 32 unless said): 8 prompts x 8 members at ctx 16384 take 62
// us, 174 MB of which 168 are the prompts' rows. The loads alone take 34 us, with the scores and weights
// but without the P V products 41: it is issue, 23.0 M VALU instructions (4 cycles each, 37 us of the
// SIMDs) and 1.6 M MFMAs (16 cycles, 10 us), about 650 and 48 per tile and 32 rows, at two waves per SIMD.
// Of a tile's VALU instructions 192 split P' in two terms, three per key, row and group. (As one fp16 value
// in one instruction for two keys the kernel took 56 us, with 11 bits of each product and the range of
// fp16.) 64 members of one prompt (group 128, fp16, ctx 8192: 256 query rows per KV head) take 37 us, the
// loads alone 13, without the P V products 24: every row block decodes the same tiles again. 2 x 8 under a
// keep-mask, ctx 4001: 19.5 us, the loads and masks alone 12.6, without the P V products 17.3. A few
// members at a short prompt (1 x 4, ctx 777: 8.0 us) are one tile per wave: latency of the loads, set-up
// and join. An additive mask is slow (8 x 8, ctx 16384: 273 us a call, 95 with the keep-mask, 68 without):
// its 16 values per lane and tile are loaded inside the tile's work, and with two column tiles at group 32
// and 64 they do not fit the registers beside it.
//
// Why 32 rows and not more per wave: the accumulators (64 registers), the query operands (32) and a tile's
// decoded values and scales fill the 256 registers of two waves per SIMD. Why a tile per wave and not one
// per workgroup: no barrier in the key loop, and up to 32 query rows (8 members of 4 heads) there is nothing
// that two waves would share.
#include <math.h>

#include "int4_f16.h"
#include "int4_shared_attention.h"
#include "lds_loads.h"

namespace lq {
namespace {

typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x2_t __attribute__((ext_vector_type(2)));

constexpr int SD = 128;     // head_dim
constexpr int TILE = 32;    // keys per wave step
constexpr int WAVES = 4;
constexpr int THREADS = 64 * WAVES;
constexpr int SEG = 16;     // tiles of a wave whose keep-mask words are made together
constexpr int OROW = SD + 4;  // floats per row of a wave's partial output (rows 4 banks apart)
constexpr float LAZY = 8.0f;  // running-max slack of the lazy rescale

enum { MASK_NONE = 0, MASK_BIAS = 1, MASK_KEEP = 2 };

// One wave's copy of a 32-key tile. K rows: 16-byte unit u of row r (r = key & 15 of the half) sits in
// slot 4 r + (u ^ ((r >> 2) & 3)), so that the 64 dwords that one QK operand read takes lie in 64
// different banks. V rows and the scales keep their order ([key][64 bytes], [key][group]).
struct alignas(16) SharedTile {
  u32x4_t k[2][64];
  u32x4_t v[2][64];
  float ks[TILE * 4];
  float vs[TILE * 4];
};

// A wave's partial result: o [row][dim], then m and l per row.
template <int QT>
struct alignas(16) WavePartial {
  float o[16 * QT][OROW];
  float m[16 * QT], l[16 * QT];
};

template <int QT>
union SharedLds {
  SharedTile tiles[3][WAVES];
  WavePartial<QT> part[WAVES];
};

struct MaskWords {
  uint32_t w[SEG][33];  // keep bits of a tile's 32 keys per member of the row block; [32]: any member
};

// A unit of work: one stretch of one cache, and the query rows that attend to it.
struct Unit {
  const CacheView* c;
  int64_t crow;      // the cache's row
  int kvh;
  int t0, t1, S;     // the split's keys, the cache's live keys
  int64_t key0;      // the mask's key of cache row 0
  int row0, rows;    // first query row of the block, query rows of the unit
  int64_t b0;        // row of member 0 in q
  int split;         // partial slot
  int waves;         // waves of the workgroup that share the unit (1, 2 or 4)
  bool pack;         // the token goes into cache row S - 1
};

template <int G>
__device__ __forceinline__ void issue_tile(const uint8_t* kb, const uint8_t* vb, const float* ksb,
                                           const float* vsb, int kvo, int tb, int S, SharedTile& B,
                                           int lane) {
  tb = __builtin_amdgcn_readfirstlane(tb);
  const int rem = S - tb;  // > 0: keys past S read as 0
  const i32x4_t rk = make_desc(kb + (int64_t)tb * 64, rem * 64);
  const i32x4_t rv = make_desc(vb + (int64_t)tb * 64, rem * 64);
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    load_to_lds(rk, &B.k[h][0], kvo + 1024 * h);
    load_to_lds(rv, &B.v[h][0], 16 * lane + 1024 * h);
  }
  const i32x4_t rks = make_desc(ksb + (int64_t)tb * G, rem * G * 4);
  const i32x4_t rvs = make_desc(vsb + (int64_t)tb * G, rem * G * 4);
  // (lane 0 always issues these two, so that every tile counts 6 loads in the waits)
  if constexpr (G == 4) {
    if (lane < 32) {
      load_to_lds(rks, &B.ks[0], 16 * lane);
      load_to_lds(rvs, &B.vs[0], 16 * lane);
    }
  } else {
    if (lane < 32 * G) {
      load_to_lds_b32(rks, &B.ks[0], 4 * lane);
      load_to_lds_b32(rvs, &B.vs[0], 4 * lane);
    }
  }
}
constexpr int LPT = 6;  // loads per tile

// The scales of the lane's 8 keys q4 + 4e, all groups.
template <int G>
__device__ __forceinline__ void read_scales(const float* s, int q4, float (&out)[8][G]) {
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const float* at = s + (q4 + 4 * e) * G;
    if constexpr (G == 4) {
      const f32x4_t v = *(const f32x4_t*)at;
#pragma unroll
      for (int m = 0; m < 4; ++m) out[e][m] = v[m];
    } else {
#pragma unroll
      for (int m = 0; m < G; ++m) out[e][m] = at[m];
    }
  }
}

// A query row's 32 values of this lane (two per word) as fp16 operands q * 2^-e, 2^e being `scale`, e such
// that the row's largest value lies in [2^14, 2^15); zeros where the row is none.
template <int DT>
__device__ __forceinline__ void scale_query(const uint32_t (&w)[4][4], bool ok, u32x4_t (&op)[4],
                                            float& scale) {
  float qv[4][8];
  float mx = 0.0f;
#pragma unroll
  for (int k = 0; k < 4; ++k) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const uint32_t x = ok ? w[k][j] : 0u;
      qv[k][2 * j] = word_elem(x, 0, DT);
      qv[k][2 * j + 1] = word_elem(x, 16, DT);
      mx = fmaxf(mx, fmaxf(fabsf(qv[k][2 * j]), fabsf(qv[k][2 * j + 1])));
    }
  }
  mx = fmaxf(mx, __shfl_xor(mx, 16, 64));
  mx = fmaxf(mx, __shfl_xor(mx, 32, 64));
  int e = mx > 0.0f ? (int)((__float_as_uint(mx) >> 23) & 0xffu) - 127 - 14 : 0;
  e = max(-100, min(100, e));
  scale = __uint_as_float((uint32_t)(127 + e) << 23);
  const float inv = __uint_as_float((uint32_t)(127 - e) << 23);
#pragma unroll
  for (int k = 0; k < 4; ++k) {
#pragma unroll
    for (int j = 0; j < 4; ++j) op[k][j] = pack_f16(qv[k][j] * inv, qv[k][j + 4] * inv);
  }
}

// Two value nibbles (bits 3:0 and 19:16 of x) as a bf16 pair n / 16 (exact).
__device__ __forceinline__ uint32_t nib_pair_16th(uint32_t x) {
  const float a = __builtin_amdgcn_cvt_off_f32_i4((int)x);
  const float b = __builtin_amdgcn_cvt_off_f32_i4((int)(x >> 16));
  return __builtin_amdgcn_perm(__float_as_uint(b), __float_as_uint(a), 0x07060302u);
}

__device__ __forceinline__ f32x4_t mfma_bf16(u32x4_t a, u32x4_t b, f32x4_t c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, a),
                                                 __builtin_bit_cast(bf16x8_t, b), c, 0, 0, 0);
}

// a and b as TERMS bf16 pairs t[0] + t[1] + ..: each rounds what is left (to nearest), which the next
// subtraction gives exactly. The subtraction a - t.lo * 1 - t.hi * 0 is one v_dot2_f32_bf16, with the
// multipliers (-1, 0) in a register: as an inline constant, -1.0 stands for another pair in this instruction.
template <int TERMS>
__device__ __forceinline__ void split_pair(float a, float b, uint32_t minus_lo, uint32_t (&t)[TERMS]) {
#pragma unroll
  for (int i = 0; i < TERMS; ++i) {
    const bf16x2_t r = __builtin_convertvector(f32x2_t{a, b}, bf16x2_t);
    t[i] = __builtin_bit_cast(uint32_t, r);
    if (i + 1 < TERMS) {
      a = __builtin_amdgcn_fdot2_f32_bf16(r, __builtin_bit_cast(bf16x2_t, minus_lo), a, false);
      b = __builtin_amdgcn_fdot2_f32_bf16(r, __builtin_bit_cast(bf16x2_t, 0xbf800000u), b, false);
    }
  }
}

template <int QT, int G, int MASK, int TERMS>
__device__ __forceinline__ void run_unit(const SharedParams& p, const Unit& u, SharedTile* ring,
                                         MaskWords* words, WavePartial<QT>* part) {
  constexpr int CPG = 4 / G;  // 32-dim chunks per group
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  const int q4 = lane >> 4;
  const int c16 = lane & 15;
  const CacheView& c = *u.c;
  const uint8_t* kb = c.kp + u.crow * c.kps[0] + u.kvh * c.kps[1];
  const uint8_t* vb = c.vp + u.crow * c.vps[0] + u.kvh * c.vps[1];
  const float* ksb = c.ks + u.crow * c.kss[0] + u.kvh * c.kss[1];
  const float* vsb = c.vs + u.crow * c.vss[0] + u.kvh * c.vss[1];
  const int ntile = (u.t1 - u.t0 + TILE - 1) / TILE;
  const int member_wave = wave & (u.waves - 1);
  const int nw = ntile > member_wave ? (ntile - member_wave + u.waves - 1) / u.waves : 0;
  auto tile_key = [&](const int i) { return u.t0 + (member_wave + u.waves * i) * TILE; };
  // K slot l of a half holds row l >> 2, unit (l & 3) ^ ((l >> 4) & 3)
  const int kvo = (lane >> 2) * 64 + 16 * ((lane & 3) ^ ((lane >> 4) & 3));
  auto tile_at = [&](const int slot) -> SharedTile& { return ring[slot * WAVES + wave]; };
  for (int i = 0; i < 2; ++i) {
    if (i < nw) issue_tile<G>(kb, vb, ksb, vsb, kvo, tile_key(i), u.S, tile_at(i), lane);
  }

  // Query operands: lane (q4, c16) of column tile qt holds query row row0 + 16 qt + c16, dims
  // 32c + 8 q4 + (0,4,1,5,2,6,3,7) for chunk c, as fp16 q * 2^-e; cs turns its raw scores into exp2
  // units. Rows past the unit's count hold 0.
  // The rows' bits are loaded here and converted behind the mask's loads.
  u32x4_t qop[QT][4];
  float cs[QT];
  int member[QT];  // the row's member, relative to the row block's first
  uint32_t qbits[QT][4][4];
  const int first_member = u.row0 / p.nrep;
#pragma unroll
  for (int qt = 0; qt < QT; ++qt) {
    const int r = min(u.row0 + 16 * qt + c16, u.rows - 1);
    const int n = r / p.nrep;
    member[qt] = n - first_member;
    const int64_t base = (u.b0 + n) * p.q.s[0] + (int64_t)(u.kvh * p.nrep + r - n * p.nrep) * p.q.s[1];
    const uint16_t* at = (const uint16_t*)p.q.data + base;
    if (p.q_rows) {
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const u32x4_t v = *(const u32x4_t*)(at + 32 * k + 8 * q4);
#pragma unroll
        for (int j = 0; j < 4; ++j) qbits[qt][k][j] = v[j];
      }
    } else {
      uint32_t e[4][8];
#pragma unroll
      for (int k = 0; k < 4; ++k) {
#pragma unroll
        for (int j = 0; j < 8; ++j) e[k][j] = at[(32 * k + 8 * q4 + j) * p.q.s[2]];
      }
#pragma unroll
      for (int k = 0; k < 4; ++k) {
#pragma unroll
        for (int j = 0; j < 4; ++j) qbits[qt][k][j] = e[k][2 * j] | (e[k][2 * j + 1] << 16);
      }
    }
  }

  float m_run[QT], l_run[QT];
  f32x4_t acc[QT][8];
#pragma unroll
  for (int qt = 0; qt < QT; ++qt) {
    m_run[qt] = -INFINITY;
    l_run[qt] = 0.0f;
#pragma unroll
    for (int k = 0; k < 8; ++k) acc[qt][k] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
  }
  uint32_t minus_lo = 0x0000bf80u;  // bf16 (-1, 0)
  asm("" : "+s"(minus_lo));

  // Keep-mask: the wave turns the next SEG tiles' rows of the mask into one word of 32 keys per member
  // of its row block, lanes 0..31 for one member and 32..63 for the next.
  const int last_row = min(u.row0 + 16 * QT, u.rows) - 1;
  const int members = last_row / p.nrep - first_member + 1;
  auto make_words = [&](const int i0) {
    constexpr int BATCH = 8;  // loads in flight
    const int pairs = (members + 1) / 2;
    const int tiles = min(SEG, nw - i0);
    int i = 0, a = 0;  // tile and pair of the batch's first load
    for (int left = tiles * pairs; left > 0; left -= BATCH) {
      int ti[BATCH], ta[BATCH];
      bool keep[BATCH];
#pragma unroll
      for (int f = 0; f < BATCH; ++f) {
        ti[f] = i;
        ta[f] = a;
        const int n = 2 * a + (lane >> 5);
        const int64_t key = u.key0 + tile_key(i0 + i) + (lane & 31);
        keep[f] = false;
        if (f < left && n < members && key < p.mask_len) {
          keep[f] = ((const int64_t*)p.mask)[(u.b0 + first_member + n) * p.mask_sb + key * p.mask_sk] != 0;
        }
        if (++a == pairs) {
          a = 0;
          ++i;
        }
      }
#pragma unroll
      for (int f = 0; f < BATCH; ++f) {
        const uint64_t bits = __ballot(keep[f]);
        if (f < left && lane < 2) {
          words->w[ti[f]][2 * ta[f] + lane] = lane == 0 ? (uint32_t)bits : (uint32_t)(bits >> 32);
        }
      }
    }
    __builtin_amdgcn_wave_barrier();
    if (lane < tiles) {
      uint32_t any = 0;
      for (int n = 0; n < members; ++n) any |= words->w[lane][n];
      words->w[lane][32] = any;
    }
    __builtin_amdgcn_wave_barrier();
  };

  if constexpr (MASK == MASK_KEEP) {
    if (nw > 0) make_words(0);
  }
#pragma unroll
  for (int qt = 0; qt < QT; ++qt) {
    const bool ok = u.row0 + 16 * qt + c16 < u.rows;
    if (p.q.dtype == LQ_BF16) scale_query<LQ_BF16>(qbits[qt], ok, qop[qt], cs[qt]);
    else scale_query<LQ_F16>(qbits[qt], ok, qop[qt], cs[qt]);
    cs[qt] *= p.scale_sm;
  }

  const int krow = 4 * (c16 & 3) + (c16 >> 2);  // key of QK A-row c16 in its half
  // byte c16 & 3 of two dwords -> bytes 0 and 2
  const uint32_t vsel = 0x0c040c00u + (c16 & 3) * 0x00010001u;

  auto process = [&](const int i, SharedTile& B) {
    const int tb = tile_key(i);
    if constexpr (MASK == MASK_KEEP) {
      if (i > 0 && i % SEG == 0) make_words(i);
    }
    if (i + 2 < nw) wait_loads<2 * LPT>();
    else if (i + 1 < nw) wait_loads<LPT>();
    else wait_loads<0>();
    if (u.pack && tb <= u.S - 1 && u.S - 1 < tb + TILE) {
      // the new token: quantised, written to cache row S - 1 and over that key's row of the tile. Lane
      // j holds dims 2j and 2j + 1, a group is GH adjacent lanes.
      constexpr int GH = SD / (2 * G);
      const int key = u.S - 1 - tb;
      const int hk = key >> 4;
      const int r = key & 15;
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        const View& x = t == 0 ? p.knew : p.vnew;
        const int64_t at = u.crow * x.s[0] + u.kvh * x.s[1];
        const float x0 = load_float(x.data, x.dtype, at + 2 * lane * x.s[2]);
        const float x1 = load_float(x.data, x.dtype, at + (2 * lane + 1) * x.s[2]);
        const float scale = token_scale(group_max<GH>(fmaxf(fabsf(x0), fabsf(x1))));
        const uint8_t byte = (uint8_t)(token_level(x0, scale) | token_level(x1, scale) << 4);
        uint8_t* row = t == 0 ? (uint8_t*)&B.k[hk][4 * r + ((lane >> 4) ^ ((r >> 2) & 3))] + (lane & 15)
                              : (uint8_t*)&B.v[hk][0] + r * 64 + lane;
        *row = byte;
        const_cast<uint8_t*>(t == 0 ? kb : vb)[(int64_t)(u.S - 1) * 64 + lane] = byte;
        if ((lane & (GH - 1)) == 0) {
          (t == 0 ? B.ks : B.vs)[key * G + lane / GH] = scale;
          const_cast<float*>(t == 0 ? ksb : vsb)[(int64_t)(u.S - 1) * G + lane / GH] = scale;
        }
      }
      __builtin_amdgcn_wave_barrier();
    }

    // ---- scores, raw units: key slot e = 4t + r of lane group q4 is key tb + 16 t + 4 r + q4
    float s[QT][8];
    {
      float ks[8][G];
      read_scales<G>(B.ks, q4, ks);
      __builtin_amdgcn_s_setprio(1);
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        const uint32_t* kd = (const uint32_t*)&B.k[t][0];
#pragma unroll
        for (int m = 0; m < G; ++m) {
          u32x4_t ka[CPG];
#pragma unroll
          for (int cc = 0; cc < CPG; ++cc) {
            ka[cc] = decode_octet_f16(kd[4 * (4 * krow + ((m * CPG + cc) ^ (c16 & 3))) + q4]);
          }
#pragma unroll
          for (int qt = 0; qt < QT; ++qt) {
            f32x4_t a = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int cc = 0; cc < CPG; ++cc) a = mfma_f16(ka[cc], qop[qt][m * CPG + cc], a);
#pragma unroll
            for (int r = 0; r < 4; ++r) {
              const int e = 4 * t + r;
              s[qt][e] = m == 0 ? a[r] * ks[e][m] : fmaf(a[r], ks[e][m], s[qt][e]);
            }
          }
        }
      }
      __builtin_amdgcn_s_setprio(0);
    }
    // V operands of 32-dim chunk c: A row i of the two products is byte i of the chunk's 16 (its low
    // and its high nibble), so that a product's 16 dims belong to one group. Lane (q4, c16) takes its
    // byte of key rows q4 + 4e, key slots (2j, 2j+1) paired.
    u32x4_t va[4][2];
    {
      const uint32_t* vrow = (const uint32_t*)&B.v[0][0] + 16 * q4 + (c16 >> 2);
#pragma unroll
      for (int k = 0; k < 4; ++k) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const uint32_t a0 = vrow[64 * (2 * j) + 4 * k], a1 = vrow[64 * (2 * j + 1) + 4 * k];
          const uint32_t y = __builtin_amdgcn_perm(a1, a0, vsel);
          uint32_t high = y >> 4;
          asm("" : "+v"(high));  // (one shift for both of its nibbles: their word is an operand select)
          va[k][0][j] = nib_pair_16th(y);
          va[k][1][j] = nib_pair_16th(high);
        }
      }
    }
    float vs[8][G];
    read_scales<G>(B.vs, q4, vs);

    // ---- masks
    if constexpr (MASK == MASK_KEEP) {
      const uint32_t* w = words->w[i % SEG];
      const uint32_t any = w[32];
#pragma unroll
      for (int qt = 0; qt < QT; ++qt) {
        const uint32_t mine = w[member[qt]];
#pragma unroll
        for (int e = 0; e < 8; ++e) s[qt][e] = (mine >> (q4 + 4 * e) & 1) != 0 ? s[qt][e] : -INFINITY;
      }
#pragma unroll
      for (int e = 0; e < 8; ++e) {
#pragma unroll
        for (int m = 0; m < G; ++m) vs[e][m] = (any >> (q4 + 4 * e) & 1) != 0 ? vs[e][m] : 0.0f;
      }
    }
    if constexpr (MASK == MASK_BIAS) {
      // additive, in exp2 units: the scores are turned into those first
      uint32_t any = 0;  // keys that some query row of the wave attends to
#pragma unroll
      for (int qt = 0; qt < QT; ++qt) {
        const float* row = (const float*)p.mask + (u.b0 + first_member + member[qt]) * p.mask_sb;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const int64_t key = u.key0 + tb + q4 + 4 * e;
          const float bias = key < p.mask_len ? row[key * p.mask_sk] : -INFINITY;
          const bool on = bias != -INFINITY;
          s[qt][e] = on ? fmaf(s[qt][e], cs[qt], bias) : -INFINITY;
          any |= ((__ballot(on) >> (16 * q4)) & 0xffffu) != 0 ? 1u << e : 0u;
        }
      }
#pragma unroll
      for (int e = 0; e < 8; ++e) {
#pragma unroll
        for (int m = 0; m < G; ++m) vs[e][m] = (any >> e & 1) != 0 ? vs[e][m] : 0.0f;
      }
    }
    if (tb + TILE > u.t1) {  // keys past the split's range (their scales read as 0)
#pragma unroll
      for (int qt = 0; qt < QT; ++qt) {
#pragma unroll
        for (int e = 0; e < 8; ++e) s[qt][e] = tb + q4 + 4 * e < u.t1 ? s[qt][e] : -INFINITY;
      }
    }

    // ---- weights, below a running maximum of each row's scores
#pragma unroll
    for (int qt = 0; qt < QT; ++qt) {
      float lm = s[qt][0];
#pragma unroll
      for (int e = 1; e < 8; ++e) lm = fmaxf(lm, s[qt][e]);
      if constexpr (MASK != MASK_BIAS) lm *= cs[qt];
      if (__any(lm > m_run[qt] + LAZY)) {
        float mt = fmaxf(lm, __shfl_xor(lm, 16, 64));
        mt = fmaxf(mt, __shfl_xor(mt, 32, 64));
        const float m_new = fmaxf(m_run[qt], mt);
        // accumulators are still zero while m_run is -inf
        const float alpha = m_run[qt] == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(m_run[qt] - m_new);
#pragma unroll
        for (int k = 0; k < 8; ++k) acc[qt][k] *= alpha;
        l_run[qt] *= alpha;
        m_run[qt] = m_new;
      }
      // -inf only while every score so far is: 0 then, for 2^(-inf)
      const float m_use = m_run[qt] == -INFINITY ? 0.0f : m_run[qt];
      float psum = 0.0f;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        if constexpr (MASK == MASK_BIAS) {
          s[qt][e] = __builtin_amdgcn_exp2f(s[qt][e] - m_use);
        } else {
          s[qt][e] = __builtin_amdgcn_exp2f(fmaf(s[qt][e], cs[qt], -m_use));
        }
        psum += s[qt][e];
      }
      l_run[qt] += psum;
    }

    // ---- P' per group and the P V products
    __builtin_amdgcn_s_setprio(1);
#pragma unroll
    for (int m = 0; m < G; ++m) {
      u32x4_t pt[TERMS][QT];
#pragma unroll
      for (int qt = 0; qt < QT; ++qt) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          uint32_t t[TERMS];
          split_pair<TERMS>(s[qt][2 * j] * vs[2 * j][m], s[qt][2 * j + 1] * vs[2 * j + 1][m], minus_lo, t);
#pragma unroll
          for (int i = 0; i < TERMS; ++i) pt[i][qt][j] = t[i];
        }
      }
#pragma unroll
      for (int k = m * CPG; k < (m + 1) * CPG; ++k) {
#pragma unroll
        for (int i = 0; i < TERMS; ++i) {
#pragma unroll
          for (int t = 0; t < 2; ++t) {
#pragma unroll
            for (int qt = 0; qt < QT; ++qt) {
              acc[qt][2 * k + t] = mfma_bf16(va[k][t], pt[i][qt], acc[qt][2 * k + t]);
            }
          }
        }
      }
    }
    __builtin_amdgcn_s_setprio(0);
    __builtin_amdgcn_wave_barrier();
  };

  // 3-deep ring: the loads of the next two tiles are in flight while one is processed. (One body for all
  // ring positions: unrolled by three, the kernel's two units fill the instruction cache.)
  int slot = 0;
  for (int i = 0; i < nw; ++i) {
    const int fill = slot == 0 ? 2 : slot - 1;
    if (i + 2 < nw) issue_tile<G>(kb, vb, ksb, vsb, kvo, tile_key(i + 2), u.S, tile_at(fill), lane);
    process(i, tile_at(slot));
    slot = slot == 2 ? 0 : slot + 1;
  }

  const int ns = p.nsp + p.nso;
  // ---- the waves' states to LDS (over the tiles, which every wave has read), joined there
  __syncthreads();
  WavePartial<QT>& mine = part[wave];
#pragma unroll
  for (int qt = 0; qt < QT; ++qt) {
    float l = l_run[qt];
    l += __shfl_xor(l, 16, 64);
    l += __shfl_xor(l, 32, 64);
    const int row = 16 * qt + c16;
    if (q4 == 0) {
      mine.m[row] = m_run[qt];
      mine.l[row] = l;
    }
#pragma unroll
    for (int k = 0; k < 4; ++k) {  // dims 32k + 8 q4 + 2r + t
      float* o = &mine.o[row][32 * k + 8 * q4];
      const f32x4_t a = acc[qt][2 * k] * 16.0f, b = acc[qt][2 * k + 1] * 16.0f;
      *(f32x4_t*)o = f32x4_t{a[0], b[0], a[1], b[1]};
      *(f32x4_t*)(o + 4) = f32x4_t{a[2], b[2], a[3], b[3]};
    }
  }
  __syncthreads();
  const int w0 = wave & ~(u.waves - 1);  // the unit's first wave
  for (int i = threadIdx.x - 64 * w0; i < 16 * QT * (SD / 4); i += 64 * u.waves) {
    const int row = i / (SD / 4);
    const int d = 4 * (i % (SD / 4));
    if (u.row0 + row >= u.rows) break;
    float M = -INFINITY, L = 0.0f;
    for (int w = w0; w < w0 + u.waves; ++w) M = fmaxf(M, part[w].m[row]);
    f32x4_t o = {0.0f, 0.0f, 0.0f, 0.0f};
    for (int w = w0; w < w0 + u.waves; ++w) {
      const float wt = partial_weight(part[w].m[row], M);
      L += wt * part[w].l[row];
      o += wt * *(const f32x4_t*)&part[w].o[row][d];
    }
    const int n = (u.row0 + row) / p.nrep;
    const int qh = u.kvh * p.nrep + u.row0 + row - n * p.nrep;
    const int64_t b = u.b0 + n;
    if (ns == 1) {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        store_float(p.out.data, p.out.dtype, b * p.out.s[0] + qh * p.out.s[1] + (d + j) * p.out.s[2],
                    o[j] / L);
      }
    } else {
      const int64_t slot = (b * p.Hq + qh) * ns + u.split;
      *(f32x4_t*)&p.ws_acc[slot * SD + d] = o;
      if (d == 0) {
        p.ws_m[slot] = M;
        p.ws_l[slot] = L;
      }
    }
  }
}

// Workgroups: the prefix units first, the longer ones (KV head fastest, so that the row blocks that share
// keys lie on the same XCD where there are 8 KV heads; then row block, split, prompt), then the own units.
template <int QT, int G, int MASK, int TERMS>
__global__ __launch_bounds__(THREADS, 2) void shared_mfma_kernel(SharedParams p) {
  __shared__ SharedLds<QT> lds;
  __shared__ MaskWords words[MASK == MASK_KEEP ? WAVES : 1];
  const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  MaskWords* mine = &words[MASK == MASK_KEEP ? wave : 0];
  uint32_t i = blockIdx.x;
  Unit u;
  if (i < p.prefix_blocks) {
    u.kvh = i % p.Hkv;
    i /= p.Hkv;
    const int rb = i % p.rb_prefix;
    i /= p.rb_prefix;
    u.split = i % p.nsp;
    const int prompt = i / p.nsp;
    u.c = &p.prefix;
    u.crow = prompt;
    u.S = (int)p.prefix_len;
    u.t0 = u.split * (int)p.chunk_p;
    u.t1 = min(u.S, u.t0 + (int)p.chunk_p);
    u.key0 = 0;
    u.row0 = rb * 16 * QT;
    u.rows = p.N * p.nrep;
    u.b0 = (int64_t)prompt * p.N;
    u.pack = false;
    u.waves = WAVES;
    run_unit<QT, G, MASK, TERMS>(p, u, &lds.tiles[0][0], mine, lds.part);
    return;
  }
  // (a wave without a unit takes the last one's place with no query rows)
  u.waves = p.own_waves;
  i = (i - p.prefix_blocks) * (WAVES / p.own_waves) + (uint32_t)wave / p.own_waves;
  const bool none = i >= p.own_units;
  if (none) i = p.own_units - 1;
  u.kvh = i % p.Hkv;
  i /= p.Hkv;
  const int rb = i % p.rb_own;
  i /= p.rb_own;
  const int split = i % p.nso;
  const int b = i / p.nso;
  u.split = p.nsp + split;
  u.c = &p.own;
  u.crow = b;
  u.S = (int)p.own_len;
  u.t0 = split * (int)p.chunk_o;
  u.t1 = min(u.S, u.t0 + (int)p.chunk_o);
  u.key0 = p.prefix_len;
  u.row0 = rb * 16;
  u.rows = p.nrep;
  u.b0 = b;
  u.pack = p.pack && u.t1 == u.S;
  if (none) {
    u.t1 = u.t0;  // no keys
    u.row0 = u.rows;
    u.pack = false;
  }
  run_unit<1, G, MASK, TERMS>(p, u, &lds.tiles[0][0], mine, (WavePartial<1>*)lds.part);
}

template <int QT, int G, int MASK>
void launch_terms(const SharedParams& p, dim3 grid, hipStream_t st) {
  if (p.out.dtype == LQ_BF16) {
    hipLaunchKernelGGL((shared_mfma_kernel<QT, G, MASK, 2>), grid, dim3(THREADS), 0, st, p);
  } else {
    hipLaunchKernelGGL((shared_mfma_kernel<QT, G, MASK, 3>), grid, dim3(THREADS), 0, st, p);
  }
}

template <int QT, int G>
void launch_mask(const SharedParams& p, dim3 grid, hipStream_t st) {
  if (p.mask == nullptr) launch_terms<QT, G, MASK_NONE>(p, grid, st);
  else if (p.mask_keep) launch_terms<QT, G, MASK_KEEP>(p, grid, st);
  else launch_terms<QT, G, MASK_BIAS>(p, grid, st);
}

template <int G>
void launch_tiles(const SharedParams& p, dim3 grid, hipStream_t st) {
  if (p.col_tiles == 1) launch_mask<1, G>(p, grid, st);
  else launch_mask<2, G>(p, grid, st);
}

bool cache_ok(const CacheView& c, int64_t len, int64_t G) {
  // contiguous key rows: 64 packed bytes per key, D/g scale words per key; 4-byte aligned; 32-bit
  // extents of one (row, KV head) block
  if (c.kps[3] != 1 || c.vps[3] != 1 || c.kps[2] != 64 || c.vps[2] != 64) return false;
  if (c.kss[3] != 1 || c.vss[3] != 1 || c.kss[2] != G || c.vss[2] != G) return false;
  for (int64_t s : {c.kps[0], c.kps[1], c.vps[0], c.vps[1]}) {
    if (s % 4 != 0) return false;
  }
  for (const void* d : {(const void*)c.kp, (const void*)c.vp, (const void*)c.ks, (const void*)c.vs}) {
    if (((uintptr_t)d & 3) != 0) return false;
  }
  return len * 64 < (int64_t)1 << 31;
}

}  // namespace

bool shared_fast_shape_ok(int64_t head_dim, int group_size) {
  return head_dim == SD && (group_size == 32 || group_size == 64 || group_size == 128);
}

bool shared_fast_ok(const SharedParams& p) {
  if (diag(LQ_DIAG_ATTN_FORCE_GENERIC)) return false;
  if (!shared_fast_shape_ok(p.D, p.g)) return false;
  if (p.q.dtype != LQ_BF16 && p.q.dtype != LQ_F16) return false;
  const int64_t G = SD / p.g;
  if (!cache_ok(p.prefix, p.prefix_len, G) || !cache_ok(p.own, p.own_len, G)) return false;
  return ((uintptr_t)p.mask & (p.mask_keep ? 7 : 3)) == 0;
}

// Workgroups that run at once: two per CU (LDS and registers).
static int64_t resident_workgroups() { return 2 * (int64_t)device_cus(); }

// Column tiles of 16 query rows per wave in the prefix units.
static int col_tiles_of(int64_t rows) { return rows <= 16 ? 1 : 2; }

SharedPlan plan_shared_fast(int64_t P, int64_t N, int64_t Hkv, int64_t nrep, int64_t prefix_len,
                            int64_t own_len) {
  const int64_t resident = resident_workgroups();
  const int64_t rows = N * nrep;
  const int64_t block = 16 * col_tiles_of(rows);
  const int64_t units = std::max<int64_t>(1, P * Hkv * ((rows + block - 1) / block));
  const int64_t own_units = std::max<int64_t>(1, P * N * Hkv * ((nrep + 15) / 16));
  constexpr int64_t STEP = WAVES * TILE;
  // One prefix workgroup per CU leaves the other place to the own units and halves the set-ups and partials;
  // two hide each other's waits. The first pays up to about 12 tiles per wave (9 with 16 query rows) and one
  // more for each of the first 6 own tiles. Measured with one and with two, group 32: 60 own rows, 1 prompt
  // x 16, 4 tiles 21.0 us for 26.9, 8 x 8, 10 tiles 32.1 for 33.8, 14 tiles 39.7 for 39.0, 18 tiles 47.1 for
  // 43.7; 200 own rows, 8 x 8, 14 tiles 39.8 for 41.5, 18 tiles 47.2 for 46.4, 24 tiles 58.2 for 53.8; 4 x 4
  // (16 query rows), 60 own rows, 10 tiles 23.3 for 25.4, 14 tiles 28.6 for 28.5, 16 tiles 31.3 for 30.0.
  const int64_t own_tiles = std::min<int64_t>(6, (own_len + TILE - 1) / TILE);
  SharedPlan plan{split_of(prefix_len, device_cus() / units, STEP),
                  split_of(own_len, resident / own_units, 2 * STEP)};
  if (plan.prefix.chunk > ((block == 16 ? 9 : 12) + own_tiles) * STEP) {
    plan.prefix = split_of(prefix_len, resident / units, STEP);
  }
  return plan;
}

int launch_shared_fast(SharedParams p, hipStream_t st) {
  const int64_t rows = (int64_t)p.N * p.nrep;
  p.col_tiles = col_tiles_of(rows);
  p.rb_prefix = (int)((rows + 16 * p.col_tiles - 1) / (16 * p.col_tiles));
  p.rb_own = (p.nrep + 15) / 16;
  const int64_t pb = (int64_t)p.P * p.Hkv * p.rb_prefix * p.nsp;
  const int64_t units = (int64_t)p.B * p.Hkv * p.rb_own * p.nso;
  // Waves per own unit: a whole workgroup where every one has its place at once, the shortest chain of
  // steps (1 prompt x 16, ctx 2000, 100 own rows: 14.9 us, 15.9 with two waves, 18.8 with one); where they
  // wait for places behind the prefix, fewer and fuller ones (8 x 8, ctx 16384: 100 rows 64.1 us with four
  // waves, 63.6 with two, 65.2 with one; 200 rows 68.0, 64.6 and 67.4; 64 rows 66.4, 66.1 and 66.5).
  const int64_t tiles = (std::min(p.chunk_o, p.own_len) + TILE - 1) / TILE;
  p.own_waves = pb + units <= resident_workgroups() ? 4 : tiles <= 2 ? 1 : tiles <= 8 ? 2 : 4;
  const int64_t ob = (units * p.own_waves + WAVES - 1) / WAVES;
  p.own_units = (uint32_t)units;
  if ((pb + ob) * THREADS >= (int64_t)1 << 32) {  // threads of a launch
    return fail(LQ_ERR_UNSUPPORTED, "%lld workgroups exceed the launch limits", (long long)(pb + ob));
  }
  p.prefix_blocks = (uint32_t)pb;
  const View& q = p.q;
  p.q_rows = q.s[2] == 1 && ((uintptr_t)q.data & 15) == 0 && q.s[0] % 8 == 0 && q.s[1] % 8 == 0;
  const dim3 grid((unsigned)(pb + ob));
  switch (SD / p.g) {
    case 4: launch_tiles<4>(p, grid, st); break;
    case 2: launch_tiles<2>(p, grid, st); break;
    default: launch_tiles<1>(p, grid, st); break;
  }
  return check_launch("lq_int4_shared_decode_attention (mfma)");
}

}  // namespace lq
