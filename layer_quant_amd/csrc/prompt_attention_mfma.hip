// prompt_attention.hip's operator for 16-bit inputs on v_mfma_f32_32x32x16_{bf16,f16}: head_dim 64 or
// 128, rows of q, k, v and out contiguous and 16-byte aligned.
//
// A workgroup of NW waves has 32 NW rows (positions x query heads, prompt_attention.hip) of one KV head
// and walks the keys in tiles of 64, which buffer loads write to one of two LDS buffers while the other
// is worked on: one barrier per tile. Per tile and wave
//   S^T[key][row] = K Q^T   A = K rows (16-byte LDS reads), B = the wave's query rows, in registers
//   p = 2^(c s - c m)       c = scale log2(e); a lane has one row's scores (32 of the 64, the lane 32
//                           away the others), so the row's maximum takes one exchange
//   O^T[dim][row] += V^T P^T   B = P^T: the eight scores that a lane holds of 16 keys are its B operand
//                           as they are, if the keys of the products' K slots are taken in that order:
//                           slots 0-3 and 4-7 of half h are keys 4 h .. + 3 and 8 + 4 h .. + 3. A = V^T
//                           by ds_read_b64_tr_b16, which hands a lane four keys of one dim.
// The rows of both tiles are swizzled by 16-byte chunks, through the addresses that the loading lanes
// read from, so that these reads meet no bank twice: K's chunk c of row r lies in chunk c ^ (r mod 16),
// V's in c ^ 4 (r mod 4) (the D = 64 forms in swizzle_k and swizzle_v).
//
// The running maximum moves only when a score exceeds it by 2^LAZY: p <= 2^8 then, and the 64
// accumulators are rescaled in a few tiles only. Weights are rounded to the inputs' type, their sum is
// fp32 and of the unrounded ones: the rounding is half a step per weight, as if the values had it. fp16 ones are
// raised by 2^7, so that this holds down to 2^-21 of the largest weight so far; below it they are off by 2^-32
// of that one.
//
// Masked keys of a row have p = 0, which a value of inf or NaN would turn into NaN. Results that are not
// finite are rare, so it is they that are looked for: a workgroup with one runs its rows again, and then
// hands such values to the rows that see them and takes them out of the tile. As unnormalised sums of values
// next to bf16's largest can leave fp32, the weights are smaller then (PROMPT_ATTENTION_DOWN). Weights that are
// too large or all 0 because scores beyond 2^30 round c m by too much are made from s - m.
//
// What it measured (MI355X, 32 query / 8 KV heads of 128, us per call): one prompt of 16384 rows 1995-2054,
// 1.07-1.10 PFLOP/s, where the library's large bf16 product reaches 1.14; 24 fp16 prompts up to 700 rows 31.6;
// one of 333 rows 11.5. Bound by issue: per tile and wave 32 matrix instructions of 32 cycles and the softmax's VALU
// instructions; the short prompt by latency, six tiles in a row behind the span search and cold instructions; the
// 24 by their order too: the one of 700 rows is the 20th, and its workgroups, of eleven tiles, begin late
// (longest first 26.5 us where the given order takes 33-35, shortest first 33-35). prompt_attention_f32 in its
// first form, one value per load, took 57 ms, 518 and 131.
#include "matrix16.h"
#include "prompt_attention.h"

namespace lq {
namespace {

constexpr int KT = 64;    // keys per tile
constexpr int ROWS = 32;  // rows per wave
constexpr float LAZY = 8.f;
constexpr float RAISE = 7.f;  // of fp16 weights' exponents: 2^(LAZY + RAISE) is in fp16

// Chunks by which a tile row's chunks are exchanged. D = 128 (256-byte rows): 16 rows' equal chunks, and
// 4 rows' runs of 4 chunks, lie in different banks. D = 64: two rows share 256 bytes.
template <int D>
__device__ __forceinline__ int swizzle_k(int r) {
  return D == 128 ? r & 15 : (r >> 1) & 7;
}
template <int D>
__device__ __forceinline__ int swizzle_v(int r) {
  return D == 128 ? 4 * (r & 3) : 4 * ((r >> 1) & 1);
}

template <int D>
using Tiles = char[2][2][KT * 2 * D];  // [buffer][K, V]

// A span's rows of a workgroup; whether they have to run again, with CAREFUL.
template <bool BF, int D, int NW, bool CAREFUL>
__device__ __forceinline__ bool attend(const PromptAttention& p, const Span& sp, int hk, int tid, Tiles<D>& tiles) {
  constexpr int ROW_BYTES = 2 * D, CH = D / 8, TILE = KT * ROW_BYTES;
  constexpr int PER_LOAD = 64 / CH;                 // rows of one load
  constexpr int LOADS = KT / PER_LOAD / NW;         // of K, and of V, per wave and tile
  static_assert(LOADS * PER_LOAD * NW == KT, "every wave loads as many rows");
  const int nrep = p.nrep, lane = tid & 63, col = lane & 31, hi = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int nrows = sp.len * nrep, parts = (nrows + NW * ROWS - 1) / (NW * ROWS);
  // the last rows of a prompt have the most keys: they go first
  const int first = (parts - 1 - sp.part) * NW * ROWS;
  const int r = first + wave * ROWS + col, at = min(r, nrows - 1);
  const int pos = at / nrep, head = hk * nrep + at - pos * nrep;
  const int64_t lead = p.spans.starts == nullptr ? sp.index : 0, row = sp.begin + pos;
  uint16_t* out = (uint16_t*)p.out.data + lead * p.out.s[0] + row * p.out.s[1] + head * p.out.s[2];
  if (!CAREFUL && sp.gap) {
    if (r < nrows) {
#pragma unroll
      for (int i = 0; i < CH / 2; ++i) *(words4_t*)(out + 8 * (2 * i + hi)) = words4_t{0, 0, 0, 0};
    }
    return false;
  }

  words4_t q[D / 16];  // dims 16 i + 8 hi .. + 7
  {
    const uint16_t* from = (const uint16_t*)p.q.data + lead * p.q.s[0] + row * p.q.s[1] + head * p.q.s[2];
#pragma unroll
    for (int i = 0; i < D / 16; ++i) {
      q[i] = *(const words4_t*)(from + 16 * i + 8 * hi);
#pragma unroll
      for (int e = 0; e < 4; ++e) q[i][e] = (q[i][e] & p.q_and) ^ p.q_xor;
    }
  }

  const int ks = (int)p.k.s[1] * 2, vs = (int)p.v.s[1] * 2;  // bytes between rows
  const char* kbase = (const char*)p.k.data + (lead * p.k.s[0] + sp.begin * p.k.s[1] + hk * p.k.s[2]) * 2;
  const char* vbase = (const char*)p.v.data + (lead * p.v.s[0] + sp.begin * p.v.s[1] + hk * p.v.s[2]) * 2;
  int koff[LOADS], voff[LOADS];
#pragma unroll
  for (int j = 0; j < LOADS; ++j) {
    const int tr = (wave * LOADS + j) * PER_LOAD + lane / CH, c = lane % CH;
    koff[j] = tr * ks + 16 * (c ^ swizzle_k<D>(tr));
    voff[j] = tr * vs + 16 * (c ^ swizzle_v<D>(tr));
  }
  auto load_tile = [&](int kb, int buf) {
    const int have = min(KT, sp.len - kb);  // rows past the prompt read as zero
    const i32x4_t kd = make_desc(kbase + (int64_t)kb * ks, (have - 1) * ks + ROW_BYTES);
    const i32x4_t vd = make_desc(vbase + (int64_t)kb * vs, (have - 1) * vs + ROW_BYTES);
    lds_t to = (lds_t)&tiles[buf][0][0] + wave * LOADS * 1024;
#pragma unroll
    for (int j = 0; j < LOADS; ++j) load_rows_to_lds(kd, to + j * 1024, koff[j]);
#pragma unroll
    for (int j = 0; j < LOADS; ++j) load_rows_to_lds(vd, to + TILE + j * 1024, voff[j]);
  };

  // LDS addresses of the lane's A operands, before the products' steps (which exchange chunks: ^)
  const int kaddr = col * ROW_BYTES + 16 * (hi ^ swizzle_k<D>(col));
  const int vrow = 4 * hi + ((lane & 15) >> 2);
  const int vaddr = vrow * ROW_BYTES + 8 * (lane & 1) +
                    16 * ((2 * ((lane >> 4) & 1) + ((lane >> 1) & 1)) ^ swizzle_v<D>(vrow));

  const int pos_first = first / nrep;                                 // of the workgroup
  const int pos_last = min(first + NW * ROWS - 1, nrows - 1) / nrep;
  const int wave_first = __builtin_amdgcn_readfirstlane(min(first + wave * ROWS, nrows - 1) / nrep);
  const int wave_last = __builtin_amdgcn_readfirstlane(min(first + wave * ROWS + ROWS - 1, nrows - 1) / nrep);
  f32x16_t o[D / 32];
  float m = -INFINITY, l = 0.f;
#pragma unroll
  for (int i = 0; i < D / 32; ++i) o[i] = f32x16_t{};
  load_tile(0, 0);
  for (int kb = 0, buf = 0; kb <= pos_last; kb += KT, buf ^= 1) {
    wait_loads<0>();
    __syncthreads();
    if (kb + KT <= pos_last) load_tile(kb + KT, buf ^ 1);
    lds_t kt = (lds_t)&tiles[buf][0][0], vt = (lds_t)&tiles[buf][1][0];
    if (CAREFUL && kb + KT - 1 > pos_first) {
      uint16_t* v = (uint16_t*)&tiles[buf][1][0];
      constexpr uint32_t INF = BF ? 0x7f80 : 0x7c00;
      for (int key = 0; key < KT; ++key) {
        if (kb + key > pos) continue;
#pragma unroll
        for (int b = 0; b < D / 32; ++b) {
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            const int d = 32 * b + 8 * (i >> 2) + 4 * hi + (i & 3);
            const uint32_t x = v[key * D + 8 * ((d >> 3) ^ swizzle_v<D>(key)) + (d & 7)];
            if ((x & INF) == INF) {
              o[b][i] += BF ? bf16_bits_to_float(x) : (float)__builtin_bit_cast(_Float16, (uint16_t)x);
            }
          }
        }
      }
      __syncthreads();
      for (int i = tid; i < KT * D; i += 64 * NW) {
        if ((v[i] & INF) == INF) v[i] = 0;
      }
      __syncthreads();
    }
    if (kb > wave_last) continue;
    f32x16_t s[2] = {};
#pragma unroll
    for (int i = 0; i < D / 16; ++i) {
#pragma unroll
      for (int b = 0; b < 2; ++b) {
        s[b] = mfma<BF>(lds_read16(kt + (kaddr ^ (32 * i)) + b * 32 * ROW_BYTES), q[i], s[b]);
      }
    }
    if (kb + KT - 1 > wave_first) {
#pragma unroll
      for (int b = 0; b < 2; ++b) {
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          if (kb + 32 * b + 8 * (i >> 2) + 4 * hi + (i & 3) > pos) s[b][i] = -INFINITY;
        }
      }
    }
    float top = s[0][0];
#pragma unroll
    for (int i = 1; i < 32; ++i) top = fmaxf(top, s[i >> 4][i & 15]);
    top = fmaxf(top, __shfl_xor(top, 32, 64));
    if (__any((top - m) * p.scale > LAZY || m == -INFINITY)) {
      const float to = fmaxf(m, top);
      // all keys so far at -inf: no weight yet
      float keep = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f((m - to) * p.scale);
      m = to;
      l *= keep;
      if (CAREFUL && __any(keep == 0.f)) {  // the infinities, this tile's among them, stay
#pragma unroll
        for (int i = 0; i < D / 2; ++i) {
          const float x = o[i >> 4][i & 15];
          o[i >> 4][i & 15] = keep == 0.f && x - x == 0.f ? 0.f : x;
        }
        keep = keep == 0.f ? 1.f : keep;
      }
#pragma unroll
      for (int b = 0; b < D / 32; ++b) o[b] *= keep;
    }
    const float rounded = m == -INFINITY ? 0.f : m * p.scale, base = BF ? rounded : rounded - RAISE;
    const bool far = fabsf(rounded) >= 0x1p24f;  // its rounding is no small factor of all weights
    words4_t pk[4];
    float sum = 0.f;  // (by itself: many small terms, each rounded beside a large l, would be off together)
#pragma unroll
    for (int b = 0; b < 2; ++b) {
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        float z = fmaf(s[b][i], p.scale, -base);
        if (CAREFUL && far) z = (s[b][i] - m) * p.scale + (BF ? 0.f : RAISE);
        s[b][i] = __builtin_amdgcn_exp2f(z);
        sum += s[b][i];
      }
      if (BF && CAREFUL) s[b] *= PROMPT_ATTENTION_DOWN;  // (fp16 values are too small to need it)
#pragma unroll
      for (int i = 0; i < 8; ++i) pk[2 * b + (i >> 2)][i & 3] = pack2<BF>(s[b][2 * i], s[b][2 * i + 1]);
    }
    l += sum;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
#pragma unroll
      for (int b = 0; b < D / 32; ++b) {
        lds_t from = vt + (vaddr ^ (64 * b)) + 16 * j * ROW_BYTES;
        o[b] = mfma<BF>(lds_read_columns(from, from + 8 * ROW_BYTES), pk[j], o[b]);
      }
    }
  }
  l += __shfl_xor(l, 32, 64);
  if (!CAREFUL) {
    // sum of the accumulators times 0: NaN if one is not finite
    float odd = l * 0.f;
#pragma unroll
    for (int b = 0; b < D / 32; ++b) {
#pragma unroll
      for (int i = 0; i < 16; ++i) odd = fmaf(o[b][i], 0.f, odd);
    }
    if (__syncthreads_or(odd != 0.f || l == 0.f)) return true;
  }
  const float inv = (BF && CAREFUL ? 1.f / PROMPT_ATTENTION_DOWN : 1.f) / l;
  if (r >= nrows) return false;
#pragma unroll
  for (int b = 0; b < D / 32; ++b) {
#pragma unroll
    for (int a = 0; a < 2; ++a) {
      // a lane has dims 0-3 (hi: 4-7) and 8-11 (12-15) of 16: the halves exchange to 8 in a row each
      uint32_t w[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) w[i] = pack2<BF>(o[b][8 * a + 2 * i] * inv, o[b][8 * a + 2 * i + 1] * inv);
      const auto x = __builtin_amdgcn_permlane32_swap(w[0], w[2], false, false);
      const auto y = __builtin_amdgcn_permlane32_swap(w[1], w[3], false, false);
      *(words4_t*)(out + 32 * b + 16 * a + 8 * hi) = words4_t{x[0], y[0], x[1], y[1]};
    }
  }
  return false;
}

template <bool BF, int D, int NW>
__global__ __launch_bounds__(64 * NW, D == 64 ? 3 : 2) void prompt_attention_mfma(PromptAttention p) {
  __shared__ __attribute__((aligned(1024))) Tiles<D> tiles;
  int hk = blockIdx.x % p.Hkv, tid = threadIdx.x;
  Span sp;
  if (!find_part(p, blockIdx.x / p.Hkv, sp)) return;
  if (!attend<BF, D, NW, false>(p, sp, hk, tid, tiles)) return;
  // Again, from values hidden from the compiler: it would keep what the first run made of them in registers
  // for the second one, through the loop.
  asm volatile("" : "+s"(sp.index), "+s"(sp.begin), "+s"(sp.len), "+s"(sp.part), "+s"(hk), "+v"(tid));
  attend<BF, D, NW, true>(p, sp, hk, tid, tiles);
}

// A row's elements in a row, every row 16-byte aligned, 64 rows within 31 bits of bytes.
bool rows_fit(const lq_tensor* t) {
  const int nd = t->ndim;
  if (t->stride[nd - 1] != 1 || ((uintptr_t)t->data & 15) != 0) return false;
  for (int i = 0; i < nd - 1; ++i) {
    if (t->shape[i] > 1 && t->stride[i] % 8 != 0) return false;
  }
  return true;
}

}  // namespace

bool prompt_attention_mfma_fits(const lq_tensor* q, const lq_tensor* k, const lq_tensor* v,
                                const lq_tensor* out) {
  const int nd = q->ndim;
  const int64_t D = q->shape[nd - 1];
  if (q->dtype == LQ_F32 || (D != 64 && D != 128)) return false;
  const lq_tensor* ts[4] = {q, k, v, out};
  for (const lq_tensor* t : ts) {
    if (!rows_fit(t)) return false;
  }
  const lq_tensor* kv[2] = {k, v};
  for (const lq_tensor* t : kv) {
    const int64_t s = t->stride[nd - 3];
    if (t->shape[nd - 3] > 1 && (s < D || s > (1 << 22))) return false;
  }
  return true;
}

int launch_prompt_attention_mfma(const PromptAttention& p, int dtype, int64_t parts, hipStream_t st) {
  const dim3 grid((unsigned)(parts * p.Hkv)), block(64 * PROMPT_ATTENTION_WAVES);
  constexpr int NW = PROMPT_ATTENTION_WAVES;
  if (dtype == LQ_BF16) {
    if (p.D == 64) hipLaunchKernelGGL((prompt_attention_mfma<true, 64, NW>), grid, block, 0, st, p);
    else hipLaunchKernelGGL((prompt_attention_mfma<true, 128, NW>), grid, block, 0, st, p);
  } else {
    if (p.D == 64) hipLaunchKernelGGL((prompt_attention_mfma<false, 64, NW>), grid, block, 0, st, p);
    else hipLaunchKernelGGL((prompt_attention_mfma<false, 128, NW>), grid, block, 0, st, p);
  }
  return check_launch("lq_prompt_attention");
}

}  // namespace lq
