// prompt_scan.hip's operator for bf16 x, B and C with head_dim 64 and a state of 128, on
// v_mfma_f32_32x32x16_bf16: prompts in chunks of 64 rows. With c the running sum of A dt log2(e) within a
// chunk, S the state in front of it and t, s rows of it,
//   Y[t] = 2^c_t S C_t + sum_{s <= t} M[t][s] x_s + D x_t,  M[t][s] = 2^(c_t - c_s) dt_s (C_t . B_s)
//   S'   = 2^c_63 S + sum_s w_s x_s B_s^T,          w_s = 2^(c_63 - c_s) dt_s
// c is summed in 64 bits and taken apart into a whole number n and a rest: 2^(c_t - c_s) is the product of
// 2^(n_t - n_s), exact, and of two factors between 0.7 and 1.42 that a row has once. So no decay overflows
// however fast a state fades, close rows behind a large c keep their digits, and no element of M takes an
// exponential. (A step's decay is held within 2^-256 and 2^256.) scan_steps_kernel makes these numbers of
// every row and head beforehand: in this kernel one wave made them while the others waited, 260 us of 539
// for a prompt of 16384 rows.
//
// A workgroup of four waves has two heads of one group; wave (head, half) keeps rows p = 32 half .. + 31 of
// its head's state, transposed, in 64 accumulators. Of B^T x that is the layout in which S is, rounded to
// bf16, the A operand of S C^T without leaving its registers, once the columns that the transposing reads
// hand to the lanes are taken in the order sigma: lane bits (8 a + 4 h + b) <-> index (8 h + 4 a + b). The
// same order makes eight consecutive values of every result meet in one lane.
// Per chunk:
//   phase 1  S C^T (16 products) with C's operands shared by the mixing scores B C^T, of which three waves
//            make one 32 x 32 block each (the fourth lies above the diagonal) for both heads and leave M in
//            LDS as bf16
//   phase 2  Y += M x + D x (6 and 4 products), stores, S' (32 or 48 products)
// B lies in two LDS buffers; x goes to registers at once, and C and the decays are read in phase 1 alone, so
// that one buffer each does, refilled from then on: 79 KB per workgroup, two of them per CU.
//
// What it measured (MI355X, 128 heads, 8 groups, us): one prompt of 16384 rows 318-328 (steps 15-18, what the
// segments add 90-103, carry 13, the segments 203-229), 24 prompts up to 700 rows with fp32 states 124 (8 + 3-5 + 5 +
// 110-112; longest first 105: the one of 700 rows is the 20th and begins late), one of 200 rows 25.3 (5 + 20). A chunk
// takes a workgroup 3.3 us alone on its CU, 3.7 with fp32 states, and 6.3-7.2 beside another one: per wave 70 matrix
// instructions (32 cycles) and 600 other VALU ones (4), which add up, are 1.9 us at 2.4 GHz; the rest is the latency
// of LDS and of three barriers. Tried, with one value of w x (50 matrix instructions, 289 us): one workgroup of eight
// waves and four heads with M in registers and a single barrier (313); loads further ahead into L2 (no gain); heads to
// XCDs in other orders (no difference); the last block's heads shared out to two waves (297).
//
// Roundings: M and S to bf16 as operands (half a step, 2^-8, of each term of a bf16 result), D to the sum of two
// bf16 values (2^-17). w x, which a state keeps, to the sum of two bf16 values (2^-16) where the state leaves in 16 bits, and of three (its 24
// bits) where it leaves in fp32: 700 rows' fp32 states are off by less than 5e-7 with three, 2e-6 with two (24
// prompts 123 us, 117), and bf16 ones by 0.0017, their own rounding, with two, 0.0024 with one (16384 rows 312
// us, 285). y is off by 0.0019-0.0022 of itself, of which its own rounding is 0.0017; with D as one bf16 value it
// was 0.0023 (16384 rows 316 us, 325 with two; D's rest in M's diagonal instead of products of its own 328, 24
// prompts 134 us against 124). Everything else is fp32.
//
// Rows behind a row in its chunk have M = 0 there, which an x of inf or NaN would turn into NaN. Such a value
// stays in the state, so that it is enough to look at the state behind a segment: one that is not finite has
// the segment run again, and then they are added to the rows that see them and left out of M x.
#include "matrix16.h"
#include "prompt_scan.h"

namespace lq {
namespace {

constexpr int Q = 64;      // rows of a chunk
constexpr int HEADS = 2;   // of a workgroup
constexpr int P = 64, N = 128;

// Inclusive sums over the wave's lanes.
template <int CTRL, int ROWS>
__device__ __forceinline__ double moved(double v) {
  const uint64_t u = __builtin_bit_cast(uint64_t, v);
  const uint32_t lo = __builtin_amdgcn_update_dpp(0, (uint32_t)u, CTRL, ROWS, 0xf, false);
  const uint32_t hi = __builtin_amdgcn_update_dpp(0, (uint32_t)(u >> 32), CTRL, ROWS, 0xf, false);
  return __builtin_bit_cast(double, ((uint64_t)hi << 32) | lo);
}
__device__ __forceinline__ double prefix_sum(double v) {
  v += moved<0x111, 0xf>(v);  // row_shr 1, 2, 4, 8
  v += moved<0x112, 0xf>(v);
  v += moved<0x114, 0xf>(v);
  v += moved<0x118, 0xf>(v);
  v += moved<0x142, 0xa>(v);  // row_bcast 15, 31
  v += moved<0x143, 0xc>(v);
  return v;
}

struct alignas(1024) ChunkLds {
  char b[2][Q * N * 2];         // rows of 256 bytes; chunk k of row r at k ^ swizzle_b(r)
  char c[Q * N * 2];            // the same with k ^ (r mod 16)
  char x[HEADS][Q * P * 2];     // rows of 128 bytes, k ^ 4 ((r / 2) mod 2)
  char m[HEADS][3][32 * 32 * 2];  // blocks (s, t) = (0, 0), (0, 1), (1, 1): row t, 64 bytes
  float weight[2][HEADS][Q];    // w_s
  int whole[HEADS][Q];          // n_s
  float rest[HEADS][Q];         // 2^(c_s - n_s)
  float step[HEADS][Q];         // dt_s 2^(n_s - c_s)
};

// scan_steps_kernel's arrays, in p.steps: [array][head][row]
enum { WEIGHT, WHOLE, REST, STEP };

constexpr int STEP_HEADS = 16;  // of a workgroup of scan_steps_kernel

// A chunk's decays and steps, lane = row.
__global__ __launch_bounds__(256) void scan_steps_kernel(PromptScan p) {
  __shared__ float tile[Q][STEP_HEADS + 1];
  const int blocks = (p.H + STEP_HEADS - 1) / STEP_HEADS, hb = blockIdx.x % blocks * STEP_HEADS;
  Span sp;
  if (!find_span<false>(p.spans, blockIdx.x / blocks, [](int len, bool) { return (len + Q - 1) / Q; },
                        [](int begin, int i) { return begin / Q + i; }, sp)) {
    return;
  }
  const int64_t lead = p.spans.starts == nullptr ? sp.index : 0, row0 = sp.begin + sp.part * Q;
  const int have = min(Q, sp.len - sp.part * Q), heads = min(STEP_HEADS, p.H - hb);
  for (int i = threadIdx.x; i < have * STEP_HEADS; i += 256) {
    const int r = i / STEP_HEADS, j = i % STEP_HEADS;
    if (j >= heads) continue;
    tile[r][j] = load_float(p.dt.data, p.dt.dtype,
                            lead * p.dt.s[0] + (row0 + r) * p.dt.s[1] + (hb + j) * p.dt.s[2]);
  }
  __syncthreads();
  const int lane = threadIdx.x & 63;
  for (int j = threadIdx.x >> 6; j < heads; j += 4) {
    const int h = hb + j;
    const double A = (double)load_float(p.A.data, p.A.dtype, h * p.A.s[0]) * 1.4426950408889634;
    const float bias = p.bias.data == nullptr ? 0.f : load_float(p.bias.data, p.bias.dtype, h * p.bias.s[0]);
    const bool in = lane < have;
    float dt = in ? scan_step(p, tile[lane][j], bias) : 0.f;
    // a decay that is NaN counts as one here, and has its NaN in what the step multiplies
    const double lg = A * dt;
    if (in && lg != lg) dt = __builtin_nanf("");
    const double c = prefix_sum(in ? fmin(fmax(lg, -256.0), 256.0) : 0.0);
    const uint64_t u = __builtin_bit_cast(uint64_t, c);
    const uint32_t lo = __builtin_amdgcn_readlane((uint32_t)u, 63);
    const uint32_t up = __builtin_amdgcn_readlane((uint32_t)(u >> 32), 63);
    const double all = __builtin_bit_cast(double, ((uint64_t)up << 32) | lo), whole = __builtin_rint(c);
    const float rest = (float)(c - whole);
    if (!in) continue;
    float* to = p.steps + h * p.rows + lead * p.spans.rows + row0 + lane;
    const int64_t array = p.H * p.rows;
    to[WEIGHT * array] = dt * __builtin_amdgcn_exp2f((float)(all - c));
    to[WHOLE * array] = __int_as_float((int)whole);
    to[REST * array] = __builtin_amdgcn_exp2f(rest);
    to[STEP * array] = dt * __builtin_amdgcn_exp2f(-rest);
  }
}

// Both four consecutive rows' runs of 4 chunks and 16 rows' equal chunks lie in different banks.
__device__ __forceinline__ int swizzle_b(int r) { return 4 * (r & 3) | ((r >> 2) & 3); }

// index of lane (or result row) m
__device__ __forceinline__ int sigma(int m) { return (m & ~12) | ((m & 4) << 1) | ((m & 8) >> 1); }

// Eight consecutive state values.
__device__ __forceinline__ void load8(const char* at, int dtype, float (&v)[8]) {
  if (dtype == LQ_F32) {
    const float4 a = ((const float4*)at)[0], b = ((const float4*)at)[1];
    v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w, v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
    return;
  }
  const words4_t w = *(const words4_t*)at;
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = word_elem(w[i >> 1], (i & 1) * 16, dtype);
}
__device__ __forceinline__ void store8(char* at, int dtype, const float (&v)[8]) {
  if (dtype == LQ_F32) {
    ((float4*)at)[0] = make_float4(v[0], v[1], v[2], v[3]);
    ((float4*)at)[1] = make_float4(v[4], v[5], v[6], v[7]);
    return;
  }
  words4_t w;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    w[i] = dtype == LQ_BF16 ? pack2<true>(v[2 * i], v[2 * i + 1]) : pack2<false>(v[2 * i], v[2 * i + 1]);
  }
  *(words4_t*)at = w;
}

__device__ __forceinline__ int size_of(int dtype) { return dtype == LQ_F32 ? 4 : 2; }

// A segment of two heads; whether it has to run again, with CAREFUL. ADDS: find_segment's. TERMS: bf16
// values that w x is the sum of.
template <bool ADDS, int TERMS, bool CAREFUL>
__device__ __forceinline__ bool run_segment(const PromptScan& p, const Segment& seg, int pair, int tid,
                                            ChunkLds& lds) {
  const Span& sp = seg.span;
  const int lane = tid & 63, col = lane & 31, hi = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), hw = wave >> 1, half = wave & 1;
  const int h0 = pair * HEADS, h = h0 + hw, g = h0 / p.ratio;
  const int64_t lead = p.spans.starts == nullptr ? sp.index : 0;
  const int from = sp.part * p.segment, to = min(sp.len, from + p.segment);
  // the state: [32-block][i], n = 32 block + 16 (i / 8) + 8 hi + i mod 8 of row pw
  const int pw = 32 * half + sigma(col);
  f32x16_t st[4];
  const int64_t slot_at = (((int64_t)seg.slot * p.H + h) * P + pw) * N + 8 * hi;
#pragma unroll
  for (int b = 0; b < 4; ++b) st[b] = f32x16_t{};
  if (!ADDS && (seg.several || p.initial.data != nullptr)) {
    const int dtype = seg.several ? (int)LQ_F32 : p.initial.dtype;
    const char* at = seg.several ? (const char*)(p.slot_state + slot_at)
                                 : (const char*)p.initial.data +
                                       (sp.index * p.initial.s[0] + h * p.initial.s[1] + pw * p.initial.s[2] + 8 * hi) *
                                           size_of(dtype);
#pragma unroll
    for (int b = 0; b < 4; ++b) {
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        float v[8];
        load8(at + (32 * b + 16 * u) * size_of(dtype), dtype, v);
#pragma unroll
        for (int i = 0; i < 8; ++i) st[b][8 * u + i] = v[i];
      }
    }
  }

  // loads of a chunk: each wave 16 rows of B and of C, and 32 of one head's x
  const int bs = (int)p.B.s[1] * 2, cs = (int)p.C.s[1] * 2, xs = (int)p.x.s[1] * 2;
  const int64_t row0 = sp.begin + from;
  const char* bbase = (const char*)p.B.data + (lead * p.B.s[0] + row0 * p.B.s[1] + g * p.B.s[2]) * 2;
  const char* cbase = (const char*)p.C.data + (lead * p.C.s[0] + row0 * p.C.s[1] + g * p.C.s[2]) * 2;
  const char* xbase = (const char*)p.x.data + (lead * p.x.s[0] + row0 * p.x.s[1] + h * p.x.s[2]) * 2;
  const char* obase = (const char*)p.out.data + (lead * p.out.s[0] + row0 * p.out.s[1] + h * p.out.s[2]) * 2;
  const int os = (int)p.out.s[1] * 2, o_at = col * os + 64 * half + 16 * hi;
  const int rows = to - from, chunks = (rows + Q - 1) / Q;
  auto load_b = [&](int k) {
    const i32x4_t bd = make_desc(bbase + (int64_t)k * Q * bs, (min(Q, rows - k * Q) - 1) * bs + N * 2);
    lds_t to = (lds_t)&lds.b[k & 1][wave * 4096];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int r = wave * 16 + j * 4 + (lane >> 4);
      load_rows_to_lds(bd, to + j * 1024, r * bs + 16 * ((lane & 15) ^ swizzle_b(r)));
    }
  };
  auto load_x = [&](int k) {
    const i32x4_t xd = make_desc(xbase + (int64_t)k * Q * xs, (min(Q, rows - k * Q) - 1) * xs + P * 2);
    lds_t to = (lds_t)&lds.x[hw][half * 4096];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int r = half * 32 + j * 8 + (lane >> 3);
      load_rows_to_lds(xd, to + j * 1024, r * xs + 16 * ((lane & 7) ^ (4 * ((r >> 1) & 1))));
    }
  };
  auto load_rest = [&](int k) {
    const int have = min(Q, rows - k * Q);
    lds_t c_to = (lds_t)&lds.c[wave * 4096];
    const char* steps = (const char*)(p.steps + h * p.rows + lead * p.spans.rows + row0 + k * Q);
    const int64_t array = (int64_t)p.H * p.rows * 4;
    float* const to[4] = {&lds.weight[k & 1][hw][0], (float*)&lds.whole[hw][0], &lds.rest[hw][0], &lds.step[hw][0]};
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const int a = 2 * half + j;
      load_words_to_lds(make_desc(steps + a * array, have * 4), (lds_t)to[a], 4 * lane);
    }
    if (!ADDS) {
      const i32x4_t cd = make_desc(cbase + (int64_t)k * Q * cs, (have - 1) * cs + N * 2);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int r = wave * 16 + j * 4 + (lane >> 4);
        load_rows_to_lds(cd, c_to + j * 1024, r * cs + 16 * ((lane & 15) ^ (r & 15)));
      }
    }
  };

  // D as the sum of two bf16 values, each in both halves of a word
  const float D = p.D.data == nullptr ? 0.f : load_float(p.D.data, p.D.dtype, h * p.D.s[0]);
  const uint32_t D16 = pack2<true>(D, D);
  const float rest = D - __uint_as_float(D16 << 16);
  const uint32_t D16_rest = rest - rest == 0.f ? pack2<true>(rest, rest) : 0;  // (an infinite D has none)
  // operand addresses within the tiles; a product step exchanges chunks (^)
  const int sb = wave >= 2, tb = wave != 0;  // the mixing block of waves 0 to 2
  const int brow = 32 * sb + sigma(col);
  int b_row_at = brow * 256 + 16 * (hi ^ swizzle_b(brow));
  int c_row_at = col * 256 + 16 * (hi ^ (col & 15));
  const int j16 = lane & 15, g1 = (lane >> 4) & 1;
  const int col_chunk = 2 * g1 + (j16 & 1), col_half = 8 * ((j16 >> 1) & 1), tr = 8 * hi + (j16 >> 2);
  int b_col_at0 = tr * 256 + 16 * (col_chunk ^ swizzle_b(tr)) + col_half;
  int b_col_at1 = (tr + 4) * 256 + 16 * (col_chunk ^ swizzle_b(tr + 4)) + col_half;
  const int x_col_at = tr * 128 + 16 * ((4 * half + col_chunk) ^ (4 * (j16 >> 3))) + col_half;
  int m_at = col * 64 + 16 * (hi ^ ((col >> 2) & 3));
  float log_decay = 0.f;
  if (chunks > 0) {
    load_b(0);
    load_x(0);
    load_rest(0);
  }
  for (int k = 0; k < chunks; ++k) {
    const int buf = k & 1;
    // the chunk's loads; the four stores of the last one's y, a whole chunk's, were issued behind them
    if (ADDS || k == 0) wait_loads<0>();
    else wait_loads<4>();
    lds_barrier();
    // hidden from the compiler, which would keep every exchanged form of them in a register of its own
    asm volatile("" : "+v"(b_row_at), "+v"(c_row_at), "+v"(b_col_at0), "+v"(b_col_at1), "+v"(m_at));
    lds_t xt = (lds_t)&lds.x[hw][0], bt = (lds_t)&lds.b[buf][0], ct = (lds_t)&lds.c[0];
    float added = 0.f;
    words4_t xa[4];  // x of rows s = 16 i + 8 hi .. + 7 in column pw
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      lds_t at = xt + x_col_at + i * 16 * 128;
      xa[i] = lds_read_columns(at, at + 4 * 128);
    }
    f32x16_t y[2] = {}, seen[2] = {};
    if (CAREFUL) {
      for (int s = 0; s < Q; ++s) {
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const int q = 32 * half + 16 * (i >> 3) + 8 * hi + (i & 7);
          const float v = bf16_bits_to_float(
              *(const uint16_t*)&lds.x[hw][s * 128 + 16 * ((q >> 3) ^ (4 * ((s >> 1) & 1))) + 2 * (q & 7)]);
          if (v - v == 0.f) continue;
          if (s <= col) seen[0][i] += v;
          if (s <= 32 + col) seen[1][i] += v;
        }
      }
      float gone = 0.f;  // of row pw: to its state as well
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        uint32_t w = xa[i >> 2][i & 3];
        const float a = __uint_as_float(w << 16), b = __uint_as_float(w & 0xffff0000u);
        if (a - a != 0.f) gone += a, w &= 0xffff0000u;
        if (b - b != 0.f) gone += b, w &= 0xffffu;
        xa[i >> 2][i & 3] = w;
      }
      added = gone + __shfl_xor(gone, 32, 64);
    }
    lds_barrier();  // x is in registers: its buffer is free
    if (k + 1 < chunks) {
      load_x(k + 1);
      load_b(k + 1);
    }
    if (!ADDS) {
      f32x16_t mix = {};
      // the next step's operands are read before this one's products (the scheduler, short of registers,
      // would read each right before its product and wait for it)
      words4_t c0 = lds_read16(ct + c_row_at), c1 = lds_read16(ct + c_row_at + 32 * 256);
      words4_t b0 = lds_read16(bt + b_row_at);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        words4_t next_c0, next_c1, next_b0;
        if (i < 7) {
          next_c0 = lds_read16(ct + (c_row_at ^ (32 * (i + 1))));
          next_c1 = lds_read16(ct + (c_row_at ^ (32 * (i + 1))) + 32 * 256);
          next_b0 = lds_read16(bt + (b_row_at ^ (32 * (i + 1))));
        }
        words4_t s16;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          s16[e] = pack2<true>(st[i >> 1][8 * (i & 1) + 2 * e], st[i >> 1][8 * (i & 1) + 2 * e + 1]);
        }
        __builtin_amdgcn_sched_barrier(0);
        mix = mfma<true>(b0, tb ? c1 : c0, mix);  // (the fourth wave's is not used)
        y[0] = mfma<true>(s16, c0, y[0]);
        y[1] = mfma<true>(s16, c1, y[1]);
        __builtin_amdgcn_sched_barrier(0);
        c0 = next_c0, c1 = next_c1, b0 = next_b0;
      }
      if (wave < 3) {
        // mix[8 u + e]: row s = 32 sb + 16 u + 8 hi + e, column t = 32 tb + col. (t is hidden from the
        // compiler, which would keep the comparisons' masks through the loop, more than there are registers.)
        int t = col;
        asm volatile("" : "+v"(t));
#pragma unroll
        for (int j = 0; j < HEADS; ++j) {
          const int at_t = lds.whole[j][32 * tb + col];
          const float rest = lds.rest[j][32 * tb + col];
          words4_t w[2];
#pragma unroll
          for (int u = 0; u < 2; ++u) {
            float v[8];
            const int s0 = 32 * sb + 16 * u + 8 * hi;
            const int4 n0 = *(const int4*)&lds.whole[j][s0], n1 = *(const int4*)&lds.whole[j][s0 + 4];
            const float4 d0 = *(const float4*)&lds.step[j][s0], d1 = *(const float4*)&lds.step[j][s0 + 4];
            const int n[8] = {n0.x, n0.y, n0.z, n0.w, n1.x, n1.y, n1.z, n1.w};
            const float d[8] = {d0.x, d0.y, d0.z, d0.w, d1.x, d1.y, d1.z, d1.w};
#pragma unroll
            for (int e = 0; e < 8; ++e) {
              v[e] = __builtin_amdgcn_ldexpf(mix[8 * u + e] * (d[e] * rest), at_t - n[e]);
            }
            if (sb == tb) {
#pragma unroll
              for (int e = 0; e < 8; ++e) v[e] = 16 * u + 8 * hi + e <= t ? v[e] : 0.f;
            }
#pragma unroll
            for (int e = 0; e < 4; ++e) w[u][e] = pack2<true>(v[2 * e], v[2 * e + 1]);
          }
          lds_t at = (lds_t)&lds.m[j][sb + tb][0];
          *(__attribute__((address_space(3))) words4_t*)(at + m_at) = w[0];
          *(__attribute__((address_space(3))) words4_t*)(at + (m_at ^ 32)) = w[1];
        }
      }
#pragma unroll
      for (int b = 0; b < 2; ++b) {
        y[b] *= __builtin_amdgcn_ldexpf(lds.rest[hw][32 * b + col], lds.whole[hw][32 * b + col]);
        if (CAREFUL) y[b] += seen[b];
      }
    }
    const int last_row = min(Q, rows - k * Q) - 1;
    const int whole = lds.whole[hw][last_row];  // the chunk's decay
    const float rest = lds.rest[hw][last_row];
    lds_barrier();
    if (k + 1 < chunks) load_rest(k + 1);
    if (!ADDS) {
      lds_t mt = (lds_t)&lds.m[hw][0][0];
      int t = col;
      asm volatile("" : "+v"(t));
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        words4_t diagonal, rest;  // D where s = t
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int s = 16 * i + 8 * hi + 2 * e;
          const uint32_t here = t == s ? 0xffffu : t == s + 1 ? 0xffff0000u : 0;
          diagonal[e] = here & D16;
          rest[e] = here & D16_rest;
        }
        y[0] = mfma<true>(xa[i], diagonal, y[0]);
        y[1] = mfma<true>(xa[i + 2], diagonal, y[1]);
        y[0] = mfma<true>(xa[i], rest, y[0]);
        y[1] = mfma<true>(xa[i + 2], rest, y[1]);
        y[0] = mfma<true>(xa[i], lds_read16(mt + (m_at ^ (32 * i))), y[0]);
        y[1] = mfma<true>(xa[i], lds_read16(mt + 2048 + (m_at ^ (32 * i))), y[1]);
        y[1] = mfma<true>(xa[i + 2], lds_read16(mt + 4096 + (m_at ^ (32 * i))), y[1]);
      }
      // (rows past the end are past the descriptor, and not stored)
      const auto od = buffer_of(obase + (int64_t)k * Q * os, (min(Q, rows - k * Q) - 1) * os + P * 2);
      if (p.z.data != nullptr) {
        const char* zbase = (const char*)p.z.data + (lead * p.z.s[0] + (row0 + k * Q) * p.z.s[1] + h * p.z.s[2]) * 2;
        const int zs = (int)p.z.s[1] * 2;
        const auto zd = buffer_of(zbase, (min(Q, rows - k * Q) - 1) * zs + P * 2);
#pragma unroll
        for (int b = 0; b < 2; ++b) {
#pragma unroll
          for (int u = 0; u < 2; ++u) {
            const words4_t z = __builtin_bit_cast(words4_t, __builtin_amdgcn_raw_buffer_load_b128(
                zd, (32 * b + col) * zs + 64 * half + 16 * hi, 32 * u, 0));
#pragma unroll
            for (int e = 0; e < 8; ++e) y[b][8 * u + e] *= scan_silu(word_elem(z[e >> 1], (e & 1) * 16, LQ_BF16));
          }
        }
      }
#pragma unroll
      for (int b = 0; b < 2; ++b) {
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          words4_t w;
#pragma unroll
          for (int e = 0; e < 4; ++e) w[e] = pack2<true>(y[b][8 * u + 2 * e], y[b][8 * u + 2 * e + 1]);
          __builtin_amdgcn_raw_buffer_store_b128(w, od, o_at + 32 * b * os, 32 * u, 0);
        }
      }
    }
    const float keep = __builtin_amdgcn_ldexpf(rest, whole);
    log_decay += (float)whole + __builtin_amdgcn_logf(rest);
    words4_t bc[4];
#pragma unroll
    for (int b = 0; b < 4; ++b) bc[b] = lds_read_columns(bt + (b_col_at0 ^ (64 * b)), bt + (b_col_at1 ^ (64 * b)));
#pragma unroll
    for (int b = 0; b < 4; ++b) {
      st[b] *= keep;
      if (CAREFUL) st[b] += added;
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float4 w0 = *(const float4*)&lds.weight[buf][hw][16 * i + 8 * hi];
      const float4 w1 = *(const float4*)&lds.weight[buf][hw][16 * i + 8 * hi + 4];
      words4_t next[4];
      if (i < 3) {
#pragma unroll
        for (int b = 0; b < 4; ++b) {
          next[b] = lds_read_columns(bt + (b_col_at0 ^ (64 * b)) + (i + 1) * 16 * 256,
                                     bt + (b_col_at1 ^ (64 * b)) + (i + 1) * 16 * 256);
        }
      }
      const float w[8] = {w0.x, w0.y, w0.z, w0.w, w1.x, w1.y, w1.z, w1.w};
      words4_t top, lower, lowest;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float a = w[2 * e] * __uint_as_float(xa[i][e] << 16);
        const float b = w[2 * e + 1] * __uint_as_float(xa[i][e] & 0xffff0000u);
        const uint32_t ab = pack2<true>(a, b);
        top[e] = ab;
        const float a1 = a - __uint_as_float(ab << 16), b1 = b - __uint_as_float(ab & 0xffff0000u);
        const uint32_t ab1 = pack2<true>(a1, b1);
        lower[e] = ab1;
        if (TERMS == 3) lowest[e] = pack2<true>(a1 - __uint_as_float(ab1 << 16), b1 - __uint_as_float(ab1 & 0xffff0000u));
      }
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int b = 0; b < 4; ++b) st[b] = mfma<true>(bc[b], top, st[b]);
#pragma unroll
      for (int b = 0; b < 4; ++b) st[b] = mfma<true>(bc[b], lower, st[b]);
      if (TERMS == 3) {
#pragma unroll
        for (int b = 0; b < 4; ++b) st[b] = mfma<true>(bc[b], lowest, st[b]);
      }
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int b = 0; b < 4; ++b) bc[b] = next[b];
    }
  }

  if (!ADDS && !CAREFUL) {
    // a value that is not finite, wherever it came from, is still in the state
    float odd = 0.f;
#pragma unroll
    for (int i = 0; i < 64; ++i) odd = fmaf(st[i >> 4][i & 15], 0.f, odd);
    if (__syncthreads_or(odd != 0.f)) return true;
  }

  if (!ADDS && (to != sp.len || p.states.data == nullptr)) return false;
  const int dtype = ADDS ? (int)LQ_F32 : p.states.dtype;
  char* at = ADDS ? (char*)(p.slot_state + slot_at + (int64_t)p.H * P * N)
                  : (char*)p.states.data +
                        (sp.index * p.states.s[0] + h * p.states.s[1] + pw * p.states.s[2] + 8 * hi) *
                            size_of(dtype);
#pragma unroll
  for (int b = 0; b < 4; ++b) {
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      float v[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = st[b][8 * u + i];
      store8(at + (32 * b + 16 * u) * size_of(dtype), dtype, v);
    }
  }
  if (ADDS && half == 0 && lane == 0) p.slot_log[(int64_t)(seg.slot + 1) * p.H + h] = log_decay;
  return false;
}

template <bool ADDS, int TERMS>
__global__ __launch_bounds__(256, 2) void scan_chunks_kernel(PromptScan p) {
  __shared__ ChunkLds lds;
  // the workgroups of a group's heads on one XCD (blocks go round the eight), as they read the same B and C
  const int pairs = p.H / HEADS, idx = blockIdx.x % pairs;
  const int pair = pairs % 8 == 0 ? (idx & 7) * (pairs / 8) + (idx >> 3) : idx;
  const Segment seg = find_segment<ADDS>(p, blockIdx.x / pairs);
  if (!seg.valid) return;
  const Span& sp = seg.span;
  if (sp.gap) {
    const int from = sp.part * p.segment, rows = min(sp.len - from, p.segment);
    uint16_t* out = (uint16_t*)p.out.data + (int64_t)(sp.begin + from) * p.out.s[1];
    for (int i = threadIdx.x; i < rows * HEADS * (P / 8); i += 256) {
      const int r = i / (HEADS * P / 8), k = i % (HEADS * P / 8);
      *(words4_t*)(out + r * p.out.s[1] + (pair * HEADS + k / (P / 8)) * p.out.s[2] + k % (P / 8) * 8) =
          words4_t{0, 0, 0, 0};
    }
    return;
  }
  if (!run_segment<ADDS, TERMS, false>(p, seg, pair, threadIdx.x, lds)) return;
  // Again, from values hidden from the compiler: it would keep what the first run made of them in registers
  // for the second one, through the loop.
  Segment again = seg;
  int tid = threadIdx.x, same = pair;
  asm volatile("" : "+s"(again.span.index), "+s"(again.span.begin), "+s"(again.span.part), "+s"(again.slot));
  asm volatile("" : "+v"(tid), "+s"(same));
  run_segment<ADDS, TERMS, true>(p, again, same, tid, lds);
}

// Values in a row, every row 16-byte aligned.
bool rows_fit(const lq_tensor* t) {
  if (t == nullptr) return true;
  const int nd = t->ndim;
  if (t->stride[nd - 1] != 1 || ((uintptr_t)t->data & 15) != 0) return false;
  for (int i = 0; i < nd - 1; ++i) {
    if (t->shape[i] > 1 && t->stride[i] * dtype_size(t->dtype) % 16 != 0) return false;
  }
  return true;
}

}  // namespace

bool prompt_scan_mfma_geometry(int dtype, int64_t heads, int64_t head_dim, int64_t dstate) {
  return dtype == LQ_BF16 && heads % HEADS == 0 && head_dim == P && dstate == N;
}

bool prompt_scan_mfma_fits(const lq_tensor* x, const lq_tensor* B, const lq_tensor* C,
                           const lq_tensor* z, const lq_tensor* initial, const lq_tensor* states,
                           const lq_tensor* out) {
  const int nd = x->ndim;
  const int64_t H = x->shape[nd - 2], G = B->shape[nd - 2];
  if (!prompt_scan_mfma_geometry(x->dtype, H, x->shape[nd - 1], B->shape[nd - 1])) return false;
  if (H / G % HEADS != 0 || out->dtype != LQ_BF16 || (z != nullptr && z->dtype != LQ_BF16)) return false;
  const lq_tensor* ts[7] = {x, B, C, z, initial, states, out};
  for (const lq_tensor* t : ts) {
    if (!rows_fit(t)) return false;
  }
  const lq_tensor* by_chunk[5] = {x, B, C, z, out};
  for (const lq_tensor* t : by_chunk) {
    if (t == nullptr) continue;
    // (a single row's too: the rows past it have to be past the descriptors)
    const int64_t s = t->stride[nd - 3];
    if (s < t->shape[nd - 1] || s > (1 << 22)) return false;
  }
  return true;
}

size_t prompt_scan_mfma_workspace(int64_t rows, int64_t heads) { return (size_t)(rows * heads) * 16; }

void launch_prompt_scan_steps(const PromptScan& p, int64_t chunks, hipStream_t st) {
  const int64_t blocks = (p.H + STEP_HEADS - 1) / STEP_HEADS;
  hipLaunchKernelGGL(scan_steps_kernel, dim3((unsigned)(chunks * blocks)), dim3(256), 0, st, p);
}

void launch_prompt_scan_mfma(const PromptScan& p, bool adds, int64_t parts, hipStream_t st) {
  const dim3 grid((unsigned)(parts * (p.H / HEADS))), block(256);
  const bool three = p.states.data != nullptr && p.states.dtype == LQ_F32;
  if (adds && three) hipLaunchKernelGGL((scan_chunks_kernel<true, 3>), grid, block, 0, st, p);
  else if (adds) hipLaunchKernelGGL((scan_chunks_kernel<true, 2>), grid, block, 0, st, p);
  else if (three) hipLaunchKernelGGL((scan_chunks_kernel<false, 3>), grid, block, 0, st, p);
  else hipLaunchKernelGGL((scan_chunks_kernel<false, 2>), grid, block, 0, st, p);
}

}  // namespace lq
