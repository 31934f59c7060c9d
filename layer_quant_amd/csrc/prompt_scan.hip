// The Mamba2 recurrence over whole prompts, packed one behind another or a batch of equal lengths (the
// single token's form is lq_selective_state_update; no reference counterpart: its remote module runs
// prompts, hybrid_quant/mamba_state_8b_kernel.py only decode steps):
//
//   S_t = exp(A dt_t) S_{t-1} + dt_t x_t B_t^T      [P, N] per head
//   y_t = S_t C_t + D x_t,  y_t *= silu(z_t)
//
// A prompt's rows fall into segments. Where a prompt has more than one, so that a few long prompts fill
// the GPU too, a first launch finds what each segment but the last adds to the state by itself, a second
// one carries the states from segment to segment, and the last launch runs every segment from the state in
// front of it. (The first segment's is a copy, as the given states may be the tensor that the last segment
// writes.) A prompt of one segment takes the last launch alone. The segment's length follows from the sizes
// (plan_segment).
//
// scan_rows_kernel walks the rows one by one with the state in registers, fp32 throughout: the kernel of
// fp32 and fp16 inputs and of every geometry that the matrix kernel does not take. A thread holds 4 p x
// (N / 16) n of the state: per row it reads N / 8 + 4 values from LDS, and four sums over 16 lanes give y.
// Blocks of 16 rows are staged in LDS, loaded a block ahead. Within a block, with c the running sum of A dt
// log2(e) and e its end, the state is held as 2^(e - c) S, so that
//   2^(e - c_t) S_t = 2^(e - c_t-1) S_t-1 + 2^(e - c_t) dt_t x_t B_t^T,   y_t = 2^(c_t - e) (2^(e - c_t) S_t) C_t
// takes two multiply-adds per value of the state instead of three, and one where y is not wanted. Only values
// that are smaller than they would be stand in registers, by 2^-40 at most: blocks that decay further, or
// grow, or have a NaN, take the steps as they are. c is summed in 64 bits, for the reason that
// prompt_scan_mfma.hip gives.
// Three fp32 prompts up to 1001 rows (2438 in all) of 128 heads x 64 x 128: 350-372 us (101-113 for what
// the segments add, 33 to carry, 234-268 for the segments, where 85 VALU instructions per row and wave, 64 of them
// these multiply-adds, are 173 at 2.4 GHz; the rest is the blocks' staging, barriers and silu, and latency at
// four waves per SIMD). With a state not scaled, loads at addresses of their own and less of the GPU's
// workgroups it was 548. Without effect or worse: z loaded ahead (350), two rows unrolled (358), five
// workgroups per CU (350, and 620 with spills), all loads of a segment's first state at once (401 against
// 393, with spills).
#include "matrix16.h"
#include "prompt_scan.h"

namespace lq {
namespace {

constexpr int TB = 16;       // rows per staged block
constexpr int PB = 64;       // p of a workgroup (16 per wave)
constexpr float LOG2E = 1.44269504088896340736f;
constexpr double MAX_SCALE = 40;  // a scaled state's, in powers of two

template <int NPL>
struct alignas(16) RowTile {
  float x[TB][PB];
  float y[TB][PB];
  float b[TB][16 * NPL];
  float c[TB][16 * NPL];
  // of 64 rows, four blocks
  float dt[64], decay[64];                // scaled: dt_s 2^(e - c_s), 2^(c_s - e); else dt_s, A dt_s log2(e)
  float keep[64 / TB], log_decay[64 / TB];  // 2^e, e
  int scaled[64 / TB];
};

// v + the value CTRL's shift away within 16 lanes (0 from outside them).
template <int CTRL>
__device__ __forceinline__ double plus_shifted(double v) {
  const uint64_t u = __builtin_bit_cast(uint64_t, v);
  const uint32_t lo = __builtin_amdgcn_update_dpp(0, (uint32_t)u, CTRL, 0xf, 0xf, false);
  const uint32_t hi = __builtin_amdgcn_update_dpp(0, (uint32_t)(u >> 32), CTRL, 0xf, 0xf, false);
  return v + __builtin_bit_cast(double, ((uint64_t)hi << 32) | lo);
}

__device__ __forceinline__ float exp2_of(double v) {
  const double whole = __builtin_rint(v);
  return __builtin_amdgcn_ldexpf(__builtin_amdgcn_exp2f((float)(v - whole)), (int)whole);
}

// v's sum over 16 lanes; lane (bit 3, bit 2) of each 16 ends with that of v[2 bit3 + bit2].
__device__ __forceinline__ float sums_of_four(const float (&v)[4], int lane) {
  const bool b3 = lane & 8, b2 = lane & 4;
  float a0 = b3 ? v[2] : v[0], a1 = b3 ? v[3] : v[1];
  const float s0 = b3 ? v[0] : v[2], s1 = b3 ? v[1] : v[3];
  // row_mirror: lane i of a row of 16 reads lane 15 - i
  a0 += __uint_as_float(__builtin_amdgcn_mov_dpp(__float_as_uint(s0), 0x140, 0xf, 0xf, true));
  a1 += __uint_as_float(__builtin_amdgcn_mov_dpp(__float_as_uint(s1), 0x140, 0xf, 0xf, true));
  float r = b2 ? a1 : a0;
  const float s = b2 ? a0 : a1;
  // row_half_mirror: lane i of 8 reads lane 7 - i; then the four lanes of a quad
  r += __uint_as_float(__builtin_amdgcn_mov_dpp(__float_as_uint(s), 0x141, 0xf, 0xf, true));
  r += __uint_as_float(__builtin_amdgcn_mov_dpp(__float_as_uint(r), 0x4e, 0xf, 0xf, true));
  r += __uint_as_float(__builtin_amdgcn_mov_dpp(__float_as_uint(r), 0xb1, 0xf, 0xf, true));
  return r;
}

// Four values in a row as they lie in memory (8 bytes of 16-bit ones in x and y).
template <int SIZE>
__device__ __forceinline__ uint4 load_raw4(const void* base, int64_t at) {
  if (SIZE == 4) return *(const uint4*)((const char*)base + at * 4);
  const uint2 w = *(const uint2*)((const char*)base + at * 2);
  return make_uint4(w.x, w.y, 0, 0);
}
template <int SIZE>
__device__ __forceinline__ uint4 buffer_load4(__amdgpu_buffer_rsrc_t rows, uint32_t offset) {
  if (SIZE == 4) return __builtin_bit_cast(uint4, __builtin_amdgcn_raw_buffer_load_b128(rows, offset, 0, 0));
  const uint2 w = __builtin_bit_cast(uint2, __builtin_amdgcn_raw_buffer_load_b64(rows, offset, 0, 0));
  return make_uint4(w.x, w.y, 0, 0);
}
template <int SIZE>
__device__ __forceinline__ float4 values_of(uint4 w, int dtype) {
  if (SIZE == 4) return make_float4(__uint_as_float(w.x), __uint_as_float(w.y), __uint_as_float(w.z), __uint_as_float(w.w));
  return make_float4(word_elem(w.x, 0, dtype), word_elem(w.x, 16, dtype), word_elem(w.y, 0, dtype),
                     word_elem(w.y, 16, dtype));
}
template <int SIZE>
__device__ __forceinline__ void store4(void* base, int dtype, int64_t at, float4 v) {
  if (SIZE == 4) {
    *(float4*)((char*)base + at * 4) = v;
    return;
  }
  uint2 w;
  if (dtype == LQ_BF16) {
    w.x = float_to_bf16_bits(v.x) | ((uint32_t)float_to_bf16_bits(v.y) << 16);
    w.y = float_to_bf16_bits(v.z) | ((uint32_t)float_to_bf16_bits(v.w) << 16);
  } else {
    w.x = __builtin_bit_cast(uint16_t, (_Float16)v.x) | ((uint32_t)__builtin_bit_cast(uint16_t, (_Float16)v.y) << 16);
    w.y = __builtin_bit_cast(uint16_t, (_Float16)v.z) | ((uint32_t)__builtin_bit_cast(uint16_t, (_Float16)v.w) << 16);
  }
  *(uint2*)((char*)base + at * 2) = w;
}

// ADDS: find_segment's. SIZE: bytes of a value of x, B, C, z and out where four in a row are loaded at once,
// a block of rows ahead, by WAVES waves; 0: any layout.
template <int NPL, bool ADDS, int SIZE, int WAVES>
__global__ __launch_bounds__(64 * WAVES, WAVES == 4 && NPL <= 8 ? 4 : 1) void scan_rows_kernel(PromptScan p) {
  __shared__ RowTile<NPL> tile;
  const int h = blockIdx.x % p.H;
  const Segment seg = find_segment<ADDS>(p, blockIdx.x / p.H);
  if (!seg.valid) return;
  const Span& sp = seg.span;
  const int tid = threadIdx.x, lane = tid & 63, nl = lane & 15;
  const int pb = blockIdx.y * PB, width = min(PB, p.P - pb);
  const int p0 = (tid >> 6) * 16 + (lane >> 4) * 4;  // of the thread's 4 p
  const int64_t lead = p.spans.starts == nullptr ? sp.index : 0;
  const int from = sp.part * p.segment, to = min(sp.len, from + p.segment);
  const int64_t row0 = sp.begin;
  const int64_t out_at = lead * p.out.s[0] + h * p.out.s[2] + pb * p.out.s[3];
  if (sp.gap) {
    for (int i = tid; i < (to - from) * width; i += blockDim.x) {
      store_float(p.out.data, p.out.dtype,
                  out_at + (row0 + from + i / width) * p.out.s[1] + (i % width) * p.out.s[3], 0.f);
    }
    return;
  }
  float st[4][NPL];
  const int64_t slot_at = (((int64_t)seg.slot * p.H + h) * p.P + pb + p0) * p.N;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
#pragma unroll
    for (int j = 0; j < NPL; ++j) {
      const int n = 64 * (j >> 2) + 4 * nl + (j & 3);
      float v = 0.f;
      if (!ADDS && p0 + i < width && n < p.N) {
        if (seg.several) {
          v = p.slot_state[slot_at + (int64_t)i * p.N + n];
        } else if (p.initial.data != nullptr) {
          v = load_float(p.initial.data, p.initial.dtype,
                         sp.index * p.initial.s[0] + h * p.initial.s[1] +
                             (pb + p0 + i) * p.initial.s[2] + n * p.initial.s[3]);
        }
      }
      st[i][j] = v;
    }
  }
  const float A_h = load_float(p.A.data, p.A.dtype, h * p.A.s[0]), A = A_h * LOG2E;
  const double A64 = (double)A_h * 1.4426950408889634;
  const float bias = p.bias.data == nullptr ? 0.f : load_float(p.bias.data, p.bias.dtype, h * p.bias.s[0]);
  const float D = p.D.data == nullptr ? 0.f : load_float(p.D.data, p.D.dtype, h * p.D.s[0]);
  const int g = h / p.ratio;
  const int64_t x_at = lead * p.x.s[0] + h * p.x.s[2] + pb * p.x.s[3];
  const int64_t z_at = lead * p.z.s[0] + h * p.z.s[2] + pb * p.z.s[3];
  const int64_t b_at = lead * p.B.s[0] + g * p.B.s[2], c_at = lead * p.C.s[0] + g * p.C.s[2];
  const int64_t dt_at = lead * p.dt.s[0] + h * p.dt.s[2];
  float log_decay = 0.f;
  // A block of x, B and C in chunks of four values: a thread has one chunk of x, and of B and of C those in
  // its column (BR rows apart). Rows past the segment are past the descriptors and read as zero, columns
  // past the row's values are sent there.
  constexpr int XC = 4 * WAVES, BC = 4 * NPL, BR = 64 * WAVES / BC, BL = SIZE == 0 ? 0 : TB / BR;
  static_assert(TB * XC == 64 * WAVES && (SIZE == 0 || BR * BL == TB), "every thread loads as many");
  constexpr uint32_t OUTSIDE = 0x7fffff00;
  const int xr = tid / XC, xc = 4 * (tid % XC), br = tid / BC, bc = 4 * (tid % BC);
  const int xs = (int)p.x.s[1] * SIZE, bs = (int)p.B.s[1] * SIZE, cs = (int)p.C.s[1] * SIZE;
  const uint32_t x_off = xc < width ? xr * xs + xc * SIZE : OUTSIDE;
  const uint32_t b_off = bc < p.N ? br * bs + bc * SIZE : OUTSIDE, c_off = bc < p.N ? br * cs + bc * SIZE : OUTSIDE;
  uint4 raw_x, raw_b[BL + 1], raw_c[BL + 1];
  auto load_block = [&](int t) {
    if (SIZE == 0) return;
    const int last = min(TB, to - t) - 1;
    const int64_t row = row0 + t;
    const auto xd = buffer_of((const char*)p.x.data + (x_at + row * p.x.s[1]) * SIZE, last < 0 ? 0 : last * xs + width * SIZE);
    const auto bd = buffer_of((const char*)p.B.data + (b_at + row * p.B.s[1]) * SIZE, last < 0 ? 0 : last * bs + p.N * SIZE);
    const auto cd = buffer_of((const char*)p.C.data + (c_at + row * p.C.s[1]) * SIZE, last < 0 ? 0 : last * cs + p.N * SIZE);
    raw_x = buffer_load4<SIZE>(xd, x_off);
#pragma unroll
    for (int j = 0; j < BL; ++j) {
      raw_b[j] = buffer_load4<SIZE>(bd, b_off + j * BR * bs);
      if (!ADDS) raw_c[j] = buffer_load4<SIZE>(cd, c_off + j * BR * cs);
    }
  };
  load_block(from);
  for (int t = from; t < to; t += TB) {
    const int rows = min(TB, to - t);
    const int64_t row = row0 + t;
    __syncthreads();
    if (SIZE != 0) {
      *(float4*)&tile.x[xr][xc] = values_of<SIZE == 0 ? 4 : SIZE>(raw_x, p.x.dtype);
#pragma unroll
      for (int j = 0; j < BL; ++j) {
        *(float4*)&tile.b[br + j * BR][bc] = values_of<SIZE == 0 ? 4 : SIZE>(raw_b[j], p.x.dtype);
        if (!ADDS) *(float4*)&tile.c[br + j * BR][bc] = values_of<SIZE == 0 ? 4 : SIZE>(raw_c[j], p.x.dtype);
      }
      load_block(t + TB);
    } else {
      for (int i = tid; i < rows * PB; i += blockDim.x) {
        const int r = i / PB, c = i % PB;
        tile.x[r][c] = c < width ? load_float(p.x.data, p.x.dtype, x_at + (row + r) * p.x.s[1] + c * p.x.s[3]) : 0.f;
      }
      for (int i = tid; i < rows * 16 * NPL; i += blockDim.x) {
        const int r = i / (16 * NPL), n = i % (16 * NPL);
        float b = 0.f, c = 0.f;
        if (n < p.N) {
          b = load_float(p.B.data, p.B.dtype, b_at + (row + r) * p.B.s[1] + n * p.B.s[3]);
          c = load_float(p.C.data, p.C.dtype, c_at + (row + r) * p.C.s[1] + n * p.C.s[3]);
        }
        tile.b[r][n] = b;
        tile.c[r][n] = c;
      }
    }
    const int block = (t - from) / TB % (64 / TB);
    if (block == 0 && tid < 64) {
      const bool in = t + tid < to;
      float dt = 0.f;
      if (in) dt = scan_step(p, load_float(p.dt.data, p.dt.dtype, dt_at + (row + tid) * p.dt.s[1]), bias);
      const float lg = in ? A * dt : 0.f;
      double c = in ? A64 * dt : 0.0;
      c = plus_shifted<0x111>(c);  // row_shr 1, 2, 4, 8
      c = plus_shifted<0x112>(c);
      c = plus_shifted<0x114>(c);
      c = plus_shifted<0x118>(c);
      const double e = __shfl(c, lane | (TB - 1), 64);
      const uint64_t falls = __ballot(lg <= 0.f) >> (lane & ~(TB - 1));
      const bool scaled = (falls & 0xffff) == 0xffff && e >= -MAX_SCALE;
      tile.dt[tid] = scaled ? dt * exp2_of(e - c) : dt;
      tile.decay[tid] = scaled ? exp2_of(c - e) : lg;
      if ((tid & (TB - 1)) == 0) {
        tile.scaled[tid / TB] = scaled;
        tile.keep[tid / TB] = scaled ? exp2_of(e) : 1.f;
        tile.log_decay[tid / TB] = (float)e;
      }
    }
    __syncthreads();
    log_decay += tile.log_decay[block];
    const bool scaled = tile.scaled[block];
    const float *dts = &tile.dt[block * TB], *decays = &tile.decay[block * TB];
    if (scaled) {
      const float keep = tile.keep[block];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
#pragma unroll
        for (int j = 0; j < NPL; ++j) st[i][j] *= keep;
      }
#pragma unroll 1
      for (int r = 0; r < rows; ++r) {
        const float dt = dts[r];
        const float4 x4 = *(const float4*)&tile.x[r][p0];
        const float dx[4] = {dt * x4.x, dt * x4.y, dt * x4.z, dt * x4.w};
        float y[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int j = 0; j < NPL; j += 4) {
          const float4 b4 = *(const float4*)&tile.b[r][16 * j + 4 * nl];
          float4 c4 = b4;
          if (!ADDS) c4 = *(const float4*)&tile.c[r][16 * j + 4 * nl];
          const float b[4] = {b4.x, b4.y, b4.z, b4.w}, c[4] = {c4.x, c4.y, c4.z, c4.w};
#pragma unroll
          for (int i = 0; i < 4; ++i) {
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              st[i][j + k] = fmaf(dx[i], b[k], st[i][j + k]);
              if (!ADDS) y[i] = fmaf(st[i][j + k], c[k], y[i]);
            }
          }
        }
        if (!ADDS) {
          const float sum = sums_of_four(y, lane) * decays[r];
          if ((lane & 3) == 0) tile.y[r][p0 + ((lane >> 2) & 3)] = sum;
        }
      }
    }
#pragma unroll 1
    for (int r = scaled ? rows : 0; r < rows; ++r) {
      const float a = __builtin_amdgcn_exp2f(decays[r]), dt = dts[r];
      const float4 x4 = *(const float4*)&tile.x[r][p0];
      const float dx[4] = {dt * x4.x, dt * x4.y, dt * x4.z, dt * x4.w};
      float y[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int j = 0; j < NPL; j += 4) {
        const float4 b4 = *(const float4*)&tile.b[r][16 * j + 4 * nl];
        float4 c4 = b4;
        if (!ADDS) c4 = *(const float4*)&tile.c[r][16 * j + 4 * nl];
        const float b[4] = {b4.x, b4.y, b4.z, b4.w}, c[4] = {c4.x, c4.y, c4.z, c4.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            st[i][j + e] = fmaf(st[i][j + e], a, dx[i] * b[e]);
            if (!ADDS) y[i] = fmaf(st[i][j + e], c[e], y[i]);
          }
        }
      }
      if (!ADDS) {
        const float sum = sums_of_four(y, lane);
        if ((lane & 3) == 0) tile.y[r][p0 + ((lane >> 2) & 3)] = sum;
      }
    }
    if (!ADDS) {
      __syncthreads();
      for (int i = tid; i < (SIZE == 0 ? 0 : rows * XC); i += 64 * WAVES) {
        const int r = i / XC, c = 4 * (i % XC);
        if (c >= width) continue;
        const float4 x4 = *(const float4*)&tile.x[r][c];
        float4 y4 = *(const float4*)&tile.y[r][c];
        y4 = make_float4(fmaf(D, x4.x, y4.x), fmaf(D, x4.y, y4.y), fmaf(D, x4.z, y4.z), fmaf(D, x4.w, y4.w));
        if (p.z.data != nullptr) {
          const float4 z4 = values_of<SIZE == 0 ? 4 : SIZE>(
              load_raw4<SIZE == 0 ? 4 : SIZE>(p.z.data, z_at + (row + r) * p.z.s[1] + c), p.x.dtype);
          y4.x *= scan_silu(z4.x);
          y4.y *= scan_silu(z4.y);
          y4.z *= scan_silu(z4.z);
          y4.w *= scan_silu(z4.w);
        }
        store4<SIZE == 0 ? 4 : SIZE>(p.out.data, p.x.dtype, out_at + (row + r) * p.out.s[1] + c, y4);
      }
      for (int i = tid; i < (SIZE == 0 ? rows * PB : 0); i += blockDim.x) {
        const int r = i / PB, c = i % PB;
        if (c >= width) continue;
        float y = fmaf(D, tile.x[r][c], tile.y[r][c]);
        if (p.z.data != nullptr) {
          y *= scan_silu(load_float(p.z.data, p.z.dtype, z_at + (row + r) * p.z.s[1] + c * p.z.s[3]));
        }
        store_float(p.out.data, p.out.dtype, out_at + (row + r) * p.out.s[1] + c * p.out.s[3], y);
      }
    }
  }
  if (ADDS) {
    const int64_t next_at = slot_at + (int64_t)p.H * p.P * p.N;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
#pragma unroll
      for (int j = 0; j < NPL; ++j) {
        const int n = 64 * (j >> 2) + 4 * nl + (j & 3);
        if (p0 + i < width && n < p.N) p.slot_state[next_at + (int64_t)i * p.N + n] = st[i][j];
      }
    }
    if (tid == 0 && blockIdx.y == 0) p.slot_log[(int64_t)(seg.slot + 1) * p.H + h] = log_decay;
  } else if (to == sp.len && p.states.data != nullptr) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
#pragma unroll
      for (int j = 0; j < NPL; ++j) {
        const int n = 64 * (j >> 2) + 4 * nl + (j & 3);
        if (p0 + i < width && n < p.N) {
          store_float(p.states.data, p.states.dtype,
                      sp.index * p.states.s[0] + h * p.states.s[1] + (pb + p0 + i) * p.states.s[2] +
                          n * p.states.s[3],
                      st[i][j]);
        }
      }
    }
  }
}

constexpr int AHEAD = 8;

// The states in front of a prompt's segments from what the segments in front of them add, in place.
// blockIdx.y: slot; a prompt's first one carries all of its own. Four consecutive values per thread.
__global__ __launch_bounds__(256) void scan_carry_kernel(PromptScan p) {
  Span sp;
  const bool mine = find_span<false>(
      p.spans, blockIdx.y, [&](int len, bool) { return slots_of_prompt(p, len); },
      [&](int begin, int i) { return slot_of(p, begin, i); }, sp);
  if (!mine || sp.part != 0) return;
  const int many = min(slots_of_prompt(p, sp.len), p.slots - (int)blockIdx.y);
  const int64_t size = (int64_t)p.H * p.P * p.N, i = ((int64_t)blockIdx.x * 256 + threadIdx.x) * 4;
  if (i >= size) return;
  float* state = p.slot_state + (int64_t)blockIdx.y * size + i;
  const int have = (int)min((int64_t)4, size - i);
  float held[4];
  int head[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const int64_t at = i + min(e, have - 1);
    const int n = (int)(at % p.N), pp = (int)(at / p.N % p.P);
    head[e] = (int)(at / ((int64_t)p.P * p.N));
    held[e] = 0.f;
    if (p.initial.data != nullptr) {
      held[e] = load_float(p.initial.data, p.initial.dtype,
                           sp.index * p.initial.s[0] + head[e] * p.initial.s[1] + pp * p.initial.s[2] +
                               n * p.initial.s[3]);
    }
  }
  if (size % 4 == 0 && p.P * p.N % 4 == 0) {
    const float* lg = p.slot_log + (int64_t)blockIdx.y * p.H + head[0];
    float4 h4 = make_float4(held[0], held[1], held[2], held[3]);
    *(float4*)state = h4;
    // eight loads go out before the first is needed
    for (int j = 1; j < many; j += AHEAD) {
      float4 add[AHEAD];
      float keep[AHEAD];
#pragma unroll
      for (int e = 0; e < AHEAD; ++e) {
        const int k = min(j + e, many - 1);
        add[e] = *(const float4*)(state + k * size);
        keep[e] = lg[(int64_t)k * p.H];
      }
#pragma unroll
      for (int e = 0; e < AHEAD; ++e) {
        if (j + e >= many) break;
        const float a = __builtin_amdgcn_exp2f(keep[e]);
        h4.x = fmaf(h4.x, a, add[e].x);
        h4.y = fmaf(h4.y, a, add[e].y);
        h4.z = fmaf(h4.z, a, add[e].z);
        h4.w = fmaf(h4.w, a, add[e].w);
        *(float4*)(state + (j + e) * size) = h4;
      }
    }
    return;
  }
  for (int e = 0; e < have; ++e) {
    float v = held[e];
    state[e] = v;
    for (int j = 1; j < many; ++j) {
      v = fmaf(v, __builtin_amdgcn_exp2f(p.slot_log[((int64_t)blockIdx.y + j) * p.H + head[e]]),
               state[j * size + e]);
      state[j * size + e] = v;
    }
  }
}

// Rows of a segment, a multiple of 64. Segments cost a part of the work again and two launches.
// Matrix kernel: as many as give two workgroups per CU (a workgroup has two heads), but at least 256 rows, and
// prompts of up to 1024 rows, as far as their mean says, stay whole (4 prompts of 512 rows and 128 heads: 71 us
// in two segments each, 41 whole; one of 2000 rows: 107 us in two of 1024, 73 in eight of 256, and 108 again with a
// prompt of 40 rows beside it, as the lengths are not known here). Eight prompts or more fill the GPU by themselves:
// twice as many rows then (24 prompts up to 700 rows: 134 -> 117 us).
// Rows kernel: as many as give eight workgroups per CU, of which it has four at a time (half as many
// workgroups: three fp32 prompts up to 1001 rows 429 us against 394, one of 4000 fp16 rows 757 against 652);
// at least 192 rows, or 256 where prompts have no more, as their mean says (4 of 200 rows, 64 heads: 137 us in two
// segments each, 84 whole, 89 in four), or 64 where the heads give few workgroups (8000 rows of 8 heads: 145 us
// with 192, 75 with 64) and for few prompts whose segments of 64 rows the GPU takes at once, or nearly, and
// that either leave CUs without work or have more than 256 rows (128 heads: one of 200 fp32 rows 83 -> 61, of
// 500 fp16 rows 154 -> 102, two of 300 fp32 rows 132 -> 109; one of 128 rows stays whole, 56 against 59).
int64_t plan_segment(bool matrix, int64_t prompts, int64_t rows, int64_t heads) {
  const int64_t many = (matrix ? 4 : 8) * device_cus(), want = (rows * heads + many - 1) / many;
  if (!matrix) {
    const bool few = rows > 128 * prompts && rows * heads <= (int64_t)64 * 5 * device_cus() &&
                     (prompts * heads < device_cus() || rows > 256 * prompts);
    const int64_t least = heads < 64 || few ? 64 : rows <= 256 * prompts ? 256 : 192;
    return max((want + 63) / 64 * 64, least);
  }
  const int64_t seg = (prompts >= 8 ? 2 * want : want) + 63;
  return max(seg / 64 * 64, rows <= 1024 * prompts ? (int64_t)1024 : (int64_t)256);
}

// Whether slot_of goes by the rows alone, as fewer slots are needed then.
bool slots_by_rows(int64_t prompts, int64_t rows, int64_t segment) {
  return 2 * rows / segment < rows / segment + prompts;
}

// Slots, at most: a prompt has a segment more than its rows fill, or, as one of several segments has more
// rows than one of them, less than two for each segment's rows.
int64_t slots_of(int64_t prompts, int64_t rows, int64_t segment, bool packed) {
  const int64_t n = (rows + segment - 1) / segment;
  if (n < 2) return 0;
  return packed ? min(rows / segment + prompts, 2 * rows / segment) : prompts * n;
}

size_t align256(size_t n) { return (n + 255) & ~(size_t)255; }

template <bool ADDS, int SIZE, int WAVES>
void launch_rows_of(const PromptScan& p, dim3 grid, hipStream_t st) {
  const dim3 block(SIZE == 0 ? 64 * min(4, (p.P + 15) / 16) : 64 * WAVES);
  if (p.N <= 64) hipLaunchKernelGGL((scan_rows_kernel<4, ADDS, SIZE, WAVES>), grid, block, 0, st, p);
  else if (p.N <= 128) hipLaunchKernelGGL((scan_rows_kernel<8, ADDS, SIZE, WAVES>), grid, block, 0, st, p);
  else if constexpr (SIZE == 0) hipLaunchKernelGGL((scan_rows_kernel<16, ADDS, 0, 4>), grid, block, 0, st, p);
}

// size: bytes of a value where all rows can be loaded four values at a time and N <= 128, else 0
template <bool ADDS>
void launch_rows(const PromptScan& p, int size, dim3 grid, hipStream_t st) {
  if (size == 4 && p.P <= 16) launch_rows_of<ADDS, 4, 1>(p, grid, st);
  else if (size == 4) launch_rows_of<ADDS, 4, 4>(p, grid, st);
  else if (size == 2 && p.P <= 16) launch_rows_of<ADDS, 2, 1>(p, grid, st);
  else if (size == 2) launch_rows_of<ADDS, 2, 4>(p, grid, st);
  else launch_rows_of<ADDS, 0, 4>(p, grid, st);
}

// Values of x's type, four in a row at addresses that are multiples of their bytes.
bool in_fours(const lq_tensor* t, int dtype) {
  if (t == nullptr) return true;
  const int nd = t->ndim, size = dtype_size(dtype);
  if (t->dtype != dtype || t->stride[nd - 1] != 1 || t->shape[nd - 1] % 4 != 0) return false;
  if (((uintptr_t)t->data & (4 * size - 1)) != 0) return false;
  for (int i = 0; i < nd - 1; ++i) {
    if (t->shape[i] > 1 && t->stride[i] % 4 != 0) return false;
  }
  // a block's rows within 31 bits of bytes (a single row's too: the rows past it have to be past the end)
  const int64_t s = t->stride[nd - 3];
  return s >= t->shape[nd - 1] && s <= (1 << 22);
}

// Sizes that a call takes, the launch limits aside (no product leaves 64 bits).
bool sizes_fit(int64_t prompts, int64_t rows, bool packed, int64_t heads, int64_t head_dim, int64_t dstate) {
  constexpr int64_t MOST = INT32_MAX / 2;
  return prompts <= 65535 && rows <= MOST && (packed || prompts * rows <= MOST) && dstate <= PROMPT_SCAN_MAX_N &&
         head_dim <= 65535 && heads <= MOST && heads * head_dim <= MOST && heads * head_dim * dstate <= MOST;
}

}  // namespace
}  // namespace lq

using namespace lq;

extern "C" size_t lq_prompt_scan_workspace(int dtype, int64_t prompts, int64_t rows, int packed,
                                           int64_t heads, int64_t head_dim, int64_t dstate) {
  if (prompts <= 0 || rows <= 0 || heads <= 0 || head_dim <= 0 || dstate <= 0) return 0;
  if (!sizes_fit(prompts, rows, packed != 0, heads, head_dim, dstate)) return 0;
  const int64_t total = packed ? rows : prompts * rows;
  const bool mfma = prompt_scan_mfma_geometry(dtype, heads, head_dim, dstate);
  const int64_t slots = slots_of(prompts, rows, plan_segment(mfma, prompts, total, heads), packed != 0);
  return align256((size_t)(slots * heads * head_dim * dstate) * 4) + align256((size_t)(slots * heads) * 4) +
         (mfma ? prompt_scan_mfma_workspace(total, heads) : 0);
}

extern "C" int lq_prompt_scan(const lq_tensor* x, const lq_tensor* dt, const lq_tensor* A,
                              const lq_tensor* B, const lq_tensor* C, const lq_tensor* starts,
                              const lq_tensor* D, const lq_tensor* z, const lq_tensor* dt_bias,
                              const lq_tensor* initial, const lq_tensor* states,
                              const lq_tensor* out, int dt_softplus, float dt_min, float dt_max,
                              void* workspace, size_t workspace_bytes, void* stream) {
  int rc;
  const int nd = starts != nullptr ? 3 : 4;
  if ((rc = check_tensor_or_empty(x, "x", nd, true)) != LQ_OK) return rc;
  if ((rc = check_tensor_or_empty(dt, "dt", nd - 1, true)) != LQ_OK) return rc;
  if ((rc = check_tensor_or_empty(B, "B", nd, true, x->dtype)) != LQ_OK) return rc;
  if ((rc = check_tensor_or_empty(C, "C", nd, true, x->dtype)) != LQ_OK) return rc;
  if (z != nullptr && (rc = check_tensor_or_empty(z, "z", nd, true)) != LQ_OK) return rc;
  if ((rc = check_tensor_or_empty(out, "out", nd, true)) != LQ_OK) return rc;
  if ((rc = check_tensor(A, "A", 1, true)) != LQ_OK) return rc;
  if (D != nullptr && (rc = check_tensor(D, "D", 1, true)) != LQ_OK) return rc;
  if (dt_bias != nullptr && (rc = check_tensor(dt_bias, "dt_bias", 1, true)) != LQ_OK) return rc;
  if (initial != nullptr && (rc = check_tensor_or_empty(initial, "initial_states", 4, true)) != LQ_OK) return rc;
  if (states != nullptr && (rc = check_tensor_or_empty(states, "states", 4, true)) != LQ_OK) return rc;
  const int64_t batch = nd == 4 ? x->shape[0] : 1, rows = x->shape[nd - 3];
  const int64_t H = x->shape[nd - 2], P = x->shape[nd - 1], G = B->shape[nd - 2], N = B->shape[nd - 1];
  for (int i = 0; i < nd; ++i) {
    if (out->shape[i] != x->shape[i] || (z != nullptr && z->shape[i] != x->shape[i])) {
      return fail(LQ_ERR_INVALID_ARG, "out and z must have x's shape");
    }
    if (C->shape[i] != B->shape[i]) return fail(LQ_ERR_INVALID_ARG, "C must have B's shape");
    if (i < nd - 2 && B->shape[i] != x->shape[i]) return fail(LQ_ERR_INVALID_ARG, "B must have x's rows");
    if (i < nd - 1 && dt->shape[i] != x->shape[i]) {
      return fail(LQ_ERR_INVALID_ARG, "dt must have x's rows and heads");
    }
  }
  PromptScan p{};
  if ((rc = make_spans(starts, batch, rows, p.spans)) != LQ_OK) return rc;
  if (H < 1 || G < 1 || H % G != 0) {
    return fail(LQ_ERR_INVALID_ARG, "%lld heads over %lld groups", (long long)H, (long long)G);
  }
  if (P < 1 || N < 1 || N > PROMPT_SCAN_MAX_N || P > 65535) {
    return fail(LQ_ERR_UNSUPPORTED, "head_dim %lld, state %lld unsupported (<= 65535, <= %d)",
                (long long)P, (long long)N, PROMPT_SCAN_MAX_N);
  }
  const lq_tensor* per_head[3] = {A, D, dt_bias};
  for (const lq_tensor* t : per_head) {
    if (t != nullptr && t->shape[0] != H) {
      return fail(LQ_ERR_INVALID_ARG, "A, D and dt_bias must be [%lld]", (long long)H);
    }
  }
  const int64_t S = p.spans.S;
  const lq_tensor* st4[2] = {initial, states};
  for (const lq_tensor* t : st4) {
    if (t != nullptr && (t->shape[0] != S || t->shape[1] != H || t->shape[2] != P || t->shape[3] != N)) {
      return fail(LQ_ERR_INVALID_ARG, "states must be [%lld, %lld, %lld, %lld]", (long long)S,
                  (long long)H, (long long)P, (long long)N);
    }
  }
  if (!(dt_min <= dt_max)) return fail(LQ_ERR_INVALID_ARG, "dt_limit %g .. %g", dt_min, dt_max);
  if (batch == 0 || (S == 0 && rows == 0)) return LQ_OK;
  const int64_t total = nd == 4 ? batch * rows : rows;
  if (!sizes_fit(S, rows, nd == 3, H, P, N)) {
    return fail(LQ_ERR_UNSUPPORTED, "%lld rows of %lld prompts exceed the launch limits",
                (long long)total, (long long)S);
  }
  p.segment = (int)plan_segment(prompt_scan_mfma_geometry(x->dtype, H, P, N), S, total, H);
  const int64_t slots = slots_of(S, rows, p.segment, nd == 3);
  const int64_t parts =
      nd == 4 ? batch * (rows == 0 ? 1 : (rows + p.segment - 1) / p.segment) : rows / p.segment + S + 2;
  const int64_t pblocks = (P + PB - 1) / PB;
  const int64_t chunks = nd == 4 ? batch * ((rows + 63) / 64) : rows / 64 + S;
  if (parts * H * pblocks >= ((int64_t)1 << 32) / 256 || slots > 65535 ||
      chunks * ((H + 31) / 32) >= ((int64_t)1 << 32) / 256) {
    return fail(LQ_ERR_UNSUPPORTED, "%lld parts of %lld heads exceed the launch limits",
                (long long)parts, (long long)H);
  }
  const size_t need = lq_prompt_scan_workspace(x->dtype, S, rows, nd == 3, H, P, N);
  if (need > 0 && (workspace == nullptr || workspace_bytes < need)) {
    return fail(LQ_ERR_WORKSPACE, "workspace of %zu bytes needed, %zu given", need,
                workspace == nullptr ? (size_t)0 : workspace_bytes);
  }
  if (need > 0 && ((uintptr_t)workspace & 255) != 0) {
    return fail(LQ_ERR_WORKSPACE, "workspace must be 256-byte aligned");
  }
  const lq_tensor* inputs[10] = {x, dt, A, B, C, starts, D, z, dt_bias, initial};
  for (int i = 0; i < 10; ++i) {
    if (inputs[i] == nullptr) continue;
    const bool in_place = i == 9 && states != nullptr && same_elements(*states, *initial);
    if (overlap(*out, *inputs[i]) || (states != nullptr && !in_place && overlap(*states, *inputs[i]))) {
      return fail(LQ_ERR_INVALID_ARG, "an output overlaps an input");
    }
  }
  if (overlaps_itself(*out) || (states != nullptr && (overlaps_itself(*states) || overlap(*out, *states)))) {
    return fail(LQ_ERR_INVALID_ARG, "the outputs overlap themselves or each other");
  }
  const lq_tensor* ts[6] = {x, B, C, z, out, dt};
  View* vs[6] = {&p.x, &p.B, &p.C, &p.z, &p.out, &p.dt};
  for (int i = 0; i < 6; ++i) {
    *vs[i] = make_view(ts[i]);
    if (ts[i] == nullptr || nd == 4) continue;
    for (int j = 3; j > 0; --j) vs[i]->s[j] = vs[i]->s[j - 1];
    vs[i]->s[0] = 0;
  }
  p.A = make_view(A);
  p.D = make_view(D);
  p.bias = make_view(dt_bias);
  p.initial = make_view(initial);
  p.states = make_view(states);
  p.H = (int)H;
  p.P = (int)P;
  p.N = (int)N;
  p.ratio = (int)(H / G);
  p.softplus = dt_softplus;
  p.slots = (int)slots;
  p.slots_by_rows = slots_by_rows(S, rows, p.segment);
  p.dt_min = dt_min;
  p.dt_max = dt_max;
  p.slot_state = (float*)workspace;
  p.slot_log = (float*)((char*)workspace + align256((size_t)(slots * H * P * N) * 4));
  p.steps = (float*)((char*)p.slot_log + align256((size_t)(slots * H) * 4));
  p.rows = total;
  const hipStream_t st = (hipStream_t)stream;
  const bool mfma = !diag(LQ_DIAG_PROMPT_FORCE_GENERIC) &&
                    prompt_scan_mfma_fits(x, B, C, z, initial, states, out);
  if (!mfma && diag(LQ_DIAG_PROMPT_REQUIRE_MFMA)) {
    return fail(LQ_ERR_INVALID_ARG, "the call takes the general kernel");
  }
  int size = dtype_size(x->dtype);
  const lq_tensor* fours[5] = {x, B, C, z, out};
  for (const lq_tensor* t : fours) size = in_fours(t, x->dtype) && N <= 128 ? size : 0;
  const unsigned blocks = (unsigned)((H * P * N + 255) / 256);
  if (mfma && chunks > 0) {  // (none where no prompt has a row)
    launch_prompt_scan_steps(p, chunks, st);
    if ((rc = check_launch("lq_prompt_scan (steps)")) != LQ_OK) return rc;
  }
  if (slots > 0) {
    if (mfma) launch_prompt_scan_mfma(p, true, slots, st);
    else launch_rows<true>(p, size, dim3((unsigned)(slots * H), (unsigned)pblocks), st);
    if ((rc = check_launch("lq_prompt_scan (segments)")) != LQ_OK) return rc;
    hipLaunchKernelGGL(scan_carry_kernel, dim3((blocks + 3) / 4, (unsigned)slots), dim3(256), 0, st, p);
    if ((rc = check_launch("lq_prompt_scan (carry)")) != LQ_OK) return rc;
  }
  if (parts > 0) {
    if (mfma) launch_prompt_scan_mfma(p, false, parts, st);
    else launch_rows<false>(p, size, dim3((unsigned)(parts * H), (unsigned)pblocks), st);
    if ((rc = check_launch("lq_prompt_scan")) != LQ_OK) return rc;
  }
  return LQ_OK;
}
