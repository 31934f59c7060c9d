// The Mamba2 recurrence over whole prompts, packed one behind another or a batch of equal lengths (the
// single token's form is lq_selective_state_update; no reference counterpart: its remote module runs
// prompts, hybrid_quant/mamba_state_8b_kernel.py only decode steps):
//
//   S_t = exp(A dt_t) S_{t-1} + dt_t x_t B_t^T      [P, N] per head
//   y_t = S_t C_t + D x_t,  y_t *= silu(z_t)
//
// A prompt's rows fall into segments. Where a prompt has more than one, so that a few long prompts fill
// the GPU too, a first launch finds the state that each segment but the last adds by itself (the first
// segment starts from the given state and is finished there), a second one carries the states from
// segment to segment, and the last launch runs the others from the state in front of them. A prompt of
// one segment takes the last launch alone. The segment's length follows from the sizes (plan_segment).
//
// scan_rows_kernel walks the rows one by one with the state in registers, fp32 throughout: the kernel of
// fp32 and fp16 inputs and of every geometry that the matrix kernel does not take. A thread holds 4 p x
// (N / 16) n of the state: per row it reads N / 8 + 4 values from LDS for N / 2 fused multiply-adds with
// the state's decay, and four sums over 16 lanes give y.
#include "prompt_scan.h"

namespace lq {
namespace {

constexpr int TB = 16;       // rows per staged block
constexpr int PB = 64;       // p of a workgroup (16 per wave)
constexpr float LOG2E = 1.44269504088896340736f;

template <int NPL>
struct alignas(16) RowTile {
  float x[TB][PB];
  float y[TB][PB];
  float b[TB][16 * NPL];
  float c[TB][16 * NPL];
  float dt[TB], decay[TB];
};

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

// FOLLOWED: the segments that others of their prompt follow (blockIdx: slot), else those that are left.
template <int NPL, bool FOLLOWED>
__global__ __launch_bounds__(256) void scan_rows_kernel(PromptScan p) {
  __shared__ RowTile<NPL> tile;
  const int h = blockIdx.x % p.H, t0 = blockIdx.x / p.H;
  Span sp;
  const bool mine = find_span(
      p.spans, t0,
      [&](int len, bool gap) { return FOLLOWED ? followed_segments_of(p, len, gap) : segments_of(p, len, gap); },
      sp);
  if (!mine) return;
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
  const int nseg = segments_of(p, sp.len, false);
  const int slot = FOLLOWED ? t0 : sp.before + sp.part;
  if (!FOLLOWED && nseg > 1 && sp.part == 0) return;  // finished by the first launch
  if (slot > p.slots) return;                         // starts out of order ask for more than there are
  const bool alone = FOLLOWED && sp.part > 0;         // from no state, and no y

  float st[4][NPL];
  const int64_t slot_at = (((int64_t)slot * p.H + h) * p.P + pb + p0) * p.N;
  const int64_t prev_at = slot_at - (int64_t)p.H * p.P * p.N;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
#pragma unroll
    for (int j = 0; j < NPL; ++j) {
      const int n = 64 * (j >> 2) + 4 * nl + (j & 3);
      float v = 0.f;
      if (!alone && p0 + i < width && n < p.N) {
        if (sp.part > 0) {
          v = p.slot_state[prev_at + (int64_t)i * p.N + n];
        } else if (p.initial.data != nullptr) {
          v = load_float(p.initial.data, p.initial.dtype,
                         sp.index * p.initial.s[0] + h * p.initial.s[1] +
                             (pb + p0 + i) * p.initial.s[2] + n * p.initial.s[3]);
        }
      }
      st[i][j] = v;
    }
  }
  const float A = load_float(p.A.data, p.A.dtype, h * p.A.s[0]) * LOG2E;
  const float bias = p.bias.data == nullptr ? 0.f : load_float(p.bias.data, p.bias.dtype, h * p.bias.s[0]);
  const float D = p.D.data == nullptr ? 0.f : load_float(p.D.data, p.D.dtype, h * p.D.s[0]);
  const int g = h / p.ratio;
  const int64_t x_at = lead * p.x.s[0] + h * p.x.s[2] + pb * p.x.s[3];
  const int64_t z_at = lead * p.z.s[0] + h * p.z.s[2] + pb * p.z.s[3];
  const int64_t b_at = lead * p.B.s[0] + g * p.B.s[2], c_at = lead * p.C.s[0] + g * p.C.s[2];
  const int64_t dt_at = lead * p.dt.s[0] + h * p.dt.s[2];
  float log_decay = 0.f;
  for (int t = from; t < to; t += TB) {
    const int rows = min(TB, to - t);
    const int64_t row = row0 + t;
    __syncthreads();
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
    if (tid < rows) {
      const float dt = scan_step(p, load_float(p.dt.data, p.dt.dtype, dt_at + (row + tid) * p.dt.s[1]), bias);
      tile.dt[tid] = dt;
      tile.decay[tid] = A * dt;
    }
    __syncthreads();
    for (int r = 0; r < rows; ++r) {
      const float lg = tile.decay[r], a = __builtin_amdgcn_exp2f(lg), dt = tile.dt[r];
      log_decay += lg;
      const float4 x4 = *(const float4*)&tile.x[r][p0];
      const float dx[4] = {dt * x4.x, dt * x4.y, dt * x4.z, dt * x4.w};
      float y[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int j = 0; j < NPL; j += 4) {
        const float4 b4 = *(const float4*)&tile.b[r][16 * j + 4 * nl];
        const float4 c4 = *(const float4*)&tile.c[r][16 * j + 4 * nl];
        const float b[4] = {b4.x, b4.y, b4.z, b4.w}, c[4] = {c4.x, c4.y, c4.z, c4.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            st[i][j + e] = fmaf(st[i][j + e], a, dx[i] * b[e]);
            y[i] = fmaf(st[i][j + e], c[e], y[i]);
          }
        }
      }
      if (!alone) {
        const float sum = sums_of_four(y, lane);
        if ((lane & 3) == 0) tile.y[r][p0 + ((lane >> 2) & 3)] = sum;
      }
    }
    if (!alone) {
      __syncthreads();
      for (int i = tid; i < rows * PB; i += blockDim.x) {
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
  if (FOLLOWED) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
#pragma unroll
      for (int j = 0; j < NPL; ++j) {
        const int n = 64 * (j >> 2) + 4 * nl + (j & 3);
        if (p0 + i < width && n < p.N) p.slot_state[slot_at + (int64_t)i * p.N + n] = st[i][j];
      }
    }
    if (tid == 0 && blockIdx.y == 0) p.slot_log[(int64_t)slot * p.H + h] = log_decay;
  } else if (sp.part == nseg - 1 && p.states.data != nullptr) {
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

// The states behind the segments of a prompt from what each adds by itself, in place. blockIdx.y: slot;
// the first slot of a prompt carries all of its own.
__global__ __launch_bounds__(256) void scan_carry_kernel(PromptScan p) {
  Span sp;
  if (!find_span(p.spans, blockIdx.y,
                 [&](int len, bool gap) { return followed_segments_of(p, len, gap); }, sp)) {
    return;
  }
  if (sp.part != 0) return;
  const int many = min(followed_segments_of(p, sp.len, false), p.slots - (int)blockIdx.y);
  const int64_t size = (int64_t)p.H * p.P * p.N, i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i >= size) return;
  const int h = (int)(i / ((int64_t)p.P * p.N));
  float* state = p.slot_state + (int64_t)blockIdx.y * size + i;
  const float* lg = p.slot_log + (int64_t)blockIdx.y * p.H + h;
  float held = state[0];
  for (int j = 1; j < many; ++j) {
    held = fmaf(held, __builtin_amdgcn_exp2f(lg[(int64_t)j * p.H]), state[j * size]);
    state[j * size] = held;
  }
}

constexpr int MIN_SEGMENT = 256;

// Rows of a segment: as many as give about four workgroups per CU, a multiple of 64 and 256 at least
// (a shorter one costs more in carried states than it wins).
int64_t plan_segment(int64_t rows, int64_t heads) {
  const int64_t want = (rows * heads + 4 * device_cus() - 1) / (4 * device_cus());
  const int64_t seg = (want + 63) / 64 * 64;
  return seg < MIN_SEGMENT ? MIN_SEGMENT : seg;
}

// Segments that others follow, at most.
int64_t slots_of(int64_t batch, int64_t rows, int64_t segment, bool packed) {
  return packed ? rows / segment : rows == 0 ? 0 : batch * ((rows + segment - 1) / segment - 1);
}

size_t align256(size_t n) { return (n + 255) & ~(size_t)255; }

template <bool FOLLOWED>
void launch_rows(const PromptScan& p, dim3 grid, hipStream_t st) {
  const dim3 block(64 * min(4, (p.P + 15) / 16));
  if (p.N <= 64) hipLaunchKernelGGL((scan_rows_kernel<4, FOLLOWED>), grid, block, 0, st, p);
  else if (p.N <= 128) hipLaunchKernelGGL((scan_rows_kernel<8, FOLLOWED>), grid, block, 0, st, p);
  else hipLaunchKernelGGL((scan_rows_kernel<16, FOLLOWED>), grid, block, 0, st, p);
}

}  // namespace
}  // namespace lq

using namespace lq;

extern "C" size_t lq_prompt_scan_workspace(int64_t batch, int64_t rows, int packed, int64_t heads,
                                           int64_t head_dim, int64_t dstate) {
  if (batch <= 0 || rows <= 0 || heads <= 0 || head_dim <= 0 || dstate <= 0) return 0;
  const int64_t total = packed ? rows : batch * rows;
  const int64_t slots = slots_of(batch, rows, plan_segment(total, heads), packed != 0);
  return align256((size_t)(slots * heads * head_dim * dstate) * 4) + align256((size_t)(slots * heads) * 4);
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
  if (total > INT32_MAX / 2 || S > 65535 || H * P * N > INT32_MAX / 2) {
    return fail(LQ_ERR_UNSUPPORTED, "%lld rows of %lld prompts exceed the launch limits",
                (long long)total, (long long)S);
  }
  p.segment = (int)plan_segment(total, H);
  const int64_t slots = slots_of(batch, rows, p.segment, nd == 3);
  const int64_t parts =
      nd == 4 ? batch * (rows == 0 ? 1 : (rows + p.segment - 1) / p.segment) : rows / p.segment + S + 2;
  const int64_t pblocks = (P + PB - 1) / PB;
  if (parts * H * pblocks >= ((int64_t)1 << 32) / 256 || slots > 65535) {
    return fail(LQ_ERR_UNSUPPORTED, "%lld parts of %lld heads exceed the launch limits",
                (long long)parts, (long long)H);
  }
  const size_t need = lq_prompt_scan_workspace(batch, rows, nd == 3, H, P, N);
  if (need > 0 && (workspace == nullptr || workspace_bytes < need)) {
    return fail(LQ_ERR_WORKSPACE, "workspace of %zu bytes needed, %zu given", need,
                workspace == nullptr ? (size_t)0 : workspace_bytes);
  }
  if (need > 0 && ((uintptr_t)workspace & 255) != 0) {
    return fail(LQ_ERR_WORKSPACE, "workspace must be 256-byte aligned");
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
  p.dt_min = dt_min;
  p.dt_max = dt_max;
  p.slot_state = (float*)workspace;
  p.slot_log = (float*)((char*)workspace + align256((size_t)(slots * H * P * N) * 4));
  const hipStream_t st = (hipStream_t)stream;
  const bool mfma = !diag(LQ_DIAG_PROMPT_FORCE_GENERIC) &&
                    prompt_scan_mfma_fits(x, B, C, z, initial, states, out);
  if (!mfma && diag(LQ_DIAG_PROMPT_REQUIRE_MFMA)) {
    return fail(LQ_ERR_INVALID_ARG, "the call takes the general kernel");
  }
  const unsigned blocks = (unsigned)((H * P * N + 255) / 256);
  if (slots > 0) {
    if (mfma) launch_prompt_scan_mfma(p, true, slots, st);
    else launch_rows<true>(p, dim3((unsigned)(slots * H), (unsigned)pblocks), st);
    if ((rc = check_launch("lq_prompt_scan (segments)")) != LQ_OK) return rc;
    hipLaunchKernelGGL(scan_carry_kernel, dim3(blocks, (unsigned)slots), dim3(256), 0, st, p);
    if ((rc = check_launch("lq_prompt_scan (carry)")) != LQ_OK) return rc;
  }
  if (parts > 0) {
    if (mfma) launch_prompt_scan_mfma(p, false, parts, st);
    else launch_rows<false>(p, dim3((unsigned)(parts * H), (unsigned)pblocks), st);
    if ((rc = check_launch("lq_prompt_scan")) != LQ_OK) return rc;
  }
  return LQ_OK;
}
