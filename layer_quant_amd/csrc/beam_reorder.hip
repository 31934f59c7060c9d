// Beam reordering of decode states, in place: row p*N + n of every listed tensor takes the contents
// of row p*N + beams[p][n].
//
// One launch moves any number of tensors (the INT4 caches' live rows, MX or float states, convolution
// states of all layers). A thread owns a few units (up to 16 bytes) of a row's contents, at the same places
// in all N rows of a prompt: it loads those of every row's source first and stores afterwards, so
// that a row may be the source of some rows and the destination of another, in any permutation, with
// no second buffer and no order between threads. Rows that keep their beam are neither read nor
// written.
#include <algorithm>
#include <cstdlib>

#include "lq_common.h"

namespace lq {
namespace {

constexpr int MAX_BEAMS = LQ_REORDER_MAX_BEAMS;
constexpr int THREADS = 256;
constexpr int MAX_SHAPES = 16;    // different row geometries in a launch
constexpr int MAX_TENSORS = 256;  // tensors in a launch
constexpr int64_t MAX_BLOCKS = ((int64_t)1 << 32) / THREADS - 1;  // a launch holds less than 2^32 threads

// Contents of a row: a n0 x n1 x n2 array of runs (byte strides s0, s1, s2) of `units` units.
struct RowShape {
  int64_t sb;           // bytes between rows
  int64_t s0, s1, s2;
  uint32_t n1, n2;
  uint32_t units;       // units per run
  uint32_t total;       // units per row
  uint32_t blocks;      // workgroups per (tensor, prompt)
  uint32_t first_block;
  uint32_t first_tensor;
  uint32_t unit_log2;   // bytes of a unit
  bool operator==(const RowShape& o) const {
    return sb == o.sb && s0 == o.s0 && s1 == o.s1 && s2 == o.s2 && n1 == o.n1 && n2 == o.n2 &&
           units == o.units && total == o.total && unit_log2 == o.unit_log2;
  }
};

// The tensors are sorted by shape; the kernel's arguments stay below the 4 KiB of a launch.
struct ReorderParams {
  const int64_t* beams;
  int64_t beams_sp, beams_sn;
  int N, P, nshapes;
  RowShape shapes[MAX_SHAPES];
  char* base[MAX_TENSORS];
};
static_assert(sizeof(ReorderParams) <= 4096, "a launch's arguments");

typedef uint32_t u32x4_t __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2_t __attribute__((ext_vector_type(2)));

// Units per thread: two keep the units of 16 rows within 128 registers. (32 rows of 24 layers' MX8 states,
// half of them moved, 1.36 GB read and written: one per thread in scratch 388 us, four 256, two 250; with
// the default cache policy 268 instead of 256. A plain copy of this size runs at 5.24 TB/s, this at 5.46.)
constexpr int units_per_thread(int nmax) { return nmax <= 16 ? 2 : 1; }

// Unit `first` + i THREADS of the row for i < U, of all rows: the sources' first, then the stores. (The
// values are vector types: an array of uint4 structs stays in scratch memory here.)
template <class T, int NMAX, int U>
__device__ __forceinline__ void move_units(const RowShape& sh, char* base, uint32_t first,
                                           const int (&src)[NMAX]) {
  char* at[U];
#pragma unroll
  for (int i = 0; i < U; ++i) {
    const uint32_t u = min(first + i * THREADS, sh.total - 1);
    if (sh.units == sh.total) {
      at[i] = base + (uint64_t)u * sizeof(T);
    } else {
      const uint32_t run = u / sh.units;
      const uint32_t i1 = run / sh.n2;
      const uint32_t i0 = i1 / sh.n1;
      at[i] = base + i0 * sh.s0 + (i1 - i0 * sh.n1) * sh.s1 + (run - i1 * sh.n2) * sh.s2 +
              (uint64_t)(u - run * sh.units) * sizeof(T);
    }
  }
  T v[NMAX][U];
#pragma unroll
  for (int n = 0; n < NMAX; ++n) {
    if (src[n] != n) {
#pragma unroll
      for (int i = 0; i < U; ++i) v[n][i] = __builtin_nontemporal_load((const T*)(at[i] + src[n] * sh.sb));
    }
  }
#pragma unroll
  for (int n = 0; n < NMAX; ++n) {
    if (src[n] != n) {
#pragma unroll
      for (int i = 0; i < U; ++i) {
        if (first + i * THREADS < sh.total) __builtin_nontemporal_store(v[n][i], (T*)(at[i] + n * sh.sb));
      }
    }
  }
}

template <int NMAX>
__global__ __launch_bounds__(THREADS) void reorder_kernel(ReorderParams p) {
  constexpr int U = units_per_thread(NMAX);
  int si = 0;
  while (si + 1 < p.nshapes && blockIdx.x >= p.shapes[si + 1].first_block) ++si;
  const RowShape& sh = p.shapes[si];
  const uint32_t rel = blockIdx.x - sh.first_block;
  const uint32_t tp = rel / sh.blocks;
  const uint32_t first = (rel - tp * sh.blocks) * (THREADS * U) + threadIdx.x;
  const uint32_t tensor = tp / p.P;
  const int64_t prompt = tp - tensor * p.P;

  int64_t beam[NMAX];
#pragma unroll
  for (int n = 0; n < NMAX; ++n) {
    beam[n] = p.beams[prompt * p.beams_sp + min(n, p.N - 1) * p.beams_sn];
  }
  int src[NMAX];
#pragma unroll
  for (int n = 0; n < NMAX; ++n) {
    src[n] = n < p.N && beam[n] >= 0 && beam[n] < p.N ? (int)beam[n] : n;
  }
  if (first >= sh.total) return;
  char* base = p.base[sh.first_tensor + tensor] + prompt * p.N * sh.sb;
  switch (sh.unit_log2) {
    case 4: move_units<u32x4_t, NMAX, U>(sh, base, first, src); break;
    case 3: move_units<u32x2_t, NMAX, U>(sh, base, first, src); break;
    case 2: move_units<uint32_t, NMAX, U>(sh, base, first, src); break;
    case 1: move_units<uint16_t, NMAX, U>(sh, base, first, src); break;
    default: move_units<uint8_t, NMAX, U>(sh, base, first, src); break;
  }
}

// One tensor as the launch takes it: its row geometry and its place in the caller's list.
struct Item {
  RowShape shape;
  char* base;
  int64_t span;  // bytes from base on
};

// The row geometry of t over its first `rows` entries of dim 2 (-1: all); total 0 when it is empty.
int row_shape(const lq_tensor& t, int64_t rows, int64_t per_block, Item& item) {
  const int64_t es = dtype_size(t.dtype);
  int64_t n[3] = {1, 1, 1}, s[3] = {0, 0, 0};  // dims 1 .. 3, in bytes
  for (int d = 1; d < t.ndim; ++d) {
    n[d - 1] = d == 2 && rows >= 0 ? rows : t.shape[d];
    s[d - 1] = t.stride[d] * es;
  }
  RowShape r{};
  r.sb = t.stride[0] * es;
  item.base = (char*)t.data;
  if (n[0] == 0 || n[1] == 0 || n[2] == 0) return LQ_OK;
  // the run that is contiguous from an element on, and the dims outside of it
  int64_t run = es, dims = 0, on[3], os[3];
  for (int d = 2; d >= 0; --d) {
    if (n[d] == 1) continue;
    if (dims == 0 && s[d] == run) {
      run *= n[d];
    } else if (dims > 0 && s[d] == on[dims - 1] * os[dims - 1]) {
      on[dims - 1] *= n[d];
    } else {
      on[dims] = n[d];
      os[dims++] = s[d];
    }
  }
  for (; dims < 3; ++dims) {
    on[dims] = 1;
    os[dims] = 0;
  }
  uint64_t align = (uint64_t)run | (uint64_t)(uintptr_t)t.data | (uint64_t)r.sb;
  for (int d = 0; d < 3; ++d) align |= (uint64_t)os[d];
  while (r.unit_log2 < 4 && (align >> r.unit_log2 & 1) == 0) ++r.unit_log2;
  const int64_t units = run >> r.unit_log2;
  const int64_t total = units * on[0] * on[1] * on[2];
  if (total >= (int64_t)1 << 31) {
    return fail(LQ_ERR_UNSUPPORTED, "a row of %lld units exceeds the launch limits",
                (long long)total);
  }
  r.n1 = (uint32_t)on[1];
  r.n2 = (uint32_t)on[0];
  r.s0 = os[2];
  r.s1 = os[1];
  r.s2 = os[0];
  r.units = (uint32_t)units;
  r.total = (uint32_t)total;
  r.blocks = (uint32_t)((total + per_block - 1) / per_block);
  item.shape = r;
  return LQ_OK;
}

// The bytes that t spans, from its first element's on.
int64_t span_bytes(const lq_tensor& t) {
  int64_t last = 0;
  for (int d = 0; d < t.ndim; ++d) last += (t.shape[d] - 1) * t.stride[d];
  return (last + 1) * dtype_size(t.dtype);
}

int launch(const ReorderParams& p, int nmax, int64_t blocks, hipStream_t st) {
  const dim3 grid((unsigned)blocks), block(THREADS);
  if (nmax == 4) hipLaunchKernelGGL(reorder_kernel<4>, grid, block, 0, st, p);
  else if (nmax == 8) hipLaunchKernelGGL(reorder_kernel<8>, grid, block, 0, st, p);
  else if (nmax == 16) hipLaunchKernelGGL(reorder_kernel<16>, grid, block, 0, st, p);
  else if (nmax == 32) hipLaunchKernelGGL(reorder_kernel<32>, grid, block, 0, st, p);
  else hipLaunchKernelGGL(reorder_kernel<64>, grid, block, 0, st, p);
  return check_launch("lq_reorder_beams");
}

}  // namespace
}  // namespace lq

using namespace lq;

extern "C" int lq_reorder_beams(const lq_tensor* tensors, const int64_t* rows, int count,
                                const lq_tensor* beams, void* stream) {
  int rc;
  if ((rc = check_tensor(beams, "beams", 2, false, LQ_I64)) != LQ_OK) return rc;
  const int64_t P = beams->shape[0], N = beams->shape[1];
  if (N > MAX_BEAMS) {
    return fail(LQ_ERR_UNSUPPORTED, "%lld beams per prompt unsupported (<= %d)", (long long)N,
                MAX_BEAMS);
  }
  if (count < 0 || (count > 0 && tensors == nullptr)) {
    return fail(LQ_ERR_INVALID_ARG, "tensors: %d descriptors at NULL", count);
  }
  if (count > LQ_REORDER_MAX_TENSORS) {
    return fail(LQ_ERR_UNSUPPORTED, "%d tensors in one call unsupported (<= %d)", count,
                LQ_REORDER_MAX_TENSORS);
  }
  const int nmax = N <= 4 ? 4 : N <= 8 ? 8 : N <= 16 ? 16 : N <= 32 ? 32 : 64;
  const int64_t per_block = (int64_t)THREADS * units_per_thread(nmax);
  Item items[LQ_REORDER_MAX_TENSORS];
  int used = 0;
  for (int i = 0; i < count; ++i) {
    const lq_tensor& t = tensors[i];
    if (t.ndim < 1 || t.ndim > 4) {
      return fail(LQ_ERR_INVALID_ARG, "tensor %d: expected 1 to 4 dims, got %d", i, t.ndim);
    }
    bool empty = false;
    for (int d = 0; d < t.ndim; ++d) empty = empty || t.shape[d] == 0;
    if (t.shape[0] != P * N) {
      return fail(LQ_ERR_INVALID_ARG, "tensor %d: %lld rows, expected %lld prompts x %lld beams", i,
                  (long long)t.shape[0], (long long)P, (long long)N);
    }
    const int64_t live = rows == nullptr ? -1 : rows[i];
    if (live != -1 && (t.ndim < 3 || live < 0 || live > t.shape[2])) {
      return fail(LQ_ERR_INVALID_ARG, "tensor %d: %lld entries of dim 2 to move", i,
                  (long long)live);
    }
    if (empty) continue;
    if ((rc = check_tensor(&t, "tensor", t.ndim, false)) != LQ_OK) return rc;
    for (int d = 0; d < t.ndim; ++d) {
      if (t.shape[d] > 1 && t.stride[d] == 0) {
        return fail(LQ_ERR_INVALID_ARG, "tensor %d: a broadcast dimension cannot be moved in place",
                    i);
      }
    }
    if (overlaps_itself(t)) {
      return fail(LQ_ERR_INVALID_ARG, "tensor %d: its elements overlap and cannot be moved in place", i);
    }
    Item it{};
    if ((rc = row_shape(t, live, per_block, it)) != LQ_OK) return rc;
    if (it.shape.total == 0) continue;
    // before anything is moved: a call that fails leaves every tensor as it was
    if (N > 1 && (int64_t)it.shape.blocks * P > MAX_BLOCKS) {
      return fail(LQ_ERR_UNSUPPORTED, "tensor %d: %lld prompts exceed the launch limits", i, (long long)P);
    }
    it.span = span_bytes(t);
    items[used++] = it;
  }
  if (used == 0 || P == 0 || N <= 1) return LQ_OK;
  std::sort(items, items + used, [](const Item& a, const Item& b) { return a.base < b.base; });
  for (int i = 1; i < used; ++i) {
    if (items[i].base == items[i - 1].base) {
      return fail(LQ_ERR_INVALID_ARG, "a tensor is listed twice");
    }
  }
  // a workgroup may read its beams after another has moved rows
  const char* beams_at = (const char*)beams->data;
  const int64_t beams_span = span_bytes(*beams);
  for (int i = 0; i < used; ++i) {
    if (beams_at < items[i].base + items[i].span && items[i].base < beams_at + beams_span) {
      return fail(LQ_ERR_INVALID_ARG, "a tensor overlaps the beams");
    }
  }

  // launches of up to MAX_SHAPES shapes and MAX_TENSORS tensors (one, for a model's states)
  const hipStream_t st = (hipStream_t)stream;
  bool done[LQ_REORDER_MAX_TENSORS] = {};
  for (int left = used; left > 0;) {
    ReorderParams p{};
    p.beams = (const int64_t*)beams->data;
    p.beams_sp = beams->stride[0];
    p.beams_sn = beams->stride[1];
    p.N = (int)N;
    p.P = (int)P;
    int64_t blocks = 0;
    int taken = 0;
    for (int i = 0; i < used && p.nshapes < MAX_SHAPES && taken < MAX_TENSORS; ++i) {
      if (done[i]) continue;
      RowShape sh = items[i].shape;
      sh.first_block = (uint32_t)blocks;
      sh.first_tensor = (uint32_t)taken;
      const int64_t each = (int64_t)sh.blocks * P;
      for (int j = i; j < used && taken < MAX_TENSORS; ++j) {
        if (done[j] || !(items[j].shape == sh)) continue;
        if (blocks + each > MAX_BLOCKS) break;
        p.base[taken++] = items[j].base;
        blocks += each;
        done[j] = true;
        --left;
      }
      if (!done[i]) break;
      p.shapes[p.nshapes++] = sh;
    }
    if ((rc = launch(p, nmax, blocks, st)) != LQ_OK) return rc;
  }
  return LQ_OK;
}
