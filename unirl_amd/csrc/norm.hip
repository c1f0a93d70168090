// Layer norm and RMS norm, forward and backward, over rows of at most 32768 elements: the norm in
// front of an AR policy's head, and the modulated norm (gain and bias per sample) in front of a
// diffusion policy's output projection.
//
//   mu = mean(x), s = 1 / sqrt(mean((x - mu)^2) + eps)        (RMS: mu = 0)
//   xh = (x - mu) s,   y = xh (offset + gain) + bias
//   a = dy (offset + gain),   dx = s (a - xh mean(a xh) - mean(a))   (RMS: without mean(a))
//   dgain = sum over rows of dy xh,   dbias = sum over rows of dy
//
// Bound by HBM: two flows of N elements forward (x, y), three backward (x, dy, dx).  A row stays in
// the registers of one wavefront or one workgroup, so it is read once and its variance is taken from
// the centred values; statistics, sums and partial sums are fp32, the result is rounded once.
#include <string.h>

#include "common_hip.h"
#include "unirl_internal.h"

namespace unirl {

constexpr int kNormMaxDim = 32768;
constexpr int kNormRowsPerBlock = 4;       // one-wavefront rows: wavefronts of a workgroup
constexpr int kNormTargetBlocks = 1024;    // backward: workgroups over all groups (4 a compute unit)
constexpr int64_t kNormMaxGroups = 65535;  // of one launch (gridDim.y)
constexpr int64_t kNormMaxBlocks = 1 << 21;  // forward: workgroups per group; the rest is looped over (a launch counts its threads in 32 bits)

struct NormArgs {
  const void* x;
  int64_t x_group_stride, x_row_stride;
  const void* dy;
  int64_t dy_group_stride, dy_row_stride;
  const void* gain;
  const void* bias;
  int64_t gain_group_stride, bias_group_stride;
  int gain_dtype;
  float gain_offset;
  int center;
  float eps, inv_d;
  int D;
  int64_t rows;
  float* mean;
  float* rstd;
  void* out;       // y or dx, dense; backward: may be NULL
  float* partial;  // [groups][blocks][D] of dgain, then of dbias; NULL = no parameter gradients
  int64_t partial_bias;
};

// VEC elements of a gain or bias whose type is known at run time (wave-uniform), from the caches:
// every row reads them.
template <typename T, int VEC>
__device__ __forceinline__ void cached_load(const T* p, float (&o)[VEC]) {
#pragma unroll
  for (int k = 0; k < VEC; ++k) o[k] = Elem<T>::load(p + k);
}
template <int VEC>
__device__ __forceinline__ void load_param(const void* base, int dtype, int64_t at, float absent, float add, float (&o)[VEC]) {
  if (!base) {
#pragma unroll
    for (int k = 0; k < VEC; ++k) o[k] = absent;
    return;
  }
  if (dtype == UNIRL_F32)
    cached_load<float, VEC>((const float*)base + at, o);
  else if (dtype == UNIRL_BF16)
    cached_load<bf16_t, VEC>((const bf16_t*)base + at, o);
  else
    cached_load<f16_t, VEC>((const f16_t*)base + at, o);
#pragma unroll
  for (int k = 0; k < VEC; ++k) o[k] += add;
}

// Sum over the row's threads, in every one of them.
template <bool ONE_WAVE>
__device__ __forceinline__ float row_sum(float v, float* lds) {
  if constexpr (ONE_WAVE)
    return wave_sum(v);
  else
    return block_sum(v, lds);
}

template <typename T, int VEC, int E, bool ONE_WAVE>
__device__ __forceinline__ void norm_fwd_row(const NormArgs& A, int64_t row, int tid, int nthreads, float* lds) {
  const int64_t group = blockIdx.y;
  const T* x = (const T*)A.x + group * A.x_group_stride + row * A.x_row_stride;
  const int64_t flat = group * A.rows + row;
  T* y = (T*)A.out + flat * A.D;
  int cols[E / VEC];
  float v[E];
#pragma unroll
  for (int j = 0; j < E / VEC; ++j) {
    cols[j] = (j * nthreads + tid) * VEC;
    float t[VEC];
#pragma unroll
    for (int k = 0; k < VEC; ++k) t[k] = 0.0f;
    if (cols[j] < A.D) Vec<T, VEC>::load(x + cols[j], t);
#pragma unroll
    for (int k = 0; k < VEC; ++k) v[j * VEC + k] = t[k];
  }
  float mean = 0.0f;
  if (A.center) {
    float s = 0.0f;
#pragma unroll
    for (int k = 0; k < E; ++k) s += v[k];
    mean = row_sum<ONE_WAVE>(s, lds) * A.inv_d;
#pragma unroll
    for (int j = 0; j < E / VEC; ++j)
      if (cols[j] < A.D)
#pragma unroll
        for (int k = 0; k < VEC; ++k) v[j * VEC + k] -= mean;
  }
  float q = 0.0f;
#pragma unroll
  for (int k = 0; k < E; ++k) q = fmaf(v[k], v[k], q);
  const float rstd = 1.0f / sqrtf(row_sum<ONE_WAVE>(q, lds) * A.inv_d + A.eps);
#pragma unroll
  for (int j = 0; j < E / VEC; ++j) {
    if (cols[j] >= A.D) continue;
    float o[VEC], w[VEC], b[VEC];
    load_param<VEC>(A.gain, A.gain_dtype, group * A.gain_group_stride + cols[j], 1.0f, A.gain_offset, w);
    load_param<VEC>(A.bias, A.gain_dtype, group * A.bias_group_stride + cols[j], 0.0f, 0.0f, b);
#pragma unroll
    for (int k = 0; k < VEC; ++k) o[k] = fmaf(v[j * VEC + k] * rstd, w[k], b[k]);
    Vec<T, VEC>::store(y + cols[j], o);
  }
  if (tid == 0) {
    if (A.mean) A.mean[flat] = mean;
    if (A.rstd) A.rstd[flat] = rstd;
  }
}

template <typename T, int VEC, int E, bool ONE_WAVE>
__global__ __launch_bounds__(ONE_WAVE ? 256 : 1024) void norm_fwd_kernel(NormArgs A) {
  __shared__ float lds[16];
  const int tid = ONE_WAVE ? threadIdx.x & (kWave - 1) : threadIdx.x;
  const int nthreads = ONE_WAVE ? kWave : blockDim.x;
  const int64_t first = ONE_WAVE ? (int64_t)blockIdx.x * kNormRowsPerBlock + __builtin_amdgcn_readfirstlane(threadIdx.x / kWave)
                                 : (int64_t)blockIdx.x;
  const int64_t stride = ONE_WAVE ? (int64_t)gridDim.x * kNormRowsPerBlock : (int64_t)gridDim.x;
  for (int64_t row = first; row < A.rows; row += stride) norm_fwd_row<T, VEC, E, ONE_WAVE>(A, row, tid, nthreads, lds);
}

// Each wavefront (or workgroup) walks over rows of one group and keeps the sums of its columns in
// registers; a workgroup leaves one partial row per sum, and norm_param_kernel adds those in order.
template <typename T, int VEC, int E, bool ONE_WAVE, bool BIAS>
__global__ __launch_bounds__(ONE_WAVE ? 256 : 1024) void norm_bwd_kernel(NormArgs A) {
  extern __shared__ float sums[];  // ONE_WAVE: D floats to join the wavefronts; else 2 x 2 x 16 floats
  const int tid = ONE_WAVE ? threadIdx.x & (kWave - 1) : threadIdx.x;
  const int nthreads = ONE_WAVE ? kWave : blockDim.x;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int64_t group = blockIdx.y;
  const T* x = (const T*)A.x + group * A.x_group_stride;
  const T* dy = (const T*)A.dy + group * A.dy_group_stride;

  int cols[E / VEC];
#pragma unroll
  for (int j = 0; j < E / VEC; ++j) cols[j] = (j * nthreads + tid) * VEC;
  float w[E];
#pragma unroll
  for (int j = 0; j < E / VEC; ++j) {
    float t[VEC];
#pragma unroll
    for (int k = 0; k < VEC; ++k) t[k] = 0.0f;
    if (cols[j] < A.D)
      load_param<VEC>(A.gain, A.gain_dtype, group * A.gain_group_stride + cols[j], 1.0f, A.gain_offset, t);
#pragma unroll
    for (int k = 0; k < VEC; ++k) w[j * VEC + k] = t[k];
  }
  float dw[E], db[E];
#pragma unroll
  for (int k = 0; k < E; ++k) dw[k] = db[k] = 0.0f;

  const int64_t first = ONE_WAVE ? (int64_t)blockIdx.x * kNormRowsPerBlock + wave : (int64_t)blockIdx.x;
  const int64_t stride = ONE_WAVE ? (int64_t)gridDim.x * kNormRowsPerBlock : (int64_t)gridDim.x;
  int parity = 0;
  for (int64_t row = first; row < A.rows; row += stride) {
    const int64_t flat = group * A.rows + row;
    const float rstd = A.rstd[flat];
    const float mean = A.center ? A.mean[flat] : 0.0f;
    float xh[E], g[E];
#pragma unroll
    for (int j = 0; j < E / VEC; ++j) {
      float tx[VEC], tg[VEC];
#pragma unroll
      for (int k = 0; k < VEC; ++k) tx[k] = tg[k] = 0.0f;
      if (cols[j] < A.D) {
        Vec<T, VEC>::load(x + row * A.x_row_stride + cols[j], tx);
        Vec<T, VEC>::load(dy + row * A.dy_row_stride + cols[j], tg);
#pragma unroll
        for (int k = 0; k < VEC; ++k) tx[k] = (tx[k] - mean) * rstd;
      }
#pragma unroll
      for (int k = 0; k < VEC; ++k) {
        xh[j * VEC + k] = tx[k];
        g[j * VEC + k] = tg[k];
      }
    }
    float c1 = 0.0f, c2 = 0.0f;
#pragma unroll
    for (int k = 0; k < E; ++k) {
      dw[k] = fmaf(g[k], xh[k], dw[k]);
      if constexpr (BIAS) db[k] += g[k];
      g[k] *= w[k];
      c1 = fmaf(g[k], xh[k], c1);
      c2 += g[k];
    }
    if constexpr (ONE_WAVE) {
      c1 = wave_sum(c1);
      c2 = A.center ? wave_sum(c2) : 0.0f;
    } else {
      // two sets of slots: a row's sums are written while slower wavefronts still read the last row's
      c1 = wave_sum(c1);
      c2 = wave_sum(c2);
      float* s = sums + parity * 32;
      parity ^= 1;
      if ((threadIdx.x & (kWave - 1)) == 0) {
        s[wave] = c1;
        s[16 + wave] = c2;
      }
      __syncthreads();
      c1 = s[0];
      c2 = s[16];
      for (int k = 1; k < (int)blockDim.x / kWave; ++k) {
        c1 += s[k];
        c2 += s[16 + k];
      }
      if (!A.center) c2 = 0.0f;
    }
    c1 *= A.inv_d;
    c2 *= A.inv_d;
    if (A.out) {
      T* dx = (T*)A.out + flat * A.D;
#pragma unroll
      for (int j = 0; j < E / VEC; ++j) {
        if (cols[j] >= A.D) continue;
        float o[VEC];
#pragma unroll
        for (int k = 0; k < VEC; ++k) o[k] = (fmaf(-xh[j * VEC + k], c1, g[j * VEC + k]) - c2) * rstd;
        Vec<T, VEC>::store(dx + cols[j], o);
      }
    }
  }
  if (!A.partial) return;

#pragma unroll
  for (int which = 0; which < (BIAS ? 2 : 1); ++which) {
    float(&acc)[E] = which ? db : dw;
    float* out = A.partial + (which ? A.partial_bias : 0) + (group * gridDim.x + blockIdx.x) * A.D;
    if constexpr (ONE_WAVE) {
      // the wavefronts add their sums in order
      for (int turn = 0; turn < kNormRowsPerBlock; ++turn) {
        __syncthreads();
        if (wave != turn) continue;
#pragma unroll
        for (int j = 0; j < E / VEC; ++j) {
          if (cols[j] >= A.D) continue;
#pragma unroll
          for (int k = 0; k < VEC; ++k) {
            const float v = turn ? sums[cols[j] + k] + acc[j * VEC + k] : acc[j * VEC + k];
            if (turn == kNormRowsPerBlock - 1)
              out[cols[j] + k] = v;
            else
              sums[cols[j] + k] = v;
          }
        }
      }
    } else {
#pragma unroll
      for (int j = 0; j < E / VEC; ++j) {
        if (cols[j] >= A.D) continue;
#pragma unroll
        for (int k = 0; k < VEC; ++k) out[cols[j] + k] = acc[j * VEC + k];
      }
    }
  }
}

// out[set][c] = sum of `n` partial rows, in a fixed order: 16 columns x 16 slices of the rows a workgroup.
template <typename O>
__global__ __launch_bounds__(256) void norm_param_kernel(const float* partial, int64_t n, int D, O* out) {
  __shared__ float lds[256];
  const int c = threadIdx.x & 15, slice = threadIdx.x >> 4;
  const int64_t col = (int64_t)blockIdx.x * 16 + c;
  const float* p = partial + (int64_t)blockIdx.y * n * D;
  float s = 0.0f;
  if (col < D)
    for (int64_t i = slice; i < n; i += 16) s += p[i * D + col];
  lds[threadIdx.x] = s;
  __syncthreads();
  if (slice == 0 && col < D) {
    for (int k = 1; k < 16; ++k) s += lds[k * 16 + c];
    Elem<O>::store(out + (int64_t)blockIdx.y * D + col, s);
  }
}

// --- shapes of launches -----------------------------------------------------
struct NormShape {
  bool one_wave;
  int vec, elems, threads;
};
// A lane holds 8, 16 or 32 elements of a row.  Rows of up to 64 * 32 elements belong to one wavefront
// (no barrier), longer ones to a workgroup of as many threads as 8 elements each ask for, up to 1024.
static NormShape norm_shape(int64_t D, int dtype, bool vectors) {
  NormShape S;
  S.vec = vectors ? 16 / (int)dtype_size(dtype) : 1;
  S.one_wave = D <= kWave * 32;
  if (S.one_wave) {
    S.elems = D <= kWave * 8 ? 8 : (D <= kWave * 16 ? 16 : 32);
    S.threads = kWave * kNormRowsPerBlock;
  } else {
    S.elems = D <= 1024 * 8 ? 8 : (D <= 1024 * 16 ? 16 : 32);
    S.threads = (int)((D + S.elems * kWave - 1) / (S.elems * kWave)) * kWave;
  }
  return S;
}
static int64_t norm_bwd_blocks(int64_t groups, int64_t rows, bool one_wave) {
  const int64_t most = one_wave ? (rows + kNormRowsPerBlock - 1) / kNormRowsPerBlock : rows;
  const int64_t want = (kNormTargetBlocks + groups - 1) / groups;
  return want < most ? want : most;
}

template <typename T, int VEC, int E>
static void launch_norm(const NormArgs& A, const NormShape& S, dim3 grid, bool backward, bool bias, hipStream_t s) {
  const dim3 block(S.threads);
  if (!backward) {
    if (S.one_wave)
      hipLaunchKernelGGL((norm_fwd_kernel<T, VEC, E, true>), grid, block, 0, s, A);
    else
      hipLaunchKernelGGL((norm_fwd_kernel<T, VEC, E, false>), grid, block, 0, s, A);
    return;
  }
  const size_t lds = S.one_wave ? (size_t)A.D * 4 : 64 * 4;
  if (S.one_wave && bias)
    hipLaunchKernelGGL((norm_bwd_kernel<T, VEC, E, true, true>), grid, block, lds, s, A);
  else if (S.one_wave)
    hipLaunchKernelGGL((norm_bwd_kernel<T, VEC, E, true, false>), grid, block, lds, s, A);
  else if (bias)
    hipLaunchKernelGGL((norm_bwd_kernel<T, VEC, E, false, true>), grid, block, lds, s, A);
  else
    hipLaunchKernelGGL((norm_bwd_kernel<T, VEC, E, false, false>), grid, block, lds, s, A);
}
template <typename T>
static void launch_norm(const NormArgs& A, const NormShape& S, dim3 grid, bool backward, bool bias, hipStream_t s) {
  constexpr int V = 16 / (int)sizeof(T);
  if (S.vec == 1) {
    if (S.elems == 8) return launch_norm<T, 1, 8>(A, S, grid, backward, bias, s);
    if (S.elems == 16) return launch_norm<T, 1, 16>(A, S, grid, backward, bias, s);
    return launch_norm<T, 1, 32>(A, S, grid, backward, bias, s);
  }
  if (S.elems == 8) return launch_norm<T, V, 8>(A, S, grid, backward, bias, s);
  if (S.elems == 16) return launch_norm<T, V, 16>(A, S, grid, backward, bias, s);
  return launch_norm<T, V, 32>(A, S, grid, backward, bias, s);
}
static void launch_norm(const NormArgs& A, const NormShape& S, int dtype, dim3 grid, bool backward, bool bias,
                        hipStream_t s) {
  if (dtype == UNIRL_F32)
    launch_norm<float>(A, S, grid, backward, bias, s);
  else if (dtype == UNIRL_BF16)
    launch_norm<bf16_t>(A, S, grid, backward, bias, s);
  else
    launch_norm<f16_t>(A, S, grid, backward, bias, s);
}

// Pointer and strides of a [groups, rows, D] operand suit 16-byte accesses.
static bool vectors_ok(const void* p, int64_t gs, int64_t rs, int64_t D, int64_t groups, int64_t rows, size_t esize) {
  const int64_t v = 16 / (int64_t)esize;
  return aligned_to(p, 16) && D % v == 0 && (rows < 2 || rs % v == 0) && (groups < 2 || gs % v == 0);
}

static int norm_check(const struct unirl_norm_desc* d) {
  if (!d) return UNIRL_E_NULL;
  if (!dtype_ok(d->dtype) || ((d->gain || d->bias) && !dtype_ok(d->gain_dtype))) return UNIRL_E_DTYPE;
  if (d->groups < 0 || d->rows < 0 || d->D < 1) return UNIRL_E_SHAPE;
  if (d->D > kNormMaxDim) return UNIRL_E_LIMIT;
  if (d->groups == 0 || d->rows == 0) return UNIRL_OK;
  if (d->x_group_stride < 0 || d->x_row_stride < 0 || d->gain_group_stride < 0 || d->bias_group_stride < 0)
    return UNIRL_E_SHAPE;
  if (!d->x) return UNIRL_E_NULL;
  if (!aligned_to(d->x, dtype_size(d->dtype)) || !aligned_to(d->mean, 4) || !aligned_to(d->rstd, 4)) return UNIRL_E_ALIGN;
  if (d->gain && !aligned_to(d->gain, dtype_size(d->gain_dtype))) return UNIRL_E_ALIGN;
  if (d->bias && !aligned_to(d->bias, dtype_size(d->gain_dtype))) return UNIRL_E_ALIGN;
  return UNIRL_OK;
}
static NormArgs norm_args(const struct unirl_norm_desc* d, int64_t group0) {
  NormArgs A;
  memset(&A, 0, sizeof(A));
  const size_t es = dtype_size(d->dtype);
  const size_t ps = (d->gain || d->bias) ? dtype_size(d->gain_dtype) : 4;
  A.x = offset_ptr(d->x, group0 * d->x_group_stride, es);
  A.x_group_stride = d->x_group_stride;
  A.x_row_stride = d->x_row_stride;
  A.gain = offset_ptr(d->gain, group0 * d->gain_group_stride, ps);
  A.bias = offset_ptr(d->bias, group0 * d->bias_group_stride, ps);
  A.gain_group_stride = d->gain_group_stride;
  A.bias_group_stride = d->bias_group_stride;
  A.gain_dtype = d->gain_dtype;
  A.gain_offset = d->gain_offset;
  A.center = d->center;
  A.eps = (float)d->eps;
  A.inv_d = 1.0f / (float)d->D;
  A.D = (int)d->D;
  A.rows = d->rows;
  A.mean = offset_f32(d->mean, group0 * d->rows);
  A.rstd = offset_f32(d->rstd, group0 * d->rows);
  return A;
}

}  // namespace unirl

using namespace unirl;

extern "C" int unirl_layer_norm_fwd(const struct unirl_norm_desc* d, void* y, void* stream) {
  const int rc = norm_check(d);
  if (rc != UNIRL_OK) return rc;
  if (d->groups == 0 || d->rows == 0) return UNIRL_OK;
  if (!y) return UNIRL_E_NULL;
  const size_t es = dtype_size(d->dtype);
  if (!aligned_to(y, es)) return UNIRL_E_ALIGN;
  const bool vectors = vectors_ok(d->x, d->x_group_stride, d->x_row_stride, d->D, d->groups, d->rows, es) && aligned_to(y, 16);
  const NormShape S = norm_shape(d->D, d->dtype, vectors);
  for (int64_t g0 = 0; g0 < d->groups; g0 += kNormMaxGroups) {
    const int64_t ng = d->groups - g0 < kNormMaxGroups ? d->groups - g0 : kNormMaxGroups;
    NormArgs A = norm_args(d, g0);
    A.out = (char*)y + g0 * d->rows * d->D * (int64_t)es;
    int64_t gx = S.one_wave ? (d->rows + kNormRowsPerBlock - 1) / kNormRowsPerBlock : d->rows;
    if (gx > kNormMaxBlocks) gx = kNormMaxBlocks;
    launch_norm(A, S, d->dtype, dim3((unsigned)gx, (unsigned)ng), false, false, (hipStream_t)stream);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return (int)e;
  }
  return UNIRL_OK;
}

extern "C" size_t unirl_layer_norm_bwd_scratch_bytes(int64_t groups, int64_t rows, int64_t D) {
  if (groups <= 0 || rows <= 0 || D <= 0 || D > kNormMaxDim) return 0;
  return (size_t)(groups * norm_bwd_blocks(groups, rows, D <= kWave * 32) * D) * 2 * sizeof(float);
}

extern "C" int unirl_layer_norm_bwd(const struct unirl_norm_desc* d, const void* dy, int64_t dy_group_stride,
                                    int64_t dy_row_stride, void* dx, void* dgain, void* dbias, int per_group,
                                    void* scratch, size_t scratch_bytes, void* stream) {
  const int rc = norm_check(d);
  if (rc != UNIRL_OK) return rc;
  const bool params = dgain || dbias;
  if (params && !dtype_ok(d->gain_dtype)) return UNIRL_E_DTYPE;
  if (params && (!aligned_to(dgain, dtype_size(d->gain_dtype)) || !aligned_to(dbias, dtype_size(d->gain_dtype))))
    return UNIRL_E_ALIGN;
  if (per_group && d->groups > kNormMaxGroups) return UNIRL_E_LIMIT;
  hipStream_t s = (hipStream_t)stream;
  const bool empty = d->groups == 0 || d->rows == 0;
  const size_t es = dtype_size(d->dtype);
  int64_t blocks = 0;
  float* part = (float*)scratch;
  int64_t part_bias = 0;
  if (!empty) {
    if (!dy || !d->rstd || (d->center && !d->mean)) return UNIRL_E_NULL;
    if (dy_group_stride < 0 || dy_row_stride < 0) return UNIRL_E_SHAPE;
    if (!aligned_to(dy, es) || !aligned_to(dx, es)) return UNIRL_E_ALIGN;
    const bool vectors = vectors_ok(d->x, d->x_group_stride, d->x_row_stride, d->D, d->groups, d->rows, es) &&
                         vectors_ok(dy, dy_group_stride, dy_row_stride, d->D, d->groups, d->rows, es) && aligned_to(dx, 16);
    const NormShape S = norm_shape(d->D, d->dtype, vectors);
    blocks = norm_bwd_blocks(d->groups, d->rows, S.one_wave);
    if (params) {
      if (!scratch || scratch_bytes < unirl_layer_norm_bwd_scratch_bytes(d->groups, d->rows, d->D)) return UNIRL_E_WORKSPACE;
      if (!aligned_to(scratch, 16)) return UNIRL_E_ALIGN;
    }
    if (!params && !dx) return UNIRL_OK;
    part_bias = d->groups * blocks * d->D;
    for (int64_t g0 = 0; g0 < d->groups; g0 += kNormMaxGroups) {
      const int64_t ng = d->groups - g0 < kNormMaxGroups ? d->groups - g0 : kNormMaxGroups;
      NormArgs A = norm_args(d, g0);
      A.dy = offset_ptr(dy, g0 * dy_group_stride, es);
      A.dy_group_stride = dy_group_stride;
      A.dy_row_stride = dy_row_stride;
      A.out = dx ? (char*)dx + g0 * d->rows * d->D * (int64_t)es : nullptr;
      A.partial = params ? part + g0 * blocks * d->D : nullptr;
      A.partial_bias = part_bias;
      launch_norm(A, S, d->dtype, dim3((unsigned)blocks, (unsigned)ng), true, dbias != nullptr, s);
      const hipError_t e = hipGetLastError();
      if (e != hipSuccess) return (int)e;
    }
  }
  if (!params) return UNIRL_OK;
  // no rows: the sums are zero (n = 0 below)
  const int64_t sets = per_group ? d->groups : 1;
  const int64_t n = empty ? 0 : (per_group ? blocks : d->groups * blocks);
  if (sets == 0) return UNIRL_OK;
  const dim3 grid((unsigned)((d->D + 15) / 16), (unsigned)sets);
  for (int which = 0; which < 2; ++which) {
    void* out = which ? dbias : dgain;
    if (!out) continue;
    const float* p = part + (which ? part_bias : 0);
    if (d->gain_dtype == UNIRL_F32)
      hipLaunchKernelGGL((norm_param_kernel<float>), grid, dim3(256), 0, s, p, n, (int)d->D, (float*)out);
    else if (d->gain_dtype == UNIRL_BF16)
      hipLaunchKernelGGL((norm_param_kernel<bf16_t>), grid, dim3(256), 0, s, p, n, (int)d->D, (bf16_t*)out);
    else
      hipLaunchKernelGGL((norm_param_kernel<f16_t>), grid, dim3(256), 0, s, p, n, (int)d->D, (f16_t*)out);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return (int)e;
  }
  return UNIRL_OK;
}
