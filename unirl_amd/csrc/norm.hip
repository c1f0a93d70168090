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
constexpr int kNormFwdRows = 4;            // one-wavefront rows: wavefronts of a workgroup, forward
constexpr int kNormBwdRows = 8;            // and backward, where fewer workgroups leave fewer partial rows
constexpr int64_t kNormMaxBlocks = 1024;   // workgroups over all groups (4 a compute unit)
constexpr int64_t kNormMaxGroups = 65535;  // of one launch (gridDim.y)

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
  bool keep;  // what is read stays cached
  float eps, inv_d;
  uint32_t D;
  int64_t rows;
  float* mean;
  float* rstd;
  void* out;       // y or dx, dense; backward: may be NULL
  float* partial;  // [groups][blocks][D] of dgain, then of dbias; NULL = no parameter gradients
  int64_t partial_bias;
};

// Rows are read and written through buffer descriptors that end with the row: a lane behind the end
// loads zeros and its stores are dropped, so no access stands behind a condition, and an address
// is one 32-bit offset.
__device__ __forceinline__ __amdgpu_buffer_rsrc_t row_rsrc(const void* row, uint32_t bytes) {
  return __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(row), 0, bytes, 0x00020000);
}
// Cache policy, measured with calls back to back on three sets of inputs (a kernel timed alone leaves the
// write-back of its cached stores to the next one).  Stores stream: cached ones take 39.2 instead of 35.0 us
// for a forward of 101 MB, 77.0 instead of 73.3 us for 201 MB.  The forward's x stays cached where it is
// read again or small: cached / streaming 15.2 / 17.5 us at 42 MB, 35.0 / 35.9 at 101 MB, 73.3 / 71.1 at 201 MB,
// but with the backward behind it 169 / 177 us there.  The backward's x and dy are cached where they are small:
// forward + backward 46.3 / 49.3 us at 42 MB, 66.1 / 65.6 at 63 MB, 179 / 169 at 201 MB.
constexpr int kStreaming = 2;
constexpr int kCached = 0;
constexpr int64_t kKeepForward = 128 << 20, kKeepBackward = 48 << 20;  // bytes of x

// VEC consecutive elements of T as loaded (up to 16 bytes), and as floats.
template <typename T, int VEC>
struct Packed {
  static constexpr int kBytes = VEC * (int)sizeof(T);
  static constexpr int kWords = (kBytes + 3) / 4;
  uint32_t w[kWords];
  template <int POLICY>
  __device__ __forceinline__ void load(__amdgpu_buffer_rsrc_t r, uint32_t off) {
    if constexpr (kBytes == 32) {
      const u32x4 a = __builtin_amdgcn_raw_buffer_load_b128(r, off, 0, POLICY);
      const u32x4 b = __builtin_amdgcn_raw_buffer_load_b128(r, off + 16, 0, POLICY);
#pragma unroll
      for (int k = 0; k < 4; ++k) w[k] = a[k], w[4 + k] = b[k];
    } else if constexpr (kBytes == 16) {
      const u32x4 a = __builtin_amdgcn_raw_buffer_load_b128(r, off, 0, POLICY);
#pragma unroll
      for (int k = 0; k < 4; ++k) w[k] = a[k];
    } else if constexpr (kBytes == 8) {
      const u32x2 a = __builtin_amdgcn_raw_buffer_load_b64(r, off, 0, POLICY);
      w[0] = a[0];
      w[1] = a[1];
    } else if constexpr (kBytes == 4) {
      w[0] = __builtin_amdgcn_raw_buffer_load_b32(r, off, 0, POLICY);
    } else {
      w[0] = __builtin_amdgcn_raw_buffer_load_b16(r, off, 0, POLICY);
    }
  }
  __device__ __forceinline__ float get(int k) const {
    if constexpr (sizeof(T) == 4)
      return __uint_as_float(w[k]);
    else if constexpr (std::is_same<T, bf16_t>::value)
      return __uint_as_float(k & 1 ? w[k / 2] & 0xffff0000u : w[k / 2] << 16);
    else
      return f16_bits_to_f32(k & 1 ? w[k / 2] >> 16 : w[k / 2] & 0xffffu);
  }
};
template <typename T, int VEC>
__device__ __forceinline__ void store_vec(__amdgpu_buffer_rsrc_t r, uint32_t off, const float (&o)[VEC]) {
  if constexpr (VEC == 1) {
    if constexpr (sizeof(T) == 4) {
      __builtin_amdgcn_raw_buffer_store_b32(__float_as_uint(o[0]), r, off, 0, kStreaming);
    } else {
      T t;
      Elem<T>::store(&t, o[0]);
      __builtin_amdgcn_raw_buffer_store_b16((short)t.bits, r, off, 0, kStreaming);
    }
  } else {
    u32x4 v;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      if constexpr (sizeof(T) == 4)
        v[k] = __float_as_uint(o[k]);
      else if constexpr (std::is_same<T, bf16_t>::value)
        v[k] = f32x2_to_bf16x2_bits(o[2 * k], o[2 * k + 1]);
      else
        v[k] = f32_to_f16_bits(o[2 * k]) | (f32_to_f16_bits(o[2 * k + 1]) << 16);
    }
    __builtin_amdgcn_raw_buffer_store_b128(v, r, off, 0, kStreaming);
  }
}

// One lane's share of a row: E elements in vectors `step` elements apart.
template <typename T, int VEC, int E>
struct RowRegs {
  Packed<T, VEC> q[E / VEC];
  template <int POLICY>
  __device__ __forceinline__ void load(const T* row, uint32_t D, uint32_t col, uint32_t step) {
    const __amdgpu_buffer_rsrc_t r = row_rsrc(row, D * (uint32_t)sizeof(T));
#pragma unroll
    for (int j = 0; j < E / VEC; ++j) q[j].template load<POLICY>(r, (col + j * step) * (uint32_t)sizeof(T));
  }
  __device__ __forceinline__ void load(const T* row, uint32_t D, uint32_t col, uint32_t step, bool keep) {
    if (keep)
      load<kCached>(row, D, col, step);
    else
      load<kStreaming>(row, D, col, step);
  }
  __device__ __forceinline__ void unpack(float (&v)[E]) const {
#pragma unroll
    for (int j = 0; j < E / VEC; ++j)
#pragma unroll
      for (int k = 0; k < VEC; ++k) v[j * VEC + k] = q[j].get(k);
  }
};

// A lane's share of a gain or bias (from the caches: every row reads it), all loads in flight at once.
template <typename W, int VEC, int E>
__device__ __forceinline__ void load_param_as(const void* base, int64_t at, uint32_t D, uint32_t col, uint32_t step, float (&o)[E]) {
  const __amdgpu_buffer_rsrc_t r = row_rsrc((const W*)base + at, D * (uint32_t)sizeof(W));
  Packed<W, VEC> q[E / VEC];
#pragma unroll
  for (int j = 0; j < E / VEC; ++j) q[j].template load<kCached>(r, (col + j * step) * (uint32_t)sizeof(W));
#pragma unroll
  for (int j = 0; j < E / VEC; ++j)
#pragma unroll
    for (int k = 0; k < VEC; ++k) o[j * VEC + k] = q[j].get(k);
}
template <int VEC, int E>
__device__ __forceinline__ void load_param(const void* base, int dtype, int64_t at, uint32_t D, uint32_t col, uint32_t step,
                                           float absent, float add, float (&o)[E]) {
  if (!base) {
#pragma unroll
    for (int k = 0; k < E; ++k) o[k] = absent;
    return;
  }
  if (dtype == UNIRL_F32)
    load_param_as<float, VEC, E>(base, at, D, col, step, o);
  else if (dtype == UNIRL_BF16)
    load_param_as<bf16_t, VEC, E>(base, at, D, col, step, o);
  else
    load_param_as<f16_t, VEC, E>(base, at, D, col, step, o);
#pragma unroll
  for (int k = 0; k < E; ++k) o[k] += add;
}

// Sum over the row's threads, in every one of them.
template <bool ONE_WAVE>
__device__ __forceinline__ float row_sum(float v, float* lds) {
  if constexpr (ONE_WAVE)
    return wave_sum(v);
  else
    return block_sum(v, lds);
}

// Both kernels: a wavefront (or workgroup) walks over rows of one group with the gain in registers and
// the next row on its way while it works on one.
template <typename T, int VEC, int E, bool ONE_WAVE, bool BIAS, int THREADS>
__global__ __launch_bounds__(THREADS) void norm_fwd_kernel(NormArgs A) {
  __shared__ float lds[16];
  const uint32_t tid = ONE_WAVE ? threadIdx.x & (kWave - 1) : threadIdx.x;
  const uint32_t step = (ONE_WAVE ? kWave : blockDim.x) * VEC;
  const uint32_t col = tid * VEC;
  const int64_t first = ONE_WAVE ? (int64_t)blockIdx.x * kNormFwdRows + __builtin_amdgcn_readfirstlane(threadIdx.x / kWave)
                                 : (int64_t)blockIdx.x;
  const int64_t stride = ONE_WAVE ? (int64_t)gridDim.x * kNormFwdRows : (int64_t)gridDim.x;
  if (first >= A.rows) return;
  const int64_t group = blockIdx.y;
  const T* x = (const T*)A.x + group * A.x_group_stride;
  RowRegs<T, VEC, E> raw;
  raw.load(x + first * A.x_row_stride, A.D, col, step, A.keep);
  // 128 registers a lane hold a row and the next, but the gain and bias only behind packed loads: fp32
  // D = 18432 77 us with them read per row, 96 us held; bf16 82 / 72 us
  constexpr bool kHeld = THREADS < 1024 || (VEC > 1 && sizeof(T) == 2);
  constexpr int kParams = kHeld ? E : 8;
  float w[kParams], b[BIAS ? kParams : 1];
  const auto load_params = [&](uint32_t at) {
    load_param<VEC, kParams>(A.gain, A.gain_dtype, group * A.gain_group_stride, A.D, at, step, 1.0f, A.gain_offset, w);
    if constexpr (BIAS) load_param<VEC, kParams>(A.bias, A.gain_dtype, group * A.bias_group_stride, A.D, at, step, 0.0f, 0.0f, b);
  };
  if constexpr (kHeld) load_params(col);

  for (int64_t row = first; row < A.rows; row += stride) {
    float v[E];
    raw.unpack(v);
    if (row + stride < A.rows) raw.load(x + (row + stride) * A.x_row_stride, A.D, col, step, A.keep);
    float mean = 0.0f;
    if (A.center) {
      float s = 0.0f;
#pragma unroll
      for (int k = 0; k < E; ++k) s = fmaf(v[k], A.inv_d, s);  // the sum itself could overflow
      mean = row_sum<ONE_WAVE>(s, lds);
#pragma unroll
      for (int j = 0; j < E / VEC; ++j)
#pragma unroll
        for (int k = 0; k < VEC; ++k) v[j * VEC + k] = col + j * step < A.D ? v[j * VEC + k] - mean : 0.0f;
    }
    float q = 0.0f;
#pragma unroll
    for (int k = 0; k < E; ++k) q = fmaf(v[k], v[k], q);
    const float rstd = 1.0f / sqrtf(row_sum<ONE_WAVE>(q, lds) * A.inv_d + A.eps);
    const int64_t flat = group * A.rows + row;
    const __amdgpu_buffer_rsrc_t y = row_rsrc((T*)A.out + flat * A.D, A.D * (uint32_t)sizeof(T));
#pragma unroll
    for (int j = 0; j < E / VEC; ++j) {
      if constexpr (!kHeld)
        if (j % (8 / VEC) == 0) load_params(col + j * step);
      float o[VEC];
#pragma unroll
      for (int k = 0; k < VEC; ++k) {
        const float xh = v[j * VEC + k] * rstd;
        const int at = kHeld ? j * VEC + k : (j * VEC + k) % 8;
        o[k] = BIAS ? fmaf(xh, w[at], b[BIAS ? at : 0]) : xh * w[at];
      }
      store_vec<T, VEC>(y, (col + j * step) * (uint32_t)sizeof(T), o);
    }
    if (tid == 0) {
      if (A.mean) A.mean[flat] = mean;
      if (A.rstd) A.rstd[flat] = rstd;
    }
  }
}

// The sums of the columns stay in registers as well; a workgroup leaves one partial row per sum, and
// norm_param_kernel adds those in order.  Sixteen wavefronts a compute unit have 128 registers each:
// there dgain's sums lie in LDS, and rows of more than 16384 elements are loaded when they are due and
// read the gain from the caches (bf16 with a bias, 100 M elements, D = 24576: 138 us, all of it in registers and
// scratch memory 462; D = 32768 195 / 763 us; one by one D = 16385 254 / 574 us, 32767 425).
template <typename T, int VEC, int E, bool ONE_WAVE, bool BIAS, int THREADS>
__global__ __launch_bounds__(THREADS) void norm_bwd_kernel(NormArgs A) {
  constexpr bool kSumsInLds = THREADS == 1024, kAhead = THREADS < 1024 || E < 24, kGainHeld = kAhead;
  extern __shared__ float sums[];  // ONE_WAVE: 4 D floats to join the wavefronts; else 2 x 2 x 16 floats
  __shared__ float dw_lds[kSumsInLds ? E * THREADS : 1];
  const uint32_t tid = ONE_WAVE ? threadIdx.x & (kWave - 1) : threadIdx.x;
  const uint32_t step = (ONE_WAVE ? kWave : blockDim.x) * VEC;
  const uint32_t col = tid * VEC;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int64_t group = blockIdx.y;
  const T* x = (const T*)A.x + group * A.x_group_stride;
  const T* dy = (const T*)A.dy + group * A.dy_group_stride;
  const int64_t first = ONE_WAVE ? (int64_t)blockIdx.x * kNormBwdRows + wave : (int64_t)blockIdx.x;
  const int64_t stride = ONE_WAVE ? (int64_t)gridDim.x * kNormBwdRows : (int64_t)gridDim.x;
  RowRegs<T, VEC, E> rx, rg;
  float rstd = 0.0f, mean = 0.0f;
  if (kAhead && first < A.rows) {
    rx.load(x + first * A.x_row_stride, A.D, col, step, A.keep);
    rg.load(dy + first * A.dy_row_stride, A.D, col, step, A.keep);
  }
  const int64_t gain_at = group * A.gain_group_stride;
  float w[kGainHeld ? E : 8];
  if constexpr (kGainHeld) load_param<VEC, E>(A.gain, A.gain_dtype, gain_at, A.D, col, step, 1.0f, A.gain_offset, w);
  float dw[kSumsInLds ? 1 : E], db[BIAS ? E : 1];
#pragma unroll
  for (int k = 0; k < E; ++k) {
    if constexpr (kSumsInLds)
      dw_lds[k * THREADS + threadIdx.x] = 0.0f;
    else
      dw[k] = 0.0f;
  }
#pragma unroll
  for (int k = 0; k < (BIAS ? E : 1); ++k) db[k] = 0.0f;

  int parity = 0;
  for (int64_t row = first; row < A.rows; row += stride) {
    const int64_t flat = group * A.rows + row;
    rstd = A.rstd[flat];
    if (A.center) mean = A.mean[flat];
    if constexpr (!kAhead) {
      rx.template load<kStreaming>(x + row * A.x_row_stride, A.D, col, step);
      rg.template load<kStreaming>(dy + row * A.dy_row_stride, A.D, col, step);
    }
    float xh[E], g[E];
    rx.unpack(xh);
    rg.unpack(g);
    if (kAhead && row + stride < A.rows) {
      rx.load(x + (row + stride) * A.x_row_stride, A.D, col, step, A.keep);
      rg.load(dy + (row + stride) * A.dy_row_stride, A.D, col, step, A.keep);
    }
    // behind the row's end x and dy are 0, and so is xh there (0 - mean could overflow on its way)
#pragma unroll
    for (int j = 0; j < E / VEC; ++j) {
      const float mu = col + j * step < A.D ? mean : 0.0f;
#pragma unroll
      for (int k = 0; k < VEC; ++k) xh[j * VEC + k] = (xh[j * VEC + k] - mu) * rstd;
    }
    float c1 = 0.0f, c2 = 0.0f;
#pragma unroll
    for (int k = 0; k < E; ++k) {
      if constexpr (!kGainHeld)
        if (k % 8 == 0)
          load_param<VEC, 8>(A.gain, A.gain_dtype, gain_at, A.D, col + k / VEC * step, step, 1.0f, A.gain_offset, w);
      if constexpr (kSumsInLds) {
        float& sum = dw_lds[k * THREADS + threadIdx.x];
        sum = fmaf(g[k], xh[k], sum);
      } else {
        dw[k] = fmaf(g[k], xh[k], dw[k]);
      }
      if constexpr (BIAS) db[k] += g[k];
      g[k] *= w[kGainHeld ? k : k % 8];
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
      const __amdgpu_buffer_rsrc_t dx = row_rsrc((T*)A.out + flat * A.D, A.D * (uint32_t)sizeof(T));
#pragma unroll
      for (int j = 0; j < E / VEC; ++j) {
        float o[VEC];
#pragma unroll
        for (int k = 0; k < VEC; ++k) o[k] = (fmaf(-xh[j * VEC + k], c1, g[j * VEC + k]) - c2) * rstd;
        store_vec<T, VEC>(dx, (col + j * step) * (uint32_t)sizeof(T), o);
      }
    }
  }
  if (!A.partial) return;

#pragma unroll
  for (int which = 0; which < (BIAS ? 2 : 1); ++which) {
    float* out = A.partial + (which ? A.partial_bias : 0) + (group * gridDim.x + blockIdx.x) * A.D;
    float acc[E];
#pragma unroll
    for (int k = 0; k < E; ++k)
      acc[k] = which ? db[BIAS ? k : 0] : (kSumsInLds ? dw_lds[k * THREADS + threadIdx.x] : dw[kSumsInLds ? 0 : k]);
    if constexpr (ONE_WAVE) {
      // the second half of the wavefronts leaves its sums in LDS, the first adds its own, then every
      // thread adds the four sums of its columns
      constexpr int kHalf = kNormBwdRows / 2;
      float* mine = sums + (wave % kHalf) * A.D;
      if (which) __syncthreads();
#pragma unroll
      for (int pass = 0; pass < 2; ++pass) {
        if (wave / kHalf != pass) {
#pragma unroll
          for (int j = 0; j < E / VEC; ++j) {
            if (col + j * step >= A.D) continue;
#pragma unroll
            for (int k = 0; k < VEC; ++k) {
              const uint32_t c = col + j * step + k;
              mine[c] = pass ? mine[c] + acc[j * VEC + k] : acc[j * VEC + k];
            }
          }
        }
        __syncthreads();
      }
      for (uint32_t c = threadIdx.x; c < A.D; c += kNormBwdRows * kWave) {
        float v = sums[c];
#pragma unroll
        for (int h = 1; h < kHalf; ++h) v += sums[h * A.D + c];
        out[c] = v;
      }
    } else {
#pragma unroll
      for (int j = 0; j < E / VEC; ++j) {
        if (col + j * step >= A.D) continue;
#pragma unroll
        for (int k = 0; k < VEC; ++k) out[col + j * step + k] = acc[j * VEC + k];
      }
    }
  }
}

// --- rows of at most 32 vectors (heads of 64 or 128): several rows share a wavefront ----------------
// Sum over each group of LANES adjacent lanes (8, 16, 32), in every one of them: swaps inside quads, then
// mirrored halves of 8 and 16 lanes (each lane of a quad, then of eight, holds the same sum by then).
template <int LANES>
__device__ __forceinline__ float lanes_sum(float v) {
  v += __int_as_float(dpp_move<0xB1, 0xf>(0, __float_as_int(v)));   // lanes 1 0 3 2
  v += __int_as_float(dpp_move<0x4E, 0xf>(0, __float_as_int(v)));   // lanes 2 3 0 1
  v += __int_as_float(dpp_move<0x141, 0xf>(0, __float_as_int(v)));  // mirrored in 8
  if constexpr (LANES >= 16) v += __int_as_float(dpp_move<0x140, 0xf>(0, __float_as_int(v)));  // mirrored in 16
  if constexpr (LANES >= 32) v += __shfl_xor(v, 16);
  return v;
}

// A wavefront takes 64 / LANES rows at a time; a lane keeps one vector of columns.  The descriptor
// covers the rows that the wavefront reads, and a lane without a row or behind its end asks for an
// offset outside it.
constexpr uint32_t kOutside = 0x80000000u;
template <typename T, int LANES>
struct NarrowRows {
  static constexpr int VEC = 16 / (int)sizeof(T), kRows = kWave / LANES;
  uint32_t sub, col;
  bool live;
  __device__ __forceinline__ NarrowRows(uint32_t D) {
    const uint32_t lane = threadIdx.x & (kWave - 1);
    sub = lane / LANES;
    col = lane % LANES * VEC;
    live = col < D;
  }
  // rows [row, row + kRows) of a tensor whose rows are `stride` elements apart
  __device__ __forceinline__ __amdgpu_buffer_rsrc_t rsrc(const T* base, int64_t row, int64_t stride) const {
    return row_rsrc(base + row * stride, kOutside - 1);
  }
  __device__ __forceinline__ uint32_t off(int64_t row, int64_t rows, int64_t stride) const {
    return live && row + sub < rows ? (sub * (uint32_t)stride + col) * (uint32_t)sizeof(T) : kOutside;
  }
};

template <typename T, int LANES, bool BIAS>
__global__ __launch_bounds__(256) void norm_narrow_fwd_kernel(NormArgs A) {
  using N = NarrowRows<T, LANES>;
  constexpr int VEC = N::VEC;
  const N at(A.D);
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int64_t group = blockIdx.y, stride = (int64_t)gridDim.x * 4 * N::kRows;
  const T* x = (const T*)A.x + group * A.x_group_stride;
  int64_t row = ((int64_t)blockIdx.x * 4 + wave) * N::kRows;
  if (row >= A.rows) return;
  Packed<T, VEC> raw;
  const auto load = [&](int64_t r) {
    if (A.keep)
      raw.template load<kCached>(at.rsrc(x, r, A.x_row_stride), at.off(r, A.rows, A.x_row_stride));
    else
      raw.template load<kStreaming>(at.rsrc(x, r, A.x_row_stride), at.off(r, A.rows, A.x_row_stride));
  };
  load(row);
  float w[VEC], b[BIAS ? VEC : 1];
  load_param<VEC, VEC>(A.gain, A.gain_dtype, group * A.gain_group_stride, A.D, at.col, 0, 1.0f, A.gain_offset, w);
  if constexpr (BIAS) load_param<VEC, VEC>(A.bias, A.gain_dtype, group * A.bias_group_stride, A.D, at.col, 0, 0.0f, 0.0f, b);
  for (; row < A.rows; row += stride) {
    float v[VEC];
#pragma unroll
    for (int k = 0; k < VEC; ++k) v[k] = raw.get(k);
    if (row + stride < A.rows) load(row + stride);
    float mean = 0.0f;
    if (A.center) {
      float s = 0.0f;
#pragma unroll
      for (int k = 0; k < VEC; ++k) s = fmaf(v[k], A.inv_d, s);  // the sum itself could overflow
      mean = lanes_sum<LANES>(s);
#pragma unroll
      for (int k = 0; k < VEC; ++k) v[k] = at.live ? v[k] - mean : 0.0f;
    }
    float q = 0.0f;
#pragma unroll
    for (int k = 0; k < VEC; ++k) q = fmaf(v[k], v[k], q);
    const float rstd = 1.0f / sqrtf(lanes_sum<LANES>(q) * A.inv_d + A.eps);
    const int64_t flat = group * A.rows + row;
    float o[VEC];
#pragma unroll
    for (int k = 0; k < VEC; ++k) {
      const float xh = v[k] * rstd;
      o[k] = BIAS ? fmaf(xh, w[k], b[BIAS ? k : 0]) : xh * w[k];
    }
    store_vec<T, VEC>(at.rsrc((const T*)A.out + group * A.rows * A.D, row, A.D), at.off(row, A.rows, A.D), o);
    if (at.col == 0 && row + at.sub < A.rows) {
      if (A.mean) A.mean[flat + at.sub] = mean;
      if (A.rstd) A.rstd[flat + at.sub] = rstd;
    }
  }
}

template <typename T, int LANES, bool BIAS>
__global__ __launch_bounds__(512) void norm_narrow_bwd_kernel(NormArgs A) {
  using N = NarrowRows<T, LANES>;
  constexpr int VEC = N::VEC;
  __shared__ float sums[512 * VEC];  // [wavefront * rows of one][LANES * VEC]
  const N at(A.D);
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int64_t group = blockIdx.y, stride = (int64_t)gridDim.x * kNormBwdRows * N::kRows;
  const T* x = (const T*)A.x + group * A.x_group_stride;
  const T* dy = (const T*)A.dy + group * A.dy_group_stride;
  int64_t row = ((int64_t)blockIdx.x * kNormBwdRows + wave) * N::kRows;
  Packed<T, VEC> rx, rg;
  float rstd = 0.0f, mean = 0.0f;
  const auto load = [&](int64_t r) {
    if (A.keep) {
      rx.template load<kCached>(at.rsrc(x, r, A.x_row_stride), at.off(r, A.rows, A.x_row_stride));
      rg.template load<kCached>(at.rsrc(dy, r, A.dy_row_stride), at.off(r, A.rows, A.dy_row_stride));
    } else {
      rx.template load<kStreaming>(at.rsrc(x, r, A.x_row_stride), at.off(r, A.rows, A.x_row_stride));
      rg.template load<kStreaming>(at.rsrc(dy, r, A.dy_row_stride), at.off(r, A.rows, A.dy_row_stride));
    }
    const int64_t flat = group * A.rows + (r + at.sub < A.rows ? r + at.sub : A.rows - 1);
    rstd = A.rstd[flat];
    if (A.center) mean = A.mean[flat];
  };
  if (row < A.rows) load(row);
  float w[VEC], dw[VEC], db[BIAS ? VEC : 1];
  load_param<VEC, VEC>(A.gain, A.gain_dtype, group * A.gain_group_stride, A.D, at.col, 0, 1.0f, A.gain_offset, w);
#pragma unroll
  for (int k = 0; k < VEC; ++k) dw[k] = 0.0f;
#pragma unroll
  for (int k = 0; k < (BIAS ? VEC : 1); ++k) db[k] = 0.0f;
  for (; row < A.rows; row += stride) {
    float xh[VEC], g[VEC];
    // behind the rows and their ends x and dy are 0, and so is xh there (0 - mean could overflow on its way)
    const float s = rstd, mu = at.live && row + at.sub < A.rows ? mean : 0.0f;
#pragma unroll
    for (int k = 0; k < VEC; ++k) {
      xh[k] = (rx.get(k) - mu) * s;
      g[k] = rg.get(k);
    }
    if (row + stride < A.rows) load(row + stride);
    float c1 = 0.0f, c2 = 0.0f;
#pragma unroll
    for (int k = 0; k < VEC; ++k) {
      dw[k] = fmaf(g[k], xh[k], dw[k]);
      if constexpr (BIAS) db[k] += g[k];
      g[k] *= w[k];
      c1 = fmaf(g[k], xh[k], c1);
      c2 += g[k];
    }
    c1 = lanes_sum<LANES>(c1) * A.inv_d;
    c2 = A.center ? lanes_sum<LANES>(c2) * A.inv_d : 0.0f;
    if (A.out) {
      float o[VEC];
#pragma unroll
      for (int k = 0; k < VEC; ++k) o[k] = (fmaf(-xh[k], c1, g[k]) - c2) * s;
      store_vec<T, VEC>(at.rsrc((const T*)A.out + group * A.rows * A.D, row, A.D), at.off(row, A.rows, A.D), o);
    }
  }
  if (!A.partial) return;
#pragma unroll
  for (int which = 0; which < (BIAS ? 2 : 1); ++which) {
    if (which) __syncthreads();
#pragma unroll
    for (int k = 0; k < VEC; ++k) sums[threadIdx.x * VEC + k] = which ? db[BIAS ? k : 0] : dw[k];
    __syncthreads();
    float* out = A.partial + (which ? A.partial_bias : 0) + (group * gridDim.x + blockIdx.x) * A.D;
    for (uint32_t c = threadIdx.x; c < A.D; c += 512) {
      float v = 0.0f;
      for (int h = 0; h < 512 / LANES; ++h) v += sums[h * (LANES * VEC) + c];
      out[c] = v;
    }
  }
}

// out[set][c] = sum of `n` partial rows, in a fixed order: 32 columns x 32 slices of the rows a
// workgroup, eight rows' loads of a lane in flight (a plain loop makes one trip to memory per row).
// blockIdx.z: dgain, dbias.
template <typename O>
__global__ __launch_bounds__(1024) void norm_param_kernel(const float* partial, int64_t partial_bias, int64_t n, uint32_t D, O* dgain,
                                                         O* dbias) {
  __shared__ float lds[32][33];
  O* out = blockIdx.z ? dbias : dgain;
  if (!out) return;
  const int c = threadIdx.x & 31, slice = threadIdx.x >> 5;
  const uint32_t col = blockIdx.x * 32 + c;
  const float* p = partial + (blockIdx.z ? partial_bias : 0) + (int64_t)blockIdx.y * n * D + (col < D ? col : D - 1);
  float s = 0.0f;
  for (int64_t i0 = slice; i0 < n; i0 += 32 * 8) {
    float t[8];
#pragma unroll
    for (int b = 0; b < 8; ++b) {
      const int64_t i = i0 + 32 * b;
      t[b] = p[(i < n ? i : n - 1) * D];
    }
#pragma unroll
    for (int b = 0; b < 8; ++b) s += i0 + 32 * b < n ? t[b] : 0.0f;
  }
  lds[slice][c] = s;
  __syncthreads();
  if (slice == 0 && col < D) {
    for (int k = 1; k < 32; ++k) s += lds[k][c];
    Elem<O>::store(out + (int64_t)blockIdx.y * D + col, s);
  }
}

// --- shapes of launches -----------------------------------------------------
struct NormShape {
  int lanes;  // of one row: 8, 16, 32 or 64 of a wavefront, 0 = a workgroup
  int vec, elems, threads;
};
// Rows of up to 32 vectors share a wavefront (forward, bf16 [781250, 128]: 77 us, one row a wavefront 183).
// Rows of up to 64 * 64 elements (forward; 64 * 32 one by one) or 64 * 32 (backward, whose lanes hold five
// numbers per element; 64 * 24 in fp32, 64 * 16 one by one, which hold their loads in more registers)
// belong to one wavefront, longer ones to a workgroup.  Backward with a bias, 100 M elements of bf16 (half
// as many of fp32), one wavefront / workgroup: bf16 D = 1000 114 / 168 us, 1600 105 / 127 us, 2048 109 / 112 us;
// fp32 equal from D = 1000 to 1536.
// A workgroup has as few elements a lane as its width allows, since wide workgroups stay resident alone
// and few registers hold a long row: backward 8 up to 768 threads (bf16 D = 5120 109 us, 16 of 320 threads
// 134; but D = 7168 115 us in 16, 150 in 8 of 896 threads), then 16 (bf16 / fp32 D = 10240 135 / 113 us, 32 of 320
// threads, some of them in scratch memory, 160 / 205), 24, 32.  Forward 8 and 16 up to 512 threads, then 32, and
// 24 where that fits 1024 threads.
static NormShape norm_shape(int64_t D, int dtype, bool vectors, bool backward) {
  NormShape S;
  S.vec = vectors ? 16 / (int)dtype_size(dtype) : 1;
  const int64_t one_wave = !backward ? (vectors ? 64 : 32) : (!vectors ? 16 : (dtype == UNIRL_F32 ? 24 : 32));
  if (vectors && D <= 32 * S.vec) {
    S.lanes = D <= 8 * S.vec ? 8 : (D <= 16 * S.vec ? 16 : 32);
    S.elems = S.vec;
    S.threads = kWave * (backward ? kNormBwdRows : kNormFwdRows);
  } else if (D <= kWave * one_wave) {
    S.lanes = 64;
    const int need = (int)((D + kWave - 1) / kWave);  // elements of a lane
    S.elems = need <= 8 ? 8 : (need <= 16 ? 16 : (need <= 32 && !vectors ? 32 : (need + 7) / 8 * 8));
    if (S.elems == 56) S.elems = 64;
    S.threads = kWave * (backward ? kNormBwdRows : kNormFwdRows);
  } else {
    S.lanes = 0;
    S.elems = D <= (backward ? 768 : 512) * 8 ? 8 : (D <= (backward ? 1024 : 512) * 16 ? 16 : (D > 512 * 32 && D <= 1024 * 24 ? 24 : 32));
    S.threads = (int)((D + S.elems * kWave - 1) / (S.elems * kWave)) * kWave;
  }
  return S;
}
// Workgroups of one group.  Forward: up to 4 a compute unit (8 where rows share a wavefront).
// Backward: as many as stay resident, since a few more would run alone behind the others, with two rows
// a wavefront at least, since each leaves a partial row of D sums.
static int64_t norm_blocks(const NormShape& S, int64_t groups, int64_t rows, bool backward, bool bias) {
  const int64_t rows_at_once = S.lanes ? S.threads / S.lanes : 1;
  const int64_t most = (rows + rows_at_once - 1) / rows_at_once;
  int64_t total = S.lanes && S.lanes < kWave ? 2 * kNormMaxBlocks : kNormMaxBlocks;
  if (backward) {
    // wavefronts that a compute unit's registers hold (16 are enough where rows share a wavefront)
    int64_t slots = S.elems <= 8 ? 28 : (S.elems <= 16 ? 16 : 8);
    if (S.vec == 1) slots = S.elems <= 8 ? 20 : (S.elems <= 16 ? 12 : 8);
    if (S.lanes && S.lanes < kWave) slots = 16;
    const int64_t waves = S.threads / kWave;
    // fewer where they do not spread evenly over its four register files, which a bias fills further (with it,
    // 28 / these, bf16 D = 3584 140 / 113 us, 4608 134 / 109; fp32 D = 3584 120 / 111 us)
    if (S.elems <= 8 && waves % 4) slots = S.vec == 8 ? (bias ? 24 : 28) : (S.vec == 4 ? (bias ? 22 : 24) : (bias ? 16 : 20));
    const int64_t resident = slots / waves;
    total = 256 * (resident > 1 ? resident : 1);
    if (total > kNormMaxBlocks) total = kNormMaxBlocks;  // what unirl_layer_norm_bwd_scratch_bytes has room for
    const int64_t enough = (rows * groups + 2 * rows_at_once - 1) / (2 * rows_at_once);
    if (total > enough) total = enough;
  }
  const int64_t want = (total + groups - 1) / groups;
  return want < most ? want : most;
}

template <typename T, int VEC, int E, bool BIAS>
static void launch_norm(const NormArgs& A, const NormShape& S, dim3 grid, bool backward, hipStream_t s) {
  const dim3 block(S.threads);
  if (S.lanes == kWave) {
    if (!backward)
      hipLaunchKernelGGL((norm_fwd_kernel<T, VEC, E, true, BIAS, kNormFwdRows * kWave>), grid, block, 0, s, A);
    else if constexpr (E <= (VEC == 1 ? 16 : (sizeof(T) == 4 ? 24 : 32)))
      hipLaunchKernelGGL((norm_bwd_kernel<T, VEC, E, true, BIAS, kNormBwdRows * kWave>), grid, block,
                         (size_t)A.D * (kNormBwdRows / 2 * 4), s, A);
  } else if constexpr (E == 8 || E == 16 || E == 24 || E == 32) {
    // what norm_shape gives: forward 8, 16, 32 up to 512 threads, 24, 32 above; backward 8 up to 768
    // threads, 16 at any width, 24, 32 above 512
    constexpr size_t kSlots = 64 * 4;
    const bool small = S.threads <= 512;
    if (backward) {
      if constexpr (E <= 16)
        if (small) hipLaunchKernelGGL((norm_bwd_kernel<T, VEC, E, false, BIAS, 512>), grid, block, kSlots, s, A);
      if constexpr (E <= 16)
        if (!small && S.threads <= 768)
          hipLaunchKernelGGL((norm_bwd_kernel<T, VEC, E, false, BIAS, 768>), grid, block, kSlots, s, A);
      if constexpr (E >= 16)
        if (S.threads > (E == 16 ? 768 : 512))
          hipLaunchKernelGGL((norm_bwd_kernel<T, VEC, E, false, BIAS, 1024>), grid, block, kSlots, s, A);
    } else {
      // vectors of rows that 8 a lane cover belong to one wavefront
      if constexpr (E != 24 && (VEC == 1 || E > 8))
        if (small) hipLaunchKernelGGL((norm_fwd_kernel<T, VEC, E, false, BIAS, 512>), grid, block, 0, s, A);
      if constexpr (E >= 24)
        if (!small) hipLaunchKernelGGL((norm_fwd_kernel<T, VEC, E, false, BIAS, 1024>), grid, block, 0, s, A);
    }
  }
}
template <typename T, int VEC, int E>
static void launch_norm(const NormArgs& A, const NormShape& S, dim3 grid, bool backward, bool bias, hipStream_t s) {
  if (bias)
    launch_norm<T, VEC, E, true>(A, S, grid, backward, s);
  else
    launch_norm<T, VEC, E, false>(A, S, grid, backward, s);
}
template <typename T, int LANES>
static void launch_narrow(const NormArgs& A, const NormShape& S, dim3 grid, bool backward, bool bias, hipStream_t s) {
  const dim3 block(S.threads);
  if (backward && bias)
    hipLaunchKernelGGL((norm_narrow_bwd_kernel<T, LANES, true>), grid, block, 0, s, A);
  else if (backward)
    hipLaunchKernelGGL((norm_narrow_bwd_kernel<T, LANES, false>), grid, block, 0, s, A);
  else if (bias)
    hipLaunchKernelGGL((norm_narrow_fwd_kernel<T, LANES, true>), grid, block, 0, s, A);
  else
    hipLaunchKernelGGL((norm_narrow_fwd_kernel<T, LANES, false>), grid, block, 0, s, A);
}
template <typename T>
static void launch_norm(const NormArgs& A, const NormShape& S, dim3 grid, bool backward, bool bias, hipStream_t s) {
  constexpr int V = 16 / (int)sizeof(T);
  switch (S.lanes) {
    case 8: return launch_narrow<T, 8>(A, S, grid, backward, bias, s);
    case 16: return launch_narrow<T, 16>(A, S, grid, backward, bias, s);
    case 32: return launch_narrow<T, 32>(A, S, grid, backward, bias, s);
    default: break;
  }
  if (S.vec == 1) {
    switch (S.elems) {
      case 8: return launch_norm<T, 1, 8>(A, S, grid, backward, bias, s);
      case 16: return launch_norm<T, 1, 16>(A, S, grid, backward, bias, s);
      case 24: return launch_norm<T, 1, 24>(A, S, grid, backward, bias, s);
      default: return launch_norm<T, 1, 32>(A, S, grid, backward, bias, s);
    }
  }
  switch (S.elems) {
    case 8: return launch_norm<T, V, 8>(A, S, grid, backward, bias, s);
    case 16: return launch_norm<T, V, 16>(A, S, grid, backward, bias, s);
    case 24: return launch_norm<T, V, 24>(A, S, grid, backward, bias, s);
    case 32: return launch_norm<T, V, 32>(A, S, grid, backward, bias, s);
    case 40: return launch_norm<T, V, 40>(A, S, grid, backward, bias, s);
    case 48: return launch_norm<T, V, 48>(A, S, grid, backward, bias, s);
    default: return launch_norm<T, V, 64>(A, S, grid, backward, bias, s);
  }
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

// Pointer and strides of a [groups, rows, D] operand suit 16-byte accesses (and the 32-bit offsets of
// eight rows that share a wavefront).
static bool vectors_ok(const void* p, int64_t gs, int64_t rs, int64_t D, int64_t groups, int64_t rows, size_t esize) {
  const int64_t v = 16 / (int64_t)esize;
  return aligned_to(p, 16) && D % v == 0 && (rows < 2 || (rs % v == 0 && rs < (1 << 24))) && (groups < 2 || gs % v == 0);
}

static bool params_vectors_ok(const struct unirl_norm_desc* d) {
  const size_t ps = (d->gain || d->bias) ? dtype_size(d->gain_dtype) : 4;
  const int64_t v = 16 / (int64_t)ps;
  return aligned_to(d->gain, 16) && aligned_to(d->bias, 16) && (!d->gain || d->gain_group_stride % v == 0) &&
         (!d->bias || d->bias_group_stride % v == 0);
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
  A.D = (uint32_t)d->D;
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
  const bool vectors = vectors_ok(d->x, d->x_group_stride, d->x_row_stride, d->D, d->groups, d->rows, es) &&
                       params_vectors_ok(d) && aligned_to(y, 16);
  const NormShape S = norm_shape(d->D, d->dtype, vectors, false);
  for (int64_t g0 = 0; g0 < d->groups; g0 += kNormMaxGroups) {
    const int64_t ng = d->groups - g0 < kNormMaxGroups ? d->groups - g0 : kNormMaxGroups;
    NormArgs A = norm_args(d, g0);
    A.keep = d->rstd || d->groups * d->rows * d->D * (int64_t)es <= kKeepForward;
    A.out = (char*)y + g0 * d->rows * d->D * (int64_t)es;
    const int64_t gx = norm_blocks(S, d->groups, d->rows, false, false);
    launch_norm(A, S, d->dtype, dim3((unsigned)gx, (unsigned)ng), false, d->bias != nullptr, (hipStream_t)stream);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return (int)e;
  }
  return UNIRL_OK;
}

extern "C" size_t unirl_layer_norm_bwd_scratch_bytes(int64_t groups, int64_t rows, int64_t D) {
  if (groups <= 0 || rows <= 0 || D <= 0 || D > kNormMaxDim) return 0;
  // at least what norm_blocks gives for any layout of the operands
  const int64_t want = (kNormMaxBlocks + groups - 1) / groups;
  return (size_t)(groups * (want < rows ? want : rows) * D) * 2 * sizeof(float);
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
  if (params && per_group && d->groups > kNormMaxGroups) return UNIRL_E_LIMIT;  // norm_param_kernel's sets lie in gridDim.y
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
                         vectors_ok(dy, dy_group_stride, dy_row_stride, d->D, d->groups, d->rows, es) &&
                         params_vectors_ok(d) && aligned_to(dx, 16);
    const NormShape S = norm_shape(d->D, d->dtype, vectors, true);
    blocks = norm_blocks(S, d->groups, d->rows, true, dbias != nullptr);
    if (params) {
      if (!scratch || scratch_bytes < unirl_layer_norm_bwd_scratch_bytes(d->groups, d->rows, d->D))
        return UNIRL_E_WORKSPACE;
      if (!aligned_to(scratch, 16)) return UNIRL_E_ALIGN;
      // the launch's own partial rows, whatever the function above says
      if ((size_t)(d->groups * blocks * d->D) * (dbias ? 2 : 1) * sizeof(float) > scratch_bytes) return UNIRL_E_WORKSPACE;
    }
    if (!params && !dx) return UNIRL_OK;
    part_bias = d->groups * blocks * d->D;
    for (int64_t g0 = 0; g0 < d->groups; g0 += kNormMaxGroups) {
      const int64_t ng = d->groups - g0 < kNormMaxGroups ? d->groups - g0 : kNormMaxGroups;
      NormArgs A = norm_args(d, g0);
      A.keep = d->groups * d->rows * d->D * (int64_t)es <= kKeepBackward;
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
  const dim3 grid((unsigned)((d->D + 31) / 32), (unsigned)sets, dbias ? 2 : 1);
#define UNIRL_NORM_PARAM(O)                                                                                               \
  hipLaunchKernelGGL((norm_param_kernel<O>), grid, dim3(1024), 0, s, part, part_bias, n, (uint32_t)d->D, (O*)dgain, (O*)dbias)
  if (d->gain_dtype == UNIRL_F32)
    UNIRL_NORM_PARAM(float);
  else if (d->gain_dtype == UNIRL_BF16)
    UNIRL_NORM_PARAM(bf16_t);
  else
    UNIRL_NORM_PARAM(f16_t);
#undef UNIRL_NORM_PARAM
  return (int)hipGetLastError();
}
