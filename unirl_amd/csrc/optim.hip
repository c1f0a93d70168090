// The optimizer's side of a policy update over many tensors at once: the global norm of the
// gradients and the AdamW step with its moments in 32 bits or in 8.
//
// Tables of tensors ride in the kernel arguments (48 or 160 tensors a launch, under 4 KB), so a call
// copies nothing to the device, keeps nothing between calls and can be captured into a graph.
// Workgroup b finds its tensor by comparing b with the tensors' first workgroups, one per lane, and
// counting the lanes that are not beyond it: one load and a ballot instead of a search.
#include <math.h>
#include <string.h>

#include "common_hip.h"
#include "unirl_internal.h"

namespace unirl {

// ---------------------------------------------------------------------------
// Global norm
// ---------------------------------------------------------------------------
constexpr int kGradNormTensors = 160;
constexpr int kGradNormThreads = 256;
constexpr int64_t kGradNormMinChunk = 8192;  // elements of one workgroup at least
constexpr int64_t kGradNormMaxTensors = kPartialCapacity / 2;

struct GradNormTensor {
  const void* p;
  int64_t n;
};
struct GradNormArgs {
  GradNormTensor t[kGradNormTensors];
  uint32_t first[kGradNormTensors];  // first workgroup of each tensor; the grid's size beyond the last
  uint8_t kind[kGradNormTensors];    // dtype | 4 when 16-byte aligned
  int64_t chunk;
  double* partials;
};

// Which of `count` (<= 192) ascending entries of `first` is the last that is not beyond `b`.
template <int COUNT>
__device__ __forceinline__ int find_tensor(const uint32_t* first, uint32_t b) {
  const int lane = threadIdx.x & (kWave - 1);
  int t = -1;
#pragma unroll
  for (int k = 0; k < COUNT; k += kWave) {
    const int i = k + lane;
    const bool in = i < COUNT && first[i < COUNT ? i : COUNT - 1] <= b;
    t += __popcll(__ballot(in));
  }
  return __builtin_amdgcn_readfirstlane(t);
}

// Sum of squares of [p, p + n) over the workgroup's threads, one value per thread.  The squares are
// formed and added in fp64: exact for every fp32 product, no overflow or underflow for any finite
// gradient.
template <typename T, bool ALIGNED>
__device__ __forceinline__ double thread_sumsq(const T* p, int64_t n) {
  constexpr int VEC = ALIGNED ? 16 / (int)sizeof(T) : 1;
  constexpr int U = 4;  // 16-byte loads in flight per lane
  double a[2] = {0.0, 0.0};
  const int64_t step = (int64_t)kGradNormThreads * VEC;
  int64_t i = (int64_t)threadIdx.x * VEC;
  for (; i + (U - 1) * step + VEC <= n; i += U * step) {
    float x[U][VEC];
#pragma unroll
    for (int u = 0; u < U; ++u) Vec<T, VEC>::load(p + i + u * step, x[u]);
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int k = 0; k < VEC; ++k) a[k & 1] = fma((double)x[u][k], (double)x[u][k], a[k & 1]);
  }
  for (; i + VEC <= n; i += step) {
    float x[VEC];
    Vec<T, VEC>::load(p + i, x);
#pragma unroll
    for (int k = 0; k < VEC; ++k) a[k & 1] = fma((double)x[k], (double)x[k], a[k & 1]);
  }
  for (; i < n; ++i) {  // fewer than VEC elements, of one lane
    const double x = (double)Elem<T>::load(p + i);
    a[0] = fma(x, x, a[0]);
  }
  return a[0] + a[1];
}

__global__ __launch_bounds__(kGradNormThreads) void grad_norm_kernel(GradNormArgs A) {
  __shared__ double lds[kGradNormThreads / kWave];
  const int t = find_tensor<kGradNormTensors>(A.first, blockIdx.x);
  const int64_t off = (int64_t)(blockIdx.x - A.first[t]) * A.chunk;
  const int64_t left = A.t[t].n - off;
  const int64_t n = left < A.chunk ? left : A.chunk;
  const int kind = A.kind[t];
  double s;
  switch (kind) {
    case UNIRL_F32 | 4: s = thread_sumsq<float, true>((const float*)A.t[t].p + off, n); break;
    case UNIRL_BF16 | 4: s = thread_sumsq<bf16_t, true>((const bf16_t*)A.t[t].p + off, n); break;
    case UNIRL_F16 | 4: s = thread_sumsq<f16_t, true>((const f16_t*)A.t[t].p + off, n); break;
    case UNIRL_F32: s = thread_sumsq<float, false>((const float*)A.t[t].p + off, n); break;
    case UNIRL_BF16: s = thread_sumsq<bf16_t, false>((const bf16_t*)A.t[t].p + off, n); break;
    default: s = thread_sumsq<f16_t, false>((const f16_t*)A.t[t].p + off, n); break;
  }
  s = block_sum(s, lds);
  if (threadIdx.x == 0) A.partials[blockIdx.x] = s;
}

// The partials in a fixed order, then the root.
__global__ __launch_bounds__(1024) void grad_norm_finish_kernel(const double* partials, int64_t n, float* out) {
  __shared__ double lds[1024 / kWave];
  double s = 0.0;
  for (int64_t i = threadIdx.x; i < n; i += 1024) s += partials[i];
  s = block_sum(s, lds);
  if (threadIdx.x == 0) *out = (float)sqrt(s);
}

// ---------------------------------------------------------------------------
// AdamW
// ---------------------------------------------------------------------------
constexpr int kAdamTensors = 48;
constexpr int kAdamThreads = 256;
constexpr int kQuantBlock = 256;  // elements that share a scale: one wavefront's four elements a lane
constexpr int kAdamUnroll = 4;    // blocks of one wavefront
constexpr int64_t kMaxGrid = 0xffffff;  // workgroups of 256 threads: a launch counts its threads in 32 bits
constexpr int kAdamChunk = kAdamThreads / kWave * kAdamUnroll * kQuantBlock;

// The scalars of one step, as the kernels read them (the first fields of the caller's control buffer).
struct AdamControl {
  float decay;       // 1 - lr * weight_decay
  float step_size;   // lr / (1 - beta1^t)
  float rsqrt_bc2;   // 1 / sqrt(1 - beta2^t)
  float clip;        // factor of the gradients
  uint32_t key;      // of the dither
  uint32_t skip;     // nothing is to be written
};
static_assert(sizeof(AdamControl) <= UNIRL_ADAMW_CONTROL_BYTES, "control buffer");

struct AdamArgs {
  struct unirl_adamw_tensor t[kAdamTensors];
  uint32_t first[kAdamTensors];
  uint64_t aligned;  // bit per tensor: every pointer suits the vector accesses
  const AdamControl* control;
  const float* norm;
  AdamControl host;
  float max_norm, beta1, beta2, one_minus_beta1, one_minus_beta2, eps;
  int skip_nonfinite;
};
static_assert(sizeof(AdamArgs) <= 4096, "kernel arguments");

// A bijection of 32-bit words whose output bits each depend on all input bits: xor-shifts and odd
// products, with the fractions of sqrt(2) and sqrt(3) as constants (flipping any input bit flips each
// output bit with a probability of 0.5 +- 0.006 over 65 536 samples, which is that count's own noise).
__host__ __device__ __forceinline__ uint32_t mix32(uint32_t x) {
  x ^= x >> 16;
  x *= 0x6A09E667u;
  x ^= x >> 15;
  x *= 0xBB67AE85u;
  return x ^ (x >> 16);
}
__host__ __device__ __forceinline__ uint32_t dither_key(uint32_t seed, int64_t step) {
  return mix32(seed + (uint32_t)step * 0x9E3779B9u);
}

// min(1, max_norm / (norm + 1e-6)); NaN stays NaN, an infinite norm gives 0.
__device__ __forceinline__ float clip_factor(float norm, float max_norm) {
  const float c = max_norm / (norm + 1e-6f);
  return c > 1.0f ? 1.0f : c;
}
__device__ __forceinline__ bool finite_f32(float x) { return (__float_as_uint(x) & 0x7f800000u) != 0x7f800000u; }

// --- moments in 8 bits ---
// m: e4m3 (sign, 4 exponent bits, 3 mantissa bits) times 2^(scale - 127); v: the upper 8 bits of a
// positive half (5 exponent bits, 3 mantissa bits) times 2^(scale - 127); one scale per block.  The
// scale is the power of two that brings the block's largest finite value into [2^7, 2^8) / [2^14, 2^15).
//
// Rounding is stochastic: with x between two codes, the upper one is taken with the probability
// that makes the expected value x.  A moving average with weights (0.999, 0.001) moves by less
// than half a code step (2^-4 of the value) in almost every step; rounding to nearest would put it
// back each time and freeze the moment.  16 random bits per value leave a bias of 2^-17 steps.
__device__ __forceinline__ float scale_of(uint32_t byte) { return __uint_as_float(byte << 23); }

// Code of a >= 0, finite: bias B of the exponent, unit 2^-S of the subnormals.
template <int B, int S>
__device__ __forceinline__ uint32_t encode3(float a, uint32_t u16) {
  const uint32_t normal = (__float_as_uint(a) + (u16 << 4) - ((uint32_t)(127 - B) << 23)) >> 20;
  const uint32_t sub = (uint32_t)(a * (float)(1 << S) + (float)u16 * 1.52587890625e-05f);
  return a < 1.0f / (float)(1 << (B - 1)) ? sub : normal;
}

typedef unsigned short u16x2 __attribute__((ext_vector_type(2)));
__device__ __forceinline__ uint32_t pk_max_u16(uint32_t a, uint32_t b) {
  union {
    uint32_t u;
    u16x2 v;
  } x, y;
  x.u = a;
  y.u = b;
  x.v = __builtin_elementwise_max(x.v, y.v);
  return x.u;
}
__device__ __forceinline__ uint32_t wave_pk_max_u16(uint32_t v) {
  UNIRL_DPP_REDUCE(v, pk_max_u16, dpp_u32_or_zero)
  return last_lane(v);
}


// One lane's four consecutive elements of one block, in registers.
template <typename P, typename G, int BITS, bool MASTER>
struct AdamLane {
  float p[4], g[4], m[4], v[4];

  __device__ __forceinline__ void update(const AdamArgs& A, const AdamControl& C) {
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const float gc = g[k] * C.clip;
      m[k] = A.beta1 * m[k] + A.one_minus_beta1 * gc;
      v[k] = A.beta2 * v[k] + A.one_minus_beta2 * (gc * gc);
      const float denom = sqrtf(v[k]) * C.rsqrt_bc2 + A.eps;
      p[k] = p[k] * C.decay - C.step_size * (m[k] / denom);
    }
  }

  // The block's scales and this lane's codes from its m and v.
  __device__ __forceinline__ void encode(uint32_t index, uint32_t key, uint32_t& codes_m, uint32_t& codes_v,
                                         uint32_t& scale_m, uint32_t& scale_v) const {
    uint32_t top = 0;  // largest biased exponents: m in the lower half, v in the upper
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const uint32_t em = finite_f32(m[k]) ? (__float_as_uint(m[k]) >> 23) & 0xffu : 0u;
      const uint32_t ev = finite_f32(v[k]) ? (__float_as_uint(v[k]) >> 23) & 0xffu : 0u;
      top = pk_max_u16(top, em | (ev << 16));
    }
    top = wave_pk_max_u16(top);
    const int em = (int)(top & 0xffffu) - 7, ev = (int)(top >> 16) - 14;
    scale_m = (uint32_t)(em > 1 ? em : 1);
    scale_v = (uint32_t)(ev > 1 ? ev : 1);
    const float inv_m = scale_of(254u - scale_m), inv_v = scale_of(254u - scale_v);
    codes_m = codes_v = 0;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const uint32_t h = mix32((index + k) ^ key);
      const uint32_t bits = __float_as_uint(m[k]);
      uint32_t cm = encode3<7, 9>(fabsf(m[k]) * inv_m, h & 0xffffu) | ((bits >> 24) & 0x80u);
      if (!finite_f32(m[k])) cm = 0x7fu;  // NaN: the format has no infinity
      uint32_t cv = encode3<15, 17>(v[k] * inv_v, h >> 16);
      // a positive second moment never becomes zero: the next step would divide by eps alone
      if (v[k] > 0.0f && cv == 0u) cv = 1u;
      if (!finite_f32(v[k])) cv = v[k] != v[k] ? 0xffu : 0xf8u;
      codes_m |= cm << (8 * k);
      codes_v |= cv << (8 * k);
    }
  }
};

__device__ __forceinline__ void decode_m4(uint32_t codes, float scale, float (&o)[4]) {
  typedef float f32x2 __attribute__((ext_vector_type(2)));
  const f32x2 lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)codes, false);
  const f32x2 hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)codes, true);
  o[0] = lo.x * scale;
  o[1] = lo.y * scale;
  o[2] = hi.x * scale;
  o[3] = hi.y * scale;
}
__device__ __forceinline__ void decode_v4(uint32_t codes, float scale, float (&o)[4]) {
#pragma unroll
  for (int k = 0; k < 4; ++k) o[k] = f16_bits_to_f32(((codes >> (8 * k)) & 0xffu) << 7) * scale;
}

// Bound by HBM: 28 bytes an element with 32-bit moments and a master, 10 with 8-bit moments and a
// 16-bit parameter.  One wavefront takes four blocks of 256 elements, four elements a lane, so that
// all loads of 1024 elements are in flight before the first is used; a block's maximum is then one
// reduction inside a wavefront.
template <typename P, typename G, int BITS, bool MASTER>
__global__ __launch_bounds__(kAdamThreads) void adamw_kernel(AdamArgs A) {
  AdamControl C = A.host;
  if (A.control) {
    C = *A.control;
  } else if (A.norm) {
    const float norm = *A.norm;
    C.clip = clip_factor(norm, A.max_norm);
    C.skip = A.skip_nonfinite && !finite_f32(norm);
  }
  if (C.skip) return;
  const int t = find_tensor<kAdamTensors>(A.first, blockIdx.x);
  const struct unirl_adamw_tensor& T = A.t[t];
  const int64_t n = T.numel;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int lane = threadIdx.x & (kWave - 1);
  const int64_t e0 = (int64_t)(blockIdx.x - A.first[t]) * kAdamChunk + (int64_t)wave * (kAdamUnroll * kQuantBlock);
  if (e0 >= n) return;
  P* param = (P*)T.param;
  const G* grad = (const G*)T.grad;
  float* master = (float*)T.master;
  using Lane = AdamLane<P, G, BITS, MASTER>;

  if (((A.aligned >> t) & 1) && e0 + kAdamUnroll * kQuantBlock <= n) {
    Lane L[kAdamUnroll];
    uint32_t cm[kAdamUnroll], cv[kAdamUnroll], sm[kAdamUnroll], sv[kAdamUnroll];
#pragma unroll
    for (int u = 0; u < kAdamUnroll; ++u) {
      const int64_t i = e0 + u * kQuantBlock + lane * 4;
      Vec<G, 4>::load(grad + i, L[u].g);
      if constexpr (MASTER)
        Vec<float, 4>::load(master + i, L[u].p);
      else
        Vec<P, 4>::load(param + i, L[u].p);
      if constexpr (BITS == 32) {
        Vec<float, 4>::load((const float*)T.exp_avg + i, L[u].m);
        Vec<float, 4>::load((const float*)T.exp_avg_sq + i, L[u].v);
      } else {
        cm[u] = __builtin_nontemporal_load((const uint32_t*)((const uint8_t*)T.exp_avg + i));
        cv[u] = __builtin_nontemporal_load((const uint32_t*)((const uint8_t*)T.exp_avg_sq + i));
        sm[u] = T.exp_avg_scale[e0 / kQuantBlock + u];
        sv[u] = T.exp_avg_sq_scale[e0 / kQuantBlock + u];
      }
    }
#pragma unroll
    for (int u = 0; u < kAdamUnroll; ++u) {
      const int64_t i = e0 + u * kQuantBlock + lane * 4;
      if constexpr (BITS == 8) {
        decode_m4(cm[u], scale_of(sm[u]), L[u].m);
        decode_v4(cv[u], scale_of(sv[u]), L[u].v);
      }
      L[u].update(A, C);
      if constexpr (MASTER) Vec<float, 4>::store(master + i, L[u].p);
      Vec<P, 4>::store(param + i, L[u].p);
      if constexpr (BITS == 32) {
        Vec<float, 4>::store((float*)T.exp_avg + i, L[u].m);
        Vec<float, 4>::store((float*)T.exp_avg_sq + i, L[u].v);
      } else {
        const uint64_t index = (uint64_t)T.index_base + (uint64_t)i;
        uint32_t wm, wv, km, kv;
        L[u].encode((uint32_t)index, C.key + (uint32_t)(index >> 32) * 0x9E3779B9u, wm, wv, km, kv);
        __builtin_nontemporal_store(wm, (uint32_t*)((uint8_t*)T.exp_avg + i));
        __builtin_nontemporal_store(wv, (uint32_t*)((uint8_t*)T.exp_avg_sq + i));
        if (lane == 0) {
          T.exp_avg_scale[e0 / kQuantBlock + u] = (uint8_t)km;
          T.exp_avg_sq_scale[e0 / kQuantBlock + u] = (uint8_t)kv;
        }
      }
    }
    return;
  }

  // element by element: a tensor's last blocks, and tensors whose pointers do not suit the vectors
  for (int u = 0; u < kAdamUnroll; ++u) {
    const int64_t b = e0 + u * kQuantBlock;
    if (b >= n) break;
    const int64_t i = b + lane * 4;
    Lane L;
    float sm = 0.0f, sv = 0.0f;
    if constexpr (BITS == 8) {
      sm = scale_of(T.exp_avg_scale[b / kQuantBlock]);
      sv = scale_of(T.exp_avg_sq_scale[b / kQuantBlock]);
    }
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const bool in = i + k < n;
      L.g[k] = in ? Elem<G>::load(grad + i + k) : 0.0f;
      if constexpr (MASTER)
        L.p[k] = in ? master[i + k] : 0.0f;
      else
        L.p[k] = in ? Elem<P>::load(param + i + k) : 0.0f;
      if constexpr (BITS == 32) {
        L.m[k] = in ? ((const float*)T.exp_avg)[i + k] : 0.0f;
        L.v[k] = in ? ((const float*)T.exp_avg_sq)[i + k] : 0.0f;
      } else {
        float om[4], ov[4];
        decode_m4(in ? ((const uint8_t*)T.exp_avg)[i + k] : 0u, sm, om);
        decode_v4(in ? ((const uint8_t*)T.exp_avg_sq)[i + k] : 0u, sv, ov);
        L.m[k] = om[0];
        L.v[k] = ov[0];
      }
    }
    L.update(A, C);
    uint32_t wm = 0, wv = 0, km = 0, kv = 0;
    if constexpr (BITS == 8) {
      // what lies behind the tensor's end stays out of the block's maximum, whatever the clip factor is
#pragma unroll
      for (int k = 0; k < 4; ++k)
        if (i + k >= n) L.m[k] = L.v[k] = 0.0f;
      const uint64_t index = (uint64_t)T.index_base + (uint64_t)i;
      L.encode((uint32_t)index, C.key + (uint32_t)(index >> 32) * 0x9E3779B9u, wm, wv, km, kv);
      if (lane == 0) {
        T.exp_avg_scale[b / kQuantBlock] = (uint8_t)km;
        T.exp_avg_sq_scale[b / kQuantBlock] = (uint8_t)kv;
      }
    }
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      if (i + k >= n) continue;
      if constexpr (MASTER) master[i + k] = L.p[k];
      Elem<P>::store(param + i + k, L.p[k]);
      if constexpr (BITS == 32) {
        ((float*)T.exp_avg)[i + k] = L.m[k];
        ((float*)T.exp_avg_sq)[i + k] = L.v[k];
      } else {
        ((uint8_t*)T.exp_avg)[i + k] = (uint8_t)(wm >> (8 * k));
        ((uint8_t*)T.exp_avg_sq)[i + k] = (uint8_t)(wv >> (8 * k));
      }
    }
  }
}

struct AdamScalars {
  double lr, beta1, beta2, weight_decay;
  uint32_t seed;
};
__host__ __device__ __forceinline__ AdamControl control_of(const AdamScalars& S, int64_t step) {
  AdamControl C;
  C.decay = (float)(1.0 - S.lr * S.weight_decay);
  C.step_size = (float)(S.lr / (1.0 - pow(S.beta1, (double)step)));
  C.rsqrt_bc2 = (float)(1.0 / sqrt(1.0 - pow(S.beta2, (double)step)));
  C.clip = 1.0f;
  C.key = dither_key(S.seed, step);
  C.skip = 0u;
  return C;
}

// One thread: the next step's number and scalars, on the device, so that a captured step counts on.
__global__ void adamw_advance_kernel(int64_t* step, AdamControl* control, AdamScalars S, const float* lr,
                                     const float* norm, float max_norm, int skip_nonfinite) {
  float factor = 1.0f;
  bool skip = false;
  if (norm) {
    const float x = *norm;
    if (max_norm >= 0.0f) factor = clip_factor(x, max_norm);
    skip = skip_nonfinite && !finite_f32(x);
  }
  if (lr) S.lr = (double)*lr;
  const int64_t t = *step + 1;
  AdamControl C = control_of(S, t);
  C.clip = factor;
  C.skip = skip ? 1u : 0u;
  *control = C;
  if (!skip) *step = t;
}

// The values that 8-bit moments stand for: four elements a lane, one block a wavefront.
template <typename O>
__global__ __launch_bounds__(256) void adamw_moments_kernel(const uint8_t* m, const uint8_t* v, const uint8_t* sm,
                                                            const uint8_t* sv, int64_t n, O* out_m, O* out_v, int aligned) {
  for (int64_t block = (int64_t)blockIdx.x * 4 + threadIdx.x / kWave; block * kQuantBlock < n; block += (int64_t)gridDim.x * 4)
#pragma unroll
  for (int which = 0; which < 2; ++which) {
    const int64_t i = block * kQuantBlock + (threadIdx.x & (kWave - 1)) * 4;
    const uint8_t* c = which ? v : m;
    O* out = which ? out_v : out_m;
    if (!out) continue;
    const float scale = scale_of((which ? sv : sm)[block]);
    float o[4];
    if (aligned && i + 4 <= n) {
      const uint32_t codes = __builtin_nontemporal_load((const uint32_t*)(c + i));
      if (which)
        decode_v4(codes, scale, o);
      else
        decode_m4(codes, scale, o);
      Vec<O, 4>::store(out + i, o);
    } else {
      for (int k = 0; k < 4 && i + k < n; ++k) {
        if (which)
          decode_v4(c[i + k], scale, o);
        else
          decode_m4(c[i + k], scale, o);
        Elem<O>::store(out + i + k, o[0]);
      }
    }
  }
}

template <typename P, typename G, int BITS>
static void launch_adamw(const AdamArgs& A, bool master, unsigned grid, hipStream_t s) {
  if constexpr (!std::is_same<P, float>::value) {  // an fp32 parameter is its own master
    if (master) {
      hipLaunchKernelGGL((adamw_kernel<P, G, BITS, true>), dim3(grid), dim3(kAdamThreads), 0, s, A);
      return;
    }
  }
  hipLaunchKernelGGL((adamw_kernel<P, G, BITS, false>), dim3(grid), dim3(kAdamThreads), 0, s, A);
}
template <typename P, typename G>
static void launch_adamw(const AdamArgs& A, int bits, bool master, unsigned grid, hipStream_t s) {
  if (bits == 32)
    launch_adamw<P, G, 32>(A, master, grid, s);
  else
    launch_adamw<P, G, 8>(A, master, grid, s);
}

}  // namespace unirl

using namespace unirl;

extern "C" int unirl_grad_norm(const void* const* grads, const int64_t* numels, const int* dtypes, int64_t n_tensors,
                               float* norm, void* workspace, size_t workspace_bytes, void* stream) {
  if (n_tensors < 0) return UNIRL_E_SHAPE;
  if (!norm || (n_tensors > 0 && (!grads || !numels || !dtypes))) return UNIRL_E_NULL;
  if (!aligned_to(norm, 4)) return UNIRL_E_ALIGN;
  if (n_tensors > kGradNormMaxTensors) return UNIRL_E_LIMIT;
  int64_t total = 0;
  for (int64_t i = 0; i < n_tensors; ++i) {
    if (!dtype_ok(dtypes[i])) return UNIRL_E_DTYPE;
    if (numels[i] < 0) return UNIRL_E_SHAPE;
    if (numels[i] > 0 && !grads[i]) return UNIRL_E_NULL;
    if (!aligned_to(grads[i], dtype_size(dtypes[i]))) return UNIRL_E_ALIGN;
    if (numels[i] > INT64_MAX / 4 - total) return UNIRL_E_LIMIT;
    total += numels[i];
  }
  if (!workspace || workspace_bytes < kWorkspaceBytes) return UNIRL_E_WORKSPACE;
  if (!aligned_to(workspace, 16)) return UNIRL_E_ALIGN;
  // about 8192 workgroups for large gradients (32 a compute unit), and at most one partial more per tensor
  const int64_t chunk = (total / 8192 / kGradNormMinChunk + 1) * kGradNormMinChunk;
  double* partials = ws_partials(workspace);
  int64_t done = 0;
  for (int64_t i = 0; i < n_tensors;) {
    GradNormArgs A;
    memset(&A, 0, sizeof(A));
    int k = 0;
    int64_t grid = 0;
    for (; i < n_tensors && k < kGradNormTensors; ++i) {
      if (numels[i] == 0) continue;
      A.t[k].p = grads[i];
      A.t[k].n = numels[i];
      A.first[k] = (uint32_t)grid;
      A.kind[k] = (uint8_t)(dtypes[i] | (aligned_to(grads[i], 16) ? 4 : 0));
      grid += (numels[i] + chunk - 1) / chunk;
      ++k;
    }
    if (k == 0) break;
    for (int j = k; j < kGradNormTensors; ++j) A.first[j] = 0xffffffffu;
    A.chunk = chunk;
    A.partials = partials + done;
    hipLaunchKernelGGL(grad_norm_kernel, dim3((unsigned)grid), dim3(kGradNormThreads), 0, (hipStream_t)stream, A);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return (int)e;
    done += grid;
  }
  hipLaunchKernelGGL(grad_norm_finish_kernel, dim3(1), dim3(1024), 0, (hipStream_t)stream, partials, done, norm);
  return (int)hipGetLastError();
}

extern "C" int unirl_adamw_advance(int64_t* step, void* control, double lr, const float* lr_ptr, double beta1,
                                   double beta2, double weight_decay, uint32_t seed, const float* grad_norm,
                                   float max_norm, int skip_nonfinite, void* stream) {
  if (!step || !control) return UNIRL_E_NULL;
  if (!aligned_to(step, 8) || !aligned_to(control, 4) || !aligned_to(lr_ptr, 4) || !aligned_to(grad_norm, 4))
    return UNIRL_E_ALIGN;
  if (!(beta1 >= 0.0 && beta1 < 1.0) || !(beta2 >= 0.0 && beta2 < 1.0)) return UNIRL_E_SHAPE;
  const AdamScalars S = {lr, beta1, beta2, weight_decay, seed};
  hipLaunchKernelGGL(adamw_advance_kernel, dim3(1), dim3(1), 0, (hipStream_t)stream, step, (AdamControl*)control, S,
                     lr_ptr, grad_norm, max_norm, skip_nonfinite);
  return (int)hipGetLastError();
}

extern "C" int unirl_adamw_step(const struct unirl_adamw_tensor* tensors, int64_t n_tensors,
                                const struct unirl_adamw_params* q, void* stream) {
  if (!q || (n_tensors > 0 && !tensors)) return UNIRL_E_NULL;
  if (n_tensors < 0) return UNIRL_E_SHAPE;
  if (!dtype_ok(q->param_dtype) || !dtype_ok(q->grad_dtype)) return UNIRL_E_DTYPE;
  if (q->grad_dtype != q->param_dtype && q->grad_dtype != UNIRL_F32) return UNIRL_E_DTYPE;
  if (q->state_bits != 8 && q->state_bits != 32) return UNIRL_E_DTYPE;
  if (q->use_master && q->param_dtype == UNIRL_F32) return UNIRL_E_DTYPE;
  if (!q->control && q->step < 1) return UNIRL_E_SHAPE;
  if (!(q->beta1 >= 0.0 && q->beta1 < 1.0) || !(q->beta2 >= 0.0 && q->beta2 < 1.0)) return UNIRL_E_SHAPE;
  if (!aligned_to(q->grad_norm, 4) || !aligned_to(q->control, 4)) return UNIRL_E_ALIGN;
  const size_t ps = dtype_size(q->param_dtype), gs = dtype_size(q->grad_dtype);
  const size_t ss = q->state_bits == 32 ? 4 : 1;
  for (int64_t i = 0; i < n_tensors; ++i) {
    const struct unirl_adamw_tensor& T = tensors[i];
    if (T.numel < 0 || T.index_base < 0) return UNIRL_E_SHAPE;
    if (T.numel == 0) continue;
    if (!T.param || !T.grad || !T.exp_avg || !T.exp_avg_sq) return UNIRL_E_NULL;
    if (q->use_master && !T.master) return UNIRL_E_NULL;
    if (q->state_bits == 8 && (!T.exp_avg_scale || !T.exp_avg_sq_scale)) return UNIRL_E_NULL;
    if (T.index_base % kQuantBlock != 0) return UNIRL_E_ALIGN;
    if (!aligned_to(T.param, ps) || !aligned_to(T.grad, gs) || !aligned_to(T.exp_avg, ss) ||
        !aligned_to(T.exp_avg_sq, ss) || !aligned_to(T.master, 4))
      return UNIRL_E_ALIGN;
    if (T.numel > kAdamChunk * kMaxGrid) return UNIRL_E_LIMIT;
  }
  AdamArgs A;
  memset(&A, 0, sizeof(A));
  A.control = (const AdamControl*)q->control;
  A.norm = q->max_norm >= 0.0f || q->skip_nonfinite ? q->grad_norm : nullptr;
  // without a bound the norm only decides whether the step is taken: an infinite bound makes the factor 1
  A.max_norm = q->max_norm >= 0.0f ? q->max_norm : INFINITY;
  A.skip_nonfinite = q->skip_nonfinite;
  A.beta1 = (float)q->beta1;
  A.beta2 = (float)q->beta2;
  A.one_minus_beta1 = (float)(1.0 - q->beta1);
  A.one_minus_beta2 = (float)(1.0 - q->beta2);
  A.eps = (float)q->eps;
  if (!A.control) {
    const AdamScalars S = {q->lr, q->beta1, q->beta2, q->weight_decay, q->seed};
    A.host = control_of(S, q->step);
  }
  for (int64_t i = 0; i < n_tensors;) {
    int k = 0;
    int64_t grid = 0;
    A.aligned = 0;
    for (; i < n_tensors && k < kAdamTensors; ++i) {
      const struct unirl_adamw_tensor& T = tensors[i];
      if (T.numel == 0) continue;
      const int64_t blocks = (T.numel + kAdamChunk - 1) / kAdamChunk;
      if (grid + blocks > kMaxGrid) break;  // the next launch takes it
      A.t[k] = T;
      A.first[k] = (uint32_t)grid;
      if (aligned_to(T.param, 4 * ps) && aligned_to(T.grad, 4 * gs) && aligned_to(T.exp_avg, 4 * ss) &&
          aligned_to(T.exp_avg_sq, 4 * ss) && aligned_to(T.master, 16))
        A.aligned |= 1ull << k;
      grid += blocks;
      ++k;
    }
    if (k == 0) break;
    for (int j = k; j < kAdamTensors; ++j) A.first[j] = 0xffffffffu;
    hipStream_t s = (hipStream_t)stream;
    const bool master = q->use_master != 0;
    if (q->param_dtype == UNIRL_F32)
      launch_adamw<float, float>(A, q->state_bits, false, (unsigned)grid, s);
    else if (q->param_dtype == UNIRL_BF16 && q->grad_dtype == UNIRL_BF16)
      launch_adamw<bf16_t, bf16_t>(A, q->state_bits, master, (unsigned)grid, s);
    else if (q->param_dtype == UNIRL_BF16)
      launch_adamw<bf16_t, float>(A, q->state_bits, master, (unsigned)grid, s);
    else if (q->grad_dtype == UNIRL_F16)
      launch_adamw<f16_t, f16_t>(A, q->state_bits, master, (unsigned)grid, s);
    else
      launch_adamw<f16_t, float>(A, q->state_bits, master, (unsigned)grid, s);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return (int)e;
  }
  return UNIRL_OK;
}

extern "C" int unirl_adamw_moments(const void* exp_avg, const void* exp_avg_sq, const uint8_t* exp_avg_scale,
                                   const uint8_t* exp_avg_sq_scale, int64_t numel, void* out_exp_avg,
                                   void* out_exp_avg_sq, int out_dtype, void* stream) {
  if (numel < 0) return UNIRL_E_SHAPE;
  if (!dtype_ok(out_dtype)) return UNIRL_E_DTYPE;
  if (numel == 0 || (!out_exp_avg && !out_exp_avg_sq)) return UNIRL_OK;
  if ((out_exp_avg && (!exp_avg || !exp_avg_scale)) || (out_exp_avg_sq && (!exp_avg_sq || !exp_avg_sq_scale)))
    return UNIRL_E_NULL;
  const size_t os = dtype_size(out_dtype);
  if (!aligned_to(out_exp_avg, os) || !aligned_to(out_exp_avg_sq, os)) return UNIRL_E_ALIGN;
  int64_t grid = (numel + 4 * kQuantBlock - 1) / (4 * kQuantBlock);
  if (grid > kMaxGrid) grid = kMaxGrid;
  const int aligned = aligned_to(exp_avg, 4) && aligned_to(exp_avg_sq, 4) && aligned_to(out_exp_avg, 4 * os) &&
                      aligned_to(out_exp_avg_sq, 4 * os);
#define UNIRL_MOMENTS(O)                                                                                            \
  hipLaunchKernelGGL((adamw_moments_kernel<O>), dim3((unsigned)grid), dim3(256), 0, (hipStream_t)stream,            \
                     (const uint8_t*)exp_avg, (const uint8_t*)exp_avg_sq, exp_avg_scale, exp_avg_sq_scale, numel, \
                     (O*)out_exp_avg, (O*)out_exp_avg_sq, aligned)
  if (out_dtype == UNIRL_F32)
    UNIRL_MOMENTS(float);
  else if (out_dtype == UNIRL_BF16)
    UNIRL_MOMENTS(bf16_t);
  else
    UNIRL_MOMENTS(f16_t);
#undef UNIRL_MOMENTS
  return (int)hipGetLastError();
}
