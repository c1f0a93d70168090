// The optimizer's side of a policy update over many tensors at once: the global norm of the
// gradients and the AdamW step with its moments in 32 bits or in 8.
//
// Tables of tensors ride in the kernel arguments (50 to 160 tensors a launch, under 4 KB), so a call
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
// gradient.  Bound by reading: 400 M bf16 elements in 117 us (6.8 TB/s).  Small lists are bound by the
// launch (160 tensors of 5 M elements together 7 us); two loads a lane in flight suit both (one: 8.5, four:
// 7.7, eight: 9.1 us for the small list, whose code is fetched anew by every launch).
template <typename T, bool ALIGNED>
__device__ __forceinline__ double thread_sumsq(const T* p, int64_t n) {
  constexpr int VEC = ALIGNED ? 16 / (int)sizeof(T) : 1;
  constexpr int U = 2;  // loads in flight per lane
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
constexpr int kAdamThreads = 256;
constexpr int kQuantBlock = 256;  // elements that share a scale: one wavefront's four elements a lane
// Blocks of one wavefront, whose loads are in flight together.  With 32-bit moments one block is enough
// (eight wavefronts a SIMD keep the memory busy) and the shorter code is fetched sooner: a launch over 1.6 M
// elements takes 10.2 us with one block, 10.4 with two, 11.3 with four, one over 400 M 2.02, 2.10, 2.06 ms.
// With 8-bit moments: 9.3 / 9.6 / 11.3 us and 1.20 / 1.14 / 1.16 ms.
constexpr int adam_unroll(int bits) { return bits == 32 ? 1 : 2; }
constexpr int64_t kMaxGrid = 0xffffff;  // workgroups of 256 threads: a launch counts its threads in 32 bits
constexpr int adam_chunk(int bits) { return kAdamThreads / kWave * adam_unroll(bits) * kQuantBlock; }

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

// A tensor's entry holds what its kind of step reads, so that as many as possible share a launch: 90
// (32-bit moments) to 52 (8-bit moments and a master).
struct AdamMaster {
  float* master;
};
struct AdamBytes {
  uint8_t *exp_avg_scale, *exp_avg_sq_scale;
  int64_t index_base;
};
template <int>
struct Nothing {};
template <int BITS, bool MASTER>
struct AdamEntry : std::conditional<MASTER, AdamMaster, Nothing<0>>::type, std::conditional<BITS == 8, AdamBytes, Nothing<1>>::type {
  void* param;
  const void* grad;
  void* exp_avg;
  void* exp_avg_sq;
  int64_t numel2;  // twice the number of elements; odd: every pointer suits the vector accesses
};
struct AdamCommon {
  const AdamControl* control;
  const float* norm;
  AdamControl host;
  float max_norm, beta1, beta2, one_minus_beta1, one_minus_beta2, eps;
  int skip_nonfinite;
};
template <int BITS, bool MASTER>
struct AdamArgs : AdamCommon {
  static constexpr int kTensors = (4096 - 96) / (int)(sizeof(AdamEntry<BITS, MASTER>) + 4) / 2 * 2;
  uint32_t first[kTensors];  // first workgroup of each tensor; above the grid's size behind the last
  AdamEntry<BITS, MASTER> t[kTensors];
};
static_assert(sizeof(AdamArgs<32, false>) <= 4096 && sizeof(AdamArgs<32, true>) <= 4096 && sizeof(AdamArgs<8, false>) <= 4096 &&
                  sizeof(AdamArgs<8, true>) <= 4096,
              "kernel arguments");

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

  __device__ __forceinline__ void update(const AdamCommon& A, const AdamControl& C) {
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

// Where one wavefront's elements lie and how its lanes reach them: four adjacent elements in one access,
// or element by element through buffer descriptors that end with the tensor (loads behind the end give
// zeros, stores there are dropped), so that neither stands behind a condition.
template <typename T, bool VECTORS>
struct Span {
  T* p;
  __amdgpu_buffer_rsrc_t r;
  __device__ __forceinline__ Span(const void* base, int64_t e0, uint32_t count) : p((T*)base + e0) {
    if constexpr (!VECTORS) r = __builtin_amdgcn_make_buffer_rsrc(p, 0, count * (uint32_t)sizeof(T), 0x00020000);
  }
  __device__ __forceinline__ void load(uint32_t i, float (&o)[4]) const {
    if constexpr (VECTORS) {
      Vec<T, 4>::load(p + i, o);
    } else {
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        if constexpr (sizeof(T) == 4) {
          o[k] = __uint_as_float(__builtin_amdgcn_raw_buffer_load_b32(r, (i + k) * 4, 0, 0));
        } else {
          T t;
          t.bits = (uint16_t)__builtin_amdgcn_raw_buffer_load_b16(r, (i + k) * 2, 0, 0);
          o[k] = Elem<T>::load(&t);
        }
      }
    }
  }
  __device__ __forceinline__ void store(uint32_t i, const float (&o)[4]) const {
    if constexpr (VECTORS && sizeof(T) == 4) {
      Vec<T, 4>::store(p + i, o);
    } else if constexpr (VECTORS) {  // streaming like the other flows (cached: 2.05 instead of 1.98 ms below)
      u32x2 w;
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        if constexpr (std::is_same<T, bf16_t>::value)
          w[k] = f32x2_to_bf16x2_bits(o[2 * k], o[2 * k + 1]);
        else
          w[k] = f32_to_f16_bits(o[2 * k]) | (f32_to_f16_bits(o[2 * k + 1]) << 16);
      }
      __builtin_nontemporal_store(w, reinterpret_cast<u32x2*>(p + i));
    } else {
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        if constexpr (sizeof(T) == 4) {
          __builtin_amdgcn_raw_buffer_store_b32(__float_as_uint(o[k]), r, (i + k) * 4, 0, 0);
        } else {
          T t;
          Elem<T>::store(&t, o[k]);
          __builtin_amdgcn_raw_buffer_store_b16((short)t.bits, r, (i + k) * 2, 0, 0);
        }
      }
    }
  }
};
template <bool VECTORS>
struct Span<uint8_t, VECTORS> {
  uint8_t* p;
  __amdgpu_buffer_rsrc_t r;
  __device__ __forceinline__ Span(const void* base, int64_t e0, uint32_t count) : p((uint8_t*)base + e0) {
    if constexpr (!VECTORS) r = __builtin_amdgcn_make_buffer_rsrc(p, 0, count, 0x00020000);
  }
  __device__ __forceinline__ uint32_t load(uint32_t i) const {
    if constexpr (VECTORS) return __builtin_nontemporal_load((const uint32_t*)(p + i));
    uint32_t w = 0;
#pragma unroll
    for (int k = 0; k < 4; ++k) w |= (uint32_t)(uint8_t)__builtin_amdgcn_raw_buffer_load_b8(r, i + k, 0, 0) << (8 * k);
    return w;
  }
  __device__ __forceinline__ void store(uint32_t i, uint32_t w) const {
    if constexpr (VECTORS) {
      __builtin_nontemporal_store(w, (uint32_t*)(p + i));
    } else {
#pragma unroll
      for (int k = 0; k < 4; ++k) __builtin_amdgcn_raw_buffer_store_b8((char)(w >> (8 * k)), r, i + k, 0, 0);
    }
  }
};

// One wavefront's blocks of 256 elements from e0 on: all their loads are in flight before the first
// is used.  `count` of the elements exist (VECTORS: all).
template <typename P, typename G, int BITS, bool MASTER, bool VECTORS>
__device__ __forceinline__ void adamw_blocks(const AdamCommon& A, const AdamControl& C, const AdamEntry<BITS, MASTER>& T, int64_t e0,
                                             uint32_t count, uint32_t lane) {
  constexpr int kUnroll = adam_unroll(BITS);
  const Span<P, VECTORS> param(T.param, e0, count);
  const Span<G, VECTORS> grad(T.grad, e0, count);
  const void* master_base = T.param;
  if constexpr (MASTER) master_base = T.master;
  const Span<float, VECTORS> master(master_base, e0, count);
  using S = typename std::conditional<BITS == 32, float, uint8_t>::type;
  const Span<S, VECTORS> avg(T.exp_avg, e0, count), sq(T.exp_avg_sq, e0, count);
  const int64_t block0 = e0 / kQuantBlock;
  AdamLane<P, G, BITS, MASTER> L[kUnroll];
  uint32_t cm[kUnroll], cv[kUnroll], sm[kUnroll], sv[kUnroll];
#pragma unroll
  for (int u = 0; u < kUnroll; ++u) {
    const uint32_t i = u * kQuantBlock + lane * 4;
    grad.load(i, L[u].g);
    if constexpr (MASTER)
      master.load(i, L[u].p);
    else
      param.load(i, L[u].p);
    if constexpr (BITS == 32) {
      avg.load(i, L[u].m);
      sq.load(i, L[u].v);
    } else {
      cm[u] = avg.load(i);
      cv[u] = sq.load(i);
      const int64_t block = block0 + (VECTORS || u * kQuantBlock < count ? u : 0);  // one that exists
      sm[u] = T.exp_avg_scale[block];
      sv[u] = T.exp_avg_sq_scale[block];
    }
  }
#pragma unroll
  for (int u = 0; u < kUnroll; ++u) {
    if (!VECTORS && u * kQuantBlock >= count) break;
    const uint32_t i = u * kQuantBlock + lane * 4;
    if constexpr (BITS == 8) {
      decode_m4(cm[u], scale_of(sm[u]), L[u].m);
      decode_v4(cv[u], scale_of(sv[u]), L[u].v);
    }
    L[u].update(A, C);
    if constexpr (MASTER) master.store(i, L[u].p);
    param.store(i, L[u].p);
    if constexpr (BITS == 32) {
      avg.store(i, L[u].m);
      sq.store(i, L[u].v);
    } else {
      // what lies behind the tensor's end stays out of the block's maximum, whatever the clip factor is
      if constexpr (!VECTORS)
#pragma unroll
        for (int k = 0; k < 4; ++k)
          if (i + k >= count) L[u].m[k] = L[u].v[k] = 0.0f;
      const uint64_t index = (uint64_t)T.index_base + (uint64_t)e0 + i;
      uint32_t wm, wv, km, kv;
      L[u].encode((uint32_t)index, C.key + (uint32_t)(index >> 32) * 0x9E3779B9u, wm, wv, km, kv);
      avg.store(i, wm);
      sq.store(i, wv);
      if (lane == 0) {
        T.exp_avg_scale[block0 + u] = (uint8_t)km;
        T.exp_avg_sq_scale[block0 + u] = (uint8_t)kv;
      }
    }
  }
}

// Bound by HBM: 28 bytes an element with 32-bit moments and a master, 16 with 8-bit moments and a master
// (10 without).  400 M bf16 elements with masters: 1.98 ms and 1.13 ms, 5.7 TB/s, the rate of a copy on this
// card; streaming accesses (cached ones: 2.10 ms), workgroups in address order (a range of its own for each
// XCD: the same).  A lane takes four elements of a block, so that a block's maximum is one
// reduction inside a wavefront.
template <typename P, typename G, int BITS, bool MASTER>
__global__ __launch_bounds__(kAdamThreads) void adamw_kernel(AdamArgs<BITS, MASTER> A) {
  AdamControl C = A.host;
  if (A.control) {
    C = *A.control;
  } else if (A.norm) {
    const float norm = *A.norm;
    C.clip = clip_factor(norm, A.max_norm);
    C.skip = A.skip_nonfinite && !finite_f32(norm);
  }
  if (C.skip) return;
  constexpr int kElements = adam_unroll(BITS) * kQuantBlock;  // of one wavefront
  const int t = find_tensor<AdamArgs<BITS, MASTER>::kTensors>(A.first, blockIdx.x);
  const AdamEntry<BITS, MASTER>& T = A.t[t];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const uint32_t lane = threadIdx.x & (kWave - 1);
  const int64_t e0 = (int64_t)(blockIdx.x - A.first[t]) * adam_chunk(BITS) + (int64_t)wave * kElements;
  const int64_t left = (T.numel2 >> 1) - e0;
  if (left <= 0) return;
  if ((T.numel2 & 1) && left >= kElements)
    adamw_blocks<P, G, BITS, MASTER, true>(A, C, T, e0, kElements, lane);
  else
    adamw_blocks<P, G, BITS, MASTER, false>(A, C, T, e0, left < kElements ? (uint32_t)left : kElements, lane);
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

// The values that 8-bit moments stand for: eight elements a lane (a lane's stores are 16 bytes in 16-bit
// types), kMomentsRounds times; blockIdx.y: m, v.  Bound by HBM: 400 M elements to bf16 in 394 us (6.1 TB/s).
constexpr int kMomentsRounds = 2;
constexpr int kMomentsChunk = 256 * 8 * kMomentsRounds;
template <typename O>
__global__ __launch_bounds__(256) void adamw_moments_kernel(const uint8_t* m, const uint8_t* v, const uint8_t* sm,
                                                            const uint8_t* sv, int64_t n, O* out_m, O* out_v, int aligned) {
  const bool second = blockIdx.y != 0;
  const uint8_t *codes = second ? v : m, *scales = second ? sv : sm;
  O* out = second ? out_v : out_m;
  if (!out) return;
  const auto decode = [second](uint32_t w, float scale, float (&o)[4]) {
    if (second)
      decode_v4(w, scale, o);
    else
      decode_m4(w, scale, o);
  };
  for (int64_t e0 = (int64_t)blockIdx.x * kMomentsChunk; e0 < n; e0 += (int64_t)gridDim.x * kMomentsChunk) {
    if (aligned && e0 + kMomentsChunk <= n) {
      u32x2 w[kMomentsRounds];
      uint32_t s[kMomentsRounds];
#pragma unroll
      for (int u = 0; u < kMomentsRounds; ++u) {
        const int64_t i = e0 + u * 2048 + threadIdx.x * 8;
        w[u] = stream_load8(codes + i);
        s[u] = scales[i / kQuantBlock];
      }
#pragma unroll
      for (int u = 0; u < kMomentsRounds; ++u) {
        float lo[4], hi[4], o[8];
        decode(w[u].x, scale_of(s[u]), lo);
        decode(w[u].y, scale_of(s[u]), hi);
#pragma unroll
        for (int k = 0; k < 4; ++k) o[k] = lo[k], o[4 + k] = hi[k];
        Vec<O, 8>::store(out + e0 + u * 2048 + threadIdx.x * 8, o);
      }
    } else {
      for (int u = 0; u < kMomentsRounds; ++u) {
        const int64_t i = e0 + u * 2048 + threadIdx.x * 8;
        if (i >= n) break;
        const float scale = scale_of(scales[i / kQuantBlock]);
        float o[4];
        if (aligned && i + 8 <= n) {
          const u32x2 w = stream_load8(codes + i);
          decode(w.x, scale, o);
          Vec<O, 4>::store(out + i, o);
          decode(w.y, scale, o);
          Vec<O, 4>::store(out + i + 4, o);
          continue;
        }
        for (int k = 0; k < 8 && i + k < n; ++k) {
          decode(codes[i + k], scale, o);
          Elem<O>::store(out + i + k, o[0]);
        }
      }
    }
  }
}

// One launch after another over the tensors of a checked call.
template <typename P, typename G, int BITS, bool MASTER>
static int launch_adamw(const AdamCommon& common, const struct unirl_adamw_tensor* tensors, int64_t n, hipStream_t s) {
  using Args = AdamArgs<BITS, MASTER>;
  constexpr size_t kState = BITS == 32 ? 4 : 1;
  Args A;
  memset(&A, 0, sizeof(A));
  static_cast<AdamCommon&>(A) = common;
  for (int64_t i = 0; i < n;) {
    int k = 0;
    int64_t grid = 0;
    for (; i < n && k < Args::kTensors; ++i) {
      const struct unirl_adamw_tensor& T = tensors[i];
      if (T.numel == 0) continue;
      const int64_t blocks = (T.numel + adam_chunk(BITS) - 1) / adam_chunk(BITS);
      if (grid + blocks > kMaxGrid) break;  // the next launch takes it
      const bool vectors = aligned_to(T.param, 4 * sizeof(P)) && aligned_to(T.grad, 4 * sizeof(G)) &&
                           aligned_to(T.exp_avg, 4 * kState) && aligned_to(T.exp_avg_sq, 4 * kState) &&
                           (!MASTER || aligned_to(T.master, 16));
      auto& E = A.t[k];
      E.param = T.param;
      E.grad = T.grad;
      E.exp_avg = T.exp_avg;
      E.exp_avg_sq = T.exp_avg_sq;
      E.numel2 = 2 * T.numel + vectors;
      if constexpr (MASTER) E.master = T.master;
      if constexpr (BITS == 8) {
        E.exp_avg_scale = T.exp_avg_scale;
        E.exp_avg_sq_scale = T.exp_avg_sq_scale;
        E.index_base = T.index_base;
      }
      A.first[k++] = (uint32_t)grid;
      grid += blocks;
    }
    if (k == 0) break;
    for (int j = k; j < Args::kTensors; ++j) A.first[j] = 0xffffffffu;
    hipLaunchKernelGGL((adamw_kernel<P, G, BITS, MASTER>), dim3((unsigned)grid), dim3(kAdamThreads), 0, s, A);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return (int)e;
  }
  return UNIRL_OK;
}
template <typename P, typename G>
static int launch_adamw(const AdamCommon& c, const struct unirl_adamw_params* q, const struct unirl_adamw_tensor* t, int64_t n,
                        hipStream_t s) {
  if constexpr (!std::is_same<P, float>::value) {  // an fp32 parameter is its own master
    if (q->use_master) return q->state_bits == 32 ? launch_adamw<P, G, 32, true>(c, t, n, s) : launch_adamw<P, G, 8, true>(c, t, n, s);
  }
  return q->state_bits == 32 ? launch_adamw<P, G, 32, false>(c, t, n, s) : launch_adamw<P, G, 8, false>(c, t, n, s);
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
    if (T.numel > adam_chunk(q->state_bits) * kMaxGrid) return UNIRL_E_LIMIT;
  }
  AdamCommon A;
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
  hipStream_t s = (hipStream_t)stream;
  if (q->param_dtype == UNIRL_F32) return launch_adamw<float, float>(A, q, tensors, n_tensors, s);
  if (q->param_dtype == UNIRL_BF16)
    return q->grad_dtype == UNIRL_BF16 ? launch_adamw<bf16_t, bf16_t>(A, q, tensors, n_tensors, s)
                                       : launch_adamw<bf16_t, float>(A, q, tensors, n_tensors, s);
  return q->grad_dtype == UNIRL_F16 ? launch_adamw<f16_t, f16_t>(A, q, tensors, n_tensors, s)
                                    : launch_adamw<f16_t, float>(A, q, tensors, n_tensors, s);
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
  int64_t grid = (numel + kMomentsChunk - 1) / kMomentsChunk;
  if (grid > kMaxGrid) grid = kMaxGrid;
  const int aligned = aligned_to(exp_avg, 8) && aligned_to(exp_avg_sq, 8) && aligned_to(out_exp_avg, 16) &&
                      aligned_to(out_exp_avg_sq, 16);
#define UNIRL_MOMENTS(O)                                                                                            \
  hipLaunchKernelGGL((adamw_moments_kernel<O>), dim3((unsigned)grid, 2), dim3(256), 0, (hipStream_t)stream,            \
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
