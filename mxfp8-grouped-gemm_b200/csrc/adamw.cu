// One AdamW step over many tensors for sm_100a.
//
// The tensors are cut into chunks of MXG_ADAMW_CHUNK elements; a persistent
// grid walks the chunk table, a warp taking 256 elements at a time (8 a lane,
// the block that shares one scale of the 8-bit moments).  Bound by HBM: every
// array passes by once, in 16-byte accesses.
//
// The moments are rounded operation by operation (no fused multiply-adds), so
// that the 8-bit codes are a function of the inputs alone.
#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <cmath>

#include "mxg.h"
#include "mxg_device.cuh"
#include "mxg_internal.h"

namespace mxg {

constexpr int kAdamThreads = 256;
constexpr int kAdamTensors = 480;              // gradient addresses a launch carries (kernel arguments: 4 KB)
constexpr uint64_t kGradF32 = uint64_t(1) << 63;

struct AdamArgs {
  const mxg_adamw_tensor* tensors;
  const int32_t* chunks;
  int64_t chunk0, n_chunks;
  int tensor0;
  bool last;                                   // this launch raises the step
  void *m, *v;
  float *m_scale, *v_scale, *master;
  int64_t* step;
  int32_t* done;
  const float* lr_ptr;
  float lr, b1, c1, b2, c2, eps;
  double ln_b1, ln_b2;
  uint32_t seed_lo, seed_hi;
  uint64_t grads[kAdamTensors];
};

// Random bits: 32x32 -> 64-bit products by odd constants, the halves xored,
// two of them for each of (seed, step), block and element.  Means, spread and
// correlations of both halves, between neighbours, blocks and steps, are
// those of independent uniform draws to within sampling error.
constexpr uint32_t kM1 = 0x6A09C55Du, kM2 = 0x5D1B8E63u, kStep = 0x9E2F4D8Bu, kAdd = 0x3C7A15E9u;
__device__ __forceinline__ uint32_t mix(uint32_t x, uint32_t by) {
  const uint64_t p = uint64_t(x) * by;
  return uint32_t(p >> 32) ^ uint32_t(p);
}
__device__ __forceinline__ uint32_t step_key(uint32_t lo, uint32_t hi, uint32_t step) {
  uint32_t k = mix(lo + kAdd, kM1);
  k = mix(k ^ hi ^ kAdd, kM2);
  return mix(k + step + kStep, kM1);
}
__device__ __forceinline__ uint32_t block_key(uint32_t k, uint64_t block) {
  const uint32_t b = mix(k + uint32_t(block) + kAdd, kM1);
  return mix((b ^ uint32_t(block >> 32)) + kStep, kM2);
}
__device__ __forceinline__ uint32_t element_bits(uint32_t kb, uint32_t j) {
  return mix(mix((kb ^ (j * kStep)) + kAdd, kM1) ^ kStep, kM2);
}
__device__ __forceinline__ uint32_t more_bits(uint32_t h) { return mix(h ^ kAdd, kM1); }

// 8-bit codes: the bits of a float whose exponent field is small enough for
// the code to be its bits 20 and up; denormals continue the grid to 0.
__device__ __forceinline__ float decode_m(uint32_t c, float scale) {
  const float x = __uint_as_float((c & 127u) << 20) * 0x1p112f * scale;
  return (c & 128u) ? -x : x;
}
__device__ __forceinline__ float decode_v(uint32_t c, float scale) {
  return __uint_as_float(c << 20) * 0x1p96f * scale;
}
__device__ __forceinline__ uint32_t encode_m(float x, float inv, uint32_t noise) {
  const float y = fabsf(x) * inv * 0x1p-112f;
  const uint32_t c = min((__float_as_uint(y) + noise) >> 20, 127u);
  return c | (x < 0.0f ? 128u : 0u);
}
__device__ __forceinline__ uint32_t encode_v(float x, float inv, uint32_t noise) {
  const float y = x * inv * 0x1p-96f;
  const uint32_t c = min((__float_as_uint(y) + noise) >> 20, 255u);
  return max(c, x > 0.0f ? 1u : 0u);
}

__device__ __forceinline__ void load8(const float* p, float (&x)[8]) {
  const float4 a = *reinterpret_cast<const float4*>(p), b = *reinterpret_cast<const float4*>(p + 4);
  x[0] = a.x, x[1] = a.y, x[2] = a.z, x[3] = a.w, x[4] = b.x, x[5] = b.y, x[6] = b.z, x[7] = b.w;
}
__device__ __forceinline__ void store8(float* p, const float (&x)[8]) {
  *reinterpret_cast<float4*>(p) = make_float4(x[0], x[1], x[2], x[3]);
  *reinterpret_cast<float4*>(p + 4) = make_float4(x[4], x[5], x[6], x[7]);
}
__device__ __forceinline__ void load8(const __nv_bfloat16* p, float (&x)[8]) {
  const uint4 a = *reinterpret_cast<const uint4*>(p);
  const uint32_t w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
  for (int q = 0; q < 4; ++q) x[2 * q] = bf16_lo(w[q]), x[2 * q + 1] = bf16_hi(w[q]);
}
__device__ __forceinline__ void store8(__nv_bfloat16* p, const float (&x)[8]) {
  *reinterpret_cast<uint4*>(p) = make_uint4(pack2_bf16(x[0], x[1]), pack2_bf16(x[2], x[3]), pack2_bf16(x[4], x[5]),
                                            pack2_bf16(x[6], x[7]));
}
__device__ __forceinline__ float as_f32(float x) { return x; }
__device__ __forceinline__ float as_f32(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ void put(float* p, float x) { *p = x; }
__device__ __forceinline__ void put(__nv_bfloat16* p, float x) { *p = __float2bfloat16_rn(x); }

struct StepConsts {
  float keep_lr, step_size, rs2;  // lr, lr / (1 - b1^t), 1 / sqrt(1 - b2^t)
  uint32_t key;
};

// 256 elements (n of them real) at element i of a tensor, `at` of the moments.
template <typename P, typename G, bool MASTER, int BITS>
__device__ __forceinline__ void adamw_block(const AdamArgs& a, const StepConsts& k, P* param, const G* grad,
                                            float* master, int64_t at, int n, float keep, bool vec, int lane) {
  float p[8], g[8], m[8], v[8];
  const int e0 = lane * 8;
  const int mine = n - e0;  // real elements of this lane (any that is <= 0: none)
  if (vec && n >= 256) {
    load8(grad + e0, g);
    if constexpr (!MASTER) load8(param + e0, p);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      g[i] = i < mine ? as_f32(grad[e0 + i]) : 0.0f;
      if constexpr (!MASTER) p[i] = i < mine ? as_f32(param[e0 + i]) : 0.0f;
    }
  }
  if constexpr (MASTER) load8(master + e0, p);

  if constexpr (BITS == 32) {
    load8(static_cast<const float*>(a.m) + at + e0, m);
    load8(static_cast<const float*>(a.v) + at + e0, v);
  } else {
    const uint2 cm = *reinterpret_cast<const uint2*>(static_cast<const uint8_t*>(a.m) + at + e0);
    const uint2 cv = *reinterpret_cast<const uint2*>(static_cast<const uint8_t*>(a.v) + at + e0);
    const float sm = a.m_scale[at >> 8], sv = a.v_scale[at >> 8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      m[i] = decode_m(((i < 4 ? cm.x : cm.y) >> (8 * (i & 3))) & 255u, sm);
      v[i] = decode_v(((i < 4 ? cv.x : cv.y) >> (8 * (i & 3))) & 255u, sv);
    }
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    m[i] = __fadd_rn(__fmul_rn(m[i], a.b1), __fmul_rn(g[i], a.c1));
    v[i] = __fadd_rn(__fmul_rn(v[i], a.b2), __fmul_rn(__fmul_rn(g[i], g[i]), a.c2));
    const float down = fmaf(sqrtf(v[i]), k.rs2, a.eps);
    p[i] = fmaf(p[i], keep, -k.step_size * (m[i] / down));
  }
  uint32_t kb = 0;
  if constexpr (BITS == 8 || (!MASTER && sizeof(P) == 2)) kb = block_key(k.key, uint64_t(at) >> 8);
  uint32_t bits[8];
  if constexpr (BITS == 8 || (!MASTER && sizeof(P) == 2)) {
#pragma unroll
    for (int i = 0; i < 8; ++i) bits[i] = element_bits(kb, e0 + i);
  }

  if constexpr (BITS == 32) {
    store8(static_cast<float*>(a.m) + at + e0, m);
    store8(static_cast<float*>(a.v) + at + e0, v);
  } else {
    uint32_t bm = 0, bv = 0;  // bit patterns order as the sizes do; a NaN is the largest
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      bm = max(bm, __float_as_uint(m[i]) & 0x7FFFFFFFu);
      bv = max(bv, __float_as_uint(v[i]) & 0x7FFFFFFFu);
    }
    bm = max(__reduce_max_sync(0xffffffffu, bm), __float_as_uint(0x1p-100f));
    bv = max(__reduce_max_sync(0xffffffffu, bv), __float_as_uint(0x1p-100f));
    const float sm = __uint_as_float(bm), sv = __uint_as_float(bv);
    const float im = 1.0f / sm, iv = 1.0f / sv;
    uint32_t cm[2] = {0, 0}, cv[2] = {0, 0};
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      cm[i >> 2] |= encode_m(m[i], im, (bits[i] >> 16) << 4 | 8u) << (8 * (i & 3));
      cv[i >> 2] |= encode_v(v[i], iv, (bits[i] & 0xFFFFu) << 4 | 8u) << (8 * (i & 3));
    }
    *reinterpret_cast<uint2*>(static_cast<uint8_t*>(a.m) + at + e0) = make_uint2(cm[0], cm[1]);
    *reinterpret_cast<uint2*>(static_cast<uint8_t*>(a.v) + at + e0) = make_uint2(cv[0], cv[1]);
    if (lane == 0) {
      a.m_scale[at >> 8] = sm;
      a.v_scale[at >> 8] = sv;
    }
  }
  if constexpr (MASTER) {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (i >= mine) p[i] = 0.0f;  // the gap behind the tensor stays zero
    store8(master + e0, p);
  } else if constexpr (sizeof(P) == 2) {
    // stochastic: 16 random bits below the last one kept (never through NaN or infinity)
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (fabsf(p[i]) < INFINITY)
        p[i] = __uint_as_float((__float_as_uint(p[i]) + (more_bits(bits[i]) & 0xFFFFu)) & 0xFFFF0000u);
  }
  if (vec && n >= 256) {
    store8(param + e0, p);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (i < mine) put(param + e0 + i, p[i]);
  }
}

template <typename P, typename G, bool MASTER, int BITS>
__device__ __forceinline__ void adamw_chunk(const AdamArgs& a, const StepConsts& k, const mxg_adamw_tensor& t,
                                            uint64_t g, int64_t i0) {
  P* param = static_cast<P*>(t.param) + i0;
  const G* grad = reinterpret_cast<const G*>(g) + i0;
  float* master = MASTER ? a.master + t.master + i0 : nullptr;
  const int n = int(min(t.numel - i0, int64_t(MXG_ADAMW_CHUNK)));
  const bool vec = ((reinterpret_cast<uintptr_t>(param) | reinterpret_cast<uintptr_t>(grad)) & 15) == 0;
  const float keep = 1.0f - k.keep_lr * t.weight_decay;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  for (int b = warp * 256; b < n; b += kAdamThreads * 8)
    adamw_block<P, G, MASTER, BITS>(a, k, param + b, grad + b, MASTER ? master + b : nullptr, t.offset + i0 + b, n - b,
                                    keep, vec, lane);
}

template <int BITS>
__global__ void __launch_bounds__(kAdamThreads) adamw_kernel(const __grid_constant__ AdamArgs a) {
  __shared__ float s_bc[2];
  const int64_t t = *a.step + 1;
  // 1 - b^t = -expm1(t ln b): exact where b^t is close to 1
  if (threadIdx.x == 0) s_bc[0] = float(-expm1(double(t) * a.ln_b1));
  if (threadIdx.x == 32) s_bc[1] = float(-expm1(double(t) * a.ln_b2));
  __syncthreads();
  StepConsts k;
  k.keep_lr = a.lr_ptr ? *a.lr_ptr : a.lr;
  k.step_size = k.keep_lr / s_bc[0];
  k.rs2 = 1.0f / sqrtf(s_bc[1]);
  k.key = step_key(a.seed_lo, a.seed_hi, uint32_t(t));
  for (int64_t c = blockIdx.x; c < a.n_chunks; c += gridDim.x) {
    const int ti = a.chunks[a.chunk0 + c];
    const mxg_adamw_tensor& T = a.tensors[ti];
    const uint64_t tagged = a.grads[ti - a.tensor0];
    if (tagged == 0) continue;
    const uint64_t g = tagged & ~kGradF32;
    const bool f32 = tagged & kGradF32;
    const int64_t i0 = (a.chunk0 + c - T.first_chunk) * MXG_ADAMW_CHUNK;
    switch (T.kind) {
      case MXG_ADAMW_F32:
        if (f32) adamw_chunk<float, float, false, BITS>(a, k, T, g, i0);
        else adamw_chunk<float, __nv_bfloat16, false, BITS>(a, k, T, g, i0);
        break;
      case MXG_ADAMW_BF16_MASTER:
        if (f32) adamw_chunk<__nv_bfloat16, float, true, BITS>(a, k, T, g, i0);
        else adamw_chunk<__nv_bfloat16, __nv_bfloat16, true, BITS>(a, k, T, g, i0);
        break;
      default:
        if (f32) adamw_chunk<__nv_bfloat16, float, false, BITS>(a, k, T, g, i0);
        else adamw_chunk<__nv_bfloat16, __nv_bfloat16, false, BITS>(a, k, T, g, i0);
    }
  }
  // every block has read the step by the time the last one is done
  __syncthreads();
  if (threadIdx.x == 0) {
    __threadfence();
    if (atomicAdd(a.done, 1) == int(gridDim.x) - 1) {
      *a.done = 0;
      if (a.last) *a.step = t;
    }
  }
}

__global__ void __launch_bounds__(256) adamw_moments_kernel(const uint2* __restrict__ m, const uint2* __restrict__ v,
                                                            const float* __restrict__ m_scale,
                                                            const float* __restrict__ v_scale, int64_t n,
                                                            float* __restrict__ m_out, float* __restrict__ v_out) {
  const int64_t stride = int64_t(gridDim.x) * blockDim.x;
  for (int64_t i = int64_t(blockIdx.x) * blockDim.x + threadIdx.x; i < n / 8; i += stride) {
    const uint2 cm = __ldcs(m + i), cv = __ldcs(v + i);
    const float sm = m_scale[i >> 5], sv = v_scale[i >> 5];
    float x[8], y[8];
#pragma unroll
    for (int q = 0; q < 8; ++q) {
      x[q] = decode_m(((q < 4 ? cm.x : cm.y) >> (8 * (q & 3))) & 255u, sm);
      y[q] = decode_v(((q < 4 ? cv.x : cv.y) >> (8 * (q & 3))) & 255u, sv);
    }
    store8(m_out + i * 8, x);
    store8(v_out + i * 8, y);
  }
}

}  // namespace mxg

using namespace mxg;

extern "C" int mxg_adamw_step(const mxg_adamw_tensor* tensors, int n_tensors, const int32_t* chunks,
                              const int64_t* chunk_begin, const uint64_t* grads, const int32_t* grad_dtypes,
                              int state_bits, void* exp_avg, void* exp_avg_sq, float* exp_avg_scale,
                              float* exp_avg_sq_scale, float* master, int64_t* step, int32_t* done, double lr,
                              const float* lr_ptr, double beta1, double beta2, double eps, uint64_t seed,
                              void* stream) {
  if (n_tensors < 1 || !tensors || !chunks || !chunk_begin || !grads || !grad_dtypes || !exp_avg || !exp_avg_sq ||
      !step || !done || (state_bits != 8 && state_bits != 32))
    return MXG_ERR_INVALID_ARGUMENT;
  if (state_bits == 8 && (!exp_avg_scale || !exp_avg_sq_scale)) return MXG_ERR_INVALID_ARGUMENT;
  if (!(lr >= 0.0) || !(beta1 >= 0.0 && beta1 < 1.0) || !(beta2 >= 0.0 && beta2 < 1.0) || !(eps >= 0.0))
    return MXG_ERR_INVALID_ARGUMENT;
  for (int i = 0; i < n_tensors; ++i) {
    if (chunk_begin[i] < 0 || chunk_begin[i + 1] < chunk_begin[i]) return MXG_ERR_INVALID_ARGUMENT;
    if (grads[i] && grad_dtypes[i] != MXG_DTYPE_BF16 && grad_dtypes[i] != MXG_DTYPE_F32)
      return MXG_ERR_INVALID_ARGUMENT;
    if (grads[i] & kGradF32 || grads[i] % (grad_dtypes[i] == MXG_DTYPE_F32 ? 4 : 2)) return MXG_ERR_MISALIGNED;
  }
  if (!aligned16(exp_avg) || !aligned16(exp_avg_sq) || !aligned16(master)) return MXG_ERR_MISALIGNED;
  int st = check_device();
  if (st) return st;
  AdamArgs a;
  a.tensors = tensors, a.chunks = chunks;
  a.m = exp_avg, a.v = exp_avg_sq, a.m_scale = exp_avg_scale, a.v_scale = exp_avg_sq_scale, a.master = master;
  a.step = step, a.done = done, a.lr_ptr = lr_ptr;
  a.lr = float(lr), a.b1 = float(beta1), a.c1 = float(1.0 - beta1), a.b2 = float(beta2), a.c2 = float(1.0 - beta2);
  a.eps = float(eps);
  a.ln_b1 = std::log(beta1), a.ln_b2 = std::log(beta2);
  a.seed_lo = uint32_t(seed), a.seed_hi = uint32_t(seed >> 32);
  int per_sm = 0;
  auto* kernel = state_bits == 8 ? adamw_kernel<8> : adamw_kernel<32>;
  if (cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per_sm, kernel, kAdamThreads, 0) != cudaSuccess || per_sm < 1)
    return MXG_ERR_CUDA;
  for (int t0 = 0; t0 < n_tensors; t0 += kAdamTensors) {
    const int t1 = std::min(n_tensors, t0 + kAdamTensors);
    a.tensor0 = t0, a.last = t1 == n_tensors;
    a.chunk0 = chunk_begin[t0], a.n_chunks = chunk_begin[t1] - chunk_begin[t0];
    for (int i = t0; i < t1; ++i)
      a.grads[i - t0] = grads[i] ? grads[i] | (grad_dtypes[i] == MXG_DTYPE_F32 ? kGradF32 : 0) : 0;
    const int64_t blocks = std::max<int64_t>(1, std::min<int64_t>(a.n_chunks, int64_t(num_sms()) * per_sm));
    kernel<<<unsigned(blocks), kAdamThreads, 0, (cudaStream_t)stream>>>(a);
    if (cudaGetLastError() != cudaSuccess) return MXG_ERR_CUDA;
  }
  return MXG_OK;
}

extern "C" int mxg_adamw_moments(const void* exp_avg, const void* exp_avg_sq, const float* exp_avg_scale,
                                 const float* exp_avg_sq_scale, int64_t n, float* exp_avg_out, float* exp_avg_sq_out,
                                 void* stream) {
  if (n < 0) return MXG_ERR_INVALID_ARGUMENT;
  if (n % MXG_ADAMW_BLOCK) return MXG_ERR_BAD_SHAPE;
  if (n == 0) return MXG_OK;
  if (!exp_avg || !exp_avg_sq || !exp_avg_scale || !exp_avg_sq_scale || !exp_avg_out || !exp_avg_sq_out)
    return MXG_ERR_INVALID_ARGUMENT;
  if (!aligned16(exp_avg) || !aligned16(exp_avg_sq) || !aligned16(exp_avg_out) || !aligned16(exp_avg_sq_out))
    return MXG_ERR_MISALIGNED;
  int st = check_device();
  if (st) return st;
  const int64_t want = (n / 8 + 255) / 256;
  adamw_moments_kernel<<<unsigned(std::min<int64_t>(want, int64_t(num_sms()) * 16)), 256, 0, (cudaStream_t)stream>>>(
      static_cast<const uint2*>(exp_avg), static_cast<const uint2*>(exp_avg_sq), exp_avg_scale, exp_avg_sq_scale, n,
      exp_avg_out, exp_avg_sq_out);
  return cuda_status(cudaGetLastError());
}
