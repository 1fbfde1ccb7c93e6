// One AdamW step over many tensors for sm_100a.
//
// The tensors are cut into chunks of MXG_ADAMW_CHUNK elements; every block takes
// an equal run of the chunk table, a warp 256 elements at a time (8 a lane, the
// block that shares one scale of the 8-bit moments).  Bound by HBM: every
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

// 8-bit codes are bits 20 and up of a float whose exponent field is small
// enough (denormals continue the grid to 0).  The first moment's are e4m3 codes
// (times 2^-8), which the conversion instruction decodes two at a time; the
// second's become floats as they are.  A scale of 2^30 and more, whose product
// with 2^96 would overflow, takes two products (the same value).
__device__ __forceinline__ void decode_m(uint32_t codes, float scale, float (&x)[8], int at) {
  const float by = scale * 0x1p-8f;
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const __half2_raw r =
        __nv_cvt_fp8x2_to_halfraw2(__nv_fp8x2_storage_t(h ? codes >> 16 : codes & 0xFFFFu), __NV_E4M3);
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&r));
    x[at + 2 * h] = f.x * by;
    x[at + 2 * h + 1] = f.y * by;
  }
}
__device__ __forceinline__ void decode_v(uint32_t codes, float scale, float (&x)[8], int at) {
  const bool big = scale >= 0x1p30f;
  const float by = big ? 0x1p96f : scale * 0x1p96f, more = big ? scale : 1.0f;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t u = i < 3 ? codes << (20 - 8 * i) : codes >> 4;
    x[at + i] = __uint_as_float(u & 0x0FF00000u) * by;
  }
  if (big) {
#pragma unroll
    for (int i = 0; i < 4; ++i) x[at + i] *= more;
  }
}
// The code as the top byte, sign apart; noise: 16 random bits, in bits 8 to 23.
// (A NaN or infinity spills over, into a block whose scale is one too.)  The
// two products are spelled out: nvcc 12.9 at -O3 drops what follows a plain
// product by 2^-112 here and yields codes of 0.
__device__ __forceinline__ uint32_t encode_m(float x, float inv, uint32_t noise) {
  const uint32_t t = __float_as_uint(__fmul_rn(__fmul_rn(fabsf(x), inv), 0x1p-112f)) * 16u + noise;
  return (t & 0x7FFFFFFFu) | (__float_as_uint(x) & 0x80000000u);
}
__device__ __forceinline__ uint32_t encode_v(float x, float inv, uint32_t noise) {
  const uint32_t t = __float_as_uint(__fmul_rn(__fmul_rn(x, inv), 0x1p-96f)) * 16u + noise;
  return x > 0.0f ? max(t, 1u << 24) : t;
}
__device__ __forceinline__ uint32_t top_bytes(uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  return __byte_perm(__byte_perm(a, b, 0x0073), __byte_perm(c, d, 0x0073), 0x5410);
}
__device__ __forceinline__ float max_nan(float a, float b) {
  float m;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(m) : "f"(a), "f"(b));
  return m;
}
__device__ __forceinline__ float warp_max_nan(float x) {
  float m;
  asm("redux.sync.max.NaN.f32 %0, %1, 0xffffffff;" : "=f"(m) : "f"(x));
  return m;
}

// A lane's 8 of a block's 256 values: four at 4 * lane and four at 128 + 4 *
// lane, so that every access of a warp to an fp32 array covers whole lines
// (8 in a row, two 16-byte stores into each 32-byte sector: 4.4, not 6 TB/s).
__device__ __forceinline__ int place(int lane, int i) { return lane * 4 + (i & 3) + (i >> 2) * 128; }
__device__ __forceinline__ void load8(const float* p, int lane, float (&x)[8]) {
  const float4 a = *reinterpret_cast<const float4*>(p + lane * 4), b = *reinterpret_cast<const float4*>(p + 128 + lane * 4);
  x[0] = a.x, x[1] = a.y, x[2] = a.z, x[3] = a.w, x[4] = b.x, x[5] = b.y, x[6] = b.z, x[7] = b.w;
}
__device__ __forceinline__ void store8(float* p, int lane, const float (&x)[8]) {
  *reinterpret_cast<float4*>(p + lane * 4) = make_float4(x[0], x[1], x[2], x[3]);
  *reinterpret_cast<float4*>(p + 128 + lane * 4) = make_float4(x[4], x[5], x[6], x[7]);
}
__device__ __forceinline__ void load8(const __nv_bfloat16* p, int lane, float (&x)[8]) {
  const uint2 a = *reinterpret_cast<const uint2*>(p + lane * 4), b = *reinterpret_cast<const uint2*>(p + 128 + lane * 4);
  const uint32_t w[4] = {a.x, a.y, b.x, b.y};
#pragma unroll
  for (int q = 0; q < 4; ++q) x[2 * q] = bf16_lo(w[q]), x[2 * q + 1] = bf16_hi(w[q]);
}
__device__ __forceinline__ void store_words(__nv_bfloat16* p, int lane, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  *reinterpret_cast<uint2*>(p + lane * 4) = make_uint2(a, b);
  *reinterpret_cast<uint2*>(p + 128 + lane * 4) = make_uint2(c, d);
}
__device__ __forceinline__ void store8(__nv_bfloat16* p, int lane, const float (&x)[8]) {
  store_words(p, lane, pack2_bf16(x[0], x[1]), pack2_bf16(x[2], x[3]), pack2_bf16(x[4], x[5]), pack2_bf16(x[6], x[7]));
}
__device__ __forceinline__ uint2 load_codes(const uint8_t* p, int lane) {
  return make_uint2(*reinterpret_cast<const uint32_t*>(p + lane * 4), *reinterpret_cast<const uint32_t*>(p + 128 + lane * 4));
}
__device__ __forceinline__ void store_codes(uint8_t* p, int lane, uint32_t a, uint32_t b) {
  *reinterpret_cast<uint32_t*>(p + lane * 4) = a;
  *reinterpret_cast<uint32_t*>(p + 128 + lane * 4) = b;
}
__device__ __forceinline__ float as_f32(float x) { return x; }
__device__ __forceinline__ float as_f32(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ void put(float* p, float x) { *p = x; }
__device__ __forceinline__ void put(__nv_bfloat16* p, float x) { *p = __float2bfloat16_rn(x); }

__device__ __forceinline__ float sqrt_fast(float x) {
  float y;
  asm("sqrt.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float rcp_fast(float x) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

struct StepConsts {
  float lr, step_size, rs2;  // lr, lr / (1 - b1^t), 1 / sqrt(1 - b2^t)
  uint32_t key;
};

// 256 elements (n of them real) at element i of a tensor, `at` of the moments.
template <typename P, typename G, bool MASTER, int BITS>
__device__ __forceinline__ void adamw_block(const AdamArgs& a, const StepConsts& k, P* param, const G* grad,
                                            float* master, int64_t at, int n, float keep, bool vec, int lane) {
  float p[8], g[8], m[8], v[8];
  if (vec && n >= 256) {
    load8(grad, lane, g);
    if constexpr (!MASTER) load8(param, lane, p);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int e = place(lane, i);
      g[i] = e < n ? as_f32(grad[e]) : 0.0f;
      if constexpr (!MASTER) p[i] = e < n ? as_f32(param[e]) : 0.0f;
    }
  }
  if constexpr (MASTER) load8(master, lane, p);

  if constexpr (BITS == 32) {
    load8(static_cast<const float*>(a.m) + at, lane, m);
    load8(static_cast<const float*>(a.v) + at, lane, v);
  } else {
    const uint2 cm = load_codes(static_cast<const uint8_t*>(a.m) + at, lane);
    const uint2 cv = load_codes(static_cast<const uint8_t*>(a.v) + at, lane);
    const float sm = a.m_scale[at >> 8], sv = a.v_scale[at >> 8];
    decode_m(cm.x, sm, m, 0), decode_m(cm.y, sm, m, 4);
    decode_v(cv.x, sv, v, 0), decode_v(cv.y, sv, v, 4);
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    m[i] = __fadd_rn(__fmul_rn(m[i], a.b1), __fmul_rn(g[i], a.c1));
    v[i] = __fadd_rn(__fmul_rn(v[i], a.b2), __fmul_rn(__fmul_rn(g[i], g[i]), a.c2));
    // the update alone goes through the approximate root and reciprocal
    // (2 units of the last place; a v under 2^-126 counts as 0 beside eps)
    p[i] = fmaf(p[i], keep, -k.step_size * (m[i] * rcp_fast(fmaf(sqrt_fast(v[i]), k.rs2, a.eps))));
  }
  constexpr bool kStochastic = !MASTER && sizeof(P) == 2;
  uint32_t bits[8];
  if constexpr (BITS == 8 || kStochastic) {
    const uint32_t kb = block_key(k.key, uint64_t(at) >> 8);
#pragma unroll
    for (int i = 0; i < 8; ++i) bits[i] = element_bits(kb, place(lane, i));
  }

  if constexpr (BITS == 32) {
    store8(static_cast<float*>(a.m) + at, lane, m);
    store8(static_cast<float*>(a.v) + at, lane, v);
  } else {
    float sm = fabsf(m[0]), sv = v[0];  // of the block: a NaN if there is one
#pragma unroll
    for (int i = 1; i < 8; ++i) sm = max_nan(sm, fabsf(m[i])), sv = max_nan(sv, v[i]);
    sm = max_nan(warp_max_nan(sm), 0x1p-100f), sv = max_nan(warp_max_nan(sv), 0x1p-100f);
    const float im = 1.0f / sm, iv = 1.0f / sv;
    uint32_t c[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) c[i] = encode_m(m[i], im, __byte_perm(bits[i], 0x80u, 0x5324));
    store_codes(static_cast<uint8_t*>(a.m) + at, lane, top_bytes(c[0], c[1], c[2], c[3]),
                top_bytes(c[4], c[5], c[6], c[7]));
#pragma unroll
    for (int i = 0; i < 8; ++i) c[i] = encode_v(v[i], iv, __byte_perm(bits[i], 0x80u, 0x5104));
    store_codes(static_cast<uint8_t*>(a.v) + at, lane, top_bytes(c[0], c[1], c[2], c[3]),
                top_bytes(c[4], c[5], c[6], c[7]));
    if (lane == 0) {
      a.m_scale[at >> 8] = sm;
      a.v_scale[at >> 8] = sv;
    }
  }
  if constexpr (MASTER) {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (place(lane, i) >= n) p[i] = 0.0f;  // the gap behind the tensor stays zero
    store8(master, lane, p);
  } else if constexpr (kStochastic) {
    // 16 random bits below the last one kept (never through NaN or infinity)
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (fabsf(p[i]) < INFINITY) p[i] = __uint_as_float(__float_as_uint(p[i]) + (more_bits(bits[i]) & 0xFFFFu));
  }
  if (vec && n >= 256) {
    if constexpr (kStochastic) {
      uint32_t w[4];
#pragma unroll
      for (int q = 0; q < 4; ++q)
        w[q] = __byte_perm(__float_as_uint(p[2 * q]), __float_as_uint(p[2 * q + 1]), 0x7632);
      store_words(param, lane, w[0], w[1], w[2], w[3]);
    } else {
      store8(param, lane, p);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      if constexpr (kStochastic) p[i] = __uint_as_float(__float_as_uint(p[i]) & 0xFFFF0000u);
      if (place(lane, i) < n) put(param + place(lane, i), p[i]);
    }
  }
}

// Elements i0 .. i1 of a tensor, i0 a multiple of 256.
template <typename P, typename G, bool MASTER, int BITS>
__device__ __forceinline__ void adamw_run(const AdamArgs& a, const StepConsts& k, const mxg_adamw_tensor& t,
                                          uint64_t g, int64_t i0, int64_t i1) {
  P* param = static_cast<P*>(t.param);
  const G* grad = reinterpret_cast<const G*>(g);
  float* master = MASTER ? a.master + t.master : nullptr;
  const int64_t offset = t.offset;
  const bool vec = ((reinterpret_cast<uintptr_t>(param) | reinterpret_cast<uintptr_t>(grad)) & 15) == 0;
  const float keep = 1.0f - k.lr * t.weight_decay;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  for (int64_t b = i0 + warp * 256; b < i1; b += kAdamThreads * 8)
    adamw_block<P, G, MASTER, BITS>(a, k, param + b, grad + b, MASTER ? master + b : nullptr, offset + b,
                                    int(min(i1 - b, int64_t(256))), keep, vec, lane);
}

// A block takes a run of neighbouring chunks: their tensor is looked up once.
template <int BITS>
__global__ void __launch_bounds__(kAdamThreads, BITS == 8 ? 3 : 4) adamw_kernel(const __grid_constant__ AdamArgs a) {
  __shared__ float s_bc[2];
  const int64_t t = *a.step + 1;
  // 1 - b^t = -expm1(t ln b): exact where b^t is close to 1
  if (threadIdx.x == 0) s_bc[0] = float(-expm1(double(t) * a.ln_b1));
  if (threadIdx.x == 32) s_bc[1] = float(-expm1(double(t) * a.ln_b2));
  __syncthreads();
  StepConsts k;
  k.lr = a.lr_ptr ? *a.lr_ptr : a.lr;
  k.step_size = k.lr / s_bc[0];
  k.rs2 = 1.0f / sqrtf(s_bc[1]);
  k.key = step_key(a.seed_lo, a.seed_hi, uint32_t(t));
  int64_t c = blockIdx.x;
  int ti = c < a.n_chunks ? a.chunks[a.chunk0 + c] : 0;
  for (; c < a.n_chunks; c += gridDim.x) {
    const mxg_adamw_tensor& T = a.tensors[ti];
    const uint64_t tagged = a.grads[ti - a.tensor0];
    const int64_t i0 = (a.chunk0 + c - T.first_chunk) * MXG_ADAMW_CHUNK, i1 = min(T.numel, i0 + MXG_ADAMW_CHUNK);
    if (c + gridDim.x < a.n_chunks) ti = a.chunks[a.chunk0 + c + gridDim.x];
    if (tagged == 0) continue;
    const uint64_t g = tagged & ~kGradF32;
    const bool f32 = tagged & kGradF32;
    switch (T.kind) {
      case MXG_ADAMW_F32:
        if (f32) adamw_run<float, float, false, BITS>(a, k, T, g, i0, i1);
        else adamw_run<float, __nv_bfloat16, false, BITS>(a, k, T, g, i0, i1);
        break;
      case MXG_ADAMW_BF16_MASTER:
        if (f32) adamw_run<__nv_bfloat16, float, true, BITS>(a, k, T, g, i0, i1);
        else adamw_run<__nv_bfloat16, __nv_bfloat16, true, BITS>(a, k, T, g, i0, i1);
        break;
      default:
        if (f32) adamw_run<__nv_bfloat16, float, false, BITS>(a, k, T, g, i0, i1);
        else adamw_run<__nv_bfloat16, __nv_bfloat16, false, BITS>(a, k, T, g, i0, i1);
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

// A warp takes blocks of 256.
__global__ void __launch_bounds__(256) adamw_moments_kernel(const uint8_t* __restrict__ m,
                                                            const uint8_t* __restrict__ v,
                                                            const float* __restrict__ m_scale,
                                                            const float* __restrict__ v_scale, int64_t blocks,
                                                            float* __restrict__ m_out, float* __restrict__ v_out) {
  const int lane = threadIdx.x & 31;
  const int64_t step = int64_t(gridDim.x) * 8;
  for (int64_t b = int64_t(blockIdx.x) * 8 + (threadIdx.x >> 5); b < blocks; b += step) {
    const uint2 cm = load_codes(m + b * 256, lane), cv = load_codes(v + b * 256, lane);
    const float sm = m_scale[b], sv = v_scale[b];
    float x[8], y[8];
    decode_m(cm.x, sm, x, 0), decode_m(cm.y, sm, x, 4);
    decode_v(cv.x, sv, y, 0), decode_v(cv.y, sv, y, 4);
    store8(m_out + b * 256, lane, x);
    store8(v_out + b * 256, lane, y);
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
  if (!(lr >= 0.0) || !(beta1 >= 0.0 && beta1 < 1.0) || !(beta2 >= 0.0 && beta2 < 1.0) || !(eps > 0.0))
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
  const int64_t blocks = n / MXG_ADAMW_BLOCK, want = (blocks + 7) / 8;
  adamw_moments_kernel<<<unsigned(std::min<int64_t>(want, int64_t(num_sms()) * 16)), 256, 0, (cudaStream_t)stream>>>(
      static_cast<const uint8_t*>(exp_avg), static_cast<const uint8_t*>(exp_avg_sq), exp_avg_scale, exp_avg_sq_scale,
      blocks, exp_avg_out, exp_avg_sq_out);
  return cuda_status(cudaGetLastError());
}
