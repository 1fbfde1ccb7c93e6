// One AdamW step over many tensors for sm_100a.
//
// The tensors are cut into chunks; a persistent grid walks their table, a warp
// taking 256 elements at a time (8 a lane, the block that shares one scale of
// the 8-bit moments).  Bound by HBM: every
// array passes by once, in 16-byte accesses.
//
// The moments are rounded operation by operation (no fused multiply-adds), so
// that the 8-bit codes are a function of the inputs alone.
#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <cfloat>
#include <cmath>
#include <type_traits>

#include "mxg.h"
#include "mxg_device.cuh"
#include "mxg_internal.h"

namespace mxg {

// One block an SM: its warps work on one run of memory (352 M weights, 8 bits: 868 us, 908 with two blocks of 512,
// 948 with four of 256; 32 bits: 1627, 1630, 1645).
constexpr int kAdamThreads = 1024;
constexpr int kAdamTensors = 480;              // gradient addresses a launch carries (kernel arguments: 4 KB)
constexpr uint64_t kGradF32 = uint64_t(1) << 63;

struct AdamArgs {
  const mxg_adamw_tensor* tensors;
  const int32_t* chunks;
  int64_t chunk0, n_chunks;
  int chunk;
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

// Two fp32 operations in one instruction, each rounded as a single one.
struct Two {
  uint64_t w;
};
__device__ __forceinline__ Two two(float a, float b) {
  Two t;
  asm("mov.b64 %0, {%1, %2};" : "=l"(t.w) : "f"(a), "f"(b));
  return t;
}
__device__ __forceinline__ Two both(float a) { return two(a, a); }
__device__ __forceinline__ void split(Two t, float& a, float& b) {
  asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(t.w));
}
__device__ __forceinline__ Two mul(Two a, Two b) {
  Two t;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(t.w) : "l"(a.w), "l"(b.w));
  return t;
}
__device__ __forceinline__ Two fma2(Two a, Two b, Two c) {
  Two t;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(t.w) : "l"(a.w), "l"(b.w), "l"(c.w));
  return t;
}

// Random bits: 32x32 -> 64-bit products by odd constants, the halves xored,
// two of them for each of (seed, step), block and element.  Means, spread and
// bits of both halves, and their correlations with one another and between
// neighbours, blocks, steps and seeds, are those of independent uniform draws
// to within the sampling error of 2^18 draws (a test).
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
// The code as the top byte, without a sign; noise: 16 random bits, in bits 8 to
// 23.  (A NaN or infinity spills over, into a block whose scale is one too.)
__device__ __forceinline__ uint32_t top_code(float x, uint32_t noise) { return __float_as_uint(x) * 16u + noise; }
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
// They travel as words; pointers are to the lane's first value.
__device__ __forceinline__ int place(int lane, int i) { return lane * 4 + (i & 3) + (i >> 2) * 128; }
template <typename T>
struct Words {
  static constexpr int N = 2 * sizeof(T);
  uint32_t w[N];
};
template <typename T>
__device__ __forceinline__ void fetch(const T* p, Words<T>& x) {
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const T* q = p + h * 128;
    uint32_t* w = x.w + h * sizeof(T);
    if constexpr (sizeof(T) == 4) {
      const uint4 v = *reinterpret_cast<const uint4*>(q);
      w[0] = v.x, w[1] = v.y, w[2] = v.z, w[3] = v.w;
    } else if constexpr (sizeof(T) == 2) {
      const uint2 v = *reinterpret_cast<const uint2*>(q);
      w[0] = v.x, w[1] = v.y;
    } else {
      w[0] = *reinterpret_cast<const uint32_t*>(q);
    }
  }
}
template <typename T>
__device__ __forceinline__ void keep_words(T* p, const Words<T>& x) {
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    T* q = p + h * 128;
    const uint32_t* w = x.w + h * sizeof(T);
    if constexpr (sizeof(T) == 4) *reinterpret_cast<uint4*>(q) = make_uint4(w[0], w[1], w[2], w[3]);
    else if constexpr (sizeof(T) == 2) *reinterpret_cast<uint2*>(q) = make_uint2(w[0], w[1]);
    else *reinterpret_cast<uint32_t*>(q) = w[0];
  }
}
__device__ __forceinline__ void unpack(const Words<float>& x, float (&f)[8]) {
#pragma unroll
  for (int i = 0; i < 8; ++i) f[i] = __uint_as_float(x.w[i]);
}
__device__ __forceinline__ void unpack(const Words<__nv_bfloat16>& x, float (&f)[8]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) f[2 * i] = bf16_lo(x.w[i]), f[2 * i + 1] = bf16_hi(x.w[i]);
}
__device__ __forceinline__ void pack(const float (&f)[8], Words<float>& x) {
#pragma unroll
  for (int i = 0; i < 8; ++i) x.w[i] = __float_as_uint(f[i]);
}
__device__ __forceinline__ void pack(const float (&f)[8], Words<__nv_bfloat16>& x) {
#pragma unroll
  for (int i = 0; i < 4; ++i) x.w[i] = pack2_bf16(f[2 * i], f[2 * i + 1]);
}
__device__ __forceinline__ float as_f32(float x) { return x; }
__device__ __forceinline__ float as_f32(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ void put(float* p, float x) { *p = x; }
__device__ __forceinline__ void put(__nv_bfloat16* p, float x) { *p = __float2bfloat16_rn(x); }

// SMALL: an x under 2^-126 has a root too, else it counts as 0.
template <bool SMALL>
__device__ __forceinline__ float sqrt_fast(float x) {
  float y;
  if constexpr (SMALL) asm("sqrt.approx.f32 %0, %1;" : "=f"(y) : "f"(x));
  else asm("sqrt.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float rcp_fast(float x) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

struct StepConsts {
  float size, rs2;   // -lr / (1 - b1^t), 1 / sqrt(1 - b2^t)
  const float* bc1;  // 1 - b1^t, in shared memory: registers are short
  uint32_t key;
};

// What a lane reads of a block: weights, gradients and moments.
template <typename P, typename G, bool MASTER, int BITS>
struct Block {
  using W = typename std::conditional<MASTER, float, P>::type;    // what takes the update
  using S = typename std::conditional<BITS == 8, uint8_t, float>::type;
  Words<W> p;
  Words<G> g;
  Words<S> m, v;
  float sm, sv;                                                    // scales
};

// The update of one block, in place; block: its number in the moments.
template <typename P, typename G, bool MASTER, int BITS, bool SMALL>
__device__ __forceinline__ void update(const AdamArgs& a, const StepConsts& k, float decay, uint64_t block, int lane,
                                       Block<P, G, MASTER, BITS>& x) {
  constexpr bool kStochastic = !MASTER && sizeof(P) == 2;
  float p[8], g[8], m[8], v[8];
  unpack(x.p, p);
  unpack(x.g, g);
  if constexpr (BITS == 32) {
    unpack(x.m, m);
    unpack(x.v, v);
  } else {
    decode_m(x.m.w[0], x.sm, m, 0), decode_m(x.m.w[1], x.sm, m, 4);
    decode_v(x.v.w[0], x.sv, v, 0), decode_v(x.v.w[1], x.sv, v, 4);
  }
  // the update alone goes through the approximate root and reciprocal (2 units
  // of the last place)
#pragma unroll
  for (int i = 0; i < 8; i += 2) {
    const Two gg = two(g[i], g[i + 1]);
    float d0, d1;
    // (the sums one by one: a packed one is contracted with its product)
    split(mul(gg, both(a.c1)), d0, d1);
    split(mul(two(m[i], m[i + 1]), both(a.b1)), m[i], m[i + 1]);
    m[i] = __fadd_rn(m[i], d0), m[i + 1] = __fadd_rn(m[i + 1], d1);
    split(mul(mul(gg, gg), both(a.c2)), d0, d1);
    split(mul(two(v[i], v[i + 1]), both(a.b2)), v[i], v[i + 1]);
    v[i] = __fadd_rn(v[i], d0), v[i + 1] = __fadd_rn(v[i + 1], d1);
    split(fma2(two(sqrt_fast<SMALL>(v[i]), sqrt_fast<SMALL>(v[i + 1])), both(k.rs2), both(a.eps)), d0, d1);
    // lr is a factor of what is finite, last of all, so that with lr 0 the weight stays whatever v is; the
    // decay joins the update: one rounding of the weight's size
    const Two by = mul(two(m[i], m[i + 1]), two(rcp_fast(d0), rcp_fast(d1)));
    const Two old = two(p[i], p[i + 1]);
    split(fma2(fma2(old, both(decay), by), both(k.size), old), p[i], p[i + 1]);
  }
  float im = 0.0f, iv = 0.0f, rm[2], rv[2];
  if constexpr (BITS == 32) {
    pack(m, x.m);
    pack(v, x.v);
  } else {
    x.sm = fabsf(m[0]), x.sv = v[0];  // of the block: a NaN if there is one
#pragma unroll
    for (int i = 1; i < 8; ++i) x.sm = max_nan(x.sm, fabsf(m[i])), x.sv = max_nan(x.sv, v[i]);
    x.sm = max_nan(warp_max_nan(x.sm), 0x1p-100f), x.sv = max_nan(warp_max_nan(x.sv), 0x1p-100f);
    im = 1.0f / x.sm, iv = 1.0f / x.sv;
  }
  if constexpr (BITS == 8 || kStochastic) {
    const uint32_t kb = block_key(k.key, block);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const uint32_t bits = element_bits(kb, place(lane, i));
      if constexpr (BITS == 8) {
        // relative to the scale, with the exponent field that makes bits 20 and up the code
        if (i % 2 == 0) {
          split(mul(mul(two(m[i], m[i + 1]), both(im)), both(0x1p-112f)), rm[0], rm[1]);
          split(mul(mul(two(v[i], v[i + 1]), both(iv)), both(0x1p-96f)), rv[0], rv[1]);
        }
        // the new code enters at the top of its word
        const uint32_t tm = top_code(rm[i % 2], __byte_perm(bits, 0x80u, 0x5324));
        const uint32_t tv = top_code(rv[i % 2], __byte_perm(bits, 0x80u, 0x5104));
        x.m.w[i >> 2] = __byte_perm(x.m.w[i >> 2], (tm & 0x7FFFFFFFu) | (__float_as_uint(m[i]) & 0x80000000u), 0x7321);
        x.v.w[i >> 2] = __byte_perm(x.v.w[i >> 2], v[i] > 0.0f ? max(tv, 1u << 24) : tv, 0x7321);
      }
      // a bf16 weight without a copy: 16 random bits below the last one kept; the sum of a NaN's bits
      // (0x7FFFFFFF, as arithmetic gives it) would pass over to a negative number
      if constexpr (kStochastic) {
        const int u = __float_as_int(p[i]);
        const uint32_t r = uint32_t(max(int(uint32_t(u) + (more_bits(bits) & 0xFFFFu)), u));
        x.p.w[i >> 1] = i & 1 ? __byte_perm(x.p.w[i >> 1], r, 0x7632) : r;
      }
    }
  }
  if constexpr (!kStochastic) pack(p, x.p);
}

// Elements i0 .. i0 + n of a tensor, i0 a multiple of 256, n at most a chunk.
// Whole blocks of 16-byte-aligned tensors are read and written in vectors,
// others element by element.  With 8-bit moments the step is bound by
// instructions, and registers are short: the next block is fetched to the L2
// cache (352 M weights, blocks of 256 threads: 979 -> 935 us; through shared
// memory instead 957, into registers 1265).  Addresses are those of the chunk, the same for
// the whole block, plus a 32-bit offset.
template <typename P, typename G, bool MASTER, int BITS, bool SMALL>
__device__ __forceinline__ void adamw_chunk(const AdamArgs& a, const StepConsts& k, const mxg_adamw_tensor& t,
                                            uint64_t g, int64_t i0, int n) {
  using B = Block<P, G, MASTER, BITS>;
  using S = typename B::S;
  constexpr uint32_t kStep = kAdamThreads * 8;
  const uint32_t lane = threadIdx.x & 31;
  const float decay = *k.bc1 * t.weight_decay;  // over -lr / (1 - b1^t), as the update is
  const int64_t at = t.offset + i0;
  P* param = static_cast<P*>(t.param) + i0;
  const G* grad = reinterpret_cast<const G*>(g) + i0;
  typename B::W* weight;
  if constexpr (MASTER) weight = a.master + t.master + i0;
  else weight = param;
  S *m = static_cast<S*>(a.m) + at, *v = static_cast<S*>(a.v) + at;
  float *ms = a.m_scale + (at >> 8), *vs = a.v_scale + (at >> 8);
  const uint64_t block = uint64_t(at) >> 8;
  const bool vec = ((reinterpret_cast<uintptr_t>(param) | reinterpret_cast<uintptr_t>(grad)) & 15) == 0;
  const uint32_t whole = vec ? uint32_t(n) & ~255u : 0;  // elements that go by in vectors

  auto load = [&](uint32_t o, B& x) {  // o: of the lane's first value
    fetch(weight + o, x.p);
    fetch(grad + o, x.g);
    fetch(m + o, x.m);
    fetch(v + o, x.v);
    if constexpr (BITS == 8) x.sm = ms[o >> 8], x.sv = vs[o >> 8];
  };
  // a line of 128 bytes a lane: gradients, weights, codes
  constexpr uint32_t kG = 2 * sizeof(G), kW = 2 * sizeof(typename B::W);
  auto prefetch = [&](uint32_t q) {
    const char* from = lane < kG        ? reinterpret_cast<const char*>(grad + q) + lane * 128
                       : lane < kG + kW ? reinterpret_cast<const char*>(weight + q) + (lane - kG) * 128
                       : lane < kG + kW + 2 ? reinterpret_cast<const char*>(m + q) + (lane - kG - kW) * 128
                                            : reinterpret_cast<const char*>(v + q) + (lane - kG - kW - 2) * 128;
    if (lane < kG + kW + 4) asm volatile("prefetch.global.L2 [%0];" ::"l"(from));
  };
  uint32_t o = (threadIdx.x >> 5) * 256 + lane * 4;
#pragma unroll 1
  for (; o < uint32_t(n) + lane * 4; o += kStep) {
    B x;
    if (o < whole) {
      load(o, x);
      if (BITS == 8 && o + kStep < whole) prefetch(o - lane * 4 + kStep);
    } else {
      float p[8], f[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const uint32_t e = o + (i & 3) + (i >> 2) * 128;
        f[i] = e < n ? as_f32(grad[e]) : 0.0f;
        p[i] = !MASTER && e < n ? as_f32(param[e]) : 0.0f;
      }
      pack(f, x.g);
      if constexpr (MASTER) fetch(weight + o, x.p);
      else pack(p, x.p);
      fetch(m + o, x.m);
      fetch(v + o, x.v);
      if constexpr (BITS == 8) x.sm = ms[o >> 8], x.sv = vs[o >> 8];
    }
    update<P, G, MASTER, BITS, SMALL>(a, k, decay, block + (o >> 8), lane, x);
    keep_words(m + o, x.m);
    keep_words(v + o, x.v);
    if (BITS == 8 && lane == 0) ms[o >> 8] = x.sm, vs[o >> 8] = x.sv;
    if (o < whole) {
      keep_words(weight + o, x.p);
      if constexpr (MASTER) {
        float f[8];
        Words<P> w;
        unpack(x.p, f);
        pack(f, w);
        keep_words(param + o, w);
      }
    } else {
      float p[8];
      unpack(x.p, p);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const uint32_t e = o + (i & 3) + (i >> 2) * 128;
        if (e < n) put(param + e, p[i]);
        else p[i] = 0.0f;  // the gap behind the tensor stays zero
      }
      if constexpr (MASTER) {
        pack(p, x.p);
        keep_words(weight + o, x.p);
      }
    }
  }
}

template <int BITS, bool SMALL>
__global__ void __launch_bounds__(kAdamThreads) adamw_kernel(const __grid_constant__ AdamArgs a) {
  __shared__ float s_bc[2];
  const int64_t t = *a.step + 1;
  // 1 - b^t = -expm1(t ln b): exact where b^t is close to 1
  if (threadIdx.x == 0) s_bc[0] = float(-expm1(double(t) * a.ln_b1));
  if (threadIdx.x == 32) s_bc[1] = float(-expm1(double(t) * a.ln_b2));
  __syncthreads();
  StepConsts k;
  k.bc1 = s_bc;
  k.size = -(a.lr_ptr ? *a.lr_ptr : a.lr) / s_bc[0];
  k.rs2 = 1.0f / sqrtf(s_bc[1]);
  k.key = step_key(a.seed_lo, a.seed_hi, uint32_t(t));
  int64_t c = blockIdx.x;
  int ti = c < a.n_chunks ? a.chunks[a.chunk0 + c] : 0;
  for (; c < a.n_chunks; c += gridDim.x) {
    const mxg_adamw_tensor& T = a.tensors[ti];
    const uint64_t tagged = a.grads[ti - a.tensor0];
    const int64_t i0 = (a.chunk0 + c - T.first_chunk) * a.chunk;
    const int n = int(min(T.numel - i0, int64_t(a.chunk)));
    if (c + gridDim.x < a.n_chunks) ti = a.chunks[a.chunk0 + c + gridDim.x];
    if (tagged == 0) continue;
    const uint64_t g = tagged & ~kGradF32;
    const bool f32 = tagged & kGradF32;
    switch (T.kind) {
      case MXG_ADAMW_F32:
        if (f32) adamw_chunk<float, float, false, BITS, SMALL>(a, k, T, g, i0, n);
        else adamw_chunk<float, __nv_bfloat16, false, BITS, SMALL>(a, k, T, g, i0, n);
        break;
      case MXG_ADAMW_BF16_MASTER:
        if (f32) adamw_chunk<__nv_bfloat16, float, true, BITS, SMALL>(a, k, T, g, i0, n);
        else adamw_chunk<__nv_bfloat16, __nv_bfloat16, true, BITS, SMALL>(a, k, T, g, i0, n);
        break;
      default:
        if (f32) adamw_chunk<__nv_bfloat16, float, false, BITS, SMALL>(a, k, T, g, i0, n);
        else adamw_chunk<__nv_bfloat16, __nv_bfloat16, false, BITS, SMALL>(a, k, T, g, i0, n);
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
    Words<uint8_t> cm, cv;
    Words<float> out;
    fetch(m + b * 256 + lane * 4, cm);
    fetch(v + b * 256 + lane * 4, cv);
    const float sm = m_scale[b], sv = v_scale[b];
    float x[8], y[8];
    decode_m(cm.w[0], sm, x, 0), decode_m(cm.w[1], sm, x, 4);
    decode_v(cv.w[0], sv, y, 0), decode_v(cv.w[1], sv, y, 4);
    pack(x, out);
    keep_words(m_out + b * 256 + lane * 4, out);
    pack(y, out);
    keep_words(v_out + b * 256 + lane * 4, out);
  }
}

}  // namespace mxg

using namespace mxg;

extern "C" int mxg_adamw_step(const mxg_adamw_args* args, void* stream) {
  if (!args) return MXG_ERR_INVALID_ARGUMENT;
  const mxg_adamw_args& r = *args;
  const int n_tensors = r.n_tensors, state_bits = r.state_bits;
  const int64_t* chunk_begin = r.chunk_begin;
  const uint64_t* grads = r.grads;
  const int32_t* grad_dtypes = r.grad_dtypes;
  if (n_tensors < 1 || !r.tensors || !r.chunks || !chunk_begin || !grads || !grad_dtypes || !r.exp_avg ||
      !r.exp_avg_sq || !r.step || !r.done || (state_bits != 8 && state_bits != 32))
    return MXG_ERR_INVALID_ARGUMENT;
  if (r.chunk < MXG_ADAMW_BLOCK || r.chunk % MXG_ADAMW_BLOCK || r.chunk > (1 << 24)) return MXG_ERR_INVALID_ARGUMENT;
  if (state_bits == 8 && (!r.exp_avg_scale || !r.exp_avg_sq_scale)) return MXG_ERR_INVALID_ARGUMENT;
  if (!(r.lr >= 0.0 && r.lr <= FLT_MAX) || !(r.beta1 >= 0.0 && r.beta1 < 1.0) ||
      !(r.beta2 >= 0.0 && r.beta2 < 1.0) || !(r.eps >= FLT_MIN && r.eps <= FLT_MAX))
    return MXG_ERR_INVALID_ARGUMENT;
  for (int i = 0; i < n_tensors; ++i) {
    if (chunk_begin[i] < 0 || chunk_begin[i + 1] < chunk_begin[i]) return MXG_ERR_INVALID_ARGUMENT;
    if (grads[i] && grad_dtypes[i] != MXG_DTYPE_BF16 && grad_dtypes[i] != MXG_DTYPE_F32)
      return MXG_ERR_INVALID_ARGUMENT;
    if (grads[i] & kGradF32 || grads[i] % (grad_dtypes[i] == MXG_DTYPE_F32 ? 4 : 2)) return MXG_ERR_MISALIGNED;
  }
  if (!aligned16(r.exp_avg) || !aligned16(r.exp_avg_sq) || !aligned16(r.master)) return MXG_ERR_MISALIGNED;
  int st = check_device();
  if (st) return st;
  AdamArgs a;
  a.tensors = r.tensors, a.chunks = r.chunks, a.chunk = r.chunk;
  a.m = r.exp_avg, a.v = r.exp_avg_sq, a.m_scale = r.exp_avg_scale, a.v_scale = r.exp_avg_sq_scale, a.master = r.master;
  a.step = r.step, a.done = r.done, a.lr_ptr = r.lr_ptr;
  a.lr = float(r.lr), a.b1 = float(r.beta1), a.c1 = float(1.0 - r.beta1);
  a.b2 = float(r.beta2), a.c2 = float(1.0 - r.beta2), a.eps = float(r.eps);
  a.ln_b1 = std::log(r.beta1), a.ln_b2 = std::log(r.beta2);
  a.seed_lo = uint32_t(r.seed), a.seed_hi = uint32_t(r.seed >> 32);
  int per_sm = 0;
  // The root of a second moment under 2^-126 is at most 2^-63, over sqrt(1 - b2) in the first step: from eps =
  // 2^24 times that on it is lost in fp32's rounding.  Below, 8-bit states take the root with subnormals too (352 M
  // weights: 1008 us for 987; 32-bit states, bound by HBM, take it always: 1626, 1624).
  const bool small = state_bits == 32 || r.eps * std::sqrt(1.0 - r.beta2) < 0x1p-39;
  auto* kernel = state_bits == 32 ? adamw_kernel<32, true> : small ? adamw_kernel<8, true> : adamw_kernel<8, false>;
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
