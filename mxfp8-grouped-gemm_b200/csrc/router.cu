// Expert router for sm_100a: scores, top-k experts and their weights of every
// token, and the gradient of the logits.
//
//   s = softmax(z) or sigmoid(z) over a token's E experts, c = s + bias;
//   with G groups of E/G experts only the topk_groups best groups stay (a
//   group counts by its best c or by the sum of its two best);
//   ids = the k largest c, descending, ties to the lowest index;
//   w = scale * s[ids], divided by their sum when renormalised.
//
// A token's experts lie in the registers of LANES lanes, V consecutive ones a
// lane, so the lowest lane that holds a maximum also holds the lowest index.
// Selection is k rounds of a maximum over the lanes.
//
// Order.  The scores rise with the logits, so without a bias the logits
// themselves are compared: exact.  With one, c is computed in fp32 and its
// error bounded; where two neighbours of the order (the first expert left out
// among them) or the last group kept and the first dropped are closer than
// the bound, the token is selected again with scores in fp64.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <cmath>
#include <type_traits>

#include "mxg.h"
#include "mxg_device.cuh"
#include "mxg_internal.h"

namespace mxg {

constexpr int kRouterThreads = 128;
constexpr unsigned kFull = 0xffffffffu;

struct RouterArgs {
  const void* z;
  int64_t ld, n;
  int experts, topk, groups, topk_groups;
  bool top2, sigmoid, renorm, vec;
  float scale;
  const float* bias;
  float* weights;
  int32_t* ids;
};

__device__ __forceinline__ float to_f32(float x) { return x; }
__device__ __forceinline__ float to_f32(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ float to_f32(__half x) { return __half2float(x); }
__device__ __forceinline__ void from_f32(float x, float& o) { o = x; }
__device__ __forceinline__ void from_f32(float x, __nv_bfloat16& o) { o = __float2bfloat16_rn(x); }
__device__ __forceinline__ void from_f32(float x, __half& o) { o = __float2half_rn(x); }

// Order-preserving key of a float: unsigned comparison of keys is comparison
// of values, -0 equals +0, a NaN counts as -inf, and 0 is below every key.
__device__ __forceinline__ uint32_t order_key(float x) {
  if (x != x) return 0x007FFFFFu;
  const uint32_t u = __float_as_uint(x + 0.0f);
  return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}
__device__ __forceinline__ float key_value(uint32_t k) {
  return __uint_as_float((k & 0x80000000u) ? (k & 0x7FFFFFFFu) : ~k);
}

template <int LANES, class F, class X>
__device__ __forceinline__ X lanes_reduce(X x, F f, unsigned mask) {
#pragma unroll
  for (int o = LANES / 2; o > 0; o >>= 1) x = f(x, __shfl_xor_sync(mask, x, o, LANES));
  return x;
}
struct MaxOp {
  __device__ float operator()(float a, float b) const { return fmaxf(a, b); }
  __device__ uint32_t operator()(uint32_t a, uint32_t b) const { return a > b ? a : b; }
};
struct MinOp {
  __device__ float operator()(float a, float b) const { return fminf(a, b); }
};
struct OrOp {
  __device__ uint32_t operator()(uint32_t a, uint32_t b) const { return a | b; }
};
struct SumOp {
  __device__ float operator()(float a, float b) const { return a + b; }
  __device__ double operator()(double a, double b) const { return a + b; }
};

template <int LANES>
__device__ __forceinline__ uint32_t lanes_max_key(uint32_t x) {
  if constexpr (LANES == 32) return __reduce_max_sync(kFull, x);
  else return lanes_reduce<LANES>(x, MaxOp(), kFull);
}

// z[v] = logit of expert lane * V + v (anything beyond the last expert: -inf).
template <typename T, int V>
__device__ __forceinline__ void load_row(const T* row, int lane, int experts, bool vec, float (&z)[V]) {
  const int e0 = lane * V;
  if (vec) {
    if (e0 < experts) {
      constexpr int B = (V * sizeof(T)) % 16 == 0 ? 16 : 8;  // bytes a load
      constexpr int P = B / sizeof(T);
      using W = typename std::conditional<B == 16, uint4, uint2>::type;
#pragma unroll
      for (int c = 0; c < V / P; ++c) {
        const W w = __ldg(reinterpret_cast<const W*>(row + e0) + c);
        const T* t = reinterpret_cast<const T*>(&w);
#pragma unroll
        for (int i = 0; i < P; ++i) z[c * P + i] = to_f32(t[i]);
      }
    } else {
#pragma unroll
      for (int v = 0; v < V; ++v) z[v] = -INFINITY;
    }
  } else {
#pragma unroll
    for (int v = 0; v < V; ++v) z[v] = e0 + v < experts ? to_f32(row[e0 + v]) : -INFINITY;
  }
}

__device__ __forceinline__ float sigmoid_f32(float z) { return 1.0f / (1.0f + __expf(-z)); }

// Selection of one token with scores in fp64 (rare: see the head of the
// file), by the LANES lanes of `mask`.  c: LANES * V doubles of shared memory.
template <typename T, int LANES, int V>
__device__ __noinline__ void select_f64(const RouterArgs& a, const T* row, int lane, unsigned mask, double* c,
                                        double* group, int32_t* out) {
  const int E = a.experts, G = a.groups, per = E / G;
  double top = -INFINITY, sum = 0.0;
  if (!a.sigmoid) {
    for (int v = 0; v < V; ++v) {
      const int e = lane * V + v;
      if (e < E) top = fmax(top, double(to_f32(row[e])));
    }
    for (int o = LANES / 2; o > 0; o >>= 1) top = fmax(top, __shfl_xor_sync(mask, top, o, LANES));
    if (top == -INFINITY) top = 0.0;
    for (int v = 0; v < V; ++v) {
      const int e = lane * V + v;
      if (e < E) sum += exp(double(to_f32(row[e])) - top);
    }
    sum = lanes_reduce<LANES>(sum, SumOp(), mask);
  }
  for (int v = 0; v < V; ++v) {
    const int e = lane * V + v;
    double x = -INFINITY;
    if (e < E) {
      const double z = double(to_f32(row[e]));
      x = a.sigmoid ? 1.0 / (1.0 + exp(-z)) : (sum == 0.0 ? 0.0 : exp(z - top) / sum);
      if (a.bias) x += double(a.bias[e]);
      if (x != x) x = -INFINITY;
    }
    c[e] = x;
  }
  __syncwarp(mask);
  uint32_t kept = 0;
  for (int g = lane; g < G; g += LANES) {
    double b1 = -INFINITY, b2 = -INFINITY;
    for (int i = 0; i < per; ++i) {
      const double x = c[g * per + i];
      if (x > b1) { b2 = b1; b1 = x; } else if (x > b2) b2 = x;
    }
    group[g] = a.top2 && per > 1 ? b1 + b2 : b1;
  }
  __syncwarp(mask);
  for (int g = lane; g < G; g += LANES) {
    int rank = 0;
    for (int h = 0; h < G; ++h) rank += group[h] > group[g] || (group[h] == group[g] && h < g);
    if (rank < a.topk_groups) kept |= 1u << g;
  }
  for (int o = LANES / 2; o > 0; o >>= 1) kept |= __shfl_xor_sync(mask, kept, o, LANES);
  uint32_t left = 0;                                    // my experts that are still to be had
  for (int v = 0; v < V; ++v) {
    const int e = lane * V + v;
    if (e < E && (kept >> (e / per) & 1)) left |= 1u << v;
  }
  // without a bias the logits give the order (the groups alone needed scores)
  for (int r = 0; r < a.topk; ++r) {
    double best = -INFINITY;
    int at = 0x7FFFFFFF;
    for (int v = 0; v < V; ++v) {
      const int e = lane * V + v;
      if (!(left >> v & 1)) continue;
      double x = a.bias ? c[e] : double(to_f32(row[e]));
      if (x != x) x = -INFINITY;
      if (at == 0x7FFFFFFF || x > best) { best = x; at = e; }
    }
    for (int o = LANES / 2; o > 0; o >>= 1) {
      const double x = __shfl_xor_sync(mask, best, o, LANES);
      const int e = __shfl_xor_sync(mask, at, o, LANES);
      if (e != 0x7FFFFFFF && (at == 0x7FFFFFFF || x > best || (x == best && e < at))) { best = x; at = e; }
    }
    if (at / V == lane) left &= ~(1u << (at % V));
    if (lane == 0) out[r] = at;
  }
  __syncwarp(mask);
}

template <typename T, int LANES, int V>
__global__ void __launch_bounds__(kRouterThreads) router_topk_kernel(const __grid_constant__ RouterArgs a) {
  constexpr int ROWS = kRouterThreads / LANES;                       // tokens a block
  constexpr int MOST = (LANES * V < 32 ? LANES * V : 32) + 1;        // choices, and the first left out
  constexpr int GMAX = LANES * V < 32 ? LANES * V : 32;
  __shared__ int32_t s_id[ROWS][MOST];
  __shared__ uint32_t s_key[ROWS][MOST];
  __shared__ double s_group[ROWS][GMAX];
  __shared__ double s_c[ROWS][LANES * V];

  const int lane = threadIdx.x % LANES, sub = threadIdx.x / LANES;
  const int64_t want = int64_t(blockIdx.x) * ROWS + sub;
  const int64_t r = want < a.n ? want : a.n - 1;                     // every lane takes part in the shuffles
  const T* row = static_cast<const T*>(a.z) + r * a.ld;
  const int E = a.experts, G = a.groups, per = E / G, k = a.topk;
  const unsigned mask = LANES == 32 ? kFull : ((1u << (LANES & 31)) - 1u) << ((threadIdx.x & 31) / LANES * LANES);

  float z[V];
  load_row<T, V>(row, lane, E, a.vec, z);

  // softmax statistics of the whole row: for its scores and for weights that are not renormalised
  const bool scored = a.bias || (G > 1 && a.top2);
  bool odd = false;                                                  // a NaN or +inf: softmax has no value
  float top = -INFINITY;
#pragma unroll
  for (int v = 0; v < V; ++v) {
    top = fmaxf(top, z[v]);
    odd |= !(z[v] < INFINITY);
  }
  top = lanes_reduce<LANES>(top, MaxOp(), kFull);
  const float base = top == -INFINITY ? 0.0f : top;
  float inv = 0.0f;
  if (!a.sigmoid) {
    odd = (__ballot_sync(kFull, odd) & mask) != 0;
    if (scored || !a.renorm) {
      float sum = 0.0f;
#pragma unroll
      for (int v = 0; v < V; ++v) sum += __expf(z[v] - base);
      sum = lanes_reduce<LANES>(sum, SumOp(), kFull);
      inv = sum > 0.0f ? 1.0f / sum : 0.0f;
    }
  }

  uint32_t key[V];
  float near = 0.0f;  // two choices closer than this may be in the wrong order
  bool again = false;
  float c[V];
  if (scored) {
    float big = 0.0f, most = 0.0f;
#pragma unroll
    for (int v = 0; v < V; ++v) {
      const int e = lane * V + v;
      float s = a.sigmoid ? sigmoid_f32(z[v]) : __expf(z[v] - base) * inv;
      if (e >= E) s = 0.0f;
      big = fmaxf(big, s);
      if (a.bias && e < E) {
        const float b = __ldg(a.bias + e);
        s += b;
        if (fabsf(b) < INFINITY) most = fmaxf(most, fabsf(b));
      }
      c[v] = s;
    }
    big = lanes_reduce<LANES>(big, MaxOp(), kFull);
    if (a.bias) most = lanes_reduce<LANES>(most, MaxOp(), kFull);
    // exp's argument is off by |z| 2^-24 in relative terms, the exponential,
    // the sum and the quotient by a few 2^-24 each; the sum with the bias by
    // 2^-24 of its size: 2^-20 and 2^-22 leave room for all of them, twice
    const float far = a.sigmoid ? fmaxf(0.0f, -top) : 0.0f;
    near = 0x1p-19f * big * (1.0f + far) + 0x1p-21f * most;
  }
#pragma unroll
  for (int v = 0; v < V; ++v) key[v] = lane * V + v < E ? order_key(a.bias ? c[v] : z[v]) : 0u;

  if (G > 1) {
    // every group's score, then its rank among the groups
    float* gs = reinterpret_cast<float*>(s_group[sub]);
    float* all = reinterpret_cast<float*>(s_c[sub]);
    const bool byz = !scored;                                        // best logit: exact
#pragma unroll
    for (int v = 0; v < V; ++v) all[lane * V + v] = byz ? z[v] : c[v];
    __syncwarp();
    for (int g = lane; g < G; g += LANES) {
      float b1 = -INFINITY, b2 = -INFINITY;
      for (int i = 0; i < per; ++i) {
        const float x = all[g * per + i];
        if (x > b1) { b2 = b1; b1 = x; } else if (x > b2) b2 = x;
      }
      gs[g] = a.top2 && per > 1 ? b1 + b2 : b1;
    }
    __syncwarp();
    uint32_t kept = 0;
    float low = INFINITY, high = -INFINITY;                          // of the kept, of the dropped
    for (int g = lane; g < G; g += LANES) {
      const float x = gs[g];
      int rank = 0;
      for (int h = 0; h < G; ++h) rank += gs[h] > x || (gs[h] == x && h < g);
      if (rank < a.topk_groups) {
        kept |= 1u << g;
        low = fminf(low, x);
      } else {
        high = fmaxf(high, x);
      }
    }
    kept = lanes_reduce<LANES>(kept, OrOp(), kFull);
    if (!byz && a.topk_groups < G) {
      low = lanes_reduce<LANES>(low, MinOp(), kFull);
      high = lanes_reduce<LANES>(high, MaxOp(), kFull);
      again = !(low - high > 2.0f * near);
    }
#pragma unroll
    for (int v = 0; v < V; ++v) {
      const int e = lane * V + v;
      if (e < E && !(kept >> (e / per) & 1)) key[v] = 0u;
    }
  }

  // k rounds, and one more for the first that is left out
  const int cand = a.topk_groups * per;
  const int rounds = a.bias && cand > k ? k + 1 : k;
  for (int q = 0; q < rounds; ++q) {
    uint32_t best = key[0];
#pragma unroll
    for (int v = 1; v < V; ++v) best = best > key[v] ? best : key[v];
    const uint32_t m = lanes_max_key<LANES>(best);
    const unsigned who = __ballot_sync(kFull, best == m) & mask;
    if (int(threadIdx.x & 31) == __ffs(who) - 1) {
      int at = 0;
#pragma unroll
      for (int v = V - 1; v >= 0; --v) at = key[v] == m ? v : at;
#pragma unroll
      for (int v = 0; v < V; ++v)
        if (v == at) key[v] = 0u;
      s_id[sub][q] = lane * V + at;
      s_key[sub][q] = m;
    }
  }
  __syncwarp();
  if (a.bias) {
    for (int q = lane; q + 1 < rounds; q += LANES) {
      const float hi = key_value(s_key[sub][q]), lo = key_value(s_key[sub][q + 1]);
      if (!(hi - lo > near)) {
        // the same logit and the same bias tie for certain, and stand in order of index
        const int i = s_id[sub][q], j = s_id[sub][q + 1];
        if (!(to_f32(row[i]) == to_f32(row[j]) && a.bias[i] == a.bias[j])) again = true;
      }
    }
  }
  again = (__ballot_sync(kFull, again) & mask) != 0;
  if (again) select_f64<T, LANES, V>(a, row, lane, mask, s_c[sub], s_group[sub], s_id[sub]);
  __syncwarp();

  // weights of the chosen, from their logits
  float most = -INFINITY;
  for (int q = lane; q < k; q += LANES) most = fmaxf(most, to_f32(row[s_id[sub][q]]));
  if (a.renorm) most = lanes_reduce<LANES>(most, MaxOp(), kFull);
  float sum = 0.0f;
  // shares of a renormalised row: sigmoid(z) up to a common factor, with
  // nothing that overflows or vanishes for the largest
  const float shift = a.sigmoid ? fminf(most, 0.0f) : most;
  auto part = [&](float x) {
    if (x == -INFINITY) return 0.0f;
    if (!a.sigmoid) return __expf(x - shift);
    return x > 0.0f ? 1.0f / (1.0f + __expf(-x)) : __expf(x - shift) / (1.0f + __expf(x));
  };
  if (a.renorm) {
    for (int q = lane; q < k; q += LANES) sum += part(to_f32(row[s_id[sub][q]]));
    sum = lanes_reduce<LANES>(sum, SumOp(), kFull);
  }
  if (want >= a.n) return;
  for (int q = lane; q < k; q += LANES) {
    const int e = s_id[sub][q];
    const float x = to_f32(row[e]);
    float w;
    if (a.renorm) w = sum == 0.0f ? 0.0f : part(x) / sum;
    else if (a.sigmoid) w = sigmoid_f32(x);
    else w = __expf(x - base) * inv;
    if (odd && !a.sigmoid) w = NAN;
    a.weights[r * k + q] = w * a.scale;
    a.ids[r * k + q] = e;
  }
}

struct RouterBwdArgs {
  const void* z;
  int64_t ld, n, ld_out;
  int experts, topk;
  bool sigmoid, renorm, vec, vec_out;
  float scale;
  const float* weights;
  const int32_t* ids;
  const float* dweights;
  void* dz;
  int* err;
};

template <typename T, int V>
__device__ __forceinline__ void store_row(T* row, int lane, int experts, bool vec, const float (&x)[V]) {
  const int e0 = lane * V;
  if (vec) {
    if (e0 >= experts) return;
    constexpr int B = (V * sizeof(T)) % 16 == 0 ? 16 : 8;
    constexpr int P = B / sizeof(T);
    using W = typename std::conditional<B == 16, uint4, uint2>::type;
#pragma unroll
    for (int c = 0; c < V / P; ++c) {
      W w;
      T* t = reinterpret_cast<T*>(&w);
#pragma unroll
      for (int i = 0; i < P; ++i) from_f32(x[c * P + i], t[i]);
      reinterpret_cast<W*>(row + e0)[c] = w;
    }
  } else {
#pragma unroll
    for (int v = 0; v < V; ++v)
      if (e0 + v < experts) from_f32(x[v], row[e0 + v]);
  }
}

// Gradient of the logits from that of the weights.  With w = scale * p:
//   softmax:              dz_i = [i chosen] w_i dw_i - s_i sum(w dw)   (every expert)
//   softmax, renormalised dz_i = w_i (dw_i - sum(p dw))                (the chosen)
//   sigmoid:              dz_i = scale dw_i s_i (1 - s_i)
//   sigmoid, renormalised dz_i = w_i (1 - s_i) (dw_i - sum(p dw))
template <typename T, int LANES, int V>
__global__ void __launch_bounds__(kRouterThreads) router_bwd_kernel(const __grid_constant__ RouterBwdArgs a) {
  constexpr int ROWS = kRouterThreads / LANES;
  constexpr int MOST = LANES * V < 32 ? LANES * V : 32;
  __shared__ float s_dz[ROWS][LANES * V];
  __shared__ int32_t s_id[ROWS][MOST];
  __shared__ float s_g[ROWS][MOST];
  const int lane = threadIdx.x % LANES, sub = threadIdx.x / LANES;
  const int64_t want = int64_t(blockIdx.x) * ROWS + sub;
  const int64_t r = want < a.n ? want : a.n - 1;
  const T* row = static_cast<const T*>(a.z) + r * a.ld;
  const int E = a.experts, k = a.topk;
  const bool dense = !a.sigmoid && !a.renorm;

  float z[V];
  float* acc = s_dz[sub];
#pragma unroll
  for (int v = 0; v < V; ++v) acc[lane * V + v] = 0.0f;
  float pull = 0.0f;
  for (int q = lane; q < k; q += LANES) pull += a.weights[r * k + q] * a.dweights[r * k + q];
  pull = lanes_reduce<LANES>(pull, SumOp(), kFull);
  if (dense) {
    load_row<T, V>(row, lane, E, a.vec, z);
    float top = -INFINITY;
#pragma unroll
    for (int v = 0; v < V; ++v) top = fmaxf(top, z[v]);
    top = lanes_reduce<LANES>(top, MaxOp(), kFull);
    const float base = top == -INFINITY ? 0.0f : top;
    float sum = 0.0f;
#pragma unroll
    for (int v = 0; v < V; ++v) {
      z[v] = __expf(z[v] - base);
      sum += z[v];
    }
    sum = lanes_reduce<LANES>(sum, SumOp(), kFull);
    const float by = sum == 0.0f ? 0.0f : -pull / sum;
#pragma unroll
    for (int v = 0; v < V; ++v) z[v] *= by;
  } else {
#pragma unroll
    for (int v = 0; v < V; ++v) z[v] = 0.0f;
  }
  const float mean = pull / a.scale;
  for (int q = lane; q < k; q += LANES) {
    int e = a.ids[r * k + q];
    float g = 0.0f;
    if (e < 0 || e >= E) {
      if (want < a.n) atomicCAS(a.err, 0, MXG_ERR_INVALID_ARGUMENT);
      e = -1;
    } else {
      const float dw = a.dweights[r * k + q], w = a.weights[r * k + q];
      if (dense) {
        g = w * dw;
      } else if (a.renorm) {
        g = w * (dw - mean);
        if (a.sigmoid) g *= sigmoid_f32(-to_f32(row[e]));
      } else {
        const float x = to_f32(row[e]);
        g = a.scale * dw * sigmoid_f32(x) * sigmoid_f32(-x);
      }
    }
    s_id[sub][q] = e;
    s_g[sub][q] = g;
  }
  __syncwarp();
  // an expert that is named more than once gets the sum, in order, from its first place
  for (int q = lane; q < k; q += LANES) {
    const int e = s_id[sub][q];
    float g = 0.0f;
    bool first = e >= 0;
    for (int h = 0; h < k; ++h) {
      const bool same = s_id[sub][h] == e;
      first &= !(same && h < q);
      g += same ? s_g[sub][h] : 0.0f;
    }
    if (first) acc[e] = g;
  }
  __syncwarp();
  if (want >= a.n) return;
#pragma unroll
  for (int v = 0; v < V; ++v) z[v] += acc[lane * V + v];
  store_row<T, V>(static_cast<T*>(a.dz) + r * a.ld_out, lane, E, a.vec_out, z);
}

constexpr size_t elem_size(int dtype) { return dtype == MXG_DTYPE_F32 ? 4 : 2; }

// Rows of V consecutive elements a lane can be read as vectors: V elements a
// lane throughout, every row on a 16-byte boundary.
inline bool rows_vectorised(const void* p, int64_t ld, int experts, int v, size_t size) {
  return experts % v == 0 && (size_t(ld) * size) % 16 == 0 && aligned16(p);
}

template <typename T, int LANES, int V>
int launch_topk(RouterArgs& a, cudaStream_t s) {
  a.vec = rows_vectorised(a.z, a.ld, a.experts, V, sizeof(T));
  const int64_t blocks = (a.n + kRouterThreads / LANES - 1) / (kRouterThreads / LANES);
  router_topk_kernel<T, LANES, V><<<unsigned(blocks), kRouterThreads, 0, s>>>(a);
  return cuda_status(cudaGetLastError());
}

template <typename T, int LANES, int V>
int launch_bwd(RouterBwdArgs& a, cudaStream_t s) {
  a.vec = rows_vectorised(a.z, a.ld, a.experts, V, sizeof(T));
  a.vec_out = rows_vectorised(a.dz, a.ld_out, a.experts, V, sizeof(T));
  const int64_t blocks = (a.n + kRouterThreads / LANES - 1) / (kRouterThreads / LANES);
  router_bwd_kernel<T, LANES, V><<<unsigned(blocks), kRouterThreads, 0, s>>>(a);
  return cuda_status(cudaGetLastError());
}

// The fewest lanes that hold the experts, 8 a lane (12 beyond 256).
#define MXG_BY_EXPERTS(FN, T, a, s)                    \
  ((a).experts <= 8     ? FN<T, 1, 8>(a, s)            \
   : (a).experts <= 16  ? FN<T, 2, 8>(a, s)            \
   : (a).experts <= 32  ? FN<T, 4, 8>(a, s)            \
   : (a).experts <= 64  ? FN<T, 8, 8>(a, s)            \
   : (a).experts <= 128 ? FN<T, 16, 8>(a, s)           \
   : (a).experts <= 256 ? FN<T, 32, 8>(a, s)           \
                        : FN<T, 32, 12>(a, s))
#define MXG_BY_TYPE(FN, dtype, a, s)                                        \
  ((dtype) == MXG_DTYPE_BF16  ? MXG_BY_EXPERTS(FN, __nv_bfloat16, a, s)     \
   : (dtype) == MXG_DTYPE_F16 ? MXG_BY_EXPERTS(FN, __half, a, s)            \
                              : MXG_BY_EXPERTS(FN, float, a, s))

int router_shape(int64_t n, int experts, int topk, int64_t ld, int dtype, int score) {
  if (n < 0 || experts < 1 || topk < 1 || (dtype != MXG_DTYPE_BF16 && dtype != MXG_DTYPE_F16 && dtype != MXG_DTYPE_F32) ||
      (score != MXG_SCORE_SOFTMAX && score != MXG_SCORE_SIGMOID))
    return MXG_ERR_INVALID_ARGUMENT;
  if (experts > MXG_EP_MAX_EXPERTS || topk > experts || topk > MXG_ROUTER_MAX_TOPK || n > INT32_MAX || ld < experts)
    return MXG_ERR_BAD_SHAPE;
  return MXG_OK;
}

}  // namespace mxg

using namespace mxg;

extern "C" int mxg_router_topk(const void* logits, int64_t ld, int dtype, int64_t n_tokens, int num_experts, int topk,
                               int score, const float* bias, int groups, int topk_groups, int group_score,
                               int renormalize, float scale, float* weights, int32_t* ids, void* stream) {
  int st = router_shape(n_tokens, num_experts, topk, ld, dtype, score);
  if (st) return st;
  if (groups < 1 || topk_groups < 1 || topk_groups > groups ||
      (group_score != MXG_GROUP_MAX && group_score != MXG_GROUP_TOP2) || !(scale > 0.0f) || !std::isfinite(scale))
    return MXG_ERR_INVALID_ARGUMENT;
  if (groups > MXG_ROUTER_MAX_GROUPS || num_experts % groups || topk > topk_groups * (num_experts / groups))
    return MXG_ERR_BAD_SHAPE;
  if (n_tokens == 0) return MXG_OK;
  if (!logits || !weights || !ids) return MXG_ERR_INVALID_ARGUMENT;
  if ((st = check_device())) return st;
  RouterArgs a{};
  a.z = logits, a.ld = ld, a.n = n_tokens, a.experts = num_experts, a.topk = topk;
  a.groups = topk_groups == groups ? 1 : groups;  // all groups stay: no groups
  a.topk_groups = topk_groups == groups ? 1 : topk_groups;
  a.top2 = group_score == MXG_GROUP_TOP2, a.sigmoid = score == MXG_SCORE_SIGMOID, a.renorm = renormalize != 0;
  a.scale = scale, a.bias = bias, a.weights = weights, a.ids = ids;
  return MXG_BY_TYPE(launch_topk, dtype, a, (cudaStream_t)stream);
}

extern "C" int mxg_router_topk_bwd(const void* logits, int64_t ld, int dtype, int64_t n_tokens, int num_experts,
                                   int topk, int score, int renormalize, float scale, const float* weights,
                                   const int32_t* ids, const float* dweights, void* dlogits, int64_t ld_out,
                                   void* stream) {
  int st = router_shape(n_tokens, num_experts, topk, ld, dtype, score);
  if (st) return st;
  if (!(scale > 0.0f) || !std::isfinite(scale)) return MXG_ERR_INVALID_ARGUMENT;
  if (ld_out < num_experts) return MXG_ERR_BAD_SHAPE;
  if (n_tokens == 0) return MXG_OK;
  if (!logits || !weights || !ids || !dweights || !dlogits) return MXG_ERR_INVALID_ARGUMENT;
  if ((st = check_device())) return st;
  RouterBwdArgs a{};
  a.z = logits, a.ld = ld, a.n = n_tokens, a.ld_out = ld_out, a.experts = num_experts, a.topk = topk;
  a.sigmoid = score == MXG_SCORE_SIGMOID, a.renorm = renormalize != 0, a.scale = scale;
  a.weights = weights, a.ids = ids, a.dweights = dweights, a.dz = dlogits, a.err = device_error_word();
  if (!a.err) return MXG_ERR_CUDA;
  return MXG_BY_TYPE(launch_bwd, dtype, a, (cudaStream_t)stream);
}
