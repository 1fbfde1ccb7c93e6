// Expert router for sm_100a: scores, top-k experts and their weights of every
// token, and the gradient of the logits.
//
//   s = softmax(z) or sigmoid(z) over a token's E experts, c = s + bias;
//   with G groups of E/G experts only the topk_groups best groups stay (a
//   group counts by its best c or by the sum of its two best);
//   ids = the k largest c, descending, ties to the lowest index;
//   w = scale * s[ids], divided by their sum when renormalised.
//
// A token's experts lie in the registers of LANES lanes, in order: the lowest
// lane that holds a value also holds its lowest index, and a group fills whole
// lanes.  Each lane sorts its own V values (a network of min and max, no
// index), groups are scored from the heads of these lists, and k rounds take
// the largest head and move that lane's list up.  Where in its lane a chosen
// value stood is looked up afterwards, for all k at once.
//
// Order.  The scores rise with the logits, so without a bias the logits
// themselves are compared: exact.  With one, c is computed in fp32 and its
// error bounded; where two neighbours of the order (the first expert left out
// among them) or the last group kept and the first dropped are closer than
// the bound, and where what is chosen has c = -inf, the token is selected
// again, slowly, with scores in fp64.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <cmath>
#include <type_traits>
#include <utility>

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
  int per, lpg_log2, cnt, rounds;  // experts a group; lanes a group (a power of 2); experts a lane; rounds
  bool top2, sigmoid, renorm, vec, vec_bias;
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

// Operations over the LANES lanes of a token; every lane of the warp takes part.
template <int LANES>
__device__ __forceinline__ float lanes_max(float x) {
  if constexpr (LANES == 32) {
    float m;
    asm("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(m) : "f"(x));
    return m;
  } else {
#pragma unroll
    for (int o = LANES / 2; o > 0; o >>= 1) x = fmaxf(x, __shfl_xor_sync(kFull, x, o));
    return x;
  }
}
template <int LANES, typename X>
__device__ __forceinline__ X lanes_sum(X x, unsigned mask = kFull) {
#pragma unroll
  for (int o = LANES / 2; o > 0; o >>= 1) x += __shfl_xor_sync(mask, x, o);
  return x;
}

__device__ __forceinline__ float max_nan(float a, float b) {
  float m;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(m) : "f"(a), "f"(b));
  return m;
}

// exp and 1 / x by the approximate instructions (2 units of the last place
// beside exp's argument, 1 unit; results under 2^-126 are 0).
__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float exp_fast(float x) { return exp2_fast(x * 1.44269504f); }
__device__ __forceinline__ float rcp_fast(float x) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// 0 below z = -88.
__device__ __forceinline__ float sigmoid_fast(float z) { return rcp_fast(1.0f + exp_fast(-z)); }
__device__ __forceinline__ float sigmoid_f32(float z) { return 1.0f / (1.0f + __expf(-z)); }

// Descending order by Batcher's odd-even merge sort (for V that is no power of
// two the missing values are the smallest and never move).
template <int V>
struct Network {
  int a[V * V]{}, b[V * V]{}, n = 0;
  constexpr Network() {
    for (int p = 1; p < V; p *= 2)
      for (int k = p; k >= 1; k /= 2)
        for (int j = k % p; j + k < V; j += 2 * k)
          for (int i = 0; i < k && i + j + k < V; ++i)
            if ((i + j) / (2 * p) == (i + j + k) / (2 * p)) a[n] = i + j, b[n] = i + j + k, ++n;
  }
};
template <int A, int B, int V>
__device__ __forceinline__ void put_in_order(float (&x)[V]) {
  const float a = x[A], b = x[B];
  x[A] = fmaxf(a, b);
  x[B] = fminf(a, b);
}
template <int V, size_t... I>
__device__ __forceinline__ void sort_down(float (&x)[V], std::index_sequence<I...>) {
  constexpr Network<V> net;
  (put_in_order<net.a[I], net.b[I]>(x), ...);
}
template <int V>
__device__ __forceinline__ void sort_down(float (&x)[V]) {
  sort_down(x, std::make_index_sequence<Network<V>().n>());
}

// x[v] = element first + v of the row for v < have, else -inf.
template <typename T, int V>
__device__ __forceinline__ void load_row(const T* row, int first, int have, bool vec, float (&x)[V]) {
  if (vec) {
    if (have > 0) {
      constexpr int B = (V * sizeof(T)) % 16 == 0 ? 16 : 8;  // bytes a load
      constexpr int P = B / sizeof(T);
      using W = typename std::conditional<B == 16, uint4, uint2>::type;
#pragma unroll
      for (int c = 0; c < V / P; ++c) {
        const W w = __ldg(reinterpret_cast<const W*>(row + first) + c);
        const T* t = reinterpret_cast<const T*>(&w);
#pragma unroll
        for (int i = 0; i < P; ++i) x[c * P + i] = to_f32(t[i]);
      }
    } else {
#pragma unroll
      for (int v = 0; v < V; ++v) x[v] = -INFINITY;
    }
  } else {
#pragma unroll
    for (int v = 0; v < V; ++v) x[v] = v < have ? to_f32(row[first + v]) : -INFINITY;
  }
}

// Bits of a double in an order of unsigned integers; 0 is below every value.
__device__ __forceinline__ uint64_t order_bits(double x) {
  const uint64_t u = uint64_t(__double_as_longlong(x + 0.0));
  return u >> 63 ? ~u : u | 1ull << 63;
}

// Selection of one token in order of the scores in fp64 (rare: see the head of
// the file), by a whole warp; lane l holds experts l, l + 32, ...  key: a word
// of shared memory for every expert.  Four experts at a time: a lane's chain of
// exponentials and loads is what it waits for, but the code has to stay small,
// since it is never at hand when it is needed.
template <typename T>
__device__ __noinline__ void select_f64(const RouterArgs& a, const T* row, uint64_t* key, int32_t* out) {
  const int E = a.experts, lane = threadIdx.x & 31;
  double top = 0.0, sum = 1.0;
  if (!a.sigmoid) {
    float m = -INFINITY;
    for (int e = lane; e < E; e += 32) m = fmaxf(m, to_f32(row[e]));
    m = lanes_max<32>(m);
    top = m == -INFINITY ? 0.0 : double(m);
  }
  for (int pass = a.sigmoid ? 1 : 0; pass < 2; ++pass) {
    double part = 0.0;
#pragma unroll 4
    for (int e = lane; e < E; e += 32) {
      const double z = double(to_f32(row[e]));
      const double f = exp(a.sigmoid ? -z : z - top);
      part += f;
      if (pass == 0) continue;
      double x = a.sigmoid ? 1.0 / (1.0 + f) : sum == 0.0 ? 0.0 : f / sum;
      if (a.bias) x += double(a.bias[e]);
      else if (!a.top2) x = z;  // the best group by its best logit
      key[e] = uint64_t(__double_as_longlong(x != x ? -INFINITY : x));
    }
    if (pass == 0) sum = lanes_sum<32>(part);
  }
  __syncwarp();
  unsigned kept = kFull;
  if (a.groups > 1) {
    int log2 = 0;
    while (a.groups << (log2 + 1) <= 32) ++log2;
    const int group = lane >> log2, some = (a.per + (1 << log2) - 1) >> log2;
    const int begin = (lane & ((1 << log2) - 1)) * some, end = group < a.groups ? min(begin + some, a.per) : 0;
    double b1 = -INFINITY, b2 = -INFINITY;
#pragma unroll 4
    for (int i = begin; i < end; ++i) {
      const double x = __longlong_as_double((long long)key[group * a.per + i]);
      b2 = fmax(b2, fmin(b1, x));
      b1 = fmax(b1, x);
    }
    for (int o = 1; o < 1 << log2; o <<= 1) {
      const double o1 = __shfl_xor_sync(kFull, b1, o), o2 = __shfl_xor_sync(kFull, b2, o);
      b2 = fmax(fmin(b1, o1), fmax(b2, o2));
      b1 = fmax(b1, o1);
    }
    double score = a.top2 && a.per > 1 ? b1 + b2 : b1;
    if (score != score) score = -INFINITY;  // inf - inf
    int better = 0;
#pragma unroll 4
    for (int g = 0; g < a.groups; ++g) {
      const double o = __shfl_sync(kFull, score, g << log2);
      better += o > score || (o == score && g < group);
    }
    const unsigned all = __ballot_sync(kFull, better < a.topk_groups);
    kept = 0;
    for (int g = 0; g < a.groups; ++g) kept |= (all >> (g << log2) & 1u) << g;
  }
  __syncwarp();
#pragma unroll 4
  for (int e = lane; e < E; e += 32) {
    double x = __longlong_as_double((long long)key[e]);
    if (!a.bias) {  // the logits give the order
      x = double(to_f32(row[e]));
      if (x != x) x = -INFINITY;
    }
    key[e] = a.groups == 1 || (kept >> (e / a.per) & 1) ? order_bits(x) : 0;
  }
  constexpr int MOST = MXG_EP_MAX_EXPERTS / 32;
  uint64_t mine[MOST];
#pragma unroll
  for (int i = 0; i < MOST; ++i) mine[i] = lane + i * 32 < E ? key[lane + i * 32] : 0;
  for (int r = 0; r < a.topk; ++r) {
    uint64_t best = 0;
    int at = 0;
#pragma unroll
    for (int i = 0; i < MOST; ++i)
      if (mine[i] > best) { best = mine[i]; at = i; }
    const uint32_t hi = __reduce_max_sync(kFull, uint32_t(best >> 32));
    const uint32_t lo = __reduce_max_sync(kFull, uint32_t(best >> 32) == hi ? uint32_t(best) : 0u);
    const bool equal = best == (uint64_t(hi) << 32 | lo);
    const int e = int(__reduce_min_sync(kFull, equal ? unsigned(at * 32 + lane) : kFull));
    if (lane == 0) out[r] = e;
#pragma unroll
    for (int i = 0; i < MOST; ++i)
      if (e == i * 32 + lane) mine[i] = 0;
  }
  __syncwarp();
}

// The order of one token's best experts where values that fp32 cannot tell
// apart stand among them, but the groups are certain: those whose value in
// fp32 is at least `from` are ordered by their scores in fp64, one a lane.
// False where there are more than 32 of them.  list: 32 words of shared memory.
template <typename T>
__device__ __noinline__ bool order_near(const RouterArgs& a, const T* row, float from, uint32_t kept, float base,
                                        float inv, int per, uint32_t* list, int32_t* out) {
  const int E = a.experts, lane = threadIdx.x & 31;
  int count = 0;
  double sum = 0.0;
#pragma unroll 4
  for (int e0 = 0; e0 < E; e0 += 32) {
    const int e = e0 + lane;
    const float z = e < E ? to_f32(row[e]) : -INFINITY;
    float x = z;
    if (a.bias) {
      x = a.sigmoid ? sigmoid_fast(z) : exp_fast(z - base) * inv;
      x = e < E ? x + a.bias[e] : -INFINITY;
      if (!a.sigmoid) sum += exp(double(z) - double(base));
    }
    const bool in = e < E && x >= from && (kept >> (e / per) & 1u);
    const unsigned all = __ballot_sync(kFull, in);
    const int at = count + __popc(all & ((1u << lane) - 1u));
    if (in && at < 32) list[at] = uint32_t(e);
    count += __popc(all);
  }
  __syncwarp();
  if (count > 32 || count < a.topk) return false;
  if (a.bias && !a.sigmoid) sum = lanes_sum<32>(sum);
  const int e = lane < count ? int(list[lane]) : 0;  // ascending: the lower lane has the lower index
  double x = double(to_f32(row[e]));
  if (a.bias) {
    if (a.sigmoid) x = 1.0 / (1.0 + exp(-x));
    else x = sum > 0.0 ? exp(x - double(base)) / sum : 0.0;          // a row without an expert has no score
    x += double(a.bias[e]);
  }
  int rank = 0;
  for (int i = 0; i < count; ++i) {
    const double o = __shfl_sync(kFull, x, i);
    rank += o > x || (o == x && i < lane);
  }
  if (lane < count && rank < a.topk) out[rank] = e;
  __syncwarp();
  return true;
}

// Weights and ids of one token, from the logits of its choices: id[i] is choice
// lane + i * LANES of the LANES lanes.
template <int LANES, int NQ, typename T>
__device__ __forceinline__ void write_weights(const RouterArgs& a, const T* row, int64_t r, bool real, int lane,
                                              const int (&id)[NQ], float base, float inv, bool odd) {
  const int k = a.topk;
  float y[NQ], most = -INFINITY;
#pragma unroll
  for (int i = 0; i < NQ; ++i) {
    y[i] = lane + i * LANES < k ? to_f32(row[id[i]]) : -INFINITY;
    most = fmaxf(most, y[i]);
  }
  float by = 1.0f;
  if (a.renorm) {
    // shares: sigmoid(z) up to a common factor, with nothing that overflows or
    // vanishes for the largest
    most = lanes_max<LANES>(most);
    const float shift = a.sigmoid ? fminf(most, 0.0f) : most;
    float sum = 0.0f;
#pragma unroll
    for (int i = 0; i < NQ; ++i) {
      float p = __expf(a.sigmoid && y[i] > 0.0f ? 0.0f : y[i] - shift);
      if (a.sigmoid) p = __fdividef(p, 1.0f + __expf(-fabsf(y[i])));
      y[i] = y[i] == -INFINITY ? 0.0f : p;
      sum += y[i];
    }
    sum = lanes_sum<LANES>(sum);
    by = sum == 0.0f ? 0.0f : __fdividef(1.0f, sum);
  } else {
#pragma unroll
    for (int i = 0; i < NQ; ++i) y[i] = a.sigmoid ? sigmoid_f32(y[i]) : __expf(y[i] - base);
    if (!a.sigmoid) by = inv;
  }
  if (!real) return;
#pragma unroll
  for (int i = 0; i < NQ; ++i) {
    const int q = lane + i * LANES;
    if (q >= k) continue;
    a.weights[r * k + q] = odd ? NAN : y[i] * by * a.scale;
    a.ids[r * k + q] = id[i];
  }
}

template <typename T, int LANES, int V>
__global__ void __launch_bounds__(kRouterThreads) router_topk_kernel(const __grid_constant__ RouterArgs a) {
  constexpr int ROWS = kRouterThreads / LANES;                       // tokens a block
  constexpr int MOST = LANES * V < 32 ? LANES * V : 32;              // choices
  constexpr int SLOW = LANES * V < MXG_EP_MAX_EXPERTS ? LANES * V : MXG_EP_MAX_EXPERTS;
  __shared__ __align__(16) float s_val[ROWS][LANES * V];             // what is ordered, as the lanes hold it
  __shared__ __align__(16) float s_list[ROWS][LANES * V];            // each lane's values, descending
  __shared__ float2 s_rec[ROWS][MOST + 1];                           // a choice: value, and lane | rank in it << 8
  __shared__ int32_t s_id[ROWS][MOST];
  __shared__ uint64_t s_key[kRouterThreads / 32][SLOW];              // of the slow selection

  const int wl = threadIdx.x & 31, lane = threadIdx.x % LANES, sub = threadIdx.x / LANES;
  const int64_t want = int64_t(blockIdx.x) * ROWS + sub;
  const int64_t r = want < a.n ? want : a.n - 1;                     // every lane takes part in the shuffles
  const T* row = static_cast<const T*>(a.z) + r * a.ld;
  const int G = a.groups, per = a.per, k = a.topk;
  const unsigned mask = LANES == 32 ? kFull : ((1u << (LANES & 31)) - 1u) << (wl / LANES * LANES);
  const int group = lane >> a.lpg_log2, sl = lane & ((1 << a.lpg_log2) - 1);
  const int first = group * per + sl * a.cnt;
  const int have = group < G ? min(per - sl * a.cnt, a.cnt) : 0;     // experts of this lane (none if <= 0)

  float z[V];
  load_row<T, V>(row, first, have, a.vec, z);

  const bool groups_scored = G > 1 && (a.bias || a.top2);            // by scores, not by a logit
  float top = z[0];
#pragma unroll
  for (int v = 1; v < V; ++v) top = fmaxf(top, z[v]);
  top = lanes_max<LANES>(fmaxf(top, -INFINITY));
  const float base = top == -INFINITY ? 0.0f : top;
  bool odd = false;                                                  // a NaN or +inf: softmax has no value

  float x[V];                                                        // what is ordered
  float inv = 0.0f;                                                  // 1 / the sum of the row's exponentials
  if (a.sigmoid) {
    if (a.bias) {
#pragma unroll
      for (int v = 0; v < V; ++v) x[v] = sigmoid_fast(z[v]);
    }
  } else {
#pragma unroll
    for (int v = 0; v < V; ++v) odd |= !(z[v] < INFINITY);
    odd = (__ballot_sync(kFull, odd) & mask) != 0;
    if (groups_scored || a.bias || !a.renorm) {
      float sum = 0.0f;
#pragma unroll
      for (int v = 0; v < V; ++v) {
        x[v] = exp_fast(z[v] - base);
        sum += x[v];
      }
      sum = lanes_sum<LANES>(sum);
      inv = sum > 0.0f ? 1.0f / sum : 0.0f;
    }
  }
  float near = 0.0f;                                                 // closer than this: perhaps the other way round
  bool again = false;
  if (a.bias || groups_scored) {
    // s (1 - s) times what is off in exp (2^-22, and 1.5 |z| 2^-24 from its
    // argument), and 3 * 2^-24 s from the sum and the reciprocal: at most
    // 2^-24 s (7 + 1.5 |z|), which is largest for the largest s (and below
    // 2^-24 s 7 where z > 0); softmax has a sum of V + 5 roundings in place of
    // 1 + exp, and |z| s is at most 0.37 of its largest s.  Twice that for a
    // pair, and what lies under 2^-126 and became 0
    const float big = a.sigmoid ? sigmoid_fast(top) : inv;
    near = 0x1p-24f * big * (a.sigmoid ? 14.0f + 3.0f * fmaxf(0.0f, -top) : 2.0f * V + 40.0f) + 0x1p-124f;
    again = a.sigmoid && top < -80.0f;                               // the scores vanish in fp32
    if (a.sigmoid && !a.bias) {
      // in a group's sum a NaN counts as -inf, a logit of -inf as its score, 0: in the order below they are one
#pragma unroll
      for (int v = 0; v < V; ++v) again |= z[v] != z[v];
    }
  }
  if (a.bias) {
    float b[V];
    load_row<float, V>(a.bias, first, have, a.vec_bias, b);
#pragma unroll
    for (int v = 0; v < V; ++v) x[v] = fmaxf(a.sigmoid ? x[v] + b[v] : fmaf(x[v], inv, b[v]), -INFINITY);
  } else {
#pragma unroll
    for (int v = 0; v < V; ++v) x[v] = fmaxf(z[v] + 0.0f, -INFINITY);  // -0 is 0, a NaN is -inf
  }
  float *vals = s_val[sub], *list = s_list[sub];
#pragma unroll
  for (int v = 0; v < V; v += 4)
    *reinterpret_cast<float4*>(vals + lane * V + v) = make_float4(x[v], x[v + 1], x[v + 2], x[v + 3]);
  sort_down<V>(x);
#pragma unroll
  for (int v = 0; v < V; v += 4)
    *reinterpret_cast<float4*>(list + lane * V + v) = make_float4(x[v], x[v + 1], x[v + 2], x[v + 3]);
  float head = x[0];
  bool kept = true;                                                  // this lane's group

  if (G > 1) {
    // the two best of the group, over its lanes
    float b1 = x[0], b2 = x[1];
    for (int o = 1; o < (1 << a.lpg_log2); o <<= 1) {
      const float o1 = __shfl_xor_sync(kFull, b1, o), o2 = __shfl_xor_sync(kFull, b2, o);
      b2 = fmaxf(fminf(b1, o1), fmaxf(b2, o2));
      b1 = fmaxf(b1, o1);
    }
    if (groups_scored && !a.bias) {  // logits so far
      b1 = a.sigmoid ? sigmoid_fast(b1) : exp_fast(b1 - base) * inv;
      b2 = a.sigmoid ? sigmoid_fast(b2) : exp_fast(b2 - base) * inv;
    }
    const bool two = a.top2 && per > 1;
    float score = fmaxf(two ? b1 + b2 : b1, -INFINITY);
    if (group >= G) score = -INFINITY;
    int better = 0;
    for (int g = 0; g < G; ++g) {
      const float o = __shfl_sync(kFull, score, g << a.lpg_log2, LANES);
      better += o > score || (o == score && g < group);
    }
    kept = better < a.topk_groups && group < G;
    const float low = -lanes_max<LANES>(kept ? -score : -INFINITY), high = lanes_max<LANES>(kept ? -INFINITY : score);
    if (groups_scored) {
      // two sums of two, and their roundings
      const float size = fabsf(b1) < INFINITY ? fabsf(b1) : 0.0f, more = fabsf(b2) < INFINITY ? fabsf(b2) : 0.0f;
      const float off = 2.0f * near + 0x1p-21f * lanes_max<LANES>(fmaxf(size, more));
      again |= !(low - high > off);
    }
    again |= low == -INFINITY;
    if (!kept) head = -INFINITY;
  }

  // k rounds, and with a bias one more for the first that is left out
  const int rounds = a.rounds;
  const unsigned below = mask & ((1u << wl) - 1u);
  int code = lane;
  float2* rec = s_rec[sub];
  const float* next = list + lane * V;
  __syncwarp();
  for (int q = 0; q < rounds; ++q) {
    const float m = lanes_max<LANES>(head);
    const bool equal = head == m;
    const unsigned who = __ballot_sync(kFull, equal);
    if (equal && (who & below) == 0) {
      rec[q] = make_float2(m, __int_as_float(code));
      code += 256;
      head = code < V * 256 ? next[code >> 8] : -INFINITY;
    }
  }
  __syncwarp();
  auto expert = [&](float2 c) {  // index of a choice
    const int l = __float_as_int(c.y) & 255;
    // of the values equal to it, the one that its rank in the lane leaves
    int skip = __float_as_int(c.y) >> 8, at = 0;
    float own[V];
#pragma unroll
    for (int v = 0; v < V; v += 4) *reinterpret_cast<float4*>(own + v) = *reinterpret_cast<float4*>(vals + l * V + v);
#pragma unroll
    for (int v = 0; v < V; ++v) skip -= own[v] > c.x;
#pragma unroll
    for (int v = 0; v < V; ++v) {
      const bool hit = own[v] == c.x;
      at = hit && skip == 0 ? v : at;
      skip -= hit;
    }
    return (l >> a.lpg_log2) * per + (l & ((1 << a.lpg_log2) - 1)) * a.cnt + at;
  };
  auto apart = [&](float u, float v) { return u - v > near + 0x1p-23f * (fabsf(u) + fabsf(v)) || v == -INFINITY; };
  bool tied = false;
  for (int q = lane; q < k; q += LANES) {
    const float2 c = rec[q];
    again |= c.x == -INFINITY;
    const int e = expert(c);
    s_id[sub][q] = e;
    if (a.bias && q + 1 < rounds) {
      const float2 d = rec[q + 1];
      if (!apart(c.x, d.x)) {
        // the same logit and the same bias tie for certain, and stand in order of index
        const int j = expert(d);
        const bool same = to_f32(row[e]) == to_f32(row[j]) && a.bias[e] == a.bias[j];
        again |= !same;
        tied |= same && q == k - 1;
      }
    }
  }
  if (__any_sync(kFull, tied)) {
    // equal to the last choice is the first left out: certain where all that follows as closely is equal too
    __syncwarp();
    const float last = rec[k - 1].x;
    const int e = s_id[sub][k - 1];
    if ((__ballot_sync(kFull, tied) & mask) && kept) {
      for (int v = 0; v < have; ++v) {
        const float c = vals[lane * V + v];
        if (c > last || apart(last, c)) continue;
        again |= !(to_f32(row[e]) == to_f32(row[first + v]) && a.bias[e] == a.bias[first + v]);
      }
    }
  }
  again = (__ballot_sync(kFull, again) & mask) != 0;
  for (unsigned todo = __ballot_sync(kFull, again && lane == 0); todo; todo &= todo - 1) {
    const int from = __ffs(todo) - 1;                                // the whole warp, token after token
    const int64_t t = __shfl_sync(kFull, r, from);
    select_f64<T>(a, static_cast<const T*>(a.z) + t * a.ld, s_key[threadIdx.x / 32],
                  s_id[(threadIdx.x - wl + from) / LANES]);
  }
  __syncwarp();

  constexpr int NQ = (MOST + LANES - 1) / LANES;                     // choices of a lane: lane, lane + LANES, ...
  int id[NQ];
#pragma unroll
  for (int i = 0; i < NQ; ++i) id[i] = lane + i * LANES < k ? s_id[sub][lane + i * LANES] : 0;
  write_weights<LANES, NQ>(a, row, r, want < a.n, lane, id, base, inv, odd);
}

// Long batches, up to 8 choices: four lanes a token, eight tokens a warp, so
// that few instructions go across lanes.  A lane holds 8 consecutive experts of
// each of NC chunks of 32 as keys that carry their index, and hence all differ:
// steps of the value below the row's largest, over the index from the top
// (16-bit logits without a bias: the 16 bits themselves, exact).  Every chunk
// is sorted in a lane, then the eight largest are merged over the chunks and
// over the lanes.  Of what the merges leave out the largest is kept, and with a
// bias the two largest, which costs 5% of the throughput: where the first places
// of these ten that hold all choices are apart from the rest, a token whose
// order is in doubt is settled by its own lanes, and no warp is alone with it at
// the end.  us before and after: 16384 rows of 256 with sigmoid, bias and groups
// 18.8, 17.6 (16 to 19: what is left are groups in doubt, some in a call or
// none); bf16 with a bias of zero (ties), 8192 rows, sigmoid 19.8, 14.4, softmax
// 23.4, 15.9; without a bias, bf16 values in fp32, 13.0, 5.6.
constexpr int kRowLanes = 4, kRowMost = 8;

template <int A, int B>
__device__ __forceinline__ void order_keys(uint32_t (&x)[8]) {
  const uint32_t a = x[A], b = x[B];
  x[A] = max(a, b);
  x[B] = min(a, b);
}
template <size_t... I>
__device__ __forceinline__ void sort_keys(uint32_t (&x)[8], std::index_sequence<I...>) {
  constexpr Network<8> net;
  (order_keys<net.a[I], net.b[I]>(x), ...);
}
__device__ __forceinline__ void sort_keys(uint32_t (&x)[8]) {
  sort_keys(x, std::make_index_sequence<Network<8>().n>());
}
// The 8 largest of two descending lists, descending; the two largest of the
// others join `out`, `out2` (with a bias: nothing else asks for them).
template <bool BIAS>
__device__ __forceinline__ void merge_keys(uint32_t (&x)[8], const uint32_t (&y)[8], uint32_t& out, uint32_t& out2) {
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const uint32_t a = x[i], b = y[7 - i], low = min(a, b);
    x[i] = max(a, b);
    if (BIAS) out2 = max(out2, min(out, low));
    out = max(out, low);
  }
  order_keys<0, 4>(x), order_keys<1, 5>(x), order_keys<2, 6>(x), order_keys<3, 7>(x);
  order_keys<0, 2>(x), order_keys<1, 3>(x), order_keys<4, 6>(x), order_keys<5, 7>(x);
  order_keys<0, 1>(x), order_keys<2, 3>(x), order_keys<4, 5>(x), order_keys<6, 7>(x);
}

template <typename T>
__device__ __forceinline__ uint32_t order16(float z) {
  uint32_t u;
  if constexpr (std::is_same<T, __half>::value) u = __half_as_ushort(__float2half_rn(z));
  else u = __float_as_uint(z) >> 16;
  return u & 0x8000u ? 0xFFFFu - u : u | 0x8000u;
}

// A choice's score + bias in fp64.
template <typename T>
__device__ __noinline__ double sigmoid_f64(const T* row, const float* bias, int e) {
  return 1.0 / (1.0 + exp(-double(to_f32(row[e])))) + double(bias[e]);
}

template <typename T, int NC, bool BIAS>
__global__ void __launch_bounds__(kRouterThreads) router_rows_kernel(const __grid_constant__ RouterArgs a) {
  constexpr int PER_WARP = 32 / kRowLanes, WARPS = kRouterThreads / 32;
  constexpr int IB = NC <= 8 ? 8 : 9;                    // bits of the index
  constexpr uint32_t kLast = (1u << IB) - 1u;
  constexpr uint32_t kNoStep = 0x80000000u + (1u << IB);  // smaller keys: the lowest step
  __shared__ __align__(16) uint32_t s_list[WARPS][PER_WARP][12];
  __shared__ int32_t s_id[WARPS][PER_WARP][kRowMost];
  __shared__ uint64_t s_key[WARPS][NC * 32 < 96 ? 96 : NC * 32];
  const int wl = threadIdx.x & 31, warp = threadIdx.x >> 5, lane = wl & (kRowLanes - 1), sub = wl / kRowLanes;
  const int64_t want = (int64_t(blockIdx.x) * WARPS + warp) * PER_WARP + sub;
  const int64_t r = want < a.n ? want : a.n - 1;
  const T* row = static_cast<const T*>(a.z) + r * a.ld;
  const int E = a.experts, k = a.topk, chunks = (E + 31) / 32;
  const bool exact = sizeof(T) == 2 && !BIAS;

  float x[NC][8];
  float top = -INFINITY;  // a NaN if there is one
#pragma unroll
  for (int c = 0; c < NC; ++c) {
    const int first = c * 32 + lane * 8;
    load_row<T, 8>(row, first, E - first, a.vec, x[c]);
  }
#pragma unroll
  for (int c = 0; c < NC; ++c)
#pragma unroll
    for (int v = 0; v < 8; ++v) top = max_nan(top, x[c][v]);
#pragma unroll
  for (int o = 1; o < kRowLanes; o <<= 1) top = max_nan(top, __shfl_xor_sync(kFull, top, o));
  const float base = top == -INFINITY ? 0.0f : top;
  const bool odd = !a.sigmoid && !(top < INFINITY);  // a NaN or +inf: softmax has no value
  float inv = 0.0f;
  if (!a.sigmoid && (BIAS || !a.renorm)) {
    float sum = 0.0f;
#pragma unroll
    for (int c = 0; c < NC; ++c)
#pragma unroll
      for (int v = 0; v < 8; ++v) {
        const float f = exp_fast(x[c][v] - base);
        sum += f;
        if (BIAS) x[c][v] = f;
      }
    sum = lanes_sum<kRowLanes>(sum);
    inv = sum > 0.0f ? 1.0f / sum : 0.0f;
  }
  float near = 0.0f, largest = top;
  bool again = !exact && !(top < INFINITY);  // selected again with scores in fp64: all of it
  if (BIAS) {
    largest = -INFINITY;
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      const int first = c * 32 + lane * 8;
      float b[8];
      load_row<float, 8>(a.bias, first, E - first, a.vec_bias, b);
#pragma unroll
      for (int v = 0; v < 8; ++v) {
        x[c][v] = a.sigmoid ? sigmoid_fast(x[c][v]) + b[v] : fmaf(x[c][v], inv, b[v]);
        largest = fmaxf(largest, x[c][v]);
      }
    }
    largest = lanes_max<kRowLanes>(largest);
    // as in router_topk_kernel; a softmax's sum has 8 NC + 2 roundings here
    const float big = a.sigmoid ? sigmoid_fast(top) : inv;
    near = 0x1p-24f * big * (a.sigmoid ? 14.0f + 3.0f * fmaxf(0.0f, -top) : 16.0f * NC + 40.0f) +
           0x1p-23f * (fabsf(largest) + 2.0f);
    again |= a.sigmoid && top < -80.0f;
  }

  // values of 16 below the largest logit, of 2 below the largest s + bias,
  // share the lowest step: where that is chosen, or holds the best of a group,
  // the slow selection decides (16384 x 256 fp32, logits of standard deviation
  // 1.5, 5 and 10: 8.4, 16.5, 37 us; a group switched off: 117)
  const float scale = BIAS ? 0.5f : 0.0625f, steps = scale * float(1u << (31 - IB));
  const float shift = __fmaf_rd(-largest, scale, 1.0f - 0x1p-22f);  // down: no value reaches 1
  uint32_t key[NC][8];
#pragma unroll
  for (int c = 0; c < NC; ++c) {
    const int first = c * 32 + lane * 8;
    if (exact) {
      const uint32_t last = 0xFFFFu - first;
#pragma unroll
      for (int v = 0; v < 8; ++v) key[c][v] = (order16<T>(fmaxf(x[c][v] + 0.0f, -INFINITY)) << 16) + (last - v);
    } else {
      // 1 + a fraction clamped to 0 .. 1: the float's low 23 bits count the steps
      const uint32_t last = kLast - first;
#pragma unroll
      for (int v = 0; v < 8; ++v) {
        const uint32_t u = __float_as_uint(1.0f + __saturatef(fmaf(x[c][v], scale, shift)));
        key[c][v] = (IB == 8 ? u * 256u : (u & ~1u) * 256u | 0x80000000u) + (last - v);
      }
    }
    if (c >= chunks - 1) {
#pragma unroll
      for (int v = 0; v < 8; ++v) key[c][v] = first + v < E ? key[c][v] : 0u;
    }
    sort_keys(key[c]);
  }

  uint32_t kept = 1;
  if (a.groups > 1) {
    // a group is a.cnt whole chunks: its two best over its chunks and the
    // lanes; steps and index in one word, so that all differ
    uint32_t score[NC], order[8];
    int in = 0;
    uint32_t b1 = 0, b2 = 0;
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      b2 = max(max(b2, key[c][1]), min(b1, key[c][0]));
      b1 = max(b1, key[c][0]);
      score[c] = 0;
      if (++in == a.cnt && c < chunks) {
#pragma unroll
        for (int o = 1; o < kRowLanes; o <<= 1) {
          const uint32_t o1 = __shfl_xor_sync(kFull, b1, o), o2 = __shfl_xor_sync(kFull, b2, o);
          b2 = max(min(b1, o1), max(b2, o2));
          b1 = max(b1, o1);
        }
        again |= !exact && (a.top2 ? b2 : b1) < kNoStep;
        // steps without bit 31 (16-bit logits as they are)
        const uint32_t s1 = exact ? b1 >> 16 : (b1 & 0x7FFFFFFFu) >> IB, s2 = (b2 & 0x7FFFFFFFu) >> IB;
        score[c] = (a.top2 ? s1 + s2 : s1) << 3 | (7u - c);
        b1 = b2 = 0;
        in = 0;
      }
    }
#pragma unroll
    for (int c = 0; c < 8; ++c) order[c] = c < NC ? score[c < NC ? c : 0] : 0u;
    sort_keys(order);
    uint32_t low = order[0], high = order[1];
#pragma unroll
    for (int c = 1; c < 7; ++c)
      if (a.topk_groups == c + 1) low = order[c], high = order[c + 1];
    // steps apart by which the order is certain: of sums of two rounded values
    if (!exact) again |= float((low >> 3) - (high >> 3)) <= 2.0f * near * steps + (BIAS ? 2.0f : 0.0f);
    kept = 0;
    bool mine = false;
    int g = a.groups, left = 0;
#pragma unroll
    for (int c = NC - 1; c >= 0; --c) {
      if (c < chunks && left-- == 0) {  // the last chunk of a group, which has its score
        mine = score[c] >= low;
        kept |= uint32_t(mine) << --g;
        left = a.cnt - 1;
      }
#pragma unroll
      for (int v = 0; v < 8; ++v) key[c][v] = mine ? key[c][v] : 0u;
    }
  }

  uint32_t out = 0, out2 = 0;
#pragma unroll
  for (int c = 1; c < NC; ++c)
    if (c < chunks) merge_keys<BIAS>(key[0], key[c], out, out2);
#pragma unroll
  for (int o = 1; o < kRowLanes; o <<= 1) {
    uint32_t other[8];
#pragma unroll
    for (int v = 0; v < 8; ++v) other[v] = __shfl_xor_sync(kFull, key[0][v], o);
    const uint32_t its = __shfl_xor_sync(kFull, out, o);
    if (BIAS) out2 = max(min(out, its), max(out2, __shfl_xor_sync(kFull, out2, o)));
    out = max(out, its);
    merge_keys<BIAS>(key[0], other, out, out2);
  }

  // every lane of the token holds the list: through shared memory, two choices a lane
  uint32_t* list = s_list[warp][sub];
  if (lane == 0) {
    *reinterpret_cast<uint4*>(list) = make_uint4(key[0][0], key[0][1], key[0][2], key[0][3]);
    *reinterpret_cast<uint4*>(list + 4) = make_uint4(key[0][4], key[0][5], key[0][6], key[0][7]);
    list[8] = out;
    list[9] = out2;
  }
  __syncwarp();
  auto index = [&](uint32_t key) { return exact ? int(0xFFFFu - (key & 0xFFFFu)) : int(kLast - (key & kLast)); };
  int id[2];
  unsigned pairs = 0;  // bit q: places q and q + 1 may be the other way round; bit 16 + q: and are not equal
  auto look = [&](int q) {
    const uint32_t mine = list[q], then = list[q + 1];
    if (then == 0 || float((mine >> IB) - (then >> IB)) > near * steps + (BIAS ? 1.0f : 0.0f)) return;
    // the same logit and the same bias tie for certain, and stand in order of index
    const int e = index(mine), f = index(then);
    const bool same = to_f32(row[e]) == to_f32(row[f]) && (!BIAS || a.bias[e] == a.bias[f]);
    pairs |= (same ? 1u : 0x10001u) << q;
  };
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int q = lane + i * kRowLanes;
    id[i] = q >= k ? 0 : index(list[q]);
    if (!exact) {
      again |= q < k && list[q] < kNoStep;
      look(q);
    }
    s_id[warp][sub][q] = id[i];
  }
  if (BIAS && lane == 0) look(8);
  const unsigned group_lanes = (1u << kRowLanes) - 1u;
  bool close = (pairs >> 16 & ((1u << k) - 1u)) || (pairs >> (k - 1) & 1u);
  if (__any_sync(kFull, close)) {
    // the first `count` places hold what they should: certain where those in doubt are equal
    constexpr int MOST = BIAS ? 9 : 8;
#pragma unroll
    for (int o = 1; o < kRowLanes; o <<= 1) pairs |= __shfl_xor_sync(kFull, pairs, o);
    const int count = k + __ffs(~(pairs >> (k - 1) & 0xFFFFu)) - 1;
    close = count > MOST || (pairs >> 16 & ((1u << (count - 1)) - 1u));
    const bool few = close && !(pairs >> 16 & ((1u << (k - 1)) - 1u));
    if (!BIAS && __any_sync(kFull, few)) {
      // only the last choice: certain where as many logits are above it as there are choices above it
      const float last = to_f32(row[index(list[k - 1])]);
      int above = 0;
      if (few) {
#pragma unroll 16
        for (int e = lane; e < E; e += kRowLanes)
          above += to_f32(row[e]) > last && (a.groups == 1 || (kept >> (e / a.per) & 1u));
      }
#pragma unroll
      for (int i = 0; i < 2; ++i) above -= lane + i * kRowLanes < k && to_f32(row[id[i]]) > last;
      above = lanes_sum<kRowLanes>(above);
      if (few && above == 0) close = false;
    }
  }
  if (BIAS && a.sigmoid && __any_sync(kFull, close)) {
    // ... else settled among them, by every token at once
    const int count = k + __ffs(~(pairs >> (k - 1) & 0xFFFFu)) - 1;
    const bool here = close && count <= 9;
    double* value = reinterpret_cast<double*>(s_key[warp]) + sub * 12;
    if (here) {
#pragma unroll 1
      for (int q = lane; q < count; q += kRowLanes) value[q] = sigmoid_f64(row, a.bias, index(list[q]));
    }
    __syncwarp();
    if (here) {
#pragma unroll 1
      for (int q = lane; q < count; q += kRowLanes) {
        const int e = index(list[q]);
        const double x = value[q];
        int rank = 0;
#pragma unroll 1
        for (int i = 0; i < count; ++i) rank += value[i] > x || (value[i] == x && index(list[i]) < e);
        if (rank < k) s_id[warp][sub][rank] = e;
      }
      close = false;
    }
    __syncwarp();
#pragma unroll
    for (int i = 0; i < 2; ++i) id[i] = lane + i * kRowLanes < k ? s_id[warp][sub][lane + i * kRowLanes] : 0;
  }
  const unsigned slow = __ballot_sync(kFull, again), any = slow | __ballot_sync(kFull, close);
  if (any) {
    // a value below the last choice by more than what makes an order uncertain
    const float from =
        largest + (float((list[k - 1] & 0x7FFFFFFFu) >> IB) - float(1u << (31 - IB)) - near * steps - 4.0f) / steps;
    __syncwarp();
#pragma unroll 1
    for (int i = 0; i < PER_WARP; ++i) {  // the whole warp, token after token
      const int lead = i * kRowLanes;
      if (!(any >> lead & group_lanes)) continue;
      const int64_t t = __shfl_sync(kFull, r, lead);
      const T* its = static_cast<const T*>(a.z) + t * a.ld;
      const float its_from = __shfl_sync(kFull, from, lead), its_base = __shfl_sync(kFull, base, lead);
      const float its_inv = __shfl_sync(kFull, inv, lead);
      const uint32_t its_kept = __shfl_sync(kFull, kept, lead);
      if ((slow >> lead & group_lanes) ||
          !order_near<T>(a, its, its_from, its_kept, its_base, its_inv, a.groups > 1 ? a.per : 512,
                         reinterpret_cast<uint32_t*>(s_key[warp]), s_id[warp][i]))
        select_f64<T>(a, its, s_key[warp], s_id[warp][i]);
    }
#pragma unroll
    for (int i = 0; i < 2; ++i) id[i] = lane + i * kRowLanes < k ? s_id[warp][sub][lane + i * kRowLanes] : 0;
  }
  write_weights<kRowLanes, 2>(a, row, r, want < a.n, lane, id, base, inv, odd);
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

// Gradient of the logits from that of the weights.  With w = scale * p:
//   softmax:              dz_i = w_i (dw_i - sum(p dw)) of the chosen, -s_i sum(w dw) of the others
//   softmax, renormalised dz_i = w_i (dw_i - sum(p dw)) of the chosen, else 0
//   sigmoid:              dz_i = scale dw_i s_i (1 - s_i)
//   sigmoid, renormalised dz_i = w_i (1 - s_i) (dw_i - sum(p dw))
// The row is put together in shared memory, the chosen over the others, and
// leaves in vectors.  LANES lanes a token hold NC chunks of 8 experts each.  The
// dense gradient lives on loads in flight: a persistent grid, every group of
// lanes reading its next token while it works on one.
template <typename T>
__device__ __forceinline__ void unpack16(const uint4& w, float* x) {
  const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (sizeof(T) == 4) {
      x[i] = __uint_as_float(u[i]);
    } else if constexpr (std::is_same<T, __half>::value) {
      const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&u[i]));
      x[2 * i] = f.x, x[2 * i + 1] = f.y;
    } else {
      x[2 * i] = bf16_lo(u[i]), x[2 * i + 1] = bf16_hi(u[i]);
    }
  }
}
template <typename T>
__device__ __forceinline__ uint4 pack16(const float* x) {
  uint32_t u[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (sizeof(T) == 4) {
      u[i] = __float_as_uint(x[i]);
    } else if constexpr (std::is_same<T, __half>::value) {
      const __half2 h = __floats2half2_rn(x[2 * i], x[2 * i + 1]);
      u[i] = *reinterpret_cast<const uint32_t*>(&h);
    } else {
      u[i] = pack2_bf16(x[2 * i], x[2 * i + 1]);
    }
  }
  return make_uint4(u[0], u[1], u[2], u[3]);
}

template <typename T, int LANES, int NC, bool DENSE>
__global__ void __launch_bounds__(kRouterThreads, DENSE ? 6 : 8) router_bwd_kernel(const __grid_constant__ RouterBwdArgs a) {
  constexpr int ROWS = kRouterThreads / LANES, MOST = LANES * NC * 8;
  constexpr int NQ = ((MOST < 32 ? MOST : 32) + LANES - 1) / LANES;
  constexpr int P = 16 / sizeof(T), NW = NC * 8 / P;                 // elements a vector, vectors a lane
  __shared__ __align__(16) T s_row[ROWS][MOST];
  __shared__ uint8_t s_at[ROWS][MOST];                               // which choice names an expert
  const int lane = threadIdx.x % LANES, sub = threadIdx.x / LANES;
  const unsigned mask = LANES == 32 ? kFull : ((1u << (LANES & 31)) - 1u) << ((threadIdx.x & 31) / LANES * LANES);
  const int E = a.experts, k = a.topk;
  T* mine = s_row[sub];
  // vector i of a lane: consecutive experts, neighbours in neighbouring lanes
  auto place = [&](int i) { return a.vec ? (i * LANES + lane) * P : i * P * LANES + lane; };

  // no expert: -inf throughout
  const uint32_t inf = sizeof(T) == 4 ? 0xFF800000u : std::is_same<T, __half>::value ? 0xFC00FC00u : 0xFF80FF80u;
  const uint4 none = make_uint4(inf, inf, inf, inf);
  uint4 raw[NW];
  int id[NQ];
  float wq[NQ], dq[NQ];
  auto fetch = [&](int64_t r) {
    const T* row = static_cast<const T*>(a.z) + r * a.ld;
    if constexpr (DENSE) {
#pragma unroll
      for (int i = 0; i < NW; ++i) {
        const int e0 = place(i);
        if (a.vec) {
          raw[i] = e0 < E ? __ldg(reinterpret_cast<const uint4*>(row + e0)) : none;
        } else {
          raw[i] = none;
#pragma unroll
          for (int v = 0; v < P; ++v)
            if (e0 + v * LANES < E) reinterpret_cast<T*>(&raw[i])[v] = row[e0 + v * LANES];
        }
      }
    }
#pragma unroll
    for (int i = 0; i < NQ; ++i) {
      const int q = lane + i * LANES;
      id[i] = -1;
      wq[i] = dq[i] = 0.0f;
      if (i * LANES >= k || q >= k) continue;
      id[i] = a.ids[r * k + q];
      wq[i] = a.weights[r * k + q];
      dq[i] = a.dweights[r * k + q];
    }
  };
  const int64_t step = int64_t(gridDim.x) * ROWS;
  int64_t want = int64_t(blockIdx.x) * ROWS + sub;
  fetch(want < a.n ? want : a.n - 1);
  // as many turns for all lanes of a warp: they reduce together
  for (int64_t base_row = int64_t(blockIdx.x) * ROWS; base_row < a.n; base_row += step, want += step) {
    const bool real = want < a.n;
    const int64_t r = real ? want : a.n - 1;
    const T* row = static_cast<const T*>(a.z) + r * a.ld;
    float z[NW][P], g[NQ], pull = 0.0f;
#pragma unroll
    for (int i = 0; i < NW; ++i)
      if constexpr (DENSE) unpack16<T>(raw[i], z[i]);
#pragma unroll
    for (int i = 0; i < NQ; ++i) {
      if (i * LANES >= k) continue;
      const int q = lane + i * LANES;
      if (q < k && (id[i] < 0 || id[i] >= E)) {
        id[i] = -1;
        if (real) atomicCAS(a.err, 0, MXG_ERR_INVALID_ARGUMENT);
      }
      g[i] = !DENSE && a.sigmoid && id[i] >= 0 ? to_f32(row[id[i]]) : 0.0f;
      if (id[i] >= 0) s_at[sub][id[i]] = uint8_t(q);
      pull += wq[i] * dq[i];
    }
    pull = lanes_sum<LANES>(pull);
    const float mean = pull / a.scale;
    int at[NQ];
#pragma unroll
    for (int i = 0; i < NQ; ++i) {
      at[i] = i * LANES < k ? id[i] : -1;
      if (DENSE || !a.sigmoid) g[i] = wq[i] * (dq[i] - mean);
      else if (a.renorm) g[i] = wq[i] * (dq[i] - mean) * sigmoid_f32(-g[i]);
      else g[i] = a.scale * dq[i] * sigmoid_f32(g[i]) * sigmoid_f32(-g[i]);
    }
    if (base_row + step < a.n) fetch(want + step < a.n ? want + step : a.n - 1);
    float by = 0.0f;
    if constexpr (DENSE) {
      float top = -INFINITY, sum = 0.0f;
#pragma unroll
      for (int i = 0; i < NW; ++i)
#pragma unroll
        for (int v = 0; v < P; ++v) top = fmaxf(top, z[i][v]);
      top = lanes_max<LANES>(top);
      // exp(z - top) as 2^(z log2 e - top log2 e) with one rounding: that of
      // top log2 e is common to all, and falls out of the quotient.  It is at
      // most 2^5 below 2^30; from there on logits that differ do so by 64 or
      // more, and 2^(z - top), which is exact, tells them apart as well (2^-64
      // for e^-64).  (A subtraction first costs an instruction an element:
      // 65536 x 256 bf16 15.8 -> 18.9 us.)
      const float product = 1.44269504f * top;
      const bool far = !(fabsf(product) < 0x1p30f);
      const float by2 = far ? 1.0f : 1.44269504f, base = top == -INFINITY ? 0.0f : far ? -top : -product;
#pragma unroll
      for (int i = 0; i < NW; ++i) {
        float part = 0.0f;
#pragma unroll
        for (int v = 0; v < P; ++v) part += z[i][v] = exp2_fast(fmaf(z[i][v], by2, base));
        sum += part;
      }
      sum = lanes_sum<LANES>(sum);
      by = sum == 0.0f ? 0.0f : -pull / sum;
    }
#pragma unroll
    for (int i = 0; i < NW; ++i) {
      const int e0 = place(i);
      uint4 t = make_uint4(0, 0, 0, 0);
      if constexpr (DENSE) {
#pragma unroll
        for (int v = 0; v < P; ++v) z[i][v] *= by;
        t = pack16<T>(z[i]);
      }
      if (a.vec) {
        *reinterpret_cast<uint4*>(mine + e0) = t;
      } else {
#pragma unroll
        for (int v = 0; v < P; ++v) mine[e0 + v * LANES] = reinterpret_cast<const T*>(&t)[v];
      }
    }
    __syncwarp();
    bool twice = false;
#pragma unroll
    for (int i = 0; i < NQ; ++i) {
      if (at[i] < 0) continue;
      twice |= s_at[sub][at[i]] != lane + i * LANES;
      from_f32(g[i], mine[at[i]]);
    }
    // an expert that is named more than once gets the sum, choice after choice
    const unsigned again = __ballot_sync(kFull, twice) & mask;
    if (again) {
      __syncwarp(mask);  // lane 0 writes after the others
      const float *w = a.weights + r * k, *dw = a.dweights + r * k;
      const int32_t* ids = a.ids + r * k;
      for (int q = 0; q < k && lane == 0; ++q) {
        const int e = ids[q];
        if (e < 0 || e >= E) continue;
        const float x = a.sigmoid ? to_f32(row[e]) : 0.0f;
        float sum = DENSE ? -mean * w[q] : 0.0f;  // of an expert that is not chosen
        for (int h = 0; h < k; ++h) {
          if (ids[h] != e) continue;
          if (DENSE) sum += w[h] * dw[h];
          else if (!a.sigmoid) sum += w[h] * (dw[h] - mean);
          else if (a.renorm) sum += w[h] * (dw[h] - mean) * sigmoid_f32(-x);
          else sum += a.scale * dw[h] * sigmoid_f32(x) * sigmoid_f32(-x);
        }
        from_f32(sum, mine[e]);
      }
    }
    __syncwarp();
    T* out = static_cast<T*>(a.dz) + r * a.ld_out;
    if (!real) {
    } else if (a.vec_out) {
#pragma unroll
      for (int i = 0; i < NW; ++i) {
        const int e = (i * LANES + lane) * P;
        if (e < E) *reinterpret_cast<uint4*>(out + e) = *reinterpret_cast<const uint4*>(mine + e);
      }
    } else {
      for (int e = lane; e < E; e += LANES) out[e] = mine[e];
    }
    __syncwarp();
  }
}

// Rows can be read as vectors: v consecutive elements a lane throughout, every
// row on a 16-byte boundary.
inline bool rows_vectorised(const void* p, int64_t ld, int v, size_t size) {
  return (size_t(ld) * size) % 16 == 0 && aligned16(p);
}

// Lanes and experts a lane of a token whose groups fill whole lanes.  False:
// LANES * V are too few.
inline bool lay_out(RouterArgs& a, int lanes, int v) {
  if (a.groups > lanes) return false;
  int log2 = 0;
  while (a.groups << (log2 + 1) <= lanes) ++log2;
  a.per = a.experts / a.groups;
  a.lpg_log2 = log2;
  a.cnt = (a.per + (1 << log2) - 1) >> log2;
  if (a.cnt > v) return false;
  if (a.per % v == 0) a.cnt = v;  // fewer lanes, but whole vectors
  return true;
}

template <typename T, int LANES, int V>
int launch_topk(RouterArgs& a, cudaStream_t s) {
  const bool whole = a.cnt == V && a.per % V == 0;
  a.vec = whole && rows_vectorised(a.z, a.ld, V, sizeof(T));
  a.vec_bias = whole && aligned16(a.bias);
  const int64_t blocks = (a.n + kRouterThreads / LANES - 1) / (kRouterThreads / LANES);
  router_topk_kernel<T, LANES, V><<<unsigned(blocks), kRouterThreads, 0, s>>>(a);
  return cuda_status(cudaGetLastError());
}

template <typename T, int NC>
int launch_rows(RouterArgs& a, cudaStream_t s) {
  a.vec = a.experts % 8 == 0 && rows_vectorised(a.z, a.ld, 8, sizeof(T));
  a.vec_bias = a.experts % 8 == 0 && aligned16(a.bias);
  a.cnt = a.per / 32;
  const int rows = kRouterThreads / kRowLanes;
  const unsigned blocks = unsigned((a.n + rows - 1) / rows);
  if (a.bias) router_rows_kernel<T, NC, true><<<blocks, kRouterThreads, 0, s>>>(a);
  else router_rows_kernel<T, NC, false><<<blocks, kRouterThreads, 0, s>>>(a);
  return cuda_status(cudaGetLastError());
}

template <typename T, int LANES, int NC>
int launch_bwd(RouterBwdArgs& a, cudaStream_t s) {
  a.vec = a.experts % 8 == 0 && rows_vectorised(a.z, a.ld, 8, sizeof(T));
  a.vec_out = a.experts % 8 == 0 && rows_vectorised(a.dz, a.ld_out, 8, sizeof(T));
  const int64_t blocks = std::min<int64_t>((a.n + kRouterThreads / LANES - 1) / (kRouterThreads / LANES),
                                           int64_t(num_sms()) * 8);
  if (!a.sigmoid && !a.renorm) router_bwd_kernel<T, LANES, NC, true><<<unsigned(blocks), kRouterThreads, 0, s>>>(a);
  else router_bwd_kernel<T, LANES, NC, false><<<unsigned(blocks), kRouterThreads, 0, s>>>(a);
  return cuda_status(cudaGetLastError());
}

// The fewest lanes that hold a token's experts, 8 a lane (up to 24 beyond).
template <typename T>
int topk_by_experts(RouterArgs& a, cudaStream_t s) {
  a.per = a.experts / a.groups;
  // Four lanes a token or all of a warp, us at (tokens, experts), fp32 logits
  // with sigmoid scores: (4, 128) 2.8 / 3.3, (65536, 128) 12 / 27; (2048, 256)
  // 4.1 / 3.5, (4096, 256) 4.2 / 4.5, (16384, 256) 7.5 / 12.2, (65536, 256)
  // 19 / 42; (4096, 384) 6.1 / 5.2, (16384, 384) 10.4 / 14.1: a warp a token
  // has the shorter chain, four lanes fewer instructions.
  const int64_t rows_from = a.experts <= 128 ? 1 : a.experts <= 256 ? 4096 : 8192;
  if (a.n >= rows_from && a.experts > 16 && a.topk <= kRowMost &&
      (a.groups == 1 || (a.per % 32 == 0 && (a.bias || !a.top2) && a.experts <= 256)))
    return a.experts <= 32    ? launch_rows<T, 1>(a, s)
           : a.experts <= 64  ? launch_rows<T, 2>(a, s)
           : a.experts <= 128 ? launch_rows<T, 4>(a, s)
           : a.experts <= 256 ? launch_rows<T, 8>(a, s)
                              : launch_rows<T, 12>(a, s);
  if (lay_out(a, 1, 8)) return launch_topk<T, 1, 8>(a, s);
  if (lay_out(a, 2, 8)) return launch_topk<T, 2, 8>(a, s);
  if (lay_out(a, 4, 8)) return launch_topk<T, 4, 8>(a, s);
  if (lay_out(a, 8, 8)) return launch_topk<T, 8, 8>(a, s);
  if (lay_out(a, 16, 8)) return launch_topk<T, 16, 8>(a, s);
  if (lay_out(a, 32, 8)) return launch_topk<T, 32, 8>(a, s);
  if (lay_out(a, 32, 12)) return launch_topk<T, 32, 12>(a, s);
  if (lay_out(a, 32, 16)) return launch_topk<T, 32, 16>(a, s);
  if (lay_out(a, 32, 24)) return launch_topk<T, 32, 24>(a, s);
  return MXG_ERR_BAD_SHAPE;
}

template <typename T>
int bwd_by_experts(RouterBwdArgs& a, cudaStream_t s) {
  if (a.experts <= 8) return launch_bwd<T, 1, 1>(a, s);
  if (a.experts <= 32) return launch_bwd<T, 4, 1>(a, s);
  if (a.experts <= 64) return launch_bwd<T, 8, 1>(a, s);
  if (a.experts <= 128) return launch_bwd<T, 16, 1>(a, s);
  if (a.experts <= 256) return launch_bwd<T, 16, 2>(a, s);
  return launch_bwd<T, 16, 3>(a, s);
}

int router_shape(const mxg_router_args* a) {
  if (!a) return MXG_ERR_INVALID_ARGUMENT;
  if (a->n_tokens < 0 || a->num_experts < 1 || a->topk < 1 ||
      (a->dtype != MXG_DTYPE_BF16 && a->dtype != MXG_DTYPE_F16 && a->dtype != MXG_DTYPE_F32) ||
      (a->score != MXG_SCORE_SOFTMAX && a->score != MXG_SCORE_SIGMOID) || !(a->scale > 0.0f) || !std::isfinite(a->scale))
    return MXG_ERR_INVALID_ARGUMENT;
  if (a->num_experts > MXG_EP_MAX_EXPERTS || a->topk > a->num_experts || a->topk > MXG_ROUTER_MAX_TOPK ||
      a->n_tokens > INT32_MAX || a->ld < a->num_experts)
    return MXG_ERR_BAD_SHAPE;
  return MXG_OK;
}

}  // namespace mxg

using namespace mxg;

extern "C" int mxg_router_topk(const mxg_router_args* args, void* stream) {
  int st = router_shape(args);
  if (st) return st;
  const mxg_router_args& r = *args;
  if (r.groups < 1 || r.topk_groups < 1 || r.topk_groups > r.groups ||
      (r.group_score != MXG_GROUP_MAX && r.group_score != MXG_GROUP_TOP2))
    return MXG_ERR_INVALID_ARGUMENT;
  if (r.groups > MXG_ROUTER_MAX_GROUPS || r.num_experts % r.groups ||
      r.topk > r.topk_groups * (r.num_experts / r.groups))
    return MXG_ERR_BAD_SHAPE;
  if (r.n_tokens == 0) return MXG_OK;
  if (!r.logits || !r.weights || !r.ids) return MXG_ERR_INVALID_ARGUMENT;
  if ((st = check_device())) return st;
  RouterArgs a{};
  a.z = r.logits, a.ld = r.ld, a.n = r.n_tokens, a.experts = r.num_experts, a.topk = r.topk;
  a.groups = r.topk_groups == r.groups ? 1 : r.groups;  // all groups stay: no groups
  a.topk_groups = r.topk_groups == r.groups ? 1 : r.topk_groups;
  a.top2 = r.group_score == MXG_GROUP_TOP2, a.sigmoid = r.score == MXG_SCORE_SIGMOID, a.renorm = r.renormalize != 0;
  a.scale = r.scale, a.bias = r.bias, a.weights = r.weights, a.ids = r.ids;
  a.rounds = r.topk + (r.bias && r.topk < a.topk_groups * (r.num_experts / a.groups) ? 1 : 0);
  cudaStream_t s = (cudaStream_t)stream;
  return r.dtype == MXG_DTYPE_BF16  ? topk_by_experts<__nv_bfloat16>(a, s)
         : r.dtype == MXG_DTYPE_F16 ? topk_by_experts<__half>(a, s)
                                    : topk_by_experts<float>(a, s);
}

extern "C" int mxg_router_topk_bwd(const mxg_router_args* args, void* stream) {
  int st = router_shape(args);
  if (st) return st;
  const mxg_router_args& r = *args;
  if (r.ld_out < r.num_experts) return MXG_ERR_BAD_SHAPE;
  if (r.n_tokens == 0) return MXG_OK;
  if (!r.logits || !r.weights || !r.ids || !r.dweights || !r.dlogits) return MXG_ERR_INVALID_ARGUMENT;
  if ((st = check_device())) return st;
  RouterBwdArgs a{};
  a.z = r.logits, a.ld = r.ld, a.n = r.n_tokens, a.ld_out = r.ld_out, a.experts = r.num_experts, a.topk = r.topk;
  a.sigmoid = r.score == MXG_SCORE_SIGMOID, a.renorm = r.renormalize != 0, a.scale = r.scale;
  a.weights = r.weights, a.ids = r.ids, a.dweights = r.dweights, a.dz = r.dlogits, a.err = device_error_word();
  if (!a.err) return MXG_ERR_CUDA;
  cudaStream_t s = (cudaStream_t)stream;
  return r.dtype == MXG_DTYPE_BF16  ? bwd_by_experts<__nv_bfloat16>(a, s)
         : r.dtype == MXG_DTYPE_F16 ? bwd_by_experts<__half>(a, s)
                                    : bwd_by_experts<float>(a, s);
}
