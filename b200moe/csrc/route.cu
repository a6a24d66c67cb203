// Routing to experts with a choice of scores, a balance bias, groups and any number of experts per token (``moe.cu`` and
// ``elementwise.cu`` hold the top-2 softmax router of the standard block).
//
//   s_e = sigmoid(x_e) or softmax(x)_e,   key_e = s_e + bias_e   (without a bias: x_e, whose order is that of s_e)
//   value of a group = its best key, or the sum of its two best;  the best groups stay, then the k best experts in them
//   w_i = scale * s_i / sum of the chosen s, or scale * s_i
//
// A warp works on one token and holds its logits in registers, so a row is read once and the choice takes k steps of a
// maximum over the lane's own values, a maximum over the warp and a removal.
//
// The choice is that of exact arithmetic.  Comparisons of logits are exact as they are.  Comparisons of scores (a bias, a
// sum of two) are made in fp32 first, and each of them that decided something is checked against a bound on the error of
// both sides; a row in which one is closer than that is worked out again in 64 bits by the same code.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <float.h>
#include <stdint.h>

#include "chain.cuh"

namespace b2 {

constexpr int ROUTE_MAX_K = 32;
constexpr unsigned ALL = 0xffffffffu;

enum LogitType : int { LOGIT_F32 = 0, LOGIT_BF16 = 1, LOGIT_F16 = 2 };
enum GroupMode : int { GROUPS_NONE = 0, GROUPS_ALIGNED = 1, GROUPS_ANY = 2 };

struct RouteParams {
  const void* logits;
  const float* bias;         // [E] or null
  float* weights;            // [T, k]
  long long* idx;            // [T, k]
  long long T;
  int E, k, type, sigmoid, groups, top_groups, two_best, renormalize;
  float scale;
};

// NaN counts as masked, infinity as the largest number.
__device__ __forceinline__ float route_clean(float x) { return x != x ? -INFINITY : fminf(x, FLT_MAX); }

__device__ __forceinline__ float load_logit(const void* p, int type, long long i) {
  float x;
  if (type == LOGIT_F32) x = static_cast<const float*>(p)[i];
  else if (type == LOGIT_BF16) x = __bfloat162float(static_cast<const __nv_bfloat16*>(p)[i]);
  else x = __half2float(static_cast<const __half*>(p)[i]);
  return route_clean(x);
}

// V values of a lane, -inf behind the last expert.  One access per lane and 16 bytes where the row allows it.
template <int V>
__device__ __forceinline__ void load_row(const void* p, int type, long long row, int E, int lane, float (&x)[V]) {
  const long long base = row * E;
  const int first = lane * V;
  const int size = type == LOGIT_F32 ? 4 : 2;
  if (V >= 4 && E % V == 0 && (reinterpret_cast<uintptr_t>(p) & 15) == 0 && (V * size) % 16 == 0) {
    if (first < E) {
      const uint4* src = reinterpret_cast<const uint4*>(static_cast<const char*>(p) + (base + first) * size);
      if (type == LOGIT_F32) {
#pragma unroll
        for (int i = 0; i < V / 4; ++i) {
          const uint4 v = src[i];
          const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
          for (int j = 0; j < 4; ++j) x[(4 * i + j) % V] = route_clean(__uint_as_float(w[j]));
        }
      } else {
#pragma unroll
        for (int i = 0; i < (V + 7) / 8; ++i) {
          const uint4 v = src[i];
          const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            float2 f;
            if (type == LOGIT_BF16) f = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&w[j]));
            else f = __half22float2(*reinterpret_cast<const __half2*>(&w[j]));
            x[(8 * i + 2 * j) % V] = route_clean(f.x);
            x[(8 * i + 2 * j + 1) % V] = route_clean(f.y);
          }
        }
      }
    } else {
#pragma unroll
      for (int j = 0; j < V; ++j) x[j] = -INFINITY;
    }
    return;
  }
#pragma unroll
  for (int j = 0; j < V; ++j) x[j] = first + j < E ? load_logit(p, type, base + first + j) : -INFINITY;
}

// Order-preserving integers; zero is below every number.  -0 counts as +0.
__device__ __forceinline__ uint32_t ordered(float v) {
  const uint32_t b = __float_as_uint(v + 0.f);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ uint64_t ordered(double v) {
  const uint64_t b = static_cast<uint64_t>(__double_as_longlong(v + 0.0));
  return b >> 63 ? ~b : b | 0x8000000000000000ull;
}
__device__ __forceinline__ float unordered(uint32_t u) {
  return __uint_as_float(u & 0x80000000u ? u & 0x7fffffffu : ~u);
}
__device__ __forceinline__ uint32_t warp_max_u(uint32_t v) { return __reduce_max_sync(ALL, v); }
__device__ __forceinline__ uint64_t warp_max_u(uint64_t v) {
  const uint32_t high = __reduce_max_sync(ALL, static_cast<uint32_t>(v >> 32));
  const uint32_t low = __reduce_max_sync(ALL, (v >> 32) == high ? static_cast<uint32_t>(v) : 0u);
  return static_cast<uint64_t>(high) << 32 | low;
}
template <typename R>
__device__ __forceinline__ R warp_add(R v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(ALL, v, o);
  return v;
}
__device__ __forceinline__ float warp_max_f(float v) { return unordered(warp_max_u(ordered(v))); }

__device__ __forceinline__ float exp_of(float v) { return expf(v); }
__device__ __forceinline__ double exp_of(double v) { return exp(v); }

template <typename R> struct Ordered { using type = uint32_t; };
template <> struct Ordered<double> { using type = uint64_t; };

// How far the fp32 form of a key s + b may be from its exact value.  expf is within 2 units in the last place (2^-23 of the value
// each); a sigmoid adds one addition and one division: 8 * 2^-24 of s covers it.  A softmax adds the rounding of x - max, which
// costs (max - x) 2^-24 of s, and s (max - x) is below 0.5; up to 32 + 5 additions of the sum, whose terms have the same errors:
// 64 * 2^-24 of s and 0.5 * 2^-24 cover it.  The addition of the bias rounds by 2^-24 of the key at most.
__device__ __forceinline__ float key_error(float s, float key, int sigmoid) {
  return 5.9604645e-8f * ((sigmoid ? 8.f : 64.f) * s + 0.5f + fabsf(key));
}

template <typename R>
struct RowStats {
  R top, total;        // softmax: the largest logit (0 where all are masked) and the sum of exp(x - top)
};

template <typename R, int V>
__device__ __forceinline__ RowStats<R> softmax_stats(const float (&x)[V]) {
  float top = -INFINITY;
#pragma unroll
  for (int j = 0; j < V; ++j) top = fmaxf(top, x[j]);
  top = warp_max_f(top);
  RowStats<R> st;
  st.top = top == -INFINITY ? R(0) : R(top);
  R sum = 0;
#pragma unroll
  for (int j = 0; j < V; ++j) sum += x[j] == -INFINITY ? R(0) : exp_of(R(x[j]) - st.top);
  sum = warp_add(sum);
  st.total = sum == R(0) ? R(1) : sum;
  return st;
}

template <typename R>
__device__ __forceinline__ R score_of(float x, const RowStats<R>& st, int sigmoid) {
  if (x == -INFINITY) return R(0);
  return sigmoid ? R(1) / (R(1) + exp_of(-R(x))) : exp_of(R(x) - st.top) / st.total;
}

// Chooses the experts of one row into ``sel`` (shared memory, k entries, one more where neighbours are checked).  ``scored``:
// scores decide (a bias, or groups by the sum of two), not the logits alone.  Returns whether a comparison that decided
// something was too close for R.
template <typename R, int V, int MODE>
__device__ __forceinline__ bool choose(const RouteParams& p, long long row, const float (&x)[V], int lane, bool scored,
                                       int* sel, R* row_keys) {
  using U = typename Ordered<R>::type;
  constexpr bool WIDE = sizeof(R) == 8;
  const int first = lane * V;
  RowStats<R> st = {R(0), R(1)};
  if (scored && !p.sigmoid) st = softmax_stats<R, V>(x);
  R key[V];
#pragma unroll
  for (int j = 0; j < V; ++j) {
    if (x[j] == -INFINITY) key[j] = -R(INFINITY);
    else if (!scored) key[j] = R(x[j]);
    else key[j] = score_of<R>(x[j], st, p.sigmoid) + (p.bias ? R(p.bias[first + j]) : R(0));
  }
  bool close = false;
  unsigned allowed = ALL;                          // one bit per group
  const int size = MODE == GROUPS_NONE ? p.E : p.E / p.groups;
  if (MODE != GROUPS_NONE) {
    R best = -R(INFINITY), second = -R(INFINITY);
    if (MODE == GROUPS_ALIGNED) {                  // a group is a run of 2^n whole lanes
#pragma unroll
      for (int j = 0; j < V; ++j) {
        second = max(second, min(best, key[j]));
        best = max(best, key[j]);
      }
      const int lanes = size / V;
      for (int o = 1; o < lanes; o <<= 1) {
        const R b = __shfl_xor_sync(ALL, best, o), s = __shfl_xor_sync(ALL, second, o);
        second = max(min(best, b), max(second, s));
        best = max(best, b);
      }
      best = __shfl_sync(ALL, best, min(lane * lanes, 31));
      second = __shfl_sync(ALL, second, min(lane * lanes, 31));
    } else {                                       // through shared memory, a lane per group
#pragma unroll
      for (int j = 0; j < V; ++j)
        if (first + j < p.E) row_keys[first + j] = key[j];
      __syncwarp();
      if (lane < p.groups) {
        for (int i = 0; i < size; ++i) {
          const R v = row_keys[lane * size + i];
          second = max(second, min(best, v));
          best = max(best, v);
        }
      }
      __syncwarp();
    }
    R value = lane < p.groups ? best : -R(INFINITY);
    if (p.two_best && value != -R(INFINITY) && second != -R(INFINITY)) value = best + second;
    int in_front = 0;
    for (int i = 0; i < p.groups; ++i) {
      const R other = __shfl_sync(ALL, value, i);
      in_front += other > value || (other == value && i < lane);
    }
    const bool group = lane < p.groups;
    allowed = __ballot_sync(ALL, group && in_front < p.top_groups);
    if (!WIDE && scored) {
      // the last group that stays against the first that goes; scores are below 1
      const unsigned last = __ballot_sync(ALL, group && in_front == p.top_groups - 1);
      const unsigned next = __ballot_sync(ALL, group && in_front == p.top_groups);
      const float a = __shfl_sync(ALL, static_cast<float>(value), __ffs(last) - 1);
      const float b = __shfl_sync(ALL, static_cast<float>(value), __ffs(next) - 1);
      const float terms = p.two_best ? 2.f : 1.f, s = p.bias ? terms : fmaxf(a, 0.f);
      // the sum of two keys rounds once more; a key is below its group's sum plus one in size, whatever the bias
      const float error = terms * (key_error(s, fabsf(a) + 1.f, p.sigmoid) + key_error(s, fabsf(b) + 1.f, p.sigmoid));
      close = b != -INFINITY && a - b <= error;
    }
  }
  // Without a bias experts are compared by their logits, whatever the groups were compared by.
  U u[V];
  const int my_group = MODE == GROUPS_ALIGNED ? min(first / size, 31) : 0;
#pragma unroll
  for (int j = 0; j < V; ++j) {
    const bool here = first + j < p.E && (MODE == GROUPS_NONE ||
                                          (allowed >> (MODE == GROUPS_ALIGNED ? my_group : (first + j) / size) & 1));
    u[j] = here ? ordered(p.bias ? key[j] : R(x[j])) : U(0);
  }
  U mine = 0;
  int at = 0;
  auto local_best = [&]() {
    mine = 0;
#pragma unroll
    for (int j = 0; j < V; ++j) {
      if (u[j] > mine) {
        mine = u[j];
        at = j;
      }
    }
  };
  local_best();
  const bool neighbours = !WIDE && p.bias;
  const int candidates = MODE == GROUPS_NONE ? p.E : size * p.top_groups;
  const int steps = min(p.k + (neighbours ? 1 : 0), candidates);
  for (int i = 0; i < steps; ++i) {
    const U top = warp_max_u(mine);
    const int winner = __ffs(__ballot_sync(ALL, mine == top)) - 1;      // the lowest lane has the lowest index
    if (lane == winner) {
      sel[i] = first + at;
#pragma unroll
      for (int j = 0; j < V; ++j)
        if (j == at) u[j] = U(0);
      local_best();
    }
  }
  __syncwarp();
  if (neighbours && lane < steps - 1) {
    // each one against the next in the order, the last against the best that was left out
    const int a = sel[lane], b = sel[lane + 1];
    const float xa = load_logit(p.logits, p.type, row * p.E + a), xb = load_logit(p.logits, p.type, row * p.E + b);
    const float ba = p.bias[a], bb = p.bias[b];
    if (xb != -INFINITY && !(xa == xb && ba == bb)) {                   // equal experts are in the order of their indices
      const RowStats<float> sf = {static_cast<float>(st.top), static_cast<float>(st.total)};
      const float sa = score_of<float>(xa, sf, p.sigmoid), sb = score_of<float>(xb, sf, p.sigmoid);
      const float ka = sa + ba, kb = sb + bb;
      close |= ka - kb <= key_error(sa, ka, p.sigmoid) + key_error(sb, kb, p.sigmoid);
    }
  }
  return __any_sync(ALL, close);
}

template <int V> constexpr int route_warps() { return V == 32 ? 4 : 8; }       // shared memory of GROUPS_ANY

template <int V, int MODE>
__global__ void __launch_bounds__(route_warps<V>() * 32) route_fwd_kernel(const RouteParams p) {
  chain_begin();
  constexpr int WARPS = route_warps<V>();
  __shared__ int sel_all[WARPS][ROUTE_MAX_K + 1];
  __shared__ double keys_all[MODE == GROUPS_ANY ? WARPS : 1][MODE == GROUPS_ANY ? 32 * V : 1];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const long long row = static_cast<long long>(blockIdx.x) * WARPS + warp;
  if (row >= p.T) return;
  int* const sel = sel_all[warp];
  double* const row_keys = keys_all[MODE == GROUPS_ANY ? warp : 0];
  float x[V];
  load_row<V>(p.logits, p.type, row, p.E, lane, x);
  const bool scored = p.bias || (MODE != GROUPS_NONE && p.two_best);
  if (choose<float, V, MODE>(p, row, x, lane, scored, sel, reinterpret_cast<float*>(row_keys))) {
    __syncwarp();
    choose<double, V, MODE>(p, row, x, lane, scored, sel, row_keys);
  }
  // Weights, a lane per chosen expert.
  const bool on = lane < p.k;
  const int e = on ? sel[lane] : 0;
  const float xe = on ? load_logit(p.logits, p.type, row * p.E + e) : -INFINITY;
  float w;
  if (p.renormalize) {
    // softmax: the other experts cancel.  Sigmoids below -60 are exp(x) to the last bit, and their sum could vanish.
    const float top = warp_max_f(xe);
    if (!p.sigmoid || top < -60.f) w = xe == -INFINITY ? 0.f : expf(xe - top);
    else w = xe == -INFINITY ? 0.f : 1.f / (1.f + expf(-xe));
    const float total = warp_add(w);
    w = total == 0.f ? 0.f : w / total;
  } else {
    RowStats<float> st = {0.f, 1.f};
    if (!p.sigmoid) st = softmax_stats<float, V>(x);
    w = score_of<float>(xe, st, p.sigmoid);
  }
  if (on) {
    p.weights[row * p.k + lane] = w * p.scale;
    p.idx[row * p.k + lane] = e;
  }
}

// Gradient of the logits.  With the weights w = scale * v and their gradient g:
//   sigmoid, renormalised   v_i (1 - s_i) (scale g_i - sum_j scale g_j v_j)          sigmoid      scale g_i v_i (1 - s_i)
//   softmax, renormalised   v_i (scale g_i - sum_j scale g_j v_j)                    softmax      the same over all experts
// for the chosen experts i; the others have none, but for a softmax over all experts: -p_e sum_j scale g_j v_j.
template <int V>
__global__ void __launch_bounds__(route_warps<V>() * 32) route_bwd_kernel(const RouteParams p, const float* __restrict__ dweights,
                                                                       void* __restrict__ dlogits) {
  chain_begin();
  constexpr int WARPS = route_warps<V>();
  __shared__ float rows[WARPS][32 * V];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const long long row = static_cast<long long>(blockIdx.x) * WARPS + warp;
  if (row >= p.T) return;
  float* const out = rows[warp];
  const bool on = lane < p.k;
  const long long at = row * p.k + lane;
  const int e = on ? min(max(static_cast<int>(p.idx[at]), 0), p.E - 1) : 0;
  const float v = on ? p.weights[at] / p.scale : 0.f;
  float g = on ? dweights[at] * p.scale : 0.f;
  const bool all = !p.sigmoid && !p.renormalize;
  const float inner = warp_add(g * v);
  if (p.renormalize) g -= inner;
  g *= v;
  if (p.sigmoid && on) g *= 1.f / (1.f + expf(load_logit(p.logits, p.type, row * p.E + e)));
  float prob[V];
#pragma unroll
  for (int j = 0; j < V; ++j) prob[j] = 0.f;
  if (all) {
    float x[V];
    load_row<V>(p.logits, p.type, row, p.E, lane, x);
    const RowStats<float> st = softmax_stats<float, V>(x);
#pragma unroll
    for (int j = 0; j < V; ++j) prob[j] = -inner * score_of<float>(x[j], st, 0);
  }
#pragma unroll
  for (int j = 0; j < V; ++j) out[j * 32 + lane] = 0.f;
  __syncwarp();
  if (on && v != 0.f) out[e % V * 32 + e / V] = g;          // the place of expert e: its lane is e / V
  __syncwarp();
  const int first = lane * V;
  const int size = p.type == LOGIT_F32 ? 4 : 2;
  float y[V];
#pragma unroll
  for (int j = 0; j < V; ++j) y[j] = out[j * 32 + lane] + prob[j];
  char* const dst = static_cast<char*>(dlogits) + (row * p.E + first) * size;
  if (V >= 4 && p.E % V == 0 && (V * size) % 16 == 0) {     // a buffer of this call's own: aligned
    if (first >= p.E) return;
    if (p.type == LOGIT_F32) {
#pragma unroll
      for (int i = 0; i < V / 4; ++i)
        reinterpret_cast<float4*>(dst)[i] = make_float4(y[4 * i], y[(4 * i + 1) % V], y[(4 * i + 2) % V], y[(4 * i + 3) % V]);
    } else {
#pragma unroll
      for (int i = 0; i < (V + 7) / 8; ++i) {
        uint32_t w[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float a = y[(8 * i + 2 * j) % V], b = y[(8 * i + 2 * j + 1) % V];
          if (p.type == LOGIT_BF16) {
            const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
            w[j] = *reinterpret_cast<const uint32_t*>(&h);
          } else {
            const __half2 h = __floats2half2_rn(a, b);
            w[j] = *reinterpret_cast<const uint32_t*>(&h);
          }
        }
        reinterpret_cast<uint4*>(dst)[i] = make_uint4(w[0], w[1], w[2], w[3]);
      }
    }
    return;
  }
#pragma unroll
  for (int j = 0; j < V; ++j) {
    if (first + j >= p.E) continue;
    if (p.type == LOGIT_F32) reinterpret_cast<float*>(dst)[j] = y[j];
    else if (p.type == LOGIT_BF16) reinterpret_cast<__nv_bfloat16*>(dst)[j] = __float2bfloat16(y[j]);
    else reinterpret_cast<__half*>(dst)[j] = __float2half(y[j]);
  }
}

template <int V>
static int launch_route(const RouteParams& p, const float* dweights, void* dlogits, cudaStream_t s) {
  constexpr int WARPS = route_warps<V>();
  const long long grid = (p.T + WARPS - 1) / WARPS;
  if (grid > 0x7fffffffLL) return -12;
  cudaError_t r;
  if (dweights) {
    r = launch_next(route_bwd_kernel<V>, static_cast<unsigned>(grid), WARPS * 32, 0, s, p, dweights, dlogits);
  } else {
    const int size = p.E / p.groups;
    const bool aligned = size % V == 0 && ((size / V) & (size / V - 1)) == 0;
    if (p.top_groups == p.groups) r = launch_next(route_fwd_kernel<V, GROUPS_NONE>, static_cast<unsigned>(grid), WARPS * 32, 0, s, p);
    else if (aligned) r = launch_next(route_fwd_kernel<V, GROUPS_ALIGNED>, static_cast<unsigned>(grid), WARPS * 32, 0, s, p);
    else r = launch_next(route_fwd_kernel<V, GROUPS_ANY>, static_cast<unsigned>(grid), WARPS * 32, 0, s, p);
  }
  if (r != cudaSuccess) cudaGetLastError();
  return r == cudaSuccess ? 0 : -1;
}

static int route(const RouteParams& p, const float* dweights, void* dlogits, cudaStream_t s) {
  if (p.E < 1 || p.E > 1024 || p.k < 1 || p.k > ROUTE_MAX_K || p.groups < 1 || p.groups > 32 || p.E % p.groups ||
      p.top_groups < 1 || p.top_groups > p.groups || p.k > p.E / p.groups * p.top_groups ||
      (p.two_best && p.top_groups < p.groups && p.E / p.groups < 2) || p.type < 0 || p.type > 2 || p.scale == 0.f)
    return -10;
  if (p.T == 0) return 0;
  if (p.E <= 32) return launch_route<1>(p, dweights, dlogits, s);
  if (p.E <= 64) return launch_route<2>(p, dweights, dlogits, s);
  if (p.E <= 128) return launch_route<4>(p, dweights, dlogits, s);
  if (p.E <= 256) return launch_route<8>(p, dweights, dlogits, s);
  if (p.E <= 512) return launch_route<16>(p, dweights, dlogits, s);
  return launch_route<32>(p, dweights, dlogits, s);
}

}  // namespace b2

using namespace b2;

extern "C" {

// logits [T, E] contiguous (type 0 fp32, 1 bf16, 2 fp16), bias fp32 [E] or null -> weights fp32 [T, k], idx int64 [T, k].
int b2_route_topk(const void* logits, const float* bias, float* weights, long long* idx, long long T, int E, int k, int type,
                  int sigmoid, int groups, int top_groups, int two_best, int renormalize, float scale, cudaStream_t s) {
  const RouteParams p = {logits, bias, weights, idx, T, E, k, type, sigmoid, groups, top_groups, two_best, renormalize, scale};
  return route(p, nullptr, nullptr, s);
}

// The gradient of the logits, in their type, from that of the weights.
int b2_route_topk_bwd(const void* logits, const float* weights, const long long* idx, const float* dweights, void* dlogits,
                      long long T, int E, int k, int type, int sigmoid, int renormalize, float scale, cudaStream_t s) {
  const RouteParams p = {logits, nullptr, const_cast<float*>(weights), const_cast<long long*>(idx), T, E, k, type, sigmoid,
                         1, 1, 0, renormalize, scale};
  return route(p, dweights, dlogits, s);
}

}  // extern "C"
