// Routing to experts with a choice of scores, a balance bias, groups and any number of experts per token (``moe.cu`` and
// ``elementwise.cu`` hold the top-2 softmax router of the standard block).
//
//   s_e = sigmoid(x_e) or softmax(x)_e,   key_e = s_e + bias_e   (without a bias: x_e, whose order is that of s_e)
//   value of a group = its best key, or the sum of its two best;  the best groups stay, then the k best experts in them
//   w_i = scale * s_i / sum of the chosen s, or scale * s_i
//
// A warp, or eight lanes of one, works on a token and holds its logits in registers, so a row is read once.  Each lane sorts its
// own keys (a network of minima and maxima, no indices), then k steps take the best of the lanes' first keys and remove it; the
// index of a chosen key is looked up afterwards among the lane's keys, for all chosen ones at once.
//
// Bound by integer minima, comparisons and selections, which the ALU issues every other cycle, beyond 100 experts.
//
// The choice is that of 64-bit arithmetic.  Comparisons of logits are exact as they are.  Comparisons of scores (a bias, a
// sum of two) are made in fp32 with the fast exponential and division first, and those that decided something are checked
// against a bound on the error of both sides; a row in which one is closer than that is worked out again in 64 bits, by a whole
// warp, plainly.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <float.h>
#include <stdint.h>

#include "chain.cuh"
#include "entries.h"

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
  int size;                  // experts of a group
  int lane_shift;            // GROUPS_ALIGNED: a group is 2^lane_shift lanes
};

// NaN counts as masked (a maximum leaves it out), infinity as the largest number.
__device__ __forceinline__ float route_clean(float x) { return fminf(fmaxf(x, -INFINITY), FLT_MAX); }

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
  if constexpr (V >= 4) {
    if (E % V == 0 && (reinterpret_cast<uintptr_t>(p) & 15) == 0 && (V * size) % 16 == 0) {
      if (first >= E) {
#pragma unroll
        for (int j = 0; j < V; ++j) x[j] = -INFINITY;
        return;
      }
      const uint4* src = reinterpret_cast<const uint4*>(static_cast<const char*>(p) + (base + first) * size);
      if (type == LOGIT_F32) {
#pragma unroll
        for (int i = 0; i < V / 4; ++i) {
          const uint4 v = src[i];
          const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
          for (int j = 0; j < 4; ++j) x[4 * i + j] = route_clean(__uint_as_float(w[j]));
        }
        return;
      }
      if constexpr (V >= 8) {
#pragma unroll
        for (int i = 0; i < V / 8; ++i) {
          const uint4 v = src[i];
          const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const float2 f = type == LOGIT_BF16 ? __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&w[j]))
                                                : __half22float2(*reinterpret_cast<const __half2*>(&w[j]));
            x[8 * i + 2 * j] = route_clean(f.x);
            x[8 * i + 2 * j + 1] = route_clean(f.y);
          }
        }
        return;
      }
    }
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
// Over the LANES lanes of a row.
template <int LANES, typename R>
__device__ __forceinline__ R row_add(R v) {
#pragma unroll
  for (int o = LANES / 2; o > 0; o >>= 1) v += __shfl_xor_sync(ALL, v, o);
  return v;
}
template <int LANES, typename U>
__device__ __forceinline__ U row_max(U v) {
  if constexpr (LANES == 32) {
    return warp_max_u(v);
  } else {
#pragma unroll
    for (int o = LANES / 2; o > 0; o >>= 1) v = max(v, __shfl_xor_sync(ALL, v, o));
    return v;
  }
}
template <int LANES>
__device__ __forceinline__ float row_max_f(float v) {
  if constexpr (LANES == 32) {
    return unordered(warp_max_u(ordered(v)));
  } else {
#pragma unroll
    for (int o = LANES / 2; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(ALL, v, o));
    return v;
  }
}
// The bits of a ballot that are this row's.
template <int LANES>
__device__ __forceinline__ unsigned row_ballot(bool b) {
  const unsigned all = __ballot_sync(ALL, b);
  return LANES == 32 ? all : (all >> (threadIdx.x & 31 & ~(LANES - 1))) & ((1u << (LANES & 31)) - 1);
}

// exp and 1 / x for comparisons that are checked: two steps of the multi-function unit each way, results below 2^-126 are zero.
__device__ __forceinline__ float fast_exp(float v) {
  float e;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(v * 1.44269504f));
  return e;
}
__device__ __forceinline__ float fast_inverse(float v) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
  return r;
}

struct RowStats {
  float top, total;        // softmax: the largest logit (0 where all are masked) and the sum of exp(x - top)
};

template <int LANES, bool FAST, int V>
__device__ __forceinline__ RowStats softmax_stats(const float (&x)[V]) {
  float top = -INFINITY;
#pragma unroll
  for (int j = 0; j < V; ++j) top = fmaxf(top, x[j]);
  top = row_max_f<LANES>(top);
  RowStats st;
  st.top = top == -INFINITY ? 0.f : top;
  float sum = 0.f;
#pragma unroll
  for (int j = 0; j < V; ++j) sum += FAST ? fast_exp(x[j] - st.top) : expf(x[j] - st.top);        // of -inf: 0
  sum = row_add<LANES>(sum);
  st.total = sum == 0.f ? 1.f : sum;
  return st;
}

__device__ __forceinline__ float score_of(float x, const RowStats& st, int sigmoid) {
  if (x == -INFINITY) return 0.f;
  return sigmoid ? 1.f / (1.f + expf(-x)) : expf(x - st.top) / st.total;
}

// How far the fast fp32 form of a key s + b may be from its exact value, in steps of 2^-24, with ``most`` a bound on s.  The base-2
// exponential is within 2^-22 of its value (4 steps), its argument v log2(e) is rounded twice (2 |v| steps of the result), the
// reciprocal within one unit in the last place (2 steps).
//   sigmoid: s (1 - s) (4 + 2 |x|) of the exponential, where s (1 - s) |x| < 0.23, the addition's s and the reciprocal's 2 s:
//            below 7 s + 0.5
//   softmax: s (4 + 3 d) of the exponential with d = max - x, where s d < 0.37; the same of the sum's terms, where the mean of d over
//            the scores is below ln E < 7, and its 32 + 5 additions; the reciprocal and the product: below 69 s + 1.2
// The addition of the bias rounds by one step of the key at most.
__device__ __forceinline__ float key_error(float most, float key, int sigmoid) {
  return 5.9604645e-8f * ((sigmoid ? 10.f : 75.f) * most + 2.f + fabsf(key));
}

template <typename U>
__device__ __forceinline__ void order_down(U& a, U& b) {
  const U high = max(a, b), low = min(a, b);
  a = high;
  b = low;
}
// Descending, by a network of minima and maxima: runs of eight by 19 exchanges, which are then merged (V is a power of two).
template <typename U, int V>
__device__ __forceinline__ void sort_down(U (&h)[V]) {
  if constexpr (V < 8) {
#pragma unroll
    for (int n = V - 1; n > 0; --n) {
#pragma unroll
      for (int i = 0; i < n; ++i) order_down(h[i], h[i + 1]);
    }
  } else {
    constexpr int pairs[19][2] = {{0, 2}, {1, 3}, {4, 6}, {5, 7}, {0, 4}, {1, 5}, {2, 6}, {3, 7}, {0, 1}, {2, 3},
                                  {4, 5}, {6, 7}, {2, 4}, {3, 5}, {1, 4}, {3, 6}, {1, 2}, {3, 4}, {5, 6}};
#pragma unroll
    for (int run = 0; run < V; run += 8) {
#pragma unroll
      for (int i = 0; i < 19; ++i) order_down(h[run + pairs[i][0]], h[run + pairs[i][1]]);
    }
#pragma unroll
    for (int size = 16; size <= V; size <<= 1) {
#pragma unroll
      for (int i = 0; i < V; ++i)                         // against the mirror image, then in halves
        if ((i ^ (size - 1)) > i) order_down(h[i], h[i ^ (size - 1)]);
#pragma unroll
      for (int step = size / 4; step > 0; step >>= 1) {
#pragma unroll
        for (int i = 0; i < V; ++i)
          if ((i ^ step) > i) order_down(h[i], h[i ^ step]);
      }
    }
  }
}

// Chooses the experts of one row: lane i of the row's returns the i-th.  ``scored``: scores decide (a bias, or groups by the sum of
// two), not the logits alone.  ``close`` tells whether a comparison that decided something was too close.
template <int LANES, int V, int MODE>
__device__ __forceinline__ int choose(const RouteParams& p, long long row, const float (&x)[V], int lane, bool scored,
                                      float* row_keys, bool& close) {
  static_assert(MODE == GROUPS_NONE || LANES == 32, "groups are chosen by a whole warp");
  const int first = lane * V;
  float key[V];
  float most = 1.f;                                // no score is above
  if (scored) {
    RowStats st = {0.f, 1.f};
    if (!p.sigmoid) {
      st = softmax_stats<LANES, true, V>(x);
      most = fast_inverse(st.total);
    }
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const float s = p.sigmoid ? fast_inverse(1.f + fast_exp(-x[j])) : fast_exp(x[j] - st.top) * most;
      key[j] = x[j] == -INFINITY ? -INFINITY : p.bias ? s + p.bias[first + j] : s;
    }
  } else {
#pragma unroll
    for (int j = 0; j < V; ++j) key[j] = x[j];
  }
  close = false;
  unsigned allowed = ALL;                          // one bit per group
  const int size = p.size;
  if (MODE != GROUPS_NONE) {
    float best = -INFINITY, second = -INFINITY;
    if (MODE == GROUPS_ALIGNED) {                  // a group is a run of 2^n whole lanes
#pragma unroll
      for (int j = 0; j < V; ++j) {
        second = fmaxf(second, fminf(best, key[j]));
        best = fmaxf(best, key[j]);
      }
      for (int o = 1; o < 1 << p.lane_shift; o <<= 1) {
        const float b = __shfl_xor_sync(ALL, best, o), s = __shfl_xor_sync(ALL, second, o);
        second = fmaxf(fminf(best, b), fmaxf(second, s));
        best = fmaxf(best, b);
      }
      best = __shfl_sync(ALL, best, min(lane << p.lane_shift, LANES - 1), LANES);
      second = __shfl_sync(ALL, second, min(lane << p.lane_shift, LANES - 1), LANES);
    } else {                                       // through shared memory, a lane per group
#pragma unroll
      for (int j = 0; j < V; ++j)
        if (first + j < p.E) row_keys[first + j] = key[j];
      __syncwarp();
      if (lane < p.groups) {
        for (int i = 0; i < size; ++i) {
          const float v = row_keys[lane * size + i];
          second = fmaxf(second, fminf(best, v));
          best = fmaxf(best, v);
        }
      }
      __syncwarp();
    }
    const bool group = lane < p.groups;
    float value = group ? best : -INFINITY;
    if (p.two_best && value != -INFINITY && second != -INFINITY) value = best + second;
    int in_front = 0;
#pragma unroll 4
    for (int i = 0; i < p.groups; ++i) {
      const float other = __shfl_sync(ALL, value, i, LANES);
      in_front += other > value || (other == value && i < lane);
    }
    allowed = row_ballot<LANES>(group && in_front < p.top_groups);
    if (scored) {
      // Each group that stays against each that goes.  A key is off by what its own size says, which the sum of two of opposite signs
      // hides.  The sum rounds once more, and so do its bounds: by a step of the sum each, at most two of the larger key.
      const float reach = value == -INFINITY ? 0.f : fmaxf(fabsf(best), p.two_best && second != -INFINITY ? fabsf(second) : 0.f);
      const float error = (p.two_best ? 2.f : 1.f) * key_error(most, 3.f * reach, p.sigmoid);
      const bool stays = group && in_front < p.top_groups, goes = group && !stays && value != -INFINITY;
      // (a value that overflowed has no lower bound)
      const uint32_t low = __reduce_min_sync(ALL, stays ? ordered(fmaxf(value - error, -INFINITY)) : ALL);
      const uint32_t high = __reduce_max_sync(ALL, goes ? ordered(value + error) : 0u);
      close = low <= high;
    }
  }
  // Without a bias experts are compared by their logits, whatever the groups were compared by.
  uint32_t h[V];
  const bool lane_here = MODE != GROUPS_ALIGNED || (first < p.E && (allowed >> (lane >> p.lane_shift) & 1));
#pragma unroll
  for (int j = 0; j < V; ++j) {
    const bool here = MODE == GROUPS_ALIGNED ? lane_here
                                             : first + j < p.E && (MODE == GROUPS_NONE || (allowed >> ((first + j) / size) & 1));
    h[j] = here ? ordered(p.bias ? key[j] : x[j]) : 0u;
  }
  // the keys in the order of the experts wait in shared memory for the look-up
  uint32_t* const unsorted = reinterpret_cast<uint32_t*>(row_keys);
  if constexpr (V >= 4) {
#pragma unroll
    for (int j = 0; j < V / 4; ++j)
      reinterpret_cast<uint4*>(unsorted + first)[j] = make_uint4(h[4 * j], h[4 * j + 1], h[4 * j + 2], h[4 * j + 3]);
  } else {
#pragma unroll
    for (int j = 0; j < V; ++j) unsorted[first + j] = h[j];
  }
  sort_down(h);
  const int candidates = MODE == GROUPS_NONE ? p.E : size * p.top_groups;
  const int steps = min(p.k + (p.bias ? 2 : 0), candidates);       // two more, for the comparison with what is left out
  uint32_t my_key = 0, extra = 0;
  int my_winner = 0;
  for (int i = 0; i < steps; ++i) {
    const uint32_t top = row_max<LANES>(h[0]);
    const int winner = __ffs(row_ballot<LANES>(h[0] == top)) - 1;      // the lowest lane has the lowest index
    if (lane == i) {
      my_key = top;
      my_winner = winner;
    }
    if (i == LANES) extra = top;                   // no lane is left for it
    if (lane == winner) {
#pragma unroll
      for (int j = 0; j + 1 < V; ++j) h[j] = h[j + 1];
      h[V - 1] = 0;
    }
  }
  // Which of the winner's keys it was: of equal ones the first, then the second, ...; a lane gives them one after the other.
  const uint32_t key_before = __shfl_up_sync(ALL, my_key, 1);
  const int winner_before = __shfl_up_sync(ALL, my_winner, 1);
  const unsigned again = row_ballot<LANES>(lane > 0 && lane < steps && my_key == key_before && my_winner == winner_before);
  int skip = lane - (31 - __clz(~again & ((2u << lane) - 1)));
  int index = my_winner * V;
  const uint32_t* const theirs = unsorted + index;
  __syncwarp();
  auto look = [&](uint32_t key, int j) {
    const bool same = key == my_key;
    if (same && skip == 0) index += j;
    skip -= same;
  };
  if constexpr (V >= 4) {
#pragma unroll
    for (int j = 0; j < V / 4; ++j) {
      const uint4 v = reinterpret_cast<const uint4*>(theirs)[j];
      look(v.x, 4 * j);
      look(v.y, 4 * j + 1);
      look(v.z, 4 * j + 2);
      look(v.w, 4 * j + 3);
    }
  } else {
#pragma unroll
    for (int j = 0; j < V; ++j) look(theirs[j], j);
  }
  __syncwarp();
  if (p.bias && steps > 1) {
    // Each one against the next in the order, the last against the best that was left out.
    const uint32_t key_after = __shfl_down_sync(ALL, my_key, 1);
    const int index_after = __shfl_down_sync(ALL, index, 1);
    const float ka = unordered(my_key), kb = unordered(lane == LANES - 1 ? extra : key_after);
    const bool near = lane < steps - 1 && kb != -INFINITY && ka - kb <= key_error(most, ka, p.sigmoid) + key_error(most, kb, p.sigmoid);
    bool doubtful = near;
    float xa = 0.f, xb = 0.f, ba = 0.f, bb = 0.f;
    if (near && lane != LANES - 1) {                // equal experts are in the order of their indices
      xa = load_logit(p.logits, p.type, row * p.E + index);
      xb = load_logit(p.logits, p.type, row * p.E + index_after);
      ba = p.bias[index];
      bb = p.bias[index_after];
      doubtful = !(xa == xb && ba == bb);
    }
    // Near pairs that follow one another are a run, equal ones among them: what belongs in front of one of two equal experts belongs
    // in front of both.  Sigmoids of a pair that is a run by itself are put in order in 64 bits on the spot.  Softmaxes, which need
    // all logits again, and longer runs are left to the row's second pass where they reach the first k.
    const unsigned nears = row_ballot<LANES>(near);
    const bool alone = doubtful && p.sigmoid && lane != LANES - 1 && !((nears << 1 | nears >> 1) >> lane & 1);
    bool swap = false;
    if (alone) {
      const double a = 1.0 / (1.0 + exp(-static_cast<double>(xa))) + ba, b = 1.0 / (1.0 + exp(-static_cast<double>(xb))) + bb;
      swap = b > a || (a == b && index_after < index);
    }
    // the run that leaves the first k between their last pair and the one behind it
    const bool leaves = p.k < LANES && (nears >> (p.k - 1) & nears >> p.k & 1);
    close |= doubtful && !alone && (lane < p.k || (lane == p.k && leaves));
    const bool beyond = leaves && steps < candidates;
    if (LANES == 32 ? beyond : __any_sync(ALL, beyond)) {      // it may go on behind the last key that was looked at
      const float next = unordered(row_max<LANES>(h[0]));
      const float last = unordered(__shfl_sync(ALL, my_key, min(steps - 1, LANES - 1), LANES));
      close |= beyond && next != -INFINITY &&
               last - next <= key_error(most, last, p.sigmoid) + key_error(most, next, p.sigmoid);
    }
    const unsigned swaps = row_ballot<LANES>(swap);
    const int index_before = __shfl_up_sync(ALL, index, 1);
    if (swaps >> lane & 1) index = index_after;
    else if (lane > 0 && (swaps >> (lane - 1) & 1)) index = index_before;
  }
  return index;
}

// The same in 64 bits, for rows in which fp32 cannot decide: lane i of the warp returns the i-th expert.  ``keys``: one per expert.
// One such row among the last ones holds up the launch, so its latency counts: four experts of a lane are on their way at a time (more take
// registers from the kernel around it).
__device__ __noinline__ int choose_in_64_bits(const RouteParams& p, long long row, int lane, double* keys) {
  constexpr int N = 4;
  const bool two = p.two_best && p.top_groups < p.groups;
  const long long base = row * p.E;
  auto load = [&](int e0, float (&x)[N]) {
#pragma unroll
    for (int i = 0; i < N; ++i) x[i] = e0 + 32 * i < p.E ? load_logit(p.logits, p.type, base + e0 + 32 * i) : -INFINITY;
  };
  double top = 0, total = 1;
  if (!p.sigmoid) {
    float most = -INFINITY;
    for (int e0 = lane; e0 < p.E; e0 += 32 * N) {
      float x[N];
      load(e0, x);
#pragma unroll
      for (int i = 0; i < N; ++i) most = fmaxf(most, x[i]);
    }
    most = unordered(warp_max_u(ordered(most)));
    top = most == -INFINITY ? 0.0 : most;
    total = 0;
    for (int e0 = lane; e0 < p.E; e0 += 32 * N) {
      float x[N];
      load(e0, x);
#pragma unroll
      for (int i = 0; i < N; ++i) total += exp(x[i] - top);
    }
    total = row_add<32>(total);
    if (total == 0) total = 1;
  }
  for (int e0 = lane; e0 < p.E; e0 += 32 * N) {
    float x[N];
    load(e0, x);
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int e = e0 + 32 * i;
      if (e >= p.E) continue;
      double key = x[i];
      if (x[i] != -INFINITY && (p.bias || two)) {
        const double power = exp(p.sigmoid ? -static_cast<double>(x[i]) : x[i] - top);
        key = (p.sigmoid ? 1.0 : power) / (p.sigmoid ? 1.0 + power : total);
        if (p.bias) key += p.bias[e];
      }
      keys[e] = key;
    }
  }
  __syncwarp();
  const int size = p.E / p.groups;
  unsigned allowed = ALL;
  if (p.top_groups < p.groups) {
    double best = -INFINITY, second = -INFINITY;
    if (lane < p.groups) {
#pragma unroll 8
      for (int i = 0; i < size; ++i) {
        const double v = keys[lane * size + i];
        second = fmax(second, fmin(best, v));
        best = fmax(best, v);
      }
    }
    if (two && second != -INFINITY) best += second;
    int in_front = 0;
    for (int i = 0; i < p.groups; ++i) {
      const double other = __shfl_sync(ALL, best, i);
      in_front += other > best || (other == best && i < lane);
    }
    allowed = __ballot_sync(ALL, lane < p.groups && in_front < p.top_groups);
    __syncwarp();
  }
  // what is compared, as integers in the place of the keys: zero for experts of other groups and for those that are gone
  uint64_t* const left = reinterpret_cast<uint64_t*>(keys);
#pragma unroll 4
  for (int e = lane; e < p.E; e += 32) {
    const double key = p.bias ? keys[e] : static_cast<double>(load_logit(p.logits, p.type, base + e));
    left[e] = allowed >> (e / size) & 1 ? ordered(key) : 0;
  }
  int mine = 0;
  for (int i = 0; i < p.k; ++i) {
    uint64_t best = 0;
    int at = lane;
    for (int e0 = lane; e0 < p.E; e0 += 32 * N) {
      uint64_t key[N];
#pragma unroll
      for (int j = 0; j < N; ++j) key[j] = e0 + 32 * j < p.E ? left[e0 + 32 * j] : 0;
#pragma unroll
      for (int j = 0; j < N; ++j) {
        if (key[j] > best) {
          best = key[j];
          at = e0 + 32 * j;
        }
      }
    }
    const uint64_t most = warp_max_u(best);
    const int chosen = __reduce_min_sync(ALL, best == most ? at : 0x7fffffff);
    if (at == chosen) left[at] = 0;                // a lane's own expert: nobody else reads it
    if (lane == i) mine = chosen;
  }
  __syncwarp();
  return mine;
}

constexpr int route_warps(int V) { return V == 32 ? 4 : 8; }       // shared memory of GROUPS_ANY

template <int LANES, int V, int MODE>
__global__ void __launch_bounds__(route_warps(V) * 32, 4) route_fwd_kernel(const RouteParams p) {
  chain_begin();
  constexpr int WARPS = route_warps(V), ROWS = 32 / LANES;
  __shared__ alignas(16) double keys_all[WARPS][ROWS == 1 ? 32 * V : 16 * V];      // fp32 keys of the warp's rows, or those of one row in 64 bits
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & (LANES - 1);
  const long long first_row = (static_cast<long long>(blockIdx.x) * WARPS + warp) * ROWS;
  if (first_row >= p.T) return;
  // rows behind the last are worked out like it and not stored
  const long long mine = first_row + (threadIdx.x & 31) / LANES, row = mine < p.T ? mine : p.T - 1;
  float x[V];
  load_row<V>(p.logits, p.type, row, p.E, lane, x);
  const bool scored = p.bias || (MODE != GROUPS_NONE && p.two_best);
  bool close;
  int e = choose<LANES, V, MODE>(p, row, x, lane, scored,
                                  reinterpret_cast<float*>(keys_all[warp]) + (threadIdx.x & 31 & ~(LANES - 1)) * V, close);
  unsigned again = __ballot_sync(ALL, close);
  while (again) {                                  // row by row
    const int r = (__ffs(again) - 1) / LANES;
    again &= LANES == 32 ? 0u : ~(((1u << (LANES & 31)) - 1) << r * LANES);
    const int chosen = choose_in_64_bits(p, min(first_row + r, p.T - 1), threadIdx.x & 31, keys_all[warp]);
    const int passed = __shfl_sync(ALL, chosen, lane);
    if ((threadIdx.x & 31) / LANES == r) e = passed;
  }
  // Weights, a lane per chosen expert.
  const bool on = lane < p.k;
  const float xe = on ? load_logit(p.logits, p.type, row * p.E + e) : -INFINITY;
  float w;
  if (p.renormalize) {
    // Softmax: the other experts cancel.  Sigmoids of negative logits are exp(x) / (1 + exp(x)), all over exp(top) where none is positive: a
    // score that fp32 does not hold may have a weight that it does.
    const float top = row_max_f<LANES>(xe);
    if (p.sigmoid) {
      const float small = expf(-fabsf(xe));
      w = xe > 0.f ? 1.f : top < 0.f ? expf(xe - top) : small;
      w = xe == -INFINITY ? 0.f : w / (1.f + small);
    } else {
      w = xe == -INFINITY ? 0.f : expf(xe - top);
    }
    const float total = row_add<LANES>(w);
    w = total == 0.f ? 0.f : w / total;
  } else {
    RowStats st = {0.f, 1.f};
    if (!p.sigmoid) st = softmax_stats<LANES, false, V>(x);
    w = score_of(xe, st, p.sigmoid);
  }
  if (on && mine < p.T) {
    p.weights[row * p.k + lane] = w * p.scale;
    p.idx[row * p.k + lane] = e;
  }
}

// Gradient of the logits.  With the weights w, which hold the scale, and their gradient g:
//   sigmoid, renormalised   w_i (1 - s_i) (g_i - sum_j g_j w_j / scale)              sigmoid      w_i (1 - s_i) g_i
//   softmax, renormalised   w_i (g_i - sum_j g_j w_j / scale)                        softmax      w_i g_i - p_i sum_j g_j w_j
// for the chosen experts i; the others have none, but for a softmax over all experts: -p_e sum_j g_j w_j.
template <int LANES, int V>
__global__ void __launch_bounds__(route_warps(V) * 32) route_bwd_kernel(const RouteParams p, const float* __restrict__ dweights,
                                                                       void* __restrict__ dlogits) {
  chain_begin();
  constexpr int WARPS = route_warps(V), ROWS = 32 / LANES;
  __shared__ float rows[WARPS][32 * V];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & (LANES - 1);
  const long long first_row = (static_cast<long long>(blockIdx.x) * WARPS + warp) * ROWS;
  if (first_row >= p.T) return;
  // rows behind the last are worked out like it and not stored
  const long long mine = first_row + (threadIdx.x & 31) / LANES, row = mine < p.T ? mine : p.T - 1;
  float* const out = rows[warp] + (threadIdx.x & 31 & ~(LANES - 1)) * V;
  const bool on = lane < p.k;
  const long long at = row * p.k + lane;
  const int e = on ? min(max(static_cast<int>(p.idx[at]), 0), p.E - 1) : 0;
  const float w = on ? p.weights[at] : 0.f;
  float g = on ? dweights[at] : 0.f;
  const bool all = !p.sigmoid && !p.renormalize;
  const float inner = row_add<LANES>(g * w);
  if (p.renormalize) g -= inner / p.scale;
  g *= w;
  if (p.sigmoid && on) g *= 1.f / (1.f + expf(load_logit(p.logits, p.type, row * p.E + e)));
  float prob[V];
#pragma unroll
  for (int j = 0; j < V; ++j) prob[j] = 0.f;
  if (all) {
    float x[V];
    load_row<V>(p.logits, p.type, row, p.E, lane, x);
    const RowStats st = softmax_stats<LANES, false, V>(x);
#pragma unroll
    for (int j = 0; j < V; ++j) prob[j] = -inner * score_of(x[j], st, 0);
  }
#pragma unroll
  for (int j = 0; j < V; ++j) out[j * LANES + lane] = 0.f;
  __syncwarp();
  if (on && w != 0.f) out[e % V * LANES + e / V] = g;          // the place of expert e: its lane is e / V
  __syncwarp();
  if (mine >= p.T) return;
  const int first = lane * V;
  const int size = p.type == LOGIT_F32 ? 4 : 2;
  float y[V];
#pragma unroll
  for (int j = 0; j < V; ++j) y[j] = out[j * LANES + lane] + prob[j];
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

// Whether a group is a run of 2^n lanes of V logits.
static bool whole_lanes(const RouteParams& p, int V) {
  return p.size % V == 0 && ((p.size / V) & (p.size / V - 1)) == 0;
}

template <int LANES, int V>
static int launch_route(RouteParams p, cudaStream_t s) {
  constexpr int WARPS = route_warps(V);
  const long long grid = (p.T + WARPS * (32 / LANES) - 1) / (WARPS * (32 / LANES));
  if (grid > 0x7fffffffLL) return -12;
  const unsigned ctas = static_cast<unsigned>(grid);
  cudaError_t r = cudaErrorInvalidValue;
  if (p.top_groups == p.groups) {
    r = launch_next(route_fwd_kernel<LANES, V, GROUPS_NONE>, ctas, WARPS * 32, 0, s, p);
  } else if constexpr (LANES == 32) {
    for (int lanes = p.size / V; lanes > 1; lanes >>= 1) ++p.lane_shift;
    if (whole_lanes(p, V)) r = launch_next(route_fwd_kernel<32, V, GROUPS_ALIGNED>, ctas, WARPS * 32, 0, s, p);
    else r = launch_next(route_fwd_kernel<32, V, GROUPS_ANY>, ctas, WARPS * 32, 0, s, p);
  }
  if (r != cudaSuccess) cudaGetLastError();
  return r == cudaSuccess ? 0 : -1;
}

template <int LANES, int V>
static int launch_route_bwd(const RouteParams& p, const float* dweights, void* dlogits, cudaStream_t s) {
  constexpr int WARPS = route_warps(V);
  const long long grid = (p.T + WARPS * (32 / LANES) - 1) / (WARPS * (32 / LANES));
  if (grid > 0x7fffffffLL) return -12;
  const cudaError_t r = launch_next(route_bwd_kernel<LANES, V>, static_cast<unsigned>(grid), WARPS * 32, 0, s, p, dweights, dlogits);
  if (r != cudaSuccess) cudaGetLastError();
  return r == cudaSuccess ? 0 : -1;
}

static int route(const RouteParams& p, const float* dweights, void* dlogits, cudaStream_t s) {
  if (p.E < 1 || p.E > 1024 || p.k < 1 || p.k > ROUTE_MAX_K || p.groups < 1 || p.groups > 32 || p.E % p.groups ||
      p.top_groups < 1 || p.top_groups > p.groups || p.k > p.E / p.groups * p.top_groups ||
      (p.two_best && p.top_groups < p.groups && p.E / p.groups < 2) || p.type < 0 || p.type > 2 || p.scale == 0.f)
    return -10;
  if (p.T == 0) return 0;
  if (dweights) {
    if (p.E <= 64 && p.k <= 8) {
      if (p.E <= 8) return launch_route_bwd<8, 1>(p, dweights, dlogits, s);
      if (p.E <= 16) return launch_route_bwd<8, 2>(p, dweights, dlogits, s);
      if (p.E <= 32) return launch_route_bwd<8, 4>(p, dweights, dlogits, s);
      return launch_route_bwd<8, 8>(p, dweights, dlogits, s);
    }
    if (p.E <= 32) return launch_route_bwd<32, 1>(p, dweights, dlogits, s);
    if (p.E <= 64) return launch_route_bwd<32, 2>(p, dweights, dlogits, s);
    if (p.E <= 128) return launch_route_bwd<32, 4>(p, dweights, dlogits, s);
    if (p.E <= 256) return launch_route_bwd<32, 8>(p, dweights, dlogits, s);
    if (p.E <= 512) return launch_route_bwd<32, 16>(p, dweights, dlogits, s);
    return launch_route_bwd<32, 32>(p, dweights, dlogits, s);
  }
  // Eight lanes per token where they hold the logits and have a lane per chosen expert: 65536 tokens, 6 of 64 experts 20 us (a warp
  // per token: 33), backward 10.  Sixteen lanes for up to 256 experts lose what they save: at 32768 tokens, 8 of
  // 256 in groups with a bias, they took 58 us where a warp per token took 55 (now 46), though they issue a fifth fewer instructions.
  if (p.E <= 64 && p.k <= 8 && p.top_groups == p.groups) {
    if (p.E <= 8) return launch_route<8, 1>(p, s);
    if (p.E <= 16) return launch_route<8, 2>(p, s);
    if (p.E <= 32) return launch_route<8, 4>(p, s);
    return launch_route<8, 8>(p, s);
  }
  if (p.E <= 32) return launch_route<32, 1>(p, s);
  if (p.E <= 64) return launch_route<32, 2>(p, s);
  if (p.E <= 128) return launch_route<32, 4>(p, s);
  if (p.E <= 256) return launch_route<32, 8>(p, s);
  if (p.E <= 512) return launch_route<32, 16>(p, s);
  return launch_route<32, 32>(p, s);
}

}  // namespace b2

using namespace b2;

extern "C" {

// logits [T, E] contiguous (type 0 fp32, 1 bf16, 2 fp16), bias fp32 [E] or null -> weights fp32 [T, k], idx int64 [T, k].
int b2_route_topk(const void* logits, const float* bias, float* weights, long long* idx, long long T, int E, int k, int type,
                  int sigmoid, int groups, int top_groups, int two_best, int renormalize, float scale, cudaStream_t s) {
  const RouteParams p = {logits, bias, weights, idx, T, E, k, type, sigmoid, groups, top_groups, two_best, renormalize, scale,
                         groups > 0 ? E / groups : 0, 0};
  return route(p, nullptr, nullptr, s);
}

// The gradient of the logits, in their type, from that of the weights.
int b2_route_topk_bwd(const void* logits, const float* weights, const long long* idx, const float* dweights, void* dlogits,
                      long long T, int E, int k, int type, int sigmoid, int renormalize, float scale, cudaStream_t s) {
  const RouteParams p = {logits, nullptr, const_cast<float*>(weights), const_cast<long long*>(idx), T, E, k, type, sigmoid,
                         1, 1, 0, renormalize, scale, E, 0};
  return route(p, dweights, dlogits, s);
}

}  // extern "C"
