// The seam between two blocks of a decoder with norms on both sides of a block, in one pass each way:
//
//   n = rms(delta) w_d          the norm of what the block put out
//   s = r x + g n               its gate and the residual sum, r a number of the caller
//   y = rms(s) w                the norm in front of the next block, of the sum before it is rounded
//
// The gate g is absent, or one value for each channel, each sequence and channel, each token, or each element.
//   dS = ds + rstd (dy w - yhat mean(dy w yhat)),  dx = r dS,  dn = g dS,  dg = dS n summed over what shares g
//   ddelta = rstd_d (dn w_d - nhat mean(dn w_d nhat)),  dw = sum dy yhat,  dw_d = sum dn nhat
// The backward pass forms s again from x and delta, which the caller keeps anyway, instead of reading the rounded sum.
//
// Both directions are bound by memory traffic: 4 tensors forward, 6 backward, a gate for each element one and two more.
// W warps work on a row, 8 columns of a lane are one access, all arithmetic is fp32.  There are two forms of each kernel.  The
// one for many rows brings blocks of rows into a ring in shared memory by bulk copies: a row goes through two
// sums over its columns one after the other, forward and backward, and without rows that arrive meanwhile an SM waits most of the
// time.  The other reads straight from global memory: for few rows, where there is nothing to read ahead, and for rows that bulk
// copies do not take (widths that are no multiple of 8, addresses off a 16-byte boundary).
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "chain.cuh"
#include "entries.h"
#include "ptx.cuh"

namespace b2 {

constexpr int GN_VECS = 2;                   // runs of 8 columns per lane
constexpr int GN_MAX_D = 8192;

enum GateKind : int { GATE_NONE = 0, GATE_CHANNEL = 1, GATE_SEQUENCE = 2, GATE_TOKEN = 3, GATE_FULL = 4 };

struct GatedNormParams {
  const void* x;
  const void* delta;
  const float* delta_weight;
  const float* weight;
  const void* gate;          // [D], [rows / seq, D], [rows] or [rows, D]
  void* summed;
  void* normed;
  float* delta_rstd;         // [rows]
  float* rstd;               // [rows]
  const void* dsummed;       // null: zero
  const void* dnormed;       // null: zero
  void* dx;
  void* ddelta;
  void* dgate;               // [rows] or [rows, D] (GATE_TOKEN, GATE_FULL)
  float* partial;            // [2][CTAs][D] column sums, then for GATE_SEQUENCE [CTAs + sequences][rows at a time][D]
  int* status;               // device word, non-zero: a wait ran out
  int rows, D, seq, gate_kind, gate_f32, aligned, stages;
  float residual_scale, eps;
};

template <typename T> __device__ __forceinline__ float to_f32(T v);
template <> __device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
template <> __device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }
template <> __device__ __forceinline__ float to_f32(float v) { return v; }
template <typename T> __device__ __forceinline__ T from_f32(float v);
template <> __device__ __forceinline__ __nv_bfloat16 from_f32(float v) { return __float2bfloat16(v); }
template <> __device__ __forceinline__ __half from_f32(float v) { return __float2half(v); }
template <> __device__ __forceinline__ float from_f32(float v) { return v; }

template <typename T> struct is_bf16 { static constexpr bool value = false; };
template <> struct is_bf16<__nv_bfloat16> { static constexpr bool value = true; };

// 8 columns from ``col`` on, zeros behind column D.
template <typename T>
struct Eight {
  alignas(16) T v[8];
  __device__ __forceinline__ void load(const T* row, int col, int D, bool aligned) {
    if (aligned) {
      if (col < D) {
#pragma unroll
        for (int i = 0; i < static_cast<int>(sizeof(v) / 16); ++i)
          reinterpret_cast<uint4*>(v)[i] = reinterpret_cast<const uint4*>(row + col)[i];
        return;
      }
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = col + i < D ? row[col + i] : from_f32<T>(0.f);
  }
  __device__ __forceinline__ void store(T* row, int col, int D, bool aligned) const {
    if (aligned) {
      if (col < D) {
#pragma unroll
        for (int i = 0; i < static_cast<int>(sizeof(v) / 16); ++i)
          reinterpret_cast<uint4*>(row + col)[i] = reinterpret_cast<const uint4*>(v)[i];
      }
      return;
    }
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (col + i < D) row[col + i] = v[i];
  }
  // two values at a time: one instruction each way for a pair of 16-bit values
  __device__ __forceinline__ void get(float (&f)[8]) const {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      float2 t;
      if constexpr (sizeof(T) == 4) t = make_float2(v[2 * i], v[2 * i + 1]);
      else if constexpr (is_bf16<T>::value) t = __bfloat1622float2(reinterpret_cast<const __nv_bfloat162*>(v)[i]);
      else t = __half22float2(reinterpret_cast<const __half2*>(v)[i]);
      f[2 * i] = t.x;
      f[2 * i + 1] = t.y;
    }
  }
  __device__ __forceinline__ void set(const float (&f)[8]) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (sizeof(T) == 4) {
        v[2 * i] = f[2 * i];
        v[2 * i + 1] = f[2 * i + 1];
      } else if constexpr (is_bf16<T>::value) {
        reinterpret_cast<__nv_bfloat162*>(v)[i] = __floats2bfloat162_rn(f[2 * i], f[2 * i + 1]);
      } else {
        reinterpret_cast<__half2*>(v)[i] = __floats2half2_rn(f[2 * i], f[2 * i + 1]);
      }
    }
  }
};

template <typename T>
__device__ __forceinline__ void load_f32x8(const T* row, int col, int D, bool aligned, float (&f)[8]) {
  Eight<T> e;
  e.load(row, col, D, aligned);
  e.get(f);
}

// The gate of 8 columns of a row.
template <typename T>
__device__ __forceinline__ void load_gate(const GatedNormParams& p, long long row, int col, float (&g)[8]) {
  if (p.gate_kind == GATE_NONE) {
#pragma unroll
    for (int i = 0; i < 8; ++i) g[i] = 1.f;
    return;
  }
  if (p.gate_kind == GATE_TOKEN) {
    const float v = p.gate_f32 ? static_cast<const float*>(p.gate)[row] : to_f32<T>(static_cast<const T*>(p.gate)[row]);
#pragma unroll
    for (int i = 0; i < 8; ++i) g[i] = v;
    return;
  }
  const long long at = (p.gate_kind == GATE_CHANNEL ? 0 : p.gate_kind == GATE_SEQUENCE ? row / p.seq : row) * p.D;
  if (p.gate_f32) load_f32x8(static_cast<const float*>(p.gate) + at, col, p.D, p.aligned, g);
  else load_f32x8(static_cast<const T*>(p.gate) + at, col, p.D, p.aligned, g);
}

// Sum over the W warps of a row.  ``scratch`` alternates between two halves, so that one barrier per sum is enough.
template <int W>
__device__ __forceinline__ float gn_row_sum(float v, float (*scratch)[W], int slot, int in_row, int lane) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  if (W == 1) return v;
  if (lane == 0) scratch[slot][in_row] = v;
  asm volatile("bar.sync %0, %1;" ::"r"(1 + slot), "r"(W * 32) : "memory");
  float total = 0.f;
#pragma unroll
  for (int i = 0; i < W; ++i) total += scratch[slot][i];
  return total;
}

template <int W> constexpr int gn_threads() { return W == 16 ? 512 : 256; }
template <int W> constexpr int gn_rows() { return gn_threads<W>() / 32 / W; }        // rows a CTA works on at a time

template <typename T, int W>
__global__ void __launch_bounds__(gn_threads<W>()) gated_norm_fwd_kernel(const GatedNormParams p) {
  chain_begin();
  constexpr int R = gn_rows<W>(), V = GN_VECS;
  __shared__ float scratch[2][R][W];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, slot = warp / W, in_row = warp % W;
  const int D = p.D;
  const float inv = 1.f / D;
  for (long long row = static_cast<long long>(blockIdx.x) * R + slot; row < p.rows; row += static_cast<long long>(gridDim.x) * R) {
    const T* x = static_cast<const T*>(p.x) + row * D;
    const T* delta = static_cast<const T*>(p.delta) + row * D;
    Eight<T> xr[V], dr[V];
#pragma unroll
    for (int c = 0; c < V; ++c) {
      const int col = ((c * W + in_row) * 32 + lane) * 8;
      dr[c].load(delta, col, D, p.aligned);
      xr[c].load(x, col, D, p.aligned);
    }
    float sum = 0.f;
#pragma unroll
    for (int c = 0; c < V; ++c) {
      float d[8];
      dr[c].get(d);
#pragma unroll
      for (int i = 0; i < 8; ++i) sum += d[i] * d[i];
    }
    const float rd = rsqrtf(gn_row_sum<W>(sum, scratch[0], slot, in_row, lane) * inv + p.eps);
    float s[V][8];
    sum = 0.f;
#pragma unroll
    for (int c = 0; c < V; ++c) {
      const int col = ((c * W + in_row) * 32 + lane) * 8;
      float d[8], xv[8], g[8], wd[8];
      dr[c].get(d);
      xr[c].get(xv);
      load_gate<T>(p, row, col, g);
      load_f32x8(p.delta_weight, col, D, p.aligned, wd);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        s[c][i] = xv[i] * p.residual_scale + d[i] * rd * wd[i] * g[i];
        sum += s[c][i] * s[c][i];
      }
      Eight<T> out;
      out.set(s[c]);
      out.store(static_cast<T*>(p.summed) + row * D, col, D, p.aligned);
    }
    const float r = rsqrtf(gn_row_sum<W>(sum, scratch[1], slot, in_row, lane) * inv + p.eps);
    if (in_row == 0 && lane == 0) {
      p.delta_rstd[row] = rd;
      p.rstd[row] = r;
    }
#pragma unroll
    for (int c = 0; c < V; ++c) {
      const int col = ((c * W + in_row) * 32 + lane) * 8;
      float w[8];
      load_f32x8(p.weight, col, D, p.aligned, w);
#pragma unroll
      for (int i = 0; i < 8; ++i) s[c][i] *= r * w[i];
      Eight<T> out;
      out.set(s[c]);
      out.store(static_cast<T*>(p.normed) + row * D, col, D, p.aligned);
    }
  }
}

// A CTA has a run of rows, at least one, which its slots (of W warps) take in turn.
__device__ __forceinline__ int gn_first_row(int cta, int rows, int ctas) { return cta * (rows / ctas) + min(cta, rows % ctas); }
__device__ __forceinline__ int gn_cta_of(int row, int rows, int ctas) {
  const int base = rows / ctas, longer = rows % ctas * (base + 1);          // the first ones have a row more
  return row < longer ? row / (base + 1) : rows % ctas + (row - longer) / base;
}

// One row of column sums per CTA: its slots' sums are added in their order through ``columns`` (a row for each of two sums).
template <int R, int W, int THREADS>
__device__ __forceinline__ void gn_store_sums(const GatedNormParams& p, float (&dw)[GN_VECS][8], float (&dwd)[GN_VECS][8],
                                              float* columns, int slot, int in_row, int lane) {
  constexpr int V = GN_VECS, WIDTH = W * 32 * 8 * V;
  if (R > 1) {
    for (int k = 0; k < R; ++k) {
      asm volatile("bar.sync 15, %0;" ::"r"(THREADS) : "memory");
      if (slot != k) continue;
#pragma unroll
      for (int c = 0; c < V; ++c) {
        const int col = ((c * W + in_row) * 32 + lane) * 8;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          columns[col + i] = dw[c][i] += k ? columns[col + i] : 0.f;
          columns[WIDTH + col + i] = dwd[c][i] += k ? columns[WIDTH + col + i] : 0.f;
        }
      }
    }
    if (slot != R - 1) return;
  }
#pragma unroll
  for (int c = 0; c < V; ++c) {
    const int col = ((c * W + in_row) * 32 + lane) * 8;
    Eight<float> f;
    f.set(dw[c]);
    f.store(p.partial + static_cast<long long>(blockIdx.x) * p.D, col, p.D, p.aligned);
    f.set(dwd[c]);
    f.store(p.partial + (static_cast<long long>(gridDim.x) + blockIdx.x) * p.D, col, p.D, p.aligned);
  }
}

// Column sums stay in registers while a worker goes through its rows: dw and, where a gate of its own has no column sum, dw_d.
// With a gate that rows share the sum a = sum of dS nhat gives both its gradient, w_d a, and dw_d, g a; for a gate per sequence a
// is stored wherever the sequence changes, in place ``sequence + CTA`` and slot, which no other has.
template <typename T, int W, int GATE>       // GATE: 0 no column sums, 1 a gate per channel, 2 a gate per sequence
__global__ void __launch_bounds__(gn_threads<W>()) gated_norm_bwd_kernel(const GatedNormParams p) {
  chain_begin();
  constexpr int R = gn_rows<W>(), V = GN_VECS;
  __shared__ float scratch[2][R][W];
  __shared__ float columns[R > 1 ? 2 * W * 32 * 8 * V : 1];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, slot = warp / W, in_row = warp % W;
  const int D = p.D;
  const float inv = 1.f / D;
  const int begin = gn_first_row(blockIdx.x, p.rows, gridDim.x), end = gn_first_row(blockIdx.x + 1, p.rows, gridDim.x);
  float dw[V][8], dwd[V][8], a[GATE == 2 ? V : 1][8];
#pragma unroll
  for (int c = 0; c < V; ++c) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      dw[c][i] = dwd[c][i] = 0.f;
      if (GATE == 2) a[c][i] = 0.f;
    }
  }
  float* const sequences = p.partial + 2LL * gridDim.x * D;
  for (int row = begin + slot; row < end; row += R) {
    const long long at = static_cast<long long>(row) * D;
    Eight<T> xr[V], dr[V], sr[V], yr[V];
#pragma unroll
    for (int c = 0; c < V; ++c) {
      const int col = ((c * W + in_row) * 32 + lane) * 8;
      xr[c].load(static_cast<const T*>(p.x) + at, col, D, p.aligned);
      dr[c].load(static_cast<const T*>(p.delta) + at, col, D, p.aligned);
      if (p.dnormed) yr[c].load(static_cast<const T*>(p.dnormed) + at, col, D, p.aligned);
      if (p.dsummed) sr[c].load(static_cast<const T*>(p.dsummed) + at, col, D, p.aligned);
    }
    const float rd = p.delta_rstd[row], r = p.rstd[row];
    float hat[V][8];                                   // of the sum
    float sum = 0.f;
#pragma unroll
    for (int c = 0; c < V; ++c) {
      const int col = ((c * W + in_row) * 32 + lane) * 8;
      float d[8], xv[8], g[8], wd[8];
      dr[c].get(d);
      xr[c].get(xv);
      load_gate<T>(p, row, col, g);
      load_f32x8(p.delta_weight, col, D, p.aligned, wd);
#pragma unroll
      for (int i = 0; i < 8; ++i) hat[c][i] = (xv[i] * p.residual_scale + d[i] * rd * wd[i] * g[i]) * r;
      if (p.dnormed) {
        float dy[8], w[8];
        yr[c].get(dy);
        load_f32x8(p.weight, col, D, p.aligned, w);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          dw[c][i] += dy[i] * hat[c][i];
          sum += dy[i] * w[i] * hat[c][i];
        }
      }
    }
    const float mean = gn_row_sum<W>(sum, scratch[0], slot, in_row, lane) * inv;
    float ds[V][8];
    sum = 0.f;
#pragma unroll
    for (int c = 0; c < V; ++c) {
      const int col = ((c * W + in_row) * 32 + lane) * 8;
      float d[8], g[8], wd[8];
      dr[c].get(d);
      load_gate<T>(p, row, col, g);
      load_f32x8(p.delta_weight, col, D, p.aligned, wd);
      if (p.dsummed) sr[c].get(ds[c]);
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (!p.dsummed) ds[c][i] = 0.f;
      if (p.dnormed) {
        float dy[8], w[8];
        yr[c].get(dy);
        load_f32x8(p.weight, col, D, p.aligned, w);
#pragma unroll
        for (int i = 0; i < 8; ++i) ds[c][i] += r * (dy[i] * w[i] - hat[c][i] * mean);
      }
      float out[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) out[i] = ds[c][i] * p.residual_scale;
      Eight<T> e;
      e.set(out);
      e.store(static_cast<T*>(p.dx) + at, col, D, p.aligned);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float nhat = d[i] * rd, part = ds[c][i] * nhat;       // columns behind D hold zeros
        if (GATE == 2) a[c][i] += part;
        dwd[c][i] += GATE == 1 ? part : part * g[i];
        out[i] = part * wd[i];                                      // dS n
        sum += p.gate_kind == GATE_TOKEN ? out[i] : out[i] * g[i];
        ds[c][i] *= g[i] * wd[i];
      }
      if (p.gate_kind == GATE_FULL) {
        if (p.gate_f32) {
          Eight<float> f;
          f.set(out);
          f.store(static_cast<float*>(p.dgate) + at, col, D, p.aligned);
        } else {
          e.set(out);
          e.store(static_cast<T*>(p.dgate) + at, col, D, p.aligned);
        }
      }
    }
    float mean_d = gn_row_sum<W>(sum, scratch[1], slot, in_row, lane);
    if (p.gate_kind == GATE_TOKEN) {
      if (in_row == 0 && lane == 0) {
        if (p.gate_f32) static_cast<float*>(p.dgate)[row] = mean_d;
        else static_cast<T*>(p.dgate)[row] = from_f32<T>(mean_d);
      }
      float g[8];
      load_gate<T>(p, row, 0, g);
      mean_d *= g[0];
    }
    mean_d *= inv;
#pragma unroll
    for (int c = 0; c < V; ++c) {
      const int col = ((c * W + in_row) * 32 + lane) * 8;
      float d[8], out[8];
      dr[c].get(d);
#pragma unroll
      for (int i = 0; i < 8; ++i) out[i] = rd * (ds[c][i] - d[i] * rd * mean_d);
      Eight<T> e;
      e.set(out);
      e.store(static_cast<T*>(p.ddelta) + at, col, D, p.aligned);
    }
    if (GATE == 2 && (row + R >= end || row / p.seq != (row + R) / p.seq)) {
      float* dst = sequences + (static_cast<long long>(row / p.seq + blockIdx.x) * R + slot) * D;
#pragma unroll
      for (int c = 0; c < V; ++c) {
        const int col = ((c * W + in_row) * 32 + lane) * 8;
        Eight<float> f;
        f.set(a[c]);
        f.store(dst, col, D, p.aligned);
#pragma unroll
        for (int i = 0; i < 8; ++i) a[c][i] = 0.f;
      }
    }
  }
  gn_store_sums<R, W, gn_threads<W>()>(p, dw, dwd, columns, slot, in_row, lane);
}

// ------------------------------------------------------------------ many rows: a ring of bulk copies
constexpr int GN_RING = 4;

// The ring of a slot: its rows ``first``, ``first + step``, ... below ``end`` of TENSORS tensors (null ones are left out).  The first
// lane of the slot issues the copies beside its own work (a warp for them would take registers of a third of the others): the
// first ones at the start, the next into a stage once the slot's warps have met at the barrier behind their last read of it.
// A row of tensor i has ``row_bytes[i]`` bytes; all but the last of a stage have those of the first.
template <int TENSORS>
struct GnRing {
  const uint8_t* src[TENSORS];
  uint32_t row_bytes[TENSORS];
  uint8_t* smem;             // this slot's part of stage 0
  uint32_t stage_bytes;      // of all slots
  int stages;
  uint64_t* full;            // a barrier per stage
  int first, step, end;

  __device__ __forceinline__ void issue(int s, int row) const {
    uint32_t bytes = 0;
#pragma unroll
    for (int i = 0; i < TENSORS; ++i) bytes += src[i] ? row_bytes[i] : 0;
    mbar_expect_tx(&full[s], bytes);
#pragma unroll
    for (int i = 0; i < TENSORS; ++i)
      if (src[i]) bulk_load(smem + s * stage_bytes + i * row_bytes[0], src[i] + static_cast<size_t>(row) * row_bytes[i], &full[s],
                            row_bytes[i]);
  }
  __device__ __forceinline__ void start() const {
    for (int s = 0; s < stages && first + s * step < end; ++s) issue(s, first + s * step);
  }
  // The stage of row ``row``, which has been read, gets the row that is ``stages`` further.
  __device__ __forceinline__ void refill(int s, int row) const {
    row += stages * step;
    if (row < end) issue(s, row);
  }
  // A slot that gave up waits (with a limit) for what may be in flight before its shared memory goes to another CTA.
  __device__ __forceinline__ void drain(int turns) const {
    for (int i = turns < stages ? 0 : turns - stages; i < turns; ++i) mbar_wait(&full[i % stages], (i / stages) & 1);
  }
};

__device__ __forceinline__ void gn_init(uint64_t* bars, int count) {
  if (static_cast<int>(threadIdx.x) < count) mbar_init(&bars[threadIdx.x], 1);
  mbar_fence_init();
  __syncthreads();
}

// Waits for a stage.  A warp whose wait ran out reports and goes on without waiting: the warps of a row meet at barriers.
__device__ __forceinline__ void gn_arrived(bool& here, uint64_t& bar, uint32_t phase, int* status, int lane) {
  if (!here) return;
  here = mbar_wait(&bar, phase);
  if (!here && lane == 0) atomicExch(status, 6);
}

template <typename T>
__device__ __forceinline__ void ring_load(const uint8_t* row, int col, float (&f)[8]) {
  Eight<T> e;
#pragma unroll
  for (int i = 0; i < static_cast<int>(sizeof(T) / 2); ++i)
    reinterpret_cast<uint4*>(e.v)[i] = reinterpret_cast<const uint4*>(row + col * sizeof(T))[i];
  e.get(f);
}

// g w_d of a lane's columns (w_d where the gate is no column vector); zeros behind column D
template <typename T, int W, int G>
__device__ __forceinline__ void load_gwd(const GatedNormParams& p, long long row, int in_row, int lane, float (&gwd)[GN_VECS][8]) {
#pragma unroll
  for (int c = 0; c < GN_VECS; ++c) {
    const int col = ((c * W + in_row) * 32 + lane) * 8;
    load_f32x8(p.delta_weight, col, p.D, true, gwd[c]);
    if (G == GATE_CHANNEL || G == GATE_SEQUENCE) {
      float g[8];
      load_gate<T>(p, row, col, g);
#pragma unroll
      for (int i = 0; i < 8; ++i) gwd[c][i] *= g[i];
    }
  }
}

template <int W> constexpr int gn_ctas_per_sm() { return W == 16 ? 1 : 2; }

// One barrier per row: the sum over delta of the next row is formed before the sum over s of the present one, and both cross the
// warps together.  A CTA has a run of rows, so that a gate per sequence is loaded once per sequence and CTA.
template <typename T, int W, int G>
__global__ void __launch_bounds__(gn_threads<W>(), gn_ctas_per_sm<W>()) gated_norm_fwd_ring_kernel(const GatedNormParams p) {
  chain_begin();
  constexpr int R = gn_rows<W>(), V = GN_VECS;
  extern __shared__ __align__(128) uint8_t gn_smem[];
  __shared__ uint64_t bars[R][GN_RING];
  __shared__ float2 scratch[2][R][W];
  gn_init(bars[0], R * GN_RING);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, slot = warp / W, in_row = warp % W, D = p.D;
  const uint32_t row_bytes = D * sizeof(T), gate_bytes = p.gate_f32 ? D * 4 : row_bytes;
  const uint32_t slot_bytes = 2 * row_bytes + (G == GATE_FULL ? gate_bytes : 0), stage_bytes = R * slot_bytes;
  const int begin = gn_first_row(blockIdx.x, p.rows, gridDim.x), end = gn_first_row(blockIdx.x + 1, p.rows, gridDim.x);
  const uint8_t* const mine = gn_smem + slot * slot_bytes;
  const GnRing<3> ring = {{static_cast<const uint8_t*>(p.x), static_cast<const uint8_t*>(p.delta),
                           G == GATE_FULL ? static_cast<const uint8_t*>(p.gate) : nullptr},
                          {row_bytes, row_bytes, gate_bytes}, gn_smem + slot * slot_bytes, stage_bytes, p.stages, bars[slot],
                          begin + slot, R, end};
  const bool leader = in_row == 0 && lane == 0;
  if (leader) ring.start();
  const float inv = 1.f / D;
  float gwd[V][8], w[V][8];
  if (G != GATE_SEQUENCE) load_gwd<T, W, G>(p, 0, in_row, lane, gwd);
#pragma unroll
  for (int c = 0; c < V; ++c) load_f32x8(p.weight, ((c * W + in_row) * 32 + lane) * 8, D, true, w[c]);
  bool here = true;
  // sum of squares of delta's columns of this lane in a stage that has arrived
  auto squares = [&](int stage) {
    float sum = 0.f;
#pragma unroll
    for (int c = 0; c < V; ++c) {
      const int col = ((c * W + in_row) * 32 + lane) * 8;
      if (col >= D) continue;
      float d[8];
      ring_load<T>(mine + stage * stage_bytes + row_bytes, col, d);
#pragma unroll
      for (int i = 0; i < 8; ++i) sum += d[i] * d[i];
    }
    return sum;
  };
  // sums of both over the warps of a row
  auto row_sums = [&](float a, float b, int half) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      a += __shfl_xor_sync(0xffffffffu, a, o);
      b += __shfl_xor_sync(0xffffffffu, b, o);
    }
    if (W == 1) return make_float2(a, b);
    if (lane == 0) scratch[half][slot][in_row] = make_float2(a, b);
    asm volatile("bar.sync %0, %1;" ::"r"(1 + slot), "r"(W * 32) : "memory");
    float2 total = make_float2(0.f, 0.f);
#pragma unroll
    for (int i = 0; i < W; ++i) {
      const float2 v = scratch[half][slot][i];
      total.x += v.x;
      total.y += v.y;
    }
    return total;
  };
  int stage = 0, turn = 0, half = 0;
  uint32_t phase = 0;
  int sequence_end = 0;
  if (begin + slot >= end) return;                   // a slot's warps meet nobody else
  gn_arrived(here, bars[slot][0], 0, p.status, lane);
  float rd = rsqrtf(row_sums(squares(0), 0.f, 1).x * inv + p.eps);
  for (int row = begin + slot; row < end; row += R, ++turn, half ^= 1) {
    if (G == GATE_SEQUENCE && row >= sequence_end) {
      sequence_end = (row / p.seq + 1) * p.seq;
      load_gwd<T, W, G>(p, row, in_row, lane, gwd);
    }
    const float token = G == GATE_TOKEN
                            ? (p.gate_f32 ? static_cast<const float*>(p.gate)[row] : to_f32<T>(static_cast<const T*>(p.gate)[row]))
                            : 1.f;
    const uint8_t* in = mine + stage * stage_bytes;
    const float factor = G == GATE_TOKEN ? rd * token : rd;
    T* const summed = static_cast<T*>(p.summed) + static_cast<size_t>(row) * D;
    T* const normed = static_cast<T*>(p.normed) + static_cast<size_t>(row) * D;
    float s[V][8], sum = 0.f;
#pragma unroll
    for (int c = 0; c < V; ++c) {
      const int col = ((c * W + in_row) * 32 + lane) * 8;
      if (col >= D) continue;
      float d[8];
      ring_load<T>(in, col, s[c]);
      ring_load<T>(in + row_bytes, col, d);
      if (G == GATE_FULL) {
        float g[8];
        if (p.gate_f32) ring_load<float>(in + 2 * row_bytes, col, g);
        else ring_load<T>(in + 2 * row_bytes, col, g);
#pragma unroll
        for (int i = 0; i < 8; ++i) d[i] *= g[i];
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        s[c][i] = s[c][i] * p.residual_scale + d[i] * factor * gwd[c][i];
        sum += s[c][i] * s[c][i];
      }
      Eight<T> out;
      out.set(s[c]);
      out.store(summed, col, D, true);
    }
    const int read = stage;
    if (++stage == p.stages) {
      stage = 0;
      phase ^= 1;
    }
    float next = 0.f;
    if (row + R < end) {
      gn_arrived(here, bars[slot][stage], phase, p.status, lane);
      next = squares(stage);
    }
    const float2 sums = row_sums(sum, next, half);
    if (leader) ring.refill(read, row);
    const float r = rsqrtf(sums.x * inv + p.eps);
    if (leader) {
      p.delta_rstd[row] = rd;
      p.rstd[row] = r;
    }
#pragma unroll
    for (int c = 0; c < V; ++c) {
      const int col = ((c * W + in_row) * 32 + lane) * 8;
      if (col >= D) continue;
#pragma unroll
      for (int i = 0; i < 8; ++i) s[c][i] *= r * w[c][i];
      Eight<T> out;
      out.set(s[c]);
      out.store(normed, col, D, true);
    }
    rd = rsqrtf(sums.y * inv + p.eps);
  }
  if (leader && !here) ring.drain(turn);
}

// A value that a second phase needs again is formed again from the row in shared memory: two CTAs per SM leave 112 registers, of
// which the column sums and g w_d take 48.  w is read from shared memory, and so is dw_d for a gate per sequence, which is
// touched once per sequence.
template <typename T, int W, int G>
__global__ void __launch_bounds__(gn_threads<W>(), gn_ctas_per_sm<W>()) gated_norm_bwd_ring_kernel(const GatedNormParams p) {
  chain_begin();
  constexpr int R = gn_rows<W>(), V = GN_VECS, THREADS = gn_threads<W>();
  extern __shared__ __align__(128) uint8_t gn_smem[];
  __shared__ uint64_t bars[R][GN_RING];
  __shared__ float scratch[2][R][W];
  gn_init(bars[0], R * GN_RING);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, slot = warp / W, in_row = warp % W, D = p.D;
  const uint32_t row_bytes = D * sizeof(T), gate_bytes = p.gate_f32 ? D * 4 : row_bytes;
  const uint32_t slot_bytes = 4 * row_bytes + (G == GATE_FULL ? gate_bytes : 0), stage_bytes = R * slot_bytes;
  const int begin = gn_first_row(blockIdx.x, p.rows, gridDim.x), end = gn_first_row(blockIdx.x + 1, p.rows, gridDim.x);
  const GnRing<5> ring = {{static_cast<const uint8_t*>(p.x), static_cast<const uint8_t*>(p.delta),
                           static_cast<const uint8_t*>(p.dnormed), static_cast<const uint8_t*>(p.dsummed),
                           G == GATE_FULL ? static_cast<const uint8_t*>(p.gate) : nullptr},
                          {row_bytes, row_bytes, row_bytes, row_bytes, gate_bytes}, gn_smem + slot * slot_bytes, stage_bytes,
                          p.stages, bars[slot], begin + slot, R, end};
  const bool leader = in_row == 0 && lane == 0;
  if (leader) ring.start();
  const float inv = 1.f / D;
  float gwd[V][8], dw[V][8], a[V][8];                // a: dw_d, or the sum of dS nhat where rows share the gate
  if (G != GATE_SEQUENCE) load_gwd<T, W, G>(p, 0, in_row, lane, gwd);
  // a thread's own columns of w, four at a time, then those of dw_d
  float4* const w_smem = reinterpret_cast<float4*>(gn_smem + p.stages * stage_bytes) + threadIdx.x;      // [V * 2][THREADS]
  float* const dwd_smem = reinterpret_cast<float*>(w_smem - threadIdx.x + V * 2 * THREADS) + threadIdx.x;      // [V * 8][THREADS]
#pragma unroll
  for (int c = 0; c < V; ++c) {
    float w[8];
    load_f32x8(p.weight, ((c * W + in_row) * 32 + lane) * 8, D, true, w);
    w_smem[2 * c * THREADS] = make_float4(w[0], w[1], w[2], w[3]);
    w_smem[(2 * c + 1) * THREADS] = make_float4(w[4], w[5], w[6], w[7]);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      dw[c][i] = a[c][i] = 0.f;
      if (G == GATE_SEQUENCE) dwd_smem[(c * 8 + i) * THREADS] = 0.f;
    }
  }
  auto load_w = [&](int c, float (&w)[8]) {
    const float4 lo = w_smem[2 * c * THREADS], hi = w_smem[(2 * c + 1) * THREADS];
    w[0] = lo.x; w[1] = lo.y; w[2] = lo.z; w[3] = lo.w; w[4] = hi.x; w[5] = hi.y; w[6] = hi.z; w[7] = hi.w;
  };
  float* const sequences = p.partial + 2LL * gridDim.x * D;
  int stage = 0, turn = 0;
  uint32_t phase = 0;
  bool here = true;
  int sequence = 0, sequence_end = 0;
  for (int row = begin + slot; row < end; row += R, ++turn) {
    const size_t at = static_cast<size_t>(row) * D;
    if (G == GATE_SEQUENCE && row >= sequence_end) {
      sequence = row / p.seq;
      sequence_end = (sequence + 1) * p.seq;
      load_gwd<T, W, G>(p, row, in_row, lane, gwd);
    }
    const float rd = p.delta_rstd[row], r = p.rstd[row];
    const float token = G == GATE_TOKEN
                            ? (p.gate_f32 ? static_cast<const float*>(p.gate)[row] : to_f32<T>(static_cast<const T*>(p.gate)[row]))
                            : 1.f;
    const uint8_t* const x_row = gn_smem + stage * stage_bytes + slot * slot_bytes;
    const uint8_t *const d_row = x_row + row_bytes, *const dy_row = d_row + row_bytes, *const ds_row = dy_row + row_bytes;
    const uint8_t* const g_row = ds_row + row_bytes;
    gn_arrived(here, bars[slot][stage], phase, p.status, lane);
    const float x_factor = p.residual_scale * r, d_factor = (G == GATE_TOKEN ? rd * token : rd) * r;
    float hat[V][8];                                   // of the sum, then dn w_d
    float sum = 0.f;
#pragma unroll
    for (int c = 0; c < V; ++c) {
      const int col = ((c * W + in_row) * 32 + lane) * 8;
      if (col >= D) continue;
      float d[8], x[8];
      ring_load<T>(x_row, col, x);
      ring_load<T>(d_row, col, d);
      if (G == GATE_FULL) {
        float g[8];
        if (p.gate_f32) ring_load<float>(g_row, col, g);
        else ring_load<T>(g_row, col, g);
#pragma unroll
        for (int i = 0; i < 8; ++i) d[i] *= g[i];
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) hat[c][i] = x[i] * x_factor + d[i] * d_factor * gwd[c][i];
      if (p.dnormed) {
        float dy[8], w[8];
        ring_load<T>(dy_row, col, dy);
        load_w(c, w);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const float t = dy[i] * hat[c][i];
          dw[c][i] += t;
          sum += t * w[i];
        }
      }
    }
    const float mean = gn_row_sum<W>(sum, scratch[0], slot, in_row, lane) * inv * r;
    Eight<T> dr[V];
    sum = 0.f;
#pragma unroll
    for (int c = 0; c < V; ++c) {
      const int col = ((c * W + in_row) * 32 + lane) * 8;
      if (col >= D) continue;
      float d[8], ds[8], out[8];
#pragma unroll
      for (int i = 0; i < static_cast<int>(sizeof(T) / 2); ++i)
        reinterpret_cast<uint4*>(dr[c].v)[i] = reinterpret_cast<const uint4*>(d_row + col * sizeof(T))[i];
      dr[c].get(d);
#pragma unroll
      for (int i = 0; i < 8; ++i) ds[i] = 0.f;
      if (p.dsummed) ring_load<T>(ds_row, col, ds);
      if (p.dnormed) {
        float dy[8], w[8];
        ring_load<T>(dy_row, col, dy);
        load_w(c, w);
#pragma unroll
        for (int i = 0; i < 8; ++i) ds[i] += dy[i] * w[i] * r - hat[c][i] * mean;
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) out[i] = ds[i] * p.residual_scale;
      Eight<T> e;
      e.set(out);
      e.store(static_cast<T*>(p.dx) + at, col, D, true);
      float g[8];
      if (G == GATE_FULL) {
        if (p.gate_f32) ring_load<float>(g_row, col, g);
        else ring_load<T>(g_row, col, g);
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float nhat = d[i] * rd;
        if (G == GATE_FULL) {
          const float part = ds[i] * nhat;
          out[i] = part * gwd[c][i];                               // dS n
          a[c][i] += part * g[i];
          hat[c][i] = ds[i] * gwd[c][i] * g[i];
        } else {
          a[c][i] += G == GATE_TOKEN ? ds[i] * nhat * token : ds[i] * nhat;
          hat[c][i] = ds[i] * gwd[c][i];                           // the token's gate follows with the mean
        }
        sum += hat[c][i] * nhat;
      }
      if (G == GATE_FULL) {
        if (p.gate_f32) {
          Eight<float> f;
          f.set(out);
          f.store(static_cast<float*>(p.dgate) + at, col, D, true);
        } else {
          e.set(out);
          e.store(static_cast<T*>(p.dgate) + at, col, D, true);
        }
      }
    }
    const int read = stage;
    if (++stage == p.stages) {
      stage = 0;
      phase ^= 1;
    }
    const float total = gn_row_sum<W>(sum, scratch[1], slot, in_row, lane);
    if (leader) ring.refill(read, row);
    if (G == GATE_TOKEN && leader) {
      if (p.gate_f32) static_cast<float*>(p.dgate)[row] = total;
      else static_cast<T*>(p.dgate)[row] = from_f32<T>(total);
    }
    const float factor = G == GATE_TOKEN ? rd * token : rd, mean_d = total * inv * rd * factor;
#pragma unroll
    for (int c = 0; c < V; ++c) {
      const int col = ((c * W + in_row) * 32 + lane) * 8;
      if (col >= D) continue;
      float d[8], out[8];
      dr[c].get(d);
#pragma unroll
      for (int i = 0; i < 8; ++i) out[i] = hat[c][i] * factor - d[i] * mean_d;
      Eight<T> e;
      e.set(out);
      e.store(static_cast<T*>(p.ddelta) + at, col, D, true);
    }
    if (G == GATE_SEQUENCE && row + R >= min(end, sequence_end)) {
      float* dst = sequences + (static_cast<long long>(sequence + blockIdx.x) * R + slot) * D;
#pragma unroll
      for (int c = 0; c < V; ++c) {
        const int col = ((c * W + in_row) * 32 + lane) * 8;
        if (col >= D) continue;
        float g[8];
        load_gate<T>(p, row, col, g);
        Eight<float> f;
        f.set(a[c]);
        f.store(dst, col, D, true);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          dwd_smem[(c * 8 + i) * THREADS] += a[c][i] * g[i];
          a[c][i] = 0.f;
        }
      }
    }
  }
  if (G == GATE_SEQUENCE) {
#pragma unroll
    for (int c = 0; c < V; ++c) {
#pragma unroll
      for (int i = 0; i < 8; ++i) a[c][i] = dwd_smem[(c * 8 + i) * THREADS];
    }
  }
  if (leader && !here) ring.drain(turn);
  // the ring's shared memory serves the sums: every copy has landed and been read
  gn_store_sums<R, W, THREADS>(p, dw, a, reinterpret_cast<float*>(gn_smem), slot, in_row, lane);
}

// Column sums of the partial rows: VEC columns a thread, 16 partial rows at a time.  blockIdx.y: 0 dw; 1 dw_d, and the gradient of a
// gate per channel; 2 + i the gradient of sequence i's gate.
template <int VEC>
__global__ void __launch_bounds__(512) gated_norm_sums_kernel(const GatedNormParams p, int ctas, int per_cta, int gate_bf16,
                                                              float* __restrict__ dw, float* __restrict__ dwd,
                                                              void* __restrict__ dgate) {
  chain_begin();
  __shared__ float parts[16][32 * VEC + 1];
  const int D = p.D, col = (blockIdx.x * 32 + threadIdx.x) * VEC;
  auto add = [&](float (&sum)[VEC], const float* src) {
    if constexpr (VEC == 4) {
      const float4 v = *reinterpret_cast<const float4*>(src);
      sum[0] += v.x; sum[1] += v.y; sum[2] += v.z; sum[3] += v.w;
    } else {
      sum[0] += *src;
    }
  };
  for (long long what = blockIdx.y; what < 2 + (p.gate_kind == GATE_SEQUENCE ? p.rows / p.seq : 0); what += gridDim.y) {
    float sum[VEC];
#pragma unroll
    for (int i = 0; i < VEC; ++i) sum[i] = 0.f;
    if (what < 2 && col < D) {
      const float* src = p.partial + what * ctas * D + col;
#pragma unroll 4
      for (int r = threadIdx.y; r < ctas; r += 16) add(sum, src + static_cast<long long>(r) * D);
    } else if (col < D) {
      const int i = static_cast<int>(what - 2), low = i * p.seq, high = low + p.seq;
      const int first = gn_cta_of(low, p.rows, ctas), last = gn_cta_of(high - 1, p.rows, ctas) + 1;
      const int base = p.rows / ctas, extra = p.rows % ctas;           // as gn_first_row
      const float* src = p.partial + (2LL * ctas + static_cast<long long>(i) * per_cta) * D + col;
      const int shift = 31 - __clz(per_cta);                           // a power of two
      for (int r = (first << shift) + threadIdx.y; r < last << shift; r += 16) {
        // a slot that had none of the sequence's rows in this CTA has stored nothing
        const int cta = r >> shift, begin = cta * base + min(cta, extra), end = begin + base + (cta < extra);
        const int from = max(low, begin), rows = min(high, end) - from;
        if ((r - (from - begin) & per_cta - 1) < rows) add(sum, src + static_cast<long long>(r) * D);
      }
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < VEC; ++i) parts[threadIdx.y][threadIdx.x * VEC + i] = sum[i];
    __syncthreads();
    const int column = threadIdx.y * 32 + threadIdx.x, at_col = blockIdx.x * 32 * VEC + column;
    if (column < 32 * VEC && at_col < D) {
      float total = 0.f;
#pragma unroll
      for (int i = 0; i < 16; ++i) total += parts[i][column];
      if (what == 0) {
        dw[at_col] = total;
        continue;
      }
      if (what == 1) {
        float g = 1.f;
        if (p.gate_kind == GATE_CHANNEL) {
          if (p.gate_f32) g = static_cast<const float*>(p.gate)[at_col];
          else if (gate_bf16) g = __bfloat162float(static_cast<const __nv_bfloat16*>(p.gate)[at_col]);
          else g = __half2float(static_cast<const __half*>(p.gate)[at_col]);
        }
        dwd[at_col] = total * g;
        if (p.gate_kind != GATE_CHANNEL) continue;
      }
      const long long at = (what >= 2 ? what - 2 : 0) * D + at_col;
      const float v = total * p.delta_weight[at_col];
      if (p.gate_f32) static_cast<float*>(dgate)[at] = v;
      else if (gate_bf16) static_cast<__nv_bfloat16*>(dgate)[at] = __float2bfloat16(v);
      else static_cast<__half*>(dgate)[at] = __float2half(v);
    }
  }
}

static int gn_sms() {
  static int sms = 0;
  if (!sms) {
    int dev = 0;
    cudaGetDevice(&dev);
    cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
  }
  return sms;
}

static int gn_width(int D) { return D <= 512 ? 1 : D <= 1024 ? 2 : D <= 2048 ? 4 : D <= 4096 ? 8 : 16; }

static int gn_rows_at_once(int D) { const int W = gn_width(D); return W == 16 ? 1 : 8 / W; }

// CTAs of the backward kernels: two per SM, at least two blocks of rows each, so that the partial sums stay small beside the rows.
static int gn_bwd_ctas(int rows, int D) {
  const int W = gn_width(D), R = gn_rows_at_once(D);
  const long long most = gn_sms() * (W == 16 ? 1LL : 2LL), wanted = (rows + 2LL * R - 1) / (2LL * R);
  return static_cast<int>(wanted < most ? wanted : most);
}

// Bytes of one stage of the ring, and how many stages fit beside the ``extra`` bytes: of 227 KiB per SM, less 1 KiB a CTA.
static uint32_t gn_stage_bytes(const GatedNormParams& p, int type, bool backward) {
  const uint32_t row = p.D * (type == 0 ? 4 : 2);
  return gn_rows_at_once(p.D) * ((backward ? 4 : 2) * row + (p.gate_kind == GATE_FULL ? (p.gate_f32 ? p.D * 4 : row) : 0));
}
static uint32_t gn_extra_bytes(const GatedNormParams& p, bool backward) {
  // backward: w, and dw_d of a gate per sequence
  return backward ? (gn_width(p.D) == 16 ? 512 : 256) * GN_VECS * 8 * 4 * (p.gate_kind == GATE_SEQUENCE ? 2 : 1) : 0;
}
static int gn_stages(const GatedNormParams& p, int type, bool backward) {
  const uint32_t per_cta = (gn_width(p.D) == 16 ? 226 : 113) * 1024u - 600u - gn_extra_bytes(p, backward);
  const uint32_t n = per_cta / gn_stage_bytes(p, type, backward);
  return static_cast<int>(n < GN_RING ? n : GN_RING);
}

template <typename... Args>
static cudaError_t gn_launch_ring(void (*kernel)(Args...), int ctas, int threads, uint32_t smem, cudaStream_t s, const GatedNormParams& p) {
  // once per kernel and process; the attribute is the largest that any width asks for
  static thread_local void* last = nullptr;
  if (last != reinterpret_cast<void*>(kernel)) {
    const cudaError_t r = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 226 * 1024 - 600);
    if (r != cudaSuccess) return r;
    last = reinterpret_cast<void*>(kernel);
  }
  return launch_next(kernel, ctas, threads, smem, s, p);
}

// Which form.  A ring of two stages or more, aligned rows, and more blocks of rows than a CTA would have in one go.
template <typename T, int W>
static cudaError_t gn_launch(GatedNormParams& p, int type, bool backward, int gate_bf16, float* dw, float* dwd, cudaStream_t s) {
  constexpr int R = gn_rows<W>(), THREADS = gn_threads<W>();
  const long long blocks = (p.rows + R - 1LL) / R, resident = gn_sms() * static_cast<long long>(gn_ctas_per_sm<W>());
  p.stages = gn_stages(p, type, backward);
  const bool ring = p.aligned && p.stages >= 2 && blocks >= 2 * resident;
  const uint32_t smem = p.stages * gn_stage_bytes(p, type, backward) + gn_extra_bytes(p, backward);
  if (!backward) {
    if (ring) {
      const int ctas = static_cast<int>(resident);
      switch (p.gate_kind) {
        case GATE_NONE:                // as a gate per channel of ones
        case GATE_CHANNEL: return gn_launch_ring(gated_norm_fwd_ring_kernel<T, W, GATE_CHANNEL>, ctas, THREADS, smem, s, p);
        case GATE_SEQUENCE: return gn_launch_ring(gated_norm_fwd_ring_kernel<T, W, GATE_SEQUENCE>, ctas, THREADS, smem, s, p);
        case GATE_TOKEN: return gn_launch_ring(gated_norm_fwd_ring_kernel<T, W, GATE_TOKEN>, ctas, THREADS, smem, s, p);
        default: return gn_launch_ring(gated_norm_fwd_ring_kernel<T, W, GATE_FULL>, ctas, THREADS, smem, s, p);
      }
    }
    const long long most = gn_sms() * (W == 16 ? 4LL : 8LL);
    return launch_next(gated_norm_fwd_kernel<T, W>, static_cast<unsigned>(blocks < most ? blocks : most), THREADS, 0, s, p);
  }
  const int ctas = gn_bwd_ctas(p.rows, p.D);
  cudaError_t r;
  if (ring) {
    switch (p.gate_kind) {
      case GATE_NONE:
      case GATE_CHANNEL: r = gn_launch_ring(gated_norm_bwd_ring_kernel<T, W, GATE_CHANNEL>, ctas, THREADS, smem, s, p); break;
      case GATE_SEQUENCE: r = gn_launch_ring(gated_norm_bwd_ring_kernel<T, W, GATE_SEQUENCE>, ctas, THREADS, smem, s, p); break;
      case GATE_TOKEN: r = gn_launch_ring(gated_norm_bwd_ring_kernel<T, W, GATE_TOKEN>, ctas, THREADS, smem, s, p); break;
      default: r = gn_launch_ring(gated_norm_bwd_ring_kernel<T, W, GATE_FULL>, ctas, THREADS, smem, s, p);
    }
  } else if (p.gate_kind == GATE_CHANNEL) {
    r = launch_next(gated_norm_bwd_kernel<T, W, 1>, ctas, THREADS, 0, s, p);
  } else if (p.gate_kind == GATE_SEQUENCE) {
    r = launch_next(gated_norm_bwd_kernel<T, W, 2>, ctas, THREADS, 0, s, p);
  } else {
    r = launch_next(gated_norm_bwd_kernel<T, W, 0>, ctas, THREADS, 0, s, p);
  }
  if (r != cudaSuccess) return r;
  const long long sums = 2 + (p.gate_kind == GATE_SEQUENCE ? p.rows / p.seq : 0);
  const unsigned y = static_cast<unsigned>(sums < 32768 ? sums : 32768);
  if (p.aligned)
    return launch_next(gated_norm_sums_kernel<4>, dim3((p.D + 127) / 128, y), dim3(32, 16), 0, s, p, ctas, R, gate_bf16, dw, dwd, p.dgate);
  return launch_next(gated_norm_sums_kernel<1>, dim3((p.D + 31) / 32, y), dim3(32, 16), 0, s, p, ctas, R, gate_bf16, dw, dwd, p.dgate);
}

template <typename T>
static cudaError_t gn_dispatch(GatedNormParams& p, int type, bool backward, int gate_bf16, float* dw, float* dwd, cudaStream_t s) {
  switch (gn_width(p.D)) {
    case 1: return gn_launch<T, 1>(p, type, backward, gate_bf16, dw, dwd, s);
    case 2: return gn_launch<T, 2>(p, type, backward, gate_bf16, dw, dwd, s);
    case 4: return gn_launch<T, 4>(p, type, backward, gate_bf16, dw, dwd, s);
    case 8: return gn_launch<T, 8>(p, type, backward, gate_bf16, dw, dwd, s);
    default: return gn_launch<T, 16>(p, type, backward, gate_bf16, dw, dwd, s);
  }
}

static int gated_norm(GatedNormParams& p, int type, bool backward, float* dw, float* dwd, cudaStream_t s) {
  if (p.rows < 0 || p.D < 1 || p.D > GN_MAX_D || type < 0 || type > 2 || p.gate_kind < 0 || p.gate_kind > 4 ||
      (p.gate_kind == GATE_SEQUENCE && (p.seq < 1 || p.rows % p.seq)) || (p.gate_kind != GATE_NONE && !p.gate))
    return -10;
  if (p.rows == 0) return 0;
  uintptr_t bits = 0;
  for (const void* t : {p.x, p.delta, static_cast<const void*>(p.delta_weight), static_cast<const void*>(p.weight),
                        p.gate_kind == GATE_TOKEN ? nullptr : p.gate, static_cast<const void*>(p.summed),
                        static_cast<const void*>(p.normed), p.dsummed, p.dnormed, static_cast<const void*>(p.dx),
                        static_cast<const void*>(p.ddelta), p.gate_kind == GATE_TOKEN ? nullptr : static_cast<const void*>(p.dgate),
                        static_cast<const void*>(p.partial)})
    bits |= reinterpret_cast<uintptr_t>(t);
  p.aligned = p.D % 8 == 0 && bits % 16 == 0;
  const cudaError_t r = type == 0   ? gn_dispatch<float>(p, type, backward, 0, dw, dwd, s)
                        : type == 1 ? gn_dispatch<__nv_bfloat16>(p, type, backward, 1, dw, dwd, s)
                                    : gn_dispatch<__half>(p, type, backward, 0, dw, dwd, s);
  if (r != cudaSuccess) cudaGetLastError();
  return r == cudaSuccess ? 0 : -1;
}

}  // namespace b2

using namespace b2;

extern "C" {

// x, delta, summed, normed [rows, D] of ``type`` (0 fp32, 1 bf16, 2 fp16); weights fp32 [D]; gate_kind see GateKind, the gate of
// ``type`` or fp32; delta_rstd, rstd fp32 [rows].
int b2_gated_norm_fwd(const void* x, const void* delta, const float* delta_weight, const float* weight, const void* gate,
                      void* summed, void* normed, float* delta_rstd, float* rstd, int rows, int D, int seq, int type,
                      int gate_kind, int gate_f32, float residual_scale, float eps, int* status, cudaStream_t s) {
  GatedNormParams p{};
  p.x = x; p.delta = delta; p.delta_weight = delta_weight; p.weight = weight; p.gate = gate; p.summed = summed;
  p.normed = normed; p.delta_rstd = delta_rstd; p.rstd = rstd; p.rows = rows; p.D = D; p.seq = seq;
  p.gate_kind = gate_kind; p.gate_f32 = gate_f32; p.residual_scale = residual_scale; p.status = status; p.eps = eps;
  return gated_norm(p, type, false, nullptr, nullptr, s);
}

// Floats of the workspace of the backward pass.
long long b2_gated_norm_bwd_floats(int rows, int D, int seq, int gate_kind) {
  if (rows < 1 || D < 1 || D > GN_MAX_D || (gate_kind == GATE_SEQUENCE && seq < 1)) return 0;
  const long long ctas = gn_bwd_ctas(rows, D);
  return (2 * ctas + (gate_kind == GATE_SEQUENCE ? (ctas + rows / seq) * gn_rows_at_once(D) : 0)) * D;
}

// Gradients; dsummed and dnormed may be null (zero).  dgate has the gate's shape and type; dw, dwd fp32 [D].
int b2_gated_norm_bwd(const void* dsummed, const void* dnormed, const void* x, const void* delta, const float* delta_weight,
                      const float* weight, const void* gate, const float* delta_rstd, const float* rstd, void* dx, void* ddelta,
                      float* dwd, float* dw, void* dgate, float* partial, int rows, int D, int seq, int type, int gate_kind,
                      int gate_f32, float residual_scale, int* status, cudaStream_t s) {
  GatedNormParams p{};
  p.x = x; p.delta = delta; p.delta_weight = delta_weight; p.weight = weight; p.gate = gate;
  p.delta_rstd = const_cast<float*>(delta_rstd); p.rstd = const_cast<float*>(rstd); p.dsummed = dsummed; p.dnormed = dnormed;
  p.dx = dx; p.ddelta = ddelta; p.dgate = dgate; p.partial = partial; p.rows = rows; p.D = D; p.seq = seq;
  p.gate_kind = gate_kind; p.gate_f32 = gate_f32; p.residual_scale = residual_scale; p.status = status;
  return gated_norm(p, type, true, dw, dwd, s);
}

}  // extern "C"
