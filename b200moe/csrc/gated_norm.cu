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
// A row is in the registers of W warps; 8 columns of a lane are one access.  All arithmetic is fp32.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "chain.cuh"

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
  float* partial;            // [2][CTAs][D] column sums, then for GATE_SEQUENCE [workers + sequences][D]
  int rows, D, seq, gate_kind, gate_f32, aligned;
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
  __device__ __forceinline__ void get(float (&f)[8]) const {
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] = to_f32<T>(v[i]);
  }
  __device__ __forceinline__ void set(const float (&f)[8]) {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = from_f32<T>(f[i]);
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

// A worker is W warps that share a row.  Each has a run of rows, at least one: those beyond the number of rows have none.
__host__ __device__ __forceinline__ long long gn_workers(long long ctas, int per_cta, long long rows) {
  return ctas * per_cta < rows ? ctas * per_cta : rows;
}
__host__ __device__ __forceinline__ long long gn_first_row(long long worker, long long rows, long long workers) {
  return worker * rows / workers;
}
__host__ __device__ __forceinline__ long long gn_worker_of(long long row, long long rows, long long workers) {
  return ((row + 1) * workers - 1) / rows;
}

// Column sums stay in registers while a worker goes through its rows: dw and, where a gate of its own has no column sum, dw_d.
// With a gate that rows share the sum a = sum of dS nhat gives both its gradient, w_d a, and dw_d, g a; for a gate per sequence a
// is stored wherever the sequence changes, in place ``sequence + worker``, which no other pair has.
template <typename T, int W, int GATE>       // GATE: 0 no column sums, 1 a gate per channel, 2 a gate per sequence
__global__ void __launch_bounds__(gn_threads<W>()) gated_norm_bwd_kernel(const GatedNormParams p) {
  chain_begin();
  constexpr int R = gn_rows<W>(), V = GN_VECS;
  __shared__ float scratch[2][R][W];
  __shared__ float columns[R > 1 ? 2 : 1][R > 1 ? W * 32 * 8 * V : 1];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, slot = warp / W, in_row = warp % W;
  const int D = p.D;
  const float inv = 1.f / D;
  const long long workers = gn_workers(gridDim.x, R, p.rows), worker = static_cast<long long>(blockIdx.x) * R + slot;
  const long long begin = worker < workers ? gn_first_row(worker, p.rows, workers) : 0;
  const long long end = worker < workers ? gn_first_row(worker + 1, p.rows, workers) : 0;
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
  long long left = GATE == 2 && begin < end ? p.seq - begin % p.seq : 0;      // rows up to the end of the sequence
  for (long long row = begin; row < end; ++row) {
    const long long at = row * D;
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
    if (GATE == 2 && (--left == 0 || row + 1 == end)) {
      left = p.seq;
      float* dst = sequences + (row / p.seq + worker) * D;
#pragma unroll
      for (int c = 0; c < V; ++c) {
        const int col = ((c * W + in_row) * 32 + lane) * 8;
        Eight<float> f;
        f.set(a[c]);
        f.store(dst, col, D, D % 4 == 0 && p.aligned);
#pragma unroll
        for (int i = 0; i < 8; ++i) a[c][i] = 0.f;
      }
    }
  }
  // one row of sums per CTA: its rows' sums are added in the order of the slots
  if (R > 1) {
    for (int k = 0; k < R; ++k) {
      __syncthreads();
      if (slot != k) continue;
#pragma unroll
      for (int c = 0; c < V; ++c) {
        const int col = ((c * W + in_row) * 32 + lane) * 8;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          columns[0][col + i] = dw[c][i] += k ? columns[0][col + i] : 0.f;
          columns[R > 1 ? 1 : 0][col + i] = dwd[c][i] += k ? columns[R > 1 ? 1 : 0][col + i] : 0.f;
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
    f.store(p.partial + static_cast<long long>(blockIdx.x) * D, col, D, p.aligned);
    f.set(dwd[c]);
    f.store(p.partial + (static_cast<long long>(gridDim.x) + blockIdx.x) * D, col, D, p.aligned);
  }
}

// Column sums of the partial rows: 32 columns per CTA, 16 partial rows at a time.  blockIdx.y: 0 dw; 1 dw_d, and the gradient of a
// gate per channel; 2 + i the gradient of sequence i's gate.
__global__ void __launch_bounds__(512) gated_norm_sums_kernel(const GatedNormParams p, int ctas, long long workers, int gate_bf16,
                                                              float* __restrict__ dw, float* __restrict__ dwd,
                                                              void* __restrict__ dgate) {
  chain_begin();
  __shared__ float parts[16][33];
  const int D = p.D, col = blockIdx.x * 32 + threadIdx.x;
  for (long long what = blockIdx.y; what < 2 + (p.gate_kind == GATE_SEQUENCE ? p.rows / p.seq : 0); what += gridDim.y) {
    const float* src = p.partial + what * ctas * D;
    long long first = 0, last = ctas;
    if (what >= 2) {
      const long long i = what - 2;
      src = p.partial + (2LL * ctas + i) * D;
      first = gn_worker_of(i * p.seq, p.rows, workers);
      last = gn_worker_of((i + 1) * p.seq - 1, p.rows, workers) + 1;
    }
    float sum = 0.f;
    if (col < D)
      for (long long r = first + threadIdx.y; r < last; r += 16) sum += src[r * D + col];
    __syncthreads();
    parts[threadIdx.y][threadIdx.x] = sum;
    __syncthreads();
    if (threadIdx.y == 0 && col < D) {
      sum = 0.f;
#pragma unroll
      for (int i = 0; i < 16; ++i) sum += parts[i][threadIdx.x];
      if (what == 0) {
        dw[col] = sum;
        continue;
      }
      if (what == 1) {
        float g = 1.f;
        if (p.gate_kind == GATE_CHANNEL) {
          if (p.gate_f32) g = static_cast<const float*>(p.gate)[col];
          else if (gate_bf16) g = __bfloat162float(static_cast<const __nv_bfloat16*>(p.gate)[col]);
          else g = __half2float(static_cast<const __half*>(p.gate)[col]);
        }
        dwd[col] = sum * g;
        if (p.gate_kind != GATE_CHANNEL) continue;
      }
      const long long at = (what >= 2 ? what - 2 : 0) * D + col;
      const float v = sum * p.delta_weight[col];
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

// CTAs of the backward kernel: two per SM (their registers allow no more), at least two rows for each worker.
static int gn_bwd_ctas(int rows, int D) {
  const int W = gn_width(D), per_cta = W == 16 ? 1 : 8 / W;
  const long long most = gn_sms() * (W == 16 ? 1LL : 2LL), wanted = (rows + 2LL * per_cta - 1) / (2LL * per_cta);
  return static_cast<int>(wanted < most ? wanted : most);
}

template <typename T, int W>
static cudaError_t gn_launch(const GatedNormParams& p, bool backward, int gate_bf16, float* dw, float* dwd, cudaStream_t s) {
  constexpr int R = gn_rows<W>();
  if (!backward) {
    const long long blocks = (p.rows + R - 1) / R, most = gn_sms() * (W == 16 ? 4LL : 8LL);
    return launch_next(gated_norm_fwd_kernel<T, W>, static_cast<unsigned>(blocks < most ? blocks : most), gn_threads<W>(), 0, s, p);
  }
  const int ctas = gn_bwd_ctas(p.rows, p.D);
  cudaError_t r;
  if (p.gate_kind == GATE_CHANNEL) r = launch_next(gated_norm_bwd_kernel<T, W, 1>, ctas, gn_threads<W>(), 0, s, p);
  else if (p.gate_kind == GATE_SEQUENCE) r = launch_next(gated_norm_bwd_kernel<T, W, 2>, ctas, gn_threads<W>(), 0, s, p);
  else r = launch_next(gated_norm_bwd_kernel<T, W, 0>, ctas, gn_threads<W>(), 0, s, p);
  if (r != cudaSuccess) return r;
  const long long sums = 2 + (p.gate_kind == GATE_SEQUENCE ? p.rows / p.seq : 0);
  return launch_next(gated_norm_sums_kernel, dim3((p.D + 31) / 32, static_cast<unsigned>(sums < 32768 ? sums : 32768)),
                     dim3(32, 16), 0, s, p, ctas, gn_workers(ctas, R, p.rows), gate_bf16, dw, dwd, p.dgate);
}

template <typename T>
static cudaError_t gn_dispatch(const GatedNormParams& p, bool backward, int gate_bf16, float* dw, float* dwd, cudaStream_t s) {
  switch (gn_width(p.D)) {
    case 1: return gn_launch<T, 1>(p, backward, gate_bf16, dw, dwd, s);
    case 2: return gn_launch<T, 2>(p, backward, gate_bf16, dw, dwd, s);
    case 4: return gn_launch<T, 4>(p, backward, gate_bf16, dw, dwd, s);
    case 8: return gn_launch<T, 8>(p, backward, gate_bf16, dw, dwd, s);
    default: return gn_launch<T, 16>(p, backward, gate_bf16, dw, dwd, s);
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
  const cudaError_t r = type == 0   ? gn_dispatch<float>(p, backward, 0, dw, dwd, s)
                        : type == 1 ? gn_dispatch<__nv_bfloat16>(p, backward, 1, dw, dwd, s)
                                    : gn_dispatch<__half>(p, backward, 0, dw, dwd, s);
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
                      int gate_kind, int gate_f32, float residual_scale, float eps, cudaStream_t s) {
  GatedNormParams p{};
  p.x = x; p.delta = delta; p.delta_weight = delta_weight; p.weight = weight; p.gate = gate; p.summed = summed;
  p.normed = normed; p.delta_rstd = delta_rstd; p.rstd = rstd; p.rows = rows; p.D = D; p.seq = seq;
  p.gate_kind = gate_kind; p.gate_f32 = gate_f32; p.residual_scale = residual_scale; p.eps = eps;
  return gated_norm(p, type, false, nullptr, nullptr, s);
}

// Floats of the workspace of the backward pass.
long long b2_gated_norm_bwd_floats(int rows, int D, int seq, int gate_kind) {
  if (rows < 1 || D < 1 || D > GN_MAX_D || (gate_kind == GATE_SEQUENCE && seq < 1)) return 0;
  const long long ctas = gn_bwd_ctas(rows, D), W = gn_width(D), R = W == 16 ? 1 : 8 / W;
  return (2 * ctas + (gate_kind == GATE_SEQUENCE ? ctas * R + rows / seq : 0)) * D;
}

// Gradients; dsummed and dnormed may be null (zero).  dgate has the gate's shape and type; dw, dwd fp32 [D].
int b2_gated_norm_bwd(const void* dsummed, const void* dnormed, const void* x, const void* delta, const float* delta_weight,
                      const float* weight, const void* gate, const float* delta_rstd, const float* rstd, void* dx, void* ddelta,
                      float* dwd, float* dw, void* dgate, float* partial, int rows, int D, int seq, int type, int gate_kind,
                      int gate_f32, float residual_scale, cudaStream_t s) {
  GatedNormParams p{};
  p.x = x; p.delta = delta; p.delta_weight = delta_weight; p.weight = weight; p.gate = gate;
  p.delta_rstd = const_cast<float*>(delta_rstd); p.rstd = const_cast<float*>(rstd); p.dsummed = dsummed; p.dnormed = dnormed;
  p.dx = dx; p.ddelta = ddelta; p.dgate = dgate; p.partial = partial; p.rows = rows; p.D = D; p.seq = seq;
  p.gate_kind = gate_kind; p.gate_f32 = gate_f32; p.residual_scale = residual_scale;
  return gated_norm(p, type, true, dw, dwd, s);
}

}  // extern "C"
