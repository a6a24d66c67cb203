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
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include <type_traits>

#include "chain.cuh"
#include "entries.h"
#include "ptx.cuh"

namespace b2 {

constexpr int GN_VECS = 2;                   // runs of 8 columns per lane
constexpr int GN_MAX_D = 8192;
constexpr int GN_MAX_ROWS = 0x7fffffff - 0xffff;      // 2^31 - 2^16: a CTA's count of rows goes up to the ring's length beyond the last one

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
  float* partial;            // [2][CTAs][D] column sums, then for GATE_SEQUENCE [CTAs + sequences][places][D]
  int* status;               // device word, non-zero: a wait ran out
  int rows, D, seq, places, gate_kind, gate_f32, aligned, stages, ctas_per_sm;
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

template <int W> constexpr int gn_threads() { return W > 8 ? W * 32 : 256; }
template <int W> constexpr int gn_rows() { return gn_threads<W>() / 32 / W; }        // rows a CTA works on at a time

// A CTA has a run of rows, at least one, which its slots (of W warps) take in turn.
__device__ __forceinline__ int gn_first_row(int cta, int rows, int ctas) { return cta * (rows / ctas) + min(cta, rows % ctas); }
__device__ __forceinline__ int gn_cta_of(int row, int rows, int ctas) {
  const int base = rows / ctas, longer = rows % ctas * (base + 1);          // the first ones have a row more
  return row < longer ? row / (base + 1) : rows % ctas + (row - longer) / base;
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

// ------------------------------------------------------------------ host side
static int gn_sms() {
  static int sms = 0;
  if (!sms) {
    int dev = 0;
    cudaGetDevice(&dev);
    cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
  }
  return sms;
}

static int gn_rows_at_once(int D) { return D <= 512 ? 8 : D <= 1024 ? 4 : D <= 2048 ? 2 : 1; }

// Sums of a sequence in a CTA, one for each of its slots, or as many as the sequence has rows (the next power of two), which lie in slots one
// after the other.
static int gn_places(int D, int seq) {
  const int R = gn_rows_at_once(D);
  int n = 1;
  while (n < R && n < seq) n *= 2;
  return n;
}

// CTAs of the backward kernels: ``per_sm`` of them, at least two blocks of rows each, so that the partial sums stay small beside the
// rows.
static int gn_bwd_ctas(int rows, int D, int per_sm) {
  const int R = gn_rows_at_once(D);
  const long long most = gn_sms() * static_cast<long long>(per_sm), wanted = (rows + 2LL * R - 1) / (2LL * R);
  return static_cast<int>(wanted < most ? wanted : most);
}

// Bytes of one stage of the ring, and how many stages fit beside the ``extra`` bytes: of 227 KiB per SM, less 1 KiB a CTA.
static uint32_t gn_stage_bytes(const GatedNormParams& p, int type, bool backward) {
  const uint32_t row = p.D * (type == 0 ? 4 : 2);
  return gn_rows_at_once(p.D) * ((backward ? 4 : 2) * row + (p.gate_kind == GATE_FULL ? (p.gate_f32 ? p.D * 4 : row) : 0));
}
static uint32_t gn_extra_bytes(const GatedNormParams& p, bool backward, int W) {
  // backward: w, and dw_d of a gate per sequence
  return backward ? (W > 8 ? W * 32 : 256) * GN_VECS * 8 * 4 * (p.gate_kind == GATE_SEQUENCE ? 2 : 1) : 0;
}
static int gn_stages_that_fit(const GatedNormParams& p, int type, bool backward, int W, int ctas_per_sm) {
  return ((ctas_per_sm == 1 ? 226 : 113) * 1024u - 600u - gn_extra_bytes(p, backward, W)) / gn_stage_bytes(p, type, backward);
}

// Warps of a row.  Ten or twelve are few enough for two CTAs per SM with their columns of the weights in registers, which hides one
// row's sums behind another's; sixteen take an SM.  Forward, 20011 x 5120: sixteen warps 169 us, ten 144 (gate per channel), 15000 x
// 6144: 131, twelve 128.  Backward, 18000 x 4608: 239, ten 207, but only where two stages of both CTAs fit (20011 x 5120 with a gate
// per element, one CTA of ten 370 us, of sixteen 323).
static int gn_width(const GatedNormParams& p, int type, bool backward) {
  if (p.D <= 4096) return 8 / gn_rows_at_once(p.D);
  if (p.D <= 5120 && (!backward || gn_stages_that_fit(p, type, true, 10, 2) >= 2)) return 10;
  return p.D <= 6144 && !backward ? 12 : 16;
}

// About 120 KB of rows on their way per SM fill the memory; more make it slower, as reads and writes spread over more DRAM pages
// (16384 x 4096 forward, gate per channel: 64 KB 109 us, 96 KB 96, 128 KB 103; 15000 x 6144 with a gate per element 144 KB 141,
// 216 KB 165; backward the same or 2 % less).  A CTA that has an SM to itself has two stages on their way beside the one in use
// (12000 x 8192 with a gate per element: two stages 201 us, three 158), but for the backward pass, whose rows take longer.
static int gn_stages(const GatedNormParams& p, int type, bool backward, int W, int ctas_per_sm) {
  const int fit = gn_stages_that_fit(p, type, backward, W, ctas_per_sm), most = fit < GN_RING ? fit : GN_RING;
  const int wanted = 120 * 1024u / (gn_stage_bytes(p, type, backward) * ctas_per_sm), least = ctas_per_sm == 1 && !backward ? 3 : 2;
  const int n = wanted < least ? least : wanted;
  return n < most ? n : most;
}

// Which form: a ring of two stages or more, aligned rows, and more blocks of rows than a CTA would have in one go.
template <int W>
static bool gn_takes_ring(GatedNormParams& p, int type, bool backward, uint32_t* smem) {
  // Two CTAs per SM; 512 threads take the registers of a whole SM, and two stages of very long rows its shared memory.
  p.ctas_per_sm = W == 16 || (W > 8 && gn_stages_that_fit(p, type, backward, W, 2) < 2) ? 1 : 2;
  p.stages = gn_stages(p, type, backward, W, p.ctas_per_sm);
  const long long blocks = (p.rows + gn_rows<W>() - 1LL) / gn_rows<W>(), resident = gn_sms() * static_cast<long long>(p.ctas_per_sm);
  *smem = p.stages * gn_stage_bytes(p, type, backward) + gn_extra_bytes(p, backward, W);
  return p.aligned && p.stages >= 2 && blocks >= 2 * resident;
}
template <auto KERNEL>
static cudaError_t gn_launch_ring(int ctas, int threads, uint32_t smem, cudaStream_t s, const GatedNormParams& p) {
  const cudaError_t r = allow_shared<KERNEL>(226 * 1024 - 600);      // the most that any width asks for
  return r != cudaSuccess ? r : launch_next(KERNEL, ctas, threads, smem, s, p);
}

// Checks and fills ``p`` up, then calls ``launch(type tag, width tag)``.
template <bool BACKWARD, typename Launch>
static int gated_norm(GatedNormParams& p, int type, Launch&& launch) {
  if (p.rows < 0 || p.rows > GN_MAX_ROWS || p.D < 1 || p.D > GN_MAX_D || type < 0 || type > 2 || p.gate_kind < 0 || p.gate_kind > 4 ||
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
  auto by_width = [&](auto tag) {
    const int width = gn_width(p, type, BACKWARD);
    if constexpr (!BACKWARD) {
      if (width == 12) return launch(tag, std::integral_constant<int, 12>());
    }
    switch (width) {
      case 1: return launch(tag, std::integral_constant<int, 1>());
      case 2: return launch(tag, std::integral_constant<int, 2>());
      case 4: return launch(tag, std::integral_constant<int, 4>());
      case 8: return launch(tag, std::integral_constant<int, 8>());
      case 10: return launch(tag, std::integral_constant<int, 10>());
      default: return launch(tag, std::integral_constant<int, 16>());
    }
  };
  const cudaError_t r = type == 0 ? by_width(float()) : type == 1 ? by_width(__nv_bfloat16()) : by_width(__half());
  if (r != cudaSuccess) cudaGetLastError();
  return r == cudaSuccess ? 0 : -1;
}

}  // namespace b2
