// The gated residual norm forward: see gated_norm.cuh.
#include "gated_norm.cuh"

namespace b2 {

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

// One barrier per row: the sum over delta of the next row is formed before the sum over s of the present one, and both cross the
// warps together.  TB/s of the tensors, gate per channel: 5.7 at 16384 x 4096, 5.3 at 131072 x 512; with a gate per element 6.2 at
// 20011 x 5120 and at 12000 x 8192.  Streaming stores gave nothing.
template <typename T, int W, int G>
__global__ void __launch_bounds__(gn_threads<W>(), W == 16 ? 1 : 2) gated_norm_fwd_ring_kernel(const GatedNormParams p) {
  chain_begin();
  constexpr int R = gn_rows<W>(), V = GN_VECS;
  extern __shared__ __align__(128) uint8_t gn_smem[];
  __shared__ uint64_t bars[R][GN_RING];
  __shared__ float2 scratch[2][R][W];
  gn_init(bars[0], R * GN_RING);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, slot = warp / W, in_row = warp % W, D = p.D;
  const uint32_t row_bytes = D * sizeof(T), gate_bytes = p.gate_f32 ? D * 4 : row_bytes;
  const uint32_t slot_bytes = 2 * row_bytes + (G == GATE_FULL ? gate_bytes : 0), stage_bytes = R * slot_bytes;
  // a run of rows for each CTA where a sequence's gate is loaded, or all CTAs side by side: neighbouring rows are in one DRAM page
  constexpr bool RUNS = G == GATE_SEQUENCE;
  const int begin = RUNS ? gn_first_row(blockIdx.x, p.rows, gridDim.x) : static_cast<int>(blockIdx.x) * R;
  const int end = RUNS ? gn_first_row(blockIdx.x + 1, p.rows, gridDim.x) : p.rows;
  const int step = RUNS ? R : static_cast<int>(gridDim.x) * R;
  const uint8_t* const mine = gn_smem + slot * slot_bytes;
  const GnRing<3> ring = {{static_cast<const uint8_t*>(p.x), static_cast<const uint8_t*>(p.delta),
                           G == GATE_FULL ? static_cast<const uint8_t*>(p.gate) : nullptr},
                          {row_bytes, row_bytes, gate_bytes}, gn_smem + slot * slot_bytes, stage_bytes, p.stages, bars[slot],
                          begin + slot, step, end};
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
  for (int row = begin + slot; row < end; row += step, ++turn, half ^= 1) {
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
    if (row + step < end) {
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

template <typename T, int W>
static cudaError_t gn_forward(GatedNormParams& p, int type, cudaStream_t s) {
  constexpr int R = gn_rows<W>(), THREADS = gn_threads<W>();
  uint32_t smem;
  if (gn_takes_ring<W>(p, type, false, &smem)) {
    const int ctas = gn_sms() * p.ctas_per_sm;
    switch (p.gate_kind) {
      case GATE_NONE:                // as a gate per channel of ones
      case GATE_CHANNEL: return gn_launch_ring<gated_norm_fwd_ring_kernel<T, W, GATE_CHANNEL>>(ctas, THREADS, smem, s, p);
      case GATE_SEQUENCE: return gn_launch_ring<gated_norm_fwd_ring_kernel<T, W, GATE_SEQUENCE>>(ctas, THREADS, smem, s, p);
      case GATE_TOKEN: return gn_launch_ring<gated_norm_fwd_ring_kernel<T, W, GATE_TOKEN>>(ctas, THREADS, smem, s, p);
      default: return gn_launch_ring<gated_norm_fwd_ring_kernel<T, W, GATE_FULL>>(ctas, THREADS, smem, s, p);
    }
  }
  const long long blocks = (p.rows + R - 1LL) / R, most = gn_sms() * (W > 8 ? 4LL : 8LL);
  return launch_next(gated_norm_fwd_kernel<T, W>, static_cast<unsigned>(blocks < most ? blocks : most), THREADS, 0, s, p);
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
  return gated_norm<false>(p, type, [&](auto tag, auto width) { return gn_forward<decltype(tag), decltype(width)::value>(p, type, s); });
}

}  // extern "C"
