// The gated residual norm backward: see gated_norm.cuh.
#include "gated_norm.cuh"

namespace b2 {

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
// is stored wherever the sequence changes, in place ``sequence + CTA`` and slot (of as many as the sequence can use), which no other has.
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
      float* dst = sequences + (static_cast<long long>(row / p.seq + blockIdx.x) * p.places + (slot & p.places - 1)) * D;
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

// A value that a second phase needs again is formed again from the row in shared memory: two CTAs per SM leave 112 registers, of
// which the column sums and g w_d take 48 (96 registers with ten warps a row, where 20 to 56 bytes are spilled).  w is read from
// shared memory, and so is dw_d for a gate per sequence, which is touched once per sequence.  TB/s of the tensors, gate per channel:
// 5.8 at 16384 x 4096, 5.1 at 20011 x 5120, 5.2 at 131072 x 512; 6.0 at 16384 x 4096 with a gate per element.
template <typename T, int W, int G>
__global__ void __launch_bounds__(gn_threads<W>(), W == 16 ? 1 : 2) gated_norm_bwd_ring_kernel(const GatedNormParams p) {
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
      float* dst = sequences + (static_cast<long long>(sequence + blockIdx.x) * p.places + (slot & p.places - 1)) * D;
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
__global__ void __launch_bounds__(512) gated_norm_sums_kernel(const GatedNormParams p, int ctas, int gate_bf16,
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
      const float* src = p.partial + (2LL * ctas + static_cast<long long>(i) * p.places) * D + col;
      const int shift = 31 - __clz(p.places);                           // a power of two
      for (int r = (first << shift) + threadIdx.y; r < last << shift; r += 16) {
        // a slot that had none of the sequence's rows in this CTA has stored nothing
        const int cta = r >> shift, begin = cta * base + min(cta, extra), end = begin + base + (cta < extra);
        const int from = max(low, begin), rows = min(high, end) - from;
        if ((r - (from - begin) & p.places - 1) < rows) add(sum, src + static_cast<long long>(r) * D);
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

template <typename T, int W>
static cudaError_t gn_backward(GatedNormParams& p, int type, float* dw, float* dwd, cudaStream_t s) {
  constexpr int THREADS = gn_threads<W>();
  const int ctas = gn_bwd_ctas(p.rows, p.D, W == 16 ? 1 : 2), gate_bf16 = type == 1;
  uint32_t smem;
  cudaError_t r;
  if (gn_takes_ring<W>(p, type, true, &smem)) {
    switch (p.gate_kind) {
      case GATE_NONE:
      case GATE_CHANNEL: r = gn_launch_ring<gated_norm_bwd_ring_kernel<T, W, GATE_CHANNEL>>(ctas, THREADS, smem, s, p); break;
      case GATE_SEQUENCE: r = gn_launch_ring<gated_norm_bwd_ring_kernel<T, W, GATE_SEQUENCE>>(ctas, THREADS, smem, s, p); break;
      case GATE_TOKEN: r = gn_launch_ring<gated_norm_bwd_ring_kernel<T, W, GATE_TOKEN>>(ctas, THREADS, smem, s, p); break;
      default: r = gn_launch_ring<gated_norm_bwd_ring_kernel<T, W, GATE_FULL>>(ctas, THREADS, smem, s, p);
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
    return launch_next(gated_norm_sums_kernel<4>, dim3((p.D + 127) / 128, y), dim3(32, 16), 0, s, p, ctas, gate_bf16, dw, dwd, p.dgate);
  return launch_next(gated_norm_sums_kernel<1>, dim3((p.D + 31) / 32, y), dim3(32, 16), 0, s, p, ctas, gate_bf16, dw, dwd, p.dgate);
}

}  // namespace b2

using namespace b2;

extern "C" {

// Floats of the workspace of the backward pass (at most: which CTAs it takes goes by the type too).
long long b2_gated_norm_bwd_floats(int rows, int D, int seq, int gate_kind) {
  if (rows < 1 || D < 1 || D > GN_MAX_D || (gate_kind == GATE_SEQUENCE && seq < 1)) return 0;
  const long long ctas = gn_bwd_ctas(rows, D, D <= 5120 ? 2 : 1);
  return (2 * ctas + (gate_kind == GATE_SEQUENCE ? (ctas + rows / seq) * gn_places(D, seq) : 0)) * D;
}

// Gradients; dsummed and dnormed may be null (zero).  dgate has the gate's shape and type; dw, dwd fp32 [D].
int b2_gated_norm_bwd(const void* dsummed, const void* dnormed, const void* x, const void* delta, const float* delta_weight,
                      const float* weight, const void* gate, const float* delta_rstd, const float* rstd, void* dx, void* ddelta,
                      float* dwd, float* dw, void* dgate, float* partial, int rows, int D, int seq, int type, int gate_kind,
                      int gate_f32, float residual_scale, int* status, cudaStream_t s) {
  GatedNormParams p{};
  p.x = x; p.delta = delta; p.delta_weight = delta_weight; p.weight = weight; p.gate = gate;
  p.delta_rstd = const_cast<float*>(delta_rstd); p.rstd = const_cast<float*>(rstd); p.dsummed = dsummed; p.dnormed = dnormed;
  p.dx = dx; p.ddelta = ddelta; p.dgate = dgate; p.partial = partial; p.rows = rows; p.D = D; p.seq = seq; p.places = gn_places(D, seq);
  p.gate_kind = gate_kind; p.gate_f32 = gate_f32; p.residual_scale = residual_scale; p.status = status;
  return gated_norm<true>(p, type, [&](auto tag, auto width) { return gn_backward<decltype(tag), decltype(width)::value>(p, type, dw, dwd, s); });
}

}  // extern "C"
