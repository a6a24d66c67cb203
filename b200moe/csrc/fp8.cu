// Products of 8-bit floating point values (e4m3) with one fp32 scale for each block of 128 along the reduction: activations
// have a scale per row and block, weights one per 128 x 128 values.
//
//   quantise   scale = max(largest / 448, 2^-120), value = x / scale rounded to e4m3 (448 is its largest number)
//   product    y[m, n] = sum over blocks b of  sa[m, b] sb[n / 128, b] * (sum over the 128 k of b of a[m, k] w[n, k])
//
// The data gradient dx = dy W takes the weight as it is stored: its rows are the reduction, so B is read along MN, and a
// 128 x 128 block has the same scale either way.
//
// Product.  The tensor cores add up one block of 128 (four instructions of 32) in an accumulator of its own; the warps of the
// epilogue multiply it by the two scales and add it to fp32 registers, while the next blocks are in flight: accumulators of
// 512 / BN blocks fit in tensor memory.  A tile of 128 x 256 has 128 sums per thread of eight warps.  A block of such a tile takes
// the tensor cores 512 cycles and the epilogue one fused multiply-add per value, 128 for each pair of lanes.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>
#include <stdint.h>

#include "chain.cuh"
#include "ptx.cuh"
#include "tensormap.cuh"

namespace b2 {

constexpr float E4M3_MAX = 448.f;
constexpr float SMALLEST_SCALE = 7.52316384526264e-37f;     // 2^-120
constexpr int F8_BM = 128, F8_BK = 128;
constexpr int F8_THREADS = 320;
constexpr int F8_GROUP_M = 8;
constexpr int F8_STAGING = 32 * 1024;

// ------------------------------------------------------------------ quantisation
enum QuantType : int { QUANT_F32 = 0, QUANT_BF16 = 1, QUANT_F16 = 2 };

// 8 values of a row from column ``col`` on, zeros behind the last column.
__device__ __forceinline__ void load8(const void* x, int type, long long at, int left, bool aligned, float (&f)[8]) {
  if (aligned && left >= 8) {
    if (type == QUANT_F32) {
      const float4* src = reinterpret_cast<const float4*>(static_cast<const float*>(x) + at);
      const float4 a = src[0], b = src[1];
      f[0] = a.x; f[1] = a.y; f[2] = a.z; f[3] = a.w; f[4] = b.x; f[5] = b.y; f[6] = b.z; f[7] = b.w;
    } else {
      const uint4 v = *reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(x) + at);
      const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float2 t = type == QUANT_BF16 ? __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&w[i]))
                                            : __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
        f[2 * i] = t.x;
        f[2 * i + 1] = t.y;
      }
    }
    return;
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    f[i] = 0.f;
    if (i < left) {
      if (type == QUANT_F32) f[i] = static_cast<const float*>(x)[at + i];
      else if (type == QUANT_BF16) f[i] = __bfloat162float(static_cast<const __nv_bfloat16*>(x)[at + i]);
      else f[i] = __half2float(static_cast<const __half*>(x)[at + i]);
    }
  }
}

// Values behind ``left`` are zero and stored too where they belong to the row's pitch.
__device__ __forceinline__ void store8(uint8_t* q, float scale, const float (&f)[8]) {
  uint32_t w[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const __nv_fp8x2_storage_t a = __nv_cvt_float2_to_fp8x2(make_float2(f[4 * i] / scale, f[4 * i + 1] / scale), __NV_SATFINITE, __NV_E4M3);
    const __nv_fp8x2_storage_t b = __nv_cvt_float2_to_fp8x2(make_float2(f[4 * i + 2] / scale, f[4 * i + 3] / scale), __NV_SATFINITE, __NV_E4M3);
    w[i] = static_cast<uint32_t>(a) | static_cast<uint32_t>(b) << 16;
  }
  *reinterpret_cast<uint2*>(q) = make_uint2(w[0], w[1]);
}

// NaN is passed over here; its value stays NaN.  Infinity makes the scale infinite and its own value NaN.
__device__ __forceinline__ float largest8(const float (&f)[8]) {
  float m = 0.f;
#pragma unroll
  for (int i = 0; i < 8; ++i) m = fmaxf(m, fabsf(f[i]));
  return m;
}

// One scale for 128 values of a row: half a warp per block, 8 values a lane.  ``pitch`` is a multiple of 16 and the row is filled with
// zeros up to it.  Bound by memory traffic.
__global__ void __launch_bounds__(256) quantize_rows_kernel(const void* __restrict__ x, int type, uint8_t* __restrict__ q,
                                                            float* __restrict__ scales, long long M, int K, long long ldx,
                                                            long long pitch, long long scale_pitch, int aligned) {
  chain_begin();
  const int lane16 = threadIdx.x & 15;
  const long long blocks = (K + 127) / 128, total = M * blocks;
  for (long long b = (static_cast<long long>(blockIdx.x) * 256 + threadIdx.x) >> 4; b < total;
       b += static_cast<long long>(gridDim.x) * 16) {
    const long long row = b / blocks;
    const int kb = static_cast<int>(b - row * blocks), col = kb * 128 + lane16 * 8;
    float f[8];
    load8(x, type, row * ldx + col, K - col, aligned, f);
    float m = largest8(f);
    const unsigned mask = 0xffffu << (threadIdx.x & 16);
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(mask, m, o));
    const float scale = fmaxf(m / E4M3_MAX, SMALLEST_SCALE);
    if (col < pitch) store8(q + row * pitch + col, scale, f);
    if (lane16 == 0) scales[kb * scale_pitch + row] = scale;
  }
}

// One scale for 128 x 128 values: a CTA per block, 64 values a thread.
__global__ void __launch_bounds__(256) quantize_blocks_kernel(const void* __restrict__ x, int type, uint8_t* __restrict__ q,
                                                              float* __restrict__ scales, int M, int K, long long ldx,
                                                              long long pitch, int aligned) {
  chain_begin();
  __shared__ float most[8];
  const int kb = blockIdx.x, lane16 = threadIdx.x & 15, col = kb * 128 + lane16 * 8;
  for (long long mb = blockIdx.y; mb * 128 < M; mb += gridDim.y) {
    const long long row0 = mb * 128 + (threadIdx.x >> 4);
    float f[8][8], m = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const long long row = row0 + i * 16;
      load8(x, type, row * ldx + col, row < M ? K - col : 0, aligned, f[i]);
      m = fmaxf(m, largest8(f[i]));
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
    __syncthreads();
    if ((threadIdx.x & 31) == 0) most[threadIdx.x >> 5] = m;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 8; ++i) m = fmaxf(m, most[i]);
    const float scale = fmaxf(m / E4M3_MAX, SMALLEST_SCALE);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const long long row = row0 + i * 16;
      if (row < M && col < pitch) store8(q + row * pitch + col, scale, f[i]);
    }
    if (threadIdx.x == 0) scales[mb * gridDim.x + kb] = scale;
  }
}

// ------------------------------------------------------------------ product
struct Fp8Params {
  CUtensorMap map_a;         // [M, K], box 128 x 128
  CUtensorMap map_b;         // NT: [N, K], box BN x 128; NN: [K, N], boxes of 128 rows x 128 columns
  const float* a_scales;     // [M, K / 128] with these strides
  const float* b_scales;     // [N / 128, K / 128] with these strides
  long long a_row, a_block, b_row, b_block;
  __nv_bfloat16* d;          // [M, N]
  int M, N, K;
  int* status;
};

template <int BN> struct F8Cfg {
  static constexpr int STAGES = BN == 256 ? 4 : BN == 128 ? 6 : 8;
  static constexpr int A_BYTES = F8_BM * F8_BK, B_BYTES = BN * F8_BK, STAGE_BYTES = A_BYTES + B_BYTES;
  static constexpr int SLOTS = 512 / BN < 4 ? 512 / BN : 4;      // accumulators in tensor memory
  static constexpr int SMEM = STAGES * STAGE_BYTES + F8_STAGING + 1024 + 256;
};

// d += s * v for two values at a time.
__device__ __forceinline__ void fma2(uint64_t& d, uint32_t lo, uint32_t hi, uint64_t s) {
  uint64_t v;
  asm("mov.b64 %0, {%1, %2};" : "=l"(v) : "r"(lo), "r"(hi));
  asm("fma.rn.f32x2 %0, %1, %2, %0;" : "+l"(d) : "l"(v), "l"(s));
}
__device__ __forceinline__ void split2(uint64_t d, float& lo, float& hi) {
  uint32_t a, b;
  asm("mov.b64 {%0, %1}, %2;" : "=r"(a), "=r"(b) : "l"(d));
  lo = __uint_as_float(a);
  hi = __uint_as_float(b);
}

// SPLIT: the CTAs of a cluster share a tile, each has a run of its blocks along k; their sums meet in the order of the CTAs through
// the cluster's shared memory.
template <int BN, int B_MN, int SPLIT>
__global__ void __launch_bounds__(F8_THREADS, 1) gemm_fp8_kernel(const __grid_constant__ Fp8Params p) {
  using C = F8Cfg<BN>;
  constexpr int STAGES = C::STAGES, SLOTS = C::SLOTS, COLS = BN / 2;      // columns of an epilogue warp
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* full_bar = reinterpret_cast<uint64_t*>(smem + STAGES * C::STAGE_BYTES + F8_STAGING);
  uint64_t* empty_bar = full_bar + STAGES;
  uint64_t* tmem_full = empty_bar + STAGES;
  uint64_t* tmem_empty = tmem_full + SLOTS;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(tmem_empty + SLOTS);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(&full_bar[s], 1);
      mbar_init(&empty_bar[s], 1);
    }
    for (int s = 0; s < SLOTS; ++s) {
      mbar_init(&tmem_full[s], 1);
      mbar_init(&tmem_empty[s], 8);
    }
    *abort_flag = 0;
    mbar_fence_init();
    tma_prefetch_desc(&p.map_a);
    tma_prefetch_desc(&p.map_b);
  }
  if (warp == 1) {
    tmem_alloc(tmem_slot, 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  chain_begin();
  const int m_tiles = (p.M + F8_BM - 1) / F8_BM, n_tiles = (p.N + BN - 1) / BN, all_blocks = (p.K + F8_BK - 1) / F8_BK;
  const int parts = SPLIT ? SPLIT : 1, part = SPLIT ? static_cast<int>(cluster_ctarank()) : 0;
  const long long tiles = static_cast<long long>(m_tiles) * n_tiles;
  const long long worker = blockIdx.x / parts, workers = gridDim.x / parts;
  const int kb_begin = static_cast<int>(static_cast<long long>(all_blocks) * part / parts);
  const int kb_end = static_cast<int>(static_cast<long long>(all_blocks) * (part + 1) / parts);
  auto place = [&](long long tile, int& m0, int& n0) {
    const long long per_group = static_cast<long long>(F8_GROUP_M) * n_tiles;
    const int group = static_cast<int>(tile / per_group), first = group * F8_GROUP_M;
    const int in_group = static_cast<int>(tile - group * per_group), rows = min(F8_GROUP_M, m_tiles - first);
    m0 = (first + in_group % rows) * F8_BM;
    n0 = in_group / rows * BN;
  };

  if (warp == 0) {
    // ------------------------------------------------------------ TMA producer
    if (elect_one()) {
      int stage = 0;
      uint32_t phase = 0;
      bool wrapped = false;
      for (long long tile = worker; tile < tiles && !*abort_flag; tile += workers) {
        int m0, n0;
        place(tile, m0, n0);
        for (int kb = kb_begin; kb < kb_end; ++kb) {
          if (!mbar_wait(&empty_bar[stage], phase ^ 1)) {
            *abort_flag = 1;
            atomicExch(p.status, 1);
            break;
          }
          uint8_t* sa = smem + stage * C::STAGE_BYTES;
          uint8_t* sb = sa + C::A_BYTES;
          mbar_expect_tx(&full_bar[stage], C::STAGE_BYTES);
          tma_load_2d(sa, &p.map_a, &full_bar[stage], kb * F8_BK, m0);
          if (B_MN) {
#pragma unroll
            for (int c = 0; c < BN / 128; ++c) tma_load_2d(sb + c * 16384, &p.map_b, &full_bar[stage], n0 + c * 128, kb * F8_BK);
          } else {
            tma_load_2d(sb, &p.map_b, &full_bar[stage], kb * F8_BK, n0);
          }
          if (++stage == STAGES) {
            stage = 0;
            phase ^= 1;
            wrapped = true;
          }
        }
      }
      // a CTA that gives up waits (with a limit) for its copies before its shared memory goes to another one
      if (*abort_flag) {
        for (int s = 0; s < STAGES; ++s)
          if (wrapped || s < stage) mbar_wait(&full_bar[s], s < stage ? phase : phase ^ 1);
      }
    }
  } else if (warp == 1) {
    // ------------------------------------------------------------ MMA issuer
    if (elect_one()) {
      constexpr uint32_t idesc = umma_idesc_e4m3(F8_BM, BN, B_MN);
      int stage = 0, slot = 0;
      uint32_t phase = 0, slot_phase = 0;
      for (long long tile = worker; tile < tiles && !*abort_flag; tile += workers) {
        for (int kb = kb_begin; kb < kb_end; ++kb) {
          if (!mbar_wait(&tmem_empty[slot], slot_phase ^ 1) || !mbar_wait(&full_bar[stage], phase)) {
            *abort_flag = 1;
            atomicExch(p.status, 2);
            break;
          }
          tc_fence_after();
          const uint32_t sa = smem_u32(smem + stage * C::STAGE_BYTES), sb = sa + C::A_BYTES;
#pragma unroll
          for (int k = 0; k < F8_BK / 32; ++k) {
            const uint64_t da = umma_smem_desc(sa + k * 32, 16, 1024);
            const uint64_t db = B_MN ? umma_smem_desc(sb + k * 4096, 16384, 1024) : umma_smem_desc(sb + k * 32, 16, 1024);
            umma_f8_ss(tmem_base + slot * BN, da, db, idesc, k != 0);
          }
          umma_commit(&empty_bar[stage]);
          umma_commit(&tmem_full[slot]);
          if (++stage == STAGES) {
            stage = 0;
            phase ^= 1;
          }
          if (++slot == SLOTS) {
            slot = 0;
            slot_phase ^= 1;
          }
        }
      }
    }
  } else {
    // ------------------------------------------------------------ scales, sums and stores (eight warps)
    const int quad = warp & 3, half = (warp - 2) >> 2;       // TMEM lanes and column half of this warp
    uint4* const staged = reinterpret_cast<uint4*>(smem + STAGES * C::STAGE_BYTES) + (warp - 2) * 256;
    auto swz = [](int r) { return (r & 1) | ((r & 2) << 1) | ((r & 4) >> 1); };
    int slot = 0;
    uint32_t slot_phase = 0;
    const bool vectors = p.N % 8 == 0;
    for (long long tile = worker; tile < tiles && !*abort_flag; tile += workers) {
      int m0, n0;
      place(tile, m0, n0);
      const int row = m0 + quad * 32 + lane;
      const float* a_scale = p.a_scales + min(row, p.M - 1) * p.a_row;
      // a column half behind the last column has no scale; its sums are not stored
      const float* b_scale = p.b_scales + (min(n0 + half * COLS, p.N - 1) / 128) * p.b_row;
      uint64_t acc[COLS / 2];
#pragma unroll
      for (int i = 0; i < COLS / 2; ++i) acc[i] = 0;
      float sa = 0.f, sb = 0.f;
      if (kb_begin < kb_end) {
        sa = a_scale[kb_begin * p.a_block];
        sb = b_scale[kb_begin * p.b_block];
      }
      for (int kb = kb_begin; kb < kb_end; ++kb) {
        const float s = sa * sb;
        if (kb + 1 < kb_end) {
          sa = a_scale[(kb + 1) * p.a_block];
          sb = b_scale[(kb + 1) * p.b_block];
        }
        uint64_t s2;
        asm("mov.b64 %0, {%1, %1};" : "=l"(s2) : "r"(__float_as_uint(s)));
        if (!mbar_wait(&tmem_full[slot], slot_phase)) {
          *abort_flag = 1;
          atomicExch(p.status, 4);
          break;
        }
        tc_fence_after();
        const uint32_t taddr = tmem_base + slot * BN + half * COLS + (static_cast<uint32_t>(quad * 32) << 16);
        uint32_t v[2][16];
        tmem_ld_32x16(taddr, v[0]);
#pragma unroll
        for (int c = 0; c < COLS / 16; ++c) {
          tmem_ld_wait();
          if (c + 1 < COLS / 16) tmem_ld_32x16(taddr + (c + 1) * 16, v[(c + 1) & 1]);
          else {
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&tmem_empty[slot]);
          }
#pragma unroll
          for (int i = 0; i < 8; ++i) fma2(acc[c * 8 + i], v[c & 1][2 * i], v[c & 1][2 * i + 1], s2);
        }
        if (++slot == SLOTS) {
          slot = 0;
          slot_phase ^= 1;
        }
      }
      if (SPLIT) {
        // [column][row] of this CTA's part, in the shared memory of its operands, which have been read
        float* mine = reinterpret_cast<float*>(smem);
#pragma unroll
        for (int i = 0; i < COLS / 2; ++i) {
          float lo, hi;
          split2(acc[i], lo, hi);
          mine[(half * COLS + 2 * i) * F8_BM + quad * 32 + lane] = lo;
          mine[(half * COLS + 2 * i + 1) * F8_BM + quad * 32 + lane] = hi;
        }
        break;                                       // one tile per cluster
      }
      // 64 columns of 32 rows at a time through shared memory, so that a row leaves in 128 contiguous bytes
#pragma unroll
      for (int c = 0; c < COLS; c += 64) {
        const int col0 = n0 + half * COLS + c;
        if (col0 >= p.N) break;
        constexpr int WIDE = COLS < 64 ? COLS : 64;
#pragma unroll
        for (int i = 0; i < WIDE / 8; ++i) {
          uint32_t w[4];
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            float lo, hi;
            split2(acc[c / 2 + i * 4 + k], lo, hi);
            w[k] = pack_bf16(lo, hi);
          }
          staged[lane * 8 + (i ^ swz(lane))] = make_uint4(w[0], w[1], w[2], w[3]);
        }
        __syncwarp();
        const int unit = lane & 7, col = col0 + unit * 8;
#pragma unroll
        for (int it = 0; it < 8; ++it) {
          const int r = it * 4 + (lane >> 3), out_row = m0 + quad * 32 + r;
          if (out_row >= p.M || unit * 8 >= WIDE || col >= p.N) continue;
          const uint4 v = staged[r * 8 + (unit ^ swz(r))];
          __nv_bfloat16* dst = p.d + static_cast<long long>(out_row) * p.N + col;
          if (vectors) {
            *reinterpret_cast<uint4*>(dst) = v;
          } else {
            const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
            for (int k = 0; k < 8; ++k)
              if (col + k < p.N) dst[k] = __ushort_as_bfloat16(static_cast<unsigned short>(w[k >> 1] >> (16 * (k & 1))));
          }
        }
        __syncwarp();
      }
    }
  }
  if (SPLIT) {
    __syncwarp();
    cluster_sync_all();
    int m0, n0;
    place(worker, m0, n0);
    // this CTA's share of the columns; consecutive threads hold consecutive rows
    constexpr int SHARE = BN / (SPLIT ? SPLIT : 1);
    const bool bad = *abort_flag != 0;
    for (int i = threadIdx.x; i < F8_BM * (SHARE / 2) && !bad; i += F8_THREADS) {
      const int r = i % F8_BM, c = part * SHARE + i / F8_BM * 2;
      if (m0 + r >= p.M || n0 + c >= p.N) continue;
      float sum[2] = {0.f, 0.f};
#pragma unroll
      for (int k = 0; k < parts; ++k) {
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          float v;
          const uint32_t at = mapa_u32(smem_u32(reinterpret_cast<float*>(smem) + (c + j) * F8_BM + r), k);
          asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(at) : "memory");
          sum[j] += v;
        }
      }
      __nv_bfloat16* dst = p.d + static_cast<long long>(m0 + r) * p.N + n0 + c;
      dst[0] = __float2bfloat16(sum[0]);
      if (n0 + c + 1 < p.N) dst[1] = __float2bfloat16(sum[1]);
    }
    cluster_sync_all();                              // the others have read this CTA's part
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 1) tmem_dealloc(tmem_base, 512);
}

static int f8_sms() {
  static int sms = 0;
  if (!sms) {
    int dev = 0;
    cudaGetDevice(&dev);
    cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
  }
  return sms;
}

template <int BN, int B_MN, int SPLIT>
static int launch_fp8(const Fp8Params& p, cudaStream_t s) {
  auto kernel = gemm_fp8_kernel<BN, B_MN, SPLIT>;
  static bool set = false;
  if (!set) {
    if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, F8Cfg<BN>::SMEM) != cudaSuccess) return -3;
    set = true;
  }
  const long long tiles = static_cast<long long>((p.M + F8_BM - 1) / F8_BM) * ((p.N + BN - 1) / BN);
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = SPLIT ? SPLIT : 1;
  attr[1].val.clusterDim.y = 1;
  attr[1].val.clusterDim.z = 1;
  cfg.gridDim = dim3(static_cast<unsigned>(SPLIT ? tiles * SPLIT : tiles < f8_sms() ? tiles : f8_sms()));
  cfg.blockDim = dim3(F8_THREADS);
  cfg.dynamicSmemBytes = F8Cfg<BN>::SMEM;
  cfg.stream = s;
  cfg.attrs = attr;
  cfg.numAttrs = SPLIT ? 2 : 1;
  if (cudaLaunchKernelEx(&cfg, kernel, p) != cudaSuccess) {
    cudaGetLastError();
    return -1;
  }
  return 0;
}

}  // namespace b2

using namespace b2;

extern "C" {

// x [M, K] (type 0 fp32, 1 bf16, 2 fp16; row pitch ldx) -> e4m3 values [M, pitch], zeros from column K on, and fp32 scales:
// block_rows 1: [ceil(K / 128), scale_pitch], the scale of row m in column m; 128: [ceil(M / 128), ceil(K / 128)].
int b2_quantize_fp8(const void* x, int type, void* q, float* scales, long long M, int K, long long ldx, long long pitch,
                    long long scale_pitch, int block_rows, cudaStream_t s) {
  if (M < 0 || M > 0x7fffffff || K < 1 || pitch < K || pitch % 16 || pitch - K >= 128 || type < 0 || type > 2 ||
      (block_rows != 1 && block_rows != 128))
    return -10;
  if (M == 0) return 0;
  const int size = type == QUANT_F32 ? 4 : 2;
  const int aligned = ldx * size % 16 == 0 && reinterpret_cast<uintptr_t>(x) % 16 == 0;
  cudaError_t r;
  if (block_rows == 1) {
    const long long ctas = (M * ((K + 127) / 128) + 15) / 16, most = f8_sms() * 8LL;
    r = launch_next(quantize_rows_kernel, static_cast<unsigned>(ctas < most ? ctas : most), 256, 0, s, x, type,
                    static_cast<uint8_t*>(q), scales, M, K, ldx, pitch, scale_pitch, aligned);
  } else {
    const long long rows = (M + 127) / 128;
    r = launch_next(quantize_blocks_kernel, dim3((K + 127) / 128, static_cast<unsigned>(rows < 32768 ? rows : 32768)), 256, 0, s, x,
                    type, static_cast<uint8_t*>(q), scales, static_cast<int>(M), K, ldx, pitch, aligned);
  }
  if (r != cudaSuccess) cudaGetLastError();
  return r == cudaSuccess ? 0 : -1;
}

// d[M, N] bf16 = a[M, K] * w[N, K]^T (nn 0) or a[M, K] * w[K, N] (nn 1), e4m3 values with row pitches lda, ldw (multiples of 16) and
// their scales; b_row, b_block: strides of w's scales along n and along k.
int b2_gemm_fp8(const void* a, const float* a_scales, const void* w, const float* b_scales, void* d, int M, int N, int K,
                long long lda, long long ldw, long long a_row, long long a_block, long long b_row, long long b_block, int nn,
                int* status, cudaStream_t s) {
  if (M < 0 || N < 1 || K < 1 || lda % 16 || ldw % 16) return -10;
  if (M == 0) return 0;
  Fp8Params p{};
  p.a_scales = a_scales; p.b_scales = b_scales; p.a_row = a_row; p.a_block = a_block; p.b_row = b_row; p.b_block = b_block;
  p.d = static_cast<__nv_bfloat16*>(d); p.M = M; p.N = N; p.K = K; p.status = status;
  if (make_map8(&p.map_a, a, K, M, lda, F8_BM)) return -11;
  const int bn = 256;
  if (nn ? make_map8(&p.map_b, w, N, K, ldw, 128) : make_map8(&p.map_b, w, K, N, ldw, bn)) return -12;
  return nn ? launch_fp8<256, 1, 0>(p, s) : launch_fp8<256, 0, 0>(p, s);
}

}  // extern "C"
