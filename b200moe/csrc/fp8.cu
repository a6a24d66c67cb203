// Products of 8-bit floating point values (e4m3) with one fp32 scale for each block of 128 along the reduction: activations
// have a scale per row and block, weights one per 128 x 128 values.
//
//   quantise   scale = max(largest / 448, 2^-120), value = x / scale rounded to e4m3 (448 is its largest number)
//   product    y[m, n] = sum over blocks b of  sa[m, b] sb[n / 128, b] * (sum over the 128 k of b of a[m, k] w[n, k])
//
// The two scales are multiplied first: results below 2^-102, whose product of scales may be subnormal, lose bits.
//
// The data gradient dx = dy W takes the weight as it is stored: its rows are the reduction, so B is read along MN, and a
// 128 x 128 block has the same scale either way.
//
// Product.  The tensor cores add up one block of 128 (four instructions of 32) in an accumulator of its own; the warps of the
// epilogue multiply it by the two scales, which two warps form ahead, and add it to fp32 registers, while the next blocks are in
// flight: accumulators of 512 / BN blocks fit in tensor memory.  A block of a 128 x 256 tile is 768 cycles of shared memory (48 KiB
// written by TMA and read by the tensor cores, which would need 512), and one fused multiply-add per value, 256 issue slots of each
// scheduler.  16384 x 6144, K 4096 takes 413 us in a launch by itself (2.0 PFLOP/s, bf16 520 us) and 482 in a loop, against the power limit
// at 1.5 GHz.  The tensor cores are busy half of the cycles either way, and no unit is near its limit: what waits is the epilogue, which
// loads columns, waits for them and adds them in turn (without the additions 320 us, three quarters of the cycles).  Pairs of CTAs
// (cta_group::2), which halve the traffic of B, were slower (616 us): an accumulator goes back and forth between two CTAs for every block.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>
#include <stdint.h>

#include "chain.cuh"
#include "entries.h"
#include "ptx.cuh"
#include "tensormap.cuh"

namespace b2 {

constexpr float E4M3_MAX = 448.f;
constexpr float SMALLEST_SCALE = 0x1p-120f;
constexpr int F8_BM = 128, F8_BK = 128;
constexpr int F8_EPI_WARPS = 8, F8_THREADS = 128 + 32 * F8_EPI_WARPS;
// Registers: 384 threads x 168 at launch and at the end, 128 x 72 + 256 x 216 in between.
constexpr int F8_EVEN = 168, F8_FEW = 72, F8_MANY = 216;
constexpr int F8_GROUP_M = 8;
constexpr int F8_AHEAD = 4;
constexpr int F8_STAGING = F8_EPI_WARPS * 2048;
constexpr int F8_MAX = 0x7fffffff - 255;       // rows and columns: their counts are rounded up to whole tiles

// ------------------------------------------------------------------ quantisation
enum QuantType : int { QUANT_F32 = 0, QUANT_BF16 = 1, QUANT_F16 = 2 };

template <typename T> __device__ __forceinline__ float quant_f32(T v);
template <> __device__ __forceinline__ float quant_f32(float v) { return v; }
template <> __device__ __forceinline__ float quant_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
template <> __device__ __forceinline__ float quant_f32(__half v) { return __half2float(v); }

// 8 values of a row from ``x`` on, zeros behind the ``left`` that there are; as they are stored, which takes fewer registers.
template <typename T>
struct Values8 {
  alignas(16) T v[8];
  __device__ __forceinline__ void load(const T* x, int left, bool aligned) {
    if (aligned && left >= 8) {
#pragma unroll
      for (int i = 0; i < static_cast<int>(sizeof(v) / 16); ++i) reinterpret_cast<uint4*>(v)[i] = reinterpret_cast<const uint4*>(x)[i];
      return;
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = i < left ? x[i] : T(0.f);
  }
  __device__ __forceinline__ void get(float (&f)[8]) const {
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] = quant_f32<T>(v[i]);
  }
};

// x / scale of a block, correctly rounded: a product with the rounded reciprocal and one correction by its remainder (P. Markstein,
// "Computation of elementary functions on the IBM RISC System/6000 processor", 1990), three operations a value where a
// division is about ten.  Scales that are infinite, or so small that a remainder would underflow, are divided by.
struct BlockScale {
  float scale, inverse;
  bool plain;
};
__device__ __forceinline__ BlockScale block_scale(float most) {
  BlockScale s;
  s.scale = fmaxf(most / E4M3_MAX, SMALLEST_SCALE);
  s.inverse = 1.f / s.scale;
  s.plain = !(s.scale > 1e-29f && s.scale < 1e36f);
  return s;
}
__device__ __forceinline__ float scaled(float x, const BlockScale& s) {
  const float first = x * s.inverse;
  return __fmaf_rn(__fmaf_rn(-first, s.scale, x), s.inverse, first);
}
// Values behind the last column are zero and stored too where they belong to the row's pitch.
template <typename T>
__device__ __forceinline__ void store8(uint8_t* q, const BlockScale& s, const Values8<T>& x) {
  float v[8], f[8];
  x.get(f);
  if (s.plain) {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = f[i] / s.scale;
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = scaled(f[i], s);
  }
  uint32_t w[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const uint32_t a = __nv_cvt_float2_to_fp8x2(make_float2(v[4 * i], v[4 * i + 1]), __NV_SATFINITE, __NV_E4M3);
    const uint32_t b = __nv_cvt_float2_to_fp8x2(make_float2(v[4 * i + 2], v[4 * i + 3]), __NV_SATFINITE, __NV_E4M3);
    w[i] = a | b << 16;
  }
  *reinterpret_cast<uint2*>(q) = make_uint2(w[0], w[1]);
}

// NaN is passed over here; its value stays NaN.  Infinity makes the scale infinite and its own value NaN.
template <typename T>
__device__ __forceinline__ float largest8(const Values8<T>& x) {
  float f[8], m = 0.f;
  x.get(f);
#pragma unroll
  for (int i = 0; i < 8; ++i) m = fmaxf(m, fabsf(f[i]));
  return m;
}

// One scale for 128 values of a row: eight lanes per block with 8 values of each half of it; a CTA has 64 consecutive blocks, 32
// where there are few.  ``pitch`` is a multiple of 16 and the row is filled with zeros up to it.  Bound by instructions, which are
// issued in 72 % of the cycles where memory is at 48 % of its peak: 16384 x 4096 bf16 values take 43 us.
template <typename T, int AHEAD>
__global__ void __launch_bounds__(256) quantize_rows_kernel(const T* __restrict__ x, uint8_t* __restrict__ q,
                                                            float* __restrict__ scales, int M, int K, long long ldx,
                                                            long long pitch, long long scale_pitch, int aligned) {
  chain_begin();
  const int lane8 = threadIdx.x & 7, blocks = (K + 127) / 128;
  const long long total = static_cast<long long>(M) * blocks;
  const long long first = static_cast<long long>(blockIdx.x) * 32 * AHEAD + (threadIdx.x >> 3);
  Values8<T> f[AHEAD][2];
  int row[AHEAD], kb[AHEAD];
#pragma unroll
  for (int i = 0; i < AHEAD; ++i) {
    const long long b = first + i * 32;
    if (total <= 0x7fffffffLL) {
      row[i] = static_cast<int>(b) / blocks;
      kb[i] = static_cast<int>(b) - row[i] * blocks;
    } else {
      row[i] = static_cast<int>(b / blocks);
      kb[i] = static_cast<int>(b - static_cast<long long>(row[i]) * blocks);
    }
    const int col = kb[i] * 128 + lane8 * 8;
    const T* src = x + row[i] * ldx + col;
#pragma unroll
    for (int h = 0; h < 2; ++h) f[i][h].load(src + 64 * h, b < total ? K - col - 64 * h : 0, aligned);
  }
#pragma unroll
  for (int i = 0; i < AHEAD; ++i) {
    float m = fmaxf(largest8(f[i][0]), largest8(f[i][1]));
#pragma unroll
    for (int o = 4; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
    if (first + i * 32 >= total) continue;
    const BlockScale s = block_scale(m);
    const int col = kb[i] * 128 + lane8 * 8;
#pragma unroll
    for (int h = 0; h < 2; ++h)
      if (col + 64 * h < pitch) store8(q + row[i] * pitch + col + 64 * h, s, f[i][h]);
    if (lane8 == 0) scales[kb[i] * scale_pitch + row[i]] = s.scale;
  }
}

// One scale for 128 x 128 values, 32 of them a thread: two CTAs per SM take the blocks in turn, and the next block is on its way while
// the present one's largest value is found.  Bound by instructions as the kernel above (78 %, memory at 46 %): 16384 x 4096 bf16 values
// take 43 us; 76 with a CTA for each block, whose loads stop while it waits for its maximum.
template <typename T>
__global__ void __launch_bounds__(512, 2) quantize_blocks_kernel(const T* __restrict__ x, uint8_t* __restrict__ q,
                                                                 float* __restrict__ scales, int M, int K, long long ldx,
                                                                 long long pitch, int aligned) {
  chain_begin();
  __shared__ float most[2][16];
  const int across = (K + 127) / 128, lane16 = threadIdx.x & 15;
  const long long total = static_cast<long long>(across) * ((M + 127) / 128);
  Values8<T> f[4], next[4];
  auto load = [&](long long b, Values8<T> (&to)[4]) {
    const long long mb = b / across;
    const int col = static_cast<int>(b - mb * across) * 128 + lane16 * 8;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const long long row = mb * 128 + (threadIdx.x >> 4) + i * 32;
      to[i].load(x + row * ldx + col, row < M ? K - col : 0, aligned);
    }
  };
  int half = 0;
  if (blockIdx.x < total) load(blockIdx.x, next);
  for (long long b = blockIdx.x; b < total; b += gridDim.x, half ^= 1) {
#pragma unroll
    for (int i = 0; i < 4; ++i) f[i] = next[i];
    if (b + gridDim.x < total) load(b + gridDim.x, next);
    float m = 0.f;
#pragma unroll
    for (int i = 0; i < 4; ++i) m = fmaxf(m, largest8(f[i]));
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
    if ((threadIdx.x & 31) == 0) most[half][threadIdx.x >> 5] = m;
    __syncthreads();                                 // the other half is read behind the next one
#pragma unroll
    for (int i = 0; i < 16; ++i) m = fmaxf(m, most[half][i]);
    const BlockScale s = block_scale(m);
    const long long mb = b / across;
    const int kb = static_cast<int>(b - mb * across), col = kb * 128 + lane16 * 8;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const long long row = mb * 128 + (threadIdx.x >> 4) + i * 32;
      if (row < M && col < pitch) store8(q + row * pitch + col, s, f[i]);
    }
    if (threadIdx.x == 0) scales[b] = s.scale;
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
  static constexpr int SMEM = STAGES * STAGE_BYTES + F8_STAGING + 1024 /*align*/ + 256 /*barriers*/ + SLOTS * 1024 /*scales*/;
};

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
  float* const scale_smem = reinterpret_cast<float*>(smem + STAGES * C::STAGE_BYTES + F8_STAGING + 256);      // [slot][column half][row]
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(&full_bar[s], 1);
      mbar_init(&empty_bar[s], 1);
    }
    for (int s = 0; s < SLOTS; ++s) {
      mbar_init(&tmem_full[s], 1 + 2);         // the products, and the scales of two warps
      mbar_init(&tmem_empty[s], F8_EPI_WARPS);
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

  if (warp < 4) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(F8_FEW));
    // ------------------------------------------------------------ TMA producer
    if (warp == 0 && elect_one()) {
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
    // ------------------------------------------------------------ MMA issuer
    if (warp == 1 && elect_one()) {
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
    // ------------------------------------------------------------ scales (two warps, two rows a thread)
    // The products of both scales of each row and column half go to shared memory beside the accumulator that they belong to.  Those
    // of the next F8_AHEAD blocks are on their way: an access to a far part of L2 takes longer than a block.
    if (warp >= 2) {
      const int r = (warp - 2) * 64 + lane * 2;
      int slot = 0;
      uint32_t slot_phase = 1;
      for (long long tile = worker; tile < tiles && !*abort_flag; tile += workers) {
        int m0, n0;
        place(tile, m0, n0);
        const float* const a0 = p.a_scales + min(m0 + r, p.M - 1) * p.a_row;
        const float* const a1 = p.a_scales + min(m0 + r + 1, p.M - 1) * p.a_row;
        // columns behind the last one have no scale; their sums are not stored
        const float* const b0 = p.b_scales + (min(n0, p.N - 1) / 128) * p.b_row;
        const float* const b1 = p.b_scales + (min(n0 + BN / 2, p.N - 1) / 128) * p.b_row;
        float4 ahead[F8_AHEAD];
        auto fetch = [&](int kb) {
          return kb < kb_end ? make_float4(a0[kb * p.a_block], a1[kb * p.a_block], b0[kb * p.b_block], b1[kb * p.b_block])
                             : make_float4(0.f, 0.f, 0.f, 0.f);
        };
#pragma unroll
        for (int i = 0; i < F8_AHEAD; ++i) ahead[i] = fetch(kb_begin + i);
        for (int kb0 = kb_begin; kb0 < kb_end && !*abort_flag; kb0 += F8_AHEAD) {
#pragma unroll
          for (int i = 0; i < F8_AHEAD; ++i) {       // unrolled: a value that moved to another register would be waited for
            if (kb0 + i >= kb_end) break;
            const float4 v = ahead[i];
            ahead[i] = fetch(kb0 + i + F8_AHEAD);
            if (!__all_sync(0xffffffffu, mbar_wait(&tmem_empty[slot], slot_phase))) {       // the lanes go on together
              *abort_flag = 1;
              atomicExch(p.status, 3);
              break;
            }
            *reinterpret_cast<float2*>(scale_smem + (slot * 2) * F8_BM + r) = make_float2(v.x * v.z, v.y * v.z);
            *reinterpret_cast<float2*>(scale_smem + (slot * 2 + 1) * F8_BM + r) = make_float2(v.x * v.w, v.y * v.w);
            __syncwarp();
            if (lane == 0) mbar_arrive(&tmem_full[slot]);
            if (++slot == SLOTS) {
              slot = 0;
              slot_phase ^= 1;
            }
          }
        }
      }
    }
    __syncwarp();
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(F8_EVEN));      // the same for all behind the branches
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(F8_MANY));
    // ------------------------------------------------------------ scales, sums and stores
    const int quad = warp & 3, part_of_n = (warp - 4) >> 2;  // TMEM lanes and columns of this warp
    uint4* const staged = reinterpret_cast<uint4*>(smem + STAGES * C::STAGE_BYTES) + (warp - 4) * 128;
    constexpr int STEP = COLS < 32 ? COLS : 32;              // columns at a time
    int slot = 0;
    uint32_t slot_phase = 0;
    const bool vectors = p.N % 8 == 0;
    for (long long tile = worker; tile < tiles && !*abort_flag; tile += workers) {
      int m0, n0;
      place(tile, m0, n0);
      float acc[COLS];
#pragma unroll
      for (int i = 0; i < COLS; ++i) acc[i] = 0.f;
      for (int kb = kb_begin; kb < kb_end; ++kb) {
        if (!__all_sync(0xffffffffu, mbar_wait(&tmem_full[slot], slot_phase))) {       // the lanes go on together
          *abort_flag = 1;
          atomicExch(p.status, 4);
          break;
        }
        tc_fence_after();
        const float s = scale_smem[(slot * 2 + part_of_n) * F8_BM + quad * 32 + lane];
        const uint32_t taddr = tmem_base + slot * BN + part_of_n * COLS + (static_cast<uint32_t>(quad * 32) << 16);
        // (Two columns per instruction, which packed arithmetic has, are slower: 501 us against 440 at 16384 x 6144, K 4096.)
#pragma unroll
        for (int c = 0; c < COLS; c += STEP) {
          uint32_t v[STEP];
          if constexpr (STEP == 32) tmem_ld_32x32(taddr + c, v);
          else tmem_ld_32x16(taddr + c, v);
          tmem_ld_wait();
          if (c + STEP == COLS) {
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&tmem_empty[slot]);
          }
#pragma unroll
          for (int i = 0; i < STEP; ++i) acc[c + i] = __fmaf_rn(__uint_as_float(v[i]), s, acc[c + i]);
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
        for (int i = 0; i < COLS; ++i) mine[(part_of_n * COLS + i) * F8_BM + quad * 32 + lane] = acc[i];
        break;                                       // one tile per cluster
      }
      // STEP columns of 32 rows at a time through shared memory (16-byte units, swizzled), so that a row leaves in 64 contiguous bytes
      constexpr int UNITS = STEP / 8;
#pragma unroll
      for (int c = 0; c < COLS; c += STEP) {
        const int col0 = n0 + part_of_n * COLS + c;
        if (col0 >= p.N) break;
#pragma unroll
        for (int i = 0; i < UNITS; ++i) {
          uint32_t w[4];
#pragma unroll
          for (int k = 0; k < 4; ++k) w[k] = pack_bf16(acc[c + i * 8 + 2 * k], acc[c + i * 8 + 2 * k + 1]);
          staged[lane * 4 + (i ^ (lane >> 1 & 3))] = make_uint4(w[0], w[1], w[2], w[3]);
        }
        __syncwarp();
        const int unit = lane & 3, col = col0 + unit * 8;
#pragma unroll
        for (int it = 0; it < 4; ++it) {
          const int r = it * 8 + (lane >> 2), out_row = m0 + quad * 32 + r;
          if (out_row >= p.M || unit >= UNITS || col >= p.N) continue;
          const uint4 v = staged[r * 4 + (unit ^ (r >> 1 & 3))];
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
    __syncwarp();
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(F8_EVEN));
  }
  if (SPLIT) {
    __syncwarp();
    cluster_sync_all();
    int m0, n0;
    place(worker, m0, n0);
    // this CTA's share of the columns, two at a time; consecutive threads hold consecutive rows
    constexpr int SHARE = BN / (SPLIT ? SPLIT : 1);
    const bool bad = *abort_flag != 0;
    const int rows = min(F8_BM, p.M - m0);
    for (int i = threadIdx.x; i < rows * (SHARE / 2) && !bad; i += F8_THREADS) {
      const int r = i % rows, c = part * SHARE + i / rows * 2;
      if (n0 + c >= p.N) continue;
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
  constexpr auto kernel = gemm_fp8_kernel<BN, B_MN, SPLIT>;
  if (allow_shared<kernel>(F8Cfg<BN>::SMEM) != cudaSuccess) return -3;
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

// Tile width and split by a model of the time, in units of a block of a 256-column tile (0.6 us): waves of tiles, each with its blocks
// along k and an end.  Fitted to, us of 256, 128 and 64 columns: 1003 x 4096, K 4096 20, 22, 36; 64 x 14336, K 4096 20, 11.5, 18; 2048
// x 4096, K 1024 15, 15, 18; 128 x 512, K 512 5, 3, 2.  Few rows leave SMs without a tile: CTAs of a cluster share the blocks of one
// (16 x 1024, K 14336, 128 columns: 29 us on one CTA a tile, 20, 11 and 7 on two, four and eight; 16 x 4096, K 4096 9.4, 9, 7 on
// one, two and four).  Joining them costs by the row: 128 x 512, K 512 3 us alone, 13 shared by two.
struct Fp8Choice {
  int bn, split;
};
static Fp8Choice choose_fp8(int M, int N, int K, int nn) {
  const long long rows = (M + F8_BM - 1) / F8_BM, blocks = (K + F8_BK - 1) / F8_BK, sms = f8_sms();
  Fp8Choice best = {256, 0};
  double least = 1e30;
  for (int bn : {256, 128, 64}) {
    if (nn && bn == 64) continue;                    // a box of B along its columns is 128 wide
    const long long tiles = rows * ((N + bn - 1) / bn);
    const double block = bn == 256 ? 1.0 : bn == 128 ? 0.55 : 0.46, end = bn == 256 ? 4.7 : bn == 128 ? 2.0 : 0.5;
    for (int split : {1, 2, 4, 8}) {
      // clusters that the device holds at a time, with a margin: they do not cross its partitions
      if (split > 1 && (M > 32 || blocks < 2 * split || tiles > (split == 2 ? 70 : split == 4 ? 32 : 14))) continue;
      const double time = (split > 1 ? 1 : (tiles + sms - 1) / sms) * ((blocks + split - 1) / split * block + end) + (split > 1 ? 3.0 : 0.0);
      if (time < least) {
        least = time;
        best = {bn, split > 1 ? split : 0};
      }
    }
  }
  return best;
}

template <int BN, int B_MN>
static int launch_fp8(const Fp8Params& p, int split, cudaStream_t s) {
  switch (split) {
    case 2: return launch_fp8<BN, B_MN, 2>(p, s);
    case 4: return launch_fp8<BN, B_MN, 4>(p, s);
    case 8: return launch_fp8<BN, B_MN, 8>(p, s);
    default: return launch_fp8<BN, B_MN, 0>(p, s);
  }
}

template <typename T>
static cudaError_t launch_quantize(const void* x, void* q, float* scales, int M, int K, long long ldx, long long pitch,
                                   long long scale_pitch, int block_rows, int aligned, cudaStream_t s) {
  const T* in = static_cast<const T*>(x);
  uint8_t* out = static_cast<uint8_t*>(q);
  const long long across = (K + 127) / 128, blocks = M * across;
  if (block_rows == 128) {
    const long long squares = across * ((M + 127) / 128), most = f8_sms() * 2LL;
    return launch_next(quantize_blocks_kernel<T>, static_cast<unsigned>(squares < most ? squares : most), 512, 0, s, in, out, scales, M, K,
                       ldx, pitch, aligned);
  }
  // few blocks are spread over more CTAs
  if (blocks <= f8_sms() * 64LL)
    return launch_next(quantize_rows_kernel<T, 1>, static_cast<unsigned>((blocks + 31) / 32), 256, 0, s, in, out, scales, M, K, ldx,
                       pitch, scale_pitch, aligned);
  return launch_next(quantize_rows_kernel<T, 2>, static_cast<unsigned>((blocks + 63) / 64), 256, 0, s, in, out, scales, M, K, ldx,
                     pitch, scale_pitch, aligned);
}

}  // namespace b2

using namespace b2;

extern "C" {

// x [M, K] (type 0 fp32, 1 bf16, 2 fp16; row pitch ldx) -> e4m3 values [M, pitch], zeros from column K on, and fp32 scales:
// block_rows 1: [ceil(K / 128), scale_pitch], the scale of row m in column m; 128: [ceil(M / 128), ceil(K / 128)].
int b2_quantize_fp8(const void* x, int type, void* q, float* scales, long long M, int K, long long ldx, long long pitch,
                    long long scale_pitch, int block_rows, cudaStream_t s) {
  if (M < 0 || M > F8_MAX || K < 1 || K > F8_MAX || pitch < K || pitch % 16 || pitch - K >= 128 || type < 0 || type > 2 ||
      (block_rows != 1 && block_rows != 128))
    return -10;
  if (M == 0) return 0;
  const int size = type == QUANT_F32 ? 4 : 2;
  const int aligned = ldx * size % 16 == 0 && reinterpret_cast<uintptr_t>(x) % 16 == 0;
  const int rows = static_cast<int>(M);
  const cudaError_t r =
      type == QUANT_F32    ? launch_quantize<float>(x, q, scales, rows, K, ldx, pitch, scale_pitch, block_rows, aligned, s)
      : type == QUANT_BF16 ? launch_quantize<__nv_bfloat16>(x, q, scales, rows, K, ldx, pitch, scale_pitch, block_rows, aligned, s)
                           : launch_quantize<__half>(x, q, scales, rows, K, ldx, pitch, scale_pitch, block_rows, aligned, s);
  if (r != cudaSuccess) cudaGetLastError();
  return r == cudaSuccess ? 0 : -1;
}

// d[M, N] bf16 = a[M, K] * w[N, K]^T (nn 0) or a[M, K] * w[K, N] (nn 1), e4m3 values with row pitches lda, ldw (multiples of 16) and
// their scales; b_row, b_block: strides of w's scales along n and along k.
int b2_gemm_fp8(const void* a, const float* a_scales, const void* w, const float* b_scales, void* d, int M, int N, int K,
                long long lda, long long ldw, long long a_row, long long a_block, long long b_row, long long b_block, int nn,
                int* status, cudaStream_t s) {
  if (M < 0 || M > F8_MAX || N < 1 || N > F8_MAX || K < 1 || K > F8_MAX || lda % 16 || ldw % 16) return -10;
  if (M == 0) return 0;
  Fp8Params p{};
  p.a_scales = a_scales; p.b_scales = b_scales; p.a_row = a_row; p.a_block = a_block; p.b_row = b_row; p.b_block = b_block;
  p.d = static_cast<__nv_bfloat16*>(d); p.M = M; p.N = N; p.K = K; p.status = status;
  if (make_map8(&p.map_a, a, K, M, lda, F8_BM)) return -11;
  const Fp8Choice c = choose_fp8(M, N, K, nn);
  if (nn ? make_map8(&p.map_b, w, N, K, ldw, 128) : make_map8(&p.map_b, w, K, N, ldw, c.bn)) return -12;
  if (nn) return c.bn == 256 ? launch_fp8<256, 1>(p, c.split, s) : launch_fp8<128, 1>(p, c.split, s);
  if (c.bn == 256) return launch_fp8<256, 0>(p, c.split, s);
  return c.bn == 128 ? launch_fp8<128, 0>(p, c.split, s) : launch_fp8<64, 0>(p, c.split, s);
}

}  // extern "C"
