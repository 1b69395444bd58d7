// Pieces of the kernels whose tiles a pair of CTAs shares (linear_nvfp4_2cta.cu, linear_nvfp4_grouped_2cta.cu): the tile's layout in shared
// and tensor memory, and the drain of an accumulator.
#pragma once

#include "gemm_common.cuh"

namespace ac4k {
using namespace ptx;

namespace pair {
static constexpr int BMP = 256;                     // output rows of the pair tile
static constexpr int KS = 4;                        // K = 64 steps per stage
static constexpr int A_BYTES = 128 * BKB;           // this CTA's 128 rows of A, K = 256
static constexpr int SFA_BYTES = KS * 512;          // [K step][32 x 16 B]
static constexpr int SFB_BYTES = 2 * KS * 512;      // [128-row block of B][K step][32 x 16 B]
static constexpr int STAGES = 5;
static constexpr int BIAS_BYTES = 8 * 128 * 4;      // one tile's bias as fp32, 128 columns per epilogue warp
static constexpr int OUT_STAGE_BYTES = 32 * 128;    // per epilogue warp: 32 rows x 64 columns of 16-bit outputs
static constexpr int BAR_BYTES = 256;
static constexpr int kThreadsPair = 448;            // 14 warps: 144 registers per thread for the epilogue
// BN_: output columns of the pair tile, 256 or 192
template <int BN_>
struct Tile {
  static constexpr int BN = BN_;
  static constexpr int B_ROWS = BN / 2;             // this CTA's rows of B
  static constexpr int B_BYTES = B_ROWS * BKB;      // K = 256
  static constexpr int STAGE_TX = A_BYTES + B_BYTES + SFA_BYTES + SFB_BYTES;    // bytes one CTA's TMA loads of a stage bring
  // Tensor memory (512 columns): two accumulators that the tiles use in turn, and the scales of one stage.  Two of 256 columns share
  // 48: the last 48 of the first accumulator's tile and the first 48 of the second one's, so between two tiles only those 48
  // columns have to be read out before the next tile's first MMA may write them - the other 208 are drained while the next
  // tile's MMAs already run.  Two of 192 share none.
  static constexpr int ACC1_COL = BN == 256 ? 208 : BN;      // accumulator 0: columns [0, BN), accumulator 1: from here
  static constexpr int SHARED_COLS = BN - ACC1_COL;          // 48, 0
  static constexpr int SF_COL = ACC1_COL + BN;      // per K step 4 columns for A, then 8 per K step for B
  static constexpr int SF_COLS = KS * 12;
  // no slack for aligning the base: the kernel declares the array 1024-byte aligned and checks it
  static constexpr int SMEM_BYTES = STAGES * STAGE_TX + 8 * OUT_STAGE_BYTES + BIAS_BYTES + BAR_BYTES;
  static_assert(SF_COL + SF_COLS <= kTmemCols, "tensor memory overflow");
  static_assert(SMEM_BYTES <= 227 * 1024, "shared memory overflow");
  static_assert(B_BYTES % 1024 == 0, "a stage's B starts on a swizzle atom");
};
}  // namespace pair

// N accumulator columns starting at COL0 of this thread's 128-column segment: * alpha (+ bias from shared
// memory), rounded to the 16-bit output type, two per word into w[COL0 / 2 ...].
template <int OUT_DT, int COL0, int N>
__device__ __forceinline__ void pack_cols(const uint32_t (&r)[N], uint32_t (&w)[64], float alpha, bool has_bias, uint32_t bias_s) {
  static_assert(COL0 % 4 == 0 && N % 4 == 0, "whole 16-byte bias groups");
  if (!has_bias) {
#pragma unroll
    for (int i = 0; i < N / 2; ++i)
      w[COL0 / 2 + i] = (OUT_DT == AC4K_DT_BF16) ? scale_pack_bf16x2(r[2 * i], r[2 * i + 1], alpha)
                                                 : scale_pack_f16x2(r[2 * i], r[2 * i + 1], alpha);
  } else {
#pragma unroll
    for (int i = 0; i < N / 4; ++i) {
      const float4 bb = ld_shared_v4f(bias_s + (COL0 + 4 * i) * 4);
      if (OUT_DT == AC4K_DT_BF16) {
        w[COL0 / 2 + 2 * i] = scale_bias_pack_bf16x2(r[4 * i], r[4 * i + 1], alpha, bb.x, bb.y);
        w[COL0 / 2 + 2 * i + 1] = scale_bias_pack_bf16x2(r[4 * i + 2], r[4 * i + 3], alpha, bb.z, bb.w);
      } else {
        w[COL0 / 2 + 2 * i] = scale_bias_pack_f16x2(r[4 * i], r[4 * i + 1], alpha, bb.x, bb.y);
        w[COL0 / 2 + 2 * i + 1] = scale_bias_pack_f16x2(r[4 * i + 2], r[4 * i + 3], alpha, bb.z, bb.w);
      }
    }
  }
}

// One output word of the row-permuted variant: accumulator values of output columns col, col + 1 of this thread's
// 128-column segment.
template <int OUT_DT, bool BIAS>
__device__ __forceinline__ uint32_t pack_pair(uint32_t lo, uint32_t hi, float alpha, uint32_t bias_s, int col) {
  if (!BIAS) return (OUT_DT == AC4K_DT_BF16) ? scale_pack_bf16x2(lo, hi, alpha) : scale_pack_f16x2(lo, hi, alpha);
  const float2 bb = ld_shared_v2f(bias_s + col * 4);
  return (OUT_DT == AC4K_DT_BF16) ? scale_bias_pack_bf16x2(lo, hi, alpha, bb.x, bb.y) : scale_bias_pack_f16x2(lo, hi, alpha, bb.x, bb.y);
}

// Drain of this warp's 128 accumulator columns in the row-permuted variant.  Column c holds output column
// 4 (c % 32) + c / 32 of the segment: output columns 4 l, 4 l + 1 (word 2 l) come from columns l and 32 + l, output
// columns 4 l + 2, 4 l + 3 (word 2 l + 1) from 64 + l and 96 + l.  Step S = 2 u + v reads columns 64 u + 16 v + [0, 16)
// and the 16 columns 32 further on and packs words 2 l + u, l = 16 v + [0, 16); the first two steps are read together,
// later ones are in flight while a step is packed.
template <int S>
__device__ __forceinline__ void drain_issue(uint32_t t_row, uint32_t (&lo)[16], uint32_t (&hi)[16]) {
  tmem_ld_32x32b_x16(t_row + (S >> 1) * 64 + (S & 1) * 16, lo);
  tmem_ld_32x32b_x16(t_row + (S >> 1) * 64 + (S & 1) * 16 + 32, hi);
}
template <int OUT_DT, bool BIAS, int S>
__device__ __forceinline__ void drain_pack(uint32_t (&w)[64], const uint32_t (&lo)[16], const uint32_t (&hi)[16], float alpha,
                                           uint32_t bias_s) {
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    constexpr int u = S >> 1, v = S & 1;
    w[2 * (16 * v + i) + u] = pack_pair<OUT_DT, BIAS>(lo[i], hi[i], alpha, bias_s, 4 * (16 * v + i) + 2 * u);
  }
}
// Steps in the order S0 .. S3; after the first two (which must cover the columns both accumulators share, if this
// warp has any of them: `arrive`) the shared columns are reported free.
template <int OUT_DT, bool BIAS, int S0, int S1, int S2, int S3>
__device__ __forceinline__ void drain_permuted(uint32_t (&w)[64], uint32_t t_row, bool arrive, float alpha, uint32_t bias_s,
                                               int lane, uint32_t leader_shared_free) {
  uint32_t a_lo[16], a_hi[16], b_lo[16], b_hi[16];
  drain_issue<S0>(t_row, a_lo, a_hi);
  drain_issue<S1>(t_row, b_lo, b_hi);
  tmem_ld_wait();
  tmem_pin(a_lo);
  tmem_pin(a_hi);
  tmem_pin(b_lo);
  tmem_pin(b_hi);
  if (arrive) {
    tc_fence_before();
    __syncwarp();
    if (lane == 0) mbar_arrive_cluster(leader_shared_free);
  }
  drain_pack<OUT_DT, BIAS, S0>(w, a_lo, a_hi, alpha, bias_s);
  drain_issue<S2>(t_row, a_lo, a_hi);
  drain_pack<OUT_DT, BIAS, S1>(w, b_lo, b_hi, alpha, bias_s);
  tmem_ld_wait();
  tmem_pin(a_lo);
  tmem_pin(a_hi);
  drain_issue<S3>(t_row, b_lo, b_hi);
  drain_pack<OUT_DT, BIAS, S2>(w, a_lo, a_hi, alpha, bias_s);
  tmem_ld_wait();
  tmem_pin(b_lo);
  tmem_pin(b_hi);
  drain_pack<OUT_DT, BIAS, S3>(w, b_lo, b_hi, alpha, bias_s);
}

}  // namespace ac4k
