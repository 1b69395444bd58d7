// NVFP4 block-scaled products with a weight per group of rows (experts): rows [offsets[e], offsets[e + 1]) of A against weight e.
//
//   D[t, n] = A_gs * B_gs[e] * sum_k A[t, k] B[e, n, k] + bias[e, n]
//
// The groups' lengths are on the device and ragged, so a launch has a block for every tile that there can be (ragged.cuh) and a block looks its
// rows up.  As in the decode-shape kernel (linear_nvfp4_skinny.cu, whose structure this one has) 128 weight rows are the M side of the MMA and the
// tile's NT activation rows the N side: a group begins at any row, and the N side may be as narrow as the groups are.  Activation boxes
// reach into the next group's rows or past the last one (zeros); their columns of the accumulator are not stored.
//
// One block: 128 weight rows x NT activation rows x one slice of K; the slices (1, 2 or 4, few tiles only) are a cluster that adds its
// partial sums through distributed shared memory.  192 threads: warp 0 TMA producer, warp 1 MMA issuer (scales to tensor memory with
// tcgen05.cp, four MMAs a stage of K = 256), warps 2-5 epilogue, which also re-order each stage's scale words [K/64][rows][4 B] into the
// 32 x 16-byte chunks that tcgen05.cp takes (a group's first row is at any word of them, which no TMA box may start at).
//
// Bound by the weights' stream where groups are short: 32 rows of 8 groups, 8192 x 4096, 30 us (151 MB, 5.0 TB/s).
//
// Kernel and tile go by the groups' mean length: the host does not know the lengths.  A long group among short ones streams its weights once a tile of the
// mean's size, through L2: 1024 rows of 128 groups, 2048 x 2048, of which one has 600 take 84 to 89 us, even ones 79 to 83, the long one alone 13 to 15.
#include "gemm_common.cuh"
#include "ragged.cuh"

namespace ac4k {
using namespace ptx;

namespace grouped {
static constexpr int KS = 4;                     // K = 64 steps per stage (K = 256)
static constexpr int W_BYTES = 128 * BKB;        // 128 weight rows x 128 bytes
static constexpr int SF_BYTES = KS * 512;        // scale chunks of one 128-row block
static constexpr int kThreads = 192;
// Groups of more rows than this on average go to the CTA pairs, whose tiles follow one another without a gap: 64 groups of 32 rows, 2048 x 1024, take
// 25.4 us there and 38.8 here, 128 of 16, 1024 x 2048, 37.4 and 37.9, 64 of 16, 1024 x 4096, 39.1 and 34.4, 2048 x 1024, 24.8 and 29.2.
constexpr int pair_rows(int64_t K) { return K <= 1024 ? 8 : 24; }
template <int NT>
struct Cfg {
  static constexpr int X_BYTES = NT * BKB;
  static constexpr int STAGES = NT >= 64 ? 3 : 4;       // two blocks fit on an SM in every configuration
  static constexpr int STAGE_BYTES = W_BYTES + X_BYTES + 2 * SF_BYTES;
  // partial sums received from the other slices, as in the decode-shape kernel; a tile of 128 rows has one slice
  static constexpr int PART_UNIT = NT * 128;
  static constexpr int PART_BYTES = NT <= 64 ? 3 * PART_UNIT : 0;
  static_assert(NT > 64 || 4 * PART_UNIT <= STAGES * W_BYTES, "the warps' own partial sums reuse the weight buffers");
  static constexpr int SMEM_BYTES = STAGES * STAGE_BYTES + PART_BYTES + 1024 /*alignment*/ + 256 /*barriers*/;
  static_assert(2 * (SMEM_BYTES + 1024 + 256) <= 228 * 1024, "shared memory per SM");
  // tensor memory: accumulator, weight scales, activation scales
  static constexpr int SFW_COL = NT <= 64 ? 64 : 128, SFX_COL = SFW_COL + 4 * KS;
  static constexpr int TMEM_COLS = NT <= 64 ? 128 : 256;
  static_assert(SFX_COL + 4 * KS <= TMEM_COLS && 2 * TMEM_COLS <= kTmemCols, "tensor memory");
};

struct Args {
  const uint8_t *sfa, *sfb;      // scales in the row layout: [K/64][rows_sfa][4], [E][K/64][rows_sfb][4]
  void *D;
  const float *a_gs, *b_gs;
  int b_gs_stride;               // 0: one global scale for all weights, 1: one each
  const void *bias;              // [E][N] or NULL
  int bias_dt;
  const int32_t *offsets;
  unsigned int *status;
  int rows, groups, N, KT;
  int rows_sfa, rows_sfb;
  int tiles_n, splits, kt_per_split;
  bool fill;                     // write zeros to the rows of no group
  unsigned long long wait_ns;
  int dbg;                       // experiment switches (builds with -DAC4K_DEBUG_HOOKS), else 0
};

// alpha and bias of a weight row (output column) of group e
struct Affine { float alpha, bias; bool has_bias; };
__device__ __forceinline__ Affine affine_of(const Args &p, int e, int n) {
  Affine f;
  f.alpha = __fmul_rn(__ldg(p.a_gs), __ldg(p.b_gs + e * p.b_gs_stride));
  f.has_bias = p.bias != nullptr;
  f.bias = 0.0f;
  if (f.has_bias && n < p.N) {
    const int64_t i = (int64_t)e * p.N + n;
    if (p.bias_dt == AC4K_DT_BF16) f.bias = __bfloat162float(static_cast<const __nv_bfloat16 *>(p.bias)[i]);
    else if (p.bias_dt == AC4K_DT_FP16) f.bias = __half2float(static_cast<const __half *>(p.bias)[i]);
    else f.bias = static_cast<const float *>(p.bias)[i];
  }
  return f;
}
__device__ __forceinline__ float apply(const Affine &f, float acc) {
  const float v = __fmul_rn(acc, f.alpha);
  return f.has_bias ? __fadd_rn(v, f.bias) : v;
}

// Several K slices: `rows` activation rows of 128 output columns, the slices added in order (see finish_split of the decode-shape kernel)
template <int SPLITS, int OUT_DT>
__device__ __forceinline__ void add_slices(uint32_t own0, uint32_t part0, int slice, int rows, int rs, const Affine &f, int N,
                                           typename OutT<OUT_DT>::type *dst) {
#pragma unroll 1
  for (int i0 = 0; i0 < rows; i0 += 8) {
    float x[SPLITS][8];
#pragma unroll
    for (int sl = 0; sl < SPLITS; ++sl) {
      const uint32_t base = (sl == slice ? own0 : part0 + (uint32_t)((sl < slice ? sl : sl - 1) * rs) * 128u) + (uint32_t)i0 * 128u;
#pragma unroll
      for (int i = 0; i < 8; ++i) x[sl][i] = i0 + i < rows ? ld_shared_f32(base + i * 128) : 0.0f;
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      float v = x[0][i];
#pragma unroll
      for (int sl = 1; sl < SPLITS; ++sl) v = __fadd_rn(v, x[sl][i]);
      if (i0 + i < rows) store_out<OUT_DT>(dst + (int64_t)(i0 + i) * N, apply(f, v));
    }
  }
}
}  // namespace grouped

template <int NT, int OUT_DT>
__global__ void __launch_bounds__(grouped::kThreads, 2)
linear_nvfp4_grouped_kernel(const __grid_constant__ CUtensorMap tma_x, const __grid_constant__ CUtensorMap tma_w, const grouped::Args p) {
  using namespace grouped;
  using C = grouped::Cfg<NT>;
  constexpr int STAGES = C::STAGES;
  using T = typename OutT<OUT_DT>::type;
  extern __shared__ uint8_t smem_raw[];
  __shared__ RaggedScratch scratch;
  const uint32_t smem_base = (smem_u32(smem_raw) + 1023u) & ~1023u;
  const uint32_t sW = smem_base;
  const uint32_t sX = sW + STAGES * W_BYTES;
  const uint32_t sSFW = sX + STAGES * C::X_BYTES;
  const uint32_t sSFX = sSFW + STAGES * SF_BYTES;
  const uint32_t sPart = sSFX + STAGES * SF_BYTES;
  const uint32_t bars = sPart + C::PART_BYTES;
  const uint32_t full_bar = bars, empty_bar = bars + 8 * STAGES;
  const uint32_t tfull_bar = bars + 16 * STAGES;
  const uint32_t part_bar = tfull_bar + 8;      // [quarter] the other slices' partial sums of this block's activation rows have landed
  const uint32_t tmem_slot = part_bar + 32;
  uint8_t *smem_gen = smem_raw + (smem_base - smem_u32(smem_raw));

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int slice = p.splits > 1 ? (int)cluster_ctarank() : 0;
  const int item = blockIdx.x / p.splits, tn = item % p.tiles_n;
  if (threadIdx.x == 0) {
    prefetch_tmap(&tma_x);
    prefetch_tmap(&tma_w);
  }
  grid_dependency_wait();
  grid_launch_dependents();
  const RaggedTile tile = ragged_tile<kThreads>(p.offsets, p.groups, p.rows, NT, item / p.tiles_n, &scratch);
  const int n0 = tn * 128;
  if (tile.group < 0) {           // (all blocks of a cluster alike)
    if (tile.group == -1 && p.fill && slice == 0 && threadIdx.x < 128 && n0 + (int)threadIdx.x < p.N)
      for (int m = tile.row0; m < tile.row1; ++m) store_out<OUT_DT>(static_cast<T *>(p.D) + (int64_t)m * p.N + n0 + threadIdx.x, 0.0f);
    return;
  }
  const int M = tile.row1 - tile.row0;
  const int k_tiles_all = (p.KT + KS - 1) / KS;
  const int kt0 = slice * p.kt_per_split, kt1 = min(k_tiles_all, kt0 + p.kt_per_split);
  // activation rows that slice s finishes: [s * rs, s * rs + rows_of(s)) of the tile
  const int rs = (M + p.splits - 1) / p.splits;
  auto rows_of = [&](int s) { return max(0, min(rs, M - s * rs)); };

  if (threadIdx.x == 0) {
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(full_bar + 8 * s, 2);            // producer's expect_tx arrival and the stage's scale warp
      mbar_init(empty_bar + 8 * s, 1);
    }
    mbar_init(tfull_bar, 1);
    for (int q = 0; q < 4; ++q) mbar_init(part_bar + 8 * q, 1);
    if (p.splits > 1 && rows_of(slice) > 0) {
      // each quarter receives one copy of this block's rows x 128 bytes from every other slice
      for (int q = 0; q < 4; ++q) mbar_arrive_expect_tx(part_bar + 8 * q, (uint32_t)((p.splits - 1) * rows_of(slice)) * 128u);
    }
    fence_barrier_init();
  }
  if (warp == 1) {
    tmem_alloc(tmem_slot, C::TMEM_COLS);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  if (p.splits > 1) cluster_sync();     // the other slices' barriers exist before anything is signalled remotely
  tc_fence_after();
  const uint32_t tmem_base = *reinterpret_cast<volatile uint32_t *>(smem_gen + (tmem_slot - smem_base));

  if (warp == 0) {
    // ------------------------------------------------------------------ TMA producer
    const uint32_t el = elect_one();
    const int w_row = tile.group * p.N + n0;
    uint32_t s = 0, ph = 0;
    bool ok = true;
    for (int kt = kt0; kt < kt1; ++kt) {
      ok = warp_all(mbar_wait(empty_bar + 8 * s, ph ^ 1, p.wait_ns));
      if (!ok) break;
      if (AC4K_DBG(p, 256) && kt == kt0 && blockIdx.x == 0) {        // wait-expiry test: this stage's operands never come
        if (++s == STAGES) { s = 0; ph ^= 1; }
        continue;
      }
      const uint32_t fb = full_bar + 8 * s;
      mbar_arrive_expect_tx_if(el, fb, W_BYTES + C::X_BYTES);
      tma_load_2d_if(el, sW + s * W_BYTES, &tma_w, kt * BKB, w_row, fb);
      tma_load_2d_if(el, sX + s * C::X_BYTES, &tma_x, kt * BKB, tile.row0, fb);
      if (++s == STAGES) { s = 0; ph ^= 1; }
    }
    if (!ok && el) atomicExch(p.status, kStatusTimeoutProducer);
  } else if (warp == 1) {
    // ------------------------------------------------------------------ MMA issuer
    const uint32_t el = elect_one();
    constexpr uint32_t idesc = make_idesc_mxf4nvf4(128, NT);
    uint32_t s = 0, ph = 0;
    bool ok = true;
    const uint64_t wdesc0 = make_smem_desc(sW, 16, 1024, kSwizzle128B);
    const uint64_t xdesc0 = make_smem_desc(sX, 16, 1024, kSwizzle128B);
    const uint64_t sfwdesc0 = make_smem_desc(sSFW, 0, 128, kSwizzleNone);
    const uint64_t sfxdesc0 = make_smem_desc(sSFX, 0, 128, kSwizzleNone);
    const uint32_t t_sfw = tmem_base + C::SFW_COL, t_sfx = tmem_base + C::SFX_COL;
    for (int kt = kt0; kt < kt1; ++kt) {
      ok = warp_all(mbar_wait(full_bar + 8 * s, ph, p.wait_ns));
      if (!ok) break;
      tc_fence_after();
      const int nk = min(KS, p.KT - kt * KS);
      const uint64_t wdesc = wdesc0 + (uint64_t)(s * (W_BYTES >> 4));
      const uint64_t xdesc = xdesc0 + (uint64_t)(s * (C::X_BYTES >> 4));
      const uint64_t sfwdesc = sfwdesc0 + (uint64_t)(s * (SF_BYTES >> 4));
      const uint64_t sfxdesc = sfxdesc0 + (uint64_t)(s * (SF_BYTES >> 4));
      if (nk == KS) {
#pragma unroll
        for (int j = 0; j < KS; ++j) {
          tmem_cp_32x128b_warpx4_if(el, t_sfw + j * 4, sfwdesc + j * 32);
          tmem_cp_32x128b_warpx4_if(el, t_sfx + j * 4, sfxdesc + j * 32);
        }
#pragma unroll
        for (int j = 0; j < KS; ++j)
          mma_mxf4nvf4_if(el, tmem_base, wdesc + 2 * j, xdesc + 2 * j, idesc, t_sfw + j * 4, t_sfx + j * 4,
                          (kt > kt0 || j > 0) ? 1u : 0u);
      } else {
        for (int j = 0; j < nk; ++j) {
          tmem_cp_32x128b_warpx4_if(el, t_sfw + j * 4, sfwdesc + j * 32);
          tmem_cp_32x128b_warpx4_if(el, t_sfx + j * 4, sfxdesc + j * 32);
        }
        for (int j = 0; j < nk; ++j)
          mma_mxf4nvf4_if(el, tmem_base, wdesc + 2 * j, xdesc + 2 * j, idesc, t_sfw + j * 4, t_sfx + j * 4,
                          (kt > kt0 || j > 0) ? 1u : 0u);
      }
      tc_commit_if(el, empty_bar + 8 * s);
      if (++s == STAGES) { s = 0; ph ^= 1; }
    }
    if (ok) tc_commit_if(el, tfull_bar);
    if (!ok && el) atomicExch(p.status, kStatusTimeoutMma);
  } else {
    // ------------------------------------------------------------------ scale re-ordering, then epilogue
    const int q = warp & 3;                   // tensor-memory lane quarter of this warp (warps 2-5 -> 2, 3, 0, 1)
    {
      // [K/64][rows][4 bytes] -> per K step 32 rows of 16 bytes, row l holding the words of rows l, 32 + l, 64 + l, 96 + l of the block;
      // warp w takes the stages whose number is w - 2 modulo NW, NW no more than the depth of the ring (a warp is then at most
      // one round of the ring ahead, which the parity of the stage's barrier can tell apart).
      constexpr int NW = STAGES < 4 ? STAGES : 4;
      constexpr int GX = (NT + 31) / 32;      // words of an activation block's row that the MMA reads
      const int w4 = warp - 2;
      uint32_t s = 0, ph = 0, it = 0;
      const uint32_t *sfx_w = reinterpret_cast<const uint32_t *>(p.sfa);
      const uint32_t *sfw_w = reinterpret_cast<const uint32_t *>(p.sfb) + (int64_t)tile.group * p.KT * p.rows_sfb;
      bool ok = true;
      for (int kt = kt0; kt < kt1; ++kt) {
        if ((int)(it % NW) == w4) {
          uint32_t ww[KS][4], wx[KS][4];
#pragma unroll
          for (int j = 0; j < KS; ++j) {
            const int k64 = kt * KS + j;
            const bool k_ok = k64 < p.KT;
#pragma unroll
            for (int g = 0; g < 4; ++g) {
              const int rw = n0 + 32 * g + lane, rx = tile.row0 + 32 * g + lane;
              ww[j][g] = (k_ok && rw < p.rows_sfb) ? __ldg(sfw_w + (int64_t)k64 * p.rows_sfb + rw) : 0u;
              wx[j][g] = (g < GX && k_ok && rx < p.rows_sfa) ? __ldg(sfx_w + (int64_t)k64 * p.rows_sfa + rx) : 0u;
            }
          }
          ok = warp_all(mbar_wait(empty_bar + 8 * s, ph ^ 1, p.wait_ns));
          if (!ok) break;
#pragma unroll
          for (int j = 0; j < KS; ++j) {
            st_shared_v4u(sSFW + s * SF_BYTES + j * 512 + lane * 16, ww[j][0], ww[j][1], ww[j][2], ww[j][3]);
            st_shared_v4u(sSFX + s * SF_BYTES + j * 512 + lane * 16, wx[j][0], wx[j][1], wx[j][2], wx[j][3]);
          }
          fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0) mbar_arrive(full_bar + 8 * s);
        }
        ++it;
        if (++s == STAGES) { s = 0; ph ^= 1; }
      }
      if (!ok && lane == 0) atomicExch(p.status, kStatusTimeoutSf);
    }
    // ---- epilogue: lane l of quarter q owns weight row (output column) n0 + 32 q + l, its NT accumulator columns are the activation rows
    const int n = n0 + q * 32 + lane;
    const Affine f = affine_of(p, tile.group, n);
    const bool tfull_ok = mbar_wait(tfull_bar, 0, p.wait_ns);
    if (!tfull_ok && lane == 0) atomicExch(p.status, kStatusTimeoutEpilogue);
    tc_fence_after();
    const uint32_t t_row = tmem_base + ((uint32_t)(q * 32) << 16);
    if (NT > 64 || p.splits == 1) {
      constexpr int CH = NT < 32 ? NT : 32;
      T *dst = static_cast<T *>(p.D) + (int64_t)tile.row0 * p.N + n;
#pragma unroll 1
      for (int c = 0; c < M; c += CH) {
        uint32_t r[CH];
        __syncwarp();
        tmem_ld_cols<CH>(t_row + c, r);
        if (n < p.N && tfull_ok) {
#pragma unroll
          for (int i = 0; i < CH; ++i)
            if (c + i < M) store_out<OUT_DT>(dst + (int64_t)(c + i) * p.N, apply(f, __uint_as_float(r[i])));
        }
      }
    } else if constexpr (NT <= 64) {
      // This warp's partial sums are laid out [activation row][lane] in this block's weight buffers (free: all its MMAs are
      // complete); the rows of every other slice travel there as one bulk copy, to unit [quarter][source slice, skipping
      // the owner's own].
      uint32_t r[NT];
      tmem_ld_cols<NT>(t_row, r);
      const uint32_t own = sW + (uint32_t)(warp - 2) * C::PART_UNIT;
#pragma unroll
      for (int m = 0; m < NT; ++m)
        if (m < M) st_shared_f32(own + m * 128 + lane * 4, __uint_as_float(r[m]));
      fence_proxy_async_smem();
      __syncwarp();
      if (tfull_ok && lane < p.splits && lane != slice && rows_of(lane) > 0) {      // (a slice that gave up sends nothing: nothing of it comes late)
        const int o = lane;
        const uint32_t unit = (uint32_t)(q * (p.splits - 1) + (slice < o ? slice : slice - 1)) * (uint32_t)rs * 128u;
        bulk_copy_to_cluster(map_to_cta(sPart + unit, o), own + (uint32_t)(o * rs) * 128u, (uint32_t)rows_of(o) * 128u,
                             map_to_cta(part_bar + 8 * q, o));
      }
      const int rows = rows_of(slice);
      if (rows > 0) {
        const bool got = mbar_wait(part_bar + 8 * q, 0, p.wait_ns);
        if (!got) {                 // a slice that is late may still send: one more limit for its copies to land before this memory is given up
          if (lane == 0) atomicExch(p.status, kStatusTimeoutEpilogue);
          mbar_wait(part_bar + 8 * q, 0, p.wait_ns);
        }
        if (n < p.N && tfull_ok && got) {
          const uint32_t own0 = own + (uint32_t)(slice * rs) * 128u + lane * 4;
          const uint32_t part0 = sPart + (uint32_t)(q * (p.splits - 1) * rs) * 128u + lane * 4;
          T *dst = static_cast<T *>(p.D) + (int64_t)(tile.row0 + slice * rs) * p.N + n;
          if (p.splits == 4) add_slices<4, OUT_DT>(own0, part0, slice, rows, rs, f, p.N, dst);
          else add_slices<2, OUT_DT>(own0, part0, slice, rows, rs, f, p.N, dst);
        }
      }
    }
  }

  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem_base, C::TMEM_COLS);
  }
  // every owner has seen its copies arrive before it reaches this barrier, so no block leaves while a copy still reads from it
  if (p.splits > 1) cluster_sync_relaxed();
}

template <int NT, int OUT_DT>
static int launch_grouped(const CUtensorMap &tx, const CUtensorMap &tw, const grouped::Args &args, int64_t blocks, cudaStream_t stream) {
  using C = grouped::Cfg<NT>;
  auto kern = linear_nvfp4_grouped_kernel<NT, OUT_DT>;
  static PerDevice<int> attr_set;
  int unused = 0;
  if (int e = attr_set.get(&unused, [&](int &v) {
        AC4K_CUDA_TRY(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, C::SMEM_BYTES));
        v = 1;
        return 0;
      }))
    return e;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)blocks);
  cfg.blockDim = dim3(grouped::kThreads);
  cfg.dynamicSmemBytes = C::SMEM_BYTES;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.numAttrs = 1;
  if (args.splits > 1) {
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = args.splits;
    attr[1].val.clusterDim.y = 1;
    attr[1].val.clusterDim.z = 1;
    cfg.numAttrs = 2;
  }
  cfg.attrs = attr;
  AC4K_CUDA_TRY(cudaLaunchKernelEx(&cfg, kern, tx, tw, args));
  return 0;
}

template <int NT>
static int launch_grouped_dt(int d_dtype, const CUtensorMap &tx, const CUtensorMap &tw, const grouped::Args &a, int64_t blocks, cudaStream_t st) {
  switch (d_dtype) {
    case AC4K_DT_BF16: return launch_grouped<NT, AC4K_DT_BF16>(tx, tw, a, blocks, st);
    case AC4K_DT_FP16: return launch_grouped<NT, AC4K_DT_FP16>(tx, tw, a, blocks, st);
    default: return launch_grouped<NT, AC4K_DT_FP32>(tx, tw, a, blocks, st);
  }
}

}  // namespace ac4k

extern "C" int ac4k_linear_nvfp4_grouped(void *D, int d_dtype, const void *A, const void *A_sf, const float *A_gs, const void *B, const void *B_sf,
                                         const float *B_gs, int b_gs_per_group, const void *bias, int bias_dtype, const int32_t *offsets, int fill,
                                         int64_t M, int64_t groups, int64_t N, int64_t K, ac4k_stream_t stream_) {
  using namespace ac4k;
  if (M < 0 || N < 0 || K < 0 || groups < 0) return fail(AC4K_ERR_SHAPE, "negative dimension");
  if (d_dtype < 0 || d_dtype > 2) return fail(AC4K_ERR_ENUM, "unknown d_dtype %d", d_dtype);
  if (bias && (bias_dtype < 0 || bias_dtype > 2)) return fail(AC4K_ERR_ENUM, "unknown bias_dtype %d", bias_dtype);
  if (M == 0 || N == 0) return 0;
  if (!D) return fail(AC4K_ERR_NULL, "a required pointer is NULL");
  const cudaStream_t stream = static_cast<cudaStream_t>(stream_);
  if (groups == 0) {
    if (fill) AC4K_CUDA_TRY(cudaMemsetAsync(D, 0, (size_t)(M * N) * (d_dtype == AC4K_DT_FP32 ? 4 : 2), stream));
    return 0;
  }
  if (!A || !B || !A_sf || !B_sf || !A_gs || !B_gs || !offsets) return fail(AC4K_ERR_NULL, "a required pointer is NULL");
  if (K == 0 || K % 64 != 0)
    return fail(AC4K_ERR_SHAPE, "K = %lld must be a positive multiple of 64 (the quantiser pads K to 64)", (long long)K);
  if (M > (1 << 30) || N > (1 << 24) || K > (1 << 24) || groups > (1 << 20) || groups * N > (1 << 30)) return fail(AC4K_ERR_SHAPE, "dimension too large");
  auto addr = [](const void *q) { return reinterpret_cast<uintptr_t>(q); };
  if ((addr(A) | addr(B) | addr(A_sf) | addr(B_sf) | addr(D)) & 15) return fail(AC4K_ERR_ALIGN, "A, B, A_sf, B_sf and D must be 16-byte aligned");
  if ((addr(offsets) | addr(A_gs) | addr(B_gs)) & 3 || (bias && (addr(bias) & (bias_dtype == AC4K_DT_FP32 ? 3 : 1))))
    return fail(AC4K_ERR_ALIGN, "a pointer is not aligned to its elements");
  DeviceInfo di;
  if (int e = get_device_info(&di)) return e;
  if (di.cc_major != 10) return fail(AC4K_ERR_DEVICE, "linear_nvfp4_grouped needs an sm_100 device (found sm_%d0)", di.cc_major);
  unsigned int *status = device_status_ptr();
  if (!status) return fail(AC4K_ERR_DEVICE, "cannot resolve the device status word");

  const int64_t used = groups < M ? groups : M;        // groups that can have rows
  const int64_t mean = ceil_div(M, used);
  const int64_t tiles_n = ceil_div(N, 128);
  const int k_tiles = (int)ceil_div(K / 64, grouped::KS);
  // as many slices of K as keep one wave of blocks (two per SM), for tiles of nt rows
  auto slices = [&](int nt) {
    const int64_t all = ragged_max_tiles(M, used, nt) - 2, busy = all < M ? all : M;
    int n = 1;
    if (nt <= 64)
      for (int cand = 4; cand >= 2; cand /= 2)
        if (busy * tiles_n * cand <= 2 * di.sms && k_tiles / cand >= 4) { n = cand; break; }
    while (n > 1 && ceil_div(k_tiles, ceil_div(k_tiles, n)) != n) n /= 2;   // every slice non-empty
    return n;
  };
  // Long groups go to the CTA pairs, but where tiles of 64 rows are so few that K can be cut: 4 groups of 175 rows, 1024 x 8192, take 15.2 us cut and
  // 19.0 in pairs, 2 of 150 11.3 and 18.4, 8 of 125, 512 x 4096, 11.2 and 13.1, 4 of 175, 1024 x 2048, 10.3 both; uncut, 4 of 250, 2048 x 4096,
  // 14.9 and 14.4.
  const int cut = mean > grouped::pair_rows(K) ? slices(64) : 1;
  if (mean > grouped::pair_rows(K) && cut == 1 && grouped_pair_takes(d_dtype, M, groups, N, K))
    return launch_linear_grouped_pair(D, d_dtype, A, A_sf, A_gs, B, B_sf, B_gs, b_gs_per_group ? 1 : 0, bias, bias_dtype, offsets, fill != 0, M, groups, N,
                                      K, di.sms, status, debug_wait_ns() ? debug_wait_ns() : kWaitTimeoutNs, stream);
  // Tiles of twice the mean: a group a little above it would have two, and stream its weights twice (64 groups of 16 rows, 1024 x 4096: 36.1 us in
  // tiles of 16, 34.4 in tiles of 32; 8 groups of 12, 8192 x 4096: 35.6 and 32.0)
  const int nt = mean <= 8 ? 16 : (mean <= 16 ? 32 : (mean <= 64 || cut > 1 ? 64 : 128));
  const int64_t tiles = ragged_max_tiles(M, used, nt);
  const int splits = slices(nt);
  if (tiles * tiles_n * splits > 0x7FFFFFFFLL) return fail(AC4K_ERR_SHAPE, "too many tiles");
  CUtensorMap tx, tw;
  if (int e = make_tmap(A, M, K / 2, nt, &tx)) return e;
  if (int e = make_tmap(B, groups * N, K / 2, 128, &tw)) return e;
  grouped::Args a = {};
  a.sfa = static_cast<const uint8_t *>(A_sf);
  a.sfb = static_cast<const uint8_t *>(B_sf);
  a.D = D;
  a.a_gs = A_gs; a.b_gs = B_gs; a.b_gs_stride = b_gs_per_group ? 1 : 0;
  a.bias = bias; a.bias_dt = bias_dtype;
  a.offsets = offsets;
  a.status = status;
  a.rows = (int)M; a.groups = (int)groups; a.N = (int)N; a.KT = (int)(K / 64);
  a.rows_sfa = (int)align_up(M, 16);
  a.rows_sfb = (int)align_up(N, 16);
  a.tiles_n = (int)tiles_n;
  a.splits = splits;
  a.kt_per_split = (int)ceil_div(k_tiles, splits);
  a.fill = fill != 0;
  a.wait_ns = debug_wait_ns() ? debug_wait_ns() : kWaitTimeoutNs;
  a.dbg = debug_flags();
  const int64_t blocks = tiles * tiles_n * splits;
  switch (nt) {
    case 16: return launch_grouped_dt<16>(d_dtype, tx, tw, a, blocks, stream);
    case 32: return launch_grouped_dt<32>(d_dtype, tx, tw, a, blocks, stream);
    case 64: return launch_grouped_dt<64>(d_dtype, tx, tw, a, blocks, stream);
    default: return launch_grouped_dt<128>(d_dtype, tx, tw, a, blocks, stream);
  }
}
