// NVFP4 products with a weight per group of rows (linear_nvfp4_grouped.cu), for groups that are long enough to fill tiles of 256 rows: the
// CTA-pair kernel (linear_nvfp4_2cta.cu) with the tiles of all groups in one list.
//
// Persistent CTA pairs over 256 x 256 tiles; A rows (the activations) are the M side, B rows (one group's weights) the N side.  The tiles go by
// group, then as in the plain kernel.  How many row tiles each group has follows from the offsets, which only the device knows: every CTA
// builds a table of their running sums (of 128 ranges of groups) and each role finds its tile's group there.
//
// Scales come in the row layout by TMA, the operands' rows in the order 4 l + q -> q * 32 + l, as in the plain kernel.  A box of scales begins at a
// multiple of four rows, so a group's first tile begins up to three rows early and its last one ends late: rows of other groups are
// multiplied with this group's weight there and not stored.  (Narrower or shifted tiles would need the scales re-ordered by threads, which
// costs the tensor pipe 12 - 30 % of every stage.)
//
// Large groups are bound as the plain kernel is, by the tensor pipe and by power.  16384 rows, 8192 x 4096, calls one after another (1000 W, SM clock 1390
// to 1510 MHz): 274 us for 8 even groups, 285 for uneven ones, 262 for `linear` with one weight; a call by itself at 1965 MHz 235, 244 and 242.  The tensor
// pipe is busy 67 % of the cycles (64 % in `linear`), L2 44 %.  Uneven groups end in row tiles that other groups' rows fill up: 4 %.
// Short groups are bound by such tiles: 4099 rows of 48 groups, 2048 x 2048, 39.5 us, are 385 tiles for rows that fill 129, 5.2 rounds run as 6; a stage
// (58 KB to a pair) takes 700 to 1000 cycles where its MMAs take 520.
#include "linear_nvfp4_pair.cuh"

namespace ac4k {
using namespace ptx;

namespace grouped_pair {
using pair::KS;
using pair::STAGES;
using Tile = pair::Tile<256>;
static constexpr int kRanges = 128;                       // ranges of groups in the table
static constexpr int kListed = 48;                        // tiles of a pair whose places are worked out at the start
static constexpr int LIST_BYTES = kListed * 24;
static constexpr int SMEM_BYTES = Tile::SMEM_BYTES - 8 * pair::OUT_STAGE_BYTES /* no tile goes out through shared memory */ + (kRanges + 4) * 4 + LIST_BYTES;
static_assert(SMEM_BYTES <= 227 * 1024, "shared memory overflow");

struct Args {
  void *D;
  const float *a_gs, *b_gs;
  int b_gs_stride;
  const void *bias;              // [groups][N] or NULL
  int bias_dt;
  const int32_t *offsets;
  unsigned int *status;
  int rows, groups, N, KT;
  int tiles_n, per;              // per: groups of a range
  int row_classes;               // classes row % 4 of A in the first of its two maps (4: one map)
  bool fill;
  bool wide;                     // rows of D begin on 32 bytes
  unsigned long long wait_ns;
  int dbg;                       // experiment switches (builds with -DAC4K_DEBUG_HOOKS), else 0
};

struct TileOf {
  int group, row0, row1;         // the group's rows
  int m0, n0;                    // the tile's first row and column
  float alpha;
};

__device__ __forceinline__ int bound_of(const Args &p, int g) { return min(max(__ldg(p.offsets + g), 0), p.rows); }
__device__ __forceinline__ int row_tiles(int lo, int hi) { return hi > lo ? (hi - (lo & ~3) + pair::BMP - 1) / pair::BMP : 0; }

// tile t of the list; `sums`: row tiles in front of each range
__device__ __forceinline__ TileOf tile_of(const Args &p, const volatile int *sums, int t) {
  int r = 0;
#pragma unroll
  for (int step = kRanges / 2; step > 0; step >>= 1)
    if (sums[r + step] * p.tiles_n <= t) r += step;
  int before = sums[r], g = r * p.per, lo = bound_of(p, g), hi = bound_of(p, g + 1), n = row_tiles(lo, hi);
  while ((before + n) * p.tiles_n <= t) {                 // (t is within the range: this ends in front of its last group)
    before += n;
    ++g;
    lo = hi;
    hi = bound_of(p, g + 1);
    n = row_tiles(lo, hi);
  }
  int tm, tn;
  tile_coords(t - before * p.tiles_n, n, p.tiles_n, tm, tn);
  return TileOf{g, lo, hi, (lo & ~3) + tm * pair::BMP, tn * Tile::BN, __fmul_rn(__ldg(p.a_gs), __ldg(p.b_gs + g * p.b_gs_stride))};
}
// the pair's tile number i, t in the list of all
__device__ __forceinline__ TileOf listed_tile(const Args &p, const volatile int *sums, const TileOf *list, int i, int t) {
  return i < kListed ? list[i] : tile_of(p, sums, t);
}
}  // namespace grouped_pair

template <bool RAGGED, int OUT_DT>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(pair::kThreadsPair, 1)
linear_nvfp4_grouped_2cta_kernel(const __grid_constant__ CUtensorMap tma_a, const __grid_constant__ CUtensorMap tma_a_hi,
                                 const __grid_constant__ CUtensorMap tma_b, const __grid_constant__ CUtensorMap tma_sfa,
                                 const __grid_constant__ CUtensorMap tma_sfb, const grouped_pair::Args p) {
  using namespace pair;
  using namespace grouped_pair;
  using T2 = grouped_pair::Tile;
  using T = typename OutT<OUT_DT>::type;
  constexpr int B_BYTES = T2::B_BYTES, STAGE_TX = T2::STAGE_TX, ACC1_COL = T2::ACC1_COL, SF_COL = T2::SF_COL;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  const uint32_t smem_base = smem_u32(smem_raw);
  if (smem_base & 1023u) {      // (as in the plain kernel)
    if (threadIdx.x == 0) atomicExch(p.status, kStatusSmemAlign);
    return;
  }
  const uint32_t sA = smem_base;
  const uint32_t sB = sA + STAGES * A_BYTES;
  const uint32_t sSFA = sB + STAGES * B_BYTES;
  const uint32_t sSFB = sSFA + STAGES * SFA_BYTES;
  const uint32_t sBias = sSFB + STAGES * SFB_BYTES;    // [8 epilogue warps][128] fp32
  const uint32_t bars = sBias + BIAS_BYTES;
  const uint32_t full_bar = bars;                     // [STAGES] leader: operands and scales of both CTAs are in shared memory
  const uint32_t empty_bar = full_bar + 8 * STAGES;   // [STAGES] both: the MMAs that used the stage are done
  const uint32_t tfull_bar = empty_bar + 8 * STAGES;  // [2] both: accumulator complete
  const uint32_t tempty_bar = tfull_bar + 16;         // [2] leader: 16 epilogue warps drained the accumulator
  const uint32_t shared_free_bar = tempty_bar + 16;   // leader: the 8 warps that own the shared columns have read them
  const uint32_t tmem_slot = shared_free_bar + 8;
  volatile int *sums = reinterpret_cast<volatile int *>(smem_raw + (bars + BAR_BYTES - smem_base));     // [kRanges + 1], then 3 words of scratch
  TileOf *list = reinterpret_cast<TileOf *>(smem_raw + (bars + BAR_BYTES + (kRanges + 4) * 4 - smem_base));
  uint8_t *smem_gen = smem_raw;

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = cluster_ctarank();
  const int cluster_id = blockIdx.x >> 1, num_clusters = gridDim.x >> 1;
  const int k_tiles = (p.KT + KS - 1) / KS;
  const int last_nk = p.KT - (k_tiles - 1) * KS;      // K = 64 steps in the last stage of a tile

  if (threadIdx.x == 0) {
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(full_bar + 8 * s, 1);
      mbar_init(empty_bar + 8 * s, 1);
    }
    for (int a = 0; a < 2; ++a) {
      mbar_init(tfull_bar + 8 * a, 1);
      mbar_init(tempty_bar + 8 * a, 16);        // 8 epilogue warps in each CTA
    }
    mbar_init(shared_free_bar, 8);              // 4 of them in each CTA
    fence_barrier_init();
    prefetch_tmap(&tma_a);
    if (RAGGED) prefetch_tmap(&tma_a_hi);
    prefetch_tmap(&tma_b);
    prefetch_tmap(&tma_sfa);
    prefetch_tmap(&tma_sfb);
  }
  if (warp == 1) {
    tmem_alloc_pair(tmem_slot, kTmemCols);
    tmem_relinquish_pair();
  }
  grid_dependency_wait();
  grid_launch_dependents();
  // the table: row tiles of each range of groups by one thread, then their running sums
  {
    int count = 0, upto = 0;
    if (threadIdx.x < kRanges) {
      const int g0 = min((int)threadIdx.x * p.per, p.groups), g1 = min(g0 + p.per, p.groups);
      int lo = g0 < g1 ? bound_of(p, g0) : 0;
      for (int g = g0; g < g1; ++g) {
        const int hi = bound_of(p, g + 1);
        count += row_tiles(lo, hi);
        lo = hi;
      }
      upto = count;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int v = __shfl_up_sync(0xFFFFFFFFu, upto, o);
        if (lane >= o) upto += v;
      }
      if (lane == 31 && warp < 3) sums[kRanges + 1 + warp] = upto;
    }
    __syncthreads();
    if (threadIdx.x < kRanges) {
      for (int w = 0; w < warp; ++w) upto += sums[kRanges + 1 + w];
      sums[threadIdx.x + 1] = upto;
      if (threadIdx.x == 0) sums[0] = 0;
    }
    __syncthreads();
    // the first tiles' places, all at once (a search of some 1000 cycles, which every role would make in front of every tile)
    const int t = cluster_id + (int)threadIdx.x * num_clusters;
    if (threadIdx.x < kListed && t < sums[kRanges] * p.tiles_n) list[threadIdx.x] = tile_of(p, sums, t);
  }
  tc_fence_before();
  __syncthreads();
  cluster_sync();          // peer's barriers are initialised before anything is signalled remotely
  tc_fence_after();
  const uint32_t tmem_base = *reinterpret_cast<volatile uint32_t *>(smem_gen + (tmem_slot - smem_base));
  const int num_tiles = sums[kRanges] * p.tiles_n;

  if (warp == 0) {
    // ------------------------------------------------------------------ TMA producer
    const uint32_t el = elect_one();
    uint32_t s = 0, ph = 0;
    const uint32_t leader_full0 = map_to_cta(full_bar, 0);
    int ti = 0;
    for (int t = cluster_id; t < num_tiles; t += num_clusters) {
      const TileOf tile = listed_tile(p, sums, list, ti++, t);
      const int m0 = tile.m0 + (int)rank * 128;                             // this CTA's rows of A
      const int nb0 = tile.group * p.N + tile.n0 + (int)rank * T2::B_ROWS;  // this CTA's rows of B
      const int sfb_k0 = tile.group * p.KT;
      // a CTA without a row of the group in its half brings no rows (what its shared memory holds makes rows that are not stored; 64
      // groups of 64 rows, 2048 x 2048: 41.9 -> 41.0 us)
      const bool rows = m0 < tile.row1;
      const uint32_t tx = tile.m0 + 128 < tile.row1 ? 2 * STAGE_TX : 2 * STAGE_TX - A_BYTES - SFA_BYTES;
      const uint32_t el_rows = rows ? el : 0;
      bool ok = true;
      for (int kt = 0; kt < k_tiles; ++kt) {
        ok = warp_all(mbar_wait(empty_bar + 8 * s, ph ^ 1, p.wait_ns));
        if (!ok) break;
        const uint32_t lf = leader_full0 + 8 * s;
        if (AC4K_DBG(p, 256) && kt == 0 && t == cluster_id) {       // wait-expiry test: the first stage of each pair never comes
          if (++s == STAGES) { s = 0; ph ^= 1; }
          continue;
        }
        // the leader announces the bytes of both CTAs; rows and K steps past the end of a tensor arrive as zeros (K steps past the end of
        // this group's as the next one's scales, unused) and count all the same
        if (rank == 0) mbar_arrive_expect_tx_if(el, full_bar + 8 * s, tx);
        tma_load_3d_pair_if(el_rows, sA + s * A_BYTES, &tma_a, kt * BKB, m0 >> 2, 0, lf);
        if (RAGGED) tma_load_3d_pair_if(el_rows, sA + s * A_BYTES + p.row_classes * (32 * BKB), &tma_a_hi, kt * BKB, m0 >> 2, 0, lf);
        tma_load_3d_pair_if(el, sB + s * B_BYTES, &tma_b, kt * BKB, nb0 >> 2, 0, lf);
        tma_load_2d_pair_if(el_rows, sSFA + s * SFA_BYTES, &tma_sfa, m0, kt * KS, lf);
        tma_load_2d_pair_if(el, sSFB + s * SFB_BYTES, &tma_sfb, tile.n0, sfb_k0 + kt * KS, lf);
        tma_load_2d_pair_if(el, sSFB + s * SFB_BYTES + KS * 512, &tma_sfb, tile.n0 + 128, sfb_k0 + kt * KS, lf);
        if (++s == STAGES) { s = 0; ph ^= 1; }
      }
      if (!ok) { if (el) atomicExch(p.status, kStatusTimeoutProducer); break; }
    }
  } else if (warp == 1) {
    // ------------------------------------------------------------------ MMA issuer (leader CTA)
    if (rank == 0) {
      const uint32_t el = elect_one();
      constexpr uint32_t idesc = make_idesc_mxf4nvf4(BMP, T2::BN);
      uint32_t s = 0, ph = 0, ti = 0, acc_phs = 0, shared_ph = 0;
      const uint64_t adesc0 = make_smem_desc(sA, 16, 1024, kSwizzle128B);
      const uint64_t bdesc0 = make_smem_desc(sB, 16, 1024, kSwizzle128B);
      const uint64_t sfadesc0 = make_smem_desc(sSFA, 0, 128, kSwizzleNone);
      const uint64_t sfbdesc0 = make_smem_desc(sSFB, 0, 128, kSwizzleNone);
      bool ok = true;
      for (int t = cluster_id; t < num_tiles && ok; t += num_clusters) {
        // the accumulator has been drained (by the tile before the previous one), and so have the columns that both share
        const uint32_t acc = ti & 1;
        ok = warp_all(mbar_wait(tempty_bar + 8 * acc, ((acc_phs >> acc) & 1) ^ 1, p.wait_ns));
        if (!ok) break;
        acc_phs ^= 1u << acc;
        ok = warp_all(mbar_wait(shared_free_bar, shared_ph ^ 1, p.wait_ns));
        if (!ok) break;
        shared_ph ^= 1;
        tc_fence_after();
        const uint32_t d_tmem = tmem_base + acc * ACC1_COL;
        for (int kt = 0; kt < k_tiles; ++kt) {
          ok = warp_all(mbar_wait(full_bar + 8 * s, ph, p.wait_ns));
          if (!ok) break;
          tc_fence_after();
          const uint32_t t_sf = tmem_base + SF_COL, t_sfb = t_sf + KS * 4;
          const uint64_t adesc = adesc0 + (uint64_t)(s * (A_BYTES >> 4));
          const uint64_t bdesc = bdesc0 + (uint64_t)(s * (B_BYTES >> 4));
          const uint64_t sfadesc = sfadesc0 + (uint64_t)(s * (SFA_BYTES >> 4));
          const uint64_t sfbdesc = sfbdesc0 + (uint64_t)(s * (SFB_BYTES >> 4));
          const int nk = (kt + 1 < k_tiles) ? KS : last_nk;
          if (nk == KS) {
#pragma unroll
            for (int j = 0; j < KS; ++j) {
              tmem_cp_32x128b_warpx4_pair_if(el, t_sf + j * 4, sfadesc + j * 32);
              tmem_cp_32x128b_warpx4_pair_if(el, t_sfb + j * 8, sfbdesc + j * 32);
              tmem_cp_32x128b_warpx4_pair_if(el, t_sfb + j * 8 + 4, sfbdesc + (KS + j) * 32);
            }
#pragma unroll
            for (int j = 0; j < KS; ++j)
              mma_mxf4nvf4_pair_if(el, d_tmem, adesc + 2 * j, bdesc + 2 * j, idesc, t_sf + j * 4, t_sfb + j * 8,
                                   (kt > 0 || j > 0) ? 1u : 0u);
          } else {
            for (int j = 0; j < nk; ++j) {
              tmem_cp_32x128b_warpx4_pair_if(el, t_sf + j * 4, sfadesc + j * 32);
              tmem_cp_32x128b_warpx4_pair_if(el, t_sfb + j * 8, sfbdesc + j * 32);
              tmem_cp_32x128b_warpx4_pair_if(el, t_sfb + j * 8 + 4, sfbdesc + (KS + j) * 32);
            }
            for (int j = 0; j < nk; ++j)
              mma_mxf4nvf4_pair_if(el, d_tmem, adesc + 2 * j, bdesc + 2 * j, idesc, t_sf + j * 4, t_sfb + j * 8,
                                   (kt > 0 || j > 0) ? 1u : 0u);
          }
          tc_commit_pair_both_if(el, empty_bar + 8 * s, 3);                 // stage free in both CTAs
          if (kt == k_tiles - 1) tc_commit_pair_both_if(el, tfull_bar + 8 * acc, 3);  // accumulator complete in both CTAs
          if (++s == STAGES) { s = 0; ph ^= 1; }
        }
        ++ti;
      }
      if (!ok && el) atomicExch(p.status, kStatusTimeoutMma);
    }
  } else if (warp < 6) {
    // ------------------------------------------------------------------ rows of no group: zeros (in a new output)
    if (p.fill) {
      const int first = bound_of(p, 0), last = max(bound_of(p, p.groups), first), vectors = p.N / 8;
      const int64_t rest = (int64_t)(p.rows - (last - first)) * vectors;
      for (int64_t i = (int64_t)blockIdx.x * 128 + (threadIdx.x - 64); i < rest; i += (int64_t)gridDim.x * 128) {
        const int64_t r = i / vectors;
        reinterpret_cast<uint4 *>(p.D)[(r < first ? r : r + (last - first)) * vectors + i % vectors] = make_uint4(0, 0, 0, 0);
      }
    }
  } else {
    // ------------------------------------------------------------------ epilogue (warps 6-13)
    // As in the plain kernel: two warps per tensor-memory lane quarter, 128 columns each; drain, * alpha, + bias, pack in registers, hand
    // the accumulator back, then store.
    const int q = warp & 3;
    const int half = warp >= 10 ? 1 : 0;
    uint32_t acc_phs = 0;
    int ti = 0;
    const bool has_bias = p.bias != nullptr;
    const uint32_t leader_tempty = map_to_cta(tempty_bar, 0);
    const uint32_t leader_shared_free = map_to_cta(shared_free_bar, 0);
    const uint32_t bias_s = sBias + (uint32_t)(half * 4 + q) * 512u;
    for (int t = cluster_id; t < num_tiles; t += num_clusters) {
      const TileOf tile = listed_tile(p, sums, list, ti, t);
      const float alpha = tile.alpha;
      const int col0 = tile.n0 + half * 128;
      const uint32_t acc = ti & 1;
      const uint32_t t_row = tmem_base + ((uint32_t)(q * 32) << 16) + acc * ACC1_COL + half * 128;
      if (has_bias) {
        float b4[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int n = col0 + lane * 4 + i;
          b4[i] = 0.0f;
          if (n < p.N) {
            const int64_t at = (int64_t)tile.group * p.N + n;
            b4[i] = p.bias_dt == AC4K_DT_BF16 ? __bfloat162float(static_cast<const __nv_bfloat16 *>(p.bias)[at])
                    : p.bias_dt == AC4K_DT_FP16 ? __half2float(static_cast<const __half *>(p.bias)[at]) : static_cast<const float *>(p.bias)[at];
          }
        }
        st_shared_v4f(bias_s + lane * 16, b4[0], b4[1], b4[2], b4[3]);
        __syncwarp();
      }
      if (!mbar_wait(tfull_bar + 8 * acc, (acc_phs >> acc) & 1, p.wait_ns)) { if (lane == 0) atomicExch(p.status, kStatusTimeoutEpilogue); break; }
      __syncwarp();
      acc_phs ^= 1u << acc;
      tc_fence_after();
      uint32_t w[64];
      // the columns both accumulators share are the first 48 of accumulator 1's columns 0 - 127 and the last 48 of
      // accumulator 0's columns 128 - 255: the first two steps cover them
      const bool shared = half != (int)acc;
      if (shared && half == 1) {
        if (has_bias) drain_permuted<OUT_DT, true, 3, 2, 0, 1>(w, t_row, true, alpha, bias_s, lane, leader_shared_free);
        else drain_permuted<OUT_DT, false, 3, 2, 0, 1>(w, t_row, true, alpha, bias_s, lane, leader_shared_free);
      } else {
        if (has_bias) drain_permuted<OUT_DT, true, 0, 1, 2, 3>(w, t_row, shared, alpha, bias_s, lane, leader_shared_free);
        else drain_permuted<OUT_DT, false, 0, 1, 2, 3>(w, t_row, shared, alpha, bias_s, lane, leader_shared_free);
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive_cluster(leader_tempty + 8 * acc);
      // This warp's lane l holds row m0 + 4 l + q, 256 bytes of it: stored as they are, a whole sector of a row at a time.  (Through shared memory, for whole
      // lines, the tile's stores took 3000 cycles beside the operands that come and go there.)
      const int row = tile.m0 + (int)rank * 128 + q + 4 * lane;
      if (row >= tile.row0 && row < tile.row1) {
        T *out = static_cast<T *>(p.D) + (int64_t)row * p.N + col0;
#pragma unroll
        for (int c = 0; c < 8; ++c) {
          const uint32_t *v = w + 8 * c;
          if (p.wide && col0 + 16 * c + 16 <= p.N) {
            asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(out + 16 * c), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]),
                         "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]) : "memory");
          } else {
            if (col0 + 16 * c < p.N) *reinterpret_cast<uint4 *>(out + 16 * c) = make_uint4(v[0], v[1], v[2], v[3]);
            if (col0 + 16 * c + 8 < p.N) *reinterpret_cast<uint4 *>(out + 16 * c + 8) = make_uint4(v[4], v[5], v[6], v[7]);
          }
        }
      }
      ++ti;
    }
  }

  tc_fence_before();
  __syncthreads();
  cluster_sync_relaxed();  // neither CTA leaves while the other may still read its memory or barriers (nothing is handed over)
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc_pair(tmem_base, kTmemCols);
  }
}

template <bool RAGGED, int OUT_DT>
static int launch_grouped_pair(const CUtensorMap &ta, const CUtensorMap &ta_hi, const CUtensorMap &tb, const CUtensorMap &tsa, const CUtensorMap &tsb,
                               const grouped_pair::Args &args, int64_t most_tiles, int sms, cudaStream_t stream) {
  auto kern = linear_nvfp4_grouped_2cta_kernel<RAGGED, OUT_DT>;
  // once per device: the shared-memory attribute, and how many CTA pairs can be resident at once
  static PerDevice<int> max_clusters;
  int clusters = 0;
  if (int e = max_clusters.get(&clusters, [&](int &v) {
        AC4K_CUDA_TRY(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, grouped_pair::SMEM_BYTES));
        cudaLaunchConfig_t cfg = {};
        cfg.gridDim = dim3(sms & ~1);
        cfg.blockDim = dim3(pair::kThreadsPair);
        cfg.dynamicSmemBytes = grouped_pair::SMEM_BYTES;
        cudaLaunchAttribute attr;
        attr.id = cudaLaunchAttributeClusterDimension;
        attr.val.clusterDim.x = 2;
        attr.val.clusterDim.y = 1;
        attr.val.clusterDim.z = 1;
        cfg.attrs = &attr;
        cfg.numAttrs = 1;
        int n = 0;
        AC4K_CUDA_TRY(cudaOccupancyMaxActiveClusters(&n, kern, &cfg));
        if (n < 1) return fail(AC4K_ERR_DEVICE, "no CTA pair of the GEMM kernel fits on this device");
        v = n;
        return 0;
      }))
    return e;
  if (most_tiles < clusters) clusters = (int)most_tiles;
  return launch_kernel<true>(kern, dim3(2 * clusters), pair::kThreadsPair, grouped_pair::SMEM_BYTES, stream, ta, ta_hi, tb, tsa, tsb, args);
}

bool grouped_pair_takes(int d_dtype, int64_t M, int64_t groups, int64_t N, int64_t K) {
  if (d_dtype == AC4K_DT_FP32 || N % 8 != 0 || N <= 128) return false;
  // the list's length fits in 32 bits, whatever the offsets are
  return M >= 4 && groups * ceil_div(K, 64) < (1 << 30) &&
         groups * (ceil_div(M, pair::BMP) + 1) < (1ll << 31) / ceil_div(N, grouped_pair::Tile::BN);
}

int launch_linear_grouped_pair(void *D, int d_dtype, const void *A, const void *A_sf, const float *A_gs, const void *B, const void *B_sf,
                               const float *B_gs, int b_gs_stride, const void *bias, int bias_dtype, const int32_t *offsets, bool fill, int64_t M,
                               int64_t groups, int64_t N, int64_t K, int sms, unsigned int *status, unsigned long long wait_ns, cudaStream_t stream) {
  CUtensorMap ta, ta_hi, tb, tb_hi, tsa, tsb;
  if (int e = make_tmap_rows4(A, M, K / 2, &ta, &ta_hi)) return e;
  if (int e = make_tmap_rows4(B, groups * N, K / 2, &tb, &tb_hi)) return e;      // (a multiple of four rows: one map)
  if (int e = make_tmap_sf_rows(A_sf, align_up(M, 16), K / 64, &tsa)) return e;
  if (int e = make_tmap_sf_rows(B_sf, align_up(N, 16), groups * (K / 64), &tsb)) return e;
  grouped_pair::Args a = {};
  a.D = D;
  a.a_gs = A_gs; a.b_gs = B_gs; a.b_gs_stride = b_gs_stride;
  a.bias = bias; a.bias_dt = bias_dtype;
  a.offsets = offsets;
  a.status = status;
  a.rows = (int)M; a.groups = (int)groups; a.N = (int)N; a.KT = (int)(K / 64);
  a.tiles_n = (int)ceil_div(N, grouped_pair::Tile::BN);
  a.per = (int)ceil_div(groups, grouped_pair::kRanges);
  a.row_classes = M % 4 ? (int)(M % 4) : 4;
  a.fill = fill;
  a.wide = N % 16 == 0 && (reinterpret_cast<uintptr_t>(D) & 31) == 0;
  a.wait_ns = wait_ns;
  a.dbg = debug_flags();
  if (a.row_classes == 4) ta_hi = ta;
  // row tiles of a group of n rows that begins up to three rows early: at most (n + 3) / 256 + 1
  const int64_t used = groups < M ? groups : M, most = (ceil_div(M + 3 * used, pair::BMP) + used) * a.tiles_n;
  if (d_dtype == AC4K_DT_BF16)
    return a.row_classes < 4 ? launch_grouped_pair<true, AC4K_DT_BF16>(ta, ta_hi, tb, tsa, tsb, a, most, sms, stream)
                             : launch_grouped_pair<false, AC4K_DT_BF16>(ta, ta_hi, tb, tsa, tsb, a, most, sms, stream);
  return a.row_classes < 4 ? launch_grouped_pair<true, AC4K_DT_FP16>(ta, ta_hi, tb, tsa, tsb, a, most, sms, stream)
                           : launch_grouped_pair<false, AC4K_DT_FP16>(ta, ta_hi, tb, tsa, tsb, a, most, sms, stream);
}

}  // namespace ac4k
