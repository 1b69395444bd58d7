// Low-rank adapters of a batch of requests beside a projection that all of them share:
//
//   out[t] = y[t] + scaling[a] * B_a (A_a x[t]),   a = adapters[request of row t], or none: out[t] = y[t]
//
// A rank of 8 to 128 makes 2 R operations per byte of x and of y, below what the memory allows for up to R = 64: the work is to read x, y and the
// adapters once and to write out once.  Two launches: `shrink` leaves A x in fp32 (R values a row), `expand` adds B of it to y.  Both take a
// tile of rows of one request against its adapter with mma.sync (16 x 8 x 16, bf16, fp32 accumulators): the tiles are small and ragged, no operand
// is read twice from global memory by a warp, and what tcgen05 would add, rate, is not what bounds them.  Operands go from global memory
// straight to registers in 16-byte vectors: a product's sum may run over k in any order, so a thread takes 8 neighbouring k of a row and
// deals them to the two MMAs of a step of 32 k, the same for both operands; and the columns of `expand` are dealt so that the 8 results
// of a thread over four MMAs are neighbours, which it loads from y and stores in vectors.
//
// A x is rounded to nothing less than fp32: `expand` splits it into two bf16 values (16 bits of mantissa together) and takes two MMAs.
// With a few rows a request the K dimension of `shrink` is cut into slices, whose sums `expand` adds in order: no atomics, the same result each time.
#include "ragged.cuh"

namespace ac4k {

namespace lora {
static constexpr int kThreads = 128;      // four warps
static constexpr int kMaxRank = 128;

struct Args {
  const uint16_t *x, *a, *b;   // x [rows, K], a [adapters, R, K], b [adapters, N, R]
  const void *y;
  void *out;
  const int32_t *offsets, *adapters;
  const float *scaling;        // or NULL: ones
  float *ws;                   // [slices][rows][RP]
  int64_t x_stride, y_stride, out_stride;
  int rows, requests, count;   // count: adapters
  int K, N, R;
  int slices, k_slice;         // K of a slice, a multiple of the step of a warp's loop
  int n_block;                 // columns of a block of `expand`
  bool x_vec, a_vec, b_vec, y_vec;
};

// 8 elements of a row from `k` on; zeros at and behind `end`
template <bool CS>
__device__ __forceinline__ uint4 load8(const uint16_t *row, int k, int end, bool vec) {
  uint4 v = make_uint4(0, 0, 0, 0);
  if (vec) {
    if (k < end) v = CS ? __ldcs(reinterpret_cast<const uint4 *>(row + k)) : __ldg(reinterpret_cast<const uint4 *>(row + k));
  } else {
    uint32_t w[4] = {0, 0, 0, 0};
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (k + i < end) w[i >> 1] |= (uint32_t)__ldg(row + k + i) << (16 * (i & 1));
    v = make_uint4(w[0], w[1], w[2], w[3]);
  }
  return v;
}

__device__ __forceinline__ void mma_bf16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
               : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// the tile's adapter, -1 for none (and for an index that there is no adapter of)
__device__ __forceinline__ int adapter_of(const Args &p, const RaggedTile &t) {
  if (t.group < 0) return -1;
  const int a = __ldg(p.adapters + t.group);
  return a >= 0 && a < p.count ? a : -1;
}

__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t *>(&h);
}
}  // namespace lora

// A x: a block takes one tile of rows and one slice of K.  TM 64: a warp per 16 rows, all of the slice; TM 16 (a few rows a request): the
// warps divide the slice's K steps, and the block adds their sums.
template <int TM, int RP>
__global__ void __launch_bounds__(lora::kThreads)
lora_shrink_kernel(const lora::Args p) {
  using namespace lora;
  constexpr int NT = RP / 8;
  __shared__ RaggedScratch scratch;
  grid_dependency_wait();
  grid_launch_dependents();
  const RaggedTile tile = ragged_tile<kThreads>(p.offsets, p.requests, p.rows, TM, blockIdx.x, &scratch);
  if (tile.group < 0) return;
  const int adapter = adapter_of(p, tile);
  if (adapter < 0) return;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int m0 = tile.row0 + (TM == 64 ? warp * 16 : 0);
  const int k0 = blockIdx.y * p.k_slice, k1 = min(p.K, k0 + p.k_slice);
  float acc[NT][4];
#pragma unroll
  for (int j = 0; j < NT; ++j)
#pragma unroll
    for (int i = 0; i < 4; ++i) acc[j][i] = 0.0f;
  if (m0 < tile.row1) {
    const int r0 = m0 + g, r1 = m0 + g + 8;
    const uint16_t *x0 = p.x + (int64_t)r0 * p.x_stride, *x1 = p.x + (int64_t)r1 * p.x_stride;
    const int end0 = r0 < tile.row1 ? k1 : 0, end1 = r1 < tile.row1 ? k1 : 0;
    const uint16_t *a = p.a + (int64_t)adapter * p.R * p.K;
    constexpr int U = RP <= 32 ? 4 : 2;          // steps of 32 k whose loads are in flight together
    constexpr int STEP = TM == 64 ? 32 : 32 * 4;
#pragma unroll 1
    for (int k = k0 + (TM == 64 ? 0 : warp * 32); k < k1; k += STEP * U) {
      uint4 xa[U], xb[U], w[U][NT];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int kk = k + u * STEP + 8 * t;
        xa[u] = load8<true>(x0, kk, end0, p.x_vec);
        xb[u] = load8<true>(x1, kk, end1, p.x_vec);
#pragma unroll
        for (int j = 0; j < NT; ++j) {
          const int r = 8 * j + g;
          w[u][j] = load8<false>(a + (int64_t)r * p.K, kk, r < p.R ? k1 : 0, p.a_vec);
        }
      }
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int j = 0; j < NT; ++j) {
          mma_bf16(acc[j], xa[u].x, xb[u].x, xa[u].y, xb[u].y, w[u][j].x, w[u][j].y);
          mma_bf16(acc[j], xa[u].z, xb[u].z, xa[u].w, xb[u].w, w[u][j].z, w[u][j].w);
        }
    }
  }
  float *ws = p.ws + (int64_t)blockIdx.y * p.rows * RP;
  if (TM == 64) {
#pragma unroll
    for (int j = 0; j < NT; ++j) {
      if (m0 + g < tile.row1) *reinterpret_cast<float2 *>(ws + (int64_t)(m0 + g) * RP + 8 * j + 2 * t) = make_float2(acc[j][0], acc[j][1]);
      if (m0 + g + 8 < tile.row1) *reinterpret_cast<float2 *>(ws + (int64_t)(m0 + g + 8) * RP + 8 * j + 2 * t) = make_float2(acc[j][2], acc[j][3]);
    }
  } else {
    __shared__ __align__(16) float sums[4][16][RP];
#pragma unroll
    for (int j = 0; j < NT; ++j) {
      *reinterpret_cast<float2 *>(&sums[warp][g][8 * j + 2 * t]) = make_float2(acc[j][0], acc[j][1]);
      *reinterpret_cast<float2 *>(&sums[warp][g + 8][8 * j + 2 * t]) = make_float2(acc[j][2], acc[j][3]);
    }
    __syncthreads();
    const int n = (tile.row1 - tile.row0) * RP;
    for (int i = threadIdx.x; i < n; i += kThreads) {
      const int m = i / RP, r = i % RP;
      ws[(int64_t)(tile.row0 + m) * RP + r] = (sums[0][m][r] + sums[1][m][r]) + (sums[2][m][r] + sums[3][m][r]);
    }
  }
}

namespace lora {
template <typename T> struct Row8;      // 8 neighbouring values of y
template <> struct Row8<__nv_bfloat16> {
  static __device__ __forceinline__ void load(const void *p, float (&f)[8]) {
    const uint4 v = *reinterpret_cast<const uint4 *>(p);
    const uint32_t u[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) { f[2 * i] = __uint_as_float(u[i] << 16); f[2 * i + 1] = __uint_as_float(u[i] & 0xFFFF0000u); }
  }
  static __device__ __forceinline__ void store(void *p, const float (&f)[8]) {
    *reinterpret_cast<uint4 *>(p) = make_uint4(pack_bf16(f[0], f[1]), pack_bf16(f[2], f[3]), pack_bf16(f[4], f[5]), pack_bf16(f[6], f[7]));
  }
  static __device__ __forceinline__ float get(const __nv_bfloat16 *p) { return __bfloat162float(*p); }
  static __device__ __forceinline__ __nv_bfloat16 put(float v) { return __float2bfloat16_rn(v); }
};
template <> struct Row8<__half> {
  static __device__ __forceinline__ void load(const void *p, float (&f)[8]) {
    const uint4 v = *reinterpret_cast<const uint4 *>(p);
    const uint32_t u[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 d = __half22float2(*reinterpret_cast<const __half2 *>(&u[i]));
      f[2 * i] = d.x; f[2 * i + 1] = d.y;
    }
  }
  static __device__ __forceinline__ void store(void *p, const float (&f)[8]) {
    uint32_t u[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) { const __half2 h = __floats2half2_rn(f[2 * i], f[2 * i + 1]); u[i] = *reinterpret_cast<const uint32_t *>(&h); }
    *reinterpret_cast<uint4 *>(p) = make_uint4(u[0], u[1], u[2], u[3]);
  }
  static __device__ __forceinline__ float get(const __half *p) { return __half2float(*p); }
  static __device__ __forceinline__ __half put(float v) { return __float2half_rn(v); }
};
template <> struct Row8<float> {
  static __device__ __forceinline__ void load(const void *p, float (&f)[8]) {
    const float4 a = reinterpret_cast<const float4 *>(p)[0], b = reinterpret_cast<const float4 *>(p)[1];
    f[0] = a.x; f[1] = a.y; f[2] = a.z; f[3] = a.w; f[4] = b.x; f[5] = b.y; f[6] = b.z; f[7] = b.w;
  }
  static __device__ __forceinline__ void store(void *p, const float (&f)[8]) {
    reinterpret_cast<float4 *>(p)[0] = make_float4(f[0], f[1], f[2], f[3]);
    reinterpret_cast<float4 *>(p)[1] = make_float4(f[4], f[5], f[6], f[7]);
  }
  static __device__ __forceinline__ float get(const float *p) { return *p; }
  static __device__ __forceinline__ float put(float v) { return v; }
};

// 8 neighbouring values of a row, the first at column n: from memory, or as far as they lie in front of N
template <typename T>
__device__ __forceinline__ void load_y(const T *row, int n, int N, bool vec, float (&f)[8]) {
  if (vec) {
    if (n < N) Row8<T>::load(row + n, f);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) if (n + i < N) f[i] = Row8<T>::get(row + n + i);
  }
}
// the same values bit for bit
template <typename T>
__device__ __forceinline__ void copy8(T *out, const T *row, int n, int N, bool vec) {
  if (vec) {
#pragma unroll
    for (int i = 0; i < (int)sizeof(T) / 2; ++i)
      if (n < N) reinterpret_cast<uint4 *>(out + n)[i] = reinterpret_cast<const uint4 *>(row + n)[i];
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) if (n + i < N) out[n + i] = row[n + i];
  }
}
template <typename T>
__device__ __forceinline__ void store_y(T *row, int n, int N, bool vec, const float (&f)[8]) {
  if (vec) {
    if (n < N) Row8<T>::store(row + n, f);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) if (n + i < N) row[n + i] = Row8<T>::put(f[i]);
  }
}
}  // namespace lora

// y + B (A x): a block takes one tile of rows and n_block columns, a warp 16 rows and 32 columns at a time.  TM 64: the warps have 16 rows each,
// the same columns; TM 16: the same rows, columns in turn.
template <int TM, int RP, typename T>
__global__ void __launch_bounds__(lora::kThreads)
lora_expand_kernel(const lora::Args p) {
  using namespace lora;
  constexpr int KC = RP / 32 > 0 ? RP / 32 : 1;      // steps of 32 k (one of 16 for rank 16)
  __shared__ RaggedScratch scratch;
  // The offsets, y and the adapters may be read in front of the wait: the shrink kernel's blocks let this one in behind their own wait, so
  // all that was enqueued before them is complete.
  const RaggedTile tile = ragged_tile<kThreads>(p.offsets, p.requests, p.rows, TM, blockIdx.x, &scratch);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int adapter = tile.group == -2 ? -1 : adapter_of(p, tile);
  const int m0 = tile.row0 + (TM == 64 ? warp * 16 : 0);
  const bool live0 = tile.group != -2 && m0 + g < tile.row1, live1 = tile.group != -2 && m0 + g + 8 < tile.row1;
  const T *y0 = static_cast<const T *>(p.y) + (int64_t)(m0 + g) * p.y_stride, *y1 = y0 + 8 * p.y_stride;
  T *o0 = static_cast<T *>(p.out) + (int64_t)(m0 + g) * p.out_stride, *o1 = o0 + 8 * p.out_stride;
  const int n_first = blockIdx.y * p.n_block + (TM == 64 ? 0 : warp * 32), n_end = min(p.N, (int)(blockIdx.y + 1) * p.n_block);
  constexpr int NSTEP = TM == 64 ? 32 : 128;
  if (tile.group == -2 || adapter < 0) {
    grid_dependency_wait();
    grid_launch_dependents();
    if (tile.group == -2 || p.out == p.y) return;
    for (int n = n_first; n < n_end; n += NSTEP) {     // rows without an adapter
      if (live0) copy8<T>(o0, y0, n + 8 * t, p.N, p.y_vec);
      if (live1) copy8<T>(o1, y1, n + 8 * t, p.N, p.y_vec);
    }
    return;
  }
  grid_dependency_wait();
  grid_launch_dependents();
  if (m0 >= tile.row1) return;
  // A x of this warp's rows, the slices added in order, scaled and split into two bf16 parts: the fragments of a step of 32 k hold
  // k = 8 t + {0, 1}, {2, 3} (first MMA) and {4, 5}, {6, 7} (second); rank 16: k = 4 t + {0, 1}, {2, 3}
  uint32_t hi[KC][2][4], lo[KC][2][4];
  const float scale = p.scaling != nullptr ? __ldg(p.scaling + adapter) : 1.0f;
  constexpr int PER = RP == 16 ? 4 : 8;
#pragma unroll
  for (int c = 0; c < KC; ++c)
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      float v[PER];
#pragma unroll
      for (int i = 0; i < PER; ++i) v[i] = 0.0f;
      if (h ? live1 : live0) {
        const float *w = p.ws + (int64_t)(m0 + g + 8 * h) * RP + c * 32 + PER * t;
        for (int s = 0; s < p.slices; ++s, w += (int64_t)p.rows * RP) {
#pragma unroll
          for (int q = 0; q < PER / 4; ++q) {
            const float4 d = *reinterpret_cast<const float4 *>(w + 4 * q);
            v[4 * q] += d.x; v[4 * q + 1] += d.y; v[4 * q + 2] += d.z; v[4 * q + 3] += d.w;
          }
        }
      }
#pragma unroll
      for (int i = 0; i < PER / 2; ++i) {
        float a[2], b[2];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          // (behind the rank: not 0 * infinity, which is what an infinity in x has left there)
          const float f = c * 32 + PER * t + 2 * i + e < p.R ? __fmul_rn(v[2 * i + e], scale) : 0.0f;
          a[e] = __bfloat162float(__float2bfloat16_rn(f));
          b[e] = isfinite(a[e]) ? __fsub_rn(f, a[e]) : 0.0f;        // (exact)
        }
        // pair i -> MMA i / 2, k half i % 2; registers {row g, row g + 8} x {k half}
        hi[c][i >> 1][2 * (i & 1) + h] = pack_bf16(a[0], a[1]);
        lo[c][i >> 1][2 * (i & 1) + h] = pack_bf16(b[0], b[1]);
      }
    }
  const uint16_t *b = p.b + (int64_t)adapter * p.N * p.R;
#pragma unroll 1
  for (int n = n_first; n < n_end; n += NSTEP) {
    float f0[8] = {}, f1[8] = {};
    if (live0) load_y<T>(y0, n + 8 * t, p.N, p.y_vec, f0);
    if (live1) load_y<T>(y1, n + 8 * t, p.N, p.y_vec, f1);
    float acc[4][4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
#pragma unroll
      for (int i = 0; i < 4; ++i) acc[j][i] = 0.0f;
      // columns of MMA j: g -> n + 8 (g / 2) + 2 j + g % 2, so that this thread's results (columns 2 t, 2 t + 1 of each) are n + 8 t + 2 j, + 1
      const int col = n + 8 * (g >> 1) + 2 * j + (g & 1);
      const uint16_t *row = b + (int64_t)col * p.R;
      if (RP == 16) {
        uint2 w = make_uint2(0, 0);
        if (p.b_vec) {
          if (col < p.N && 4 * t < p.R) w = __ldg(reinterpret_cast<const uint2 *>(row + 4 * t));
        } else if (col < p.N) {
          uint32_t u[2] = {0, 0};
#pragma unroll
          for (int i = 0; i < 4; ++i) if (4 * t + i < p.R) u[i >> 1] |= (uint32_t)__ldg(row + 4 * t + i) << (16 * (i & 1));
          w = make_uint2(u[0], u[1]);
        }
        mma_bf16(acc[j], hi[0][0][0], hi[0][0][1], hi[0][0][2], hi[0][0][3], w.x, w.y);
        mma_bf16(acc[j], lo[0][0][0], lo[0][0][1], lo[0][0][2], lo[0][0][3], w.x, w.y);
      } else {
#pragma unroll
        for (int c = 0; c < KC; ++c) {
          const uint4 w = load8<false>(row, c * 32 + 8 * t, col < p.N ? p.R : 0, p.b_vec);
          mma_bf16(acc[j], hi[c][0][0], hi[c][0][1], hi[c][0][2], hi[c][0][3], w.x, w.y);
          mma_bf16(acc[j], lo[c][0][0], lo[c][0][1], lo[c][0][2], lo[c][0][3], w.x, w.y);
          mma_bf16(acc[j], hi[c][1][0], hi[c][1][1], hi[c][1][2], hi[c][1][3], w.z, w.w);
          mma_bf16(acc[j], lo[c][1][0], lo[c][1][1], lo[c][1][2], lo[c][1][3], w.z, w.w);
        }
      }
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      f0[2 * j] = __fadd_rn(f0[2 * j], acc[j][0]); f0[2 * j + 1] = __fadd_rn(f0[2 * j + 1], acc[j][1]);
      f1[2 * j] = __fadd_rn(f1[2 * j], acc[j][2]); f1[2 * j + 1] = __fadd_rn(f1[2 * j + 1], acc[j][3]);
    }
    if (live0) store_y<T>(o0, n + 8 * t, p.N, p.y_vec, f0);
    if (live1) store_y<T>(o1, n + 8 * t, p.N, p.y_vec, f1);
  }
}

namespace lora {
struct Plan {
  int tm, rp, slices, k_slice, n_block;
  int64_t tiles;
};

// How a call is cut, from its sizes alone.  Tiles of 64 rows where a request has 32 or more on average, else of 16.
static Plan plan_of(int64_t rows, int64_t requests, int64_t K, int64_t N, int64_t R, int sms) {
  Plan pl;
  pl.tm = rows >= 32 * requests ? 64 : 16;
  pl.rp = R <= 16 ? 16 : (R <= 32 ? 32 : (R <= 64 ? 64 : 128));
  pl.tiles = ragged_max_tiles(rows, requests, pl.tm);
  // tiles with rows: at most the bound less the two of no request
  const int64_t busy = pl.tiles - 2 < rows ? pl.tiles - 2 : rows;
  // slices of K: blocks enough for four on an SM, each with a loop of 512 k at least
  const int64_t unit = pl.tm == 64 ? 128 : 512;
  int64_t slices = ceil_div((int64_t)4 * sms, busy);
  const int64_t most = ceil_div(K, 512);
  if (slices > most) slices = most;
  if (slices > 16) slices = 16;
  pl.k_slice = (int)align_up(ceil_div(K, slices), unit);
  pl.slices = (int)ceil_div(K, pl.k_slice);
  // columns of a block: as many as leave eight blocks for an SM, 128 to 1024
  int64_t blocks = ceil_div((int64_t)8 * sms, busy);
  int64_t nb = align_up(ceil_div(N, blocks), 128);
  if (nb > 1024) nb = 1024;
  pl.n_block = (int)nb;
  return pl;
}

template <int TM, int RP>
static int launch_rank(const Args &p, const Plan &pl, int dt, cudaStream_t stream) {
  if (int e = launch_kernel<true>(lora_shrink_kernel<TM, RP>, dim3((unsigned)pl.tiles, (unsigned)pl.slices), kThreads, 0, stream, p)) return e;
  const dim3 grid((unsigned)pl.tiles, (unsigned)ceil_div(p.N, pl.n_block));
  if (dt == AC4K_DT_BF16) return launch_kernel<true>(lora_expand_kernel<TM, RP, __nv_bfloat16>, grid, kThreads, 0, stream, p);
  if (dt == AC4K_DT_FP16) return launch_kernel<true>(lora_expand_kernel<TM, RP, __half>, grid, kThreads, 0, stream, p);
  return launch_kernel<true>(lora_expand_kernel<TM, RP, float>, grid, kThreads, 0, stream, p);
}
template <int TM>
static int launch_tm(const Args &p, const Plan &pl, int dt, cudaStream_t stream) {
  switch (pl.rp) {
    case 16: return launch_rank<TM, 16>(p, pl, dt, stream);
    case 32: return launch_rank<TM, 32>(p, pl, dt, stream);
    case 64: return launch_rank<TM, 64>(p, pl, dt, stream);
    default: return launch_rank<TM, 128>(p, pl, dt, stream);
  }
}

static int check_sizes(int64_t rows, int64_t requests, int64_t adapters, int64_t K, int64_t N, int64_t R) {
  if (rows < 0 || requests < 0 || adapters < 0 || K < 0 || N < 0 || R < 0) return fail(AC4K_ERR_SHAPE, "negative size");
  if (rows > (1 << 30) || requests > (1 << 24) || adapters > (1 << 24) || K > (1 << 24) || N > (1 << 22))
    return fail(AC4K_ERR_SHAPE, "size too large");
  if (R > kMaxRank) return fail(AC4K_ERR_UNSUPPORTED, "rank %lld is above %d", (long long)R, kMaxRank);
  return 0;
}
}  // namespace lora

}  // namespace ac4k

extern "C" int ac4k_lora_workspace(int64_t rows, int64_t requests, int64_t K, int64_t N, int64_t R, int64_t *bytes) {
  using namespace ac4k;
  if (!bytes) return fail(AC4K_ERR_NULL, "bytes is NULL");
  *bytes = 0;
  if (int e = lora::check_sizes(rows, requests, 0, K, N, R)) return e;
  if (rows == 0 || requests == 0 || K == 0 || N == 0 || R == 0) return 0;
  DeviceInfo di;
  if (int e = get_device_info(&di)) return e;
  const lora::Plan pl = lora::plan_of(rows, requests, K, N, R, di.sms);
  *bytes = (int64_t)pl.slices * rows * pl.rp * (int64_t)sizeof(float);
  return 0;
}

extern "C" int ac4k_lora(void *out, const void *y, int y_dtype, const void *x, const void *a, const void *b, const int32_t *offsets,
                         const int32_t *adapters, const float *scaling, void *workspace, int64_t workspace_bytes, int64_t rows, int64_t requests,
                         int64_t n_adapters, int64_t K, int64_t N, int64_t R, int64_t x_stride, int64_t y_stride, int64_t out_stride,
                         ac4k_stream_t stream_) {
  using namespace ac4k;
  if (y_dtype < 0 || y_dtype > 2) return fail(AC4K_ERR_ENUM, "unknown y_dtype %d", y_dtype);
  if (int e = lora::check_sizes(rows, requests, n_adapters, K, N, R)) return e;
  if (x_stride < 0 || y_stride < 0 || out_stride < 0) return fail(AC4K_ERR_SHAPE, "negative stride");
  if (rows == 0 || N == 0) return 0;
  if (rows > 1 && out_stride < N) return fail(AC4K_ERR_SHAPE, "the rows of out overlap");
  if (!out || !y) return fail(AC4K_ERR_NULL, "a required pointer is NULL");
  const int size = y_dtype == AC4K_DT_FP32 ? 4 : 2;
  auto addr = [](const void *q) { return reinterpret_cast<uintptr_t>(q); };
  if ((addr(y) | addr(out)) & (size - 1)) return fail(AC4K_ERR_ALIGN, "y or out is not aligned to its elements");
  const uintptr_t y_end = addr(y) + ((rows - 1) * y_stride + N) * size, o_end = addr(out) + ((rows - 1) * out_stride + N) * size;
  if (out == y ? out_stride != y_stride : (addr(out) < y_end && addr(y) < o_end))
    return fail(AC4K_ERR_SHAPE, "out is y itself or does not overlap it");
  const cudaStream_t stream = static_cast<cudaStream_t>(stream_);
  if (n_adapters == 0 || requests == 0 || K == 0 || R == 0) {       // no adapter adds anything
    if (rows > 1 && y_stride < N) return fail(AC4K_ERR_SHAPE, "the rows of y overlap");
    auto pitch = [&](int64_t stride) { return (size_t)((stride < N ? N : stride) * size); };
    if (out != y) AC4K_CUDA_TRY(cudaMemcpy2DAsync(out, pitch(out_stride), y, pitch(y_stride), (size_t)(N * size), (size_t)rows, cudaMemcpyDeviceToDevice, stream));
    return 0;
  }
  if (!x || !a || !b || !offsets || !adapters) return fail(AC4K_ERR_NULL, "a required pointer is NULL");
  if (((addr(x) | addr(a) | addr(b)) & 1) || ((addr(offsets) | addr(adapters) | addr(scaling)) & 3)) return fail(AC4K_ERR_ALIGN, "a pointer is not aligned to its elements");
  DeviceInfo di;
  if (int e = get_device_info(&di)) return e;
  const lora::Plan pl = lora::plan_of(rows, requests, K, N, R, di.sms);
  if (!workspace || workspace_bytes < (int64_t)pl.slices * rows * pl.rp * (int64_t)sizeof(float))
    return fail(AC4K_ERR_SHAPE, "the workspace is smaller than ac4k_lora_workspace says");
  if (addr(workspace) & 15) return fail(AC4K_ERR_ALIGN, "the workspace is not 16-byte aligned");
  lora::Args p = {};
  p.x = static_cast<const uint16_t *>(x); p.a = static_cast<const uint16_t *>(a); p.b = static_cast<const uint16_t *>(b);
  p.y = y; p.out = out;
  p.offsets = offsets; p.adapters = adapters; p.scaling = scaling;
  p.ws = static_cast<float *>(workspace);
  p.x_stride = x_stride; p.y_stride = y_stride; p.out_stride = out_stride;
  p.rows = (int)rows; p.requests = (int)requests; p.count = (int)n_adapters;
  p.K = (int)K; p.N = (int)N; p.R = (int)R;
  p.slices = pl.slices; p.k_slice = pl.k_slice; p.n_block = pl.n_block;
  // 16-byte vectors (b: 8 bytes of a rank up to 16): whole ones in every row, and rows that begin on one
  p.x_vec = K % 8 == 0 && x_stride % 8 == 0 && (addr(x) & 15) == 0;
  p.a_vec = K % 8 == 0 && (addr(a) & 15) == 0;
  p.b_vec = (R % 8 == 0 || (pl.rp == 16 && R % 4 == 0)) && (addr(b) & 15) == 0;
  const int lanes = 16 / size;
  p.y_vec = N % 8 == 0 && y_stride % lanes == 0 && out_stride % lanes == 0 && ((addr(y) | addr(out)) & 15) == 0;
  if (pl.tm == 64) return lora::launch_tm<64>(p, pl, y_dtype, stream);
  return lora::launch_tm<16>(p, pl, y_dtype, stream);
}
