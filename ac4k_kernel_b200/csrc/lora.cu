// Low-rank adapters of a batch of requests beside a projection that all of them share:
//
//   out[t] = y[t] + scaling[a] * B_a (A_a x[t]),   a = adapters[request of row t], or none: out[t] = y[t]
//
// A row takes 2 R (K + N) operations and, in bf16, 2 K + 4 N bytes: with K = N 2 R / 3 operations a byte, 85 for R = 128 (128 with the second half's two
// MMAs each), where the tensor pipe and the memory meet at 253 (tcgen05; 1.66 PFLOP/s, 6.55 TB/s).  So the work is to read x, y and the adapters once and
// to write out once; what these kernels reach of that is a matter of latency (29 % of the issue slots, tensor pipe 35 % at rank 64).  One launch: a cluster of up to 16 blocks takes a tile of rows of one request.  Each block sums A x over its
// slice of K ("shrink"), the blocks add their sums in order through distributed shared memory (no atomics, the same result each time), and each
// adds B of that to its slice of y's columns ("expand").  Nothing goes through global memory in between, and the second half's first operands
// are on their way while the sums are exchanged.  (As two launches with A x in a workspace: 15.7 us for 64 requests of one token, rank 16,
// 8192 x 8192; 52 us for 4099 rows, rank 64, 4096 x 4096; 89 us for 8192 rows, rank 32, 8192 x 8192.
// Now 13.2, 38 and 81 - 86.)
//
// Both halves use mma.sync (16 x 8 x 16, bf16, fp32 accumulators): the tiles are small and ragged, no operand
// is read twice from global memory by a warp, and what tcgen05 would add, rate, is not what bounds them.  Operands come through
// rings in shared memory (cp.async), x and y each thread's own 16-byte vectors, the adapter's shared by the block: a product's sum may run
// over k in any order, so a thread takes 8 neighbouring k of a row and deals them to the two MMAs of a step of 32 k, the same for both
// operands, and needs no ldmatrix; the columns of the second half are dealt so that the 8 results
// of a thread over four MMAs are neighbours, which it loads from y and stores in vectors.
//
// A x is summed in fp32 and handed over as two bf16 values (16 bits of mantissa together: below the rounding of a 16-bit y), for which the second half
// takes two MMAs; for an fp32 y as three, all of its bits (2000 rows, rank 128, 4096 x 4096: 58 us, with two 51; 8192 rows, rank 32, 8192 x 8192: 179
// both).  They have the sign of A x, and none is zero unless it is (or is below 2^-110): an infinite B gives infinity from each, and not
// 0 * infinity or infinity - infinity, which the formula does not have.
#include "ragged.cuh"
#include "sm100_ptx.cuh"

namespace ac4k {

namespace lora {
static constexpr int kThreads = 128;      // four warps
static constexpr int kMaxRank = 128;
static constexpr int kMaxSlices = 16;     // blocks of a cluster

// Blocks that an SM's 228 KB take (1 KB each is the system's, and the block has some hundred bytes more)
constexpr int blocks_of(int bytes) { return bytes <= 55 * 1024 ? 4 : (bytes <= 74 * 1024 ? 3 : (bytes <= 111 * 1024 ? 2 : 1)); }
// Stages of a ring: as many as leave room for four blocks on an SM; for the adapters of high ranks three or two
constexpr int stages_of(int tm, int rp, int stage) { return (rp <= 32 || (tm == 64 && rp == 64) ? 54 : (rp == 64 || tm == 64 ? 73 : 110)) * 1024 / stage; }

struct Args {
  const uint16_t *x, *a, *b;   // x [rows, K], a [adapters, R, K], b [adapters, N, R]
  const void *y;
  void *out;
  const int32_t *offsets, *adapters;
  const float *scaling;        // or NULL: ones
  int64_t x_stride, y_stride, out_stride;
  int rows, requests, count;   // count: adapters
  int K, N, R;
  int slices;                  // blocks of a cluster
  int k_slice, n_slice;        // K and columns of a block, multiples of a stage's
  bool x_vec, a_vec, b_vec, y_vec;
};

// 16 bytes of shared memory from 8 elements of a row, beginning at element k; zeros at and behind `end`.  Vectors (k and end multiples of 8,
// 16-byte aligned) arrive asynchronously, single elements at once.
__device__ __forceinline__ void stage8(uint32_t dst, const uint16_t *row, int k, int end, bool vec) {
  if (vec) {
    const uint32_t bytes = k < end ? 16u : 0u;
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(bytes ? row + k : row), "r"(bytes) : "memory");
  } else {
    uint32_t w[4] = {0, 0, 0, 0};
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (k + i < end) w[i >> 1] |= (uint32_t)__ldg(row + k + i) << (16 * (i & 1));
    asm volatile("st.shared::cta.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(dst), "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3]) : "memory");
  }
}
__device__ __forceinline__ void stage16(uint32_t dst, const void *src, uint32_t bytes) {      // 16 bytes, those behind the first `bytes` zeros
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void stage_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void stage_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }
__device__ __forceinline__ uint4 lds16(uint32_t addr) {
  uint4 v;
  asm volatile("ld.shared::cta.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(addr) : "memory");
  return v;
}
__device__ __forceinline__ uint2 lds8(uint32_t addr) {
  uint2 v;
  asm volatile("ld.shared::cta.v2.b32 {%0, %1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(addr) : "memory");
  return v;
}
__device__ __forceinline__ uint32_t shared_addr(const void *p) { return static_cast<uint32_t>(__cvta_generic_to_shared(p)); }

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

// Takes a bf16 part off a finite a: its first eight bits, or half of a where it has no more, so that the part and what is left both have a's sign and
// are exact.  Of one that is not finite both are a itself.
__device__ __forceinline__ float take_part(float &a) {
  if (!isfinite(a)) return a;
  float h = __uint_as_float(__float_as_uint(a) & 0xFFFF0000u);
  if (h == a) h = __fmul_rn(a, 0.5f);
  a = __fsub_rn(a, h);
  return h;
}
// a in two bf16 parts, the larger one in the low half: within 2^-16 of it (the rest, at most 2^-7 of a's power of two, is rounded to eight bits, by half
// a step of 2^-8 at most)
__device__ __forceinline__ uint32_t two_parts(float a) {
  const float h = take_part(a);
  return pack_bf16(h, a);
}
// two values in three bf16 parts each, the whole of them: 24 bits by eight at a time
__device__ __forceinline__ void three_parts(float a, float b, uint32_t (&parts)[3]) {
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const float ha = take_part(a), hb = take_part(b);
    parts[i] = pack_bf16(ha, hb);
  }
  parts[2] = pack_bf16(a, b);
}
}  // namespace lora

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
  static __device__ __forceinline__ float put(float v) { return v; }
};

// 8 neighbouring values of a row, the first at column n, into this thread's places of the ring (16 bytes each, kThreads apart); those at and
// behind N: zeros or nothing
template <typename T>
__device__ __forceinline__ void stage_y(uint32_t dst, const T *row, int n, int N, bool live, bool vec) {
  constexpr int PARTS = sizeof(T) / 2;
  if (!live) return;
  if (vec) {
#pragma unroll
    for (int i = 0; i < PARTS; ++i)
      if (n < N) asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst + i * kThreads * 16), "l"(row + n + 8 / PARTS * i) : "memory");
  } else {
    T v[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = n + i < N ? row[n + i] : T(0.0f);
    const uint32_t *w = reinterpret_cast<const uint32_t *>(v);
#pragma unroll
    for (int i = 0; i < PARTS; ++i)
      asm volatile("st.shared::cta.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(dst + i * kThreads * 16), "r"(w[4 * i]), "r"(w[4 * i + 1]), "r"(w[4 * i + 2]),
                   "r"(w[4 * i + 3]) : "memory");
  }
}
template <typename T>
__device__ __forceinline__ void staged_y(uint32_t src, float (&f)[8]) {
  constexpr int PARTS = sizeof(T) / 2;
  uint4 v[PARTS];
#pragma unroll
  for (int i = 0; i < PARTS; ++i) v[i] = lds16(src + i * kThreads * 16);
  Row8<T>::load(v, f);
}
// Columns n, n + step, ... of two rows, 8 neighbouring values at each, the same values bit for bit.  Vectors by batches of loads (one at a time, the rows
// without an adapter held up a call of 4099 rows, rank 16, 4096 x 4096: 31.6 us, so 25.5).
template <typename T>
__device__ __forceinline__ void copy_rows(T *o0, T *o1, const T *y0, const T *y1, bool live0, bool live1, int n, int end, int step, int N, bool vec) {
  if (vec) {
    constexpr int PARTS = sizeof(T) / 2, B = 8 / PARTS;
    for (; n < end; n += B * step) {
      uint4 v[2][B][PARTS];
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int i = 0; i < B; ++i)
#pragma unroll
          for (int q = 0; q < PARTS; ++q)
            if ((h ? live1 : live0) && n + i * step < min(end, N)) v[h][i][q] = __ldcs(reinterpret_cast<const uint4 *>((h ? y1 : y0) + n + i * step) + q);
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int i = 0; i < B; ++i)
#pragma unroll
          for (int q = 0; q < PARTS; ++q)
            if ((h ? live1 : live0) && n + i * step < min(end, N)) reinterpret_cast<uint4 *>((h ? o1 : o0) + n + i * step)[q] = v[h][i][q];
    }
  } else {
    for (; n < end; n += step)
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (n + i < N) {
          if (live0) o0[n + i] = y0[n + i];
          if (live1) o1[n + i] = y1[n + i];
        }
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

namespace lora {
// What a stage of the first half's ring holds.  KW: k of a warp in a stage; TM 64: all warps the same k, TM 16: in turn.
template <int TM, int RP>
struct Shrink {
  static constexpr int KW = (TM == 64 && RP <= 64) || RP <= 16 ? 64 : 32;
  static constexpr int KB = TM == 64 ? KW : 4 * KW;             // k of the block
  static constexpr int PARTS = KB / KW;
  static constexpr int CH = KW / 8;                             // 16-byte chunks of a row
  static constexpr int X_BYTES = kThreads * (KW / 32) * 2 * 16; // each thread its own two rows' chunks
  static constexpr int A_PART = RP * KW * 2;
  static constexpr int STAGE = X_BYTES + PARTS * A_PART;
  static constexpr int D = stages_of(TM, RP, STAGE);
  // chunk c of adapter row r: rows of 8 chunks lie with their halves exchanged in every other row, so that the eight threads of a phase
  // (two rows, four chunks) meet all banks; two rows of 4 chunks do by themselves
  static __device__ __forceinline__ uint32_t a_at(int r, int c) { return (uint32_t)(r * CH + (CH == 8 ? c ^ ((r & 1) << 2) : c)) * 16u; }
};
// What a stage of the second half's ring holds: the rows of B of NC columns, and y's values for each thread's results
template <int TM, int RP, typename T>
struct Expand {
  static constexpr int UNITS = TM == 64 && (RP == 16 || (RP == 32 && sizeof(T) == 2)) ? 2 : 1;      // of 32 columns, for each warp
  static constexpr int NC = (TM == 64 ? 32 : 128) * UNITS;
  static constexpr int CH = RP / 8;
  static constexpr int B_BYTES = NC * RP * 2;
  static constexpr int Y_UNIT = kThreads * (int)sizeof(T) * 8;  // one row's values of a unit
  static constexpr int STAGE = B_BYTES + UNITS * 2 * Y_UNIT;
  // In front of the first stage that may be filled while the sums are exchanged: the block's own sums, and the total in two parts
  static constexpr int SUMS = (TM == 64 ? 1 : 4) * TM * RP * 4, PARTS2 = TM * RP * 4;
  static constexpr int FIRST = (SUMS + PARTS2 + STAGE - 1) / STAGE;
  static constexpr int D0 = stages_of(TM, RP, STAGE);
  static constexpr int D = D0 > FIRST ? D0 : FIRST;
  static constexpr int EARLY = D - FIRST < D - 1 ? D - FIRST : D - 1;             // stages filled that early
  static constexpr int SMEM = D * STAGE > Shrink<TM, RP>::D * Shrink<TM, RP>::STAGE ? D * STAGE : Shrink<TM, RP>::D * Shrink<TM, RP>::STAGE;
  static constexpr int BLOCKS = blocks_of(SMEM);                // on an SM
  static_assert(D >= 2 && Shrink<TM, RP>::D >= 2 && SMEM + 2048 <= 227 * 1024, "a ring has two stages");
  // chunk c of B's row n.  The eight threads of a phase read four chunks of rows n, n + 1: as in Shrink.  Rank 16: sixteen threads read halves
  // of chunks of rows n, n + 1, n + 8, n + 9; pairs of rows change places in every other eight.
  static __device__ __forceinline__ uint32_t b_at(int n, int c) {
    if (RP == 16) return (uint32_t)((n ^ (((n >> 3) & 1) << 1)) * 2 + c) * 16u;
    return (uint32_t)(n * CH + (CH >= 8 ? c ^ ((n & 1) << 2) : c)) * 16u;
  }
};
}  // namespace lora

// A block takes one tile of rows, one slice of K and one of the columns.  TM 64: a warp per 16 rows; TM 16 (a few rows a request): the warps divide
// each stage's k and add their sums, then its columns.  The adapter's rows are shared by the block, x and y by nobody: a
// thread loads just what it feeds to its MMAs and what it adds to its results.
template <int TM, int RP, typename T>
__global__ void __launch_bounds__(lora::kThreads, lora::Expand<TM, RP, T>::BLOCKS)
lora_kernel(const lora::Args p) {
  using namespace lora;
  using S1 = Shrink<TM, RP>;
  using S2 = Expand<TM, RP, T>;
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ RaggedScratch scratch;
  grid_dependency_wait();
  grid_launch_dependents();
  const int slice = p.slices > 1 ? (int)ptx::cluster_ctarank() : 0;
  const RaggedTile tile = ragged_tile<kThreads>(p.offsets, p.requests, p.rows, TM, blockIdx.x / p.slices, &scratch);
  if (tile.group == -2) return;             // (the blocks of a cluster have the same tile)
  const int adapter = adapter_of(p, tile);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int m0 = tile.row0 + (TM == 64 ? warp * 16 : 0), r0 = m0 + g, r1 = m0 + g + 8;
  const bool live0 = r0 < tile.row1, live1 = r1 < tile.row1;
  const int n_first = min(p.N, slice * p.n_slice), n_end = min(p.N, n_first + p.n_slice), column = TM == 64 ? 0 : warp * 32;
  const T *y0 = static_cast<const T *>(p.y) + (int64_t)r0 * p.y_stride, *y1 = y0 + 8 * p.y_stride;
  T *o0 = static_cast<T *>(p.out) + (int64_t)r0 * p.out_stride, *o1 = o0 + 8 * p.out_stride;
  if (adapter < 0) {
    if (p.out == p.y) return;
    copy_rows<T>(o0, o1, y0, y1, live0, live1, n_first + column + 8 * t, n_end, TM == 64 ? 32 : 128, p.N, p.y_vec);     // rows without an adapter
    return;
  }
  const uint32_t base = shared_addr(smem);
  if (TM == 16 && p.b_vec && n_first < n_end)      // the block's rows of B, read by no other tile: on their way to L2 from the start
    ptx::bulk_prefetch_l2_if(threadIdx.x == 0, p.b + ((int64_t)adapter * p.N + n_first) * p.R, (uint32_t)min((n_end - n_first) * p.R * 2ll, 65536ll));
  {
    // ------------------------------------------------------------------ A x over the block's k
    constexpr int NT = RP / 8;
    const int k0 = min(p.K, slice * p.k_slice), k1 = min(p.K, k0 + p.k_slice);
    const uint16_t *x0 = p.x + (int64_t)(live0 ? r0 : tile.row0) * p.x_stride, *x1 = p.x + (int64_t)(live1 ? r1 : tile.row0) * p.x_stride;
    const uint16_t *a = p.a + (int64_t)adapter * p.R * p.K;
    const int part = TM == 64 ? 0 : warp;
    float acc[NT][4];
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
      for (int i = 0; i < 4; ++i) acc[j][i] = 0.0f;
    // A stage, from k on.  In whole vectors a thread has its places worked out once: its two rows of x, and of the adapter one row in every ROWS, which
    // move on by a stage's k each time (worked out anew for each load, a stage of rank 32 took 294 instructions a warp, 16 of them MMAs: 50 us
    // for 8192 x 8192, and the memory idle two thirds of the time).
    constexpr int LOADS = RP * S1::CH * S1::PARTS / kThreads, ROWS = kThreads / S1::CH;
    static_assert(RP % ROWS == 0, "a thread's loads lie in one column of chunks");
    const int a_c = threadIdx.x % S1::CH, a_r = threadIdx.x / S1::CH;
    const uint16_t *xp0 = x0 + k0 + part * S1::KW + 8 * t, *xp1 = x1 + k0 + part * S1::KW + 8 * t;
    const uint16_t *ap = a + (int64_t)a_r * p.K + k0 + a_c * 8;
    const int64_t a_rows = (int64_t)ROWS * p.K;
    const uint32_t x_to = base + threadIdx.x * 16, a_to = base + S1::X_BYTES + S1::a_at(a_r, a_c);
    const uint32_t bytes0 = live0 ? 16 : 0, bytes1 = live1 ? 16 : 0;
    auto fill = [&](uint32_t off, int k) {
      if (p.x_vec && p.a_vec && k + S1::KB <= k1) {
#pragma unroll
        for (int u = 0; u < S1::KW / 32; ++u) {
          stage16(x_to + off + (2 * u) * kThreads * 16, xp0 + u * 32, bytes0);
          stage16(x_to + off + (2 * u + 1) * kThreads * 16, xp1 + u * 32, bytes1);
        }
#pragma unroll
        for (int i = 0; i < LOADS; ++i) {
          const int r = i * ROWS % RP, q = i * ROWS / RP;
          stage16(a_to + off + q * S1::A_PART + r * S1::CH * 16, ap + (r / ROWS) * a_rows + q * S1::KW, a_r + r < p.R ? 16 : 0);
        }
        xp0 += S1::KB;
        xp1 += S1::KB;
        ap += S1::KB;
        return;
      }
#pragma unroll
      for (int u = 0; u < S1::KW / 32; ++u) {
        const int kk = k + part * S1::KW + u * 32 + 8 * t;
        stage8(x_to + off + (2 * u) * kThreads * 16, x0, kk, live0 ? k1 : 0, p.x_vec);
        stage8(x_to + off + (2 * u + 1) * kThreads * 16, x1, kk, live1 ? k1 : 0, p.x_vec);
      }
#pragma unroll 1
      for (int i = threadIdx.x; i < RP * S1::CH * S1::PARTS; i += kThreads) {
        const int q = i / (RP * S1::CH), r = i / S1::CH % RP, c = i % S1::CH;
        stage8(base + off + S1::X_BYTES + q * S1::A_PART + S1::a_at(r, c), a + (int64_t)(r < p.R ? r : 0) * p.K, k + q * S1::KW + c * 8, r < p.R ? k1 : 0, p.a_vec);
      }
    };
    const int steps = (k1 - k0 + S1::KB - 1) / S1::KB;
#pragma unroll
    for (int i = 0; i < S1::D - 1; ++i) {
      if (i < steps) fill(i * S1::STAGE, k0 + i * S1::KB);
      stage_commit();
    }
    uint32_t now = 0, next = (S1::D - 1) * S1::STAGE;         // stages that are read and filled
    const uint32_t x_at = base + threadIdx.x * 16, a_at0 = base + S1::X_BYTES + part * S1::A_PART + S1::a_at(g, t);
    const uint32_t a_at1 = base + S1::X_BYTES + part * S1::A_PART + S1::a_at(g, S1::CH == 8 ? 4 + t : t);
#pragma unroll 1
    for (int i = 0; i < steps; ++i) {
      stage_wait<S1::D - 2>();
      __syncthreads();              // stage i is there for all, and all are done with the one that is filled next
      if (i + S1::D - 1 < steps) fill(next, k0 + (i + S1::D - 1) * S1::KB);
      stage_commit();
#pragma unroll
      for (int u = 0; u < S1::KW / 32; ++u) {
        const uint4 xa = lds16(x_at + now + (2 * u) * kThreads * 16), xb = lds16(x_at + now + (2 * u + 1) * kThreads * 16);
#pragma unroll
        for (int j = 0; j < NT; ++j) {
          const uint4 w = lds16((u ? a_at1 : a_at0) + now + j * 8 * S1::CH * 16);
          mma_bf16(acc[j], xa.x, xb.x, xa.y, xb.y, w.x, w.y);
          mma_bf16(acc[j], xa.z, xb.z, xa.w, xb.w, w.z, w.w);
        }
      }
      now = now + S1::STAGE == S1::D * S1::STAGE ? 0 : now + S1::STAGE;
      next = next + S1::STAGE == S1::D * S1::STAGE ? 0 : next + S1::STAGE;
    }
    // the sums of this slice: [row of the tile][RP], one such array a warp where the warps divide k
    stage_wait<0>();
    __syncthreads();
    float *sums = reinterpret_cast<float *>(smem);
#pragma unroll
    for (int j = 0; j < NT; ++j) {
      float *d = sums + (warp * 16 + g) * RP + 8 * j + 2 * t;
      *reinterpret_cast<float2 *>(d) = make_float2(acc[j][0], acc[j][1]);
      *reinterpret_cast<float2 *>(d + 8 * RP) = make_float2(acc[j][2], acc[j][3]);
    }
  }
  // ------------------------------------------------------------------ the ring of the second half, and what may be loaded already
  const uint16_t *b = p.b + (int64_t)adapter * p.N * p.R;
  // A stage, from column n on; whole vectors of whole columns as in `shrink`
  constexpr int LOADS = S2::NC * S2::CH / kThreads, COLS = kThreads / S2::CH;
  static_assert(S2::NC % COLS == 0, "every thread has its part of a stage");
  const int b_c = threadIdx.x % S2::CH, b_n = threadIdx.x / S2::CH;
  const uint16_t *bp = b + (int64_t)(n_first + b_n) * p.R + b_c * 8;
  const int64_t b_cols = (int64_t)COLS * p.R, b_step = (int64_t)S2::NC * p.R;
  const T *yp0 = y0 + n_first + column + 8 * t, *yp1 = y1 + n_first + column + 8 * t;
  const uint32_t b_to = base + S2::b_at(b_n, b_c), y_to = base + S2::B_BYTES + threadIdx.x * 16, b_bytes = b_c * 8 < p.R ? 16 : 0;
  auto fill = [&](uint32_t off, int n) {
    if (p.b_vec && p.y_vec && n + S2::NC <= p.N) {
#pragma unroll
      for (int i = 0; i < LOADS; ++i) stage16(b_to + off + i * COLS * S2::CH * 16, bp + i * b_cols, b_bytes);
#pragma unroll
      for (int u = 0; u < S2::UNITS; ++u)
#pragma unroll
        for (int h = 0; h < 2; ++h)
          if (h ? live1 : live0) {
#pragma unroll
            for (int q = 0; q < (int)sizeof(T) / 2; ++q)
              stage16(y_to + off + (2 * u + h) * S2::Y_UNIT + q * kThreads * 16, (h ? yp1 : yp0) + 32 * u + q * (16 / (int)sizeof(T)), 16);
          }
      bp += b_step;
      yp0 += S2::NC;
      yp1 += S2::NC;
      return;
    }
#pragma unroll 1
    for (int i = threadIdx.x; i < S2::NC * S2::CH; i += kThreads) {
      const int col = i / S2::CH, c = i % S2::CH;
      const bool in = n + col < p.N;
      stage8(base + off + S2::b_at(col, c), b + (int64_t)(in ? n + col : 0) * p.R, c * 8, in ? p.R : 0, p.b_vec);
    }
#pragma unroll
    for (int u = 0; u < S2::UNITS; ++u) {
      const int col = n + column + 32 * u + 8 * t;
      stage_y<T>(y_to + off + 2 * u * S2::Y_UNIT, y0, col, p.N, live0, p.y_vec);
      stage_y<T>(y_to + off + (2 * u + 1) * S2::Y_UNIT, y1, col, p.N, live1, p.y_vec);
    }
  };
  const int steps = (n_end - n_first + S2::NC - 1) / S2::NC;
  constexpr int kFrom = S2::D - S2::EARLY;             // where the first stage lies: those in front of it hold the sums
#pragma unroll
  for (int i = 0; i < S2::EARLY; ++i) {
    if (i < steps) fill((kFrom + i) * S2::STAGE, n_first + i * S2::NC);
    stage_commit();
  }
  // ------------------------------------------------------------------ the sums of all slices
  // The blocks of the cluster take a share of the values each, add them in the order of the slices, scale and round them to two bf16 parts (a value
  // in the low half of a word, what it leaves in the high one) and write them to every block; as they are where there will be three parts.
  const uint32_t total = base + S2::SUMS;
  {
    constexpr int WARPS = TM == 64 ? 1 : 4;               // sums of a row
    if (p.slices > 1) ptx::cluster_sync();
    else __syncthreads();
    const float scale = p.scaling != nullptr ? __ldg(p.scaling + adapter) : 1.0f;
    const int n = (tile.row1 - tile.row0) * RP;
    for (int i = (slice * kThreads + threadIdx.x) * 4; i < n; i += p.slices * kThreads * 4) {
      float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
      for (int q = 0; q < p.slices; ++q) {
        const uint32_t at = p.slices > 1 ? ptx::map_to_cta(base + i * 4, q) : base + i * 4;
#pragma unroll
        for (int w = 0; w < WARPS; ++w) {
          const float4 d = ptx::ld_shared_cluster_v4f(at + w * 16 * RP * 4);
          v.x += d.x; v.y += d.y; v.z += d.z; v.w += d.w;
        }
      }
      const float f[4] = {v.x, v.y, v.z, v.w};
      uint32_t u[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        // (behind the rank: not 0 * infinity, which is what an infinity in x has left there)
        const float a = i % RP + e < p.R ? __fmul_rn(f[e], scale) : 0.0f;
        u[e] = sizeof(T) == 4 ? __float_as_uint(a) : two_parts(a);
      }
      for (int q = 0; q < p.slices; ++q) {
        const uint32_t at = p.slices > 1 ? ptx::map_to_cta(total + i * 4, q) : total + i * 4;
        ptx::st_shared_cluster_v4u(at, u[0], u[1], u[2], u[3]);
      }
    }
    if (p.slices > 1) ptx::cluster_sync();              // behind this no block touches another's memory
    else __syncthreads();
  }
  // ------------------------------------------------------------------ y + B of the sum over the block's columns
  constexpr int KC = RP / 32 > 0 ? RP / 32 : 1;      // steps of 32 k (one of 16 for rank 16)
  // The parts of A x for this warp's rows: the fragments of a step of 32 k hold k = 8 t + {0, 1}, {2, 3} (first MMA) and {4, 5}, {6, 7} (second);
  // rank 16: k = 4 t + {0, 1}, {2, 3}.  Pair i -> MMA i / 2, k half i % 2; registers {row g, row g + 8} x {k half}
  constexpr int CUTS = sizeof(T) == 4 ? 3 : 2;
  uint32_t part[CUTS][KC][2][4];
  constexpr int PER = RP == 16 ? 4 : 8;
#pragma unroll
  for (int c = 0; c < KC; ++c)
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      uint4 v[PER / 4];
#pragma unroll
      for (int q = 0; q < PER / 4; ++q) {
        v[q] = make_uint4(0, 0, 0, 0);
        if (h ? live1 : live0) v[q] = lds16(total + (uint32_t)((r0 - tile.row0 + 8 * h) * RP + c * 32 + PER * t + 4 * q) * 4u);
        if constexpr (CUTS == 3) {
          uint32_t a[3], b[3];
          three_parts(__uint_as_float(v[q].x), __uint_as_float(v[q].y), a);
          three_parts(__uint_as_float(v[q].z), __uint_as_float(v[q].w), b);
#pragma unroll
          for (int i = 0; i < 3; ++i) { part[i][c][q][h] = a[i]; part[i][c][q][2 + h] = b[i]; }
        } else {
          part[0][c][q][h] = __byte_perm(v[q].x, v[q].y, 0x5410); part[1][c][q][h] = __byte_perm(v[q].x, v[q].y, 0x7632);
          part[0][c][q][2 + h] = __byte_perm(v[q].z, v[q].w, 0x5410); part[1][c][q][2 + h] = __byte_perm(v[q].z, v[q].w, 0x7632);
        }
      }
    }
  __syncthreads();              // all have read the sums: their place is the ring's now
#pragma unroll
  for (int i = S2::EARLY; i < S2::D - 1; ++i) {
    if (i < steps) fill((kFrom + i) % S2::D * S2::STAGE, n_first + i * S2::NC);
    stage_commit();
  }
  uint32_t now = kFrom % S2::D * S2::STAGE, next = (kFrom + S2::D - 1) % S2::D * S2::STAGE;
  uint32_t b_from[4];       // this thread's chunk of each MMA's rows of B (the ring begins at a multiple of 128: chunks 4 further on are 64 bytes apart by a bit)
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int col = column + 8 * (g >> 1) + 2 * j + (g & 1);
    b_from[j] = base + (RP == 16 ? S2::b_at(col, t >> 1) + (t & 1) * 8 : S2::b_at(col, t));
  }
  T *op0 = o0 + n_first + column + 8 * t, *op1 = o1 + n_first + column + 8 * t;
#pragma unroll 1
  for (int i = 0; i < steps; ++i) {
    stage_wait<S2::D - 2>();
    __syncthreads();
    if (i + S2::D - 1 < steps) fill(next, n_first + (i + S2::D - 1) * S2::NC);
    stage_commit();
#pragma unroll
    for (int u = 0; u < S2::UNITS; ++u) {
      const int n = n_first + i * S2::NC + column + 32 * u;
      float acc[4][4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
#pragma unroll
        for (int q = 0; q < 4; ++q) acc[j][q] = 0.0f;
        // columns of MMA j: g -> n + 8 (g / 2) + 2 j + g % 2, so that this thread's results (columns 2 t, 2 t + 1 of each) are n + 8 t + 2 j, + 1
        if (RP == 16) {
          const uint2 w = lds8(b_from[j] + now + u * 32 * S2::CH * 16);
#pragma unroll
          for (int i = 0; i < CUTS; ++i) mma_bf16(acc[j], part[i][0][0][0], part[i][0][0][1], part[i][0][0][2], part[i][0][0][3], w.x, w.y);
        } else {
#pragma unroll
          for (int c = 0; c < KC; ++c) {
            const uint4 w = lds16((b_from[j] ^ (S2::CH >= 8 ? (c & 1) * 64 : 0)) + (c >> 1) * 128 + now + u * 32 * S2::CH * 16);
#pragma unroll
            for (int i = 0; i < CUTS; ++i) mma_bf16(acc[j], part[i][c][0][0], part[i][c][0][1], part[i][c][0][2], part[i][c][0][3], w.x, w.y);
#pragma unroll
            for (int i = 0; i < CUTS; ++i) mma_bf16(acc[j], part[i][c][1][0], part[i][c][1][1], part[i][c][1][2], part[i][c][1][3], w.z, w.w);
          }
        }
      }
      const uint32_t y_at = y_to + now + u * 2 * S2::Y_UNIT;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        if (!(h ? live1 : live0)) continue;
        float f[8];
        staged_y<T>(y_at + h * S2::Y_UNIT, f);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          f[2 * j] = __fadd_rn(f[2 * j], acc[j][2 * h]);
          f[2 * j + 1] = __fadd_rn(f[2 * j + 1], acc[j][2 * h + 1]);
        }
        if (p.y_vec && i + 1 < steps) Row8<T>::store((h ? op1 : op0) + 32 * u, f);        // (only the last step may pass N)
        else store_y<T>(h ? o1 : o0, n + 8 * t, p.N, p.y_vec, f);
      }
    }
    op0 += S2::NC;
    op1 += S2::NC;
    now = now + S2::STAGE == S2::D * S2::STAGE ? 0 : now + S2::STAGE;
    next = next + S2::STAGE == S2::D * S2::STAGE ? 0 : next + S2::STAGE;
  }
}

namespace lora {
struct Plan {
  int slices, k_slice, n_slice;
  int64_t tiles;
};

// Blocks that are resident at once, by the size of their clusters (a cluster's blocks share a GPC, whose SMs it need not fill)
struct Waves { int of[kMaxSlices + 1]; };

// How a call is cut, from its sizes and the device alone: slices of K and of the columns, as many blocks of a cluster as keep the grid in one wave (75
// tiles of rank 64 in clusters of 8, four more than there was room for, took 42 us, in clusters of 7 38 us) and 512 of K and N together in a block.
// More than the 8 blocks that every GPC has room for where they are at most one an SM: one token, rank 128, 8192 x 8192 takes 11.0 us in a cluster of
// 16 and 14.7 in one of 8, 200 tokens, rank 32, 4096 x 4096 9.5 and 12.1; with more blocks 32 tokens, rank 16, 8192 x 8192 took 11.7 and 9.6.
static Plan plan_of(int64_t rows, int64_t requests, int64_t K, int64_t N, int tm, int kb, int nc, const Waves &waves, int sms) {
  Plan pl;
  pl.tiles = ragged_max_tiles(rows, requests, tm);
  const int64_t busy = pl.tiles - 2 < rows ? pl.tiles - 2 : rows;        // tiles of requests: at most the bound less the two of none
  pl.slices = 1;
  for (int s = 2; s <= kMaxSlices; ++s)
    if (busy * s <= (s > 8 && waves.of[s] > sms ? sms : waves.of[s]) && K + N >= 512 * s) pl.slices = s;
  pl.k_slice = (int)align_up(ceil_div(K, pl.slices), kb);
  pl.n_slice = (int)align_up(ceil_div(N, pl.slices), nc);
  return pl;
}

template <int TM, int RP, typename T>
static int launch_lora(Args p, int sms, cudaStream_t stream) {
  using C = Expand<TM, RP, T>;
  auto kern = lora_kernel<TM, RP, T>;
  cudaLaunchConfig_t cfg = {};
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = C::SMEM;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  cfg.attrs = attr;
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  // once per device: the shared-memory attribute, and how many clusters of each size can be resident at once
  static PerDevice<Waves> once;
  Waves waves;
  if (int e = once.get(&waves, [&](Waves &v) {
        AC4K_CUDA_TRY(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, C::SMEM));
        AC4K_CUDA_TRY(cudaFuncSetAttribute(kern, cudaFuncAttributeNonPortableClusterSizeAllowed, 1));
        cfg.numAttrs = 1;
        for (int s = 2; s <= kMaxSlices; ++s) {
          int n = 0;
          cfg.gridDim = dim3((unsigned)(sms * C::BLOCKS / s * s));
          attr[0].val.clusterDim.x = s;
          if (cudaOccupancyMaxActiveClusters(&n, kern, &cfg) != cudaSuccess) {        // (a size that this device does not have)
            cudaGetLastError();
            n = 0;
          }
          v.of[s] = n * s;
        }
        return 0;
      }))
    return e;
  const Plan pl = plan_of(p.rows, p.requests, p.K, p.N, TM, Shrink<TM, RP>::KB, C::NC, waves, sms);
  p.slices = pl.slices; p.k_slice = pl.k_slice; p.n_slice = pl.n_slice;
  cfg.gridDim = dim3((unsigned)(pl.tiles * pl.slices));
  attr[0].val.clusterDim.x = pl.slices;
  cfg.numAttrs = 2;
  AC4K_CUDA_TRY(cudaLaunchKernelEx(&cfg, kern, p));
  return 0;
}

template <int TM, int RP>
static int launch_dtype(const Args &p, int dt, int sms, cudaStream_t stream) {
  if (dt == AC4K_DT_BF16) return launch_lora<TM, RP, __nv_bfloat16>(p, sms, stream);
  if (dt == AC4K_DT_FP16) return launch_lora<TM, RP, __half>(p, sms, stream);
  return launch_lora<TM, RP, float>(p, sms, stream);
}
template <int TM>
static int launch_tm(const Args &p, int dt, int sms, cudaStream_t stream) {
  if (p.R <= 16) return launch_dtype<TM, 16>(p, dt, sms, stream);
  if (p.R <= 32) return launch_dtype<TM, 32>(p, dt, sms, stream);
  if (p.R <= 64) return launch_dtype<TM, 64>(p, dt, sms, stream);
  return launch_dtype<TM, 128>(p, dt, sms, stream);
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

extern "C" int ac4k_lora(void *out, const void *y, int y_dtype, const void *x, const void *a, const void *b, const int32_t *offsets,
                         const int32_t *adapters, const float *scaling, int64_t rows, int64_t requests, int64_t n_adapters,
                         int64_t K, int64_t N, int64_t R, int64_t x_stride, int64_t y_stride, int64_t out_stride,
                         ac4k_stream_t stream_) {
  using namespace ac4k;
  if (y_dtype < 0 || y_dtype > 2) return fail(AC4K_ERR_ENUM, "unknown y_dtype %d", y_dtype);
  if (int e = lora::check_sizes(rows, requests, n_adapters, K, N, R)) return e;
  if (x_stride < 0 || y_stride < 0 || out_stride < 0) return fail(AC4K_ERR_SHAPE, "negative stride");
  if (rows == 0 || N == 0) return 0;
  if (rows == 1) { x_stride = K; y_stride = out_stride = N; }         // (what one row's stride is means nothing)
  if (rows > 1 && out_stride < N) return fail(AC4K_ERR_SHAPE, "the rows of out overlap");
  if (!out || !y) return fail(AC4K_ERR_NULL, "a required pointer is NULL");
  const int size = y_dtype == AC4K_DT_FP32 ? 4 : 2;
  auto addr = [](const void *q) { return reinterpret_cast<uintptr_t>(q); };
  if ((addr(y) | addr(out)) & (size - 1)) return fail(AC4K_ERR_ALIGN, "y or out is not aligned to its elements");
  if (out == y ? out_stride != y_stride : rows_overlap(addr(out), out_stride * size, N * size, addr(y), y_stride * size, N * size, rows))
    return fail(AC4K_ERR_SHAPE, "out is y itself or does not overlap it");
  const cudaStream_t stream = static_cast<cudaStream_t>(stream_);
  const bool nothing = n_adapters == 0 || requests == 0 || K == 0 || R == 0;       // no adapter adds anything: y's rows as they are
  if (nothing) {
    if (rows > 1 && y_stride < N && y_stride != 0) return fail(AC4K_ERR_SHAPE, "the rows of y overlap");
    if (out == y) return 0;
    if (y_stride >= N && (y_stride > out_stride ? y_stride : out_stride) * size <= INT32_MAX) {       // (the longest pitch that there is)
      AC4K_CUDA_TRY(cudaMemcpy2DAsync(out, (size_t)(out_stride * size), y, (size_t)(y_stride * size), (size_t)(N * size), (size_t)rows,
                                      cudaMemcpyDeviceToDevice, stream));
      return 0;
    }
    requests = K = R = 0;         // one row of y for all, or rows far apart: the kernel's copy of rows of no request
  } else {
    if (!x || !a || !b || !offsets || !adapters) return fail(AC4K_ERR_NULL, "a required pointer is NULL");
    if (((addr(x) | addr(a) | addr(b)) & 1) || ((addr(offsets) | addr(adapters) | addr(scaling)) & 3)) return fail(AC4K_ERR_ALIGN, "a pointer is not aligned to its elements");
    // (the columns of a row are written while other blocks still read their x)
    if (rows_overlap(addr(out), out_stride * size, N * size, addr(x), x_stride * 2, K * 2, rows)) return fail(AC4K_ERR_SHAPE, "out overlaps x");
  }
  DeviceInfo di;
  if (int e = get_device_info(&di)) return e;
  lora::Args p = {};
  p.x = static_cast<const uint16_t *>(x); p.a = static_cast<const uint16_t *>(a); p.b = static_cast<const uint16_t *>(b);
  p.y = y; p.out = out;
  p.offsets = offsets; p.adapters = adapters; p.scaling = scaling;
  p.x_stride = x_stride; p.y_stride = y_stride; p.out_stride = out_stride;
  p.rows = (int)rows; p.requests = (int)requests; p.count = (int)n_adapters;
  p.K = (int)K; p.N = (int)N; p.R = (int)R;
  // 16-byte vectors: whole ones in every row, and rows that begin on one
  p.x_vec = K % 8 == 0 && x_stride % 8 == 0 && (addr(x) & 15) == 0;
  p.a_vec = K % 8 == 0 && (addr(a) & 15) == 0;
  p.b_vec = R % 8 == 0 && (addr(b) & 15) == 0;
  const int lanes = 16 / size;
  p.y_vec = N % 8 == 0 && y_stride % lanes == 0 && out_stride % lanes == 0 && ((addr(y) | addr(out)) & 15) == 0;
  // Tiles of 64 rows where a request has 32 or more on average, else of 16.  (The lengths are on the device.  A long request among short ones goes
  // in tiles of 16, which read its adapter anew each: 2000 rows and 127 of one, 4096 x 4096, 20.8 us at rank 16 and 50.7 at rank 64; in two calls, 11.0 + 15.8
  // and 20.8 + 24.3, so at rank 64 two are faster.)
  if (rows >= 32 * requests) return lora::launch_tm<64>(p, y_dtype, di.sms, stream);
  return lora::launch_tm<16>(p, y_dtype, di.sms, stream);
}
