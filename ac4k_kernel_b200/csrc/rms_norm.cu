// The residual's addition and the RMS norm of a row, written in bf16, in e4m3 with one scale a row, or in NVFP4 (the operand of
// ac4k_linear_nvfp4) with a given global scale:
//
//   s = x + residual,  v = (s * rstd) * weight,  rstd = 1 / sqrt(mean(s^2) + eps)
//   residual' = s rounded to the residual's type;  out = v rounded once
//
// Everything between the loads and the last rounding is fp32: the quantised forms take v itself and not v rounded to bf16, and the norm
// takes s and not the residual that is stored.  What has to be read and written is all there is to it (7 bytes an element with a bf16
// residual and e4m3 out against some ten operations), so a row is read once, held in registers and reduced once: the row's
// maximum of |v|, which the e4m3 scale needs, is rstd times the maximum of |s * weight|, so both reductions share one exchange.
#include "common.cuh"

namespace ac4k {

namespace norm {
enum { kBf16 = AC4K_NORM_BF16, kE4m3 = AC4K_NORM_E4M3, kNvfp4 = AC4K_NORM_NVFP4 };
static constexpr int kMaxCols = 32768;
static constexpr float kE4m3Max = 448.0f;

struct Args {
  const uint16_t *x;
  const void *residual;       // bf16 or fp32, or NULL
  const void *weight;         // bf16 or fp32, or NULL (ones)
  uint8_t *out;
  uint8_t *sf;
  const float *gs;
  uint16_t *normed;           // v in bf16 beside a quantised out, or NULL
  void *residual_out;
  int64_t M, K, x_stride, residual_stride;
  int64_t rows_sf;            // rows of the scale tensor, padding included
  float eps;
  bool residual_f32, weight_f32, tiled;
};

// max that keeps a NaN
__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

// two fp32 operations in one instruction, each rounded as the single one is
__device__ __forceinline__ void add2(float &a, float &b, float c, float d) {
  asm("{\n.reg .b64 p, q;\nmov.b64 p, {%0, %1};\nmov.b64 q, {%2, %3};\nadd.rn.f32x2 p, p, q;\nmov.b64 {%0, %1}, p;\n}" : "+f"(a), "+f"(b) : "f"(c), "f"(d));
}
__device__ __forceinline__ void mul2(float &a, float &b, float c, float d) {
  asm("{\n.reg .b64 p, q;\nmov.b64 p, {%0, %1};\nmov.b64 q, {%2, %3};\nmul.rn.f32x2 p, p, q;\nmov.b64 {%0, %1}, p;\n}" : "+f"(a), "+f"(b) : "f"(c), "f"(d));
}
__device__ __forceinline__ void square_add2(float &a, float &b, float c, float d) {       // a += c * c, b += d * d
  asm("{\n.reg .b64 p, q;\nmov.b64 p, {%0, %1};\nmov.b64 q, {%2, %3};\nfma.rn.f32x2 p, q, q, p;\nmov.b64 {%0, %1}, p;\n}" : "+f"(a), "+f"(b) : "f"(c), "f"(d));
}

__device__ __forceinline__ void unpack8(const uint4 &w, float (&f)[8]) {
  const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    f[2 * i] = __uint_as_float(u[i] << 16);
    f[2 * i + 1] = __uint_as_float(u[i] & 0xFFFF0000u);
  }
}
__device__ __forceinline__ uint4 pack8(const float (&f)[8]) {
  uint32_t u[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(f[2 * i], f[2 * i + 1]);
    u[i] = *reinterpret_cast<const uint32_t *>(&h);
  }
  return make_uint4(u[0], u[1], u[2], u[3]);
}
__device__ __forceinline__ void load8_f32(const float *p, float (&f)[8]) {
  const float4 a = __ldg(reinterpret_cast<const float4 *>(p)), b = __ldg(reinterpret_cast<const float4 *>(p) + 1);
  f[0] = a.x; f[1] = a.y; f[2] = a.z; f[3] = a.w; f[4] = b.x; f[5] = b.y; f[6] = b.z; f[7] = b.w;
}

// 8 weights from column `at` on; ones where there is no weight
__device__ __forceinline__ void weight8(const Args &p, int at, float (&w)[8]) {
  if (p.weight == nullptr) {
#pragma unroll
    for (int i = 0; i < 8; ++i) w[i] = 1.0f;
  } else if (p.weight_f32) {
    load8_f32(static_cast<const float *>(p.weight) + at, w);
  } else {
    unpack8(__ldg(reinterpret_cast<const uint4 *>(static_cast<const uint16_t *>(p.weight) + at)), w);
  }
}

__device__ __forceinline__ float rstd_of(float sum, const Args &p) {
  return __fdiv_rn(1.0f, __fsqrt_rn(__fadd_rn(__fdiv_rn(sum, (float)p.K), p.eps)));
}
// Scale of an e4m3 row with the maximum `amax` of |s * weight|, and the factors that its elements take in front of the weight and behind it.  rstd is in
// an element and in the row's maximum alike, so a code is s * weight times 448 over that maximum: two roundings less than by way of v, half as many
// codes on the other side of a border.  By way of v where that maximum or rstd are beyond what fp32 holds.  A row of zeros has the scale 0 and
// codes 0, and so has one whose largest value is so small (below 2^-117) that the factor would pass fp32's range.
struct RowScale { float scale, pre, r; };
__device__ __forceinline__ RowScale e4m3_scale(float amax, float rstd) {
  const float top = __fmul_rn(amax, rstd);
  RowScale q{__fdiv_rn(top, kE4m3Max), rstd, __fdiv_rn(kE4m3Max, top)};
  if (top < 0x1p-117f) q.scale = q.r = 0.0f;
  else if (amax >= 0x1p-117f && amax < INFINITY && top < INFINITY) { q.pre = 1.0f; q.r = __fdiv_rn(kE4m3Max, amax); }
  return q;
}

// byte offset of the scale word (four blocks of 16) of row `row`, K step `k64`
__device__ __forceinline__ int64_t sf_word(const Args &p, int64_t row, int64_t k64) {
  if (!p.tiled) return (k64 * p.rows_sf + row) * 4;
  return ((row >> 7) * ceil_div(p.K, 64) + k64) * 512 + (row & 31) * 16 + ((row >> 5) & 3) * 4;
}

// Scales of a padding row: zero
template <int FMT>
__device__ __forceinline__ void zero_scales(const Args &p, int64_t row, int t, int threads) {
  if (FMT == kE4m3 && t == 0) reinterpret_cast<float *>(p.sf)[row] = 0.0f;
  if (FMT == kNvfp4)
    for (int64_t k64 = t; k64 < ceil_div(p.K, 64); k64 += threads) *reinterpret_cast<uint32_t *>(p.sf + sf_word(p, row, k64)) = 0u;
}

// (sum, max) over the G threads that share a row; `part`: 2 * (threads / 32) floats of shared memory
template <int G>
__device__ __forceinline__ void reduce_row(float &sum, float &amax, float *part) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    sum += __shfl_xor_sync(0xFFFFFFFFu, sum, o);
    amax = max_nan(amax, __shfl_xor_sync(0xFFFFFFFFu, amax, o));
  }
  if (G > 32) {
    constexpr int W = G / 32;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (lane == 0) { part[warp] = sum; part[W + warp] = amax; }
    __syncthreads();
    sum = lane < W ? part[lane] : 0.0f;
    amax = lane < W ? part[W + lane] : 0.0f;
#pragma unroll
    for (int o = W / 2; o > 0; o >>= 1) {     // (lanes past W hold zeros and are not read by those below)
      sum += __shfl_xor_sync(0xFFFFFFFFu, sum, o);
      amax = max_nan(amax, __shfl_xor_sync(0xFFFFFFFFu, amax, o));
    }
    sum = __shfl_sync(0xFFFFFFFFu, sum, 0);
    amax = __shfl_sync(0xFFFFFFFFu, amax, 0);
  }
}

}  // namespace norm

namespace norm {
// Blocks on an SM that the compiler is to leave registers for: as many rows in flight as a row's 8 C values and its two loads of 4 C words allow.
// Left to itself it took 86 registers for C = 5, and 4099 rows of 5120 (bf16 residual, e4m3 out) 28.3 us, now 27.4; without a residual 20.9 and 19.0; 6144
// 37.0 and 35.2; 12288 69.1 and 62.8.  (8 blocks for C = 5 spill: 29.2.  All back to back, over four inputs in turn; a call among calls on new inputs each
// takes 29.7.)  Bytes and time of the other forms of 4099 x 5120: bf16 out 168 MB 27.6 us, NVFP4 138 MB 26.6; with an fp32 residual e4m3 231 MB 43.6, NVFP4
// 222 MB 47.8.
constexpr int blocks_for(int c, int threads) {
  return c == 8 ? 512 / threads : (c == 6 ? 768 / threads : (c == 5 ? 896 / threads : (c == 4 ? 1024 / threads : 1)));
}
}  // namespace norm

// Rows of 16-byte vectors: G threads share a row (a warp, or the block), C chunks of 8 elements in registers each.
template <int FMT, int G, int C, int THREADS>
__global__ void __launch_bounds__(THREADS, norm::blocks_for(C, THREADS))
rms_norm_kernel(const norm::Args p) {
  using namespace norm;
  static_assert(G == 32 || G == THREADS, "a row per warp or per block");
  __shared__ float part[2 * (THREADS / 32)];
  const int g = threadIdx.x / G, t = threadIdx.x % G;
  const int64_t row = (int64_t)blockIdx.x * (THREADS / G) + g;
  grid_dependency_wait();
  if (row >= p.M) {           // (a whole block where the block shares a row)
    grid_launch_dependents();
    if (row < p.rows_sf) zero_scales<FMT>(p, row, t, G);
    return;
  }
  const int nfull = (int)(p.K / 8);
  float s[C][8];
  if (p.residual != nullptr && !p.residual_f32) {
    // all loads in front of the first use: x and the residual of the whole row are in flight together
    const uint16_t *res = static_cast<const uint16_t *>(p.residual) + row * p.residual_stride;
    uint4 v[C], u[C];
#pragma unroll
    for (int c = 0; c < C; ++c) {
      const int ch = c * G + t;
      v[c] = u[c] = make_uint4(0, 0, 0, 0);
      if (ch < nfull) {
        v[c] = __ldcs(reinterpret_cast<const uint4 *>(p.x + row * p.x_stride + ch * 8));
        u[c] = __ldcs(reinterpret_cast<const uint4 *>(res + ch * 8));
      }
    }
#pragma unroll
    for (int c = 0; c < C; ++c) {
      float r[8];
      unpack8(v[c], s[c]);
      unpack8(u[c], r);
#pragma unroll
      for (int i = 0; i < 8; i += 2) add2(s[c][i], s[c][i + 1], r[i], r[i + 1]);
    }
  } else {
    uint4 v[C];
#pragma unroll
    for (int c = 0; c < C; ++c) {
      const int ch = c * G + t;
      v[c] = make_uint4(0, 0, 0, 0);
      if (ch < nfull) v[c] = __ldcs(reinterpret_cast<const uint4 *>(p.x + row * p.x_stride + ch * 8));
    }
#pragma unroll
    for (int c = 0; c < C; ++c) unpack8(v[c], s[c]);
    if (p.residual != nullptr) {
#pragma unroll
      for (int c = 0; c < C; ++c) {
        const int ch = c * G + t;
        if (ch < nfull) {
          const float4 *q = reinterpret_cast<const float4 *>(static_cast<const float *>(p.residual) + row * p.residual_stride + ch * 8);
          const float4 a = __ldcs(q), b = __ldcs(q + 1);
          const float r[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
#pragma unroll
          for (int i = 0; i < 8; ++i) s[c][i] = __fadd_rn(s[c][i], r[i]);
        }
      }
    }
  }
  grid_launch_dependents();
  float sum = 0.0f, odd = 0.0f, amax = 0.0f;
#pragma unroll
  for (int c = 0; c < C; ++c) {
    const int ch = c * G + t;
    if (p.residual_out != nullptr && ch < nfull) {
      if (p.residual_f32) {
        float4 *d = reinterpret_cast<float4 *>(static_cast<float *>(p.residual_out) + row * p.K + ch * 8);
        d[0] = make_float4(s[c][0], s[c][1], s[c][2], s[c][3]);
        d[1] = make_float4(s[c][4], s[c][5], s[c][6], s[c][7]);
      } else {
        *reinterpret_cast<uint4 *>(static_cast<uint16_t *>(p.residual_out) + row * p.K + ch * 8) = pack8(s[c]);
      }
    }
#pragma unroll
    for (int i = 0; i < 8; i += 2) square_add2(sum, odd, s[c][i], s[c][i + 1]);
    if (FMT == kE4m3 && ch < nfull) {
      float w[8];             // (loaded again behind the reduction: held, they would cost as many registers as the row)
      weight8(p, ch * 8, w);
#pragma unroll
      for (int i = 0; i < 8; i += 2) {
        mul2(w[i], w[i + 1], s[c][i], s[c][i + 1]);
        amax = max_nan(max_nan(amax, fabsf(w[i])), fabsf(w[i + 1]));
      }
    }
  }
  sum = __fadd_rn(sum, odd);
  reduce_row<G>(sum, amax, part);
  const float rstd = rstd_of(sum, p);
  RowScale q = {};
  float alpha = 0.0f;
  if (FMT == kE4m3) {
    q = e4m3_scale(amax, rstd);
    if (t == 0) reinterpret_cast<float *>(p.sf)[row] = q.scale;
  }
  if (FMT == kNvfp4) alpha = load_alpha(p.gs);
  const int64_t Kp = FMT == kBf16 ? p.K : (FMT == kE4m3 ? align_up(p.K, 16) : align_up(p.K, 64));
#pragma unroll
  for (int c = 0; c < C; ++c) {
    const int ch = c * G + t;
    float v[8] = {}, w[8] = {};
    if (ch < nfull) weight8(p, ch * 8, w);
    if (ch < nfull && (FMT != kE4m3 || p.normed != nullptr)) {
#pragma unroll
      for (int i = 0; i < 8; i += 2) {
        v[i] = s[c][i]; v[i + 1] = s[c][i + 1];
        mul2(v[i], v[i + 1], rstd, rstd);
        mul2(v[i], v[i + 1], w[i], w[i + 1]);
      }
    }
    if (FMT == kBf16) {
      if (ch < nfull) *reinterpret_cast<uint4 *>(p.out + (row * p.K + ch * 8) * 2) = pack8(v);
      continue;
    }
    if (p.normed != nullptr && ch < nfull) *reinterpret_cast<uint4 *>(p.normed + row * p.K + ch * 8) = pack8(v);
    if (FMT == kE4m3) {
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = s[c][i];
      if (q.pre != 1.0f)              // (seldom, and the whole row alike)
#pragma unroll
        for (int i = 0; i < 8; i += 2) mul2(v[i], v[i + 1], q.pre, q.pre);
#pragma unroll
      for (int i = 0; i < 8; i += 2) {
        mul2(v[i], v[i + 1], w[i], w[i + 1]);
        mul2(v[i], v[i + 1], q.r, q.r);
      }
      uint2 *d = reinterpret_cast<uint2 *>(p.out + row * Kp + ch * 8);
      if (ch < nfull) *d = make_uint2(f32x4_to_e4m3x4(v[0], v[1], v[2], v[3]), f32x4_to_e4m3x4(v[4], v[5], v[6], v[7]));
      else if (ch * 8 < Kp) *d = make_uint2(0, 0);            // (padding: zeros, whatever the factor of the row)
    }
    if (FMT == kNvfp4) {
      // two neighbouring lanes hold a block of 16, eight a word of four scales (G is a multiple of 8, so they stay in step)
      float m = 0.0f;
#pragma unroll
      for (int i = 0; i < 8; ++i) m = max_nan(m, fabsf(v[i]));
      m = max_nan(m, __shfl_xor_sync(0xFFFFFFFFu, m, 1));
      const BlockScale b = block_scale(m, alpha);
      float y[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) y[i] = __fmul_rn(v[i], b.r);
      uint32_t word = (uint32_t)b.byte << (8 * ((ch >> 1) & 3));
      word |= __shfl_xor_sync(0xFFFFFFFFu, word, 2);
      word |= __shfl_xor_sync(0xFFFFFFFFu, word, 4);
      if (ch * 8 < Kp) {
        *reinterpret_cast<uint32_t *>(p.out + row * (Kp / 2) + ch * 4) = ch < nfull ? f32x8_to_e2m1x8(y) : 0u;
        if ((ch & 7) == 0) *reinterpret_cast<uint32_t *>(p.sf + sf_word(p, row, ch >> 3)) = word;
      }
    }
  }
}

// Any K, stride and alignment: a block of T threads per row, the row as fp32 in shared memory.  x, the residual and outputs of the same width go by single
// elements, neighbours by neighbouring threads, a batch of loads in front of its first use; the quantised row begins on 16 bytes
// and goes by four elements a thread.  Threads by K: 30000 rows of 1001 (bf16 residual, e4m3 out) take 107 us, 299 with 512 threads a row; 9999 rows of
// 11003 take 427 us (1.8 TB/s: seven loads and stores of a warp for every 32 elements), 461 with an element and a code at a time.
template <int FMT, int T>
__global__ void __launch_bounds__(T)
rms_norm_any_kernel(const norm::Args p) {
  using namespace norm;
  extern __shared__ __align__(16) float row_s[];            // [K to 64]
  __shared__ float part[2 * (T / 32)];
  const int t = threadIdx.x;
  const int64_t row = blockIdx.x;
  grid_dependency_wait();
  grid_launch_dependents();
  if (row >= p.M) {
    if (row < p.rows_sf) zero_scales<FMT>(p, row, t, T);
    return;
  }
  const int K = (int)p.K;
  auto weight = [&](int i) {
    if (p.weight == nullptr) return 1.0f;
    return p.weight_f32 ? __ldg(static_cast<const float *>(p.weight) + i) : bf16_bits_to_f32(__ldg(static_cast<const uint16_t *>(p.weight) + i));
  };
  float sum = 0.0f, amax = 0.0f;
  constexpr int U = 8;
  const uint16_t *x = p.x + row * p.x_stride;
  for (int base = t; base < K; base += U * T) {
    uint16_t v[U];
    float r[U];
#pragma unroll
    for (int u = 0; u < U; ++u) v[u] = base + u * T < K ? x[base + u * T] : (uint16_t)0;
    if (p.residual != nullptr) {
      const int64_t at = row * p.residual_stride + base;
#pragma unroll
      for (int u = 0; u < U; ++u) {
        r[u] = 0.0f;
        if (base + u * T < K)
          r[u] = p.residual_f32 ? static_cast<const float *>(p.residual)[at + u * T] : bf16_bits_to_f32(static_cast<const uint16_t *>(p.residual)[at + u * T]);
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int i = base + u * T;
      if (i >= K) break;
      float s = bf16_bits_to_f32(v[u]);
      if (p.residual != nullptr) s = __fadd_rn(s, r[u]);
      if (p.residual_out != nullptr) {          // (the element's own address where this is the residual itself)
        if (p.residual_f32) static_cast<float *>(p.residual_out)[row * p.K + i] = s;
        else static_cast<__nv_bfloat16 *>(p.residual_out)[row * p.K + i] = __float2bfloat16_rn(s);
      }
      sum = __fmaf_rn(s, s, sum);
      if (FMT == kE4m3) amax = max_nan(amax, fabsf(__fmul_rn(s, weight(i))));
      row_s[i] = s;
    }
  }
  reduce_row<T>(sum, amax, part);             // (its barrier is in front of the reads of row_s below)
  const float rstd = rstd_of(sum, p);
  __nv_bfloat16 *wide = reinterpret_cast<__nv_bfloat16 *>(FMT == kBf16 ? static_cast<void *>(p.out) : p.normed);
  if (wide != nullptr) {
    wide += row * p.K;
    for (int i = t; i < K; i += T) wide[i] = __float2bfloat16_rn(__fmul_rn(__fmul_rn(row_s[i], rstd), weight(i)));
  }
  if (FMT == kBf16) return;
  RowScale q = {};
  float alpha = 0.0f;
  if (FMT == kE4m3) {
    q = e4m3_scale(amax, rstd);
    if (t == 0) reinterpret_cast<float *>(p.sf)[row] = q.scale;
  }
  if (FMT == kNvfp4) alpha = load_alpha(p.gs);
  const int Kp = (int)(FMT == kE4m3 ? align_up(K, 16) : align_up(K, 64));
  for (int base = 0; base < Kp; base += 4 * T) {           // (whole warps in step: NVFP4 exchanges among the four lanes of a block of 16)
    const int i = base + 4 * t;
    float v[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    if (i < Kp) {
      const float4 s = *reinterpret_cast<const float4 *>(row_s + i);
      const float f[4] = {s.x, s.y, s.z, s.w};
#pragma unroll
      for (int j = 0; j < 4; ++j) v[j] = i + j < K ? __fmul_rn(__fmul_rn(f[j], FMT == kE4m3 ? q.pre : rstd), weight(i + j)) : 0.0f;
    }
    if (FMT == kE4m3) {
      if (i < Kp) *reinterpret_cast<uint32_t *>(p.out + row * Kp + i) = f32x4_to_e4m3x4(__fmul_rn(v[0], q.r), __fmul_rn(v[1], q.r), __fmul_rn(v[2], q.r), __fmul_rn(v[3], q.r));
    }
    if (FMT == kNvfp4) {
      float m = max_nan(max_nan(fabsf(v[0]), fabsf(v[1])), max_nan(fabsf(v[2]), fabsf(v[3])));
      m = max_nan(m, __shfl_xor_sync(0xFFFFFFFFu, m, 1));
      m = max_nan(m, __shfl_xor_sync(0xFFFFFFFFu, m, 2));
      const BlockScale b = block_scale(m, alpha);
      if (i < Kp) {
        const float y[8] = {__fmul_rn(v[0], b.r), __fmul_rn(v[1], b.r), __fmul_rn(v[2], b.r), __fmul_rn(v[3], b.r), 0.f, 0.f, 0.f, 0.f};
        *reinterpret_cast<uint16_t *>(p.out + row * (Kp / 2) + i / 2) = (uint16_t)f32x8_to_e2m1x8(y);
        if ((i & 15) == 0) p.sf[sf_word(p, row, i >> 6) + ((i >> 4) & 3)] = b.byte;
      }
    }
  }
  // Padding is zeros, whatever the factor of the row (0 * NaN is none): the threads that wrote codes behind K take them back.  (In the loop above, a
  // comparison for every four elements: 30000 rows of 1001 into NVFP4 83.9 -> 87.3 us.)
  const int i = (K & ~3) + 4 * ((t - (K >> 2)) & (T - 1));
  if (i < Kp) {
    if (FMT == kE4m3) {
      uint32_t *d = reinterpret_cast<uint32_t *>(p.out + row * Kp + i);
      *d = i < K ? *d & (0xFFFFFFFFu >> (8 * (i + 4 - K))) : 0u;
    } else {
      uint16_t *d = reinterpret_cast<uint16_t *>(p.out + row * (Kp / 2) + i / 2);
      *d = i < K ? (uint16_t)(*d & (0xFFFFu >> (4 * (i + 4 - K)))) : (uint16_t)0;
    }
  }
}

template <int FMT, int G, int C, int THREADS>
static int launch_norm(const norm::Args &p, int64_t rows, cudaStream_t stream) {
  return launch_kernel<true>(rms_norm_kernel<FMT, G, C, THREADS>, dim3((unsigned)ceil_div(rows, THREADS / G)), THREADS, 0, stream, p);
}

template <int FMT, int T>
static int launch_any(const norm::Args &p, int64_t rows, cudaStream_t stream) {
  static PerDevice<int> attr_set;
  int unused = 0;
  if (int e = attr_set.get(&unused, [&](int &v) {
        AC4K_CUDA_TRY(cudaFuncSetAttribute(rms_norm_any_kernel<FMT, T>, cudaFuncAttributeMaxDynamicSharedMemorySize, norm::kMaxCols * (int)sizeof(float)));
        v = 1;
        return 0;
      }))
    return e;
  return launch_kernel<true>(rms_norm_any_kernel<FMT, T>, dim3((unsigned)rows), T, (size_t)align_up(p.K, 64) * sizeof(float), stream, p);
}

template <int FMT>
static int launch_norm_fmt(const norm::Args &p, bool vectors, cudaStream_t stream) {
  const int64_t rows = p.rows_sf > p.M ? p.rows_sf : p.M;
  const int64_t Kp = FMT == norm::kNvfp4 ? align_up(p.K, 64) : align_up(p.K, 16);
  if (!vectors) {
    if (Kp <= 512) return launch_any<FMT, 64>(p, rows, stream);
    if (Kp <= 1024) return launch_any<FMT, 128>(p, rows, stream);
    if (Kp <= 4096) return launch_any<FMT, 256>(p, rows, stream);
    return launch_any<FMT, 512>(p, rows, stream);
  }
  if (Kp <= 512) return launch_norm<FMT, 32, 2, 128>(p, rows, stream);
  if (Kp <= 1024) return launch_norm<FMT, 32, 4, 128>(p, rows, stream);
  if (Kp <= 2048) return launch_norm<FMT, 128, 2, 128>(p, rows, stream);
  if (rows < 1024) {
    if (Kp <= 4096) return launch_norm<FMT, 256, 2, 256>(p, rows, stream);
    if (Kp <= 8192) return launch_norm<FMT, 512, 2, 512>(p, rows, stream);
    if (Kp <= 16384) return launch_norm<FMT, 1024, 2, 1024>(p, rows, stream);
    return launch_norm<FMT, 1024, 4, 1024>(p, rows, stream);
  }
  if (Kp <= 4096) return launch_norm<FMT, 128, 4, 128>(p, rows, stream);
  if (Kp <= 5120) return launch_norm<FMT, 128, 5, 128>(p, rows, stream);
  if (Kp <= 6144) return launch_norm<FMT, 128, 6, 128>(p, rows, stream);
  if (Kp <= 8192) return launch_norm<FMT, 128, 8, 128>(p, rows, stream);
  if (Kp <= 12288) return launch_norm<FMT, 256, 6, 256>(p, rows, stream);
  if (Kp <= 16384) return launch_norm<FMT, 256, 8, 256>(p, rows, stream);
  return launch_norm<FMT, 512, 8, 512>(p, rows, stream);
}

}  // namespace ac4k

extern "C" int ac4k_rms_norm(void *out, void *sf, const float *global_scale, int precision, int sf_layout, void *normed, void *residual_out,
                             const void *x, const void *residual, int residual_dtype, const void *weight, int weight_dtype, float eps,
                             int64_t M, int64_t K, int64_t x_stride, int64_t residual_stride, ac4k_stream_t stream_) {
  using namespace ac4k;
  if (precision < AC4K_NORM_BF16 || precision > AC4K_NORM_NVFP4) return fail(AC4K_ERR_ENUM, "unknown precision %d", precision);
  if (precision == AC4K_NORM_NVFP4 && sf_layout != AC4K_SF_AC4K && sf_layout != AC4K_SF_TILE128X4)
    return fail(AC4K_ERR_ENUM, "unknown sf_layout %d", sf_layout);
  if (residual && residual_dtype != AC4K_DT_BF16 && residual_dtype != AC4K_DT_FP32) return fail(AC4K_ERR_ENUM, "the residual is bf16 or fp32");
  if (weight && weight_dtype != AC4K_DT_BF16 && weight_dtype != AC4K_DT_FP32) return fail(AC4K_ERR_ENUM, "the weight is bf16 or fp32");
  if (M < 0 || K < 0 || x_stride < 0 || residual_stride < 0) return fail(AC4K_ERR_SHAPE, "negative size or stride");
  if (M == 0) return 0;
  if (K == 0) return fail(AC4K_ERR_SHAPE, "rows of no elements have no norm");
  if (K > norm::kMaxCols) return fail(AC4K_ERR_UNSUPPORTED, "K = %lld is above %d", (long long)K, norm::kMaxCols);
  if (M > 0x7FFFFF00LL) return fail(AC4K_ERR_SHAPE, "too many rows");
  if (!(eps >= 0.0f)) return fail(AC4K_ERR_SHAPE, "eps must not be negative");
  if (!out || !x) return fail(AC4K_ERR_NULL, "a required pointer is NULL");
  if (precision != AC4K_NORM_BF16 && !sf) return fail(AC4K_ERR_NULL, "sf is NULL");
  if (precision == AC4K_NORM_NVFP4 && !global_scale) return fail(AC4K_ERR_NULL, "global_scale is NULL");
  if (residual_out && !residual) return fail(AC4K_ERR_NULL, "residual is NULL where residual_out is not");
  if (normed && precision == AC4K_NORM_BF16) return fail(AC4K_ERR_UNSUPPORTED, "normed stands beside a quantised output only");
  auto addr = [](const void *q) { return reinterpret_cast<uintptr_t>(q); };
  const int rsize = residual && residual_dtype == AC4K_DT_FP32 ? 4 : 2, wsize = weight && weight_dtype == AC4K_DT_FP32 ? 4 : 2;
  if ((addr(x) & 1) || (addr(residual) & (rsize - 1)) || (addr(residual_out) & (rsize - 1)) || (addr(weight) & (wsize - 1)) || (addr(normed) & 1) ||
      (addr(out) & (precision == AC4K_NORM_BF16 ? 1 : 3)) || (addr(sf) & 3) || (addr(global_scale) & 3))
    return fail(AC4K_ERR_ALIGN, "a pointer is not aligned to its elements");
  if (M == 1) x_stride = residual_stride = K;            // (what one row's stride is means nothing)
  if (residual_out) {
    // each element is read and written by one thread where the rows coincide; any other overlap has rows read after they were written
    auto meets = [&](const void *q, int64_t stride, int size) {
      return q && rows_overlap(addr(residual_out), K * rsize, K * rsize, addr(q), stride * size, K * size, M);
    };
    if ((meets(x, x_stride, 2) && !(residual_out == x && x_stride == K && rsize == 2)) ||
        (meets(residual, residual_stride, rsize) && !(residual_out == residual && residual_stride == K)))
      return fail(AC4K_ERR_SHAPE, "residual_out is the residual or x itself, element by element, or overlaps neither");
  }
  norm::Args p = {};
  p.x = static_cast<const uint16_t *>(x);
  p.residual = residual;
  p.weight = weight;
  p.out = static_cast<uint8_t *>(out);
  p.sf = static_cast<uint8_t *>(sf);
  p.gs = global_scale;
  p.normed = static_cast<uint16_t *>(normed);
  p.residual_out = residual_out;
  p.M = M; p.K = K; p.x_stride = x_stride; p.residual_stride = residual_stride;
  p.eps = eps;
  p.residual_f32 = rsize == 4;
  p.weight_f32 = wsize == 4;
  p.tiled = precision == AC4K_NORM_NVFP4 && sf_layout == AC4K_SF_TILE128X4;
  p.rows_sf = precision == AC4K_NORM_BF16 ? M : align_up(M, p.tiled ? 128 : 16);
  // 16-byte vectors: 8 elements of bf16 or two vectors of fp32; every row of every tensor begins on one
  const bool vectors = K % 8 == 0 && x_stride % 8 == 0 && (!residual || residual_stride % (rsize == 4 ? 4 : 8) == 0) &&
                       ((addr(x) | addr(residual) | addr(residual_out) | addr(weight) | addr(normed) | addr(out)) & 15) == 0;
  const cudaStream_t stream = static_cast<cudaStream_t>(stream_);
  if (precision == AC4K_NORM_BF16) return launch_norm_fmt<norm::kBf16>(p, vectors, stream);
  if (precision == AC4K_NORM_E4M3) return launch_norm_fmt<norm::kE4m3>(p, vectors, stream);
  return launch_norm_fmt<norm::kNvfp4>(p, vectors, stream);
}
