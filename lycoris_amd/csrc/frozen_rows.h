// frozen_rows.h -- the row kernels around the products of frozen_gemm.h: quantisation, weight planes, operand staging, the gated
// backward's elementwise pass, column sums.  All of them are bound by HBM (or, for one row, by the launch).
#pragma once
#include <cfloat>

#include "frozen_gemm.h"

namespace lyc {

// 8 elements of a row from column k on (beyond K: 0); `vec`: 16-byte loads are aligned and K % 8 == 0
template <typename T>
__device__ __forceinline__ void fz_row8(const T* row, int k, int K, bool vec, float (&v)[8]) {
  fz_load8<T>(row, k, k, K, vec && k < K, v);
}

// ---- rows to 8-bit integers: scale = max|x| / 127, q = round-half-even(127 x / max|x|) ----------------------------------------------
// 127 x is exact in fp32 for 16-bit inputs, and the correctly rounded quotient of two such numbers is a half exactly when the true
// quotient is (they are at least 2^-20 apart otherwise): fp32 decides every element as exact arithmetic would.  fp32 inputs take the same
// quotient in fp64 for the same reason.  The maximum is taken over the BIT PATTERNS of |x|, which order like the values and put infinity
// and NaN on top: a row that holds one gets scale NaN and q = 0, so its outputs are NaN rather than silently finite.
template <typename T>
__device__ __forceinline__ int fz_quant(float x, float amax) {
  if constexpr (sizeof(T) == 4) return (int)rint(127.0 * (double)x / (double)amax);
  else return (int)rintf(127.f * x / amax);
}
__device__ __forceinline__ float fz_amax_of(unsigned bits, float* scale) {
  if (bits >= 0x7f800000u) {
    *scale = __uint_as_float(0x7fc00000u);
    return 0.f;
  }
  const float a = __uint_as_float(bits);
  *scale = a / 127.f;
  return a;
}
template <typename T>
__device__ __forceinline__ u32x2 fz_pack_q(const float (&v)[8], float amax) {
  u32x2 o = {0u, 0u};
  if (amax > 0.f) {
    const float down = amax > 1e36f ? 0x1p-16f : 1.f;  // 127 x stays finite; what this flushes rounds to 0 anyway
#pragma unroll
    for (int e = 0; e < 8; ++e) o[e >> 2] |= ((unsigned)fz_quant<T>(v[e] * down, amax * down) & 0xffu) << (8 * (e & 3));
  }
  return o;
}

// the largest of the TPR threads of a row, to each of them
template <int TPR>
__device__ __forceinline__ unsigned fz_row_max(unsigned bits, unsigned (&red)[4]) {
#pragma unroll
  for (int o = 1; o < (TPR < 64 ? TPR : 64); o <<= 1) bits = max(bits, (unsigned)__shfl_xor((int)bits, o));
  if constexpr (TPR > 64) {
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = bits;
    __syncthreads();
    bits = max(max(red[0], red[1]), max(red[2], red[3]));
  }
  return bits;
}

// TPR threads a row, each holding NV chunks of 8 elements in registers: x is read once.  Columns K .. ldq are written as zeros.
// Bound by HBM: bf16 16384 x 5120 in 59 us (4.3 TB/s of reading and writing), 16384 x 640 out of the caches in 13; one row by the launch.
template <typename T, int TPR, int NV>
__global__ __launch_bounds__(256) void fz_quant_kernel(const T* __restrict__ x, int64_t ldx, int8_t* __restrict__ q, int64_t ldq, float* __restrict__ scale,
                                                       int64_t M, int K, int vec) {
  __shared__ unsigned red[4];
  const int t = threadIdx.x % TPR;
  const int64_t m = (int64_t)blockIdx.x * (256 / TPR) + threadIdx.x / TPR;
  float v[NV][8];
  unsigned bits = 0;
  if (m < M) {
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      fz_row8<T>(x + m * ldx, (i * TPR + t) * 8, K, vec, v[i]);
#pragma unroll
      for (int e = 0; e < 8; ++e) bits = max(bits, __float_as_uint(v[i][e]) & 0x7fffffffu);
    }
  }
  bits = fz_row_max<TPR>(bits, red);
  if (m >= M) return;
  float sc;
  const float amax = fz_amax_of(bits, &sc);
  if (t == 0) scale[m] = sc;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int64_t k = (int64_t)(i * TPR + t) * 8;
    if (k < ldq) *reinterpret_cast<u32x2*>(q + m * ldq + k) = fz_pack_q<T>(v[i], amax);
  }
}
// rows too long for the registers of a workgroup: two passes, the second out of the caches
template <typename T>
__global__ __launch_bounds__(256) void fz_quant_long_kernel(const T* __restrict__ x, int64_t ldx, int8_t* __restrict__ q, int64_t ldq, float* __restrict__ scale,
                                                            int64_t M, int K, int vec) {
  __shared__ unsigned red[4];
  const int64_t m = blockIdx.x;
  const T* row = x + m * ldx;
  unsigned bits = 0;
  float v[8];
  for (int k = threadIdx.x * 8; k < K; k += 2048) {
    fz_row8<T>(row, k, K, vec, v);
#pragma unroll
    for (int e = 0; e < 8; ++e) bits = max(bits, __float_as_uint(v[e]) & 0x7fffffffu);
  }
  bits = fz_row_max<256>(bits, red);
  float sc;
  const float amax = fz_amax_of(bits, &sc);
  if (threadIdx.x == 0) scale[m] = sc;
  for (int64_t k = threadIdx.x * 8; k < ldq; k += 2048) {
    fz_row8<T>(row, (int)k, K, vec, v);
    *reinterpret_cast<u32x2*>(q + m * ldq + k) = fz_pack_q<T>(v, amax);
  }
}

// ---- rows to fp16, scaled: out = 2^e g[m, n] col[n], scale[m] = 2^-e, the operand of dx over an 8-bit weight ------------------------------
// The largest of a row comes to [2^14, 2^15), so that fp16 holds it with 11 bits down to 2^-28 of it and with a fixed step of 2^-38 below.
// For bf16 gradients one plane is enough: g col in bf16 instead (8 bits), or col in the weight's plane, costs dx 1.4 times the error of its own
// rounding (2.35e-3 of its norm against 1.66e-3; this way 1.67e-3).  fp16 gradients take a second plane of what the first leaves.
// A row that holds an infinity or a NaN is not scaled.  Columns N .. up(N, 8) are zeros.
__device__ __forceinline__ float fz_up_of(unsigned bits, float* down) {
  const int e = bits >= 0x7f800000u ? 0 : min(14 + 127 - (int)(bits >> 23), 126);
  *down = __uint_as_float((unsigned)(127 - e) << 23);
  return __uint_as_float((unsigned)(127 + e) << 23);
}
template <typename T>
__device__ __forceinline__ void fz_scaled8(const T* row, const float* col, int k, int N, bool vec, bool vcol, float (&v)[8]) {
  float c[8];
  fz_row8<T>(row, k, N, vec, v);
  fz_load8<float>(col, k, k, N, vcol && k < N, c);
#pragma unroll
  for (int e = 0; e < 8; ++e) v[e] *= c[e];
}
template <int NP>
__device__ __forceinline__ void fz_store_planes(_Float16* out, int64_t plane, float (&v)[8], float up) {
#pragma unroll
  for (int e = 0; e < 8; ++e) v[e] *= up;
#pragma unroll
  for (int p = 0; p < NP; ++p) {
    _Float16 t[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      t[e] = (_Float16)v[e];
      v[e] = fabsf((float)t[e]) <= FLT_MAX ? v[e] - (float)t[e] : 0.f;
    }
    *reinterpret_cast<u32x4*>(out + p * plane) = *reinterpret_cast<u32x4*>(t);
  }
}
// the split over threads is fz_quant_kernel's
template <typename T, int NP, int TPR, int NV>
__global__ __launch_bounds__(256) void fz_scale_kernel(const T* __restrict__ g, const float* __restrict__ col, _Float16* __restrict__ out, int64_t plane,
                                                       float* __restrict__ scale, int64_t M, int N, int vec, int vcol) {
  __shared__ unsigned red[4];
  const int t = threadIdx.x % TPR, ldo = (N + 7) & ~7;
  const int64_t m = (int64_t)blockIdx.x * (256 / TPR) + threadIdx.x / TPR;
  float v[NV][8];
  unsigned bits = 0;
  if (m < M) {
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      fz_scaled8<T>(g + m * N, col, (i * TPR + t) * 8, N, vec, vcol, v[i]);
#pragma unroll
      for (int e = 0; e < 8; ++e) bits = max(bits, __float_as_uint(v[i][e]) & 0x7fffffffu);
    }
  }
  bits = fz_row_max<TPR>(bits, red);
  if (m >= M) return;
  float down;
  const float up = fz_up_of(bits, &down);
  if (t == 0) scale[m] = down;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int k = (i * TPR + t) * 8;
    if (k < ldo) fz_store_planes<NP>(out + m * ldo + k, plane, v[i], up);
  }
}
template <typename T, int NP>
__global__ __launch_bounds__(256) void fz_scale_long_kernel(const T* __restrict__ g, const float* __restrict__ col, _Float16* __restrict__ out, int64_t plane,
                                                            float* __restrict__ scale, int64_t M, int N, int vec, int vcol) {
  __shared__ unsigned red[4];
  const int64_t m = blockIdx.x, ldo = (N + 7) & ~7;
  const T* row = g + m * N;
  unsigned bits = 0;
  float v[8];
  for (int k = threadIdx.x * 8; k < N; k += 2048) {
    fz_scaled8<T>(row, col, k, N, vec, vcol, v);
#pragma unroll
    for (int e = 0; e < 8; ++e) bits = max(bits, __float_as_uint(v[e]) & 0x7fffffffu);
  }
  bits = fz_row_max<256>(bits, red);
  float down;
  const float up = fz_up_of(bits, &down);
  if (threadIdx.x == 0) scale[m] = down;
  for (int k = threadIdx.x * 8; k < N; k += 2048) {
    fz_scaled8<T>(row, col, k, N, vec, vcol, v);
    fz_store_planes<NP>(out + m * ldo + k, plane, v, up);
  }
}

// ---- fp16 only: the power of two that brings an 8-bit weight's scales into its range --------------------------------------------------
// The gated backward takes sw inside dx's other operand (sw dp).  fp16 has 5 exponent bits and the scales of a weight may lie anywhere: they are multiplied by f[0] = 2^e, which brings 127 max|sw| to [2^-1, 1) 2^`top`, and the product's
// alpha, f[1] = 2^-e, takes it out again.
__global__ __launch_bounds__(256) void fz_range_kernel(const float* __restrict__ sw, int n, int top, float* __restrict__ f) {
  __shared__ float red[4];
  float mx = 0.f;
  for (int i = threadIdx.x; i < n; i += 256) {
    const float a = fabsf(sw[i]);
    if (a <= 3.4e38f) mx = fmaxf(mx, a);
  }
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) mx = fmaxf(mx, __shfl_xor(mx, o));
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = mx;
  __syncthreads();
  if (threadIdx.x) return;
  mx = fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
  const int e = mx > 1e-30f && mx < 1e30f ? top - 8 - ilogbf(mx) : 0;  // 127 mx < 2^(ilogb + 8)
  f[0] = ldexpf(1.f, e);
  f[1] = ldexpf(1.f, -e);
}

// ---- the 16-bit plane of an 8-bit weight (the backward pass's operand): its integers, which 16 bits hold exactly; the scales go to the other
// operand.  Columns I .. ldo are zeros.  A workgroup takes four rows: 10240 x 1280 in 10 us (39 MB), and 5 - 8 us, most of them the launch,
// for 1280 x 1280 and 1280 x 5120
template <typename T>
__global__ __launch_bounds__(256) void fz_plane_kernel(const int8_t* __restrict__ q, int64_t ldq, T* __restrict__ out, int64_t ldo, int O, int I,
                                                       int rows_per_wg) {
  const int chunks = (int)(ldo >> 3);
  for (int r = 0; r < rows_per_wg; ++r) {
    const int o = blockIdx.x * rows_per_wg + r;
    if (o >= O) return;
    for (int c = threadIdx.x; c < chunks; c += 256) {
      T t[8];
      if (8 * c + 8 <= I) {
        const u32x2 w = *reinterpret_cast<const u32x2*>(q + (int64_t)o * ldq + 8 * c);
#pragma unroll
        for (int e = 0; e < 8; ++e) t[e] = (T)(float)(int8_t)(w[e >> 2] >> (8 * (e & 3)));
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) t[e] = (T)(8 * c + e < I ? (float)q[(int64_t)o * ldq + 8 * c + e] : 0.f);
      }
      *reinterpret_cast<u32x4*>(out + (int64_t)o * ldo + 8 * c) = *reinterpret_cast<u32x4*>(t);
    }
  }
}

// ---- staging: a row matrix into 16-byte aligned rows of 16-bit elements, NP planes -----------------------------------------------------
// NP = 1: a copy (rows whose length or base is not a multiple of 16 bytes).  NP = 3, fp32: x = h + m + l in bf16, each the rounding of
// what the ones before left; `col` scales the columns first.  Columns cols .. ldo are zeros.
// At the ends of the range: above the largest bf16 (the upper 0.2 % of the last binade) h is that one and not infinity, and m takes the rest;
// below 2^-108 the lower planes leave the normal numbers, and a term of a product is off by up to 2^-125 of its other factor.
// One launch stages up to three operands, one per blockIdx.y: they are small where it is needed most, and a launch costs 4 us.
struct FzStageJob {
  const void* x;
  const float* col;
  void* out;
  int64_t rows;
  int cols, vec;
};
struct FzStage {
  FzStageJob job[3];
};
constexpr float BF16_MAX = 0x1.fep127f;
template <typename TI, typename TO, int NP>
__global__ __launch_bounds__(256) void fz_stage_kernel(FzStage jobs) {
  const FzStageJob& j = jobs.job[blockIdx.y];
  const TI* x = static_cast<const TI*>(j.x);
  const int64_t chunks = (j.cols + 7) >> 3, ldo = chunks * 8, n = j.rows * chunks, plane = j.rows * ldo;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256) {
    const int64_t r = i / chunks;
    const int k = (int)(i - r * chunks) * 8;
    float v[8];
    fz_row8<TI>(x + r * j.cols, k, j.cols, j.vec, v);
    if (j.col) {
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] *= k + e < j.cols ? j.col[k + e] : 0.f;
    }
#pragma unroll
    for (int p = 0; p < NP; ++p) {
      TO t[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        t[e] = (TO)v[e];
        float h = (float)t[e];
        if (NP == 3 && fabsf(h) > BF16_MAX && fabsf(v[e]) <= FLT_MAX) t[e] = (TO)(h = copysignf(BF16_MAX, h));
        v[e] = fabsf(h) <= FLT_MAX ? v[e] - h : 0.f;
      }
      *reinterpret_cast<u32x4*>(static_cast<TO*>(j.out) + p * plane + r * ldo + k) = *reinterpret_cast<u32x4*>(t);
    }
  }
}

// ---- gated backward, elementwise: dp = (g act(gate), g value act'(gate)) in the order of p's halves -----------------------------------
// One pass over g and p writes what the rest of the backward pass reads: dp (rounded to the activation type: a gradient, and the operand of
// dw and dx), dps = sw f[0] dp (one rounding; dx over an 8-bit weight whose plane is its integers, [M, up(2 F, 8)]), and the column sums of
// dp before rounding, as one partial row per workgroup row (fixed order: the same bits every time).
// A workgroup takes DG_COLS columns of each half and `rows` rows; a thread 8 columns of every 8th row, two rows in flight.
// Bound by HBM, at the rate of a copy: bf16 8192 x 2560 in 48 us (252 MB), 4096 x 5120 with dp and dps in 65 (336 MB).
constexpr int DG_COLS = 256;
template <typename T, typename E>
__global__ __launch_bounds__(256) void fz_dgate_kernel(const T* __restrict__ g, const void* __restrict__ pre, T* __restrict__ dp, E* __restrict__ dps,
                                                       const float* __restrict__ sw, const float* __restrict__ f, float* __restrict__ part, int64_t M, int F,
                                                       int act, int gate_first, int vec, int rows) {
  __shared__ float sums[2][DG_COLS];
  const int tx = threadIdx.x & 31, ty = threadIdx.x >> 5;
  const int across = (F + DG_COLS - 1) / DG_COLS, slab = (int)(blockIdx.x / across), c0 = ((int)blockIdx.x - slab * across) * DG_COLS;
  const int k = c0 + tx * 8;
  const int64_t m0 = (int64_t)slab * rows;
  const int vo = gate_first ? F : 0, go = gate_first ? 0 : F;
  const bool full = vec && k + 8 <= F;
  const int64_t N = 2 * (int64_t)F, lds = (N + 7) & ~7;
  float sv[8], st[8], cv[8], ct[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) cv[e] = ct[e] = 0.f;
  if (dps && k < F) {
    fz_load8<float>(sw, vo + k, k, F, false, sv);
    fz_load8<float>(sw, go + k, k, F, false, st);
    const float scale = f ? f[0] : 1.f;
#pragma unroll
    for (int e = 0; e < 8; ++e) sv[e] *= scale, st[e] *= scale;
  }
  auto each = [&](auto ac, auto fc) {
    constexpr bool FULL = decltype(fc)::value;
#pragma unroll 2
    for (int r = ty; r < rows && m0 + r < M; r += 8) {
      const int64_t m = m0 + r;
      float gv[8], v[8], t[8], dv[8], dt[8];
      fz_load8<T>(g, m * F + k, k, F, FULL, gv);
      fz_load_pre8<T>(pre, M * N, m * N + vo + k, k, F, FULL, v);
      fz_load_pre8<T>(pre, M * N, m * N + go + k, k, F, FULL, t);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        float a, da;
        fz_act_grad<decltype(ac)::value>(t[e], a, da);
        dv[e] = gv[e] * a;
        dt[e] = gv[e] * v[e] * da;
        cv[e] += dv[e];
        ct[e] += dt[e];
      }
      if (dp) {
        fz_store8<T>(dp, m * N + vo + k, k, F, FULL, dv);
        fz_store8<T>(dp, m * N + go + k, k, F, FULL, dt);
      }
      if (dps) {
#pragma unroll
        for (int e = 0; e < 8; ++e) dv[e] *= sv[e], dt[e] *= st[e];
        fz_store8<E>(dps, m * lds + vo + k, k, F, FULL, dv);
        fz_store8<E>(dps, m * lds + go + k, k, F, FULL, dt);
        if (!FULL && k + 8 >= F)  // the product reads whole 16-byte chunks
          for (int64_t c = N; c < lds; ++c) dps[m * lds + c] = (E)0.f;
      }
    }
  };
  if (full) fz_for_act(act, [&](auto ac) { each(ac, std::true_type{}); });
  else if (k < F) fz_for_act(act, [&](auto ac) { each(ac, std::false_type{}); });
  if (!part) return;
  for (int i = 0; i < 8; ++i) {  // rows of threads one after the other
    if (ty == i) {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        sums[0][tx * 8 + e] = cv[e] + (i ? sums[0][tx * 8 + e] : 0.f);
        sums[1][tx * 8 + e] = ct[e] + (i ? sums[1][tx * 8 + e] : 0.f);
      }
    }
    __syncthreads();
  }
  for (int h = 0; h < 2; ++h) {
    const int c = c0 + (int)threadIdx.x;
    if (c < F) part[(int64_t)slab * N + (h ? go : vo) + c] = sums[h][threadIdx.x];
  }
}
// the partial rows' sum: 8 threads a column, joined in a fixed order (128 rows of 5120: 4 us, the launch)
template <typename T>
__global__ __launch_bounds__(256) void fz_join_kernel(const float* __restrict__ part, T* __restrict__ out, int64_t parts, int N) {
  __shared__ float red[8][32];
  const int tx = threadIdx.x & 31, ty = threadIdx.x >> 5, n = blockIdx.x * 32 + tx;
  float s = 0.f;
  if (n < N) {
#pragma unroll 8
    for (int64_t r = ty; r < parts; r += 8) s += part[r * N + n];
  }
  red[ty][tx] = s;
  __syncthreads();
  if (ty || n >= N) return;
#pragma unroll
  for (int i = 1; i < 8; ++i) s += red[i][tx];
  out[n] = (T)s;
}

}  // namespace lyc
