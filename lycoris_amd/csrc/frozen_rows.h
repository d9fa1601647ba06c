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

// ---- the 16-bit plane of an 8-bit weight (the backward pass's operand): its integers, which 16 bits hold exactly; the scales go to the other
// operand.  Columns I .. ldo are zeros.  A workgroup takes four rows: 10240 x 1280 in 11 us (39 MB), and 5 - 8 us, most of them the launch,
// for 1280 x 1280 and 1280 x 5120
// The bytes are taken out by bit-field extracts: written as shifts, the two words become one of 64 bits for the compiler, and its v_lshlrev_b64 by the last
// register that the kernel has (v23 of 24) gave wrong results now and then on this card, a wave at a time.
constexpr int FZ_PLANE_ROWS = 4;
struct FzPlane {
  const int8_t* q;
  void* out;
  int64_t ldq;
  int O, I, groups;  // groups: workgroups that take rows of it
};
template <typename T>
__device__ __forceinline__ void fz_plane_rows(const FzPlane& p, int group) {
  const int chunks = (p.I + 7) >> 3;
  for (int r = 0; r < FZ_PLANE_ROWS; ++r) {
    const int o = group * FZ_PLANE_ROWS + r;
    if (o >= p.O) return;
    const int8_t* q = p.q + (int64_t)o * p.ldq;
    for (int c = threadIdx.x; c < chunks; c += 256) {
      T t[8];
      if (8 * c + 8 <= p.I) {
        const u32x2 w = *reinterpret_cast<const u32x2*>(q + 8 * c);
#pragma unroll
        for (int e = 0; e < 8; ++e) t[e] = (T)(float)(int)__builtin_amdgcn_sbfe(w[e >> 2], 8 * (e & 3), 8);  // (the builtin is unsigned)
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) t[e] = (T)(8 * c + e < p.I ? (float)q[8 * c + e] : 0.f);
      }
      *reinterpret_cast<u32x4*>(static_cast<T*>(p.out) + ((int64_t)o * chunks + c) * 8) = *reinterpret_cast<u32x4*>(t);
    }
  }
}
template <typename T>
__global__ __launch_bounds__(256) void fz_plane_kernel(FzPlane p) {
  fz_plane_rows<T>(p, (int)blockIdx.x);
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
// The split over threads is fz_quant_kernel's.  The weight's plane is made in the same launch, by the first w.groups workgroups: dx of a layer is short,
// and a launch costs 4 us (4096 x 1280 x 1280, forward and dx: 60 -> 56 us).
template <typename T, int NP, int TPR, int NV>
__global__ __launch_bounds__(256) void fz_scale_kernel(const T* __restrict__ g, const float* __restrict__ col, _Float16* __restrict__ out, int64_t plane,
                                                       float* __restrict__ scale, int64_t M, int N, int vec, int vcol, FzPlane w) {
  __shared__ unsigned red[4];
  if ((int)blockIdx.x < w.groups) return fz_plane_rows<_Float16>(w, (int)blockIdx.x);
  const int t = threadIdx.x % TPR, ldo = (N + 7) & ~7;
  const int64_t m = ((int64_t)blockIdx.x - w.groups) * (256 / TPR) + threadIdx.x / TPR;
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
                                                            float* __restrict__ scale, int64_t M, int N, int vec, int vcol, FzPlane w) {
  __shared__ unsigned red[4];
  if ((int)blockIdx.x < w.groups) return fz_plane_rows<_Float16>(w, (int)blockIdx.x);
  const int64_t m = (int64_t)blockIdx.x - w.groups, ldo = (N + 7) & ~7;
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

// the gated backward's 8 columns from k on of row m: the value half's and the gate half's part of dp
template <int ACT>
__device__ __forceinline__ void fz_dgate_of(const float (&gv)[8], const float (&v)[8], const float (&t)[8], float (&dv)[8], float (&dt)[8]) {
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    float a, da;
    fz_act_grad<ACT>(t[e], a, da);
    dv[e] = gv[e] * a;
    dt[e] = gv[e] * v[e] * da;
  }
}
template <typename T, int ACT>
__device__ __forceinline__ void fz_dgate8(const T* g, const void* pre, int64_t m, int64_t M, int k, int F, int vo, int go, bool full, float (&dv)[8],
                                          float (&dt)[8]) {
  const int64_t N = 2 * (int64_t)F;
  float gv[8], v[8], t[8];
  fz_load8<T>(g, m * F + k, k, F, full, gv);
  fz_load_pre8<T>(pre, M * N, m * N + vo + k, k, F, full, v);
  fz_load_pre8<T>(pre, M * N, m * N + go + k, k, F, full, t);
  fz_dgate_of<ACT>(gv, v, t, dv, dt);
}
// what is read for it, 16 bits and whole chunks, as it lies in memory (loads that are in flight while another row is worked on)
struct FzDgateRaw {
  u32x4 g, v, t;
  u32x2 vl, tl;
  template <typename T>
  __device__ __forceinline__ void load(const T* gp, const void* pre, int64_t m, int64_t M, int k, int F, int vo, int go) {
    const int64_t N = 2 * (int64_t)F;
    const uint16_t* hi = static_cast<const uint16_t*>(pre) + m * N + k;
    const uint8_t* lo = reinterpret_cast<const uint8_t*>(static_cast<const uint16_t*>(pre) + M * N) + m * N + k;
    g = *reinterpret_cast<const u32x4*>(gp + m * F + k);
    v = *reinterpret_cast<const u32x4*>(hi + vo);
    t = *reinterpret_cast<const u32x4*>(hi + go);
    vl = *reinterpret_cast<const u32x2*>(lo + vo);
    tl = *reinterpret_cast<const u32x2*>(lo + go);
  }
  template <typename T, int ACT>
  __device__ __forceinline__ void use(float (&dv)[8], float (&dt)[8]) const {
    float gv[8], vv[8], tv[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) gv[e] = (float)reinterpret_cast<const T*>(&g)[e];
    fz_join24(v, vl, vv);
    fz_join24(t, tl, tv);
    fz_dgate_of<ACT>(gv, vv, tv, dv, dt);
  }
};

// ---- gated backward, elementwise: dp = (g act(gate), g value act'(gate)) in the order of p's halves -----------------------------------
// One pass over g and p writes what the rest of the backward pass reads.  fz_dgate_kernel, where dp itself is all that is wanted, and for 32 bits:
// dp, rounded to the activation type (it is the gradient of `base`), and the column sums of dp before rounding, as one partial row per
// workgroup row (fixed order: the same bits every time).
// A workgroup takes DG_COLS columns of each half and `rows` rows; a thread 8 columns of every 8th row, two rows in flight.
constexpr int DG_COLS = 256;
template <typename T>
__global__ __launch_bounds__(256) void fz_dgate_kernel(const T* __restrict__ g, const void* __restrict__ pre, T* __restrict__ dp, float* __restrict__ part,
                                                       int64_t M, int F, int act, int gate_first, int vec, int rows) {
  __shared__ float sums[2][DG_COLS];
  const int tx = threadIdx.x & 31, ty = threadIdx.x >> 5;
  const int across = (F + DG_COLS - 1) / DG_COLS, slab = (int)(blockIdx.x / across), c0 = ((int)blockIdx.x - slab * across) * DG_COLS;
  const int k = c0 + tx * 8;
  const int64_t m0 = (int64_t)slab * rows;
  const int vo = gate_first ? F : 0, go = gate_first ? 0 : F;
  const bool full = vec && k + 8 <= F;
  const int64_t N = 2 * (int64_t)F;
  float cv[8], ct[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) cv[e] = ct[e] = 0.f;
  auto each = [&](auto ac, auto fc) {
    constexpr bool FULL = decltype(fc)::value;
#pragma unroll 2
    for (int r = ty; r < rows && m0 + r < M; r += 8) {
      const int64_t m = m0 + r;
      float dv[8], dt[8];
      fz_dgate8<T, decltype(ac)::value>(g, pre, m, M, k, F, vo, go, FULL, dv, dt);
#pragma unroll
      for (int e = 0; e < 8; ++e) cv[e] += dv[e], ct[e] += dt[e];
      if (dp) {
        fz_store8<T>(dp, m * N + vo + k, k, F, FULL, dv);
        fz_store8<T>(dp, m * N + go + k, k, F, FULL, dt);
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

// The same where products follow, 16 bits: beside dp (or without it) their operand, 2^e c[n] dp[m, n] in NP fp16 planes with a power of two a
// row as in fz_scale_kernel, and scale[m] = 2^-e.  c: the scales of an 8-bit weight, or null.  dp rounded to bf16 as an operand cost dx and
// dw 1.4 times the error of their own rounding each (2.34e-3 of the norm against 1.66e-3; this way 1.67e-3).
// The largest of a row is known when all of it has been computed, so a row stays in the registers of its threads: a wave's where it has up to
// 512 columns a half (WAVE: four waves a workgroup, each with rows of its own), else a workgroup's, a chunk of 8 columns a thread; rows of more than 8192
// columns are computed twice, the second time out of the caches (NV = 0; two chunks a thread do not fit the 128 registers of 1024 threads).  `rows` rows follow each other; the column sums stay with the threads of their columns.
// top: the largest scale of the slab's rows, for the other operand of dw.
// Bound by HBM, short of a copy's rate by the meeting for each row's largest: bf16 4096 x 5120 with dp 69 us (336 MB, 4.9 TB/s), 8192 x 2560 without, with column sums, 62 (252 MB, 4.0 TB/s).
struct FzDgate {
  const void *g, *pre;
  void* dp;
  _Float16* out;
  const float* c;
  float *scale, *top, *part;
  int64_t M, plane;
  int F, act, gate_first, vec, rows;
};
template <typename T, int NP, int NV, bool WAVE, bool SUMS>
__global__ __launch_bounds__(WAVE ? 256 : 1024) void fz_dgate_rows_kernel(FzDgate a) {
  __shared__ unsigned red[2][16];
  const int F = a.F, nt = WAVE ? 64 : (int)blockDim.x, t = WAVE ? (int)threadIdx.x & 63 : (int)threadIdx.x;
  const int64_t slab = WAVE ? (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6) : (int64_t)blockIdx.x, m0 = slab * a.rows;
  const int vo = a.gate_first ? F : 0, go = a.gate_first ? 0 : F;
  const int64_t N = 2 * (int64_t)F, lds = (N + 7) & ~7;
  const T* g = static_cast<const T*>(a.g);
  float top = 0.f;
  int at = 0;
  auto largest = [&](unsigned bits) {  // of the row, to each of its threads
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) bits = max(bits, (unsigned)__shfl_xor((int)bits, o));
    if constexpr (!WAVE) {
      if ((threadIdx.x & 63) == 0) red[at][threadIdx.x >> 6] = bits;
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // the LDS write; __syncthreads() might wait for the next row's loads too
      __builtin_amdgcn_s_barrier();
      asm volatile("" ::: "memory");
      bits = 0;
      for (int w = 0; w < nt / 64; ++w) bits = max(bits, red[at][w]);
      at ^= 1;  // the next row's go where nobody reads this row's any more
    }
    return bits;
  };
  auto peak = [](const float (&v)[8], unsigned bits) {  // of the finite ones
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const unsigned u = __float_as_uint(v[e]) & 0x7fffffffu;
      bits = u < 0x7f800000u ? max(bits, u) : bits;
    }
    return bits;
  };
  auto put = [&](int64_t m, int k, bool full, const float (&dv)[8], const float (&dt)[8]) {
    if (a.dp) {
      fz_store8<T>(a.dp, m * N + vo + k, k, F, full, dv);
      fz_store8<T>(a.dp, m * N + go + k, k, F, full, dt);
    }
  };
  auto times_c = [&](int k, bool full, float (&dv)[8], float (&dt)[8]) {
    if (!a.c) return;
    float cv[8], ct[8];
    fz_load8<float>(a.c, vo + k, k, F, full, cv);
    fz_load8<float>(a.c, go + k, k, F, full, ct);
#pragma unroll
    for (int e = 0; e < 8; ++e) dv[e] *= cv[e], dt[e] *= ct[e];
  };
  auto planes = [&](int64_t m, int k, bool full, float up, float (&v)[8], int half) {
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] *= up;
#pragma unroll
    for (int p = 0; p < NP; ++p) {
      _Float16* out = a.out + p * a.plane;
      fz_store8<_Float16>(out, m * lds + half + k, k, F, full, v);
      if (p + 1 < NP) {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const float h = (float)(_Float16)v[e];
          v[e] = fabsf(h) <= FLT_MAX ? v[e] - h : 0.f;
        }
      }
      if (!full && k + 8 >= F)  // the products read whole 16-byte chunks
        for (int64_t c = N; c < lds; ++c) out[m * lds + c] = (_Float16)0.f;
    }
  };
  fz_for_act(a.act, [&](auto ac) {
    constexpr int ACT = decltype(ac)::value;
    if constexpr (NV == 1) {
      const int k = t * 8;
      const bool in = k < F;
      float sv[8], st[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) sv[e] = st[e] = 0.f;
      FzDgateRaw raw;
      if (a.vec && in && m0 < a.M) raw.template load<T>(g, a.pre, m0, a.M, k, F, vo, go);
      for (int r = 0; r < a.rows && m0 + r < a.M; ++r) {
        const int64_t m = m0 + r;
        float dv[8], dt[8];
        unsigned bits = 0;
        if (in) {
          if (a.vec) {
            const FzDgateRaw now = raw;
            if (r + 1 < a.rows && m + 1 < a.M) raw.template load<T>(g, a.pre, m + 1, a.M, k, F, vo, go);  // in flight while this row is worked on
            now.template use<T, ACT>(dv, dt);
          } else {
            fz_dgate8<T, ACT>(g, a.pre, m, a.M, k, F, vo, go, false, dv, dt);
          }
          if constexpr (SUMS) {
#pragma unroll
            for (int e = 0; e < 8; ++e) sv[e] += dv[e], st[e] += dt[e];
          }
          put(m, k, a.vec, dv, dt);
          times_c(k, a.vec, dv, dt);
          bits = peak(dv, peak(dt, 0));
        }
        float down;
        const float up = fz_up_of(largest(bits), &down);
        if (t == 0) a.scale[m] = down;
        top = fmaxf(top, down);
        if (in) {
          planes(m, k, a.vec, up, dv, vo);
          planes(m, k, a.vec, up, dt, go);
        }
      }
      if (SUMS && in && m0 < a.M) {
        fz_store8<float>(a.part, slab * N + vo + k, k, F, a.vec, sv);
        fz_store8<float>(a.part, slab * N + go + k, k, F, a.vec, st);
      }
    } else {
      for (int r = 0; r < a.rows && m0 + r < a.M; ++r) {
        const int64_t m = m0 + r;
        float dv[8], dt[8];
        unsigned bits = 0;
        for (int k = t * 8; k < F; k += nt * 8) {
          fz_dgate8<T, ACT>(g, a.pre, m, a.M, k, F, vo, go, a.vec, dv, dt);
          put(m, k, a.vec, dv, dt);
          if constexpr (SUMS) {  // the slab's partial sums, each the same thread's in every row
            float s[8];
            const int64_t pv = slab * N + vo + k, pt = slab * N + go + k;
            fz_load8<float>(a.part, pv, k, r ? F : 0, r && a.vec, s);
#pragma unroll
            for (int e = 0; e < 8; ++e) s[e] += dv[e];
            fz_store8<float>(a.part, pv, k, F, a.vec, s);
            fz_load8<float>(a.part, pt, k, r ? F : 0, r && a.vec, s);
#pragma unroll
            for (int e = 0; e < 8; ++e) s[e] += dt[e];
            fz_store8<float>(a.part, pt, k, F, a.vec, s);
          }
          times_c(k, a.vec, dv, dt);
          bits = peak(dv, peak(dt, bits));
        }
        float down;
        const float up = fz_up_of(largest(bits), &down);
        if (t == 0) a.scale[m] = down;
        top = fmaxf(top, down);
        for (int k = t * 8; k < F; k += nt * 8) {
          fz_dgate8<T, ACT>(g, a.pre, m, a.M, k, F, vo, go, a.vec, dv, dt);
          times_c(k, a.vec, dv, dt);
          planes(m, k, a.vec, up, dv, vo);
          planes(m, k, a.vec, up, dt, go);
        }
      }
    }
  });
  if (a.top && t == 0 && m0 < a.M) a.top[slab] = top;
}

// ---- the 16-bit weight and x as fp16 operands of dx and dw, 16 bits ---------------------------------------------------------------------
// Each takes one power of two: the weight 2^f that brings its largest entry to [2^14, 2^15); x 2^f scale[m] (the row scales of dp's operand come
// back in here, along the K of dw), its f from the largest of x and the largest scale.  What fp16 loses of bf16 values that way lies 2^-28 and more
// below the largest.  fz_peak_kernel takes the largest finite entries, one partial a workgroup; fz_level_kernel joins the partials, writes the
// operands, and 2^-f for the products' alpha.  blockIdx.y: the operand.
constexpr int FZ_PEAKS = 1024;
struct FzLevelJob {
  const void* x;
  _Float16* out;
  const float *row, *top;  // row scales and their largest a slab, or null
  unsigned* part;
  float* alpha;
  int64_t rows;
  int cols, vec, tops;
};
struct FzLevel {
  FzLevelJob job[2];
};
template <typename T>
__global__ __launch_bounds__(256) void fz_peak_kernel(FzLevel jobs) {
  __shared__ unsigned red[4];
  const FzLevelJob& j = jobs.job[blockIdx.y];
  const T* x = static_cast<const T*>(j.x);
  const int64_t n = j.rows * j.cols;
  const bool vec = fz_al16(x);
  unsigned bits = 0;
  for (int64_t i = ((int64_t)blockIdx.x * 256 + threadIdx.x) * 8; i < n; i += (int64_t)gridDim.x * 2048) {
    float v[8];
    fz_load8<T>(x, i, 0, n - i < 8 ? (int)(n - i) : 8, vec && n - i >= 8, v);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const unsigned u = __float_as_uint(v[e]) & 0x7fffffffu;
      bits = u < 0x7f800000u ? max(bits, u) : bits;
    }
  }
  bits = fz_row_max<256>(bits, red);
  if (threadIdx.x == 0) j.part[blockIdx.x] = bits;
}
template <typename T>
__global__ __launch_bounds__(256) void fz_level_kernel(FzLevel jobs, int peaks) {
  __shared__ unsigned red[2][4];
  const FzLevelJob& j = jobs.job[blockIdx.y];
  const T* x = static_cast<const T*>(j.x);
  unsigned bits = 0, top = 0;
  for (int i = threadIdx.x; i < peaks; i += 256) bits = max(bits, j.part[i]);
  for (int i = threadIdx.x; i < j.tops; i += 256) top = max(top, __float_as_uint(j.top[i]));  // powers of two: ordered like their bits
  bits = fz_row_max<256>(bits, red[0]);
  top = fz_row_max<256>(top, red[1]);
  const int f = max(-126, min(126, 14 - ((int)(bits >> 23) - 127) - (j.tops ? (int)(top >> 23) - 127 : 0)));
  if (blockIdx.x == 0 && threadIdx.x == 0) *j.alpha = __uint_as_float((unsigned)(127 - f) << 23);
  const int64_t chunks = (j.cols + 7) >> 3, ldo = chunks * 8, n = j.rows * chunks;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256) {
    const int64_t r = i / chunks;
    const int k = (int)(i - r * chunks) * 8;
    const int e2 = f + (j.row ? (int)(__float_as_uint(j.row[r]) >> 23) - 127 : 0);
    const float up = e2 < -126 ? 0.f : __uint_as_float((unsigned)(min(e2, 127) + 127) << 23);
    float v[8];
    _Float16 t[8];
    fz_row8<T>(x + r * j.cols, k, j.cols, j.vec, v);
#pragma unroll
    for (int e = 0; e < 8; ++e) t[e] = (_Float16)(v[e] * up);
    *reinterpret_cast<u32x4*>(j.out + r * ldo + k) = *reinterpret_cast<u32x4*>(t);
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
