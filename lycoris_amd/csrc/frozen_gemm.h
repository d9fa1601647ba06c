// frozen_gemm.h -- the matrix products of the 8-bit frozen layer and of the gated projection.
//
//     8-bit forward   acc[m, n] = sum_k aq[m, k] bq[n, k]          both operands K-contiguous, int32 accumulators
//     gated forward   p[m, n]   = sum_k x[m, k] w[n, k]            both operands K-contiguous; w is [2 F, K]
//     dx              dx[m, i]  = sum_o dp[m, o] w[o, i]           A K-contiguous, B K-strided
//     dw              dw[o, i]  = sum_m dp[m, o] x[m, i]           both K-strided
//
// The skeleton is gemm16d.h's: both operands go HBM -> LDS by LDS-DMA into a ring of K steps, fragments are read one step ahead of the
// MFMAs that use them, the MFMA roles are swapped and the n tiles formed in pairs so that a lane owns 8 consecutive output columns of one
// row.  Every address is formed in bytes, so 8-bit operands (64 k per step, v_mfma_i32_16x16x64_i8) and 16-bit ones (32 k,
// v_mfma_f32_16x16x32) run the same loop: a step is 64 bytes of K, a fragment 16 bytes of one row, an MFMA 16 cycles either way.
//
// What bounds the loop, measured inside it (256 x 256 tile, 8 waves, cycles per 64-byte step; the MFMAs alone are 1024): 1450 with the
// descriptor and tail arithmetic of every step in line (~100 scalar instructions between the barrier and the first MFMA), 1250 with a
// handful.  The clock then is 1.75 - 1.95 GHz: the matrix pipe is near what the card's power allows (1.68 PFLOP/s bf16, 2.4 - 2.7 POP/s int8
// inside the loop).  The LDS pipe is a quarter busy and the L2 order matters at 8192^3 only (988 -> 872 us).  On inputs out of HBM the
// granularity of the DMA counts: with slots of 64 bytes of K every row is asked for in half cache lines, with 128 bytes in whole ones, and a
// product like dx 8192 x 640 x 5120 takes 64 instead of 76 us (55 with its inputs in the caches).
//
//   * the buffer descriptor is rebased on every K step: an operand may be larger than 4 GiB;
//   * rows, columns and K outside the operand are masked in the DMA's lane offsets, 16 bytes at a time (both operands: 0 times a stray NaN
//     would not be 0);
//   * a product may be a sum of SEGMENTS over pairs of operand planes: 32-bit operands are held as three bf16 planes each
//     (x = h + m + l, 24 bits) and multiplied as hh + hm + mh + hl + lh + mm; what is left out is below 2^-24 of a term;
//   * GATED: the tile's B rows are BN / 2 rows of the value half and the BN / 2 rows of the gate half that belong to the same output
//     columns; a wave owns both, so value * act(gate) is formed in its registers and only [M, F] is written.
#pragma once
#include <type_traits>
#include <utility>

#include "gemm16d.h"

namespace lyc {

typedef __attribute__((ext_vector_type(4))) int i32x4;

template <typename E>
struct FE {  // 16-bit
  static constexpr int SIZE = 2;
  using acc = f32x4;
  static __device__ __forceinline__ acc mma(u32x4 a, u32x4 b, acc c) {
    using F8 = typename TT<E>::frag;
    return TT<E>::mma(__builtin_bit_cast(F8, a), __builtin_bit_cast(F8, b), c);
  }
};
template <>
struct FE<int8_t> {
  static constexpr int SIZE = 1;
  using acc = i32x4;
  static __device__ __forceinline__ acc mma(u32x4 a, u32x4 b, acc c) {
    return __builtin_amdgcn_mfma_i32_16x16x64_i8(__builtin_bit_cast(i32x4, a), __builtin_bit_cast(i32x4, b), c, 0, 0, 0);
  }
};

enum { FZ_ACT_GELU = 0, FZ_ACT_GELU_TANH = 1, FZ_ACT_SILU = 2 };

// Phi(t) = erfc(-t / sqrt 2) / 2 with erfc(z) = w P(w) exp(-z^2), w = 1 / (1 + 0.45 z): P is the degree-7 polynomial of least largest
// relative error on z = 0 .. 14 (3.5e-7, fitted to erfc in 64 bits).  Measured against 64 bits at two million points each, relative to Phi: 6.4e-7 on
// [0, 8], 1.0e-6 on [-3, 0], 2.2e-6 on [-6, -3], 3.9e-6 on [-9, -6] (the rounding of t^2, which the exponential magnifies by t^2 / 2); it
// underflows with exp(-t^2 / 2), below t = -13.  About 20 operations, where the library's erfc takes three times that and a branch.
__device__ __forceinline__ void fz_phi(float t, float& phi, float& e) {
  const float z = 0.70710678f * fabsf(t);
  const float w = __builtin_amdgcn_rcpf(fmaf(0.45f, z, 1.f));
  float q = 0.0689046234f;
  q = fmaf(q, w, -0.248889327f);
  q = fmaf(q, w, 0.223910257f);
  q = fmaf(q, w, 0.026233878f);
  q = fmaf(q, w, 0.196168676f);
  q = fmaf(q, w, 0.225782961f);
  q = fmaf(q, w, 0.254004091f);
  q = fmaf(q, w, 0.25388521f);
  e = __builtin_amdgcn_exp2f(-0.72134752f * t * t);  // exp(-t^2 / 2)
  const float h = 0.5f * q * w * e;
  phi = t >= 0.f ? 1.f - h : h;
}
__device__ __forceinline__ float fz_sigmoid(float t) { return __builtin_amdgcn_rcpf(1.f + __expf(-t)); }

// act(t) and its derivative in fp32
template <int ACT>
__device__ __forceinline__ float fz_act(float t) {
  if constexpr (ACT == FZ_ACT_SILU) return t * fz_sigmoid(t);
  if constexpr (ACT == FZ_ACT_GELU) {
    float phi, e;
    fz_phi(t, phi, e);
    return t * phi;
  }
  return t * fz_sigmoid(1.5957691216057308f * (t + 0.044715f * t * t * t));  // 0.5 t (1 + tanh u) = t sigmoid(2 u)
}
template <int ACT>
__device__ __forceinline__ void fz_act_grad(float t, float& a, float& da) {
  if constexpr (ACT == FZ_ACT_SILU) {
    const float s = fz_sigmoid(t);
    a = t * s;
    da = s + a * (1.f - s);
  } else if constexpr (ACT == FZ_ACT_GELU) {
    float phi, e;
    fz_phi(t, phi, e);
    a = t * phi;
    da = phi + t * 0.39894228040143268f * e;
  } else {
    const float s = fz_sigmoid(1.5957691216057308f * (t + 0.044715f * t * t * t));
    a = t * s;
    da = s + a * (1.f - s) * 1.5957691216057308f * (1.f + 0.134145f * fminf(t * t, 1e30f));  // (0 times infinity would be NaN)
  }
}
// f(the activation as a constant): one branch for as many values as f works on (a branch for each keeps the compiler from interleaving them)
template <typename F>
__device__ __forceinline__ void fz_for_act(int act, F f) {
  if (act == FZ_ACT_SILU) f(std::integral_constant<int, FZ_ACT_SILU>{});
  else if (act == FZ_ACT_GELU) f(std::integral_constant<int, FZ_ACT_GELU>{});
  else f(std::integral_constant<int, FZ_ACT_GELU_TANH>{});
}

// One product.  lda / ldb in bytes.  kb: bytes of K along a K-contiguous operand, rounded up to 16 (what the operand's rows hold up to
// there has to be finite in 16 bits, and zero in A's rows in 8 bits).  Planes of segment s: (pa >> 4 s) & 15 and (pb >> 4 s) & 15.
struct FzProb {
  const void *A, *B;
  int64_t lda, ldb, a_plane, b_plane;
  int M, N, K, kb;
  int nseg;
  unsigned pa, pb;
  int ksplit;  // the steps go to this many workgroups a tile (blockIdx.y); more than one: raw sums to FzEpi::part
};

enum { FZ_PLAIN = 0, FZ_LINEAR = 1, FZ_GATED = 2 };
struct FzEpi {
  void* part;          // ksplit > 1: [ksplit, M, N] fp32 (8-bit: int32), which fz_reduce_kernel finishes
  void* out;           // [M, N] (GATED: [M, F]), row pitch = N (F) elements
  void* pre;           // GATED: p [M, 2 F] for the backward pass (fz_store_pre8) or null
  const float* alpha;  // PLAIN: device scalar on the result, or null
  const float *sa, *sw;  // scales of A's rows (PLAIN too), of B's rows (8-bit only), or null
  const void* bias;    // [N] (GATED: [2 F]) or null; fp32 when bias_f32, else the output's type
  const void* base;    // [M, N] (GATED: [M, 2 F]) in the output's type, or null
  int64_t pre_total;   // elements of p
  int bias_f32, act, gate_first, F;
};

// what the DMA pieces of one operand's K step need
struct FzStep {
  __amdgpu_buffer_rsrc_t rs;
  unsigned mask;
};

// One operand of one workgroup tile: DMA addressing (issue) and fragment addressing (read).  A ring slot holds SB = 64 (both operands
// K-strided) or 128 bytes of K: one or two MFMA steps.
//   ROWS: tile extent; W: waves along it; NW: waves in all; KS: K-strided in memory; PAIRED: the n operand (paired tile order; with an odd
//   number of 16-row tiles a wave, as in 160 rows over two waves, the last one is in natural order)
// K-contiguous: LDS rows of 128 bytes, their 16-byte chunks XOR-permuted on the DMA's source address so that a fragment read falls on
// different slots of the 256-byte bank row (gemm16d.h).
// K-strided (16-bit): the image in memory order, read transposed (gemm16d.h).
template <int ROWS, int W, int NW, int SB, bool KS, bool PAIRED, bool GATED>
struct FzOperand {
  static constexpr int PIECES = ROWS * SB / 1024, PPW = (PIECES + NW - 1) / NW;  // 1 KiB DMA pieces of a K step; a wave without one fetches nothing
  static constexpr bool SPARE = PIECES % NW != 0;                          // ... into a spare piece of LDS: every wave's count is the same
  static constexpr int WEXT = ROWS / W, NT = WEXT / 16, NP = NT / 2;
  static constexpr bool ODD = PAIRED && NT % 2 != 0;
  static constexpr int CH = ROWS / 8, PITCH = ROWS * 2;  // KS: chunks and bytes per k row
  static constexpr bool XOR = PITCH % 128 == 0;          // KS: 320-byte rows fall on different banks by themselves
  static constexpr int HALVES = SB / 64, KROWS = SB / 2;  // MFMA steps a slot; KS: k rows a slot
  static constexpr int NADDR = KS ? (PAIRED ? NP + ODD : NT) : HALVES * (1 + ODD);
  static constexpr int SLOT = ROWS * SB;
  static_assert(KS || SB == 128, "64-byte slots: K-strided operands");
  static_assert(WEXT % 16 == 0 && (!GATED || (PAIRED && !KS && NT % 4 == 0 && !SPARE)), "tile shape");

  unsigned voff[PPW], rd[NADDR], beyond;  // beyond: K-contiguous: K4_OOB where this lane's chunk lies beyond K in the last step of a segment
  const char *org, *cur;                  // the tile's first byte in plane 0; the next K step's
  unsigned kstep, tail_bytes;             // bytes a step advances; K-strided: bytes of the rows that the last step of a segment has
  static __device__ __forceinline__ int piece_row(int j) {  // row (KC) or k row (KS) of this lane in piece j of its wave
    const int wave = (int)(threadIdx.x >> 6), lane = (int)threadIdx.x & 63;
    if constexpr (!KS) return 1024 / SB * (wave + NW * j) + lane / (SB / 16);
    else return (64 * (wave + NW * j) + lane) / CH;
  }
  static __device__ __forceinline__ int piece_chunk(int j) {
    const int lane = (int)threadIdx.x & 63;
    if constexpr (!KS) return (lane % (SB / 16)) ^ g16d_swz_kc<PAIRED>(piece_row(j));
    else return ((64 * (int)((threadIdx.x >> 6) + NW * j) + lane) % CH) ^ (XOR ? g16d_swz_ks<PAIRED, CH>(piece_row(j)) : 0);
  }
  __device__ __forceinline__ void setup(const void* base, int64_t ld, int r0, int ext, int kdim, int kb, int stage_off, int wsel, int second) {
    const int lane = threadIdx.x & 63, li = lane & 15, g = lane >> 4;
    if constexpr (!KS) {
      org = static_cast<const char*>(base) + (int64_t)r0 * ld;
      kstep = SB;
#pragma unroll
      for (int j = 0; j < PPW; ++j) {
        const int r = piece_row(j);
        // GATED: rows 0 .. BN / 2 are the half whose first row is `base`, the others the half `second` rows further on
        const int gr = !GATED || r < ROWS / 2 ? r : second + r - ROWS / 2;
        voff[j] = r0 + gr < ext && (!SPARE || r < ROWS) ? (unsigned)gr * (unsigned)ld + (unsigned)piece_chunk(j) * 16u : K4_OOB;
      }
      beyond = (unsigned)piece_chunk(0) * 16u > (unsigned)((kb - 1) & (SB - 1)) ? K4_OOB : 0u;  // (the chunk does not depend on the piece)
      const int r = wsel * (GATED ? WEXT / 2 : WEXT) + (PAIRED ? 8 * (li >> 2) + (li & 3) : li);
      const int o = wsel * WEXT + 32 * NP + li;  // ODD: the last tile's row
#pragma unroll
      for (int h = 0; h < HALVES; ++h) {
        rd[h] = (unsigned)(stage_off + r * SB + (((4 * h + g) ^ g16d_swz_kc<PAIRED>(r)) << 4));
        if constexpr (ODD) rd[HALVES + h] = (unsigned)(stage_off + o * SB + (((4 * h + g) ^ g16d_swz_kc<PAIRED>(o)) << 4));
      }
    } else {
      org = static_cast<const char*>(base) + (int64_t)r0 * 2;
      kstep = (unsigned)KROWS * (unsigned)ld;
      tail_bytes = (unsigned)((kdim - 1) & (KROWS - 1)) * (unsigned)ld + (unsigned)(((ext + 7) & ~7) - r0) * 2u;
      beyond = 0;
#pragma unroll
      for (int j = 0; j < PPW; ++j) {
        const int c = piece_chunk(j);
        voff[j] = r0 + 8 * c < ext && (!SPARE || piece_row(j) < KROWS) ? (unsigned)piece_row(j) * (unsigned)ld + (unsigned)c * 16u : K4_OOB;
      }
      const int rho = li >> 2, quad = li & 3, x = XOR ? g16d_swz_ks<PAIRED, CH>(rho) : 0, krow = 8 * g + rho;
#pragma unroll
      for (int t = 0; t < NADDR; ++t) {
        const int col = wsel * WEXT + (!PAIRED ? 16 * t + 4 * quad : ODD && t == NP ? 32 * NP + 4 * quad : 32 * t + 8 * quad);
        rd[t] = (unsigned)(stage_off + krow * PITCH + (((col >> 3) ^ x) << 4) + (col & 7) * 2);
      }
    }
  }
  // the byte offset of line part + S i of the tile's K step (K-strided: 128 bytes of a k row, of whole steps only), beyond the tile: K4_OOB
  template <int S>
  __device__ __forceinline__ unsigned ahead(int part, int i, int64_t ld, int r0, int ext) const {
    const int l = part + S * i;
    if constexpr (!KS) return l < ROWS && r0 + l < ext ? (unsigned)l * (unsigned)ld : K4_OOB;
    constexpr int LINES = (PITCH + 127) / 128;
    const int kr = l / LINES, c = l % LINES;
    return kr < KROWS && r0 + 64 * c < ext ? (unsigned)kr * (unsigned)ld + 128u * c : K4_OOB;
  }
  __device__ __forceinline__ void seek(int64_t plane_off) { cur = org + plane_off; }
  // the next K step: the descriptor is rebased to it (an operand may exceed 4 GiB; rows and columns are masked in the lane offsets, so any
  // size will do).  last: what lies beyond K reads as zero, by the lanes' chunks or by the descriptor's end; dead: nothing is left to fetch,
  // the refills behind the last step store zeros
  __device__ __forceinline__ FzStep next(bool last, bool dead) {
    const unsigned bytes = dead ? 0u : KS && last ? tail_bytes : 0x7fffffffu;
    const FzStep st{__builtin_amdgcn_make_buffer_rsrc(const_cast<char*>(cur), 0, (int)bytes, K4_RSRC_FLAGS), !KS && last ? beyond : 0u};
    cur += kstep;
    return st;
  }
  template <int J>
  __device__ __forceinline__ void issue_piece(const FzStep& st, char* slot_of_wave, char* spare) const {
    char* dst = slot_of_wave + NW * J * 1024;
    if constexpr (SPARE && (J + 1) * NW > PIECES) {
      if (__builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6)) + NW * J >= PIECES) dst = spare;
    }
    __builtin_amdgcn_raw_ptr_buffer_load_lds(st.rs, (k4_lds_ptr)dst, 16, (int)(KS ? voff[J] : voff[J] | st.mask), 0, 0, 0);
  }
  template <int... J>
  __device__ __forceinline__ void issue(const FzStep& st, char* slot_of_wave, char* spare, std::integer_sequence<int, J...>) const {
    (issue_piece<J>(st, slot_of_wave, spare), ...);
  }
  __device__ __forceinline__ void issue(const FzStep& st, char* slot_of_wave, char* spare) const {
    issue(st, slot_of_wave, spare, std::make_integer_sequence<int, PPW>{});
  }

  static constexpr int NRAW = KS ? 2 * NT : NT;
  using RawT = typename std::conditional<KS, u32x2, u32x4>::type;
  // LDS byte offset of tile TI behind rd[0]: K-contiguous tiles of 16 rows (natural) or pairs of 32 (paired); GATED: the second half of
  // the tiles lies BN / 2 rows further on
  static constexpr int kc_off(int ti) {
    if (!PAIRED) return ti * 16 * SB;
    const int half = GATED && ti >= NT / 2, t = half ? ti - NT / 2 : ti;
    return (half * (ROWS / 2) + (t >> 1) * 32 + (t & 1) * 4) * SB;
  }
  // read I of the NRAW that make up the wave's fragments of MFMA step H of the slot at LDS byte address sb
  template <int H, int I>
  __device__ __forceinline__ void read(unsigned sb, RawT (&f)[NRAW]) const {
    if constexpr (!KS) {
      if constexpr (ODD && I == NT - 1) f[I] = g16d_read128(sb + rd[HALVES + H], 0);
      else f[I] = g16d_read128(sb + rd[H], kc_off(I));
    } else {
      constexpr int TI = I / 2;
      f[I] = g16d_read_tr(sb + rd[PAIRED ? TI >> 1 : TI], H * 32 * PITCH + (PAIRED ? (TI & 1) * 8 : 0) + (I & 1) * 4 * PITCH);
    }
  }
  static __device__ __forceinline__ void tie(RawT (&f)[NRAW]) {
#pragma unroll
    for (int t = 0; t < NRAW; ++t) asm volatile("" : "+v"(f[t]));
  }
  static __device__ __forceinline__ u32x4 get(const RawT (&f)[NRAW], int t) {
    if constexpr (!KS) return f[t];
    else return u32x4{f[2 * t][0], f[2 * t][1], f[2 * t + 1][0], f[2 * t + 1][1]};
  }
};

// CN (4 or 8) consecutive entries of a row vector (out of range: 0)
template <typename T, int CN>
__device__ __forceinline__ void fz_load(const void* p, int64_t at, int n, int N, bool vec, float (&v)[CN]) {
  const T* src = static_cast<const T*>(p) + at;
  if (vec) {
    using V = typename std::conditional<sizeof(T) * CN == 8, u32x2, u32x4>::type;
    T t[CN];
    constexpr int Q = (int)(sizeof(T) * CN / sizeof(V));
#pragma unroll
    for (int q = 0; q < Q; ++q) reinterpret_cast<V*>(t)[q] = reinterpret_cast<const V*>(src)[q];
#pragma unroll
    for (int e = 0; e < CN; ++e) v[e] = (float)t[e];
  } else {
#pragma unroll
    for (int e = 0; e < CN; ++e) v[e] = n + e < N ? (float)src[e] : 0.f;
  }
}
template <typename T>
__device__ __forceinline__ void fz_load8(const void* p, int64_t at, int n, int N, bool vec, float (&v)[8]) {
  fz_load<T, 8>(p, at, n, N, vec, v);
}
template <typename T>
__device__ __forceinline__ void fz_store8(void* p, int64_t at, int n, int N, bool vec, const float (&v)[8]) {
  T* dst = static_cast<T*>(p) + at;
  if (vec) {
    T t[8];
    constexpr int Q = (int)sizeof(T) * 8 / 16;
#pragma unroll
    for (int e = 0; e < 8; ++e) t[e] = (T)v[e];
#pragma unroll
    for (int q = 0; q < Q; ++q) reinterpret_cast<u32x4*>(dst)[q] = reinterpret_cast<const u32x4*>(t)[q];
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (n + e < N) dst[e] = (T)v[e];
  }
}
template <typename T, int CN>
__device__ __forceinline__ void fz_bias(const FzEpi& ep, int64_t at, int n, int N, bool vec, float (&v)[CN]) {
  if (ep.bias_f32) fz_load<float, CN>(ep.bias, at, n, N, vec, v);
  else fz_load<T, CN>(ep.bias, at, n, N, vec, v);
}
// p for the backward pass: fp32 as it is; 16-bit types keep 24 bits of the fp32 value (sign, exponent, 15 bits) rounded to nearest, off by at
// most 2^-16 of it, as a plane of its upper 16 bits and, behind it, one of the next 8.  Rounded to 16 bits, p alone would cost the gradients as
// much as their own rounding does.  total: elements of p
//
// The bits of v with half a unit of the 24 added, whose upper 24 are the rounded value: a carry runs into the exponent as it should, and an
// infinity stays one.  A NaN is left alone: the carry out of a full payload would run into the sign.
__device__ __forceinline__ unsigned fz_near24(float v) { return __float_as_uint(v) + (v == v ? 0x80u : 0u); }
__device__ __forceinline__ void fz_split24(const float (&v)[8], u32x4& hi, u32x2& lo) {
  unsigned u[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) u[e] = fz_near24(v[e]);
#pragma unroll
  for (int e = 0; e < 4; ++e) hi[e] = __builtin_amdgcn_perm(u[2 * e + 1], u[2 * e], 0x07060302u);
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    const unsigned x = __builtin_amdgcn_perm(u[4 * e + 1], u[4 * e], 0x0c0c0501u), y = __builtin_amdgcn_perm(u[4 * e + 3], u[4 * e + 2], 0x0c0c0501u);
    lo[e] = __builtin_amdgcn_perm(y, x, 0x05040100u);
  }
}
template <typename TO>
__device__ __forceinline__ void fz_store_pre8(void* pre, int64_t total, int64_t at, int n, int N, const float (&v)[8]) {
  if constexpr (sizeof(TO) == 4) {
    fz_store8<float>(pre, at, n, N, false, v);
  } else {
    uint16_t* hi = static_cast<uint16_t*>(pre) + at;
    uint8_t* lo = reinterpret_cast<uint8_t*>(static_cast<uint16_t*>(pre) + total) + at;
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (n + e < N) {
        hi[e] = (uint16_t)(fz_near24(v[e]) >> 16);
        lo[e] = (uint8_t)(fz_near24(v[e]) >> 8);
      }
  }
}
// 8 values of the two planes
__device__ __forceinline__ void fz_join24(const u32x4& h, const u32x2& l, float (&v)[8]) {
#pragma unroll
  for (int e = 0; e < 8; ++e)  // bytes: two of h, one of l, a zero
    v[e] = __uint_as_float(__builtin_amdgcn_perm(h[e >> 1], l[e >> 2], (e & 1 ? 0x07060000u : 0x05040000u) | ((e & 3) << 8) | 0x0cu));
}
template <typename TO>
__device__ __forceinline__ void fz_load_pre8(const void* pre, int64_t total, int64_t at, int n, int N, bool vec, float (&v)[8]) {
  if constexpr (sizeof(TO) == 4) {
    fz_load8<float>(pre, at, n, N, vec, v);
  } else {
    const uint16_t* hi = static_cast<const uint16_t*>(pre) + at;
    const uint8_t* lo = reinterpret_cast<const uint8_t*>(static_cast<const uint16_t*>(pre) + total) + at;
    if (vec) {
      fz_join24(*reinterpret_cast<const u32x4*>(hi), *reinterpret_cast<const u32x2*>(lo), v);
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = n + e < N ? __uint_as_float(((unsigned)hi[e] << 16) | ((unsigned)lo[e] << 8)) : 0.f;
    }
  }
}
inline __host__ __device__ bool fz_al16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

// Workgroup -> tile.  The tiles are numbered in bands of 8 row tiles, column by column inside a band, and each of the 8 XCDs (workgroups go
// round-robin over them) takes one contiguous eighth of the numbers: the 32 or 64 tiles in flight on an XCD are a block that shares both
// operands in its L2, and no XCD has more than one tile more than another (a grid of XCDs over the output left 35 tiles to one and 10 to
// another of a 51 x 5 problem: two rounds of its 32 CUs instead of one).
__host__ __device__ inline int fz_per_xcd(int64_t tiles) { return (int)((tiles + 7) >> 3); }
__device__ __forceinline__ bool fz_tile(int b, int tiles_m, int tiles_n, int& tm, int& tn) {
  constexpr int BAND = 8;
  const int tiles = tiles_m * tiles_n, per = fz_per_xcd(tiles);
  const int t = (b & 7) * per + (b >> 3);
  if ((b >> 3) >= per || t >= tiles) return false;
  const int band = t / (BAND * tiles_n), in = t - band * BAND * tiles_n;
  const int h = min(BAND, tiles_m - band * BAND);
  tn = in / h;
  tm = band * BAND + in - tn * h;
  return true;
}

// items issued before MFMA q when n are spread evenly over the first `over` MFMAs
constexpr int fz_share(int q, int n, int over) { return over < 1 || q >= over ? n : (q * n + over - 1) / over; }

// E: operand type; TO: type of out / base / pre; BM x BN tile, waves WR x WC; D: ring slots
template <typename E, typename TO, int BM, int BN, int WR, int WC, int SB, int D, bool A_KS, bool B_KS, int EPI>
struct FzKernel {
  static constexpr int NW = WR * WC, BNO = EPI == FZ_GATED ? BN / 2 : BN;  // BNO: output columns of a tile
  static constexpr bool GATED = EPI == FZ_GATED;
  using OA = FzOperand<BM, WR, NW, SB, A_KS, false, false>;
  using OB = FzOperand<BN, WC, NW, SB, B_KS, true, GATED>;
  static constexpr int STAGE = OA::SLOT + OB::SLOT, SPARE = OA::SPARE || OB::SPARE ? 1024 : 0;
  // A third slot of 64 KiB does not fit the LDS, and what HBM takes to deliver the next one shows.  The 256 x 256 tile's waves therefore ask for one
  // word of every cache line of the slot PFD ahead of the one they fill (into spare LDS: nobody reads it), so that the lines are in the
  // L2 when their turn comes.  The workgroups of an XCD that share rows share them out: 8 row tiles those of B, 4 columns of tiles
  // those of A, one instruction a wave and slot.  dx 4096 x 1280, K = 10240 in three parts: 124 -> 105 us.  Not for other tiles (deeper
  // rings or a second workgroup hide the same: 0 to 3 % slower with it), and not for K of fewer than FAR slots (16384 x 5120, K = 1280: 190 -> 195).
  static constexpr int PF = SB == 128 && BM * BN == 256 * 256 && !GATED, PFD = 2, FAR = 32;
  static constexpr int LDS = D * STAGE + SPARE + (PF ? 256 : 0);
  static constexpr int MI = OA::NT, NI = OB::NT, C = OA::PPW + OB::PPW;
  static_assert(D >= (SB == 64 ? 4 : 2) && (D - 1) * (C + 1) <= 63 && (FE<E>::SIZE == 2 || (!A_KS && !B_KS)), "ring");

  static __device__ __forceinline__ void run(const FzProb& p, const FzEpi& ep, char* smem, int b, int z) {
    const int NO = GATED ? ep.F : p.N;
    const int tiles_m = (p.M + BM - 1) / BM, tiles_n = (NO + BNO - 1) / BNO;
    int tm, tn;
    if (!fz_tile(b, tiles_m, tiles_n, tm, tn)) return;
    const int m0 = tm * BM, n0 = tn * BNO;
    const int lane = threadIdx.x & 63, li = lane & 15, g = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
    const int wr = wave / WC, wc = wave - wr * WC;
    const int vrow = GATED && ep.gate_first ? ep.F : 0, grow = GATED && !ep.gate_first ? ep.F : 0;  // first rows of value and gate in w

    OA oa;
    OB ob;
    oa.setup(p.A, p.lda, m0, p.M, p.K, p.kb, 0, wr, 0);
    // the value rows lead the tile: with the gate half first in memory the descriptor starts at the gate rows and the halves swap
    // places in the tile instead of the offset becoming negative
    ob.setup(p.B, p.ldb, n0, p.N, p.K, p.kb, OA::SLOT, wc, GATED ? ep.F : 0);

    constexpr int ES = FE<E>::SIZE, STEP = SB / ES;
    const int nk = (p.K + STEP - 1) / STEP;
    int slots = nk * p.nseg;
    int seg = 0, left = nk;  // of the next slot to issue: its segment, the slots left in it
    int todo = slots;        // slots left to issue at all
    auto plane = [](unsigned t, int s) { return (int64_t)((t >> (4 * s)) & 15u); };
    int first = 0;
    if constexpr (!GATED) {
      if (p.ksplit > 1) {
        const int from = (int)((int64_t)slots * z / p.ksplit), to = (int)((int64_t)slots * (z + 1) / p.ksplit);
        seg = from / nk;
        first = from - seg * nk;
        left = nk - first;
        slots = todo = to - from;
      }
    }
    oa.seek(plane(p.pa, seg) * p.a_plane + (int64_t)first * oa.kstep);
    ob.seek(plane(p.pb, seg) * p.b_plane + (int64_t)first * ob.kstep);
    struct Steps {
      FzStep a, b;
    };
    auto next = [&]() {
      if (left == 0) {
        if (++seg < p.nseg) {
          oa.seek(plane(p.pa, seg) * p.a_plane);
          ob.seek(plane(p.pb, seg) * p.b_plane);
        }
        left = nk;
      }
      const bool last = --left == 0, dead = todo-- <= 0;
      return Steps{oa.next(last, dead), ob.next(last, dead)};
    };
    const bool far = PF && slots >= FAR, ofb = wave & 1;  // odd waves: B's lines
    unsigned line = K4_OOB;
    if constexpr (PF) {
      const int i = (wave >> 1) + NW / 2 * lane;
      line = ofb ? ob.template ahead<8>(tm & 7, i, p.ldb, n0, p.N) : oa.template ahead<4>(tn & 3, i, p.lda, m0, p.M);
    }
    auto fetch_ahead = [&]() {  // behind the slot that next() has just given; an operation in any case, the waits count it
      if constexpr (PF) {
        const char *const la = oa.cur + (int64_t)(PFD - 1) * oa.kstep, *const lb = ob.cur + (int64_t)(PFD - 1) * ob.kstep;
        const __amdgpu_buffer_rsrc_t rs = __builtin_amdgcn_make_buffer_rsrc(const_cast<char*>(ofb ? lb : la), 0,
                                                                            far && todo >= 0 && left > PFD ? 0x7fffffff : 0, K4_RSRC_FLAGS);
        __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, (k4_lds_ptr)(smem + D * STAGE + SPARE), 4, (int)line, 0, 0, 0);
      }
    };
    char *const wslot = smem + wave * 1024, *const spare = smem + D * STAGE;  // this wave's first DMA piece of slot 0
    constexpr int AHEAD = D == 2 ? 2 : D - 1;  // slots filled before the loop
    for (int s = 0; s < AHEAD; ++s) {
      const Steps n = next();
      oa.issue(n.a, wslot + s * STAGE, spare);
      ob.issue(n.b, wslot + s * STAGE + OA::SLOT, spare);
      fetch_ahead();
    }

    using Acc = typename FE<E>::acc;
    Acc acc[MI][NI];
#pragma unroll
    for (int mi = 0; mi < MI; ++mi)
#pragma unroll
      for (int ni = 0; ni < NI; ++ni) acc[mi][ni] = Acc{0, 0, 0, 0};

    // SB = 64: two steps between barriers.  When the waves meet before step s (even), its fragments are in everyone's registers and step s - 1 is
    // done: both slots are free and take steps s - 1 + D and s + D; steps s + 1 and s + 2 have landed (all DMA but the
    // newest D - 4 steps').  The fragments of the next step are read and its refill is issued BETWEEN the MFMAs: reads over the first
    // 5/8 of the step, so that they have landed at its end, the DMA pieces evenly.
    constexpr int NH = MI * NI, RA = OA::NRAW, RB = OB::NRAW, R = RA + RB;
    const unsigned sbase = (unsigned)(size_t)(k4_lds_ptr)smem;
    struct Frags {
      typename OA::RawT a[RA];
      typename OB::RawT b[RB];
    } f0, f1;
    auto read_one = [&](auto hc, auto ic, unsigned sb, Frags& f) {
      constexpr int H = decltype(hc)::value, I = decltype(ic)::value;
      if constexpr (I < RB) ob.template read<H, I>(sb, f.b);
      else oa.template read<H, I - RB>(sb, f.a);
    };
    k4_wait_vm<(AHEAD - 1) * (C + PF) + PF>();  // (PF: of the operations behind a slot's own, fetch_ahead's)
    __builtin_amdgcn_s_barrier();  // raw: __syncthreads() would drain the DMA queue
    asm volatile("" ::: "memory");
    g16d_for_each([&](auto ic) { read_one(std::integral_constant<int, 0>{}, ic, sbase, f0); }, std::make_integer_sequence<int, R>{});
    int read_at = 0, fill_at = (D - 1) * STAGE;  // bytes
    auto advance = [&](int at) { return at == (D - 1) * STAGE ? 0 : at + STAGE; };
    // The MFMAs of the fragments `now`; between them the reads of the next step's (MFMA step H of the slot at sn) and DMA pieces FROM .. TO
    // of the refill n
    auto compute = [&](Frags& now, Frags& then, auto hc, unsigned sn, const Steps& n, char* fill, auto from, auto to) {
      constexpr int F = decltype(from)::value, ND = decltype(to)::value - F;
      g16d_lgkm<0>();
      OB::tie(now.b);
      OA::tie(now.a);
      __builtin_amdgcn_sched_barrier(0);
      g16d_for_each([&](auto qc) {
        constexpr int Q = decltype(qc)::value;
        acc[Q % MI][Q / MI] = FE<E>::mma(OB::get(now.b, Q / MI), OA::get(now.a, Q % MI), acc[Q % MI][Q / MI]);
        constexpr int r0 = fz_share(Q, R, NH * 5 / 8), r1 = fz_share(Q + 1, R, NH * 5 / 8), d0 = Q * ND / NH, d1 = (Q + 1) * ND / NH;
        if constexpr (r1 > r0 || d1 > d0) {
          __builtin_amdgcn_sched_barrier(0);
          g16d_for_each([&](auto ic) { read_one(hc, std::integral_constant<int, r0 + decltype(ic)::value>{}, sn, then); },
                        std::make_integer_sequence<int, r1 - r0>{});
          g16d_for_each([&](auto ic) {
            constexpr int P = F + d0 + decltype(ic)::value;
            if constexpr (P < OA::PPW) oa.template issue_piece<P>(n.a, fill, spare);
            else ob.template issue_piece<P - OA::PPW>(n.b, fill + OA::SLOT, spare);
          }, std::make_integer_sequence<int, d1 - d0>{});
          __builtin_amdgcn_sched_barrier(0);
        }
      }, std::make_integer_sequence<int, NH>{});
    };
    auto meet = [&](auto outstanding) {  // the fragments that are about to be used have been read, and so many DMA operations may be in flight
      k4_wait_vm<decltype(outstanding)::value>();
      g16d_lgkm<0>();
      __builtin_amdgcn_s_barrier();
      asm volatile("" ::: "memory");
    };
    using I0 = std::integral_constant<int, 0>;
    using IC = std::integral_constant<int, C>;
    if constexpr (SB == 64) {
      for (int s = 0; s < slots; s += 2) {  // an odd number of steps ends with one of zeros
        auto step = [&](Frags& now, Frags& then, auto first) {
          char* fill = wslot + fill_at;
          fill_at = advance(fill_at);
          read_at = advance(read_at);
          const Steps n = next();
          if constexpr (decltype(first)::value) meet(std::integral_constant<int, (D - 4) * C>{});
          compute(now, then, I0{}, sbase + (unsigned)read_at, n, fill, I0{}, IC{});
        };
        step(f0, f1, std::true_type{});
        step(f1, f0, std::false_type{});
      }
    } else if constexpr (D == 2) {
      // SB = 128, two slots: the waves meet in the middle of slot k, when all of it is in registers; it takes slot k + 2 while slot k + 1,
      // landed by then, is read
      int at = 0;
      for (int s = 0; s < slots; ++s) {
        const Steps n = next();
        compute(f0, f1, std::integral_constant<int, OA::HALVES - 1>{}, sbase + (unsigned)at, n, wslot, I0{}, I0{});
        meet(std::integral_constant<int, PF>{});
        compute(f1, f0, I0{}, sbase + (unsigned)(STAGE - at), n, wslot + at, I0{}, IC{});
        fetch_ahead();
        at = STAGE - at;
      }
    } else {
      // SB = 128: one slot, two steps, between barriers.  When the waves meet before slot k, slot k - 1 is free and takes slot k - 1 + D, and
      // slot k + 1 has landed (all DMA but the newest D - 3 slots').  (With D = 3 nothing may be in flight at a meeting: 140 -> 184 us for
      // dx 4096 x 1280 x 10240 on 128 x 160; with D = 4: 117.)
      for (int s = 0; s < slots; ++s) {
        char* fill = wslot + fill_at;
        fill_at = advance(fill_at);
        const unsigned sb = sbase + (unsigned)read_at;
        read_at = advance(read_at);
        const Steps n = next();
        meet(std::integral_constant<int, (D - 3) * (C + PF) + PF>{});
        using IH = std::integral_constant<int, C / 2>;
        compute(f0, f1, std::integral_constant<int, OA::HALVES - 1>{}, sb, n, fill, I0{}, IH{});
        compute(f1, f0, I0{}, sbase + (unsigned)read_at, n, fill, IH{}, IC{});
        fetch_ahead();
      }
    }
    // the reads and refills behind the last step have landed before their registers and LDS are given up
    g16d_lgkm<0>();
    OB::tie(f0.b);
    OA::tie(f0.a);
    OB::tie(f1.b);
    OA::tie(f1.a);
    k4_wait_vm<0>();
    __builtin_amdgcn_sched_barrier(0);

    if constexpr (!GATED) {
      if (p.ksplit > 1) {  // raw sums, 16 bytes a lane
        char* part = static_cast<char*>(ep.part) + (int64_t)z * p.M * p.N * 4;
        const bool v4 = (p.N & 3) == 0;
#pragma unroll
        for (int mi = 0; mi < MI; ++mi) {
          const int m = m0 + wr * (BM / WR) + 16 * mi + li;
#pragma unroll
          for (int ni = 0; ni < NI; ++ni) {
            const int n = n0 + wc * (BN / WC) + (OB::ODD && ni == NI - 1 ? 16 * ni + 4 * g : 32 * (ni >> 1) + 8 * g + 4 * (ni & 1));
            if (m >= p.M || n >= p.N) continue;
            char* at = part + ((int64_t)m * p.N + n) * 4;
            if (v4) {
              *reinterpret_cast<Acc*>(at) = acc[mi][ni];
            } else {
#pragma unroll
              for (int e = 0; e < 4; ++e)
                if (n + e < p.N) reinterpret_cast<decltype(+acc[mi][ni][0])*>(at)[e] = acc[mi][ni][e];
            }
          }
        }
        return;
      }
    }

    // ---- epilogue: acc[mi][2 q + e] of lane (li, g) is row 16 mi + li, columns 32 q + 8 g + 4 e .. + 3 of the wave's part; an odd last
    //      tile is columns 16 ni + 4 g .. + 3.  It is vector work that the matrix pipe waits for with one workgroup a CU, so addresses
    //      are 32-bit offsets into descriptors of the tile's rows: rows beyond M lie beyond them, columns beyond NO are masked.
    //      Measured on 256 x 256 tiles: 4 us with two scales and no more, 8 us with the gelu of 128 columns; a workgroup's beginning,
    //      before its first step's operands have landed, is 1.3 - 2 us --------------------------------------------------------------
    constexpr int TS = (int)sizeof(TO), H = GATED ? 2 : 1;
    const float alpha = EPI == FZ_PLAIN && ep.alpha ? *ep.alpha : 1.f;
    const bool vec = (NO & 7) == 0 && fz_al16(ep.out) && fz_al16(ep.base) && fz_al16(ep.pre) && fz_al16(ep.bias) && fz_al16(ep.sw);
    const int row0 = wr * (BM / WR) + li, colw = n0 + wc * (BNO / WC);
    float sa[MI];
#pragma unroll
    for (int mi = 0; mi < MI; ++mi) sa[mi] = ep.sa && m0 + row0 + 16 * mi < p.M ? ep.sa[m0 + row0 + 16 * mi] : 1.f;

    const int64_t rows = p.M - m0;
    auto open_rows = [&](const void* base, int64_t row, int64_t pitch, bool have) {
      const int64_t bytes = have ? rows * pitch : 0;
      return __builtin_amdgcn_make_buffer_rsrc(const_cast<char*>(static_cast<const char*>(base)) + row * pitch, 0,
                                               (int)(bytes > 0x7fffffff ? 0x7fffffff : bytes), K4_RSRC_FLAGS);
    };
    const int po = NO * TS, pb = po * H, ph = NO * (TS == 4 ? 8 : 4), pl = NO * 2;  // pitches: out, base, p and its 8-bit plane
    const __amdgpu_buffer_rsrc_t ro = open_rows(ep.out, m0, po, true), rb = open_rows(ep.base, m0, pb, ep.base != nullptr);
    const __amdgpu_buffer_rsrc_t rh = open_rows(ep.pre, m0, ph, GATED && ep.pre),
                                 rl = open_rows(static_cast<char*>(ep.pre) + 2 * ep.pre_total, m0, pl, GATED && ep.pre && TS == 2);

    // CN columns from n on, of every row tile; get(mi, e, half): their sums
    auto emit = [&](auto cn, int n, auto get) {
      constexpr int CN = decltype(cn)::value;
      const bool in = n < NO;
      float s1[CN], s2[CN], c1[CN], c2[CN];
#pragma unroll
      for (int e = 0; e < CN; ++e) s1[e] = s2[e] = 1.f, c1[e] = c2[e] = 0.f;
      if (EPI != FZ_PLAIN && in) {
        if (FE<E>::SIZE == 1) {
          fz_load<float, CN>(ep.sw, vrow + n, n, NO, vec, s1);
          if (GATED) fz_load<float, CN>(ep.sw, grow + n, n, NO, vec, s2);
        }
        if (ep.bias) {
          fz_bias<TO, CN>(ep, vrow + n, n, NO, vec, c1);
          if (GATED) fz_bias<TO, CN>(ep, grow + n, n, NO, vec, c2);
        }
      }
      struct Row {
        TO x[CN];
      };
      auto fetch = [&](const __amdgpu_buffer_rsrc_t& r, unsigned off, Row& t) {
        if constexpr (TS * CN == 8) {
          reinterpret_cast<u32x2*>(t.x)[0] = __builtin_bit_cast(u32x2, __builtin_amdgcn_raw_buffer_load_b64(r, (int)off, 0, 0));
        } else {
#pragma unroll
          for (int i = 0; i < TS * CN / 16; ++i)
            reinterpret_cast<u32x4*>(t.x)[i] = __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(r, (int)(off + 16 * i), 0, 0));
        }
      };
      auto store = [&](const __amdgpu_buffer_rsrc_t& r, unsigned off, const float (&x)[CN]) {
        TO t[CN];
#pragma unroll
        for (int e = 0; e < CN; ++e) t[e] = (TO)x[e];
        if constexpr (TS * CN == 8) {
          __builtin_amdgcn_raw_buffer_store_b64(reinterpret_cast<u32x2*>(t)[0], r, (int)off, 0, 0);
        } else {
#pragma unroll
          for (int i = 0; i < TS * CN / 16; ++i) __builtin_amdgcn_raw_buffer_store_b128(reinterpret_cast<u32x4*>(t)[i], r, (int)(off + 16 * i), 0, 0);
        }
      };
      auto keep = [&](unsigned hoff, unsigned loff, int col, const float (&x)[CN]) {  // p for the backward pass
        if constexpr (GATED) {
          if constexpr (TS == 4) {
            store(rh, hoff + col * 4, x);
          } else {
            u32x4 hi;
            u32x2 lo;
            fz_split24(x, hi, lo);
            __builtin_amdgcn_raw_buffer_store_b128(hi, rh, (int)(hoff + col * 2), 0, 0);
            __builtin_amdgcn_raw_buffer_store_b64(lo, rl, (int)(loff + col), 0, 0);
          }
        }
      };
      // the base operand of GR row tiles is asked for at once: behind a store the next load would wait for itself
      constexpr int GR = TS == 2 ? (MI < 4 ? MI : 4) : 2;
      Row bv[GR], bt[GR];
#pragma unroll
      for (int mi = 0; mi < MI; ++mi) {
        const int r = row0 + 16 * mi;
        const int64_t m = m0 + r;
        if (EPI != FZ_PLAIN && vec && ep.base && mi % GR == 0) {
#pragma unroll
          for (int j = 0; j < GR; ++j) {
            const unsigned off = in ? (unsigned)((r + 16 * j) * pb + n * TS) : K4_OOB;
            fetch(rb, off + vrow * TS, bv[j]);
            if (GATED) fetch(rb, off + grow * TS, bt[j]);
          }
        }
        if (!vec && (m >= p.M || !in)) continue;
        float v[CN], t[CN];
#pragma unroll
        for (int e = 0; e < CN; ++e) {
          const float a = (float)get(mi, e, 0), b = GATED ? (float)get(mi, e, 1) : 0.f;
          v[e] = GATED && ep.gate_first ? b : a;  // the tile's first half holds the rows that come first in w
          t[e] = ep.gate_first ? a : b;
        }
        if constexpr (EPI == FZ_PLAIN) {
#pragma unroll
          for (int e = 0; e < CN; ++e) v[e] = v[e] * alpha * sa[mi];
        } else {
#pragma unroll
          for (int e = 0; e < CN; ++e) {
            v[e] = FE<E>::SIZE == 1 ? fmaf(v[e] * sa[mi], s1[e], c1[e]) : v[e] + c1[e];
            if (GATED) t[e] = FE<E>::SIZE == 1 ? fmaf(t[e] * sa[mi], s2[e], c2[e]) : t[e] + c2[e];
          }
          if (ep.base) {
            if (vec) {
#pragma unroll
              for (int e = 0; e < CN; ++e) {
                v[e] += (float)bv[mi % GR].x[e];
                if (GATED) t[e] += (float)bt[mi % GR].x[e];
              }
            } else {
              float x[CN];
              fz_load<TO, CN>(ep.base, m * H * NO + vrow + n, n, NO, false, x);
#pragma unroll
              for (int e = 0; e < CN; ++e) v[e] += x[e];
              if (GATED) {
                fz_load<TO, CN>(ep.base, m * H * NO + grow + n, n, NO, false, x);
#pragma unroll
                for (int e = 0; e < CN; ++e) t[e] += x[e];
              }
            }
          }
          if constexpr (GATED) {
            if (ep.pre) {
              if (vec) {
                const unsigned hoff = in ? (unsigned)(r * ph + n * (TS == 4 ? 4 : 2)) : K4_OOB, loff = in ? (unsigned)(r * pl + n) : K4_OOB;
                keep(hoff, loff, vrow, v);
                keep(hoff, loff, grow, t);
              } else {
                const int64_t at = m * 2 * NO;
                fz_store_pre8<TO>(ep.pre, ep.pre_total, at + vrow + n, n, NO, v);
                fz_store_pre8<TO>(ep.pre, ep.pre_total, at + grow + n, n, NO, t);
              }
            }
            fz_for_act(ep.act, [&](auto ac) {
#pragma unroll
              for (int e = 0; e < CN; ++e) v[e] *= fz_act<decltype(ac)::value>(t[e]);
            });
          }
        }
        if (vec) {
          store(ro, in ? (unsigned)(r * po + n * TS) : K4_OOB, v);
        } else {
          TO* dst = static_cast<TO*>(ep.out) + m * NO + n;
#pragma unroll
          for (int e = 0; e < CN; ++e)
            if (n + e < NO) dst[e] = (TO)v[e];
        }
      }
    };
    constexpr int NQ = GATED ? NI / 4 : NI / 2;
    g16d_for_each([&](auto qc) {
      constexpr int Q = decltype(qc)::value;
      emit(std::integral_constant<int, 8>{}, colw + 32 * Q + 8 * g, [&](int mi, int e, int half) { return acc[mi][half * (NI / 2) + 2 * Q + (e >> 2)][e & 3]; });
    }, std::make_integer_sequence<int, NQ>{});
    if constexpr (OB::ODD)
      emit(std::integral_constant<int, 4>{}, colw + 16 * (NI - 1) + 4 * g, [&](int mi, int e, int) { return acc[mi][NI - 1][e]; });
  }
};

template <typename K>
constexpr int fz_waves_per_simd() { return K::NW * (2 * K::LDS <= 160 * 1024 ? 2 : 1) / 4; }

template <typename K>
__global__ __launch_bounds__(K::NW * 64, fz_waves_per_simd<K>()) void fz_gemm_kernel(FzProb p, FzEpi ep) {
  extern __shared__ __attribute__((aligned(1024))) char fz_smem[];
  K::run(p, ep, fz_smem, (int)blockIdx.x, (int)blockIdx.y);
}

// the sums of a split K joined in the order of K, then the epilogue (PLAIN, LINEAR).  Bound by HBM (4 parts of 5120 x 640: 10 us, 59 MB) or, for
// few outputs, by the latency of its loads: four parts are in flight
template <typename E, typename TO>
__global__ __launch_bounds__(256) void fz_reduce_kernel(FzProb p, FzEpi ep) {
  using S = typename std::conditional<FE<E>::SIZE == 1, int, float>::type;
  const int N = p.N, chunks = (N + 7) >> 3;
  const int64_t plane = (int64_t)p.M * N, total = (int64_t)p.M * chunks;
  const bool pitch8 = (N & 7) == 0, vo = pitch8 && fz_al16(ep.out) && fz_al16(ep.base), vb = pitch8 && fz_al16(ep.bias), vs = pitch8 && fz_al16(ep.sw);
  const float alpha = ep.alpha ? *ep.alpha : 1.f;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < total; i += (int64_t)gridDim.x * 256) {
    const int64_t m = i / chunks;
    const int n = (int)(i - m * chunks) * 8;
    const S* src = static_cast<const S*>(ep.part) + m * N + n;
    S s[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) s[e] = 0;
    for (int z0 = 0; z0 < p.ksplit; z0 += 4) {  // four parts' loads in flight: what lies beyond the last part or column is read again, not used
      S part[4][8];
#pragma unroll
      for (int z = 0; z < 4; ++z) {
        const S* at = src + min(z0 + z, p.ksplit - 1) * plane;
        if (pitch8) {
          const u32x4 a = reinterpret_cast<const u32x4*>(at)[0], b = reinterpret_cast<const u32x4*>(at)[1];
#pragma unroll
          for (int e = 0; e < 8; ++e) part[z][e] = __builtin_bit_cast(S, e < 4 ? a[e & 3] : b[e & 3]);
        } else {
#pragma unroll
          for (int e = 0; e < 8; ++e) part[z][e] = at[min(e, N - 1 - n)];
        }
      }
#pragma unroll
      for (int z = 0; z < 4; ++z)
#pragma unroll
        for (int e = 0; e < 8; ++e) s[e] += z0 + z < p.ksplit ? part[z][e] : 0;
    }
    float v[8], t[8];
    const float sa = ep.sa ? ep.sa[m] : 1.f;
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = (float)s[e] * alpha * sa;
    if (ep.sw) {
      fz_load8<float>(ep.sw, n, n, N, vs, t);
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] *= t[e];
    }
    if (ep.bias) {
      fz_bias<TO, 8>(ep, n, n, N, vb, t);
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] += t[e];
    }
    if (ep.base) {
      fz_load8<TO>(ep.base, m * N + n, n, N, vo, t);
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] += t[e];
    }
    fz_store8<TO>(ep.out, m * N + n, n, N, vo, v);
  }
}

}  // namespace lyc
