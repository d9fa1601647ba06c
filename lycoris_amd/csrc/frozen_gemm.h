// frozen_gemm.h -- the matrix products of the 8-bit frozen layer and of the gated projection.
//
//     8-bit forward   acc[m, n] = sum_k aq[m, k] bq[n, k]          both operands K-contiguous, int32 accumulators
//     gated forward   p[m, n]   = sum_k x[m, k] w[n, k]            both operands K-contiguous; w is [2 F, K]
//     dx              dx[m, i]  = sum_o dp[m, o] w[o, i]           A K-contiguous, B K-strided
//     dw              dw[o, i]  = sum_m dp[m, o] x[m, i]           both K-strided
//
// The skeleton is gemm16d.h's: both operands go HBM -> LDS by LDS-DMA into a ring of K steps of 128 BYTES, fragments are read one K half
// ahead of the MFMAs that use them, the MFMA roles are swapped and the n tiles formed in pairs so that a lane owns 8 consecutive output
// columns of one row.  Since every address is formed in bytes, 8-bit operands (128 k per step, v_mfma_i32_16x16x64_i8) and 16-bit ones
// (64 k, v_mfma_f32_16x16x32) run the same loop: a fragment is 16 bytes of one row either way, and the matrix pipe takes the same
// 16 cycles for it.  What differs from gemm16d.h:
//
//   * the buffer descriptor is rebased on every K step (scalar adds beside the matrix pipe) instead of walked with a 32-bit offset: an
//     operand may be larger than 4 GiB;
//   * a K that is not a multiple of the step is masked in the DMA of the last step, 16 bytes at a time (both operands: 0 times a stray NaN
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

// act(t) and its derivative in fp32
__device__ __forceinline__ float fz_act(int act, float t) {
  if (act == FZ_ACT_SILU) return t / (1.f + __expf(-t));
  if (act == FZ_ACT_GELU) return 0.5f * t * erfcf(-0.70710678118654752f * t);
  const float u = 0.79788456080286536f * (t + 0.044715f * t * t * t);
  return t / (1.f + __expf(-2.f * u));  // 0.5 t (1 + tanh u)
}
__device__ __forceinline__ void fz_act_grad(int act, float t, float& a, float& da) {
  if (act == FZ_ACT_SILU) {
    const float s = 1.f / (1.f + __expf(-t));
    a = t * s;
    da = s + a * (1.f - s);
  } else if (act == FZ_ACT_GELU) {
    const float cdf = 0.5f * erfcf(-0.70710678118654752f * t);
    a = t * cdf;
    da = cdf + t * 0.39894228040143268f * __expf(-0.5f * t * t);
  } else {
    const float u = 0.79788456080286536f * (t + 0.044715f * t * t * t);
    const float s = 1.f / (1.f + __expf(-2.f * u));
    a = t * s;
    da = s + 2.f * a * (1.f - s) * 0.79788456080286536f * (1.f + 0.134145f * t * t);
  }
}

// One product.  lda / ldb in bytes.  kb: bytes of K along a K-contiguous operand, rounded up to 16 (what the operand's rows hold up to
// there has to be finite in 16 bits, and zero in A's rows in 8 bits).  Planes of segment s: (pa >> 4 s) & 15 and (pb >> 4 s) & 15.
struct FzProb {
  const void *A, *B;
  int64_t lda, ldb, a_plane, b_plane;
  int M, N, K, kb;
  int nseg;
  unsigned pa, pb;
};

enum { FZ_PLAIN = 0, FZ_LINEAR = 1, FZ_GATED = 2 };
struct FzEpi {
  void* out;           // [M, N] (GATED: [M, F]), row pitch = N (F) elements
  void* pre;           // GATED: p [M, 2 F] or null
  const float* alpha;  // PLAIN: device scalar on the result, or null
  const float *sa, *sw;  // 8-bit: scales of A's rows, of B's rows
  const void* bias;    // [N] (GATED: [2 F]) or null; fp32 when bias_f32, else the output's type
  const void* base;    // [M, N] (GATED: [M, 2 F]) in the output's type, or null
  int bias_f32, act, gate_first, F;
};

// One operand of one workgroup tile; gemm16d.h's G16DOperand with the tile split over W waves along this extent, NW in all.
template <int ROWS, int W, int NW, bool KS, bool PAIRED, bool GATED>
struct FzOperand {
  static constexpr int PIECES = ROWS / 8, PPW = PIECES / NW;
  static constexpr int WEXT = ROWS / W, NT = WEXT / 16;
  static constexpr int CH = ROWS / 8, PITCH = ROWS * 2;  // KS (16-bit): chunks and bytes per k row
  static constexpr int NADDR = KS ? (PAIRED ? NT / 2 : NT) : 2;
  static_assert(PIECES % NW == 0 && (!PAIRED || NT % 2 == 0) && (!GATED || (PAIRED && !KS && NT % 4 == 0)), "tile shape");

  unsigned voff[PPW], rd[NADDR];
  bool tail;             // K-contiguous: this lane's chunk lies beyond K in the last step of a segment
  const char *org, *cur;  // the tile's first byte in plane 0; the next K step's
  int64_t total, left;   // bytes behind them
  unsigned kstep;
  __amdgpu_buffer_rsrc_t rs;

  __device__ __forceinline__ void setup(const void* base, int64_t ld, int r0, int ext, int kdim, int kb, int stage_off, int wsel, int second) {
    const int lane = threadIdx.x & 63, li = lane & 15, g = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
    if constexpr (!KS) {
      const int64_t skip = (int64_t)r0 * ld;
      org = static_cast<const char*>(base) + skip;
      total = (int64_t)(ext - 1) * ld + kb - skip;
      kstep = 128;
#pragma unroll
      for (int j = 0; j < PPW; ++j) {
        const int r = 8 * (wave + NW * j) + (lane >> 3), c = (lane & 7) ^ g16d_swz_kc<PAIRED>(r);
        // GATED: rows 0 .. BN / 2 are the half whose first row is `base`, the others the half `second` rows further on
        const int gr = !GATED || r < ROWS / 2 ? r : second + r - ROWS / 2;
        voff[j] = (unsigned)gr * (unsigned)ld + (unsigned)c * 16u;
        tail = ((kb - 1) & ~127) + c * 16 >= kb;  // c does not depend on j: 8 NW rows are a multiple of the swizzle's period
      }
      const int r = wsel * (GATED ? WEXT / 2 : WEXT) + (PAIRED ? 8 * (li >> 2) + (li & 3) : li);
      const int x = g16d_swz_kc<PAIRED>(r);
#pragma unroll
      for (int kk = 0; kk < 2; ++kk) rd[kk] = (unsigned)(stage_off + r * 128 + (((4 * kk + g) ^ x) << 4));
    } else {
      const int64_t skip = (int64_t)r0 * 2;
      org = static_cast<const char*>(base) + skip;
      total = (int64_t)(kdim - 1) * ld + (((int64_t)ext + 7) & ~7) * 2 - skip;
      kstep = 64u * (unsigned)ld;
      tail = false;
      constexpr int RP = 1024 / PITCH;
#pragma unroll
      for (int j = 0; j < PPW; ++j) {
        const int kr = RP * (wave + NW * j) + lane / CH, c = (lane % CH) ^ g16d_swz_ks<PAIRED, CH>(kr);
        voff[j] = (r0 + 8 * c < ext) ? (unsigned)kr * (unsigned)ld + (unsigned)c * 16u : K4_OOB;
      }
      const int rho = li >> 2, quad = li & 3, x = g16d_swz_ks<PAIRED, CH>(rho), krow = 8 * g + rho;
#pragma unroll
      for (int t = 0; t < NADDR; ++t) {
        const int col = wsel * WEXT + (PAIRED ? 32 * t + 8 * quad : 16 * t + 4 * quad);
        rd[t] = (unsigned)(stage_off + krow * PITCH + (((col >> 3) ^ x) << 4) + (col & 7) * 2);
      }
    }
  }
  __device__ __forceinline__ void seek(int64_t plane_off) {
    cur = org + plane_off;
    left = total;
  }
  // descriptor of the next K step; `dead`: nothing is left to fetch (the refills behind the last step read nothing and store zeros)
  __device__ __forceinline__ void open(bool dead) {
    const int64_t n = dead ? 0 : left;
    rs = __builtin_amdgcn_make_buffer_rsrc(const_cast<char*>(cur), 0, (int)(n < 0 ? 0 : n > 0x7fffffff ? 0x7fffffff : n), K4_RSRC_FLAGS);
    cur += kstep;
    left -= kstep;
  }
  template <int J>
  __device__ __forceinline__ void issue_piece(char* slot, bool last) const {
    const int wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
    const unsigned v = (!KS && last && tail) ? K4_OOB : voff[J];
    __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, (k4_lds_ptr)(slot + (wave + NW * J) * 1024), 16, (int)v, 0, 0, 0);
  }
  template <int... J>
  __device__ __forceinline__ void issue(char* slot, bool last, std::integer_sequence<int, J...>) const {
    (issue_piece<J>(slot, last), ...);
  }
  __device__ __forceinline__ void issue(char* slot, bool last) const { issue(slot, last, std::make_integer_sequence<int, PPW>{}); }

  static constexpr int NRAW = KS ? 2 * NT : NT;
  using RawT = typename std::conditional<KS, u32x2, u32x4>::type;
  // LDS byte offset of tile TI behind rd[]: K-contiguous tiles of 16 rows (natural) or pairs of 32 (paired); GATED: the second half of
  // the tiles lies BN / 2 rows further on
  static constexpr int kc_off(int ti) {
    if (!PAIRED) return ti * 2048;
    const int half = GATED && ti >= NT / 2, t = half ? ti - NT / 2 : ti;
    return half * (ROWS / 2) * 128 + (t >> 1) * 4096 + (t & 1) * 512;
  }
  template <int KK, int... TI>
  __device__ __forceinline__ void read(unsigned sb, RawT (&f)[NRAW], std::integer_sequence<int, TI...>) const {
    if constexpr (!KS) {
      ((f[TI] = g16d_read128(sb + rd[KK], kc_off(TI))), ...);
    } else {
      ((f[2 * TI] = g16d_read_tr(sb + rd[PAIRED ? TI >> 1 : TI], KK * 32 * PITCH + (PAIRED ? (TI & 1) * 8 : 0)),
        f[2 * TI + 1] = g16d_read_tr(sb + rd[PAIRED ? TI >> 1 : TI], KK * 32 * PITCH + (PAIRED ? (TI & 1) * 8 : 0) + 4 * PITCH)),
       ...);
    }
  }
  template <int KK>
  __device__ __forceinline__ void read(unsigned sb, RawT (&f)[NRAW]) const {
    read<KK>(sb, f, std::make_integer_sequence<int, NT>{});
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

// 8 consecutive entries of a row vector (out of range: 0)
template <typename T>
__device__ __forceinline__ void fz_load8(const void* p, int64_t at, int n, int N, bool vec, float (&v)[8]) {
  const T* src = static_cast<const T*>(p) + at;
  if (vec) {
    T t[8];
    constexpr int Q = (int)sizeof(T) * 8 / 16;
#pragma unroll
    for (int q = 0; q < Q; ++q) reinterpret_cast<u32x4*>(t)[q] = reinterpret_cast<const u32x4*>(src)[q];
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = (float)t[e];
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = n + e < N ? (float)src[e] : 0.f;
  }
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
template <typename T>
__device__ __forceinline__ void fz_bias8(const FzEpi& ep, int64_t at, int n, int N, bool vec, float (&v)[8]) {
  if (ep.bias_f32) fz_load8<float>(ep.bias, at, n, N, vec, v);
  else fz_load8<T>(ep.bias, at, n, N, vec, v);
}
inline __host__ __device__ bool fz_al16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

// E: operand type; TO: type of out / base / pre; BM x BN tile, waves WR x WC; D: ring slots
template <typename E, typename TO, int BM, int BN, int WR, int WC, int D, bool A_KS, bool B_KS, int EPI>
struct FzKernel {
  static constexpr int NW = WR * WC, STAGE = (BM + BN) * 128, LDS = D * STAGE;
  static constexpr bool GATED = EPI == FZ_GATED;
  using OA = FzOperand<BM, WR, NW, A_KS, false, false>;
  using OB = FzOperand<BN, WC, NW, B_KS, true, GATED>;
  static constexpr int MI = OA::NT, NI = OB::NT, C = OA::PPW + OB::PPW;
  static_assert(D >= 2 && (D - 1) * C <= 63 && (FE<E>::SIZE == 2 || (!A_KS && !B_KS)), "ring");

  static __device__ __forceinline__ void run(const FzProb& p, const FzEpi& ep, char* smem, int b) {
    constexpr int BNO = GATED ? BN / 2 : BN;  // output columns of a tile
    const int NO = GATED ? ep.F : p.N;
    const int tiles_m = (p.M + BM - 1) / BM, tiles_n = (NO + BNO - 1) / BNO;
    const G16DMap mp = gemm16d_map(tiles_m, tiles_n, p.M, p.N);
    const int xcd = b & 7, idx = b >> 3;
    const int ln = idx / mp.tm_per, lm = idx - ln * mp.tm_per;
    const int tm = (xcd & ((1 << mp.lgm) - 1)) * mp.tm_per + lm, tn = (xcd >> mp.lgm) * mp.tn_per + ln;
    if (ln >= mp.tn_per || tm >= tiles_m || tn >= tiles_n) return;
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
    ob.setup(p.B, p.ldb, n0, p.N, p.K, p.kb, BM * 128, wc, GATED ? ep.F : 0);

    constexpr int ES = FE<E>::SIZE, STEP = 128 / ES;
    const int nk = (p.K + STEP - 1) / STEP, steps = nk * p.nseg;
    int seg = 0, kin = 0;  // of the next step to issue
    auto plane = [](unsigned t, int s) { return (int64_t)((t >> (4 * s)) & 15u); };
    oa.seek(plane(p.pa, 0) * p.a_plane);
    ob.seek(plane(p.pb, 0) * p.b_plane);
    bool last = false;
    auto open = [&]() {
      const bool dead = seg >= p.nseg;
      last = kin == nk - 1;
      oa.open(dead);
      ob.open(dead);
      if (++kin == nk) {
        kin = 0;
        ++seg;
        if (seg < p.nseg) {
          oa.seek(plane(p.pa, seg) * p.a_plane);
          ob.seek(plane(p.pb, seg) * p.b_plane);
        }
      }
    };
    for (int s = 0; s < D; ++s) {
      open();
      oa.issue(smem + s * STAGE, last);
      ob.issue(smem + s * STAGE + BM * 128, last);
    }

    using Acc = typename FE<E>::acc;
    Acc acc[MI][NI];
#pragma unroll
    for (int mi = 0; mi < MI; ++mi)
#pragma unroll
      for (int ni = 0; ni < NI; ++ni) acc[mi][ni] = Acc{0, 0, 0, 0};

    constexpr int NH = MI * NI, STRIDE = NH / C, R1 = OA::NRAW + OB::NRAW;
    static_assert(STRIDE >= 1, "refill interleave");
    const unsigned sbase = (unsigned)(size_t)(k4_lds_ptr)smem;
    typename OA::RawT a0[OA::NRAW], a1[OA::NRAW];
    typename OB::RawT b0[OB::NRAW], b1[OB::NRAW];
    k4_wait_vm<(D - 1) * C>();
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    ob.template read<0>(sbase, b0);
    oa.template read<0>(sbase, a0);
    int slot = 0;
    for (int ks = 0; ks < steps; ++ks) {
      const unsigned sb = sbase + (unsigned)(slot * STAGE);
      char* fill = smem + slot * STAGE;
      const int next = slot + 1 == D ? 0 : slot + 1;
      ob.template read<1>(sb, b1);
      oa.template read<1>(sb, a1);
      g16d_lgkm<(R1 > 15 ? 15 : R1)>();
      OB::tie(b0);
      OA::tie(a0);
      __builtin_amdgcn_sched_barrier(0);
      g16d_for_each([&](auto qc) {
        constexpr int Q = decltype(qc)::value;
        acc[Q % MI][Q / MI] = FE<E>::mma(OB::get(b0, Q / MI), OA::get(a0, Q % MI), acc[Q % MI][Q / MI]);
      }, std::make_integer_sequence<int, NH>{});
      __builtin_amdgcn_sched_barrier(0);
      g16d_lgkm<0>();
      OB::tie(b1);
      OA::tie(a1);
      k4_wait_vm<(D - 2) * C>();
      __builtin_amdgcn_s_barrier();
      asm volatile("" ::: "memory");
      const unsigned sn = sbase + (unsigned)(next * STAGE);
      ob.template read<0>(sn, b0);
      oa.template read<0>(sn, a0);
      open();
      __builtin_amdgcn_sched_barrier(0);
      g16d_for_each([&](auto qc) {
        constexpr int Q = decltype(qc)::value;
        acc[Q % MI][Q / MI] = FE<E>::mma(OB::get(b1, Q / MI), OA::get(a1, Q % MI), acc[Q % MI][Q / MI]);
        if constexpr ((Q + 1) % STRIDE == 0 && (Q + 1) / STRIDE <= C) {
          constexpr int P = (Q + 1) / STRIDE - 1;
          __builtin_amdgcn_sched_barrier(0);
          if constexpr (P < OA::PPW) oa.template issue_piece<P>(fill, last);
          else ob.template issue_piece<P - OA::PPW>(fill + BM * 128, last);
          __builtin_amdgcn_sched_barrier(0);
        }
      }, std::make_integer_sequence<int, NH>{});
      slot = next;
    }
    // the reads and refills behind the last step have landed before their registers and LDS are given up
    g16d_lgkm<0>();
    OB::tie(b0);
    OA::tie(a0);
    k4_wait_vm<0>();
    __builtin_amdgcn_sched_barrier(0);

    // ---- epilogue: acc[mi][2 q + e] of lane (li, g) is row 16 mi + li, columns 32 q + 8 g + 4 e .. + 3 of the wave's part ----------
    constexpr int NQ = GATED ? NI / 4 : NI / 2;
    const bool pitch8 = (NO & 7) == 0;
    const bool vo = pitch8 && fz_al16(ep.out) && (!GATED || (fz_al16(ep.pre) && fz_al16(ep.base))) && fz_al16(ep.base);
    const bool vb = pitch8 && fz_al16(ep.bias), vs = pitch8 && fz_al16(ep.sw);
    const float alpha = EPI == FZ_PLAIN && ep.alpha ? *ep.alpha : 1.f;
#pragma unroll
    for (int q = 0; q < NQ; ++q) {
      const int n = n0 + wc * (BNO / WC) + 32 * q + 8 * g;
      const bool nok = n < NO, full = n + 8 <= NO;
      float s1[8], s2[8], c1[8], c2[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) s1[e] = s2[e] = 1.f, c1[e] = c2[e] = 0.f;
      if (nok && EPI != FZ_PLAIN) {
        if (ep.sw) {
          fz_load8<float>(ep.sw, vrow + n, n, NO, vs && full, s1);
          if (GATED) fz_load8<float>(ep.sw, grow + n, n, NO, vs && full, s2);
        }
        if (ep.bias) {
          fz_bias8<TO>(ep, vrow + n, n, NO, vb && full, c1);
          if (GATED) fz_bias8<TO>(ep, grow + n, n, NO, vb && full, c2);
        }
      }
#pragma unroll
      for (int mi = 0; mi < MI; ++mi) {
        const int m = m0 + wr * (BM / WR) + 16 * mi + li;
        if (m >= p.M || !nok) continue;
        float v[8];
        if constexpr (!GATED) {
#pragma unroll
          for (int e = 0; e < 8; ++e) v[e] = (float)acc[mi][2 * q + (e >> 2)][e & 3];
          if constexpr (EPI == FZ_LINEAR) {
            const float sa = ep.sa[m];
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] = v[e] * sa * s1[e] + c1[e];
            if (ep.base) {
              float bs[8];
              fz_load8<TO>(ep.base, (int64_t)m * NO + n, n, NO, vo && full, bs);
#pragma unroll
              for (int e = 0; e < 8; ++e) v[e] += bs[e];
            }
          } else {
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] *= alpha;
          }
          fz_store8<TO>(ep.out, (int64_t)m * NO + n, n, NO, vo && full, v);
        } else {
          float t[8];
          // the tile's first half holds the rows that come first in w: the gate's when gate_first
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const float f = (float)acc[mi][2 * q + (e >> 2)][e & 3], h = (float)acc[mi][NI / 2 + 2 * q + (e >> 2)][e & 3];
            v[e] = ep.gate_first ? h : f;
            t[e] = ep.gate_first ? f : h;
          }
          const float sa = ep.sa ? ep.sa[m] : 1.f;
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            v[e] = v[e] * sa * s1[e] + c1[e];
            t[e] = t[e] * sa * s2[e] + c2[e];
          }
          const int64_t row = (int64_t)m * 2 * NO;
          if (ep.base) {
            float bs[8];
            fz_load8<TO>(ep.base, row + vrow + n, n, NO, vo && full, bs);
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] += bs[e];
            fz_load8<TO>(ep.base, row + grow + n, n, NO, vo && full, bs);
#pragma unroll
            for (int e = 0; e < 8; ++e) t[e] += bs[e];
          }
          if (ep.pre) {  // what the backward pass reads, rounded to the activation type
            fz_store8<TO>(ep.pre, row + vrow + n, n, NO, vo && full, v);
            fz_store8<TO>(ep.pre, row + grow + n, n, NO, vo && full, t);
          }
#pragma unroll
          for (int e = 0; e < 8; ++e) v[e] *= fz_act(ep.act, t[e]);
          fz_store8<TO>(ep.out, (int64_t)m * NO + n, n, NO, vo && full, v);
        }
      }
    }
  }
};

template <typename K>
constexpr int fz_waves_per_simd() { return K::NW * (2 * K::LDS <= 160 * 1024 ? 2 : 1) / 4; }

template <typename K>
__global__ __launch_bounds__(K::NW * 64, fz_waves_per_simd<K>()) void fz_gemm_kernel(FzProb p, FzEpi ep) {
  extern __shared__ __attribute__((aligned(1024))) char fz_smem[];
  K::run(p, ep, fz_smem, (int)blockIdx.x);
}

}  // namespace lyc
