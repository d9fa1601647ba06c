// frozen_skinny.h -- the forward products for up to 32 rows (single tokens, small batches): y = x w^T reads the weight once and is bound by
// that, or by the launch.
//
// A workgroup owns 16 output columns (gated: 16 of each half) and all of K, its waves take 128-byte pieces of K in turn: a weight row's 128
// bytes go to four lanes as two 16-byte loads each, straight into the registers that an MFMA reads (the MFMA's A operand are the 16 weight
// rows, its B operand the activation rows, 16 per row tile; k is permuted alike in both, which no sum notices).  The loads of a wave's first
// PRE pieces are issued before anything is waited for.  Partial sums meet in LDS, 256 threads run the epilogue.
//
// FUSED (8-bit, few activations): every workgroup quantises the rows itself into LDS while its first weight pieces are in flight -- one
// launch instead of two.  The rows are read by all workgroups, out of the L2, so this pays while they are small beside the weight slice.
//
// Measured: 1 x 1280 -> 1280 in 5.3 us and gated 1 x 1280 -> 2 x 5120 (13 MB) in 7.1, quantisation included; 16 x 4096 -> 4096 (17 MB) in 5.4 - 6.8
// behind a quantisation of 3.7.  An empty launch takes about 4.
#pragma once
#include "frozen_rows.h"

namespace lyc {

constexpr int SK_FUSED_ELEMS = 16384;  // M * K up to which the rows are quantised in the kernel (32 KiB of 16-bit activations a workgroup)
__host__ __device__ inline int sk_pitch(int K) { return ((K + 127) & ~127) + 16; }  // LDS row pitch: rows on different banks

template <typename E, typename TI, typename TO, int MT, int W, bool GATED, bool FUSED>
__global__ __launch_bounds__(W * 64) void fz_skinny_kernel(const TI* __restrict__ x, FzProb p, FzEpi ep) {
  using Acc = typename FE<E>::acc;
  constexpr int H = GATED ? 2 : 1, PRE = 2;
  extern __shared__ __attribute__((aligned(16))) char sk_smem[];
  __shared__ float xs[16 * MT];
  const int lane = threadIdx.x & 63, li = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
  const int NO = GATED ? ep.F : p.N, n0 = blockIdx.x * 16;
  const int vrow = GATED && ep.gate_first ? ep.F : 0, grow = GATED && !ep.gate_first ? ep.F : 0;
  const int pieces = (p.kb + 127) >> 7;
  const char* wr[H];
  bool wok = n0 + li < NO;
  wr[0] = static_cast<const char*>(p.B) + (int64_t)(vrow + (wok ? n0 + li : 0)) * p.ldb;
  if (GATED) wr[H - 1] = static_cast<const char*>(p.B) + (int64_t)(grow + (wok ? n0 + li : 0)) * p.ldb;
  const u32x4 zero = {0u, 0u, 0u, 0u};
  // the two 16-byte chunks of piece c that belong to this lane
  auto load = [&](const char* row, bool ok, int c, u32x4 (&o)[2]) {
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      const int k = c * 128 + 32 * g + 16 * s;
      o[s] = ok && k < p.kb ? *reinterpret_cast<const u32x4*>(row + k) : zero;
    }
  };
  u32x4 pre[PRE][H][2];
#pragma unroll
  for (int i = 0; i < PRE; ++i)
#pragma unroll
    for (int h = 0; h < H; ++h) load(wr[h], wok && wave + i * W < pieces, wave + i * W, pre[i][h]);

  const int pitch = sk_pitch(p.K);
  if constexpr (FUSED) {
    const int vec = fz_al16(x) && (p.K & 7) == 0;
    for (int m = wave; m < p.M; m += W) {
      const TI* row = x + (int64_t)m * p.K;
      unsigned bits = 0;
      float v[8];
      for (int k = lane * 8; k < p.K; k += 512) {
        fz_row8<TI>(row, k, p.K, vec, v);
#pragma unroll
        for (int e = 0; e < 8; ++e) bits = max(bits, __float_as_uint(v[e]) & 0x7fffffffu);
      }
#pragma unroll
      for (int o = 1; o < 64; o <<= 1) bits = max(bits, (unsigned)__shfl_xor((int)bits, o));
      float sc;
      const float amax = fz_amax_of(bits, &sc);
      if (lane == 0) xs[m] = sc;
      for (int k = lane * 8; k < pieces * 128; k += 512) {  // (the second reading hits the L1)
        fz_row8<TI>(row, k, p.K, vec, v);
        *reinterpret_cast<u32x2*>(sk_smem + m * pitch + k) = fz_pack_q<TI>(v, amax);
      }
    }
    __syncthreads();
  }

  Acc acc[H][MT];
#pragma unroll
  for (int h = 0; h < H; ++h)
#pragma unroll
    for (int t = 0; t < MT; ++t) acc[h][t] = Acc{0, 0, 0, 0};
  auto use = [&](int c, const u32x4 (&w)[H][2]) {
#pragma unroll
    for (int t = 0; t < MT; ++t) {
      const int m = 16 * t + li;
      u32x4 a[2];
      if constexpr (FUSED) {
#pragma unroll
        for (int s = 0; s < 2; ++s) a[s] = m < p.M ? *reinterpret_cast<const u32x4*>(sk_smem + m * pitch + c * 128 + 32 * g + 16 * s) : zero;
      } else {
        load(static_cast<const char*>(p.A) + (int64_t)(m < p.M ? m : 0) * p.lda, m < p.M, c, a);
      }
#pragma unroll
      for (int h = 0; h < H; ++h)
#pragma unroll
        for (int s = 0; s < 2; ++s) acc[h][t] = FE<E>::mma(w[h][s], a[s], acc[h][t]);
    }
  };
#pragma unroll
  for (int i = 0; i < PRE; ++i)
    if (wave + i * W < pieces) use(wave + i * W, pre[i]);
  int c = wave + PRE * W;
  for (; c + W < pieces; c += 2 * W) {
    u32x4 w0[H][2], w1[H][2];
#pragma unroll
    for (int h = 0; h < H; ++h) {
      load(wr[h], wok, c, w0[h]);
      load(wr[h], wok, c + W, w1[h]);
    }
    use(c, w0);
    use(c + W, w1);
  }
  if (c < pieces) {
    u32x4 w0[H][2];
#pragma unroll
    for (int h = 0; h < H; ++h) load(wr[h], wok, c, w0[h]);
    use(c, w0);
  }

  // partial sums [h][row tile][wave][16 rows][16 columns + pad]; the quantised rows are no longer read
  using S = typename std::conditional<FE<E>::SIZE == 1, int, float>::type;
  S* red = reinterpret_cast<S*>(sk_smem);
  constexpr int RP = 20;
  if constexpr (FUSED) __syncthreads();
#pragma unroll
  for (int h = 0; h < H; ++h)
#pragma unroll
    for (int t = 0; t < MT; ++t)  // acc: row (weight row) 4 g + e, column (activation row) li
      *reinterpret_cast<Acc*>(red + ((((h * MT + t) * W + wave) * 16) + li) * RP + 4 * g) = acc[h][t];
  __syncthreads();
  for (int i = threadIdx.x; i < 256 * MT; i += W * 64) {
    const int t = i >> 8, r = (i >> 4) & 15, j = i & 15;
    const int m = 16 * t + r, n = n0 + j;
    if (m >= p.M || n >= NO) continue;
    float v[H];
#pragma unroll
    for (int h = 0; h < H; ++h) {
      S s = 0;
#pragma unroll
      for (int w = 0; w < W; ++w) s += red[((((h * MT + t) * W + w) * 16) + r) * RP + j];
      v[h] = (float)s;
    }
    const float sa = FUSED ? xs[m] : ep.sa ? ep.sa[m] : 1.f;
    const int row[2] = {vrow, grow};
#pragma unroll
    for (int h = 0; h < H; ++h) {
      const int64_t at = (GATED ? row[h] : 0) + n;
      v[h] = v[h] * sa * (ep.sw ? ep.sw[at] : 1.f);
      if (ep.bias) v[h] += ep.bias_f32 ? static_cast<const float*>(ep.bias)[at] : (float)static_cast<const TO*>(ep.bias)[at];
      if (ep.base) v[h] += (float)static_cast<const TO*>(ep.base)[(int64_t)m * H * NO + at];
      if (GATED && ep.pre) {
        float one[8] = {v[h]};
        fz_store_pre8<TO>(ep.pre, ep.pre_total, (int64_t)m * 2 * NO + at, NO - 1, NO, one);
      }
    }
    float y = v[0];
    if constexpr (GATED) fz_for_act(ep.act, [&](auto ac) { y *= fz_act<decltype(ac)::value>(v[H - 1]); });
    static_cast<TO*>(ep.out)[(int64_t)m * NO + n] = (TO)y;
  }
}

}  // namespace lyc
