// frozen.hip -- C ABI of the 8-bit frozen layer and the gated projection (include/lycoris_amd.h).  gfx950 only.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <atomic>

#include "../../include/lycoris_amd.h"
#include "errors.h"
#include "frozen_skinny.h"

using namespace lyc;

namespace {

inline int64_t cdiv(int64_t a, int64_t b) { return (a + b - 1) / b; }
inline int64_t up(int64_t a, int64_t b) { return cdiv(a, b) * b; }

#define FZ_DTYPE(dtype_, ...)                                        \
  switch (dtype_) {                                                  \
    case LYC_BF16: { using T = __bf16; __VA_ARGS__; } break;         \
    case LYC_F16: { using T = _Float16; __VA_ARGS__; } break;        \
    case LYC_F32: { using T = float; __VA_ARGS__; } break;           \
    default: return fail(LYC_ERR_ARG, "unknown dtype %d", dtype_);   \
  }

// a workspace handed out piece by piece; with a null base it only counts
struct Carve {
  char* base;
  int64_t used = 0;
  template <typename T>
  T* take(int64_t n) {
    used = up(used, 256);
    T* r = base ? reinterpret_cast<T*>(base + used) : nullptr;
    used += n * (int64_t)sizeof(T);
    return r;
  }
};

int check_dims(const char* who, int64_t M, int64_t N, int64_t K, int dtype) {
  if (dtype != LYC_F32 && dtype != LYC_F16 && dtype != LYC_BF16) return fail(LYC_ERR_ARG, "%s: unknown dtype %d", who, dtype);
  if (M < 0 || N < 1 || K < 1) return fail(LYC_ERR_ARG, "%s: bad dims M=%ld N=%ld K=%ld", who, (long)M, (long)N, (long)K);
  // K: 2^17 products of -128 and -128 would sum to 2^31; M: launches stay below 2^32 threads, and 2 M bytes below 2^31 where rows are summed
  if (M > (1 << 26) || N > (1 << 20) || K >= (1 << 17))
    return fail(LYC_ERR_UNSUPPORTED, "%s: M=%ld N=%ld K=%ld exceed 2^26 rows, 2^20 outputs or 2^17 - 1 inputs", who, (long)M, (long)N, (long)K);
  return LYC_OK;
}
#define FZ_TRY(expr)                  \
  do {                                \
    const int rc_ = (expr);           \
    if (rc_ != LYC_OK) return rc_;    \
  } while (0)

int need16(const char* who, const char* what, const void* p, bool optional = false) {
  if (!p) return optional ? LYC_OK : fail(LYC_ERR_ARG, "%s: null pointer (%s)", who, what);
  return fz_al16(p) ? LYC_OK : fail(LYC_ERR_ARG, "%s: %s must be 16-byte aligned", who, what);
}

// Dynamic LDS above 64 KiB is allowed per kernel AND device: the kernel is a template argument (of one type are all products), so that each
// has its own flags.  Devices beyond the flags are set on every launch.
template <auto Kern>
int allow_lds(int bytes) {
  static std::atomic<uint64_t> done{0};
  int dev = 0;
  if (hipGetDevice(&dev) != hipSuccess) return fail(LYC_ERR_LAUNCH, "hipGetDevice failed");
  const uint64_t bit = dev < 64 ? 1ull << dev : 0;
  if (done.load(std::memory_order_relaxed) & bit) return LYC_OK;
  const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(Kern), hipFuncAttributeMaxDynamicSharedMemorySize, bytes);
  if (e != hipSuccess) return fail(LYC_ERR_LAUNCH, "hipFuncSetAttribute: %s", hipGetErrorString(e));
  done.fetch_or(bit, std::memory_order_relaxed);
  return LYC_OK;
}

int grid_of(int64_t chunks) { return (int)(cdiv(chunks, 256) < 16384 ? cdiv(chunks, 256) : 16384); }

template <typename K, int BM>
int launch_tile(const FzProb& p, const FzEpi& ep, hipStream_t st) {
  const int per = fz_per_xcd(cdiv(p.M, BM) * cdiv(K::GATED ? ep.F : p.N, K::BNO));
  FZ_TRY((allow_lds<&fz_gemm_kernel<K>>(K::LDS)));
  hipLaunchKernelGGL((fz_gemm_kernel<K>), dim3((unsigned)(8 * per), p.ksplit > 1 ? p.ksplit : 1), dim3(K::NW * 64), K::LDS, st, p, ep);
  return check_launch("fz_gemm");
}

// Which tiles, and into how many parts of K, for a product of M x NO outputs and `steps` 64-byte steps of K.
//   256 x 256, 128 x 160 (one workgroup of 8 waves a CU), 128 x 128 (two), 64 x 64 (two of 4 waves; gated: 64 x 128, one); where the tiles are
//   few and K is long, K in parts whose sums a second launch joins.
// The tile of 160 columns is there for outputs of 320, 640 and 1280 channels, which it cuts into as many tiles as CUs (dx 8192 x 640, K = 5120: 64
// us, against 83 with 128 x 128 and 127 with 256 x 256); with whole rounds of the larger tile that wins (dx 16384 x 5120, K = 1280: 190 us,
// against 247 and 283, on bf16 operands; 212 on fp16 ones), and in parts of a long K (dx 4096 x 1280, K = 10240, three parts: 106 + 12 us, against 157 with 128 x 128 and 127 with
// 128 x 160).
// The rule compares estimates in microseconds, from sweeps of 30 shapes with inputs out of HBM: a round costs what a step costs times the
// steps, plus what a tile's beginning and end leave exposed -- of its epilogue's bytes, at a CU's share of HBM, less where a second
// workgroup computes meanwhile.
struct Plan {
  int tile = 128, ksplit = 1;  // tile: 64, 128, 160 (128 x 160), 256
  double us = 1e30;
};
struct Rate {
  double step, tile, shown;
};
struct Tile {
  int id, bm, bn, wgs;
  Rate rate[2];  // with 1, 2 workgroups on the CU
};
constexpr Tile TILES[] = {{128, 128, 128, 2, {{0.30, 3.0, 1.0}, {0.54, 2.5, 0.5}}},
                          {64, 64, 64, 2, {{0.18, 2.5, 1.0}, {0.26, 2.0, 0.5}}},
                          {160, 128, 160, 1, {{0.35, 3.5, 1.0}}},
                          {256, 256, 256, 1, {{0.73, 5.0, 0.7}}}};
constexpr double CU_BYTES_PER_US = 19900.0;
double rounds_cost(int64_t tiles, const Tile& t, double steps, double bytes) {
  const int64_t per = fz_per_xcd(tiles), slots = 32 * t.wgs, full = per / slots, rest = per % slots;
  auto one = [&](int load) { return t.rate[load - 1].step * steps + t.rate[load - 1].tile + t.rate[load - 1].shown * load * bytes / CU_BYTES_PER_US; };
  return (double)full * one(t.wgs) + (rest ? one((int)cdiv(rest, 32)) : 0.0);
}
// eb: bytes the epilogue moves per output
Plan plan_gemm(int64_t M, int64_t NO, double steps, bool gated, double eb) {
  Plan best;
  for (const Tile& t : TILES) {
    if (gated && t.id == 160) continue;
    Tile u = t;
    const int bno = !gated || t.id == 64 ? t.bn : t.bn / 2;
    if (gated) {  // the activation's vector work, and 64 x 64 outputs take 128 rows of w
      if (t.id == 64) u.wgs = 1;
      for (Rate& r : u.rate) {
        r.tile += t.id == 256 ? 4.0 : t.id == 128 ? 1.0 : 2.0;
        if (t.id == 64) r.step *= 1.4;
      }
    }
    const int64_t tiles = cdiv(M, t.bm) * cdiv(NO, bno);
    const double area = (double)t.bm * bno;
    for (int ks = 1; ks == 1 || (!gated && ks <= 8 && steps / ks >= 12); ++ks) {
      double us = rounds_cost(tiles * ks, u, ks == 1 ? steps : cdiv((int64_t)steps, ks), area * (ks == 1 ? eb : 4.0));
      if (ks > 1) us += 4.0 + (double)M * NO * (4.0 * ks + eb) / (256 * CU_BYTES_PER_US);
      if (us < best.us) best = Plan{t.id, ks, us};
    }
  }
  return best;
}
template <typename E, int EPI>
Plan plan_of(int64_t M, int64_t NO, int64_t K, int nseg, double eb) {
  return plan_gemm(M, NO, (double)cdiv(K * FE<E>::SIZE, 64) * nseg, EPI == FZ_GATED, eb);
}
// bytes of a plan's partial sums
int64_t part_bytes(const Plan& pl, int64_t M, int64_t N) { return pl.ksplit > 1 ? pl.ksplit * M * N * 4 : 0; }

template <typename E, typename TO, bool A_KS, bool B_KS, int EPI>
int launch_gemm(const Plan& pl, FzProb p, FzEpi ep, void* part, hipStream_t st) {
  constexpr bool G = EPI == FZ_GATED;
  // ring slots of 128 bytes of K (cold inputs), but 64 where neither operand's rows lie along K: 128 x 128 dw 5120 x 640, K = 8192: 101 us
  // against 123, 256 x 256 dw 10240 x 1280, K = 4096: 104 against 110
  constexpr int SB = A_KS && B_KS ? 64 : 128, D = A_KS && B_KS ? 5 : 2;
  using K256 = FzKernel<E, TO, 256, 256, 2, 4, SB, D, A_KS, B_KS, EPI>;
  using K128 = FzKernel<E, TO, 128, 128, 4, 2, SB, D, A_KS, B_KS, EPI>;
  using K64 = FzKernel<E, TO, 64, G ? 128 : 64, 2, 2, 128, 4, A_KS, B_KS, EPI>;
  p.ksplit = pl.ksplit;
  ep.part = part;
  switch (pl.tile) {
    case 64: FZ_TRY((launch_tile<K64, 64>(p, ep, st))); break;
    case 128: FZ_TRY((launch_tile<K128, 128>(p, ep, st))); break;
    case 160:
      if constexpr (!G) FZ_TRY((launch_tile<FzKernel<E, TO, 128, 160, 4, 2, 128, 4, A_KS, B_KS, EPI>, 128>(p, ep, st)));
      break;
    default: FZ_TRY((launch_tile<K256, 256>(p, ep, st)));
  }
  if constexpr (!G) {
    if (p.ksplit > 1) {
      hipLaunchKernelGGL((fz_reduce_kernel<E, TO>), dim3(grid_of((int64_t)p.M * cdiv(p.N, 8))), dim3(256), 0, st, p, ep);
      return check_launch("fz_reduce");
    }
  }
  return LYC_OK;
}

// up to 32 rows: frozen_skinny.h.  x: the activations when the kernel quantises them itself, else null
template <typename E, typename TI, typename TO, int MT, bool GATED, bool FUSED>
int launch_skinny2(const TI* x, const FzProb& p, const FzEpi& ep, hipStream_t st) {
  const int64_t NO = GATED ? ep.F : p.N;
  auto go = [&](auto wc) {
    constexpr int W = decltype(wc)::value;
    const int red = (GATED ? 2 : 1) * MT * W * 16 * 20 * 4, rows = FUSED ? p.M * sk_pitch(p.K) : 0;
    const int lds = red > rows ? red : rows;
    FZ_TRY((allow_lds<&fz_skinny_kernel<E, TI, TO, MT, W, GATED, FUSED>>(96 * 1024)));
    hipLaunchKernelGGL((fz_skinny_kernel<E, TI, TO, MT, W, GATED, FUSED>), dim3((unsigned)cdiv(NO, 16)), dim3(W * 64), lds, st, x, p, ep);
    return check_launch("fz_skinny");
  };
  // 8 waves share K; 16 where K is long and the columns alone do not fill the CUs twice
  if (p.kb >= 4096 && NO <= 16 * 512) return go(std::integral_constant<int, 16>{});
  return go(std::integral_constant<int, 8>{});
}
template <typename E, typename TI, typename TO, bool GATED, bool FUSED>
int launch_skinny(const TI* x, const FzProb& p, const FzEpi& ep, hipStream_t st) {
  if (p.M <= 16) return launch_skinny2<E, TI, TO, 1, GATED, FUSED>(x, p, ep, st);
  return launch_skinny2<E, TI, TO, 2, GATED, FUSED>(x, p, ep, st);
}
constexpr int64_t SKINNY_ROWS = 32;
inline bool skinny_fused(int64_t M, int64_t K) { return M <= SKINNY_ROWS && M * K <= SK_FUSED_ELEMS; }

// How a row of c chunks of 8 is spread over threads: go(threads a row, chunks a thread) while registers hold it -- a wave a row, rows of 2048 columns
// and more over a workgroup -- else whole()
template <typename Go, typename Whole>
void row_shape(int64_t c, Go go, Whole whole) {
  using std::integral_constant;
  if (c <= 64) go(integral_constant<int, 64>{}, integral_constant<int, 1>{});
  else if (c <= 128) go(integral_constant<int, 64>{}, integral_constant<int, 2>{});
  else if (c <= 192) go(integral_constant<int, 64>{}, integral_constant<int, 3>{});
  else if (c <= 256) go(integral_constant<int, 64>{}, integral_constant<int, 4>{});
  else if (c <= 512) go(integral_constant<int, 256>{}, integral_constant<int, 2>{});
  else if (c <= 768) go(integral_constant<int, 256>{}, integral_constant<int, 3>{});
  else if (c <= 1024) go(integral_constant<int, 256>{}, integral_constant<int, 4>{});
  else whole();
}
constexpr int64_t ROW_SLAB = 1 << 22;  // rows a launch: a workgroup a row stays below 2^32 threads

template <typename T>
int launch_quant(const T* x, int64_t ldx, int8_t* q, int64_t ldq, float* scale, int64_t M, int K, hipStream_t st) {
  if (M > ROW_SLAB) {
    FZ_TRY(launch_quant<T>(x, ldx, q, ldq, scale, ROW_SLAB, K, st));
    return launch_quant<T>(x + ROW_SLAB * ldx, ldx, q + ROW_SLAB * ldq, ldq, scale + ROW_SLAB, M - ROW_SLAB, K, st);
  }
  const int vec = fz_al16(x) && (ldx * (int64_t)sizeof(T)) % 16 == 0 && K % 8 == 0;
  row_shape(ldq / 8, [&](auto tpr, auto nv) {
    constexpr int TPR = decltype(tpr)::value, NV = decltype(nv)::value;
    hipLaunchKernelGGL((fz_quant_kernel<T, TPR, NV>), dim3((unsigned)cdiv(M, 256 / TPR)), dim3(256), 0, st, x, ldx, q, ldq, scale, M, K, vec);
  }, [&] { hipLaunchKernelGGL((fz_quant_long_kernel<T>), dim3((unsigned)M), dim3(256), 0, st, x, ldx, q, ldq, scale, M, K, vec); });
  return check_launch("int8_quantize");
}

FzPlane plane_job(const int8_t* q, int64_t ldq, void* out, int64_t O, int64_t I) { return FzPlane{q, out, ldq, (int)O, (int)I, (int)cdiv(O, FZ_PLANE_ROWS)}; }
template <typename T>
int launch_plane(const FzPlane& w, hipStream_t st) {
  hipLaunchKernelGGL((fz_plane_kernel<T>), dim3((unsigned)w.groups), dim3(256), 0, st, w);
  return check_launch("weight plane");
}

// g [M, N] times col into NP fp16 planes, `plane` elements apart, rows of up(N, 8); and the weight's plane
template <typename T, int NP>
int launch_scale(const T* g, const float* col, _Float16* out, int64_t plane, float* scale, int64_t M, int64_t N, FzPlane w, hipStream_t st) {
  if (M > ROW_SLAB) {
    FZ_TRY((launch_scale<T, NP>(g, col, out, plane, scale, ROW_SLAB, N, w, st)));
    w.groups = 0;
    return launch_scale<T, NP>(g + ROW_SLAB * N, col, out + ROW_SLAB * up(N, 8), plane, scale + ROW_SLAB, M - ROW_SLAB, N, w, st);
  }
  const int vec = fz_al16(g) && N % 8 == 0, vcol = fz_al16(col) && N % 8 == 0;
  row_shape(cdiv(N, 8), [&](auto tpr, auto nv) {
    constexpr int TPR = decltype(tpr)::value, NV = decltype(nv)::value;
    hipLaunchKernelGGL((fz_scale_kernel<T, NP, TPR, NV>), dim3((unsigned)(w.groups + cdiv(M, 256 / TPR))), dim3(256), 0, st, g, col, out, plane, scale, M, (int)N, vec,
                       vcol, w);
  }, [&] { hipLaunchKernelGGL((fz_scale_long_kernel<T, NP>), dim3((unsigned)(w.groups + M)), dim3(256), 0, st, g, col, out, plane, scale, M, (int)N, vec, vcol, w); });
  return check_launch("scaled rows");
}

// The operands of a pass that have to be staged, and their one launch
template <typename T>
struct Stages {
  using E = typename std::conditional<sizeof(T) == 4, __bf16, T>::type;
  FzStage list;
  int n = 0;
  int64_t most = 0;
  void add(const T* x, const float* col, void* out, int64_t rows, int64_t cols) {
    list.job[n++] = FzStageJob{x, col, out, rows, (int)cols, fz_al16(x) && cols % 8 == 0};
    most = std::max(most, rows * cdiv(cols, 8));
  }
  int run(hipStream_t st) {
    if (!n) return LYC_OK;
    hipLaunchKernelGGL((fz_stage_kernel<T, E, sizeof(T) == 4 ? 3 : 1>), dim3(grid_of(most), n), dim3(256), 0, st, list);
    return check_launch("stage");
  }
};
// One operand of a product in the type the matrix cores take: the tensor itself, its staged copy, or its three bf16 planes.
template <typename T>
struct Operand {
  using E = typename Stages<T>::E;
  const void* p = nullptr;
  int64_t ld = 0, plane = 0;  // bytes
  void* room = nullptr;
  int64_t rows, cols;
  bool own;
  Operand(Carve& ws, int64_t rows_, int64_t cols_, bool wanted) : rows(rows_), cols(cols_), own(sizeof(T) == 4 || cols_ % 8 != 0) {
    if (wanted && own) room = ws.take<E>((sizeof(T) == 4 ? 3 : 1) * rows * up(cols, 8));
  }
  // x [rows, cols], contiguous; to be read after `stages` has run
  void fill(const T* x, const float* col, Stages<T>& stages) {
    p = own ? room : x;
    ld = own ? up(cols, 8) * 2 : cols * (int64_t)sizeof(T);
    plane = own ? rows * ld : 0;
    if (own) stages.add(x, col, room, rows, cols);
  }
};
// segments: of one plane each 1; of 2 or 3 planes of A 2 or 3; fp32 x fp32 6.  The small terms come first.
void segments(FzProb& p, int n) {
  p.nseg = n;
  p.pa = n == 6 ? 0x010120u : n == 3 ? 0x012u : n == 2 ? 0x01u : 0u;
  p.pb = n == 6 ? 0x001102u : 0u;
}

FzProb prob(const void* A, int64_t lda, int64_t a_plane, const void* B, int64_t ldb, int64_t b_plane, int64_t M, int64_t N, int64_t K, int es) {
  FzProb p{};
  p.A = A; p.B = B; p.lda = lda; p.ldb = ldb; p.a_plane = a_plane; p.b_plane = b_plane;
  p.M = (int)M; p.N = (int)N; p.K = (int)K;
  p.kb = (int)up(K * es, 16);
  p.nseg = 1;
  return p;
}

// (the estimate takes a base operand for granted: the workspace is sized before it is known)
Plan plan8(int64_t M, int64_t N, int64_t K, int dtype) { return plan_of<int8_t, FZ_LINEAR>(M, N, K, 1, dtype == LYC_F32 ? 8.0 : 4.0); }
int64_t part8(int64_t M, int64_t N, int64_t K, int dtype) { return M <= SKINNY_ROWS ? 0 : part_bytes(plan8(M, N, K, dtype), M, N); }
int matmul8(const int8_t* aq, int64_t lda, const float* sa, const int8_t* bq, int64_t ldb, const float* sb, const void* bias, int bias_f32, const void* base,
            void* y, void* part, int64_t M, int64_t N, int64_t K, int dtype, hipStream_t st) {
  FzProb p = prob(aq, lda, 0, bq, ldb, 0, M, N, K, 1);
  FzEpi ep{};
  ep.out = y; ep.sa = sa; ep.sw = sb; ep.bias = bias; ep.bias_f32 = bias_f32; ep.base = base;
  if (M <= SKINNY_ROWS) {
    FZ_DTYPE(dtype, return (launch_skinny<int8_t, T, T, false, false>(nullptr, p, ep, st)));
  }
  FZ_DTYPE(dtype, return (launch_gemm<int8_t, T, false, false, FZ_LINEAR>(plan8(M, N, K, dtype), p, ep, part, st)));
  return LYC_OK;
}

int check_q(const char* who, const char* what, const void* q, int64_t ld, int64_t K) {
  FZ_TRY(need16(who, what, q));
  if (ld < K || ld % 16 || ld > (1 << 22)) return fail(LYC_ERR_ARG, "%s: the row pitch of %s must be a multiple of 16, at least K and at most 2^22 (%ld)", who, what, (long)ld);
  return LYC_OK;
}

// the operand type of the backward pass's products, and the planes of the gradient's operand
template <typename T>
using GradE = typename std::conditional<sizeof(T) == 4, __bf16, _Float16>::type;
template <typename T>
constexpr int grad_planes() { return sizeof(T) == 4 ? 3 : std::is_same<T, _Float16>::value ? 2 : 1; }
template <typename T>
Plan plan_dx8(int64_t M, int64_t K, int64_t N) { return plan_of<GradE<T>, FZ_PLAIN>(M, K, N, grad_planes<T>(), sizeof(T)); }

// ---- dx of a frozen 8-bit layer: (g sw) [M, N] times the integers wq [N, K], which 16 bits hold exactly.  g sw takes a power of two a row in fp16
//      (fz_scale_kernel; fp16 gradients: two planes), for fp32 gradients three bf16 planes ---------------------------------------------
template <typename T>
int dx8(const T* g, const int8_t* wq, int64_t ldw, const float* sw, T* dx, Carve ws, int64_t* bytes, int64_t M, int64_t N, int64_t K, hipStream_t st) {
  constexpr bool F32 = sizeof(T) == 4;
  constexpr int NP = grad_planes<T>();
  using E = GradE<T>;
  const int64_t ld = up(N, 8);
  E* plane = ws.take<E>(N * up(K, 8));
  E* rows = ws.take<E>(NP * M * ld);
  float* scale = F32 ? nullptr : ws.take<float>(M);
  const Plan pl = plan_dx8<T>(M, K, N);
  char* part = ws.take<char>(part_bytes(pl, M, K));
  if (bytes) {
    *bytes = ws.used;
    return LYC_OK;
  }
  const FzPlane w = plane_job(wq, ldw, plane, N, K);
  if constexpr (F32) {
    FZ_TRY(launch_plane<E>(w, st));
    Stages<T> stages;
    stages.add(g, sw, rows, M, N);
    FZ_TRY(stages.run(st));
  } else {
    FZ_TRY((launch_scale<T, NP>(g, sw, rows, M * ld, scale, M, N, w, st)));
  }
  FzProb p = prob(rows, ld * 2, M * ld * 2, plane, up(K, 8) * 2, 0, M, K, N, 2);
  segments(p, NP);
  FzEpi ep{};
  ep.out = dx;
  ep.sa = scale;
  return launch_gemm<E, T, false, true, FZ_PLAIN>(pl, p, ep, part, st);
}

// ---- gated projection ---------------------------------------------------------------------------------------------------------------------
struct Gated {
  const void* w;
  int64_t ldw;
  const float* sw;
  int64_t M, I, F;
  int act, gate_first;
};

// eb: what the epilogue moves per output
template <typename T>
Plan plan_gated_fwd(int64_t M, int64_t I, int64_t F, bool held, bool base, bool keep) {
  const double eb = (double)sizeof(T) * (base ? 3 : 1) + (keep ? sizeof(T) == 4 ? 8.0 : 6.0 : 0.0);
  return held ? plan_of<int8_t, FZ_GATED>(M, F, I, 1, eb) : plan_of<typename Operand<T>::E, FZ_GATED>(M, F, I, sizeof(T) == 4 ? 6 : 1, eb);
}
template <typename T>
int gated_segments(bool held) { return sizeof(T) == 4 && !held ? 6 : grad_planes<T>(); }
template <typename T>
Plan plan_gated_dx(int64_t M, int64_t I, int64_t F, bool held) { return plan_of<GradE<T>, FZ_PLAIN>(M, I, 2 * F, gated_segments<T>(held), sizeof(T)); }
template <typename T>
Plan plan_gated_dw(int64_t M, int64_t I, int64_t F) { return plan_of<GradE<T>, FZ_PLAIN>(2 * F, I, M, gated_segments<T>(false), sizeof(T)); }

template <typename T>
int gated_fwd(const Gated& q, const T* x, const void* bias, int bias_f32, const T* base, T* h, void* pre, Carve ws, int64_t* bytes, hipStream_t st) {
  using E = typename Operand<T>::E;
  FzEpi ep{};
  ep.out = h; ep.pre = pre; ep.bias = bias; ep.bias_f32 = bias_f32; ep.base = base; ep.sw = q.sw; ep.act = q.act; ep.gate_first = q.gate_first; ep.F = (int)q.F;
  ep.pre_total = 2 * q.M * q.F;
  const Plan pl = plan_gated_fwd<T>(q.M, q.I, q.F, q.sw != nullptr, base != nullptr, pre != nullptr);
  if (q.sw) {
    const int64_t ldq = up(q.I, 16);
    const bool fused = skinny_fused(q.M, q.I);
    int8_t* xq = fused ? nullptr : ws.take<int8_t>(q.M * ldq);
    float* sa = fused ? nullptr : ws.take<float>(q.M);
    if (bytes) {
      *bytes = ws.used;
      return LYC_OK;
    }
    if (fused) {
      FzProb p = prob(nullptr, 0, 0, q.w, q.ldw, 0, q.M, 2 * q.F, q.I, 1);
      return launch_skinny<int8_t, T, T, true, true>(x, p, ep, st);
    }
    FZ_TRY(launch_quant<T>(x, q.I, xq, ldq, sa, q.M, (int)q.I, st));
    ep.sa = sa;
    FzProb p = prob(xq, ldq, 0, q.w, q.ldw, 0, q.M, 2 * q.F, q.I, 1);
    if (q.M <= SKINNY_ROWS) return launch_skinny<int8_t, T, T, true, false>(nullptr, p, ep, st);
    return launch_gemm<int8_t, T, false, false, FZ_GATED>(pl, p, ep, nullptr, st);
  }
  Operand<T> a(ws, q.M, q.I, true), b(ws, 2 * q.F, q.I, true);
  if (bytes) {
    *bytes = ws.used;
    return LYC_OK;
  }
  Stages<T> stages;
  a.fill(x, nullptr, stages);
  b.fill(static_cast<const T*>(q.w), nullptr, stages);
  FZ_TRY(stages.run(st));
  FzProb p = prob(a.p, a.ld, a.plane, b.p, b.ld, b.plane, q.M, 2 * q.F, q.I, 2);
  segments(p, sizeof(T) == 4 ? 6 : 1);
  if constexpr (sizeof(T) == 2) {
    if (q.M <= SKINNY_ROWS) return launch_skinny<E, T, T, true, false>(nullptr, p, ep, st);
  }
  return launch_gemm<E, T, false, false, FZ_GATED>(pl, p, ep, nullptr, st);
}

// rows a workgroup of the elementwise pass takes: as many as leave 1024 workgroups (four a CU), 64 at most (fewer partial column sums)
int dgate_rows(int64_t M, int64_t F) {
  int rows = 64;
  while (rows > 8 && cdiv(F, DG_COLS) * cdiv(M, rows) < 1024) rows /= 2;
  return rows;
}

// The elementwise pass where products follow, 16 bits: rows of a slab.  512 slabs (of waves: 2048) are two workgroups a CU, whose rows follow each other
// with the next one's loads in flight: 8192 x 2560 in 69 us, against 82 in the same run with 1024 slabs (and twice the partial column sums); 4096 x 5120 in 75, against 78.
int dgate_slab_rows(int64_t M, int64_t F) { return (int)cdiv(M, (F <= 512 ? 4 : 1) * 512); }
template <typename T, int NP, bool SUMS>
int launch_dgate_rows(const FzDgate& a, int64_t slabs, hipStream_t st) {
  const int64_t chunks = cdiv(a.F, 8);
  const dim3 grid((unsigned)slabs), block((unsigned)std::min<int64_t>(1024, up(chunks, 64)));
  if (chunks <= 64) hipLaunchKernelGGL((fz_dgate_rows_kernel<T, NP, 1, true, SUMS>), dim3((unsigned)cdiv(slabs, 4)), dim3(256), 0, st, a);
  else if (chunks <= 1024) hipLaunchKernelGGL((fz_dgate_rows_kernel<T, NP, 1, false, SUMS>), grid, block, 0, st, a);
  else hipLaunchKernelGGL((fz_dgate_rows_kernel<T, NP, 0, false, SUMS>), grid, block, 0, st, a);
  return check_launch("gated backward");
}

// dp is formed once, by one elementwise pass.  The products' operands:
//   16 bits   dp (over an 8-bit weight sw dp) in fp16 with a power of two a row (fp16 gradients: two planes); the weight's integers, which fp16 holds
//             exactly, or the 16-bit weight and x in fp16 with one power of two each (fz_level_kernel)
//   32 bits   three bf16 planes each of dp (sw dp), the weight and x
template <typename T>
int gated_bwd(const Gated& q, const T* g, const void* pre, const T* x, T* dp, T* dx, T* dw, void* dbias, bool dbias_f32, int flags, Carve ws, int64_t* bytes, hipStream_t st) {
  constexpr bool F32 = sizeof(T) == 4;
  constexpr int NP = grad_planes<T>(), NB = F32 ? 3 : 1;  // planes of dp, of the weight and of x
  using E = GradE<T>;
  const bool held = flags & LYC_GATED_INT8, want_dx = flags & LYC_GATED_DX, want_dw = flags & LYC_GATED_DW, want_db = flags & LYC_GATED_DBIAS;
  const bool products = want_dx || want_dw, by_row = products && !F32, level = by_row && !held;
  const int rows = by_row ? dgate_slab_rows(q.M, q.F) : dgate_rows(q.M, q.F);
  const int64_t N = 2 * q.F, ld = up(N, 8), ldi = up(q.I, 8), parts = cdiv(q.M, rows);
  if (!(flags & LYC_GATED_DBASE)) dp = products && F32 ? ws.take<T>(q.M * N) : nullptr;
  E* a = products ? ws.take<E>(NP * q.M * ld) : nullptr;
  float* scale = by_row ? ws.take<float>(q.M) : nullptr;
  float* top = level && want_dw ? ws.take<float>(parts) : nullptr;
  E* b = want_dx ? ws.take<E>((held ? 1 : NB) * N * ldi) : nullptr;
  E* xo = want_dw ? ws.take<E>(NB * q.M * ldi) : nullptr;
  unsigned* peaks = level ? ws.take<unsigned>(2 * FZ_PEAKS) : nullptr;
  float* alpha = level ? ws.take<float>(2) : nullptr;
  float* part = want_db ? ws.take<float>(parts * N) : nullptr;
  const Plan pdx = plan_gated_dx<T>(q.M, q.I, q.F, held), pdw = plan_gated_dw<T>(q.M, q.I, q.F);
  char* sums = ws.take<char>(std::max(want_dx ? part_bytes(pdx, q.M, q.I) : 0, want_dw ? part_bytes(pdw, N, q.I) : 0));
  if (bytes) {
    *bytes = ws.used;
    return LYC_OK;
  }
  const int vec = q.F % 8 == 0 && fz_al16(g) && fz_al16(pre) && fz_al16(dp) && (!held || fz_al16(q.sw));
  FzProb p;
  FzEpi ep{};
  if constexpr (F32) {
    hipLaunchKernelGGL((fz_dgate_kernel<T>), dim3((unsigned)(cdiv(q.F, DG_COLS) * parts)), dim3(256), 0, st, g, pre, dp, part, q.M, (int)q.F, q.act,
                       q.gate_first, vec, rows);
    FZ_TRY(check_launch("gated backward"));
    Stages<T> stages;
    if (products) stages.add(dp, held ? q.sw : nullptr, a, q.M, N);
    if (want_dx && !held) stages.add(static_cast<const T*>(q.w), nullptr, b, N, q.I);
    if (want_dw) stages.add(x, nullptr, xo, q.M, q.I);
    FZ_TRY(stages.run(st));
  } else if (!products) {
    hipLaunchKernelGGL((fz_dgate_kernel<T>), dim3((unsigned)(cdiv(q.F, DG_COLS) * parts)), dim3(256), 0, st, g, pre, dp, part, q.M, (int)q.F, q.act,
                       q.gate_first, vec, rows);
    FZ_TRY(check_launch("gated backward"));
  } else {
    FzLevel jobs;
    int n = 0;
    int64_t most = 0;
    auto add = [&](const void* v, E* out, const float* row, int64_t r) {
      jobs.job[n] = FzLevelJob{v, out, row, row ? top : nullptr, peaks + n * FZ_PEAKS, alpha + n, r, (int)q.I, fz_al16(v) && q.I % 8 == 0, row ? (int)parts : 0};
      most = std::max(most, r * cdiv(q.I, 8));
      ++n;
    };
    if (level && want_dx) add(q.w, b, nullptr, N);
    if (level && want_dw) add(x, xo, scale, q.M);
    const int spread = (int)std::min<int64_t>(FZ_PEAKS, cdiv(most, 256));
    if (level) {
      hipLaunchKernelGGL((fz_peak_kernel<T>), dim3(spread, n), dim3(256), 0, st, jobs);
      FZ_TRY(check_launch("operand range"));
    }
    const FzDgate d{g, pre, dp, a, held ? q.sw : nullptr, scale, top, part, q.M, q.M * ld, (int)q.F, q.act, q.gate_first, vec, rows};
    FZ_TRY((part ? launch_dgate_rows<T, NP, true>(d, parts, st) : launch_dgate_rows<T, NP, false>(d, parts, st)));
    if (level) {
      hipLaunchKernelGGL((fz_level_kernel<T>), dim3((unsigned)std::min<int64_t>(2048, cdiv(most, 256)), n), dim3(256), 0, st, jobs, spread);
      FZ_TRY(check_launch("operands"));
    }
  }
  if (want_dx) {
    if (held) FZ_TRY(launch_plane<E>(plane_job(static_cast<const int8_t*>(q.w), q.ldw, b, N, q.I), st));
    p = prob(a, ld * 2, q.M * ld * 2, b, ldi * 2, N * ldi * 2, q.M, q.I, N, 2);
    segments(p, gated_segments<T>(held));
    ep.out = dx;
    ep.sa = scale;
    ep.alpha = alpha;
    FZ_TRY((launch_gemm<E, T, false, true, FZ_PLAIN>(pdx, p, ep, sums, st)));
  }
  if (want_dw) {
    p = prob(a, ld * 2, q.M * ld * 2, xo, ldi * 2, q.M * ldi * 2, N, q.I, q.M, 2);
    segments(p, gated_segments<T>(false));
    ep.out = dw;
    ep.sa = nullptr;
    ep.alpha = alpha ? alpha + want_dx : nullptr;
    FZ_TRY((launch_gemm<E, T, true, true, FZ_PLAIN>(pdw, p, ep, sums, st)));
  }
  if (part) {
    const dim3 grid((unsigned)cdiv(N, 32));
    if (dbias_f32) hipLaunchKernelGGL((fz_join_kernel<float>), grid, dim3(256), 0, st, part, static_cast<float*>(dbias), parts, (int)N);
    else hipLaunchKernelGGL((fz_join_kernel<T>), grid, dim3(256), 0, st, part, static_cast<T*>(dbias), parts, (int)N);
    FZ_TRY(check_launch("column sums"));
  }
  return LYC_OK;
}

int check_gated(const char* who, const Gated& q, bool held, int dtype) {
  if (q.F > (1 << 19)) return fail(LYC_ERR_UNSUPPORTED, "%s: F=%ld exceeds 2^19", who, (long)q.F);
  FZ_TRY(check_dims(who, q.M, q.F < 1 ? 0 : 2 * q.F, q.I, dtype));
  if (q.act < 0 || q.act > 2) return fail(LYC_ERR_ARG, "%s: unknown activation %d", who, q.act);
  if ((q.F + 512) * (held ? q.ldw : up(q.I, 8) * 2) >= ((int64_t)1 << 30)) return fail(LYC_ERR_UNSUPPORTED, "%s: half a weight of 1 GiB or more", who);
  return LYC_OK;
}

}  // namespace

extern "C" {

int lyc_int8_quantize(const void* x, int64_t ldx, int8_t* q, int64_t ldq, float* scale, int64_t M, int64_t K, int dtype, void* stream) {
  FZ_TRY(check_dims("int8_quantize", M, 1, K, dtype));
  if (M == 0) return LYC_OK;
  if (!x || !scale) return fail(LYC_ERR_ARG, "int8_quantize: null pointer");
  if (ldx < K) return fail(LYC_ERR_ARG, "int8_quantize: the row pitch of x is %ld, below K=%ld", (long)ldx, (long)K);
  FZ_TRY(check_q("int8_quantize", "q", q, ldq, K));
  FZ_DTYPE(dtype, return launch_quant<T>(static_cast<const T*>(x), ldx, q, ldq, scale, M, (int)K, static_cast<hipStream_t>(stream)));
  return LYC_OK;
}

int64_t lyc_int8_matmul_workspace_bytes(int64_t M, int64_t N, int64_t K, int dtype) {
  return check_dims("int8_matmul", M, N, K, dtype) == LYC_OK ? part8(M, N, K, dtype) : -1;
}

int lyc_int8_matmul(const int8_t* aq, int64_t lda, const float* sa, const int8_t* bq, int64_t ldb, const float* sb, const void* bias, int bias_f32,
                    const void* base, void* y, void* ws, int64_t M, int64_t N, int64_t K, int dtype, void* stream) {
  FZ_TRY(check_dims("int8_matmul", M, N, K, dtype));
  if (M == 0) return LYC_OK;
  if (!sa || !sb || !y) return fail(LYC_ERR_ARG, "int8_matmul: null pointer");
  FZ_TRY(check_q("int8_matmul", "a", aq, lda, K));
  FZ_TRY(check_q("int8_matmul", "b", bq, ldb, K));
  FZ_TRY(need16("int8_matmul", "workspace", ws, lyc_int8_matmul_workspace_bytes(M, N, K, dtype) == 0));
  return matmul8(aq, lda, sa, bq, ldb, sb, bias, bias_f32, base, y, ws, M, N, K, dtype, static_cast<hipStream_t>(stream));
}

int64_t lyc_int8_linear_workspace_bytes(int64_t M, int64_t N, int64_t K, int dtype, int backward) {
  if (check_dims("int8_linear", M, N, K, dtype) != LYC_OK) return -1;
  Carve ws{nullptr};
  if (!backward) {
    if (skinny_fused(M, K)) return 0;
    ws.take<int8_t>(M * up(K, 16));
    ws.take<float>(M);
    ws.take<char>(part8(M, N, K, dtype));
    return ws.used;
  }
  int64_t n = 0;
  FZ_DTYPE(dtype, (void)dx8<T>(nullptr, nullptr, 0, nullptr, nullptr, ws, &n, M, N, K, nullptr));
  return n;
}

int lyc_int8_linear_fwd(const void* x, const int8_t* wq, int64_t ldw, const float* sw, const void* bias, int bias_f32, const void* base, void* y, void* ws,
                        int64_t M, int64_t N, int64_t K, int dtype, void* stream) {
  const char* who = "int8_linear_fwd";
  FZ_TRY(check_dims(who, M, N, K, dtype));
  if (M == 0) return LYC_OK;
  if (!x || !sw || !y) return fail(LYC_ERR_ARG, "%s: null pointer", who);
  FZ_TRY(need16(who, "workspace", ws, skinny_fused(M, K)));
  FZ_TRY(check_q(who, "wq", wq, ldw, K));
  Carve c{static_cast<char*>(ws)};
  const int64_t ldq = up(K, 16);
  int8_t* xq = c.take<int8_t>(M * ldq);
  float* sa = c.take<float>(M);
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (skinny_fused(M, K)) {
    FzProb p = prob(nullptr, 0, 0, wq, ldw, 0, M, N, K, 1);
    FzEpi ep{};
    ep.out = y; ep.sw = sw; ep.bias = bias; ep.bias_f32 = bias_f32; ep.base = base;
    FZ_DTYPE(dtype, return (launch_skinny<int8_t, T, T, false, true>(static_cast<const T*>(x), p, ep, st)));
  }
  FZ_DTYPE(dtype, FZ_TRY(launch_quant<T>(static_cast<const T*>(x), K, xq, ldq, sa, M, (int)K, st)));
  return matmul8(xq, ldq, sa, wq, ldw, sw, bias, bias_f32, base, y, c.take<char>(part8(M, N, K, dtype)), M, N, K, dtype, st);
}

int lyc_int8_linear_bwd(const void* g, const int8_t* wq, int64_t ldw, const float* sw, void* dx, void* ws, int64_t M, int64_t N, int64_t K, int dtype,
                        void* stream) {
  const char* who = "int8_linear_bwd";
  FZ_TRY(check_dims(who, M, N, K, dtype));
  if (M == 0) return LYC_OK;
  if (!sw || !dx) return fail(LYC_ERR_ARG, "%s: null pointer", who);
  FZ_TRY(need16(who, "g", g));
  FZ_TRY(need16(who, "workspace", ws));
  FZ_TRY(check_q(who, "wq", wq, ldw, K));
  FZ_DTYPE(dtype, return dx8<T>(static_cast<const T*>(g), wq, ldw, sw, static_cast<T*>(dx), Carve{static_cast<char*>(ws)}, nullptr, M, N, K,
                                static_cast<hipStream_t>(stream)));
  return LYC_OK;
}

int64_t lyc_gated_linear_workspace_bytes(int64_t M, int64_t I, int64_t F, int dtype, int flags) {
  Gated q{nullptr, 16, nullptr, M, I, F, 0, 0};
  if (check_gated("gated_linear", q, true, dtype) != LYC_OK) return -1;
  int64_t n = 0;
  const float one = 1.f;
  Carve ws{nullptr};
  if (flags & LYC_GATED_BACKWARD) {
    FZ_DTYPE(dtype, (void)gated_bwd<T>(q, nullptr, nullptr, nullptr, nullptr, nullptr, nullptr, nullptr, false, flags, ws, &n, nullptr));
  } else {
    q.sw = flags & LYC_GATED_INT8 ? &one : nullptr;
    FZ_DTYPE(dtype, (void)gated_fwd<T>(q, nullptr, nullptr, 0, nullptr, nullptr, nullptr, ws, &n, nullptr));
  }
  return n;
}

int lyc_frozen_plan(int product, int64_t M, int64_t K, int64_t N, int dtype, int flags) {
  const bool gated = product >= LYC_PRODUCT_GATED_FWD, held = flags & LYC_GATED_INT8;
  const Gated q{nullptr, 16, nullptr, M, K, N, 0, 0};
  if (product < 0 || product > LYC_PRODUCT_GATED_DW || (gated ? check_gated("frozen_plan", q, true, dtype) : check_dims("frozen_plan", M, N, K, dtype)) != LYC_OK) return -1;
  const bool few = M <= SKINNY_ROWS && (product == LYC_PRODUCT_INT8_FWD || (product == LYC_PRODUCT_GATED_FWD && (held || dtype != LYC_F32)));
  Plan pl;
  FZ_DTYPE(dtype, switch (product) {
    case LYC_PRODUCT_INT8_FWD: pl = plan8(M, N, K, dtype); break;
    case LYC_PRODUCT_INT8_DX: pl = plan_dx8<T>(M, K, N); break;
    case LYC_PRODUCT_GATED_FWD: pl = plan_gated_fwd<T>(M, K, N, held, flags & LYC_GATED_DBASE, flags & LYC_GATED_BACKWARD); break;
    case LYC_PRODUCT_GATED_DX: pl = plan_gated_dx<T>(M, K, N, held); break;
    default: pl = plan_gated_dw<T>(M, K, N);
  });
  return few ? 32 + (1 << 16) : pl.tile + (pl.ksplit << 16);
}

int lyc_gated_linear_fwd(const void* x, const void* w, int64_t ldw, const float* sw, const void* bias, int bias_f32, const void* base, void* h, void* pre,
                         void* ws, int64_t M, int64_t I, int64_t F, int act, int gate_first, int dtype, void* stream) {
  const char* who = "gated_linear_fwd";
  const Gated q{w, ldw, sw, M, I, F, act, gate_first};
  FZ_TRY(check_gated(who, q, sw != nullptr, dtype));
  if (M == 0) return LYC_OK;
  if (!h) return fail(LYC_ERR_ARG, "%s: null pointer", who);
  FZ_TRY(need16(who, "x", x));
  FZ_TRY(need16(who, "workspace", ws, lyc_gated_linear_workspace_bytes(M, I, F, dtype, sw ? LYC_GATED_INT8 : 0) == 0));
  if (sw) FZ_TRY(check_q(who, "w", w, ldw, I));
  else FZ_TRY(need16(who, "w", w));
  FZ_DTYPE(dtype, return gated_fwd<T>(q, static_cast<const T*>(x), bias, bias_f32, static_cast<const T*>(base), static_cast<T*>(h), pre,
                                      Carve{static_cast<char*>(ws)}, nullptr, static_cast<hipStream_t>(stream)));
  return LYC_OK;
}

int lyc_gated_linear_bwd(const void* g, const void* pre, const void* x, const void* w, int64_t ldw, const float* sw, void* dbase, void* dx, void* dw,
                         void* dbias, void* ws, int64_t M, int64_t I, int64_t F, int act, int gate_first, int dtype, void* stream) {
  const char* who = "gated_linear_bwd";
  const bool dbias_f32 = dtype & LYC_F32_DBIAS;
  dtype &= ~LYC_F32_DBIAS;
  const Gated q{w, ldw, sw, M, I, F, act, gate_first};
  FZ_TRY(check_gated(who, q, sw != nullptr, dtype));
  if (dw && sw) return fail(LYC_ERR_UNSUPPORTED, "%s: an 8-bit weight is frozen", who);
  if (M == 0) return LYC_OK;
  if (!g || !pre) return fail(LYC_ERR_ARG, "%s: null pointer", who);
  if (dx && sw) FZ_TRY(check_q(who, "w", w, ldw, I));
  else if (dx) FZ_TRY(need16(who, "w", w));
  if (dw) FZ_TRY(need16(who, "x", x));
  FZ_TRY(need16(who, "dbase", dbase, true));
  const int flags = LYC_GATED_BACKWARD | (sw ? LYC_GATED_INT8 : 0) | (dbase ? LYC_GATED_DBASE : 0) | (dx ? LYC_GATED_DX : 0) | (dw ? LYC_GATED_DW : 0) |
                    (dbias ? LYC_GATED_DBIAS : 0);
  FZ_TRY(need16(who, "workspace", ws, lyc_gated_linear_workspace_bytes(M, I, F, dtype, flags) == 0));
  FZ_DTYPE(dtype, return gated_bwd<T>(q, static_cast<const T*>(g), pre, static_cast<const T*>(x), static_cast<T*>(dbase),
                                      static_cast<T*>(dx), static_cast<T*>(dw), dbias, dbias_f32, flags, Carve{static_cast<char*>(ws)}, nullptr,
                                      static_cast<hipStream_t>(stream)));
  return LYC_OK;
}

}  // extern "C"
