// Products with bias, activation and residual: y = residual + act(x . w + bias), for any number of rows, K a multiple of 8, any N, rows of
// any pitch.  Sums are fp32 on the MFMA units, the epilogue is fp32, and a result is rounded once.
#include <climits>
#include <cstring>

#include "activations.h"
#include "gemm_device.h"
#include "spans.h"

#pragma clang fp contract(off)

namespace frhip {

struct LinearArgs {
  const h1* x;
  const unsigned char* w;       // [N][K] binary16 or uint8
  const h1 *mx, *rx, *my, *ry;  // uint8 only
  const float* bias;
  const void* res;
  void* y;
  int T, K, N, ldx, ldr, ldy, act, strips;
};

template <bool FINE>
__device__ __forceinline__ float activate(float v, int act) {
  switch (act) {
    case FRHIP_ACT_SIGMOID: return sigmoid_f<FINE>(v);
    case FRHIP_ACT_RELU2: return v > 0.f ? v * v : (v != v ? v : 0.f);
    case FRHIP_ACT_SILU: return silu_f<FINE>(v);
    case FRHIP_ACT_GELU: return 0.5f * v * erfcf(v * -0.70710678118654752440f);
    case FRHIP_ACT_SOFTPLUS: return softplus_f<FINE>(v);
    default: return v;
  }
}

// W consecutive outputs of a row, the first n of them stored; O: the type of y and the residual
template <class O, int W>
__device__ __forceinline__ void finish_outputs(const LinearArgs& a, const float (&acc)[W], int row, int col, int n) {
  typedef O any __attribute__((ext_vector_type(W), aligned(sizeof(O))));
  constexpr bool FINE = sizeof(O) == 4;
  O* const y = static_cast<O*>(a.y) + (size_t)row * a.ldy + col;
  const O* const res = a.res ? static_cast<const O*>(a.res) + (size_t)row * a.ldr + col : nullptr;
  float r[W], v[W];
#pragma unroll
  for (int i = 0; i < W; i++) r[i] = 0.f;
  if (res) {
    if (n >= W) {
      const any t = *reinterpret_cast<const any*>(res);
#pragma unroll
      for (int i = 0; i < W; i++) r[i] = (float)t[i];
    } else {
#pragma unroll
      for (int i = 0; i < W; i++)
        if (i < n) r[i] = (float)res[i];
    }
  }
#pragma unroll
  for (int i = 0; i < W; i++) v[i] = acc[i] + (a.bias && i < n ? a.bias[col + i] : 0.f);
#pragma unroll
  for (int i = 0; i < W; i++) {
    v[i] = activate<FINE>(v[i], a.act);
    if (res) v[i] += r[i];
  }
  if (n >= W) {
    any t;
#pragma unroll
    for (int i = 0; i < W; i++) t[i] = (O)v[i];
    *reinterpret_cast<any*>(y) = t;
  } else {
#pragma unroll
    for (int i = 0; i < W; i++)
      if (i < n) y[i] = (O)v[i];
  }
}

// ---------------------------------------------------------------------------
// Few rows: what counts is that all compute units pull at the weights.  A workgroup owns MT x 16 rows and NT x 16 columns; its waves take
// the K-steps in turn and their sums meet in LDS, in wave order.  Operands go from memory to the registers of the lanes that
// multiply them: a lane of the 16 x 16 x 32 MFMA takes 8 consecutive k, 16 bytes (8 codes of a uint8 weight), kLinDepth steps ahead.
// ---------------------------------------------------------------------------
constexpr int kLinWaves = 8, kLinDepth = 4;

template <int MT, int NT, bool U8, class O>
__global__ __launch_bounds__(kLinWaves * 64) void linear_few_kernel(LinearArgs a) {
  extern __shared__ __attribute__((aligned(16))) unsigned char lin_smem[];
  const int n = gridDim.x, lin = blockIdx.x, xcd = lin & 7;  // the strips that share weights share an L2
  const int id = xcd * (n >> 3) + min(xcd, n & 7) + (lin >> 3), tile = id / a.strips, strip = id - tile * a.strips;
  const int m0 = strip * (MT * 16), n0 = tile * (NT * 16), K = a.K;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), c16 = lane & 15, grp = lane >> 4;

  typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
  const h1* xp[MT];
  const unsigned char* wp[NT];
  float c[NT], m[NT];
#pragma unroll
  for (int i = 0; i < MT; i++) xp[i] = a.x + (size_t)min(m0 + i * 16 + c16, a.T - 1) * a.ldx + grp * 8;
#pragma unroll
  for (int j = 0; j < NT; j++) {
    const int col = min(n0 + j * 16 + c16, a.N - 1);
    wp[j] = a.w + ((size_t)col * K + grp * 8) * (U8 ? 1 : 2);
    if constexpr (U8) {
      c[j] = dequant_c(a.rx[col]);
      m[j] = (float)a.mx[col];
    }
  }
  f4v acc[MT][NT];
#pragma unroll
  for (int i = 0; i < MT; i++)
#pragma unroll
    for (int j = 0; j < NT; j++) acc[i][j] = (f4v){0.f, 0.f, 0.f, 0.f};

  struct Step {
    h8 x[MT], w[U8 ? 1 : NT], ry, my;
    u32x2 q[U8 ? NT : 1];
  };
  auto load = [&](Step& s, int k) {  // k: a multiple of 32; this lane's eight begin at k + 8 grp
#pragma unroll
    for (int j = 0; j < NT; j++) {
      if constexpr (U8) s.q[j] = *reinterpret_cast<const u32x2*>(wp[j] + k);
      else s.w[j] = *reinterpret_cast<const h8*>(wp[j] + (size_t)k * 2);
    }
    if constexpr (U8) {
      s.ry = *reinterpret_cast<const h8_any*>(a.ry + k + grp * 8);
      s.my = *reinterpret_cast<const h8_any*>(a.my + k + grp * 8);
    }
#pragma unroll
    for (int i = 0; i < MT; i++) s.x[i] = *reinterpret_cast<const h8*>(xp[i] + k);
  };
  auto weight = [&](const Step& s, int j) {
    if constexpr (U8) {
      const h2 p0 = few_dequant<0>(s.q[j][0], c[j], m[j], s.ry.s01, s.my.s01), p1 = few_dequant<1>(s.q[j][0], c[j], m[j], s.ry.s23, s.my.s23);
      const h2 p2 = few_dequant<0>(s.q[j][1], c[j], m[j], s.ry.s45, s.my.s45), p3 = few_dequant<1>(s.q[j][1], c[j], m[j], s.ry.s67, s.my.s67);
      return (h8){p0.x, p0.y, p1.x, p1.y, p2.x, p2.y, p3.x, p3.y};
    } else {
      return s.w[j];
    }
  };
  auto multiply = [&](const Step& s) {
#pragma unroll
    for (int j = 0; j < NT; j++) {
      const h8 w = weight(s, j);
#pragma unroll
      for (int i = 0; i < MT; i++) acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(w, s.x[i], acc[i][j], 0, 0, 0);
    }
  };
  const int full = K / 32, cnt = wave < full ? (full - wave - 1) / kLinWaves + 1 : 0;
  if (cnt > 0) {
    Step s[kLinDepth];
    auto at = [&](int i) { return (wave + min(i, cnt - 1) * kLinWaves) * 32; };  // past the last step: the last one again, not multiplied
#pragma unroll
    for (int p = 0; p < kLinDepth; p++) load(s[p], at(p));
    int i = 0;
    for (; i + kLinDepth < cnt; i += kLinDepth)
#pragma unroll
      for (int p = 0; p < kLinDepth; p++) {
        multiply(s[p]);
        load(s[p], at(i + kLinDepth + p));
      }
#pragma unroll
    for (int p = 0; p < kLinDepth; p++)
      if (i + p < cnt) multiply(s[p]);
  }
  if (full * 32 < K && wave == full % kLinWaves) {  // what is left of K
    Step s;
    memset(&s, 0, sizeof(s));
    const bool in = full * 32 + grp * 8 < K;
    if (in) load(s, full * 32);
#pragma unroll
    for (int j = 0; j < NT; j++) {
      h8 w = weight(s, j);
      if (!in) w = (h8)(h1)0.f;
#pragma unroll
      for (int i = 0; i < MT; i++) acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(w, s.x[i], acc[i][j], 0, 0, 0);
    }
  }
  // a lane's four sums are four consecutive columns of row c16
  f4v* const sums = reinterpret_cast<f4v*>(lin_smem);
#pragma unroll
  for (int i = 0; i < MT; i++)
#pragma unroll
    for (int j = 0; j < NT; j++) sums[((wave * MT + i) * NT + j) * 64 + lane] = acc[i][j];
  __syncthreads();
  for (int t = wave; t < MT * NT; t += kLinWaves) {
    const int i = t / NT, j = t - i * NT, row = m0 + i * 16 + c16, col = n0 + j * 16 + grp * 4;
    f4v s = sums[t * 64 + lane];
#pragma unroll
    for (int w = 1; w < kLinWaves; w++) s += sums[(w * MT * NT + t) * 64 + lane];
    if (row < a.T && col < a.N) {
      const float v[4] = {s[0], s[1], s[2], s[3]};
      finish_outputs<O>(a, v, row, col, a.N - col);
    }
  }
}

template <int MT, int NT, bool U8, class O>
static void few_launch(LinearArgs a, hipStream_t st) {
  a.strips = (a.T + MT * 16 - 1) / (MT * 16);
  const int tiles = (a.N + NT * 16 - 1) / (NT * 16);
  hipLaunchKernelGGL((linear_few_kernel<MT, NT, U8, O>), dim3((unsigned)((size_t)tiles * a.strips)), dim3(kLinWaves * 64), kLinWaves * MT * NT * 1024, st, a);
}

template <bool U8, class O>
static int linear_run(const LinearArgs& a, hipStream_t st) {
  if (a.T <= 16) few_launch<1, 1, U8, O>(a, st);
  else if (a.T <= 32) few_launch<2, 1, U8, O>(a, st);
  else few_launch<4, 2, U8, O>(a, st);
  return check_launch("linear");
}

}  // namespace frhip

using namespace frhip;

extern "C" size_t frhip_linear_workspace_bytes(int T, const frhip_weight* w) {
  (void)T;
  (void)w;
  return 0;
}

extern "C" int frhip_linear(const void* x, int ldx, const frhip_weight* w, const float* bias, int act, const void* residual, int ldr, void* y,
                            int ldy, int T, int out_dtype, void* workspace, frhip_stream s) {
  if (!w || !w->data) return set_error(FRHIP_EINVAL, "linear: null pointer");
  if (out_dtype != FRHIP_F16 && out_dtype != FRHIP_F32) return set_error(FRHIP_EINVAL, "linear: out_dtype must be F16 or F32");
  if (act != FRHIP_ACT_NONE && (act < FRHIP_ACT_SIGMOID || act > FRHIP_ACT_SOFTPLUS)) return set_error(FRHIP_EINVAL, "linear: unknown act");
  if (w->dtype != FRHIP_F16 && w->dtype != FRHIP_U8) return set_error(FRHIP_EINVAL, "linear: weight dtype must be F16 or U8");
  if (w->dtype == FRHIP_U8 && (!w->mx || !w->rx || !w->my || !w->ry)) return set_error(FRHIP_EINVAL, "linear: uint8 weight without mx/rx/my/ry");
  if (T < 0 || w->K <= 0 || w->N <= 0 || w->K % 8 != 0) return set_error(FRHIP_ESHAPE, "linear: K must be a multiple of 8, T not negative");
  if (ldx < w->K || ldx % 8 != 0 || ldy < w->N || (residual && ldr < w->N)) return set_error(FRHIP_ESHAPE, "linear: rows closer than their elements, or ldx no multiple of 8");
  if (T == 0) return 0;
  if (!x || !y) return set_error(FRHIP_EINVAL, "linear: null pointer");
  const size_t elem = out_dtype == FRHIP_F16 ? 2 : 4, rows = T, K = w->K, N = w->N;
  if (off_grid(16, {x, w->data}) || off_grid(4, {bias}) || off_grid(elem, {residual, y}) || off_grid(2, {w->mx, w->rx, w->my, w->ry}))
    return set_error(FRHIP_EINVAL, "linear: pointer not aligned");
  const size_t ye = ((rows - 1) * ldy + N) * elem;
  auto hits = [&](const void* p, size_t bytes) { return rows_overlap(p, bytes, y, ye, 1, bytes, ye, 1); };
  const size_t xe = ((rows - 1) * ldx + K) * 2;
  if (out_dtype == FRHIP_F16 ? rows_overlap(x, ldx, y, ldy, rows, K, N, 2) : hits(x, xe)) return set_error(FRHIP_EINVAL, "linear: y overlaps x");
  if (residual && !(residual == y && ldr == ldy) && rows_overlap(residual, ldr, y, ldy, rows, N, N, elem))
    return set_error(FRHIP_EINVAL, "linear: y overlaps the residual in part");
  if (hits(w->data, N * K * (w->dtype == FRHIP_U8 ? 1 : 2)) || hits(bias, N * 4) || hits(w->mx, N * 2) || hits(w->rx, N * 2) || hits(w->my, K * 2) ||
      hits(w->ry, K * 2))
    return set_error(FRHIP_EINVAL, "linear: y overlaps the weight");
  LinearArgs a;
  memset(&a, 0, sizeof(a));
  a.x = static_cast<const h1*>(x);
  a.w = static_cast<const unsigned char*>(w->data);
  a.mx = static_cast<const h1*>(w->mx);
  a.rx = static_cast<const h1*>(w->rx);
  a.my = static_cast<const h1*>(w->my);
  a.ry = static_cast<const h1*>(w->ry);
  a.bias = bias;
  a.res = residual;
  a.y = y;
  a.T = T;
  a.K = w->K;
  a.N = w->N;
  a.ldx = ldx;
  a.ldr = ldr;
  a.ldy = ldy;
  a.act = act;
  hipStream_t st = static_cast<hipStream_t>(s);
  (void)workspace;
  if (w->dtype == FRHIP_U8) return out_dtype == FRHIP_F16 ? linear_run<true, h1>(a, st) : linear_run<true, float>(a, st);
  return out_dtype == FRHIP_F16 ? linear_run<false, h1>(a, st) : linear_run<false, float>(a, st);
}
