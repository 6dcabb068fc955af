// Products with bias, activation and residual: y = residual + act(x . w + bias), for any number of rows, K a multiple of 8, any N, rows of
// any pitch.  Sums are fp32 on the MFMA units, the epilogue is fp32, and a result is rounded once.
#include <climits>
#include <cstring>

#include "activations.h"
#include "gemm_ring_device.h"
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

// ---------------------------------------------------------------------------
// More rows: tiles of 64 or 128 rows, four waves that multiply and four that load (gemm_ring.hip has the form and its reasons), here with
// rows of any pitch and a K that need not fill its last step.  The sums go through LDS to the epilogue, which all waves share.
// ---------------------------------------------------------------------------
struct LinearTiles {
  LinearArgs l;
  int base, wide, maxw;  // tiles are `base` blocks of 32 columns wide, the first `wide` of them one more; the widest
};

// The waves that multiply: the nk steps of a wave's 32 BM / 64 rows and 32 NJ columns (from row `brow0` of the tile's B)
template <int BM, int S, int NJ, bool TAIL>
__device__ __forceinline__ void ring_products(f16v (&acc)[BM / 64][NJ], const unsigned char* smem, int stage, int brow0, int nk, int lane, int wm,
                                              int krest) {
  constexpr int MI = BM / 64, KG = MI * NJ >= 6 ? 2 : 4;
#pragma unroll
  for (int i = 0; i < MI; i++)
#pragma unroll
    for (int j = 0; j < NJ; j++)
#pragma unroll
      for (int v = 0; v < 16; v++) acc[i][j][v] = 0.f;
  const unsigned char* as = smem;
  for (int k = 0; k < nk; k++) {
    step_barrier();
    const unsigned char* bs = as + BM * 128;
#pragma unroll
    for (int kh = 0; kh < 4; kh += KG) {
      h8 fa[KG][MI], fb[KG][NJ];
#pragma unroll
      for (int kb = 0; kb < KG; kb++) {
        const int q = (kh + kb) * 2 + (lane >> 5);
#pragma unroll
        for (int i = 0; i < MI; i++) fa[kb][i] = *reinterpret_cast<const h8*>(as + ldw_at(wm * (BM / 2) + i * 32 + (lane & 31), q));
#pragma unroll
        for (int j = 0; j < NJ; j++) fb[kb][j] = *reinterpret_cast<const h8*>(bs + ldw_at(brow0 + j * 32 + (lane & 31), q));
        if constexpr (TAIL) {
          if (k == nk - 1) {
            const h8 none = (h8)(h1)0.f;
#pragma unroll
            for (int i = 0; i < MI; i++) fa[kb][i] = q * 8 < krest ? fa[kb][i] : none;
#pragma unroll
            for (int j = 0; j < NJ; j++) fb[kb][j] = q * 8 < krest ? fb[kb][j] : none;
          }
        }
      }
#pragma unroll
      for (int kb = 0; kb < KG; kb++)
#pragma unroll
        for (int i = 0; i < MI; i++)
#pragma unroll
          for (int j = 0; j < NJ; j++)
            acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_f16(fa[kb][i], fb[kb][j], acc[i][j], 0, 0, 0);
    }
    as += stage;
    as = as == smem + S * stage ? smem : as;
  }
}

template <int BM, int S, int NJ, bool TAIL>
__device__ __forceinline__ void linear_mma(unsigned char* smem, int stage, int maxw, int brow0, int nk, int krest, int lane, int wm) {
  if constexpr (NJ == 0) {  // a tile of one block: the first wave column has it
    for (int k = 0; k < nk; k++) step_barrier();
    step_barrier();
  } else {
    f16v acc[BM / 64][NJ];
    ring_products<BM, S, NJ, TAIL>(acc, smem, stage, brow0, nk, lane, wm, krest);
    step_barrier();  // all fragments have been read
    const int pitch = sums_pitch(maxw);
#pragma unroll
    for (int i = 0; i < BM / 64; i++) sums_to_lds(acc[i], reinterpret_cast<float*>(smem) + (wm * (BM / 2) + i * 32) * pitch + brow0, pitch, lane);
  }
}

template <int BM, int S, bool TAIL, class O>
__global__ __launch_bounds__(kRingThreads) void linear_ring_kernel(LinearTiles a) {
  extern __shared__ __attribute__((aligned(16))) unsigned char ring_smem[];
  constexpr int kMost = BM == 128 && S == 4 ? 6 : kRingMostBlocks;
  int bx, by;
  xcd_tile(bx, by);
  const int width = a.base + (bx < a.wide ? 1 : 0), n0 = (bx * a.base + min(bx, a.wide)) * 32, m0 = by * BM;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int nk = (a.l.K + kLdwBK - 1) / kLdwBK, krest = a.l.K - (nk - 1) * kLdwBK, stage = BM * 128 + a.maxw * 4096;
  if (wave >= 4) {
    const int p = wave - 4;
    const RingOperands o = {a.l.x, a.l.w, a.l.T, a.l.N, a.l.ldx, a.l.K};
    switch (width) {
      case 1: ring_loader<BM, S, 1, TAIL>(o, ring_smem, stage, p, m0, n0, 0, nk, lane, krest); break;
      case 2: ring_loader<BM, S, 2, TAIL>(o, ring_smem, stage, p, m0, n0, 0, nk, lane, krest); break;
      case 3: ring_loader<BM, S, 3, TAIL>(o, ring_smem, stage, p, m0, n0, 0, nk, lane, krest); break;
      case 4: ring_loader<BM, S, 4, TAIL>(o, ring_smem, stage, p, m0, n0, 0, nk, lane, krest); break;
      case 5: ring_loader<BM, S, 5, TAIL>(o, ring_smem, stage, p, m0, n0, 0, nk, lane, krest); break;
      case 6: ring_loader<BM, S, 6, TAIL>(o, ring_smem, stage, p, m0, n0, 0, nk, lane, krest); break;
      case 7: ring_loader<BM, S, kMost < 7 ? kMost : 7, TAIL>(o, ring_smem, stage, p, m0, n0, 0, nk, lane, krest); break;
      default: ring_loader<BM, S, kMost, TAIL>(o, ring_smem, stage, p, m0, n0, 0, nk, lane, krest); break;
    }
    step_barrier();
  } else {
    const int wm = wave >> 1, nj0 = (width + 1) >> 1, nj = (wave & 1) ? width - nj0 : nj0, brow0 = (wave & 1) ? nj0 * 32 : 0;
    switch (nj) {  // every wave passes the same barriers, whatever its width
      case 0: linear_mma<BM, S, 0, TAIL>(ring_smem, stage, a.maxw, brow0, nk, krest, lane, wm); break;
      case 1: linear_mma<BM, S, 1, TAIL>(ring_smem, stage, a.maxw, brow0, nk, krest, lane, wm); break;
      case 2: linear_mma<BM, S, 2, TAIL>(ring_smem, stage, a.maxw, brow0, nk, krest, lane, wm); break;
      case 3: linear_mma<BM, S, 3, TAIL>(ring_smem, stage, a.maxw, brow0, nk, krest, lane, wm); break;
      default: linear_mma<BM, S, kMost / 2, TAIL>(ring_smem, stage, a.maxw, brow0, nk, krest, lane, wm); break;
    }
  }
  __syncthreads();
  const float* const sums = reinterpret_cast<const float*>(ring_smem);
  const int pitch = sums_pitch(a.maxw), groups = width * 4;  // of 8 outputs
  for (int i = threadIdx.x; i < BM * groups; i += kRingThreads) {
    const int row = i / groups, col = (i - row * groups) * 8;
    if (m0 + row >= a.l.T || n0 + col >= a.l.N) continue;
    float s[8];
    read_sums(s, sums + row * pitch + col);
    finish_outputs<O>(a.l, s, m0 + row, n0 + col, a.l.N - n0 - col);
  }
}

template <int BM, int S, bool TAIL, class O>
static void ring_launch(const TilePlan& p, const LinearTiles& t, hipStream_t st) {
  static const bool raised = [] {
    (void)hipFuncSetAttribute(reinterpret_cast<const void*>(&linear_ring_kernel<BM, S, TAIL, O>), hipFuncAttributeMaxDynamicSharedMemorySize, 160 * 1024);
    return true;
  }();
  (void)raised;
  const int ring = S * (BM * 128 + t.maxw * 4096), sums = BM * sums_pitch(t.maxw) * 4;
  hipLaunchKernelGGL((linear_ring_kernel<BM, S, TAIL, O>), p.grid, dim3(kRingThreads), ring > sums ? ring : sums, st, t);
}

// The cut of such a launch is that of the same product on gemm_ring_kernel; rows = 0: operands whose rows are too long for its offsets
static TilePlan plan_tiles(const LinearArgs& a) {
  GemmArgs g;
  memset(&g, 0, sizeof(g));
  if (a.K > INT_MAX - kLdwBK || (size_t)a.ldx * 2 * 256 > 0xffffffffull) return TilePlan();
  g.M = a.T;
  g.K = (a.K + kLdwBK - 1) / kLdwBK * kLdwBK;
  g.nseg = 1;
  g.seg[0].N = a.N;
  return plan_ring(g, compute_units());
}

template <bool TAIL, class O>
static int launch_tiles(const LinearArgs& a, const TilePlan& p, hipStream_t st) {
  const LinearTiles t = {a, p.a.vw_base[0], p.a.vw_wide[0], p.a.vw_maxw};
  if (p.rows == 64) ring_launch<64, 4, TAIL, O>(p, t, st);
  else if (ring_stages(128, t.maxw) == 4) ring_launch<128, 4, TAIL, O>(p, t, st);
  else ring_launch<128, 3, TAIL, O>(p, t, st);
  return check_launch("linear");
}

constexpr int kLinFewRows = 64;  // rows up to which a product goes out as one of few rows

template <bool U8, class O>
static int linear_run(const LinearArgs& a, hipStream_t st) {
  if (a.T <= 16) few_launch<1, 1, U8, O>(a, st);
  else if (a.T <= 32) few_launch<2, 1, U8, O>(a, st);
  else few_launch<4, 2, U8, O>(a, st);
  return check_launch("linear");
}

template <class O>
static int linear_any(LinearArgs a, bool u8, void* workspace, hipStream_t st) {
  if (a.T > kLinFewRows) {
    const TilePlan p = plan_tiles(a);
    if (p.rows) {
      if (u8) {
        if (int rc = dequant_u8_async(a.w, a.mx, a.rx, a.my, a.ry, static_cast<h1*>(workspace), a.K, a.N, st)) return rc;
        a.w = static_cast<const unsigned char*>(workspace);
      }
      return a.K % kLdwBK ? launch_tiles<true, O>(a, p, st) : launch_tiles<false, O>(a, p, st);
    }
  }
  return u8 ? linear_run<true, O>(a, st) : linear_run<false, O>(a, st);
}

}  // namespace frhip

using namespace frhip;

extern "C" size_t frhip_linear_workspace_bytes(int T, const frhip_weight* w) {
  if (!w || T <= kLinFewRows || w->dtype != FRHIP_U8 || w->K <= 0 || w->N <= 0) return 0;
  return ((size_t)w->K * w->N * 2 + 255) / 256 * 256;  // the weight in binary16
}

extern "C" int frhip_linear(const void* x, int ldx, const frhip_weight* w, const float* bias, int act, const void* residual, int ldr, void* y,
                            int ldy, int T, int out_dtype, void* workspace, frhip_stream s) {
  if (!w || !w->data) return set_error(FRHIP_EINVAL, "linear: null pointer");
  if (out_dtype != FRHIP_F16 && out_dtype != FRHIP_F32) return set_error(FRHIP_EINVAL, "linear: out_dtype must be F16 or F32");
  if (act != FRHIP_ACT_NONE && (act < FRHIP_ACT_SIGMOID || act > FRHIP_ACT_SOFTPLUS)) return set_error(FRHIP_EINVAL, "linear: unknown act");
  if (w->dtype != FRHIP_F16 && w->dtype != FRHIP_U8) return set_error(FRHIP_EINVAL, "linear: weight dtype must be F16 or U8");
  if (w->dtype == FRHIP_U8 && (!w->mx || !w->rx || !w->my || !w->ry)) return set_error(FRHIP_EINVAL, "linear: uint8 weight without mx/rx/my/ry");
  if (T < 0 || T > 1 << 30 || w->K <= 0 || w->N <= 0 || w->K % 8 != 0) return set_error(FRHIP_ESHAPE, "linear: K must be a multiple of 8, T 0 to 2^30");
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
  const bool u8 = w->dtype == FRHIP_U8;
  if (frhip_linear_workspace_bytes(T, w) > 0) {
    if (!workspace) return set_error(FRHIP_EINVAL, "linear: null workspace");
    if (off_grid(16, {workspace})) return set_error(FRHIP_EINVAL, "linear: workspace must be 16-byte aligned");
  }
  return out_dtype == FRHIP_F16 ? linear_any<h1>(a, u8, workspace, st) : linear_any<float>(a, u8, workspace, st);
}
