// Norms before and after a block, fused with what stands between them.
//
//   norm_gate      y = (norm(x) w + b) act(z), every head of a row normalised by itself: behind a recurrence, ahead of the product out of it
//   norm_residual  h = x + scale channels act(gate) norm(block), y = norm(h): from one block's output to the next one's input
//
// A norm is v / sqrt(mean v^2 + eps), of v itself or of v less its mean.  Both are bound by memory: every element once in and once out.  A row (a
// head of it) lies in the registers of a group of lanes, which sums its squares there; the mean is taken out ahead of them, so that
// a large one costs no digits.  The widest forms, of heads above 8192 and residual rows above 16384, have more than registers hold: part of a row goes to
// scratch memory and back (512 heads of 16384 of binary16: 386 us, 0.13 TB/s; 512 residual rows of 32768: 51 to 115 us, 2.3 to 2.6 TB/s).
#include <algorithm>
#include <cstring>

#include "activations.h"
#include "frhip_internal.h"
#include "groups.h"
#include "lanes.h"
#include "prompts.h"
#include "spans.h"

#pragma clang fp contract(off)

namespace frhip {

constexpr int kNormLanes = 8;        // elements of a lane's group: 16 bytes of binary16
constexpr int kMostCols = 1 << 15;   // of a norm: 32 elements a thread of the largest workgroup

struct Norm {
  const float *w, *b;
  float eps;
  int kind;
};

// A lane's eight elements as they are in memory, the first n - at of a row's from `at` on
template <class T>
struct Raw {
  typedef T any __attribute__((ext_vector_type(kNormLanes), aligned(sizeof(T))));
  any v;
  __device__ __forceinline__ void load(const T* row, int at, int n) {
    if (n - at >= kNormLanes) {
      v = *reinterpret_cast<const any*>(row + at);
    } else {
#pragma unroll
      for (int i = 0; i < kNormLanes; i++) v[i] = at + i < n ? row[at + i] : (T)0.f;
    }
  }
};

// The sum over a row's lanes: LANES of them, up to a wave, or (0) the workgroup's
template <int LANES>
__device__ __forceinline__ float row_sum(float v, float* red) {
  if constexpr (LANES > 0) {
    return lane_sum<LANES>(v);
  } else {
    v = lane_sum<64>(v);
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
    __syncthreads();
    float t = red[0];
    for (int i = 1; i < (int)blockDim.x / 64; i++) t += red[i];
    return t;
  }
}

// Of n elements, group g of a lane begins at `at` + g `step`; what is behind them is zero and stays so
template <int LANES, int G>
__device__ __forceinline__ void normalise(float (&v)[G][kNormLanes], int at, int step, int n, int kind, float eps, float (*red)[16], int& turn) {
  const float inv = 1.0f / (float)n;
  if (kind == FRHIP_NORM_MEAN) {
    float s = 0.f;
#pragma unroll
    for (int g = 0; g < G; g++)
#pragma unroll
      for (int i = 0; i < kNormLanes; i++) s += v[g][i];
    const float mean = row_sum<LANES>(s, red[turn]) * inv;
    turn ^= 1;
#pragma unroll
    for (int g = 0; g < G; g++)
#pragma unroll
      for (int i = 0; i < kNormLanes; i++) v[g][i] = at + g * step + i < n ? v[g][i] - mean : 0.f;
  }
  float s = 0.f;
#pragma unroll
  for (int g = 0; g < G; g++)
#pragma unroll
    for (int i = 0; i < kNormLanes; i++) s = __builtin_fmaf(v[g][i], v[g][i], s);
  const float r = __builtin_amdgcn_rsqf(__builtin_fmaf(row_sum<LANES>(s, red[turn]), inv, eps));
  turn ^= 1;
#pragma unroll
  for (int g = 0; g < G; g++)
#pragma unroll
    for (int i = 0; i < kNormLanes; i++) v[g][i] *= r;
}

template <int G, class T>
__device__ __forceinline__ void load_row(float (&v)[G][kNormLanes], const T* p, int at, int step, int n) {
#pragma unroll
  for (int g = 0; g < G; g++) {
    const int c = at + g * step;
    load_group<T, kNormLanes>(v[g], p + (c < n ? c : 0), n - c);
  }
}
template <int G, class T>
__device__ __forceinline__ void store_row(T* p, const float (&v)[G][kNormLanes], int at, int step, int n) {
#pragma unroll
  for (int g = 0; g < G; g++) {
    const int c = at + g * step;
    if (c < n) store_group<T, kNormLanes>(p + c, v[g], n - c);
  }
}

template <bool FINE, int G>
__device__ __forceinline__ void times_act(float (&v)[G][kNormLanes], const float (&z)[G][kNormLanes], int act) {
#pragma unroll
  for (int g = 0; g < G; g++)
#pragma unroll
    for (int i = 0; i < kNormLanes; i++) {
      const float e = act == FRHIP_ACT_NONE ? z[g][i] : sigmoid_f<FINE>(z[g][i]);
      v[g][i] *= act == FRHIP_ACT_SILU ? z[g][i] * e : e;
    }
}

// ---------------------------------------------------------------------------
// norm_gate
// ---------------------------------------------------------------------------
template <class T>
struct GateArgs {
  const T *x, *z;
  T* y;
  Norm norm;
  int rows, heads, dim, ldx, ldz, ldy, act;
  int shift;  // 2^shift neighbouring groups of a workgroup take neighbouring heads, the others further rows
};

// blockIdx.x: heads, blockIdx.y, and so on by gridDim.y: rows.  A group of LANES lanes (0: the workgroup) keeps its head, and so the head's parameters.
// 4096 rows of 32 heads of 128 of binary16: 20.4 us, 4.9 TB/s, as a large copy has.
template <class T, int LANES, int G>
__global__ __launch_bounds__(LANES ? 256 : 1024) void norm_gate_kernel(GateArgs<T> a) {
  constexpr int GROUPS = LANES ? 256 / (LANES ? LANES : 1) : 1;
  __shared__ float red[2][16];
  const int lanes = LANES ? LANES : blockDim.x, group = LANES ? threadIdx.x / lanes : 0, at = (threadIdx.x - group * lanes) * kNormLanes, n = a.dim;
  const int grid_step = lanes * kNormLanes;
  const int head = (blockIdx.x << a.shift) + (group & ((1 << a.shift) - 1)), step = GROUPS >> a.shift;
  if (head >= a.heads) return;  // a workgroup that has one head stays together
  const size_t c0 = (size_t)head * n;
  float w[G][kNormLanes], b[G][kNormLanes];
  if (a.norm.w) load_row<G>(w, a.norm.w + c0, at, grid_step, n);
  if (a.norm.b) load_row<G>(b, a.norm.b + c0, at, grid_step, n);
  int turn = 0;
  for (int row = blockIdx.y * step + (group >> a.shift); row < a.rows; row += gridDim.y * step) {
    float v[G][kNormLanes], z[G][kNormLanes];
    load_row<G>(v, a.x + (size_t)row * a.ldx + c0, at, grid_step, n);
    if (a.z) load_row<G>(z, a.z + (size_t)row * a.ldz + c0, at, grid_step, n);
    normalise<LANES, G>(v, at, grid_step, n, a.norm.kind, a.norm.eps, red, turn);
#pragma unroll
    for (int g = 0; g < G; g++)
#pragma unroll
      for (int i = 0; i < kNormLanes; i++) {
        if (a.norm.w) v[g][i] *= w[g][i];
        if (a.norm.b) v[g][i] += b[g][i];
      }
    if (a.z) times_act<sizeof(T) == 4, G>(v, z, a.act);
    store_row<G>(a.y + (size_t)row * a.ldy + c0, v, at, grid_step, n);
  }
}

template <class T, int LANES, int G>
static int gate_launch(GateArgs<T> a, hipStream_t st) {
  constexpr int GROUPS = LANES ? 256 / (LANES ? LANES : 1) : 1;
  const int threads = LANES ? 256 : std::min(1024, ((a.dim - 1) / kNormLanes / 64 + 1) * 64);
  a.shift = 0;
  while ((1 << a.shift) < GROUPS && (1 << a.shift) < a.heads) a.shift++;
  const int step = GROUPS >> a.shift, blocks = (a.heads - 1) / (1 << a.shift) + 1;
  // rows over about 32 waves a compute unit, so that a group's parameters serve several of them
  const int want = compute_units() * std::max(1, 2048 / threads) / blocks + 1, most = (a.rows - 1) / step + 1;
  hipLaunchKernelGGL((norm_gate_kernel<T, LANES, G>), dim3(blocks, std::min(std::min(want, most), 65535)), dim3(threads), 0, st, a);
  return check_launch("norm_gate");
}

template <class T>
static int gate_run(const GateArgs<T>& a, hipStream_t st) {
  const int n = a.dim;
  if (n <= 64) return gate_launch<T, 8, 1>(a, st);
  if (n <= 128) return gate_launch<T, 16, 1>(a, st);
  if (n <= 256) return gate_launch<T, 32, 1>(a, st);
  if (n <= 512) return gate_launch<T, 64, 1>(a, st);
  if (n <= 8192) return gate_launch<T, 0, 1>(a, st);
  return gate_launch<T, 0, 4>(a, st);
}

// ---------------------------------------------------------------------------
// norm_residual
// ---------------------------------------------------------------------------
template <class S, class T>
struct ResidualArgs {
  const S* x;
  const T *block, *gate;
  S* h;
  T* y;
  Norm after, before;
  const float* channels;
  int rows, cols, ldx, ldb, ldg, ldh, ldy, act;
  float scale;
};

// A row of at most 512 elements a wave (WIDE: a workgroup, G groups of eight a thread); blockIdx.x, and so on by gridDim.x: the rows.  A row's
// loads go out ahead of the sums of the row before.
// 4096 rows of 2560, two norms, a gate, a stream in fp32: 35 us, 4.2 TB/s; twelve workgroups of five waves a compute unit (six: 37).
template <class S, class T, int G, bool WIDE>
__global__ __launch_bounds__(WIDE ? 1024 : 256) void norm_residual_kernel(ResidualArgs<S, T> a) {
  constexpr bool FINE = sizeof(S) == 4 || sizeof(T) == 4;
  constexpr int GROUPS = WIDE ? 1 : 4;
  __shared__ float red[2][16];
  const int group = WIDE ? 0 : threadIdx.x / 64, lanes = WIDE ? blockDim.x : 64, at = (WIDE ? threadIdx.x : threadIdx.x & 63) * kNormLanes, n = a.cols;
  const int step = lanes * kNormLanes;
  constexpr bool AHEAD = G == 1;  // rows of more than 8192 have no registers to spare
  // f(i, parameter) for the lane's eight of group g.  (In registers from row to row they cost as many waves as they save: 41 us instead of 37.)
  auto with = [&](const float* params, int g, auto f) {
    if (!params) return;
    const int c = at + g * step;
    float p[kNormLanes];
    load_group<float, kNormLanes>(p, params + (c < n ? c : 0), n - c);
#pragma unroll
    for (int i = 0; i < kNormLanes; i++) f(i, p[i]);
  };
  Raw<S> xr[G];
  Raw<T> br[G], gr[G];
  const int first = blockIdx.x * GROUPS + group, stride = gridDim.x * GROUPS;
  auto request = [&](int row) {
#pragma unroll
    for (int g = 0; g < G; g++) {
      const int c = at + g * step;
      if (a.block) br[g].load(a.block + (size_t)row * a.ldb, c, n);
      if (a.gate) gr[g].load(a.gate + (size_t)row * a.ldg, c, n);
      xr[g].load(a.x + (size_t)row * a.ldx, c, n);
    }
  };
  if (AHEAD && first < a.rows) request(first);
  int turn = 0;
  for (int row = first; row < a.rows; row += stride) {
    if (!AHEAD) request(row);
    float h[G][kNormLanes], v[G][kNormLanes], z[G][kNormLanes];
#pragma unroll
    for (int g = 0; g < G; g++)
#pragma unroll
      for (int i = 0; i < kNormLanes; i++) {
        h[g][i] = (float)xr[g].v[i];
        v[g][i] = a.block ? (float)br[g].v[i] : 0.f;
        z[g][i] = a.gate ? (float)gr[g].v[i] : 0.f;
      }
    if (AHEAD && a.rows - row > stride) request(row + stride);
    if (a.block) {
      if (a.after.kind != FRHIP_NORM_NONE) {
        normalise<WIDE ? 0 : 64, G>(v, at, step, n, a.after.kind, a.after.eps, red, turn);
#pragma unroll
        for (int g = 0; g < G; g++) {
          with(a.after.w, g, [&](int i, float p) { v[g][i] *= p; });
          with(a.after.b, g, [&](int i, float p) { v[g][i] += p; });
        }
      }
      if (a.gate) times_act<FINE, G>(v, z, a.act);
#pragma unroll
      for (int g = 0; g < G; g++) {
        with(a.channels, g, [&](int i, float p) { v[g][i] *= p; });
#pragma unroll
        for (int i = 0; i < kNormLanes; i++) h[g][i] = __builtin_fmaf(a.scale, v[g][i], h[g][i]);
      }
    }
    if (a.h) store_row<G>(a.h + (size_t)row * a.ldh, h, at, step, n);
    if (a.y) {
      if (a.before.kind != FRHIP_NORM_NONE) {
        normalise<WIDE ? 0 : 64, G>(h, at, step, n, a.before.kind, a.before.eps, red, turn);
#pragma unroll
        for (int g = 0; g < G; g++) {
          with(a.before.w, g, [&](int i, float p) { h[g][i] *= p; });
          with(a.before.b, g, [&](int i, float p) { h[g][i] += p; });
        }
      }
      store_row<G>(a.y + (size_t)row * a.ldy, h, at, step, n);
    }
  }
}

template <class S, class T, int G, bool WIDE>
static int residual_launch(const ResidualArgs<S, T>& a, hipStream_t st) {
  const int groups = (a.cols - 1) / kNormLanes + 1, threads = WIDE ? std::min(1024, (groups + 63) / 64 * 64) : 256;
  const int per = WIDE ? 1 : 4, want = compute_units() * std::max(1, 4096 / threads), most = (a.rows - 1) / per + 1;
  hipLaunchKernelGGL((norm_residual_kernel<S, T, G, WIDE>), dim3(std::min(want, most)), dim3(threads), 0, st, a);
  return check_launch("norm_residual");
}

template <class S, class T>
static int residual_run(const frhip_block_norm& p, int rows, const void* x, int ldx, const void* block, int ldb, const void* gate, int ldg, void* h,
                        int ldh, void* y, int ldy, hipStream_t st) {
  ResidualArgs<S, T> a;
  memset(&a, 0, sizeof(a));
  a.x = static_cast<const S*>(x);
  a.block = static_cast<const T*>(block);
  a.gate = static_cast<const T*>(gate);
  a.h = static_cast<S*>(h);
  a.y = static_cast<T*>(y);
  a.after = {p.after_w, p.after_b, p.eps, p.after};
  a.before = {p.before_w, p.before_b, p.eps, p.before};
  a.channels = p.channels;
  a.rows = rows;
  a.cols = p.cols;
  a.ldx = ldx;
  a.ldb = ldb;
  a.ldg = ldg;
  a.ldh = ldh;
  a.ldy = ldy;
  a.act = p.gate_act;
  a.scale = p.scale;
  if (p.cols <= 512) return residual_launch<S, T, 1, false>(a, st);
  if (p.cols <= 8192) return residual_launch<S, T, 1, true>(a, st);
  if (p.cols <= 16384) return residual_launch<S, T, 2, true>(a, st);
  return residual_launch<S, T, 4, true>(a, st);
}

// ---------------------------------------------------------------------------
// Host side
// ---------------------------------------------------------------------------
static bool is_norm(int kind) { return kind == FRHIP_NORM_RMS || kind == FRHIP_NORM_MEAN; }
static bool is_gate_act(int act) { return act == FRHIP_ACT_NONE || act == FRHIP_ACT_SIGMOID || act == FRHIP_ACT_SILU; }
static bool is_type(int dtype) { return dtype == FRHIP_F16 || dtype == FRHIP_F32; }
static size_t type_size(int dtype) { return dtype == FRHIP_F16 ? 2 : 4; }

struct Rows {
  const void* p;
  size_t ld, cols, elem;
  size_t bytes(size_t rows) const { return ((rows - 1) * ld + cols) * elem; }
};
// Whether two sets of `rows` rows share memory; of one pitch in bytes they may lie side by side
static bool rows_meet(const Rows& a, const Rows& b, size_t rows) {
  return rows_overlap(a.p, a.ld * a.elem, b.p, b.ld * b.elem, rows, a.cols * a.elem, b.cols * b.elem, 1);
}

}  // namespace frhip

using namespace frhip;

extern "C" int frhip_norm_gate(int rows, int heads, int dim, int kind, const float* w, const float* b, float eps, const void* x, int ldx, const void* z,
                               int ldz, int act, void* y, int ldy, int dtype, frhip_stream s) {
  if (!is_type(dtype)) return set_error(FRHIP_EINVAL, "norm_gate: dtype must be F16 or F32");
  if (!is_norm(kind) || !is_gate_act(act)) return set_error(FRHIP_EINVAL, "norm_gate: no such norm or activation");
  if (!(eps >= 0.f)) return set_error(FRHIP_EINVAL, "norm_gate: eps must not be negative");
  if (rows < 0 || rows > kMostRows) return set_error(FRHIP_ESHAPE, "norm_gate: rows must be 0 to 2^30");
  if (dim <= 0 || dim > kMostCols || heads <= 0 || (long long)heads * dim > kMostChannels)
    return set_error(FRHIP_ESHAPE, "norm_gate: heads of 1 to 2^15 elements, a row up to 2^24");
  const int n = heads * dim;
  if (ldx < n || ldy < n || (z && ldz < n)) return set_error(FRHIP_ESHAPE, "norm_gate: rows closer than their elements");
  if (rows && (!x || !y)) return set_error(FRHIP_EINVAL, "norm_gate: null pointer");
  const size_t e = type_size(dtype), cols = n;
  if (off_grid(e, {x, z, y}) || off_grid(4, {w, b})) return set_error(FRHIP_EINVAL, "norm_gate: pointer not aligned to its element");
  if (rows == 0) return 0;
  const Rows in = {x, (size_t)ldx, cols, e}, gate = {z, (size_t)ldz, cols, e}, out = {y, (size_t)ldy, cols, e};
  if (((y != x || ldy != ldx) && rows_meet(in, out, rows)) || rows_meet(gate, out, rows) || spans_meet(y, out.bytes(rows), w, cols * 4) ||
      spans_meet(y, out.bytes(rows), b, cols * 4))
    return set_error(FRHIP_EINVAL, "norm_gate: the output overlaps what is read");
  auto run = [&](auto t) {
    typedef decltype(t) T;
    GateArgs<T> a;
    memset(&a, 0, sizeof(a));
    a.x = static_cast<const T*>(x);
    a.z = static_cast<const T*>(z);
    a.y = static_cast<T*>(y);
    a.norm = {w, b, eps, kind};
    a.rows = rows;
    a.heads = heads;
    a.dim = dim;
    a.ldx = ldx;
    a.ldz = ldz;
    a.ldy = ldy;
    a.act = act;
    return gate_run(a, static_cast<hipStream_t>(s));
  };
  return dtype == FRHIP_F16 ? run(h1()) : run(float());
}

extern "C" int frhip_norm_residual(const frhip_block_norm* p, int rows, const void* x, int ldx, const void* block, int ldb, const void* gate, int ldg,
                                   void* h, int ldh, int stream_dtype, void* y, int ldy, int dtype, frhip_stream s) {
  if (!p) return set_error(FRHIP_EINVAL, "norm_residual: null pointer");
  if (!is_type(dtype) || !is_type(stream_dtype)) return set_error(FRHIP_EINVAL, "norm_residual: types must be F16 or F32");
  for (int kind : {p->after, p->before})
    if (kind != FRHIP_NORM_NONE && !is_norm(kind)) return set_error(FRHIP_EINVAL, "norm_residual: no such norm");
  if (!is_gate_act(p->gate_act)) return set_error(FRHIP_EINVAL, "norm_residual: no such activation");
  if (!(p->eps >= 0.f)) return set_error(FRHIP_EINVAL, "norm_residual: eps must not be negative");
  if (rows < 0 || rows > kMostRows) return set_error(FRHIP_ESHAPE, "norm_residual: rows must be 0 to 2^30");
  const int n = p->cols;
  if (n <= 0 || n > kMostCols) return set_error(FRHIP_ESHAPE, "norm_residual: rows of 1 to 2^15 elements");
  if (ldx < n || (block && ldb < n) || (block && gate && ldg != 0 && ldg < n) || (h && ldh < n) || (y && ldy < n))
    return set_error(FRHIP_ESHAPE, "norm_residual: rows closer than their elements");
  if (rows && (!x || (!h && !y))) return set_error(FRHIP_EINVAL, "norm_residual: null pointer");
  if (gate && !block) return set_error(FRHIP_EINVAL, "norm_residual: a gate without a block");
  const size_t se = type_size(stream_dtype), e = type_size(dtype), cols = n;
  const float* params[] = {p->after_w, p->after_b, p->before_w, p->before_b, p->channels};
  if (off_grid(se, {x, h}) || off_grid(e, {block, gate, y}) || off_grid(4, {params[0], params[1], params[2], params[3], params[4]}))
    return set_error(FRHIP_EINVAL, "norm_residual: pointer not aligned to its element");
  if (rows == 0) return 0;
  const Rows xr = {x, (size_t)ldx, cols, se}, br = {block, (size_t)ldb, cols, e}, gr = {gate, (size_t)ldg, cols, e};
  const Rows hr = {h, (size_t)ldh, cols, se}, yr = {y, (size_t)ldy, cols, e};
  for (const Rows* out : {&hr, &yr}) {
    if (!out->p) continue;
    bool bad = rows_meet(br, *out, rows);
    bad |= gate && (ldg == 0 ? spans_meet(gate, cols * e, out->p, out->bytes(rows)) : rows_meet(gr, *out, rows));
    bad |= !(out == &hr && h == x && ldh == ldx) && rows_meet(xr, *out, rows);
    for (const float* v : params) bad |= spans_meet(v, cols * 4, out->p, out->bytes(rows));
    if (bad) return set_error(FRHIP_EINVAL, "norm_residual: an output overlaps what is read");
  }
  if (rows_meet(hr, yr, rows)) return set_error(FRHIP_EINVAL, "norm_residual: the outputs overlap");
  hipStream_t st = static_cast<hipStream_t>(s);
  if (stream_dtype == FRHIP_F16 && dtype == FRHIP_F16) return residual_run<h1, h1>(*p, rows, x, ldx, block, ldb, gate, ldg, h, ldh, y, ldy, st);
  if (stream_dtype == FRHIP_F16) return residual_run<h1, float>(*p, rows, x, ldx, block, ldb, gate, ldg, h, ldh, y, ldy, st);
  if (dtype == FRHIP_F16) return residual_run<float, h1>(*p, rows, x, ldx, block, ldb, gate, ldg, h, ldh, y, ldy, st);
  return residual_run<float, float>(*p, rows, x, ldx, block, ldb, gate, ldg, h, ldh, y, ldy, st);
}
