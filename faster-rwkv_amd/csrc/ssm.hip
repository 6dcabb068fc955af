// Operators of a selective state space layer: the short causal convolution and the scan whose decay depends on the input.
//
// The scan of a channel d with states n is linear in h,
//   h_t = a_t h_{t-1} + b_t,   a_t = exp(dt_t A[n]),   b_t = dt_t x_t B_t[n],
// and its decay over a stretch of time is exp(A[n] * (sum of dt_t)): a stretch is summed up by that sum, one number a channel, and
// by the state that it ends in from an empty one.  So a prompt is cut into chunks of time:
//   1. every chunk but a prompt's last is scanned from an empty state -> its end state and its sum of dt;
//   2. every chunk folds the chunks before it into its true start state and is scanned again, with outputs.
// One token is the formula itself.
#include <cfloat>
#include <climits>
#include <cstring>
#include <type_traits>

#include "activations.h"
#include "frhip_internal.h"
#include "groups.h"
#include "prompts.h"
#include "spans.h"

#pragma clang fp contract(off)

namespace frhip {

// ---------------------------------------------------------------------------
// Short causal convolution.  Bound by memory: every element once in and once out (4096 x 4096 binary16 out of rows of 8192: 16.8 us, 4.0
// TB/s).  A thread has 16 bytes of channels and walks a tile of rows with the last W - 1 in registers and the next four requested ahead.
// ---------------------------------------------------------------------------
template <class T>
struct ConvArgs {
  const T *x, *state;
  T *state_out, *y;
  const float *w, *bias;
  int ldx, ldy, C, silu;
  int nseq, tile;  // conv_seq: rows of a tile
  int rows;        // conv_one
};

template <class T>
constexpr int kConvLanes = kGroup<T>;  // channels of a thread
constexpr int kConvBatch = 4;               // rows that are requested together

template <class T, int W>
struct ConvTaps {
  static constexpr int V = kConvLanes<T>;
  float w[W][V], b[V];
  __device__ __forceinline__ void load(const ConvArgs<T>& a, int c, int n) {
    float t[V * W];
    load_group<float, V * W>(t, a.w + (size_t)c * W, n * W);
#pragma unroll
    for (int i = 0; i < V; i++) {
      b[i] = 0.f;
#pragma unroll
      for (int j = 0; j < W; j++) w[j][i] = t[i * W + j];
    }
    if (a.bias) load_group<float, V>(b, a.bias + c, n);
  }
  // past: the last W rows, oldest first
  __device__ __forceinline__ void apply(const float (&past)[W][V], float (&y)[V], int silu) const {
#pragma unroll
    for (int i = 0; i < V; i++) {
      float s = b[i];
#pragma unroll
      for (int j = 0; j < W; j++) s = __builtin_fmaf(w[j][i], past[j][i], s);
      y[i] = silu ? silu_f<sizeof(T) == 4>(s) : s;
    }
  }
};

// blockIdx.x: a block of channels; blockIdx.y, and so on by gridDim.y: the sequences
template <class T, int W>
__global__ __launch_bounds__(64) void conv_one_kernel(ConvArgs<T> a) {
  constexpr int V = kConvLanes<T>;
  const int c = (blockIdx.x * 64 + threadIdx.x) * V, n = a.C - c;
  if (n <= 0) return;
  ConvTaps<T, W> taps;
  taps.load(a, c, n);
  for (int row = blockIdx.y; row < a.rows; row += gridDim.y) {
    float past[W][V], y[V];
    const size_t st = (size_t)row * (W - 1) * a.C + c;
#pragma unroll
    for (int j = 0; j < W - 1; j++) load_group<T, V>(past[j], a.state + st + (size_t)j * a.C, n);
    load_group<T, V>(past[W - 1], a.x + (size_t)row * a.ldx + c, n);
    taps.apply(past, y, a.silu);
    store_group<T, V>(a.y + (size_t)row * a.ldy + c, y, n);
#pragma unroll
    for (int j = 0; j < W - 1; j++) store_group<T, V>(a.state_out + st + (size_t)j * a.C, past[j + 1], n);
  }
}

// blockIdx.x: a tile of rows of one prompt, blockIdx.y: a block of channels.  The threads of a prompt's first tile read its state and
// write the new one, so that the two may be the same memory.
template <class T, int W>
__global__ __launch_bounds__(256) void conv_seq_kernel(ConvArgs<T> a, SeqTable tab) {
  constexpr int V = kConvLanes<T>;
  const int j0 = blockIdx.x, i = find_seq(a.nseq, j0, [&](int k) { return tab.chunk[k]; });
  const int c = (blockIdx.y * blockDim.x + threadIdx.x) * V, n = a.C - c;
  if (n <= 0) return;
  const int first = tab.start[i], end = tab.start[i + 1], t0 = first + (j0 - tab.chunk[i]) * a.tile;
  const int t1 = end - t0 < a.tile ? end : t0 + a.tile;
  typedef T group __attribute__((ext_vector_type(V), aligned(sizeof(T))));
  ConvTaps<T, W> taps;
  taps.load(a, c, n);
  float past[W - 1][V];  // the rows ahead of the next one, oldest first
  const T* const x = a.x + c;
  if (t0 == first) {
    const size_t st = (size_t)i * (W - 1) * a.C + c;
#pragma unroll
    for (int j = 0; j < W - 1; j++) load_group<T, V>(past[j], a.state + st + (size_t)j * a.C, n);
    const int len = end - first;
#pragma unroll
    for (int j = 0; j < W - 1; j++) {  // the input W - 1 - j tokens ahead of the end, or what the old state holds of it
      float v[V];
      const int t = end - (W - 1) + j;
      if (t >= first) {
        load_group<T, V>(v, x + (size_t)t * a.ldx, n);
      } else {
#pragma unroll
        for (int k = 0; k < W - 1; k++)
          if (k == j + len) {
#pragma unroll
            for (int q = 0; q < V; q++) v[q] = past[k][q];
          }
      }
      store_group<T, V>(a.state_out + st + (size_t)j * a.C, v, n);
    }
  } else {  // a tile has W - 1 rows at least
#pragma unroll
    for (int j = 0; j < W - 1; j++) load_group<T, V>(past[j], x + (size_t)(t0 - (W - 1) + j) * a.ldx, n);
  }
  auto step = [&](const float (&in)[V], int t) {
    float rows[W][V], y[V];
#pragma unroll
    for (int v = 0; v < V; v++) {
#pragma unroll
      for (int j = 0; j < W - 1; j++) rows[j][v] = past[j][v];
      rows[W - 1][v] = in[v];
#pragma unroll
      for (int j = 0; j < W - 1; j++) past[j][v] = rows[j + 1][v];
    }
    taps.apply(rows, y, a.silu);
    store_group<T, V>(a.y + (size_t)t * a.ldy + c, y, n);
  };
  int t = t0;
  if (n >= V && t + kConvBatch <= t1) {
    group raw[kConvBatch];
    auto request = [&](int at) {  // rows past the tile repeat its last one
#pragma unroll
      for (int r = 0; r < kConvBatch; r++) raw[r] = *reinterpret_cast<const group*>(x + (size_t)min(at + r, t1 - 1) * a.ldx);
    };
    request(t);
    for (; t + kConvBatch <= t1; t += kConvBatch) {
      float in[kConvBatch][V];
#pragma unroll
      for (int r = 0; r < kConvBatch; r++)
#pragma unroll
        for (int v = 0; v < V; v++) in[r][v] = (float)raw[r][v];
      if (t + 2 * kConvBatch <= t1) request(t + kConvBatch);
#pragma unroll
      for (int r = 0; r < kConvBatch; r++) step(in[r], t + r);
    }
  }
  for (; t < t1; t++) {
    float in[V];
    load_group<T, V>(in, x + (size_t)t * a.ldx, n);
    step(in, t);
  }
}

// ---------------------------------------------------------------------------
// Selective scan
// ---------------------------------------------------------------------------
// A rate as exp2 takes it.  One of minus infinity stays a number: it forgets at any step but that of width zero, which keeps the state (0 times
// infinity would be a NaN).
__device__ __forceinline__ float exp2_rate(float A) {
  const float r = A * kLog2e;
  return r < -FLT_MAX ? -FLT_MAX : r;
}

template <class T>
struct SsmArgs {
  const T *x, *dt, *B, *C, *z;
  T* y;
  const float *A, *D, *dt_bias, *state;
  float* state_out;
  float *ends, *sums;  // of the chunks that are not a prompt's last: [local chunks, then prompts][N / 4][D][4], [local chunks][D]
  int ldx, lddt, ldb, ldc, ldz, ldy;
  int D_, N, cpg, softplus;  // channels, states, channels of a group
  int nblk;                  // workgroups of a group's channels
  int chunk, nlocal;         // rows of a chunk; chunks that are not a prompt's last
  int nseq, rows;            // prompts of the launch; scan of one token: rows
};

// Waves of a workgroup: NW of them share the states of 64 channels, NPL a lane, and there are four or NW in all.
constexpr int scan_waves(int nw) { return nw < 4 ? 4 : nw; }
constexpr int scan_rows(int nw) { return nw == 1 ? 8 : 16; }  // of a block of time, the rows that go through LDS together

// LOCAL: step 1 of the scan, otherwise step 2.  PAD: the waves have room for more states than there are; step 2 leaves those out, since zero times
// a step or an input that is not finite is no zero (step 1's are never read).  A workgroup walks its chunk in blocks of time.  Of a block, every wave
//   A. takes some rows to LDS: dt and dt x of a channel a lane, and B and C as fp32;
//   B. runs all of its rows with NPL states a lane in registers, and leaves its part of y in LDS;
//   C. adds the parts of the rows that it took in A, applies skip and gate and stores them.
// The step width's softplus and the gate are so evaluated once a channel and row, not once a wave, and a chunk's states are over several
// waves, which a SIMD needs to keep issuing.  4096 rows of 4096 channels x 16 states, binary16: 125 us (launched by themselves the steps take 50
// and 75), memory alone would be 26; a lane with all 16 states of a channel and one wave a SIMD took 368.  What bounds it are vector instructions: a
// state and row takes two products, two multiply-adds and an exponential (3.6 and 8.4 cycles a wave), in step 1 a multiply-add less, which is
// 70 us; softplus, gate, conversions, addresses and the sums of A and C are about half as many instructions again, and a quarter of the cycles issue none.
// Shorter chunks issue in less: 2077 rows of nine prompts of 1536 x 16 (36 us) in 0.4 of the cycles, between the fold, the first block's way to LDS and its end.
// Not kept: dt x times B as an outer product on the matrix units, 152; shorter blocks of time or five to eight workgroups a compute unit, 127 to
// 136; rows through buffer descriptors, 131.
template <class T, int NPL, int NW, bool LOCAL, bool PAD>
__global__ __launch_bounds__(scan_waves(NW) * 64, NW < 4 ? 3 : 4) void ssm_scan_kernel(SsmArgs<T> a, SeqTable tab) {
  constexpr int WAVES = scan_waves(NW), CW = WAVES / NW, NT = NPL * NW, TB = scan_rows(NW), CH = CW * 64;
  constexpr int ROWS = TB * CW / WAVES;                                  // rows of a wave in A and C: of its 64 channels
  constexpr int STAGE = (TB * 2 * NT + WAVES * 64 - 1) / (WAVES * 64);  // elements of B and C of a thread
  static_assert(ROWS * NW == TB, "every row has its wave");
  constexpr int UNROLL = NPL == 4 ? 4 : 2;  // rows in B; 8 and 16 of four states took 1 and 8 % longer, 4 of eight spilled
  constexpr bool FINE = sizeof(T) == 4;
  constexpr int BUFS = LOCAL ? 2 : 1;  // LOCAL takes the next block's rows while waves still scan this one
  __shared__ __attribute__((aligned(16))) float bc[BUFS][TB][2][NT];
  __shared__ float2 du[BUFS][TB][CH];
  __shared__ float part[LOCAL || NW == 1 ? 1 : NW][TB][CH];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), cw = wave / NW, nw = wave % NW;
  const int j0 = blockIdx.y;
  const int i = LOCAL ? find_seq(a.nseq, j0, [&](int k) { return tab.chunk[k] - k; })
                      : find_seq(a.nseq, j0, [&](int k) { return tab.chunk[k]; });
  const int nchunk = tab.chunk[i + 1] - tab.chunk[i], ci = j0 - tab.chunk[i] + (LOCAL ? i : 0), local0 = tab.chunk[i] - i;
  const int end = tab.start[i + 1], t0 = tab.start[i] + ci * a.chunk, t1 = end - t0 < a.chunk ? end : t0 + a.chunk;
  const int g = blockIdx.x / a.nblk, at = cw * 64 + lane, cg = (blockIdx.x - g * a.nblk) * CH + at;
  const bool mine = cg < a.cpg;
  const int d = g * a.cpg + (mine ? cg : a.cpg - 1), n0 = nw * NPL;

  const float bias = a.dt_bias ? a.dt_bias[d] : 0.f, skip = !LOCAL && a.D ? a.D[d] : 0.f;
  const unsigned at_row = (unsigned)d * sizeof(T);  // of x, dt, z and y: rows are uniform addresses, a lane adds this
  auto in_row = [&](const T* rows, int ld, int row) {
    unsigned lane_part = at_row;
    asm("" : "+v"(lane_part));  // or the compiler adds it to the base ahead of the loop, and the row's 64 bits to a vector here
    return *reinterpret_cast<const T*>(reinterpret_cast<const char*>(rows + (size_t)row * ld) + lane_part);
  };
  const T* const zp = a.z ? a.z : a.x;  // without a gate some row that is there, for nothing
  const int ldz = a.z ? a.ldz : a.ldx;
  float sum = 0.f;
  T xr[ROWS], dr[ROWS], zr[ROWS], st[STAGE];
  // B and C of a block: element e = (row, which, state), a thread takes every WAVES x 64th
  const T* bcp[STAGE];
  int bcrow[STAGE];
  unsigned bcld[STAGE];
#pragma unroll
  for (int q = 0; q < STAGE; q++) {
    const int e = threadIdx.x + q * (WAVES * 64), r = e / (2 * NT), c = (e / NT) & 1, n = e % NT;
    bcrow[q] = e < TB * 2 * NT && n < a.N ? r : INT_MAX;
    bcld[q] = c ? a.ldc : a.ldb;
    bcp[q] = (c ? a.C : a.B) + (size_t)g * a.N + (n < a.N ? n : 0);
  }
  auto request = [&](int t) {  // of the block that begins at row t; rows past the chunk repeat its last one
#pragma unroll
    for (int r = 0; r < ROWS; r++) {
      const int row = min(t + nw * ROWS + r, t1 - 1);
      xr[r] = in_row(a.x, a.ldx, row);
      dr[r] = in_row(a.dt, a.lddt, row);
      if constexpr (!LOCAL) zr[r] = in_row(zp, ldz, row);
    }
#pragma unroll
    for (int q = 0; q < STAGE; q++) st[q] = bcp[q][(size_t)(unsigned)(t + min(bcrow[q], t1 - 1 - t)) * bcld[q]];
  };
  if (t0 < t1) request(t0);  // on its way while the state is found

  float A2[NPL], h[NPL];
#pragma unroll
  for (int k = 0; k < NPL; k += 4) {
    float v[4];
    load_group<float, 4>(v, a.A + (size_t)d * a.N + n0 + k, a.N - n0 - k);
#pragma unroll
    for (int e = 0; e < 4; e++) {
      A2[k + e] = exp2_rate(v[e]);  // rows past the chunk have a step of zero
      h[k + e] = 0.f;
    }
  }
  // a chunk's end state in the workspace: [N / 4, rounded up][D][4], 16 bytes a lane and access
  const int quads = (a.N + 3) / 4;
  const size_t slot = (size_t)quads * a.D_ * 4;
  auto quad = [&](size_t chunk, int k) { return reinterpret_cast<f32x4*>(a.ends + chunk * slot + ((size_t)(n0 + k) * a.D_ + (size_t)d * 4)); };
  const size_t start = (size_t)a.nlocal + local0;  // the prompt's state ahead, of prompts of several chunks
  const float* const state = a.state + ((size_t)i * a.D_ + d) * a.N + n0;
  if constexpr (LOCAL) {
    if (ci == 0 && mine) {  // step 2 reads it here: its last chunk may overwrite the state
#pragma unroll
      for (int k = 0; k < NPL; k += 4)
        if (n0 + k < a.N) {
          float v[4];
          load_group<float, 4>(v, state + k, a.N - n0 - k);
          *quad(start, k) = (f32x4){v[0], v[1], v[2], v[3]};
        }
    }
  } else if (nchunk == 1) {
#pragma unroll
    for (int k = 0; k < NPL; k += 4) {
      float v[4];
      load_group<float, 4>(v, state + k, a.N - n0 - k);
#pragma unroll
      for (int e = 0; e < 4; e++) h[k + e] = v[e];
    }
  } else {
    const float* const sums = a.sums + (size_t)local0 * a.D_ + d;
    constexpr int AHEAD = NPL == 4 ? 8 : NPL == 8 ? 4 : 2;  // chunks that are requested together
#pragma unroll
    for (int k = 0; k < NPL; k += 4)
      if (n0 + k < a.N) {
        const f32x4 v = *quad(start, k);
#pragma unroll
        for (int e = 0; e < 4; e++) h[k + e] = v[e];
      }
    for (int p0 = 0; p0 < ci; p0 += AHEAD) {
      float sum[AHEAD];
      f32x4 v[AHEAD][NPL / 4];
#pragma unroll
      for (int p = 0; p < AHEAD; p++) {
        const int c = min(p0 + p, ci - 1);
        sum[p] = sums[(size_t)c * a.D_];
#pragma unroll
        for (int k = 0; k < NPL; k += 4) v[p][k / 4] = *quad(local0 + c, n0 + k < a.N ? k : -n0);
      }
#pragma unroll
      for (int p = 0; p < AHEAD; p++)
        if (p0 + p < ci) {
#pragma unroll
          for (int k = 0; k < NPL; k++) h[k] = __builtin_fmaf(__builtin_amdgcn_exp2f(sum[p] * A2[k]), h[k], v[p][k / 4][k % 4]);
        }
    }
#pragma unroll
    for (int k = 0; k < NPL; k++) h[k] = n0 + k < a.N ? h[k] : 0.f;
  }

  float x[ROWS], z[ROWS];  // of the block that is scanned
  auto take = [&](int t, int buf, float (&xn)[ROWS], float (&zn)[ROWS]) {
    float dt[ROWS];
#pragma unroll
    for (int r = 0; r < ROWS; r++) dt[r] = (float)dr[r] + bias;
    if (a.softplus) {
#pragma unroll
      for (int r = 0; r < ROWS; r++) dt[r] = softplus_f<FINE>(dt[r]);
    }
    if (t + TB > t1) {  // rows past the chunk: no step, no input
#pragma unroll
      for (int r = 0; r < ROWS; r++)
        if (t + nw * ROWS + r >= t1) dt[r] = 0.f, xr[r] = (T)0.f;
    }
#pragma unroll
    for (int r = 0; r < ROWS; r++) {
      xn[r] = (float)xr[r];
      if constexpr (!LOCAL) zn[r] = (float)zr[r];
      du[buf][nw * ROWS + r][at] = make_float2(dt[r], dt[r] * xn[r]);
      if constexpr (LOCAL) sum += dt[r];
    }
#pragma unroll
    for (int q = 0; q < STAGE; q++) {
      const int e = threadIdx.x + q * (WAVES * 64);
      if (TB * 2 * NT % (WAVES * 64) == 0 || e < TB * 2 * NT) (&bc[buf][0][0][0])[e] = bcrow[q] < t1 - t ? (float)st[q] : 0.f;
    }
  };
  if (t0 < t1) {
    take(t0, 0, x, z);
    if (t0 + TB < t1) request(t0 + TB);
  }
  int buf = 0;
  for (int t = t0; t < t1; t += TB, buf ^= BUFS - 1) {
    __syncthreads();
    auto scan = [&](auto whole) {  // whole: all of the wave's states are there
#pragma unroll UNROLL
      for (int r = 0; r < TB; r++) {
        const float2 v = du[buf][r][at];
        float y = 0.f;
#pragma unroll
        for (int k = 0; k < NPL; k++) {
          if (!decltype(whole)::value && n0 + k >= a.N) break;
          const float decay = __builtin_amdgcn_exp2f(v.x * A2[k]);
          h[k] = __builtin_fmaf(decay, h[k], v.y * bc[buf][r][0][n0 + k]);
          if constexpr (!LOCAL) y = k ? __builtin_fmaf(bc[buf][r][1][n0 + k], h[k], y) : bc[buf][r][1][n0] * h[0];
        }
        if constexpr (!LOCAL) part[NW == 1 ? 0 : nw][r][at] = y;
      }
    };
    if (PAD && n0 + NPL > a.N) scan(std::false_type());
    else scan(std::true_type());
    if constexpr (!LOCAL) {
      __syncthreads();
#pragma unroll
      for (int r = 0; r < ROWS; r++) {
        const int row = nw * ROWS + r;
        float y = part[0][row][at];
#pragma unroll
        for (int w = 1; w < NW; w++) y += part[w][row][at];
        y = __builtin_fmaf(skip, x[r], y);
        if (a.z) y *= silu_f<FINE>(z[r]);
        if (mine && t + row < t1) *reinterpret_cast<T*>(reinterpret_cast<char*>(a.y + (size_t)(t + row) * a.ldy) + at_row) = (T)y;
      }
    }
    if (t + TB < t1) {
      take(t + TB, buf ^ (BUFS - 1), x, z);
      if (t + 2 * TB < t1) request(t + 2 * TB);
    }
  }
  if constexpr (LOCAL) {  // the waves' sums of dt, in wave order
    __shared__ float total[NW][CH];
    total[nw][at] = sum;
    __syncthreads();
    if (nw == 0 && mine) {
#pragma unroll
      for (int w = 1; w < NW; w++) sum += total[w][at];
      a.sums[(size_t)j0 * a.D_ + d] = sum;
    }
  }
  if (!mine) return;
  if constexpr (LOCAL) {
#pragma unroll
    for (int k = 0; k < NPL; k += 4)
      if (n0 + k < a.N) *quad(j0, k) = (f32x4){h[k], h[k + 1], h[k + 2], h[k + 3]};
  } else if (ci == nchunk - 1) {
#pragma unroll
    for (int k = 0; k < NPL; k += 4) {
      const float v[4] = {h[k], h[k + 1], h[k + 2], h[k + 3]};
      store_group<float, 4>(a.state_out + ((size_t)i * a.D_ + d) * a.N + n0 + k, v, a.N - n0 - k);
    }
  }
}

// One token each of a.rows sequences.  Bound by memory: the states once in and once out.  LANES lanes share a channel, four states each;
// a thread takes R sequences (blockIdx.y, and so on by gridDim.y), whose loads go out together, and holds A for all.  VEC: the states are
// a multiple of four.
template <class T, int LANES, int R, bool VEC>
__global__ __launch_bounds__(256) void ssm_one_kernel(SsmArgs<T> a) {
  typedef T t4 __attribute__((ext_vector_type(4), aligned(sizeof(T))));
  typedef float f4 __attribute__((ext_vector_type(4), aligned(4)));
  constexpr bool FINE = sizeof(T) == 4;
  const int q = threadIdx.x % LANES, n0 = q * 4, d = blockIdx.x * (256 / LANES) + threadIdx.x / LANES;
  if (d >= a.D_) return;  // lanes of a channel leave together
  const int gn = d / a.cpg * a.N + n0, left = a.N - n0;
  auto four = [&](const auto* p) {
    f4 v;
    if constexpr (VEC) {
      if (left > 0) {
        if constexpr (sizeof(*p) == 2) {
          const t4 t = *reinterpret_cast<const t4*>(p);
#pragma unroll
          for (int k = 0; k < 4; k++) v[k] = (float)t[k];
        } else {
          v = *reinterpret_cast<const f4*>(p);
        }
      } else {
        v = (f4){0.f, 0.f, 0.f, 0.f};
      }
    } else {
#pragma unroll
      for (int k = 0; k < 4; k++) v[k] = k < left ? (float)p[k] : 0.f;
    }
    return v;
  };
  f4 A2 = four(a.A + (size_t)d * a.N + n0);
#pragma unroll
  for (int k = 0; k < 4; k++) A2[k] = exp2_rate(A2[k]);
  const float bias = a.dt_bias ? a.dt_bias[d] : 0.f, skip = a.D ? a.D[d] : 0.f;
  for (int r0 = blockIdx.y * R; r0 < a.rows; r0 += gridDim.y * R) {
    f4 h[R], B[R], C[R];
    float dt[R], x[R], z[R];
#pragma unroll
    for (int r = 0; r < R; r++) {
      const int row = min(r0 + r, a.rows - 1);
      h[r] = four(a.state + ((size_t)row * a.D_ + d) * a.N + n0);
      dt[r] = (float)a.dt[(size_t)row * a.lddt + d];
      x[r] = (float)a.x[(size_t)row * a.ldx + d];
      B[r] = four(a.B + (size_t)row * a.ldb + gn);
      C[r] = four(a.C + (size_t)row * a.ldc + gn);
      z[r] = a.z ? (float)a.z[(size_t)row * a.ldz + d] : 0.f;
    }
#pragma unroll
    for (int r = 0; r < R; r++) {
      if (R > 1 && r0 + r >= a.rows) break;
      const float v = dt[r] + bias, step = a.softplus ? softplus_f<FINE>(v) : v, u = step * x[r];
      float y = 0.f;
#pragma unroll
      for (int k = 0; k < 4; k++) {
        h[r][k] = __builtin_fmaf(__builtin_amdgcn_exp2f(step * A2[k]), h[r][k], u * B[r][k]);
        y = VEC || k < left ? __builtin_fmaf(C[r][k], h[r][k], y) : y;
      }
      if (VEC && left <= 0) y = 0.f;  // lanes without a state: not what 0 times a step that is not finite would leave
      float* const out = a.state_out + ((size_t)(r0 + r) * a.D_ + d) * a.N + n0;
      if constexpr (VEC) {
        if (left > 0) *reinterpret_cast<f4*>(out) = h[r];
      } else {
#pragma unroll
        for (int k = 0; k < 4; k++)
          if (k < left) out[k] = h[r][k];
      }
#pragma unroll
      for (int m = 1; m < LANES; m *= 2) y += __shfl_xor(y, m);
      if (q == 0) {
        y = __builtin_fmaf(skip, x[r], y);
        a.y[(size_t)(r0 + r) * a.ldy + d] = (T)(a.z ? y * silu_f<FINE>(z[r]) : y);
      }
    }
  }
}

// ---------------------------------------------------------------------------
// Host side
// ---------------------------------------------------------------------------
struct ScanShape {
  int npl, nw, nblk, wgs;  // states of a wave, waves that share a channel's states, workgroups of a group, workgroups of a chunk
};
static ScanShape scan_shape(const frhip_ssm& p) {
  ScanShape s;
  s.npl = p.states <= 16 ? 4 : p.states <= 64 ? 8 : 16;
  s.nw = 1;
  while (s.nw * s.npl < p.states) s.nw *= 2;
  const int per = 64 * (scan_waves(s.nw) / s.nw), cpg = p.channels / p.groups;
  s.nblk = (cpg + per - 1) / per;
  s.wgs = p.groups * s.nblk;
  return s;
}

constexpr int kScanLeast = 16;         // rows of a chunk, at least
constexpr int kScanMostUnits = 1024;   // workgroups of all chunks, at most about: what the workspace is sized for
constexpr int kScanRows = 16;          // a chunk is a multiple of it
constexpr int kScanWhole = 32;         // prompts of up to so many rows are not cut

// Rows of a chunk: enough chunks for four workgroups a compute unit (4096 rows of 4096 channels x 16 states, with two, three, four: 165, 142,
// 130 us, six and eight in shorter blocks 136 and 127; 830 rows of 1280 x 64, workgroups of eight waves, with two, four: 46, 41).  A compute unit holds four of the forms with
// four waves, but of step 2 of those with eight and sixteen (33 states and more) two and one: what is over runs in further rounds (1280 x 64: 540 workgroups of
// step 2 over 512 places; 1024 rows of 2560 x 128, 880 over 512: 146 us; 4096 of 1280 x 256, 860 over 256: 638).
// Where no prompt has more than kScanWhole rows the first launch costs more than it shares out (1536 channels x 16 states, in chunks of 16 and
// whole: 17 rows 8.8 and 7.0 us, 32 rows 8.9 and 7.0, 48 rows 8.9 and 9.1; x 64 states: 13.6 and 10.6, 13.6 and 10.7, 13.9 and 14.7).
static int scan_chunk(const ScanShape& s, int nseq, const int32_t* start, int cus) {
  const int T = start[nseq] - start[0];
  int longest = 0;
  for (int i = 0; i < nseq; i++)
    if (start[i + 1] - start[i] > longest) longest = start[i + 1] - start[i];
  const int units = cus < kScanMostUnits / 4 ? cus * 4 : kScanMostUnits;
  const int q = units / s.wgs > 1 ? units / s.wgs : 1;
  int len = T / q + (T % q ? 1 : 0);
  if (len < kScanLeast) len = kScanLeast;
  if (longest <= kScanWhole && len < longest) len = longest;
  return len > INT_MAX - kScanRows ? INT_MAX : (len + kScanRows - 1) / kScanRows * kScanRows;
}

static size_t scan_most_local(const ScanShape& s, int T) {  // sum of (chunks - 1) <= T / chunk <= both
  const size_t by_rows = (size_t)T / kScanLeast, by_units = (size_t)(kScanMostUnits / s.wgs > 1 ? kScanMostUnits / s.wgs : 1);
  return by_rows < by_units ? by_rows : by_units;
}

template <class T>
static int conv_one_run(const ConvArgs<T>& a, int W, hipStream_t st) {
  const int lanes = (a.C - 1) / kConvLanes<T> + 1;
  const dim3 grid((lanes + 63) / 64, a.rows < 65535 ? a.rows : 65535);
  if (W == 2) hipLaunchKernelGGL((conv_one_kernel<T, 2>), grid, dim3(64), 0, st, a);
  else if (W == 3) hipLaunchKernelGGL((conv_one_kernel<T, 3>), grid, dim3(64), 0, st, a);
  else hipLaunchKernelGGL((conv_one_kernel<T, 4>), grid, dim3(64), 0, st, a);
  return check_launch("conv_one");
}

template <class T>
static int conv_seq_run(ConvArgs<T> a, int W, int nseq, const int32_t* start, hipStream_t st) {
  constexpr int V = kConvLanes<T>;
  const int ncv = (a.C - 1) / V + 1, blocks = (ncv + 255) / 256, threads = ((ncv + blocks - 1) / blocks + 63) / 64 * 64;
  // A tile reads W - 1 rows more than its own, which costs where memory is busy; a short one starts sooner.  us with tiles of 4 and 8 rows:
  // 300 x 2048 4.9 and 5.5, 2077 x 1536 of fp32 8.0 and 8.7, 1000 x 4096 8.0 and 7.5, 4096 x 4096 19.6 and 16.8
  a.tile = (size_t)(start[nseq] - start[0]) * a.C < (size_t)4000000 ? kConvBatch : 2 * kConvBatch;
  const T *state = a.state;
  T* state_out = a.state_out;
  for (int s0 = 0; s0 < nseq; s0 += kSeqTable) {
    SeqTable tab;
    a.nseq = nseq - s0 < kSeqTable ? nseq - s0 : kSeqTable;
    int tiles = 0;
    for (int i = 0; i < a.nseq; i++) {
      const int len = start[s0 + i + 1] - start[s0 + i];
      tab.start[i] = start[s0 + i];
      tab.chunk[i] = tiles;
      tiles += len ? (len - 1) / a.tile + 1 : 1;
    }
    tab.start[a.nseq] = start[s0 + a.nseq];
    tab.chunk[a.nseq] = tiles;
    a.state = state + (size_t)s0 * (W - 1) * a.C;
    a.state_out = state_out + (size_t)s0 * (W - 1) * a.C;
    const dim3 grid(tiles, blocks);
    if (W == 2) hipLaunchKernelGGL((conv_seq_kernel<T, 2>), grid, dim3(threads), 0, st, a, tab);
    else if (W == 3) hipLaunchKernelGGL((conv_seq_kernel<T, 3>), grid, dim3(threads), 0, st, a, tab);
    else hipLaunchKernelGGL((conv_seq_kernel<T, 4>), grid, dim3(threads), 0, st, a, tab);
    if (int rc = check_launch("conv_seq")) return rc;
  }
  return 0;
}

// What frhip_conv_one and frhip_conv_seq check alike; row0, rows: the rows of x and y, nstate: sequences
static int conv_check(int C, int W, const void* x, int ldx, const float* w, const float* bias, int act, const void* state, void* state_out,
                      void* y, int ldy, int dtype, size_t row0, size_t rows, size_t nstate) {
  if (dtype != FRHIP_F16 && dtype != FRHIP_F32) return set_error(FRHIP_EINVAL, "conv: dtype must be F16 or F32");
  if (act != FRHIP_ACT_NONE && act != FRHIP_ACT_SILU) return set_error(FRHIP_EINVAL, "conv: act must be NONE or SILU");
  if (C <= 0 || C > kMostChannels || W < 2 || W > 4) return set_error(FRHIP_ESHAPE, "conv: W must be 2, 3 or 4 and C 1 to 2^24");
  if (ldx < C || ldy < C) return set_error(FRHIP_ESHAPE, "conv: rows closer than C elements");
  if (!w || !state || !state_out || (rows && (!x || !y))) return set_error(FRHIP_EINVAL, "conv: null pointer");
  const size_t elem = dtype == FRHIP_F16 ? 2 : 4, sbytes = nstate * (W - 1) * C * elem;
  if (off_grid(elem, {x, y, state, state_out}) || off_grid(4, {w, bias})) return set_error(FRHIP_EINVAL, "conv: pointer not aligned to its element");
  const char* xr = static_cast<const char*>(x) + row0 * ldx * elem;
  char* yr = static_cast<char*>(y) + row0 * ldy * elem;
  const size_t se = sbytes / elem;
  if (rows && (rows_overlap(xr, ldx, yr, ldy, rows, C, C, elem) || rows_overlap(yr, (rows - 1) * ldy + C, state, se, 1, (rows - 1) * ldy + C, se, elem) ||
               rows_overlap(yr, (rows - 1) * ldy + C, state_out, se, 1, (rows - 1) * ldy + C, se, elem) ||
               rows_overlap(xr, (rows - 1) * ldx + C, state_out, se, 1, (rows - 1) * ldx + C, se, elem)))
    return set_error(FRHIP_EINVAL, "conv: an output overlaps what is read");
  const size_t ye = rows ? ((rows - 1) * ldy + C) * elem : 0;
  for (const void* out : {static_cast<const void*>(yr), static_cast<const void*>(state_out)}) {
    const size_t bytes = out == yr ? ye : sbytes;
    if (spans_meet(out, bytes, w, (size_t)C * W * 4) || spans_meet(out, bytes, bias, (size_t)C * 4))
      return set_error(FRHIP_EINVAL, "conv: an output overlaps a parameter");
  }
  if (spans_clash(state, state_out, sbytes)) return set_error(FRHIP_EINVAL, "conv: states overlap in part");
  return 0;
}

template <class T>
static ConvArgs<T> conv_args(int C, const void* x, int ldx, const float* w, const float* bias, int act, const void* state, void* state_out,
                             void* y, int ldy) {
  ConvArgs<T> a;
  memset(&a, 0, sizeof(a));
  a.x = static_cast<const T*>(x);
  a.state = static_cast<const T*>(state);
  a.state_out = static_cast<T*>(state_out);
  a.y = static_cast<T*>(y);
  a.w = w;
  a.bias = bias;
  a.ldx = ldx;
  a.ldy = ldy;
  a.C = C;
  a.silu = act == FRHIP_ACT_SILU;
  return a;
}

static int ssm_check_params(const frhip_ssm* p) {
  if (!p || !p->A) return set_error(FRHIP_EINVAL, "ssm: null pointer");
  if (p->channels <= 0 || p->groups <= 0 || p->channels % p->groups != 0 || p->channels > kMostChannels)
    return set_error(FRHIP_ESHAPE, "ssm: channels must be a multiple of groups, at most 2^24");
  if (p->states < 1 || p->states > 256) return set_error(FRHIP_ESHAPE, "ssm: states must be 1 to 256");
  if ((long long)p->groups * p->states > INT_MAX) return set_error(FRHIP_ESHAPE, "ssm: too many groups");
  if (off_grid(4, {p->A, p->D, p->dt_bias})) return set_error(FRHIP_EINVAL, "ssm: pointer not aligned to its element");
  return 0;
}

struct SsmCall {
  const void *x, *dt, *B, *C, *z;
  int ldx, lddt, ldb, ldc, ldz;
  const float* state;
  float* state_out;
  void* y;
  int ldy, dtype;
};

static int ssm_check(const frhip_ssm& p, const SsmCall& c, size_t row0, size_t rows, size_t nstate) {
  if (c.dtype != FRHIP_F16 && c.dtype != FRHIP_F32) return set_error(FRHIP_EINVAL, "ssm: dtype must be F16 or F32");
  const int bn = p.groups * p.states;
  if (c.ldx < p.channels || c.lddt < p.channels || c.ldy < p.channels || (c.z && c.ldz < p.channels) || c.ldb < bn || c.ldc < bn)
    return set_error(FRHIP_ESHAPE, "ssm: rows closer than their elements");
  if (!c.state || !c.state_out || (rows && (!c.x || !c.dt || !c.B || !c.C || !c.y))) return set_error(FRHIP_EINVAL, "ssm: null pointer");
  const size_t elem = c.dtype == FRHIP_F16 ? 2 : 4, sn = nstate * p.channels * p.states;
  if (off_grid(elem, {c.x, c.dt, c.B, c.C, c.z, c.y}) || off_grid(4, {c.state, c.state_out}))
    return set_error(FRHIP_EINVAL, "ssm: pointer not aligned to its element");
  if (spans_clash(c.state, c.state_out, sn * 4)) return set_error(FRHIP_EINVAL, "ssm: states overlap in part");
  const size_t dn = (size_t)p.channels * 4;
  auto meets_parameter = [&](const void* out, size_t bytes) {
    return spans_meet(out, bytes, p.A, dn * p.states) || spans_meet(out, bytes, p.D, dn) || spans_meet(out, bytes, p.dt_bias, dn);
  };
  if (meets_parameter(c.state_out, sn * 4)) return set_error(FRHIP_EINVAL, "ssm: an output overlaps a parameter");
  if (!rows) return 0;
  struct In { const void* p; int ld, cols; };
  const char* y = static_cast<const char*>(c.y) + row0 * c.ldy * elem;
  const size_t ye = (rows - 1) * c.ldy + p.channels;
  if (meets_parameter(y, ye * elem)) return set_error(FRHIP_EINVAL, "ssm: an output overlaps a parameter");
  for (const In& in : {In{c.x, c.ldx, p.channels}, In{c.dt, c.lddt, p.channels}, In{c.B, c.ldb, bn}, In{c.C, c.ldc, bn}, In{c.z, c.ldz, p.channels}}) {
    if (!in.p) continue;
    const char* q = static_cast<const char*>(in.p) + row0 * in.ld * elem;
    const size_t qe = ((rows - 1) * in.ld + in.cols) * elem;
    if (rows_overlap(q, in.ld, y, c.ldy, rows, in.cols, p.channels, elem) || rows_overlap(q, qe, c.state_out, sn * 4, 1, qe, sn * 4, 1))
      return set_error(FRHIP_EINVAL, "ssm: an output overlaps what is read");
  }
  if (rows_overlap(y, ye * elem, c.state, sn * 4, 1, ye * elem, sn * 4, 1) || rows_overlap(y, ye * elem, c.state_out, sn * 4, 1, ye * elem, sn * 4, 1))
    return set_error(FRHIP_EINVAL, "ssm: an output overlaps what is read");
  return 0;
}

template <class T>
static SsmArgs<T> ssm_args(const frhip_ssm& p, const SsmCall& c) {
  SsmArgs<T> a;
  memset(&a, 0, sizeof(a));
  a.x = static_cast<const T*>(c.x);
  a.dt = static_cast<const T*>(c.dt);
  a.B = static_cast<const T*>(c.B);
  a.C = static_cast<const T*>(c.C);
  a.z = static_cast<const T*>(c.z);
  a.y = static_cast<T*>(c.y);
  a.A = p.A;
  a.D = p.D;
  a.dt_bias = p.dt_bias;
  a.state = c.state;
  a.state_out = c.state_out;
  a.ldx = c.ldx;
  a.lddt = c.lddt;
  a.ldb = c.ldb;
  a.ldc = c.ldc;
  a.ldz = c.ldz;
  a.ldy = c.ldy;
  a.D_ = p.channels;
  a.N = p.states;
  a.cpg = p.channels / p.groups;
  a.softplus = p.dt_softplus != 0;
  return a;
}

template <class T, int NPL, int NW>
static int scan_launch(const SsmArgs<T>& a, const SeqTable& tab, int wgs, int chunks, hipStream_t st) {
  constexpr int threads = scan_waves(NW) * 64;
  if (a.nlocal) {
    hipLaunchKernelGGL((ssm_scan_kernel<T, NPL, NW, true, false>), dim3(wgs, a.nlocal), dim3(threads), 0, st, a, tab);
    if (int rc = check_launch("ssm_seq")) return rc;
  }
  if (a.N == NPL * NW) hipLaunchKernelGGL((ssm_scan_kernel<T, NPL, NW, false, false>), dim3(wgs, chunks), dim3(threads), 0, st, a, tab);
  else hipLaunchKernelGGL((ssm_scan_kernel<T, NPL, NW, false, true>), dim3(wgs, chunks), dim3(threads), 0, st, a, tab);
  return check_launch("ssm_seq");
}

// Prompts s0 .. s0 + a.nseq - 1 in one table; returns the chunks
static int scan_table(SeqTable& tab, const int32_t* start, int s0, int n, int chunk) {
  int chunks = 0;
  for (int i = 0; i < n; i++) {
    const int len = start[s0 + i + 1] - start[s0 + i];
    tab.start[i] = start[s0 + i];
    tab.chunk[i] = chunks;
    chunks += len ? (len - 1) / chunk + 1 : 1;
  }
  tab.start[n] = start[s0 + n];
  tab.chunk[n] = chunks;
  return chunks;
}

template <class T>
static int ssm_seq_run(const frhip_ssm& p, const SsmCall& c, int nseq, const int32_t* start, void* workspace, hipStream_t st) {
  const ScanShape s = scan_shape(p);
  SsmArgs<T> a = ssm_args<T>(p, c);
  const int rows = start[nseq] - start[0];
  a.nblk = s.nblk;
  const size_t per = (size_t)p.channels * p.states;
  for (int s0 = 0; s0 < nseq; s0 += kSeqTable) {
    SeqTable tab;
    a.nseq = nseq - s0 < kSeqTable ? nseq - s0 : kSeqTable;
    a.chunk = scan_chunk(s, a.nseq, start + s0, compute_units());
    const int chunks = scan_table(tab, start, s0, a.nseq, a.chunk);
    a.nlocal = chunks - a.nseq;
    if ((size_t)a.nlocal > scan_most_local(s, rows)) return set_error(FRHIP_ESTATE, "ssm_seq: more chunks than the workspace holds");
    a.state = c.state + (size_t)s0 * per;
    a.state_out = c.state_out + (size_t)s0 * per;
    a.ends = static_cast<float*>(workspace);
    a.sums = a.ends + 2 * (size_t)a.nlocal * p.channels * ((p.states + 3) / 4 * 4);
    int rc = FRHIP_ESHAPE;
    if (s.npl == 4 && s.nw == 1) rc = scan_launch<T, 4, 1>(a, tab, s.wgs, chunks, st);
    else if (s.npl == 4 && s.nw == 2) rc = scan_launch<T, 4, 2>(a, tab, s.wgs, chunks, st);
    else if (s.npl == 4) rc = scan_launch<T, 4, 4>(a, tab, s.wgs, chunks, st);
    else if (s.npl == 8 && s.nw == 4) rc = scan_launch<T, 8, 4>(a, tab, s.wgs, chunks, st);
    else if (s.npl == 8) rc = scan_launch<T, 8, 8>(a, tab, s.wgs, chunks, st);
    else if (s.nw == 8) rc = scan_launch<T, 16, 8>(a, tab, s.wgs, chunks, st);
    else rc = scan_launch<T, 16, 16>(a, tab, s.wgs, chunks, st);
    if (rc) return rc;
  }
  return 0;
}

template <class T, int LANES, int R>
static void one_launch(const SsmArgs<T>& a, int groups, hipStream_t st) {
  const dim3 grid((a.D_ - 1) / (256 / LANES) + 1, groups < 65535 ? groups : 65535);
  if (a.N % 4 == 0) hipLaunchKernelGGL((ssm_one_kernel<T, LANES, R, true>), grid, dim3(256), 0, st, a);
  else hipLaunchKernelGGL((ssm_one_kernel<T, LANES, R, false>), grid, dim3(256), 0, st, a);
}

template <class T, int LANES>
static void one_rows(const SsmArgs<T>& a, hipStream_t st) {
  // four sequences a thread from where that still leaves every SIMD several waves
  const size_t waves = ((size_t)a.D_ * LANES + 63) / 64 * ((a.rows - 1) / 4 + 1);
  if (waves >= (size_t)compute_units() * 8) one_launch<T, LANES, 4>(a, (a.rows - 1) / 4 + 1, st);
  else one_launch<T, LANES, 1>(a, a.rows, st);
}

template <class T>
static int ssm_one_run(const frhip_ssm& p, const SsmCall& c, int rows, hipStream_t st) {
  SsmArgs<T> a = ssm_args<T>(p, c);
  a.rows = rows;
  int lanes = 1;
  while (lanes * 4 < p.states) lanes *= 2;
  switch (lanes) {
    case 1: one_rows<T, 1>(a, st); break;
    case 2: one_rows<T, 2>(a, st); break;
    case 4: one_rows<T, 4>(a, st); break;
    case 8: one_rows<T, 8>(a, st); break;
    case 16: one_rows<T, 16>(a, st); break;
    case 32: one_rows<T, 32>(a, st); break;
    default: one_rows<T, 64>(a, st); break;
  }
  return check_launch("ssm_one");
}

}  // namespace frhip

using namespace frhip;

extern "C" int frhip_conv_one(int rows, int C, int W, const void* x, int ldx, const float* w, const float* bias, int act, const void* state,
                              void* state_out, void* y, int ldy, int dtype, frhip_stream s) {
  if (rows < 0 || rows > kMostRows) return set_error(FRHIP_ESHAPE, "conv_one: rows must be 0 to 2^30");
  if (int rc = conv_check(C, W, x, ldx, w, bias, act, state, state_out, y, ldy, dtype, 0, rows, rows)) return rc;
  if (rows == 0) return 0;
  hipStream_t st = static_cast<hipStream_t>(s);
  if (dtype == FRHIP_F16) {
    auto a = conv_args<h1>(C, x, ldx, w, bias, act, state, state_out, y, ldy);
    a.rows = rows;
    return conv_one_run(a, W, st);
  }
  auto a = conv_args<float>(C, x, ldx, w, bias, act, state, state_out, y, ldy);
  a.rows = rows;
  return conv_one_run(a, W, st);
}

extern "C" int frhip_conv_seq(int nseq, const int32_t* seq_start, int C, int W, const void* x, int ldx, const float* w, const float* bias,
                              int act, const void* state, void* state_out, void* y, int ldy, int dtype, frhip_stream s) {
  if (int rc = check_seqs(nseq, seq_start, kMostTime, "conv_seq: seq_start must be nseq + 1 row numbers up to 2^28 that do not descend")) return rc;
  const size_t row0 = nseq ? seq_start[0] : 0, rows = nseq ? seq_start[nseq] - seq_start[0] : 0;
  if (int rc = conv_check(C, W, x, ldx, w, bias, act, state, state_out, y, ldy, dtype, row0, rows, nseq)) return rc;
  if (nseq == 0) return 0;
  hipStream_t st = static_cast<hipStream_t>(s);
  if (dtype == FRHIP_F16) return conv_seq_run(conv_args<h1>(C, x, ldx, w, bias, act, state, state_out, y, ldy), W, nseq, seq_start, st);
  return conv_seq_run(conv_args<float>(C, x, ldx, w, bias, act, state, state_out, y, ldy), W, nseq, seq_start, st);
}

extern "C" int frhip_ssm_one(const frhip_ssm* p, int rows, const void* x, int ldx, const void* dt, int lddt, const void* B, int ldb,
                             const void* C, int ldc, const void* z, int ldz, const float* state, float* state_out, void* y, int ldy,
                             int dtype, frhip_stream s) {
  if (int rc = ssm_check_params(p)) return rc;
  if (rows < 0 || rows > kMostRows) return set_error(FRHIP_ESHAPE, "ssm_one: rows must be 0 to 2^30");
  const SsmCall c = {x, dt, B, C, z, ldx, lddt, ldb, ldc, ldz, state, state_out, y, ldy, dtype};
  if (int rc = ssm_check(*p, c, 0, rows, rows)) return rc;
  if (rows == 0) return 0;
  return dtype == FRHIP_F16 ? ssm_one_run<h1>(*p, c, rows, static_cast<hipStream_t>(s)) : ssm_one_run<float>(*p, c, rows, static_cast<hipStream_t>(s));
}

extern "C" size_t frhip_ssm_workspace_bytes(const frhip_ssm* p, int nseq, int T) {
  if (!p || p->channels <= 0 || p->groups <= 0 || p->channels % p->groups != 0 || p->states < 1 || p->states > 256 || nseq <= 0 || T <= 0) return 0;
  const ScanShape s = scan_shape(*p);
  const size_t bytes = scan_most_local(s, T) * (2 * (size_t)((p->states + 3) / 4 * 4) + 1) * p->channels * 4;
  return (bytes + 255) / 256 * 256;
}

extern "C" int frhip_ssm_seq(const frhip_ssm* p, int nseq, const int32_t* seq_start, const void* x, int ldx, const void* dt, int lddt,
                             const void* B, int ldb, const void* C, int ldc, const void* z, int ldz, const float* state, float* state_out,
                             void* y, int ldy, int dtype, void* workspace, frhip_stream s) {
  if (int rc = ssm_check_params(p)) return rc;
  if (int rc = check_seqs(nseq, seq_start, kMostTime, "ssm_seq: seq_start must be nseq + 1 row numbers up to 2^28 that do not descend")) return rc;
  const SsmCall c = {x, dt, B, C, z, ldx, lddt, ldb, ldc, ldz, state, state_out, y, ldy, dtype};
  const size_t row0 = nseq ? seq_start[0] : 0, rows = nseq ? seq_start[nseq] - seq_start[0] : 0;
  if (int rc = ssm_check(*p, c, row0, rows, nseq)) return rc;
  if (nseq == 0) return 0;
  if (scan_shape(*p).wgs > (1 << 21)) return set_error(FRHIP_ESHAPE, "ssm_seq: too many groups");
  if (frhip_ssm_workspace_bytes(p, nseq, (int)rows) > 0) {
    if (!workspace) return set_error(FRHIP_EINVAL, "ssm_seq: null workspace");
    if (reinterpret_cast<uintptr_t>(workspace) % 16 != 0) return set_error(FRHIP_EINVAL, "ssm_seq: workspace must be 16-byte aligned");
  }
  hipStream_t st = static_cast<hipStream_t>(s);
  return dtype == FRHIP_F16 ? ssm_seq_run<h1>(*p, c, nseq, seq_start, workspace, st) : ssm_seq_run<float>(*p, c, nseq, seq_start, workspace, st);
}

extern "C" int frhip_ssm_cut(const frhip_ssm* p, int nseq, const int32_t* seq_start, int compute_units, int* out) {
  if (int rc = ssm_check_params(p)) return rc;
  if (!out) return set_error(FRHIP_EINVAL, "ssm_cut: null pointer");
  if (compute_units < 1) return set_error(FRHIP_ESHAPE, "ssm_cut: no such scan");
  if (int rc = check_seqs(nseq, seq_start, INT_MAX, "ssm_cut: seq_start must be nseq + 1 row numbers that do not descend")) return rc;
  if (nseq < 1 || nseq > kSeqTable) return set_error(FRHIP_ESHAPE, "ssm_cut: 1 to 128 prompts");
  const ScanShape s = scan_shape(*p);
  SeqTable tab;
  out[0] = scan_chunk(s, nseq, seq_start, compute_units);
  out[1] = scan_table(tab, seq_start, 0, nseq, out[0]);
  out[2] = s.wgs;
  return 0;
}
