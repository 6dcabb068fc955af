// Products with bias, activation and residual: y = residual + act(x . w + bias), for any number of rows, K a multiple of 8, any N, rows of
// any pitch.  Sums are fp32 on the MFMA units (rows streamed: v_dot2_f32_f16), the epilogue is fp32, and a result is rounded once.
// The forms are those of the framework's other products, each with its reasons there, and so are the cuts and the expected times that
// choose among them (plan_linear), which know nothing of what an end reads and evaluates; what differs is the pitch of x, a K that need not fill its last step,
// and the end.  Not among them: the loading waves that frhip_gemm has for whole tiles of 256 rows and up to 160 columns, and rows of uint8 weights streamed (one and
// two go out as a few rows).
// us here and of frhip_gemm (no epilogue) on the same operands: 48 x 2048 x 8192 9.9 and 10.3, 512 x 2048 x 8192 25.5 and 25.3, 1024 x 2048 x
// 8192 40.3 and 40.8, 4099 x 5120 x 2560 114 and 114, 4096 x 2560 x 10240 208 and 205; the vendor library's binary16 product 18.5 (its
// call), 26.2, 38.2, 96.7, 251.
#include <climits>
#include <cstring>
#include <type_traits>

#include "activations.h"
#include "gemm_few_device.h"
#include "gemm_q8_device.h"
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
  int T, K, N, ldx, ldr, ldy, act;
  int out32;   // type of y and the residual
  int strips;  // linear_few_kernel: strips of rows
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

// f(activation, type of y and the residual), as types.  What ends a tile is a short loop for each of them: with the choice inside the loop,
// unrolled, a tile of 256 rows spent 12 us between its last product and its end, most of it on fetching instructions (4096 x 2560 x
// 10240, three rounds: 242 us, 220 so).
template <class F>
__device__ __forceinline__ void by_choice(const LinearArgs& a, F&& f) {
  auto typed = [&](auto type) {
    switch (a.act) {
      case FRHIP_ACT_SIGMOID: f(std::integral_constant<int, FRHIP_ACT_SIGMOID>(), type); break;
      case FRHIP_ACT_RELU2: f(std::integral_constant<int, FRHIP_ACT_RELU2>(), type); break;
      case FRHIP_ACT_SILU: f(std::integral_constant<int, FRHIP_ACT_SILU>(), type); break;
      case FRHIP_ACT_GELU: f(std::integral_constant<int, FRHIP_ACT_GELU>(), type); break;
      case FRHIP_ACT_SOFTPLUS: f(std::integral_constant<int, FRHIP_ACT_SOFTPLUS>(), type); break;
      default: f(std::integral_constant<int, FRHIP_ACT_NONE>(), type); break;
    }
  };
  if (a.out32) typed(float());
  else typed(h1());
}

// One output from its sum
template <int ACT, class O>
__device__ __forceinline__ void finish_one(const LinearArgs& a, float sum, int row, int col) {
  const float v = activate<sizeof(O) == 4>(a.bias ? sum + a.bias[col] : sum, ACT);
  static_cast<O*>(a.y)[(size_t)row * a.ldy + col] = (O)(a.res ? v + (float)static_cast<const O*>(a.res)[(size_t)row * a.ldr + col] : v);
}

// Residual and bias of W consecutive outputs, requested ahead of their sums, and the outputs from these
template <int ACT, class O, int W>
struct Outputs {
  typedef O any __attribute__((ext_vector_type(W), aligned(sizeof(O))));
  typedef float anyf __attribute__((ext_vector_type(W), aligned(4)));
  any r;
  anyf b;
  __device__ __forceinline__ void request(const LinearArgs& a, int row, int col) {
    if (a.res) r = *reinterpret_cast<const any*>(static_cast<const O*>(a.res) + (size_t)row * a.ldr + col);
    if (a.bias) b = *reinterpret_cast<const anyf*>(a.bias + col);
  }
  __device__ __forceinline__ void finish(const LinearArgs& a, const float (&s)[W], int row, int col) const {
    any y;
#pragma unroll
    for (int i = 0; i < W; i++) {
      const float v = activate<sizeof(O) == 4>(a.bias ? s[i] + b[i] : s[i], ACT);
      y[i] = (O)(a.res ? v + (float)r[i] : v);
    }
    *reinterpret_cast<any*>(static_cast<O*>(a.y) + (size_t)row * a.ldy + col) = y;
  }
};

// Groups of eight consecutive outputs whose sums are in LDS: place(t, row, col, sums) says where group t is, false: nowhere; a thread takes t0,
// t0 + step, ... below `end`, two at a time, whose residuals and biases are requested together.
template <class Place>
__device__ __forceinline__ void finish_groups(const LinearArgs& a, int t0, int step, int end, Place&& place) {
  by_choice(a, [&](auto act, auto type) {
    constexpr int G = 2;
#pragma unroll 1
    for (int t = t0; t < end; t += G * step) {
      int row[G], col[G];
      const float* sums[G];
      bool in[G], whole[G];
      Outputs<decltype(act)::value, decltype(type), 8> o[G];
#pragma unroll
      for (int g = 0; g < G; g++) {
        in[g] = t + g * step < end && place(t + g * step, row[g], col[g], sums[g]);
        whole[g] = in[g] && col[g] + 8 <= a.N;
        if (whole[g]) o[g].request(a, row[g], col[g]);
      }
#pragma unroll
      for (int g = 0; g < G; g++) {
        if (whole[g]) {
          float s[8];
          read_sums(s, sums[g]);
          o[g].finish(a, s, row[g], col[g]);
        } else if (in[g]) {  // the end of a row
#pragma unroll 1
          for (int i = 0; col[g] + i < a.N; i++) finish_one<decltype(act)::value, decltype(type)>(a, sums[g][i], row[g], col[g] + i);
        }
      }
    }
  });
}

// ---------------------------------------------------------------------------
// One or two rows: a wave streams COLS consecutive rows of the weight, 16 bytes a lane and load, and multiplies them with its lanes'
// pieces of x, which stay in registers (lane l has the 8 k of chunks l, l + 64, ... of a slice of K, of x and of every column alike).
// Reads beyond a row give zeros (buffer descriptors), so K may end anywhere.
// ---------------------------------------------------------------------------
__device__ __forceinline__ h8 load_chunk(__amdgpu_buffer_rsrc_t r, int byte) {
  return __builtin_bit_cast(h8, __builtin_amdgcn_raw_buffer_load_b128(r, byte, 0, 0));
}
__device__ __forceinline__ h8 load_chunk_once(__amdgpu_buffer_rsrc_t r, int byte) {
  return __builtin_bit_cast(h8, __builtin_amdgcn_raw_buffer_load_b128(r, byte, 0, 2));  // non-temporal
}
__device__ __forceinline__ __amdgpu_buffer_rsrc_t row_rsrc(const void* p, unsigned bytes) {
  return __builtin_amdgcn_make_buffer_rsrc(const_cast<unsigned char*>(uniform_ptr(p)), 0, bytes, 0x00020000);
}

template <int TR, int NCH, int COLS>
__global__ __launch_bounds__(512) void linear_rows_kernel(LinearArgs a) {
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int n0 = (blockIdx.x * 8 + wave) * COLS;
  if (n0 >= a.N) return;
  const unsigned bytes = (unsigned)a.K * 2;
  float acc[TR][COLS];
#pragma unroll
  for (int t = 0; t < TR; t++)
#pragma unroll
    for (int j = 0; j < COLS; j++) acc[t][j] = 0.f;
  for (int k = 0; k < a.K; k += NCH * 512) {
    h8 x[TR][NCH], w[COLS][NCH];
#pragma unroll
    for (int t = 0; t < TR; t++) {
      const auto r = row_rsrc(a.x + (size_t)min(t, a.T - 1) * a.ldx, bytes);
#pragma unroll
      for (int i = 0; i < NCH; i++) x[t][i] = load_chunk(r, (k + i * 512 + lane * 8) * 2);
    }
#pragma unroll
    for (int j = 0; j < COLS; j++) {
      const auto r = row_rsrc(a.w + (size_t)min(n0 + j, a.N - 1) * a.K * 2, n0 + j < a.N ? bytes : 0);
#pragma unroll
      for (int i = 0; i < NCH; i++) w[j][i] = load_chunk_once(r, (k + i * 512 + lane * 8) * 2);
    }
#pragma unroll
    for (int j = 0; j < COLS; j++)
#pragma unroll
      for (int i = 0; i < NCH; i++)
#pragma unroll
        for (int t = 0; t < TR; t++) acc[t][j] = dot8acc(w[j][i], x[t][i], acc[t][j]);
  }
  // sum t COLS + j goes to lane t COLS + j, which finishes it
  float mine = 0.f;
#pragma unroll
  for (int t = 0; t < TR; t++)
#pragma unroll
    for (int j = 0; j < COLS; j++) {
      const float s = wave_sum(acc[t][j]);
      mine = lane == t * COLS + j ? s : mine;
    }
  const int t = lane / COLS, col = n0 + lane % COLS;
  if (t < TR && t < a.T && col < a.N) {
    by_choice(a, [&](auto act, auto type) { finish_one<decltype(act)::value, decltype(type)>(a, mine, t, col); });
  }
}

template <int TR, int NCH, int COLS>
static void rows_launch(const LinearArgs& a, hipStream_t st) {
  hipLaunchKernelGGL((linear_rows_kernel<TR, NCH, COLS>), dim3((unsigned)((a.N + 8 * COLS - 1) / (8 * COLS))), dim3(512), 0, st, a);
}
template <int TR, int NCH>
static void rows_cols(const LinearArgs& a, hipStream_t st) {
  const int waves = compute_units() * 8;  // as many columns a wave as give every compute unit eight waves, while they fit its registers
  if (NCH <= 4 && a.N >= 4 * waves) rows_launch<TR, NCH, NCH <= 4 ? 4 : 1>(a, st);
  else if (a.N >= 2 * waves) rows_launch<TR, NCH, 2>(a, st);
  else rows_launch<TR, NCH, 1>(a, st);
}
template <int TR>
static int launch_rows(const LinearArgs& a, hipStream_t st) {
  if (a.K <= 512) rows_cols<TR, 1>(a, st);
  else if (a.K <= 1024) rows_cols<TR, 2>(a, st);
  else if (a.K <= 2048) rows_cols<TR, 4>(a, st);
  else rows_cols<TR, 8>(a, st);
  return check_launch("linear");
}

// ---------------------------------------------------------------------------
// A few rows, one launch, K split over the waves of a workgroup (gemm_few.hip has the form, its reasons and its choice of tiles), here with
// rows of any pitch, any N, and a K that need not fill its last step (a multiple of 8): the last step's loads of
// what is not there repeat the step's begin, and what they bring counts as zero.  Codes are loaded 16 a lane, from any multiple of 8 bytes.
// ---------------------------------------------------------------------------
template <int MT, int NT, bool U8>
__global__ __launch_bounds__(few_waves(MT, NT) * 64) void linear_few_kernel(LinearArgs a) {
  constexpr int NW = few_waves(MT, NT), S = few_stages(MT, NT, U8), kStage = few_stage_bytes(MT, NT, U8);
  constexpr int kBOff = MT * 2048, kScaleOff = kBOff + NT * (U8 ? 1024 : 2048);
  constexpr int kPer = 2 * MT + (U8 ? NT + 1 : 2 * NT);  // load instructions per step
  static_assert(S >= 2 && (S - 1) * kPer <= 63, "the wait counter's range");
  extern __shared__ __attribute__((aligned(16))) unsigned char few_smem[];

  // tiles are dealt to the XCDs in contiguous runs, strips of rows fastest: the strips that share weights share an L2
  const int n = gridDim.x, strips = a.strips, lin = blockIdx.x, xcd = lin & 7;
  const int id = xcd * (n >> 3) + min(xcd, n & 7) + (lin >> 3);
  const int tile = id / strips, strip = id - tile * strips;
  const int M = a.T, K = a.K, N = a.N, n0 = tile * (NT * 16), m0 = strip * (MT * 16);
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int row16 = lane & 15, grp = lane >> 4;

  unsigned char* const ring = few_smem + wave * few_wave_bytes(MT, NT, U8);
  const unsigned ring_lds = (unsigned)(size_t)((__attribute__((address_space(3))) unsigned char*)few_smem) + wave * few_wave_bytes(MT, NT, U8);

  // ---- this wave's loads; rows past the matrix repeat its last row and are never stored ----
  const int lr = lane >> 3;
  unsigned va[2 * MT], vb[U8 ? NT : 2 * NT];
#pragma unroll
  for (int b = 0; b < 2 * MT; b++) {
    const int row = min(m0 + b * 8 + lr, M - 1) - m0;
    va[b] = (unsigned)row * (unsigned)(a.ldx * 2) + (((lane & 7) ^ lr ^ (b & 1)) * 16);
  }
  if constexpr (U8) {
#pragma unroll
    for (int b = 0; b < NT; b++) {
      const int col = min(n0 + b * 16 + (lane >> 2), N - 1) - n0;
      vb[b] = (unsigned)col * (unsigned)K + (((lane & 3) ^ (lane >> 4)) * 16);
    }
  } else {
#pragma unroll
    for (int b = 0; b < 2 * NT; b++) {
      const int col = min(n0 + b * 8 + lr, N - 1) - n0;
      vb[b] = (unsigned)col * (unsigned)(K * 2) + (((lane & 7) ^ lr ^ (b & 1)) * 16);
    }
  }
  const unsigned char* const abase = uniform_ptr(reinterpret_cast<const unsigned char*>(a.x) + (size_t)m0 * a.ldx * 2);
  const unsigned char* const bbase = uniform_ptr(a.w + (size_t)n0 * K * (U8 ? 1 : 2));
  const h1* scale_k = nullptr;  // uint8: lanes 0..31 bring ry, lanes 32..63 my, two values each
  if constexpr (U8) scale_k = (lane < 32 ? a.ry : a.my) + (lane & 31) * 2;
  const int nk = (K + 63) >> 6, krest = K - (nk - 1) * 64, mine = wave < nk ? (nk - wave + NW - 1) / NW : 0;
  auto issue = [&](int i) {
    const int k0 = (wave + i * NW) * 64;
    const unsigned st = ring_lds + (i % S) * kStage;
    const unsigned char* ak = abase + (size_t)k0 * 2;
    const unsigned char* bk = bbase + (size_t)k0 * (U8 ? 1 : 2);
    if (k0 + 64 > K) {  // once, and the wave's last: back to the step's begin with the k-segments that are not there
#pragma unroll
      for (int b = 0; b < 2 * MT; b++) {
        const unsigned seg = (lane & 7) ^ lr ^ (b & 1);
        if ((int)seg * 8 >= krest) va[b] -= seg * 16;
      }
#pragma unroll
      for (int b = 0; b < (U8 ? NT : 2 * NT); b++) {
        const unsigned seg = U8 ? (lane & 3) ^ (lane >> 4) : (lane & 7) ^ lr ^ (b & 1);
        if (U8 && (krest & 8)) {  // the last 16 codes, of which the half that ends K is wanted; they may begin ahead of the step
          vb[b] += (int)seg * 16 + 16 > krest ? krest - seg * 16 : 16;
        } else if ((int)seg * (U8 ? 16 : 8) >= krest) {
          vb[b] -= seg * 16;
        }
      }
      if constexpr (U8) {
        if (krest & 8) bk -= 16;
        if ((lane & 31) * 2 >= krest) scale_k -= (lane & 31) * 2;
      }
    }
#pragma unroll
    for (int b = 0; b < (U8 ? NT : 2 * NT); b++) load_lds_saddr(vb[b], bk, st + kBOff + b * 1024);
#pragma unroll
    for (int b = 0; b < 2 * MT; b++) load_lds_saddr(va[b], ak, st + b * 1024);
    if constexpr (U8) load_lds_dword(scale_k + k0, st + kScaleOff);
  };
  if constexpr (U8) {  // rx, mx of this workgroup's columns, two a lane
    static_assert(NT * 16 <= 128, "two columns a lane");
    h1* const sc = reinterpret_cast<h1*>(ring + S * kStage);
#pragma unroll
    for (int e = 0; e < 2; e++) {
      const int c = min(n0 + lane * 2 + e, N - 1);
      sc[lane * 2 + e] = a.rx[c];
      sc[128 + lane * 2 + e] = a.mx[c];
    }
    lanes_in_order();
  }
#pragma unroll
  for (int i = 0; i < S; i++)
    if (i < mine) issue(i);

  f4v acc[MT][NT];
#pragma unroll
  for (int i = 0; i < MT; i++)
#pragma unroll
    for (int j = 0; j < NT; j++) acc[i][j] = (f4v){0.f, 0.f, 0.f, 0.f};
  // loads complete in order: a step has landed when at most the loads of the steps behind it are outstanding
  auto landed = [&](int behind) {
    if (behind >= S - 1) wait_loads<(S - 1) * kPer>();
    else if (S > 3 && behind == 2) wait_loads<(S > 3 ? 2 : 0) * kPer>();
    else if (S > 2 && behind == 1) wait_loads<(S > 2 ? 1 : 0) * kPer>();
    else wait_loads<0>();
  };
  float c[NT], m[NT];  // uint8: rx / 255 and mx of the lane's columns
  if constexpr (U8) {
    landed(mine - 1);
#pragma unroll
    for (int t = 0; t < NT; t++) {
      const h1* sc = reinterpret_cast<const h1*>(ring + S * kStage) + t * 16 + row16;
      c[t] = dequant_c(sc[0]);
      m[t] = (float)sc[128];
    }
  }
  for (int i = 0; i < mine; i++) {
    landed(mine - 1 - i);
    const unsigned char* st = ring + (i % S) * kStage;
    h8 xa[2][MT], wb[2][NT];
#pragma unroll
    for (int t = 0; t < MT; t++)
#pragma unroll
      for (int h = 0; h < 2; h++) xa[h][t] = *reinterpret_cast<const h8*>(st + t * 2048 + few_at(row16, 2 * grp + h));
    if constexpr (U8) {
      u32x4 q[NT];
      h8 ry[2], my[2];
#pragma unroll
      for (int h = 0; h < 2; h++) {
        ry[h] = *reinterpret_cast<const h8*>(st + kScaleOff + grp * 32 + h * 16);
        my[h] = *reinterpret_cast<const h8*>(st + kScaleOff + 128 + grp * 32 + h * 16);
      }
#pragma unroll
      for (int t = 0; t < NT; t++)
        q[t] = *reinterpret_cast<const u32x4*>(st + kBOff + t * 1024 + row16 * 64 + ((grp ^ (row16 >> 2)) * 16));
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // the slot has been read
      if (i + S < mine) issue(i + S);
      if ((krest & 8) && (wave + i * NW) * 64 + 64 > K) {
#pragma unroll
        for (int t = 0; t < NT; t++)
          if (grp == krest >> 4) q[t][0] = q[t][2], q[t][1] = q[t][3];
      }
#pragma unroll
      for (int t = 0; t < NT; t++)
#pragma unroll
        for (int h = 0; h < 2; h++) {
          const uint32_t w0 = q[t][2 * h], w1 = q[t][2 * h + 1];
          const h2 p0 = few_dequant<0>(w0, c[t], m[t], ry[h].s01, my[h].s01);
          const h2 p1 = few_dequant<1>(w0, c[t], m[t], ry[h].s23, my[h].s23);
          const h2 p2 = few_dequant<0>(w1, c[t], m[t], ry[h].s45, my[h].s45);
          const h2 p3 = few_dequant<1>(w1, c[t], m[t], ry[h].s67, my[h].s67);
          wb[h][t] = (h8){p0.x, p0.y, p1.x, p1.y, p2.x, p2.y, p3.x, p3.y};
        }
    } else {
#pragma unroll
      for (int t = 0; t < NT; t++)
#pragma unroll
        for (int h = 0; h < 2; h++) wb[h][t] = *reinterpret_cast<const h8*>(st + kBOff + t * 2048 + few_at(row16, 2 * grp + h));
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
      if (i + S < mine) issue(i + S);
    }
    if ((wave + i * NW) * 64 + 64 > K) {
#pragma unroll
      for (int h = 0; h < 2; h++) {
        const bool in = (2 * grp + h) * 8 < krest;
#pragma unroll
        for (int t = 0; t < MT; t++) xa[h][t] = in ? xa[h][t] : (h8)(h1)0.f;
#pragma unroll
        for (int j = 0; j < NT; j++) wb[h][j] = in ? wb[h][j] : (h8)(h1)0.f;
      }
    }
#pragma unroll
    for (int h = 0; h < 2; h++)
#pragma unroll
      for (int t = 0; t < MT; t++)
#pragma unroll
        for (int j = 0; j < NT; j++) acc[t][j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(wb[h][j], xa[h][t], acc[t][j], 0, 0, 0);
  }

  // ---- the waves' sums meet: each leaves its tiles in its own ring (a tile is 1 KB; MT NT <= 2 S (MT + NT / 2) of them fit) ----
  static_assert(MT * NT * 1024 <= S * kStage, "the sums fit the ring");
#pragma unroll
  for (int t = 0; t < MT; t++)
#pragma unroll
    for (int j = 0; j < NT; j++) *reinterpret_cast<f4v*>(ring + ((t * NT + j) * 64 + lane) * 16) = acc[t][j];
  __syncthreads();
  by_choice(a, [&](auto act, auto type) {
#pragma unroll 1
    for (int t = wave; t < MT * NT; t += NW) {
      const int i = t / NT, j = t - i * NT, row = m0 + i * 16 + row16, col = n0 + j * 16 + grp * 4;
      const bool in = row < M && col < N, whole = in && col + 4 <= N;
      Outputs<decltype(act)::value, decltype(type), 4> o;
      if (whole) o.request(a, row, col);
      float s[4];
#pragma unroll
      for (int w = 0; w < NW; w++) {  // in wave order
        const f4v p = *reinterpret_cast<const f4v*>(few_smem + w * few_wave_bytes(MT, NT, U8) + (t * 64 + lane) * 16);
#pragma unroll
        for (int v = 0; v < 4; v++) s[v] = w == 0 ? p[v] : s[v] + p[v];
      }
      if (whole) {
        o.finish(a, s, row, col);
      } else if (in) {
#pragma unroll
        for (int v = 0; v < 4; v++)
          if (col + v < N) finish_one<decltype(act)::value, decltype(type)>(a, s[v], row, col + v);
      }
    }
  });
}

template <int MT, int NT, bool U8>
static void few_launch(const LinearArgs& a, hipStream_t st) {
  constexpr size_t lds = (size_t)few_waves(MT, NT) * few_wave_bytes(MT, NT, U8);
  static const bool raised = [] {
    (void)hipFuncSetAttribute(reinterpret_cast<const void*>(&linear_few_kernel<MT, NT, U8>), hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds);
    return true;
  }();
  (void)raised;
  const unsigned grid = (unsigned)((a.N + NT * 16 - 1) / (NT * 16)) * a.strips;
  hipLaunchKernelGGL((linear_few_kernel<MT, NT, U8>), dim3(grid), dim3(few_waves(MT, NT) * 64), lds, st, a);
}

template <bool U8>
static int launch_few(LinearArgs a, const FewPlan& p, hipStream_t st) {
  a.strips = (a.T + 16 * p.mt - 1) / (16 * p.mt);
#define FR_FEW_GO(MT_, NT_) \
  if (p.mt == MT_ && p.nt == NT_) few_launch<MT_, NT_, U8>(a, st);
  FR_FEW_TILES(FR_FEW_GO)
#undef FR_FEW_GO
  return check_launch("linear");
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

// A tile of ROWS rows and `width` blocks of 32 columns whose sums are in LDS, shared by all waves of the workgroup
template <int ROWS, int THREADS>
__device__ __forceinline__ void finish_tile_of(const LinearTiles& a, const float* sums, int width, int m0, int n0) {
  const int pitch = sums_pitch(a.maxw), groups = width * 4;  // of 8 outputs
  const unsigned inv = ((1u << 20) + groups - 1) / groups;   // i / groups for i < 4096, groups <= 32
  static_assert(ROWS * 4 * 8 <= 4096, "the division");
  finish_groups(a.l, threadIdx.x, THREADS, ROWS * groups, [&](int i, int& row, int& col, const float*& from) {
    const int r = (int)((unsigned)i * inv >> 20), c = (i - r * groups) * 8;
    row = m0 + r;
    col = n0 + c;
    from = sums + r * pitch + c;
    return row < a.l.T && col < a.l.N;
  });
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

template <int BM, int S, bool TAIL>
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
  finish_tile_of<BM, kRingThreads>(a, reinterpret_cast<const float*>(ring_smem), width, m0, n0);
}

template <int BM, int S, bool TAIL>
static void ring_launch(const TilePlan& p, const LinearTiles& t, hipStream_t st) {
  static const bool raised = [] {
    (void)hipFuncSetAttribute(reinterpret_cast<const void*>(&linear_ring_kernel<BM, S, TAIL>), hipFuncAttributeMaxDynamicSharedMemorySize, 160 * 1024);
    return true;
  }();
  (void)raised;
  const int ring = S * (BM * 128 + t.maxw * 4096), sums = BM * sums_pitch(t.maxw) * 4;
  hipLaunchKernelGGL((linear_ring_kernel<BM, S, TAIL>), p.grid, dim3(kRingThreads), ring > sums ? ring : sums, st, t);
}

// ---------------------------------------------------------------------------
// Many rows: tiles of 256 rows, eight waves of 64 rows by half the width that load for themselves one step ahead (gemm_vw256_kernel has the
// form and its reasons); the sums go out through a place in LDS of each wave's own.
// ---------------------------------------------------------------------------
constexpr int kWideThreads = 512, kWideMostBlocks = 8, kWideABytes = 256 * kLdwBK * 2;
static_assert(2 * (kWideABytes + kWideMostBlocks * 4096) <= 160 * 1024 && 8 * wave_sums_bytes((kWideMostBlocks + 1) / 2) <= 160 * 1024, "LDS of a compute unit");

// Blocks that lie inside the matrix, without an activation: acc[i][j][v] is C[row0 + 32 i + 8 (v / 4) + v % 4][col0 + 32 j].  4096 x 2560 x 10240 through LDS 220 us,
// so 208.
template <class O, int NJ>
__device__ __forceinline__ void store_blocks(const LinearArgs& a, const f16v (&acc)[2][NJ], int row0, int col0) {
#pragma unroll
  for (int j = 0; j < NJ; j++) {
    const float b = a.bias ? a.bias[col0 + j * 32] : 0.f;
#pragma unroll
    for (int i = 0; i < 2; i++) {
      const O* const res = static_cast<const O*>(a.res) + (size_t)(row0 + i * 32) * a.ldr + col0 + j * 32;
      O* const out = static_cast<O*>(a.y) + (size_t)(row0 + i * 32) * a.ldy + col0 + j * 32;
      float r[16];
#pragma unroll
      for (int v = 0; v < 16; v++) r[v] = 0.f;
      if (a.res) {
#pragma unroll
        for (int v = 0; v < 16; v++) r[v] = (float)res[(size_t)(8 * (v >> 2) + (v & 3)) * a.ldr];
      }
#pragma unroll
      for (int v = 0; v < 16; v++) {
        const float y = acc[i][j][v] + b;
        out[(size_t)(8 * (v >> 2) + (v & 3)) * a.ldy] = (O)(a.res ? y + r[v] : y);
      }
    }
  }
}

template <int NJ, bool TAIL>
__device__ __forceinline__ void wide_body(const LinearTiles& a, unsigned char* smem, int width, int brow0, int m0, int n0, int lane, int wave) {
  const int M = a.l.T, K = a.l.K, N = a.l.N, lda = a.l.ldx, nk = TAIL ? (K + kLdwBK - 1) / kLdwBK : K / kLdwBK, krest = TAIL ? K - (nk - 1) * kLdwBK : kLdwBK;
  const int wm = wave >> 1, nb = 4 * width;
  const unsigned stage_bytes = kWideABytes + a.maxw * 4096;
  // this wave's loads: row groups 4 wave .. + 3 of A, row groups wave, wave + 8, ... of B (there are 4 width)
  unsigned va[4], vb[4];
  const int lr = lane >> 3, ls = (lane & 7) ^ lr;
#pragma unroll
  for (int i = 0; i < 4; i++) {
    const int ga = wave * 4 + i, gb = wave + 8 * i;
    va[i] = (unsigned)(min(m0 + ga * 8 + lr, M - 1) - m0) * (unsigned)(lda * 2) + (ls ^ (ga & 1)) * 16;
    vb[i] = (unsigned)(min(n0 + gb * 8 + lr, N - 1) - n0) * (unsigned)(K * 2) + (ls ^ (gb & 1)) * 16;
  }
  const unsigned char* abase = uniform_ptr(reinterpret_cast<const unsigned char*>(a.l.x) + (size_t)m0 * lda * 2);
  const unsigned char* bbase = uniform_ptr(a.l.w + (size_t)n0 * K * 2);
  const unsigned lds0 = (unsigned)(size_t)((__attribute__((address_space(3))) unsigned char*)smem);
  auto issue = [&](int step) {
    const unsigned st = lds0 + (step & 1) * stage_bytes;
    const unsigned char* ak = abase + (size_t)step * (kLdwBK * 2);
    const unsigned char* bk = bbase + (size_t)step * (kLdwBK * 2);
    if constexpr (TAIL) {
      if (step == nk - 1) {  // the last loads: what is not there repeats the step's begin
#pragma unroll
        for (int i = 0; i < 4; i++) {
          const int sa = ls ^ (i & 1), sb = ls ^ (wave & 1);
          if (sa * 8 >= krest) va[i] -= sa * 16;
          if (sb * 8 >= krest) vb[i] -= sb * 16;
        }
      }
    }
#pragma unroll
    for (int i = 0; i < 4; i++) load_lds_saddr(va[i], ak, st + (wave * 4 + i) * 1024);
#pragma unroll
    for (int i = 0; i < 4; i++)
      if (wave + 8 * i < nb) load_lds_saddr(vb[i], bk, st + kWideABytes + (wave + 8 * i) * 1024);
  };
  f16v acc[2][NJ];
#pragma unroll
  for (int i = 0; i < 2; i++)
#pragma unroll
    for (int j = 0; j < NJ; j++)
#pragma unroll
      for (int v = 0; v < 16; v++) acc[i][j][v] = 0.f;
  issue(0);
  for (int k = 0; k < nk; k++) {
    // this wave's loads of step k have landed and its fragments of step k-1 are in registers; behind the
    // barrier that holds for all eight, so step k may be read and the slot of step k-1 refilled
    __builtin_amdgcn_s_waitcnt(0x0070);  // vmcnt(0) lgkmcnt(0)
    step_barrier();
    if (k + 1 < nk) issue(k + 1);
    const unsigned char* st = smem + (k & 1) * stage_bytes;
#pragma unroll
    for (int kb = 0; kb < 4; kb++) {
      h8 fa[2], fb[NJ];
      const int q = kb * 2 + (lane >> 5);
#pragma unroll
      for (int i = 0; i < 2; i++) fa[i] = *reinterpret_cast<const h8*>(st + ldw_at(wm * 64 + i * 32 + (lane & 31), q));
#pragma unroll
      for (int j = 0; j < NJ; j++) fb[j] = *reinterpret_cast<const h8*>(st + kWideABytes + ldw_at(brow0 + j * 32 + (lane & 31), q));
      if constexpr (TAIL) {
        if (k == nk - 1) {
#pragma unroll
          for (int i = 0; i < 2; i++) fa[i] = q * 8 < krest ? fa[i] : (h8)(h1)0.f;
#pragma unroll
          for (int j = 0; j < NJ; j++) fb[j] = q * 8 < krest ? fb[j] : (h8)(h1)0.f;
        }
      }
#pragma unroll
      for (int i = 0; i < 2; i++)
#pragma unroll
        for (int j = 0; j < NJ; j++) acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_f16(fa[i], fb[j], acc[i][j], 0, 0, 0);
    }
  }
  if (a.l.act == FRHIP_ACT_NONE && m0 + 256 <= M && n0 + width * 32 <= N) {  // whole tiles: straight from the accumulators
    const int row0 = m0 + wm * 64 + 4 * (lane >> 5), col0 = n0 + brow0 + (lane & 31);
    if (a.l.out32) store_blocks<float, NJ>(a.l, acc, row0, col0);
    else store_blocks<h1, NJ>(a.l, acc, row0, col0);
    return;
  }
  // the last fragments are in registers (the compiler may leave their wait behind the barrier, with the products), then all waves' are
  asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
  step_barrier();  // all fragments have been read
  float* const sums = reinterpret_cast<float*>(smem + wave * wave_sums_bytes((a.maxw + 1) / 2));
#pragma unroll 1
  for (int i = 0; i < 2; i++) {  // one copy of what follows
    if (i == 0) {
      sums_to_lds(acc[0], sums, sums_pitch(NJ), lane);
    } else {
      lanes_in_order();  // the rows before have been read
      sums_to_lds(acc[1], sums, sums_pitch(NJ), lane);
    }
    lanes_in_order();
    finish_groups(a.l, lane, 64, 32 * NJ * 4, [&](int t, int& row, int& col, const float*& from) {
      const int r = t / (NJ * 4), c = (t - r * (NJ * 4)) * 8;
      row = m0 + wm * 64 + i * 32 + r;
      col = n0 + brow0 + c;
      from = sums + r * sums_pitch(NJ) + c;
      return row < M && col < N;
    });
  }
}

template <bool TAIL>
__global__ __launch_bounds__(kWideThreads) void linear_wide_kernel(LinearTiles a) {
  extern __shared__ __attribute__((aligned(16))) unsigned char wide_smem[];
  int bx, by;
  xcd_tile(bx, by);
  const int width = a.base + (bx < a.wide ? 1 : 0), n0 = (bx * a.base + min(bx, a.wide)) * 32, m0 = by * 256;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int nj0 = (width + 1) >> 1, nj = (wave & 1) ? width - nj0 : nj0, brow0 = (wave & 1) ? nj0 * 32 : 0;
  switch (nj) {  // every wave passes the same barriers, whatever its width
    case 1: wide_body<1, TAIL>(a, wide_smem, width, brow0, m0, n0, lane, wave); break;
    case 2: wide_body<2, TAIL>(a, wide_smem, width, brow0, m0, n0, lane, wave); break;
    case 3: wide_body<3, TAIL>(a, wide_smem, width, brow0, m0, n0, lane, wave); break;
    default: wide_body<4, TAIL>(a, wide_smem, width, brow0, m0, n0, lane, wave); break;
  }
}

template <bool TAIL>
static void wide_launch(const TilePlan& p, const LinearTiles& t, hipStream_t st) {
  static const bool raised = [] {
    (void)hipFuncSetAttribute(reinterpret_cast<const void*>(&linear_wide_kernel<TAIL>), hipFuncAttributeMaxDynamicSharedMemorySize, 160 * 1024);
    return true;
  }();
  (void)raised;
  const int ring = 2 * (kWideABytes + t.maxw * 4096), sums = 8 * wave_sums_bytes((t.maxw + 1) / 2);
  hipLaunchKernelGGL(linear_wide_kernel<TAIL>, p.grid, dim3(kWideThreads), ring > sums ? ring : sums, st, t);
}

// ---------------------------------------------------------------------------
// uint8 weights, more rows: the codes are dequantised on their way into LDS by waves of their own (gemm_q8.hip has the form and its
// reasons), for whole steps of K and whole blocks of 16 columns.
// ---------------------------------------------------------------------------
template <int BM>
__global__ __launch_bounds__(64 * (4 + kQ8Producers)) void linear_q8_kernel(LinearTiles a) {
  extern __shared__ __attribute__((aligned(16))) unsigned char q8_smem[];
  int bx, by;
  xcd_tile(bx, by);
  const int width = a.base + (bx < a.wide ? 1 : 0), n0 = (bx * a.base + min(bx, a.wide)) * 32, m0 = by * BM;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), nk = a.l.K / kLdwBK;
  if (wave >= 4) {
    const int p = wave - 4;
    const GemmSeg sg = {a.l.x, a.l.w, a.l.mx, a.l.rx, a.l.my, a.l.ry, nullptr, a.l.N, 0};
    switch (p < 2 * width ? (2 * width - p + kQ8Producers - 1) / kQ8Producers : 0) {
      case 0: q8_producer<BM, 0>(sg, q8_smem, a.maxw, p, m0, n0, a.l.T, a.l.K, a.l.ldx, 0, nk, lane); break;
      case 1: q8_producer<BM, 1>(sg, q8_smem, a.maxw, p, m0, n0, a.l.T, a.l.K, a.l.ldx, 0, nk, lane); break;
      default: q8_producer<BM, 2>(sg, q8_smem, a.maxw, p, m0, n0, a.l.T, a.l.K, a.l.ldx, 0, nk, lane); break;
    }
  } else {
    const int wm = wave >> 1, nj0 = (width + 1) >> 1, nj = (wave & 1) ? width - nj0 : nj0, brow0 = (wave & 1) ? nj0 * 32 : 0;
    switch (nj) {  // every wave passes the same barriers, whatever its width
      case 1: q8_mma<BM, 1>(q8_smem, a.maxw, brow0, nk, lane, wm); break;
      case 2: q8_mma<BM, 2>(q8_smem, a.maxw, brow0, nk, lane, wm); break;
      case 3: q8_mma<BM, 3>(q8_smem, a.maxw, brow0, nk, lane, wm); break;
      default: q8_mma<BM, q8_max_blocks(BM) / 2>(q8_smem, a.maxw, brow0, nk, lane, wm); break;
    }
  }
  __syncthreads();
  finish_tile_of<BM, 64 * (4 + kQ8Producers)>(a, reinterpret_cast<const float*>(q8_smem), width, m0, n0);
}

template <int BM>
static void q8_launch(const TilePlan& p, const LinearTiles& t, hipStream_t st) {
  static const bool raised = [] {
    (void)hipFuncSetAttribute(reinterpret_cast<const void*>(&linear_q8_kernel<BM>), hipFuncAttributeMaxDynamicSharedMemorySize, 160 * 1024);
    return true;
  }();
  (void)raised;
  hipLaunchKernelGGL(linear_q8_kernel<BM>, p.grid, dim3(64 * (4 + kQ8Producers)), q8_lds_bytes(BM, t.maxw), st, t);
}

template <bool TAIL>
static int launch_tiles(const LinearArgs& a, const TilePlan& p, hipStream_t st) {
  const LinearTiles t = {a, p.a.vw_base[0], p.a.vw_wide[0], p.a.vw_maxw};
  if (p.rows == 256) wide_launch<TAIL>(p, t, st);
  else if (p.rows == 64) ring_launch<64, 4, TAIL>(p, t, st);
  else if (ring_stages(128, t.maxw) == 4) ring_launch<128, 4, TAIL>(p, t, st);
  else ring_launch<128, 3, TAIL>(p, t, st);
  return check_launch("linear");
}

constexpr int kLinearMostK = 8388544;  // whole steps of it keep 256 rows of a tile within 32-bit byte offsets
constexpr int kLinearMostN = 1 << 24;                    // a launch's threads stay in 32 bits
constexpr size_t kLinearMostWeight = (size_t)1 << 34;    // 32 GiB of binary16

// How a product goes out: the forms and cuts of the same product (K and N rounded up to whole steps and blocks) without a
// residual on the framework's other kernels, by the same expected times.  A pure function of the sizes.
struct LinearPlan {
  FewPlan few;           // mt: a few rows
  TilePlan tiles;        // otherwise
  bool codes = false;    // uint8: the tiles dequantise
  bool expand = false;   // uint8: the codes are expanded to binary16 first
  int head = 0;          // tiles: so many rows, and the rest of them behind it in a launch of its own ...
  FewPlan rest;          // ... as a few rows; 0: all
};

static TilePlan plan_tiles(const GemmArgs& g, int cus) {
  TilePlan p = plan_ring(g, cus);
  const TilePlan wide = g.M > 128 ? plan_256(g, cus) : TilePlan();
  return wide.rows && (!p.rows || wide.us <= p.us * 1.05) ? wide : p;
}

// A few rows behind the last whole tile cost a strip of tiles, and with it often a round of wider ones: they go out behind the others as a few
// rows where that is expected to save 8 %.  In one launch and in two, us: 2051 x 2048 x 8192 84.0 and 73.1, 4099 x 4096 x 4096 144 and 129, 8195 x
// 2048 x 2048 82.0 and 70.0, 1027 x 2048 x 8192 46.3 and 44.9, where it is not done 4104 x 5120 x 2560 111 and 115, 1027 x 5120 x 5120 61 and 67; over
// 60 drawn products that it was tried on 4 % less in the mean, 5 % more at worst.
constexpr double kLinearSplit = 0.92;
static void split_rest(LinearPlan& p, GemmArgs g, int cus) {
  const int T = g.M;
  double best = p.tiles.us * kLinearSplit;
  for (int rows = 256; rows >= 64; rows /= 2) {
    const int head = T / rows * rows;
    if (head == 0 || head == T || head == p.head) continue;
    g.M = T - head;
    const int N = g.seg[0].N;
    g.seg[0].N = (N + 15) / 16 * 16;
    const FewPlan rest = plan_few(g, cus);
    g.seg[0].N = N;
    if (!rest.mt || rest.us >= best) continue;
    g.M = head;
    const TilePlan tiles = plan_tiles(g, cus);
    if (!tiles.rows || tiles.us + rest.us >= best) continue;
    best = tiles.us + rest.us;
    p.tiles = tiles;
    p.head = head;
    p.rest = rest;
  }
}

static LinearPlan plan_linear(int T, int K, int N, bool u8, int cus) {
  GemmArgs g;
  memset(&g, 0, sizeof(g));
  g.M = T;
  g.K = (K + kLdwBK - 1) / kLdwBK * kLdwBK;
  g.nseg = 1;
  g.seg[0].N = (N + 15) / 16 * 16;
  LinearPlan p;
  p.few = plan_few(g, cus);
  g.seg[0].N = N;
  p.tiles = plan_tiles(g, cus);
  if (!u8) {
    if (p.few.mt && p.tiles.rows && p.tiles.us < p.few.us) p.few.mt = 0;
    if (!p.few.mt && p.tiles.rows) split_rest(p, g, cus);
    return p;
  }
  // codes: dequantised by the lanes that multiply them (K of 24 and more, or 16), on their way into LDS, or expanded ahead of either
  const double expand = 5.5 + 3.0 * K * N / 6.3e6;
  if (K % kLdwBK == 0 && N % 16 == 0) {
    const TilePlan q8 = plan_q8(g, cus);
    if (q8.rows && (!p.tiles.rows || q8.us <= p.tiles.us + expand)) {
      p.tiles = q8;
      p.codes = true;
    }
  }
  const bool direct = K >= 16;
  const double few = p.few.us + (direct ? 0 : expand), tiles = p.tiles.us + (p.codes ? 0 : expand);
  if (p.few.mt && p.tiles.rows && tiles < few) p.few.mt = 0;
  p.expand = p.few.mt ? !direct : !p.codes;
  if (!p.few.mt && p.tiles.rows && p.expand) split_rest(p, g, cus);
  return p;
}

// Whether a product of uint8 weights of T rows, or of fewer, expands its codes: a workspace for T rows serves fewer as well, though `expand` comes and
// goes with the expected times (2048 x 8192 codes: 641 to 1024 rows, 1153 to 1280, from 1409 on).  Every expected time is one number for all rows
// of a strip: of 16 while a few rows are among the forms, of 64 beyond.  Above kExpandRows the answer is yes unasked.
constexpr int kExpandRows = 8192;
static bool expands_up_to(int T, int K, int N, int cus) {
  if (T > kExpandRows || plan_linear(T, K, N, true, cus).expand) return true;
  for (int rows = 16; rows < T; rows += rows < kFewKernelRows ? 16 : 64)
    if (plan_linear(rows, K, N, true, cus).expand) return true;
  return false;
}

static bool linear_shape(int T, const frhip_weight* w) {
  return T >= 0 && T <= 1 << 30 && w->K > 0 && w->K <= kLinearMostK && w->K % 8 == 0 && w->N > 0 && w->N <= kLinearMostN &&
         (size_t)w->K * w->N <= kLinearMostWeight;
}

constexpr int kLinearRows = 2;  // binary16 weights, us: 2 x 4096 x 2048 5.2 in rows, 5.5 as a few rows; 3 and 4 x 2048 x 8192 11.2 and 8.6

static int launch_linear(LinearArgs a, bool u8, void* workspace, hipStream_t st) {
  if (!u8 && a.T <= kLinearRows) return a.T == 1 ? launch_rows<1>(a, st) : launch_rows<2>(a, st);
  const LinearPlan p = plan_linear(a.T, a.K, a.N, u8, compute_units());
  if (!p.few.mt && !p.tiles.rows) return set_error(FRHIP_ESHAPE, "linear: no tiles for this shape");
  if (p.expand) {
    if (!workspace) return set_error(FRHIP_EINVAL, "linear: null workspace");
    if (off_grid(16, {workspace})) return set_error(FRHIP_EINVAL, "linear: workspace must be 16-byte aligned");
    if (int rc = dequant_u8_async(a.w, a.mx, a.rx, a.my, a.ry, static_cast<h1*>(workspace), a.K, a.N, st)) return rc;
    a.w = static_cast<const unsigned char*>(workspace);
    u8 = false;
  }
  if (!p.few.mt && p.codes) {
    const LinearTiles t = {a, p.tiles.a.vw_base[0], p.tiles.a.vw_wide[0], p.tiles.a.vw_maxw};
    if (p.tiles.rows == 128) q8_launch<128>(p.tiles, t, st);
    else q8_launch<64>(p.tiles, t, st);
    return check_launch("linear");
  }
  if (p.few.mt) return u8 ? launch_few<true>(a, p.few, st) : launch_few<false>(a, p.few, st);
  LinearArgs head = a;
  if (p.head) head.T = p.head;
  const int rc = a.K % kLdwBK ? launch_tiles<true>(head, p.tiles, st) : launch_tiles<false>(head, p.tiles, st);
  if (rc || !p.head) return rc;
  const size_t elem = a.out32 ? 4 : 2;
  a.T -= p.head;
  a.x += (size_t)p.head * a.ldx;
  a.y = static_cast<char*>(a.y) + (size_t)p.head * a.ldy * elem;
  if (a.res) a.res = static_cast<const char*>(a.res) + (size_t)p.head * a.ldr * elem;
  return launch_few<false>(a, p.rest, st);
}

}  // namespace frhip

using namespace frhip;

extern "C" size_t frhip_linear_workspace_bytes(int T, const frhip_weight* w) {
  if (!w || T <= 0 || w->dtype != FRHIP_U8 || !linear_shape(T, w) || !expands_up_to(T, w->K, w->N, compute_units()))
    return 0;
  return ((size_t)w->K * w->N * 2 + 255) / 256 * 256;  // the weight in binary16
}

extern "C" int frhip_linear_form(int T, const frhip_weight* w, int compute_units, int* out) {
  if (!w || !out) return set_error(FRHIP_EINVAL, "linear_form: null pointer");
  if (w->dtype != FRHIP_F16 && w->dtype != FRHIP_U8) return set_error(FRHIP_EINVAL, "linear_form: weight dtype must be F16 or U8");
  if (T <= 0 || compute_units < 1 || !linear_shape(T, w)) return set_error(FRHIP_ESHAPE, "linear_form: no such product");
  const bool u8 = w->dtype == FRHIP_U8;
  out[0] = out[1] = out[2] = 0;
  if (!u8 && T <= kLinearRows) return FRHIP_LINEAR_ROWS;
  const LinearPlan p = plan_linear(T, w->K, w->N, u8, compute_units);
  out[0] = p.few.mt ? p.few.mt * 16 : p.tiles.rows;
  out[1] = p.few.mt ? p.few.nt * 16 : p.tiles.a.vw_maxw * 32;
  out[2] = (p.expand ? 1 : 0) + (!p.few.mt && p.head ? 2 : 0);
  return p.few.mt ? FRHIP_LINEAR_FEW : p.codes ? FRHIP_LINEAR_CODES : FRHIP_LINEAR_TILES;
}

extern "C" int frhip_linear(const void* x, int ldx, const frhip_weight* w, const float* bias, int act, const void* residual, int ldr, void* y,
                            int ldy, int T, int out_dtype, void* workspace, frhip_stream s) {
  if (!w || !w->data) return set_error(FRHIP_EINVAL, "linear: null pointer");
  if (out_dtype != FRHIP_F16 && out_dtype != FRHIP_F32) return set_error(FRHIP_EINVAL, "linear: out_dtype must be F16 or F32");
  if (act != FRHIP_ACT_NONE && (act < FRHIP_ACT_SIGMOID || act > FRHIP_ACT_SOFTPLUS)) return set_error(FRHIP_EINVAL, "linear: unknown act");
  if (w->dtype != FRHIP_F16 && w->dtype != FRHIP_U8) return set_error(FRHIP_EINVAL, "linear: weight dtype must be F16 or U8");
  if (w->dtype == FRHIP_U8 && (!w->mx || !w->rx || !w->my || !w->ry)) return set_error(FRHIP_EINVAL, "linear: uint8 weight without mx/rx/my/ry");
  if (!linear_shape(T, w) || ldx > kLinearMostK) return set_error(FRHIP_ESHAPE, "linear: K must be a multiple of 8, T at most 2^30, N 2^24, K N 2^34, rows at most 8388544 elements apart");
  if (ldx < w->K || ldx % 8 != 0 || ldy < w->N || (residual && ldr < w->N)) return set_error(FRHIP_ESHAPE, "linear: rows closer than their elements, or ldx no multiple of 8");
  if (T == 0) return 0;
  if (!x || !y) return set_error(FRHIP_EINVAL, "linear: null pointer");
  const size_t elem = out_dtype == FRHIP_F16 ? 2 : 4, rows = T, K = w->K, N = w->N;
  if (off_grid(16, {x, w->data}) || off_grid(4, {bias}) || off_grid(elem, {residual, y}) || off_grid(4, {w->mx, w->rx, w->my, w->ry}))
    return set_error(FRHIP_EINVAL, "linear: pointer not aligned");
  const size_t ye = ((rows - 1) * ldy + N) * elem;
  auto hits = [&](const void* p, size_t bytes) { return rows_overlap(p, bytes, y, ye, 1, bytes, ye, 1); };
  if (rows_overlap(x, (size_t)ldx * 2, y, ldy * elem, rows, K * 2, N * elem, 1)) return set_error(FRHIP_EINVAL, "linear: y overlaps x");
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
  a.out32 = out_dtype == FRHIP_F32;
  hipStream_t st = static_cast<hipStream_t>(s);
  const bool u8 = w->dtype == FRHIP_U8;
  return launch_linear(a, u8, workspace, st);
}
