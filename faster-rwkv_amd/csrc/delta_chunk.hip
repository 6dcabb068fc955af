// The gated delta rule chunk by chunk, on the matrix units.
//
// In a chunk of 64 rows that begins at the state S, with a_ij the decay from row j to row i, a_i0 that from the chunk's start and k, q of unit length,
//   R_i = b_i (v_i - a_i0 S^T k_i),   U = T R,   T = (1 + L)^-1,   L_ij = b_i a_ij k_i . k_j  (j < i)
//   y_i = scale a_i0 S^T q_i + (P R)_i,   P = A T,   A_ij = scale a_ij q_i . k_j  (j <= i)
//   S' = a_C0 S + sum_i k_i (a_Ci U_i)^T
// T and P do not depend on S: a first launch finds them for all chunks at once; a second one walks the chunks of a prompt, a head and 16 columns of S
// a workgroup, with three products a chunk that wait for each other: [K; Q] S, [T; P] R, K^T U.
//
// The products multiply binary16 with fp32 sums.  What is fp32 goes in as a pair hi + lo, 22 bits and more, scaled by a power of two: rows of T and P, of q
// and k where they are fp32, columns of S, R and U.  Rows of q and k go in as they are but for a power of two, binary16 exactly, and their lengths are made good behind the products.
#include <algorithm>
#include <climits>
#include <cstring>

#include "delta.h"

#pragma clang fp contract(off)

namespace frhip {

constexpr int kChunk = 64;
constexpr float kLeastLog = -1e4f;  // of a row's decay, which is zero there; sums of a chunk's stay exact enough in float64

// Per chunk and head: [T: 6 blocks][P: 6 blocks], a block 32 columns of 16 rows as {hi, lo}[64 lanes] operands; [5][64] row factors; bounds
constexpr int kBlockBytes = 2 * 64 * 16;
constexpr int kTriBytes = 6 * kBlockBytes;
__device__ __forceinline__ constexpr int block_of(int tile, int ks) { return (tile == 3 ? 4 : tile) + ks; }  // tiles 0 and 1 have one block
enum { kRowBeta, kRowK, kRowQ, kRowP, kRowT, kRowKinds };
struct ChunkBounds {
  float key[4], tri[4], back[4];  // of each wave's rows, see the scan
  float keep;                     // the decay of the whole chunk
  int bad;                        // the first row of which something is not finite, or kChunk
  float pad[2];
};
constexpr int kRowsAt = 2 * kTriBytes, kBoundsAt = kRowsAt + kRowKinds * kChunk * 4, kHeadBytes = (kBoundsAt + (int)sizeof(ChunkBounds) + 255) / 256 * 256;

// Per chunk and head of keys: [K][Q], each [4 tiles of 16 rows][steps of 32 dimensions][parts][64 lanes] operands
constexpr size_t key_bytes(int dkp, int parts) { return (size_t)kChunk * dkp * 2 * parts * 2; }

template <class T>
constexpr int kParts = sizeof(T) == 4 ? 2 : 1;

__device__ __forceinline__ f32x4 mfma_h(h8 a, h8 b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }
__device__ __forceinline__ f32x4 mfma_f(float a, float b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x4f32(a, b, c, 0, 0, 0); }

__device__ __forceinline__ float max_across_rows(float v) {  // over the four lanes that share lane % 16
  const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  v = __builtin_fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
  const auto s = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return __builtin_fmaxf(__uint_as_float(s[0]), __uint_as_float(s[1]));
}
__device__ __forceinline__ uint32_t max_across_rows(uint32_t v) {
  const auto r = __builtin_amdgcn_permlane16_swap(v, v, false, false);
  v = max((uint32_t)r[0], (uint32_t)r[1]);
  const auto s = __builtin_amdgcn_permlane32_swap(v, v, false, false);
  return max((uint32_t)s[0], (uint32_t)s[1]);
}
template <class F>
__device__ __forceinline__ float wave_fold(float v, F f) {
#pragma unroll
  for (int m = 1; m < 64; m *= 2) v = f(v, __shfl_xor(v, m));
  return v;
}

// A power of two that takes what is not above `bound` (its bits, sign off) below 2^15, and its reciprocal.  For no bound that is finite: any
__device__ __forceinline__ float scale_for(uint32_t bound) {
  const int field = 268 - (int)(bound >> 23);
  return __uint_as_float((uint32_t)min(field, 253) << 23);
}
__device__ __forceinline__ float inverse_of(float power) { return __uint_as_float((254u << 23) - __float_as_uint(power)); }
__device__ __forceinline__ uint32_t magnitude(float v) { return __float_as_uint(v) & 0x7fffffffu; }
constexpr uint32_t kNotFinite = 0x7f800000u;  // magnitudes from here on

// v as hi + lo
__device__ __forceinline__ void split(float v, h1& hi, h1& lo) {
  asm("" : "+v"(v));  // rounded to fp32 ahead of both conversions: a product that v_fma_mixlo_f16 rounds once gives another hi, now and then
  hi = (h1)v;
  lo = (h1)(v - (float)hi);
}

// ---------------------------------------------------------------------------
// First launch: T, P and the row factors of every chunk and head, and q and k as operands of every chunk and head of keys
// ---------------------------------------------------------------------------
// A tile of 16 rows as operands: lane l has row l % 16, of step ks the dimensions 32 ks + 8 (l / 16) and on, times a power of two that takes the
// row's largest value to [2^8, 2^9), fp32 as hi + lo.  Of the lane's row: the sum of squares, the sum of magnitudes and the largest one of what the operands
// hold, and the power of two; a row with something that is not finite is zero.
template <class T, int KS>
struct KeyTile {
  h8 f[KS][kParts<T>];
  float squares, sum, most, power;
  bool finite;

  __device__ __forceinline__ void load(const T* rows, size_t ld, int row0, int nrows, int dk) {
    const int lane = threadIdx.x & 63, row = row0 + (lane & 15), d0 = (lane >> 4) * 8;
    const bool there = row < nrows;
    const T* const p = rows + (size_t)(there ? row : 0) * ld;
    float v[KS][8];
    uint32_t top = 0;
#pragma unroll
    for (int ks = 0; ks < KS; ks++) {
      const int d = ks * 32 + d0;
      load_group<T, 8>(v[ks], p + (d < dk ? d : 0), there ? dk - d : 0);
#pragma unroll
      for (int i = 0; i < 8; i++) top = max(top, magnitude(v[ks][i]));
    }
    top = max_across_rows(top);
    finite = top < kNotFinite;
    power = __uint_as_float((uint32_t)max(1, min(262 - (int)(top >> 23), 127 + 60)) << 23);  // 2^60 at most: its square times norm_eps stays in fp32
    squares = sum = 0.f;
#pragma unroll
    for (int ks = 0; ks < KS; ks++)
#pragma unroll
      for (int i = 0; i < 8; i++) {
        const float x = finite ? v[ks][i] * power : 0.f;
        squares = __builtin_fmaf(x, x, squares);
        sum += __builtin_fabsf(x);
        if constexpr (kParts<T> == 2) {
          h1 hi, lo;
          split(x, hi, lo);
          f[ks][0][i] = hi;
          f[ks][1][i] = lo;
        } else {
          f[ks][0][i] = (h1)x;
        }
      }
    squares = add_across_32(add_across_16(squares));
    sum = add_across_32(add_across_16(sum));
    most = finite ? __uint_as_float(top) * power : 0.f;
  }
  // what the operands' row is to be multiplied by
  __device__ __forceinline__ float factor(float eps) const {
    if (eps < 0.f) return inverse_of(power);
    return __builtin_amdgcn_rsqf(__builtin_fmaf(eps * power, power, squares));
  }
  __device__ __forceinline__ void store(h8* to) const {
#pragma unroll
    for (int ks = 0; ks < KS; ks++)
#pragma unroll
      for (int n = 0; n < kParts<T>; n++) to[(ks * kParts<T> + n) * 64 + (threadIdx.x & 63)] = f[ks][n];
  }
};

template <class T, int KS>
__device__ __forceinline__ f32x4 gram(const KeyTile<T, KS>& a, const KeyTile<T, KS>& b) {
  f32x4 s = {0.f, 0.f, 0.f, 0.f};
  if constexpr (kParts<T> == 2) {
#pragma unroll
    for (int ks = 0; ks < KS; ks++) {
      s = mfma_h(a.f[ks][1], b.f[ks][0], s);
      s = mfma_h(a.f[ks][0], b.f[ks][1], s);
    }
  }
#pragma unroll
  for (int ks = 0; ks < KS; ks++) s = mfma_h(a.f[ks][0], b.f[ks][0], s);
  return s;
}

constexpr int kLd = kChunk + 4;  // of a matrix in LDS: 16 rows apart, 16 bytes each, on all banks

// The operands of 16 rows of a lower triangular matrix m, by rows' powers of two; returns the sum of magnitudes of the lane's row
__device__ __forceinline__ float store_tri(const float (*m)[kLd], int tile, char* to, float* inv) {
  const int lane = threadIdx.x & 63, row = tile * 16 + (lane & 15), g = lane >> 4;
  float v[2][8], sum = 0.f;
  uint32_t top = 0;
#pragma unroll
  for (int ks = 0; ks < 2; ks++) {
    const bool there = 2 * ks + (g >> 1) <= tile;  // the others were never written
#pragma unroll
    for (int i = 0; i < 8; i += 4) {
      f32x4 t = {0.f, 0.f, 0.f, 0.f};
      if (there) t = *reinterpret_cast<const f32x4*>(&m[row][ks * 32 + g * 8 + i]);
#pragma unroll
      for (int e = 0; e < 4; e++) {
        v[ks][i + e] = t[e];
        top = max(top, magnitude(t[e]));
        sum += __builtin_fabsf(t[e]);
      }
    }
  }
  const float power = scale_for(max_across_rows(top));
  *inv = inverse_of(power);
#pragma unroll
  for (int ks = 0; ks < 2; ks++) {
    if (ks * 2 > tile) break;
    h8 hi, lo;
#pragma unroll
    for (int i = 0; i < 8; i++) {
      h1 a, b;
      split(v[ks][i] * power, a, b);
      hi[i] = a;
      lo[i] = b;
    }
    h8* const block = reinterpret_cast<h8*>(to + block_of(tile, ks) * kBlockBytes);
    block[lane] = hi;
    block[64 + lane] = lo;
  }
  return add_across_32(add_across_16(sum));
}

// blockIdx.x: a chunk, blockIdx.y: a head.  Wave w has the rows 16 w to 16 w + 15 of every matrix, but of T behind its diagonal the columns.
template <class T, int KS>
__global__ __launch_bounds__(256) void delta_prep_kernel(DeltaArgs<T> a, DeltaTable tab, char* keys, char* heads) {
  __shared__ __attribute__((aligned(16))) float Lm[kChunk][kLd], Am[kChunk][kLd], Tm[kChunk][kLd];
  __shared__ double Gs[kChunk];
  __shared__ float fk[kChunk], fq[kChunk], beta[kChunk], l1[kChunk];
  __shared__ int spoilt[kChunk];
  const int lane = threadIdx.x & 63, c = lane & 15, g = lane >> 4, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int cj = blockIdx.x, head = blockIdx.y, kh = head / a.share;
  const int i0 = find_seq(a.nseq, cj, [&](int k) { return tab.chunk[k]; });
  const int t0 = tab.start[i0] + (cj - tab.chunk[i0]) * kChunk, len = min(tab.end[i0] - t0, kChunk);
  const T* const kr = a.k + (size_t)t0 * a.ldk + (size_t)kh * a.dk;
  const T* const qr = a.q + (size_t)t0 * a.ldq + (size_t)kh * a.dk;
  KeyTile<T, KS> K, Q;
  K.load(kr, a.ldk, w * 16, len, a.dk);
  Q.load(qr, a.ldq, w * 16, len, a.dk);
  if (head % a.share == 0) {
    constexpr int tile = KS * kParts<T> * 64;
    h8* const to = reinterpret_cast<h8*>(keys + ((size_t)cj * (a.heads / a.share) + kh) * key_bytes(KS * 32, kParts<T>));
    K.store(to + w * tile);
    Q.store(to + (4 + w) * tile);
  }
  if (g == 0) {
    const float f = K.factor(a.eps);
    fk[w * 16 + c] = f;
    fq[w * 16 + c] = (Q.finite ? Q.factor(a.eps) : __builtin_nanf("")) * a.scale;
    l1[w * 16 + c] = K.sum;
    spoilt[w * 16 + c] = !K.finite || magnitude(f) >= kNotFinite;  // (nothing divided by its length)
  }
  __syncthreads();
  // a lane a row, in every wave alike
  int bad;
  double G;
  {
    const bool there = lane < len;
    const size_t t = t0 + (there ? lane : 0);
    const float rate = a.A ? finite_rate(a.A[head]) : 1.f, bias = a.dt_bias ? a.dt_bias[head] : 0.f;
    const float lg = there ? log_decay(a, (float)a.dt[t * a.lddt + head], rate, bias) : 0.f, raw = there ? (float)a.beta[t * a.ldbeta + head] : 0.f;
    float b = there ? (a.sigmoid ? sigmoid_f<true>(raw) : raw) : 0.f;
    const unsigned long long off = __ballot(there && (spoilt[lane] || magnitude(b) >= kNotFinite || !(lg < __builtin_inff())));
    bad = off ? __builtin_ctzll(off) : kChunk;
    G = lane < bad ? (double)__builtin_fmaxf(lg, kLeastLog) : 0.0;
    if (lane >= bad) b = 0.f;
#pragma unroll
    for (int m = 1; m < 64; m *= 2) {
      const double up = __shfl_up(G, m);
      if (lane >= m) G += up;
    }
    if (w == 0) {
      Gs[lane] = G;
      beta[lane] = b;
    }
  }
  __syncthreads();
  const int r0 = w * 16 + g * 4;  // the lane's rows of a tile of results, whose column is c
  double Gi[4];
  float bi[4], fi[4], qi[4];
#pragma unroll
  for (int r = 0; r < 4; r++) {
    Gi[r] = Gs[r0 + r];
    bi[r] = beta[r0 + r];
    fi[r] = fk[r0 + r];
    qi[r] = fq[r0 + r];
  }
  for (int j = 0; j <= w; j++) {
    KeyTile<T, KS> B;
    if (j < w) B.load(kr, a.ldk, j * 16, len, a.dk);
    else B = K;
    const f32x4 kk = gram<T, KS>(K, B), qk = gram<T, KS>(Q, B);
    const int col = j * 16 + c;
    const double Gj = Gs[col];
    const float fj = fk[col];
#pragma unroll
    for (int r = 0; r < 4; r++) {
      const int row = r0 + r;
      const float d = decay_f((float)(Gi[r] - Gj)) * fj;
      Lm[row][col] = col < row && row < bad ? bi[r] * fi[r] * (d * kk[r]) : 0.f;
      Am[row][col] = col <= row && row < bad ? qi[r] * (d * qk[r]) : 0.f;
    }
  }
  // (a wave's own rows of Lm and Am: written and read by the same wave, in order)
  __builtin_amdgcn_wave_barrier();
  {  // T on its diagonal, column c of 16, row by row
    float t[16];
#pragma unroll
    for (int i = 0; i < 16; i++) {
      float s = i == c ? 1.f : 0.f;
#pragma unroll
      for (int j = 0; j < i; j++) s = __builtin_fmaf(-Lm[w * 16 + i][w * 16 + j], t[j], s);
      t[i] = s;
    }
    if (g == 0) {
#pragma unroll
      for (int i = 0; i < 16; i++) Tm[w * 16 + i][w * 16 + c] = t[i];
    }
  }
  __syncthreads();
  // T behind its diagonal, wave j the columns of tile j: T_ij = -T_ii sum_m L_im T_mj (m = j to i - 1).  An operand of results as they lie (row 4 g + s of
  // step s) goes with the columns 4 g + s of the other matrix.
  f32x4 X[4];
#pragma unroll
  for (int s = 0; s < 4; s++) X[0][s] = Tm[w * 16 + g * 4 + s][w * 16 + c];  // X[n]: tile w + n
#pragma unroll
  for (int n = 1; n < 4; n++) {
    if (w + n > 3) break;
    const int i = w + n;
    f32x4 acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int m = 0; m < n; m++) {
      const f32x4 l = *reinterpret_cast<const f32x4*>(&Lm[i * 16 + c][(w + m) * 16 + g * 4]);
#pragma unroll
      for (int s = 0; s < 4; s++) acc = mfma_f(l[s], X[m][s], acc);
    }
    const f32x4 ti = *reinterpret_cast<const f32x4*>(&Tm[i * 16 + c][i * 16 + g * 4]);
    f32x4 x = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int s = 0; s < 4; s++) x = mfma_f(ti[s], -acc[s], x);
    X[n] = x;
#pragma unroll
    for (int s = 0; s < 4; s++) Tm[i * 16 + g * 4 + s][w * 16 + c] = x[s];
  }
  __syncthreads();
  // P = A T, the wave's rows
  f32x4 Pt[4];
#pragma unroll
  for (int j = 0; j < 4; j++) {
    if (j > w) break;
    f32x4 acc = {0.f, 0.f, 0.f, 0.f};
    for (int m = j; m <= w; m++) {
      const f32x4 am = *reinterpret_cast<const f32x4*>(&Am[w * 16 + c][m * 16 + g * 4]);
#pragma unroll
      for (int s = 0; s < 4; s++) acc = mfma_f(am[s], Tm[m * 16 + g * 4 + s][j * 16 + c], acc);
    }
    Pt[j] = acc;
  }
  __builtin_amdgcn_wave_barrier();
#pragma unroll
  for (int j = 0; j < 4; j++) {
    if (j > w) break;
#pragma unroll
    for (int r = 0; r < 4; r++) Am[r0 + r][j * 16 + c] = Pt[j][r];
  }
  __builtin_amdgcn_wave_barrier();
  char* const out = heads + ((size_t)cj * a.heads + head) * kHeadBytes;
  float invt, invp;
  const float rowsum = store_tri(Tm, w, out, &invt);
  store_tri(Am, w, out + kTriBytes, &invp);
  // of row 16 w + c
  const int row = w * 16 + c;
  const double Grow = Gs[row], Gend = Gs[kChunk - 1];
  const float from = decay_f((float)Grow), back = row < bad ? decay_f((float)(Gend - Grow)) * fk[row] : 0.f;
  const float key = row < bad ? beta[row] * from * fk[row] : 0.f;
  float* const rows = reinterpret_cast<float*>(out + kRowsAt);
  if (g == 0) {
    rows[kRowBeta * kChunk + row] = beta[row];
    rows[kRowK * kChunk + row] = key;
    rows[kRowQ * kChunk + row] = fq[row] * from;
    rows[kRowP * kChunk + row] = invp;
    rows[kRowT * kChunk + row] = back * invt;
  }
  const auto larger = [](float x, float y) { return __builtin_fmaxf(x, y); };
  const float bkey = wave_fold(__builtin_fabsf(key) * l1[row], larger), btri = wave_fold(__builtin_fabsf(back) * rowsum, larger);
  const float bback = wave_fold(g == 0 ? K.most * __builtin_fabsf(back) * rowsum : 0.f, [](float x, float y) { return x + y; });
  if (lane == 0) {
    ChunkBounds* const b = reinterpret_cast<ChunkBounds*>(out + kBoundsAt);
    b->key[w] = bkey;
    b->tri[w] = btri;
    b->back[w] = bback;
    if (w == 0) {
      b->keep = decay_f((float)Gend);
      b->bad = bad;
    }
  }
}

// ---------------------------------------------------------------------------
// Second launch: the chunks of a prompt one after another
// ---------------------------------------------------------------------------
// LDS alone: loads that are on their way to registers stay on it
__device__ __forceinline__ void lds_barrier() {
  asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}

typedef short s4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) s4 lds_s4;
// Four rows of 16 columns of a matrix in LDS by the 16 lanes of a row of lanes: lane p gives row p / 4, columns 4 (p % 4) and on, and gets column p
__device__ __forceinline__ h4 read_columns(const h1* p) {
  return __builtin_bit_cast(h4, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4*)(void*)p));
}

template <class T, int KS, int NT>
struct ScanLds {
  static constexpr int DK = KS * 32, SL = DK + 8, RL = kChunk + 8, KL = DK + 16;
  h1 S[2][NT * 16][SL], R[2][NT * 16][RL], U[2][NT * 16][RL];  // [column][row], hi and lo
  h1 K[kParts<T>][kChunk][KL];
  uint32_t smost[NT * 16][4], vmost[NT * 16][4];  // of each wave's rows
};

// blockIdx.x: a prompt, a head and 16 NT columns of its state.  A wave has 16 rows of a chunk, of K, Q, T and P, and a quarter of the rows of S.  A lane has
// column c of every tile of 16 columns, rows 4 g and on of one of 16 rows.
//
// The powers of two by which columns are scaled come from bounds, a step ahead of the values and without waiting for the other waves' values:
//   |R| <= max |b v| + max_i |b_i a_i0| |k_i|_1 max |S|,   |a U| <= max_i |a_Ci| |T_i|_1 max |R|,   |S'| <= a max |S| + sum_i max_d |k_id| |a_Ci| |T_i|_1 max |R|
// They may be 2^16 too high before a pair holds a column's largest value to less than fp32 does.
template <class T, int KS, int NT>
__global__ __launch_bounds__(256) void delta_scan_kernel(DeltaArgs<T> a, DeltaTable tab, const char* keys, const char* heads) {
  constexpr int NK = kParts<T>, ST = KS / 2;  // ST: tiles of 16 rows of S of a wave
  typedef ScanLds<T, KS, NT> Lds;
  __shared__ __attribute__((aligned(16))) Lds lds;
  const int lane = threadIdx.x & 63, c = lane & 15, g = lane >> 4, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int slices = (a.dv + NT * 16 - 1) / (NT * 16), per = a.heads * slices;
  const int i0 = blockIdx.x / per, head = (blockIdx.x - i0 * per) / slices, col0 = (blockIdx.x - i0 * per - head * slices) * (NT * 16), kh = head / a.share;
  const int begin = tab.start[i0], end = tab.end[i0], nchunk = tab.chunk[i0 + 1] - tab.chunk[i0];
  const size_t st = ((size_t)tab.seq[i0] * a.heads + head) * a.dk * a.dv;
  const float* const from = i0 == 0 && tab.ahead ? a.state_out : a.state;
  int col[NT];
  bool mine[NT];
  f32x4 S[ST][NT];
  const int d0 = w * (ST * 16) + g * 4;  // row of S[.][.][0], 16 rows a tile
#pragma unroll
  for (int n = 0; n < NT; n++) {
    mine[n] = col0 + n * 16 + c < a.dv;
    col[n] = mine[n] ? col0 + n * 16 + c : a.dv - 1;
#pragma unroll
    for (int t = 0; t < ST; t++)
#pragma unroll
      for (int r = 0; r < 4; r++) {
        const int d = d0 + t * 16 + r;
        S[t][n][r] = d < a.dk ? from[st + (size_t)d * a.dv + col[n]] : 0.f;
      }
  }
  h8 Kf[KS][NK], Qf[KS][NK], Tf[2][2], Pf[2][2];
  T v[NT][4];
  f32x4 rb, rk, rq, rp, rt;
  const int nkh = a.heads / a.share;
  auto load_keys = [&](int j) {
    const h8* const p = reinterpret_cast<const h8*>(keys + ((size_t)j * nkh + kh) * key_bytes(KS * 32, NK)) + lane;
#pragma unroll
    for (int ks = 0; ks < KS; ks++)
#pragma unroll
      for (int n = 0; n < NK; n++) {
        Kf[ks][n] = p[((w * KS + ks) * NK + n) * 64];
        Qf[ks][n] = p[(((4 + w) * KS + ks) * NK + n) * 64];
      }
  };
  auto load_values = [&](int t0) {
#pragma unroll
    for (int r = 0; r < 4; r++) {
      const int t = t0 + w * 16 + g * 4 + r;
#pragma unroll
      for (int n = 0; n < NT; n++) v[n][r] = t < end ? a.v[(size_t)t * a.ldv + (size_t)head * a.dv + col[n]] : (T)0.f;
    }
  };
  auto head_of = [&](int j) { return heads + ((size_t)j * a.heads + head) * kHeadBytes; };
  auto load_tri = [&](int j) {
    const char* const p = head_of(j);
#pragma unroll
    for (int ks = 0; ks < 2; ks++)
#pragma unroll
      for (int n = 0; n < 2; n++) {
        if (2 * ks > w) break;
        Tf[ks][n] = reinterpret_cast<const h8*>(p + block_of(w, ks) * kBlockBytes)[n * 64 + lane];
        Pf[ks][n] = reinterpret_cast<const h8*>(p + kTriBytes + block_of(w, ks) * kBlockBytes)[n * 64 + lane];
      }
  };
  auto row_factors = [&](int j, int kind) { return *reinterpret_cast<const f32x4*>(head_of(j) + kRowsAt + (kind * kChunk + w * 16 + g * 4) * 4); };
  const int first = tab.chunk[i0];
  if (nchunk > 0) {
    load_keys(first);
    load_values(begin);
    load_tri(first);
    rb = row_factors(first, kRowBeta), rk = row_factors(first, kRowK), rq = row_factors(first, kRowQ);
    rp = row_factors(first, kRowP), rt = row_factors(first, kRowT);
  }
  uint32_t sbound[NT];  // of the columns of S; the first chunk's is its own largest value
#pragma unroll
  for (int n = 0; n < NT; n++) {
    uint32_t m = 0;
#pragma unroll
    for (int t = 0; t < ST; t++)
#pragma unroll
      for (int r = 0; r < 4; r++) m = max(m, magnitude(S[t][n][r]));
    m = max_across_rows(m);
    if (g == 0) lds.smost[n * 16 + c][w] = m;
  }
  lds_barrier();
#pragma unroll
  for (int n = 0; n < NT; n++) {
    const u32x4 m = *reinterpret_cast<const u32x4*>(lds.smost[n * 16 + c]);
    sbound[n] = max(max(m[0], m[1]), max(m[2], m[3]));
  }
  lds_barrier();
  for (int j = 0; j < nchunk; j++) {
    const int t0 = begin + j * kChunk, next = first + (j + 1 < nchunk ? j + 1 : j);
    const ChunkBounds& bounds = *reinterpret_cast<const ChunkBounds*>(head_of(first + j) + kBoundsAt);
    const float keep = bounds.keep, bkey = __builtin_fmaxf(__builtin_fmaxf(bounds.key[0], bounds.key[1]), __builtin_fmaxf(bounds.key[2], bounds.key[3]));
    const float btri = __builtin_fmaxf(__builtin_fmaxf(bounds.tri[0], bounds.tri[1]), __builtin_fmaxf(bounds.tri[2], bounds.tri[3]));
    const float bback = bounds.back[0] + bounds.back[1] + bounds.back[2] + bounds.back[3];
    const int bad = bounds.bad;
    float sinv[NT], bv[NT][4];
    // S to LDS, and the largest values of S and b v
#pragma unroll
    for (int n = 0; n < NT; n++) {
      const float power = scale_for(sbound[n]);
      sinv[n] = inverse_of(power);
      uint32_t m = 0, mv = 0;
#pragma unroll
      for (int t = 0; t < ST; t++) {
        h4 hi, lo;
#pragma unroll
        for (int r = 0; r < 4; r++) {
          h1 x, y;
          m = max(m, magnitude(S[t][n][r]));
          split(S[t][n][r] * power, x, y);
          hi[r] = x;
          lo[r] = y;
        }
        *reinterpret_cast<h4*>(&lds.S[0][n * 16 + c][d0 + t * 16]) = hi;
        *reinterpret_cast<h4*>(&lds.S[1][n * 16 + c][d0 + t * 16]) = lo;
      }
#pragma unroll
      for (int r = 0; r < 4; r++) {
        bv[n][r] = rb[r] * (float)v[n][r];
        mv = max(mv, magnitude(bv[n][r]));
      }
      m = max_across_rows(m);
      mv = max_across_rows(mv);
      if (g == 0) {
        lds.smost[n * 16 + c][w] = m;
        lds.vmost[n * 16 + c][w] = mv;
      }
    }
    lds_barrier();
    // [K; Q] S
    f32x4 ks_[NT], qs[NT];
#pragma unroll
    for (int n = 0; n < NT; n++) {
      ks_[n] = qs[n] = (f32x4){0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int ks = 0; ks < KS; ks++) {
        const h8 hi = *reinterpret_cast<const h8*>(&lds.S[0][n * 16 + c][ks * 32 + g * 8]), lo = *reinterpret_cast<const h8*>(&lds.S[1][n * 16 + c][ks * 32 + g * 8]);
        ks_[n] = mfma_h(Kf[ks][0], lo, ks_[n]);
        qs[n] = mfma_h(Qf[ks][0], lo, qs[n]);
        if constexpr (NK == 2) {
          ks_[n] = mfma_h(Kf[ks][1], hi, ks_[n]);
          qs[n] = mfma_h(Qf[ks][1], hi, qs[n]);
        }
        ks_[n] = mfma_h(Kf[ks][0], hi, ks_[n]);
        qs[n] = mfma_h(Qf[ks][0], hi, qs[n]);
      }
    }
#pragma unroll
    for (int ks = 0; ks < KS; ks++)
#pragma unroll
      for (int n = 0; n < NK; n++) *reinterpret_cast<h8*>(&lds.K[n][w * 16 + c][ks * 32 + g * 8]) = Kf[ks][n];
    load_keys(next);
    int spoilt[NT];  // the column's first row of which something is not finite
    bool any = bad < kChunk;
    float rinv[NT], upower[NT], uinv[NT];
#pragma unroll
    for (int n = 0; n < NT; n++) {
      const u32x4 ms = *reinterpret_cast<const u32x4*>(lds.smost[n * 16 + c]), mv = *reinterpret_cast<const u32x4*>(lds.vmost[n * 16 + c]);
      const uint32_t sm = max(max(ms[0], ms[1]), max(ms[2], ms[3]));
      uint32_t vm = max(max(mv[0], mv[1]), max(mv[2], mv[3]));
      spoilt[n] = bad;
      if (__ballot(vm >= kNotFinite)) {  // seldom: every wave looks for the first such value itself
        if (vm >= kNotFinite) {
          const float* const b = reinterpret_cast<const float*>(head_of(first + j) + kRowsAt) + kRowBeta * kChunk;
          vm = 0;
          for (int r = min(end - t0, kChunk) - 1; r >= 0; r--) {
            const uint32_t m = magnitude(b[r] * (float)a.v[(size_t)(t0 + r) * a.ldv + (size_t)head * a.dv + col[n]]);
            if (m >= kNotFinite) spoilt[n] = min(spoilt[n], r);
            else vm = max(vm, m);
          }
#pragma unroll
          for (int r = 0; r < 4; r++)
            if (magnitude(bv[n][r]) >= kNotFinite) bv[n][r] = 0.f;
        }
        any = true;
      }
      const float rbound = __builtin_fmaf(bkey, __uint_as_float(sm), __uint_as_float(vm)), ubound = btri * rbound;
      const float rpower = scale_for(magnitude(rbound));
      rinv[n] = inverse_of(rpower);
      upower[n] = scale_for(magnitude(ubound));
      uinv[n] = inverse_of(upower[n]);
      sbound[n] = magnitude(__builtin_fmaf(keep, __uint_as_float(sm), bback * rbound));
      h4 hi, lo;
#pragma unroll
      for (int r = 0; r < 4; r++) {
        h1 x, y;
        split((bv[n][r] - rk[r] * (sinv[n] * ks_[n][r])) * rpower, x, y);
        hi[r] = x;
        lo[r] = y;
      }
      *reinterpret_cast<h4*>(&lds.R[0][n * 16 + c][w * 16 + g * 4]) = hi;
      *reinterpret_cast<h4*>(&lds.R[1][n * 16 + c][w * 16 + g * 4]) = lo;
    }
    if (j + 1 < nchunk) load_values(t0 + kChunk);
    rb = row_factors(next, kRowBeta), rk = row_factors(next, kRowK);
    lds_barrier();
    // [T; P] R
    f32x4 tr[NT], pr[NT];
#pragma unroll
    for (int n = 0; n < NT; n++) {
      tr[n] = pr[n] = (f32x4){0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int ks = 0; ks < 2; ks++) {
        if (2 * ks > w) break;
        const h8 hi = *reinterpret_cast<const h8*>(&lds.R[0][n * 16 + c][ks * 32 + g * 8]), lo = *reinterpret_cast<const h8*>(&lds.R[1][n * 16 + c][ks * 32 + g * 8]);
        tr[n] = mfma_h(Tf[ks][0], lo, tr[n]);
        pr[n] = mfma_h(Pf[ks][0], lo, pr[n]);
        tr[n] = mfma_h(Tf[ks][1], hi, tr[n]);
        pr[n] = mfma_h(Pf[ks][1], hi, pr[n]);
        tr[n] = mfma_h(Tf[ks][0], hi, tr[n]);
        pr[n] = mfma_h(Pf[ks][0], hi, pr[n]);
      }
      h4 hi, lo;
      const float to = rinv[n] * upower[n];
#pragma unroll
      for (int r = 0; r < 4; r++) {
        h1 x, y;
        split(rt[r] * (to * tr[n][r]), x, y);
        hi[r] = x;
        lo[r] = y;
      }
      *reinterpret_cast<h4*>(&lds.U[0][n * 16 + c][w * 16 + g * 4]) = hi;
      *reinterpret_cast<h4*>(&lds.U[1][n * 16 + c][w * 16 + g * 4]) = lo;
    }
    load_tri(next);
    rt = row_factors(next, kRowT);
    lds_barrier();
    // S' = keep S + K^T U
    f32x4 ku[ST][NT];
#pragma unroll
    for (int t = 0; t < ST; t++)
#pragma unroll
      for (int n = 0; n < NT; n++) ku[t][n] = (f32x4){0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int ks = 0; ks < 2; ks++) {
      h8 hi[NT], lo[NT];
#pragma unroll
      for (int n = 0; n < NT; n++) {
        hi[n] = *reinterpret_cast<const h8*>(&lds.U[0][n * 16 + c][ks * 32 + g * 8]);
        lo[n] = *reinterpret_cast<const h8*>(&lds.U[1][n * 16 + c][ks * 32 + g * 8]);
      }
#pragma unroll
      for (int t = 0; t < ST; t++) {
        h8 kt[NK];
#pragma unroll
        for (int p = 0; p < NK; p++) {
          const h1* const at = &lds.K[p][ks * 32 + g * 8 + c / 4][w * (ST * 16) + t * 16 + (c & 3) * 4];
          const h4 x = read_columns(at), y = read_columns(at + 4 * Lds::KL);
          kt[p] = __builtin_shufflevector(x, y, 0, 1, 2, 3, 4, 5, 6, 7);
        }
#pragma unroll
        for (int n = 0; n < NT; n++) {
          ku[t][n] = mfma_h(kt[0], lo[n], ku[t][n]);
          if constexpr (NK == 2) ku[t][n] = mfma_h(kt[1], hi[n], ku[t][n]);
          ku[t][n] = mfma_h(kt[0], hi[n], ku[t][n]);
        }
      }
    }
#pragma unroll
    for (int n = 0; n < NT; n++) {
#pragma unroll
      for (int t = 0; t < ST; t++)
#pragma unroll
        for (int r = 0; r < 4; r++) S[t][n][r] = __builtin_fmaf(uinv[n], ku[t][n][r], keep * S[t][n][r]);
      float y[4];
#pragma unroll
      for (int r = 0; r < 4; r++) y[r] = __builtin_fmaf(rq[r], sinv[n] * qs[n][r], rp[r] * (rinv[n] * pr[n][r]));
      if (any) {
        const float nan = __builtin_nanf("");
#pragma unroll
        for (int r = 0; r < 4; r++)
          if (w * 16 + g * 4 + r >= spoilt[n]) y[r] = nan;
        if (spoilt[n] < kChunk) {
#pragma unroll
          for (int t = 0; t < ST; t++) S[t][n] = (f32x4){nan, nan, nan, nan};
        }
      }
#pragma unroll
      for (int r = 0; r < 4; r++) {
        const int t = t0 + w * 16 + g * 4 + r;
        if (mine[n] && t < end) a.y[(size_t)t * a.ldy + (size_t)head * a.dv + col[n]] = (T)y[r];
      }
    }
    rq = row_factors(next, kRowQ), rp = row_factors(next, kRowP);
  }
#pragma unroll
  for (int n = 0; n < NT; n++)
#pragma unroll
    for (int t = 0; t < ST; t++)
#pragma unroll
      for (int r = 0; r < 4; r++) {
        const int d = d0 + t * 16 + r;
        if (mine[n] && d < a.dk) a.state_out[st + (size_t)d * a.dv + col[n]] = S[t][n][r];
      }
}

// ---------------------------------------------------------------------------
// Host side
// ---------------------------------------------------------------------------
constexpr size_t kPassBytes = (size_t)256 << 20;  // scratch of a pair of launches, about: longer calls go out in several
static int key_steps(int dk) { return dk <= 64 ? 2 : dk <= 128 ? 4 : 8; }
static size_t chunk_bytes(int heads, int key_heads, int dk, int parts) {
  return (size_t)heads * kHeadBytes + (size_t)key_heads * key_bytes(key_steps(dk) * 32, parts);
}
// Chunks of a pair of launches: prompts have kDeltaChunkLeast rows at least, so there are no more chunks than rows / kDeltaChunkLeast + 1
static size_t most_chunks(size_t per, int T) {
  const size_t by_rows = (size_t)T / kDeltaChunkLeast + 1, by_bytes = std::max<size_t>(kPassBytes / per, 16);
  return std::min(by_rows, by_bytes);
}

size_t delta_chunk_bytes(const frhip_delta& p, int elem, int T) {
  if (T < kDeltaChunkLeast) return 0;
  const size_t per = chunk_bytes(p.heads, p.key_heads, p.key_dim, elem == 4 ? 2 : 1);
  return most_chunks(per, T) * per;
}

template <class T, int KS>
static int chunk_launch(const DeltaArgs<T>& a, const DeltaTable& tab, char* keys, char* heads, hipStream_t st) {
  const int chunks = tab.chunk[a.nseq], slices = (a.dv + 15) / 16;
  if (chunks > 0) {
    hipLaunchKernelGGL((delta_prep_kernel<T, KS>), dim3(chunks, a.heads), dim3(256), 0, st, a, tab, keys, heads);
    if (int rc = check_launch("delta_seq")) return rc;
  }
  hipLaunchKernelGGL((delta_scan_kernel<T, KS, 1>), dim3(a.nseq * a.heads * slices), dim3(256), 0, st, a, tab, keys, heads);
  return check_launch("delta_seq");
}

template <class T>
int delta_chunk_run(const DeltaArgs<T>& args, const int* seqs, int nseq, const int32_t* start, int rows, void* workspace, hipStream_t st) {
  DeltaArgs<T> a = args;
  const int nkh = a.heads / a.share, steps = key_steps(a.dk);
  const size_t per = chunk_bytes(a.heads, nkh, a.dk, kParts<T>), most = most_chunks(per, rows);
  const int together = std::min(kSeqTable, (1 << 23) / (a.heads * ((a.dv + 15) / 16)));  // prompts of a launch, which has less than 2^32 threads
  char* const keys = static_cast<char*>(workspace);
  char* const heads = keys + most * nkh * key_bytes(steps * 32, kParts<T>);
  DeltaTable tab;
  memset(&tab, 0, sizeof(tab));
  int i = 0, done = 0;  // prompt, and its chunks that have gone out
  while (i < nseq) {
    a.nseq = 0;
    tab.ahead = done > 0;
    size_t left = most;
    while (i < nseq && left > 0 && a.nseq < together) {
      const int s = seqs[i], len = start[s + 1] - start[s], chunks = (len - 1) / kChunk + 1 - done;
      const int now = (size_t)chunks < left ? chunks : (int)left;
      tab.start[a.nseq] = start[s] + done * kChunk;
      tab.end[a.nseq] = now == chunks ? start[s + 1] : tab.start[a.nseq] + now * kChunk;
      tab.seq[a.nseq] = s;
      tab.chunk[a.nseq + 1] = tab.chunk[a.nseq] + now;
      a.nseq++;
      left -= now;
      if (now == chunks) i++, done = 0;
      else done += now;
    }
    int rc;
    if (steps == 2) rc = chunk_launch<T, 2>(a, tab, keys, heads, st);
    else if (steps == 4) rc = chunk_launch<T, 4>(a, tab, keys, heads, st);
    else rc = chunk_launch<T, 8>(a, tab, keys, heads, st);
    if (rc) return rc;
  }
  return 0;
}
template int delta_chunk_run<h1>(const DeltaArgs<h1>&, const int*, int, const int32_t*, int, void*, hipStream_t);
template int delta_chunk_run<float>(const DeltaArgs<float>&, const int*, int, const int32_t*, int, void*, hipStream_t);

}  // namespace frhip
