// The gated delta rule chunk by chunk, on the matrix units.
//
// In a chunk of 64 rows that begins at the state S, with a_ij the decay from row j to row i, a_i0 that from the chunk's start, a_Ci that to its end and k, q of
// unit length, the rows write the values U:
//   R_i = b_i (v_i - a_i0 S^T k_i),   U = T R,   T = (1 + L)^-1,   L_ij = b_i a_ij k_i . k_j  (j < i)
//   y_i = scale a_i0 S^T q_i + (P R)_i,   P = A T,   A_ij = scale a_ij q_i . k_j  (j <= i)
//   S' = a_C0 S + W R,   W = sum_i k_i (a_Ci T_i)^T
// P and W do not depend on S: a first launch finds them for all chunks at once; a second one walks the chunks of a prompt, a head and 16 columns of S
// a workgroup, with two products a chunk that wait for each other: [K; Q] S and [W; P] R.
//
// The products multiply binary16 with fp32 sums.  What is fp32 goes in as a pair hi + lo, scaled by a power of two: rows of W and P, of q
// and k where they are fp32, columns of S and R.  Where a row or column has decays in it (W, P, R, S) lo goes in times 2^11, in sums of its own: a pair is
// 22 bits and more of what is within 2^29 of the largest, and off by 2^-51 of that below it (without the 2^11, 2^18 and 2^-40).  Where rows of R are so far below
// their column's bound that results would show it, they go token by token (see the scan).
// Rows of k go in as they are but for a power of two, those of q as they are, and their lengths are made good behind the products.
#include <algorithm>
#include <cstring>

#include "delta.h"

#pragma clang fp contract(off)

namespace frhip {

constexpr int kChunk = 64;
constexpr int kXcds = 8;
constexpr float kLeastLog = -1e4f;  // of a row's decay, which is zero there; sums of a chunk's stay exact enough in float64

// Per chunk and head: P, W, the rows' factors, W's rows' factors, bounds.  A block is 64 columns' half of 16 rows as {hi, lo}[64 lanes] operands: lane l has
// row l % 16, and of block ks the columns 32 ks + 4 (l / 16) and on and those 16 further, four each: as the results lie that it is made of.
constexpr int kBlockBytes = 2 * 64 * 16;
__device__ __forceinline__ constexpr int block_of(int tile, int ks) { return (tile == 3 ? 4 : tile) + ks; }  // of P; its tiles 0 and 1 have one
constexpr int kTriBytes = 6 * kBlockBytes;
enum { kRowBeta, kRowK, kRowQ, kRowP, kRowKeep, kRowKinds };  // kRowKeep: a row's own decay; -1 for none, or from what is not finite on
struct ChunkBounds {
  float key, back, both;  // see the scan
  float keep;             // the decay of the whole chunk
  int bad;                // the first row of which something is not finite, or kChunk
  int none[3];
};
template <int KS>
struct HeadLayout {
  static constexpr int W = kTriBytes, rows = W + KS * 2 * 2 * kBlockBytes, back = rows + kRowKinds * kChunk * 4, bounds = back + KS * 32 * 4,
                       bytes = (bounds + (int)sizeof(ChunkBounds) + 255) / 256 * 256;
};

// Per chunk and head of keys: [K][Q], each [4 tiles of 16 rows][steps of 32 dimensions][parts][64 lanes] operands
constexpr size_t key_bytes(int dkp, int parts) { return (size_t)kChunk * dkp * 2 * parts * 2; }

template <class T>
constexpr int kParts = sizeof(T) == 4 ? 2 : 1;

typedef float f32x2 __attribute__((ext_vector_type(2)));

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
constexpr int kLoBits = 11;
constexpr float kLoUp = 1 << kLoBits, kLoDown = 1.f / kLoUp;
// A power of two (kLoUp times which is a number) that takes what is not above `bound` (its bits, sign off) below 2^15, and its reciprocal.  For no bound that is finite: any
__device__ __forceinline__ float scale_for(uint32_t bound) {
  const int field = 268 - (int)(bound >> 23);
  return __uint_as_float((uint32_t)min(field, 253 - kLoBits) << 23);
}
__device__ __forceinline__ float inverse_of(float power) { return __uint_as_float((254u << 23) - __float_as_uint(power)); }
__device__ __forceinline__ uint32_t magnitude(float v) { return __float_as_uint(v) & 0x7fffffffu; }
constexpr uint32_t kNotFinite = 0x7f800000u;  // magnitudes from here on

// x, y as hi + lo
__device__ __forceinline__ void split(float x, float y, h2& hi, h2& lo) {
  asm("" : "+v"(x), "+v"(y));  // rounded to fp32 first: a product that a conversion rounds once gives another hi, now and then
  hi = __builtin_convertvector((f32x2){x, y}, h2);
  lo = __builtin_convertvector((f32x2){__builtin_fmaf((float)hi[0], -1.f, x), __builtin_fmaf((float)hi[1], -1.f, y)}, h2);
}
__device__ __forceinline__ void split(const f32x4& v, h4& hi, h4& lo) {
  h2 h[2], l[2];
  split(v[0], v[1], h[0], l[0]);
  split(v[2], v[3], h[1], l[1]);
  hi = __builtin_shufflevector(h[0], h[1], 0, 1, 2, 3);
  lo = __builtin_shufflevector(l[0], l[1], 0, 1, 2, 3);
}

// ---------------------------------------------------------------------------
// First launch: P, W and the factors of every chunk and head, and q and k as operands of every chunk and head of keys
// ---------------------------------------------------------------------------
// A tile of 16 rows as operands: lane l has row l % 16, of step ks the dimensions 32 ks + 8 (l / 16) and on.  fp32 goes in times a power of two that takes the
// row's largest value to [2^8, 2^9), as hi + lo; binary16 as it is or (SCALED) times one that takes the row's length to [2^7, 2^8], in the range of
// binary16.  Of the lane's row: the sum of squares of what the operands hold, and the power; a row with something that is not finite is zero.
template <class T, int KS>
struct KeyTile {
  h8 f[KS][kParts<T>];
  float squares, power;
  bool finite;
  typedef T any8 __attribute__((ext_vector_type(8), aligned(sizeof(T))));
  any8 v[KS];  // as it is in memory

  // All requests of a row go out together: of whole groups they have no branches, where the compiler waits for what is on its way
  __device__ __forceinline__ void request(const T* rows, size_t ld, int row0, int nrows, int dk) {
    const int lane = threadIdx.x & 63, row = row0 + (lane & 15), d0 = (lane >> 4) * 8;
    const T* const p = rows + (size_t)(row < nrows ? row : 0) * ld;
    if (dk % 8 == 0) {
#pragma unroll
      for (int ks = 0; ks < KS; ks++) v[ks] = *reinterpret_cast<const any8*>(p + (ks * 32 + d0 < dk ? ks * 32 + d0 : 0));
    } else {
#pragma unroll
      for (int ks = 0; ks < KS; ks++)
#pragma unroll
        for (int i = 0; i < 8; i++) v[ks][i] = ks * 32 + d0 + i < dk ? p[ks * 32 + d0 + i] : (T)0.f;
    }
  }

  template <bool SCALED>
  __device__ __forceinline__ void take(int row0, int nrows, int dk) {
    const int lane = threadIdx.x & 63, d0 = (lane >> 4) * 8;
    const bool there = row0 + (lane & 15) < nrows;
#pragma unroll
    for (int ks = 0; ks < KS; ks++)
      if (!there || ks * 32 + d0 >= dk) v[ks] = (any8){};
    squares = 0.f;
    if constexpr (kParts<T> == 2) {
      uint32_t top = 0;
#pragma unroll
      for (int ks = 0; ks < KS; ks++)
#pragma unroll
        for (int i = 0; i < 8; i++) top = max(top, magnitude(v[ks][i]));
      top = max_across_rows(top);
      finite = top < kNotFinite;
      power = __uint_as_float((uint32_t)max(1, min(262 - (int)(top >> 23), 127 + 60)) << 23);  // 2^60 at most: its square times norm_eps stays in fp32
#pragma unroll
      for (int ks = 0; ks < KS; ks++)
#pragma unroll
        for (int i = 0; i < 8; i += 2) {
          const float x = finite ? v[ks][i] * power : 0.f, y = finite ? v[ks][i + 1] * power : 0.f;
          squares = __builtin_fmaf(x, x, squares);
          squares = __builtin_fmaf(y, y, squares);
          h2 hi, lo;
          split(x, y, hi, lo);
          f[ks][0][i] = hi[0], f[ks][0][i + 1] = hi[1];
          f[ks][1][i] = lo[0], f[ks][1][i + 1] = lo[1];
        }
      squares = add_across_32(add_across_16(squares));
    } else {
#pragma unroll
      for (int ks = 0; ks < KS; ks++) f[ks][0] = v[ks];
#pragma unroll
      for (int ks = 0; ks < KS; ks++) squares = dot8acc(f[ks][0], f[ks][0], squares);
      squares = add_across_32(add_across_16(squares));
      finite = magnitude(squares) < kNotFinite;
      power = 1.f;
      if constexpr (SCALED) power = __uint_as_float((uint32_t)(127 + min(8 - (((int)(__float_as_uint(squares) >> 23) - 125) >> 1), 15)) << 23);
      if (!finite) power = 0.f;
      if (SCALED || !finite) {
        const h1 by = (h1)power;
#pragma unroll
        for (int ks = 0; ks < KS; ks++) f[ks][0] = finite ? f[ks][0] * by : (h8){};
        squares = finite ? squares * power * power : 0.f;
      }
      if (!finite) power = 1.f;
    }
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

// Values as hi + lo 2^-kLoBits, from 2^kLoBits times them
__device__ __forceinline__ void split_far(const f32x4& up, h4& hi, h4& lo) {
  f32x4 v = up * kLoDown;
#pragma unroll
  for (int i = 0; i < 4; i += 2) {
    asm("" : "+v"(v[i]), "+v"(v[i + 1]));  // (or the compiler finds hi twice, by itself and for lo)
    const h2 h = __builtin_convertvector((f32x2){v[i], v[i + 1]}, h2);
    hi[i] = h[0], hi[i + 1] = h[1];
    lo[i] = (h1)__builtin_fmaf((float)h[0], -kLoUp, up[i]);
    lo[i + 1] = (h1)__builtin_fmaf((float)h[1], -kLoUp, up[i + 1]);
  }
}
__device__ __forceinline__ float join(float hi, float lo) { return __builtin_fmaf(lo, kLoDown, hi); }
__device__ __forceinline__ f32x4 join(const f32x4& hi, const f32x4& lo) {
  return (f32x4){join(hi[0], lo[0]), join(hi[1], lo[1]), join(hi[2], lo[2]), join(hi[3], lo[3])};
}

constexpr int kLd = kChunk + 4;  // of an fp32 matrix in LDS: 16 rows, 16 bytes each, are on all banks
constexpr int kLdT = kChunk + 8;

typedef short s4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) s4 lds_s4;
// Four rows of 16 columns of a matrix in LDS by the 16 lanes of a row of lanes: lane p gives row p / 4, columns 4 (p % 4) and on, and gets column p
__device__ __forceinline__ h4 read_columns(const h1* p) {
  return __builtin_bit_cast(h4, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4*)(void*)p));
}

// Operands of a block, of its row's power, of two tiles of results whose rows are its columns
__device__ __forceinline__ void store_block(char* to, const f32x4& a, const f32x4& b, float power) {
  const int lane = threadIdx.x & 63;
  const float up = power * kLoUp;
  h4 h[2], l[2];
  split_far(a * up, h[0], l[0]);
  split_far(b * up, h[1], l[1]);
  reinterpret_cast<h8*>(to)[lane] = __builtin_shufflevector(h[0], h[1], 0, 1, 2, 3, 4, 5, 6, 7);
  reinterpret_cast<h8*>(to)[64 + lane] = __builtin_shufflevector(l[0], l[1], 0, 1, 2, 3, 4, 5, 6, 7);
}
__device__ __forceinline__ float larger(float x, float y) { return __builtin_fmaxf(x, y); }
__device__ __forceinline__ float most_of(const f32x4& v) {
  return larger(larger(__builtin_fabsf(v[0]), __builtin_fabsf(v[1])), larger(__builtin_fabsf(v[2]), __builtin_fabsf(v[3])));
}
__device__ __forceinline__ float most_of_16(float v) {  // over the lanes that share lane / 16
  v = larger(v, dpp_mov<0xB1>(v));
  v = larger(v, dpp_mov<0x4E>(v));
  v = larger(v, dpp_mov<0x141>(v));
  return larger(v, dpp_mov<0x140>(v));
}

template <class T, int KS>
struct PrepLds {
  h1 K[kParts<T>][kChunk][KS * 32 + 8];
  union {
    float LT[kChunk][kLd];  // blocks of 16: behind the diagonal L's, as they are; on it T's, as they are; ahead of it T's from behind it, transposed
    h1 C[2][kChunk][kLdT];  // [column][row] of T with its rows' a_Ci, hi and lo
  };
  double G[kChunk];  // sums of the logarithms of the rows' decays
  float fk[kChunk], fq[kChunk], length[kChunk], write[kChunk], back[kChunk], inv[kChunk], ref[4][kChunk];
  __attribute__((aligned(16))) float most[2][4];
  int bad;
};

// blockIdx.x: a chunk, blockIdx.y: a head.  Wave w has the rows 16 w to 16 w + 15 of K, Q, L and P, those columns of T, and a quarter of W; wave 0 the gates.
// 4096 rows of 32 heads 128 x 128 of binary16: 44 us, four workgroups a compute unit (LDS), bound by instructions: 1470 of vectors a wave, 60 % of the cycles.
template <class T, int KS>
__global__ __launch_bounds__(256, KS * kParts<T> <= 4 ? 4 : KS * kParts<T> <= 8 ? 2 : 1) void delta_prep_kernel(DeltaArgs<T> a, DeltaTable tab, char* keys, char* heads) {
  constexpr int NK = kParts<T>, ST = KS / 2;
  typedef PrepLds<T, KS> Lds;
  typedef HeadLayout<KS> Out;
  __shared__ __attribute__((aligned(16))) Lds lds;
  const int lane = threadIdx.x & 63, c = lane & 15, g = lane >> 4, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int cj = blockIdx.x, head = blockIdx.y, kh = head / a.share;
  const int i0 = find_seq(a.nseq, cj, [&](int k) { return tab.chunk[k]; });
  const int t0 = tab.start[i0] + (cj - tab.chunk[i0]) * kChunk, len = min(tab.end[i0] - t0, kChunk);
  char* const out = heads + ((size_t)head * gridDim.x + cj) * Out::bytes;  // a head's chunks one behind the other: pages stay
  const int row = w * 16 + c, r0 = w * 16 + g * 4;  // the lane's row of an operand, the first one of results
  KeyTile<T, KS> K, Q;
  K.request(a.k + (size_t)t0 * a.ldk + (size_t)kh * a.dk, a.ldk, w * 16, len, a.dk);
  Q.request(a.q + (size_t)t0 * a.ldq + (size_t)kh * a.dk, a.ldq, w * 16, len, a.dk);
  const bool there = lane < len;  // wave 0: a lane a row
  float rate = 1.f, bias = 0.f;
  T dt = (T)0.f, raw = (T)0.f;
  if (w == 0) {
    const int t = t0 + min(lane, len - 1);
    dt = a.dt[(size_t)t * a.lddt + head];
    raw = a.beta[(size_t)t * a.ldbeta + head];
    if (a.A) rate = a.A[head];
    if (a.dt_bias) bias = a.dt_bias[head];
  }
  K.template take<true>(w * 16, len, a.dk);
  Q.template take<false>(w * 16, len, a.dk);
#pragma unroll
  for (int ks = 0; ks < KS; ks++)
#pragma unroll
    for (int n = 0; n < NK; n++) *reinterpret_cast<h8*>(&lds.K[n][row][ks * 32 + g * 8]) = K.f[ks][n];
  if (g == 0) {
    const float nan = __builtin_nanf("");
    const bool real = row < len;  // (of no row, and with a.eps zero, there is no length)
    lds.fk[row] = !real ? 0.f : K.finite ? K.factor(a.eps) : nan;
    lds.fq[row] = !real ? 0.f : (Q.finite ? Q.factor(a.eps) : nan) * a.scale;
    lds.length[row] = __builtin_sqrtf(K.squares * (KS * 32));  // not below the sum of the row's magnitudes
  }
  if (head % a.share == 0) {
    constexpr int tile = KS * NK * 64;
    h8* const to = reinterpret_cast<h8*>(keys + ((size_t)kh * gridDim.x + cj) * key_bytes(KS * 32, NK));
    K.store(to + w * tile);
    Q.store(to + (4 + w) * tile);
  }
  __syncthreads();
  f32x4 kk[4], kq[4];  // K K^T, rows 4 g and on of the wave's, column c of tile j; K Q^T, rows 4 g and on of tile j, column c of the wave's
#pragma unroll
  for (int j = 0; j < 4; j++) {
    kk[j] = kq[j] = (f32x4){0.f, 0.f, 0.f, 0.f};
    if (j > w) continue;
#pragma unroll
    for (int ks = 0; ks < KS; ks++) {
      const h8 b = *reinterpret_cast<const h8*>(&lds.K[0][j * 16 + c][ks * 32 + g * 8]);
      if constexpr (NK == 2) {
        const h8 lo = *reinterpret_cast<const h8*>(&lds.K[1][j * 16 + c][ks * 32 + g * 8]);
        kk[j] = mfma_h(K.f[ks][0], lo, kk[j]);
        kq[j] = mfma_h(lo, Q.f[ks][0], kq[j]);
        kk[j] = mfma_h(K.f[ks][1], b, kk[j]);
        kq[j] = mfma_h(b, Q.f[ks][1], kq[j]);
      }
      kk[j] = mfma_h(K.f[ks][0], b, kk[j]);
      kq[j] = mfma_h(b, Q.f[ks][0], kq[j]);
    }
  }
  if (w == 0) {
    const float lg = log_decay(a, (float)dt, finite_rate(rate), bias), fk = lds.fk[lane];
    float b = there ? (a.sigmoid ? sigmoid_f<true>((float)raw) : (float)raw) : 0.f;
    const unsigned long long off = __ballot(there && (magnitude(fk) >= kNotFinite || magnitude(b) >= kNotFinite || !(lg < __builtin_inff())));
    const int bad = off ? __builtin_ctzll(off) : kChunk;
    double G = there && lane < bad ? (double)__builtin_fmaxf(lg, kLeastLog) : 0.0;
    if (lane >= bad) b = 0.f;
#pragma unroll
    for (int m = 1; m < 64; m *= 2) {
      const double up = __shfl_up(G, m);
      if (lane >= m) G += up;
    }
    const float f = lane < bad ? fk : 0.f, from = decay_f((float)G), key = b * from * f;
    lds.G[lane] = G;
    lds.write[lane] = b * f;
    lds.back[lane] = f * decay_f((float)(__shfl(G, 63) - G));
    float* const rows = reinterpret_cast<float*>(out + Out::rows) + lane;
    rows[kRowBeta * kChunk] = b;
    rows[kRowK * kChunk] = key;
    rows[kRowQ * kChunk] = lds.fq[lane] * from;
    rows[kRowKeep * kChunk] = there && lane < bad ? decay_f(lg) : -1.f;
    const float reach = __builtin_fabsf(key) * lds.length[lane], bkey = max_across_rows(most_of_16(reach));
    lds.length[lane] = reach;
    if (lane == 63) {
      lds.bad = bad;
      ChunkBounds* const to = reinterpret_cast<ChunkBounds*>(out + Out::bounds);
      to->key = bkey;
      to->keep = from;
      to->bad = bad;
    }
  }
  __syncthreads();
  const int bad = lds.bad;
  f32x4 X[4];  // T's tiles (w + n, w), as results
  {
    // Decays between a row of the wave's and one ahead of them go by way of the row in between: each half is at most one where decays are
    const double Gref = lds.G[w ? w * 16 - 1 : 0], Gl = lds.G[lane];
    const bool ahead = lane < w * 16;
    lds.ref[w][lane] = decay_f((float)(ahead ? Gref - Gl : Gl - Gref)) * (ahead ? (lane < bad ? lds.fk[lane] : 0.f) : 1.f);
    __builtin_amdgcn_wave_barrier();
    const f32x4 lw = *reinterpret_cast<const f32x4*>(&lds.write[r0]), lref = *reinterpret_cast<const f32x4*>(&lds.ref[w][r0]);
    const float qi = row < bad ? lds.fq[row] : 0.f, qref = lds.ref[w][row];
    f32x4 ld;  // L on the diagonal
#pragma unroll
    for (int j = 0; j < 4; j++) {
      if (j > w) continue;
      const int col = j * 16 + c, col4 = j * 16 + g * 4;
      if (j < w) {
        const float at = lds.ref[w][col];
        const f32x4 at4 = *reinterpret_cast<const f32x4*>(&lds.ref[w][col4]);
#pragma unroll
        for (int r = 0; r < 4; r++) {
          lds.LT[r0 + r][col] = lw[r] * (lref[r] * at * kk[j][r]);
          kq[j][r] = qi * (qref * at4[r] * kq[j][r]);
        }
      } else {
        const double Gc = lds.G[col];  // of the lane's column of L, and of its row of A
        const float fc = col < bad ? lds.fk[col] : 0.f;
#pragma unroll
        for (int r = 0; r < 4; r++) {
          const double Gr = lds.G[r0 + r];
          const float f4 = r0 + r < bad ? lds.fk[r0 + r] : 0.f;
          ld[r] = col < r0 + r ? lw[r] * (decay_f((float)(Gr - Gc)) * fc * kk[j][r]) : 0.f;
          kq[j][r] = r0 + r <= col ? qi * (decay_f((float)(Gc - Gr)) * f4 * kq[j][r]) : 0.f;
        }
      }
    }
    // T on the diagonal: column c, row by row, L's values from their lanes
    float t[16];
#pragma unroll
    for (int i = 0; i < 16; i++) t[i] = i == c ? 1.f : 0.f;
#pragma unroll
    for (int j = 0; j < 15; j++)
#pragma unroll
      for (int i = 1; i < 16; i++) {
        if (i <= j) continue;
        const float l = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(ld[i % 4]), i / 4 * 16 + j));
        t[i] = __builtin_fmaf(-l, t[j], t[i]);
      }
#pragma unroll
    for (int s = 0; s < 4; s++) {
      const float ta = t[s], tb = t[4 + s], tc = t[8 + s], td = t[12 + s];
      const float x = g & 1 ? tb : ta, y = g & 1 ? td : tc;
      X[0][s] = g & 2 ? y : x;
      lds.LT[r0 + s][w * 16 + c] = X[0][s];
    }
  }
  __syncthreads();
  // T behind it: T_ij = -T_ii sum_m L_im T_mj (m = j to i - 1).  An operand of results as they lie (row 4 g + s of step s) goes with the columns 4 g + s of
  // the other matrix.
#pragma unroll
  for (int n = 1; n < 4; n++) {
    X[n] = (f32x4){0.f, 0.f, 0.f, 0.f};
    if (w + n > 3) continue;
    const int i = w + n;
    f32x4 acc[2] = {X[n], X[n]};
#pragma unroll
    for (int m = 0; m < 3; m++) {
      if (m >= n) continue;
      const f32x4 l = *reinterpret_cast<const f32x4*>(&lds.LT[i * 16 + c][(w + m) * 16 + g * 4]);
#pragma unroll
      for (int s = 0; s < 4; s++) acc[s & 1] = mfma_f(l[s], X[m][s], acc[s & 1]);
    }
    const f32x4 ti = *reinterpret_cast<const f32x4*>(&lds.LT[i * 16 + c][i * 16 + g * 4]), sum = acc[0] + acc[1];
#pragma unroll
    for (int s = 0; s < 4; s++) X[n] = mfma_f(ti[s], -sum[s], X[n]);
    *reinterpret_cast<f32x4*>(&lds.LT[w * 16 + c][i * 16 + g * 4]) = X[n];
  }
  __syncthreads();
  {  // P = A T, as its transpose T^T A^T: a lane has columns 4 g and on of every tile, of its row
    f32x4 P[4];
    float top = 0.f;
#pragma unroll
    for (int j = 0; j < 4; j++) {
      P[j] = (f32x4){0.f, 0.f, 0.f, 0.f};
      if (j > w) continue;
#pragma unroll
      for (int m = 0; m < 4; m++) {
        if (m < j || m > w) continue;
        f32x4 t;
        if (m == j) {
#pragma unroll
          for (int s = 0; s < 4; s++) t[s] = lds.LT[j * 16 + g * 4 + s][j * 16 + c];
        } else {
          t = *reinterpret_cast<const f32x4*>(&lds.LT[j * 16 + c][m * 16 + g * 4]);
        }
#pragma unroll
        for (int s = 0; s < 4; s++) P[j] = mfma_f(t[s], kq[m][s], P[j]);
      }
    }
#pragma unroll
    for (int j = 0; j < 4; j++) top = larger(top, most_of(P[j]));
    const float power = scale_for(magnitude(max_across_rows(top)));
    store_block(out + block_of(w, 0) * kBlockBytes, P[0], P[1], power);
    if (w >= 2) store_block(out + block_of(w, 1) * kBlockBytes, P[2], P[3], power);
    if (g == 0) reinterpret_cast<float*>(out + Out::rows)[kRowP * kChunk + row] = inverse_of(power);
  }
  float top = 0.f;  // T with a_Ci
#pragma unroll
  for (int n = 0; n < 4; n++) {
    if (w + n > 3) continue;
    X[n] *= *reinterpret_cast<const f32x4*>(&lds.back[(w + n) * 16 + g * 4]);
    top = larger(top, most_of(X[n]));
  }
  const float power = scale_for(magnitude(max_across_rows(top)));
  if (g == 0) lds.inv[row] = inverse_of(power);
  __syncthreads();
  if (w & 1) {  // the block of 32 rows begins ahead of the diagonal
    *reinterpret_cast<h4*>(&lds.C[0][row][(w - 1) * 16 + g * 4]) = (h4){};
    *reinterpret_cast<h4*>(&lds.C[1][row][(w - 1) * 16 + g * 4]) = (h4){};
  }
#pragma unroll
  for (int n = 0; n < 4; n++) {
    if (w + n > 3) continue;
    h4 hi, lo;
    split(X[n] * power, hi, lo);
    *reinterpret_cast<h4*>(&lds.C[0][row][(w + n) * 16 + g * 4]) = hi;
    *reinterpret_cast<h4*>(&lds.C[1][row][(w + n) * 16 + g * 4]) = lo;
  }
  __syncthreads();
  // W = K^T T, as its transpose: a lane has columns 4 g and on of every tile, of row c of a tile
  float wide = 0.f, both = 0.f;
#pragma unroll
  for (int t = 0; t < ST; t++) {
    const int d0 = (w * ST + t) * 16;
    f32x4 W[4];
#pragma unroll
    for (int j = 0; j < 4; j++) W[j] = (f32x4){0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int ks = 0; ks < 2; ks++) {
      h8 k[NK];
#pragma unroll
      for (int n = 0; n < NK; n++) {
        const h1* const at = &lds.K[n][ks * 32 + g * 8 + c / 4][d0 + (c & 3) * 4];
        k[n] = __builtin_shufflevector(read_columns(at), read_columns(at + 4 * (KS * 32 + 8)), 0, 1, 2, 3, 4, 5, 6, 7);
      }
#pragma unroll
      for (int j = 0; j < 4; j++) {
        if (j >= 2 + 2 * ks) continue;
        const h8 hi = *reinterpret_cast<const h8*>(&lds.C[0][j * 16 + c][ks * 32 + g * 8]), lo = *reinterpret_cast<const h8*>(&lds.C[1][j * 16 + c][ks * 32 + g * 8]);
        W[j] = mfma_h(lo, k[0], W[j]);
        if constexpr (NK == 2) W[j] = mfma_h(hi, k[1], W[j]);
        W[j] = mfma_h(hi, k[0], W[j]);
      }
    }
    float most = 0.f, sum = 0.f, reach = 0.f;
#pragma unroll
    for (int j = 0; j < 4; j++) {
      const f32x4 far = *reinterpret_cast<const f32x4*>(&lds.length[j * 16 + g * 4]);
      W[j] *= *reinterpret_cast<const f32x4*>(&lds.inv[j * 16 + g * 4]);
      most = larger(most, most_of(W[j]));
#pragma unroll
      for (int s = 0; s < 4; s++) {
        sum += __builtin_fabsf(W[j][s]);
        reach = __builtin_fmaf(__builtin_fabsf(W[j][s]), far[s], reach);
      }
    }
    const float by = scale_for(magnitude(max_across_rows(most)));
    wide = larger(wide, add_across_32(add_across_16(sum)));
    both = larger(both, add_across_32(add_across_16(reach)));
    char* const to = out + Out::W + (w * ST + t) * 2 * kBlockBytes;
    store_block(to, W[0], W[1], by);
    store_block(to + kBlockBytes, W[2], W[3], by);
    if (g == 0) reinterpret_cast<float*>(out + Out::back)[d0 + c] = inverse_of(by);
  }
  wide = most_of_16(wide);
  both = most_of_16(both);
  if (lane == 0) {
    lds.most[0][w] = wide;
    lds.most[1][w] = both;
  }
  __syncthreads();
  if (threadIdx.x < 2) {
    const f32x4 m = *reinterpret_cast<const f32x4*>(lds.most[threadIdx.x]);
    (&reinterpret_cast<ChunkBounds*>(out + Out::bounds)->back)[threadIdx.x] = most_of(m);
  }
}

// ---------------------------------------------------------------------------
// Second launch: the chunks of a prompt one after another
// ---------------------------------------------------------------------------
constexpr float kLeastSize = 0x1p-12f * kLoUp;  // see the scan

// LDS alone: loads that are on their way to registers stay on it
__device__ __forceinline__ void lds_barrier() {
  asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}

template <class T, int KS>
struct ScanLds {
  h1 S[2][16][KS * 32], R[2][16][kChunk];          // [column][row: see place], hi and lo; R's rows as the blocks of P and W have their columns
  float bv[2][4][64][4];                           // b v of this chunk and the next one, of the lanes of waves 0 to 3
  float qs[4][64][4];                              // Q S, of their lanes
  float most[16][20];                              // of S, of each lane's rows
  uint32_t vmost[16][4];                           // of b v of the next chunk (as bits, which tell what is not finite)
  float cols[16][2], inv[16][2];                   // of each column: the largest b v, the decay of the chunk (or NaN: see spoilt); R's inverse power, S's
  float sums[2][5][16][4];                         // of a row that goes token by token and the next one, of waves 0 to 3
  int gone[4], far;                                // rows that go token by token; the last chunk that has rows of R or columns of S far below their bounds
};

// Where the eight rows from 8 b on of column c are in S (64 rows and more) and R: rows of 16 bytes, 16 of which are on all banks, change places
// so that the 16 columns' ones of the same b are, and those of any b that the lanes of a read mix
template <int ROWS>
__device__ __forceinline__ int place(int c, int b) { return (b ^ (ROWS == 64 ? c >> 1 : c)) * 8; }

// An element `off` bytes behind a uniform address (or the compiler adds the two ahead of the loop, and keeps 64 bits a lane)
template <class T>
__device__ __forceinline__ T* behind(T* uniform, uint32_t off) {
  asm("" : "+v"(off));
  return reinterpret_cast<T*>(const_cast<char*>(reinterpret_cast<const char*>(uniform)) + off);
}

__device__ __forceinline__ void in_order() { __builtin_amdgcn_sched_barrier(0); }

// Rows of v or y of a chunk as a buffer of the rows that are there: what lies behind its end is read as zero and not written.  So the code
// has no branches around requests, where the compiler would have to wait for all that may be on their way.
template <class T>
__device__ __forceinline__ __amdgpu_buffer_rsrc_t rows_of(T* rows, int nrows, int ld) {
  const int there = __builtin_amdgcn_readfirstlane(nrows < 0 ? 0 : nrows < kChunk ? nrows : kChunk);  // (or the compiler takes it for the lanes' own)
  return __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(static_cast<const void*>(rows)), 0, (int)((uint32_t)there * (uint32_t)ld * (uint32_t)sizeof(T)), 0x00027000);
}
template <class T>
__device__ __forceinline__ T load_row(__amdgpu_buffer_rsrc_t rows, uint32_t at) {
  if constexpr (sizeof(T) == 2) return __builtin_bit_cast(T, (uint16_t)__builtin_amdgcn_raw_buffer_load_b16(rows, at, 0, 0));
  else return __builtin_bit_cast(T, (uint32_t)__builtin_amdgcn_raw_buffer_load_b32(rows, at, 0, 0));
}
template <class T>
__device__ __forceinline__ void store_row(__amdgpu_buffer_rsrc_t rows, uint32_t at, T v) {
  if constexpr (sizeof(T) == 2) __builtin_amdgcn_raw_buffer_store_b16(__builtin_bit_cast(uint16_t, v), rows, at, 0, 0);
  else __builtin_amdgcn_raw_buffer_store_b32(__builtin_bit_cast(uint32_t, v), rows, at, 0, 0);
}

// The lane, found anew: where it is seldom needed, so that nothing that is made of it stays in registers until then
__device__ __forceinline__ int this_lane() { return __builtin_amdgcn_mbcnt_hi(~0u, __builtin_amdgcn_mbcnt_lo(~0u, 0u)); }

// Four rows' factors of the one that each lane of a quad requested
__device__ __forceinline__ f32x4 of_quad(float f) { return (f32x4){dpp_mov<0x00>(f), dpp_mov<0x55>(f), dpp_mov<0xAA>(f), dpp_mov<0xFF>(f)}; }
template <int LANE>
__device__ __forceinline__ float of_lane(float f) { return __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(f), LANE)); }

// blockIdx.x: a prompt, a head and 16 columns of its state.  A lane has column c of a tile, rows 4 g and on of one of 16 rows.
//
// What the next chunk waits for is a row of dependent steps, S to LDS, K S, R to LDS, W R, and it is their latency that counts: waves 0 to 3 do them, with
// 16 rows each of K and a quarter of those of W and S, and Q S, whose operands of S they have, besides.  Waves 4 to 7 do the rest, with 16 rows each of
// P and v: they hand over b v and what belongs to it, and make y.  LDS passes 128 bytes a cycle, 16 bytes a lane in eight whether the lanes read
// the same or not: rows' factors go from memory to registers, one a lane, and round the quads of lanes.
//
// The powers of two by which columns are scaled come from bounds, of S ahead of its values (without waiting for the other waves' ones):
//   |R| <= max |b v| + key max |S|,   key = max_i |b_i a_i0| |k_i|_1
//   |S'| <= a_C0 max |S| + back max |b v| + both max |S|,   back = max_d sum_i |W_di|,   both = max_d sum_i |W_di| |b_i a_i0| |k_i|_1
// They may be 2^27 too high before a pair holds a column's largest value to less than fp32 does.
//
// The 64 rows of a column of R share a power, so one that is 2^-s of the bound is off by 2^(s - 51) of itself, and by as much in the results of a row is what
// W's and P's pairs make of those ahead of it.  It shows where nothing of a row's own size stands behind it: ahead of a value that is far above the others, and
// behind one (or a state) that has been forgotten.  So a row i whose size, the largest a_ij max(|R_j|, |b_j v_j|) of the rows up to it, is below 2^-26 of the
// bound or so, and all ahead of it, go token by token from S (far_rows, walk); others are off by 2^-23 of their size at most for each row that is at the bound,
// as the roundings of 64 fp32 products are.  So do all rows of a chunk whose S is 2^27 and more below its bound, which is too high where a value was
// forgotten in the chunk before.  Only chunks with a row of R that is that low look for them, hardly any of a layer's ordinary values (without the 2^11 it would
// be one in some hundred); a look takes 1 us, a row 0.8 to 2.6 (64 to 256 keys).
//
// 4096 rows of 32 heads 128 x 128 of binary16: 109 us, 1.7 a chunk, 130 to 139 where operands and rows come from memory.  Vector instructions take 36 % of the
// cycles, matrix ones 15 %; the rest is the latency of the dependent steps, and of 76 KB of operands a chunk.
template <class T, int KS>
__global__ __launch_bounds__(512, KS * kParts<T> <= 2 ? 4 : 2) void delta_scan_kernel(DeltaArgs<T> a, DeltaTable tab, const char* keys, const char* heads) {
  constexpr int NK = kParts<T>, ST = KS / 2;  // ST: tiles of 16 rows of S of a wave
  typedef ScanLds<T, KS> Lds;
  typedef HeadLayout<KS> In;
  __shared__ __attribute__((aligned(16))) Lds lds;
  const int lane = threadIdx.x & 63, c = lane & 15, g = lane >> 4, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), w = wave & 3;
  // Workgroups go round the eight XCDs: those of a prompt and head of keys, which read the same operands, come to be on one
  const int slices = (a.dv + 15) / 16, nkh = a.heads / a.share, alike = a.share * slices, sets = a.nseq * nkh;
  const int whole_sets = sets / kXcds * kXcds, at = blockIdx.x < whole_sets * alike ? blockIdx.x : blockIdx.x - whole_sets * alike;
  const int round = blockIdx.x < whole_sets * alike ? kXcds : sets - whole_sets;
  const int turn = at / round, set = (blockIdx.x < whole_sets * alike ? turn / alike * kXcds : whole_sets) + at % round, member = turn % alike;
  const int i0 = set / nkh, kh = set % nkh, head = kh * a.share + member / slices, col0 = member % slices * 16;
  const int begin = tab.start[i0], end = tab.end[i0], nchunk = tab.chunk[i0 + 1] - tab.chunk[i0], first = tab.chunk[i0];
  const size_t nall = tab.chunk[a.nseq];
  const bool mine = col0 + c < a.dv;
  const int col = mine ? col0 + c : a.dv - 1;
  // Whether rows of chunk j are far below their bounds, behind the barrier behind R; and how many go token by token, behind two more
  auto is_far = [](int seen, int j) { return __builtin_expect(__builtin_amdgcn_readfirstlane(seen) == j, 0); };  // lds.far
  auto gone_of = [&] { return max(max(__builtin_amdgcn_readfirstlane(lds.gone[0]), __builtin_amdgcn_readfirstlane(lds.gone[1])),
                                  max(__builtin_amdgcn_readfirstlane(lds.gone[2]), __builtin_amdgcn_readfirstlane(lds.gone[3]))); };
  if (nchunk == 0) {  // no rows: the state as it was
    const float* const from = a.state;
    const size_t st = ((size_t)tab.seq[i0] * a.heads + head) * a.dk * a.dv;
    for (int d = wave * 4 + g; d < a.dk; d += 32)
      if (mine) a.state_out[st + (size_t)d * a.dv + col] = from[st + (size_t)d * a.dv + col];
    return;
  }
  constexpr size_t head_step = In::bytes, key_step = key_bytes(KS * 32, NK);
  const char* here = heads + (head * nall + first) * head_step;  // of the chunk that is requested next
  const int row0 = w * 16 + g * 4, quad0 = row0 + (c & 3);       // the lane's rows of a chunk; the one of which it requests factors
  const uint32_t limits_at = In::bounds + (lane & 7) * 4;
  if (wave < 4) {
    __builtin_amdgcn_s_setprio(2);
    const char* own = keys + (kh * nall + first) * key_step;
    const uint32_t own_at = (w * KS * NK * 64 + lane) * 16;
    h8 Kf[KS][NK], Qf[KS][NK];
    auto load_step = [&](const char* p, h8 (&f)[KS][NK], int ks) {
      const h8* const q = reinterpret_cast<const h8*>(behind(p, own_at));
#pragma unroll
      for (int n = 0; n < NK; n++) f[ks][n] = q[(ks * NK + n) * 64];
    };
    auto load_own = [&](const char* p, h8 (&f)[KS][NK]) {
#pragma unroll
      for (int ks = 0; ks < KS; ks++) load_step(p, f, ks);
    };
    constexpr size_t queries = (size_t)4 * KS * NK * 64 * 16;  // behind the keys
    const size_t st = ((size_t)tab.seq[i0] * a.heads + head) * a.dk * a.dv;
    const float* const from = i0 == 0 && tab.ahead ? a.state_out : a.state;
    const int d0 = w * (ST * 16) + g * 4, at_row = place<kChunk>(c, (w >> 1) * 4 + g) + (w & 1) * 4;  // the lane's rows of S[0], of R
    const uint32_t back_at = In::W + (w * ST * 2 * 2 * 64 + lane) * 16, key_at = In::rows + (kRowK * kChunk + quad0) * 4,
                   scale_at = In::back + (d0 + (c & 3)) * 4;
    h8 Wf[ST][2][2];
    float key, limits, scale[ST];
    auto load_back = [&](const char* p, int t) {
      const h8* const q = reinterpret_cast<const h8*>(behind(p, back_at));
#pragma unroll
      for (int ks = 0; ks < 2; ks++)
#pragma unroll
        for (int n = 0; n < 2; n++) Wf[t][ks][n] = q[((t * 2 + ks) * 2 + n) * 64];
      scale[t] = *reinterpret_cast<const float*>(behind(p + t * 64, scale_at));
    };
    auto load_key = [&](const char* p) {
      key = *reinterpret_cast<const float*>(behind(p, key_at));
      limits = *reinterpret_cast<const float*>(behind(p, limits_at));
    };
    load_own(own, Kf);
    load_key(here);
    load_own(own + queries, Qf);
#pragma unroll
    for (int t = 0; t < ST; t++) load_back(here, t);
    f32x4 S[ST];
    auto most_of_S = [&] {
      float m = 0.f;
#pragma unroll
      for (int t = 0; t < ST; t++) m = larger(m, most_of(S[t]));
      lds.most[c][w * 4 + g] = m;
    };
    // How many rows of chunk j, up to the last one that must, are to go token by token.  What a row is off by is carried on like its size, and grows with
    // decays that do.  A lane's rows are taken together, then the wave's, then those of all four.
    auto far_rows = [&](int j, const f32x4& size) {
      const int lane = this_lane(), c = lane & 15, g = lane >> 4;
      const f32x4 keep = *reinterpret_cast<const f32x4*>(heads + (head * nall + first + j) * head_step + In::rows + (kRowKeep * kChunk + w * 16 + g * 4) * 4);
      float s[4], o[4], k[4];  // of its rows by themselves: size, what they are off by, and what is left of a size ahead of them
      auto of_row = [&](int r) { return keep[r] < 0.f ? __builtin_inff() : size[r]; };
      s[0] = of_row(0), o[0] = 1.f, k[0] = keep[0];
#pragma unroll
      for (int r = 1; r < 4; r++) s[r] = larger(of_row(r), keep[r] * s[r - 1]), o[r] = larger(1.f, keep[r] * o[r - 1]), k[r] = keep[r] * k[r - 1];
      float S1 = s[3], O1 = o[3], K1 = k[3];
#pragma unroll
      for (int m = 16; m < 64; m *= 2) {
        const float sm = __shfl_up(S1, m), om = __shfl_up(O1, m), km = __shfl_up(K1, m);
        if (lane >= m) S1 = larger(S1, K1 * sm), O1 = larger(O1, K1 * om), K1 *= km;
      }
      f32x4* const waves = reinterpret_cast<f32x4*>(&lds.sums[0][0][0][0]);
      if (g == 3) waves[w * 16 + c] = (f32x4){S1, O1, K1, 0.f};
      float sa = __shfl_up(S1, 16), oa = __shfl_up(O1, 16), ka = __shfl_up(K1, 16);  // of the rows ahead of the lane's: in the wave
      if (g == 0) sa = oa = 0.f, ka = 1.f;
      lds_barrier();
      float sb = 0.f, ob = 1.f;  // and in those before
      for (int i = 0; i < w; i++) {
        const f32x4 m = waves[i * 16 + c];
        sb = larger(m[0], m[2] * sb), ob = larger(m[1], m[2] * ob);
      }
      sa = larger(sa, ka * sb), oa = larger(oa, ka * ob);
      int rows = 0;
#pragma unroll
      for (int r = 0; r < 4; r++) {
        const float z = larger(s[r], k[r] * sa);
        const unsigned long long off = __ballot(z > 0.f && z < kLeastSize * larger(o[r], k[r] * oa));
        if (off) rows = max(rows, w * 16 + (63 - __builtin_clzll(off)) / 16 * 4 + r + 1);
      }
      lds.gone[w] = rows;
      lds_barrier();
      return gone_of();
    };
    // The first rows of chunk j token by token, y and, in LDS, S: each wave has its rows of S, whose sums meet there.  In few registers, and loops that are not
    // unrolled: what counts is that the chunks that do not come here are not held up.
    auto state_of = [&](int lane) { return reinterpret_cast<float*>(&lds.S[0][0][0]) + (w * (ST * 16) + (lane >> 4) * 4) * 16 + (lane & 15); };  // [row][column]
    auto walk = [&](int j, int rows) {
      const int lane = this_lane(), c = lane & 15, g = lane >> 4, d0 = w * (ST * 16) + g * 4, col = min(col0 + c, a.dv - 1);
      float* const state = state_of(lane);
      const float* const factors = reinterpret_cast<const float*>(heads + (head * nall + first + j) * head_step + In::rows);
      const float keeps = factors[kRowKeep * kChunk + lane], writes = factors[kRowBeta * kChunk + lane];
#pragma unroll
      for (int t = 0; t < ST; t++)
#pragma unroll
        for (int r = 0; r < 4; r++) state[(t * 16 + r) * 16] = S[t][r];
#pragma clang loop unroll(disable)
      for (int i = 0; i < rows; i++) {
        const size_t t = (size_t)begin + j * kChunk + i;
        const T* const kr = a.k + t * a.ldk + (size_t)kh * a.dk;
        const T* const qr = a.q + t * a.ldq + (size_t)kh * a.dk;
        const float v = (float)a.v[t * a.ldv + (size_t)head * a.dv + col];
        const float keep = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(keeps), i));
        const float b = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(writes), i));
        float sum[5] = {};  // k k, q q, q k, k S, q S
#pragma clang loop unroll(disable)
        for (int e = 0; e < ST * 16; e += 16) {
          T k[4], q[4];
#pragma unroll
          for (int r = 0; r < 4; r++) {
            const int d = min(d0 + e + r, a.dk - 1);
            k[r] = kr[d], q[r] = qr[d];
          }
#pragma unroll
          for (int r = 0; r < 4; r++) {
            const float x = d0 + e + r < a.dk ? (float)k[r] : 0.f, y = d0 + e + r < a.dk ? (float)q[r] : 0.f, s = state[(e + r) * 16];
            sum[0] = __builtin_fmaf(x, x, sum[0]);
            sum[1] = __builtin_fmaf(y, y, sum[1]);
            sum[2] = __builtin_fmaf(y, x, sum[2]);
            sum[3] = __builtin_fmaf(x, s, sum[3]);
            sum[4] = __builtin_fmaf(y, s, sum[4]);
          }
        }
#pragma unroll
        for (int n = 0; n < 5; n++) {
          const float all = add_across_32(add_across_16(sum[n]));
          if (g == 0) lds.sums[i & 1][n][c][w] = all;  // the next row's go elsewhere: a barrier a row
        }
        lds_barrier();
#pragma unroll
        for (int n = 0; n < 5; n++) {
          const f32x4 m = *reinterpret_cast<const f32x4*>(lds.sums[i & 1][n][c]);
          sum[n] = (m[0] + m[1]) + (m[2] + m[3]);
        }
        float kn = 1.f, qn = a.scale;
        if (a.eps >= 0.f) {
          kn = __builtin_amdgcn_rsqf(sum[0] + a.eps);
          qn = __builtin_amdgcn_rsqf(sum[1] + a.eps) * a.scale;
        }
        const float u = kn * (b * (v - keep * kn * sum[3]));
#pragma clang loop unroll(disable)
        for (int e = 0; e < ST * 16; e += 16) {
          T k[4];
#pragma unroll
          for (int r = 0; r < 4; r++) k[r] = kr[min(d0 + e + r, a.dk - 1)];
#pragma unroll
          for (int r = 0; r < 4; r++) state[(e + r) * 16] = __builtin_fmaf(d0 + e + r < a.dk ? (float)k[r] : 0.f, u, keep * state[(e + r) * 16]);
        }
        if (w == 0 && g == 0 && col0 + c < a.dv) a.y[t * a.ldy + (size_t)head * a.dv + col] = (T)(qn * __builtin_fmaf(keep, sum[4], sum[2] * u));
      }
    };
#pragma unroll
    for (int t = 0; t < ST; t++)
#pragma unroll
      for (int r = 0; r < 4; r++) {
        const int d = d0 + t * 16 + r;
        S[t][r] = d < a.dk ? from[st + (size_t)d * a.dv + col] : 0.f;
      }
    auto most_of_all = [&] { return max_across_rows(most_of(*reinterpret_cast<const f32x4*>(&lds.most[c][g * 4]))); };
    most_of_S();
    if (threadIdx.x == 0) lds.far = -1;
    lds_barrier();
    float sbound = most_of_all();  // of the column of S; the first chunk's is its own largest value
    lds_barrier();
    const int last = end - begin - (nchunk - 1) * kChunk;  // rows of the last chunk
    auto sizes_of = [&](const f32x4& R, const f32x4& bv) {  // of the lane's rows
      f32x4 size;
#pragma unroll
      for (int r = 0; r < 4; r++) size[r] = larger(__builtin_fabsf(R[r]), __builtin_fabsf(bv[r]));
      return size;
    };
    auto sizes_there = [&](f32x4 size) {  // rows behind the last one have none that is too small
      asm volatile("");  // (a branch: a row's selects would be made of every chunk)
#pragma unroll
      for (int r = 0; r < 4; r++) size[r] = row0 + r < last ? size[r] : __builtin_inff();
      return size;
    };
    for (int j = 0; j < nchunk; j++) {
      const bool more = j + 1 < nchunk;
      const float power = scale_for(magnitude(sbound)), sinv = inverse_of(power), sup = power * kLoUp;
#pragma unroll
      for (int t = 0; t < ST; t++) {
        h4 hi, lo;
        split_far(S[t] * sup, hi, lo);
        const int to = place<KS * 32>(c, (d0 + t * 16) / 8) + (g & 1) * 4;
        *reinterpret_cast<h4*>(&lds.S[0][c][to]) = hi;
        *reinterpret_cast<h4*>(&lds.S[1][c][to]) = lo;
        if (t > 0) {
          load_back(here, t);
          in_order();
        }
      }
      most_of_S();
      lds_barrier();
      h8 hi[KS], lo[KS];
#pragma unroll
      for (int ks = 0; ks < KS; ks++) {
        lo[ks] = *reinterpret_cast<const h8*>(&lds.S[1][c][place<KS * 32>(c, ks * 4 + g)]);
        hi[ks] = *reinterpret_cast<const h8*>(&lds.S[0][c][place<KS * 32>(c, ks * 4 + g)]);
      }
      const float vm = lds.cols[c][0];
      float keep = lds.cols[c][1];
      f32x4 bv = *reinterpret_cast<const f32x4*>(lds.bv[j & 1][w][lane]), kf = of_quad(key);
      const float sm = most_of_all();
      f32x4 s[4];  // hi and lo apart, and both in two sums: a product waits for the one ahead of it
#pragma unroll
      for (int k = 0; k < 4; k++) s[k] = (f32x4){0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int ks = 0; ks < KS; ks++) {
        s[ks & 1] = mfma_h(Kf[ks][0], lo[ks], s[ks & 1]);
        s[2 + (ks & 1)] = mfma_h(Kf[ks][0], hi[ks], s[2 + (ks & 1)]);
        if constexpr (NK == 2) s[2 + (ks & 1)] = mfma_h(Kf[ks][1], hi[ks], s[2 + (ks & 1)]);
      }
      const float reach = __builtin_fmaf(of_lane<0>(limits), sm, vm), rpower = scale_for(magnitude(reach)), rup = rpower * kLoUp;
      float rinv = inverse_of(rpower);
      sbound = __builtin_fmaf(of_lane<3>(limits) + of_lane<2>(limits), sm, of_lane<1>(limits) * vm);
      kf *= rup;  // (one by one: their product may be no number)
      kf *= sinv;
      bv *= rup;
      // A row's least size: none is below that of a column of zeros, all are where S is not zero but more than 2^27 below its bound
      const float least = magnitude(sm * sup) - 1 < magnitude(0.5f) - 1 ? __builtin_inff() : reach * (rup * (kLeastSize * 0x1p-26f));
      f32x4 q[2];
      q[0] = q[1] = (f32x4){0.f, 0.f, 0.f, 0.f};
      own = more ? own + key_step : own;
      here = more ? here + head_step : here;
#pragma unroll
      for (int ks = 0; ks < KS; ks++) {
        in_order();
        load_step(own, Kf, ks);
        q[0] = mfma_h(Qf[ks][0], lo[ks], q[0]);
        q[1] = mfma_h(Qf[ks][0], hi[ks], q[1]);
        if constexpr (NK == 2) q[1] = mfma_h(Qf[ks][1], hi[ks], q[1]);
      }
      in_order();
      load_own(own + queries, Qf);
      f32x4 R;
#pragma unroll
      for (int r = 0; r < 4; r++) R[r] = __builtin_fmaf(-kf[r], join(s[2][r] + s[3][r], s[0][r] + s[1][r]), bv[r]);
      h4 rhi, rlo;
      split_far(R, rhi, rlo);
      *reinterpret_cast<h4*>(&lds.R[0][c][at_row]) = rhi;
      *reinterpret_cast<h4*>(&lds.R[1][c][at_row]) = rlo;
      f32x4 size = sizes_of(R, bv);
      if (!more) size = sizes_there(size);
      if (__builtin_expect(__ballot(__builtin_fminf(__builtin_fminf(size[0], size[1]), __builtin_fminf(size[2], size[3])) < least) != 0, 0)) lds.far = j;
      load_key(here);
      lds_barrier();
      const int seen = lds.far;
      h8 rh[2], rl[2];
#pragma unroll
      for (int ks = 0; ks < 2; ks++) {
        rl[ks] = *reinterpret_cast<const h8*>(&lds.R[1][c][place<kChunk>(c, ks * 4 + g)]);
        rh[ks] = *reinterpret_cast<const h8*>(&lds.R[0][c][place<kChunk>(c, ks * 4 + g)]);
      }
      in_order();
      *reinterpret_cast<f32x4*>(lds.qs[w][lane]) = join(q[1], q[0]);
      if (w == 0 && g == 0) *reinterpret_cast<f32x2*>(lds.inv[c]) = (f32x2){rinv, sinv};
      f32x4 rw[ST], ws[ST][2];
#pragma unroll
      for (int t = 0; t < ST; t++) {
        ws[t][0] = ws[t][1] = (f32x4){0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int ks = 0; ks < 2; ks++) {
          ws[t][0] = mfma_h(Wf[t][ks][0], rl[ks], ws[t][0]);
          ws[t][1] = mfma_h(Wf[t][ks][0], rh[ks], ws[t][1]);
          ws[t][0] = mfma_h(Wf[t][ks][1], rh[ks], ws[t][0]);
        }
      }
      if (is_far(seen, j)) {
        const int lane = this_lane(), c = lane & 15, at = place<kChunk>(c, (w >> 1) * 4 + (lane >> 4)) + (w & 1) * 4;
        const h4 hi = *reinterpret_cast<const h4*>(&lds.R[0][c][at]), lo = *reinterpret_cast<const h4*>(&lds.R[1][c][at]);
        const f32x4 v = *reinterpret_cast<const f32x4*>(lds.bv[j & 1][w][lane]) * (inverse_of(rinv) * kLoUp);
        f32x4 Rj;  // what has become zero in a pair may have been less than nothing else is
#pragma unroll
        for (int r = 0; r < 4; r++) Rj[r] = larger(__builtin_fabsf(join((float)hi[r], (float)lo[r]) * kLoUp), 0x1p-60f);
        f32x4 size = sizes_of(Rj, v);
        const bool some = least > 0.f && most_of_all() < __builtin_inff();  // not a column of zeros, and finite
        if (!some || least == __builtin_inff()) size = (f32x4){} + (some ? 0x1p-60f : __builtin_inff());
        const int len = more ? kChunk : last, gone = far_rows(j, size);
        if (gone > 0) walk(j, gone);
        if (gone == len) {  // S is that behind the chunk, to which nothing is left to add
#pragma unroll
          for (int t = 0; t < ST; t++)
#pragma unroll
            for (int r = 0; r < 4; r++) S[t][r] = state_of(lane)[(t * 16 + r) * 16];
          if (keep == keep) keep = 1.f;
          rinv = 0.f;
          most_of_S();
        }
        lds_barrier();
        if (gone == len) sbound = most_of_all();
        __builtin_amdgcn_s_waitcnt(0x0f70);  // all that is on its way: what follows need not wait for more than it does without this
      }
#pragma unroll
      for (int t = 0; t < ST; t++) {
        rw[t] = of_quad(scale[t]) * rinv;
        S[t] *= keep;
      }
      in_order();
      load_back(here, 0);
#pragma unroll
      for (int t = 0; t < ST; t++) {
#pragma unroll
        for (int r = 0; r < 4; r++) S[t][r] = __builtin_fmaf(rw[t][r], join(ws[t][1][r], ws[t][0][r]), S[t][r]);
      }
    }
    lds_barrier();
#pragma unroll
    for (int t = 0; t < ST; t++)
#pragma unroll
      for (int r = 0; r < 4; r++) {
        const int d = d0 + t * 16 + r;
        if (mine && d < a.dk) a.state_out[st + (size_t)d * a.dv + col] = S[t][r];
      }
    return;
  }
  uint32_t vat[4], yat[4];  // of the lane's values in a chunk, bytes
#pragma unroll
  for (int r = 0; r < 4; r++) {
    vat[r] = ((uint32_t)(row0 + r) * a.ldv + col) * sizeof(T);
    yat[r] = mine ? ((uint32_t)(row0 + r) * a.ldy + col) * sizeof(T) : ~0u;
  }
  const uint32_t tri_at = block_of(w, 0) * kBlockBytes + lane * 16, tri_on = w < 2 ? 0 : kBlockBytes, factor_at = In::rows + quad0 * 4;
  h8 Pf[2][2];
  T v[4];
  float query, tri, beta, limits;
  auto load_tri = [&](const char* p) {
#pragma unroll
    for (int ks = 0; ks < 2; ks++) {  // (waves 4 and 5 have one block and take it twice)
      const h8* const q = reinterpret_cast<const h8*>(behind(p + ks * tri_on, tri_at));
#pragma unroll
      for (int n = 0; n < 2; n++) Pf[ks][n] = q[n * 64];
    }
    query = *reinterpret_cast<const float*>(behind(p + kRowQ * kChunk * 4, factor_at));
    tri = *reinterpret_cast<const float*>(behind(p + kRowP * kChunk * 4, factor_at));
  };
  auto load_limits = [&](const char* p) { limits = *reinterpret_cast<const float*>(behind(p, limits_at)); };
  auto load_values = [&](int t0, const char* p) {  // (behind the end: none)
    const auto rows = rows_of(a.v + (size_t)min(t0, end) * a.ldv + (size_t)head * a.dv, end - t0, a.ldv);
#pragma unroll
    for (int r = 0; r < 4; r++) v[r] = load_row<T>(rows, vat[r]);
    beta = *reinterpret_cast<const float*>(behind(p + kRowBeta * kChunk * 4, factor_at));
  };
  f32x4 bv;
  auto take_values = [&](int buf) {  // b v of a chunk and its largest value, to LDS
    const f32x4 rb = of_quad(beta);
    uint32_t m = 0;
#pragma unroll
    for (int r = 0; r < 4; r++) {
      bv[r] = rb[r] * (float)v[r];
      m = max(m, magnitude(bv[r]));
    }
    *reinterpret_cast<f32x4*>(lds.bv[buf][w][lane]) = bv;
    m = max_across_rows(m);
    if (g == 0) lds.vmost[c][w] = m;
  };
  int spoilt = kChunk;  // of the column, the first row of which something is not finite
  // What belongs to b v of a chunk, to LDS
  auto hand_over = [&](const char* p, int t0, int buf) {
    const u32x4 mv = *reinterpret_cast<const u32x4*>(lds.vmost[c]);
    uint32_t m = max(max(mv[0], mv[1]), max(mv[2], mv[3]));
    spoilt = (int)__float_as_uint(of_lane<4>(limits));
    if (__ballot(m >= kNotFinite)) {  // seldom: every wave looks for the first such value itself
      if (m >= kNotFinite) {
        const float* const b = reinterpret_cast<const float*>(p + In::rows) + kRowBeta * kChunk;
        m = 0;
        for (int r = min(end - t0, kChunk) - 1; r >= 0; r--) {
          const uint32_t x = magnitude(b[r] * (float)a.v[(size_t)(t0 + r) * a.ldv + (size_t)head * a.dv + col]);
          if (x >= kNotFinite) spoilt = min(spoilt, r);
          else m = max(m, x);
        }
#pragma unroll
        for (int r = 0; r < 4; r++)
          if (magnitude(bv[r]) >= kNotFinite) bv[r] = 0.f;
        *reinterpret_cast<f32x4*>(lds.bv[buf][w][lane]) = bv;
      }
    }
    if (w == 0 && g == 0) {
      lds.cols[c][0] = __uint_as_float(m);
      lds.cols[c][1] = spoilt < kChunk ? __builtin_nanf("") : of_lane<3>(limits);
    }
  };
  const char* ahead = nchunk > 1 ? here + head_step : here;  // the next chunk's
  load_values(begin, here);
  load_limits(here);
  load_tri(here);
  take_values(0);
  load_values(begin + kChunk, ahead);
  lds_barrier();
  hand_over(here, begin, 0);
  load_limits(ahead);
  lds_barrier();
  // Of the chunk before: its P R, its rows' factors, its first row that is not finite.  Its y is made while the next one's K S is.
  f32x4 yp = {0.f, 0.f, 0.f, 0.f}, yt = yp, yq = yp;
  int none = kChunk, gone = 0;  // gone: rows that went token by token, whose y is there
  auto finish = [&](int t0, int nrows) {
    const f32x4 qs = *reinterpret_cast<const f32x4*>(lds.qs[w][lane]);
    const f32x2 inv = *reinterpret_cast<const f32x2*>(lds.inv[c]);
    f32x4 y;  // (powers of two last: what a row of q or P has makes the other factor no larger than a result)
#pragma unroll
    for (int r = 0; r < 4; r++) y[r] = __builtin_fmaf(yt[r] * inv[0], yp[r], yq[r] * qs[r] * inv[1]);
    if (__ballot(none < kChunk)) {
#pragma unroll
      for (int r = 0; r < 4; r++)
        if (row0 + r >= none) y[r] = __builtin_nanf("");
    }
    const auto rows = rows_of(a.y + (size_t)t0 * a.ldy + (size_t)head * a.dv, nrows, a.ldy);
#pragma unroll
    for (int r = 0; r < 4; r++) store_row<T>(rows, row0 + r < gone ? ~0u : yat[r], (T)y[r]);
  };
  int t0 = begin;
  for (int j = 0; j < nchunk; j++, t0 += kChunk) {
    const char* const far = j + 2 < nchunk ? ahead + head_step : ahead;
    lds_barrier();
    take_values(~j & 1);
    load_values(t0 + 2 * kChunk, far);
    finish(j ? t0 - kChunk : t0, j ? kChunk : 0);  // (a chunk with another one behind it is whole)
    lds_barrier();
    h8 rh[2], rl[2];
#pragma unroll
    for (int ks = 0; ks < 2; ks++) {
      rl[ks] = *reinterpret_cast<const h8*>(&lds.R[1][c][place<kChunk>(c, ks * 4 + g)]);
      rh[ks] = *reinterpret_cast<const h8*>(&lds.R[0][c][place<kChunk>(c, ks * 4 + g)]);
    }
    none = spoilt;
    hand_over(ahead, t0 + kChunk, ~j & 1);  // (behind the last chunk: nobody's)
    load_limits(far);
    f32x4 p[2];
    p[0] = p[1] = (f32x4){0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int ks = 0; ks < 2; ks++) {
      if (2 * ks > w) break;
      p[0] = mfma_h(Pf[ks][0], rl[ks], p[0]);
      p[1] = mfma_h(Pf[ks][0], rh[ks], p[1]);
      p[0] = mfma_h(Pf[ks][1], rh[ks], p[0]);
    }
    yq = of_quad(query);
    yt = of_quad(tri);
    load_tri(ahead);
    yp = join(p[1], p[0]);
    ahead = far;
    gone = 0;
    if (is_far(lds.far, j)) {  // the same barriers as waves 0 to 3
      lds_barrier();
      lds_barrier();
      gone = gone_of();
      for (int i = 0; i <= gone; i++) lds_barrier();
    }
  }
  lds_barrier();
  finish(t0 - kChunk, end - (t0 - kChunk));
}

// ---------------------------------------------------------------------------
// Host side
// ---------------------------------------------------------------------------
constexpr size_t kPassBytes = (size_t)256 << 20;  // scratch of a pair of launches, about: longer calls go out in several
static int key_steps(int dk) { return dk <= 64 ? 2 : dk <= 128 ? 4 : 8; }
static size_t chunk_bytes(int heads, int key_heads, int dk, int parts) {
  const int ks = key_steps(dk), head = ks == 2 ? HeadLayout<2>::bytes : ks == 4 ? HeadLayout<4>::bytes : HeadLayout<8>::bytes;
  return (size_t)heads * head + (size_t)key_heads * key_bytes(ks * 32, parts);
}
// Chunks of a pair of launches.  Prompts of kDeltaChunkLeast rows and more have rows / kDeltaChunkLeast + 1 at most.
static size_t most_chunks(size_t per, int T) {
  const size_t by_rows = (size_t)T / kDeltaChunkLeast + 1, by_bytes = std::max<size_t>(kPassBytes / per, 16);
  return std::min(by_rows, by_bytes);
}

size_t delta_chunk_bytes(const frhip_delta& p, int elem, int T) {
  if (T < kDeltaChunkLeast) return 0;
  const size_t per = chunk_bytes(p.heads, p.key_heads, p.key_dim, elem == 4 ? 2 : 1);
  return most_chunks(per, T) * per;
}

bool delta_chunks_fit(const frhip_delta& p, int elem, const int32_t* start, int nseq, int T) {
  size_t chunks = 0;
  int longest = 0;
  for (int i = 0; i < nseq; i++) {
    const int len = start[i + 1] - start[i];
    longest = std::max(longest, len);
    chunks += len ? (len - 1) / kChunk + 1 : 0;
  }
  return longest >= kDeltaChunkLeast && chunks <= most_chunks(chunk_bytes(p.heads, p.key_heads, p.key_dim, elem == 4 ? 2 : 1), T);
}

template <class T, int KS>
static int chunk_launch(const DeltaArgs<T>& a, const DeltaTable& tab, char* keys, char* heads, hipStream_t st) {
  const int chunks = tab.chunk[a.nseq], slices = (a.dv + 15) / 16;
  if (chunks > 0) {
    hipLaunchKernelGGL((delta_prep_kernel<T, KS>), dim3(chunks, a.heads), dim3(256), 0, st, a, tab, keys, heads);
    if (int rc = check_launch("delta_seq")) return rc;
  }
  hipLaunchKernelGGL((delta_scan_kernel<T, KS>), dim3(a.nseq * a.heads * slices), dim3(512), 0, st, a, tab, keys, heads);
  return check_launch("delta_seq");
}

template <class T>
int delta_chunk_run(const DeltaArgs<T>& args, const int* seqs, int nseq, const int32_t* start, int rows, void* workspace, hipStream_t st) {
  DeltaArgs<T> a = args;
  const int nkh = a.heads / a.share, steps = key_steps(a.dk);
  const size_t per = chunk_bytes(a.heads, nkh, a.dk, kParts<T>), most = most_chunks(per, rows);
  const int together = std::min(kSeqTable, (1 << 22) / (a.heads * ((a.dv + 15) / 16)));  // prompts of a launch, which has less than 2^32 threads
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
      const int s = seqs[i], len = start[s + 1] - start[s], chunks = (len ? (len - 1) / kChunk + 1 : 0) - done;
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
