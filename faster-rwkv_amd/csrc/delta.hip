// The gated delta rule: a matrix per head as the state of a recurrence.
//
//   S = a S + b k (v - a S^T k)^T,   y = scale S^T q,   a = exp(A dt'), dt' = softplus(dt + dt_bias), b = sigmoid(beta)
//
// with q and k divided by their length.  S is [key][value] and its columns do not mix: a column of S, v and y is a recurrence of its own.
#include <algorithm>
#include <cstring>

#include "delta.h"
#include "spans.h"

#pragma clang fp contract(off)

namespace frhip {

// ---------------------------------------------------------------------------
// Token by token.  A wave has CL x 4 columns of a head, and CL lanes of a row of S: lane l has its columns 4 (l % CL) and the R keys from R (l / CL) on.
// Bound by memory where there are many sequences of one token, the states once in and once out: 64 of 32 heads 128 x 128 in 55 us, 4.9 TB/s.  A prompt's
// tokens are bound by the instructions of its waves, of which a compute unit has few: so sums over rows of lanes leave each with a column of its own, whose
// value and result it works out, the lengths are a wave's scalars, and 64 tokens' gates are evaluated at once, a lane each.
// ---------------------------------------------------------------------------
// R elements as they are in memory, the first n of them.  WHOLE: all or none, and p can be read in either case
template <class T, int R, bool WHOLE>
struct RawRow {
  static constexpr int P = R < kGroup<T> ? R : kGroup<T>;
  typedef T any __attribute__((ext_vector_type(P), aligned(sizeof(T))));
  any v[R / P];
  __device__ __forceinline__ void load(const T* p, int n) {
    if (WHOLE || n >= R) {
#pragma unroll
      for (int k = 0; k < R / P; k++) v[k] = *reinterpret_cast<const any*>(p + k * P);
    }
    if (!WHOLE && n < R) {
#pragma unroll
      for (int i = 0; i < R; i++) v[i / P][i % P] = i < n ? p[i] : (T)0.f;
    }
  }
  __device__ __forceinline__ float operator[](int i) const { return (float)v[i / P][i % P]; }
};

// Two values' sums of each lane's and the one's 32 (16) away: the first value's in the even halves (rows), the second one's in the odd ones
__device__ __forceinline__ float halves_sum(float x, float y) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(y), false, false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}
__device__ __forceinline__ float rows_sum(float x, float y) {
  const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(y), false, false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}
// Value j's sum over the lanes that share lane % CL, in row j of 16 lanes
template <int CL>
__device__ __forceinline__ float sum_by_row(float v0, float v1, float v2, float v3) {
  float v = rows_sum(halves_sum(v0, v2), halves_sum(v1, v3));
  v += dpp_mov<0x128>(v);  // row_ror:8
  if constexpr (CL == 4) v += dpp_mov<0x124>(v);
  return v;
}
// What the four rows of lanes have, to all of them
__device__ __forceinline__ void of_rows(float v, float (&to)[4]) {
  const uint32_t u = __float_as_uint(v);
  const auto h = __builtin_amdgcn_permlane32_swap(u, u, false, false);
  const auto lo = __builtin_amdgcn_permlane16_swap(h[0], h[0], false, false), hi = __builtin_amdgcn_permlane16_swap(h[1], h[1], false, false);
  to[0] = __uint_as_float(lo[0]);
  to[1] = __uint_as_float(lo[1]);
  to[2] = __uint_as_float(hi[0]);
  to[3] = __uint_as_float(hi[1]);
}
__device__ __forceinline__ float lane_of(float v, int lane) { return __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(v), lane)); }

template <class T, int CL, int R, bool ONE, bool WHOLE>
__global__ __launch_bounds__(256) void delta_step_kernel(DeltaArgs<T> a, DeltaTable tab) {
  constexpr int W = 4 * CL;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int slices = (a.dv + W - 1) / W, unit = blockIdx.x * 4 + wave;
  if (unit >= a.heads * slices) return;  // whole waves; nothing here waits for another one
  const int head = unit / slices, kh = head / a.share, c = (unit - head * slices) * W + (lane % CL) * 4, d0 = lane / CL * R, col = c + lane / 16;
  const int nc = a.dv - c, nd = a.dk - d0;
  const bool mine = (lane & 15) < CL && col < a.dv;
  const float rate = a.A ? finite_rate(a.A[head]) : 1.f, bias = a.dt_bias ? a.dt_bias[head] : 0.f;
  const size_t kat = (size_t)kh * a.dk + (nd > 0 ? d0 : 0), vat = (size_t)head * a.dv + (col < a.dv ? col : 0);
  const int nseq = ONE ? a.rows : a.nseq;
  RawRow<T, R, WHOLE> qr, kr;
  T vr;
  float keeps, writes;  // of this token, or of 64 tokens, a lane each
  auto request = [&](int t) {
    kr.load(a.k + (size_t)t * a.ldk + kat, nd);
    qr.load(a.q + (size_t)t * a.ldq + kat, nd);
    vr = a.v[(size_t)t * a.ldv + vat];
  };
  auto gates = [&](int t) {
    const float dt = (float)a.dt[(size_t)t * a.lddt + head], raw = (float)a.beta[(size_t)t * a.ldbeta + head];
    const float log = log_decay(a, dt, rate, bias);
    keeps = log < __builtin_inff() ? decay_f(log) : __builtin_nanf("");  // one that grows without end is no number, as chunk by chunk
    writes = a.sigmoid ? sigmoid_f<true>(raw) : raw;
  };
  for (int i = blockIdx.y; i < nseq; i += gridDim.y) {
    const size_t st = ((size_t)(ONE ? i : tab.seq[i]) * a.heads + head) * a.dk * a.dv + c;
    const int begin = ONE ? i : tab.start[i], end = ONE ? i + 1 : tab.end[i];
    if (ONE || begin < end) request(begin);
    float S[R][4];
#pragma unroll
    for (int r = 0; r < R; r++) load_group<float, 4>(S[r], a.state + st + (size_t)(r < nd ? d0 + r : 0) * a.dv, r < nd ? nc : 0);
    if (ONE) gates(begin);
    for (int t = begin; t < end; t++) {
      const int nth = (t - begin) & 63;
      if (!ONE && nth == 0) gates(min(t + lane, end - 1));
      float q[R], k[R];
#pragma unroll
      for (int r = 0; r < R; r++) {
        q[r] = !WHOLE || nd > 0 ? qr[r] : 0.f;
        k[r] = !WHOLE || nd > 0 ? kr[r] : 0.f;
      }
      const float v = (float)vr, keep = ONE ? keeps : lane_of(keeps, nth), b = ONE ? writes : lane_of(writes, nth);
      if (!ONE) request(min(t + 1, end - 1));  // on its way while this one is worked on
      float kk = 0.f, qq = 0.f, qk = 0.f, kS[4] = {}, qS[4] = {};
#pragma unroll
      for (int r = 0; r < R; r++) {
        kk = __builtin_fmaf(k[r], k[r], kk);
        qq = __builtin_fmaf(q[r], q[r], qq);
        qk = __builtin_fmaf(q[r], k[r], qk);
#pragma unroll
        for (int j = 0; j < 4; j++) {
          kS[j] = __builtin_fmaf(k[r], S[r][j], kS[j]);
          qS[j] = __builtin_fmaf(q[r], S[r][j], qS[j]);
        }
      }
      const float sums = sum_by_row<CL>(kk, qq, qk, qq), ks = sum_by_row<CL>(kS[0], kS[1], kS[2], kS[3]), qs = sum_by_row<CL>(qS[0], qS[1], qS[2], qS[3]);
      float kn = 1.f, qn = a.scale;
      if (a.eps >= 0.f) {
        kn = __builtin_amdgcn_rsqf(lane_of(sums, 0) + a.eps);
        qn = __builtin_amdgcn_rsqf(lane_of(sums, 16) + a.eps) * a.scale;
      }
      const float u = kn * (b * (v - keep * kn * ks));
      float to[4];
      of_rows(u, to);
#pragma unroll
      for (int r = 0; r < R; r++)
#pragma unroll
        for (int j = 0; j < 4; j++) S[r][j] = __builtin_fmaf(k[r], to[j], keep * S[r][j]);
      if (mine) a.y[(size_t)t * a.ldy + vat] = (T)(qn * __builtin_fmaf(keep, qs, lane_of(sums, 32) * u));
    }
#pragma unroll
    for (int r = 0; r < R; r++)
      if (r < nd && nc > 0) store_group<float, 4>(a.state_out + st + (size_t)(d0 + r) * a.dv, S[r], nc);
  }
}

// ---------------------------------------------------------------------------
// Host side
// ---------------------------------------------------------------------------
template <class T, int CL, bool ONE, bool WHOLE>
static int step_launch_of(const DeltaArgs<T>& a, const DeltaTable& tab, int nseq, hipStream_t st) {
  const int slices = (a.dv + 4 * CL - 1) / (4 * CL), units = a.heads * slices;
  const dim3 grid((units + 3) / 4, nseq < 65535 ? nseq : 65535);
  const int rows = (a.dk + 64 / CL - 1) / (64 / CL);  // keys of a lane
  if (rows <= 4) hipLaunchKernelGGL((delta_step_kernel<T, CL, 4, ONE, WHOLE>), grid, dim3(256), 0, st, a, tab);
  else if (rows <= 8) hipLaunchKernelGGL((delta_step_kernel<T, CL, 8, ONE, WHOLE>), grid, dim3(256), 0, st, a, tab);
  else if (rows <= 16) hipLaunchKernelGGL((delta_step_kernel<T, CL, 16, ONE, WHOLE>), grid, dim3(256), 0, st, a, tab);
  else if constexpr (CL == 8) hipLaunchKernelGGL((delta_step_kernel<T, CL, 32, ONE, WHOLE>), grid, dim3(256), 0, st, a, tab);
  return check_launch("delta");
}
template <class T, int CL, bool ONE>
static int step_launch(const DeltaArgs<T>& a, const DeltaTable& tab, int nseq, hipStream_t st) {
  const int rows = (a.dk + 64 / CL - 1) / (64 / CL), part = rows <= 4 ? 4 : rows <= 8 ? 8 : rows <= 16 ? 16 : 32;
  return a.dk % part == 0 && a.dv % 4 == 0 ? step_launch_of<T, CL, ONE, true>(a, tab, nseq, st) : step_launch_of<T, CL, ONE, false>(a, tab, nseq, st);
}

static int delta_check_params(const frhip_delta* p) {
  if (!p) return set_error(FRHIP_EINVAL, "delta: null pointer");
  if (p->heads <= 0 || p->key_heads <= 0 || p->heads % p->key_heads != 0) return set_error(FRHIP_ESHAPE, "delta: heads must be a multiple of key_heads");
  if (p->heads > kMostHeads) return set_error(FRHIP_ESHAPE, "delta: up to 65535 heads");
  if (p->key_dim < 1 || p->key_dim > kMostDim || p->value_dim < 1 || p->value_dim > kMostDim) return set_error(FRHIP_ESHAPE, "delta: dimensions must be 1 to 256");
  if ((long long)p->heads * p->value_dim > kMostPitch || (long long)p->key_heads * p->key_dim > kMostPitch)
    return set_error(FRHIP_ESHAPE, "delta: a row may have up to 2^23 elements");
  if (off_grid(4, {p->A, p->dt_bias})) return set_error(FRHIP_EINVAL, "delta: pointer not aligned to its element");
  if (!(p->norm_eps < 3e38f)) return set_error(FRHIP_EINVAL, "delta: norm_eps must be a number, or negative");
  return 0;
}

struct DeltaCall {
  const void *q, *k, *v, *dt, *beta;
  int ldq, ldk, ldv, lddt, ldbeta;
  const float* state;
  float* state_out;
  void* y;
  int ldy, dtype;
};

static int delta_check(const frhip_delta& p, const DeltaCall& c, size_t row0, size_t rows, size_t nstate) {
  if (c.dtype != FRHIP_F16 && c.dtype != FRHIP_F32) return set_error(FRHIP_EINVAL, "delta: dtype must be F16 or F32");
  const int kn = p.key_heads * p.key_dim, vn = p.heads * p.value_dim;
  if (c.ldq < kn || c.ldk < kn || c.ldv < vn || c.lddt < p.heads || c.ldbeta < p.heads || c.ldy < vn)
    return set_error(FRHIP_ESHAPE, "delta: rows closer than their elements");
  for (int ld : {c.ldq, c.ldk, c.ldv, c.lddt, c.ldbeta, c.ldy})
    if (ld > kMostPitch) return set_error(FRHIP_ESHAPE, "delta: rows more than 2^23 elements apart");
  if (!c.state || !c.state_out || (rows && (!c.q || !c.k || !c.v || !c.dt || !c.beta || !c.y))) return set_error(FRHIP_EINVAL, "delta: null pointer");
  const size_t elem = c.dtype == FRHIP_F16 ? 2 : 4, sbytes = nstate * p.heads * p.key_dim * p.value_dim * 4, pbytes = (size_t)p.heads * 4;
  if (off_grid(elem, {c.q, c.k, c.v, c.dt, c.beta, c.y}) || off_grid(4, {c.state, c.state_out}))
    return set_error(FRHIP_EINVAL, "delta: pointer not aligned to its element");
  if (spans_clash(c.state, c.state_out, sbytes)) return set_error(FRHIP_EINVAL, "delta: states overlap in part");
  if (spans_meet(c.state_out, sbytes, p.A, pbytes) || spans_meet(c.state_out, sbytes, p.dt_bias, pbytes))
    return set_error(FRHIP_EINVAL, "delta: an output overlaps a parameter");
  if (!rows) return 0;
  struct In { const void* p; int ld, cols; };
  const char* y = static_cast<const char*>(c.y) + row0 * c.ldy * elem;
  const size_t ybytes = ((rows - 1) * c.ldy + vn) * elem;
  if (spans_meet(y, ybytes, p.A, pbytes) || spans_meet(y, ybytes, p.dt_bias, pbytes)) return set_error(FRHIP_EINVAL, "delta: an output overlaps a parameter");
  for (const In& in : {In{c.q, c.ldq, kn}, In{c.k, c.ldk, kn}, In{c.v, c.ldv, vn}, In{c.dt, c.lddt, p.heads}, In{c.beta, c.ldbeta, p.heads}}) {
    const char* r = static_cast<const char*>(in.p) + row0 * in.ld * elem;
    if (rows_overlap(r, in.ld, y, c.ldy, rows, in.cols, vn, elem) || spans_meet(r, ((rows - 1) * in.ld + in.cols) * elem, c.state_out, sbytes))
      return set_error(FRHIP_EINVAL, "delta: an output overlaps what is read");
  }
  if (spans_meet(y, ybytes, c.state, sbytes) || spans_meet(y, ybytes, c.state_out, sbytes)) return set_error(FRHIP_EINVAL, "delta: an output overlaps what is read");
  return 0;
}

template <class T>
static DeltaArgs<T> delta_args(const frhip_delta& p, const DeltaCall& c) {
  DeltaArgs<T> a;
  memset(&a, 0, sizeof(a));
  a.q = static_cast<const T*>(c.q);
  a.k = static_cast<const T*>(c.k);
  a.v = static_cast<const T*>(c.v);
  a.dt = static_cast<const T*>(c.dt);
  a.beta = static_cast<const T*>(c.beta);
  a.y = static_cast<T*>(c.y);
  a.A = p.A;
  a.dt_bias = p.dt_bias;
  a.state = c.state;
  a.state_out = c.state_out;
  a.ldq = c.ldq;
  a.ldk = c.ldk;
  a.ldv = c.ldv;
  a.lddt = c.lddt;
  a.ldbeta = c.ldbeta;
  a.ldy = c.ldy;
  a.heads = p.heads;
  a.share = p.heads / p.key_heads;
  a.dk = p.key_dim;
  a.dv = p.value_dim;
  a.scale = p.scale;
  a.eps = p.norm_eps;
  a.softplus = p.dt_softplus != 0;
  a.sigmoid = p.beta_sigmoid != 0;
  return a;
}

template <class T>
static int delta_one_run(const frhip_delta& p, const DeltaCall& c, int rows, hipStream_t st) {
  DeltaArgs<T> a = delta_args<T>(p, c);
  a.rows = rows;
  DeltaTable none;
  memset(&none, 0, sizeof(none));
  return step_launch<T, 8, true>(a, none, rows, st);
}

// Rows, at least, of the prompts of a call that go chunk by chunk.  Either form's time (us), 32 heads 128 x 128, by the rows of each prompt:
//   one prompt    8: 9 / 17   16: 13 / 16   20: 16 / 16   32: 23 / 17   64: 42 / 17
//   16 prompts    8: 22 / 77  16: 35 / 77   32: 60 / 77   48: 85 / 79   64: 110 / 80
// A chunk of few rows costs what a whole one does, which counts where there are more of them than compute units to work on them.  For the same reason short
// prompts join long ones if they are few: launches that are there anyway take them for nothing (nine prompts of 24 heads 64 x 64, four of them of 31 rows at
// most: 62 -> 45 us).
static int chunk_least(const frhip_delta& p, const int32_t* start, int n, int elem, int rows) {
  const long long each = (long long)p.heads * ((p.value_dim + 15) / 16), room = 2LL * compute_units();  // workgroups
  int some = 0;
  for (int i = 0; i < n; i++) some += start[i + 1] - start[i] >= kDeltaChunkLeast;
  const int least = some * each <= room ? kDeltaChunkLeast : 2 * kDeltaChunkLeast;
  int below = 0;
  for (int i = 0; i < n; i++) below += start[i + 1] - start[i] < least;
  return below < n && below * each <= room && delta_chunks_fit(p, elem, start, n, rows) ? 0 : least;
}

template <class T>
static int delta_seq_run(const frhip_delta& p, const DeltaCall& c, int nseq, const int32_t* start, void* workspace, hipStream_t st) {
  DeltaArgs<T> a = delta_args<T>(p, c);
  const size_t per = (size_t)p.heads * p.key_dim * p.value_dim;
  const int rows = start[nseq] - start[0];
  for (int s0 = 0; s0 < nseq; s0 += kSeqTable) {  // short prompts token by token, the others chunk by chunk
    const int n = nseq - s0 < kSeqTable ? nseq - s0 : kSeqTable;
    a.state = c.state + (size_t)s0 * per;
    a.state_out = c.state_out + (size_t)s0 * per;
    DeltaTable tab;
    memset(&tab, 0, sizeof(tab));
    const int least = chunk_least(p, start + s0, n, sizeof(T), rows);
    int many[kSeqTable], nmany = 0;
    a.nseq = 0;
    for (int i = 0; i < n; i++) {
      const int from = start[s0 + i], to = start[s0 + i + 1];
      if (to - from >= least) {
        many[nmany++] = i;
        continue;
      }
      tab.start[a.nseq] = from;
      tab.end[a.nseq] = to;
      tab.seq[a.nseq++] = i;
    }
    std::sort(many, many + nmany, [&](int x, int y) {  // long ones first
      const int lx = start[s0 + x + 1] - start[s0 + x], ly = start[s0 + y + 1] - start[s0 + y];
      return lx != ly ? lx > ly : x < y;
    });
    if (a.nseq)
      if (int rc = step_launch<T, 4, false>(a, tab, a.nseq, st)) return rc;
    if (nmany)
      if (int rc = delta_chunk_run<T>(a, many, nmany, start + s0, rows, workspace, st)) return rc;
  }
  return 0;
}

}  // namespace frhip

using namespace frhip;

extern "C" int frhip_delta_one(const frhip_delta* p, int rows, const void* q, int ldq, const void* k, int ldk, const void* v, int ldv, const void* dt,
                               int lddt, const void* beta, int ldbeta, const float* state, float* state_out, void* y, int ldy, int dtype,
                               frhip_stream s) {
  if (int rc = delta_check_params(p)) return rc;
  if (rows < 0 || rows > kMostRows) return set_error(FRHIP_ESHAPE, "delta_one: rows must be 0 to 2^30");
  const DeltaCall c = {q, k, v, dt, beta, ldq, ldk, ldv, lddt, ldbeta, state, state_out, y, ldy, dtype};
  if (int rc = delta_check(*p, c, 0, rows, rows)) return rc;
  if (rows == 0) return 0;
  hipStream_t st = static_cast<hipStream_t>(s);
  return dtype == FRHIP_F16 ? delta_one_run<h1>(*p, c, rows, st) : delta_one_run<float>(*p, c, rows, st);
}

extern "C" size_t frhip_delta_workspace_bytes(const frhip_delta* p, int nseq, int T) {
  if (nseq <= 0 || T <= 0 || delta_check_params(p)) return 0;
  const size_t bytes = delta_chunk_bytes(*p, 4, T) > delta_chunk_bytes(*p, 2, T) ? delta_chunk_bytes(*p, 4, T) : delta_chunk_bytes(*p, 2, T);
  return (bytes + 255) / 256 * 256;
}

extern "C" int frhip_delta_seq(const frhip_delta* p, int nseq, const int32_t* seq_start, const void* q, int ldq, const void* k, int ldk, const void* v,
                               int ldv, const void* dt, int lddt, const void* beta, int ldbeta, const float* state, float* state_out, void* y, int ldy,
                               int dtype, void* workspace, frhip_stream s) {
  if (int rc = delta_check_params(p)) return rc;
  if (int rc = check_seqs(nseq, seq_start, kMostTime, "delta_seq: seq_start must be nseq + 1 row numbers up to 2^28 that do not descend")) return rc;
  const DeltaCall c = {q, k, v, dt, beta, ldq, ldk, ldv, lddt, ldbeta, state, state_out, y, ldy, dtype};
  const size_t row0 = nseq ? seq_start[0] : 0, rows = nseq ? seq_start[nseq] - seq_start[0] : 0;
  if (int rc = delta_check(*p, c, row0, rows, nseq)) return rc;
  if (nseq == 0) return 0;
  if (frhip_delta_workspace_bytes(p, nseq, (int)rows) > 0) {
    if (!workspace) return set_error(FRHIP_EINVAL, "delta_seq: null workspace");
    if (reinterpret_cast<uintptr_t>(workspace) % 16 != 0) return set_error(FRHIP_EINVAL, "delta_seq: workspace must be 16-byte aligned");
  }
  hipStream_t st = static_cast<hipStream_t>(s);
  return dtype == FRHIP_F16 ? delta_seq_run<h1>(*p, c, nseq, seq_start, workspace, st) : delta_seq_run<float>(*p, c, nseq, seq_start, workspace, st);
}
