// Tiles of 64 or 128 rows whose operands waves of their own bring to LDS, shared by gemm_ring.hip and linear.hip (gemm_ring.hip has the
// reasons and the figures).
#pragma once

#include "gemm_device.h"

#pragma clang fp contract(off)

namespace frhip {

constexpr int kRingLoaders = 4, kRingThreads = 64 * (4 + kRingLoaders), kRingMostBlocks = 8;
// K-steps in LDS: as many as 160 KB hold, up to four; tiles of 64 rows and up to 96 columns run two workgroups on a compute unit
constexpr int ring_stages(int bm, int w) { return bm == 128 && w > 6 ? 3 : 4; }
static_assert(4 * (128 * 128 + 6 * 4096) <= 160 * 1024 && 3 * (128 * 128 + 8 * 4096) <= 160 * 1024 && 4 * (64 * 128 + 8 * 4096) <= 160 * 1024, "LDS");

// The operands of a tile: rows of A and B, lda and ldb elements apart
struct RingOperands {
  const h1* A;
  const unsigned char* B;  // binary16
  int M, N, lda, ldb;
};

// The waves that load.  TAIL: the last step has krest of its 64 k (a multiple of 8); the places of the others get what lies at the step's
// begin, and what multiplies takes zeros there.
template <int BM, int S, int W, bool TAIL = false>
__device__ __forceinline__ void ring_loader(const RingOperands& o, unsigned char* smem, int stage, int p, int m0, int n0, int kbase, int nk,
                                            int lane, int krest = 64) {
  constexpr int NA = BM / 8 / kRingLoaders, NL = NA + W;
  static_assert(S == 3 || S == 4, "the waits of the last steps");
  static_assert((S - 1) * NL <= 63, "the wait counter's range");
  const int M = o.M, N = o.N, lr = lane >> 3;
  unsigned va[NA], vb[W];
#pragma unroll
  for (int i = 0; i < NA; i++) {  // groups of 8 rows; rows past the matrix repeat its last one and are never stored
    const int g = p + kRingLoaders * i;
    va[i] = (unsigned)(min(m0 + g * 8 + lr, M - 1) - m0) * (unsigned)(o.lda * 2) + (((lane & 7) ^ lr ^ (g & 1)) * 16);
  }
#pragma unroll
  for (int i = 0; i < W; i++) {
    const int g = p + kRingLoaders * i;
    vb[i] = (unsigned)(min(n0 + g * 8 + lr, N - 1) - n0) * (unsigned)(o.ldb * 2) + (((lane & 7) ^ lr ^ (g & 1)) * 16);
  }
  const unsigned char* ak = uniform_ptr(reinterpret_cast<const unsigned char*>(o.A) + ((size_t)m0 * o.lda + kbase) * 2);
  const unsigned char* bk = uniform_ptr(o.B + ((size_t)n0 * o.ldb + kbase) * 2);
  const unsigned lds0 = (unsigned)(size_t)((__attribute__((address_space(3))) unsigned char*)smem) + p * 1024;
  unsigned at = lds0;
  const unsigned end = lds0 + S * stage;
  int issued = 0;
  auto issue = [&] {
    if constexpr (TAIL) {
      if (++issued == nk) {  // all groups of this wave have one parity, so a lane has one k-segment
        const unsigned seg = (lane & 7) ^ lr ^ (p & 1), back = seg * 8 >= (unsigned)krest ? seg * 16 : 0;
#pragma unroll
        for (int i = 0; i < W; i++) vb[i] -= back;
#pragma unroll
        for (int i = 0; i < NA; i++) va[i] -= back;
      }
    }
#pragma unroll
    for (int i = 0; i < W; i++) load_lds_saddr(vb[i], bk, at + BM * 128 + i * (kRingLoaders * 1024));
#pragma unroll
    for (int i = 0; i < NA; i++) load_lds_saddr(va[i], ak, at + i * (kRingLoaders * 1024));
    ak += 128;
    bk += 128;
    at += stage;
    at = at == end ? lds0 : at;
  };
#pragma unroll
  for (int i = 0; i < S - 1; i++)
    if (i < nk) issue();
  int k = 0;
  for (; k + S - 1 < nk; k++) {
    wait_loads<(S - 2) * NL>();  // step k has landed
    step_barrier();              // and step k - 1 has been read
    issue();                     // step k + S - 1, into the slot of step k - 1
  }
  for (; k < nk; k++) {
    const int behind = nk - 1 - k;
    if (S > 3 && behind >= 2) wait_loads<2 * NL>();
    else if (behind >= 1) wait_loads<NL>();
    else wait_loads<0>();
    step_barrier();
  }
}

}  // namespace frhip
