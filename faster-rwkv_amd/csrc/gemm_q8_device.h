// Tiles whose uint8 codes waves of their own dequantise on their way into LDS, shared by gemm_q8.hip (which has the form, its reasons and
// the figures) and linear.hip.
#pragma once

#include <type_traits>

#include "gemm_device.h"

#pragma clang fp contract(off)

namespace frhip {

constexpr int kQ8Stages = 4;  // K-steps of X in LDS: one multiplied, three in flight
constexpr int kQ8Codes = 3;   // K-steps of codes, per producer
constexpr int q8_max_blocks(int bm) { return bm == 128 ? 6 : 8; }  // of 32 columns: what 160 KB hold
constexpr int kQ8Producers = 8;
// A producer's codes, ry and my of a step; its rx and mx behind the slots.  Tiles of up to w blocks of 32 columns.
__host__ __device__ constexpr int q8_blocks_before(int p, int w) {
  const int r = 2 * w % kQ8Producers;
  return p * (2 * w / kQ8Producers) + (p < r ? p : r);
}
__host__ __device__ constexpr int q8_producer_at(int p, int w) { return kQ8Codes * (q8_blocks_before(p, w) * 1024 + p * 256) + p * 256; }
constexpr int q8_lds_bytes(int bm, int w) { return kQ8Stages * bm * 128 + 2 * w * 4096 + q8_producer_at(kQ8Producers, w); }
static_assert(128 * sums_pitch(6) * 4 <= q8_lds_bytes(128, 6) && 128 * sums_pitch(2) * 4 <= q8_lds_bytes(128, 2) &&
                  64 * sums_pitch(8) * 4 <= q8_lds_bytes(64, 8) && 64 * sums_pitch(2) * 4 <= q8_lds_bytes(64, 2), "the sums fit");
static_assert(q8_lds_bytes(128, q8_max_blocks(128)) <= 160 * 1024 && q8_lds_bytes(64, q8_max_blocks(64)) <= 160 * 1024, "LDS of a compute unit");

// few_dequant's two values, the same bits, in 8 instructions: a code in the low byte of a binary16 is the subnormal q 2^-24, which
// v_fma_mix_f32 reads as it is; c24 is c 2^24 and the product the same real number (c ry is far from fp32's subnormals).
template <int HI>
__device__ __forceinline__ h2 q8_dequant(uint32_t word, float c24, float mx, h2 ry, h2 my) {
  const uint32_t q = __builtin_amdgcn_perm(0u, word, HI ? 0x0c030c02u : 0x0c010c00u);
  float w0, w1;
  asm("v_fma_mix_f32 %0, %1, %2, %3 op_sel_hi:[1,0,0]" : "=v"(w0) : "v"(q), "v"(mul_h<0>(c24, ry)), "v"(add_h<0>(mx, my)));
  asm("v_fma_mix_f32 %0, %1, %2, %3 op_sel:[1,0,0] op_sel_hi:[1,0,0]" : "=v"(w1) : "v"(q), "v"(mul_h<1>(c24, ry)), "v"(add_h<1>(mx, my)));
  return (h2){(h1)w0, (h1)w1};
}

// NB: blocks of 16 columns of this wave (p, p + 8); rows of A are lda elements apart
template <int BM, int NB>
__device__ __forceinline__ void q8_producer(const GemmSeg& sg, unsigned char* smem, int maxw, int p, int m0, int n0, int M, int K, int lda,
                                            int kbase, int nk, int lane) {
  constexpr int NA = BM / 8 / kQ8Producers, NC = NB + 1;  // loads of a step: 8 rows of X each; 16 columns each, and the scales
  const int N = sg.N, lr = lane >> 3, row16 = lane & 15, grp = lane >> 4;
  unsigned char* const bsm = smem + kQ8Stages * BM * 128;
  const int slot_bytes = (q8_blocks_before(p + 1, maxw) - q8_blocks_before(p, maxw)) * 1024 + 256;
  unsigned char* const own = bsm + 2 * maxw * 4096 + q8_producer_at(p, maxw);
  const unsigned lds0 = (unsigned)(size_t)((__attribute__((address_space(3))) unsigned char*)smem);
  const unsigned own_lds = lds0 + (unsigned)(own - smem);
  unsigned va[NA], vb[NB + 1];
#pragma unroll
  for (int i = 0; i < NA; i++) {  // rows past the matrix repeat its last row and are never stored
    const int g = p * NA + i;
    va[i] = (unsigned)(min(m0 + g * 8 + lr, M - 1) - m0) * (unsigned)(lda * 2) + (((lane & 7) ^ lr ^ (g & 1)) * 16);
  }
#pragma unroll
  for (int t = 0; t < NB; t++) {
    const int col = min(n0 + (p + kQ8Producers * t) * 16 + (lane >> 2), N - 1) - n0;
    vb[t] = (unsigned)col * (unsigned)K + (((lane & 3) ^ (lane >> 4)) * 16);
  }
  const unsigned char* const abase = uniform_ptr(reinterpret_cast<const unsigned char*>(sg.A) + ((size_t)m0 * lda + kbase) * 2);
  const unsigned char* const bbase = uniform_ptr(sg.B + (size_t)n0 * K + kbase);
  const h1* scale_k = (lane < 32 ? sg.ry : sg.my) + kbase + (lane & 31) * 2;  // lanes 0..31 ry, 32..63 my, two each
  {
    // rx (lanes 0..31) and mx of the wave's up to 64 columns, two a lane
    const int c = min(n0 + (p + kQ8Producers * ((lane & 31) >> 3)) * 16 + (lane & 7) * 2, N - 2);
    load_lds_dword((lane < 32 ? sg.rx : sg.mx) + c, own_lds + kQ8Codes * slot_bytes);
  }
  // Where the next loads come from and go to, in the order of their steps
  const unsigned char *ak = abase, *bk = bbase;
  unsigned a_lds = lds0 + p * (NA * 1024), c_lds = own_lds;
  const unsigned a_end = a_lds + kQ8Stages * (BM * 128), c_end = own_lds + kQ8Codes * slot_bytes;
  auto issue_a = [&] {
#pragma unroll
    for (int i = 0; i < NA; i++) load_lds_saddr(va[i], ak, a_lds + i * 1024);
    ak += 128;
    a_lds += BM * 128;
    a_lds = a_lds == a_end ? a_end - kQ8Stages * (BM * 128) : a_lds;
  };
  auto issue_codes = [&] {
#pragma unroll
    for (int t = 0; t < NB; t++) load_lds_saddr(vb[t], bk, c_lds + 256 + t * 1024);
    load_lds_dword(scale_k, c_lds);
    bk += 64;
    scale_k += 64;
    c_lds += slot_bytes;
    c_lds = c_lds == c_end ? own_lds : c_lds;
  };
  struct Step {  // a lane's codes of one step, and the scales of their rows
    u32x4 q[NB + 1];
    h8 ry[2], my[2];
  };
  const unsigned char* from = own;  // the slot that is read next
  auto read = [&](Step& r) {
    const unsigned char* st = from;
    from += slot_bytes;
    from = from == own + kQ8Codes * slot_bytes ? own : from;
#pragma unroll
    for (int h = 0; h < 2; h++) {
      r.ry[h] = *reinterpret_cast<const h8*>(st + grp * 32 + h * 16);
      r.my[h] = *reinterpret_cast<const h8*>(st + 128 + grp * 32 + h * 16);
    }
#pragma unroll
    for (int t = 0; t < NB; t++)
      r.q[t] = *reinterpret_cast<const u32x4*>(st + 256 + t * 1024 + row16 * 64 + ((grp ^ (row16 >> 2)) * 16));
  };
  // Loads complete in order, and they are issued in the order codes 0, codes 1, X 0, codes 2, X 1, codes 3, X 2, ...: what
  // has to have landed is told by how many of the loads behind it are outstanding.
  issue_codes();
  if (nk > 1) issue_codes();
  issue_a();
  if (nk > 2) issue_codes();
  if (nk > 1) issue_a();
  if (nk > 2) wait_loads<2 * NA + 2 * NC>();
  else if (nk > 1) wait_loads<2 * NA + NC>();
  else wait_loads<NA>();
  float c[NB + 1], m[NB + 1];
  const h1* cols = reinterpret_cast<const h1*>(own + kQ8Codes * slot_bytes);
#pragma unroll
  for (int t = 0; t < NB; t++) {
    c[t] = dequant_c(cols[t * 16 + row16]) * 16777216.0f;  // q8_dequant
    m[t] = (float)cols[64 + t * 16 + row16];
  }
  __builtin_amdgcn_s_setprio(2);  // the step waits for its producers: 1-5 % of a launch
  Step s0, s1;
  read(s0);
  asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
  if (nk > 3) issue_codes();
  unsigned char* bst = bsm;
  int b_step = maxw * 4096;  // to the other stage, and back
  // Step j between barriers j - 1 and j: behind barrier j - 1 step j - 2 has been read by all, and its slots may be written.
  auto step = [&](const Step& cur, Step& next, int behind, auto all) {
    constexpr bool ALL = decltype(all)::value;  // four steps or more behind this one
    if (ALL || behind >= 2) issue_a();
    if (ALL || behind >= 3) wait_loads<3 * NA + 2 * NC>();
    else if (behind == 2) wait_loads<3 * NA + NC>();
    else if (behind == 1) wait_loads<2 * NA>();
    if (ALL || behind >= 1) read(next);  // arrives while this step's codes are dequantised
#pragma unroll
    for (int t = 0; t < NB; t++)
#pragma unroll
      for (int h = 0; h < 2; h++) {
        const uint32_t w0 = cur.q[t][2 * h], w1 = cur.q[t][2 * h + 1];
        const h2 p0 = q8_dequant<0>(w0, c[t], m[t], cur.ry[h].s01, cur.my[h].s01);
        const h2 p1 = q8_dequant<1>(w0, c[t], m[t], cur.ry[h].s23, cur.my[h].s23);
        const h2 p2 = q8_dequant<0>(w1, c[t], m[t], cur.ry[h].s45, cur.my[h].s45);
        const h2 p3 = q8_dequant<1>(w1, c[t], m[t], cur.ry[h].s67, cur.my[h].s67);
        // 16 lanes write 16 columns' k-segment: free of bank conflicts
        *reinterpret_cast<h8*>(bst + ldw_at((p + kQ8Producers * t) * 16 + row16, 2 * grp + h)) = (h8){p0.x, p0.y, p1.x, p1.y, p2.x, p2.y, p3.x, p3.y};
      }
    bst += b_step;
    b_step = -b_step;
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // the step is written, the next one read
    if (ALL || behind >= 4) issue_codes();
    if (ALL || behind >= 4) wait_loads<2 * NA + 3 * NC>();  // X j has landed
    else if (behind == 3) wait_loads<2 * NA + 2 * NC>();
    else if (behind == 2) wait_loads<2 * NA + NC>();
    else if (behind == 1) wait_loads<NA>();
    else wait_loads<0>();
    step_barrier();  // barrier j
  };
  int behind = nk - 1;
  for (; behind >= 5; behind -= 2) {
    step(s0, s1, behind, std::true_type());
    step(s1, s0, behind - 1, std::true_type());
  }
  for (; behind >= 0; behind -= 2) {
    step(s0, s1, behind, std::false_type());
    if (behind >= 1) step(s1, s0, behind - 1, std::false_type());
  }
  step_barrier();
}

template <int BM, int NJ>
__device__ __forceinline__ void q8_mma(unsigned char* smem, int maxw, int brow0, int nk, int lane, int wm) {
  constexpr int MI = BM / 64, KG = MI * NJ >= 6 ? 2 : 4;
  const unsigned char* const bsm = smem + kQ8Stages * BM * 128;
  f16v acc[MI][NJ];
#pragma unroll
  for (int i = 0; i < MI; i++)
#pragma unroll
    for (int j = 0; j < NJ; j++)
#pragma unroll
      for (int v = 0; v < 16; v++) acc[i][j][v] = 0.f;
  for (int k = 0; k < nk; k++) {
    step_barrier();
    const unsigned char* as = smem + (k % kQ8Stages) * (BM * 128);
    const unsigned char* bs = bsm + (k & 1) * (maxw * 4096);
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
      }
#pragma unroll
      for (int kb = 0; kb < KG; kb++)
#pragma unroll
        for (int i = 0; i < MI; i++)
#pragma unroll
          for (int j = 0; j < NJ; j++)
            acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_f16(fa[kb][i], fb[kb][j], acc[i][j], 0, 0, 0);
    }
  }
  step_barrier();  // all fragments have been read
  const int pitch = sums_pitch(maxw);
#pragma unroll
  for (int i = 0; i < MI; i++) sums_to_lds(acc[i], reinterpret_cast<float*>(smem) + (wm * (BM / 2) + i * 32) * pitch + brow0, pitch, lane);
}

}  // namespace frhip
