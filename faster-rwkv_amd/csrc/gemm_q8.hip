// Products of uint8 weights on the MFMA units, the codes dequantised on their way into LDS by waves that do nothing else.
//
// Workgroup tile BM x (32 w): four MFMA waves (2 x 2, as in gemm_vw_kernel: the same MFMAs in the same k order, so the same
// bits as the binary16 kernels give on the expanded matrix) and eight producer waves, two per SIMD.  A producer
// brings its share of X and of the codes, global -> LDS directly, three K-steps of 64 ahead, turns its codes into binary16
// with the formula of the standalone dequantisation and leaves them where the MFMA waves read their fragments, one step
// ahead of them.  A wave dequantises the codes that it loaded itself, so only the finished step needs a barrier: one a step,
// for all twelve waves.  The sums go through LDS to the epilogue, which all of them share.
//
// What bounds it: a wave issues an instruction every 6 to 10 cycles here, whatever the other waves of its SIMD do, so what
// counts is the producer's instructions from barrier to barrier (110 for one block of 16 columns, 182 for two: 64 a block for
// its codes, 4 a code).  512 x 2560 x (4 x 2560), us: four producers 55, eight 61 (1100 spilled registers in an epilogue of the
// four MFMA waves) -> 50 with the sums through LDS -> 46 with the loop free of branches and address arithmetic; the
// expansion of the codes and the binary16 product 59.  Products of a layer, expansion and binary16 kernels -> this one:
//   13 rows (codes dequantised in registers, 64 x 128 tiles): 2560 x (4 x 2560) 25.7 -> 18.6, 8192 x 2048 17.5 -> 14.9
//   128 rows: 4096 x (4 x 4096) 73.5 -> 38.9, 14336 x 4096 71.6 -> 37.3;  300 rows: 2560 x (2560 + 8960) 62.8 -> 41.9
//   512 rows: 2560 x 2560 28.1 -> 22.6, 2560 x (2560 + 8960) 56.7 -> 49.1, 8960 x 2560 63.2 -> 45.4
#include <climits>
#include <cmath>
#include <cstring>

#include "gemm_q8_device.h"

#pragma clang fp contract(off)

namespace frhip {

template <int BM>
__global__ __launch_bounds__(64 * (4 + kQ8Producers)) void gemm_q8_kernel(GemmArgs a) {
  extern __shared__ __attribute__((aligned(16))) unsigned char q8_smem[];
  int bx, by;
  xcd_tile(bx, by);
  int sidx = 0;
#pragma unroll
  for (int i = 1; i < kGemmMaxSeg; i++) sidx += (i < a.nseg && bx >= a.tile_start[i]) ? 1 : 0;
  GemmSeg sg = a.seg[sidx];
  const int ti = bx - a.tile_start[sidx], base = a.vw_base[sidx], wide = a.vw_wide[sidx];
  const int width = base + (ti < wide ? 1 : 0);  // 32-column blocks of this tile
  const int n0 = (ti * base + (ti < wide ? ti : wide)) * 32, m0 = by * BM;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  // slice z of ksplit takes K-steps [z base + min(z, rem), ...): the first rem slices one step more
  const int ksplit = a.ksplit > 1 ? a.ksplit : 1, kz = blockIdx.z, ksteps = a.K / kLdwBK, kper = ksteps / ksplit, krem = ksteps % ksplit;
  const int nk = kper + (kz < krem ? 1 : 0), kbase = (kz * kper + (kz < krem ? kz : krem)) * kLdwBK;
  if (wave >= 4) {
    const int p = wave - 4;
    static_assert(2 * q8_max_blocks(BM) <= 2 * kQ8Producers, "a producer has at most two blocks of 16 columns");
    switch (p < 2 * width ? (2 * width - p + kQ8Producers - 1) / kQ8Producers : 0) {
      case 0: q8_producer<BM, 0>(sg, q8_smem, a.vw_maxw, p, m0, n0, a.M, a.K, a.K, kbase, nk, lane); break;
      case 1: q8_producer<BM, 1>(sg, q8_smem, a.vw_maxw, p, m0, n0, a.M, a.K, a.K, kbase, nk, lane); break;
      default: q8_producer<BM, 2>(sg, q8_smem, a.vw_maxw, p, m0, n0, a.M, a.K, a.K, kbase, nk, lane); break;
    }
  } else {
    const int wm = wave >> 1, nj0 = (width + 1) >> 1, nj = (wave & 1) ? width - nj0 : nj0, brow0 = (wave & 1) ? nj0 * 32 : 0;
    switch (nj) {  // every wave passes the same barriers, whatever its width
      case 1: q8_mma<BM, 1>(q8_smem, a.vw_maxw, brow0, nk, lane, wm); break;
      case 2: q8_mma<BM, 2>(q8_smem, a.vw_maxw, brow0, nk, lane, wm); break;
      case 3: q8_mma<BM, 3>(q8_smem, a.vw_maxw, brow0, nk, lane, wm); break;
      default: q8_mma<BM, q8_max_blocks(BM) / 2>(q8_smem, a.vw_maxw, brow0, nk, lane, wm); break;
    }
  }
  __syncthreads();
  if (a.ksplit > 1) {  // this slice's sums go out as fp32; the epilogue proper follows in gemm_splitk_reduce_kernel
    sg.out = a.partial + (size_t)kz * a.partial_stride + a.part_off[sidx];
    sg.epi = G_STORE_F32;
  }
  finish_tile<BM, 64 * (4 + kQ8Producers)>(a, sg, reinterpret_cast<const float*>(q8_smem), sums_pitch(a.vw_maxw), width, m0, n0, a.M, sg.N);
}

// What a launch of such tiles is expected to take, us: fitted to 1793 measured ones (13 to 1536 rows, widths 1024 to 4096, the
// products of a layer, weights from memory; 7 % rms, the tile chosen by it 0.6 % slower than the best of 11).  Per round a fixed
// part and its K-steps, and no faster than the codes arrive; slices of K and their reduction launch.
static double q8_us(const GemmArgs& a, int bm, int rounds, int w) {
  const int S = a.ksplit > 1 ? a.ksplit : 1, steps = (a.K / kLdwBK + S - 1) / S;
  double cols = 0;
  for (int s = 0; s < a.nseg; s++) cols += a.seg[s].N;
  const double x = rounds * (bm == 128 ? 3.17 + 0.102 * w + steps * (0.194 + 0.120 * w) : 2.41 + 0.261 * w + steps * (0.181 + 0.085 * w));
  const double y = cols * a.K / 3.44e6;
  return 4.2 + sqrt(sqrt(x * x * x * x + y * y * y * y)) + (S > 1 ? 1.6 + S * a.M * cols * 8 / 4.2e6 : 0);
}

TilePlan plan_q8(const GemmArgs& args, int cus) {
  TilePlan best;
  const int S = args.ksplit > 1 ? args.ksplit : 1;
  if ((size_t)args.K * 2 * 128 > 0xffffffffull) return best;  // 32-bit byte offsets within a tile
  for (int s = 0; s < args.nseg; s++)
    if (args.seg[s].N % 16 != 0) return best;
  for (int bm : {128, 64}) {
    const int strips = (args.M + bm - 1) / bm;
    for (int w = q8_max_blocks(bm); w >= 2; w--) {
      // as few tiles as this width allows, then as many as their rounds hold
      long need = 0;
      for (int s = 0; s < args.nseg; s++) need += ((args.seg[s].N + 31) / 32 + w - 1) / w;
      const int rounds = (int)((need * strips * S + cus - 1) / cus);
      TilePlan p;
      p.a = args;
      auto dealt = [&](long tiles) {  // the MFMA waves take two blocks or more of a tile
        if (!deal_tiles(p.a, (int)tiles) || p.a.vw_maxw > w) return false;
        for (int s = 0; s < args.nseg; s++)
          if (p.a.vw_base[s] < 2) return false;
        return true;
      };
      if (!dealt((long)rounds * cus / ((long)strips * S)) && !dealt(need)) continue;
      p.us = q8_us(args, bm, rounds, p.a.vw_maxw);
      p.rows = bm;
      p.rounds = rounds;
      p.grid = dim3(p.a.tile_start[p.a.nseg], strips, S);
      if (!best.rows || p.us < best.us) best = p;
    }
  }
  return best;
}

// codes are loaded 16 bytes at a time, rows' and columns' scales 4
bool q8_takes(const GemmArgs& a) {
  uintptr_t v16 = 0, v4 = 0;
  for (int s = 0; s < a.nseg; s++) {
    v16 |= reinterpret_cast<uintptr_t>(a.seg[s].A) | reinterpret_cast<uintptr_t>(a.seg[s].B);
    for (const h1* p : {a.seg[s].mx, a.seg[s].rx, a.seg[s].my, a.seg[s].ry}) v4 |= reinterpret_cast<uintptr_t>(p);
  }
  return (v16 & 15) == 0 && (v4 & 3) == 0;
}

int launch_gemm_q8(const TilePlan& p, hipStream_t st, const char* what) {
  static const bool raised = [] {
    for (const void* f : {reinterpret_cast<const void*>(&gemm_q8_kernel<128>), reinterpret_cast<const void*>(&gemm_q8_kernel<64>)})
      (void)hipFuncSetAttribute(f, hipFuncAttributeMaxDynamicSharedMemorySize, 160 * 1024);
    return true;
  }();
  (void)raised;
  const size_t lds = q8_lds_bytes(p.rows, p.a.vw_maxw);
  if (p.rows == 128)
    hipLaunchKernelGGL(gemm_q8_kernel<128>, p.grid, dim3(64 * (4 + kQ8Producers)), lds, st, p.a);
  else
    hipLaunchKernelGGL(gemm_q8_kernel<64>, p.grid, dim3(64 * (4 + kQ8Producers)), lds, st, p.a);
  return check_launch(what);
}

}  // namespace frhip
