// Sizes and layout of the products of a few rows (gemm_few.hip has the form and its reasons), shared with linear.hip.
#pragma once

#include "gemm_device.h"

#pragma clang fp contract(off)

namespace frhip {

constexpr int kFewScaleBytes = 512;  // uint8: rx, then mx of up to 128 columns, behind a wave's ring
// The waves decide the order of the sums: the same for both weight types.  The ring is as deep as 160 KB of LDS allow, up to
// four steps.
constexpr int few_waves(int mt, int nt) { return mt + nt <= 5 ? 8 : 4; }
constexpr int few_stage_bytes(int mt, int nt, bool u8) { return mt * 2048 + (u8 ? nt * 1024 + 256 : nt * 2048); }
constexpr int few_stages(int mt, int nt, bool u8) {
  const int s = (160 * 1024 / few_waves(mt, nt) - (u8 ? kFewScaleBytes : 0)) / few_stage_bytes(mt, nt, u8);
  return s > 4 ? 4 : s;
}
constexpr int few_wave_bytes(int mt, int nt, bool u8) { return few_stages(mt, nt, u8) * few_stage_bytes(mt, nt, u8) + (u8 ? kFewScaleBytes : 0); }

// A tile of 16 rows x 64 binary16: rows of 128 bytes, k-segment q (8 halves) of row r in slot q ^ (r % 8) ^ (r / 8)
// (the layout of the tiled kernels: fragment reads of 16 rows are free of bank conflicts)
__device__ __forceinline__ int few_at(int r, int q) { return r * 128 + ((q ^ (r & 7) ^ (r >> 3)) * 16); }

// The tiles (16-row by 16-column blocks of a workgroup) that are built: within 2 % of the best of all 30 on 1360 measured products.
#define FR_FEW_TILES(X) \
  X(1, 1) X(1, 2) X(1, 3) X(1, 4) X(2, 1) X(2, 2) X(2, 3) X(2, 4) X(3, 1) X(3, 2) X(3, 3) X(3, 4) X(3, 5) \
  X(4, 2) X(4, 3) X(4, 4) X(5, 2) X(5, 3) X(5, 4) X(5, 5) X(6, 4)

}  // namespace frhip
