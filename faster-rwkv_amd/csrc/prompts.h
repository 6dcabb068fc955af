// Prompts that lie one behind the other in the rows of a call: their table on the device, and what the host checks of them.
#pragma once

#include <cstdint>

#include "device_utils.h"
#include "frhip_internal.h"

namespace frhip {

constexpr int kMostRows = 1 << 30;     // of a call of single tokens: a loop over them counts in steps of up to 2^18
constexpr int kMostTime = 1 << 28;     // row numbers of prompts: sums of a few of them stay in 32 bits, and so do a launch's threads
constexpr int kMostChannels = 1 << 24;

constexpr int kSeqTable = 128;  // prompts of a launch; more go out in several
struct SeqTable {
  int start[kSeqTable + 1];  // first row
  int chunk[kSeqTable + 1];  // first chunk (every prompt has one at least)
};

// The prompt that chunk `j` belongs to: the last i with first(i) <= j, for all lanes of a wave at once (all of them are here).  `first` does
// not descend and first(0) is 0.  One load of a lane each: a search by halves waits for one after another.
template <class F>
__device__ __forceinline__ int find_seq(int nseq, int j, F first) {
  static_assert(kSeqTable <= 128, "two prompts a lane");
  if (nseq == 1) return 0;
  const int l = threadIdx.x & 63;
  int n = __builtin_popcountll(__ballot(l < nseq && first(min(l, nseq - 1)) <= j));
  if (nseq > 64) n += __builtin_popcountll(__ballot(l + 64 < nseq && first(min(l + 64, nseq - 1)) <= j));
  return __builtin_amdgcn_readfirstlane(n - 1);
}

inline int check_seqs(int nseq, const int32_t* seq_start, int most, const char* what) {
  if (nseq < 0) return set_error(FRHIP_ESHAPE, what);
  if (nseq > 0) {
    if (!seq_start) return set_error(FRHIP_EINVAL, what);
    if (seq_start[0] < 0) return set_error(FRHIP_ESHAPE, what);
    for (int i = 0; i < nseq; i++)
      if (seq_start[i + 1] < seq_start[i]) return set_error(FRHIP_ESHAPE, what);
    if (seq_start[nseq] > most) return set_error(FRHIP_ESHAPE, what);
  }
  return 0;
}

}  // namespace frhip
