// The gated delta rule: what its two forms share (delta.hip: token by token; delta_chunk.hip: chunk by chunk).
#pragma once

#include "activations.h"
#include "frhip_internal.h"
#include "groups.h"
#include "lanes.h"
#include "prompts.h"

#pragma clang fp contract(off)

namespace frhip {

constexpr int kMostDim = 256;         // of a key, of a value
constexpr int kMostHeads = 65535;     // a launch's second dimension
constexpr int kMostPitch = 1 << 23;   // of rows: the bytes of a chunk of them, 64, stay in 32 bits
constexpr int kDeltaChunkLeast = 21;  // rows of a prompt, at least, that goes chunk by chunk

template <class T>
struct DeltaArgs {
  const T *q, *k, *v, *dt, *beta;
  T* y;
  const float *A, *dt_bias, *state;
  float* state_out;
  int ldq, ldk, ldv, lddt, ldbeta, ldy;
  int heads, share, dk, dv;  // share: heads of values to a head of keys
  float scale, eps;          // eps < 0: q and k as they are
  int softplus, sigmoid;
  int nseq, rows;  // prompts of the launch; of single tokens: rows
};

// The prompts of a launch, or parts of them
struct DeltaTable {
  int start[kSeqTable], end[kSeqTable];  // rows
  int seq[kSeqTable];                    // which state
  int chunk[kSeqTable + 1];              // first chunk, of the form by chunks
  int ahead;                             // the first one goes on from what an earlier launch left in state_out
};

// exp(g) for the logarithm of a decay, which is a number: below -120 it is zero in fp32, above 88 it stays there
__device__ __forceinline__ float decay_f(float g) { return exp_neg_fine(__builtin_fmaxf(__builtin_fminf(-g, 120.f), -88.f)); }

// The logarithm of a row's decay.  A rate of minus infinity stays a number (times a step of width zero it keeps the state).
template <class T>
__device__ __forceinline__ float log_decay(const DeltaArgs<T>& a, float dt, float rate, float bias) {
  const float v = dt + bias;
  return rate * (a.softplus ? softplus_f<true>(v) : v);
}
__device__ __forceinline__ float finite_rate(float r) { return r < -__FLT_MAX__ ? -__FLT_MAX__ : r; }

// The form by chunks, host side: its scratch for T rows, and prompts of a call by it (indices into start; in any order)
size_t delta_chunk_bytes(const frhip_delta& p, int elem, int T);
// Whether prompts, some of them of kDeltaChunkLeast rows, have no more chunks than one pair of launches for T rows takes
bool delta_chunks_fit(const frhip_delta& p, int elem, const int32_t* start, int nseq, int T);
template <class T>
int delta_chunk_run(const DeltaArgs<T>& a, const int* seqs, int nseq, const int32_t* start, int rows, void* workspace, hipStream_t st);

}  // namespace frhip
