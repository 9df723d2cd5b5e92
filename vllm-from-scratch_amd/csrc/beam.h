// Host/device interface of the beam-search kernels (beam.hip, beam_states.hip).
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "../../include/mvsd.h"

namespace mvsd {

constexpr int kMaxBeams = 64;        // a group's beams fit the lanes of a wave
constexpr int kMaxCandidates = 256;  // of a group
constexpr int kMaxBeamStates = 24;   // state tensors of one launch (kernel arguments)

#ifdef __HIPCC__
// len^alpha, len >= 1, inside 2^-1000 .. 2^1000: 2^y, y = alpha log2(len), to about (1 + |y| / 4) 2^-50; the
// logarithm of the mantissa m in [1/sqrt 2, sqrt 2) from the series of atanh((m - 1) / (m + 1)), the power
// of the fraction from that of exp.  (The library's pow, exact to the last bit, took 3000 cycles of a
// group's 20000.)
__device__ inline double len_power(int len, double alpha) {
  if (alpha == 1.0) return (double)len;
  int e = 32 - __clz(len);  // len = m 2^e
  double m = ldexp((double)len, -e);
  if (m < 0.70710678118654752) {
    m *= 2.0;
    --e;
  }
  const double s = (m - 1.0) / (m + 1.0), s2 = s * s;
  double ln = 0.0;
#pragma unroll
  for (int k = 19; k >= 1; k -= 2) ln = fma(ln, s2, 1.0 / k);
  ln *= 2.0 * s;
  const double y = alpha * ((double)e + ln * 1.4426950408889634074);
  const double in = fmin(fmax(y, -1000.0), 1000.0), n = rint(in);
  const double f = (in - n) * 0.69314718055994530942;
  double x = 1.0;
#pragma unroll
  for (int k = 14; k >= 1; --k) x = fma(x, f * (1.0 / k), 1.0);
  return ldexp(x, (int)n);
}

// A candidate's score: fl32(total), and fp32's lowest value below it, since -inf says that there is no beam
// (two tokens masked by the type's lowest value in one sequence).
__device__ inline float candidate_score(double total) {
  return fmaxf((float)total, -3.402823466e38f);
}

// A hypothesis' score: fl32(total / power), and fp32's largest value beyond it, since -inf says that there
// is no hypothesis (a negative alpha: 20 tokens to the 30th).
__device__ inline float hypothesis_score(float total, double power) {
  return fminf(fmaxf((float)((double)total / power), -3.402823466e38f), 3.402823466e38f);
}
#endif

struct BeamScanParams {
  const void* logits;
  int64_t stride;       // elements
  int64_t num_rows;     // rows of `logits` that a row index is clamped to
  const int32_t* rows;  // [G * W] row of each beam, or null (row g * W + w)
  const float* scores;  // [G, W]
  const int32_t* lengths;  // step: [G], else null
  const uint8_t* done;     // step: [G], else null
  int G, W, V, C;
  int max_length;  // step: T
  int nchunks, tops_per_chunk;
  struct alignas(16) Stat {
    double sum;  // of exp(x - max)
    float max;
  };
  Stat* stats;    // [G * W, nchunks] chunk maximum and sum
  float* tops;    // [G * W, nchunks, tops_per_chunk] the largest entry of 16 or 2 lanes each
};

struct BeamSelectOut {
  int32_t* token_ids;  // [G, C]
  int32_t* parents;
  float* scores;
};

int64_t beam_workspace_bytes(int64_t G, int64_t W, int64_t V, int64_t C);
hipError_t launch_beam_select(BeamScanParams p, const BeamSelectOut& out, int dtype,
                              void* workspace, hipStream_t stream);
hipError_t launch_beam_step(BeamScanParams p, const mvsd_beam_step_args& a, void* workspace,
                            hipStream_t stream);

struct BeamStatesParams {
  mvsd_beam_state state[kMaxBeamStates];
  const int32_t* parents;  // [G, W]
  const int32_t* starts;   // [G] or null
  const int32_t* lengths;  // [G] or null
  const int32_t* slots;    // [G, W] or null
  int64_t first_group;     // group 0 of this launch
  int G, W, n;
};

hipError_t launch_beam_reorder(const BeamStatesParams& p, bool in_place, hipStream_t stream);
int64_t beam_finish_workspace_bytes(int64_t G, int64_t W, int64_t T, int64_t n);
hipError_t launch_beam_finish(const mvsd_beam_finish_args& a, hipStream_t stream);

}  // namespace mvsd
