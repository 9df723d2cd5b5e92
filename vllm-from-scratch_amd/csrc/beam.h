// Host/device interface of the beam-search kernels (beam.hip, beam_states.hip).
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "../../include/mvsd.h"

namespace mvsd {

constexpr int kMaxBeams = 64;        // a group's beams fit the lanes of a wave
constexpr int kMaxCandidates = 256;  // of a group
constexpr int kMaxBeamStates = 24;   // state tensors of one launch (kernel arguments)

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
  int nchunks;
  float2* stats;  // [G * W, nchunks] chunk maximum and sum of exp(x - maximum)
  float* tops;    // [G * W, nchunks, 16] the largest entry of 16 lanes each
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
