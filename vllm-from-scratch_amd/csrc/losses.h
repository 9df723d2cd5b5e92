// Host/device interface of the training losses on rows of logits (losses.hip).
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "../../include/mvsd.h"

namespace mvsd {

constexpr int kMaxTeacher = 512;            // teacher entries of a row: two a thread of a finishing workgroup
constexpr int kRecord = 8;                  // floats of a row that its gradient needs
constexpr int kNormParts = 1024;            // partial sums of the rows' weights

// A row's record for the gradient of unit upstream: with e_j = 2^((x_j - M) c1) of the tokens that are
// none of the row's given ones ("the rest", M their maximum), g the upstream times c and gH the entropy's
// times cH, the gradient is  -e_j k (g + gH (h + ln 2 * log2 e_j)), and  g o1 + gH o2  at the given token.
struct LossRecord {
  float M, k, h, o1, o2, c, cH;
  int pair;  // preference: the upstream's index
};
static_assert(sizeof(LossRecord) == kRecord * sizeof(float));

// What a row's entries give without the rest of the row: their maximum, and sums of e_k = exp((x_k - top) / T)
// and of what the divergence needs.
struct EntrySums {
  float top, z, s1, s2;
};

struct LossTeacher {
  EntrySums sums;
  float value;   // the mass of the rest, or without a tail the log of the entries' sum
  float weight;  // 0: the row is left out
  float unused[2];
};

struct LossParams {
  mvsd_loss_args a;
  float c1;     // log2(e) / temperature
  float inv_t;  // 1 / temperature
  int V;
  int K;        // given tokens of a row
  int chunk, nch;   // columns of a workgroup, workgroups of a row
  int active;       // threads that hold a row
  void* aside;      // a span of them for each workgroup
  bool entropy;
  bool whole;       // the statistics' kernel finishes token rows, of one chunk each
  float4* parts;      // [N, nch] maximum, sum, sum of e log2 e
  float* norm;        // [kNormParts] partial sums of weights (mean)
  int norm_parts;
  int* counters;      // [2], see losses.hip
  float* row_loss;    // [N] (preference: [pairs]), weighted
  float* row_lp;      // preference: [N]
  LossTeacher* teach;   // distillation: [N]
  float* entry_logits;  // [N, K]
  LossRecord* records;    // [N] or null
  float* over;            // distillation: [N, K] gradients of the given tokens for unit upstream
  int32_t* over_ids;      // [N, K] the entries that count, -1: none
};

bool loss_one_pass(const mvsd_loss_args& a);
int64_t loss_workspace_bytes(const mvsd_loss_args& a);
int64_t loss_saved_bytes(const mvsd_loss_args& a);
hipError_t launch_loss(const mvsd_loss_args& a, hipStream_t stream);
hipError_t launch_loss_gradient(const mvsd_loss_args& a, const float* up, int64_t up_stride,
                                const float* up_entropy, int64_t up_entropy_stride, hipStream_t stream);

}  // namespace mvsd
