// Beam search: the states of the beams follow their parents, and the sequences of the answers.
#include "beam.h"
#include "mvsd_device.h"

namespace mvsd {

// ------------------------------------------------------------------ reorder ----------
// Row of beam (g, w): state row slots[g, w], or g * W + w.  A row is `outer` pieces of `length`
// entries of `inner` bytes; entries [start_g, length_g) of every piece are copied from the row of the
// parent.  A parent outside [0, W) is the beam itself.
//
// In place, a thread owns a few bytes of all W rows of a group: it loads what each row needs into
// registers, then stores, so no row is overwritten before it has been read, with no second buffer and
// no order among threads.  Rows that keep their beam are neither read nor written.

typedef u32x4 u32x4_align1 __attribute__((aligned(1)));
typedef u32x2 u32x2_align1 __attribute__((aligned(1)));

template <typename T>
struct AnyAlign;
template <>
struct AnyAlign<u32x4> {
  using type = u32x4_align1;
};
template <>
struct AnyAlign<u32x2> {
  using type = u32x2_align1;
};
template <>
struct AnyAlign<uint8_t> {
  using type = uint8_t;
};

template <int ROWS, typename T, bool IN_PLACE>
__device__ inline void move_rows(const char* src, char* dst, int64_t src_stride,
                                 int64_t dst_stride, int64_t off, uint64_t moves, int from, int to,
                                 int W) {
  using U = typename AnyAlign<T>::type;
  for (int b = 0; b < W; b += ROWS) {  // one round in place (ROWS >= W)
    T v[ROWS];
#pragma unroll
    for (int w = 0; w < ROWS; ++w)
      if ((moves >> (b + w)) & 1)
        v[w] = *reinterpret_cast<const U*>(
            src + (int64_t)__builtin_amdgcn_readlane(from, b + w) * src_stride + off);
#pragma unroll
    for (int w = 0; w < ROWS; ++w)
      if ((moves >> (b + w)) & 1)
        *reinterpret_cast<U*>(dst + (int64_t)__builtin_amdgcn_readlane(to, b + w) * dst_stride +
                              off) = v[w];
  }
}

template <int ROWS, typename T, bool IN_PLACE>
__global__ __launch_bounds__(kThreads) void beam_reorder_kernel(BeamStatesParams p) {
  const int64_t g = p.first_group + blockIdx.y / p.n;
  const int k = blockIdx.y % p.n;
  const mvsd_beam_state s = p.state[k];
  const int lane = lane_id(), W = p.W;
  // lane w: where the row of beam w comes from and goes to
  int from = -1, to = -1;
  bool move = false;
  if (lane < W) {
    const int64_t first = g * W;
    int parent = p.parents[first + lane];
    if (parent < 0 || parent >= W) parent = lane;
    from = p.slots ? p.slots[first + parent] : (int)first + parent;
    to = p.slots ? p.slots[first + lane] : (int)first + lane;
    move = from >= 0 && from < s.num_rows && to >= 0 && to < s.num_rows &&
           !(IN_PLACE && from == to);
  }
  const uint64_t moves = __ballot(move);
  if (moves == 0) return;
  const int64_t start = p.starts ? min(max((int64_t)p.starts[g], (int64_t)0), s.length) : 0;
  const int64_t end = p.lengths ? min((int64_t)p.lengths[g], s.length) : s.length;
  const int64_t seg = (end - start) * s.inner;
  if (seg <= 0) return;
  // a piece: whole vectors, then single bytes
  const uint32_t whole = (uint32_t)(seg / (int64_t)sizeof(T));
  const uint32_t units = whole + (uint32_t)(seg - (int64_t)whole * (int64_t)sizeof(T));
  const int64_t total = (int64_t)s.outer * units;
  const int64_t piece = s.length * s.inner;
  for (int64_t u = (int64_t)blockIdx.x * kThreads + threadIdx.x; u < total;
       u += (int64_t)gridDim.x * kThreads) {
    const int64_t o = u / units;
    const uint32_t i = (uint32_t)(u - o * units);
    const int64_t at = o * piece + start * s.inner;
    if (i < whole)
      move_rows<ROWS, T, IN_PLACE>((const char*)s.src, (char*)s.dst, s.src_stride, s.dst_stride,
                                   at + (int64_t)i * (int64_t)sizeof(T), moves, from, to, W);
    else
      move_rows<ROWS, uint8_t, IN_PLACE>((const char*)s.src, (char*)s.dst, s.src_stride,
                                         s.dst_stride,
                                         at + (int64_t)whole * (int64_t)sizeof(T) + (i - whole),
                                         moves, from, to, W);
  }
}

template <int ROWS, typename T, bool IN_PLACE>
static void launch_rows(const BeamStatesParams& p, hipStream_t stream) {
  int64_t most = 1;
  for (int k = 0; k < p.n; ++k) {
    const mvsd_beam_state& s = p.state[k];
    const int64_t units = s.outer * (s.length * s.inner / (int64_t)sizeof(T) + 1);
    most = units > most ? units : most;
  }
  int64_t x = (most + kThreads - 1) / kThreads;
  const int64_t y = (int64_t)p.G * p.n;
  const int64_t cap = y < 65536 ? 65536 / y + 1 : 1;
  if (x > cap) x = cap;
  hipLaunchKernelGGL((beam_reorder_kernel<ROWS, T, IN_PLACE>), dim3((unsigned)x, (unsigned)y),
                     dim3(kThreads), 0, stream, p);
}

hipError_t launch_beam_reorder(const BeamStatesParams& p, bool in_place, hipStream_t stream) {
  if (!in_place) launch_rows<8, u32x4, false>(p, stream);
  else if (p.W <= 8) launch_rows<8, u32x4, true>(p, stream);
  else if (p.W <= 16) launch_rows<16, u32x4, true>(p, stream);
  else if (p.W <= 32) launch_rows<32, u32x4, true>(p, stream);
  else launch_rows<64, u32x2, true>(p, stream);
  return hipGetLastError();
}

// ------------------------------------------------------------------ finish -----------
// Of each group the n best of its finished hypotheses and, unless it is done, its running beams (a
// running beam is its last token appended to its parent), the finished ones first where they are
// equal; then each one's tokens, from the last step back: the token and the parent recorded in the
// beam's place.  A parent outside [0, W) is the beam itself.

__global__ __launch_bounds__(kThreads) void beam_finish_hyps_kernel(mvsd_beam_finish_args a) {
  __shared__ float s_key[2 * kMaxBeams];
  __shared__ int s_beam[kMaxBeams], s_token[kMaxBeams], s_len[kMaxBeams];
  const int g = blockIdx.x, tid = threadIdx.x, W = (int)a.beam_width, n = (int)a.num_return;
  const int64_t first = (int64_t)g * W, T = a.max_length;
  const int len = (int)min(max((int64_t)a.lengths[g], (int64_t)0), T);
  if (tid < 2 * W) {
    float v = -INFINITY;
    if (tid < W) v = a.finished_scores[first + tid];
    else if (a.done[g] == 0 && len > 0 && fabsf(a.scores[first + tid - W]) < INFINITY)
      v = (float)((double)a.scores[first + tid - W] / pow((double)len, a.length_penalty));
    s_key[tid] = v > -INFINITY ? v : -INFINITY;
  }
  __syncthreads();
  if (tid < 2 * W) {
    const float v = s_key[tid];
    int rank = 0;
    for (int j = 0; j < 2 * W; ++j) rank += s_key[j] > v || (s_key[j] == v && j < tid);
    if (rank < n) {
      int beam = -1, token = -1, l = 0;
      if (v > -INFINITY) {
        if (tid < W) {
          beam = a.finished_beams[first + tid];
          token = a.finished_token_ids[first + tid];
          l = (int)min(max((int64_t)a.finished_lengths[first + tid], (int64_t)0), T);
        } else {
          const int64_t at = ((int64_t)g * T + len - 1) * W + tid - W;
          beam = a.parent_history[at];
          token = a.token_history[at];
          l = len;
        }
      }
      a.out_scores[(int64_t)g * n + rank] = v;
      a.out_lengths[(int64_t)g * n + rank] = l;
      s_beam[rank] = beam >= 0 && beam < W ? beam : 0;
      s_token[rank] = token;
      s_len[rank] = l;
    }
  }
  __syncthreads();
  for (int h = 0; h < n; ++h) {
    int32_t* out = a.out_token_ids + ((int64_t)g * n + h) * T;
    for (int64_t t = s_len[h] + tid; t < T; t += kThreads) out[t] = -1;
  }
  if (tid < n) {
    int32_t* out = a.out_token_ids + ((int64_t)g * n + tid) * T;
    const int l = s_len[tid];
    int slot = s_beam[tid];
    if (l > 0) out[l - 1] = s_token[tid];
    for (int t = l - 2; t >= 0; --t) {
      const int64_t at = ((int64_t)g * T + t) * W + slot;
      out[t] = a.token_history[at];
      const int parent = a.parent_history[at];
      if (parent >= 0 && parent < W) slot = parent;
    }
  }
}

hipError_t launch_beam_finish(const mvsd_beam_finish_args& a, hipStream_t stream) {
  hipLaunchKernelGGL(beam_finish_hyps_kernel, dim3((unsigned)a.num_groups), dim3(kThreads), 0,
                     stream, a);
  return hipGetLastError();
}

}  // namespace mvsd
