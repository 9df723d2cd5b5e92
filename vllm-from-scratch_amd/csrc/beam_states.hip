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
//
// With b_t the beam at step t, b_(t-1) = parent_t(b_t): a chain of T dependent reads.  The steps'
// maps are composed instead.  A workgroup holds the parents of a chunk of steps in LDS, a byte each;
//   - the chunk's sub-chunks of kSub steps are walked from every beam at once, which gives their maps;
//   - the hypotheses go through the sub-chunks' maps, which gives their beam at the top of each;
//   - every sub-chunk is walked again from there, all at once, and leaves the beam of each step, by
//     which the tokens are gathered and the sequences written, coalesced.
// Histories of one chunk take one launch.  Longer ones take two: the first leaves every chunk's map
// and, for a hypothesis that ends in the chunk, its beam below it; the second starts from those.

constexpr int kTThreads = 512;
constexpr int kSub = 32;
constexpr int kTraceLds = 56 * 1024;
constexpr int kMapPiece = 4096;  // bytes of chunk maps held at a time
enum { kTraceWhole, kTraceMaps, kTraceEmit };

// Steps per chunk: the whole history where it fits LDS and is short, else 1024 steps or fewer.
static int trace_chunk(int64_t W, int64_t n, int64_t T) {
  if (T <= 4096 && T * (W + n) <= kTraceLds) return (int)T;
  return W + n <= 48 ? 1024 : 384;
}

// Dynamic LDS: parents [S, W], beams [n, S], sub-chunk maps [nsub, W], tops [n, nsub] in bytes.
static int trace_lds(int64_t W, int64_t n, int64_t S) {
  const int64_t nsub = (S + kSub - 1) / kSub;
  return (int)(((S + 3) / 4 * 4) * W + n * S + nsub * (W + n));
}

int64_t beam_finish_workspace_bytes(int64_t G, int64_t W, int64_t T, int64_t n) {
  const int64_t S = trace_chunk(W, n, T), chunks = (T + S - 1) / S;
  return chunks > 1 ? G * (chunks * W + n) : 0;
}

template <int MODE>
__global__ __launch_bounds__(kTThreads) void beam_trace_kernel(mvsd_beam_finish_args a, int S,
                                                                int chunks, uint8_t* maps,
                                                                uint8_t* exits) {
  __shared__ float s_key[2 * kMaxBeams];
  __shared__ int s_token[kMaxBeams], s_len[kMaxBeams];
  __shared__ uint8_t s_beam[kMaxBeams];
  __shared__ int s_longest;
  __shared__ uint8_t s_maps[MODE == kTraceEmit ? kMapPiece : 1];
  extern __shared__ __align__(16) uint8_t lds[];
  const int tid = threadIdx.x, W = (int)a.beam_width, n = (int)a.num_return;
  const int64_t T = a.max_length;
  const int64_t g = blockIdx.x / chunks;
  const int chunk = (int)(blockIdx.x - g * chunks);
  const int64_t first = g * W;
  const int nsub = (S + kSub - 1) / kSub;
  uint8_t* parent = lds;
  uint8_t* sub_map = parent + (int64_t)((S + 3) / 4 * 4) * W;
  uint8_t* tops = sub_map + nsub * W;
  uint8_t* beams = tops + n * nsub;
  // ---- the n best hypotheses ----
  const int len = (int)min(max((int64_t)a.lengths[g], (int64_t)0), T);
  if (tid == 0) s_longest = 0;
  float v = -INFINITY;
  if (tid < W) v = a.finished_scores[first + tid];
  else if (tid < 2 * W && a.done[g] == 0 && len > 0 &&
           fabsf(a.scores[first + tid - W]) < INFINITY)
    v = (float)((double)a.scores[first + tid - W] / pow((double)len, a.length_penalty));
  if (!(v > -INFINITY)) v = -INFINITY;
  if (tid < 2 * W) s_key[tid] = v;
  __syncthreads();
  if (tid < 2 * W) {
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
          const int64_t at = (g * T + len - 1) * W + tid - W;
          beam = a.parent_history[at];
          token = a.token_history[at];
          l = len;
        }
      }
      if (MODE != kTraceMaps && chunk == 0) {
        a.out_scores[g * n + rank] = v;
        a.out_lengths[g * n + rank] = l;
      }
      s_beam[rank] = (uint8_t)(beam >= 0 && beam < W ? beam : 0);
      s_token[rank] = token;
      s_len[rank] = l;
      atomicMax(&s_longest, l);
    }
  }
  __syncthreads();
  // ---- the parents of the steps [c0, c0 + steps) that some hypothesis goes through ----
  const int64_t c0 = (int64_t)chunk * S;
  const int steps = (int)min(max((int64_t)s_longest - 1 - c0, (int64_t)0), (int64_t)S);
  if (MODE == kTraceMaps && steps == 0) return;
  {
    const int32_t* from = a.parent_history + (g * T + c0) * W;
    const int count = steps * W;
    for (int i = tid * 4; i < count; i += kTThreads * 4) {
      uint32_t four = 0;
      int p[4];
      if (i + 4 <= count) {
        const u32x4 q = *reinterpret_cast<const u32x4_align4*>(from + i);
#pragma unroll
        for (int e = 0; e < 4; ++e) p[e] = (int)q[e];
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) p[e] = i + e < count ? from[i + e] : 0;
      }
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        if ((unsigned)p[e] >= (unsigned)W) p[e] = (i + e) % W;
        four |= (uint32_t)p[e] << (8 * e);
      }
      *reinterpret_cast<uint32_t*>(parent + i) = four;
    }
  }
  __syncthreads();
  // ---- the sub-chunks' maps ----
  const int subs = (steps + kSub - 1) / kSub;
  for (int i = tid; i < subs * W; i += kTThreads) {
    const int s = i / W;
    int b = i - s * W;
    for (int t = min(steps, (s + 1) * kSub) - 1; t >= s * kSub; --t) b = parent[t * W + b];
    sub_map[i] = (uint8_t)b;
  }
  __syncthreads();
  if (MODE == kTraceMaps) {
    // the whole chunk's map, and the hypotheses that end in it (at step len - 2)
    if (tid < W) {
      int b = tid;
      for (int s = subs - 1; s >= 0; --s) b = sub_map[s * W + b];
      maps[(g * chunks + chunk) * W + tid] = (uint8_t)b;
    } else if (tid >= kTThreads / 2 && tid < kTThreads / 2 + n) {
      const int h = tid - kTThreads / 2;
      const int64_t end = (int64_t)s_len[h] - 2 - c0;
      if (end >= 0 && end < S) {
        int b = s_beam[h], t = (int)end;
        for (; t >= 0 && (t + 1) % kSub != 0; --t) b = parent[t * W + b];
        for (int s = (t + 1) / kSub - 1; s >= 0; --s) b = sub_map[s * W + b];
        exits[g * n + h] = (uint8_t)b;
      }
    }
    return;
  }
  // ---- each hypothesis' beam at the top of every sub-chunk ----
  int b = 0;
  int64_t end = -1;  // its last step, from c0
  if (tid < n) {
    b = s_beam[tid];
    end = (int64_t)s_len[tid] - 2 - c0;
    if (MODE == kTraceEmit && end >= S) b = exits[g * n + tid];
  }
  if (MODE == kTraceEmit) {
    // down through the chunks above this one, a piece of their maps at a time
    const int per = kMapPiece / W;
    const int last = (int)((max((int64_t)s_longest - 2, (int64_t)0)) / S);  // uniform
    for (int hi = last; hi > chunk; hi -= per) {
      const int lo = max(chunk + 1, hi - per + 1);
      const uint8_t* from = maps + (g * chunks + lo) * W;
      for (int i = tid; i < (hi - lo + 1) * W; i += kTThreads) s_maps[i] = from[i];
      __syncthreads();
      if (tid < n && end >= S) {
        const int mine = (int)((int64_t)(s_len[tid] - 2) / S) - 1;  // the first one below its own
        for (int c = min(hi, mine); c >= lo; --c) b = s_maps[(c - lo) * W + b];
      }
      __syncthreads();
    }
  }
  if (tid < n && end >= 0) {
    int s = (int)(min(end, (int64_t)steps - 1) / kSub);
    tops[tid * nsub + s] = (uint8_t)b;
    if (s > 0) {
      // the first one from the hypothesis' own last step
      for (int t = (int)min(end, (int64_t)steps - 1); t >= s * kSub; --t) b = parent[t * W + b];
      for (--s; s >= 0; --s) {
        tops[tid * nsub + s] = (uint8_t)b;
        b = sub_map[s * W + b];
      }
    }
  }
  __syncthreads();
  // ---- the beam of every step ----
  for (int i = tid; i < subs * n; i += kTThreads) {
    const int h = i / subs, s = i - h * subs;
    const int64_t top = min((int64_t)s_len[h] - 2 - c0, (int64_t)(s + 1) * kSub - 1);
    if (top < s * kSub) continue;
    int at = tops[h * nsub + s];
    for (int t = (int)min(top, (int64_t)steps - 1); t >= s * kSub; --t) {
      beams[h * S + t] = (uint8_t)at;
      at = parent[t * W + at];
    }
  }
  __syncthreads();
  // ---- the tokens ----
  const int width = (int)min((int64_t)S, T - c0);
  const int32_t* tokens = a.token_history + (g * T + c0) * W;
  for (int h = 0; h < n; ++h) {
    int32_t* out = a.out_token_ids + (g * n + h) * T + c0;
    const int64_t end_h = (int64_t)s_len[h] - 2 - c0;
    for (int t = tid; t < width; t += kTThreads) {
      int32_t id = -1;
      if (t <= end_h) id = tokens[(int64_t)t * W + beams[h * S + t]];
      else if (t == end_h + 1 && s_len[h] > 0) id = s_token[h];
      out[t] = id;
    }
  }
}

hipError_t launch_beam_finish(const mvsd_beam_finish_args& a, hipStream_t stream) {
  const int S = trace_chunk(a.beam_width, a.num_return, a.max_length);
  const int chunks = (int)((a.max_length + S - 1) / S);
  const int lds = trace_lds(a.beam_width, a.num_return, S);
  const dim3 grid((unsigned)(a.num_groups * chunks)), block(kTThreads);
  if (chunks == 1) {
    hipLaunchKernelGGL((beam_trace_kernel<kTraceWhole>), grid, block, lds, stream, a, S, chunks,
                       nullptr, nullptr);
    return hipGetLastError();
  }
  uint8_t* maps = static_cast<uint8_t*>(a.workspace);
  uint8_t* exits = maps + a.num_groups * chunks * a.beam_width;
  hipLaunchKernelGGL((beam_trace_kernel<kTraceMaps>), grid, block, lds, stream, a, S, chunks, maps,
                     exits);
  hipLaunchKernelGGL((beam_trace_kernel<kTraceEmit>), grid, block, lds, stream, a, S, chunks, maps,
                     exits);
  return hipGetLastError();
}

}  // namespace mvsd
