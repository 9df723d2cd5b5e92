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
//
// What bounds it: memory.  Each moved byte is read once (a parent of several beams once for each, the
// others from the caches) and stored past the caches, since nothing here reads it again: 1355 MB of
// eight caches move in 250 us with such stores and 271 with ordinary ones (5.4 TB/s read and written; a
// large copy reaches 4.9), 72 MB of pages in 14.2 us and 17.6.  Sixteen bytes a thread of 8, 16 or 32
// rows (the least that holds W) and eight of 64 stay in registers.  64 rows of eight caches, 4.2 MB a
// row, half of the beams copied onto the others, TB/s: W = 8 5.8, 16 5.6, 24 5.0, 32 5.0, 48 4.0, 64 3.7
// (a copy of 1 GiB there 5.1); with vectors of eight bytes for 16 and 32 rows 5.0 and 4.5, of sixteen for
// 64 (past the registers) 3.8 with 48 and 64 beams.  Into `out`, eight rows at a time, the others read
// again: W = 4 5.6, 8 5.4, 16 4.7, 32 4.5, 64 4.1.

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

template <int ROWS, typename T>
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
        __builtin_nontemporal_store(
            v[w], reinterpret_cast<U*>(
                      dst + (int64_t)__builtin_amdgcn_readlane(to, b + w) * dst_stride + off));
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
      move_rows<ROWS, T>((const char*)s.src, (char*)s.dst, s.src_stride, s.dst_stride,
                         at + (int64_t)i * (int64_t)sizeof(T), moves, from, to, W);
    else
      move_rows<ROWS, uint8_t>((const char*)s.src, (char*)s.dst, s.src_stride, s.dst_stride,
                               at + (int64_t)whole * (int64_t)sizeof(T) + (i - whole), moves, from,
                               to, W);
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
// beam's place.  A parent outside [0, W) is the beam itself; a finished hypothesis' beam outside it, of
// which there is no other record, counts as beam 0.
//
// With b_t the beam at step t, b_(t-1) = parent_t(b_t): a chain of T dependent reads.  The steps'
// maps are composed instead.  A workgroup holds the parents of a chunk of steps in LDS, a byte each,
// in sub-chunks of kSub steps and spans of kSpan sub-chunks:
//   1 every sub-chunk is walked from every beam at once: its map (and each hypothesis down to the
//     bottom of the sub-chunk that it ends in);
//   2 the maps of a span's sub-chunks are composed (and each hypothesis down to its span's bottom);
//   3 the hypotheses go down through the spans;
//   4 and, for every span at once, through its sub-chunks;
//   5 every sub-chunk is walked again from there, all at once, and leaves the beam of each step, by
//     which the workgroup writes the sequences' tokens, on their way since the start.
// What bounds it: latencies in a row.  Of a workgroup's 23400 cycles (27400 the slowest) of 64 groups of 8
// beams and 2048 steps, 10 MB in 15.6 us, the lengths, histories and hypotheses take 6400, the walks 3300,
// 1800, 1500, 1800 and 2700 (16 dependent LDS reads each in 1 and 5, up to 8 in the others) and the tokens'
// way out 6000; an empty launch is 2.8 us.  One group of 64 steps takes 7.9 us, 16500 cycles: 4600, 8700
// and 3000.
// Where there are few groups, several workgroups share a group's hypotheses; all of them compose.
// Histories of one chunk take one launch.  Longer ones take two: the first leaves the hypotheses,
// every chunk's map and, for a hypothesis that ends in the chunk, its beam below it; the second starts
// from those (4 groups of 4 beams and 65536 steps: 7.0 and 11.4 us).

constexpr int kTThreads = 512;
constexpr int kSub = 16, kSpan = 8, kSpanSteps = kSub * kSpan;
constexpr int kTraceLds = 50 * 1024;  // of W + n bytes a step; the maps and the padding add a fifth
constexpr int kMapPiece = 4096;       // bytes of chunk maps held at a time
constexpr int kAhead = 8;             // vectors of parents, and of tokens, that a thread holds
constexpr int kTraceGroups = 256;     // workgroups that a launch is split into at least
enum { kTraceWhole, kTraceMaps, kTraceEmit };

// Steps per chunk: the whole history where it fits LDS and is short, else 2048 steps or fewer.
static int trace_chunk(int64_t W, int64_t n, int64_t T) {
  if (T <= 4096 && T * (W + n) <= kTraceLds) return (int)T;
  return W + n <= 24 ? 2048 : W + n <= 48 ? 1024 : 384;
}

// Dynamic LDS, bytes.  A sub-chunk's parents, and its beams of one hypothesis, take four bytes more
// than they need: lanes that walk neighbouring sub-chunks then read different banks (a stride of 16
// steps of 8 beams has 32 lanes on one: step 5 over 2048 steps took 9200 cycles, with them 5400).
__host__ __device__ constexpr int parents_stride(int W) { return kSub * W + 4; }
constexpr int kBeamsStride = kSub + 4;
static int trace_lds(int64_t W, int64_t n, int64_t S) {
  const int64_t subs = (S + kSub - 1) / kSub, spans = (S + kSpanSteps - 1) / kSpanSteps;
  return (int)(subs * (parents_stride((int)W) + n * kBeamsStride + W + n) + spans * (W + n));
}

// Workspace of two launches: hypotheses (beam, last token, length, beam below its chunk) and maps.
int64_t beam_finish_workspace_bytes(int64_t G, int64_t W, int64_t T, int64_t n) {
  const int64_t S = trace_chunk(W, n, T), chunks = (T + S - 1) / S;
  return chunks > 1 ? G * (n * 16 + chunks * W) : 0;
}

struct TraceSmem {
  float score[kMaxBeams];
  int beam[kMaxBeams], token[kMaxBeams], len[kMaxBeams];
  uint8_t exit[kMaxBeams];  // a hypothesis' beam below the sub-chunk that it ends in
};

// The group's n best hypotheses, by one wave: lane w holds finished hypothesis w and running beam w.
__device__ inline void best_hypotheses(const mvsd_beam_finish_args& a, int64_t g, int len,
                                       TraceSmem& sm) {
  const int lane = lane_id(), W = (int)a.beam_width, n = (int)a.num_return, T = (int)a.max_length;
  const int64_t at = g * W + min(lane, W - 1);
  const int64_t last = (g * T + max(len - 1, 0)) * W + min(lane, W - 1);
  float old = a.finished_scores[at];
  const float running = a.scores[at];
  const int old_beam = a.finished_beams[at], old_token = a.finished_token_ids[at];
  const int old_len = a.finished_lengths[at];
  const int beam = a.parent_history[last], token = a.token_history[last];
  const bool runs = a.done[g] == 0 && len > 0 && fabsf(running) < INFINITY;
  float now = runs ? hypothesis_score(running, len_power(len, a.length_penalty)) : -INFINITY;
  if (!(old > -INFINITY) || lane >= W) old = -INFINITY;
  if (!(now > -INFINITY) || lane >= W) now = -INFINITY;
  int rank_old = 0, rank_now = 0;
  for (int j = 0; j < W; ++j) {
    const float o = readlane_f32(old, j), r = readlane_f32(now, j);
    rank_old += (o > old || (o == old && j < lane)) + (r > old);
    rank_now += (o >= now) + (r > now || (r == now && j < lane));
  }
  auto put = [&](int rank, float score, int b, int own, int id, int l) {
    const bool any = score > -INFINITY;
    sm.beam[rank] = !any ? 0 : b >= 0 && b < W ? b : own;
    sm.token[rank] = id;
    sm.len[rank] = any ? min(max(l, 0), T) : 0;
    sm.score[rank] = score;
  };
  if (lane < W && rank_old < n) put(rank_old, old, old_beam, 0, old_token, old_len);
  if (lane < W && rank_now < n) put(rank_now, now, beam, lane, token, len);
}

// Workgroup (group, chunk, part): hypotheses [part * per, part * per + per) of the group.  Sizes of
// one group stay below 2^31 (the entry point checks), so offsets within it are ints.
template <int MODE>
__global__ __launch_bounds__(kTThreads) void beam_trace_kernel(mvsd_beam_finish_args a, int S,
                                                                int chunks, int parts, int per,
                                                                int32_t* hyps, uint8_t* maps) {
  __shared__ TraceSmem sm;
  __shared__ uint8_t s_maps[MODE == kTraceEmit ? kMapPiece : 1];
  extern __shared__ __align__(16) uint8_t lds[];
  const int tid = threadIdx.x, lane = lane_id(), wid = wave_id();
  const int W = (int)a.beam_width, n = (int)a.num_return, T = (int)a.max_length;
  const int gc = blockIdx.x / parts, part = blockIdx.x - gc * parts;
  const int64_t g = gc / chunks;
  const int chunk = gc - (int)g * chunks, c0 = chunk * S;
  const int h0 = part * per, nh = min(per, n - h0);
  const int max_subs = (S + kSub - 1) / kSub, max_spans = (S + kSpanSteps - 1) / kSpanSteps;
  const int sub_bytes = parents_stride(W);
  uint8_t* parent = lds;                                      // [subs, sub_bytes]: 16 steps of W
  uint8_t* beams = parent + max_subs * sub_bytes;             // [per, subs, kBeamsStride]
  uint8_t* sub_map = beams + max_subs * per * kBeamsStride;   // [subs, W]
  uint8_t* sub_top = sub_map + max_subs * W;                  // [per, subs]
  uint8_t* span_map = sub_top + max_subs * per;               // [spans, W]
  uint8_t* span_top = span_map + max_spans * W;               // [per, spans]
  // ---- how far the parents are needed: no hypothesis is longer (every wave for itself) ----
  const int len = min(max(a.lengths[g], 0), T);
  int longest = 0;
  if (MODE == kTraceEmit) longest = lane < n ? hyps[(g * n + lane) * 4 + 2] : 0;
  else longest = min(max(a.finished_lengths[g * W + min(lane, W - 1)], len), T);
  longest = (int)wave_max_u32((uint32_t)max(longest, 0));
  const int steps = min(max(longest - 1 - c0, 0), S);
  if (MODE == kTraceMaps && steps == 0 && chunk > 0) return;  // (the first has the hypotheses to write)
  // ---- parents and tokens on their way, the hypotheses meanwhile ----
  const int32_t* parents = a.parent_history + (g * T + c0) * W;
  const int32_t* tokens = a.token_history + (g * T + c0) * W;
  const int count = steps * W, vecs = count / 4;
  auto vec_of = [&](const int32_t* from, int i) {
    return *reinterpret_cast<const u32x4_align4*>(from + 4 * min(i, vecs - 1));
  };
  u32x4 q[kAhead], id[kAhead];
  if (vecs > 0) {  // uniform
#pragma unroll
    for (int k = 0; k < kAhead; ++k) q[k] = vec_of(parents, tid + k * kTThreads);
    if (MODE != kTraceMaps) {
#pragma unroll
      for (int k = 0; k < kAhead; ++k) id[k] = vec_of(tokens, tid + k * kTThreads);
    }
  }
  if (wid == 0) {
    if (MODE == kTraceEmit) {
      if (lane < n) {
        const int32_t* h = hyps + (g * n + lane) * 4;
        sm.beam[lane] = h[0];
        sm.token[lane] = h[1];
        sm.len[lane] = h[2];
      }
    } else {
      best_hypotheses(a, g, len, sm);
    }
  }
  // a vector's four parents lie in one sub-chunk (16 W is a multiple of four)
  bool outside = false;
  auto pack = [&](int i, const u32x4& v) {
    outside |= max(max(v[0], v[1]), max(v[2], v[3])) >= (uint32_t)W;
    *reinterpret_cast<uint32_t*>(parent + 4 * i + 4 * (i / (4 * W))) =
        v[0] | v[1] << 8 | v[2] << 16 | v[3] << 24;
  };
#pragma unroll
  for (int k = 0; k < kAhead; ++k)
    if (tid + k * kTThreads < vecs) pack(tid + k * kTThreads, q[k]);
  for (int i0 = kAhead * kTThreads + tid; i0 < vecs; i0 += kAhead * kTThreads) {
#pragma unroll
    for (int k = 0; k < kAhead; ++k) q[k] = vec_of(parents, i0 + k * kTThreads);
#pragma unroll
    for (int k = 0; k < kAhead; ++k)
      if (i0 + k * kTThreads < vecs) pack(i0 + k * kTThreads, q[k]);
  }
  // one by one: what is left, and the vectors of a thread that saw a parent outside the group
  auto one = [&](int i) {
    const uint32_t p = (uint32_t)parents[i];
    parent[i + 4 * (i / (kSub * W))] = (uint8_t)(p >= (uint32_t)W ? (uint32_t)(i % W) : p);
  };
  if (4 * vecs + tid < count) one(4 * vecs + tid);
  if (outside)
    for (int i = tid; i < vecs; i += kTThreads)
      for (int e = 0; e < 4; ++e) one(4 * i + e);
  __syncthreads();
  if (MODE != kTraceEmit && chunk == 0 && part == 0 && tid < n) {
    a.out_scores[g * n + tid] = sm.score[tid];
    a.out_lengths[g * n + tid] = sm.len[tid];
    if (MODE == kTraceMaps) {
      int32_t* h = hyps + (g * n + tid) * 4;
      h[0] = sm.beam[tid];
      h[1] = sm.token[tid];
      h[2] = sm.len[tid];
    }
  }
  const int subs = (steps + kSub - 1) / kSub, spans = (steps + kSpanSteps - 1) / kSpanSteps;
  // the last step of this workgroup's hypothesis h, from c0: in the chunk, below (negative), or above
  auto end_of = [&](int h) { return sm.len[h0 + h] - 2 - c0; };
  auto ends_here = [&](int end) { return end >= 0 && end < S; };
  // Two walks of a thread side by side, down the 16 steps of sub-chunks s[k] from beams b[k], which
  // enter at steps top[k] (from the sub-chunk's bottom; above it a walk stands still: what the parents
  // say there is not used, and may be anything).
  auto walk = [&](const int (&s)[2], int (&b)[2], const int (&top)[2], auto&& seen) {
    const uint8_t* base[2] = {parent + s[0] * sub_bytes, parent + s[1] * sub_bytes};
#pragma unroll
    for (int t = kSub - 1; t >= 0; --t)
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        seen(k, t, b[k]);
        const int next = base[k][t * W + b[k]];
        b[k] = t <= top[k] ? next : b[k];
      }
  };
  // ---- 1: sub-chunks ----
  for (int i0 = tid; i0 < subs * W + nh; i0 += 2 * kTThreads) {
    int s[2], b[2], top[2];
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const int i = i0 + k * kTThreads;
      s[k] = b[k] = 0;
      top[k] = -1;
      if (i < subs * W) {
        s[k] = i / W;
        b[k] = i - s[k] * W;
        top[k] = min(steps - s[k] * kSub, kSub) - 1;
      } else if (i < subs * W + nh) {
        const int end = end_of(i - subs * W);
        if (ends_here(end)) {
          b[k] = sm.beam[h0 + i - subs * W];
          s[k] = end / kSub;
          top[k] = end % kSub;
        }
      }
    }
    walk(s, b, top, [](int, int, int) {});
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const int i = i0 + k * kTThreads;
      if (i < subs * W) sub_map[i] = (uint8_t)b[k];
      else if (i < subs * W + nh) sm.exit[i - subs * W] = (uint8_t)b[k];
    }
  }
  __syncthreads();
  // ---- 2: spans ----
  for (int i = tid; i < spans * W; i += kTThreads) {
    const int p = i / W;
    int m = i - p * W;
    for (int s = min(subs, (p + 1) * kSpan) - 1; s >= p * kSpan; --s) m = sub_map[s * W + m];
    span_map[i] = (uint8_t)m;
  }
  int end = -1, b = 0;
  if (tid < nh) {
    end = end_of(tid);
    b = sm.exit[tid];
    if (ends_here(end)) {
      const int e = end / kSub;
      for (int s = e - 1; s >= e / kSpan * kSpan; --s) b = sub_map[s * W + b];
    }
  }
  __syncthreads();
  if (MODE == kTraceMaps) {
    // the whole chunk's map, and the hypotheses that end in it
    if (tid >= kTThreads / 2 && tid < kTThreads / 2 + W && steps > 0) {
      int m = tid - kTThreads / 2;
      for (int p = spans - 1; p >= 0; --p) m = span_map[p * W + m];
      maps[(g * chunks + chunk) * W + tid - kTThreads / 2] = (uint8_t)m;
    }
    if (tid < nh && ends_here(end)) {
      for (int p = end / kSpanSteps - 1; p >= 0; --p) b = span_map[p * W + b];
      hyps[(g * n + h0 + tid) * 4 + 3] = b;
    }
    return;
  }
  // ---- 3: down through the spans ----
  if (MODE == kTraceEmit) {
    // first through the chunks above this one, a piece of their maps at a time
    if (tid < nh && end >= S) b = hyps[(g * n + h0 + tid) * 4 + 3];
    const int piece = kMapPiece / W;
    const int last = max(longest - 2, 0) / S;
    for (int hi = last; hi > chunk; hi -= piece) {
      const int lo = max(chunk + 1, hi - piece + 1);
      const uint8_t* m = maps + (g * chunks + lo) * W;
      for (int i = tid; i < (hi - lo + 1) * W; i += kTThreads) s_maps[i] = m[i];
      __syncthreads();
      if (tid < nh && end >= S) {
        const int mine = (end + c0) / S - 1;  // the first one below its own
        for (int c = min(hi, mine); c >= lo; --c) b = s_maps[(c - lo) * W + b];
      }
      __syncthreads();
    }
  }
  if (tid < nh && end >= 0) {
    // the spans it goes through as a whole; its own, where it has one here, starts at its end
    for (int p = ends_here(end) ? end / kSpanSteps - 1 : spans - 1; p >= 0; --p) {
      span_top[tid * max_spans + p] = (uint8_t)b;
      b = span_map[p * W + b];
    }
  }
  __syncthreads();
  // ---- 4: through every span's sub-chunks ----
  for (int i = tid; i < spans * nh; i += kTThreads) {
    const int p = i / nh, h = i - p * nh, e = end_of(h);
    if (e < p * kSpanSteps) continue;
    int s = min(subs, (p + 1) * kSpan) - 1, at;
    if (ends_here(e) && e / kSpanSteps == p) {
      s = e / kSub;
      sub_top[h * max_subs + s] = (uint8_t)sm.beam[h0 + h];
      --s;
      at = sm.exit[h];
    } else {
      at = span_top[h * max_spans + p];
    }
    for (; s >= p * kSpan; --s) {
      sub_top[h * max_subs + s] = (uint8_t)at;
      at = sub_map[s * W + at];
    }
  }
  __syncthreads();
  // ---- 5: the beam of every step ----
  for (int i0 = tid; i0 < subs * nh; i0 += 2 * kTThreads) {
    int s[2], at[2], top[2];
    uint32_t four[2] = {0, 0};
    uint32_t* to[2];
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const int i = min(i0 + k * kTThreads, subs * nh - 1), h = i / subs;
      s[k] = i - h * subs;
      const int e = end_of(h) - s[k] * kSub;
      top[k] = min(e, kSub - 1);
      at[k] = e >= 0 ? sub_top[h * max_subs + s[k]] : 0;
      to[k] = reinterpret_cast<uint32_t*>(beams + (h * max_subs + s[k]) * kBeamsStride);
    }
    walk(s, at, top, [&](int k, int t, int beam) {
      four[k] = four[k] << 8 | (uint32_t)beam;
      if (t % 4 == 0) to[k][t / 4] = four[k];
    });
  }
  __syncthreads();
  // ---- the tokens: who holds a step's tokens writes those of the hypotheses that go through them ----
  const int width = min(S, T - c0);
  int32_t* out = a.out_token_ids + (g * n + h0) * T + c0;
  auto beam_at = [&](int h, int t) {
    return (int)beams[(h * max_subs + t / kSub) * kBeamsStride + t % kSub];
  };
  auto write = [&](int i0) {
    if (W % 4 == 0) {  // uniform: a vector is four beams of one step
      int t[kAhead], w0[kAhead];
#pragma unroll
      for (int k = 0; k < kAhead; ++k) {
        const int i = 4 * min(i0 + k * kTThreads, vecs - 1);
        t[k] = i / W;
        w0[k] = i - t[k] * W;
        if (i0 + k * kTThreads >= vecs) t[k] = INT32_MAX;
      }
      for (int h = 0; h < nh; ++h) {
        const int e = end_of(h);
        int32_t* row = out + h * T;
#pragma unroll
        for (int k = 0; k < kAhead; ++k) {
          const uint32_t d = (uint32_t)(beam_at(h, min(t[k], steps - 1)) - w0[k]);
          const uint32_t low = d & 1 ? id[k][1] : id[k][0], high = d & 1 ? id[k][3] : id[k][2];
          if (d < 4 && t[k] <= e) row[t[k]] = (int32_t)(d & 2 ? high : low);
        }
      }
    } else {
#pragma unroll
      for (int k = 0; k < kAhead; ++k)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int i = 4 * (i0 + k * kTThreads) + e, t = i / W, w = i - t * W;
          if (i >= 4 * vecs) continue;
          for (int h = 0; h < nh; ++h)
            if (beam_at(h, t) == w && t <= end_of(h)) out[h * T + t] = (int32_t)id[k][e];
        }
    }
  };
  if (tid < vecs) write(tid);
  for (int i0 = kAhead * kTThreads + tid; i0 < vecs; i0 += kAhead * kTThreads) {
#pragma unroll
    for (int k = 0; k < kAhead; ++k) id[k] = vec_of(tokens, i0 + k * kTThreads);
    write(i0);
  }
  if (4 * vecs + tid < count) {  // the last one to three
    const int i = 4 * vecs + tid, t = i / W, w = i - t * W;
    for (int h = 0; h < nh; ++h)
      if (beam_at(h, t) == w && t <= end_of(h)) out[h * T + t] = tokens[i];
  }
  for (int h = 0; h < nh; ++h) {  // the last token, and what is behind the sequence
    const int e = end_of(h);
    for (int t = max(e + 1, 0) + tid; t < width; t += kTThreads)
      out[h * T + t] = t == e + 1 && sm.len[h0 + h] > 0 ? sm.token[h0 + h] : -1;
  }
}

hipError_t launch_beam_finish(const mvsd_beam_finish_args& a, hipStream_t stream) {
  const int W = (int)a.beam_width, n = (int)a.num_return;
  const int S = trace_chunk(W, n, a.max_length);
  const int chunks = (int)((a.max_length + S - 1) / S);
  const int64_t wgs = a.num_groups * chunks;
  // hypotheses shared out until there are kTraceGroups workgroups, one per compute unit: 64 groups of 8
  // beams and 2048 steps take 19.4 us unshared, 15.9 with 128, 14.2 with 256 and 19.4 with 512 (every
  // workgroup reads the group's histories); 8 groups of 32 beams and 512 steps 16.7, 14.8, 13.7, 13.8
  const int64_t want = wgs < kTraceGroups ? (kTraceGroups + wgs - 1) / wgs : 1;
  const int per = want < n ? (int)((n + want - 1) / want) : 1;
  const int parts = (n + per - 1) / per;
  const int lds = trace_lds(W, per, S);
  const dim3 grid((unsigned)(wgs * parts)), block(kTThreads);
  if (chunks == 1) {
    hipLaunchKernelGGL((beam_trace_kernel<kTraceWhole>), grid, block, lds, stream, a, S, chunks,
                       parts, per, nullptr, nullptr);
    return hipGetLastError();
  }
  int32_t* hyps = static_cast<int32_t*>(a.workspace);
  uint8_t* maps = reinterpret_cast<uint8_t*>(hyps + a.num_groups * n * 4);
  hipLaunchKernelGGL((beam_trace_kernel<kTraceMaps>), dim3((unsigned)wgs), block,
                     trace_lds(W, n, S), stream, a, S, chunks, 1, n, hyps, maps);
  hipLaunchKernelGGL((beam_trace_kernel<kTraceEmit>), grid, block, lds, stream, a, S, chunks, parts,
                     per, hyps, maps);
  return hipGetLastError();
}

}  // namespace mvsd
