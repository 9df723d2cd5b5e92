// Beam search: the selection over beams and vocabulary, and a decoding step around it.
//
// A group is one request with W beams.  Beam b has the summed log-probability s_b and a row of
// logits x_b over V tokens:
//   lse_b       = log sum_v exp(x_bv)
//   total(b, v) = s_b + (x_bv - lse_b)
// and the group's candidates are its C largest totals, in the order (total descending, beam
// ascending, logit descending, token ascending).  A beam whose score or lse is not finite (no beam,
// a row masked everywhere, a NaN or +inf) proposes nothing; entries of -inf are no candidates.
//
//   beam_scan_kernel    one 256-thread workgroup per (beam, chunk of columns) reads the chunk once,
//                       into registers, and leaves its maximum, its sum of exp(x - maximum) and the
//                       largest entry of every 16 or 2 lanes (a "top").
//   beam_select_kernel, beam_step_kernel: the finish, one 512-thread workgroup per group:
//     - lse_b in 64 bits from the chunks' sums;
//     - theta, the C-th largest of the maxima of 512 disjoint unions of tops (64 for C <= 32), as
//       totals: at least C entries of the group reach it, so the candidates are among the entries
//       that do, and these lie under the tops that do (a few more than C);
//     - per beam the logit that theta stands for (rounded down), so that tops and entries are compared
//       as they are; the entries under the tops that reach it are gathered into LDS, their totals
//       formed in 64 bits, and ranked by counting;
//     - more entries than LDS holds (long runs of one value: masks of the type's lowest value, a
//       uniform row): the beams one after the other, each one's C largest by a radix selection.
//   A step goes on in the same workgroup: stop tokens, finished hypotheses, histories.
//
// Order: a lane's sum of up to 32 exponentials is fp32, in pairs, everything after it fp64, which leaves
// an lse with a deviation of 2e-8 (rows of 1000 columns) to 6e-9 (151936) from the 64-bit one, at most
// 9.1e-7 for any row (at kNear) and 2^-18 of a log-probability close to zero (at kPeaked).  Candidates of
// one beam are ordered by their logits; where two neighbouring candidates of different beams are closer
// than kNear, both beams' lse are formed again with 64-bit exponentials: the order is the 64-bit one.
//
// What bounds it (bf16 rows of 151936 columns, one MI355X): 1024 rows the scan, 48 us of 57 (6.45 TB/s);
// four rows the chain of two launches, 3 and 6 us.  Scans of 20 to 30 MB are one round of workgroups, whose
// reads and arithmetic follow each other: of 10.5 us for 512 fp16 rows of 32000 columns an empty kernel
// takes 2.8, the reads 4.0 more and the arithmetic 3.7 (0.7 of it the exponentials).  The finish is a chain
// too: the scan's results, 7 barriers, one gather.  One launch in which the last workgroup of a group
// finishes it was no faster (four rows 9.7 us against 8.8, 256 rows 38 against 22: the agent-scope stores
// and counters).
#include "beam.h"
#include "mvsd_device.h"

namespace mvsd {

constexpr int kFThreads = 512;
constexpr int kFWaves = kFThreads / kWave;
constexpr int kListCap = 1024;     // tops that reach theta
constexpr int kCandCap = 1024;     // gathered entries
constexpr int kHeld = 4;           // vectors of tops a thread keeps in registers
constexpr int kStats = 2;          // chunks that a lane of a beam loads at a time
constexpr int kPowerBits = 8, kPowers = 1 << kPowerBits;  // of a 64-bit exponential's table
constexpr int kFoldC = 32;         // the largest C whose theta is read off 64 keys

// How rows are split: columns per chunk, and the lanes that share a top (each holds NV vectors of the
// chunk).  Long chunks, unless they leave compute units idle (fewer than 4 workgroups each) or give a
// row fewer than two tops per candidate (a group may have one beam only), so that theta is a poor bound
// or none.  Short rows can have too few even then: tops of two lanes (6 groups of 16 bf16 beams, 64
// candidates: rows of 1088 columns 114 us with tops of 16 lanes and 23.6 with tops of 2; of 4096 columns
// 1285, where theta leaves more entries than LDS holds, and 19.0; 8 candidates of 1088 10.5 and 9.8).
constexpr int kBeamLong = 8192, kBeamShort = 2048;
constexpr int kCoarse = 16, kFine = 2;

struct BeamSplit {
  int chunk, lanes;
  int64_t chunks;
  int tops() const { return kThreads / lanes; }  // of a chunk
};

static BeamSplit beam_split(int64_t rows, int64_t V, int64_t C) {
  const int64_t large = (V + kBeamLong - 1) / kBeamLong, small = (V + kBeamShort - 1) / kBeamShort;
  if (rows * large >= 1024 && V / (kCoarse * 32) >= 2 * C) return {kBeamLong, kCoarse, large};
  return {kBeamShort, V / (kCoarse * 8) >= 2 * C ? kCoarse : kFine, small};
}

// exp(d), d <= 0, as 2^(d log2(e)) with log2(e) in two parts, so that its rounding leaves no bias: the
// mean error of a row's lse went from 4.0e-8 to 3e-9 and less.
__device__ inline float exp_of(float d) {
  return __builtin_amdgcn_exp2f(fmaf(d, 1.44269504f, d * 1.92596304e-8f));
}

// The sum of f(0) ... f(N - 1), N a power of two, in pairs: at most log2(N) roundings of each term.
template <int N, typename F>
__device__ inline float pair_sum(F&& f, int from = 0) {
  if constexpr (N == 1) return f(from);
  else return pair_sum<N / 2>(f, from) + pair_sum<N / 2>(f, from + N / 2);
}

__device__ inline bool finite(float x) { return fabsf(x) < INFINITY; }

// Sums and maxima over `lanes` (a power of two from 8 to 64) neighbouring lanes, in each of them.
template <int CTRL>
__device__ inline double dpp_f64(double v) {
  return __builtin_bit_cast(double, dpp_u64<CTRL>(__builtin_bit_cast(uint64_t, v)));
}
__device__ inline double lanes_sum(double v, int lanes) {
  v += dpp_f64<kDppXor1>(v);
  v += dpp_f64<kDppXor2>(v);
  v += dpp_f64<kDppHalfMirror>(v);
  if (lanes > 8) v += dpp_f64<kDppMirror>(v);
  for (int off = 16; off < lanes; off *= 2) v += __shfl_xor(v, off, kWave);
  return v;
}
__device__ inline float lanes_max(float v, int lanes) {
  v = fmaxf(v, dpp_f32<kDppXor1>(v));
  v = fmaxf(v, dpp_f32<kDppXor2>(v));
  v = fmaxf(v, dpp_f32<kDppHalfMirror>(v));
  if (lanes > 8) v = fmaxf(v, dpp_f32<kDppMirror>(v));
  for (int off = 16; off < lanes; off *= 2) v = fmaxf(v, __shfl_xor(v, off, kWave));
  return v;
}

// Whether a step leaves the group as it is.
__device__ inline bool group_rests(const BeamScanParams& p, int g) {
  if (!p.lengths) return false;
  const int len = p.lengths[g];
  return p.done[g] != 0 || len < 0 || len >= p.max_length;
}

template <typename S>
__device__ inline const S* beam_row(const BeamScanParams& p, int64_t r) {
  int64_t row = r;
  if (p.rows) row = min(max((int64_t)p.rows[r], (int64_t)0), p.num_rows - 1);
  return static_cast<const S*>(p.logits) + row * p.stride;
}

// Rows of kStreamBytes together are read past the caches: what the model's last product left of them
// does not fit the 256 MB that the memory side keeps, and nothing of a scan is read again but the few
// entries of the finish.  bf16 rows, cached and past the caches: 78 MB 21.9 and
// 22.0 us, 102 MB 26.4 and 26.7, 160 MB 35.7 and 34.2, 311 MB 61.8 and 56.4.
constexpr int64_t kStreamBytes = 128ll << 20;

template <int DT, bool STREAM>
__device__ inline u32x4 load_scan(const typename Elem<DT>::storage* row, int col, int V) {
  if (!STREAM || V < Elem<DT>::kVec) return load_vec_inside<DT>(row, col, V);
  return __builtin_nontemporal_load(
      reinterpret_cast<const Vec16<DT>*>(row + min(col, V - Elem<DT>::kVec)));
}

// A wave whose sum, its maximum's 1 included, is below kPeaked adds its exponentials again without that one
// (no other is 1: the sum would be 2), which then comes in 64 bits.  In its lane's fp32 sum, what is below
// 2^-24 beside it would be lost, and the log-probability of a confident model's best token is
// -log(1 + rest) of such waves: with 151936 entries 20 below the best one it was 2e-4 of itself off, now at
// most the 1.7e-6 of an exponential.  Above kPeaked the partial sums' 3.0e-7 are at most 1.4e-6 of
// log(kPeaked).  (The branch costs nothing measurable where it is not taken; the largest entry left out
// everywhere took 63 us instead of 58 for 128 groups of 8 bf16 rows of 151936.)
constexpr double kPeaked = 1.25;

template <int DT, int NV, int LANES, bool STREAM>
__global__ __launch_bounds__(kThreads) void beam_scan_kernel(BeamScanParams p) {
  constexpr int kTops = kThreads / LANES;
  using S = typename Elem<DT>::storage;
  constexpr int VEC = Elem<DT>::kVec;
  constexpr int CH = NV * kThreads * VEC;
  __shared__ float s_m[kWaves];
  __shared__ double s_s[kWaves];
  const int r = blockIdx.x / p.nchunks, c = blockIdx.x - r * p.nchunks;
  if (!finite(p.scores[r]) || group_rests(p, r / p.W)) return;  // the finish does the same test
  const S* row = beam_row<S>(p, r);
  const int tid = threadIdx.x;
  const int64_t base = (int64_t)c * CH;
  const int left = (int)min((int64_t)p.V - base, (int64_t)CH);  // columns of the chunk
  row += base;
  u32x4 q[NV];
#pragma unroll
  for (int j = 0; j < NV; ++j) q[j] = load_scan<DT, STREAM>(row, (j * kThreads + tid) * VEC, left);
  float v[NV][VEC];
#pragma unroll
  for (int j = 0; j < NV; ++j)
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
      v[j][e] = vec_elem<DT>(q[j], e);
      if (left < CH)
        v[j][e] = inside_col<DT>((j * kThreads + tid) * VEC, e, left) < 0 ? -INFINITY : v[j][e];
    }
  float m = -INFINITY;
#pragma unroll
  for (int j = 0; j < NV; ++j)
#pragma unroll
    for (int e = 0; e < VEC; ++e) m = fmaxf(m, v[j][e]);
  const float pair = fmaxf(m, dpp_f32<kDppXor1>(m)), top16 = max16(m);
  const float top = LANES == kFine ? pair : top16;
  const float wm = fmaxf(fmaxf(readlane_f32(top16, 0), readlane_f32(top16, 16)),
                         fmaxf(readlane_f32(top16, 32), readlane_f32(top16, 48)));
  float s = 0.f;
  if (wm != -INFINITY) {  // +inf gives a NaN sum, as a NaN does
#pragma unroll
    for (int j = 0; j < NV; ++j)
#pragma unroll
      for (int e = 0; e < VEC; ++e) v[j][e] = exp_of(v[j][e] - wm);
    s = pair_sum<NV * VEC>([&](int i) { return v[i / VEC][i % VEC]; });
  } else {  // every entry is -inf or NaN
#pragma unroll
    for (int j = 0; j < NV; ++j)
#pragma unroll
      for (int e = 0; e < VEC; ++e) s += v[j][e] != v[j][e] ? NAN : 0.f;
  }
  double sum64 = lanes_sum((double)s, kWave);
  if (wm != -INFINITY && sum64 < kPeaked) {  // wave-uniform; a NaN sum is not
    s = pair_sum<NV * VEC>([&](int i) {
      const float e = v[i / VEC][i % VEC];
      return e == 1.f ? 0.f : e;
    });
    sum64 = 1.0 + lanes_sum((double)s, kWave);
  }
  const int64_t slot = (int64_t)r * p.nchunks + c;
  if (tid % LANES == 0) p.tops[slot * kTops + tid / LANES] = top;
  if (lane_id() == 0) {
    s_m[wave_id()] = wm;
    s_s[wave_id()] = sum64;
  }
  __syncthreads();
  if (wave_id() != 0) return;
  // the waves' sums, each with its own maximum
  float M = s_m[0];
#pragma unroll
  for (int w = 1; w < kWaves; ++w) M = fmaxf(M, s_m[w]);
  const int w = tid % kWaves;
  double sum = s_m[w] == -INFINITY ? s_s[w] : s_s[w] * exp((double)s_m[w] - (double)M);
  sum += dpp_f64<kDppXor1>(sum);
  sum += dpp_f64<kDppXor2>(sum);
  if (tid == 0) p.stats[slot] = {sum, M};
}

// ------------------------------------------------------------------ finish -----------

// Candidates in LDS, an array each.
template <int N>
struct Candidates {
  double total[N];
  float x[N];
  int token[N], beam[N];
};

struct Candidate {
  double total;
  float x;
  int token, beam;
};

template <int N>
__device__ inline Candidate get(const Candidates<N>& c, int i) {
  return {c.total[i], c.x[i], c.token[i], c.beam[i]};
}
template <int N>
__device__ inline void put(Candidates<N>& c, int i, const Candidate& o) {
  c.total[i] = o.total;
  c.x[i] = o.x;
  c.token[i] = o.token;
  c.beam[i] = o.beam;
}

// Whether candidate j of c comes before `mine` (equal totals are rare: the rest is read only then).
template <int N>
__device__ inline bool before(const Candidates<N>& c, int j, const Candidate& mine) {
  const double t = c.total[j];
  bool yes = t > mine.total;
  if (t == mine.total) {
    const int beam = c.beam[j], token = c.token[j];
    const float x = c.x[j];
    yes = beam != mine.beam ? beam < mine.beam : x != mine.x ? x > mine.x : token < mine.token;
  }
  return yes;
}

struct BeamSmem {
  Candidates<kCandCap> cand;
  Candidates<kMaxCandidates> best;  // the group's candidates in order
  int2 list[kListCap];  // beam, top of the beam's row
  __align__(16) float key[kFThreads];
  float fold[kFWaves];
  int above_key[kWave];
  int64_t row[kMaxBeams];  // the first element of each beam's row
  double lse[kMaxBeams];
  float score[kMaxBeams];  // -inf: proposes nothing
  float most[kMaxBeams];   // the row's largest entry
  double red[kFWaves];
  double power[kPowers];   // 2^(k / kPowers)
  uint64_t near_ties, edge;  // beams whose candidates' order depends on their lse's last digits
  float floor[kMaxBeams];  // the least logit that can be a candidate (+inf: none)
  int hist[256];
  int wave_cnt[kFWaves];
  uint64_t stop_mask[kMaxCandidates / kWave], on_mask[kMaxCandidates / kWave];
  int stop[kMaxCandidates];  // a step's stop tokens
  float pool[2 * kMaxBeams];
  int listed, count, above, digit;
  float worst;
};

// The C-th largest of the workgroup's keys (in sm.key, `own` the thread's): fewer than C keys are above
// it, and it is the least such key.
__device__ inline float block_theta(float own, int C, BeamSmem& sm) {
  int above = 0;
  const float4* keys = reinterpret_cast<const float4*>(sm.key);
#pragma unroll 8
  for (int j = 0; j < kFThreads / 4; ++j) {
    const float4 o = keys[j];
    above += (o.x > own) + (o.y > own) + (o.z > own) + (o.w > own);
  }
  const float least = wave_max(above < C ? -own : -INFINITY);
  if (lane_id() == 0) sm.fold[wave_id()] = least;
  __syncthreads();
  float all = -INFINITY;
#pragma unroll
  for (int k = 0; k < kFWaves; ++k) all = fmaxf(all, sm.fold[k]);
  return -all;
}

// Calls see(col, x) for a workgroup's share of the columns [from, to) of a row whose entries pass
// test(x): four vectors of a thread in flight, a vector without such an entry is one comparison.
template <int DT, typename Test, typename See>
__device__ inline void sweep(const typename Elem<DT>::storage* row, int from, int to, Test&& test,
                             See&& see) {
  constexpr int VEC = Elem<DT>::kVec, kDeep = 4;
  const int tid = threadIdx.x;
  if (to - from < VEC) {
    for (int i = from + tid; i < to; i += kFThreads) {
      const float x = Elem<DT>::cvt(row[i]);
      if (test(x)) see(i, x);
    }
    return;
  }
  for (int64_t b = from; b < to; b += kDeep * kFThreads * VEC) {
    u32x4 q[kDeep];
    int64_t col[kDeep];
#pragma unroll
    for (int k = 0; k < kDeep; ++k) {
      col[k] = b + (int64_t)(k * kFThreads + tid) * VEC;
      q[k] = load_vec_any<DT>(row + min(col[k], (int64_t)to - VEC));
    }
#pragma unroll
    for (int k = 0; k < kDeep; ++k) {
      const int64_t at = min(col[k], (int64_t)to - VEC);  // moved back at the end
      bool any = false;
#pragma unroll
      for (int e = 0; e < VEC; ++e) any |= test(vec_elem<DT>(q[k], e));
      if (!any) continue;
#pragma unroll
      for (int e = 0; e < VEC; ++e)
        if (at + e >= col[k] && test(vec_elem<DT>(q[k], e))) see((int)(at + e), vec_elem<DT>(q[k], e));
    }
  }
}

// The C largest entries of beam w's row, by (value desc, token asc), into cand[at ..]; returns how
// many.  Fewer than C unions of the row's tops are above the C-th largest union, theta.  Where fewer
// than C entries are above theta (runs of one value: the case that comes here), they and the first
// entries equal to theta are the answer: one sweep over the row, and one that ends early.  Otherwise a
// radix selection of the C-th largest key, eight bits at a time, and those two sweeps again.
template <int DT>
__device__ inline int row_largest(const BeamScanParams& p, int64_t beam_row, int beam, BeamSmem& sm,
                                  int at) {
  using S = typename Elem<DT>::storage;
  const int tid = threadIdx.x, lane = lane_id(), wid = wave_id();
  constexpr uint32_t kNinf = 0x007fffffu;  // ordered_bits(-inf): not a candidate
  const S* row = static_cast<const S*>(p.logits) + sm.row[beam];
  const int V = p.V, C = p.C;
  float theta;
  {
    const int row_tops = p.nchunks * p.tops_per_chunk;
    const float* tops = p.tops + beam_row * row_tops;
    float own = -INFINITY;
    for (int i = tid; i < row_tops; i += kFThreads) own = fmaxf(own, tops[i]);
    sm.key[tid] = own;
    if (tid == 0) sm.count = 0;
    __syncthreads();
    theta = block_theta(own, C, sm);
  }
  auto keep = [&](int col, float x) {
    const int pos = atomicAdd(&sm.count, 1);
    if (pos < C) put(sm.cand, at + pos, {0.0, x, col, beam});
  };
  sweep<DT>(row, 0, V, [&](float x) { return x > theta; }, keep);
  __syncthreads();
  int found = sm.count;
  if (found < C) {
    if (theta == -INFINITY) return found;
  } else {
    theta = -INFINITY;  // to be found
  }
  if (theta == -INFINITY) {
    __syncthreads();
    uint32_t prefix = 0, mask = 0;
    int want = C;
    for (int shift = 24; shift >= 0; shift -= 8) {
      for (int i = tid; i < 256; i += kFThreads) sm.hist[i] = 0;
      __syncthreads();
      sweep<DT>(
          row, 0, V,
          [&](float x) {
            const uint32_t key = ordered_bits(x);
            return key > kNinf && (key & mask) == prefix;
          },
          [&](int, float x) { atomicAdd(&sm.hist[(ordered_bits(x) >> shift) & 255u], 1); });
      __syncthreads();
      if (tid == 0) {
        int above = 0, d = 255;  // at least C entries: every round finds its digit
        while (d > 0 && above + sm.hist[d] < want) above += sm.hist[d--];
        sm.digit = d;
        sm.above = above;
        sm.count = 0;
      }
      __syncthreads();
      want -= sm.above;
      prefix |= (uint32_t)sm.digit << shift;
      mask |= 255u << shift;
      __syncthreads();
    }
    theta = key_float(prefix);
    sweep<DT>(row, 0, V, [&](float x) { return x > theta; }, keep);
    __syncthreads();
    found = min(sm.count, C);
  }
  // as many entries equal to theta as are missing, from the first column
  const int block = 8 * kFThreads * Elem<DT>::kVec;
  for (int64_t b = 0; b < V && found < C; b += block) {
    const int end = (int)min(b + block, (int64_t)V);
    bool here = false;
    sweep<DT>(row, (int)b, end, [&](float x) { return x == theta; }, [&](int, float) { here = true; });
    if (!__syncthreads_or(here)) continue;
    for (int64_t i0 = b; i0 < end && found < C; i0 += kFThreads) {
      const int64_t i = i0 + tid;
      const float x = i < end ? Elem<DT>::cvt(row[i]) : NAN;
      const uint64_t hit = __ballot(x == theta);
      if (lane == 0) sm.wave_cnt[wid] = __popcll(hit);
      __syncthreads();
      int pos = found, total = 0;
      for (int w = 0; w < kFWaves; ++w) {
        pos += w < wid ? sm.wave_cnt[w] : 0;
        total += sm.wave_cnt[w];
      }
      pos += __popcll(hit & ((1ull << lane) - 1ull));
      if (x == theta && pos < C) put(sm.cand, at + pos, {0.0, x, (int)i, beam});
      found = min(found + total, C);
      __syncthreads();
    }
  }
  return found;
}

// The lse of a beam in 64 bits throughout, into sm.lse.  exp(d), d <= 0: with k = round(256 d / ln 2) and
// r = d - k ln 2 / 256 it is 2^(k / 256) exp(r), the first from a table of 256 and k's upper bits in the
// exponent, the second, |r| < 0.0014, its series up to r^4 (4e-17).  One compute unit's vector pipes
// bound it.
template <int DT>
__device__ inline void exact_lse(const BeamScanParams& p, int w, BeamSmem& sm) {
  using S = typename Elem<DT>::storage;
  constexpr double kStep = 0.69314718055994530942 / kPowers;
  constexpr int kDeep = 8;
  const int tid = threadIdx.x, V = p.V;
  const S* row = static_cast<const S*>(p.logits) + sm.row[w];
  const float most = sm.most[w];
  if (tid < kPowers) sm.power[tid] = exp2(tid / (double)kPowers);
  __syncthreads();
  double s = 0.0;
  auto add = [&](float x) {
    // (-600 for masks and -inf: nothing beside the sum, which is at least 1)
    const double d = fmax((double)x - (double)most, -600.0);
    const float n = rintf(fmaxf(x - most, -600.f) * (float)(1.0 / kStep));
    const double r = fma((double)n, -kStep, d);
    double e = fma(r, 1.0 / 24, 1.0 / 6);
    e = fma(e, r, 0.5);
    e = fma(e, r, 1.0);
    e = fma(e, r, 1.0);
    const int k = (int)n;
    const uint64_t power = __builtin_bit_cast(uint64_t, sm.power[k & (kPowers - 1)]);
    const uint32_t high = (uint32_t)(power >> 32) + ((uint32_t)(k & -kPowers) << (20 - kPowerBits));
    s = fma(e, __builtin_bit_cast(double, (uint64_t)high << 32 | (uint32_t)power), s);
  };
  const int whole = V / (kDeep * kFThreads) * (kDeep * kFThreads);
  for (int b = 0; b < whole; b += kDeep * kFThreads) {
    S x[kDeep];
#pragma unroll
    for (int k = 0; k < kDeep; ++k) x[k] = row[b + k * kFThreads + tid];
#pragma unroll
    for (int k = 0; k < kDeep; ++k) add(Elem<DT>::cvt(x[k]));
  }
  for (int i = whole + tid; i < V; i += kFThreads) add(Elem<DT>::cvt(row[i]));
  s = lanes_sum(s, kWave);
  if (lane_id() == 0) sm.red[wave_id()] = s;
  __syncthreads();
  if (tid == 0) {
    double all = 0.0;
    for (int k = 0; k < kFWaves; ++k) all += sm.red[k];
    sm.lse[w] = (double)most + log(all);
  }
  __syncthreads();
}

// How close two totals of different beams have to be for the scan's lse not to decide: twice the most
// that an lse is off by, 9.1e-7, whatever the row's type and length.  Every wave sums its 2048 columns (512
// in short chunks) below their own maximum, and the waves' sums are joined in 64 bits, so the worst
// relative error of a wave's sum is that of the row's.  An exponential at distance D below the maximum is
// off by the power's own rounding (2^-23), its argument's (D < 5.54: ln 2 2^-22, < 11.1: ln 2 2^-21, and so
// on) and, unless the values' exponents are near each other, the distance's (D < 8: 2^-22, < 16: 2^-21);
// all of them together have at most 2047 e^-D / (1 + 2047 e^-D) of the sum.  The product is largest at
// D = 5.55: 6.9e-7 of 0.89.  Five roundings of partial sums add 3.0e-7.  (The worst of waves searched for
// it: 5.8e-7; rows drawn at random: 1e-8.)
// Totals past 2^30 add their own rounding; past kFar it hides any lse's.
constexpr double kNear = 0x1p-19, kFar = 0x1p44;

__device__ inline double near_by(double total) { return kNear + fabs(total) * 0x1p-51; }

// Of the `found` gathered candidates, the first C in sm.best: where two neighbours of different beams
// are closer than kNear, or several beams have candidates so close to the last place, in it or behind
// it, the lse of those beams is formed again, in 64 bits throughout, and true returned: the totals have
// to be formed and ranked again.  A row of 151936 entries takes 22 us more; a group of 8 beams and 16
// candidates has such a pair about once in 2500.
template <int DT>
__device__ inline bool settle_near_ties(const BeamScanParams& p, int found, BeamSmem& sm) {
  const int tid = threadIdx.x, have = min(found, p.C);
  if (tid == 0) sm.near_ties = sm.edge = 0;
  __syncthreads();
  if (tid + 1 < have) {
    const int a = sm.best.beam[tid], b = sm.best.beam[tid + 1];
    const double t = sm.best.total[tid];
    if (a != b && fabs(t) < kFar && t - sm.best.total[tid + 1] < near_by(t))
      atomicOr((unsigned long long*)&sm.near_ties, 1ull << a | 1ull << b);
  }
  if (found > have) {
    const double last = sm.best.total[have - 1];
    if (fabs(last) < kFar)
      for (int i = tid; i < found; i += kFThreads)
        if (fabs(sm.cand.total[i] - last) < near_by(last))
          atomicOr((unsigned long long*)&sm.edge, 1ull << sm.cand.beam[i]);
  }
  __syncthreads();
  const uint64_t beams = sm.near_ties | (__popcll(sm.edge) > 1 ? sm.edge : 0);
  for (uint64_t left = beams; left != 0; left &= left - 1)
    exact_lse<DT>(p, __ffsll((long long)left) - 1, sm);
  return beams != 0;
}

// The group's candidates, in order, in sm.best; returns how many.
template <int DT, int NV, int LANES>
__device__ inline int group_candidates(const BeamScanParams& p, int g, BeamSmem& sm) {
  using S = typename Elem<DT>::storage;
  constexpr int VEC = Elem<DT>::kVec;
  constexpr int CH = NV * kThreads * VEC;
  constexpr int kTops = kThreads / LANES;
  const int tid = threadIdx.x, lane = lane_id(), wid = wave_id();
  const int W = p.W, C = p.C, nch = p.nchunks;
  const int64_t first = (int64_t)g * W;
  // ---- what the scan left: every load is issued before the first is waited for, so indices are
  //      clamped instead of branched on.  A beam that was not scanned has whatever is there. ----
  // tops: four of one chunk at a time, the first ones stay in registers
  const int per_row = nch * (kTops / 4), quads = W * per_row;
  const float4* top4 = reinterpret_cast<const float4*>(p.tops + first * nch * kTops);
  float4 held[kHeld];
#pragma unroll
  for (int k = 0; k < kHeld; ++k) held[k] = top4[min(tid + k * kFThreads, quads - 1)];
  // log-sums: as many lanes per beam as there are, a power of two from 8 to 64
  const int lanes = max(8, min(kWave, 1 << (31 - __clz(kFThreads / W))));
  const int lse_w = tid / lanes, l = tid & (lanes - 1);
  const BeamScanParams::Stat* st = p.stats + (first + min(lse_w, W - 1)) * nch;
  BeamScanParams::Stat v[kStats];
#pragma unroll
  for (int k = 0; k < kStats; ++k) v[k] = st[min(l + k * lanes, nch - 1)];
  const float score = p.scores[first + min(lse_w, W - 1)];
  int64_t row = first + min(tid, W - 1);
  if (p.rows) row = min(max((int64_t)p.rows[row], (int64_t)0), p.num_rows - 1);
  if (tid < W) sm.row[tid] = row * p.stride;
  int held_row[kHeld];
#pragma unroll
  for (int k = 0; k < kHeld; ++k) {
    const int i = tid + k * kFThreads;
    held_row[k] = i < quads ? i / per_row : -1;
  }
  // ---- lse of every beam ----
  {
    const int w = lse_w;
    float M = -INFINITY;
#pragma unroll
    for (int k = 0; k < kStats; ++k) {
      if (w >= W || l + k * lanes >= nch) v[k] = {0.0, -INFINITY};
      M = fmaxf(M, v[k].max);
    }
    if (w < W)
      for (int c = l + kStats * lanes; c < nch; c += lanes) M = fmaxf(M, st[c].max);
    const float all = lanes_max(M, lanes);
    // a chunk of -inf alone adds its sum, 0 (NaN where it holds a NaN)
    auto term = [&](const BeamScanParams::Stat& t) {
      return t.max == -INFINITY ? t.sum : t.sum * exp((double)t.max - (double)all);
    };
    double s = 0.0;
#pragma unroll
    for (int k = 0; k < kStats; ++k) s += term(v[k]);
    if (w < W)
      for (int c = l + kStats * lanes; c < nch; c += lanes) s += term(st[c]);
    s = lanes_sum(s, lanes);
    if (w < W && l == 0) {
      const double lse = (double)all + log(s);
      const bool live = finite(score) && fabs(lse) < (double)INFINITY;
      sm.lse[w] = live ? lse : 0.0;
      sm.score[w] = live ? score : -INFINITY;
      sm.most[w] = all;
    }
  }
  if (tid < kWave) sm.above_key[tid] = 0;
  if (tid == 0) sm.listed = sm.count = 0;
  __syncthreads();
  // ---- theta: the C-th largest of the 512 threads' keys, or of 64 maxima of eight of them: fewer
  //      than C keys are above it, and it is the least such key ----
  // (what is left of a beam that proposes nothing: whatever plus -inf, -inf or NaN)
  auto total_of = [&](float x, int w) {
    return (float)((double)sm.score[w] + ((double)x - sm.lse[w]));
  };
  float theta;
  const int live = __popcll(__ballot(lane < W && sm.score[min(lane, W - 1)] != -INFINITY));
  if (live * per_row < 2 * C) {  // block-uniform
    // few vectors of tops (the first step's one beam, short rows): unions of single tops
    uint32_t* bits = reinterpret_cast<uint32_t*>(sm.key);
    bits[tid] = 0;
    __syncthreads();
    for (int i = tid; i < quads; i += kFThreads) {
      const float4 v = top4[i];
      const float e[4] = {v.x, v.y, v.z, v.w};
      const int w = i / per_row;
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const float t = total_of(e[k], w);
        if (t > -INFINITY) atomicMax(&bits[(4 * i + k) % kFThreads], ordered_bits(t));
      }
    }
    __syncthreads();
    const float own = bits[tid] == 0 ? -INFINITY : key_float(bits[tid]);
    sm.key[tid] = own;
    __syncthreads();
    theta = block_theta(own, C, sm);
  } else {
    float own = -INFINITY;
#pragma unroll
    for (int k = 0; k < kHeld; ++k)
      if (held_row[k] >= 0) {
        const float4 v = held[k];
        own = fmaxf(own, total_of(fmaxf(fmaxf(v.x, v.y), fmaxf(v.z, v.w)), held_row[k]));
      }
    for (int i = tid + kHeld * kFThreads; i < quads; i += kFThreads) {
      const float4 v = top4[i];
      own = fmaxf(own, total_of(fmaxf(fmaxf(v.x, v.y), fmaxf(v.z, v.w)), i / per_row));
    }
    sm.key[tid] = own;
    __syncthreads();
    if (C <= kFoldC) {  // block-uniform
      // every wave folds the keys, counts an eighth of the comparisons and reads the sums
#pragma unroll
      for (int k = 1; k < kFWaves; ++k) own = fmaxf(own, sm.key[((wid + k) % kFWaves) * kWave + lane]);
      int above = 0;
#pragma unroll
      for (int j = 0; j < kWave / kFWaves; ++j)
        above += readlane_f32(own, wid * (kWave / kFWaves) + j) > own;
      atomicAdd(&sm.above_key[lane], above);
      __syncthreads();
      theta = -wave_max(sm.above_key[lane] < C ? -own : -INFINITY);
    } else {
      theta = block_theta(own, C, sm);
    }
  }
  // ---- the least logit of each beam that can reach theta, rounded down: lane w's of every wave ----
  float floor_w = INFINITY;
  if (lane < W && sm.score[lane] != -INFINITY) {
    floor_w = -3.402823466e38f;  // -inf is no candidate
    if (theta != -INFINITY) {
      // a rounded total at or above theta stands for one of at least theta - |theta| 2^-24
      // (and the scan's lse for one near by)
      const double t = (double)theta - fabs((double)theta) * 0x1p-23 - kNear;
      floor_w = fmaxf(floor_w, __double2float_rd(t - (double)sm.score[lane] + sm.lse[lane]));
    }
  }
  if (tid < W) sm.floor[tid] = floor_w;
  auto list = [&](const float4& v, int i, int w, float f) {
    const float e[4] = {v.x, v.y, v.z, v.w};
    if (!(fmaxf(fmaxf(v.x, v.y), fmaxf(v.z, v.w)) >= f) || f == INFINITY) return;
#pragma unroll
    for (int k = 0; k < 4; ++k)
      if (e[k] >= f) {
        const int pos = atomicAdd(&sm.listed, 1);
        if (pos < kListCap) sm.list[pos] = make_int2(w, (i - w * per_row) * 4 + k);
      }
  };
#pragma unroll
  for (int k = 0; k < kHeld; ++k) {
    const float f = __shfl(floor_w, max(held_row[k], 0), kWave);
    if (held_row[k] >= 0) list(held[k], tid + k * kFThreads, held_row[k], f);
  }
  for (int i0 = kHeld * kFThreads; i0 < quads; i0 += kFThreads) {
    const int i = i0 + tid, w = min(i, quads - 1) / per_row;
    const float f = __shfl(floor_w, w, kWave);
    if (i < quads) list(top4[i], i, w, f);
  }
  __syncthreads();
  const int listed = sm.listed;
  int found = 0;
  if (listed <= kListCap) {
    const S* x0 = static_cast<const S*>(p.logits);
    if (p.V < VEC) {  // uniform: rows shorter than a vector
      for (int i = tid; i < W * p.V; i += kFThreads) {
        const int w = i / p.V, col = i - w * p.V;
        if (sm.floor[w] == INFINITY) continue;  // proposes nothing, whatever its row holds
        const float x = Elem<DT>::cvt(x0[sm.row[w] + col]);
        if (x >= sm.floor[w]) {
          const int pos = atomicAdd(&sm.count, 1);
          if (pos < kCandCap) put(sm.cand, pos, {0.0, x, col, w});
        }
      }
    } else {
      // ---- the entries under the listed tops, LANES lanes each, two tops at a time ----
      constexpr int kTeams = kFThreads / LANES;
      for (int b = tid / LANES; b < listed; b += 2 * kTeams) {
        u32x4 q[2][NV];
        int64_t col0[2];
        int row_of[2];
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          const int2 i = sm.list[min(b + k * kTeams, listed - 1)];
          const int w = i.x, c = i.y / kTops;
          row_of[k] = w;
          col0[k] = (int64_t)c * CH + ((i.y % kTops) * LANES + tid % LANES) * VEC;
          const S* row = x0 + sm.row[w];
          // as load_vec_inside: the vector is moved back where it would pass the row's end
#pragma unroll
          for (int j = 0; j < NV; ++j)
            q[k][j] = load_vec_any<DT>(row + min(col0[k] + j * kThreads * VEC, (int64_t)p.V - VEC));
        }
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          if (b + k * kTeams >= listed) continue;
          // the lane's entries that reach the floor, a bit each; one or two of a top's lanes have any
          const int w = row_of[k];
          const float f = sm.floor[w];
          const int64_t end = (int64_t)p.V - VEC;
          uint32_t mask = 0;
#pragma unroll
          for (int j = 0; j < NV; ++j)
#pragma unroll
            for (int e = 0; e < VEC; ++e)
              mask |= vec_elem<DT>(q[k][j], e) >= f ? 1u << (j * VEC + e) : 0u;
          if (mask == 0) continue;
          if (col0[k] + (NV - 1) * kThreads * VEC > end) {
            // vectors that were moved back: not what is in front of their own columns
#pragma unroll
            for (int j = 0; j < NV; ++j) {
              const int64_t over = min(max(col0[k] + j * kThreads * VEC - end, (int64_t)0),
                                       (int64_t)VEC);
              mask &= ~(((1u << over) - 1u) << (j * VEC));
            }
          }
          int pos = atomicAdd(&sm.count, __popc(mask));
          const S* row = x0 + sm.row[w];
          for (; mask != 0; mask &= mask - 1u, ++pos) {
            const int bit = __ffs(mask) - 1;
            const int64_t at = min(col0[k] + (bit / VEC) * kThreads * VEC, end) + bit % VEC;
            if (pos < kCandCap)
              put(sm.cand, pos, {0.0, Elem<DT>::cvt(row[at]), (int)at, w});
          }
        }
      }
    }
    __syncthreads();
    found = sm.count;
  }
  if (listed <= kListCap && found <= kCandCap) {
    int settled = 0;
    do {
      for (int i = tid; i < found; i += kFThreads)
        sm.cand.total[i] = (double)sm.score[sm.cand.beam[i]] +
                           ((double)sm.cand.x[i] - sm.lse[sm.cand.beam[i]]);
      __syncthreads();
      // ranked by counting, eight threads to a candidate
      for (int i0 = 0; i0 < found; i0 += kFThreads / 8) {
        const int i = i0 + tid / 8;
        const Candidate mine = get(sm.cand, min(i, found - 1));
        int rank = 0, equal = 0;
  #pragma unroll 4
        for (int j = tid & 7; j < found; j += 8) {
          const double t = sm.cand.total[j];
          rank += t > mine.total;
          equal += t == mine.total;
        }
        if (equal > ((i & 7) == (tid & 7))) {  // others than itself
          rank = 0;
          for (int j = tid & 7; j < found; j += 8) rank += before(sm.cand, j, mine);
        }
        rank += dpp_i32<kDppXor1>(rank);
        rank += dpp_i32<kDppXor2>(rank);
        rank += dpp_i32<kDppHalfMirror>(rank);
        if (i < found && rank < C && (tid & 7) == 0) put(sm.best, rank, mine);
      }
      __syncthreads();
    } while (!settled++ && settle_near_ties<DT>(p, found, sm));
    return min(found, C);
  }
  // ---- too many: the beams one after the other, by their lse in 64 bits where it can matter for the
  //      last place; once more where candidates in front of it are near ties ----
  const bool exact = W > 1 && (fabsf(theta) < (float)kFar || theta == -INFINITY);
  if (exact)
    for (int w = 0; w < W; ++w)
      if (sm.floor[w] < INFINITY) exact_lse<DT>(p, w, sm);
  int settled = 0;
  do {
    found = 0;
    for (int w = 0; w < W; ++w) {
      __syncthreads();
      if (sm.floor[w] == INFINITY) continue;
      const int got = row_largest<DT>(p, first + w, w, sm, 0);
      __syncthreads();
      // the best so far and the beam's own: at most 2 C = 512, one a thread
      Candidate mine;
      const bool have = tid < found + got;
      if (have) {
        mine = tid < found ? get(sm.best, tid) : get(sm.cand, tid - found);
        if (tid >= found) mine.total = (double)sm.score[w] + ((double)mine.x - sm.lse[w]);
      }
      __syncthreads();
      if (have) put(sm.cand, tid, mine);
      __syncthreads();
      int rank = 0;
      if (have)
        for (int j = 0; j < found + got; ++j) rank += before(sm.cand, j, mine);
      if (have && rank < C) put(sm.best, rank, mine);
      found = min(found + got, C);
    }
    __syncthreads();
  } while (!exact && !settled++ && settle_near_ties<DT>(p, found, sm));
  return found;
}

template <int DT, int NV, int LANES>
__global__ __launch_bounds__(kFThreads) void beam_select_kernel(BeamScanParams p,
                                                                 BeamSelectOut o) {
  __shared__ BeamSmem sm;
  const int g = blockIdx.x;
  const int found = group_candidates<DT, NV, LANES>(p, g, sm);
  for (int i = threadIdx.x; i < p.C; i += kFThreads) {
    const int64_t at = (int64_t)g * p.C + i;
    const bool on = i < found;
    o.token_ids[at] = on ? sm.best.token[i] : -1;
    o.parents[at] = on ? sm.best.beam[i] : -1;
    o.scores[at] = on ? candidate_score(sm.best.total[i]) : -INFINITY;
  }
}

// ------------------------------------------------------------------ step -------------
// Candidates in order; those of rank below W that are stop tokens end a hypothesis of
// length + 1 tokens with the normalised score fl32(fl32(total) / (length + 1)^alpha); the first W
// that are no stop tokens are the next beams.  W (1 + E) candidates always hold W of the latter if
// there are as many.  Finished hypotheses: the W best of the old and the new ones, the old first
// where they are equal.
template <int DT, int NV, int LANES>
__global__ __launch_bounds__(kFThreads) void beam_step_kernel(BeamScanParams p,
                                                               mvsd_beam_step_args a) {
  __shared__ BeamSmem sm;
  const int g = blockIdx.x, tid = threadIdx.x, lane = lane_id(), wid = wave_id();
  const int W = p.W;
  const int64_t first = (int64_t)g * W, at = first + min(tid, W - 1);
  // the state, before anything is written (outputs may be inputs) and while the scan's results arrive
  const int len = p.lengths[g];
  const uint8_t was = a.done[g];
  float hyp = a.finished_scores[at];
  int hyp_beam = a.finished_beams[at], hyp_token = a.finished_token_ids[at];
  int hyp_len = a.finished_lengths[at];
  const float old_score = a.scores[at];
  const int E = (int)a.num_stop_ids;
  if (tid < E) sm.stop[tid] = a.stop_token_ids[tid];
  if (was != 0 || len < 0 || len >= p.max_length) {  // the group rests (block-uniform)
    if (tid < W) {
      a.token_ids[first + tid] = -1;
      a.parents[first + tid] = -1;
      a.out_scores[first + tid] = old_score;
      a.out_finished_scores[first + tid] = hyp;
      a.out_finished_beams[first + tid] = hyp_beam;
      a.out_finished_token_ids[first + tid] = hyp_token;
      a.out_finished_lengths[first + tid] = hyp_len;
    }
    if (tid == 0) {
      a.out_lengths[g] = len;
      a.out_done[g] = was;
    }
    return;
  }
  const int found = group_candidates<DT, NV, LANES>(p, g, sm);
  const int new_len = len + 1;
  const double power = len_power(new_len, a.length_penalty);
  if (wid < kMaxCandidates / kWave) {
    bool stop = false;
    if (tid < found) {
      const int token = sm.best.token[tid];
      for (int e = 0; e < E; ++e) stop |= token == sm.stop[e];
    }
    const uint64_t sb = __ballot(stop), ob = __ballot(tid < found && !stop);
    if (lane == 0) {
      sm.stop_mask[wid] = sb;
      sm.on_mask[wid] = ob;
    }
  }
  if (tid >= W || !(hyp > -INFINITY)) {
    hyp = -INFINITY;
    hyp_beam = hyp_token = -1;
    hyp_len = 0;
  }
  __syncthreads();
  // ---- next beams ----
  int going = 0;
  for (int k = 0; k < kMaxCandidates / kWave; ++k) going += __popcll(sm.on_mask[k]);
  going = min(going, W);
  float next_best = -INFINITY;
  {
    // the first candidate that goes on is the best running beam
    for (int k = kMaxCandidates / kWave - 1; k >= 0; --k)
      if (sm.on_mask[k])
        next_best =
            candidate_score(sm.best.total[k * kWave + __ffsll((long long)sm.on_mask[k]) - 1]);
  }
  const int64_t hist = ((int64_t)g * a.max_length + len) * W;
  auto put = [&](int w, float score, int token, int parent) {
    a.out_scores[first + w] = score;
    a.token_ids[first + w] = token;
    a.parents[first + w] = parent;
    a.token_history[hist + w] = token;
    a.parent_history[hist + w] = parent;
  };
  if (wid < kMaxCandidates / kWave && ((sm.on_mask[wid] >> lane) & 1)) {
    int place = __popcll(sm.on_mask[wid] & ((1ull << lane) - 1ull));
    for (int k = 0; k < wid; ++k) place += __popcll(sm.on_mask[k]);
    if (place < W)
      put(place, candidate_score(sm.best.total[tid]), sm.best.token[tid], sm.best.beam[tid]);
  }
  if (tid >= going && tid < W) put(tid, -INFINITY, -1, -1);
  // ---- finished hypotheses: entries [0, W) are the old ones, [W, 2 W) the candidates of rank < W ----
  if (tid >= W && tid < 2 * W) {
    const int r = tid - W;
    if (r < found && ((sm.stop_mask[r / kWave] >> (r % kWave)) & 1)) {
      hyp = hypothesis_score(candidate_score(sm.best.total[r]), power);
      hyp_beam = sm.best.beam[r];
      hyp_token = sm.best.token[r];
      hyp_len = new_len;
    }
  }
  if (tid < 2 * W) sm.pool[tid] = hyp;
  __syncthreads();
  if (tid < 2 * W) {
    int rank = 0;
    for (int j = 0; j < 2 * W; ++j) {
      const float o = sm.pool[j];
      rank += o > hyp || (o == hyp && j < tid);
    }
    if (rank < W) {
      const bool any = hyp > -INFINITY;
      a.out_finished_scores[first + rank] = hyp;
      a.out_finished_beams[first + rank] = any ? hyp_beam : -1;
      a.out_finished_token_ids[first + rank] = any ? hyp_token : -1;
      a.out_finished_lengths[first + rank] = any ? hyp_len : 0;
      if (rank == W - 1) sm.worst = hyp;  // the worst one kept
    }
  }
  __syncthreads();
  if (tid == 0) {
    const float worst = sm.worst;
    const bool full = worst > -INFINITY;
    const float reach = hypothesis_score(next_best, power);
    const bool over = going == 0 || (full && (a.early_stopping || worst >= reach));
    a.out_lengths[g] = new_len;
    a.out_done[g] = over ? 1 : 0;
  }
}

// ------------------------------------------------------------------ launches ---------

int64_t beam_workspace_bytes(int64_t G, int64_t W, int64_t V, int64_t C) {
  if (G <= 0 || W <= 0 || V <= 0) return 0;
  const BeamSplit split = beam_split(G * W, V, C);
  const int64_t slots = G * W * split.chunks;
  if (slots >= (1ll << 24)) return 0;  // the scan's threads stay below 2^32
  return slots * (int64_t)(sizeof(BeamScanParams::Stat) + split.tops() * sizeof(float));
}

template <int DT, int NV, int LANES, bool STREAM>
static void launch_split(const BeamScanParams& p, const BeamSelectOut* o,
                         const mvsd_beam_step_args* a, hipStream_t stream) {
  hipLaunchKernelGGL((beam_scan_kernel<DT, NV, LANES, STREAM>),
                     dim3((unsigned)(p.G * p.W) * (unsigned)p.nchunks), dim3(kThreads), 0, stream, p);
  const dim3 groups(p.G), block(kFThreads);
  if (o) hipLaunchKernelGGL((beam_select_kernel<DT, NV, LANES>), groups, block, 0, stream, p, *o);
  else hipLaunchKernelGGL((beam_step_kernel<DT, NV, LANES>), groups, block, 0, stream, p, *a);
}

template <int DT>
static void launch_dt(const BeamScanParams& p, const BeamSelectOut* o,
                      const mvsd_beam_step_args* a, const BeamSplit& split, hipStream_t stream) {
  constexpr int kLong = kBeamLong / (kThreads * Elem<DT>::kVec);
  constexpr int kShort = kBeamShort / (kThreads * Elem<DT>::kVec);
  const int64_t bytes = (int64_t)p.G * p.W * p.V * (int64_t)sizeof(typename Elem<DT>::storage);
  if (split.chunk == kBeamLong && bytes >= kStreamBytes)
    launch_split<DT, kLong, kCoarse, true>(p, o, a, stream);
  else if (split.chunk == kBeamLong)
    launch_split<DT, kLong, kCoarse, false>(p, o, a, stream);
  else if (split.lanes == kCoarse)
    launch_split<DT, kShort, kCoarse, false>(p, o, a, stream);
  else
    launch_split<DT, kShort, kFine, false>(p, o, a, stream);
}

static hipError_t launch(BeamScanParams p, const BeamSelectOut* o, const mvsd_beam_step_args* a,
                         int dtype, void* workspace, hipStream_t stream) {
  const int64_t rows = (int64_t)p.G * p.W;
  const BeamSplit split = beam_split(rows, p.V, p.C);
  p.nchunks = (int)split.chunks;
  p.tops_per_chunk = split.tops();
  p.tops = static_cast<float*>(workspace);
  p.stats = reinterpret_cast<BeamScanParams::Stat*>(p.tops + rows * split.chunks * split.tops());
  switch (dtype) {
    case MVSD_F32: launch_dt<MVSD_F32>(p, o, a, split, stream); break;
    case MVSD_BF16: launch_dt<MVSD_BF16>(p, o, a, split, stream); break;
    case MVSD_F16: launch_dt<MVSD_F16>(p, o, a, split, stream); break;
    default: return hipErrorInvalidValue;
  }
  return hipGetLastError();
}

hipError_t launch_beam_select(BeamScanParams p, const BeamSelectOut& out, int dtype,
                              void* workspace, hipStream_t stream) {
  return launch(p, &out, nullptr, dtype, workspace, stream);
}

hipError_t launch_beam_step(BeamScanParams p, const mvsd_beam_step_args& a, void* workspace,
                            hipStream_t stream) {
  return launch(p, nullptr, &a, a.dtype, workspace, stream);
}

}  // namespace mvsd
