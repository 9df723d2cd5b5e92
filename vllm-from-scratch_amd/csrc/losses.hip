// Training losses on rows of logits and their gradients: log-probabilities of given tokens, distillation
// from a teacher's top tokens, a clipped policy loss, a preference loss over pairs of answers
// (mvsd_row_loss, mvsd_loss_gradient in include/mvsd.h; the reference has none of them).
//
// Mathematics.  Every one of them needs of a row x, p = softmax(x / T), only
//   * "the rest", the tokens that are not given ones: their maximum M, s = sum e_j, e_j = 2^((x_j - M) c1),
//     c1 = log2(e) / T, and for an entropy t = sum e_j log2 e_j;
//   * the given tokens' logits.
// The rest is summed without the given tokens, so that 1 - p of a confident token and the mass of a
// distillation's tail are sums of positive terms and no differences.  With the log-odds against a token
// l = ln s + (M - x_t) / T its log-probability is -log(1 + e^l).  Every gradient is, at the rest,
// e_j (a + b log2 e_j) with two numbers of the row, and a value of its own at each given token.
//
// Statistics and sums are fp32: a lane adds up to 1024 terms of a chunk (594 of 151936 columns), in one pass up to
// 144 that it holds and a 1024th of the columns behind, then trees.  The gradient is rounded once, to the logits' dtype.
//
// All of it is bound by memory: a logit is 2 or 4 bytes for two exponentials at most and some 16 vector
// instructions.  Two ways through:
//   * split: the statistics of (row, chunk) by workgroups of their own, then the rows' or pairs' values, and in
//     the backward pass the gradient from a record of 32 bytes a row.  Reads a row twice, works for any upstream;
//   * one pass (loss_rows_kernel), where the loss is a scalar whose rows do not wait for each other: a row stays
//     in registers until its gradient for an upstream of 1 is written.  Reads a row once.
// Times below are medians of a kernel trace on one MI355X, whose large copies reach 5.25 TB/s.
#include <float.h>

#include <algorithm>
#include <atomic>
#include <cmath>

#include "losses.h"
#include "mvsd_device.h"

namespace mvsd {

int record_hip_error(hipError_t err);  // capi.hip: keeps err for mvsd_last_hip_error()

namespace {

constexpr float kLn2 = 0.69314718055994531f;
constexpr int kLossThreads = 256;
constexpr float kLeast = -16384.f;  // below every exponent whose power is not 0: no 0 * -inf in e log2 e

// ------------------------------------------------------------------ a row's place and tokens ----

template <int DT>
__device__ inline const typename Elem<DT>::storage* logits_row(const mvsd_loss_args& a, int64_t row) {
  const int64_t outer = row / a.inner_rows;
  return static_cast<const typename Elem<DT>::storage*>(a.logits) + outer * a.outer_stride +
         (row - outer * a.inner_rows) * a.stride;
}

// Token id i, V for every one of V or more, -1 for every one below 0.  Its two halves are loaded (one word
// twice of an int32), so that several ids' loads need no branch between them.
__device__ inline int token_at(const mvsd_loss_args& a, int64_t i, int V) {
  const int words = a.ids_dtype == MVSD_I64 ? 2 : 1;
  const int32_t* id = static_cast<const int32_t*>(a.token_ids) + i * words;
  const int low = id[0], high = id[words - 1];
  return high < 0 ? -1 : (words == 2 && high > 0) || (uint32_t)low >= (uint32_t)V ? V : low;
}

// A row's weight before the mean's division (a preference's weights are its pairs').
__device__ inline float row_weight(const mvsd_loss_args& a, int64_t row) {
  return a.weights && a.kind != MVSD_LOSS_PREFERENCE ? a.weights[row] : 1.f;
}

// The log-odds' reference: -inf (nothing but masked tokens) gives sums of 0.
__device__ inline float base_of(float m) { return m == -INFINITY ? 0.f : m; }

// ------------------------------------------------------------------ statistics of the rest ------

struct Stat {
  float m, s, t;
};

// Both parts' sums against their common maximum.
__device__ inline Stat join(Stat a, Stat b, float c1) {
  const float m = fmaxf(a.m, b.m);
  const float base = base_of(m);
  const float da = fmaxf((a.m - base) * c1, kLeast), db = fmaxf((b.m - base) * c1, kLeast);
  const float fa = __builtin_amdgcn_exp2f(da), fb = __builtin_amdgcn_exp2f(db);
  return {m, a.s * fa + b.s * fb, (a.t + a.s * da) * fa + (b.t + b.s * db) * fb};
}

template <int CTRL>
__device__ inline Stat dpp_stat(Stat v) {
  return {dpp_f32<CTRL>(v.m), dpp_f32<CTRL>(v.s), dpp_f32<CTRL>(v.t)};
}
__device__ inline Stat readlane_stat(Stat v, int lane) {
  return {readlane_f32(v.m, lane), readlane_f32(v.s, lane), readlane_f32(v.t, lane)};
}
__device__ inline Stat wave_join(Stat v, float c1) {
  v = join(v, dpp_stat<kDppXor1>(v), c1);
  v = join(v, dpp_stat<kDppXor2>(v), c1);
  v = join(v, dpp_stat<kDppHalfMirror>(v), c1);
  v = join(v, dpp_stat<kDppMirror>(v), c1);
  return join(join(readlane_stat(v, 0), readlane_stat(v, 16), c1),
              join(readlane_stat(v, 32), readlane_stat(v, 48), c1), c1);
}

// The vector of columns [col, col + VEC), -inf behind `end`.
template <int DT>
__device__ inline void load_filled(const typename Elem<DT>::storage* row, int col, int end,
                                   float (&x)[Elem<DT>::kVec]) {
  constexpr int VEC = Elem<DT>::kVec;
  if (col + VEC <= end) {
    const u32x4 raw = load_vec_any<DT>(row + col);
#pragma unroll
    for (int e = 0; e < VEC; ++e) x[e] = vec_elem<DT>(raw, e);
  } else {
#pragma unroll
    for (int e = 0; e < VEC; ++e) x[e] = col + e < end ? Elem<DT>::cvt(row[col + e]) : -INFINITY;
  }
}

// Marks of the given tokens among a chunk's columns, a bit each.
__device__ inline unsigned marks_at(const uint32_t* bits, unsigned col, int n) {  // n divides 32, col is its multiple
  return (bits[col >> 5] >> (col & 31)) & ((1u << n) - 1u);
}

// The elements of `marks` become -inf.
template <int DT>
__device__ inline void mask_vec(u32x4& r, unsigned marks) {
  if constexpr (DT == MVSD_F32) {
#pragma unroll
    for (int e = 0; e < 4; ++e) r[e] = marks >> e & 1 ? 0xff800000u : r[e];
  } else {
    constexpr uint32_t ninf = DT == MVSD_BF16 ? 0xff80u : 0xfc00u;
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      r[w] = marks >> (2 * w) & 1 ? (r[w] & 0xffff0000u) | ninf : r[w];
      r[w] = marks >> (2 * w + 1) & 1 ? (r[w] & 0x0000ffffu) | ninf << 16 : r[w];
    }
  }
}

// vec_elem, by instructions of its own: the compiler would keep what the statistics converted until the
// gradient converts it again, and a row would take twice the registers.
template <int DT>
__device__ inline float vec_elem_again(const u32x4& r, int j) {
  if constexpr (DT == MVSD_F32) {
    return __uint_as_float(r[j]);
  } else {
    float v;
    const uint32_t w = r[j / 2];
    if (DT == MVSD_BF16 && j % 2 == 0)
      asm("v_lshlrev_b32 %0, 16, %1" : "=v"(v) : "v"(w));
    else if (DT == MVSD_BF16)
      asm("v_and_b32 %0, 0xffff0000, %1" : "=v"(v) : "v"(w));
    else if (j % 2 == 0)
      asm("v_cvt_f32_f16 %0, %1" : "=v"(v) : "v"(w));
    else
      asm("v_cvt_f32_f16_sdwa %0, %1 dst_sel:DWORD dst_unused:UNUSED_PAD src0_sel:WORD_1" : "=v"(v) : "v"(w));
    return v;
  }
}

// Adds values to a thread's statistics.
template <bool ENT, int N>
__device__ inline void add_values(Stat& st, const float (&v)[N], float c1) {
  float m = st.m;
#pragma unroll
  for (int e = 0; e < N; ++e) m = fmaxf(m, v[e]);
  const float base = base_of(m);
  const float d = fmaxf((st.m - base) * c1, kLeast), f = __builtin_amdgcn_exp2f(d);
  if constexpr (ENT) st.t = fmaf(st.s, d, st.t) * f;
  st.s *= f;
  st.m = m;
#pragma unroll
  for (int e = 0; e < N; ++e) {
    const float y = (v[e] - base) * c1, w = __builtin_amdgcn_exp2f(y);
    st.s += w;
    if constexpr (ENT) st.t = fmaf(w, fmaxf(y, kLeast), st.t);
  }
}
template <int DT, bool ENT, int N>
__device__ inline void add_vecs(Stat& st, const u32x4 (&r)[N], float c1) {
  constexpr int VEC = Elem<DT>::kVec;
  float v[N * VEC];
#pragma unroll
  for (int i = 0; i < N * VEC; ++i) v[i] = vec_elem<DT>(r[i / VEC], i % VEC);
  add_values<ENT, N * VEC>(st, v, c1);
}

// Both sums against a new maximum.
__device__ inline void rebase(Stat& st, float m, float c1) {
  const float d = fmaxf((st.m - base_of(m)) * c1, kLeast), f = __builtin_amdgcn_exp2f(d);
  st.t = fmaf(st.s, d, st.t) * f;
  st.s *= f;
  st.m = m;
}

// ------------------------------------------------------------------ the loss of all rows --------

// counters[0]: rows that loss_rows_kernel's workgroups have taken behind their first; [1]: workgroups whose rows
// have their losses.  An earlier launch of the call clears them.
__device__ inline void clear_counters(const LossParams& p) {
  if (threadIdx.x < 2) p.counters[threadIdx.x] = 0;
}

// loss[0] = the sum of n row losses, by a workgroup, in one order.
__device__ inline void sum_losses(const LossParams& p, int64_t n) {
  __shared__ float s_sum[16];
  float sum = 0.f;
  for (int64_t i = threadIdx.x; i < n; i += blockDim.x) sum += p.row_loss[i];
  sum = wave_sum(sum);
  if (lane_id() == 0) s_sum[wave_id()] = sum;
  __syncthreads();
  if (threadIdx.x == 0) {
    sum = 0.f;
    for (int w = 0; w < (int)blockDim.x / kWave; ++w) sum += s_sum[w];
    p.a.loss[0] = sum;
  }
}

// The same by the last of a launch's workgroups, each of which comes here once, behind its rows' losses.
__device__ inline void sum_by_the_last(const LossParams& p, int64_t n) {
  if (p.a.reduction == MVSD_REDUCE_NONE) return;
  __shared__ int s_last;
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // each wave's losses have left it: a barrier waits for no stores
  __syncthreads();
  if (threadIdx.x == 0) s_last = atomic_add_acq_rel(p.counters + 1, 1) == (int)gridDim.x - 1;
  __syncthreads();
  if (s_last) sum_losses(p, n);
}

// Behind loss_rows_kernel (4.7 us, latency), whose workgroups would write their gradients back from L2 before they count
// themselves (12 us of 260, 30 of 125, against 6 for this launch); and for calls without rows.
__global__ __launch_bounds__(1024) void loss_sum_kernel(LossParams p, int64_t n) { sum_losses(p, n); }

// ------------------------------------------------------------------ the mean's divisor ----------

// Partial sums of the weights of the rows that are not left out, or of the pairs: 3 to 5 us, latency.
__global__ __launch_bounds__(kLossThreads) void loss_norm_kernel(LossParams p) {
  __shared__ float scratch[kWaves];
  const bool pairs = p.a.kind == MVSD_LOSS_PREFERENCE;
  const int64_t n = pairs ? p.a.num_pairs : p.a.num_rows;
  const int64_t each = (n + gridDim.x - 1) / gridDim.x;
  const int64_t first = blockIdx.x * each, last = min(n, first + each);
  float sum[1] = {0.f};
  for (int64_t i = first + threadIdx.x; i < last; i += kLossThreads)
    if (pairs || token_at(p.a, i, p.V) >= 0) sum[0] += p.a.weights ? p.a.weights[i] : 1.f;
  block_sum<1>(sum, scratch);
  if (threadIdx.x == 0) p.norm[blockIdx.x] = sum[0];
  if (blockIdx.x == 0) clear_counters(p);
}

// What a row's weight is multiplied by, in every thread of a wave.
__device__ inline float mean_factor(const LossParams& p) {
  if (p.a.reduction != MVSD_REDUCE_MEAN) return 1.f;
  float sum = 0.f;
  if (p.norm_parts == 0) {  // a policy's few rows, added by whom it concerns
    for (int64_t row = lane_id(); row < p.a.num_rows; row += kWave)
      sum += token_at(p.a, row, p.V) >= 0 ? row_weight(p.a, row) : 0.f;
  }
  for (int i = lane_id(); i < p.norm_parts; i += kWave) sum += p.norm[i];
  sum = wave_sum(sum);
  return sum == 0.f ? 0.f : 1.f / sum;
}

// ------------------------------------------------------------------ rows with one given token ---

struct TokenRow {
  float lp, H;
  LossRecord rec;  // c, cH and pair are the caller's
};

// From the statistics of the rest and the token's logit (a NaN where the id is no token).
__device__ inline TokenRow token_row(const LossParams& p, Stat st, float x) {
  TokenRow r;
  const float base = base_of(st.m);
  if (x == INFINITY) x = NAN;  // as inf - inf
  const float log_s = logf(st.s);
  // of all others against the token; one operation, so that an x / T beyond fp32 is finite beside a log_s of -inf
  const float odds = fmaf(base - x, p.inv_t, log_s);
  const float z = expf(-fabsf(odds)), soft = log1pf(z);
  r.lp = -(fmaxf(odds, 0.f) + soft);
  const float log_q = -(fmaxf(-odds, 0.f) + soft);  // q = 1 - p
  const float small = z / (1.f + z), large = 1.f / (1.f + z);
  const float pt = odds >= 0.f ? small : large;
  const float q = odds >= 0.f ? large : odds < 0.f ? small : NAN;
  const bool none = st.s == 0.f;  // nothing beside the token
  const float h_rest = none ? 0.f : log_s - kLn2 * (st.t / st.s);
  const float own = pt > 0.f ? pt * r.lp : 0.f, rest = q > 0.f ? q * log_q : 0.f;
  r.H = -own - rest + q * h_rest;
  r.rec.M = base;
  r.rec.k = none ? 0.f : q / st.s * p.inv_t;
  r.rec.h = q == 0.f ? 0.f : log_q - log_s + r.H;
  r.rec.o1 = q * p.inv_t;
  r.rec.o2 = -(own + pt * r.H) * p.inv_t;
  if (odds != odds) r.lp = r.H = r.rec.k = NAN;
  return r;
}

struct PolicyRow {
  float loss, c, kl;
};

// What a policy's row is given besides its logits.
struct PolicyIn {
  float A, old, ref;
};
__device__ inline PolicyIn policy_in(const mvsd_loss_args& a, int64_t row) {
  return {a.advantages[row], a.old_logprobs ? a.old_logprobs[row] : 0.f,
          a.ref_logprobs ? a.ref_logprobs[row] : 0.f};
}

__device__ inline PolicyRow policy_row(const mvsd_loss_args& a, const PolicyIn& in, float lp, float H) {
  PolicyRow o;
  const float A = in.A;
  const float gap = lp - in.old;
  const float r = a.old_logprobs ? expf(gap) : lp == lp ? 1.f : lp;
  const float free = A == 0.f && gap < INFINITY ? 0.f : r * A;  // 0 too where the ratio is beyond fp32
  const float bound = fminf(fmaxf(r, (float)(1.0 - a.clip_low)), (float)(1.0 + a.clip_high)) * A;
  const bool clipped = free > bound;
  o.loss = clipped ? -bound : -free;
  o.c = clipped ? 0.f : -free;
  o.kl = 0.f;
  if (a.ref_logprobs) {
    const float d = in.ref - lp, e1 = expm1f(d);
    // e^d - d - 1: its series where the difference of the two would be rounding
    o.kl = fabsf(d) < 0.25f
               ? d * d * (0.5f + d * (1.f / 6 + d * (1.f / 24 + d * (1.f / 120 + d * (1.f / 720 + d * (1.f / 5040 + d * (1.f / 40320)))))))
               : d == -INFINITY ? INFINITY : d == INFINITY ? INFINITY : e1 - d;
    if (a.kl_coef != 0.0) {
      o.loss += (float)a.kl_coef * o.kl;
      o.c -= (float)a.kl_coef * e1;
    }
  }
  if (a.entropy_coef != 0.0) o.loss -= (float)a.entropy_coef * H;
  return o;
}

// The row's values and its record, by a wave, from the statistics of its rest; `out`: it is left out.
template <int DT>
__device__ inline void finish_token_row(const LossParams& p, int64_t row, int token, bool out, Stat st) {
  const mvsd_loss_args& a = p.a;
  TokenRow r;
  PolicyRow o = {0.f, 0.f, 0.f};
  float w = 0.f;
  r.lp = r.H = 0.f;
  r.rec = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0};
  if (!out) {
    const float x = token < p.V ? Elem<DT>::cvt(logits_row<DT>(a, row)[token]) : NAN;
    r = token_row(p, st, x);
    r.rec.pair = 0;
    r.rec.c = 1.f;
    r.rec.cH = 1.f;
    if (a.kind == MVSD_LOSS_POLICY) {
      o = policy_row(a, policy_in(a, row), r.lp, r.H);
      w = row_weight(a, row) * mean_factor(p);
      r.rec.c = o.c * w;
      r.rec.cH = -(float)a.entropy_coef * w;
    } else if (a.kind == MVSD_LOSS_PREFERENCE) {
      r.rec.c = r.rec.cH = 0.f;  // its sequence's, once that is known
    }
  }
  if (lane_id() != 0) return;
  if (a.kind == MVSD_LOSS_PREFERENCE) {
    p.row_lp[row] = r.lp;
  } else {
    a.logprobs[row] = r.lp;
    if (a.entropy) a.entropy[row] = r.H;
  }
  if (a.kind == MVSD_LOSS_POLICY) {
    p.row_loss[row] = out ? 0.f : o.loss * w;
    if (a.kl) a.kl[row] = o.kl;
  }
  if (p.records) p.records[row] = r.rec;
}

// A wave a row: the chunks' statistics together, then the row's loss.  A chain of latencies: 3.1 us for 4 rows,
// 6.1 where a mean's weights and the losses are summed too.
template <int DT>
__global__ __launch_bounds__(kLossThreads) void loss_token_rows_kernel(LossParams p) {
  const int64_t row = (int64_t)blockIdx.x * kWaves + wave_id();
  if (row < p.a.num_rows) {
    const int token = token_at(p.a, row, p.V);
    const bool out = token < 0 || row_weight(p.a, row) == 0.f;
    Stat st = {-INFINITY, 0.f, 0.f};
    if (!out) {
      for (int i = lane_id(); i < p.nch; i += kWave) {
        const float4 v = p.parts[row * p.nch + i];
        st = join(st, {v.x, v.y, v.z}, p.c1);
      }
      st = wave_join(st, p.c1);
    }
    finish_token_row<DT>(p, row, token, out, st);
  }
  if (p.a.kind == MVSD_LOSS_POLICY) sum_by_the_last(p, p.a.num_rows);
}

// One workgroup a chunk of a row: statistics of its rest.  Blocks of kBlock vectors a thread, the next one's
// loads in flight while one is added.  A row of one chunk (of token rows) is finished on the spot.  Bound by
// reads: 1843 bf16 rows of 151936 in 102.5 us, 5.5 TB/s (71 us for 1250 rows, 5.4); 4.5 us for 4 rows in 1024
// chunks, most of it the launch and one read's latency.
template <int DT, bool LIST, bool ENT>
__global__ __launch_bounds__(kLossThreads) void loss_stats_kernel(LossParams p) {
  constexpr int VEC = Elem<DT>::kVec, kBlock = 4, kStep = kLossThreads * VEC;
  extern __shared__ uint32_t bits[];
  __shared__ Stat s_stat[kWaves];
  const int64_t row = blockIdx.x / p.nch;
  const int part = blockIdx.x - (int)(row * p.nch);
  const int begin = part * p.chunk, end = min(p.V, begin + p.chunk);
  const bool whole = !LIST && p.whole;
  int token = -1;
  if (!LIST && p.norm_parts == 0 && blockIdx.x == 0) clear_counters(p);  // a later kernel counts
  if constexpr (LIST) {
    if (p.teach[row].weight == 0.f) return;
    for (int i = threadIdx.x; i < (p.chunk + 31) / 32; i += kLossThreads) bits[i] = 0;
    __syncthreads();
    for (int k = threadIdx.x; k < p.K; k += kLossThreads) {
      const int id = p.over_ids[row * p.K + k];
      if (id >= begin && id < end) atomicOr(&bits[(id - begin) >> 5], 1u << ((id - begin) & 31));
    }
    __syncthreads();
  } else {
    token = token_at(p.a, row, p.V);
    if (token < 0 || row_weight(p.a, row) == 0.f) {
      if (whole && wave_id() == 0) finish_token_row<DT>(p, row, token, true, {-INFINITY, 0.f, 0.f});
      if (whole && p.a.kind == MVSD_LOSS_POLICY) sum_by_the_last(p, p.a.num_rows);
      return;
    }
  }
  const auto* x = logits_row<DT>(p.a, row);
  Stat st = {-INFINITY, 0.f, 0.f};
  const int mine = begin + (int)threadIdx.x * VEC;
  const int blocks = (end - begin) / (kStep * kBlock);
  auto load = [&](u32x4 (&v)[kBlock], int block) {
#pragma unroll
    for (int u = 0; u < kBlock; ++u) v[u] = load_vec_any<DT>(x + mine + (block * kBlock + u) * kStep);
  };
  auto add = [&](u32x4 (&v)[kBlock], int block) {
#pragma unroll
    for (int u = 0; u < kBlock; ++u) {
      const int col = mine + (block * kBlock + u) * kStep;
      if constexpr (LIST) {
        const unsigned marks = marks_at(bits, col - begin, VEC);
        if (marks) mask_vec<DT>(v[u], marks);
      } else if (token >= col && token < col + VEC) {
        mask_vec<DT>(v[u], 1u << (token - col));
      }
    }
    add_vecs<DT, ENT, kBlock>(st, v, p.c1);
  };
  if (blocks > 0) {
    u32x4 a[kBlock], b[kBlock];
    load(a, 0);
    int k = 0;
    for (; k + 2 < blocks; k += 2) {
      load(b, k + 1);
      add(a, k);
      load(a, k + 2);
      add(b, k + 1);
    }
    if (k + 1 < blocks) {
      load(b, k + 1);
      add(a, k);
      add(b, k + 1);
    } else {
      add(a, k);
    }
  }
  for (int col = mine + blocks * kBlock * kStep; col < end; col += kStep) {
    float v[VEC];
    load_filled<DT>(x, col, end, v);
    const unsigned marks = LIST ? marks_at(bits, col - begin, VEC) : 0;
#pragma unroll
    for (int e = 0; e < VEC; ++e) v[e] = (LIST ? marks >> e & 1 : token == col + e) ? -INFINITY : v[e];
    add_values<ENT, VEC>(st, v, p.c1);
  }
  st = wave_join(st, p.c1);
  if (lane_id() == 0) s_stat[wave_id()] = st;
  __syncthreads();
  if (wave_id() == 0) {
    st = join(join(s_stat[0], s_stat[1], p.c1), join(s_stat[2], s_stat[3], p.c1), p.c1);
    if (whole)
      finish_token_row<DT>(p, row, token, false, st);
    else if (lane_id() == 0)
      p.parts[blockIdx.x] = make_float4(st.m, st.s, st.t, 0.f);
  }
  if (whole && p.a.kind == MVSD_LOSS_POLICY) sum_by_the_last(p, p.a.num_rows);
}

// A workgroup a pair: the sums over its two sequences, its loss, its rows' factors.  Latencies, 5 us for one
// pair and 8 for 16.
__global__ __launch_bounds__(kLossThreads) void loss_pairs_kernel(LossParams p) {
  __shared__ float scratch[4 * kWaves];
  const mvsd_loss_args& a = p.a;
  const int64_t pair = blockIdx.x, B = a.num_pairs, N = a.num_rows;
  float w = a.weights ? a.weights[pair] : 1.f;
  if (a.reduction == MVSD_REDUCE_MEAN) {
    float all[1] = {0.f};  // of many pairs, loss_norm_kernel's sums
    const float* some = p.norm_parts ? p.norm : a.weights;
    const int n = p.norm_parts ? p.norm_parts : (int)B;
    for (int i = threadIdx.x; some && i < n; i += kLossThreads) all[0] += some[i];
    block_sum<1>(all, scratch);
    if (!some) all[0] = (float)B;
    w = all[0] == 0.f ? 0.f : w / all[0];
  }
  int64_t begin[2], end[2];
  float v[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int side = 0; side < 2; ++side) {
    const int64_t s = pair + side * B;
    if (a.cu_num_tokens) {
      begin[side] = s == 0 ? 0 : a.cu_num_tokens[s - 1];
      end[side] = a.cu_num_tokens[s];
    } else {
      begin[side] = s * (N / (2 * B));
      end[side] = begin[side] + N / (2 * B);
    }
    begin[side] = min(max(begin[side], (int64_t)0), N);
    end[side] = min(max(end[side], begin[side]), N);
    for (int64_t row = begin[side] + threadIdx.x; row < end[side]; row += kLossThreads) {
      v[side] += p.row_lp[row];
      v[2 + side] += token_at(a, row, p.V) >= 0 ? 1.f : 0.f;
    }
  }
  block_sum<4>(v, scratch);
  float unit[2], S[2];
#pragma unroll
  for (int side = 0; side < 2; ++side) {
    unit[side] = a.average ? 1.f / fmaxf(v[2 + side], 1.f) : 1.f;
    S[side] = a.average ? v[side] / fmaxf(v[2 + side], 1.f) : v[side];
  }
  const float chosen = a.ref_logprobs ? S[0] - a.ref_logprobs[pair] : S[0];
  const float rejected = a.ref_logprobs ? S[1] - a.ref_logprobs[pair + B] : S[1];
  const float m = chosen - rejected, beta = (float)a.beta, margin = (float)a.margin;
  const float h = beta * m - margin, e = (float)a.label_smoothing;
  float loss, c;
  if (a.loss_type == MVSD_PREF_SIGMOID) {
    const float z = expf(-fabsf(h)), soft = log1pf(z);
    loss = soft + (1.f - e) * fmaxf(-h, 0.f) + e * fmaxf(h, 0.f);
    const float small = z / (1.f + z), large = 1.f / (1.f + z);
    const float up = h >= 0.f ? large : h < 0.f ? small : NAN, down = h >= 0.f ? small : large;
    c = beta * (e * up - (1.f - e) * down);
    if (h != h) loss = NAN;
  } else if (a.loss_type == MVSD_PREF_HINGE) {
    loss = h < 1.f ? 1.f - h : h >= 1.f ? 0.f : NAN;
    c = h < 1.f ? -beta : h >= 1.f ? 0.f : NAN;
  } else {
    const float off = m - margin - (float)(0.5 / a.beta);
    loss = off * off;
    c = 2.f * off;
  }
  const bool out = w == 0.f;
  if (threadIdx.x == 0) {
    p.row_loss[pair] = out ? 0.f : loss * w;
    a.logprobs[pair] = S[0];
    a.logprobs[pair + B] = S[1];
  }
  if (a.num_rows > 0) sum_by_the_last(p, B);
  if (!p.records || out) return;
#pragma unroll
  for (int side = 0; side < 2; ++side)
    for (int64_t row = begin[side] + threadIdx.x; row < end[side]; row += kLossThreads) {
      if (token_at(a, row, p.V) < 0) continue;
      LossRecord& r = p.records[row];
      r.c = (side ? -c : c) * unit[side] * w;
      r.pair = (int)pair;
    }
}

// ------------------------------------------------------------------ distillation ----------------

__device__ inline double wave_sum_f64(double v) {
#pragma unroll
  for (int d = 1; d < kWave; d *= 2) v += __shfl_xor(v, d);
  return v;
}

__device__ inline void teacher_of(const LossParams& p, float v, float teacher, float& q, float& log_q) {
  log_q = p.a.tail ? v : v * p.inv_t - teacher;
  q = expf(log_q);
}

// What needs the row's given tokens alone, a wave a row: which entries count (over_ids, -1: not) and their
// logits; the mass of the rest (0 where the rest is no outcome) or, without a tail, the log of the entries'
// sum; the row's weight (0: left out) and the partial sums of the weights; the entries' sums.  Here, because the
// workgroup of a row would spend four barriers on them (1024 rows of 33 entries: 171 us a pass against 160).
// 4.5 us for few rows, 6.7 for 1024 of 33 entries, 19.8 for 2048 of 128, whose 250000 logits are a line each.
template <int DT, int E>  // entries a lane
__global__ __launch_bounds__(kLossThreads) void loss_teacher_kernel(LossParams p) {
  __shared__ __attribute__((aligned(16))) int s_ids[kWaves][E * kWave];
  __shared__ float scratch[kWaves];
  const mvsd_loss_args& a = p.a;
  const int64_t each = (a.num_rows + gridDim.x - 1) / gridDim.x;
  const int64_t first = blockIdx.x * each, last = min(a.num_rows, first + each);
  const int K = p.K, lane = lane_id();
  int* ids = s_ids[wave_id()];
  float weights[1] = {0.f};
  for (int64_t row = first + wave_id(); row < last; row += kWaves) {
    int id[E];
    float v[E];
#pragma unroll
    for (int i = 0; i < E; ++i) {
      const int k = min(i * kWave + lane, K - 1);
      id[i] = token_at(a, row * K + k, p.V);
      v[i] = a.teacher_logprobs[row * K + k];
    }
#pragma unroll
    for (int i = 0; i < E; ++i) {
      if (i * kWave + lane >= K) id[i] = -1;
      ids[i * kWave + lane] = id[i];  // a wave's own places: its reads below follow
    }
    __builtin_amdgcn_wave_barrier();
    bool before[E] = {};
    for (int j = 0; j < K; j += 4) {
      const int4 other = *reinterpret_cast<const int4*>(ids + j);
#pragma unroll
      for (int i = 0; i < E; ++i) {
        if (i * kWave >= K) break;
        const int k = i * kWave + lane;
        before[i] |= (other.x == id[i] && j < k) | (other.y == id[i] && j + 1 < k) |
                     (other.z == id[i] && j + 2 < k) | (other.w == id[i] && j + 3 < k);
      }
    }
    __builtin_amdgcn_wave_barrier();
    int count = 0;
    float top = -INFINITY;
#pragma unroll
    for (int i = 0; i < E; ++i) {
      if (i * kWave >= K) break;
      const int k = i * kWave + lane;
      if (id[i] >= 0 && before[i]) id[i] = -1;
      if (id[i] < 0) v[i] = -INFINITY;
      count += __popcll(__ballot(id[i] >= 0));
      top = fmaxf(top, v[i]);
      if (k < K) p.over_ids[row * K + k] = id[i];
    }
    float value;
    if (a.tail) {
      double mass = 0.0;
#pragma unroll
      for (int i = 0; i < E; ++i)
        if (i * kWave < K) mass += exp((double)v[i]);
      mass = wave_sum_f64(mass);
      value = count >= p.V ? 0.f : mass != mass ? NAN : (float)fmax(1.0 - mass, 0x1p-24);
    } else {
      top = base_of(wave_max(top));
      float sum = 0.f;
#pragma unroll
      for (int i = 0; i < E; ++i)
        if (i * kWave < K) sum += expf((v[i] - top) * p.inv_t);
      value = top * p.inv_t + logf(wave_sum(sum));
    }
    const float w = count == 0 ? 0.f : row_weight(a, row);
    weights[0] += w;
    EntrySums sums = {0.f, 0.f, 0.f, 0.f};
    if (w != 0.f) {
      const auto* x = logits_row<DT>(a, row);
      float g[E];
#pragma unroll
      for (int i = 0; i < E; ++i)
        if (i * kWave < K) g[i] = id[i] >= 0 && id[i] < p.V ? Elem<DT>::cvt(x[id[i]]) : id[i] < 0 ? -INFINITY : NAN;
      top = -INFINITY;
#pragma unroll
      for (int i = 0; i < E; ++i) {
        if (i * kWave >= K) break;
        if (g[i] == INFINITY) g[i] = NAN;
        top = fmaxf(top, g[i]);
      }
      sums.top = top = base_of(wave_max(top));
#pragma unroll
      for (int i = 0; i < E; ++i) {
        if (i * kWave >= K) break;
        const int k = i * kWave + lane;
        if (k < K) p.entry_logits[row * K + k] = g[i];
        const float d = (g[i] - top) * p.inv_t, e = expf(d);
        float q, log_q;
        teacher_of(p, v[i], value, q, log_q);
        if (id[i] < 0) continue;
        sums.z += e;
        if (a.divergence == MVSD_KL_FORWARD) {
          sums.s1 += q == 0.f ? 0.f : q * (log_q - d);
          sums.s2 += q;
        } else {
          sums.s1 += e == 0.f ? 0.f : e * (d - log_q);
        }
      }
      sums = {top, wave_sum(sums.z), wave_sum(sums.s1), wave_sum(sums.s2)};
    }
    if (lane == 0) p.teach[row] = {sums, value, w, 0.f, 0.f};
  }
  if (lane != 0) weights[0] = 0.f;
  block_sum<1>(weights, scratch);
  if (threadIdx.x == 0) p.norm[blockIdx.x] = weights[0];
  if (blockIdx.x == 0) clear_counters(p);
}

// A row's entries, entry i * T + thread in each of T threads.
template <int E>
struct Entries {
  int id[E];  // -1: it does not count
  float x[E], v[E];
};

template <int E>
__device__ inline void load_entry_values(const LossParams& p, int64_t row, int T, Entries<E>& in) {
#pragma unroll
  for (int i = 0; i < E; ++i) {
    const int k = i * T + (int)threadIdx.x;
    in.v[i] = 0.f;
    in.x[i] = -INFINITY;
    if (k < p.K) {
      in.v[i] = p.a.teacher_logprobs[row * p.K + k];
      in.x[i] = p.entry_logits[row * p.K + k];
    }
  }
}

__device__ inline float sum16(float v) {
  v += dpp_f32<kDppXor1>(v);
  v += dpp_f32<kDppXor2>(v);
  v += dpp_f32<kDppHalfMirror>(v);
  return v + dpp_f32<kDppMirror>(v);
}

// Sums over the NW waves of a workgroup, in one order; two barriers.
template <int N>
__device__ inline void waves_sum(float (&v)[N], float* red, int NW) {
#pragma unroll
  for (int g = 0; g < N; ++g) v[g] = wave_sum(v[g]);
  if (lane_id() == 0) {
#pragma unroll
    for (int g = 0; g < N; ++g) red[g * NW + wave_id()] = v[g];
  }
  __syncthreads();
  const int part = lane_id() % 16;
#pragma unroll
  for (int g = 0; g < N; ++g) v[g] = readlane_f32(sum16(part < NW ? red[g * NW + part] : 0.f), 0);
  __syncthreads();
}
// One row's loss by a workgroup of NW waves, from the statistics of its rest, its entries and what the
// teacher's kernel gave of it.  Gives the gradients of the given tokens (over, at id, -1: none) and returns
// the loss; *k is the record's.  `weight` is the row's, after the mean.  With d_k = (x_k - top) / T and lz the
// log of the row's sum against top, the entries' part of sum q (log q - log p) is s1 + lz s2, that of
// sum p (log p - log q) is (s1 - lz z) / e^lz; only a Jensen-Shannon divergence needs sums behind lz.
template <int E>
__device__ inline float distill_row(const LossParams& p, Stat st, const EntrySums& k, float teacher, float weight,
                                    float* red, int NW, Entries<E>& in, float (&over)[E], float* k_out) {
  const mvsd_loss_args& a = p.a;
  const bool tail = a.tail && teacher != 0.f;
  // entries that are all masked have no maximum: the rest's is the row's
  const float top = k.z == 0.f ? base_of(st.m) : k.top;
  // infinite where a mask of the type's lowest value over T leaves fp32: the sum is against the larger maximum, and
  // the rest's log-probability is formed without lz
  const float rest_d = st.m == -INFINITY ? 0.f : (st.m - top) * p.inv_t, far = fmaxf(rest_d, 0.f);
  const float near = fminf(rest_d, 0.f), log_sum = logf(k.z * expf(-far) + st.s * expf(near)), lz = far + log_sum;
  const float rest_lp = near + logf(st.s) - log_sum, rest_p = st.s > 0.f ? expf(rest_lp) : st.s;
  // the divergence's term, and p dL/dp, of an outcome
  auto outcome = [&](float q, float log_q, float pr, float lp, float& term, float& pd) {
    if (a.divergence == MVSD_KL_FORWARD) {
      term = q == 0.f ? 0.f : q * (log_q - lp);
      pd = -q;
    } else if (a.divergence == MVSD_KL_REVERSE) {
      term = pd = pr == 0.f ? 0.f : pr * (lp - log_q);
    } else {
      const float mix = 0.5f * (pr + q), lm = logf(mix);
      pd = pr == 0.f ? 0.f : 0.5f * pr * (lp - lm);
      term = pd + (q == 0.f ? 0.f : 0.5f * q * (log_q - lm));
    }
  };
  float both[2] = {0.f, 0.f}, pr[E], pd[E];  // the sums of terms, and of p dL/dp
#pragma unroll
  for (int i = 0; i < E; ++i) {
    const float lp = (in.x[i] - top) * p.inv_t - lz;
    float q, log_q, term = 0.f;
    teacher_of(p, in.v[i], teacher, q, log_q);
    pr[i] = expf(lp);
    pd[i] = 0.f;
    if (in.id[i] >= 0) outcome(q, log_q, pr[i], lp, term, pd[i]);
    both[0] += term;
    both[1] += pd[i];
  }
  if (a.divergence == MVSD_KL_FORWARD) {
    both[0] = k.s2 == 0.f && lz == INFINITY ? k.s1 : k.s1 + lz * k.s2;
    both[1] = -k.s2;
  } else if (a.divergence == MVSD_KL_REVERSE) {
    // entries whose probabilities are all below fp32's range are 0, also where the teacher has none
    const float scale = expf(-lz);
    both[0] = both[1] = scale == 0.f && k.s1 == k.s1 ? 0.f : (k.s1 - lz * k.z) * scale;
  } else {
    waves_sum<2>(both, red, NW);
  }
  float rest_pd = 0.f;
  if (tail) {
    float term;
    outcome(teacher, logf(teacher), rest_p, rest_lp, term, rest_pd);
    both[0] += term;
    both[1] += rest_pd;
  }
  const float f = weight * p.inv_t;
  if (lz != lz || log_sum == -INFINITY)  // a NaN in the row, or nothing but -inf
    *k_out = NAN;
  else
    *k_out = st.s == 0.f ? 0.f : -f * (rest_pd - rest_p * both[1]) / st.s;
#pragma unroll
  for (int i = 0; i < E; ++i) {
    over[i] = f * (pd[i] - pr[i] * both[1]);
    if (in.id[i] >= p.V) in.id[i] = -1;
  }
  return both[0] * weight;
}

template <int E>
__device__ inline void save_over(const LossParams& p, int64_t row, int T, const float (&over)[E]) {
#pragma unroll
  for (int i = 0; i < E; ++i) {
    const int k = i * T + (int)threadIdx.x;
    if (k < p.K) p.over[row * p.K + k] = over[i];
  }
}

// A workgroup a row: 7.5 us for 16 rows, a chain of latencies.
__global__ __launch_bounds__(kLossThreads) void loss_distill_rows_kernel(LossParams p) {
  constexpr int E = kMaxTeacher / kLossThreads;
  __shared__ float red[2 * kWaves];
  const int64_t row = blockIdx.x;
  const LossTeacher teacher = p.teach[row];
  float loss = 0.f;
  LossRecord rec = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0};
  if (teacher.weight != 0.f) {
    Entries<E> in;
#pragma unroll
    for (int i = 0; i < E; ++i) {
      const int k = i * kLossThreads + (int)threadIdx.x;
      in.id[i] = k < p.K ? p.over_ids[row * p.K + k] : -1;
    }
    load_entry_values<E>(p, row, kLossThreads, in);
    Stat st = {-INFINITY, 0.f, 0.f};
    for (int i = lane_id(); i < p.nch; i += kWave) {
      const float4 v = p.parts[row * p.nch + i];
      st = join(st, {v.x, v.y, v.z}, p.c1);
    }
    st = wave_join(st, p.c1);
    rec.M = base_of(st.m);
    rec.c = 1.f;
    float over[E];
    loss = distill_row<E>(p, st, teacher.sums, teacher.value, teacher.weight * mean_factor(p), red, kWaves, in, over,
                          &rec.k);
    if (p.records) save_over<E>(p, row, kLossThreads, over);
  }
  if (threadIdx.x == 0) {
    p.row_loss[row] = loss;
    if (p.records) p.records[row] = rec;
  }
  sum_by_the_last(p, p.a.num_rows);
}

// ------------------------------------------------------------------ the gradient ----------------

// The gradient at the rest, e (a + b log2 e), and at the given token, for the factors g and gH.  Both
// gradient kernels go through these, so that they give the same bits.
struct RestGradient {
  float a, b;
};
__device__ inline RestGradient rest_gradient(const LossRecord& r, float g, float gH) {
  return {-r.k * fmaf(gH, r.h, g), -r.k * gH * kLn2};
}
__device__ inline float token_gradient(const LossRecord& r, float g, float gH) {
  return fmaf(gH, r.o2, g * r.o1);
}
template <bool ENT>
__device__ inline float rest_value(float x, float M, float c1, RestGradient k) {
  const float y = (x - M) * c1, w = __builtin_amdgcn_exp2f(y);
  return w * (ENT ? fmaf(k.b, fmaxf(y, kLeast), k.a) : k.a);
}

template <int DT>
__device__ inline u32x4 pack_vec(const float (&g)[Elem<DT>::kVec]) {
  u32x4 r;
  if constexpr (DT == MVSD_F32) {
#pragma unroll
    for (int e = 0; e < 4; ++e) r[e] = __float_as_uint(g[e]);
  } else {
    using H = std::conditional_t<DT == MVSD_BF16, __bf16, _Float16>;
    typedef H pair_t __attribute__((ext_vector_type(2)));
    typedef float float2_t __attribute__((ext_vector_type(2)));
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float2_t f = {g[2 * e], g[2 * e + 1]};
      r[e] = __builtin_bit_cast(uint32_t, __builtin_convertvector(f, pair_t));
    }
  }
  return r;
}

template <int DT>
__device__ inline typename Elem<DT>::storage to_storage(float g) {
  if constexpr (DT == MVSD_F32) return g;
  else if constexpr (DT == MVSD_F16) return (_Float16)g;
  else return __builtin_bit_cast(uint16_t, (__bf16)g);
}

// PAST: past the caches.
template <int DT, bool PAST = false>
__device__ inline void store_filled(typename Elem<DT>::storage* row, int col, int end,
                                    const float (&g)[Elem<DT>::kVec]) {
  constexpr int VEC = Elem<DT>::kVec;
  if (col + VEC <= end) {
    if constexpr (PAST)
      __builtin_nontemporal_store(pack_vec<DT>(g), reinterpret_cast<Vec16<DT>*>(row + col));
    else
      *reinterpret_cast<Vec16<DT>*>(row + col) = pack_vec<DT>(g);
  } else {
#pragma unroll
    for (int e = 0; e < VEC; ++e)
      if (col + e < end) row[col + e] = to_storage<DT>(g[e]);
  }
}

// A chunk of a row by a workgroup, from the row's record.
template <int DT, bool LIST, bool ENT, bool PAST>
__device__ inline void gradient_chunk(const LossParams& p, const float* up, int64_t us, const float* up_h,
                                      int64_t uhs, int64_t chunk) {
  constexpr int VEC = Elem<DT>::kVec;
  const int64_t at = chunk / p.nch, row = p.a.num_rows - 1 - at;
  const int part = chunk - at * p.nch;
  const int begin = part * p.chunk, end = min(p.V, begin + p.chunk);
  const LossRecord rec = p.records[row];
  const int64_t n = p.a.kind == MVSD_LOSS_PREFERENCE ? rec.pair : row;
  const float g = rec.c == 0.f || !up ? 0.f : rec.c * up[n * us];
  const float gH = !ENT || rec.cH == 0.f || !up_h ? 0.f : rec.cH * up_h[n * uhs];
  auto* out = static_cast<typename Elem<DT>::storage*>(p.a.grad) + row * p.V;
  if (g == 0.f && gH == 0.f) {
    const float zero[VEC] = {};
    for (int col = begin + (int)threadIdx.x * VEC; col < end; col += kLossThreads * VEC)
      store_filled<DT, PAST>(out, col, end, zero);
    return;
  }
  const auto* x = logits_row<DT>(p.a, row);
  const RestGradient rest = rest_gradient(rec, g, gH);
  const int token = LIST ? -1 : token_at(p.a, row, p.V);
  const float at_token = token_gradient(rec, g, gH);
  for (int col = begin + (int)threadIdx.x * VEC; col < end; col += kLossThreads * VEC) {
    float v[VEC];
    load_filled<DT>(x, col, end, v);
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
      v[e] = rest_value<ENT>(v[e], rec.M, p.c1, rest);
    }
    if (!LIST && token >= col && token < col + VEC) {
#pragma unroll
      for (int e = 0; e < VEC; ++e) v[e] = token == col + e ? at_token : v[e];
    }
    store_filled<DT, PAST>(out, col, end, v);
  }
  if constexpr (LIST) {
    __syncthreads();
    for (int k = threadIdx.x; k < p.K; k += kLossThreads) {
      const int id = p.over_ids[row * p.K + k];
      if (id >= begin && id < end) out[id] = to_storage<DT>(g * p.over[row * p.K + k]);
    }
  }
}

// The last rows first: the statistics were read in the rows' order, so that the last of them are still in
// the caches, where a gradient that is larger than those (PAST) leaves them by being stored past them.  At a
// copy's rate: 380 MB read and 471 written in 163 us, 5.2 TB/s; fp32 rows with entropies, 301 MB written, 104 us
// (a pass of theirs 157 us; in the rows' order and with ordinary stores 195).
template <int DT, bool LIST, bool ENT, bool PAST>
__global__ __launch_bounds__(kLossThreads) void loss_gradient_kernel(LossParams p, const float* up, int64_t us,
                                                                     const float* up_h, int64_t uhs) {
  if (p.a.unit_gradient && up[0] == 1.f) return;  // it is there already
  for (int64_t chunk = blockIdx.x; chunk < p.a.num_rows * p.nch; chunk += gridDim.x)
    gradient_chunk<DT, LIST, ENT, PAST>(p, up, us, up_h, uhs, chunk);
}

// ------------------------------------------------------------------ values and gradient in one pass ---

constexpr int kMostHeld = 18;  // vectors of a row in each thread's registers (72 of 128)
constexpr int kRowThreads = 1024;

// A value that all lanes have, in a scalar register.
__device__ inline float scalar(float v) { return readlane_f32(v, 0); }

// Rows by a workgroup, one after the other (by tickets: some are left out), every row in its registers: read
// once, written once.  A turn of the loop writes the gradient of one row and, vector by vector, loads the next
// one in its place and adds it to its statistics kDelay vectors later (4, 6, 8, 10 and 12 are within 4 %), so
// that memory is busy except in the reductions and the row's own loss between two turns.  `active` threads hold NV
// vectors each, those of one i side by side (a span, a multiple of 32 columns); the columns behind the spans (few, or
// what the registers do not hold: 78208 of 151936 fp32) are read again, a vector at a time.
// A turn's loads and stores are unconditional, with a first turn that only loads and a last one that only
// stores (a conditional load makes the compiler wait for all of them at once); rows that are left out are
// passed by, their gradient written on the way.
// Bytes read and written a second (a copy: 5.25 TB/s): 2048 policy rows of 151936 bf16 248 us, 4.8 TB/s; 2000 of
// 32001 fp32 with entropies 117 us, 4.4; distillation, 1024 rows of 151936 bf16 and 33 entries, 149 us, 4.2, 2048
// of 128 entries 277 us, 4.4; 4096 of 32000 fp16 133 us, 4.0; 2048 policy rows of 151936 fp32 624 us, 4.0, or 5.0 with
// what is read again.  What is lost: the gap between two turns, and in a distillation the marks (4 us of 160) and the
// entries' own values, which follow the row's stores (3; 17 of 298).
template <int DT, int NV, bool LIST, bool ENT, bool WANT>
__global__ __launch_bounds__(kRowThreads, 4) void loss_rows_kernel(LossParams p) {
  using S = typename Elem<DT>::storage;
  constexpr int VEC = Elem<DT>::kVec, E = 1, kDelay = NV > 4 ? 4 : 2;
  extern __shared__ uint32_t bits[];
  __shared__ float4 s_part[2][kRowThreads / kWave];
  __shared__ float red[2 * kRowThreads / kWave];
  __shared__ int s_ticket[2], s_next;  // two of what is read behind a turn's one barrier: a wave may be a turn ahead
  const mvsd_loss_args& a = p.a;
  const int tid = threadIdx.x, V = p.V, N = (int)a.num_rows, T = blockDim.x, NW = T / kWave;
  const int span = p.active * VEC, behind = NV * span;
  // threads behind the active ones do what the last of those does, and count for nothing
  const unsigned own = min(tid, p.active - 1) * VEC;
  const int tail_col = behind + tid * VEC;
  const float mean = scalar(mean_factor(p)), c1 = p.c1;
  const int words = (V + 31) / 32;
  uint32_t* marked = bits;  // the marks of this turn's row: two sets in turn, the other one is cleared
  if constexpr (LIST) {
    for (int i = tid; i < 2 * words; i += T) bits[i] = 0;
    __syncthreads();
  }

  // What a row is given beside its logits, and what its gradient is formed from.
  int row = blockIdx.x, ticket = 0, token = -1, parity = 0;
  float w = 0.f, xt = NAN;
  PolicyIn given = {0.f, 0.f, 0.f};
  Entries<E> in = {};
  LossTeacher teacher = {};
  const S* x = nullptr;
  int cur = -1, cur_token = -1, pend_id[E];
  float pend[E], cur_M = 0.f, at_token = 0.f;
  RestGradient rest = {0.f, 0.f};
  bool zeros = true;  // the gradient is 0
  const S* cur_x = nullptr;
#pragma unroll
  for (int i = 0; i < E; ++i) pend_id[i] = -1;
  // of the row after it, loaded while this one's loss is formed
  int next_token = -1, next_id = -1;
  float next_w = 0.f;
  auto announce = [&](int n) {
    if (n >= N) return;
    if constexpr (LIST) {
      if (tid < p.K) next_id = p.over_ids[(int64_t)n * p.K + tid];
      next_w = p.teach[n].weight;
    } else {
      next_token = token_at(a, n, V);
      next_w = row_weight(a, n);
    }
  };
  // The next row that is not left out becomes `row`; false: there is none.
  auto advance = [&]() {
    for (; row < N; announce(row)) {
      if constexpr (LIST) {
        in.id[0] = next_id;
      } else {
        token = __builtin_amdgcn_readfirstlane(next_token);
      }
      w = scalar(next_w);
      if (w != 0.f && (LIST || token >= 0)) break;
      if (tid == 0) {
        p.row_loss[row] = 0.f;
        if (p.records) p.records[row] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0};
        if constexpr (!LIST) {
          a.logprobs[row] = 0.f;
          if (a.entropy) a.entropy[row] = 0.f;
          if (a.kl) a.kl[row] = 0.f;
        }
      }
      if (WANT) {
        const float zero[VEC] = {};
        S* out = static_cast<S*>(a.grad) + (int64_t)row * V;
        for (int col = tid * VEC; col < V; col += T * VEC) store_filled<DT>(out, col, V, zero);
      }
      if (tid == 0) s_next = atomicAdd(p.counters, 1);
      __syncthreads();
      row = gridDim.x + __builtin_amdgcn_readfirstlane(s_next);
      __syncthreads();
    }
    if (row >= N) return false;
    if (tid == 0) ticket = atomicAdd(p.counters, 1);  // the next row's, which finish() gives to all
    x = logits_row<DT>(a, row);
    if constexpr (!LIST) {
      xt = token < V ? Elem<DT>::cvt(x[token]) : NAN;
      given = policy_in(a, row);
    }
    return true;
  };

  Stat st;
  u32x4 r[NV] = {};
  bool more = true;
  // A turn's loads and stores are unconditional: a conditional one makes the compiler wait for all of them at
  // once.  The first turn stores to a place of the workgroup's own, the last loads one span again and again.
  S* const aside = static_cast<S*>(p.aside) + (int64_t)blockIdx.x * span;
  auto turn = [&]() {
    st = {-INFINITY, 0.f, 0.f};
    const bool stores = cur >= 0;
    S* out = WANT && stores ? static_cast<S*>(a.grad) + (int64_t)cur * V : aside;
    const unsigned to_step = stores ? span : 0, from_step = more ? span : 0;
    // the span and thread that hold a given token
    const int spot = token >= 0 && token < behind ? token / VEC : -1;
    const int at_span = spot < 0 ? -1 : spot / p.active;
    const bool holds = (int)own == (spot - at_span * p.active) * VEC;
    const int cur_spot = !zeros && cur_token >= 0 && cur_token < behind ? cur_token / VEC : -1;
    const int cur_span = cur_spot < 0 ? -1 : cur_spot / p.active;
    const bool cur_holds = (int)own == (cur_spot - cur_span * p.active) * VEC;
    // uniform offsets, kept so: the compiler would keep each thread's for every vector
    unsigned from = 0, to = 0;
    const uint32_t* marks_from = marked + (own >> 5);
    auto clean = [&](u32x4& v, int i) {  // the given tokens become -inf
      if constexpr (LIST) {
        const unsigned marks = *marks_from >> (own & 31) & ((1u << VEC) - 1);
        marks_from += span / 32;
        asm("" : "+v"(marks_from));
        if (marks) mask_vec<DT>(v, marks);
      } else if (i == at_span) {
        if (holds) mask_vec<DT>(v, 1u << token % VEC);
      }
    };
    auto vector = [&](int i) {
      if (i < NV) {
        if constexpr (WANT) {
          u32x4 v = {0u, 0u, 0u, 0u};
          if (!zeros) {
            float g[VEC];
#pragma unroll
            for (int e = 0; e < VEC; ++e) g[e] = rest_value<ENT>(vec_elem_again<DT>(r[i], e), cur_M, c1, rest);
            if (!LIST && i == cur_span) {
#pragma unroll
              for (int e = 0; e < VEC; ++e) g[e] = cur_holds && cur_token % VEC == e ? at_token : g[e];
            }
            v = pack_vec<DT>(g);
          }
          asm("" : "+s"(to));
          *reinterpret_cast<Vec16<DT>*>(out + to + own) = v;
          to += to_step;
        }
        asm("" : "+s"(from));
        r[i] = load_vec_any<DT>(x + from + own);
        from += from_step;
      }
      const int j = i - kDelay;  // pairs, and a last one alone
      if (more && (j == NV - 1 || (j >= 0 && j % 2 == 1))) {
        if (j % 2 == 1) {
          clean(r[j - 1], j - 1);
          clean(r[j], j);
          add_vecs<DT, ENT, 2>(st, {r[j - 1], r[j]}, c1);
        } else {
          clean(r[j], j);
          add_vecs<DT, ENT, 1>(st, {r[j]}, c1);
        }
      }
      __builtin_amdgcn_sched_barrier(0);  // vectors in their order: more of them at once do not fit the registers
    };
#pragma unroll
    for (int i = 0; i < kDelay; ++i) vector(i);
    if (LIST && more) {  // while the first vectors come: the marks
#pragma unroll
      for (int n = 0; n < E; ++n)
        if (in.id[n] >= 0 && in.id[n] < V) atomicOr(&marked[in.id[n] >> 5], 1u << (in.id[n] & 31));
      __syncthreads();
    }
#pragma unroll
    for (int i = kDelay; i < NV; ++i) vector(i);
    if (LIST && more) {  // what finish() needs, behind the vectors
      teacher = p.teach[row];
      load_entry_values<E>(p, row, T, in);
    }
#pragma unroll
    for (int i = NV; i < NV + kDelay; ++i) vector(i);
    if (tid >= p.active) st = {-INFINITY, 0.f, 0.f};
    for (int col = tail_col; col < V; col += T * VEC) {
      float v[VEC];
      if (WANT && stores) {
        load_filled<DT>(cur_x, col, V, v);
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
          const float g = rest_value<ENT>(v[e], cur_M, c1, rest);
          v[e] = zeros ? 0.f : !LIST && cur_token == col + e ? at_token : g;
        }
        store_filled<DT>(out, col, V, v);
      }
      if (more) {
        load_filled<DT>(x, col, V, v);
        const unsigned marks = LIST ? marks_at(marked, col, VEC) : 0;
#pragma unroll
        for (int e = 0; e < VEC; ++e) v[e] = (LIST ? marks >> e & 1 : token == col + e) ? -INFINITY : v[e];
        add_values<ENT, VEC>(st, v, c1);
      }
    }
  };
  // Behind every store of a row: its given tokens' own values.
  auto give = [&]() {
    if constexpr (LIST && WANT) {
      S* out = static_cast<S*>(a.grad) + (int64_t)cur * V;
#pragma unroll
      for (int i = 0; i < E; ++i)
        if (pend_id[i] >= 0) out[pend_id[i]] = to_storage<DT>(pend[i]);
    }
  };
  // The loss of `row`, which becomes `cur`.
  auto finish = [&]() {
    rebase(st, wave_max(st.m), c1);
    st.s = wave_sum(st.s);
    if constexpr (ENT) st.t = wave_sum(st.t);
    if (lane_id() == 0) s_part[parity][wave_id()] = make_float4(st.m, st.s, st.t, 0.f);
    if (tid == 0) s_ticket[parity] = ticket;
    __syncthreads();
    const int next = gridDim.x + __builtin_amdgcn_readfirstlane(s_ticket[parity]);  // one of all, in a scalar register
    announce(next);
    give();
    const int part = lane_id() % 16;
    const float4 v = part < NW ? s_part[parity][part] : make_float4(-INFINITY, 0.f, 0.f, 0.f);
    st = {v.x, v.y, v.z};
    rebase(st, readlane_f32(max16(st.m), 0), c1);
    st.s = readlane_f32(sum16(st.s), 0);  // one lane's: a sum's last bit may be another in each
    if constexpr (ENT) st.t = readlane_f32(sum16(st.t), 0);
    parity ^= 1;
    LossRecord rec = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0};
    float loss;
    if constexpr (LIST) {
#pragma unroll
      for (int i = 0; i < E; ++i)
        if (in.id[i] >= 0 && in.id[i] < V) marked[in.id[i] >> 5] = 0;
      marked = marked == bits ? bits + words : bits;
      rec.M = base_of(st.m);
      rec.c = 1.f;
      loss = distill_row<E>(p, st, teacher.sums, teacher.value, w * mean, red, NW, in, pend, &rec.k);
      if (p.records) save_over<E>(p, row, T, pend);
#pragma unroll
      for (int i = 0; i < E; ++i) pend_id[i] = in.id[i];
    } else {
      const TokenRow o = token_row(p, st, xt);
      const PolicyRow q = policy_row(a, given, o.lp, o.H);
      rec = o.rec;
      rec.c = q.c * w * mean;
      rec.cH = -(float)a.entropy_coef * w * mean;
      rec.pair = 0;
      loss = q.loss * w * mean;
      if (tid == 0) {
        a.logprobs[row] = o.lp;
        if (a.entropy) a.entropy[row] = o.H;
        if (a.kl) a.kl[row] = q.kl;
      }
    }
    if (tid == 0) {
      p.row_loss[row] = loss;
      if (p.records) p.records[row] = rec;
    }
    const float gH = ENT ? rec.cH : 0.f;
    zeros = rec.c == 0.f && gH == 0.f;
    cur_M = scalar(rec.M);
    rest = rest_gradient(rec, rec.c, gH);
    rest = {scalar(rest.a), scalar(rest.b)};
    at_token = scalar(token_gradient(rec, rec.c, gH));
    cur = row;
    cur_x = x;
    cur_token = token;
    row = next;
  };

  announce(row);
  if (advance()) {
    for (;;) {
      turn();
      if (!more) break;
      finish();
      more = advance();
      if (!WANT && !more) break;
    }
    __syncthreads();
    give();
  }
}

// ------------------------------------------------------------------ host ------------------------

int64_t up16(int64_t v) { return (v + 15) / 16 * 16; }

bool has_list(const mvsd_loss_args& a) { return a.kind == MVSD_LOSS_DISTILL; }

// Columns of a workgroup in the split kernels: enough workgroups for the card's 256 CUs, each of at least
// one vector a thread and of so many columns that their marks fit LDS (32 KiB).
constexpr int64_t kMaxChunk = 1 << 18;
int chunk_of(int64_t rows, int V, int dtype) {
  const int step = kLossThreads * (dtype == MVSD_F32 ? 4 : 8);
  const int64_t want = (1024 + rows - 1) / std::max(rows, (int64_t)1);
  const int64_t steps = (V + step - 1) / step;
  const int64_t each = (steps + want - 1) / want;
  return (int)std::min(std::max(each, (int64_t)1) * step, kMaxChunk);
}

int num_cus() {
  static std::atomic<int> cus[64];
  int device = 0, n = 0;
  if (hipGetDevice(&device) != hipSuccess || device < 0 || device >= 64) return 256;
  if ((n = cus[device].load(std::memory_order_relaxed)) > 0) return n;
  if (hipDeviceGetAttribute(&n, hipDeviceAttributeMultiprocessorCount, device) != hipSuccess || n < 1) n = 256;
  cus[device].store(n, std::memory_order_relaxed);
  return n;
}

// How loss_rows_kernel holds a row of V columns: NV vectors in each of `active` threads.
struct RowPlan {
  int held, active, threads;
};
RowPlan row_plan(const mvsd_loss_args& a) {
  const int64_t vectors = a.vocab_size / (a.dtype == MVSD_F32 ? 4 : 8);
  RowPlan best = {0, 0, 0};
  int most = 0;
  for (int held : {18, 16, 13, 10, 6, 3}) {
    if (held < kMostHeld && vectors / held > kRowThreads) break;  // columns would be read again
    RowPlan r;
    r.held = held;
    r.active = (int)std::min(vectors / held, (int64_t)kRowThreads) / 8 * 8;
    r.threads = (r.active + kWave - 1) / kWave * kWave;
    if (has_list(a)) r.threads = std::max(r.threads, (int)(a.num_teacher + kWave - 1) / kWave * kWave);  // an entry each
    // the active threads of a CU, whose registers hold 1024
    const int busy = r.active == 0 ? 0 : kRowThreads / r.threads * r.active;
    if (busy > most) best = r, most = busy;
  }
  return best;
}

// Its workgroups: as many as run at once.
int64_t row_groups(const mvsd_loss_args& a, const RowPlan& plan) {
  return std::min(a.num_rows, (int64_t)num_cus() * (kRowThreads / plan.threads));
}

// What its first turns store.
int64_t aside_bytes(const mvsd_loss_args& a) {
  if (!loss_one_pass(a)) return 0;
  const RowPlan plan = row_plan(a);
  return row_groups(a, plan) * plan.active * 16;
}

constexpr int64_t kMaxMarked = 3 << 16;  // columns whose two sets of marks are 48 KiB

constexpr int64_t kFewRows = 512;    // whose weights every wave adds by itself (a launch less)
constexpr int64_t kFewPairs = 2048;  // the same of pairs and workgroups
constexpr int64_t kCacheBytes = 256ll << 20;  // of the last level

LossParams make_params(const mvsd_loss_args& a) {
  LossParams p = {};
  p.a = a;
  p.V = (int)a.vocab_size;
  p.K = has_list(a) ? (int)a.num_teacher : 1;
  p.c1 = (float)(1.4426950408889634 / a.temperature);
  p.inv_t = (float)(1.0 / a.temperature);
  p.chunk = chunk_of(a.num_rows, p.V, a.dtype);
  p.nch = (p.V + p.chunk - 1) / p.chunk;
  p.entropy = (a.kind == MVSD_LOSS_LOGPROBS || a.kind == MVSD_LOSS_POLICY) && (a.entropy || a.entropy_coef != 0.0);
  const int64_t N = a.num_rows;
  char* w = static_cast<char*>(a.workspace);
  p.aside = w;
  w += aside_bytes(a);
  p.parts = reinterpret_cast<float4*>(w);
  w += N * p.nch * sizeof(float4);
  p.norm = reinterpret_cast<float*>(w);
  w += kNormParts * sizeof(float);
  p.counters = reinterpret_cast<int*>(w);
  w += 16;
  p.row_loss = a.reduction == MVSD_REDUCE_NONE && a.loss ? a.loss : reinterpret_cast<float*>(w);
  w += up16(std::max(N, a.num_pairs) * 4);
  p.row_lp = reinterpret_cast<float*>(w);
  p.teach = reinterpret_cast<LossTeacher*>(w);  // of a distillation, which has no row_lp
  w += up16(N * (has_list(a) ? (int64_t)sizeof(LossTeacher) : 4));
  p.entry_logits = reinterpret_cast<float*>(w);
  if (has_list(a)) w += up16(N * p.K * 4);
  p.over_ids = reinterpret_cast<int32_t*>(w);
  if (a.saved) {
    p.records = static_cast<LossRecord*>(a.saved);
    p.over = reinterpret_cast<float*>(p.records + N);
    p.over_ids = reinterpret_cast<int32_t*>(p.over + N * p.K);
  }
  // the distillation's kernel has a wave a row where there are few
  if (a.kind == MVSD_LOSS_DISTILL)
    p.norm_parts = (int)std::min((N + kWaves - 1) / kWaves, (int64_t)kNormParts);
  else if (a.kind == MVSD_LOSS_POLICY && a.reduction != MVSD_REDUCE_NONE && (N > kFewRows || loss_one_pass(a)))
    p.norm_parts = (int)std::min(N / 64 + 1, (int64_t)kNormParts);
  else if (a.kind == MVSD_LOSS_PREFERENCE && a.reduction == MVSD_REDUCE_MEAN && a.weights && a.num_pairs > kFewPairs)
    p.norm_parts = (int)std::min(a.num_pairs / 1024 + 1, (int64_t)kNormParts);
  // a workgroup that counts itself needs counters that an earlier launch cleared
  p.whole = p.nch == 1 && (a.kind != MVSD_LOSS_POLICY || a.reduction == MVSD_REDUCE_NONE || p.norm_parts > 0);
  return p;
}

template <int DT, int NV, bool WANT>
void launch_rows_of(const LossParams& p, const RowPlan& plan, hipStream_t stream) {
  const dim3 grid((unsigned)row_groups(p.a, plan));
  const dim3 block(plan.threads);
  if (has_list(p.a))
    hipLaunchKernelGGL((loss_rows_kernel<DT, NV, true, false, WANT>), grid, block, (unsigned)((p.V + 31) / 32 * 8), stream, p);
  else if (p.entropy)
    hipLaunchKernelGGL((loss_rows_kernel<DT, NV, false, true, WANT>), grid, block, 0, stream, p);
  else
    hipLaunchKernelGGL((loss_rows_kernel<DT, NV, false, false, WANT>), grid, block, 0, stream, p);
}

template <int DT, int NV>
void launch_rows(const LossParams& p, const RowPlan& plan, hipStream_t stream) {
  if (p.a.grad)
    launch_rows_of<DT, NV, true>(p, plan, stream);
  else
    launch_rows_of<DT, NV, false>(p, plan, stream);
}

template <int DT>
hipError_t launch_dt(const LossParams& p, hipStream_t stream) {
  const mvsd_loss_args& a = p.a;
  const dim3 grid((unsigned)(a.num_rows * p.nch)), block(kLossThreads);
  if (p.norm_parts && a.kind != MVSD_LOSS_PREFERENCE) {
    if (has_list(a))
      hipLaunchKernelGGL((p.K <= kWave       ? loss_teacher_kernel<DT, 1>
                          : p.K <= 2 * kWave ? loss_teacher_kernel<DT, 2>
                                             : loss_teacher_kernel<DT, kMaxTeacher / kWave>),
                         dim3(p.norm_parts), block, 0, stream, p);
    else
      hipLaunchKernelGGL(loss_norm_kernel, dim3(p.norm_parts), block, 0, stream, p);
  }
  if (loss_one_pass(a)) {
    const RowPlan plan = row_plan(a);
    LossParams q = p;
    q.active = plan.active;
    switch (plan.held) {
      case 3: launch_rows<DT, 3>(q, plan, stream); break;
      case 6: launch_rows<DT, 6>(q, plan, stream); break;
      case 10: launch_rows<DT, 10>(q, plan, stream); break;
      case 13: launch_rows<DT, 13>(q, plan, stream); break;
      case 16: launch_rows<DT, 16>(q, plan, stream); break;
      default: launch_rows<DT, kMostHeld>(q, plan, stream); break;
    }
    return hipGetLastError();
  }
  if (has_list(a)) {
    const unsigned lds = (unsigned)((p.chunk + 31) / 32 * 4);
    hipLaunchKernelGGL((loss_stats_kernel<DT, true, false>), grid, block, lds, stream, p);
    hipLaunchKernelGGL(loss_distill_rows_kernel, dim3((unsigned)a.num_rows), block, 0, stream, p);
  } else {
    if (p.entropy)
      hipLaunchKernelGGL((loss_stats_kernel<DT, false, true>), grid, block, 0, stream, p);
    else
      hipLaunchKernelGGL((loss_stats_kernel<DT, false, false>), grid, block, 0, stream, p);
    if (!p.whole)
      hipLaunchKernelGGL(loss_token_rows_kernel<DT>, dim3((unsigned)((a.num_rows + kWaves - 1) / kWaves)), block, 0,
                       stream, p);
  }
  return hipGetLastError();
}

template <int DT>
hipError_t launch_gradient_dt(const LossParams& p, const float* up, int64_t us, const float* up_h, int64_t uhs,
                              hipStream_t stream) {
  // Mostly the gradient is there where a value of 1 is expected: few workgroups look for it (4.6 us).  For another
  // upstream these few form it, at 2.8 TB/s (2048 rows of 151936 bf16: 445 us, distillation of 1024: 233).
  const int64_t chunks = p.a.num_rows * p.nch;
  const dim3 grid((unsigned)(p.a.unit_gradient ? std::min(chunks, (int64_t)num_cus()) : chunks)), block(kLossThreads);
  const bool past = p.a.num_rows * p.V * (DT == MVSD_F32 ? 4 : 2) > kCacheBytes;
  auto launch = [&](auto kernel) { hipLaunchKernelGGL(kernel, grid, block, 0, stream, p, up, us, up_h, uhs); };
  if (has_list(p.a))
    past ? launch(loss_gradient_kernel<DT, true, false, true>) : launch(loss_gradient_kernel<DT, true, false, false>);
  else if (p.entropy)
    past ? launch(loss_gradient_kernel<DT, false, true, true>) : launch(loss_gradient_kernel<DT, false, true, false>);
  else
    past ? launch(loss_gradient_kernel<DT, false, false, true>) : launch(loss_gradient_kernel<DT, false, false, false>);
  return hipGetLastError();
}

}  // namespace

bool loss_one_pass(const mvsd_loss_args& a) {
  if ((a.kind != MVSD_LOSS_DISTILL && a.kind != MVSD_LOSS_POLICY) || a.reduction == MVSD_REDUCE_NONE) return false;
  if (a.vocab_size < 256 || (has_list(a) && a.vocab_size > kMaxMarked)) return false;
  // Where rows are few, workgroups that share a row are faster.  Forward and backward pass, us, one pass / split:
  //   policy, bf16, V = 151936: 96 rows 35.1 / 28.5, 128 36.3 / 31.3, 160 38.4 / 36.0, 256 43.1 / 51.5;
  //     V = 32000: 96 19.0 / 16.7, 128 19.5 / 18.0, 160 20.0 / 20.0, 256 22.7 / 23.1;
  //   distillation, bf16, V = 151936: 64 39.3 / 35.1, 80 40.6 / 39.8, 96 41.5 / 43.3, 160 44.4 / 57.0;
  //     V = 32000: 48 22.9 / 24.1, 80 25.0 / 27.4;
  //   rows of which the registers hold a half, fp32, V = 151936: policy 128 59.4 / 46.8, 512 184 / 180, 2048 656 / 755,
  //     distillation 128 65.8 / 70.8, 2048 655 / 815;
  //   values alone, policy, bf16, V = 151936: 128 22.6 / 20.5, 2048 144 / 221.
  // One border for all of a kind, although a policy's 128 to some 180 rows would be faster split.
  return a.num_rows >= (has_list(a) ? 80 : 128);
}

int64_t loss_workspace_bytes(const mvsd_loss_args& a) {
  const int64_t chunk = chunk_of(a.num_rows, (int)a.vocab_size, a.dtype);
  const int64_t nch = (a.vocab_size + chunk - 1) / chunk;
  return aside_bytes(a) + a.num_rows * nch * (int64_t)sizeof(float4) + kNormParts * 4 + 16 +
         up16(std::max(a.num_rows, a.num_pairs) * 4) + up16(a.num_rows * (has_list(a) ? (int64_t)sizeof(LossTeacher) : 4)) +
         (has_list(a) ? 2 * up16(a.num_rows * a.num_teacher * 4) : 0);
}

int64_t loss_saved_bytes(const mvsd_loss_args& a) {
  return a.num_rows * ((int64_t)sizeof(LossRecord) + (has_list(a) ? a.num_teacher * 8 : 0));
}

hipError_t launch_loss(const mvsd_loss_args& a, hipStream_t stream) {
  const LossParams p = make_params(a);
  hipError_t err = hipSuccess;
  if (a.num_rows > 0) {
    switch (a.dtype) {
      case MVSD_F32: err = launch_dt<MVSD_F32>(p, stream); break;
      case MVSD_BF16: err = launch_dt<MVSD_BF16>(p, stream); break;
      default: err = launch_dt<MVSD_F16>(p, stream); break;
    }
    if (err != hipSuccess) return err;
  }
  if (a.kind == MVSD_LOSS_PREFERENCE && p.norm_parts)
    hipLaunchKernelGGL(loss_norm_kernel, dim3(p.norm_parts), dim3(kLossThreads), 0, stream, p);
  if (a.kind == MVSD_LOSS_PREFERENCE && a.num_pairs > 0)
    hipLaunchKernelGGL(loss_pairs_kernel, dim3((unsigned)a.num_pairs), dim3(kLossThreads), 0, stream, p);
  const int64_t losses = a.kind == MVSD_LOSS_PREFERENCE ? a.num_pairs : a.num_rows;
  if (a.kind != MVSD_LOSS_LOGPROBS && a.reduction != MVSD_REDUCE_NONE &&
      (losses == 0 || a.num_rows == 0 || loss_one_pass(a)))
    hipLaunchKernelGGL(loss_sum_kernel, dim3(1), dim3(1024), 0, stream, p, losses);
  return hipGetLastError();
}

hipError_t launch_loss_gradient(const mvsd_loss_args& a, const float* up, int64_t us, const float* up_h,
                                int64_t uhs, hipStream_t stream) {
  const LossParams p = make_params(a);
  if (a.kind == MVSD_LOSS_POLICY) up_h = up, uhs = us;
  switch (a.dtype) {
    case MVSD_F32: return launch_gradient_dt<MVSD_F32>(p, up, us, up_h, uhs, stream);
    case MVSD_BF16: return launch_gradient_dt<MVSD_BF16>(p, up, us, up_h, uhs, stream);
    default: return launch_gradient_dt<MVSD_F16>(p, up, us, up_h, uhs, stream);
  }
}

}  // namespace mvsd

// ------------------------------------------------------------------ C ABI -----------------------

namespace {

// What every call of these arguments checks first.
int check_sizes(const mvsd_loss_args* a) {
  if (!a || a->kind < MVSD_LOSS_LOGPROBS || a->kind > MVSD_LOSS_PREFERENCE) return MVSD_E_INVALID;
  if (a->dtype != MVSD_F32 && a->dtype != MVSD_BF16 && a->dtype != MVSD_F16) return MVSD_E_INVALID;
  if (a->num_rows < 0 || a->vocab_size < 1) return MVSD_E_INVALID;
  if (a->vocab_size > 0x7fffffff - (1 << 20)) return MVSD_E_RANGE;
  // a launch has fewer than 2^32 threads
  if (a->num_rows > (1 << 23) / ((a->vocab_size / mvsd::kMaxChunk) + 1)) return MVSD_E_RANGE;
  if (a->kind == MVSD_LOSS_DISTILL) {
    if (a->num_teacher < 1) return MVSD_E_INVALID;
    if (a->num_teacher > mvsd::kMaxTeacher) return MVSD_E_RANGE;
  }
  if (a->kind == MVSD_LOSS_PREFERENCE) {
    if (a->num_pairs < 0) return MVSD_E_INVALID;
    if (a->num_pairs > 1 << 23) return MVSD_E_RANGE;
  }
  return MVSD_OK;
}

int check_call(const mvsd_loss_args* a) {
  const int status = check_sizes(a);
  if (status != MVSD_OK) return status;
  const bool rows = a->num_rows > 0;
  if (!(a->temperature >= 1e-6 && a->temperature <= 1e6)) return MVSD_E_INVALID;
  if (a->ids_dtype != MVSD_I32 && a->ids_dtype != MVSD_I64) return MVSD_E_INVALID;
  if (rows && (!a->logits || !a->token_ids || a->inner_rows < 1 || a->stride < 0 || a->outer_stride < 0))
    return MVSD_E_INVALID;
  if (a->reduction < MVSD_REDUCE_SUM || a->reduction > MVSD_REDUCE_NONE) return MVSD_E_INVALID;
  if (a->kind == MVSD_LOSS_DISTILL) {
    if (a->divergence < MVSD_KL_FORWARD || a->divergence > MVSD_JS) return MVSD_E_INVALID;
    if (a->divergence != MVSD_KL_FORWARD && !a->tail) return MVSD_E_INVALID;
    if (rows && !a->teacher_logprobs) return MVSD_E_INVALID;
  }
  if (a->kind == MVSD_LOSS_POLICY) {
    if (rows && !a->advantages) return MVSD_E_INVALID;
    for (const double v : {a->clip_low, a->clip_high, a->kl_coef, a->entropy_coef})
      if (!std::isfinite(v)) return MVSD_E_INVALID;
  }
  if (a->kind == MVSD_LOSS_PREFERENCE) {
    for (const double v : {a->beta, a->margin, a->label_smoothing})
      if (!std::isfinite(v)) return MVSD_E_INVALID;
    if (a->loss_type < MVSD_PREF_SIGMOID || a->loss_type > MVSD_PREF_SQUARED) return MVSD_E_INVALID;
    if (a->num_pairs == 0 && a->reduction == MVSD_REDUCE_NONE && !rows) return MVSD_OK;
    if (!a->cu_num_tokens && a->num_pairs > 0 && a->num_rows % (2 * a->num_pairs)) return MVSD_E_INVALID;
    if (a->loss_type == MVSD_PREF_SQUARED && !(a->beta != 0.0)) return MVSD_E_INVALID;
  }
  return MVSD_OK;
}

bool misaligned(const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 != 0; }

}  // namespace

extern "C" {

int64_t mvsd_loss_saved_bytes(const mvsd_loss_args* args) {
  const int status = check_sizes(args);
  return status != MVSD_OK ? status : mvsd::loss_saved_bytes(*args);
}

int64_t mvsd_loss_workspace_bytes(const mvsd_loss_args* args) {
  const int status = check_sizes(args);
  return status != MVSD_OK ? status : mvsd::loss_workspace_bytes(*args);
}

int mvsd_loss_one_pass(const mvsd_loss_args* args) {
  const int status = check_sizes(args);
  return status != MVSD_OK ? status : mvsd::loss_one_pass(*args) ? 1 : 0;
}

int mvsd_loss_plan(mvsd_loss_args* args) {
  const int status = check_sizes(args);
  if (status != MVSD_OK) return status;
  args->workspace_bytes = mvsd::loss_workspace_bytes(*args);
  args->saved_bytes = mvsd::loss_saved_bytes(*args);
  args->one_pass = mvsd::loss_one_pass(*args) ? 1 : 0;
  return MVSD_OK;
}

int mvsd_row_loss(const mvsd_loss_args* args, mvsd_stream_t stream) {
  const int status = check_call(args);
  if (status != MVSD_OK) return status;
  const mvsd_loss_args& a = *args;
  const bool sums = a.kind != MVSD_LOSS_LOGPROBS;
  const int64_t values = a.kind == MVSD_LOSS_PREFERENCE ? 2 * a.num_pairs : a.num_rows;
  if (sums && !a.loss && (a.reduction != MVSD_REDUCE_NONE || values > 0)) return MVSD_E_INVALID;
  if (a.kind != MVSD_LOSS_DISTILL && values > 0 && !a.logprobs) return MVSD_E_INVALID;
  if (!a.workspace || misaligned(a.workspace) || misaligned(a.saved) ||
      a.workspace_bytes < mvsd::loss_workspace_bytes(a))
    return MVSD_E_WORKSPACE;
  return mvsd::record_hip_error(mvsd::launch_loss(a, (hipStream_t)stream));
}

int mvsd_loss_gradient(const mvsd_loss_args* args, const float* upstream, int64_t up_stride,
                       const float* upstream_entropy, int64_t up_entropy_stride, mvsd_stream_t stream) {
  const int status = check_call(args);
  if (status != MVSD_OK) return status;
  const mvsd_loss_args& a = *args;
  if (a.num_rows == 0) return MVSD_OK;
  if (!a.grad || up_stride < 0 || up_entropy_stride < 0) return MVSD_E_INVALID;
  if (a.unit_gradient && !mvsd::loss_one_pass(a)) return MVSD_E_INVALID;
  const bool none = a.kind == MVSD_LOSS_PREFERENCE && a.num_pairs == 0;  // rows of no pair: zeros
  if (!upstream && a.kind != MVSD_LOSS_LOGPROBS && !none) return MVSD_E_INVALID;
  if (!a.saved || misaligned(a.saved)) return MVSD_E_WORKSPACE;
  return mvsd::record_hip_error(mvsd::launch_loss_gradient(a, upstream, up_stride, upstream_entropy,
                                                           up_entropy_stride, (hipStream_t)stream));
}

}  // extern "C"
