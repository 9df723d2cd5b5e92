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
// Statistics and sums are fp32 (a lane adds at most some hundred terms, then trees); the gradient is
// rounded once, to the logits' dtype.
#include <float.h>

#include <algorithm>

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

// A token id, V for every one of V or more, -1 for every one below 0.
__device__ inline int clean_id(int64_t id, int V) { return id < 0 ? -1 : id >= V ? V : (int)id; }
__device__ inline int token_at(const mvsd_loss_args& a, int64_t i, int V) {
  return clean_id(a.ids_dtype == MVSD_I64 ? static_cast<const int64_t*>(a.token_ids)[i]
                                          : (int64_t) static_cast<const int32_t*>(a.token_ids)[i], V);
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
__device__ inline unsigned marks_at(const uint32_t* bits, int col, int n) {  // n divides 32, col is its multiple
  return (bits[col >> 5] >> (col & 31)) & ((1u << n) - 1u);
}

// One workgroup a chunk of a row: statistics of its rest.
template <int DT, bool LIST, bool ENT>
__global__ __launch_bounds__(kLossThreads) void loss_stats_kernel(LossParams p) {
  constexpr int VEC = Elem<DT>::kVec, U = 4;
  extern __shared__ uint32_t bits[];
  __shared__ Stat s_stat[kWaves];
  const int64_t row = blockIdx.x / p.nch;
  const int part = blockIdx.x - (int)(row * p.nch);
  const int begin = part * p.chunk, end = min(p.V, begin + p.chunk);
  int token = -1;
  if (row_weight(p.a, row) == 0.f) return;
  if constexpr (LIST) {
    for (int i = threadIdx.x; i < (p.chunk + 31) / 32; i += kLossThreads) bits[i] = 0;
    __syncthreads();
    int any = 0;
    for (int k = threadIdx.x; k < p.K; k += kLossThreads) {
      const int id = token_at(p.a, row * p.K + k, p.V);
      any |= id >= 0;
      if (id >= begin && id < end) atomicOr(&bits[(id - begin) >> 5], 1u << ((id - begin) & 31));
    }
    if (!__syncthreads_or(any)) return;
  } else {
    token = token_at(p.a, row, p.V);
    if (token < 0) return;
  }
  const auto* x = logits_row<DT>(p.a, row);
  Stat st = {-INFINITY, 0.f, 0.f};
  for (int col = begin + (int)threadIdx.x * VEC; col < end; col += kLossThreads * VEC * U) {
    float v[U][VEC];
    float m = st.m;
#pragma unroll
    for (int u = 0; u < U; ++u) load_filled<DT>(x, col + u * kLossThreads * VEC, end, v[u]);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int at = col + u * kLossThreads * VEC;
      if constexpr (LIST) {
        const unsigned marks = at < end ? marks_at(bits, at - begin, VEC) : 0;
        if (marks)
#pragma unroll
          for (int e = 0; e < VEC; ++e) v[u][e] = marks >> e & 1 ? -INFINITY : v[u][e];
      } else if (token >= at && token < at + VEC) {
#pragma unroll
        for (int e = 0; e < VEC; ++e) v[u][e] = token == at + e ? -INFINITY : v[u][e];
      }
#pragma unroll
      for (int e = 0; e < VEC; ++e) m = fmaxf(m, v[u][e]);
    }
    const float base = base_of(m);
    const float d = fmaxf((st.m - base) * p.c1, kLeast), f = __builtin_amdgcn_exp2f(d);
    if constexpr (ENT) st.t = (st.t + st.s * d) * f;
    st.s *= f;
    st.m = m;
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        const float y = (v[u][e] - base) * p.c1, w = __builtin_amdgcn_exp2f(y);
        st.s += w;
        if constexpr (ENT) st.t += w * fmaxf(y, kLeast);
      }
  }
  st = wave_join(st, p.c1);
  if (lane_id() == 0) s_stat[wave_id()] = st;
  __syncthreads();
  if (threadIdx.x == 0) {
    st = join(join(s_stat[0], s_stat[1], p.c1), join(s_stat[2], s_stat[3], p.c1), p.c1);
    p.parts[blockIdx.x] = make_float4(st.m, st.s, st.t, 0.f);
  }
}

// ------------------------------------------------------------------ the mean's divisor ----------

// Partial sums of the weights of the rows that are not left out: a wave a row where it has a list.
template <bool LIST>
__global__ __launch_bounds__(kLossThreads) void loss_norm_kernel(LossParams p) {
  __shared__ float scratch[kWaves];
  const int64_t each = (p.a.num_rows + gridDim.x - 1) / gridDim.x;
  const int64_t first = blockIdx.x * each, last = min(p.a.num_rows, first + each);
  float sum[1] = {0.f};
  if constexpr (LIST) {
    for (int64_t row = first + wave_id(); row < last; row += kWaves) {
      bool any = false;
      for (int k = lane_id(); k < p.K; k += kWave) any |= token_at(p.a, row * p.K + k, p.V) >= 0;
      if (__any(any) && lane_id() == 0) sum[0] += row_weight(p.a, row);
    }
  } else {
    for (int64_t row = first + threadIdx.x; row < last; row += kLossThreads)
      if (token_at(p.a, row, p.V) >= 0) sum[0] += row_weight(p.a, row);
  }
  block_sum<1>(sum, scratch);
  if (threadIdx.x == 0) p.norm[blockIdx.x] = sum[0];
}

// What a row's weight is multiplied by, in every thread of a wave.
__device__ inline float mean_factor(const LossParams& p) {
  if (p.a.reduction != MVSD_REDUCE_MEAN || p.norm_parts == 0) return 1.f;
  float sum = 0.f;
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
  const float odds = log_s + (base - x) * p.inv_t;  // of all others against the token
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

__device__ inline PolicyRow policy_row(const mvsd_loss_args& a, int64_t row, float lp, float H) {
  PolicyRow o;
  const float A = a.advantages[row];
  const float r = a.old_logprobs ? expf(lp - a.old_logprobs[row]) : lp == lp ? 1.f : lp;
  const float free = r * A;
  const float bound = fminf(fmaxf(r, (float)(1.0 - a.clip_low)), (float)(1.0 + a.clip_high)) * A;
  const bool clipped = free > bound;
  o.loss = clipped ? -bound : -free;
  o.c = clipped ? 0.f : -free;
  o.kl = 0.f;
  if (a.ref_logprobs) {
    const float d = a.ref_logprobs[row] - lp, e1 = expm1f(d);
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

// A wave a row: the chunks' statistics together, then the row's loss.
template <int DT>
__global__ __launch_bounds__(kLossThreads) void loss_token_rows_kernel(LossParams p) {
  const int64_t row = (int64_t)blockIdx.x * kWaves + wave_id();
  if (row >= p.a.num_rows) return;
  const mvsd_loss_args& a = p.a;
  const float mean = mean_factor(p);
  const int token = token_at(a, row, p.V);
  const float w = row_weight(a, row);
  const bool out = token < 0 || w == 0.f;
  TokenRow r;
  PolicyRow o = {0.f, 0.f, 0.f};
  r.lp = r.H = 0.f;
  r.rec = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0};
  if (!out) {
    const float x = token < p.V ? Elem<DT>::cvt(logits_row<DT>(a, row)[token]) : NAN;
    Stat st = {-INFINITY, 0.f, 0.f};
    for (int i = lane_id(); i < p.nch; i += kWave) {
      const float4 v = p.parts[row * p.nch + i];
      st = join(st, {v.x, v.y, v.z}, p.c1);
    }
    st = wave_join(st, p.c1);
    r = token_row(p, st, x);
    r.rec.pair = 0;
    r.rec.c = 1.f;
    r.rec.cH = 1.f;
    if (a.kind == MVSD_LOSS_POLICY) {
      o = policy_row(a, row, r.lp, r.H);
      r.rec.c = o.c * w * mean;
      r.rec.cH = -(float)a.entropy_coef * w * mean;
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
    p.row_loss[row] = out ? 0.f : o.loss * w * mean;
    if (a.kl) a.kl[row] = o.kl;
  }
  if (p.records) p.records[row] = r.rec;
}

// A workgroup a pair: the sums over its two sequences, its loss, its rows' factors.
__global__ __launch_bounds__(kLossThreads) void loss_pairs_kernel(LossParams p) {
  __shared__ float scratch[4 * kWaves];
  const mvsd_loss_args& a = p.a;
  const int64_t pair = blockIdx.x, B = a.num_pairs, N = a.num_rows;
  float w = a.weights ? a.weights[pair] : 1.f;
  if (a.reduction == MVSD_REDUCE_MEAN) {
    float all[1] = {0.f};
    for (int64_t i = threadIdx.x; i < B; i += kLossThreads) all[0] += a.weights ? a.weights[i] : 1.f;
    block_sum<1>(all, scratch);
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

template <int T>
struct DistillScratch {
  int ids[kMaxTeacher];
  float red[4 * (T / kWave)];
  double sum[T / kWave];
};

__device__ inline double wave_sum_f64(double v) {
#pragma unroll
  for (int d = 1; d < kWave; d *= 2) v += __shfl_xor(v, d);
  return v;
}

// One row's loss by a workgroup of T threads, from the statistics of its rest.  Writes the gradients of the
// given tokens (over, over_ids: -1 where an entry does not count) and returns the loss; *k is the record's.
// `weight` is the row's, after the mean.
template <int DT, int T>
__device__ inline float distill_row(const LossParams& p, int64_t row, Stat st, float weight,
                                    DistillScratch<T>& sm, float* over, int32_t* over_ids, float* k_out) {
  constexpr int NW = T / kWave, E = (kMaxTeacher + T - 1) / T;
  const mvsd_loss_args& a = p.a;
  const int tid = threadIdx.x, K = p.K;
  const auto* xrow = logits_row<DT>(a, row);
  int id[E];
  float x[E], v[E];
#pragma unroll
  for (int i = 0; i < E; ++i) {
    const int k = i * T + tid;
    id[i] = k < K ? token_at(a, row * K + k, p.V) : -1;
    x[i] = id[i] < 0 ? -INFINITY : id[i] < p.V ? Elem<DT>::cvt(xrow[id[i]]) : NAN;
    if (x[i] == INFINITY) x[i] = NAN;
    v[i] = id[i] < 0 ? -INFINITY : a.teacher_logprobs[row * K + k];
    if (k < K) sm.ids[k] = id[i];
  }
  __syncthreads();
  // an id that stands before does not count
#pragma unroll
  for (int i = 0; i < E; ++i) {
    const int k = i * T + tid;
    if (i * T >= K) break;
    bool twice = false;
    const int last = min(K, (i + 1) * T);
    for (int j = 0; j < last; ++j) twice |= j < k && sm.ids[j] == id[i];
    if (twice) id[i] = -1, x[i] = v[i] = -INFINITY;
  }
  // the row's maximum, the teacher's, and the number of entries
  float top[2] = {st.m, -INFINITY}, count[1] = {0.f};
  double mass = 0.0;
#pragma unroll
  for (int i = 0; i < E; ++i) {
    top[0] = fmaxf(top[0], x[i]);
    top[1] = fmaxf(top[1], v[i]);
    count[0] += id[i] >= 0 ? 1.f : 0.f;
    if (id[i] >= 0 && a.tail) mass += exp((double)v[i]);
  }
  block_max<2, NW>(top, sm.red);
  block_sum<1, NW>(count, sm.red);
  const float base = base_of(top[0]), rest_base = base_of(st.m);
  float q[E], log_q[E], rest_q = 0.f;
  bool tail = false;
  if (a.tail) {
    mass = wave_sum_f64(mass);
    if (lane_id() == 0) sm.sum[wave_id()] = mass;
    __syncthreads();
    mass = 0.0;
#pragma unroll
    for (int w = 0; w < NW; ++w) mass += sm.sum[w];
    tail = (int)count[0] < p.V;
    rest_q = tail ? (float)fmax(1.0 - mass, 0x1p-24) : 0.f;
    if (mass != mass) rest_q = NAN;
#pragma unroll
    for (int i = 0; i < E; ++i) {
      log_q[i] = v[i];
      q[i] = expf(v[i]);
    }
  } else {
    float sum[1] = {0.f};
    const float vb = base_of(top[1]);
#pragma unroll
    for (int i = 0; i < E; ++i) {
      log_q[i] = (v[i] - vb) * p.inv_t;
      q[i] = expf(log_q[i]);
      sum[0] += q[i];
    }
    block_sum<1, NW>(sum, sm.red);
    const float lg = logf(sum[0]), inv = 1.f / sum[0];
#pragma unroll
    for (int i = 0; i < E; ++i) {
      log_q[i] -= lg;
      q[i] *= inv;
    }
  }
  // the student's normaliser
  float z[1] = {0.f};
#pragma unroll
  for (int i = 0; i < E; ++i) z[0] += expf((x[i] - base) * p.inv_t);
  block_sum<1, NW>(z, sm.red);
  const float rest_d = st.m == -INFINITY ? 0.f : (rest_base - base) * p.inv_t;
  const float log_z = logf(z[0] + st.s * expf(rest_d));
  const float rest_lp = rest_d + logf(st.s) - log_z, rest_p = st.s > 0.f ? expf(rest_lp) : st.s;
  // the divergence's terms, and p dL/dp of every outcome
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
  float both[2] = {0.f, 0.f}, pr[E], pd[E];
#pragma unroll
  for (int i = 0; i < E; ++i) {
    const float lp = (x[i] - base) * p.inv_t - log_z;
    float term = 0.f;
    pr[i] = expf(lp);
    pd[i] = 0.f;
    if (id[i] >= 0) outcome(q[i], log_q[i], pr[i], lp, term, pd[i]);
    both[0] += term;
    both[1] += pd[i];
  }
  block_sum<2, NW>(both, sm.red);
  float rest_pd = 0.f;
  if (tail) {
    float term;
    outcome(rest_q, logf(rest_q), rest_p, rest_lp, term, rest_pd);
    both[0] += term;
    both[1] += rest_pd;
  }
  const float f = weight * p.inv_t;
  *k_out = st.s == 0.f ? 0.f : -f * (rest_pd - rest_p * both[1]) / st.s;
  if (over) {
#pragma unroll
    for (int i = 0; i < E; ++i) {
      const int k = i * T + tid;
      if (k < K) {
        over[k] = f * (pd[i] - pr[i] * both[1]);
        over_ids[k] = id[i] < p.V ? id[i] : -1;
      }
    }
  }
  return both[0] * weight;
}

// A workgroup a row.
template <int DT>
__global__ __launch_bounds__(kLossThreads) void loss_distill_rows_kernel(LossParams p) {
  __shared__ DistillScratch<kLossThreads> sm;
  const int64_t row = blockIdx.x;
  const mvsd_loss_args& a = p.a;
  const float w = row_weight(a, row) * mean_factor(p);
  bool any = false;
  for (int k = threadIdx.x; k < p.K; k += kLossThreads) any |= token_at(a, row * p.K + k, p.V) >= 0;
  const bool out = !__syncthreads_or(any) || row_weight(a, row) == 0.f;
  float loss = 0.f;
  LossRecord rec = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0};
  if (!out) {
    Stat st = {-INFINITY, 0.f, 0.f};
    for (int i = lane_id(); i < p.nch; i += kWave) {
      const float4 v = p.parts[row * p.nch + i];
      st = join(st, {v.x, v.y, v.z}, p.c1);
    }
    st = wave_join(st, p.c1);
    rec.M = base_of(st.m);
    rec.c = 1.f;
    loss = distill_row<DT, kLossThreads>(p, row, st, w, sm, p.records ? p.over + row * p.K : nullptr,
                                         p.over_ids + row * p.K, &rec.k);
  }
  if (threadIdx.x == 0) {
    p.row_loss[row] = loss;
    if (p.records) p.records[row] = rec;
  }
}

// ------------------------------------------------------------------ sums ------------------------

// loss[0] = sum of n values, in one order.
__global__ __launch_bounds__(1024) void loss_sum_kernel(float* loss, const float* v, int64_t n) {
  __shared__ float scratch[16];
  float sum[1] = {0.f};
  for (int64_t i = threadIdx.x; i < n; i += 1024) sum[0] += v[i];
  block_sum<1, 16>(sum, scratch);
  if (threadIdx.x == 0) loss[0] = sum[0];
}

// ------------------------------------------------------------------ the gradient ----------------

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

template <int DT>
__device__ inline void store_filled(typename Elem<DT>::storage* row, int col, int end,
                                    const float (&g)[Elem<DT>::kVec]) {
  constexpr int VEC = Elem<DT>::kVec;
  if (col + VEC <= end) {
    *reinterpret_cast<Vec16<DT>*>(row + col) = pack_vec<DT>(g);
  } else {
#pragma unroll
    for (int e = 0; e < VEC; ++e)
      if (col + e < end) row[col + e] = to_storage<DT>(g[e]);
  }
}

// One workgroup a chunk of a row, from its record.
template <int DT, bool LIST, bool ENT>
__global__ __launch_bounds__(kLossThreads) void loss_gradient_kernel(LossParams p, const float* up, int64_t us,
                                                                     const float* up_h, int64_t uhs) {
  constexpr int VEC = Elem<DT>::kVec;
  const int64_t row = blockIdx.x / p.nch;
  const int part = blockIdx.x - (int)(row * p.nch);
  const int begin = part * p.chunk, end = min(p.V, begin + p.chunk);
  const LossRecord rec = p.records[row];
  const int64_t n = p.a.kind == MVSD_LOSS_PREFERENCE ? rec.pair : row;
  const float g = rec.c == 0.f || !up ? 0.f : rec.c * up[n * us];
  const float gH = !ENT || rec.cH == 0.f || !up_h ? 0.f : rec.cH * up_h[n * uhs];
  auto* out = static_cast<typename Elem<DT>::storage*>(p.a.grad) + row * p.V;
  if (g == 0.f && gH == 0.f) {
    const float zero[VEC] = {};
    for (int col = begin + (int)threadIdx.x * VEC; col < end; col += kLossThreads * VEC)
      store_filled<DT>(out, col, end, zero);
    return;
  }
  const auto* x = logits_row<DT>(p.a, row);
  const float ka = -rec.k * (g + gH * rec.h), kb = -rec.k * gH * kLn2;
  const int token = LIST ? -1 : token_at(p.a, row, p.V);
  const float at_token = g * rec.o1 + gH * rec.o2;
  for (int col = begin + (int)threadIdx.x * VEC; col < end; col += kLossThreads * VEC) {
    float v[VEC];
    load_filled<DT>(x, col, end, v);
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
      const float y = (v[e] - rec.M) * p.c1, w = __builtin_amdgcn_exp2f(y);
      v[e] = w * (ENT ? fmaf(kb, fmaxf(y, kLeast), ka) : ka);
    }
    if (!LIST && token >= col && token < col + VEC) {
#pragma unroll
      for (int e = 0; e < VEC; ++e) v[e] = token == col + e ? at_token : v[e];
    }
    store_filled<DT>(out, col, end, v);
  }
  if constexpr (LIST) {
    __syncthreads();
    for (int k = threadIdx.x; k < p.K; k += kLossThreads) {
      const int id = p.over_ids[row * p.K + k];
      if (id >= begin && id < end) out[id] = to_storage<DT>(g * p.over[row * p.K + k]);
    }
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
  p.parts = reinterpret_cast<float4*>(w);
  w += N * p.nch * sizeof(float4);
  p.norm = reinterpret_cast<float*>(w);
  w += kNormParts * sizeof(float);
  p.row_loss = a.reduction == MVSD_REDUCE_NONE && a.loss ? a.loss : reinterpret_cast<float*>(w);
  w += up16(std::max(N, a.num_pairs) * 4);
  p.row_lp = reinterpret_cast<float*>(w);
  if (a.saved) {
    p.records = static_cast<LossRecord*>(a.saved);
    p.over = reinterpret_cast<float*>(p.records + N);
    p.over_ids = reinterpret_cast<int32_t*>(p.over + N * p.K);
  }
  const bool weighs = a.kind == MVSD_LOSS_DISTILL || a.kind == MVSD_LOSS_POLICY;
  p.norm_parts = weighs && a.reduction == MVSD_REDUCE_MEAN
                     ? (int)std::min(N / 64 + 1, (int64_t)kNormParts)
                     : 0;
  return p;
}

template <int DT>
hipError_t launch_dt(const LossParams& p, hipStream_t stream) {
  const mvsd_loss_args& a = p.a;
  const dim3 grid((unsigned)(a.num_rows * p.nch)), block(kLossThreads);
  if (p.norm_parts) {
    if (has_list(a))
      hipLaunchKernelGGL(loss_norm_kernel<true>, dim3(p.norm_parts), block, 0, stream, p);
    else
      hipLaunchKernelGGL(loss_norm_kernel<false>, dim3(p.norm_parts), block, 0, stream, p);
  }
  if (has_list(a)) {
    const unsigned lds = (unsigned)((p.chunk + 31) / 32 * 4);
    hipLaunchKernelGGL((loss_stats_kernel<DT, true, false>), grid, block, lds, stream, p);
    hipLaunchKernelGGL(loss_distill_rows_kernel<DT>, dim3((unsigned)a.num_rows), block, 0, stream, p);
  } else {
    if (p.entropy)
      hipLaunchKernelGGL((loss_stats_kernel<DT, false, true>), grid, block, 0, stream, p);
    else
      hipLaunchKernelGGL((loss_stats_kernel<DT, false, false>), grid, block, 0, stream, p);
    hipLaunchKernelGGL(loss_token_rows_kernel<DT>, dim3((unsigned)((a.num_rows + kWaves - 1) / kWaves)), block, 0,
                       stream, p);
  }
  return hipGetLastError();
}

template <int DT>
hipError_t launch_gradient_dt(const LossParams& p, const float* up, int64_t us, const float* up_h, int64_t uhs,
                              hipStream_t stream) {
  const dim3 grid((unsigned)(p.a.num_rows * p.nch)), block(kLossThreads);
  if (has_list(p.a))
    hipLaunchKernelGGL((loss_gradient_kernel<DT, true, false>), grid, block, 0, stream, p, up, us, up_h, uhs);
  else if (p.entropy)
    hipLaunchKernelGGL((loss_gradient_kernel<DT, false, true>), grid, block, 0, stream, p, up, us, up_h, uhs);
  else
    hipLaunchKernelGGL((loss_gradient_kernel<DT, false, false>), grid, block, 0, stream, p, up, us, up_h, uhs);
  return hipGetLastError();
}

}  // namespace

int64_t loss_workspace_bytes(const mvsd_loss_args& a) {
  const int64_t chunk = chunk_of(a.num_rows, (int)a.vocab_size, a.dtype);
  const int64_t nch = (a.vocab_size + chunk - 1) / chunk;
  return a.num_rows * nch * (int64_t)sizeof(float4) + kNormParts * 4 +
         up16(std::max(a.num_rows, a.num_pairs) * 4) + up16(a.num_rows * 4);
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
  int64_t losses = a.num_rows;
  if (a.kind == MVSD_LOSS_PREFERENCE) {
    losses = a.num_pairs;
    if (losses > 0) hipLaunchKernelGGL(loss_pairs_kernel, dim3((unsigned)losses), dim3(kLossThreads), 0, stream, p);
  }
  if (a.kind != MVSD_LOSS_LOGPROBS && a.reduction != MVSD_REDUCE_NONE)
    hipLaunchKernelGGL(loss_sum_kernel, dim3(1), dim3(1024), 0, stream, a.loss, p.row_loss, losses);
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
    if (a->num_pairs > 0x3fffffff) return MVSD_E_RANGE;
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
  if (a->kind == MVSD_LOSS_POLICY && rows && !a->advantages) return MVSD_E_INVALID;
  if (a->kind == MVSD_LOSS_PREFERENCE) {
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
  if (!upstream && a.kind != MVSD_LOSS_LOGPROBS) return MVSD_E_INVALID;
  if (!a.saved || misaligned(a.saved)) return MVSD_E_WORKSPACE;
  return mvsd::record_hip_error(mvsd::launch_loss_gradient(a, upstream, up_stride, upstream_entropy,
                                                           up_entropy_stride, (hipStream_t)stream));
}

}  // extern "C"
