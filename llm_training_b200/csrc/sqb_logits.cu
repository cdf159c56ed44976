// Token log-probabilities of logits and the two losses that train on them
// (include/sqb_train.h): a preference loss over pairs of answers and a clipped
// policy loss with a KL term, forward and backward.
//
// A row of V logits x with target t:  m = max x,  s = sum exp(x - m),
//   logp = (x_t - m) - log s,   d logp / d x_c = [c == t] - exp(x_c - m) / s.
// (m, s) is kept for the backward instead of log-sum-exp: exp(x - m) / s has the
// rounding of one subtraction of nearby numbers, exp(x - lse) that of lse itself.
// The row's sum is fp32 over at most a few hundred terms a thread and a tree over
// threads; logp, and everything per token or per sequence above it, is computed in
// 64 bits by one thread, since a sequence's sum of logps is hundreds to thousands
// and the losses are made of small differences of such sums.
//
// All kernels over logits are bound by HBM: they read each row once, all of its
// loads independent, and rows whose target is ignored are not read at all.

#include <cuda_bf16.h>
#include <math.h>
#include <stdint.h>

#include "sqb_train.h"

namespace sqb {
namespace logits {
namespace {

constexpr float kLog2e = 1.4426950408889634f;

struct View {  // (S, T, V) logits, unit stride on V; strides in elements
  int64_t T, V, ss, st;
};

__device__ __forceinline__ int64_t row_offset(int64_t r, int64_t T, int64_t ss, int64_t st) {
  const int64_t s = r / T;
  return s * ss + (r - s * T) * st;
}

__device__ __forceinline__ float to_f(float x) { return x; }
__device__ __forceinline__ float to_f(__nv_bfloat16 x) { return __bfloat162float(x); }
template <typename T>
__device__ __forceinline__ T from_f(float x);
template <>
__device__ __forceinline__ float from_f<float>(float x) {
  return x;
}
template <>
__device__ __forceinline__ __nv_bfloat16 from_f<__nv_bfloat16>(float x) {
  return __float2bfloat16_rn(x);
}

__device__ __forceinline__ float exp2_approx(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// exp(x - m): the difference first, so that no rounding of m * log2(e) is shared by
// the whole row.
__device__ __forceinline__ float exp_diff(float x, float m) {
  return exp2_approx((x - m) * kLog2e);
}

// The max a running sum is taken against: 0 while every element so far is -inf
// (their exponentials are then 0, and a NaN still shows).
__device__ __forceinline__ float finite_ref(float m) { return m == -INFINITY ? 0.f : m; }

// Adds a sum over another part of the row, (m2, s2), to (m, s).
__device__ __forceinline__ void join(float& m, float& s, float m2, float s2) {
  const float top = fmaxf(m, m2), ref = finite_ref(top);
  s = s * exp_diff(m, ref) + s2 * exp_diff(m2, ref);
  m = top;
}

// Elements before the first 16-byte boundary of `p`, at most V.
template <typename T>
__device__ __forceinline__ int64_t head_of(const T* p, int64_t V) {
  const int64_t h = ((16 - (reinterpret_cast<uintptr_t>(p) & 15)) & 15) / sizeof(T);
  return h < V ? h : V;
}

// (max, sum of exp(x - max)) over a row, the same in every thread of the CTA.
// red: 2 * 32 floats of shared memory.
template <typename T, int kThreads>
__device__ void row_stats(const T* row, int64_t V, float* red, float& m_out, float& s_out) {
  constexpr int kN = 16 / sizeof(T);
  const int64_t head = head_of(row, V), nvec = (V - head) / kN;
  float m = -INFINITY, s = 0.f;
  auto one = [&](float x) { join(m, s, x, 1.f); };
  if (threadIdx.x < head) one(to_f(row[threadIdx.x]));
  const T* body = row + head;
  for (int64_t i = threadIdx.x; i < nvec; i += kThreads) {
    const uint4 u = *reinterpret_cast<const uint4*>(body + i * kN);
    const T* e = reinterpret_cast<const T*>(&u);
    float x[kN], top = m;
#pragma unroll
    for (int j = 0; j < kN; ++j) {
      x[j] = to_f(e[j]);
      top = fmaxf(top, x[j]);
    }
    const float ref = finite_ref(top);
    s *= exp_diff(m, ref);
#pragma unroll
    for (int j = 0; j < kN; ++j) s += exp_diff(x[j], ref);
    m = top;
  }
  const int64_t tail = head + nvec * kN + threadIdx.x;
  if (tail < V) one(to_f(row[tail]));
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const float m2 = __shfl_xor_sync(0xffffffffu, m, o), s2 = __shfl_xor_sync(0xffffffffu, s, o);
    join(m, s, m2, s2);
  }
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (lane == 0) {
    red[warp] = m;
    red[32 + warp] = s;
  }
  __syncthreads();
  m = lane < kThreads / 32 ? red[lane] : -INFINITY;
  s = lane < kThreads / 32 ? red[32 + lane] : 0.f;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const float m2 = __shfl_xor_sync(0xffffffffu, m, o), s2 = __shfl_xor_sync(0xffffffffu, s, o);
    join(m, s, m2, s2);
  }
  m_out = m;
  s_out = s;
}

// drow[c] = g * ([c == t] - exp(row[c] - m) / s) for c < V, by the whole CTA.
template <typename T, int kThreads>
__device__ void write_grad(const T* row, T* drow, int64_t V, int64_t t, float m, float s,
                           float g) {
  constexpr int kN = 16 / sizeof(T);
  const float k = -g / s;
  auto grad = [&](float x, int64_t c) {
    const float p = k * exp_diff(x, m);
    return from_f<T>(c == t ? g + p : p);
  };
  if (((reinterpret_cast<uintptr_t>(row) ^ reinterpret_cast<uintptr_t>(drow)) & 15) != 0) {
    for (int64_t c = threadIdx.x; c < V; c += kThreads) drow[c] = grad(to_f(row[c]), c);
    return;
  }
  const int64_t head = head_of(row, V), nvec = (V - head) / kN;
  if (threadIdx.x < head) drow[threadIdx.x] = grad(to_f(row[threadIdx.x]), threadIdx.x);
  for (int64_t i = threadIdx.x; i < nvec; i += kThreads) {
    const int64_t c = head + i * kN;
    const uint4 u = *reinterpret_cast<const uint4*>(row + c);
    const T* e = reinterpret_cast<const T*>(&u);
    uint4 o;
    T* d = reinterpret_cast<T*>(&o);
#pragma unroll
    for (int j = 0; j < kN; ++j) d[j] = grad(to_f(e[j]), c + j);
    *reinterpret_cast<uint4*>(drow + c) = o;
  }
  const int64_t tail = head + nvec * kN + threadIdx.x;
  if (tail < V) drow[tail] = grad(to_f(row[tail]), tail);
}

template <typename T, int kThreads>
__device__ void write_zeros(T* drow, int64_t V) {
  constexpr int kN = 16 / sizeof(T);
  const int64_t head = head_of(drow, V), nvec = (V - head) / kN;
  if (threadIdx.x < head) drow[threadIdx.x] = from_f<T>(0.f);
  for (int64_t i = threadIdx.x; i < nvec; i += kThreads)
    *reinterpret_cast<uint4*>(drow + head + i * kN) = make_uint4(0, 0, 0, 0);
  const int64_t tail = head + nvec * kN + threadIdx.x;
  if (tail < V) drow[tail] = from_f<T>(0.f);
}

// Log-probability of target t in 64 bits (NaN for a t past the vocabulary).
template <typename T>
__device__ __forceinline__ double logp_of(const T* row, int64_t V, int64_t t, float m, float s) {
  if (t >= V) return NAN;
  return ((double)to_f(row[t]) - (double)m) - log((double)s);
}

constexpr int kThreads = 512;

template <typename T>
__global__ void __launch_bounds__(kThreads)
    logp_fwd_kernel(const T* x, const int64_t* targets, float* logp, double* logp64,
                    float2* stats, View v) {
  __shared__ float red[64];
  const int64_t r = blockIdx.x, t = targets[r];
  float m = 0.f, s = 1.f;
  double lp = 0.0;
  if (t >= 0) {
    const T* row = x + row_offset(r, v.T, v.ss, v.st);
    row_stats<T, kThreads>(row, v.V, red, m, s);
    if (threadIdx.x == 0) lp = logp_of(row, v.V, t, m, s);
  }
  if (threadIdx.x == 0) {
    stats[r] = make_float2(m, s);
    if (logp) logp[r] = (float)lp;
    if (logp64) logp64[r] = lp;
  }
}

template <typename T>
__global__ void __launch_bounds__(kThreads)
    logp_bwd_kernel(const T* x, const int64_t* targets, const float2* stats, const float* g_row,
                    const float* scale, T* dx, View v, int64_t dss, int64_t dst) {
  const int64_t r = blockIdx.x, t = targets[r];
  T* drow = dx + row_offset(r, v.T, dss, dst);
  const float2 ms = stats[r];
  float g = t < 0 ? 0.f : g_row[r];
  if (t >= 0 && scale) g *= *scale;
  if (t >= v.V) g = NAN;
  // a zero factor (an ignored token, a clipped one) makes a zero row, which needs no
  // logits - unless they hold a NaN or an infinity, which the sum then shows
  if (t < 0 || (g == 0.f && isfinite(ms.x) && isfinite(ms.y)))
    write_zeros<T, kThreads>(drow, v.V);
  else
    write_grad<T, kThreads>(x + row_offset(r, v.T, v.ss, v.st), drow, v.V, t, ms.x, ms.y, g);
}

// Per-row terms of the policy loss.  In all of it NaN arguments give NaN results.
struct Policy {
  const float* old_logp;  // (N), null: the current ones (ratio 1)
  const float* ref_logp;  // (N), null: no KL term
  const float* adv;       // (N), or (S) if by_seq
  const int32_t* seq;     // row -> sequence of a packed batch, null: r / T
  const float* weight;    // (N), 0 for a row that is not counted
  bool by_seq;
  double lo, hi, kl_coef;  // ratio held in [lo, hi]
};

// term: {-min(ratio A, held A), KL, 1 if the held one counts}; returns d loss / d logp.
__device__ double policy_terms(const Policy& p, int64_t r, int64_t T, double lp, double* term) {
  const int64_t a = p.by_seq ? (p.seq ? p.seq[r] : r / T) : r;
  const double A = p.adv[a];
  const double ratio = p.old_logp ? exp(lp - (double)p.old_logp[r]) : exp(lp - lp);
  const double kept = ratio < p.lo ? p.lo : ratio > p.hi ? p.hi : ratio;
  const double open = ratio * A, held = kept * A;
  const bool clipped = held < open;
  term[0] = clipped ? -held : -open;
  term[2] = clipped ? 1.0 : 0.0;
  double d = clipped ? 0.0 : -open;
  term[1] = 0.0;
  if (p.ref_logp) {
    const double gap = (double)p.ref_logp[r] - lp;
    term[1] = expm1(gap) - gap;
    d -= p.kl_coef * expm1(gap);
  }
  return d;
}

// One row of the policy loss: log-probability, terms and d loss / d logp; with dx,
// also the row's gradient times `scale`, the row read again where it is still in L2.
template <typename T>
__global__ void __launch_bounds__(kThreads)
    policy_kernel(const T* x, const int64_t* targets, Policy p, float* logp, float2* stats,
                  float* g_row, double* terms, T* dx, float scale, View v, int64_t dss,
                  int64_t dst, int64_t N) {
  __shared__ float red[64];
  __shared__ float bcast;
  const int64_t r = blockIdx.x, t = targets[r];
  const float w = p.weight[r];
  T* drow = dx ? dx + row_offset(r, v.T, dss, dst) : nullptr;
  if (t < 0 || w == 0.f) {
    if (threadIdx.x == 0) {
      if (logp) logp[r] = 0.f;
      if (stats) stats[r] = make_float2(0.f, 1.f);
      if (g_row) g_row[r] = 0.f;
      terms[r] = terms[N + r] = terms[2 * N + r] = 0.0;
    }
    if (dx) write_zeros<T, kThreads>(drow, v.V);
    return;
  }
  const T* row = x + row_offset(r, v.T, v.ss, v.st);
  float m, s;
  row_stats<T, kThreads>(row, v.V, red, m, s);
  if (threadIdx.x == 0) {
    double term[3];
    const double lp = logp_of(row, v.V, t, m, s);
    const float g = (float)(policy_terms(p, r, v.T, lp, term) * (double)w);
    if (logp) logp[r] = (float)lp;
    if (stats) stats[r] = make_float2(m, s);
    if (g_row) g_row[r] = g;
    terms[r] = term[0];
    terms[N + r] = term[1];
    terms[2 * N + r] = term[2];
    bcast = g * scale;
  }
  if (!dx) return;
  __syncthreads();
  const float g = bcast;
  if (g == 0.f && isfinite(m) && isfinite(s))
    write_zeros<T, kThreads>(drow, v.V);
  else
    write_grad<T, kThreads>(row, drow, v.V, t, m, s, g);
}

// ---- sequences ------------------------------------------------------------------

// Block-wide sum in a fixed order, the same in every thread.  red: 32 doubles.
__device__ double block_sum(double v, double* red) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  __syncthreads();  // red may still be read by a previous reduction
  if (lane == 0) red[warp] = v;
  __syncthreads();
  v = lane < (int)blockDim.x / 32 ? red[lane] : 0.0;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// Rows [a, b) of sequence s: cu's, held inside [0, N], or s * T and on.
__device__ __forceinline__ void rows_of(const int64_t* cu, int64_t s, int64_t T, int64_t N,
                                        int64_t& a, int64_t& b) {
  if (cu) {
    a = min(max(cu[s], (int64_t)0), N);
    b = min(max(cu[s + 1], a), N);
  } else {
    a = s * T;
    b = a + T;
  }
}

// log(1 + exp(z)) and 1 / (1 + exp(-z)) without overflow
__device__ __forceinline__ double softplus(double z) { return fmax(z, 0.0) + log1p(exp(-fabs(z))); }
__device__ __forceinline__ double sigmoid(double z) {
  const double e = exp(-fabs(z));
  return (z >= 0 ? 1.0 : e) / (1.0 + e);
}

constexpr int kSeqThreads = 256;

// One CTA per pair (chosen sequence p, rejected sequence P + p): both sums of
// logps, the pair's loss, and d loss / d logp of each of its rows.
__global__ void __launch_bounds__(kSeqThreads)
    preference_pair_kernel(const double* logp, const int64_t* cu, const float* ref, int64_t P,
                           int64_t T, int64_t N, double beta, double smooth, double* pair_loss,
                           float* rewards, float* g_row) {
  __shared__ double red[32];
  const int64_t p = blockIdx.x;
  int64_t a[2], b[2];
  double ratio[2];
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    rows_of(cu, p + k * P, T, N, a[k], b[k]);
    double v = 0.0;
    for (int64_t r = a[k] + threadIdx.x; r < b[k]; r += kSeqThreads) v += logp[r];
    ratio[k] = block_sum(v, red) - (ref ? (double)ref[p + k * P] : 0.0);
  }
  const double z = beta * (ratio[0] - ratio[1]);
  const double dz = smooth * sigmoid(z) - (1.0 - smooth) * sigmoid(-z);
  const float g = (float)(dz * beta / (double)P);
  if (threadIdx.x == 0) {
    pair_loss[p] = (1.0 - smooth) * softplus(-z) + smooth * softplus(z);
    rewards[p] = (float)(beta * ratio[0]);
    rewards[P + p] = (float)(beta * ratio[1]);
  }
#pragma unroll
  for (int k = 0; k < 2; ++k)
    for (int64_t r = a[k] + threadIdx.x; r < b[k]; r += kSeqThreads) g_row[r] = k ? -g : g;
}

__global__ void __launch_bounds__(kSeqThreads)
    preference_mean_kernel(const double* pair_loss, int64_t P, float* loss) {
  __shared__ double red[32];
  double v = 0.0;
  for (int64_t p = threadIdx.x; p < P; p += kSeqThreads) v += pair_loss[p];
  v = block_sum(v, red);
  if (threadIdx.x == 0) *loss = (float)(v / (double)P);
}

constexpr int kWeightThreads = 1024;

// Weight of every row in the policy loss, and the sequence of every row of a packed
// batch (-1 for a row outside every sequence).  One CTA: the counts of all sequences
// are needed before the first weight, and 64K targets are 512 KB.
__global__ void __launch_bounds__(kWeightThreads)
    policy_weights_kernel(const int64_t* targets, const int64_t* cu, int64_t S, int64_t T,
                          int64_t N, bool per_sequence, int32_t* counts, float* weight,
                          int32_t* seq) {
  __shared__ double red[32];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  for (int64_t s = warp; s < S; s += kWeightThreads / 32) {
    int64_t a, b;
    rows_of(cu, s, T, N, a, b);
    int n = 0;
    for (int64_t r = a + lane; r < b; r += 32) n += targets[r] >= 0;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) n += __shfl_xor_sync(0xffffffffu, n, o);
    if (lane == 0) counts[s] = n;
  }
  __syncthreads();
  double total = 0.0;
  for (int64_t s = threadIdx.x; s < S; s += kWeightThreads)
    total += per_sequence ? (counts[s] > 0 ? 1.0 : 0.0) : (double)counts[s];
  total = block_sum(total, red);  // whole numbers: exact
  for (int64_t r = threadIdx.x; r < N; r += kWeightThreads) {
    int64_t s = r / (T > 0 ? T : 1);
    bool inside = true;
    if (cu) {  // the last s with cu[s] <= r
      int64_t lo = 0, hi = S;
      while (lo < hi) {
        const int64_t mid = (lo + hi) / 2;
        if (cu[mid + 1] <= r)
          lo = mid + 1;
        else
          hi = mid;
      }
      s = lo;
      inside = s < S && cu[s] <= r;
      seq[r] = inside ? (int32_t)s : -1;
    }
    float w = 0.f;
    if (inside && targets[r] >= 0)
      w = (float)(1.0 / (per_sequence ? total * (double)counts[s] : total));
    weight[r] = w;
  }
}

// loss = sum of weight * (policy term + kl_coef * KL); stats: policy term, KL and
// clipped share, each so weighted.
__global__ void __launch_bounds__(kWeightThreads)
    policy_sum_kernel(const double* terms, const float* weight, int64_t N, double kl_coef,
                      float* loss, float* stats) {
  __shared__ double red[32];
  double v[3] = {0.0, 0.0, 0.0};
  for (int64_t r = threadIdx.x; r < N; r += kWeightThreads) {
    const double w = weight[r];
    if (w != 0.0)
#pragma unroll
      for (int k = 0; k < 3; ++k) v[k] += w * terms[k * N + r];
  }
#pragma unroll
  for (int k = 0; k < 3; ++k) v[k] = block_sum(v[k], red);
  if (threadIdx.x == 0) {
    *loss = (float)(v[0] + (kl_coef != 0.0 ? kl_coef * v[1] : 0.0));
    for (int k = 0; k < 3; ++k) stats[k] = (float)v[k];
  }
}

int elt_of(int dtype) { return dtype == SQB_BF16 ? 2 : dtype == SQB_F32 ? 4 : 0; }

bool dims_ok(int64_t S, int64_t T, int64_t V) {
  return S > 0 && T > 0 && V > 0 && S <= INT32_MAX && T <= INT32_MAX / S;
}

int launched() { return cudaGetLastError() == cudaSuccess ? SQB_OK : SQB_ERR_LAUNCH; }

}  // namespace
}  // namespace logits
}  // namespace sqb

using namespace sqb::logits;

extern "C" int sqb_logp_fwd(const void* logits, const int64_t* targets, float* logp,
                            double* logp_double, float* stats, int64_t S, int64_t T, int64_t V,
                            int64_t ss, int64_t st, int dtype, void* stream) {
  if (!logits || !targets || !stats || !dims_ok(S, T, V)) return SQB_ERR_ARG;
  if (!elt_of(dtype)) return SQB_ERR_DTYPE;
  cudaStream_t q = static_cast<cudaStream_t>(stream);
  const unsigned grid = (unsigned)(S * T);
  const View v{T, V, ss, st};
  float2* ms = reinterpret_cast<float2*>(stats);
  if (dtype == SQB_BF16)
    logp_fwd_kernel<<<grid, kThreads, 0, q>>>(static_cast<const __nv_bfloat16*>(logits), targets,
                                              logp, logp_double, ms, v);
  else
    logp_fwd_kernel<<<grid, kThreads, 0, q>>>(static_cast<const float*>(logits), targets, logp,
                                              logp_double, ms, v);
  return launched();
}

extern "C" int sqb_logp_bwd(const void* logits, const int64_t* targets, const float* stats,
                            const float* g_row, const float* scale, void* dlogits, int64_t S,
                            int64_t T, int64_t V, int64_t ss, int64_t st, int64_t dss,
                            int64_t dst, int dtype, void* stream) {
  if (!logits || !targets || !stats || !g_row || !dlogits || !dims_ok(S, T, V))
    return SQB_ERR_ARG;
  if (!elt_of(dtype)) return SQB_ERR_DTYPE;
  cudaStream_t q = static_cast<cudaStream_t>(stream);
  const unsigned grid = (unsigned)(S * T);
  const View v{T, V, ss, st};
  const float2* ms = reinterpret_cast<const float2*>(stats);
  if (dtype == SQB_BF16)
    logp_bwd_kernel<<<grid, kThreads, 0, q>>>(static_cast<const __nv_bfloat16*>(logits), targets,
                                              ms, g_row, scale,
                                              static_cast<__nv_bfloat16*>(dlogits), v, dss, dst);
  else
    logp_bwd_kernel<<<grid, kThreads, 0, q>>>(static_cast<const float*>(logits), targets, ms,
                                              g_row, scale, static_cast<float*>(dlogits), v, dss,
                                              dst);
  return launched();
}

extern "C" int sqb_preference_finish(const double* logp, const int64_t* cu_seqlens,
                                     const float* ref_logps, int64_t P, int64_t T, int64_t N,
                                     double beta, double label_smoothing, double* pair_loss,
                                     float* loss, float* rewards, float* g_row, void* stream) {
  if (!pair_loss || !loss || !rewards || P <= 0 || P > INT32_MAX / 2 || N < 0 || T < 0)
    return SQB_ERR_ARG;
  if (N > 0 && (!logp || !g_row)) return SQB_ERR_ARG;
  if (!cu_seqlens && (T == 0 ? N != 0 : N / T != 2 * P || N % T != 0)) return SQB_ERR_ARG;
  cudaStream_t q = static_cast<cudaStream_t>(stream);
  preference_pair_kernel<<<(unsigned)P, kSeqThreads, 0, q>>>(
      logp, cu_seqlens, ref_logps, P, T, N, beta, label_smoothing, pair_loss, rewards, g_row);
  preference_mean_kernel<<<1, kSeqThreads, 0, q>>>(pair_loss, P, loss);
  return launched();
}

extern "C" int sqb_policy_weights(const int64_t* targets, const int64_t* cu_seqlens, int64_t S,
                                  int64_t T, int64_t N, int per_sequence, int32_t* counts,
                                  float* weight, int32_t* row_seq, void* stream) {
  if (!targets || !counts || !weight || S <= 0 || S > INT32_MAX || N <= 0 || N > INT32_MAX ||
      T < 0 || (cu_seqlens && !row_seq))
    return SQB_ERR_ARG;
  if (!cu_seqlens && (T == 0 || N / T != S || N % T != 0)) return SQB_ERR_ARG;
  policy_weights_kernel<<<1, kWeightThreads, 0, static_cast<cudaStream_t>(stream)>>>(
      targets, cu_seqlens, S, T, N, per_sequence != 0, counts, weight, row_seq);
  return launched();
}

extern "C" int sqb_policy_rows(const void* logits, const int64_t* targets, const float* old_logp,
                               const float* ref_logp, const float* adv, int adv_by_seq,
                               const int32_t* row_seq, const float* weight, double clip_low,
                               double clip_high, double kl_coef, float* logp, float* stats,
                               float* g_row, double* terms, void* dlogits, float grad_scale,
                               int64_t S, int64_t T, int64_t V, int64_t ss, int64_t st,
                               int64_t dss, int64_t dst, int dtype, void* stream) {
  if (!logits || !targets || !adv || !weight || !terms || !dims_ok(S, T, V)) return SQB_ERR_ARG;
  if (!elt_of(dtype)) return SQB_ERR_DTYPE;
  cudaStream_t q = static_cast<cudaStream_t>(stream);
  const int64_t N = S * T;
  const View v{T, V, ss, st};
  const Policy p{old_logp, ref_logp,       adv,           row_seq,        weight,
                 adv_by_seq != 0, 1.0 - clip_low, 1.0 + clip_high, kl_coef};
  float2* ms = reinterpret_cast<float2*>(stats);
  if (dtype == SQB_BF16)
    policy_kernel<<<(unsigned)N, kThreads, 0, q>>>(
        static_cast<const __nv_bfloat16*>(logits), targets, p, logp, ms, g_row, terms,
        static_cast<__nv_bfloat16*>(dlogits), grad_scale, v, dss, dst, N);
  else
    policy_kernel<<<(unsigned)N, kThreads, 0, q>>>(static_cast<const float*>(logits), targets, p,
                                                   logp, ms, g_row, terms,
                                                   static_cast<float*>(dlogits), grad_scale, v,
                                                   dss, dst, N);
  return launched();
}

extern "C" int sqb_policy_finish(const double* terms, const float* weight, int64_t N,
                                 double kl_coef, float* loss, float* stats, void* stream) {
  if (!terms || !weight || !loss || !stats || N <= 0 || N > INT32_MAX) return SQB_ERR_ARG;
  policy_sum_kernel<<<1, kWeightThreads, 0, static_cast<cudaStream_t>(stream)>>>(
      terms, weight, N, kl_coef, loss, stats);
  return launched();
}
