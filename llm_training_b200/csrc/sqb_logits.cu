// Token log-probabilities of logits and the two losses that train on them
// (include/sqb_train.h): a preference loss over pairs of answers and a clipped
// policy loss with a KL term, forward and backward.
//
// A row of V logits x with target t, m a number near its maximum:
//   s = sum exp(x - m),  logp = x_t - m - log s,  d logp / d x_c = [c == t] - exp(x_c - m) / s.
// (m, s) is kept for the backward.  A sequence's log-probability is a sum of hundreds
// to thousands of logps and the losses are made of small differences of such sums, so
// an error that all rows share grows with the length: everything above s is computed
// in 64 bits by one thread, and s itself is summed without such an error (below).
//
// The kernels over logits are bound by HBM: they read each row once, with independent
// 16-byte loads, and rows whose target is ignored are not read at all.  The exponentials
// come next (one special-function result for each logit, 16 a clock and SM, against 11.7
// bf16 logits a clock and SM at 6.56 TB/s), which is why the sum is shaped around them.
//
// Sum of exponentials: of 2^(x log2(e) - c), c a whole number no smaller than the largest
// x log2(e), so that a new maximum rescales by an exact power of two.  The product x log2(e)
// must not be rounded either: its rounding is the same for all rows that hold the same logit,
// and with it, or with an approximate exponential to rescale by, 1e-7 of s is left in every
// row, the same sign in all - 5e-5 of a 512-token answer's log-probability, against 1e-6 to
// 1e-5 this way (2e-9 to 2e-8 a row).  The difference is then rounded at most where |x log2(e)|
// is smaller than it: by 2^-24 of a difference d whose exponential is 2^-d, 2^-25 of s at most
// and of either sign.  What is left is ex2.approx itself: where bf16 logits are so large that
// they take a handful of values (600, in steps of 4), what it is off at these is shared by the
// rows: 6e-8.
//   bf16: with H = log2(e) cut to 15 bits, x H has at most 23 bits and x H - c is formed in
//     one fused multiply-add.  What H lacks, exp(x) = 2^(x H) exp(x d) with
//     d = 1 - H ln 2 (5e-6), is made up for once a row: sum e (1 + (x - x0) d) from the sums
//     of e and of e x (the next term, ((x - x0) d)^2 / 2, is below 1e-8 where e counts).
//   fp32: h = fl(x L), and the rest of x log2(e), an fma's residual and the constant's low
//     part, is summed as e r beside e.
// Rows whose maximum is beyond 2800 are summed again by one warp, with rounded arguments.

#include <cuda_bf16.h>
#include <math.h>
#include <stdint.h>

#include <type_traits>

#include "sqb_train.h"

namespace sqb {
namespace logits {
namespace {

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLog2eLow = (float)(1.4426950408889634 - (double)kLog2e);
constexpr double kLn2 = 0.6931471805599453;
// log2(e) cut to 15 bits, and 1 - H ln 2 (4.9e-6)
constexpr float kH = 23637.0f / 16384.0f;
constexpr double kLack = 1.0 - (double)kH * kLn2;
constexpr int kBound = 4096;  // of c in the exact form
// ex2.approx of arguments below 0 falls short by 5.06e-8 in the mean (measured on B200, 2^18
// arguments a binade: 4.9e-8 to 5.1e-8 in [-16, -1), 2e-8 to 6e-8 in [-1, 0) by the last bits of
// the arguments; 3e-8 around the mean), about a fifth of its largest error.  All of a row's
// terms share it, and all rows: it is made up for in the sum.
constexpr double kExp2Short = 5.06e-8;

struct View {  // (S, T, V) logits, unit stride on V; strides in elements
  int64_t T, V, ss, st;
};

__device__ __forceinline__ int64_t row_offset(uint32_t r, int64_t T, int64_t ss, int64_t st) {
  const uint32_t s = r / (uint32_t)T;
  return s * ss + (r - s * (uint32_t)T) * st;
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
// max that keeps a NaN
__device__ __forceinline__ float max_nan(float a, float b) {
  float y;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(y) : "f"(a), "f"(b));
  return y;
}

__device__ __forceinline__ float exp_diff(float x, float m) {
  return exp2_approx((x - m) * kLog2e);
}

// The number a running sum is taken against: 0 while every element so far is -inf
// (their exponentials are then 0, and a NaN still shows).
__device__ __forceinline__ float finite_ref(float m) { return m == -INFINITY ? 0.f : m; }

// Elements before the first 16-byte boundary of `p`, at most V.
template <typename T>
__device__ __forceinline__ int head_of(const T* p, int V) {
  const int h = (int)((16 - (reinterpret_cast<uintptr_t>(p) & 15)) & 15) / (int)sizeof(T);
  return h < V ? h : V;
}

// A group of kThreads threads works on a row: a CTA of kThreads, or (32) one of its warps.
template <int kThreads>
__device__ __forceinline__ int rank() {
  return kThreads == 32 ? (threadIdx.x & 31) : threadIdx.x;
}
template <int kThreads>
__device__ __forceinline__ void group_sync() {
  if constexpr (kThreads == 32)
    __syncwarp();
  else
    __syncthreads();
}

// Part of a row's sum: e = 2^(x log2(e) - ref) and its correction (e x for bf16, e r for fp32).
// e is added up in fp32 over a group of up to 32 elements and from there in 64 bits: next to a
// longer fp32 sum, what is below 2^-25 of it is lost, 1e-7 of s in all for logits whose
// standard deviation is 4.
struct Part {
  int ref;
  double a;
  float b;
};
constexpr int kNone = -65536;  // ref before the first element

// 2^k for k <= 0
__device__ __forceinline__ float power_of_2(int k) {
  return __int_as_float((max(k, -127) + 127) << 23);
}

__device__ __forceinline__ void rescale(Part& p, int ref) {
  const float f = power_of_2(p.ref - ref);
  p.a *= f;
  p.b *= f;
  p.ref = ref;
}

// The sum of the warp's parts, in all its lanes.
__device__ __forceinline__ void join_warp(Part& p) {
  rescale(p, __reduce_max_sync(0xffffffffu, p.ref));
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    p.a += __shfl_xor_sync(0xffffffffu, p.a, o);
    p.b += __shfl_xor_sync(0xffffffffu, p.b, o);
  }
}

// Stand for -inf and below: their exponentials are 0 as well, and their corrections finite.
constexpr float kLowestBf16 = -3.3e38f, kLowest = -1e30f;

// Makes p's ref no smaller than top's.
template <typename T>
__device__ __forceinline__ void raise(Part& p, float top) {
  const int c = min(__float2int_ru(top * (sizeof(T) == 2 ? kH : kLog2e)), -kNone);
  if (c > p.ref) rescale(p, c);
}

template <typename T>
__device__ __forceinline__ void add(Part& p, float& a, float c, float x) {
  if constexpr (sizeof(T) == 2) {
    const float e = exp2_approx(fmaf(x, kH, -c));
    a += e;
    p.b = fmaf(e, x, p.b);
  } else {
    const float h = x * kLog2e, e = exp2_approx(h - c);
    a += e;
    p.b = fmaf(e, fmaf(x, kLog2eLow, fmaf(x, kLog2e, -h)), p.b);
  }
}

template <typename T>
__device__ __forceinline__ void add_one(Part& p, T v) {
  const float x = max_nan(to_f(v), sizeof(T) == 2 ? kLowestBf16 : kLowest);
  float a = 0.f;
  raise<T>(p, x);
  add<T>(p, a, (float)p.ref, x);
  p.a += a;
}

// Adds the n 16-byte vectors u.
template <typename T, int n>
__device__ __forceinline__ void add_vectors(Part& p, uint4 (&u)[n]) {
  uint32_t* w = reinterpret_cast<uint32_t*>(u);
  float a = 0.f;
  if constexpr (sizeof(T) == 4) {
    float top = kLowest;
#pragma unroll
    for (int j = 0; j < 4 * n; ++j) {
      w[j] = __float_as_uint(max_nan(__uint_as_float(w[j]), kLowest));
      top = fmaxf(top, __uint_as_float(w[j]));
    }
    raise<T>(p, top);
    const float c = (float)p.ref;
#pragma unroll
    for (int j = 0; j < 4 * n; ++j) add<T>(p, a, c, __uint_as_float(w[j]));
  } else {
    const __nv_bfloat162 low = __float2bfloat162_rn(kLowestBf16);
    __nv_bfloat162 top = low;
#pragma unroll
    for (int j = 0; j < 4 * n; ++j) {
      const __nv_bfloat162 v = __hmax2_nan(*reinterpret_cast<__nv_bfloat162*>(&w[j]), low);
      top = __hmax2(top, v);
      w[j] = *reinterpret_cast<const uint32_t*>(&v);
    }
    raise<T>(p, fmaxf(__low2float(top), __high2float(top)));
    const float c = (float)p.ref;
#pragma unroll
    for (int j = 0; j < 4 * n; ++j) {
      add<T>(p, a, c, __uint_as_float(w[j] << 16));
      add<T>(p, a, c, __uint_as_float(w[j] & 0xffff0000u));
    }
  }
  p.a += a;
}

constexpr int kUnroll = 4;

// (m, s) of a row whose maximum is out of the exact form's range, by one warp: rounded
// arguments, 64-bit sums.
template <typename T>
__device__ void far_stats(const T* row, int V, float& m, double& s) {
  const int lane = threadIdx.x & 31;
  float top = -INFINITY;
  for (int c = lane; c < V; c += 32) top = fmaxf(top, to_f(row[c]));
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
  const float ref = finite_ref(top);
  s = 0.0;
  for (int c = lane; c < V; c += 32) s += exp_diff(to_f(row[c]), ref);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
  m = top;
}

// A row's (m, s), by its group of threads; in the lanes of the group's first warp alone.
// red: shared memory of a CTA's warps.
template <typename T, int kThreads>
__device__ void row_stats(const T* row, int V, Part* red, float& m, double& s) {
  constexpr int kN = 16 / sizeof(T);
  Part p{kNone, 0.0, 0.f};
  const int head = head_of(row, V), nvec = (V - head) / kN, me = rank<kThreads>();
  const uint4* body = reinterpret_cast<const uint4*>(row + head);
  int i = me;
  for (; i + (kUnroll - 1) * kThreads < nvec; i += kUnroll * kThreads) {
    uint4 u[kUnroll];
#pragma unroll
    for (int k = 0; k < kUnroll; ++k) u[k] = body[i + k * kThreads];
    add_vectors<T>(p, u);
  }
  for (; i < nvec; i += kThreads) {
    uint4 u[1] = {body[i]};
    add_vectors<T>(p, u);
  }
  if (me < head) add_one<T>(p, row[me]);
  const int tail = head + nvec * kN + me;
  if (tail < V) add_one<T>(p, row[tail]);
  join_warp(p);
  if constexpr (kThreads > 32) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (lane == 0) red[warp] = p;
    __syncthreads();
    if (warp) return;
    p = lane < kThreads / 32 ? red[lane] : Part{kNone, 0.0, 0.f};
    join_warp(p);
  }
  if (abs(p.ref) >= kBound) {
    far_stats(row, V, m, s);
    return;
  }
  const double x0 = p.ref * kLn2;
  m = (float)x0;
  double y = x0 - (double)m;  // sum e^x = 2^ref sum = e^(m + y) sum
  if constexpr (sizeof(T) == 2) {
    s = p.a + kLack * ((double)p.b - x0 * p.a);  // sum e^(x lack) e = e^(x0 lack) s
    y += x0 * kLack;                             // below 0.02
  } else {
    s = p.a + kLn2 * (double)p.b;
  }
  s *= 1.0 + kExp2Short + y * (1.0 + y * (0.5 + y * (1.0 / 6 + y / 24)));
}

// A vector's load and store; kLast: nothing of either is wanted in L2 any longer (where rows
// that will be read a second time lie).
template <bool kLast>
__device__ __forceinline__ uint4 get(const uint4* p) {
  return kLast ? __ldcs(p) : *p;
}
template <bool kLast>
__device__ __forceinline__ void put(uint4* p, uint4 v) {
  if (kLast)
    __stcs(p, v);
  else
    *p = v;
}

// drow[c] = g [c == t] + k exp(row[c] - m) for c < V, k = -g / s, by the group.
template <typename T, int kThreads, bool kLast>
__device__ void write_grad(const T* row, T* drow, int V, int64_t t, float m, float k, float g) {
  constexpr int kN = 16 / sizeof(T);
  const int me = rank<kThreads>();
  auto grad = [&](float x, int c) {
    const float p = k * exp_diff(x, m);
    return from_f<T>(c == t ? g + p : p);
  };
  if (((reinterpret_cast<uintptr_t>(row) ^ reinterpret_cast<uintptr_t>(drow)) & 15) != 0) {
    for (int c = me; c < V; c += kThreads) drow[c] = grad(to_f(row[c]), c);
    return;
  }
  const int head = head_of(row, V), nvec = (V - head) / kN;
  if (me < head) drow[me] = grad(to_f(row[me]), me);
  const uint4* body = reinterpret_cast<const uint4*>(row + head);
  uint4* out = reinterpret_cast<uint4*>(drow + head);
  auto vector = [&](uint4 u) {
    const T* e = reinterpret_cast<const T*>(&u);
    uint4 o;
    T* d = reinterpret_cast<T*>(&o);
#pragma unroll
    for (int j = 0; j < kN; ++j) d[j] = from_f<T>(k * exp_diff(to_f(e[j]), m));
    return o;
  };
  int i = me;
  for (; i + (kUnroll - 1) * kThreads < nvec; i += kUnroll * kThreads) {
    uint4 u[kUnroll];
#pragma unroll
    for (int j = 0; j < kUnroll; ++j) u[j] = get<kLast>(body + i + j * kThreads);
#pragma unroll
    for (int j = 0; j < kUnroll; ++j) put<kLast>(out + i + j * kThreads, vector(u[j]));
  }
  for (; i < nvec; i += kThreads) put<kLast>(out + i, vector(get<kLast>(body + i)));
  const int tail = head + nvec * kN + me;
  if (tail < V) drow[tail] = grad(to_f(row[tail]), tail);
  // the target's element, by the thread that wrote its vector
  const int64_t at = t - head;  // one past the vocabulary may be past 32 bits
  if (at >= 0 && at < nvec * kN && ((int)at / kN) % kThreads == me)
    drow[t] = grad(to_f(row[t]), (int)t);
}

template <typename T, int kThreads, bool kLast>
__device__ void write_zeros(T* drow, int V) {
  constexpr int kN = 16 / sizeof(T);
  const int head = head_of(drow, V), nvec = (V - head) / kN, me = rank<kThreads>();
  if (me < head) drow[me] = from_f<T>(0.f);
  uint4* out = reinterpret_cast<uint4*>(drow + head);
  for (int i = me; i < nvec; i += kThreads) put<kLast>(out + i, make_uint4(0, 0, 0, 0));
  const int tail = head + nvec * kN + me;
  if (tail < V) drow[tail] = from_f<T>(0.f);
}

// Log-probability of a target whose logit is x (NaN for one past the vocabulary).  In 64
// bits, and never inlined, like the policy's terms: one thread of a row calls them, and what
// registers they need is not to be taken from all the others.
__device__ __noinline__ double logp_of(double x, float m, double s) {
  return (x - (double)m) - log(s);
}
template <typename T>
__device__ __forceinline__ double logp_of(const T* row, int V, int64_t t, float m, double s) {
  return logp_of(t < V ? (double)to_f(row[t]) : (double)NAN, m, s);
}
// What is kept of a row for its gradient: NaN for a target past the vocabulary.
__device__ __forceinline__ float2 stats_of(int64_t V, int64_t t, float m, double s) {
  return make_float2(m, t < V ? (float)s : NAN);
}

// ---- rows -------------------------------------------------------------------------

// Threads of a row's CTA: of the kernels that only read it (4685 of 8192 rows of 50304 bf16:
// 88 us, 92 with 512), and of those that write its gradient (193 us, 201 with 256).
constexpr int kReadThreads = 256, kWriteThreads = 512;
constexpr int kWarpRows = 8;       // or a warp, eight rows to a CTA
// A warp takes a row of at most 2 KB, and one of up to 16 KB when there are rows for eight
// warps on every SM.  Forward and backward, warp against CTA: 32768 rows of 1024 bf16 21 + 26
// us, 59 + 121; 4096 of 8192 bf16 16 + 22, 17 + 31; 4096 of 16384 bf16 30 + 51, 28 + 43; 64
// rows of 4096 bf16 4.7 + 4.5, 3.1 + 2.7.
constexpr int64_t kWarpRowBytes = 16384, kFewRowBytes = 2048, kFewRows = 148 * 8;

template <int kThreads>
constexpr int block_of() {
  return kThreads == 32 ? 32 * kWarpRows : kThreads;
}
// The group's row; >= N for a warp that has none.
template <int kThreads>
__device__ __forceinline__ uint32_t row_of() {
  return kThreads == 32 ? blockIdx.x * kWarpRows + (threadIdx.x >> 5) : blockIdx.x;
}

// Rows of a packed batch that lie in a sequence: [cu[0], cu[seqs]), all for a null cu.
struct Inside {
  const int64_t* cu;
  int64_t seqs;
};

// The row's target; negative for a row that is left out: without one, or in no sequence.
__device__ __forceinline__ int64_t target_of(const int64_t* targets, const Inside& in,
                                             uint32_t r) {
  const int64_t t = targets[r];
  return in.cu && (r < in.cu[0] || r >= in.cu[in.seqs]) ? -1 : t;
}

// The statistics of a row that is left out, which tell the backward so: a softmax's sum is at
// least a half, or 0 next to a maximum of -inf.
__device__ __forceinline__ float2 left_out() { return make_float2(0.f, 0.f); }

// Per-row outputs: logp (either or both), stats = (m, s), and a zero for g_row.
struct RowOut {
  float* logp;
  double* logp64;
  float2* stats;
  float* g_row;
};

template <typename T, int kThreads>
__global__ void __launch_bounds__(block_of<kThreads>())
    logp_fwd_kernel(const T* x, const int64_t* targets, Inside in, RowOut out, View v,
                    uint32_t N) {
  __shared__ Part red[32];
  const uint32_t r = row_of<kThreads>();
  if (kThreads == 32 && r >= N) return;
  const int64_t t = target_of(targets, in, r);
  float2 ms = left_out();
  double lp = 0.0;
  if (t >= 0) {
    const T* row = x + row_offset(r, v.T, v.ss, v.st);
    float m;
    double s;
    row_stats<T, kThreads>(row, (int)v.V, red, m, s);
    if (rank<kThreads>() == 0) {
      lp = logp_of(row, (int)v.V, t, m, s);
      ms = stats_of(v.V, t, m, s);
    }
  }
  if (rank<kThreads>() == 0) {
    out.stats[r] = ms;
    if (out.logp) out.logp[r] = (float)lp;
    if (out.logp64) out.logp64[r] = lp;
    if (out.g_row) out.g_row[r] = 0.f;
  }
}

template <typename T, int kThreads>
__global__ void __launch_bounds__(block_of<kThreads>())
    logp_bwd_kernel(const T* x, const int64_t* targets, const float2* stats, const float* g_row,
                    const float* scale, T* dx, View v, int64_t dss, int64_t dst, uint32_t N) {
  const uint32_t r = row_of<kThreads>();
  if (kThreads == 32 && r >= N) return;
  const int64_t t = targets[r];
  T* drow = dx + row_offset(r, v.T, dss, dst);
  const float2 ms = stats[r];
  const bool left = t < 0 || (ms.x == 0.f && ms.y == 0.f);
  float g = left ? 0.f : g_row[r];
  if (!left && scale) g *= *scale;
  // a zero factor (a clipped token) makes a zero row, which needs no logits - unless they
  // hold a NaN or an infinity or have no such target, which the sum then shows
  if (left || (g == 0.f && isfinite(ms.x) && isfinite(ms.y)))
    write_zeros<T, kThreads, false>(drow, (int)v.V);
  else
    write_grad<T, kThreads, false>(x + row_offset(r, v.T, v.ss, v.st), drow, (int)v.V, t, ms.x,
                                   -g / ms.y, g);
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
__device__ __noinline__ double policy_terms(double A, bool has_old, double old_logp,
                                            bool has_ref, double ref_logp, double lo, double hi,
                                            double kl_coef, double lp, double* term) {
  // without an old one 1, also for a -inf log-probability
  const double ratio = has_old ? exp(lp - old_logp) : isnan(lp) ? lp : 1.0;
  const double kept = ratio < lo ? lo : ratio > hi ? hi : ratio;
  const double open = ratio * A, held = kept * A;
  const bool clipped = held < open;
  term[0] = clipped ? -held : -open;
  term[2] = clipped ? 1.0 : 0.0;
  double d = clipped ? 0.0 : -open;
  term[1] = 0.0;
  if (has_ref) {
    const double gap = ref_logp - lp, e = expm1(gap);
    term[1] = e - gap;
    if (kl_coef != 0.0) d -= kl_coef * e;  // e may be infinite where the KL is only logged
  }
  return d;
}

// One row of the policy loss: log-probability, terms and d loss / d logp; with dx, also the
// row's gradient times `scale`, the row read again where it is still in L2.  Launched while
// the weights are still being counted: it waits for them once it has its sum.
// Three CTAs of 512 threads an SM, the second reading and the gradient passing through L2 as
// what is needed last: 8192 rows of 50304 bf16, 4975 of them counted, 237 us, 5.6 TB/s of the
// 1.32 GB it cannot do without.  Measured: 250 us without those hints, 272 with four CTAs
// besides (59 MB of rows wait in L2 between their readings; 234 with the hints and some
// spilled registers); the row kept in shared memory, two an SM, 284 us.
template <typename T, int kThreads>
__global__ void __launch_bounds__(block_of<kThreads>(), kThreads == 32 ? 1 : 1536 / kThreads)
    policy_kernel(const T* x, const int64_t* targets, Inside in, Policy p, RowOut out,
                  double* terms, T* dx, float scale, View v, int64_t dss, int64_t dst,
                  uint32_t N) {
  __shared__ Part red[32];
  __shared__ float3 known;
  const uint32_t r = row_of<kThreads>();
  if (kThreads == 32 && r >= N) return;
  const int64_t t = target_of(targets, in, r);
  const int me = rank<kThreads>(), V = (int)v.V;
  T* drow = dx ? dx + row_offset(r, v.T, dss, dst) : nullptr;
  if (t < 0) {
    if (me == 0) {
      out.logp[r] = 0.f;
      if (out.stats) out.stats[r] = left_out();
      if (out.g_row) out.g_row[r] = 0.f;
      terms[r] = terms[(size_t)N + r] = terms[2 * (size_t)N + r] = 0.0;
    }
    if (dx) write_zeros<T, kThreads, true>(drow, V);
    // no kernel behind this one may start before the weights are there, whatever rows there are
    if (r == 0 && me == 0) cudaGridDependencySynchronize();
    return;
  }
  const T* row = x + row_offset(r, v.T, v.ss, v.st);
  float m = 0.f, old_logp = 0.f, ref_logp = 0.f;
  double s = 1.0;
  if (me == 0) {
    if (p.old_logp) old_logp = p.old_logp[r];
    if (p.ref_logp) ref_logp = p.ref_logp[r];
  }
  row_stats<T, kThreads>(row, V, red, m, s);
  float3 f;  // m, -g / s (0: a zero row) and g
  if (me == 0) {
    const double lp = logp_of(row, V, t, m, s);
    cudaGridDependencySynchronize();
    const float w = p.weight[r];
    double term[3] = {0.0, 0.0, 0.0};
    float g = 0.f;
    float2 ms = left_out();
    if (w != 0.f) {  // else between sequences that do not follow one another: left out
      ms = stats_of(V, t, m, s);
      const uint32_t a = p.by_seq ? (p.seq ? (uint32_t)p.seq[r] : r / (uint32_t)v.T) : r;
      g = (float)(policy_terms(p.adv[a], p.old_logp, old_logp, p.ref_logp, ref_logp, p.lo, p.hi,
                               p.kl_coef, lp, term) *
                  (double)w);
    }
    out.logp[r] = w != 0.f ? (float)lp : 0.f;
    if (out.stats) out.stats[r] = ms;
    if (out.g_row) out.g_row[r] = g;
    terms[r] = term[0];
    terms[(size_t)N + r] = term[1];
    terms[2 * (size_t)N + r] = term[2];
    const float gs = w != 0.f ? g * scale : 0.f;
    f = make_float3(ms.x, gs == 0.f && isfinite(ms.x) && isfinite(ms.y) ? 0.f : -gs / ms.y, gs);
    if (kThreads > 32) known = f;
  }
  if (!dx) return;
  if constexpr (kThreads == 32) {
    f.x = __shfl_sync(0xffffffffu, f.x, 0);
    f.y = __shfl_sync(0xffffffffu, f.y, 0);
    f.z = __shfl_sync(0xffffffffu, f.z, 0);
  } else {
    __syncthreads();
    f = known;
  }
  if (f.y == 0.f && f.z == 0.f)
    write_zeros<T, kThreads, true>(drow, V);
  else
    write_grad<T, kThreads, true>(row, drow, V, t, f.x, f.y, f.z);
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
  cudaGridDependencySynchronize();
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
    // a term without weight is not there: its softplus may be infinite
    pair_loss[p] = (smooth != 1.0 ? (1.0 - smooth) * softplus(-z) : 0.0) +
                   (smooth != 0.0 ? smooth * softplus(z) : 0.0);
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
  cudaGridDependencySynchronize();
  for (int64_t p = threadIdx.x; p < P; p += kSeqThreads) v += pair_loss[p];
  v = block_sum(v, red);
  if (threadIdx.x == 0) *loss = (float)(v / (double)P);
}

constexpr int kWeightThreads = 1024;

// Weight of every row in the policy loss, and the sequence of every row of a packed
// batch (-1 for a row outside every sequence).  One CTA: the counts of all sequences
// are needed before the first weight, and 64K targets are 512 KB.
__global__ void __launch_bounds__(kWeightThreads)
    policy_weights_kernel(const int64_t* targets, const int64_t* cu, uint32_t S, uint32_t T,
                          uint32_t N, bool per_sequence, uint32_t* counts, float* weight,
                          int32_t* seq) {
  __shared__ double red[32];
  cudaTriggerProgrammaticLaunchCompletion();  // the rows' kernel may start
  for (uint32_t s = threadIdx.x; s < S; s += kWeightThreads) counts[s] = 0;
  __syncthreads();
  auto sequence = [&](uint32_t r) -> uint32_t {  // S for none
    if (!cu) return r / T;
    uint32_t lo = 0, hi = S;  // the first s with cu[s + 1] > r
    while (lo < hi) {
      const uint32_t mid = (lo + hi) / 2;
      if (cu[mid + 1] <= (int64_t)r)
        lo = mid + 1;
      else
        hi = mid;
    }
    return lo < S && cu[lo] <= (int64_t)r ? lo : S;
  };
  for (uint32_t base = 0; base < N; base += kWeightThreads) {
    const uint32_t r = base + threadIdx.x;
    const uint32_t s = r < N ? sequence(r) : S;
    if (seq && r < N) seq[r] = s < S ? (int32_t)s : -1;
    const bool counted = s < S && targets[r] >= 0;
    // whole numbers: their order does not show.  Most warps lie in one sequence.
    const uint32_t s0 = __shfl_sync(0xffffffffu, s, 0);
    if (__all_sync(0xffffffffu, s == s0)) {
      const uint32_t n = __popc(__ballot_sync(0xffffffffu, counted));
      if ((threadIdx.x & 31) == 0 && n) atomicAdd(&counts[s0], n);
    } else if (counted) {
      atomicAdd(&counts[s], 1u);
    }
  }
  __syncthreads();
  double total = 0.0;
  for (uint32_t s = threadIdx.x; s < S; s += kWeightThreads) {
    const uint32_t n = *reinterpret_cast<volatile uint32_t*>(&counts[s]);
    total += per_sequence ? (n > 0 ? 1.0 : 0.0) : (double)n;
  }
  total = block_sum(total, red);
  for (uint32_t r = threadIdx.x; r < N; r += kWeightThreads) {
    const uint32_t s = seq ? (uint32_t)seq[r] : r / T;  // -1 is beyond S
    float w = 0.f;
    if (s < S && targets[r] >= 0)
      w = (float)(1.0 / (per_sequence
                             ? total * (double)*reinterpret_cast<volatile uint32_t*>(&counts[s])
                             : total));
    weight[r] = w;
  }
}

// loss = sum of weight * (policy term + kl_coef * KL); statistics: policy term, KL and
// clipped share, each so weighted.
__global__ void __launch_bounds__(kWeightThreads)
    policy_sum_kernel(const double* terms, const float* weight, uint32_t N, double kl_coef,
                      float* loss, float* statistics) {
  __shared__ double red[32];
  double v[3] = {0.0, 0.0, 0.0};
  cudaGridDependencySynchronize();
#pragma unroll 4
  for (uint32_t r = threadIdx.x; r < N; r += kWeightThreads) {
    const double w = weight[r];  // the terms of a row without weight are 0
#pragma unroll
    for (int k = 0; k < 3; ++k) v[k] += w * terms[k * (size_t)N + r];
  }
#pragma unroll
  for (int k = 0; k < 3; ++k) v[k] = block_sum(v[k], red);
  if (threadIdx.x == 0) {
    *loss = (float)(v[0] + (kl_coef != 0.0 ? kl_coef * v[1] : 0.0));
    for (int k = 0; k < 3; ++k) statistics[k] = (float)v[k];
  }
}

int elt_of(int dtype) { return dtype == SQB_BF16 ? 2 : dtype == SQB_F32 ? 4 : 0; }

bool dims_ok(int64_t S, int64_t T, int64_t V) {
  return S > 0 && T > 0 && V > 0 && V <= (1 << 30) && S <= INT32_MAX && T <= INT32_MAX / S;
}

// Launches a kernel that may start before the one in front of it on the stream has ended: it
// waits for that one's results itself (cudaGridDependencySynchronize).
template <typename... P, typename... A>
void launch_early(void (*kernel)(P...), unsigned grid, unsigned block, cudaStream_t q, A... args) {
  cudaLaunchAttribute early;
  early.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  early.val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t config = {};
  config.gridDim = dim3(grid);
  config.blockDim = dim3(block);
  config.stream = q;
  config.attrs = &early;
  config.numAttrs = 1;
  cudaLaunchKernelEx(&config, kernel, static_cast<P>(args)...);
}

int launched() { return cudaGetLastError() == cudaSuccess ? SQB_OK : SQB_ERR_LAUNCH; }

// Calls f(type, threads, grid) for the rows' type and width: a warp for a short row, else a
// CTA of kCta threads.
template <int kCta, typename F>
void dispatch(int dtype, int64_t N, int64_t V, F&& f) {
  const unsigned rows = (unsigned)N, packed = (unsigned)((N + kWarpRows - 1) / kWarpRows);
  const int64_t bytes = V * elt_of(dtype);
  const bool warp = bytes <= (N < kFewRows ? kFewRowBytes : kWarpRowBytes);
  using W = std::integral_constant<int, 32>;
  using B = std::integral_constant<int, kCta>;
  if (dtype == SQB_BF16)
    warp ? f(__nv_bfloat16(), W(), packed) : f(__nv_bfloat16(), B(), rows);
  else
    warp ? f(float(), W(), packed) : f(float(), B(), rows);
}

void launch_logp(const void* x, const int64_t* targets, const Inside& in, const RowOut& out,
                 int64_t S, int64_t T, int64_t V, int64_t ss, int64_t st, int dtype,
                 cudaStream_t q) {
  dispatch<kReadThreads>(dtype, S * T, V, [&](auto type, auto threads, unsigned grid) {
    using X = decltype(type);
    constexpr int kThreads = decltype(threads)::value;
    logp_fwd_kernel<X, kThreads><<<grid, block_of<kThreads>(), 0, q>>>(
        static_cast<const X*>(x), targets, in, out, View{T, V, ss, st}, (uint32_t)(S * T));
  });
}

size_t align256(size_t n) { return (n + 255) / 256 * 256; }

// Whether every pointer (a null one, too) is a multiple of `bytes`.
template <typename... P>
bool aligned(uintptr_t bytes, P... p) {
  return (... && (reinterpret_cast<uintptr_t>(p) % bytes == 0));
}

}  // namespace
}  // namespace logits
}  // namespace sqb

using namespace sqb::logits;

extern "C" int sqb_logp_fwd(const void* logits, const int64_t* targets, float* logp, float* stats,
                            int64_t S, int64_t T, int64_t V, int64_t ss, int64_t st, int dtype,
                            void* stream) {
  if (!logits || !targets || !logp || !stats || !dims_ok(S, T, V)) return SQB_ERR_ARG;
  const int elt = elt_of(dtype);
  if (!elt) return SQB_ERR_DTYPE;
  if (!aligned(elt, logits) || !aligned(8, targets, stats) || !aligned(4, logp))
    return SQB_ERR_ALIGN;
  const RowOut out{logp, nullptr, reinterpret_cast<float2*>(stats), nullptr};
  launch_logp(logits, targets, Inside{nullptr, 0}, out, S, T, V, ss, st, dtype,
              static_cast<cudaStream_t>(stream));
  return launched();
}

extern "C" int sqb_logp_bwd(const void* logits, const int64_t* targets, const float* stats,
                            const float* g_row, const float* scale, void* dlogits, int64_t S,
                            int64_t T, int64_t V, int64_t ss, int64_t st, int64_t dss,
                            int64_t dst, int dtype, void* stream) {
  if (!logits || !targets || !stats || !g_row || !dlogits || !dims_ok(S, T, V))
    return SQB_ERR_ARG;
  const int elt = elt_of(dtype);
  if (!elt) return SQB_ERR_DTYPE;
  if (!aligned(elt, logits, dlogits) || !aligned(8, targets, stats) || !aligned(4, g_row, scale))
    return SQB_ERR_ALIGN;
  dispatch<kWriteThreads>(dtype, S * T, V, [&](auto type, auto threads, unsigned grid) {
    using X = decltype(type);
    constexpr int kThreads = decltype(threads)::value;
    logp_bwd_kernel<X, kThreads>
        <<<grid, block_of<kThreads>(), 0, static_cast<cudaStream_t>(stream)>>>(
            static_cast<const X*>(logits), targets, reinterpret_cast<const float2*>(stats), g_row,
            scale, static_cast<X*>(dlogits), View{T, V, ss, st}, dss, dst, (uint32_t)(S * T));
  });
  return launched();
}

extern "C" size_t sqb_preference_workspace_bytes(int64_t N, int64_t P) {
  if (N < 0 || P <= 0) return 0;
  return align256((size_t)N * sizeof(double)) + (size_t)P * sizeof(double);
}

extern "C" int sqb_preference_fwd(const void* logits, const int64_t* targets,
                                  const int64_t* cu_seqlens, const float* ref_logps, int64_t P,
                                  double beta, double label_smoothing, float* loss,
                                  float* rewards, float* stats, float* g_row, int64_t S,
                                  int64_t T, int64_t V, int64_t ss, int64_t st, int dtype,
                                  void* workspace, size_t ws_bytes, void* stream) {
  if (!loss || !rewards || P <= 0 || P > INT32_MAX / 2 || S <= 0 || T < 0) return SQB_ERR_ARG;
  if (T > 0 && (!logits || !targets || !stats || !g_row || !dims_ok(S, T, V)))
    return SQB_ERR_ARG;
  if (cu_seqlens ? S != 1 : S != 2 * P) return SQB_ERR_ARG;
  const int elt = elt_of(dtype);
  if (!elt) return SQB_ERR_DTYPE;
  const int64_t N = S * T;
  if (!workspace || ws_bytes < sqb_preference_workspace_bytes(N, P)) return SQB_ERR_WORKSPACE;
  if (!aligned(elt, logits) || !aligned(8, targets, cu_seqlens, stats) ||
      !aligned(4, ref_logps, loss, rewards, g_row) ||
      !aligned(8, workspace))
    return SQB_ERR_ALIGN;
  cudaStream_t q = static_cast<cudaStream_t>(stream);
  double* logp = static_cast<double*>(workspace);
  double* pair_loss = logp + align256((size_t)N * sizeof(double)) / sizeof(double);
  // rows of a packed batch that belong to no sequence keep the zero written here
  const RowOut out{nullptr, logp, reinterpret_cast<float2*>(stats), cu_seqlens ? g_row : nullptr};
  if (N > 0)
    launch_logp(logits, targets, Inside{cu_seqlens, 2 * P}, out, S, T, V, ss, st, dtype, q);
  if (N > 0)
    launch_early(preference_pair_kernel, (unsigned)P, kSeqThreads, q, logp, cu_seqlens, ref_logps,
                 P, T, N, beta, label_smoothing, pair_loss, rewards, g_row);
  else
    preference_pair_kernel<<<(unsigned)P, kSeqThreads, 0, q>>>(logp, cu_seqlens, ref_logps, P, T,
                                                               N, beta, label_smoothing,
                                                               pair_loss, rewards, g_row);
  launch_early(preference_mean_kernel, 1, kSeqThreads, q, pair_loss, P, loss);
  return launched();
}

extern "C" size_t sqb_policy_workspace_bytes(int64_t N, int64_t seqs) {
  if (N <= 0 || seqs <= 0) return 0;
  return align256((size_t)N * 3 * sizeof(double)) +
         ((size_t)N * 2 + (size_t)seqs) * sizeof(float);
}

extern "C" int sqb_policy_fwd(const void* logits, const int64_t* targets,
                              const int64_t* cu_seqlens, int64_t seqs, const float* old_logp,
                              const float* ref_logp, const float* adv, int adv_by_seq,
                              double clip_low, double clip_high, double kl_coef,
                              int per_sequence, float* loss, float* statistics, float* logp,
                              float* stats, float* g_row, void* dlogits, float grad_scale,
                              int64_t S, int64_t T, int64_t V, int64_t ss, int64_t st,
                              int64_t dss, int64_t dst, int dtype, void* workspace,
                              size_t ws_bytes, void* stream) {
  if (!logits || !targets || !adv || !loss || !statistics || !logp || !dims_ok(S, T, V) ||
      seqs <= 0 || seqs > INT32_MAX || (cu_seqlens ? S != 1 : S != seqs))
    return SQB_ERR_ARG;
  const int elt = elt_of(dtype);
  if (!elt) return SQB_ERR_DTYPE;
  const int64_t N = S * T;
  if (!workspace || ws_bytes < sqb_policy_workspace_bytes(N, seqs)) return SQB_ERR_WORKSPACE;
  if (!aligned(elt, logits, dlogits) || !aligned(8, targets, cu_seqlens, stats) ||
      !aligned(4, old_logp, ref_logp, adv, loss, statistics, logp, g_row) ||
      !aligned(8, workspace))
    return SQB_ERR_ALIGN;
  cudaStream_t q = static_cast<cudaStream_t>(stream);
  double* terms = static_cast<double*>(workspace);
  float* weight = reinterpret_cast<float*>(static_cast<char*>(workspace) +
                                           align256((size_t)N * 3 * sizeof(double)));
  int32_t* seq = reinterpret_cast<int32_t*>(weight + N);
  uint32_t* counts = reinterpret_cast<uint32_t*>(seq + N);
  policy_weights_kernel<<<1, kWeightThreads, 0, q>>>(targets, cu_seqlens, (uint32_t)seqs,
                                                     (uint32_t)T, (uint32_t)N, per_sequence != 0,
                                                     counts, weight, cu_seqlens ? seq : nullptr);
  const Policy p{old_logp,        ref_logp,       adv,    cu_seqlens ? seq : nullptr, weight,
                 adv_by_seq != 0, 1.0 - clip_low, 1.0 + clip_high, kl_coef};
  const RowOut out{logp, nullptr, reinterpret_cast<float2*>(stats), g_row};
  auto rows = [&](auto type, auto threads, unsigned grid) {
    using X = decltype(type);
    constexpr int kThreads = decltype(threads)::value;
    launch_early(policy_kernel<X, kThreads>, grid, block_of<kThreads>(), q,
                 static_cast<const X*>(logits), targets, Inside{cu_seqlens, seqs}, p, out, terms,
                 static_cast<X*>(dlogits), grad_scale, View{T, V, ss, st}, dss, dst, (uint32_t)N);
  };
  if (dlogits)
    dispatch<kWriteThreads>(dtype, N, V, rows);
  else
    dispatch<kReadThreads>(dtype, N, V, rows);
  launch_early(policy_sum_kernel, 1, kWeightThreads, q, terms, weight, (uint32_t)N, kl_coef, loss,
               statistics);
  return launched();
}
