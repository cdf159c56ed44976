// Residual step between two norms (include/sqb_train.h): the norm behind a block,
// its gate and scale, the residual add, and the norm before the next block.
//
//   n  = Norm(h; post weight, post bias)      (n = h without a post weight)
//   x' = x + scale * gate * n,   y = Norm(x'; weight, bias)
//   Norm(v; w, b) = (v - mean) / sqrt(mean of (v - mean)^2 + eps) * w + b, mean = 0 for RMS
//
// Backward, with u = dy * w, x^ and h^ the normalised rows, r and r_h their 1/std:
//   D  = dx' + r (u - [mean u] - x^ mean(u x^)),   dx = D
//   dn = D * scale * gate,  v = dn * post weight
//   dh = r_h (v - [mean v] - h^ mean(v h^))       ([mean] terms: layer norm only)
//   d weight = sum dy x^, d bias = sum dy, d post weight = sum dn h^, d post bias = sum dn,
//   d gate = sum scale D n over the rows that share the gate
//
// Both norms' statistics are saved; the backward forms x' again from x and h in fp32, so
// that a stream kept in bf16 is not rounded between the two passes.  Variances are of
// differences from the mean (two sweeps over registers), never E[v^2] - mean^2.
// Bound by HBM for large batches: forward reads x, h and writes x', y; backward reads
// x, h, dy, dx' and writes dx, dh.

#include <cuda_bf16.h>
#include <math.h>
#include <stdint.h>

#include <type_traits>

#include "sqb_train.h"

namespace sqb {
namespace resnorm {
namespace {

constexpr int kMaxC = 4096;
constexpr int kParts = 5;  // d weight, d bias, d post weight, d post bias, d gate (if one)

struct Args {
  const void *x, *h;
  const float *w, *b, *wp, *bp, *gate;
  float scale, eps;
  uint32_t N, T;  // rows, rows that share a gate (N for one gate)
  int C;
  bool rms;
};

template <typename T, int W>
struct Raw;  // W elements as they lie in memory
template <>
struct Raw<float, 4> {
  float4 v;
};
template <>
struct Raw<__nv_bfloat16, 4> {
  uint2 v;
};
template <>
struct Raw<float, 1> {
  float v;
};
template <>
struct Raw<__nv_bfloat16, 1> {
  __nv_bfloat16 v;
};

template <typename T, int W>
__device__ __forceinline__ Raw<T, W> fetch(const T* p) {
  return *reinterpret_cast<const Raw<T, W>*>(p);
}
__device__ __forceinline__ void unpack(Raw<float, 4> r, float* v) {
  v[0] = r.v.x, v[1] = r.v.y, v[2] = r.v.z, v[3] = r.v.w;
}
__device__ __forceinline__ void unpack(Raw<__nv_bfloat16, 4> r, float* v) {
  v[0] = __uint_as_float(r.v.x << 16), v[1] = __uint_as_float(r.v.x & 0xffff0000u);
  v[2] = __uint_as_float(r.v.y << 16), v[3] = __uint_as_float(r.v.y & 0xffff0000u);
}
__device__ __forceinline__ void unpack(Raw<float, 1> r, float* v) { v[0] = r.v; }
__device__ __forceinline__ void unpack(Raw<__nv_bfloat16, 1> r, float* v) {
  v[0] = __bfloat162float(r.v);
}

template <int W>
__device__ __forceinline__ void store(float* p, const float* v) {
  if constexpr (W == 4)
    *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]);
  else
    p[0] = v[0];
}
template <int W>
__device__ __forceinline__ void store(__nv_bfloat16* p, const float* v) {
  if constexpr (W == 4) {
    const __nv_bfloat162 a = __floats2bfloat162_rn(v[0], v[1]);
    const __nv_bfloat162 b = __floats2bfloat162_rn(v[2], v[3]);
    *reinterpret_cast<uint2*>(p) = make_uint2(*reinterpret_cast<const uint32_t*>(&a),
                                              *reinterpret_cast<const uint32_t*>(&b));
  } else {
    p[0] = __float2bfloat16_rn(v[0]);
  }
}

// W parameters of columns c.., or `none` for a null p.
template <int W>
__device__ __forceinline__ void param(const float* p, int c, float none, float* v) {
  if (p)
    unpack(fetch<float, W>(p + c), v);
  else
#pragma unroll
    for (int j = 0; j < W; ++j) v[j] = none;
}

// ---- rows ---------------------------------------------------------------------------
//
// G warps (1 to 16) hold a row, E columns a lane, each warp 32 E consecutive ones, and walk a
// run of consecutive rows.  A CTA is one such group, or eight groups of one warp.  A warp
// whose columns all exist takes a path without a comparison for each.  More warps before more
// columns a lane: 2728 rows of 4001 (bf16, y fp32) take 52 + 62 us, forward + backward, and
// took 69 + 96 with eight warps of 16 columns; and fewer columns where one warp has room: 51155
// rows of 102 take 37 + 50 us with 4 a lane, 59 + 93 with 8.

constexpr int kMaxWarps = 16;               // of a row
constexpr int kBwdWarps = 16, kFwdWarps = 24;  // on an SM, as registers allow

// The CTA's barrier: its warps arrive from two places in the code.
__device__ __forceinline__ void group_barrier() { asm volatile("bar.sync 0;" ::: "memory"); }

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// ---- forward ------------------------------------------------------------------------

// Mean (0 for RMS) and 1/std of a row over its G warps.  Each warp finds its own columns'
// mean and squared differences (two sweeps over registers); the warps' are joined by
//   M2 = sum M2_i + n_i (mean_i - mean)^2,  one barrier for both.
// red: a pair for each warp; uses alternate between two.
template <int E, int W, typename On>
__device__ __forceinline__ void moments(const float (&v)[E], const Args& a, On on, int G,
                                        int member, float2* red, float& mean, float& rstd) {
  const int n = min(32 * E, a.C - member * 32 * E);
  float m = 0.f, q = 0.f;
  if (!a.rms) {
#pragma unroll
    for (int e = 0; e < E; ++e) m += v[e];  // columns that are not there hold 0
    m = warp_sum(m) / n;
  }
#pragma unroll
  for (int e = 0; e < E; ++e) {
    const float d = v[e] - m;
    if (on(e / W)) q = fmaf(d, d, q);
  }
  q = warp_sum(q);
  mean = m;
  if (G > 1) {
    if ((threadIdx.x & 31) == 0) red[member] = make_float2(m, q);
    group_barrier();
    if (!a.rms) {
      mean = 0.f;
      for (int i = 0; i < G; ++i) mean += red[i].x * min(32 * E, a.C - i * 32 * E);
      mean /= a.C;
    }
    q = 0.f;
    for (int i = 0; i < G; ++i) {
      const float2 p = red[i];
      const float d = p.x - mean;
      q += p.y;
      if (!a.rms) q += d * d * min(32 * E, a.C - i * 32 * E);
    }
  }
  rstd = rsqrtf(q / a.C + a.eps);
}

template <typename X, typename H, typename Y, int E, int W, bool kBias, bool kFull>
__device__ __forceinline__ void fwd_rows(const Args& a, X* xo, Y* y, float4* stats, float2* red,
                                         uint32_t first, uint32_t last, int c0, int member,
                                         int G) {
  constexpr int K = E / W, kStep = 32 * W;
  constexpr bool kKeep = !kBias;  // parameters in registers
  const int C = a.C;
  auto on = [&](int k) { return kFull || c0 + k * kStep < C; };
  float w[kKeep ? E : W], wp[kKeep ? E : W], gw[kKeep ? E : W], b[W], bp[W];
  auto load_post = [&](const float* gate, int k, int i) {
    param<W>(on(k) ? a.wp : nullptr, c0 + k * kStep, 1.f, wp + i);
    param<W>(on(k) ? gate : nullptr, c0 + k * kStep, 1.f, gw + i);
#pragma unroll
    for (int j = 0; j < W; ++j) gw[i + j] *= a.scale;
  };
  uint32_t grp = first / a.T, turn = (grp + 1) * a.T;
  const float* gate = a.gate ? a.gate + (size_t)grp * C : nullptr;
  if (kKeep)
#pragma unroll
    for (int k = 0; k < K; ++k) {
      load_post(gate, k, k * W);
      param<W>(on(k) ? a.w : nullptr, c0 + k * kStep, 1.f, w + k * W);
    }
  for (uint32_t r = first; r < last; ++r) {
    const size_t base = (size_t)r * C + c0;
    const X* xr = static_cast<const X*>(a.x) + base;
    const H* hr = static_cast<const H*>(a.h) + base;
    Raw<X, W> xw[K];
    Raw<H, W> hw[K];
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int i = on(k) ? k * kStep : -c0;  // a column that is not there: the row's first
      hw[k] = fetch<H, W>(hr + i);
      xw[k] = fetch<X, W>(xr + i);
    }
    if (r == turn) {
      turn += a.T;
      if (a.gate) {
        gate += C;
        if (kKeep)
#pragma unroll
          for (int k = 0; k < K; ++k) load_post(gate, k, k * W);
      }
    }
    float h[E], x[E];
#pragma unroll
    for (int k = 0; k < K; ++k) {
      unpack(hw[k], h + k * W);
      unpack(xw[k], x + k * W);
      if (!on(k))
#pragma unroll
        for (int j = 0; j < W; ++j) h[k * W + j] = x[k * W + j] = 0.f;
    }
    float mh = 0.f, rh = 1.f, mx, rx;
    if (a.wp) moments<E, W>(h, a, on, G, member, red, mh, rh);
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int i = kKeep ? k * W : 0;
      if (!kKeep) load_post(gate, k, 0);
      param<W>(kBias && on(k) ? a.bp : nullptr, c0 + k * kStep, 0.f, bp);
#pragma unroll
      for (int j = 0; j < W; ++j) {
        const int e = k * W + j;
        x[e] = fmaf(gw[i + j], fmaf((h[e] - mh) * rh, wp[i + j], bp[j]), x[e]);
        if (!on(k)) x[e] = 0.f;
      }
      if (on(k)) store<W>(xo + base + k * kStep, x + k * W);
    }
    moments<E, W>(x, a, on, G, member, red + kMaxWarps, mx, rx);
    if (G > 1 && !a.wp) group_barrier();  // these are written again before another barrier
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int i = kKeep ? k * W : 0;
      float o[W];
      if (!kKeep) param<W>(on(k) ? a.w : nullptr, c0 + k * kStep, 1.f, w);
      param<W>(kBias && on(k) ? a.b : nullptr, c0 + k * kStep, 0.f, b);
#pragma unroll
      for (int j = 0; j < W; ++j) o[j] = fmaf((x[k * W + j] - mx) * rx, w[i + j], b[j]);
      if (on(k)) store<W>(y + base + k * kStep, o);
    }
    if (member == 0 && (threadIdx.x & 31) == 0) stats[r] = make_float4(mh, rh, mx, rx);
  }
}

template <typename X, typename H, typename Y, int E, int W, bool kBias>
__global__ void __launch_bounds__(kFwdWarps * 32)  // for its registers: CTAs are smaller
    fwd_kernel(const Args a, X* xo, Y* y, float4* stats, int G, uint32_t rows) {
  __shared__ float2 red[2 * kMaxWarps];
  const int warp = threadIdx.x >> 5, groups = G == 1 ? (int)blockDim.x >> 5 : 1;
  const int group = G == 1 ? warp : 0, member = G == 1 ? 0 : warp;
  const int c0 = member * 32 * E + (threadIdx.x & 31) * W;
  const uint32_t run = blockIdx.x * groups + group;
  const uint32_t first = min(run * rows, a.N), last = min(first + rows, a.N);
  if (first >= last) return;  // the whole group
  if ((member + 1) * 32 * E <= a.C)
    fwd_rows<X, H, Y, E, W, kBias, true>(a, xo, y, stats, red, first, last, c0, member, G);
  else
    fwd_rows<X, H, Y, E, W, kBias, false>(a, xo, y, stats, red, first, last, c0, member, G);
}

// A warp for a row of up to 1024 columns, K * 4 a lane, when they can be read four at a time:
// no barriers, and rows enough in flight (16384 rows of 768: 31 us, against 41 us with three
// warps a row; wider rows would leave too few registers, single elements too many
// instructions: 9006 x 1999 53 us with eight warps a row, 89 us with four and more columns
// a lane).
constexpr int kWarpRows = 8;  // rows of a CTA
template <typename X, typename H, typename Y, int K>
__global__ void __launch_bounds__(kWarpRows * 32)
    fwd_warp_kernel(const Args a, X* xo, Y* y, float4* stats) {
  const int lane = threadIdx.x & 31, C = a.C;
  const uint32_t r = blockIdx.x * kWarpRows + (threadIdx.x >> 5);
  if (r >= a.N) return;
  const size_t base = (size_t)r * C;
  const X* xr = static_cast<const X*>(a.x) + base;
  const H* hr = static_cast<const H*>(a.h) + base;
  const float* gate = a.gate ? a.gate + (size_t)(r / a.T) * C : nullptr;
  auto column = [&](int k) { return (k * 32 + lane) * 4; };
  auto on = [&](int k) { return column(k) < C; };
  Raw<X, 4> xw[K];
  Raw<H, 4> hw[K];
#pragma unroll
  for (int k = 0; k < K; ++k)
    if (on(k)) {
      hw[k] = fetch<H, 4>(hr + column(k));
      xw[k] = fetch<X, 4>(xr + column(k));
    }
  float h[K * 4], x[K * 4];
#pragma unroll
  for (int k = 0; k < K; ++k) {
    if (on(k)) {
      unpack(hw[k], h + k * 4);
      unpack(xw[k], x + k * 4);
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j) h[k * 4 + j] = x[k * 4 + j] = 0.f;
    }
  }
  auto moments = [&](const float* v, float& mean, float& rstd) {
    mean = 0.f;
    if (!a.rms) {
      float s = 0.f;
#pragma unroll
      for (int e = 0; e < K * 4; ++e) s += v[e];
      mean = warp_sum(s) / C;
    }
    float q = 0.f;
#pragma unroll
    for (int e = 0; e < K * 4; ++e) {
      const float d = v[e] - mean;
      if (on(e / 4)) q = fmaf(d, d, q);
    }
    rstd = rsqrtf(warp_sum(q) / C + a.eps);
  };
  float mh = 0.f, rh = 1.f, mx, rx;
  if (a.wp) moments(h, mh, rh);
#pragma unroll
  for (int k = 0; k < K; ++k) {
    if (!on(k)) continue;
    float g[4], w[4], b[4];
    param<4>(gate, column(k), 1.f, g);
    param<4>(a.wp, column(k), 1.f, w);
    param<4>(a.bp, column(k), 0.f, b);
#pragma unroll
    for (int j = 0; j < 4; ++j)
      x[k * 4 + j] =
          fmaf(a.scale * g[j], fmaf((h[k * 4 + j] - mh) * rh, w[j], b[j]), x[k * 4 + j]);
    store<4>(xo + base + column(k), x + k * 4);
  }
  moments(x, mx, rx);
#pragma unroll
  for (int k = 0; k < K; ++k) {
    if (!on(k)) continue;
    float w[4], b[4], o[4];
    param<4>(a.w, column(k), 1.f, w);
    param<4>(a.b, column(k), 0.f, b);
#pragma unroll
    for (int j = 0; j < 4; ++j) o[j] = fmaf((x[k * 4 + j] - mx) * rx, w[j], b[j]);
    store<4>(y + base + column(k), o);
  }
  if (lane == 0) stats[r] = make_float4(mh, rh, mx, rx);
}

// ---- backward -----------------------------------------------------------------------
//
// The columns' sums (d weight and so on) stay in registers over a run of rows; each CTA
// writes one partial row of each (parts: (kParts, grid, pitch)), which a second kernel adds
// in a fixed order (bit-reproducible).  A gate for each sample has its sums written where the
// gate changes: one row for each (run, gate) that meet, at slot run + gate (each step along
// the rows raises one of the two, so no slot is shared).
// What binds it first is the issue of instructions, with 16 warps an SM to cover their
// latencies: some 25 for each element are the mathematics.  No more is kept in registers than
// 16 warps of 128 have room for.  16384 rows of 768 (fp32 stream, bf16 h and dy): 49 us, 4.6
// TB/s of the 226 MB; 9006 of 1999, bf16: 85 us.  Measured on the way: loads straight into
// registers 55 us, 24 columns a lane 62 us, rows shared by whole CTAs 85 to 108 us.

// Sums of a pair over the G warps of a row, the same in all of them.  red: the group's,
// member: this warp's place in it.
__device__ __forceinline__ void pair_sums(float& u, float& v, float2* red, int G, int member) {
  const int lane = threadIdx.x & 31;
  const bool upper = lane & 16;  // the upper lanes go on with v
  const float send = upper ? u : v;
  float t = (upper ? v : u) + __shfl_xor_sync(0xffffffffu, send, 16);
#pragma unroll
  for (int o = 8; o > 0; o >>= 1) t += __shfl_xor_sync(0xffffffffu, t, o);
  if (G == 1) {
    u = __shfl_sync(0xffffffffu, t, 0);
    v = __shfl_sync(0xffffffffu, t, 16);
    return;
  }
  if ((lane & 15) == 0) reinterpret_cast<float*>(red + member)[lane >> 4] = t;
  group_barrier();
  // the places of members that are not there hold zeros
  const float4* all = reinterpret_cast<const float4*>(red);
  const float4 p = all[0], q = all[1];
  u = (p.x + p.z) + (q.x + q.z);
  v = (p.y + p.w) + (q.y + q.w);
  if (G > 4) {
    const float4 r = all[2], t = all[3];
    u += (r.x + r.z) + (t.x + t.z);
    v += (r.y + r.w) + (t.y + t.w);
  }
  if (G > 8)
#pragma unroll
    for (int i = 4; i < kMaxWarps / 2; i += 2) {
      const float4 r = all[i], t = all[i + 1];
      u += (r.x + r.z) + (t.x + t.z);
      v += (r.y + r.w) + (t.y + t.w);
    }
}

// A warp's 32 E columns of a row on their way through shared memory, a row ahead of its use:
// the next row's loads then neither wait for this one's barriers nor take registers.
// Four elements a lane: each lane copies and reads its own.  Single elements: the warp copies
// the stretch in whole 16-byte pieces, from the boundary before it to the one after (other
// elements there are not used), so that rows of any phase arrive at full speed; a piece that
// would reach past the tensor is copied element by element.
template <typename T, int E>
__host__ __device__ constexpr int stage_bytes() {
  return 32 * E * (int)sizeof(T) + 32;
}

template <typename X, typename H, typename Y, int E>
__host__ __device__ constexpr int bwd_slot() {  // x, dx', h and dy
  return 2 * stage_bytes<X, E>() + stage_bytes<H, E>() + stage_bytes<Y, E>();
}

template <int kBytes>
__device__ __forceinline__ void cp_async(uint32_t to, const void* from) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"(to), "l"(from), "n"(kBytes)
               : "memory");
}

// Starts the copy of elements [at, at + n) of p, which has `all`, to `to` (kFull: n = 32 E), of
// which `to_shared` is the address in shared memory.
template <typename T, int E, int W, bool kFull>
__device__ __forceinline__ void stage_in(char* to, uint32_t to_shared, const T* p, size_t at, int n,
                                         size_t all) {
  const int lane = threadIdx.x & 31;
  if constexpr (W == 4) {
    const T* from = p + at + lane * 4;
    to_shared += lane * 4 * sizeof(T);
#pragma unroll
    for (int k = 0; k < E / 4; ++k)
      if (kFull || (k * 32 + lane) * 4 < n)
        cp_async<4 * sizeof(T)>(to_shared + k * 128 * sizeof(T), from + k * 128);
  } else {
    const uintptr_t from = reinterpret_cast<uintptr_t>(p + at), first = from & ~(uintptr_t)15;
    const uintptr_t lo = reinterpret_cast<uintptr_t>(p), hi = reinterpret_cast<uintptr_t>(p + all);
    const int pieces = (int)((from + n * sizeof(T) - first + 15) / 16);
    for (int i = lane; i < pieces; i += 32) {
      const uintptr_t piece = first + (uintptr_t)i * 16;
      if (piece >= lo && piece + 16 <= hi)
        cp_async<16>(to_shared + i * 16, reinterpret_cast<const void*>(piece));
      else
        for (uintptr_t b = piece; b < piece + 16; b += sizeof(T))
          if (b >= lo && b < hi)
            *reinterpret_cast<T*>(to + (b - first)) = *reinterpret_cast<const T*>(b);
    }
  }
}
// The lane's k-th group of those elements.
template <typename T, int W>
__device__ __forceinline__ Raw<T, W> staged(const char* to, const T* p, size_t at, int k) {
  const int c = (k * 32 + (int)(threadIdx.x & 31)) * W;
  const int phase = W == 4 ? 0 : (int)(reinterpret_cast<uintptr_t>(p + at) & 15);
  return *reinterpret_cast<const Raw<T, W>*>(to + phase + c * sizeof(T));
}

template <int E>
struct ColumnSums {
  float w[E], b[E], wp[E], bp[E], g[E];
};

struct BwdArgs {
  const float4* stats;
  float *parts, *gate_parts;
  int pitch, G;
  uint32_t rows;
};

// Rows [first, last) of one warp, whose lanes' columns start at c0.  kFull: all of them exist.
template <typename X, typename H, typename Y, int E, int W, bool kBias, bool kFull>
__device__ __forceinline__ void bwd_rows(const Args& a, const BwdArgs& p, const Y* dy,
                                         const X* dxo, X* dx, H* dh, ColumnSums<E>& sum,
                                         float2* red, char* stage, uint32_t run, uint32_t first,
                                         uint32_t last, int c0, int member) {
  constexpr int K = E / W, kStep = 32 * W;
  constexpr bool kKeep = !kBias;  // the gate and post weight in registers
  const int C = a.C;
  auto on = [&](int k) { return kFull || c0 + k * kStep < C; };
  const float inv = 1.f / C, mean_inv = a.rms ? 0.f : inv;
  float w[W], bp[W], wp[kKeep ? E : W], gw[kKeep ? E : W];
  auto load_wp = [&](int k, int i) { param<W>(on(k) ? a.wp : nullptr, c0 + k * kStep, 1.f, wp + i); };
  auto load_gate = [&](const float* gate, int k, int i) {
    param<W>(on(k) ? gate : nullptr, c0 + k * kStep, 1.f, gw + i);
#pragma unroll
    for (int j = 0; j < W; ++j) gw[i + j] *= a.scale;
  };
  uint32_t grp = first / a.T, turn = (grp + 1) * a.T;  // the gate, and the row where it ends
  const float* gate = a.gate ? a.gate + (size_t)grp * C : nullptr;
  if (kKeep)
#pragma unroll
    for (int k = 0; k < K; ++k) {
      load_wp(k, k * W);
      load_gate(gate, k, k * W);
    }
  const X* xp = static_cast<const X*>(a.x);
  const H* hp = static_cast<const H*>(a.h);
  const size_t all = (size_t)a.N * C;
  const int w0 = member * 32 * E, here = kFull ? 32 * E : C - w0;  // the warp's columns
  constexpr int kX = stage_bytes<X, E>(), kH = stage_bytes<H, E>(), kY = stage_bytes<Y, E>();
  constexpr int kSlot = bwd_slot<X, H, Y, E>();
  const uint32_t stage_shared = (uint32_t)__cvta_generic_to_shared(stage);
  auto start = [&](uint32_t r, int slot) {
    if (r < last) {
      char* to = stage + slot * kSlot;
      const uint32_t ts = stage_shared + slot * kSlot;
      const size_t at = (size_t)r * C + w0;
      stage_in<H, E, W, kFull>(to, ts, hp, at, here, all);
      stage_in<X, E, W, kFull>(to + kH, ts + kH, xp, at, here, all);
      stage_in<Y, E, W, kFull>(to + kH + kX, ts + kH + kX, dy, at, here, all);
      if (dxo)
        stage_in<X, E, W, kFull>(to + kH + kX + kY, ts + kH + kX + kY, dxo, at, here, all);
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  start(first, 0);
  float4 st = p.stats[first];
  int flip = 0, slot = 0;
  for (uint32_t r = first; r < last; ++r, slot ^= 1) {
    const size_t base = (size_t)r * C + c0, at = (size_t)r * C + w0;
    const char* in = stage + slot * kSlot;
    if (W == 1) __syncwarp();  // the other slot has been read
    start(r + 1, slot ^ 1);
    const float4 next = r + 1 < last ? p.stats[r + 1] : st;
    asm volatile("cp.async.wait_group 1;" ::: "memory");
    if (W == 1) __syncwarp();
    Raw<X, W> xw[K];
    Raw<H, W> hw[K];
    Raw<Y, W> yw[K];
#pragma unroll
    for (int k = 0; k < K; ++k) {
      hw[k] = staged<H, W>(in, hp, at, k);
      xw[k] = staged<X, W>(in + kH, xp, at, k);
      yw[k] = staged<Y, W>(in + kH + kX, dy, at, k);
    }
    if (r == turn) {
      ++grp, turn += a.T;
      if (a.gate) {
        gate += C;
        if (kKeep)
#pragma unroll
          for (int k = 0; k < K; ++k) load_gate(gate, k, k * W);
      }
    }
    const float mh = -st.x * st.y, mx = -st.z * st.w;
    float D[E], xh[E], hh[E], s0 = 0.f, s1 = 0.f, t0 = 0.f, t1 = 0.f;  // D is u
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int i = kKeep ? k * W : 0;
      if (!kKeep) load_wp(k, 0), load_gate(gate, k, 0);
      if (on(k))
        unpack(fetch<float, W>(a.w + c0 + k * kStep), w);
      else
#pragma unroll
        for (int j = 0; j < W; ++j) w[j] = 0.f;
      param<W>(kBias && on(k) ? a.bp : nullptr, c0 + k * kStep, 0.f, bp);
      unpack(hw[k], hh + k * W);
      unpack(xw[k], xh + k * W);
      unpack(yw[k], D + k * W);
#pragma unroll
      for (int j = 0; j < W; ++j) {
        const int e = k * W + j;
        hh[e] = fmaf(hh[e], st.y, mh);  // h itself without a post norm
        xh[e] = fmaf(fmaf(gw[i + j], fmaf(hh[e], wp[i + j], bp[j]), xh[e]), st.w, mx);
        if (!on(k)) D[e] = xh[e] = hh[e] = 0.f;
        sum.w[e] = fmaf(D[e], xh[e], sum.w[e]);
        if (kBias) sum.b[e] += D[e];
        D[e] *= w[j];
        (e & 1 ? t0 : s0) += D[e];
        float& s = e & 1 ? t1 : s1;
        s = fmaf(D[e], xh[e], s);
      }
    }
    s0 += t0, s1 += t1;
    pair_sums(s0, s1, red + flip * kMaxWarps, p.G, member);
    flip ^= 1;
    const float k0 = -st.w * (s0 * mean_inv), k1 = -s1 * inv;
    float q0 = 0.f, q1 = 0.f;
    t0 = t1 = 0.f;
    X* dxr = dx + base;
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int i = kKeep ? k * W : 0;
      float d[W];
      if (dxo)
        unpack(staged<X, W>(in + kH + kX + kY, dxo, at, k), d);
      else
#pragma unroll
        for (int j = 0; j < W; ++j) d[j] = 0.f;
      if (!kKeep) load_wp(k, 0), load_gate(gate, k, 0);
      param<W>(kBias && on(k) ? a.bp : nullptr, c0 + k * kStep, 0.f, bp);
#pragma unroll
      for (int j = 0; j < W; ++j) {
        const int e = k * W + j;
        d[j] += fmaf(st.w, fmaf(xh[e], k1, D[e]), k0);
        if (!on(k)) d[j] = 0.f;
        sum.g[e] = fmaf(d[j], fmaf(hh[e], wp[i + j], bp[j]), sum.g[e]);
        const float dn = d[j] * gw[i + j];
        sum.wp[e] = fmaf(dn, hh[e], sum.wp[e]);
        if (kBias) sum.bp[e] += dn;
        D[e] = dn * wp[i + j];
        (e & 1 ? t0 : q0) += D[e];
        float& q = e & 1 ? t1 : q1;
        q = fmaf(D[e], hh[e], q);
      }
      if (on(k)) store<W>(dxr + k * kStep, d);
    }
    float l0 = 0.f, l1 = 0.f;
    if (a.wp) {
      q0 += t0, q1 += t1;
      pair_sums(q0, q1, red + flip * kMaxWarps, p.G, member);
      flip ^= 1;
      l0 = -st.y * (q0 * mean_inv), l1 = -q1 * inv;
    }
    H* dhr = dh + base;
#pragma unroll
    for (int k = 0; k < K; ++k) {
      float o[W];
#pragma unroll
      for (int j = 0; j < W; ++j)  // 1/std is 1 without a post norm
        o[j] = fmaf(st.y, fmaf(hh[k * W + j], l1, D[k * W + j]), l0);
      if (on(k)) store<W>(dhr + k * kStep, o);
    }
    if (p.gate_parts && (r + 1 == last || r + 1 == turn)) {
      float* out = p.gate_parts + ((size_t)run + grp) * p.pitch + c0;
#pragma unroll
      for (int k = 0; k < K; ++k)
#pragma unroll
        for (int j = 0; j < W; ++j) {
          if (on(k)) out[k * kStep + j] = a.scale * sum.g[k * W + j];
          sum.g[k * W + j] = 0.f;
        }
    }
    st = next;
  }
  asm volatile("cp.async.wait_group 0;" ::: "memory");
}

template <typename X, typename H, typename Y, int E, int W, bool kBias>
__global__ void __launch_bounds__(kBwdWarps * 32)
    bwd_kernel(const Args a, const BwdArgs p, const Y* dy, const X* dxo, X* dx, H* dh) {
  constexpr int K = E / W, kStep = 32 * W;
  extern __shared__ __align__(16) char stages[];
  static_assert(2 * bwd_slot<X, H, Y, E>() >= 32 * E * (int)sizeof(float), "a warp's sums");
  __shared__ __align__(16) float2 red[2 * kMaxWarps];
  const int C = a.C, warp = threadIdx.x >> 5, groups = p.G == 1 ? (int)blockDim.x >> 5 : 1;
  const int group = p.G == 1 ? warp : 0, member = p.G == 1 ? 0 : warp;
  const int c0 = member * 32 * E + (threadIdx.x & 31) * W;
  const uint32_t run = blockIdx.x * groups + group;
  const uint32_t first = min(run * p.rows, a.N), last = min(first + p.rows, a.N);
  if (threadIdx.x < 2 * kMaxWarps) red[threadIdx.x] = make_float2(0.f, 0.f);
  __syncthreads();
  ColumnSums<E> sum;
#pragma unroll
  for (int e = 0; e < E; ++e) sum.w[e] = sum.b[e] = sum.wp[e] = sum.bp[e] = sum.g[e] = 0.f;
  char* stage = stages + warp * (2 * bwd_slot<X, H, Y, E>());
  if (first < last) {
    if ((member + 1) * 32 * E <= C)
      bwd_rows<X, H, Y, E, W, kBias, true>(a, p, dy, dxo, dx, dh, sum, red, stage, run, first,
                                           last, c0, member);
    else
      bwd_rows<X, H, Y, E, W, kBias, false>(a, p, dy, dxo, dx, dh, sum, red, stage, run, first,
                                            last, c0, member);
  }
  // the groups' sums, added in order: a row of each, where the staged rows were
  float* sums = reinterpret_cast<float*>(stages);
  auto total = [&](const float* v, float f, int part) {
    __syncthreads();
#pragma unroll
    for (int k = 0; k < K; ++k)
      if (c0 + k * kStep < C)
#pragma unroll
        for (int j = 0; j < W; ++j) sums[group * C + c0 + k * kStep + j] = v[k * W + j];
    __syncthreads();
    float* out = p.parts + ((size_t)part * gridDim.x + blockIdx.x) * p.pitch;
    for (int c = threadIdx.x; c < C; c += blockDim.x) {
      float t = 0.f;
      for (int i = 0; i < groups; ++i) t += sums[i * C + c];
      out[c] = f * t;
    }
  };
  total(sum.w, 1.f, 0);
  if (kBias && a.b) total(sum.b, 1.f, 1);
  if (a.wp) total(sum.wp, 1.f, 2);
  if (kBias && a.bp) total(sum.bp, 1.f, 3);
  if (a.gate && !p.gate_parts) total(sum.g, a.scale, 4);
}

struct Sums {
  const float* parts;
  float* out[kParts];
  const float* gate_parts;
  float* dgate;
  int64_t N, T, rows;
  int C, pitch, ctas;
};

// Column sums of the partial rows: blockIdx.y < kParts one parameter's gradient, else that of
// gate blockIdx.y - kParts from the rows of the runs it meets.  A CTA takes 32 columns: thread
// (g, j) of 64 x 8 adds rows g, g + 64, ... of four columns, then the 64 are added in order.
__global__ void __launch_bounds__(512) sums_kernel(const Sums s) {
  constexpr int kGroups = 64;
  __shared__ float red[kGroups][33];
  const int j = threadIdx.x & 7, grp = threadIdx.x >> 3;
  const int c = blockIdx.x * 32 + j * 4;
  const int y = blockIdx.y;
  const float* in;
  float* out;
  int count = s.ctas;
  if (y < kParts) {
    in = s.parts + (size_t)y * s.ctas * s.pitch;
    out = s.out[y];
  } else {
    const int64_t g = y - kParts, first = g * s.T / s.rows;
    const int64_t end = min((g + 1) * s.T, s.N);
    count = (int)((end - 1) / s.rows - first + 1);
    in = s.gate_parts + (first + g) * s.pitch;
    out = s.dgate ? s.dgate + g * s.C : nullptr;
  }
  if (!out) return;
  float4 t = make_float4(0.f, 0.f, 0.f, 0.f);
  if (c < s.pitch) {
#pragma unroll 8
    for (int r = grp; r < count; r += kGroups) {
      const float4 v = *reinterpret_cast<const float4*>(in + (size_t)r * s.pitch + c);
      t.x += v.x, t.y += v.y, t.z += v.z, t.w += v.w;
    }
  }
  red[grp][j * 4] = t.x, red[grp][j * 4 + 1] = t.y;
  red[grp][j * 4 + 2] = t.z, red[grp][j * 4 + 3] = t.w;
  __syncthreads();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;  // two columns a warp
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    const int col = warp * 2 + k, at = blockIdx.x * 32 + col;
    const float u = warp_sum(red[lane][col] + red[lane + 32][col]);
    if (lane == 0 && at < s.C) out[at] = u;
  }
}

bool aligned(const void* p, int bytes) {
  return (reinterpret_cast<uintptr_t>(p) & (bytes - 1)) == 0;
}

bool known(int dtype) { return dtype == SQB_BF16 || dtype == SQB_F32; }
int elt_of(int dtype) { return dtype == SQB_BF16 ? 2 : 4; }

// How N rows of C columns are dealt out: groups of G warps whose lanes hold E columns (8, or 4
// where one warp then has the row), as many CTAs of one group (or of eight groups of one warp)
// on each of 148 SMs as `warps` allow, runs of as many rows each.
struct Plan {
  int G, E, groups, ctas, runs, pitch;
  uint32_t rows;
};

Plan plan_of(int64_t N, int64_t C, int warps) {
  Plan p;
  p.E = C <= 128 ? 4 : 8;
  p.G = (int)((C + 32 * p.E - 1) / (32 * p.E));
  p.groups = p.G == 1 ? 8 : 1;
  const int per_sm = warps / (p.G * p.groups);
  const int64_t all = (int64_t)148 * per_sm * p.groups;
  p.rows = (uint32_t)((N + all - 1) / all);
  p.runs = (int)((N + p.rows - 1) / p.rows);
  p.ctas = (p.runs + p.groups - 1) / p.groups;
  p.pitch = (int)((C + 3) / 4 * 4);
  return p;
}

int check(const Args& a, int64_t N, int64_t C, int x_dtype, int h_dtype, int y_dtype,
          int64_t gates) {
  if (!a.x || !a.h || !a.w || N <= 0 || N > INT32_MAX || (a.bp && !a.wp)) return SQB_ERR_ARG;
  if (a.gate && (gates <= 0 || N % gates != 0)) return SQB_ERR_ARG;
  if (!known(x_dtype) || !known(h_dtype) || !known(y_dtype)) return SQB_ERR_DTYPE;
  if (C <= 0 || C > kMaxC) return SQB_ERR_UNSUPPORTED;
  const float* const parameters[] = {a.w, a.b, a.wp, a.bp, a.gate};
  for (const float* p : parameters)
    if (!aligned(p, 4)) return SQB_ERR_ALIGN;
  return aligned(a.x, elt_of(x_dtype)) && aligned(a.h, elt_of(h_dtype)) ? SQB_OK : SQB_ERR_ALIGN;
}

// Whether every row can be read four elements at a time.
bool wide(const Args& a, const void* const* more, int n) {
  if (a.C % 4) return false;
  const void* all[] = {a.x, a.h, a.w, a.b, a.wp, a.bp, a.gate};
  for (const void* p : all)
    if (!aligned(p, 16)) return false;
  for (int i = 0; i < n; ++i)
    if (!aligned(more[i], 16)) return false;
  return true;
}

Args make_args(const void* x, const void* h, const float* w, const float* b, const float* wp,
               const float* bp, const float* gate, int64_t gates, float scale, float eps, int rms,
               int64_t N, int64_t C) {
  Args a;
  a.x = x, a.h = h, a.w = w, a.b = b, a.wp = wp, a.bp = bp, a.gate = gate;
  a.scale = scale, a.eps = eps, a.N = (uint32_t)N;
  a.T = (uint32_t)(gate && gates > 0 && N >= gates ? N / gates : N);
  a.C = (int)C;
  a.rms = rms != 0;
  return a;
}

// Calls f(X(), H(), Y()) for the three dtypes.
template <typename F>
void by_type(int x, int h, int y, F&& f) {
  auto second = [&](auto X) {
    auto third = [&](auto H) {
      if (y == SQB_BF16)
        f(X, H, __nv_bfloat16());
      else
        f(X, H, float());
    };
    if (h == SQB_BF16)
      third(__nv_bfloat16());
    else
      third(float());
  };
  if (x == SQB_BF16)
    second(__nv_bfloat16());
  else
    second(float());
}

}  // namespace
}  // namespace resnorm
}  // namespace sqb

using namespace sqb::resnorm;

extern "C" int sqb_residual_norm_fwd(const void* x, int x_dtype, const void* h, int h_dtype,
                                     const float* weight, const float* bias,
                                     const float* post_weight, const float* post_bias,
                                     const float* gate, int64_t gates, float scale, float eps,
                                     int rms, void* x_out, void* y, int y_dtype, float* stats,
                                     int64_t N, int64_t C, void* stream) {
  const Args a = make_args(x, h, weight, bias, post_weight, post_bias, gate, gates, scale, eps,
                           rms, N, C);
  if (const int rc = check(a, N, C, x_dtype, h_dtype, y_dtype, gates)) return rc;
  if (!x_out || !y || !stats) return SQB_ERR_ARG;
  if (!aligned(stats, 16) || !aligned(x_out, elt_of(x_dtype)) || !aligned(y, elt_of(y_dtype)))
    return SQB_ERR_ALIGN;
  cudaStream_t q = static_cast<cudaStream_t>(stream);
  const void* more[] = {x_out, y};
  const bool w4 = wide(a, more, 2), biased = bias || post_bias;
  const Plan p = plan_of(N, C, kFwdWarps);
  float4* st = reinterpret_cast<float4*>(stats);
  by_type(x_dtype, h_dtype, y_dtype, [&](auto tx, auto th, auto ty) {
    using X = decltype(tx);
    using H = decltype(th);
    using Y = decltype(ty);
    auto run = [&](auto kernel) {
      kernel<<<p.ctas, 32 * p.G * p.groups, 0, q>>>(a, static_cast<X*>(x_out),
                                                    static_cast<Y*>(y), st, p.G, p.rows);
    };
    auto sized = [&](auto biased_) {
      constexpr bool kb = decltype(biased_)::value;
      if (p.E == 8)
        w4 ? run(fwd_kernel<X, H, Y, 8, 4, kb>) : run(fwd_kernel<X, H, Y, 8, 1, kb>);
      else
        w4 ? run(fwd_kernel<X, H, Y, 4, 4, kb>) : run(fwd_kernel<X, H, Y, 4, 1, kb>);
    };
    auto one_warp = [&](auto kernel) {
      kernel<<<(unsigned)((N + kWarpRows - 1) / kWarpRows), kWarpRows * 32, 0, q>>>(a, static_cast<X*>(x_out),
                                                             static_cast<Y*>(y), st);
    };
    if (w4 && C <= 128)
      one_warp(fwd_warp_kernel<X, H, Y, 1>);
    else if (w4 && C <= 256)
      one_warp(fwd_warp_kernel<X, H, Y, 2>);
    else if (w4 && C <= 512)
      one_warp(fwd_warp_kernel<X, H, Y, 4>);
    else if (w4 && C <= 768)
      one_warp(fwd_warp_kernel<X, H, Y, 6>);
    else if (w4 && C <= 1024)
      one_warp(fwd_warp_kernel<X, H, Y, 8>);
    else
      biased ? sized(std::true_type()) : sized(std::false_type());
  });
  return cudaGetLastError() == cudaSuccess ? SQB_OK : SQB_ERR_LAUNCH;
}

extern "C" size_t sqb_residual_norm_workspace_bytes(int64_t N, int64_t C, int64_t gates) {
  if (N <= 0 || N > INT32_MAX || C <= 0 || C > kMaxC || gates < 0) return 0;
  // partial rows of the CTAs, and one for each run and gate that meet
  const Plan p = plan_of(N, C, kBwdWarps);
  return ((size_t)kParts * p.ctas + (gates > 1 ? (size_t)p.runs + gates : 0)) * p.pitch *
         sizeof(float);
}

extern "C" int sqb_residual_norm_bwd(const void* dy, int y_dtype, const void* dx_out,
                                     const void* x, int x_dtype, const void* h, int h_dtype,
                                     const float* weight, const float* bias,
                                     const float* post_weight, const float* post_bias,
                                     const float* gate, int64_t gates, float scale, float eps,
                                     int rms, const float* stats, void* dx, void* dh,
                                     float* dweight, float* dbias, float* dpost_weight,
                                     float* dpost_bias, float* dgate, void* workspace,
                                     size_t ws_bytes, int64_t N, int64_t C, void* stream) {
  const Args a = make_args(x, h, weight, bias, post_weight, post_bias, gate, gates, scale, eps,
                           rms, N, C);
  if (const int rc = check(a, N, C, x_dtype, h_dtype, y_dtype, gates)) return rc;
  if (!dy || !stats || !dx || !dh || !dweight || (bias && !dbias) ||
      (post_weight && !dpost_weight) || (post_bias && !dpost_bias) || (gate && !dgate))
    return SQB_ERR_ARG;
  if (gate && gates > 65535 - kParts) return SQB_ERR_UNSUPPORTED;
  if (!workspace || ws_bytes < sqb_residual_norm_workspace_bytes(N, C, gate ? gates : 0))
    return SQB_ERR_WORKSPACE;
  if (!aligned(stats, 16) || !aligned(workspace, 16) || !aligned(dy, elt_of(y_dtype)) ||
      !aligned(dx_out, elt_of(x_dtype)) || !aligned(dx, elt_of(x_dtype)) ||
      !aligned(dh, elt_of(h_dtype)))
    return SQB_ERR_ALIGN;
  const float* const gradients[] = {dweight, dbias, dpost_weight, dpost_bias, dgate};
  for (const float* p : gradients)
    if (!aligned(p, 4)) return SQB_ERR_ALIGN;
  cudaStream_t q = static_cast<cudaStream_t>(stream);
  const void* more[] = {dy, dx_out, dx, dh};
  const bool w4 = wide(a, more, 4), biased = bias || post_bias;
  const Plan p = plan_of(N, C, kBwdWarps);
  float* parts = static_cast<float*>(workspace);
  float* gate_parts = gate && gates > 1 ? parts + (size_t)kParts * p.ctas * p.pitch : nullptr;
  const BwdArgs more_args{reinterpret_cast<const float4*>(stats), parts, gate_parts, p.pitch, p.G,
                          p.rows};
  bool ok = true;
  by_type(x_dtype, h_dtype, y_dtype, [&](auto tx, auto th, auto ty) {
    using X = decltype(tx);
    using H = decltype(th);
    using Y = decltype(ty);
    auto run = [&](auto kernel) {
      const int warps = p.G * p.groups;
      const int warp = 2 * (p.E == 8 ? bwd_slot<X, H, Y, 8>() : bwd_slot<X, H, Y, 4>());
      const int smem = warps * warp;
      // the limit belongs to the kernel, whatever thread launches it: always the most that any
      // width takes
      ok = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                kMaxWarps * warp) == cudaSuccess;
      if (!ok) return;
      kernel<<<p.ctas, 32 * warps, smem, q>>>(
          a, more_args, static_cast<const Y*>(dy), static_cast<const X*>(dx_out),
          static_cast<X*>(dx), static_cast<H*>(dh));
    };
    auto sized = [&](auto biased_) {
      constexpr bool kb = decltype(biased_)::value;
      if (p.E == 8)
        w4 ? run(bwd_kernel<X, H, Y, 8, 4, kb>) : run(bwd_kernel<X, H, Y, 8, 1, kb>);
      else
        w4 ? run(bwd_kernel<X, H, Y, 4, 4, kb>) : run(bwd_kernel<X, H, Y, 4, 1, kb>);
    };
    biased ? sized(std::true_type()) : sized(std::false_type());
  });
  if (!ok) return SQB_ERR_CUDA;
  Sums s;
  s.parts = parts;
  s.out[0] = dweight, s.out[1] = bias ? dbias : nullptr;
  s.out[2] = post_weight ? dpost_weight : nullptr, s.out[3] = post_bias ? dpost_bias : nullptr;
  s.out[4] = gate && !gate_parts ? dgate : nullptr;
  s.gate_parts = gate_parts, s.dgate = dgate;
  s.N = N, s.T = a.T, s.rows = p.rows, s.C = (int)C, s.pitch = p.pitch, s.ctas = p.ctas;
  const dim3 grid((unsigned)((C + 31) / 32), (unsigned)(kParts + (gate_parts ? gates : 0)));
  sums_kernel<<<grid, 512, 0, q>>>(s);
  return cudaGetLastError() == cudaSuccess ? SQB_OK : SQB_ERR_LAUNCH;
}
