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
// One CTA per row, the row in registers (E elements a thread).  Both norms' statistics
// are saved; the backward forms x' again from x and h in fp32, so that a stream kept
// in bf16 is not rounded between the two passes.  Variances are of differences from
// the mean (two sweeps over registers), never E[v^2] - mean^2.  The backward's CTAs
// each take a run of rows, keep their columns' sums in registers and write one partial
// row; a second kernel adds the partials in a fixed order (bit-reproducible).
// Bound by HBM for large batches: forward reads x, h and writes x', y; backward reads
// x, h, dy, dx' and writes dx, dh.

#include <cuda_bf16.h>
#include <math.h>
#include <stdint.h>

#include "sqb_train.h"

namespace sqb {
namespace resnorm {
namespace {

constexpr int kMaxC = 4096;
constexpr int kParts = 4;  // d weight, d bias, d post weight, d post bias

struct Args {
  const void *x, *h;
  const float *w, *b, *wp, *bp, *gate;
  float scale, eps;
  int64_t N, T;  // rows, rows that share a gate (N for one gate)
  int C;
  bool rms, x_bf16, h_bf16, y_bf16;
};

// W consecutive elements of a row of either type, and their stores.
template <int W>
__device__ __forceinline__ void load(const void* p, bool bf16, int64_t i, float* v) {
  if constexpr (W == 4) {
    if (bf16) {
      const uint2 u = *reinterpret_cast<const uint2*>(static_cast<const __nv_bfloat16*>(p) + i);
      const float2 a = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&u.x));
      const float2 b = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&u.y));
      v[0] = a.x, v[1] = a.y, v[2] = b.x, v[3] = b.y;
    } else {
      const float4 a = *reinterpret_cast<const float4*>(static_cast<const float*>(p) + i);
      v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w;
    }
  } else {
    v[0] = bf16 ? __bfloat162float(static_cast<const __nv_bfloat16*>(p)[i])
                : static_cast<const float*>(p)[i];
  }
}

template <int W>
__device__ __forceinline__ void store(void* p, bool bf16, int64_t i, const float* v) {
  if constexpr (W == 4) {
    if (bf16) {
      const __nv_bfloat162 a = __floats2bfloat162_rn(v[0], v[1]);
      const __nv_bfloat162 b = __floats2bfloat162_rn(v[2], v[3]);
      uint2 u;
      u.x = *reinterpret_cast<const uint32_t*>(&a);
      u.y = *reinterpret_cast<const uint32_t*>(&b);
      *reinterpret_cast<uint2*>(static_cast<__nv_bfloat16*>(p) + i) = u;
    } else {
      *reinterpret_cast<float4*>(static_cast<float*>(p) + i) =
          make_float4(v[0], v[1], v[2], v[3]);
    }
  } else {
    if (bf16)
      static_cast<__nv_bfloat16*>(p)[i] = __float2bfloat16_rn(v[0]);
    else
      static_cast<float*>(p)[i] = v[0];
  }
}

// Column of the thread's k-th group of W elements.
template <int W>
__device__ __forceinline__ int column(int k) {
  return (k * (int)blockDim.x + (int)threadIdx.x) * W;
}

// Sums of K values over the CTA, the same in every thread.  red: K * 32 floats; the
// caller alternates two such buffers, so one barrier separates a buffer's uses.
template <int K>
__device__ __forceinline__ void block_sums(float* v, float* red) {
#pragma unroll
  for (int k = 0; k < K; ++k)
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v[k] += __shfl_xor_sync(0xffffffffu, v[k], o);
  const int warps = blockDim.x >> 5;
  if (warps == 1) return;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (lane == 0)
#pragma unroll
    for (int k = 0; k < K; ++k) red[k * 32 + warp] = v[k];
  __syncthreads();
#pragma unroll
  for (int k = 0; k < K; ++k) {
    v[k] = lane < warps ? red[k * 32 + lane] : 0.f;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v[k] += __shfl_xor_sync(0xffffffffu, v[k], o);
  }
}

// Mean (0 for RMS) and 1/std of a row held as v[E], columns past C excluded.
template <int E, int W>
__device__ __forceinline__ void moments(const float* v, const Args& a, float* red0, float* red1,
                                        float& mean, float& rstd) {
  mean = 0.f;
  if (!a.rms) {
    float s = 0.f;
#pragma unroll
    for (int e = 0; e < E; ++e) s += v[e];  // columns past C hold 0
    block_sums<1>(&s, red0);
    mean = s / a.C;
  }
  float q = 0.f;
#pragma unroll
  for (int k = 0; k < E / W; ++k)
    if (column<W>(k) < a.C)
#pragma unroll
      for (int j = 0; j < W; ++j) {
        const float d = v[k * W + j] - mean;
        q += d * d;
      }
  block_sums<1>(&q, red1);
  rstd = rsqrtf(q / a.C + a.eps);
}

// scale * gate and the post norm's weight and bias for the thread's columns.
template <int W>
__device__ __forceinline__ void gate_of(const Args& a, const float* gate, int c, float* g) {
  if (gate)
    load<W>(gate, false, c, g);
  else
#pragma unroll
    for (int j = 0; j < W; ++j) g[j] = 1.f;
#pragma unroll
  for (int j = 0; j < W; ++j) g[j] *= a.scale;
}

template <int E, int W>
__global__ void __launch_bounds__(E == 4 ? 256 : 512) fwd_kernel(Args a, void* xo, void* y, float4* stats) {
  __shared__ float red[4][32];
  const int64_t r = blockIdx.x, base = r * a.C;
  const float* gate = a.gate ? a.gate + (r / a.T) * a.C : nullptr;
  float h[E], x[E];
#pragma unroll
  for (int k = 0; k < E / W; ++k) {
    const int c = column<W>(k);
    if (c < a.C) {
      load<W>(a.h, a.h_bf16, base + c, h + k * W);
      load<W>(a.x, a.x_bf16, base + c, x + k * W);
    } else {
#pragma unroll
      for (int j = 0; j < W; ++j) h[k * W + j] = x[k * W + j] = 0.f;
    }
  }
  float mh = 0.f, rh = 1.f, mx, rx;
  if (a.wp) moments<E, W>(h, a, red[0], red[1], mh, rh);
#pragma unroll
  for (int k = 0; k < E / W; ++k) {
    const int c = column<W>(k);
    if (c >= a.C) continue;
    float g[W], w[W], b[W];
    gate_of<W>(a, gate, c, g);
    if (a.wp) load<W>(a.wp, false, c, w);
    if (a.bp) load<W>(a.bp, false, c, b);
#pragma unroll
    for (int j = 0; j < W; ++j) {
      float n = h[k * W + j];
      if (a.wp) n = (n - mh) * rh * w[j] + (a.bp ? b[j] : 0.f);
      x[k * W + j] += g[j] * n;
    }
    store<W>(xo, a.x_bf16, base + c, x + k * W);
  }
  moments<E, W>(x, a, red[2], red[3], mx, rx);
#pragma unroll
  for (int k = 0; k < E / W; ++k) {
    const int c = column<W>(k);
    if (c >= a.C) continue;
    float w[W], b[W], o[W];
    load<W>(a.w, false, c, w);
    if (a.b) load<W>(a.b, false, c, b);
#pragma unroll
    for (int j = 0; j < W; ++j)
      o[j] = (x[k * W + j] - mx) * rx * w[j] + (a.b ? b[j] : 0.f);
    store<W>(y, a.y_bf16, base + c, o);
  }
  if (threadIdx.x == 0) stats[r] = make_float4(mh, rh, mx, rx);
}

// CTA i takes rows [i * rows, (i + 1) * rows).  parts: (kParts, grid, C) column sums of
// the CTAs; gate_parts: one row of C for each (CTA, gate) that meet, at slot
// CTA + gate (each step along the rows raises one of the two, so no slot is shared).
template <int E, int W>
__global__ void __launch_bounds__(E == 4 ? 256 : 512) bwd_kernel(Args a, const void* dy, const void* dxo, const float4* stats, void* dx,
                           void* dh, float* parts, float* gate_parts, int64_t rows) {
  __shared__ float red[2][64];
  const int64_t first = (int64_t)blockIdx.x * rows, last = min(first + rows, a.N);
  float sw[E], sb[E], swp[E], sbp[E], sg[E];
#pragma unroll
  for (int e = 0; e < E; ++e) sw[e] = sb[e] = swp[e] = sbp[e] = sg[e] = 0.f;
  for (int64_t r = first; r < last; ++r) {
    const int64_t base = r * a.C, grp = r / a.T;
    const float* gate = a.gate ? a.gate + grp * a.C : nullptr;
    const float4 st = stats[r];
    // D starts as u; hh and xh are the normalised rows
    float D[E], xh[E], hh[E];
    float s[2] = {0.f, 0.f};
#pragma unroll
    for (int k = 0; k < E / W; ++k) {
      const int c = column<W>(k);
      if (c < a.C) {
        float g[W], w[W], wp[W], bp[W];
        load<W>(a.h, a.h_bf16, base + c, hh + k * W);
        load<W>(a.x, a.x_bf16, base + c, xh + k * W);
        load<W>(dy, a.y_bf16, base + c, D + k * W);
        load<W>(a.w, false, c, w);
        gate_of<W>(a, gate, c, g);
        if (a.wp) load<W>(a.wp, false, c, wp);
        if (a.bp) load<W>(a.bp, false, c, bp);
#pragma unroll
        for (int j = 0; j < W; ++j) {
          const int e = k * W + j;
          float n = hh[e];
          if (a.wp) {
            hh[e] = (n - st.x) * st.y;
            n = hh[e] * wp[j] + (a.bp ? bp[j] : 0.f);
          }
          xh[e] = (xh[e] + g[j] * n - st.z) * st.w;
          sw[e] += D[e] * xh[e];
          sb[e] += D[e];
          D[e] *= w[j];
          s[0] += D[e];
          s[1] += D[e] * xh[e];
        }
      } else {
#pragma unroll
        for (int j = 0; j < W; ++j) D[k * W + j] = xh[k * W + j] = hh[k * W + j] = 0.f;
      }
    }
    block_sums<2>(s, red[0]);
    const float mu = a.rms ? 0.f : s[0] / a.C, mux = s[1] / a.C;
    float q[2] = {0.f, 0.f};
#pragma unroll
    for (int k = 0; k < E / W; ++k) {
      const int c = column<W>(k);
      if (c >= a.C) continue;
      float up[W], g[W], wp[W], bp[W];
      if (dxo)
        load<W>(dxo, a.x_bf16, base + c, up);
      else
#pragma unroll
        for (int j = 0; j < W; ++j) up[j] = 0.f;
      gate_of<W>(a, gate, c, g);
      if (a.wp) load<W>(a.wp, false, c, wp);
      if (a.bp) load<W>(a.bp, false, c, bp);
#pragma unroll
      for (int j = 0; j < W; ++j) {
        const int e = k * W + j;
        up[j] += st.w * (D[e] - mu - xh[e] * mux);
        const float n = a.wp ? hh[e] * wp[j] + (a.bp ? bp[j] : 0.f) : hh[e];
        sg[e] += up[j] * n;
        const float dn = up[j] * g[j];
        swp[e] += dn * hh[e];
        sbp[e] += dn;
        D[e] = a.wp ? dn * wp[j] : dn;
        q[0] += D[e];
        q[1] += D[e] * hh[e];
      }
      store<W>(dx, a.x_bf16, base + c, up);
    }
    float mv = 0.f, mvh = 0.f;
    if (a.wp) {
      block_sums<2>(q, red[1]);
      mv = a.rms ? 0.f : q[0] / a.C;
      mvh = q[1] / a.C;
    } else {
      __syncthreads();  // red[0] is free for the next row
    }
#pragma unroll
    for (int k = 0; k < E / W; ++k) {
      const int c = column<W>(k);
      if (c >= a.C) continue;
      float o[W];
#pragma unroll
      for (int j = 0; j < W; ++j) {
        const int e = k * W + j;
        o[j] = a.wp ? st.y * (D[e] - mv - hh[e] * mvh) : D[e];
      }
      store<W>(dh, a.h_bf16, base + c, o);
    }
    if (gate_parts && (r + 1 == last || (r + 1) / a.T != grp)) {
      float* out = gate_parts + ((int64_t)blockIdx.x + grp) * a.C;
#pragma unroll
      for (int k = 0; k < E / W; ++k) {
        const int c = column<W>(k);
        if (c >= a.C) continue;
#pragma unroll
        for (int j = 0; j < W; ++j) {
          out[c + j] = a.scale * sg[k * W + j];
          sg[k * W + j] = 0.f;
        }
      }
    }
  }
  const int64_t plane = (int64_t)gridDim.x * a.C;
  float* out = parts + (int64_t)blockIdx.x * a.C;
#pragma unroll
  for (int k = 0; k < E / W; ++k) {
    const int c = column<W>(k);
    if (c >= a.C) continue;
    store<W>(out, false, c, sw + k * W);
    if (a.b) store<W>(out + plane, false, c, sb + k * W);
    if (a.wp) store<W>(out + 2 * plane, false, c, swp + k * W);
    if (a.bp) store<W>(out + 3 * plane, false, c, sbp + k * W);
  }
}

struct Sums {
  const float* parts;
  float* out[kParts];
  const float* gate_parts;
  float* dgate;
  int64_t N, T, rows;
  int C, ctas;
};

// Column sums of the partial rows: blockIdx.y < kParts one parameter's gradient, else
// the gate's gradient of group blockIdx.y - kParts.  A CTA of 8 x 32 threads takes 32
// columns, thread (g, j) adds rows g, g + 8, ... of column j, then the eight are added.
__global__ void __launch_bounds__(256) sums_kernel(Sums s) {
  __shared__ float red[8][33];
  const int j = threadIdx.x & 31, grp = threadIdx.x >> 5;
  const int c = blockIdx.x * 32 + j;
  const int64_t y = blockIdx.y;
  const float* in;
  float* out;
  int64_t count = s.ctas;
  if (y < kParts) {
    in = s.parts + y * s.ctas * s.C;
    out = s.out[y];
  } else {
    const int64_t g = y - kParts, first = g * s.T / s.rows;
    const int64_t end = min((g + 1) * s.T, s.N);
    count = (end - 1) / s.rows - first + 1;
    in = s.gate_parts + (first + g) * s.C;
    out = s.dgate ? s.dgate + g * s.C : nullptr;
  }
  if (!out) return;
  float t = 0.f;
  if (c < s.C)
    for (int64_t r = grp; r < count; r += 8) t += in[r * s.C + c];
  red[grp][j] = t;
  __syncthreads();
  if (grp == 0 && c < s.C) {
    float u = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) u += red[i][j];
    out[c] = u;
  }
}

bool aligned(const void* p, int bytes) {
  return (reinterpret_cast<uintptr_t>(p) & (bytes - 1)) == 0;
}

bool known(int dtype) { return dtype == SQB_BF16 || dtype == SQB_F32; }

constexpr int kMaxCtas = 148 * 4;

int ctas_of(int64_t N) { return (int)(N < kMaxCtas ? N : kMaxCtas); }
int64_t rows_of(int64_t N) { return (N + ctas_of(N) - 1) / ctas_of(N); }

// Elements a thread holds, and threads for C columns.
int elements_of(int64_t C) { return C <= 1024 ? 4 : 8; }
int threads_of(int64_t C) {
  const int64_t e = elements_of(C);
  return (int)(((C + e - 1) / e + 31) / 32 * 32);
}

int check(const Args& a, int x_dtype, int h_dtype, int y_dtype, int64_t gates) {
  if (!a.x || !a.h || !a.w || a.N <= 0 || a.N > INT32_MAX || (a.bp && !a.wp)) return SQB_ERR_ARG;
  if (a.gate && (gates <= 0 || a.N % gates != 0)) return SQB_ERR_ARG;
  if (!known(x_dtype) || !known(h_dtype) || !known(y_dtype)) return SQB_ERR_DTYPE;
  if (a.C <= 0 || a.C > kMaxC) return SQB_ERR_UNSUPPORTED;
  return SQB_OK;
}

// Whether every row can be read four elements at a time.
bool wide(const Args& a, const void* const* more, int n) {
  if (a.C % 4) return false;
  for (const void* p : {a.x, a.h, (const void*)a.w, (const void*)a.b, (const void*)a.wp,
                        (const void*)a.bp, (const void*)a.gate})
    if (!aligned(p, 16)) return false;
  for (int i = 0; i < n; ++i)
    if (!aligned(more[i], 16)) return false;
  return true;
}

Args make_args(const void* x, int x_dtype, const void* h, int h_dtype, int y_dtype,
               const float* w, const float* b, const float* wp, const float* bp,
               const float* gate, int64_t gates, float scale, float eps, int rms, int64_t N,
               int64_t C) {
  Args a;
  a.x = x, a.h = h, a.w = w, a.b = b, a.wp = wp, a.bp = bp, a.gate = gate;
  a.scale = scale, a.eps = eps, a.N = N, a.T = gate && gates > 0 ? N / gates : N;
  if (a.T <= 0) a.T = 1;
  a.C = C > kMaxC ? kMaxC + 1 : (int)C;
  a.rms = rms != 0, a.x_bf16 = x_dtype == SQB_BF16, a.h_bf16 = h_dtype == SQB_BF16;
  a.y_bf16 = y_dtype == SQB_BF16;
  return a;
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
  const Args a = make_args(x, x_dtype, h, h_dtype, y_dtype, weight, bias, post_weight, post_bias,
                           gate, gates, scale, eps, rms, N, C);
  if (const int rc = check(a, x_dtype, h_dtype, y_dtype, gates)) return rc;
  if (!x_out || !y || !stats) return SQB_ERR_ARG;
  if (!aligned(stats, 16)) return SQB_ERR_ALIGN;
  cudaStream_t q = static_cast<cudaStream_t>(stream);
  const void* more[] = {x_out, y};
  const bool w4 = wide(a, more, 2);
  const int nt = threads_of(C);
  const unsigned grid = (unsigned)N;
  float4* st = reinterpret_cast<float4*>(stats);
  if (elements_of(C) == 4) {
    if (w4)
      fwd_kernel<4, 4><<<grid, nt, 0, q>>>(a, x_out, y, st);
    else
      fwd_kernel<4, 1><<<grid, nt, 0, q>>>(a, x_out, y, st);
  } else {
    if (w4)
      fwd_kernel<8, 4><<<grid, nt, 0, q>>>(a, x_out, y, st);
    else
      fwd_kernel<8, 1><<<grid, nt, 0, q>>>(a, x_out, y, st);
  }
  return cudaGetLastError() == cudaSuccess ? SQB_OK : SQB_ERR_LAUNCH;
}

extern "C" size_t sqb_residual_norm_workspace_bytes(int64_t N, int64_t C, int64_t gates) {
  if (N <= 0 || C <= 0 || gates < 0) return 0;
  const int64_t rows = kParts * (int64_t)ctas_of(N) + (gates ? ctas_of(N) + gates : 0);
  return (size_t)rows * (size_t)C * sizeof(float);
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
  const Args a = make_args(x, x_dtype, h, h_dtype, y_dtype, weight, bias, post_weight, post_bias,
                           gate, gates, scale, eps, rms, N, C);
  if (const int rc = check(a, x_dtype, h_dtype, y_dtype, gates)) return rc;
  if (!dy || !stats || !dx || !dh || !dweight || (bias && !dbias) ||
      (post_weight && !dpost_weight) || (post_bias && !dpost_bias) || (gate && !dgate))
    return SQB_ERR_ARG;
  if (gate && gates > 65535 - kParts) return SQB_ERR_UNSUPPORTED;
  if (!workspace || ws_bytes < sqb_residual_norm_workspace_bytes(N, C, gate ? gates : 0))
    return SQB_ERR_WORKSPACE;
  if (!aligned(stats, 16) || !aligned(workspace, 16)) return SQB_ERR_ALIGN;
  cudaStream_t q = static_cast<cudaStream_t>(stream);
  const void* more[] = {dy, dx_out, dx, dh};
  const bool w4 = wide(a, more, 4);
  const int nt = threads_of(C), ctas = ctas_of(N);
  const int64_t rows = rows_of(N);
  float* parts = static_cast<float*>(workspace);
  float* gate_parts = gate ? parts + (int64_t)kParts * ctas * C : nullptr;
  const float4* st = reinterpret_cast<const float4*>(stats);
  // rows are dealt out evenly, so the last CTAs may have none: they write zero sums
  if (elements_of(C) == 4) {
    if (w4)
      bwd_kernel<4, 4><<<ctas, nt, 0, q>>>(a, dy, dx_out, st, dx, dh, parts, gate_parts, rows);
    else
      bwd_kernel<4, 1><<<ctas, nt, 0, q>>>(a, dy, dx_out, st, dx, dh, parts, gate_parts, rows);
  } else {
    if (w4)
      bwd_kernel<8, 4><<<ctas, nt, 0, q>>>(a, dy, dx_out, st, dx, dh, parts, gate_parts, rows);
    else
      bwd_kernel<8, 1><<<ctas, nt, 0, q>>>(a, dy, dx_out, st, dx, dh, parts, gate_parts, rows);
  }
  Sums s;
  s.parts = parts;
  s.out[0] = dweight, s.out[1] = bias ? dbias : nullptr;
  s.out[2] = post_weight ? dpost_weight : nullptr, s.out[3] = post_bias ? dpost_bias : nullptr;
  s.gate_parts = gate_parts, s.dgate = dgate;
  s.N = N, s.T = a.T, s.rows = rows, s.C = (int)C, s.ctas = ctas;
  const dim3 grid((unsigned)((C + 31) / 32), (unsigned)(kParts + (gate ? gates : 0)));
  sums_kernel<<<grid, 256, 0, q>>>(s);
  return cudaGetLastError() == cudaSuccess ? SQB_OK : SQB_ERR_LAUNCH;
}
