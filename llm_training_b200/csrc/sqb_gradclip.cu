// Global gradient norm over many tensors, and clipping (include/sqb_train.h).
//
//   norm = sqrt(sum of g^2 over every tensor),  out = g * min(1, max_norm / (norm + 1e-6))
//
// The squares are summed in 64 bits: a square of an fp32 gradient overflows or
// vanishes in 32 bits from 1e19 up and 1e-19 down, and the B200's 64-bit units keep
// up with HBM (two operations for each 4 bytes).  One CTA's sum is written to its own
// slot and the slots are added in a fixed order, so the norm is the same bits on
// every run and on every data-parallel rank that holds the same gradients.
//
// The tensors' pointers and sizes travel as a kernel argument (no table in device
// memory to fill, and a captured graph keeps its own copy).  The work is cut into pieces
// that never cross a tensor; CTAs take pieces in turn and find a piece's tensor by a
// binary search in the table.  Bound by HBM: one read for the norm, one read and one write
// for the scaling.  Four loads in flight a thread, pieces of 32768: 124M fp32 gradients
// (497 MB) norm 90 us, 5.5 TB/s, scaling 160 us, 6.2 TB/s; 362M bf16 ones (724 MB) into fp32
// 136 and 372 us.  Measured and not kept: sums in 32 bits (2 to 4 % of the norm's time),
// equal contiguous spans for the CTAs (norm 121 us), 32-byte loads (93 us), pieces taken
// from the end and streaming hints, for what the norm leaves in L2 (1 % of the total).

#include <cuda_bf16.h>
#include <math.h>
#include <stdint.h>

#include "sqb_train.h"

namespace sqb {
namespace gradclip {
namespace {

constexpr int kThreads = 512;
constexpr int kPerSm = 4;
constexpr int kGrid = 148 * kPerSm;  // CTAs on 148 SMs
// Tensors of a launch, and of one whose smaller table (2 of 23 KB) the host has copied sooner.
constexpr int kMaxTensors = 768, kFewTensors = 64;
constexpr int kPiece = 32768;  // elements

template <int kMax>
struct Table {
  const void* in[kMax];
  void* out[kMax];
  int64_t numel[kMax];
  int32_t end[kMax];  // pieces of tensors 0..i
  uint8_t in_bf16[kMax], out_bf16[kMax];
  int32_t n;
};
static_assert(sizeof(Table<kMaxTensors>) <= 32000, "a kernel's arguments are at most 32764 bytes");

// Calls f(tensor, first element, elements) for this CTA's pieces.
template <int kMax, typename F>
__device__ __forceinline__ void for_pieces(const Table<kMax>& t, F&& f) {
  const int all = t.end[t.n - 1];
  for (int c = blockIdx.x; c < all; c += gridDim.x) {
    int lo = 0, hi = t.n - 1;  // the first tensor that ends beyond c
    while (lo < hi) {
      const int mid = (lo + hi) / 2;
      if (t.end[mid] <= c)
        lo = mid + 1;
      else
        hi = mid;
    }
    const int64_t at = (int64_t)(c - (lo ? t.end[lo - 1] : 0)) * kPiece;
    f(lo, at, (int)min((int64_t)kPiece, t.numel[lo] - at));
  }
}

__device__ __forceinline__ float to_f(float x) { return x; }
__device__ __forceinline__ float to_f(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ void put(float* p, float v) { *p = v; }
__device__ __forceinline__ void put(__nv_bfloat16* p, float v) { *p = __float2bfloat16_rn(v); }

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

// Elements before the first `bytes` boundary of p, at most n.
template <typename T>
__device__ __forceinline__ int head_of(const T* p, int n, int bytes) {
  const int h = (int)((bytes - (reinterpret_cast<uintptr_t>(p) & (bytes - 1))) & (bytes - 1)) /
                (int)sizeof(T);
  return h < n ? h : n;
}

constexpr int kUnroll = 4;  // loads in flight a thread

template <typename T>
__device__ double square_sum(const T* p, int n) {
  constexpr int kN = 16 / sizeof(T);
  const int head = head_of(p, n, 16), nvec = (n - head) / kN;
  double v[2] = {0.0, 0.0};
  auto one = [&](float x, int j) { v[j & 1] = fma((double)x, (double)x, v[j & 1]); };
  auto vector = [&](const uint4& u) {
    const T* e = reinterpret_cast<const T*>(&u);
#pragma unroll
    for (int j = 0; j < kN; ++j) one(to_f(e[j]), j);
  };
  if ((int)threadIdx.x < head) one(to_f(p[threadIdx.x]), 0);
  const uint4* body = reinterpret_cast<const uint4*>(p + head);
  int i = threadIdx.x;
  for (; i + (kUnroll - 1) * kThreads < nvec; i += kUnroll * kThreads) {
    uint4 u[kUnroll];
#pragma unroll
    for (int k = 0; k < kUnroll; ++k) u[k] = body[i + k * kThreads];
#pragma unroll
    for (int k = 0; k < kUnroll; ++k) vector(u[k]);
  }
  for (; i < nvec; i += kThreads) vector(body[i]);
  const int tail = head + nvec * kN + threadIdx.x;
  if (tail < n) one(to_f(p[tail]), 0);
  return v[0] + v[1];
}

template <int kMax>
__global__ void __launch_bounds__(kThreads, kPerSm)
    norm_kernel(const __grid_constant__ Table<kMax> t, double* partial) {
  __shared__ double red[32];
  double v = 0.0;
  for_pieces(t, [&](int i, int64_t at, int n) {
    v += t.in_bf16[i] ? square_sum(static_cast<const __nv_bfloat16*>(t.in[i]) + at, n)
                      : square_sum(static_cast<const float*>(t.in[i]) + at, n);
  });
  v = block_sum(v, red);
  if (threadIdx.x == 0) partial[blockIdx.x] = v;
}

// The norm from the CTAs' sums, the same in every thread of every CTA.
__device__ float norm_of(const double* partial, int slots, double* red) {
  double v = 0.0;
  for (int i = threadIdx.x; i < slots; i += blockDim.x) v += partial[i];
  return (float)sqrt(block_sum(v, red));
}

__global__ void __launch_bounds__(kThreads, kPerSm)
    finish_kernel(const double* partial, int slots, float* norm) {
  __shared__ double red[32];
  const float n = norm_of(partial, slots, red);
  if (threadIdx.x == 0) *norm = n;
}

// N elements as they lie in memory.
template <typename T, int N>
struct alignas(sizeof(T) * N) Pack {
  T v[N];
};

// o = f p over n elements.  A thread moves 16 bytes of the wider of the two types at a time
// (4 elements between the types), so that a warp's loads and stores are both contiguous.
template <typename I, typename O>
__device__ void scale_piece(const I* p, O* o, int n, float f) {
  constexpr int kN = sizeof(I) == 2 && sizeof(O) == 2 ? 8 : 4;
  const int head = head_of(p, n, kN * sizeof(I));
  if ((reinterpret_cast<uintptr_t>(o + head) & (kN * sizeof(O) - 1)) != 0) {
    for (int i = threadIdx.x; i < n; i += kThreads) put(o + i, to_f(p[i]) * f);
    return;
  }
  const int nvec = (n - head) / kN;
  if ((int)threadIdx.x < head) put(o + threadIdx.x, to_f(p[threadIdx.x]) * f);
  const Pack<I, kN>* in = reinterpret_cast<const Pack<I, kN>*>(p + head);
  Pack<O, kN>* out = reinterpret_cast<Pack<O, kN>*>(o + head);
  auto scaled = [&](const Pack<I, kN>& u) {
    Pack<O, kN> d;
#pragma unroll
    for (int j = 0; j < kN; ++j) put(d.v + j, to_f(u.v[j]) * f);
    return d;
  };
  int i = threadIdx.x;
  for (; i + (kUnroll - 1) * kThreads < nvec; i += kUnroll * kThreads) {
    Pack<I, kN> u[kUnroll];
#pragma unroll
    for (int k = 0; k < kUnroll; ++k) u[k] = in[i + k * kThreads];
#pragma unroll
    for (int k = 0; k < kUnroll; ++k) out[i + k * kThreads] = scaled(u[k]);
  }
  for (; i < nvec; i += kThreads) out[i] = scaled(in[i]);
  const int tail = head + nvec * kN + threadIdx.x;
  if (tail < n) put(o + tail, to_f(p[tail]) * f);
}

template <int kMax>
__global__ void __launch_bounds__(kThreads, kPerSm)
    clip_kernel(const __grid_constant__ Table<kMax> t, const double* partial, int slots,
                float max_norm, bool in_place, float* norm) {
  __shared__ double red[32];
  const float n = norm_of(partial, slots, red);
  if (blockIdx.x == 0 && threadIdx.x == 0) *norm = n;
  float f = max_norm / (n + 1e-6f);
  if (f > 1.f) f = 1.f;  // a NaN stays
  if (in_place && f == 1.f) return;
  for_pieces(t, [&](int i, int64_t at, int n) {
    const float* pf = static_cast<const float*>(t.in[i]) + at;
    const __nv_bfloat16* pb = static_cast<const __nv_bfloat16*>(t.in[i]) + at;
    float* of = static_cast<float*>(t.out[i]) + at;
    __nv_bfloat16* ob = static_cast<__nv_bfloat16*>(t.out[i]) + at;
    if (t.in_bf16[i]) {
      if (t.out_bf16[i])
        scale_piece(pb, ob, n, f);
      else
        scale_piece(pb, of, n, f);
    } else {
      if (t.out_bf16[i])
        scale_piece(pf, ob, n, f);
      else
        scale_piece(pf, of, n, f);
    }
  });
}

// Fills `t` from the next tensors at `at`; returns how many were passed.  Empty
// tensors take no slot.
template <int kMax>
int64_t fill(Table<kMax>& t, const void* const* in, void* const* out, const int64_t* numel,
             const int32_t* in_dtype, const int32_t* out_dtype, int64_t n, int64_t at) {
  t.n = 0;
  int32_t pieces = 0;
  int64_t i = at;
  for (; i < n && t.n < kMax; ++i) {
    if (numel[i] == 0) continue;
    pieces += (int32_t)((numel[i] + kPiece - 1) / kPiece);
    t.in[t.n] = in[i];
    t.out[t.n] = out ? out[i] : nullptr;
    t.numel[t.n] = numel[i];
    t.end[t.n] = pieces;
    t.in_bf16[t.n] = in_dtype[i] == SQB_BF16;
    t.out_bf16[t.n] = out_dtype && out_dtype[i] == SQB_BF16;
    ++t.n;
  }
  return i - at;
}

bool known(int32_t dtype) { return dtype == SQB_BF16 || dtype == SQB_F32; }

int check(const void* const* in, void* const* out, const int64_t* numel,
          const int32_t* in_dtype, const int32_t* out_dtype, int64_t n) {
  int64_t pieces = 0;  // of all tensors: held in 32 bits
  for (int64_t i = 0; i < n; ++i) {
    if (numel[i] < 0 || numel[i] > (int64_t)INT32_MAX * kPiece) return SQB_ERR_ARG;
    pieces += (numel[i] + kPiece - 1) / kPiece;
    if (pieces > INT32_MAX) return SQB_ERR_ARG;
    if (!known(in_dtype[i]) || (out_dtype && !known(out_dtype[i]))) return SQB_ERR_DTYPE;
    if (numel[i] && (!in[i] || (out && !out[i]))) return SQB_ERR_ARG;
    const uintptr_t a = reinterpret_cast<uintptr_t>(in[i]);
    const uintptr_t b = out ? reinterpret_cast<uintptr_t>(out[i]) : 0;
    if (a % (in_dtype[i] == SQB_BF16 ? 2 : 4)) return SQB_ERR_ALIGN;
    if (out && b % (out_dtype[i] == SQB_BF16 ? 2 : 4)) return SQB_ERR_ALIGN;
  }
  return SQB_OK;
}

template <int kMax>
int grid_of(const Table<kMax>& t) {
  return t.end[t.n - 1] < kGrid ? t.end[t.n - 1] : kGrid;
}

// One launch for each table of tensors; returns the slots of `partial` they write.
template <int kMax>
int launch_norms(Table<kMax>& t, const void* const* in, const int64_t* numel, const int32_t* in_dtype,
                 int64_t n, double* partial, cudaStream_t q) {
  int slots = 0;
  for (int64_t at = 0; at < n;) {
    at += fill(t, in, nullptr, numel, in_dtype, nullptr, n, at);
    if (t.n == 0) continue;
    norm_kernel<<<grid_of(t), kThreads, 0, q>>>(t, partial + slots);
    slots += grid_of(t);
  }
  return slots;
}

// Calls f with a table for n tensors.
template <typename F>
void with_table(int64_t n, F&& f) {
  if (n <= kFewTensors) {
    Table<kFewTensors> t;
    f(t);
  } else {
    Table<kMaxTensors> t;
    f(t);
  }
}

// The scratch's doubles and the norm on their boundaries.
bool aligned(const void* workspace, const float* norm) {
  return reinterpret_cast<uintptr_t>(workspace) % sizeof(double) == 0 &&
         reinterpret_cast<uintptr_t>(norm) % sizeof(float) == 0;
}

int launched() { return cudaGetLastError() == cudaSuccess ? SQB_OK : SQB_ERR_LAUNCH; }

}  // namespace
}  // namespace gradclip
}  // namespace sqb

using namespace sqb::gradclip;

extern "C" size_t sqb_grad_norm_workspace_bytes(int64_t n_tensors) {
  if (n_tensors <= 0) return 0;
  return (size_t)((n_tensors + kMaxTensors - 1) / kMaxTensors) * kGrid * sizeof(double);
}

extern "C" int sqb_grad_norm(const void* const* grads, const int64_t* numel,
                             const int32_t* dtypes, int64_t n, void* workspace, size_t ws_bytes,
                             float* norm, void* stream) {
  if (!grads || !numel || !dtypes || n <= 0 || !norm) return SQB_ERR_ARG;
  if (const int rc = check(grads, nullptr, numel, dtypes, nullptr, n)) return rc;
  if (!workspace || ws_bytes < sqb_grad_norm_workspace_bytes(n)) return SQB_ERR_WORKSPACE;
  if (!aligned(workspace, norm)) return SQB_ERR_ALIGN;
  cudaStream_t q = static_cast<cudaStream_t>(stream);
  double* partial = static_cast<double*>(workspace);
  with_table(n, [&](auto& t) {
    const int slots = launch_norms(t, grads, numel, dtypes, n, partial, q);
    finish_kernel<<<1, kThreads, 0, q>>>(partial, slots, norm);
  });
  return launched();
}

extern "C" int sqb_grad_clip(const void* const* grads, void* const* outs, const int64_t* numel,
                             const int32_t* dtypes, const int32_t* out_dtypes, int64_t n,
                             float max_norm, void* workspace, size_t ws_bytes, float* norm,
                             void* stream) {
  if (!grads || !outs || !numel || !dtypes || !out_dtypes || n <= 0 || !norm ||
      !(max_norm >= 0.f))
    return SQB_ERR_ARG;
  if (const int rc = check(grads, outs, numel, dtypes, out_dtypes, n)) return rc;
  if (!workspace || ws_bytes < sqb_grad_norm_workspace_bytes(n)) return SQB_ERR_WORKSPACE;
  if (!aligned(workspace, norm)) return SQB_ERR_ALIGN;
  cudaStream_t q = static_cast<cudaStream_t>(stream);
  double* partial = static_cast<double*>(workspace);
  bool in_place = true;
  for (int64_t i = 0; i < n; ++i)
    in_place = in_place && (numel[i] == 0 || (grads[i] == outs[i] && dtypes[i] == out_dtypes[i]));
  with_table(n, [&](auto& t) {
    const int slots = launch_norms(t, grads, numel, dtypes, n, partial, q);
    if (slots == 0) finish_kernel<<<1, kThreads, 0, q>>>(partial, 0, norm);
    for (int64_t at = 0; at < n;) {
      at += fill(t, grads, outs, numel, dtypes, out_dtypes, n, at);
      if (t.n == 0) continue;
      clip_kernel<<<grid_of(t), kThreads, 0, q>>>(t, partial, slots, max_norm, in_place, norm);
    }
  });
  return launched();
}
