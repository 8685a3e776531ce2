// Layer norm over the last axis, forward and backward.
//
//   h = (x - mean) * rstd,  y = h * w + b,  rstd = 1 / sqrt(var + eps)
//   dx = rstd * (g - mean(g) - h * mean(g h)),  g = dy * w;   dw = sum_rows dy h,  db = sum_rows dy
//
// Both passes are bound by HBM bandwidth: x is read once and y written once forwards, x and dy read and dx written backwards.
// A row is held in the registers of a group of 32 .. 512 threads (kPer = 8, 16 or 32 elements each), so the mean and
// then the centred squares are summed from registers: two reductions, no cancellation between E[x^2] and
// E[x]^2. Groups walk over the rows with the weights in registers and the next row's loads in flight. The weight's and the bias's
// gradients stay in each thread's registers over all rows of its group; a CTA adds its groups' sums in shared memory,
// writes one partial row, and a second kernel adds those rows in a fixed order: no atomics, the same bits every run.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <atomic>

#include "../../include/hyfft.h"
#include "common.cuh"

namespace hyfft {

extern std::atomic<long long> g_launches;
int set_error(int code, const char* msg);  // engine.cu: the message hyfft_last_error returns

namespace {

constexpr int kMaxRow = 512 * 32;  // widest row held in registers
constexpr int kLoopThreads = 512;  // threads of the kernels for wider rows

struct NormArgs {
  const void *x, *w, *b, *dy;
  void *y, *dx;
  float *mean, *rstd;
  float *part;           // [ctas, 2, C]
  long long rows, xs, ds;  // row strides of x and dy; y and dx are contiguous
  int C, tpr, groups;
  int w32;  // weight and bias are float32
  float eps, invC;
};

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// Sums of (a, b) over the group's threads; `slot` alternates between calls, so one barrier is enough.
__device__ __forceinline__ float2 group_sum(float2 v, int tpr, int group, float2 (*red)[16], int& slot) {
  v.x = warp_sum(v.x);
  v.y = warp_sum(v.y);
  if (tpr == 32) return v;
  const int t = threadIdx.x - group * tpr;
  float2* r = red[group * 3 + slot];
  slot = slot == 2 ? 0 : slot + 1;
  if ((t & 31) == 0) r[t >> 5] = v;
  asm volatile("bar.sync %0, %1;" ::"r"(group + 1), "r"(tpr) : "memory");
  const int n = tpr >> 5;
  float2 s = r[0];
  for (int i = 1; i < n; ++i) s = cadd(s, r[i]);
  return s;
}

// Element e of a thread's kPer: column (t + tpr * (e / V)) * V + e % V.
template <typename T, int V, int PER>
__device__ __forceinline__ void load_row(T (&e)[PER], const T* __restrict__ p, int t, int tpr, int C) {
#pragma unroll
  for (int j = 0; j < PER / V; ++j) {
    const int c = (t + tpr * j) * V;
    if (c < C) {
      if constexpr (V > 1)
        *reinterpret_cast<uint4*>(e + j * V) = *reinterpret_cast<const uint4*>(p + c);
      else
        e[j] = p[c];
    }
  }
}
template <typename T, int V, int PER>
__device__ __forceinline__ void store_row(T* __restrict__ p, const T (&e)[PER], int t, int tpr, int C) {
#pragma unroll
  for (int j = 0; j < PER / V; ++j) {
    const int c = (t + tpr * j) * V;
    if (c < C) {
      if constexpr (V > 1)
        *reinterpret_cast<uint4*>(p + c) = *reinterpret_cast<const uint4*>(e + j * V);
      else
        p[c] = e[j];
    }
  }
}
template <typename T>
__device__ __forceinline__ float param(const void* p, int c, int w32) {
  return w32 ? static_cast<const float*>(p)[c] : DT<T>::load(static_cast<const T*>(p) + c);
}

template <typename T, int V, int PER>
__global__ void __launch_bounds__(512) layer_norm_fwd_kernel(const NormArgs A) {
  __shared__ float2 red[15 * 3][16];
  const int group = threadIdx.x / A.tpr, t = threadIdx.x - group * A.tpr;
  int slot = 0;
  float w[PER], b[PER];
#pragma unroll
  for (int e = 0; e < PER; ++e) {
    const int c = (t + A.tpr * (e / V)) * V + e % V;
    w[e] = A.w && c < A.C ? param<T>(A.w, c, A.w32) : 1.f;
    b[e] = A.b && c < A.C ? param<T>(A.b, c, A.w32) : 0.f;
  }
  const long long step = (long long)gridDim.x * A.groups;
  long long row = (long long)blockIdx.x * A.groups + group;
  const T* x = static_cast<const T*>(A.x);
  T* y = static_cast<T*>(A.y);
  alignas(16) T cur[PER];
  if (row < A.rows) load_row<T, V, PER>(cur, x + row * A.xs, t, A.tpr, A.C);
  for (; row < A.rows; row += step) {
    float f[PER];
    float s = 0.f;
#pragma unroll
    for (int e = 0; e < PER; ++e) {
      const int c = (t + A.tpr * (e / V)) * V + e % V;
      f[e] = c < A.C ? DT<T>::load(cur + e) : 0.f;
      s += f[e];
    }
    if (row + step < A.rows) load_row<T, V, PER>(cur, x + (row + step) * A.xs, t, A.tpr, A.C);
    const float mean = group_sum(make_float2(s, 0.f), A.tpr, group, red, slot).x * A.invC;
    s = 0.f;
#pragma unroll
    for (int e = 0; e < PER; ++e) {
      const int c = (t + A.tpr * (e / V)) * V + e % V;
      f[e] -= mean;
      if (c < A.C) s = fmaf(f[e], f[e], s);
    }
    const float var = group_sum(make_float2(s, 0.f), A.tpr, group, red, slot).x * A.invC;
    const float rstd = 1.f / sqrtf(var + A.eps);
    alignas(16) T o[PER];
#pragma unroll
    for (int e = 0; e < PER; ++e) DT<T>::store(o + e, fmaf(f[e] * rstd, w[e], b[e]));
    store_row<T, V, PER>(y + row * A.C, o, t, A.tpr, A.C);
    if (t == 0 && A.mean) A.mean[row] = mean, A.rstd[row] = rstd;
  }
}

template <typename T, int V, int PER>
__global__ void __launch_bounds__(512) layer_norm_bwd_kernel(const NormArgs A) {
  __shared__ float2 red[15 * 3][16];
  extern __shared__ float sums[];  // [groups, 2, C] where there is more than one group
  const int group = threadIdx.x / A.tpr, t = threadIdx.x - group * A.tpr;
  int slot = 0;
  float w[PER], dw[PER], db[PER];
#pragma unroll
  for (int e = 0; e < PER; ++e) {
    const int c = (t + A.tpr * (e / V)) * V + e % V;
    w[e] = A.w && c < A.C ? param<T>(A.w, c, A.w32) : 1.f;
    dw[e] = db[e] = 0.f;
  }
  const long long step = (long long)gridDim.x * A.groups;
  long long row = (long long)blockIdx.x * A.groups + group;
  const T* x = static_cast<const T*>(A.x);
  const T* dy = static_cast<const T*>(A.dy);
  alignas(16) T cx[PER];
  alignas(16) T cd[PER];
  float mean = 0.f, rstd = 0.f;
  if (row < A.rows) {
    load_row<T, V, PER>(cx, x + row * A.xs, t, A.tpr, A.C);
    load_row<T, V, PER>(cd, dy + row * A.ds, t, A.tpr, A.C);
    mean = A.mean[row], rstd = A.rstd[row];
  }
  for (; row < A.rows; row += step) {
    float h[PER], g[PER];
    float2 s = make_float2(0.f, 0.f);
#pragma unroll
    for (int e = 0; e < PER; ++e) {
      const int c = (t + A.tpr * (e / V)) * V + e % V;
      const float d = c < A.C ? DT<T>::load(cd + e) : 0.f;
      h[e] = c < A.C ? (DT<T>::load(cx + e) - mean) * rstd : 0.f;
      g[e] = d * w[e];
      dw[e] = fmaf(d, h[e], dw[e]);
      db[e] += d;
      s.x += g[e];
      s.y = fmaf(g[e], h[e], s.y);
    }
    const float r = rstd;
    if (row + step < A.rows) {
      load_row<T, V, PER>(cx, x + (row + step) * A.xs, t, A.tpr, A.C);
      load_row<T, V, PER>(cd, dy + (row + step) * A.ds, t, A.tpr, A.C);
      mean = A.mean[row + step], rstd = A.rstd[row + step];
    }
    s = group_sum(s, A.tpr, group, red, slot);
    s.x *= A.invC, s.y *= A.invC;
    if (A.dx) {
      alignas(16) T o[PER];
#pragma unroll
      for (int e = 0; e < PER; ++e) DT<T>::store(o + e, r * (g[e] - s.x - h[e] * s.y));
      store_row<T, V, PER>(static_cast<T*>(A.dx) + row * A.C, o, t, A.tpr, A.C);
    }
  }
  if (!A.part) return;
  float* out = A.part + (long long)blockIdx.x * 2 * A.C;
  float* to = A.groups == 1 ? out : sums + (long long)group * 2 * A.C;
#pragma unroll
  for (int e = 0; e < PER; ++e) {
    const int c = (t + A.tpr * (e / V)) * V + e % V;
    if (c < A.C) to[c] = dw[e], to[A.C + c] = db[e];
  }
  if (A.groups == 1) return;
  __syncthreads();
  for (int c = threadIdx.x; c < 2 * A.C; c += blockDim.x) {
    float s = 0.f;
    for (int i = 0; i < A.groups; ++i) s += sums[i * 2 * A.C + c];
    out[c] = s;
  }
}

// Rows wider than the registers of 512 threads: one CTA per row, the row read again for each sum.
template <typename T>
__global__ void __launch_bounds__(kLoopThreads) layer_norm_fwd_loop_kernel(const NormArgs A) {
  __shared__ float2 red[3][16];
  int slot = 0;
  for (long long row = blockIdx.x; row < A.rows; row += gridDim.x) {
    const T* x = static_cast<const T*>(A.x) + row * A.xs;
    T* y = static_cast<T*>(A.y) + row * A.C;
    float s = 0.f;
    for (int c = threadIdx.x; c < A.C; c += kLoopThreads) s += DT<T>::load(x + c);
    const float mean = group_sum(make_float2(s, 0.f), kLoopThreads, 0, red, slot).x * A.invC;
    s = 0.f;
    for (int c = threadIdx.x; c < A.C; c += kLoopThreads) {
      const float d = DT<T>::load(x + c) - mean;
      s = fmaf(d, d, s);
    }
    const float var = group_sum(make_float2(s, 0.f), kLoopThreads, 0, red, slot).x * A.invC;
    const float rstd = 1.f / sqrtf(var + A.eps);
    for (int c = threadIdx.x; c < A.C; c += kLoopThreads) {
      const float w = A.w ? param<T>(A.w, c, A.w32) : 1.f, b = A.b ? param<T>(A.b, c, A.w32) : 0.f;
      DT<T>::store(y + c, fmaf((DT<T>::load(x + c) - mean) * rstd, w, b));
    }
    if (threadIdx.x == 0 && A.mean) A.mean[row] = mean, A.rstd[row] = rstd;
  }
}

// The same backwards; a CTA's sums of dw and db live in its own row of `part`, each column touched by one thread.
template <typename T>
__global__ void __launch_bounds__(kLoopThreads) layer_norm_bwd_loop_kernel(const NormArgs A) {
  __shared__ float2 red[3][16];
  int slot = 0;
  float* out = A.part ? A.part + (long long)blockIdx.x * 2 * A.C : nullptr;
  if (out)
    for (int c = threadIdx.x; c < A.C; c += kLoopThreads) out[c] = out[A.C + c] = 0.f;
  for (long long row = blockIdx.x; row < A.rows; row += gridDim.x) {
    const T* x = static_cast<const T*>(A.x) + row * A.xs;
    const T* dy = static_cast<const T*>(A.dy) + row * A.ds;
    const float mean = A.mean[row], rstd = A.rstd[row];
    float2 s = make_float2(0.f, 0.f);
    for (int c = threadIdx.x; c < A.C; c += kLoopThreads) {
      const float d = DT<T>::load(dy + c), h = (DT<T>::load(x + c) - mean) * rstd;
      const float g = A.w ? d * param<T>(A.w, c, A.w32) : d;
      s.x += g;
      s.y = fmaf(g, h, s.y);
      if (out) {
        out[c] = fmaf(d, h, out[c]);
        out[A.C + c] += d;
      }
    }
    s = group_sum(s, kLoopThreads, 0, red, slot);
    s.x *= A.invC, s.y *= A.invC;
    if (A.dx) {
      T* dx = static_cast<T*>(A.dx) + row * A.C;
      for (int c = threadIdx.x; c < A.C; c += kLoopThreads) {
        const float d = DT<T>::load(dy + c), h = (DT<T>::load(x + c) - mean) * rstd;
        const float g = A.w ? d * param<T>(A.w, c, A.w32) : d;
        DT<T>::store(dx + c, rstd * (g - s.x - h * s.y));
      }
    }
  }
}

// part [n, 2 C] -> dw, db: 32 columns by 8 strands per CTA, each strand every eighth row, then the strands in order.
template <typename P>
__global__ void __launch_bounds__(256) layer_norm_reduce_kernel(const float* __restrict__ part, int n, int C, P* dw, P* db) {
  __shared__ float red[8][33];
  const int lane = threadIdx.x & 31, strand = threadIdx.x >> 5;
  const int c = blockIdx.x * 32 + lane;
  float s = 0.f;
  if (c < 2 * C)
    for (int i = strand; i < n; i += 8) s += part[(long long)i * 2 * C + c];
  red[strand][lane] = s;
  __syncthreads();
  if (strand == 0 && c < 2 * C) {
#pragma unroll
    for (int i = 1; i < 8; ++i) s += red[i][lane];
    if (c < C) {
      if (dw) DT<P>::store(dw + c, s);
    } else if (db) {
      DT<P>::store(db + c - C, s);
    }
  }
}

int launched() {
  if (cudaGetLastError() != cudaSuccess) return set_error(HYFFT_ERR_CUDA, "layer norm: kernel launch failed");
  g_launches.fetch_add(1, std::memory_order_relaxed);
  return HYFFT_OK;
}

struct NormPlan {
  int per, tpr, groups, ctas;  // per 0: the loop kernels
};

NormPlan plan(long long rows, int C, bool backward) {
  NormPlan p{};
  if (C > kMaxRow) {
    p.tpr = kLoopThreads, p.groups = 1;
    p.ctas = (int)std::min<long long>(rows, 2 * 148);
    return p;
  }
  p.per = C <= 512 * 8 ? 8 : C <= 512 * 16 ? 16 : 32;
  p.tpr = std::max(32, ((C + p.per - 1) / p.per + 31) / 32 * 32);
  p.groups = std::max(1, std::min(8, 256 / p.tpr));
  // rows that stay in flight on an SM: 2048 threads forwards, 1024 backwards, where a thread holds twice as much
  const int threads = p.tpr * p.groups;
  const int per_sm = std::max(1, (backward ? 1024 : 2048) / threads / (p.per / 8));
  p.ctas = (int)std::max<long long>(1, std::min<long long>((rows + p.groups - 1) / p.groups, 148ll * per_sm));
  return p;
}

template <typename T, int V, int PER>
int launch_rows(const NormArgs& A, const NormPlan& p, bool backward, cudaStream_t st) {
  const int threads = p.tpr * p.groups;
  if (!backward) {
    layer_norm_fwd_kernel<T, V, PER><<<p.ctas, threads, 0, st>>>(A);
  } else {
    const size_t sm = p.groups > 1 && A.part ? sizeof(float) * 2 * (size_t)p.groups * A.C : 0;
    auto kern = layer_norm_bwd_kernel<T, V, PER>;
    if (sm > 32 * 1024 && !kernel_smem_once((const void*)kern, sm)) return set_error(HYFFT_ERR_CUDA, "layer norm: shared memory");
    kern<<<p.ctas, threads, sm, st>>>(A);
  }
  return launched();
}

template <typename T, int V>
int launch_v(const NormArgs& A, const NormPlan& p, bool backward, cudaStream_t st) {
  if (p.per == 8) return launch_rows<T, V, 8>(A, p, backward, st);
  if (p.per == 16) return launch_rows<T, V, 16>(A, p, backward, st);
  return launch_rows<T, V, 32>(A, p, backward, st);
}

bool aligned(const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }

template <typename T>
int launch_t(NormArgs& A, bool backward, cudaStream_t st) {
  const NormPlan p = plan(A.rows, A.C, backward);
  A.tpr = p.tpr, A.groups = p.groups;
  A.invC = 1.f / (float)A.C;
  if (p.per == 0) {
    if (backward)
      layer_norm_bwd_loop_kernel<T><<<p.ctas, kLoopThreads, 0, st>>>(A);
    else
      layer_norm_fwd_loop_kernel<T><<<p.ctas, kLoopThreads, 0, st>>>(A);
    return launched();
  }
  constexpr int V = 16 / (int)sizeof(T);
  bool vec = A.C % V == 0 && A.xs % V == 0 && aligned(A.x) && aligned(A.y) && aligned(A.dx);
  if (backward) vec = vec && A.ds % V == 0 && aligned(A.dy);
  return vec ? launch_v<T, V>(A, p, backward, st) : launch_v<T, 1>(A, p, backward, st);
}

int check_args(int64_t rows, int64_t C, int32_t dtype, int32_t param_dtype) {
  if (rows < 1 || C < 1 || C > 0x3fffffff) return set_error(HYFFT_ERR_INVALID, "layer norm: rows and columns must be positive");
  if (dtype < HYFFT_F32 || dtype > HYFFT_F16) return set_error(HYFFT_ERR_INVALID, "layer norm: bad dtype");
  if (param_dtype != HYFFT_F32 && param_dtype != dtype)
    return set_error(HYFFT_ERR_INVALID, "layer norm: weight and bias have x's dtype or float32");
  return HYFFT_OK;
}

int run(NormArgs& A, int32_t dtype, bool backward, cudaStream_t st) {
  if (dtype == HYFFT_F32) return launch_t<float>(A, backward, st);
  if (dtype == HYFFT_BF16) return launch_t<__nv_bfloat16>(A, backward, st);
  return launch_t<__half>(A, backward, st);
}

}  // namespace
}  // namespace hyfft

using namespace hyfft;

extern "C" {

int hyfft_layer_norm_workspace_size(int64_t rows, int64_t C, size_t* bwd_bytes) {
  const int rc = check_args(rows, C, HYFFT_F32, HYFFT_F32);
  if (rc != HYFFT_OK) return rc;
  if (bwd_bytes) *bwd_bytes = sizeof(float) * 2 * (size_t)C * plan(rows, (int)C, true).ctas;
  return HYFFT_OK;
}

int hyfft_layer_norm_forward(const void* x, const void* weight, const void* bias, void* y, float* mean, float* rstd,
                             int64_t rows, int64_t C, int64_t x_stride, float eps, int32_t dtype, int32_t param_dtype,
                             void* stream) {
  const int rc = check_args(rows, C, dtype, param_dtype);
  if (rc != HYFFT_OK) return rc;
  if (!x || !y || (mean == nullptr) != (rstd == nullptr)) return set_error(HYFFT_ERR_INVALID, "layer norm: null tensor");
  if (bind_device_of(x) != HYFFT_OK) return set_error(HYFFT_ERR_CUDA, "layer norm: device");
  NormArgs A{};
  A.x = x, A.w = weight, A.b = bias, A.y = y, A.mean = mean, A.rstd = rstd;
  A.rows = rows, A.C = (int)C, A.xs = x_stride, A.eps = eps, A.w32 = param_dtype == HYFFT_F32;
  return run(A, dtype, false, static_cast<cudaStream_t>(stream));
}

int hyfft_layer_norm_backward(const void* x, const void* weight, const float* mean, const float* rstd, const void* dy,
                              void* dx, void* dweight, void* dbias, int64_t rows, int64_t C, int64_t x_stride,
                              int64_t dy_stride, int32_t dtype, int32_t param_dtype, void* workspace,
                              size_t workspace_bytes, void* stream) {
  const int rc = check_args(rows, C, dtype, param_dtype);
  if (rc != HYFFT_OK) return rc;
  if (!x || !dy || !mean || !rstd) return set_error(HYFFT_ERR_INVALID, "layer norm: null tensor in the backward");
  if (bind_device_of(x) != HYFFT_OK) return set_error(HYFFT_ERR_CUDA, "layer norm: device");
  const bool sums = dweight || dbias;
  const NormPlan p = plan(rows, (int)C, true);
  if (sums && (!workspace || workspace_bytes < sizeof(float) * 2 * (size_t)C * p.ctas))
    return set_error(HYFFT_ERR_WORKSPACE, "layer norm: workspace too small");
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  NormArgs A{};
  A.x = x, A.w = weight, A.dy = dy, A.dx = dx;
  A.mean = const_cast<float*>(mean), A.rstd = const_cast<float*>(rstd);
  A.rows = rows, A.C = (int)C, A.xs = x_stride, A.ds = dy_stride, A.w32 = param_dtype == HYFFT_F32;
  A.part = sums ? static_cast<float*>(workspace) : nullptr;
  int r = run(A, dtype, true, st);
  if (r != HYFFT_OK || !sums) return r;
  const unsigned grid = (unsigned)((2 * C + 31) / 32);
  if (param_dtype == HYFFT_F32)
    layer_norm_reduce_kernel<float><<<grid, 256, 0, st>>>(A.part, p.ctas, (int)C, (float*)dweight, (float*)dbias);
  else if (dtype == HYFFT_BF16)
    layer_norm_reduce_kernel<__nv_bfloat16><<<grid, 256, 0, st>>>(A.part, p.ctas, (int)C, (__nv_bfloat16*)dweight,
                                                                 (__nv_bfloat16*)dbias);
  else
    layer_norm_reduce_kernel<__half><<<grid, 256, 0, st>>>(A.part, p.ctas, (int)C, (__half*)dweight, (__half*)dbias);
  return launched();
}

}  // extern "C"
