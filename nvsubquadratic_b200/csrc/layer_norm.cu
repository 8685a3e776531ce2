// Layer norm over the last axis, forward and backward.
//
//   h = (x - mean) * rstd,  y = h * w + b,  rstd = 1 / sqrt(var + eps)
//   dx = rstd * (g - mean(g) - h * mean(g h)),  g = dy * w;   dw = sum_rows dy h,  db = sum_rows dy
//
// Both passes are bound by HBM bandwidth: x is read once and y written once forwards, x and dy read and dx written backwards.
// A row is held in the registers of a group of 32 .. 512 threads (kPer = 8, 16 or 32 elements each), so the mean and
// then the centred squares are summed from registers: two reductions, no cancellation between E[x^2] and
// E[x]^2. Groups walk over the rows with the weights in registers. Rows that start on 16 bytes come through a ring of up
// to four in shared memory for each group, filled by bulk copies (65536 rows of 4096 bfloat16: 210 us forwards, 282
// backwards; with the next row's loads in registers instead 246 and 330). Other rows are loaded one ahead into registers.
// Forwards 16-bit weights stay packed, which leaves room for four CTAs an SM instead of three (210 against 228 us); joining
// the warps' own means and squares with one barrier instead of two cost more instructions than it saved (251).
// Everything per element runs on packed pairs (element by element, with a test of the column for each, it was 314 and
// 422 us: instructions were the bound). The weight's and the bias's gradients stay in each thread's registers over
// all rows of its group; a CTA adds its groups' sums in shared memory, writes one partial row, and a second kernel adds those rows in a fixed order: no atomics, the same bits every run.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <atomic>
#include <map>
#include <mutex>
#include <tuple>

#include "../../include/hyfft.h"
#include "common.cuh"
#include "umma.cuh"
#include "waits.cuh"

namespace hyfft {

extern std::atomic<long long> g_launches;
int set_error(int code, const char* msg);  // engine.cu: the message hyfft_last_error returns

namespace {

constexpr int kMaxRow = 512 * 32;  // widest row held in registers
constexpr int kMaxGroups = 8, kMaxWarps = 16, kStages = 4;
constexpr int kLoopThreads = 512;  // threads of the kernels for wider rows

struct NormArgs {
  const void *x, *w, *b, *dy;
  void *y, *dx;
  float *mean, *rstd;
  float *part;           // [ctas, 2, C]
  long long rows, xs, ds;  // row strides of x and dy; y and dx are contiguous
  int C, tpr, groups;
  int stages;  // rows in a group's ring
  unsigned patience;  // clocks after which a wait gives up
  float eps, invC;
};

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// A group's warps leave their sums in shared memory and every thread adds all of them (read as 16-byte broadcasts).
// `slot` alternates between calls, so that one barrier is enough.
struct Sums {
  float4 v[2][kMaxGroups][kMaxWarps / 4];
};
__device__ __forceinline__ float read_sums(const float4* r, int warps) {
  float s = 0.f;
  for (int i = 0; i < warps; i += 4) {  // the entries past the last warp are zero
    const float4 q = r[i >> 2];
    s += (q.x + q.y) + (q.z + q.w);
  }
  return s;
}
__device__ __forceinline__ float group_sum(float v, int tpr, int group, Sums& sm, int& slot) {
  v = warp_sum(v);
  if (tpr == 32) return v;
  const int t = threadIdx.x - group * tpr;
  float4* r = sm.v[slot][group];
  slot ^= 1;
  if ((t & 31) == 0) reinterpret_cast<float*>(r)[t >> 5] = v;
  asm volatile("bar.sync %0, %1;" ::"r"(group + 1), "r"(tpr) : "memory");
  return read_sums(r, tpr >> 5);
}
__device__ __forceinline__ float2 group_sum(float2 v, int tpr, int group, Sums& sx, Sums& sy, int& slot) {
  v.x = warp_sum(v.x);
  v.y = warp_sum(v.y);
  if (tpr == 32) return v;
  const int t = threadIdx.x - group * tpr;
  float4 *x = sx.v[slot][group], *y = sy.v[slot][group];
  slot ^= 1;
  if ((t & 31) == 0) reinterpret_cast<float*>(x)[t >> 5] = v.x, reinterpret_cast<float*>(y)[t >> 5] = v.y;
  asm volatile("bar.sync %0, %1;" ::"r"(group + 1), "r"(tpr) : "memory");
  return make_float2(read_sums(x, tpr >> 5), read_sums(y, tpr >> 5));
}
// All entries zero, before the first sum.
__device__ __forceinline__ void clear(Sums& s) {
  float* f = reinterpret_cast<float*>(&s);
  for (int i = threadIdx.x; i < (int)(sizeof(Sums) / sizeof(float)); i += blockDim.x) f[i] = 0.f;
}

// One row (or two, of x and dy) into a place of the ring; one thread.
__device__ __forceinline__ void bulk_row(unsigned char* dst, const void* src, int bytes, uint64_t* bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(umma::su32(dst)),
               "l"(src), "r"(bytes), "r"(umma::su32(bar))
               : "memory");
}
__device__ __forceinline__ void expect(uint64_t* bar, int bytes) {
  asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(umma::su32(bar)), "r"(bytes) : "memory");
}
__device__ __forceinline__ void init_ring(uint64_t (*full)[kStages]) {
  if (threadIdx.x == 0) {
    for (int i = 0; i < kMaxGroups * kStages; ++i) umma::mbar_init(&full[0][i], 1);
    umma::fence_mbar_init();
  }
}

// What a group's fetching thread has in flight once a wait of its own has run out: the rows from `row` on, that one at place
// `at` in phase `phase` of the ring. It fetches no more, and waits for these before it leaves.
struct Lost {
  long long row;
  int at, phase;
};
__device__ __forceinline__ void drain(uint64_t* full, Lost l, int stages, long long step, long long rows) {
  for (int i = 0; i < stages && l.row + i * step < rows; ++i) {
    wait_phase(&full[l.at], l.phase, kWaitClocks);
    if (++l.at == stages) l.at = 0, l.phase ^= 1;
  }
}

// A thread's PER elements as PER / 2 pairs, so that the arithmetic runs as packed float32 pairs: element e is column
// (t + tpr * (e / V)) * V + e % V. Places past C hold zeros (WHOLE: there are none, C = tpr * PER).
template <typename T>
__device__ __forceinline__ float2 two(const T* p) {
  return make_float2(DT<T>::load(p), DT<T>::load(p + 1));
}
template <>
__device__ __forceinline__ float2 two<__nv_bfloat16>(const __nv_bfloat16* p) {
  const uint32_t u = *reinterpret_cast<const uint32_t*>(p);
  return make_float2(__uint_as_float(u << 16), __uint_as_float(u & 0xffff0000u));
}
template <>
__device__ __forceinline__ float2 two<__half>(const __half* p) {
  return __half22float2(*reinterpret_cast<const __half2*>(p));
}
template <typename T>
__device__ __forceinline__ void put_two(T* p, float2 v) {
  DT<T>::store(p, v.x);
  DT<T>::store(p + 1, v.y);
}
template <>
__device__ __forceinline__ void put_two<__nv_bfloat16>(__nv_bfloat16* p, float2 v) {
  *reinterpret_cast<__nv_bfloat162*>(p) = __floats2bfloat162_rn(v.x, v.y);
}
template <>
__device__ __forceinline__ void put_two<__half>(__half* p, float2 v) {
  *reinterpret_cast<__half2*>(p) = __floats2half2_rn(v.x, v.y);
}
__device__ __forceinline__ float2 mul2(float2 a, float2 b) { return make_float2(a.x * b.x, a.y * b.y); }
__device__ __forceinline__ float2 dup(float a) { return make_float2(a, a); }

template <int V>
__device__ __forceinline__ int column(int e, int t, int tpr) {
  return (t + tpr * (e / V)) * V + e % V;
}
template <typename T, int V, int PER, bool WHOLE>
__device__ __forceinline__ void load_row(T (&e)[PER], const T* __restrict__ p, int t, int tpr, int C) {
#pragma unroll
  for (int j = 0; j < PER / V; ++j) {
    const int c = (t + tpr * j) * V;
    const bool in = WHOLE || c < C;
    if constexpr (V > 1)
      *reinterpret_cast<uint4*>(e + j * V) = in ? *reinterpret_cast<const uint4*>(p + c) : make_uint4(0, 0, 0, 0);
    else
      DT<T>::store(e + j, in ? DT<T>::load(p + c) : 0.f);
  }
}
template <typename T, int PER>
__device__ __forceinline__ void no_row(T (&e)[PER]) {
#pragma unroll
  for (int j = 0; j < PER; ++j) DT<T>::store(e + j, __int_as_float(0x7fffffff));
}
template <typename T, int V, int PER, bool WHOLE>
__device__ __forceinline__ void store_row(T* __restrict__ p, const T (&e)[PER], int t, int tpr, int C) {
#pragma unroll
  for (int j = 0; j < PER / V; ++j) {
    const int c = (t + tpr * j) * V;
    if (WHOLE || c < C) {
      if constexpr (V > 1)
        *reinterpret_cast<uint4*>(p + c) = *reinterpret_cast<const uint4*>(e + j * V);
      else
        p[c] = e[j];
    }
  }
}
// Pairs that lie past C are zeroed (with V = 1 the two halves of a pair are tpr columns apart).
template <int V, bool WHOLE>
__device__ __forceinline__ float2 inside(float2 v, int e, int t, int tpr, int C) {
  if (WHOLE) return v;
  const bool a = column<V>(e, t, tpr) < C, b = V > 1 ? a : column<V>(e + 1, t, tpr) < C;
  return make_float2(a ? v.x : 0.f, b ? v.y : 0.f);
}
template <typename P, int V, int PER>
__device__ __forceinline__ void load_param(float2 (&f)[PER / 2], const void* p, float none, int t, int tpr, int C) {
#pragma unroll
  for (int e = 0; e < PER; ++e) {
    const int c = column<V>(e, t, tpr);
    (&f[e / 2].x)[e & 1] = p && c < C ? DT<P>::load(static_cast<const P*>(p) + c) : none;
  }
}

// Keeps 16-bit parameters packed: what is converted inside the loop must not be moved out of it.
template <typename P, int PER>
__device__ __forceinline__ void opaque(P (&f)[PER]) {
  if constexpr (sizeof(P) == 2) {
    uint32_t* u = reinterpret_cast<uint32_t*>(f);
#pragma unroll
    for (int i = 0; i < PER / 2; ++i) asm volatile("" : "+r"(u[i]));
  }
}

// The same in the parameters' own type: half the registers for 16-bit ones.
template <typename P, int V, int PER>
__device__ __forceinline__ void keep_param(P (&f)[PER], const void* p, float none, int t, int tpr, int C) {
#pragma unroll
  for (int e = 0; e < PER; ++e) {
    const int c = column<V>(e, t, tpr);
    DT<P>::store(f + e, p && c < C ? DT<P>::load(static_cast<const P*>(p) + c) : none);
  }
}

// 16-bit rows of up to 16 elements a thread: 64 registers, for four CTAs of 256 threads an SM.
template <typename T, typename P, int V, int PER, bool WHOLE>
__global__ void __launch_bounds__(512, V == 8 && sizeof(P) == 2 && PER <= 16 ? 2 : 1) layer_norm_fwd_kernel(const NormArgs A) {
  extern __shared__ __align__(16) unsigned char ring[];  // [groups, stages, C]
  __shared__ uint64_t full[kMaxGroups][kStages];
  __shared__ Lost lost[kMaxGroups];
  __shared__ Sums sums;
  clear(sums);
  init_ring(full);
  __syncthreads();
  const int group = threadIdx.x / A.tpr, t = threadIdx.x - group * A.tpr;
  int slot = 0;
  alignas(16) P w[PER], b[PER];
  keep_param<P, V, PER>(w, A.w, 1.f, t, A.tpr, A.C);
  keep_param<P, V, PER>(b, A.b, 0.f, t, A.tpr, A.C);
  const long long step = (long long)gridDim.x * A.groups;
  long long row = (long long)blockIdx.x * A.groups + group;
  const T* x = static_cast<const T*>(A.x);
  T* y = static_cast<T*>(A.y);
  constexpr bool kRing = V > 1;
  const int bytes = A.C * (int)sizeof(T);
  unsigned char* mine = ring + (size_t)group * A.stages * bytes;
  const auto fetch = [&](int i, long long r) {
    expect(&full[group][i], bytes);
    bulk_row(mine + (size_t)i * bytes, x + r * A.xs, bytes, &full[group][i]);
  };
  alignas(16) T cur[PER];
  if (kRing) {
    if (t == 0)
      for (int i = 0; i < A.stages; ++i)
        if (row + i * step < A.rows) fetch(i, row + i * step);
  } else if (row < A.rows) {
    load_row<T, V, PER, WHOLE>(cur, x + row * A.xs, t, A.tpr, A.C);
  }
  int at = 0, phase = 0;
  // phase: from 2 on once a wait has run out; this thread's part of a row is NaN then, and so are its group's results
  for (; row < A.rows; row += step) {
    if (kRing) {
      if (phase < 2 && !wait_phase(&full[group][at], phase, A.patience)) {
        if (t == 0) lost[group] = {row, at, phase};
        phase |= 2;
        atomicExch(&g_ran_out, 1u);
      }
      if (phase < 2)
        load_row<T, V, PER, WHOLE>(cur, reinterpret_cast<const T*>(mine + (size_t)at * bytes), t, A.tpr, A.C);
      else
        no_row(cur);
    }
    float2 f[PER / 2], s2 = dup(0.f);
#pragma unroll
    for (int p = 0; p < PER / 2; ++p) {
      f[p] = two<T>(cur + 2 * p);
      s2 = cadd(s2, f[p]);
    }
    if (!kRing && row + step < A.rows) load_row<T, V, PER, WHOLE>(cur, x + (row + step) * A.xs, t, A.tpr, A.C);
    const float mean = group_sum(s2.x + s2.y, A.tpr, group, sums, slot) * A.invC;
    if (kRing) {  // every thread of the group has read its part of the row
      if (t == 0 && phase < 2 && row + A.stages * step < A.rows) fetch(at, row + A.stages * step);
      if (++at == A.stages) at = 0, phase ^= 1;
    }
    s2 = dup(0.f);
#pragma unroll
    for (int p = 0; p < PER / 2; ++p) {
      f[p] = inside<V, WHOLE>(csub(f[p], dup(mean)), 2 * p, t, A.tpr, A.C);
      s2 = ffma2(f[p], f[p], s2);
    }
    const float var = group_sum(s2.x + s2.y, A.tpr, group, sums, slot) * A.invC;
    const float rstd = 1.f / sqrtf(var + A.eps);
    opaque(w);
    opaque(b);
    alignas(16) T o[PER];
#pragma unroll
    for (int p = 0; p < PER / 2; ++p) put_two<T>(o + 2 * p, ffma2(mul2(f[p], dup(rstd)), two<P>(w + 2 * p), two<P>(b + 2 * p)));
    store_row<T, V, PER, WHOLE>(y + row * A.C, o, t, A.tpr, A.C);
    if (t == 0 && A.mean) A.mean[row] = mean, A.rstd[row] = rstd;
  }
  if (kRing && t == 0 && phase >= 2) drain(full[group], lost[group], A.stages, step, A.rows);
}

template <typename T, typename P, int V, int PER, bool WHOLE>
__global__ void __launch_bounds__(512) layer_norm_bwd_kernel(const NormArgs A) {
  extern __shared__ __align__(16) unsigned char ring[];  // [groups, stages, 2, C]; at the end the groups' sums [groups, 2, C]
  float* sums = reinterpret_cast<float*>(ring);
  __shared__ uint64_t full[kMaxGroups][kStages];
  __shared__ Lost lost[kMaxGroups];
  __shared__ Sums sx, sy;
  clear(sx);
  clear(sy);
  init_ring(full);
  __syncthreads();
  const int group = threadIdx.x / A.tpr, t = threadIdx.x - group * A.tpr;
  int slot = 0;
  float2 w[PER / 2], dw[PER / 2], db[PER / 2];
  load_param<P, V, PER>(w, A.w, 1.f, t, A.tpr, A.C);
#pragma unroll
  for (int p = 0; p < PER / 2; ++p) dw[p] = db[p] = dup(0.f);
  const long long step = (long long)gridDim.x * A.groups;
  long long row = (long long)blockIdx.x * A.groups + group;
  const T* x = static_cast<const T*>(A.x);
  const T* dy = static_cast<const T*>(A.dy);
  constexpr bool kRing = V > 1;
  const int bytes = A.C * (int)sizeof(T);
  unsigned char* mine = ring + (size_t)group * A.stages * 2 * bytes;
  const auto fetch = [&](int i, long long r) {
    expect(&full[group][i], 2 * bytes);
    bulk_row(mine + (size_t)i * 2 * bytes, x + r * A.xs, bytes, &full[group][i]);
    bulk_row(mine + ((size_t)i * 2 + 1) * bytes, dy + r * A.ds, bytes, &full[group][i]);
  };
  alignas(16) T cx[PER];
  alignas(16) T cd[PER];
  float mean = 0.f, rstd = 0.f;
  if (row < A.rows) mean = A.mean[row], rstd = A.rstd[row];
  if (kRing) {
    if (t == 0)
      for (int i = 0; i < A.stages; ++i)
        if (row + i * step < A.rows) fetch(i, row + i * step);
  } else if (row < A.rows) {
    load_row<T, V, PER, WHOLE>(cx, x + row * A.xs, t, A.tpr, A.C);
    load_row<T, V, PER, WHOLE>(cd, dy + row * A.ds, t, A.tpr, A.C);
  }
  int at = 0, phase = 0;
  // phase: from 2 on once a wait has run out; this thread's part of a row is NaN then, and so are its group's results
  for (; row < A.rows; row += step) {
    if (kRing) {
      if (phase < 2 && !wait_phase(&full[group][at], phase, A.patience)) {
        if (t == 0) lost[group] = {row, at, phase};
        phase |= 2;
        atomicExch(&g_ran_out, 1u);
      }
      if (phase < 2) {
        load_row<T, V, PER, WHOLE>(cx, reinterpret_cast<const T*>(mine + (size_t)at * 2 * bytes), t, A.tpr, A.C);
        load_row<T, V, PER, WHOLE>(cd, reinterpret_cast<const T*>(mine + ((size_t)at * 2 + 1) * bytes), t, A.tpr, A.C);
      } else {
        no_row(cx);
        no_row(cd);
      }
    }
    const float r = rstd;  // of this row: the next one's is fetched below
    float2 h[PER / 2], g[PER / 2], s1 = dup(0.f), s2 = dup(0.f);
#pragma unroll
    for (int p = 0; p < PER / 2; ++p) {
      const float2 d = two<T>(cd + 2 * p);  // zero past C, and so is all that it multiplies
      h[p] = mul2(csub(two<T>(cx + 2 * p), dup(mean)), dup(r));
      g[p] = mul2(d, w[p]);
      dw[p] = ffma2(d, h[p], dw[p]);
      db[p] = cadd(db[p], d);
      s1 = cadd(s1, g[p]);
      s2 = ffma2(g[p], h[p], s2);
    }
    if (row + step < A.rows) {
      if (!kRing) {
        load_row<T, V, PER, WHOLE>(cx, x + (row + step) * A.xs, t, A.tpr, A.C);
        load_row<T, V, PER, WHOLE>(cd, dy + (row + step) * A.ds, t, A.tpr, A.C);
      }
      mean = A.mean[row + step], rstd = A.rstd[row + step];
    }
    float2 s = group_sum(make_float2(s1.x + s1.y, s2.x + s2.y), A.tpr, group, sx, sy, slot);
    if (kRing) {  // every thread of the group has read its part of both rows
      if (t == 0 && phase < 2 && row + A.stages * step < A.rows) fetch(at, row + A.stages * step);
      if (++at == A.stages) at = 0, phase ^= 1;
    }
    s.x *= A.invC, s.y *= A.invC;
    if (A.dx) {
      alignas(16) T o[PER];
#pragma unroll
      for (int p = 0; p < PER / 2; ++p)
        put_two<T>(o + 2 * p, mul2(csub(ffma2(h[p], dup(-s.y), g[p]), dup(s.x)), dup(r)));
      store_row<T, V, PER, WHOLE>(static_cast<T*>(A.dx) + row * A.C, o, t, A.tpr, A.C);
    }
  }
  if (kRing && t == 0 && phase >= 2) drain(full[group], lost[group], A.stages, step, A.rows);
  if (!A.part) return;
  __syncthreads();  // the ring is read
  float* out = A.part + (long long)blockIdx.x * 2 * A.C;
  float* to = A.groups == 1 ? out : sums + (long long)group * 2 * A.C;
#pragma unroll
  for (int e = 0; e < PER; ++e) {
    const int c = column<V>(e, t, A.tpr);
    if (WHOLE || c < A.C) to[c] = (&dw[e / 2].x)[e & 1], to[A.C + c] = (&db[e / 2].x)[e & 1];
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
template <typename T, typename P>
__global__ void __launch_bounds__(kLoopThreads) layer_norm_fwd_loop_kernel(const NormArgs A) {
  __shared__ Sums sums;
  int slot = 0;
  for (long long row = blockIdx.x; row < A.rows; row += gridDim.x) {
    const T* x = static_cast<const T*>(A.x) + row * A.xs;
    T* y = static_cast<T*>(A.y) + row * A.C;
    float s = 0.f;
    for (int c = threadIdx.x; c < A.C; c += kLoopThreads) s += DT<T>::load(x + c);
    const float mean = group_sum(s, kLoopThreads, 0, sums, slot) * A.invC;
    s = 0.f;
    for (int c = threadIdx.x; c < A.C; c += kLoopThreads) {
      const float d = DT<T>::load(x + c) - mean;
      s = fmaf(d, d, s);
    }
    const float var = group_sum(s, kLoopThreads, 0, sums, slot) * A.invC;
    const float rstd = 1.f / sqrtf(var + A.eps);
    for (int c = threadIdx.x; c < A.C; c += kLoopThreads) {
      const float w = A.w ? DT<P>::load(static_cast<const P*>(A.w) + c) : 1.f, b = A.b ? DT<P>::load(static_cast<const P*>(A.b) + c) : 0.f;
      DT<T>::store(y + c, fmaf((DT<T>::load(x + c) - mean) * rstd, w, b));
    }
    if (threadIdx.x == 0 && A.mean) A.mean[row] = mean, A.rstd[row] = rstd;
  }
}

// The same backwards; a CTA's sums of dw and db live in its own row of `part`, each column touched by one thread.
template <typename T, typename P>
__global__ void __launch_bounds__(kLoopThreads) layer_norm_bwd_loop_kernel(const NormArgs A) {
  __shared__ Sums sx, sy;
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
      const float g = A.w ? d * DT<P>::load(static_cast<const P*>(A.w) + c) : d;
      s.x += g;
      s.y = fmaf(g, h, s.y);
      if (out) {
        out[c] = fmaf(d, h, out[c]);
        out[A.C + c] += d;
      }
    }
    s = group_sum(s, kLoopThreads, 0, sx, sy, slot);
    s.x *= A.invC, s.y *= A.invC;
    if (A.dx) {
      T* dx = static_cast<T*>(A.dx) + row * A.C;
      for (int c = threadIdx.x; c < A.C; c += kLoopThreads) {
        const float d = DT<T>::load(dy + c), h = (DT<T>::load(x + c) - mean) * rstd;
        const float g = A.w ? d * DT<P>::load(static_cast<const P*>(A.w) + c) : d;
        DT<T>::store(dx + c, rstd * (g - s.x - h * s.y));
      }
    }
  }
}

// part [n, 2 C] -> dw, db: 32 columns by 32 strands per CTA, each strand every 32nd row, then the strands in order.
template <typename P>
__global__ void __launch_bounds__(1024) layer_norm_reduce_kernel(const float* __restrict__ part, int n, int C, P* dw, P* db) {
  __shared__ float red[32][33];
  const int lane = threadIdx.x & 31, strand = threadIdx.x >> 5;
  const int c = blockIdx.x * 32 + lane;
  float s = 0.f;
  if (c < 2 * C) {
#pragma unroll 4
    for (int i = strand; i < n; i += 32) s += part[(long long)i * 2 * C + c];
  }
  red[strand][lane] = s;
  __syncthreads();
  s = warp_sum(red[lane][strand]);  // column blockIdx.x * 32 + strand, in a fixed order
  const int d = blockIdx.x * 32 + strand;
  if (lane == 0 && d < 2 * C) {
    if (d < C) {
      if (dw) DT<P>::store(dw + d, s);
    } else if (db) {
      DT<P>::store(db + d - C, s);
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

// Few warps for each row (their sums meet at a barrier), enough rows on an SM to keep its share of HBM's latency covered.
// ctas is an upper bound (and the number of partial rows of the backward): the launch takes what is resident at once.
NormPlan plan(long long rows, int C) {
  NormPlan p{};
  if (C > kMaxRow) {
    p.tpr = kLoopThreads, p.groups = 1;
    p.ctas = (int)std::min<long long>(rows, 2 * 148);
    return p;
  }
  p.per = C <= 256 * 8 ? 8 : C <= 512 * 16 ? 16 : 32;
  p.tpr = std::max(32, ((C + p.per - 1) / p.per + 31) / 32 * 32);
  p.groups = std::max(1, std::min(kMaxGroups, 256 / p.tpr));
  p.ctas = (int)std::max<long long>(1, std::min<long long>((rows + p.groups - 1) / p.groups, 148ll * 8));
  return p;
}

// CTAs of a kernel that fit the device at once, asked once for each kernel, block and device.
int resident(const void* fn, int threads, size_t smem) {
  static std::mutex mu;
  static std::map<std::tuple<const void*, int, size_t, int>, int> known;
  int dev = 0;
  cudaGetDevice(&dev);
  std::lock_guard<std::mutex> lock(mu);
  auto it = known.find({fn, threads, smem, dev});
  if (it != known.end()) return it->second;
  int per_sm = 1, sms = 148;
  if (cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per_sm, fn, threads, smem) != cudaSuccess || per_sm < 1) per_sm = 1;
  cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
  cudaGetLastError();
  return known[{fn, threads, smem, dev}] = per_sm * sms;
}

template <typename T, typename P, int V, int PER, bool WHOLE>
int launch_rows(NormArgs& A, NormPlan& p, bool backward, cudaStream_t st) {
  const int threads = p.tpr * p.groups;
  // the ring: as many rows as 64 KB hold (three CTAs on an SM), two at least where 200 KB hold them
  const size_t row = (size_t)A.C * sizeof(T) * (backward ? 2 : 1) * p.groups;
  A.stages = (int)std::max<size_t>(2 * row <= 200 * 1024 ? 2 : 1, std::min<size_t>(kStages, 64 * 1024 / row));
  size_t sm = V > 1 ? row * A.stages : 0;
  if (backward && A.part && p.groups > 1) sm = std::max(sm, sizeof(float) * 2 * (size_t)p.groups * A.C);
  const void* fn = backward ? (const void*)layer_norm_bwd_kernel<T, P, V, PER, WHOLE> : (const void*)layer_norm_fwd_kernel<T, P, V, PER, WHOLE>;
  if (!kernel_smem_once(fn, sm)) return set_error(HYFFT_ERR_CUDA, "layer norm: shared memory");
  p.ctas = std::min(p.ctas, resident(fn, threads, sm));
  if (backward)
    layer_norm_bwd_kernel<T, P, V, PER, WHOLE><<<p.ctas, threads, sm, st>>>(A);
  else
    layer_norm_fwd_kernel<T, P, V, PER, WHOLE><<<p.ctas, threads, sm, st>>>(A);
  return launched();
}

template <typename T, typename P, int V, int PER>
int launch_per(NormArgs& A, NormPlan& p, bool backward, cudaStream_t st) {
  return A.C == p.tpr * PER ? launch_rows<T, P, V, PER, true>(A, p, backward, st)
                            : launch_rows<T, P, V, PER, false>(A, p, backward, st);
}

template <typename T, typename P, int V>
int launch_v(NormArgs& A, NormPlan& p, bool backward, cudaStream_t st) {
  if (p.per == 8) return launch_per<T, P, V, 8>(A, p, backward, st);
  if (p.per == 16) return launch_per<T, P, V, 16>(A, p, backward, st);
  return launch_per<T, P, V, 32>(A, p, backward, st);
}

bool aligned(const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }

template <typename T, typename P>
int launch_t(NormArgs& A, NormPlan& p, bool backward, cudaStream_t st) {
  A.tpr = p.tpr, A.groups = p.groups;
  A.patience = g_wait_clocks.load(std::memory_order_relaxed);
  A.invC = 1.f / (float)A.C;
  if (p.per == 0) {
    if (backward)
      layer_norm_bwd_loop_kernel<T, P><<<p.ctas, kLoopThreads, 0, st>>>(A);
    else
      layer_norm_fwd_loop_kernel<T, P><<<p.ctas, kLoopThreads, 0, st>>>(A);
    return launched();
  }
  constexpr int V = 16 / (int)sizeof(T);
  bool vec = A.C % V == 0 && A.xs % V == 0 && aligned(A.x) && aligned(A.y) && aligned(A.dx);
  if (backward) vec = vec && A.ds % V == 0 && aligned(A.dy);
  return vec ? launch_v<T, P, V>(A, p, backward, st) : launch_v<T, P, 1>(A, p, backward, st);
}

int check_args(int64_t rows, int64_t C, int32_t dtype, int32_t param_dtype) {
  if (rows < 1 || C < 1 || C > 0x3fffffff) return set_error(HYFFT_ERR_INVALID, "layer norm: rows and columns must be positive");
  if (dtype < HYFFT_F32 || dtype > HYFFT_F16) return set_error(HYFFT_ERR_INVALID, "layer norm: bad dtype");
  if (param_dtype != HYFFT_F32 && param_dtype != dtype)
    return set_error(HYFFT_ERR_INVALID, "layer norm: weight and bias have x's dtype or float32");
  return HYFFT_OK;
}

}  // namespace

int norm_wait_status(bool clear, unsigned* ran_out) { return read_ran_out(clear, ran_out) == cudaSuccess ? HYFFT_OK : HYFFT_ERR_CUDA; }

namespace {

int run(NormArgs& A, NormPlan& p, int32_t dtype, int32_t param_dtype, bool backward, cudaStream_t st) {
  if (dtype == HYFFT_F32) return launch_t<float, float>(A, p, backward, st);
  if (dtype == HYFFT_BF16)
    return param_dtype == HYFFT_F32 ? launch_t<__nv_bfloat16, float>(A, p, backward, st)
                                    : launch_t<__nv_bfloat16, __nv_bfloat16>(A, p, backward, st);
  return param_dtype == HYFFT_F32 ? launch_t<__half, float>(A, p, backward, st) : launch_t<__half, __half>(A, p, backward, st);
}

}  // namespace
}  // namespace hyfft

using namespace hyfft;

extern "C" {

int hyfft_layer_norm_workspace_size(int64_t rows, int64_t C, size_t* bwd_bytes) {
  const int rc = check_args(rows, C, HYFFT_F32, HYFFT_F32);
  if (rc != HYFFT_OK) return rc;
  if (bwd_bytes) *bwd_bytes = sizeof(float) * 2 * (size_t)C * plan(rows, (int)C).ctas;
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
  A.rows = rows, A.C = (int)C, A.xs = x_stride, A.eps = eps;
  NormPlan p = plan(rows, (int)C);
  return run(A, p, dtype, param_dtype, false, static_cast<cudaStream_t>(stream));
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
  NormPlan p = plan(rows, (int)C);
  if (sums && (!workspace || workspace_bytes < sizeof(float) * 2 * (size_t)C * p.ctas))
    return set_error(HYFFT_ERR_WORKSPACE, "layer norm: workspace too small");
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  NormArgs A{};
  A.x = x, A.w = weight, A.dy = dy, A.dx = dx;
  A.mean = const_cast<float*>(mean), A.rstd = const_cast<float*>(rstd);
  A.rows = rows, A.C = (int)C, A.xs = x_stride, A.ds = dy_stride;
  A.part = sums ? static_cast<float*>(workspace) : nullptr;
  int r = run(A, p, dtype, param_dtype, true, st);
  if (r != HYFFT_OK || !sums) return r;
  const unsigned grid = (unsigned)((2 * C + 31) / 32);
  if (param_dtype == HYFFT_F32)
    layer_norm_reduce_kernel<float><<<grid, 1024, 0, st>>>(A.part, p.ctas, (int)C, (float*)dweight, (float*)dbias);
  else if (dtype == HYFFT_BF16)
    layer_norm_reduce_kernel<__nv_bfloat16><<<grid, 1024, 0, st>>>(A.part, p.ctas, (int)C, (__nv_bfloat16*)dweight,
                                                                 (__nv_bfloat16*)dbias);
  else
    layer_norm_reduce_kernel<__half><<<grid, 1024, 0, st>>>(A.part, p.ctas, (int)C, (__half*)dweight, (__half*)dbias);
  return launched();
}

}  // extern "C"
