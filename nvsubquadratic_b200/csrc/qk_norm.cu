// The norm of every head of queries and keys, and rotary positions, in one pass, forward and backward.
//
//   r = 1 / sqrt(mean(x^2) + eps),  h = x r,  y = R (h w)         R: the turn of rotary.cu, scaled by the amplitude
//   t = R^T dy,  g = t w,  dx = r (g - h mean(g h)),  dw = sum over tokens and heads of t h
//
// Bound by HBM bandwidth: x is read once and y written once forwards; x and dy read, dx written backwards (the norm is computed
// again from x, which has to be read anyway). A group of 2^k lanes holds one row (a head of one token) in registers, so the sums
// are a few shuffles; a lane holds the same features of every row it sees, so it keeps their weights, turns the angle of its pairs
// once for all heads of a token, and adds its part of the weights' gradients in registers. A CTA adds those in shared memory into one
// partial row, and a second kernel adds the rows in a fixed order: no atomics, the same bits every run.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <math_constants.h>

#include <algorithm>
#include <atomic>
#include <type_traits>

#include "../../include/hyfft.h"
#include "common.cuh"

namespace hyfft {

extern std::atomic<long long> g_launches;
int set_error(int code, const char* msg);  // engine.cu: the message hyfft_last_error returns

namespace {

constexpr int kThreads = 256;
constexpr int kMaxDim = 256;
constexpr int kMaxCtas = 296;  // partial rows of a weight's gradient: two CTAs an SM

struct QkArgs {
  const void* x[2];
  const void* dy[2];
  void* out[2];                   // y; backwards dx. contiguous
  const void* w[2];
  long long xb[2], xl[2], xh[2];  // element strides of batch, token, head
  long long db[2], dl[2], dh[2];  // of dy
  int heads[2];
  const long long* turns;
  const void* pos;
  long long pb, pl;
  int pos32, w32;                 // the weights are float32
  float amplitude, eps;
  float* partial;                 // [2][CTAs][D]
  int D, half, want_dw;
  int groups[2], ctas[2];         // groups of heads of a token; CTAs (q's first)
  long long L, tokens, items[2];  // items: (token, group of heads)
};

// Where the features of lane j are: U units of 2 V features, two runs of V (halves; units past the pairs hold the features that are not
// turned) or one of 2 V (neighbours).
template <typename T, int V> struct alignas(16) Unit { T e[2 * V]; };

template <typename T, int R>
__device__ __forceinline__ void move_run(T* dst, const T* src) {
  if constexpr (R * sizeof(T) == 16) {
    *reinterpret_cast<uint4*>(dst) = *reinterpret_cast<const uint4*>(src);
  } else {
    static_assert(R <= 2, "longer runs are aligned");
#pragma unroll
    for (int u = 0; u < R; ++u) dst[u] = src[u];
  }
}

// V: pairs of a unit; U: units of a lane; G: lanes of a row.
template <typename T, int V, int U, bool INTER, bool BACK>
struct Rows {
  static constexpr int E = 2 * V * U;  // features of a lane

  // The first feature of each run of a unit, and how many features it has. Neighbours: one run, whether its pairs are turned or not.
  static __device__ __forceinline__ void runs(const QkArgs& A, int unit, int (&c)[2], int (&n)[2]) {
    if constexpr (INTER) {
      c[0] = unit * 2 * V, n[0] = min(max(A.D - c[0], 0), 2 * V), c[1] = 0, n[1] = 0;
    } else {
      const int pairs = (A.half + V - 1) / V;
      if (unit < pairs) {
        const int p = unit * V, k = min(V, A.half - p);
        c[0] = p, n[0] = k, c[1] = p + A.half, n[1] = k;
      } else {
        const int p = 2 * A.half + (unit - pairs) * 2 * V, left = max(min(2 * V, A.D - p), 0);
        c[0] = p, n[0] = min(V, left), c[1] = p + V, n[1] = left - n[0];
      }
    }
  }
  // places of the runs' features within the unit
  static constexpr int kFirst = INTER ? 2 * V : V;

  static constexpr bool kWide = V > 1;
  static __device__ __forceinline__ void fetch(const QkArgs& A, const T* row, int unit, Unit<T, V>& d) {
    int c[2], n[2];
    runs(A, unit, c, n);
    if constexpr (kWide) {
      if (n[0]) move_run<T, kFirst>(d.e, row + c[0]);
      if constexpr (!INTER)
        if (n[1]) move_run<T, V>(d.e + V, row + c[1]);
    } else {
#pragma unroll
      for (int u = 0; u < kFirst; ++u)
        if (u < n[0]) d.e[u] = row[c[0] + u];
      if constexpr (!INTER)
#pragma unroll
        for (int u = 0; u < V; ++u)
          if (u < n[1]) d.e[V + u] = row[c[1] + u];
    }
  }
  static __device__ __forceinline__ void unpack(const Unit<T, V>& d, float* v) {
#pragma unroll
    for (int u = 0; u < V; ++u) {
      float2 f;
      if constexpr (std::is_same<T, float>::value) {
        f = make_float2(d.e[2 * u], d.e[2 * u + 1]);
      } else if constexpr (std::is_same<T, __half>::value) {
        f = __half22float2(*reinterpret_cast<const __half2*>(d.e + 2 * u));
      } else {
        const uint32_t w = *reinterpret_cast<const uint32_t*>(d.e + 2 * u);
        f = make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
      }
      v[2 * u] = f.x, v[2 * u + 1] = f.y;
    }
  }
  static __device__ __forceinline__ void store(const QkArgs& A, T* row, int unit, const float* v) {
    int c[2], n[2];
    runs(A, unit, c, n);
    if constexpr (kWide) {
      Unit<T, V> d;
#pragma unroll
      for (int u = 0; u < V; ++u) {
        if constexpr (std::is_same<T, float>::value) {
          d.e[2 * u] = v[2 * u], d.e[2 * u + 1] = v[2 * u + 1];
        } else if constexpr (std::is_same<T, __half>::value) {
          *reinterpret_cast<__half2*>(d.e + 2 * u) = __floats2half2_rn(v[2 * u], v[2 * u + 1]);
        } else {
          *reinterpret_cast<__nv_bfloat162*>(d.e + 2 * u) = __floats2bfloat162_rn(v[2 * u], v[2 * u + 1]);
        }
      }
      if (n[0]) move_run<T, kFirst>(row + c[0], d.e);
      if constexpr (!INTER)
        if (n[1]) move_run<T, V>(row + c[1], d.e + V);
    } else {
#pragma unroll
      for (int u = 0; u < kFirst; ++u)
        if (u < n[0]) DT<T>::store(row + c[0] + u, v[u]);
      if constexpr (!INTER)
#pragma unroll
        for (int u = 0; u < V; ++u)
          if (u < n[1]) DT<T>::store(row + c[1] + u, v[V + u]);
    }
  }
};

// The pairs of a unit turned (back: turned back), the first `on` of them; places (2 u, 2 u + 1) or (u, V + u).
template <int V, bool INTER>
__device__ __forceinline__ void turn(float* v, const float* cs, const float* sn, int on) {
  const auto one = [&](int u) {
    float &a = v[INTER ? 2 * u : u], &b = v[INTER ? 2 * u + 1 : V + u];
    const float x = a, y = b;
    a = fmaf(x, cs[u], -y * sn[u]);
    b = fmaf(x, sn[u], y * cs[u]);
  };
  if (on >= V) {
#pragma unroll
    for (int u = 0; u < V; ++u) one(u);
  } else if (INTER && V > 1 && on > 0) {  // a unit that the turned features end in
#pragma unroll
    for (int u = 0; u < V; ++u)
      if (u < on) one(u);
  }
}

template <int G> __device__ __forceinline__ float sum_of(float v) {
#pragma unroll
  for (int d = 1; d < G; d *= 2) v += __shfl_xor_sync(0xffffffffu, v, d);
  return v;
}

// Squares below this have fewer digits, or none, in the sum: mean + eps of a row that needs them.
constexpr float kSmallMean = 8.0779357e-28f;  // 2^-90
// 1 / sqrt(mean + eps) of a row whose squares leave float32's range although its features do not: of the row times 2^-100 or 2^100.
template <int E, int G> __device__ __forceinline__ float of_extreme(const float (&v)[E], float ss, float r, float inv, float eps) {
  float m = 0.0f, s = 0.0f;
#pragma unroll
  for (int e = 0; e < E; ++e) m = fmaxf(m, fabsf(v[e]));
#pragma unroll
  for (int d = 1; d < G; d *= 2) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, d));
  const float up = m > 1.0f ? 7.8886091e-31f : 1.2676506e30f;
#pragma unroll
  for (int e = 0; e < E; ++e) s = fmaf(v[e] * up, v[e] * up, s);
  s = sum_of<G>(s);
  const bool large = ss == CUDART_INF_F && m < CUDART_INF_F, small = fmaf(ss, inv, eps) < kSmallMean && m > 0.0f;
  // below 2^-126 a row counts as if it were there
  return large || small ? fminf(rsqrtf(fmaf(s, inv, eps * up * up)) * up, 3.4028235e38f) : r;
}

// Groups of G lanes walk over the items of one tensor (q's CTAs and k's are apart: one set of weights and of their sums in registers). The
// next HB rows' loads are in flight while HB are worked on. 65536 tokens of 32 + 32 heads of 128, bfloat16: 414 us forwards (79%
// of a copy's rate) and 652 backwards (75%; the 16-bit kernels with 8 pairs a lane are at their 128 registers and spill 52 to 68 bytes); without
// the loads ahead 424 with four rows at once, and 789 with two backwards; with 8 bytes a run instead of 16, twice the lanes of a row, 449 and 812.
// Neighbouring pairs have 8 features a lane, and room for three CTAs an SM instead of two forwards (32 + 8 heads: 265 against 338 us); turned or
// not they lie side by side, so their runs are aligned wherever the turned features end (26 x 3238 tokens, 2 + 2 heads of 128, 18 turned,
// training: 476 -> 189 us).
template <typename T, int V, int U, int G, bool INTER, bool BACK>
__global__ void __launch_bounds__(kThreads, BACK || 2 * V * U > 8 ? 2 : 3) qk_norm_kernel(const QkArgs A) {
  using R = Rows<T, V, U, INTER, BACK>;
  constexpr int E = R::E, HB = BACK ? 1 : 2;
  const int lane = threadIdx.x % G;
  const int k = blockIdx.x >= A.ctas[0];
  const int cta = blockIdx.x - (k ? A.ctas[0] : 0), ctas = A.ctas[k], heads = A.heads[k], groups = A.groups[k];
  const long long items = A.items[k];
  float w[E], dw[BACK ? E : 1];
#pragma unroll
  for (int n = 0; n < U; ++n) {
    int c[2], m[2];
    R::runs(A, lane + n * G, c, m);
#pragma unroll
    for (int e = 0; e < 2 * V; ++e) {  // one by one: the weights' alignment is not known, and they are read once
      const int run = e < R::kFirst ? 0 : 1, at = e - run * R::kFirst;
      float& to = w[n * 2 * V + e];
      to = 1.0f;
      if (A.w[k] && at < m[run])
        to = A.w32 ? static_cast<const float*>(A.w[k])[c[run] + at] : DT<T>::load(static_cast<const T*>(A.w[k]) + c[run] + at);
    }
  }
  if constexpr (BACK) {
#pragma unroll
    for (int e = 0; e < E; ++e) dw[e] = 0.0f;
  }
  const float inv = 1.0f / A.D;
  const long long stride = (long long)ctas * (kThreads / G);
  const long long xh = A.xh[k], dh = BACK ? A.dh[k] : 0;
  // all lanes of a warp take the same number of turns (the sums are over whole warps)
  const long long base = (long long)cta * (kThreads / G) + threadIdx.x / 32 * (32 / G);
  for (long long first = base; first < items; first += stride) {
    const long long item = first + threadIdx.x % 32 / G;
    const bool live = item < items;
    long long tok = 0, b = 0;
    if (live && items < (1ll << 31) && A.L < (1ll << 31)) {  // a 64-bit division costs as much as a row
      tok = (unsigned)item / (unsigned)groups;
      b = (unsigned)tok / (unsigned)A.L;
    } else if (live) {
      tok = item / groups;
      b = tok / A.L;
    }
    const int grp = live ? (int)(item - tok * groups) : heads;
    const long long l = tok - b * A.L;
    const T* x = static_cast<const T*>(A.x[k]) + b * A.xb[k] + l * A.xl[k];
    const T* dy = BACK ? static_cast<const T*>(A.dy[k]) + b * A.db[k] + l * A.dl[k] : nullptr;
    T* out = static_cast<T*>(A.out[k]) + tok * heads * (long long)A.D;
    struct Raw {
      Unit<T, V> x[HB][U], d[BACK ? HB : 1][U];
    };
    const auto fetch = [&](int h0, Raw& raw) {  // heads h0, h0 + groups, ...
#pragma unroll
      for (int j = 0; j < HB; ++j) {
        const int h = h0 + j * groups;
#pragma unroll
        for (int n = 0; n < U; ++n) {
          raw.x[j][n] = Unit<T, V>{};
          if constexpr (BACK) raw.d[j][n] = Unit<T, V>{};
          if (h < heads) {
            R::fetch(A, x + h * xh, lane + n * G, raw.x[j][n]);
            if constexpr (BACK) R::fetch(A, dy + h * dh, lane + n * G, raw.d[j][n]);
          }
        }
      }
    };
    Raw raw, ahead;
    fetch(grp, raw);
    float cs[U][V], sn[U][V];
    {
      long long p = l;
      if (A.pos) {
        const long long at = b * A.pb + l * A.pl;
        p = A.pos32 ? (long long)static_cast<const int*>(A.pos)[at] : static_cast<const long long*>(A.pos)[at];
      }
#pragma unroll
      for (int n = 0; n < U; ++n)
#pragma unroll
        for (int u = 0; u < V; ++u) {
          const int pair = (lane + n * G) * V + u;
          cs[n][u] = 1.0f, sn[n][u] = 0.0f;
          if (pair < A.half) {
            const unsigned long long t = (unsigned long long)p * (unsigned long long)A.turns[pair];
            float s, c;
            sincospif((float)(int)(t >> 32) * 4.656612873077393e-10f, &s, &c);  // half turns of 2^-31
            cs[n][u] = c * A.amplitude;
            sn[n][u] = BACK ? -s * A.amplitude : s * A.amplitude;
          }
        }
    }
    const int rounds = (heads + groups - 1) / groups;
#pragma unroll 2
    for (int i = 0; i < rounds; i += HB) {
      const int h0 = grp + i * groups;
      if (i + HB < rounds) fetch(h0 + HB * groups, ahead);  // while these are worked on
#pragma unroll
      for (int j = 0; j < HB; ++j) {
        const int h = h0 + j * groups;
        const bool on = h < heads;
        float v[E];
#pragma unroll
        for (int n = 0; n < U; ++n) R::unpack(raw.x[j][n], v + n * 2 * V);
        float ss = 0.0f;
#pragma unroll
        for (int e = 0; e < E; ++e) ss = fmaf(v[e], v[e], ss);
        ss = sum_of<G>(ss);
        const float mean = fmaf(ss, inv, A.eps);
        float r = rsqrtf(mean);
        if (__any_sync(0xffffffffu, mean < kSmallMean || ss == CUDART_INF_F)) r = of_extreme<E, G>(v, ss, r, inv, A.eps);
        if (!on) r = 0.0f;
        if constexpr (!BACK) {
#pragma unroll
          for (int e = 0; e < E; ++e) v[e] = v[e] * r * w[e];
#pragma unroll
          for (int n = 0; n < U; ++n) {
            turn<V, INTER>(v + n * 2 * V, cs[n], sn[n], A.half - (lane + n * G) * V);
            if (on) R::store(A, out + (long long)h * A.D, lane + n * G, v + n * 2 * V);
          }
        } else {
          float t[E], gh = 0.0f;
#pragma unroll
          for (int n = 0; n < U; ++n) {
            R::unpack(raw.d[j][n], t + n * 2 * V);
            turn<V, INTER>(t + n * 2 * V, cs[n], sn[n], A.half - (lane + n * G) * V);
          }
#pragma unroll
          for (int e = 0; e < E; ++e) {
            v[e] *= r;
            dw[e] = fmaf(t[e], v[e], dw[e]);
            t[e] *= w[e];
            gh = fmaf(t[e], v[e], gh);
          }
          gh = sum_of<G>(gh) * inv;
#pragma unroll
          for (int e = 0; e < E; ++e) v[e] = r * fmaf(-gh, v[e], t[e]);
#pragma unroll
          for (int n = 0; n < U; ++n)
            if (on) R::store(A, out + (long long)h * A.D, lane + n * G, v + n * 2 * V);
        }
      }
      raw = ahead;
    }
  }
  if constexpr (BACK) {
    if (!A.want_dw || !A.w[k]) return;
    // this CTA's sums over its groups, in their order
    extern __shared__ float part[];  // [groups of the CTA][D]
    float* mine = part + threadIdx.x / G * A.D;
#pragma unroll
    for (int n = 0; n < U; ++n) {
      int c[2], m[2];
      R::runs(A, lane + n * G, c, m);
#pragma unroll
      for (int e = 0; e < 2 * V; ++e) {
        const int run = e < R::kFirst ? 0 : 1, at = e - run * R::kFirst;
        if (at < m[run]) mine[c[run] + at] = dw[n * 2 * V + e];
      }
    }
    __syncthreads();
    for (int c = threadIdx.x; c < A.D; c += kThreads) {
      float s = 0.0f;
      for (int i = 0; i < kThreads / G; ++i) s += part[i * A.D + c];
      A.partial[((long long)k * kMaxCtas + cta) * A.D + c] = s;
    }
  }
}

// dw[k][c]: column c of the partial rows, in a fixed order. Eight columns (a sector) for each CTA.
template <typename W>
__global__ void __launch_bounds__(256) qk_norm_reduce_kernel(const float* partial, W* dwq, W* dwk, int D, int rows_q, int rows_k) {
  W* dw = blockIdx.y ? dwk : dwq;
  if (!dw) return;
  const int rows = blockIdx.y ? rows_k : rows_q;
  const int c = blockIdx.x * 8 + threadIdx.x % 8, i0 = threadIdx.x / 8;
  __shared__ float part[32][9];
  float s = 0.0f;
  if (c < D) {
    const float* p = partial + (long long)blockIdx.y * kMaxCtas * D + c;
#pragma unroll 4
    for (int i = i0; i < rows; i += 32) s += p[(long long)i * D];
  }
  part[i0][threadIdx.x % 8] = s;
  __syncthreads();
  if (threadIdx.x < 8 && c < D) {
    float t = 0.0f;
    for (int i = 0; i < 32; ++i) t += part[i][threadIdx.x];
    DT<W>::store(dw + c, t);
  }
}

template <typename T, int V, int U, int G, bool INTER, bool BACK>
int launch(QkArgs A, int* ctas, cudaStream_t st) {
  for (int k = 0; k < 2; ++k) {
    const int nh = A.heads[k];
    if (!nh) continue;
    // heads a group takes at one token: as many as share the turned angles, while there are 512 threads for each SM
    int per = std::min(nh, 16);
    while (per > 1 && A.tokens * G * ((nh + per - 1) / per) < 148ll * 512) per = (per + 1) / 2;
    A.groups[k] = (nh + per - 1) / per;
    A.items[k] = A.tokens * A.groups[k];
  }
  const long long most = kMaxCtas, all = A.heads[0] + A.heads[1];
  long long grid = 0;
  for (int k = 0; k < 2; ++k) {
    if (!A.heads[k]) continue;
    long long n = (A.items[k] + kThreads / G - 1) / (kThreads / G);
    // backwards the weights' sums stay in registers over many tokens: the CTAs that run at once, shared by the heads
    if (BACK) n = std::min(n, std::max(1ll, most * A.heads[k] / all));
    if (n > 0x3fffffffLL) return set_error(HYFFT_ERR_UNSUPPORTED, "qk norm: too many elements");
    A.ctas[k] = (int)n, grid += n;
  }
  if (ctas) ctas[0] = A.ctas[0], ctas[1] = A.ctas[1];
  const size_t smem = BACK ? sizeof(float) * (kThreads / G) * A.D : 0;
  const auto fn = qk_norm_kernel<T, V, U, G, INTER, BACK>;
  if (smem > 48 * 1024 && !kernel_smem_once(reinterpret_cast<const void*>(fn), smem))
    return set_error(HYFFT_ERR_CUDA, "qk norm: shared memory");
  fn<<<(unsigned)grid, kThreads, smem, st>>>(A);
  if (cudaGetLastError() != cudaSuccess) return set_error(HYFFT_ERR_CUDA, "qk norm: kernel launch failed");
  g_launches.fetch_add(1, std::memory_order_relaxed);
  return HYFFT_OK;
}

template <typename T, int V, int U, bool INTER, bool BACK>
int launch_lanes(const QkArgs& A, int lanes, int* ctas, cudaStream_t st) {
  if (lanes <= 4) return launch<T, V, U, 4, INTER, BACK>(A, ctas, st);
  if (lanes <= 8) return launch<T, V, U, 8, INTER, BACK>(A, ctas, st);
  if (lanes <= 16) return launch<T, V, U, 16, INTER, BACK>(A, ctas, st);
  return launch<T, V, U, 32, INTER, BACK>(A, ctas, st);
}

template <typename T, bool INTER, bool BACK> int launch_t(const QkArgs& A, int* ctas, cudaStream_t st) {
  constexpr int V = (INTER ? 8 : 16) / (int)sizeof(T), E = INTER ? 2 * V : V;  // pairs of a unit, elements of a run
  // Runs of 16 bytes where every run of every row starts on a 16-byte boundary, pairs of elements otherwise. 4 x 4096 tokens, 8 + 8 heads,
  // us forwards and backwards: 128 features turned of 128, bfloat16 39 and 88, float32 51 and 89; 24 of 96 (halves on 8 bytes, and on 16 in
  // float32) 98 and 185, 52 and 89; 76 of 77 82 and 160, 71 and 117.
  bool al = A.D % E == 0 && (INTER || A.half % E == 0);
  for (int k = 0; k < 2; ++k) {
    if (!A.heads[k]) continue;
    al = al && reinterpret_cast<uintptr_t>(A.x[k]) % (E * sizeof(T)) == 0 && reinterpret_cast<uintptr_t>(A.out[k]) % (E * sizeof(T)) == 0 &&
         A.xb[k] % E == 0 && A.xl[k] % E == 0 && A.xh[k] % E == 0;
    if (BACK) al = al && reinterpret_cast<uintptr_t>(A.dy[k]) % (E * sizeof(T)) == 0 && A.db[k] % E == 0 && A.dl[k] % E == 0 && A.dh[k] % E == 0;
  }
  const int v = al ? V : 1;
  const int units = INTER ? (A.D + 2 * v - 1) / (2 * v) : (A.half + v - 1) / v + (A.D - 2 * A.half + 2 * v - 1) / (2 * v);
  if (al) {
    if constexpr (V * 2 * 32 < kMaxDim)
      if (units > 32) return launch<T, V, 2, 32, INTER, BACK>(A, ctas, st);
    return launch_lanes<T, V, 1, INTER, BACK>(A, units, ctas, st);
  }
  if (units > 64) return launch<T, 1, 4, 32, INTER, BACK>(A, ctas, st);
  if (units > 32) return launch<T, 1, 2, 32, INTER, BACK>(A, ctas, st);
  return launch_lanes<T, 1, 1, INTER, BACK>(A, units, ctas, st);
}

template <bool BACK> int run(const hyfft_qk_norm_desc* d, const QkArgs& A, int* ctas, cudaStream_t st) {
  if (d->dtype == HYFFT_F32) return d->interleaved ? launch_t<float, true, BACK>(A, ctas, st) : launch_t<float, false, BACK>(A, ctas, st);
  if (d->dtype == HYFFT_BF16)
    return d->interleaved ? launch_t<__nv_bfloat16, true, BACK>(A, ctas, st) : launch_t<__nv_bfloat16, false, BACK>(A, ctas, st);
  return d->interleaved ? launch_t<__half, true, BACK>(A, ctas, st) : launch_t<__half, false, BACK>(A, ctas, st);
}

int check_desc(const hyfft_qk_norm_desc* d) {
  if (!d) return set_error(HYFFT_ERR_INVALID, "qk norm: null descriptor");
  if (d->batch < 1 || d->length < 1 || d->heads < 1 || d->kv_heads < 0 || d->dim < 1)
    return set_error(HYFFT_ERR_INVALID, "qk norm: every extent must be positive");
  if (d->rot_dim < 0 || d->rot_dim % 2 || d->rot_dim > d->dim)
    return set_error(HYFFT_ERR_INVALID, "qk norm: rot_dim must be even and at most the head size");
  if (d->dtype < HYFFT_F32 || d->dtype > HYFFT_F16) return set_error(HYFFT_ERR_INVALID, "qk norm: bad dtype");
  if (d->weight_dtype != d->dtype && d->weight_dtype != HYFFT_F32)
    return set_error(HYFFT_ERR_INVALID, "qk norm: the weights have the rows' dtype or float32");
  if (d->dim > kMaxDim) return set_error(HYFFT_ERR_UNSUPPORTED, "qk norm: heads above 256 features");
  return HYFFT_OK;
}

QkArgs args_of(const hyfft_qk_norm_desc* d, const void* q, const void* k, const void* qw, const void* kw, const int64_t* turns,
               const void* positions) {
  QkArgs A{};
  A.x[0] = q, A.x[1] = k, A.w[0] = qw, A.w[1] = kw;
  A.xb[0] = d->q_stride[0], A.xl[0] = d->q_stride[1], A.xh[0] = d->q_stride[2];
  A.xb[1] = d->k_stride[0], A.xl[1] = d->k_stride[1], A.xh[1] = d->k_stride[2];
  A.heads[0] = d->heads, A.heads[1] = d->kv_heads;
  A.turns = reinterpret_cast<const long long*>(turns);
  A.pos = positions, A.pb = d->pos_stride[0], A.pl = d->pos_stride[1], A.pos32 = d->pos_int32;
  A.amplitude = d->amplitude, A.eps = d->eps, A.w32 = d->weight_dtype == HYFFT_F32 && d->dtype != HYFFT_F32;
  A.D = d->dim, A.half = d->rot_dim / 2, A.L = d->length, A.tokens = (long long)d->batch * d->length;
  return A;
}

}  // namespace
}  // namespace hyfft

using namespace hyfft;

extern "C" int hyfft_qk_norm_workspace_size(const hyfft_qk_norm_desc* d, size_t* bwd_bytes) {
  if (int rc = check_desc(d)) return rc;
  if (!bwd_bytes) return set_error(HYFFT_ERR_INVALID, "qk norm: null size");
  *bwd_bytes = sizeof(float) * 2 * kMaxCtas * (size_t)d->dim;
  return HYFFT_OK;
}

extern "C" int hyfft_qk_norm_forward(const hyfft_qk_norm_desc* d, const void* q, const void* k, const void* q_weight,
                                     const void* k_weight, const int64_t* turns, const void* positions, void* out_q,
                                     void* out_k, void* stream) {
  if (int rc = check_desc(d)) return rc;
  if (!q || !out_q || (d->rot_dim && !turns) || (d->kv_heads && (!k || !out_k)))
    return set_error(HYFFT_ERR_INVALID, "qk norm: null tensor");
  if (bind_device_of(q) != HYFFT_OK) return set_error(HYFFT_ERR_CUDA, "qk norm: device");
  QkArgs A = args_of(d, q, k, q_weight, k_weight, turns, positions);
  A.out[0] = out_q, A.out[1] = out_k;
  return run<false>(d, A, nullptr, static_cast<cudaStream_t>(stream));
}

extern "C" int hyfft_qk_norm_backward(const hyfft_qk_norm_desc* d, const void* q, const void* k, const void* q_weight,
                                      const void* k_weight, const int64_t* turns, const void* positions, const void* dq_out,
                                      const void* dk_out, void* dq, void* dk, void* dq_weight, void* dk_weight,
                                      void* workspace, size_t workspace_bytes, void* stream) {
  if (int rc = check_desc(d)) return rc;
  if (!q || !dq_out || !dq || (d->rot_dim && !turns) || (d->kv_heads && (!k || !dk_out || !dk)))
    return set_error(HYFFT_ERR_INVALID, "qk norm: null tensor");
  if ((dq_weight && !q_weight) || (dk_weight && (!k_weight || !d->kv_heads)))
    return set_error(HYFFT_ERR_INVALID, "qk norm: a gradient of a weight that is not there");
  const bool want = dq_weight || dk_weight;
  size_t need = 0;
  if (int rc = hyfft_qk_norm_workspace_size(d, &need)) return rc;
  if (want && (!workspace || workspace_bytes < need)) return set_error(HYFFT_ERR_WORKSPACE, "qk norm: workspace too small");
  if (bind_device_of(q) != HYFFT_OK) return set_error(HYFFT_ERR_CUDA, "qk norm: device");
  QkArgs A = args_of(d, q, k, q_weight, k_weight, turns, positions);
  A.dy[0] = dq_out, A.dy[1] = dk_out, A.out[0] = dq, A.out[1] = dk;
  A.db[0] = d->dq_stride[0], A.dl[0] = d->dq_stride[1], A.dh[0] = d->dq_stride[2];
  A.db[1] = d->dk_stride[0], A.dl[1] = d->dk_stride[1], A.dh[1] = d->dk_stride[2];
  A.partial = static_cast<float*>(workspace), A.want_dw = want;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  int ctas[2] = {0, 0};
  if (int rc = run<true>(d, A, ctas, st)) return rc;
  if (!want) return HYFFT_OK;
  const dim3 grid((d->dim + 7) / 8, 2);
  if (d->weight_dtype == HYFFT_F32)
    qk_norm_reduce_kernel<float><<<grid, 256, 0, st>>>(A.partial, (float*)dq_weight, (float*)dk_weight, A.D, ctas[0], ctas[1]);
  else if (d->weight_dtype == HYFFT_BF16)
    qk_norm_reduce_kernel<__nv_bfloat16>
        <<<grid, 256, 0, st>>>(A.partial, (__nv_bfloat16*)dq_weight, (__nv_bfloat16*)dk_weight, A.D, ctas[0], ctas[1]);
  else
    qk_norm_reduce_kernel<__half><<<grid, 256, 0, st>>>(A.partial, (__half*)dq_weight, (__half*)dk_weight, A.D, ctas[0], ctas[1]);
  if (cudaGetLastError() != cudaSuccess) return set_error(HYFFT_ERR_CUDA, "qk norm: kernel launch failed");
  g_launches.fetch_add(1, std::memory_order_relaxed);
  return HYFFT_OK;
}
