// Linear attention with one decay for each head, over whole sequences and for single tokens.
//
//   S_t = a S_{t-1} + k_t v_t^T,   o_t = scale * S_t^T q_t,   a = exp(log_decay[h]),   S [Dk, Dv] float32
//
// The gradients are the same scan with other operands. With G_t = dL/dS_t running backwards,
//   dq_t = scale * S_t do_t               scan(do, v, k) forwards
//   dk_t = G_t v_t,  dv_t = G_t^T k_t     scan(v, do, q) and scan(k, q, do) backwards
//   G_t  = U_{t+1} + scale * q_t do_t^T,  U_t = a G_t,  U_L = dL/dS_L,  dL/dS_0 = U_0
// and the decay's, with T_t = dS_t / dlog_decay = a (T_{t-1} + S_{t-1}) carried beside S:
//   dlog_decay = scale * sum_t q_t^T T_t do_t + <dL/dS_L, T_L>.
//
// The scan kernel below takes every type and every head size up to 256 and computes in float32 multiply-adds. A thread
// owns four columns of the state and up to 32 of its rows in registers, packed in pairs of rows: a token costs two packed
// multiply-adds per pair (S += k v, o += q S). q and k are read from shared memory as broadcasts, which the register
// file takes at 128 bytes a cycle: one 16-byte read serves 16 multiply-adds here (with one column per thread it served four
// and the reads were the bound: 2.08 ms for 16 x 4096 tokens, 12 heads of 64, float16, instead of 1.04). The two halves of a
// warp hold two parts of the rows, their sums meet in one shuffle; states of more than 64 rows take more warps.
// Inside a chunk of 16 tokens the state is kept divided by a^i, which takes the decay out of the inner loop: v is
// multiplied by a^-i and o by a^i, each from a table, and the chunk's a^n is applied once, as the sum of two floats
// (a rounded a^n would be off by its rounding error times the number of chunks in a head's memory). Heads that
// forget more than e^-46 within a chunk, where a^-i would overflow, multiply the state for each token; so does a CTA whose
// results came out infinite or NaN, once more from the start, in case only the division by a^i made them so.
// What of this runs on the tensor cores instead (decay_mma.cu) says use_mma below.
// Few rows and a long axis: the axis is cut into segments; a first pass adds up each segment from a zero
// state, a small kernel chains the segments' states, and the second pass starts every segment from its own.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <atomic>
#include <type_traits>

#include "../../include/hyfft.h"
#include "common.cuh"
#include "decay_attn.h"

namespace hyfft {

extern std::atomic<long long> g_launches;
int set_error(int code, const char* msg);  // engine.cu: the message hyfft_last_error returns

namespace {

constexpr int kTok = 16;   // tokens per chunk
constexpr int kCols = 64;  // columns per CTA: 16 lanes x 4
constexpr int kMaxDim = 256;
constexpr double kFastLimit = 46.0;  // |log_decay| * kTok below this: a^-i stays below 1e20

using Op = ScanOp;

__device__ __forceinline__ float2 mul2(float2 a, float b) { return make_float2(a.x * b, a.y * b); }
__device__ __forceinline__ float2 dup(float a) { return make_float2(a, a); }

// Columns [c0, c0 + W) of n tokens (zeros past D); token of row i: t0 + i * step. Left in flight.
template <typename T, int W>
__device__ __forceinline__ void fetch_tile(T* dst, const T* __restrict__ src, long long sl, int n, int c0, int D,
                                           long long t0, int step) {
  constexpr int V = 16 / sizeof(T), kPer = W / V;
  for (int i = threadIdx.x; i < n * kPer; i += blockDim.x) {
    const int r = i / kPer, c = (i - r * kPer) * V;
    const bool ok = c0 + c < D;
    const T* s = ok ? src + (t0 + (long long)r * step) * sl + c0 + c : src;
    const unsigned d = (unsigned)__cvta_generic_to_shared(dst + r * W + c);
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;\n" ::"r"(d), "l"(s), "r"(ok ? 16 : 0) : "memory");
  }
}
// The same as floats, from any address, at once.
template <typename T, int W>
__device__ __forceinline__ void load_tile(float* dst, const T* __restrict__ src, long long sl, int n, int c0, int D,
                                          long long t0, int step) {
  for (int i = threadIdx.x; i < n * W; i += blockDim.x) {
    const int r = i / W, c = i - r * W;
    dst[i] = c0 + c < D ? DT<T>::load(src + (t0 + (long long)r * step) * sl + c0 + c) : 0.f;
  }
}
// n rows of a 16-bit tile to floats.
template <typename T, int W>
__device__ __forceinline__ void widen_tile(float* dst, const T* src, int n) {
  for (int i = threadIdx.x; i < n * W / 8; i += blockDim.x) {
    const uint4 raw = reinterpret_cast<const uint4*>(src)[i];
    const T* e = reinterpret_cast<const T*>(&raw);
    float4* d = reinterpret_cast<float4*>(dst) + 2 * i;
    d[0] = make_float4(DT<T>::load(e), DT<T>::load(e + 1), DT<T>::load(e + 2), DT<T>::load(e + 3));
    d[1] = make_float4(DT<T>::load(e + 4), DT<T>::load(e + 5), DT<T>::load(e + 6), DT<T>::load(e + 7));
  }
}

// Floats of shared memory: tiles as the inner loop reads them, two chunks as they arrive (16-bit types; a float32 chunk is
// read where it arrived), the parts of o where warps share a row.
template <typename T, int RH, int KW, bool LEARN>
struct Smem {
  static constexpr int W = 2 * RH * KW;
  static constexpr int chunk = kTok * (2 * W + kCols * (LEARN ? 2 : 1));  // elements
  static constexpr bool wide = sizeof(T) == 4;
  static constexpr int raw = wide ? 0 : chunk;                           // where the arriving chunks begin, in floats
  static constexpr int os = raw + (wide ? 2 * chunk : chunk);
  static constexpr int floats = os + (KW > 1 ? KW * kTok * kCols : 0);
};

// RH rows of the state in each thread (two halves of a warp: 2 RH rows), KW warps over its rows.
template <typename T, typename TO, int RH, int KW, bool LEARN>
__global__ void __launch_bounds__(32 * KW) decay_scan_kernel(const ScanArgs A) {
  using M = Smem<T, RH, KW, LEARN>;
  constexpr int W = M::W;
  extern __shared__ __align__(16) float smem[];
  float* os = smem + M::os;  // [KW][kTok][kCols]
  __shared__ float apow[kTok], ainv[kTok];

  long long id = blockIdx.x;
  const int slice = (int)(id % A.nslice);
  id /= A.nslice;
  const int seg = (int)(id % A.nseg);
  const long long bh = id / A.nseg;
  const int h = (int)(bh % A.H);
  const long long b = bh / A.H;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int c0 = slice * kCols, col = (lane & 15) * 4, row0 = (warp * 2 + (lane >> 4)) * RH;
  const int left = A.DV - c0 - col;  // columns from this thread's first on that exist

  int len = A.L;
  if (A.lengths) len = min(max(A.lengths[b], 0), A.L);
  const long long t_lo = (long long)seg * A.seglen;
  const long long t_end = min(t_lo + A.seglen, (long long)A.L);  // tokens of the segment
  const long long t_hi = min(t_end, (long long)len);             // those that count
  const int n_all = t_hi > t_lo ? (int)(t_hi - t_lo) : 0;

  const float g = A.log_decay[h];
  const int lag = A.reverse ? 0 : 1;
  float a1, a1lo, achi, aclo;
  two_floats(exp((double)g), &a1, &a1lo);
  two_floats(exp((double)g * kTok), &achi, &aclo);

  // rows row0 + 2 p, row0 + 2 p + 1 of column col + c; D: the same of T
  float2 S[RH / 2][4], D[LEARN ? RH / 2 : 1][4];
  const long long per_state = (long long)A.DK * A.DV;
  const T* qp = static_cast<const T*>(A.q.p) + b * A.q.sb + (long long)(h / A.q.group) * A.q.sh;
  const T* kp = static_cast<const T*>(A.k.p) + b * A.k.sb + (long long)(h / A.k.group) * A.k.sh;
  const T* vp = static_cast<const T*>(A.v.p) + b * A.v.sb + (long long)(h / A.v.group) * A.v.sh;
  const T* xp = LEARN ? static_cast<const T*>(A.x.p) + b * A.x.sb + (long long)(h / A.x.group) * A.x.sh : nullptr;
  TO* op = static_cast<TO*>(A.o) + (A.o ? b * A.ob + (long long)h * A.oh + c0 : 0);
  const int step = A.reverse ? -1 : 1;
  float dg;

  // A chunk's tiles: q [kTok][W], k [kTok][W], v [kTok][kCols], x [kTok][kCols].
  const auto fetch = [&](int i0) {
    const int n = min(kTok, n_all - i0);
    const long long t0 = A.reverse ? t_hi - 1 - i0 : t_lo + i0;
    T* raw = reinterpret_cast<T*>(smem + M::raw) + (i0 / kTok & 1) * M::chunk;
    if (A.o) fetch_tile<T, W>(raw, qp, A.q.sl, n, 0, A.DK, t0, step);
    fetch_tile<T, W>(raw + kTok * W, kp, A.k.sl, n, 0, A.DK, t0, step);
    fetch_tile<T, kCols>(raw + 2 * kTok * W, vp, A.v.sl, n, c0, A.DV, t0, step);
    if (LEARN && A.o) fetch_tile<T, kCols>(raw + 2 * kTok * W + kTok * kCols, xp, A.x.sl, n, c0, A.DV, t0, step);
  };
  // whether a result was infinite or NaN
  const auto run = [&](auto divided) {
    constexpr bool fast = divided;
    float2 odd = dup(0.f);  // NaN once a result was infinite or NaN
    dg = 0.f;
    if (threadIdx.x < kTok) {
      const int e = threadIdx.x + lag;
      apow[threadIdx.x] = fast ? (float)(e ? exp((double)g * e) : 1.0) : 1.f;
      ainv[threadIdx.x] = (fast ? (float)(e ? exp(-(double)g * e) : 1.0) : 1.f) * A.vscale;
    }
#pragma unroll
    for (int p = 0; p < RH / 2; ++p)
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        S[p][c] = dup(0.f);
        if (LEARN) D[LEARN ? p : 0][c] = dup(0.f);
      }
    if (A.o) {
      const float* src = nullptr;
      long long sr = A.DV, sc = 1;
      if (A.nseg > 1) {
        src = A.seg + (bh * A.nseg + seg) * per_state;
        sr = A.segrow, sc = A.segcol;
      } else if (A.start) {
        src = A.start + bh * per_state;
        sr = A.srow, sc = A.scol;
      }
      const float* srcT = LEARN && A.nseg > 1 ? A.segT + (bh * A.nseg + seg) * per_state : nullptr;
#pragma unroll
      for (int r = 0; r < RH; ++r)
#pragma unroll
        for (int c = 0; c < 4; ++c)
          if (row0 + r < A.DK && c < left) {
            if (src) (&S[r >> 1][c].x)[r & 1] = src[(row0 + r) * sr + (c0 + col + c) * sc];
            if (LEARN && srcT) (&D[LEARN ? r >> 1 : 0][c].x)[r & 1] = srcT[(long long)(row0 + r) * A.DV + c0 + col + c];
          }
    }

    if (A.vec) {
      if (n_all > 0) fetch(0);
      asm volatile("cp.async.commit_group;\n" ::: "memory");
    }
    for (int i0 = 0; i0 < n_all; i0 += kTok) {
      const int n = min(kTok, n_all - i0);
      const long long t0 = A.reverse ? t_hi - 1 - i0 : t_lo + i0;
      float* tile = smem + (M::wide ? (i0 / kTok & 1) * M::chunk : 0);
      __syncthreads();  // the last chunk has been read
      if (A.vec) {
        if (i0 + kTok < n_all) fetch(i0 + kTok);
        asm volatile("cp.async.commit_group;\ncp.async.wait_group 1;\n" ::: "memory");
        if constexpr (!M::wide) {
          __syncthreads();
          const T* raw = reinterpret_cast<const T*>(smem + M::raw) + (i0 / kTok & 1) * M::chunk;
          if (A.o) widen_tile<T, W>(tile, raw, n);
          widen_tile<T, W>(tile + kTok * W, raw + kTok * W, n);
          widen_tile<T, kCols>(tile + 2 * kTok * W, raw + 2 * kTok * W, n);
          if (LEARN && A.o) widen_tile<T, kCols>(tile + 2 * kTok * W + kTok * kCols, raw + 2 * kTok * W + kTok * kCols, n);
        }
      } else {
        if (A.o) load_tile<T, W>(tile, qp, A.q.sl, n, 0, A.DK, t0, step);
        load_tile<T, W>(tile + kTok * W, kp, A.k.sl, n, 0, A.DK, t0, step);
        load_tile<T, kCols>(tile + 2 * kTok * W, vp, A.v.sl, n, c0, A.DV, t0, step);
        if (LEARN && A.o) load_tile<T, kCols>(tile + 2 * kTok * W + kTok * kCols, xp, A.x.sl, n, c0, A.DV, t0, step);
      }
      __syncthreads();
      const float *qs = tile, *ks = tile + kTok * W, *vs = ks + kTok * W, *xs = vs + kTok * kCols;
      for (int i = 0; i < n; ++i) {
        const float4 v4 = *reinterpret_cast<const float4*>(vs + i * kCols + col);
        const float ai = ainv[i];
        const float2 vj[4] = {dup(v4.x * ai), dup(v4.y * ai), dup(v4.z * ai), dup(v4.w * ai)};
        const float4* k4 = reinterpret_cast<const float4*>(ks + i * W + row0);
        const float4* q4 = reinterpret_cast<const float4*>(qs + i * W + row0);
        if (!fast && lag) {
#pragma unroll
          for (int p = 0; p < RH / 2; ++p)
#pragma unroll
            for (int c = 0; c < 4; ++c) {
              if (LEARN) {
                const float2 x = cadd(D[LEARN ? p : 0][c], S[p][c]);
                D[LEARN ? p : 0][c] = ffma2(x, dup(a1), mul2(x, a1lo));
              }
              S[p][c] = ffma2(S[p][c], dup(a1), mul2(S[p][c], a1lo));
            }
        }
        float2 acc[4] = {dup(0.f), dup(0.f), dup(0.f), dup(0.f)};  // of o, or of q T
#pragma unroll
        for (int r = 0; r < RH / 4; ++r) {
          const float4 kk = k4[r];
          const float2 ka = make_float2(kk.x, kk.y), kb = make_float2(kk.z, kk.w);
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            if (LEARN && fast) {
              D[LEARN ? 2 * r : 0][c] = cadd(D[LEARN ? 2 * r : 0][c], S[2 * r][c]);
              D[LEARN ? 2 * r + 1 : 0][c] = cadd(D[LEARN ? 2 * r + 1 : 0][c], S[2 * r + 1][c]);
            }
            S[2 * r][c] = ffma2(ka, vj[c], S[2 * r][c]);
            S[2 * r + 1][c] = ffma2(kb, vj[c], S[2 * r + 1][c]);
          }
          if constexpr (!fast) {  // rows past the head's size stay zero, where zero times an infinity does not
            const int rows = A.DK - row0 - 4 * r;
            if (rows < 4) {
#pragma unroll
              for (int c = 0; c < 4; ++c) {
                if (rows < 1) S[2 * r][c].x = 0.f;
                if (rows < 2) S[2 * r][c].y = 0.f;
                if (rows < 3) S[2 * r + 1][c].x = 0.f;
                S[2 * r + 1][c].y = 0.f;
              }
            }
          }
          if (A.o) {
            const float4 qq = q4[r];
            const float2 qa = make_float2(qq.x, qq.y), qb = make_float2(qq.z, qq.w);
#pragma unroll
            for (int c = 0; c < 4; ++c) {
              acc[c] = ffma2(qa, LEARN ? D[LEARN ? 2 * r : 0][c] : S[2 * r][c], acc[c]);
              acc[c] = ffma2(qb, LEARN ? D[LEARN ? 2 * r + 1 : 0][c] : S[2 * r + 1][c], acc[c]);
            }
          }
        }
        if (A.o) {
          if (LEARN) {
            const float4 x4 = *reinterpret_cast<const float4*>(xs + i * kCols + col);
            float s = (acc[0].x + acc[0].y) * x4.x;
            s = fmaf(acc[1].x + acc[1].y, x4.y, s);
            s = fmaf(acc[2].x + acc[2].y, x4.z, s);
            s = fmaf(acc[3].x + acc[3].y, x4.w, s);
            dg = fmaf(s, apow[i], dg);
          } else {
            const float as = apow[i] * A.oscale;
            float o[4];
#pragma unroll
            for (int c = 0; c < 4; ++c) {
              o[c] = acc[c].x + acc[c].y;
              o[c] = (o[c] + __shfl_xor_sync(0xffffffffu, o[c], 16)) * as;
            }
            if (fast) {
              odd = ffma2(make_float2(o[0], o[1]), dup(0.f), odd);
              odd = ffma2(make_float2(o[2], o[3]), dup(0.f), odd);
            }
            if (lane < 16) {
              if (KW > 1) {
                *reinterpret_cast<float4*>(os + (warp * kTok + i) * kCols + col) = make_float4(o[0], o[1], o[2], o[3]);
              } else {
                TO* d = op + (t0 + (long long)i * step) * A.ol + col;
                if (sizeof(TO) == 4 && A.ovec && left > 0) {
                  *reinterpret_cast<float4*>(d) = make_float4(o[0], o[1], o[2], o[3]);
                } else {
#pragma unroll
                  for (int c = 0; c < 4; ++c)
                    if (c < left) DT<TO>::store(d + c, o[c]);
                }
              }
            }
          }
        }
        if (!fast && !lag) {
#pragma unroll
          for (int p = 0; p < RH / 2; ++p)
#pragma unroll
            for (int c = 0; c < 4; ++c) S[p][c] = ffma2(S[p][c], dup(a1), mul2(S[p][c], a1lo));
        }
      }
      if (fast) {
        float hi = achi, lo = aclo;
        if (n != kTok) {
          two_floats(exp((double)g * n), &hi, &lo);
        }
#pragma unroll
        for (int p = 0; p < RH / 2; ++p)
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            S[p][c] = ffma2(S[p][c], dup(hi), mul2(S[p][c], lo));
            if (LEARN) D[LEARN ? p : 0][c] = ffma2(D[LEARN ? p : 0][c], dup(hi), mul2(D[LEARN ? p : 0][c], lo));
          }
      }
      if (KW > 1 && A.o && !LEARN) {
        __syncthreads();
        for (int i = threadIdx.x; i < n * kCols; i += 32 * KW) {
          const int r = i / kCols, c = i - r * kCols;
          if (c0 + c < A.DV) {
            float o = 0.f;
#pragma unroll
            for (int j = 0; j < KW; ++j) o += os[j * kTok * kCols + i];
            DT<TO>::store(op + (t0 + (long long)r * step) * A.ol + c, o);
          }
        }
      }
    }

    if constexpr (fast) {
#pragma unroll
      for (int p = 0; p < RH / 2; ++p)
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          odd = ffma2(S[p][c], dup(0.f), odd);
          if (LEARN) odd = ffma2(D[LEARN ? p : 0][c], dup(0.f), odd);
        }
      if (LEARN) odd.x = fmaf(dg, 0.f, odd.x);
    }
    return __syncthreads_or(odd.x != 0.f || odd.y != 0.f) != 0;
  };
  const bool fast = !(fabs((double)g) * kTok > kFastLimit);
  if (!fast || run(std::true_type{})) run(std::false_type{});

  if (A.o && !LEARN) {  // tokens past the length: zeros
    const long long z0 = max(t_lo, t_hi);
    for (long long i = threadIdx.x; i < (t_end - z0) * kCols; i += 32 * KW) {
      const long long r = i / kCols;
      const int c = (int)(i - r * kCols);
      if (c0 + c < A.DV) DT<TO>::store(op + (z0 + r) * A.ol + c, 0.f);
    }
  }
  float* dst = nullptr;
  long long sr = A.DV, sc = 1;
  if (!A.o) {
    dst = A.seg + (bh * A.nseg + seg) * per_state;
  } else if (A.nseg == 1 && A.finish) {
    dst = A.finish + bh * per_state;
    sr = A.srow, sc = A.scol;
  }
  float* dT = LEARN && (!A.o || A.nseg == 1) ? A.segT + (bh * A.nseg + seg) * per_state : nullptr;
#pragma unroll
  for (int r = 0; r < RH; ++r)
#pragma unroll
    for (int c = 0; c < 4; ++c)
      if (row0 + r < A.DK && c < left) {
        if (dst) dst[(row0 + r) * sr + (c0 + col + c) * sc] = (&S[r >> 1][c].x)[r & 1];
        if (LEARN && dT) dT[(long long)(row0 + r) * A.DV + c0 + col + c] = (&D[LEARN ? r >> 1 : 0][c].x)[r & 1];
      }
  if (LEARN && A.o) A.dg[((bh * A.nseg + seg) * A.nslice + slice) * (32 * KW) + threadIdx.x] = dg * A.oscale;
}

// Chains the segments: seg[s] becomes the state before segment s (in scan order), finish the state after the last.
// T_out = a^n T_in + n a^n S_in + T_segment. 
constexpr int kChainLoads = 8;
__global__ void __launch_bounds__(256) decay_chain_kernel(float* seg, float* segT, float* finalT, const float* start,
                                                          float* finish, const float* log_decay, const int* lengths,
                                                          int H, int L, int DK, int DV, int srow, int scol, int nseg,
                                                          int seglen, int reverse) {
  const long long bh = blockIdx.y;
  const int e = blockIdx.x * 256 + threadIdx.x;
  if (e >= DK * DV) return;
  const int r = e / DV, c = e - r * DV;
  const long long per = (long long)DK * DV;
  const float g = log_decay[bh % H];
  int len = L;
  if (lengths) len = min(max(lengths[bh / H], 0), L);
  // a power that is too small even for a double is not zero all the same: an infinite state stays infinite
  const double least = g > -INFINITY ? 1e-300 : 0.0;
  const double af = fmax(exp((double)g * seglen), least);
  float s = start ? start[bh * per + (long long)r * srow + (long long)c * scol] : 0.f, t = 0.f;
  for (int i0 = 0; i0 < nseg; i0 += kChainLoads) {  // loads of several segments in flight
    float add[kChainLoads], addT[kChainLoads];
    const int m = min(kChainLoads, nseg - i0);
#pragma unroll
    for (int i = 0; i < kChainLoads; ++i)
      if (i < m) {
        const long long at = (bh * nseg + (reverse ? nseg - 1 - i0 - i : i0 + i)) * per + e;
        add[i] = seg[at];
        if (segT) addT[i] = segT[at];
      }
#pragma unroll
    for (int i = 0; i < kChainLoads; ++i)
      if (i < m) {
        const int j = reverse ? nseg - 1 - i0 - i : i0 + i;
        const long long at = (bh * nseg + j) * per + e, lo = (long long)j * seglen;
        const long long n = max(0ll, min(lo + seglen, (long long)len) - lo);
        const double an = n == seglen ? af : n ? fmax(exp((double)g * (double)n), least) : 1.0;
        seg[at] = s;
        if (segT) {
          segT[at] = t;
          t = (float)(an * ((double)t + (double)n * (double)s) + (double)addT[i]);
        }
        s = (float)(an * (double)s + (double)add[i]);
      }
  }
  if (finish) finish[bh * per + (long long)r * srow + (long long)c * scol] = s;
  if (finalT) finalT[bh * per + e] = t;
}

// dlog_decay[h] = sum over rows of head h of the partial sums, plus <dfinal, T_final>; one CTA per head, in a fixed order.
__global__ void __launch_bounds__(256) decay_dg_kernel(const float* part, long long per, const float* finalT,
                                                       const float* dfinal, long long state, int B, int H, float* out) {
  const int h = blockIdx.x;
  double s = 0.0;
  for (int b = 0; b < B; ++b) {
    const long long bh = (long long)b * H + h;
    for (long long i = threadIdx.x; i < per; i += 256) s += (double)part[bh * per + i];
    if (dfinal)
      for (long long i = threadIdx.x; i < state; i += 256) s += (double)finalT[bh * state + i] * (double)dfinal[bh * state + i];
  }
  __shared__ double red[256];
  red[threadIdx.x] = s;
  __syncthreads();
  for (int w = 128; w > 0; w >>= 1) {
    if (threadIdx.x < w) red[threadIdx.x] += red[threadIdx.x + w];
    __syncthreads();
  }
  if (threadIdx.x == 0) out[h] = (float)red[0];
}

// Gradients of a shared head: the sum over its query heads, src [B * L, H, D] float32 -> dst [B * L, Hk, D].
template <typename T>
__global__ void __launch_bounds__(256) decay_group_sum_kernel(const float* src, T* dst, long long n, int D, int group) {
  const long long i = (long long)blockIdx.x * 256 + threadIdx.x;
  if (i >= n) return;
  const long long hk = i / D;
  const int d = (int)(i - hk * D);
  float s = 0.f;
  for (int j = 0; j < group; ++j) s += src[(hk * group + j) * D + d];
  DT<T>::store(dst + i, s);
}

// ---------------------------------------------------------------- single tokens
// One token of each request: a pass over the state, read and written once (8 bytes per element, nothing else of
// size). A CTA takes one head's state (a slice of 32 columns when there are few heads, so that all SMs have work);
// a thread reads four neighbouring columns of every (kStepThreads / columns * 4)-th row. 172 requests of 32 heads of
// 128 x 128: 133 us, 5.5 TB/s (84% of a copy's rate); one request of 12 heads of 64 x 64: 3 us.
constexpr int kStepThreads = 256;

struct StepArgs {
  Op q, k, v;
  void* o;
  long long ob, oh;
  const float* log_decay;
  const int* slots;
  const float* state;
  float* out_state;
  float scale;
  long long pool;
  int H, DK, DV, cols, nslice;
};

template <typename T, int V>
__global__ void __launch_bounds__(kStepThreads) decay_step_kernel(const StepArgs A) {
  extern __shared__ float sm[];
  float* qs = sm;             // [DK]
  float* ks = qs + A.DK;      // [DK]
  float* red = ks + A.DK;     // [rows][cols]
  const int slice = blockIdx.x % A.nslice;
  const long long bh = blockIdx.x / A.nslice;
  const int h = (int)(bh % A.H);
  const long long b = bh / A.H;
  const int c0 = slice * A.cols;
  const int ncol = min(A.cols, A.DV - c0);
  T* o = static_cast<T*>(A.o) + b * A.ob + (long long)h * A.oh + c0;
  const long long slot = A.slots ? (long long)A.slots[b] : b;
  if (slot < 0 || slot >= A.pool) {  // an idle request
    for (int c = threadIdx.x; c < ncol; c += kStepThreads) DT<T>::store(o + c, 0.f);
    return;
  }
  const T* qp = static_cast<const T*>(A.q.p) + b * A.q.sb + (long long)h * A.q.sh;
  const T* kp = static_cast<const T*>(A.k.p) + b * A.k.sb + (long long)(h / A.k.group) * A.k.sh;
  const T* vp = static_cast<const T*>(A.v.p) + b * A.v.sb + (long long)(h / A.v.group) * A.v.sh + c0;
  for (int i = threadIdx.x; i < A.DK; i += kStepThreads) {
    qs[i] = DT<T>::load(qp + i) * A.scale;
    ks[i] = DT<T>::load(kp + i);
  }
  const float a = expf(A.log_decay[h]);
  __syncthreads();
  const int per = A.cols / V, rows = kStepThreads / per;
  const int c = (threadIdx.x % per) * V, r0 = threadIdx.x / per;
  const long long base = (slot * A.H + h) * (long long)A.DK * A.DV + c0 + c;
  float acc[V], vv[V];
#pragma unroll
  for (int u = 0; u < V; ++u) acc[u] = 0.f, vv[u] = 0.f;
  if (r0 < rows && c < ncol) {
#pragma unroll
    for (int u = 0; u < V; ++u) vv[u] = DT<T>::load(vp + c + u);
#pragma unroll 4
    for (int r = r0; r < A.DK; r += rows) {
      const float* src = A.state + base + (long long)r * A.DV;
      float s[V];
      if (V == 4) {
        const float4 x = *reinterpret_cast<const float4*>(src);
        s[0] = x.x, s[V > 1 ? 1 : 0] = x.y, s[V > 2 ? 2 : 0] = x.z, s[V > 3 ? 3 : 0] = x.w;
      } else {
        s[0] = src[0];
      }
      const float kk = ks[r], qq = qs[r];
#pragma unroll
      for (int u = 0; u < V; ++u) {
        s[u] = fmaf(a, s[u], kk * vv[u]);
        acc[u] = fmaf(qq, s[u], acc[u]);
      }
      float* dst = A.out_state + base + (long long)r * A.DV;
      if (V == 4)
        *reinterpret_cast<float4*>(dst) = make_float4(s[0], s[V > 1 ? 1 : 0], s[V > 2 ? 2 : 0], s[V > 3 ? 3 : 0]);
      else
        dst[0] = s[0];
    }
  }
  if (r0 < rows)
#pragma unroll
    for (int u = 0; u < V; ++u) red[r0 * A.cols + c + u] = acc[u];
  __syncthreads();
  for (int i = threadIdx.x; i < ncol; i += kStepThreads) {
    float s = 0.f;
    for (int r = 0; r < rows; ++r) s += red[r * A.cols + i];
    DT<T>::store(o + i, s);
  }
}

// ---------------------------------------------------------------- host

int launched() {
  if (cudaGetLastError() != cudaSuccess) return set_error(HYFFT_ERR_CUDA, "decay attention: kernel launch failed");
  g_launches.fetch_add(1, std::memory_order_relaxed);
  return HYFFT_OK;
}

// Rows of the state that a thread holds, and warps over them, for a state of DK rows.
void scan_shape(int DK, int* rh, int* kw) {
  *kw = 1;
  while (*kw * 32 < DK) *kw *= 2;
  *rh = DK <= 16 ? 8 : 16;
}

// The tensor cores take every bfloat16 scan whose state has up to 128 rows, and float16 and float32 ones (as sums of
// bfloat16 terms) from half a chunk of tokens on: below, the scan's time is latency either way and laying out the terms is one
// launch more (12 heads of 64, float32, multiply-adds: 11 us for 16 tokens, 28 for 64; tensor cores: 10 for 64). All
// scans of a call go one way.
bool use_mma(const hyfft_decay_desc* d, int DK) {
  if (d->dtype == HYFFT_BF16) return DK <= kMmaMaxDK;
  return std::max(d->dk, d->dv) <= kMmaMaxDK && d->length >= kMmaTok / 2;
}
// bfloat16 terms of an operand, 0: none are laid out. bfloat16 heads of a size that 16-byte copies cannot take are laid out
// as one term (8 x 4096 tokens, 8 heads of 65, forward and backward: 0.94 ms; element by element in the scan itself 4.14).
int terms(const hyfft_decay_desc* d) {
  if (d->dtype != HYFFT_BF16) return !use_mma(d, d->dk) ? 0 : d->dtype == HYFFT_F16 ? 2 : 3;
  return (d->dk % 8 || d->dv % 8) && std::max(d->dk, d->dv) <= kMmaMaxDK && d->length >= kMmaTok / 2 ? 1 : 0;
}

int slices(int DV) { return (DV + kCols - 1) / kCols; }  // 64 columns a CTA on either path
static_assert(kCols == kMmaCols && kMmaTok % kTok == 0, "one plan for both paths");

struct Segments {
  int n, len;
};

// All scans of a call cut the axis at the same places, so that one pass over the segments serves several. Tensor
// cores: as many CTAs as fit; rows alone where they give every SM one (200 rows of 4096 tokens of 64: 155 us forwards, as two
// segments each 204; of 1024 tokens 46 and 79; 150 rows of 4096 153 and 199) or are shorter than eight chunks, else as many segments
// as there is room for, none shorter than two chunks (1024 tokens, 12 heads of 64, forward and backward: segments of four chunks
// or more 63 us, of two 52, of one 59; 256 tokens: one segment 42 us, two 48). Else: twelve warps for each SM, segments of
// one chunk at least.
Segments segments(const hyfft_decay_desc* d, bool learn) {
  const long long rows = (long long)d->batch * d->heads;
  long long want, most;
  if (!learn && use_mma(d, d->dk) && use_mma(d, d->dv)) {
    const long long ctas = rows * std::max(slices(d->dk), slices(d->dv));
    // two CTAs share an SM but where the terms of float32, or of heads above 64, fill it
    const int fit = terms(d) == 3 || (terms(d) == 2 && std::max(d->dk, d->dv) > 64) ? 148 : 296;
    want = ctas >= 148 ? 1 : fit / ctas;
    most = d->length >= 8 * kMmaTok ? d->length / (2 * kMmaTok) : 1;
  } else {
    int rh, kw, rh2, kw2;
    scan_shape(d->dk, &rh, &kw);
    scan_shape(d->dv, &rh2, &kw2);
    const long long warps = rows * (learn ? slices(d->dv) * kw : std::max(slices(d->dv) * kw, slices(d->dk) * kw2));
    want = (12 * 148 + warps - 1) / warps;
    most = (d->length + kMmaTok - 1) / kMmaTok;
  }
  const long long n = std::max<long long>(1, std::min(want, most));
  const long long len = std::max<long long>(kMmaTok, ((d->length + n - 1) / n + kMmaTok - 1) / kMmaTok * kMmaTok);
  Segments g;
  g.len = (int)std::min<long long>(len, 1ll << 30);
  g.n = (int)std::max<long long>(1, (d->length + g.len - 1) / g.len);
  return g;
}

template <typename T, typename TO, int RH, int KW, bool LEARN>
int launch_scan_rh(const ScanArgs& A, long long ctas, cudaStream_t st) {
  const size_t sm = sizeof(float) * Smem<T, RH, KW, LEARN>::floats;
  auto kern = decay_scan_kernel<T, TO, RH, KW, LEARN>;
  if (!kernel_smem_once((const void*)kern, sm, true)) return set_error(HYFFT_ERR_CUDA, "decay attention: shared memory");
  kern<<<(unsigned)ctas, 32 * KW, sm, st>>>(A);
  return launched();
}

template <typename T, typename TO, bool LEARN>
int launch_scan(const ScanArgs& A, int rh, int kw, long long ctas, cudaStream_t st) {
  if (ctas > 0x7fffffffLL) return set_error(HYFFT_ERR_UNSUPPORTED, "decay attention: too many rows");
  if constexpr (LEARN || !std::is_same<T, __nv_bfloat16>::value) {  // bfloat16 states of up to 128 rows run on the tensor cores
    if (rh == 8) return launch_scan_rh<T, TO, 8, 1, LEARN>(A, ctas, st);
    if (kw == 1) return launch_scan_rh<T, TO, 16, 1, LEARN>(A, ctas, st);
    if (kw == 2) return launch_scan_rh<T, TO, 16, 2, LEARN>(A, ctas, st);
    if (kw == 4) return launch_scan_rh<T, TO, 16, 4, LEARN>(A, ctas, st);
  }
  return launch_scan_rh<T, TO, 16, 8, LEARN>(A, ctas, st);
}

bool op_vec(const Op& o, int D, int es) {
  const int v = 16 / es;
  return D % v == 0 && reinterpret_cast<uintptr_t>(o.p) % 16 == 0 && o.sb % v == 0 && o.sl % v == 0 && o.sh % v == 0;
}

size_t align256(size_t n) { return (n + 255) / 256 * 256; }

// Bytes of the segments' states; 0 where the axis is not cut.
size_t seg_bytes(const hyfft_decay_desc* d) {
  const Segments g = segments(d, false);
  return g.n > 1 ? align256(sizeof(float) * (size_t)d->batch * d->heads * g.n * d->dk * d->dv) : 0;
}

void set_segments(const hyfft_decay_desc* d, ScanArgs& A, bool learn) {
  const Segments g = segments(d, learn);
  A.B = d->batch;
  A.H = d->heads;
  A.L = (int)d->length;
  A.nseg = g.n;
  A.seglen = g.len;
  A.nslice = slices(A.DV);
}

template <typename T, typename TO>
int run_pass(const hyfft_decay_desc* d, ScanArgs A, cudaStream_t st) {
  const int es = (int)sizeof(T);
  A.vec = (!A.o || op_vec(A.q, A.DK, es)) && op_vec(A.k, A.DK, es) && op_vec(A.v, A.DV, es);
  A.ovec = A.DV % 8 == 0 && reinterpret_cast<uintptr_t>(A.o) % 16 == 0;
  const long long ctas = (long long)d->batch * d->heads * A.nseg * A.nslice;
  if (use_mma(d, A.DK)) {
    if (terms(d)) A.vec = 1;  // laid out so
    return launch_scan_mma(A, d->dtype, sizeof(TO) == 4, ctas, st);
  }
  int rh, kw;
  scan_shape(A.DK, &rh, &kw);
  return launch_scan<T, TO, false>(A, rh, kw, ctas, st);
}

// The segments' start states, [B * H, nseg, dk, dv], and the state after the last one; nothing where the axis is not cut.
template <typename T>
int run_states(const hyfft_decay_desc* d, ScanArgs A, float* seg, cudaStream_t st) {
  set_segments(d, A, false);
  if (A.nseg == 1) return HYFFT_OK;
  A.o = nullptr;
  A.seg = seg;
  const long long rows = (long long)d->batch * d->heads;
  if (rows > 65535) return set_error(HYFFT_ERR_UNSUPPORTED, "decay attention: too many rows");
  const int rc = run_pass<T, T>(d, A, st);
  if (rc != HYFFT_OK) return rc;
  decay_chain_kernel<<<dim3((A.DK * A.DV + 255) / 256, (unsigned)rows), 256, 0, st>>>(
      seg, nullptr, nullptr, A.start, A.finish, A.log_decay, A.lengths, A.H, A.L, A.DK, A.DV, A.srow, A.scol, A.nseg,
      A.seglen, A.reverse);
  return launched();
}

// The outputs, from segment states of either orientation (`turned`: the states' rows are this scan's columns).
template <typename T, typename TO>
int run_outputs(const hyfft_decay_desc* d, ScanArgs A, const float* seg, bool turned, cudaStream_t st) {
  set_segments(d, A, false);
  A.seg = const_cast<float*>(seg);
  A.segrow = turned ? 1 : A.DV;
  A.segcol = turned ? A.DK : 1;
  return run_pass<T, TO>(d, A, st);
}

// The decay's gradient: the forward scan once more with T beside S.
template <typename T>
int run_learn(const hyfft_decay_desc* d, ScanArgs A, const float* dfinal, float* ws, float* out, cudaStream_t st) {
  set_segments(d, A, true);
  int rh, kw;
  scan_shape(A.DK, &rh, &kw);
  A.segrow = A.DV, A.segcol = 1;
  const int es = (int)sizeof(T);
  A.vec = op_vec(A.q, A.DK, es) && op_vec(A.k, A.DK, es) && op_vec(A.v, A.DV, es) && op_vec(A.x, A.DV, es);
  const long long rows = (long long)d->batch * d->heads;
  const size_t states = (size_t)rows * A.nseg * d->dk * d->dv;
  float* finalT = ws;
  A.seg = ws + (size_t)rows * d->dk * d->dv;
  A.segT = A.nseg > 1 ? A.seg + states : finalT;
  A.dg = A.seg + (A.nseg > 1 ? 2 * states : 0);
  A.finish = nullptr;
  const long long ctas = rows * A.nseg * A.nslice;
  if (A.nseg > 1) {
    ScanArgs P = A;
    P.o = nullptr;
    int rc = launch_scan<T, T, true>(P, rh, kw, ctas, st);
    if (rc != HYFFT_OK) return rc;
    if (rows > 65535) return set_error(HYFFT_ERR_UNSUPPORTED, "decay attention: too many rows");
    decay_chain_kernel<<<dim3((A.DK * A.DV + 255) / 256, (unsigned)rows), 256, 0, st>>>(
        A.seg, A.segT, finalT, A.start, nullptr, A.log_decay, A.lengths, A.H, A.L, A.DK, A.DV, A.srow, A.scol, A.nseg,
        A.seglen, 0);
    if ((rc = launched()) != HYFFT_OK) return rc;
  }
  A.o = ws;  // not written by this scan: only says that it is the second pass
  int rc = launch_scan<T, T, true>(A, rh, kw, ctas, st);
  if (rc != HYFFT_OK) return rc;
  decay_dg_kernel<<<d->heads, 256, 0, st>>>(A.dg, (long long)A.nseg * A.nslice * 32 * kw, finalT, dfinal,
                                            (long long)d->dk * d->dv, d->batch, d->heads, out);
  return launched();
}

size_t learn_bytes(const hyfft_decay_desc* d) {
  const Segments g = segments(d, true);
  int rh, kw;
  scan_shape(d->dk, &rh, &kw);
  const size_t rows = (size_t)d->batch * d->heads, per = (size_t)d->dk * d->dv;
  return align256(sizeof(float) * (rows * per * (1 + (g.n > 1 ? 2 * (size_t)g.n : 0)) + rows * g.n * slices(d->dv) * 32 * kw));
}

int check_desc(const hyfft_decay_desc* d) {
  if (!d) return set_error(HYFFT_ERR_INVALID, "decay attention: null descriptor");
  if (d->batch < 1 || d->length < 0 || d->heads < 1 || d->kv_heads < 1 || d->dk < 1 || d->dv < 1)
    return set_error(HYFFT_ERR_INVALID, "decay attention: every extent must be positive");
  if (d->heads % d->kv_heads) return set_error(HYFFT_ERR_INVALID, "decay attention: kv_heads must divide heads");
  if (d->dtype < HYFFT_F32 || d->dtype > HYFFT_F16) return set_error(HYFFT_ERR_INVALID, "decay attention: bad dtype");
  if (d->dk > kMaxDim || d->dv > kMaxDim)
    return set_error(HYFFT_ERR_UNSUPPORTED, "decay attention: head sizes above 256 are not covered");
  if (d->length > 0x7fffffffLL - 4096) return set_error(HYFFT_ERR_UNSUPPORTED, "decay attention: sequence too long");
  return HYFFT_OK;
}

struct Rows {  // strides of a contiguous [B, L, heads, D]
  long long b, l, h;
};
Rows dense(const hyfft_decay_desc* d, int heads, int D) {
  return {(long long)d->length * heads * D, (long long)heads * D, (long long)D};
}

template <typename T>
int forward_t(const hyfft_decay_desc* d, const void* q, const void* k, const void* v, const float* g, const int* lengths,
              const float* s0, void* o, float* s1, float* ws, cudaStream_t st) {
  const int r = d->heads / d->kv_heads;
  const Rows ro = dense(d, d->heads, d->dv);
  ScanArgs A{};
  A.q = {q, d->q_stride[0], d->q_stride[1], d->q_stride[2], 1};
  A.k = {k, d->k_stride[0], d->k_stride[1], d->k_stride[2], r};
  A.v = {v, d->v_stride[0], d->v_stride[1], d->v_stride[2], r};
  A.o = o, A.ob = ro.b, A.ol = ro.l, A.oh = ro.h;
  A.log_decay = g, A.lengths = lengths, A.start = s0, A.finish = s1;
  A.vscale = 1.f, A.oscale = d->scale;
  A.DK = d->dk, A.DV = d->dv, A.srow = d->dv, A.scol = 1;
  int rc = HYFFT_OK;
  if (terms(d)) {
    ScanOp ops[3] = {A.q, A.k, A.v};
    const int heads[3] = {d->heads, d->kv_heads, d->kv_heads}, D[3] = {d->dk, d->dk, d->dv};
    rc = launch_split_terms(ops, heads, D, 3, d->batch, d->length, d->dtype, terms(d),
                            reinterpret_cast<char*>(ws) + seg_bytes(d), st);
    A.q = ops[0], A.k = ops[1], A.v = ops[2];
  }
  if (rc == HYFFT_OK) rc = run_states<T>(d, A, ws, st);
  return rc == HYFFT_OK ? run_outputs<T, T>(d, A, ws, false, st) : rc;
}

// dk or dv: straight to the output where no head is shared, else in float32 per query head and summed.
template <typename T>
int shared_scan(const hyfft_decay_desc* d, ScanArgs A, void* out, int D, const float* seg, bool turned, float* per_head,
                cudaStream_t st) {
  if (d->heads == d->kv_heads) {
    const Rows ro = dense(d, d->heads, D);
    A.o = out, A.ob = ro.b, A.ol = ro.l, A.oh = ro.h;
    return run_outputs<T, T>(d, A, seg, turned, st);
  }
  const Rows ro = dense(d, d->heads, D);
  A.o = per_head, A.ob = ro.b, A.ol = ro.l, A.oh = ro.h;
  int rc = run_outputs<T, float>(d, A, seg, turned, st);
  if (rc != HYFFT_OK) return rc;
  const long long n = (long long)d->batch * d->length * d->kv_heads * D;
  if (n == 0) return HYFFT_OK;
  decay_group_sum_kernel<T><<<(unsigned)((n + 255) / 256), 256, 0, st>>>(per_head, static_cast<T*>(out), n, D,
                                                                         d->heads / d->kv_heads);
  return launched();
}

template <typename T>
int backward_t(const hyfft_decay_desc* d, const void* q, const void* k, const void* v, const float* g,
               const int* lengths, const float* s0, const float* saved, const void* dout, const float* ds1, void* dq,
               void* dk, void* dv,
               float* dg, float* ds0, char* ws, size_t seg_size, size_t group_size, cudaStream_t st) {
  const int r = d->heads / d->kv_heads;
  Op oq{q, d->q_stride[0], d->q_stride[1], d->q_stride[2], 1};
  Op ok{k, d->k_stride[0], d->k_stride[1], d->k_stride[2], r};
  Op ov{v, d->v_stride[0], d->v_stride[1], d->v_stride[2], r};
  Op od{dout, d->o_stride[0], d->o_stride[1], d->o_stride[2], 1};
  float* seg = reinterpret_cast<float*>(ws);
  float* per_head = reinterpret_cast<float*>(ws + seg_size);
  float* learn = reinterpret_cast<float*>(ws + seg_size + group_size);
  const Op plain[4] = {oq, ok, ov, od};
  ScanArgs A{};
  A.log_decay = g, A.lengths = lengths;
  int rc;
  if (terms(d) && (dq || dk || dv)) {
    Op ops[4] = {oq, ok, ov, od};
    const int heads[4] = {d->heads, d->kv_heads, d->kv_heads, d->heads}, D[4] = {d->dk, d->dk, d->dv, d->dv};
    if ((rc = launch_split_terms(ops, heads, D, 4, d->batch, d->length, d->dtype, terms(d),
                                 ws + seg_size + group_size + learn_bytes(d), st)) != HYFFT_OK)
      return rc;
    oq = ops[0], ok = ops[1], ov = ops[2], od = ops[3];
  }
  if (dq) {  // forwards over (do, v, k), the state transposed
    if (!saved) {
      ScanArgs P = A;
      P.k = ok, P.v = ov, P.start = s0, P.vscale = 1.f;
      P.DK = d->dk, P.DV = d->dv, P.srow = d->dv, P.scol = 1;
      if ((rc = run_states<T>(d, P, seg, st)) != HYFFT_OK) return rc;
      saved = seg;
    }
    ScanArgs P = A;
    const Rows ro = dense(d, d->heads, d->dk);
    P.q = od, P.k = ov, P.v = ok;
    P.o = dq, P.ob = ro.b, P.ol = ro.l, P.oh = ro.h;
    P.start = s0, P.vscale = 1.f, P.oscale = d->scale;
    P.DK = d->dv, P.DV = d->dk, P.srow = 1, P.scol = d->dv;
    if ((rc = run_outputs<T, T>(d, P, saved, true, st)) != HYFFT_OK) return rc;
  }
  ScanArgs G = A;  // backwards over (k, q, do): the state's gradient, in the state's own orientation
  G.q = ok, G.k = oq, G.v = od;
  G.start = ds1, G.finish = ds0, G.vscale = d->scale, G.oscale = 1.f, G.reverse = 1;
  G.DK = d->dk, G.DV = d->dv, G.srow = d->dv, G.scol = 1;
  if ((dk || dv) && (rc = run_states<T>(d, G, seg, st)) != HYFFT_OK) return rc;
  if (dk) {  // and over (v, do, q), transposed
    ScanArgs P = A;
    P.q = ov, P.k = od, P.v = oq;
    P.start = ds1, P.vscale = d->scale, P.oscale = 1.f, P.reverse = 1;
    P.DK = d->dv, P.DV = d->dk, P.srow = 1, P.scol = d->dv;
    if ((rc = shared_scan<T>(d, P, dk, d->dk, seg, true, per_head, st)) != HYFFT_OK) return rc;
  }
  if (dv && (rc = shared_scan<T>(d, G, dv, d->dv, seg, false, per_head, st)) != HYFFT_OK) return rc;
  if (dg) {
    ScanArgs P = A;
    P.q = plain[0], P.k = plain[1], P.v = plain[2], P.x = plain[3];
    P.start = s0, P.vscale = 1.f, P.oscale = d->scale;
    P.DK = d->dk, P.DV = d->dv, P.srow = d->dv, P.scol = 1;
    if ((rc = run_learn<T>(d, P, ds1, learn, dg, st)) != HYFFT_OK) return rc;
  }
  return HYFFT_OK;
}

struct Sizes {
  size_t seg, group, learn, terms3, terms4;  // the terms of q, k, v, and those with the output's gradient
};
Sizes sizes(const hyfft_decay_desc* d) {
  Sizes s;
  s.seg = seg_bytes(d);
  s.group = d->heads == d->kv_heads
                ? 0
                : align256(sizeof(float) * (size_t)d->batch * d->length * d->heads * std::max(d->dk, d->dv));
  s.learn = learn_bytes(d);
  s.terms3 = s.terms4 = 0;
  if (const int t = terms(d)) {
    s.terms3 = mma_terms_bytes(d->batch, d->length, d->heads, d->dk, t) +
               mma_terms_bytes(d->batch, d->length, d->kv_heads, d->dk, t) +
               mma_terms_bytes(d->batch, d->length, d->kv_heads, d->dv, t);
    s.terms4 = s.terms3 + mma_terms_bytes(d->batch, d->length, d->heads, d->dv, t);
  }
  return s;
}

}  // namespace
}  // namespace hyfft

using namespace hyfft;

extern "C" {

int hyfft_decay_workspace_size(const hyfft_decay_desc* d, size_t* fwd_bytes, size_t* bwd_bytes) {
  const int rc = check_desc(d);
  if (rc != HYFFT_OK) return rc;
  const Sizes s = sizes(d);
  if (fwd_bytes) *fwd_bytes = s.seg + s.terms3;
  if (bwd_bytes) *bwd_bytes = s.seg + s.group + s.learn + s.terms4;
  return HYFFT_OK;
}

int hyfft_decay_saved_size(const hyfft_decay_desc* d, size_t* saved_bytes) {
  const int rc = check_desc(d);
  if (rc != HYFFT_OK) return rc;
  if (!saved_bytes) return set_error(HYFFT_ERR_INVALID, "decay attention: null size");
  *saved_bytes = sizes(d).seg;
  return HYFFT_OK;
}

int hyfft_decay_forward(const hyfft_decay_desc* d, const void* q, const void* k, const void* v, const float* log_decay,
                        const int32_t* lengths, const float* initial_state, void* o, float* final_state,
                        void* workspace, size_t workspace_bytes, void* stream) {
  const int rc = check_desc(d);
  if (rc != HYFFT_OK) return rc;
  if (!log_decay || (d->length > 0 && (!q || !k || !v || !o)))
    return set_error(HYFFT_ERR_INVALID, "decay attention: null tensor");
  const Sizes s = sizes(d);
  if (workspace_bytes < s.seg + s.terms3 || (s.seg + s.terms3 && !workspace))
    return set_error(HYFFT_ERR_WORKSPACE, "decay attention: workspace too small");
  if (bind_device_of(log_decay) != HYFFT_OK) return set_error(HYFFT_ERR_CUDA, "decay attention: device");
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (d->length == 0 && !o) o = const_cast<float*>(log_decay);  // no token writes it
  float* ws = static_cast<float*>(workspace);
  if (d->dtype == HYFFT_F32) return forward_t<float>(d, q, k, v, log_decay, lengths, initial_state, o, final_state, ws, st);
  if (d->dtype == HYFFT_BF16)
    return forward_t<__nv_bfloat16>(d, q, k, v, log_decay, lengths, initial_state, o, final_state, ws, st);
  return forward_t<__half>(d, q, k, v, log_decay, lengths, initial_state, o, final_state, ws, st);
}

int hyfft_decay_backward(const hyfft_decay_desc* d, const void* q, const void* k, const void* v, const float* log_decay,
                         const int32_t* lengths, const float* initial_state, const void* saved, const void* dout,
                         const float* dfinal_state,
                         void* dq, void* dk, void* dv, float* dlog_decay, float* dinitial_state, void* workspace,
                         size_t workspace_bytes, void* stream) {
  const int rc = check_desc(d);
  if (rc != HYFFT_OK) return rc;
  if (!log_decay || (d->length > 0 && (!q || !k || !v || !dout)))
    return set_error(HYFFT_ERR_INVALID, "decay attention: null tensor in the backward");
  if (d->length > 0 && dinitial_state && !dv)
    return set_error(HYFFT_ERR_INVALID, "decay attention: the initial state's gradient comes with dv");
  const Sizes s = sizes(d);
  if (workspace_bytes < s.seg + s.group + s.learn + s.terms4 || !workspace)
    return set_error(HYFFT_ERR_WORKSPACE, "decay attention: workspace too small");
  if (bind_device_of(log_decay) != HYFFT_OK) return set_error(HYFFT_ERR_CUDA, "decay attention: device");
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  char* ws = static_cast<char*>(workspace);
  if (d->length == 0) dq = dk = dv = nullptr;
  if (d->length == 0 && dinitial_state) dv = ws;  // no token writes it
  if (d->dtype == HYFFT_F32)
    return backward_t<float>(d, q, k, v, log_decay, lengths, initial_state, static_cast<const float*>(saved), dout, dfinal_state, dq, dk, dv, dlog_decay,
                             dinitial_state, ws, s.seg, s.group, st);
  if (d->dtype == HYFFT_BF16)
    return backward_t<__nv_bfloat16>(d, q, k, v, log_decay, lengths, initial_state, static_cast<const float*>(saved), dout, dfinal_state, dq, dk, dv,
                                     dlog_decay, dinitial_state, ws, s.seg, s.group, st);
  return backward_t<__half>(d, q, k, v, log_decay, lengths, initial_state, static_cast<const float*>(saved), dout, dfinal_state, dq, dk, dv, dlog_decay,
                            dinitial_state, ws, s.seg, s.group, st);
}

int hyfft_decay_step(const hyfft_decay_desc* d, const void* q, const void* k, const void* v, const float* log_decay,
                     const int32_t* slots, int64_t pool, const float* state, float* out_state, void* o, void* stream) {
  const int rc = check_desc(d);
  if (rc != HYFFT_OK) return rc;
  if (!q || !k || !v || !log_decay || !state || !out_state || !o)
    return set_error(HYFFT_ERR_INVALID, "decay attention step: null tensor");
  if (bind_device_of(q) != HYFFT_OK) return set_error(HYFFT_ERR_CUDA, "decay attention step: device");
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const int r = d->heads / d->kv_heads;
  StepArgs A{};
  A.q = {q, d->q_stride[0], 0, d->q_stride[2], 1};
  A.k = {k, d->k_stride[0], 0, d->k_stride[2], r};
  A.v = {v, d->v_stride[0], 0, d->v_stride[2], r};
  A.o = o, A.ob = (long long)d->heads * d->dv, A.oh = d->dv;
  A.log_decay = log_decay, A.slots = slots, A.state = state, A.out_state = out_state, A.scale = d->scale;
  A.H = d->heads, A.DK = d->dk, A.DV = d->dv, A.pool = pool;
  const bool vec = d->dv % 4 == 0 && reinterpret_cast<uintptr_t>(state) % 16 == 0 &&
                   reinterpret_cast<uintptr_t>(out_state) % 16 == 0;
  const long long rows = (long long)d->batch * d->heads;
  // all columns in one CTA when the heads fill the machine, slices of 32 otherwise
  const int whole = vec ? (d->dv + 3) / 4 * 4 : d->dv;
  A.cols = rows >= 2 * 148 ? whole : std::min(whole, 32);
  A.nslice = (d->dv + A.cols - 1) / A.cols;
  const long long ctas = rows * A.nslice;
  if (ctas > 0x7fffffffLL) return set_error(HYFFT_ERR_UNSUPPORTED, "decay attention step: too many rows");
  const int per = vec ? A.cols / 4 : A.cols;
  const size_t sm = sizeof(float) * (2 * (size_t)A.DK + (size_t)(kStepThreads / per) * A.cols);
#define HYFFT_STEP(T)                                                               \
  do {                                                                              \
    if (vec)                                                                        \
      decay_step_kernel<T, 4><<<(unsigned)ctas, kStepThreads, sm, st>>>(A);         \
    else                                                                            \
      decay_step_kernel<T, 1><<<(unsigned)ctas, kStepThreads, sm, st>>>(A);         \
  } while (0)
  if (d->dtype == HYFFT_F32)
    HYFFT_STEP(float);
  else if (d->dtype == HYFFT_BF16)
    HYFFT_STEP(__nv_bfloat16);
  else
    HYFFT_STEP(__half);
#undef HYFFT_STEP
  return launched();
}

}  // extern "C"
