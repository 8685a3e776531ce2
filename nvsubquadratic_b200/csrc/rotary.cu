// Rotary positions of queries and keys: feature pair i of the first rot_dim features of every head is turned by
// the angle position * frequency_i (and scaled by an amplitude); the remaining features are copied.
//
//   (a, b) -> amplitude * (a cos - b sin, a sin + b cos)
//
// Pairs are (2i, 2i + 1) (interleaved) or (i, i + rot_dim / 2). The transpose, which is the gradient, is the turn back.
//
// Frequencies come as whole numbers, turns per position in units of 2^-64: the product with the position wraps at
// whole turns, so the remaining fraction of a turn is exact for any 64-bit position, and its sine and cosine are as
// good at position 2^40 as at 1 (a float32 angle is off by 0.004 radians at position 10^5 already).
//
// Every element is read once and written once (that is all the traffic; bound by HBM bandwidth). A thread computes the sines
// and cosines of one vector of pairs at one token and applies them to several heads of q and of k in one launch, so
// their cost is shared; no table is stored or read. 65536 tokens of 32 + 32 heads of 128, bfloat16: 319 us either way, 6.6
// TB/s, the rate of a copy (470 us with elements converted one by one and 64-bit divisions for the thread's place).
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

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

struct RotArgs {
  const void* x[2];
  void* y[2];
  long long xb[2], xl[2], xh[2];  // element strides of batch, token, head; outputs are contiguous
  int heads[2];
  const long long* turns;
  const void* pos;
  long long pb, pl;  // element strides of the positions
  int pos32;
  float amplitude;
  int back, inter;
  int D, half, units, tail, groups, per;  // units: pair vectors, then tail copies; per: heads a thread handles
  long long L, items;
};

// Elements of one pair vector: V pairs as two runs of V (halves) or one run of 2 V (interleaved).
template <typename T, int V>
struct alignas(16) Pairs {
  T e[2 * V];
};

// A run of R elements: 16 bytes on a 16-byte boundary, or (runs of one or two elements) one at a time, from any address.
template <typename T, int R>
__device__ __forceinline__ void copy_run(T* dst, const T* src) {
  if constexpr (R * sizeof(T) == 16) {
    *reinterpret_cast<uint4*>(dst) = *reinterpret_cast<const uint4*>(src);
  } else {
    static_assert(R <= 2, "longer runs are aligned");
#pragma unroll
    for (int u = 0; u < R; ++u) dst[u] = src[u];
  }
}

// Two neighbouring elements as float32 and back; the packed forms where V > 1 says that they lie on an even place.
template <typename T, bool PACKED>
__device__ __forceinline__ float2 two(const T* p) {
  if constexpr (PACKED && sizeof(T) == 2) {
    if constexpr (std::is_same<T, __half>::value) {
      return __half22float2(*reinterpret_cast<const __half2*>(p));
    } else {
      const uint32_t u = *reinterpret_cast<const uint32_t*>(p);
      return make_float2(__uint_as_float(u << 16), __uint_as_float(u & 0xffff0000u));
    }
  }
  return make_float2(DT<T>::load(p), DT<T>::load(p + 1));
}
template <typename T, bool PACKED>
__device__ __forceinline__ void put_two(T* p, float2 v) {
  if constexpr (PACKED && sizeof(T) == 2) {
    if constexpr (std::is_same<T, __half>::value)
      *reinterpret_cast<__half2*>(p) = __floats2half2_rn(v.x, v.y);
    else
      *reinterpret_cast<__nv_bfloat162*>(p) = __floats2bfloat162_rn(v.x, v.y);
  } else {
    DT<T>::store(p, v.x);
    DT<T>::store(p + 1, v.y);
  }
}

// V: pairs per thread. INTER: the pairs are neighbours. ID: the type that counts threads (64-bit divisions would cost as
// much as four heads do).
template <typename T, int V, bool INTER, typename ID>
__global__ void __launch_bounds__(kThreads) rotary_kernel(const RotArgs A) {
  const ID id = (ID)blockIdx.x * kThreads + threadIdx.x;
  if (id >= (ID)A.items) return;
  const ID all = (ID)(A.units + A.tail);
  const int unit = (int)(id % all);
  const ID rest = id / all;
  const int grp = (int)(rest % (ID)A.groups);
  const long long tok = (long long)(rest / (ID)A.groups);
  const long long b = (long long)((ID)tok / (ID)A.L), l = tok - b * A.L;
  const int nh = A.heads[0] + A.heads[1];
  constexpr int R = INTER ? 2 * V : V;  // elements of one run
  const T* src[2];
  T* dst[2];
#pragma unroll
  for (int w = 0; w < 2; ++w) {
    src[w] = static_cast<const T*>(A.x[w]) + b * A.xb[w] + l * A.xl[w];
    dst[w] = static_cast<T*>(A.y[w]) + tok * A.heads[w] * (long long)A.D;
  }
  // head h of q and k counted through
  const auto from = [&](int h) { return h < A.heads[0] ? src[0] + h * A.xh[0] : src[1] + (h - A.heads[0]) * A.xh[1]; };
  const auto to = [&](int h) {
    return h < A.heads[0] ? dst[0] + (long long)h * A.D : dst[1] + (long long)(h - A.heads[0]) * A.D;
  };

  if (unit >= A.units) {  // features that are not turned
    const int c = 2 * A.half + (unit - A.units) * R;
    for (int h = grp; h < nh; h += A.groups) {
      const T* s = from(h) + c;
      T* d = to(h) + c;
      if (c + R <= A.D) {
        copy_run<T, R>(d, s);
      } else {
        for (int u = 0; c + u < A.D; ++u) d[u] = s[u];
      }
    }
    return;
  }

  long long p = l;
  if (A.pos) {
    const long long at = b * A.pb + l * A.pl;
    p = A.pos32 ? (long long)static_cast<const int*>(A.pos)[at] : static_cast<const long long*>(A.pos)[at];
  }
  float cs[V], sn[V];
#pragma unroll
  for (int u = 0; u < V; ++u) {
    const unsigned long long t = (unsigned long long)p * (unsigned long long)A.turns[unit * V + u];
    const float half_turns = (float)(int)(t >> 32) * 4.656612873077393e-10f;  // 2^-31
    float s, c;
    sincospif(half_turns, &s, &c);
    cs[u] = c * A.amplitude;
    sn[u] = A.back ? -s * A.amplitude : s * A.amplitude;
  }
  const int c0 = INTER ? unit * 2 * V : unit * V;
  const int c1 = INTER ? c0 + V : c0 + A.half;
  for (int h0 = grp; h0 < nh; h0 += 4 * A.groups) {  // four heads' loads in flight
    Pairs<T, V> d[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int h = h0 + j * A.groups;
      if (h < nh) {
        const T* s = from(h);
        if constexpr (INTER) {
          copy_run<T, 2 * V>(d[j].e, s + c0);
        } else {
          copy_run<T, V>(d[j].e, s + c0);
          copy_run<T, V>(d[j].e + V, s + c1);
        }
      }
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int h = h0 + j * A.groups;
      if (h < nh) {
        T* o = to(h);
        if constexpr (INTER) {
#pragma unroll
          for (int u = 0; u < V; ++u) {
            const float2 ab = two<T, (V > 1)>(d[j].e + 2 * u);
            put_two<T, (V > 1)>(d[j].e + 2 * u, ffma2(make_float2(ab.y, ab.x), make_float2(-sn[u], sn[u]), cscale(ab, cs[u])));
          }
          copy_run<T, 2 * V>(o + c0, d[j].e);
        } else {
          if constexpr (V == 1) {
            const float a = DT<T>::load(d[j].e), bb = DT<T>::load(d[j].e + 1);
            DT<T>::store(d[j].e, fmaf(a, cs[0], -bb * sn[0]));
            DT<T>::store(d[j].e + 1, fmaf(a, sn[0], bb * cs[0]));
          } else {
#pragma unroll
            for (int u = 0; u < V; u += 2) {
              const float2 a = two<T, true>(d[j].e + u), bb = two<T, true>(d[j].e + V + u);
              const float2 c = make_float2(cs[u], cs[u + 1]), s = make_float2(sn[u], sn[u + 1]);
              const float2 n = make_float2(-sn[u], -sn[u + 1]);
              put_two<T, true>(d[j].e + u, ffma2(bb, n, make_float2(a.x * c.x, a.y * c.y)));
              put_two<T, true>(d[j].e + V + u, ffma2(a, s, make_float2(bb.x * c.x, bb.y * c.y)));
            }
          }
          copy_run<T, V>(o + c0, d[j].e);
          copy_run<T, V>(o + c1, d[j].e + V);
        }
      }
    }
  }
}

template <typename T, int V, bool INTER>
int launch(RotArgs A, long long tokens, cudaStream_t st) {
  const int run = INTER ? 2 * V : V;
  A.units = A.half / V;
  A.tail = (A.D - 2 * A.half + run - 1) / run;
  const int nh = A.heads[0] + A.heads[1];
  // heads per thread: as many as share the sines, while there are two thousand threads for each SM
  int per = std::min(nh, 16);
  while (per > 1 && tokens * (A.units + A.tail) * ((nh + per - 1) / per) < 148ll * 2048) per = (per + 1) / 2;
  A.groups = (nh + per - 1) / per;
  A.items = tokens * (A.units + A.tail) * A.groups;
  const long long ctas = (A.items + kThreads - 1) / kThreads;
  if (ctas > 0x7fffffffLL) return set_error(HYFFT_ERR_UNSUPPORTED, "rotary: too many elements");
  if (ctas * kThreads < (1ll << 32))
    rotary_kernel<T, V, INTER, unsigned><<<(unsigned)ctas, kThreads, 0, st>>>(A);
  else
    rotary_kernel<T, V, INTER, unsigned long long><<<(unsigned)ctas, kThreads, 0, st>>>(A);
  if (cudaGetLastError() != cudaSuccess) return set_error(HYFFT_ERR_CUDA, "rotary: kernel launch failed");
  g_launches.fetch_add(1, std::memory_order_relaxed);
  return HYFFT_OK;
}

template <typename T>
int launch_t(const RotArgs& A, long long tokens, cudaStream_t st) {
  // 16-byte runs where every run of a row starts on a 16-byte boundary, single pairs otherwise
  constexpr int E = 16 / (int)sizeof(T);
  bool al = A.D % E == 0 && (A.inter ? (2 * A.half) % E == 0 : A.half % E == 0);
  for (int w = 0; w < 2; ++w)
    if (A.heads[w])
      al = al && reinterpret_cast<uintptr_t>(A.x[w]) % 16 == 0 && reinterpret_cast<uintptr_t>(A.y[w]) % 16 == 0 &&
           A.xb[w] % E == 0 && A.xl[w] % E == 0 && A.xh[w] % E == 0;
  if (A.inter) return al ? launch<T, E / 2, true>(A, tokens, st) : launch<T, 1, true>(A, tokens, st);
  return al ? launch<T, E, false>(A, tokens, st) : launch<T, 1, false>(A, tokens, st);
}

}  // namespace
}  // namespace hyfft

using namespace hyfft;

extern "C" int hyfft_rotary(const hyfft_rotary_desc* d, const void* q, const void* k, const int64_t* turns,
                            const void* positions, void* out_q, void* out_k, void* stream) {
  if (!d) return set_error(HYFFT_ERR_INVALID, "rotary: null descriptor");
  if (d->batch < 1 || d->length < 1 || d->heads < 1 || d->kv_heads < 0 || d->dim < 1)
    return set_error(HYFFT_ERR_INVALID, "rotary: every extent must be positive");
  if (d->rot_dim < 2 || d->rot_dim % 2 || d->rot_dim > d->dim)
    return set_error(HYFFT_ERR_INVALID, "rotary: rot_dim must be even and at most the head size");
  if (d->dtype < HYFFT_F32 || d->dtype > HYFFT_F16) return set_error(HYFFT_ERR_INVALID, "rotary: bad dtype");
  if (!q || !out_q || !turns || (d->kv_heads && (!k || !out_k)))
    return set_error(HYFFT_ERR_INVALID, "rotary: null tensor");
  if (bind_device_of(q) != HYFFT_OK) return set_error(HYFFT_ERR_CUDA, "rotary: device");
  RotArgs A{};
  A.x[0] = q, A.x[1] = k, A.y[0] = out_q, A.y[1] = out_k;
  A.xb[0] = d->q_stride[0], A.xl[0] = d->q_stride[1], A.xh[0] = d->q_stride[2];
  A.xb[1] = d->k_stride[0], A.xl[1] = d->k_stride[1], A.xh[1] = d->k_stride[2];
  A.heads[0] = d->heads, A.heads[1] = d->kv_heads;
  A.turns = reinterpret_cast<const long long*>(turns);
  A.pos = positions, A.pb = d->pos_stride[0], A.pl = d->pos_stride[1], A.pos32 = d->pos_int32;
  A.amplitude = d->amplitude, A.back = d->backward ? 1 : 0, A.inter = d->interleaved ? 1 : 0;
  A.D = d->dim, A.half = d->rot_dim / 2, A.L = d->length;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const long long tokens = (long long)d->batch * d->length;
  if (d->dtype == HYFFT_F32) return launch_t<float>(A, tokens, st);
  if (d->dtype == HYFFT_BF16) return launch_t<__nv_bfloat16>(A, tokens, st);
  return launch_t<__half>(A, tokens, st);
}
