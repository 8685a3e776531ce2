// Gated linear recurrence over sequences (forward, backward) and for single tokens.
//
//   a_t = sigmoid(g_t) or exp(g_t),  u_t = 1 - a_t,  s_t = u_t or 1
//   h_t = a_t h_{t-1} + s_t x_t,     y_t = h_t  or  h_t * silu(o_t)
//
//   dh_t = dy_t (* silu(o_t)),  G_t = dh_t + c_{t+1},  c_t = a_t G_t,  c_{T+1} = the final state's gradient
//   dx_t = s_t G_t,  dg_t = G_t (h_{t-1} - [s_t = u_t] x_t) * (a_t u_t or a_t),  do_t = dy_t h_t silu'(o_t),  dh_0 = c_1
//
// Every channel is a recurrence of its own; there is nothing to share but the loads, so the floor is one read of the inputs and one write
// of the outputs. A CTA takes a row of 128 bytes of channels (a lane: two of 16 bits or one of 32) and 64 tokens at a time, 16 (backwards
// 8) for each warp, copied to shared memory one tile ahead. A lane runs its tokens from a zero state, which gives the segment's map
//   h -> A h + H  (backwards: c -> A c + C),
// the maps go through shared memory in token order, and the tokens are finished with the state that enters them. Every eighth token's
// state is kept for the backward pass (four bytes for eight tokens of a channel), which then needs nothing else of the forward's.
//
// Where there are fewer rows than CTAs that fit the machine, the CTAs of a cluster take a row's tiles in turn: each passes the state that
// leaves its tile on to the next one's shared memory. In steady state a CTA has its tile's map before the state arrives, so a hop is a
// wait, one map and one remote store (0.25 us), and the data still goes through once; no workspace, no order of arrival in the results.
//
// Measured, bfloat16 with output gates and logits (8 bytes an element forwards, 14 backwards): 64 x 2048 tokens of 1024 channels, one CTA a
// row, 184 us forwards (89% of a copy's rate) and 358 backwards (80%); 65536 tokens of 4096 channels, 8 and 4 CTAs a cluster, 477 us (69%; one
// CTA a row 1.54 ms, all of a cluster's maps exchanged behind a barrier 0.73) and 923 us (62%). On the first: logs 213 and 375, float16 192 and
// 363, float32 344 (95%) and 624 (92%). What is left in 16 bits is latency: 31 instructions an element forwards and 59 backwards keep the issue
// slots busy for 54 to 61% of the time, DRAM for 47 to 57%, and the registers leave room for 4 warps a scheduler, which wait for their own
// arithmetic more than for anything else; and with clusters the turns of the tiles.
//
// What is exact: A is carried as P + l. P is the product of the rounded decays, whose relative error grows with every token; l = (1 - P) - D
// with D = 1 - A, accumulated as D += u P, which keeps the digits of slow decays (0 where decays above 1 made P large on the way, and D
// inexact). So a state that remembers 10^5 tokens is off by the roundings of its 10^4 segments, not by those of its decays; within a segment,
// by 16 products of rounded decays. Sums are float32.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <math_constants.h>

#include <algorithm>
#include <atomic>
#include <map>
#include <mutex>
#include <tuple>
#include <type_traits>

#include "../../include/hyfft.h"
#include "common.cuh"
#include "waits.cuh"

namespace hyfft {

extern std::atomic<long long> g_launches;
int set_error(int code, const char* msg);  // engine.cu: the message hyfft_last_error returns

namespace {

// A pass's tile: SEG tokens for each of a row's lanes, LANES lanes a row (a warp has 32 / LANES segments, one behind the other), WARPS
// warps, and how many CTAs of it an SM holds at least.
template <int SEG, int WARPS, int CTAS, int LANES> struct Shape {
  static constexpr int kSeg = SEG, kWarps = WARPS, kCtas = CTAS, kLanes = LANES, kThreads = 32 * WARPS;
  static constexpr int kSegs = WARPS * 32 / LANES, kTile = SEG * kSegs, kWidth = 4 * LANES;  // bytes of a tile's row
};
template <int LANES> using Fwd = Shape<16, 4, 4, LANES>;
template <int LANES> using Bwd = Shape<8, 8, 2, LANES>;
constexpr int kSaved = 8;              // tokens from one saved state to the next: the backward pass's segments
static_assert(Fwd<32>::kSeg % kSaved == 0 && Bwd<32>::kSeg == kSaved, "both passes have the saved states at hand");
constexpr int kMaxCluster = 16;        // above 8 by a kernel attribute
constexpr unsigned kLanding = 1u << 24; // clocks for a message that has been sent (about 0.25 us) to land

struct ScanArgs {
  const char* in[4];          // x, gate, out_gate, dy
  long long batch[4], tok[4]; // their strides in bytes
  char* out[3];               // y; or dx, dgate, dout_gate; contiguous
  const int* lengths;
  const float* first;         // the state before the first token; backwards the final state's gradient; or NULL
  float* last;                // the state after the last token; backwards the initial state's gradient; or NULL
  float* saved;               // [B, segments, C]: the state that enters each segment; or NULL
  int L, C, cols, segments, complement;
  int n;                      // CTAs of a cluster
  unsigned patience;          // clocks that a wait may take
};

// ---------------------------------------------------------------- a lane's channels: float2 for 16-bit types, float for float32

template <typename T> struct Lane { using F = float2; static constexpr int N = 2; };
template <> struct Lane<float> { using F = float; static constexpr int N = 1; };

__device__ __forceinline__ float fma_(float a, float b, float c) { return fmaf(a, b, c); }
__device__ __forceinline__ float2 fma_(float2 a, float2 b, float2 c) { return ffma2(a, b, c); }
__device__ __forceinline__ float mul_(float a, float b) { return a * b; }
__device__ __forceinline__ float2 mul_(float2 a, float2 b) {
  float2 r;
  asm("{\n.reg .b64 ra, rb, rd;\nmov.b64 ra, {%2, %3};\nmov.b64 rb, {%4, %5};\nmul.rn.f32x2 rd, ra, rb;\n"
      "mov.b64 {%0, %1}, rd;\n}"
      : "=f"(r.x), "=f"(r.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return r;
}
__device__ __forceinline__ float add_(float a, float b) { return a + b; }
__device__ __forceinline__ float2 add_(float2 a, float2 b) { return cadd(a, b); }
__device__ __forceinline__ float sub_(float a, float b) { return a - b; }
__device__ __forceinline__ float2 sub_(float2 a, float2 b) { return csub(a, b); }
template <typename F> __device__ __forceinline__ F all_(float v);
template <> __device__ __forceinline__ float all_<float>(float v) { return v; }
template <> __device__ __forceinline__ float2 all_<float2>(float v) { return make_float2(v, v); }
// op on every channel of up to three values
template <typename Op> __device__ __forceinline__ float each_(float a, Op op) { return op(a); }
template <typename Op> __device__ __forceinline__ float2 each_(float2 a, Op op) { return make_float2(op(a.x), op(a.y)); }
template <typename Op> __device__ __forceinline__ float each_(float a, float b, Op op) { return op(a, b); }
template <typename Op> __device__ __forceinline__ float2 each_(float2 a, float2 b, Op op) {
  return make_float2(op(a.x, b.x), op(a.y, b.y));
}
template <typename Op> __device__ __forceinline__ float each_(float a, float b, float c, Op op) { return op(a, b, c); }
template <typename Op> __device__ __forceinline__ float2 each_(float2 a, float2 b, float2 c, Op op) {
  return make_float2(op(a.x, b.x, c.x), op(a.y, b.y, c.y));
}
template <typename Op> __device__ __forceinline__ bool any_(float a, Op op) { return op(a); }
template <typename Op> __device__ __forceinline__ bool any_(float2 a, Op op) { return op(a.x) || op(a.y); }
template <typename Op> __device__ __forceinline__ bool any_(float a, float b, Op op) { return op(a, b); }
template <typename Op> __device__ __forceinline__ bool any_(float2 a, float2 b, Op op) { return op(a.x, b.x) || op(a.y, b.y); }

// 2^x and 1 / x to 2 units in the last place, results below 2^-126 flushed to zero.
__device__ __forceinline__ float exp2_(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
__device__ __forceinline__ float inverse(float x) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
constexpr float kLog2E = 1.4426950408889634f;
// exp(s g), s = 1 or -1. 16-bit inputs: off by the exponent's rounding, 2^-24 of s g, and by exp2_ (what is left of both in a 16-bit result is
// below its rounding). float32: the rest of the exponent's product too, as a factor 1 + rest.
template <int SIGN> __device__ __forceinline__ float2 exp_of(float2 g) {
  return each_(mul_(g, all_<float2>(SIGN * kLog2E)), exp2_);
}
template <int SIGN> __device__ __forceinline__ float exp_of(float g) {
  constexpr float kLow = 1.925963e-8f;  // log2(e) - kLog2E
  const float t = SIGN * kLog2E * g;
  const float rest = fmaf(SIGN * kLow, g, fmaf(SIGN * kLog2E, g, -t)), e = exp2_(t);
  return fabsf(t) < 126.0f ? fmaf(e * 0.6931472f, rest, e) : e;
}
template <typename F> __device__ __forceinline__ F sigmoid_of(F o) {
  const F e = exp_of<-1>(o);
  return each_(add_(e, all_<F>(1.0f)), inverse);
}

// The decay and what it leaves, a + u = 1, each without cancellation.
template <bool LOG, typename F> __device__ __forceinline__ void decay_of(F g, F& a, F& u) {
  if constexpr (LOG) {
    a = exp_of<1>(g);
    // 1 - exp(g) near 0 by its series (the rest at 0.35 is below 2e-8 of it)
    const F one = all_<F>(1.0f);
    F s = fma_(g, all_<F>(1.0f / 7), one);
    s = fma_(s, mul_(g, all_<F>(1.0f / 6)), one);
    s = fma_(s, mul_(g, all_<F>(1.0f / 5)), one);
    s = fma_(s, mul_(g, all_<F>(1.0f / 4)), one);
    s = fma_(s, mul_(g, all_<F>(1.0f / 3)), one);
    s = fma_(s, mul_(g, all_<F>(-1.0f / 2)), all_<F>(-1.0f));
    // below 0 for decays above 1 alone: a gate of 0 leaves +0
    u = each_(g, fma_(g, s, all_<F>(0.0f)), sub_(one, a), [](float v, float near, float far) { return fabsf(v) < 0.35f ? near : far; });
  } else {
    const F e = exp_of<-1>(g);
    a = each_(add_(e, all_<F>(1.0f)), inverse);
    // e a, which is 1 - a; where e has overflowed and a is 0 that is a NaN or 0, and 1 - 2 a is 1 (below 1 - a everywhere)
    u = each_(mul_(e, a), fma_(a, all_<F>(-2.0f), all_<F>(1.0f)), [](float v, float w) { return fmaxf(v, w); });
  }
}

// ---------------------------------------------------------------- maps h -> (P + l) h + H

template <typename F> struct Map { F P, l, H; };

// Where a map does not give what the recurrence holds in float32, its result is NaN and the tokens are run one by one instead:
// a product of decays or a state from zero that overflows (what enters may be small, or of the other sign); and, where decays may be above
// 1 (form log) and make small states large again, a product that has lost digits (below kLeast: off by up to 2^-149) and grows, or is
// most of a result. A product of 0 has a decay of exactly 0 in it and loses nothing. A decay of 1 at most needs no such care: what a
// product below kLeast leaves of a state is 2^-100 of it.
constexpr float kLeast = 7.888609e-31f;  // 2^-100
constexpr float kLost = 9.403955e-38f;   // 2^-123: 2^-149 of what enters is at most a quarter of a larger result's last place
__device__ __forceinline__ float above_zero(float p) { return p == 0.0f ? __int_as_float(1) : p; }

__device__ __forceinline__ bool infinite(float v) { return fabsf(v) == CUDART_INF_F; }
__device__ __forceinline__ bool finite(float v) { return fabsf(v) < CUDART_INF_F; }
// P, or NaN. A product of decays that are 1 at most does not overflow.
template <bool LOG, typename F> __device__ __forceinline__ F held(F P, F H) {
  return each_(P, H, [](float p, float h) { return (!LOG || finite(p)) && finite(h) ? p : CUDART_NAN_F; });
}
template <typename F> __device__ __forceinline__ F apply(const Map<F>& m, F h) { return fma_(m.P, h, fma_(m.l, h, m.H)); }
__device__ __forceinline__ bool lossy(float P) { return P > 0.0f && P < kLeast; }
// r = P h + H, NaN where it needs digits of P that are not there.
template <typename F> __device__ __forceinline__ F checked(F r, F P, F h) {
  return each_(r, P, h, [](float v, float p, float w) { return lossy(p) && fabsf(w) * kLost > fabsf(v) ? CUDART_NAN_F : v; });
}
// Whether a map made a NaN of what was none.
template <typename F> __device__ __forceinline__ bool fresh_nan(F to, F from) {
  return any_(to, from, [](float t, float f) { return t != t && f == f; });
}

// First f, then s.
template <bool LOG, typename F> __device__ __forceinline__ Map<F> then(const Map<F>& f, const Map<F>& s) {
  Map<F> r;
  r.H = apply(s, f.H);
  const F p = mul_(f.P, s.P);
  const F e = fma_(f.P, s.P, each_(p, [](float v) { return -v; }));
  r.l = fma_(f.P, s.l, fma_(s.P, f.l, e));
  r.P = p;
  if constexpr (LOG) {
    const F of_some = each_(p, f.P, s.P, [](float v, float a, float b) { return a > 0.0f && b > 0.0f ? above_zero(v) : v; });
    r.P = each_(of_some, f.P, s.P, [](float v, float a, float b) { return b > 1.0f && lossy(a) ? CUDART_NAN_F : v; });
  }
  r.P = held<LOG>(r.P, r.H);
  return r;
}

// l of a segment with the product P of its decays and D = 1 - A. Beyond D = 1/2 P is as exact as it gets.
template <typename F> __device__ __forceinline__ F low_part(F P, F D) {
  return each_(P, D, [](float p, float d) { return fabsf(d) < 0.5f ? (1.0f - p) - d : 0.0f; });
}
// The sign bits of what decays leave: set where a decay is above 1.
__device__ __forceinline__ int signs_of(float u) { return __float_as_int(u); }
__device__ __forceinline__ int signs_of(float2 u) { return __float_as_int(u.x) | __float_as_int(u.y); }
// The map of a segment that has decays above 1, for each product on the way and the one before it. D has the roundings of the largest
// product, so it corrects nothing where that is far above 1.
template <typename F> __device__ __forceinline__ void grown(Map<F>& m, F P, F before) {
  m.l = each_(m.l, P, [](float v, float p) { return p > 2.0f ? 0.0f : v; });
  m.P = each_(m.P, P, before, [](float v, float p, float q) { return q < kLeast && p >= q ? CUDART_NAN_F : v; });
}
// Nothing in the channels that are not there (what a tile holds in their place is not defined).
__device__ __forceinline__ float there(float v, int have) { return have > 0 ? v : 0.0f; }
__device__ __forceinline__ float2 there(float2 v, int have) { return make_float2(have > 0 ? v.x : 0.0f, have > 1 ? v.y : 0.0f); }
template <typename F> __device__ __forceinline__ Map<F> there(const Map<F>& m, int have) {
  return Map<F>{there(m.P, have), there(m.l, have), there(m.H, have)};
}

// ---------------------------------------------------------------- tiles

__device__ __forceinline__ uint32_t smem_of(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }
template <int BYTES> __device__ __forceinline__ void copy_async(uint32_t dst, const char* src, int valid) {
  if constexpr (BYTES == 16)
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(valid) : "memory");
  else
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src), "r"(valid) : "memory");
}

// Rows of S::kWidth bytes where every row starts on 16 bytes (ALIGNED), else the 32-bit words that cover them: one more, and a pitch of 16
// bytes more. The halves of a warp that has two segments read rows a segment apart: 64 bytes between segments keep their banks apart.
template <typename S, bool ALIGNED> struct Tile {
  static constexpr int kPitch = S::kWidth + (ALIGNED ? 0 : 16), kPad = S::kLanes < 32 ? 64 : 0;
  static constexpr int kBytes = S::kTile * kPitch + S::kSegs * kPad;
  static __device__ __forceinline__ int row(int r) { return r * kPitch + (kPad ? r / S::kSeg * kPad : 0); }
};

// `rows` tokens from `src` on (the tile's first channel of its first token), `width` bytes of each.
template <typename S, bool ALIGNED>
__device__ __forceinline__ void load_tile(unsigned char* tile, const char* src, long long stride, int rows, int width) {
  using L = Tile<S, ALIGNED>;
  const uint32_t to = smem_of(tile);
  if constexpr (ALIGNED) {
    constexpr int kChunks = S::kWidth / 16;
    const int c = 16 * (threadIdx.x % kChunks), valid = min(16, width - c);
    if (valid > 0) {
#pragma unroll
      for (int i = 0; i < S::kTile * kChunks / S::kThreads; ++i) {
        const int r = threadIdx.x / kChunks + i * (S::kThreads / kChunks);
        if (r < rows) copy_async<16>(to + L::row(r) + c, src + r * stride + c, valid);
      }
    }
  } else {
    const int lane = threadIdx.x & 31;
    for (int r = threadIdx.x >> 5; r < rows; r += S::kWarps) {
      const char* p = src + r * stride;
      const int off = (int)(reinterpret_cast<uintptr_t>(p) & 3);
      for (int w = 4 * lane; w < off + width; w += 128) copy_async<4>(to + L::row(r) + w, p - off + w, min(4, off + width - w));
    }
  }
}

// A lane's channels at p in the tile, of row r; `src` as for load_tile.
template <typename T, bool ALIGNED>
__device__ __forceinline__ typename Lane<T>::F lane_of(const unsigned char* p, const char* src, long long stride, int r) {
  if constexpr (std::is_same<T, float>::value) {
    return *reinterpret_cast<const float*>(p);
  } else if constexpr (ALIGNED) {
    const uint32_t w = *reinterpret_cast<const uint32_t*>(p);
    if constexpr (std::is_same<T, __half>::value)
      return __half22float2(*reinterpret_cast<const __half2*>(&w));
    else
      return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
  } else {
    p += reinterpret_cast<uintptr_t>(src + r * stride) & 2;
    const T* t = reinterpret_cast<const T*>(p);
    return make_float2(DT<T>::load(t), DT<T>::load(t + 1));
  }
}

// base + i * stride (elements): the compiler keeps the three bases and one stride of the backward pass in registers.
template <typename T> __device__ __forceinline__ T* row_at(T* base, unsigned stride, unsigned i) {
  T* r;
  asm("mad.wide.u32 %0, %1, %2, %3;" : "=l"(r) : "r"(stride), "r"(i * (unsigned)sizeof(T)), "l"(base));
  return r;
}
// A lane's channels to the output; `have` (1 at least) of them exist.
template <typename T, bool ALIGNED>
__device__ __forceinline__ void put(T* p, typename Lane<T>::F v, int have) {
  if constexpr (std::is_same<T, float>::value) {
    *p = v;
  } else if constexpr (!ALIGNED) {
    DT<T>::store(p, v.x);
    if (have > 1) DT<T>::store(p + 1, v.y);
  } else if constexpr (std::is_same<T, __half>::value) {
    *reinterpret_cast<__half2*>(p) = __floats2half2_rn(v.x, v.y);
  } else {
    *reinterpret_cast<__nv_bfloat162*>(p) = __floats2bfloat162_rn(v.x, v.y);
  }
}
__device__ __forceinline__ float get_state(const float* p, int have, float) { return have > 0 ? *p : 0.0f; }
__device__ __forceinline__ float2 get_state(const float* p, int have, float2) {
  return make_float2(have > 0 ? p[0] : 0.0f, have > 1 ? p[1] : 0.0f);
}
__device__ __forceinline__ void put_state(float* p, int have, float v) {
  if (have > 0) *p = v;
}
__device__ __forceinline__ void put_state(float* p, int have, float2 v) {
  if (have > 0) p[0] = v.x;
  if (have > 1) p[1] = v.y;
}

// ---------------------------------------------------------------- a row's tiles among the CTAs of a cluster

__device__ __forceinline__ void cluster_meet() {
  asm volatile("barrier.cluster.arrive.release.aligned;\nbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ uint32_t at_rank(uint32_t own, int rank) {
  uint32_t p;
  asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(p) : "r"(own), "r"(rank));
  return p;
}
// Writes to another CTA's shared memory and counts the bytes at a barrier there.
__device__ __forceinline__ void send(uint32_t to, uint32_t bar, float v) {
  asm volatile("st.async.weak.shared::cluster.mbarrier::complete_tx::bytes.b32 [%0], %1, [%2];" ::"r"(to),
               "r"(__float_as_uint(v)), "r"(bar)
               : "memory");
}
__device__ __forceinline__ void send(uint32_t to, uint32_t bar, float2 v) {
  asm volatile("st.async.weak.shared::cluster.mbarrier::complete_tx::bytes.v2.b32 [%0], {%1, %2}, [%3];" ::"r"(to),
               "r"(__float_as_uint(v.x)), "r"(__float_as_uint(v.y)), "r"(bar)
               : "memory");
}
__device__ __forceinline__ void arm(uint32_t bar, int bytes) {
  asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
}
__device__ __forceinline__ bool try_message(uint32_t bar, uint32_t parity) {
  uint32_t done;
  asm volatile(
      "{\n.reg .pred p;\nmbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\nselp.u32 %0, 1, 0, p;\n}\n"
      : "=r"(done)
      : "r"(bar), "r"(parity)
      : "memory");
  return done != 0;
}
__device__ __forceinline__ bool test_message(uint32_t bar, uint32_t parity) {
  uint32_t done;
  asm volatile(
      "{\n.reg .pred p;\nmbarrier.test_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\nselp.u32 %0, 1, 0, p;\n}\n"
      : "=r"(done)
      : "r"(bar), "r"(parity)
      : "memory");
  return done != 0;
}
// Waits for a message; false after `patience` clocks (0: without waiting).
__device__ __forceinline__ bool wait_message(uint32_t bar, uint32_t parity, unsigned patience) {
  if (patience ? try_message(bar, parity) : test_message(bar, parity)) return true;
  const unsigned t0 = (unsigned)clock64();
  do {
    if ((unsigned)clock64() - t0 >= patience) return false;
  } while (!try_message(bar, parity));
  return true;
}

// The maps of a tile's segments, and the states that enter tiles: two, used in turn. Where another CTA has the tile before, it sends
// them. The next one into a place is written only after this CTA's last warp has handed on the one in between, so after all warps have read it.
template <typename F, typename S> struct Board {
  F P[S::kSegs][S::kLanes], l[S::kSegs][S::kLanes], H[S::kSegs][S::kLanes];
  F inbox[2][S::kLanes];
  unsigned long long full[2];
};

// Where a CTA works: one batch row and S::kWidth bytes of channels. The n CTAs of a cluster take the row's tiles in turn, each passing the
// state that leaves its tile to the next.
struct Place {
  int n, rank, b, col, ch, have, len, tiles;
  int seg;  // this lane's segment of a tile
};
template <typename T, typename S> __device__ __forceinline__ Place place_of(const ScanArgs& A) {
  Place p;
  p.n = A.n, p.rank = blockIdx.x % A.n;  // a cluster's CTAs are neighbours
  const int row = blockIdx.x / A.n;
  p.b = row / A.cols, p.col = row % A.cols;
  p.ch = (p.col * S::kLanes + threadIdx.x % S::kLanes) * Lane<T>::N;
  p.seg = threadIdx.x / S::kLanes;
  p.have = A.C - p.ch;
  p.len = A.lengths ? min(max(A.lengths[p.b], 0), A.L) : A.L;
  p.tiles = (p.len + S::kTile - 1) / S::kTile;
  return p;
}

template <typename F, typename S> __device__ __forceinline__ void open_board(Board<F, S>& B, const Place& p) {
  if (p.n == 1) return;
  if (threadIdx.x == 0) {
    for (int i = 0; i < 2; ++i) {
      asm volatile("mbarrier.init.shared::cta.b64 [%0], 1;" ::"r"(smem_of(&B.full[i])) : "memory");
      arm(smem_of(&B.full[i]), sizeof(B.inbox[0]));
    }
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  cluster_meet();  // the others run, and their barriers are there
}
// What a warp has heard of its CTA's messages. After one that did not come in time (lost) it takes none.
struct Mail {
  int heard = 0;
  bool lost = false;
};
// Messages that come late after all: their barriers are armed again, so that what the next ones count stays in range.
template <typename F, typename S> __device__ __forceinline__ void hear(Board<F, S>& B, Mail& mail, int messages, unsigned patience) {
  while (mail.heard < messages && wait_message(smem_of(&B.full[mail.heard & 1]), (mail.heard >> 1) & 1, patience)) {
    arm(smem_of(&B.full[mail.heard & 1]), sizeof(B.inbox[0]));
    ++mail.heard;
  }
}
// No CTA leaves while another may still write to it: behind the barrier all messages are sent, and one that has given up waits for those
// that it has not heard. steps: the tiles that this CTA has handed on.
template <typename F, typename S> __device__ __forceinline__ void close_board(Board<F, S>& B, const Place& p, Mail& mail, int steps) {
  if (p.n == 1) return;
  cluster_meet();
  if (threadIdx.x == 0 && mail.lost) hear(B, mail, steps - (p.rank == 0 && steps > 0 ? 1 : 0), kLanding);
}

// Hands the maps of a tile's segments on. k: the tile's number in the order of the recurrence, step: how many this CTA has done
// before; order: this lane's segment's place within the tile. state: what enters the first tile; in the last segment, what leaves each.
// tokens(j, h): the state that leaves the segment in place j, by its tokens, where h enters it.
// Returns what enters this lane's segment: NaN from the first message on that did not come (lost).
template <bool LOG, typename F, typename S, typename Tokens>
__device__ __forceinline__ F hand_on(Board<F, S>& B, const Place& p, int k, int step, int order, const Map<F>& mine, F& state,
                                     unsigned patience, Mail& mail, const Tokens& tokens) {
  const int lane = threadIdx.x % S::kLanes;
  B.P[order][lane] = mine.P, B.l[order][lane] = mine.l, B.H[order][lane] = mine.H;
  // Maps of lost digits are looked at one by one, where a tile has any (looked for in every chain, 64 x 2048 tokens of 1024
  // channels in bfloat16 took 392 us backwards instead of 377).
  bool careful = false;
  if constexpr (LOG)
    careful = __syncthreads_or(any_(mine.P, lossy)) != 0;
  else
    __syncthreads();
  const auto map_of = [&](int j) { return Map<F>{B.P[j][lane], B.l[j][lane], B.H[j][lane]}; };
  const auto through = [&](int j, F h) {
    const Map<F> m = map_of(j);
    F r = apply(m, h);
    if constexpr (LOG) r = checked(r, m.P, h);
    if (!fresh_nan(r, h)) return r;
    return each_(r, tokens(j, h), [](float v, float t) { return v != v ? t : v; });
  };
  // What leaves the tile goes by one map over all of it, which is there before the message is: the next CTA waits for nothing else.
  const bool last = order == S::kSegs - 1, sends = last && p.n > 1;
  Map<F> whole = mine;
  bool digits = false;  // that whole has lost
  if (sends) {
    whole = map_of(0);
#pragma unroll 1
    for (int j = 1; j < S::kSegs; ++j) {
      const Map<F> m = map_of(j), both = then<LOG>(whole, m);
      const F h = whole.H;
      whole = both;
      if (careful) whole.P = each_(both.P, checked(both.H, m.P, h), [](float v, float w) { return w != w ? w : v; });
    }
    digits = LOG && any_(whole.P, lossy);
  }
  if (p.n == 1 && S::kSegs <= 4) {  // few enough for every warp to go through all of them
    F h = state, in = state;
#pragma unroll
    for (int j = 0; j < S::kSegs; ++j) {
      if (j == order) in = h;
      h = apply(map_of(j), h);
    }
    if (careful || fresh_nan(h, state)) {
      h = in = state;
#pragma unroll 1
      for (int j = 0; j < S::kSegs; ++j) {
        if (j == order) in = h;
        h = through(j, h);
      }
    }
    state = h;
    return in;
  }
  F h = state;
  if (k > 0) {
    // the message's number: the first CTA of a cluster gets none for its first tile, a CTA alone leaves them to itself
    const int m = p.rank > 0 ? step : step - 1;
    if (p.n > 1) {
      const uint32_t bar = smem_of(&B.full[m & 1]);
      if (!mail.lost) mail.lost = !__all_sync(0xffffffffu, wait_message(bar, (m >> 1) & 1, patience));
      if (!mail.lost) {
        if (threadIdx.x == 0) arm(bar, sizeof(B.inbox[0]));
        mail.heard = m + 1;
      } else if (threadIdx.x % 32 == 0) {
        atomicExch(&g_ran_out, 1u);
        if (threadIdx.x == 0) hear(B, mail, m + 1, 0);
      }
    }
    h = mail.lost ? all_<F>(CUDART_NAN_F) : B.inbox[m & 1][lane];
  }
  const auto pass_on = [&] {
    if (k + 1 < p.tiles) {
      const int next = p.rank + 1 == p.n ? 0 : p.rank + 1;
      send(at_rank(smem_of(&B.inbox[step & 1][lane]), next), at_rank(smem_of(&B.full[step & 1]), next), state);
    }
  };
  bool late = false;
  if (sends) {
    state = apply(whole, h);
    late = fresh_nan(digits ? checked(state, whole.P, h) : state, h);
    if (!late) pass_on();
  }
  F in = h;
#pragma unroll 1
  for (int j = 0; j < order; ++j) in = apply(map_of(j), in);
  if (late || careful || fresh_nan(in, h)) {
    in = h;
#pragma unroll 1
    for (int j = 0; j < order; ++j) in = through(j, in);
  }
  if (last && p.n == 1) {
    state = apply(mine, in);
    if (careful || fresh_nan(state, in)) state = through(order, in);
    B.inbox[step & 1][lane] = state;
  }
  if (late) {
    state = through(order, in);
    pass_on();
  }
  return in;
}

// ---------------------------------------------------------------- the passes

// Tokens past the last tile: zeros.
template <typename T, typename S, bool ALIGNED, int OUTS>
__device__ __forceinline__ void zeros_behind(const ScanArgs& A, const Place& p) {
  if (p.have < 1) return;
  for (int t = p.tiles * S::kTile + p.rank * S::kSegs + p.seg; t < A.L; t += p.n * S::kSegs)
#pragma unroll
    for (int k = 0; k < OUTS; ++k)
      put<T, ALIGNED>(reinterpret_cast<T*>(A.out[k]) + ((long long)p.b * A.L + t) * A.C + p.ch, all_<typename Lane<T>::F>(0.0f), p.have);
}

template <typename T, int LANES, bool LOG, bool GATE, bool COMP, bool ALIGNED>
__global__ void __launch_bounds__(Fwd<LANES>::kThreads, Fwd<LANES>::kCtas) gated_fwd_kernel(const ScanArgs A) {
  using F = typename Lane<T>::F;
  using S = Fwd<LANES>;
  constexpr int K = GATE ? 3 : 2, TB = Tile<S, ALIGNED>::kBytes, kSeg = S::kSeg;
  extern __shared__ __align__(128) unsigned char smem[];
  auto& B = *reinterpret_cast<Board<F, S>*>(smem + 2 * K * TB);
  const Place p = place_of<T, S>(A);
  const int width = min(S::kWidth, A.C * (int)sizeof(T) - p.col * S::kWidth);
  const char* in[K];
#pragma unroll
  for (int k = 0; k < K; ++k) in[k] = A.in[k] + p.b * A.batch[k] + p.col * S::kWidth;
  const auto fetch = [&](int step, int tile) {
    const int t = tile * S::kTile, rows = min(S::kTile, p.len - t);
#pragma unroll
    for (int k = 0; k < K; ++k)
      load_tile<S, ALIGNED>(smem + ((step & 1) * K + k) * TB, in[k] + t * A.tok[k], A.tok[k], rows, width);
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  F state = all_<F>(0.0f);
  if (A.first) state = get_state(A.first + (long long)p.b * A.C + p.ch, p.have, state);
  Mail mail;
  open_board(B, p);
  if (p.rank < p.tiles) fetch(0, p.rank);
  // Whole tiles, and the tile that the row ends in, are apart from each other: a test for each token keeps the tokens' latencies apart too.
  const auto run = [&](int k, int step, auto all_live) {
    constexpr bool whole = decltype(all_live)::value;
    asm volatile("cp.async.wait_group 0;" ::: "memory");
    __syncthreads();
    if (k + p.n < p.tiles) fetch(step + 1, k + p.n);
    const unsigned char* tile = smem + (step & 1) * K * TB;
    const int tile0 = k * S::kTile, r0 = p.seg * kSeg, t0 = tile0 + r0;
    const int live = whole ? kSeg : min(kSeg, p.len - t0);  // below 1: none
    const unsigned char* mine = tile + Tile<S, ALIGNED>::row(r0) + 4 * (threadIdx.x % LANES);
    const auto value = [&](int k, int i) {
      return lane_of<T, ALIGNED>(mine + k * TB + i * Tile<S, ALIGNED>::kPitch, in[k] + tile0 * A.tok[k], A.tok[k], r0 + i);
    };
    const auto token = [&](int i, F& a, F& u, F& b) {
      const F x = value(0, i);
      decay_of<LOG>(value(1, i), a, u);
      b = COMP ? mul_(u, x) : x;
    };
    F hl[kSeg], Pl[kSeg];
    F h = all_<F>(0.0f), P = all_<F>(1.0f), D = all_<F>(0.0f);
    [[maybe_unused]] int signs = 0;
#pragma unroll
    for (int i = 0; i < kSeg; ++i) {
      if (whole || i < live) {
        F a, u, b;
        token(i, a, u, b);
        h = fma_(a, h, b);
        D = fma_(u, P, D);
        P = mul_(P, a);
        if constexpr (LOG) signs |= signs_of(u);
      }
      hl[i] = h, Pl[i] = P;
    }
    Map<F> map{P, low_part(P, D), h};
    if constexpr (LOG) {
      if (signs < 0) {  // a decay above 1
#pragma unroll
        for (int i = 0; i < kSeg; ++i) grown(map, Pl[i], i ? Pl[i ? i - 1 : 0] : all_<F>(1.0f));
      }
      if (any_(P, [](float v) { return v == 0.0f; })) {  // lost, or a decay of 0?
        F least = all_<F>(1.0f);
#pragma unroll 1
        for (int i = 0; i < live; ++i) {
          F a, u;
          decay_of<LOG>(value(1, i), a, u);
          least = each_(least, a, [](float v, float w) { return fminf(v, w); });
        }
        map.P = each_(map.P, least, [](float v, float w) { return w > 0.0f ? above_zero(v) : v; });
      }
    }
    map.P = held<LOG>(map.P, map.H);
    if (p.have < Lane<T>::N) map = there(map, p.have);
    const auto tokens = [&](int seg, F state) {
      const int r = seg * kSeg, n = min(kSeg, p.len - tile0 - r);
      const unsigned char* at = tile + Tile<S, ALIGNED>::row(r) + 4 * (threadIdx.x % LANES);
#pragma unroll 1
      for (int i = 0; i < n; ++i, at += Tile<S, ALIGNED>::kPitch) {
        const F x = lane_of<T, ALIGNED>(at, in[0] + tile0 * A.tok[0], A.tok[0], r + i);
        F a, u;
        decay_of<LOG>(lane_of<T, ALIGNED>(at + TB, in[1] + tile0 * A.tok[1], A.tok[1], r + i), a, u);
        state = fma_(a, state, COMP ? mul_(u, x) : x);
      }
      return state;
    };
    const F carry = hand_on<LOG>(B, p, k, step, p.seg, map, state, A.patience, mail, tokens);
    if (p.have < 1) return;
    T* const y = reinterpret_cast<T*>(A.out[0]) + ((long long)p.b * A.L + t0) * A.C + p.ch;
    float* const s = A.saved + ((long long)p.b * A.segments + t0 / kSaved) * A.C + p.ch;
    bool alone = any_(carry, infinite) || any_(map.P, [](float v) { return v != v; });
    if constexpr (LOG) {
      if (any_(P, [](float v) { return v < kLeast; })) {  // digits lost on the way: does an output need them?
        F low = all_<F>(3.4e38f);
#pragma unroll
        for (int i = 0; i < kSeg; ++i) low = each_(low, fma_(Pl[i], carry, hl[i]), [](float v, float w) { return fminf(v, fabsf(w)); });
        alone = alone || any_(low, carry, [](float v, float c) { return fabsf(c) * kLost > v; });
      }
    }
    // token by token, as the recurrence has it; apart from the rest, which keeps its registers
    if (alone) {
      F full = carry;
#pragma unroll 1
      for (int i = 0; i < kSeg && t0 + i < A.L; ++i) {
        F v = all_<F>(0.0f);
        if (i < live) {
          if (A.saved && i % kSaved == 0) put_state(s + (long long)(i / kSaved) * A.C, p.have, full);
          F a, u, b;
          token(i, a, u, b);
          v = full = fma_(a, full, b);
          if constexpr (GATE) {
            const F o = value(2, i);
            v = mul_(v, mul_(o, sigmoid_of(o)));
          }
        }
        put<T, ALIGNED>(y + (long long)i * A.C, v, p.have);
      }
      return;
    }
    if (A.saved) {
#pragma unroll
      for (int i = 0; i < kSeg; i += kSaved)
        if (whole || i < live)
          put_state(s + (long long)(i / kSaved) * A.C, p.have, i ? fma_(Pl[i ? i - 1 : 0], carry, hl[i ? i - 1 : 0]) : carry);
    }
#pragma unroll
    for (int i = 0; i < kSeg; ++i) {
      if (whole || t0 + i < A.L) {
        F v = all_<F>(0.0f);
        if (whole || i < live) {
          v = fma_(Pl[i], carry, hl[i]);
          if constexpr (GATE) {
            const F o = value(2, i);
            v = mul_(v, mul_(o, sigmoid_of(o)));
          }
        }
        put<T, ALIGNED>(y + (long long)i * A.C, v, p.have);
      }
    }
  };
  const int full = p.len / S::kTile;
  int k = p.rank, step = 0;
  for (; k < full; k += p.n, ++step) run(k, step, std::true_type{});
  if (k < p.tiles) {
    run(k, step, std::false_type{});
    ++step;
  }
  // the last tile's CTA has the state in its last segment; a row without tokens keeps what it was given
  if (A.last && p.seg == S::kSegs - 1 && p.rank == max(p.tiles - 1, 0) % p.n)
    put_state(A.last + (long long)p.b * A.C + p.ch, p.have, state);
  zeros_behind<T, S, ALIGNED, 1>(A, p);
  close_board(B, p, mail, step);
}

template <typename T, int LANES, bool LOG, bool GATE, bool COMP, bool ALIGNED>
__global__ void __launch_bounds__(Bwd<LANES>::kThreads, Bwd<LANES>::kCtas) gated_bwd_kernel(const ScanArgs A) {
  using F = typename Lane<T>::F;
  using S = Bwd<LANES>;
  constexpr int K = GATE ? 4 : 3, TB = Tile<S, ALIGNED>::kBytes, kSeg = S::kSeg;
  constexpr int kDy = K - 1;  // x, gate, (out_gate,) dy
  extern __shared__ __align__(128) unsigned char smem[];
  auto& B = *reinterpret_cast<Board<F, S>*>(smem + 2 * K * TB);
  const Place p = place_of<T, S>(A);
  const int width = min(S::kWidth, A.C * (int)sizeof(T) - p.col * S::kWidth);
  const char* in[K];
  long long tok[K];
#pragma unroll
  for (int k = 0; k < K; ++k) {
    const int from = k == kDy ? 3 : k;
    in[k] = A.in[from] + p.b * A.batch[from] + p.col * S::kWidth;
    tok[k] = A.tok[from];
  }
  const auto fetch = [&](int step, int tile) {
    const int t = tile * S::kTile, rows = min(S::kTile, p.len - t);
#pragma unroll
    for (int k = 0; k < K; ++k)
      load_tile<S, ALIGNED>(smem + ((step & 1) * K + k) * TB, in[k] + t * tok[k], tok[k], rows, width);
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  unsigned stride = A.C;
  asm volatile("" : "+r"(stride));  // in a register, not fetched again for each store
  F state = all_<F>(0.0f);
  if (A.first) state = get_state(A.first + (long long)p.b * A.C + p.ch, p.have, state);
  Mail mail;
  open_board(B, p);
  if (p.rank < p.tiles) fetch(0, p.tiles - 1 - p.rank);
  const auto run = [&](int k, int step, auto all_live) {
    constexpr bool whole = decltype(all_live)::value;
    const int tile0 = (p.tiles - 1 - k) * S::kTile, r0 = p.seg * kSeg, t0 = tile0 + r0;
    const int live = whole ? kSeg : min(kSeg, p.len - t0);
    F before[kSeg + 1];  // before[i]: the state that enters token i
    before[0] = all_<F>(0.0f);
    if (live > 0) before[0] = get_state(A.saved + ((long long)p.b * A.segments + t0 / kSaved) * A.C + p.ch, p.have, before[0]);
    asm volatile("cp.async.wait_group 0;" ::: "memory");
    __syncthreads();
    if (k + p.n < p.tiles) fetch(step + 1, p.tiles - 1 - k - p.n);
    const unsigned char* tile = smem + (step & 1) * K * TB;
    const unsigned char* mine = tile + Tile<S, ALIGNED>::row(r0) + 4 * (threadIdx.x % LANES);
    const auto value = [&](int k, int i) {
      return lane_of<T, ALIGNED>(mine + k * TB + i * Tile<S, ALIGNED>::kPitch, in[k] + tile0 * tok[k], tok[k], r0 + i);
    };
    F a[kSeg], u[kSeg], sig[kSeg];
    F c = all_<F>(0.0f), P = all_<F>(1.0f), D = all_<F>(0.0f);
    [[maybe_unused]] int signs = 0;
#pragma unroll
    for (int i = 0; i < kSeg; ++i) {
      before[i + 1] = before[i];
      if (whole || i < live) {
        const F x = value(0, i);
        decay_of<LOG>(value(1, i), a[i], u[i]);
        before[i + 1] = fma_(a[i], before[i], COMP ? mul_(u[i], x) : x);
      }
    }
#pragma unroll
    for (int i = kSeg - 1; i >= 0; --i) {
      if (whole || i < live) {
        F dh = value(kDy, i);
        if constexpr (GATE) {
          const F o = value(2, i);
          sig[i] = sigmoid_of(o);
          dh = mul_(dh, mul_(o, sig[i]));
        }
        c = mul_(a[i], add_(dh, c));
        D = fma_(u[i], P, D);
        P = mul_(P, a[i]);
        if constexpr (LOG) signs |= signs_of(u[i]);
      }
    }
    Map<F> map{P, low_part(P, D), c};
    if constexpr (LOG) {
      if (signs < 0) {  // a decay above 1
        F q = all_<F>(1.0f);
#pragma unroll 1
        for (int i = live - 1; i >= 0; --i) {
          const F before_it = q;
          F decay, left;
          decay_of<LOG>(value(1, i), decay, left);
          q = mul_(q, decay);
          grown(map, q, before_it);
        }
      }
      if (any_(P, [](float v) { return v == 0.0f; })) {  // lost, or a decay of 0?
        F least = all_<F>(1.0f);
#pragma unroll
        for (int i = 0; i < kSeg; ++i)
          if (whole || i < live) least = each_(least, a[i], [](float v, float w) { return fminf(v, w); });
        map.P = each_(map.P, least, [](float v, float w) { return w > 0.0f ? above_zero(v) : v; });
      }
    }
    map.P = held<LOG>(map.P, map.H);
    if (p.have < Lane<T>::N) map = there(map, p.have);
    const auto tokens = [&](int place, F state) {
      const int r = (S::kSegs - 1 - place) * kSeg, n = min(kSeg, p.len - tile0 - r);
      const unsigned char* first = tile + Tile<S, ALIGNED>::row(r) + 4 * (threadIdx.x % LANES);
#pragma unroll 1
      for (int i = n - 1; i >= 0; --i) {
        const unsigned char* at = first + i * Tile<S, ALIGNED>::kPitch;
        const auto of = [&](int j) { return lane_of<T, ALIGNED>(at + j * TB, in[j] + tile0 * tok[j], tok[j], r + i); };
        F a, u, dh = of(kDy);
        decay_of<LOG>(of(1), a, u);
        if constexpr (GATE) {
          const F o = of(2);
          dh = mul_(dh, mul_(o, sigmoid_of(o)));
        }
        state = mul_(a, add_(dh, state));
      }
      return state;
    };
    c = hand_on<LOG>(B, p, k, step, S::kSegs - 1 - p.seg, map, state, A.patience, mail, tokens);
    const long long at = ((long long)p.b * A.L + t0) * A.C + p.ch;
    T* const dx_at = reinterpret_cast<T*>(A.out[0]) + at;
    T* const dg_at = reinterpret_cast<T*>(A.out[1]) + at;
    [[maybe_unused]] T* const do_at = reinterpret_cast<T*>(A.out[2]) + at;
    if (p.have < 1) return;
#pragma unroll
    for (int i = kSeg - 1; i >= 0; --i) {
      if (whole || t0 + i < A.L) {
        F dx = all_<F>(0.0f), dg = dx;
        [[maybe_unused]] F dO = dx;
        if (whole || i < live) {
          const F dy = value(kDy, i);
          F dh = dy;
          if constexpr (GATE) {
            const F o = value(2, i);
            dh = mul_(dy, mul_(o, sig[i]));
            // silu'(o) = sig + o sig (1 - sig)
            const F slope = mul_(sig[i], fma_(o, sub_(all_<F>(1.0f), sig[i]), all_<F>(1.0f)));
            dO = mul_(mul_(dy, before[i + 1]), slope);
          }
          const F G = add_(dh, c);
          c = mul_(a[i], G);
          dx = COMP ? mul_(u[i], G) : G;
          const F da = mul_(G, COMP ? sub_(before[i], value(0, i)) : before[i]);
          dg = mul_(da, LOG ? a[i] : mul_(a[i], u[i]));
        }
        put<T, ALIGNED>(row_at(dx_at, stride, i), dx, p.have);
        put<T, ALIGNED>(row_at(dg_at, stride, i), dg, p.have);
        if constexpr (GATE) put<T, ALIGNED>(row_at(do_at, stride, i), dO, p.have);
      }
    }
  };
  int k = p.rank, step = 0;
  if (k == 0 && p.len % S::kTile) {
    run(k, step, std::false_type{});
    k += p.n, ++step;
  }
  for (; k < p.tiles; k += p.n, ++step) run(k, step, std::true_type{});
  if (A.last && p.seg == 0 && p.rank == max(p.tiles - 1, 0) % p.n)
    put_state(A.last + (long long)p.b * A.C + p.ch, p.have, state);
  zeros_behind<T, S, ALIGNED, GATE ? 3 : 2>(A, p);
  close_board(B, p, mail, step);
}

// ---------------------------------------------------------------- single tokens

struct StepArgs {
  const void *x, *g, *o;
  long long xb, gb, ob;  // element strides of the batch
  const int* slots;
  const float* state;
  float* out_state;
  void* y;
  long long pool;
  int B, C, complement, units;
};

// One thread for V neighbouring channels of a request.
template <typename T, bool LOG, int V>
__global__ void __launch_bounds__(256) gated_step_kernel(const StepArgs A) {
  const long long id = (long long)blockIdx.x * 256 + threadIdx.x;
  if (id >= (long long)A.B * A.units) return;
  const int b = (int)(id / A.units), c = (int)(id % A.units) * V;
  struct alignas(V * sizeof(T)) Row { T e[V]; };
  struct alignas(V * 4) State { float e[V]; };
  Row& y = *reinterpret_cast<Row*>(static_cast<T*>(A.y) + (long long)b * A.C + c);
  const long long slot = A.slots ? A.slots[b] : b;
  Row out;
  if (slot < 0 || slot >= A.pool) {
#pragma unroll
    for (int i = 0; i < V; ++i) DT<T>::store(&out.e[i], 0.0f);
    y = out;
    return;
  }
  const Row x = *reinterpret_cast<const Row*>(static_cast<const T*>(A.x) + b * A.xb + c);
  const Row g = *reinterpret_cast<const Row*>(static_cast<const T*>(A.g) + b * A.gb + c);
  Row o{};
  if (A.o) o = *reinterpret_cast<const Row*>(static_cast<const T*>(A.o) + b * A.ob + c);
  State h = *reinterpret_cast<const State*>(A.state + slot * A.C + c);
#pragma unroll
  for (int i = 0; i < V; ++i) {
    float a, u;
    decay_of<LOG>(DT<T>::load(&g.e[i]), a, u);
    const float xi = DT<T>::load(&x.e[i]);
    h.e[i] = fmaf(a, h.e[i], A.complement ? u * xi : xi);
    float v = h.e[i];
    if (A.o) {
      const float oi = DT<T>::load(&o.e[i]);
      v *= oi * sigmoid_of(oi);
    }
    DT<T>::store(&out.e[i], v);
  }
  *reinterpret_cast<State*>(A.out_state + slot * A.C + c) = h;
  y = out;
}

// ---------------------------------------------------------------- host

using Kernel = void (*)(ScanArgs);

struct Form {
  bool back, log, gate, complement, aligned;
};
template <typename T, int LANES, bool LOG, bool GATE, bool COMP> Kernel pick3(const Form& f) {
  if (f.back) return f.aligned ? gated_bwd_kernel<T, LANES, LOG, GATE, COMP, true> : gated_bwd_kernel<T, LANES, LOG, GATE, COMP, false>;
  return f.aligned ? gated_fwd_kernel<T, LANES, LOG, GATE, COMP, true> : gated_fwd_kernel<T, LANES, LOG, GATE, COMP, false>;
}
template <typename T, int LANES, bool LOG, bool GATE> Kernel pick2(const Form& f) {
  return f.complement ? pick3<T, LANES, LOG, GATE, true>(f) : pick3<T, LANES, LOG, GATE, false>(f);
}
template <typename T, int LANES> Kernel pick1(const Form& f) {
  if (f.log) return f.gate ? pick2<T, LANES, true, true>(f) : pick2<T, LANES, true, false>(f);
  return f.gate ? pick2<T, LANES, false, true>(f) : pick2<T, LANES, false, false>(f);
}
template <int LANES> Kernel pick(int dtype, const Form& f) {
  if (dtype == HYFFT_F32) return pick1<float, LANES>(f);
  return dtype == HYFFT_BF16 ? pick1<__nv_bfloat16, LANES>(f) : pick1<__half, LANES>(f);
}

// Clusters of n CTAs that can run at once (0: unknown), asked once for each kernel, size and device.
int room_for(Kernel fn, int n, int threads, size_t smem) {
  static std::mutex mu;
  static std::map<std::tuple<const void*, int, int>, int> known;
  int dev = 0;
  cudaGetDevice(&dev);
  std::lock_guard<std::mutex> lock(mu);
  const auto key = std::make_tuple(reinterpret_cast<const void*>(fn), n, dev);
  const auto it = known.find(key);
  if (it != known.end()) return it->second;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(n), cfg.blockDim = dim3(threads), cfg.dynamicSmemBytes = smem;
  cudaLaunchAttribute at{};
  at.id = cudaLaunchAttributeClusterDimension;
  at.val.clusterDim.x = n, at.val.clusterDim.y = 1, at.val.clusterDim.z = 1;
  cfg.attrs = &at, cfg.numAttrs = 1;
  int room = 0;
  if (n > 8) cudaFuncSetAttribute(reinterpret_cast<const void*>(fn), cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
  if (cudaOccupancyMaxActiveClusters(&room, reinterpret_cast<const void*>(fn), &cfg) != cudaSuccess) {
    cudaGetLastError();
    room = 0;
  }
  known[key] = room;
  return room;
}

struct Bytes {
  int tile, threads;
  size_t smem;
};
template <int LANES> Bytes bytes_of(const Form& f, int e) {
  const auto of = [&](auto shape, int tensors) {
    using S = decltype(shape);
    const size_t tile = f.aligned ? Tile<S, true>::kBytes : Tile<S, false>::kBytes;
    return Bytes{S::kTile, S::kThreads, 2 * tile * tensors + (e == 4 ? sizeof(Board<float, S>) : sizeof(Board<float2, S>))};
  };
  return f.back ? of(Bwd<LANES>{}, f.gate ? 4 : 3) : of(Fwd<LANES>{}, f.gate ? 3 : 2);
}

// step: a single token of each request, whose descriptor has no length.
int check_desc(const hyfft_gated_desc* d, const char* null_msg, bool step = false) {
  if (!d) return set_error(HYFFT_ERR_INVALID, null_msg);
  if (d->batch < 1 || (!step && d->length < 1) || d->channels < 1)
    return set_error(HYFFT_ERR_INVALID, "gated scan: every extent must be positive");
  if (d->dtype < HYFFT_F32 || d->dtype > HYFFT_F16) return set_error(HYFFT_ERR_INVALID, "gated scan: bad dtype");
  if (d->form != HYFFT_GATED_LOGIT && d->form != HYFFT_GATED_LOG)
    return set_error(HYFFT_ERR_INVALID, "gated scan: bad form");
  // token numbers and the cluster's tiles past the end are 32-bit
  if ((!step && d->length > (1ll << 30)) || d->channels > (1 << 28) || (long long)d->batch * ((d->channels + 31) / 32) > (1ll << 27))
    return set_error(HYFFT_ERR_UNSUPPORTED, "gated scan: too many tokens, channels or rows");
  return HYFFT_OK;
}

int run_scan(const hyfft_gated_desc* d, ScanArgs A, bool back, cudaStream_t st) {
  const int e = d->dtype == HYFFT_F32 ? 4 : 2;
  const bool gate = A.in[2] != nullptr;
  A.L = (int)d->length, A.C = d->channels, A.complement = d->complement ? 1 : 0;
  A.segments = (A.L + kSaved - 1) / kSaved;
  const int64_t* strides[4] = {d->x_stride, d->gate_stride, d->out_gate_stride, d->dy_stride};
  bool aligned = (long long)A.C * e % 4 == 0;
  for (int k = 0; k < 4; ++k) {
    if (!A.in[k]) continue;
    A.batch[k] = strides[k][0] * e, A.tok[k] = strides[k][1] * e;
    aligned = aligned && reinterpret_cast<uintptr_t>(A.in[k]) % 16 == 0 && A.batch[k] % 16 == 0 && A.tok[k] % 16 == 0;
  }
  for (int k = 0; k < 3; ++k) aligned = aligned && reinterpret_cast<uintptr_t>(A.out[k]) % 4 == 0;
  const Form form{back, d->form == HYFFT_GATED_LOG, gate, d->complement != 0, aligned};
  const auto rows_of = [&](int width) { return (long long)d->batch * (((long long)A.C * e + width - 1) / width); };
  // Few rows: half as wide ones, so twice as many, of tiles with twice the tokens, so half the hops. Measured, bfloat16 with output gates,
  // wide | narrow, us forwards and backwards: rows of 128 bytes 4 (1 x 65536 x 256): 248 | 127, 298 | 165; 16 (4 x 16384 x 256): 73 | 48, 92 | 86;
  // 32 (8 x 16384 x 256): 83 | 73, 127 | 147; 48 (3 x 8192 x 1024): 57 | 59, 99 | 141; 64 (1 x 65536 x 4096): 476 | 517, 921 | 1055. The same
  // rows in float32 (half the channels): 217 | 105, 208 | 126; 64 | 41, 70 | 70; 70 | 58, 97 | 116; 45 | 47, 78 | 114; 370 | 400, 692 | 848; in
  // bfloat16 without output gates: 238 | 126, 236 | 129; 68 | 43, 74 | 63; 77 | 57, 95 | 115; 45 | 47, 77 | 113; 355 | 395, 677 | 838. Rows of one
  // tile take the same rule (47 x 60 x 64: 6.3 | 8.2).
  const bool narrow = rows_of(128) < (back ? 24 : 48);
  const Kernel fn = narrow ? pick<16>(d->dtype, form) : pick<32>(d->dtype, form);
  const long long rows = rows_of(narrow ? 64 : 128);
  A.cols = (int)(rows / d->batch);
  const Bytes by = narrow ? bytes_of<16>(form, e) : bytes_of<32>(form, e);
  const int tile = by.tile, threads = by.threads;
  const size_t smem = by.smem;
  A.patience = g_wait_clocks.load(std::memory_order_relaxed);
  if (!kernel_smem_once(reinterpret_cast<const void*>(fn), smem, true))
    return set_error(HYFFT_ERR_CUDA, "gated scan: shared memory");
  // As many CTAs for a row as the machine can run at once for all rows, and as the row has tiles.
  int n = (int)std::min<long long>(kMaxCluster, (A.L + tile - 1) / tile);
  while (n > 1 && room_for(fn, n, threads, smem) < rows) --n;
  A.n = n;
  if (n > 1) {
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3((unsigned)(rows * n)), cfg.blockDim = dim3(threads), cfg.dynamicSmemBytes = smem, cfg.stream = st;
    cudaLaunchAttribute at{};
    at.id = cudaLaunchAttributeClusterDimension;
    at.val.clusterDim.x = n, at.val.clusterDim.y = 1, at.val.clusterDim.z = 1;
    cfg.attrs = &at, cfg.numAttrs = 1;
    if (cudaLaunchKernelEx(&cfg, fn, A) != cudaSuccess) {
      cudaGetLastError();
      return set_error(HYFFT_ERR_CUDA, "gated scan: kernel launch failed");
    }
  } else {
    fn<<<(unsigned)rows, threads, smem, st>>>(A);
  }
  if (cudaGetLastError() != cudaSuccess) return set_error(HYFFT_ERR_CUDA, "gated scan: kernel launch failed");
  g_launches.fetch_add(1, std::memory_order_relaxed);
  return HYFFT_OK;
}

template <typename T, bool LOG> int launch_step(StepArgs A, cudaStream_t st) {
  // 16 bytes of state and 4 elements at once where all rows start on their boundaries
  constexpr int V = 4;
  bool wide = A.C % V == 0 && A.xb % V == 0 && A.gb % V == 0 && (!A.o || A.ob % V == 0);
  for (const void* p : {A.x, A.g, A.o, (const void*)A.y}) wide = wide && reinterpret_cast<uintptr_t>(p) % (V * sizeof(T)) == 0;
  for (const void* p : {(const void*)A.state, (const void*)A.out_state}) wide = wide && reinterpret_cast<uintptr_t>(p) % 16 == 0;
  A.units = wide ? A.C / V : A.C;
  const long long ctas = ((long long)A.B * A.units + 255) / 256;
  if (ctas > 0x7fffffffLL) return set_error(HYFFT_ERR_UNSUPPORTED, "gated step: too many elements");
  if (wide)
    gated_step_kernel<T, LOG, V><<<(unsigned)ctas, 256, 0, st>>>(A);
  else
    gated_step_kernel<T, LOG, 1><<<(unsigned)ctas, 256, 0, st>>>(A);
  if (cudaGetLastError() != cudaSuccess) return set_error(HYFFT_ERR_CUDA, "gated step: kernel launch failed");
  g_launches.fetch_add(1, std::memory_order_relaxed);
  return HYFFT_OK;
}
template <typename T> int launch_step(const StepArgs& A, bool log, cudaStream_t st) {
  return log ? launch_step<T, true>(A, st) : launch_step<T, false>(A, st);
}

}  // namespace
}  // namespace hyfft

namespace hyfft {
int gated_wait_status(bool clear, unsigned* ran_out) { return read_ran_out(clear, ran_out) == cudaSuccess ? HYFFT_OK : HYFFT_ERR_CUDA; }
}  // namespace hyfft

using namespace hyfft;

extern "C" int hyfft_gated_saved_size(const hyfft_gated_desc* d, size_t* saved_bytes) {
  if (int rc = check_desc(d, "gated scan: null descriptor")) return rc;
  if (!saved_bytes) return set_error(HYFFT_ERR_INVALID, "gated scan: null size");
  *saved_bytes = sizeof(float) * (size_t)d->batch * (size_t)((d->length + kSaved - 1) / kSaved) * (size_t)d->channels;
  return HYFFT_OK;
}

extern "C" int hyfft_gated_forward(const hyfft_gated_desc* d, const void* x, const void* gate, const void* out_gate,
                                   const int32_t* lengths, const float* initial_state, void* y, float* final_state,
                                   void* saved, size_t saved_bytes, void* stream) {
  if (int rc = check_desc(d, "gated scan: null descriptor")) return rc;
  if (!x || !gate || !y) return set_error(HYFFT_ERR_INVALID, "gated scan: null tensor");
  size_t need = 0;
  if (int rc = hyfft_gated_saved_size(d, &need)) return rc;
  if (saved && saved_bytes < need) return set_error(HYFFT_ERR_WORKSPACE, "gated scan: saved buffer too small");
  if (bind_device_of(x) != HYFFT_OK) return set_error(HYFFT_ERR_CUDA, "gated scan: device");
  ScanArgs A{};
  A.in[0] = static_cast<const char*>(x), A.in[1] = static_cast<const char*>(gate);
  A.in[2] = static_cast<const char*>(out_gate);
  A.out[0] = static_cast<char*>(y);
  A.lengths = lengths, A.first = initial_state, A.last = final_state, A.saved = static_cast<float*>(saved);
  return run_scan(d, A, false, static_cast<cudaStream_t>(stream));
}

extern "C" int hyfft_gated_backward(const hyfft_gated_desc* d, const void* x, const void* gate, const void* out_gate,
                                    const int32_t* lengths, const void* saved, size_t saved_bytes, const void* dy,
                                    const float* dfinal_state, void* dx, void* dgate, void* dout_gate,
                                    float* dinitial_state, void* stream) {
  if (int rc = check_desc(d, "gated scan: null descriptor")) return rc;
  if (!x || !gate || !dy || !dx || !dgate || (out_gate && !dout_gate))
    return set_error(HYFFT_ERR_INVALID, "gated scan: null tensor");
  size_t need = 0;
  if (int rc = hyfft_gated_saved_size(d, &need)) return rc;
  if (!saved || saved_bytes < need) return set_error(HYFFT_ERR_WORKSPACE, "gated scan: saved buffer missing or too small");
  if (bind_device_of(x) != HYFFT_OK) return set_error(HYFFT_ERR_CUDA, "gated scan: device");
  ScanArgs A{};
  A.in[0] = static_cast<const char*>(x), A.in[1] = static_cast<const char*>(gate);
  A.in[2] = static_cast<const char*>(out_gate), A.in[3] = static_cast<const char*>(dy);
  A.out[0] = static_cast<char*>(dx), A.out[1] = static_cast<char*>(dgate);
  A.out[2] = out_gate ? static_cast<char*>(dout_gate) : nullptr;
  A.lengths = lengths, A.first = dfinal_state, A.last = dinitial_state;
  A.saved = const_cast<float*>(static_cast<const float*>(saved));
  return run_scan(d, A, true, static_cast<cudaStream_t>(stream));
}

extern "C" int hyfft_gated_step(const hyfft_gated_desc* d, const void* x, const void* gate, const void* out_gate,
                                const int32_t* slots, int64_t pool, const float* state, float* out_state, void* y,
                                void* stream) {
  if (int rc = check_desc(d, "gated step: null descriptor", true)) return rc;
  if (!x || !gate || !state || !out_state || !y) return set_error(HYFFT_ERR_INVALID, "gated step: null tensor");
  if (pool < 1 || (!slots && pool < d->batch)) return set_error(HYFFT_ERR_INVALID, "gated step: too few states");
  if (bind_device_of(x) != HYFFT_OK) return set_error(HYFFT_ERR_CUDA, "gated step: device");
  StepArgs A{};
  A.x = x, A.g = gate, A.o = out_gate, A.slots = slots, A.state = state, A.out_state = out_state, A.y = y;
  A.xb = d->x_stride[0], A.gb = d->gate_stride[0], A.ob = d->out_gate_stride[0];
  A.pool = pool, A.B = d->batch, A.C = d->channels, A.complement = d->complement ? 1 : 0;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const bool log = d->form == HYFFT_GATED_LOG;
  if (d->dtype == HYFFT_F32) return launch_step<float>(A, log, st);
  if (d->dtype == HYFFT_BF16) return launch_step<__nv_bfloat16>(A, log, st);
  return launch_step<__half>(A, log, st);
}
