// The decayed linear attention's scan on the tensor cores (tcgen05), bfloat16 operands, float32 state.
//
// A CTA walks over one row's tokens (or a segment of them) in chunks of 64 and keeps 64 columns of the state. With
// i, j the tokens of a chunk in scan order, n of them valid, S the state before it (e = 1 forwards, 0 backwards, where
// the decay is applied after a token's output):
//
//   P = Q K^T                      [64, 64]     masked and decayed: P_ij a^(i-j), j <= i
//   R = Q S                        [64, 64 columns]
//   o_i = a^(i+e) R_i + (P V)_i
//   S  <- a^n S + K^T (a^(n-j-e) V_j)
//
// All four products accumulate in float32 in TMEM. P and the copy of S that R reads are rounded to bfloat16 (each is
// one operand of one product: together with the output's own rounding the error is 1.4 times that of one rounding). The state
// itself is a result in float32, so the decayed V is not rounded: it is split into three bfloat16 terms (24 bits),
// three products into one accumulator; S lives in registers and takes the chunk's decay as the sum of two floats.
//
// Operand tiles sit in shared memory as 8 x 16-byte core matrices, [D / 8][tokens / 8][8][16 B], which the tensor core
// reads along either axis, so K serves as K^T and V, S as they lie. cp.async brings them in (zeros past a length, a row or a
// head size), K and V of the next chunk while this one is computed, Q as soon as P and R are done. Two CTAs of 256 threads
// share an SM (<= 112 KB, 256 TMEM columns each) so that one's products run under the other's epilogues.
#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include <atomic>

#include "../../include/hyfft.h"
#include "common.cuh"
#include "decay_attn.h"
#include "umma.cuh"

namespace hyfft {

extern std::atomic<long long> g_launches;
int set_error(int code, const char* msg);  // engine.cu: the message hyfft_last_error returns

namespace {

using bf16 = __nv_bfloat16;

constexpr int kT = kMmaTok, kC = kMmaCols;
constexpr int kThreads = 256;
constexpr int kColP = 0, kColR = 64, kColO = 128, kColS = 192, kTmemCols = 256;

// Bytes of the shared-memory layout for a state of DK (64 or 128) rows.
template <int DK, bool OUT>
struct Layout {
  static constexpr int qk = DK * kT * 2, v = kC * kT * 2;
  static constexpr int q = 0;
  static constexpr int k = q + (OUT ? qk : 0);
  static constexpr int vv = k + 2 * qk;
  static constexpr int w = vv + 2 * v;                 // the decayed V in three terms
  static constexpr int p = w + 3 * v;                  // P
  static constexpr int s = p + (OUT ? kT * kT * 2 : 0);  // the rounded state
  static constexpr int tab = s + (OUT ? DK * kC * 2 : 0);  // a^d for d = -64 .. 64 (zeros below 0)
  static constexpr int bar = tab + (2 * kT + 4) * 4;
  static constexpr int bytes = bar + 64;
};

__device__ __forceinline__ void cp16(uint32_t dst, const void* src, bool valid) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;\n" ::"r"(dst), "l"(src), "r"(valid ? 16 : 0) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;\n" ::: "memory"); }
__device__ __forceinline__ void cp_wait() { asm volatile("cp.async.wait_group 0;\n" ::: "memory"); }

__device__ __forceinline__ uint32_t pack2(float a, float b) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ float2 unpack2(uint32_t u) {
  return make_float2(__uint_as_float(u << 16), __uint_as_float(u & 0xffff0000u));
}

// Columns [c0, c0 + W) of n tokens (scan order from token t0) into a tile of kT tokens, zeros past n and past D.
template <int W>
__device__ __forceinline__ void load_tile(unsigned char* dst, const bf16* __restrict__ src, long long sl, int n, int c0,
                                          int D, long long t0, int step, bool vec) {
  // a quarter warp writes 8 tokens of one 16-byte column (128 contiguous bytes); a warp reads 64 bytes of each token
  for (int i = threadIdx.x; i < kT * W / 8; i += kThreads) {
    const int r = i & 7, j = ((i >> 3) & 3) | ((i / (kT * 4)) << 2), t = ((i >> 5) % (kT / 8)) * 8 + r;
    const int c = c0 + j * 8;
    unsigned char* d = dst + j * (kT * 16) + t * 16;
    const bool ok = t < n && c < D;
    const bf16* s = src + (t0 + (long long)(ok ? t : 0) * step) * sl + (ok ? c : 0);
    if (vec) {
      cp16(umma::su32(d), s, ok);
    } else {
      uint4 u = make_uint4(0, 0, 0, 0);
      bf16* e = reinterpret_cast<bf16*>(&u);
      if (ok)
#pragma unroll
        for (int x = 0; x < 8; ++x)
          if (c + x < D) e[x] = s[x];
      *reinterpret_cast<uint4*>(d) = u;
    }
  }
}

__device__ __forceinline__ void tmem_ld32(uint32_t a, float (&v)[32]) {
  uint32_t r[32];
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,"
      "%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];\n"
      "tcgen05.wait::ld.sync.aligned;\n"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
        "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
        "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(a)
      : "memory");
#pragma unroll
  for (int i = 0; i < 32; ++i) v[i] = __uint_as_float(r[i]);
}

// OUT: the pass with outputs; without it, segments' sums alone (K and V only).
template <int DK, bool OUT, typename TO>
__global__ void __launch_bounds__(kThreads, 2) decay_mma_kernel(const ScanArgs A) {
  using L = Layout<DK, OUT>;
  extern __shared__ __align__(1024) unsigned char smem[];
  float* tab = reinterpret_cast<float*>(smem + L::tab);
  uint64_t* bar = reinterpret_cast<uint64_t*>(smem + L::bar);  // P and R; K^T V; P V
  uint32_t* tslot = reinterpret_cast<uint32_t*>(smem + L::bar + 32);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;

  long long id = blockIdx.x;
  const int slice = (int)(id % A.nslice);
  id /= A.nslice;
  const int seg = (int)(id % A.nseg);
  const long long bh = id / A.nseg;
  const int h = (int)(bh % A.H);
  const long long b = bh / A.H;
  const int c0 = slice * kC;

  int len = A.L;
  if (A.lengths) len = min(max(A.lengths[b], 0), A.L);
  const long long t_lo = (long long)seg * A.seglen;
  const long long t_end = min(t_lo + A.seglen, (long long)A.L);
  const long long t_hi = min(t_end, (long long)len);
  const int n_all = t_hi > t_lo ? (int)(t_hi - t_lo) : 0;
  const int step = A.reverse ? -1 : 1;
  const long long t_first = A.reverse ? t_hi - 1 : t_lo;
  const int lag = A.reverse ? 0 : 1;

  const bf16* qp = static_cast<const bf16*>(A.q.p) + b * A.q.sb + (long long)(h / A.q.group) * A.q.sh;
  const bf16* kp = static_cast<const bf16*>(A.k.p) + b * A.k.sb + (long long)(h / A.k.group) * A.k.sh;
  const bf16* vp = static_cast<const bf16*>(A.v.p) + b * A.v.sb + (long long)(h / A.v.group) * A.v.sh;

  if (n_all > 0) {
    const int n = min(kT, n_all);
    if (OUT) load_tile<DK>(smem + L::q, qp, A.q.sl, n, 0, A.DK, t_first, step, A.vec);
    load_tile<DK>(smem + L::k, kp, A.k.sl, n, 0, A.DK, t_first, step, A.vec);
    load_tile<kC>(smem + L::vv, vp, A.v.sl, n, c0, A.DV, t_first, step, A.vec);
  }
  cp_commit();
  if (warp == 0) umma::tmem_alloc(tslot, kTmemCols);
  if (tid == 0) {
    for (int i = 0; i < 3; ++i) umma::mbar_init(&bar[i], 1);
    umma::fence_mbar_init();
  }
  const double g = (double)A.log_decay[h];
  if (tid <= 2 * kT) tab[tid] = tid < kT ? 0.f : tid == kT ? 1.f : (float)exp(g * (tid - kT));
  const float a64hi = (float)exp(g * kT), a64lo = (float)(exp(g * kT) - (double)a64hi);

  // This thread's part of the state: one row and 32 columns. Rows of a 64-row product lie in lanes 0 .. 15 of each warp.
  const int wq = warp & 3, half = (warp >> 2) * 32;
  const int srow = DK == 128 ? wq * 32 + lane : wq * 16 + lane;
  const int trow = wq * 16 + lane;  // and of a 64-token product
  const bool sact = DK == 128 || lane < 16, tact = lane < 16;
  float S[32];
#pragma unroll
  for (int c = 0; c < 32; ++c) S[c] = 0.f;
  const long long per_state = (long long)A.DK * A.DV;
  if (OUT && sact && srow < A.DK) {
    const float* src = nullptr;
    long long sr = A.DV, sc = 1;
    if (A.nseg > 1) {
      src = A.seg + (bh * A.nseg + seg) * per_state;
    } else if (A.start) {
      src = A.start + bh * per_state;
      sr = A.srow, sc = A.scol;
    }
    if (src)
#pragma unroll
      for (int c = 0; c < 32; ++c)
        if (c0 + half + c < A.DV) S[c] = src[srow * sr + (c0 + half + c) * sc];
  }
  if (OUT && sact) {
    unsigned char* d = smem + L::s + srow * 16;
#pragma unroll
    for (int j = 0; j < 4; ++j)
      *reinterpret_cast<uint4*>(d + (half / 8 + j) * (DK * 16)) =
          make_uint4(pack2(S[8 * j], S[8 * j + 1]), pack2(S[8 * j + 2], S[8 * j + 3]), pack2(S[8 * j + 4], S[8 * j + 5]),
                     pack2(S[8 * j + 6], S[8 * j + 7]));
  }
  __syncthreads();
  umma::fence_after_sync();
  const uint32_t tmem = *tslot;
  const uint32_t lanes = tmem + ((uint32_t)(wq * 32) << 16);
  const uint32_t sq = umma::su32(smem + L::q), sk0 = umma::su32(smem + L::k), sv0 = umma::su32(smem + L::vv);
  const uint32_t sw = umma::su32(smem + L::w), sp = umma::su32(smem + L::p), ss = umma::su32(smem + L::s);
  constexpr uint32_t kIdP = umma::idesc_bf16(kT, kT, 0, 0);
  constexpr uint32_t kIdR = umma::idesc_bf16(kT, kC, 0, 1);
  constexpr uint32_t kIdS = umma::idesc_bf16(DK, kC, 1, 1);
  TO* op = static_cast<TO*>(A.o) + (OUT ? b * A.ob + (long long)h * A.oh + c0 : 0);
  bool ok = true;

  int it = 0;
  for (int i0 = 0; i0 < n_all; i0 += kT, ++it) {
    const int n = min(kT, n_all - i0), buf = it & 1;
    const uint32_t sk = sk0 + buf * L::qk, sv = sv0 + buf * L::v;
    const int nn = min(kT, n_all - i0 - kT);  // tokens of the next chunk
    const long long t0 = t_first + (long long)i0 * step, t1 = t0 + (long long)kT * step;
    cp_wait();
    umma::fence_async_smem();
    umma::fence_before_sync();
    __syncthreads();  // this chunk's operands and the state are in place; the last chunk's accumulators have been read
    if (OUT && tid == 0) {
      umma::fence_after_sync();
#pragma unroll
      for (int x = 0; x < DK / 16; ++x)
        umma::mma(tmem + kColP, umma::sdesc(sq + x * 2 * kT * 16, kT * 16, 128), umma::sdesc(sk + x * 2 * kT * 16, kT * 16, 128),
                  kIdP, x > 0);
#pragma unroll
      for (int x = 0; x < DK / 16; ++x)
        umma::mma(tmem + kColR, umma::sdesc(sq + x * 2 * kT * 16, kT * 16, 128), umma::sdesc(ss + x * 256, 128, DK * 16), kIdR,
                  x > 0);
      umma::commit(&bar[0]);
    }
    if (nn > 0) {
      load_tile<DK>(smem + L::k + (buf ^ 1) * L::qk, kp, A.k.sl, nn, 0, A.DK, t1, step, A.vec);
      load_tile<kC>(smem + L::vv + (buf ^ 1) * L::v, vp, A.v.sl, nn, c0, A.DV, t1, step, A.vec);
    }
    cp_commit();
    // the decayed V, in three terms
    for (int i = tid; i < kT * kC / 8; i += kThreads) {
      const int t = i & (kT - 1);
      const float w = t < n ? tab[kT + n - t - lag] * A.vscale : 0.f;
      const uint4 u = *reinterpret_cast<const uint4*>(smem + L::vv + buf * L::v + i * 16);
      uint4 hi, mid, lo;
      const uint32_t* up = &u.x;
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        float2 f = unpack2(up[x]);
        f.x *= w, f.y *= w;
        const uint32_t a = pack2(f.x, f.y);
        const float2 fa = unpack2(a);
        f.x -= fa.x, f.y -= fa.y;
        const uint32_t c = pack2(f.x, f.y);
        const float2 fc = unpack2(c);
        (&hi.x)[x] = a, (&mid.x)[x] = c, (&lo.x)[x] = pack2(f.x - fc.x, f.y - fc.y);
      }
      *reinterpret_cast<uint4*>(smem + L::w + i * 16) = hi;
      *reinterpret_cast<uint4*>(smem + L::w + L::v + i * 16) = mid;
      *reinterpret_cast<uint4*>(smem + L::w + 2 * L::v + i * 16) = lo;
    }
    umma::fence_async_smem();
    __syncthreads();
    if (tid == 0) {
      umma::fence_after_sync();
#pragma unroll
      for (int y = 0; y < 3; ++y)
#pragma unroll
        for (int x = 0; x < kT / 16; ++x)
          umma::mma(tmem + kColS, umma::sdesc(sk + x * 256, 128, kT * 16), umma::sdesc(sw + y * L::v + x * 256, 128, kT * 16),
                    kIdS, x + y > 0);
      umma::commit(&bar[1]);
    }
    if (OUT) {
      ok &= umma::mbar_wait(&bar[0], it & 1);
      umma::fence_after_sync();
      if (nn > 0) load_tile<DK>(smem + L::q, qp, A.q.sl, nn, 0, A.DK, t1, step, A.vec);
      cp_commit();
      float p[32];
      tmem_ld32(lanes + kColP + half, p);
      if (tact) {
        const float* tb = tab + kT + trow - half;
        unsigned char* d = smem + L::p + (half / 8) * (kT * 16) + trow * 16;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          uint4 u;
#pragma unroll
          for (int x = 0; x < 4; ++x) {
            const int c = 8 * j + 2 * x;
            (&u.x)[x] = pack2(p[c] * tb[-c], p[c + 1] * tb[-c - 1]);
          }
          *reinterpret_cast<uint4*>(d + j * (kT * 16)) = u;
        }
      }
      umma::fence_async_smem();
      umma::fence_before_sync();
      __syncthreads();
      if (tid == 0) {
        umma::fence_after_sync();
#pragma unroll
        for (int x = 0; x < kT / 16; ++x)
          umma::mma(tmem + kColO, umma::sdesc(sp + x * 2 * kT * 16, kT * 16, 128), umma::sdesc(sv + x * 256, 128, kT * 16), kIdR,
                    x > 0);
        umma::commit(&bar[2]);
      }
    }
    // the state
    ok &= umma::mbar_wait(&bar[1], it & 1);
    umma::fence_after_sync();
    {
      float d[32];
      tmem_ld32(lanes + kColS + half, d);
      float hi = a64hi, lo = a64lo;
      if (n != kT) {
        const double an = exp(g * n);
        hi = (float)an, lo = (float)(an - (double)hi);
      }
#pragma unroll
      for (int c = 0; c < 32; ++c) S[c] = fmaf(S[c], hi, fmaf(S[c], lo, d[c]));
      if (OUT && sact) {
        unsigned char* t = smem + L::s + srow * 16;
#pragma unroll
        for (int j = 0; j < 4; ++j)
          *reinterpret_cast<uint4*>(t + (half / 8 + j) * (DK * 16)) =
              make_uint4(pack2(S[8 * j], S[8 * j + 1]), pack2(S[8 * j + 2], S[8 * j + 3]),
                         pack2(S[8 * j + 4], S[8 * j + 5]), pack2(S[8 * j + 6], S[8 * j + 7]));
      }
    }
    if (OUT) {
      ok &= umma::mbar_wait(&bar[2], it & 1);
      umma::fence_after_sync();
      float r[32], o[32];
      tmem_ld32(lanes + kColR + half, r);
      tmem_ld32(lanes + kColO + half, o);
      if (tact && trow < n) {
        const float rs = tab[kT + trow + lag] * A.oscale, os = A.vscale * A.oscale;
        TO* d = op + (t0 + (long long)trow * step) * A.ol + half;
        const int left = A.DV - c0 - half;
#pragma unroll
        for (int c = 0; c < 32; ++c) o[c] = ok ? fmaf(r[c], rs, o[c] * os) : __int_as_float(0x7fffffff);
        if (A.ovec && left >= 32) {
          if constexpr (sizeof(TO) == 2) {
#pragma unroll
            for (int j = 0; j < 4; ++j)
              reinterpret_cast<uint4*>(d)[j] =
                  make_uint4(pack2(o[8 * j], o[8 * j + 1]), pack2(o[8 * j + 2], o[8 * j + 3]),
                             pack2(o[8 * j + 4], o[8 * j + 5]), pack2(o[8 * j + 6], o[8 * j + 7]));
          } else {
#pragma unroll
            for (int j = 0; j < 8; ++j)
              reinterpret_cast<float4*>(d)[j] = make_float4(o[4 * j], o[4 * j + 1], o[4 * j + 2], o[4 * j + 3]);
          }
        } else {
#pragma unroll
          for (int c = 0; c < 32; ++c)
            if (c < left) DT<TO>::store(d + c, o[c]);
        }
      }
    }
  }
  cp_wait();

  if (OUT) {  // tokens past the length: zeros
    const long long z0 = max(t_lo, t_hi);
    for (long long i = tid; i < (t_end - z0) * kC; i += kThreads) {
      const long long r = i / kC;
      const int c = (int)(i - r * kC);
      if (c0 + c < A.DV) DT<TO>::store(op + (z0 + r) * A.ol + c, 0.f);
    }
  }
  if (sact && srow < A.DK) {
    float* dst = nullptr;
    long long sr = A.DV, sc = 1;
    if (!OUT) {
      dst = A.seg + (bh * A.nseg + seg) * per_state;
    } else if (A.nseg == 1 && A.finish) {
      dst = A.finish + bh * per_state;
      sr = A.srow, sc = A.scol;
    }
    if (dst)
#pragma unroll
      for (int c = 0; c < 32; ++c)
        if (c0 + half + c < A.DV) dst[srow * sr + (c0 + half + c) * sc] = ok ? S[c] : __int_as_float(0x7fffffff);
  }
  umma::fence_before_sync();
  __syncthreads();
  if (warp == 0) umma::tmem_dealloc(tmem, kTmemCols);
}

template <int DK, bool OUT, typename TO>
int launch(const ScanArgs& A, long long ctas, cudaStream_t st) {
  auto kern = decay_mma_kernel<DK, OUT, TO>;
  constexpr size_t sm = Layout<DK, OUT>::bytes;
  if (!kernel_smem_once((const void*)kern, sm, true)) return set_error(HYFFT_ERR_CUDA, "decay attention: shared memory");
  kern<<<(unsigned)ctas, kThreads, sm, st>>>(A);
  if (cudaGetLastError() != cudaSuccess) return set_error(HYFFT_ERR_CUDA, "decay attention: kernel launch failed");
  g_launches.fetch_add(1, std::memory_order_relaxed);
  return HYFFT_OK;
}

template <int DK>
int launch_dk(const ScanArgs& A, bool out_f32, long long ctas, cudaStream_t st) {
  if (!A.o) return launch<DK, false, bf16>(A, ctas, st);
  return out_f32 ? launch<DK, true, float>(A, ctas, st) : launch<DK, true, bf16>(A, ctas, st);
}

}  // namespace

int launch_scan_mma(const ScanArgs& A, bool out_f32, long long ctas, cudaStream_t st) {
  if (ctas > 0x7fffffffLL) return set_error(HYFFT_ERR_UNSUPPORTED, "decay attention: too many rows");
  return A.DK <= 64 ? launch_dk<64>(A, out_f32, ctas, st) : launch_dk<128>(A, out_f32, ctas, st);
}

}  // namespace hyfft
