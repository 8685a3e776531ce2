// The decayed linear attention's scan on the tensor cores (tcgen05), bfloat16 operands, float32 state.
//
// float16 and float32 operands come as sums of NT = 2 and 3 bfloat16 terms (8 bits each; a small kernel lays them out
// first, NT = 1 below is bfloat16 itself). A product of two sums runs the pairs of terms whose order is below NT, 3 or 6 of
// them, into one float32 accumulator, and what the kernel rounds for a product (P, the state's copy) it keeps to NT terms too, so
// float32 results are float32's (16 x 4096 tokens, 12 heads of 64: 0.62 ms, multiply-adds take 1.06; float16 0.46 and 1.04).
// The tensor cores' own float16 would do with fewer products but not hold a state beyond 65504.
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
// All four products accumulate in float32 in TMEM. P and the copy of S that R reads are operands of bfloat16 products too: of
// bfloat16 tensors they are kept as two terms (16 bits), so that the one error that shows in an output is its own
// rounding (one term each made it 1.4 times as large). The state
// itself is a result in float32, so the decayed V is not rounded: it is split into three bfloat16 terms (24 bits),
// three products into one accumulator; S lives in registers and takes the chunk's decay as the sum of two floats.
//
// Operand tiles sit in shared memory as rows of 128 bytes (64 columns of a token, or of a row of P or S) whose 16-byte
// chunks are swizzled by the row's number (chunk ^ row % 8). The tensor core reads such a tile along either axis, so K serves
// as K^T and V, S as they lie; and both halves of a 32-byte sector stay neighbours, which tiles of 8 x 16-byte core
// matrices did not give: cp.async then fetched every sector twice. Rows are in the order of time in either direction.
// Sixteen warps: three load (TMA; the last, partial chunk and tensors that TMA cannot take by cp.async, with zeros past a
// length or a head size; two take turns with K and V, one brings Q), one issues the products, eight compute: they decay P,
// update the state and split the next chunk's V; four write the outputs. Only mbarriers order them. The computing warps' chain
// of TMEM reads, shared-memory writes and barriers sets the pace, so what need not be in it is not (a pass with outputs
// over the 128 x 128 grid, 32 rows of 16384 tokens of 64, with P and the state's copy as one term: 134 us with eight warps
// doing everything, 69 with loads and products issued by others, 58 with the outputs written by others too, Q in several buffers
// and no register spilled; as two terms 72; its traffic at the copy's rate takes 41).
// A result that is infinite or NaN is computed again at the end, token by token in scan order (scan_by_token).
// Registers move from the loading to the computing warps. Two CTAs share an SM (<= 113 KB, 256 TMEM columns each).
//
// 64-row products lie in 16 of a warp's 32 TMEM lanes, and the 16 x 256-bit load shape spreads those over all 32 threads
// (two rows, pairs of columns).
#include <cuda.h>
#include <cudaTypedefs.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <atomic>
#include <mutex>
#include <type_traits>

#include "../../include/hyfft.h"
#include "common.cuh"
#include "decay_attn.h"
#include "umma.cuh"
#include "waits.cuh"

namespace hyfft {

extern std::atomic<long long> g_launches;
int set_error(int code, const char* msg);  // engine.cu: the message hyfft_last_error returns

namespace {

using bf16 = __nv_bfloat16;

constexpr int kT = kMmaTok, kC = kMmaCols;
constexpr int kThreads = 256;  // computing
constexpr int kLoader = kThreads / 32, kIssuer = kLoader + 3;  // first loading warp, issuing warp
constexpr int kWriter = kIssuer + 1, kWriters = 4;
constexpr int kAll = 32 * (kWriter + kWriters);
// Registers of a thread: computing, loading and issuing, writing; together those of the launch (64 for each of 512). Chosen
// so that little spills (bfloat16 heads of 64: nothing): with the shared memory that is taken here a spilled register comes
// back from L2.
// Where all warps have something to run at the end, they take the launch's 64 again: after a barrier, since a warp that
// did so before the computing warps have got their registers would leave them waiting forever.
template <int DK, bool OUT>
struct Regs {
  static constexpr int compute = DK == 64 && OUT ? 72 : 80, load = DK == 64 && OUT ? 56 : 48, write = load;
  static constexpr int launch = 64;
  static_assert(kThreads * compute + 128 * load + 128 * write <= launch * kAll, "setmaxnreg would wait forever");
};
constexpr int kColP = 0, kColR = 64, kColO = 128, kColS = 192, kTmemCols = 256;  // kColS - 64: a second one without outputs

// What each mbarrier says: full for the loads, done by the tensor core, the others by the warps. One commit tells all that
// wait for a product, the loading warps too: a second commit behind it held the issuing warp for a thousand cycles.
// A barrier with two phases behind its waiter cannot be told from one with none: where a waiter may fall behind (several
// buffers in use), each buffer has its own.
enum Bar {
  kFull = 0,     // K and V of a buffer are in place
  kFullQ = 4,    // Q of a buffer
  kDoneR = 7,    // R is there, Q (of a buffer) and the rounded state have been read
  kDoneO = 10,   // P V is there, K and V of a buffer have been read
  kDoneS = 14,   // K^T V is there (without outputs: K and V of a buffer have been read)
  kDoneP = 18,
  kHaveV = 19,   // the decayed V is in place, of buffer 0, 1
  kHaveS = 21,   // the rounded state is in place, the accumulator of buffer 0, 1 free
  kHaveP = 23,   // P is in place (and its accumulator free)
  kReadO = 24,   // R and P V have been read, by the writing warps
  kDrain = 25,   // all products are over; after a wait that ran out
  kBars = 26
};
// Words behind the barriers: the TMEM address, whether a wait has run out (or the tiles lie off the swizzle's pattern), and the
// last chunk that each loading warp brought (two of K and V, one of Q; -1: none).
enum Word { kTmem = 0, kFailed = 1, kLast = 2, kOdd = 5, kWords = 6 };  // kOdd: a result is infinite or NaN

// Bytes of the shared-memory layout for a state of DK (64 or 128) rows, operands of NT terms, a state update from TERMS
// terms of the decayed V. Tiles start on 1024 bytes, where the swizzle's pattern does.
constexpr int kTile = kT * 128;
// Terms of what a pass rounds itself, P and the state's copy: 16 bits at least.
constexpr int round_terms(int nt) { return nt == 1 ? 2 : nt; }
template <int DK, bool OUT, int NT, int TERMS>
struct Layout {
  static constexpr int RT = round_terms(NT);
  static constexpr bool two = NT == 1 || (NT == 2 && DK == 64);  // CTAs on an SM
  static constexpr int qk = NT * DK / 64 * kTile, vt = NT * kTile;
  // as many buffers of K and V, of Q and of the decayed V as there is room for (bfloat16 heads of 128 with outputs: one of each
  // and two CTAs; one CTA with four is slower, 8 heads of 65536 tokens 303 us against 295)
  static constexpr int nbuf = NT == 1 ? (OUT ? (DK == 64 ? (TERMS == 2 ? 3 : 2) : 1) : (DK == 64 ? 4 : 2))
                                      : (OUT ? (NT == 3 && DK == 64 ? 2 : 1) : (NT == 3 && DK == 64 ? 3 : 2));
  static constexpr int qbuf = NT == 1 && DK == 64 ? (TERMS == 2 ? 2 : 3) : 1;
  static constexpr int wbuf = OUT || (NT == 2 && DK == 64) ? 1 : 2;
  static constexpr int q = 0;
  static constexpr int k = q + (OUT ? qbuf * qk : 0);
  static constexpr int v = k + nbuf * qk;
  static constexpr int w = v + nbuf * vt;                    // the decayed V
  static constexpr int p = w + wbuf * TERMS * kTile;         // P
  static constexpr int s = p + (OUT ? RT * kTile : 0);       // the state in RT terms
  static constexpr int tab = s + (OUT ? RT * DK * 128 : 0);  // a^d for d = -64 .. 64 (zeros below 0)
  static constexpr int bar = tab + (2 * kT + 4) * 4;
  static constexpr int bytes = bar + kBars * 8 + kWords * 4;
  static_assert((two ? 2 : 1) * (bytes + 1024) <= 228 * 1024 && bytes <= 227 * 1024, "does not fit an SM");
};
// Byte of column c (even) of a row in a swizzled tile of 64 columns.
__device__ __forceinline__ int swz(int row, int c) { return row * 128 + ((((c >> 3) ^ row) & 7) << 4) + (c & 7) * 2; }
// Descriptor of a swizzled tile, as two words of which only the low one depends on the address. Rows along M or N, 64
// columns along K: groups of 8 rows 1024 bytes apart, 32 bytes for each 16 columns. Rows along K, columns along M or N:
// groups of 8 rows 1024 bytes apart (2048 for each 16 rows), blocks of 64 columns a tile apart.
constexpr uint32_t kDescHigh = (1024u >> 4) | (1u << 14) | (2u << 29);
__device__ __forceinline__ uint32_t desc_low(const void* p) {
  return (umma::su32(p) >> 4) | ((uint32_t)(kTile >> 4) << 16);
}
constexpr int kAlongK = 32 >> 4, kAlongRows = 2048 >> 4, kNextTile = kTile >> 4;  // steps of the low word
__device__ __forceinline__ void mma(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc, bool add) {
  asm volatile(
      "{\n.reg .pred p;\n.reg .b64 da, db;\nmov.b64 da, {%1, %5};\nmov.b64 db, {%2, %5};\nsetp.ne.b32 p, %4, 0;\n"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], da, db, %3, p;\n}\n" ::"r"(d),
      "r"(a), "r"(b), "r"(idesc), "r"((uint32_t)add), "n"(kDescHigh)
      : "memory");
}

__device__ __forceinline__ void cp16(uint32_t dst, const void* src, bool valid) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;\n" ::"r"(dst), "l"(src), "r"(valid ? 16 : 0) : "memory");
}
__device__ __forceinline__ void cp_wait() { asm volatile("cp.async.wait_all;\n" ::: "memory"); }

__device__ __forceinline__ void arrive(uint64_t* bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(umma::su32(bar)) : "memory");
}
// This warp's shared-memory writes and TMEM reads are over; the writes are visible to the tensor core.
__device__ __forceinline__ void hand_over(uint64_t* bar) {
  umma::fence_async_smem();
  umma::fence_before_sync();
  __syncwarp();
  if ((threadIdx.x & 31) == 0) arrive(bar);
}
__device__ __forceinline__ bool elect() {
  uint32_t p;
  asm volatile("{\n.reg .pred q;\nelect.sync _|q, 0xffffffff;\nselp.u32 %0, 1, 0, q;\n}\n" : "=r"(p));
  return p != 0;
}

// Lanes `by` apart exchange: the lane whose bit is clear keeps a and gives b, the other keeps b and gives a.
__device__ __forceinline__ void swap_pairs(uint32_t& a, uint32_t& b, int by, int lane) {
  const bool up = lane & by;
  const uint32_t got = __shfl_xor_sync(0xffffffffu, up ? a : b, by);
  if (up)
    a = got;
  else
    b = got;
}

__device__ __forceinline__ uint32_t pack2(float a, float b) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}
template <typename TO>
__device__ __forceinline__ uint32_t pack_out(float2 f) {
  if constexpr (std::is_same<TO, __half>::value) {
    const __half2 h = __floats2half2_rn(f.x, f.y);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
  return pack2(f.x, f.y);
}
__device__ __forceinline__ float2 unpack2(uint32_t u) {
  return make_float2(__uint_as_float(u << 16), __uint_as_float(u & 0xffff0000u));
}

// Maps of q, k, v as [batch, token, head, feature], boxes of 64 tokens x 64 features of one head.
struct Maps {
  CUtensorMap q, k, v;
  int on;
};

// Columns [c0, c0 + W) of 64 tokens from t0 on, all of them inside the sequence, by TMA; one lane.
template <int W>
__device__ __forceinline__ void load_box(uint32_t dst, const CUtensorMap* map, uint64_t* bar, int c0, int head, int t0, int b) {
#pragma unroll
  for (int x = 0; x < W / 64; ++x)
    asm volatile(
        "cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];" ::
            "r"(dst + x * kTile), "l"(map), "r"(c0 + 64 * x), "r"(head), "r"(t0), "r"(b), "r"(umma::su32(bar))
        : "memory");
}
__device__ __forceinline__ void expect(uint64_t* bar, int bytes) {
  asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(umma::su32(bar)), "r"(bytes) : "memory");
}

// Columns [c0, c0 + W) of n tokens from t0 on into tiles of kT tokens x 64 columns, zeros past n and past D.
// One warp: eight lanes copy 128 bytes of a token. Addresses advance by constants: recomputed for each copy they held a
// loading warp up for 180 cycles a copy.
template <int W>
__device__ __forceinline__ void load_tile(unsigned char* dst, const bf16* __restrict__ src, long long sl, int n, int c0,
                                          int D, long long t0, bool vec) {
  const int lane = threadIdx.x & 31, j = lane & 7, r = lane >> 3;
  const int c = c0 + j * 8;
  const bf16* s = src + (t0 + r) * sl + c;
  const long long jump = 4 * sl;
  // rows r + 4 m: their chunk's place alternates between two
  const int at0 = r * 128 + ((j ^ r) << 4), at1 = (r + 4) * 128 + ((j ^ (r + 4)) << 4);
  if (vec) {
    const uint32_t d0 = umma::su32(dst + at0), d1 = umma::su32(dst + at1);
#pragma unroll
    for (int t = 0; t < kT; t += 4) {
#pragma unroll
      for (int x = 0; x < W / 64; ++x) {
        const bool ok = t + r < n && c + 64 * x < D;
        cp16((t & 4 ? d1 : d0) + (t >> 3) * 1024 + x * kTile, ok ? s + 64 * x : src, ok);
      }
      s += jump;
    }
  } else {
    for (int t = 0; t < kT; t += 4) {
#pragma unroll
      for (int x = 0; x < W / 64; ++x) {
        uint4 u = make_uint4(0, 0, 0, 0);
        bf16* e = reinterpret_cast<bf16*>(&u);
        if (t + r < n)
#pragma unroll
          for (int y = 0; y < 8; ++y)
            if (c + 64 * x + y < D) e[y] = s[64 * x + y];
        *reinterpret_cast<uint4*>(dst + (t & 4 ? at1 : at0) + (t >> 3) * 1024 + x * kTile) = u;
      }
      s += jump;
    }
  }
}

// Two neighbouring values of a tile row in NT terms, the terms `apart` bytes from each other.
template <int NT>
__device__ __forceinline__ void put_terms(unsigned char* d, int apart, float2 f) {
#pragma unroll
  for (int y = 0; y < NT; ++y) {
    const uint32_t u = pack2(f.x, f.y);
    *reinterpret_cast<uint32_t*>(d + y * apart) = u;
    if (y + 1 < NT) f = csub(f, unpack2(u));
  }
}
// 16 TMEM lanes x 32 columns over a warp: register 4 j + 2 y + x holds row lane / 4 + 8 y, column 8 j + 2 (lane % 4) + x.
__device__ __forceinline__ void tmem_ld(uint32_t a, uint32_t (&u)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.16x256b.x4.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];\n"
      "tcgen05.wait::ld.sync.aligned;\n"
      : "=r"(u[0]), "=r"(u[1]), "=r"(u[2]), "=r"(u[3]), "=r"(u[4]), "=r"(u[5]), "=r"(u[6]), "=r"(u[7]), "=r"(u[8]),
        "=r"(u[9]), "=r"(u[10]), "=r"(u[11]), "=r"(u[12]), "=r"(u[13]), "=r"(u[14]), "=r"(u[15])
      : "r"(a)
      : "memory");
}
__device__ __forceinline__ void tmem_ld2(uint32_t a, uint32_t b, uint32_t (&u)[16], uint32_t (&v)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.16x256b.x4.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%32];\n"
      "tcgen05.ld.sync.aligned.16x256b.x4.b32 {%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%33];\n"
      "tcgen05.wait::ld.sync.aligned;\n"
      : "=r"(u[0]), "=r"(u[1]), "=r"(u[2]), "=r"(u[3]), "=r"(u[4]), "=r"(u[5]), "=r"(u[6]), "=r"(u[7]), "=r"(u[8]),
        "=r"(u[9]), "=r"(u[10]), "=r"(u[11]), "=r"(u[12]), "=r"(u[13]), "=r"(u[14]), "=r"(u[15]),
        "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]),
        "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15])
      : "r"(a), "r"(b)
      : "memory");
}

// The products of a sum of na terms and one of nb: the pairs whose order (the terms' numbers added) is below `orders`, the
// smallest products first. The accumulator cuts off below its last bit at every step, so steps at the full size are to be few
// (largest first, float32 outputs were off by 1.2e-6 of their norm instead of 1.3e-7).
constexpr int term_a(int y, int na, int nb, int orders) {
  for (int o = orders - 1; o >= 0; --o)
    for (int a = 0; a < na; ++a)
      if (o - a >= 0 && o - a < nb && y-- == 0) return a;
  return -1;
}
constexpr int term_b(int y, int na, int nb, int orders) {
  for (int o = orders - 1; o >= 0; --o)
    for (int a = 0; a < na; ++a)
      if (o - a >= 0 && o - a < nb && y-- == 0) return o - a;
  return -1;
}
constexpr int pairs(int na, int nb, int orders) {
  int n = 0;
  while (term_a(n, na, nb, orders) >= 0) ++n;
  return n;
}

// What a CTA works on.
struct Place {
  int slice, seg, h, n;      // n: tokens that count
  long long bh, b, lo, hi, end;  // tokens of the segment: lo .. end, up to hi they count
  __device__ __forceinline__ Place(const ScanArgs& A, unsigned cta) {
    long long id = cta;
    slice = (int)(id % A.nslice);
    id /= A.nslice;
    seg = (int)(id % A.nseg);
    bh = id / A.nseg;
    h = (int)(bh % A.H);
    b = bh / A.H;
    int len = A.L;
    if (A.lengths) len = min(max(A.lengths[b], 0), A.L);
    lo = (long long)seg * A.seglen;
    end = min(lo + A.seglen, (long long)A.L);
    hi = min(end, (long long)len);
    n = hi > lo ? (int)(hi - lo) : 0;
  }
};

// The CTA's work once more, strictly token by token, for results that are infinite or NaN. The products above run over
// all pairs of a chunk's tokens and multiply what is masked by zero, so an infinity or a NaN in one token reaches earlier ones, and
// a difference of two terms makes a NaN of an infinity. Here neither happens: a value reaches what the recurrence lets it reach.
// A thread holds DK / 8 rows of one column. Slow, and only CTAs with such results pay for it (with every one of them: 128 x 128 grid
// training 6.8 ms instead of 0.38, 65536 tokens of 8 heads of 128 10.2 instead of 0.30).
template <int DK, bool OUT, int NT, typename TO>
__device__ __forceinline__ void scan_by_token(const ScanArgs& A, const Place& z, float* sm) {
  constexpr int kN = 16, kG = kAll / kC, kR = DK / kG;
  float *qs = sm, *ks = qs + kN * DK, *vs = ks + kN * DK, *red = vs + kN * kC;
  const int tid = threadIdx.x, col = z.slice * kC, c = tid % kC, grp = tid / kC;
  const int rows = min(kR, A.DK - grp * kR);
  float hi, lo;
  two_floats(exp((double)A.log_decay[z.h]), &hi, &lo);
  const long long per = (long long)A.DK * A.DV;
  const float* src = nullptr;
  long long sr = A.DV, sc = 1;
  if (OUT && A.nseg > 1)
    src = A.seg + (z.bh * A.nseg + z.seg) * per, sr = A.segrow, sc = A.segcol;
  else if (OUT && A.start)
    src = A.start + z.bh * per, sr = A.srow, sc = A.scol;
  float S[kR];
#pragma unroll
  for (int r = 0; r < kR; ++r) S[r] = src && r < rows && col + c < A.DV ? src[(grp * kR + r) * sr + (col + c) * sc] : 0.f;
  const auto get = [&](const ScanOp& x, int d, long long t) {
    const bf16* p = static_cast<const bf16*>(x.p) + z.b * x.sb + (long long)(z.h / x.group) * x.sh + t * x.sl + d;
    float f = __bfloat162float(p[(NT - 1) * x.st]);
#pragma unroll
    for (int y = NT - 2; y >= 0; --y) f += __bfloat162float(p[y * x.st]);
    return f;
  };
  const auto when = [&](int i) { return A.reverse ? z.hi - 1 - i : z.lo + i; };
  for (int i0 = 0; i0 < z.n; i0 += kN) {
    const int n = min(kN, z.n - i0);
    for (int i = tid; i < n * DK; i += kAll) {
      const int d = i % DK;
      const bool in = d < A.DK;
      ks[i] = in ? get(A.k, d, when(i0 + i / DK)) : 0.f;
      if (OUT) qs[i] = in ? get(A.q, d, when(i0 + i / DK)) : 0.f;
    }
    for (int i = tid; i < n * kC; i += kAll)
      vs[i] = col + i % kC < A.DV ? get(A.v, col + i % kC, when(i0 + i / kC)) * A.vscale : 0.f;
    __syncthreads();
    for (int t = 0; t < n; ++t) {
      const float v = vs[t * kC + c];
      float o = 0.f;
#pragma unroll
      for (int r = 0; r < kR; ++r)
        if (r < rows) {
          const int at = t * DK + grp * kR + r;
          if (!A.reverse) S[r] = fmaf(S[r], hi, S[r] * lo);
          S[r] = fmaf(ks[at], v, S[r]);
          if (OUT) o = fmaf(qs[at], S[r], o);
          if (A.reverse) S[r] = fmaf(S[r], hi, S[r] * lo);
        }
      if (OUT) red[(t * kG + grp) * kC + c] = o;
    }
    __syncthreads();
    if (OUT)
      for (int i = tid; i < n * kC; i += kAll) {
        const int t = i / kC, d = col + i % kC;
        float o = 0.f;
        for (int y = 0; y < kG; ++y) o += red[(t * kG + y) * kC + i % kC];
        if (d < A.DV)
          DT<TO>::store(static_cast<TO*>(A.o) + z.b * A.ob + (long long)z.h * A.oh + when(i0 + t) * A.ol + d, o * A.oscale);
      }
  }
  float* dst = !OUT ? A.seg + (z.bh * A.nseg + z.seg) * per : A.nseg == 1 && A.finish ? A.finish + z.bh * per : nullptr;
  if (dst)
#pragma unroll
    for (int r = 0; r < kR; ++r)
      if (r < rows && col + c < A.DV)
        dst[(long long)(grp * kR + r) * (OUT ? A.srow : A.DV) + (long long)(col + c) * (OUT ? A.scol : 1)] = S[r];
}

// OUT: the pass with outputs; without it, segments' sums alone (K and V only).
template <int DK, bool OUT, int NT, int TERMS, typename TO>
__global__ void __launch_bounds__(kAll, 2) decay_mma_kernel(const ScanArgs A, const __grid_constant__ Maps M) {
  using L = Layout<DK, OUT, NT, TERMS>;
  constexpr int RT = L::RT;
  extern __shared__ __align__(1024) unsigned char smem[];
  float* tab = reinterpret_cast<float*>(smem + L::tab);
  uint64_t* bar = reinterpret_cast<uint64_t*>(smem + L::bar);
  volatile int* word = reinterpret_cast<volatile int*>(smem + L::bar + kBars * 8);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;

  const Place at(A, blockIdx.x);
  const int h = at.h, c0 = at.slice * kC, seg = at.seg, n_all = at.n;
  const long long b = at.b, bh = at.bh, t_lo = at.lo, t_hi = at.hi, t_end = at.end;
  const int chunks = (n_all + kT - 1) / kT;
  const bool rev = A.reverse;
  const auto tokens = [&](int i) { return min(kT, n_all - i * kT); };  // of chunk i, and the first of them in time
  const auto first = [&](int i) { return rev ? t_hi - i * kT - tokens(i) : t_lo + i * kT; };

  if (warp == 0) umma::tmem_alloc(reinterpret_cast<uint32_t*>(smem + L::bar + kBars * 8), kTmemCols);
  if (tid == 0) {
    for (int i = 0; i < kBars; ++i)
      umma::mbar_init(&bar[i], i < kHaveV || i == kDrain ? 1 : i == kReadO ? kWriters : kThreads / 32);
    umma::fence_mbar_init();
    word[kFailed] = (umma::su32(smem) & 1023) != 0;
    for (int i = kLast; i < kOdd; ++i) word[i] = -1;
    word[kOdd] = 0;
  }
  umma::fence_before_sync();
  __syncthreads();
  umma::fence_after_sync();
  const uint32_t tmem = (uint32_t)word[kTmem];
  // False once a wait of this thread has run out: no more waits. A loading or issuing warp then copies nothing and issues no
  // product any more, the others go on over what there is; warps that wait for it run out themselves. What is in flight is
  // waited for at the end, and all results of the CTA become NaN there.
  bool ok = !word[kFailed];
  const auto wait = [&](int i, int phase) {
    ok = ok && wait_phase(&bar[i], phase & 1, A.patience);
    umma::fence_after_sync();
  };
  // The same for the loading warps. Where they have one buffer a chunk's loads begin when the last chunk's products end, and
  // being woken takes longer than seeing it (8 heads of 128, 65536 tokens: 309 us, 295; with more buffers 382, 391).
  const auto wait_free = [&](int i, int phase) {
    if (L::nbuf > 1) return wait(i, phase);
    const uint32_t a = umma::su32(&bar[i]);
    const unsigned t0 = (unsigned)clock64();
    while (ok && !test_phase(a, phase & 1)) ok = (unsigned)clock64() - t0 < A.patience;
    umma::fence_after_sync();
  };
  const auto stopped = [&] { return __any_sync(0xffffffffu, !ok) != 0; };  // the same for the whole warp

  const float g = A.log_decay[h];
  // a^d, d = -64 .. 64, by the computing and writing warps for themselves
  const auto fill_table = [&](int i) {
    if (i <= 2 * kT) tab[i] = i < kT ? 0.f : i == kT ? 1.f : expf(g * (i - kT));
    asm volatile("bar.sync 1, %0;" ::"n"(kThreads + 32 * kWriters) : "memory");
  };
  if (warp >= kLoader && warp < kWriter) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(Regs<DK, OUT>::load));
  }
  if (warp >= kLoader && warp < kIssuer) {
    const int who = warp - kLoader;
    int last = -1;  // chunk brought
    if (who < 2) {
      const int hk = h / A.k.group, hv = h / A.v.group;
      const bf16* kp = static_cast<const bf16*>(A.k.p) + b * A.k.sb + hk * A.k.sh;
      const bf16* vp = static_cast<const bf16*>(A.v.p) + b * A.v.sb + hv * A.v.sh;
      // one buffer: one warp fills it. A warp that skips a buffer's phase could take the one before for the one that it waits
      // for; with more buffers each wait is preceded by one for a later chunk than the phase that was skipped.
      constexpr int kTurns = L::nbuf == 1 ? 1 : 2;
      for (int i = who < kTurns ? who : chunks; i < chunks; i += kTurns) {
        const int nb = i % L::nbuf;
        unsigned char *kd = smem + L::k + nb * L::qk, *vd = smem + L::v + nb * L::vt;
        if (i >= L::nbuf) wait_free((OUT ? kDoneO : kDoneS) + nb, i / L::nbuf - 1);
        if (M.on && tokens(i) == kT) {
          if (lane == 0 && ok) {
            last = i;
            expect(&bar[kFull + nb], L::qk + L::vt);
#pragma unroll
            for (int y = 0; y < NT; ++y) {
              load_box<DK>(umma::su32(kd + y * L::qk / NT), &M.k, &bar[kFull + nb], 0, hk, (int)first(i), (int)b + y * A.B);
              load_box<kC>(umma::su32(vd + y * kTile), &M.v, &bar[kFull + nb], c0, hv, (int)first(i), (int)b + y * A.B);
            }
          }
          __syncwarp();
        } else if (!stopped()) {
          last = i;
#pragma unroll
          for (int y = 0; y < NT; ++y) {
            load_tile<DK>(kd + y * L::qk / NT, kp + y * A.k.st, A.k.sl, tokens(i), 0, A.DK, first(i), A.vec);
            load_tile<kC>(vd + y * kTile, vp + y * A.v.st, A.v.sl, tokens(i), c0, A.DV, first(i), A.vec);
          }
          cp_wait();
          hand_over(&bar[kFull + nb]);
        }
      }
    } else if (OUT) {
      const int hq = h / A.q.group;
      const bf16* qp = static_cast<const bf16*>(A.q.p) + b * A.q.sb + hq * A.q.sh;
      for (int i = 0; i < chunks; ++i) {
        const int qb = i % L::qbuf;
        unsigned char* qd = smem + L::q + qb * L::qk;
        if (i >= L::qbuf) wait_free(kDoneR + qb, i / L::qbuf - 1);
        if (M.on && tokens(i) == kT) {
          if (lane == 0 && ok) {
            last = i;
            expect(&bar[kFullQ + qb], L::qk);
#pragma unroll
            for (int y = 0; y < NT; ++y)
              load_box<DK>(umma::su32(qd + y * L::qk / NT), &M.q, &bar[kFullQ + qb], 0, hq, (int)first(i), (int)b + y * A.B);
          }
          __syncwarp();
        } else if (!stopped()) {
          last = i;
#pragma unroll
          for (int y = 0; y < NT; ++y)
            load_tile<DK>(qd + y * L::qk / NT, qp + y * A.q.st, A.q.sl, tokens(i), 0, A.DK, first(i), A.vec);
          cp_wait();
          hand_over(&bar[kFullQ + qb]);
        }
      }
    }
    if (lane == 0) word[kLast + who] = last;
  } else if (warp == kIssuer) {
    // every descriptor is one of these plus a constant: built anew for each product, they held the issue up
    const uint32_t dq = desc_low(smem + L::q), dw = desc_low(smem + L::w), dp = desc_low(smem + L::p), ds = desc_low(smem + L::s);
    const uint32_t dk0 = desc_low(smem + L::k), dv0 = desc_low(smem + L::v);
    constexpr uint32_t kIdP = umma::idesc_bf16(kT, kT, 0, 0);
    constexpr uint32_t kIdR = umma::idesc_bf16(kT, kC, 0, 1);
    constexpr uint32_t kIdS = umma::idesc_bf16(DK, kC, 1, 1);
    for (int i = 0; i < chunks; ++i) {
      if (stopped()) break;
      const int nb = i % L::nbuf, wb = i % L::wbuf;
      const uint32_t dk = dk0 + nb * (L::qk >> 4), dv = dv0 + nb * (L::vt >> 4);
      wait(kFull + nb, i / L::nbuf);
      if (OUT) {
        const uint32_t dqi = dq + i % L::qbuf * (L::qk >> 4);
        wait(kFullQ + i % L::qbuf, i / L::qbuf);
        if (elect() && ok) {
#pragma unroll
          for (int y = 0; y < pairs(NT, NT, NT); ++y)
#pragma unroll
            for (int x = 0; x < DK / 16; ++x) {
              const int at = (x >> 2) * kNextTile + (x & 3) * kAlongK;
              mma(tmem + kColP, dqi + term_a(y, NT, NT, NT) * (L::qk / NT >> 4) + at,
                  dk + term_b(y, NT, NT, NT) * (L::qk / NT >> 4) + at, kIdP, x + y > 0);
            }
          umma::commit(&bar[kDoneP]);
        }
        __syncwarp();
      }
      wait(kHaveS + wb, i / L::wbuf);
      wait(kHaveV + wb, i / L::wbuf);
      if (elect() && ok) {
#pragma unroll
        for (int y = 0; y < pairs(NT, TERMS, TERMS); ++y)
#pragma unroll
          for (int x = 0; x < kT / 16; ++x)
            mma(tmem + kColS - 64 * wb, dk + term_a(y, NT, TERMS, TERMS) * (L::qk / NT >> 4) + x * kAlongRows,
                dw + (wb * TERMS + term_b(y, NT, TERMS, TERMS)) * kNextTile + x * kAlongRows, kIdS, x + y > 0);
        umma::commit(&bar[kDoneS + (OUT ? 0 : nb)]);
      }
      __syncwarp();
      if (OUT) {
        const uint32_t dqi = dq + i % L::qbuf * (L::qk >> 4);
        if (i) wait(kReadO, i - 1);
        if (elect() && ok) {
#pragma unroll
          for (int y = 0; y < pairs(NT, RT, RT); ++y)
#pragma unroll
            for (int x = 0; x < DK / 16; ++x)
              mma(tmem + kColR, dqi + term_a(y, NT, RT, RT) * (L::qk / NT >> 4) + (x >> 2) * kNextTile + (x & 3) * kAlongK,
                  ds + term_b(y, NT, RT, RT) * (DK * 128 >> 4) + x * kAlongRows, kIdR, x + y > 0);
          umma::commit(&bar[kDoneR + i % L::qbuf]);
        }
        __syncwarp();
        wait(kHaveP, i);
        if (elect() && ok) {
#pragma unroll
          for (int y = 0; y < pairs(RT, NT, RT); ++y)
#pragma unroll
            for (int x = 0; x < kT / 16; ++x)
              mma(tmem + kColO, dp + term_a(y, RT, NT, RT) * kNextTile + x * kAlongK,
                  dv + term_b(y, RT, NT, RT) * kNextTile + x * kAlongRows, kIdR, x + y > 0);
          umma::commit(&bar[kDoneO + nb]);
        }
        __syncwarp();
      }
    }
  } else if (warp >= kWriter) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(Regs<DK, OUT>::write));
    fill_table(2 * kT + 1);
    if (OUT) {
      const int wq = warp & 3, row = wq * 16 + (lane >> 2), quad = lane & 3;
      const uint32_t lanes = tmem + ((uint32_t)(wq * 32) << 16);
      TO* op = static_cast<TO*>(A.o) + b * A.ob + (long long)h * A.oh + c0;
      float2 odd = make_float2(0.f, 0.f);  // NaN once a result was infinite or NaN
      for (int i = 0; i < chunks; ++i) {
        const int n = tokens(i);
        wait(kDoneO + i % L::nbuf, i / L::nbuf);
        const float os = A.vscale * A.oscale;
#pragma unroll
        for (int half = 0; half < kC; half += 32) {
          uint32_t r[16], o[16];
          tmem_ld2(lanes + kColR + half, lanes + kColO + half, r, o);
          if (half) {  // all of it has been read
            umma::fence_before_sync();
            __syncwarp();
            if (lane == 0) arrive(&bar[kReadO]);
          }
#pragma unroll
          for (int y = 0; y < 2; ++y) {
            const int rw = row + 8 * y;
            const float rs = tab[kT + (rev ? n - 1 - rw : rw + 1)] * A.oscale;
            TO* d = op + (first(i) + rw) * A.ol + half;
            float2 f[4];  // columns half + 8 j + 2 quad, + 1
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              const int at = 4 * j + 2 * y;
              f[j] = make_float2(fmaf(__uint_as_float(r[at]), rs, __uint_as_float(o[at]) * os),
                                 fmaf(__uint_as_float(r[at + 1]), rs, __uint_as_float(o[at + 1]) * os));
              odd = ffma2(f[j], make_float2(0.f, 0.f), odd);
            }
            if (sizeof(TO) == 2 && A.ovec) {
              // transposed among four lanes: each stores 16 bytes of the row, together 64
              uint4 u = make_uint4(pack_out<TO>(f[0]), pack_out<TO>(f[1]), pack_out<TO>(f[2]), pack_out<TO>(f[3]));
              swap_pairs(u.x, u.y, 1, quad);
              swap_pairs(u.z, u.w, 1, quad);
              swap_pairs(u.x, u.z, 2, quad);
              swap_pairs(u.y, u.w, 2, quad);
              if (rw < n && c0 + half + 8 * quad < A.DV) *reinterpret_cast<uint4*>(d + 8 * quad) = u;
            } else if (rw < n) {
#pragma unroll
              for (int j = 0; j < 4; ++j) {
                const int c = 8 * j + 2 * quad, left = A.DV - c0 - half - c;
                if (sizeof(TO) == 4 && A.ovec && left > 0) {
                  *reinterpret_cast<float2*>(d + c) = f[j];
                } else {
                  if (left > 0) DT<TO>::store(d + c, f[j].x);
                  if (left > 1) DT<TO>::store(d + c + 1, f[j].y);
                }
              }
            }
          }
        }
      }
      if (odd.x != 0.f || odd.y != 0.f) word[kOdd] = 1;
      const long long z0 = max(t_lo, t_hi);  // tokens past the length: zeros
      for (long long i = tid - 32 * kWriter; i < (t_end - z0) * kC; i += 32 * kWriters) {
        const long long r = i / kC;
        const int c = (int)(i - r * kC);
        if (c0 + c < A.DV) DT<TO>::store(op + (z0 + r) * A.ol + c, 0.f);
      }
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(Regs<DK, OUT>::compute));
    // This thread's part of a 64 x 64 product: rows row and row + 8, columns half + 8 j + pair + {0, 1}, j < 4. Of a
    // state of 128 rows it has two such parts, 16 TMEM lanes apart (SB).
    constexpr int SB = DK / 64;
    const auto power = [&](int n) {  // a^n as the sum of two floats
      const double an = exp((double)g * n);
      return make_float2((float)an, (float)(an - (double)(float)an));
    };
    const float2 a64 = power(kT);
    const int wq = warp & 3, half = (warp >> 2) * 32;
    const int row = wq * 16 + (lane >> 2), pair = 2 * (lane & 3);
    const int srow = SB == 1 ? row : wq * 32 + (lane >> 2);
    const uint32_t lanes = tmem + ((uint32_t)(wq * 32) << 16) + half;
    const long long per_state = (long long)A.DK * A.DV;
    const int left = A.DV - c0 - half - pair;  // columns from this thread's first on that exist
    float S[SB][16];
    const auto put_state = [&] {  // the rounded state, for R
#pragma unroll
      for (int y = 0; y < SB; ++y) {
        const int rw = srow + 16 * y;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          unsigned char* d = smem + L::s + swz(rw, half + 8 * j + pair);
          put_terms<RT>(d, DK * 128, make_float2(S[y][4 * j], S[y][4 * j + 1]));
          put_terms<RT>(d + 1024, DK * 128, make_float2(S[y][4 * j + 2], S[y][4 * j + 3]));
        }
      }
    };
    {
      const float* src = nullptr;
      long long sr = A.DV, sc = 1;
      if (OUT && A.nseg > 1) {
        src = A.seg + (bh * A.nseg + seg) * per_state;
        sr = A.segrow, sc = A.segcol;
      } else if (OUT && A.start) {
        src = A.start + bh * per_state;
        sr = A.srow, sc = A.scol;
      }
#pragma unroll
      for (int y = 0; y < SB; ++y)
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          const int c = 8 * (r >> 2) + (r & 1), rw = srow + 16 * y + 8 * ((r >> 1) & 1);
          S[y][r] = src && rw < A.DK && c < left ? src[rw * sr + (c0 + half + pair + c) * sc] : 0.f;
        }
      if (OUT) put_state();
      hand_over(&bar[kHaveS]);
      if (L::wbuf == 2) hand_over(&bar[kHaveS + 1]);
    }
    // The V of chunk i, decayed, in TERMS terms.
    const auto split_v = [&](int i) {
      const int wb = i % L::wbuf, n = tokens(i);
      const unsigned char* v = smem + L::v + i % L::nbuf * L::vt;
      unsigned char* terms = smem + L::w + wb * (TERMS * kTile);
      wait(kFull + i % L::nbuf, i / L::nbuf);
#pragma unroll
      for (int x = 0; x < kT * kC / 8 / kThreads; ++x) {
        const int at = tid + x * kThreads, t = at >> 3;  // V's place in the tile is its terms' place
        const float w = t < n ? tab[kT + (rev ? t + 1 : n - 1 - t)] * A.vscale : 0.f;
        uint4 u[NT], hi, mid, lo;
#pragma unroll
        for (int y = 0; y < NT; ++y) u[y] = *reinterpret_cast<const uint4*>(v + y * kTile + at * 16);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          float2 f = unpack2((&u[NT - 1].x)[e]);  // the terms from the least on: exact
#pragma unroll
          for (int y = NT - 2; y >= 0; --y) f = cadd(f, unpack2((&u[y].x)[e]));
          f.x *= w, f.y *= w;
          const uint32_t p = pack2(f.x, f.y);
          f = csub(f, unpack2(p));
          const uint32_t q = pack2(f.x, f.y);
          (&hi.x)[e] = p, (&mid.x)[e] = q;
          if (TERMS == 3) {
            f = csub(f, unpack2(q));
            (&lo.x)[e] = pack2(f.x, f.y);
          }
        }
        *reinterpret_cast<uint4*>(terms + at * 16) = hi;
        *reinterpret_cast<uint4*>(terms + kTile + at * 16) = mid;
        if (TERMS == 3) *reinterpret_cast<uint4*>(terms + 2 * kTile + at * 16) = lo;
      }
      hand_over(&bar[kHaveV + wb]);
    };
    fill_table(tid);
    // a^|row - column| of this thread's part of P, zero where the column is later in scan order: entries 2 m, 2 m + 1 for
    // columns 8 (m - 1), + 1 of its first row. In registers where there is room.
    const float* tb = tab + kT + (rev ? half + pair - 8 - row : row - half - pair + 8);
    const int along = rev ? 1 : -1;
    float dec[SB == 1 ? 10 : 1];
    if (SB == 1)
#pragma unroll
      for (int m = 0; m < (SB == 1 ? 10 : 1); ++m) dec[m] = tb[along * (8 * (m / 2) + (m & 1))];
    const auto decay = [&](int m) { return SB == 1 ? dec[SB == 1 ? m : 0] : tb[along * (8 * (m / 2) + (m & 1))]; };
    if (chunks) split_v(0);
    for (int i = 0; i < chunks; ++i) {
      const int n = tokens(i);
      if (L::wbuf == 2 && i + 1 < chunks) split_v(i + 1);  // both buffers are in use: beside the last chunk's product
      if (OUT) {  // P
        wait(kDoneP, i);
        uint32_t p[16];
        tmem_ld(lanes + kColP, p);
#pragma unroll
        for (int j = 0; j < 4; ++j) {  // row + 8 at column block j decays like row at block j - 1
          unsigned char* d = smem + L::p + swz(row, half + 8 * j + pair);
          put_terms<RT>(d, kTile, make_float2(__uint_as_float(p[4 * j]) * decay(2 * j + 2),
                                              __uint_as_float(p[4 * j + 1]) * decay(2 * j + 3)));
          put_terms<RT>(d + 1024, kTile, make_float2(__uint_as_float(p[4 * j + 2]) * decay(2 * j),
                                                     __uint_as_float(p[4 * j + 3]) * decay(2 * j + 1)));
        }
        hand_over(&bar[kHaveP]);
      }
      {  // the state
        const float2 an = n == kT ? a64 : power(n);
        if (OUT) wait(kDoneR + i % L::qbuf, i / L::qbuf);
        wait(kDoneS + (OUT ? 0 : i % L::nbuf), OUT ? i : i / L::nbuf);
#pragma unroll
        for (int y = 0; y < SB; ++y) {
          uint32_t d[16];
          tmem_ld(lanes + kColS - 64 * (i % L::wbuf) + ((uint32_t)(16 * y) << 16), d);
#pragma unroll
          for (int r = 0; r < 16; ++r) S[y][r] = fmaf(S[y][r], an.x, fmaf(S[y][r], an.y, __uint_as_float(d[r])));
        }
        if (OUT) put_state();
        hand_over(&bar[kHaveS + i % L::wbuf]);
      }
      if (L::wbuf == 1 && i + 1 < chunks) split_v(i + 1);
    }
    float* dst = nullptr;
    long long sr = A.DV, sc = 1;
    if (!OUT) {
      dst = A.seg + (bh * A.nseg + seg) * per_state;
    } else if (A.nseg == 1 && A.finish) {
      dst = A.finish + bh * per_state;
      sr = A.srow, sc = A.scol;
    }
    if (dst) {
      float odd = 0.f;
#pragma unroll
      for (int y = 0; y < SB; ++y)
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          const int c = 8 * (r >> 2) + (r & 1), rw = srow + 16 * y + 8 * ((r >> 1) & 1);
          odd = fmaf(S[y][r], 0.f, odd);
          if (rw < A.DK && c < left) dst[rw * sr + (c0 + half + pair + c) * sc] = S[y][r];
        }
      if (odd != 0.f) word[kOdd] = 1;
    }
  }
  if (!ok) word[kFailed] = 1;
  umma::fence_before_sync();
  __syncthreads();
  if (word[kFailed] || word[kOdd]) {
    if (warp < kLoader)
      asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(Regs<DK, OUT>::launch));
    else
      asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(Regs<DK, OUT>::launch));
    // asked anew: kept in registers all along, the place cost the loops some of theirs
    unsigned cta;
    asm volatile("mov.u32 %0, %%ctaid.x;" : "=r"(cta));
    const Place z(A, cta);
    if (word[kFailed]) {
      // products and copies in flight end by themselves; shared memory and TMEM are given back after them
      if (warp == kIssuer) {
        if (elect()) umma::commit(&bar[kDrain]);
        wait_phase(&bar[kDrain], 0, kWaitClocks);
      } else if (warp == kLoader && lane < L::nbuf) {
        constexpr int kTurns = L::nbuf == 1 ? 1 : 2;
        const int i = max(word[kLast], word[kLast + 1]) - lane;  // the last chunk of one of the buffers
        if (i >= 0 && i <= word[kLast + i % kTurns]) wait_phase(&bar[kFull + i % L::nbuf], i / L::nbuf & 1, kWaitClocks);
      } else if (OUT && warp == kLoader + 2 && lane < L::qbuf) {
        const int i = word[kLast + 2] - lane;
        if (i >= 0) wait_phase(&bar[kFullQ + i % L::qbuf], i / L::qbuf & 1, kWaitClocks);
      }
      umma::fence_before_sync();
      __syncthreads();
      const int col = z.slice * kC, DV = A.DV;
      const float nan = __int_as_float(0x7fffffff);
      if (OUT)
        for (long long i = threadIdx.x; i < (long long)z.n * kC; i += kAll) {
          const int c = col + (int)(i % kC);
          if (c < DV) DT<TO>::store(static_cast<TO*>(A.o) + z.b * A.ob + (long long)z.h * A.oh + (z.lo + i / kC) * A.ol + c, nan);
        }
      float* dst = !OUT ? A.seg + (z.bh * A.nseg + z.seg) * A.DK * DV
                        : A.nseg == 1 && A.finish ? A.finish + z.bh * A.DK * DV : nullptr;
      if (dst)
        for (int i = threadIdx.x; i < A.DK * kC; i += kAll) {
          const int c = col + i % kC;
          if (c < DV) dst[(long long)(i / kC) * (OUT ? A.srow : DV) + (long long)c * (OUT ? A.scol : 1)] = nan;
        }
      if (threadIdx.x == 0) atomicExch(&g_ran_out, 1u);
    } else {
      scan_by_token<DK, OUT, NT, TO>(A, z, reinterpret_cast<float*>(smem));
    }
  }
  if (warp == 0) umma::tmem_dealloc(tmem, kTmemCols);
}

PFN_cuTensorMapEncodeTiled_v12000 encode_fn() {
  static std::once_flag once;
  static PFN_cuTensorMapEncodeTiled_v12000 fn = nullptr;
  std::call_once(once, [] {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) == cudaSuccess &&
        q == cudaDriverEntryPointSuccess)
      fn = reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(p);
  });
  return fn;
}

// False where TMA cannot address the tensor (a head size, an address or a stride off 16 bytes, a stride of zero).
bool make_map(CUtensorMap* m, const ScanOp& x, int D, int heads, int L, int B) {  // B: batches times terms
  PFN_cuTensorMapEncodeTiled_v12000 enc = encode_fn();
  if (!enc || !x.p) return false;
  const cuuint64_t dims[4] = {(cuuint64_t)D, (cuuint64_t)heads, (cuuint64_t)L, (cuuint64_t)B};
  const long long s[3] = {x.sh, x.sl, x.sb};
  cuuint64_t strides[3];
  for (int i = 0; i < 3; ++i) {
    const long long bytes = dims[i + 1] == 1 ? (long long)((D + 7) / 8 * 16) : 2 * s[i];  // one of them: never stepped over
    if (bytes <= 0 || bytes % 16 || bytes >= (1ll << 40)) return false;
    strides[i] = (cuuint64_t)bytes;
  }
  const cuuint32_t box[4] = {64, 1, kT, 1}, one[4] = {1, 1, 1, 1};
  return enc(m, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4, const_cast<void*>(x.p), dims, strides, box, one,
             CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_128B,
             CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <int DK, bool OUT, int NT, int TERMS, typename TO>
int launch(const ScanArgs& A, const Maps& M, long long ctas, cudaStream_t st) {
  auto kern = decay_mma_kernel<DK, OUT, NT, TERMS, TO>;
  constexpr size_t sm = Layout<DK, OUT, NT, TERMS>::bytes;
  if (!kernel_smem_once((const void*)kern, sm, true)) return set_error(HYFFT_ERR_CUDA, "decay attention: shared memory");
  kern<<<(unsigned)ctas, kAll, sm, st>>>(A, M);
  if (cudaGetLastError() != cudaSuccess) return set_error(HYFFT_ERR_CUDA, "decay attention: kernel launch failed");
  g_launches.fetch_add(1, std::memory_order_relaxed);
  return HYFFT_OK;
}

template <int DK, int NT, typename T>
int launch_dk(const ScanArgs& A, const Maps& M, bool out_f32, long long ctas, cudaStream_t st) {
  if (!A.o) return launch<DK, false, NT, 3, T>(A, M, ctas, st);
  // where segments were added up before, the state only serves this pass's outputs: those of bfloat16 read it in 16 bits,
  // and as many of the decayed V are enough (not by whether the caller wants the final state, so that asking for it changes no output)
  if (NT == 1 && A.nseg > 1)
    return out_f32 ? launch<DK, true, NT, NT == 1 ? 2 : 3, float>(A, M, ctas, st)
                   : launch<DK, true, NT, NT == 1 ? 2 : 3, T>(A, M, ctas, st);
  return out_f32 ? launch<DK, true, NT, 3, float>(A, M, ctas, st) : launch<DK, true, NT, 3, T>(A, M, ctas, st);
}

// ---------------------------------------------------------------- terms
struct SplitArgs {
  const void* src[4];
  bf16* dst[4];
  long long sb[4], sl[4], sh[4], begin[5];  // strides; where each tensor's work begins, in runs of eight features
  int heads[4], D[4], n;
  int B, L, terms;
};

// The bfloat16 nearest to f; of a finite f never an infinity (float32 reaches a little further: the next term has the rest).
__device__ __forceinline__ uint32_t finite_bits(float f) {
  uint32_t u = __bfloat16_as_ushort(__float2bfloat16_rn(f));
  if ((u & 0x7fff) == 0x7f80 && isfinite(f)) --u;
  return u;
}

// x = sum of bfloat16 terms, largest first; an infinity or NaN is the first term alone.
template <typename T>
__global__ void __launch_bounds__(256) decay_split_kernel(const SplitArgs A) {
  const long long id = (long long)blockIdx.x * 256 + threadIdx.x;
  if (id >= A.begin[A.n]) return;
  int w = 0;
  while (id >= A.begin[w + 1]) ++w;
  const int D = A.D[w], runs = (D + 7) / 8;
  long long i = id - A.begin[w];
  const int c = (int)(i % runs) * 8;
  i /= runs;
  const int h = (int)(i % A.heads[w]);
  i /= A.heads[w];  // b * L + l
  const long long b = i / A.L, l = i - b * A.L;
  const T* src = static_cast<const T*>(A.src[w]) + b * A.sb[w] + l * A.sl[w] + h * A.sh[w] + c;
  float f[8];
#pragma unroll
  for (int u = 0; u < 8; ++u) f[u] = c + u < D ? DT<T>::load(src + u) : 0.f;
  const long long per = (long long)A.B * A.L * A.heads[w] * runs * 8;
  bf16* dst = A.dst[w] + ((i * A.heads[w] + h) * runs * 8 + c);
  for (int t = 0; t < A.terms; ++t) {
    uint4 out;
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      uint32_t p = pack2(f[2 * u], f[2 * u + 1]);
      float2 r = unpack2(p);
      if (!isfinite(r.x) || !isfinite(r.y)) {
        p = finite_bits(f[2 * u]) | finite_bits(f[2 * u + 1]) << 16;
        r = unpack2(p);
        f[2 * u] = isfinite(r.x) ? f[2 * u] - r.x : 0.f;
        f[2 * u + 1] = isfinite(r.y) ? f[2 * u + 1] - r.y : 0.f;
      } else {
        f[2 * u] -= r.x;
        f[2 * u + 1] -= r.y;
      }
      (&out.x)[u] = p;
    }
    *reinterpret_cast<uint4*>(dst + t * per) = out;
  }
}

size_t term_elements(int B, long long L, int heads, int D, int terms) {
  return (size_t)terms * B * L * heads * ((D + 7) / 8 * 8);
}

}  // namespace

size_t mma_terms_bytes(int B, long long L, int heads, int D, int terms) {
  return (sizeof(bf16) * term_elements(B, L, heads, D, terms) + 255) / 256 * 256;
}

int launch_split_terms(ScanOp* ops, const int* heads, const int* D, int n, int B, long long L, int dtype, int terms,
                       char* ws, cudaStream_t st) {
  SplitArgs A{};
  A.B = B, A.L = (int)L, A.terms = terms, A.n = n;
  for (int w = 0; w < n; ++w) {
    const int runs = (D[w] + 7) / 8;
    A.src[w] = ops[w].p, A.sb[w] = ops[w].sb, A.sl[w] = ops[w].sl, A.sh[w] = ops[w].sh;
    A.heads[w] = heads[w], A.D[w] = D[w];
    A.dst[w] = reinterpret_cast<bf16*>(ws);
    ws += mma_terms_bytes(B, L, heads[w], D[w], terms);
    A.begin[w + 1] = A.begin[w] + (long long)B * L * heads[w] * runs;
    ops[w].p = A.dst[w];
    ops[w].sh = runs * 8, ops[w].sl = (long long)heads[w] * runs * 8, ops[w].sb = L * ops[w].sl, ops[w].st = B * ops[w].sb;
  }
  const long long ctas = (A.begin[n] + 255) / 256;
  if (ctas > 0x7fffffffLL) return set_error(HYFFT_ERR_UNSUPPORTED, "decay attention: too many elements");
  if (dtype == HYFFT_F32)
    decay_split_kernel<float><<<(unsigned)ctas, 256, 0, st>>>(A);
  else if (dtype == HYFFT_BF16)
    decay_split_kernel<bf16><<<(unsigned)ctas, 256, 0, st>>>(A);
  else
    decay_split_kernel<__half><<<(unsigned)ctas, 256, 0, st>>>(A);
  if (cudaGetLastError() != cudaSuccess) return set_error(HYFFT_ERR_CUDA, "decay attention: kernel launch failed");
  g_launches.fetch_add(1, std::memory_order_relaxed);
  return HYFFT_OK;
}

int decay_wait_status(bool clear, unsigned* ran_out) { return read_ran_out(clear, ran_out) == cudaSuccess ? HYFFT_OK : HYFFT_ERR_CUDA; }

int launch_scan_mma(ScanArgs A, int dtype, bool out_f32, long long ctas, cudaStream_t st) {
  if (ctas > 0x7fffffffLL) return set_error(HYFFT_ERR_UNSUPPORTED, "decay attention: too many rows");
  const int nt = dtype == HYFFT_BF16 ? 1 : dtype == HYFFT_F16 ? 2 : 3;
  Maps M{};
  A.patience = g_wait_clocks.load(std::memory_order_relaxed);
  M.on = A.L >= kT && A.vec && make_map(&M.k, A.k, A.DK, A.H / A.k.group, A.L, A.B * nt) &&
         make_map(&M.v, A.v, A.DV, A.H / A.v.group, A.L, A.B * nt) &&
         (!A.o || make_map(&M.q, A.q, A.DK, A.H / A.q.group, A.L, A.B * nt));
  const bool wide = A.DK > 64;
  if (nt == 1) return wide ? launch_dk<128, 1, bf16>(A, M, out_f32, ctas, st) : launch_dk<64, 1, bf16>(A, M, out_f32, ctas, st);
  if (nt == 2)
    return wide ? launch_dk<128, 2, __half>(A, M, out_f32, ctas, st) : launch_dk<64, 2, __half>(A, M, out_f32, ctas, st);
  return wide ? launch_dk<128, 3, float>(A, M, true, ctas, st) : launch_dk<64, 3, float>(A, M, true, ctas, st);
}

}  // namespace hyfft
