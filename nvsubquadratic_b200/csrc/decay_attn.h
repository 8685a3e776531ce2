// One scan of the decayed linear attention, as decay_attn.cu plans it and its kernels run it.
#pragma once

#include <cuda_runtime.h>

namespace hyfft {

struct ScanOp {  // strides in elements: batch, token, head
  const void* p;
  long long sb, sl, sh;
  int group;         // query heads that share one head of this operand
  long long st = 0;  // between the bfloat16 terms of a split operand
};

// o_i = oscale * S_i^T q_i with S_i = a S_{i-1} + vscale * k_i v_i^T over a row's tokens, forwards or backwards in time.
struct ScanArgs {
  ScanOp q, k, v, x;  // x: the output's gradient (learned decays only)
  void* o;            // nullptr: the pass that adds up each segment from a zero state
  long long ob, ol, oh;
  const float* log_decay;
  const int* lengths;  // [B] or nullptr
  const float* start;  // state before a row's first token [B, H, ...], nullptr: zero
  float* finish;       // state after its last
  float* seg;          // [B * H, nseg, DK, DV] segment sums, then segment start states
  float* segT;         // the same of T (learned decays)
  float* dg;           // [B * H, nseg, ...] partial sums of the decay's gradient
  float vscale, oscale;
  int B, H, L, DK, DV;  // DK: rows of the state in this scan's order, DV: its columns
  int srow, scol;        // strides of start and finish
  int segrow, segcol;    // strides of a segment's start state as it is read
  int nseg, seglen, nslice;
  int reverse;  // the decay is applied after a token's output instead of before
  int vec;      // q, k, v (and x) can be read in 16-byte pieces
  int ovec;     // o can be written in 16-byte pieces
  unsigned patience;   // clocks after which a wait inside the kernel gives up
};

// a as the sum of two floats, both of a's sign and neither zero, so that infinity times a is infinity plus infinity.
__device__ __forceinline__ void two_floats(double a, float* hi, float* lo) {
  *hi = __double2float_rz(a);
  *lo = (float)(a - (double)*hi);
  if (*hi > 0.f) *lo = fmaxf(*lo, 1.1754944e-38f);
}

// decay_mma.cu: DK <= 128, columns in slices of 64, segments of whole 64-token chunks. float16 and float32 operands are
// first split into bfloat16 terms (2, 3): launch_split_terms does up to four tensors [B, L, heads[w], D[w]] into `ws` and makes
// the ops point there.
constexpr int kMmaTok = 64;
constexpr int kMmaCols = 64;
constexpr int kMmaMaxDK = 128;
int launch_scan_mma(ScanArgs A, int dtype, bool out_f32, long long ctas, cudaStream_t st);
size_t mma_terms_bytes(int B, long long L, int heads, int D, int terms);
int decay_wait_status(bool clear, unsigned* ran_out);
int launch_split_terms(ScanOp* ops, const int* heads, const int* D, int n, int B, long long L, int dtype, int terms, char* ws,
                       cudaStream_t st);

}  // namespace hyfft
