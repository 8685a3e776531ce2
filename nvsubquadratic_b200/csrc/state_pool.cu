// Slots of pools of states: copied to other slots all at once (requests forked, reordered in place, cleared), and running requests
// moved into the lowest slots. A pool is a row of bytes for each slot; several pools (a layer's states, positions, other layers')
// go through one launch.
//
// Bound by HBM bandwidth (source rows read once, target rows written once). A source may be a target of another move, in chains and
// cycles, so every source has to be read before its row is written. A CTA takes the same few bytes of every row that takes part: it copies
// them to shared memory, waits, and writes them out, so nothing crosses HBM twice and no second buffer is needed. A kernel of one CTA
// comes first and drops what is not to be copied: targets outside the pool, and all but the last move into a slot.
// 224 rows of 2 MB in another order: 155 us (93% of a copy's rate); 2000 rows of 16 KB: 18.6 us in a graph, 24.7 among other passes (54 and 41%;
// 56 us with one unit looked up at a time): the list takes 5 us to make by one CTA, and 64 bytes of 2000 rows fill an SM's shared memory, so
// 257 CTAs take two waves, each reading all before it writes. Rows are copied 16 bytes at a time where all of them start on 16 bytes, else 8, 4 or 1:
// those 2000 rows with 8188, 8190 and 8191 elements of 16 bits instead of 8192 take 33, 53 and 232 us.
// Compaction fills the lowest free slots with the highest running requests; sources and targets are apart, and rows are copied through
// registers.
#include <cuda_runtime.h>

#include <algorithm>
#include <atomic>

#include "../../include/hyfft.h"
#include "common.cuh"

namespace hyfft {

extern std::atomic<long long> g_launches;
int set_error(int code, const char* msg);  // engine.cu: the message hyfft_last_error returns

namespace {

constexpr int kThreads = 256;
constexpr int kPlanThreads = 1024;
constexpr size_t kStageBytes = 64 * 1024;       // of shared memory for a CTA where that is enough
constexpr size_t kStageMost = 200 * 1024;
constexpr int kSkip = -2;

struct PoolArgs {
  char* base[HYFFT_MAX_POOLS];
  long long row[HYFFT_MAX_POOLS];    // bytes
  int unit[HYFFT_MAX_POOLS];         // bytes copied at once: 16, 8, 4 or 1
  int width[HYFFT_MAX_POOLS];        // bytes of a row that a CTA takes
  int first[HYFFT_MAX_POOLS + 1];    // a pool's first CTA
  int pools;
  const int* source;                 // the row that each move reads, kSkip for none
  const int* target;                 // the row that it writes, or what plan_copy_kernel says
  const int* count;                  // moves, on the device (compaction); or NULL
  int moves;
};

// from [moves]: the row that each move reads, to [moves]: the row that it writes; kSkip where it does not, and rows that become zeros are
// counted down from kSkip - 1. owner [slots]: the last move into each slot.
__global__ void __launch_bounds__(kPlanThreads) plan_copy_kernel(const int* source, const int* target, int moves, int slots, int* owner,
                                                                 int* from, int* to) {
  for (int i = threadIdx.x; i < moves; i += kPlanThreads) {
    const int t = target[i];
    if (t >= 0 && t < slots) owner[t] = -1;
  }
  __syncthreads();
  for (int i = threadIdx.x; i < moves; i += kPlanThreads) {
    const int t = target[i];
    if (t >= 0 && t < slots) atomicMax(owner + t, i);
  }
  __syncthreads();
  for (int i = threadIdx.x; i < moves; i += kPlanThreads) {
    const int t = target[i], s = source[i];
    const bool made = t >= 0 && t < slots && atomicMax(owner + t, -1) == i && s != t;
    const bool row = s >= 0 && s < slots;
    from[i] = made && row ? s : kSkip;
    to[i] = !made ? kSkip : row ? t : kSkip - 1 - t;
  }
}

// Sum of v over the threads before this one, and over all (whole).
__device__ __forceinline__ int scan_block(int v, int* warps, int& whole) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int s = v;
#pragma unroll
  for (int d = 1; d < 32; d *= 2) {
    const int u = __shfl_up_sync(0xffffffffu, s, d);
    if (lane >= d) s += u;
  }
  __syncthreads();
  if (lane == 31) warps[warp] = s;
  __syncthreads();
  int before = 0;
  whole = 0;
  for (int w = 0; w < kPlanThreads / 32; ++w) {
    if (w < warp) before += warps[w];
    whole += warps[w];
  }
  return before + s - v;
}

// holes[k], movers[k]: the k-th free slot below the number of running requests, the k-th running request above it; as many of one as of
// the other. count: how many. moved [slots]: where each slot's request is afterwards, -1 for none.
__global__ void __launch_bounds__(kPlanThreads) plan_compact_kernel(const unsigned char* live, int slots, int* movers, int* holes, int* count,
                                                                    int* moved) {
  __shared__ int warps[kPlanThreads / 32];
  int running = 0, whole;
  for (int i0 = 0; i0 < slots; i0 += kPlanThreads) {
    const int i = i0 + threadIdx.x;
    scan_block(i < slots && live[i], warps, whole);
    running += whole;
  }
  int h = 0, m = 0;
  for (int i0 = 0; i0 < slots; i0 += kPlanThreads) {
    const int i = i0 + threadIdx.x;
    const bool in = i < slots, on = in && live[i];
    const int kh = h + scan_block(in && !on && i < running, warps, whole);
    h += whole;
    const int km = m + scan_block(on && i >= running, warps, whole);
    m += whole;
    if (in && !on && i < running) holes[kh] = i;
    if (on && i >= running) movers[km] = i;
    if (in && !(on && i >= running)) moved[i] = on ? i : -1;
  }
  if (threadIdx.x == 0) *count = m;
  __syncthreads();
  for (int k = threadIdx.x; k < m; k += kPlanThreads) moved[movers[k]] = holes[k];
}

template <int U> __device__ __forceinline__ void to_shared(unsigned char* dst, const char* src) {
  const uint32_t d = (uint32_t)__cvta_generic_to_shared(dst);
  if constexpr (U == 16)
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(d), "l"(src) : "memory");
  else if constexpr (U == 8)
    asm volatile("cp.async.ca.shared.global [%0], [%1], 8;" ::"r"(d), "l"(src) : "memory");
  else if constexpr (U == 4)
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(d), "l"(src) : "memory");
  else
    *dst = *reinterpret_cast<const unsigned char*>(src);
}
template <int U> struct Word;
template <> struct Word<16> { using T = uint4; };
template <> struct Word<8> { using T = uint2; };
template <> struct Word<4> { using T = uint32_t; };
template <> struct Word<1> { using T = unsigned char; };

// `width` bytes (a whole number of units) from `base` on of every row. A thread has N units' rows looked up before it copies them.
template <int U> __device__ __forceinline__ void copy_slice(const PoolArgs& A, char* base, long long row, int width, unsigned char* stage) {
  constexpr int N = 8;
  using W = typename Word<U>::T;
  const int per = width / U, all = A.moves * per;  // below 2^18: the stage holds them
  const int dm = kThreads / per, du = kThreads % per;
  const int m0 = threadIdx.x / per, u0 = threadIdx.x % per;
  const auto each = [&](auto look, auto act) {
    int m = m0, u = u0;
    for (int i = threadIdx.x; i < all; i += N * kThreads) {
      int ms[N], us[N], rows[N];
#pragma unroll
      for (int j = 0; j < N; ++j) {
        ms[j] = m, us[j] = u * U;
        rows[j] = i + j * kThreads < all ? look(m) : kSkip;
        m += dm, u += du;
        if (u >= per) u -= per, ++m;
      }
#pragma unroll
      for (int j = 0; j < N; ++j)
        if (rows[j] != kSkip) act(ms[j], us[j], rows[j]);
    }
  };
  each([&](int m) { return A.source[m]; },
       [&](int m, int u, int s) { to_shared<U>(stage + m * width + u, base + s * row + u); });
  asm volatile("cp.async.wait_all;" ::: "memory");
  __syncthreads();
  each([&](int m) { return A.target[m]; },
       [&](int m, int u, int t) {
         W w{};
         if (t >= 0) w = *reinterpret_cast<const W*>(stage + m * width + u);
         *reinterpret_cast<W*>(base + (t >= 0 ? t : kSkip - 1 - t) * row + u) = w;
       });
}

__global__ void __launch_bounds__(kThreads) pool_copy_kernel(const PoolArgs A) {
  extern __shared__ __align__(16) unsigned char stage[];
  int p = 0;
  while (p + 1 < A.pools && (int)blockIdx.x >= A.first[p + 1]) ++p;
  const long long at = (long long)(blockIdx.x - A.first[p]) * A.width[p];
  const int width = (int)min((long long)A.width[p], A.row[p] - at);
  char* base = A.base[p] + at;
  if (A.unit[p] == 16)
    copy_slice<16>(A, base, A.row[p], width, stage);
  else if (A.unit[p] == 8)
    copy_slice<8>(A, base, A.row[p], width, stage);
  else if (A.unit[p] == 4)
    copy_slice<4>(A, base, A.row[p], width, stage);
  else
    copy_slice<1>(A, base, A.row[p], width, stage);
}

// Rows that no other move reads or writes, in pieces of kPiece bytes.
constexpr int kPiece = 16 * 1024;
template <int U> __device__ __forceinline__ void copy_piece(char* to, const char* from, int bytes) {
  using W = typename Word<U>::T;
  constexpr int N = 4;
  for (int i = threadIdx.x * U; i < bytes; i += N * kThreads * U) {
    W w[N];
#pragma unroll
    for (int j = 0; j < N; ++j)
      if (i + j * kThreads * U < bytes) w[j] = *reinterpret_cast<const W*>(from + i + j * kThreads * U);
#pragma unroll
    for (int j = 0; j < N; ++j)
      if (i + j * kThreads * U < bytes) *reinterpret_cast<W*>(to + i + j * kThreads * U) = w[j];
  }
}
__global__ void __launch_bounds__(kThreads) pool_move_kernel(const PoolArgs A) {
  const int moves = *A.count;
  for (int p = 0; p < A.pools; ++p) {
    const long long row = A.row[p], pieces = (row + kPiece - 1) / kPiece;
    for (long long i = blockIdx.x; i < moves * pieces; i += gridDim.x) {
      const long long m = i / pieces, at = (i - m * pieces) * kPiece;
      const int bytes = (int)min((long long)kPiece, row - at);
      char* to = A.base[p] + A.target[m] * row + at;
      const char* from = A.base[p] + A.source[m] * row + at;
      if (A.unit[p] == 16)
        copy_piece<16>(to, from, bytes);
      else if (A.unit[p] == 8)
        copy_piece<8>(to, from, bytes);
      else if (A.unit[p] == 4)
        copy_piece<4>(to, from, bytes);
      else
        copy_piece<1>(to, from, bytes);
    }
  }
}

int check_pools(const hyfft_pool* pools, int32_t n, int64_t slots) {
  if (!pools || n < 1 || n > HYFFT_MAX_POOLS) return set_error(HYFFT_ERR_INVALID, "slots: 1 to 16 pools");
  if (slots < 1) return set_error(HYFFT_ERR_INVALID, "slots: a pool needs a slot");
  if (slots > (1ll << 30)) return set_error(HYFFT_ERR_UNSUPPORTED, "slots: more than 2^30");
  for (int p = 0; p < n; ++p)
    if (!pools[p].data || pools[p].row_bytes < 1) return set_error(HYFFT_ERR_INVALID, "slots: null or empty pool");
  return HYFFT_OK;
}

PoolArgs args_of(const hyfft_pool* pools, int32_t n) {
  PoolArgs A{};
  A.pools = n;
  for (int p = 0; p < n; ++p) {
    A.base[p] = static_cast<char*>(pools[p].data), A.row[p] = pools[p].row_bytes;
    const uintptr_t both = reinterpret_cast<uintptr_t>(pools[p].data) | (uintptr_t)pools[p].row_bytes;
    A.unit[p] = both % 16 == 0 ? 16 : both % 8 == 0 ? 8 : both % 4 == 0 ? 4 : 1;
  }
  return A;
}

}  // namespace
}  // namespace hyfft

using namespace hyfft;

extern "C" int hyfft_pool_workspace_size(int64_t slots, int64_t moves, size_t* copy_bytes, size_t* compact_bytes) {
  if (slots < 1 || moves < 0) return set_error(HYFFT_ERR_INVALID, "slots: bad sizes");
  if (!copy_bytes || !compact_bytes) return set_error(HYFFT_ERR_INVALID, "slots: null size");
  *copy_bytes = sizeof(int) * (size_t)(slots + 2 * moves);
  *compact_bytes = sizeof(int) * (size_t)(2 * slots + 1);
  return HYFFT_OK;
}

extern "C" int hyfft_pool_copy(const hyfft_pool* pools, int32_t n, int64_t slots, const int32_t* source, const int32_t* target,
                               int64_t moves, void* workspace, size_t workspace_bytes, void* stream) {
  if (int rc = check_pools(pools, n, slots)) return rc;
  if (moves < 0) return set_error(HYFFT_ERR_INVALID, "slots: negative number of moves");
  if (!moves) return HYFFT_OK;
  if (!source || !target) return set_error(HYFFT_ERR_INVALID, "slots: null list");
  if (moves * 16 > (long long)kStageMost) return set_error(HYFFT_ERR_UNSUPPORTED, "slots: more than 12800 moves at once");
  size_t need = 0, other = 0;
  if (int rc = hyfft_pool_workspace_size(slots, moves, &need, &other)) return rc;
  if (!workspace || workspace_bytes < need) return set_error(HYFFT_ERR_WORKSPACE, "slots: workspace too small");
  if (bind_device_of(pools[0].data) != HYFFT_OK) return set_error(HYFFT_ERR_CUDA, "slots: device");
  PoolArgs A = args_of(pools, n);
  int* owner = static_cast<int*>(workspace);
  int* from = owner + slots;
  int* to = from + moves;
  A.source = from, A.target = to, A.moves = (int)moves;
  // As wide a slice of the rows as a CTA's share of shared memory holds, and narrow enough for two CTAs an SM
  long long total = 0;
  for (int p = 0; p < n; ++p) total += A.row[p];
  long long width = std::min<long long>(kStageBytes / moves, std::max(128ll, total / 296));
  // below 64 bytes rather more shared memory (2000 rows of 16 KB reordered: 24.6 us with 64, 30.5 with 32)
  if (width < 64) width = std::min<long long>(64, kStageMost / moves);
  width = width >= 128 ? width / 128 * 128 : width >= 64 ? 64 : width >= 32 ? 32 : 16;
  long long ctas = 0;
  size_t smem = 0;
  for (int p = 0; p < n; ++p) {
    A.width[p] = (int)std::min(width, A.row[p]);
    A.first[p] = (int)ctas;
    ctas += (A.row[p] + A.width[p] - 1) / A.width[p];
    smem = std::max(smem, (size_t)A.width[p] * (size_t)moves);
    if (ctas > 0x7fffffffLL) return set_error(HYFFT_ERR_UNSUPPORTED, "slots: rows too long");
  }
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (smem > 48 * 1024 && !kernel_smem_once(reinterpret_cast<const void*>(pool_copy_kernel), kStageMost))
    return set_error(HYFFT_ERR_CUDA, "slots: shared memory");
  plan_copy_kernel<<<1, kPlanThreads, 0, st>>>(source, target, (int)moves, (int)slots, owner, from, to);
  pool_copy_kernel<<<(unsigned)ctas, kThreads, smem, st>>>(A);
  if (cudaGetLastError() != cudaSuccess) return set_error(HYFFT_ERR_CUDA, "slots: kernel launch failed");
  g_launches.fetch_add(2, std::memory_order_relaxed);
  return HYFFT_OK;
}

extern "C" int hyfft_pool_compact(const hyfft_pool* pools, int32_t n, int64_t slots, const uint8_t* live, int32_t* moved,
                                  void* workspace, size_t workspace_bytes, void* stream) {
  if (int rc = check_pools(pools, n, slots)) return rc;
  if (!live || !moved) return set_error(HYFFT_ERR_INVALID, "slots: null list");
  size_t need = 0, other = 0;
  if (int rc = hyfft_pool_workspace_size(slots, 0, &other, &need)) return rc;
  if (!workspace || workspace_bytes < need) return set_error(HYFFT_ERR_WORKSPACE, "slots: workspace too small");
  if (bind_device_of(pools[0].data) != HYFFT_OK) return set_error(HYFFT_ERR_CUDA, "slots: device");
  PoolArgs A = args_of(pools, n);
  int* movers = static_cast<int*>(workspace);
  int* holes = movers + slots;
  int* count = holes + slots;
  A.source = movers, A.target = holes, A.count = count;
  long long pieces = 0;
  for (int p = 0; p < n; ++p) pieces = std::max(pieces, (A.row[p] + kPiece - 1) / kPiece * ((slots + 1) / 2));
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  plan_compact_kernel<<<1, kPlanThreads, 0, st>>>(live, (int)slots, movers, holes, count, moved);
  pool_move_kernel<<<(unsigned)std::min<long long>(pieces, 148 * 8), kThreads, 0, st>>>(A);
  if (cudaGetLastError() != cudaSuccess) return set_error(HYFFT_ERR_CUDA, "slots: kernel launch failed");
  g_launches.fetch_add(2, std::memory_order_relaxed);
  return HYFFT_OK;
}
