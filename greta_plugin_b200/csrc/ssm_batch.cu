// Metadata of a packed serving batch from the requests' lengths, in one launch:
// token offsets, has_initial, request and position of every token, block
// tables grown from a list of free blocks, and the tokens' slots in a paged
// cache.
//
// A few numbers per request and token, so latency is all: one launch in place
// of a chain of prefix sums, searches and gathers (and of a repeat_interleave
// that waits for the host). Every CTA sums the lengths of all requests for
// itself, in shared memory (2 x 4 bytes a request), rather than waiting for a
// first kernel, and then takes its 512 tokens: a binary search for the token's
// request there, one table entry. A new block of a request always begins at
// one of the step's tokens (position b * block_size >= its context), so that
// token's thread writes the table entry; no thread reads an entry that another
// writes, since what a new block is follows from the sums alone. 256 requests of
// one token: 4.0 us; 1024 requests, 8192 tokens: 6.0 us.
#include "ssm_launch.cuh"

namespace greta {
namespace ssm {
namespace {

constexpr int kThreads = 512;
constexpr int kMaxRequests = 16384;  // 128 KB of sums

struct BatchParams {
  const int *query, *context;
  int n;
  long long T;
  int *starts, *seq_idx;
  signed char* has_initial;
  long long *positions, *slot_map;
  int* tables;  // null: no paged cache
  long long s_row;
  int width, bs;
  const int* free_list;
  long long nfree;
  int* used;
};

__device__ __forceinline__ long long blocks_of(long long tokens, int bs) { return (tokens + bs - 1) / bs; }

__global__ void __launch_bounds__(kThreads) batch_metadata_kernel(const BatchParams p) {
  extern __shared__ int sums[];  // starts [n + 1], first new block [n + 1]
  __shared__ long long warp_q[kThreads / 32], warp_b[kThreads / 32];
  int* starts = sums;
  int* first = sums + p.n + 1;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  pdl_wait();
  pdl_trigger();
  long long run_q = 0, run_b = 0;
  const long long kMost = INT_MAX;
  for (int base = 0; base < p.n; base += kThreads) {
    const int i = base + threadIdx.x;
    long long q = 0, c = 0, b = 0;
    if (i < p.n) {
      q = max(p.query[i], 0);
      c = max(p.context[i], 0);
      if (p.tables != nullptr) b = blocks_of(c + q, p.bs) - blocks_of(c, p.bs);
      if (blockIdx.x == 0) p.has_initial[i] = c > 0;
    }
    long long sq = q, sb = b;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const long long xq = __shfl_up_sync(0xffffffffu, sq, o), xb = __shfl_up_sync(0xffffffffu, sb, o);
      if (lane >= o) {
        sq += xq;
        sb += xb;
      }
    }
    if (lane == 31) {
      warp_q[warp] = sq;
      warp_b[warp] = sb;
    }
    __syncthreads();
    long long before_q = run_q, before_b = run_b;
    for (int w = 0; w < kThreads / 32; ++w) {
      if (w < warp) {
        before_q += warp_q[w];
        before_b += warp_b[w];
      }
      run_q += warp_q[w];
      run_b += warp_b[w];
    }
    if (i < p.n) {
      // offsets past the rows that there are end there (the packed calls read
      // no further); sums past 2^31 stay at its end
      starts[i] = (int)min(before_q + sq - q, p.T);
      first[i] = (int)min(before_b + sb - b, kMost);
      if (blockIdx.x == 0) p.starts[i] = starts[i];
    }
    __syncthreads();
  }
  if (threadIdx.x == 0) {
    starts[p.n] = (int)min(run_q, p.T);
    if (blockIdx.x == 0) {
      p.starts[p.n] = starts[p.n];
      if (p.used != nullptr) *p.used = (int)min(run_b, kMost);
    }
  }
  __syncthreads();
  const long long t = (long long)blockIdx.x * kThreads + threadIdx.x;
  if (t >= p.T) return;
  int req = -1;
  long long pos = 0, slot = -1;
  if (t < starts[p.n]) {
    int lo = 0, hi = p.n;  // starts[lo] <= t < starts[hi]
    while (hi - lo > 1) {
      const int mid = (lo + hi) / 2;
      if (starts[mid] <= t)
        lo = mid;
      else
        hi = mid;
    }
    req = lo;
    const long long c = max(p.context[req], 0);
    pos = c + t - starts[req];
    if (p.tables != nullptr) {
      const long long blk = pos / p.bs, fresh = blk - blocks_of(c, p.bs);
      if (blk < p.width) {
        int* entry = p.tables + req * p.s_row + blk;
        int id;
        if (fresh >= 0) {
          const long long at = first[req] + fresh;
          id = at < p.nfree ? p.free_list[at] : -1;
          if (pos % p.bs == 0) *entry = id;
        } else {
          id = *entry;
        }
        if (id >= 0) slot = (long long)id * p.bs + pos % p.bs;
      }
    }
  }
  p.seq_idx[t] = req;
  p.positions[t] = pos;
  if (p.slot_map != nullptr) p.slot_map[t] = slot;
}

}  // namespace
}  // namespace ssm
}  // namespace greta

using namespace greta;
using namespace greta::ssm;

extern "C" int greta_ssm_batch_metadata(const int32_t* query_lens, const int32_t* context_lens, int64_t num_reqs,
                                        int64_t T, int32_t* starts, int8_t* has_initial, int32_t* seq_idx,
                                        int64_t* positions, int32_t* block_tables, int64_t s_row, int64_t width,
                                        int64_t block_size, const int32_t* free_blocks, int64_t num_free,
                                        int64_t* slot_map, int32_t* blocks_used, void* stream) {
  if (num_reqs < 0 || T < 0 || T >= INT_MAX) return GRETA_ERR_INVALID_ARG;
  if (num_reqs > kMaxRequests) return GRETA_ERR_UNSUPPORTED;
  if (starts == nullptr || (num_reqs > 0 && (query_lens == nullptr || context_lens == nullptr || has_initial == nullptr)))
    return GRETA_ERR_INVALID_ARG;
  if (T > 0 && (seq_idx == nullptr || positions == nullptr)) return GRETA_ERR_INVALID_ARG;
  if (block_tables != nullptr) {
    if (block_size < 1 || block_size > INT_MAX || width < 0 || width > INT_MAX || s_row < width || num_free < 0)
      return GRETA_ERR_INVALID_ARG;
    if ((num_free > 0 && free_blocks == nullptr) || blocks_used == nullptr || (T > 0 && slot_map == nullptr))
      return GRETA_ERR_INVALID_ARG;
  }
  BatchParams p{};
  p.query = query_lens; p.context = context_lens; p.n = (int)num_reqs; p.T = T;
  p.starts = starts; p.seq_idx = seq_idx;
  p.has_initial = reinterpret_cast<signed char*>(has_initial);
  p.positions = reinterpret_cast<long long*>(positions);
  if (block_tables != nullptr) {
    p.tables = block_tables; p.s_row = s_row; p.width = (int)width; p.bs = (int)block_size;
    p.free_list = free_blocks; p.nfree = num_free;
    p.slot_map = reinterpret_cast<long long*>(slot_map);
    p.used = blocks_used;
  }
  const size_t smem = sizeof(int) * 2 * (size_t)(num_reqs + 1);
  // (the limit is the kernel's, for all host threads: a call that set its own size
  // could take away what another's launch was just allowed)
  cudaError_t e = cudaSuccess;
  if (smem > 48 * 1024) e = allow_smem(batch_metadata_kernel, sizeof(int) * 2 * (kMaxRequests + 1));
  if (e != cudaSuccess) return GRETA_ERR_LAUNCH;
  const unsigned blocks = (unsigned)(T > 0 ? cdiv(T, kThreads) : 1);
  return finish(launch(batch_metadata_kernel, dim3(blocks), dim3(kThreads), smem,
                       reinterpret_cast<cudaStream_t>(stream), p));
}
