// What a choice of beams moves: pages of the paged cache and rows of the recurrent states.
//
// A copy is a pair (source, target); no target is a source or the target of another pair, so copies need no order.  A pair with an
// index outside the pool copies nothing.
// Bound by bytes: 192 pages of 32 layers of 8 heads of 128 (428 MB read and written) 67 us, 6.4 TB/s; 20 states of 13.8 MB 66 us (a
// source that two targets share is read once).
#include "common.cuh"

using namespace kvf;

namespace {

constexpr int THREADS = 256;

struct PageTensor {
  char* base;        // [entries][blocks][heads][block_size][row bytes]
  int row;           // bytes of one position of one head
};

template <typename U>
__device__ __forceinline__ void copy_runs(const PageTensor& t, long long entry, int src, int dst, int blocks, int heads, int bs, int tokens) {
  const int run = tokens * (t.row / (int)sizeof(U)), page = bs * (t.row / (int)sizeof(U));
  U* base = reinterpret_cast<U*>(t.base) + entry * blocks * ((long long)heads * page);
  const U* from = base + (long long)src * heads * page;
  U* to = base + (long long)dst * heads * page;
  for (int i = threadIdx.x; i < heads * run; i += THREADS) {
    const int h = i / run, r = i - h * run;
    to[h * page + r] = from[h * page + r];
  }
}

// grid: (pairs, entries)
template <typename U>
__global__ void __launch_bounds__(THREADS) copy_pages_kernel(PageTensor k, PageTensor v, const int* __restrict__ src, const int* __restrict__ dst,
                                                              const int* __restrict__ tokens, int blocks, int heads, int bs) {
  pdl_launch();
  pdl_wait();
  const int p = blockIdx.x;
  const int s = src[p], d = dst[p], n = tokens ? min(tokens[p], bs) : bs;
  if (s < 0 || s >= blocks || d < 0 || d >= blocks || n <= 0 || s == d) return;
  copy_runs<U>(k, blockIdx.y, s, d, blocks, heads, bs, n);
  if (v.base) copy_runs<U>(v, blockIdx.y, s, d, blocks, heads, bs, n);
}

struct StateRow {
  char* base;
  long long stride;  // bytes from a slot to the next
  long long bytes;   // of a slot's state
};

// grid: (stretches, pairs, tensors)
template <typename U, int PER>
__global__ void __launch_bounds__(THREADS) copy_states_kernel(const StateRow* __restrict__ rows, const int* __restrict__ src, const int* __restrict__ dst, int slots) {
  pdl_launch();
  const StateRow r = rows[blockIdx.z];
  pdl_wait();
  const int s = src[blockIdx.y], d = dst[blockIdx.y];
  if (s < 0 || s >= slots || d < 0 || d >= slots || s == d) return;
  const long long n = r.bytes / (long long)sizeof(U);
  const U* from = reinterpret_cast<const U*>(r.base + s * r.stride);
  U* to = reinterpret_cast<U*>(r.base + d * r.stride);
  const long long at = (long long)blockIdx.x * (THREADS * PER) + threadIdx.x;
  U buf[PER];
#pragma unroll
  for (int i = 0; i < PER; ++i)
    if (at + i * THREADS < n) buf[i] = from[at + i * THREADS];
#pragma unroll
  for (int i = 0; i < PER; ++i)
    if (at + i * THREADS < n) to[at + i * THREADS] = buf[i];
}

}  // namespace

KVF_API int kvf_copy_pages(void* k, void* v, int k_row, int v_row, const int* src, const int* dst, const int* tokens, int pairs, int entries, int blocks, int heads, int bs,
                           int unit, cudaStream_t st) {
  if (pairs <= 0 || entries <= 0) return 0;
  if (entries > 65535 || (unit != 16 && unit != 4 && unit != 2)) return (int)cudaErrorInvalidValue;
  const PageTensor tk{(char*)k, k_row}, tv{(char*)v, v_row};
  const dim3 grid(pairs, entries), block(THREADS);
  if (unit == 16) return launch(copy_pages_kernel<uint4>, grid, block, 0, st, tk, tv, src, dst, tokens, blocks, heads, bs);
  if (unit == 4) return launch(copy_pages_kernel<uint32_t>, grid, block, 0, st, tk, tv, src, dst, tokens, blocks, heads, bs);
  return launch(copy_pages_kernel<uint16_t>, grid, block, 0, st, tk, tv, src, dst, tokens, blocks, heads, bs);
}

// rows: per tensor (base, bytes from slot to slot, bytes of a slot), 64 bits each, on the device; most: the largest of the last
KVF_API int kvf_copy_states(const void* rows, int tensors, long long most, const int* src, const int* dst, int pairs, int slots, int unit, cudaStream_t st) {
  if (pairs <= 0 || tensors <= 0 || most <= 0) return 0;
  if (pairs > 65535 || tensors > 65535 || (unit != 16 && unit != 4)) return (int)cudaErrorInvalidValue;
  constexpr int PER = 4;
  const long long each = (long long)THREADS * PER * unit;
  const dim3 grid((unsigned)((most + each - 1) / each), pairs, tensors), block(THREADS);
  const StateRow* r = reinterpret_cast<const StateRow*>(rows);
  if (unit == 16) return launch(copy_states_kernel<uint4, PER>, grid, block, 0, st, r, src, dst, slots);
  return launch(copy_states_kernel<uint32_t, PER>, grid, block, 0, st, r, src, dst, slots);
}
