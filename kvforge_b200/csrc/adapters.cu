// Low-rank adapters of many requests at once, beside a projection that they share: row n of the result is
//   out[n][c] = base[n][c] + sum_r B[s][c][r] * (scale[s] * sum_k A[s][section(c)][r][k] x[n][k]),   s = ids[n],
// and base[n] where s is -1.  A section is one of the matrices that are stacked in the projection (queries, keys, values);
// of gates and ups that alternate in blocks of 8 columns the sections alternate too.
#include "common.cuh"

using namespace kvf;

namespace {

constexpr int THREADS = 256;
constexpr int MAX_SECTIONS = 4;

struct AdapterParams {
  const void* x;
  const void* a;        // [S][sections][R][K]
  const void* b;        // [S][N][R]
  const float* scales;  // [S]
  const int* ranks;     // [S] or null: all R
  const int* ids;       // [n]
  const void* base;
  void* out;
  int* err;
  long long x_stride, base_stride, out_stride;
  int n, S, sections, R, K, N;
  int ends[MAX_SECTIONS];  // sections' last columns + 1 (not alternating)
  int alternating;
};

__device__ __forceinline__ int section_of(const AdapterParams& p, int c) {
  if (p.alternating) return (c >> 3) & 1;
  int s = 0;
  while (s + 1 < p.sections && c >= p.ends[s]) ++s;
  return s;
}

template <typename T, typename O>
__global__ void __launch_bounds__(THREADS) adapter_rows_kernel(AdapterParams p) {
  pdl_launch();
  pdl_wait();
  extern __shared__ float h[];  // [sections][R]
  const int row = blockIdx.x;
  int s = p.ids[row];
  if (s < -1 || s >= p.S) {
    if (threadIdx.x == 0 && p.err) atomicOr(p.err, 32);
    s = -1;
  }
  const O* base = reinterpret_cast<const O*>(p.base) + row * p.base_stride;
  O* out = reinterpret_cast<O*>(p.out) + row * p.out_stride;
  if (s < 0) {
    if (p.out != p.base)
      for (int c = threadIdx.x; c < p.N; c += THREADS) out[c] = base[c];
    return;
  }
  const int total = p.sections * p.R, rank = p.ranks ? min(p.ranks[s], p.R) : p.R;
  const T* x = reinterpret_cast<const T*>(p.x) + row * p.x_stride;
  const T* a = reinterpret_cast<const T*>(p.a) + (long long)s * total * p.K;
  const T* b = reinterpret_cast<const T*>(p.b) + (long long)s * p.N * p.R;
  for (int t = threadIdx.x >> 5; t < total; t += THREADS / 32) {
    float sum = 0.f;
    for (int k = threadIdx.x & 31; k < p.K; k += 32) sum += to_float(a[(long long)t * p.K + k]) * to_float(x[k]);
    sum = warp_sum(sum);
    if ((threadIdx.x & 31) == 0) h[t] = sum * p.scales[s];
  }
  __syncthreads();
  for (int c = threadIdx.x; c < p.N; c += THREADS) {
    const float* hs = h + section_of(p, c) * p.R;
    float sum = 0.f;
    for (int r = 0; r < rank; ++r) sum += to_float(b[(long long)c * p.R + r]) * hs[r];
    out[c] = from_float<O>(to_float(base[c]) + sum);
  }
}

}  // namespace

KVF_API int kvf_adapters_set_pdl(int on) {
  g_pdl_enabled = on;
  return 0;
}

#define KVF_ADAPTER_API(SUF, T)                                                                                                                                          \
  KVF_API int kvf_adapter_add_##SUF(const void* x, long long x_stride, const void* a, const void* b, const float* scales, const int* ranks, const int* ids, int n, int S, \
                                    int sections, int R, int K, int N, int end0, int end1, int end2, int alternating, const void* base, long long base_stride, void* out, \
                                    long long out_stride, int wide, int* err, cudaStream_t st) {                                                                         \
    if (n <= 0) return 0;                                                                                                                                                \
    if (sections < 1 || sections > MAX_SECTIONS) return (int)cudaErrorInvalidValue;                                                                                      \
    AdapterParams p{x, a, b, scales, ranks, ids, base, out, err, x_stride, base_stride, out_stride, n, S, sections, R, K, N, {end0, end1, end2, N}, alternating};         \
    const size_t smem = (size_t)sections * R * sizeof(float);                                                                                                            \
    if (wide) return launch(adapter_rows_kernel<T, float>, dim3(n), dim3(THREADS), smem, st, p);                                                                         \
    return launch(adapter_rows_kernel<T, T>, dim3(n), dim3(THREADS), smem, st, p);                                                                                       \
  }
KVF_ADAPTER_API(f32, float)
KVF_ADAPTER_API(bf16, bf16)
