// The best continuations of a prompt's beams: of score[b] + logit[b][t] - log(sum_t' exp(logit[b][t'])) over the W rows of
// a prompt and the V tokens the K highest, best first, of equal ones the lowest b V + t.
// A score that is no number (a row with a NaN, an infinity or nothing but masked tokens) and a beam whose own score is not
// finite count as minus infinity; a place without a candidate above that gets parent and token -1.
//
// Kernel 1, a CTA a row: maximum, sum of exponentials, then the K highest logits one after another.
// Kernel 2, a CTA a prompt: the K highest of the W K scores, in 64 bits.
#include "common.cuh"

using namespace kvf;

namespace {

constexpr int MAX_K = 64;
constexpr int MAX_W = 64;
constexpr int THREADS = 256;

typedef unsigned long long u64;

__device__ __forceinline__ unsigned ordered_key(float v) {  // (-0 and 0 are one value)
  const unsigned b = __float_as_uint(v + 0.f);
  return (b & 0x80000000u) ? ~b : (b | 0x80000000u);
}
__device__ __forceinline__ float key_value(unsigned k) { return __uint_as_float((k & 0x80000000u) ? (k & 0x7fffffffu) : ~k); }
// logit and place as one number, larger for a larger logit and, of equal ones, a lower place
__device__ __forceinline__ u64 pack(float v, unsigned at) { return ((u64)ordered_key(v) << 32) | (0xffffffffu - at); }

__device__ __forceinline__ u64 block_max_u64(u64 v, u64* red) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const u64 t = __shfl_xor_sync(0xffffffffu, v, o);
    v = t > v ? t : v;
  }
  __syncthreads();
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  u64 r = 0;
  for (int i = 0; i < THREADS / 32; ++i) r = red[i] > r ? red[i] : r;
  return r;
}

// row record in the workspace: log of the sum, then K candidates
__global__ void __launch_bounds__(THREADS) beam_rows_kernel(const float* __restrict__ logits, long long stride, int V, int K, double* __restrict__ lse, u64* __restrict__ cand) {
  __shared__ u64 red[THREADS / 32];
  __shared__ double sums[THREADS / 32];
  const float* row = logits + blockIdx.x * stride;
  float m = -INFINITY;
  bool bad = false;
  for (int i = threadIdx.x; i < V; i += THREADS) {
    m = fmaxf(m, row[i]);
    bad |= isnan(row[i]);
  }
  m = key_value((unsigned)(block_max_u64((u64)ordered_key(m), red)));
  bad = __syncthreads_or(bad);
  double s = 0;
  for (int i = threadIdx.x; i < V; i += THREADS) s += (double)expf(row[i] - m);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
  if ((threadIdx.x & 31) == 0) sums[threadIdx.x >> 5] = s;
  __syncthreads();
  if (threadIdx.x == 0) {
    double t = 0;
    for (int i = 0; i < THREADS / 32; ++i) t += sums[i];
    lse[blockIdx.x] = (bad || isinf(m)) ? (double)NAN : (double)m + log(t);
  }
  u64 last = ~0ull;
  for (int k = 0; k < K; ++k) {
    u64 best = 0;
    for (int i = threadIdx.x; i < V; i += THREADS) {
      const u64 c = pack(row[i], i);
      if (c < last && c > best) best = c;
    }
    best = block_max_u64(best, red);
    if (threadIdx.x == 0) cand[(long long)blockIdx.x * K + k] = best;
    last = best;
  }
}

__global__ void __launch_bounds__(THREADS) beam_merge_kernel(const float* __restrict__ scores, int W, int K, const double* __restrict__ lse, const u64* __restrict__ cand,
                                                              int* __restrict__ parents, int* __restrict__ tokens, float* __restrict__ best) {
  extern __shared__ double sc[];  // W K scores, then what rows and tokens they have
  u64* at = reinterpret_cast<u64*>(sc + W * K);
  const int row0 = blockIdx.x * W;
  for (int i = threadIdx.x; i < W * K; i += THREADS) {
    const int b = row0 + i / K;
    const u64 c = cand[(long long)b * K + i % K];
    double v = (double)scores[b] + ((double)key_value((unsigned)(c >> 32)) - lse[b]);
    if (c == 0 || isnan(v) || !isfinite(scores[b])) v = -INFINITY;
    sc[i] = v;
    at[i] = ((u64)(i / K) << 32) | (0xffffffffu - (unsigned)c);
  }
  __syncthreads();
  // rank of every candidate by (score, then place)
  const int o = blockIdx.x * K;
  for (int i = threadIdx.x; i < W * K; i += THREADS) {
    int rank = 0;
    for (int j = 0; j < W * K; ++j) rank += sc[j] > sc[i] || (sc[j] == sc[i] && (at[j] < at[i] || (at[j] == at[i] && j < i)));
    if (rank < K) {
      const bool none = sc[i] == -INFINITY;
      parents[o + rank] = none ? -1 : (int)(at[i] >> 32);
      tokens[o + rank] = none ? -1 : (int)(unsigned)at[i];
      best[o + rank] = (float)sc[i];
    }
  }
}

}  // namespace

KVF_API int kvf_beams_set_pdl(int on) {
  g_pdl_enabled = on;
  return 0;
}

KVF_API int kvf_beam_select_f32(const float* logits, long long stride, int prompts, int W, int V, int K, const float* scores, void* work, int* parents, int* tokens,
                                float* best, cudaStream_t st) {
  if (prompts <= 0) return 0;
  if (W < 1 || W > MAX_W || K < 1 || K > MAX_K || V < 1) return (int)cudaErrorInvalidValue;
  double* lse = reinterpret_cast<double*>(work);
  u64* cand = reinterpret_cast<u64*>(lse + (long long)prompts * W);
  int rc = launch(beam_rows_kernel, dim3(prompts * W), dim3(THREADS), 0, st, logits, stride, V, K, lse, cand);
  if (rc) return rc;
  const size_t smem = (size_t)W * K * 16;
  if (smem > 48 * 1024) cudaFuncSetAttribute(beam_merge_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
  return launch(beam_merge_kernel, dim3(prompts), dim3(THREADS), smem, st, scores, W, K, (const double*)lse, (const u64*)cand, parents, tokens, best);
}
