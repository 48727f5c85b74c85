// The best continuations of a prompt's beams: of score[b] + logit[b][t] - log(sum_t' exp(logit[b][t'])) over the W rows of
// a prompt and the V tokens the K highest, best first, of equal ones the lowest b V + t.
// A score that is no number (a row with a NaN, an infinity or nothing but masked tokens) and a beam whose own score is not
// finite count as minus infinity; a place without a candidate above that gets parent and token -1.
//
// One pass over the logits, one launch.  A CTA holds a stretch of a row in registers (8 or 32 logits a thread) and leaves the
// stretch's maximum, its sum of exponentials below that maximum and its K highest logits; the CTA that finishes a row's last
// stretch does the same with the stretches' candidates, and the one that finishes a prompt's last row chooses among the rows'.
// In each of the three steps the K highest are found without a sort: every warp's m-th highest thread maximum (m = K / 8 rounded
// up) has at least K numbers of the CTA at or above the least of them, a bound that a few dozen numbers pass; those are gathered
// and each counts the ones above it.  Where too many pass (rows of one value), the K highest are taken one after another.
// Order is decided in 64 bits (a logit with its place; a score in double with its place), so equal numbers never depend on
// which thread comes first; the sums of exponentials are joined in double in the order of the stretches.
#include "common.cuh"

using namespace kvf;

namespace {

constexpr int MAX_K = 64;
constexpr int MAX_W = 64;
constexpr int THREADS = 256;
constexpr int WARPS = THREADS / 32;
constexpr int CAP = 512;  // candidates that are ranked by counting

typedef unsigned long long u64;

__device__ __forceinline__ unsigned ordered_key(float v) {
  const unsigned b = __float_as_uint(v + 0.f);  // (-0 and 0 are one value)
  return (b & 0x80000000u) ? ~b : (b | 0x80000000u);
}
__device__ __forceinline__ float key_value(unsigned k) { return __uint_as_float((k & 0x80000000u) ? (k & 0x7fffffffu) : ~k); }
__device__ __forceinline__ u64 ordered_key64(double v) {
  const u64 b = (u64)__double_as_longlong(v + 0.0);
  return (b >> 63) ? ~b : (b | 0x8000000000000000ull);
}
__device__ __forceinline__ double key_value64(u64 k) { return __longlong_as_double((long long)((k >> 63) ? (k & 0x7fffffffffffffffull) : ~k)); }
// logit and place as one number, larger for a larger logit and, of equal ones, a lower place
__device__ __forceinline__ u64 pack(float v, unsigned at) { return ((u64)ordered_key(v) << 32) | (0xffffffffu - at); }
constexpr unsigned NOTHING = 0x007fffffu;  // ordered_key(-inf): what does not count

// A candidate: `hi`, then `lo`, the larger one first.
struct Cand {
  u64 hi;
  unsigned lo;
};
__device__ __forceinline__ bool above(const Cand& a, const Cand& b) { return a.hi > b.hi || (a.hi == b.hi && a.lo > b.lo); }

struct Shared {
  u64 hi[CAP];
  unsigned lo[CAP];
  u64 out_hi[MAX_K];
  unsigned out_lo[MAX_K];
  unsigned least[WARPS];
  float warp_max[WARPS];
  double warp_sum[WARPS];
  Cand round[WARPS];
  int n, last, bad;
};

// A bound that at least K of the CTA's numbers reach, if it holds that many (`top`: the thread's highest, ordered).
__device__ __forceinline__ unsigned bound_of(unsigned top, int K, Shared& sh) {
  const int m = (K + WARPS - 1) / WARPS;
  unsigned w = 0;
  for (int i = 0; i < m; ++i) {
    w = __reduce_max_sync(0xffffffffu, top);
    const unsigned who = __ballot_sync(0xffffffffu, top == w);
    if ((threadIdx.x & 31) == __ffs(who) - 1) top = 0;
  }
  if ((threadIdx.x & 31) == 0) sh.least[threadIdx.x >> 5] = w;
  if (threadIdx.x == 0) sh.n = 0;
  __syncthreads();
  unsigned least = sh.least[0];
#pragma unroll
  for (int i = 1; i < WARPS; ++i) least = min(least, sh.least[i]);
  return max(least, NOTHING + 1);
}

// The K highest of what `each(f)` hands to f(candidate) on every thread, into out_hi / out_lo, best first; returns how many there are.
// `gather(put)`: calls put(candidate) for those at or above the bound.
template <class Gather, class Each>
__device__ __forceinline__ int k_highest(int K, Shared& sh, Gather gather, Each each) {
  gather([&](const Cand& c) {
    const int at = atomicAdd(&sh.n, 1);
    if (at < CAP) {
      sh.hi[at] = c.hi;
      sh.lo[at] = c.lo;
    }
  });
  __syncthreads();
  const int n = sh.n;
  if (n <= CAP) {
    for (int i = threadIdx.x; i < n; i += THREADS) {
      const Cand c{sh.hi[i], sh.lo[i]};
      int rank = 0;
      for (int j = 0; j < n; ++j) rank += above(Cand{sh.hi[j], sh.lo[j]}, c);
      if (rank < K) {
        sh.out_hi[rank] = c.hi;
        sh.out_lo[rank] = c.lo;
      }
    }
    __syncthreads();
    return min(n, K);
  }
  Cand last{~0ull, ~0u};
  for (int k = 0; k < K; ++k) {
    Cand best{0, 0};
    each([&](const Cand& c) {
      if (above(last, c) && above(c, best)) best = c;
    });
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      const Cand t{__shfl_xor_sync(0xffffffffu, best.hi, o), __shfl_xor_sync(0xffffffffu, best.lo, o)};
      if (above(t, best)) best = t;
    }
    __syncthreads();
    if ((threadIdx.x & 31) == 0) sh.round[threadIdx.x >> 5] = best;
    __syncthreads();
    best = sh.round[0];
    for (int i = 1; i < WARPS; ++i)
      if (above(sh.round[i], best)) best = sh.round[i];
    if (threadIdx.x == 0) {
      sh.out_hi[k] = best.hi;
      sh.out_lo[k] = best.lo;
    }
    last = best;
  }
  __syncthreads();
  return K;
}

struct BeamParams {
  const float* logits;
  long long stride;
  const float* scores;
  int prompts, W, V, K, stretches;
  int* tickets;    // [rows] stretches done, [prompts] rows done: zeros between calls
  double* sums;    // [rows][stretches]
  float* maxima;   // [rows][stretches]
  u64* cands;      // [rows][stretches][K]
  double* lse;     // [rows]
  u64* row_cands;  // [rows][K]
  int* parents;
  int* tokens;
  float* best;
};

// Whether this CTA is the last of `of` that come here; what the others wrote before is then visible.
__device__ __forceinline__ bool last_of(int* ticket, int of, Shared& sh) {
  if (of == 1) {
    __syncthreads();
    return true;
  }
  __threadfence();
  __syncthreads();
  if (threadIdx.x == 0) {
    const int t = atomicAdd(ticket, 1);
    sh.last = t == of - 1;
    if (sh.last) *ticket = 0;
  }
  __syncthreads();
  if (sh.last) __threadfence();
  return sh.last;
}

// VEC: rows begin at multiples of 16 bytes, four logits a load.  All rows of a call are dealt out to threads alike, so that equal rows have
// equal sums and their candidates are ties.
template <int E, bool VEC>
__global__ void __launch_bounds__(THREADS, E > 16 ? 3 : 4) beam_select_kernel(BeamParams p) {
  pdl_launch();
  __shared__ Shared sh;
  const int row = blockIdx.x / p.stretches, stretch = blockIdx.x - row * p.stretches;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const float* x = p.logits + (long long)row * p.stride;
  const int K = p.K;
  float v[E];
  const int first = stretch * (THREADS * E) + (VEC ? 4 : 1) * threadIdx.x;
  const auto place = [&](int e) { return first + (VEC ? (e >> 2) * (4 * THREADS) + (e & 3) : e * THREADS); };
  pdl_wait();
  if (VEC) {
#pragma unroll
    for (int q = 0; q < E / 4; ++q) {
      const int i = place(4 * q);
      if (i + 4 <= p.V) {
        const float4 f = __ldcs(reinterpret_cast<const float4*>(x + i));
        v[4 * q] = f.x, v[4 * q + 1] = f.y, v[4 * q + 2] = f.z, v[4 * q + 3] = f.w;
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) v[4 * q + e] = i + e < p.V ? __ldcs(x + i + e) : -INFINITY;
      }
    }
  } else {
#pragma unroll
    for (int e = 0; e < E; ++e) v[e] = place(e) < p.V ? __ldcs(x + place(e)) : -INFINITY;
  }
  float top = v[0];
  bool bad = false;
#pragma unroll
  for (int e = 0; e < E; ++e) {
    top = fmaxf(top, v[e]);
    bad |= isnan(v[e]);
  }
  if (isnan(top)) top = -INFINITY;
  {
    const float w = warp_max(top);
    if (lane == 0) sh.warp_max[warp] = w;
  }
  const unsigned bound = bound_of(ordered_key(top), K, sh);  // (a barrier lies in it)
  float m = sh.warp_max[0];
#pragma unroll
  for (int i = 1; i < WARPS; ++i) m = fmaxf(m, sh.warp_max[i]);
  const float least = key_value(bound);
  {
    // a stretch with nothing in it has no sum; a NaN or an infinity leaves NaN
    float s = 0.f;
    if (m > -INFINITY) {
#pragma unroll
      for (int e = 0; e < E; ++e) s += expf(v[e] - m);
    }
    if (bad) s = NAN;
    double d = s;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) d += __shfl_xor_sync(0xffffffffu, d, o);
    if (lane == 0) sh.warp_sum[warp] = d;
  }
  const int found = k_highest(
      K, sh,
      [&](auto put) {
        if (top >= least) {
#pragma unroll
          for (int e = 0; e < E; ++e)
            if (v[e] >= least) put(Cand{pack(v[e], place(e)), 0});
        }
      },
      [&](auto see) {
#pragma unroll
        for (int e = 0; e < E; ++e)
          if (v[e] > -INFINITY) see(Cand{pack(v[e], place(e)), 0});
      });
  const long long rec = (long long)row * p.stretches + stretch;
  for (int k = threadIdx.x; k < K; k += THREADS) p.cands[rec * K + k] = k < found ? sh.out_hi[k] : 0;
  if (threadIdx.x == 0) {
    double s = 0;
#pragma unroll
    for (int i = 0; i < WARPS; ++i) s += sh.warp_sum[i];
    p.sums[rec] = s;
    p.maxima[rec] = m;
  }
  if (!last_of(p.tickets + row, p.stretches, sh)) return;

  // ---- the row: its logarithm of the sum, and the K highest of the stretches' candidates
  const long long rec0 = (long long)row * p.stretches;
  {
    float rm = -INFINITY;
    for (int i = threadIdx.x; i < p.stretches; i += THREADS) rm = fmaxf(rm, __ldcg(p.maxima + rec0 + i));
    rm = warp_max(rm);
    if (lane == 0) sh.warp_max[warp] = rm;
    __syncthreads();
    rm = sh.warp_max[0];
#pragma unroll
    for (int i = 1; i < WARPS; ++i) rm = fmaxf(rm, sh.warp_max[i]);
    double s = 0;
    for (int i = threadIdx.x; i < p.stretches; i += THREADS) {
      const float sm = __ldcg(p.maxima + rec0 + i);
      const double part = __ldcg(p.sums + rec0 + i);
      if (sm > -INFINITY || isnan(part)) s += part * exp((double)sm - (double)rm);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    if (lane == 0) sh.warp_sum[warp] = s;
    __syncthreads();
    if (threadIdx.x == 0) {
      double t = 0;
#pragma unroll
      for (int i = 0; i < WARPS; ++i) t += sh.warp_sum[i];
      p.lse[row] = isinf(rm) ? (double)NAN : (double)rm + log(t);
    }
  }
  const u64* cands = p.cands + rec0 * K;
  const int total = p.stretches * K;
  unsigned high = 0;
  for (int i = threadIdx.x; i < total; i += THREADS) high = max(high, (unsigned)(__ldcg(cands + i) >> 32));
  const unsigned row_bound = bound_of(high, K, sh);
  const int row_found = k_highest(
      K, sh,
      [&](auto put) {
        for (int i = threadIdx.x; i < total; i += THREADS) {
          const u64 c = __ldcg(cands + i);
          if ((unsigned)(c >> 32) >= row_bound) put(Cand{c, 0});
        }
      },
      [&](auto see) {
        for (int i = threadIdx.x; i < total; i += THREADS) {
          const u64 c = __ldcg(cands + i);
          if (c) see(Cand{c, 0});
        }
      });
  for (int k = threadIdx.x; k < K; k += THREADS) p.row_cands[(long long)row * K + k] = k < row_found ? sh.out_hi[k] : 0;
  const int prompt = row / p.W, row0 = prompt * p.W;
  if (!last_of(p.tickets + p.prompts * p.W + prompt, p.W, sh)) return;

  // ---- the prompt: scores in double; the bound goes by the scores rounded to floats (a rounding keeps the order)
  const int all = p.W * K;
  auto candidate = [&](int i) {
    const int b = i / K;
    const u64 c = __ldcg(p.row_cands + (long long)row0 * K + i);
    const float own = __ldg(p.scores + row0 + b);
    double s = (double)own + ((double)key_value((unsigned)(c >> 32)) - __ldcg(p.lse + row0 + b));
    if (c == 0 || isnan(s) || !isfinite(own) || (float)s == -INFINITY) s = -INFINITY;
    return Cand{ordered_key64(s), 0xffffffffu - ((unsigned)b * p.V + (0xffffffffu - (unsigned)c))};
  };
  unsigned score = 0;
  for (int i = threadIdx.x; i < all; i += THREADS) score = max(score, ordered_key((float)key_value64(candidate(i).hi)));
  const unsigned prompt_bound = bound_of(score, K, sh);
  const int chosen = k_highest(
      K, sh,
      [&](auto put) {
        for (int i = threadIdx.x; i < all; i += THREADS) {
          const Cand c = candidate(i);
          if (ordered_key((float)key_value64(c.hi)) >= prompt_bound) put(c);
        }
      },
      [&](auto see) {
        for (int i = threadIdx.x; i < all; i += THREADS) {
          const Cand c = candidate(i);
          if (key_value64(c.hi) > -INFINITY) see(c);
        }
      });
  for (int k = threadIdx.x; k < K; k += THREADS) {
    const bool none = k >= chosen || sh.out_hi[k] == 0;
    const unsigned at = 0xffffffffu - sh.out_lo[k];
    p.parents[prompt * K + k] = none ? -1 : (int)(at / p.V);
    p.tokens[prompt * K + k] = none ? -1 : (int)(at % p.V);
    p.best[prompt * K + k] = none ? -INFINITY : (float)key_value64(sh.out_hi[k]);
  }
}

// Logits a CTA: 32 a thread where that still makes four CTAs for every SM (three are on one at a time), else 8.
int stretches_of(int V, int per) { return (V + THREADS * per - 1) / (THREADS * per); }
int per_thread(long long rows, int V) { return rows * stretches_of(V, 32) >= 4 * 148 ? 32 : 8; }

}  // namespace

KVF_API int kvf_beams_set_pdl(int on) {
  g_pdl_enabled = on;
  return 0;
}

// work: `words` eight-byte words; the first quarter holds the tickets, zeros between calls, whatever the sizes of a call.  The rest takes
// the records: K + 2 words a stretch (of at least 2,048 logits) and K + 1 a row.
KVF_API int kvf_beam_select_f32(const float* logits, long long stride, int prompts, int W, int V, int K, const float* scores, void* work, long long words, int* parents,
                                int* tokens, float* best, cudaStream_t st) {
  if (prompts <= 0) return 0;
  const long long rows = (long long)prompts * W;
  if (W < 1 || W > MAX_W || K < 1 || K > MAX_K || V < 1 || (long long)W * V > 0x7fff0000ll) return (int)cudaErrorInvalidValue;
  const int per = per_thread(rows, V), s = stretches_of(V, per);
  const long long quarter = words / 4;
  if (rows > quarter || rows * (s * (K + 2ll) + K + 1) > words - quarter || rows * s > 0x7fffffffll) return (int)cudaErrorInvalidValue;
  BeamParams p;
  p.logits = logits, p.stride = stride, p.scores = scores;
  p.prompts = prompts, p.W = W, p.V = V, p.K = K, p.stretches = s;
  p.tickets = reinterpret_cast<int*>(work);
  u64* at = reinterpret_cast<u64*>(work) + quarter;
  p.cands = at, at += rows * s * K;
  p.row_cands = at, at += rows * K;
  p.sums = reinterpret_cast<double*>(at), at += rows * s;
  p.lse = reinterpret_cast<double*>(at), at += rows;
  p.maxima = reinterpret_cast<float*>(at);
  p.parents = parents, p.tokens = tokens, p.best = best;
  const dim3 grid((unsigned)(rows * s)), block(THREADS);
  const bool vec = stride % 4 == 0 && (reinterpret_cast<uintptr_t>(logits) & 15) == 0;
  if (per == 32) return vec ? launch(beam_select_kernel<32, true>, grid, block, 0, st, p) : launch(beam_select_kernel<32, false>, grid, block, 0, st, p);
  return vec ? launch(beam_select_kernel<8, true>, grid, block, 0, st, p) : launch(beam_select_kernel<8, false>, grid, block, 0, st, p);
}
