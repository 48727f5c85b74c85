// The best continuations of a prompt's beams: of score[b] + logit[b][t] - log(sum_t' exp(logit[b][t'])) over the W rows of
// a prompt and the V tokens the K highest, best first, of equal ones the lowest b V + t.
// A score that is no number (a row with a NaN, an infinity or nothing but masked tokens) and a beam whose own score is not
// finite count as minus infinity; a place without a candidate above that gets parent and token -1.
//
// One pass over the logits, one launch.  A CTA walks a stretch of a row, sixteen logits a thread at a time with the next sixteen on
// their way, and leaves the stretch's maximum, its sum of exponentials below that maximum and its K highest logits; the CTA that
// finishes a prompt's last stretch joins the sums and chooses among the stretches' candidates.
// The K highest are found without a sort: every warp's m-th highest thread maximum (m = K / 8 rounded up) has at least K numbers of the CTA
// at or above the least of the eight, a bound that rises as the walk goes on and that a few dozen numbers of a stretch pass; those are
// gathered, and each counts the ones above it.  Where too many pass (rows of one value), the K highest are taken one after another.
// Measured: 512 rows of 128,256 logits (64 prompts of eight beams, K = 16) 56 us, 4.7 TB/s.  No unit is full: 14 instructions a logit and warp
// take 43 % of the issue slots, DRAM is busy half of the time; of the 12.2 cycles between two instructions of a warp 3.7 go to logits on their
// way, 3.0 to instructions before it, and the 512 CTAs leave every seventh of the 592 places empty.  Four rows 9.4 us, of which the walk is 1.5,
// the choice 1, the ticket 1, the join 3 and the launch the rest.
// Order is decided in 64 bits (a logit with its place; a score in double with its place), so equal numbers never depend on which
// thread comes first; sums of sixteen exponentials are in float, all that joins them is in double and in one order.
#include "common.cuh"

using namespace kvf;

namespace {

constexpr int MAX_K = 64;
constexpr int MAX_W = 64;
constexpr int THREADS = 256;
constexpr int WARPS = THREADS / 32;
constexpr int E = 16;               // logits a thread holds at a time
constexpr int BATCH = THREADS * E;  // logits a CTA holds at a time
constexpr int CAP = 768;            // candidates that are gathered

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
__device__ __forceinline__ float ex2(float v) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
  return r;
}

__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}
// two floats at once
__device__ __forceinline__ u64 two(float a, float b) {
  u64 r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ void apart(u64 v, float& a, float& b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v)); }
__device__ __forceinline__ u64 add2(u64 a, u64 b) {
  u64 r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ u64 mul2(u64 a, u64 b) {
  u64 r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ u64 fma2(u64 a, u64 b, u64 c) {
  u64 r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}

// A candidate: `hi`, then `lo`, the larger one first.
struct Cand {
  u64 hi;
  unsigned lo;
};
__device__ __forceinline__ int above(const Cand& a, const Cand& b) { return (a.hi > b.hi) | ((a.hi == b.hi) & (a.lo > b.lo)); }  // (without a branch)

struct Shared {
  u64 hi[CAP];
  u64 hi2[CAP];
  unsigned lo[CAP];
  unsigned lo2[CAP];
  u64 out_hi[MAX_K];
  unsigned out_lo[MAX_K];
  alignas(16) unsigned least[WARPS];
  float warp_max[WARPS];
  double warp_sum[WARPS];
  double lse[MAX_W];
  Cand round[WARPS];
  int n, n2, last;
};

// The warp's m-th highest of its threads' numbers (not 0).
__device__ __forceinline__ unsigned warp_mth(unsigned top, int m) {
  unsigned w = 0;
  for (int i = 0; i < m; ++i) {
    w = __reduce_max_sync(0xffffffffu, top);
    if (i + 1 < m) {
      const unsigned who = __ballot_sync(0xffffffffu, top == w);
      if ((threadIdx.x & 31) == __ffs(who) - 1) top = 0;
    }
  }
  return w;
}
// The least of what the warps have posted; they post numbers that rise, so one posted before is a bound too.
__device__ __forceinline__ unsigned posted_bound(const Shared& sh) {
  static_assert(WARPS == 8, "two loads of four");
  uint32_t a, b, c, d, e, f, g, h;
  const uint32_t at = (uint32_t)__cvta_generic_to_shared(sh.least);
  asm volatile("ld.volatile.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(a), "=r"(b), "=r"(c), "=r"(d) : "r"(at) : "memory");
  asm volatile("ld.volatile.shared.v4.u32 {%0, %1, %2, %3}, [%4 + 16];" : "=r"(e), "=r"(f), "=r"(g), "=r"(h) : "r"(at) : "memory");
  return max(min(min(min(a, b), min(c, d)), min(min(e, f), min(g, h))), NOTHING + 1);
}
template <bool LO>
__device__ __forceinline__ void put(const Cand& c, Shared& sh) {
  const int at = atomicAdd(&sh.n, 1);
  if (at < CAP) {
    sh.hi[at] = c.hi;
    if (LO) sh.lo[at] = c.lo;
  }
}

// The K highest of what was put (all of those at or above `bound`, a number of `key`), into out_hi / out_lo, best first; returns how many
// there are.  `each(f)` hands every number there is to f, for when more were put than there is room for.  Begins and ends with a barrier.
// LO: `lo` differs between candidates of equal `hi` (else there are none).
template <bool LO, class Key, class Each>
__device__ __forceinline__ int k_highest(int K, Shared& sh, unsigned bound, Key key, Each each) {
  if (threadIdx.x == 0) sh.n2 = 0;
  __syncthreads();
  int n = sh.n;
  if (n <= CAP) {
    // the bound rose after some had been put
    for (int i = threadIdx.x; i < n; i += THREADS) {
      if (key(sh.hi[i]) >= bound) {
        const int at = atomicAdd(&sh.n2, 1);
        sh.hi2[at] = sh.hi[i];
        if (LO) sh.lo2[at] = sh.lo[i];
      }
    }
    __syncthreads();
    n = sh.n2;
    for (int i = threadIdx.x; i < n; i += THREADS) {
      const Cand c{sh.hi2[i], LO ? sh.lo2[i] : 0};
      int rank = 0;
#pragma unroll 8
      for (int j = 0; j < n; ++j) rank += LO ? above(Cand{sh.hi2[j], sh.lo2[j]}, c) : (int)(sh.hi2[j] > c.hi);
      if (rank < K) {
        sh.out_hi[rank] = c.hi;
        if (LO) sh.out_lo[rank] = c.lo;
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
  int prompts, W, V, K;
  int batches;    // of a stretch
  int stretches;  // of a row
  int* tickets;   // [prompts] stretches done: zeros between calls
  double* sums;   // [rows][stretches]
  float* maxima;  // [rows][stretches]
  u64* cands;     // [rows][stretches][K]
  int* parents;
  int* tokens;
  float* best;
};

template <bool VEC>
__device__ __forceinline__ int place(int first, int e) { return first + (VEC ? 4 * threadIdx.x + (e >> 2) * (4 * THREADS) + (e & 3) : threadIdx.x + e * THREADS); }

template <bool VEC>
__device__ __forceinline__ void load_batch(float (&v)[E], const float* x, int first, int V) {
  if (first + BATCH <= V) {
    if (VEC) {
#pragma unroll
      for (int q = 0; q < E / 4; ++q) {
        const float4 f = __ldcs(reinterpret_cast<const float4*>(x + place<VEC>(first, 4 * q)));
        v[4 * q] = f.x, v[4 * q + 1] = f.y, v[4 * q + 2] = f.z, v[4 * q + 3] = f.w;
      }
    } else {
#pragma unroll
      for (int e = 0; e < E; ++e) v[e] = __ldcs(x + place<VEC>(first, e));
    }
  } else {  // the row's last batch
#pragma unroll
    for (int e = 0; e < E; ++e) v[e] = place<VEC>(first, e) < V ? __ldcs(x + place<VEC>(first, e)) : -INFINITY;
  }
}

// What a thread knows of its part of the stretch.
struct Walk {
  float high = -INFINITY;  // the thread's highest logit
  float m = -INFINITY;     // the warp's
  double s = 0.;           // the thread's sum of exponentials below m
};

template <bool VEC>
__device__ __forceinline__ void walk_batch(Walk& t, const float (&v)[E], int at, bool begins, int mth, Shared& sh) {
  constexpr float L2E = 1.4426950408889634f, L2E_LOW = (float)(1.4426950408889634 - (double)L2E);
  float top = max3(v[0], v[1], -INFINITY);  // (a NaN is passed over here and shows in the sum)
#pragma unroll
  for (int e = 2; e < E; e += 2) top = max3(top, v[e], v[e + 1]);
  t.high = fmaxf(t.high, top);
  const unsigned key = ordered_key(t.high);
  const float wm = key_value(__reduce_max_sync(0xffffffffu, key));
  const unsigned w = warp_mth(key, mth);
  if ((threadIdx.x & 31) == 0) *(volatile unsigned*)&sh.least[threadIdx.x >> 5] = w;
  if (begins) __syncthreads();
  const float least = key_value(posted_bound(sh));
  if (top >= least) {
#pragma unroll
    for (int e = 0; e < E; ++e)
      if (v[e] >= least) put<false>(Cand{pack(v[e], place<VEC>(at, e)), 0}, sh);
  }
  if (wm > t.m) {
    t.s *= (double)ex2((t.m - wm) * L2E);
    t.m = wm;
  }
  const float below = t.m > -INFINITY ? -t.m : 0.f;
  const u64 shift = two(below, below), scale = two(L2E, L2E), low = two(L2E_LOW, L2E_LOW);
  u64 part = 0;
#pragma unroll
  for (int e = 0; e < E; e += 2) {
    const u64 d = add2(two(v[e], v[e + 1]), shift);  // exact for the logits that weigh most
    float a, b;
    apart(fma2(d, scale, mul2(d, low)), a, b);
    part = add2(part, two(ex2(a), ex2(b)));
  }
  float a, b;
  apart(part, a, b);
  t.s += (double)(a + b);
}

// VEC: rows begin at multiples of 16 bytes, four logits a load.  All rows of a call are dealt out to threads alike, so that equal rows have
// equal sums and their candidates are ties.
template <bool VEC>
__global__ void __launch_bounds__(THREADS, 4) beam_select_kernel(BeamParams p) {
  pdl_launch();
  __shared__ Shared sh;
  const int row = blockIdx.x / p.stretches, stretch = blockIdx.x - row * p.stretches;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const float* x = p.logits + (long long)row * p.stride;
  const int K = p.K, V = p.V, mth = (K + WARPS - 1) / WARPS;
  const int first = stretch * p.batches * BATCH;
  const int batches = min(p.batches, (V - first + BATCH - 1) / BATCH);
  if (threadIdx.x == 0) sh.n = 0;
  float v[E], next[E];
  Walk t;
  pdl_wait();
  load_batch<VEC>(v, x, first, V);
  for (int b = 0; b < batches; b += 2) {
    const int at = first + b * BATCH;
    if (b + 1 < batches) load_batch<VEC>(next, x, at + BATCH, V);
    walk_batch<VEC>(t, v, at, b == 0, mth, sh);
    if (b + 1 < batches) {
      if (b + 2 < batches) load_batch<VEC>(v, x, at + 2 * BATCH, V);
      walk_batch<VEC>(t, next, at + BATCH, false, mth, sh);
    }
  }
  {
    double d = t.s;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) d += __shfl_xor_sync(0xffffffffu, d, o);
    if (lane == 0) {
      sh.warp_max[warp] = t.m;
      sh.warp_sum[warp] = d;
    }
  }
  __syncthreads();
  const long long rec = (long long)row * p.stretches + stretch;
  const int found = k_highest<false>(
      K, sh, posted_bound(sh), [](u64 hi) { return (unsigned)(hi >> 32); },
      [&](auto see) {
        for (int i = first + threadIdx.x; i < min(V, first + batches * BATCH); i += THREADS)
          if (x[i] > -INFINITY) see(Cand{pack(x[i], i), 0});
      });
  for (int k = threadIdx.x; k < K; k += THREADS) p.cands[rec * K + k] = k < found ? sh.out_hi[k] : 0;
  if (warp == 1) {
    float hi = lane < WARPS ? sh.warp_max[lane] : -INFINITY;
    const float all = warp_max(hi);
    double d = 0;
    if (lane < WARPS) {
      d = sh.warp_sum[lane];
      if (hi > -INFINITY) d *= (double)expf(hi - all);
    }
#pragma unroll
    for (int o = 4; o > 0; o >>= 1) d += __shfl_xor_sync(0xffffffffu, d, o);
    if (lane == 0) {
      p.sums[rec] = d;
      p.maxima[rec] = all;
    }
  }
  const int prompt = row / p.W, row0 = prompt * p.W;
  __syncthreads();
  if (threadIdx.x == 0) {
    // what the CTA wrote is seen by whoever sees its ticket
    int done;
    asm volatile("atom.acq_rel.gpu.global.add.s32 %0, [%1], 1;" : "=r"(done) : "l"(p.tickets + prompt) : "memory");
    sh.last = done == p.W * p.stretches - 1;
    if (sh.last) p.tickets[prompt] = 0;
    sh.n = 0;
  }
  __syncthreads();
  if (!sh.last) return;

  // ---- the prompt: the rows' logarithms of the sums, a warp a row
  for (int b = warp; b < p.W; b += WARPS) {
    const long long r0 = (long long)(row0 + b) * p.stretches;
    // (a lane joins its stretches one after another: one each up to 32 stretches)
    float hi = -INFINITY;
    double d = 0;
    for (int i = lane; i < p.stretches; i += 32) {
      const float next = __ldcg(p.maxima + r0 + i);
      const double part = __ldcg(p.sums + r0 + i);
      const float both = fmaxf(hi, next);
      if (both > -INFINITY || isnan(part)) d = d * (double)expf(hi - both) + part * (double)expf(next - both);
      hi = both;
    }
    const float all = warp_max(hi);
    if (hi > -INFINITY) d *= (double)expf(hi - all);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) d += __shfl_xor_sync(0xffffffffu, d, o);
    if (lane == 0) sh.lse[b] = isinf(all) ? (double)NAN : (double)all + log(d);
  }
  __syncthreads();
  // ---- the K highest of the stretches' candidates: scores in double; the bound goes by the scores rounded to floats (a rounding keeps the order)
  const int each_row = p.stretches * K, every = p.W * each_row;
  const u64* cands = p.cands + (long long)row0 * each_row;
  auto candidate = [&](int i) {
    const int b = i / each_row;
    const u64 c = __ldcg(cands + i);
    const float own = __ldg(p.scores + row0 + b);
    double sc = (double)own + ((double)key_value((unsigned)(c >> 32)) - sh.lse[b]);
    if (c == 0 || isnan(sc) || !isfinite(own) || (float)sc == -INFINITY) sc = -INFINITY;
    return Cand{ordered_key64(sc), 0xffffffffu - ((unsigned)b * V + (0xffffffffu - (unsigned)c))};
  };
  auto score_key = [](u64 hi) { return ordered_key((float)key_value64(hi)); };
  // (a stretch's candidates are in order: every warp takes some of all ranks, or the least of the warps' bounds would be a low one)
  unsigned top = 0;
  for (int i0 = 0, turn = 0; i0 < every; i0 += THREADS, turn += 37) {
    const int i = i0 + ((threadIdx.x * 5 + turn) & (THREADS - 1));
    if (i >= every) continue;
    const Cand c = candidate(i);
    top = max(top, score_key(c.hi));
    if (every <= CAP) sh.hi[i] = c.hi, sh.lo[i] = c.lo;  // all of them have room
  }
  const unsigned w = warp_mth(top, mth);
  if (lane == 0) sh.least[warp] = w;
  if (threadIdx.x == 0 && every <= CAP) sh.n = every;
  __syncthreads();
  const unsigned bound = posted_bound(sh);
  if (every > CAP) {
    for (int i = threadIdx.x; i < every; i += THREADS) {
      const Cand c = candidate(i);
      if (score_key(c.hi) >= bound) put<true>(c, sh);
    }
  }
  const int chosen = k_highest<true>(K, sh, bound, score_key, [&](auto see) {
    for (int i = threadIdx.x; i < every; i += THREADS) {
      const Cand c = candidate(i);
      if (key_value64(c.hi) > -INFINITY) see(c);
    }
  });
  for (int k = threadIdx.x; k < K; k += THREADS) {
    const bool none = k >= chosen || sh.out_hi[k] == 0;
    const unsigned at = 0xffffffffu - sh.out_lo[k];
    p.parents[prompt * K + k] = none ? -1 : (int)(at / V);
    p.tokens[prompt * K + k] = none ? -1 : (int)(at % V);
    p.best[prompt * K + k] = none ? -INFINITY : (float)key_value64(sh.out_hi[k]);
  }
}

// Batches a CTA walks: CTAs run four to an SM, each costs about two batches besides those it walks, and what counts is the number of
// times the device fills up with them.
int batches_of(long long rows, int V) {
  const int all = (V + BATCH - 1) / BATCH;
  int best = 1;
  long long least = -1;
  for (int b = 1; b <= all; ++b) {
    const long long ctas = rows * ((all + b - 1) / b);
    const long long cost = ((ctas + 4 * 148 - 1) / (4 * 148)) * (b + 2);
    if (least < 0 || cost < least) least = cost, best = b;
    if (b > 64) break;
  }
  return best;
}

}  // namespace

KVF_API int kvf_beams_set_pdl(int on) {
  g_pdl_enabled = on;
  return 0;
}

// work: `words` eight-byte words; the first quarter holds the tickets, zeros between calls, whatever the sizes of a call.  The rest takes
// the records: K + 2 words a stretch (of at least 4,096 logits).
KVF_API int kvf_beam_select_f32(const float* logits, long long stride, int prompts, int W, int V, int K, const float* scores, void* work, long long words, int* parents,
                                int* tokens, float* best, cudaStream_t st) {
  if (prompts <= 0) return 0;
  const long long rows = (long long)prompts * W;
  if (W < 1 || W > MAX_W || K < 1 || K > MAX_K || V < 1 || (long long)W * V > 0x7fff0000ll) return (int)cudaErrorInvalidValue;
  BeamParams p;
  p.batches = batches_of(rows, V);
  p.stretches = ((V + BATCH - 1) / BATCH + p.batches - 1) / p.batches;
  const long long quarter = words / 4, records = rows * p.stretches;
  if (prompts > 2 * quarter || records * (K + 2) > words - quarter || records > 0x7fffffffll) return (int)cudaErrorInvalidValue;
  p.logits = logits, p.stride = stride, p.scores = scores;
  p.prompts = prompts, p.W = W, p.V = V, p.K = K;
  p.tickets = reinterpret_cast<int*>(work);
  u64* at = reinterpret_cast<u64*>(work) + quarter;
  p.cands = at, at += records * K;
  p.sums = reinterpret_cast<double*>(at), at += records;
  p.maxima = reinterpret_cast<float*>(at);
  p.parents = parents, p.tokens = tokens, p.best = best;
  const dim3 grid((unsigned)records), block(THREADS);
  const bool vec = stride % 4 == 0 && (reinterpret_cast<uintptr_t>(logits) & 15) == 0;
  return vec ? launch(beam_select_kernel<true>, grid, block, 0, st, p) : launch(beam_select_kernel<false>, grid, block, 0, st, p);
}
