// Low-rank adapters of many requests at once, beside a projection that they share: row n of the result is
//   out[n][c] = base[n][c] + sum_r B[s][c][r] * (scale[s] * sum_k A[s][section(c)][r][k] x[n][k]),   s = ids[n],
// and base[n] where s is -1.  A section is one of the matrices that are stacked in the projection (queries, keys, values);
// of gates and ups that alternate in blocks of 8 columns the sections alternate too.
//
// Neither product needs its operands in shared memory: a lane takes 16 bytes of a row at a time, and which of its k come first in a
// tensor-core step is its own affair as long as x and A (or the inner numbers and B) agree.  bfloat16 goes to the tensor cores
// (mma.sync m16n8k16: sixteen flops or so a byte of x and of A, so bytes and latency bound it, not the products); the numbers between the two
// products are sums in 32 bits and are multiplied as two bfloat16 numbers (2^-17 of each is lost beside a result that is rounded to
// 2^-8), or as three where the result is float.  float32 stays on the FP32 pipes.
//
// Few rows (and float32): one launch.  16 rows of one adapter go to a cluster of eight CTAs: their 64 warps share out the columns of x and A,
// the partial sums meet in shared memory (of the CTA, then of every CTA of the cluster, summed in one order), and each CTA adds its
// eighth of the result's columns.
// Many rows: two launches.  64 rows of one adapter go to a cluster of eight CTAs that make their inner numbers, and then to a CTA every 256
// columns of the result: the first kernel reads x once, the second reads and writes the rows once.
//
// Which rows make a tile: up to 64 rows every cluster finds out for itself; for more a kernel of one CTA sorts the rows once a step.
#include "common.cuh"

using namespace kvf;

namespace {

constexpr int THREADS = 256;
constexpr int WARPS = THREADS / 32;
constexpr int MAX_SECTIONS = 4;
constexpr int TILE = 16;        // rows of a cluster that makes both products
constexpr int LIST = 64;        // rows of a tile of the list
constexpr int CLUSTER = 8;      // CTAs a tile
constexpr int DIRECT = 64;      // up to so many rows are grouped by every cluster itself
constexpr int CHUNK = 48;       // rows of A a warp multiplies at a time
constexpr int PART = CHUNK + 4; // floats from one row of the partial sums to the next
constexpr int AHEAD = 2;        // groups of columns that a warp fetches ahead
constexpr int MOST = 256;       // numbers between the products of a row that are in shared memory at a time (whole sections)

struct AdapterParams {
  const void* x;
  const void* a;        // [S][sections][R][K]
  const void* b;        // [S][N][R]
  const float* scales;  // [S]
  const int* ranks;     // [S] or null: all R
  const int* ids;       // [n]
  const int* rows;      // the rows by adapter, and
  const int* tiles;     // (adapter, first of `rows`, count) of up to LIST rows: null where clusters group for themselves
  bf16* inner;          // the inner numbers of many rows: [tile][split][LIST][sections R]
  const void* base;
  void* out;
  int* err;
  long long x_stride, base_stride, out_stride;
  int n, S, sections, R, K, N;
  // sections: where they begin, how wide they are, and the groups of 32 columns up to their end
  int begin[MAX_SECTIONS], width[MAX_SECTIONS], groups[MAX_SECTIONS];
  int alternating;
};

// A section as a lane needs it (taken from the parameters with fixed indices: an index known only at run time costs a constant load's
// latency each time).
struct Section {
  int sec, begin, width;
};
// The section of group `gi` of 32 columns; gi becomes its number there.
__device__ __forceinline__ Section section_of_group(const AdapterParams& p, int& gi) {
  Section s{0, p.begin[0], p.width[0]};
  int before = 0;
#pragma unroll
  for (int i = 1; i < MAX_SECTIONS; ++i)
    if (gi >= p.groups[i - 1]) s = Section{i, p.begin[i], p.width[i]}, before = p.groups[i - 1];
  gi -= before;
  return s;
}

__device__ __forceinline__ uint32_t sm32(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }
__device__ __forceinline__ void mma(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
               : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void st_cluster(uint32_t addr, uint32_t cta, float4 v) {
  asm volatile(
      "{\n\t.reg .b32 at;\n\t"
      "mapa.shared::cluster.u32 at, %0, %1;\n\t"
      "st.shared::cluster.v4.f32 [at], {%2, %3, %4, %5};\n\t}" ::"r"(addr), "r"(cta), "f"(v.x), "f"(v.y), "f"(v.z), "f"(v.w)
      : "memory");
}
__device__ __forceinline__ void prefetch(const void* p) { asm volatile("prefetch.global.L2 [%0];" ::"l"(p)); }

// Column of the result that is number u of a section.
__device__ __forceinline__ int column(const AdapterParams& p, const Section& s, int u) { return p.alternating ? (u >> 3) * 16 + s.sec * 8 + (u & 7) : s.begin + u; }

// ---- the first product: partial sums over a warp's share of k for 16 rows and CHUNK rows of A, into part[16][PART]
// k goes in steps of 32, eight a lane; step st belongs to warp st % 64 of the cluster
struct Rows {
  const char* lo;  // the lane's row g, or null
  const char* hi;  // and g + 8
};

__device__ __forceinline__ void first_product(const AdapterParams& p, const bf16* a, const Rows& x, int t0, int total, int R16, int gw, float* part) {
  const int lane = threadIdx.x & 31, g = lane >> 2, q = lane & 3;
  float acc[CHUNK / 8][4];
#pragma unroll
  for (int j = 0; j < CHUNK / 8; ++j)
#pragma unroll
    for (int i = 0; i < 4; ++i) acc[j][i] = 0.f;
  const bf16* rows[CHUNK / 8];
#pragma unroll
  for (int j = 0; j < CHUNK / 8; ++j) {
    const int t = t0 + j * 8 + g;
    const int sec = (t >= R16) + (t >= 2 * R16) + (t >= 3 * R16);
    rows[j] = t < total ? a + (long long)(sec * (p.R - R16) + t) * p.K : nullptr;
  }
  const uint4 zero = make_uint4(0, 0, 0, 0);
  constexpr int STEP = 32 * CLUSTER * WARPS;
  for (int k0 = gw * 32; k0 < p.K; k0 += 2 * STEP) {  // (all lanes take every step: K may end inside one)
    // the loads of two steps go out together
    uint4 lo[2], hi[2], w[2][CHUNK / 8];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int k = k0 + i * STEP + q * 8;
      const bool in = k < p.K;
      lo[i] = x.lo && in ? __ldg(reinterpret_cast<const uint4*>(x.lo + 2ll * k)) : zero;
      hi[i] = x.hi && in ? __ldg(reinterpret_cast<const uint4*>(x.hi + 2ll * k)) : zero;
#pragma unroll
      for (int j = 0; j < CHUNK / 8; ++j) w[i][j] = rows[j] && in ? __ldg(reinterpret_cast<const uint4*>(rows[j] + k)) : zero;
    }
#pragma unroll
    for (int i = 0; i < 2; ++i) {
#pragma unroll
      for (int j = 0; j < CHUNK / 8; ++j) {
        mma(acc[j], lo[i].x, hi[i].x, lo[i].y, hi[i].y, w[i][j].x, w[i][j].y);
        mma(acc[j], lo[i].z, hi[i].z, lo[i].w, hi[i].w, w[i][j].z, w[i][j].w);
      }
    }
  }
#pragma unroll
  for (int j = 0; j < CHUNK / 8; ++j) {
    *reinterpret_cast<float2*>(part + g * PART + j * 8 + 2 * q) = make_float2(acc[j][0], acc[j][1]);
    *reinterpret_cast<float2*>(part + (g + 8) * PART + j * 8 + 2 * q) = make_float2(acc[j][2], acc[j][3]);
  }
}

__device__ __forceinline__ float dot8(const float4& a0, const float4& a1, const float4& b0, const float4& b1, float c) {
  c = fmaf(a0.x, b0.x, c), c = fmaf(a0.y, b0.y, c), c = fmaf(a0.z, b0.z, c), c = fmaf(a0.w, b0.w, c);
  return fmaf(a1.w, b1.w, fmaf(a1.z, b1.z, fmaf(a1.y, b1.y, fmaf(a1.x, b1.x, c))));
}

__device__ __forceinline__ void first_product(const AdapterParams& p, const float* a, const Rows& x, int t0, int total, int R16, int gw, float* part) {
  const int lane = threadIdx.x & 31, g = lane >> 2, q = lane & 3;
  const float4 zero = make_float4(0, 0, 0, 0);
  for (int c0 = 0; c0 < CHUNK && t0 + c0 < total; c0 += 8) {
    const int t = t0 + c0, sec = (t >= R16) + (t >= 2 * R16) + (t >= 3 * R16);
    const float* row = a + (long long)(sec * (p.R - R16) + t) * p.K;  // eight rows of one section
    float lo[8], hi[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) lo[j] = hi[j] = 0.f;
    for (int k = gw * 32 + q * 8; k < p.K; k += 32 * CLUSTER * WARPS) {
      const float4* xl = reinterpret_cast<const float4*>(x.lo + 4ll * k);
      const float4* xh = reinterpret_cast<const float4*>(x.hi + 4ll * k);
      const float4 l0 = x.lo ? __ldg(xl) : zero, l1 = x.lo ? __ldg(xl + 1) : zero;
      const float4 h0 = x.hi ? __ldg(xh) : zero, h1 = x.hi ? __ldg(xh + 1) : zero;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float4* w = reinterpret_cast<const float4*>(row + (long long)j * p.K + k);
        const float4 w0 = __ldg(w), w1 = __ldg(w + 1);
        lo[j] = dot8(l0, l1, w0, w1, lo[j]);
        hi[j] = dot8(h0, h1, w0, w1, hi[j]);
      }
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) {
#pragma unroll
      for (int o = 1; o < 4; o <<= 1) {
        lo[j] += __shfl_xor_sync(0xffffffffu, lo[j], o);
        hi[j] += __shfl_xor_sync(0xffffffffu, hi[j], o);
      }
      if (q == 0) {
        part[g * PART + c0 + j] = lo[j];
        part[(g + 8) * PART + c0 + j] = hi[j];
      }
    }
  }
}

// ---- the numbers between the products in shared memory, and the second product: 16 rows and 32 columns a warp
// (bf16: `SPLITS` numbers of 16 bits that add up to each; a row's stride makes the eight rows of a load lie in different banks)
__host__ __device__ inline int inner_stride(int total, int size) { return size == 4 ? total + 4 : total % 32 == 0 ? total + 16 : total; }

template <int SPLITS>
__device__ __forceinline__ void keep_inner(bf16* inner, int total, int row, int t, float v) {
  const int stride = inner_stride(total, 2);
#pragma unroll
  for (int i = 0; i < SPLITS; ++i) {
    const bf16 h = __float2bfloat16_rn(v);
    inner[(i * TILE + row) * stride + t] = h;
    const float f = __bfloat162float(h);
    v = isinf(f) ? 0.f : v - f;  // (an infinity has no rest)
  }
}
template <int SPLITS>
__device__ __forceinline__ void keep_inner(float* inner, int total, int row, int t, float v) {
  inner[row * inner_stride(total, 4) + t] = v;
}

// Where a group of 32 columns of a section lies for a lane, and what of it can be fetched before the inner numbers are there: the first
// sixteen numbers of its rows of B (bf16) and the rows that are added to.
template <typename T, typename O>
struct Group {
  Section s;         // sec < 0: none
  int u0;            // its first column in the section
  int col;           // the lane's first column of the result, or -1
  uint2 w[4];        // bf16: B
  uint4 base[2][sizeof(O) / 2];
};

__device__ __forceinline__ const bf16* b_row(const AdapterParams& p, const bf16* b, const Section& s, int u0, int j) {
  // column 2q + e of the j-th of four tensor-core tiles is column 8q + 2j + e of the 32: a lane's eight results lie side by side
  const int g = (threadIdx.x & 31) >> 2, u = u0 + (g >> 1) * 8 + 2 * j + (g & 1);
  return u < s.width ? b + (long long)column(p, s, u) * p.R : nullptr;
}

template <typename T, typename O>
__device__ __forceinline__ void fetch(Group<T, O>& gr, const AdapterParams& p, const T* b, const O* base0, const O* base1) {
  const int q = threadIdx.x & 3;
  gr.col = -1;
  if (gr.s.sec < 0) return;
  const int u = gr.u0 + 8 * q;
  if (u < gr.s.width) gr.col = column(p, gr.s, u);
  if constexpr (sizeof(T) == 2) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const T* row = b_row(p, b, gr.s, gr.u0, j);
      gr.w[j] = row ? __ldg(reinterpret_cast<const uint2*>(row + 4 * q)) : make_uint2(0, 0);
    }
  }
#pragma unroll
  for (int i = 0; i < (int)sizeof(O) / 2; ++i) {
    if (gr.col >= 0 && base0) gr.base[0][i] = *(reinterpret_cast<const uint4*>(base0 + gr.col) + i);
    if (gr.col >= 0 && base1) gr.base[1][i] = *(reinterpret_cast<const uint4*>(base1 + gr.col) + i);
  }
}

// acc[row half][column]: eight columns a lane
template <int SPLITS, typename O>
__device__ __forceinline__ void second_product(const AdapterParams& p, const bf16* b, const bf16* inner, int total, const Group<bf16, O>& gr, int R16, float (&acc)[2][8]) {
  const int lane = threadIdx.x & 31, g = lane >> 2, q = lane & 3;
  const int stride = inner_stride(total, 2);
  float c[4][4];
#pragma unroll
  for (int j = 0; j < 4; ++j)
#pragma unroll
    for (int i = 0; i < 4; ++i) c[j][i] = 0.f;
  for (int r0 = 0; r0 < R16; r0 += 16) {
    uint2 w[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if (r0 == 0) {
        w[j] = gr.w[j];
      } else {
        const bf16* row = b_row(p, b, gr.s, gr.u0, j);
        w[j] = row ? __ldg(reinterpret_cast<const uint2*>(row + r0 + 4 * q)) : make_uint2(0, 0);
      }
    }
#pragma unroll
    for (int i = 0; i < SPLITS; ++i) {
      const bf16* h = inner + (i * TILE + g) * stride + r0 + 4 * q;
      const uint2 lo = *reinterpret_cast<const uint2*>(h), hi = *reinterpret_cast<const uint2*>(h + 8 * stride);
#pragma unroll
      for (int j = 0; j < 4; ++j) mma(c[j], lo.x, hi.x, lo.y, hi.y, w[j].x, w[j].y);
    }
  }
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    acc[0][2 * j] = c[j][0], acc[0][2 * j + 1] = c[j][1];
    acc[1][2 * j] = c[j][2], acc[1][2 * j + 1] = c[j][3];
  }
}

template <int SPLITS, typename O>
__device__ __forceinline__ void second_product(const AdapterParams& p, const float* b, const float* inner, int total, const Group<float, O>& gr, int R16, float (&acc)[2][8]) {
  const int lane = threadIdx.x & 31, g = lane >> 2;
  const int stride = inner_stride(total, 4);
#pragma unroll
  for (int i = 0; i < 8; ++i) acc[0][i] = acc[1][i] = 0.f;
  if (gr.col < 0) return;
  const float* rows = b + (long long)gr.col * p.R;
  const float* lo = inner + g * stride;
  const float* hi = lo + 8 * stride;
  for (int r = 0; r < R16; r += 4) {
    const float4 l = *reinterpret_cast<const float4*>(lo + r), h = *reinterpret_cast<const float4*>(hi + r);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float4 w = __ldg(reinterpret_cast<const float4*>(rows + (long long)i * p.R + r));
      acc[0][i] = fmaf(w.w, l.w, fmaf(w.z, l.z, fmaf(w.y, l.y, fmaf(w.x, l.x, acc[0][i]))));
      acc[1][i] = fmaf(w.w, h.w, fmaf(w.z, h.z, fmaf(w.y, h.y, fmaf(w.x, h.x, acc[1][i]))));
    }
  }
}

// eight columns of a row: what they were and what is added
__device__ __forceinline__ void add_eight(const uint4 (&base)[2], float* out, const float (&v)[8]) {
#pragma unroll
  for (int i = 0; i < 2; ++i)
    reinterpret_cast<float4*>(out)[i] = make_float4(__uint_as_float(base[i].x) + v[4 * i], __uint_as_float(base[i].y) + v[4 * i + 1], __uint_as_float(base[i].z) + v[4 * i + 2],
                                                    __uint_as_float(base[i].w) + v[4 * i + 3]);
}
__device__ __forceinline__ void add_eight(const uint4 (&base)[1], bf16* out, const float (&v)[8]) {
  float f[8];
  bf16x8_to_float(base[0], f);
  __nv_bfloat162 r[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) r[i] = __floats2bfloat162_rn(f[2 * i] + v[2 * i], f[2 * i + 1] + v[2 * i + 1]);
  *reinterpret_cast<uint4*>(out) = *reinterpret_cast<const uint4*>(r);
}

template <typename O>
__device__ __forceinline__ void copy_rows(const AdapterParams& p, const int* rows, int count, int part, int parts) {
  if (p.out == p.base) return;
  constexpr int PER = 16 / sizeof(O);
  const int each = p.N / PER;  // 16-byte pieces of a row (N is a multiple of 8)
  for (int i = part * THREADS + threadIdx.x; i < count * each; i += parts * THREADS) {
    const int r = rows[i / each], c = i % each * PER;
    *reinterpret_cast<uint4*>(reinterpret_cast<O*>(p.out) + r * p.out_stride + c) = *reinterpret_cast<const uint4*>(reinterpret_cast<const O*>(p.base) + r * p.base_stride + c);
  }
}

// The adapter of a row, -1 for one outside the bank.
__device__ __forceinline__ int valid_id(int id, int S, int* err) {
  if (id >= -1 && id < S) return id;
  if (err) atomicOr(err, 32);
  return -1;
}

// The rows of tile t without a list: the t-th among the rows that are the 1st, 17th, ... of their adapter, and the fifteen of that adapter
// that follow; the count (0: there are fewer tiles).  Tiles that there are come first, so that their CTAs are not kept waiting by those
// of tiles that there are not.  All warps work it out; the first leaves the rows in `rows`.
__device__ __forceinline__ int own_rows(const AdapterParams& p, int t, int* rows, int& s) {
  const int lane = threadIdx.x & 31;
  const unsigned below = (1u << lane) - 1;
  int* err = t == 0 && threadIdx.x < 32 ? p.err : nullptr;
  const int a = lane < p.n ? valid_id(p.ids[lane], p.S, err) : -2;
  const int b = lane + 32 < p.n ? valid_id(p.ids[lane + 32], p.S, err) : -2;
  const int least = p.out == p.base ? 0 : -1;  // rows without an adapter are copied, or stay
  const int ra = __popc(__match_any_sync(0xffffffffu, a) & below);
  int rb = 0;
  if (p.n > 32) {
    rb = __popc(__match_any_sync(0xffffffffu, b) & below);
#pragma unroll
    for (int i = 0; i < 32; ++i) rb += __shfl_sync(0xffffffffu, a, i) == b;
  }
  const unsigned la = __ballot_sync(0xffffffffu, a >= least && ra % TILE == 0), lb = __ballot_sync(0xffffffffu, b >= least && rb % TILE == 0);
  if (t >= __popc(la) + __popc(lb)) return 0;
  const bool mine_a = (la >> lane & 1) && __popc(la & below) == t, mine_b = (lb >> lane & 1) && __popc(la) + __popc(lb & below) == t;
  const int who = __ffs(__ballot_sync(0xffffffffu, mine_a || mine_b)) - 1;
  s = __shfl_sync(0xffffffffu, mine_a ? a : b, who);
  const int before = __shfl_sync(0xffffffffu, mine_a ? ra : rb, who);
  const int count = min(TILE, __popc(__ballot_sync(0xffffffffu, a == s)) + __popc(__ballot_sync(0xffffffffu, b == s)) - before);
  if (threadIdx.x < 32) {
    if (a == s && ra >= before && ra < before + TILE) rows[ra - before] = lane;
    if (b == s && rb >= before && rb < before + TILE) rows[rb - before] = lane + 32;
  }
  return count;
}

// T: type of x, A and B; O: of base and out
template <typename T, typename O, int SPLITS>
__global__ void __cluster_dims__(CLUSTER, 1, 1) __launch_bounds__(THREADS, 2) adapter_tile_kernel(const __grid_constant__ AdapterParams p) {
  extern __shared__ __align__(16) float smem[];  // the warps' partial sums (then the numbers between the products), the CTAs' sums
  __shared__ int rows[TILE];
  pdl_launch();
  pdl_wait();
  const int tile = blockIdx.x / CLUSTER, rank = blockIdx.x % CLUSTER;  // (of the list: a quarter of a tile)
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2;
  int s, count;
  if (p.tiles) {
    const int* entry = p.tiles + tile / (LIST / TILE) * 3;
    const int first = tile % (LIST / TILE) * TILE;
    s = entry[0], count = min(TILE, entry[2] - first);
    if (count > 0 && threadIdx.x < count) rows[threadIdx.x] = p.rows[entry[1] + first + threadIdx.x];
  } else {
    count = own_rows(p, tile, rows, s);
  }
  if (count <= 0) return;  // (the whole cluster)
  __syncthreads();
  const int R = s < 0 ? 0 : p.ranks ? min(max(p.ranks[s], 0), p.R) : p.R;
  if (R == 0) {
    copy_rows<O>(p, rows, count, rank, CLUSTER);
    return;
  }
  asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");
  const int R16 = (R + 15) & ~15;
  const T* a = reinterpret_cast<const T*>(p.a) + (long long)s * p.sections * p.R * p.K;
  const T* b = reinterpret_cast<const T*>(p.b) + (long long)s * p.N * p.R;
  // this CTA's eighth of B and of the rows that are added to comes on its way
  const int per = (p.N / 8 + CLUSTER - 1) / CLUSTER * 8, c0 = rank * per, c1 = min(p.N, c0 + per);
  if (c0 < c1) {
    const char* from = reinterpret_cast<const char*>(b + (long long)c0 * p.R);
    const int bytes = (c1 - c0) * p.R * (int)sizeof(T);
    for (int i = threadIdx.x * 128; i < bytes; i += THREADS * 128) prefetch(from + i);
    const int row = threadIdx.x / (THREADS / TILE), row_bytes = (c1 - c0) * (int)sizeof(O);
    if (row < count) {
      const char* at = reinterpret_cast<const char*>(reinterpret_cast<const O*>(p.base) + rows[row] * p.base_stride + c0);
      for (int i = threadIdx.x % (THREADS / TILE) * 128; i < row_bytes; i += 128 * (THREADS / TILE)) prefetch(at + i);
    }
  }

  // whole sections at a time, as many as there is room for
  const int together = min(p.sections, MOST / R16);
  float* part = smem;                        // [WARPS][TILE][PART]
  float* sums = part + WARPS * TILE * PART;  // [CLUSTER][TILE][total]
  T* inner = reinterpret_cast<T*>(part);     // (once the partial sums are out of the way)
  Rows x;
  {
    const char* from = reinterpret_cast<const char*>(p.x);
    x.lo = g < count ? from + rows[g] * p.x_stride * (long long)sizeof(T) : nullptr;
    x.hi = g + 8 < count ? from + rows[g + 8] * p.x_stride * (long long)sizeof(T) : nullptr;
  }
  const float scale = p.scales[s];
  const O* base0 = g < count ? reinterpret_cast<const O*>(p.base) + rows[g] * p.base_stride : nullptr;
  const O* base1 = g + 8 < count ? reinterpret_cast<const O*>(p.base) + rows[g + 8] * p.base_stride : nullptr;
  O* out0 = g < count ? reinterpret_cast<O*>(p.out) + rows[g] * p.out_stride : nullptr;
  O* out1 = g + 8 < count ? reinterpret_cast<O*>(p.out) + rows[g + 8] * p.out_stride : nullptr;
  for (int sec0 = 0; sec0 < p.sections; sec0 += together) {
    const int sec1 = min(p.sections, sec0 + together), total = (sec1 - sec0) * R16;
    for (int t0 = 0; t0 < total; t0 += CHUNK) {
      first_product(p, a + (long long)sec0 * p.R * p.K, x, t0, total, R16, rank * WARPS + warp, part + warp * TILE * PART);
      // the CTAs of the cluster run, and have read the sums of the sections before: their memory may be written
      if (t0 == 0) asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
      __syncthreads();
      const int wide = min(CHUNK, total - t0);
      const int row = threadIdx.x / (THREADS / TILE), t = threadIdx.x % (THREADS / TILE) * 4;
      static_assert(CHUNK / 4 <= THREADS / TILE, "sixteen threads a row take four numbers each");
      if (t < wide) {
        float4 v = *reinterpret_cast<const float4*>(part + row * PART + t);
#pragma unroll
        for (int w = 1; w < WARPS; ++w) {
          const float4 o = *reinterpret_cast<const float4*>(part + (w * TILE + row) * PART + t);
          v.x += o.x, v.y += o.y, v.z += o.z, v.w += o.w;
        }
        const uint32_t to = sm32(sums + (rank * TILE + row) * total + t0 + t);
#pragma unroll
        for (int c = 0; c < CLUSTER; ++c) st_cluster(to, c, v);
      }
      __syncthreads();
    }
    asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
    // groups of 32 columns of one section, a warp each; the first ones are fetched while the cluster meets
    const int before = sec0 ? p.groups[sec0 - 1] : 0, groups = p.groups[sec1 - 1] - before, mine = (groups + CLUSTER - 1) / CLUSTER;
    const auto group = [&](Group<T, O>& gr, int i) {
      int gi = rank * mine + i;
      gr.s.sec = -1;
      if (i < mine && gi < groups) {
        gi += before;
        gr.s = section_of_group(p, gi);
        gr.u0 = gi * 32;
      }
      fetch(gr, p, b, base0, base1);
    };
    Group<T, O> ahead[AHEAD];
#pragma unroll
    for (int i = 0; i < AHEAD; ++i) group(ahead[i], warp + i * WARPS);
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
    for (int row = threadIdx.x / (THREADS / TILE), t = threadIdx.x % (THREADS / TILE); t < total; t += THREADS / TILE) {
      float v = 0.f;
#pragma unroll
      for (int c = 0; c < CLUSTER; ++c) v += sums[(c * TILE + row) * total + t];
      keep_inner<SPLITS>(inner, total, row, t, v * scale);
    }
    __syncthreads();
    if (sec1 < p.sections) asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");

    for (int i = warp; i < mine; i += AHEAD * WARPS) {
#pragma unroll
      for (int j = 0; j < AHEAD; ++j) {
        const Group<T, O> gr = ahead[j];
        if (gr.s.sec < 0) continue;
        group(ahead[j], i + (j + AHEAD) * WARPS);
        float acc[2][8];
        second_product<SPLITS>(p, b, inner + (gr.s.sec - sec0) * R16, total, gr, R16, acc);
        if (gr.col >= 0 && out0) add_eight(gr.base[0], out0 + gr.col, acc[0]);
        if (gr.col >= 0 && out1) add_eight(gr.base[1], out1 + gr.col, acc[1]);
      }
    }
    __syncthreads();
  }
}

// ---- many rows, first kernel: the inner numbers of 64 rows by a cluster.  A warp multiplies 64 rows by 32 rows of A over its share of k
// (x and A are each read once by a CTA); the eight warps' sums meet in shared memory, and CTA c of the cluster gets all of rows 8c .. 8c + 7.
constexpr int WIDE_CHUNK = 32;
constexpr int WIDE_PART = WIDE_CHUNK + 4;
constexpr int SHARE = LIST / CLUSTER;

template <int SPLITS>
__global__ void __cluster_dims__(CLUSTER, 1, 1) __launch_bounds__(THREADS, 2) adapter_inner_kernel(const __grid_constant__ AdapterParams p) {
  extern __shared__ __align__(16) float smem[];  // [WARPS][LIST][WIDE_PART] partial sums, then [CLUSTER][SHARE][total] sums
  __shared__ long long offset[LIST];  // of the tile's rows in x (bytes), or -1
  pdl_launch();
  pdl_wait();
  const int tile = blockIdx.x / CLUSTER, rank = blockIdx.x % CLUSTER;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, q = lane & 3;
  const int s = p.tiles[3 * tile], first = p.tiles[3 * tile + 1], count = p.tiles[3 * tile + 2];
  if (s < 0 || count <= 0) return;
  const int R = p.ranks ? min(max(p.ranks[s], 0), p.R) : p.R;
  if (R == 0) return;
  if (threadIdx.x < LIST) offset[threadIdx.x] = threadIdx.x < count ? (long long)p.rows[first + threadIdx.x] * p.x_stride * 2 : -1;
  __syncthreads();
  asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");
  const int R16 = (R + 15) & ~15, total = p.sections * R16;
  const bf16* a = reinterpret_cast<const bf16*>(p.a) + (long long)s * p.sections * p.R * p.K;
  const char* x = reinterpret_cast<const char*>(p.x);
  float* sums = smem + WARPS * LIST * WIDE_PART;
  const uint4 zero = make_uint4(0, 0, 0, 0);
  const int tall = (count + 15) / 16;  // sixteens of rows that there are
  for (int t0 = 0; t0 < total; t0 += WIDE_CHUNK) {
    float acc[4][4][4];
#pragma unroll
    for (int m = 0; m < 4; ++m)
#pragma unroll
      for (int j = 0; j < 4; ++j)
#pragma unroll
        for (int i = 0; i < 4; ++i) acc[m][j][i] = 0.f;
    const bf16* rows[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int t = t0 + j * 8 + g, sec = (t >= R16) + (t >= 2 * R16) + (t >= 3 * R16);
      rows[j] = t < total ? a + (long long)(sec * (p.R - R16) + t) * p.K : nullptr;
    }
    for (int k0 = (rank * WARPS + warp) * 32; k0 < p.K; k0 += 32 * CLUSTER * WARPS) {
      const int k = k0 + q * 8;
      const bool in = k < p.K;
      uint4 w[4], lo[4], hi[4];
#pragma unroll
      for (int m = 0; m < 4; ++m) {
        const long long l = offset[m * 16 + g], h = offset[m * 16 + g + 8];
        lo[m] = l >= 0 && in ? __ldg(reinterpret_cast<const uint4*>(x + l + 2ll * k)) : zero;
        hi[m] = h >= 0 && in ? __ldg(reinterpret_cast<const uint4*>(x + h + 2ll * k)) : zero;
      }
#pragma unroll
      for (int j = 0; j < 4; ++j) w[j] = rows[j] && in ? __ldg(reinterpret_cast<const uint4*>(rows[j] + k)) : zero;
#pragma unroll
      for (int m = 0; m < 4; ++m) {
        if (m < tall) {
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            mma(acc[m][j], lo[m].x, hi[m].x, lo[m].y, hi[m].y, w[j].x, w[j].y);
            mma(acc[m][j], lo[m].z, hi[m].z, lo[m].w, hi[m].w, w[j].z, w[j].w);
          }
        }
      }
    }
    if (t0) __syncthreads();  // the sums of the chunk before are read
    float* part = smem + warp * LIST * WIDE_PART;
#pragma unroll
    for (int m = 0; m < 4; ++m)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        *reinterpret_cast<float2*>(part + (m * 16 + g) * WIDE_PART + j * 8 + 2 * q) = make_float2(acc[m][j][0], acc[m][j][1]);
        *reinterpret_cast<float2*>(part + (m * 16 + g + 8) * WIDE_PART + j * 8 + 2 * q) = make_float2(acc[m][j][2], acc[m][j][3]);
      }
    if (t0 == 0) asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");  // all CTAs of the cluster run: their memory may be written
    __syncthreads();
    // eight threads a row take four numbers each; rows 8c .. 8c + 7 go to CTA c
#pragma unroll
    for (int i = 0; i < LIST * 8 / THREADS; ++i) {
      const int row = threadIdx.x / 8 + i * (THREADS / 8), t = threadIdx.x % 8 * 4;
      if (row < count && t0 + t < total) {
        float4 v = *reinterpret_cast<const float4*>(smem + row * WIDE_PART + t);
#pragma unroll
        for (int w = 1; w < WARPS; ++w) {
          const float4 o = *reinterpret_cast<const float4*>(smem + (w * LIST + row) * WIDE_PART + t);
          v.x += o.x, v.y += o.y, v.z += o.z, v.w += o.w;
        }
        st_cluster(sm32(sums + (rank * SHARE + row % SHARE) * total + t0 + t), row / SHARE, v);
      }
    }
  }
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
  const float scale = p.scales[s];
  const int wide = p.sections * p.R;  // numbers of a row of `inner`
  bf16* inner = p.inner + (long long)tile * SPLITS * LIST * wide;
  // a warp a row, two numbers a lane
  const int row = rank * SHARE + warp;
  if (row >= count) return;
  for (int t = 2 * lane; t < total; t += 64) {
    float v0 = 0.f, v1 = 0.f;
#pragma unroll
    for (int c = 0; c < CLUSTER; ++c) {
      const float2 v = *reinterpret_cast<const float2*>(sums + (c * SHARE + warp) * total + t);
      v0 += v.x, v1 += v.y;
    }
    v0 *= scale, v1 *= scale;
#pragma unroll
    for (int i = 0; i < SPLITS; ++i) {
      const __nv_bfloat162 h = __floats2bfloat162_rn(v0, v1);
      *reinterpret_cast<__nv_bfloat162*>(inner + ((long long)i * LIST + row) * wide + t) = h;
      const float2 f = __bfloat1622float2(h);
      v0 = isinf(f.x) ? 0.f : v0 - f.x;
      v1 = isinf(f.y) ? 0.f : v1 - f.y;
    }
  }
}

// ---- many rows, second kernel: 64 rows and 256 columns a CTA, 32 columns a warp
template <typename O, int SPLITS>
__global__ void __launch_bounds__(THREADS, 2) adapter_outer_kernel(const __grid_constant__ AdapterParams p) {
  extern __shared__ __align__(16) bf16 held[];  // the tile's inner numbers: [SPLITS][LIST][stride]
  __shared__ int rows[LIST];
  pdl_launch();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, q = lane & 3;
  const int tile = blockIdx.y;
  pdl_wait();
  const int s = p.tiles[3 * tile], first = p.tiles[3 * tile + 1], count = p.tiles[3 * tile + 2];
  if (count <= 0) return;
  if (threadIdx.x < LIST) rows[threadIdx.x] = threadIdx.x < count ? p.rows[first + threadIdx.x] : -1;
  __syncthreads();
  const int R = s < 0 ? 0 : p.ranks ? min(max(p.ranks[s], 0), p.R) : p.R;
  if (R == 0) {
    copy_rows<O>(p, rows, count, blockIdx.x, gridDim.x);
    return;
  }
  const int R16 = (R + 15) & ~15, total = p.sections * R16, wide = p.sections * p.R;
  int gi = blockIdx.x * WARPS + warp;
  const bool none = gi >= p.groups[MAX_SECTIONS - 1];
  const Section sec = section_of_group(p, gi);
  const int u = gi * 32 + 8 * q;
  const int col = !none && u < sec.width ? column(p, sec, u) : -1;
  const bf16* b = reinterpret_cast<const bf16*>(p.b) + (long long)s * p.N * p.R;
  const bf16* brow[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int ub = gi * 32 + (g >> 1) * 8 + 2 * j + (g & 1);
    brow[j] = !none && ub < sec.width ? b + (long long)column(p, sec, ub) * p.R + 4 * q : nullptr;
  }
  // the rows that are added to and the first of B come while the inner numbers do
  constexpr int PIECES = sizeof(O) / 2;  // 16-byte pieces of eight columns
  constexpr int EARLY = sizeof(O) == 2 ? 4 : 2;  // sixteens of rows whose pieces come early
  uint4 base[4][2][PIECES];
  const auto fetch = [&](int m) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int r = rows[m * 16 + h * 8 + g];
      if (r >= 0 && col >= 0) {
        const uint4* at = reinterpret_cast<const uint4*>(reinterpret_cast<const O*>(p.base) + r * p.base_stride + col);
#pragma unroll
        for (int i = 0; i < PIECES; ++i) base[m][h][i] = at[i];
      }
    }
  };
#pragma unroll
  for (int m = 0; m < EARLY; ++m) fetch(m);
  uint2 w0[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) w0[j] = brow[j] ? __ldg(reinterpret_cast<const uint2*>(brow[j])) : make_uint2(0, 0);
  const int stride = inner_stride(total, 2), tall = (count + 15) / 16;
  {
    const bf16* inner = p.inner + (long long)tile * SPLITS * LIST * wide;
    const int pieces = total / 8;
    for (int r = threadIdx.x / 8; r < SPLITS * LIST; r += THREADS / 8) {
      if (r % LIST >= tall * 16) continue;
      const bool live = r % LIST < count;
      for (int i = threadIdx.x % 8; i < pieces; i += 8)
        *reinterpret_cast<uint4*>(held + r * stride + i * 8) = live ? *reinterpret_cast<const uint4*>(inner + (long long)r * wide + i * 8) : make_uint4(0, 0, 0, 0);
    }
  }
  __syncthreads();
  if (none) return;
  float acc[4][4][4];
#pragma unroll
  for (int m = 0; m < 4; ++m)
#pragma unroll
    for (int j = 0; j < 4; ++j)
#pragma unroll
      for (int i = 0; i < 4; ++i) acc[m][j][i] = 0.f;
  const bf16* mine = held + g * stride + sec.sec * R16 + 4 * q;
  for (int r0 = 0; r0 < R16; r0 += 16) {
    uint2 w[4], next[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      w[j] = w0[j];
      next[j] = r0 + 16 < R16 && brow[j] ? __ldg(reinterpret_cast<const uint2*>(brow[j] + r0 + 16)) : make_uint2(0, 0);
    }
#pragma unroll
    for (int m = 0; m < 4; ++m) {
      if (m < tall) {
#pragma unroll
        for (int i = 0; i < SPLITS; ++i) {
          const bf16* h = mine + (i * LIST + m * 16) * stride + r0;
          const uint2 lo = *reinterpret_cast<const uint2*>(h), hi = *reinterpret_cast<const uint2*>(h + 8 * stride);
#pragma unroll
          for (int j = 0; j < 4; ++j) mma(acc[m][j], lo.x, hi.x, lo.y, hi.y, w[j].x, w[j].y);
        }
      }
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) w0[j] = next[j];
  }
#pragma unroll
  for (int m = EARLY; m < 4; ++m) fetch(m);
  if (col < 0) return;
#pragma unroll
  for (int m = 0; m < 4; ++m)
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int r = rows[m * 16 + h * 8 + g];
      if (r < 0) continue;
      const float v[8] = {acc[m][0][2 * h], acc[m][0][2 * h + 1], acc[m][1][2 * h], acc[m][1][2 * h + 1], acc[m][2][2 * h], acc[m][2][2 * h + 1], acc[m][3][2 * h], acc[m][3][2 * h + 1]};
      add_eight(base[m][h], reinterpret_cast<O*>(p.out) + r * p.out_stride + col, v);
    }
}

template <typename O, int SPLITS>
int run_wide(const AdapterParams& p, int tiles, cudaStream_t st) {
  const int total = p.sections * p.R;
  const size_t one = (size_t)(WARPS * LIST * WIDE_PART + CLUSTER * SHARE * total) * 4, two = (size_t)SPLITS * LIST * inner_stride(total, 2) * 2;
  const auto inner = adapter_inner_kernel<SPLITS>;
  const auto outer = adapter_outer_kernel<O, SPLITS>;
  cudaError_t rc = cudaFuncSetAttribute(inner, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)one);
  if (rc == cudaSuccess) rc = cudaFuncSetAttribute(outer, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)two);
  if (rc != cudaSuccess) return (int)rc;
  const int r = launch(inner, dim3(tiles * CLUSTER), dim3(THREADS), one, st, p);
  if (r) return r;
  return launch(outer, dim3((p.groups[MAX_SECTIONS - 1] + WARPS - 1) / WARPS, tiles), dim3(THREADS), two, st, p);
}

// ---- the rows of a step by adapter: one CTA.  Rows without an adapter come last.
constexpr int SORT = 1024;
__global__ void __launch_bounds__(SORT) adapter_group_kernel(const int* __restrict__ ids, int n, int S, int tile, int max_tiles, int* __restrict__ rows, int* __restrict__ tiles,
                                                             int* __restrict__ err) {
  pdl_launch();
  pdl_wait();
  extern __shared__ int count[];  // [S + 1] rows, then [S + 1] where they begin
  int* from = count + S + 1;
  __shared__ int warp_rows[32], warp_tiles[32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  for (int i = threadIdx.x; i <= S; i += SORT) count[i] = 0;
  __syncthreads();
  const int rounds = (n + SORT - 1) / SORT;
  for (int r = 0; r < rounds; ++r) {
    const int i = r * SORT + threadIdx.x;
    int s = i < n ? valid_id(ids[i], S, err) : -2;
    if (s == -1) s = S;
    const unsigned same = __match_any_sync(0xffffffffu, s);
    if (s >= 0 && lane == __ffs(same) - 1) atomicAdd(&count[s], __popc(same));
  }
  __syncthreads();
  // rows and tiles before each adapter: every thread takes a run of adapters
  const int run = (S + 1 + SORT - 1) / SORT, lo = threadIdx.x * run, hi = min(S + 1, lo + run);
  int rows_here = 0, tiles_here = 0;
  for (int i = lo; i < hi; ++i) {
    rows_here += count[i];
    tiles_here += (count[i] + tile - 1) / tile;
  }
  int rs = rows_here, ts = tiles_here;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int r = __shfl_up_sync(0xffffffffu, rs, o), t = __shfl_up_sync(0xffffffffu, ts, o);
    if (lane >= o) rs += r, ts += t;
  }
  if (lane == 31) warp_rows[warp] = rs, warp_tiles[warp] = ts;
  __syncthreads();
  int r0 = rs - rows_here, t0 = ts - tiles_here, all = 0;
  for (int w = 0; w < SORT / 32; ++w) {
    if (w < warp) r0 += warp_rows[w], t0 += warp_tiles[w];
    all += warp_tiles[w];
  }
  for (int i = lo; i < hi; ++i) {
    from[i] = r0;
    for (int at = 0; at < count[i]; at += tile, ++t0) {
      tiles[3 * t0] = i == S ? -1 : i;
      tiles[3 * t0 + 1] = r0 + at;
      tiles[3 * t0 + 2] = min(tile, count[i] - at);
    }
    r0 += count[i];
  }
  for (int i = all + threadIdx.x; i < max_tiles; i += SORT) tiles[3 * i] = -1, tiles[3 * i + 1] = 0, tiles[3 * i + 2] = 0;
  __syncthreads();
  for (int r = 0; r < rounds; ++r) {
    const int i = r * SORT + threadIdx.x;
    int s = i < n ? valid_id(ids[i], S, nullptr) : -2;
    if (s == -1) s = S;
    const unsigned same = __match_any_sync(0xffffffffu, s);
    const int first = __ffs(same) - 1;
    int at = 0;
    if (s >= 0 && lane == first) at = atomicAdd(&from[s], __popc(same));
    at = __shfl_sync(0xffffffffu, at, first);
    if (s >= 0) rows[at + __popc(same & ((1u << lane) - 1))] = i;
  }
}

template <typename T, typename O, int SPLITS>
int run_tiles(const AdapterParams& p, int tiles, cudaStream_t st) {
  static_assert(3 * TILE * (MOST + 16) * 2 <= WARPS * TILE * PART * 4 && TILE * (MOST + 4) * 4 <= WARPS * TILE * PART * 4, "the numbers between the products take the partial sums' place");
  const int total = min(p.sections * p.R, MOST);
  const size_t smem = (size_t)(WARPS * TILE * PART + CLUSTER * TILE * total) * 4;
  const auto kernel = adapter_tile_kernel<T, O, SPLITS>;
  const cudaError_t rc = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
  if (rc != cudaSuccess) return (int)rc;
  return launch(kernel, dim3(tiles * CLUSTER), dim3(THREADS), smem, st, p);
}

}  // namespace

KVF_API int kvf_adapters_set_pdl(int on) {
  g_pdl_enabled = on;
  return 0;
}

KVF_API int kvf_adapter_group(const int* ids, int n, int S, int tile, int max_tiles, int* rows, int* tiles, int* err, cudaStream_t st) {
  if (n <= 0) return 0;
  const size_t smem = (size_t)2 * (S + 1) * sizeof(int);
  if (smem > 40 * 1024) return (int)cudaErrorInvalidValue;
  return launch(adapter_group_kernel, dim3(1), dim3(SORT), smem, st, ids, n, S, tile, max_tiles, rows, tiles, err);
}

namespace {

template <typename T, int WIDE_SPLITS>
int run(AdapterParams& p, const int* ends, int wide, int max_tiles, int two, cudaStream_t st) {
  if (p.n <= 0) return 0;
  if (p.sections < 1 || p.sections > MAX_SECTIONS || p.R % 16 || p.K % 8 || p.N % 8 || (!p.tiles && p.n > DIRECT)) return (int)cudaErrorInvalidValue;
  for (int i = 0, from = 0; i < MAX_SECTIONS; ++i) {
    const int end = i < p.sections - 1 ? ends[i] : p.N;
    p.begin[i] = p.alternating ? 0 : from;
    p.width[i] = i >= p.sections ? 0 : p.alternating ? p.N / 2 : end - from;
    p.groups[i] = (i ? p.groups[i - 1] : 0) + (p.width[i] + 31) / 32;
    from = end;
  }
  if constexpr (sizeof(T) == 2) {
    if (two && p.tiles && p.inner && max_tiles <= 65535) return wide ? run_wide<float, 3>(p, max_tiles, st) : run_wide<bf16, 2>(p, max_tiles, st);
  }
  const int tiles = p.tiles ? max_tiles * (LIST / TILE) : p.n;
  if (wide) return run_tiles<T, float, WIDE_SPLITS>(p, tiles, st);
  return run_tiles<T, T, sizeof(T) == 2 ? 2 : 1>(p, tiles, st);
}

}  // namespace

#define KVF_ADAPTER_API(SUF, T, WIDE_SPLITS)                                                                                                                              \
  KVF_API int kvf_adapter_add_##SUF(const void* x, long long x_stride, const void* a, const void* b, const float* scales, const int* ranks, const int* ids, int n, int S,  \
                                    int sections, int R, int K, int N, int end0, int end1, int end2, int alternating, const void* base, long long base_stride, void* out,  \
                                    long long out_stride, int wide, const int* rows, const int* tiles, int max_tiles, void* inner, int two, int* err, cudaStream_t st) {   \
    AdapterParams p{x, a, b, scales, ranks, ids, rows, tiles, (bf16*)inner, base, out, err, x_stride, base_stride, out_stride, n, S, sections, R, K, N, {}, {}, {}, alternating}; \
    const int ends[3] = {end0, end1, end2};                                                                                                                               \
    return run<T, WIDE_SPLITS>(p, ends, wide, max_tiles, two, st);                                                                                                             \
  }
KVF_ADAPTER_API(f32, float, 1)
KVF_ADAPTER_API(bf16, bf16, 3)
