// Low-rank adapters of many requests at once, beside a projection that they share: row n of the result is
//   out[n][c] = base[n][c] + sum_r B[s][c][r] * (scale[s] * sum_k A[s][section(c)][r][k] x[n][k]),   s = ids[n],
// and base[n] where s is -1.  A section is one of the matrices that are stacked in the projection (queries, keys, values);
// of gates and ups that alternate in blocks of 8 columns the sections alternate too.
//
// Up to 16 rows of one adapter are a tile and go to a cluster of eight CTAs: their 64 warps share out the columns of x and A, the partial
// sums meet in shared memory (of the CTA, then of every CTA of the cluster, summed in one order), and each CTA adds its eighth of the
// result's columns.  Neither product needs its operands in shared memory: a lane takes 16 bytes of a row at a time, and which of its k
// come first in a tensor-core step is its own affair as long as x and A (or the inner numbers and B) agree.
// bfloat16 goes to the tensor cores (mma.sync m16n8k16: sixteen flops or so a byte of x and of A, so bytes and latency bound it, not the
// products); the numbers between the two products are sums in 32 bits and are multiplied as two bfloat16 numbers (2^-17 of each is lost
// beside a result that is rounded to 2^-8), or as three where the result is float.  float32 stays on the FP32 pipes.
//
// Which rows make a tile: up to 64 rows every cluster finds out for itself (cluster t is row t's, and works if the row is the 1st,
// 17th, ... of its adapter); for more a kernel of one CTA sorts the rows once a step.
#include "common.cuh"

using namespace kvf;

namespace {

constexpr int THREADS = 256;
constexpr int WARPS = THREADS / 32;
constexpr int MAX_SECTIONS = 4;
constexpr int TILE = 16;        // rows of a tile
constexpr int CLUSTER = 8;      // CTAs a tile
constexpr int DIRECT = 64;      // up to so many rows are grouped by every cluster itself
constexpr int CHUNK = 48;       // rows of A a warp multiplies at a time
constexpr int PART = CHUNK + 4; // floats from one row of the partial sums to the next
constexpr int MOST = 256;       // numbers between the products of a row that are in shared memory at a time (whole sections)

struct AdapterParams {
  const void* x;
  const void* a;        // [S][sections][R][K]
  const void* b;        // [S][N][R]
  const float* scales;  // [S]
  const int* ranks;     // [S] or null: all R
  const int* ids;       // [n]
  const int* rows;      // the rows by adapter, and
  const int* tiles;     // (adapter, first of `rows`, count) a tile: null where clusters group for themselves
  const void* base;
  void* out;
  int* err;
  long long x_stride, base_stride, out_stride;
  int n, S, sections, R, K, N;
  int ends[MAX_SECTIONS];  // sections' last columns + 1 (not alternating)
  int alternating;
};

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

// Column of the result that is number u of section `sec`.
__device__ __forceinline__ int column(const AdapterParams& p, int sec, int u) {
  return p.alternating ? (u >> 3) * 16 + sec * 8 + (u & 7) : (sec ? p.ends[sec - 1] : 0) + u;
}
__device__ __forceinline__ int width(const AdapterParams& p, int sec) { return p.alternating ? p.N / 2 : p.ends[sec] - (sec ? p.ends[sec - 1] : 0); }

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
    rows[j] = t < total ? a + ((long long)(t / R16) * p.R + t % R16) * p.K : nullptr;
  }
  const uint4 zero = make_uint4(0, 0, 0, 0);
#pragma unroll 2
  for (int k0 = gw * 32; k0 < p.K; k0 += 32 * CLUSTER * WARPS) {  // (all lanes take every step: K may end inside one)
    const int k = k0 + q * 8;
    const bool in = k < p.K;
    const uint4 lo = x.lo && in ? __ldg(reinterpret_cast<const uint4*>(x.lo + 2ll * k)) : zero;
    const uint4 hi = x.hi && in ? __ldg(reinterpret_cast<const uint4*>(x.hi + 2ll * k)) : zero;
    uint4 w[CHUNK / 8];
#pragma unroll
    for (int j = 0; j < CHUNK / 8; ++j) w[j] = rows[j] && in ? __ldg(reinterpret_cast<const uint4*>(rows[j] + k)) : zero;
#pragma unroll
    for (int j = 0; j < CHUNK / 8; ++j) {
      mma(acc[j], lo.x, hi.x, lo.y, hi.y, w[j].x, w[j].y);
      mma(acc[j], lo.z, hi.z, lo.w, hi.w, w[j].z, w[j].w);
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
    const float* row = a + ((long long)((t0 + c0) / R16) * p.R + (t0 + c0) % R16) * p.K;  // eight rows of one section
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

// acc[row half][column]: eight columns a lane
template <int SPLITS>
__device__ __forceinline__ void second_product(const AdapterParams& p, const bf16* b, const bf16* inner, int total, int sec, int u0, int R16, float (&acc)[2][8]) {
  const int lane = threadIdx.x & 31, g = lane >> 2, q = lane & 3;
  const int stride = inner_stride(total, 2);
  // column 2q + e of the j-th of four tensor-core tiles is column 8q + 2j + e of the 32: a lane's eight results lie side by side
  const bf16* rows[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int u = u0 + (g >> 1) * 8 + 2 * j + (g & 1);
    rows[j] = u < width(p, sec) ? b + (long long)column(p, sec, u) * p.R : nullptr;
  }
  float c[4][4];
#pragma unroll
  for (int j = 0; j < 4; ++j)
#pragma unroll
    for (int i = 0; i < 4; ++i) c[j][i] = 0.f;
  for (int r = 4 * q; r < R16; r += 16) {
    uint2 w[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) w[j] = rows[j] ? __ldg(reinterpret_cast<const uint2*>(rows[j] + r)) : make_uint2(0, 0);
#pragma unroll
    for (int i = 0; i < SPLITS; ++i) {
      const bf16* h = inner + (i * TILE + g) * stride + r;
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

template <int SPLITS>
__device__ __forceinline__ void second_product(const AdapterParams& p, const float* b, const float* inner, int total, int sec, int u0, int R16, float (&acc)[2][8]) {
  const int lane = threadIdx.x & 31, g = lane >> 2, q = lane & 3;
  const int stride = inner_stride(total, 4);
#pragma unroll
  for (int i = 0; i < 8; ++i) acc[0][i] = acc[1][i] = 0.f;
  if (u0 + 8 * q >= width(p, sec)) return;
  const float* rows = b + (long long)column(p, sec, u0 + 8 * q) * p.R;
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

// eight columns of a row: read, added to, written
__device__ __forceinline__ void add_eight(const float* base, float* out, const float (&v)[8]) {
  float4 a = *reinterpret_cast<const float4*>(base), b = *reinterpret_cast<const float4*>(base + 4);
  a.x += v[0], a.y += v[1], a.z += v[2], a.w += v[3];
  b.x += v[4], b.y += v[5], b.z += v[6], b.w += v[7];
  *reinterpret_cast<float4*>(out) = a;
  *reinterpret_cast<float4*>(out + 4) = b;
}
__device__ __forceinline__ void add_eight(const bf16* base, bf16* out, const float (&v)[8]) {
  const uint4 u = *reinterpret_cast<const uint4*>(base);
  float f[8];
  bf16x8_to_float(u, f);
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

// The rows of tile t without a list: row t's adapter's, if row t is the 1st, 17th, ... of them; the count (0: not a tile's first row).
// All warps work it out; the first leaves the rows in `rows`.
__device__ __forceinline__ int own_rows(const AdapterParams& p, int t, int* rows, int& s) {
  const int lane = threadIdx.x & 31;
  int* err = t == 0 && threadIdx.x < 32 ? p.err : nullptr;
  const int a = lane < p.n ? valid_id(p.ids[lane], p.S, err) : -2;
  const int b = lane + 32 < p.n ? valid_id(p.ids[lane + 32], p.S, err) : -2;
  s = __shfl_sync(0xffffffffu, t < 32 ? a : b, t & 31);
  const unsigned ma = __ballot_sync(0xffffffffu, a == s), mb = __ballot_sync(0xffffffffu, b == s);
  const unsigned long long all = ma | ((unsigned long long)mb << 32);
  const int before = __popcll(all & ((1ull << t) - 1));
  if (before % TILE) return 0;
  const int count = min(TILE, __popcll(all) - before);
  if (threadIdx.x < 32) {
    const int ra = __popc(ma & ((1u << lane) - 1)) - before, rb = __popc(ma) + __popc(mb & ((1u << lane) - 1)) - before;
    if (a == s && ra >= 0 && ra < TILE) rows[ra] = lane;
    if (b == s && rb >= 0 && rb < TILE) rows[rb] = lane + 32;
  }
  return count;
}

// T: type of x, A and B; O: of base and out
template <typename T, typename O, int SPLITS>
__global__ void __cluster_dims__(CLUSTER, 1, 1) __launch_bounds__(THREADS) adapter_tile_kernel(const __grid_constant__ AdapterParams p) {
  extern __shared__ __align__(16) float smem[];  // the warps' partial sums, the CTAs' sums, the numbers between the products
  __shared__ int rows[TILE];
  pdl_launch();
  pdl_wait();
  const int tile = blockIdx.x / CLUSTER, rank = blockIdx.x % CLUSTER;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, q = lane & 3;
  int s, count;
  if (p.tiles) {
    s = p.tiles[3 * tile], count = p.tiles[3 * tile + 2];
    if (count > 0 && threadIdx.x < count) rows[threadIdx.x] = p.rows[p.tiles[3 * tile + 1] + threadIdx.x];
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
    const int row_bytes = (c1 - c0) * (int)sizeof(O), lines = (row_bytes + 127) / 128;
    for (int i = threadIdx.x; i < count * lines; i += THREADS)
      prefetch(reinterpret_cast<const char*>(reinterpret_cast<const O*>(p.base) + rows[i / lines] * p.base_stride + c0) + min(i % lines * 128, row_bytes - 1));
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
  const O* base = reinterpret_cast<const O*>(p.base);
  O* out = reinterpret_cast<O*>(p.out);
  for (int sec0 = 0; sec0 < p.sections; sec0 += together) {
    const int sec1 = min(p.sections, sec0 + together), total = (sec1 - sec0) * R16;
    for (int t0 = 0; t0 < total; t0 += CHUNK) {
      first_product(p, a + (long long)sec0 * p.R * p.K, x, t0, total, R16, rank * WARPS + warp, part + warp * TILE * PART);
      // the CTAs of the cluster run, and have read the sums of the sections before: their memory may be written
      if (t0 == 0) asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
      __syncthreads();
      const int wide = min(CHUNK, total - t0) / 4;
      for (int i = threadIdx.x; i < TILE * wide; i += THREADS) {
        const int row = i / wide, t = i % wide * 4;
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
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
    for (int i = threadIdx.x; i < TILE * total; i += THREADS) {
      float v = 0.f;
#pragma unroll
      for (int c = 0; c < CLUSTER; ++c) v += sums[c * TILE * total + i];
      keep_inner<SPLITS>(inner, total, i / total, i % total, v * scale);
    }
    __syncthreads();
    if (sec1 < p.sections) asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");

    // ---- groups of 32 columns of one section, a warp each
    int groups = 0;
    for (int i = sec0; i < sec1; ++i) groups += (width(p, i) + 31) / 32;
    const int mine = (groups + CLUSTER - 1) / CLUSTER;
    for (int i = warp; i < mine; i += WARPS) {
      int gi = rank * mine + i, sec = sec0;
      if (gi >= groups) break;
      while (gi >= (width(p, sec) + 31) / 32) gi -= (width(p, sec++) + 31) / 32;
      float acc[2][8];
      second_product<SPLITS>(p, b, inner + (sec - sec0) * R16, total, sec, gi * 32, R16, acc);
      const int u = gi * 32 + 8 * q;
      if (u < width(p, sec)) {
        const int c = column(p, sec, u);
        if (g < count) add_eight(base + rows[g] * p.base_stride + c, out + rows[g] * p.out_stride + c, acc[0]);
        if (g + 8 < count) add_eight(base + rows[g + 8] * p.base_stride + c, out + rows[g + 8] * p.out_stride + c, acc[1]);
      }
    }
    __syncthreads();
  }
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

#define KVF_ADAPTER_API(SUF, T, WIDE_SPLITS)                                                                                                                             \
  KVF_API int kvf_adapter_add_##SUF(const void* x, long long x_stride, const void* a, const void* b, const float* scales, const int* ranks, const int* ids, int n, int S, \
                                    int sections, int R, int K, int N, int end0, int end1, int end2, int alternating, const void* base, long long base_stride, void* out, \
                                    long long out_stride, int wide, const int* rows, const int* tiles, int max_tiles, int* err, cudaStream_t st) {                        \
    if (n <= 0) return 0;                                                                                                                                                \
    if (sections < 1 || sections > MAX_SECTIONS || R % 16 || K % 8 || N % 8 || (!tiles && n > DIRECT)) return (int)cudaErrorInvalidValue;                                 \
    AdapterParams p{x, a, b, scales, ranks, ids, rows, tiles, base, out, err, x_stride, base_stride, out_stride, n, S, sections, R, K, N, {end0, end1, end2, N}, alternating}; \
    const int count = tiles ? max_tiles : n;                                                                                                                             \
    if (wide) return run_tiles<T, float, WIDE_SPLITS>(p, count, st);                                                                                                     \
    return run_tiles<T, T, 2>(p, count, st);                                                                                                                             \
  }
KVF_ADAPTER_API(bf16, bf16, 3)
KVF_API int kvf_adapter_add_f32(const void* x, long long x_stride, const void* a, const void* b, const float* scales, const int* ranks, const int* ids, int n, int S, int sections,
                                int R, int K, int N, int end0, int end1, int end2, int alternating, const void* base, long long base_stride, void* out, long long out_stride, int,
                                const int* rows, const int* tiles, int max_tiles, int* err, cudaStream_t st) {
  if (n <= 0) return 0;
  if (sections < 1 || sections > MAX_SECTIONS || R % 16 || K % 8 || N % 8 || (!tiles && n > DIRECT)) return (int)cudaErrorInvalidValue;
  AdapterParams p{x, a, b, scales, ranks, ids, rows, tiles, base, out, err, x_stride, base_stride, out_stride, n, S, sections, R, K, N, {end0, end1, end2, N}, alternating};
  return run_tiles<float, float, 1>(p, tiles ? max_tiles : n, st);
}
