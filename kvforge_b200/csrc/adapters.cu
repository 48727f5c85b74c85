// Low-rank adapters of many requests at once, beside a projection that they share: row n of the result is
//   out[n][c] = base[n][c] + sum_r B[s][c][r] * (scale[s] * sum_k A[s][section(c)][r][k] x[n][k]),   s = ids[n],
// and base[n] where s is -1.  A section is one of the matrices that are stacked in the projection (queries, keys, values);
// of gates and ups that alternate in blocks of 8 columns the sections alternate too.
//
// What bounds it is bytes (about a rank's flops a byte of x and of the rows) and, for few rows, latency.  The numbers between the two
// products ("inner" numbers) are sums in 32 bits; bfloat16 multiplies them as two bfloat16 numbers (2^-17 of each is lost beside a result that
// is rounded to 2^-8), or as three where the result is float.  float32 stays on the FP32 pipes, and is bound by latency too (515 rows on three
// adapters, rank 16, 2048 -> 2048: 16.4 us, of which the sort is 4; the pipes are busy 9 % of the time, issue slots 18 %, and a warp waits most for x
// and A, which come straight into registers).  A row's sums come in one order whatever
// else is in the step: partial sums of k meet in shared memory and are added warp by warp and CTA by CTA.
//
// Few rows (and float32), one launch (`adapter_tile_kernel`): 16 rows of one adapter go to a cluster of eight CTAs.  Each warp multiplies blocks of
// 64 columns of k of its own (mma.sync; A comes by TMA, the rows of x by TMA, gathered, four at a time); the CTAs' sums go to all eight through
// their shared memory; then each CTA adds its share of the columns, B and the rows that are added to coming by bulk copies, a piece
// ahead.  Where there are few tiles several clusters make the same inner numbers and share out the columns.
// Many rows, two launches: `adapter_inner_kernel`, 128 rows by a cluster (tcgen05: the adapter's rows of A are the lanes of the accumulator, the
// tile's rows its columns; rows of A past the adapter's are whatever lies there in shared memory, and their lanes are not read), and
// `adapter_outer_tensor_kernel`, 128 rows and a stripe of columns a CTA on tcgen05, or, where that has no room for the inner numbers of a tile,
// `adapter_outer_kernel`, 32 rows and some hundred columns a CTA.
//
// Which rows make a tile: up to 64 rows every cluster finds out for itself; for more a kernel of one CTA sorts the rows once a step.
#include "tcgen05.cuh"

using namespace kvf;

namespace {

constexpr int THREADS = 256;
constexpr int WARPS = THREADS / 32;
constexpr int MAX_SECTIONS = 4;
constexpr int TILE = 16;        // rows of a cluster that makes both products
constexpr int LIST = 128;       // rows of a tile of the list
constexpr int CLUSTER = 8;      // CTAs a tile
constexpr int DIRECT = 64;      // up to so many rows are grouped by every cluster itself
constexpr int CHUNK = 48;       // rows of A a warp multiplies at a time
constexpr int PART = CHUNK + 4; // floats from one row of the partial sums to the next
constexpr int MOST = 128;       // numbers between the products of a row that are in shared memory at a time (whole sections)

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
  int begin[MAX_SECTIONS], width[MAX_SECTIONS];  // of the sections
  int alternating;
  int most;   // inner numbers of a row that shared memory holds at a time (whole sections of rank R)
  int stage;  // bytes of shared memory that columns of B and of the rows take in turn (few rows)
  int shares; // clusters of a tile (few rows)
  int slots;  // blocks of 64 columns of k that it holds (of a warp, where there are few rows; bf16)
  int tmem;   // columns of tensor memory
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
__device__ __forceinline__ void tmem_ld16(uint32_t at, uint32_t (&r)[16]) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]),
                 "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
               : "r"(at)
               : "memory");
}
// (naming the registers keeps the compiler from using them before the wait)
__device__ __forceinline__ void tmem_wait16(uint32_t (&r)[16]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]), "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]),
                 "+r"(r[13]), "+r"(r[14]), "+r"(r[15])
               :
               : "memory");
}
__device__ __forceinline__ void prefetch_map(const void* map) { asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(map)) : "memory"); }

// ---- the first product in float32: partial sums over a warp's share of k for 16 rows and CHUNK rows of A, into part[16][PART]
// k goes in steps of 32, eight a lane; step st belongs to warp st % 64 of the cluster
struct Rows {
  const char* lo;  // the lane's row g, or null
  const char* hi;  // and g + 8
};

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

// ---- the first product in bfloat16
constexpr int BLOCK_K = 64;  // columns of a block: a 128-byte row of the swizzled tiles
constexpr int MAX_SLOTS = WARPS - 1;  // (a slot has a warp of its own that fills it)
constexpr int BARS = 2 * MAX_SLOTS + 1;
constexpr int FEW_SLOTS = 2;  // of a warp
constexpr int SUM_ROW = 20;  // floats from the sums of one row of A to the next's: of 16 rows of x, and room against bank conflicts

struct Maps {
  CUtensorMap x, run, a, whole;  // rows of x, twice, and of all adapters' A, twice, 64 columns a box: one row, 32 rows; sixteen rows, `most`
};

__host__ __device__ constexpr int slot_bytes(int nr, int rows) { return (nr + rows) * BLOCK_K * 2; }

__device__ __forceinline__ void tma_gather4(uint32_t dst, const CUtensorMap* map, int x, int y0, int y1, int y2, int y3, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cluster.global.tile::gather4.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5, %6}], [%7];"
      ::"r"(dst), "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y0), "r"(y1), "r"(y2), "r"(y3), "r"(bar)
      : "memory");
}

// Few rows: a warp fetches blocks of its own, waits for them and multiplies them (a tcgen05 product of 128 x 16 x 16 takes 128 cycles for its
// operand A alone: 4,100 for 512 columns of k, where eight warps of mma.sync take some 300).  Block j of the CTA is warp j % 8's.
struct Few {
  uint32_t ring, bar;  // the warp's slots ([16 rows of x | rows of A] each) and their barriers
  int block;           // blocks so far
};

__device__ __forceinline__ void ldsm_x4(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];\n" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}

// The warp's share of x[16 rows][k] a[total rows][k] into part[16][total + 4] (in its first slot).
__device__ __forceinline__ void first_product(const AdapterParams& p, const Maps& maps, int a0, const int* rows, int total, int R16, int rank, Few& few, float* part) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, q = lane & 3;
  const int every = (p.K + BLOCK_K - 1) / BLOCK_K, all = (every - rank + CLUSTER - 1) / CLUSTER;  // the CTA's blocks
  const int blocks = (all - warp + WARPS - 1) / WARPS;                                           // the warp's (none for some where K is short)
  const uint32_t bytes = slot_bytes(TILE, total);
  const bool whole = R16 == p.R && total == p.most;
  const auto load = [&](int j) {
    const int slot = (few.block + j) % p.slots;
    const uint32_t to = few.ring + slot * slot_bytes(TILE, p.most), bar = few.bar + 8 * slot;
    const int k = (rank + CLUSTER * (warp + WARPS * j)) * BLOCK_K;
    tc::bar_expect_tx(bar, bytes);
    if (whole) tc::tma_load_2d(to + TILE * 128, &maps.whole, k, a0, bar);
    for (int t = whole ? total : 0, sec = 0, in = 0; t < total; t += 16) {
      tc::tma_load_2d(to + (TILE + t) * 128, &maps.a, k, a0 + sec * p.R + in, bar);
      in += 16;
      if (in == R16) in = 0, ++sec;
    }
#pragma unroll
    for (int r = 0; r < TILE; r += 4) tma_gather4(to + r * 128, &maps.x, k, rows[r], rows[r + 1], rows[r + 2], rows[r + 3], bar);
  };
  if (elect_one())
    for (int j = 0; j < min(blocks, p.slots); ++j) load(j);
  __syncwarp();
  float acc[MOST / 8][4];
#pragma unroll
  for (int j = 0; j < MOST / 8; ++j)
#pragma unroll
    for (int i = 0; i < 4; ++i) acc[j][i] = 0.f;
  // lane l names row l % 16 of a 16 x 16 piece, columns 8 (l / 16) on
  const int lr = lane & 15, lc = lane >> 4;
  for (int j = 0; j < blocks; ++j) {
    const int slot = (few.block + j) % p.slots, turn = (few.block + j) / p.slots;
    const uint32_t at = few.ring + slot * slot_bytes(TILE, p.most);
    tc::bar_wait(few.bar + 8 * slot, turn & 1, p.err);
#pragma unroll
    for (int i = 0; i < BLOCK_K / 16; ++i) {
      uint32_t x[4];
      ldsm_x4(x, at + tc::sw128(lr, 2 * i + lc));
#pragma unroll
      for (int t = 0; t < MOST / 16; ++t) {
        if (t * 16 < total) {
          uint32_t w[4];
          ldsm_x4(w, at + tc::sw128(TILE + t * 16 + lr, 2 * i + lc));
          mma(acc[2 * t], x[0], x[1], x[2], x[3], w[0], w[2]);
          mma(acc[2 * t + 1], x[0], x[1], x[2], x[3], w[1], w[3]);
        }
      }
    }
    __syncwarp();
    if (j + p.slots < blocks && elect_one()) load(j + p.slots);
    __syncwarp();
  }
  few.block += max(blocks, 0);
#pragma unroll
  for (int j = 0; j < MOST / 8; ++j) {
    if (j * 8 < total) {
      *reinterpret_cast<float2*>(part + g * (total + 4) + j * 8 + 2 * q) = make_float2(acc[j][0], acc[j][1]);
      *reinterpret_cast<float2*>(part + (g + 8) * (total + 4) + j * 8 + 2 * q) = make_float2(acc[j][2], acc[j][3]);
    }
  }
}

struct Tensor {
  uint32_t ring, bars, tmem;  // blocks ([NR rows of x | rows of A] each); barriers: a slot is filled, its products are done, all are; accumulator
  int block, pass;            // blocks and passes so far: what phase the barriers are in
};



// Many rows: this CTA's share of a[total rows][k] x[128 rows][k], sent to where it is needed: CTA c of the cluster gets the sums of rows
// 16c .. 16c + 15 of x, in `sums[rank][t][SUM_ROW]`.  a0: the first of the sections' rows of A among all adapters'; rows:
// of x, `count`, to the next multiple of four each valid; runs: bit i, rows 32i .. 32i + 31 follow one another in x.  What lies where no rows are fetched
// reaches only the sums of those.  Blocks are the cluster's in turn: block j of the CTA is block
// rank + 8 j of k.  Warp 0 multiplies; a slot is filled by a thread of a warp of its own (a warp takes some 90 cycles for each copy that it starts).
__device__ __forceinline__ void first_product(const AdapterParams& p, const Maps& maps, int a0, const int* rows, unsigned runs, int count, int total, int R16, int rank, Tensor& tn, float* sums) {
  constexpr int NR = LIST;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int every = (p.K + BLOCK_K - 1) / BLOCK_K, blocks = (every - rank + CLUSTER - 1) / CLUSTER;  // (none for some where K is short)
  const uint32_t bytes = slot_bytes(NR, total), filled = tn.bars, done = filled + 8 * MAX_SLOTS, all = done + 8 * MAX_SLOTS;
  const int tiles = (total + 127) / 128;
  const bool whole = R16 == p.R && total == p.most;
  if (warp > 0) {
    // Warp w fills slot w - 1 and no other, one block after another: what it waits for is never more than one phase ahead of the barrier
    // (a parity tells only two neighbouring phases apart).
    // Where all rows follow one another a block is a few copies, and one warp starts them block after block: the first block is there first.
    const bool alone = runs == (1u << LIST / 32) - 1;
    const int fetched = (count + 3) / 4 * 4;
    if (warp <= (alone ? 1 : p.slots) && elect_one()) {
      const int begin = tn.block % p.slots, own = warp - 1;
      for (int j = alone ? 0 : own - begin + (own < begin ? p.slots : 0); j < blocks; j += alone ? 1 : p.slots) {
        const int turn = (tn.block + j) / p.slots, slot = (tn.block + j) % p.slots;
        if (turn) tc::bar_wait(done + 8 * slot, (turn - 1) & 1, p.err);
        const uint32_t to = tn.ring + slot * bytes, bar = filled + 8 * slot;
        tc::bar_expect_tx(bar, bytes - (NR - fetched) * 128);
        const int k = (rank + CLUSTER * j) * BLOCK_K;
        if (whole) tc::tma_load_2d(to + NR * 128, &maps.whole, k, a0, bar);
        for (int t = whole ? total : 0, sec = 0, in = 0; t < total; t += 16) {
          tc::tma_load_2d(to + (NR + t) * 128, &maps.a, k, a0 + sec * p.R + in, bar);
          in += 16;
          if (in == R16) in = 0, ++sec;
        }
#pragma unroll
        for (int i = 0; i < (NR + 31) / 32; ++i) {
          if (runs >> i & 1) {
            tc::tma_load_2d(to + i * 4096, &maps.run, k, rows[32 * i], bar);
          } else {
#pragma unroll
            for (int r = 32 * i; r < min(NR, 32 * i + 32); r += 4)
              if (r < fetched) tma_gather4(to + r * 128, &maps.x, k, rows[r], rows[r + 1], rows[r + 2], rows[r + 3], bar);
          }
        }
      }
    }
  } else {
    int slot = tn.block % p.slots, turn = tn.block / p.slots;
    for (int j = 0; j < blocks; ++j) {
      tc::bar_wait(filled + 8 * slot, turn & 1, p.err);
      asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
      if (elect_one()) {
        const uint32_t at = tn.ring + slot * bytes;
        for (int m = 0; m < tiles; ++m) {
          const uint64_t da = tc::sdesc(at + NR * 128 + m * 128 * 128), db = tc::sdesc(at);
#pragma unroll
          for (int i = 0; i < BLOCK_K / 16; ++i) tc::umma(tn.tmem + m * NR, da + 2 * i, db + 2 * i, tc::idesc(NR, 0), j | i);
        }
        tc::umma_commit(done + 8 * slot);
        if (j + 1 == blocks) tc::umma_commit(all);
      }
      __syncwarp();
      if (++slot == p.slots) slot = 0, ++turn;
    }
  }
  __syncwarp();
  if (blocks > 0) {
    tc::bar_wait(all, tn.pass & 1, p.err);
    tn.block += blocks;
    ++tn.pass;
  }
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
  // the CTAs of the cluster run, and have read the sums of the sections before: their memory may be written
  asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
  // warps w and w + 4 have the same lanes of the accumulator: the first goes to CTAs 0 .. 3, the second to 4 .. 7
  for (int m = 0; m < tiles; ++m) {
    const int t = m * 128 + (warp & 3) * 32;
    if (t >= total) break;
    const uint32_t from = tn.tmem + m * NR + ((uint32_t)((warp & 3) * 32) << 16);
    const uint32_t to = sm32(sums + (rank * total + t + lane) * SUM_ROW);
    uint32_t r[16];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int cta = (warp >> 2) * 4 + i;
      tmem_ld16(from + cta * 16, r);
      tmem_wait16(r);
      if (t + lane < total) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float4 v = blocks > 0 ? make_float4(__uint_as_float(r[4 * e]), __uint_as_float(r[4 * e + 1]), __uint_as_float(r[4 * e + 2]), __uint_as_float(r[4 * e + 3]))
                                      : make_float4(0.f, 0.f, 0.f, 0.f);
          st_cluster(to + 16 * e, cta, v);
        }
      }
    }
  }
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
}

// Barriers and tensor memory of a CTA (by all threads; ends with a barrier); what the CTA's ring begins with lies at a multiple of 1,024 bytes.
__device__ __forceinline__ Tensor make_tensor(const AdapterParams& p, float* ring, unsigned long long* bars, uint32_t* slot) {
  if (threadIdx.x == 0) {
    for (int i = 0; i < BARS; ++i) tc::bar_init(sm32(bars + i), 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (threadIdx.x < 32) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(sm32(slot)), "r"(p.tmem) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
  return Tensor{sm32(ring), sm32(bars), *slot, 0, 0};
}
__device__ __forceinline__ void free_tensor(const AdapterParams& p, const Tensor& tn) {
  if (threadIdx.x < 32) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tn.tmem), "r"(p.tmem) : "memory");
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

// Of a group of columns (32, or 64 where the sections alternate) the 32 of one section: rows of B in shared memory (`b`, the group's first column's,
// `last` what is there after it) and the section's inner numbers make acc[row half][column], eight columns a lane: 8q .. 8q + 7 of the 32.
// Column 2q + e of the j-th of four tensor-core tiles is column 8q + 2j + e of the 32, so that a lane's eight results lie side by side.
__device__ __forceinline__ int in_group(const AdapterParams& p, int sec, int u) { return p.alternating ? (u >> 3) * 16 + sec * 8 + (u & 7) : u; }

template <int SPLITS>
__device__ __forceinline__ void second_product(const AdapterParams& p, const bf16* b, int last, const bf16* inner, int total, int sec, int R16, float (&acc)[2][8]) {
  const int lane = threadIdx.x & 31, g = lane >> 2, q = lane & 3;
  const int stride = inner_stride(total, 2);
  const bf16* rows[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) rows[j] = b + min(in_group(p, sec, (g >> 1) * 8 + 2 * j + (g & 1)), last) * p.R + 4 * q;  // (columns past the last are not written)
  float c[4][4];
#pragma unroll
  for (int j = 0; j < 4; ++j)
#pragma unroll
    for (int i = 0; i < 4; ++i) c[j][i] = 0.f;
  const bf16* mine = inner + g * stride + 4 * q;
  for (int r = 0; r < R16; r += 16) {
    uint2 w[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) w[j] = *reinterpret_cast<const uint2*>(rows[j] + r);
#pragma unroll
    for (int i = 0; i < SPLITS; ++i) {
      const bf16* h = mine + i * TILE * stride + r;
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
__device__ __forceinline__ void second_product(const AdapterParams& p, const float* b, int last, const float* inner, int total, int sec, int R16, float (&acc)[2][8]) {
  const int lane = threadIdx.x & 31, g = lane >> 2, q = lane & 3;
  const int stride = inner_stride(total, 4);
#pragma unroll
  for (int i = 0; i < 8; ++i) acc[0][i] = acc[1][i] = 0.f;
  const int first = in_group(p, sec, 8 * q);
  if (first > last) return;
  const float* rows = b + first * p.R;
  const float* lo = inner + g * stride;
  const float* hi = lo + 8 * stride;
  // (the four column groups of a warp go round the numbers from places of their own: rows of B lie a multiple of all banks apart)
  int r = 4 * q;
  for (int n = 0; n < R16; n += 4) {
    const float4 l = *reinterpret_cast<const float4*>(lo + r), h = *reinterpret_cast<const float4*>(hi + r);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float4 w = *reinterpret_cast<const float4*>(rows + i * p.R + r);
      acc[0][i] = fmaf(w.w, l.w, fmaf(w.z, l.z, fmaf(w.y, l.y, fmaf(w.x, l.x, acc[0][i]))));
      acc[1][i] = fmaf(w.w, h.w, fmaf(w.z, h.z, fmaf(w.y, h.y, fmaf(w.x, h.x, acc[1][i]))));
    }
    r = r + 4 < R16 ? r + 4 : 0;
  }
}

__device__ __forceinline__ void bulk_load(uint32_t dst, const void* src, uint32_t bytes, uint32_t bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst), "l"(src), "r"(bytes), "r"(bar) : "memory");
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
    __syncwarp();
    if (lane >= count && lane < TILE) rows[lane] = rows[0];  // (what comes of them is not read)
  }
  return count;
}

// Measured (replayed launches, inputs from three states in turn): eight rows with adapters of their own, rank 16, 4096 -> 6144 9.3 us for 5.0
// MB; 64 rows on 20 adapters, rank 32, 8192 -> 2048 in float 10.9 us for 15 MB; one row, 4096 -> 28672 8.4 us; 512 rows of one adapter, 4096 ->
// 4096 13 us for 13 MB.  Of the 9.3 us some 1 goes to the ids, 2 to x and A, 2 to the sums and the cluster's barrier, 2 to B and the rows.
// T: type of x, A and B; O: of base and out
template <typename T, typename O, int SPLITS>
__global__ void __cluster_dims__(CLUSTER, 1, 1) __launch_bounds__(THREADS, 2) adapter_tile_kernel(const __grid_constant__ AdapterParams p, const __grid_constant__ Maps maps) {
  // the warps' blocks (bfloat16) or partial sums (float32), whose place columns of B and of the rows take later; the CTAs' sums; the inner numbers
  extern __shared__ __align__(1024) float smem[];
  __shared__ int rows[TILE];
  __shared__ __align__(8) unsigned long long bars[WARPS * FEW_SLOTS], halves[2];
  constexpr bool TENSOR = sizeof(T) == 2;
  pdl_launch();
  if (TENSOR && threadIdx.x == 0) {
    prefetch_map(&maps.x);
    prefetch_map(&maps.whole);
  }
  pdl_wait();
  // a tile (of the list: part of a tile) is `shares` clusters', which all make its inner numbers and share out the columns
  const int rank = blockIdx.x % CLUSTER, tile = blockIdx.x / CLUSTER / p.shares, share = blockIdx.x / CLUSTER % p.shares * CLUSTER + rank;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2;
  int s, count;
  if (p.tiles) {
    const int* entry = p.tiles + tile / (LIST / TILE) * 3;
    const int first = tile % (LIST / TILE) * TILE;
    s = entry[0], count = min(TILE, entry[2] - first);
    if (count > 0 && threadIdx.x < TILE) rows[threadIdx.x] = p.rows[entry[1] + first + min((int)threadIdx.x, count - 1)];  // (rows past the last: what comes of them is not read)
  } else {
    count = own_rows(p, tile, rows, s);
  }
  if (count <= 0) return;  // (the whole cluster)
  const int R = s < 0 ? 0 : p.ranks ? min(max(p.ranks[s], 0), p.R) : p.R;
  if (R == 0) {
    __syncthreads();
    copy_rows<O>(p, rows, count, share, CLUSTER * p.shares);
    return;
  }
  asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");
  const int R16 = (R + 15) & ~15;
  const T* a = reinterpret_cast<const T*>(p.a) + (long long)s * p.sections * p.R * p.K;
  const T* b = reinterpret_cast<const T*>(p.b) + (long long)s * p.N * p.R;
  // whole sections at a time, as many as there is room for
  const int together = min(p.sections, p.most / R16);
  if (threadIdx.x < WARPS * FEW_SLOTS + 2) {
    tc::bar_init(threadIdx.x < 2 ? sm32(halves + threadIdx.x) : sm32(bars + threadIdx.x - 2), threadIdx.x < 2 ? WARPS : 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  __syncthreads();
  float* part = smem;                       // float32: [WARPS][TILE][PART]
  float* sums = reinterpret_cast<float*>(reinterpret_cast<char*>(smem) + p.stage);
  T* inner = reinterpret_cast<T*>(sums + CLUSTER * TILE * p.most);
  const int warp_floats = p.slots * slot_bytes(TILE, p.most) / 4;  // from a warp's slots to the next warp's
  Few few{sm32(smem + warp * warp_floats), sm32(bars + warp * FEW_SLOTS), 0};
  Rows x;
  if constexpr (!TENSOR) {
    const char* from = reinterpret_cast<const char*>(p.x);
    x.lo = g < count ? from + rows[g] * p.x_stride * (long long)sizeof(T) : nullptr;
    x.hi = g + 8 < count ? from + rows[g + 8] * p.x_stride * (long long)sizeof(T) : nullptr;
  }
  const float scale = p.scales[s];
  // groups of 32 columns, in pieces whose columns of B and of the rows take half the stage each
  const int half_bytes = p.stage / 2;
  int pieces = 0;  // so far: what phase the halves' barriers are in
  for (int sec0 = 0; sec0 < p.sections; sec0 += together) {
    const int sec1 = min(p.sections, sec0 + together), total = (sec1 - sec0) * R16;
    for (int t0 = 0; t0 < total; t0 += TENSOR ? MOST : CHUNK) {
      // the warps' partial sums of `wide` numbers, `step` floats from one row to the next
      const int wide = TENSOR ? total : min(CHUNK, total - t0), step = TENSOR ? total + 4 : PART, from = TENSOR ? warp_floats : TILE * PART;
      if constexpr (TENSOR) {
        first_product(p, maps, (s * p.sections + sec0) * p.R, rows, total, R16, rank, few, smem + warp * warp_floats);
      } else {
        first_product(p, a + (long long)sec0 * p.R * p.K, x, t0, total, R16, rank * WARPS + warp, part + warp * TILE * PART);
      }
      // the CTAs of the cluster run, and have read the sums of the sections before: their memory may be written
      if (t0 == 0) asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
      __syncthreads();
      const int row = threadIdx.x / (THREADS / TILE);
      for (int t = threadIdx.x % (THREADS / TILE) * 4; t < wide; t += THREADS / TILE * 4) {
        float4 v = *reinterpret_cast<const float4*>(smem + row * step + t);
#pragma unroll
        for (int w = 1; w < WARPS; ++w) {
          const float4 o = *reinterpret_cast<const float4*>(smem + w * from + row * step + t);
          v.x += o.x, v.y += o.y, v.z += o.z, v.w += o.w;
        }
        const uint32_t to = sm32(sums + (rank * TILE + row) * total + t0 + t);
#pragma unroll
        for (int c = 0; c < CLUSTER; ++c) st_cluster(to, c, v);
      }
      tc::fence_async_smem();  // what was written and read here comes before the copies into the same place: the columns', the next sections'
      __syncthreads();
    }
    asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
    // the sections' columns lie side by side (alternating ones among each other), from `left` to `right`, in groups of `group` columns
    int left = 0, right = p.N;
    if (!p.alternating) {
#pragma unroll
      for (int i = 1; i < MAX_SECTIONS; ++i) {
        if (sec0 == i) left = p.begin[i];
        if (sec1 == i) right = p.begin[i];
      }
    }
    const int group = p.alternating ? 64 : 32, groups = (right - left + group - 1) / group, mine = (groups + CLUSTER * p.shares - 1) / (CLUSTER * p.shares);
    const int begin = share * mine, end = min(groups, begin + mine);
    const int each = max(1, (half_bytes - TILE * 128) / (group * (p.R * (int)sizeof(T) + TILE * (int)sizeof(O))));  // groups of a piece
    const auto row_stride = [&](int columns) { return (columns * (int)sizeof(O) + 63) / 128 * 128 + 64; };  // (two rows in all banks)
    const auto load = [&](int g0, int half) {  // a thread of every warp
      const int c0 = left + g0 * group, columns = min(right, left + min(end, g0 + each) * group) - c0;
      const uint32_t bar = sm32(halves + half), at = sm32(smem) + half * half_bytes;
      const uint32_t b_bytes = columns * p.R * sizeof(T), r_bytes = columns * sizeof(O);
      tc::bar_expect_tx(bar, (warp == 0 ? b_bytes : 0) + (warp < count ? r_bytes : 0) + (warp + WARPS < count ? r_bytes : 0));
      if (warp == 0) bulk_load(at, b + (long long)c0 * p.R, b_bytes, bar);
      for (int r = warp; r < count; r += WARPS)
        bulk_load(at + b_bytes + r * row_stride(columns), reinterpret_cast<const O*>(p.base) + rows[r] * p.base_stride + c0, r_bytes, bar);
    };
    if (begin < end && elect_one()) load(begin, pieces & 1);
    __syncwarp();
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
    for (int row = threadIdx.x / (THREADS / TILE), t = threadIdx.x % (THREADS / TILE); t < total; t += THREADS / TILE) {
      float v = 0.f;
#pragma unroll
      for (int c = 0; c < CLUSTER; ++c) v += sums[(c * TILE + row) * total + t];
      keep_inner<SPLITS>(inner, total, row, t, v * scale);
    }
    __syncthreads();
    if (sec1 < p.sections) asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
    for (int g0 = begin; g0 < end; g0 += each, ++pieces) {
      const int half = pieces & 1;
      // (the other half has been read: a barrier lies behind its piece)
      if (g0 + each < end && elect_one()) load(g0 + each, half ^ 1);
      __syncwarp();
      tc::bar_wait(sm32(halves + half), pieces >> 1 & 1, p.err);
      const int c0 = left + g0 * group, columns = min(right, left + min(end, g0 + each) * group) - c0, stride = row_stride(columns);
      const char* at = reinterpret_cast<const char*>(smem) + half * half_bytes;
      const char* base = at + columns * p.R * sizeof(T);
      // units: a group's columns of one section where they alternate, a group's where they do not
      const int parts = p.alternating ? sec1 - sec0 : 1;
      for (int u = warp; u < parts * (min(end, g0 + each) - g0); u += WARPS) {
        const int from = (u >> (parts - 1)) * group;  // the group's first column, from the piece's
#pragma unroll
        for (int i = 0; i < MAX_SECTIONS; ++i) {
          // (a group may reach over the end of a section: each takes its own columns)
          if (i < sec0 || i >= sec1 || (p.alternating ? i != sec0 + (u & (parts - 1)) : c0 + from >= p.begin[i] + p.width[i] || c0 + from + 32 <= p.begin[i])) continue;
          float acc[2][8];
          second_product<SPLITS>(p, reinterpret_cast<const T*>(at) + from * p.R, columns - 1 - from, inner + (i - sec0) * R16, total, i, R16, acc);
          const int c = from + in_group(p, i, 8 * (lane & 3));
          const bool own = c < columns && (p.alternating || (c0 + c >= p.begin[i] && c0 + c < p.begin[i] + p.width[i]));
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const int r = g + 8 * h;
            if (own && r < count) {
              uint4 old[sizeof(O) / 2];
#pragma unroll
              for (int k = 0; k < (int)sizeof(O) / 2; ++k) old[k] = reinterpret_cast<const uint4*>(base + r * stride + c * sizeof(O))[k];
              add_eight(old, reinterpret_cast<O*>(p.out) + rows[r] * p.out_stride + c0 + c, acc[h]);
            }
          }
          __syncwarp();  // (the next products take the whole warp)
        }
      }
      tc::fence_async_smem();  // what was read here comes before what is copied here next
      __syncthreads();
    }
  }
}

// ---- many rows, first kernel: the inner numbers of 128 rows by a cluster, of which CTA c keeps rows 16c .. 16c + 15.  2,048 rows of 4096 columns and
// 48 rows of A (17 MB) 11 us behind the kernel that sorts them (4 us): the loads take 3, the eight products of a block some 0.3 each behind the
// last of them, the sums and the cluster's barrier 3.
template <int SPLITS>
__global__ void __cluster_dims__(CLUSTER, 1, 1) __launch_bounds__(THREADS) adapter_inner_kernel(const __grid_constant__ AdapterParams p, const __grid_constant__ Maps maps) {
  extern __shared__ __align__(1024) float smem[];  // the ring of blocks, then the sums
  __shared__ int rows[LIST];
  __shared__ unsigned runs_of[LIST / 32];
  __shared__ __align__(8) unsigned long long bars[BARS];
  __shared__ uint32_t tmem_slot;
  if (threadIdx.x == 0) {
    prefetch_map(&maps.run);
    prefetch_map(&maps.whole);
  }
  pdl_wait();
  const int tile = blockIdx.x / CLUSTER, rank = blockIdx.x % CLUSTER;
  const int s = p.tiles[3 * tile], first = p.tiles[3 * tile + 1], count = p.tiles[3 * tile + 2];
  const int R = s < 0 || count <= 0 ? 0 : p.ranks ? min(max(p.ranks[s], 0), p.R) : p.R;
  if (R == 0) return;
  if (threadIdx.x < LIST) {
    const int row = p.rows[first + (threadIdx.x < count ? threadIdx.x : 0)];  // (any row past the last: what comes of it is not read)
    const bool run = __all_sync(0xffffffffu, row == __shfl_sync(0xffffffffu, row, 0) + (int)(threadIdx.x & 31));
    rows[threadIdx.x] = row;
    if ((threadIdx.x & 31) == 0) runs_of[threadIdx.x / 32] = run;
  }
  asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");
  Tensor tn = make_tensor(p, smem, bars, &tmem_slot);  // (a barrier)
  pdl_launch();  // not before it has its tensor memory: a kernel that waits for this one could hold it
  const unsigned runs = runs_of[0] | runs_of[1] << 1 | runs_of[2] << 2 | runs_of[3] << 3;
  static_assert(LIST == 128, "four runs");
  const int R16 = (R + 15) & ~15, together = min(p.sections, p.most / R16);
  float* sums = reinterpret_cast<float*>(reinterpret_cast<char*>(smem) + p.slots * slot_bytes(LIST, p.most));
  const float scale = p.scales[s];
  const int wide = p.sections * p.R;  // numbers of a row of `inner`
  for (int sec0 = 0; sec0 < p.sections; sec0 += together) {
    const int sec1 = min(p.sections, sec0 + together), total = (sec1 - sec0) * R16;
    first_product(p, maps, (s * p.sections + sec0) * p.R, rows, runs, count, total, R16, rank, tn, sums);
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
    // two neighbouring numbers of a row a thread
    bf16* inner = p.inner + ((long long)tile * SPLITS * LIST + rank * TILE) * wide + sec0 * R16;
    const int live = min(TILE, count - rank * TILE);
    for (int i = threadIdx.x; i < TILE * (total / 2); i += THREADS) {
      const int row = i / (total / 2), t = i % (total / 2) * 2;
      if (row >= live) break;
      float v0 = 0.f, v1 = 0.f;
#pragma unroll
      for (int c = 0; c < CLUSTER; ++c) {
        v0 += sums[(c * total + t) * SUM_ROW + row];
        v1 += sums[(c * total + t + 1) * SUM_ROW + row];
      }
      v0 *= scale, v1 *= scale;
#pragma unroll
      for (int k = 0; k < SPLITS; ++k) {
        const __nv_bfloat162 h = __floats2bfloat162_rn(v0, v1);
        *reinterpret_cast<__nv_bfloat162*>(inner + ((long long)k * LIST + row) * wide + t) = h;
        const float2 f = __bfloat1622float2(h);
        v0 = isinf(f.x) ? 0.f : v0 - f.x;
        v1 = isinf(f.y) ? 0.f : v1 - f.y;
      }
    }
    __syncthreads();
    if (sec1 < p.sections) asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
  }
  free_tensor(p, tn);
}

// ---- many rows, second kernel, where the inner numbers of 128 rows have no room in shared memory (two sections and more of rank 128, or of a float
// result): 32 rows and a stripe of columns a CTA, 256 columns at a time.  A warp of its own fetches what the pieces need (the rows by TMA, 32
// that follow one another a box or four gathered; the columns' rows of B are one stretch), several pieces ahead; eight warps multiply, add
// and write 32 columns each.  What is on its way is in shared memory, not in registers.  Bound by its products and by their operands' way from
// shared memory: a call of 1,057 rows on 24 adapters of rank 128, 28672 columns alternating (356 MB with both products' reads) 309 us; of 2,048 rows on
// two, rank 128, 4096 -> 6144 in three sections 172.
constexpr int PIECE = 256;  // columns
constexpr int ROWS = 32;
constexpr int MAX_STAGES = 4;

struct RowMaps {
  CUtensorMap run, row;  // the rows that are added to, 128 bytes a box: 32 rows, one row
};

// KEPT: sixteens of inner numbers that stay in registers from piece to piece
template <typename O, int SPLITS, int KEPT>
__global__ void __launch_bounds__(THREADS + 32, KEPT > 1 ? 1 : 2) adapter_outer_kernel(const __grid_constant__ AdapterParams p, const __grid_constant__ RowMaps maps, int stripe, int stages) {
  extern __shared__ __align__(1024) char ring[];  // a piece: [128 bytes' columns][ROWS][128 bytes], then its rows of B
  __shared__ int rows[ROWS];
  __shared__ unsigned run_of;
  __shared__ __align__(8) unsigned long long filled[MAX_STAGES], empty[MAX_STAGES];
  constexpr int COLUMNS = 128 / (int)sizeof(O);  // of a box
  constexpr int ROW_BYTES = PIECE / COLUMNS * ROWS * 128;
  pdl_launch();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, q = lane & 3, tile = blockIdx.y / (LIST / ROWS), r0 = blockIdx.y % (LIST / ROWS) * ROWS;
  if (threadIdx.x < MAX_STAGES) {
    tc::bar_init(sm32(filled + threadIdx.x), 1);
    tc::bar_init(sm32(empty + threadIdx.x), WARPS);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (threadIdx.x == THREADS) {
    prefetch_map(&maps.run);
    prefetch_map(&maps.row);
  }
  pdl_wait();
  const int s = p.tiles[3 * tile], first = p.tiles[3 * tile + 1] + r0, count = min(ROWS, p.tiles[3 * tile + 2] - r0);
  if (count <= 0) return;
  if (warp == 0) {
    const int row = p.rows[first + min(lane, count - 1)];  // (rows past the last are fetched and not used)
    const bool run = __all_sync(0xffffffffu, row == __shfl_sync(0xffffffffu, row, 0) + lane);
    rows[lane] = row;
    if (lane == 0) run_of = run;
  }
  __syncthreads();
  const int R = s < 0 ? 0 : p.ranks ? min(max(p.ranks[s], 0), p.R) : p.R;
  if (R == 0) {
    if (threadIdx.x < THREADS) copy_rows<O>(p, rows, count, blockIdx.x, gridDim.x);
    return;
  }
  const int R16 = (R + 15) & ~15, wide = p.sections * p.R;
  const bf16* b = reinterpret_cast<const bf16*>(p.b) + (long long)s * p.N * p.R;
  const int left = blockIdx.x * stripe * PIECE, right = min(p.N, left + stripe * PIECE);
  const int stage_bytes = ROW_BYTES + PIECE * p.R * 2;
  if (warp == WARPS) {
    if (elect_one()) {
      int slot = 0, turn = 0;
      const int fetched = run_of ? 32 : (count + 3) / 4 * 4;
      for (int c0 = left; c0 < right; c0 += PIECE) {
        if (turn) tc::bar_wait(sm32(empty + slot), (turn - 1) & 1, p.err);
        const int columns = min(PIECE, right - c0), boxes = (columns + COLUMNS - 1) / COLUMNS;
        const uint32_t bar = sm32(filled + slot), at = sm32(ring) + slot * stage_bytes;
        tc::bar_expect_tx(bar, boxes * fetched * 128 + columns * p.R * 2);
        for (int k = 0; k < boxes; ++k) {
          if (run_of) {
            tc::tma_load_2d(at + k * ROWS * 128, &maps.run, c0 + k * COLUMNS, rows[0], bar);
          } else {
            for (int r = 0; r < count; r += 4) tma_gather4(at + (k * ROWS + r) * 128, &maps.row, c0 + k * COLUMNS, rows[r], rows[r + 1], rows[r + 2], rows[r + 3], bar);
          }
        }
        bulk_load(at + ROW_BYTES, b + (long long)c0 * p.R, columns * p.R * 2, bar);
        if (++slot == stages) slot = 0, ++turn;
      }
    }
    return;
  }
  // What a warp does with a piece is the same for every piece, and is worked out here (worked out anew each time, 346 instructions for 16 x 32
  // numbers, the kernel was bound by them).  Warp w has columns 32w .. 32w + 31, or those of section w % 2 in the 64 from
  // 64 (w / 2) on where they alternate.
  const int from = p.alternating ? 64 * (warp >> 1) : 32 * warp, half = warp & 1;
  const int own = from + in_group(p, half, 8 * q);  // the lane's first column in the piece
  int w_at[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) w_at[j] = from + in_group(p, half, (g >> 1) * 8 + 2 * j + (g & 1));
  const long long split = (long long)LIST * wide;
  const bf16* held = p.inner + ((long long)tile * SPLITS * LIST + r0 + g) * wide + 4 * q;
  O* out[2][2];
  int old_at[2][2];
  bool live[2][2];
#pragma unroll
  for (int k = 0; k < 2; ++k)
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int r = k * 16 + 8 * h + g, byte = own * (int)sizeof(O);
      live[k][h] = r < count;
      out[k][h] = reinterpret_cast<O*>(p.out) + (live[k][h] ? rows[r] : 0) * p.out_stride + own;
      old_at[k][h] = byte / 128 * ROWS * 128 + (int)tc::sw128(r, byte % 128 / 16);
    }
  uint2 kept[2][KEPT][SPLITS][2];  // the first inner numbers of the section `kept_of`
  int kept_of = -1;
  int slot = 0, turn = 0;
  for (int c0 = left; c0 < right; c0 += PIECE) {
    tc::bar_wait(sm32(filled + slot), turn & 1, p.err);
    const char* at = ring + slot * stage_bytes;
    const bf16* bs = reinterpret_cast<const bf16*>(at + ROW_BYTES) + 4 * q;
    const int columns = min(PIECE, right - c0);
#pragma unroll
    for (int i = 0; i < MAX_SECTIONS; ++i) {
      // (32 columns may reach over the end of a section: each takes its own)
      if (i >= p.sections || from >= columns || (p.alternating ? half != i : c0 + from >= p.begin[i] + p.width[i] || c0 + from + 32 <= p.begin[i])) continue;
      if (i != kept_of) {
        kept_of = i;
#pragma unroll
        for (int k = 0; k < 2; ++k)
#pragma unroll
          for (int e = 0; e < KEPT; ++e)
#pragma unroll
            for (int t = 0; t < SPLITS; ++t) {
              const bf16* h = held + (long long)k * 16 * wide + t * split + i * R16 + 16 * e;
              kept[k][e][t][0] = live[k][0] && 16 * e < R16 ? *reinterpret_cast<const uint2*>(h) : make_uint2(0, 0);
              kept[k][e][t][1] = live[k][1] && 16 * e < R16 ? *reinterpret_cast<const uint2*>(h + 8 * wide) : make_uint2(0, 0);
            }
      }
      const bool mine = own < columns && (p.alternating || (c0 + own >= p.begin[i] && c0 + own < p.begin[i] + p.width[i]));
      float acc[2][4][4];
#pragma unroll
      for (int k = 0; k < 2; ++k)
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
          for (int e = 0; e < 4; ++e) acc[k][j][e] = 0.f;
      const auto step = [&](int r, auto inner_numbers) {
        uint2 x[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) x[j] = *reinterpret_cast<const uint2*>(bs + min(w_at[j], columns - 1) * p.R + r);  // (columns past the last are not written)
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          if (k && count <= 16) continue;
#pragma unroll
          for (int t = 0; t < SPLITS; ++t) {
            uint2 lo, hi;
            inner_numbers(k, t, lo, hi);
#pragma unroll
            for (int j = 0; j < 4; ++j) mma(acc[k][j], lo.x, hi.x, lo.y, hi.y, x[j].x, x[j].y);
          }
        }
      };
#pragma unroll
      for (int e = 0; e < KEPT; ++e)
        if (16 * e < R16) step(16 * e, [&](int k, int t, uint2& lo, uint2& hi) { lo = kept[k][e][t][0], hi = kept[k][e][t][1]; });
      for (int r = 16 * KEPT; r < R16; r += 16)
        step(r, [&](int k, int t, uint2& lo, uint2& hi) {
          const bf16* h = held + (long long)k * 16 * wide + t * split + i * R16 + r;
          lo = live[k][0] ? *reinterpret_cast<const uint2*>(h) : make_uint2(0, 0);
          hi = live[k][1] ? *reinterpret_cast<const uint2*>(h + 8 * wide) : make_uint2(0, 0);
        });
#pragma unroll
      for (int k = 0; k < 2; ++k)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          if (mine && live[k][h]) {
            uint4 old[sizeof(O) / 2];
#pragma unroll
            for (int e = 0; e < (int)sizeof(O) / 2; ++e) old[e] = *reinterpret_cast<const uint4*>(at + (old_at[k][h] ^ (16 * e)));  // (the next sixteen bytes of a swizzled row)
            const float v[8] = {acc[k][0][2 * h], acc[k][0][2 * h + 1], acc[k][1][2 * h], acc[k][1][2 * h + 1], acc[k][2][2 * h], acc[k][2][2 * h + 1], acc[k][3][2 * h], acc[k][3][2 * h + 1]};
            add_eight(old, out[k][h] + c0, v);
          }
        }
      __syncwarp();  // (the next products take the whole warp)
    }
    __syncwarp();
    if (lane == 0) tc::bar_arrive(sm32(empty + slot));
    if (++slot == stages) slot = 0, ++turn;
  }
}

// ---- many rows, second kernel on tcgen05: a CTA an SM, each with 128 rows and a stripe of columns, 128 columns at a time.  The tile's inner
// numbers (every section, every 16-bit part) stay in shared memory for a stripe.  Four warps fetch the pieces (one of them B), several ahead; a
// warp multiplies (128 x 128 into one half of tensor memory while the other is read); eight warps add and write: a lane adds 64 columns of one
// row where the rows lie in shared memory, and the warp writes them from there, 128 bytes a row.  What the table of tiles says decides how many
// pieces a stripe has: the host does not know how many adapters there are.
// Replayed calls (sort and both products), and with the kernel above in place of this one: 2,048 rows of one adapter, rank 16, 28672 columns (235
// MB) 62 us, 119; of two, rank 64, 8192 -> 4096 in float 50, 81; 1,057 rows on 24 adapters, rank 64, 28672 columns (238 MB) 123, 171; 700 rows
// on 24, rank 16, 6144 columns 35, 31 (tiles of 30 rows: too few to fill the pieces).  Bound by latency: of the first piece (the table, the
// rows' numbers, their TMA; 4 us), and of a piece's way through three kinds of warps where tiles are many and short.  One warp that fetched, some 90
// cycles for each four rows, took 143 us for the third; products of all columns for both alternating sections 128 for 143.
constexpr int SPAN = 128;  // columns of a piece
constexpr int ADDERS = 8;  // warps that add
constexpr int FETCHERS = LIST / 32;

struct OuterMaps {
  CUtensorMap run, row, inner, b;  // the rows that are added to (128 bytes: 32 rows, one row); the inner numbers (64: 128 rows); B (64: 128 rows)
};

// Pieces do not reach from one section into the next.
__host__ __device__ __forceinline__ int outer_pieces(const AdapterParams& p) {
  if (p.alternating) return (p.N + SPAN - 1) / SPAN;
  int pieces = 0;
  for (int i = 0; i < MAX_SECTIONS; ++i)
    if (i < p.sections) pieces += (p.width[i] + SPAN - 1) / SPAN;
  return pieces;
}

// Pieces of a stripe, of which CTAs take one to four after another (a lane tries each): a stripe begins with the inner numbers, in the time of some
// four pieces.
constexpr int SMS = 148;
__device__ __forceinline__ int pieces_of_stripe(int tiles, int pieces) {
  const int stripes = max(1, ((int)(threadIdx.x & 3) + 1) * SMS / tiles), each = (pieces + stripes - 1) / stripes;
  const int time = (tiles * ((pieces + each - 1) / each) + SMS - 1) / SMS * (each + 4);
  return (int)(__reduce_min_sync(0xffffffffu, (unsigned)min(time, 65535) << 16 | (unsigned)min(each, 65535)) & 65535u);
}

template <typename O, int SPLITS>
__global__ void __launch_bounds__(32 * (ADDERS + FETCHERS + 1), 1) adapter_outer_tensor_kernel(const __grid_constant__ AdapterParams p, const __grid_constant__ OuterMaps maps, int tiles, int stages) {
  extern __shared__ __align__(1024) char pool[];  // the inner numbers [section][part][64 numbers][LIST][128 bytes]; pieces: [128 bytes' columns][LIST][128 bytes], B [64 numbers][SPAN][128 bytes]
  __shared__ __align__(16) int rows[LIST];
  __shared__ unsigned run_of[FETCHERS];
  __shared__ __align__(8) unsigned long long filled[MAX_STAGES], empty[MAX_STAGES], made[2], taken[2], held_bar;
  __shared__ uint32_t tmem_slot;
  constexpr int COLUMNS = 128 / (int)sizeof(O), BOXES = SPAN / COLUMNS, BLOCK = LIST * 128;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  if (threadIdx.x == 0) {
    for (int i = 0; i < MAX_STAGES; ++i) {
      tc::bar_init(sm32(filled + i), FETCHERS);
      tc::bar_init(sm32(empty + i), ADDERS);
    }
    for (int i = 0; i < 2; ++i) {
      tc::bar_init(sm32(made + i), 1);
      tc::bar_init(sm32(taken + i), ADDERS);
    }
    tc::bar_init(sm32(&held_bar), 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    prefetch_map(&maps.run);
    prefetch_map(&maps.inner);
    prefetch_map(&maps.b);
  }
  // (tensor memory before the wait: the kernel before has its own by then, and only then lets this one begin; the one after waits for this one's)
  if (warp == ADDERS) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(sm32(&tmem_slot)), "r"(2u * SPAN) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
  const uint32_t tmem = tmem_slot;
  pdl_launch();
  pdl_wait();
  int with = 0, used = 0;  // tiles that have an adapter, all tiles: the former come first
  int3 mine = make_int3(-1, 0, 0);
  for (int i = 0; i < tiles; i += 32) {
    const int* t = p.tiles + 3 * (i + lane);
    const int3 at = i + lane < tiles ? make_int3(t[0], t[1], t[2]) : make_int3(-1, 0, 0);
    if (i == 0) mine = at;
    with += __popc(__ballot_sync(0xffffffffu, at.z > 0 && at.x >= 0));
    used += __popc(__ballot_sync(0xffffffffu, at.z > 0));
  }
  if (threadIdx.x < THREADS)
    for (int t = with; t < used; ++t) copy_rows<O>(p, p.rows + p.tiles[3 * t + 1], p.tiles[3 * t + 2], blockIdx.x, gridDim.x);
  const int all = outer_pieces(p), stripe = pieces_of_stripe(max(1, with), all), stripes = (all + stripe - 1) / stripe;
  const int held_blocks = (p.R + 63) / 64;
  const int part_bytes = held_blocks * BLOCK, ring = p.sections * SPLITS * part_bytes, b_bytes = held_blocks * SPAN * 128, stage_bytes = BOXES * BLOCK + b_bytes;
  // piece i: its first column, how many it has, its section
  const auto piece = [&](int i, int& c0, int& end, int& sec) {
    sec = 0, c0 = i * SPAN, end = min(SPAN, p.N - c0);
    if (p.alternating) return;
#pragma unroll
    for (int k = 0; k < MAX_SECTIONS; ++k) {
      const int pieces = k < p.sections ? (p.width[k] + SPAN - 1) / SPAN : 0;
      if (i >= 0 && i < pieces) sec = k, c0 = p.begin[k] + i * SPAN, end = min(SPAN, p.width[k] - i * SPAN);
      i -= pieces;
    }
  };
  int c0, end, sec;
  int slot = 0, turn = 0, done = 0, begun = 0;  // the ring, pieces and stripes so far: what phases the barriers are in
  for (int unit = blockIdx.x; unit < with * stripes; unit += gridDim.x) {
    const int tile = unit / stripes, left = unit % stripes * stripe, right = min(all, left + stripe);
    int s = __shfl_sync(0xffffffffu, mine.x, tile & 31), first = __shfl_sync(0xffffffffu, mine.y, tile & 31), count = __shfl_sync(0xffffffffu, mine.z, tile & 31);
    if (tile >= 32) s = p.tiles[3 * tile], first = p.tiles[3 * tile + 1], count = p.tiles[3 * tile + 2];
    if (unit != (int)blockIdx.x) __syncthreads();  // (the stripe before is done with the rows and the inner numbers)
    if (warp < FETCHERS) {
      const int row = p.rows[first + min((int)threadIdx.x, count - 1)];  // (rows past the last are fetched and not used)
      const bool run = __all_sync(0xffffffffu, row == __shfl_sync(0xffffffffu, row, 0) + lane);
      rows[threadIdx.x] = row;
      if (lane == 0) run_of[warp] = run;
    }
    __syncthreads();
    const int R = p.ranks ? min(max(p.ranks[s], 0), p.R) : p.R;
    if (R == 0) {
      if (threadIdx.x < THREADS) copy_rows<O>(p, rows, count, unit % stripes, stripes);
      continue;
    }
    const int R16 = (R + 15) & ~15, blocks = (R16 + 63) / 64;
    if (warp >= ADDERS && warp < ADDERS + FETCHERS) {
      // 32 rows a warp, which takes some 90 cycles for each copy that it starts; the first fetches the inner numbers and B too
      const int part = warp - ADDERS, r0 = 32 * part;
      const bool run = run_of[part], issues = elect_one();
      const int fetched = r0 >= count ? 0 : run ? 32 : (min(32, count - r0) + 3) / 4 * 4;
      if (part == 0 && issues) {
        const uint32_t held = sm32(&held_bar);
        tc::bar_expect_tx(held, p.sections * SPLITS * blocks * BLOCK);
        for (int i = 0; i < p.sections; ++i)
          for (int t = 0; t < SPLITS; ++t)
            for (int k = 0; k < blocks; ++k) tc::tma_load_2d(sm32(pool) + (i * SPLITS + t) * part_bytes + k * BLOCK, &maps.inner, i * R16 + 64 * k, (tile * SPLITS + t) * LIST, held);
      }
      for (int i = left; i < right; ++i) {
        piece(i, c0, end, sec);
        if (issues) {
          if (turn) tc::bar_wait(sm32(empty + slot), (turn - 1) & 1, p.err);
          const uint32_t bar = sm32(filled + slot), at = sm32(pool) + ring + slot * stage_bytes;
          const int boxes = (end + COLUMNS - 1) / COLUMNS;
          tc::bar_expect_tx(bar, boxes * fetched * 128 + (part == 0 ? blocks * SPAN * 128 : 0));
          if (part == 0)
            for (int k = 0; k < blocks; ++k) tc::tma_load_2d(at + BOXES * BLOCK + k * SPAN * 128, &maps.b, 64 * k, s * p.N + c0, bar);
          for (int k = 0; k < boxes && fetched; ++k) {
            const uint32_t to = at + k * BLOCK + r0 * 128;
            if (run) {
              tc::tma_load_2d(to, &maps.run, c0 + k * COLUMNS, rows[r0], bar);
            } else {
              for (int r = 0; r < fetched; r += 4) {
                const int4 four = *reinterpret_cast<const int4*>(rows + r0 + r);
                tma_gather4(to + r * 128, &maps.row, c0 + k * COLUMNS, four.x, four.y, four.z, four.w, bar);
              }
            }
          }
        }
        __syncwarp();
        if (++slot == stages) slot = 0, ++turn;
      }
    } else if (warp == ADDERS + FETCHERS) {
      tc::bar_wait(sm32(&held_bar), begun++ & 1, p.err);
      for (int i = left; i < right; ++i, ++done) {
        piece(i, c0, end, sec);
        tc::bar_wait(sm32(filled + slot), turn & 1, p.err);
        const int half = done & 1;
        if (done >= 2) tc::bar_wait(sm32(taken + half), (done / 2 - 1) & 1, p.err);
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        if (elect_one()) {
          const uint32_t at = sm32(pool) + ring + slot * stage_bytes + BOXES * BLOCK;
          // where two sections alternate, each takes every second eight rows of B (descriptors of 2,048 bytes from eight to eight)
          const int alternating = p.alternating ? 1 : 0;
          for (int h = 0; h <= alternating; ++h) {
            uint32_t accumulate = 0;
            for (int t = 0; t < SPLITS; ++t)
              for (int k = 0; k < R16 / 16; ++k) {
                const uint64_t da = tc::sdesc(sm32(pool) + ((alternating ? h : sec) * SPLITS + t) * part_bytes + k / 4 * BLOCK) + 2 * (k % 4);
                const uint64_t db = tc::sdesc(at + k / 4 * SPAN * 128 + h * 1024) + 2 * (k % 4) + ((uint64_t)(alternating * (1024 >> 4)) << 32);
                tc::umma(tmem + half * SPAN + h * (SPAN / 2), da, db, alternating ? tc::idesc(SPAN / 2, 0) : tc::idesc(SPAN, 0), accumulate);
                accumulate = 1;
              }
          }
          tc::umma_commit(sm32(made + half));
        }
        __syncwarp();
        if (++slot == stages) slot = 0, ++turn;
      }
    } else {
      // warp w: rows 32 (w % 4) on, columns 64 (w / 4) on
      const int quarter = warp & 3, columns0 = (warp >> 2) * 64, r = quarter * 32 + lane;
      for (int i = left; i < right; ++i, ++done) {
        piece(i, c0, end, sec);
        const int half = done & 1;
        tc::bar_wait(sm32(filled + slot), turn & 1, p.err);
        tc::bar_wait(sm32(made + half), done / 2 & 1, p.err);
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        char* at = pool + ring + slot * stage_bytes;
        if (quarter * 32 < count && columns0 < end) {
#pragma unroll
          for (int part = 0; part < 2; ++part) {
            const int c = columns0 + part * 32;
            const uint32_t from = tmem + half * SPAN + ((uint32_t)(quarter * 32) << 16);
            uint32_t v[32];
            if (p.alternating) {
              uint32_t w[2][16];
              tmem_ld16(from + c / 2, w[0]);
              tmem_ld16(from + SPAN / 2 + c / 2, w[1]);
              tmem_wait16(w[0]);
              tmem_wait16(w[1]);
#pragma unroll
              for (int e = 0; e < 32; ++e) v[e] = w[e >> 3 & 1][(e >> 4) * 8 + (e & 7)];
            } else {
              tc::tmem_ld32(from + c, v);
              tc::tmem_wait(v);
            }
#pragma unroll
            for (int e = 0; e < 32; e += 16 / (int)sizeof(O)) {
              const int byte = (c + e) * (int)sizeof(O);
              uint4* old = reinterpret_cast<uint4*>(at + byte / 128 * BLOCK + tc::sw128(r, byte % 128 / 16));
              uint4 o = *old;
              if constexpr (sizeof(O) == 2) {
                float f[8];
                bf16x8_to_float(o, f);
                o.x = tc::pk(f[0] + __uint_as_float(v[e]), f[1] + __uint_as_float(v[e + 1]));
                o.y = tc::pk(f[2] + __uint_as_float(v[e + 2]), f[3] + __uint_as_float(v[e + 3]));
                o.z = tc::pk(f[4] + __uint_as_float(v[e + 4]), f[5] + __uint_as_float(v[e + 5]));
                o.w = tc::pk(f[6] + __uint_as_float(v[e + 6]), f[7] + __uint_as_float(v[e + 7]));
              } else {
                o.x = __float_as_uint(__uint_as_float(o.x) + __uint_as_float(v[e]));
                o.y = __float_as_uint(__uint_as_float(o.y) + __uint_as_float(v[e + 1]));
                o.z = __float_as_uint(__uint_as_float(o.z) + __uint_as_float(v[e + 2]));
                o.w = __float_as_uint(__uint_as_float(o.w) + __uint_as_float(v[e + 3]));
              }
              *old = o;
            }
          }
          __syncwarp();
          // eight lanes a row of 128 bytes
          const int chunk = lane & 7;
#pragma unroll
          for (int k = 0; k < 64 / COLUMNS; ++k) {
            const int box = columns0 / COLUMNS + k, c = box * COLUMNS + chunk * 16 / (int)sizeof(O);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
              const int rr = quarter * 32 + i * 4 + (lane >> 3);
              const uint4 o = *reinterpret_cast<const uint4*>(at + box * BLOCK + tc::sw128(rr, chunk));
              if (rr < count && c < end) *reinterpret_cast<uint4*>(reinterpret_cast<O*>(p.out) + rows[rr] * p.out_stride + c0 + c) = o;
            }
          }
        }
        asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
        tc::fence_async_smem();  // what was written here comes before what is copied here next
        __syncwarp();
        if (lane == 0) {
          tc::bar_arrive(sm32(taken + half));
          tc::bar_arrive(sm32(empty + slot));
        }
        if (++slot == stages) slot = 0, ++turn;
      }
    }
  }
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  if (warp == ADDERS) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(2u * SPAN) : "memory");
}

// Few rows: slots a warp (one where it has one block, or where two keep a second CTA off the SM), the stage, and the bytes for it, the sums and
// the inner numbers.
template <typename T, typename O>
size_t few_smem(AdapterParams& p, int splits) {
  const size_t rest = (size_t)CLUSTER * TILE * p.most * 4 + (sizeof(T) == 2 ? (size_t)splits * TILE * (p.most + 16) * 2 : (size_t)TILE * (p.most + 4) * 4);
  p.slots = 1;
  size_t stage = 64 * 1024;
  if (sizeof(T) == 2) {
    const int blocks = ((p.K + BLOCK_K - 1) / BLOCK_K + CLUSTER - 1) / CLUSTER;
    const size_t slots = (size_t)WARPS * slot_bytes(TILE, p.most);
    if (blocks > WARPS && rest + 2 * slots <= 112 * 1024) p.slots = FEW_SLOTS;
    stage = max(p.slots * slots, min(stage, (size_t)(112 * 1024 - min(rest, (size_t)48 * 1024))));
  }
  // in each half a group at least, and 32 columns for every warp where there is room for them (with one group of 64 columns a piece six warps
  // of eight had nothing to do: 300 float rows of rank 64 and 28672 columns 800 us)
  const size_t column = p.R * sizeof(T) + TILE * sizeof(O);
  stage = max(stage, min(2 * (WARPS * 32 * column + TILE * 128), (size_t)224 * 1024 - rest));
  stage = max(stage, 2 * (64 * column + TILE * 128));
  p.stage = (int)((stage + 2047) / 2048 * 2048);
  return rest + p.stage;
}

// Tensor memory has 512 columns, four CTAs' of the inner kernel.  A fifth on the same SM would wait for some with the CTAs of its cluster
// waiting for it, theirs kept: clusters that have them on different SMs could wait for one another for good.  So each CTA takes at least so much shared
// memory that a fifth has no room.  (Up to 512 columns of k one block is all that a CTA has, and six CTAs of rank 16 found room.)
constexpr int INNER_LEAST = 46 * 1024;
static_assert(512 / LIST == 4 && 5 * (INNER_LEAST + 1024) > 228 * 1024, "a fifth CTA has no room (each has 1 KB besides what it asks for)");

// Many rows: blocks of k that shared memory holds, columns of tensor memory, and the bytes for the ring and the sums (16 KB at least: the last
// lanes of the accumulator read past the rows of A).
size_t many_smem(AdapterParams& p) {
  const size_t sums = (size_t)CLUSTER * p.most * SUM_ROW * 4, rest = max(sums, (size_t)16 * 1024), slot = slot_bytes(LIST, p.most);
  const int blocks = ((p.K + BLOCK_K - 1) / BLOCK_K + CLUSTER - 1) / CLUSTER;
  // Two CTAs an SM where that leaves three blocks each: with one, sixteen clusters of eight did not find room at the same time (a cluster
  // lies within a GPC), and 2,048 rows took two rounds, 18 us for 10.
  const int two = rest < 112 * 1024 ? (int)((112 * 1024 - rest) / slot) : 0, one = (int)((220 * 1024 - rest) / slot);
  p.slots = max(1, min(min(two >= 3 ? two : one, MAX_SLOTS), blocks));
  p.tmem = LIST;
  return max(p.slots * slot + rest, (size_t)INNER_LEAST);
}
static_assert(MOST <= 128 && CLUSTER * MOST * SUM_ROW * 4 + 16 * 1024 + slot_bytes(LIST, MOST) <= 220 * 1024, "one tile of the accumulator; room for a block");
static_assert(CLUSTER * TILE * MOST * 4 + 3 * TILE * (MOST + 16) * 2 + WARPS * slot_bytes(TILE, MOST) <= 226 * 1024, "room for a block a warp");
static_assert(CLUSTER * TILE * MOST * 4 + TILE * (MOST + 4) * 4 + 2 * (64 * (128 * 4 + TILE * 4) + TILE * 128) + 2048 <= 226 * 1024, "... and for a float32 group a half");
static_assert(TILE * (MOST + 4) * 4 <= slot_bytes(TILE, MOST) && TILE * (16 + 4) * 4 <= slot_bytes(TILE, 16), "partial sums take a slot's place");

// x: [n][K], one row a box and 32; A: [S sections R][K], sixteen rows a box and `most`; zeros past K
int make_maps(const AdapterParams& p, Maps& maps) {
  tc::EncodeTiledFn fn = tc::encode_tiled();
  if (!fn) return (int)cudaErrorNotSupported;
  const cuuint32_t ones[2] = {1, 1};
  const auto encode = [&](CUtensorMap* map, const void* at, long long rows, long long stride, int box_rows) {
    const cuuint64_t dims[2] = {(cuuint64_t)p.K, (cuuint64_t)rows}, strides[1] = {(cuuint64_t)stride * 2};
    const cuuint32_t box[2] = {(cuuint32_t)BLOCK_K, (cuuint32_t)box_rows};
    return fn(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, const_cast<void*>(at), dims, strides, box, ones, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
              CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
  };
  return encode(&maps.x, p.x, p.n, p.x_stride, 1) && encode(&maps.run, p.x, p.n, p.x_stride, 32) && encode(&maps.a, p.a, (long long)p.S * p.sections * p.R, p.K, 16) &&
                 encode(&maps.whole, p.a, (long long)p.S * p.sections * p.R, p.K, p.most)
             ? 0 : (int)cudaErrorInvalidValue;
}

// A tensor map of rows of 128 bytes, swizzled.
template <typename E>
bool map_rows(CUtensorMap* map, const void* at, long long columns, long long rows, long long stride, int box_rows) {
  const cuuint64_t dims[2] = {(cuuint64_t)columns, (cuuint64_t)rows}, strides[1] = {(cuuint64_t)stride * sizeof(E)};
  const cuuint32_t box[2] = {(cuuint32_t)(128 / sizeof(E)), (cuuint32_t)box_rows}, ones[2] = {1, 1};
  return tc::encode_tiled()(map, sizeof(E) == 2 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT32, 2, const_cast<void*>(at), dims, strides, box, ones,
                            CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <typename O, int SPLITS>
int run_wide(AdapterParams p, const Maps& maps, int tiles, cudaStream_t st) {
  OuterMaps outer;
  if (!map_rows<O>(&outer.run, p.base, p.N, p.n, p.base_stride, 32) || !map_rows<O>(&outer.row, p.base, p.N, p.n, p.base_stride, 1)) return (int)cudaErrorInvalidValue;
  const size_t one = many_smem(p);
  const auto inner = adapter_inner_kernel<SPLITS>;
  cudaError_t rc = cudaFuncSetAttribute(inner, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)one);
  if (rc != cudaSuccess) return (int)rc;
  const int r = launch(inner, dim3(tiles * CLUSTER), dim3(THREADS), one, st, p, maps);
  if (r) return r;

  // on tcgen05, where the inner numbers of a tile and two pieces have room (and rows of B are counted in 31 bits)
  const size_t parts = (p.R + 63) / 64, held = (size_t)p.sections * SPLITS * parts * LIST * 128, fed = (size_t)SPAN * sizeof(O) * LIST + parts * SPAN * 128;
  if (held + 2 * fed <= 224 * 1024 && (long long)p.S * p.N <= 0x7fffffff - SPAN) {
    const long long wide = (long long)p.sections * p.R;
    if (!map_rows<bf16>(&outer.inner, p.inner, wide, (long long)tiles * SPLITS * LIST, wide, LIST) || !map_rows<bf16>(&outer.b, p.b, p.R, (long long)p.S * p.N, p.R, SPAN))
      return (int)cudaErrorInvalidValue;
    const auto kernel = adapter_outer_tensor_kernel<O, SPLITS>;
    const int stages = min(MAX_STAGES, (int)((224 * 1024 - held) / fed));
    rc = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)(held + stages * fed));
    if (rc != cudaSuccess) return (int)rc;
    return launch(kernel, dim3(SMS), dim3(32 * (ADDERS + FETCHERS + 1)), held + stages * fed, st, p, outer, tiles, stages);
  }

  // Float results of two sections and more: two CTAs an SM where few inner numbers stay in registers (2,048 rows on eight adapters, two sections of 2048
  // columns: rank 16 34 us so and 56 with one CTA and more numbers, rank 32 46 and 64; 28672 columns alternating, rank 32: 227 and 284).
  const bool few_ranks = sizeof(O) == 4 && p.R <= 32;
  const int places = few_ranks ? 2 : 1;
  const size_t stage = (size_t)PIECE * sizeof(O) * ROWS + (size_t)PIECE * p.R * 2;
  const int stages = min(MAX_STAGES, (int)(220 * 1024 / places / stage));  // (of 96 KB at the most: two at least)
  auto kernel = adapter_outer_kernel<O, SPLITS, 4>;
  if constexpr (sizeof(O) == 4) kernel = few_ranks ? adapter_outer_kernel<O, SPLITS, 1> : kernel;
  rc = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)(stages * stage));
  if (rc != cudaSuccess) return (int)rc;
  // pieces of a CTA: as many as leave a CTA for every place there is
  const int pieces = (p.N + PIECE - 1) / PIECE, full = (p.n + ROWS - 1) / ROWS;
  const int stripe = max(1, min(pieces, (int)(((long long)pieces * full + places * SMS - 1) / (places * SMS))));
  return launch(kernel, dim3((pieces + stripe - 1) / stripe, tiles * (LIST / ROWS)), dim3(THREADS + 32), stages * stage, st, p, RowMaps{outer.run, outer.row}, stripe, stages);
}

// ---- the rows of a step by adapter: one CTA.  Rows without an adapter come last.  The rows of an adapter keep their order within a
// warp's 32; whoever places the first row of a tile writes the tile.
constexpr int SORT = 1024;
__global__ void __launch_bounds__(SORT) adapter_group_kernel(const int* __restrict__ ids, int n, int S, int tile, int max_tiles, int* __restrict__ rows, int* __restrict__ tiles,
                                                             int* __restrict__ err) {
  pdl_launch();
  pdl_wait();
  extern __shared__ int count[];  // [S + 1] rows, then [S + 1] where they and [S + 1] where their tiles begin, then [S + 1] how many are placed
  int* from = count + S + 1;
  int* tile0 = from + S + 1;
  int* placed = tile0 + S + 1;
  __shared__ int warp_rows[32], warp_tiles[32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  for (int i = threadIdx.x; i <= S; i += SORT) count[i] = placed[i] = 0;
  const int rounds = (n + SORT - 1) / SORT;
  constexpr int KEPT = 4;  // rounds whose ids stay in registers
  int kept[KEPT];
#pragma unroll
  for (int r = 0; r < KEPT; ++r) kept[r] = r * SORT + (int)threadIdx.x < n ? ids[r * SORT + threadIdx.x] : -2;
  const auto check = [&](int raw, int i) {
    if (i < n && (raw < -1 || raw >= S) && err) atomicOr(err, 32);
    return i >= n ? -2 : raw >= 0 && raw < S ? raw : S;
  };
  __syncthreads();
#pragma unroll
  for (int r = 0; r < KEPT; ++r) kept[r] = check(kept[r], r * SORT + threadIdx.x);
  for (int r = 0; r < rounds; ++r) {
    const int i = r * SORT + threadIdx.x;
    const int s = r == 0 ? kept[0] : r == 1 ? kept[1] : r == 2 ? kept[2] : r == 3 ? kept[3] : check(i < n ? ids[i] : -2, i);
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
  // (the warps' sums, scanned by every warp for itself)
  int wr = warp_rows[lane], wt = warp_tiles[lane];
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int r = __shfl_up_sync(0xffffffffu, wr, o), t = __shfl_up_sync(0xffffffffu, wt, o);
    if (lane >= o) wr += r, wt += t;
  }
  const int all = __shfl_sync(0xffffffffu, wt, 31);
  const int wr0 = __shfl_sync(0xffffffffu, wr, max(warp - 1, 0)), wt0 = __shfl_sync(0xffffffffu, wt, max(warp - 1, 0));
  int r0 = rs - rows_here + (warp ? wr0 : 0), t0 = ts - tiles_here + (warp ? wt0 : 0);
  for (int i = lo; i < hi; ++i) {
    from[i] = r0, tile0[i] = t0;
    r0 += count[i], t0 += (count[i] + tile - 1) / tile;
  }
  for (int i = all + threadIdx.x; i < max_tiles; i += SORT) tiles[3 * i] = -1, tiles[3 * i + 1] = 0, tiles[3 * i + 2] = 0;
  __syncthreads();
  for (int r = 0; r < rounds; ++r) {
    const int i = r * SORT + threadIdx.x;
    const int s = r == 0 ? kept[0] : r == 1 ? kept[1] : r == 2 ? kept[2] : r == 3 ? kept[3] : check(i < n ? ids[i] : -2, i);
    const unsigned same = __match_any_sync(0xffffffffu, s);
    const int leader = __ffs(same) - 1;
    int at = 0;
    if (s >= 0 && lane == leader) at = atomicAdd(&placed[s], __popc(same));
    at = __shfl_sync(0xffffffffu, at, leader) + __popc(same & ((1u << lane) - 1));
    if (s >= 0) {
      rows[from[s] + at] = i;
      if (at % tile == 0) {
        int* t = tiles + 3 * (tile0[s] + at / tile);
        t[0] = s == S ? -1 : s, t[1] = from[s] + at, t[2] = min(tile, count[s] - at);
      }
    }
  }
}

template <typename T, typename O, int SPLITS>
int run_tiles(AdapterParams p, const Maps& maps, int tiles, cudaStream_t st) {
  static_assert(WARPS * TILE * PART * 4 <= 64 * 1024, "the partial sums take the stage's place");
  const size_t smem = few_smem<T, O>(p, SPLITS);
  // A cluster streams all columns of B through eight SMs; where there are few tiles several clusters take shares of the columns (one row and 28672
  // columns: 15 us with one cluster, 9 with sixteen), each of two groups or more.
  const int groups = p.N / (p.alternating ? 64 : 32);
  p.shares = max(1, min((smem > 112 * 1024 ? 1 : 2) * 148 / (tiles * CLUSTER), groups / (2 * CLUSTER)));
  const auto kernel = adapter_tile_kernel<T, O, SPLITS>;
  const cudaError_t rc = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
  if (rc != cudaSuccess) return (int)rc;
  return launch(kernel, dim3(tiles * CLUSTER * p.shares), dim3(THREADS), smem, st, p, maps);
}

}  // namespace

KVF_API int kvf_adapters_set_pdl(int on) {
  g_pdl_enabled = on;
  return 0;
}

// Bytes of shared memory of a CTA that makes the inner numbers of many rows.
KVF_API int kvf_adapter_inner_bytes(int sections, int R, int K) {
  AdapterParams p{};
  p.sections = sections, p.R = R, p.K = K, p.most = min(sections, MOST / R) * R;
  return (int)many_smem(p);
}

KVF_API int kvf_adapter_group(const int* ids, int n, int S, int tile, int max_tiles, int* rows, int* tiles, int* err, cudaStream_t st) {
  if (n <= 0) return 0;
  const size_t smem = (size_t)4 * (S + 1) * sizeof(int);
  if (smem > 96 * 1024) return (int)cudaErrorInvalidValue;
  if (smem > 40 * 1024) {
    const cudaError_t rc = cudaFuncSetAttribute(adapter_group_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
    if (rc != cudaSuccess) return (int)rc;
  }
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
    from = end;
  }
  p.most = min(p.sections, MOST / p.R) * p.R;
  Maps maps;
  if constexpr (sizeof(T) == 2) {
    const int rc = make_maps(p, maps);
    if (rc) return rc;
    if (two && p.tiles && p.inner && max_tiles * (LIST / ROWS) <= 65535) return wide ? run_wide<float, 3>(p, maps, max_tiles, st) : run_wide<bf16, 2>(p, maps, max_tiles, st);
  }
  const int tiles = p.tiles ? max_tiles * (LIST / TILE) : p.n;
  if (wide) return run_tiles<T, float, WIDE_SPLITS>(p, maps, tiles, st);
  return run_tiles<T, T, sizeof(T) == 2 ? 2 : 1>(p, maps, tiles, st);
}

}  // namespace

// A bank as the host keeps it for all calls: A, B, scales, ranks (or null), adapters, sections, R, K, N, the first three sections' ends,
// whether they alternate; 64 bits each.
#define KVF_ADAPTER_API(SUF, T, WIDE_SPLITS)                                                                                                                              \
  KVF_API int kvf_adapter_add_##SUF(const void* x, long long x_stride, const long long* bank, const int* ids, int n, const void* base, long long base_stride, void* out,  \
                                    long long out_stride, int wide, const int* rows, const int* tiles, int max_tiles, void* inner, int two, int* err, cudaStream_t st) {   \
    AdapterParams p{x, (const void*)bank[0], (const void*)bank[1], (const float*)bank[2], (const int*)bank[3], ids, rows, tiles, (bf16*)inner, base, out, err, x_stride,    \
                    base_stride, out_stride, n, (int)bank[4], (int)bank[5], (int)bank[6], (int)bank[7], (int)bank[8], {}, {}, (int)bank[12], 0, 0, 0, 0, 0};               \
    const int ends[3] = {(int)bank[9], (int)bank[10], (int)bank[11]};                                                                                                      \
    return run<T, WIDE_SPLITS>(p, ends, wide, max_tiles, two, st);                                                                                                        \
  }
KVF_ADAPTER_API(f32, float, 1)
KVF_ADAPTER_API(bf16, bf16, 3)
