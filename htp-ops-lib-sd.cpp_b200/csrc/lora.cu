// Low-rank adapters of many requests beside a shared projection:
//
//   out_i = base_i + scale_s (x_i A_s^T) B_s^T,  s = the adapter of row i.
#include <algorithm>
#include <cmath>
#include <exception>

#include "ops.h"
#include "ptx.cuh"

namespace htpg {
namespace {

constexpr int kLoraMaxRank = 128;

struct LoraArgs {
  float *out;
  const float *base, *x;
  const int *ids, *ranks;
  const float *scales;
  const void *a, *b;
  long long ldx, ldb, ldo;
  int m, k, n, adapters, max_rank;
  int wide;  // rows of out are 32-byte aligned
};

constexpr int kLoraThreads = 256, kLoraWarps = 8;

// ---------------------------------------------------------------- rows by adapter
// A tile of TM neighbouring rows, ordered by adapter (stable) and cut into
// blocks of up to BS rows of one adapter, so that requests in any order cost no
// more products than (rows / BS + adapters in the tile) blocks.
template <int TM>
struct RowBlocks {
  int row[TM];                       // row of the tile at each place of the order
  int rank[TM];                      // of its adapter; 0 without one
  float scale[TM];
  int key[TM], ordered[TM], first[TM];
  int start[TM], count[TM], adapter[TM];  // per block; adapter -1: none
  int blocks;
};

constexpr int kNoAdapter = 0x7fffffff;

template <int TM, int BS>
__device__ void find_blocks(RowBlocks<TM> &r, const LoraArgs &p, int row0) {
  const int i = threadIdx.x, rows = min(TM, p.m - row0);
  int key = kNoAdapter, head = p.ids[row0];
  if (head < 0 || head >= p.adapters) head = kNoAdapter;
  if (i < rows) {
    key = p.ids[row0 + i];
    if (key < 0 || key >= p.adapters) key = kNoAdapter;
    r.key[i] = key;
  }
  if (__syncthreads_and(i >= rows || key == head)) {  // one adapter
    if (i < rows) {
      r.row[i] = i;
      const int block = i / BS;
      if (i % BS == 0) {
        r.start[block] = i;
        r.count[block] = min(BS, rows - i);
        r.adapter[block] = key == kNoAdapter ? -1 : key;
      }
    }
    if (i == 0) r.blocks = (rows + BS - 1) / BS;
  } else {
    if (i < rows) {
      int place = 0;
#pragma unroll 8
      for (int j = 0; j < rows; ++j) place += r.key[j] < key || (r.key[j] == key && j < i);
      r.row[place] = i;
      r.ordered[place] = key;
    }
    __syncthreads();
    if (i < rows) {
      int before = 0;
      key = r.ordered[i];
#pragma unroll 8
      for (int j = 0; j < i; ++j) before += r.ordered[j] == key;
      r.first[i] = before % BS == 0;
    }
    __syncthreads();
    if (i < rows && r.first[i]) {
      int block = 0, n = 1;
#pragma unroll 8
      for (int j = 0; j < i; ++j) block += r.first[j];
      while (n < BS && i + n < rows && r.ordered[i + n] == key) ++n;
      r.start[block] = i;
      r.count[block] = n;
      r.adapter[block] = key == kNoAdapter ? -1 : key;
      if (i + n == rows) r.blocks = block + 1;
    }
  }
  if (i < rows) {  // key: that of place i
    r.rank[i] = key == kNoAdapter ? 0 : min(max(p.ranks[key], 0), p.max_rank);
    r.scale[i] = key == kNoAdapter ? 0.0f : p.scales[key];
  }
  __syncthreads();
}

// ---------------------------------------------------------------- x A^T
__device__ __forceinline__ void mma_tf32(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// Shared memory of the down kernel: a ring of steps per warp, a step's 16-byte
// pieces by lane (every lane reads only what it copied: no barrier).
template <int RK>
struct DownSmem {
  static constexpr int kPieces = 4 + RK / 8;  // of two rows of x, of A
  static constexpr int kSteps = RK == 128 ? 2 : 3;
  static constexpr int kRing = kLoraWarps * kSteps * kPieces * 32 * 16;
  static constexpr int kRed = kLoraWarps * (RK / 8) * 32 * 16;
  static constexpr int kBytes = kRing > kRed ? kRing : kRed;
};

// Partial sums over K range blockIdx.y of t = x A^T for a tile's blocks
// blockIdx.z, + gridDim.z, ...: part[range][row][max_rank].  Up to eight blocks
// at once: the warps are shared out evenly, and a block's warps (with more than
// 16 rows: those of each half) take turns at the range's 32-element steps; within
// a step lane t of a quad holds elements 8t .. 8t + 7 of its rows of x and of A
// (any order of k will do, as long as both sides have it).  x = hi + lo, hi with
// the 11 significant bits that TF32 keeps, lo the rest, which TF32 cuts to 11
// more; A is exact in TF32.  The tensor core's own sums round towards zero, so
// they are added up outside of it every step.
// Bound by the chain of a step (16384 x 1536, rank 64, 101 MB: 67 us in tiles of 32
// rows, 57 in tiles of 128, where a CTA's set-up and its warps' sums come less
// often; tensor pipe 57 % busy, issue slots 43 %): x is split and A widened in
// registers.  Both halves of 32 rows in one warp save A's second reading but leave
// 255 registers and less in flight: 76 us.
// One CTA per SM: registers for all of a step's loads (rank 32: 166 instead of 128,
// 12867 x 1152 x 4608 145 -> 131 us in all).
template <typename T, int RK, int TM>
__global__ void __launch_bounds__(kLoraThreads, 1)
    lora_down_kernel(const __grid_constant__ LoraArgs p, float *part, int k_range, int early) {
  using S = DownSmem<RK>;
  constexpr int NT = RK / 8, NS = S::kSteps;
  __shared__ RowBlocks<TM> rb;
  extern __shared__ __align__(16) uint4 smem[];
  grid_dependency_wait();
  if (early) grid_dependents_launch();
  const int row0 = blockIdx.x * TM;
  // 128 rows: a block of 16 rows per warp, and what is left over shared by all
  find_blocks<TM, TM == 128 ? 16 : 32>(rb, p, row0);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int k0 = blockIdx.y * k_range, k1 = min(k0 + k_range, p.k);
  part += static_cast<long long>(blockIdx.y) * p.m * p.max_rank;
  uint4 *ring = smem + warp * (NS * S::kPieces * 32) + lane;
  float4 *red = reinterpret_cast<float4 *>(smem);
  const int z = blockIdx.z, zs = gridDim.z, mine = (rb.blocks - z + zs - 1) / zs;
  auto store = [&](int start, int count, int place, int r, float x, float y) {
    if (place < count && r < p.max_rank)
      *reinterpret_cast<float2 *>(part + static_cast<long long>(row0 + rb.row[start + place]) * p.max_rank + r) = make_float2(x, y);
  };
  for (int done = 0; done < mine;) {
    int group = kLoraWarps;  // warps per block
    while (group > 1 && kLoraWarps / group < mine - done) group >>= 1;
    const int at = done + warp / group, in_group = warp % group, block = z + at * zs;
    const bool live = at < mine;
    const int start = live ? rb.start[block] : 0, count = live ? rb.count[block] : 0, rank = live ? rb.rank[start] : 0;
    const bool halves = count > 16, side = halves && group > 1;  // side: both halves of the rows at once
    const T *a = static_cast<const T *>(p.a) + static_cast<long long>(g) * p.k;
    if (rank) a += static_cast<long long>(rb.adapter[block]) * p.max_rank * p.k;
    float sum[NT][4];
    for (int turn = 0; turn < (halves && !side ? 2 : 1); ++turn) {
      const int half = side ? in_group & 1 : turn, place = half * 16 + g;
#pragma unroll
      for (int j = 0; j < NT; ++j) sum[j][0] = sum[j][1] = sum[j][2] = sum[j][3] = 0.0f;
      if (rank) {
        const float *xa = p.x + (row0 + rb.row[start + min(place, count - 1)]) * p.ldx;
        const float *xb = p.x + (row0 + rb.row[start + min(place + 8, count - 1)]) * p.ldx;
        const int k_first = k0 + (side ? in_group >> 1 : in_group) * 32 + 8 * t, k_step = (side ? group / 2 : group) * 32;
        const long long a_step = 8LL * p.k;
        auto load = [&](int k, int slot) {
          const bool in = k < k1;
          uint4 *to = ring + slot * (S::kPieces * 32);
          copy16(to, xa + (in ? k : 0), in);
          copy16(to + 32, xa + (in ? k + 4 : 0), in);
          copy16(to + 64, xb + (in ? k : 0), in);
          copy16(to + 96, xb + (in ? k + 4 : 0), in);
          const T *from = a + (in ? k : 0);
#pragma unroll
          for (int j = 0; j < NT; ++j, from += a_step) {
            const bool rank_in = in && 8 * j + g < rank;
            copy16(to + (4 + j) * 32, rank_in ? from : static_cast<const T *>(p.a), rank_in);
          }
          copy_commit();
        };
#pragma unroll
        for (int i = 0; i < NS - 1; ++i) load(k_first + i * k_step, i);
        int slot = 0;
        for (int k = k_first; k - 8 * t < k1; k += k_step) {
          load(k + (NS - 1) * k_step, slot == 0 ? NS - 1 : slot - 1);
          copy_wait<NS - 1>();
          const uint4 *from = ring + slot * (S::kPieces * 32);
          slot = slot + 1 == NS ? 0 : slot + 1;
          float c[NT][4];
#pragma unroll
          for (int j = 0; j < NT; ++j) c[j][0] = c[j][1] = c[j][2] = c[j][3] = 0.0f;
#pragma unroll
          for (int h = 0; h < 2; ++h) {  // elements 4h .. 4h + 3 of the lane's eight
            const float4 va = *reinterpret_cast<const float4 *>(from + h * 32);
            const float4 vb = *reinterpret_cast<const float4 *>(from + (2 + h) * 32);
            uint2 w[NT];
#pragma unroll
            for (int j = 0; j < NT; ++j) w[j] = reinterpret_cast<const uint2 *>(from + (4 + j) * 32)[h];
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              // a0, a1: rows g, g + 8 of element 2e; a2, a3: of element 2e + 1
              const float f[4] = {e ? va.z : va.x, e ? vb.z : vb.x, e ? va.w : va.y, e ? vb.w : vb.y};
              uint32_t xh[4], xl[4];
#pragma unroll
              for (int y = 0; y < 4; ++y) {
                xh[y] = __float_as_uint(f[y]) & 0xffffe000u;
                xl[y] = __float_as_uint(f[y] - __uint_as_float(xh[y]));
              }
              float2 b[NT];
#pragma unroll
              for (int j = 0; j < NT; ++j) {
                b[j] = unpack2<T>(e ? w[j].y : w[j].x);
                mma_tf32(c[j], xl, __float_as_uint(b[j].x), __float_as_uint(b[j].y));
              }
#pragma unroll
              for (int j = 0; j < NT; ++j) mma_tf32(c[j], xh, __float_as_uint(b[j].x), __float_as_uint(b[j].y));
            }
          }
#pragma unroll
          for (int j = 0; j < NT; ++j)
#pragma unroll
            for (int y = 0; y < 4; ++y) sum[j][y] += c[j][y];
        }
        copy_wait<0>();
      }
      if (group == 1 && rank) {
#pragma unroll
        for (int j = 0; j < NT; ++j) {
          store(start, count, place, 8 * j + 2 * t, sum[j][0], sum[j][1]);
          store(start, count, place + 8, 8 * j + 2 * t, sum[j][2], sum[j][3]);
        }
      }
    }
    if (group > 1) {
      __syncthreads();  // the rings become the warps' sums, added in order
#pragma unroll
      for (int j = 0; j < NT; ++j)
        red[(warp * NT + j) * 32 + lane] = make_float4(sum[j][0], sum[j][1], sum[j][2], sum[j][3]);
      __syncthreads();
      // the block's own warps add: fragment i of half i / (32 NT)
      for (int i = in_group * 32 + lane; rank && i < (side ? 2 : 1) * NT * 32; i += group * 32) {
        const int h = i / (NT * 32), j = i / 32 % NT;
        float4 o = make_float4(0, 0, 0, 0);
        for (int w = h; w < group; w += side ? 2 : 1) {
          const float4 v = red[((warp - in_group + w) * NT + j) * 32 + lane];
          o.x += v.x, o.y += v.y, o.z += v.z, o.w += v.w;
        }
        store(start, count, h * 16 + g, 8 * j + 2 * t, o.x, o.y);
        store(start, count, h * 16 + g + 8, 8 * j + 2 * t, o.z, o.w);
      }
      __syncthreads();
    }
    done += kLoraWarps / group;
  }
}

// ---------------------------------------------------------------- out = base + t B^T
// Word i of a vector of words (i known when compiling).
__device__ __forceinline__ uint32_t &word(uint4 &v, int i) { return i == 0 ? v.x : i == 1 ? v.y : i == 2 ? v.z : v.w; }
__device__ __forceinline__ uint32_t &word(uint2 &v, int i) { return i == 0 ? v.x : v.y; }
__device__ __forceinline__ uint32_t word(const uint4 &v, int i) { return i == 0 ? v.x : i == 1 ? v.y : i == 2 ? v.z : v.w; }
__device__ __forceinline__ uint32_t word(const uint2 &v, int i) { return i == 0 ? v.x : v.y; }

template <typename T, int RK>
struct UpSmem {
  static constexpr int TM = RK == 128 ? 32 : 64;
  // elements from row to row: the rows of one access phase (2 of 64 bytes, 4 of
  // 32 at rank 16) lie on different banks
  static constexpr int PITCH = RK == 64 ? 96 : RK == 128 ? 160 : RK;
  static constexpr int kVec = RK >= 32 ? 8 : 4;  // ranks a lane holds together
  static constexpr int PARTS = std::is_same<T, __half>::value ? 2 : 3;
  // Blocks of base in flight per warp, less one: more leave less L1 for the rest
  // (16384 x 1536 x 6144, rank 64: two 214 us, three 208, four 217, five 265).
  static constexpr int kDepth = 3;
  // The next item's part of B is read ahead, the first before t (one row, 4096 x
  // 14336: 8.6 -> 8.0 us; 16384 mixed rows of rank 16: 300 -> 283); above rank 32
  // the registers do not reach.
  static constexpr bool kAhead = RK <= 32;
  static constexpr int kBytes = kLoraWarps * kDepth * 4 * 32 * 16;
};

// A tile of rows, its blocks blockIdx.z, + gridDim.z, ..., and the column range
// blockIdx.y, 32 columns per warp at a time.  t (the sum of the K ranges,
// times the adapter's scale) becomes the 16-bit A operand in parts that add up
// to its FP32 value: two for FP16, the row scaled by a power of two to a
// largest element in [2^10, 2^11) (undone at the end), so that what the parts
// leave out is below 2^-22 of an element or 2^-35 of the row's largest; three for BF16.
// Lane t of a quad holds ranks 8t .. 8t + 7 of each 32 (4t .. 4t + 3 of 16), and
// columns 8t .. 8t + 7 of 32 in four MMA tiles, so that B and base move in 16-byte
// pieces and a row's 32 outputs are one 128-byte line of one store.  Each warp keeps
// kDepth blocks (16 rows x 32 columns) of base in flight in a ring of its own, read
// back by the lanes that copied them.
// Many rows: bound by L1 and the chain of an item, then HBM (16384 rows x 6144, rank
// 64: 169 us under ncu for 805 MB, L1 78 % busy; both passes 211 to 216 us alone, 228
// in a sequence of calls on other rows); few rows by the chain ids -> t -> out (one
// row, both passes: 8 us).
template <typename T, int RK>
__global__ void __launch_bounds__(kLoraThreads, 2)
    lora_up_kernel(const __grid_constant__ LoraArgs p, const float *part, int ranges, int n_range) {
  using S = UpSmem<T, RK>;
  constexpr int TM = S::TM, PITCH = S::PITCH, PARTS = S::PARTS, D = S::kDepth;
  __shared__ RowBlocks<TM> rb;
  __shared__ int4 blocks[TM];                     // start, rows, adapter, rank
  __shared__ long long at_base[TM], at_out[TM];  // of the rows, by place
  __shared__ float undo[TM], shared_sums[kLoraWarps][(RK + 31) / 32 * 32];
  extern __shared__ __align__(16) uint4 smem[];
  __shared__ __align__(16) T ts[PARTS][TM][PITCH];
  // what the kernel before the down pass wrote is visible: that pass waited for
  // it before it let this one start
  const int row0 = blockIdx.x * TM;
  find_blocks<TM, 16>(rb, p, row0);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int z = blockIdx.z, zs = gridDim.z;
  const int mine = (rb.blocks - z + zs - 1) / zs;  // blocks of this CTA
  const bool in_place = p.base == p.out && p.ldb == p.ldo;
  if (threadIdx.x < TM && row0 + static_cast<int>(threadIdx.x) < p.m) {
    const long long row = row0 + rb.row[threadIdx.x];
    at_base[threadIdx.x] = row * p.ldb;
    at_out[threadIdx.x] = row * p.ldo;
  }
  if (threadIdx.x < rb.blocks)
    blocks[threadIdx.x] = make_int4(rb.start[threadIdx.x], rb.count[threadIdx.x], rb.adapter[threadIdx.x], rb.rank[rb.start[threadIdx.x]]);
  __syncthreads();
  // work: column groups of 32 (this warp's), each over the CTA's blocks
  const int c_first = blockIdx.y * n_range + warp * 32, c_end = min(static_cast<int>(blockIdx.y + 1) * n_range, p.n);
  const int groups = c_first < c_end ? (c_end - c_first + kLoraWarps * 32 - 1) / (kLoraWarps * 32) : 0;
  const int items = groups * mine;
  uint4 *ring = smem + warp * (D * 4 * 32) + lane;
  int f_item = 0, f_block = 0, f_col = c_first + 8 * t;  // of the next item to fetch
  auto fetch = [&] {
    if (f_item < items && p.base) {
      const int4 block = blocks[z + f_block * zs];
      const bool in = f_col < p.n;
      const float *src = p.base + (in ? f_col : 0);
      uint4 *to = ring + f_item % D * (4 * 32);
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const float *row = src + at_base[block.x + min(g + 8 * i, block.y - 1)];
        const bool ok = in && g + 8 * i < block.y;
        copy16(to + 2 * i * 32, row, ok);
        copy16(to + (2 * i + 1) * 32, row + 4, ok);
      }
      if (++f_block == mine) f_block = 0, f_col += kLoraWarps * 32;
    }
    ++f_item;
    copy_commit();
  };
  constexpr int V = S::kVec, NVEC = RK / (4 * V);  // vectors of V ranks per lane
  using Vec = std::conditional_t<V == 8, uint4, uint2>;
  // B's vectors for the 32 columns of one group, as they lie
  auto take = [&](Vec (&w)[4][NVEC], int block, int group) {
    const int rank = blocks[block].w;
    const T *b = static_cast<const T *>(p.b) + static_cast<long long>(max(blocks[block].z, 0)) * p.n * p.max_rank;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int c = c_first + group * (kLoraWarps * 32) + 8 * (g >> 1) + 2 * j + (g & 1);
      const T *row = b + static_cast<long long>(c) * p.max_rank + V * t;
#pragma unroll
      for (int k = 0; k < NVEC; ++k) {
        w[j][k] = Vec{};
        if (c < p.n && 4 * V * k + V * t < rank) w[j][k] = *reinterpret_cast<const Vec *>(row + 4 * V * k);
      }
    }
  };
  Vec w[4][NVEC], next[4][NVEC];
  if (S::kAhead && items > 0) take(next, z, 0);
  grid_dependency_wait();
#pragma unroll
  for (int i = 0; i < D - 1; ++i) fetch();
  {
    // one warp per place, every eighth, a warp's loads of four ranges in flight together
    constexpr int PLACES = TM / kLoraWarps, NV = (RK + 31) / 32;
    const int rows = min(TM, p.m - row0);
    const long long range_step = static_cast<long long>(p.m) * p.max_rank;
    const float *src = part + static_cast<long long>(row0) * p.max_rank + lane;
    float v[PLACES][NV];
#pragma unroll
    for (int u = 0; u < PLACES; ++u)
#pragma unroll
      for (int j = 0; j < NV; ++j) v[u][j] = 0.0f;
    if (rows <= kLoraWarps / 2) {
      // fewer places than warps: several warps share a place's ranges, and the
      // place's own warp adds their sums in order
      const int share = kLoraWarps / (rows <= 1 ? 1 : rows <= 2 ? 2 : 4), at = warp / share, rank = at < rows ? rb.rank[at] : 0;
      float sum[NV];
#pragma unroll
      for (int j = 0; j < NV; ++j) sum[j] = 0.0f;
#pragma unroll 4
      for (int range = warp % share; range < ranges; range += share)
#pragma unroll
        for (int j = 0; j < NV; ++j)
          if (lane + 32 * j < rank) sum[j] += src[range * range_step + rb.row[at] * p.max_rank + 32 * j];
#pragma unroll
      for (int j = 0; j < NV; ++j) shared_sums[warp][lane + 32 * j] = sum[j];
      __syncthreads();
      if (warp < rows)
        for (int w = warp * share; w < (warp + 1) * share; ++w)
#pragma unroll
          for (int j = 0; j < NV; ++j) v[0][j] += shared_sums[w][lane + 32 * j];
    } else {
      int offset[PLACES], rank[PLACES];
#pragma unroll
      for (int u = 0; u < PLACES; ++u) {
        const int at = warp + kLoraWarps * u;
        rank[u] = at < rows ? rb.rank[at] : 0;
        offset[u] = rank[u] ? rb.row[at] * p.max_rank : 0;
      }
      const int used = (rows + kLoraWarps - 1) / kLoraWarps;  // places of a warp
      if (used <= 2) {
#pragma unroll 8
        for (int range = 0; range < ranges; ++range, src += range_step)
#pragma unroll
          for (int u = 0; u < 2; ++u)
#pragma unroll
            for (int j = 0; j < NV; ++j)
              if (lane + 32 * j < rank[u]) v[u][j] += src[offset[u] + 32 * j];
      } else {
#pragma unroll 2
        for (int range = 0; range < ranges; ++range, src += range_step)
#pragma unroll
          for (int u = 0; u < PLACES; ++u)
#pragma unroll
            for (int j = 0; j < NV; ++j)
              if (lane + 32 * j < rank[u]) v[u][j] += src[offset[u] + 32 * j];
      }
    }
#pragma unroll
    for (int u = 0; u < PLACES; ++u) {
      const int at = warp + kLoraWarps * u;
#pragma unroll
      for (int j = 0; j < NV; ++j) v[u][j] = at < rows && lane + 32 * j < rb.rank[at] ? v[u][j] * rb.scale[at] : 0.0f;
    }
#pragma unroll
    for (int u = 0; u < PLACES; ++u) {
      const int at = warp + kLoraWarps * u;
      float up = 1.0f, down = 1.0f;
      if (PARTS == 2) {
        float most = 0.0f;
#pragma unroll
        for (int j = 0; j < NV; ++j) most = fmaxf(most, fabsf(v[u][j]));
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, o));
        // 2^(10 - e), e the exponent of the largest (subnormals: the nearest that stays finite)
        if (most > 0.0f && most < INFINITY) {
          const int e = max(static_cast<int>(__float_as_uint(most) >> 23) - 127, -110);
          up = __uint_as_float(static_cast<uint32_t>(127 + 10 - e) << 23);
          down = __uint_as_float(static_cast<uint32_t>(127 + e - 10) << 23);
        }
      }
      if (lane == 0) undo[at] = down;
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        const int r = lane + 32 * j;
        if (r >= RK) continue;
        float rest = v[u][j] * up;
#pragma unroll
        for (int q = 0; q < PARTS; ++q) {
          const T h = from_f32<T>(rest);
          ts[q][at][r] = h;
          rest = fabsf(to_f32(h)) < INFINITY ? rest - to_f32(h) : 0.0f;
        }
      }
    }
  }
  __syncthreads();
  int held = -1, held_group = -1, group = 0, at = 0;
  for (int item = 0; item < items; ++item) {
    fetch();
    const int4 block = blocks[z + at * zs];
    const int start = block.x, count = block.y, s = block.z, rank = block.w;
    const int c = c_first + group * (kLoraWarps * 32) + 8 * t;
    if (rank && (s != held || group != held_group)) {
      held = s, held_group = group;
      if (S::kAhead) {
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
          for (int k = 0; k < NVEC; ++k) w[j][k] = next[j][k];
      } else {
        take(w, z + at * zs, group);
      }
      if (rank % V) {  // what lies past the rank may be anything
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
          for (int k = 0; k < NVEC; ++k)
#pragma unroll
            for (int e = 0; e < V / 2; ++e) {
              const int left = rank - (4 * V * k + V * t + 2 * e);
              word(w[j][k], e) &= left >= 2 ? 0xffffffffu : left == 1 ? 0xffffu : 0u;
            }
      }
    }
    if (++at == mine) at = 0, ++group;
    if (S::kAhead && item + 1 < items && (blocks[z + at * zs].z != held || group != held_group))
      take(next, z + at * zs, group);
    copy_wait<D - 1>();
    if (rank == 0 && in_place) continue;
    // base joins after the products: 16 registers fewer next to B (16384 x 1536 x 1536, rank
    // 128: 210 -> 190 us)
    float acc[4][4];
#pragma unroll
    for (int j = 0; j < 4; ++j) acc[j][0] = acc[j][1] = acc[j][2] = acc[j][3] = 0.0f;
    // places past the block's rows: those of other blocks, whose results are not stored
    const int r0 = min(start + g, TM - 1), r1 = min(start + g + 8, TM - 1);
#pragma unroll
    for (int k = 0; k < NVEC; ++k) {
      if (4 * V * k >= rank) break;
#pragma unroll
      for (int q = PARTS - 1; q >= 0; --q) {
        const Vec v0 = *reinterpret_cast<const Vec *>(&ts[q][r0][4 * V * k + V * t]);
        const Vec v1 = *reinterpret_cast<const Vec *>(&ts[q][r1][4 * V * k + V * t]);
#pragma unroll
        for (int e = 0; e < V / 4; ++e) {
          const uint32_t a[4] = {word(v0, 2 * e), word(v1, 2 * e), word(v0, 2 * e + 1), word(v1, 2 * e + 1)};
#pragma unroll
          for (int j = 0; j < 4; ++j) mma_16<T>(acc[j], a, word(w[j][k], 2 * e), word(w[j][k], 2 * e + 1));
        }
      }
    }
    const float down[2] = {undo[r0], undo[r1]};
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      if (g + 8 * i >= count || c >= p.n) continue;
      float4 o[2];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const float *x = acc[2 * h], *y = acc[2 * h + 1];
        o[h] = make_float4(0, 0, 0, 0);
        if (p.base) o[h] = *reinterpret_cast<const float4 *>(ring + (item % D * 4 + 2 * i + h) * 32);
        if (rank) {
          o[h].x = fmaf(x[2 * i], down[i], o[h].x);
          o[h].y = fmaf(x[2 * i + 1], down[i], o[h].y);
          o[h].z = fmaf(y[2 * i], down[i], o[h].z);
          o[h].w = fmaf(y[2 * i + 1], down[i], o[h].w);
        }
      }
      float *out = p.out + at_out[start + g + 8 * i] + c;
      if (p.wide) {
        asm volatile("st.global.cs.v8.f32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(out), "f"(o[0].x),
                     "f"(o[0].y), "f"(o[0].z), "f"(o[0].w), "f"(o[1].x), "f"(o[1].y), "f"(o[1].z), "f"(o[1].w)
                     : "memory");
      } else {
        __stcs(reinterpret_cast<float4 *>(out), o[0]);
        __stcs(reinterpret_cast<float4 *>(out + 4), o[1]);
      }
    }
  }
  copy_wait<0>();
}

template <typename T, int RK>
int launch_lora(const LoraArgs &p, const OpDevice &d, cudaStream_t st) {
  using U = UpSmem<T, RK>;
  using D = DownSmem<RK>;
  // Down: ranges of K until every SM has a tile (multiples of 128, none shorter
  // than a step per warp: 1000 mixed rows 21.5 us in all; multiples of 256 22.5;
  // two CTAs per SM 23.9), then a tile's blocks side by side.  Tiles of 32 or, up
  // to rank 64, 128 rows, whichever takes fewer rounds of (rows x elements + a CTA's
  // set-up, about as long as 32 rows x 1024 elements): 16384 x 1536 x 6144, rank 64:
  // 226 us in all with 32, 216 with 128; mixed, rank 16: 269, 247; 16384 x 1536 x 1536,
  // rank 128: 210, 215.
  struct Plan {
    int tiles, k_range, k_ranges;
    long long cost;
  };
  auto plan = [&](int rows) {
    Plan r;
    r.tiles = (p.m + rows - 1) / rows;
    const int parts = (p.k + 127) / 128, ranges = std::max(1, std::min(parts / 2, d.sms / r.tiles));
    r.k_range = (parts + ranges - 1) / ranges * 128;
    r.k_ranges = (p.k + r.k_range - 1) / r.k_range;
    const long long rounds = (static_cast<long long>(r.tiles) * r.k_ranges + d.sms - 1) / d.sms;
    r.cost = rounds * (rows / 32 * static_cast<long long>(std::min(r.k_range, p.k)) + 1024);
    return r;
  };
  const Plan small = plan(32), large = plan(128);
  const bool wide_tiles = RK <= 64 && large.cost < small.cost;
  const Plan down_plan = wide_tiles ? large : small;
  const int tiles = down_plan.tiles, k_range = down_plan.k_range, k_ranges = down_plan.k_ranges;
  const int z_down = std::max(1, std::min({8, p.adapters, p.m, d.sms / (tiles * k_ranges)}));
  // Up: the column ranges that take least, in sixths of a step of 256 columns: two
  // CTAs of one SM take 5/3 of the time of one, and a CTA's set-up as long as two
  // steps; then blocks of rows side by side.  Against whole rounds of two per SM,
  // 12867 rows of 1152 x 4608, in all: rank 64 173 -> 160 us (BF16) and 156 -> 162 (FP16),
  // rank 16 114 -> 123, rank 32 176 -> 158 (131 as it is now).
  const int up_tiles = (p.m + U::TM - 1) / U::TM, n_steps = (p.n + kLoraWarps * 32 - 1) / (kLoraWarps * 32);
  int n_range = n_steps;
  long long least = -1;
  for (int per = 1; per <= n_steps; ++per) {
    const long long ctas = static_cast<long long>(up_tiles) * ((n_steps + per - 1) / per);
    const long long each = (ctas + d.sms - 1) / d.sms;  // per SM
    const long long cost = (each == 1 ? 6 : 5 * each) * per + 12 * each;
    if (least < 0 || cost <= least) least = cost, n_range = per;
  }
  n_range *= kLoraWarps * 32;
  const int n_ranges = (p.n + n_range - 1) / n_range;
  const int z_up = std::max(1, std::min({8, p.adapters, p.m, 2 * d.sms / (up_tiles * n_ranges)}));
  // The second pass is let in early, to find its blocks meanwhile, for few rows only:
  // with many its CTAs crowd on the SMs that are free then (rank 32, both passes:
  // 1000 rows 16.5 us early, 18.9 late; 4096 x 1536 x 4608 63.6 and 50.3).
  const int early = p.m <= 2048;
  auto lock = op_lock();
  uint32_t *counters;
  uint8_t *scratch;
  const int rc = op_scratch(st, static_cast<size_t>(k_ranges) * p.m * p.max_rank * sizeof(float), &counters, &scratch);
  if (rc) return rc;
  float *part = reinterpret_cast<float *>(scratch);
  auto *down = wide_tiles ? lora_down_kernel<T, RK, RK <= 64 ? 128 : 32> : lora_down_kernel<T, RK, 32>;
  auto *up = lora_up_kernel<T, RK>;
  cudaError_t e = cudaFuncSetAttribute(down, cudaFuncAttributeMaxDynamicSharedMemorySize, D::kBytes);
  if (e == cudaSuccess) e = cudaFuncSetAttribute(up, cudaFuncAttributeMaxDynamicSharedMemorySize, U::kBytes);
  if (e == cudaSuccess) e = op_launch(down, dim3(tiles, k_ranges, z_down), kLoraThreads, D::kBytes, st, p, part, k_range, early);
  if (e == cudaSuccess) e = op_launch(up, dim3(up_tiles, n_ranges, z_up), kLoraThreads, U::kBytes, st, p, part, k_ranges, n_range);
  return op_result(e);
}

template <typename T>
int run_lora(const LoraArgs &p, const OpDevice &d, cudaStream_t st) {
  if (p.max_rank <= 16) return launch_lora<T, 16>(p, d, st);
  if (p.max_rank <= 32) return launch_lora<T, 32>(p, d, st);
  if (p.max_rank <= 64) return launch_lora<T, 64>(p, d, st);
  return launch_lora<T, 128>(p, d, st);
}

}  // namespace
}  // namespace htpg

using namespace htpg;

extern "C" int htpg_lora_run(const struct htpg_lora_params *p, float *out, const float *base, const float *x,
                             const int32_t *row_adapter, const void *a, const void *b, const int32_t *ranks,
                             const float *scales, void *stream) {
  if (!p || (p->type != HTPG_TYPE_F16 && p->type != HTPG_TYPE_BF16) || p->m < 0 || p->k < 1 || p->n < 1 ||
      p->adapters < 1 || p->max_rank < 1 || p->ldx < 0 || p->ldb < 0 || p->ldo < 0)
    return HTPG_EARGS;
  if (p->k % 8 || p->n % 8 || p->max_rank % 8 || p->max_rank > kLoraMaxRank) return HTPG_ECAPACITY;
  if (std::max({p->m, p->k, p->n}) > kOpMaxExtent) return HTPG_ECAPACITY;
  if (p->m == 0) return HTPG_OK;
  if (!out || !x || !row_adapter || !a || !b || !ranks || !scales) return HTPG_EARGS;
  LoraArgs r = {};
  r.ldx = p->ldx ? p->ldx : p->k;
  r.ldb = p->ldb ? p->ldb : p->n;
  r.ldo = p->ldo ? p->ldo : p->n;
  if (p->m > 1 && (r.ldx < p->k || r.ldo < p->n || (base && r.ldb < p->n))) return HTPG_EARGS;
  if (((reinterpret_cast<uintptr_t>(out) | reinterpret_cast<uintptr_t>(base) | reinterpret_cast<uintptr_t>(x) |
        reinterpret_cast<uintptr_t>(a) | reinterpret_cast<uintptr_t>(b)) & 15u) ||
      ((reinterpret_cast<uintptr_t>(row_adapter) | reinterpret_cast<uintptr_t>(ranks) |
        reinterpret_cast<uintptr_t>(scales)) & 3u) ||
      (p->m > 1 && (r.ldx % 4 || r.ldo % 4 || (base && r.ldb % 4))))
    return HTPG_ECONTROL;
  // in place a row's base is where the row goes; elsewhere another CTA may have been
  if (p->m > 1 && base == out && r.ldb != r.ldo) return HTPG_EARGS;
  OpDevice d;
  const int rc = op_device(&d);
  if (rc) return rc;
  r.out = out;
  r.base = base;
  r.x = x;
  r.ids = row_adapter;
  r.ranks = ranks;
  r.scales = scales;
  r.a = a;
  r.b = b;
  r.m = p->m;
  r.k = p->k;
  r.n = p->n;
  r.adapters = p->adapters;
  r.max_rank = p->max_rank;
  r.wide = reinterpret_cast<uintptr_t>(out) % 32 == 0 && (p->m == 1 || r.ldo % 8 == 0);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  try {
    return p->type == HTPG_TYPE_F16 ? run_lora<__half>(r, d, st) : run_lora<__nv_bfloat16>(r, d, st);
  } catch (const std::exception &) {
    return HTPG_ENOMEM;
  }
}
