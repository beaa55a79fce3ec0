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
};

constexpr int kLoraThreads = 256, kLoraWarps = 8;

// ---------------------------------------------------------------- rows by adapter
// A tile of TM neighbouring rows, ordered by adapter (stable) and cut into
// blocks of up to BS rows of one adapter, so that requests in any order cost no
// more products than (rows / BS + adapters in the tile) blocks.
template <int TM>
struct RowBlocks {
  int row[TM];                            // row of the tile at each place of the order
  int key[TM], ordered[TM], first[TM];
  int start[TM], count[TM], adapter[TM];  // per block; adapter -1: none
  int blocks;
};

template <int TM, int BS>
__device__ void find_blocks(RowBlocks<TM> &r, const LoraArgs &p, int row0) {
  const int i = threadIdx.x, rows = min(TM, p.m - row0);
  int key = 0;
  if (i < rows) {
    key = p.ids[row0 + i];
    if (key < 0 || key >= p.adapters) key = 0x7fffffff;
    r.key[i] = key;
  }
  __syncthreads();
  if (i < rows) {
    int place = 0;
    for (int j = 0; j < rows; ++j) place += r.key[j] < key || (r.key[j] == key && j < i);
    r.row[place] = i;
    r.ordered[place] = key;
  }
  __syncthreads();
  int before = 0;
  if (i < rows) {
    key = r.ordered[i];
    for (int j = 0; j < i; ++j) before += r.ordered[j] == key;
    r.first[i] = before % BS == 0;
  }
  __syncthreads();
  if (i < rows && r.first[i]) {
    int block = 0, n = 1;
    for (int j = 0; j < i; ++j) block += r.first[j];
    while (n < BS && i + n < rows && r.ordered[i + n] == key) ++n;
    r.start[block] = i;
    r.count[block] = n;
    r.adapter[block] = key == 0x7fffffff ? -1 : key;
    if (i + n == rows) r.blocks = block + 1;
  }
  __syncthreads();
}

__device__ __forceinline__ int rank_of(const LoraArgs &p, int s) { return min(max(p.ranks[s], 0), p.max_rank); }

// ---------------------------------------------------------------- x A^T
__device__ __forceinline__ void mma_tf32(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// Partial sums over K range blockIdx.y of t = x A^T for a tile's blocks
// blockIdx.z, + gridDim.z, ...: part[range][row][max_rank].  The warps split
// the range by 32-element steps; within a step lane t of a quad holds elements
// 8t .. 8t + 7 of its rows of x and of A (any order of k will do, as long as
// both sides have it), so every load is 16 or 32 contiguous bytes.
// x = hi + lo, hi with the 11 significant bits that TF32 keeps, lo the rest,
// which TF32 cuts to 11 more; A is exact in TF32.  The accumulators are added
// up outside of the tensor core every kRun steps, whose own sums round towards zero.
constexpr int kRun = 8;

template <typename T, int RK, int MB>
__global__ void __launch_bounds__(kLoraThreads) lora_down_kernel(const __grid_constant__ LoraArgs p, float *part,
                                                                 int k_range) {
  constexpr int TM = 32, NT = RK / 8;
  __shared__ RowBlocks<TM> rb;
  __shared__ float4 red[4][NT * MB][32];
  grid_dependency_wait();
  grid_dependents_launch();
  const int row0 = blockIdx.x * TM;
  find_blocks<TM, 16 * MB>(rb, p, row0);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int k0 = blockIdx.y * k_range, k1 = min(k0 + k_range, p.k);
  part += static_cast<long long>(blockIdx.y) * p.m * p.max_rank;
  for (int block = blockIdx.z; block < rb.blocks; block += gridDim.z) {
    const int s = rb.adapter[block];
    if (s < 0) continue;
    const int rank = rank_of(p, s), start = rb.start[block], count = rb.count[block];
    const T *a = static_cast<const T *>(p.a) + static_cast<long long>(s) * p.max_rank * p.k;
    const float *x[2 * MB];
#pragma unroll
    for (int i = 0; i < 2 * MB; ++i)
      x[i] = g + 8 * i < count ? p.x + (row0 + rb.row[start + g + 8 * i]) * p.ldx : nullptr;
    float sum[MB][NT][4];
#pragma unroll
    for (int i = 0; i < MB; ++i)
#pragma unroll
      for (int j = 0; j < NT; ++j) sum[i][j][0] = sum[i][j][1] = sum[i][j][2] = sum[i][j][3] = 0.0f;
    for (int kb = k0 + warp * 32; kb < k1; kb += kLoraWarps * 32) {
      const int k = kb + 8 * t;
      const bool in = k < k1;
      float v[2 * MB][8];
#pragma unroll
      for (int i = 0; i < 2 * MB; ++i) {
        float4 lo = make_float4(0, 0, 0, 0), hi = lo;
        if (in && x[i]) {
          lo = *reinterpret_cast<const float4 *>(x[i] + k);
          hi = *reinterpret_cast<const float4 *>(x[i] + k + 4);
        }
        v[i][0] = lo.x, v[i][1] = lo.y, v[i][2] = lo.z, v[i][3] = lo.w;
        v[i][4] = hi.x, v[i][5] = hi.y, v[i][6] = hi.z, v[i][7] = hi.w;
      }
      uint4 w[NT];
#pragma unroll
      for (int j = 0; j < NT; ++j) {
        w[j] = make_uint4(0, 0, 0, 0);
        if (in && 8 * j + g < rank) w[j] = *reinterpret_cast<const uint4 *>(a + static_cast<long long>(8 * j + g) * p.k + k);
      }
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        uint32_t xh[MB][4], xl[MB][4];
#pragma unroll
        for (int i = 0; i < MB; ++i)
#pragma unroll
          for (int y = 0; y < 4; ++y) {
            // a0, a1: rows g, g + 8 of element 2e; a2, a3: of element 2e + 1
            const float f = v[2 * i + (y & 1)][2 * e + (y >> 1)];
            xh[i][y] = __float_as_uint(f) & 0xffffe000u;
            xl[i][y] = __float_as_uint(f - __uint_as_float(xh[i][y]));
          }
#pragma unroll
        for (int j = 0; j < NT; ++j) {
          const float2 b = unpack2<T>(e == 0 ? w[j].x : e == 1 ? w[j].y : e == 2 ? w[j].z : w[j].w);
          const uint32_t b0 = __float_as_uint(b.x), b1 = __float_as_uint(b.y);
#pragma unroll
          for (int i = 0; i < MB; ++i) {
            mma_tf32(sum[i][j], xl[i], b0, b1);
            mma_tf32(sum[i][j], xh[i], b0, b1);
          }
        }
      }
    }
    // the warps' sums, in a fixed tree
#pragma unroll
    for (int half = kLoraWarps / 2; half > 0; half /= 2) {
      __syncthreads();
      if (warp >= half && warp < 2 * half) {
#pragma unroll
        for (int i = 0; i < MB; ++i)
#pragma unroll
          for (int j = 0; j < NT; ++j)
            red[warp - half][i * NT + j][lane] = make_float4(sum[i][j][0], sum[i][j][1], sum[i][j][2], sum[i][j][3]);
      }
      __syncthreads();
      if (warp < half) {
#pragma unroll
        for (int i = 0; i < MB; ++i)
#pragma unroll
          for (int j = 0; j < NT; ++j) {
            const float4 o = red[warp][i * NT + j][lane];
            sum[i][j][0] += o.x, sum[i][j][1] += o.y, sum[i][j][2] += o.z, sum[i][j][3] += o.w;
          }
      }
    }
    if (warp == 0) {
#pragma unroll
      for (int i = 0; i < 2 * MB; ++i) {
        if (g + 8 * i >= count) continue;
        float *out = part + static_cast<long long>(row0 + rb.row[start + g + 8 * i]) * p.max_rank;
#pragma unroll
        for (int j = 0; j < NT; ++j)
          if (8 * j + 2 * t < p.max_rank)
            *reinterpret_cast<float2 *>(out + 8 * j + 2 * t) =
                make_float2(sum[i / 2][j][i % 2 * 2], sum[i / 2][j][i % 2 * 2 + 1]);
      }
    }
  }
}

// ---------------------------------------------------------------- out = base + t B^T
template <typename T>
__device__ __forceinline__ void mma_16(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if constexpr (std::is_same<T, __half>::value)
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// A tile of rows x 256 columns, 32 columns per warp.  t (the sum of the ranges,
// times the adapter's scale) becomes the 16-bit A operand in parts that add up
// to its FP32 value: two for FP16, the row scaled by a power of two to a
// largest element in [2^10, 2^11) (undone at the end), so that what the parts
// leave out is below 2^-22 of an element or 2^-35 of the row's largest; three for BF16.
// Lane t of a quad holds ranks 4t .. 4t + 3 of each 16, and columns 4t .. 4t + 3
// of each 16 in two MMA tiles, so that B, base and out move in 8- and 16-byte pieces.
template <typename T, int RK>
__global__ void __launch_bounds__(kLoraThreads) lora_up_kernel(const __grid_constant__ LoraArgs p, const float *part,
                                                               int ranges) {
  constexpr int TM = RK == 128 ? 32 : 64, KS = RK / 16, PITCH = RK + 8;
  constexpr int PARTS = std::is_same<T, __half>::value ? 2 : 3;
  __shared__ RowBlocks<TM> rb;
  __shared__ __align__(16) T ts[PARTS][TM][PITCH];  // by place in the order
  __shared__ float undo[TM];
  // what the kernel before the down pass wrote is visible: that pass waited for
  // it before it let this one start
  const int row0 = blockIdx.x * TM;
  find_blocks<TM, 16>(rb, p, row0);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  grid_dependency_wait();
  for (int block = blockIdx.z; block < rb.blocks; block += gridDim.z) {
    const int s = rb.adapter[block];
    if (s < 0) continue;
    const int rank = rank_of(p, s);
    const float scale = p.scales[s];
    for (int i = warp; i < 16; i += kLoraWarps) {
      const int at = rb.start[block] + i;
      if (i >= rb.count[block]) continue;
      const float *src = part + static_cast<long long>(row0 + rb.row[at]) * p.max_rank;
      float v[(RK + 31) / 32], most = 0.0f;
#pragma unroll
      for (int j = 0; j < (RK + 31) / 32; ++j) {
        const int r = lane + 32 * j;
        v[j] = 0.0f;
        if (r < rank)
          for (int range = 0; range < ranges; ++range) v[j] += src[static_cast<long long>(range) * p.m * p.max_rank + r];
        v[j] *= scale;
        most = fmaxf(most, fabsf(v[j]));
      }
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, o));
      float up = 1.0f, down = 1.0f;
      if (PARTS == 2 && most > 0.0f && most < INFINITY) {
        const int e = max(ilogbf(most), -110);
        up = ldexpf(1.0f, 10 - e);
        down = ldexpf(1.0f, e - 10);
      }
      if (lane == 0) undo[at] = down;
#pragma unroll
      for (int j = 0; j < (RK + 31) / 32; ++j) {
        const int r = lane + 32 * j;
        if (r >= RK) continue;
        float rest = v[j] * up;
#pragma unroll
        for (int q = 0; q < PARTS; ++q) {
          const T h = from_f32<T>(rest);
          ts[q][at][r] = h;
          rest = isfinite(rest) ? rest - to_f32(h) : 0.0f;
        }
      }
    }
  }
  __syncthreads();
  const int c0 = blockIdx.y * (kLoraWarps * 32) + warp * 32;
  if (c0 >= p.n) return;
  const bool in_place = p.base == p.out && p.ldb == p.ldo;
  uint2 w[4][KS];
  int held = -1;
  for (int block = blockIdx.z; block < rb.blocks; block += gridDim.z) {
    const int s = rb.adapter[block], start = rb.start[block], count = rb.count[block];
    const int rank = s < 0 ? 0 : rank_of(p, s);
    if (rank == 0 && in_place) continue;
    float4 o[2][2];
    long long row[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const bool ok = g + 8 * i < count;
      row[i] = ok ? row0 + rb.row[start + g + 8 * i] : -1;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int c = c0 + 16 * h + 4 * t;
        o[i][h] = make_float4(0, 0, 0, 0);
        if (ok && p.base && c < p.n) o[i][h] = __ldcs(reinterpret_cast<const float4 *>(p.base + row[i] * p.ldb + c));
      }
    }
    if (rank) {
      if (s != held) {
        held = s;
        const T *b = static_cast<const T *>(p.b) + static_cast<long long>(s) * p.n * p.max_rank;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int c = c0 + 16 * (j >> 1) + 4 * (g >> 1) + 2 * (j & 1) + (g & 1);
#pragma unroll
          for (int k = 0; k < KS; ++k) {
            const int r = 16 * k + 4 * t;
            w[j][k] = make_uint2(0, 0);
            if (c < p.n && r < rank) {
              w[j][k] = *reinterpret_cast<const uint2 *>(b + static_cast<long long>(c) * p.max_rank + r);
              if (r + 1 >= rank) w[j][k].x &= 0xffffu;
              if (r + 2 >= rank) w[j][k].y = 0;
              if (r + 3 >= rank) w[j][k].y &= 0xffffu;
            }
          }
        }
      }
      float acc[4][4];
#pragma unroll
      for (int j = 0; j < 4; ++j) acc[j][0] = acc[j][1] = acc[j][2] = acc[j][3] = 0.0f;
#pragma unroll
      for (int k = 0; k < KS; ++k) {
        if (16 * k >= rank) break;
#pragma unroll
        for (int q = PARTS - 1; q >= 0; --q) {
          uint32_t a[4] = {0, 0, 0, 0};
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            if (row[i] < 0) continue;
            const uint2 v = *reinterpret_cast<const uint2 *>(&ts[q][start + g + 8 * i][16 * k + 4 * t]);
            a[i] = v.x, a[2 + i] = v.y;
          }
#pragma unroll
          for (int j = 0; j < 4; ++j) mma_16<T>(acc[j], a, w[j][k].x, w[j][k].y);
        }
      }
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        if (row[i] < 0) continue;
        const float down = undo[start + g + 8 * i];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          o[i][h].x = fmaf(acc[2 * h][2 * i], down, o[i][h].x);
          o[i][h].y = fmaf(acc[2 * h][2 * i + 1], down, o[i][h].y);
          o[i][h].z = fmaf(acc[2 * h + 1][2 * i], down, o[i][h].z);
          o[i][h].w = fmaf(acc[2 * h + 1][2 * i + 1], down, o[i][h].w);
        }
      }
    }
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int c = c0 + 16 * h + 4 * t;
        if (row[i] >= 0 && c < p.n) __stcs(reinterpret_cast<float4 *>(p.out + row[i] * p.ldo + c), o[i][h]);
      }
  }
}

template <typename T, int RK>
int launch_lora(const LoraArgs &p, const OpDevice &d, cudaStream_t st) {
  // Down: ranges of K until the SMs have a block each (no shorter than one step
  // per warp), and blocks of few tiles side by side.
  constexpr int MB = RK == 128 ? 1 : 2;
  const int tiles = (p.m + 31) / 32;
  const int steps = (p.k + kLoraWarps * 32 - 1) / (kLoraWarps * 32);
  const int ranges = std::max(1, std::min(steps, d.sms / tiles));
  const int k_range = (steps + ranges - 1) / ranges * kLoraWarps * 32;
  const int z_down = std::max(1, std::min({8, p.adapters, p.m, 2 * d.sms / (tiles * ranges)}));
  constexpr int TM = RK == 128 ? 32 : 64;
  const int up_tiles = (p.m + TM - 1) / TM, n_tiles = (p.n + kLoraWarps * 32 - 1) / (kLoraWarps * 32);
  const int z_up = std::max(1, std::min({8, p.adapters, p.m, 4 * d.sms / (up_tiles * n_tiles)}));
  auto lock = op_lock();
  uint32_t *counters;
  uint8_t *scratch;
  const int rc = op_scratch(st, static_cast<size_t>(ranges) * p.m * p.max_rank * sizeof(float), &counters, &scratch);
  if (rc) return rc;
  float *part = reinterpret_cast<float *>(scratch);
  cudaError_t e = op_launch(lora_down_kernel<T, RK, MB>, dim3(tiles, (p.k + k_range - 1) / k_range, z_down), kLoraThreads,
                            0, st, p, part, k_range);
  if (e == cudaSuccess)
    e = op_launch(lora_up_kernel<T, RK>, dim3(up_tiles, n_tiles, z_up), kLoraThreads, 0, st, p, part,
                  (p.k + k_range - 1) / k_range);
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
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  try {
    return p->type == HTPG_TYPE_F16 ? run_lora<__half>(r, d, st) : run_lora<__nv_bfloat16>(r, d, st);
  } catch (const std::exception &) {
    return HTPG_ENOMEM;
  }
}
