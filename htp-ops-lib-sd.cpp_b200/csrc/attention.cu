// Attention over an encoder's states:
//
//   out_i = sum_j w_ij v_j / sum_j w_ij,  w_ij = exp(scale q_i . k_j + bias_j)
//
// in one pass over the keys with the running maximum and sum of the softmax.
// Few rows: mma.sync, bound by the bytes of K and V.  Tiles of 128 rows: tcgen05.
#include <algorithm>
#include <cmath>
#include <exception>

#include "ops.h"
#include "ptx.cuh"

namespace htpg {
namespace {

constexpr int kAttnMaxDim = 192;

struct AttnArgs {
  const void *q, *k, *v;
  void *out;
  const int *lens;
  const float *bias;
  long long qs[3], ks[3], vs[3], os[3];
  long long bias_stride;
  int batch, q_len, kv_len, q_heads, group, dim;
  float scale;
};

// ------------------------------------------------------------ tiles of rows
// 128 query rows of one head are one tile: S = Q K^T (128 rows x up to 64 keys)
// and O += P V are tcgen05.mma into TMEM, softmax in registers, one thread per
// row.  A CTA holds two tiles that share their keys and values (neighbouring
// rows of one head, or heads of one group):
//   warps 0-3, 4-7  softmax of tile 0, 1: S from TMEM, running maximum and sum,
//                   P (16 bits) back into TMEM over S, and the tile's output
//   warps 8, 10     issue the MMAs of tile 0, 1; warp 9 the TMA loads (11 only
//                   makes the warpgroup whole, to hand its registers to the others:
//                   256 x 216 + 128 x 72 = 384 x 168, what the launch gives)
// TMEM columns: per tile two buffers of S (64 each, P in place; one buffer for
// heads above 128) and O (DP).  With two, the scores of the next two key tiles are
// made while the softmax of one runs, so the chain scores -> softmax -> weights
// never waits for the tensor core.  P is the A operand in TMEM; V, as loaded
// ([key][dim]), the MN-major B operand.
// Rounding: scores and sums are FP32; the weights are rounded to the 16 bits of
// the tensor core's A operand (with FP32 outputs the rest follows as a second
// operand), the sum they are divided by is of the unrounded ones.  16-bit outputs
// are then off by a third more than the exact result rounded once (0.00028 against
// 0.00021 of the norm, FP16); the second operand would take that away for the time
// that FP32 outputs show below.  The maximum is
// only raised (and O rescaled) once a score passes it by 2^kLazy, which changes
// no weight's relative error and lets most tiles skip the rescale.
// Bound by the latency of one step's chain, with no unit full (tensor pipe 34 %,
// issue slots 37 %).  Times alone (the call repeated in a graph): 4 x 4096 queries
// of 12 heads of 128 over 4096 keys, FP16: 407 us = 1010 TFLOP/s (0.61 of cuBLAS)
// for ten after a pause, 457 to 468 kept up, where the power cap lowers the clocks;
// 16384 over 512, BF16: 79 us.  64 keys a tile: 128 with one buffer of S 611 us.
// Turns at the exponentials 489 -> 455, one elected lane issuing 548 -> 489.  Few
// keys are bound by an item's chain load -> scores -> weights -> output, about
// 3.5 us: 2 x 4096 queries of 24 heads of 64 over 77 keys 27.5 us (FP32 out 29.3).
constexpr int kTileThreads = 384;
constexpr int kLensHeld = 256;   // batches whose lengths are kept in shared memory
constexpr float kLazy = 8.0f;    // log2 of how far a score may pass the held maximum
constexpr float kLog2e = 1.4426950408889634f;

struct TileArgs {
  AttnArgs a;
  int pack;            // heads of a group that share a tile (rows token by token), a power of two, or 1
  int log_pack;
  int row_tiles;       // tiles of one head, or of one group's heads together
  int tiles;           // tiles of one key/value head
  int pairs;           // tile pairs of one key/value head
  int kv_heads;
  int units;           // batch * kv_heads * pairs
  int whole;           // the first units are one item each,
  int splits;          // the others this many: ranges of their keys
  int items;           // whole + (units - whole) * splits
  int q_batch, q_head, k_batch, k_head, v_batch, v_head;  // 0: that dimension's stride is 0 (one copy)
  int staged;          // the output has a tensor map (boxes of one warp's 32 rows)
  int wide;            // output rows are 32-byte aligned
  float *part_o;       // of split items: [item - whole][tile][128 rows][dim] sums
  float2 *part_ml;     // [item - whole][tile][128 rows] maximum (log2) and sum
  float4 *sums;        // FP32 outputs over more than kFlush tiles: [CTA][tile][dim / 4][128 rows]
  uint32_t *watchdog;
};

// STAGED: output rows leave through shared memory (FP32 rows of up to 128: twice
// the stores of 16-bit ones, which gain nothing: 2 x 4096 rows of 64 over 77 keys
// 32.7 -> 29.4 us with FP32 outputs, 28.6 -> 30.4 with FP16).
template <int DP, int KT, bool STAGED>
struct TileSmem {
  static constexpr int kQ = 128 * DP * 2;
  static constexpr int kStage = KT * DP * 2;
  static constexpr int kStages = DP == 128 ? (STAGED ? 7 : 8) : DP == 64 ? 10 : 5;
  static constexpr int kBuffers = DP == 192 ? 1 : 2;  // of S, per tile
  static constexpr int kBarriers = 2 * kStages + 18;
  static constexpr int kOut = 2 * kQ + kStages * kStage;
  static constexpr int kBars = kOut + (STAGED ? 8 * 4096 : 0);  // 4 KB per softmax warp
  static constexpr int kLens = kBars + 8 * kBarriers + 24;
  static constexpr int kBias = (kLens + 4 * kLensHeld + 15) / 16 * 16;  // [tile][2][KT]
  static constexpr int kBytes = kBias + 16 * KT + 1024;                 // + alignment
};

template <typename TO>
constexpr bool tile_staged(int dp) {
  return sizeof(TO) == 4 && dp <= 128;
}

// FP32 outputs: the tensor core's sums round towards zero, which takes 2^-24 or
// so of O away with every product and would show over thousands of keys. Every
// kFlush key tiles O is added (to nearest) to sums in global memory, [dim / 4][row]
// per CTA and tile, and begins anew. Four tiles keep the loss below what FP32
// sums over thousands of keys lose anyway: 4096 queries over 4096 keys of 128,
// error 5.2e-6 without, 1.7e-6 with eight, 1.1e-6 with four (FP32 products summed
// in order: 1.4e-6). The sums stay in L2; four floats per atomic: 2 x 4096 queries
// of 12 heads of 128 over 4096 keys 530 us (one per atomic 677); of 24 heads of 64
// 609, where 16-bit outputs take 378.
constexpr int kFlush = 4;

struct TileItem {
  int b, kvh, n, j0, j1, split;  // n keys take part, tiles [j0, j1) of them are this item's
  int head[2], row0[2];  // first head and token of each tile
  bool two;
};

__device__ __forceinline__ int clamped_len(const AttnArgs &a, int b) {
  return a.lens ? min(max(a.lens[b], 0), a.kv_len) : a.kv_len;
}

template <int KT>
__device__ __forceinline__ TileItem tile_item(const TileArgs &t, int item, const int *lens) {
  TileItem r;
  uint32_t u = item, pair;
  int splits = 1;
  r.split = 0;
  if (item >= t.whole) {
    splits = t.splits;
    u = (item - t.whole) / splits;
    r.split = item - t.whole - u * splits;
    u += t.whole;
  }
  pair = u;
  u = u / t.pairs;
  pair -= u * t.pairs;
  r.b = u / t.kv_heads;
  r.kvh = u - r.b * t.kv_heads;
  r.n = r.b < kLensHeld ? lens[r.b] : clamped_len(t.a, r.b);
  const int tiles = (r.n + KT - 1) / KT, per = (tiles + splits - 1) / splits;
  r.j0 = min(r.split * per, tiles);
  r.j1 = min(r.j0 + per, tiles);
  r.two = 2 * static_cast<int>(pair) + 1 < t.tiles;
#pragma unroll
  for (int w = 0; w < 2; ++w) {
    const uint32_t tile = 2 * pair + w, head = t.tiles == t.row_tiles ? 0 : tile / t.row_tiles;
    r.head[w] = r.kvh * t.a.group + head;
    r.row0[w] = (tile - head * t.row_tiles) * (128 >> t.log_pack);
  }
  return r;
}

// A key's bias in units of log2.  The lowest finite ones stay finite (-inf would
// take their keys out); NaN stays NaN.
__device__ __forceinline__ float bias_log2(float add) {
  add *= kLog2e;
  return add == -INFINITY ? -3.402823466e38f : add;
}

__device__ __forceinline__ void store32(void *p, const uint32_t (&v)[8], bool wide) {
  if (wide) {
    asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "r"(v[0]), "r"(v[1]), "r"(v[2]),
                 "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7])
                 : "memory");
  } else {
    reinterpret_cast<uint4 *>(p)[0] = make_uint4(v[0], v[1], v[2], v[3]);
    reinterpret_cast<uint4 *>(p)[1] = make_uint4(v[4], v[5], v[6], v[7]);
  }
}

// 32 output columns [c, c + 32) of one row, those below dim.
template <typename TO>
__device__ __forceinline__ void store_columns(TO *row, int c, int dim, const float (&o)[32], bool wide) {
  if constexpr (sizeof(TO) == 4) {
#pragma unroll
    for (int j = 0; j < 32; j += 8) {
      if (c + j >= dim) break;
      uint32_t v[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = __float_as_uint(o[j + i]);
      store32(row + c + j, v, wide);
    }
  } else {
#pragma unroll
    for (int j = 0; j < 32; j += 16) {
      if (c + j >= dim) break;
      uint32_t v[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = pack2<TO>(o[j + 2 * i], o[j + 2 * i + 1]);
      if (c + j + 16 <= dim)
        store32(row + c + j, v, wide);
      else
        *reinterpret_cast<uint4 *>(row + c + j) = make_uint4(v[0], v[1], v[2], v[3]);
    }
  }
}

template <typename T, typename TO, int DP, int KT>
__global__ void __launch_bounds__(kTileThreads, 1)
    attn_tile_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k,
                     const __grid_constant__ CUtensorMap map_v, const __grid_constant__ CUtensorMap map_out,
                     const __grid_constant__ TileArgs t) {
  constexpr bool kStaged = tile_staged<TO>(DP);
  using L = TileSmem<DP, KT, kStaged>;
  // FP32 outputs: P in two 16-bit parts, high and low, each KT / 2 TMEM columns
  constexpr bool kParts = sizeof(TO) == 4;
  // FP16 weights are 2^7 times larger, so that those down to 2^-21 of the
  // largest keep their 11 bits; with kLazy they stay at 2^15 or below
  constexpr float kShift = std::is_same<T, __half>::value ? 7.0f : 0.0f;
  constexpr uint32_t kFormat = std::is_same<T, __half>::value ? 0u : 1u;
  constexpr uint32_t kIdesc = (1u << 4) | (kFormat << 7) | (kFormat << 10) | (8u << 24);  // F32 sums, M = 128
  constexpr int NS = L::kStages;
  constexpr int NB = L::kBuffers;
  constexpr uint32_t kO = 2 * NB * KT;  // first TMEM column of O

  extern __shared__ uint8_t raw[];
  uint8_t *base = raw + ((1024u - (smem_u32(raw) & 1023u)) & 1023u);
  const uint32_t q_s = smem_u32(base), kv_s = q_s + 2 * L::kQ;
  const uint32_t bars = q_s + L::kBars;
  const uint32_t kv_full = bars, kv_empty = bars + 8 * NS, q_full = bars + 16 * NS, q_empty = q_full + 16;
  // per tile and buffer; per tile
  const uint32_t s_full = q_empty + 16, p_ready = s_full + 32, pv_done = p_ready + 32, mma_done = pv_done + 32;
  uint32_t *slot = reinterpret_cast<uint32_t *>(base + L::kBars + 8 * L::kBarriers);
  volatile uint32_t *abort = slot + 1;
  int *lens = reinterpret_cast<int *>(base + L::kLens);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    *abort = 0;
    for (int i = 0; i < NS; ++i) mbar_init(kv_full + 8 * i, 1), mbar_init(kv_empty + 8 * i, 2);
    for (int w = 0; w < 2; ++w) {
      mbar_init(q_full + 8 * w, 1);
      mbar_init(q_empty + 8 * w, 1);
      // (one of each per buffer: a wait for step n then cannot take step n - 1's phase for its own)
      for (int i = 0; i < 2; ++i) {
        mbar_init(s_full + 16 * w + 8 * i, 1);
        mbar_init(p_ready + 16 * w + 8 * i, 4);
        mbar_init(pv_done + 16 * w + 8 * i, 1);
      }
      mbar_init(mma_done + 8 * w, 1);
    }
    fence_barrier_init();
  }
  if (warp == 8) {
    tmem_alloc(smem_u32(slot), 512);
    tmem_relinquish();
  }
  if (warp == 9 && lane == 0) {
    tma_prefetch_desc(&map_q);
    tma_prefetch_desc(&map_k);
    tma_prefetch_desc(&map_v);
  }
  grid_dependency_wait();
  for (int i = threadIdx.x; i < min(t.a.batch, kLensHeld); i += kTileThreads) lens[i] = clamped_len(t.a, i);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *slot;
  const int dim = t.a.dim;

  if (warp >= 8) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 72;");
    if (warp == 9) {
      // ------------------------------------------------------------ loads
      bool ok = true;
      uint32_t loads = 0, tiles[2] = {0, 0};  // K and V tiles, query tiles issued
      const int panels = (dim + 63) / 64;
      auto wait = [&](uint32_t bar, uint32_t parity) {
        return __all_sync(0xffffffffu, mbar_wait(bar, parity, t.watchdog, kWatchProducer, abort)) != 0;
      };
      auto load = [&](const CUtensorMap *map, int j, int h, int b) {
        const uint32_t s = loads % NS, bar = kv_full + 8 * s;
        if (!wait(kv_empty + 8 * s, (loads / NS & 1u) ^ 1u)) return false;
        if (elect_one()) {
          mbar_arrive_expect_tx(bar, panels * KT * 128);
          for (int p = 0; p < panels; ++p)
            tma_load_4d(kv_s + s * L::kStage + p * KT * 128, map, bar, p * 64, j * KT, h, b);
        }
        ++loads;
        return true;
      };
      for (int item = blockIdx.x; ok && item < t.items; item += gridDim.x) {
        const TileItem it = tile_item<KT>(t, item, lens);
        if (it.j0 == it.j1) continue;
        for (int w = 0; ok && w < (it.two ? 2 : 1); ++w) {
          ok = wait(q_empty + 8 * w, (tiles[w] & 1u) ^ 1u);
          if (!ok) break;
          if (elect_one()) {
            mbar_arrive_expect_tx(q_full + 8 * w, panels * 128 * 128);
            for (int p = 0; p < panels; ++p)
              tma_load_5d(q_s + w * L::kQ + p * 128 * 128, &map_q, q_full + 8 * w, p * 64, 0, w ? it.row0[1] : it.row0[0],
                          (t.pack > 1 ? it.kvh : w ? it.head[1] : it.head[0]) * t.q_head, it.b * t.q_batch);
          }
          ++tiles[w];
          // the first keys right after the first tile's queries
          if (w == 0) ok = load(&map_k, it.j0, it.kvh * t.k_head, it.b * t.k_batch);
        }
        for (int j = it.j0; ok && j < it.j1; ++j) {
          if (j > it.j0) ok = load(&map_k, j, it.kvh * t.k_head, it.b * t.k_batch);
          ok = ok && load(&map_v, j, it.kvh * t.v_head, it.b * t.v_batch);
        }
      }
      // never leave the CTA with a copy still landing in its shared memory
      for (uint32_t i = loads > NS ? loads - NS : 0; i < loads; ++i)
        mbar_wait(kv_full + 8 * (i % NS), i / NS & 1u, t.watchdog, kWatchProducer, abort);
      for (int w = 0; w < 2; ++w)
        if (tiles[w]) mbar_wait(q_full + 8 * w, (tiles[w] - 1) & 1u, t.watchdog, kWatchProducer, abort);
    }
    if (warp == 8 || warp == 10) {
      // ------------------------------------------------------------- MMAs
      // The whole warp runs the loop, so that descriptors stay in uniform
      // registers; one lane issues.
      const int w = warp == 10;
      const int ksteps = (dim + 15) / 16;
      const uint64_t desc_q = umma_desc_sw128(q_s + w * L::kQ), desc_k = umma_desc_sw128(kv_s);
      const uint64_t desc_v = umma_desc_sw128_mn(kv_s, KT * 128);
      const uint32_t idesc_v = kIdesc | (1u << 16) | (static_cast<uint32_t>(ksteps * 2) << 17);  // V: MN-major, N = dim
      const uint32_t s_t = tmem + w * NB * KT, o_t = tmem + kO + w * DP;
      auto wait = [&](uint32_t bar, uint32_t parity) {
        const bool got = mbar_wait(bar, parity, t.watchdog, kWatchMma, abort);
        tc_fence_after();
        return __all_sync(0xffffffffu, got) != 0;
      };
      // Steps: the key tiles of this CTA's items, one after the other.  At each:
      // O += P V of the step NB before, then S = Q K^T of this one into the buffer
      // that frees.  Slots: K of step n in 2n, V in 2n + 1; both tiles' warps
      // release them, this one at once where the item has no second tile.
      struct Step {
        int keys = 0;  // 0: none
        bool mine = false, opens = false, first = false, last = false;
      } past[NB];
      uint32_t queries = 0, made = 0, taken = 0, n = 0;  // made, taken: steps of this tile
      TileItem it;
      int item = blockIdx.x, j = 0;
      bool ok = true, open = false;
      for (; ok; ++n) {
        Step now;
        while (!open && item < t.items) {
          it = tile_item<KT>(t, item, lens);
          it.n = __shfl_sync(0xffffffffu, it.n, 0);
          it.j0 = __shfl_sync(0xffffffffu, it.j0, 0);
          it.j1 = __shfl_sync(0xffffffffu, it.j1, 0);
          item += gridDim.x;
          j = it.j0;
          open = it.j0 < it.j1;
        }
        if (open) {
          now.keys = min(KT, it.n - j * KT);
          now.mine = w == 0 || it.two;
          now.first = kParts ? (j - it.j0) % kFlush == 0 : j == it.j0;  // O is overwritten
          now.opens = j == it.j0;
          now.last = ++j == it.j1;
          open = !now.last;
        }
        const Step old = past[0];
        if (!now.keys && !old.keys && (NB == 1 || !past[NB - 1].keys)) break;
        if (old.keys) {
          const uint32_t v_slot = (2 * (n - NB) + 1) % NS, v_phase = (2 * (n - NB) + 1) / NS & 1u;
          const uint32_t buf = taken % NB;
          if (old.mine) ok = wait(p_ready + 16 * w + 8 * buf, taken / NB & 1u);
          ok = ok && wait(kv_full + 8 * v_slot, v_phase);
          if (!ok) break;
          if (!old.mine) {
            if (elect_one()) mbar_arrive(kv_empty + 8 * v_slot);
          } else {
            ++taken;
            if (elect_one()) {
              // P of 32 keys (two K = 16 steps): 16 columns high parts, 16 low, where their scores were
              const uint64_t dv = desc_v + v_slot * (L::kStage / 16);
              const uint32_t p_t = s_t + buf * KT;
              uint32_t more = !old.first;  // 0: O is overwritten
#pragma unroll
              for (int i = 0; i < KT / 32; ++i) {
                if (i * 32 >= old.keys) break;
                umma_f16_ta(o_t, p_t + i * 32, dv + i * 256, idesc_v, more);
                if (kParts) umma_f16_ta(o_t, p_t + i * 32 + 16, dv + i * 256, idesc_v, 1);
                more = 1;
                if (i * 32 + 16 < old.keys) {
                  umma_f16_ta(o_t, p_t + i * 32 + 8, dv + i * 256 + 128, idesc_v, 1);
                  if (kParts) umma_f16_ta(o_t, p_t + i * 32 + 24, dv + i * 256 + 128, idesc_v, 1);
                }
              }
              tc_commit(pv_done + 16 * w + 8 * buf);
              tc_commit(kv_empty + 8 * v_slot);
            }
          }
        }
        if (now.keys) {
          const uint32_t k_slot = 2 * n % NS;
          if (now.mine && now.opens) ok = wait(q_full + 8 * w, queries++ & 1u);
          ok = ok && wait(kv_full + 8 * k_slot, 2 * n / NS & 1u);
          if (!ok) break;
          if (!now.mine) {
            if (elect_one()) mbar_arrive(kv_empty + 8 * k_slot);
          } else {
            const uint32_t buf = made++ % NB;
            if (elect_one()) {
              uint64_t dq = desc_q, dk = desc_k + k_slot * (L::kStage / 16);
              const uint32_t idesc = kIdesc | (static_cast<uint32_t>((now.keys + 15) / 16 * 2) << 17);
              int i = 0;
#pragma unroll
              for (int panel = 0; panel < DP / 64; ++panel) {
                if (i + 4 > ksteps) break;
                umma_f16_kblock(s_t + buf * KT, dq, dk, idesc, i > 0);
                i += 4, dq += 128 * 128 / 16, dk += KT * 128 / 16;
              }
#pragma unroll 1
              for (; i < ksteps; ++i, dq += 2, dk += 2) umma_f16(s_t + buf * KT, dq, dk, idesc, i > 0);
              tc_commit(s_full + 16 * w + 8 * buf);
              tc_commit(kv_empty + 8 * k_slot);
              if (now.last) tc_commit(q_empty + 8 * w);
            }
          }
        }
        if (NB > 1) past[0] = past[NB - 1];
        past[NB - 1] = now;
      }
      if (elect_one()) {
        tc_commit(mma_done + 8 * w);  // every MMA is complete before TMEM is freed
        mbar_wait(mma_done + 8 * w, 0, t.watchdog, kWatchMma, abort);
      }
    }
  } else {
    // ------------------------------------------------------------ softmax
    asm volatile("setmaxnreg.inc.sync.aligned.u32 216;");
    const int w = warp >> 2, quad = warp & 3, r = quad * 32 + lane;  // row of the tile = TMEM lane
    const uint32_t s_at0 = tmem + w * NB * KT + (static_cast<uint32_t>(quad) << 21);
    const uint32_t o_at = tmem + kO + w * DP + (static_cast<uint32_t>(quad) << 21);
    const float c = t.a.scale * kLog2e;
    const bool wide = t.wide != 0;
    float *bias_s = reinterpret_cast<float *>(base + L::kBias) + w * 2 * KT;
    uint32_t seen = 0, used = 0;  // steps of this tile; slots passed
    float4 *sums = nullptr;
    if (kParts && t.sums) sums = t.sums + (static_cast<long long>(blockIdx.x) * 2 + w) * (dim / 4) * 128 + r;
    bool ok = true;
    auto wait = [&](bool go, uint32_t bar, uint32_t parity) {
      const bool got = go && mbar_wait(bar, parity, t.watchdog, kWatchEpilogue, abort);
      tc_fence_after();
      return __all_sync(0xffffffffu, got) != 0;
    };
    // No early exit: a tile's threads meet at its named barriers in every
    // iteration; after a wait that gave up they skip the work.
    for (int item = blockIdx.x; item < t.items; item += gridDim.x) {
      const TileItem it = tile_item<KT>(t, item, lens);
      const int row0 = w ? it.row0[1] : it.row0[0], head0 = w ? it.head[1] : it.head[0];
      const int nt = it.j1 - it.j0;
      if (w == 1 && !it.two) {
        used += 2 * nt;
        continue;
      }
      const int token = row0 + (r >> t.log_pack), head = head0 + (r & (t.pack - 1));
      const bool mine = token < t.a.q_len;
      const float *bias = t.a.bias ? t.a.bias + it.b * t.a.bias_stride : nullptr;
      const float unit = bias ? 1.0f : c;  // of the scores in s[], in log2
      // top: what weights are relative to, the held maximum less kShift.  It is kept as
      // rounded, so that weights, sums and key ranges agree where scores are so large
      // that FP32 cannot take kShift off exactly, and is compared by differences
      // (exact there), so that weights stay within 2^(kLazy + kShift).
      float top = -INFINITY, sum = 0.0f;
      if (w == 1 && nt) named_bar_arrive(3 + quad, 64);  // tile 0 begins
      for (int j = 0; j < nt; ++j, used += 2) {
        const int k0 = (it.j0 + j) * KT, keys = min(KT, it.n - k0);
        bool dead = r < KT && r >= keys;
        if (bias) {
          // one key per thread; two buffers, taken in turn over all steps (a thread
          // may be one barrier ahead of the slowest reader), so one barrier a step is
          // enough
          float add = r < keys ? ld_dep(bias + k0 + r) : -INFINITY;
          dead = r < KT && add == -INFINITY;
          if (!dead) add = bias_log2(add);
          if (r < KT) bias_s[(seen & 1) * KT + r] = add;
          named_bar_sync(1 + w, 128);
        }
        const uint32_t buf = seen % NB, s_at = s_at0 + buf * KT;
        ok = wait(ok, s_full + 16 * w + 8 * buf, seen / NB & 1u);
        ++seen;
        float2 s[KT / 32][16];
        if (ok) {
          tmem_ld32(s_at, s[0]);
          if (keys > 32) tmem_ld32(s_at + 32, s[1]);
          tmem_ld_wait();
          // What takes no part becomes -inf; with a bias the scores come in units of log2.
          if (bias) {
            const float4 *add = reinterpret_cast<const float4 *>(bias_s + (~seen & 1) * KT);  // seen: counted on
#pragma unroll
            for (int x = 0; x < KT / 2; x += 2) {
              const float4 y = add[x / 2];
              float2 &s0 = s[x / 16][x % 16], &s1 = s[x / 16][x % 16 + 1];
              const float2 c2 = make_float2(c, c);
              const float2 f0 = fma2(s0, c2, make_float2(y.x, y.y)), f1 = fma2(s1, c2, make_float2(y.z, y.w));
              s0 = make_float2(y.x == -INFINITY ? -INFINITY : f0.x, y.y == -INFINITY ? -INFINITY : f0.y);
              s1 = make_float2(y.z == -INFINITY ? -INFINITY : f1.x, y.w == -INFINITY ? -INFINITY : f1.y);
            }
          } else if (keys < KT) {
#pragma unroll
            for (int x = 0; x < KT / 2; ++x) {
              float2 &s0 = s[x / 16][x % 16];
              if (2 * x >= keys) s0.x = -INFINITY;
              if (2 * x + 1 >= keys) s0.y = -INFINITY;
            }
          }
          // Four running maxima and sums: one of each would be a chain of 64 dependent operations.
          float most4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
          for (int x = 0; x < KT / 2; ++x)
            most4[x % 4] = fmaxf(most4[x % 4], fmaxf(s[x / 16][x % 16].x, s[x / 16][x % 16].y));
          const float most = fmaxf(fmaxf(most4[0], most4[1]), fmaxf(most4[2], most4[3])) * unit;
          const bool raise = most - top > kLazy + kShift;  // from -inf too; NaN where both are -inf: no
          if (__any_sync(0xffffffffu, raise)) {
            const float to = most - kShift, keep = raise ? ex2_approx(top - to) : 1.0f;
            if (raise) {
              top = to;
              sum *= keep;
            }
            if (j > 0) {
              ok = wait(ok, pv_done + 16 * w + 8 * ((seen - 2) % NB), (seen - 2) / NB & 1u);  // the step before's
#pragma unroll 1
              for (int i = 0; ok && i < dim; i += 32) {
                uint32_t o[32];
                tmem_ld32(o_at + i, o);
                tmem_ld_wait();
#pragma unroll
                for (int x = 0; x < 32; ++x) o[x] = __float_as_uint(__uint_as_float(o[x]) * keep);
                tmem_st32(o_at + i, o);
              }
              if (kParts && j > kFlush && keep != 1.0f) {
#pragma unroll 4
                for (int i = 0; i < dim / 4; ++i) {
                  const float4 y = __ldcg(sums + i * 128);
                  __stcg(sums + i * 128, make_float4(y.x * keep, y.y * keep, y.z * keep, y.w * keep));
                }
              }
            }
          }
        }
        // The two tiles' warps of one scheduler take turns at the exponentials, so
        // that one's run while the other waits, loads and compares (left alone
        // they fall into step, and the exponential unit idles in between).
        if (it.two) named_bar_sync(3 + 4 * w + quad, 64);
        if (ok) {
          const float from = top == -INFINITY ? 0.0f : top;
          const float2 zero2 = make_float2(0.0f, 0.0f);
          float2 sum4[4] = {make_float2(sum, 0.0f), zero2, zero2, zero2};
#pragma unroll
          for (int h = 0; h < KT / 32; ++h) {
            if (32 * h >= keys) break;
            uint32_t w32[32];  // 16 words high parts, 16 low
#pragma unroll
            for (int x = 0; x < 16; ++x) {
              float2 p = fma2(s[h][x], make_float2(unit, unit), make_float2(-from, -from));
              p = make_float2(ex2_approx(p.x), ex2_approx(p.y));
              sum4[x % 4] = add2(sum4[x % 4], p);
              w32[x] = pack2<T>(p.x, p.y);
              if (kParts) {
                const float2 rest = fma2(unpack2<T>(w32[x]), make_float2(-1.0f, -1.0f), p);
                w32[16 + x] = pack2<T>(rest.x, rest.y);
              }
            }
            if (kParts)
              tmem_st32(s_at + 32 * h, w32);
            else
              tmem_st16(s_at + 32 * h, *reinterpret_cast<const uint32_t(*)[16]>(w32));
          }
          sum4[0] = add2(add2(sum4[0], sum4[1]), add2(sum4[2], sum4[3]));
          sum = sum4[0].x + sum4[0].y;
        }
        if (it.two && (w == 0 || j + 1 < nt)) named_bar_arrive(3 + 4 * (1 - w) + quad, 64);
        if (kParts && j > 0 && j % kFlush == 0) {
          // by now the product of the step before is done, and this step's waits for its weights
          ok = wait(ok, pv_done + 16 * w + 8 * ((seen - 2) % NB), (seen - 2) / NB & 1u);
          tmem_st_wait();  // O as raised above
#pragma unroll 1
          for (int i = 0; ok && i < dim; i += 32) {
            float o[32];
            tmem_ld32(o_at + i, o);
            tmem_ld_wait();
#pragma unroll
            for (int x = 0; x < 32; x += 4) {
              if (i + x >= dim) break;
              const float4 y = make_float4(o[x], o[x + 1], o[x + 2], o[x + 3]);
              float4 *at = sums + (i + x) / 4 * 128;
              if (j == kFlush)
                __stcg(at, y);
              else
                atomicAdd(at, y);  // this thread's alone, in order; nothing waits for its result
            }
          }
        }
        if (!ok) continue;
        tmem_st_wait();
        tc_fence_before();
        // Values of keys that take no part may be infinite or NaN, which a
        // zero weight would not remove: each tile's threads, one key each, clear
        // them before its product reads them (both tiles write the same zeros).
        if (bias || it.n < t.a.kv_len) {
          dead = dead && r < (keys + 15) / 16 * 16;
          if (__any_sync(0xffffffffu, dead)) {
            const uint32_t v_slot = (used + 1) % NS;
            ok = wait(ok, kv_full + 8 * v_slot, (used + 1) / NS & 1u);
            if (!ok) continue;
            if (dead) {
              const uint32_t at = q_s + 2 * L::kQ + v_slot * L::kStage + r * 128;
              for (int p = 0; p * 64 < dim; ++p)
#pragma unroll
                for (int x = 0; x < 8; ++x)  // in an order that spreads neighbouring rows over the banks
                  sts_u32x4(at + p * KT * 128 + ((x ^ (r & 7)) << 4), 0, 0, 0, 0);
            }
            fence_proxy_async_smem();
          }
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(p_ready + 16 * w + 8 * buf);
      }
      if (nt) ok = wait(ok, pv_done + 16 * w + 8 * ((seen - 1) % NB), (seen - 1) / NB & 1u);
      if (!ok) continue;
      auto load_o = [&](int i, float (&o)[32]) {  // 32 columns
        tmem_ld32(o_at + i, o);
        tmem_ld_wait();
        if (kParts && nt > kFlush) {
#pragma unroll
          for (int x = 0; x < 32; x += 4) {
            if (i + x >= dim) break;
            const float4 y = __ldcg(sums + (i + x) / 4 * 128);
            o[x] += y.x, o[x + 1] += y.y, o[x + 2] += y.z, o[x + 3] += y.w;
          }
        }
      };
      const bool none = sum == 0.0f;  // then O is zero, or there was no tile
      const bool split = item >= t.whole;
      const float inv = split || none ? 1.0f : 1.0f / sum;
      const long long row = (static_cast<long long>(item - t.whole) * 2 + w) * 128 + r;  // of the parts
      TO *out = static_cast<TO *>(t.a.out) + it.b * t.a.os[0] + token * t.a.os[1] + head * t.a.os[2];
      float *part = split ? t.part_o + row * dim : nullptr;
      if (kStaged && t.staged && !split) {
        // Rows of one thread become 128-byte pieces of 32 rows, stored by TMA
        // (which leaves out rows and columns past the ends): straight from the
        // threads, every store would touch 32 lines.
        const uint32_t stage = q_s + L::kOut + warp * 4096, at = stage + lane * 128;
        const int first = row0 + (quad * 32 >> t.log_pack);
#pragma unroll 1
        for (int i = 0; i < dim; i += 32) {
          float o[32];
          if (nt) load_o(i, o);
          uint32_t words[32];
#pragma unroll
          for (int x = 0; x < 32; ++x) words[x] = nt ? __float_as_uint(o[x] * inv) : 0u;
          if (elect_one()) bulk_wait_read_all();  // the piece before has left
          __syncwarp();
#pragma unroll
          for (int x = 0; x < 8; ++x)
            sts_u32x4(at + ((x ^ (lane & 7)) << 4), words[4 * x], words[4 * x + 1], words[4 * x + 2], words[4 * x + 3]);
          fence_proxy_async_smem();
          __syncwarp();
          if (first < t.a.q_len && elect_one()) {
            tma_store_5d(&map_out, stage, i, 0, first, t.pack > 1 ? it.kvh : head0, it.b);
            bulk_commit();
          }
        }
      } else {
#pragma unroll 1
        for (int i = 0; i < dim; i += 32) {
          float o[32];
          if (nt) load_o(i, o);
#pragma unroll
          for (int x = 0; x < 32; ++x) o[x] = nt ? o[x] * inv : 0.0f;
          if (mine) {
            if (part)
              store_columns<float>(part, i, dim, o, true);
            else
              store_columns<TO>(out, i, dim, o, wide);
          }
        }
      }
      if (part && mine) t.part_ml[row] = make_float2(none ? -INFINITY : top, sum);
      tc_fence_before();  // O has been read before the next tile's P is announced
    }
  }
  if (kStaged && warp < 8 && elect_one()) bulk_wait_all();  // output pieces still leaving
  tc_fence_before();
  __syncthreads();
  if (warp == 8) {
    __syncwarp();
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

// Joins the key ranges of the split units' rows, in order: one warp per row.
template <typename TO>
__global__ void __launch_bounds__(256) attn_join_kernel(const __grid_constant__ TileArgs t) {
  grid_dependency_wait();
  const int lane = threadIdx.x & 31;
  const int index = blockIdx.x * 8 + (threadIdx.x >> 5);  // unit, tile, row
  const int unit = index / 256, w = index / 128 % 2, r = index % 128;
  const uint32_t u = t.whole + unit, pair = u % t.pairs, tile = 2 * pair + w;
  const int kvh = u / t.pairs % t.kv_heads, b = u / t.pairs / t.kv_heads;
  if (tile >= static_cast<uint32_t>(t.tiles)) return;
  const int i = tile % t.row_tiles * (128 / t.pack) + r / t.pack;
  const int h = kvh * t.a.group + tile / t.row_tiles + r % t.pack;
  if (i >= t.a.q_len) return;
  const long long first = (static_cast<long long>(unit) * t.splits * 2 + w) * 128 + r;  // the ranges: 256 rows apart
  float top = -INFINITY;
  for (int s = 0; s < t.splits; ++s) top = fmaxf(top, t.part_ml[first + s * 256].x);
  const float from = top == -INFINITY ? 0.0f : top;
  float sum = 0.0f;
  for (int s = 0; s < t.splits; ++s) {
    const float2 ml = t.part_ml[first + s * 256];
    sum += ml.y * ex2_approx(ml.x - from);
  }
  const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
  TO *out = static_cast<TO *>(t.a.out) + b * t.a.os[0] + i * t.a.os[1] + h * t.a.os[2];
  for (int d = lane; d < t.a.dim; d += 32) {
    float o = 0.0f;
    for (int s = 0; s < t.splits; ++s)
      o += t.part_o[(first + s * 256) * t.a.dim + d] * ex2_approx(t.part_ml[first + s * 256].x - from);
    out[d] = from_f32<TO>(sum == 0.0f ? 0.0f : o * inv);
  }
}

// ------------------------------------------------------------ few rows
// Up to 16 query rows that share one key/value head (the tokens of a decode
// step times the heads of a group): bound by reading K and V once.  Four warps
// take every fourth chunk of 16 keys; each has a ring of chunks of its own,
// filled by asynchronous copies, so about 100 KB are in flight per SM.  S and O
// are m16n8k16 products on rows of the ring (ldmatrix, transposed for V), with
// a running maximum and sum per warp, joined at the end through shared
// memory, and over the key ranges of a unit by its last CTA, in order.  Keys
// that take no part are never copied: their rows are zeros.  Weights are rounded
// as in the tiles above (two parts for FP32 outputs).
// 16 requests, 32 heads in 8 groups of 128, over 1500 keys and fewer, FP32 out: 22 us
// for 74 MB with K and V in part in L2, 28.6 in a sequence of calls on other ones (2.6
// TB/s; the wave's tail and the chain copy -> scores -> weights of each warp's
// chunks, 25 % issue); one request over 8192 keys: 13 us for 34 MB.
constexpr int kFewWarps = 4, kFewRows = 16, kFewKeys = 16;

struct FewArgs {
  AttnArgs a;
  int kv_heads, splits, per;  // per: chunks of one range
  int unit16;                 // 16-byte pieces of a row in shared memory that hold data or zeros
  uint32_t magic;             // i / unit16 = i * magic >> 16
  float *part_o;              // [unit][split][16][dim]
  float2 *part_ml;            // [unit][split][16]
  uint32_t *counters;         // [unit], left zero
};

template <int DB>
struct FewSmem {
  static constexpr int kPitch = DB * 2 + 16;  // an odd number of 16-byte pieces: 8 rows on different banks
  static constexpr int kStage = 2 * kFewKeys * kPitch;
  static constexpr int kStages = DB == 64 ? 5 : DB == 128 ? 3 : 2;
  static constexpr int kRing = kFewWarps * kStages * kStage;
  static constexpr int kJoin = kFewWarps * kFewRows * (DB + 2) * 4;
  static constexpr int kBytes = kRing > kJoin ? kRing : kJoin;
};

__device__ __forceinline__ void ldmatrix4(uint32_t (&r)[4], uint32_t at) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(at)
               : "memory");
}
__device__ __forceinline__ void ldmatrix4t(uint32_t (&r)[4], uint32_t at) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(at)
               : "memory");
}

// FULL: heads of exactly DB elements (a lane then always copies the same pieces).
template <typename T, typename TO, int DB, bool FULL>
__global__ void __launch_bounds__(kFewWarps * 32, 2) attn_few_kernel(const __grid_constant__ FewArgs f) {
  using S = FewSmem<DB>;
  constexpr int KS = DB / 16, NS = S::kStages;
  constexpr bool kParts = sizeof(TO) == 4;
  constexpr float kShift = std::is_same<T, __half>::value ? 7.0f : 0.0f;
  extern __shared__ __align__(16) uint8_t smem[];
  __shared__ bool last;
  grid_dependency_wait();
  const AttnArgs &a = f.a;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int split = blockIdx.x % f.splits, unit = blockIdx.x / f.splits;
  const int kvh = unit % f.kv_heads, b = unit / f.kv_heads;
  const int rows = a.q_len * a.group, n = clamped_len(a, b), dim = FULL ? DB : a.dim;
  const T *k = static_cast<const T *>(a.k) + b * a.ks[0] + kvh * a.ks[2];
  const T *v = static_cast<const T *>(a.v) + b * a.vs[0] + kvh * a.vs[2];
  const float *bias = a.bias ? a.bias + b * a.bias_stride : nullptr;
  const int chunks = (n + kFewKeys - 1) / kFewKeys;
  const int first = min(split * f.per, chunks), end = min(first + f.per, chunks);

  uint8_t *ring = smem + warp * (NS * S::kStage);
  auto load = [&](int chunk, int slot) {
    if (chunk < end) {
      const int key0 = chunk * kFewKeys;
      bool in = lane < kFewKeys && key0 + lane < n;
      if (bias && in) in = ld_dep(bias + key0 + lane) != -INFINITY;
      const uint32_t live = __ballot_sync(0xffffffffu, in);
      uint8_t *ks = ring + slot * S::kStage, *vs = ks + kFewKeys * S::kPitch;
      if constexpr (FULL) {
        constexpr int kUnit = DB / 8, kRows = 32 / kUnit;  // pieces of a row, rows of one pass
        const int row0 = lane / kUnit, d = lane % kUnit * 8;
        const T *kp = k + static_cast<long long>(key0 + row0) * a.ks[1] + d;
        const T *vp = v + static_cast<long long>(key0 + row0) * a.vs[1] + d;
        const uint32_t to = row0 * S::kPitch + d * 2;
#pragma unroll
        for (int i = 0; i < kFewKeys / kRows; ++i) {
          const bool take = live >> (row0 + i * kRows) & 1u;
          copy16(ks + to + i * kRows * S::kPitch, take ? kp : k, take);
          copy16(vs + to + i * kRows * S::kPitch, take ? vp : v, take);
          kp += kRows * a.ks[1], vp += kRows * a.vs[1];
        }
      } else {
        for (int i = lane; i < kFewKeys * f.unit16; i += 32) {
          const int row = i * f.magic >> 16, piece = i - row * f.unit16;
          const bool take = (live >> row & 1u) && piece * 8 < dim;
          const long long key = take ? key0 + row : 0;
          const int d = take ? piece * 8 : 0;
          copy16(ks + row * S::kPitch + piece * 16, k + key * a.ks[1] + d, take);
          copy16(vs + row * S::kPitch + piece * 16, v + key * a.vs[1] + d, take);
        }
      }
    }
    copy_commit();
  };
#pragma unroll
  for (int i = 0; i < NS - 1; ++i) load(first + warp + i * kFewWarps, i);

  // the rows' queries as A operand: rows g and g + 8, elements 2t, 2t + 1 and 2t + 8, 2t + 9 of each 16
  uint32_t q[KS][4];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int r = g + 8 * i;
    const T *src = static_cast<const T *>(a.q) + b * a.qs[0] + static_cast<long long>(r < rows ? r / a.group : 0) * a.qs[1] +
                   static_cast<long long>(kvh * a.group + (r < rows ? r % a.group : 0)) * a.qs[2];
#pragma unroll
    for (int s = 0; s < KS; ++s)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int d = 16 * s + 8 * h + 2 * t;
        q[s][2 * h + i] = r < rows && d < dim ? ld_dep(reinterpret_cast<const uint32_t *>(src + d)) : 0u;
      }
  }
  const float c = a.scale * kLog2e;
  float o[DB / 8][4];
#pragma unroll
  for (int j = 0; j < DB / 8; ++j) o[j][0] = o[j][1] = o[j][2] = o[j][3] = 0.0f;
  float top[2] = {-INFINITY, -INFINITY}, sum[2] = {0.0f, 0.0f};  // of rows g, g + 8; sum: this lane's keys
  int slot = 0;
  for (int chunk = first + warp; chunk < end; chunk += kFewWarps) {
    load(chunk + (NS - 1) * kFewWarps, slot == 0 ? NS - 1 : slot - 1);
    copy_wait<NS - 1>();
    __syncwarp();
    const uint32_t ks = smem_u32(ring + slot * S::kStage), vs = ks + kFewKeys * S::kPitch;
    slot = slot + 1 == NS ? 0 : slot + 1;
    // s[h]: keys 8h + 2t, 8h + 2t + 1 of rows g (0, 1) and g + 8 (2, 3)
    float s[2][4];
#pragma unroll
    for (int h = 0; h < 2; ++h) s[h][0] = s[h][1] = s[h][2] = s[h][3] = 0.0f;
#pragma unroll
    for (int x = 0; x < KS; ++x) {
      if (16 * x >= dim) break;
      // matrices: keys 0-7 and 8-15 of elements 0-7, then of 8-15
      uint32_t m[4];
      ldmatrix4(m, ks + (lane & 15) * S::kPitch + x * 32 + (lane >> 4) * 16);
      mma_16<T>(s[0], q[x], m[0], m[2]);
      mma_16<T>(s[1], q[x], m[1], m[3]);
    }
    const int key0 = chunk * kFewKeys;
    if (bias || key0 + kFewKeys > n) {
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int key = key0 + 8 * h + 2 * t + e;
          float add = key < n ? 0.0f : -INFINITY;
          if (bias && key < n) {
            add = ld_dep(bias + key);
            if (add != -INFINITY) add = bias_log2(add);
          }
          s[h][e] = add == -INFINITY ? -INFINITY : fmaf(s[h][e], c, add);
          s[h][2 + e] = add == -INFINITY ? -INFINITY : fmaf(s[h][2 + e], c, add);
        }
    } else {
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int e = 0; e < 4; ++e) s[h][e] *= c;
    }
    float keep[2];
    bool moved = false;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      float most = fmaxf(fmaxf(s[0][2 * i], s[0][2 * i + 1]), fmaxf(s[1][2 * i], s[1][2 * i + 1]));
      most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 1));
      most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 2));
      most -= kShift;  // as rounded: weights, sums and ranges agree where it is not exact
      const bool up = most > top[i];
      keep[i] = up ? ex2_approx(top[i] - most) : 1.0f;
      if (up) top[i] = most;
      moved |= up;
      sum[i] *= keep[i];
    }
    if (__any_sync(0xffffffffu, moved)) {
#pragma unroll
      for (int j = 0; j < DB / 8; ++j) o[j][0] *= keep[0], o[j][1] *= keep[0], o[j][2] *= keep[1], o[j][3] *= keep[1];
    }
    uint32_t hi[4], lo[4];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const float from = top[i] == -INFINITY ? 0.0f : top[i];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const float p0 = ex2_approx(s[h][2 * i] - from), p1 = ex2_approx(s[h][2 * i + 1] - from);
        sum[i] += p0 + p1;
        hi[2 * h + i] = pack2<T>(p0, p1);
        if (kParts) {
          const float2 back = unpack2<T>(hi[2 * h + i]);
          lo[2 * h + i] = pack2<T>(p0 - back.x, p1 - back.y);
        }
      }
    }
#pragma unroll
    for (int x = 0; x < KS; ++x) {
      if (16 * x >= dim) break;
      // transposed matrices: keys 0-7 and 8-15 of elements 0-7, then of 8-15
      uint32_t m[4];
      ldmatrix4t(m, vs + (lane & 15) * S::kPitch + x * 32 + (lane >> 4) * 16);
      if (kParts) {
        // the tensor core's sums round towards zero: added up outside of it
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          float y[4] = {0.0f, 0.0f, 0.0f, 0.0f};
          mma_16<T>(y, lo, m[2 * h], m[2 * h + 1]);
          mma_16<T>(y, hi, m[2 * h], m[2 * h + 1]);
#pragma unroll
          for (int e = 0; e < 4; ++e) o[2 * x + h][e] += y[e];
        }
      } else {
        mma_16<T>(o[2 * x], hi, m[0], m[1]);
        mma_16<T>(o[2 * x + 1], hi, m[2], m[3]);
      }
    }
    __syncwarp();  // every lane is done with the chunk before its slot is filled again
  }
  copy_wait<0>();
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    sum[i] += __shfl_xor_sync(0xffffffffu, sum[i], 1);
    sum[i] += __shfl_xor_sync(0xffffffffu, sum[i], 2);
  }
  // join the warps: [warp][row][maximum, sum, dim sums]
  __syncthreads();
  float *join = reinterpret_cast<float *>(smem);
  constexpr int kRow = DB + 2;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    float *row = join + (warp * kFewRows + g + 8 * i) * kRow;
    if (t == 0) row[0] = top[i], row[1] = sum[i];
#pragma unroll
    for (int j = 0; j < DB / 8; ++j)
      *reinterpret_cast<float2 *>(row + 2 + 8 * j + 2 * t) = make_float2(o[j][2 * i], o[j][2 * i + 1]);
  }
  __syncthreads();
  auto out_row = [&](int r) {
    return static_cast<TO *>(a.out) + b * a.os[0] + static_cast<long long>(r / a.group) * a.os[1] +
           static_cast<long long>(kvh * a.group + r % a.group) * a.os[2];
  };
  // one warp per row, lanes over the elements
  for (int r = warp; r < rows; r += kFewWarps) {
    float m = -INFINITY, l = 0.0f, w[kFewWarps];
#pragma unroll
    for (int x = 0; x < kFewWarps; ++x) m = fmaxf(m, join[(x * kFewRows + r) * kRow]);
    const float from = m == -INFINITY ? 0.0f : m;
#pragma unroll
    for (int x = 0; x < kFewWarps; ++x) {
      w[x] = ex2_approx(join[(x * kFewRows + r) * kRow] - from);
      l += w[x] * join[(x * kFewRows + r) * kRow + 1];
    }
    const long long at = (static_cast<long long>(unit) * f.splits + split) * kFewRows + r;
    for (int d = lane; d < dim; d += 32) {
      float y = 0.0f;
#pragma unroll
      for (int x = 0; x < kFewWarps; ++x) y += w[x] * join[(x * kFewRows + r) * kRow + 2 + d];
      if (f.splits > 1)
        f.part_o[at * dim + d] = y;
      else
        out_row(r)[d] = from_f32<TO>(l == 0.0f ? 0.0f : y / l);
    }
    if (f.splits > 1 && lane == 0) f.part_ml[at] = make_float2(m, l);
  }
  if (f.splits == 1) return;
  // the unit's last CTA joins its ranges
  __threadfence();
  __syncthreads();
  if (threadIdx.x == 0) last = atomicAdd(f.counters + unit, 1u) == static_cast<uint32_t>(f.splits - 1);
  __syncthreads();
  if (!last) return;
  __threadfence();
  for (int r = warp; r < rows; r += kFewWarps) {
    const long long at = static_cast<long long>(unit) * f.splits * kFewRows + r;
    // the ranges' maxima and sums, two per lane, then their weighted rows
    float2 ml[2];
    float m = -INFINITY, l = 0.0f, weight[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int x = lane + 32 * i;
      ml[i] = x < f.splits ? __ldcg(&f.part_ml[at + x * kFewRows]) : make_float2(-INFINITY, 0.0f);
      m = fmaxf(m, ml[i].x);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
    const float from = m == -INFINITY ? 0.0f : m;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      weight[i] = ex2_approx(ml[i].x - from);
      l += weight[i] * ml[i].y;
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) l += __shfl_xor_sync(0xffffffffu, l, o);
    float y[DB / 32];
#pragma unroll
    for (int j = 0; j < DB / 32; ++j) y[j] = 0.0f;
#pragma unroll 8
    for (int x = 0; x < f.splits; ++x) {
      const float w = __shfl_sync(0xffffffffu, x < 32 ? weight[0] : weight[1], x & 31);
#pragma unroll
      for (int j = 0; j < DB / 32; ++j) {
        const int d = lane + 32 * j;
        if (d < dim) y[j] += w * __ldcg(&f.part_o[(at + x * kFewRows) * dim + d]);
      }
    }
#pragma unroll
    for (int j = 0; j < DB / 32; ++j) {
      const int d = lane + 32 * j;
      if (d < dim) out_row(r)[d] = from_f32<TO>(l == 0.0f ? 0.0f : y[j] / l);
    }
  }
  if (threadIdx.x == 0) f.counters[unit] = 0;
}

// Stride (bytes) of an extent: its own where it is stepped along, any valid one otherwise.
uint64_t step_of(bool stepped, int64_t stride, int dim, int bytes) {
  return static_cast<uint64_t>(stepped ? stride : dim) * bytes;
}

// A map {dim, tokens, heads, batch} of K or V, boxes of 64 x box_rows.  Heads or
// batches that share one copy (stride 0) become one.
int kv_map(CUtensorMap *map, const struct htpg_attention_params *p, const void *base, const int64_t *stride, int box_rows,
           int *head_step, int *batch_step) {
  *head_step = p->kv_heads > 1 && stride[2] != 0;
  *batch_step = p->batch > 1 && stride[0] != 0;
  const uint64_t heads = *head_step ? p->kv_heads : 1, batches = *batch_step ? p->batch : 1;
  const uint64_t dims[4] = {static_cast<uint64_t>(p->head_dim), static_cast<uint64_t>(p->kv_len), heads, batches};
  const uint64_t strides[3] = {step_of(p->kv_len > 1, stride[1], p->head_dim, 2),
                               step_of(*head_step, stride[2], p->head_dim, 2),
                               step_of(*batch_step, stride[0], p->head_dim, 2)};
  const uint32_t box[4] = {64, static_cast<uint32_t>(box_rows), 1, 1};
  return op_tensor_map(map, p->type, base, 4, dims, strides, box);
}

// A map {dim, packed heads, tokens, heads or groups, batch} of Q or the output,
// boxes of 128 bytes x `rows` rows: rows / pack tokens, each with `pack` heads.
int rows_map(CUtensorMap *map, const struct htpg_attention_params *p, const void *base, int type, const int64_t *stride,
             int pack, int rows, int *head_step, int *batch_step) {
  *head_step = p->q_heads > pack && stride[2] != 0;
  *batch_step = p->batch > 1 && stride[0] != 0;
  const int others = *head_step ? p->q_heads / pack : 1, bytes = type_bytes(type);
  const uint64_t dims[5] = {static_cast<uint64_t>(p->head_dim), static_cast<uint64_t>(pack),
                            static_cast<uint64_t>(p->q_len), static_cast<uint64_t>(others),
                            static_cast<uint64_t>(*batch_step ? p->batch : 1)};
  const uint64_t strides[4] = {step_of(pack > 1, stride[2], p->head_dim, bytes),
                               step_of(p->q_len > 1, stride[1], p->head_dim, bytes),
                               step_of(others > 1, stride[2] * pack, p->head_dim, bytes),
                               step_of(*batch_step, stride[0], p->head_dim, bytes)};
  const uint32_t box[5] = {static_cast<uint32_t>(128 / bytes), static_cast<uint32_t>(pack),
                           static_cast<uint32_t>(rows / pack), 1, 1};
  return op_tensor_map(map, type, base, 5, dims, strides, box);
}

template <typename T, typename TO, int DP, int KT>
int run_tiles(const struct htpg_attention_params *p, const AttnArgs &a, const OpDevice &d, cudaStream_t st) {
  TileArgs t = {};
  t.a = a;
  // A group's heads share tiles where their number divides 128: few tokens then
  // fill a tile (16 tokens x 4 heads in one tile instead of four).
  t.pack = (a.group & (a.group - 1)) == 0 && a.group <= 128 && p->q_stride[2] != 0 ? a.group : 1;
  while (1 << t.log_pack < t.pack) ++t.log_pack;
  t.kv_heads = p->kv_heads;
  const long long row_tiles = (static_cast<long long>(a.q_len) * t.pack + 127) / 128;
  const long long tiles_kv = row_tiles * (a.group / t.pack);
  const long long pairs = (tiles_kv + 1) / 2;
  if (pairs > 0x3ffffff) return HTPG_ECAPACITY;
  t.row_tiles = static_cast<int>(row_tiles);
  t.tiles = static_cast<int>(tiles_kv);
  t.pairs = static_cast<int>(pairs);
  t.watchdog = d.watchdog;
  const long long units = pairs * t.kv_heads * a.batch;
  const int tiles = (a.kv_len + KT - 1) / KT;
  if (units * 64 > 0x3fffffff) return HTPG_ECAPACITY;
  // Rounds of one unit per SM; the units of a last round that would leave half
  // of the SMs idle or more are cut into ranges of keys of two tiles or
  // more, where the round gets shorter by 12 tiles (8 tiles cut in four: 84 -> 88 us
  // in all; 64 cut in five: 455 -> 416).
  const int rest = static_cast<int>(units % d.sms);
  int splits = rest ? std::min(d.sms / rest, tiles / 2) : 1;
  if (splits < 2 || tiles - (tiles + splits - 1) / splits < 12) splits = 1;
  t.units = static_cast<int>(units);
  t.whole = splits > 1 ? t.units - rest : t.units;
  t.splits = splits;
  t.items = t.whole + (t.units - t.whole) * splits;
  t.wide = (reinterpret_cast<uintptr_t>(a.out) & 31u) == 0;
  const int qe[3] = {a.batch, a.q_len, a.q_heads};
  for (int i = 0; i < 3; ++i)
    if (qe[i] > 1 && a.os[i] * sizeof(TO) % 32) t.wide = 0;
  CUtensorMap mq, mk, mv;
  int rc;
  if ((rc = rows_map(&mq, p, a.q, p->type, p->q_stride, t.pack, 128, &t.q_head, &t.q_batch)) ||
      (rc = kv_map(&mk, p, a.k, p->k_stride, KT, &t.k_head, &t.k_batch)) ||
      (rc = kv_map(&mv, p, a.v, p->v_stride, KT, &t.v_head, &t.v_batch)))
    return rc;
  // the output's, where a warp's 32 rows are whole tokens and no two rows are one
  CUtensorMap mo = mq;
  int own_head = 0, own_batch = 0;
  if (tile_staged<TO>(DP) && t.pack <= 32) {
    if ((rc = rows_map(&mo, p, a.out, p->out_type, p->out_stride, t.pack, 32, &own_head, &own_batch))) return rc;
    t.staged = (own_head || p->q_heads == t.pack) && (own_batch || p->batch == 1);
  }
  std::unique_lock<std::mutex> lock;
  const int grid = std::min(t.items, d.sms);
  const bool flushes = sizeof(TO) == 4 && tiles > kFlush;
  if (t.splits > 1 || flushes) {
    lock = op_lock();
    uint32_t *counters;
    uint8_t *scratch;
    const size_t rows = static_cast<size_t>(t.items - t.whole) * 256, ml = rows * sizeof(float2), parts = rows * a.dim * 4;
    rc = op_scratch(st, ml + parts + (flushes ? static_cast<size_t>(grid) * 256 * a.dim * 4 : 0), &counters, &scratch);
    if (rc) return rc;
    t.part_ml = reinterpret_cast<float2 *>(scratch);
    t.part_o = reinterpret_cast<float *>(scratch + ml);
    if (flushes) t.sums = reinterpret_cast<float4 *>(scratch + ml + parts);
  }
  auto *fn = attn_tile_kernel<T, TO, DP, KT>;
  using L = TileSmem<DP, KT, tile_staged<TO>(DP)>;
  cudaError_t e = cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, L::kBytes);
  if (e != cudaSuccess) return op_result(e);
  e = op_launch(fn, dim3(grid), kTileThreads, L::kBytes, st, mq, mk,
                mv, mo, t);
  if (e == cudaSuccess && t.splits > 1)
    e = op_launch(attn_join_kernel<TO>, dim3((t.units - t.whole) * 32), 256, 0, st, t);
  return op_result(e);
}

// No keys: every row is zero.
__global__ void __launch_bounds__(256) attn_zero_kernel(AttnArgs a, int out_bytes) {
  grid_dependency_wait();
  const long long rows = static_cast<long long>(a.batch) * a.q_heads * a.q_len, total = rows * a.dim;
  for (long long i = static_cast<long long>(blockIdx.x) * 256 + threadIdx.x; i < total; i += gridDim.x * 256LL) {
    const long long row = i / a.dim, q = row % a.q_len, h = row / a.q_len % a.q_heads, b = row / a.q_len / a.q_heads;
    const long long at = b * a.os[0] + q * a.os[1] + h * a.os[2] + i % a.dim;
    if (out_bytes == 4)
      static_cast<uint32_t *>(a.out)[at] = 0;
    else
      static_cast<uint16_t *>(a.out)[at] = 0;
  }
}

template <typename T, typename TO, int DB, bool FULL>
int run_few(const struct htpg_attention_params *p, const AttnArgs &a, const OpDevice &d, cudaStream_t st) {
  using S = FewSmem<DB>;
  FewArgs f = {};
  f.a = a;
  f.kv_heads = p->kv_heads;
  f.unit16 = (a.dim + 15) / 16 * 2;
  f.magic = (65536 + f.unit16 - 1) / f.unit16;
  const long long units = static_cast<long long>(a.batch) * p->kv_heads;
  if (units > (1 << 30)) return HTPG_ECAPACITY;
  const int chunks = (a.kv_len + kFewKeys - 1) / kFewKeys;
  // Key ranges: as many as make the rounds of CTAs (two per SM) shortest, in
  // chunks per warp; set-up counts as 2 chunks, with several ranges as 6 and half
  // a chunk for each that is joined (one request, 32 heads over 8192 keys: 16
  // ranges 12.8 us, 37 ranges, a CTA on every slot, 14.9; 16 requests over 1500:
  // 1, 2, 3 ranges 23, 21, 25 us).
  const long long slots = 2LL * d.sms;
  f.splits = 1;
  long long least = -1;
  for (int s = 1; s <= 64 && (s == 1 || (units * s <= 4 * slots && s * kFewWarps <= chunks)); ++s) {
    const int per = (chunks + s - 1) / s;
    const long long rounds = (units * s + slots - 1) / slots;
    const long long cost = rounds * ((per + kFewWarps - 1) / kFewWarps + (s > 1 ? 6 : 2)) * 4 + (s > 1 ? 2 * s : 0);
    if (least < 0 || cost < least) least = cost, f.splits = s;
  }
  f.per = (chunks + f.splits - 1) / f.splits;
  std::unique_lock<std::mutex> lock;
  if (f.splits > 1) {
    lock = op_lock();
    uint8_t *scratch;
    const size_t ml = static_cast<size_t>(units) * f.splits * kFewRows * sizeof(float2);
    const int rc = op_scratch(st, ml + static_cast<size_t>(units) * f.splits * kFewRows * a.dim * 4, &f.counters, &scratch);
    if (rc) return rc;
    f.part_ml = reinterpret_cast<float2 *>(scratch);
    f.part_o = reinterpret_cast<float *>(scratch + ml);
  }
  auto *fn = attn_few_kernel<T, TO, DB, FULL>;
  const cudaError_t e = cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, S::kBytes);
  if (e != cudaSuccess) return op_result(e);
  return op_result(op_launch(fn, dim3(static_cast<unsigned>(units * f.splits)), kFewWarps * 32, S::kBytes, st, f));
}

template <typename T, typename TO>
int run_attention(const struct htpg_attention_params *p, const AttnArgs &a, const OpDevice &d, cudaStream_t st) {
  if (a.kv_len == 0) {
    const long long blocks = (static_cast<long long>(a.batch) * a.q_heads * a.q_len * a.dim + 255) / 256;
    return op_result(op_launch(attn_zero_kernel, dim3(static_cast<unsigned>(std::min<long long>(blocks, 16LL * d.sms))), 256,
                               0, st, a, static_cast<int>(sizeof(TO))));
  }
  if (static_cast<long long>(a.q_len) * a.group <= kFewRows) {
    if (a.dim == 64) return run_few<T, TO, 64, true>(p, a, d, st);
    if (a.dim == 128) return run_few<T, TO, 128, true>(p, a, d, st);
    if (a.dim <= 64) return run_few<T, TO, 64, false>(p, a, d, st);
    if (a.dim <= 128) return run_few<T, TO, 128, false>(p, a, d, st);
    return run_few<T, TO, 192, false>(p, a, d, st);
  }
  if (a.dim <= 64) return run_tiles<T, TO, 64, 64>(p, a, d, st);
  if (a.dim <= 128) return run_tiles<T, TO, 128, 64>(p, a, d, st);
  return run_tiles<T, TO, 192, 64>(p, a, d, st);
}

// 16-byte vectors along every dimension that is stepped along, forwards, and
// within a tensor map's reach; tokens, and everything written, have rows of their own.
bool strides_fit(const int64_t *s, const int (&extent)[3], int per16, bool written) {
  for (int i = 0; i < 3; ++i)
    if (extent[i] > 1 && (s[i] % per16 || s[i] < (i == 1 || written) || s[i] >= (int64_t{1} << 38))) return false;
  return true;
}

}  // namespace
}  // namespace htpg

using namespace htpg;

extern "C" int htpg_cross_attention(const struct htpg_attention_params *p, void *out, const void *q, const void *k,
                                    const void *v, const int32_t *kv_lens, const float *key_bias, void *stream) {
  if (!p || (p->type != HTPG_TYPE_F16 && p->type != HTPG_TYPE_BF16) ||
      (p->out_type != p->type && p->out_type != HTPG_TYPE_F32) || p->reserved)
    return HTPG_EARGS;
  if (p->batch < 0 || p->q_len < 0 || p->kv_len < 0 || p->q_heads < 1 || p->kv_heads < 1 || p->head_dim < 1 ||
      !(p->scale > 0.0f) || !std::isfinite(p->scale))
    return HTPG_EARGS;
  if (p->q_heads % p->kv_heads || p->head_dim % 8 || p->head_dim > kAttnMaxDim) return HTPG_ECAPACITY;
  if (std::max(p->q_len, p->kv_len) > kOpMaxExtent) return HTPG_ECAPACITY;
  if (p->batch == 0 || p->q_len == 0) return HTPG_OK;
  if (!out || !q || (p->kv_len && (!k || !v))) return HTPG_EARGS;
  const int qe[3] = {p->batch, p->q_len, p->q_heads}, ke[3] = {p->batch, p->kv_len, p->kv_heads};
  if (((reinterpret_cast<uintptr_t>(out) | reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(k) |
        reinterpret_cast<uintptr_t>(v)) & 15u) ||
      ((reinterpret_cast<uintptr_t>(kv_lens) | reinterpret_cast<uintptr_t>(key_bias)) & 3u) ||
      !strides_fit(p->q_stride, qe, 8, false) || !strides_fit(p->k_stride, ke, 8, false) ||
      !strides_fit(p->v_stride, ke, 8, false) || !strides_fit(p->out_stride, qe, 16 / type_bytes(p->out_type), true))
    return HTPG_ECONTROL;
  OpDevice d;
  const int rc = op_device(&d);
  if (rc) return rc;
  AttnArgs a = {};
  a.q = q;
  a.k = k;
  a.v = v;
  a.out = out;
  a.lens = kv_lens;
  a.bias = key_bias;
  for (int i = 0; i < 3; ++i) {
    a.qs[i] = p->q_stride[i];
    a.ks[i] = p->k_stride[i];
    a.vs[i] = p->v_stride[i];
    a.os[i] = p->out_stride[i];
  }
  a.bias_stride = p->bias_stride;
  a.batch = p->batch;
  a.q_len = p->q_len;
  a.kv_len = p->kv_len;
  a.q_heads = p->q_heads;
  a.group = p->q_heads / p->kv_heads;
  a.dim = p->head_dim;
  a.scale = p->scale;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  try {
    if (p->type == HTPG_TYPE_F16)
      return p->out_type == HTPG_TYPE_F32 ? run_attention<__half, float>(p, a, d, st)
                                          : run_attention<__half, __half>(p, a, d, st);
    return p->out_type == HTPG_TYPE_F32 ? run_attention<__nv_bfloat16, float>(p, a, d, st)
                                        : run_attention<__nv_bfloat16, __nv_bfloat16>(p, a, d, st);
  } catch (const std::exception &) {
    return HTPG_ENOMEM;
  }
}
