// Per-head RMS norm and rotary positions of projected queries and keys, with
// the conversion of the values in the same pass, and the table of cosines and
// sines they use.
//
//   y = x rsqrt(mean(x^2) + eps) w;   (a', b') = (a cos - b sin, a sin + b cos)
//
// Every element is read and written once and does some ten operations, so the
// pass is bound by HBM: (in + out) bytes per element.
#include <algorithm>
#include <cmath>

#include "ops.h"
#include "ptx.cuh"

namespace htpg {
namespace {

// ---------------------------------------------------------------- the table
// One thread per (position, pair).  Angles in FP64: at position 2^17 an FP32
// angle is off by up to 2^-8 rad, an FP64 one by 2^-37; the values are rounded once.
// Bound by the FP64 power and sine, which a table is worth once: 131072 x 64 pairs
// 120 us.
__global__ void rope_table_kernel(float2 *table, int rows, int pairs, htpg_rope_scaling s, double base, double low,
                                  double high, double mult) {
  const long long i = static_cast<long long>(blockIdx.x) * blockDim.x + threadIdx.x;
  grid_dependency_wait();
  if (i >= static_cast<long long>(rows) * pairs) return;
  const int pair = static_cast<int>(i % pairs);
  const long long pos = i / pairs;
  double f = pow(base, -static_cast<double>(pair) / pairs);
  if (s.scaling == HTPG_ROPE_LINEAR) f /= s.factor;
  if (s.scaling == HTPG_ROPE_YARN) {
    // 0: turns often enough within the trained context, kept; 1: interpolated
    const double ramp = fmin(fmax((pair - low) / (high - low), 0.0), 1.0);
    f = f / s.factor * ramp + f * (1.0 - ramp);
  }
  double sn, cs;
  sincos(static_cast<double>(pos) * f, &sn, &cs);
  table[i] = make_float2(static_cast<float>(cs * mult), static_cast<float>(sn * mult));
}

// ---------------------------------------------------------------- the pass
struct RopePart {
  const void *in;
  void *out;
  const float *weight;
  long long in_stride[3], out_stride[3];
  int heads, rotate;
};

struct RopeArgs {
  RopePart part[3];
  const float2 *table;
  const int *positions;
  int batch, seq, dim, rot, half, table_rows;
  int heads;  // of all parts
  float eps, inv_dim;
};

constexpr int kRopeWarps = 8, kRopeMaxDim = 512;

// Any size and alignment (odd head dims, rotations that are no multiple of 4):
// one warp per (token, head) row, the row staged in shared memory as FP32.  Bound
// by latency: 16384 tokens of 24 heads of 70, FP32 to FP16: 186 us (heads of 72,
// in vectors: 51).
template <typename TI, typename TO>
__global__ void __launch_bounds__(kRopeWarps * 32) rope_row_kernel(RopeArgs a) {
  __shared__ float rows[kRopeWarps][kRopeMaxDim];
  grid_dependency_wait();
  const int lane = threadIdx.x & 31;
  float *row = rows[threadIdx.x >> 5];
  const long long total = static_cast<long long>(a.batch) * a.seq * a.heads;
  for (long long t = static_cast<long long>(blockIdx.x) * kRopeWarps + (threadIdx.x >> 5); t < total;
       t += static_cast<long long>(gridDim.x) * kRopeWarps) {
    int h = static_cast<int>(t % a.heads);
    const long long token = t / a.heads;
    const long long b = token / a.seq, i = token % a.seq;
    int which = 0;
    while (h >= a.part[which].heads) h -= a.part[which++].heads;
    const RopePart &p = a.part[which];
    const TI *x = static_cast<const TI *>(p.in) + b * p.in_stride[0] + i * p.in_stride[1] + h * p.in_stride[2];
    TO *y = static_cast<TO *>(p.out) + b * p.out_stride[0] + i * p.out_stride[1] + h * p.out_stride[2];
    float sum = 0.0f;
    for (int d = lane; d < a.dim; d += 32) {
      row[d] = to_f32(x[d]);
      sum += row[d] * row[d];
    }
    if (p.weight) {
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
      const float inv = 1.0f / sqrtf(sum / static_cast<float>(a.dim) + a.eps);
      for (int d = lane; d < a.dim; d += 32) row[d] = row[d] * inv * p.weight[d];
    }
    __syncwarp();
    const int rot = p.rotate ? a.rot : 0;
    if (rot) {
      const long long pos = a.positions ? a.positions[token] : i;
      const bool ok = pos >= 0 && pos < a.table_rows;
      const float2 *cs = a.table + pos * (rot / 2);
      for (int j = lane; ok && j < rot / 2; j += 32) {  // outside: the table may have no row at all
        const int d0 = a.half ? j : 2 * j, d1 = a.half ? j + rot / 2 : 2 * j + 1;
        const float2 w = cs[j];
        const float u = row[d0], v = row[d1];
        row[d0] = u * w.x - v * w.y;
        row[d1] = u * w.y + v * w.x;
      }
      __syncwarp();
      if (!ok)
        for (int d = lane; d < a.dim; d += 32) row[d] = __int_as_float(0x7fffffff);
    }
    for (int d = lane; d < a.dim; d += 32) y[d] = from_f32<TO>(row[d]);
    __syncwarp();
  }
}

// ---------------------------------------------------------------- vectors
// N consecutive elements as FP32 (ONCE: evicted first), and back.
template <typename T, int N, bool ONCE = true>
__device__ __forceinline__ void load_n(const T *p, float *v) {
  auto get = [](auto *q) { return ONCE ? __ldcs(q) : *q; };
  if constexpr (sizeof(T) == 4) {
    if constexpr (N % 4 == 0) {
#pragma unroll
      for (int i = 0; i < N; i += 4) {
        const float4 x = get(reinterpret_cast<const float4 *>(p + i));
        v[i] = x.x, v[i + 1] = x.y, v[i + 2] = x.z, v[i + 3] = x.w;
      }
    } else {
      const float2 x = get(reinterpret_cast<const float2 *>(p));
      v[0] = x.x, v[1] = x.y;
    }
  } else {
    uint32_t r[(N + 1) / 2];
    if constexpr (N == 8) {
      const uint4 x = get(reinterpret_cast<const uint4 *>(p));
      r[0] = x.x, r[1] = x.y, r[2] = x.z, r[3] = x.w;
    } else if constexpr (N == 4) {
      const uint2 x = get(reinterpret_cast<const uint2 *>(p));
      r[0] = x.x, r[1] = x.y;
    } else {
      r[0] = get(reinterpret_cast<const uint32_t *>(p));
    }
#pragma unroll
    for (int i = 0; i < N; i += 2) {
      const float2 x = unpack2<T>(r[i / 2]);
      v[i] = x.x, v[i + 1] = x.y;
    }
  }
}
template <typename T, int N>
__device__ __forceinline__ void store_n(T *p, const float *v) {
  if constexpr (sizeof(T) == 4) {
    if constexpr (N % 4 == 0) {
#pragma unroll
      for (int i = 0; i < N; i += 4) *reinterpret_cast<float4 *>(p + i) = make_float4(v[i], v[i + 1], v[i + 2], v[i + 3]);
    } else {
      *reinterpret_cast<float2 *>(p) = make_float2(v[0], v[1]);
    }
  } else {
    uint32_t r[(N + 1) / 2];
#pragma unroll
    for (int i = 0; i < N; i += 2) r[i / 2] = pack2<T>(v[i], v[i + 1]);
    if constexpr (N == 8)
      *reinterpret_cast<uint4 *>(p) = make_uint4(r[0], r[1], r[2], r[3]);
    else if constexpr (N == 4)
      *reinterpret_cast<uint2 *>(p) = make_uint2(r[0], r[1]);
    else
      *reinterpret_cast<uint32_t *>(p) = r[0];
  }
}

// A row is dim / (2 W) slots of W pairs, one per lane of a group of 2^log_g
// lanes: both halves' W elements (half layout) or 2 W neighbours (interleaved,
// and past rot in both).  A group takes kHeads neighbouring heads of one part
// of one token: their loads are all in flight together, with the lane's
// weights, cosines and sines, which they share.  Nothing is staged: partners sit
// in the same thread, and the norm is log_g shuffles.
// HBM-bound once the instructions are few: part, heads and batch come from the
// block's index (with one flat index, divided per thread, 212 instructions per
// 8 elements left the pass issue-bound: 4.8 TB/s), and products are packed
// pairs.  16384 tokens of 36 heads x 128, FP32 to FP16, cold L2: 80 us = 5.7
// TB/s with two heads per group (one: 92; four: 82; six: 94; 16 elements per
// lane and part: 80, but 104 against 88 with interleaved pairs).  FP16 to FP16:
// 74 us = 4.1 TB/s (one head: 90; four: 86; 16 elements: 84).
constexpr int kHeads = 2;
template <typename TI, typename TO, bool HALF, int W>
__global__ void __launch_bounds__(256) rope_vec_kernel(const __grid_constant__ RopeArgs a, int log_g) {
  constexpr int U = kHeads;
  grid_dependency_wait();
  const unsigned g = 1u << log_g, slot = threadIdx.x & (g - 1);
  // blocks: x tokens of one sequence, y a part's U heads, z the batch
  const unsigned i = blockIdx.x * (blockDim.x >> log_g) + (threadIdx.x >> log_g), b = blockIdx.z;
  if (i >= static_cast<unsigned>(a.seq)) return;  // whole groups; `mask` names the group alone
  const unsigned mask = g == 32 ? 0xffffffffu : ((1u << g) - 1) << ((threadIdx.x & 31) & ~(g - 1));
  const int per_q = (a.part[0].heads + U - 1) / U, per_k = (a.part[1].heads + U - 1) / U;
  int h0 = blockIdx.y;
  const int which = h0 < per_q ? 0 : h0 < per_q + per_k ? 1 : 2;
  h0 = (h0 - (which > 0 ? per_q : 0) - (which > 1 ? per_k : 0)) * U;
  const RopePart &p = a.part[which];
  const bool live = slot * 2 * W < static_cast<unsigned>(a.dim);
  const int rot = p.rotate ? a.rot : 0;
  const bool turns = slot * 2 * W < static_cast<unsigned>(rot);
  // offsets of the slot's two W-element parts
  const int o0 = HALF && turns ? W * slot : 2 * W * slot, o1 = HALF && turns ? rot / 2 + W * slot : o0 + W;

  const TI *in0 = static_cast<const TI *>(p.in) + b * p.in_stride[0] + i * p.in_stride[1] + h0 * p.in_stride[2];
  float x[U][2 * W], w[2 * W];
  float2 cs[W];
#pragma unroll
  for (int u = 0; u < U; ++u) {
#pragma unroll
    for (int e = 0; e < 2 * W; ++e) x[u][e] = 0.0f;
    const TI *in = in0 + u * p.in_stride[2];
    if (!live || h0 + u >= p.heads) continue;
    if (HALF) {
      load_n<TI, W>(in + o0, x[u]);
      load_n<TI, W>(in + o1, x[u] + W);
    } else {
      load_n<TI, 2 * W>(in + o0, x[u]);
    }
  }
  bool inside = true;
  if (rot) {
    const int pos = a.positions ? a.positions[static_cast<long long>(b) * a.seq + i] : static_cast<int>(i);
    inside = pos >= 0 && pos < a.table_rows;
    if (inside && turns) {
      const float4 *t = reinterpret_cast<const float4 *>(a.table + static_cast<long long>(pos) * (rot / 2) + W * slot);
#pragma unroll
      for (int e = 0; e < W; e += 2) {
        const float4 v = t[e / 2];
        cs[e] = make_float2(v.x, v.y), cs[e + 1] = make_float2(v.z, v.w);
      }
    }
  }
  if (p.weight && live) {
    load_n<float, W, false>(p.weight + o0, w);
    load_n<float, W, false>(p.weight + o1, w + W);
  }
  float2 cos2[W / 2], sin2[W / 2], neg2[W / 2];  // of two neighbouring pairs
#pragma unroll
  for (int e = 0; e < W / 2; ++e) {
    cos2[e] = make_float2(cs[2 * e].x, cs[2 * e + 1].x);
    sin2[e] = make_float2(cs[2 * e].y, cs[2 * e + 1].y);
    neg2[e] = make_float2(-sin2[e].x, -sin2[e].y);
  }
  TO *out = static_cast<TO *>(p.out) + b * p.out_stride[0] + i * p.out_stride[1] + h0 * p.out_stride[2];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    if (p.weight) {
      float2 sq = make_float2(0.0f, 0.0f);
#pragma unroll
      for (int e = 0; e < 2 * W; e += 2) {
        const float2 v = make_float2(x[u][e], x[u][e + 1]);
        sq = fma2(v, v, sq);
      }
      float sum = sq.x + sq.y;
      for (unsigned o = g / 2; o > 0; o >>= 1) sum += __shfl_xor_sync(mask, sum, o);
      const float inv = rsqrtf(fmaf(sum, a.inv_dim, a.eps));
#pragma unroll
      for (int e = 0; e < 2 * W; e += 2) {
        const float2 v = mul2(mul2(make_float2(x[u][e], x[u][e + 1]), make_float2(inv, inv)), make_float2(w[e], w[e + 1]));
        x[u][e] = v.x, x[u][e + 1] = v.y;
      }
    }
    if (!live || h0 + u >= p.heads) continue;
    if (turns) {
#pragma unroll
      for (int e = 0; e < W / 2; ++e) {
        const int e0 = HALF ? 2 * e : 4 * e, e1 = HALF ? 2 * e + 1 : 4 * e + 2;  // first elements of two pairs
        const int f0 = HALF ? W + e0 : e0 + 1, f1 = HALF ? W + e1 : e1 + 1;      // their second ones
        const float2 p0 = make_float2(x[u][e0], x[u][e1]), p1 = make_float2(x[u][f0], x[u][f1]);
        const float2 q0 = fma2(p1, neg2[e], mul2(p0, cos2[e])), q1 = fma2(p1, cos2[e], mul2(p0, sin2[e]));
        x[u][e0] = q0.x, x[u][e1] = q0.y, x[u][f0] = q1.x, x[u][f1] = q1.y;
      }
    }
    if (!inside) {
#pragma unroll
      for (int e = 0; e < 2 * W; ++e) x[u][e] = __int_as_float(0x7fffffff);
    }
    if (HALF) {
      store_n<TO, W>(out + u * p.out_stride[2] + o0, x[u]);
      store_n<TO, W>(out + u * p.out_stride[2] + o1, x[u] + W);
    } else {
      store_n<TO, 2 * W>(out + u * p.out_stride[2] + o0, x[u]);
    }
  }
}

// Whether every vector of the W-pair kernel is aligned, and a row fits one warp.
bool vectors_fit(const RopeArgs &a, int w, int in_bytes, int out_bytes) {
  if (a.dim % (2 * w) || a.rot % (2 * w) || a.dim / (2 * w) > 32) return false;
  const int elements = a.half ? w : 2 * w;
  const uintptr_t in_vec = std::min(16, elements * in_bytes), out_vec = std::min(16, elements * out_bytes);
  if (reinterpret_cast<uintptr_t>(a.table) % 16) return false;
  const int extent[3] = {a.batch, a.seq, 0};
  for (const RopePart &p : a.part) {
    if (!p.heads) continue;
    if (reinterpret_cast<uintptr_t>(p.in) % in_vec || reinterpret_cast<uintptr_t>(p.out) % out_vec ||
        reinterpret_cast<uintptr_t>(p.weight) % (4u * w))
      return false;
    for (int j = 0; j < 3; ++j)
      if ((j == 2 ? p.heads : extent[j]) > 1 && (p.in_stride[j] * in_bytes % static_cast<int64_t>(in_vec) ||
                                                 p.out_stride[j] * out_bytes % static_cast<int64_t>(out_vec)))
        return false;
  }
  return true;
}

template <typename TI, typename TO, int W>
cudaError_t launch_vectors(const RopeArgs &a, cudaStream_t st) {
  int log_g = 0;
  while ((2 * W << log_g) < a.dim) ++log_g;
  int y = 0;
  for (const RopePart &p : a.part) y += (p.heads + kHeads - 1) / kHeads;
  unsigned threads = 256;  // fewer where a sequence has fewer tokens
  while (threads > 32 && (threads >> 1 >> log_g) >= static_cast<unsigned>(a.seq)) threads >>= 1;
  const unsigned tokens = threads >> log_g;
  const dim3 grid((a.seq + tokens - 1) / tokens, y, a.batch);
  return a.half ? op_launch(rope_vec_kernel<TI, TO, true, W>, grid, threads, 0, st, a, log_g)
                : op_launch(rope_vec_kernel<TI, TO, false, W>, grid, threads, 0, st, a, log_g);
}

template <typename TI, typename TO>
cudaError_t launch_rope(const RopeArgs &a, int sms, cudaStream_t st) {
  const long long rows = static_cast<long long>(a.batch) * a.seq * a.heads;
  if (a.batch < 65536 && a.heads < 65536) {  // the grid's limits
    if (vectors_fit(a, 4, sizeof(TI), sizeof(TO))) return launch_vectors<TI, TO, 4>(a, st);
    if (vectors_fit(a, 2, sizeof(TI), sizeof(TO))) return launch_vectors<TI, TO, 2>(a, st);
  }
  const long long blocks = (rows + kRopeWarps - 1) / kRopeWarps;
  const unsigned grid = static_cast<unsigned>(blocks < 32LL * sms ? blocks : 32LL * sms);
  return op_launch(rope_row_kernel<TI, TO>, dim3(grid), kRopeWarps * 32, 0, st, a);
}

template <typename TI>
cudaError_t launch_rope_out(int out_type, const RopeArgs &a, int sms, cudaStream_t st) {
  if (out_type == HTPG_TYPE_F32) return launch_rope<TI, float>(a, sms, st);
  if (out_type == HTPG_TYPE_F16) return launch_rope<TI, __half>(a, sms, st);
  return launch_rope<TI, __nv_bfloat16>(a, sms, st);
}

}  // namespace
}  // namespace htpg

using namespace htpg;

extern "C" int htpg_rope_table(float *table, int rows, int rot_dim, const struct htpg_rope_scaling *s, void *stream) {
  if (!table || !s || rows < 0 || rot_dim < 2 || rot_dim % 2 || s->scaling < HTPG_ROPE_PLAIN ||
      s->scaling > HTPG_ROPE_YARN || !(s->base > 1.0) || !std::isfinite(s->base))
    return HTPG_EARGS;
  if (s->scaling != HTPG_ROPE_PLAIN && (!(s->factor >= 1.0) || !std::isfinite(s->factor))) return HTPG_EARGS;
  if (s->scaling == HTPG_ROPE_NTK && rot_dim <= 2) return HTPG_EARGS;
  if (reinterpret_cast<uintptr_t>(table) & 7u) return HTPG_ECONTROL;
  const int pairs = rot_dim / 2;
  double base = s->base, low = 0.0, high = 1.0, mult = 1.0;
  if (s->scaling == HTPG_ROPE_NTK) base *= std::pow(s->factor, static_cast<double>(rot_dim) / (rot_dim - 2));
  if (s->scaling == HTPG_ROPE_YARN) {
    if (s->original_rows < 1 || !(s->beta_fast > 0) || !(s->beta_slow > 0) || !(s->beta_fast >= s->beta_slow) ||
        !std::isfinite(s->beta_fast))
      return HTPG_EARGS;
    // pair i turns original_rows * base^(-i / pairs) / (2 pi) times over the trained context
    const double two_pi = 6.283185307179586;
    auto pair_of = [&](double turns) { return pairs * std::log(s->original_rows / (turns * two_pi)) / std::log(base); };
    low = std::fmax(std::floor(pair_of(s->beta_fast)), 0.0);
    high = std::fmin(std::ceil(pair_of(s->beta_slow)), rot_dim - 1.0);
    if (high <= low) high = low + 0.001;
    mult = 0.1 * std::log(s->factor) + 1.0;
  }
  if (rows == 0) return HTPG_OK;
  OpDevice d;
  const int rc = op_device(&d);
  if (rc) return rc;
  const long long n = static_cast<long long>(rows) * pairs;
  if ((n + 255) / 256 > 0x7fffffffLL) return HTPG_ECAPACITY;
  return op_result(op_launch(rope_table_kernel, dim3(static_cast<unsigned>((n + 255) / 256)), 256, 0,
                             static_cast<cudaStream_t>(stream), reinterpret_cast<float2 *>(table), rows, pairs, *s, base,
                             low, high, mult));
}

extern "C" int htpg_qkv_rope(const struct htpg_rope_params *p, void *q_out, void *k_out, void *v_out, const void *q,
                             const void *k, const void *v, const float *q_weight, const float *k_weight,
                             const float *table, const int32_t *positions, void *stream) {
  if (!p || !type_bytes(p->in_type) || !type_bytes(p->out_type) || p->batch < 0 || p->seq < 0 || p->reserved)
    return HTPG_EARGS;
  if (!q != !q_out || !k != !k_out || !v != !v_out || (!q && !k && !v)) return HTPG_EARGS;
  if ((q && p->q_heads < 1) || ((k || v) && p->kv_heads < 1) || p->head_dim < 1 || p->table_rows < 0) return HTPG_EARGS;
  if (p->rot_dim < 0 || p->rot_dim % 2 || (p->layout != HTPG_ROPE_INTERLEAVED && p->layout != HTPG_ROPE_HALF) ||
      !(p->eps >= 0.0f) || !std::isfinite(p->eps) || (p->rot_dim && !table && (q || k)))
    return HTPG_EARGS;
  if (p->head_dim > kRopeMaxDim || p->rot_dim > p->head_dim) return HTPG_ECAPACITY;
  if (p->q_heads > (1 << 20) || p->kv_heads > (1 << 20)) return HTPG_ECAPACITY;
  if (p->rot_dim && (q || k) && !positions && p->seq > p->table_rows) return HTPG_ECAPACITY;
  const uintptr_t in_bits = reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v);
  const uintptr_t out_bits =
      reinterpret_cast<uintptr_t>(q_out) | reinterpret_cast<uintptr_t>(k_out) | reinterpret_cast<uintptr_t>(v_out);
  const uintptr_t f32_bits = reinterpret_cast<uintptr_t>(q_weight) | reinterpret_cast<uintptr_t>(k_weight) |
                             reinterpret_cast<uintptr_t>(positions);
  if (in_bits % type_bytes(p->in_type) || out_bits % type_bytes(p->out_type) || f32_bits % 4 ||
      reinterpret_cast<uintptr_t>(table) % 8)
    return HTPG_ECONTROL;
  if (p->batch == 0 || p->seq == 0) return HTPG_OK;
  OpDevice d;
  const int rc = op_device(&d);
  if (rc) return rc;
  RopeArgs a = {};
  auto part = [&](int i, const void *in, void *out, const float *w, int heads, int rotate, const int64_t *is,
                  const int64_t *os) {
    if (!in) return;
    a.part[i].in = in;
    a.part[i].out = out;
    a.part[i].weight = w;
    a.part[i].heads = heads;
    a.part[i].rotate = rotate;
    for (int j = 0; j < 3; ++j) a.part[i].in_stride[j] = is[j], a.part[i].out_stride[j] = os[j];
    a.heads += heads;
  };
  part(0, q, q_out, q_weight, p->q_heads, 1, p->q_stride, p->q_out_stride);
  part(1, k, k_out, k_weight, p->kv_heads, 1, p->k_stride, p->k_out_stride);
  part(2, v, v_out, nullptr, p->kv_heads, 0, p->v_stride, p->v_out_stride);
  a.table = reinterpret_cast<const float2 *>(table);
  a.positions = positions;
  a.batch = p->batch;
  a.seq = p->seq;
  a.dim = p->head_dim;
  a.rot = p->rot_dim;
  a.half = p->layout == HTPG_ROPE_HALF;
  a.table_rows = p->table_rows;
  a.eps = p->eps;
  a.inv_dim = 1.0f / static_cast<float>(p->head_dim);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (p->in_type == HTPG_TYPE_F32) return op_result(launch_rope_out<float>(p->out_type, a, d.sms, st));
  if (p->in_type == HTPG_TYPE_F16) return op_result(launch_rope_out<__half>(p->out_type, a, d.sms, st));
  return op_result(launch_rope_out<__nv_bfloat16>(p->out_type, a, d.sms, st));
}
