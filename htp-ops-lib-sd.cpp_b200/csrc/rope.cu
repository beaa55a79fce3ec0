// Per-head RMS norm and rotary positions of projected queries and keys, with
// the conversion of the values in the same pass, and the table of cosines and
// sines they use.
//
//   y = x rsqrt(mean(x^2) + eps) w;   (a', b') = (a cos - b sin, a sin + b cos)
//
// Every element is read and written once and does some ten operations, so the
// pass is bound by HBM: (in + out) bytes per element.
#include <cmath>
#include <new>

#include "ops.h"
#include "ptx.cuh"

namespace htpg {
namespace {

// ---------------------------------------------------------------- the table
// One thread per (position, pair).  Angles in FP64: at position 2^17 an FP32
// angle is off by up to 2^-8 rad, an FP64 one by 2^-37; the values are rounded once.
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
  float eps;
};

constexpr int kRopeWarps = 8, kRopeMaxDim = 512;

// One warp per (token, head) row, the row staged in shared memory as FP32.
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
      const float2 *cs = a.table + (ok ? pos : 0) * (rot / 2);
      for (int j = lane; j < rot / 2; j += 32) {
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

template <typename TI, typename TO>
cudaError_t launch_rope(const RopeArgs &a, int sms, cudaStream_t st) {
  const long long rows = static_cast<long long>(a.batch) * a.seq * a.heads;
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
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (p->in_type == HTPG_TYPE_F32) return op_result(launch_rope_out<float>(p->out_type, a, d.sms, st));
  if (p->in_type == HTPG_TYPE_F16) return op_result(launch_rope_out<__half>(p->out_type, a, d.sms, st));
  return op_result(launch_rope_out<__nv_bfloat16>(p->out_type, a, d.sms, st));
}
