// Attention over an encoder's states:
//
//   out_i = sum_j w_ij v_j / sum_j w_ij,  w_ij = exp(scale q_i . k_j + bias_j)
//
// in one pass over the keys with the running maximum and sum of the softmax.
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

constexpr int kRowWarps = 8;

// One warp per query row: lanes split the head, every key is one dot product.
template <typename T, typename TO>
__global__ void __launch_bounds__(kRowWarps * 32) attn_row_kernel(AttnArgs a) {
  grid_dependency_wait();
  const int lane = threadIdx.x & 31;
  const long long rows = static_cast<long long>(a.batch) * a.q_heads * a.q_len;
  constexpr int kPer = kAttnMaxDim / 32;
  for (long long r = static_cast<long long>(blockIdx.x) * kRowWarps + (threadIdx.x >> 5); r < rows;
       r += static_cast<long long>(gridDim.x) * kRowWarps) {
    const long long i = r % a.q_len, h = r / a.q_len % a.q_heads, b = r / a.q_len / a.q_heads;
    const T *q = static_cast<const T *>(a.q) + b * a.qs[0] + i * a.qs[1] + h * a.qs[2];
    const T *k = static_cast<const T *>(a.k) + b * a.ks[0] + h / a.group * a.ks[2];
    const T *v = static_cast<const T *>(a.v) + b * a.vs[0] + h / a.group * a.vs[2];
    const int n = a.lens ? min(max(a.lens[b], 0), a.kv_len) : a.kv_len;
    float qr[kPer], o[kPer];
#pragma unroll
    for (int j = 0; j < kPer; ++j) {
      const int d = lane + 32 * j;
      qr[j] = d < a.dim ? to_f32(q[d]) : 0.0f;
      o[j] = 0.0f;
    }
    float top = -INFINITY, sum = 0.0f;
    for (int t = 0; t < n; ++t) {
      const float add = a.bias ? a.bias[b * a.bias_stride + t] : 0.0f;
      if (add == -INFINITY) continue;
      float s = 0.0f;
#pragma unroll
      for (int j = 0; j < kPer; ++j) {
        const int d = lane + 32 * j;
        if (d < a.dim) s += qr[j] * to_f32(k[t * a.ks[1] + d]);
      }
#pragma unroll
      for (int w = 16; w > 0; w >>= 1) s += __shfl_xor_sync(0xffffffffu, s, w);
      s = s * a.scale + add;
      const float m = fmaxf(top, s);
      const float keep = m == top ? 1.0f : expf(top - m), p = expf(s - (m == -INFINITY ? 0.0f : m));
      top = m;
      sum = sum * keep + p;
#pragma unroll
      for (int j = 0; j < kPer; ++j) {
        const int d = lane + 32 * j;
        if (d < a.dim) o[j] = o[j] * keep + p * to_f32(v[t * a.vs[1] + d]);
      }
    }
    TO *out = static_cast<TO *>(a.out) + b * a.os[0] + i * a.os[1] + h * a.os[2];
#pragma unroll
    for (int j = 0; j < kPer; ++j) {
      const int d = lane + 32 * j;
      if (d < a.dim) out[d] = from_f32<TO>(sum == 0.0f ? 0.0f : o[j] / sum);
    }
  }
}

template <typename T, typename TO>
cudaError_t launch_attn(const AttnArgs &a, int sms, cudaStream_t st) {
  const long long rows = static_cast<long long>(a.batch) * a.q_heads * a.q_len;
  const long long blocks = (rows + kRowWarps - 1) / kRowWarps;
  const unsigned grid = static_cast<unsigned>(blocks < 64LL * sms ? blocks : 64LL * sms);
  return op_launch(attn_row_kernel<T, TO>, dim3(grid), kRowWarps * 32, 0, st, a);
}

// 16-byte vectors along every dimension that is stepped along.
bool strides_fit(const int64_t *s, const int (&extent)[3], int per16) {
  for (int i = 0; i < 3; ++i)
    if (extent[i] > 1 && s[i] % per16) return false;
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
  if (p->batch == 0 || p->q_len == 0) return HTPG_OK;
  if (!out || !q || (p->kv_len && (!k || !v))) return HTPG_EARGS;
  const int qe[3] = {p->batch, p->q_len, p->q_heads}, ke[3] = {p->batch, p->kv_len, p->kv_heads};
  if (((reinterpret_cast<uintptr_t>(out) | reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(k) |
        reinterpret_cast<uintptr_t>(v)) & 15u) ||
      ((reinterpret_cast<uintptr_t>(kv_lens) | reinterpret_cast<uintptr_t>(key_bias)) & 3u) ||
      !strides_fit(p->q_stride, qe, 8) || !strides_fit(p->k_stride, ke, 8) || !strides_fit(p->v_stride, ke, 8) ||
      !strides_fit(p->out_stride, qe, 16 / type_bytes(p->out_type)))
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
  cudaError_t e;
  if (p->type == HTPG_TYPE_F16)
    e = p->out_type == HTPG_TYPE_F32 ? launch_attn<__half, float>(a, d.sms, st) : launch_attn<__half, __half>(a, d.sms, st);
  else
    e = p->out_type == HTPG_TYPE_F32 ? launch_attn<__nv_bfloat16, float>(a, d.sms, st)
                                     : launch_attn<__nv_bfloat16, __nv_bfloat16>(a, d.sms, st);
  return op_result(e);
}
