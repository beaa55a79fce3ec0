// Low-rank adapters of many requests beside a shared projection:
//
//   out_i = base_i + scale_s (x_i A_s^T) B_s^T,  s = the adapter of row i.
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

constexpr int kLoraThreads = 256;

// One block per row: the rank's dot products by its warps, then the columns.
template <typename T>
__global__ void __launch_bounds__(kLoraThreads) lora_row_kernel(LoraArgs p) {
  __shared__ float t[kLoraMaxRank];
  grid_dependency_wait();
  const int row = blockIdx.x, lane = threadIdx.x & 31;
  const int s = p.ids[row];
  const int rank = s >= 0 && s < p.adapters ? min(max(p.ranks[s], 0), p.max_rank) : 0;
  const float *x = p.x + row * p.ldx;
  const T *a = static_cast<const T *>(p.a) + (rank ? static_cast<long long>(s) * p.max_rank * p.k : 0);
  const T *b = static_cast<const T *>(p.b) + (rank ? static_cast<long long>(s) * p.n * p.max_rank : 0);
  for (int r = threadIdx.x >> 5; r < rank; r += kLoraThreads / 32) {
    float sum = 0.0f;
    for (int c = lane; c < p.k; c += 32) sum += x[c] * to_f32(a[static_cast<long long>(r) * p.k + c]);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    if (lane == 0) t[r] = sum * p.scales[s];
  }
  __syncthreads();
  for (int c = threadIdx.x; c < p.n; c += kLoraThreads) {
    float v = 0.0f;
    for (int r = 0; r < rank; ++r) v += t[r] * to_f32(b[static_cast<long long>(c) * p.max_rank + r]);
    p.out[row * p.ldo + c] = (p.base ? p.base[row * p.ldb + c] : 0.0f) + v;
  }
}

template <typename T>
cudaError_t launch_lora(const LoraArgs &p, cudaStream_t st) {
  return op_launch(lora_row_kernel<T>, dim3(p.m), kLoraThreads, 0, st, p);
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
  return op_result(p->type == HTPG_TYPE_F16 ? launch_lora<__half>(r, st) : launch_lora<__nv_bfloat16>(r, st));
}
