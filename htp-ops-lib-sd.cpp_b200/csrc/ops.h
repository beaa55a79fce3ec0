// Shared by the transformer-block operators (rope.cu, attention.cu, lora.cu):
// the library's device state, stream scratch and launches, and element types.
// Internal to libhtp_ops_b200.so.
#pragma once

#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <cstdint>
#include <mutex>
#include <type_traits>

#include "../../include/htp_ops_b200.h"
#include "kernels.h"
#include "ptx.cuh"

namespace htpg {

// ---- device state (capi.cu)
struct OpDevice {
  int sms = 0;
  uint32_t *watchdog = nullptr;
};
// The current device, initialised when this is its first use.
int op_device(OpDevice *d);
// Text for htpg_last_cuda_error; HTPG_OK or HTPG_ELAUNCH.
int op_result(cudaError_t e);
// The library's lock: held from op_scratch to the launch that uses the scratch,
// so that no other host thread grows (moves) it in between.
std::unique_lock<std::mutex> op_lock();
// Scratch of one stream: `bytes` of it, preceded by kOpCounters zero words that
// every launch leaves zero.  Grows when a larger call arrives and is kept
// otherwise.  While the stream is being captured it is the graph's own, so that
// graphs run beside each other and beside the stream; with the graph and its
// executables it goes to the next user.  Called with op_lock() held.
constexpr int kOpCounters = 16384;
int op_scratch(cudaStream_t st, size_t bytes, uint32_t **counters, uint8_t **scratch);
// Tensor map of an array (any HTPG_TYPE_*) of `rank` <= 5 dimensions (innermost first;
// strides in bytes of dimensions 1 .. rank - 1), zero fill, 128-byte swizzle.
int op_tensor_map(CUtensorMap *map, int type, const void *base, int rank, const uint64_t *dims, const uint64_t *strides,
                  const uint32_t *box);

// Launch as a programmatic dependent: the kernel waits (grid_dependency_wait)
// before it touches memory, so only its set-up overlaps the kernel before it.
template <typename... P, typename... A>
cudaError_t op_launch(void (*fn)(P...), dim3 grid, unsigned block, size_t smem, cudaStream_t st, A... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(block, 1, 1);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return counted(cudaLaunchKernelEx(&cfg, fn, static_cast<P>(args)...));
}

// Extents up to this one can be rounded up to tiles, and passed by a step, in 32 bits.
constexpr int kOpMaxExtent = 1 << 30;

// ---- element types
inline int type_bytes(int type) {
  return type == HTPG_TYPE_F32 ? 4 : type == HTPG_TYPE_F16 || type == HTPG_TYPE_BF16 ? 2 : 0;
}

template <typename T>
__device__ __forceinline__ float to_f32(T v) {
  if constexpr (sizeof(T) == 4)
    return v;
  else if constexpr (std::is_same<T, __half>::value)
    return __half2float(v);
  else
    return __bfloat162float(v);
}
// Round to nearest even.
template <typename T>
__device__ __forceinline__ T from_f32(float v) {
  if constexpr (sizeof(T) == 4)
    return v;
  else if constexpr (std::is_same<T, __half>::value)
    return __float2half_rn(v);
  else
    return __float2bfloat16_rn(v);
}

// Two FP32 values as one 16-bit pair (the first in the low half), to nearest even.
template <typename T>
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
  uint32_t r;
  if constexpr (std::is_same<T, __half>::value)
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  else
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}
template <typename T>
__device__ __forceinline__ float2 unpack2(uint32_t v) {
  if constexpr (std::is_same<T, __half>::value) return __half22float2(*reinterpret_cast<const __half2 *>(&v));
  return make_float2(__uint_as_float(v << 16), __uint_as_float(v & 0xffff0000u));
}

// ---- packed pairs of FP32 values (one instruction for both)
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
  unsigned long long r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(reinterpret_cast<const unsigned long long &>(a)), "l"(reinterpret_cast<const unsigned long long &>(b)));
  return reinterpret_cast<float2 &>(r);
}
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
  unsigned long long r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(reinterpret_cast<const unsigned long long &>(a)), "l"(reinterpret_cast<const unsigned long long &>(b)));
  return reinterpret_cast<float2 &>(r);
}
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  unsigned long long r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(reinterpret_cast<const unsigned long long &>(a)), "l"(reinterpret_cast<const unsigned long long &>(b)), "l"(reinterpret_cast<const unsigned long long &>(c)));
  return reinterpret_cast<float2 &>(r);
}

// ---- asynchronous copies and 16-bit products
// 16 bytes to shared memory, zeros where `in` is false (src is not read then).
__device__ __forceinline__ void copy16(void *dst, const void *src, bool in) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 16, %2;" ::"r"(smem_u32(dst)), "l"(src), "r"(in ? 16 : 0) : "memory");
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copy_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

// C += A B, m16n8k16, FP32 sums.
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

}  // namespace htpg
