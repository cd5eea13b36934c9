// gg_ops.h -- what the device-memory operators (gg_ops.cu, gg_kv8.cu) share: error messages,
// checks of streams and views, and loads of rows of any of the three element types.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "../../include/gemma_b200.h"
#include "gg_device.cuh"
#include "gg_launch.h"

#include <atomic>

// Keeps the message for gg_last_error(NULL) and returns `code`.
int ops_fail(int code, const char* fmt, ...);
// GG_OK if `stream` belongs to the current device (NULL does).
int ops_check_stream(const char* fn, cudaStream_t s);
// GG_OK if the view is usable for `rows` rows of head_dim values.
int ops_check_rows(const char* fn, const char* name, const gg_rows* v, int rows, int head_dim);
int ops_check_cache(const char* fn, const gg_kv8_cache* c);
// gg_kv8_attention whose waits are bounded by timeout_ns; one that runs out sets GG_ERR_WAIT_MBAR in *err
// (device memory, or NULL) and leaves NaN in the rows concerned.
int kv8_attention_bounded(const gg_kv8_cache* c, const gg_kv8_attention_call* call, cudaStream_t s, uint32_t* err, uint64_t timeout_ns);
constexpr uint64_t KV8_TIMEOUT_NS = 2000000000ull;  // of gg_kv8_attention

inline int ops_type_bytes(int type) { return type == GG_T_F32 ? 4 : 2; }
// Every head of the view starts on a 16-byte boundary.
inline bool ops_aligned16(const gg_rows& v) {
  const int64_t es = ops_type_bytes(v.type);
  return ((uintptr_t)v.data & 15) == 0 && (v.row_stride * es) % 16 == 0 && (v.heads == 1 || (v.head_stride * es) % 16 == 0);
}

namespace gg {

// launch_pdl of a kernel that needs more dynamic shared memory than the default limit. The limit is
// raised on the kernel's first launch on a device, and again when a launch is refused: a context made
// after cudaDeviceReset has forgotten it.
template <auto Kernel, typename... Args>
inline cudaError_t launch_big_smem(dim3 grid, dim3 block, size_t smem, cudaStream_t s, const Args&... args) {
  static std::atomic<uint64_t> raised;  // devices, by bit
  int dev = 0;
  cudaError_t r = cudaGetDevice(&dev);
  if (r != cudaSuccess) return r;
  const uint64_t bit = dev < 64 ? 1ull << dev : 0;
  if (raised.load(std::memory_order_acquire) & bit) {
    r = launch_pdl(Kernel, grid, block, smem, s, args...);
    if (r != cudaErrorInvalidValue) return r;
    cudaGetLastError();
  }
  r = cudaFuncSetAttribute(Kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
  if (r != cudaSuccess) return r;
  raised.fetch_or(bit, std::memory_order_acq_rel);
  return launch_pdl(Kernel, grid, block, smem, s, args...);
}

GG_DEV float to_f32(float v) { return v; }
GG_DEV float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
GG_DEV float to_f32(__half v) { return __half2float(v); }
template <class T> GG_DEV T from_f32(float v);
template <> GG_DEV float from_f32<float>(float v) { return v; }
template <> GG_DEV __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <> GG_DEV __half from_f32<__half>(float v) { return __float2half_rn(v); }

// N elements next to each other, widened; vec: p is aligned to the N elements (16 bytes at least).
template <class T, int N, bool VEC>
GG_DEV void load_row(const T* p, float (&v)[N]) {
  if constexpr (VEC) {
    constexpr int W = N * (int)sizeof(T) / 16;
    static_assert(W >= 1 && N * sizeof(T) % 16 == 0, "whole 16-byte words");
    uint4 w[W];
#pragma unroll
    for (int i = 0; i < W; i++) w[i] = reinterpret_cast<const uint4*>(p)[i];
    const T* e = reinterpret_cast<const T*>(w);
#pragma unroll
    for (int i = 0; i < N; i++) v[i] = to_f32(e[i]);
  } else {
#pragma unroll
    for (int i = 0; i < N; i++) v[i] = to_f32(p[i]);
  }
}
template <class T, int N, bool VEC>
GG_DEV void store_row(T* p, const float (&v)[N]) {
  if constexpr (VEC) {
    constexpr int W = N * (int)sizeof(T) / 16;
    uint4 w[W];
    T* e = reinterpret_cast<T*>(w);
#pragma unroll
    for (int i = 0; i < N; i++) e[i] = from_f32<T>(v[i]);
#pragma unroll
    for (int i = 0; i < W; i++) reinterpret_cast<uint4*>(p)[i] = w[i];
  } else {
#pragma unroll
    for (int i = 0; i < N; i++) p[i] = from_f32<T>(v[i]);
  }
}

}  // namespace gg
