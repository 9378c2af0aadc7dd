// Shared by the kernels on 4-bit weight matrices and the distillation loss: storage types, the code layout, checks.
#pragma once
#include "hyb_internal.h"
#include <hyacin_b200.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <utility>

namespace hyb {

// ---- storage types -------------------------------------------------------------------------------------------
inline bool is_w4_type(hyacinPrecision_t t) { return t == HYACIN_F32 || t == HYACIN_F16 || t == HYACIN_B200_BF16; }
inline size_t w4_type_bytes(hyacinPrecision_t t) { return t == HYACIN_F32 ? 4 : 2; }

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
template <class T> __device__ __forceinline__ T from_f32(float v);
template <> __device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <> __device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// Calls f(T{}) for the storage type of t.
template <class F> void with_w4_type(hyacinPrecision_t t, F&& f) {
  if (t == HYACIN_F32) f(float{});
  else if (t == HYACIN_F16) f(__half{});
  else f(__nv_bfloat16{});
}

// ---- code layout ---------------------------------------------------------------------------------------------
// A block of 128 rows is sixteen words; word w = 4 c + i holds rows 32 i + 8 c .. + 7, row 2 p + h of these eight in nibble
// p + 4 h.  A 16-byte quarter c then carries eight rows of each 32-row subset i, and the nibbles (p, p + 4), which one
// mask extracts into the two halves of a register, are neighbouring rows.
constexpr int kW4Block = 128;
__host__ __device__ inline int w4_word_row(int word) { return 32 * (word & 3) + 8 * (word >> 2); }     // within the block
__host__ __device__ inline int w4_nibble_row(int nibble) { return 2 * (nibble & 3) + (nibble >> 2); }  // within the word
__host__ __device__ inline int w4_row_nibble(int row8) { return (row8 >> 1) + 4 * (row8 & 1); }

// Segments of a column of m rows.  The sum before the division passes 2^31 when seg is near its upper end ("one scale per column").
__host__ __device__ inline int w4_segments(int m, int seg) { return int((int64_t(m) + seg - 1) / seg); }

// ---- argument checks -----------------------------------------------------------------------------------------
inline int32_t w4_refuse(const char* fn, const char* why) {
  std::fprintf(stderr, "hyacin-b200: %s: %s\n", fn, why);
  return -1;
}
// Pointers lie on a boundary of their type's size: the kernels' loads would fault otherwise.
inline bool w4_on_boundary(const void* p, size_t bytes) { return reinterpret_cast<uintptr_t>(p) % bytes == 0; }
template <class... P> bool w4_on_boundary(size_t bytes, P... p) { return (w4_on_boundary(static_cast<const void*>(p), bytes) && ...); }
// The handle's device must be the current one: launches would otherwise go to the wrong GPU.  A zero-initialised handle names device 0,
// but has neither its number of SMs, by which grids are divided, nor a pool.
inline int32_t w4_refuse_handle(const char* fn, const hyacinHandle_t* handle) {
  int device = -1;
  if (cudaGetDevice(&device) != cudaSuccess || device != handle->DeviceID) return w4_refuse(fn, "the handle belongs to another device than the current one");
  if (handle->DeviceSMs < 1 || !handle->mempool) return w4_refuse(fn, "the handle has not been through hyacinCreate");
  return 0;
}
// A launch that returns its own error: the thread's last one may be of an earlier, unrelated call.
template <class... P, class... A> cudaError_t w4_start(void (*kernel)(P...), dim3 grid, unsigned threads, size_t smem, cudaStream_t stream, A&&... args) {
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = grid; cfg.blockDim = dim3(threads); cfg.dynamicSmemBytes = smem; cfg.stream = stream;
  return cudaLaunchKernelEx(&cfg, kernel, std::forward<A>(args)...);
}
// The return value of an entry point.  An error that is reported here is not left for the next call that asks for the thread's last one.
inline int32_t w4_result(cudaError_t e, const char* what) {
  if (e == cudaSuccess) return 0;
  report_cuda_error(e, what, __FILE__, __LINE__);
  cudaGetLastError();
  return -3;
}

}  // namespace hyb
