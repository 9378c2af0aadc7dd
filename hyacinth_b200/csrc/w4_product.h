// Interfaces between the kernels of hyacinB200ProductW4.
#pragma once
#include "w4.cuh"
#include <cuda.h>

namespace hyb {

struct ProductArgs {
  const uint8_t* codes; int64_t ldq; int m, n, t, seg;
  const void* scales; const uint8_t* zeros; int64_t lds;
  const void* x; int64_t ldx;
  // correction: second (outputs x rank) times mid = first^T x (rank x t)
  int rank; const void* first; int64_t ld1; const void* second; int64_t ld2;
  void* y; int64_t ldy;
};

// The descriptor of a tensor map, a kernel's argument, on its way before the first copy needs it.
__device__ __forceinline__ void prefetch_map(const CUtensorMap* map) { asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(map)) : "memory"); }

// Fifth-generation tensor cores, 16-bit types, both directions.  Returns 0 or -3.
int32_t launch_product_umma(const hyacinHandle_t* handle, const char* fn, bool trans, hyacinPrecision_t type, const ProductArgs& a);

// mid(k, t) = sum_r first(r, k) x(r, t) in single precision, [t][k], for the 16-bit types.
cudaError_t launch_mid_float(const hyacinHandle_t* handle, hyacinPrecision_t type, const void* first, int64_t ld1, int rows, int rank, const void* x, int64_t ldx, int t, float* mid, bool aligned);
// Few vectors, opW 'T', all types, any number of passes over W; product_stream_vectors: vectors per pass (0: not even one fits).
int product_stream_vectors(hyacinPrecision_t type, const ProductArgs& a);
int32_t launch_product_stream(const hyacinHandle_t* handle, const char* fn, hyacinPrecision_t type, const ProductArgs& a);

// Single precision, both directions, any size.
int32_t launch_product_single(const hyacinHandle_t* handle, const char* fn, bool trans, const ProductArgs& a);

}  // namespace hyb
