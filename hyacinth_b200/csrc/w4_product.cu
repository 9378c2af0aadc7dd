// Products of a few vectors with a 4-bit weight matrix, Y = Wq^T X + V (U^T X) and Y = Wq X + U (V^T X), with
// Wq(r, j) = s(j, r / segM) (q(r, j) - zero(j, r / segM)).
#include "w4_product.h"
#include <algorithm>

namespace hyb {
namespace {

struct PlainArgs : ProductArgs { const float* mid = nullptr; };

// y += sum_k second(row, k) mid(k, token)
template <class T> __device__ __forceinline__ float add_correction(const PlainArgs& a, float y, int row, int token) {
  const T* f = static_cast<const T*>(a.second) + row;
  const float* m = a.mid + int64_t(token) * a.rank;
  for (int k = 0; k < a.rank; ++k) y += to_f32(f[k * a.ld2]) * m[k];
  return y;
}

// mid(k, token) = sum_r first(r, k) x(r, token): one warp per entry.
template <class T> __global__ void __launch_bounds__(256) correction_mid_kernel(const T* first, int64_t ld1, int rows, int rank, const T* x, int64_t ldx, int t, float* mid) {
  const int64_t task = int64_t(blockIdx.x) * 8 + (threadIdx.x >> 5);
  if (task >= int64_t(rank) * t) return;
  const int lane = threadIdx.x & 31, k = int(task % rank), token = int(task / rank);
  float s = 0.f;
  for (int r = lane; r < rows; r += 32) s += to_f32(first[k * ld1 + r]) * to_f32(x[token * ldx + r]);
  for (int d = 16; d; d >>= 1) s += __shfl_xor_sync(~0u, s, d);
  if (lane == 0) mid[task] = s;
}

constexpr int kPlainTokens = 4;

// op 'T', plain: one warp per column, the lanes share its words.  For single-precision x too long for the streaming kernel's shared memory
// (more than about 20 000 rows) and for sums over nothing.
template <class T> __global__ void __launch_bounds__(256) product_t_plain_kernel(PlainArgs a) {
  const int lane = threadIdx.x & 31, col = blockIdx.x * 8 + (threadIdx.x >> 5);
  if (col >= a.n) return;
  const T* x = static_cast<const T*>(a.x);
  const T* scales = static_cast<const T*>(a.scales) + col * a.lds;
  const int words = (a.m + kW4Block - 1) / kW4Block * 16;
  for (int64_t t0 = int64_t(blockIdx.y) * kPlainTokens; t0 < a.t; t0 += int64_t(gridDim.y) * kPlainTokens) {
    float acc[kPlainTokens] = {};
    for (int w = lane; w < words; w += 32) {
      const int row = w / 16 * kW4Block + w4_word_row(w & 15);
      if (row >= a.m) continue;
      const uint32_t word = *reinterpret_cast<const uint32_t*>(a.codes + col * a.ldq + int64_t(w) * 4);
      const int seg = row / a.seg;
      const float s = to_f32(scales[seg]); const int zero = a.zeros ? a.zeros[col * a.lds + seg] : 8;
      for (int e = 0; e < 8 && row + e < a.m; ++e) {
        const float v = s * float(int((word >> (4 * w4_row_nibble(e))) & 15u) - zero);
        for (int t = 0; t < kPlainTokens; ++t) if (t0 + t < a.t) acc[t] += v * to_f32(x[(t0 + t) * a.ldx + row + e]);
      }
    }
    for (int t = 0; t < kPlainTokens; ++t) {
      for (int d = 16; d; d >>= 1) acc[t] += __shfl_xor_sync(~0u, acc[t], d);
      if (lane == 0 && t0 + t < a.t) static_cast<T*>(a.y)[(t0 + t) * a.ldy + col] = from_f32<T>(add_correction<T>(a, acc[t], col, int(t0 + t)));
    }
  }
}

// op 'N' in single precision (and for 16-bit types when there is nothing to sum): a block of 256 threads takes 128 rows, thread (word,
// lane) the eight rows of a word in every 16th column, for four vectors at a time; x times the scale is formed once per word.
// A cluster of up to eight such blocks splits the columns; sums meet in shared memory, in a fixed order.
// Bound: the floating-point pipe, 8 conversions and 32 multiply-adds per word and four vectors; 4096 x 4096, four vectors: 24 us.
constexpr int kSingleLanes = 16, kSingleThreads = 16 * kSingleLanes;
__device__ __forceinline__ float ld_cluster(const float* at, uint32_t rank) {
  uint32_t remote; float v;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(remote) : "r"(uint32_t(__cvta_generic_to_shared(at))), "r"(rank));
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(remote) : "memory");
  return v;
}
__device__ __forceinline__ void cluster_sync_all() {
  asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
  asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}
template <class T> __global__ void __launch_bounds__(kSingleThreads) product_n_single_kernel(PlainArgs a, int splits) {
  __shared__ float red[kPlainTokens][8][16][kSingleLanes + 1], sum[kPlainTokens][kW4Block];
  const int word = threadIdx.x & 15, lane = threadIdx.x >> 4, split = blockIdx.x % splits, block = blockIdx.x / splits;
  const int row = block * kW4Block + w4_word_row(word), seg = min(row, a.m - 1) / a.seg;
  const int j0 = int(int64_t(a.n) * split / splits), j1 = int(int64_t(a.n) * (split + 1) / splits);
  const T* x = static_cast<const T*>(a.x);
  const T* scales = static_cast<const T*>(a.scales) + seg;
  const uint8_t* zeros = a.zeros ? a.zeros + seg : nullptr;
  const uint8_t* codes = a.codes + int64_t(block) * 64 + word * 4;
  for (int64_t t0 = int64_t(blockIdx.y) * kPlainTokens; t0 < a.t; t0 += int64_t(gridDim.y) * kPlainTokens) {
    float acc[kPlainTokens][8] = {};
#pragma unroll 4
    for (int j = j0 + lane; j < j1; j += kSingleLanes) {
      const uint32_t q = __ldg(reinterpret_cast<const uint32_t*>(codes + j * a.ldq));
      const float s = to_f32(scales[j * a.lds]), offset = 8388608.f + float(zeros ? int(zeros[j * a.lds]) : 8);
      float xs[kPlainTokens], w[8];
#pragma unroll
      for (int t = 0; t < kPlainTokens; ++t) xs[t] = t0 + t < a.t ? s * to_f32(x[(t0 + t) * a.ldx + j]) : 0.f;
#pragma unroll
      for (int e = 0; e < 8; ++e) w[e] = __uint_as_float(((q >> (4 * w4_row_nibble(e))) & 15u) | 0x4b000000u) - offset;      // 2^23 + q, exact
#pragma unroll
      for (int t = 0; t < kPlainTokens; ++t)
#pragma unroll
        for (int e = 0; e < 8; ++e) acc[t][e] += w[e] * xs[t];
    }
#pragma unroll
    for (int t = 0; t < kPlainTokens; ++t)
#pragma unroll
      for (int e = 0; e < 8; ++e) red[t][e][word][lane] = acc[t][e];
    __syncthreads();
    for (int i = threadIdx.x; i < kPlainTokens * kW4Block; i += kSingleThreads) {
      const int t = i / kW4Block, r = i % kW4Block, e = r & 7, w = r >> 3;
      float v = 0.f;
#pragma unroll
      for (int l = 0; l < kSingleLanes; ++l) v += red[t][e][w][l];
      sum[t][w4_word_row(w) + e] = v;
    }
    if (splits > 1) cluster_sync_all(); else __syncthreads();
    const int share = kW4Block / splits;
    for (int i = threadIdx.x; i < kPlainTokens * share; i += kSingleThreads) {
      const int t = i / share, local = split * share + i % share, out = block * kW4Block + local;
      if (out >= a.m || t0 + t >= a.t) continue;
      float v = 0.f;
      for (int c = 0; c < splits; ++c) v += splits > 1 ? ld_cluster(&sum[t][local], c) : sum[t][local];
      static_cast<T*>(a.y)[(t0 + t) * a.ldy + out] = from_f32<T>(add_correction<T>(a, v, out, int(t0 + t)));
    }
    if (splits > 1) cluster_sync_all(); else __syncthreads();
  }
}

}  // namespace
}  // namespace hyb

extern "C" int32_t hyacinB200ProductW4(const hyacinHandle_t* handle, char opW, int32_t M, int32_t N, int32_t T, hyacinPrecision_t Xtype,
                                       const uint8_t* codes, int64_t ldq, int32_t segM, const void* scales, const uint8_t* zeros,
                                       int32_t lds, const void* X, int32_t ldx, int32_t rank, const void* U, int32_t ldu, const void* V,
                                       int32_t ldv, void* Y, int32_t ldy) {
  using namespace hyb;
  const char* fn = "hyacinB200ProductW4";
  if (!handle) return w4_refuse(fn, "no handle");
  const bool trans = opW == 'T' || opW == 't';
  if (!trans && opW != 'N' && opW != 'n') return w4_refuse(fn, "opW must be 'T' or 'N'");
  if (!is_w4_type(Xtype)) return w4_refuse(fn, "type not supported");
  if (M < 0 || N < 0 || T < 0 || rank < 0 || segM <= 0 || segM % 32) return w4_refuse(fn, "sizes: M, N, T, rank >= 0 and segM a positive multiple of 32");
  if (M > 0x7fffff00 || N > 0x7fffff00 || T > 0x7fffff00) return w4_refuse(fn, "sizes: M, N, T at most 2^31 - 256");
  if (rank > 1 << 20) return w4_refuse(fn, "rank: at most 2^20");
  const int in = trans ? M : N, out = trans ? N : M;
  if (T == 0 || out == 0) return 0;
  if (!Y || ldy < out) return w4_refuse(fn, "Y: null or leading dimension too small");
  if (in > 0) {
    if (!X || ldx < in) return w4_refuse(fn, "X: null or leading dimension too small");
    if (!codes || !scales) return w4_refuse(fn, "null pointer");
    if (lds < (int64_t(M) + segM - 1) / segM) return w4_refuse(fn, "lds too small");
    if (ldq % 16 || ldq < (int64_t(M) + 127) / 128 * 64 || reinterpret_cast<uintptr_t>(codes) % 16) return w4_refuse(fn, "codes: 16-byte aligned, ldq a multiple of 16 and at least 64 ceil(M / 128)");
    if (rank > 0 && (!U || !V || ldu < M || ldv < N)) return w4_refuse(fn, "U, V: null or leading dimension too small");
  }
  if (!w4_on_boundary(w4_type_bytes(Xtype), Y) || (in > 0 && !w4_on_boundary(w4_type_bytes(Xtype), X, scales)) || (in > 0 && rank > 0 && !w4_on_boundary(w4_type_bytes(Xtype), U, V)))
    return w4_refuse(fn, "a pointer that is not on a boundary of its type");
  if (!w4_device_ok(handle)) return w4_refuse(fn, "the handle belongs to another device than the current one");
  cudaStream_t stream = handle->cudaStream;
  PlainArgs a;
  static_cast<ProductArgs&>(a) = ProductArgs{codes, ldq, M, N, T, segM, scales, zeros, lds, X, ldx, in > 0 ? rank : 0,
                                             trans ? U : V, trans ? ldu : ldv, trans ? V : U, trans ? ldv : ldu, Y, ldy};
  timer_mark(handle, Segment::Replicated);
  if (in > 0 && trans) {
    const int per = product_stream_vectors(Xtype, a);
    // Up to eight vectors stream (17 against 23 us, 4096 x 16384); up to sixteen where the tensor-core kernel cannot fetch a block's
    // scales at once (24 against 58 us, 5001 x 6003, segments of 32 rows, odd table pitch).
    const bool scattered = segM % 128 != 0 && (segM == 96 || lds % (128 / std::min(segM, 64)) != 0 || reinterpret_cast<uintptr_t>(scales) % (256 / std::min(segM, 64)) != 0);
    if (per > 0 && (Xtype == HYACIN_F32 || (per >= T && (T <= 8 || scattered)))) return launch_product_stream(handle, fn, Xtype, a);
  }
  if (in > 0 && Xtype != HYACIN_F32) return launch_product_umma(handle, fn, trans, Xtype, a);
  float* mid = nullptr;
  int32_t rc = 0;
  with_w4_type(Xtype, [&](auto tag) {
    using E = decltype(tag);
    if (a.rank) {
      const int64_t entries = int64_t(a.rank) * T;
      const cudaError_t e = cudaMallocFromPoolAsync(reinterpret_cast<void**>(&mid), entries * sizeof(float), handle->mempool, stream);
      if (e != cudaSuccess) { report_cuda_error(e, "cudaMallocFromPoolAsync", __FILE__, __LINE__); rc = -3; return; }
      a.mid = mid;
      count_launch();
      correction_mid_kernel<E><<<unsigned((entries + 7) / 8), 256, 0, stream>>>(static_cast<const E*>(a.first), a.ld1, in, a.rank, static_cast<const E*>(X), ldx, T, mid);
    }
    const unsigned ty = unsigned(min((T + kPlainTokens - 1) / kPlainTokens, 65535));
    count_launch();
    if (trans) product_t_plain_kernel<E><<<dim3((N + 7) / 8, ty), 256, 0, stream>>>(a);
    else {
      const int blocks = (M + kW4Block - 1) / kW4Block;
      int splits = 1;
      while (splits < 8 && int64_t(blocks) * ty * splits < 4 * int64_t(handle->DeviceSMs) && splits * 2 * kSingleLanes <= N) splits *= 2;
      cudaLaunchConfig_t cfg{};
      cfg.gridDim = dim3(unsigned(blocks) * splits, ty); cfg.blockDim = dim3(kSingleThreads); cfg.stream = stream;
      cudaLaunchAttribute attr[1];
      attr[0].id = cudaLaunchAttributeClusterDimension; attr[0].val.clusterDim.x = splits; attr[0].val.clusterDim.y = 1; attr[0].val.clusterDim.z = 1;
      cfg.attrs = attr; cfg.numAttrs = splits > 1 ? 1 : 0;
      const cudaError_t e = cudaLaunchKernelEx(&cfg, product_n_single_kernel<E>, a, splits);
      if (e != cudaSuccess) { report_cuda_error(e, fn, __FILE__, __LINE__); rc = -3; return; }
    }
    rc = w4_launched(fn);
  });
  if (mid) HYB_CUDA(cudaFreeAsync(mid, stream));
  return rc;
}
