// Products with a 4-bit weight matrix, Y = Wq^T X + V (U^T X) and Y = Wq X + U (V^T X), with
// Wq(r, j) = s(j, r / segM) (q(r, j) - zero(j, r / segM)).
#include "w4_product.h"
#include <algorithm>

namespace hyb {
namespace {

// The sum over nothing.
__global__ void __launch_bounds__(256) zero_kernel(uint8_t* y, int64_t pitch, int64_t bytes, int t) {
  for (int64_t v = blockIdx.y; v < t; v += gridDim.y)
    for (int64_t i = int64_t(blockIdx.x) * 256 + threadIdx.x; i < bytes; i += int64_t(gridDim.x) * 256) y[v * pitch + i] = 0;
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
    if (lds < w4_segments(M, segM)) return w4_refuse(fn, "lds too small");
    if (ldq % 16 || ldq < (int64_t(M) + 127) / 128 * 64 || reinterpret_cast<uintptr_t>(codes) % 16) return w4_refuse(fn, "codes: 16-byte aligned, ldq a multiple of 16 and at least 64 ceil(M / 128)");
    if (rank > 0 && (!U || !V || ldu < M || ldv < N)) return w4_refuse(fn, "U, V: null or leading dimension too small");
  }
  if (!w4_on_boundary(w4_type_bytes(Xtype), Y) || (in > 0 && !w4_on_boundary(w4_type_bytes(Xtype), X, scales)) || (in > 0 && rank > 0 && !w4_on_boundary(w4_type_bytes(Xtype), U, V)))
    return w4_refuse(fn, "a pointer that is not on a boundary of its type");
  if (w4_refuse_handle(fn, handle)) return -1;
  const ProductArgs a{codes, ldq, M, N, T, segM, scales, zeros, lds, X, ldx, rank, trans ? U : V, trans ? ldu : ldv, trans ? V : U, trans ? ldv : ldu, Y, ldy};
  timer_mark(handle, Segment::Replicated);
  if (in == 0) {
    const int64_t size = int64_t(w4_type_bytes(Xtype));
    count_launch();
    return w4_result(w4_start(zero_kernel, dim3(unsigned(std::min<int64_t>((out * size + 255) / 256, 1024)), unsigned(std::min(T, 4096))), 256, 0, handle->cudaStream, static_cast<uint8_t*>(Y), ldy * size, out * size, T), fn);
  }
  const int per = trans ? product_stream_vectors(Xtype, a) : 0;
  if (Xtype == HYACIN_F32) {
    // Five passes of the streaming kernel are where it meets the tiled one: 4096 x 4096 times 16, four passes, 39.6 against 42.5 us, times 20,
    // five, 49.3 against 49.0, six would be 59 against 49.7; 8192 x 4096 times 10, five of two vectors, 62 against 81; 4096 x 16384 times 20 99
    // against 182.  With few columns the streaming kernel leaves SMs idle and the tiled one splits the rows (16384 x 200 times 4: 49 against 16).
    const bool filled = N >= (T <= per ? 2 : 8) * handle->DeviceSMs;
    if (per > 0 && T <= 5 * per && filled) return launch_product_stream(handle, fn, Xtype, a);
    return launch_product_single(handle, fn, trans, a);
  }
  // Up to eight vectors stream (17 against 23 us, 4096 x 16384); up to sixteen where the tensor-core kernel cannot fetch a block's
  // scales at once (24 against 58 us, 5001 x 6003, segments of 32 rows, odd table pitch).
  const bool scattered = segM % 128 != 0 && (segM == 96 || lds % (128 / std::min(segM, 64)) != 0 || reinterpret_cast<uintptr_t>(scales) % (256 / std::min(segM, 64)) != 0);
  if (per >= T && (T <= 8 || scattered)) return launch_product_stream(handle, fn, Xtype, a);
  return launch_product_umma(handle, fn, trans, Xtype, a);
}
