// 4-bit form of a weight matrix: per (column, segment) scale s = max|w| / 7 (or (hi - lo) / 15 with a zero point), codes
// q = rint(w / s) + zero, and the residual w - s (q - zero) that a low-rank fit takes.
//
// The quotient decides a whole number, so it is taken in 64 bits: w and s carry at most 24 bits, a quotient that is not
// exactly a half differs from it by at least 2^-28 relative, and rint of the 64-bit quotient is that of the exact one.
#include "w4.cuh"

namespace hyb {
namespace {

struct QuantizeArgs {
  const void* w; int64_t ldw; int m, n, seg, segs;
  uint8_t* codes; int64_t ldq; void* scales; uint8_t* zeros; int64_t lds;
  float* r; int64_t ldr;
};

struct SegmentCode {        // what a segment's codes are computed with
  double s; int zero; bool live;
  __device__ __forceinline__ int code(float v, bool symmetric) const {
    if (!live) return zero;
    const double q = rint(double(v) / s);
    return symmetric ? int(fmin(fmax(q, -7.), 7.)) + 8 : int(fmin(fmax(q + zero, 0.), 15.));
  }
};

// lo, hi: extremes of the segment together with 0; bad: it holds a NaN or an infinity.
template <class S> __device__ __forceinline__ SegmentCode segment_code(float lo, float hi, bool bad, bool symmetric, S* scale) {
  SegmentCode c;
  const double span = symmetric ? double(fmaxf(-lo, hi)) / 7. : (double(hi) - double(lo)) / 15.;
  *scale = bad ? from_f32<S>(__int_as_float(0x7fc00000)) : from_f32<S>(float(span));
  c.s = double(to_f32(*scale));
  c.live = c.s > 0.;                                   // false for NaN as well
  c.zero = symmetric ? 8 : c.live ? int(fmin(fmax(rint(-double(lo) / c.s), 0.), 15.)) : 0;
  return c;
}

// One warp per (column, segment): a pass for the extremes, a pass for the codes.
template <class T, class S> __global__ void __launch_bounds__(256) quantize_w4_kernel(QuantizeArgs a) {
  const int lane = threadIdx.x & 31;
  const int64_t task = int64_t(blockIdx.x) * 8 + (threadIdx.x >> 5);
  if (task >= int64_t(a.n) * a.segs) return;
  const int col = int(task / a.segs), seg = int(task % a.segs);
  const T* w = static_cast<const T*>(a.w) + col * a.ldw;
  const int row0 = seg * a.seg, row1 = min(row0 + a.seg, a.m);
  float lo = 0.f, hi = 0.f; bool bad = false;
  for (int r = row0 + lane; r < row1; r += 32) {
    const float v = to_f32(w[r]);
    bad |= !(fabsf(v) <= 3.402823466e38f); lo = fminf(lo, v); hi = fmaxf(hi, v);
  }
  for (int d = 16; d; d >>= 1) { lo = fminf(lo, __shfl_xor_sync(~0u, lo, d)); hi = fmaxf(hi, __shfl_xor_sync(~0u, hi, d)); }
  bad = __any_sync(~0u, bad);
  const bool symmetric = a.zeros == nullptr;
  S scale; const SegmentCode c = segment_code<S>(lo, hi, bad, symmetric, &scale);
  if (lane == 0) {
    static_cast<S*>(a.scales)[col * a.lds + seg] = scale;
    if (!symmetric) a.zeros[col * a.lds + seg] = uint8_t(c.zero);
  }
  // words of the segment's 32-row subsets; the last segment also fills its block up
  const int sub0 = row0 / 32, sub1 = (row0 + a.seg >= a.m) ? (a.m + kW4Block - 1) / kW4Block * 4 : (row0 + a.seg) / 32;
  for (int k = lane; k < (sub1 - sub0) * 4; k += 32) {
    const int sub = sub0 + k / 4, quarter = k & 3, row = 32 * sub + 8 * quarter;
    uint32_t word = 0;
    for (int e = 0; e < 8; ++e) {
      if (row + e >= a.m) break;
      const float v = to_f32(w[row + e]);
      const int q = c.code(v, symmetric);
      word |= uint32_t(q) << (4 * w4_row_nibble(e));
      if (a.r) a.r[col * a.ldr + row + e] = float(double(v) - c.s * double(q - c.zero));
    }
    *reinterpret_cast<uint32_t*>(a.codes + col * a.ldq + int64_t(sub / 4) * 64 + (4 * quarter + (sub & 3)) * 4) = word;
  }
}

}  // namespace
}  // namespace hyb

extern "C" int32_t hyacinB200QuantizeW4(const hyacinHandle_t* handle, hyacinPrecision_t Wtype, int32_t M, int32_t N, const void* W,
                                        int32_t ldw, int32_t segM, hyacinPrecision_t Stype, uint8_t* codes, int64_t ldq, void* scales,
                                        uint8_t* zeros, int32_t lds, float* R, int32_t ldr) {
  using namespace hyb;
  const char* fn = "hyacinB200QuantizeW4";
  if (!handle) return w4_refuse(fn, "no handle");
  if (!is_w4_type(Wtype) || !is_w4_type(Stype)) return w4_refuse(fn, "type not supported");
  if (M < 0 || N < 0 || segM <= 0 || segM % 32) return w4_refuse(fn, "sizes: M, N >= 0 and segM a positive multiple of 32");
  if (M == 0 || N == 0) return 0;
  const int segs = (int64_t(M) + segM - 1) / segM;
  if (!W || !codes || !scales) return w4_refuse(fn, "null pointer");
  if (ldw < M || lds < segs || (R && ldr < M)) return w4_refuse(fn, "leading dimension too small");
  if (ldq % 16 || ldq < (int64_t(M) + 127) / 128 * 64 || reinterpret_cast<uintptr_t>(codes) % 16) return w4_refuse(fn, "codes: 16-byte aligned, ldq a multiple of 16 and at least 64 ceil(M / 128)");
  if (!w4_device_ok(handle)) return w4_refuse(fn, "the handle belongs to another device than the current one");
  QuantizeArgs a{W, ldw, M, N, segM, segs, codes, ldq, scales, zeros, lds, R, ldr};
  const int64_t blocks = (int64_t(N) * segs + 7) / 8;
  if (blocks > 0x7fffffff) return w4_refuse(fn, "too many segments");
  timer_mark(handle, Segment::Replicated);
  count_launch();
  with_w4_type(Wtype, [&](auto t) { with_w4_type(Stype, [&](auto s) {
    quantize_w4_kernel<decltype(t), decltype(s)><<<unsigned(blocks), 256, 0, handle->cudaStream>>>(a);
  }); });
  return w4_launched("quantize_w4_kernel");
}
