// 4-bit form of a weight matrix: per (column, segment) scale s = max|w| / 7 (or (hi - lo) / 15 with a zero point), codes
// q = rint(w / s) + zero, and the residual w - s (q - zero) that a low-rank fit takes.
//
// The quotient decides a whole number, so it is rounded as if it were exact.  In 64 bits that needs no care: w and s carry at most 24
// bits, a quotient that is not exactly a half differs from it by at least 2^-28 relative, and rint of the 64-bit quotient is that of the exact
// one.  Scales and quotients of ordinary size are done in 32 bits with one correction step, as said at rounded_quotient and quotient_bits.
#include "w4.cuh"
#include <algorithm>

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

// rint(v / s), ties to even, as if the quotient were exact, given `inverse` = 1 / s to within 2^-22.  v * inverse then finds the nearest
// whole number, or next to a half its neighbour.  The remainder v - whole s is exact in 32 bits (a multiple of the smaller of
// the two last places, and at most about s / 2), and twice that against s decides.  Adding and subtracting 1.5 * 2^23 rounds to
// a whole number on the floating-point pipe: the conversion instructions, four per weight, took longer than DRAM.
constexpr float kRound = 12582912.f;
__device__ __forceinline__ float rounded_quotient(float v, float s, float inverse) {
  const float m = __fmaf_rn(v, inverse, kRound), whole = __fadd_rn(m, -kRound), r = __fmaf_rn(-whole, s, v), twice = 2.f * fabsf(r);
  const bool off = twice > s || (twice == s && (__float_as_int(m) & 1));
  return off ? whole + copysignf(1.f, r) : whole;
}
// That holds for ordinary scales and quotients below 32 in magnitude; `largest`: of the segment's weights.
__device__ __forceinline__ bool ordinary(float s, float inverse, float largest) { return s > 1e-30f && s < 1e30f && largest * inverse < 32.f; }
__device__ __noinline__ float quotient_in_64_bits(float v, float s) { return float(fmin(fmax(rint(double(v) / double(s)), -64.), 64.)); }
__device__ __forceinline__ float reciprocal(float s) { float r; asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(s)); return r; }

// x / by for 7 and 15.  A product with the rounded reciprocal is within a last place, and one step corrects it (Markstein, IBM J. Res. Dev.
// 34, 1990; a test compares all 2^23 fractions with the division); the range keeps the remainder's last place above the smallest number.
__device__ __forceinline__ float divided(float x, float by) {
  if (!(x > 1e-28f && x < 1e30f)) return __fdiv_rn(x, by);
  const float inverse = by == 7.f ? 1.f / 7.f : 1.f / 15.f, q = __fmul_rn(x, inverse);
  return __fmaf_rn(__fmaf_rn(-by, q, x), inverse, q);
}
// lo, hi: extremes of the segment together with 0; bad: it holds a NaN or an infinity.  float(double / 7) is the 32-bit quotient;
// so is float(double / 15) of a difference that 32 bits hold.
template <class S> __device__ __forceinline__ S segment_scale(float lo, float hi, bool bad, bool symmetric) {
  float span;
  if (symmetric) span = divided(fmaxf(-lo, hi), 7.f);
  else {
    const float more = fmaxf(hi, -lo), less = fminf(hi, -lo), f = __fadd_rn(more, less);
    span = __fsub_rn(f, more) == less ? divided(f, 15.f) : float((double(hi) - double(lo)) / 15.);   // the sum is exact or it is not
  }
  return from_f32<S>(bad ? __int_as_float(0x7fc00000) : span);
}
template <class S> __device__ __forceinline__ SegmentCode segment_code(float lo, float hi, bool bad, bool symmetric, S* scale) {
  SegmentCode c;
  *scale = segment_scale<S>(lo, hi, bad, symmetric);
  const float s = to_f32(*scale);
  c.s = double(s);
  c.live = s > 0.f;                                    // false for NaN as well
  if (symmetric) c.zero = 8;
  else if (!c.live) c.zero = 0;
  else {
    const float inverse = reciprocal(s);
    c.zero = int(fminf(fmaxf(ordinary(s, inverse, -lo) ? rounded_quotient(-lo, s, inverse) : quotient_in_64_bits(-lo, s), 0.f), 15.f));
  }
  return c;
}

// kRound + rint(v / s), the form that the codes are read from.  For a 16-bit scale the quotient itself is cheaper than the remainder above:
// one correction step (Markstein, IBM J. Res. Dev. 34, 1990) leaves it within 2^-22 of a last place of its rounding to 32 bits, and that
// rounding hits a half only where the quotient is one: half * s is a 32-bit number then, so v is at least a last place away from
// it, the quotient at least (1 + 2^-11) half places from the half.
template <class S> __device__ __forceinline__ float quotient_bits(float v, float s, float inverse) {
  if (sizeof(S) == 4) return rounded_quotient(v, s, inverse) + kRound;
  const float q = __fmul_rn(v, inverse);
  return __fadd_rn(__fmaf_rn(__fmaf_rn(-q, s, v), inverse, q), kRound);
}
__device__ __forceinline__ float largest_of(float a, float b, float c) { float d; asm("max.NaN.abs.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c)); return d; }

// Segments of 32, 64, 128 or 256 rows: a lane owns eight consecutive rows, one word of codes, a warp 256 rows of a column; a
// segment's lanes are neighbours and find its extremes with shuffles, so W is read once and everything stays in registers.
// Rows that are not 16-byte aligned pass through shared memory, so that DRAM sees whole lines all the same.
// A warp walks down the columns of its row group with the next columns' loads in flight.
// Bound: with residual (4 more bytes written per weight) DRAM and issue, 60 and 64 % of either; without it instruction issue, 78 % of the slots
// beside 32 % of DRAM (4096 x 16384 bfloat16), and for small matrices the start and end of a walk over few columns.  Measured: 16384 x
// 4096 bfloat16 with residual 77 us, 5.6 TB/s; 4096 x 4096 bfloat16 15.4 us, 2.7 TB/s; 8190 x 2049 float, rows off their alignment, zero
// points and residual 31 us, 4.6 TB/s (23.7 us aligned).
template <class T, class S, bool SYMMETRIC, bool WIDE> __device__ __forceinline__ void quantize_columns(const QuantizeArgs& a, int r_aligned, float* turn) {
  constexpr int kWords = int(sizeof(T)) * 8 / 16, kDepth = WIDE && sizeof(T) == 2 ? 2 : 1;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int row0 = blockIdx.x * 256, row = row0 + lane * 8, valid = WIDE ? 8 : a.m - row, all = WIDE ? 256 : a.m - row0;
  const int step = gridDim.y * 8, lanes = a.seg / 8, r8 = row / 8, col0 = blockIdx.y * 8 + warp;
  const bool writes = r8 < (a.m + kW4Block - 1) / kW4Block * 16, leads = lane % lanes == 0 && valid > 0;
  uint8_t* codes = a.codes + col0 * a.ldq + int64_t(r8 / 16) * 64 + (4 * (r8 & 3) + ((r8 >> 2) & 3)) * 4;
  const T* from = static_cast<const T*>(a.w) + col0 * a.ldw + row0;
  int64_t table = col0 * a.lds + row / a.seg;
  float* to = a.r ? a.r + col0 * a.ldr + row0 : nullptr;
  const int64_t w_step = step * a.ldw, q_step = step * a.ldq, s_step = step * a.lds, r_step = step * a.ldr;
  int partner[5];
#pragma unroll
  for (int i = 0; i < 5; ++i) partner[i] = (1 << i) < lanes ? 1 << i : 0;
  uint4 raw[kDepth][kWords]; T part[8];
  auto fetch = [&](int64_t col, int buf) {
    if (col < a.n) {
      if (WIDE) {
#pragma unroll
        for (int i = 0; i < kWords; ++i) raw[buf][i] = __ldcs(reinterpret_cast<const uint4*>(from + lane * 8) + i);
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) if (i * 32 + lane < all) part[i] = from[i * 32 + lane];
      }
    }
    from += w_step;
  };
  auto column = [&](int64_t col, int buf) {
    float v[8];
    if (WIDE) {
      const T* e = reinterpret_cast<const T*>(raw[buf]);
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = to_f32(e[i]);
    } else {
      __syncwarp();
#pragma unroll
      for (int i = 0; i < 8; ++i) turn[i * 32 + lane] = i * 32 + lane < all ? to_f32(part[i]) : 0.f;
      __syncwarp();
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = turn[lane * 8 + i];
      __syncwarp();
    }
    fetch(col + kDepth * step, buf);
    // the largest magnitude, infinities and NaNs among them; as an integer a NaN is the largest
    const float most = largest_of(largest_of(v[0], v[1], v[2]), largest_of(v[3], v[4], v[5]), largest_of(v[6], v[7], 0.f));
    int size = __float_as_int(most) & 0x7fffffff;
    float lo = 0.f, hi = 0.f;
    if (!SYMMETRIC) {
#pragma unroll
      for (int i = 0; i < 8; ++i) { lo = fminf(lo, v[i]); hi = fmaxf(hi, v[i]); }
    }
#pragma unroll
    for (int i = 0; i < 5; ++i) {                    // a lane beyond the segment's is taken for itself
      size = max(size, __shfl_xor_sync(~0u, size, partner[i]));
      if (!SYMMETRIC) { lo = fminf(lo, __shfl_xor_sync(~0u, lo, partner[i])); hi = fmaxf(hi, __shfl_xor_sync(~0u, hi, partner[i])); }
    }
    const float largest = __int_as_float(size);
    if (SYMMETRIC) hi = largest;
    const S scale = segment_scale<S>(lo, hi, size >= 0x7f800000, SYMMETRIC);
    const float s = to_f32(scale), inverse = reciprocal(s);
    float zero = SYMMETRIC ? 8.f : 0.f, whole[8];    // whole: kRound + the code minus its zero point
    // With the largest quotient below 7.44 (15.44) nothing has to be clamped but the upper end beside a zero point, where both ends may
    // have been rounded up: rint is monotonic and odd, so no code falls below 1 (0).
    if (ordinary(s, inverse, largest) && largest * inverse < (SYMMETRIC ? 7.4375f : 15.4375f)) {
      if (!SYMMETRIC) zero = quotient_bits<S>(-lo, s, inverse) - kRound;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        whole[i] = quotient_bits<S>(v[i], s, inverse);
        if (!SYMMETRIC) whole[i] = fminf(whole[i], kRound + 15.f - zero);
      }
    } else if (s > 0.f) {                            // the same with quotients in 64 bits
      if (!SYMMETRIC) zero = fminf(fmaxf(quotient_in_64_bits(-lo, s), 0.f), 15.f);
      const float low = SYMMETRIC ? -7.f : -zero, high = SYMMETRIC ? 7.f : 15.f - zero;
#pragma unroll
      for (int i = 0; i < 8; ++i) whole[i] = kRound + fminf(fmaxf(quotient_in_64_bits(v[i], s), low), high);
    } else {                                         // no scale: nothing but zeros, or a NaN
#pragma unroll
      for (int i = 0; i < 8; ++i) whole[i] = kRound;
    }
    if (leads) {
      static_cast<S*>(a.scales)[table] = scale;
      if (!SYMMETRIC) a.zeros[table] = uint8_t(int(zero));
    }
    table += s_step;
    // the last places of kRound + k are 0x4b400000 + k: summed with shifts, the codes come out where they belong
    uint32_t word = (__float_as_uint(kRound + zero) - 0x4b400000u) * 0x11111111u - 0x4b400000u * 0x11111111u;
#pragma unroll
    for (int i = 0; i < 8; ++i) word += __float_as_uint(whole[i]) << (4 * w4_row_nibble(i));
    if (!WIDE && valid < 8) {                        // rows behind the last one are stored as 0
#pragma unroll
      for (int i = 0; i < 8; ++i) if (i >= valid) word &= ~(15u << (4 * w4_row_nibble(i)));
    }
    if (writes) *reinterpret_cast<uint32_t*>(codes) = word;
    codes += q_step;
    if (to) {
      float r[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) r[i] = fmaf(-s, whole[i] - kRound, v[i]);
      if (r_aligned && all >= 256) {
        __stcs(reinterpret_cast<float4*>(to + lane * 8), make_float4(r[0], r[1], r[2], r[3]));
        __stcs(reinterpret_cast<float4*>(to + lane * 8) + 1, make_float4(r[4], r[5], r[6], r[7]));
      } else {
        __syncwarp();
#pragma unroll
        for (int i = 0; i < 8; ++i) turn[lane * 8 + i] = r[i];
        __syncwarp();
#pragma unroll
        for (int i = 0; i < 8; ++i) if (i * 32 + lane < all) __stcs(to + i * 32 + lane, turn[i * 32 + lane]);
      }
      to += r_step;
    }
  };
#pragma unroll
  for (int d = 0; d < kDepth; ++d) fetch(col0 + d * step, d);
  for (int64_t col = col0; col < a.n; col += kDepth * step) {
#pragma unroll
    for (int d = 0; d < kDepth; ++d) if (col + d * step < a.n) column(col + d * step, d);
  }
}
template <class T, class S, bool SYMMETRIC> __global__ void __launch_bounds__(256, 4) quantize_w4_warp_kernel(QuantizeArgs a, int w_aligned, int r_aligned) {
  __shared__ __align__(16) float turns[8][256];
  float* turn = turns[threadIdx.x >> 5];
  if (w_aligned && a.m - int(blockIdx.x) * 256 >= 256) quantize_columns<T, S, SYMMETRIC, true>(a, r_aligned, turn);
  else quantize_columns<T, S, SYMMETRIC, false>(a, r_aligned, turn);
}

// Any other segment length: one warp per (column, segment), a pass for the extremes, a pass for the codes; latency of its own two passes.
template <class T, class S> __global__ void __launch_bounds__(256) quantize_w4_kernel(QuantizeArgs a) {
  const int lane = threadIdx.x & 31;
  const int64_t task = int64_t(blockIdx.x) * 8 + (threadIdx.x >> 5);
  if (task >= int64_t(a.n) * a.segs) return;
  const int col = int(task / a.segs), seg = int(task % a.segs);
  const T* w = static_cast<const T*>(a.w) + col * a.ldw;
  const int row0 = seg * a.seg, row1 = int(min(int64_t(row0) + a.seg, int64_t(a.m)));
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
  const int sub0 = row0 / 32, sub1 = seg + 1 == a.segs ? (a.m + kW4Block - 1) / kW4Block * 4 : row1 / 32;
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
  if (M > 0x7fffff00 || N > 0x7fffff00) return w4_refuse(fn, "sizes: M, N at most 2^31 - 256");
  if (M == 0 || N == 0) return 0;
  const int segs = w4_segments(M, segM);
  if (!W || !codes || !scales) return w4_refuse(fn, "null pointer");
  if (ldw < M || lds < segs || (R && ldr < M)) return w4_refuse(fn, "leading dimension too small");
  if (ldq % 16 || ldq < (int64_t(M) + 127) / 128 * 64 || reinterpret_cast<uintptr_t>(codes) % 16) return w4_refuse(fn, "codes: 16-byte aligned, ldq a multiple of 16 and at least 64 ceil(M / 128)");
  if (!w4_on_boundary(w4_type_bytes(Wtype), W) || !w4_on_boundary(w4_type_bytes(Stype), scales) || !w4_on_boundary(4, R)) return w4_refuse(fn, "a pointer that is not on a boundary of its type");
  if (w4_refuse_handle(fn, handle)) return -1;
  QuantizeArgs a{W, ldw, M, N, segM, segs, codes, ldq, scales, zeros, lds, R, ldr};
  const int64_t blocks = (int64_t(N) * segs + 7) / 8;
  if (blocks > 0x7fffffff) return w4_refuse(fn, "too many segments");
  timer_mark(handle, Segment::Replicated);
  count_launch();
  cudaError_t e = cudaSuccess;
  if (segM == 32 || segM == 64 || segM == 128 || segM == 256) {
    const int64_t groups = (int64_t(M) + 255) / 256;
    const int w_aligned = reinterpret_cast<uintptr_t>(W) % 16 == 0 && int64_t(ldw) * int64_t(w4_type_bytes(Wtype)) % 16 == 0;
    const int r_aligned = reinterpret_cast<uintptr_t>(R) % 16 == 0 && ldr % 4 == 0;
    // about eight blocks per SM, so that a warp sees several columns
    const int64_t chunks = std::max<int64_t>(1, std::min<int64_t>({(int64_t(N) + 7) / 8, 8 * int64_t(handle->DeviceSMs) / groups, 65535}));
    with_w4_type(Wtype, [&](auto t) { with_w4_type(Stype, [&](auto s) {
      auto* kernel = zeros ? quantize_w4_warp_kernel<decltype(t), decltype(s), false> : quantize_w4_warp_kernel<decltype(t), decltype(s), true>;
      e = w4_start(kernel, dim3(unsigned(groups), unsigned(chunks)), 256, 0, handle->cudaStream, a, w_aligned, r_aligned);
    }); });
    return w4_result(e, "quantize_w4_warp_kernel");
  }
  with_w4_type(Wtype, [&](auto t) { with_w4_type(Stype, [&](auto s) {
    e = w4_start(quantize_w4_kernel<decltype(t), decltype(s)>, dim3(unsigned(blocks)), 256, 0, handle->cudaStream, a);
  }); });
  return w4_result(e, "quantize_w4_kernel");
}
