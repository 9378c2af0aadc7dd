// Distillation loss against a teacher's top logits, and its gradient.
//
// Per token, with u = z / tau and the list i = 1 .. K of classes c_i with teacher logits t_i:
//     p_i = exp(t_i / tau - teacherLse), p_r = max(0, 1 - sum p), 0 when every class is listed   or, without teacherLse, p_i = softmax over the list, p_r = 0
//     lse = log sum_j exp u_j,  lse_r = log sum over the classes outside the list
//     KL  = sum_i p_i (log p_i - (u_{c_i} - lse)) + p_r (log p_r - (lse_r - lse))
//     dKL/dz_j = (q_j mass - P_j) / tau                        listed: P_j = sum of its p_i, mass = sum p + p_r
//     dKL/dz_j = exp(u_j - lse_r) (mass exp(lse_r - lse) - p_r) / tau    outside the list
// The sum over the classes outside is accumulated without the listed ones, so p_r / q_r never comes from a difference, and
// what concerns the list (K terms) is done in 64 bits: where student and teacher agree, q - p is the difference of two numbers
// close to one.
//
// Two kernels.  distill_cluster_kernel keeps a token's logits in the shared memory of a cluster of one to eight CTAs: they are read
// from DRAM once, with bulk copies, and the gradient is written from there; one exchange of (maximum, sum) per CTA is all the
// communication.  Several CTAs per SM (see kSliceBytes) overlap their loads, arithmetic and stores.
// distill_plain_kernel (one block per token, passes over global memory) takes rows that do not fit a cluster.
// Bound: the phases of a token (copy, maximum, sum, exchange, gradient), which three CTAs per SM do not hide: 34 % of DRAM, 48 % of the issue
// slots and of the exponentials' pipe.  512 tokens of 128000 bfloat16 logits, a fifth masked, loss and gradient: 70 us with the launch,
// 3.4 TB/s; the plain kernel took 590.
// exp is taken as 2^(z scale - c), scale = log2(e) / tau and c = float(top scale), one fused multiply-add and one ex2 per entry;
// what rounding c loses, kappa = top scale - c, is known in 64 bits and put back into the sum, so the loss does not see it.  Beyond
// |c| = 2^27 kappa itself would leave the range of 2^x; there the difference z - top is formed first, one instruction more per entry.
#include "w4.cuh"
#include "ptx_sm100.cuh"
#include <atomic>
#include <algorithm>
#include <type_traits>

namespace hyb {
namespace {

constexpr int kMaxList = 1024;
constexpr int kMaxClasses = 1 << 20;

struct DistillArgs {
  const void* z; int64_t ldz; int n, t, k;
  const int32_t* ids; const float* teacher; int64_t ldk; double tau, inv_tau;
  const float* teacher_lse; const float* weight;
  float* loss; float* stats_out; const float* stats_in;
  void* dz; int64_t lddz;
  int splits, list_at;      // cluster kernel: CTAs per token, start of the list in shared memory
};

__device__ __forceinline__ float ex2(float x) { float r; asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x)); return r; }
// 2^(z scale - c) relative to top: c and the factor that puts kappa back.  top = 0 stands for "nothing there".
struct Exponent {
  float scale, c, top;
  __device__ __forceinline__ Exponent(double tau, float t) : scale(float(1.4426950408889634 / tau)), c(t * scale), top(t) {}
  __device__ double fix() const {
    const double x = (double(c) - double(top) * double(scale)) * 0.69314718055994530942;
    return fabs(x) < 1e-4 ? 1. + x * (1. + x * (0.5 + x * (1. / 6.))) : exp(x);
  }
  __device__ __forceinline__ float operator()(float z) const { return ex2(fmaf(z, scale, -c)); }
  __device__ __forceinline__ bool far() const { return !(fabsf(c) < 134217728.f); }
};
struct FarExponent {
  float scale, top;
  __device__ double fix() const { return 1.; }
  __device__ __forceinline__ float operator()(float z) const { return ex2((z - top) * scale); }
};
// f with the form that serves; the same for every thread of a token.
template <class F> __device__ __forceinline__ void with_exponent(double tau, float top, F&& f) {
  const Exponent e(tau, top);
  if (e.far()) f(FarExponent{e.scale, top}); else f(e);
}

// Sum / maximum over the block, the same in every thread.  buf: 32 entries.
template <class V, class F> __device__ V block_reduce(V v, F f, V* buf) {
  for (int d = 16; d; d >>= 1) v = f(v, __shfl_xor_sync(~0u, v, d));
  __syncthreads();
  if ((threadIdx.x & 31) == 0) buf[threadIdx.x >> 5] = v;
  __syncthreads();
  V r = buf[0];
  for (unsigned i = 1; i < blockDim.x / 32; ++i) r = f(r, buf[i]);
  return r;
}
struct Add { template <class V> __device__ V operator()(V a, V b) const { return a + b; } };
struct Max { template <class V> __device__ V operator()(V a, V b) const { return a > b ? a : b; } };

// The list of one token in shared memory, `k` entries each.
struct List {
  double *p, *logp, *psum;   // teacher probability, its logarithm, sum over the entries of the same class
  double* e;                 // exp(z / tau - top of the list), 0 for entries that are skipped
  float* z;                  // student logit
  int *id, *first;           // class, -1 when skipped; 1 for the first entry of its class
  double* buf; float* fbuf;  // 32 entries each, for reductions
  __device__ List(uint8_t* at, int k) {
    buf = reinterpret_cast<double*>(at); p = buf + 32; logp = p + k; psum = logp + k; e = psum + k;
    fbuf = reinterpret_cast<float*>(e + k); z = fbuf + 32; id = reinterpret_cast<int*>(z + k); first = id + k;
  }
};
__host__ __device__ constexpr size_t list_bytes(int k) { return 32 * 12 + size_t(k) * 44; }

// What is known of the teacher, and of the student's listed classes, before the rest of the row has been seen.
struct Listed { double rest, mass, top, sum; };      // p_r, sum p + p_r; log-sum-exp of the student's listed classes as top + log(sum), top = -inf without any

// exp(z / tau - top), top the maximum over the listed classes.  Maxima leave NaNs out, so a list of NaNs has no top, but its sum is one.
__device__ __forceinline__ double relative_exp(float z, double inv_tau, double top) { return top == -INFINITY ? (z == -INFINITY ? 0. : double(z)) : exp(double(z) * inv_tau - top); }

// Reads the list.  Ends with a barrier.
template <class T> __device__ Listed load_list(const DistillArgs& a, int64_t token, const T* z, List& s) {
  double top = -INFINITY, student = -INFINITY;
  for (int i = threadIdx.x; i < a.k; i += blockDim.x) {
    const int id = a.ids[token * a.ldk + i];
    const bool ok = id >= 0 && id < a.n;
    s.id[i] = ok ? id : -1;
    const double t = ok ? double(a.teacher[token * a.ldk + i]) * a.inv_tau : -INFINITY;
    s.logp[i] = t; s.z[i] = ok ? to_f32(z[id]) : 0.f;
    top = fmax(top, t);
    if (ok) student = fmax(student, double(s.z[i]) * a.inv_tau);
  }
  double norm;
  if (a.teacher_lse) norm = double(a.teacher_lse[token]);
  else {
    top = block_reduce(top, Max{}, s.buf);
    double e = 0.;
    for (int i = threadIdx.x; i < a.k; i += blockDim.x) if (s.id[i] >= 0) e += exp(s.logp[i] - top);
    norm = top + log(block_reduce(e, Add{}, s.buf));
  }
  double sum = 0.;
  for (int i = threadIdx.x; i < a.k; i += blockDim.x) {
    const double l = s.logp[i] - norm;
    s.logp[i] = l; s.p[i] = s.id[i] >= 0 ? exp(l) : 0.;
    sum += s.p[i];
  }
  sum = block_reduce(sum, Add{}, s.buf);
  Listed r;
  r.top = block_reduce(student, Max{}, s.buf);
  double e = 0.; int classes = 0;
  for (int i = threadIdx.x; i < a.k; i += blockDim.x) {
    int first = s.id[i] >= 0; double ps = 0.;
    for (int j = 0; j < a.k; ++j) if (s.id[j] == s.id[i]) { ps += s.p[j]; if (j < i) first = 0; }
    s.first[i] = first; s.psum[i] = ps;
    s.e[i] = s.id[i] >= 0 ? relative_exp(s.z[i], a.inv_tau, r.top) : 0.;
    if (first) e += s.e[i];
    classes += first;
  }
  r.sum = block_reduce(e, Add{}, s.buf);
  r.rest = a.teacher_lse ? fmax(0., 1. - sum) : 0.;
  if (a.k >= a.n && int(block_reduce(double(classes), Add{}, s.buf)) == a.n) r.rest = 0.;      // what sum p leaves of 1 is rounding
  r.mass = sum + r.rest;
  __syncthreads();
  return r;
}

// The student's normaliser from the listed classes and the sum over the others, outside 2^(top scale), everything relative to the larger of
// the two references: total = listed + outside shares.  Logarithms are left to the loss.
struct Student {
  double ref, list_share, outside_share, total; bool no_outside;      // exp(l.top - ref), exp(top / tau - ref)
  __device__ __forceinline__ Student(const DistillArgs& a, const Listed& l, float top, float outside) {
    no_outside = outside == 0.f;
    const double out = double(top) * a.inv_tau;
    ref = no_outside ? l.top : fmax(l.top, out);
    if (ref == -INFINITY) ref = 0.;
    list_share = l.top == -INFINITY ? 0. : exp(l.top - ref);
    outside_share = no_outside ? 0. : exp(out - ref);
    total = l.sum * list_share + double(outside) * outside_share;
  }
  // log q of a listed class, and of everything outside
  __device__ __forceinline__ double log_q(double u, double log_total) const { return total == 0. ? -INFINITY : u - ref - log_total; }
};
// This thread's part of the loss over its entries of the list.
__device__ __forceinline__ double listed_loss(const DistillArgs& a, const List& s, const Student& st, double log_total, int first, int step) {
  double kl = 0.;
  for (int i = first; i < a.k; i += step) if (s.p[i] != 0.) kl += s.p[i] * (s.logp[i] - st.log_q(double(s.z[i]) * a.inv_tau, log_total));
  return kl;
}
__device__ __forceinline__ double outside_loss(const DistillArgs& a, const Listed& l, const Student& st, double log_total, float top, float outside) {
  return l.rest > 0. ? l.rest * (log(l.rest) - (st.no_outside ? -INFINITY : log(double(outside)) + double(top) * a.inv_tau - st.ref - log_total)) : 0.;
}
// dKL/dz = factor * 2^(z scale - top scale) outside the list; without anything there 0, or what a list of NaNs makes of it
__device__ __forceinline__ double outside_factor(const DistillArgs& a, const Listed& l, const Student& st, float outside, float weight) {
  return st.no_outside ? 0. * st.total : double(weight) * a.inv_tau * (l.mass * st.outside_share / st.total - l.rest / double(outside));
}
__device__ __forceinline__ float listed_gradient(const DistillArgs& a, const List& s, const Listed& l, const Student& st, float weight, int i) {
  return float(double(weight) * a.inv_tau * ((st.total == 0. ? 0. : l.mass * s.e[i] * st.list_share / st.total) - s.psum[i]));
}

template <class T> __global__ void __launch_bounds__(512) distill_plain_kernel(DistillArgs a) {
  extern __shared__ __align__(128) uint8_t smem[];
  uint32_t* listed = reinterpret_cast<uint32_t*>(smem + (list_bytes(a.k) + 15) / 16 * 16);
  List s(smem, a.k);
  const T* z_all = static_cast<const T*>(a.z);
  for (int64_t token = blockIdx.x; token < a.t; token += gridDim.x) {
    const T* z = z_all + token * a.ldz;
    T* dz = a.dz ? static_cast<T*>(a.dz) + token * a.lddz : nullptr;
    const float weight = a.weight ? a.weight[token] : 1.f;
    __syncthreads();
    if (weight == 0.f) {
      if (threadIdx.x == 0) {
        if (a.loss) a.loss[token] = 0.f;
        if (a.stats_out) a.stats_out[2 * token] = a.stats_out[2 * token + 1] = __int_as_float(0x7fc00000);
      }
      if (dz) for (int j = threadIdx.x; j < a.n; j += blockDim.x) dz[j] = from_f32<T>(0.f);
      continue;
    }
    for (int j = threadIdx.x; j < (a.n + 31) / 32; j += blockDim.x) listed[j] = 0;
    const Listed l = load_list<T>(a, token, z, s);
    for (int i = threadIdx.x; i < a.k; i += blockDim.x) if (s.id[i] >= 0) atomicOr(&listed[s.id[i] >> 5], 1u << (s.id[i] & 31));
    __syncthreads();
    float top, outside;
    if (a.stats_in) { top = a.stats_in[2 * token]; outside = a.stats_in[2 * token + 1]; }
    else {
      top = -INFINITY;
      for (int j = threadIdx.x; j < a.n; j += blockDim.x) if (!(listed[j >> 5] >> (j & 31) & 1)) top = fmaxf(top, to_f32(z[j]));
      top = block_reduce(top, Max{}, s.fbuf);
      if (top == -INFINITY) top = 0.f;
      with_exponent(a.tau, top, [&](auto e) {
        double sum = 0.;
        for (int j = threadIdx.x; j < a.n; j += blockDim.x) if (!(listed[j >> 5] >> (j & 31) & 1)) sum += e(to_f32(z[j]));
        outside = float(block_reduce(sum, Add{}, s.buf) * e.fix());
      });
    }
    const Student st(a, l, top, outside);
    if (a.loss || a.stats_out) {
      const double log_total = log(st.total);
      const double loss = block_reduce(listed_loss(a, s, st, log_total, threadIdx.x, blockDim.x), Add{}, s.buf) + outside_loss(a, l, st, log_total, top, outside);
      if (threadIdx.x == 0) {
        if (a.loss) a.loss[token] = float(loss * weight);
        if (a.stats_out) { a.stats_out[2 * token] = top; a.stats_out[2 * token + 1] = outside; }
      }
    }
    if (dz) {
      with_exponent(a.tau, top, [&](auto e) {
        const float factor = float(outside_factor(a, l, st, outside, weight) * e.fix());
        for (int j = threadIdx.x; j < a.n; j += blockDim.x)
          if (!(listed[j >> 5] >> (j & 31) & 1)) dz[j] = from_f32<T>(factor * e(to_f32(z[j])));
      });
      for (int i = threadIdx.x; i < a.k; i += blockDim.x) if (s.first[i]) dz[s.id[i]] = from_f32<T>(listed_gradient(a, s, l, st, weight, i));
    }
  }
}

// ---- cluster kernel ------------------------------------------------------------------------------------------------
constexpr int kMainThreads = 256, kClusterThreads = kMainThreads + 32;      // the last warp works on the list
constexpr int kHashWords = 2048;                  // 65536 bits: finds out cheaply that no class is listed twice
__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }
__device__ __forceinline__ void main_sync() { asm volatile("bar.sync 1, %0;" ::"n"(kMainThreads) : "memory"); }
__device__ __forceinline__ float ld_cluster(const void* at, uint32_t rank) {
  uint32_t remote; float v;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(remote) : "r"(ptx::smem_u32(at)), "r"(rank));
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(remote) : "memory");
  return v;
}
template <class V, class F> __device__ __forceinline__ V warp_reduce(V v, F f) {
#pragma unroll
  for (int d = 16; d; d >>= 1) v = f(v, __shfl_xor_sync(~0u, v, d));
  return v;
}
// The entries of a 16-byte vector as floats, and back; their maximum together with m, two at a time for the 16-bit types.
template <class T> __device__ __forceinline__ void unpack(const uint4& v, float (&f)[16 / sizeof(T)]) {
  const T* p = reinterpret_cast<const T*>(&v);
#pragma unroll
  for (int i = 0; i < int(16 / sizeof(T)); ++i) f[i] = to_f32(p[i]);
}
template <class T> __device__ __forceinline__ uint4 pack(const float (&f)[16 / sizeof(T)]) {
  uint4 v;
  if constexpr (sizeof(T) == 4) v = make_uint4(__float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]), __float_as_uint(f[3]));
  else {
    uint32_t* o = reinterpret_cast<uint32_t*>(&v);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (std::is_same<T, __half>::value) { const __half2 h = __floats2half2_rn(f[2 * i], f[2 * i + 1]); o[i] = *reinterpret_cast<const uint32_t*>(&h); }
      else { const __nv_bfloat162 h = __floats2bfloat162_rn(f[2 * i], f[2 * i + 1]); o[i] = *reinterpret_cast<const uint32_t*>(&h); }
    }
  }
  return v;
}
template <class T> struct RowMax;
template <> struct RowMax<float> {
  float m = -INFINITY;
  __device__ __forceinline__ void add(const uint4& v) { m = fmaxf(fmaxf(m, fmaxf(__uint_as_float(v.x), __uint_as_float(v.y))), fmaxf(__uint_as_float(v.z), __uint_as_float(v.w))); }
  __device__ __forceinline__ float value() const { return m; }
};
template <> struct RowMax<__half> {
  __half2 m = __float2half2_rn(-INFINITY);
  __device__ __forceinline__ void add(const uint4& v) {
    const __half2* h = reinterpret_cast<const __half2*>(&v);
    m = __hmax2(__hmax2(m, __hmax2(h[0], h[1])), __hmax2(h[2], h[3]));
  }
  __device__ __forceinline__ float value() const { return fmaxf(__low2float(m), __high2float(m)); }
};
template <> struct RowMax<__nv_bfloat16> {
  __nv_bfloat162 m = __float2bfloat162_rn(-INFINITY);
  __device__ __forceinline__ void add(const uint4& v) {
    const __nv_bfloat162* h = reinterpret_cast<const __nv_bfloat162*>(&v);
    m = __hmax2(__hmax2(m, __hmax2(h[0], h[1])), __hmax2(h[2], h[3]));
  }
  __device__ __forceinline__ float value() const { return fmaxf(__low2float(m), __high2float(m)); }
};

// The list by one warp: first the classes, for the warps that wait to take them out of the row, then the arithmetic.
__device__ __forceinline__ bool list_classes(const DistillArgs& a, int64_t token, List& s, uint32_t* hash) {
  const int lane = threadIdx.x & 31;
  const int32_t* ids = a.ids + token * a.ldk;
  int id = lane < a.k ? ids[lane] : -1;
#pragma unroll
  for (int i = 0; i < kHashWords / 128; ++i) reinterpret_cast<uint4*>(hash)[i * 32 + lane] = make_uint4(0, 0, 0, 0);
  __syncwarp();
  bool twice = false;                                // some class may be listed twice
  for (int i = lane; i < a.k; i += 32) {
    const int next = i + 32 < a.k ? ids[i + 32] : -1;
    const bool ok = id >= 0 && id < a.n;
    s.id[i] = ok ? id : -1;
    if (ok) { const uint32_t bit = 1u << (id & 31); twice |= (atomicOr(&hash[(id >> 5) & (kHashWords - 1)], bit) & bit) != 0; }
    id = next;
  }
  return __any_sync(~0u, twice);
}
template <class T> __device__ Listed list_by_warp(const DistillArgs& a, int64_t token, const T* z, List& s, bool twice) {
  const int lane = threadIdx.x & 31;
  float top32 = -INFINITY, student32 = -INFINITY;
#pragma unroll 4
  for (int i = lane; i < a.k; i += 32) {
    const int id = s.id[i];
    const float t = id >= 0 ? a.teacher[token * a.ldk + i] : -INFINITY, v = id >= 0 ? to_f32(z[id]) : -INFINITY;
    s.logp[i] = double(t) * a.inv_tau; s.z[i] = v;
    top32 = fmaxf(top32, t); student32 = fmaxf(student32, v);
  }
  top32 = warp_reduce(top32, Max{}); student32 = warp_reduce(student32, Max{});
  Listed r;
  r.top = double(student32) * a.inv_tau;
  // with the teacher's log-sum-exp p = exp(t - lse), without it the exponentials over their sum
  const double norm = a.teacher_lse ? double(a.teacher_lse[token]) : top32 == -INFINITY ? 0. : double(top32) * a.inv_tau;
  double sum = 0.;
  for (int i = lane; i < a.k; i += 32) {
    const bool ok = s.id[i] >= 0;
    const double l = s.logp[i] - norm, p = ok ? exp(l) : 0.;
    s.logp[i] = l; s.p[i] = p; s.first[i] = ok;
    s.e[i] = ok ? relative_exp(s.z[i], a.inv_tau, r.top) : 0.;
    sum += p;
  }
  sum = warp_reduce(sum, Add{});
  const double share = a.teacher_lse ? 1. : 1. / sum, log_sum = a.teacher_lse ? 0. : log(sum);
  for (int i = lane; i < a.k; i += 32) { s.p[i] = s.psum[i] = s.id[i] >= 0 ? s.p[i] * share : 0.; s.logp[i] -= log_sum; }
  __syncwarp();
  if (twice)
    for (int i = lane; i < a.k; i += 32) {
      int first = s.id[i] >= 0; double ps = 0.;
      for (int j = 0; j < a.k; ++j) if (s.id[j] == s.id[i]) { ps += s.p[j]; if (j < i) first = 0; }
      s.first[i] = first; s.psum[i] = ps;
    }
  double e = 0.; int classes = 0;
  for (int i = lane; i < a.k; i += 32) if (s.first[i]) { e += s.e[i]; ++classes; }
  r.sum = warp_reduce(e, Add{});
  if (a.teacher_lse) {
    r.rest = fmax(0., 1. - sum);
    if (a.k >= a.n && warp_reduce(classes, Add{}) == a.n) r.rest = 0.;      // what sum p leaves of 1 is rounding
    r.mass = sum + r.rest;
  }
  else { r.rest = 0.; r.mass = sum > 0. ? 1. : sum == 0. ? 0. : sum; }
  return r;
}

// A token's row is cut at the 16-byte boundaries of its address: up to V - 1 entries before the first one belong to CTA 0, those behind
// the last one to the last CTA (both kept as floats in `edge`), the vectors between are shared out evenly.
// Eight warps run over the slice; a ninth does the list's 64-bit arithmetic meanwhile.
template <class T> __global__ void __launch_bounds__(kClusterThreads, 3) distill_cluster_kernel(const __grid_constant__ DistillArgs a, uint32_t* status) {
  constexpr int V = 16 / sizeof(T);
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ float edge[2 * V], part[2], warp_max[8], shared_top, shared_factor;
  __shared__ double warp_sum[8];
  __shared__ uint64_t bar; __shared__ uint32_t abort_flag;
  __shared__ __align__(16) uint32_t hash[kHashWords];
  uint4* slice = reinterpret_cast<uint4*>(smem);
  List s(smem + a.list_at, a.k);
  const int rank = int(blockIdx.x % unsigned(a.splits)); const int64_t token = blockIdx.x / unsigned(a.splits);
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const T* z = static_cast<const T*>(a.z) + token * a.ldz;
  T* dz = a.dz ? static_cast<T*>(a.dz) + token * a.lddz : nullptr;
  const int mis = int(reinterpret_cast<uintptr_t>(z) / sizeof(T) % V), head = min((V - mis) % V, a.n), vectors = (a.n - head) / V, tail0 = head + vectors * V;
  const int v0 = int(int64_t(vectors) * rank / a.splits), v1 = int(int64_t(vectors) * (rank + 1) / a.splits);
  const bool first = rank == 0, last = rank == a.splits - 1;
  const bool same = dz && int(reinterpret_cast<uintptr_t>(dz) / sizeof(T) % V) == mis;      // gradient and logits share their alignment
  const float weight = a.weight ? a.weight[token] : 1.f;
  if (weight == 0.f) {                               // the same for the whole cluster: nobody waits
    if (first && threadIdx.x == 0) {
      if (a.loss) a.loss[token] = 0.f;
      if (a.stats_out) a.stats_out[2 * token] = a.stats_out[2 * token + 1] = __int_as_float(0x7fc00000);
    }
    if (dz) {
      if (same) for (int v = v0 + threadIdx.x; v < v1; v += kClusterThreads) *reinterpret_cast<uint4*>(dz + head + v * V) = make_uint4(0, 0, 0, 0);
      else for (int j = head + v0 * V + threadIdx.x; j < head + v1 * V; j += kClusterThreads) dz[j] = from_f32<T>(0.f);
      if (first && int(threadIdx.x) < head) dz[threadIdx.x] = from_f32<T>(0.f);
      if (last && tail0 + int(threadIdx.x) < a.n) dz[tail0 + threadIdx.x] = from_f32<T>(0.f);
    }
    return;
  }
  if (threadIdx.x == 0) {
    ptx::mbar_init(&bar, 1); abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    const uint32_t bytes = uint32_t(v1 - v0) * 16;
    ptx::mbar_expect_tx(&bar, bytes);
    for (uint32_t at = 0; at < bytes; at += 16384) ptx::bulk_load(ptx::smem_u32(smem) + at, reinterpret_cast<const uint8_t*>(z + head + v0 * V) + at, min(16384u, bytes - at), &bar);
  }
  Listed l{};
  if (warp == 8) {
    const bool twice = list_classes(a, token, s, hash);
    asm volatile("bar.arrive 2, %0;" ::"n"(kClusterThreads) : "memory");      // the classes are there
    l = list_by_warp<T>(a, token, z, s, twice);
  } else {
    if (threadIdx.x < 2 * V) {
      const int j = int(threadIdx.x) < V ? int(threadIdx.x) : tail0 + int(threadIdx.x) - V;
      const bool mine = int(threadIdx.x) < V ? first && j < head : last && j < a.n;
      edge[threadIdx.x] = mine ? to_f32(z[j]) : -INFINITY;
    }
    main_sync();
    // expired: the status word says so, the values are then undefined, and the copies get a second term before shared memory goes
    if (!ptx::mbar_wait(&bar, 0u, &abort_flag, status, 41u)) { uint32_t ignore = 0; ptx::mbar_wait(&bar, 0u, &ignore, status, 42u); }
    asm volatile("bar.sync 2, %0;" ::"n"(kClusterThreads) : "memory");        // every thread has seen the copy land, and the classes
    for (int i = threadIdx.x; i < a.k; i += kMainThreads) {  // listed classes leave the row (equal values for a class listed twice)
      const int id = s.id[i];
      if (id < 0) continue;
      if (id < head) { if (first) edge[id] = -INFINITY; }
      else if (id >= tail0) { if (last) edge[V + id - tail0] = -INFINITY; }
      else { const int v = (id - head) / V; if (v >= v0 && v < v1) reinterpret_cast<T*>(slice)[id - head - v0 * V] = from_f32<T>(-INFINITY); }
    }
    main_sync();
  }
  if (warp < 8 && !a.stats_in) {
    // maximum and sum of this slice
    RowMax<T> row_max;
    for (int v = threadIdx.x; v < v1 - v0; v += kMainThreads) row_max.add(slice[v]);
    float m = row_max.value();
    if (threadIdx.x < 2 * V) m = fmaxf(m, edge[threadIdx.x]);
    m = warp_reduce(m, Max{});
    if (lane == 0) warp_max[warp] = m;
    main_sync();
#pragma unroll
    for (int w = 0; w < 8; ++w) m = fmaxf(m, warp_max[w]);
    with_exponent(a.tau, m == -INFINITY ? 0.f : m, [&](auto e) {
      float sum = threadIdx.x < 2 * V ? e(edge[threadIdx.x]) : 0.f;
#pragma unroll 2
      for (int v = threadIdx.x; v < v1 - v0; v += kMainThreads) {
        float f[V]; unpack<T>(slice[v], f);
#pragma unroll
        for (int i = 0; i < V; ++i) f[i] = e(f[i]);
#pragma unroll
        for (int d = V / 2; d; d /= 2)
#pragma unroll
          for (int i = 0; i < d; ++i) f[i] += f[i + d];
        sum += f[0];
      }
      const double mine = warp_reduce(double(sum), Add{});
      if (lane == 0) warp_sum[warp] = mine;
      main_sync();
      if (threadIdx.x == 0) {
        double total = 0.;
#pragma unroll
        for (int w = 0; w < 8; ++w) total += warp_sum[w];
        part[0] = m; part[1] = float(total * e.fix());
      }
    });
  }
  if (a.splits > 1) { __syncwarp(); cluster_arrive(); cluster_wait(); }      // also: every CTA has read the listed logits, the gradient may go in their place
  else __syncthreads();
  if (warp == 8) {
    float top, outside;
    if (a.stats_in) { top = a.stats_in[2 * token]; outside = a.stats_in[2 * token + 1]; }
    else {
      // one CTA's part per lane
      const float pm = lane >= a.splits ? -INFINITY : a.splits > 1 ? ld_cluster(&part[0], lane) : part[0];
      const float ps = lane >= a.splits ? 0.f : a.splits > 1 ? ld_cluster(&part[1], lane) : part[1];
      top = warp_reduce(pm, Max{});
      if (top == -INFINITY) top = 0.f;
      const double scale = double(float(1.4426950408889634 * a.inv_tau));
      // a part without a maximum holds nothing, or nothing but NaNs: its sum says which
      const double share = pm == -INFINITY || pm == top ? double(ps) : double(ps) * exp2((double(pm) - double(top)) * scale);
      outside = float(warp_reduce(share, Add{}));
    }
    const Student st(a, l, top, outside);
    if (lane == 0) with_exponent(a.tau, top, [&](auto e) { shared_top = top; shared_factor = float(outside_factor(a, l, st, outside, weight) * e.fix()); });
    __syncthreads();
    if (a.splits > 1) cluster_arrive();              // peers may leave once everybody has read
    if (first && (a.loss || a.stats_out)) {
      const double log_total = log(st.total);
      const double kl = warp_reduce(listed_loss(a, s, st, log_total, lane, 32), Add{}) + outside_loss(a, l, st, log_total, top, outside);
      if (lane == 0) {
        if (a.loss) a.loss[token] = float(kl * weight);
        if (a.stats_out) { a.stats_out[2 * token] = top; a.stats_out[2 * token + 1] = outside; }
      }
    }
    if (dz) {
      for (int i = lane; i < a.k; i += 32) if (s.first[i]) s.psum[i] = double(listed_gradient(a, s, l, st, weight, i));
      __syncthreads();                               // the listed classes are written last
      for (int i = lane; i < a.k; i += 32) {
        const int id = s.id[i];
        if (!s.first[i]) continue;
        const bool mine = id < head ? first : id >= tail0 ? last : (id - head) / V >= v0 && (id - head) / V < v1;
        if (mine) dz[id] = from_f32<T>(float(s.psum[i]));
      }
    }
  } else {
    __syncthreads();
    if (a.splits > 1) cluster_arrive();
    if (dz) {
      const float factor = shared_factor;
      with_exponent(a.tau, shared_top, [&](auto e) {
#pragma unroll 2
        for (int v = threadIdx.x; v < v1 - v0; v += kMainThreads) {
          float f[V]; unpack<T>(slice[v], f);
#pragma unroll
          for (int i = 0; i < V; ++i) f[i] = factor * e(f[i]);
          T* to = dz + head + (v0 + v) * V;
          if (same) __stcs(reinterpret_cast<uint4*>(to), pack<T>(f));
          else
#pragma unroll
            for (int i = 0; i < V; ++i) to[i] = from_f32<T>(f[i]);
        }
        if (threadIdx.x < 2 * V) {
          const int j = int(threadIdx.x) < V ? int(threadIdx.x) : tail0 + int(threadIdx.x) - V;
          if (int(threadIdx.x) < V ? first && j < head : last && j < a.n) dz[j] = from_f32<T>(factor * e(edge[threadIdx.x]));
        }
      });
      __syncthreads();
    }
  }
  if (a.splits > 1) cluster_wait();
}

// Slices of at most 72 KiB where eight CTAs allow it, otherwise what one CTA per SM takes.  With the list and 8 KiB of tables three CTAs fit
// an SM up to slices of some 64 KiB and two beyond, which still beat three or four of half the slice, whose phases are as long: 512
// x 131072 bfloat16 (64 KiB) 96 us, in twice the CTAs 113; 1024 x 32768 (64 KiB) 49 against 56; 1024 x 36000 (70 KiB) 51 against 58.
constexpr int kSliceBytes = 72 * 1024, kSmemMost = 216 * 1024;

template <class T> cudaError_t raise_limit(const hyacinHandle_t* handle, T* kernel, std::atomic<uint64_t>& ready) {
  const uint64_t bit = uint64_t(1) << (handle->DeviceID & 63);      // per device
  if (ready.load() & bit) return cudaSuccess;
  const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmemMost);
  if (e == cudaSuccess) ready.fetch_or(bit);
  return e;
}

int32_t launch_distill(const char* fn, const hyacinHandle_t* handle, hyacinPrecision_t type, DistillArgs a) {
  const int64_t row = int64_t(a.n) * int64_t(w4_type_bytes(type)) + 16;
  int splits = 1;
  while (splits < 8 && (row + splits - 1) / splits > kSliceBytes) splits *= 2;
  cudaError_t e = cudaSuccess;
  count_launch();
  const int64_t slice = ((row / 16 + splits - 1) / splits + 1) * 16;
  if (slice + int64_t(list_bytes(a.k)) <= kSmemMost && int64_t(a.t) * splits <= 0x7fffffff) {
    a.splits = splits; a.list_at = int(slice);
    const size_t smem = size_t(slice) + list_bytes(a.k);
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(unsigned(a.t) * splits); cfg.blockDim = dim3(kClusterThreads); cfg.dynamicSmemBytes = smem; cfg.stream = handle->cudaStream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension; attr[0].val.clusterDim.x = splits; attr[0].val.clusterDim.y = 1; attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr; cfg.numAttrs = splits > 1 ? 1 : 0;
    uint32_t* status = status_word_device(handle->DeviceID);
    with_w4_type(type, [&](auto tag) {
      auto* kernel = distill_cluster_kernel<decltype(tag)>;
      static std::atomic<uint64_t> ready{0};
      e = raise_limit(handle, kernel, ready);
      if (e == cudaSuccess) e = cudaLaunchKernelEx(&cfg, kernel, a, status);
    });
  } else {
    const size_t smem = (list_bytes(a.k) + 15) / 16 * 16 + size_t((a.n + 31) / 32) * 4;
    with_w4_type(type, [&](auto tag) {
      auto* kernel = distill_plain_kernel<decltype(tag)>;
      static std::atomic<uint64_t> ready{0};
      e = raise_limit(handle, kernel, ready);
      if (e == cudaSuccess) e = w4_start(kernel, dim3(unsigned(std::min(a.t, 1 << 20))), 512, smem, handle->cudaStream, a);
    });
  }
  return w4_result(e, fn);
}

int32_t check_distill(const char* fn, const hyacinHandle_t* handle, hyacinPrecision_t type, const DistillArgs& a) {
  if (!handle) return w4_refuse(fn, "no handle");
  if (!is_w4_type(type)) return w4_refuse(fn, "type not supported");
  if (a.n < 1 || a.t < 0 || a.k < 0 || a.k > kMaxList || a.n > kMaxClasses) return w4_refuse(fn, "sizes: 1 <= N <= 2^20, T >= 0, 0 <= K <= 1024");
  if (!(a.tau >= 1e-30 && a.tau <= 1e30)) return w4_refuse(fn, "tau must lie in [1e-30, 1e30]");
  if (a.t == 0) return 1;
  if (!a.z || a.ldz < a.n) return w4_refuse(fn, "Z: null or leading dimension too small");
  if (a.k > 0 && (!a.ids || !a.teacher || a.ldk < a.k)) return w4_refuse(fn, "ids, teacher: null or leading dimension too small");
  if (a.dz && a.lddz < a.n) return w4_refuse(fn, "dZ: leading dimension too small");
  if (a.dz == a.z && a.lddz != a.ldz) return w4_refuse(fn, "dZ in place of Z needs the same leading dimension");
  if (!w4_on_boundary(w4_type_bytes(type), a.z, a.dz) || !w4_on_boundary(4, a.ids, a.teacher, a.teacher_lse, a.weight, a.loss, a.stats_out, a.stats_in))
    return w4_refuse(fn, "a pointer that is not on a boundary of its type");
  if (w4_refuse_handle(fn, handle)) return -1;
  return 0;
}

}  // namespace
}  // namespace hyb

extern "C" int32_t hyacinB200DistillLoss(const hyacinHandle_t* handle, hyacinPrecision_t Ztype, int32_t N, int32_t T, const void* Z,
                                         int32_t ldz, int32_t K, const int32_t* ids, const float* teacher, int32_t ldk, double tau,
                                         const float* teacherLse, const float* weight, float* loss, float* stats, void* dZ, int32_t lddz) {
  using namespace hyb;
  const char* fn = "hyacinB200DistillLoss";
  DistillArgs a{Z, ldz, N, T, K, ids, teacher, ldk, tau, 1. / tau, teacherLse, weight, loss, stats, nullptr, dZ, lddz, 1, 0};
  const int32_t rc = check_distill(fn, handle, Ztype, a);
  if (rc) return rc < 0 ? rc : 0;
  if (!loss && !stats && !dZ) return 0;
  timer_mark(handle, Segment::Replicated);
  return launch_distill(fn, handle, Ztype, a);
}

extern "C" int32_t hyacinB200DistillGrad(const hyacinHandle_t* handle, hyacinPrecision_t Ztype, int32_t N, int32_t T, const void* Z,
                                         int32_t ldz, int32_t K, const int32_t* ids, const float* teacher, int32_t ldk, double tau,
                                         const float* teacherLse, const float* weight, const float* stats, void* dZ, int32_t lddz) {
  using namespace hyb;
  const char* fn = "hyacinB200DistillGrad";
  DistillArgs a{Z, ldz, N, T, K, ids, teacher, ldk, tau, 1. / tau, teacherLse, weight, nullptr, nullptr, stats, dZ, lddz, 1, 0};
  const int32_t rc = check_distill(fn, handle, Ztype, a);
  if (rc) return rc < 0 ? rc : 0;
  if (!stats || !dZ) return w4_refuse(fn, "null pointer");
  timer_mark(handle, Segment::Replicated);
  return launch_distill(fn, handle, Ztype, a);
}
