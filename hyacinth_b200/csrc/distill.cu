// Distillation loss against a teacher's top logits, and its gradient.
//
// Per token, with u = z / tau and the list i = 1 .. K of classes c_i with teacher logits t_i:
//     p_i = exp(t_i / tau - teacherLse), p_r = max(0, 1 - sum p)   or, without teacherLse, p_i = softmax over the list, p_r = 0
//     lse = log sum_j exp u_j,  lse_r = log sum over the classes outside the list
//     KL  = sum_i p_i (log p_i - (u_{c_i} - lse)) + p_r (log p_r - (lse_r - lse))
//     dKL/dz_j = (q_j mass - P_j) / tau                        listed: P_j = sum of its p_i, mass = sum p + p_r
//     dKL/dz_j = exp(u_j - lse_r) (mass exp(lse_r - lse) - p_r) / tau    outside the list
// The sum over the classes outside is accumulated without the listed ones, so p_r / q_r never comes from a difference, and
// what concerns the list (K terms) is done in 64 bits: where student and teacher agree, q - p is the difference of two numbers
// close to one.
#include "w4.cuh"
#include <algorithm>

namespace hyb {
namespace {

constexpr int kMaxList = 1024;
constexpr int kMaxClasses = 1 << 20;
constexpr float kLog2e = 1.4426950408889634f;

struct DistillArgs {
  const void* z; int64_t ldz; int n, t, k;
  const int32_t* ids; const float* teacher; int64_t ldk; double tau;
  const float* teacher_lse; const float* weight;
  float* loss; float* stats_out; const float* stats_in;
  void* dz; int64_t lddz;
};

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

// The list of one token in shared memory.
struct List {
  double p[kMaxList];        // teacher probability
  double logp[kMaxList];
  double psum[kMaxList];     // sum over the entries of the same class, at the first of them
  float z[kMaxList];         // student logit
  int id[kMaxList];          // class, -1 when skipped
  int first[kMaxList];       // 1: first entry of its class
  double buf[32]; float fbuf[32];
};

// Reads the list; returns p_r and the mass.  Ends with a barrier.
template <class T> __device__ void load_list(const DistillArgs& a, int64_t token, const T* z, List& s, double& rest, double& mass) {
  double top = -INFINITY;
  for (int i = threadIdx.x; i < a.k; i += blockDim.x) {
    const int id = a.ids[token * a.ldk + i];
    const bool ok = id >= 0 && id < a.n;
    s.id[i] = ok ? id : -1;
    const double t = ok ? double(a.teacher[token * a.ldk + i]) / a.tau : -INFINITY;
    s.logp[i] = t; s.z[i] = ok ? to_f32(z[id]) : 0.f;
    top = fmax(top, t);
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
  for (int i = threadIdx.x; i < a.k; i += blockDim.x) {
    int first = s.id[i] >= 0; double ps = 0.;
    for (int j = 0; j < a.k; ++j) if (s.id[j] == s.id[i]) { ps += s.p[j]; if (j < i) first = 0; }
    s.first[i] = first; s.psum[i] = ps;
  }
  rest = a.teacher_lse ? fmax(0., 1. - sum) : 0.;
  mass = sum + rest;
  __syncthreads();
}

// Plain form: one block per token, two passes over the logits, a bit per class for the list.
// Mode: loss from this pass's sums, or gradient from saved ones.
template <class T> __global__ void __launch_bounds__(512) distill_plain_kernel(DistillArgs a) {
  extern __shared__ uint32_t listed[];
  __shared__ List s;
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
    double rest, mass;
    load_list<T>(a, token, z, s, rest, mass);
    for (int i = threadIdx.x; i < a.k; i += blockDim.x) if (s.id[i] >= 0) atomicOr(&listed[s.id[i] >> 5], 1u << (s.id[i] & 31));
    __syncthreads();
    const float scale = kLog2e / float(a.tau);
    float top, outside;
    if (a.stats_in) { top = a.stats_in[2 * token]; outside = a.stats_in[2 * token + 1]; }
    else {
      top = -INFINITY;
      for (int j = threadIdx.x; j < a.n; j += blockDim.x) if (!(listed[j >> 5] >> (j & 31) & 1)) top = fmaxf(top, to_f32(z[j]));
      top = block_reduce(top, Max{}, s.fbuf);
      if (top == -INFINITY) top = 0.f;
      double sum = 0.;
      for (int j = threadIdx.x; j < a.n; j += blockDim.x) if (!(listed[j >> 5] >> (j & 31) & 1)) sum += exp2f((to_f32(z[j]) - top) * scale);
      outside = float(block_reduce(sum, Add{}, s.buf));
    }
    // log-sum-exps in 64 bits, relative to the larger of the two maxima
    double ltop = -INFINITY;
    for (int i = threadIdx.x; i < a.k; i += blockDim.x) if (s.id[i] >= 0) ltop = fmax(ltop, double(s.z[i]) / a.tau);
    ltop = block_reduce(ltop, Max{}, s.buf);
    const double lse_out = log(double(outside)) + double(top) / a.tau;
    double ref = fmax(ltop, lse_out);
    if (ref == -INFINITY) ref = 0.;
    double e = 0.;
    for (int i = threadIdx.x; i < a.k; i += blockDim.x) if (s.first[i]) e += exp(double(s.z[i]) / a.tau - ref);
    const double total = block_reduce(e, Add{}, s.buf) + (outside == 0.f ? 0. : exp(lse_out - ref));
    const double lse = ref + log(total);
    if (a.loss || a.stats_out) {
      double kl = 0.;
      for (int i = threadIdx.x; i < a.k; i += blockDim.x) if (s.p[i] != 0.) kl += s.p[i] * (s.logp[i] - (total == 0. ? -INFINITY : double(s.z[i]) / a.tau - lse));
      kl = block_reduce(kl, Add{}, s.buf);
      if (rest > 0.) kl += rest * (log(rest) - (outside == 0.f ? -INFINITY : lse_out - lse));
      if (threadIdx.x == 0) {
        if (a.loss) a.loss[token] = float(kl * weight);
        if (a.stats_out) { a.stats_out[2 * token] = top; a.stats_out[2 * token + 1] = outside; }
      }
    }
    if (dz) {
      const double w = double(weight) / a.tau;
      const float factor = outside == 0.f ? 0.f : float(w * (mass * exp(double(top) / a.tau - lse) - rest / double(outside)));
      for (int j = threadIdx.x; j < a.n; j += blockDim.x)
        if (!(listed[j >> 5] >> (j & 31) & 1)) dz[j] = from_f32<T>(factor * exp2f((to_f32(z[j]) - top) * scale));
      for (int i = threadIdx.x; i < a.k; i += blockDim.x)
        if (s.first[i]) dz[s.id[i]] = from_f32<T>(float(w * (mass * (total == 0. ? 0. : exp(double(s.z[i]) / a.tau - lse)) - s.psum[i])));
    }
  }
}

int32_t launch_distill(const char* fn, const hyacinHandle_t* handle, hyacinPrecision_t type, const DistillArgs& a) {
  const size_t bits = size_t((a.n + 31) / 32) * 4;
  int32_t rc = 0;
  with_w4_type(type, [&](auto tag) {
    auto* kernel = distill_plain_kernel<decltype(tag)>;
    if (bits > 8192) {
      const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kMaxClasses / 8);
      if (e != cudaSuccess) { report_cuda_error(e, "cudaFuncSetAttribute", __FILE__, __LINE__); rc = -3; return; }
    }
    count_launch();
    kernel<<<unsigned(std::min(a.t, 1 << 20)), 512, bits, handle->cudaStream>>>(a);
    rc = w4_launched(fn);
  });
  return rc;
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
  if (!w4_device_ok(handle)) return w4_refuse(fn, "the handle belongs to another device than the current one");
  return 0;
}

}  // namespace
}  // namespace hyb

extern "C" int32_t hyacinB200DistillLoss(const hyacinHandle_t* handle, hyacinPrecision_t Ztype, int32_t N, int32_t T, const void* Z,
                                         int32_t ldz, int32_t K, const int32_t* ids, const float* teacher, int32_t ldk, double tau,
                                         const float* teacherLse, const float* weight, float* loss, float* stats, void* dZ, int32_t lddz) {
  using namespace hyb;
  const char* fn = "hyacinB200DistillLoss";
  DistillArgs a{Z, ldz, N, T, K, ids, teacher, ldk, tau, teacherLse, weight, loss, stats, nullptr, dZ, lddz};
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
  DistillArgs a{Z, ldz, N, T, K, ids, teacher, ldk, tau, teacherLse, weight, nullptr, nullptr, stats, dZ, lddz};
  const int32_t rc = check_distill(fn, handle, Ztype, a);
  if (rc) return rc < 0 ? rc : 0;
  if (!stats || !dZ) return w4_refuse(fn, "null pointer");
  timer_mark(handle, Segment::Replicated);
  return launch_distill(fn, handle, Ztype, a);
}
