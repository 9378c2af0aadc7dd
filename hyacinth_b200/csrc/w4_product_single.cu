// Products with a 4-bit weight matrix in single precision where the streaming kernel does not serve: opW 'N', many vectors, very long x.
//
// Y (out x T) = A X, A = Wq^T or Wq, in 32 bits throughout: scale times code (or, for few vectors, scale times x) is rounded to 32 bits, then the
// sums.  A block of 128 threads computes 128 outputs x TOK vectors: steps of 32 along the sum
// bring the dequantised weights and x to shared memory as floats, a thread holds 8 x TOK / 8 sums.  A step's sums start from
// zero and are then added to the total, so no term passes through more than 32 + K / 32 additions.  The next step's words are on their way
// in registers meanwhile.  The correction V (U^T X) is more steps of the same sum with mid = U^T X as x, and mid itself the same
// kernel over a plain matrix.  Few tiles: a cluster of up to 8 blocks splits the steps, sums joined in a fixed order.
// Bound: the floating-point pipe, 128 multiply-adds per clock and SM (72 TFLOP/s at 1.9 GHz), and shared memory beside it: four 16-byte loads, sixteen
// wavefronts, per 64 multiply-adds of a warp.  8 x 8 sums per thread need half the loads of 8 x 4 (276 -> 236 us below); two blocks per SM
// leave eight warps to cover what remains: 32 % of the multiply pipe and 43 % of the issue slots for 256 vectors.  Measured, 4096 x 4096 with
// segments of 64 rows: opW 'N', 16 vectors 37 us, 32 44 us, 64 63 us, 256 234 us (37 TFLOP/s); opW 'T', 16 vectors 42 us, 256 255 us;
// 200 x 32768 times 32, opW 'N' (two tiles, 1024 steps) 45 us, 263 without the second split.  The kernel for few vectors would take two
// passes of 21 us for eight, where this one takes 36.
#include "w4_product.h"
#include <algorithm>

namespace hyb {
namespace {

constexpr int kOut = 128, kStep = 32, kThreads = 128, kPitch = kOut + 4;
enum Mode { kCodesT, kCodesN, kDense };           // weights: Wq^T, Wq, or the transpose of a plain matrix

struct SingleArgs {
  const uint8_t* codes; int64_t ldq; const float* scales; const uint8_t* zeros; int64_t lds;
  int m, n, seg, in, out, t;
  const float* x; int64_t ldx;
  int rank; const float* second; int64_t ld2; const float* mid;          // second: also the plain matrix
  float* y; int64_t ldy;
  int code_steps, steps, splits, parts, x_aligned;      // splits: blocks of a cluster, parts: clusters that share a tile's steps
  float* scratch;                                 // a part's share of Y, [part][vector][output]
};

__device__ __forceinline__ float4 ld_cluster4(const float* at, uint32_t rank) {
  uint32_t remote; float4 v;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(remote) : "r"(uint32_t(__cvta_generic_to_shared(at))), "r"(rank));
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(remote) : "memory");
  return v;
}
__device__ __forceinline__ void cluster_sync_all() {
  asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
  asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}

// Loads that stay where they are written: left to the compiler, those for the next step moved behind the arithmetic that they are to overlap.
__device__ __forceinline__ uint32_t now(const uint32_t* p) { uint32_t v; asm volatile("ld.global.nc.u32 %0, [%1];" : "=r"(v) : "l"(p)); return v; }
__device__ __forceinline__ float now(const float* p) { float v; asm volatile("ld.global.nc.f32 %0, [%1];" : "=f"(v) : "l"(p)); return v; }
__device__ __forceinline__ int now(const uint8_t* p) { uint16_t v; asm volatile("ld.global.nc.u8 %0, [%1];" : "=h"(v) : "l"(p)); return v; }
__device__ __forceinline__ float4 now(const float4* p) { float4 v; asm volatile("ld.global.nc.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "l"(p)); return v; }
// q - zero of row e of a word, exact: 2^23 + q from the bits, less 2^23 + zero
__device__ __forceinline__ float code(uint32_t word, int e, float offset) { return __uint_as_float(((word >> (4 * w4_row_nibble(e))) & 15u) | 0x4b000000u) - offset; }
// Two sums at once: one instruction of the packed form does the work of two, and the scalar ones do not fill the pipe.
struct Two { uint64_t v; };
__device__ __forceinline__ Two two(float lo, float hi) { Two r; asm("mov.b64 %0, {%1, %2};" : "=l"(r.v) : "f"(lo), "f"(hi)); return r; }
__device__ __forceinline__ float2 unpack(Two t) { float2 r; asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(t.v)); return r; }
__device__ __forceinline__ Two fma2(Two a, Two b, Two c) { Two r; asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r.v) : "l"(a.v), "l"(b.v), "l"(c.v)); return r; }
__device__ __forceinline__ Two add2(Two a, Two b) { Two r; asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v)); return r; }
__device__ __forceinline__ Two mul2(Two a, Two b) { Two r; asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v)); return r; }

template <Mode MODE, int TOK> __global__ void __launch_bounds__(kThreads, 2) product_single_kernel(const __grid_constant__ SingleArgs a) {
  constexpr int kTok = TOK / 8, kXPitch = TOK + 4, kXPer = kStep * TOK / kThreads;       // sums of a thread along the vectors; values of x it brings
  constexpr int kTiles = kStep * kPitch + kStep * kXPitch, kSums = TOK * kOut;
  __shared__ __align__(16) float smem[kTiles > kSums ? kTiles : kSums];
  float* ws = smem;                                // [k][output]
  float* xs = smem + kStep * kPitch;               // [k][vector]
  const int tid = threadIdx.x, split = blockIdx.x % a.splits, out0 = blockIdx.x / a.splits * kOut;
  const int piece = int(blockIdx.z) * a.splits + split, pieces = a.parts * a.splits;
  const int step0 = int(int64_t(a.steps) * piece / pieces), step1 = int(int64_t(a.steps) * (piece + 1) / pieces);
  float* y = a.parts > 1 ? a.scratch + int64_t(blockIdx.z) * a.t * a.out : a.y;
  const int64_t ldy = a.parts > 1 ? a.out : a.ldy;
  const int o = tid;                               // output that this thread brings ('T', plain, correction)
  const int word = tid & 15, lane = tid >> 4;      // 'N': word of the block, column modulo 8
  const int xt = tid % TOK, xk = tid / TOK * kXPer;
  for (int64_t t0 = int64_t(blockIdx.y) * TOK; t0 < a.t; t0 += int64_t(gridDim.y) * TOK) {
    Two total[4][kTok] = {};
    uint32_t q[4] = {}; float s[4] = {}; int zero[4] = {}; float xv[kXPer];
    auto fetch = [&](int k) {
      const bool more = k >= a.code_steps;         // a step of the correction
      const int k0 = (more ? k - a.code_steps : k) * kStep, length = more ? a.rank : a.in;
      if (more || MODE == kDense) {                // few of these: read when they are stored
      } else if (MODE == kCodesT) {
        const int col = min(out0 + o, a.n - 1), sub = k, seg = k0 / a.seg;
        const uint8_t* from = a.codes + col * a.ldq + int64_t(sub >> 2) * 64 + (sub & 3) * 4;
#pragma unroll
        for (int u = 0; u < 4; ++u) q[u] = now(reinterpret_cast<const uint32_t*>(from + 16 * u));
        s[0] = now(a.scales + col * a.lds + seg); zero[0] = a.zeros ? now(a.zeros + col * a.lds + seg) : 8;
      } else {
        const int seg = min(out0 + w4_word_row(word), a.m - 1) / a.seg;
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          const int col = min(k0 + lane + 8 * u, a.n - 1);                  // behind the last column x is zero and the weights are not used
          q[u] = now(reinterpret_cast<const uint32_t*>(a.codes + col * a.ldq + int64_t(out0 / kOut) * 64 + word * 4));
          s[u] = now(a.scales + col * a.lds + seg); zero[u] = a.zeros ? now(a.zeros + col * a.lds + seg) : 8;
        }
      }
      const float* x = more ? a.mid : a.x; const int64_t ldx = more ? a.rank : a.ldx;
      const float* from = x + (t0 + xt) * ldx + k0 + xk;
      const bool there = t0 + xt < a.t;
      if (!more && a.x_aligned && there && kXPer % 4 == 0 && k0 + xk + kXPer <= length) {
#pragma unroll
        for (int i = 0; i < kXPer / 4; ++i) { const float4 v = now(reinterpret_cast<const float4*>(from) + i); xv[4 * i] = v.x; xv[4 * i + 1] = v.y; xv[4 * i + 2] = v.z; xv[4 * i + 3] = v.w; }
      } else {
#pragma unroll
        for (int i = 0; i < kXPer; ++i) xv[i] = there && k0 + xk + i < length ? now(from + i) : 0.f;
      }
    };
    auto store = [&](int k) {
      const bool more = k >= a.code_steps;
      const int k0 = (more ? k - a.code_steps : k) * kStep, length = more ? a.rank : a.in;
      float offset[4];
#pragma unroll
      for (int u = 0; u < 4; ++u) offset[u] = 8388608.f + float(zero[MODE == kCodesT ? 0 : u]);
      if (more || MODE == kDense) {
        const float* from = more ? a.second + k0 * a.ld2 + out0 + o : a.second + (out0 + o) * a.ld2 + k0;
        const int64_t pitch = more ? a.ld2 : 1;
#pragma unroll 16
        for (int r = 0; r < kStep; ++r) ws[r * kPitch + o] = k0 + r < length && out0 + o < a.out ? __ldg(from + r * pitch) : 0.f;
      } else if (MODE == kCodesT) {
        // rows behind the last one: whatever scale and codes say there, it is not multiplied
#pragma unroll
        for (int u = 0; u < 4; ++u)
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const int r = 8 * u + e;
            ws[r * kPitch + o] = k0 + r < a.in ? s[0] * code(q[u], e, offset[0]) : 0.f;
          }
      } else {
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          float w[8];
#pragma unroll
          for (int e = 0; e < 8; ++e) w[e] = k0 + lane + 8 * u < a.in ? s[u] * code(q[u], e, offset[u]) : 0.f;
          float4* to = reinterpret_cast<float4*>(ws + (lane + 8 * u) * kPitch + w4_word_row(word));
          to[0] = make_float4(w[0], w[1], w[2], w[3]); to[1] = make_float4(w[4], w[5], w[6], w[7]);
        }
      }
#pragma unroll
      for (int i = 0; i < kXPer; ++i) xs[(xk + i) * kXPitch + xt] = xv[i];
    };
    // outputs 4 ox .. + 3 and 64 + 4 ox .. + 3, vectors kTok og .. + kTok - 1
    const int ox = tid & 15, og = tid >> 4;
    if (step0 < step1) fetch(step0);
    for (int k = step0; k < step1; ++k) {
      __syncthreads();
      store(k);
      __syncthreads();
      if (k + 1 < step1) fetch(k + 1);
      Two sum[4][kTok];
#pragma unroll
      for (int r = 0; r < kStep; ++r) {
        const ulonglong2 w0 = *reinterpret_cast<const ulonglong2*>(ws + r * kPitch + 4 * ox), w1 = *reinterpret_cast<const ulonglong2*>(ws + r * kPitch + 64 + 4 * ox);
        const Two w[4] = {{w0.x}, {w0.y}, {w1.x}, {w1.y}};
        Two x[kTok];
        if constexpr (kTok % 4 == 0) {
#pragma unroll
          for (int j = 0; j < kTok; j += 4) {
            const float4 v = *reinterpret_cast<const float4*>(xs + r * kXPitch + kTok * og + j);
            x[j] = two(v.x, v.x); x[j + 1] = two(v.y, v.y); x[j + 2] = two(v.z, v.z); x[j + 3] = two(v.w, v.w);
          }
        } else {
          const float2 v = *reinterpret_cast<const float2*>(xs + r * kXPitch + kTok * og);
          x[0] = two(v.x, v.x); x[1] = two(v.y, v.y);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int j = 0; j < kTok; ++j) sum[i][j] = r == 0 ? mul2(w[i], x[j]) : fma2(w[i], x[j], sum[i][j]);
      }
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < kTok; ++j) total[i][j] = add2(total[i][j], sum[i][j]);
    }
    if (a.splits == 1) {
#pragma unroll
      for (int j = 0; j < kTok; ++j)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int out = out0 + 64 * (i >> 1) + 4 * ox + 2 * (i & 1); const int64_t t = t0 + kTok * og + j;
          const float2 v = unpack(total[i][j]);
          if (out < a.out && t < a.t) y[t * ldy + out] = v.x;
          if (out + 1 < a.out && t < a.t) y[t * ldy + out + 1] = v.y;
        }
      continue;
    }
    __syncthreads();                               // the tiles are read; the sums take their place, [vector][output]
#pragma unroll
    for (int j = 0; j < kTok; ++j)
#pragma unroll
      for (int h = 0; h < 2; ++h)
        *reinterpret_cast<ulonglong2*>(smem + (kTok * og + j) * kOut + 64 * h + 4 * ox) = make_ulonglong2(total[2 * h][j].v, total[2 * h + 1][j].v);
    cluster_sync_all();
    const int share = kSums / 4 / a.splits;
    for (int e = split * share + tid; e < (split + 1) * share; e += kThreads) {
      float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
      for (int c = 0; c < a.splits; ++c) { const float4 p = ld_cluster4(smem + 4 * e, c); v.x += p.x; v.y += p.y; v.z += p.z; v.w += p.w; }
      const int out = out0 + 4 * e % kOut; const int64_t t = t0 + 4 * e / kOut;
      if (t >= a.t) continue;
      const float p[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
      for (int i = 0; i < 4; ++i) if (out + i < a.out) y[t * ldy + out + i] = p[i];
    }
    cluster_sync_all();                            // shared memory stays until every peer has read it
  }
}

// Few vectors, opW 'N': a block of 256 threads takes 128 rows, thread (word, lane) the eight rows of a word in every 16th column, for up to
// four vectors; x times the scale is formed once per word.  A cluster of up to eight such blocks splits the columns; sums meet
// in shared memory, in a fixed order.
// Bound: the latency of plain loads, one scale and up to four x for each word, four columns of a thread in flight; 35 % of the issue slots
// and 19 % of the multiply pipe are used.  4096 x 4096, one vector 21 us, four 22.
constexpr int kFew = 4, kFewLanes = 16, kFewThreads = 16 * kFewLanes;
__device__ __forceinline__ float ld_cluster(const float* at, uint32_t rank) {
  uint32_t remote; float v;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(remote) : "r"(uint32_t(__cvta_generic_to_shared(at))), "r"(rank));
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(remote) : "memory");
  return v;
}
__global__ void __launch_bounds__(kFewThreads) product_few_kernel(const __grid_constant__ SingleArgs a) {
  __shared__ float red[kFew][8][16][kFewLanes + 1], sum[kFew][kW4Block];
  const int word = threadIdx.x & 15, lane = threadIdx.x >> 4, split = blockIdx.x % a.splits, block = blockIdx.x / a.splits;
  const int row = block * kW4Block + w4_word_row(word), seg = min(row, a.m - 1) / a.seg;
  const int j0 = int(int64_t(a.n) * split / a.splits), j1 = int(int64_t(a.n) * (split + 1) / a.splits);
  const float* x = a.x;
  const float* scales = a.scales + seg;
  const uint8_t* zeros = a.zeros ? a.zeros + seg : nullptr;
  const uint8_t* codes = a.codes + int64_t(block) * 64 + word * 4;
  float acc[kFew][8] = {};
#pragma unroll 4
  for (int j = j0 + lane; j < j1; j += kFewLanes) {
    const uint32_t q = __ldg(reinterpret_cast<const uint32_t*>(codes + j * a.ldq));
    const float s = scales[j * a.lds], offset = 8388608.f + float(zeros ? int(zeros[j * a.lds]) : 8);
    float xs[kFew], w[8];
#pragma unroll
    for (int t = 0; t < kFew; ++t) xs[t] = t < a.t ? s * x[t * a.ldx + j] : 0.f;
#pragma unroll
    for (int e = 0; e < 8; ++e) w[e] = __uint_as_float(((q >> (4 * w4_row_nibble(e))) & 15u) | 0x4b000000u) - offset;      // 2^23 + q, exact
#pragma unroll
    for (int t = 0; t < kFew; ++t)
#pragma unroll
      for (int e = 0; e < 8; ++e) acc[t][e] += w[e] * xs[t];
  }
#pragma unroll
  for (int t = 0; t < kFew; ++t)
#pragma unroll
    for (int e = 0; e < 8; ++e) red[t][e][word][lane] = acc[t][e];
  __syncthreads();
  for (int i = threadIdx.x; i < kFew * kW4Block; i += kFewThreads) {
    const int t = i / kW4Block, r = i % kW4Block, e = r & 7, w = r >> 3;
    float v = 0.f;
#pragma unroll
    for (int l = 0; l < kFewLanes; ++l) v += red[t][e][w][l];
    sum[t][w4_word_row(w) + e] = v;
  }
  if (a.splits > 1) cluster_sync_all(); else __syncthreads();
  const int share = kW4Block / a.splits;
  for (int i = threadIdx.x; i < kFew * share; i += kFewThreads) {
    const int t = i / share, local = split * share + i % share, out = block * kW4Block + local;
    if (out >= a.m || t >= a.t) continue;
    float v = 0.f;
    for (int c = 0; c < a.splits; ++c) v += a.splits > 1 ? ld_cluster(&sum[t][local], c) : sum[t][local];
    for (int k = 0; k < a.rank; ++k) v += a.second[k * a.ld2 + out] * a.mid[t * a.rank + k];
    a.y[t * a.ldy + out] = v;
  }
  if (a.splits > 1) cluster_sync_all();            // shared memory stays until every peer has read it
}

// Y = the sum of the parts, in their order.
__global__ void __launch_bounds__(256) join_kernel(const float* scratch, int parts, int out, int t, float* y, int64_t ldy) {
  const int64_t size = int64_t(out) * t, e = int64_t(blockIdx.x) * 256 + threadIdx.x;
  if (e >= size) return;
  float v = 0.f;
#pragma unroll 8
  for (int p = 0; p < parts; ++p) v += scratch[p * size + e];
  y[e / out * ldy + e % out] = v;
}

template <Mode MODE, int TOK> cudaError_t start(const hyacinHandle_t* handle, SingleArgs a) {
  a.code_steps = int((int64_t(a.in) + kStep - 1) / kStep); a.steps = a.code_steps + (a.rank + kStep - 1) / kStep;
  const int64_t tiles = (int64_t(a.out) + kOut - 1) / kOut, groups = std::min<int64_t>((int64_t(a.t) + TOK - 1) / TOK, 65535);
  // two blocks fit an SM; at least four steps for each block.  Where a cluster of eight leaves most of the GPU idle several share a tile
  // and a second kernel adds their shares (200 x 32768 times 32, opW 'N': 263 us without).
  a.splits = a.parts = 1;
  while (a.splits < 8 && tiles * groups * a.splits * 2 <= 2 * int64_t(handle->DeviceSMs) && a.steps >= 8 * a.splits) a.splits *= 2;
  if (a.splits == 8) a.parts = int(std::max<int64_t>(1, std::min<int64_t>({2 * int64_t(handle->DeviceSMs) / (tiles * groups * 8), a.steps / 32, 64})));
  a.x_aligned = reinterpret_cast<uintptr_t>(a.x) % 16 == 0 && a.ldx % 4 == 0;
  if (a.parts > 1) {
    const cudaError_t e = cudaMallocFromPoolAsync(reinterpret_cast<void**>(&a.scratch), size_t(a.parts) * a.t * a.out * sizeof(float), handle->mempool, handle->cudaStream);
    if (e != cudaSuccess) return e;
  }
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(unsigned(tiles * a.splits), unsigned(groups), unsigned(a.parts)); cfg.blockDim = dim3(kThreads); cfg.stream = handle->cudaStream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension; attr[0].val.clusterDim.x = a.splits; attr[0].val.clusterDim.y = 1; attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr; cfg.numAttrs = a.splits > 1 ? 1 : 0;
  count_launch();
  cudaError_t e = cudaLaunchKernelEx(&cfg, product_single_kernel<MODE, TOK>, a);
  if (a.parts > 1) {
    if (e == cudaSuccess) {
      count_launch();
      e = w4_start(join_kernel, dim3(unsigned((int64_t(a.out) * a.t + 255) / 256)), 256, 0, handle->cudaStream, a.scratch, a.parts, a.out, a.t, a.y, a.ldy);
    }
    HYB_CUDA(cudaFreeAsync(a.scratch, handle->cudaStream));
  }
  return e;
}
cudaError_t start_few(const hyacinHandle_t* handle, SingleArgs a) {
  const int64_t blocks = (int64_t(a.m) + kOut - 1) / kOut;
  a.splits = 1;
  while (a.splits < 8 && blocks * a.splits < 4 * int64_t(handle->DeviceSMs) && a.splits * 2 * kFewLanes <= a.n) a.splits *= 2;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(unsigned(blocks * a.splits)); cfg.blockDim = dim3(kFewThreads); cfg.stream = handle->cudaStream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension; attr[0].val.clusterDim.x = a.splits; attr[0].val.clusterDim.y = 1; attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr; cfg.numAttrs = a.splits > 1 ? 1 : 0;
  count_launch();
  return cudaLaunchKernelEx(&cfg, product_few_kernel, a);
}
template <Mode MODE> cudaError_t start_for(const hyacinHandle_t* handle, const SingleArgs& a) {
  return a.t <= 16 ? start<MODE, 16>(handle, a) : a.t <= 32 ? start<MODE, 32>(handle, a) : start<MODE, 64>(handle, a);
}

}  // namespace

int32_t launch_product_single(const hyacinHandle_t* handle, const char* fn, bool trans, const ProductArgs& p) {
  cudaStream_t stream = handle->cudaStream;
  SingleArgs a{};
  a.codes = p.codes; a.ldq = p.ldq; a.scales = static_cast<const float*>(p.scales); a.zeros = p.zeros; a.lds = p.lds;
  a.m = p.m; a.n = p.n; a.seg = p.seg; a.in = trans ? p.m : p.n; a.out = trans ? p.n : p.m; a.t = p.t;
  a.x = static_cast<const float*>(p.x); a.ldx = p.ldx; a.y = static_cast<float*>(p.y); a.ldy = p.ldy;
  float* mid = nullptr;
  cudaError_t e = cudaSuccess;
  if (p.rank) {
    e = cudaMallocFromPoolAsync(reinterpret_cast<void**>(&mid), size_t(p.rank) * p.t * sizeof(float), handle->mempool, stream);
    if (e != cudaSuccess) return w4_result(e, "cudaMallocFromPoolAsync");
    SingleArgs b = a;                              // mid(k, t) = sum_r first(r, k) x(r, t)
    b.second = static_cast<const float*>(p.first); b.ld2 = p.ld1; b.out = p.rank; b.y = mid; b.ldy = p.rank;
    e = start_for<kDense>(handle, b);
    a.rank = p.rank; a.second = static_cast<const float*>(p.second); a.ld2 = p.ld2; a.mid = mid;
  }
  if (e == cudaSuccess) e = trans ? start_for<kCodesT>(handle, a) : p.t <= kFew && p.m >= 8 * kOut ? start_few(handle, a) : start_for<kCodesN>(handle, a);
  if (mid) HYB_CUDA(cudaFreeAsync(mid, stream));
  return w4_result(e, fn);
}

}  // namespace hyb
