// Products with a 4-bit weight matrix on the fifth-generation tensor cores (16-bit types, both directions).
//
// Y (out x T) = A X, A = Wq^T or Wq.  A CTA computes 128 outputs x NT tokens (NT <= 256, accumulators in tensor memory) over a
// range of K steps of 128:
//   warp 0     TMA producer: the step's codes (128 columns x 64 bytes, 8 KiB) and the step's X tile (NT tokens x 128, K-major)
//              into a ring, so that the code stream from DRAM never waits for the arithmetic;
//   warps 2-9  turn codes into the scaled 16-bit weights s (q - zero) of a 128 x 128 operand tile in shared memory;
//   warp 1     issues tcgen05.mma (M128, N NT, K16) on it.
// Both directions share the dequantisation: a thread owns one column of W and a word of its codes is eight consecutive rows, one
// 16-byte chunk.  With opW 'T' the tile's rows are columns of W and the chunk runs along K (K-major operand); with 'N' the rows of
// shared memory are K and the chunk runs along the outputs (MN-major operand).  Address and swizzle are the same, only the
// descriptor differs.
// The correction V (U^T X) is two more operands of the same product: K steps whose A tile is V and whose X tile is
// mid = U^T X, kept as two 16-bit parts (value and remainder), so that it adds no rounding of its own.
// Few tiles: a cluster of up to 8 CTAs splits the K steps of one tile and adds the partial sums through distributed shared memory
// in a fixed order.
// Rounding: s (q - zero) has up to 15 significant bits (8 of s, 5 of q for bfloat16) and is rounded to the operand type, which
// is what the matrix instruction takes; one half step, independent per weight, well below the rounding of Y after a sum.
#include "w4_product.h"
#include "ptx_sm100.cuh"
#include <algorithm>
#include <atomic>

namespace hyb {
namespace {
using namespace ptx;

constexpr int kOut = 128;                         // outputs per tile
constexpr int kStep = 128;                        // K per step
constexpr uint32_t kCodeBytes = 128 * 64;
constexpr uint32_t kOperandBytes = kOut * kStep * 2;
constexpr int kMaxRing = 8;
constexpr int kThreads = 320;
constexpr int kWorkers = 8;                       // dequantising warps
constexpr uint32_t kSmemLimit = 232448;

struct UmmaParams {
  const void* scales; const uint8_t* zeros; int64_t lds;
  int m, n, t, out;
  int segs, seg_sub, seg_shift;                   // 32-row subsets per segment; shift when that is a power of two, else -1
  int code_steps, steps;                          // K steps of codes, and with those of the correction
  int rank; const void* second; int64_t ld2;
  void* y; int64_t ldy;
  int nt, ring, splits; uint32_t tmem_cols, idesc;
  uint32_t* status;
};

struct UmmaBars {
  uint64_t full[kMaxRing], empty[kMaxRing], a_full[2], a_empty[2], done;
  uint32_t tmem_base; uint32_t abort_flag;
};

__device__ __forceinline__ void umma_f16(uint32_t d, uint64_t adesc, uint64_t bdesc, uint32_t idesc, uint32_t accumulate) {
  asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
               "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}"
               ::"r"(d), "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate) : "memory");
}
__device__ __forceinline__ void tmem_ld8(uint32_t addr, float (&v)[8]) {
  uint32_t r[8];
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]) : "r"(addr) : "memory");
  tmem_ld_wait();
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = __uint_as_float(r[i]);
}
// 128-byte-swizzled operand: groups of 8 rows 1024 bytes apart (stride offset); the leading offset is the distance of the
// 64-element halves along M, used by the MN-major form only.
__device__ __forceinline__ uint64_t operand_desc(uint32_t addr, uint32_t leading) {
  return uint64_t((addr & 0x3FFFFu) >> 4) | (uint64_t(leading >> 4) << 16) | (uint64_t(1024 >> 4) << 32) | (uint64_t(1) << 46) | (uint64_t(2) << 61);
}
__device__ __forceinline__ void cluster_sync_all() {
  asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
  asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ float4 ld_cluster4(uint32_t addr, uint32_t rank) {
  uint32_t remote; float4 v;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(remote) : "r"(addr), "r"(rank));
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(remote) : "memory");
  return v;
}
__device__ __forceinline__ uint4 lds128(uint32_t addr) {
  uint4 v; asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(addr)); return v;
}
__device__ __forceinline__ void sts128(uint32_t addr, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(addr), "r"(a), "r"(b), "r"(c), "r"(d) : "memory");
}

// Scale and zero point of one (column, segment), as the pairs that the dequantisation multiplies and subtracts.
template <class T> struct Scale;
// half: 0x6400 | q is 1024 + q and 0x6400 | 16 q is 1024 + 16 q, both exact
template <> struct Scale<__half> {
  uint16_t bits = 0; int zero = 0;
  struct Ready { __half2 s, low, high; };
  __device__ __forceinline__ Ready ready() const {
    Ready r; r.s = __half2half2(__ushort_as_half(bits)); r.low = __float2half2_rn(float(-(1024 + zero))); r.high = __float2half2_rn(float(-(64 + zero))); return r;
  }
  static __device__ __forceinline__ uint32_t u(__half2 v) { return *reinterpret_cast<uint32_t*>(&v); }
  static __device__ __forceinline__ __half2 h(uint32_t v) { return *reinterpret_cast<__half2*>(&v); }
  static __device__ __forceinline__ void word(uint32_t w, const Ready& r, uint32_t (&o)[4]) {
    const __half2 sixteenth = __float2half2_rn(0.0625f);
    const uint32_t v = w >> 8;
    o[0] = u(__hmul2(__hadd2(h((w & 0x000f000fu) | 0x64006400u), r.low), r.s));
    o[1] = u(__hmul2(__hfma2(h((w & 0x00f000f0u) | 0x64006400u), sixteenth, r.high), r.s));
    o[2] = u(__hmul2(__hadd2(h((v & 0x000f000fu) | 0x64006400u), r.low), r.s));
    o[3] = u(__hmul2(__hfma2(h((v & 0x00f000f0u) | 0x64006400u), sixteenth, r.high), r.s));
  }
};
// bfloat16: 0x4300 | q is 128 + q; the seven bits of the fraction hold one nibble at a time
template <> struct Scale<__nv_bfloat16> {
  uint16_t bits = 0; int zero = 0;
  struct Ready { __nv_bfloat162 s, low; };
  __device__ __forceinline__ Ready ready() const {
    Ready r; r.s = __bfloat162bfloat162(__ushort_as_bfloat16(bits)); r.low = __float2bfloat162_rn(float(-(128 + zero))); return r;
  }
  static __device__ __forceinline__ uint32_t u(__nv_bfloat162 v) { return *reinterpret_cast<uint32_t*>(&v); }
  static __device__ __forceinline__ __nv_bfloat162 h(uint32_t v) { return *reinterpret_cast<__nv_bfloat162*>(&v); }
  static __device__ __forceinline__ void word(uint32_t w, const Ready& r, uint32_t (&o)[4]) {
#pragma unroll
    for (int p = 0; p < 4; ++p) o[p] = u(__hmul2(__hadd2(h(((w >> (4 * p)) & 0x000f000fu) | 0x43004300u), r.low), r.s));
  }
};

template <class T, bool TRANS>
__global__ void __launch_bounds__(kThreads, 1)
product_umma_kernel(const __grid_constant__ CUtensorMap code_map, const __grid_constant__ CUtensorMap x_map, const __grid_constant__ CUtensorMap mid_map,
                    const __grid_constant__ UmmaParams p) {
  extern __shared__ uint8_t smem_raw[];
  const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u;
  uint8_t* aligned = smem_raw + (base - smem_u32(smem_raw));
  const uint32_t x_bytes = uint32_t(p.nt) * kStep * 2;
  const uint32_t operand = base + p.ring * kCodeBytes, x_ring = operand + 2 * kOperandBytes;
  UmmaBars* bars = reinterpret_cast<UmmaBars*>(aligned + size_t(p.ring) * kCodeBytes + 2 * kOperandBytes + size_t(p.ring) * x_bytes);
  volatile uint32_t* abort_flag = &bars->abort_flag;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int part = int(blockIdx.x) % p.splits, tile = int(blockIdx.x) / p.splits, t0 = int(blockIdx.y) * p.nt;
  const int step0 = int(int64_t(p.steps) * part / p.splits), step1 = int(int64_t(p.steps) * (part + 1) / p.splits);

  if (threadIdx.x == 0) {
    for (int s = 0; s < p.ring; ++s) { mbar_init(&bars->full[s], 1); mbar_init(&bars->empty[s], 1); }
    for (int a = 0; a < 2; ++a) { mbar_init(&bars->a_full[a], kWorkers); mbar_init(&bars->a_empty[a], 1); }
    mbar_init(&bars->done, 1);
    bars->abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 1) tmem_alloc(&bars->tmem_base, p.tmem_cols);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = bars->tmem_base;

  bool ok = true;
  if (warp == 0) {
    if (lane == 0) {
      uint32_t stage = 0, phase = 0; int issued = 0; bool waited = false;
      for (int k = step0; k < step1; ++k) {
        if (!(ok = mbar_wait(&bars->empty[stage], phase ^ 1u, abort_flag, p.status, 11u))) break;
        uint64_t* bar = &bars->full[stage];
        const uint32_t sx = x_ring + stage * x_bytes;
        if (k < p.code_steps) {
          mbar_expect_tx(bar, kCodeBytes + x_bytes);
          if (TRANS) tma_load_2d(base + stage * kCodeBytes, &code_map, bar, k * 64, tile * kOut);
          else tma_load_2d(base + stage * kCodeBytes, &code_map, bar, tile * 64, k * kStep);
          tma_load_2d(sx, &x_map, bar, k * kStep, t0);
          tma_load_2d(sx + x_bytes / 2, &x_map, bar, k * kStep + 64, t0);
        } else {
          // mid comes from the kernel before this one, which may still be running
          if (!waited) { asm volatile("griddepcontrol.wait;" ::: "memory"); waited = true; }
          mbar_expect_tx(bar, x_bytes);
          const int c = (k - p.code_steps) * kStep;
          tma_load_2d(sx, &mid_map, bar, c, t0);
          tma_load_2d(sx + x_bytes / 2, &mid_map, bar, c + 64, t0);
        }
        ++issued;
        if (++stage == uint32_t(p.ring)) { stage = 0; phase ^= 1u; }
      }
      if (!ok) {      // some role gave up: let the copies in flight land before the block can end
        uint32_t ignore = 0;
        for (int b = 0; b < (issued < p.ring ? issued : p.ring); ++b) {
          if (stage == 0) { stage = p.ring; phase ^= 1u; }
          --stage;
          mbar_wait(&bars->full[stage], phase, &ignore, p.status, 12u);
        }
      }
    }
  } else if (warp == 1) {
    if (lane == 0) {
      uint32_t stage = 0, phase = 0, buf = 0, buf_phase = 0;
      for (int k = step0; k < step1; ++k) {
        if (!(ok = mbar_wait(&bars->full[stage], phase, abort_flag, p.status, 13u))) break;
        if (!(ok = mbar_wait(&bars->a_full[buf], buf_phase, abort_flag, p.status, 14u))) break;
        tc_fence_after();
        const uint32_t sa = operand + buf * kOperandBytes, sx = x_ring + stage * x_bytes;
#pragma unroll
        for (int q = 0; q < kStep / 16; ++q) {
          const uint64_t ad = TRANS ? operand_desc(sa + (q >> 2) * (kOperandBytes / 2) + (q & 3) * 32, 16)
                                    : operand_desc(sa + q * 2048, kOperandBytes / 2);
          const uint64_t bd = operand_desc(sx + (q >> 2) * (x_bytes / 2) + (q & 3) * 32, 16);
          umma_f16(tmem, ad, bd, p.idesc, (k > step0 || q > 0) ? 1u : 0u);
        }
        umma_commit(&bars->empty[stage]);
        umma_commit(&bars->a_empty[buf]);
        if (++stage == uint32_t(p.ring)) { stage = 0; phase ^= 1u; }
        if (++buf == 2) { buf = 0; buf_phase ^= 1u; }
      }
      umma_commit(&bars->done);
      if (!ok) { uint32_t ignore = 0; mbar_wait(&bars->done, 0u, &ignore, p.status, 15u); }      // instructions in flight end before tensor memory is freed
    }
  } else {
    const int id = threadIdx.x - 64, row = id & 127, half = id >> 7;      // row: column of W within the step's 128
    const bool uniform = (p.seg_sub & 3) == 0;
    Scale<T> cur[4];
    auto load_scales = [&](int k) {
      const int col = TRANS ? tile * kOut + row : k * kStep + row;
      const int sub = (TRANS ? k : tile) * 4;
      const bool live = col < p.n;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if (i > 0 && uniform) { cur[i] = cur[0]; continue; }
        int s = p.seg_shift >= 0 ? (sub + i) >> p.seg_shift : (sub + i) / p.seg_sub;
        s = min(s, p.segs - 1);
        cur[i].bits = live ? static_cast<const uint16_t*>(p.scales)[col * p.lds + s] : uint16_t(0);
        cur[i].zero = p.zeros ? (live ? int(p.zeros[col * p.lds + s]) : 0) : 8;
      }
    };
    uint32_t stage = 0, phase = 0, buf = 0, buf_phase = 0;
    if (step0 < min(step1, p.code_steps)) load_scales(step0);
    for (int k = step0; k < step1; ++k) {
      const uint32_t dst = operand + buf * kOperandBytes + row * 128, swz = (row & 7) << 4;
      if (k < p.code_steps) {
        ok = __all_sync(~0u, mbar_wait(&bars->full[stage], phase, abort_flag, p.status, 16u));
        if (!ok) break;
        uint4 q[2];
#pragma unroll
        for (int c = 0; c < 2; ++c) q[c] = lds128(base + stage * kCodeBytes + row * 64 + (((2 * half + c) ^ ((row >> 1) & 3)) << 4));
        typename Scale<T>::Ready r[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) r[i] = cur[i].ready();
        if (k + 1 < min(step1, p.code_steps)) load_scales(k + 1);
        ok = __all_sync(~0u, mbar_wait(&bars->a_empty[buf], buf_phase ^ 1u, abort_flag, p.status, 17u));
        if (!ok) break;
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          const uint32_t w[4] = {q[c].x, q[c].y, q[c].z, q[c].w};
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            uint32_t o[4]; Scale<T>::word(w[i], r[i], o);
            sts128(dst + (i >> 1) * (kOperandBytes / 2) + (((4 * (i & 1) + 2 * half + c) << 4) ^ swz), o[0], o[1], o[2], o[3]);
          }
        }
      } else {
        // correction step: entry (output, c) of the operand is second(output, c mod rank), c < 2 rank
        ok = __all_sync(~0u, mbar_wait(&bars->a_empty[buf], buf_phase ^ 1u, abort_flag, p.status, 18u));
        if (!ok) break;
        const uint16_t* second = static_cast<const uint16_t*>(p.second);
#pragma unroll 1
        for (int j = 0; j < 8; ++j) {
          uint32_t o[4] = {0, 0, 0, 0};
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const int along = 64 * half + 8 * j + e;
            const int c = (k - p.code_steps) * kStep + (TRANS ? along : row), out = tile * kOut + (TRANS ? row : along);
            if (c < 2 * p.rank && out < p.out) o[e >> 1] |= uint32_t(second[out + int64_t(c < p.rank ? c : c - p.rank) * p.ld2]) << (16 * (e & 1));
          }
          sts128(dst + half * (kOperandBytes / 2) + ((j << 4) ^ swz), o[0], o[1], o[2], o[3]);
        }
      }
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      __syncwarp();
      if (lane == 0) mbar_arrive(&bars->a_full[buf]);
      if (++stage == uint32_t(p.ring)) { stage = 0; phase ^= 1u; }
      if (++buf == 2) { buf = 0; buf_phase ^= 1u; }
    }
    // ---- accumulators: to Y, or to shared memory for the cluster's sum ----
    ok = __all_sync(~0u, ok && mbar_wait(&bars->done, 0u, abort_flag, p.status, 19u));
    if (ok) {
      tc_fence_after();
      const int quarter = warp & 3, side = (warp - 2) >> 2, o = quarter * 32 + lane, out = tile * kOut + o;
      const uint32_t addr = tmem + (uint32_t(quarter * 32) << 16);
      float* red = reinterpret_cast<float*>(aligned);
      for (int c = side * (p.nt / 2); c < (side + 1) * (p.nt / 2); c += 8) {
        if (p.splits == 1 && t0 + c >= p.t) break;
        float v[8];
        tmem_ld8(addr + c, v);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          if (p.splits > 1) red[(c + e) * kOut + o] = v[e];
          else if (out < p.out && t0 + c + e < p.t) static_cast<T*>(p.y)[int64_t(t0 + c + e) * p.ldy + out] = from_f32<T>(v[e]);
        }
      }
      tc_fence_before();
    }
  }
  __syncthreads();
  if (warp == 1) { tc_fence_after(); tmem_dealloc(tmem, p.tmem_cols); }
  if (p.splits > 1) {
    cluster_sync_all();
    const int c0 = p.nt * part / p.splits, c1 = p.nt * (part + 1) / p.splits;
    for (int e = threadIdx.x; e < (c1 - c0) * (kOut / 4); e += kThreads) {
      const int c = c0 + e / (kOut / 4), o = (e % (kOut / 4)) * 4;
      if (t0 + c >= p.t) break;
      float4 s = ld_cluster4(base + (c * kOut + o) * 4, 0);
      for (int r = 1; r < p.splits; ++r) {
        const float4 v = ld_cluster4(base + (c * kOut + o) * 4, r);
        s.x += v.x; s.y += v.y; s.z += v.z; s.w += v.w;
      }
      T* y = static_cast<T*>(p.y) + int64_t(t0 + c) * p.ldy + tile * kOut + o;
      const float v[4] = {s.x, s.y, s.z, s.w};
#pragma unroll
      for (int i = 0; i < 4; ++i) if (tile * kOut + o + i < p.out) y[i] = from_f32<T>(v[i]);
    }
    cluster_sync_all();                            // shared memory stays until every peer has read it
  }
}

// ---- mid = first^T X for many tokens, as two 16-bit parts: [token][value 0 .. rank, remainder 0 .. rank] ----------------------
template <class T> __device__ __forceinline__ uint4 load8(const T* p, int valid, bool aligned) {
  if (valid >= 8 && aligned) return *reinterpret_cast<const uint4*>(p);
  uint32_t o[4] = {0, 0, 0, 0};
#pragma unroll
  for (int e = 0; e < 8; ++e) if (e < valid) o[e >> 1] |= uint32_t(reinterpret_cast<const uint16_t*>(p)[e]) << (16 * (e & 1));
  return make_uint4(o[0], o[1], o[2], o[3]);
}
template <class T> __device__ __forceinline__ void mma16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1);
template <> __device__ __forceinline__ void mma16816<__half>(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
template <> __device__ __forceinline__ void mma16816<__nv_bfloat16>(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

constexpr int kMidWarps = 16;
// A block: 16 entries of the rank x 16 tokens; its warps split the rows.  A lane feeds eight consecutive rows of each operand
// row to two instructions: the order of K inside an instruction is free as long as both operands agree.
template <class T> __global__ void __launch_bounds__(kMidWarps * 32)
mid_split_kernel(const T* first, int64_t ld1, int rows, int rank, const T* x, int64_t ldx, int t, T* mid, int64_t ldm, int aligned) {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  __shared__ float red[kMidWarps][16][17];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, c = lane & 3;
  const int k0 = blockIdx.x * 16; const int64_t t0 = int64_t(blockIdx.y) * 16;
  const T* fp[2] = {first + int64_t(k0 + g) * ld1, first + int64_t(k0 + g + 8) * ld1};
  const T* xp[2] = {x + (t0 + g) * ldx, x + (t0 + g + 8) * ldx};
  const bool fl[2] = {k0 + g < rank, k0 + g + 8 < rank}, xl[2] = {t0 + g < t, t0 + g + 8 < t};
  float acc[2][4] = {};
#pragma unroll 4
  for (int r = warp * 32 + c * 8; r < (rows + 31) / 32 * 32; r += kMidWarps * 32) {
    const int valid = rows - r;
    uint4 a[2], b[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      a[i] = load8(fp[i] + r, fl[i] ? valid : 0, aligned); b[i] = load8(xp[i] + r, xl[i] ? valid : 0, aligned);
    }
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      mma16816<T>(acc[i], a[0].x, a[1].x, a[0].y, a[1].y, b[i].x, b[i].y);
      mma16816<T>(acc[i], a[0].z, a[1].z, a[0].w, a[1].w, b[i].z, b[i].w);
    }
  }
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int e = 0; e < 4; ++e) red[warp][g + 8 * (e >> 1)][8 * i + 2 * c + (e & 1)] = acc[i][e];
  __syncthreads();
  if (threadIdx.x < 256) {
    const int k = threadIdx.x & 15, tok = threadIdx.x >> 4;
    float s = 0.f;
#pragma unroll
    for (int w = 0; w < kMidWarps; ++w) s += red[w][k][tok];
    if (k0 + k < rank && t0 + tok < t) {
      T* m = mid + (t0 + tok) * ldm + k0 + k;
      const T value = from_f32<T>(s);
      m[0] = value; m[rank] = from_f32<T>(s - to_f32(value));
    }
  }
}

// X with rows that TMA can address (16-byte pitch and start).
__global__ void __launch_bounds__(256) align_rows_kernel(const uint16_t* x, int64_t ldx, int rows, uint16_t* out, int64_t ldo) {
  for (int r = blockIdx.x * 256 + threadIdx.x; r < rows; r += gridDim.x * 256) out[int64_t(blockIdx.y) * ldo + r] = x[int64_t(blockIdx.y) * ldx + r];
}

bool encode_2d(CUtensorMap* map, CUtensorMapDataType type, const void* ptr, uint64_t inner, uint64_t outer, uint64_t pitch, uint32_t box_inner, uint32_t box_outer,
               CUtensorMapSwizzle swizzle) {
  EncodeTiledFn encode = encode_tiled();
  if (!encode) return false;
  const cuuint64_t dims[2] = {inner, outer}, strides[1] = {pitch};
  const cuuint32_t box[2] = {box_inner, box_outer}, elem[2] = {1, 1};
  const CUresult r = encode(map, type, 2, const_cast<void*>(ptr), dims, strides, box, elem, CU_TENSOR_MAP_INTERLEAVE_NONE, swizzle,
                            CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) std::fprintf(stderr, "hyacin-b200: cuTensorMapEncodeTiled failed (%d)\n", int(r));
  return r == CUDA_SUCCESS;
}

// CTAs that share a tile's K steps: the whole takes ceil(tiles s / SMs) rounds of ceil(steps / s) steps plus about six steps' worth of
// start, drain and exchange.
int choose_splits(int64_t tiles, int steps, int sms) {
  int best = 1; double cost = 1e300;
  for (int s = 1; s <= 8 && s * 2 <= std::max(steps, 2); ++s) {
    const double c = double((tiles * s + sms - 1) / sms) * ((steps + s - 1) / s + 6.);
    if (c < cost * 0.999) { cost = c; best = s; }
  }
  return best;
}

template <class T, bool TRANS> int32_t launch(const hyacinHandle_t* handle, const char* fn, hyacinPrecision_t type, const ProductArgs& a) {
  cudaStream_t stream = handle->cudaStream;
  const int in = TRANS ? a.m : a.n, out = TRANS ? a.n : a.m;
  void *x_copy = nullptr, *mid = nullptr;
  auto cleanup = [&] { if (x_copy) HYB_CUDA(cudaFreeAsync(x_copy, stream)); if (mid) HYB_CUDA(cudaFreeAsync(mid, stream)); };
  auto allocate = [&](void** p, size_t bytes) {
    const cudaError_t e = cudaMallocFromPoolAsync(p, bytes, handle->mempool, stream);
    if (e != cudaSuccess) { report_cuda_error(e, "cudaMallocFromPoolAsync", __FILE__, __LINE__); *p = nullptr; }
    return e == cudaSuccess;
  };
  const void* x = a.x; int64_t ldx = a.ldx;
  if (a.t == 1) ldx = (int64_t(in) + 7) / 8 * 8;                 // a single column has no pitch
  if (reinterpret_cast<uintptr_t>(x) % 16 || ldx % 8) {
    const int64_t ldo = (int64_t(in) + 7) / 8 * 8;
    if (!allocate(&x_copy, size_t(ldo) * a.t * 2)) return -3;
    for (int64_t t = 0; t < a.t; t += 65535) {
      count_launch();
      align_rows_kernel<<<dim3((in + 255) / 256, unsigned(std::min<int64_t>(65535, a.t - t))), 256, 0, stream>>>(
          static_cast<const uint16_t*>(a.x) + t * a.ldx, a.ldx, in, static_cast<uint16_t*>(x_copy) + t * ldo, ldo);
    }
    x = x_copy; ldx = ldo;
  }
  UmmaParams p{};
  p.scales = a.scales; p.zeros = a.zeros; p.lds = a.lds; p.m = a.m; p.n = a.n; p.t = a.t; p.out = out;
  p.segs = (a.m + a.seg - 1) / a.seg; p.seg_sub = a.seg / 32; p.seg_shift = -1;
  for (int s = 0; s < 27; ++s) if (p.seg_sub == 1 << s) p.seg_shift = s;
  p.code_steps = (in + kStep - 1) / kStep;
  p.rank = a.rank; p.second = a.second; p.ld2 = a.ld2; p.y = a.y; p.ldy = a.ldy;
  p.steps = p.code_steps + (2 * a.rank + kStep - 1) / kStep;
  const int64_t token_tiles = (int64_t(a.t) + 255) / 256;
  p.nt = int((int64_t(a.t) + token_tiles - 1) / token_tiles + 15) / 16 * 16;
  p.tmem_cols = 32;
  while (p.tmem_cols < uint32_t(p.nt)) p.tmem_cols *= 2;
  const uint32_t x_bytes = uint32_t(p.nt) * kStep * 2;
  const uint32_t fixed = 2 * kOperandBytes + 1024 + sizeof(UmmaBars);
  p.ring = int(std::min<uint32_t>(kMaxRing, (kSmemLimit - fixed) / (kCodeBytes + x_bytes)));
  const uint32_t smem = fixed + p.ring * (kCodeBytes + x_bytes);
  const int tiles = (out + kOut - 1) / kOut;
  p.splits = choose_splits(int64_t(tiles) * token_tiles, p.steps, handle->DeviceSMs);
  const uint32_t fmt = type == HYACIN_F16 ? 0u : 1u;
  p.idesc = (1u << 4) | (fmt << 7) | (fmt << 10) | ((TRANS ? 0u : 1u) << 15) | (uint32_t(p.nt >> 3) << 17) | (uint32_t(kOut >> 4) << 24);
  p.status = status_word_device(handle->DeviceID);
  const CUtensorMapDataType dt = type == HYACIN_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
  CUtensorMap code_map{}, x_map{}, mid_map{};
  bool fine = encode_2d(&code_map, CU_TENSOR_MAP_DATA_TYPE_UINT8, a.codes, uint64_t((a.m + 127) / 128) * 64, a.n, a.ldq, 64, 128, CU_TENSOR_MAP_SWIZZLE_64B) &&
              encode_2d(&x_map, dt, x, in, a.t, uint64_t(ldx) * 2, 64, p.nt, CU_TENSOR_MAP_SWIZZLE_128B);
  mid_map = x_map;
  if (fine && a.rank) {
    const int64_t ldm = (2 * int64_t(a.rank) + 7) / 8 * 8;
    if (!allocate(&mid, size_t(ldm) * a.t * 2)) { cleanup(); return -3; }
    fine = encode_2d(&mid_map, dt, mid, 2 * uint64_t(a.rank), a.t, uint64_t(ldm) * 2, 64, p.nt, CU_TENSOR_MAP_SWIZZLE_128B);
    const int aligned = reinterpret_cast<uintptr_t>(x) % 16 == 0 && ldx % 8 == 0 && reinterpret_cast<uintptr_t>(a.first) % 16 == 0 && a.ld1 % 8 == 0;
    count_launch();
    mid_split_kernel<T><<<dim3((a.rank + 15) / 16, unsigned((int64_t(a.t) + 15) / 16)), kMidWarps * 32, 0, stream>>>(
        static_cast<const T*>(a.first), a.ld1, in, a.rank, static_cast<const T*>(x), ldx, a.t, static_cast<T*>(mid), ldm, aligned);
  }
  if (!fine) { cleanup(); return -3; }
  auto* kernel = product_umma_kernel<T, TRANS>;
  static std::atomic<uint64_t> ready{0};                         // per device: shared memory limit raised
  const uint64_t bit = uint64_t(1) << (handle->DeviceID & 63);
  if (!(ready.load() & bit)) {
    const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmemLimit);
    if (e != cudaSuccess) { report_cuda_error(e, "cudaFuncSetAttribute", __FILE__, __LINE__); cleanup(); return -3; }
    ready.fetch_or(bit);
  }
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(unsigned(tiles) * p.splits, unsigned(token_tiles)); cfg.blockDim = dim3(kThreads); cfg.dynamicSmemBytes = smem; cfg.stream = stream;
  cudaLaunchAttribute attr[2]; int attrs = 0;
  attr[attrs].id = cudaLaunchAttributeClusterDimension; attr[attrs].val.clusterDim.x = p.splits; attr[attrs].val.clusterDim.y = 1; attr[attrs++].val.clusterDim.z = 1;
  if (a.rank) { attr[attrs].id = cudaLaunchAttributeProgrammaticStreamSerialization; attr[attrs++].val.programmaticStreamSerializationAllowed = 1; }
  cfg.attrs = attr; cfg.numAttrs = attrs;
  count_launch();
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, code_map, x_map, mid_map, p);
  if (e != cudaSuccess) report_cuda_error(e, fn, __FILE__, __LINE__);
  cleanup();
  return e == cudaSuccess ? w4_launched(fn) : -3;
}

}  // namespace

int32_t launch_product_umma(const hyacinHandle_t* handle, const char* fn, bool trans, hyacinPrecision_t type, const ProductArgs& a) {
  if (type == HYACIN_F16) return trans ? launch<__half, true>(handle, fn, type, a) : launch<__half, false>(handle, fn, type, a);
  return trans ? launch<__nv_bfloat16, true>(handle, fn, type, a) : launch<__nv_bfloat16, false>(handle, fn, type, a);
}

}  // namespace hyb
