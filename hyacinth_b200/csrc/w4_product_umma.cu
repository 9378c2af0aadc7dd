// Products with a 4-bit weight matrix on the fifth-generation tensor cores (16-bit types, both directions).
//
// Y (out x T) = A X, A = Wq^T or Wq.  A CTA computes 128 outputs x NT tokens (NT <= 256, accumulators in tensor memory) over a
// range of K steps:
//   warp 0     TMA producer: the step's codes and the step's X tile (NT tokens, K-major) into a ring, so that the code stream from
//              DRAM never waits for the arithmetic;
//   warp 1     issues tcgen05.mma (M128, N NT, K16);
//   warps 2-5  fetch the step's scales and zero points into the ring;
//   warps 6-21 turn codes into scaled 16-bit weights s (q - zero), in four groups of four warps that take every fourth step, into up
//              to six operand buffers: from the dequantised tile to the freed buffer takes some 1700 cycles, several steps' worth.
// opW 'T': a step is 128 rows of W, a thread owns one output and writes its K values to tensor memory, the A operand of the
// instruction (an instruction with A in shared memory takes 40 cycles for its 4 KiB however small NT is, from tensor memory
// 10 to 33).  opW 'N': a step is 128 columns of W (64 beside tiles of more than 128 tokens); a word of codes is eight consecutive outputs
// at one K, a 16-byte chunk of an MN-major operand in shared memory.
// The correction V (U^T X) is two more operands of the same product: K steps whose A tile is V and whose X tile is mid = U^T X, both in
// bfloat16 parts, whose exponents hold every 32-bit mid (a half ends at 65504 and loses small remainders).  bfloat16: mid in two
// parts, value and remainder, 16 bits, 2^-8 of the rounding of Y.  Half: V in two parts, exact, mid in three, all of its 24 bits; of
// their six products the last, 2^-24, is left out.
// Few tiles: a cluster of up to 8 CTAs splits the K steps of one tile and adds the partial sums through distributed shared memory
// in a fixed order.
// Rounding: s (q - zero) has up to 15 significant bits (8 of s, 5 of q for bfloat16) and is rounded to the operand type, which
// is what the matrix instruction takes; one half step, independent per weight, of the size of the rounding of Y itself (error against
// 64 bits 0.0021 instead of the 0.0017 of that rounding alone for bfloat16, 0.00027 instead of 0.00021 for half).  A weight beyond 65504 is an
// infinity for half.
// Bound: the hand-overs between the roles: 4096 x 16384 bfloat16 times 32 tokens keeps the tensor pipe busy for 9 % of the time, the issue
// slots for 41 % and DRAM for 16 %, times 256 tokens for 47, 33 and 10 %.  Measured, matrices cycled through more than the L2: 32 tokens 22.0
// us (1.6 TB/s), 128 tokens 25.0 us (690 TFLOP/s), 256 tokens 33.0 us (1040 TFLOP/s, 0.65 of measured); half with segments of 64 rows and
// zero points, opW 'N', 64 tokens 27.4 us.  The correction, rank 64, adds 5.0 us to the first of these and 7.5 to the third (half: 8 and 10).
#include "w4_product.h"
#include "ptx_sm100.cuh"
#include <algorithm>
#include <atomic>
#include <type_traits>

namespace hyb {
namespace {
using namespace ptx;

constexpr int kOut = 128;                         // outputs per tile
constexpr int kMaxRing = 8;
constexpr int kMaxTokens = 256;                   // per tile
constexpr int kLoaders = 4;                       // warps that fetch scales
constexpr int kGroups = 4, kGroupWarps = 4;       // dequantising warps
constexpr int kMaxBufs = 6;                       // operand buffers
constexpr int kThreads = 32 * (2 + kLoaders + kGroups * kGroupWarps);
// More than half of the shared memory, always: one CTA per SM, so tensor memory is not contended for, which clusters whose CTAs
// wait for one another could not afford.
constexpr uint32_t kSmemLimit = 232448, kSmemFloor = 120 * 1024;
template <bool TRANS, int STEP> struct Geometry {
  static constexpr int step = STEP;                                      // K per step
  static constexpr int cols = TRANS ? kOut : step;                       // columns of W per step
  static constexpr uint32_t code_bytes = cols * 64;
  static constexpr uint32_t scale_bytes = cols * 12;                     // four 16-bit scales and four zero points per column
  static constexpr uint32_t operand_bytes = TRANS ? 0 : kOut * step * 2; // in shared memory, per group
  static constexpr uint32_t operand_cols = TRANS ? step / 2 : 0;         // in tensor memory, per group
};

struct UmmaParams {
  const void* scales; const uint8_t* zeros; int64_t lds;
  int m, n, t, out;
  int segs, seg_sub, seg_shift;                   // 32-row subsets per segment; shift when that is a power of two, else -1
  int wide;                                       // segments of a block that one aligned load fetches (1, 2, 4)
  int code_steps, steps;                          // K steps of codes, and with those of the correction
  int rank, rank16; const void* second; int64_t ld2;      // rank16: rank rounded up to 16, the width of a part of mid
  void* y; int64_t ldy;
  int nt, ring, bufs, groups, splits, second_aligned; uint32_t nt_cols, tmem_cols, idesc, idesc_more;      // idesc_more: of the correction
  uint32_t* status;
};

struct UmmaBars {
  uint64_t full[kMaxRing], empty[kMaxRing], a_full[kMaxBufs], done;
  uint32_t tmem_base; uint32_t abort_flag;
};

__device__ __forceinline__ void umma_f16(uint32_t d, uint64_t adesc, uint64_t bdesc, uint32_t idesc, uint32_t accumulate) {
  asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
               "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}"
               ::"r"(d), "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate) : "memory");
}
__device__ __forceinline__ void umma_f16_ts(uint32_t d, uint32_t a, uint64_t bdesc, uint32_t idesc, uint32_t accumulate) {
  asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
               "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}"
               ::"r"(d), "r"(a), "l"(bdesc), "r"(idesc), "r"(accumulate) : "memory");
}
__device__ __forceinline__ void tmem_st32(uint32_t addr, const uint32_t (&v)[32]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], "
      "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, "
      "%17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32};"
      ::"r"(addr), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]),
        "r"(v[8]), "r"(v[9]), "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15]),
        "r"(v[16]), "r"(v[17]), "r"(v[18]), "r"(v[19]), "r"(v[20]), "r"(v[21]), "r"(v[22]), "r"(v[23]),
        "r"(v[24]), "r"(v[25]), "r"(v[26]), "r"(v[27]), "r"(v[28]), "r"(v[29]), "r"(v[30]), "r"(v[31])
      : "memory");
}
__device__ __forceinline__ void tmem_st4(uint32_t addr, const uint32_t (&v)[4]) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x4.b32 [%0], {%1, %2, %3, %4};" ::"r"(addr), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]) : "memory");
}
// Bounded waits for the pipelines of this kernel, executed by whole warps: a poll by a single lane is not suspended by the
// hardware, and many warps that poll slow the multiplying warp down (a satisfied wait took it 800 cycles with 20 single-lane
// pollers).  So few warps poll at a time, the ones that run ahead with pauses in between.
template <bool PAUSE> __device__ __forceinline__ bool warp_wait(uint64_t* bar, uint32_t parity, volatile uint32_t* abort_flag, uint32_t* status, uint32_t code) {
#pragma unroll 1
  for (uint32_t it = 0; it < (1u << 20); ++it) {
    uint32_t done;
    asm volatile("{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, %3;\n\tselp.u32 %0, 1, 0, p;\n\t}"
                 : "=r"(done) : "r"(smem_u32(bar)), "r"(parity), "r"(20000u) : "memory");
    if (__all_sync(~0u, done)) return true;
    if (__any_sync(~0u, *abort_flag)) break;
    if (PAUSE) __nanosleep(64);
  }
  if ((threadIdx.x & 31) == 0 && !*abort_flag) { *abort_flag = 1u; *reinterpret_cast<volatile uint32_t*>(status) = code; }
  __syncwarp();
  return false;
}
__device__ __forceinline__ bool elect_one() {
  uint32_t r;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(r));
  return r != 0;
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

// Eight consecutive values, the first `valid` of them, zeros behind.
template <class T> __device__ __forceinline__ uint4 load8(const T* p, int valid, bool aligned) {
  if (valid >= 8 && aligned) return *reinterpret_cast<const uint4*>(p);
  uint32_t o[4] = {0, 0, 0, 0};
#pragma unroll
  for (int e = 0; e < 8; ++e) if (e < valid) o[e >> 1] |= uint32_t(reinterpret_cast<const uint16_t*>(p)[e]) << (16 * (e & 1));
  return make_uint4(o[0], o[1], o[2], o[3]);
}

// (w & mask) | bits in one instruction: left to the compiler, two constants became two instructions
__device__ __forceinline__ uint32_t and_or(uint32_t w, uint32_t mask, uint32_t bits) {
  uint32_t r;
  asm("lop3.b32 %0, %1, %2, %3, 0xEA;" : "=r"(r) : "r"(w), "r"(mask), "r"(bits));
  return r;
}

// The first `left` of a word's eight rows, the zero point in the others.
__device__ __forceinline__ uint32_t rows_only(uint32_t w, int left, uint32_t zero) {
  left = min(max(left, 0), 8);
  const uint32_t mask = ((1u << 4 * ((left + 1) >> 1)) - 1u) | ((1u << 4 * (left >> 1)) - 1u) << 16;
  return (w & mask) | (zero * 0x11111111u & ~mask);
}

// Scale and zero point of one (column, segment), as the pairs that the dequantisation multiplies and subtracts.
template <class T> struct Scale;
// half: 0x6400 | q is 1024 + q and 0x6400 | 16 q is 1024 + 16 q, both exact (published for 4-bit weights by Kim et al., arXiv:2211.10017, 2022)
template <> struct Scale<__half> {
  uint16_t bits = 0; int zero = 0;
  struct Ready { __half2 s, low, high; };
  __device__ __forceinline__ Ready ready() const {
    Ready r; r.s = __half2half2(__ushort_as_half(bits)); r.low = __float2half2_rn(float(-(1024 + zero))); r.high = __float2half2_rn(float(-(64 + zero))); return r;
  }
  static __device__ __forceinline__ uint32_t u(__half2 v) { return *reinterpret_cast<uint32_t*>(&v); }
  static __device__ __forceinline__ __half2 h(uint32_t v) { return *reinterpret_cast<__half2*>(&v); }
  static __device__ __forceinline__ void word(uint32_t w, const Ready& r, uint32_t* o) {
    const __half2 sixteenth = __float2half2_rn(0.0625f);
    const uint32_t v = w >> 8;
    o[0] = u(__hmul2(__hadd2(h(and_or(w, 0x000f000fu, 0x64006400u)), r.low), r.s));
    o[1] = u(__hmul2(__hfma2(h(and_or(w, 0x00f000f0u, 0x64006400u)), sixteenth, r.high), r.s));
    o[2] = u(__hmul2(__hadd2(h(and_or(v, 0x000f000fu, 0x64006400u)), r.low), r.s));
    o[3] = u(__hmul2(__hfma2(h(and_or(v, 0x00f000f0u, 0x64006400u)), sixteenth, r.high), r.s));
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
  static __device__ __forceinline__ void word(uint32_t w, const Ready& r, uint32_t* o) {
#pragma unroll
    for (int p = 0; p < 4; ++p) o[p] = u(__hmul2(__hadd2(h(and_or(w >> (4 * p), 0x000f000fu, 0x43004300u)), r.low), r.s));
  }
};

// Parts of the correction's operands, the same K range after another: with mid part i (i < mid) V, or what of it is left beyond
// bfloat16 with part i - mid.
template <class T> struct Parts { static constexpr bool split = std::is_same<T, __half>::value; static constexpr int mid = split ? 3 : 2, all = split ? 5 : 2; };
// Two halves as bfloat16: the nearest, or what it leaves (3 bits, exact; of an infinity a NaN).
__device__ __forceinline__ uint32_t factor_part(uint32_t v, bool rest) {
  const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&v));
  __nv_bfloat162 b = __floats2bfloat162_rn(f.x, f.y);
  if (rest) b = __floats2bfloat162_rn(f.x - __low2float(b), f.y - __high2float(b));
  return *reinterpret_cast<const uint32_t*>(&b);
}

template <class T, bool TRANS, int STEP>
__global__ void __launch_bounds__(kThreads, 1)
product_umma_kernel(const __grid_constant__ CUtensorMap code_map, const __grid_constant__ CUtensorMap x_map, const __grid_constant__ CUtensorMap mid_map,
                    const __grid_constant__ UmmaParams p) {
  extern __shared__ uint8_t smem_raw[];
  const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u;
  uint8_t* aligned = smem_raw + (base - smem_u32(smem_raw));
  using G = Geometry<TRANS, STEP>;
  constexpr int kStep = G::step;
  constexpr bool kFull = STEP == 128;
  const uint32_t x_bytes = uint32_t(p.nt) * kStep * 2;
  const uint32_t operand = base + p.ring * G::code_bytes, x_ring = operand + p.bufs * G::operand_bytes, scale_ring = x_ring + p.ring * x_bytes;
  UmmaBars* bars = reinterpret_cast<UmmaBars*>(aligned + (scale_ring - base) + p.ring * G::scale_bytes);
  volatile uint32_t* abort_flag = &bars->abort_flag;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int part = int(blockIdx.x) % p.splits, tile = int(blockIdx.x) / p.splits, t0 = int(blockIdx.y) * p.nt;
  const int step0 = int(int64_t(p.steps) * part / p.splits), step1 = int(int64_t(p.steps) * (part + 1) / p.splits);

  // The first copies start before the block has met: the thread that issues them has initialised their barriers itself.
  const int early = step1 - step0 < p.ring ? step1 - step0 : p.ring;
  auto issue = [&](int k, uint32_t stage) {
    uint64_t* bar = &bars->full[stage];
    const uint32_t sx = x_ring + stage * x_bytes;
    if (k < p.code_steps) {
      mbar_expect_tx(bar, G::code_bytes + x_bytes);
      if (TRANS) tma_load_2d(base + stage * G::code_bytes, &code_map, bar, k * 64, tile * kOut);
      else tma_load_2d(base + stage * G::code_bytes, &code_map, bar, tile * 64, k * kStep);
      tma_load_2d(sx, &x_map, bar, k * kStep, t0);
      if (kFull) tma_load_2d(sx + x_bytes / 2, &x_map, bar, k * kStep + 64, t0);
    } else {
      mbar_expect_tx(bar, x_bytes);
      const int c = (k - p.code_steps) * kStep;
      tma_load_2d(sx, &mid_map, bar, c, t0);
      if (kFull) tma_load_2d(sx + x_bytes / 2, &mid_map, bar, c + 64, t0);
    }
  };
  if (threadIdx.x == 0) {
    prefetch_map(&code_map); prefetch_map(&x_map);
    for (int s = 0; s < p.ring; ++s) { mbar_init(&bars->full[s], 2); mbar_init(&bars->empty[s], 1); }
    for (int a = 0; a < p.bufs; ++a) mbar_init(&bars->a_full[a], kGroupWarps);
    mbar_init(&bars->done, 1);
    bars->abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    for (int k = step0; k < step0 + early && k < p.code_steps; ++k) issue(k, k - step0);
  }
  if (warp == 1) tmem_alloc(&bars->tmem_base, p.tmem_cols);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = bars->tmem_base;

  bool ok = true;
  if (warp == 0) {
    uint32_t stage = 0, phase = 0; int issued = 0; bool waited = false;
    for (int k = step0; k < step1; ++k) {
      if (!(issued < early && k < p.code_steps)) {
        if (issued >= p.ring && !(ok = warp_wait<true>(&bars->empty[stage], phase ^ 1u, abort_flag, p.status, 11u))) break;
        // mid comes from the kernel before this one, which may still be running
        if (k >= p.code_steps && !waited) { asm volatile("griddepcontrol.wait;" ::: "memory"); waited = true; }
        if (lane == 0) issue(k, stage);
        __syncwarp();
      }
      ++issued;
      if (++stage == uint32_t(p.ring)) { stage = 0; phase ^= 1u; }
    }
    if (!ok && lane == 0) {      // some role gave up: let the copies in flight land before the block can end
      uint32_t ignore = 0;
      for (int b = 0; b < (issued < p.ring ? issued : p.ring); ++b) {
        if (stage == 0) { stage = p.ring; phase ^= 1u; }
        --stage;
        mbar_wait(&bars->full[stage], phase, &ignore, p.status, 12u);
      }
    }
  } else if (warp == 1) {
    // The whole warp runs the loop and one elected lane issues: descriptors then stay in uniform registers.  With the loop inside
    // a single-lane branch an instruction took 69 cycles to issue, more than it runs for with NT <= 128.
    uint32_t stage = 0, buf = 0, buf_phase = 0;
    for (int k = step0; k < step1; ++k) {
      // the group that filled the operand buffer had seen the step's copies land
      if (!(ok = warp_wait<false>(&bars->a_full[buf], buf_phase, abort_flag, p.status, 14u))) break;
      tc_fence_after();
      const uint32_t sx = x_ring + stage * x_bytes, ta = tmem + p.nt_cols + buf * G::operand_cols;
      const uint64_t a0 = operand_desc(operand + buf * G::operand_bytes, G::operand_bytes / 2), b0 = operand_desc(sx, 16);
      const uint32_t b_half = x_bytes / 32, idesc = Parts<T>::split && k >= p.code_steps ? p.idesc_more : p.idesc;
      if (elect_one()) {
#pragma unroll
        for (int q = 0; q < kStep / 16; ++q) {
          const uint64_t bd = b0 + ((q >> 2) * b_half + (q & 3) * 2);
          if (TRANS) umma_f16_ts(tmem, ta + q * 8, bd, idesc, (k > step0 || q > 0) ? 1u : 0u);
          else umma_f16(tmem, a0 + q * 128, bd, idesc, (k > step0 || q > 0) ? 1u : 0u);
        }
        umma_commit(&bars->empty[stage]);
      }
      __syncwarp();
      if (++stage == uint32_t(p.ring)) stage = 0;
      if (++buf == uint32_t(p.bufs)) { buf = 0; buf_phase ^= 1u; }
    }
    if (elect_one()) umma_commit(&bars->done);
    __syncwarp();
    if (!ok) { uint32_t ignore = 0; mbar_wait(&bars->done, 0u, &ignore, p.status, 15u); }      // instructions in flight end before tensor memory is freed
  } else if (warp < 2 + kLoaders) {
    // Scales and zero points of a step, [column][subset]: they lie one row of the table per column, so every load touches as many
    // lines as lanes.  Each loader takes every fourth step and has the next one's loads in flight while it hands one over.
    const int loaders = p.ring < kLoaders ? p.ring : kLoaders;
    constexpr int kPer = G::cols / 32;                             // columns per lane
    struct Entry { uint32_t s01, s23, z; } even[kPer], odd[kPer];
    enum Form { kNothing, kOne, kPair, kFour, kMixed };
    auto segment = [&](int sub) { return p.seg_shift >= 0 ? sub >> p.seg_shift : sub / p.seg_sub; };
    auto form = [&](int k) {
      if (k >= p.code_steps || k >= step1) return kNothing;
      const int first = segment((TRANS ? k : tile) * 4);
      return p.wide == 4 && first + 4 <= p.segs ? kFour : p.wide == 2 && first + 2 <= p.segs ? kPair : (p.seg_sub & 3) == 0 ? kOne : kMixed;
    };
    auto fetch = [&](int k, Entry (&e)[kPer]) {
      const int sub = (TRANS ? k : tile) * 4, first = segment(sub);
      const Form f = form(k);
#pragma unroll
      for (int j = 0; j < kPer; ++j) {
        const int col = (TRANS ? tile * kOut : k * kStep) + 32 * j + lane;
        e[j].s01 = e[j].s23 = 0; e[j].z = p.zeros ? 0u : 0x08080808u;
        if (f == kNothing || col >= p.n) continue;
        const uint16_t* scales = static_cast<const uint16_t*>(p.scales) + col * p.lds;
        const uint8_t* zeros = p.zeros + col * p.lds;
        if (f == kFour) {
          const uint2 v = *reinterpret_cast<const uint2*>(scales + first);
          e[j].s01 = v.x; e[j].s23 = v.y;
          if (p.zeros) e[j].z = *reinterpret_cast<const uint32_t*>(zeros + first);
        } else if (f == kPair) {
          e[j].s01 = *reinterpret_cast<const uint32_t*>(scales + first);
          if (p.zeros) e[j].z = *reinterpret_cast<const uint16_t*>(zeros + first);
        } else if (f == kOne) {
          e[j].s01 = scales[first];
          if (p.zeros) e[j].z = zeros[first];
        } else {
          uint32_t s[4], z = 0;
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int g = min(segment(sub + i), p.segs - 1);
            s[i] = scales[g];
            if (p.zeros) z |= uint32_t(zeros[g]) << (8 * i);
          }
          e[j].s01 = s[0] | s[1] << 16; e[j].s23 = s[2] | s[3] << 16;
          if (p.zeros) e[j].z = z;
        }
      }
    };
    if (p.rank && step1 == p.steps) {                // the correction's factor comes last: into the L2 meanwhile
      const char* from = static_cast<const char*>(p.second) + int64_t(tile) * kOut * 2;
      for (int k = threadIdx.x - 64; k < 2 * p.rank; k += 32 * kLoaders)
        if (tile * kOut + 64 * (k & 1) < p.out) asm volatile("prefetch.global.L2 [%0];" ::"l"(from + int64_t(k >> 1) * p.ld2 * 2 + 128 * (k & 1)));
    }
    uint32_t stage = (warp - 2) % p.ring, phase = 0;
    auto hand_over = [&](int k, const Entry (&e)[kPer]) {
      if (!warp_wait<true>(&bars->empty[stage], phase ^ 1u, abort_flag, p.status, 20u)) return false;
      const uint32_t at = scale_ring + stage * G::scale_bytes;
      const Form f = form(k);
#pragma unroll
      for (int j = 0; j < kPer; ++j) {
        uint32_t s01 = e[j].s01, s23 = e[j].s23, z = e[j].z;
        if (f == kPair) { s23 = __byte_perm(s01, 0, 0x3232); s01 = __byte_perm(s01, 0, 0x1010); if (p.zeros) z = __byte_perm(z, 0, 0x1100); }
        else if (f == kOne) { s23 = s01 = __byte_perm(s01, 0, 0x1010); if (p.zeros) z = __byte_perm(z, 0, 0x0000); }
        asm volatile("st.shared.v2.u32 [%0], {%1, %2};" ::"r"(at + (32 * j + lane) * 8), "r"(s01), "r"(s23) : "memory");
        asm volatile("st.shared.u32 [%0], %1;" ::"r"(at + G::cols * 8 + (32 * j + lane) * 4), "r"(z) : "memory");
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&bars->full[stage]);
      stage += loaders;
      while (stage >= uint32_t(p.ring)) { stage -= p.ring; phase ^= 1u; }
      return true;
    };
    // A loader that waits for step k has handed over step k - loaders, so step k - loaders - ring has left the
    // ring; with loaders <= ring that covers step k - 2 ring, and the parity it waits for cannot be that of the phase before.
    int k = warp - 2 < loaders ? step0 + warp - 2 : step1;
    fetch(k, even);
    while (k < step1) {
      fetch(k + loaders, odd);
      if (!(ok = hand_over(k, even))) break;
      if ((k += loaders) >= step1) break;
      fetch(k + loaders, even);
      if (!(ok = hand_over(k, odd))) break;
      k += loaders;
    }
  } else {
    const int id = threadIdx.x - 32 * (2 + kLoaders), group = id >> 7;
    // column of W within the step; for 'T' that is the output, which has to be this thread's lane of tensor memory
    const int row = TRANS ? 32 * (warp & 3) + lane : kFull ? id & 127 : id & 63, half = kFull ? 0 : (id >> 6) & 1;
    const uint32_t swz = (row & 7) << 4;
    const int ragged = p.m % kStep ? p.code_steps - 1 : -1;        // 'T': the step that ends behind the last row
    // An operand buffer is free when the step before on it, k - bufs, was multiplied: the barrier that also frees that step's ring
    // stage.  A group waits for its own steps only and a barrier cannot overtake it: step k + ring is not loaded, and step
    // k - bufs + ring >= k not multiplied, before step k was, which needs this group (bufs <= ring).  It cannot be early either:
    // after its first wait all steps up to k - bufs are known to be multiplied, so step k's stage is in its last or this phase, and
    // its wait for step k - groups before told the same of step k - groups - bufs (groups <= ring).
    // The group's first warp polls, the others wait at a barrier that also tells them whether it gave up.
    auto group_wait = [&](uint64_t* free, uint32_t free_parity, uint64_t* full, uint32_t full_parity) {
      uint32_t good = 1;
      if (((id >> 5) & 3) == 0) {
        if (free) good = warp_wait<false>(free, free_parity, abort_flag, p.status, 17u);
        if (good) good = warp_wait<false>(full, full_parity, abort_flag, p.status, 16u);
      }
      asm volatile("{\n\t.reg .pred p, q;\n\tsetp.ne.u32 p, %0, 0;\n\tbar.red.and.pred q, %1, 128, p;\n\tselp.u32 %0, 1, 0, q;\n\t}"
                   : "+r"(good) : "r"(group + 1) : "memory");
      return good != 0;
    };
    auto group_sync = [&] { asm volatile("bar.sync %0, 128;" ::"r"(group + 1) : "memory"); };
    uint32_t stage = group, phase = 0, buf = group;
    for (int k = group < p.groups ? step0 + group : step1; k < step1; k += p.groups) {
      const int s = k - step0 - p.bufs;
      if (!(ok = group_wait(s >= 0 ? &bars->empty[s % p.ring] : nullptr, (s / p.ring) & 1, &bars->full[stage], phase))) break;
      const uint32_t dst = operand + buf * G::operand_bytes + row * 128;
      const uint32_t tdst = tmem + (uint32_t(32 * (warp & 3)) << 16) + p.nt_cols + buf * G::operand_cols;
      if (TRANS) tc_fence_after();
      if (k < p.code_steps) {
        const uint32_t at = scale_ring + stage * G::scale_bytes, codes = base + stage * G::code_bytes + row * 64, chunk = (row >> 1) & 3;
        constexpr int kQuarters = kFull ? 4 : 2;
        uint32_t s[2], z; uint4 q[kQuarters];
        asm volatile("ld.shared.v2.u32 {%0, %1}, [%2];" : "=r"(s[0]), "=r"(s[1]) : "r"(at + row * 8));
        asm volatile("ld.shared.u32 %0, [%1];" : "=r"(z) : "r"(at + G::cols * 8 + row * 4));
        if (TRANS && k == ragged) {
          // rows behind the last one: their X is zero, but what is stored there times the scale may be infinite.  Done in place, so that the
          // other steps keep their loads together.
#pragma unroll 1
          for (int c = 0; c < 4; ++c) {
            const uint32_t there = codes + ((c ^ chunk) << 4);
            const uint4 w = lds128(there);
            const int left = p.m - k * kStep - 8 * c;
            sts128(there, rows_only(w.x, left, z & 15), rows_only(w.y, left - 32, (z >> 8) & 15), rows_only(w.z, left - 64, (z >> 16) & 15), rows_only(w.w, left - 96, (z >> 24) & 15));
          }
        }
#pragma unroll
        for (int c = 0; c < kQuarters; ++c) q[c] = lds128(codes + (((2 * half + c) ^ chunk) << 4));
#pragma unroll
        for (int pair = 0; pair < 2; ++pair) {
          typename Scale<T>::Ready r[2];
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            Scale<T> sc; sc.bits = uint16_t(s[pair] >> (16 * i)); sc.zero = (z >> (16 * pair + 8 * i)) & 0xff;
            r[i] = sc.ready();
          }
          auto word = [&](int i, int c) { return pair == 0 ? (i == 0 ? q[c].x : q[c].y) : (i == 0 ? q[c].z : q[c].w); };
          if constexpr (TRANS) {
            uint32_t o[32];
#pragma unroll
            for (int i = 0; i < 2; ++i)
#pragma unroll
              for (int c = 0; c < kQuarters; ++c) Scale<T>::word(word(i, c), r[i], o + 16 * i + 4 * c);
            tmem_st32(tdst + pair * 32, o);
          } else {
#pragma unroll
            for (int i = 0; i < 2; ++i)
#pragma unroll
              for (int c = 0; c < kQuarters; ++c) {
                uint32_t o[4]; Scale<T>::word(word(i, c), r[i], o);
                sts128(dst + pair * (G::operand_bytes / 2) + (((4 * i + 2 * half + c) << 4) ^ swz), o[0], o[1], o[2], o[3]);
              }
          }
        }
      } else {
        // correction step: entry (output, c) of the operand is second(output, c mod rank16), c < Parts::all rank16; mid is zero behind the rank
        const uint16_t* second = static_cast<const uint16_t*>(p.second);
        const int c0 = (k - p.code_steps) * kStep;
        if constexpr (TRANS) {
          // 32 columns from c at a time through the stage's own, now idle, code buffer: rows of 128 outputs in, one output's values out
          uint32_t o[32];
          const uint32_t turn = base + stage * G::code_bytes;
          const uint16_t* from = second + tile * kOut;
          const int valid = p.out - tile * kOut;
          auto gather = [&](int c, uint32_t* to) {
            uint4 v[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const int e = (id & 127) + 128 * i, chunk = e & 15;
              int a = c + (e >> 4);
              if (a >= 2 * p.rank16) a -= 2 * p.rank16;
              if (a >= p.rank16) a -= p.rank16;
              v[i] = load8(reinterpret_cast<const T*>(from + int64_t(a) * p.ld2) + chunk * 8, a < p.rank ? valid - chunk * 8 : 0, p.second_aligned != 0);
            }
            group_sync();
#pragma unroll
            for (int i = 0; i < 4; ++i) sts128(turn + ((id & 127) + 128 * i) * 16, v[i].x, v[i].y, v[i].z, v[i].w);
            group_sync();
#pragma unroll
            for (int e = 0; e < 16; ++e) {
              uint16_t lo, hi;
              asm volatile("ld.shared.u16 %0, [%1];" : "=h"(lo) : "r"(turn + (2 * e) * 256 + row * 2));
              asm volatile("ld.shared.u16 %0, [%1];" : "=h"(hi) : "r"(turn + (2 * e + 1) * 256 + row * 2));
              to[e] = uint32_t(lo) | uint32_t(hi) << 16;
            }
          };
          // of half the parts are made here; they begin at multiples of 16 columns
          auto store = [&](int pair) {
            if constexpr (Parts<T>::split) {
#pragma unroll
              for (int e = 0; e < 32; e += 4) {
                const int column = c0 + 64 * pair + 2 * e;
                uint32_t part[4] = {};
                if (column < Parts<T>::all * p.rank16) {
#pragma unroll
                  for (int i = 0; i < 4; ++i) part[i] = factor_part(o[e + i], column >= Parts<T>::mid * p.rank16);
                }
                tmem_st4(tdst + pair * 32 + e, part);
              }
            } else tmem_st32(tdst + pair * 32, o);
          };
          if (p.rank16 <= 64 && 64 % p.rank16 == 0) {                // the pattern repeats every 64 columns
            gather(0, o);
            if (p.rank16 == 64) gather(32, o + 16);
            else {
#pragma unroll
              for (int e = 0; e < 16; ++e) o[16 + e] = o[e];
            }
            store(0); store(1);
          } else {
#pragma unroll 1
            for (int pair = 0; pair < 2; ++pair) {
              const int c = (c0 + pair * 64) % (2 * p.rank16);
              gather(c, o); gather((c + 32) % (2 * p.rank16), o + 16);
              store(pair);
            }
          }
        } else {
          const int c = c0 + row, of = Parts<T>::split ? c % p.rank16 : c < p.rank16 ? c : c - p.rank16;
          const uint16_t* from = second + int64_t(of) * p.ld2 + tile * kOut + 64 * half;
          const int valid = c < Parts<T>::all * p.rank16 && of < p.rank ? p.out - tile * kOut - 64 * half : 0;
#pragma unroll 4
          for (int j = 0; j < (kFull ? 16 : 8); ++j) {
            uint4 v = load8(reinterpret_cast<const T*>(from) + 8 * j, valid - 8 * j, p.second_aligned != 0);
            if (Parts<T>::split) { const bool rest = c >= Parts<T>::mid * p.rank16; v = make_uint4(factor_part(v.x, rest), factor_part(v.y, rest), factor_part(v.z, rest), factor_part(v.w, rest)); }
            sts128(dst + (half + (j >> 3)) * (G::operand_bytes / 2) + (((j & 7) << 4) ^ swz), v.x, v.y, v.z, v.w);
          }
        }
      }
      if (TRANS) {
        asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
        tc_fence_before();
      } else asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      __syncwarp();
      if (lane == 0) mbar_arrive(&bars->a_full[buf]);
      if ((buf += p.groups) >= uint32_t(p.bufs)) buf -= p.bufs;
      stage += p.groups;
      while (stage >= uint32_t(p.ring)) { stage -= p.ring; phase ^= 1u; }
    }
    // ---- accumulators: to Y, or to shared memory for the cluster's sum ----
    ok = ok && warp_wait<true>(&bars->done, 0u, abort_flag, p.status, 19u);
    if (ok) {
      tc_fence_after();
      const int quarter = warp & 3, side = (warp - 2 - kLoaders) >> 2, o = quarter * 32 + lane, out = tile * kOut + o;
      const uint32_t addr = tmem + (uint32_t(quarter * 32) << 16);
      float* red = reinterpret_cast<float*>(aligned);
      for (int c = side * 8; c < p.nt; c += 8 * kGroups) {
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

// ---- mid = first^T X for many tokens, in bfloat16 parts: [token][Parts::all][entry of the rank], each padded with zeros to a multiple of 16 ----------
template <class T> __device__ __forceinline__ void mma16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1);
template <> __device__ __forceinline__ void mma16816<__half>(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
template <> __device__ __forceinline__ void mma16816<__nv_bfloat16>(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

constexpr int kMidWarps = 8, kMidSplits = 8;
// A cluster of eight blocks: 16 entries of the rank x 16 tokens, the blocks and their warps split the rows, sums joined in shared memory
// and across the cluster in a fixed order.  A lane feeds eight consecutive rows of each operand row to two instructions: the
// order of K inside an instruction is free as long as both operands agree.  The product waits for this kernel, so what counts is
// its latency: 4096 rows, rank 64, 256 tokens took 9 us with one block per tile.
template <class T> __global__ void __launch_bounds__(kMidWarps * 32)
mid_split_kernel(const T* first, int64_t ld1, int rows, int rank, const T* x, int64_t ldx, int t, __nv_bfloat16* mid, int64_t ldm, int aligned, float* mid32) {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  __shared__ float red[kMidWarps][16][17];
  __shared__ __align__(16) float part[256];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, c = lane & 3;
  const int split = blockIdx.x % kMidSplits, k0 = blockIdx.x / kMidSplits * 16; const int64_t t0 = int64_t(blockIdx.y) * 16;
  const T* fp[2] = {first + int64_t(k0 + g) * ld1, first + int64_t(k0 + g + 8) * ld1};
  const T* xp[2] = {x + (t0 + g) * ldx, x + (t0 + g + 8) * ldx};
  const bool fl[2] = {k0 + g < rank, k0 + g + 8 < rank}, xl[2] = {t0 + g < t, t0 + g + 8 < t};
  float acc[2][4] = {};
#pragma unroll 4
  for (int64_t r0 = (split * kMidWarps + warp) * 32; r0 < rows; r0 += kMidSplits * kMidWarps * 32) {
    const int64_t r = r0 + c * 8; const int valid = int(rows - r);
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
  {
    for (int e = threadIdx.x; e < 256; e += kMidWarps * 32) {
      float s = 0.f;
#pragma unroll
      for (int w = 0; w < kMidWarps; ++w) s += red[w][e & 15][e >> 4];
      part[e] = s;
    }
  }
  cluster_sync_all();
  if (threadIdx.x < 256 / kMidSplits / 4) {
    const int e = split * (256 / kMidSplits) + threadIdx.x * 4;
    float4 s = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int r = 0; r < kMidSplits; ++r) { const float4 v = ld_cluster4(smem_u32(part + e), r); s.x += v.x; s.y += v.y; s.z += v.z; s.w += v.w; }
    const float v[4] = {s.x, s.y, s.z, s.w};
    const int tok = e >> 4;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int k = k0 + (e & 15) + i;
      if (mid32) { if (t0 + tok < t && k < rank) mid32[(t0 + tok) * rank + k] = v[i]; }      // for the streaming kernel, in one part
      else if (t0 + tok < t) {                       // zeros behind the rank
        __nv_bfloat16* m = mid + (t0 + tok) * ldm + k;
        const int64_t next = ldm / Parts<T>::all;
        const bool finite = fabsf(v[i]) <= 3.402823466e38f;      // an infinity or a NaN is one part: what it left would be a NaN
        if constexpr (Parts<T>::split) {
          float rest = v[i];
          __nv_bfloat16 p[3];
#pragma unroll
          for (int q = 0; q < 3; ++q) { p[q] = __float2bfloat16_rz(rest); rest = finite ? rest - __bfloat162float(p[q]) : 0.f; }
#pragma unroll
          for (int q = 0; q < 3; ++q) m[q * next] = p[q];
          m[3 * next] = finite ? p[0] : __float2bfloat16_rn(0.f); m[4 * next] = p[1];
        } else {
          const __nv_bfloat16 value = __float2bfloat16_rn(v[i]);
          m[0] = value; m[next] = __float2bfloat16_rn(finite ? v[i] - __bfloat162float(value) : 0.f);
        }
      }
    }
  }
  cluster_sync_all();
}

template <class T> cudaError_t start_mid(const hyacinHandle_t* handle, const T* first, int64_t ld1, int rows, int rank, const T* x, int64_t ldx, int t, __nv_bfloat16* mid, int64_t ldm, int aligned, float* mid32) {
  cudaLaunchConfig_t mc{};
  mc.gridDim = dim3(unsigned((rank + 15) / 16) * kMidSplits, unsigned((int64_t(t) + 15) / 16)); mc.blockDim = dim3(kMidWarps * 32); mc.stream = handle->cudaStream;
  cudaLaunchAttribute ma[1];
  ma[0].id = cudaLaunchAttributeClusterDimension; ma[0].val.clusterDim.x = kMidSplits; ma[0].val.clusterDim.y = 1; ma[0].val.clusterDim.z = 1;
  mc.attrs = ma; mc.numAttrs = 1;
  // the product's blocks move in beside this kernel's only if the SM is already split between cache and shared memory their way
  static std::atomic<uint64_t> carved{0};
  const uint64_t bit = uint64_t(1) << (handle->DeviceID & 63);
  if (!(carved.load() & bit)) {
    HYB_CUDA(cudaFuncSetAttribute(mid_split_kernel<T>, cudaFuncAttributePreferredSharedMemoryCarveout, cudaSharedmemCarveoutMaxShared));
    carved.fetch_or(bit);
  }
  count_launch();
  return cudaLaunchKernelEx(&mc, mid_split_kernel<T>, first, ld1, rows, rank, x, ldx, t, mid, ldm, aligned, mid32);
}

// X with rows that TMA can address (16-byte pitch and start).
__global__ void __launch_bounds__(256) align_rows_kernel(const uint16_t* x, int64_t ldx, int rows, uint16_t* out, int64_t ldo) {
  const int64_t r = int64_t(blockIdx.x) * 256 + threadIdx.x;
  if (r < rows) out[int64_t(blockIdx.y) * ldo + r] = x[int64_t(blockIdx.y) * ldx + r];
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

// CTAs that share a tile's K steps: the whole takes ceil(tiles s / slots) rounds of ceil(steps / s) steps plus `overhead` steps' worth of
// start, drain and exchange.
int choose_splits(int64_t tiles, int steps, int slots, int overhead) {
  int best = 1; double cost = 1e300;
  for (int s = 1; s <= 8 && s * 2 <= std::max(steps, 2); ++s) {
    const double c = double((tiles * s + slots - 1) / slots) * ((steps + s - 1) / s + overhead);
    if (c < cost * 0.999) { cost = c; best = s; }
  }
  return best;
}

template <class T, bool TRANS, int STEP> int32_t launch(const hyacinHandle_t* handle, const char* fn, hyacinPrecision_t type, const ProductArgs& a) {
  cudaStream_t stream = handle->cudaStream;
  const int in = TRANS ? a.m : a.n, out = TRANS ? a.n : a.m;
  void *x_copy = nullptr, *mid = nullptr;
  auto cleanup = [&] { if (x_copy) HYB_CUDA(cudaFreeAsync(x_copy, stream)); if (mid) HYB_CUDA(cudaFreeAsync(mid, stream)); };
  auto allocate = [&](void** p, size_t bytes) {
    const cudaError_t e = cudaMallocFromPoolAsync(p, bytes, handle->mempool, stream);
    if (w4_result(e, "cudaMallocFromPoolAsync")) *p = nullptr;
    return e == cudaSuccess;
  };
  const void* x = a.x; int64_t ldx = a.ldx;
  if (a.t == 1) ldx = (int64_t(in) + 7) / 8 * 8;                 // a single column has no pitch
  if (reinterpret_cast<uintptr_t>(x) % 16 || ldx % 8) {
    const int64_t ldo = (int64_t(in) + 7) / 8 * 8;
    if (!allocate(&x_copy, size_t(ldo) * a.t * 2)) return -3;
    for (int64_t t = 0; t < a.t; t += 65535) {
      count_launch();
      const cudaError_t e = w4_start(align_rows_kernel, dim3((in + 255) / 256, unsigned(std::min<int64_t>(65535, a.t - t))), 256, 0, stream,
                                     static_cast<const uint16_t*>(a.x) + t * a.ldx, a.ldx, in, static_cast<uint16_t*>(x_copy) + t * ldo, ldo);
      if (e != cudaSuccess) { cleanup(); return w4_result(e, fn); }
    }
    x = x_copy; ldx = ldo;
  }
  UmmaParams p{};
  p.scales = a.scales; p.zeros = a.zeros; p.lds = a.lds; p.m = a.m; p.n = a.n; p.t = a.t; p.out = out;
  p.segs = w4_segments(a.m, a.seg); p.seg_sub = a.seg / 32; p.seg_shift = -1;
  for (int s = 0; s < 27; ++s) if (p.seg_sub == 1 << s) p.seg_shift = s;
  // two or four segments per block of 128 rows, fetched at once where the table's rows allow it
  const int per_block = p.seg_sub == 1 ? 4 : p.seg_sub == 2 ? 2 : 1;
  p.wide = per_block > 1 && a.lds % per_block == 0 && reinterpret_cast<uintptr_t>(a.scales) % (2 * per_block) == 0 &&
           reinterpret_cast<uintptr_t>(a.zeros) % per_block == 0 ? per_block : 1;
  using G = Geometry<TRANS, STEP>;
  constexpr int kStep = G::step;
  p.code_steps = (in + kStep - 1) / kStep;
  p.rank = a.rank; p.rank16 = (a.rank + 15) / 16 * 16; p.second = a.second; p.ld2 = a.ld2; p.y = a.y; p.ldy = a.ldy;
  p.steps = p.code_steps + (Parts<T>::all * p.rank16 + kStep - 1) / kStep;
  const int64_t token_tiles = (int64_t(a.t) + kMaxTokens - 1) / kMaxTokens;
  p.nt = int((int64_t(a.t) + token_tiles - 1) / token_tiles + 15) / 16 * 16;
  p.nt_cols = (p.nt + 31) / 32 * 32;

  const uint32_t x_bytes = uint32_t(p.nt) * kStep * 2, stage_bytes = G::code_bytes + x_bytes + G::scale_bytes;
  // operand buffers: as many as leave the ring as many stages; with 'T' they share the 512 columns with the accumulators
  const uint32_t fixed = 1024 + sizeof(UmmaBars);
  p.bufs = TRANS ? std::min<int>(kMaxBufs, (512 - p.nt_cols) / std::max<uint32_t>(G::operand_cols, 1)) : kMaxBufs;
  for (;; --p.bufs) {
    p.ring = int(std::min<uint32_t>(kMaxRing, (kSmemLimit - fixed - p.bufs * G::operand_bytes) / stage_bytes));
    if (p.ring >= p.bufs) break;
  }
  p.groups = std::min(kGroups, p.bufs);
  p.tmem_cols = 32;
  while (p.tmem_cols < p.nt_cols + p.bufs * G::operand_cols) p.tmem_cols *= 2;
  const uint32_t smem = std::max(fixed + p.bufs * G::operand_bytes + p.ring * stage_bytes, kSmemFloor);
  p.second_aligned = reinterpret_cast<uintptr_t>(a.second) % 16 == 0 && a.ld2 % 8 == 0;
  const int tiles = (out + kOut - 1) / kOut;
  p.splits = choose_splits(int64_t(tiles) * token_tiles, p.steps, handle->DeviceSMs, kStep == 128 ? 6 : 12);
  const uint32_t fmt = type == HYACIN_F16 ? 0u : 1u;
  p.idesc_more = (1u << 4) | (1u << 7) | (1u << 10) | ((TRANS ? 0u : 1u) << 15) | (uint32_t(p.nt >> 3) << 17) | (uint32_t(kOut >> 4) << 24);
  p.idesc = (p.idesc_more & ~((1u << 7) | (1u << 10))) | (fmt << 7) | (fmt << 10);
  p.status = status_word_device(handle->DeviceID);
  const CUtensorMapDataType dt = type == HYACIN_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
  CUtensorMap code_map{}, x_map{}, mid_map{};
  bool fine = encode_2d(&code_map, CU_TENSOR_MAP_DATA_TYPE_UINT8, a.codes, uint64_t((a.m + 127) / 128) * 64, a.n, a.ldq, 64, G::cols, CU_TENSOR_MAP_SWIZZLE_64B) &&
              encode_2d(&x_map, dt, x, in, a.t, uint64_t(ldx) * 2, 64, p.nt, CU_TENSOR_MAP_SWIZZLE_128B);
  mid_map = x_map;
  if (fine && a.rank) {
    const int64_t ldm = Parts<T>::all * int64_t(p.rank16);
    if (!allocate(&mid, size_t(ldm) * a.t * 2)) { cleanup(); return -3; }
    fine = encode_2d(&mid_map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, mid, uint64_t(ldm), a.t, uint64_t(ldm) * 2, 64, p.nt, CU_TENSOR_MAP_SWIZZLE_128B);
    const int aligned = reinterpret_cast<uintptr_t>(x) % 16 == 0 && ldx % 8 == 0 && reinterpret_cast<uintptr_t>(a.first) % 16 == 0 && a.ld1 % 8 == 0;
    const cudaError_t e = start_mid<T>(handle, static_cast<const T*>(a.first), a.ld1, in, a.rank, static_cast<const T*>(x), ldx, a.t, static_cast<__nv_bfloat16*>(mid), ldm, aligned, nullptr);
    if (w4_result(e, fn)) fine = false;
  }
  if (!fine) { cleanup(); return -3; }
  auto* kernel = product_umma_kernel<T, TRANS, STEP>;
  static std::atomic<uint64_t> ready{0};                         // per device: shared memory limit raised
  const uint64_t bit = uint64_t(1) << (handle->DeviceID & 63);
  if (!(ready.load() & bit)) {
    const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmemLimit);
    if (e != cudaSuccess) { cleanup(); return w4_result(e, "cudaFuncSetAttribute"); }
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
  cleanup();
  return w4_result(e, fn);
}

}  // namespace

cudaError_t launch_mid_float(const hyacinHandle_t* handle, hyacinPrecision_t type, const void* first, int64_t ld1, int rows, int rank, const void* x, int64_t ldx, int t, float* mid, bool aligned) {
  if (type == HYACIN_F16) return start_mid<__half>(handle, static_cast<const __half*>(first), ld1, rows, rank, static_cast<const __half*>(x), ldx, t, nullptr, 0, aligned, mid);
  return start_mid<__nv_bfloat16>(handle, static_cast<const __nv_bfloat16*>(first), ld1, rows, rank, static_cast<const __nv_bfloat16*>(x), ldx, t, nullptr, 0, aligned, mid);
}

int32_t launch_product_umma(const hyacinHandle_t* handle, const char* fn, bool trans, hyacinPrecision_t type, const ProductArgs& a) {
  constexpr int kMostTokens = 1 << 19;                           // of one launch: the grids' second dimensions end at 65535
  if (a.t > kMostTokens) {
    int32_t rc = 0;
    for (int64_t t0 = 0; t0 < a.t && rc == 0; t0 += kMostTokens) {
      ProductArgs b = a;
      b.t = int(std::min<int64_t>(kMostTokens, a.t - t0));
      b.x = static_cast<const uint16_t*>(a.x) + t0 * a.ldx; b.y = static_cast<uint16_t*>(a.y) + t0 * a.ldy;
      rc = launch_product_umma(handle, fn, trans, type, b);
    }
    return rc;
  }
  // opW 'N' keeps its operand in shared memory.  Steps of 128 columns halve the hand-overs between the warps' roles (4096 x 16384 times 64
  // tokens 28 against 36 us), but beside tiles of more than 128 tokens only two of them fit (times 256: 47 against 42 us).
  const bool small = a.t <= 128;
  if (type == HYACIN_F16) return trans ? launch<__half, true, 128>(handle, fn, type, a) : small ? launch<__half, false, 128>(handle, fn, type, a) : launch<__half, false, 64>(handle, fn, type, a);
  return trans ? launch<__nv_bfloat16, true, 128>(handle, fn, type, a) : small ? launch<__nv_bfloat16, false, 128>(handle, fn, type, a) : launch<__nv_bfloat16, false, 64>(handle, fn, type, a);
}

}  // namespace hyb
