// Y = Wq^T X + V (U^T X) for few vectors: every SM streams its columns' codes through shared memory with bulk copies and feeds
// warp-level matrix instructions from there.
//
// Mathematics.  Y(j, t) = sum over segments of s(j, seg) sum_{r in seg} (q(r, j) - zero) x(r, t).  A mask turns two codes into two
// 16-bit numbers offset + q (offset 1024 for half, 128 for bfloat16), and one subtraction into the exact whole numbers q - zero, which
// go into the instruction.  (Offset codes in the instruction and (offset + zero) sum x taken off afterwards would save those four of eleven
// instructions per eight codes, but for x of one sign the sums to be cancelled are a hundred times the result for half, the
// error a rounding of Y; and an infinite or very large x ends in infinity minus infinity.)  A segment's sum is multiplied by its scale in
// 32 bits; the only rounding to 16 bits is that of Y.  Single-precision x is split into three bfloat16 parts of 8 bits that add up to it
// exactly (down to 2^-110), three columns of the right-hand operand: the result is that of 32-bit sums.
// Layout.  A CTA (one per SM) takes every 148th tile of 16 columns, the rows of the m16n8k16 instruction.  A column's codes are
// contiguous; a stage of the ring holds 4096 rows of the tile (2048 for more than eight operand columns), one TMA box, so the copies for the next
// stages and tiles are in flight all the time (up to 190 KiB per SM) whatever the arithmetic does.  Each of 16 warps takes two
// blocks of 128 rows of the stage (one).  Lane (g, c) reads quarter c of the block's 64 bytes of columns g and g + 8: four words, word i
// holding rows 32 i + 8 c .. + 7.  The order of K inside an instruction is free as long as both operands use the same one, so the
// lane's four code pairs of a word meet the lane's 16 bytes of x for those eight rows, read from shared memory in their natural
// order.  Six more warps fetch scales and zero points, coalesced along a table row, into the
// same ring, and one adds the partial sums of the multiplying warps.
// Bound.  Latency: barrier, shared load, extraction, matrix instruction and scaling follow one another in each of the 16 warps.  Half 8192 x
// 16384 with zero points for every 64 rows uses 57 % of the issue slots, 15 % of the matrix pipe and 32 % of DRAM.  Measured, matrices
// cycled through more than the L2: that case 26.3 us (2.8 TB/s; 22.9 with segments of 128 rows); bfloat16 4096 x 16384, one vector 15.4 us
// (2.2 TB/s), eight 16.6 us; 4096 x 4096 7.0 us.  The subtraction of the offsets costs 0 to 5 % of these.
#include "w4_product.h"
#include "ptx_sm100.cuh"
#include <algorithm>
#include <atomic>
#include <type_traits>

namespace hyb {
namespace {
using namespace ptx;

constexpr int kTile = 16;                         // columns
constexpr int kWarps = 16;                        // multiplying warps
// blocks of 128 rows a warp takes from a stage: two while x leaves room for four such stages
__host__ __device__ constexpr int blocks_per_warp(int tiles) { return tiles == 1 ? 2 : 1; }
constexpr int kLoaders = 6;                       // warps that fetch scales
constexpr int kJoints = 2;                        // buffers for the partial sums of a tile
constexpr int kThreads = 32 * (kWarps + kLoaders + 2);
constexpr int kMaxRing = 8;
constexpr int kSmemLimit = 232448;

struct StreamParams {
  int m, n, t;
  const void* scales; const uint8_t* zeros; int64_t lds;
  const void* x; int64_t ldx;
  int rank; const void* second; int64_t ld2; const float* mid;
  void* y; int64_t ldy;
  int segs, seg_sub, seg_shift;                   // 32-row subsets per segment, its logarithm or -1
  int blocks, cols, tiles, ring, pitch, x_aligned;       // pitch: of x in shared memory, elements
  int ring_at, pairs_at, red_at, bars_at;
  uint32_t* status;
};

struct StreamBars { uint64_t full[kMaxRing], empty[kMaxRing], joint_full[kJoints], joint_empty[kJoints]; uint32_t abort_flag; };

// Two codes each: offset + q as extracted, by joining the code's bits to the exponent of a number whose last places are whole (the classic
// conversion of integers, e.g. Warren, Hacker's Delight, 2003; for 4-bit weights in half Kim et al., arXiv:2211.10017, 2022).
template <bool HALF> struct Codes;
template <> struct Codes<true> {       // 0x6400 | q = 1024 + q
  static constexpr uint32_t kBits = 0x64006400u; static constexpr int kOffset = 1024;
  static __device__ __forceinline__ void mma(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  }
};
template <> struct Codes<false> {      // 0x4300 | q = 128 + q
  static constexpr uint32_t kBits = 0x43004300u; static constexpr int kOffset = 128;
  static __device__ __forceinline__ void mma(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  }
};
// (w & mask) | bits in one instruction: left to the compiler, two constants became two instructions
__device__ __forceinline__ uint32_t and_or(uint32_t w, uint32_t mask, uint32_t bits) {
  uint32_t r;
  asm("lop3.b32 %0, %1, %2, %3, 0xEA;" : "=r"(r) : "r"(w), "r"(mask), "r"(bits));
  return r;
}
template <bool HALF> __device__ __forceinline__ void code_pairs(uint32_t w, uint32_t (&o)[4]) {
#pragma unroll
  for (int p = 0; p < 4; ++p) o[p] = and_or(w >> (4 * p), 0x000f000fu, Codes<HALF>::kBits);
}
// Pairs q - zero; low: -(offset + zero) twice.
template <bool HALF> __device__ __forceinline__ void subtract_zero(uint32_t (&o)[4], uint32_t low) {
  using Two = std::conditional_t<HALF, __half2, __nv_bfloat162>;
#pragma unroll
  for (int p = 0; p < 4; ++p) {
    const Two v = __hadd2(*reinterpret_cast<Two*>(&o[p]), *reinterpret_cast<const Two*>(&low));
    o[p] = *reinterpret_cast<const uint32_t*>(&v);
  }
}

// Scale and -(offset + zero) of one (column, segment), as kept in shared memory: two numbers of the scale's own type, which holds
// offset + zero exactly (float: the second as bfloat16, twice).
template <class X> struct Pair {
  uint32_t bits;
  __device__ __forceinline__ float scale() const { const uint16_t s = uint16_t(bits); return to_f32(*reinterpret_cast<const X*>(&s)); }
  __device__ __forceinline__ uint32_t low() const { return __byte_perm(bits, 0, 0x3232); }
};
template <> struct Pair<float> {
  float s; uint32_t twice;
  __device__ __forceinline__ float scale() const { return s; }
  __device__ __forceinline__ uint32_t low() const { return twice; }
};
template <class X> __device__ __forceinline__ Pair<X> make_pair(X scale, int zero) {
  if constexpr (sizeof(X) == 4) return {scale, 0xc300c300u + uint32_t(zero) * 0x10001u};
  else {
    const X off = from_f32<X>(-float(Codes<std::is_same<X, __half>::value>::kOffset + zero));
    return {uint32_t(*reinterpret_cast<const uint16_t*>(&scale)) | uint32_t(*reinterpret_cast<const uint16_t*>(&off)) << 16};
  }
}


__device__ __forceinline__ int segment_of(int sub, const StreamParams& p) { return p.seg_shift >= 0 ? sub >> p.seg_shift : sub / p.seg_sub; }

// Bounded wait of a whole warp (a poll by a single lane is not suspended by the hardware and costs the others issue slots).
__device__ __forceinline__ bool warp_wait(uint64_t* bar, uint32_t parity, volatile uint32_t* abort_flag, uint32_t* status, uint32_t code) {
#pragma unroll 1
  for (uint32_t it = 0; it < (1u << 20); ++it) {
    if (__all_sync(~0u, mbar_try_wait(bar, parity))) return true;
    if (__any_sync(~0u, *abort_flag)) return false;
    if (it > 1024) __nanosleep(256);
  }
  if ((threadIdx.x & 31) == 0) { *abort_flag = 1u; *reinterpret_cast<volatile uint32_t*>(status) = code; }
  __syncwarp();
  return false;
}

// X: type of x; TILES: eights of operand columns (vectors, or their parts); GRAIN: 32-row subsets that share a scale for sure: 4 when
// segments are whole blocks, else 2 or 1.
template <class X, int TILES, int GRAIN>
__global__ void __launch_bounds__(kThreads, 1) product_stream_kernel(const __grid_constant__ CUtensorMap code_map, const __grid_constant__ StreamParams p) {
  constexpr bool kSplit = sizeof(X) == 4, kHalf = std::is_same<X, __half>::value;
  constexpr int kPer = blocks_per_warp(TILES), kStageBlocks = kWarps * kPer, kColumnPitch = kStageBlocks * 64;      // pitch: bytes of a column in a stage
  constexpr int kPairs = 4 / GRAIN * kStageBlocks + 1;       // scales of a column in a stage; odd, so that columns fall into different banks
  constexpr int kRed = 8 * TILES + 1;
  extern __shared__ __align__(128) uint8_t smem[];
  uint16_t* xs = reinterpret_cast<uint16_t*>(smem);                // [operand column][row]
  uint8_t* ring = smem + p.ring_at;
  Pair<X>* pairs = reinterpret_cast<Pair<X>*>(smem + p.pairs_at);  // [stage][column][segment of the stage]
  float* red = reinterpret_cast<float*>(smem + p.red_at);          // [joint][warp][column][operand column]
  StreamBars* bars = reinterpret_cast<StreamBars*>(smem + p.bars_at);
  volatile uint32_t* abort_flag = &bars->abort_flag;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int tiles = (p.n + kTile - 1) / kTile, stages = (p.blocks + kStageBlocks - 1) / kStageBlocks;      // stages per tile

  // stage number `at` of this CTA: tile blockIdx.x + (at / stages) gridDim.x, chunk at % stages of the rows
  const int my_tiles = (tiles - int(blockIdx.x) + int(gridDim.x) - 1) / int(gridDim.x), total = my_tiles * stages;
  auto copy = [&](int tile, int chunk, int stage) {
    mbar_expect_tx(&bars->full[stage], kTile * kColumnPitch);
    tma_load_2d(smem_u32(ring) + stage * kTile * kColumnPitch, &code_map, &bars->full[stage], chunk * (kColumnPitch / 8), tile * kTile);
  };
  if (threadIdx.x == 0) {
    prefetch_map(&code_map);
    for (int s = 0; s < p.ring; ++s) { mbar_init(&bars->full[s], 2); mbar_init(&bars->empty[s], kWarps); }
    for (int j = 0; j < kJoints; ++j) { mbar_init(&bars->joint_full[j], kWarps); mbar_init(&bars->joint_empty[j], 1); }
    bars->abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  __syncthreads();

  bool ok = true;
  if (warp == 0) {
    // ---- codes ----
    int tile = blockIdx.x, chunk = 0; uint32_t stage = 0, phase = 0;
    for (int at = 0; at < total; ++at) {
      if (at >= p.ring && !(ok = warp_wait(&bars->empty[stage], phase ^ 1u, abort_flag, p.status, 31u))) break;
      if (lane == 0) copy(tile, chunk, stage);
      __syncwarp();
      if (++chunk == stages) { chunk = 0; tile += gridDim.x; }
      if (++stage == uint32_t(p.ring)) { stage = 0; phase ^= 1u; }
    }
    if (!ok) {      // some role gave up: let the copies in flight land before the block can end
      uint32_t ignore = 0;
      for (int s = 0; s < p.ring; ++s) {
        if (stage == 0) { stage = p.ring; phase ^= 1u; }
        --stage;
        if (lane == 0) mbar_wait(&bars->full[stage], phase, &ignore, p.status, 32u);
      }
    }
  } else if (warp <= kLoaders) {
    // ---- scales and zero points: loader l takes stages l, l + loaders, ... ----
    // A loader that waits for stage number `at` has handed over number at - loaders, so number at - loaders - ring has left the ring;
    // with loaders <= ring that covers at - 2 ring, and the parity it waits for cannot be that of the phase before.
    const int loaders = min(kLoaders, p.ring), l = warp - 1;
    for (int at = l < loaders ? l : total; at < total; at += loaders) {
      const int tile = int(blockIdx.x) + at / stages * int(gridDim.x), chunk = at % stages;
      const int sub0 = chunk * kStageBlocks * 4, seg0 = segment_of(sub0, p);
      const int count = min(segment_of(min(sub0 + kStageBlocks * 4, p.blocks * 4) - 1, p), p.segs - 1) - seg0 + 1;
      const int cols = min(kTile, p.n - tile * kTile);
      const uint32_t stage = at % p.ring, phase = (at / p.ring) & 1;
      // lanes per column: as many as it has segments here, so that a load's lanes touch few lines
      const int log = count > 16 ? 5 : count > 8 ? 4 : count > 4 ? 3 : count > 2 ? 2 : count > 1 ? 1 : 0;
      const int first = lane >> log, step = 32 >> log;
      Pair<X>* out = pairs + stage * kTile * kPairs;
      bool waited = false;
      for (int s0 = 0; s0 < count; s0 += 32) {
        const int s = s0 + (lane & ((1 << log) - 1));
#pragma unroll 1
        for (int c0 = 0; c0 < cols; c0 += 16 * step) {
          X scale[16]; uint8_t zero[16];
#pragma unroll
          for (int u = 0; u < 16; ++u) {
            const int col = c0 + first + u * step;
            const int64_t at_table = int64_t(tile * kTile + col) * p.lds + seg0 + s;
            if (col < cols && s < count) { scale[u] = static_cast<const X*>(p.scales)[at_table]; zero[u] = p.zeros ? p.zeros[at_table] : uint8_t(8); }
          }
          if (!waited) { if (!(ok = warp_wait(&bars->empty[stage], phase ^ 1u, abort_flag, p.status, 33u))) break; waited = true; }
#pragma unroll
          for (int u = 0; u < 16; ++u) {
            const int col = c0 + first + u * step;
            if (col < cols && s < count) out[col * kPairs + s] = make_pair<X>(scale[u], int(zero[u]));
          }
        }
        if (!ok) break;
      }
      if (!ok) break;
      __syncwarp();
      if (lane == 0) mbar_arrive(&bars->full[stage]);
    }
  } else if (warp == 1 + kLoaders) {
    // ---- joining: adds the multiplying warps' partial sums of a tile, so that they need not wait for one another ----
    uint32_t joint = 0, phase = 0;
    for (int tile = blockIdx.x; tile < tiles; tile += gridDim.x) {
      if (!(ok = warp_wait(&bars->joint_full[joint], phase, abort_flag, p.status, 35u))) break;
#pragma unroll 2
      for (int e = lane; e < kTile * p.t; e += 32) {
        const int col = e & (kTile - 1), t = e / kTile, out = tile * kTile + col;
        const float* from = red + joint * kWarps * kTile * kRed + col * kRed + (kSplit ? 3 * t : t);
        float v = 0.f;
#pragma unroll
        for (int q = 0; q < kWarps; ++q)
#pragma unroll
          for (int i = 0; i < (kSplit ? 3 : 1); ++i) v += from[q * kTile * kRed + i];
        if (out < p.n) static_cast<X*>(p.y)[int64_t(t) * p.ldy + out] = from_f32<X>(v);
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&bars->joint_empty[joint]);
      if (++joint == kJoints) { joint = 0; phase ^= 1u; }
    }
  } else {
    // ---- products ----
    const int w = warp - 2 - kLoaders, g = lane >> 2, c = lane & 3;
    // First x, one operand column per line, zeros behind the last row, while the first codes arrive.
    {
      const int rows = p.blocks * kW4Block, tid = threadIdx.x - 32 * (2 + kLoaders), step = kWarps * 32;
      if constexpr (kSplit) {
        for (int t = 0; t < p.t; ++t)
#pragma unroll 4
          for (int r = tid; r < rows; r += step) {
            float v = r < p.m ? __ldg(static_cast<const float*>(p.x) + t * p.ldx + r) : 0.f;
#pragma unroll
            for (int k = 0; k < 3; ++k) {
              const __nv_bfloat16 h = __float2bfloat16_rz(v);
              xs[(3 * t + k) * p.pitch + r] = __bfloat16_as_ushort(h);
              v = fabsf(v) <= 3.402823466e38f ? v - __bfloat162float(h) : 0.f;
            }
          }
      } else {
        // eight rows per thread and step
        const int per = rows / 8, chunks = p.t * per;
#pragma unroll 4
        for (int e = tid; e < chunks; e += step) {
          const int t = e / per, r = (e - t * per) * 8, valid = p.m - r;
          const uint16_t* src = static_cast<const uint16_t*>(p.x) + t * p.ldx + r;
          uint4 v;
          if (p.x_aligned && valid >= 8) v = __ldg(reinterpret_cast<const uint4*>(src));
          else {
            uint32_t o[4] = {0, 0, 0, 0};
#pragma unroll
            for (int i = 0; i < 8; ++i) if (i < valid) o[i >> 1] |= uint32_t(__ldg(src + i)) << (16 * (i & 1));
            v = make_uint4(o[0], o[1], o[2], o[3]);
          }
          *reinterpret_cast<uint4*>(xs + t * p.pitch + r) = v;
        }
      }
      asm volatile("bar.sync 1, %0;" ::"n"(kWarps * 32) : "memory");
    }
    const uint16_t* xl[TILES];
#pragma unroll
    for (int j = 0; j < TILES; ++j) xl[j] = xs + min(8 * j + g, p.cols - 1) * p.pitch + 8 * c;
    uint32_t stage = 0, phase = 0, joint = 0, joint_phase = 0;
    for (int tile = blockIdx.x; tile < tiles; tile += gridDim.x) {
      float sum[TILES][4] = {};
      for (int chunk = 0; chunk < stages; ++chunk) {
        if (!(ok = warp_wait(&bars->full[stage], phase, abort_flag, p.status, 34u))) break;
        const uint8_t* from = ring + (stage * kTile + g) * kColumnPitch + w * 64 + c * 16;
        const Pair<X>* pa = pairs + (stage * kTile + g) * kPairs - segment_of(chunk * kStageBlocks * 4, p);
        const Pair<X>* pb = pa + 8 * kPairs;
        // one block: (q - zero) x in the matrix pipe, times the scale
        auto block = [&](int b, const uint4& qa, const uint4& qb) {
#pragma unroll
          for (int i0 = 0; i0 < 4; i0 += GRAIN) {
            // rows behind the last one meet zeros of x under the last segment's scale
            const int seg = GRAIN < 4 ? min(segment_of(4 * b + i0, p), p.segs - 1) : segment_of(4 * b, p);
            const Pair<X> va = pa[seg], vb = pb[seg];
            float acc[TILES][4] = {}, odd[TILES][4] = {};          // two chains of instructions that do not wait for each other
            const float sa = va.scale(), sb = vb.scale();
            const uint32_t la = va.low(), lb = vb.low();
#pragma unroll
            for (int i = i0; i < i0 + GRAIN; ++i) {
              uint32_t a[4], e[4];
              code_pairs<kHalf>(i == 0 ? qa.x : i == 1 ? qa.y : i == 2 ? qa.z : qa.w, a);
              code_pairs<kHalf>(i == 0 ? qb.x : i == 1 ? qb.y : i == 2 ? qb.z : qb.w, e);
              subtract_zero<kHalf>(a, la); subtract_zero<kHalf>(e, lb);
#pragma unroll
              for (int j = 0; j < TILES; ++j) {
                const uint4 x = *reinterpret_cast<const uint4*>(xl[j] + b * kW4Block + 32 * i);
                Codes<kHalf>::mma(acc[j], a[0], e[0], a[1], e[1], x.x, x.y);
                if (GRAIN > 1) Codes<kHalf>::mma(odd[j], a[2], e[2], a[3], e[3], x.z, x.w);
                else Codes<kHalf>::mma(acc[j], a[2], e[2], a[3], e[3], x.z, x.w);
              }
            }
#pragma unroll
            for (int j = 0; j < TILES; ++j) {
              if (GRAIN > 1)
#pragma unroll
                for (int q = 0; q < 4; ++q) acc[j][q] += odd[j][q];
              sum[j][0] += sa * acc[j][0]; sum[j][1] += sa * acc[j][1]; sum[j][2] += sb * acc[j][2]; sum[j][3] += sb * acc[j][3];
            }
          }
        };
        const int b0 = chunk * kStageBlocks + w;
        if (b0 + (kPer - 1) * kWarps < p.blocks) {
          uint4 q[kPer][2];
#pragma unroll
          for (int u = 0; u < kPer; ++u) { q[u][0] = *reinterpret_cast<const uint4*>(from + u * kWarps * 64); q[u][1] = *reinterpret_cast<const uint4*>(from + u * kWarps * 64 + 8 * kColumnPitch); }
#pragma unroll
          for (int u = 0; u < kPer; ++u) block(b0 + u * kWarps, q[u][0], q[u][1]);
        } else {
#pragma unroll 1
          for (int u = 0; b0 + u * kWarps < p.blocks; ++u)
            block(b0 + u * kWarps, *reinterpret_cast<const uint4*>(from + u * kWarps * 64), *reinterpret_cast<const uint4*>(from + u * kWarps * 64 + 8 * kColumnPitch));
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&bars->empty[stage]);
        if (++stage == uint32_t(p.ring)) { stage = 0; phase ^= 1u; }
      }
      if (!ok) break;
      // correction: this warp's share of the rank, straight into its partial sums (the first of the parts of a vector)
      if (p.rank) {
        asm volatile("griddepcontrol.wait;" ::: "memory");         // mid comes from the kernel before this one
        const X* second = static_cast<const X*>(p.second) + tile * kTile + g;
        const bool la = tile * kTile + g < p.n, lb = tile * kTile + g + 8 < p.n;
#pragma unroll 4
        for (int k = w; k < p.rank; k += kWarps) {
          const float va = la ? to_f32(second[k * p.ld2]) : 0.f, vb = lb ? to_f32(second[k * p.ld2 + 8]) : 0.f;
#pragma unroll
          for (int j = 0; j < TILES; ++j)
#pragma unroll
            for (int q = 0; q < 2; ++q) {
              const int col = 8 * j + 2 * c + q, t = kSplit ? col / 3 : col;
              if (t < p.t && (!kSplit || col == 3 * t)) {
                const float m = p.mid[int64_t(t) * p.rank + k];
                sum[j][q] += va * m; sum[j][2 + q] += vb * m;
              }
            }
        }
      }
      // the warps' partial sums meet in shared memory
      if (!(ok = warp_wait(&bars->joint_empty[joint], joint_phase ^ 1u, abort_flag, p.status, 36u))) break;
      float* mine = red + (joint * kWarps + w) * kTile * kRed;
#pragma unroll
      for (int j = 0; j < TILES; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) mine[(g + 8 * (e >> 1)) * kRed + 8 * j + 2 * c + (e & 1)] = sum[j][e];
      __syncwarp();
      if (lane == 0) mbar_arrive(&bars->joint_full[joint]);
      if (++joint == kJoints) { joint = 0; joint_phase ^= 1u; }
    }
  }
}

// mid(k, t) = sum_r first(r, k) x(r, t): one block per k and up to eight vectors, its threads share the rows, eight at a time where
// both operands allow it.  For one vector two warps: the block then fits beside the product's, which starts meanwhile.
template <class X> __global__ void __launch_bounds__(256) mid_kernel(const X* first, int64_t ld1, int rows, int rank, const X* x, int64_t ldx, int t, float* mid, int aligned) {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  __shared__ float red[8][8];
  constexpr int kWide = 16 / sizeof(X);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, k = blockIdx.x, t0 = blockIdx.y * 8;
  float s[8] = {};
  const X* f = first + int64_t(k) * ld1;
  const X* xt = x + int64_t(t0) * ldx;
  const int r0 = aligned ? rows / kWide * kWide : 0;
  auto wide = [&](int count) {
    if (count == 1) {
#pragma unroll 8
      for (int r = threadIdx.x * kWide; r < r0; r += int(blockDim.x) * kWide) {
        const uint4 fw = __ldg(reinterpret_cast<const uint4*>(f + r)), xw = __ldg(reinterpret_cast<const uint4*>(xt + r));
        const X *fv = reinterpret_cast<const X*>(&fw), *xv = reinterpret_cast<const X*>(&xw);
#pragma unroll
        for (int e = 0; e < kWide; ++e) s[0] += to_f32(fv[e]) * to_f32(xv[e]);
      }
      return;
    }
#pragma unroll 2
    for (int r = threadIdx.x * kWide; r < r0; r += int(blockDim.x) * kWide) {
      const uint4 fw = __ldg(reinterpret_cast<const uint4*>(f + r));
      const X* fv = reinterpret_cast<const X*>(&fw);
#pragma unroll
      for (int i = 0; i < 8; ++i) if (i < count) {
        const uint4 xw = __ldg(reinterpret_cast<const uint4*>(xt + i * ldx + r));
        const X* xv = reinterpret_cast<const X*>(&xw);
#pragma unroll
        for (int e = 0; e < kWide; ++e) s[i] += to_f32(fv[e]) * to_f32(xv[e]);
      }
    }
  };
  const int count = min(8, t - t0);
  wide(count);
#pragma unroll 4
  for (int r = r0 + threadIdx.x; r < rows; r += int(blockDim.x)) {
    const float v = to_f32(f[r]);
#pragma unroll
    for (int i = 0; i < 8; ++i) if (i < count) s[i] += v * to_f32(xt[i * ldx + r]);
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    for (int d = 16; d; d >>= 1) s[i] += __shfl_xor_sync(~0u, s[i], d);
    if (lane == 0) red[warp][i] = s[i];
  }
  __syncthreads();
  if (int(threadIdx.x) < count) {
    float v = 0.f;
    for (int w = 0; w < int(blockDim.x) / 32; ++w) v += red[w][threadIdx.x];
    mid[int64_t(t0 + threadIdx.x) * rank + k] = v;
  }
}

template <class X, int TILES, int GRAIN> cudaError_t start(const hyacinHandle_t* handle, const CUtensorMap& map, const StreamParams& p, int smem) {
  auto* kernel = product_stream_kernel<X, TILES, GRAIN>;
  static std::atomic<uint64_t> ready{0};                           // per device: shared memory limit raised
  const uint64_t bit = uint64_t(1) << (handle->DeviceID & 63);
  if (!(ready.load() & bit)) {
    const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmemLimit);
    if (e != cudaSuccess) return e;
    ready.fetch_or(bit);
  }
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(unsigned(std::min((p.n + kTile - 1) / kTile, handle->DeviceSMs))); cfg.blockDim = dim3(kThreads); cfg.dynamicSmemBytes = smem; cfg.stream = handle->cudaStream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization; attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr; cfg.numAttrs = p.rank ? 1 : 0;
  count_launch();
  return cudaLaunchKernelEx(&cfg, kernel, map, p);
}

template <class X, int GRAIN> cudaError_t dispatch(const hyacinHandle_t* handle, const CUtensorMap& map, const StreamParams& p, int smem) {
  return p.tiles == 1 ? start<X, 1, GRAIN>(handle, map, p, smem) : start<X, 2, GRAIN>(handle, map, p, smem);
}

constexpr int kMaxColumns = 16;
int parts(hyacinPrecision_t type) { return type == HYACIN_F32 ? 3 : 1; }

// Shared memory of the form with `tiles` eights of operand columns, 0 when it leaves no ring of four stages.
int layout(StreamParams& p, hyacinPrecision_t type, int tiles) {
  const int per_block = p.seg_sub % 4 == 0 ? 1 : p.seg_sub % 2 == 0 ? 2 : 4, stage_blocks = kWarps * blocks_per_warp(tiles);
  const int64_t pitch = int64_t(p.blocks) * kW4Block + 32;          // 64 bytes over a multiple of 256: lanes g, g + 1 in different halves of the banks
  const int64_t x_bytes = (p.cols * pitch * 2 + 127) / 128 * 128;
  const int64_t red = kJoints * kWarps * kTile * (8 * tiles + 1) * 4, pair_stage = int64_t(kTile) * (per_block * stage_blocks + 1) * (type == HYACIN_F32 ? 8 : 4);
  const int64_t fixed = x_bytes + red + int64_t(sizeof(StreamBars)), stage_codes = kTile * stage_blocks * 64, stage = stage_codes + pair_stage;
  const int64_t ring = std::min<int64_t>(kMaxRing, (kSmemLimit - fixed) / stage);
  if (fixed > kSmemLimit || ring < 4) return 0;
  p.tiles = tiles; p.ring = int(ring); p.pitch = int(pitch); p.ring_at = int(x_bytes);
  p.pairs_at = int(p.ring_at + ring * stage_codes); p.red_at = int(p.pairs_at + ring * pair_stage); p.bars_at = int(p.red_at + red);
  return int(fixed + ring * stage);
}
// Geometry for `vectors` vectors; returns the shared memory, or 0 when they do not fit.  A long x may need the form with smaller stages.
int place(StreamParams& p, hyacinPrecision_t type, const ProductArgs& a, int vectors) {
  p.t = vectors; p.cols = vectors * parts(type); p.rank = a.rank; p.m = a.m; p.n = a.n;
  p.segs = w4_segments(a.m, a.seg); p.seg_sub = a.seg / 32; p.seg_shift = -1;
  for (int s = 0; s < 27; ++s) if (p.seg_sub == 1 << s) p.seg_shift = s;
  p.blocks = (a.m + kW4Block - 1) / kW4Block;
  int bytes = p.cols <= 8 ? layout(p, type, 1) : 0;
  if (!bytes) bytes = layout(p, type, 2);
  return bytes;
}

}  // namespace

int product_stream_vectors(hyacinPrecision_t type, const ProductArgs& a) {
  StreamParams p{};
  int v = std::min(a.t, kMaxColumns / parts(type));
  while (v > 0 && !place(p, type, a, v)) --v;
  return v;
}

int32_t launch_product_stream(const hyacinHandle_t* handle, const char* fn, hyacinPrecision_t type, const ProductArgs& a) {
  cudaStream_t stream = handle->cudaStream;
  float* mid = nullptr;
  int32_t rc = 0;
  const int per = product_stream_vectors(type, a);
  with_w4_type(type, [&](auto tag) {
    using X = decltype(tag);
    if (a.rank) {
      const cudaError_t e = cudaMallocFromPoolAsync(reinterpret_cast<void**>(&mid), size_t(a.rank) * a.t * sizeof(float), handle->mempool, stream);
      if (e != cudaSuccess) { rc = w4_result(e, "cudaMallocFromPoolAsync"); mid = nullptr; return; }
    }
    for (int64_t t0 = 0; t0 < a.t && rc == 0; t0 += per) {
      StreamParams p{};
      const int smem = place(p, type, a, int(std::min<int64_t>(per, a.t - t0)));
      // the codes as eight-byte elements: a box row is a column's share of a stage
      EncodeTiledFn encode = encode_tiled();
      CUtensorMap map{};
      const cuuint64_t dims[2] = {cuuint64_t(p.blocks) * 8, cuuint64_t(a.n)}, strides[1] = {cuuint64_t(a.ldq)};
      const cuuint32_t box[2] = {cuuint32_t(kWarps * blocks_per_warp(p.tiles) * 8), kTile}, elem[2] = {1, 1};
      if (!encode || encode(&map, CU_TENSOR_MAP_DATA_TYPE_UINT64, 2, const_cast<uint8_t*>(a.codes), dims, strides, box, elem, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_NONE,
                            CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) != CUDA_SUCCESS) {
        std::fprintf(stderr, "hyacin-b200: %s: cuTensorMapEncodeTiled failed\n", fn);
        rc = -3; return;
      }
      p.scales = a.scales; p.zeros = a.zeros; p.lds = a.lds;
      p.x = static_cast<const X*>(a.x) + t0 * a.ldx; p.ldx = a.ldx; p.y = static_cast<X*>(a.y) + t0 * a.ldy; p.ldy = a.ldy;
      p.second = a.second; p.ld2 = a.ld2; p.mid = mid ? mid + t0 * a.rank : nullptr;
      p.status = status_word_device(handle->DeviceID);
      const bool wide = reinterpret_cast<uintptr_t>(p.x) % 16 == 0 && (p.ldx * sizeof(X) % 16 == 0 || p.t == 1);
      p.x_aligned = sizeof(X) == 2 && wide;
      if (a.rank) {
        const bool both = wide && reinterpret_cast<uintptr_t>(a.first) % 16 == 0 && a.ld1 * sizeof(X) % 16 == 0;
        if (sizeof(X) == 2 && (p.t > 2 || !both)) {                  // a cluster per 16 x 16 entries
          const cudaError_t e = launch_mid_float(handle, type, a.first, a.ld1, a.m, a.rank, p.x, a.ldx, p.t, mid + t0 * a.rank, both);
          if (e != cudaSuccess) { rc = w4_result(e, fn); return; }
        } else {
          // the product's blocks move in beside this kernel's only if the SM is already split between cache and shared memory their way
          static std::atomic<uint64_t> carved{0};
          const uint64_t mine = uint64_t(1) << (handle->DeviceID & 63);
          if (!(carved.load() & mine)) { HYB_CUDA(cudaFuncSetAttribute(mid_kernel<X>, cudaFuncAttributePreferredSharedMemoryCarveout, cudaSharedmemCarveoutMaxShared)); carved.fetch_or(mine); }
          count_launch();
          const cudaError_t e = w4_start(mid_kernel<X>, dim3(a.rank, (p.t + 7) / 8), p.t == 1 ? 64 : 256, 0, stream, static_cast<const X*>(a.first), a.ld1, a.m, a.rank, static_cast<const X*>(p.x), a.ldx, p.t, mid + t0 * a.rank, int(both));
          if (e != cudaSuccess) { rc = w4_result(e, fn); return; }
        }
      }
      const cudaError_t e = p.seg_sub % 4 == 0 ? dispatch<X, 4>(handle, map, p, smem) : p.seg_sub % 2 == 0 ? dispatch<X, 2>(handle, map, p, smem) : dispatch<X, 1>(handle, map, p, smem);
      rc = w4_result(e, fn);
    }
  });
  if (mid) HYB_CUDA(cudaFreeAsync(mid, stream));
  return rc;
}

}  // namespace hyb
