// Products of a few activation rows with a 4-bit weight (sm_100a):
//   out[m, n] = sum_k x[m, k] * (q[n, k] - z[n, k / group]) * s[n, k / group] (+ bias[n]),   group 32, 64 or 128.
//
// A few rows read the weight once: the call is bound by HBM, N K / 2 bytes, as long as the 4-bit values can be turned into
// operands fast enough - at 6.5 TB/s every SM has to unpack about 50 of them per cycle.  So:
//   * 16 weight rows x 16 k are the A operand of mma.sync (m16n8k16) and 8 activation rows the B operand, with A formed in
//     registers: a 32-bit word holds 8 consecutive k of one row; (w & 0x000f000f) | magic is a pair of 16-bit floats 128 + q
//     (1024 + q in fp16), and one fused multiply-add per pair subtracts 128 + z.  q - z is exact, so the tensor core sees
//     the exact integers, sums of a group are formed in fp32, and the scale multiplies the group's fp32 sum.  tcgen05 would
//     need the unpacked operand in shared memory, four times the bytes that come from HBM.
//   * which k a thread's operand register stands for is free as long as A and B agree: a thread owns 8 consecutive k of each
//     32, the word as it lies in memory, and pairs (k, k + 4) of x by byte permutes.
//   * the weight streams through a ring of shared-memory stages, 512 k of the CTA's rows each, by TMA; x comes with it, and one
//     warp per 8 activation rows (16 of 32) makes the permutes once for all others.  Scales and zero points go from global memory to
//     the registers of the warp that has their rows, up to 1024 k ahead, and from there to its shared memory as fp32 scale
//     and 16-bit offset.
//   * a CTA has R rows (a multiple of 16) and a slice of K: R and the cluster size are chosen so that the CTAs fill the SMs
//     once with the least per CTA (w4_plan).  Inside the CTA the warps split R and, where that leaves warps over, the k of
//     a stage, evenly over the SM's schedulers; the CTAs of a cluster add their sums through distributed shared memory.  All
//     sums in a fixed order.
// Measured: 10.3 us for 1 x 14336 x 4096 (2.9 TB/s), 31 us for 8 x 28672 x 8192 with groups of 64 (4.1 TB/s).  The copies alone
// take 7 and 19.6 us; what bounds it is unpacking, 8 LOP3, 8 HFMA2 and 2 to 6 shifts per 512 weights and warp, in chains that
// three or four warps per scheduler do not hide (the multiplication alone of resident data took 9 us, and 28 of 32 before
// four warps shared the rows left over).
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "common.cuh"
#include "ptx.cuh"

namespace bfp8 {

bool weights_at_rest();

namespace {

constexpr long long kDefaultWaitLimit = 2000000000LL;      // about a second
constexpr int kStageK = 512;                               // k per stage: twice 128 bytes of a code row
constexpr int kMaxStages = 16;
constexpr int kSmemBytes = 225 * 1024;
constexpr int kSmemLimit = 227 * 1024;                     // what one SM has for a CTA
constexpr int kMaxCluster = 8;

struct W4Params {
  const uint16_t* scales;      // [n, groups]
  const uint8_t* zeros;        // [n, groups] or NULL: 8
  const float* bias;           // [n] or NULL
  void* out;
  int64_t ldo;
  int m, n, k, groups;
  int rows;                    // R
  uint32_t row_share;          // 2^32 / R, rounded up: i / R = __umulhi(i, row_share) for the few thousand sums of a CTA
  int stages;                  // ring depth
  int cluster;
  int out_f32;
  int scale_vec;               // the scales and zero points of a step can be loaded together
  int w_early;
  long long wait_limit;
  uint32_t* status;
};

struct W4Tail {
  uint64_t full[kMaxStages], ready[kMaxStages], empty[kMaxStages];
  uint32_t abort_flag;
};

template <bool kBf16>
struct Half16;
template <>
struct Half16<true> {
  static constexpr uint32_t kMagic = 0x43004300u, kOne = 0x3f803f80u, kSixteenth = 0u, kStep = 0u, kMinus = 0xc300c300u;
  static __device__ __forceinline__ uint32_t fma(uint32_t a, uint32_t b, uint32_t c) {
    uint32_t r;
    asm("fma.rn.bf16x2 %0, %1, %2, %3;" : "=r"(r) : "r"(a), "r"(b), "r"(c));
    return r;
  }
  static __device__ __forceinline__ float value(uint32_t bits) { return __uint_as_float(bits << 16); }
  static __device__ __forceinline__ uint16_t round(float v) { return static_cast<uint16_t>(float_to_bf16_bits(v)); }
  static __device__ __forceinline__ void mma(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  }
  // the same from zero
  static __device__ __forceinline__ void mma0(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
                 : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.0f));
  }
};
template <>
struct Half16<false> {
  static constexpr uint32_t kMagic = 0x64006400u, kOne = 0x3c003c00u, kSixteenth = 0x2c002c00u, kMinus = 0xe400e400u;
  static constexpr uint32_t kStep = 0x63806380u;           // 960 = 1024 - 64
  static __device__ __forceinline__ uint32_t fma(uint32_t a, uint32_t b, uint32_t c) {
    uint32_t r;
    asm("fma.rn.f16x2 %0, %1, %2, %3;" : "=r"(r) : "r"(a), "r"(b), "r"(c));
    return r;
  }
  static __device__ __forceinline__ float value(uint32_t bits) {
    return __half2float(__ushort_as_half(static_cast<unsigned short>(bits)));
  }
  static __device__ __forceinline__ uint16_t round(float v) { return __half_as_ushort(__float2half_rn(v)); }
  static __device__ __forceinline__ void mma(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  }
  static __device__ __forceinline__ void mma0(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
                 : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.0f));
  }
};

// (w & mask) | magic in one instruction
__device__ __forceinline__ uint32_t pick(uint32_t w, uint32_t mask, uint32_t magic) {
  uint32_t r;
  asm("lop3.b32 %0, %1, %2, %3, 0xea;" : "=r"(r) : "r"(w), "r"(mask), "r"(magic));
  return r;
}
__device__ __forceinline__ void named_sync(int id, int threads) {
  asm volatile("bar.sync %0, %1;" ::"r"(id), "r"(threads) : "memory");
}
__device__ __forceinline__ float ld_cluster_f32(uint32_t addr) {
  float v;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(addr) : "memory");
  return v;
}

// An SM's warps run on four schedulers, warp w on number w % 4, and the one with most work sets the pace.  A CTA's groups of 16
// rows (units) go to whole warps, each a stage's four pieces of 128 k, or two where a pair of warps shares a unit.  Without a
// rest that is all; with one, only as many units as divide evenly over the schedulers go to whole warps, and of each unit left
// over four more warps take a piece each (8 x 28672 x 8192, 13 units: 32.4 us without, 31.1 with; 8 x 35520 x 8192, 15 units:
// 50 us in two waves without, 36 with; 16 x 65536 x 1024: 21.1 and 18.6).  The rest's code costs 0.5 us where nothing is left.
// (Quarters of a stage for all warps alike, which needs every unit's scales in reach of four warps: 36 us for 28672 x 8192.)
// Beside them a warp per 8 rows of x and the producer; of 32 rows a warp has 16, which leaves 13 multiplying warps instead of
// 11 and 28672 x 8192 in one wave: 58.7 us, not 83.
__host__ __device__ constexpr int x_warps(int nt) { return nt < 4 ? nt : 2; }
__host__ __device__ constexpr int whole_warps(int nt, bool rest) { return rest ? 12 : 15 - x_warps(nt); }
__host__ __device__ constexpr int consumers(int nt, bool rest) { return whole_warps(nt, rest) + (rest ? 4 : 0); }
__host__ __device__ constexpr int threads_of(int nt, bool rest) { return 32 * (consumers(nt, rest) + x_warps(nt) + 1); }
__host__ __device__ constexpr int whole_units(int units, int slices, bool rest) {
  return !rest ? units : slices == 2 ? units & ~1 : min(units & ~3, whole_warps(1, true));
}
// Scales are fetched for up to 1024 k at once: from the [n, groups] layout 256 k of a row are 4 to 16 bytes of a 128-byte line,
// and a warp-wide load costs a cycle per line
__host__ __device__ constexpr int super_steps(int shift) { return shift == 0 ? 1 : 2; }
__host__ __device__ constexpr int step_groups(int shift) { return kStageK >> (5 + shift); }
__host__ __device__ constexpr int warp_area(int shift) { return 16 * super_steps(shift) * step_groups(shift) * 8; }
__host__ __device__ constexpr int rest_area(int shift) { return 3 * 16 * (step_groups(shift) / 4) * 8; }
__host__ __device__ constexpr int scale_bytes(int nt, int shift, bool rest) {
  return whole_warps(nt, rest) * warp_area(shift) + (rest ? 4 * rest_area(shift) : 0);
}
__host__ __device__ constexpr int ring_bytes(int nt, int shift, bool rest) { return (kSmemBytes - scale_bytes(nt, shift, rest)) & ~1023; }
constexpr int64_t kMaxM = 65535 * 16;                      // activation rows: chunks of 16 or more on the grid's y axis
constexpr int kMaxRows = 16 * (whole_warps(1, true) + 3);                // weight rows per CTA, within a TMA box
__host__ __device__ constexpr int stage_size(int rows, int mp) { return rows * (kStageK / 2) + mp * kStageK * 2; }

// Scales and zero points of kGroups neighbouring groups of one row as they lie in memory, loaded well before they are used
template <int kGroups>
struct RawScales {
  uint32_t s[(kGroups + 1) / 2];
  uint32_t z[(kGroups + 3) / 4];
  __device__ __forceinline__ void load(const W4Params& p, int row, int g0) {
#pragma unroll
    for (int i = 0; i < (kGroups + 1) / 2; ++i) s[i] = 0u;
#pragma unroll
    for (int i = 0; i < (kGroups + 3) / 4; ++i) z[i] = 0x08080808u;
    if (row >= p.n || g0 >= p.groups) return;
    const int64_t at = static_cast<int64_t>(row) * p.groups + g0;
    if (p.scale_vec) {                                             // groups % kGroups == 0: they exist together
      if constexpr (kGroups == 1) {
        s[0] = __ldg(p.scales + at);
        if (p.zeros != nullptr) z[0] = __ldg(p.zeros + at);
      } else if constexpr (kGroups == 2) {
        s[0] = __ldg(reinterpret_cast<const uint32_t*>(p.scales + at));
        if (p.zeros != nullptr) z[0] = __ldg(reinterpret_cast<const uint16_t*>(p.zeros + at));
      } else if constexpr (kGroups == 4) {
        const uint2 v = __ldg(reinterpret_cast<const uint2*>(p.scales + at));
        s[0] = v.x; s[1] = v.y;
        if (p.zeros != nullptr) z[0] = __ldg(reinterpret_cast<const uint32_t*>(p.zeros + at));
      } else {
        const uint4 v = __ldg(reinterpret_cast<const uint4*>(p.scales + at));
        s[0] = v.x; s[1] = v.y; s[2] = v.z; s[3] = v.w;
        if (p.zeros != nullptr) {
          const uint2 u = __ldg(reinterpret_cast<const uint2*>(p.zeros + at));
          z[0] = u.x; z[1] = u.y;
        }
      }
    } else {
#pragma unroll
      for (int j = 0; j < kGroups; ++j)
        if (g0 + j < p.groups) {
          s[j >> 1] |= static_cast<uint32_t>(__ldg(p.scales + at + j)) << (16 * (j & 1));
          if (p.zeros != nullptr)
            z[j >> 2] = (z[j >> 2] & ~(0xffu << (8 * (j & 3)))) | static_cast<uint32_t>(__ldg(p.zeros + at + j)) << (8 * (j & 3));
        }
    }
  }
  // group j as the kernel uses it: fp32 scale, and -(128 + z) or -(1024 + z) twice
  template <typename H>
  __device__ __forceinline__ uint2 ready(int j) const {
    const uint32_t sc = (s[j >> 1] >> (16 * (j & 1))) & 0xffffu, zp = (z[j >> 2] >> (8 * (j & 3))) & 0xffu;
    return make_uint2(__float_as_uint(H::value(sc)), H::kMinus + zp * 0x10001u);
  }
};

// kNT: activation rows / 8, 1, 2 or 4; kShift: group = 32 << kShift; kSlices: warps that share 16 rows, 2 take a half of each stage's k
// each; kRest: four more warps for the units left over.
template <bool kBf16, int kNT, int kShift, int kSlices, bool kRest>
__global__ void __launch_bounds__(threads_of(kNT, kRest), 1)
w4_kernel(const __grid_constant__ CUtensorMap tmap_w, const __grid_constant__ CUtensorMap tmap_x, const W4Params p) {
  using H = Half16<kBf16>;
  constexpr int kWhole = whole_warps(kNT, kRest), kConsumers = consumers(kNT, kRest), kProducer = kConsumers + x_warps(kNT);
  constexpr int kWarpRows = 16, kThreads = threads_of(kNT, kRest), kRing = ring_bytes(kNT, kShift, kRest);
  constexpr int kMp = kNT * 8;
  constexpr int kXBytes = kMp * kStageK * 2;
  constexpr int kStepGroups = step_groups(kShift), kSuper = super_steps(kShift);
  constexpr int kLaneGroups = kSuper * kStepGroups / 2;            // 4 or 8: two lanes per row
  constexpr int kPieceGroups = kStepGroups / 4;                    // 4, 2 or 1
  constexpr int kRestUnits = kSlices == 2 ? 1 : 3;                 // groups of rows left over, at most
  extern __shared__ uint8_t smem_raw[];
  const uint32_t smem_base = (ptx::smem_u32(smem_raw) + 1023u) & ~1023u;
  uint8_t* smem = smem_raw + (smem_base - ptx::smem_u32(smem_raw));
  W4Tail* tail = reinterpret_cast<W4Tail*>(smem + kRing + scale_bytes(kNT, kShift, kRest));
  volatile uint32_t* abort_flag = &tail->abort_flag;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int units = p.rows / kWarpRows;
  constexpr int slices = kSlices;
  const int whole = whole_units(units, slices, kRest), rest = units - whole;
  const uint32_t stage_bytes = static_cast<uint32_t>(stage_size(p.rows, kMp));
  const int rank = p.cluster > 1 ? static_cast<int>(blockIdx.x) % p.cluster : 0;
  const int n0 = static_cast<int>(blockIdx.x) / p.cluster * p.rows;
  const int m0 = blockIdx.y * kMp;
  const int all_steps = (p.k + kStageK - 1) / kStageK;
  const int step0 = static_cast<int>(static_cast<long long>(all_steps) * rank / p.cluster);
  const int step1 = static_cast<int>(static_cast<long long>(all_steps) * (rank + 1) / p.cluster);

  if (threadIdx.x == 0) {
    for (int s = 0; s < p.stages; ++s) {
      ptx::mbar_init(ptx::smem_u32(&tail->full[s]), 1);
      ptx::mbar_init(ptx::smem_u32(&tail->ready[s]), x_warps(kNT));
      ptx::mbar_init(ptx::smem_u32(&tail->empty[s]), static_cast<uint32_t>(whole * slices + (rest > 0 ? 4 : 0)));
    }
    tail->abort_flag = 0;
    ptx::fence_mbar_init();
  }
  __syncthreads();
  ptx::griddep_launch_dependents();

  const int g = lane >> 2, t = lane & 3;
  // activation row of column g of the B operand: neighbouring columns lie in different halves of the swizzled 128 bytes
  const int xrow = (g >> 1) + 4 * (g & 1);
  uint32_t stage = 0, parity = 0;
  auto advance = [&] {
    if (++stage == static_cast<uint32_t>(p.stages)) { stage = 0; parity ^= 1u; }
  };

  if (warp == kProducer) {
    // ------------------------------------------------------------------ TMA producer
    if (lane == 0) {
      ptx::prefetch_tensormap(&tmap_w);
      ptx::prefetch_tensormap(&tmap_x);
      const uint64_t once = ptx::l2_policy_evict_first();
      int early = 0;
      if (p.w_early)                                               // codes at rest: asked for before the previous kernel has ended
        for (; early < p.stages && step0 + early < step1; ++early) {
          const uint32_t full = ptx::smem_u32(&tail->full[early]);
          ptx::mbar_arrive_expect_tx(full, stage_bytes);
          for (int h = 0; h < 2; ++h)
            ptx::tma_load_2d_hint(smem_base + early * stage_bytes + h * p.rows * 128, &tmap_w, full, (step0 + early) * 256 + h * 128, n0, once);
        }
      ptx::griddep_wait();
      for (int s = step0; s < step1; ++s) {
        const uint32_t full = ptx::smem_u32(&tail->full[stage]), dst = smem_base + stage * stage_bytes;
        if (early > 0) {
          --early;
        } else {
          if (!ptx::mbar_wait(ptx::smem_u32(&tail->empty[stage]), parity ^ 1u, abort_flag, p.wait_limit)) break;
          ptx::mbar_arrive_expect_tx(full, stage_bytes);
          for (int h = 0; h < 2; ++h) ptx::tma_load_2d_hint(dst + h * p.rows * 128, &tmap_w, full, s * 256 + h * 128, n0, once);
        }
#pragma unroll
        for (int b = 0; b < kStageK / 64; ++b)
          ptx::tma_load_2d(dst + p.rows * 256 + b * kMp * 128, &tmap_x, full, s * kStageK + b * 64, m0);
        advance();
      }
    }
  } else if (warp >= kConsumers) {
    // ------------------------------------------------------------------ x of 8 rows: pairs (k, k + 4) side by side, once for all consumers
    constexpr int kEach = kNT / x_warps(kNT);
    const uint32_t first = p.rows * 256 + ((warp - kConsumers) * kEach * 8 + xrow) * 128 + ((t ^ xrow) << 4);
    ptx::griddep_wait();                                           // x comes only then: the previous kernel's time is not this wait's
    for (int s = step0; s < step1; ++s) {
      if (!__all_sync(0xffffffffu, ptx::mbar_wait(ptx::smem_u32(&tail->full[stage]), parity, abort_flag, p.wait_limit))) break;
      uint8_t* at = smem + stage * stage_bytes;
#pragma unroll
      for (int h = 0; h < kEach * (kStageK / 256); ++h) {
        uint8_t* half = at + (h / kEach) * 4 * (kMp * 128) + (h % kEach) * 1024;
        uint4 v[8];
#pragma unroll
        for (int q = 0; q < 8; ++q) v[q] = *reinterpret_cast<const uint4*>(half + (first ^ ((q & 1) << 6)) + (q >> 1) * (kMp * 128));
#pragma unroll
        for (int q = 0; q < 8; ++q)
          *reinterpret_cast<uint4*>(half + (first ^ ((q & 1) << 6)) + (q >> 1) * (kMp * 128)) =
              make_uint4(__byte_perm(v[q].x, v[q].z, 0x5410), __byte_perm(v[q].x, v[q].z, 0x7632),
                         __byte_perm(v[q].y, v[q].w, 0x5410), __byte_perm(v[q].y, v[q].w, 0x7632));
      }
      ptx::fence_proxy_async_smem();                               // the stage's next copy may not pass these stores
      __syncwarp();
      ptx::mbar_arrive_lane0(ptx::smem_u32(&tail->ready[stage]), lane);
      advance();
    }
  } else {
    // ------------------------------------------------------------------ multiplying warps
    const uint32_t w_lane = g * 128 + (g << 4) + t * 4;                    // chunk c of 16 bytes of row r lies at c ^ (r & 7)
    const uint32_t x_first = p.rows * 256 + xrow * 128 + ((t ^ xrow) << 4);
    // 16 rows x 128 k: `at` the stage, codes those of the rows' 256 k that hold the piece, scales its first group
    auto multiply = [&](const uint8_t* at, const uint8_t* codes, const uint8_t* scales, int quarter, float (&acc)[kNT][4]) {
      float part[kNT][4], scale[2];
      uint32_t sub0[2], sub1[2];
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        constexpr int kMask = (1 << kShift) - 1;
        if ((q & kMask) == 0) {                                            // a new group
#pragma unroll
          for (int r = 0; r < 2; ++r) {
            const uint2 v = *reinterpret_cast<const uint2*>(scales + ((q >> kShift) * kWarpRows + r * 8) * 8);
            scale[r] = __uint_as_float(v.x);
            sub0[r] = v.y;
            if (!kBf16) sub1[r] = H::fma(sub0[r], H::kOne, H::kStep);      // -(64 + z)
          }
        }
        uint4 x[kNT];
#pragma unroll
        for (int b = 0; b < kNT; ++b)
          x[b] = *reinterpret_cast<const uint4*>(at + (x_first ^ ((q & 1) << 6)) + (quarter * 2 + (q >> 1)) * (kMp * 128) + b * 1024);
        uint32_t w[2][4];
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          const uint32_t lo = *reinterpret_cast<const uint32_t*>(codes + (w_lane ^ (q << 4) ^ ((quarter & 1) << 6)) + r * 1024);
          const uint32_t hi = lo >> 8;
          w[r][0] = H::fma(pick(lo, 0x000f000fu, H::kMagic), H::kOne, sub0[r]);
          w[r][2] = H::fma(pick(hi, 0x000f000fu, H::kMagic), H::kOne, sub0[r]);
          if (kBf16) {                                                     // seven bits of fraction: no room for a value shifted by four
            w[r][1] = H::fma(pick(lo >> 4, 0x000f000fu, H::kMagic), H::kOne, sub0[r]);
            w[r][3] = H::fma(pick(lo >> 12, 0x000f000fu, H::kMagic), H::kOne, sub0[r]);
          } else {                                                         // 1024 + 16 q, times 1/16
            w[r][1] = H::fma(pick(lo, 0x00f000f0u, H::kMagic), H::kSixteenth, sub1[r]);
            w[r][3] = H::fma(pick(hi, 0x00f000f0u, H::kMagic), H::kSixteenth, sub1[r]);
          }
        }
#pragma unroll
        for (int b = 0; b < kNT; ++b) {
          if ((q & kMask) == 0) H::mma0(part[b], w[0][0], w[1][0], w[0][1], w[1][1], x[b].x, x[b].y);
          else H::mma(part[b], w[0][0], w[1][0], w[0][1], w[1][1], x[b].x, x[b].y);
          H::mma(part[b], w[0][2], w[1][2], w[0][3], w[1][3], x[b].z, x[b].w);
        }
        if ((q & kMask) == kMask)
#pragma unroll
          for (int b = 0; b < kNT; ++b)
#pragma unroll
            for (int c = 0; c < 4; ++c) acc[b][c] = fmaf(part[b][c], scale[c >> 1], acc[b][c]);
      }
    };
    // sums of 16 rows as [part][activation row][weight row], once every stage has been read and the ring is free
    auto keep = [&](const float (&acc)[kNT][4], int part, int unit) {
      float* red = reinterpret_cast<float*>(smem);
#pragma unroll
      for (int b = 0; b < kNT; ++b)
#pragma unroll
        for (int c = 0; c < 4; ++c)
          red[(part * kMp + b * 8 + t + 4 * (c & 1)) * p.rows + unit * 16 + g + 8 * (c >> 1)] = acc[b][c];
    };
    // x is ready: so are the codes, whose copies the x warps waited for
    auto wait_stage = [&] {
      return __all_sync(0xffffffffu, ptx::mbar_wait(ptx::smem_u32(&tail->ready[stage]), parity, abort_flag, p.wait_limit));
    };
    auto leave_stage = [&] {
      __syncwarp();
      ptx::mbar_arrive_lane0(ptx::smem_u32(&tail->empty[stage]), lane);
      advance();
    };
    const int row = lane & 15;
    if (warp < kWhole) {
      const int unit = slices == 2 ? warp >> 1 : warp, slice = slices == 2 ? warp & 1 : 0;
      float acc[kNT][4] = {};
      if (unit < whole) {
        const uint32_t area = kRing + warp * warp_area(kShift);
        const int share = (lane >> 4) * kLaneGroups;                       // this lane's part of the scales: one half of a row's groups
        ptx::griddep_wait();
        RawScales<kLaneGroups> raw;
        raw.load(p, n0 + unit * kWarpRows + row, step0 * kStepGroups + share);
        bool ok = true;
        for (int s0 = step0; s0 < step1 && ok; s0 += kSuper) {
          __syncwarp();                                                    // the last scales have been read
#pragma unroll
          for (int j = 0; j < kLaneGroups; ++j)
            *reinterpret_cast<uint2*>(smem + area + ((share + j) * kWarpRows + row) * 8) = raw.template ready<H>(j);
          __syncwarp();
          if (s0 + kSuper < step1) raw.load(p, n0 + unit * kWarpRows + row, (s0 + kSuper) * kStepGroups + share);
          const int s1 = min(s0 + kSuper, step1);
          for (int s = s0; s < s1; ++s) {
            ok = wait_stage();
            if (!ok) break;
            const uint8_t* at = smem + stage * stage_bytes;
            const uint8_t* scales = smem + area + ((s - s0) * kStepGroups * kWarpRows + g) * 8;
            const uint8_t* codes = at + unit * 2048 + (slices == 2 ? slice * p.rows * 128 : 0);
#pragma unroll(kNT == 4 ? 1 : 4)                           // with 32 rows the registers do not hold what four overlapping pieces need
            for (int piece = 0; piece < 4 / slices; ++piece) {
              const int quarter = slices == 2 ? slice * 2 + piece : piece;
              multiply(at, codes + (slices == 1 ? (piece >> 1) * p.rows * 128 : 0), scales + quarter * kPieceGroups * kWarpRows * 8, quarter, acc);
            }
            leave_stage();
          }
        }
      }
      named_sync(1, kThreads);
      if (unit < whole) keep(acc, slice, unit);
    } else if constexpr (kRest) {
      const int quarter = warp - kWhole;
      float acc[kRestUnits][kNT][4] = {};
      if (rest > 0) {
        const uint32_t area = kRing + kWhole * warp_area(kShift) + quarter * rest_area(kShift);
        const int first = whole + (lane >> 4);                             // a lane's scales: its row of every other unit
        RawScales<kPieceGroups> raw[(kRestUnits + 1) / 2];
        auto load = [&](int s) {
#pragma unroll
          for (int i = 0; i < (kRestUnits + 1) / 2; ++i)
            if (first + 2 * i < units) raw[i].load(p, n0 + (first + 2 * i) * kWarpRows + row, s * kStepGroups + quarter * kPieceGroups);
        };
        ptx::griddep_wait();
        load(step0);
        for (int s = step0; s < step1; ++s) {
          __syncwarp();
#pragma unroll
          for (int i = 0; i < (kRestUnits + 1) / 2; ++i)
            if (first + 2 * i < units)
#pragma unroll
              for (int j = 0; j < kPieceGroups; ++j)
                *reinterpret_cast<uint2*>(smem + area + (((first - whole + 2 * i) * kPieceGroups + j) * kWarpRows + row) * 8) =
                    raw[i].template ready<H>(j);
          __syncwarp();
          if (s + 1 < step1) load(s + 1);
          if (!wait_stage()) break;
          const uint8_t* at = smem + stage * stage_bytes;
          const uint8_t* codes = at + (quarter >> 1) * p.rows * 128 + whole * 2048;
#pragma unroll
          for (int i = 0; i < kRestUnits; ++i)
            if (i < rest) multiply(at, codes + i * 2048, smem + area + (i * kPieceGroups * kWarpRows + g) * 8, quarter, acc[i]);
          leave_stage();
        }
      }
      named_sync(1, kThreads);
#pragma unroll
      for (int i = 0; i < kRestUnits; ++i)
        if (i < rest) keep(acc[i], quarter, whole + i);
    }
  }

  // ------------------------------------------------------------------ sums of the warps, then of the cluster's CTAs
  if (warp >= kConsumers) named_sync(1, kThreads);                 // every stage has been read
  __syncthreads();
  float* red = reinterpret_cast<float*>(smem);
  const int width = p.rows;
  const bool done = *abort_flag == 0;
  const int count = min(kMp, p.m - m0) * width;
  auto sum_of = [&](int i, int n) {
    const int q = kMp * width;
    float v = red[i];
    if (kRest && n >= whole * kWarpRows) v += (red[q + i] + red[2 * q + i]) + red[3 * q + i];
    else if (slices == 2) v += red[q + i];
    return v;
  };
  auto split = [&](int i, int& m, int& n) {
    m = static_cast<int>(__umulhi(static_cast<uint32_t>(i), p.row_share));
    n = i - m * width;
  };
  if (p.cluster > 1) {
    for (int i = threadIdx.x; i < count; i += kThreads) {
      int m, n;
      split(i, m, n);
      red[i] = sum_of(i, n);
    }
    ptx::cluster_sync_all();
  }
  auto store = [&](int m, int n, float v) {
    n += n0;
    if (n >= p.n) return;
    if (p.bias != nullptr) v += __ldg(p.bias + n);
    const int64_t at = static_cast<int64_t>(m0 + m) * p.ldo + n;
    if (p.out_f32) static_cast<float*>(p.out)[at] = v;
    else static_cast<uint16_t*>(p.out)[at] = H::round(v);
  };
  if (p.cluster > 1) {
    // CTA `rank` finishes its share of the outputs, adding the CTAs' sums in rank order, which is K order
    const int i1 = static_cast<int>(static_cast<long long>(count) * (rank + 1) / p.cluster);
    for (int i = static_cast<int>(static_cast<long long>(count) * rank / p.cluster) + threadIdx.x; i < i1 && done; i += kThreads) {
      float part[kMaxCluster], v = 0.0f;                           // on their way together
#pragma unroll
      for (int c = 0; c < kMaxCluster; ++c) part[c] = c < p.cluster ? ld_cluster_f32(ptx::cluster_map(smem_base + i * 4, c)) : 0.0f;
#pragma unroll
      for (int c = 0; c < kMaxCluster; ++c) v += part[c];
      int m, n;
      split(i, m, n);
      store(m, n, v);
    }
    ptx::cluster_sync_all();                                       // nobody leaves while its sums are being read
  } else if (done) {
    for (int i = threadIdx.x; i < count; i += kThreads) {
      int m, n;
      split(i, m, n);
      store(m, n, sum_of(i, n));
    }
  }
  ptx::idle_after_abort(abort_flag);
  if (threadIdx.x == 0 && tail->abort_flag != 0) atomicOr(p.status, BFP8_STATUS_WAIT_TIMEOUT);
}

// Rows per CTA and CTAs per cluster: the least time for the CTA that has most to do, priced with what B200 measured, in 0.01 us.
// The SM's four schedulers have a quarter of the warps each, and the one with most of them sets the pace: one warp unpacks
// 3.5 KB of codes per us, two 6.6, three 8.5 and four 10 (with 16 activation rows 3, 5.3, 6.5 and 7.5, with 32 rows 2.2, 4, 5 and 5.6).
// A stage costs 0.15 us beside that, a wave of CTAs 1.5 us to start (with 32 rows 3.5 us after the first) and a cluster
// 1.2 us to form and exchange its sums (3 rows x 1003 x 4000: 5.0 us with clusters of four, 7.2 us without; 1 row x 1024 x
// 1024: 2.8 us without, 4.4 us with pairs).  resident(c): clusters of c CTAs that the device holds at once - 74 of two, but
// 33 of four and 15 of eight on 148 SMs.
// A rest's warps count for the share of a whole warp's work that they have, and cost 0.3 us.
struct Plan {
  int rows, cluster, slices;
  bool rest;
  int64_t cost;
};
template <typename Resident>
Plan w4_plan(int64_t n, int64_t k, int64_t chunks, int nt, Resident resident) {
  const int64_t steps = (k + kStageK - 1) / kStageK;
  Plan best = {16, 1, 1, false, INT64_MAX};
  constexpr int64_t kRate[3][5] = {{0, 35, 66, 85, 100}, {0, 30, 53, 65, 75}, {0, 22, 40, 50, 56}};   // bytes per 0.01 us
  const int64_t* rates = kRate[nt / 2];
  for (int cluster = 1; cluster <= kMaxCluster; cluster *= 2) {
    if (cluster > steps) break;
    const int64_t together = resident(cluster);
    if (together <= 0) continue;
    const int64_t each = (steps + cluster - 1) / cluster;
    for (int units = 1; units <= kMaxRows / 16; ++units) {
      const int64_t waves = ((n + units * 16 - 1) / (units * 16) * chunks + together - 1) / together;
      for (int form = 0; form < (nt == 4 ? 1 : 2); ++form) {
        const bool rest = form != 0;
        const int slices = 2 * whole_units(units, 2, rest) <= whole_warps(nt, rest) ? 2 : 1;
        const int whole = whole_units(units, slices, rest), warps = (whole * slices + 3) / 4, more = (units - whole) * slices;
        if (whole * slices > whole_warps(nt, rest) || rest != (more > 0)) continue;
        // of the scheduler that has most: bytes of codes, and how fast its warps take them
        const int64_t codes = each * 1024 * (rest ? units : 4 / slices * warps);
        const int64_t rate = rates[warps] + (more > 0 ? (rates[warps + 1] - rates[warps]) * more / 4 : 0);
        const int64_t cost = waves * (codes / rate + each * 15 + 150 + (cluster > 1 ? 120 : 0) + (rest ? 30 : 0)) +
                             (nt == 4 ? (waves - 1) * 200 : 0);
        if (cost < best.cost || (cost == best.cost && cluster > best.cluster)) best = {units * 16, cluster, slices, rest, cost};
      }
      if (waves == 1) break;                                       // more rows per CTA only take longer
    }
  }
  return best;
}

template <bool kBf16, int kNT, int kShift, int kSlices, bool kRest>
int launch_form(cudaLaunchConfig_t& cfg, const CUtensorMap& tmap_w, const CUtensorMap& tmap_x, W4Params& p) {
  constexpr int kRing = ring_bytes(kNT, kShift, kRest);
  constexpr int smem = 1024 + kRing + scale_bytes(kNT, kShift, kRest) + static_cast<int>(sizeof(W4Tail));
  static_assert(smem <= kSmemLimit, "shared memory of one SM");
  static_assert(kRing / stage_size(kRest ? kMaxRows : 16 * whole_warps(kNT, false), kNT * 8) >= 2, "two stages at least");
  static_assert(4 * kNT * 8 * kMaxRows * 4 <= kRing, "the warps' sums");
  auto kernel = w4_kernel<kBf16, kNT, kShift, kSlices, kRest>;
  static DeviceFlags done;
  const int rc = ensure_smem_limit(kernel, kSmemLimit, done);
  if (rc != BFP8_OK) return rc;
  const int most = kRing / stage_size(p.rows, kNT * 8);
  p.stages = most < kMaxStages ? most : kMaxStages;
  cfg.blockDim = dim3(threads_of(kNT, kRest), 1, 1);
  cfg.dynamicSmemBytes = smem;
  BFP8_CUDA_TRY(cudaLaunchKernelEx(&cfg, kernel, tmap_w, tmap_x, p));
  return BFP8_OK;
}

cudaLaunchConfig_t overlapped(cudaLaunchAttribute (&attr)[2], cudaStream_t st) {
  cudaLaunchConfig_t cfg = {};
  cfg.stream = st;
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim = {1, 1, 1};
  cfg.attrs = attr;
  return cfg;
}

template <bool kBf16, int kNT, int kShift>
Plan plan_for(const W4Params& p) {
  return w4_plan(p.n, p.k, (p.m + kNT * 8 - 1) / (kNT * 8), kNT, [&](int cluster) -> int {
    if (cluster == 1) return sm_count();
    // one CTA per SM in every form; asked for with the plain one
    auto kernel = w4_kernel<kBf16, kNT, kShift, 1, false>;
    static DeviceFlags done;
    static ClusterCaps caps;
    if (ensure_smem_limit(kernel, kSmemLimit, done) != BFP8_OK) return 0;
    cudaLaunchAttribute attr[2];
    cudaLaunchConfig_t ask = overlapped(attr, nullptr);
    attr[1].val.clusterDim.x = static_cast<unsigned>(cluster);
    ask.blockDim = dim3(threads_of(kNT, false), 1, 1);
    ask.dynamicSmemBytes = 1024 + kSmemBytes;
    ask.gridDim = dim3(static_cast<unsigned>(cluster), 1, 1);
    ask.attrs = attr + 1;
    ask.numAttrs = 1;
    return max_active_clusters(kernel, ask, cluster, caps);
  });
}

template <bool kBf16, int kNT, int kShift>
int launch_w4(const Plan& plan, const uint8_t* codes, const void* x, int64_t ldx, W4Params& p, cudaStream_t st) {
  constexpr int kLaneGroups = super_steps(kShift) * step_groups(kShift) / 2;
  static_assert(kLaneGroups == 4 || kLaneGroups == 8, "what RawScales loads at once");
  cudaLaunchAttribute attr[2];
  cudaLaunchConfig_t cfg = overlapped(attr, st);
  p.rows = plan.rows;
  p.cluster = plan.cluster;
  p.row_share = 0xffffffffu / static_cast<uint32_t>(plan.rows) + 1u;
  p.scale_vec = p.groups % kLaneGroups == 0 && aligned(p.scales, 2 * kLaneGroups) && (p.zeros == nullptr || aligned(p.zeros, kLaneGroups));
  alignas(64) CUtensorMap tmap_w, tmap_x;
  int rc = make_tensor_map_2d(&tmap_w, CU_TENSOR_MAP_DATA_TYPE_UINT8, codes, p.k / 2, p.n, p.k / 2, 128, p.rows);
  if (rc != BFP8_OK) return rc;
  rc = make_tensor_map_2d(&tmap_x, kBf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, x, p.k, p.m,
                          ldx * 2, 64, kNT * 8);
  if (rc != BFP8_OK) return rc;
  cfg.gridDim = dim3(static_cast<unsigned>((p.n + p.rows - 1) / p.rows * p.cluster), static_cast<unsigned>((p.m + kNT * 8 - 1) / (kNT * 8)), 1);
  attr[1].val.clusterDim.x = static_cast<unsigned>(p.cluster);
  cfg.numAttrs = p.cluster > 1 ? 2 : 1;
  if constexpr (kNT < 4)                                           // w4_plan knows no rest with 32 rows
    if (plan.rest)
      return plan.slices == 2 ? launch_form<kBf16, kNT, kShift, 2, true>(cfg, tmap_w, tmap_x, p)
                              : launch_form<kBf16, kNT, kShift, 1, true>(cfg, tmap_w, tmap_x, p);
  return plan.slices == 2 ? launch_form<kBf16, kNT, kShift, 2, false>(cfg, tmap_w, tmap_x, p)
                          : launch_form<kBf16, kNT, kShift, 1, false>(cfg, tmap_w, tmap_x, p);
}

// Up to 8 activation rows, 16, or more in several passes over the weight: of 32 rows where the price is no higher (the
// prices of the two are good to a few percent), or a fifth lower where the passes would hold 16 rows of nothing; else of 16.
// bf16 in passes of 16 and of 32: 32 rows, 4096 x 14336 22.0 and 20.1 us, 14336 x 4096 with groups of 64 23.5 and 20.8, 28672 x
// 8192 73.5 and 58.7; 48 rows, 10240 x 8192 with groups of 32 52.5 and 60, 14336 x 4096 with groups of 64 42.7 and 33.
template <bool kBf16, int kShift>
int launch_rows(const uint8_t* codes, const void* x, int64_t ldx, W4Params& p, cudaStream_t st) {
  if (p.m <= 8) return launch_w4<kBf16, 1, kShift>(plan_for<kBf16, 1, kShift>(p), codes, x, ldx, p, st);
  const Plan two = plan_for<kBf16, 2, kShift>(p);
  if (p.m > 16) {
    const Plan four = plan_for<kBf16, 4, kShift>(p);
    const bool filled = (p.m + 31) / 32 * 32 - p.m < 16;
    if (four.cost - two.cost <= (filled ? two.cost / 50 : -two.cost / 5)) return launch_w4<kBf16, 4, kShift>(four, codes, x, ldx, p, st);
  }
  return launch_w4<kBf16, 2, kShift>(two, codes, x, ldx, p, st);
}

template <bool kBf16>
int launch_group(int group, const uint8_t* codes, const void* x, int64_t ldx, W4Params& p, cudaStream_t st) {
  if (group == 32) return launch_rows<kBf16, 0>(codes, x, ldx, p, st);
  if (group == 64) return launch_rows<kBf16, 1>(codes, x, ldx, p, st);
  return launch_rows<kBf16, 2>(codes, x, ldx, p, st);
}

// ---------------------------------------------------------------------------------------------------------------------
// Quantizer: one warp per group of a row
// ---------------------------------------------------------------------------------------------------------------------
template <bool kBf16>
__device__ __forceinline__ float rounded16(float v) { return Half16<kBf16>::value(Half16<kBf16>::round(v)); }

// zeros != NULL: s = rounded((max(max w, 0) - min(min w, 0)) / 15), z = clamp(rne(-min / s), 0, 15); otherwise
// s = rounded(max|w| / 7), z = 8.  q = clamp(rne(w / s) + z, 0, 15).  A group of zeros gets s = 1, one
// with a NaN s = NaN; where s overflows it is infinite, and the weights read back are not finite.
template <bool kBf16>
__global__ void __launch_bounds__(256)
quant_group_w4_kernel(const float* __restrict__ w, int64_t n, int k, int64_t ldw, int group, int groups,
                      uint8_t* __restrict__ codes, uint16_t* __restrict__ scales, uint8_t* __restrict__ zeros) {
  const int64_t item = static_cast<int64_t>(blockIdx.x) * 8 + (threadIdx.x >> 5);
  if (item >= n * groups) return;
  const int lane = threadIdx.x & 31;
  const int64_t row = item / groups;
  const int k0 = static_cast<int>(item - row * groups) * group, len = min(group, k - k0);
  const float* src = w + row * ldw + k0;
  float lo = 0.0f, hi = 0.0f;
  bool nan = false;
  for (int c = lane; c < len; c += 32) {
    const float v = src[c];
    nan |= v != v;
    lo = fminf(lo, v);
    hi = fmaxf(hi, v);
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    lo = fminf(lo, __shfl_xor_sync(0xffffffffu, lo, o));
    hi = fmaxf(hi, __shfl_xor_sync(0xffffffffu, hi, o));
  }
  float s = rounded16<kBf16>(zeros != nullptr ? __fdiv_rn(hi - lo, 15.0f) : __fdiv_rn(fmaxf(hi, -lo), 7.0f));
  if (s == 0.0f) s = 1.0f;
  if (__any_sync(0xffffffffu, nan)) s = __uint_as_float(0x7fffffffu);
  const int z = zeros != nullptr ? static_cast<int>(fminf(fmaxf(rintf(__fdiv_rn(-lo, s)), 0.0f), 15.0f)) : 8;
  if (lane == 0) {
    scales[item] = Half16<kBf16>::round(s);
    if (zeros != nullptr) zeros[item] = static_cast<uint8_t>(z);
  }
  auto code = [&](int c) {
    const float q = rintf(__fdiv_rn(src[c], s)) + static_cast<float>(z);
    return static_cast<uint32_t>(static_cast<int>(fminf(fmaxf(q, 0.0f), 15.0f)));
  };
  for (int c = 2 * lane; c < len; c += 64)                         // k % 32 == 0: pairs are whole
    codes[row * (k / 2) + (k0 + c) / 2] = static_cast<uint8_t>(code(c) | (code(c + 1) << 4));
}

}  // namespace
}  // namespace bfp8

using namespace bfp8;

extern "C" int bfp8_gemm_group_w4(const void* x, int64_t ldx, int x_dtype, const uint8_t* codes, const uint16_t* scales,
                                  const uint8_t* zeros, int group, const float* bias, void* out, int out_f32, int64_t ldo,
                                  int64_t m, int64_t n, int64_t k, uint32_t* status_dev, void* stream, int64_t wait_limit_cycles) {
  if (!x || !codes || !scales || !out || !status_dev) return BFP8_ERR_NULL;
  const bool fresh_codes = (x_dtype & BFP8_W4_FRESH_CODES) != 0;
  x_dtype &= ~BFP8_W4_FRESH_CODES;
  if (m <= 0 || n <= 0 || k <= 0 || m > kMaxM || n > (1 << 30) || k > (1 << 30) || ldx < k || ldo < n) return BFP8_ERR_SHAPE;
  if (x_dtype != BFP8_W4_BF16 && x_dtype != BFP8_W4_F16) return BFP8_ERR_SHAPE;
  if (group != 32 && group != 64 && group != 128) return BFP8_ERR_UNSUPPORTED;
  if (k % 32 != 0) return BFP8_ERR_UNSUPPORTED;
  if (!aligned(x, 16) || ldx % 8 != 0 || !aligned(codes, 16) || !aligned(scales, 2) || !aligned(out, out_f32 ? 4 : 2) ||
      (bias && !aligned(bias, 4)) || !aligned(status_dev, 4))
    return BFP8_ERR_ALIGN;
  W4Params p = {};
  p.scales = scales;
  p.zeros = zeros;
  p.bias = bias;
  p.out = out;
  p.ldo = ldo;
  p.m = static_cast<int>(m);
  p.n = static_cast<int>(n);
  p.k = static_cast<int>(k);
  p.groups = static_cast<int>((k + group - 1) / group);
  p.out_f32 = out_f32 != 0;
  p.w_early = weights_at_rest() && !fresh_codes ? 1 : 0;
  p.wait_limit = wait_limit_cycles > 0 ? wait_limit_cycles : kDefaultWaitLimit;
  p.status = status_dev;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  return x_dtype == BFP8_W4_BF16 ? launch_group<true>(group, codes, x, ldx, p, st) : launch_group<false>(group, codes, x, ldx, p, st);
}

extern "C" int bfp8_quant_group_w4_f32(const float* w, int64_t n, int64_t k, int64_t ldw, int group, uint8_t* codes,
                                       uint16_t* scales, uint8_t* zeros, int scale_dtype, void* stream) {
  if (!w || !codes || !scales) return BFP8_ERR_NULL;
  if (n <= 0 || k <= 0 || n > (1 << 30) || k > (1 << 30) || ldw < k) return BFP8_ERR_SHAPE;
  if (scale_dtype != BFP8_W4_BF16 && scale_dtype != BFP8_W4_F16) return BFP8_ERR_SHAPE;
  if ((group != 32 && group != 64 && group != 128) || k % 32 != 0) return BFP8_ERR_UNSUPPORTED;
  if (!aligned(w, 4) || !aligned(scales, 2)) return BFP8_ERR_ALIGN;
  const int64_t groups = (k + group - 1) / group, blocks = (n * groups + 7) / 8;
  if (blocks > 2147483647LL) return BFP8_ERR_SHAPE;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const dim3 grid(static_cast<unsigned>(blocks)), block(256);
  if (scale_dtype == BFP8_W4_BF16)
    quant_group_w4_kernel<true><<<grid, block, 0, st>>>(w, n, static_cast<int>(k), ldw, group, static_cast<int>(groups), codes, scales, zeros);
  else
    quant_group_w4_kernel<false><<<grid, block, 0, st>>>(w, n, static_cast<int>(k), ldw, group, static_cast<int>(groups), codes, scales, zeros);
  BFP8_CUDA_TRY(cudaGetLastError());
  return BFP8_OK;
}
