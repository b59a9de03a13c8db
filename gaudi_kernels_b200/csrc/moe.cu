// Routed experts for a few tokens (sm_100a): the router's top-k and a whole block-FP8 mixture-of-experts layer.
//
//   l[t, e] = fp32(sum_h x[t, h] r[e, h]);   (ids, w)[t] = top-k of the scores;
//   xq = E4M3(x) by groups of 128;   h[s] = silu(xq . Wg[id_s]^T) * (xq . Wu[id_s]^T) of slot s = (token, choice);
//   hq = E4M3(h) by groups of 128;   y[t] = sum_s w_s (hq[s] . Wd[id_s]^T).
//
// A few tokens read every weight of the experts they reach once and do little arithmetic with it, so the layer is bound by
// HBM and, for one token, by the latency of its dependent steps.  Two kernels:
//   * moe_front_kernel: the router's products (scores) and the activation quantizer, independent work of one launch; it
//     also zeroes the synchronisation words of the second kernel, so no state outlives a call and workspaces need no
//     preparation.
//   * moe_experts_kernel: one CTA per SM, launched cooperatively (its CTAs wait for one another).  Every CTA picks the
//     top-k itself (a few microseconds of redundant work instead of a third launch), sorts the slots by expert, and cuts
//     the list of units - 256 weight rows x one 128-wide K block, 32 KB - evenly over the CTAs, first for gate/up, then
//     for down: each SM streams the same number of bytes whatever the routing is.
// In one expert 128 weight rows are the M dimension of a tcgen05.mma and the tokens that chose it the N dimension (16 at a
// time), so padding costs no HBM traffic; a unit holds the gate and the up rows of the same 128 outputs, which are one
// quantization group of h: the SwiGLU step and the second quantizer are the epilogue of the first product and h never
// leaves the chip in more than 8 bits.  The second product of a chunk of an expert's slots waits until all of the chunk's h is
// there (a counter per chunk, no barrier of the grid: 150 -> 144 us where 128 tokens reach 31 experts of H = 4096, I = 2048); the
// weight producer does not wait, it fills the pipeline with the down projection's first units meanwhile.
#include <cuda.h>

#include "common.cuh"
#include "ptx.cuh"

namespace bfp8 {

namespace {

constexpr int kMaxTokens = 128;
constexpr int kMaxTopK = 32;
constexpr int kMaxSlots = 2048;        // tokens * top_k
constexpr int kMaxExperts = 512;
constexpr int kMaxWidth = 1 << 16;     // h and inter: a phase's units fit 32 bits
constexpr int kMaxGrid = 256;          // the workspace holds this many CTAs' partial sums
constexpr long long kDefaultWaitLimit = 2000000000LL;      // about a second

// Synchronisation words at the start of the workspace (zeroed by the first kernel of every call)
constexpr int kMaxChunks = kMaxExperts + kMaxSlots / 16;
constexpr int kSyncBarrier = 0;                    // grid barrier
constexpr int kSyncFlags = 32;                     // [CTA][tile]: partial sum of the first product stored
constexpr int kSyncChunks = kSyncFlags + 2 * kMaxGrid;       // [chunk]: groups of h finished
constexpr int kSyncWords = kSyncChunks + kMaxChunks;

// ---------------------------------------------------------------------------------------------------------------------
// Top-k of one token's scores, by one warp
// ---------------------------------------------------------------------------------------------------------------------

struct RouteRule {
  const float* bias;     // [experts] added for the choice alone, or NULL
  int softmax;           // weights: softmax of the scores, else the scores themselves
  int renorm;            // over the chosen ones only
  float scale;
};

// Order-preserving map of fp32 to unsigned: NaN below everything, +0 and -0 alike.  0 is left for "taken".
__device__ __forceinline__ uint32_t order_key(float v) {
  if (v != v) return 1u;
  const uint32_t b = __float_as_uint(v + 0.0f);
  return (b & 0x80000000u) ? ~b : (b | 0x80000000u);
}

// Largest keys first, ties to the lowest index.  Lane j (j < k) returns the j-th choice and its weight.
template <int kPer>
__device__ __forceinline__ void topk_token(const float* __restrict__ row, int experts, int k, const RouteRule& r, int lane,
                                           int& my_id, float& my_weight) {
  float score[kPer], bias[kPer];
  uint32_t key[kPer];
  float top = -INFINITY;
  // all loads on their way before the first is used
#pragma unroll
  for (int q = 0; q < kPer; ++q) score[q] = __ldcg(row + min(q * 32 + lane, experts - 1));
#pragma unroll
  for (int q = 0; q < kPer; ++q) bias[q] = r.bias != nullptr ? __ldg(r.bias + min(q * 32 + lane, experts - 1)) : 0.0f;
#pragma unroll
  for (int q = 0; q < kPer; ++q) key[q] = q * 32 + lane < experts ? order_key(score[q] + bias[q]) : 0u;
  my_id = -1;
  float my_score = 0.0f;
  // every lane keeps the largest of its own keys; only the lane whose key was taken looks for its next one
  uint32_t best = 0u;
  int best_q = 0;
  float best_score = 0.0f;
  auto own_best = [&] {
    best = 0u;
#pragma unroll
    for (int q = 0; q < kPer; ++q)
      if (key[q] > best) { best = key[q]; best_q = q; best_score = score[q]; }
  };
  own_best();
  for (int j = 0; j < k; ++j) {
    const uint32_t most = __reduce_max_sync(0xffffffffu, best);
    const uint32_t mine = best == most ? static_cast<uint32_t>(best_q * 32 + lane) : 0xffffffffu;
    const uint32_t id = __reduce_min_sync(0xffffffffu, mine);
    const float s = __shfl_sync(0xffffffffu, best_score, id & 31u);
    if (j == 0) top = s;
    if (lane == j) { my_id = static_cast<int>(id); my_score = s; }
    if (mine == id) {
#pragma unroll
      for (int q = 0; q < kPer; ++q)
        if (q == best_q) key[q] = 0u;
      own_best();
    }
    __syncwarp();
  }
  float w = lane < k ? my_score : 0.0f;
  if (r.softmax) {
    // without a bias the first choice is the largest score
    w = lane < k ? expf(my_score - top) : 0.0f;
    float sum = w;
    if (!r.renorm) {
      sum = 0.0f;
#pragma unroll
      for (int q = 0; q < kPer; ++q)
        if (q * 32 + lane < experts) sum += expf(score[q] - top);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    w /= sum;
  } else if (r.renorm) {
    float sum = w;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    w /= sum + 1e-20f;
  }
  my_weight = w * r.scale;
}

__device__ __forceinline__ void topk_any(const float* __restrict__ row, int experts, int k, const RouteRule& r, int lane, int& my_id,
                                         float& my_weight) {
  if (experts <= 128) topk_token<4>(row, experts, k, r, lane, my_id, my_weight);
  else if (experts <= 256) topk_token<8>(row, experts, k, r, lane, my_id, my_weight);
  else topk_token<kMaxExperts / 32>(row, experts, k, r, lane, my_id, my_weight);
}

__global__ void __launch_bounds__(128)
moe_topk_kernel(const float* __restrict__ scores, int64_t tokens, int experts, int k, RouteRule rule, int32_t* __restrict__ ids,
                float* __restrict__ weights) {
  ptx::griddep_launch_dependents();
  ptx::griddep_wait();
  const int64_t t = static_cast<int64_t>(blockIdx.x) * 4 + (threadIdx.x >> 5);
  if (t >= tokens) return;
  const int lane = threadIdx.x & 31;
  int id;
  float w;
  topk_any(scores + t * experts, experts, k, rule, lane, id, w);
  if (lane < k) {
    ids[t * k + lane] = id;
    weights[t * k + lane] = w;
  }
}

// ---------------------------------------------------------------------------------------------------------------------
// First kernel: router scores and activation quantizer
// ---------------------------------------------------------------------------------------------------------------------
constexpr int kFrontWarps = 16;

struct FrontParams {
  const uint16_t* x;
  int64_t ldx;
  int64_t t;
  int h;
  int vec;                     // rows of x and of the router start on 16 bytes and h % 8 == 0
  // quantizer (quant_blocks == 0: none)
  int quant_blocks;
  int groups, half;
  uint8_t* codes;              // [t, h]
  float* scales;               // [groups, t]
  uint32_t* sync;
  // router (router == NULL: none)
  const uint16_t* router;
  int64_t ldr;
  int experts, sigmoid;
  float* scores;               // [t, experts]
};

// Eight bf16 values at column c of a row as packed pairs, zero beyond h
__device__ __forceinline__ uint4 load8(const uint16_t* row, int c, int h, bool vec) {
  uint4 v = make_uint4(0u, 0u, 0u, 0u);
  if (vec) {
    if (c < h) v = __ldg(reinterpret_cast<const uint4*>(row + c));
  } else {
    uint32_t* w = reinterpret_cast<uint32_t*>(&v);
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (c + j < h) w[j >> 1] |= static_cast<uint32_t>(__ldg(row + c + j)) << (16 * (j & 1));
  }
  return v;
}

// A score decides which experts run, so its sum is formed in fp64: products of bf16 numbers are exact there, and the sum is off by
// 2^-53 of its terms per addition.  (Sums of 16 or 32 terms in fp32 first, as the tensor core forms them, cost half the time for
// many tokens, but put one of a hundred scores off by a step of fp32 where two columns of x are a thousand times the others, and
// differ between batch sizes.  Both launches of the router, 1 x 64 x 2048, 8 x 256 x 4096, 128 x 256 x 4096: 4.2, 8.9 and 15.2 us,
// with fp32 sums in blocks of 16 x 16 and a warp per token and expert 5.6, 8.0 and 9.8.)
__device__ __forceinline__ float score_of(const FrontParams& p, double sum) {
  const float l = static_cast<float>(sum);
  return p.sigmoid ? static_cast<float>(1.0 / (1.0 + exp(-static_cast<double>(l)))) : l;
}

__device__ __forceinline__ double bf16_lo_to_double(uint32_t v) { return static_cast<double>(bf16_lo_to_float(v)); }
__device__ __forceinline__ double bf16_hi_to_double(uint32_t v) { return static_cast<double>(bf16_hi_to_float(v)); }

// c += a b, 8 rows x 4 k x 8 columns in fp64: lane 4 g + t has row g (column g) at one k of its choice and columns 2 t, 2 t + 1 of row g
__device__ __forceinline__ void mma_f64(double (&c)[2], double a, double b) {
  asm("mma.sync.aligned.m8n8k4.row.col.f64.f64.f64.f64 {%0,%1}, {%2}, {%3}, {%0,%1};" : "+d"(c[0]), "+d"(c[1]) : "d"(a), "d"(b));
}

// Up to four tokens: eight warps per expert, each with every eighth 256 columns of its row, for all tokens.
constexpr int kDotTokens = 4, kDotSlices = 8, kDotExperts = kFrontWarps / kDotSlices;
__device__ __forceinline__ void router_dot(const FrontParams& p, int e0, int warp, int lane, double* red) {
  double acc[kDotTokens] = {};
  const bool vec = p.vec != 0;
  const int e = e0 + warp / kDotSlices;
  if (e < p.experts) {
    const uint16_t* wr = p.router + e * p.ldr;
#pragma unroll 2
    for (int c = (warp % kDotSlices * 32 + lane) * 8; c < p.h; c += kDotSlices * 256) {
      const uint4 w = load8(wr, c, p.h, vec);
      uint4 x[kDotTokens];
#pragma unroll
      for (int t = 0; t < kDotTokens; ++t)
        if (t < p.t) x[t] = load8(p.x + t * p.ldx, c, p.h, vec);
      const uint32_t a[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
      for (int t = 0; t < kDotTokens; ++t)
        if (t < p.t) {
          const uint32_t b[4] = {x[t].x, x[t].y, x[t].z, x[t].w};
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            acc[t] = fma(bf16_lo_to_double(a[j]), bf16_lo_to_double(b[j]), acc[t]);
            acc[t] = fma(bf16_hi_to_double(a[j]), bf16_hi_to_double(b[j]), acc[t]);
          }
        }
    }
  }
#pragma unroll
  for (int t = 0; t < kDotTokens; ++t)
    if (t < p.t) {
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) acc[t] += __shfl_xor_sync(0xffffffffu, acc[t], o);
      if (lane == 0) red[warp * kDotTokens + t] = acc[t];
    }
  __syncthreads();
  const int i = threadIdx.x / kDotTokens, t = threadIdx.x % kDotTokens;
  if (i < kDotExperts && e0 + i < p.experts && t < p.t) {
    double v = 0.0;
    for (int w = 0; w < kDotSlices; ++w) v += red[(i * kDotSlices + w) * kDotTokens + t];
    p.scores[t * p.experts + e0 + i] = score_of(p, v);
  }
}

// More tokens: a block has 8 kA experts (rows of the fp64 mma.sync) and 8 kB tokens (columns); its warps take turns in K, 32 at a
// time.  A thread's operands are 8 consecutive k of its rows as they lie in memory: which k an operand stands for is free as long
// as both agree.  fp64 bounds it, 64 multiplications per SM and cycle: 128 tokens, 256 experts and H = 4096 need 7.4 us, the kernel
// takes 11.
template <int kA, int kB>
__device__ __forceinline__ void router_tile(const FrontParams& p, int64_t t0, int e0, double* red) {
  constexpr int kE = 8 * kA, kT = 8 * kB;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const bool vec = p.vec != 0;
  double acc[kA][kB][2] = {};
  const uint4 none = make_uint4(0u, 0u, 0u, 0u);
#pragma unroll 4
  for (int c = warp * 32; c < p.h; c += kFrontWarps * 32) {
    const int k = c + t * 8;
    uint4 w[kA], x[kB];
#pragma unroll
    for (int a = 0; a < kA; ++a) {
      const int row = e0 + a * 8 + g;
      w[a] = row < p.experts ? load8(p.router + row * p.ldr, k, p.h, vec) : none;
    }
#pragma unroll
    for (int b = 0; b < kB; ++b) {
      const int64_t row = t0 + b * 8 + g;
      x[b] = row < p.t ? load8(p.x + row * p.ldx, k, p.h, vec) : none;
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      auto value = [&](const uint4& v) {
        const uint32_t two = j < 2 ? v.x : j < 4 ? v.y : j < 6 ? v.z : v.w;
        return j & 1 ? bf16_hi_to_double(two) : bf16_lo_to_double(two);
      };
      double d[kB];
#pragma unroll
      for (int b = 0; b < kB; ++b) d[b] = value(x[b]);
#pragma unroll
      for (int a = 0; a < kA; ++a) {
        const double v = value(w[a]);
#pragma unroll
        for (int b = 0; b < kB; ++b) mma_f64(acc[a][b], v, d[b]);
      }
    }
  }
  // the warps' sums, [warp][token][expert]
#pragma unroll
  for (int a = 0; a < kA; ++a)
#pragma unroll
    for (int b = 0; b < kB; ++b)
#pragma unroll
      for (int j = 0; j < 2; ++j) red[(warp * kT + b * 8 + 2 * t + j) * kE + a * 8 + g] = acc[a][b][j];
  __syncthreads();
  for (int i = threadIdx.x; i < kT * kE; i += kFrontWarps * 32) {
    const int64_t token = t0 + i / kE;
    const int e = e0 + i % kE;
    if (token < p.t && e < p.experts) {
      double v = 0.0;
      for (int w = 0; w < kFrontWarps; ++w) v += red[w * kT * kE + i];
      p.scores[token * p.experts + e] = score_of(p, v);
    }
  }
}

// Scale of a group whose largest magnitude has these bits; NaN where that is inf or NaN, so the whole group becomes NaN.
__device__ __forceinline__ float group_scale(uint32_t bits) {
  return bits < 0x7f800000u ? scale_from_amax(__uint_as_float(bits)) : __uint_as_float(0x7fffffffu);
}

// One warp: 128 columns of one token to E4M3 (the rule of bfp8_quant_act_1x128_bf16, four columns per lane).
__device__ __forceinline__ void quantize_group(const FrontParams& p, int64_t t, int g, int lane) {
  const int c = g * 128 + lane * 4;
  const uint16_t* row = p.x + t * p.ldx;
  float f[4] = {0.0f, 0.0f, 0.0f, 0.0f};
  if (p.vec) {
    if (c < p.h) {                                         // h % 8 == 0
      const uint2 v = __ldg(reinterpret_cast<const uint2*>(row + c));
      f[0] = bf16_lo_to_float(v.x); f[1] = bf16_hi_to_float(v.x);
      f[2] = bf16_lo_to_float(v.y); f[3] = bf16_hi_to_float(v.y);
    }
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (c + j < p.h) f[j] = bf16_bits_to_float(__ldg(row + c + j));
  }
  uint32_t bits = 0u;                                      // |f| as an integer: NaN is the largest
#pragma unroll
  for (int j = 0; j < 4; ++j) bits = max(bits, __float_as_uint(f[j]) & 0x7fffffffu);
  const float scale = group_scale(__reduce_max_sync(0xffffffffu, bits));
  const float rcp = __frcp_rn(scale);
  const uint32_t q = p.half ? quant_half_e4m3x4(f[0], f[1], f[2], f[3], scale, rcp) : quant_e4m3x4(f[0], f[1], f[2], f[3], scale, rcp);
  if (c < p.h) *reinterpret_cast<uint32_t*>(p.codes + t * p.h + c) = q;      // h % 16 == 0
  if (lane == 0) p.scales[static_cast<int64_t>(g) * p.t + t] = p.half ? scale * 2.0f : scale;
}

// kA, kB: a router block's experts and tokens / 8, 0: up to four tokens
template <int kA, int kB>
__global__ void __launch_bounds__(kFrontWarps * 32)
moe_front_kernel(const FrontParams p) {
  __shared__ double red[kB > 0 ? kFrontWarps * 64 * kA * kB : kFrontWarps * kDotTokens];
  ptx::griddep_launch_dependents();
  ptx::griddep_wait();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (p.sync != nullptr && blockIdx.x == 0)
    for (int i = threadIdx.x; i < kSyncWords; i += blockDim.x) p.sync[i] = 0u;
  if (static_cast<int>(blockIdx.x) < p.quant_blocks) {
    const int64_t item = static_cast<int64_t>(blockIdx.x) * kFrontWarps + warp;
    if (item < p.t * p.groups) quantize_group(p, item / p.groups, static_cast<int>(item % p.groups), lane);
    return;
  }
  const int64_t block = blockIdx.x - p.quant_blocks;
  if (kB == 0) {
    router_dot(p, static_cast<int>(block) * kDotExperts, warp, lane, red);
  } else {
    const int eb = (p.experts + 8 * kA - 1) / (8 * kA);
    router_tile<kA, kB == 0 ? 1 : kB>(p, block / eb * (8 * kB), static_cast<int>(block % eb) * (8 * kA), red);
  }
}

int launch_front(FrontParams& p, cudaStream_t st) {
  const int64_t quant = p.quant_blocks ? (p.t * p.groups + kFrontWarps - 1) / kFrontWarps : 0;
  p.quant_blocks = static_cast<int>(quant);
  // router blocks as small as lets the device hold them at once, one per SM
  const int64_t e8 = (p.experts + 7) / 8, e16 = (p.experts + 15) / 16, t8 = (p.t + 7) / 8, t16 = (p.t + 15) / 16;
  const int form = p.t <= kDotTokens ? 0 : e8 * t8 <= sm_count() ? 1 : e16 * t8 <= sm_count() ? 2 : 3;
  int64_t route = 0;
  if (p.router != nullptr)
    route = form == 0 ? (p.experts + kDotExperts - 1) / kDotExperts : form == 1 ? e8 * t8 : form == 2 ? e16 * t8 : e16 * t16;
  if (quant + route > 2147483647LL) return BFP8_ERR_SHAPE;
  const dim3 grid(static_cast<unsigned>(quant + route)), block(kFrontWarps * 32);
  switch (form) {
    case 0: return launch_overlapped(moe_front_kernel<1, 0>, grid, block, 0, st, p);
    case 1: return launch_overlapped(moe_front_kernel<1, 1>, grid, block, 0, st, p);
    case 2: return launch_overlapped(moe_front_kernel<2, 1>, grid, block, 0, st, p);
    default: return launch_overlapped(moe_front_kernel<2, 2>, grid, block, 0, st, p);
  }
}

// ---------------------------------------------------------------------------------------------------------------------
// Second kernel: the experts
// ---------------------------------------------------------------------------------------------------------------------
constexpr int BK = 128;
constexpr int kTileBytes = 128 * BK;               // 128 weight rows x one K block
constexpr int kWBytes = 2 * kTileBytes;            // gate and up, or two neighbouring down tiles
constexpr int kAccBufs = 4;
constexpr int kStageBudget = 200 * 1024;
constexpr int kMaxStages = 6;
constexpr int kRowProducer = 8, kTokenProducer = 9, kIssuer = 10, kScaleWarp = 12, kWarps = 13;
constexpr int kThreads = kWarps * 32;
constexpr int kScaleAhead = 4;

// NC: slots of one expert that are multiplied together (a chunk); an expert with more has its weight read again, from L2.
template <int NC>
struct Cfg {
  static constexpr int kStageBytes = kWBytes + NC * BK;
  static constexpr int kStages = kStageBudget / kStageBytes < kMaxStages ? kStageBudget / kStageBytes : kMaxStages;
  static constexpr int kTmemCols = 2 * kAccBufs * NC;
};

struct Routing {
  int16_t slot_expert[kMaxSlots];      // -1: no expert here
  uint16_t count[kMaxExperts];
  uint16_t start[kMaxExperts];
  uint16_t chunk[kMaxExperts];
};
struct Exchange {
  float value[2][8][128];              // [up to the gate side / gate to the up side][column][row]
  float most[8][8];                    // [warp][column] largest magnitude of the warp's rows
};

struct Tail {
  uint64_t full[kMaxStages], empty[kMaxStages];
  uint64_t tmem_full[2][kAccBufs], tmem_empty[2][kAccBufs];
  float scale[kAccBufs][2][64];
  uint16_t place_of_slot[kMaxSlots];   // chunk * 64 + column of a slot, 0xffff: none
  uint8_t token_of_pos[kMaxSlots];
  uint16_t chunk_expert[kMaxChunks];
  uint16_t chunk_start[kMaxChunks];
  uint8_t chunk_count[kMaxChunks];
  union {
    Routing routing;                   // until the work list stands
    Exchange ex;                       // from then on
  };
  uint32_t tmem_base, abort_flag, flag[2];
  int chunks;
};

struct ExpertParams {
  const float* x_scales;   // [groups_h][t]
  const float* scores;     // [t][experts]: the choice is made here; NULL: ids and weights are given
  RouteRule rule;
  const int32_t* ids;      // [t][k]
  float* weights;          // [t][k]
  int32_t* ids_out;        // written where scores are given
  const float* s13;        // [experts][2][ceil(i / 128)][ceil(h / 128)]
  const float* s2;         // [experts][ceil(h / 128)][ceil(i / 128)]
  uint8_t* hq;             // [slots + pad][i] in the order of experts
  float* h_scales;         // [ceil(i / 128)][spad]
  float* partials;         // [product][CTA][tile][NC][128]: a CTA may store its second while its first is still to be read
  float* y;                // [slots][h]
  uint32_t* sync;
  uint16_t* out;
  int64_t ldo;
  int t, k, experts, h, i, gh, gi, hpairs, spad, half;
  long long wait_limit;
  uint32_t* status;
};

// `total` units cut evenly over `parts` CTAs, each of which has at least one.
struct Shares {
  uint32_t total, parts, base, extra;                  // the first `extra` CTAs have base + 1 units
  __device__ __forceinline__ Shares(uint32_t total_, uint32_t ctas) : total(total_), parts(min(total_, ctas)) {
    base = parts > 0 ? total / parts : 0u;
    extra = total - base * parts;
  }
  __device__ __forceinline__ uint32_t first(uint32_t c) const { return c < parts ? c * base + min(c, extra) : total; }
  __device__ __forceinline__ uint32_t cta_of(uint32_t u) const {
    const uint32_t large = extra * (base + 1);
    return u < large ? u / (base + 1) : extra + (u - large) / base;
  }
};

// Position in the unit list of a phase: (chunk, pair of tiles, K block).  Both products go through the chunks in the same
// order, so a CTA's share of the second one needs h of the chunks whose first product it and its neighbours have just done.
struct Cursor {
  int chunk, j, g, groups, pairs;
  __device__ __forceinline__ Cursor(uint32_t u, int pairs_, int groups_) : groups(groups_), pairs(pairs_) {
    const uint32_t item = u / static_cast<uint32_t>(groups);
    g = static_cast<int>(u - item * groups);
    chunk = static_cast<int>(item / static_cast<uint32_t>(pairs));
    j = static_cast<int>(item % static_cast<uint32_t>(pairs));
  }
  __device__ __forceinline__ void next() {
    if (++g < groups) return;
    g = 0;
    if (++j == pairs) { j = 0; ++chunk; }
  }
};

// Bounded wait for *word >= want, by one thread.
__device__ __forceinline__ bool wait_word(const uint32_t* word, uint32_t want, volatile uint32_t* abort_flag, long long limit) {
  const long long t0 = clock64();
  while (ptx::ld_acquire_gpu_u32(word) < want) {
    if (*abort_flag != 0) return false;
    if (clock64() - t0 > limit) { *abort_flag = 1; return false; }
  }
  return true;
}

__device__ __forceinline__ void red_release_add(uint32_t* word) {
  asm volatile("red.release.gpu.global.add.u32 [%0], 1;" ::"l"(word) : "memory");
}
__device__ __forceinline__ void fence_proxy_async() { asm volatile("fence.proxy.async;" ::: "memory"); }
__device__ __forceinline__ void named_sync(int id, int threads) {
  asm volatile("bar.sync %0, %1;" ::"r"(id), "r"(threads) : "memory");
}
__device__ __forceinline__ void tma_load_3d_hint(uint32_t dst, const CUtensorMap* m, uint32_t bar, int x, int y, int z,
                                                 uint64_t policy) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes.L2::cache_hint [%0], [%1, {%3, %4, %5}], [%2], %6;"
      ::"r"(dst), "l"(reinterpret_cast<uint64_t>(m)), "r"(bar), "r"(x), "r"(y), "r"(z), "l"(policy) : "memory");
}
__device__ __forceinline__ uint64_t l2_policy_evict_normal() {
  uint64_t policy;
  asm volatile("createpolicy.fractional.L2::evict_normal.b64 %0, 1.0;" : "=l"(policy));
  return policy;
}

// The work list: slots sorted by expert (stable, so every CTA gets the same order), experts in chunks of NC slots.
template <int NC>
__device__ __forceinline__ void build_work_list(const ExpertParams& p, Tail* tail, int warp, int lane) {
  Routing& rt = tail->routing;
  const int slots = p.t * p.k;
  for (int e = threadIdx.x; e < p.experts; e += kThreads) rt.count[e] = 0;
  if (p.scores != nullptr) {
    for (int t = warp; t < p.t; t += kWarps) {
      int id;
      float w;
      topk_any(p.scores + static_cast<int64_t>(t) * p.experts, p.experts, p.k, p.rule, lane, id, w);
      if (lane < p.k) {
        rt.slot_expert[t * p.k + lane] = static_cast<int16_t>(id);
        if (blockIdx.x == 0) {
          p.ids_out[t * p.k + lane] = id;
          p.weights[t * p.k + lane] = w;
        }
      }
    }
  } else {
    bool bad = false;
    for (int s = threadIdx.x; s < slots; s += kThreads) {
      const int id = __ldg(p.ids + s);
      bad |= id >= p.experts;
      rt.slot_expert[s] = static_cast<int16_t>(id >= 0 && id < p.experts ? id : -1);
    }
    if (bad && blockIdx.x == 0) atomicOr(p.status, BFP8_STATUS_BAD_INDEX);
  }
  __syncthreads();
  if (warp == 0) {
    for (int base = 0; base < slots; base += 32) {                 // place of each slot inside its expert
      const int s = base + lane;
      const int e = s < slots ? rt.slot_expert[s] : -1;
      const uint32_t same = __match_any_sync(0xffffffffu, e);
      const int before = __popc(same & ((1u << lane) - 1u));
      const int have = e >= 0 ? rt.count[e] : 0;
      __syncwarp();
      if (s < slots) tail->place_of_slot[s] = static_cast<uint16_t>(e >= 0 ? have + before : 0xffff);
      if (e >= 0 && (same >> lane) == 1u) rt.count[e] = static_cast<uint16_t>(have + before + 1);   // the last of them
      __syncwarp();
    }
    int pos = 0, chunk = 0;
    for (int base = 0; base < p.experts; base += 32) {
      const int e = base + lane;
      const int c = e < p.experts ? rt.count[e] : 0;
      const int n = (c + NC - 1) / NC;
      int upto = c, chunks_upto = n;                               // inclusive sums over the lanes
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int a = __shfl_up_sync(0xffffffffu, upto, o), b = __shfl_up_sync(0xffffffffu, chunks_upto, o);
        if (lane >= o) { upto += a; chunks_upto += b; }
      }
      const int first = pos + upto - c;
      if (e < p.experts) { rt.start[e] = static_cast<uint16_t>(first); rt.chunk[e] = static_cast<uint16_t>(chunk + chunks_upto - n); }
      for (int q = 0; q < n; ++q) {
        const int at = chunk + chunks_upto - n + q;
        tail->chunk_expert[at] = static_cast<uint16_t>(e);
        tail->chunk_start[at] = static_cast<uint16_t>(first + q * NC);
        tail->chunk_count[at] = static_cast<uint8_t>(min(NC, c - q * NC));
      }
      pos += __shfl_sync(0xffffffffu, upto, 31);
      chunk += __shfl_sync(0xffffffffu, chunks_upto, 31);
    }
    if (lane == 0) tail->chunks = chunk;
  }
  __syncthreads();
  for (int s = threadIdx.x; s < slots; s += kThreads) {
    const int e = rt.slot_expert[s];
    if (e >= 0) {
      const int at = tail->place_of_slot[s];
      tail->place_of_slot[s] = static_cast<uint16_t>((rt.chunk[e] + at / NC) * 64 + at % NC);
      tail->token_of_pos[rt.start[e] + at] = static_cast<uint8_t>(s / p.k);
    }
  }
  __syncthreads();
}

template <int NC>
__global__ void __launch_bounds__(kThreads, 1)
moe_experts_kernel(const __grid_constant__ CUtensorMap tmap_w13, const __grid_constant__ CUtensorMap tmap_w2,
                   const __grid_constant__ CUtensorMap tmap_x, const __grid_constant__ CUtensorMap tmap_h,
                   const ExpertParams p) {
  using C = Cfg<NC>;
  extern __shared__ uint8_t smem_raw[];
  const uint32_t smem_base = (ptx::smem_u32(smem_raw) + 1023u) & ~1023u;
  Tail* tail = reinterpret_cast<Tail*>(smem_raw + (smem_base - ptx::smem_u32(smem_raw)) + C::kStages * C::kStageBytes);
  volatile uint32_t* abort_flag = &tail->abort_flag;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  if (threadIdx.x == 0) {
    for (int s = 0; s < C::kStages; ++s) {
      ptx::mbar_init(ptx::smem_u32(&tail->full[s]), 2);            // weight rows, token rows
      ptx::mbar_init(ptx::smem_u32(&tail->empty[s]), 2);           // one commit per tile
    }
    for (int w = 0; w < 2; ++w)
      for (int b = 0; b < kAccBufs; ++b) {
        ptx::mbar_init(ptx::smem_u32(&tail->tmem_full[w][b]), 2);  // MMAs, scales
        ptx::mbar_init(ptx::smem_u32(&tail->tmem_empty[w][b]), 4);
      }
    tail->abort_flag = 0;
    ptx::fence_mbar_init();
  }
  if (threadIdx.x == kRowProducer * 32) {
    ptx::prefetch_tensormap(&tmap_w13);
    ptx::prefetch_tensormap(&tmap_w2);
  }
  if (threadIdx.x == kTokenProducer * 32) {
    ptx::prefetch_tensormap(&tmap_x);
    ptx::prefetch_tensormap(&tmap_h);
  }
  if (warp == kIssuer) {
    ptx::tmem_alloc(ptx::smem_u32(&tail->tmem_base), C::kTmemCols);
    ptx::tmem_relinquish();
  }
  ptx::griddep_wait();
  build_work_list<NC>(p, tail, warp, lane);
  ptx::tc_fence_before_sync();
  __syncthreads();
  ptx::tc_fence_after_sync();
  const uint32_t tmem_base = tail->tmem_base;
  const int chunks = tail->chunks;
  const Shares shares[2] = {Shares(static_cast<uint32_t>(chunks) * p.gi * p.gh, gridDim.x),
                            Shares(static_cast<uint32_t>(p.hpairs) * chunks * p.gi, gridDim.x)};
  auto cursor = [&](int phase, uint32_t u) {
    return phase == 0 ? Cursor(u, p.gi, p.gh) : Cursor(u, p.hpairs, p.gi);
  };
  const uint32_t barrier_count = 2u * gridDim.x;                   // both tile halves of every CTA arrive

  if (warp == kRowProducer) {
    // ------------------------------------------------------------------ weight rows
    if (lane == 0) {
      const uint64_t once = ptx::l2_policy_evict_first(), again = l2_policy_evict_normal();
      uint32_t stage = 0, parity = 0;
      bool ok = true;
      for (int phase = 0; phase < 2 && ok; ++phase) {
        const uint32_t u0 = shares[phase].first(blockIdx.x), u1 = shares[phase].first(blockIdx.x + 1);
        if (u0 >= u1) continue;
        Cursor c = cursor(phase, u0);
        for (uint32_t u = u0; u < u1; ++u, c.next()) {
          const uint32_t full = ptx::smem_u32(&tail->full[stage]), dst = smem_base + stage * C::kStageBytes;
          ok = ptx::mbar_wait(ptx::smem_u32(&tail->empty[stage]), parity ^ 1u, abort_flag, p.wait_limit);
          if (!ok) break;
          ptx::mbar_arrive_expect_tx(full, kWBytes);
          const int e = tail->chunk_expert[c.chunk];
          const uint64_t policy = (c.chunk + 1 < chunks && tail->chunk_expert[c.chunk + 1] == e) ||
                                  (c.chunk > 0 && tail->chunk_expert[c.chunk - 1] == e) ? again : once;
          if (phase == 0) {
            tma_load_3d_hint(dst, &tmap_w13, full, c.g * BK, c.j * 128, 2 * e, policy);
            tma_load_3d_hint(dst + kTileBytes, &tmap_w13, full, c.g * BK, c.j * 128, 2 * e + 1, policy);
          } else {
            tma_load_3d_hint(dst, &tmap_w2, full, c.g * BK, c.j * 256, e, policy);
            tma_load_3d_hint(dst + kTileBytes, &tmap_w2, full, c.g * BK, c.j * 256 + 128, e, policy);
          }
          if (++stage == C::kStages) { stage = 0; parity ^= 1u; }
        }
      }
    }
  } else if (warp == kTokenProducer) {
    // ------------------------------------------------------------------ token rows
    uint32_t stage = 0, parity = 0;
    bool ok = true;
    for (int phase = 0; phase < 2 && ok; ++phase) {
      const uint32_t u0 = shares[phase].first(blockIdx.x), u1 = shares[phase].first(blockIdx.x + 1);
      if (u0 >= u1) continue;
      Cursor c = cursor(phase, u0);
      int seen = -1;
      for (uint32_t u = u0; u < u1; ++u, c.next()) {
        if (phase == 1 && c.chunk != seen) {                       // all of the chunk's h
          bool there = true;
          if (lane == 0) there = wait_word(p.sync + kSyncChunks + c.chunk, p.gi, abort_flag, p.wait_limit);
          ok = __all_sync(0xffffffffu, there);
          if (!ok) break;
          __syncwarp();                                            // a vote alone orders no memory
          fence_proxy_async();                                     // h was written by ordinary stores, TMA reads it
          seen = c.chunk;
        }
        ok = __all_sync(0xffffffffu, ptx::mbar_wait(ptx::smem_u32(&tail->empty[stage]), parity ^ 1u, abort_flag, p.wait_limit));
        if (!ok) break;
        const uint32_t full = ptx::smem_u32(&tail->full[stage]), dst = smem_base + stage * C::kStageBytes + kWBytes;
        const int pos = tail->chunk_start[c.chunk], n = tail->chunk_count[c.chunk];
        if (phase == 0) {
          // rows of x are gathered: a copy of one row per lane.  Rows beyond n keep what an earlier unit left; a column
          // of the product depends on its own row alone and theirs are not looked at
          if (lane == 0) ptx::mbar_arrive_expect_tx(full, static_cast<uint32_t>(n) * BK);
          __syncwarp();
          for (int r = lane; r < n; r += 32) ptx::tma_load_2d(dst + r * BK, &tmap_x, full, c.g * BK, tail->token_of_pos[pos + r]);
        } else {
          const int boxes = (n + 15) / 16;
          if (lane == 0) ptx::mbar_arrive_expect_tx(full, static_cast<uint32_t>(boxes) * 16 * BK);
          __syncwarp();
          if (lane < boxes) ptx::tma_load_2d(dst + lane * 16 * BK, &tmap_h, full, c.g * BK, pos + lane * 16);
        }
        if (++stage == C::kStages) { stage = 0; parity ^= 1u; }
      }
    }
  } else if (warp == kIssuer || warp == kIssuer + 1) {
    // ------------------------------------------------------------------ MMA issuers, one per tile
    if (lane == 0) {
      const int tile = warp - kIssuer;
      uint32_t stage = 0, parity = 0, kb = 0;
      bool ok = true;
      for (int phase = 0; phase < 2 && ok; ++phase) {
        const uint32_t u0 = shares[phase].first(blockIdx.x), u1 = shares[phase].first(blockIdx.x + 1);
        if (u0 >= u1) continue;
        Cursor c = cursor(phase, u0);
        for (uint32_t u = u0; u < u1; ++u, ++kb, c.next()) {
          const uint32_t buf = kb % kAccBufs, acc_parity = (kb / kAccBufs) & 1u;
          ok = ptx::mbar_wait(ptx::smem_u32(&tail->tmem_empty[tile][buf]), acc_parity ^ 1u, abort_flag, p.wait_limit) &&
               ptx::mbar_wait(ptx::smem_u32(&tail->full[stage]), parity, abort_flag, p.wait_limit);
          if (!ok) break;
          ptx::tc_fence_after_sync();
          const int cols = (tail->chunk_count[c.chunk] + 15) & ~15;
          const uint32_t idesc = ptx::umma_idesc_e4m3(128, cols);
          const uint32_t base = smem_base + stage * C::kStageBytes;
          const uint64_t w_desc = ptx::umma_desc_k128(base + tile * kTileBytes);
          const uint64_t x_desc = ptx::umma_desc_k128(base + kWBytes);
          const uint32_t d = tmem_base + (tile * kAccBufs + buf) * NC;
#pragma unroll
          for (int k4 = 0; k4 < BK / 32; ++k4) ptx::umma_f8(d, w_desc + 2u * k4, x_desc + 2u * k4, idesc, k4 > 0);
          ptx::umma_commit(ptx::smem_u32(&tail->empty[stage]));
          ptx::umma_commit(ptx::smem_u32(&tail->tmem_full[tile][buf]));
          if (++stage == C::kStages) { stage = 0; parity ^= 1u; }
        }
      }
    }
  } else if (warp == kScaleWarp) {
    // ------------------------------------------------------------------ scale products of the units ahead
    constexpr int kPer = (NC + 31) / 32;
    uint32_t kb = 0;
    bool ok = true;
    for (int phase = 0; phase < 2 && ok; ++phase) {
      const uint32_t u0 = shares[phase].first(blockIdx.x), u1 = shares[phase].first(blockIdx.x + 1);
      if (u0 >= u1) continue;
      int seen = -1;
      float va[kScaleAhead][kPer], vw[kScaleAhead][2];
      Cursor f = cursor(phase, u0);
      auto fetch = [&](float (&a)[kPer], float (&w)[2]) {
        const int e = tail->chunk_expert[f.chunk], pos = tail->chunk_start[f.chunk], n = tail->chunk_count[f.chunk];
        if (phase == 1 && f.chunk != seen) {
          bool there = true;
          if (lane == 0) there = wait_word(p.sync + kSyncChunks + f.chunk, p.gi, abort_flag, p.wait_limit);
          ok = ok && __all_sync(0xffffffffu, there);
          __syncwarp();
          seen = f.chunk;
        }
        if (phase == 0) {
          const float* s = p.s13 + (static_cast<int64_t>(2 * e) * p.gi + f.j) * p.gh + f.g;
          w[0] = __ldg(s);
          w[1] = __ldg(s + static_cast<int64_t>(p.gi) * p.gh);
        } else {
          const float* s = p.s2 + (static_cast<int64_t>(e) * p.gh + 2 * f.j) * p.gi + f.g;
          w[0] = __ldg(s);
          w[1] = 2 * f.j + 1 < p.gh ? __ldg(s + p.gi) : 0.0f;
        }
#pragma unroll
        for (int q = 0; q < kPer; ++q) {
          const int r = lane + 32 * q;
          a[q] = 0.0f;
          if (r < n) a[q] = phase == 0 ? __ldg(p.x_scales + static_cast<int64_t>(f.g) * p.t + tail->token_of_pos[pos + r])
                                       : __ldcg(p.h_scales + static_cast<int64_t>(f.g) * p.spad + pos + r);
        }
        f.next();
      };
#pragma unroll
      for (int i = 0; i < kScaleAhead; ++i)
        if (u0 + i < u1) fetch(va[i], vw[i]);
      for (uint32_t base = u0; base < u1 && ok; base += kScaleAhead) {
#pragma unroll
        for (int i = 0; i < kScaleAhead; ++i) {
          if (base + i < u1 && ok) {
            const uint32_t buf = kb % kAccBufs, acc_parity = (kb / kAccBufs) & 1u;
            ok = __all_sync(0xffffffffu,
                            ptx::mbar_wait(ptx::smem_u32(&tail->tmem_empty[0][buf]), acc_parity ^ 1u, abort_flag, p.wait_limit) &&
                            ptx::mbar_wait(ptx::smem_u32(&tail->tmem_empty[1][buf]), acc_parity ^ 1u, abort_flag, p.wait_limit));
            if (ok) {
#pragma unroll
              for (int q = 0; q < kPer; ++q)
                if (lane + 32 * q < NC) {
                  tail->scale[buf][0][lane + 32 * q] = va[i][q] * vw[i][0];
                  tail->scale[buf][1][lane + 32 * q] = va[i][q] * vw[i][1];
                }
              __syncwarp();
              ptx::mbar_arrive_lane0(ptx::smem_u32(&tail->tmem_full[0][buf]), lane);
              ptx::mbar_arrive_lane0(ptx::smem_u32(&tail->tmem_full[1][buf]), lane);
              if (base + i + kScaleAhead < u1) fetch(va[i], vw[i]);
              ++kb;
            }
          }
        }
      }
    }
  } else {
    // ------------------------------------------------------------------ epilogue: two groups of four warps, one per tile
    const int tile = warp >> 2;
    const int row = (warp & 3) * 32 + lane;                        // weight row inside the tile = TMEM lane
    const int tid = threadIdx.x & 127;
    const uint32_t lane_addr = static_cast<uint32_t>((warp & 3) * 32) << 16;
    float acc[NC];
#pragma unroll
    for (int j = 0; j < NC; ++j) acc[j] = 0.0f;
    uint32_t kb = 0;
    bool ok = true;
    for (int phase = 0; phase < 2; ++phase) {
      const uint32_t u0 = shares[phase].first(blockIdx.x), u1 = shares[phase].first(blockIdx.x + 1);
      if (u0 < u1) {
        Cursor c = cursor(phase, u0);
        uint32_t seg_start = u0;
        auto segment_end = [&](uint32_t u, bool alive) {
          const int pos = tail->chunk_start[c.chunk], n = tail->chunk_count[c.chunk];
          const uint32_t item_first = u - c.g;
          const int c_first = static_cast<int>(shares[phase].cta_of(item_first));
          const int c_last = static_cast<int>(shares[phase].cta_of(item_first + c.groups - 1));
          uint32_t* flags = p.sync + kSyncFlags;
          bool finish = alive;
          if (seg_start != item_first) {
            // The item's first CTA finishes it: this one hands its sums over (an item that began before this CTA's range is
            // the first thing in it, so there is one such partial per CTA and phase).  In the second phase they are added
            // behind the grid barrier, by whoever sums the token.
            float* dst = p.partials + (static_cast<int64_t>(phase * kMaxGrid + blockIdx.x) * 2 + tile) * (NC * 128) + row;
#pragma unroll
            for (int j = 0; j < NC; ++j)
              if (j < n) __stcg(dst + j * 128, acc[j]);
            if (phase == 0) {
              named_sync(1 + tile, 128);
              if (tid == 0) red_release_add(flags + blockIdx.x * 2 + tile);
            }
            finish = false;
          } else if (phase == 0 && c_last != c_first) {
            // Its own part is the last thing in its range; the others' partials are added in the order of the K range,
            // whatever the timing.  One thread waits for each of the others.
            if (tid == 0) tail->flag[tile] = 1u;
            named_sync(1 + tile, 128);
            for (int o = c_first + 1 + tid; o <= c_last; o += 128)
              if (!wait_word(flags + o * 2 + tile, 1u, abort_flag, p.wait_limit)) tail->flag[tile] = 0u;
            named_sync(1 + tile, 128);
            const bool there = tail->flag[tile] != 0;
            finish = finish && there;
            if (there) {
              const int64_t pitch = 2 * NC * 128;
              const float* src = p.partials + (static_cast<int64_t>(c_first + 1) * 2 + tile) * (NC * 128) + row;
              for (int o = c_last - c_first; o > 0; o -= 4, src += 4 * pitch) {
                // four CTAs' sums of four columns on their way at a time
#pragma unroll
                for (int j0 = 0; j0 < NC; j0 += 4) {
                  if (j0 < n) {
                    float v[4][4];
#pragma unroll
                    for (int w = 0; w < 4; ++w)
#pragma unroll
                      for (int j = 0; j < 4; ++j) v[w][j] = w < o && j0 + j < n ? __ldcg(src + w * pitch + (j0 + j) * 128) : 0.0f;
#pragma unroll
                    for (int w = 0; w < 4; ++w)
#pragma unroll
                      for (int j = 0; j < 4; ++j) acc[j0 + j] += v[w][j];
                  }
                }
              }
            }
          }
          if (seg_start == item_first) {
            if (phase == 0) {
              // SwiGLU and the quantizer of h, 16 columns at a time: each side finishes eight of them, with the other
              // side's factor from shared memory; 128 outputs of a column are one quantization group
              const int col = c.j * 128 + row;
#pragma unroll
              for (int q = 0; q < NC / 16; ++q) {
                if (q * 16 < n) {
#pragma unroll
                  for (int j = 0; j < 8; ++j)
                    tail->ex.value[1 - tile][j][row] = tile == 0 ? acc[q * 16 + 8 + j] : acc[q * 16 + j];
                  named_sync(3, 256);
                  float v[8];
#pragma unroll
                  for (int j = 0; j < 8; ++j) {
                    if (q * 16 + tile * 8 + j >= n) { v[j] = 0.0f; continue; }
                    const float other = tail->ex.value[tile][j][row], own = tile == 0 ? acc[q * 16 + j] : acc[q * 16 + 8 + j];
                    v[j] = col < p.i ? (tile == 0 ? silu_mul(own, other) : silu_mul(other, own)) : 0.0f;
                    const uint32_t most = __reduce_max_sync(0xffffffffu, __float_as_uint(v[j]) & 0x7fffffffu);
                    if (lane == 0) tail->ex.most[warp][j] = __uint_as_float(most);
                  }
                  named_sync(1 + tile, 128);
#pragma unroll
                  for (int j = 0; j < 8; ++j) {
                    const int place = q * 16 + tile * 8 + j;
                    if (place >= n) continue;
                    uint32_t bits = 0u;                            // as integers: a NaN is the largest
#pragma unroll
                    for (int w = 0; w < 4; ++w) bits = max(bits, __float_as_uint(tail->ex.most[tile * 4 + w][j]));
                    const float scale = group_scale(bits);
                    const float rcp = __frcp_rn(scale);
                    const uint32_t code = p.half ? quant_half_e4m3x2(v[j], 0.0f, scale, rcp) : quant_e4m3x2(v[j], 0.0f, scale, rcp);
                    if (finish) {
                      if (col < p.i) p.hq[static_cast<int64_t>(pos + place) * p.i + col] = static_cast<uint8_t>(code);
                      if (row == 0) p.h_scales[static_cast<int64_t>(c.j) * p.spad + pos + place] = p.half ? scale * 2.0f : scale;
                    }
                  }
                  named_sync(3, 256);
                }
              }
              fence_proxy_async();
              named_sync(3, 256);
              if (threadIdx.x == 0) red_release_add(p.sync + kSyncChunks + c.chunk);
            } else if (finish) {
              const int col = c.j * 256 + tile * 128 + row;
              if (col < p.h) {
                float* dst = p.y + static_cast<int64_t>(pos) * p.h + col;
#pragma unroll
                for (int j = 0; j < NC; ++j)
                  if (j < n) __stcg(dst + static_cast<int64_t>(j) * p.h, acc[j]);
              }
            }
          }
#pragma unroll
          for (int j = 0; j < NC; ++j) acc[j] = 0.0f;
          seg_start = u + 1;
        };
        uint32_t u = u0;
        for (; u < u1; ++u, ++kb) {
          const uint32_t buf = kb % kAccBufs, acc_parity = (kb / kAccBufs) & 1u;
          ok = ok && __all_sync(0xffffffffu, ptx::mbar_wait(ptx::smem_u32(&tail->tmem_full[tile][buf]), acc_parity, abort_flag, p.wait_limit));
          if (!ok) break;
          ptx::tc_fence_after_sync();
          const int n = tail->chunk_count[c.chunk];
          const uint32_t taddr = tmem_base + lane_addr + (tile * kAccBufs + buf) * NC;
#pragma unroll
          for (int q = 0; q < NC / 16; ++q) {
            if (q * 16 < n) {
              uint32_t r[16];
              ptx::tmem_ld16(taddr + q * 16, r);
              float s[16];
#pragma unroll
              for (int j = 0; j < 16; j += 4) {
                const float4 t4 = *reinterpret_cast<const float4*>(&tail->scale[buf][tile][q * 16 + j]);
                s[j] = t4.x; s[j + 1] = t4.y; s[j + 2] = t4.z; s[j + 3] = t4.w;
              }
              ptx::tmem_wait_ld16(r);
#pragma unroll
              for (int j = 0; j < 16; ++j) acc[q * 16 + j] = fmaf(__uint_as_float(r[j]), s[j], acc[q * 16 + j]);
            }
          }
          ptx::tc_fence_before_sync();
          __syncwarp();
          ptx::mbar_arrive_lane0(ptx::smem_u32(&tail->tmem_empty[tile][buf]), lane);
          if (c.g == c.groups - 1 || u == u1 - 1) segment_end(u, true);
          c.next();
        }
        // a thread that gave up keeps every appointment with the other group and the other CTAs
        for (; u < u1; ++u) {
          if (c.g == c.groups - 1 || u == u1 - 1) segment_end(u, false);
          c.next();
        }
      }
    }
    // ---- grid barrier: everything this half of the CTA wrote is visible
    named_sync(1 + tile, 128);
    if (tid == 0) red_release_add(p.sync + kSyncBarrier);
    // ---- weighted sum over each token's slots, the columns spread over all warps of the grid
    if (tid == 0) tail->flag[tile] = wait_word(p.sync + kSyncBarrier, barrier_count, abort_flag, p.wait_limit) ? 1u : 0u;
    named_sync(1 + tile, 128);
    if (tail->flag[tile] != 0) {
      const int per_token = (p.h + 127) / 128;                     // a warp takes 128 columns of a token
      for (uint32_t w = warp * gridDim.x + blockIdx.x; w < static_cast<uint32_t>(p.t) * per_token; w += 8u * gridDim.x) {
        const int t = static_cast<int>(w / per_token), block = static_cast<int>(w % per_token), col = block * 128 + lane * 4;
        // lane j looks up slot j: where its sum lies, and how many more CTAs hold parts of its K range
        int more = -1;
        const float *own = nullptr, *parts = nullptr;
        float weight = 0.0f;
        if (lane < p.k) {
          const int place = tail->place_of_slot[t * p.k + lane];
          if (place != 0xffff) {
            const int chunk = place >> 6, column = place & 63;
            const uint32_t u = (static_cast<uint32_t>(chunk) * p.hpairs + (block >> 1)) * p.gi;
            const int first = static_cast<int>(shares[1].cta_of(u));
            more = static_cast<int>(shares[1].cta_of(u + p.gi - 1)) - first;
            own = p.y + static_cast<int64_t>(tail->chunk_start[chunk] + column) * p.h + block * 128;
            parts = p.partials + ((static_cast<int64_t>(kMaxGrid + first + 1) * 2 + (block & 1)) * NC + column) * 128;
            weight = __ldcg(p.weights + t * p.k + lane);
          }
        }
        const int deepest = __reduce_max_sync(0xffffffffu, more);
        float4 sum = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        for (int j0 = 0; j0 < p.k; j0 += 4) {                      // four slots' loads on their way at a time
          float4 v[4];
          const float* at[4];
          int n[4];
          float wt[4];
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const int from = min(j0 + j, 31);
            const unsigned long long a = __shfl_sync(0xffffffffu, reinterpret_cast<unsigned long long>(own), from);
            at[j] = reinterpret_cast<const float*>(__shfl_sync(0xffffffffu, reinterpret_cast<unsigned long long>(parts), from));
            n[j] = __shfl_sync(0xffffffffu, more, from);
            wt[j] = __shfl_sync(0xffffffffu, weight, from);
            if (j0 + j >= p.k || col >= p.h) n[j] = -1;
            v[j] = n[j] >= 0 ? __ldcg(reinterpret_cast<const float4*>(reinterpret_cast<const float*>(a) + lane * 4))
                             : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
          }
          for (int o = 0; o < deepest; o += 3) {
            float4 a[3][4];
#pragma unroll
            for (int i = 0; i < 3; ++i)
#pragma unroll
              for (int j = 0; j < 4; ++j)
                a[i][j] = o + i < n[j] ? __ldcg(reinterpret_cast<const float4*>(at[j] + static_cast<int64_t>(o + i) * (2 * NC * 128) + lane * 4))
                                       : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
            for (int i = 0; i < 3; ++i)
#pragma unroll
              for (int j = 0; j < 4; ++j) { v[j].x += a[i][j].x; v[j].y += a[i][j].y; v[j].z += a[i][j].z; v[j].w += a[i][j].w; }
          }
#pragma unroll
          for (int j = 0; j < 4; ++j)
            if (n[j] >= 0) {
              sum.x = fmaf(wt[j], v[j].x, sum.x); sum.y = fmaf(wt[j], v[j].y, sum.y);
              sum.z = fmaf(wt[j], v[j].z, sum.z); sum.w = fmaf(wt[j], v[j].w, sum.w);
            }
        }
        if (col < p.h)
          *reinterpret_cast<uint2*>(p.out + t * p.ldo + col) = make_uint2(pack_bf16x2(sum.x, sum.y), pack_bf16x2(sum.z, sum.w));
      }
    }
  }

  // ------------------------------------------------------------------ teardown
  ptx::tc_fence_before_sync();
  __syncthreads();
  ptx::tc_fence_after_sync();
  ptx::idle_after_abort(abort_flag);
  if (warp == kIssuer) ptx::tmem_dealloc(tmem_base, C::kTmemCols);
  if (threadIdx.x == 0 && tail->abort_flag != 0) atomicOr(p.status, BFP8_STATUS_WAIT_TIMEOUT);
}

// Layout of the workspace
struct Layout {
  size_t sync, x_codes, x_scales, scores, hq, h_scales, partials, y, bytes;
  int spad;
};
Layout layout_of(int64_t t, int64_t k, int64_t e, int64_t h, int64_t i) {
  Layout l;
  size_t at = 0;
  auto take = [&](size_t n) { const size_t a = at; at += (n + 255) & ~static_cast<size_t>(255); return a; };
  const int64_t slots = t * k;
  l.spad = static_cast<int>((slots + 15) / 16 * 16);
  l.sync = take(kSyncWords * 4);
  l.x_codes = take(static_cast<size_t>(t) * h);
  l.x_scales = take(static_cast<size_t>((h + 127) / 128) * t * 4);
  l.scores = take(static_cast<size_t>(t) * e * 4);
  l.hq = take(static_cast<size_t>(l.spad) * i);
  l.h_scales = take(static_cast<size_t>((i + 127) / 128) * l.spad * 4);
  l.partials = take(static_cast<size_t>(kMaxGrid) * 2 * 2 * (t <= 16 ? 16 : 64) * 128 * 4);
  l.y = take(static_cast<size_t>(slots) * h * 4);
  l.bytes = at;
  return l;
}

template <int NC>
int launch_experts(const CUtensorMap& w13, const CUtensorMap& w2, const CUtensorMap& x, const CUtensorMap& hm, const ExpertParams& p,
                   int max_ctas, cudaStream_t st) {
  using C = Cfg<NC>;
  constexpr int smem = 1024 + C::kStages * C::kStageBytes + static_cast<int>(sizeof(Tail));
  static_assert(smem <= 227 * 1024, "shared memory of one SM");
  static DeviceFlags done;
  const int rc = ensure_smem_limit(moe_experts_kernel<NC>, smem, done);
  if (rc != BFP8_OK) return rc;
  int grid = sm_count();
  if (grid > kMaxGrid) grid = kMaxGrid;
  if (max_ctas > 0 && max_ctas < grid) grid = max_ctas;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(grid), 1, 1);
  cfg.blockDim = dim3(kThreads, 1, 1);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  // the CTAs wait for one another: the launch has to put all of them on the device together
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeCooperative;
  attr[0].val.cooperative = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  BFP8_CUDA_TRY(cudaLaunchKernelEx(&cfg, moe_experts_kernel<NC>, w13, w2, x, hm, p));
  return BFP8_OK;
}

struct Router {
  const uint16_t* weight;
  int64_t ld;
  RouteRule rule;
  int sigmoid;
};

int moe_layer(const uint16_t* x, int64_t ldx, const Router* router, const int32_t* ids, const float* weights, int32_t* ids_out,
              float* weights_out, const uint8_t* w13, const float* s13, const uint8_t* w2, const float* s2, uint16_t* out,
              int64_t ldo, int64_t t, int64_t k, int64_t e, int64_t h, int64_t i, int native_half, void* workspace,
              size_t workspace_bytes, uint32_t* status_dev, void* stream, int max_ctas, int64_t wait_limit_cycles) {
  if (!x || !w13 || !s13 || !w2 || !s2 || !out || !status_dev || !workspace) return BFP8_ERR_NULL;
  if (router ? !router->weight : (!ids || !weights)) return BFP8_ERR_NULL;
  if (!router && (!aligned(ids, 4) || !aligned(weights, 4))) return BFP8_ERR_ALIGN;
  if (t <= 0 || k <= 0 || e <= 0 || h <= 0 || i <= 0 || h > kMaxWidth || i > kMaxWidth || ldx < h || ldo < h) return BFP8_ERR_SHAPE;
  if (t > kMaxTokens || k > kMaxTopK || e > kMaxExperts || t * k > kMaxSlots || h % 16 != 0 || i % 16 != 0)
    return BFP8_ERR_UNSUPPORTED;
  if (router && (k > e || router->ld < h)) return BFP8_ERR_SHAPE;
  if (!aligned(x, 2) || !aligned(w13, 16) || !aligned(w2, 16) || !aligned(s13, 4) || !aligned(s2, 4) || !aligned(status_dev, 4) ||
      !aligned(out, 8) || ldo % 4 != 0 || !aligned(workspace, 256))
    return BFP8_ERR_ALIGN;
  const Layout l = layout_of(t, k, e, h, i);
  if (workspace_bytes < l.bytes) return BFP8_ERR_WORKSPACE;
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  cudaStream_t st = static_cast<cudaStream_t>(stream);

  FrontParams f = {};
  f.x = x;
  f.ldx = ldx;
  f.t = t;
  f.h = static_cast<int>(h);
  f.vec = aligned(x, 16) && ldx % 8 == 0;
  f.quant_blocks = 1;
  f.groups = static_cast<int>((h + 127) / 128);
  f.half = native_half != 0;
  f.codes = ws + l.x_codes;
  f.scales = reinterpret_cast<float*>(ws + l.x_scales);
  f.sync = reinterpret_cast<uint32_t*>(ws + l.sync);
  if (router) {
    f.vec = f.vec && aligned(router->weight, 16) && router->ld % 8 == 0;
    f.router = router->weight;
    f.ldr = router->ld;
    f.experts = static_cast<int>(e);
    f.sigmoid = router->sigmoid;
    f.scores = reinterpret_cast<float*>(ws + l.scores);
  }

  ExpertParams p = {};
  p.x_scales = f.scales;
  p.scores = f.scores;
  if (router) {
    p.rule = router->rule;
    p.ids_out = ids_out;
    p.weights = weights_out;
  } else {
    p.ids = ids;
    p.weights = const_cast<float*>(weights);
  }
  p.s13 = s13;
  p.s2 = s2;
  p.hq = ws + l.hq;
  p.h_scales = reinterpret_cast<float*>(ws + l.h_scales);
  p.partials = reinterpret_cast<float*>(ws + l.partials);
  p.y = reinterpret_cast<float*>(ws + l.y);
  p.sync = f.sync;
  p.out = out;
  p.ldo = ldo;
  p.t = static_cast<int>(t);
  p.k = static_cast<int>(k);
  p.experts = static_cast<int>(e);
  p.h = static_cast<int>(h);
  p.i = static_cast<int>(i);
  p.gh = static_cast<int>((h + 127) / 128);
  p.gi = static_cast<int>((i + 127) / 128);
  p.hpairs = static_cast<int>((h + 255) / 256);
  p.spad = l.spad;
  p.half = f.half;
  p.wait_limit = wait_limit_cycles > 0 ? wait_limit_cycles : kDefaultWaitLimit;
  p.status = status_dev;

  alignas(64) CUtensorMap m13, m2, mx, mh;
  int rc = make_tensor_map_3d(&m13, CU_TENSOR_MAP_DATA_TYPE_UINT8, w13, h, i, 2 * e, BK, 128);
  if (rc == BFP8_OK) rc = make_tensor_map_3d(&m2, CU_TENSOR_MAP_DATA_TYPE_UINT8, w2, i, h, e, BK, 128);
  if (rc == BFP8_OK) rc = make_tensor_map_2d(&mx, CU_TENSOR_MAP_DATA_TYPE_UINT8, f.codes, h, t, h, BK, 1);
  if (rc == BFP8_OK) rc = make_tensor_map_2d(&mh, CU_TENSOR_MAP_DATA_TYPE_UINT8, p.hq, i, l.spad, i, BK, 16);
  if (rc != BFP8_OK) return rc;
  rc = launch_front(f, st);
  if (rc != BFP8_OK) return rc;
  return t <= 16 ? launch_experts<16>(m13, m2, mx, mh, p, max_ctas, st) : launch_experts<64>(m13, m2, mx, mh, p, max_ctas, st);
}

}  // namespace
}  // namespace bfp8

using namespace bfp8;

extern "C" size_t bfp8_moe_route_workspace_bytes(int64_t t, int64_t experts) {
  return t > 0 && experts > 0 ? static_cast<size_t>(t) * experts * sizeof(float) : 0;
}

extern "C" int bfp8_moe_route(const uint16_t* x, int64_t ldx, const uint16_t* router, int64_t ld_router, const float* bias,
                              int64_t t, int64_t h, int64_t experts, int64_t top_k, int scoring, int renormalize, float scale,
                              int32_t* ids, float* weights, void* workspace, size_t workspace_bytes, void* stream) {
  if (!x || !router || !ids || !weights || !workspace) return BFP8_ERR_NULL;
  if (t <= 0 || h <= 0 || experts <= 0 || top_k <= 0 || top_k > experts || ldx < h || ld_router < h || h > (1 << 20))
    return BFP8_ERR_SHAPE;
  if (scoring != BFP8_ROUTE_SOFTMAX && scoring != BFP8_ROUTE_SIGMOID) return BFP8_ERR_SHAPE;
  if (top_k > kMaxTopK || experts > kMaxExperts || (bias && scoring == BFP8_ROUTE_SOFTMAX)) return BFP8_ERR_UNSUPPORTED;
  if (!aligned(x, 2) || !aligned(router, 2) || (bias && !aligned(bias, 4)) || !aligned(ids, 4) || !aligned(weights, 4) ||
      !aligned(workspace, 4))
    return BFP8_ERR_ALIGN;
  if (workspace_bytes < bfp8_moe_route_workspace_bytes(t, experts)) return BFP8_ERR_WORKSPACE;
  if ((t + 3) / 4 > 2147483647LL) return BFP8_ERR_SHAPE;
  FrontParams f = {};
  f.x = x;
  f.ldx = ldx;
  f.t = t;
  f.h = static_cast<int>(h);
  f.vec = aligned(x, 16) && ldx % 8 == 0 && aligned(router, 16) && ld_router % 8 == 0 && h % 8 == 0;
  f.router = router;
  f.ldr = ld_router;
  f.experts = static_cast<int>(experts);
  f.sigmoid = scoring == BFP8_ROUTE_SIGMOID;
  f.scores = static_cast<float*>(workspace);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const int rc = launch_front(f, st);
  if (rc != BFP8_OK) return rc;
  const RouteRule rule = {bias, scoring == BFP8_ROUTE_SOFTMAX, renormalize != 0, scale};
  return launch_overlapped(moe_topk_kernel, dim3(static_cast<unsigned>((t + 3) / 4)), dim3(128), 0, st, f.scores, t,
                           static_cast<int>(experts), static_cast<int>(top_k), rule, ids, weights);
}

extern "C" size_t bfp8_moe_block128_workspace_bytes(int64_t t, int64_t top_k, int64_t experts, int64_t h, int64_t inter) {
  if (t <= 0 || top_k <= 0 || experts <= 0 || h <= 0 || inter <= 0 || t > kMaxTokens || t * top_k > kMaxSlots ||
      experts > kMaxExperts || h > kMaxWidth || inter > kMaxWidth)
    return 0;
  return layout_of(t, top_k, experts, h, inter).bytes;
}

extern "C" int bfp8_moe_block128(const uint16_t* x, int64_t ldx, const int32_t* ids, const float* weights,
                                 const uint8_t* w_gate_up, const float* s_gate_up, const uint8_t* w_down, const float* s_down,
                                 uint16_t* out, int64_t ldo, int64_t t, int64_t top_k, int64_t experts, int64_t h, int64_t inter,
                                 int native_half, void* workspace, size_t workspace_bytes, uint32_t* status_dev, void* stream,
                                 int max_ctas, int64_t wait_limit_cycles) {
  return moe_layer(x, ldx, nullptr, ids, weights, nullptr, nullptr, w_gate_up, s_gate_up, w_down, s_down, out, ldo, t, top_k,
                   experts, h, inter, native_half, workspace, workspace_bytes, status_dev, stream, max_ctas, wait_limit_cycles);
}

extern "C" int bfp8_moe_layer_block128_ex(const uint16_t* x, int64_t ldx, const uint16_t* router, int64_t ld_router,
                                          const float* bias, int scoring, int renormalize, float scale, int32_t* ids,
                                          float* weights, const uint8_t* w_gate_up, const float* s_gate_up, const uint8_t* w_down,
                                          const float* s_down, uint16_t* out, int64_t ldo, int64_t t, int64_t top_k,
                                          int64_t experts, int64_t h, int64_t inter, int native_half, void* workspace,
                                          size_t workspace_bytes, uint32_t* status_dev, void* stream, int max_ctas,
                                          int64_t wait_limit_cycles) {
  if (!router || !ids || !weights) return BFP8_ERR_NULL;
  if (scoring != BFP8_ROUTE_SOFTMAX && scoring != BFP8_ROUTE_SIGMOID) return BFP8_ERR_SHAPE;
  if (bias && scoring == BFP8_ROUTE_SOFTMAX) return BFP8_ERR_UNSUPPORTED;
  if (!aligned(router, 2) || (bias && !aligned(bias, 4)) || !aligned(ids, 4) || !aligned(weights, 4)) return BFP8_ERR_ALIGN;
  const Router r = {router, ld_router, {bias, scoring == BFP8_ROUTE_SOFTMAX, renormalize != 0, scale}, scoring == BFP8_ROUTE_SIGMOID};
  return moe_layer(x, ldx, &r, nullptr, nullptr, ids, weights, w_gate_up, s_gate_up, w_down, s_down, out, ldo, t, top_k, experts,
                   h, inter, native_half, workspace, workspace_bytes, status_dev, stream, max_ctas, wait_limit_cycles);
}

extern "C" int bfp8_moe_layer_block128(const uint16_t* x, int64_t ldx, const uint16_t* router, int64_t ld_router, const float* bias,
                                       int scoring, int renormalize, float scale, int32_t* ids, float* weights,
                                       const uint8_t* w_gate_up, const float* s_gate_up, const uint8_t* w_down,
                                       const float* s_down, uint16_t* out, int64_t ldo, int64_t t, int64_t top_k,
                                       int64_t experts, int64_t h, int64_t inter, int native_half, void* workspace,
                                       size_t workspace_bytes, uint32_t* status_dev, void* stream) {
  return bfp8_moe_layer_block128_ex(x, ldx, router, ld_router, bias, scoring, renormalize, scale, ids, weights, w_gate_up, s_gate_up,
                                    w_down, s_down, out, ldo, t, top_k, experts, h, inter, native_half, workspace, workspace_bytes,
                                    status_dev, stream, 0, 0);
}
