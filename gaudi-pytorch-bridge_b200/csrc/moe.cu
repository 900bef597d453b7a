// A mixture-of-experts layer for a few tokens: router, choice of the experts, their gated products, and the weighted sum.
#include <type_traits>

#include "layer.cuh"
#include "tcgen05_ptx.cuh"
#include "tma_host.cuh"

namespace b200q {

constexpr int64_t kMoeChunk = 256;  // tokens taken at a time
constexpr size_t moe_align(size_t n) { return (n + 255) / 256 * 256; }

// Where the parts of the workspace lie.
struct MoeSpace {
  size_t logits, x_top, control, h_top, hidden, outputs, x_terms, h_terms, parts, bytes;
  int clear_words;  // from control on
  MoeSpace(int64_t tokens, int64_t h, int64_t f, int experts, int top_k);
};

// Tokens to route of those that `a` stands for, which are the call's from `first` on.
__device__ __forceinline__ int moe_tokens(const b200q_moe_args& a, int64_t first) {
  return a.num_tokens ? (int)min(max((int64_t)*a.num_tokens - first, (int64_t)0), a.tokens) : (int)a.tokens;
}
__device__ __forceinline__ float moe_weight(const void* p, int dtype, int64_t at) {
  return dtype == B200Q_BF16 ? __bfloat162float(static_cast<const __nv_bfloat16*>(p)[at]) : fp8_to_float<B200Q_E4M3>(static_cast<const uint8_t*>(p)[at]);
}
__device__ __forceinline__ float moe_x(const b200q_moe_args& a, int64_t t, int64_t i) {
  return __bfloat162float(static_cast<const __nv_bfloat16*>(a.x)[t * a.x_stride + i]);
}
__device__ __forceinline__ float moe_silu(float g) { return g / (1.f + expf(-g)); }
// An infinite value of h has no terms (e4m3 has no infinity, and inf - inf is no rest): NaN in all kernels, so that layouts do not differ.
__device__ __forceinline__ float moe_finite(float h) { return fabsf(h) <= 3.402823466e38f ? h : __int_as_float(0x7FC00000); }

// ---------------------------------------------------------------------------- router
// Sums in fp64: neighbours in the order of the experts may be closer than the rounding of a sum in fp32, and another expert is another answer.
constexpr int kMoeThreads = 256;

// The power of two that brings a largest value (its bits) to [128, 256), and its inverse.
__device__ __forceinline__ float moe_up_factor(uint32_t top) {
  const int e = (int)(top >> 23) - 127;
  const int up = e == 128 ? 0 : max(-126, min(7 - e, 126));
  return __uint_as_float((uint32_t)(127 + up) << 23);
}
__device__ __forceinline__ float moe_down_factor(uint32_t top) {
  const int e = (int)(top >> 23) - 127;
  const int up = e == 128 ? 0 : max(-126, min(7 - e, 126));
  return __uint_as_float((uint32_t)(127 - up) << 23);
}

// Eight values in TERMS terms of e4m3, each the rounded rest of the one before times 32 (a rest is at most 8 where the largest value is below 256).
template <int TERMS>
__device__ __forceinline__ void moe_terms_fp8(float (&v)[8], uint2 (&out)[TERMS]) {
#pragma unroll
  for (int t = 0; t < TERMS; ++t) {
    uint32_t w[2] = {0, 0};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t pair = cvt_fp8x2<B200Q_E4M3>(v[2 * i], v[2 * i + 1]);
      w[i / 2] |= pair << (16 * (i & 1));
      if (t + 1 < TERMS) {
        v[2 * i] = (v[2 * i] - fp8_to_float<B200Q_E4M3>(pair & 0xFFu)) * 32.f;
        v[2 * i + 1] = (v[2 * i + 1] - fp8_to_float<B200Q_E4M3>(pair >> 8)) * 32.f;
      }
    }
    out[t] = make_uint2(w[0], w[1]);
  }
}

template <typename W>
__device__ __forceinline__ void moe_load8(const W* p, bool wide, int64_t i, int64_t n, float (&v)[8]) {
  if (wide) {
    if (sizeof(W) == 2) {
      const uint4 u = __ldg(reinterpret_cast<const uint4*>(p + i));
      const uint32_t x[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        v[2 * c] = __uint_as_float(x[c] << 16);
        v[2 * c + 1] = __uint_as_float(x[c] & 0xFFFF0000u);
      }
    } else {
      const float4 x = __ldg(reinterpret_cast<const float4*>(p + i)), y = __ldg(reinterpret_cast<const float4*>(p + i) + 1);
      v[0] = x.x; v[1] = x.y; v[2] = x.z; v[3] = x.w;
      v[4] = y.x; v[5] = y.y; v[6] = y.z; v[7] = y.w;
    }
  } else {
#pragma unroll
    for (int c = 0; c < 8; ++c) v[c] = i + c < n ? (float)p[i + c] : 0.f;
  }
}

// A block has EB experts' rows and TB tokens', its warps an eighth of the row each: all of a warp's loads of a row of 4096 are then in flight at once.  What the
// fused kernel wants cleared, and the tokens' largest values, come from here too.
template <typename W, int EB, int TB>
__global__ void __launch_bounds__(kMoeThreads) moe_logits_kernel(const b200q_moe_args a, int64_t first, double* logits, uint32_t* x_top, uint8_t* x_terms, uint32_t* clear, int clear_words, bool wide) {
  constexpr int kWarps = kMoeThreads / 32;
  __shared__ double s_sum[kWarps][EB * TB];
  __shared__ uint32_t s_top[kWarps][TB];
  pdl_enter();
  for (int i = blockIdx.x * kMoeThreads + threadIdx.x; i < clear_words; i += gridDim.x * kMoeThreads) clear[i] = 0;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, tokens = moe_tokens(a, first);
  const int64_t expert_blocks = (a.experts + EB - 1) / EB;
  const int64_t t0 = blockIdx.x / expert_blocks * TB, e0 = (blockIdx.x % expert_blocks) * EB;
  if (t0 >= tokens) return;
  const W* router[EB];
  const __nv_bfloat16* x[TB];
#pragma unroll
  for (int e = 0; e < EB; ++e) router[e] = static_cast<const W*>(a.router) + min(e0 + e, (int64_t)a.experts - 1) * a.hidden;
#pragma unroll
  for (int t = 0; t < TB; ++t) x[t] = static_cast<const __nv_bfloat16*>(a.x) + min(t0 + t, (int64_t)tokens - 1) * a.x_stride;
  double sum[EB * TB] = {};
  uint32_t top[TB] = {};
#pragma unroll 2
  for (int64_t i = 8 * threadIdx.x; i < a.hidden; i += 8 * kMoeThreads) {
    float xv[TB][8], wv[EB][8];
#pragma unroll
    for (int t = 0; t < TB; ++t) moe_load8(x[t], wide, i, a.hidden, xv[t]);
#pragma unroll
    for (int e = 0; e < EB; ++e) moe_load8(router[e], wide, i, a.hidden, wv[e]);
#pragma unroll
    for (int c = 0; c < 8; ++c) {
      double xd[TB];
#pragma unroll
      for (int t = 0; t < TB; ++t) {
        xd[t] = (double)xv[t][c];
        top[t] = max(top[t], __float_as_uint(xv[t][c]) & 0x7FFFFFFFu);
      }
#pragma unroll
      for (int e = 0; e < EB; ++e) {
        const double wd = (double)wv[e][c];
#pragma unroll
        for (int t = 0; t < TB; ++t) sum[e * TB + t] += wd * xd[t];
      }
    }
  }
#pragma unroll
  for (int i = 0; i < EB * TB; ++i) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum[i] += __shfl_xor_sync(0xFFFFFFFFu, sum[i], o);
    if (lane == 0) s_sum[warp][i] = sum[i];
  }
#pragma unroll
  for (int t = 0; t < TB; ++t) {
    top[t] = __reduce_max_sync(0xFFFFFFFFu, top[t]);
    if (lane == 0) s_top[warp][t] = top[t];
  }
  __syncthreads();
  if (threadIdx.x < EB * TB) {
    const int e = threadIdx.x / TB, t = threadIdx.x % TB;
    double all = 0.0;
#pragma unroll
    for (int i = 0; i < kWarps; ++i) all += s_sum[i][threadIdx.x];
    if (t0 + t < tokens && e0 + e < a.experts) logits[(t0 + t) * a.experts + e0 + e] = all;
    if (e0 == 0 && e == 0 && t0 + t < tokens) {
      uint32_t most = 0;
#pragma unroll
      for (int i = 0; i < kWarps; ++i) most = max(most, s_top[i][t]);
      x_top[t0 + t] = most;
    }
  }
  if (!x_terms) return;
  // the tokens' two terms for 8-bit weights, a token by each of the blocks that have it
#pragma unroll 1
  for (int64_t t = e0 / EB; t < TB && t0 + t < tokens; t += expert_blocks) {
    uint32_t most = 0;
    for (int i = 0; i < kWarps; ++i) most = max(most, s_top[i][t]);
    const float factor = moe_up_factor(most);
    const __nv_bfloat16* row = static_cast<const __nv_bfloat16*>(a.x) + (t0 + t) * a.x_stride;
    for (int64_t i = 8 * threadIdx.x; i < a.hidden; i += 8 * kMoeThreads) {
      float v[8];
      moe_load8(row, true, i, a.hidden, v);
#pragma unroll
      for (int c = 0; c < 8; ++c) v[c] *= factor;
      uint2 term[2];
      moe_terms_fp8<2>(v, term);
#pragma unroll
      for (int c = 0; c < 2; ++c) *reinterpret_cast<uint2*>(x_terms + (c * a.tokens + t0 + t) * a.hidden + i) = term[c];
    }
  }
}

// A logit as an integer that is ordered as the choice is: a NaN above all; the two zeros are one.  0 is below every logit.
__device__ __forceinline__ unsigned long long moe_key(double v) {
  if (v != v) return ~0ull;
  const long long b = __double_as_longlong(v + 0.0);  // (-0 + 0 = 0)
  return (unsigned long long)b ^ (b < 0 ? ~0ull : 1ull << 63);
}
__device__ __forceinline__ double moe_value(unsigned long long key) {
  return key == ~0ull ? __longlong_as_double(~0ll) : __longlong_as_double((long long)(key ^ (key >> 63 ? 1ull << 63 : ~0ull)));
}

// The choice for one token by one warp: lane j has the j-th expert.  A lane has each 32nd logit and knows the best of those it has left, so that a
// round is a maximum over the lanes in three steps of 32 bits: upper half of the key, lower half, lowest index.
struct MoeChoice {
  int id;
  float weight;
};
template <int MINE>
__device__ __forceinline__ MoeChoice moe_choose_of(const b200q_moe_args& a, const double* logits, int lane) {
  MoeChoice c = {-1, 0.f};
  double mine[MINE];
#pragma unroll
  for (int i = 0; i < MINE; ++i) mine[i] = lane + 32 * i < a.experts ? __ldcg(logits + lane + 32 * i) : 0.0;
  unsigned long long key[MINE];  // 0: taken, or behind the last expert
#pragma unroll
  for (int i = 0; i < MINE; ++i) key[i] = lane + 32 * i < a.experts ? moe_key(mine[i]) : 0;
  unsigned long long best, first = 0, value = 0;
  int at;
  auto look = [&] {
    best = key[0];
    at = lane;
#pragma unroll
    for (int i = 1; i < MINE; ++i)
      if (key[i] > best) {
        best = key[i];
        at = lane + 32 * i;
      }
  };
  look();
  for (int j = 0; j < a.top_k; ++j) {
    const uint32_t hi = (uint32_t)(best >> 32), hi_most = __reduce_max_sync(0xFFFFFFFFu, hi);
    const uint32_t lo = hi == hi_most ? (uint32_t)best : 0u, lo_most = __reduce_max_sync(0xFFFFFFFFu, lo);
    const int id = (int)__reduce_min_sync(0xFFFFFFFFu, hi == hi_most && (uint32_t)best == lo_most ? (uint32_t)at : 0x7FFFu);
    const unsigned long long most = (unsigned long long)hi_most << 32 | lo_most;
    if (j == 0) first = most;
    if (lane == j) {
      c.id = id;
      value = most;
    }
    if (id == at) {
#pragma unroll
      for (int i = 0; i < MINE; ++i)
        if (id >> 5 == i) key[i] = 0;
      look();
    }
  }
  // exponents are differences taken in fp64, and small ones exact enough in fp32
  const double top = moe_value(first);
  const float p = lane < a.top_k ? expf((float)(moe_value(value) - top)) : 0.f;
  float sum = 0.f;
  if (a.renormalize) {
    sum = p;
  } else {
#pragma unroll
    for (int i = 0; i < MINE; ++i)
      if (lane + 32 * i < a.experts) sum += expf((float)(mine[i] - top));
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xFFFFFFFFu, sum, o);
  c.weight = p / sum;
  return c;
}
__device__ __forceinline__ MoeChoice moe_choose(const b200q_moe_args& a, const double* logits, bool live, int lane) {
  if (!live) return {-1, 0.f};
  return a.experts <= 128 ? moe_choose_of<4>(a, logits, lane) : moe_choose_of<kMoeMaxExperts / 32>(a, logits, lane);
}
__device__ __forceinline__ void moe_store_choice(const b200q_moe_args& a, int64_t t, int lane, const MoeChoice& c) {
  a.ids[t * a.top_k + lane] = c.id;
  a.weights[t * a.top_k + lane] = c.weight;
}

__global__ void __launch_bounds__(32) moe_choose_kernel(const b200q_moe_args a, int64_t first, const double* logits) {
  pdl_enter();
  const int64_t t = blockIdx.x;
  const int lane = threadIdx.x;
  const MoeChoice c = moe_choose(a, logits + t * a.experts, t < moe_tokens(a, first), lane);
  if (lane < a.top_k) moe_store_choice(a, t, lane, c);
}

// ---------------------------------------------------------------------------- plain
// Any sizes and alignment: a warp per (slot, unit) for h, a warp per (slot, output) for the second product.
__global__ void __launch_bounds__(kMoeThreads) moe_plain_up_kernel(const b200q_moe_args a, float* hidden) {
  pdl_enter();
  const int lane = threadIdx.x & 31;
  const int64_t at = (int64_t)blockIdx.x * (kMoeThreads / 32) + (threadIdx.x >> 5);
  if (at >= a.tokens * a.top_k * a.inner) return;
  const int64_t slot = at / a.inner, unit = at - slot * a.inner, t = slot / a.top_k, e = a.ids[slot];
  if (e < 0) return;
  const int64_t gate = e * 2 * a.inner + unit, up = gate + a.inner;
  float g = 0.f, u = 0.f;
  for (int64_t i = lane; i < a.hidden; i += 32) {
    const float x = moe_x(a, t, i);
    g += x * moe_weight(a.gate_up, a.weight_dtype, gate * a.hidden + i);
    u += x * moe_weight(a.gate_up, a.weight_dtype, up * a.hidden + i);
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    g += __shfl_xor_sync(0xFFFFFFFFu, g, o);
    u += __shfl_xor_sync(0xFFFFFFFFu, u, o);
  }
  if (a.gate_up_scale) {
    g *= a.gate_up_scale[gate];
    u *= a.gate_up_scale[up];
  }
  if (lane == 0) hidden[at] = moe_finite(moe_silu(g) * u);
}
__global__ void __launch_bounds__(kMoeThreads) moe_plain_down_kernel(const b200q_moe_args a, const float* hidden, float* outputs) {
  pdl_enter();
  const int lane = threadIdx.x & 31;
  const int64_t at = (int64_t)blockIdx.x * (kMoeThreads / 32) + (threadIdx.x >> 5);
  if (at >= a.tokens * a.top_k * a.hidden) return;
  const int64_t slot = at / a.hidden, c = at - slot * a.hidden, e = a.ids[slot];
  if (e < 0) return;
  float sum = 0.f;
  for (int64_t i = lane; i < a.inner; i += 32) sum += hidden[slot * a.inner + i] * moe_weight(a.down, a.weight_dtype, (e * a.hidden + c) * a.inner + i);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xFFFFFFFFu, sum, o);
  if (lane == 0) outputs[at] = sum * (a.down_scale ? a.down_scale[e * a.hidden + c] : 1.f);
}
__global__ void __launch_bounds__(kMoeThreads) moe_sum_kernel(const b200q_moe_args a, const float* outputs) {
  pdl_enter();
  const int64_t per_row = (a.hidden + kMoeThreads - 1) / kMoeThreads;
  const int64_t t = blockIdx.x / per_row, c = (blockIdx.x - t * per_row) * kMoeThreads + threadIdx.x;
  if (c >= a.hidden) return;
  float sum = 0.f;
  for (int j = 0; j < a.top_k; ++j) {
    const int64_t slot = t * a.top_k + j;
    if (a.ids[slot] >= 0) sum += a.weights[slot] * outputs[slot * a.hidden + c];
  }
  if (a.out_dtype == B200Q_F32) static_cast<float*>(a.out)[t * a.hidden + c] = sum;
  else static_cast<__nv_bfloat16*>(a.out)[t * a.hidden + c] = __float2bfloat16_rn(sum);
}

// ---------------------------------------------------------------------------- tensor cores
// Bound by the weights of the chosen experts, each read once: a product of a weight tile with the few tokens of an expert has the weights as the
// 128 rows of tcgen05.mma and the tokens as its columns.  What 8-bit weights meet has to be 8 bits too, so that a value becomes several e4m3
// terms, a column each, scaled by powers of two: bf16 values of a token two terms (8 bits, which is all they have), h three (12 bits; for an fp32 output six, 24 bits).  The
// weights then go from global memory to the tensor core as they are, by TMA alone; f16 operands would want every weight converted in
// registers first.
//
// One persistent CTA per SM; the units of the work are (group of an expert's tokens, tile of weight rows), which the CTAs take from a counter: in equal
// runs of one list the SMs that get at the memory fastest were done after 203 us and the last ones after 272 (29 tokens, 108 experts of 4096 x 1792).  Long
// tiles are cut into parts of a few steps of 128 bytes of a row where they do not come out even, so that all end together, and few experts load every SM; a cut
// tile is summed, in the parts' order, by a CTA that its number gives.  (By the one whose part comes last, a CTA that falls behind gets the sums too.)
// Both products are one stream of units without a barrier between: the second one of a group waits for the group's first.
//
// The terms of x are made by the router's kernel, those of a slot's h when its last tile is finished (its largest value gives their scale), and come by
// TMA as the weights do, an expert's tokens by gathered rows.  (Made by each CTA for itself, step by step from registers, they paced the kernel.)
//   warp 0: weights     warp 1: MMAs     warp 2: terms     warps 3-6: sums of cut tiles, terms of h     warps 7-10: results
constexpr int kMoeWarps = 11;
constexpr int kMoeErrWeights = 821, kMoeErrTokens = 822, kMoeErrMma = 823, kMoeErrResults = 824, kMoeErrGrid = 825;  // status codes: a wait ran out
constexpr int kMoeGroupTokens = 32;     // of an expert, at a time
constexpr int kMoeFineTokens = 16;      // the same for an fp32 output of 8-bit weights, whose six terms are that many columns more
constexpr int kMoeSubBytes = 128 * 128;  // a weight tile: 128 rows of 128 bytes; a step has two (gate and up, or 256 outputs)
constexpr int kMoeMostDim = 65536;
constexpr uint32_t kMoeGridPolls = 1u << 21;  // some two seconds
constexpr uint32_t kMoeTestPolls = 1u << 14;  // of the self-test: some ten milliseconds

constexpr int kMoeCutTiles = kNumSMs * 5 / 4 + 1, kMoeMostParts = 8, kMoeSumTokens = 4;
constexpr int kMoeMostGroups = kMoeMaxExperts + (int)kMoeChunk * kMoeMaxTopK / kMoeFineTokens;
struct MoeControl {  // cleared by the router's kernel
  uint32_t chosen, done, next[2];
  uint32_t parts[2][kMoeCutTiles];  // of a cut tile that are there, four warps each
  uint32_t up[kMoeMostGroups];      // of a group's first product: tiles times blocks of four tokens that are finished, four warps each
  uint32_t terms[kMoeMostGroups];   // slots of a group whose terms are there, four warps each
};

// FINE: the output is fp32.  Then h has as many terms as hold its 24 bits, and no more than 256 products are added inside the tensor core, whose additions drop what does not fit 24
// bits of the sum so far (lora.cu has the figures): the results' warps add those sums in fp32.  Otherwise both would be far below the output's rounding to bf16.
template <bool FP8, int MAXN, bool FINE>
struct MoeTile {
  static constexpr int kUpTerms = FP8 ? 2 : 1, kDownTerms = FINE ? (FP8 ? 6 : 3) : FP8 ? 3 : 2;
  static constexpr int kCols = (kDownTerms * MAXN + 15) / 16 * 16;  // columns of an accumulator
  static constexpr int kTokenBytes = kCols * 128;
  static constexpr int kStage = 2 * kMoeSubBytes + kTokenBytes;
  static constexpr int kStages = 200 * 1024 / kStage < 5 ? 200 * 1024 / kStage : 5;
  static constexpr int kTmem = 4 * kCols <= 64 ? 64 : 4 * kCols <= 128 ? 128 : 4 * kCols <= 256 ? 256 : 512;  // two accumulators of two tiles
  static constexpr int kStep = FP8 ? 128 : 64;  // values of K in a step
  static constexpr int kSub = 256 / kStep;      // steps that are added inside the tensor core where FINE
  static constexpr int kPart = 2 * MAXN * 128;  // floats of a partial result: [tile][token][row]
  static_assert(kTokenBytes % 1024 == 0, "tiles lie on boundaries of the swizzle");
  static_assert(4 * kCols <= 512, "two accumulators of two tiles are in tensor memory");
};

struct MoeFused {
  const double* logits;
  const uint32_t* x_top;   // bits of max |x| per token
  uint32_t* h_top;         // bits of max |h| per slot
  float *hidden, *outputs;  // [slots][inner] (8-bit weights), [slots][hidden]: slots in the order of experts
  uint8_t* h_terms;        // [terms][slots][inner], of a byte or two
  int slots;               // of that
  float* parts;            // [products][cut tiles][parts][kPart]
  MoeControl* control;
  int* status;
  int up_tiles, up_steps, down_tiles, down_steps;
  int lost;  // self-test: what never comes (MoeLost)
};
// What a self-test waits for in vain: a CTA's choices, a CTA's results, the weights of a step, the tokens of a step (the last two in CTA 0).
enum MoeLost { kMoeLostChoice, kMoeLostResults, kMoeLostWeights, kMoeLostTokens, kMoeLostCount };

__device__ __forceinline__ uint32_t moe_ld_acquire(const uint32_t* p) {
  uint32_t v;
  asm volatile("ld.acquire.gpu.global.u32 %0, [%1];" : "=r"(v) : "l"(p) : "memory");
  return v;
}
__device__ __forceinline__ void moe_add_release(uint32_t* p, int n = 1) { asm volatile("red.release.gpu.global.add.u32 [%0], %1;" ::"l"(p), "r"(n) : "memory"); }
// until all CTAs have arrived (one warp); false when they do not
__device__ __forceinline__ bool moe_grid_wait(const uint32_t* p, uint32_t want, volatile int* abort_flag, int* status, uint32_t polls) {
  for (uint32_t i = 0; i < polls; ++i) {
    if (__all_sync(0xFFFFFFFFu, moe_ld_acquire(p) >= want)) return true;
    if ((i & 63u) == 63u && __any_sync(0xFFFFFFFFu, *abort_flag)) return false;
    if (i > 64u) __nanosleep(64);
  }
  *abort_flag = 1;
  atomicCAS(status, 0, kMoeErrGrid);
  return false;
}
// between ordinary accesses to memory and those of copies
__device__ __forceinline__ void moe_fence_async() { asm volatile("fence.proxy.async;" ::: "memory"); }
// x / d for -d < x < 2^22 (0 below 0) from 1 / d: (x + 1/2) / d is at least 1 / 2d from a whole number, and its two roundings are off by less than x / d * 2^-22.  (A division of
// integers is a hundred cycles, and some ten of them stood before the first copy.)
__device__ __forceinline__ int moe_divide(int x, float inverse) { return (int)(((float)x + 0.5f) * inverse); }

// The units of a product: `whole` tiles, then the parts of the others.  Fewer than 2^22 of them: at most 768 groups, of 512 tiles each.
// Cut are the tiles that do not come out even, and a quarter of a round of all CTAs at least; but not
// * tiles of up to 8 steps;
// * tiles of up to 32 steps (4096 bytes of a row) where there is one for each third CTA or more: fewer CTAs draw more each, and the sums come on top.  us with cuts above 8 steps, above
//   32 and none at all: 64 tokens of 32 experts 2048 x 688 (192 tiles) 66, 60, 60; 16 tokens of 64 experts 2048 x 1408 94, 86, 86; 29 tokens of 128 experts 4096 x 1792 383, 378, 377.
//   One token, with and without: 14 tiles of 32 steps 26.6, 34.2; 28 28.7, 35.4; 32 28.8, 34.2; 32 of 16 steps 25.7, 27.2; 64 of 32 42.8, 39.4; 64 of 16 32.8, 29.3; 64 and 32 of 32 as now 42.0,
//   uncut 45.2; bf16 weights, 8 and 8 of 32 and 16 steps 21.1, 31.5;
// * any where a product has less than a round of the CTAs, but 70 % of one: those draw all that the memory gives.  One token of a bf16 expert of 4096 x 128 n, n tiles of 64 steps, us with
//   and without: n = 40 42.2, -; 75 57.5, 58.6; 90 64.2, 64.8; 100 69.3, 68.6; 105 72.2, 70.3; 112 76.1, 73.8; 120 79.0, 74.7; 148 91.3, 88.1; in e4m3 (8192 x 128 n) 90 76.3, 75.0; 105 83.7,
//   80.8; 140 102.9, 98.3.
struct MoeUnits {
  int tiles, steps, whole, cut, parts, units;  // tiles of a group, steps of a tile
  float per_group, per_tile;
  __device__ __forceinline__ MoeUnits(int groups, int tiles_, int steps_, int ctas) {
    tiles = tiles_;
    steps = steps_;
    const int total = groups * tiles, rounds = max(0, moe_divide(total - ctas / 4, __frcp_rn((float)ctas)));
    cut = total - rounds * ctas;
    if (steps <= 8 || (steps <= 32 && 3 * total > ctas) || (total <= ctas && 10 * total >= 7 * ctas)) cut = 0;
    const int length = max(3, min((int)((float)(cut * steps) * __frcp_rn((float)(3 * ctas))), 8));
    parts = min(moe_divide(steps + length - 1, __frcp_rn((float)length)), kMoeMostParts);
    whole = total - cut;
    units = whole + cut * parts;
    per_group = __frcp_rn((float)tiles);
    per_tile = __frcp_rn((float)parts);
  }
};
struct MoeUnit {
  int group, row, part, cut, k0, k1;  // part: -1 for a whole tile; cut: index among the cut tiles
  __device__ __forceinline__ MoeUnit(const MoeUnits& u, int i) {
    int tile = i;
    part = -1;
    cut = 0;
    k0 = 0;
    k1 = u.steps;
    if (i >= u.whole) {
      cut = moe_divide(i - u.whole, u.per_tile);
      part = (i - u.whole) - cut * u.parts;
      tile = u.whole + cut;
      k0 = moe_divide(part * u.steps, u.per_tile);
      k1 = moe_divide((part + 1) * u.steps, u.per_tile);
    }
    group = moe_divide(tile, u.per_group);
    row = tile - group * u.tiles;
  }
};

template <bool FP8, int MAXN, bool FINE, bool TEST>  // TEST: short waits, one of them in vain
__global__ void __launch_bounds__(32 * kMoeWarps, 1)
    moe_fused_kernel(const __grid_constant__ CUtensorMap map_up, const __grid_constant__ CUtensorMap map_down, const __grid_constant__ CUtensorMap map_x,
                     const __grid_constant__ CUtensorMap map_h, const b200q_moe_args a, int64_t first, const MoeFused w) {
  using Tile = MoeTile<FP8, MAXN, FINE>;
  constexpr int kStages = Tile::kStages, kSteps = Tile::kStep;
  constexpr uint32_t kLimit = TEST ? kMoeTestPolls : ptx::kWaitLimit, kPolls = TEST ? kMoeTestPolls : kMoeGridPolls;
  constexpr int kMostSlots = MAXN == 8 ? 8 * kMoeMaxTopK : (int)kMoeChunk * kMoeMaxTopK;
  constexpr int kMostGroups = MAXN == 8 ? 8 * kMoeMaxTopK : kMoeMaxExperts + kMostSlots / MAXN;
  constexpr int kMaskWords = MAXN == 8 ? 1 : (int)kMoeChunk / 32;
  extern __shared__ __align__(1024) uint8_t s_raw[];
  uint8_t* const s_ring = s_raw + (0u - ptx::smem_u32(s_raw) & 1023u);
  __shared__ uint16_t s_slot_of[kMostSlots], s_token_of[kMostSlots];  // slot of (token, j); token of a slot
  __shared__ uint16_t s_group_expert[kMostGroups], s_group_slot[kMostGroups];
  __shared__ uint8_t s_group_tokens[kMostGroups];
  constexpr int kQueue = 4;  // units that the producer is ahead of the others at most
  __shared__ __align__(8) uint64_t s_bars[3 * kStages + 4 + 2 * kQueue + 1];
  __shared__ uint32_t s_tmem;
  __shared__ int s_abort, s_groups, s_slots, s_scan[2][kMoeWarps], s_unit[kQueue];
  __shared__ uint16_t s_expert_slot[kMoeMaxExperts];  // an expert's first slot
  // before the ring is in use: a bit per token of each expert
  uint32_t* const s_mask = reinterpret_cast<uint32_t*>(s_ring);
  int16_t* const s_ids = reinterpret_cast<int16_t*>(s_ring + sizeof(uint32_t) * kMoeMaxExperts * kMaskWords);  // [tokens][top_k]

  const int tid = threadIdx.x, lane = tid & 31, warp = ptx::uniform_warp_index();
  const int cta = blockIdx.x, ctas = gridDim.x;
  const uint32_t bar_weights = ptx::smem_u32(s_bars), bar_tokens = bar_weights + 8 * kStages, bar_empty = bar_tokens + 8 * kStages;
  const uint32_t bar_full = bar_empty + 8 * kStages, bar_free = bar_full + 16;  // of the two accumulators
  const uint32_t bar_unit = bar_free + 16, bar_taken = bar_unit + 8 * kQueue, bar_last = bar_taken + 8 * kQueue;
  const uint32_t ring = ptx::smem_u32(s_ring);
  if (tid == 0) {
    for (int i = 0; i < kStages; ++i) {
      ptx::mbar_init(bar_weights + 8 * i, 1);
      ptx::mbar_init(bar_tokens + 8 * i, 1);
      ptx::mbar_init(bar_empty + 8 * i, 1);
    }
    for (int i = 0; i < 2; ++i) {
      ptx::mbar_init(bar_full + 8 * i, 1);
      ptx::mbar_init(bar_free + 8 * i, 4);
    }
    for (int i = 0; i < kQueue; ++i) {
      ptx::mbar_init(bar_unit + 8 * i, 1);
      ptx::mbar_init(bar_taken + 8 * i, 6);  // (MMAs, terms, four of the results)
    }
    ptx::mbar_init(bar_last, 1);
    s_abort = 0;
    ptx::fence_barrier_init();
    ptx::tma_prefetch_desc(&map_up);
    ptx::tma_prefetch_desc(&map_down);
    ptx::tma_prefetch_desc(&map_x);
    ptx::tma_prefetch_desc(&map_h);
  }
  if (warp == 1) {
    ptx::tmem_alloc(ptx::smem_u32(&s_tmem), Tile::kTmem);
    ptx::tmem_relinquish();
  }
  pdl_enter();

  // ---- the choice: by every CTA for itself where a warp has few tokens (29 tokens of 128 experts: a barrier between the CTAs takes longer than three more
  // rounds), else a token per warp of the grid
  const int tokens = (int)a.tokens, live = moe_tokens(a, first), top_k = a.top_k, slots = live * top_k;
  bool ok = true;
  for (int i = tid; i < a.experts * kMaskWords; i += 32 * kMoeWarps) s_mask[i] = 0;
  if (MAXN == 8 || tokens <= 4 * kMoeWarps) {
    for (int t = warp; t < tokens; t += kMoeWarps) {
      const MoeChoice c = moe_choose(a, w.logits + (int64_t)t * a.experts, t < live, lane);
      if (lane < top_k) {
        s_ids[t * top_k + lane] = (int16_t)c.id;
        if (cta == 0) moe_store_choice(a, t, lane, c);
      }
    }
    __syncthreads();
  } else {
    for (int t = warp * ctas + cta; t < tokens; t += kMoeWarps * ctas) {
      const MoeChoice c = moe_choose(a, w.logits + (int64_t)t * a.experts, t < live, lane);
      if (lane < top_k) moe_store_choice(a, t, lane, c);
    }
    __threadfence();
    __syncthreads();
    if (tid == 0) moe_add_release(&w.control->chosen);
    ok = moe_grid_wait(&w.control->chosen, (uint32_t)ctas + (TEST && w.lost == kMoeLostChoice), &s_abort, w.status, kPolls);
    for (int i = tid; i < slots; i += 32 * kMoeWarps) s_ids[i] = (int16_t)__ldcg(a.ids + i);
    ok = __syncthreads_and(ok);
  }

  // ---- the list: slots in the order of experts, and tokens, and groups of at most MAXN tokens of an expert
  for (int i = tid; i < slots; i += 32 * kMoeWarps) {
    const int t = i / top_k, e = s_ids[i];
    if (e >= 0 && e < a.experts) atomicOr(&s_mask[e * kMaskWords + t / 32], 1u << (t & 31));
  }
  __syncthreads();
  {
    int slots_before = 0, groups_before = 0;
    for (int base = 0, turn = 0; base < a.experts; base += 32 * kMoeWarps, turn ^= 1) {
      const int e = base + tid;
      int n = 0;
      if (e < a.experts)
        for (int i = 0; i < kMaskWords; ++i) n += __popc(s_mask[e * kMaskWords + i]);
      const int mine = n | ((n + MAXN - 1) / MAXN) << 16;  // (both sums stay below 2^15)
      int scan = mine;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int v = __shfl_up_sync(0xFFFFFFFFu, scan, o);
        if (lane >= o) scan += v;
      }
      if (lane == 31) s_scan[turn][warp] = scan;
      __syncthreads();  // (the other half is written next, and this one only behind the next barrier)
      int before = slots_before | groups_before << 16, all = before;
      for (int i = 0; i < kMoeWarps; ++i) {
        if (i < warp) before += s_scan[turn][i];
        all += s_scan[turn][i];
      }
      before += scan - mine;
      slots_before = all & 0xFFFF;
      groups_before = all >> 16;
      if (n) {
        const int slot = before & 0xFFFF;
        int group = before >> 16;
        s_expert_slot[e] = (uint16_t)slot;
        for (int i = 0; i < n; i += MAXN, ++group) {
          s_group_expert[group] = (uint16_t)e;
          s_group_slot[group] = (uint16_t)(slot + i);
          s_group_tokens[group] = (uint8_t)min(n - i, MAXN);
        }
      }
    }
    if (tid == 0) {
      s_groups = groups_before;
      s_slots = slots_before;
    }
  }
  __syncthreads();
  for (int i = tid; i < slots; i += 32 * kMoeWarps) {  // an expert's slots are in the order of its tokens
    const int t = i / top_k, e = s_ids[i];
    if (e < 0 || e >= a.experts) continue;
    int slot = s_expert_slot[e];
    for (int k = 0; k < t / 32; ++k) slot += __popc(s_mask[e * kMaskWords + k]);
    slot += __popc(s_mask[e * kMaskWords + t / 32] & ((1u << (t & 31)) - 1u));
    s_slot_of[i] = (uint16_t)slot;
    s_token_of[slot] = (uint16_t)t;
  }
  ptx::tc_fence_before();
  __syncthreads();
  ptx::tc_fence_after();
  // (the ring's first bytes were written and read by ordinary accesses; the copies come through another path)
  ptx::fence_proxy_async_smem();
  __syncthreads();
  const uint32_t tmem = s_tmem;
  const int groups = s_groups, slots_here = s_slots;
  auto units_of = [&](int product) { return MoeUnits(groups, product ? w.down_tiles : w.up_tiles, product ? w.down_steps : w.up_steps, ctas); };

  // The next unit as the producer has passed it on, or -1 at the end of a product; the same for all warps but the producer.
  uint32_t turn = 0, turn_phase = 0;
  auto next_unit = [&](int code) {
    int unit = -1;
    ok = ptx::mbar_wait_uniform(bar_unit + 8 * turn, turn_phase, &s_abort, w.status, code, kLimit);
    if (!ok) return unit;
    unit = *(volatile int*)&s_unit[turn];
    __syncwarp();
    if (lane == 0) ptx::mbar_arrive(bar_taken + 8 * turn);
    if (++turn == kQueue) {
      turn = 0;
      turn_phase ^= 1;
    }
    return unit;
  };

  // a role's place in the ring, and its copies so far
  uint32_t stage = 0, phase = 0;
  int made = 0;
  // where a wait has run out: the copies in flight are waited for, as far as they come
  auto drain = [&](uint32_t bars) {
    for (int i = 0; i < min(made, kStages); ++i) {
      phase ^= stage == 0;
      stage = stage == 0 ? kStages - 1 : stage - 1;
      for (int k = 0; k < 4096 && !ptx::mbar_try_wait(bars + 8 * stage, phase); ++k) __nanosleep(64);
    }
  };
  // blocks of tokens that a group's results are counted in
  auto blocks_of = [&](int group) { return (s_group_tokens[group] + kMoeSumTokens - 1) / kMoeSumTokens; };
  // the terms of a slot's h, by the four warps of the sums
  auto terms_of_h = [&](int slot) {
    int group = 0;
    for (int hi = groups - 1; group < hi;) {  // the last group that does not begin behind the slot
      const int mid = (group + hi + 1) >> 1;
      if (s_group_slot[mid] <= slot) group = mid;
      else hi = mid - 1;
    }
    ok = moe_grid_wait(&w.control->up[group], 4 * (uint32_t)(w.up_tiles * blocks_of(group)), &s_abort, w.status, kPolls);
    if (!ok) return;
    const float factor = moe_up_factor(__ldcg(w.h_top + slot));
    for (int64_t i = 8 * (tid - 96); i < a.inner; i += 8 * 128) {
      const float4* p = reinterpret_cast<const float4*>(w.hidden + slot * a.inner + i);
      const float4 x = __ldcg(p), y = __ldcg(p + 1);
      float v[8] = {x.x, x.y, x.z, x.w, y.x, y.y, y.z, y.w};
#pragma unroll
      for (int c = 0; c < 8; ++c) {
        v[c] = moe_finite(v[c] * factor);
      }
      uint2 term[Tile::kDownTerms];
      moe_terms_fp8<Tile::kDownTerms>(v, term);
#pragma unroll
      for (int c = 0; c < Tile::kDownTerms; ++c) *reinterpret_cast<uint2*>(w.h_terms + ((int64_t)c * w.slots + slot) * a.inner + i) = term[c];
    }
    moe_fence_async();
    __syncwarp();
    if (lane == 0) moe_add_release(&w.control->terms[group]);
  };
  // what a group's values are to be multiplied by: lane j has token j's
  auto backs_of = [&](auto which, const MoeUnit& unit) {
    constexpr int product = decltype(which)::value;
    const int slot = s_group_slot[unit.group] + lane;
    if (!FP8 || lane >= s_group_tokens[unit.group]) return 1.f;
    return moe_down_factor(product ? __ldcg(w.h_top + slot) : __ldcg(w.x_top + s_token_of[slot]));
  };
  // a result: token j of a group's values in row `row` of the two tiles of a unit
  auto finish = [&](auto which, const MoeUnit& unit, int row, int j, float v0, float v1, const float (&scale)[2], float backs) {
    constexpr int product = decltype(which)::value;
    const int slot = s_group_slot[unit.group] + j;
    const float back = __shfl_sync(0xFFFFFFFFu, backs, j);
    if (product == 0) {
      const int64_t r = unit.row * 128 + row;
      const float h = r < a.inner ? moe_silu(v0 * back * scale[0]) * (v1 * back * scale[1]) : 0.f;
      if constexpr (FP8) {
        if (r < a.inner) __stcg(w.hidden + (int64_t)slot * a.inner + r, h);
        const uint32_t top = __reduce_max_sync(0xFFFFFFFFu, __float_as_uint(h) & 0x7FFFFFFFu);
        if (lane == 0) atomicMax(w.h_top + slot, top);
      } else if (r < a.inner) {
        __nv_bfloat16* to = reinterpret_cast<__nv_bfloat16*>(w.h_terms) + (int64_t)slot * a.inner + r;
        // (all terms but the last stay within bf16, so that what lies between the ends of bf16 and fp32 has a rest)
        float v = moe_finite(h);
#pragma unroll
        for (int t = 0; t < Tile::kDownTerms; ++t) {
          const __nv_bfloat16 term = __float2bfloat16_rn(t + 1 < Tile::kDownTerms ? fminf(fmaxf(v, -3.3895313892515355e38f), 3.3895313892515355e38f) : v);
          to[t * (int64_t)w.slots * a.inner] = term;
          v -= __bfloat162float(term);
        }
      }
    } else {
      const int64_t r = unit.row * 256 + row;
      if (r < a.hidden) __stcg(w.outputs + (int64_t)slot * a.hidden + r, v0 * back * scale[0]);
      if (r + 128 < a.hidden) __stcg(w.outputs + (int64_t)slot * a.hidden + r + 128, v1 * back * scale[1]);
    }
  };
  // the scales of a row of the two tiles
  auto scales_of = [&](auto which, const MoeUnit& unit, int row, float (&scale)[2]) {
    constexpr int product = decltype(which)::value;
    const int64_t e = s_group_expert[unit.group], r = (product ? unit.row * 256 : unit.row * 128) + row;
    const float* scales = product ? a.down_scale : a.gate_up_scale;
    scale[0] = scale[1] = 1.f;
    if (!scales) return;
    if (product == 0 && r < a.inner) {
      scale[0] = scales[e * 2 * a.inner + r];
      scale[1] = scales[e * 2 * a.inner + a.inner + r];
    } else if (product == 1) {
      if (r < a.hidden) scale[0] = scales[e * a.hidden + r];
      if (r + 128 < a.hidden) scale[1] = scales[e * a.hidden + r + 128];
    }
  };
  // behind the last unit: the warps of the sums and of the results together, whatever became of their waits
  auto finished_all = [&] {
    __threadfence();
    ok = layer_bar_and(3, 256, ok);
    if (ok && tid == 96) moe_add_release(&w.control->done);
  };
  // some blocks of tokens of a tile of a group's first product are finished (one of four warps)
  auto finished_up = [&](int group, int blocks) {
    if (!FP8) moe_fence_async();
    __syncwarp();
    if (lane == 0) moe_add_release(&w.control->up[group], blocks);
  };

  if (!ok && warp < 3) {
    // (a CTA did not come: nothing is in flight, and nobody goes on)
  } else if (warp == 0) {
    // ------------------------------------------------------------ weights
    auto publish = [&](int u) {
      ok = ok && ptx::mbar_wait_uniform(bar_taken + 8 * turn, turn_phase ^ 1, &s_abort, w.status, kMoeErrWeights, kLimit);
      if (!ok) return;
      if (lane == 0) {
        *(volatile int*)&s_unit[turn] = u;
        ptx::mbar_arrive(bar_unit + 8 * turn);
      }
      if (++turn == kQueue) {
        turn = 0;
        turn_phase ^= 1;
      }
    };
    auto stream = [&](auto which) {
      constexpr int product = decltype(which)::value;
      const MoeUnits list = units_of(product);
      // The first units, `dealt` each, are the CTA's by its index.  The others come from the counter, whose answer takes a microsecond or two behind the copies
      // and is asked for before a unit's copies are.
      const int dealt = max(1, (int)((float)list.units / (float)ctas) * 5 / 8);
      for (int i = 0, u = cta; ok; ++i) {
        publish(u < list.units ? u : -1);
        if (!ok || u >= list.units) break;
        const bool ask = i + 1 >= dealt && dealt * ctas < list.units;
        uint32_t taken = 0;  // (nothing is computed from it before the copies are on their way: that would wait for the answer)
        if (ask && lane == 0) asm volatile("atom.global.add.u32 %0, [%1], 1;" : "=r"(taken) : "l"(&w.control->next[product]) : "memory");
        const MoeUnit unit(list, u);
        const int e = s_group_expert[unit.group];
        for (int k = unit.k0; k < unit.k1; ++k) {
          ok = ptx::mbar_wait_uniform(bar_empty + 8 * stage, phase ^ 1, &s_abort, w.status, kMoeErrWeights, kLimit);
          if (!ok) break;
          if (ptx::elect_one()) {
            const uint32_t bar = bar_weights + 8 * stage, dst = ring + stage * Tile::kStage;
            ptx::mbar_arrive_expect_tx(bar, 2 * kMoeSubBytes);
            if (TEST && w.lost == kMoeLostWeights && cta == 0 && made == 0) {
              // (never copied)
            } else if (product == 0) {
              ptx::tma_load_3d(dst, &map_up, bar, k * kSteps, unit.row * 128, 2 * e);
              ptx::tma_load_3d(dst + kMoeSubBytes, &map_up, bar, k * kSteps, unit.row * 128, 2 * e + 1);
            } else {
              ptx::tma_load_3d(dst, &map_down, bar, k * kSteps, unit.row * 256, e);
              ptx::tma_load_3d(dst + kMoeSubBytes, &map_down, bar, k * kSteps, unit.row * 256 + 128, e);
            }
          }
          ++made;
          if (++stage == kStages) {
            stage = 0;
            phase ^= 1;
          }
        }
        taken = __shfl_sync(0xFFFFFFFFu, taken, 0);
        u = ask ? dealt * ctas + (int)taken : u + ctas;
      }
    };
    stream(std::integral_constant<int, 0>());
    if (ok) stream(std::integral_constant<int, 1>());
  } else if (warp == 1) {
    // ------------------------------------------------------------ products
    int pieces = 0;
    const uint64_t a0 = ptx::smem_desc_k_sw128(ring), b0 = ptx::smem_desc_k_sw128(ring + 2 * kMoeSubBytes);
    for (int product = 0; product < 2 && ok; ++product) {
      const int terms = product ? Tile::kDownTerms : Tile::kUpTerms;
      const MoeUnits list = units_of(product);
      while (ok) {
        const int u = next_unit(kMoeErrMma);
        if (u < 0) break;
        const MoeUnit unit(list, u);
        const int cols = ((s_group_tokens[unit.group] + 7) / 8 * 8 * terms + 15) / 16 * 16;
        const uint32_t idesc = FP8 ? ptx::umma_idesc(0, 0, 128, cols) : ptx::umma_idesc(1, 1, 128, cols);
        uint32_t acc = 0, d = 0;
        for (int k = unit.k0, sub_step = 0; k < unit.k1; ++k) {
          if (sub_step == 0) {
            acc = pieces & 1;
            d = tmem + acc * 2 * Tile::kCols;
            ok = ptx::mbar_wait_uniform(bar_free + 8 * acc, ((pieces >> 1) & 1) ^ 1, &s_abort, w.status, kMoeErrMma, kLimit);
            if (!ok) break;
            ++pieces;
            ptx::tc_fence_after();
          }
          ok = ptx::mbar_wait2_uniform(bar_weights + 8 * stage, phase, bar_tokens + 8 * stage, phase, &s_abort, w.status, kMoeErrMma, kLimit);
          if (!ok) break;
          ptx::tc_fence_after();
          const uint64_t off = stage * (uint32_t)(Tile::kStage >> 4);
          if (ptx::elect_one()) {
#pragma unroll
            for (int sub = 0; sub < 2; ++sub) {
              if (FP8) ptx::umma_f8_x4(d + sub * Tile::kCols, a0 + off + sub * (kMoeSubBytes >> 4), b0 + off, idesc, sub_step != 0, 2, 2);
              else ptx::umma_f16_x4(d + sub * Tile::kCols, a0 + off + sub * (kMoeSubBytes >> 4), b0 + off, idesc, sub_step != 0, 2, 2);
            }
            ptx::umma_commit(bar_empty + 8 * stage);
            if (k + 1 == unit.k1 || (FINE && sub_step + 1 == Tile::kSub)) ptx::umma_commit(bar_full + 8 * acc);
          }
          __syncwarp();
          if (++sub_step == Tile::kSub && FINE) sub_step = 0;
          if (++stage == kStages) {
            stage = 0;
            phase ^= 1;
          }
        }
      }
    }
  } else if (warp == 2) {
    // ------------------------------------------------------------ terms
    auto stream = [&](auto which) {
      constexpr int product = decltype(which)::value, terms = product ? Tile::kDownTerms : Tile::kUpTerms;
      const MoeUnits list = units_of(product);
      int there = -1;  // the group whose h is known to be there
      while (ok) {
        const int u = next_unit(kMoeErrTokens);
        if (u < 0) break;
        const MoeUnit unit(list, u);
        const int slot = s_group_slot[unit.group], n = s_group_tokens[unit.group], blocks = (n + 7) / 8;
        if (product == 1 && unit.group != there) {
          ok = FP8 ? moe_grid_wait(&w.control->terms[unit.group], 4 * (uint32_t)n, &s_abort, w.status, kPolls)
                   : moe_grid_wait(&w.control->up[unit.group], 4 * (uint32_t)(w.up_tiles * blocks_of(unit.group)), &s_abort, w.status, kPolls);
          if (!ok) break;
          moe_fence_async();
          there = unit.group;
        }
        // x: lane i fetches four tokens' rows of a term (columns behind the last token are that token's again, and not looked at)
        const int four = lane & 1, term = (lane >> 1) % terms, block = (lane >> 1) / terms;
        int rows[4] = {};
        if (product == 0 && block < blocks) {
#pragma unroll
          for (int i = 0; i < 4; ++i) rows[i] = term * tokens + s_token_of[slot + min(8 * block + 4 * four + i, n - 1)];
        }
        for (int k = unit.k0; k < unit.k1; ++k) {
          ok = ptx::mbar_wait_uniform(bar_empty + 8 * stage, phase ^ 1, &s_abort, w.status, kMoeErrTokens, kLimit);
          if (!ok) break;
          if (ptx::elect_one()) {
            const uint32_t bar = bar_tokens + 8 * stage, dst = ring + stage * Tile::kStage + 2 * kMoeSubBytes;
            ptx::mbar_arrive_expect_tx(bar, blocks * terms * 1024);
            if (product == 1)
              for (int g = 0; g < blocks; ++g) ptx::tma_load_3d(dst + g * terms * 1024, &map_h, bar, k * kSteps, slot + 8 * g, 0);
          }
          __syncwarp();
          if (product == 0 && block < blocks && !(TEST && w.lost == kMoeLostTokens && cta == 0 && made == 0))
            layer_gather4(ring + stage * Tile::kStage + 2 * kMoeSubBytes + (lane >> 1) * 1024 + four * 512, &map_x, bar_tokens + 8 * stage, k * kSteps, rows);
          __syncwarp();
          ++made;
          if (++stage == kStages) {
            stage = 0;
            phase ^= 1;
          }
        }
      }
    };
    stream(std::integral_constant<int, 0>());
    if (ok) stream(std::integral_constant<int, 1>());
  } else if (warp < 7) {
    // ------------------------------------------------------------ sums of cut tiles, terms of h
    const int row = tid - 96;
    auto sums_of = [&](auto which) {
      constexpr int product = decltype(which)::value;
      const MoeUnits list = units_of(product);
      // A task is four tokens of a tile, so that all CTAs have some where tiles are few; those of the tiles' first tokens come first.
      constexpr int kBlocks = MAXN / kMoeSumTokens;
      const float per_block = __frcp_rn((float)max(list.cut, 1));
      for (int i = cta; i < list.cut * kBlocks && ok; i += ctas) {
        const int block = moe_divide(i, per_block), c = i - block * list.cut, j0 = kMoeSumTokens * block;
        const MoeUnit unit(list, list.whole + c * list.parts);
        const int n = s_group_tokens[unit.group];
        if (j0 >= n) continue;
        ok = moe_grid_wait(&w.control->parts[product][c], 4 * (uint32_t)list.parts, &s_abort, w.status, kPolls);
        if (!ok) break;
        float scale[2];
        scales_of(which, unit, row, scale);
        const float backs = backs_of(which, unit);
        const float* p = w.parts + ((int64_t)product * kMoeCutTiles + unit.cut) * kMoeMostParts * Tile::kPart + row;
        float v[kMoeSumTokens][2][kMoeMostParts];
#pragma unroll
        for (int b = 0; b < kMoeSumTokens; ++b)
#pragma unroll
          for (int sub = 0; sub < 2; ++sub)
#pragma unroll
            for (int k = 0; k < kMoeMostParts; ++k) v[b][sub][k] = k < list.parts && j0 + b < n ? __ldcg(p + k * Tile::kPart + (sub * MAXN + j0 + b) * 128) : 0.f;
#pragma unroll
        for (int b = 0; b < kMoeSumTokens; ++b) {
#pragma unroll
          for (int k = 1; k < kMoeMostParts; ++k) {
            v[b][0][0] += v[b][0][k];
            v[b][1][0] += v[b][1][k];
          }
          if (j0 + b < n) finish(which, unit, row, j0 + b, v[b][0][0], v[b][1][0], scale, backs);
        }
        if (product == 0) finished_up(unit.group, 1);
      }
    };
    // the slots of groups without cut tiles are ready before those tiles are, the others behind them
    const MoeUnits ups = units_of(0);
    const int first_cut = moe_divide(ups.whole, ups.per_group), early = first_cut < groups ? s_group_slot[first_cut] : slots_here;
    int mine = cta;
    if (FP8)
      for (; ok && mine < early; mine += ctas) terms_of_h(mine);
    sums_of(std::integral_constant<int, 0>());
    if (FP8)
      for (; ok && mine < slots_here; mine += ctas) terms_of_h(mine);
    sums_of(std::integral_constant<int, 1>());
    finished_all();
  } else {
    // ------------------------------------------------------------ results
    const int row = 32 * (warp & 3) + lane;  // of a tile: the lane of tensor memory that this thread reads
    const uint32_t lane_base = (uint32_t)(32 * (warp & 3)) << 16;
    int pieces = 0;
    auto results_of = [&](auto which) {
      constexpr int product = decltype(which)::value, terms = product ? Tile::kDownTerms : Tile::kUpTerms;
      const MoeUnits list = units_of(product);
      for (;;) {
        const int u = next_unit(kMoeErrResults);
        if (u < 0) break;
        const MoeUnit unit(list, u);
        const bool whole = unit.part < 0;
        const int n = s_group_tokens[unit.group];
        float scale[2], backs = 1.f;
        if (whole) {
          scales_of(which, unit, row, scale);
          if (product == 0) backs = backs_of(which, unit);
        }
        float* part = w.parts + (((int64_t)product * kMoeCutTiles + unit.cut) * kMoeMostParts + unit.part) * Tile::kPart + row;
        // the next sums that are there, in tensor memory at d
        uint32_t acc, d;
        auto wait = [&] {
          acc = pieces & 1;
          d = tmem + acc * 2 * Tile::kCols + lane_base;
          ok = ptx::mbar_wait_uniform(bar_full + 8 * acc, (pieces >> 1) & 1, &s_abort, w.status, kMoeErrResults, kLimit);
          if (!ok) return;
          ++pieces;
          ptx::tc_fence_after();
        };
        // eight tokens' of them, their terms put together
        auto get = [&](int j0, float (&v)[2][8]) {
#pragma unroll
          for (int sub = 0; sub < 2; ++sub) {
            float term[terms][8];
#pragma unroll
            for (int t = 0; t < terms; ++t) layer_tmem_ld8(d + sub * Tile::kCols + j0 * terms + 8 * t, term[t]);
            ptx::tmem_ld_wait();
#pragma unroll
            for (int i = 0; i < 8; ++i) {
              v[sub][i] = term[terms - 1][i];
#pragma unroll
              for (int t = terms - 2; t >= 0; --t) v[sub][i] = term[t][i] + (FP8 ? 1.f / 32.f : 1.f) * v[sub][i];
            }
          }
        };
        auto put = [&](int j, float v0, float v1) {
          if (whole) {
            finish(which, unit, row, j, v0, v1, scale, backs);
          } else {
            __stcg(part + j * 128, v0);
            __stcg(part + (MAXN + j) * 128, v1);
          }
        };
        auto release = [&] {
          ptx::tc_fence_before();
          __syncwarp();
          if (lane == 0) ptx::mbar_arrive(bar_free + 8 * acc);
        };
        if constexpr (FINE) {
          float sums[MAXN][2] = {};
          for (int k = unit.k0; k < unit.k1; k += Tile::kSub) {
            wait();
            if (!ok) break;
#pragma unroll
            for (int j0 = 0; j0 < MAXN; j0 += 8) {
              if (j0 >= n) break;
              float v[2][8];
              get(j0, v);
#pragma unroll
              for (int i = 0; i < 8; ++i) {
                sums[j0 + i][0] += v[0][i];
                sums[j0 + i][1] += v[1][i];
              }
            }
            release();
          }
          if (!ok) break;
          if (whole && product == 1) backs = backs_of(which, unit);  // (h's largest value is known now that it has been multiplied)
#pragma unroll
          for (int j = 0; j < MAXN; ++j) {
            if (j >= n) break;
            put(j, sums[j][0], sums[j][1]);
          }
        } else {
          wait();
          if (!ok) break;
          if (whole && product == 1) backs = backs_of(which, unit);  // (as above)
          for (int j0 = 0; j0 < n; j0 += 8) {
            float v[2][8];
            get(j0, v);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
              if (j0 + i >= n) break;
              put(j0 + i, v[0][i], v[1][i]);
            }
          }
          release();
        }
        if (!whole) {
          __syncwarp();
          if (lane == 0) moe_add_release(&w.control->parts[product][unit.cut]);
        } else if (product == 0) {
          finished_up(unit.group, blocks_of(unit.group));
        }
      }
    };
    if (ok) results_of(std::integral_constant<int, 0>());
    if (ok) results_of(std::integral_constant<int, 1>());
    finished_all();
    // ---- the weighted sums.  Where a wait has run out nothing is read: the list may have been made of choices that were never written, and a token's slots with it.
    if (ok) ok = moe_grid_wait(&w.control->done, (uint32_t)ctas + (TEST && w.lost == kMoeLostResults), &s_abort, w.status, kPolls);
    const int et = tid - 224;
    const int64_t quads = (a.hidden + 3) / 4;
    for (int64_t i = (int64_t)cta * 128 + et; i < tokens * quads; i += (int64_t)ctas * 128) {
      const int t = (int)(i / quads);
      const int64_t c = (i - t * quads) * 4;
      float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
      if (ok && t < live)
        for (int j = 0; j < top_k; ++j) {
          const float p = __ldcg(a.weights + t * top_k + j);
          const float4 y = __ldcg(reinterpret_cast<const float4*>(w.outputs + (int64_t)s_slot_of[t * top_k + j] * a.hidden + c));
          sum.x += p * y.x; sum.y += p * y.y; sum.z += p * y.z; sum.w += p * y.w;
        }
      if (!ok) sum.x = sum.y = sum.z = sum.w = __int_as_float(0x7FC00000);
      if (a.out_dtype == B200Q_F32) *reinterpret_cast<float4*>(static_cast<float*>(a.out) + t * a.hidden + c) = sum;
      else *reinterpret_cast<uint2*>(static_cast<__nv_bfloat16*>(a.out) + t * a.hidden + c) = make_uint2(pack_bf16x2(sum.x, sum.y), pack_bf16x2(sum.z, sum.w));
    }
  }
  __syncwarp();
  ptx::tc_fence_before();
  __syncthreads();
  if (s_abort) {  // (a role may have been done before another's wait ran out)
    if (warp == 0) drain(bar_weights);
    if (warp == 2) drain(bar_tokens);
    if (warp == 1) {  // nor do products outlive the tensor memory and the ring
      if (ptx::elect_one()) ptx::umma_commit(bar_last);
      __syncwarp();
      for (int k = 0; k < 4096 && !ptx::mbar_try_wait(bar_last, 0); ++k) __nanosleep(64);
    }
  }
  if (warp == 1) ptx::tmem_dealloc(tmem, Tile::kTmem);
}

// ---------------------------------------------------------------------------- host
MoeSpace::MoeSpace(int64_t tokens, int64_t h, int64_t f, int experts, int top_k) {
  const size_t t = (size_t)(tokens < kMoeChunk ? tokens : kMoeChunk), slots = t * (size_t)top_k;
  logits = 0;
  x_top = moe_align(logits + sizeof(double) * t * (size_t)experts);
  control = moe_align(x_top + sizeof(uint32_t) * t);
  h_top = control + sizeof(MoeControl);
  clear_words = (int)((sizeof(MoeControl) + sizeof(uint32_t) * slots) / sizeof(uint32_t));
  hidden = moe_align(h_top + sizeof(uint32_t) * slots);
  outputs = moe_align(hidden + sizeof(float) * slots * (size_t)f);
  x_terms = moe_align(outputs + sizeof(float) * slots * (size_t)h);  // [2][tokens][h]
  h_terms = moe_align(x_terms + 2 * t * (size_t)h);                    // three of a byte or two of two; for an fp32 output six or three
  parts = moe_align(h_terms + 6 * slots * (size_t)f);
  const size_t group = t <= 8 ? 8 : kMoeGroupTokens;
  bytes = moe_align(parts + sizeof(float) * 2 * kMoeCutTiles * kMoeMostParts * 2 * group * 128);
}

size_t moe_workspace_bytes_impl(int64_t tokens, int64_t hidden, int64_t inner, int experts, int top_k) {
  return MoeSpace(tokens, hidden, inner, experts, top_k).bytes;
}

static int64_t moe_blocks(int64_t warps) { return (warps + kMoeThreads / 32 - 1) / (kMoeThreads / 32); }

static bool moe_fits_tensor_cores(const b200q_moe_args& a) {
  const int64_t size = a.weight_dtype == B200Q_BF16 ? 2 : 1;
  if (a.force_plain || a.hidden <= 0 || a.inner <= 0 || a.hidden > kMoeMostDim || a.inner > kMoeMostDim || a.hidden * size % 16 || a.inner * size % 16) return false;
  if (a.tokens > 1 && (a.x_stride % 8 || a.x_stride < a.hidden)) return false;
  for (const void* p : {a.x, a.gate_up, a.down, static_cast<const void*>(a.out)})
    if (reinterpret_cast<uintptr_t>(p) % 16) return false;
  return true;
}

// [planes][rows][depth] of weights, or of terms, in boxes of rows of 128 bytes
static int moe_map(CUtensorMap* map, const void* base, bool fp8, int64_t depth, int64_t rows, int64_t planes, int box_rows = 128, int box_planes = 1) {
  EncodeTiledFn enc = get_encode_fn();
  if (!enc) return B200Q_ERR_CUDA;
  const cuuint64_t size = fp8 ? 1 : 2;
  const cuuint64_t dims[3] = {(cuuint64_t)depth, (cuuint64_t)rows, (cuuint64_t)planes}, strides[2] = {depth * size, rows * depth * size};
  const cuuint32_t box[3] = {fp8 ? 128u : 64u, (cuuint32_t)box_rows, (cuuint32_t)box_planes}, step[3] = {1, 1, 1};
  const CUresult r = enc(map, fp8 ? CU_TENSOR_MAP_DATA_TYPE_UINT8 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, const_cast<void*>(base), dims, strides, box, step,
                         CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return r == CUDA_SUCCESS ? B200Q_OK : B200Q_ERR_UNSUPPORTED;
}

template <bool FP8, int MAXN, bool FINE, bool TEST = false>
static int moe_launch_fused(const b200q_moe_args& a, int64_t first, const MoeSpace& space, cudaStream_t st, int lost = 0) {
  using Tile = MoeTile<FP8, MAXN, FINE>;
  auto kernel = moe_fused_kernel<FP8, MAXN, FINE, TEST>;
  constexpr int kSmem = Tile::kStages * Tile::kStage + 1024;
  static std::atomic<int> grid_of[kMaxDevices];  // CTAs that are resident together
  const int dev = current_device_index();
  if (dev < 0) return B200Q_ERR_CUDA;
  int grid = grid_of[dev].load(std::memory_order_acquire);
  if (!grid) {
    int per_sm = 0, sms = 0;
    B200Q_CUDA_OK(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmem));
    B200Q_CUDA_OK(cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per_sm, kernel, 32 * kMoeWarps, kSmem));
    B200Q_CUDA_OK(cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev));
    if (per_sm < 1) return B200Q_ERR_UNSUPPORTED;
    grid = sms < kNumSMs ? sms : kNumSMs;
    grid_of[dev].store(grid, std::memory_order_release);
  }
  CUtensorMap map_up, map_down;
  if (int rc = moe_map(&map_up, a.gate_up, FP8, a.hidden, a.inner, 2 * (int64_t)a.experts)) return rc;
  if (int rc = moe_map(&map_down, a.down, FP8, a.inner, a.hidden, a.experts)) return rc;
  uint8_t* p = static_cast<uint8_t*>(a.workspace);
  MoeFused w;
  w.lost = lost;
  w.slots = (int)a.tokens * a.top_k;
  w.h_terms = p + space.h_terms;
  CUtensorMap map_x, map_h;
  {  // rows one by one: the terms of x, or x itself
    EncodeTiledFn enc = get_encode_fn();
    if (!enc) return B200Q_ERR_CUDA;
    const cuuint64_t dims[2] = {(cuuint64_t)a.hidden, (cuuint64_t)a.tokens * Tile::kUpTerms};
    const cuuint64_t stride[1] = {FP8 ? (cuuint64_t)a.hidden : (cuuint64_t)(a.tokens > 1 ? a.x_stride : a.hidden) * 2};
    const cuuint32_t box[2] = {FP8 ? 128u : 64u, 1}, step[2] = {1, 1};
    const CUresult r = enc(&map_x, FP8 ? CU_TENSOR_MAP_DATA_TYPE_UINT8 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, FP8 ? p + space.x_terms : const_cast<void*>(a.x), dims, stride, box,
                           step, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) return B200Q_ERR_UNSUPPORTED;
  }
  if (int rc = moe_map(&map_h, w.h_terms, FP8, a.inner, w.slots, Tile::kDownTerms, 8, Tile::kDownTerms)) return rc;
  w.logits = reinterpret_cast<const double*>(p + space.logits);
  w.x_top = reinterpret_cast<const uint32_t*>(p + space.x_top);
  w.h_top = reinterpret_cast<uint32_t*>(p + space.h_top);
  w.hidden = reinterpret_cast<float*>(p + space.hidden);
  w.outputs = reinterpret_cast<float*>(p + space.outputs);
  w.parts = reinterpret_cast<float*>(p + space.parts);
  w.control = reinterpret_cast<MoeControl*>(p + space.control);
  w.status = device_status_ptr();
  if (!w.status) return B200Q_ERR_CUDA;
  w.up_tiles = (int)((a.inner + 127) / 128);
  w.up_steps = (int)((a.hidden + Tile::kStep - 1) / Tile::kStep);
  w.down_tiles = (int)((a.hidden + 255) / 256);
  w.down_steps = (int)((a.inner + Tile::kStep - 1) / Tile::kStep);
  // CTAs wait for one another: a cooperative launch has them all resident
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)grid);
  cfg.blockDim = dim3(32 * kMoeWarps);
  cfg.dynamicSmemBytes = kSmem;
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeCooperative;
  attr[0].val.cooperative = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  (void)cudaLaunchKernelEx(&cfg, kernel, map_up, map_down, map_x, map_h, a, first, w);
  B200Q_LAUNCH_CHECK();
  return B200Q_OK;
}

template <typename W, int EB, int TB>
static int moe_launch_logits(const b200q_moe_args& a, int64_t first, const MoeSpace& space, cudaStream_t st) {
  uint8_t* p = static_cast<uint8_t*>(a.workspace);
  const int64_t blocks = ((a.experts + EB - 1) / EB) * ((a.tokens + TB - 1) / TB);
  bool wide = a.hidden % 8 == 0 && (a.tokens == 1 || a.x_stride % 8 == 0);
  for (const void* q : {a.x, a.router}) wide = wide && reinterpret_cast<uintptr_t>(q) % 16 == 0;
  launch_dependent(moe_logits_kernel<W, EB, TB>, dim3((unsigned)blocks), dim3(kMoeThreads), 0, st, a, first, reinterpret_cast<double*>(p + space.logits),
                   reinterpret_cast<uint32_t*>(p + space.x_top), a.weight_dtype == B200Q_E4M3 && moe_fits_tensor_cores(a) ? p + space.x_terms : nullptr,
                   reinterpret_cast<uint32_t*>(p + space.control), space.clear_words, wide);
  B200Q_LAUNCH_CHECK();
  return B200Q_OK;
}
template <typename W>
static int moe_launch_router(const b200q_moe_args& a, int64_t first, const MoeSpace& space, cudaStream_t st) {
  const int64_t dots = a.tokens * a.experts;
  if (dots >= 16 * kNumSMs) return moe_launch_logits<W, 4, 4>(a, first, space, st);
  if (dots >= 4 * kNumSMs) return moe_launch_logits<W, 2, 2>(a, first, space, st);
  return moe_launch_logits<W, 1, 1>(a, first, space, st);
}

static int moe_chunk(const b200q_moe_args& a, int64_t first, cudaStream_t st) {
  const MoeSpace space(a.tokens, a.hidden, a.inner, a.experts, a.top_k);
  if (int rc = a.router_dtype == B200Q_BF16 ? moe_launch_router<__nv_bfloat16>(a, first, space, st) : moe_launch_router<float>(a, first, space, st)) return rc;
  if (moe_fits_tensor_cores(a)) {
    const bool few = a.tokens <= 8, fine = a.out_dtype == B200Q_F32;
    int rc;
    if (a.weight_dtype == B200Q_E4M3) {
      if (fine) rc = few ? moe_launch_fused<true, 8, true>(a, first, space, st) : moe_launch_fused<true, kMoeFineTokens, true>(a, first, space, st);
      else rc = few ? moe_launch_fused<true, 8, false>(a, first, space, st) : moe_launch_fused<true, kMoeGroupTokens, false>(a, first, space, st);
    } else {
      if (fine) rc = few ? moe_launch_fused<false, 8, true>(a, first, space, st) : moe_launch_fused<false, kMoeGroupTokens, true>(a, first, space, st);
      else rc = few ? moe_launch_fused<false, 8, false>(a, first, space, st) : moe_launch_fused<false, kMoeGroupTokens, false>(a, first, space, st);
    }
    if (rc != B200Q_ERR_UNSUPPORTED) return rc;  // (a layout that has no tensor map takes the plain kernels)
  }
  uint8_t* p = static_cast<uint8_t*>(a.workspace);
  const double* logits = reinterpret_cast<const double*>(p + space.logits);
  float *hidden = reinterpret_cast<float*>(p + space.hidden), *outputs = reinterpret_cast<float*>(p + space.outputs);
  const int64_t slots = a.tokens * a.top_k, up = moe_blocks(slots * a.inner), down = moe_blocks(slots * a.hidden);
  const int64_t sum = a.tokens * ((a.hidden + kMoeThreads - 1) / kMoeThreads);
  if (up > INT32_MAX || down > INT32_MAX || sum > INT32_MAX) return B200Q_ERR_TOO_LARGE;
  launch_dependent(moe_choose_kernel, dim3((unsigned)a.tokens), dim3(32), 0, st, a, first, logits);
  B200Q_LAUNCH_CHECK();
  if (up) {  // (a grid of no blocks is an error)
    launch_dependent(moe_plain_up_kernel, dim3((unsigned)up), dim3(kMoeThreads), 0, st, a, hidden);
    B200Q_LAUNCH_CHECK();
  }
  if (down) {
    launch_dependent(moe_plain_down_kernel, dim3((unsigned)down), dim3(kMoeThreads), 0, st, a, static_cast<const float*>(hidden), outputs);
    B200Q_LAUNCH_CHECK();
    launch_dependent(moe_sum_kernel, dim3((unsigned)sum), dim3(kMoeThreads), 0, st, a, static_cast<const float*>(outputs));
    B200Q_LAUNCH_CHECK();
  }
  return B200Q_OK;
}

static bool moe_has_workspace(const b200q_moe_args& a) {
  return a.workspace && a.workspace_bytes >= moe_workspace_bytes_impl(a.tokens, a.hidden, a.inner, a.experts, a.top_k) && reinterpret_cast<uintptr_t>(a.workspace) % 16 == 0;
}

int moe_layer_impl(const b200q_moe_args& a, cudaStream_t st) {
  if (!moe_has_workspace(a)) return B200Q_ERR_BAD_ARGUMENT;
  for (int64_t t = 0; t < a.tokens; t += kMoeChunk) {
    b200q_moe_args c = a;
    c.tokens = a.tokens - t < kMoeChunk ? a.tokens - t : kMoeChunk;
    c.x = static_cast<const uint8_t*>(a.x) + 2 * t * a.x_stride;
    c.out = static_cast<uint8_t*>(a.out) + (a.out_dtype == B200Q_F32 ? 4 : 2) * t * a.hidden;
    c.weights = a.weights + t * a.top_k;
    c.ids = a.ids + t * a.top_k;
    if (int rc = moe_chunk(c, t, st)) return rc;
  }
  return B200Q_OK;
}

// The kernel for 8-bit weights and more tokens than a CTA chooses for by itself, with a wait that is in vain.
int moe_selftest_impl(const b200q_moe_args& a, int lost, cudaStream_t st) {
  if (lost < 0 || lost >= kMoeLostCount || !moe_has_workspace(a)) return B200Q_ERR_BAD_ARGUMENT;
  if (!moe_fits_tensor_cores(a) || a.weight_dtype != B200Q_E4M3 || a.out_dtype != B200Q_BF16 || a.router_dtype != B200Q_BF16 || a.tokens <= 4 * kMoeWarps || a.tokens > kMoeChunk)
    return B200Q_ERR_UNSUPPORTED;
  const MoeSpace space(a.tokens, a.hidden, a.inner, a.experts, a.top_k);
  if (int rc = moe_launch_router<__nv_bfloat16>(a, 0, space, st)) return rc;
  return moe_launch_fused<true, kMoeGroupTokens, false, true>(a, 0, space, st, lost);
}

}  // namespace b200q
