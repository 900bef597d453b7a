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
  size_t logits, x_top, control, h_top, hidden, outputs, parts, bytes;
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

// ---------------------------------------------------------------------------- router
// Sums in fp64: neighbours in the order of the experts may be closer than the rounding of a sum in fp32, and another expert is another answer.
constexpr int kMoeThreads = 256;

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

// A warp has EB experts' rows and TB tokens'.  What the fused kernel wants cleared, and the tokens' largest values, come from here too.
template <typename W, int EB, int TB>
__global__ void __launch_bounds__(kMoeThreads) moe_logits_kernel(const b200q_moe_args a, int64_t first, double* logits, uint32_t* x_top, uint32_t* clear, int clear_words, bool wide) {
  pdl_enter();
  for (int i = blockIdx.x * kMoeThreads + threadIdx.x; i < clear_words; i += gridDim.x * kMoeThreads) clear[i] = 0;
  const int lane = threadIdx.x & 31, tokens = moe_tokens(a, first);
  const int64_t at = (int64_t)blockIdx.x * (kMoeThreads / 32) + (threadIdx.x >> 5), expert_blocks = (a.experts + EB - 1) / EB;
  const int64_t t0 = at / expert_blocks * TB, e0 = (at % expert_blocks) * EB;
  if (t0 >= tokens) return;
  const W* router[EB];
  const __nv_bfloat16* x[TB];
#pragma unroll
  for (int e = 0; e < EB; ++e) router[e] = static_cast<const W*>(a.router) + min(e0 + e, (int64_t)a.experts - 1) * a.hidden;
#pragma unroll
  for (int t = 0; t < TB; ++t) x[t] = static_cast<const __nv_bfloat16*>(a.x) + min(t0 + t, (int64_t)tokens - 1) * a.x_stride;
  double sum[EB][TB] = {};
  uint32_t top[TB] = {};
  for (int64_t i = 8 * lane; i < a.hidden; i += 256) {
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
        for (int t = 0; t < TB; ++t) sum[e][t] += wd * xd[t];
      }
    }
  }
#pragma unroll
  for (int t = 0; t < TB; ++t) {
#pragma unroll
    for (int e = 0; e < EB; ++e) {
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) sum[e][t] += __shfl_xor_sync(0xFFFFFFFFu, sum[e][t], o);
      if (lane == 0 && t0 + t < tokens && e0 + e < a.experts) logits[(t0 + t) * a.experts + e0 + e] = sum[e][t];
    }
    if (e0 == 0 && t0 + t < tokens) {
      top[t] = __reduce_max_sync(0xFFFFFFFFu, top[t]);
      if (lane == 0) x_top[t0 + t] = top[t];
    }
  }
}

// whether (v, i) comes before (w, j) in the order of choice
__device__ __forceinline__ bool moe_before(double v, int i, double w, int j) {
  const bool vn = v != v, wn = w != w;
  if (vn || wn) return vn && wn ? i < j : vn;
  return v > w || (v == w && i < j);
}

// The choice for one token by one warp: lane j has the j-th expert.  top_k rounds of a maximum over the logits, of which a lane has each 32nd.
struct MoeChoice {
  int id;
  float weight;
};
__device__ __forceinline__ MoeChoice moe_choose(const b200q_moe_args& a, const double* logits, bool live, int lane) {
  MoeChoice c = {-1, 0.f};
  if (!live) return c;
  constexpr int kMine = kMoeMaxExperts / 32;
  double mine[kMine];
#pragma unroll
  for (int i = 0; i < kMine; ++i) mine[i] = lane + 32 * i < a.experts ? __ldcg(logits + lane + 32 * i) : 0.0;
  uint32_t taken = 0;  // bit i: expert lane + 32 i
  double first = 0.0, value = 0.0;
  for (int j = 0; j < a.top_k; ++j) {
    double best = 0.0;
    int at = -1;
#pragma unroll
    for (int i = 0; i < kMine; ++i) {
      if (32 * i >= a.experts) break;
      if (lane + 32 * i >= a.experts || (taken >> i & 1u)) continue;
      if (at < 0 || moe_before(mine[i], lane + 32 * i, best, at)) {
        best = mine[i];
        at = lane + 32 * i;
      }
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      const double v = __shfl_xor_sync(0xFFFFFFFFu, best, o);
      const int k = __shfl_xor_sync(0xFFFFFFFFu, at, o);
      if (k >= 0 && (at < 0 || moe_before(v, k, best, at))) {
        best = v;
        at = k;
      }
    }
    if (lane == (at & 31)) taken |= 1u << (at >> 5);
    if (j == 0) first = best;
    if (lane == j) {
      c.id = at;
      value = best;
    }
  }
  // exponents are differences taken in fp64, and small ones exact enough in fp32
  const float p = lane < a.top_k ? expf((float)(value - first)) : 0.f;
  float sum = 0.f;
  if (a.renormalize) {
    sum = p;
  } else {
#pragma unroll
    for (int i = 0; i < kMine; ++i)
      if (lane + 32 * i < a.experts) sum += expf((float)(mine[i] - first));
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xFFFFFFFFu, sum, o);
  c.weight = p / sum;
  return c;
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
  if (lane == 0) hidden[at] = moe_silu(g) * u;
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
// terms, a column each, scaled by powers of two: bf16 values of a token two terms (8 bits, which is all they have), h three (12 bits).  The
// weights then go from global memory to the tensor core as they are, by TMA alone; f16 operands would want every weight converted in
// registers first.
//
// One persistent CTA per SM; the list of (expert, 32 tokens of it at most), weight rows and steps of 128 bytes of a row is cut into equal runs for the
// CTAs, so that few experts and ragged sizes load every SM alike.  A row tile that several CTAs have a part of is summed by the one that finishes
// last, in the CTAs' order.  Both products are one stream of weights: while the last tiles of the first product are finished, and all CTAs wait for them, the
// second one's weights fill the ring.
//   warp 0: weights, by TMA     warp 1: MMAs     warps 2-5: tokens' terms into shared memory     warps 6-9: results
constexpr int kMoeWarps = 10;
constexpr int kMoeErrWeights = 821, kMoeErrTokens = 822, kMoeErrMma = 823, kMoeErrResults = 824, kMoeErrGrid = 825;  // status codes: a wait ran out
constexpr int kMoeGroupTokens = 32;     // of an expert, at a time
constexpr int kMoeSubBytes = 128 * 128;  // a weight tile: 128 rows of 128 bytes; a step has two (gate and up, or 256 outputs)
constexpr int kMoeMostDim = 65536;
constexpr uint32_t kMoeGridPolls = 1u << 23;

struct MoeControl {  // cleared by the router's kernel
  uint32_t chosen, up_done, down_done, unused;
  uint32_t joins[2][kNumSMs];  // parts that have arrived, by the CTA that has the first one
};

template <bool FP8, int MAXN>
struct MoeTile {
  static constexpr int kUpTerms = FP8 ? 2 : 1, kDownTerms = FP8 ? 3 : 2;
  static constexpr int kCols = (kDownTerms * MAXN + 15) / 16 * 16;  // columns of an accumulator
  static constexpr int kTokenBytes = kCols * 128;
  static constexpr int kStage = 2 * kMoeSubBytes + kTokenBytes;
  static constexpr int kStages = 200 * 1024 / kStage < 5 ? 200 * 1024 / kStage : 5;
  static constexpr int kTmem = 4 * kCols <= 64 ? 64 : 4 * kCols <= 128 ? 128 : 4 * kCols <= 256 ? 256 : 512;  // two accumulators of two tiles
  static constexpr int kStep = FP8 ? 128 : 64;  // values of K in a step
  static constexpr int kPart = 2 * MAXN * 128;  // floats of a partial result: [tile][token][row]
  static_assert(kTokenBytes % 1024 == 0, "tiles lie on boundaries of the swizzle");
};

struct MoeFused {
  const double* logits;
  const uint32_t* x_top;   // bits of max |x| per token
  uint32_t* h_top;         // bits of max |h| per slot
  float *hidden, *outputs;  // [slots][inner], [slots][hidden]: slots in the order of experts
  float* parts;            // [grid][2][kPart]
  MoeControl* control;
  int* status;
  int up_tiles, up_steps, down_tiles, down_steps;
};

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

__device__ __forceinline__ uint32_t moe_ld_acquire(const uint32_t* p) {
  uint32_t v;
  asm volatile("ld.acquire.gpu.global.u32 %0, [%1];" : "=r"(v) : "l"(p) : "memory");
  return v;
}
__device__ __forceinline__ void moe_add_release(uint32_t* p) { asm volatile("red.release.gpu.global.add.u32 [%0], 1;" ::"l"(p) : "memory"); }
// until all CTAs have arrived (one warp); false when they do not
__device__ __forceinline__ bool moe_grid_wait(const uint32_t* p, uint32_t want, volatile int* abort_flag, int* status) {
  for (uint32_t i = 0; i < kMoeGridPolls; ++i) {
    if (__all_sync(0xFFFFFFFFu, moe_ld_acquire(p) >= want)) return true;
    if ((i & 63u) == 63u && __any_sync(0xFFFFFFFFu, *abort_flag)) return false;
    if (i > 64u) __nanosleep(64);
  }
  *abort_flag = 1;
  atomicCAS(status, 0, kMoeErrGrid);
  return false;
}
__device__ __forceinline__ void moe_tmem_ld8(uint32_t taddr, float (&v)[8]) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
               : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]), "=f"(v[4]), "=f"(v[5]), "=f"(v[6]), "=f"(v[7])
               : "r"(taddr)
               : "memory");
}

// A CTA's run of the list of steps of a product, and the pieces of tiles in it.
struct MoeRun {
  int steps, begin, end;  // steps of a tile; of the run
  int each, more;
  __device__ __forceinline__ MoeRun(int groups, int tiles, int steps_, int cta, int ctas) {
    steps = steps_;
    const int total = groups * tiles * steps;
    each = total / ctas;
    more = total - each * ctas;
    begin = at(cta);
    end = at(cta + 1);
  }
  __device__ __forceinline__ int at(int cta) const { return cta * each + min(cta, more); }
  __device__ __forceinline__ int cta_of(int step) const {
    const int longer = more * (each + 1);
    return step < longer ? step / (each + 1) : more + (step - longer) / each;
  }
};

template <bool FP8, int MAXN>
__global__ void __launch_bounds__(32 * kMoeWarps, 1)
    moe_fused_kernel(const __grid_constant__ CUtensorMap map_up, const __grid_constant__ CUtensorMap map_down, const b200q_moe_args a, int64_t first,
                     const MoeFused w) {
  using Tile = MoeTile<FP8, MAXN>;
  constexpr int kStages = Tile::kStages, kSteps = Tile::kStep;
  constexpr int kMostSlots = MAXN == 8 ? 8 * kMoeMaxTopK : (int)kMoeChunk * kMoeMaxTopK;
  constexpr int kMostGroups = MAXN == 8 ? 8 * kMoeMaxTopK : kMoeMaxExperts + kMostSlots / kMoeGroupTokens;
  constexpr int kMaskWords = MAXN == 8 ? 1 : (int)kMoeChunk / 32;
  extern __shared__ __align__(1024) uint8_t s_raw[];
  uint8_t* const s_ring = s_raw + (0u - ptx::smem_u32(s_raw) & 1023u);
  __shared__ uint16_t s_slot_of[kMostSlots], s_token_of[kMostSlots];  // slot of (token, j); token of a slot
  __shared__ uint16_t s_group_expert[kMostGroups], s_group_slot[kMostGroups];
  __shared__ uint8_t s_group_tokens[kMostGroups];
  __shared__ __align__(8) uint64_t s_bars[3 * kStages + 4];
  __shared__ uint32_t s_tmem;
  __shared__ int s_abort, s_groups, s_last, s_scan[2][kMoeWarps];
  // before the ring is in use: a bit per token of each expert
  uint32_t* const s_mask = reinterpret_cast<uint32_t*>(s_ring);
  int16_t* const s_ids = reinterpret_cast<int16_t*>(s_ring + sizeof(uint32_t) * kMoeMaxExperts * kMaskWords);  // [tokens][top_k]

  const int tid = threadIdx.x, lane = tid & 31, warp = ptx::uniform_warp_index();
  const int cta = blockIdx.x, ctas = gridDim.x;
  const uint32_t bar_weights = ptx::smem_u32(s_bars), bar_tokens = bar_weights + 8 * kStages, bar_empty = bar_tokens + 8 * kStages;
  const uint32_t bar_full = bar_empty + 8 * kStages, bar_free = bar_full + 16;  // of the two accumulators
  const uint32_t ring = ptx::smem_u32(s_ring);
  if (tid == 0) {
    for (int i = 0; i < kStages; ++i) {
      ptx::mbar_init(bar_weights + 8 * i, 1);
      ptx::mbar_init(bar_tokens + 8 * i, 4);
      ptx::mbar_init(bar_empty + 8 * i, 1);
    }
    for (int i = 0; i < 2; ++i) {
      ptx::mbar_init(bar_full + 8 * i, 1);
      ptx::mbar_init(bar_free + 8 * i, 4);
    }
    s_abort = 0;
    ptx::fence_barrier_init();
    ptx::tma_prefetch_desc(&map_up);
    ptx::tma_prefetch_desc(&map_down);
  }
  if (warp == 1) {
    ptx::tmem_alloc(ptx::smem_u32(&s_tmem), Tile::kTmem);
    ptx::tmem_relinquish();
  }
  pdl_enter();

  // ---- the choice: by every CTA for itself where a warp has two tokens at most, else a token per warp of the grid
  const int tokens = (int)a.tokens, live = moe_tokens(a, first), top_k = a.top_k, slots = live * top_k;
  bool ok = true;
  if (MAXN == 8) {
    for (int t = warp; t < tokens; t += kMoeWarps) {
      const MoeChoice c = moe_choose(a, w.logits + (int64_t)t * a.experts, t < live, lane);
      if (lane < top_k) {
        s_ids[t * top_k + lane] = (int16_t)c.id;
        if (cta == 0) moe_store_choice(a, t, lane, c);
      }
    }
    for (int i = tid; i < a.experts * kMaskWords; i += 32 * kMoeWarps) s_mask[i] = 0;
    __syncthreads();
  } else {
    for (int t = warp * ctas + cta; t < tokens; t += kMoeWarps * ctas) {
      const MoeChoice c = moe_choose(a, w.logits + (int64_t)t * a.experts, t < live, lane);
      if (lane < top_k) moe_store_choice(a, t, lane, c);
    }
    for (int i = tid; i < a.experts * kMaskWords; i += 32 * kMoeWarps) s_mask[i] = 0;
    __threadfence();
    __syncthreads();
    if (tid == 0) moe_add_release(&w.control->chosen);
    ok = moe_grid_wait(&w.control->chosen, (uint32_t)ctas, &s_abort, w.status);
    for (int i = tid; i < slots; i += 32 * kMoeWarps) s_ids[i] = (int16_t)__ldcg(a.ids + i);
    __syncthreads();
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
        int slot = before & 0xFFFF, group = before >> 16;
        for (int i = 0; i < n; i += MAXN, ++group) {
          s_group_expert[group] = (uint16_t)e;
          s_group_slot[group] = (uint16_t)(slot + i);
          s_group_tokens[group] = (uint8_t)min(n - i, MAXN);
        }
        for (int i = 0; i < kMaskWords; ++i)
          for (uint32_t m = s_mask[e * kMaskWords + i]; m; m &= m - 1, ++slot) s_token_of[slot] = (uint16_t)(32 * i + __ffs(m) - 1);
      }
    }
    if (tid == 0) s_groups = groups_before;
  }
  __syncthreads();
  // slot of (t, j): the expert's first slot and the tokens before t.  (The slots' order is in s_token_of; found by the expert's group.)
  for (int g = tid; g < s_groups; g += 32 * kMoeWarps) {
    const int e = s_group_expert[g], s0 = s_group_slot[g];
    for (int i = 0; i < s_group_tokens[g]; ++i) {
      const int t = s_token_of[s0 + i];
      for (int j = 0; j < top_k; ++j)
        if (s_ids[t * top_k + j] == e) s_slot_of[t * top_k + j] = (uint16_t)(s0 + i);
    }
  }
  ptx::tc_fence_before();
  __syncthreads();
  ptx::tc_fence_after();
  // (the ring's first bytes were written and read by ordinary accesses; the copies come through another path)
  ptx::fence_proxy_async_smem();
  __syncthreads();
  const uint32_t tmem = s_tmem;
  const int groups = s_groups;
  const MoeRun runs[2] = {MoeRun(groups, w.up_tiles, w.up_steps, cta, ctas), MoeRun(groups, w.down_tiles, w.down_steps, cta, ctas)};

  if (!ok) {
    // (a CTA did not come: nothing is in flight, and nobody goes on)
  } else if (warp == 0) {
    // ------------------------------------------------------------ weights
    uint32_t stage = 0, phase = 0;
    int made = 0;
    for (int product = 0; product < 2 && ok; ++product) {
      const MoeRun& run = runs[product];
      const int tiles = product ? w.down_tiles : w.up_tiles;
      int tile = run.begin / run.steps, k = run.begin - tile * run.steps;
      for (int at = run.begin; at < run.end; ++at) {
        ok = ptx::mbar_wait_uniform(bar_empty + 8 * stage, phase ^ 1, &s_abort, w.status, kMoeErrWeights);
        if (!ok) break;
        const int group = tile / tiles, row = tile - group * tiles, e = s_group_expert[group];
        if (ptx::elect_one()) {
          const uint32_t bar = bar_weights + 8 * stage, dst = ring + stage * Tile::kStage;
          ptx::mbar_arrive_expect_tx(bar, 2 * kMoeSubBytes);
          if (product == 0) {
            ptx::tma_load_3d(dst, &map_up, bar, k * kSteps, row * 128, 2 * e);
            ptx::tma_load_3d(dst + kMoeSubBytes, &map_up, bar, k * kSteps, row * 128, 2 * e + 1);
          } else {
            ptx::tma_load_3d(dst, &map_down, bar, k * kSteps, row * 256, e);
            ptx::tma_load_3d(dst + kMoeSubBytes, &map_down, bar, k * kSteps, row * 256 + 128, e);
          }
        }
        ++made;
        if (++k == run.steps) {
          k = 0;
          ++tile;
        }
        if (++stage == kStages) {
          stage = 0;
          phase ^= 1;
        }
      }
    }
    if (!ok) {  // the copies in flight are waited for, as far as they come
      for (int i = 0; i < min(made, kStages); ++i) {
        phase ^= stage == 0;
        stage = stage == 0 ? kStages - 1 : stage - 1;
        for (int k = 0; k < 4096 && !ptx::mbar_try_wait(bar_weights + 8 * stage, phase); ++k) __nanosleep(64);
      }
    }
  } else if (warp == 1) {
    // ------------------------------------------------------------ products
    uint32_t stage = 0, phase = 0;
    int pieces = 0;
    const uint64_t a0 = ptx::smem_desc_k_sw128(ring), b0 = ptx::smem_desc_k_sw128(ring + 2 * kMoeSubBytes);
    for (int product = 0; product < 2 && ok; ++product) {
      const MoeRun& run = runs[product];
      const int tiles = product ? w.down_tiles : w.up_tiles, terms = product ? Tile::kDownTerms : Tile::kUpTerms;
      for (int at = run.begin; at < run.end && ok; ++pieces) {
        const int tile = run.begin < run.end ? at / run.steps : 0, end = min(run.end, (tile + 1) * run.steps);
        const int cols = (terms * ((s_group_tokens[tile / tiles] + 7) / 8 * 8) + 15) / 16 * 16;
        const uint32_t idesc = FP8 ? ptx::umma_idesc(0, 0, 128, cols) : ptx::umma_idesc(1, 1, 128, cols);
        const uint32_t acc = pieces & 1, d = tmem + acc * 2 * Tile::kCols;
        ok = ptx::mbar_wait_uniform(bar_free + 8 * acc, ((pieces >> 1) & 1) ^ 1, &s_abort, w.status, kMoeErrMma);
        if (!ok) break;
        ptx::tc_fence_after();
        for (int k = 0; at < end; ++at, ++k) {
          ok = ptx::mbar_wait2_uniform(bar_weights + 8 * stage, phase, bar_tokens + 8 * stage, phase, &s_abort, w.status, kMoeErrMma);
          if (!ok) break;
          ptx::tc_fence_after();
          const uint64_t off = stage * (uint32_t)(Tile::kStage >> 4);
          if (ptx::elect_one()) {
#pragma unroll
            for (int sub = 0; sub < 2; ++sub) {
              if (FP8) ptx::umma_f8_x4(d + sub * Tile::kCols, a0 + off + sub * (kMoeSubBytes >> 4), b0 + off, idesc, k != 0, 2, 2);
              else ptx::umma_f16_x4(d + sub * Tile::kCols, a0 + off + sub * (kMoeSubBytes >> 4), b0 + off, idesc, k != 0, 2, 2);
            }
            ptx::umma_commit(bar_empty + 8 * stage);
            if (at + 1 == end) ptx::umma_commit(bar_full + 8 * acc);
          }
          __syncwarp();
          if (++stage == kStages) {
            stage = 0;
            phase ^= 1;
          }
        }
      }
    }
  } else if (warp < 6) {
    // ------------------------------------------------------------ tokens
    constexpr int kPieces = MAXN * (kSteps / 8) / 128 > 0 ? MAXN * (kSteps / 8) / 128 : 1;  // of eight values, per thread
    const int lt = tid - 64;
    uint32_t stage = 0, phase = 0;
    for (int product = 0; product < 2 && ok; ++product) {
      const MoeRun& run = runs[product];
      if (product == 1) {
        ok = moe_grid_wait(&w.control->up_done, (uint32_t)ctas, &s_abort, w.status);
        if (!ok) break;
      }
      const int tiles = product ? w.down_tiles : w.up_tiles;
      const int64_t depth = product ? a.inner : a.hidden;
      int tile = run.begin / run.steps, k = run.begin - tile * run.steps, group = tile / tiles;
      uint4 raw[kPieces][2];
      float factor[kPieces];
      const uint4 zero = make_uint4(0, 0, 0, 0);
      // piece i of a thread: token j's values 8 c ... of a step
      auto token_of = [&](int i) { return (lt + 128 * i) / (kSteps / 8); };
      auto fetch = [&](int group, int k) {
        const int n = s_group_tokens[group], slot = s_group_slot[group];
#pragma unroll
        for (int i = 0; i < kPieces; ++i) {
          const int j = token_of(i);
          const int64_t at = (int64_t)k * kSteps + (lt + 128 * i) % (kSteps / 8) * 8;
          raw[i][0] = raw[i][1] = zero;
          if (j >= n || at >= depth) continue;
          if (product == 0) {
            raw[i][0] = __ldg(reinterpret_cast<const uint4*>(static_cast<const __nv_bfloat16*>(a.x) + s_token_of[slot + j] * a.x_stride + at));
          } else {
            const uint4* p = reinterpret_cast<const uint4*>(w.hidden + (int64_t)(slot + j) * a.inner + at);
            raw[i][0] = __ldcg(p);
            raw[i][1] = __ldcg(p + 1);
          }
        }
      };
      auto factors = [&](int group) {
        const int n = s_group_tokens[group], slot = s_group_slot[group];
#pragma unroll
        for (int i = 0; i < kPieces; ++i) {
          const int j = token_of(i);
          factor[i] = 1.f;
          if (FP8 && j < n) factor[i] = moe_up_factor(product ? __ldcg(w.h_top + slot + j) : __ldcg(w.x_top + s_token_of[slot + j]));
        }
      };
      if (run.begin < run.end) {
        factors(group);
        fetch(group, k);
      }
      for (int at = run.begin; at < run.end; ++at) {
        const int n8 = (s_group_tokens[group] + 7) / 8 * 8;
        // the terms, while the stage is still in use
        uint2 low[kPieces][FP8 ? 3 : 1];
        uint4 wide[kPieces][FP8 ? 1 : 2];
#pragma unroll
        for (int i = 0; i < kPieces; ++i) {
          float v[8];
          if (product == 0) {
            if (!FP8) {
              wide[i][0] = raw[i][0];
              continue;
            }
            const uint32_t u[4] = {raw[i][0].x, raw[i][0].y, raw[i][0].z, raw[i][0].w};
#pragma unroll
            for (int c = 0; c < 4; ++c) {
              v[2 * c] = __uint_as_float(u[c] << 16) * factor[i];
              v[2 * c + 1] = __uint_as_float(u[c] & 0xFFFF0000u) * factor[i];
            }
          } else {
            const uint32_t u[8] = {raw[i][0].x, raw[i][0].y, raw[i][0].z, raw[i][0].w, raw[i][1].x, raw[i][1].y, raw[i][1].z, raw[i][1].w};
#pragma unroll
            for (int c = 0; c < 8; ++c) {
              v[c] = __uint_as_float(u[c]) * factor[i];
              if (FP8 && !(fabsf(v[c]) <= 3.4e38f)) v[c] = __int_as_float(0x7FC00000);  // (e4m3 has no infinity, and would make it 448)
            }
          }
          if (FP8) {
            if (product == 0) {
              uint2 two[2];
              moe_terms_fp8<2>(v, two);
              low[i][0] = two[0];
              low[i][FP8 ? 1 : 0] = two[1];
            } else {
              uint2 three[3];
              moe_terms_fp8<3>(v, three);
#pragma unroll
              for (int c = 0; c < 3; ++c) low[i][FP8 ? c : 0] = three[c];
            }
          } else {
            uint32_t hi[4], lo[4];
#pragma unroll
            for (int c = 0; c < 4; ++c) {
              hi[c] = pack_bf16x2(v[2 * c], v[2 * c + 1]);
              lo[c] = pack_bf16x2(v[2 * c] - __uint_as_float(hi[c] << 16), v[2 * c + 1] - __uint_as_float(hi[c] & 0xFFFF0000u));
            }
            wide[i][0] = make_uint4(hi[0], hi[1], hi[2], hi[3]);
            wide[i][FP8 ? 0 : 1] = make_uint4(lo[0], lo[1], lo[2], lo[3]);
          }
        }
        const int here = s_group_tokens[group];
        // the next step's values are asked for
        int next_k = k + 1, next_tile = tile;
        if (next_k == run.steps) {
          next_k = 0;
          ++next_tile;
        }
        const int next_group = next_tile / tiles;
        if (at + 1 < run.end) {
          if (next_group != group) factors(next_group);
          fetch(next_group, next_k);
        }
        ok = ptx::mbar_wait_uniform(bar_empty + 8 * stage, phase ^ 1, &s_abort, w.status, kMoeErrTokens);
        if (!ok) break;
        const uint32_t dst = ring + stage * Tile::kStage + 2 * kMoeSubBytes;
#pragma unroll
        for (int i = 0; i < kPieces; ++i) {
          const int j = token_of(i), c = (lt + 128 * i) % (kSteps / 8);
          if (j >= here) continue;
          const int terms = product ? Tile::kDownTerms : Tile::kUpTerms;
#pragma unroll
          for (int t = 0; t < Tile::kDownTerms; ++t) {
            if (t >= terms) break;
            const uint32_t row = (uint32_t)(t * n8 + j);
            if (FP8) {
              const uint32_t to = dst + row * 128 + ((((uint32_t)c >> 1) ^ (row & 7)) << 4) + (c & 1) * 8;
              asm volatile("st.shared.v2.u32 [%0], {%1, %2};" ::"r"(to), "r"(low[i][FP8 ? t : 0].x), "r"(low[i][FP8 ? t : 0].y) : "memory");
            } else {
              const uint32_t to = dst + row * 128 + (((uint32_t)c ^ (row & 7)) << 4);
              const uint4 x = wide[i][FP8 ? 0 : t];
              asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(to), "r"(x.x), "r"(x.y), "r"(x.z), "r"(x.w) : "memory");
            }
          }
        }
        ptx::fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) ptx::mbar_arrive(bar_tokens + 8 * stage);
        k = next_k;
        tile = next_tile;
        group = next_group;
        if (++stage == kStages) {
          stage = 0;
          phase ^= 1;
        }
      }
    }
  } else {
    // ------------------------------------------------------------ results
    const int row = 32 * (warp & 3) + lane;  // of a tile: the lane of tensor memory that this thread reads
    const uint32_t lane_base = (uint32_t)(32 * (warp & 3)) << 16;
    auto barrier = [] { ptx::named_bar_sync(1, 128); };
    int pieces = 0;
    auto results_of = [&](auto which) {
      constexpr int product = decltype(which)::value, terms = product ? Tile::kDownTerms : Tile::kUpTerms;
      const MoeRun& run = runs[product];
      const int tiles = product ? w.down_tiles : w.up_tiles;
      for (int at = run.begin; at < run.end; ++pieces) {
        const int tile = at / run.steps, tile0 = tile * run.steps, end = min(run.end, tile0 + run.steps);
        const int group = tile / tiles, row_tile = tile - group * tiles, e = s_group_expert[group], slot = s_group_slot[group], n = s_group_tokens[group];
        const int n8 = (n + 7) / 8 * 8;
        const uint32_t acc = pieces & 1, d = tmem + acc * 2 * Tile::kCols + lane_base;
        ok = ptx::mbar_wait_uniform(bar_full + 8 * acc, (pieces >> 1) & 1, &s_abort, w.status, kMoeErrResults);
        if (!ok) return;
        ptx::tc_fence_after();
        const bool whole = at == tile0 && end == tile0 + run.steps;
        // of the rows that this thread has: the two tiles' scales
        const int64_t r0 = product ? row_tile * 256 + row : row_tile * 128 + row, r1 = product ? r0 + 128 : r0;
        const int64_t width = product ? a.hidden : a.inner;
        float scale[2] = {1.f, 1.f};
        const float* scales = product ? a.down_scale : a.gate_up_scale;
        if (scales) {
          if (r0 < width) scale[0] = scales[product ? e * a.hidden + r0 : e * 2 * a.inner + r0];
          if (r1 < width) scale[1] = scales[product ? e * a.hidden + r1 : e * 2 * a.inner + a.inner + r1];
        }
        auto finish = [&](int j, float v0, float v1) {  // token j's values of the two tiles
          if (product == 0) {
            const float back = FP8 ? moe_down_factor(__ldcg(w.x_top + s_token_of[slot + j])) : 1.f;
            const float g = v0 * back * scale[0], u = v1 * back * scale[1];
            const float h = r0 < width ? moe_silu(g) * u : 0.f;
            if (r0 < width) __stcg(w.hidden + (int64_t)(slot + j) * a.inner + r0, h);
            if (FP8) {
              const uint32_t top = __reduce_max_sync(0xFFFFFFFFu, __float_as_uint(h) & 0x7FFFFFFFu);
              if (lane == 0) atomicMax(w.h_top + slot + j, top);
            }
          } else {
            const float back = FP8 ? moe_down_factor(__ldcg(w.h_top + slot + j)) : 1.f;
            if (r0 < width) __stcg(w.outputs + (int64_t)(slot + j) * a.hidden + r0, v0 * back * scale[0]);
            if (r1 < width) __stcg(w.outputs + (int64_t)(slot + j) * a.hidden + r1, v1 * back * scale[1]);
          }
        };
        float* part = w.parts + ((int64_t)cta * 2 + (at == tile0 ? 1 : 0)) * Tile::kPart;
        for (int j0 = 0; j0 < n8; j0 += 8) {
          float v[2][8];
#pragma unroll
          for (int sub = 0; sub < 2; ++sub) {
            float term[terms][8];
#pragma unroll
            for (int t = 0; t < terms; ++t) moe_tmem_ld8(d + sub * Tile::kCols + t * n8 + j0, term[t]);
            ptx::tmem_ld_wait();
#pragma unroll
            for (int i = 0; i < 8; ++i) {
              v[sub][i] = term[terms - 1][i];
#pragma unroll
              for (int t = terms - 2; t >= 0; --t) v[sub][i] = term[t][i] + (FP8 ? 1.f / 32.f : 1.f) * v[sub][i];
            }
          }
          if (whole) {
#pragma unroll
            for (int i = 0; i < 8; ++i)
              if (j0 + i < n) finish(j0 + i, v[0][i], v[1][i]);
          } else {
#pragma unroll
            for (int i = 0; i < 8; ++i)
              if (j0 + i < n) {
                __stcg(part + (j0 + i) * 128 + row, v[0][i]);
                __stcg(part + (MAXN + j0 + i) * 128 + row, v[1][i]);
              }
          }
        }
        ptx::tc_fence_before();
        __syncwarp();
        if (lane == 0) ptx::mbar_arrive(bar_free + 8 * acc);
        if (!whole) {
          const int c0 = run.cta_of(tile0), c1 = run.cta_of(tile0 + run.steps - 1);
          __threadfence();
          barrier();
          if (warp == 6 && lane == 0) s_last = atomicAdd(&w.control->joins[product][c0], 1u) == (uint32_t)(c1 - c0);
          barrier();
          if (s_last) {
            __threadfence();
            for (int j = 0; j < n; ++j) {
              float v0 = 0.f, v1 = 0.f;
              for (int c = c0; c <= c1; ++c) {
                const float* p = w.parts + ((int64_t)c * 2 + (c == c0 ? 1 : 0)) * Tile::kPart;
                v0 += __ldcg(p + j * 128 + row);
                v1 += __ldcg(p + (MAXN + j) * 128 + row);
              }
              finish(j, v0, v1);
            }
          }
        }
        at = end;
      }
      __threadfence();
      barrier();
      if (warp == 6 && lane == 0) moe_add_release(product ? &w.control->down_done : &w.control->up_done);
    };
    results_of(std::integral_constant<int, 0>());
    if (ok) results_of(std::integral_constant<int, 1>());
    // ---- the weighted sums
    if (ok) ok = moe_grid_wait(&w.control->down_done, (uint32_t)ctas, &s_abort, w.status);
    const int et = tid - 192;
    const int64_t quads = (a.hidden + 3) / 4;
    for (int64_t i = (int64_t)cta * 128 + et; i < tokens * quads; i += (int64_t)ctas * 128) {
      const int t = (int)(i / quads);
      const int64_t c = (i - t * quads) * 4;
      float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
      if (t < live)
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
  parts = moe_align(outputs + sizeof(float) * slots * (size_t)h);
  const int group = t <= 8 ? 8 : kMoeGroupTokens;
  bytes = moe_align(parts + sizeof(float) * 2 * (size_t)kNumSMs * 2 * group * 128);
}

size_t moe_workspace_bytes_impl(int64_t tokens, int64_t hidden, int64_t inner, int experts, int top_k) {
  return MoeSpace(tokens, hidden, inner, experts, top_k).bytes;
}

static int64_t moe_blocks(int64_t warps) { return (warps + kMoeThreads / 32 - 1) / (kMoeThreads / 32); }

static bool moe_fits_tensor_cores(const b200q_moe_args& a) {
  const int64_t size = a.weight_dtype == B200Q_BF16 ? 2 : 1;
  if (a.force_plain || a.hidden <= 0 || a.inner <= 0 || a.hidden > kMoeMostDim || a.inner > kMoeMostDim || a.hidden * size % 16 || a.inner * size % 16) return false;
  if (a.tokens > 1 && a.x_stride % 8) return false;
  for (const void* p : {a.x, a.gate_up, a.down, static_cast<const void*>(a.out)})
    if (reinterpret_cast<uintptr_t>(p) % 16) return false;
  return true;
}

// [planes][rows][depth] of weights in boxes of 128 rows of 128 bytes
static int moe_map(CUtensorMap* map, const void* base, bool fp8, int64_t depth, int64_t rows, int64_t planes) {
  EncodeTiledFn enc = get_encode_fn();
  if (!enc) return B200Q_ERR_CUDA;
  const cuuint64_t size = fp8 ? 1 : 2;
  const cuuint64_t dims[3] = {(cuuint64_t)depth, (cuuint64_t)rows, (cuuint64_t)planes}, strides[2] = {depth * size, rows * depth * size};
  const cuuint32_t box[3] = {fp8 ? 128u : 64u, 128, 1}, step[3] = {1, 1, 1};
  const CUresult r = enc(map, fp8 ? CU_TENSOR_MAP_DATA_TYPE_UINT8 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, const_cast<void*>(base), dims, strides, box, step,
                         CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return r == CUDA_SUCCESS ? B200Q_OK : B200Q_ERR_UNSUPPORTED;
}

template <bool FP8, int MAXN>
static int moe_launch_fused(const b200q_moe_args& a, int64_t first, const MoeSpace& space, cudaStream_t st) {
  using Tile = MoeTile<FP8, MAXN>;
  auto kernel = moe_fused_kernel<FP8, MAXN>;
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
  (void)cudaLaunchKernelEx(&cfg, kernel, map_up, map_down, a, first, w);
  B200Q_LAUNCH_CHECK();
  return B200Q_OK;
}

template <typename W, int EB, int TB>
static int moe_launch_logits(const b200q_moe_args& a, int64_t first, const MoeSpace& space, cudaStream_t st) {
  uint8_t* p = static_cast<uint8_t*>(a.workspace);
  const int64_t warps = ((a.experts + EB - 1) / EB) * ((a.tokens + TB - 1) / TB);
  bool wide = a.hidden % 8 == 0 && (a.tokens == 1 || a.x_stride % 8 == 0);
  for (const void* q : {a.x, a.router}) wide = wide && reinterpret_cast<uintptr_t>(q) % 16 == 0;
  launch_dependent(moe_logits_kernel<W, EB, TB>, dim3((unsigned)moe_blocks(warps)), dim3(kMoeThreads), 0, st, a, first, reinterpret_cast<double*>(p + space.logits),
                   reinterpret_cast<uint32_t*>(p + space.x_top), reinterpret_cast<uint32_t*>(p + space.control), space.clear_words, wide);
  B200Q_LAUNCH_CHECK();
  return B200Q_OK;
}
template <typename W>
static int moe_launch_router(const b200q_moe_args& a, int64_t first, const MoeSpace& space, cudaStream_t st) {
  const int64_t dots = a.tokens * a.experts;
  if (dots >= 16 * 4 * kNumSMs) return moe_launch_logits<W, 4, 4>(a, first, space, st);
  if (dots >= 4 * 4 * kNumSMs) return moe_launch_logits<W, 2, 2>(a, first, space, st);
  return moe_launch_logits<W, 1, 1>(a, first, space, st);
}

static int moe_chunk(const b200q_moe_args& a, int64_t first, cudaStream_t st) {
  const MoeSpace space(a.tokens, a.hidden, a.inner, a.experts, a.top_k);
  if (int rc = a.router_dtype == B200Q_BF16 ? moe_launch_router<__nv_bfloat16>(a, first, space, st) : moe_launch_router<float>(a, first, space, st)) return rc;
  if (moe_fits_tensor_cores(a)) {
    int rc;
    if (a.weight_dtype == B200Q_E4M3) rc = a.tokens <= 8 ? moe_launch_fused<true, 8>(a, first, space, st) : moe_launch_fused<true, kMoeGroupTokens>(a, first, space, st);
    else rc = a.tokens <= 8 ? moe_launch_fused<false, 8>(a, first, space, st) : moe_launch_fused<false, kMoeGroupTokens>(a, first, space, st);
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

int moe_layer_impl(const b200q_moe_args& a, cudaStream_t st) {
  if (!a.workspace || a.workspace_bytes < moe_workspace_bytes_impl(a.tokens, a.hidden, a.inner, a.experts, a.top_k) ||
      reinterpret_cast<uintptr_t>(a.workspace) % 16)
    return B200Q_ERR_BAD_ARGUMENT;
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

}  // namespace b200q
