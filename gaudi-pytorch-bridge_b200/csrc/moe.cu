// A mixture-of-experts layer for a few tokens: router, choice of the experts, their gated products, and the weighted sum.
#include "layer.cuh"

namespace b200q {

constexpr int64_t kMoeChunk = 256;  // tokens taken at a time
constexpr size_t moe_align(size_t n) { return (n + 255) / 256 * 256; }

// Where the parts of the workspace lie.  Slot t * top_k + j belongs to token t's j-th expert.
struct MoeSpace {
  size_t logits, hidden, outputs, bytes;
  MoeSpace(int64_t tokens, int64_t h, int64_t f, int experts, int top_k) {
    const size_t t = (size_t)(tokens < kMoeChunk ? tokens : kMoeChunk), slots = t * (size_t)top_k;
    logits = 0;
    hidden = moe_align(logits + sizeof(double) * t * (size_t)experts);
    outputs = moe_align(hidden + sizeof(float) * slots * (size_t)f);
    bytes = moe_align(outputs + sizeof(float) * slots * (size_t)h);
  }
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

__global__ void __launch_bounds__(kMoeThreads) moe_logits_kernel(const b200q_moe_args a, int64_t first, double* logits) {
  pdl_enter();
  const int lane = threadIdx.x & 31;
  const int64_t at = (int64_t)blockIdx.x * (kMoeThreads / 32) + (threadIdx.x >> 5);
  if (at >= a.tokens * a.experts) return;
  const int64_t t = at / a.experts, e = at - t * a.experts;
  if (t >= moe_tokens(a, first)) return;
  double sum = 0.0;
  for (int64_t i = lane; i < a.hidden; i += 32) {
    const float w = a.router_dtype == B200Q_F32 ? static_cast<const float*>(a.router)[e * a.hidden + i]
                                                : __bfloat162float(static_cast<const __nv_bfloat16*>(a.router)[e * a.hidden + i]);
    sum += (double)w * (double)moe_x(a, t, i);
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xFFFFFFFFu, sum, o);
  if (lane == 0) logits[at] = sum;
}

// whether (v, i) comes before (w, j) in the order of choice
__device__ __forceinline__ bool moe_before(double v, int i, double w, int j) {
  const bool vn = v != v, wn = w != w;
  if (vn || wn) return vn && wn ? i < j : vn;
  return v > w || (v == w && i < j);
}

// The choice for one token by one warp: top_k rounds of a maximum over the logits.
__device__ __forceinline__ void moe_choose(const b200q_moe_args& a, int64_t t, const double* logits, int lane) {
  uint32_t taken = 0;  // bit i: expert lane + 32 i
  double first = 0.0, mine = 0.0;
  int chosen = -1;  // of round `lane`
  for (int j = 0; j < a.top_k; ++j) {
    double best = 0.0;
    int at = -1;
    for (int i = 0; lane + 32 * i < a.experts; ++i) {
      if (taken >> i & 1u) continue;
      const double v = __ldcg(logits + lane + 32 * i);
      if (at < 0 || moe_before(v, lane + 32 * i, best, at)) {
        best = v;
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
      chosen = at;
      mine = best;
    }
  }
  // exponents are differences taken in fp64, and small ones exact enough in fp32
  float p = lane < a.top_k ? expf((float)(mine - first)) : 0.f, sum = 0.f;
  if (a.renormalize) {
    sum = p;
  } else {
    for (int e = lane; e < a.experts; e += 32) sum += expf((float)(__ldcg(logits + e) - first));
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xFFFFFFFFu, sum, o);
  if (lane < a.top_k) {
    a.ids[t * a.top_k + lane] = chosen;
    a.weights[t * a.top_k + lane] = p / sum;
  }
}
__device__ __forceinline__ void moe_choose_none(const b200q_moe_args& a, int64_t t, int lane) {
  if (lane < a.top_k) {
    a.ids[t * a.top_k + lane] = -1;
    a.weights[t * a.top_k + lane] = 0.f;
  }
}

__global__ void __launch_bounds__(32) moe_choose_kernel(const b200q_moe_args a, int64_t first, const double* logits) {
  pdl_enter();
  const int64_t t = blockIdx.x;
  if (t < moe_tokens(a, first)) moe_choose(a, t, logits + t * a.experts, threadIdx.x);
  else moe_choose_none(a, t, threadIdx.x);
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

// ---------------------------------------------------------------------------- host
size_t moe_workspace_bytes_impl(int64_t tokens, int64_t hidden, int64_t inner, int experts, int top_k) {
  return MoeSpace(tokens, hidden, inner, experts, top_k).bytes;
}

static int64_t moe_blocks(int64_t warps) { return (warps + kMoeThreads / 32 - 1) / (kMoeThreads / 32); }

static int moe_chunk(const b200q_moe_args& a, int64_t first, cudaStream_t st) {
  const MoeSpace space(a.tokens, a.hidden, a.inner, a.experts, a.top_k);
  uint8_t* p = static_cast<uint8_t*>(a.workspace);
  double* logits = reinterpret_cast<double*>(p + space.logits);
  float *hidden = reinterpret_cast<float*>(p + space.hidden), *outputs = reinterpret_cast<float*>(p + space.outputs);
  const int64_t slots = a.tokens * a.top_k, up = moe_blocks(slots * a.inner), down = moe_blocks(slots * a.hidden);
  const int64_t sum = a.tokens * ((a.hidden + kMoeThreads - 1) / kMoeThreads);
  if (up > INT32_MAX || down > INT32_MAX || sum > INT32_MAX) return B200Q_ERR_TOO_LARGE;
  launch_dependent(moe_logits_kernel, dim3((unsigned)moe_blocks(a.tokens * a.experts)), dim3(kMoeThreads), 0, st, a, first, logits);
  B200Q_LAUNCH_CHECK();
  launch_dependent(moe_choose_kernel, dim3((unsigned)a.tokens), dim3(32), 0, st, a, first, static_cast<const double*>(logits));
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
