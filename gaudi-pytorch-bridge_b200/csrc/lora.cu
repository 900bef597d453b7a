// Low-rank adapters of many requests beside a product that they share: y[t] += scale * b (a x[t]) with the adapter of each token.
#include "layer.cuh"

namespace b200q {

constexpr int64_t kLoraChunk = 8192;  // tokens taken at a time
constexpr size_t lora_align(size_t n) { return (n + 255) / 256 * 256; }

__device__ __forceinline__ float lora_bf16(const void* p, int64_t at) { return __bfloat162float(static_cast<const __nv_bfloat16*>(p)[at]); }
__device__ __forceinline__ int lora_adapter(const b200q_lora_args& a, int64_t t) {  // or -1
  const int i = a.adapter[t];
  return i >= 0 && i < a.adapters ? i : -1;
}

// ---------------------------------------------------------------------------- plain
// Any sizes, strides and alignment: a warp per (token, rank), then a thread per value of y.
constexpr int kLoraPlainThreads = 256;

__global__ void __launch_bounds__(kLoraPlainThreads) lora_plain_down_kernel(const b200q_lora_args a, float* low) {
  pdl_enter();
  const int lane = threadIdx.x & 31;
  const int64_t at = (int64_t)blockIdx.x * (kLoraPlainThreads / 32) + (threadIdx.x >> 5);
  if (at >= a.tokens * a.rank) return;
  const int64_t t = at / a.rank, r = at - t * a.rank;
  const int i = lora_adapter(a, t);
  if (i < 0) return;
  float sum = 0.f;
  for (int64_t k = lane; k < a.k; k += 32) sum += lora_bf16(a.a, i * a.a_stride + r * a.a_row_stride + k) * lora_bf16(a.x, t * a.x_stride + k);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xFFFFFFFFu, sum, o);
  if (lane == 0) low[at] = sum * (a.scales ? a.scales[i] : 1.f);
}
__global__ void __launch_bounds__(kLoraPlainThreads) lora_plain_up_kernel(const b200q_lora_args a, const float* low) {
  pdl_enter();
  const int64_t per_row = (a.n + kLoraPlainThreads - 1) / kLoraPlainThreads;
  const int64_t t = blockIdx.x / per_row, n = (blockIdx.x - t * per_row) * kLoraPlainThreads + threadIdx.x;
  const int i = lora_adapter(a, t);
  if (i < 0 || n >= a.n) return;
  float sum = 0.f;
  for (int64_t r = 0; r < a.rank; ++r) sum += low[t * a.rank + r] * lora_bf16(a.b, i * a.b_stride + n * a.b_row_stride + r);
  if (a.y_dtype == B200Q_F32) {
    static_cast<float*>(a.y)[t * a.y_stride + n] += sum;
  } else {
    __nv_bfloat16* y = static_cast<__nv_bfloat16*>(a.y) + t * a.y_stride + n;
    *y = __float2bfloat16_rn(__bfloat162float(*y) + sum);
  }
}

size_t lora_workspace_bytes_impl(int64_t tokens, int64_t k, int64_t n, int64_t rank, int64_t adapters) {
  (void)k;
  (void)n;
  (void)adapters;
  return lora_align(sizeof(float) * (size_t)((tokens < kLoraChunk ? tokens : kLoraChunk) * rank));
}

static int lora_chunk(const b200q_lora_args& a, cudaStream_t st) {
  float* low = static_cast<float*>(a.workspace);
  const int64_t warps = a.tokens * a.rank, down = (warps + kLoraPlainThreads / 32 - 1) / (kLoraPlainThreads / 32);
  const int64_t up = a.tokens * ((a.n + kLoraPlainThreads - 1) / kLoraPlainThreads);
  if (down > INT32_MAX || up > INT32_MAX) return B200Q_ERR_TOO_LARGE;
  launch_dependent(lora_plain_down_kernel, dim3((unsigned)down), dim3(kLoraPlainThreads), 0, st, a, low);
  B200Q_LAUNCH_CHECK();
  launch_dependent(lora_plain_up_kernel, dim3((unsigned)up), dim3(kLoraPlainThreads), 0, st, a, static_cast<const float*>(low));
  B200Q_LAUNCH_CHECK();
  return B200Q_OK;
}

int lora_add_impl(const b200q_lora_args& a, cudaStream_t st) {
  if (!a.workspace || a.workspace_bytes < lora_workspace_bytes_impl(a.tokens, a.k, a.n, a.rank, a.adapters) ||
      reinterpret_cast<uintptr_t>(a.workspace) % 16)
    return B200Q_ERR_BAD_ARGUMENT;
  for (int64_t t = 0; t < a.tokens; t += kLoraChunk) {
    b200q_lora_args c = a;
    c.tokens = a.tokens - t < kLoraChunk ? a.tokens - t : kLoraChunk;
    c.x = static_cast<const uint8_t*>(a.x) + 2 * t * a.x_stride;
    c.y = static_cast<uint8_t*>(a.y) + (a.y_dtype == B200Q_F32 ? 4 : 2) * t * a.y_stride;
    c.adapter = a.adapter + t;
    if (int rc = lora_chunk(c, st)) return rc;
  }
  return B200Q_OK;
}

}  // namespace b200q
