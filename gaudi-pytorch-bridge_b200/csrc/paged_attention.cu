// Attention of one new token per request over a key/value cache in pages:
//   s_j = softmax_scale * k_scale_inv * <q, k_j>,  j in [max(0, len - window), len);   p = softmax(s)
//   out = v_scale_inv * sum_j p_j v_j,   lse = log sum_j exp(s_j);   nothing to see: out = 0, lse = -inf.
#include "paged.cuh"

namespace b200q {

__device__ __forceinline__ float paged_value(const void* p, int dtype, int64_t at) {
  if (dtype == B200Q_BF16) return __bfloat162float(static_cast<const __nv_bfloat16*>(p)[at]);
  const uint32_t byte = static_cast<const uint8_t*>(p)[at];
  return dtype == B200Q_E4M3 ? fp8_to_float<B200Q_E4M3>(byte) : fp8_to_float<B200Q_E5M2>(byte);
}
__device__ __forceinline__ void paged_store(void* out, int dtype, int64_t at, float v) {
  if (dtype == B200Q_BF16) static_cast<__nv_bfloat16*>(out)[at] = __float2bfloat16_rn(v);
  else if (dtype == B200Q_F32) static_cast<float*>(out)[at] = v;
  else static_cast<uint8_t*>(out)[at] = (uint8_t)(cvt_fp8x2<B200Q_E4M3>(v, 0.f) & 0xFFu);
}
// tokens of the request that its table can hold
__device__ __forceinline__ int64_t paged_length(const b200q_paged_attention_args& a, int64_t b) {
  const int64_t most = a.table_width * a.page_size;
  return min((int64_t)max(a.kv_lens[b], 0), most);
}

// ---------------------------------------------------------------------------- plain
// Any head dimension up to 256, any page size, strides and alignment: a block per (request, query head), a thread per key
// of a tile for the scores and per dimension for the values.
constexpr int kPlainThreads = 256;

__device__ __forceinline__ float plain_block_reduce(float v, bool maximum) {
  __shared__ float s[kPlainThreads / 32];
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const float w = __shfl_xor_sync(0xFFFFFFFFu, v, o);
    v = maximum ? (v > w || v != v ? v : w) : v + w;  // (a NaN stays)
  }
  __syncthreads();
  if ((threadIdx.x & 31) == 0) s[threadIdx.x >> 5] = v;
  __syncthreads();
  v = s[0];
#pragma unroll
  for (int i = 1; i < kPlainThreads / 32; ++i) v = maximum ? (v > s[i] || v != v ? v : s[i]) : v + s[i];
  return v;
}

__global__ void __launch_bounds__(kPlainThreads) paged_attention_plain_kernel(const b200q_paged_attention_args a) {
  __shared__ float s_q[256], s_p[kPlainThreads];
  __shared__ int s_page[kPlainThreads];
  pdl_enter();
  const int tid = threadIdx.x;
  const int64_t b = blockIdx.x / a.heads, head = blockIdx.x % a.heads, kv = head / (a.heads / a.kv_heads);
  const int64_t len = paged_length(a, b);
  const int64_t first = a.window > 0 ? max(len - a.window, (int64_t)0) : 0;
  if (tid < a.dim) s_q[tid] = __bfloat162float(static_cast<const __nv_bfloat16*>(a.q)[b * a.q_token_stride + head * a.q_head_stride + tid]);
  __syncthreads();
  const float scale = a.softmax_scale * (a.k_scale_inv ? *a.k_scale_inv : 1.f);
  float m = -INFINITY, l = 0.f, acc = 0.f;
  for (int64_t tile = first; tile < len; tile += kPlainThreads) {
    const int64_t j = tile + tid;
    int page = -1;
    float s = -INFINITY;
    if (j < len) {
      page = a.block_table[b * a.table_stride + j / a.page_size];
      if (page >= a.num_pages) page = -1;
      if (page >= 0) {
        const int64_t at = page * a.k_page_stride + (j % a.page_size) * a.k_slot_stride + kv * a.k_head_stride;
        float dot = 0.f;
        for (int d = 0; d < a.dim; ++d) dot += s_q[d] * paged_value(a.k_cache, a.cache_dtype, at + d);
        s = dot * scale;
      }
    }
    const float top = fmaxf(m, plain_block_reduce(s, true));
    const float keep = m == -INFINITY ? 0.f : expf(m - top);
    const float prob = page < 0 || s == -INFINITY ? 0.f : expf(s - (top == -INFINITY ? 0.f : top));  // (a NaN comes through)
    m = top;
    l = l * keep + plain_block_reduce(prob, false);
    s_p[tid] = prob;
    s_page[tid] = page;
    __syncthreads();
    if (tid < a.dim) {
      acc *= keep;
      const int n = (int)min((int64_t)kPlainThreads, len - tile);
      for (int i = 0; i < n; ++i) {
        if (s_page[i] < 0) continue;
        const int64_t at = s_page[i] * a.v_page_stride + ((tile + i) % a.page_size) * a.v_slot_stride + kv * a.v_head_stride;
        acc += s_p[i] * paged_value(a.v_cache, a.cache_dtype, at + tid);
      }
    }
    __syncthreads();
  }
  // (l is NaN where a score is: that is not an empty row)
  const bool empty = l == 0.f;
  if (tid < a.dim) {
    const float v_scale = (a.v_scale_inv ? *a.v_scale_inv : 1.f) * (a.out_scale ? *a.out_scale : 1.f);
    paged_store(a.out, a.out_dtype, (b * a.heads + head) * a.dim + tid, empty ? 0.f : acc / l * v_scale);
  }
  if (tid == 0 && a.lse) a.lse[b * a.heads + head] = empty ? -INFINITY : m + logf(l);
}

size_t paged_attention_workspace_bytes_impl(int64_t requests, int heads, int kv_heads, int dim, int cache_dtype) { return 0; }

int paged_attention_impl(const b200q_paged_attention_args& a, cudaStream_t st) {
  const int64_t blocks = a.requests * a.heads;
  if (blocks > 0x7FFFFFFF) return B200Q_ERR_TOO_LARGE;
  launch_dependent(paged_attention_plain_kernel, dim3((unsigned)blocks), dim3(kPlainThreads), 0, st, a);
  B200Q_LAUNCH_CHECK();
  return B200Q_OK;
}

}  // namespace b200q
