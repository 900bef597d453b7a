// The paged key/value cache before its attention: the plan of a step (which slot every new token gets, built on the
// device from the requests' lengths) and the append (norm of the query and key heads, rotation by the position, cast,
// write into the pages).
#include "paged.cuh"

namespace b200q {

// ---------------------------------------------------------------------------- plan
// Request b holds c_b tokens and gets n_b new ones: of its pages ceil(c_b / ps) are in the table already and the ones up
// to ceil((c_b + n_b) / ps) come from the free list, in request order.  So everything follows from two prefix sums over
// the requests (new tokens, new pages); a block forms both in shared memory for itself, and then no block waits for
// another: a token reads its page either from an old table entry, which nobody writes, or from the free list.
// All of it is latency (a few KB to 1 MB of output).
constexpr int kPlanThreads = 256;
constexpr int kPlanTokensPerBlock = 1024;

__device__ __forceinline__ int sat_add(int a, int b) {  // of non-negative numbers
  return (int)min((uint32_t)a + (uint32_t)b, 0x7FFFFFFFu);
}
// index of the first entry of the ascending end[0..n) that is above x; x < end[n - 1]
__device__ __forceinline__ int first_above(const int* end, int n, int x) {
  int lo = 0, hi = n - 1;
  while (lo < hi) {
    const int mid = (lo + hi) >> 1;
    if (end[mid] > x) hi = mid;
    else lo = mid + 1;
  }
  return lo;
}

struct PlanRequest {
  uint32_t context, total;  // tokens held, tokens after the step
  int have, need;           // pages of both, within the table's width
};
__device__ __forceinline__ PlanRequest plan_request(const PagedPlanParams& p, int b) {
  PlanRequest r;
  r.context = (uint32_t)max(p.context_lens[b], 0);
  r.total = r.context + (uint32_t)max(p.new_lens[b], 0);
  const uint32_t ps = (uint32_t)p.page_size, w = (uint32_t)p.table_width;
  r.have = (int)min(r.context / ps + (r.context % ps != 0), w);
  r.need = (int)min(r.total / ps + (r.total % ps != 0), w);
  return r;
}

__global__ void __launch_bounds__(kPlanThreads) paged_plan_kernel(const PagedPlanParams p) {
  extern __shared__ int s_end[];  // [requests] new tokens, [requests] new pages: inclusive sums
  __shared__ int s_warp[2][kPlanThreads / 32];
  int* tok_end = s_end;
  int* page_end = s_end + p.requests;
  pdl_enter();
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int per = (p.requests + kPlanThreads - 1) / kPlanThreads;
  const int b0 = min(tid * per, p.requests), b1 = min(b0 + per, p.requests);
  int toks = 0, pages = 0;
  for (int b = b0; b < b1; ++b) {
    const PlanRequest r = plan_request(p, b);
    toks = sat_add(toks, (int)(r.total - r.context));
    pages += r.need - r.have;
    tok_end[b] = toks;
    page_end[b] = pages;
  }
  int t_scan = toks, p_scan = pages;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int t = __shfl_up_sync(0xFFFFFFFFu, t_scan, o), g = __shfl_up_sync(0xFFFFFFFFu, p_scan, o);
    if (lane >= o) {
      t_scan = sat_add(t_scan, t);
      p_scan += g;
    }
  }
  if (lane == 31) {
    s_warp[0][warp] = t_scan;
    s_warp[1][warp] = p_scan;
  }
  int t_before = __shfl_up_sync(0xFFFFFFFFu, t_scan, 1), p_before = __shfl_up_sync(0xFFFFFFFFu, p_scan, 1);
  if (lane == 0) t_before = p_before = 0;
  __syncthreads();
  int total_toks = 0, total_pages = 0;
#pragma unroll
  for (int w = 0; w < kPlanThreads / 32; ++w) {
    if (w == warp) {
      t_before = sat_add(t_before, total_toks);
      p_before += total_pages;
    }
    total_toks = sat_add(total_toks, s_warp[0][w]);
    total_pages += s_warp[1][w];
  }
  for (int b = b0; b < b1; ++b) {
    tok_end[b] = sat_add(tok_end[b], t_before);
    page_end[b] += p_before;
  }
  __syncthreads();

  const int head = p.free_head ? max(*p.free_head, 0) : 0;
  auto free_page = [&](int i) -> int {  // the i-th page that this step takes
    const int64_t at = (int64_t)head + i;
    return at < p.free_count ? p.free_pages[at] : -1;
  };
  if (blockIdx.x == 0) {
    for (int b = tid; b < p.requests; b += kPlanThreads) {
      p.query_start[b + 1] = tok_end[b];
      p.kv_lens[b] = (int)min(plan_request(p, b).total, 0x7FFFFFFFu);
    }
    if (tid == 0) {
      p.query_start[0] = 0;
      *p.free_head_out = sat_add(head, total_pages);
    }
  }
  const int stride = gridDim.x * kPlanThreads;
  for (int i = blockIdx.x * kPlanThreads + tid; i < total_pages; i += stride) {
    const int b = first_above(page_end, p.requests, i);
    const PlanRequest r = plan_request(p, b);
    p.table[b * p.table_stride + r.need - (page_end[b] - i)] = free_page(i);
  }
  for (int64_t t64 = blockIdx.x * kPlanThreads + tid; t64 < p.num_tokens; t64 += stride) {
    const int t = (int)t64;
    int64_t pos = 0, slot = -1;
    if (t < total_toks) {
      const int b = first_above(tok_end, p.requests, t);
      const PlanRequest r = plan_request(p, b);
      const uint32_t at = r.context + (uint32_t)(t - (b ? tok_end[b - 1] : 0));
      const uint32_t j = at / (uint32_t)p.page_size, off = at % (uint32_t)p.page_size;
      pos = at;
      if (j < (uint32_t)p.table_width) {
        const int page = (int)j < r.have ? p.table[b * p.table_stride + j] : free_page((b ? page_end[b - 1] : 0) + (int)j - r.have);
        if (page >= 0) slot = (int64_t)page * p.page_size + off;
      }
    }
    p.positions[t] = pos;
    p.slot_map[t] = slot;
  }
}

int paged_plan_impl(const PagedPlanParams& p, cudaStream_t st) {
  const size_t smem = 2 * sizeof(int) * (size_t)p.requests;
  static std::atomic<int> ready[kMaxDevices];
  const int dev = current_device_index();
  if (dev < 0) return B200Q_ERR_CUDA;
  if (!ready[dev].load(std::memory_order_acquire)) {
    B200Q_CUDA_OK(cudaFuncSetAttribute(paged_plan_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)(2 * sizeof(int) * kPagedMaxRequests)));
    ready[dev].store(1, std::memory_order_release);
  }
  int64_t blocks = ((int64_t)p.num_tokens + kPlanTokensPerBlock - 1) / kPlanTokensPerBlock;
  if (blocks < 1) blocks = 1;
  if (blocks > kNumSMs) blocks = kNumSMs;
  launch_dependent(paged_plan_kernel, dim3((unsigned)blocks), dim3(kPlanThreads), smem, st, p);
  B200Q_LAUNCH_CHECK();
  return B200Q_OK;
}

// ---------------------------------------------------------------------------- norm, rotation, append
// y = x * rsqrt(mean(x^2) + eps) * w over a head of D values (no norm without w); the first r of them turn by the angle of
// the token's position in pairs (i, i + r/2) or (2i, 2i + 1); one rounding from fp32 to the output's type.
// Memory bound.  D / 8 lanes own a head: a lane holds four values and the four they are paired with, so that the rotation needs
// no exchange between lanes, and its four cosines and sines serve every head of the token that it walks through.
constexpr int kAppendThreads = 128;

template <typename Src>
__device__ __forceinline__ void load4(const Src* p, float (&v)[4]);
template <>
__device__ __forceinline__ void load4<__nv_bfloat16>(const __nv_bfloat16* p, float (&v)[4]) {
  const uint2 w = *reinterpret_cast<const uint2*>(p);
  v[0] = bf16_bits_to_float(w.x & 0xFFFFu);
  v[1] = bf16_bits_to_float(w.x >> 16);
  v[2] = bf16_bits_to_float(w.y & 0xFFFFu);
  v[3] = bf16_bits_to_float(w.y >> 16);
}
template <>
__device__ __forceinline__ void load4<float>(const float* p, float (&v)[4]) {
  const float4 w = *reinterpret_cast<const float4*>(p);
  v[0] = w.x; v[1] = w.y; v[2] = w.z; v[3] = w.w;
}
__device__ __forceinline__ void load4_any(const void* p, int dtype, int64_t at, float (&v)[4]) {
  if (dtype == B200Q_BF16) load4(static_cast<const __nv_bfloat16*>(p) + at, v);
  else load4(static_cast<const float*>(p) + at, v);
}

// four values to elements [at, at + 4) of a bf16 / e4m3 / e5m2 tensor
__device__ __forceinline__ void store4(void* p, int dtype, int64_t at, const float (&v)[4]) {
  if (dtype == B200Q_BF16) {
    *reinterpret_cast<uint2*>(static_cast<__nv_bfloat16*>(p) + at) = make_uint2(pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]));
  } else if (dtype == B200Q_E4M3) {
    *reinterpret_cast<uint32_t*>(static_cast<uint8_t*>(p) + at) = cvt_fp8x2<B200Q_E4M3>(v[0], v[1]) | (cvt_fp8x2<B200Q_E4M3>(v[2], v[3]) << 16);
  } else {
    *reinterpret_cast<uint32_t*>(static_cast<uint8_t*>(p) + at) = cvt_fp8x2<B200Q_E5M2>(v[0], v[1]) | (cvt_fp8x2<B200Q_E5M2>(v[2], v[3]) << 16);
  }
}

// Row r of a token: query heads, key heads, value heads.
template <typename Src, int LANES>
__global__ void __launch_bounds__(kAppendThreads) qk_norm_rope_append_kernel(const b200q_append_args a, int rows_per_block) {
  constexpr int kGroups = kAppendThreads / LANES;
  pdl_enter();
  const int64_t t = blockIdx.x;
  const int lane = threadIdx.x % LANES, group = threadIdx.x / LANES;
  const bool on = lane < a.dim / 8;
  const int rot = a.cos_sin ? a.rotary_dim : 0, half = rot / 2;
  const bool turned = lane < rot / 8;
  // where the lane's values are: four at lo, and at hi the four that they are paired with (or the next four)
  const bool apart = turned && !a.interleaved;
  const int lo = apart ? 4 * lane : 8 * lane;
  const int hi = apart ? half + 4 * lane : lo + 4;
  float cs[4] = {1.f, 1.f, 1.f, 1.f}, sn[4] = {0.f, 0.f, 0.f, 0.f};
  if (turned) {
    const int64_t pos = a.positions[t];
    if (pos >= 0 && pos < a.max_positions) {
      load4(a.cos_sin + pos * rot + 4 * lane, cs);
      load4(a.cos_sin + pos * rot + half + 4 * lane, sn);
    } else {  // no such position: the heads become NaN
#pragma unroll
      for (int i = 0; i < 4; ++i) cs[i] = sn[i] = __int_as_float(0x7FC00000);
    }
  }
  const int64_t slot = a.slot_map[t];
  const bool kept = slot >= 0 && slot < a.num_pages * a.page_size;
  const int64_t page = kept ? (uint32_t)slot / (uint32_t)a.page_size : 0, off = kept ? (uint32_t)slot % (uint32_t)a.page_size : 0;
  const float q_scale = a.q_scale ? *a.q_scale : 1.f, k_scale = a.k_scale ? *a.k_scale : 1.f, v_scale = a.v_scale ? *a.v_scale : 1.f;

  const int rows = a.heads + 2 * a.kv_heads;
  const int r0 = blockIdx.y * rows_per_block, r1 = min(r0 + rows_per_block, rows);
  for (int base = r0; base < r1; base += kGroups) {  // (every lane of a warp makes the same number of rounds)
    const int row = base + group;
    const bool is_q = row < a.heads, is_v = row >= a.heads + a.kv_heads;
    const int h = is_q ? row : row - a.heads - (is_v ? a.kv_heads : 0);
    const bool live = on && row < r1 && (is_q || kept);
    float x[4] = {0.f, 0.f, 0.f, 0.f}, y[4] = {0.f, 0.f, 0.f, 0.f};
    if (live) {
      const Src* src = is_q ? static_cast<const Src*>(a.q) + t * a.q_token_stride + h * a.q_head_stride
                            : is_v ? static_cast<const Src*>(a.v) + t * a.v_token_stride + h * a.v_head_stride
                                   : static_cast<const Src*>(a.k) + t * a.k_token_stride + h * a.k_head_stride;
      load4(src + lo, x);
      load4(src + hi, y);
    }
    const void* w = is_q ? a.q_weight : is_v ? nullptr : a.k_weight;
    float sum = 0.f;
#pragma unroll
    for (int i = 0; i < 4; ++i) sum += x[i] * x[i] + y[i] * y[i];
#pragma unroll
    for (int o = LANES / 2; o > 0; o >>= 1) sum += __shfl_xor_sync(0xFFFFFFFFu, sum, o, LANES);
    if (!live) continue;
    if (w) {
      const float inv = rsqrtf(sum / (float)a.dim + a.eps);
      float wx[4], wy[4];
      load4_any(w, a.weight_dtype, lo, wx);
      load4_any(w, a.weight_dtype, hi, wy);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        x[i] = x[i] * inv * wx[i];
        y[i] = y[i] * inv * wy[i];
      }
    }
    if (turned && !is_v) {
      if (a.interleaved) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const float u0 = x[2 * i], u1 = x[2 * i + 1], w0 = y[2 * i], w1 = y[2 * i + 1];
          x[2 * i] = u0 * cs[i] - u1 * sn[i];
          x[2 * i + 1] = u1 * cs[i] + u0 * sn[i];
          y[2 * i] = w0 * cs[2 + i] - w1 * sn[2 + i];
          y[2 * i + 1] = w1 * cs[2 + i] + w0 * sn[2 + i];
        }
      } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float u = x[i], v = y[i];
          x[i] = u * cs[i] - v * sn[i];
          y[i] = v * cs[i] + u * sn[i];
        }
      }
    }
    const float scale = is_q ? q_scale : is_v ? v_scale : k_scale;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      x[i] *= scale;
      y[i] *= scale;
    }
    if (is_q) {
      const int64_t at = (t * a.heads + h) * a.dim;
      store4(a.q_out, a.q_out_dtype, at + lo, x);
      store4(a.q_out, a.q_out_dtype, at + hi, y);
    } else {
      const int64_t at = is_v ? page * a.v_page_stride + off * a.v_slot_stride + h * a.v_cache_head_stride
                              : page * a.k_page_stride + off * a.k_slot_stride + h * a.k_cache_head_stride;
      void* cache = is_v ? a.v_cache : a.k_cache;
      store4(cache, a.cache_dtype, at + lo, x);
      store4(cache, a.cache_dtype, at + hi, y);
    }
  }
}

template <typename Src>
static void append_launch(const b200q_append_args& a, cudaStream_t st) {
  const int rows = a.heads + 2 * a.kv_heads;
  auto go = [&](auto kernel, int lanes) {
    const int groups = kAppendThreads / lanes;
    // few tokens: a block per round of rows, so that the whole device takes part
    const int rounds = (rows + groups - 1) / groups;
    const int split = a.tokens * rounds <= 4 * kNumSMs ? rounds : 1;
    launch_dependent(kernel, dim3((unsigned)a.tokens, (unsigned)split), dim3(kAppendThreads), 0, st, a, (split > 1 ? 1 : rounds) * groups);
  };
  if (a.dim <= 64) go(qk_norm_rope_append_kernel<Src, 8>, 8);
  else if (a.dim <= 128) go(qk_norm_rope_append_kernel<Src, 16>, 16);
  else go(qk_norm_rope_append_kernel<Src, 32>, 32);
}

int qk_norm_rope_append_impl(const b200q_append_args& a, cudaStream_t st) {
  if (a.src_dtype == B200Q_BF16) append_launch<__nv_bfloat16>(a, st);
  else append_launch<float>(a, st);
  B200Q_LAUNCH_CHECK();
  return B200Q_OK;
}

}  // namespace b200q
