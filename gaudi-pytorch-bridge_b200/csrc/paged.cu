// The paged key/value cache before its attention: the plan of a step (which slot every new token gets, built on the
// device from the requests' lengths) and the append (norm of the query and key heads, rotation by the position, cast,
// write into the pages).
#include <type_traits>

#include "paged.cuh"

namespace b200q {

// ---------------------------------------------------------------------------- plan
// Request b holds c_b tokens and gets n_b new ones: of its pages ceil(c_b / ps) are in the table already and the ones up
// to ceil((c_b + n_b) / ps) come from the free list, in request order.  So everything follows from two prefix sums over
// the requests (new tokens, new pages); a block forms both in shared memory for itself, and then no block waits for
// another: a token reads its page either from an old table entry, which nobody writes, or from the free list.
// All of it is latency (a few KB to 1 MB of output): 3.1 us for 64 requests, 5.1 for 32 prompts of 80 000 tokens together, 7.7 for 1024 requests and
// 24 for 8192, whose sums are taken 256 requests at a time.  Every block forms the sums again, so that more blocks cost SMs, not time: in blocks of 256 /
// 1024 / 4096 tokens the 32 prompts take 4.6 / 5.1 / 12.8 us, 64 requests of 256 tokens each 3.1 / 6.2 / 16.4, 1024 of 16 4.8 / 8.2 / 21.5, one of 16384
// 2.6 / 3.6 / 8.2, and steps of a token each up to 64 requests the same.
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
__device__ __forceinline__ PlanRequest plan_request(const PagedPlanParams& p, int context, int added) {
  PlanRequest r;
  r.context = (uint32_t)max(context, 0);
  r.total = r.context + (uint32_t)max(added, 0);
  const uint32_t ps = (uint32_t)p.page_size, w = (uint32_t)p.table_width;
  const uint32_t have = r.context / ps, need = r.total / ps;
  r.have = (int)min(have + (have * ps != r.context), w);
  r.need = (int)min(need + (need * ps != r.total), w);
  return r;
}

__device__ __forceinline__ PlanRequest plan_request(const PagedPlanParams& p, int b) { return plan_request(p, p.context_lens[b], p.new_lens[b]); }

__global__ void __launch_bounds__(kPlanThreads) paged_plan_kernel(const PagedPlanParams p) {
  extern __shared__ int s_end[];  // [requests] new tokens, [requests] new pages: inclusive sums
  __shared__ int s_warp[2][2][kPlanThreads / 32];
  int* tok_end = s_end;
  int* page_end = s_end + p.requests;
  pdl_enter();
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  int total_toks = 0, total_pages = 0;
  int context = 0, added = 0;  // of the next requests, on their way while the ones before are summed up
  if (tid < p.requests) {
    context = p.context_lens[tid];
    added = p.new_lens[tid];
  }
  for (int base = 0, turn = 0; base < p.requests; base += kPlanThreads, turn ^= 1) {
    const int b = base + tid;
    int toks = 0, pages = 0;
    if (b < p.requests) {
      const PlanRequest r = plan_request(p, context, added);
      toks = (int)(r.total - r.context);
      pages = r.need - r.have;
    }
    if (b + kPlanThreads < p.requests) {
      context = p.context_lens[b + kPlanThreads];
      added = p.new_lens[b + kPlanThreads];
    }
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int t = __shfl_up_sync(0xFFFFFFFFu, toks, o), g = __shfl_up_sync(0xFFFFFFFFu, pages, o);
      if (lane >= o) {
        toks = sat_add(toks, t);
        pages += g;
      }
    }
    if (lane == 31) {
      s_warp[turn][0][warp] = toks;
      s_warp[turn][1][warp] = pages;
    }
    __syncthreads();  // (the other half of s_warp is written next, and this one only behind the next barrier)
    int t_before = total_toks, p_before = total_pages;
#pragma unroll
    for (int w = 0; w < kPlanThreads / 32; ++w) {
      if (w == warp) {
        t_before = total_toks;
        p_before = total_pages;
      }
      total_toks = sat_add(total_toks, s_warp[turn][0][w]);
      total_pages += s_warp[turn][1][w];
    }
    if (b < p.requests) {
      tok_end[b] = sat_add(toks, t_before);
      page_end[b] = pages + p_before;
    }
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
  for (int64_t i64 = blockIdx.x * kPlanThreads + tid; i64 < total_pages; i64 += stride) {  // (up to 2^31 - 1 of them)
    const int i = (int)i64, b = first_above(page_end, p.requests, i);
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
// Memory bound, if the instructions are few: 16 lanes own a head of 128, 8 values each, and a first version of 221 instructions per
// lane and head was bound by them (82 % of the issue slots, 4.0 TB/s).  So a lane holds four values and the four that they are paired
// with: the rotation needs no exchange between lanes.  Weight, cosine and sine are multiplied once per token into four factors
// per pair, which serve every head that the lane walks through; norm and scale are one factor at the end.
constexpr int kAppendThreads = 128;
constexpr int kAppendBatch = 2;  // rounds of heads in flight: what more would bring costs as many registers, and with them blocks per SM

__device__ __forceinline__ void load4(const float* p, float (&v)[4]) {
  const float4 w = *reinterpret_cast<const float4*>(p);
  v[0] = w.x; v[1] = w.y; v[2] = w.z; v[3] = w.w;
}
__device__ __forceinline__ void load4(const __nv_bfloat16* p, float (&v)[4]) {
  const uint2 w = *reinterpret_cast<const uint2*>(p);
  v[0] = bf16_bits_to_float(w.x & 0xFFFFu);
  v[1] = bf16_bits_to_float(w.x >> 16);
  v[2] = bf16_bits_to_float(w.y & 0xFFFFu);
  v[3] = bf16_bits_to_float(w.y >> 16);
}
__device__ __forceinline__ void load4_any(const void* p, int dtype, int64_t at, float (&v)[4]) {
  if (dtype == B200Q_BF16) load4(static_cast<const __nv_bfloat16*>(p) + at, v);
  else load4(static_cast<const float*>(p) + at, v);
}

// Four values as they come.
template <typename Src>
struct Raw4 {
  typename std::conditional<sizeof(Src) == 2, uint2, float4>::type w;
  __device__ __forceinline__ void load(const Src* p) { w = *reinterpret_cast<const decltype(w)*>(p); }
  __device__ __forceinline__ void get(float (&v)[4]) const;
};
template <>
__device__ __forceinline__ void Raw4<__nv_bfloat16>::get(float (&v)[4]) const {
  v[0] = __uint_as_float(w.x << 16);
  v[1] = __uint_as_float(w.x & 0xFFFF0000u);
  v[2] = __uint_as_float(w.y << 16);
  v[3] = __uint_as_float(w.y & 0xFFFF0000u);
}
template <>
__device__ __forceinline__ void Raw4<float>::get(float (&v)[4]) const {
  v[0] = w.x; v[1] = w.y; v[2] = w.z; v[3] = w.w;
}

// values lo .. lo + 3 and hi .. hi + 3 of a head that begins at element `at` of a bf16 / e4m3 / e5m2 tensor
__device__ __forceinline__ void store8(void* p, int dtype, int64_t at, int lo, int hi, const float (&x)[4], const float (&y)[4]) {
  if (dtype == B200Q_BF16) {
    __nv_bfloat16* to = static_cast<__nv_bfloat16*>(p) + at;
    *reinterpret_cast<uint2*>(to + lo) = make_uint2(pack_bf16x2(x[0], x[1]), pack_bf16x2(x[2], x[3]));
    *reinterpret_cast<uint2*>(to + hi) = make_uint2(pack_bf16x2(y[0], y[1]), pack_bf16x2(y[2], y[3]));
  } else {
    uint8_t* to = static_cast<uint8_t*>(p) + at;
    uint32_t a, b;
    if (dtype == B200Q_E4M3) {
      a = cvt_fp8x2<B200Q_E4M3>(x[0], x[1]) | (cvt_fp8x2<B200Q_E4M3>(x[2], x[3]) << 16);
      b = cvt_fp8x2<B200Q_E4M3>(y[0], y[1]) | (cvt_fp8x2<B200Q_E4M3>(y[2], y[3]) << 16);
    } else {
      a = cvt_fp8x2<B200Q_E5M2>(x[0], x[1]) | (cvt_fp8x2<B200Q_E5M2>(x[2], x[3]) << 16);
      b = cvt_fp8x2<B200Q_E5M2>(y[0], y[1]) | (cvt_fp8x2<B200Q_E5M2>(y[2], y[3]) << 16);
    }
    *reinterpret_cast<uint32_t*>(to + lo) = a;
    *reinterpret_cast<uint32_t*>(to + hi) = b;
  }
}

// A block walks through tokens; of each it takes rounds [y rounds_per_block, ...): first the query heads, then the key heads, then the value
// heads, as many at a time as it has groups of LANES lanes.
template <typename Src, int LANES, bool INTERLEAVED>
__global__ void __launch_bounds__(kAppendThreads) qk_norm_rope_append_kernel(const b200q_append_args a, float inv_dim, int rounds_per_block) {
  constexpr int kGroups = kAppendThreads / LANES;
  __shared__ __align__(16) float s_weight[2][8 * LANES];  // of query and key heads
  __shared__ float s_scale[2];
  pdl_enter();
  const int lane = threadIdx.x % LANES, group = threadIdx.x / LANES;
  const bool on = lane < a.dim / 8;
  const int rot = a.cos_sin ? a.rotary_dim : 0, half = rot / 2;
  const bool turned = lane < rot / 8;
  // where the lane's values are: four at lo, and at hi the four that they are paired with (or the next four)
  const bool apart = turned && !INTERLEAVED;
  const int lo = apart ? 4 * lane : 8 * lane;
  const int hi = apart ? half + 4 * lane : lo + 4;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const void* weight = i ? a.k_weight : a.q_weight;
    for (int d = threadIdx.x; d < a.dim; d += kAppendThreads)
      s_weight[i][d] = !weight ? 1.f : a.weight_dtype == B200Q_BF16 ? __bfloat162float(static_cast<const __nv_bfloat16*>(weight)[d]) : static_cast<const float*>(weight)[d];
  }
  if (threadIdx.x == 0) {
    s_scale[0] = a.q_scale ? *a.q_scale : 1.f;
    s_scale[1] = a.k_scale ? *a.k_scale : 1.f;
  }
  const float v_scale = a.v_scale ? *a.v_scale : 1.f;
  const int k_begin = (a.heads + kGroups - 1) / kGroups, v_begin = k_begin + (a.kv_heads + kGroups - 1) / kGroups;
  const int y0 = blockIdx.y * rounds_per_block, y1 = min(y0 + rounds_per_block, 2 * v_begin - k_begin);
  __syncthreads();

  const bool turns = rot > 0;
  int64_t next_slot = a.slot_map[blockIdx.x], next_pos = turns ? a.positions[blockIdx.x] : 0;  // (a token ahead)
  for (int64_t t = blockIdx.x; t < a.tokens; t += gridDim.x) {
    const int64_t slot = next_slot, pos = next_pos;
    if (t + gridDim.x < a.tokens) {
      next_slot = a.slot_map[t + gridDim.x];
      if (turns) next_pos = a.positions[t + gridDim.x];
    }
    const bool kept = slot >= 0 && slot < a.num_pages * a.page_size;
    float cs[4] = {1.f, 1.f, 1.f, 1.f}, sn[4] = {0.f, 0.f, 0.f, 0.f};
    if (turned) {
      if (pos >= 0 && pos < a.max_positions) {
        load4(a.cos_sin + pos * rot + 4 * lane, cs);
        load4(a.cos_sin + pos * rot + half + 4 * lane, sn);
      } else {  // no such position: the heads become NaN
#pragma unroll
        for (int i = 0; i < 4; ++i) cs[i] = sn[i] = __int_as_float(0x7FC00000);
      }
    }
    // rounds [r0, r1) of one kind of heads; f(x, y) makes them what is stored
    auto heads = [&](int r0, int r1, int n_heads, const Src* src, int64_t src_stride, void* out, int dtype, int64_t out_at, int64_t out_stride, auto f) {
      src += (int64_t)(r0 * kGroups + group) * src_stride;
      out_at += (int64_t)(r0 * kGroups + group) * out_stride;
      const int64_t src_step = kGroups * src_stride, out_step = kGroups * out_stride;
      for (int r = r0; r < r1; r += kAppendBatch) {  // (every lane of a warp makes the same number of rounds)
        Raw4<Src> raw[kAppendBatch][2];
        const int left = on ? n_heads - r * kGroups - group : 0;  // heads from this lane's on
#pragma unroll
        for (int u = 0; u < kAppendBatch; ++u) {
          if (u * kGroups < left && r + u < r1) {
            raw[u][0].load(src + lo);
            raw[u][1].load(src + hi);
          } else {
            raw[u][0].w = {};
            raw[u][1].w = {};
          }
          src += src_step;
        }
#pragma unroll
        for (int u = 0; u < kAppendBatch; ++u) {
          if (kAppendBatch > 1 && r + u >= r1) break;
          float x[4], y[4];
          raw[u][0].get(x);
          raw[u][1].get(y);
          f(x, y);
          if (u * kGroups < left) store8(out, dtype, out_at, lo, hi, x, y);
          out_at += out_step;
        }
      }
    };
    auto norm_rope_heads = [&](int r0, int r1, int n_heads, const Src* src, int64_t src_stride, int which, bool normed, void* out, int dtype, int64_t out_at,
                               int64_t out_stride) {
      if (r0 >= r1) return;
      // pairs (a, b) become (fa a - gb b, fb b + ga a) times the norm
      float fa[4], fb[4], ga[4], gb[4], wx[4] = {}, wy[4] = {};
      if (on) {
        load4(&s_weight[which][lo], wx);
        load4(&s_weight[which][hi], wy);
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float wa = INTERLEAVED ? (i < 2 ? wx[2 * i] : wy[2 * i - 4]) : wx[i], wb = INTERLEAVED ? (i < 2 ? wx[2 * i + 1] : wy[2 * i - 3]) : wy[i];
        fa[i] = wa * cs[i];
        fb[i] = wb * cs[i];
        ga[i] = wa * sn[i];
        gb[i] = wb * sn[i];
      }
      heads(r0, r1, n_heads, src, src_stride, out, dtype, out_at, out_stride, [&](float (&x)[4], float (&y)[4]) {
        // (the scale comes last: a rotation of values that it has made infinite would be NaN)
        float norm = s_scale[which];
        if (normed) {
          float sum = 0.f;
#pragma unroll
          for (int i = 0; i < 4; ++i) sum += x[i] * x[i] + y[i] * y[i];
#pragma unroll
          for (int o = LANES / 2; o > 0; o >>= 1) sum += __shfl_xor_sync(0xFFFFFFFFu, sum, o, LANES);
          norm *= rsqrtf(sum * inv_dim + a.eps);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          float& va = INTERLEAVED ? (i < 2 ? x[2 * i] : y[2 * i - 4]) : x[i];
          float& vb = INTERLEAVED ? (i < 2 ? x[2 * i + 1] : y[2 * i - 3]) : y[i];
          float na = va * fa[i], nb = vb * fb[i];
          if (turned) {
            na -= vb * gb[i];
            nb += va * ga[i];
          }
          va = na * norm;
          vb = nb * norm;
        }
      });
    };
    norm_rope_heads(y0, min(y1, k_begin), a.heads, static_cast<const Src*>(a.q) + t * a.q_token_stride, a.q_head_stride, 0, a.q_weight != nullptr, a.q_out,
                    a.q_out_dtype, t * a.heads * a.dim, a.dim);
    if (!kept) continue;
    const uint32_t page = (uint32_t)slot / (uint32_t)a.page_size, off = (uint32_t)slot - page * (uint32_t)a.page_size;
    norm_rope_heads(max(y0 - k_begin, 0), min(y1, v_begin) - k_begin, a.kv_heads, static_cast<const Src*>(a.k) + t * a.k_token_stride, a.k_head_stride, 1,
                    a.k_weight != nullptr, a.k_cache, a.cache_dtype, page * a.k_page_stride + off * a.k_slot_stride, a.k_cache_head_stride);
    heads(max(y0 - v_begin, 0), y1 - v_begin, a.kv_heads, static_cast<const Src*>(a.v) + t * a.v_token_stride, a.v_head_stride, a.v_cache, a.cache_dtype,
          page * a.v_page_stride + off * a.v_slot_stride, a.v_cache_head_stride, [&](float (&x)[4], float (&y)[4]) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              x[i] *= v_scale;
              y[i] *= v_scale;
            }
          });
  }
}

template <typename Src, int LANES, bool INTERLEAVED>
static int append_launch(const b200q_append_args& a, cudaStream_t st) {
  auto kernel = qk_norm_rope_append_kernel<Src, LANES, INTERLEAVED>;
  static std::atomic<int> resident[kMaxDevices];  // blocks per SM
  const int dev = current_device_index();
  if (dev < 0) return B200Q_ERR_CUDA;
  int per_sm = resident[dev].load(std::memory_order_acquire);
  if (!per_sm) {
    B200Q_CUDA_OK(cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per_sm, kernel, kAppendThreads, 0));
    if (per_sm < 1) per_sm = 1;
    resident[dev].store(per_sm, std::memory_order_release);
  }
  constexpr int kGroups = kAppendThreads / LANES;
  const int rounds = (a.heads + kGroups - 1) / kGroups + 2 * ((a.kv_heads + kGroups - 1) / kGroups);
  // Few tokens: a block per round or per batch of rounds, so that the whole device takes part.  Many: one resident set of blocks walks through
  // them (8192 tokens of 64 + 2 x 8 heads of 128 in bf16, caches in e4m3: 65.8 us = 4.9 TB/s, against 71 with a block per token).
  // us with a block per round / per batch / for all rounds of a token, of that shape (10 rounds): 16 tokens 2.57 / 2.70 / 4.87, 32 2.70 / 2.82 / 5.00,
  // 64 2.95 / 2.95 / 5.00, 96 3.98 / 3.21 / 5.01, 256 7.70 / 5.65 / 8.36, 384 10.5 / 8.21 / 8.87, 512 13.0 / 9.34 / 9.22, 1024 23.0 / 15.3 / 11.8: the limits
  // below are at 59 and 473 tokens.  3 rounds (8 + 2 x 1 heads): 64 2.57 / 2.95 / 3.33, 256 3.84 / 3.21 / 3.46, 1024 7.18 / 6.15 / 5.77 (limits 197 and 1184).
  const int64_t batches = (rounds + kAppendBatch - 1) / kAppendBatch;
  const int per = a.tokens * rounds <= 4 * kNumSMs ? 1 : a.tokens * batches <= 16 * kNumSMs ? kAppendBatch : rounds;
  const int64_t most = (int64_t)per_sm * kNumSMs;
  launch_dependent(kernel, dim3((unsigned)(a.tokens < most ? a.tokens : most), (unsigned)((rounds + per - 1) / per)), dim3(kAppendThreads), 0, st, a,
                   1.f / (float)a.dim, per);
  B200Q_LAUNCH_CHECK();
  return B200Q_OK;
}
template <typename Src, bool INTERLEAVED>
static int append_launch_dim(const b200q_append_args& a, cudaStream_t st) {
  if (a.dim <= 64) return append_launch<Src, 8, INTERLEAVED>(a, st);
  if (a.dim <= 128) return append_launch<Src, 16, INTERLEAVED>(a, st);
  return append_launch<Src, 32, INTERLEAVED>(a, st);
}

int qk_norm_rope_append_impl(const b200q_append_args& a, cudaStream_t st) {
  if (a.src_dtype == B200Q_BF16) return a.interleaved ? append_launch_dim<__nv_bfloat16, true>(a, st) : append_launch_dim<__nv_bfloat16, false>(a, st);
  return a.interleaved ? append_launch_dim<float, true>(a, st) : append_launch_dim<float, false>(a, st);
}

}  // namespace b200q
