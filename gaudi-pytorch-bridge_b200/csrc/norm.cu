// The norm in front of an FP8 product: the residual's addition, the root-mean-square norm and the cast to 8 bits (one scale for the
// tensor, or one per token from the token's own maximum), in one pass over the data.  Bound by memory where tokens are many (8192 x 8192 in bf16 with residual, to e4m3: 470 MB,
// 77 us, 6.1 TB/s, 0.93 of what a plain copy reaches) and by a trip to memory, a reduction and a trip back where they are few (1 x 8192: 3.2 us; 64 x 4096: 2.5 us).
#include <float.h>

#include "layer.cuh"
#include "tcgen05_ptx.cuh"

namespace b200q {

// ---------------------------------------------------------------------------- the mathematics of a token
// z = x (+ residual, rounded to its type), r = rsqrt(mean(z^2) + eps), y = (z w) r.  |y| is largest where |z w| is, whatever r (rounding is
// monotone), so that the sum of squares and the maximum come from one reduction, and a token's values are needed once.
struct NormSums {
  float squares;
  uint32_t top;  // bits of max |z w|: as integers, so that a NaN is above all and stays
};
__device__ __forceinline__ NormSums norm_join(const NormSums& a, const NormSums& b) { return {a.squares + b.squares, max(a.top, b.top)}; }

struct NormFactors {
  float norm;   // y = z w norm
  float scale;  // out = y scale
  float inverse;
};
__device__ __forceinline__ NormFactors norm_factors(const b200q_norm_args& a, const NormSums& s, float inv_dim, float given_scale) {
  NormFactors f;
  f.norm = rsqrtf(s.squares * inv_dim + a.eps);
  f.scale = given_scale;
  f.inverse = 1.f;
  if (a.scale_inv) {
    const float most = a.out_dtype == B200Q_E4M3 ? Fp8Fmt<B200Q_E4M3>::kMax : Fp8Fmt<B200Q_E5M2>::kMax;
    const float top = __uint_as_float(s.top) * f.norm;
    if (top != 0.f) {
      f.inverse = top / most;
      f.scale = most / top;
      if (f.scale > FLT_MAX) f.scale = FLT_MAX;  // (a NaN stays one)
    } else {
      f.scale = 1.f;
    }
  }
  return f;
}

// ---------------------------------------------------------------------------- values of a row, eight at a time or one at a time
template <typename T>
__device__ __forceinline__ float norm_get(const T* p);
template <>
__device__ __forceinline__ float norm_get(const float* p) { return *p; }
template <>
__device__ __forceinline__ float norm_get(const __nv_bfloat16* p) { return __bfloat162float(*p); }
__device__ __forceinline__ float norm_rounded(float v, const float*) { return v; }
__device__ __forceinline__ float norm_rounded(float v, const __nv_bfloat16*) { return round_to_bf16(v); }

__device__ __forceinline__ void norm_load8(const float* p, float (&v)[8]) {
  const float4 a = reinterpret_cast<const float4*>(p)[0], b = reinterpret_cast<const float4*>(p)[1];
  v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
  v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
}
__device__ __forceinline__ void norm_load8(const __nv_bfloat16* p, float (&v)[8]) {
  const uint4 w = *reinterpret_cast<const uint4*>(p);
  const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    v[2 * i] = __uint_as_float(u[i] << 16);
    v[2 * i + 1] = __uint_as_float(u[i] & 0xFFFF0000u);
  }
}
__device__ __forceinline__ void norm_store8(float* p, const float (&v)[8]) {
  reinterpret_cast<float4*>(p)[0] = make_float4(v[0], v[1], v[2], v[3]);
  reinterpret_cast<float4*>(p)[1] = make_float4(v[4], v[5], v[6], v[7]);
}
__device__ __forceinline__ void norm_store8(__nv_bfloat16* p, const float (&v)[8]) {
  *reinterpret_cast<uint4*>(p) = make_uint4(pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]), pack_bf16x2(v[4], v[5]), pack_bf16x2(v[6], v[7]));
}
template <int FMT>
__device__ __forceinline__ void norm_store8_fp8(uint8_t* p, const float (&v)[8]) {
  *reinterpret_cast<uint2*>(p) = make_uint2(cvt_fp8x2<FMT>(v[0], v[1]) | (cvt_fp8x2<FMT>(v[2], v[3]) << 16),
                                            cvt_fp8x2<FMT>(v[4], v[5]) | (cvt_fp8x2<FMT>(v[6], v[7]) << 16));
}
__device__ __forceinline__ void norm_out8(const b200q_norm_args& a, int64_t at, float (&v)[8]) {
  if (a.out_dtype == B200Q_E4M3) norm_store8_fp8<B200Q_E4M3>(static_cast<uint8_t*>(a.out) + at, v);
  else if (a.out_dtype == B200Q_E5M2) norm_store8_fp8<B200Q_E5M2>(static_cast<uint8_t*>(a.out) + at, v);
  else norm_store8(static_cast<__nv_bfloat16*>(a.out) + at, v);
}
__device__ __forceinline__ void norm_out1(const b200q_norm_args& a, int64_t at, float v) {
  if (a.out_dtype == B200Q_E4M3) static_cast<uint8_t*>(a.out)[at] = (uint8_t)cvt_fp8x2<B200Q_E4M3>(v, 0.f);
  else if (a.out_dtype == B200Q_E5M2) static_cast<uint8_t*>(a.out)[at] = (uint8_t)cvt_fp8x2<B200Q_E5M2>(v, 0.f);
  else static_cast<__nv_bfloat16*>(a.out)[at] = __float2bfloat16_rn(v);
}
__device__ __forceinline__ float norm_weight(const b200q_norm_args& a, int64_t at) {
  if (!a.weight) return 1.f;
  return a.weight_dtype == B200Q_BF16 ? norm_get(static_cast<const __nv_bfloat16*>(a.weight) + at) : static_cast<const float*>(a.weight)[at];
}

// How a row lies: on boundaries of eight values (16-byte accesses); on any boundary, but the same in x, residual and the outputs (rows of an
// odd length one behind the other: 16-byte accesses between the row's ends); or in any other way (value by value).
enum NormForm { kNormEven, kNormShifted, kNormLoose };

// the weights of the eight values from `at` on, of a row that begins `shift` values behind such a boundary; 0 outside the row
template <int FORM, int THREADS>
__device__ __forceinline__ void norm_weights(const b200q_norm_args& a, int at, int v, int tid, int dim, float (&w)[8]) {
#pragma unroll
  for (int i = 0; i < 8; ++i) w[i] = a.weight ? 0.f : 1.f;
  if (!a.weight) return;
  if (FORM == kNormEven) {
    if (at >= dim) return;
    if (a.weight_dtype == B200Q_BF16) norm_load8(static_cast<const __nv_bfloat16*>(a.weight) + at, w);
    else norm_load8(static_cast<const float*>(a.weight) + at, w);
  } else {
    if (FORM == kNormShifted && at >= dim) return;
    const int off = -at & 7;  // of the eight, so many lie before the next boundary; the same for all vectors of a row
    if (FORM == kNormShifted && a.weight_dtype == B200Q_BF16 && off != 0 && at >= 0 && at + off + 8 <= dim) {
      // sixteen values on boundaries, moved by 8 - off places: value by value the weights would be half of a row's instructions
      const uint4* p = reinterpret_cast<const uint4*>(static_cast<const __nv_bfloat16*>(a.weight) + (at + off - 8));
      const uint4 lo = p[0], hi = p[1];
      uint32_t u[8] = {lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w};
      const int by = 8 - off;
#pragma unroll
      for (int i = 0; i < 6; ++i) u[i] = by & 4 ? u[i + 2] : u[i];
#pragma unroll
      for (int i = 0; i < 5; ++i) u[i] = by & 2 ? u[i + 1] : u[i];
#pragma unroll
      for (int i = 0; i < 4; ++i) u[i] = by & 1 ? __funnelshift_r(u[i], u[i + 1], 16) : u[i];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        w[2 * i] = __uint_as_float(u[i] << 16);
        w[2 * i + 1] = __uint_as_float(u[i] & 0xFFFF0000u);
      }
      return;
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int k = FORM == kNormShifted ? at + i : (v * 8 + i) * THREADS + tid;
      if (k >= 0 && k < dim) w[i] = norm_weight(a, k);
    }
  }
}

// ---------------------------------------------------------------------------- rows of any length
// Three passes by one block; the second and third find the row in L2 (z lies in residual where there is one).
constexpr int kNormLongThreads = 1024;
template <typename T>
__global__ void __launch_bounds__(kNormLongThreads) norm_long_kernel(const b200q_norm_args a, float inv_dim) {
  __shared__ NormSums s_warp[kNormLongThreads / 32];
  pdl_enter();
  const int tid = threadIdx.x;
  const float given = a.scale ? *a.scale : 1.f;
  for (int64_t t = blockIdx.x; t < a.tokens; t += gridDim.x) {
    const T* x = static_cast<const T*>(a.x) + t * a.x_stride;
    T* residual = a.residual ? static_cast<T*>(a.residual) + t * a.residual_stride : nullptr;
    NormSums s = {0.f, 0u};
    for (int64_t i = tid; i < a.dim; i += kNormLongThreads) {
      float z = norm_get(x + i);
      if (residual) {
        z = norm_rounded(norm_get(residual + i) + z, x);
        residual[i] = T(z);
      }
      s = norm_join(s, {z * z, __float_as_uint(z * norm_weight(a, i)) & 0x7FFFFFFFu});
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) s = norm_join(s, {__shfl_xor_sync(0xFFFFFFFFu, s.squares, o), __shfl_xor_sync(0xFFFFFFFFu, s.top, o)});
    __syncthreads();
    if ((tid & 31) == 0) s_warp[tid >> 5] = s;
    __syncthreads();
    s = s_warp[0];
    for (int i = 1; i < kNormLongThreads / 32; ++i) s = norm_join(s, s_warp[i]);
    const NormFactors f = norm_factors(a, s, inv_dim, given);
    if (a.scale_inv && tid == 0) a.scale_inv[t] = f.inverse;
    const T* z = residual ? residual : x;
    for (int64_t i = tid; i < a.dim; i += kNormLongThreads) {
      const float y = norm_get(z + i) * norm_weight(a, i) * f.norm;
      if (a.kept) static_cast<__nv_bfloat16*>(a.kept)[t * a.dim + i] = __float2bfloat16_rn(y);
      norm_out1(a, t * a.dim + i, y * f.scale);
    }
  }
}

// ---------------------------------------------------------------------------- rows that fit the registers
// A row belongs to THREADS threads (a warp, or a whole block), which hold it in registers: VECS times eight values each, in 16-byte accesses
// (WIDE), or 8 VECS times one value where rows do not lie on such boundaries.  Everything is loaded before anything is used.
template <typename T>
struct NormRaw8;
template <>
struct NormRaw8<__nv_bfloat16> {
  uint4 w;
  __device__ __forceinline__ void load(const __nv_bfloat16* p) { w = *reinterpret_cast<const uint4*>(p); }
  __device__ __forceinline__ void get(float (&v)[8]) const {
    const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      v[2 * i] = __uint_as_float(u[i] << 16);
      v[2 * i + 1] = __uint_as_float(u[i] & 0xFFFF0000u);
    }
  }
};
template <>
struct NormRaw8<float> {
  float4 a, b;
  __device__ __forceinline__ void load(const float* p) {
    a = reinterpret_cast<const float4*>(p)[0];
    b = reinterpret_cast<const float4*>(p)[1];
  }
  __device__ __forceinline__ void get(float (&v)[8]) const {
    v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
    v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
  }
};

template <typename T, int FORM, int THREADS, int VECS>
__global__ void __launch_bounds__(THREADS < 128 ? 128 : THREADS) norm_row_kernel(const b200q_norm_args a, float inv_dim) {
  constexpr int kBlock = THREADS < 128 ? 128 : THREADS, kRows = kBlock / THREADS, kWarps = THREADS / 32;
  __shared__ NormSums s_warp[2][kWarps];  // (the other half is written for the next row, and this one only behind its barrier)
  pdl_enter();
  const int tid = threadIdx.x % THREADS, dim = (int)a.dim;
  const float given = a.scale ? *a.scale : 1.f;
  const int64_t step = (int64_t)gridDim.x * kRows;
  // a thread's vector v of row t: values at .. at + 7, of which (kNormShifted) some may lie outside the row
  auto shift_of = [&](int64_t t) { return FORM == kNormShifted ? (int)((t * dim) & 7) : 0; };
  auto begin = [&](int v, int shift) { return (v * THREADS + tid) * 8 - shift; };
  auto inside = [&](int at) { return at >= 0 && at + 8 <= dim; };
  NormRaw8<T> rx[VECS], rr[VECS];  // of the row that is next: on its way while the one before is reduced
  auto load = [&](int64_t t) {
    const T* x = static_cast<const T*>(a.x) + t * a.x_stride;
    const T* residual = static_cast<const T*>(a.residual) + t * a.residual_stride;
    const int shift = shift_of(t);
#pragma unroll
    for (int v = 0; v < VECS; ++v) {
      const int at = begin(v, shift);
      if (inside(at)) {
        rx[v].load(x + at);
        if (a.residual) rr[v].load(residual + at);
      }
    }
  };
  int64_t t = (int64_t)blockIdx.x * kRows + threadIdx.x / THREADS;
  if (FORM != kNormLoose && t < a.tokens) load(t);
  for (int turn = 0; t < a.tokens; t += step, turn ^= 1) {
    const T* x = static_cast<const T*>(a.x) + t * a.x_stride;
    T* residual = a.residual ? static_cast<T*>(a.residual) + t * a.residual_stride : nullptr;
    const int shift = shift_of(t);
    float z[VECS][8];
    NormSums s = {0.f, 0u};
    if (FORM != kNormLoose) {
#pragma unroll
      for (int v = 0; v < VECS; ++v) {
        const int at = begin(v, shift);
        if (inside(at)) {
          rx[v].get(z[v]);
          if (residual) {
            float r[8];
            rr[v].get(r);
#pragma unroll
            for (int i = 0; i < 8; ++i) z[v][i] = norm_rounded(r[i] + z[v][i], x);
            norm_store8(residual + at, z[v]);
          }
        } else {
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            z[v][i] = 0.f;
            if (FORM == kNormShifted && at + i >= 0 && at + i < dim) {  // (an end of the row)
              z[v][i] = norm_get(x + at + i);
              if (residual) {
                z[v][i] = norm_rounded(norm_get(residual + at + i) + z[v][i], x);
                residual[at + i] = T(z[v][i]);
              }
            }
          }
        }
      }
      if (t + step < a.tokens) load(t + step);
    } else {
#pragma unroll
      for (int v = 0; v < VECS; ++v)
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const int at = (v * 8 + i) * THREADS + tid;
          z[v][i] = at < dim ? norm_get(x + at) : 0.f;
        }
      if (residual) {
#pragma unroll
        for (int v = 0; v < VECS; ++v) {
          float r[8];
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const int at = (v * 8 + i) * THREADS + tid;
            r[i] = at < dim ? norm_get(residual + at) : 0.f;
          }
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const int at = (v * 8 + i) * THREADS + tid;
            z[v][i] = norm_rounded(r[i] + z[v][i], x);
            if (at < dim) residual[at] = T(z[v][i]);
          }
        }
      }
    }
#pragma unroll
    for (int v = 0; v < VECS; ++v) {
      float w[8];
      norm_weights<FORM, THREADS>(a, begin(v, shift), v, tid, dim, w);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        s.squares += z[v][i] * z[v][i];
        z[v][i] *= w[i];
        s.top = max(s.top, __float_as_uint(z[v][i]) & 0x7FFFFFFFu);
      }
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) s = norm_join(s, {__shfl_xor_sync(0xFFFFFFFFu, s.squares, o), __shfl_xor_sync(0xFFFFFFFFu, s.top, o)});
    if (kWarps > 1) {
      if ((tid & 31) == 0) s_warp[turn][tid >> 5] = s;
      __syncthreads();
      s = s_warp[turn][tid & (kWarps - 1)];
#pragma unroll
      for (int o = kWarps / 2; o > 0; o >>= 1) s = norm_join(s, {__shfl_xor_sync(0xFFFFFFFFu, s.squares, o), __shfl_xor_sync(0xFFFFFFFFu, s.top, o)});
    }
    const NormFactors f = norm_factors(a, s, inv_dim, given);
    if (a.scale_inv && tid == 0) a.scale_inv[t] = f.inverse;
#pragma unroll
    for (int v = 0; v < VECS; ++v) {
      const int at = begin(v, shift);
      if (FORM != kNormLoose && inside(at)) {
#pragma unroll
        for (int i = 0; i < 8; ++i) z[v][i] *= f.norm;
        if (a.kept) norm_store8(static_cast<__nv_bfloat16*>(a.kept) + t * dim + at, z[v]);
#pragma unroll
        for (int i = 0; i < 8; ++i) z[v][i] *= f.scale;
        norm_out8(a, t * dim + at, z[v]);
      } else if (FORM != kNormEven) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const int k = FORM == kNormShifted ? at + i : (v * 8 + i) * THREADS + tid;
          if (k < 0 || k >= dim) continue;
          const float y = z[v][i] * f.norm;
          if (a.kept) static_cast<__nv_bfloat16*>(a.kept)[t * dim + k] = __float2bfloat16_rn(y);
          norm_out1(a, t * dim + k, y * f.scale);
        }
      }
    }
  }
}

template <typename T, int FORM, int THREADS, int VECS>
static int norm_launch(const b200q_norm_args& a, float inv_dim, cudaStream_t st) {
  auto kernel = norm_row_kernel<T, FORM, THREADS, VECS>;
  constexpr int kBlock = THREADS < 128 ? 128 : THREADS, kRows = kBlock / THREADS;
  static std::atomic<int> resident[kMaxDevices];  // blocks per SM
  const int dev = current_device_index();
  if (dev < 0) return B200Q_ERR_CUDA;
  int per_sm = resident[dev].load(std::memory_order_acquire);
  if (!per_sm) {
    B200Q_CUDA_OK(cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per_sm, kernel, kBlock, 0));
    if (per_sm < 1) per_sm = 1;
    resident[dev].store(per_sm, std::memory_order_release);
  }
  const int64_t blocks = (a.tokens + kRows - 1) / kRows, most = (int64_t)per_sm * kNumSMs;
  launch_dependent(kernel, dim3((unsigned)(blocks < most ? blocks : most)), dim3(kBlock), 0, st, a, inv_dim);
  B200Q_LAUNCH_CHECK();
  return B200Q_OK;
}

// ---------------------------------------------------------------------------- many long rows
// The same with the rows on their way to shared memory, as bulk copies: what is in flight then costs no registers, and a block that
// waits for its sums has its next rows coming: 77 us for 8192 x 8192 where rows ahead in registers took 91.  In fp32 138 us (6.3 TB/s); 16384 x 4096 77, 32768 x 2048 78,
// 65536 x 1024 88, 4096 x 16384 79, 2000 x 32768 84 us.  Blocks of 512 threads with two vectors each, two on an SM, are the best for 8192 values: 256 threads with four 82, 128
// with eight 87, 512 with four 86, one block on an SM 107.  A row that begins between boundaries (kNormShifted) is fetched from the boundary before it to the one
// behind it; what that brings of its neighbours is masked out, and behind the last row nothing is fetched: its end is read value by value.  8000 x 8189: 180 us, bound by
// instructions (masks, and weights that have to be moved into place), where value by value it was 288; 4096 x 13433: 114 us.
constexpr int kNormErrCopy = 811;  // status code: a copy of a row did not arrive
constexpr uint32_t kNormTestPolls = 1u << 14;  // of the self-test: some ten milliseconds
constexpr int kNormRingBytes = 216 * 1024;  // of an SM

__device__ __forceinline__ void norm_bulk_copy(uint32_t dst, const void* src, uint32_t bytes, uint32_t bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst), "l"(src), "r"(bytes), "r"(bar) : "memory");
}

template <typename T>
__host__ __device__ constexpr int64_t norm_slot_row(int64_t dim, int form) {  // bytes of a row's place
  return (dim + (form == kNormShifted ? 7 : 0) + 7) / 8 * 8 * (int64_t)sizeof(T);  // (all vectors that begin in the row end in its place)
}

template <typename T, int FORM, int THREADS, int VECS, int BLOCKS, bool TEST>  // TEST: short waits, and block 0's first row is never copied
__global__ void __launch_bounds__(THREADS, BLOCKS) norm_ring_kernel(const b200q_norm_args a, float inv_dim, int depth, int* status) {
  constexpr int kWarps = THREADS / 32, kMostDepth = 8;
  extern __shared__ __align__(128) uint8_t s_ring[];  // [depth] rows of x, with that of residual behind it
  __shared__ __align__(8) uint64_t s_bars[kMostDepth];
  __shared__ NormSums s_warp[2][kWarps];
  __shared__ int s_abort;
  const int tid = threadIdx.x, dim = (int)a.dim;
  constexpr bool kShifted = FORM == kNormShifted;
  const uint32_t bars = ptx::smem_u32(s_bars), ring = ptx::smem_u32(s_ring);
  const uint32_t row = (uint32_t)norm_slot_row<T>(dim, FORM), slot_bytes = a.residual ? 2 * row : row;
  auto shift_of = [&](int64_t t) { return kShifted ? (int)((t * dim) & 7) : 0; };
  auto bytes_of = [&](int64_t t) {  // of a row that are fetched
    const uint32_t n = (uint32_t)((shift_of(t) + dim) * sizeof(T));
    return !kShifted || t + 1 < a.tokens ? (n + 15u) & ~15u : n & ~15u;
  };
  if (tid == 0) {
    for (int i = 0; i < depth; ++i) ptx::mbar_init(bars + 8 * i, 1);
    s_abort = 0;
    ptx::fence_barrier_init();
  }
  __syncthreads();
  pdl_enter();
  const float given = a.scale ? *a.scale : 1.f;
  auto copy = [&](int64_t t, int slot) {  // (one thread)
    const uint32_t bytes = bytes_of(t);
    const int64_t back = shift_of(t);
    ptx::mbar_arrive_expect_tx(bars + 8 * slot, a.residual ? 2 * bytes : bytes);
    if (TEST && t == 0) return;
    norm_bulk_copy(ring + slot * slot_bytes, static_cast<const T*>(a.x) + (t * a.x_stride - back), bytes, bars + 8 * slot);
    if (a.residual)
      norm_bulk_copy(ring + slot * slot_bytes + row, static_cast<const T*>(a.residual) + (t * a.residual_stride - back), bytes, bars + 8 * slot);
  };
  if (tid == 0)
    for (int i = 0; i < depth && (int64_t)blockIdx.x + (int64_t)i * gridDim.x < a.tokens; ++i) copy((int64_t)blockIdx.x + (int64_t)i * gridDim.x, i);
  int slot = 0, turn = 0;
  uint32_t phase = 0;
  for (int64_t t = blockIdx.x; t < a.tokens; t += gridDim.x, turn ^= 1) {
    const bool here = ptx::mbar_wait(bars + 8 * slot, phase, &s_abort, status, kNormErrCopy, 0, TEST ? kNormTestPolls : ptx::kWaitLimit);
    const T* x = reinterpret_cast<const T*>(s_ring + slot * slot_bytes);
    T* residual = static_cast<T*>(a.residual) + t * a.residual_stride;
    const int shift = shift_of(t);
    auto begin = [&](int v) { return (v * THREADS + tid) * 8 - shift; };
    auto inside = [&](int at) { return at >= 0 && at + 8 <= dim; };
    // values at .. at + 7 of the row in shared memory at p, which lies at `from` in global memory
    auto get = [&](const T* p, const T* from, int at, float (&v)[8]) {
      norm_load8(p + at + shift, v);
      if (kShifted && !inside(at)) {
        const int there = (int)(bytes_of(t) / sizeof(T)) - shift;
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = at + i < 0 || at + i >= dim ? 0.f : at + i < there ? v[i] : norm_get(from + at + i);
      }
    };
    float z[VECS][8];
    NormSums s = {0.f, 0u};
#pragma unroll
    for (int v = 0; v < VECS; ++v) {
      const int at = begin(v);
      if (here && at < dim) {
        get(x, static_cast<const T*>(a.x) + t * a.x_stride, at, z[v]);
        if (a.residual) {
          float r[8];
          get(x + row / sizeof(T), residual, at, r);
#pragma unroll
          for (int i = 0; i < 8; ++i) z[v][i] = norm_rounded(r[i] + z[v][i], x);
          if (inside(at)) {
            norm_store8(residual + at, z[v]);
          } else if (kShifted) {
#pragma unroll
            for (int i = 0; i < 8; ++i)
              if (at + i >= 0 && at + i < dim) residual[at + i] = T(z[v][i]);
          }
        }
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) z[v][i] = 0.f;
      }
    }
#pragma unroll
    for (int v = 0; v < VECS; ++v) {
      float w[8];
      norm_weights<FORM, THREADS>(a, begin(v), v, tid, dim, w);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        s.squares += z[v][i] * z[v][i];
        z[v][i] *= w[i];
        s.top = max(s.top, __float_as_uint(z[v][i]) & 0x7FFFFFFFu);
      }
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) s = norm_join(s, {__shfl_xor_sync(0xFFFFFFFFu, s.squares, o), __shfl_xor_sync(0xFFFFFFFFu, s.top, o)});
    if ((tid & 31) == 0) s_warp[turn][tid >> 5] = s;
    __syncthreads();  // (and the slot has been read by all)
    // A copy is missing: nothing more is written, and the copies in flight are waited for, as far as they come.  (All threads see the same: one that waits for the next row in vain
    // says so long after the others have looked.  A flag for each of two rows, or a barrier that carries it, cost registers: rows of odd lengths 180 -> 191 to 194 us.)
    if (s_abort) {
      if (tid == 0)
        for (int i = 0; i < depth && t + (int64_t)i * gridDim.x < a.tokens; ++i) {
          const int at = slot + i < depth ? slot + i : slot + i - depth;
          for (int k = 0; k < 4096 && !ptx::mbar_try_wait(bars + 8 * at, slot + i < depth ? phase : phase ^ 1); ++k) __nanosleep(64);
        }
      break;
    }
    if (tid == 0 && t + (int64_t)depth * gridDim.x < a.tokens) copy(t + (int64_t)depth * gridDim.x, slot);
    s = s_warp[turn][tid & (kWarps - 1)];
#pragma unroll
    for (int o = kWarps / 2; o > 0; o >>= 1) s = norm_join(s, {__shfl_xor_sync(0xFFFFFFFFu, s.squares, o), __shfl_xor_sync(0xFFFFFFFFu, s.top, o)});
    const NormFactors f = norm_factors(a, s, inv_dim, given);
    if (a.scale_inv && tid == 0) a.scale_inv[t] = f.inverse;
#pragma unroll
    for (int v = 0; v < VECS; ++v) {
      const int at = begin(v);
      if (at >= dim) continue;
#pragma unroll
      for (int i = 0; i < 8; ++i) z[v][i] *= f.norm;
      if (inside(at)) {
        if (a.kept) norm_store8(static_cast<__nv_bfloat16*>(a.kept) + t * dim + at, z[v]);
#pragma unroll
        for (int i = 0; i < 8; ++i) z[v][i] *= f.scale;
        norm_out8(a, t * dim + at, z[v]);
      } else if (kShifted) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          if (at + i < 0 || at + i >= dim) continue;
          if (a.kept) static_cast<__nv_bfloat16*>(a.kept)[t * dim + at + i] = __float2bfloat16_rn(z[v][i]);
          norm_out1(a, t * dim + at + i, z[v][i] * f.scale);
        }
      }
    }
    if (++slot == depth) {
      slot = 0;
      phase ^= 1;
    }
  }
}

template <typename T, int FORM, int THREADS, int VECS, int BLOCKS, bool TEST = false>
static int norm_launch_ring(const b200q_norm_args& a, float inv_dim, cudaStream_t st) {
  auto kernel = norm_ring_kernel<T, FORM, THREADS, VECS, BLOCKS, TEST>;
  constexpr int kMost = kNormRingBytes / BLOCKS / 1024 * 1024;
  static std::atomic<int> ready[kMaxDevices];
  const int dev = current_device_index();
  if (dev < 0) return B200Q_ERR_CUDA;
  if (!ready[dev].load(std::memory_order_acquire)) {
    B200Q_CUDA_OK(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kMost));
    ready[dev].store(1, std::memory_order_release);
  }
  int* status = device_status_ptr();
  if (!status) return B200Q_ERR_CUDA;
  const int64_t bytes = norm_slot_row<T>(a.dim, FORM) * (a.residual ? 2 : 1);
  const int64_t fits = kMost / bytes;
  const int depth = fits < 1 ? 0 : fits < 8 ? (int)fits : 8;
  if (!depth) return B200Q_ERR_UNSUPPORTED;
  const int64_t most = (int64_t)BLOCKS * kNumSMs;
  launch_dependent(kernel, dim3((unsigned)(a.tokens < most ? a.tokens : most)), dim3(THREADS), (size_t)(depth * bytes), st, a, inv_dim, depth, status);
  B200Q_LAUNCH_CHECK();
  return B200Q_OK;
}

// At most a row to an SM: as many threads to a row as it has use for, everything asked for at once.  (A ring would add the trip through shared memory.)
template <typename T, int FORM>
static int norm_launch_few(const b200q_norm_args& a, float inv_dim, cudaStream_t st) {
  const int64_t dim = a.dim + (FORM == kNormShifted ? 7 : 0);
  if (dim <= 256) return norm_launch<T, FORM, 32, 1>(a, inv_dim, st);
  if (dim <= 1024) return norm_launch<T, FORM, 128, 1>(a, inv_dim, st);
  if (dim <= 4096) return norm_launch<T, FORM, 512, 1>(a, inv_dim, st);
  if (dim <= 8192) return norm_launch<T, FORM, 1024, 1>(a, inv_dim, st);
  if (dim <= 16384) return norm_launch<T, FORM, 1024, 2>(a, inv_dim, st);
  return norm_launch<T, FORM, 1024, 4>(a, inv_dim, st);
}
template <typename T, int FORM>
static int norm_launch_many(const b200q_norm_args& a, float inv_dim, cudaStream_t st) {
  const int64_t dim = a.dim + (FORM == kNormShifted ? 7 : 0);
  if (dim <= 256) return norm_launch<T, FORM, 32, 1>(a, inv_dim, st);
  if (dim <= 512) return norm_launch<T, FORM, 32, 2>(a, inv_dim, st);
  if constexpr (FORM != kNormLoose) {
    int rc = B200Q_ERR_UNSUPPORTED;
    if (dim <= 1024) rc = norm_launch_ring<T, FORM, 64, 2, 12>(a, inv_dim, st);
    else if (dim <= 2048) rc = norm_launch_ring<T, FORM, 128, 2, 6>(a, inv_dim, st);
    // (us with six blocks of 128 threads an SM and with four of 256, 60e6 values, bf16 with residual / without / fp32 with, half as many / without: 2624 88, 93 / 64, 78 / 67, 72 / 71, 78; 2816 76,
    // 87 / 61, 73 / 68, 70 / 61, 73; 3008 75, 83 / 58, 70 / 70, 69 / 60, 69; 3200 86, 81 / 63, 68 / 69, 66 / 61, 67; 3584 79, 75 / 54, 62 / 69, 66 / 60, 62; 4096 75, 71 / 49, 56 / 68, 67 / 55, 57.
    // Rows of odd lengths, bf16 with residual: 2817 143, 175; 3001 136, 139; 3201 180, 135; 4001 120, 114)
    else if (dim <= 3008 || (dim <= 4096 && !a.residual && FORM == kNormEven)) rc = norm_launch_ring<T, FORM, 128, 4, 6>(a, inv_dim, st);
    else if (dim <= 4096) rc = norm_launch_ring<T, FORM, 256, 2, 4>(a, inv_dim, st);
    else if (dim <= 8192) rc = norm_launch_ring<T, FORM, 512, 2, 2>(a, inv_dim, st);
    else if (dim <= 16384) rc = norm_launch_ring<T, FORM, 512, 4, 2>(a, inv_dim, st);
    else rc = norm_launch_ring<T, FORM, 1024, 4, 1>(a, inv_dim, st);
    if (rc != B200Q_ERR_UNSUPPORTED) return rc;  // (rows too long for shared memory)
    return norm_launch<T, FORM, 1024, 4>(a, inv_dim, st);
  }
  if (dim <= 1024) return norm_launch<T, FORM, 128, 1>(a, inv_dim, st);
  if (dim <= 4096) return norm_launch<T, FORM, 256, 2>(a, inv_dim, st);
  if (dim <= 16384) return norm_launch<T, FORM, 512, 4>(a, inv_dim, st);
  return norm_launch<T, FORM, 1024, 4>(a, inv_dim, st);
}
template <typename T, int FORM>
static int norm_launch_form(const b200q_norm_args& a, float inv_dim, cudaStream_t st) {
  return a.tokens <= kNumSMs ? norm_launch_few<T, FORM>(a, inv_dim, st) : norm_launch_many<T, FORM>(a, inv_dim, st);
}

static NormForm norm_form(const b200q_norm_args& a) {
  bool aligned = true;
  for (const void* p : {a.x, static_cast<const void*>(a.residual), a.weight, static_cast<const void*>(a.out), static_cast<const void*>(a.kept)})
    aligned = aligned && reinterpret_cast<uintptr_t>(p) % 16 == 0;
  const int64_t strides[2] = {a.x_stride, a.residual ? a.residual_stride : a.x_stride};
  const bool one = a.tokens == 1;  // (no stride is used)
  if (aligned && a.dim % 8 == 0 && (one || (strides[0] % 8 == 0 && strides[1] % 8 == 0))) return kNormEven;
  // (rows that overlap: what is fetched beyond a row could lie behind the last one)
  if (aligned && (one || ((strides[0] - a.dim) % 8 == 0 && (strides[1] - a.dim) % 8 == 0 && strides[0] >= a.dim))) return kNormShifted;
  return kNormLoose;
}

template <typename T>
static int norm_launch_type(const b200q_norm_args& a, float inv_dim, cudaStream_t st) {
  if (a.dim > 32768 || (a.dim > 32760 && a.dim % 8)) {
    const unsigned grid = (unsigned)(a.tokens < 2 * kNumSMs ? a.tokens : 2 * kNumSMs);
    launch_dependent(norm_long_kernel<T>, dim3(grid), dim3(kNormLongThreads), 0, st, a, inv_dim);
    B200Q_LAUNCH_CHECK();
    return B200Q_OK;
  }
  switch (norm_form(a)) {
    case kNormEven: return norm_launch_form<T, kNormEven>(a, inv_dim, st);
    case kNormShifted: return norm_launch_form<T, kNormShifted>(a, inv_dim, st);
    default: return norm_launch_form<T, kNormLoose>(a, inv_dim, st);
  }
}

int add_rms_norm_cast_impl(const b200q_norm_args& a, cudaStream_t st) {
  const float inv_dim = a.dim ? 1.f / (float)a.dim : 0.f;
  return a.x_dtype == B200Q_BF16 ? norm_launch_type<__nv_bfloat16>(a, inv_dim, st) : norm_launch_type<float>(a, inv_dim, st);
}

int norm_selftest_impl(const b200q_norm_args& a, cudaStream_t st) {
  if (a.x_dtype != B200Q_BF16 || a.dim <= 4096 || a.dim > 8192 || a.tokens <= kNumSMs || norm_form(a) != kNormEven) return B200Q_ERR_UNSUPPORTED;
  return norm_launch_ring<__nv_bfloat16, kNormEven, 512, 2, 2, true>(a, 1.f / (float)a.dim, st);
}

}  // namespace b200q
