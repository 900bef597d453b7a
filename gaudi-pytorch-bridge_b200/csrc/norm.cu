// The norm in front of an FP8 product: the residual's addition, the root-mean-square norm and the cast to 8 bits (one scale for the
// tensor, or one per token from the token's own maximum), in one pass over the data.
#include <float.h>

#include "layer.cuh"

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

int add_rms_norm_cast_impl(const b200q_norm_args& a, cudaStream_t st) {
  const float inv_dim = a.dim ? 1.f / (float)a.dim : 0.f;
  const unsigned grid = (unsigned)(a.tokens < 2 * kNumSMs ? a.tokens : 2 * kNumSMs);
  if (a.x_dtype == B200Q_BF16) launch_dependent(norm_long_kernel<__nv_bfloat16>, dim3(grid), dim3(kNormLongThreads), 0, st, a, inv_dim);
  else launch_dependent(norm_long_kernel<float>, dim3(grid), dim3(kNormLongThreads), 0, st, a, inv_dim);
  B200Q_LAUNCH_CHECK();
  return B200Q_OK;
}

}  // namespace b200q
