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

// ---------------------------------------------------------------------------- tensor cores
// Bound by memory: the adapters that are used where tokens are few, y (read and written) where they are many.  Tokens of one adapter have to be
// taken together, in whatever order they come, or its matrices are read again for each: a first kernel sorts the tokens by adapter into tiles of 32.
// Then a x and b (a x) are m16n8k16 products on fragments that come straight from global memory, 16 bytes a lane: the values of K may be taken in any
// order as long as both operands take the same one, and so may the columns of y, whose order is such that a lane has 16 neighbours.
constexpr int kLoraTile = 32;
constexpr int kLoraSortThreads = 1024;
constexpr int kLoraThreads = 256;

struct LoraTile {
  int adapter, first, count, unused;  // tokens sorted[first] ...
};
struct LoraPlan {
  int* tiles_used;
  LoraTile* tiles;
  int* sorted;
  float* low;  // [splits][tokens][rank]: a x, in parts over k
  int splits, slice;  // values of k per part
};
struct LoraSpace {
  size_t tiles, sorted, low, bytes;
  LoraSpace(int64_t tokens, int64_t rank, int64_t splits) {
    const size_t t = (size_t)(tokens < kLoraChunk ? tokens : kLoraChunk);
    tiles = 256;
    sorted = lora_align(tiles + sizeof(LoraTile) * t);
    low = lora_align(sorted + sizeof(int) * t);
    bytes = lora_align(low + sizeof(float) * t * (size_t)(rank * splits));
  }
};
// tiles that the tokens may need at most; parts of k and of n such that as many CTAs have work as there are SMs, twice over
static int64_t lora_most_tiles(int64_t tokens, int64_t adapters) {
  const int64_t t = tokens < kLoraChunk ? tokens : kLoraChunk, shared = adapters + t / kLoraTile;
  return t < shared ? t : shared;
}
static int64_t lora_splits(int64_t tokens, int64_t k, int64_t adapters) {
  const int64_t most = (k + 255) / 256, wanted = (2 * kNumSMs + lora_most_tiles(tokens, adapters) - 1) / lora_most_tiles(tokens, adapters);
  return wanted < 1 ? 1 : wanted < most ? (wanted < 16 ? wanted : 16) : (most < 16 ? most : 16);
}

__device__ __forceinline__ void lora_mma(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
               : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// A stable counting sort by one block: each warp has a run of the tokens and counts of its own.
__global__ void __launch_bounds__(kLoraSortThreads) lora_sort_kernel(const b200q_lora_args a, const LoraPlan p) {
  constexpr int kWarps = kLoraSortThreads / 32;
  extern __shared__ uint16_t s_count[];  // [warps][adapters], then [adapters]: an adapter's first place
  __shared__ int s_scan[2][kWarps];
  pdl_enter();
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, adapters = (int)a.adapters, tokens = (int)a.tokens;
  uint16_t* const mine = s_count + warp * adapters;
  uint16_t* const s_first = s_count + kWarps * adapters;
  for (int i = tid; i < kWarps * adapters; i += kLoraSortThreads) s_count[i] = 0;
  __syncthreads();
  const int per = (tokens + 32 * kWarps - 1) / (32 * kWarps) * 32, begin = warp * per, end = min(begin + per, tokens);
  for (int base = begin; base < end; base += 32) {
    const int t = base + lane, i = t < end ? lora_adapter(a, t) : -1;
    const uint32_t same = __match_any_sync(0xFFFFFFFFu, i);
    if (i >= 0 && lane == __ffs(same) - 1) mine[i] += (uint16_t)__popc(same);
    __syncwarp();
  }
  __syncthreads();
  int tokens_before = 0, tiles_before = 0;
  for (int base = 0, turn = 0; base < adapters; base += kLoraSortThreads, turn ^= 1) {
    const int i = base + tid;
    int n = 0;
    if (i < adapters)
      for (int w = 0; w < kWarps; ++w) {
        const int c = s_count[w * adapters + i];
        s_count[w * adapters + i] = (uint16_t)n;
        n += c;
      }
    const int tiles = (n + kLoraTile - 1) / kLoraTile, both = n | tiles << 16;  // (sums of at most 8192 each)
    int scan = both;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int v = __shfl_up_sync(0xFFFFFFFFu, scan, o);
      if (lane >= o) scan += v;
    }
    if (lane == 31) s_scan[turn][warp] = scan;
    __syncthreads();  // (the other half is written next, and this one only behind the next barrier)
    int before = tokens_before | tiles_before << 16, all = before;
    for (int w = 0; w < kWarps; ++w) {
      if (w < warp) before += s_scan[turn][w];
      all += s_scan[turn][w];
    }
    before += scan - both;
    tokens_before = all & 0xFFFF;
    tiles_before = all >> 16;
    if (i < adapters) s_first[i] = (uint16_t)(before & 0xFFFF);
    for (int j = 0; j < tiles; ++j) p.tiles[(before >> 16) + j] = {i, (before & 0xFFFF) + j * kLoraTile, min(n - j * kLoraTile, kLoraTile), 0};
  }
  if (tid == 0) *p.tiles_used = tiles_before;
  __syncthreads();
  for (int base = begin; base < end; base += 32) {
    const int t = base + lane, i = t < end ? lora_adapter(a, t) : -1;
    const uint32_t same = __match_any_sync(0xFFFFFFFFu, i);
    if (i >= 0) {
      const int at = mine[i];
      p.sorted[s_first[i] + at + __popc(same & ((1u << lane) - 1u))] = t;
    }
    __syncwarp();
    if (i >= 0 && lane == __ffs(same) - 1) mine[i] += (uint16_t)__popc(same);
    __syncwarp();
  }
}

// The plan as a CTA finds it: made by the kernel in front, or, for up to 32 tokens, here, by one warp (a launch takes longer).
struct LoraHere {
  int tiles, adapter[kLoraTile];
  uint32_t tokens[kLoraTile];  // a bit per token
};
__device__ __forceinline__ int lora_tiles(const b200q_lora_args& a, const LoraPlan& p, LoraHere& here) {
  if (p.tiles_used) return *p.tiles_used;
  if (threadIdx.x < 32) {
    const int lane = threadIdx.x, i = lane < a.tokens ? lora_adapter(a, lane) : -1;
    const uint32_t same = __match_any_sync(0xFFFFFFFFu, i);
    const bool first = i >= 0 && lane == __ffs(same) - 1;
    const uint32_t all = __ballot_sync(0xFFFFFFFFu, first);
    if (first) {
      const int tile = __popc(all & ((1u << lane) - 1u));
      here.adapter[tile] = i;
      here.tokens[tile] = same;
    }
    if (lane == 0) here.tiles = __popc(all);
  }
  __syncthreads();
  return here.tiles;
}
// the tile's adapter, number of tokens, and tokens (the last one again behind it); the block's threads together, between two barriers
__device__ __forceinline__ LoraTile lora_tile(const LoraPlan& p, const LoraHere& here, int index, int (&s_token)[kLoraTile]) {
  LoraTile tile;
  const int tid = threadIdx.x;
  if (p.tiles_used) {
    tile = p.tiles[index];
    if (tid < kLoraTile) s_token[tid] = p.sorted[tile.first + min(tid, tile.count - 1)];
  } else {
    const uint32_t mask = here.tokens[index];
    tile = {here.adapter[index], 0, __popc(mask), 0};
    if (tid < kLoraTile) {
      const int last = 31 - __clz((int)mask);
      if (mask >> tid & 1u) s_token[__popc(mask & ((1u << tid) - 1u))] = tid;
      if (tid >= tile.count) s_token[tid] = last;
    }
  }
  return tile;
}

// a x of a tile's tokens over a part of k: ranks are the rows of the product, tokens its columns.  Each warp has every eighth 64 bytes of the rows of both, so
// that nothing is loaded twice; the warps' sums are added in shared memory.
template <int MT>  // tiles of 16 ranks
__global__ void __launch_bounds__(kLoraThreads) lora_down_kernel(const b200q_lora_args a, const LoraPlan p) {
  constexpr int kWarps = kLoraThreads / 32, kRanks = 16 * MT, kPitch = kRanks + 4, NT = kLoraTile / 8;
  constexpr int kBatch = MT <= 2 ? 4 : MT == 4 ? 2 : 1;  // steps of 32 values of k on their way together
  extern __shared__ float s_sum[];                       // [warps][tokens][kPitch]
  __shared__ int s_token[kLoraTile];
  __shared__ LoraHere s_here;
  pdl_enter();
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t = lane & 3;
  const int blocks = ((int)a.rank + kRanks - 1) / kRanks, items = lora_tiles(a, p, s_here) * p.splits * blocks;
  for (int item = blockIdx.x; item < items; item += gridDim.x) {
    const int block = item % blocks, part = item / blocks % p.splits;
    __syncthreads();  // (the item before this one is done with shared memory)
    const LoraTile tile = lora_tile(p, s_here, item / blocks / p.splits, s_token);
    __syncthreads();
    const __nv_bfloat16* x[NT];
    const __nv_bfloat16* rows = static_cast<const __nv_bfloat16*>(a.a) + tile.adapter * a.a_stride + (int64_t)(block * kRanks + g) * a.a_row_stride + 8 * t;
#pragma unroll
    for (int n = 0; n < NT; ++n) x[n] = static_cast<const __nv_bfloat16*>(a.x) + s_token[8 * n + g] * a.x_stride + 8 * t;
    const int ranks = (int)a.rank - block * kRanks - g, nt = (tile.count + 7) / 8;  // (of this lane's first row on)
    float acc[MT][NT][4];
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int i = 0; i < 4; ++i) acc[m][n][i] = 0.f;
    const int64_t end = min((int64_t)(part + 1) * p.slice, a.k);
    const uint4 zero = make_uint4(0, 0, 0, 0);
    for (int64_t k0 = (int64_t)part * p.slice + 32 * warp; k0 < end; k0 += 32 * kWarps * kBatch) {
      uint4 ra[kBatch][MT][2], rx[kBatch][NT];
#pragma unroll
      for (int b = 0; b < kBatch; ++b) {
        const int64_t k = k0 + 32 * kWarps * b;
        const bool in = k + 8 * t < end;
#pragma unroll
        for (int m = 0; m < MT; ++m)
#pragma unroll
          for (int h = 0; h < 2; ++h) ra[b][m][h] = in && 16 * m + 8 * h < ranks ? __ldg(reinterpret_cast<const uint4*>(rows + (16 * m + 8 * h) * a.a_row_stride + k)) : zero;
#pragma unroll
        for (int n = 0; n < NT; ++n) rx[b][n] = in && n < nt ? __ldg(reinterpret_cast<const uint4*>(x[n] + k)) : zero;
      }
#pragma unroll
      for (int b = 0; b < kBatch; ++b)
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          if (n >= nt) break;
#pragma unroll
          for (int m = 0; m < MT; ++m) {
            lora_mma(acc[m][n], ra[b][m][0].x, ra[b][m][1].x, ra[b][m][0].y, ra[b][m][1].y, rx[b][n].x, rx[b][n].y);
            lora_mma(acc[m][n], ra[b][m][0].z, ra[b][m][1].z, ra[b][m][0].w, ra[b][m][1].w, rx[b][n].z, rx[b][n].w);
          }
        }
    }
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      if (n >= nt) break;
#pragma unroll
      for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int i = 0; i < 4; ++i) s_sum[(warp * kLoraTile + 8 * n + 2 * t + (i & 1)) * kPitch + 16 * m + g + 8 * (i >> 1)] = acc[m][n][i];
    }
    __syncthreads();
    for (int i = tid; i < tile.count * kRanks; i += kLoraThreads) {
      const int j = i / kRanks, r = i % kRanks;
      if (block * kRanks + r >= a.rank) continue;
      float sum = 0.f;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) sum += s_sum[(w * kLoraTile + j) * kPitch + r];
      p.low[((int64_t)part * a.tokens + s_token[j]) * a.rank + block * kRanks + r] = sum;
    }
  }
}

// y += b (scale a x): tokens are the rows of the product, 32 values of y of a warp its columns, of which a lane has 8 neighbours in four rows.  The values of y for
// the next step are on their way while this one's products are formed.
template <typename Y, bool WIDE>  // WIDE: ranks 32 at a time, in 16 bytes a lane; else 16 at a time
__global__ void __launch_bounds__(kLoraThreads, 2) lora_up_kernel(const b200q_lora_args a, const LoraPlan p, int parts, int width) {
  constexpr int kTerms = sizeof(Y) == 4 ? 3 : 2, kWarps = kLoraThreads / 32, kStep = WIDE ? 32 : 16, kHalves = WIDE ? 2 : 1;
  constexpr int kY = sizeof(Y) == 4 ? 2 : 1, kPer = 16 / sizeof(Y);  // 16-byte pieces of a lane's 8 values; values of a piece
  extern __shared__ __align__(16) uint8_t s_raw[];                   // [terms][tokens][pitch] of bf16
  __shared__ int s_token[kLoraTile];
  __shared__ LoraHere s_here;
  pdl_enter();
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t = lane & 3;
  const int rank = (int)a.rank, steps = (rank + kStep - 1) / kStep, pitch = steps * kStep + 8, items = lora_tiles(a, p, s_here) * parts;
  __nv_bfloat16* const s_low = reinterpret_cast<__nv_bfloat16*>(s_raw);
  for (int item = blockIdx.x; item < items; item += gridDim.x) {
    const int part = item % parts;
    __syncthreads();
    const LoraTile tile = lora_tile(p, s_here, item / parts, s_token);
    const float scale = a.scales ? a.scales[tile.adapter] : 1.f;
    __syncthreads();
    const int n_end = (int)min((int64_t)(part + 1) * width, a.n);
    int n0 = part * width + 32 * warp;
    Y* rows[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) rows[i] = static_cast<Y*>(a.y) + s_token[g + 8 * i] * a.y_stride + 8 * t;
    uint4 next[4][kY];
    auto ask = [&](int n) {
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int c = 0; c < kY; ++c)
          if (g + 8 * i < tile.count && n < n_end && n + 8 * t + c * kPer < a.n) next[i][c] = *reinterpret_cast<const uint4*>(rows[i] + n + c * kPer);
    };
    ask(n0);
    for (int i = tid; i < kLoraTile * steps * kStep; i += kLoraThreads) {
      const int j = i / (steps * kStep), r = i - j * (steps * kStep);
      float v = 0.f;
      if (j < tile.count && r < rank) {
        for (int s = 0; s < p.splits; ++s) v += __ldcg(p.low + ((int64_t)s * a.tokens + s_token[j]) * rank + r);
        v *= scale;
      }
#pragma unroll
      for (int c = 0; c < kTerms; ++c) {
        const __nv_bfloat16 hi = __float2bfloat16_rn(v);
        s_low[(c * kLoraTile + j) * pitch + r] = hi;
        v -= __bfloat162float(hi);
      }
    }
    __syncthreads();
    const bool two = tile.count > 16;
    // column g of product c is y's n0 + 8 (g / 2) + 2 c + g % 2
    const int column = 8 * (g >> 1) + (g & 1);
    const __nv_bfloat16* const b0 = static_cast<const __nv_bfloat16*>(a.b) + tile.adapter * a.b_stride + column * a.b_row_stride + (WIDE ? 8 : 4) * t;
    for (; n0 < n_end; n0 += 32 * kWarps) {
      uint4 now[4][kY];
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int c = 0; c < kY; ++c) now[i][c] = next[i][c];
      ask(n0 + 32 * kWarps);
      float acc[2][4][4];
#pragma unroll
      for (int m = 0; m < 2; ++m)
#pragma unroll
        for (int c = 0; c < 4; ++c)
#pragma unroll
          for (int i = 0; i < 4; ++i) acc[m][c][i] = 0.f;
      const __nv_bfloat16* b = b0 + n0 * a.b_row_stride;
      for (int k = 0; k < steps; ++k) {
        uint32_t rb[4][2 * kHalves];
        const bool in = k * kStep + (WIDE ? 8 : 4) * t < rank;
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          const bool there = in && n0 + column + 2 * c < a.n;
          if constexpr (WIDE) {
            const uint4 v = there ? __ldg(reinterpret_cast<const uint4*>(b + 2 * c * a.b_row_stride + k * kStep)) : make_uint4(0, 0, 0, 0);
            rb[c][0] = v.x; rb[c][1] = v.y; rb[c][2] = v.z; rb[c][3] = v.w;
          } else {
            const uint2 v = there ? __ldg(reinterpret_cast<const uint2*>(b + 2 * c * a.b_row_stride + k * kStep)) : make_uint2(0, 0);
            rb[c][0] = v.x; rb[c][1] = v.y;
          }
        }
#pragma unroll
        for (int m = 0; m < 2; ++m) {
          if (m == 1 && !two) break;
#pragma unroll
          for (int e = 0; e < kTerms; ++e) {
            const __nv_bfloat16* low = s_low + (e * kLoraTile + 16 * m + g) * pitch + k * kStep + (WIDE ? 8 : 4) * t;
            uint32_t lo[2 * kHalves], hi[2 * kHalves];
            if constexpr (WIDE) {
              const uint4 u = *reinterpret_cast<const uint4*>(low), v = *reinterpret_cast<const uint4*>(low + 8 * pitch);
              lo[0] = u.x; lo[1] = u.y; lo[2] = u.z; lo[3] = u.w;
              hi[0] = v.x; hi[1] = v.y; hi[2] = v.z; hi[3] = v.w;
            } else {
              const uint2 u = *reinterpret_cast<const uint2*>(low), v = *reinterpret_cast<const uint2*>(low + 8 * pitch);
              lo[0] = u.x; lo[1] = u.y;
              hi[0] = v.x; hi[1] = v.y;
            }
#pragma unroll
            for (int h = 0; h < kHalves; ++h)
#pragma unroll
              for (int c = 0; c < 4; ++c) lora_mma(acc[m][c], lo[2 * h], hi[2 * h], lo[2 * h + 1], hi[2 * h + 1], rb[c][2 * h], rb[c][2 * h + 1]);
          }
        }
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if (g + 8 * i >= tile.count) continue;
#pragma unroll
        for (int c = 0; c < kY; ++c) {
          if (n0 + 8 * t + c * kPer >= a.n) continue;
          // the lane's values 2 q and 2 q + 1 are in product q
          Y* y = rows[i] + n0 + c * kPer;
          if constexpr (sizeof(Y) == 4) {
            const float* v0 = acc[i >> 1][2 * c] + 2 * (i & 1);
            const float* v1 = acc[i >> 1][2 * c + 1] + 2 * (i & 1);
            *reinterpret_cast<float4*>(y) = make_float4(__uint_as_float(now[i][c].x) + v0[0], __uint_as_float(now[i][c].y) + v0[1],
                                                        __uint_as_float(now[i][c].z) + v1[0], __uint_as_float(now[i][c].w) + v1[1]);
          } else {
            const uint32_t u[4] = {now[i][c].x, now[i][c].y, now[i][c].z, now[i][c].w};
            uint32_t w[4];
#pragma unroll
            for (int q = 0; q < 4; ++q) {
              const float* v = acc[i >> 1][q] + 2 * (i & 1);
              w[q] = pack_bf16x2(__uint_as_float(u[q] << 16) + v[0], __uint_as_float(u[q] & 0xFFFF0000u) + v[1]);
            }
            *reinterpret_cast<uint4*>(y) = make_uint4(w[0], w[1], w[2], w[3]);
          }
        }
      }
    }
  }
}

// ---------------------------------------------------------------------------- host
size_t lora_workspace_bytes_impl(int64_t tokens, int64_t k, int64_t n, int64_t rank, int64_t adapters) {
  (void)n;
  return LoraSpace(tokens, rank, lora_splits(tokens, k, adapters)).bytes;
}

static bool lora_fits_tensor_cores(const b200q_lora_args& a) {
  if (a.force_plain || a.rank % 8 || a.k % 8 || a.n % 8) return false;
  const bool many = a.tokens > 1;
  if (many && (a.x_stride % 8 || a.y_stride % 8)) return false;
  if (a.adapters > 1 && (a.a_stride % 8 || a.b_stride % 8)) return false;
  if ((a.rank > 1 && a.a_row_stride % 8) || (a.n > 1 && a.b_row_stride % 8)) return false;
  for (const void* p : {a.x, static_cast<const void*>(a.y), a.a, a.b})
    if (reinterpret_cast<uintptr_t>(p) % 16) return false;
  return true;
}

static int lora_ready(const void* kernel, std::atomic<int> (&done)[kMaxDevices], int smem) {
  const int dev = current_device_index();
  if (dev < 0) return B200Q_ERR_CUDA;
  if (!done[dev].load(std::memory_order_acquire)) {
    B200Q_CUDA_OK(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
    done[dev].store(1, std::memory_order_release);
  }
  return B200Q_OK;
}

template <int MT>
static int lora_launch_down(const b200q_lora_args& a, const LoraPlan& p, int64_t tiles, cudaStream_t st) {
  constexpr int kSmem = (int)sizeof(float) * (kLoraThreads / 32) * kLoraTile * (16 * MT + 4);
  static std::atomic<int> done[kMaxDevices];
  if (int rc = lora_ready(reinterpret_cast<const void*>(lora_down_kernel<MT>), done, kSmem)) return rc;
  const int64_t items = tiles * p.splits * ((a.rank + 16 * MT - 1) / (16 * MT)), most = 4 * kNumSMs;
  launch_dependent(lora_down_kernel<MT>, dim3((unsigned)(items < most ? items : most)), dim3(kLoraThreads), kSmem, st, a, p);
  B200Q_LAUNCH_CHECK();
  return B200Q_OK;
}
template <typename Y, bool WIDE>
static int lora_launch_up(const b200q_lora_args& a, const LoraPlan& p, int64_t tiles, cudaStream_t st) {
  constexpr int kTerms = sizeof(Y) == 4 ? 3 : 2, kStep = WIDE ? 32 : 16;
  constexpr int kMost = 2 * kTerms * kLoraTile * ((int)kLoraMaxRank + 8);
  static std::atomic<int> done[kMaxDevices];
  if (int rc = lora_ready(reinterpret_cast<const void*>(lora_up_kernel<Y, WIDE>), done, kMost)) return rc;
  const int64_t most_parts = (a.n + 255) / 256, wanted = (4 * kNumSMs + tiles - 1) / tiles, parts = wanted < most_parts ? wanted : most_parts;
  const int64_t width = ((a.n + parts - 1) / parts + 255) / 256 * 256, used = (a.n + width - 1) / width;
  const int64_t items = tiles * used, most = 4 * kNumSMs;
  const size_t smem = (size_t)(2 * kTerms * kLoraTile) * ((a.rank + kStep - 1) / kStep * kStep + 8);
  launch_dependent(lora_up_kernel<Y, WIDE>, dim3((unsigned)(items < most ? items : most)), dim3(kLoraThreads), smem, st, a, p, (int)used, (int)width);
  B200Q_LAUNCH_CHECK();
  return B200Q_OK;
}

static int lora_chunk_fast(const b200q_lora_args& a, cudaStream_t st) {
  const int64_t splits = lora_splits(a.tokens, a.k, a.adapters), tiles = lora_most_tiles(a.tokens, a.adapters);
  const LoraSpace space(a.tokens, a.rank, splits);
  uint8_t* w = static_cast<uint8_t*>(a.workspace);
  LoraPlan p;
  p.tiles_used = reinterpret_cast<int*>(w);
  p.tiles = reinterpret_cast<LoraTile*>(w + space.tiles);
  p.sorted = reinterpret_cast<int*>(w + space.sorted);
  p.low = reinterpret_cast<float*>(w + space.low);
  p.splits = (int)splits;
  p.slice = (int)(((a.k + splits - 1) / splits + 255) / 256 * 256);
  static std::atomic<int> done[kMaxDevices];
  constexpr int kMost = (int)sizeof(uint16_t) * (kLoraSortThreads / 32 + 1) * (int)kLoraMaxAdapters;
  if (int rc = lora_ready(reinterpret_cast<const void*>(lora_sort_kernel), done, kMost)) return rc;
  if (a.tokens <= kLoraTile) {
    p.tiles_used = nullptr;  // (each CTA makes the plan for itself)
  } else {
    launch_dependent(lora_sort_kernel, dim3(1), dim3(kLoraSortThreads), sizeof(uint16_t) * (kLoraSortThreads / 32 + 1) * (size_t)a.adapters, st, a, p);
    B200Q_LAUNCH_CHECK();
  }
  int rc;
  if (a.rank <= 16) rc = lora_launch_down<1>(a, p, tiles, st);
  else if (a.rank <= 32) rc = lora_launch_down<2>(a, p, tiles, st);
  else if (a.rank <= 64) rc = lora_launch_down<4>(a, p, tiles, st);
  else rc = lora_launch_down<8>(a, p, tiles, st);
  if (rc) return rc;
  if (a.y_dtype == B200Q_F32) return a.rank % 32 ? lora_launch_up<float, false>(a, p, tiles, st) : lora_launch_up<float, true>(a, p, tiles, st);
  return a.rank % 32 ? lora_launch_up<__nv_bfloat16, false>(a, p, tiles, st) : lora_launch_up<__nv_bfloat16, true>(a, p, tiles, st);
}

static int lora_chunk_plain(const b200q_lora_args& a, cudaStream_t st) {
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
    if (int rc = lora_fits_tensor_cores(a) ? lora_chunk_fast(c, st) : lora_chunk_plain(c, st)) return rc;
  }
  return B200Q_OK;
}

}  // namespace b200q
