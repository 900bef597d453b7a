// Attention of one new token per request over a key/value cache in pages:
//   s_j = softmax_scale * k_scale_inv * <q, k_j>,  j in [max(0, len - window), len);   p = softmax(s)
//   out = v_scale_inv * sum_j p_j v_j,   lse = log sum_j exp(s_j);   nothing to see: out = 0, lse = -inf.
#include "paged.cuh"
#include "tcgen05_ptx.cuh"
#include "tma_host.cuh"

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
__device__ __forceinline__ int paged_length(const b200q_paged_attention_args& a, int64_t b) {
  const int64_t most = a.table_width * a.page_size;
  return (int)min((int64_t)max(a.kv_lens[b], 0), most);
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

// ---------------------------------------------------------------------------- tensor cores
// Memory bound: every cached key and value is used once for the 8 or 16 query heads that share it.  What the kernel does
// beside reading must stay under the reads: 16 flops a byte and head group are beyond the CUDA cores' rate in fp32, so both
// products are m16n8k16 matrix instructions with the CACHE as the operand of 16 rows (keys of K, dimensions of V) and the heads as
// the 8 columns, which fills the instruction when eight heads share a key/value head.
//
// A warp works on steps of 16 keys.  It has a ring of its own in shared memory that TMA fills, a box of 16 keys and 128 bytes
// at a time (cp.async of the same bytes, 16 at a time, ends at 4.4 TB/s), and nothing to wait for but its own copies.
// Lane (g = lane / 4, t = lane % 4) reads the operands' fragments as they lie:
//   of K: keys R(g) and R(g) + 8, bytes 64 c + 16 t ... + 15 of their rows   (the dimensions of a dot product may come in any
//         order: the queries are laid out to match; so may the keys, as long as V follows)
//   of V: the keys of rows 2t, 2t + 1, 2t + 8, 2t + 9, that is t, t + 4, t + 8, t + 12, bytes (8 c + R(g)) * 16 ... + 15  (the
//         dimensions are the rows of the second product, which may come in any order too)
// R(0 ... 7) = 0, 4, 1, 5, 2, 6, 3, 7: with it the eight lanes of a 16-byte access lie in different banks of the swizzled tile.  (Where a row
// is 64 bytes the pieces of V are 8 bytes, and a lane's the g-th.)
// fp8 values become f16 exactly.  The probabilities of an fp8 cache are f16 too, scaled by 2^7 so that the small ones stay normal: one term
// (11 bits) where the output is bf16 or e4m3, whose own rounding is 8 bits or fewer, and two terms (22 bits) that take a product each
// where it is fp32.  Two terms everywhere would be 124 -> 131 us for 64 requests of 2048 to 8192 tokens (8 key/value heads of 128), and a branch
// in the loop would cost all outputs 5 %; that case's bf16 output is 1.5e-3 from 64-bit arithmetic with one term, with two and with 24 bits.  For a bf16 cache
// they are two bf16 terms (16 bits), twice as fine as any bf16 output.  Queries meet fp8 keys as f16, scaled
// by a power of two per head, which is exact over 2^22 of a head's largest value.
//
// Work is the list of all steps (request-major, then key/value head, then the length), cut into equal runs for the CTAs, so that
// ragged lengths and few requests load every SM alike.  In a CTA `lanes` warps take neighbouring heads of the same keys -- the
// whole row of a token is read at one time, which is worth 5.0 -> 6.2 TB/s where the heads of a token lie together -- and the
// kWarps / lanes groups of such warps cut the run again.  A run may begin or end inside a row of steps: such partial results
// (maximum, sum, output) are joined in the CTA, and, where a row goes on in another CTA, by a second kernel.
//
// Measured (from a CUDA graph, shuffled pages): 64 requests of 8192 tokens, 8 key/value heads of 128 in e4m3, 175 us = 6.1 TB/s (fp32 output 180); the same in
// bf16, 32 requests, 165 us = 6.5 TB/s.  About 9 us of a call do not depend on the length: 3 of dependent loads (lengths, page numbers, first keys),
// joining (a kernel of 5 to 11 us by itself, in part behind this one's end), and the launches.
constexpr int kPagedGrid = kNumSMs;
constexpr int kPagedRingBytes = 192 * 1024;
constexpr int kPagedLaneSteps = 14;   // a warp's steps from which on heads go side by side
constexpr int kPagedMinSteps = 2;     // a warp gets at least this many steps while there are enough for the others
constexpr float kPagedNoMax = -3.402823466e38f;  // the lowest finite number: no finite score is below it
constexpr int kPagedLengthsHere = (int)kPagedMaxRequests / 2;  // up to so many requests' lengths lie in shared memory beside the sums
constexpr int kPagedErrCopy = 801;  // status code: a copy of keys and values did not arrive

constexpr int paged_warps_of(int dim) { return dim == 256 ? 4 : 8; }  // of a CTA

template <int DIM, int FMT, int NT>
struct PagedTile {
  static constexpr int kElt = FMT == B200Q_BF16 ? 2 : 1;
  static constexpr int kRow = DIM * kElt;           // bytes of a key
  static constexpr int kStage = 2 * 16 * kRow;      // keys and values of a step
  static constexpr int kWarps = paged_warps_of(DIM);
  static constexpr int kStages = kPagedRingBytes / kWarps / kStage < 8 ? kPagedRingBytes / kWarps / kStage : 8;
  static constexpr int kKChunks = kRow / 64;        // 16-byte pieces of a key per lane
  static constexpr int kVPiece = kRow / 8 < 16 ? 8 : 16;
  static constexpr int kVChunks = kRow / 8 / kVPiece;
  static constexpr int kVPer = kVPiece / kElt;      // values of a piece
  static constexpr int kBox = kRow < 128 ? kRow : 128;  // bytes of a key in one copy
  static constexpr int kBoxes = kRow / kBox;
  static constexpr int kTiles = DIM / 16;           // k-steps of the first product, row tiles of the second
  static constexpr int kRows = 8 * NT;              // query heads
  // Probabilities are held relative to 2^(maximum - kShift), and the maximum is raised when one would pass 2^kRescale.  f16 ends at 2^16, and
  // below 2^-14 it loses bits: 2^7 and 2^15.  bf16 has the range of fp32, and so have the values that it meets, whose products with
  // probabilities of at most 1 do not overflow: 2^-8 and 1.
  static constexpr float kShift = FMT == B200Q_BF16 ? -8.f : 7.f, kRescale = FMT == B200Q_BF16 ? 0.f : 15.f;
  static constexpr int kPart = kRows * (DIM + 2);   // floats of a partial result: output, maxima, sums
  static constexpr int kRing = kStages * kStage;    // bytes per warp
  static_assert(2 * kPart * 4 <= kRing && kStages >= 2, "both partial results of a warp take the place of the ring");
};

// The row (of `lanes` neighbouring heads, `sub` the index of their group) that is first cut by the first step of a CTA: it begins in the CTA
// before and goes on in `count` CTAs from here.
struct alignas(16) PagedJoin {
  int lanes, request, sub, count;  // lanes: 0 where no row is first cut here
};

struct PagedWork {
  int heads_per_request;  // key/value heads x row tiles
  int row_tiles;
  int group;              // query heads per key/value head
  int lane_bits;          // log2 of the largest power of two, at most the warps of a CTA, that divides heads_per_request
  PagedJoin* joins;       // [grid]
  float* cta_part;        // [grid][2][warps][kPart]: rows from the CTA before, rows into the CTA behind, of each lane
  float* warp_part;       // [grid][warps][kPart]: rows from the warp before that end inside a warp's run
  int* status;
  int drop_cta, drop_warp, drop_step;  // self-test: the step of the warp's run whose copies are never made
};

__device__ __forceinline__ uint32_t paged_smem(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }
// a box of a cache: `kBox` bytes from x on of 16 tokens' head
__device__ __forceinline__ void paged_copy(uint32_t dst, const CUtensorMap* map, uint32_t bar, int x, int head, int slot, int page) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5, %6}], [%2];"
      ::"r"(dst), "l"(reinterpret_cast<uint64_t>(map)), "r"(bar), "r"(x), "r"(head), "r"(slot), "r"(page)
      : "memory");
}
__device__ __forceinline__ uint4 paged_lds16(uint32_t at) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(at) : "memory");
  return v;
}
__device__ __forceinline__ uint2 paged_lds8(uint32_t at) {
  uint2 v;
  asm volatile("ld.shared.v2.u32 {%0, %1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(at) : "memory");
  return v;
}
__device__ __forceinline__ float paged_exp2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
template <int FMT>
__device__ __forceinline__ void paged_mma(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  if (FMT == B200Q_BF16)
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  else
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// rows of 8 x 8 16-bit values held as fragments become columns
__device__ __forceinline__ uint32_t paged_transpose(uint32_t v) {
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}
// four fp8 values -> (0, 1) and (2, 3) as f16 pairs, exactly
template <int FMT>
__device__ __forceinline__ void paged_f16(uint32_t w, uint32_t& lo, uint32_t& hi) {
  if (FMT == B200Q_E4M3) {
    asm("{\n.reg .b16 a, b;\nmov.b32 {a, b}, %2;\ncvt.rn.f16x2.e4m3x2 %0, a;\ncvt.rn.f16x2.e4m3x2 %1, b;\n}" : "=r"(lo), "=r"(hi) : "r"(w));
  } else {  // (an e5m2 value is the upper byte of the f16 one)
    lo = __byte_perm(w, 0u, 0x1404);
    hi = __byte_perm(w, 0u, 0x3424);
  }
}
__device__ __forceinline__ uint32_t paged_pack_f16(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}
__device__ __forceinline__ float2 paged_unpack_f16(uint32_t v) {
  float2 r;
  asm("{\n.reg .b16 a, b;\nmov.b32 {a, b}, %2;\ncvt.f32.f16 %0, a;\ncvt.f32.f16 %1, b;\n}" : "=f"(r.x), "=f"(r.y) : "r"(v));
  return r;
}
__device__ __forceinline__ void paged_store4(void* out, int dtype, int64_t at, const float (&v)[4]) {
  if (dtype == B200Q_BF16)
    *reinterpret_cast<uint2*>(static_cast<__nv_bfloat16*>(out) + at) = make_uint2(pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]));
  else if (dtype == B200Q_F32) *reinterpret_cast<float4*>(static_cast<float*>(out) + at) = make_float4(v[0], v[1], v[2], v[3]);
  else *reinterpret_cast<uint32_t*>(static_cast<uint8_t*>(out) + at) = cvt_fp8x2<B200Q_E4M3>(v[0], v[1]) | (cvt_fp8x2<B200Q_E4M3>(v[2], v[3]) << 16);
}
__device__ __forceinline__ float paged_lse(float m, float l) { return l == 0.f ? -INFINITY : (m + log2f(l)) * 0.693147180559945309f; }
__device__ __forceinline__ float paged_out_scale(const b200q_paged_attention_args& a) {
  return (a.v_scale_inv ? *a.v_scale_inv : 1.f) * (a.out_scale ? *a.out_scale : 1.f);
}

// the keys that a request's token sees: [first, len); its steps begin at a multiple of 16
struct PagedSpan {
  int len, first;
  __device__ __forceinline__ PagedSpan(const b200q_paged_attention_args& a, int length) {
    len = length;
    first = a.window > 0 && len > a.window ? len - (int)a.window : 0;
  }
  __device__ __forceinline__ int steps() const { return (int)(((uint32_t)len + 15u) / 16u) - first / 16; }
};

// A place in the list of steps (of fewer than 2^31).
struct PagedCursor {
  int b, sub, step, steps;
  // the place of step `at`; prefix: inclusive sums of the requests' steps
  __device__ __forceinline__ void locate(const int* prefix, int requests, int heads, int at) {
    int lo = 0, hi = requests - 1;
    while (lo < hi) {
      const int mid = (lo + hi) >> 1;
      if (prefix[mid] * heads > at) hi = mid;
      else lo = mid + 1;
    }
    b = lo;
    const int before = b ? prefix[b - 1] : 0;
    steps = prefix[b] - before;
    const uint32_t r = (uint32_t)(at - before * heads);
    sub = (int)(r / (uint32_t)steps);
    step = (int)r - sub * steps;
  }
  // to the first step of the next row; there is one
  __device__ __forceinline__ bool next_row(const int* prefix, int requests, int heads) {
    step = 0;
    if (++sub < heads) return true;
    sub = 0;
    do {
      if (++b >= requests) return false;
      steps = prefix[b] - prefix[b - 1];
    } while (steps == 0);
    return true;
  }
};

// The list in equal runs: the first `more` of `ctas` have a step more than the others.
struct PagedRuns {
  int ctas, each, more;
  __device__ __forceinline__ PagedRuns(int total, int ctas_) {
    ctas = ctas_;
    each = (int)((uint32_t)total / (uint32_t)ctas);
    more = total - each * ctas;
  }
  __device__ __forceinline__ int begin(int c) const { return c * each + min(c, more); }
  __device__ __forceinline__ int cta_of(int at) const {  // (each > 0)
    const int longer = more * (each + 1);
    return at < longer ? (int)((uint32_t)at / (uint32_t)(each + 1)) : more + (int)((uint32_t)(at - longer) / (uint32_t)each);
  }
};

// One of a warp's partial results, in the order in which rows are written out: [kRows][DIM], then maxima, then sums.
template <int DIM, int FMT, int NT>
struct PagedAcc {
  using Tile = PagedTile<DIM, FMT, NT>;
  float o[Tile::kTiles][NT][4];  // dimensions x heads: fragment j holds the lane's values 2j (0, 1) and 2j + 1 (2, 3) for heads 2t, 2t + 1
  float m[NT][2], l[NT][2];

  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int n = 0; n < NT; ++n) {
#pragma unroll
      for (int j = 0; j < Tile::kTiles; ++j)
#pragma unroll
        for (int i = 0; i < 4; ++i) o[j][n][i] = 0.f;
      m[n][0] = m[n][1] = kPagedNoMax;
      l[n][0] = l[n][1] = 0.f;
    }
  }
  // every lane has the whole sums
  __device__ __forceinline__ void sum_lanes() {
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int s = 4; s < 32; s <<= 1) l[n][i] += __shfl_xor_sync(0xFFFFFFFFu, l[n][i], s);
  }
  // calls f(head row, first dimension, four values) for all that the lane holds
  template <typename F>
  __device__ __forceinline__ void each4(int piece, int t, F f) const {
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int e = 0; e < Tile::kVChunks * Tile::kVPer; e += 4) {
          const float v[4] = {o[e / 2][n][i], o[e / 2][n][i + 2], o[e / 2 + 1][n][i], o[e / 2 + 1][n][i + 2]};
          f(8 * n + 2 * t + i, (e / Tile::kVPer * 8 + piece) * Tile::kVPer + e % Tile::kVPer, v, n, i);
        }
  }
  __device__ __forceinline__ void save(float* to, int g, int piece, int t) const {
    each4(piece, t, [&](int row, int d, const float (&v)[4], int, int) {
      *reinterpret_cast<float4*>(to + row * DIM + d) = make_float4(v[0], v[1], v[2], v[3]);
    });
    if (g == 0) {
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const int row = 8 * n + 2 * t + i;
          to[Tile::kRows * DIM + row] = m[n][i];
          to[Tile::kRows * DIM + Tile::kRows + row] = l[n][i];
        }
    }
  }
};

// Joins one head's results from `count` places (at(i): a partial result): the values of dimensions lane, lane + 32, ...  Eight places at a
// time, all their loads in flight together (a trip to L2 is what a join costs).
template <int DIM, int ROWS, typename At>
__device__ __forceinline__ void paged_merge(At at, int count, int row, int lane, float (&o)[DIM / 32], float& m, float& l) {
  constexpr int kBatch = 8;
  m = kPagedNoMax;
  l = 0.f;
#pragma unroll
  for (int d = 0; d < DIM / 32; ++d) o[d] = 0.f;
  for (int base = 0; base < count; base += kBatch) {
    float pm[kBatch], pl[kBatch], x[kBatch][DIM / 32];
#pragma unroll
    for (int i = 0; i < kBatch; ++i) {
      const float* p = at(min(base + i, count - 1));  // (written by other CTAs: read past L1)
      pm[i] = __ldcg(p + ROWS * DIM + row);
      pl[i] = __ldcg(p + ROWS * DIM + ROWS + row);
#pragma unroll
      for (int d = 0; d < DIM / 32; ++d) x[i][d] = __ldcg(p + row * DIM + d * 32 + lane);
    }
    float top = m;
#pragma unroll
    for (int i = 0; i < kBatch; ++i) top = fmaxf(top, pm[i]);
    const float keep = exp2f(m - top);  // (inf - inf: a NaN row, as its parts are)
    m = top;
    l *= keep;
#pragma unroll
    for (int d = 0; d < DIM / 32; ++d) o[d] *= keep;
#pragma unroll
    for (int i = 0; i < kBatch; ++i) {
      if (base + i >= count) break;
      const float weight = exp2f(pm[i] - top);
      l += weight * pl[i];
#pragma unroll
      for (int d = 0; d < DIM / 32; ++d) o[d] += weight * x[i][d];
    }
  }
}
template <int DIM>
__device__ __forceinline__ void paged_finish(const b200q_paged_attention_args& a, int b, int head, int lane, const float (&o)[DIM / 32], float m, float l,
                                             float scale) {
  const int64_t at = ((int64_t)b * a.heads + head) * DIM;
  const float inv = l == 0.f ? 0.f : scale / l;
#pragma unroll
  for (int d = 0; d < DIM / 32; ++d) paged_store(a.out, a.out_dtype, at + d * 32 + lane, o[d] * inv);
  if (lane == 0 && a.lse) a.lse[(int64_t)b * a.heads + head] = paged_lse(m, l);
}

// DROP: the instance of the self-test, in which one step's copies are never made and waits are short.
template <int DIM, int FMT, int NT, int TERMS, bool DROP = false>
__global__ void __launch_bounds__(32 * PagedTile<DIM, FMT, NT>::kWarps, 1)
    paged_attention_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v,
                           const b200q_paged_attention_args a, const PagedWork w) {
  using Tile = PagedTile<DIM, FMT, NT>;
  static_assert(TERMS == 2 || FMT != B200Q_BF16, "a bf16 term alone would be 8 bits");
  constexpr int kWarps = Tile::kWarps, kWarpBits = kWarps == 8 ? 3 : 2, kStages = Tile::kStages, kTiles = Tile::kTiles;
  static_assert(1 << kWarpBits == kWarps, "a power of two");
  extern __shared__ __align__(1024) uint8_t s_raw[];
  uint8_t* const s_ring = s_raw + (0u - paged_smem(s_raw) & 1023u);  // [warps][kRing] (swizzled tiles repeat every 1024 bytes), then the prefix sums
  __shared__ __align__(8) uint64_t s_bars[kWarps * kStages];
  __shared__ int s_abort;
  __shared__ int s_sum[2][kWarps];
  __shared__ int s_state[kWarps], s_b[kWarps], s_sub[kWarps], s_cut_b, s_cut_sub;
  int* prefix = reinterpret_cast<int*>(s_ring + kWarps * Tile::kRing);
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t = lane & 3;
  const int requests = (int)a.requests;
  const uint32_t bars = paged_smem(s_bars + warp * kStages);
  if (lane < kStages) {
    ptx::mbar_init(bars + 8 * lane, 1);
    ptx::fence_barrier_init();
  }
  if (tid == 0) {
    s_abort = 0;
    ptx::tma_prefetch_desc(&map_k);
    ptx::tma_prefetch_desc(&map_v);
  }
  pdl_enter();

  // (asked for before anything else, used much later)
  const float k_scale = a.k_scale_inv ? *a.k_scale_inv : 1.f, v_scale = a.v_scale_inv ? *a.v_scale_inv : 1.f, o_scale = a.out_scale ? *a.out_scale : 1.f;

  // ---- the list of steps
  int* const lengths = prefix + requests;  // (where there is room: the rows of the loop then need no loads that wait behind the copies)
  const bool lengths_here = requests <= kPagedLengthsHere;
  {
    int sums = 0;
    for (int base = 0, turn = 0; base < requests; base += 32 * kWarps, turn ^= 1) {
      const int b = base + tid;
      int scan = 0;
      if (b < requests) {
        const int len = paged_length(a, b);
        scan = PagedSpan(a, len).steps();
        if (lengths_here) lengths[b] = len;
      }
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int v = __shfl_up_sync(0xFFFFFFFFu, scan, o);
        if (lane >= o) scan += v;
      }
      if (lane == 31) s_sum[turn][warp] = scan;
      __syncthreads();  // (the other half of s_sum is written next, and this one only behind the next barrier)
      int before = sums;
#pragma unroll
      for (int i = 0; i < kWarps; ++i) {
        if (i < warp) before += s_sum[turn][i];
        sums += s_sum[turn][i];
      }
      if (b < requests) prefix[b] = before + scan;
    }
    __syncthreads();
  }
  auto span_of = [&](int b) { return PagedSpan(a, lengths_here ? lengths[b] : paged_length(a, b)); };
  // Heads side by side where a warp's share is long enough to pay for a partial result of its own, or where rows are so many that few of
  // them are cut (and no warps of a CTA have parts of the same one), and only where a token's head is short of 512 bytes.  us, side by
  // side / one head per CTA, 8 key/value heads of 128 in e4m3: 64 x 8192 tokens 175 / 221, 8 x 16000 56 / 62, 64 x 1000 36.1 / 40.6, 256 x 200 37.4 / 43.3,
  // 2 x 34000 36.0 / 37.9, 1 x 131072 58.1 / 62.8, 4 x 10000 25.3 / 25.6; below the limit 8 x 4000 24.8 / 23.4, 1 x 16384 20.8 / 16.9, 1 x 8192 18.3 / 15.2.
  // 4 heads, 100 of 75 to 300 26.7 / 20.3; 2 heads of 256 in bf16, 40 x 4000 64.4 / 61.8.  The total of steps does not tell all of it: 16 requests of 1024 to
  // 4096 30.0 / 26.2, 16 x 2600 28.0 / 27.1, 1 x 34000 26.5 / 23.2 and 1 x 65536 37.3 / 36.1 lie above the limit, 32 x 400 17.3 / 18.4 below.
  const int key_steps = prefix[requests - 1], warps = kWarps * (int)gridDim.x;
  const bool beside = Tile::kRow < 512 && (key_steps * w.heads_per_request >= kPagedLaneSteps * warps ||
                                           (w.lane_bits == kWarpBits && requests * w.heads_per_request >= warps / 4));
  const int shift = beside ? w.lane_bits : 0;
  const int lanes = 1 << shift, groups = kWarps >> shift, my_lane = warp & (lanes - 1), my_group = warp >> shift;
  const int heads = w.heads_per_request >> shift, total = key_steps * heads;
  // of the `sub`-th row tile of a request: its key/value head, and its first query head in that head's group
  auto kv_of = [&](int sub) { return w.row_tiles == 1 ? sub : sub / w.row_tiles; };
  auto row_of = [&](int sub) { return w.row_tiles == 1 ? 0 : sub % w.row_tiles * Tile::kRows; };
  const float out_scale = v_scale * o_scale;

  auto write_empty = [&] {  // requests that see nothing
    for (int b = blockIdx.x; b < requests; b += gridDim.x) {
      if (prefix[b] != (b ? prefix[b - 1] : 0)) continue;
      const float zero[4] = {0.f, 0.f, 0.f, 0.f};
      for (int64_t i = tid; i < (int64_t)a.heads * (DIM / 4); i += 32 * kWarps) paged_store4(a.out, a.out_dtype, (int64_t)b * a.heads * DIM + 4 * i, zero);
      if (a.lse)
        for (int64_t i = tid; i < a.heads; i += 32 * kWarps) a.lse[(int64_t)b * a.heads + i] = -INFINITY;
    }
  };

  // ---- this CTA's run, and this warp's
  const int c = blockIdx.x;
  const int wanted = (int)(((uint32_t)total + (uint32_t)(groups * kPagedMinSteps - 1)) / (uint32_t)(groups * kPagedMinSteps));
  const int ctas = min(wanted, (int)gridDim.x);
  if (c >= ctas) {
    if (tid == 0) w.joins[c].lanes = 0;
    write_empty();
    return;
  }
  const PagedRuns runs(total, ctas);
  const int run0 = runs.begin(c), run1 = runs.begin(c + 1);
  const int group_bits = kWarpBits - shift;
  auto group_begin = [&](int i) { return run0 + (int)(((int64_t)(run1 - run0) * i + groups - 1) >> group_bits); };
  const int first_step = group_begin(my_group);
  const int todo = group_begin(my_group + 1) - first_step;

  const uint32_t ring = paged_smem(s_ring + warp * Tile::kRing);
  int final_part = 0, from_here = 0, row_done = 0;  // of the row that the warp's run ends in
  int cut = 0, early = 0;                           // the run begins inside a row; which ends inside the run
  PagedCursor cc = {0, 0, 0, 0};

  if (todo > 0) {
    // ---- copies, kStages - 1 steps ahead.  Where steps lie is found out for 32 of them at a time, one per lane, a whole such batch before
    // it is needed: behind the copies of all SMs a load (of a page's number, above all) takes 2 to 3 us.
    cc.locate(prefix, requests, heads, first_step);
    cut = cc.step > 0;
    if (warp == 0 && lane == 0) {
      s_cut_b = cc.b;
      s_cut_sub = cc.sub;
    }
    const int steps_per_page = (int)a.page_size / 16;
    const __nv_bfloat16* const q = static_cast<const __nv_bfloat16*>(a.q);
    struct Place {
      int page, slot, kv;
    };
    auto plan = [&](int base) {
      Place at = {-1, 0, 0};
      if (base + lane < todo) {
        PagedCursor pc = cc;
        pc.step += lane;
        if (base > 0 || pc.step >= pc.steps) pc.locate(prefix, requests, heads, first_step + base + lane);  // (cc: where the run begins, while base is 0)
        const int step = span_of(pc.b).first / 16 + pc.step, index = step / steps_per_page, sub = pc.sub * lanes + my_lane;
        at.page = a.block_table[(int64_t)pc.b * a.table_stride + index];  // (a step lies within a request's length, which its table covers)
        at.slot = 16 * (step - index * steps_per_page);
        at.kv = kv_of(sub);
        if (pc.step == 0 && base + lane > 0) {  // the queries of a row that begins here, into L1
          const int row0 = row_of(sub);
          const __nv_bfloat16* src = q + (int64_t)pc.b * a.q_token_stride + (int64_t)(at.kv * w.group + row0) * a.q_head_stride;
          for (int i = 0; i < min(Tile::kRows, w.group - row0); ++i)
#pragma unroll
            for (int d = 0; d < DIM; d += 64) {
              uint32_t unused;
              asm volatile("ld.global.ca.u32 %0, [%1];" : "=r"(unused) : "l"(src + i * a.q_head_stride + d));
            }
        }
      }
      return at;
    };
    Place now, soon;  // of steps [copied / 32 * 32, ...), and of the 32 behind them
    int copied = 0;
    uint32_t bad = 0;  // bit s: the step in stage s has no page
    auto copy_step = [&](int stage) {
      if (copied == todo) return;
      const int p = __shfl_sync(0xFFFFFFFFu, now.page, copied & 31);
      const int page = (uint32_t)p < (uint32_t)a.num_pages ? p : (int)a.num_pages;  // (behind the last page a copy brings zeros)
      const int slot = __shfl_sync(0xFFFFFFFFu, now.slot, copied & 31), kv = __shfl_sync(0xFFFFFFFFu, now.kv, copied & 31);
      const uint32_t bar = bars + 8 * stage, dst = ring + stage * Tile::kStage;
      bad = (bad & ~(1u << stage)) | ((uint32_t)(page == (int)a.num_pages) << stage);
      const bool made = !DROP || c != w.drop_cta || warp != w.drop_warp || copied != w.drop_step;
      if (made && ptx::elect_one()) {
        ptx::mbar_arrive_expect_tx(bar, Tile::kStage);
#pragma unroll
        for (int i = 0; i < Tile::kBoxes; ++i) paged_copy(dst + i * 16 * Tile::kBox, &map_k, bar, i * Tile::kBox, kv, slot, page);
#pragma unroll
        for (int i = 0; i < Tile::kBoxes; ++i)
          paged_copy(dst + 16 * Tile::kRow + i * 16 * Tile::kBox, &map_v, bar, i * Tile::kBox, kv, slot, page);
      }
      if ((++copied & 31) == 0) {
        now = soon;
        soon = plan(copied + 32);
      }
    };

    // ---- the products
    PagedAcc<DIM, FMT, NT> acc;
    uint32_t qf[kTiles][NT][2];
    float coef[NT][2];  // scores in powers of two for heads 2t, 2t + 1
    int c_lo = 0, c_end = 0, c_left = 0;  // keys of this step before c_lo are not seen, nor those of the row's last step from c_end on
    const float score_scale = a.softmax_scale * k_scale * 1.44269504088896341f;
    constexpr int kQ = Tile::kKChunks * (FMT == B200Q_BF16 ? 4 : 8);  // words of a head per lane
    auto load_queries = [&](const PagedCursor& at, uint32_t (&raw)[NT][kQ]) {
      const int sub = at.sub * lanes + my_lane, kv = kv_of(sub), row0 = row_of(sub);
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        const int row = row0 + 8 * n + g;
        const bool live = row < w.group;
        const __nv_bfloat16* src = q + (int64_t)at.b * a.q_token_stride + (int64_t)(kv * w.group + (live ? row : 0)) * a.q_head_stride;
#pragma unroll
        for (int i = 0; i < kQ / 4; ++i) {  // values as they meet the keys' bytes 64 c + 16 t ... + 15
          const uint4 v = *reinterpret_cast<const uint4*>(src + (FMT == B200Q_BF16 ? (4 * i + t) * 8 : (4 * (i / 2) + t) * 16 + 8 * (i % 2)));
          raw[n][4 * i] = v.x; raw[n][4 * i + 1] = v.y; raw[n][4 * i + 2] = v.z; raw[n][4 * i + 3] = v.w;
        }
      }
    };
    auto begin_row = [&](uint32_t (&raw)[NT][kQ]) {
      const PagedSpan span = span_of(cc.b);
      c_lo = cc.step == 0 ? span.first % 16 : 0;
      c_end = (span.len - 1) % 16 + 1;
      c_left = cc.steps - cc.step;
      from_here = cc.step == 0;
      acc.clear();
      const int rows = w.group - row_of(cc.sub * lanes + my_lane);
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        if (8 * n + g >= rows) {  // (a head that the group does not have: the loads brought another's)
#pragma unroll
          for (int i = 0; i < kQ; ++i) raw[n][i] = 0;
        }
        if (FMT == B200Q_BF16) {
#pragma unroll
          for (int i = 0; i < kQ; ++i) qf[i / 2][n][i % 2] = raw[n][i];
          coef[n][0] = coef[n][1] = score_scale;
        } else {
          uint32_t top = 0;
#pragma unroll
          for (int i = 0; i < kQ; ++i) top = __vmaxu2(top, raw[n][i] & 0x7FFF7FFFu);
          top = max(top & 0xFFFFu, top >> 16);
          top = max(top, __shfl_xor_sync(0xFFFFFFFFu, top, 1));
          top = max(top, __shfl_xor_sync(0xFFFFFFFFu, top, 2));
          // largest exponent of the head -> 2^8 (nothing to do for zeros; infinities and NaN stay what they are)
          const int e = (int)(top >> 7) - 127;
          const int up = top == 0 || e == 128 ? 0 : min(8 - e, 120);
          const float mul = __uint_as_float((uint32_t)(127 + up) << 23), back = __uint_as_float((uint32_t)(127 - up) << 23);
#pragma unroll
          for (int i = 0; i < kQ; ++i)
            qf[i / 2][n][i % 2] = paged_pack_f16(bf16_bits_to_float(raw[n][i] & 0xFFFFu) * mul, bf16_bits_to_float(raw[n][i] >> 16) * mul);
          coef[n][0] = score_scale * __shfl_sync(0xFFFFFFFFu, back, 8 * t);
          coef[n][1] = score_scale * __shfl_sync(0xFFFFFFFFu, back, 8 * t + 4);
        }
      }
    };
    {
      // the first queries are asked for before the copies: behind them a load takes 3 us
      uint32_t raw[NT][kQ];
      load_queries(cc, raw);
      now = plan(0);
      for (int s = 0; s < kStages - 1; ++s) copy_step(s);
      soon = plan(32);
      begin_row(raw);
    }
    if (tid == 0) {  // (while the first copies are on their way)
      PagedJoin join = {0, cc.b, cc.sub, 0};
      const int row0 = run0 - cc.step, row1 = row0 + cc.steps;
      if (cc.step > 0 && row0 >= runs.begin(c - 1)) {  // the row is cut here for the first time
        join.lanes = lanes;
        join.count = runs.cta_of(row1 - 1) - c + 1;
      }
      w.joins[c] = join;
    }

    // where the lane's pieces are in a stage: of keys R(g) + 8 h in box c / 2 at k_at ^ 64 (c % 2); of values key t + 4 i + 8 h
    const int rg = (g >> 1) | ((g & 1) << 2);
    const uint32_t k_at = Tile::kBox == 128 ? rg * 128 + ((t ^ rg) << 4) : rg * 64 + ((t ^ (rg >> 1)) << 4);
    const uint32_t v_at = Tile::kBox == 128 ? t * 128 + ((rg ^ t) << 4) : t * 64 + (((g >> 1) ^ (t >> 1)) << 4) + (g & 1) * 8;
    int stage = 0;
    uint32_t phase = 0;
    auto step_products = [&] {
      const uint32_t src = ring + stage * Tile::kStage, src_v = src + 16 * Tile::kRow + v_at;
      // scores: keys x heads
      float s[NT][4], s2[NT][4];
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int i = 0; i < 4; ++i) s[n][i] = s2[n][i] = 0.f;
#pragma unroll
      for (int i = 0; i < Tile::kKChunks; ++i) {
        const uint32_t at = src + (i >> 1) * 16 * Tile::kBox + (k_at ^ (64 * (i & 1)));
        const uint4 lo4 = paged_lds16(at), hi4 = paged_lds16(at + 8 * Tile::kBox);
        const uint32_t lo[4] = {lo4.x, lo4.y, lo4.z, lo4.w}, hi[4] = {hi4.x, hi4.y, hi4.z, hi4.w};
        if (FMT == B200Q_BF16) {
#pragma unroll
          for (int n = 0; n < NT; ++n) {
            paged_mma<FMT>(s[n], lo[0], hi[0], lo[1], hi[1], qf[2 * i][n][0], qf[2 * i][n][1]);
            paged_mma<FMT>(s2[n], lo[2], hi[2], lo[3], hi[3], qf[2 * i + 1][n][0], qf[2 * i + 1][n][1]);
          }
        } else {
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            uint32_t a0, a1, a2, a3;
            paged_f16<FMT>(lo[j], a0, a2);
            paged_f16<FMT>(hi[j], a1, a3);
#pragma unroll
            for (int n = 0; n < NT; ++n) paged_mma<FMT>(j & 1 ? s2[n] : s[n], a0, a1, a2, a3, qf[4 * i + j][n][0], qf[4 * i + j][n][1]);
          }
        }
      }
      const bool nowhere = bad >> stage & 1u;
      const bool edge = nowhere || c_lo > 0 || c_left == 1;  // some of its keys are not to be seen
      const int lo = nowhere ? 16 : c_lo, end = c_left == 1 ? c_end : 16;
      bool ok0 = true, ok1 = true;  // keys R(g), R(g) + 8
      if (edge) {
        ok0 = rg >= lo && rg < end;
        ok1 = 8 + rg >= lo && 8 + rg < end;
      }
      uint32_t p_hi[NT][2], p_lo[NT][2];
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        float x[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) s[n][i] += s2[n][i];
        // The product is rounded before the maximum is taken away, as it is where the maximum is found: the difference of a fused and a rounded
        // product of scores of 2^27 and more is a large number itself, and the largest probability then infinite, or none at all.
#pragma unroll
        for (int i = 0; i < 4; ++i) s[n][i] = (i < 2 ? ok0 : ok1) ? __fmul_rn(s[n][i], coef[n][i & 1]) : -INFINITY;
        auto exponents = [&] {
#pragma unroll
          for (int i = 0; i < 4; ++i) x[i] = __fsub_rn(s[n][i], acc.m[n][i & 1]);
        };
        exponents();
        if (__any_sync(0xFFFFFFFFu, fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3])) > Tile::kRescale)) {
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            float top = fmaxf(s[n][i], s[n][i + 2]);
#pragma unroll
            for (int o = 4; o < 32; o <<= 1) top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, o));
            const float raised = __fsub_rn(top, acc.m[n][i]) > Tile::kRescale ? top - Tile::kShift : acc.m[n][i];  // (by the exponent itself: m + 15 may be rounded up)
            const float keep = paged_exp2(acc.m[n][i] - raised);
            acc.m[n][i] = raised;
            acc.l[n][i] *= keep;
#pragma unroll
            for (int j = 0; j < kTiles; ++j) {
              acc.o[j][n][i] *= keep;
              acc.o[j][n][i + 2] *= keep;
            }
          }
          exponents();
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) x[i] = paged_exp2(x[i]);
        acc.l[n][0] += x[0] + x[2];
        acc.l[n][1] += x[1] + x[3];
        if (FMT == B200Q_BF16) {
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const uint32_t hi = pack_bf16x2(x[2 * i], x[2 * i + 1]);
            const uint32_t lo = pack_bf16x2(x[2 * i] - bf16_bits_to_float(hi & 0xFFFFu), x[2 * i + 1] - bf16_bits_to_float(hi >> 16));
            p_hi[n][i] = paged_transpose(hi);
            p_lo[n][i] = paged_transpose(lo);
          }
        } else {
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const uint32_t hi = paged_pack_f16(x[2 * i], x[2 * i + 1]);
            p_hi[n][i] = paged_transpose(hi);
            if (TERMS == 2) {
              const float2 back = paged_unpack_f16(hi);
              p_lo[n][i] = paged_transpose(paged_pack_f16(x[2 * i] - back.x, x[2 * i + 1] - back.y));
            }
          }
        }
      }
      // output: dimensions x heads
      // the piece of the key four rows on: the swizzle turns its place by 64 (rows of 128 bytes) or 32 bytes (of 64)
      auto v_four = [&](uint32_t at) { return (at + 4 * Tile::kBox) ^ (Tile::kBox == 128 ? 64 : 32); };
#pragma unroll
      for (int i = 0; i < Tile::kVChunks; ++i) {
        uint32_t v[4][Tile::kVPiece / 4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          // key t + 4 (k % 2) + 8 (k / 2): four rows on, the swizzled piece is the one across
          const uint32_t at = src_v + i * 16 * Tile::kBox + (k >> 1) * 8 * Tile::kBox;
          if (Tile::kVPiece == 16) {
            const uint4 x = paged_lds16(k & 1 ? v_four(at) : at);
            v[k][0] = x.x; v[k][1] = x.y; v[k][Tile::kVPiece / 4 - 2] = x.z; v[k][Tile::kVPiece / 4 - 1] = x.w;
          } else {
            const uint2 x = paged_lds8(k & 1 ? v_four(at) : at);
            v[k][0] = x.x; v[k][1] = x.y;
          }
          if (edge) {  // whatever lies there, 0 times it must be 0
            const int key = t + 4 * (k & 1) + 8 * (k >> 1);
            if (key < lo || key >= end) {
#pragma unroll
              for (int j = 0; j < Tile::kVPiece / 4; ++j) v[k][j] = 0;
            }
          }
        }
#pragma unroll
        for (int j = 0; j < Tile::kVPiece / 4; ++j) {
          if (FMT == B200Q_BF16) {
            const uint32_t a0 = __byte_perm(v[0][j], v[1][j], 0x5410), a1 = __byte_perm(v[0][j], v[1][j], 0x7632);
            const uint32_t a2 = __byte_perm(v[2][j], v[3][j], 0x5410), a3 = __byte_perm(v[2][j], v[3][j], 0x7632);
#pragma unroll
            for (int n = 0; n < NT; ++n) {
              paged_mma<FMT>(acc.o[i * 4 + j][n], a0, a1, a2, a3, p_hi[n][0], p_hi[n][1]);
              paged_mma<FMT>(acc.o[i * 4 + j][n], a0, a1, a2, a3, p_lo[n][0], p_lo[n][1]);
            }
          } else {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              const uint32_t sel = h ? 0x7362 : 0x5140;  // (key, next key) of two dimensions
              uint32_t a0, a1, a2, a3;
              paged_f16<FMT>(__byte_perm(v[0][j], v[1][j], sel), a0, a1);
              paged_f16<FMT>(__byte_perm(v[2][j], v[3][j], sel), a2, a3);
#pragma unroll
              for (int n = 0; n < NT; ++n) {
                auto& o = acc.o[(i * Tile::kVPiece + j * 4) / 2 + h][n];
                paged_mma<FMT>(o, a0, a1, a2, a3, p_hi[n][0], p_hi[n][1]);
                if (TERMS == 2) paged_mma<FMT>(o, a0, a1, a2, a3, p_lo[n][0], p_lo[n][1]);
              }
            }
          }
        }
      }
    };
    bool failed = false;  // a wait ran out: the rows of what is left of the run become NaN
    for (int done = 0; done < todo; ++done) {
      if (!failed && !ptx::mbar_wait_uniform(bars + 8 * stage, phase, &s_abort, w.status, kPagedErrCopy, DROP ? 1u << 12 : ptx::kWaitLimit)) {
        // gives up: makes no more copies, and waits for the others in flight, as far as they come
        failed = true;
        for (int s = 1; s < kStages && done + s < copied; ++s) {
          const int next = (stage + s) % kStages;
          for (int i = 0; i < 4096 && !ptx::mbar_try_wait(bars + 8 * next, phase ^ (stage + s >= kStages)); ++i) __nanosleep(64);
        }
        copied = todo;
      }
      if (failed) {
#pragma unroll
        for (int n = 0; n < NT; ++n) acc.l[n][0] = acc.l[n][1] = __int_as_float(0x7FC00000);
      } else {
        step_products();
        // the stage of the step before this one is free
        __syncwarp();
        copy_step(stage == 0 ? kStages - 1 : stage - 1);
      }
      if (++stage == kStages) {
        stage = 0;
        phase ^= 1;
      }
      c_lo = 0;

      const bool row_end = --c_left == 0, last = done + 1 == todo;
      if (row_end || last) {
        // the next row's queries are on their way while this one is finished, where there are registers for them
        constexpr bool kAhead = NT == 1 && DIM < 256;
        PagedCursor next = cc;
        uint32_t raw[NT][kQ];
        const bool more = !last && next.next_row(prefix, requests, heads);
        if (kAhead && more) load_queries(next, raw);
        acc.sum_lanes();
        if (row_end && from_here) {
          const int sub = cc.sub * lanes + my_lane, rows = w.group - row_of(sub);
          const int64_t head = (int64_t)cc.b * a.heads + kv_of(sub) * w.group + row_of(sub);
          float inv[NT][2];
#pragma unroll
          for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int i = 0; i < 2; ++i) inv[n][i] = acc.l[n][i] == 0.f ? 0.f : __fdividef(out_scale, acc.l[n][i]);
          auto write = [&](int dtype) {
            acc.each4(Tile::kVPiece == 16 ? rg : g, t, [&](int row, int d, const float (&v)[4], int n, int i) {
              const float r[4] = {v[0] * inv[n][i], v[1] * inv[n][i], v[2] * inv[n][i], v[3] * inv[n][i]};
              if (row < rows) paged_store4(a.out, dtype, head * DIM + (row * DIM + d), r);
            });
          };
          if (a.out_dtype == B200Q_BF16) write(B200Q_BF16);
          else write(a.out_dtype);
          if (a.lse && g == 0) {
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
              for (int i = 0; i < 2; ++i) {
                const int row = 8 * n + 2 * t + i;
                if (row < rows) a.lse[head + row] = paged_lse(acc.m[n][i], acc.l[n][i]);
              }
          }
        } else {
          // to the joining kernel, where no other warp of the CTA has a part of the row; else to where the CTA joins it
          float* to = groups == 1 ? w.cta_part + (((int64_t)c * 2 + from_here) * kWarps + my_lane) * Tile::kPart
                      : last      ? reinterpret_cast<float*>(s_ring + warp * Tile::kRing)
                                  : w.warp_part + ((int64_t)c * kWarps + warp) * Tile::kPart;
          __syncwarp();
          acc.save(to, g, Tile::kVPiece == 16 ? rg : g, t);
          if (last) {
            final_part = 1;
            row_done = row_end;
          } else {
            early = groups > 1;
          }
        }
        if (more) {
          cc = next;
          if (!kAhead) load_queries(cc, raw);
          begin_row(raw);
        }
      }
    }
  }
  write_empty();
  if (groups == 1) return;
  if (early) {  // into shared memory too, behind the part of the last row
    const float4* from = reinterpret_cast<const float4*>(w.warp_part + ((int64_t)c * kWarps + warp) * Tile::kPart);
    float4* to = reinterpret_cast<float4*>(s_ring + warp * Tile::kRing + 4 * Tile::kPart);
    __syncwarp();
#pragma unroll 9
    for (int i = lane; i < Tile::kPart / 4; i += 32) to[i] = from[i];
  }
  // what each warp leaves: 1 it had steps, 2 a part of its last row, 4 which it began, 8 which is done, 16 its run began inside a row
  if (lane == 0) {
    s_state[warp] = todo > 0 ? 1 | final_part << 1 | from_here << 2 | row_done << 3 | cut << 4 : 0;
    s_b[warp] = cc.b;
    s_sub[warp] = cc.sub;
  }
  __syncthreads();

  // ---- rows that several groups of warps have a part of; a task is one head of one lane
  const int state = lane < groups ? s_state[lane << shift] : 0;  // (the lanes of a group are alike in all but the head)
  const uint32_t has = __ballot_sync(0xFFFFFFFFu, state & 1), last_part = __ballot_sync(0xFFFFFFFFu, state & 2);
  const uint32_t began = __ballot_sync(0xFFFFFFFFu, state & 4), done_bits = __ballot_sync(0xFFFFFFFFu, state & 8);
  const uint32_t through = last_part & ~began;            // the group's last row came from the one before: its part is in shared memory
  const uint32_t on = through & ~done_bits;               // ... and goes on
  uint32_t starts = last_part & began;                    // rows that begin in a group and go on
  bool from_cut = __shfl_sync(0xFFFFFFFFu, state, 0) & 16;  // the row from the CTA before comes first
  while (from_cut || starts) {
    const int first = from_cut ? 0 : __ffs(starts) - 1;
    if (!from_cut) starts &= starts - 1;
    uint32_t parts = 1u << first;
    bool ended = from_cut && !(on & 1u);
    if (!ended) {  // the groups behind, up to the first one in which the row does not go on
      const uint32_t behind = has & ~((2u << first) - 1u), stops = behind & ~on;
      ended = stops != 0;
      parts |= ended ? behind & ((stops & (0u - stops)) * 2u - 1u) : behind;
    }
    const uint32_t here = (from_cut ? through : through | 1u << first) & parts;  // the others ended in the middle of a run
    const int b = from_cut ? s_cut_b : s_b[first << shift], group = from_cut ? s_cut_sub : s_sub[first << shift];
    for (int task = warp; task < lanes * Tile::kRows; task += kWarps) {
      const int l_head = task & (lanes - 1), row = task >> shift;
      const int sub = (group << shift) + l_head, kv = kv_of(sub), row0 = row_of(sub);
      if (row0 + row >= w.group) continue;
      auto part_of = [&](int v) {
        return reinterpret_cast<const float*>(s_ring + ((v << shift) + l_head) * Tile::kRing + (here >> v & 1u ? 0 : 4 * Tile::kPart));
      };
      const bool mine = lane < kWarps && (parts >> lane & 1u);
      float pm = kPagedNoMax, pl = 0.f, x[kWarps][DIM / 32];
      if (mine) {
        const float* p = part_of(lane) + Tile::kRows * DIM + row;
        pm = p[0];
        pl = s_abort ? __int_as_float(0x7FC00000) : p[Tile::kRows];  // (where a wait ran out, a late copy may yet land on a part)
      }
#pragma unroll
      for (int v = 0; v < kWarps; ++v) {
        const bool part = parts >> v & 1u;
        const float* p = part_of(part ? v : first) + row * DIM + lane;
#pragma unroll
        for (int d = 0; d < DIM / 32; ++d) x[v][d] = part ? p[d * 32] : 0.f;
      }
      float m = pm;
#pragma unroll
      for (int s = kWarps / 2; s > 0; s >>= 1) m = fmaxf(m, __shfl_xor_sync(0xFFFFFFFFu, m, s));
      m = __shfl_sync(0xFFFFFFFFu, m, 0);
      const float weight = mine ? exp2f(pm - m) : 0.f;  // (inf - inf: a NaN row, as its parts are)
      float l = weight * pl, o[DIM / 32];
#pragma unroll
      for (int s = kWarps / 2; s > 0; s >>= 1) l += __shfl_xor_sync(0xFFFFFFFFu, l, s);
      l = __shfl_sync(0xFFFFFFFFu, l, 0);
#pragma unroll
      for (int d = 0; d < DIM / 32; ++d) o[d] = 0.f;
#pragma unroll
      for (int v = 0; v < kWarps; ++v) {
        const float y = __shfl_sync(0xFFFFFFFFu, weight, v);
#pragma unroll
        for (int d = 0; d < DIM / 32; ++d) o[d] += y * x[v][d];
      }
      if (!from_cut && ended) {
        paged_finish<DIM>(a, b, kv * w.group + row0 + row, lane, o, m, l, out_scale);
      } else {
        float* to = w.cta_part + (((int64_t)c * 2 + (from_cut ? 0 : 1)) * kWarps + l_head) * Tile::kPart;
#pragma unroll
        for (int d = 0; d < DIM / 32; ++d) to[row * DIM + d * 32 + lane] = o[d];
        if (lane == 0) {
          to[Tile::kRows * DIM + row] = m;
          to[Tile::kRows * DIM + Tile::kRows + row] = l;
        }
      }
    }
    from_cut = false;
  }
}

// Rows that several CTAs have a part of.  Every block makes the list of them; one (row of heads, lane, head) is a task, of a warp where
// there are many, and of a whole block where there are fewer than blocks (long rows of few requests, with up to a part per CTA).
constexpr int kPagedJoinBlocks = 2 * kNumSMs;  // (all resident at once; one per SM leaves 128 x 200 tokens at 31.4 instead of 26.5 us)
constexpr int kPagedJoinWarps = 8;

template <int DIM, int ROWS, int WARPS>
__global__ void __launch_bounds__(32 * kPagedJoinWarps) paged_join_kernel(const b200q_paged_attention_args a, const PagedWork w, int ctas) {
  constexpr int kPart = ROWS * (DIM + 2);
  __shared__ float s_o[kPagedJoinWarps][DIM], s_m[kPagedJoinWarps], s_l[kPagedJoinWarps];
  __shared__ PagedJoin s_join[kPagedGrid];
  __shared__ int s_cta[kPagedGrid], s_count[kPagedJoinWarps];
  static_assert(kPagedGrid <= 32 * kPagedJoinWarps, "a thread per CTA");
  pdl_enter();
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  int4 v = make_int4(0, 0, 0, 0);
  if (tid < ctas) v = __ldcg(reinterpret_cast<const int4*>(w.joins) + tid);
  const uint32_t vote = __ballot_sync(0xFFFFFFFFu, v.x != 0);
  if (lane == 0) s_count[warp] = __popc(vote);
  __syncthreads();
  int rows = 0, before = __popc(vote & ((1u << lane) - 1u));
#pragma unroll
  for (int i = 0; i < kPagedJoinWarps; ++i) {
    if (i < warp) before += s_count[i];
    rows += s_count[i];
  }
  if (v.x != 0) {
    s_join[before] = {v.x, v.y, v.z, v.w};
    s_cta[before] = tid;
  }
  __syncthreads();
  if (rows == 0) return;
  const int lanes = s_join[0].lanes, per_row = lanes * ROWS, tasks = rows * per_row;
  // a warp's task takes a trip to L2 per 8 parts, of which a row has 1 + (ctas - 1) / rows on average; a block's takes one or two
  const bool by_block = (tasks - 1) / (int)gridDim.x <= (ctas - 1) / (8 * rows);
  const float scale = paged_out_scale(a);
  for (int task = blockIdx.x + (by_block ? 0 : gridDim.x * warp); task < tasks; task += by_block ? gridDim.x : gridDim.x * kPagedJoinWarps) {
    const PagedJoin join = s_join[task / per_row];
    const int c = s_cta[task / per_row], l_head = task % per_row / ROWS, row = task % ROWS;
    const int sub = join.sub * lanes + l_head, kv = sub / w.row_tiles, row0 = (sub - kv * w.row_tiles) * ROWS;
    if (row0 + row >= w.group) continue;
    const int head = kv * w.group + row0 + row;
    // part 0: the CTA before's last row; part i: the first row of CTA c + i - 1
    const int count = join.count + 1, per = by_block ? (count + kPagedJoinWarps - 1) / kPagedJoinWarps : count;
    const int i0 = by_block ? min(warp * per, count) : 0, n = min(per, count - i0);
    float m, l, o[DIM / 32];
    paged_merge<DIM, ROWS>(
        [&](int i) { return w.cta_part + ((i0 + i == 0 ? (int64_t)(c - 1) * 2 + 1 : (int64_t)(c + i0 + i - 1) * 2) * WARPS + l_head) * kPart; }, n, row, lane, o, m,
        l);
    if (by_block) {
#pragma unroll
      for (int d = 0; d < DIM / 32; ++d) s_o[warp][d * 32 + lane] = o[d];
      if (lane == 0) {
        s_m[warp] = m;
        s_l[warp] = l;
      }
      __syncthreads();
      if (warp == 0) {
        m = kPagedNoMax;
#pragma unroll
        for (int i = 0; i < kPagedJoinWarps; ++i) m = fmaxf(m, s_m[i]);
        l = 0.f;
#pragma unroll
        for (int d = 0; d < DIM / 32; ++d) o[d] = 0.f;
#pragma unroll
        for (int i = 0; i < kPagedJoinWarps; ++i) {
          if (i * per >= count) break;
          const float x = exp2f(s_m[i] - m);
          l += x * s_l[i];
#pragma unroll
          for (int d = 0; d < DIM / 32; ++d) o[d] += x * s_o[i][d * 32 + lane];
        }
      }
      __syncthreads();
      if (warp != 0) continue;
    }
    paged_finish<DIM>(a, join.request, head, lane, o, m, l, scale);
  }
}

// ---------------------------------------------------------------------------- host
static bool paged_tensor_dim(int dim) { return dim == 64 || dim == 128 || dim == 256; }
// query heads of a row tile: 16 where more than 8 share a key/value head, which then is read once for them; heads of 256
// values in two tiles do not fit the registers
static int paged_rows_of(int group, int dim) { return group <= 8 || dim == 256 ? 8 : 16; }

// Where the three parts of the workspace lie, for the size that a caller is told and for the kernels alike.
struct PagedSpace {
  size_t cta_part, warp_part, bytes;
  static constexpr size_t align(size_t n) { return (n + 255) / 256 * 256; }
  constexpr PagedSpace(int rows, int dim, int warps)
      : cta_part(align(sizeof(PagedJoin) * kPagedGrid)),
        warp_part(cta_part + align(sizeof(float) * rows * (dim + 2) * 2 * warps * kPagedGrid)),
        bytes(warp_part + align(sizeof(float) * rows * (dim + 2) * warps * kPagedGrid)) {}
};

size_t paged_attention_workspace_bytes_impl(int64_t requests, int heads, int kv_heads, int dim, int cache_dtype) {
  (void)requests;  // (rows are joined per CTA, whatever the number of requests)
  (void)cache_dtype;
  if (!paged_tensor_dim(dim)) return 0;
  return PagedSpace(paged_rows_of(heads / kv_heads, dim), dim, paged_warps_of(dim)).bytes;
}

// A cache as [pages][slots][heads][bytes of a head], whatever the order of its strides, in boxes of 16 slots
static int paged_map(CUtensorMap* map, const void* base, const b200q_paged_attention_args& a, int64_t size, int64_t page_stride, int64_t slot_stride,
                     int64_t head_stride) {
  EncodeTiledFn enc = get_encode_fn();
  if (!enc) return B200Q_ERR_CUDA;
  const cuuint64_t row = (cuuint64_t)(a.dim * size);
  const cuuint32_t inner = row < 128 ? (cuuint32_t)row : 128;
  // (the stride of a dimension of one entry is never used, and may be anything in the caller's view)
  const cuuint64_t dims[4] = {row, (cuuint64_t)a.kv_heads, (cuuint64_t)a.page_size, (cuuint64_t)a.num_pages};
  const cuuint64_t strides[3] = {a.kv_heads > 1 ? (cuuint64_t)(head_stride * size) : row, (cuuint64_t)(slot_stride * size),
                                 a.num_pages > 1 ? (cuuint64_t)(page_stride * size) : row};
  const cuuint32_t box[4] = {inner, 1, 16, 1}, step[4] = {1, 1, 1, 1};
  const CUresult r = enc(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 4, const_cast<void*>(base), dims, strides, box, step, CU_TENSOR_MAP_INTERLEAVE_NONE,
                         inner == 128 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B, CU_TENSOR_MAP_L2_PROMOTION_L2_128B,
                         CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return r == CUDA_SUCCESS ? B200Q_OK : B200Q_ERR_UNSUPPORTED;
}

struct PagedDrop {
  int cta, warp, step;
};
template <int DIM, int FMT, int NT, int TERMS, bool DROP = false>
static int paged_launch(const b200q_paged_attention_args& a, cudaStream_t st, PagedDrop drop = {}) {
  using Tile = PagedTile<DIM, FMT, NT>;
  auto kernel = paged_attention_kernel<DIM, FMT, NT, TERMS, DROP>;
  static std::atomic<int> ready[kMaxDevices];
  const int dev = current_device_index();
  if (dev < 0) return B200Q_ERR_CUDA;
  if (!ready[dev].load(std::memory_order_acquire)) {
    B200Q_CUDA_OK(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)(Tile::kWarps * Tile::kRing + 1024 + 4 * kPagedMaxRequests)));
    ready[dev].store(1, std::memory_order_release);
  }
  CUtensorMap map_k, map_v;
  if (int rc = paged_map(&map_k, a.k_cache, a, Tile::kElt, a.k_page_stride, a.k_slot_stride, a.k_head_stride)) return rc;
  if (int rc = paged_map(&map_v, a.v_cache, a, Tile::kElt, a.v_page_stride, a.v_slot_stride, a.v_head_stride)) return rc;
  PagedWork w;
  w.drop_cta = drop.cta;
  w.drop_warp = drop.warp;
  w.drop_step = drop.step;
  w.status = device_status_ptr();
  if (!w.status) return B200Q_ERR_CUDA;
  w.group = a.heads / a.kv_heads;
  w.row_tiles = (w.group + Tile::kRows - 1) / Tile::kRows;
  w.heads_per_request = a.kv_heads * w.row_tiles;
  w.lane_bits = 0;
  while ((2 << w.lane_bits) <= Tile::kWarps && w.heads_per_request % (2 << w.lane_bits) == 0) ++w.lane_bits;
  constexpr PagedSpace space(Tile::kRows, DIM, Tile::kWarps);
  static_assert(Tile::kPart == Tile::kRows * (DIM + 2), "the size of a part in PagedSpace");
  if (a.workspace_bytes < space.bytes) return B200Q_ERR_BAD_ARGUMENT;  // (this instance's own need, whatever the caller was told)
  uint8_t* p = static_cast<uint8_t*>(a.workspace);
  w.joins = reinterpret_cast<PagedJoin*>(p);
  w.cta_part = reinterpret_cast<float*>(p + space.cta_part);
  w.warp_part = reinterpret_cast<float*>(p + space.warp_part);
  // no more CTAs than the longest list that the tables can hold would fill
  const int64_t most = a.requests * ((a.table_width * a.page_size + 15) / 16) * w.heads_per_request;
  int64_t grid = (most + Tile::kWarps * kPagedMinSteps - 1) / (Tile::kWarps * kPagedMinSteps);
  if (grid < 1) grid = 1;
  if (grid > kPagedGrid) grid = kPagedGrid;
  launch_dependent(kernel, dim3((unsigned)grid), dim3(32 * Tile::kWarps), Tile::kWarps * Tile::kRing + 1024 + (a.requests <= kPagedLengthsHere ? 8 : 4) * (size_t)a.requests, st, map_k, map_v, a, w);
  B200Q_LAUNCH_CHECK();
  if (grid > 1) {
    launch_dependent(paged_join_kernel<DIM, 8 * NT, Tile::kWarps>, dim3(kPagedJoinBlocks), dim3(32 * kPagedJoinWarps), 0, st, a, w, (int)grid);
    B200Q_LAUNCH_CHECK();
  }
  return B200Q_OK;
}

template <int DIM, int FMT, int TERMS>
static int paged_launch_rows(const b200q_paged_attention_args& a, cudaStream_t st) {
  if constexpr (DIM < 256) {
    if (paged_rows_of(a.heads / a.kv_heads, DIM) == 16) return paged_launch<DIM, FMT, 2, TERMS>(a, st);
  }
  return paged_launch<DIM, FMT, 1, TERMS>(a, st);
}
// One term for an fp8 cache where the output is rounded to 8 bits or fewer, two where it is fp32 (see above).
template <int DIM, int FMT>
static int paged_launch_terms(const b200q_paged_attention_args& a, cudaStream_t st) {
  return a.out_dtype == B200Q_F32 ? paged_launch_rows<DIM, FMT, 2>(a, st) : paged_launch_rows<DIM, FMT, 1>(a, st);
}
template <int DIM>
static int paged_launch_dtype(const b200q_paged_attention_args& a, cudaStream_t st) {
  switch (a.cache_dtype) {
    case B200Q_BF16: return paged_launch_rows<DIM, B200Q_BF16, 2>(a, st);
    case B200Q_E4M3: return paged_launch_terms<DIM, B200Q_E4M3>(a, st);
    default: return paged_launch_terms<DIM, B200Q_E5M2>(a, st);
  }
}

static bool paged_fits_tensor_cores(const b200q_paged_attention_args& a) {
  if (a.force_plain || !paged_tensor_dim(a.dim) || a.page_size % 16 || a.num_pages == 0) return false;
  const int64_t size = a.cache_dtype == B200Q_BF16 ? 2 : 1;
  for (const void* p : {a.q, a.k_cache, a.v_cache, static_cast<const void*>(a.out)})
    if (reinterpret_cast<uintptr_t>(p) % 16) return false;
  for (int64_t s : {a.k_page_stride, a.k_slot_stride, a.k_head_stride, a.v_page_stride, a.v_slot_stride, a.v_head_stride})
    if (s < 0 || s * size % 16) return false;
  return a.q_token_stride % 8 == 0 && a.q_head_stride % 8 == 0;
}

static int paged_check_tensor_cores(const b200q_paged_attention_args& a) {
  if (a.requests > kPagedMaxRequests) return B200Q_ERR_TOO_LARGE;
  // the steps that the tables can hold, of all heads' row tiles, are counted in 31 bits
  const int rows = paged_rows_of(a.heads / a.kv_heads, a.dim);
  const int64_t tiles = (int64_t)a.kv_heads * ((a.heads / a.kv_heads + rows - 1) / rows), row_steps = (a.table_width * a.page_size + 15) / 16;
  if (row_steps > INT32_MAX || tiles > INT32_MAX || (row_steps > 0 && a.requests > INT32_MAX / row_steps / tiles)) return B200Q_ERR_TOO_LARGE;
  if (a.workspace_bytes < paged_attention_workspace_bytes_impl(a.requests, a.heads, a.kv_heads, a.dim, a.cache_dtype) || !a.workspace ||
      reinterpret_cast<uintptr_t>(a.workspace) % 16)
    return B200Q_ERR_BAD_ARGUMENT;
  return B200Q_OK;
}

int paged_attention_impl(const b200q_paged_attention_args& a, cudaStream_t st) {
  if (paged_fits_tensor_cores(a)) {
    if (int rc = paged_check_tensor_cores(a)) return rc;
    const int rc = a.dim == 64 ? paged_launch_dtype<64>(a, st) : a.dim == 128 ? paged_launch_dtype<128>(a, st) : paged_launch_dtype<256>(a, st);
    if (rc != B200Q_ERR_UNSUPPORTED) return rc;  // (a layout that has no tensor map takes the plain kernel)
  }
  const int64_t blocks = a.requests * a.heads;
  if (blocks > 0x7FFFFFFF) return B200Q_ERR_TOO_LARGE;
  launch_dependent(paged_attention_plain_kernel, dim3((unsigned)blocks), dim3(kPlainThreads), 0, st, a);
  B200Q_LAUNCH_CHECK();
  return B200Q_OK;
}

// The kernel for heads of 128 in e4m3 with a step whose keys and values never arrive.
int paged_selftest_impl(const b200q_paged_attention_args& a, int cta, int warp, int step, cudaStream_t st) {
  if (!paged_fits_tensor_cores(a) || a.dim != 128 || a.cache_dtype != B200Q_E4M3 || a.out_dtype != B200Q_BF16 || paged_rows_of(a.heads / a.kv_heads, 128) != 8)
    return B200Q_ERR_UNSUPPORTED;
  if (int rc = paged_check_tensor_cores(a)) return rc;
  return paged_launch<128, B200Q_E4M3, 1, 1, true>(a, st, {cta, warp, step});
}

}  // namespace b200q
