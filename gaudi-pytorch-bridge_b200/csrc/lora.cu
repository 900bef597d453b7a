// Low-rank adapters of many requests beside a product that they share: y[t] += scale * b (a x[t]) with the adapter of each token.
#include "layer.cuh"
#include "tma_host.cuh"

namespace b200q {

constexpr int64_t kLoraChunk = 8192;  // tokens taken at a time
constexpr size_t lora_align(size_t n) { return (n + 255) / 256 * 256; }

__device__ __forceinline__ float lora_bf16(const void* p, int64_t at) { return __bfloat162float(static_cast<const __nv_bfloat16*>(p)[at]); }
__device__ __forceinline__ int lora_adapter(const b200q_lora_args& a, int64_t t) {  // or -1
  const int i = __ldcg(a.adapter + t);
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
// taken together, in whatever order they come, or its matrices are read again for each: a first kernel sorts the tokens by adapter into tiles.  In both products
// the adapter's matrix has the 128 rows of tcgen05.mma (ranks, or columns of y) and the tile's tokens are its columns, so that a warp's results are
// neighbours in memory: a x is bf16 times bf16, both by TMA (tokens by gathered rows); b (a x) has a x in bf16 terms that follow one another along K.
//
// us: 4096 tokens of 4096 -> 14336, rank 64, 8 adapters in runs of 512 tokens 78 to 86 (floor, y twice and x once, 38: the sorting 5, a x 18, the rest b (a x)); 64 tokens of 8192 -> 8192 with
// 56 of 64 adapters of rank 32 22 (floor 9.4: the steps of two kernels one behind the other); one token of 4096 -> 4096, rank 16, 8.6 (7.2 on the device), two kernels' latency.
// With mma.sync and the tokens as rows these were 162, 32 and 6.2.
constexpr int kLoraSortThreads = 1024;
constexpr int kLoraFew = 128;  // tokens up to which each CTA sorts for itself
constexpr int kLoraErrCopy = 831, kLoraErrMma = 832, kLoraErrResults = 833;  // status codes: a wait ran out
constexpr uint32_t kLoraTestPolls = 1u << 14;  // of the self-test: some ten milliseconds

struct __align__(16) LoraTile {
  int adapter, first, count, unused;  // tokens sorted[first] ...
};
struct LoraPlan {
  int* tiles_used;  // or null: the plan is made by each CTA
  LoraTile* tiles;
  int* sorted;
  float* low;  // [splits][tokens][rank]: a x, in parts over k
  int splits, slots;  // parts of k at most; CTAs that share a x
  int steps;          // of 64 values of k
  int tile;                       // tokens of a tile at most
  int* status;
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

// Tiles of 128 tokens read the adapters' matrices less often, and tiles of 16 are more, take less shared memory and so have more copies on their way.  us with 16 and with 128, bf16, k = n =
// 4096 and 8 adapters where nothing else is said:
// * tokens: rank 16 to 64: 1024 22, 31 to 34; 2600 35, 40; 3500 45, 42; 5000 72, 48; 8192 82, 67 to 87, 67; fp32, rank 64: 2600 45, 53; 3500 68, 59.  A rank of 129 and more is two blocks of rows
//   that fetch the tokens twice, rank 192: 1024 57, 89; 2048 81, 75 (n = 14336 159, 98); 4096 131, 85 (285, 132);
// * tokens times k + n, 2^20: k = n = 1024 (4096 to 8192 tokens, 8 to 16) 22, 26 and 32, 33; k = 4096, n = 1024 (20) 29, 32; k = 1024, n = 4096 (20) 39, 38; (27) as above; rank 128, whose terms leave room
//   for one CTA: 3500 tokens (27) 62, 71; 4096 (32) 65, 74; 5000 (39) 99, 75; n = 14336 (72) 138, 122; in fp32 (32) 98, 76;
// * adapters: 8192 tokens of 128 adapters 79, 89 (k = 14336 133, 190), because their tiles and those that there might be leave a x whole; 4096 tokens of 64 53, 47, of 128 53, 60; 8192 of 84 90, 76.
// What counts is the table's adapters, which the host knows, not those that are used: 4096 tokens of one of 256 60, 55.
static int lora_tile_tokens(int64_t tokens, int64_t k, int64_t n, int64_t rank, int64_t adapters, bool wide) {
  const int64_t t = tokens < kLoraChunk ? tokens : kLoraChunk, blocks = (wide ? 3 : 2) * ((rank + 63) / 64);
  if (blocks > 6 || adapters + t / 128 > kNumSMs) return 16;  // (more terms leave no room for the copies)
  if (rank > 128) return t >= 2048 ? 128 : 16;
  const int64_t least = rank > 64 && !wide ? 36 : 24;
  return t >= 3200 && t * (k + n) >= least << 20 ? 128 : 16;
}
// CTAs of an SM that share a x: more where ranks are few, because an item is a chain of steps
// (64 tokens of 56 adapters of rank 32, 8192 values each: 24.3 us with two, 22.6 with four)
static int lora_down_ctas(int64_t rank, int tile) { return tile == 16 && rank <= 64 ? 4 : 2; }
// tiles that the tokens may need at most, and parts of k at most.  The kernels, which know how many tiles there are, take as many parts as leave no CTA a second item (a second
// round costs as much as the first); the workspace has room for as many as that can be, which is little where tokens are few, and where they are many for what the most tiles leave.
static int64_t lora_most_tiles(int64_t tokens, int64_t adapters, int tile) {
  const int64_t t = tokens < kLoraChunk ? tokens : kLoraChunk, shared = adapters + t / tile;
  return t < shared ? t : shared;
}
static int64_t lora_splits(int64_t tokens, int64_t k, int64_t rank, int64_t adapters, int tile) {
  const int64_t most = (k + 255) / 256, items = lora_most_tiles(tokens, adapters, tile) * ((rank + 127) / 128);
  const int64_t wanted = tokens <= kLoraFew ? 16 : lora_down_ctas(rank, tile) * kNumSMs / items;
  const int64_t splits = wanted < most ? wanted : most;
  return splits < 1 ? 1 : splits < 16 ? splits : 16;
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
  constexpr int kKept = (int)kLoraChunk / kLoraSortThreads;  // tokens of a thread
  const int per = (tokens + 32 * kWarps - 1) / (32 * kWarps), begin = warp * per * 32;
  int adapter[kKept];
#pragma unroll
  for (int i = 0; i < kKept; ++i) adapter[i] = i < per && begin + 32 * i + lane < tokens ? lora_adapter(a, begin + 32 * i + lane) : -1;
  for (int i = tid; i < kWarps * adapters; i += kLoraSortThreads) s_count[i] = 0;
  __syncthreads();
  int place[kKept];  // among the warp's tokens of the adapter
#pragma unroll
  for (int i = 0; i < kKept; ++i) {
    if (i >= per) break;
    const uint32_t same = __match_any_sync(0xFFFFFFFFu, adapter[i]);
    place[i] = adapter[i] >= 0 ? mine[adapter[i]] + __popc(same & ((1u << lane) - 1u)) : 0;
    __syncwarp();
    if (adapter[i] >= 0 && lane == __ffs(same) - 1) mine[adapter[i]] += (uint16_t)__popc(same);
    __syncwarp();
  }
  __syncthreads();
  int tokens_before = 0, tiles_before = 0;
  for (int base = 0, turn = 0; base < adapters; base += kLoraSortThreads, turn ^= 1) {
    const int i = base + tid;
    int n = 0;
    if (i < adapters) {
#pragma unroll 8
      for (int w = 0; w < kWarps; ++w) {
        const int c = s_count[w * adapters + i];
        s_count[w * adapters + i] = (uint16_t)n;
        n += c;
      }
    }
    const int tiles = (n + p.tile - 1) / p.tile, both = n | tiles << 16;  // (sums of at most 8192 each)
    int scan = both;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int v = __shfl_up_sync(0xFFFFFFFFu, scan, o);
      if (lane >= o) scan += v;
    }
    if (lane == 31) s_scan[turn][warp] = scan;
    __syncthreads();  // (the other half is written next, and this one only behind the next barrier)
    int sums = s_scan[turn][lane];
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int v = __shfl_up_sync(0xFFFFFFFFu, sums, o);
      if (lane >= o) sums += v;
    }
    const int here = tokens_before | tiles_before << 16, all = here + __shfl_sync(0xFFFFFFFFu, sums, 31);
    int before = __shfl_sync(0xFFFFFFFFu, sums, warp == 0 ? 0 : warp - 1);
    before = here + (warp == 0 ? 0 : before) + scan - both;
    tokens_before = all & 0xFFFF;
    tiles_before = all >> 16;
    if (i < adapters) s_first[i] = (uint16_t)(before & 0xFFFF);
    for (int j = 0; j < tiles; ++j) p.tiles[(before >> 16) + j] = {i, (before & 0xFFFF) + j * p.tile, min(n - j * p.tile, p.tile), 0};
  }
  if (tid == 0) *p.tiles_used = tiles_before;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kKept; ++i)
    if (i < per && adapter[i] >= 0) p.sorted[s_first[adapter[i]] + mine[adapter[i]] + place[i]] = begin + 32 * i + lane;
}

// The plan as a CTA finds it: made by the kernel in front, or, for few tokens, here (a launch takes longer): a thread per token counts those that come before it in the order.
struct LoraFew {
  int adapter[kLoraFew], sorted[kLoraFew];
  LoraTile tiles[kLoraFew];
  uint32_t first[kLoraFew / 32];  // a bit for each place that a tile begins at
};
struct LoraView {
  int tiles_used;
  bool made;  // by a kernel: in global memory, and before a kernel has waited read past L1, which may be older than it
  const LoraTile* tiles;
  const int* sorted;
  __device__ __forceinline__ LoraTile tile(int i) const {
    if (!made) return tiles[i];
    const int4 v = __ldcg(reinterpret_cast<const int4*>(tiles) + i);
    return {v.x, v.y, v.z, v.w};
  }
  __device__ __forceinline__ int token(int i) const { return made ? __ldcg(sorted + i) : sorted[i]; }
};
__device__ __forceinline__ int lora_parts(const LoraPlan& p, int items) { return max(1, min(p.splits, p.slots / max(items, 1))); }
template <int TILE>
__device__ __forceinline__ LoraView lora_view(const b200q_lora_args& a, const LoraPlan& p, LoraFew& few) {
  if (TILE > 16 || p.tiles_used) return {__ldcg(p.tiles_used), true, p.tiles, p.sorted};
  constexpr int kNone = 0x7FFFFFFF;
  const int t = threadIdx.x, tokens = (int)a.tokens;
  int mine = kNone;
  if (t < kLoraFew) {
    if (t < tokens) {
      const int i = lora_adapter(a, t);
      mine = i < 0 ? kNone : i;
    }
    few.adapter[t] = mine;
    if (t < kLoraFew / 32) few.first[t] = 0;
  }
  __syncthreads();
  int lower = 0, same = 0, same_before = 0;
  if (mine != kNone) {
#pragma unroll 4
    for (int j = 0; j < tokens; j += 4) {
      const int4 other = *reinterpret_cast<const int4*>(few.adapter + j);
      const int v[4] = {other.x, other.y, other.z, other.w};
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        lower += v[c] < mine;
        same += v[c] == mine;
        same_before += v[c] == mine && j + c < t;
      }
    }
  }
  const int place = lower + same_before;
  const bool first = mine != kNone && same_before % p.tile == 0;
  if (mine != kNone) few.sorted[place] = t;
  if (first) atomicOr(&few.first[place / 32], 1u << (place & 31));
  __syncthreads();
  int used = 0, tile = 0;
#pragma unroll
  for (int i = 0; i < kLoraFew / 32; ++i) {
    used += __popc(few.first[i]);
    tile += __popc(few.first[i] & (place >= 32 * i + 32 ? ~0u : place <= 32 * i ? 0u : (1u << (place & 31)) - 1u));
  }
  if (first) few.tiles[tile] = {mine, place, min(same - same_before, p.tile), 0};
  __syncthreads();
  return {used, false, few.tiles, few.sorted};
}

// Before a CTA ends its last copies are waited for, as far as they come.  (Where no wait has run out they have been multiplied, or will be next.)
__device__ __forceinline__ void lora_drain(uint32_t bars, int stages, int made, uint32_t stage, uint32_t phase) {
  for (int i = 0; i < min(made, stages); ++i) {
    phase ^= stage == 0;
    stage = stage == 0 ? stages - 1 : stage - 1;
    for (int k = 0; k < 4096 && !ptx::mbar_try_wait(bars + 8 * stage, phase); ++k) __nanosleep(64);
  }
}
// nor do products outlive the tensor memory and the ring (the warp that issued them; `bar` is for this alone)
__device__ __forceinline__ void lora_drain_products(uint32_t bar) {
  if (ptx::elect_one()) ptx::umma_commit(bar);
  __syncwarp();
  for (int k = 0; k < 4096 && !ptx::mbar_try_wait(bar, 0); ++k) __nanosleep(64);
}
__host__ __device__ constexpr int lora_columns(int tokens) { return (tokens + 15) / 16 * 16; }

// a x of a tile's tokens over a part of k: ranks are the rows of the product, tokens its columns.  A step is 64 values of k of up to 128 ranks and the tile's tokens.
constexpr int kLoraMostStages = 8;
constexpr int kLoraDownWarps = 6;  // copies, MMAs, four of results
// An addition inside the tensor core drops what does not fit 24 bits: behind a row of 2048 products a y in fp32 would be off by 5e-7 where plain fp32 sums are by 1e-7.  So for
// such a y no more than 256 are added there (2e-7).
constexpr int kLoraSub = 4;
struct LoraDownShape {
  int rows, row_bytes, stage, stages;  // ranks of a block; bytes of them and of a stage
  LoraDownShape(int rank, int tile, int smem) {
    rows = rank < 128 ? rank : 128;
    row_bytes = rows * 128;
    stage = row_bytes + tile * 128;
    stages = (smem - 16384) / stage;
    if (stages > kLoraMostStages) stages = kLoraMostStages;
  }
};

// EXACT: no more than kLoraSub steps are added inside the tensor core.  TEST: short waits, and the first copy of block 0 is never made.
template <int TILE, bool EXACT, bool TEST>
__global__ void __launch_bounds__(32 * kLoraDownWarps, TILE == 16 ? 4 : 2)
    lora_down_kernel(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_x, const __grid_constant__ CUtensorMap map_run, const b200q_lora_args a, const LoraPlan p, const LoraDownShape d) {
  extern __shared__ uint8_t s_raw[];
  uint8_t* const s_ring = s_raw + (0u - ptx::smem_u32(s_raw) & 1023u);
  __shared__ __align__(8) uint64_t s_bars[2 * kLoraMostStages + 5];
  __shared__ uint32_t s_tmem;
  __shared__ int s_abort;
  __shared__ __align__(16) LoraFew s_few;
  constexpr int kTmem = 2 * TILE < 32 ? 32 : 2 * TILE;
  constexpr uint32_t kLimit = TEST ? kLoraTestPolls : ptx::kWaitLimit;
  const int tid = threadIdx.x, lane = tid & 31, warp = ptx::uniform_warp_index();
  const uint32_t ring = ptx::smem_u32(s_ring), bar_full = ptx::smem_u32(s_bars), bar_empty = bar_full + 8 * kLoraMostStages;
  const uint32_t bar_done = bar_empty + 8 * kLoraMostStages, bar_free = bar_done + 16, bar_last = bar_free + 16;
  if (tid == 0) {
    for (int i = 0; i < d.stages; ++i) {
      ptx::mbar_init(bar_full + 8 * i, 1);
      ptx::mbar_init(bar_empty + 8 * i, 1);
    }
    for (int i = 0; i < 2; ++i) {
      ptx::mbar_init(bar_done + 8 * i, 1);
      ptx::mbar_init(bar_free + 8 * i, 4);
    }
    ptx::mbar_init(bar_last, 1);
    s_abort = 0;
    ptx::fence_barrier_init();
    ptx::tma_prefetch_desc(&map_a);
    ptx::tma_prefetch_desc(&map_x);
    if (TILE > 16) ptx::tma_prefetch_desc(&map_run);
  }
  if (warp == 1) {
    ptx::tmem_alloc(ptx::smem_u32(&s_tmem), kTmem);
    ptx::tmem_relinquish();
  }
  ptx::tc_fence_before();
  __syncthreads();
  ptx::tc_fence_after();
  const uint32_t tmem = s_tmem;
  pdl_enter();
  const LoraView view = lora_view<TILE>(a, p, s_few);
  const int blocks = ((int)a.rank + 127) / 128, splits = lora_parts(p, view.tiles_used * blocks), part_steps = (p.steps + splits - 1) / splits;
  const int items = view.tiles_used * splits * blocks;
  bool ok = true;
  // item: block of ranks, part of k, tile
  struct Item {
    int block, k0, k1, part;
    LoraTile tile;
  };
  auto item_of = [&](int i) {
    Item it;
    it.block = blocks == 1 ? 0 : i & 1;  // (at most two)
    const int rest = blocks == 1 ? i : i >> 1;
    const int tile = rest / splits;
    it.part = rest - tile * splits;
    it.k0 = it.part * part_steps;
    it.k1 = min(it.k0 + part_steps, p.steps);
    it.tile = view.tile(tile);
    return it;
  };
  if (warp == 0) {
    uint32_t stage = 0, phase = 0;
    int made = 0;
    for (int i = blockIdx.x; i < items && ok; i += gridDim.x) {
      const Item it = item_of(i);
      const int eights = (it.tile.count + 7) / 8;
      int rows[4] = {};
      if (lane < 2 * eights) {
#pragma unroll
        for (int r = 0; r < 4; ++r) rows[r] = view.sorted[it.tile.first + min(4 * lane + r, it.tile.count - 1)];
      }
      // Tokens that follow one another, as those of a prompt do, come as one box: 32 gathers of four rows each take a microsecond.
      bool run = TILE > 16 && it.tile.count > TILE / 2;
      const int first = __shfl_sync(0xFFFFFFFFu, rows[0], 0);
#pragma unroll
      for (int r = 0; r < 4; ++r) run = run && (4 * lane + r >= it.tile.count || rows[r] == first + 4 * lane + r);
      run = __all_sync(0xFFFFFFFFu, run);
      for (int k = it.k0; k < it.k1; ++k) {
        ok = ptx::mbar_wait_uniform(bar_empty + 8 * stage, phase ^ 1, &s_abort, p.status, kLoraErrCopy, kLimit);
        if (!ok) break;
        const uint32_t bar = bar_full + 8 * stage, dst = ring + stage * d.stage;
        if (ptx::elect_one()) {
          ptx::mbar_arrive_expect_tx(bar, d.row_bytes + (run ? TILE * 128 : eights * 1024));
          if (!(TEST && blockIdx.x == 0 && made == 0)) ptx::tma_load_3d(dst, &map_a, bar, 64 * k, 128 * it.block, it.tile.adapter);
          if (run) ptx::tma_load_2d(dst + d.row_bytes, &map_run, bar, 64 * k, first);  // (rows behind the tile's are columns that nobody looks at)
        }
        __syncwarp();
        if (!run && lane < 2 * eights) layer_gather4(dst + d.row_bytes + 512 * lane, &map_x, bar, 64 * k, rows);
        __syncwarp();
        ++made;
        if (++stage == (uint32_t)d.stages) {
          stage = 0;
          phase ^= 1;
        }
      }
    }
    lora_drain(bar_full, d.stages, made, stage, phase);
  } else if (warp == 1) {
    uint32_t stage = 0, phase = 0;
    int n = 0;
    const uint64_t a0 = ptx::smem_desc_k_sw128(ring), b0 = ptx::smem_desc_k_sw128(ring + d.row_bytes);
    for (int i = blockIdx.x; i < items && ok; i += gridDim.x) {
      const Item it = item_of(i);
      if (it.k0 >= it.k1) continue;
      const uint32_t idesc = ptx::umma_idesc(1, 1, 128, lora_columns(it.tile.count));
      uint32_t acc = 0, out = 0;
      for (int k = it.k0, sub = 0; k < it.k1; ++k) {
        if (sub == 0) {
          acc = n & 1;
          out = tmem + acc * TILE;
          ok = ptx::mbar_wait_uniform(bar_free + 8 * acc, ((n >> 1) & 1) ^ 1, &s_abort, p.status, kLoraErrMma, kLimit);
          if (!ok) break;
          ++n;
          ptx::tc_fence_after();
        }
        ok = ptx::mbar_wait_uniform(bar_full + 8 * stage, phase, &s_abort, p.status, kLoraErrMma, kLimit);
        if (!ok) break;
        ptx::tc_fence_after();
        if (ptx::elect_one()) {
          const uint64_t off = stage * (uint32_t)(d.stage >> 4);
          ptx::umma_f16_x4(out, a0 + off, b0 + off, idesc, sub != 0, 2, 2);
          ptx::umma_commit(bar_empty + 8 * stage);
          if (k + 1 == it.k1 || (EXACT && sub + 1 == kLoraSub)) ptx::umma_commit(bar_done + 8 * acc);
        }
        __syncwarp();
        if (++sub == kLoraSub && EXACT) sub = 0;
        if (++stage == (uint32_t)d.stages) {
          stage = 0;
          phase ^= 1;
        }
      }
    }
    lora_drain_products(bar_last);
  } else {
    // Where a wait has run out, what should be there is NaN: the other kernel would make finite values of whatever lay there.
    int n = 0;
    const int quarter = warp & 3;
    for (int i = blockIdx.x; i < items; i += gridDim.x) {
      const Item it = item_of(i);
      const int r = 128 * it.block + 32 * quarter + lane;
      constexpr int kHeld = (TILE + 31) / 32;
      int held[kHeld];  // a lane has each 32nd token, fetched while the products run
#pragma unroll
      for (int h = 0; h < kHeld; ++h) held[h] = 32 * h + lane < it.tile.count ? view.sorted[it.tile.first + 32 * h + lane] : 0;
      // (a part behind the end of k: zeros)
      for (int k = it.k0; k == it.k0 || (EXACT && k < it.k1); k += kLoraSub) {
        bool none = it.k0 >= it.k1;
        const uint32_t acc = n & 1, in = tmem + acc * TILE + ((uint32_t)(32 * quarter) << 16);
        if (!none) {
          ok = ok && ptx::mbar_wait_uniform(bar_done + 8 * acc, (n >> 1) & 1, &s_abort, p.status, kLoraErrResults, kLimit);
          none = !ok;
          ++n;
          ptx::tc_fence_after();
        }
        const float nothing = ok ? 0.f : __int_as_float(0x7FC00000);
#pragma unroll
        for (int h = 0; h < kHeld; ++h)
          for (int j0 = 32 * h; j0 < min(it.tile.count, 32 * h + 32); j0 += 8) {
            float v[8] = {nothing, nothing, nothing, nothing, nothing, nothing, nothing, nothing};
            if (!none) {
              layer_tmem_ld8(in + j0, v);
              ptx::tmem_ld_wait();
            }
            float* to[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) to[j] = p.low + ((int64_t)it.part * a.tokens + __shfl_sync(0xFFFFFFFFu, held[h], j0 + j - 32 * h)) * a.rank + r;
            if (EXACT && k > it.k0) {  // (a thread's own sums)
              float before[8];
#pragma unroll
              for (int j = 0; j < 8; ++j) before[j] = r < a.rank && j0 + j < it.tile.count ? *to[j] : 0.f;
#pragma unroll
              for (int j = 0; j < 8; ++j) v[j] += before[j];
            }
#pragma unroll
            for (int j = 0; j < 8; ++j)
              if (j0 + j < it.tile.count && r < a.rank) *to[j] = v[j];
          }
        if (!none) {
          ptx::tc_fence_before();
          __syncwarp();
          if (lane == 0) ptx::mbar_arrive(bar_free + 8 * acc);
        }
      }
    }
  }
  ptx::tc_fence_before();
  __syncthreads();
  if (warp == 1) ptx::tmem_dealloc(tmem, kTmem);
}

// y += b (scale a x): columns of y are the rows of the product, tokens its columns.  A tile's terms of a x lie in shared memory and meet one block of 128 columns
// after the other.  A warp has 32 columns and half of the tokens; it turns its results around in shared memory, eight tokens at a time, so that a lane has 16 bytes of
// a row of y, and has always asked for the next block's.  (A column and two bytes per lane, 16 of them asked for at a time, was 150 us where this is 45: 4096 tokens of
// 14336 columns.)
constexpr int lora_result_warps(int tile) { return tile == 16 ? 4 : 8; }
constexpr int lora_up_threads(int tile) { return 64 + 32 * lora_result_warps(tile); }  // copies, MMAs, results
constexpr int lora_up_ctas(int wide, int tile) { return tile == 16 ? (wide ? 3 : 4) : wide ? 1 : 2; }  // of an SM, as many as the registers are enough for
struct LoraUpShape {
  int chunks, terms_bytes, stages;  // chunks of 64 ranks; bytes of the terms
};

// 16 bytes of a row, at once or (rows between boundaries) value by value; PAST: past L1, which the kernels before may have left older than y
template <bool WHOLE, bool PAST, typename Y>
__device__ __forceinline__ uint4 lora_load16(const Y* p) {
  auto load = [](const auto* q) {
    if constexpr (PAST) return __ldcg(q);
    else return *q;
  };
  if constexpr (WHOLE) {
    return load(reinterpret_cast<const uint4*>(p));
  } else if constexpr (sizeof(Y) == 4) {
    const unsigned* u = reinterpret_cast<const unsigned*>(p);
    return make_uint4(load(u), load(u + 1), load(u + 2), load(u + 3));
  } else {
    const unsigned short* u = reinterpret_cast<const unsigned short*>(p);
    auto two = [&](int i) { return (uint32_t)load(u + 2 * i) | (uint32_t)load(u + 2 * i + 1) << 16; };
    return make_uint4(two(0), two(1), two(2), two(3));
  }
}
template <bool WHOLE, typename Y>
__device__ __forceinline__ void lora_store16(Y* p, const uint4& w) {
  const uint32_t v[4] = {w.x, w.y, w.z, w.w};
  if constexpr (WHOLE) {
    *reinterpret_cast<uint4*>(p) = w;
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (sizeof(Y) == 4) {
        p[i] = __uint_as_float(v[i]);
      } else {
        reinterpret_cast<uint16_t*>(p)[2 * i] = (uint16_t)v[i];
        reinterpret_cast<uint16_t*>(p)[2 * i + 1] = (uint16_t)(v[i] >> 16);
      }
    }
  }
}

// All terms but the last stay finite, so that the rest of an infinity is that infinity (and of a NaN a NaN), not inf - inf, and what lies between the ends of bf16 and fp32 has a rest.
__device__ __forceinline__ float lora_within_bf16(float v) { return fminf(fmaxf(v, -3.3895313892515355e38f), 3.3895313892515355e38f); }

template <typename Y, int TILE, bool WHOLE, bool TEST>  // TEST: short waits, and the first copy of block 0 is never made
__global__ void __launch_bounds__(lora_up_threads(TILE), lora_up_ctas(sizeof(Y) == 4, TILE)) lora_up_kernel(const __grid_constant__ CUtensorMap map_b, const b200q_lora_args a, const LoraPlan p, const LoraUpShape d) {
  constexpr int kTerms = sizeof(Y) == 4 ? 3 : 2, kStage = 128 * 128, kWarps = lora_result_warps(TILE), kHalf = TILE / (kWarps / 4);
  constexpr int kPer = 16 / sizeof(Y), kLanes = 32 / kPer, kRows = 32 / kLanes, kPieces = kHalf / kRows;  // values of a lane's piece of a row; lanes of a row
  constexpr int kBatch = kHalf < 16 ? kHalf : 16, kPitch = 36;  // tokens turned around together; floats of a token's 32 results
  extern __shared__ uint8_t s_raw[];
  uint8_t* const s_terms = s_raw + (0u - ptx::smem_u32(s_raw) & 1023u);  // [terms][chunks][tokens][128 bytes], then the ring
  __shared__ __align__(8) uint64_t s_bars[2 * kLoraMostStages + 7];
  __shared__ uint32_t s_tmem;
  __shared__ __align__(16) float s_turn[kWarps][kBatch * kPitch];
  __shared__ int s_abort;
  __shared__ __align__(16) LoraFew s_few;
  constexpr int kTmem = 2 * TILE < 32 ? 32 : 2 * TILE;
  constexpr uint32_t kLimit = TEST ? kLoraTestPolls : ptx::kWaitLimit;
  const int tid = threadIdx.x, lane = tid & 31, warp = ptx::uniform_warp_index();
  const uint32_t terms = ptx::smem_u32(s_terms), ring = terms + d.terms_bytes;
  const uint32_t bar_full = ptx::smem_u32(s_bars), bar_empty = bar_full + 8 * kLoraMostStages, bar_done = bar_empty + 8 * kLoraMostStages, bar_free = bar_done + 16;
  const uint32_t bar_terms = bar_free + 16, bar_used = bar_terms + 8, bar_last = bar_used + 8;
  if (tid == 0) {
    for (int i = 0; i < d.stages; ++i) {
      ptx::mbar_init(bar_full + 8 * i, 1);
      ptx::mbar_init(bar_empty + 8 * i, 1);
    }
    for (int i = 0; i < 2; ++i) {
      ptx::mbar_init(bar_done + 8 * i, 1);
      ptx::mbar_init(bar_free + 8 * i, kWarps);
    }
    ptx::mbar_init(bar_terms, kWarps);
    ptx::mbar_init(bar_used, 1);
    ptx::mbar_init(bar_last, 1);
    s_abort = 0;
    ptx::fence_barrier_init();
    ptx::tma_prefetch_desc(&map_b);
  }
  if (warp == 1) {
    ptx::tmem_alloc(ptx::smem_u32(&s_tmem), kTmem);
    ptx::tmem_relinquish();
  }
  ptx::tc_fence_before();
  __syncthreads();
  ptx::tc_fence_after();
  const uint32_t tmem = s_tmem;
  // The kernel in front (a x) was waiting for all before it when it let this one begin, so that all but its own results may be read: the plan, b, and y.  Only the
  // warps of the results wait for it, behind their first loads of y.
  constexpr bool kEarly = TILE == 16;
  if (!kEarly) pdl_enter();
  const LoraView view = lora_view<TILE>(a, p, s_few);
  // parts of n (every `parts`-th block of 128 columns): as many as leave no CTA a second item.  (Found by the host from the most tiles that there may be, they left every fourth
  // CTA without one where 8 adapters have 512 tokens each: 91 us, now 81 to 89.)
  const int n_blocks = (int)((a.n + 127) / 128), parts = max(1, min(n_blocks, (int)gridDim.x / max(view.tiles_used, 1))), items = view.tiles_used * parts;
  bool ok = true;
  if (warp == 0) {
    uint32_t stage = 0, phase = 0;
    int made = 0;
    for (int i = blockIdx.x; i < items && ok; i += gridDim.x) {
      const int tile = i / parts, part = i - tile * parts, adapter = view.tile(tile).adapter;
      for (int n = part; n < n_blocks && ok; n += parts)
        for (int c = 0; c < d.chunks; ++c) {
          ok = ptx::mbar_wait_uniform(bar_empty + 8 * stage, phase ^ 1, &s_abort, p.status, kLoraErrCopy, kLimit);
          if (!ok) break;
          if (ptx::elect_one()) {
            ptx::mbar_arrive_expect_tx(bar_full + 8 * stage, kStage);
            if (!(TEST && blockIdx.x == 0 && made == 0)) ptx::tma_load_3d(ring + stage * kStage, &map_b, bar_full + 8 * stage, 64 * c, 128 * n, adapter);
          }
          __syncwarp();
          ++made;
          if (++stage == (uint32_t)d.stages) {
            stage = 0;
            phase ^= 1;
          }
        }
    }
    lora_drain(bar_full, d.stages, made, stage, phase);
  } else if (warp == 1) {
    uint32_t stage = 0, phase = 0;
    int done = 0, item = 0;
    const uint64_t a0 = ptx::smem_desc_k_sw128(ring), b0 = ptx::smem_desc_k_sw128(terms);
    for (int i = blockIdx.x; i < items && ok; i += gridDim.x, ++item) {
      const int tile = i / parts, part = i - tile * parts;
      const uint32_t idesc = ptx::umma_idesc(1, 1, 128, lora_columns(view.tile(tile).count));
      ok = ptx::mbar_wait_uniform(bar_terms, item & 1, &s_abort, p.status, kLoraErrMma, kLimit);
      for (int n = part; n < n_blocks && ok; n += parts, ++done) {
        const uint32_t acc = done & 1, out = tmem + acc * TILE;
        ok = ptx::mbar_wait_uniform(bar_free + 8 * acc, ((done >> 1) & 1) ^ 1, &s_abort, p.status, kLoraErrMma, kLimit);
        if (!ok) break;
        ptx::tc_fence_after();
        for (int c = 0; c < d.chunks; ++c) {
          ok = ptx::mbar_wait_uniform(bar_full + 8 * stage, phase, &s_abort, p.status, kLoraErrMma, kLimit);
          if (!ok) break;
          ptx::tc_fence_after();
          if (ptx::elect_one()) {
            for (int e = kTerms - 1; e >= 0; --e)  // (the small ones first)
              ptx::umma_f16_x4(out, a0 + stage * (uint32_t)(kStage >> 4), b0 + (e * d.chunks + c) * (TILE * 128 >> 4), idesc, c > 0 || e < kTerms - 1, 2, 2);
            ptx::umma_commit(bar_empty + 8 * stage);
            if (c + 1 == d.chunks) ptx::umma_commit(bar_done + 8 * acc);
          }
          __syncwarp();
          if (++stage == (uint32_t)d.stages) {
            stage = 0;
            phase ^= 1;
          }
        }
      }
      if (ok && ptx::elect_one()) ptx::umma_commit(bar_used);
      __syncwarp();
    }
    lora_drain_products(bar_last);
  } else {
    int done = 0, item = 0;
    const int wt = tid - 64, quarter = warp & 3, half = (warp - 2) >> 2, my_row = lane / kLanes, my_column = 32 * quarter + lane % kLanes * kPer;
    float* const turn = s_turn[warp - 2];
    for (int i = blockIdx.x; i < items; i += gridDim.x, ++item) {  // (all its warps come to each item's barrier, whatever became of their waits)
      const int index = i / parts, part = i - index * parts;
      const LoraTile tile = view.tile(index);
      const int first = tile.first + kHalf * half, count = min(tile.count - kHalf * half, kHalf);  // of this half
      int token[kPieces];  // of a lane's pieces; -1 behind the last one
      uint4 old[kPieces];
      Y* const columns = static_cast<Y*>(a.y) + my_column;
      auto ask = [&](int c, int n) {
        if (token[c] >= 0 && 128 * n + my_column < a.n) old[c] = lora_load16<WHOLE, kEarly>(columns + token[c] * a.y_stride + 128 * n);
      };
#pragma unroll
      for (int c = 0; c < kPieces; ++c) token[c] = c * kRows + my_row < count ? view.token(first + c * kRows + my_row) : -1;
      if constexpr (kEarly) {
#pragma unroll
        for (int c = 0; c < kPieces; ++c) ask(c, part);
        if (item == 0) pdl_enter();
      }
      ok = ok && ptx::mbar_wait_uniform(bar_used, (item & 1) ^ 1, &s_abort, p.status, kLoraErrResults, kLimit);  // (the products with the terms before are done)
      const float scale = a.scales ? a.scales[tile.adapter] : 1.f;
      // The terms: a thread has four ranks of a token or two at a time, eight parts of k at once.  (Eight ranks of a token, two parts at once: twice the sectors, 89 us for
      // 4096 tokens where this is 86; what spills, four tokens and two parts for instance, 110.)
      const int pieces = 16 * d.chunks, total = tile.count * pieces;  // of four ranks
      const int splits = lora_parts(p, view.tiles_used * ((d.chunks + 1) / 2));
      constexpr int kSets = TILE == 16 ? 1 : 2, kTogether = 8;
      for (int q0 = wt; ok && q0 < total; q0 += 32 * kWarps * kSets) {
        const float* low[kSets];
        float v[kSets][4] = {};
#pragma unroll
        for (int e = 0; e < kSets; ++e) {
          const int q = q0 + 32 * kWarps * e, j = q / pieces, r = 4 * (q - j * pieces);
          low[e] = q < total && r < a.rank ? p.low + (int64_t)view.sorted[tile.first + j] * a.rank + r : nullptr;
        }
        const int64_t step = a.tokens * a.rank;
        for (int s0 = 0; s0 < splits; s0 += kTogether) {
          float4 x[kSets][kTogether];
#pragma unroll
          for (int s = 0; s < kTogether; ++s)
#pragma unroll
            for (int e = 0; e < kSets; ++e)
              x[e][s] = low[e] && s0 + s < splits ? __ldcg(reinterpret_cast<const float4*>(low[e] + (s0 + s) * step)) : make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
          for (int s = 0; s < kTogether; ++s)
#pragma unroll
            for (int e = 0; e < kSets; ++e) {
              v[e][0] += x[e][s].x; v[e][1] += x[e][s].y; v[e][2] += x[e][s].z; v[e][3] += x[e][s].w;
            }
        }
#pragma unroll
        for (int e = 0; e < kSets; ++e) {
          const int q = q0 + 32 * kWarps * e, j = q / pieces, r = 4 * (q - j * pieces);
          if (q >= total) break;
#pragma unroll
          for (int c = 0; c < 4; ++c) v[e][c] *= scale;
#pragma unroll
          for (int t = 0; t < kTerms; ++t) {
            uint32_t w[2];
#pragma unroll
            for (int c = 0; c < 2; ++c) {
              w[c] = t + 1 < kTerms ? pack_bf16x2(lora_within_bf16(v[e][2 * c]), lora_within_bf16(v[e][2 * c + 1])) : pack_bf16x2(v[e][2 * c], v[e][2 * c + 1]);
              v[e][2 * c] -= __uint_as_float(w[c] << 16);
              v[e][2 * c + 1] -= __uint_as_float(w[c] & 0xFFFF0000u);
            }
            *reinterpret_cast<uint2*>(s_terms + ((t * d.chunks + r / 64) * TILE + j) * 128 + (((r / 8 & 7) ^ (j & 7)) << 4) + 2 * (r & 4)) = make_uint2(w[0], w[1]);
          }
        }
      }
      if constexpr (!kEarly) {  // (here, because the registers are wanted for the terms before)
#pragma unroll
        for (int c = 0; c < kPieces; ++c) ask(c, part);
      }
      ptx::fence_proxy_async_smem();
      ok = layer_bar_and(1, 32 * kWarps, ok);
      if (!ok) break;
      if (lane == 0) ptx::mbar_arrive(bar_terms);
      for (int n = part; n < n_blocks && ok; n += parts, ++done) {
        const uint32_t acc = done & 1, in = tmem + acc * TILE + kHalf * half + ((uint32_t)(32 * quarter) << 16);
        ok = ptx::mbar_wait_uniform(bar_done + 8 * acc, (done >> 1) & 1, &s_abort, p.status, kLoraErrResults, kLimit);
        if (!ok) break;
        ptx::tc_fence_after();
        const bool there = 128 * n + my_column < a.n;
#pragma unroll
        for (int j0 = 0; j0 < kHalf; j0 += kBatch) {
          if (j0 >= count) break;
          float v[kBatch / 8][8];
#pragma unroll
          for (int h = 0; h < kBatch / 8; ++h)
            if (j0 + 8 * h < count) layer_tmem_ld8(in + j0 + 8 * h, v[h]);
          ptx::tmem_ld_wait();
          __syncwarp();
#pragma unroll
          for (int h = 0; h < kBatch / 8; ++h)
            if (j0 + 8 * h < count) {
#pragma unroll
              for (int j = 0; j < 8; ++j) turn[(8 * h + j) * kPitch + lane] = v[h][j];
            }
          __syncwarp();
#pragma unroll
          for (int c = j0 / kRows; c < (j0 + kBatch) / kRows; ++c) {
            const float4* from = reinterpret_cast<const float4*>(turn + (c * kRows - j0 + my_row) * kPitch + lane % kLanes * kPer);
            uint4 w;
            const float4 x = from[0];
            if constexpr (sizeof(Y) == 4) {
              w = make_uint4(__float_as_uint(__uint_as_float(old[c].x) + x.x), __float_as_uint(__uint_as_float(old[c].y) + x.y),
                             __float_as_uint(__uint_as_float(old[c].z) + x.z), __float_as_uint(__uint_as_float(old[c].w) + x.w));
            } else {
              const float4 z = from[1];
              w.x = pack_bf16x2(__uint_as_float(old[c].x << 16) + x.x, __uint_as_float(old[c].x & 0xFFFF0000u) + x.y);
              w.y = pack_bf16x2(__uint_as_float(old[c].y << 16) + x.z, __uint_as_float(old[c].y & 0xFFFF0000u) + x.w);
              w.z = pack_bf16x2(__uint_as_float(old[c].z << 16) + z.x, __uint_as_float(old[c].z & 0xFFFF0000u) + z.y);
              w.w = pack_bf16x2(__uint_as_float(old[c].w << 16) + z.z, __uint_as_float(old[c].w & 0xFFFF0000u) + z.w);
            }
            if (there && token[c] >= 0) lora_store16<WHOLE>(columns + token[c] * a.y_stride + 128 * n, w);
            ask(c, n + parts);
          }
        }
        ptx::tc_fence_before();
        __syncwarp();
        if (lane == 0) ptx::mbar_arrive(bar_free + 8 * acc);
      }
    }
    if (kEarly && blockIdx.x >= items) pdl_enter();  // (no kernel is done before those in front of it)
  }
  ptx::tc_fence_before();
  __syncthreads();
  if (warp == 1) ptx::tmem_dealloc(tmem, kTmem);
}

// ---------------------------------------------------------------------------- host
size_t lora_workspace_bytes_impl(int64_t tokens, int64_t k, int64_t n, int64_t rank, int64_t adapters) {
  (void)n;
  size_t bytes = 0;
  for (int tile : {16, 128})  // (which one depends on y's type)
    for (int64_t t : {tokens, tokens % kLoraChunk}) {  // (the last tokens of a long call may be cut into more parts of k than those before)
      const size_t b = t ? LoraSpace(t, rank, lora_splits(t, k, rank, adapters, tile)).bytes : 0;
      if (b > bytes) bytes = b;
    }
  return bytes;
}

static bool lora_fits_tensor_cores(const b200q_lora_args& a) {
  if (a.force_plain || a.rank % 8 || a.k % 8 || a.n % 8) return false;
  if (a.k > 1 << 30 || a.n > 1 << 30) return false;  // (columns are counted in 32 bits, and past the last one)
  if (a.tokens > 1 && (a.x_stride % 8 || a.x_stride < a.k)) return false;
  if (a.adapters > 1 && (a.a_stride % 8 || a.b_stride % 8 || a.a_stride <= 0 || a.b_stride <= 0)) return false;
  if ((a.rank > 1 && (a.a_row_stride % 8 || a.a_row_stride < a.k)) || (a.n > 1 && (a.b_row_stride % 8 || a.b_row_stride < a.rank))) return false;
  for (const void* p : {a.x, a.a, a.b})
    if (reinterpret_cast<uintptr_t>(p) % 16) return false;
  return true;
}

// bf16 [planes][rows][depth] in boxes of 64 values of `box` rows
static int lora_map(CUtensorMap* map, const void* base, int64_t depth, int64_t rows, int64_t planes, int64_t row_stride, int64_t plane_stride, int box_rows, int rank) {
  EncodeTiledFn enc = get_encode_fn();
  if (!enc) return B200Q_ERR_CUDA;
  const cuuint64_t dims[3] = {(cuuint64_t)depth, (cuuint64_t)rows, (cuuint64_t)planes};
  const cuuint64_t strides[2] = {(cuuint64_t)(rows > 1 ? row_stride : (depth + 7) / 8 * 8) * 2, (cuuint64_t)(planes > 1 ? plane_stride : (depth + 7) / 8 * 8) * 2};
  const cuuint32_t box[3] = {64, (cuuint32_t)box_rows, 1}, step[3] = {1, 1, 1};
  const CUresult r = enc(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, (cuuint32_t)rank, const_cast<void*>(base), dims, strides, box, step, CU_TENSOR_MAP_INTERLEAVE_NONE,
                         CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return r == CUDA_SUCCESS ? B200Q_OK : B200Q_ERR_UNSUPPORTED;
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

constexpr int kLoraShared = 100 * 1024;  // of a CTA where two share an SM, beside what its kernel has of its own

template <int TILE, bool EXACT, bool TEST = false>
static int lora_launch_down(const b200q_lora_args& a, const LoraPlan& p, int64_t tiles, cudaStream_t st) {
  static std::atomic<int> done[kMaxDevices];
  if (int rc = lora_ready(reinterpret_cast<const void*>(lora_down_kernel<TILE, EXACT, TEST>), done, kLoraShared)) return rc;
  const int ctas = lora_down_ctas(a.rank, TILE);
  const LoraDownShape d((int)a.rank, TILE, (ctas == 2 ? kLoraShared : 220 * 1024 / ctas - 4096) - 1024);
  CUtensorMap map_a, map_x, map_run;
  if (int rc = lora_map(&map_a, a.a, a.k, a.rank, a.adapters, a.a_row_stride, a.a_stride, d.rows, 3)) return rc;
  if (int rc = lora_map(&map_x, a.x, a.k, a.tokens, 1, a.x_stride, 0, 1, 2)) return rc;
  if (int rc = lora_map(&map_run, a.x, a.k, a.tokens, 1, a.x_stride, 0, TILE, 2)) return rc;
  const int64_t items = tiles * p.splits * ((a.rank + 127) / 128), most = p.slots;
  // (the rows behind a block's ranks, which the product reads too and whose results nobody looks at, are within the allocation)
  launch_dependent(lora_down_kernel<TILE, EXACT, TEST>, dim3((unsigned)(items < most ? items : most)), dim3(32 * kLoraDownWarps), (size_t)d.stages * d.stage + 16384 + 1024, st, map_a, map_x,
                   map_run, a, p, d);
  B200Q_LAUNCH_CHECK();
  return B200Q_OK;
}
template <typename Y, int TILE, bool WHOLE, bool TEST = false>
static int lora_launch_up(const b200q_lora_args& a, const LoraPlan& p, int64_t tiles, cudaStream_t st) {
  constexpr int kTerms = sizeof(Y) == 4 ? 3 : 2, kMost = 200 * 1024;
  static std::atomic<int> done[kMaxDevices];
  if (int rc = lora_ready(reinterpret_cast<const void*>(lora_up_kernel<Y, TILE, WHOLE, TEST>), done, kMost)) return rc;
  CUtensorMap map_b;
  if (int rc = lora_map(&map_b, a.b, a.rank, a.n, a.adapters, a.b_row_stride, a.b_stride, 128, 3)) return rc;
  LoraUpShape d;
  d.chunks = (int)((a.rank + 63) / 64);
  d.terms_bytes = kTerms * d.chunks * TILE * 128;
  // as many stages as leave room for the SM's other CTAs, if that is two; else as many as there is room for
  constexpr int kCtas = lora_up_ctas(sizeof(Y) == 4, TILE), kHere = 4 * lora_result_warps(TILE) * 16 * 36 + (int)sizeof(LoraFew) + 512;  // (static memory)
  constexpr int kOne = (226 * 1024 / kCtas - 1024 - kHere) / 1024 * 1024, kShare = kOne < kMost ? kOne : kMost;
  const int room = (d.terms_bytes + 2 * 16384 + 1024 <= kShare ? kShare : kMost) - 1024 - d.terms_bytes;
  d.stages = room / 16384 < kLoraMostStages ? room / 16384 : kLoraMostStages;
  const int64_t items = tiles * ((a.n + 127) / 128), most = kCtas * kNumSMs;
  launch_dependent(lora_up_kernel<Y, TILE, WHOLE, TEST>, dim3((unsigned)(items < most ? items : most)), dim3(lora_up_threads(TILE)), (size_t)d.terms_bytes + d.stages * 16384 + 1024, st, map_b, a, p,
                   d);
  B200Q_LAUNCH_CHECK();
  return B200Q_OK;
}

static bool lora_y_whole(const b200q_lora_args& a) {  // rows of y on boundaries of 16 bytes
  return reinterpret_cast<uintptr_t>(a.y) % 16 == 0 && (a.tokens == 1 || a.y_stride * (a.y_dtype == B200Q_F32 ? 4 : 2) % 16 == 0);
}
template <typename Y>
static int lora_launch_up_tile(const b200q_lora_args& a, const LoraPlan& p, int64_t tiles, cudaStream_t st) {
  const bool whole = lora_y_whole(a);
  if (p.tile == 16) return whole ? lora_launch_up<Y, 16, true>(a, p, tiles, st) : lora_launch_up<Y, 16, false>(a, p, tiles, st);
  return whole ? lora_launch_up<Y, 128, true>(a, p, tiles, st) : lora_launch_up<Y, 128, false>(a, p, tiles, st);
}

enum LoraLost { kLoraLostNothing = -1, kLoraLostA, kLoraLostB, kLoraLostCount };  // what a self-test waits for in vain: the first copy of a, or of b, of block 0

static int lora_chunk_fast(const b200q_lora_args& a, cudaStream_t st, int lost = kLoraLostNothing) {
  const int tile = lora_tile_tokens(a.tokens, a.k, a.n, a.rank, a.adapters, a.y_dtype == B200Q_F32);
  const int64_t splits = lora_splits(a.tokens, a.k, a.rank, a.adapters, tile), tiles = lora_most_tiles(a.tokens, a.adapters, tile);
  const LoraSpace space(a.tokens, a.rank, splits);
  uint8_t* w = static_cast<uint8_t*>(a.workspace);
  LoraPlan p;
  p.tiles_used = reinterpret_cast<int*>(w);
  p.tiles = reinterpret_cast<LoraTile*>(w + space.tiles);
  p.sorted = reinterpret_cast<int*>(w + space.sorted);
  p.low = reinterpret_cast<float*>(w + space.low);
  p.splits = (int)splits;
  p.steps = (int)((a.k + 63) / 64);
  p.slots = lora_down_ctas(a.rank, tile) * kNumSMs;
  p.tile = tile;
  p.status = device_status_ptr();
  if (!p.status) return B200Q_ERR_CUDA;
  if (a.tokens <= kLoraFew) {
    p.tiles_used = nullptr;
  } else {
    static std::atomic<int> done[kMaxDevices];
    constexpr int kMost = (int)sizeof(uint16_t) * (kLoraSortThreads / 32 + 1) * (int)kLoraMaxAdapters;
    if (int rc = lora_ready(reinterpret_cast<const void*>(lora_sort_kernel), done, kMost)) return rc;
    launch_dependent(lora_sort_kernel, dim3(1), dim3(kLoraSortThreads), sizeof(uint16_t) * (kLoraSortThreads / 32 + 1) * (size_t)a.adapters, st, a, p);
    B200Q_LAUNCH_CHECK();
  }
  if (lost != kLoraLostNothing) {  // (tiles of 16 tokens, y in bf16 and on boundaries of 16 bytes)
    if (int rc = lost == kLoraLostA ? lora_launch_down<16, false, true>(a, p, tiles, st) : lora_launch_down<16, false>(a, p, tiles, st)) return rc;
    return lost == kLoraLostB ? lora_launch_up<__nv_bfloat16, 16, true, true>(a, p, tiles, st) : lora_launch_up<__nv_bfloat16, 16, true>(a, p, tiles, st);
  }
  int rc;
  if (a.y_dtype == B200Q_F32) rc = tile == 16 ? lora_launch_down<16, true>(a, p, tiles, st) : lora_launch_down<128, true>(a, p, tiles, st);
  else rc = tile == 16 ? lora_launch_down<16, false>(a, p, tiles, st) : lora_launch_down<128, false>(a, p, tiles, st);
  if (rc) return rc;
  return a.y_dtype == B200Q_F32 ? lora_launch_up_tile<float>(a, p, tiles, st) : lora_launch_up_tile<__nv_bfloat16>(a, p, tiles, st);
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

static bool lora_has_workspace(const b200q_lora_args& a) {
  return a.workspace && a.workspace_bytes >= lora_workspace_bytes_impl(a.tokens, a.k, a.n, a.rank, a.adapters) && reinterpret_cast<uintptr_t>(a.workspace) % 16 == 0;
}

int lora_add_impl(const b200q_lora_args& a, cudaStream_t st) {
  if (!lora_has_workspace(a)) return B200Q_ERR_BAD_ARGUMENT;
  for (int64_t t = 0; t < a.tokens; t += kLoraChunk) {
    b200q_lora_args c = a;
    c.tokens = a.tokens - t < kLoraChunk ? a.tokens - t : kLoraChunk;
    c.x = static_cast<const uint8_t*>(a.x) + 2 * t * a.x_stride;
    c.y = static_cast<uint8_t*>(a.y) + (a.y_dtype == B200Q_F32 ? 4 : 2) * t * a.y_stride;
    c.adapter = a.adapter + t;
    int rc = lora_fits_tensor_cores(a) ? lora_chunk_fast(c, st) : B200Q_ERR_UNSUPPORTED;
    if (rc == B200Q_ERR_UNSUPPORTED) rc = lora_chunk_plain(c, st);  // (or a layout that has no tensor map)
    if (rc) return rc;
  }
  return B200Q_OK;
}

int lora_selftest_impl(const b200q_lora_args& a, int lost, cudaStream_t st) {
  if (lost < 0 || lost >= kLoraLostCount || !lora_has_workspace(a)) return B200Q_ERR_BAD_ARGUMENT;
  if (!lora_fits_tensor_cores(a) || a.y_dtype != B200Q_BF16 || !lora_y_whole(a) || a.tokens > kLoraChunk || lora_tile_tokens(a.tokens, a.k, a.n, a.rank, a.adapters, false) != 16)
    return B200Q_ERR_UNSUPPORTED;
  return lora_chunk_fast(a, st, lost);
}

}  // namespace b200q
