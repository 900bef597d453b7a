// What stands around the FP8 products of a decoder layer: the entry points of norm.cu, lora.cu and moe.cu, called by the C ABI wrappers
// once their arguments are checked.
#pragma once

#include "common.cuh"
#include "tcgen05_ptx.cuh"

namespace b200q {

constexpr int64_t kLoraMaxRank = 256, kLoraMaxAdapters = 2048;
constexpr int kMoeMaxExperts = 512, kMoeMaxTopK = 16;

int add_rms_norm_cast_impl(const b200q_norm_args& a, cudaStream_t st);
int norm_selftest_impl(const b200q_norm_args& a, cudaStream_t st);
size_t lora_workspace_bytes_impl(int64_t tokens, int64_t k, int64_t n, int64_t rank, int64_t adapters);
int lora_add_impl(const b200q_lora_args& a, cudaStream_t st);
int lora_selftest_impl(const b200q_lora_args& a, int lost, cudaStream_t st);
size_t moe_workspace_bytes_impl(int64_t tokens, int64_t hidden, int64_t inner, int experts, int top_k);
int moe_layer_impl(const b200q_moe_args& a, cudaStream_t st);
int moe_selftest_impl(const b200q_moe_args& a, int lost, cudaStream_t st);

// A named barrier that tells whether all its threads say yes.  Warps that share a barrier must all come to it, also where the waits of some have run out.
__device__ __forceinline__ bool layer_bar_and(int id, int threads, bool yes) {
  uint32_t all;
  __syncwarp();  // (an aligned barrier wants a warp's threads together, and they may come from a loop that each left when it was done)
  asm volatile(
      "{\n"
      ".reg .pred p, q;\n"
      "setp.ne.u32 p, %3, 0;\n"
      "barrier.cta.red.and.aligned.pred q, %1, %2, p;\n"
      "selp.u32 %0, 1, 0, q;\n"
      "}\n"
      : "=r"(all)
      : "r"(id), "r"(threads), "r"((uint32_t)yes)
      : "memory");
  return all != 0;
}
// four rows of a matrix, 128 bytes of each from column x on
__device__ __forceinline__ void layer_gather4(uint32_t dst, const CUtensorMap* map, uint32_t bar, int x, const int (&rows)[4]) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cluster.global.tile::gather4.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5, %6, %7}], [%2];" ::"r"(dst),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(bar), "r"(x), "r"(rows[0]), "r"(rows[1]), "r"(rows[2]), "r"(rows[3])
      : "memory");
}
__device__ __forceinline__ void layer_tmem_ld8(uint32_t taddr, float (&v)[8]) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
               : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]), "=f"(v[4]), "=f"(v[5]), "=f"(v[6]), "=f"(v[7])
               : "r"(taddr)
               : "memory");
}

}  // namespace b200q
