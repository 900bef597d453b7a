// What stands around the FP8 products of a decoder layer: the entry points of norm.cu, lora.cu and moe.cu, called by the C ABI wrappers
// once their arguments are checked.
#pragma once

#include "common.cuh"

namespace b200q {

constexpr int64_t kLoraMaxRank = 256, kLoraMaxAdapters = 2048;
constexpr int kMoeMaxExperts = 512, kMoeMaxTopK = 16;

int add_rms_norm_cast_impl(const b200q_norm_args& a, cudaStream_t st);
size_t lora_workspace_bytes_impl(int64_t tokens, int64_t k, int64_t n, int64_t rank, int64_t adapters);
int lora_add_impl(const b200q_lora_args& a, cudaStream_t st);
size_t moe_workspace_bytes_impl(int64_t tokens, int64_t hidden, int64_t inner, int experts, int top_k);
int moe_layer_impl(const b200q_moe_args& a, cudaStream_t st);

}  // namespace b200q
