// Argument blocks of the paged-cache kernels (shared by the kernel files and the C ABI wrappers).
#pragma once

#include "common.cuh"

namespace b200q {

constexpr int64_t kPagedMaxRequests = 8192;  // the prefix sums over the requests live in shared memory

struct PagedPlanParams {
  const int32_t *context_lens, *new_lens;
  int requests;
  int32_t* table;
  int table_width;
  int64_t table_stride;
  const int32_t* free_pages;
  int64_t free_count;
  const int32_t* free_head;  // or null: 0
  int page_size;
  int num_tokens;
  int64_t *slot_map, *positions;
  int32_t *query_start, *kv_lens, *free_head_out;
};

}  // namespace b200q
