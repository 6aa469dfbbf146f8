// Host-side launchers of the operators on the caller's device memory
// (qd_paged.hip, qd_select.hip; C ABI in qd_operators.cpp). The launchers take
// checked arguments and return what the launch returned.
#pragma once

#include <hip/hip_runtime.h>

#include <cstddef>
#include <cstdint>

#include "qd/qd_operators.h"

namespace qd {

// A workspace starts with arrival counters, which every kernel finds and leaves
// zero; the rest is scratch of the call.
constexpr size_t kOpCounters = 65536;
constexpr size_t kOpCounterBytes = kOpCounters * sizeof(uint32_t);

struct OpScratch {
  uint32_t *counters;  // [kOpCounters]
  char *scratch;
};

constexpr uint32_t kPageSizeLeast = 16, kPageSizeMost = 1024;
constexpr uint32_t kForkRows = 1024, kForkMemories = 4;
constexpr uint32_t kSelectBeams = 32, kSelectK = 64, kSelectVocab = 1u << 24;
constexpr uint32_t kTreeNodes = 64;

hipError_t launch_op_clear(hipStream_t s, uint32_t *counters, size_t n);

// `slots`: where each token goes, or null: its position.
hipError_t launch_paged_append(hipStream_t s, const qd_paged_cache &c, const qd_append_args &a, const int32_t *slots = nullptr);

// Scratch bytes of an attention over `rows` rows, and the most of one over up to so many.
size_t paged_attention_scratch(uint32_t rows, uint32_t heads, uint32_t kv_heads, uint32_t head_dim);
size_t paged_attention_scratch_most(uint32_t rows, uint32_t heads, uint32_t kv_heads, uint32_t head_dim);
// `head_table`: elements from one KV head's table of a row to the next one's; 0: they share it.
hipError_t launch_paged_attention(hipStream_t s, const qd_paged_cache &c, const qd_attention_args &a, const OpScratch &w,
                                  int64_t head_table = 0);

size_t pages_fork_scratch(uint32_t rows, uint32_t pages);
hipError_t launch_pages_fork(hipStream_t s, const qd_fork_args &a, const OpScratch &w);

// What one call needs, and the most that any call of up to these sizes does.
size_t beam_select_scratch(uint32_t groups, uint32_t beams, uint32_t k, uint32_t vocab);
size_t beam_select_scratch_most(uint32_t groups, uint32_t beams, uint32_t k, uint32_t vocab);
hipError_t launch_beam_select(hipStream_t s, const qd_select_args &a, const OpScratch &w);

size_t tree_attention_scratch(uint32_t dtype, uint32_t rows, uint32_t nodes, uint32_t heads, uint32_t kv_heads, uint32_t head_dim);
size_t tree_attention_scratch_most(uint32_t rows, uint32_t nodes, uint32_t heads, uint32_t kv_heads, uint32_t head_dim);
hipError_t launch_tree_attention(hipStream_t s, const qd_paged_cache &c, const qd_tree_attention_args &a, const OpScratch &w);

size_t tree_accept_scratch(uint32_t rows, uint32_t nodes);
hipError_t launch_tree_accept(hipStream_t s, const qd_accept_args &a, const OpScratch &w);
hipError_t launch_tree_commit(hipStream_t s, const qd_commit_args &a);

hipError_t launch_page_bounds(hipStream_t s, const qd_paged_cache &c, void *bounds, uint32_t recent);
size_t sparse_attention_scratch(uint32_t rows, uint32_t heads, uint32_t kv_heads, uint32_t head_dim, uint32_t width, uint32_t budget);
size_t sparse_attention_scratch_most(uint32_t rows, uint32_t heads, uint32_t kv_heads, uint32_t head_dim, uint32_t width,
                                     uint32_t budget);
hipError_t launch_sparse_attention(hipStream_t s, const qd_paged_cache &c, const qd_sparse_args &a, const OpScratch &w);

}  // namespace qd
