// Shared-prefix decode (shared_prefix.cu): the step's plan and the launch of the
// attention of whole groups of requests over the INT2 history they share.
#pragma once

#include "history_common.cuh"

namespace oscar {

// Plan (int32 words, device): header, then per request the end of the history that its
// group's tiles cover (0: none) and the split slots they fill, then the work items.
constexpr int kSharedHead = 8;  // [0] items, [1] CTAs that work on them
struct SharedItem {
  int32_t tok0;            // first token of the group
  int32_t row0, rows;      // this tile's rows of the group (row i: token i / G, query head i % G)
  int32_t leader;          // request whose block table is read
  int32_t tile0, tile1;    // 64-token tiles of this split
  int32_t end;             // history positions [sink, end) count
  int32_t slot;            // split slot of the partial
};
constexpr int kSharedTile = 64, kSharedRows = 128;

inline int64_t shared_up4(int64_t x) { return (x + 3) / 4 * 4; }
inline int64_t shared_words(int64_t max_reqs, int64_t items) {
  return kSharedHead + 2 * shared_up4(max_reqs) + 8 * items;
}

struct SharedLaunch {
  const __nv_bfloat16 *query;  // rotated, [n, hq, 256] contiguous
  const uint8_t *history;
  int64_t num_pages;
  int64_t n;              // tokens of the step
  int32_t table_rows;
  const int32_t *table, *plan;
  int32_t max_reqs, items;  // plan capacities
  float *partials, *lse;
  int32_t split_slots, slot_base;
  oscar_geometry geo;
  float scale_log2;
  int32_t *status;
};
int shared_prefix_launch(const SharedLaunch &L, cudaStream_t stream, int priority);

int sm_count();  // SMs of the current device (attention.cu)
int32_t test_hook_withhold();
uint32_t test_hook_wait_probes();

}  // namespace oscar
