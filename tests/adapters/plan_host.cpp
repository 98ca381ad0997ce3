// The host side of an adapter plan behind a C interface, for tests that need
// no device.
#include <cstring>

#include "../../go-semantica_b200/csrc/host/adapter_plan.h"

extern "C" {

const char* ph_check(const int32_t* offsets, const int32_t* adapters, int32_t n_seqs, int64_t max_rows,
                     int32_t max_seqs, int32_t* bad) {
  const char* why = sem::adapter_plan_check(offsets, adapters, n_seqs, max_rows, max_seqs, bad);
  return why ? why : "";
}

// tiles: room for max_large + max_small of {adapter, pos0, rows, row0}; order: n_seqs,
// pos: n_seqs + 1. counts: large, small, rows, max adapter.
void ph_build(const int32_t* offsets, const int32_t* adapters, int32_t n_seqs, int32_t* order, int32_t* pos,
              int32_t* large, int32_t* small, int32_t* counts) {
  const sem::AdapterPlanHost p = sem::adapter_plan_build(offsets, adapters, n_seqs);
  if (n_seqs > 0) std::memcpy(order, p.order.data(), p.order.size() * 4);
  std::memcpy(pos, p.pos.data(), p.pos.size() * 4);
  if (!p.large.empty()) std::memcpy(large, p.large.data(), p.large.size() * sizeof(sem::AdapterTile));
  if (!p.small.empty()) std::memcpy(small, p.small.data(), p.small.size() * sizeof(sem::AdapterTile));
  counts[0] = (int32_t)p.large.size();
  counts[1] = (int32_t)p.small.size();
  counts[2] = p.rows;
  counts[3] = p.max_adapter;
}

int64_t ph_max_large(int64_t max_rows, int32_t max_seqs) { return sem::adapter_plan_max_large(max_rows, max_seqs); }
int32_t ph_tile_rows() { return sem::kAdapterTileRows; }
int32_t ph_small_rows() { return sem::kAdapterSmallRows; }
}
