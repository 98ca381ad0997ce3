// The host side of an adapter plan: which adapter every row of a packed batch
// uses, as tiles of rows that share one. Plain C++ (no CUDA), so that the tile
// arithmetic can be checked without a device.
#pragma once

#include <algorithm>
#include <cstdint>
#include <vector>

#include "../../../include/semantica_b200.h"

namespace sem {

// Rows of a large tile, and the most rows of a small one (the kernels of
// kernels.h, launch_lowrank_*).
constexpr int kAdapterTileRows = 64;
constexpr int kAdapterSmallRows = 16;

// Up to kAdapterTileRows positions [pos0, pos0 + rows) of the order by adapter
// that all use `adapter` (-1: none). row0: their rows are [row0, row0 + rows),
// or -1 when they do not follow each other.
struct alignas(16) AdapterTile {
  int32_t adapter, pos0, rows, row0;
};

// The rows of a batch ordered by adapter: its sequences sorted by adapter
// (stable), sequence order[i] at positions [pos[i], pos[i + 1]).
struct AdapterPlanHost {
  std::vector<int32_t> order, pos;
  std::vector<AdapterTile> large, small;
  int32_t rows = 0, max_adapter = -1;
};

// Bounds on the tiles of any plan of at most max_rows rows in max_seqs
// sequences: every group of rows of one adapter holds a sequence, gives a
// large tile per kAdapterTileRows rows and at most one more tile.
inline int64_t adapter_plan_max_large(int64_t max_rows, int32_t max_seqs) {
  return max_rows / kAdapterTileRows + max_seqs;
}

// Why (offsets, adapters) is no batch of at most max_rows rows and max_seqs
// sequences; nullptr when it is one. *bad receives the offending sequence.
inline const char* adapter_plan_check(const int32_t* offsets, const int32_t* adapters, int32_t n_seqs,
                                      int64_t max_rows, int32_t max_seqs, int32_t* bad) {
  *bad = -1;
  if (n_seqs < 0) return "negative sequence count";
  if (n_seqs > max_seqs) return "more sequences than the plan was created for";
  if (n_seqs > 0 && (!offsets || !adapters)) return "null argument";
  if (n_seqs > 0 && offsets[0] != 0) return "offsets[0] must be 0";
  for (int32_t s = 0; s < n_seqs; ++s) {
    *bad = s;
    if (offsets[s + 1] < offsets[s]) return "offsets must not decrease";
    if (adapters[s] < -1) return "an adapter is -1 (none) or an index";
  }
  *bad = -1;
  if (n_seqs > 0 && offsets[n_seqs] > max_rows) return "more rows than the plan was created for";
  return nullptr;
}

// What n_absmax activation scales of a call belong to: *per_seq 1, one per
// sequence of a plan of n_seqs; 0, one for every row. A capture keeps the
// answer for batches of other counts, so there the count has to tell the two
// apart. Returns why not, nullptr when it does.
inline const char* lowrank_scales(int32_t n_absmax, int32_t n_seqs, bool captured, int32_t* per_seq) {
  *per_seq = n_absmax == SEM_ABSMAX_PER_SEQUENCE || (n_absmax != 1 && n_absmax == n_seqs);
  if (*per_seq || n_absmax == SEM_ABSMAX_ALL_ROWS) return nullptr;
  if (n_absmax != 1) return "neither one for all rows nor one per sequence";
  if (captured && n_seqs == 1)
    return "a call captured with 1 activation scale for a plan of 1 sequence has to say SEM_ABSMAX_ALL_ROWS or "
           "SEM_ABSMAX_PER_SEQUENCE";
  return nullptr;
}

inline AdapterPlanHost adapter_plan_build(const int32_t* offsets, const int32_t* adapters, int32_t n_seqs) {
  AdapterPlanHost p;
  p.order.resize(n_seqs);
  for (int32_t s = 0; s < n_seqs; ++s) p.order[s] = s;
  std::stable_sort(p.order.begin(), p.order.end(), [&](int32_t a, int32_t b) { return adapters[a] < adapters[b]; });
  p.pos.resize((size_t)n_seqs + 1);
  int32_t at = 0;
  for (int32_t i = 0; i < n_seqs; ++i) {
    p.pos[i] = at;
    at += offsets[p.order[i] + 1] - offsets[p.order[i]];
  }
  p.pos[n_seqs] = p.rows = at;
  auto row_at = [&](int32_t q) {  // the last sequence that starts at or before position q holds it
    const int32_t i = (int32_t)(std::upper_bound(p.pos.begin(), p.pos.end() - 1, q) - p.pos.begin()) - 1;
    return offsets[p.order[i]] + (q - p.pos[i]);
  };
  for (int32_t i = 0; i < n_seqs;) {  // one group of sequences per adapter
    const int32_t a = adapters[p.order[i]];
    int32_t j = i;
    while (j < n_seqs && adapters[p.order[j]] == a) ++j;
    const int32_t end = p.pos[j];
    if (end > p.pos[i]) p.max_adapter = std::max(p.max_adapter, a);
    for (int32_t r = p.pos[i]; r < end;) {
      const int32_t n = std::min(kAdapterTileRows, end - r);
      // the rows of a group increase with its positions
      const int32_t first = row_at(r), last = row_at(r + n - 1);
      (n <= kAdapterSmallRows ? p.small : p.large).push_back(AdapterTile{a, r, n, last - first == n - 1 ? first : -1});
      r += n;
    }
    i = j;
  }
  return p;
}

}  // namespace sem
