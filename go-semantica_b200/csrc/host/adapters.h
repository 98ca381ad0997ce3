// Handles of the adapter operators, shared with the model's adapted forward.
#pragma once

#include "internal.h"

struct sem_adapter_plan {
  sem_context* ctx = nullptr;
  int64_t max_rows = 0;
  int32_t max_seqs = 0;
  std::mutex mu;            // the host fields below, and set against use
  int32_t n_large = 0, n_small = 0, small_rows = 0, rows = 0, n_seqs = 0, max_adapter = -1;
  sem::DevBuf up;           // counts, sorted sequences, tiles (uploaded)
  sem::DevBuf maps;         // pos_row, pos_seq, row_adapter [max_rows] each
  sem::HostBuf staging;     // the upload's pinned image
  cudaEvent_t staged = nullptr;  // the last upload has been read
  size_t up_bytes = 0;
  ~sem_adapter_plan();
};

struct sem_lowrank {
  sem_context* ctx = nullptr;
  sem::LowRankBank bank{};
  sem::DevBuf weights;  // the adapter table, then every adapter's a and b
  sem::DevBuf err;      // error bits of a timed-out pipeline wait
};

struct sem_block_norm {
  sem_context* ctx = nullptr;
  int32_t dim = 0, n_adapters = 0;
  float eps = 0.0f;
  sem::DevBuf weights;
  const float *post = nullptr, *pre = nullptr, *gates = nullptr, *scales = nullptr;
};

namespace sem {

constexpr int32_t kLowRankMaxDim = 65536;

// plan_create enqueues on the context's stream, plan_set on `st`: the caller holds the context's lock where that is it.
int plan_create(sem_context* ctx, int64_t max_rows, int32_t max_seqs, sem_adapter_plan** out);
int plan_set(sem_adapter_plan* p, const int32_t* offsets, const int32_t* adapters, int32_t n_seqs, cudaStream_t st);
AdapterPlanDev plan_device(const sem_adapter_plan* p);
int lowrank_create(sem_context* ctx, int32_t k_in, int32_t n_out, int32_t n_adapters, const int32_t* ranks,
                   const float* scales, const void* const* a, const void* const* b, int32_t dtype, sem_lowrank** out);
int lowrank_enqueue(const LowRankBank& bank, const sem_adapter_plan* plan, const LowRankArgs& args, bool captured,
                    uint32_t* err, cudaStream_t st);

// The arguments of a block norm over packed rows with the plan's adapters.
BlockNormArgs block_norm_args(const sem_block_norm* b, const sem_adapter_plan* plan, int64_t rows);
int block_norm_create(sem_context* ctx, int32_t dim, float eps, const float* post_w, const float* pre_w,
                      int32_t n_adapters, const float* gates, const float* scales, sem_block_norm** out);

}  // namespace sem
