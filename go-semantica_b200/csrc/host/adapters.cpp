// Adapters of many requests: which adapter every row of a packed batch uses
// (sem_adapter_plan), banks of low-rank adapters beside a shared projection
// (sem_lowrank) and block norms with gates and residual scales
// (sem_block_norm). No reference counterpart: the reference serves one model
// without adapters.
#include "adapters.h"

#include <array>
#include <atomic>
#include <cmath>
#include <cstring>
#include <memory>

namespace sem {

namespace {

std::atomic<int> g_lowrank_path{SEM_LOWRANK_PATH_AUTO};
int get_lowrank_path() { return g_lowrank_path.load(std::memory_order_relaxed); }

bool valid_dtype(int32_t t) { return t == SEM_DTYPE_F32 || t == SEM_DTYPE_F16 || t == SEM_DTYPE_BF16; }
size_t dtype_size(int32_t t) { return t == SEM_DTYPE_F32 ? 4 : 2; }
int64_t round_up(int64_t x, int64_t to) { return (x + to - 1) / to * to; }

// A plan, a bank or a block norm works on its own device only.
int same_device(const sem_context* a, const sem_context* b) {
  if (a->device == b->device) return SEM_OK;
  return set_error(SEM_EINVAL, "the plan is on device %d, the operator on device %d", b->device, a->device);
}

// Holds a context's lock while a call enqueues on the context's own stream: the model's forward may be capturing that
// stream on another thread, and would take the call into its graph. (Taken before a plan's lock.)
std::unique_lock<std::mutex> own_stream(sem_context* ctx, cudaStream_t st) {
  return st == ctx->stream ? std::unique_lock<std::mutex>(ctx->mu) : std::unique_lock<std::mutex>();
}

int capturing(cudaStream_t st, bool* out) {
  cudaStreamCaptureStatus s = cudaStreamCaptureStatusNone;
  SEM_CUDA(cudaStreamIsCapturing(st, &s));
  *out = s != cudaStreamCaptureStatusNone;
  return SEM_OK;
}

}  // namespace

int plan_create(sem_context* ctx, int64_t max_rows, int32_t max_seqs, sem_adapter_plan** out) {
  if (max_rows < 0 || max_rows > 0x7fffffff || max_seqs < 0 || max_seqs == 0x7fffffff)
    return set_error(SEM_EINVAL, "adapter plan: at most 2147483647 rows and 2147483646 sequences");
  if (!ctx || !out) return set_error(SEM_EINVAL, "null argument");
  DeviceGuard dg(ctx->device);
  std::unique_ptr<sem_adapter_plan> p(new sem_adapter_plan());
  p->ctx = ctx;
  p->max_rows = max_rows;
  p->max_seqs = max_seqs;
  const int64_t large = adapter_plan_max_large(max_rows, max_seqs);
  // one buffer: counts and sequences (pos, row0, seq, adapter), large tiles, small tiles; what a batch fills of the three
  // goes up in a copy each
  p->up_bytes = 16 + (size_t)round_up((size_t)4 * max_seqs + 4, 4) * 4 + ((size_t)large + max_seqs + 1) * sizeof(AdapterTile);
  cudaError_t e = p->up.ensure(p->up_bytes);
  if (e == cudaSuccess) e = p->maps.ensure((size_t)3 * (max_rows > 0 ? max_rows : 1) * 4);
  if (e == cudaSuccess) e = p->staging.ensure(p->up_bytes);
  if (e != cudaSuccess) return set_error(SEM_ENOMEM, "adapter plan: %s", cudaGetErrorString(e));
  SEM_CUDA(cudaEventCreateWithFlags(&p->staged, cudaEventDisableTiming));
  SEM_CUDA(cudaMemsetAsync(p->up.p, 0, 16, ctx->stream));
  SEM_CUDA(cudaStreamSynchronize(ctx->stream));
  *out = p.release();
  return SEM_OK;
}

AdapterPlanDev plan_device(const sem_adapter_plan* p) {
  const uint8_t* up = p->up.as<uint8_t>();
  const AdapterTile* tiles = reinterpret_cast<const AdapterTile*>(up + 16 + (size_t)round_up((size_t)4 * p->max_seqs + 4, 4) * 4);
  const int32_t* maps = p->maps.as<int32_t>();
  return AdapterPlanDev{reinterpret_cast<const int32_t*>(up), tiles,
                        tiles + adapter_plan_max_large(p->max_rows, p->max_seqs), maps, maps + p->max_rows,
                        maps + 2 * p->max_rows, p->max_rows, p->max_seqs};
}

int plan_set(sem_adapter_plan* p, const int32_t* offsets, const int32_t* adapters, int32_t n_seqs, cudaStream_t st) {
  int32_t bad = -1;
  if (const char* why = adapter_plan_check(offsets, adapters, n_seqs, p->max_rows, p->max_seqs, &bad)) {
    if (bad >= 0) return set_error(SEM_EINVAL, "adapter plan: %s (sequence %d)", why, bad);
    return set_error(SEM_EINVAL, "adapter plan: %s", why);
  }
  DeviceGuard dg(p->ctx->device);
  std::lock_guard<std::mutex> lk(p->mu);
  bool cap = false;
  if (int rc = capturing(st, &cap)) return rc;
  if (cap) return set_error(SEM_EINVAL, "adapter plan: set it outside stream capture (its tables come from the host)");
  AdapterPlanHost h = adapter_plan_build(offsets, adapters, n_seqs);
  // the previous upload has left the staging buffer
  SEM_CUDA(cudaEventSynchronize(p->staged));
  const size_t seq_ints = (size_t)round_up((size_t)4 * p->max_seqs + 4, 4);  // the tiles start on 16 bytes
  uint8_t* s = p->staging.as<uint8_t>();
  int32_t* counts = reinterpret_cast<int32_t*>(s);
  counts[0] = (int32_t)h.large.size();
  counts[1] = (int32_t)h.small.size();
  counts[2] = h.rows;
  counts[3] = n_seqs;
  int32_t* pos = counts + 4;
  int32_t *row0 = pos + n_seqs + 1, *seq = row0 + n_seqs, *adp = seq + n_seqs;
  for (int32_t i = 0; i < n_seqs; ++i) {
    pos[i] = h.pos[i];
    row0[i] = offsets[h.order[i]];
    seq[i] = h.order[i];
    adp[i] = adapters[h.order[i]];
  }
  pos[n_seqs] = h.rows;
  const int64_t max_large = adapter_plan_max_large(p->max_rows, p->max_seqs);
  uint8_t* tiles = s + 16 + seq_ints * 4;
  uint8_t* small = tiles + (size_t)max_large * sizeof(AdapterTile);
  if (!h.large.empty()) std::memcpy(tiles, h.large.data(), h.large.size() * sizeof(AdapterTile));
  if (!h.small.empty()) std::memcpy(small, h.small.data(), h.small.size() * sizeof(AdapterTile));
  uint8_t* d = p->up.as<uint8_t>();
  auto upload = [&](size_t at, size_t bytes) {
    return bytes ? cudaMemcpyAsync(d + at, s + at, bytes, cudaMemcpyHostToDevice, st) : cudaSuccess;
  };
  SEM_CUDA(upload(0, 16 + ((size_t)4 * n_seqs + 1) * 4));
  SEM_CUDA(upload((size_t)(tiles - s), h.large.size() * sizeof(AdapterTile)));
  SEM_CUDA(upload((size_t)(small - s), h.small.size() * sizeof(AdapterTile)));
  SEM_CUDA(cudaEventRecord(p->staged, st));
  const int32_t* dpos = reinterpret_cast<const int32_t*>(d) + 4;
  int32_t* maps = p->maps.as<int32_t>();
  SEM_CUDA(launch_adapter_plan(dpos, dpos + n_seqs + 1, dpos + 2 * n_seqs + 1, dpos + 3 * n_seqs + 1, n_seqs, h.rows,
                               maps, maps + p->max_rows, maps + 2 * p->max_rows, st));
  p->n_large = (int32_t)h.large.size();
  p->n_small = (int32_t)h.small.size();
  p->small_rows = 0;
  for (const AdapterTile& t : h.small) p->small_rows += t.rows;
  p->rows = h.rows;
  p->n_seqs = n_seqs;
  p->max_adapter = h.max_adapter;
  return SEM_OK;
}

int lowrank_create(sem_context* ctx, int32_t k_in, int32_t n_out, int32_t n_adapters, const int32_t* ranks,
                   const float* scales, const void* const* a, const void* const* b, int32_t dtype,
                   sem_lowrank** out) {
  if (k_in <= 0 || n_out <= 0 || k_in > kLowRankMaxDim || n_out > kLowRankMaxDim)
    return set_error(SEM_EINVAL, "low-rank adapters %d x %d: both dimensions must be in 1..%d", k_in, n_out,
                     kLowRankMaxDim);
  if (n_adapters < 0) return set_error(SEM_EINVAL, "low-rank adapters: negative count %d", n_adapters);
  if (!valid_dtype(dtype)) return set_error(SEM_EINVAL, "low-rank adapters: unknown element type %d", dtype);
  if (n_adapters > 0 && (!ranks || !scales || !a || !b)) return set_error(SEM_EINVAL, "null argument");
  for (int32_t i = 0; i < n_adapters; ++i) {
    if (ranks[i] < 0 || ranks[i] > kLowRankMaxRank)
      return set_error(SEM_EINVAL, "low-rank adapter %d: rank %d out of range (0..%d)", i, ranks[i], kLowRankMaxRank);
    if (ranks[i] > 0 && (!a[i] || !b[i])) return set_error(SEM_EINVAL, "low-rank adapter %d: null weights", i);
  }
  if (!ctx || !out) return set_error(SEM_EINVAL, "null argument");
  DeviceGuard dg(ctx->device);
  std::unique_ptr<sem_lowrank> w(new sem_lowrank());
  w->ctx = ctx;
  const size_t es = dtype_size(dtype);
  const int32_t ka = (int32_t)round_up(k_in, 64);
  // host image: the adapter table, then every adapter's a and b, rows padded with zeros
  size_t bytes = (size_t)round_up((int64_t)n_adapters * sizeof(LowRankAdapter), 256);
  std::vector<size_t> at_a(n_adapters), at_b(n_adapters), at_tb(n_adapters), at_us(n_adapters);
  std::vector<std::array<size_t, 3>> at_ta(n_adapters);
  int32_t max_rank = 0;
  for (int32_t i = 0; i < n_adapters; ++i) {
    const int64_t rp = round_up(ranks[i], 8);
    at_a[i] = bytes;
    bytes += (size_t)round_up((int64_t)ranks[i] * ka * es, 256);
    at_b[i] = bytes;
    bytes += (size_t)round_up((int64_t)n_out * rp * es, 256);
    if (ranks[i] > max_rank) max_rank = ranks[i];
  }
  // behind the image, filled on the device: the weights as the tensor-core kernel's tiles
  size_t total = bytes;
  for (int32_t i = 0; i < n_adapters; ++i) {
    const int32_t rp = (int32_t)round_up(ranks[i], 8);
    for (int x = 0; x < 3; ++x) {
      at_ta[i][x] = total;
      total += lowrank_tile_bytes_a(ranks[i], ka, dtype, x);  // these are multiples of 128 bytes
    }
    at_tb[i] = total;
    total += lowrank_tile_bytes_b(rp, n_out, dtype);
    at_us[i] = total;
    total += (size_t)round_up(rp * 4, 128);
  }
  cudaError_t e = w->weights.ensure(total > 0 ? total : 256);
  if (e != cudaSuccess)
    return set_error(SEM_ENOMEM, "device allocation of %zu bytes failed: %s", total, cudaGetErrorString(e));
  e = w->err.ensure(16);
  if (e != cudaSuccess) return set_error(SEM_ENOMEM, "device allocation failed: %s", cudaGetErrorString(e));
  std::vector<uint8_t> img(bytes, 0);
  uint8_t* d = w->weights.as<uint8_t>();
  for (int32_t i = 0; i < n_adapters; ++i) {
    const int32_t r = ranks[i], rp = (int32_t)round_up(r, 8);
    for (int32_t j = 0; j < r; ++j)
      std::memcpy(&img[at_a[i] + (size_t)j * ka * es], static_cast<const uint8_t*>(a[i]) + (size_t)j * k_in * es,
                  (size_t)k_in * es);
    for (int32_t n = 0; r > 0 && n < n_out; ++n)
      std::memcpy(&img[at_b[i] + (size_t)n * rp * es], static_cast<const uint8_t*>(b[i]) + (size_t)n * r * es,
                  (size_t)r * es);
    const LowRankAdapter ad{d + at_a[i],
                            d + at_b[i],
                            d + at_tb[i],
                            {d + at_ta[i][0], d + at_ta[i][1], d + at_ta[i][2]},
                            lowrank_has_unscale(dtype) ? reinterpret_cast<const float*>(d + at_us[i]) : nullptr,
                            r,
                            rp,
                            scales[i]};
    std::memcpy(&img[(size_t)i * sizeof(LowRankAdapter)], &ad, sizeof ad);
  }
  w->bank = LowRankBank{reinterpret_cast<const LowRankAdapter*>(d), n_adapters, k_in, n_out, ka, dtype, max_rank};
  std::lock_guard<std::mutex> lk(ctx->mu);
  if (bytes) SEM_CUDA(cudaMemcpyAsync(d, img.data(), bytes, cudaMemcpyHostToDevice, ctx->stream));
  SEM_CUDA(launch_lowrank_tiles(w->bank, ctx->stream));
  SEM_CUDA(cudaMemsetAsync(w->err.p, 0, 16, ctx->stream));
  SEM_CUDA(cudaStreamSynchronize(ctx->stream));
  *out = w.release();
  return SEM_OK;
}

namespace {

// What both forms of the call share. The plan is looked at and the call enqueued under one lock, so that the batch
// that the checks saw is the one that the call runs on. n_absmax: the activation scales given (null: none).
int lowrank_launch(sem_lowrank* w, sem_adapter_plan* plan, LowRankArgs args, const int32_t* n_absmax, void* stream) {
  if (int rc = same_device(w->ctx, plan->ctx)) return rc;
  DeviceGuard dg(w->ctx->device);
  cudaStream_t st = stream ? static_cast<cudaStream_t>(stream) : w->ctx->stream;
  const auto own = own_stream(w->ctx, st);
  std::lock_guard<std::mutex> lk(plan->mu);
  if (plan->max_adapter >= w->bank.n_adapters)
    return set_error(SEM_EINVAL, "low-rank adapters: the plan uses adapter %d, the bank has %d", plan->max_adapter,
                     w->bank.n_adapters);
  bool cap = false;
  if (int rc = capturing(st, &cap)) return rc;
  if (n_absmax)
    if (const char* why = lowrank_scales(*n_absmax, plan->n_seqs, cap, &args.per_seq))
      return set_error(SEM_EINVAL, "low-rank adapters: %d activation scales for a plan of %d sequences: %s", *n_absmax,
                       plan->n_seqs, why);
  return lowrank_enqueue(w->bank, plan, args, cap, w->err.as<uint32_t>(), st);
}

}  // namespace

// Up to this many multiply-adds a call runs on the CUDA cores as a whole: the
// tensor-core kernel's pipeline takes longer to fill than they take. Measured
// (CUDA cores / tensor cores, 768 x 768, rank 16, per call of a CUDA graph):
// INT8 codes 12.6 M 7.8 / 12.0 us, 25 M 11.5 / 13.5, 50 M 18.2 / 14.8; float32
// rows, whose conversion the tensor cores wait for, 25 M 11.0 / 20.2, 63 M
// 21.3 / 21.9; 517 x 1001, 212 M 43.2 / 34.9. A tile of up to 16 rows counts as
// eight (256 single fp16 rows of as many adapters: 32.1 / 26.7 us; 64 tiles of 12
// rows: 11.1 / 15.7).
constexpr int64_t kLowRankSmallWork = 28000000, kLowRankSmallWorkF32 = 60000000;

// One launch for all tiles of the plan, also for an empty plan when it is
// captured (a replay may find the plan set to another batch).
int lowrank_enqueue(const LowRankBank& bank, const sem_adapter_plan* plan, const LowRankArgs& args, bool captured,
                    uint32_t* err, cudaStream_t st) {
  const AdapterPlanDev dev = plan_device(plan);
  const int64_t rows = (int64_t)plan->rows - plan->small_rows + 8 * (int64_t)plan->n_small;
  const int64_t work = rows * bank.max_rank * (bank.k_in + bank.n_out);
  const int path = get_lowrank_path();
  const bool cuda_cores = path == SEM_LOWRANK_PATH_CUDA_CORES || (path == SEM_LOWRANK_PATH_AUTO && work <= (args.xtype == kDtF32 ? kLowRankSmallWorkF32 : kLowRankSmallWork));
  if (plan->rows == 0 && !captured) return SEM_OK;
  const int n_large = plan->n_large, n_small = n_large || plan->n_small ? plan->n_small : 1;
  if (cuda_cores) SEM_CUDA(launch_lowrank_small(bank, dev, n_large, n_small, args, st));
  else SEM_CUDA(launch_lowrank_tc(bank, dev, n_large, n_small, args, err, st));
  return SEM_OK;
}

namespace {

int check_ld(const char* what, int64_t* ld, int64_t width) {
  if (*ld == 0) *ld = width;
  if (*ld < width) return set_error(SEM_EINVAL, "%s: row stride %lld below the %lld values of a row", what,
                                    (long long)*ld, (long long)width);
  return SEM_OK;
}

bool misaligned(const void* p, int32_t dtype) { return (reinterpret_cast<uintptr_t>(p) & (dtype_size(dtype) - 1)) != 0; }

int lowrank_apply(sem_lowrank* w, sem_adapter_plan* plan, const void* d_x, int32_t x_dtype, int64_t ldx,
                  const void* d_base, int64_t ld_base, void* d_y, int32_t y_dtype, int64_t ldy, void* stream) {
  if (!valid_dtype(x_dtype) || !valid_dtype(y_dtype) || (y_dtype != x_dtype && y_dtype != SEM_DTYPE_F32))
    return set_error(SEM_EINVAL, "low-rank adapters: no form for inputs of type %d and outputs of type %d", x_dtype,
                     y_dtype);
  if (!w || !plan || !d_x || !d_y) return set_error(SEM_EINVAL, "null argument");
  int rc;
  if ((rc = check_ld("low-rank adapters: inputs", &ldx, w->bank.k_in))) return rc;
  if ((rc = check_ld("low-rank adapters: base", &ld_base, w->bank.n_out))) return rc;
  if ((rc = check_ld("low-rank adapters: outputs", &ldy, w->bank.n_out))) return rc;
  if (misaligned(d_x, x_dtype) || misaligned(d_y, y_dtype) || misaligned(d_base, y_dtype))
    return set_error(SEM_EINVAL, "low-rank adapters: a pointer is not aligned to its element type");
  if (d_base == d_y && ld_base != ldy)
    return set_error(SEM_EINVAL, "low-rank adapters: base and outputs are one buffer with two row strides");
  LowRankArgs a{d_x, d_base, d_y, ldx, ld_base, ldy, x_dtype, y_dtype, nullptr, 0};
  return lowrank_launch(w, plan, a, nullptr, stream);
}

int lowrank_apply_int8(sem_lowrank* w, sem_adapter_plan* plan, const void* d_codes, const uint32_t* d_absmax,
                       int32_t n_absmax, const float* d_base, int64_t ld_base, float* d_y, int64_t ldy,
                       void* stream) {
  if (!w || !plan || !d_codes || !d_absmax || !d_y) return set_error(SEM_EINVAL, "null argument");
  int rc;
  if ((rc = check_ld("low-rank adapters: base", &ld_base, w->bank.n_out))) return rc;
  if ((rc = check_ld("low-rank adapters: outputs", &ldy, w->bank.n_out))) return rc;
  if (misaligned(d_codes, SEM_DTYPE_F16) || misaligned(d_absmax, SEM_DTYPE_F32) || misaligned(d_y, SEM_DTYPE_F32) ||
      misaligned(d_base, SEM_DTYPE_F32))
    return set_error(SEM_EINVAL, "low-rank adapters: a pointer is not aligned to its element type");
  if (d_base == d_y && ld_base != ldy)
    return set_error(SEM_EINVAL, "low-rank adapters: base and outputs are one buffer with two row strides");
  LowRankArgs a{d_codes, d_base, d_y, w->bank.k_in, ld_base, ldy, SEM_DTYPE_F16, SEM_DTYPE_F32, d_absmax, 0};
  return lowrank_launch(w, plan, a, &n_absmax, stream);
}

int lowrank_check(sem_lowrank* w) {
  if (!w) return set_error(SEM_EINVAL, "null argument");
  DeviceGuard dg(w->ctx->device);
  std::lock_guard<std::mutex> lk(w->ctx->mu);
  SEM_CUDA(cudaDeviceSynchronize());
  uint32_t bits = 0;
  SEM_CUDA(cudaMemcpyAsync(&bits, w->err.p, 4, cudaMemcpyDeviceToHost, w->ctx->stream));
  SEM_CUDA(cudaMemsetAsync(w->err.p, 0, 4, w->ctx->stream));
  SEM_CUDA(cudaStreamSynchronize(w->ctx->stream));
  if (bits)
    return set_error(SEM_EDEVICE, "low-rank adapters: a tensor-core pipeline wait timed out (error bits 0x%x)", bits);
  return SEM_OK;
}

}  // namespace

int block_norm_create(sem_context* ctx, int32_t dim, float eps, const float* post_w, const float* pre_w,
                      int32_t n_adapters, const float* gates, const float* scales, sem_block_norm** out) {
  if (dim <= 0 || dim > kBlockNormMaxDim)
    return set_error(SEM_EINVAL, "block norm: %d values per row, 1..%d are supported", dim, kBlockNormMaxDim);
  if (!(eps >= 0.0f) || std::isinf(eps)) return set_error(SEM_EINVAL, "block norm: eps must be finite and not negative");
  if (n_adapters < 0) return set_error(SEM_EINVAL, "block norm: negative adapter count %d", n_adapters);
  if (!ctx || !out) return set_error(SEM_EINVAL, "null argument");
  DeviceGuard dg(ctx->device);
  std::unique_ptr<sem_block_norm> b(new sem_block_norm());
  b->ctx = ctx;
  b->dim = dim;
  b->eps = eps;
  b->n_adapters = n_adapters;
  // post, pre and each gate from a 16-byte boundary on when dim is a multiple of 4 (the vector kernels' case)
  const size_t vec = (size_t)round_up(dim, 4);
  const size_t n_gates = gates ? (size_t)n_adapters * dim : 0;
  const size_t total = 2 * vec + (size_t)round_up((int64_t)n_gates, 4) + (scales ? n_adapters : 0) + 4;
  cudaError_t e = b->weights.ensure(total * 4);
  if (e != cudaSuccess)
    return set_error(SEM_ENOMEM, "device allocation of %zu bytes failed: %s", total * 4, cudaGetErrorString(e));
  float* d = b->weights.as<float>();
  std::lock_guard<std::mutex> lk(ctx->mu);
  auto put = [&](const float* src, size_t at, size_t n, const float** dst) -> cudaError_t {
    *dst = nullptr;
    if (!src || !n) return cudaSuccess;
    *dst = d + at;
    return cudaMemcpyAsync(d + at, src, n * 4, cudaMemcpyHostToDevice, ctx->stream);
  };
  SEM_CUDA(put(post_w, 0, dim, &b->post));
  SEM_CUDA(put(pre_w, vec, dim, &b->pre));
  SEM_CUDA(put(gates, 2 * vec, n_gates, &b->gates));
  SEM_CUDA(put(scales, 2 * vec + (size_t)round_up((int64_t)n_gates, 4), scales ? n_adapters : 0, &b->scales));
  SEM_CUDA(cudaStreamSynchronize(ctx->stream));
  *out = b.release();
  return SEM_OK;
}

BlockNormArgs block_norm_args(const sem_block_norm* b, const sem_adapter_plan* plan, int64_t rows) {
  BlockNormArgs a{};
  a.ldo = a.ldh = a.ldho = a.ldy = b->dim;
  a.dtype = a.htype = kDtF32;
  a.rows = rows;
  a.dim = b->dim;
  a.eps = b->eps;
  a.post = b->post;
  a.pre = b->pre;
  a.gates = b->gates;
  a.scales = b->scales;
  a.n_adapters = b->n_adapters;
  a.row_adapter = plan ? plan_device(plan).row_adapter : nullptr;
  return a;
}

namespace {

int block_norm_run(sem_block_norm* b, sem_adapter_plan* plan, int64_t rows, const void* d_o, int64_t ldo,
                   int32_t dtype, const void* d_h, int64_t ldh, int32_t h_dtype, void* d_h_out, int64_t ldho,
                   void* d_y, int64_t ldy, void* stream) {
  if (!valid_dtype(dtype) || !valid_dtype(h_dtype) || (h_dtype != dtype && h_dtype != SEM_DTYPE_F32))
    return set_error(SEM_EINVAL, "block norm: no form for block outputs of type %d and a residual of type %d", dtype,
                     h_dtype);
  if (rows < 0 || rows > 0x7fffffff) return set_error(SEM_EINVAL, "block norm: %lld rows", (long long)rows);
  if (!b) return set_error(SEM_EINVAL, "null argument");
  if (rows > 0 && (!d_o || !d_h || !d_h_out || (b->pre && !d_y))) return set_error(SEM_EINVAL, "null argument");
  int rc;
  if ((rc = check_ld("block norm: block outputs", &ldo, b->dim))) return rc;
  if ((rc = check_ld("block norm: residual", &ldh, b->dim))) return rc;
  if ((rc = check_ld("block norm: new residual", &ldho, b->dim))) return rc;
  if ((rc = check_ld("block norm: outputs", &ldy, b->dim))) return rc;
  if (misaligned(d_o, dtype) || misaligned(d_y, dtype) || misaligned(d_h, h_dtype) || misaligned(d_h_out, h_dtype))
    return set_error(SEM_EINVAL, "block norm: a pointer is not aligned to its element type");
  if ((d_h_out == d_h && ldho != ldh) || (b->pre && d_y == d_o && ldy != ldo))
    return set_error(SEM_EINVAL, "block norm: one buffer with two row strides");
  DeviceGuard dg(b->ctx->device);
  cudaStream_t st = stream ? static_cast<cudaStream_t>(stream) : b->ctx->stream;
  const auto own = own_stream(b->ctx, st);
  std::unique_lock<std::mutex> lk;  // until the call is enqueued, as in lowrank_launch
  if (plan) {
    if ((rc = same_device(b->ctx, plan->ctx))) return rc;
    lk = std::unique_lock<std::mutex>(plan->mu);
    if (plan->rows != rows)
      return set_error(SEM_EINVAL, "block norm: %lld rows, the plan has %d", (long long)rows, plan->rows);
    if ((b->gates || b->scales) && plan->max_adapter >= b->n_adapters)
      return set_error(SEM_EINVAL, "block norm: the plan uses adapter %d, there are %d", plan->max_adapter,
                       b->n_adapters);
  }
  BlockNormArgs a = block_norm_args(b, plan, rows);
  a.o = d_o;
  a.h = d_h;
  a.h_out = d_h_out;
  a.y = b->pre ? d_y : nullptr;
  a.ldo = ldo;
  a.ldh = ldh;
  a.ldho = ldho;
  a.ldy = ldy;
  a.dtype = dtype;
  a.htype = h_dtype;
  SEM_CUDA(launch_block_norm(a, st));
  return SEM_OK;
}

// Frees a handle once the work enqueued on its device is done (not while the context's stream is captured: a device
// with a captured stream cannot be waited for).
template <class T>
int free_handle(T* h) {
  if (!h) return SEM_OK;
  DeviceGuard dg(h->ctx->device);
  std::lock_guard<std::mutex> lk(h->ctx->mu);
  cudaDeviceSynchronize();
  delete h;
  return SEM_OK;
}

}  // namespace
}  // namespace sem

sem_adapter_plan::~sem_adapter_plan() {
  if (staged) cudaEventDestroy(staged);
}

extern "C" {

int sem_adapter_plan_create(sem_context* ctx, int64_t max_rows, int32_t max_seqs, sem_adapter_plan** out) {
  return sem::guarded([&]() -> int {
    const auto own = ctx ? sem::own_stream(ctx, ctx->stream) : std::unique_lock<std::mutex>();
    return sem::plan_create(ctx, max_rows, max_seqs, out);
  });
}

int sem_adapter_plan_set(sem_adapter_plan* plan, const int32_t* offsets, const int32_t* adapters, int32_t n_seqs,
                         void* stream) {
  return sem::guarded([&]() -> int {
    if (!plan) return sem::set_error(SEM_EINVAL, "null argument");
    cudaStream_t st = stream ? static_cast<cudaStream_t>(stream) : plan->ctx->stream;
    const auto own = sem::own_stream(plan->ctx, st);
    return sem::plan_set(plan, offsets, adapters, n_seqs, st);
  });
}

int sem_adapter_plan_free(sem_adapter_plan* plan) {
  return sem::guarded([&]() -> int { return sem::free_handle(plan); });
}

int sem_lowrank_create(sem_context* ctx, int32_t k_in, int32_t n_out, int32_t n_adapters, const int32_t* ranks,
                       const float* scales, const void* const* a, const void* const* b, int32_t dtype,
                       sem_lowrank** out) {
  return sem::guarded([&]() -> int {
    return sem::lowrank_create(ctx, k_in, n_out, n_adapters, ranks, scales, a, b, dtype, out);
  });
}

int sem_lowrank_free(sem_lowrank* w) {
  return sem::guarded([&]() -> int { return sem::free_handle(w); });
}

int sem_lowrank_apply(sem_lowrank* w, sem_adapter_plan* plan, const void* d_x, int32_t x_dtype, int64_t ldx,
                      const void* d_base, int64_t ld_base, void* d_y, int32_t y_dtype, int64_t ldy, void* stream) {
  return sem::guarded([&]() -> int {
    return sem::lowrank_apply(w, plan, d_x, x_dtype, ldx, d_base, ld_base, d_y, y_dtype, ldy, stream);
  });
}

int sem_lowrank_apply_int8(sem_lowrank* w, sem_adapter_plan* plan, const void* d_codes, const uint32_t* d_absmax,
                           int32_t n_absmax, const float* d_base, int64_t ld_base, float* d_y, int64_t ldy,
                           void* stream) {
  return sem::guarded([&]() -> int {
    return sem::lowrank_apply_int8(w, plan, d_codes, d_absmax, n_absmax, d_base, ld_base, d_y, ldy, stream);
  });
}

int sem_lowrank_path(int32_t mode) {
  return sem::guarded([&]() -> int {
    if (mode < SEM_LOWRANK_PATH_AUTO || mode > SEM_LOWRANK_PATH_TENSOR) return -1;
    return sem::g_lowrank_path.exchange(mode);
  });
}

int sem_lowrank_check(sem_lowrank* w) {
  return sem::guarded([&]() -> int { return sem::lowrank_check(w); });
}

int sem_block_norm_create(sem_context* ctx, int32_t dim, float eps, const float* post_w, const float* pre_w,
                          int32_t n_adapters, const float* gates, const float* scales, sem_block_norm** out) {
  return sem::guarded([&]() -> int {
    return sem::block_norm_create(ctx, dim, eps, post_w, pre_w, n_adapters, gates, scales, out);
  });
}

int sem_block_norm_free(sem_block_norm* b) {
  return sem::guarded([&]() -> int { return sem::free_handle(b); });
}

int sem_block_norm_run(sem_block_norm* b, sem_adapter_plan* plan, int64_t rows, const void* d_o, int64_t ldo,
                       int32_t dtype, const void* d_h, int64_t ldh, int32_t h_dtype, void* d_h_out, int64_t ldho,
                       void* d_y, int64_t ldy, void* stream) {
  return sem::guarded([&]() -> int {
    return sem::block_norm_run(b, plan, rows, d_o, ldo, dtype, d_h, ldh, h_dtype, d_h_out, ldho, d_y, ldy, stream);
  });
}

}  // extern "C"
