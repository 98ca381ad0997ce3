// Adapters of many requests (sm_100a): the plan's row maps, the low-rank
// adapters of small tiles on CUDA cores, and the block norm with its gate and
// residual scale. The tensor-core kernel of the large tiles is lowrank_tc.cu.
#include <cooperative_groups.h>
#include <cuda_bf16.h>

#include <type_traits>

#include "common.cuh"
#include "kernels.h"

namespace sem {

namespace cg = cooperative_groups;

namespace {

// ---------------------------------------------------------------------------
// Plan: row maps
// ---------------------------------------------------------------------------
// A thread per position finds its sequence by bisection over the sorted
// prefix (log2 of the sequence count steps, all in L1) and writes the three
// maps: 12 bytes a row, once per batch, against kilobytes a row in every
// operator that goes by them.
__global__ void adapter_plan_kernel(const int32_t* __restrict__ pos, const int32_t* __restrict__ row0,
                                    const int32_t* __restrict__ seq, const int32_t* __restrict__ adapter,
                                    int32_t n_seqs, int32_t rows, int32_t* __restrict__ pos_row,
                                    int32_t* __restrict__ pos_seq, int32_t* __restrict__ row_adapter) {
  const int64_t p = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
  if (p >= rows) return;
  int lo = 0, hi = n_seqs - 1;  // the last i with pos[i] <= p (empty sequences share a position: the last one holds it)
  while (lo < hi) {
    const int mid = lo + (hi - lo + 1) / 2;
    if (pos[mid] <= p) lo = mid;
    else hi = mid - 1;
  }
  const int32_t row = row0[lo] + (int32_t)(p - pos[lo]);
  pos_row[p] = row;
  pos_seq[p] = seq[lo];
  row_adapter[row] = adapter[lo];
}

// ---------------------------------------------------------------------------
// Element access
// ---------------------------------------------------------------------------
__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
template <class T>
__device__ __forceinline__ T from_f32(float v) {
  if constexpr (std::is_same<T, float>::value) return v;
  else if constexpr (std::is_same<T, __half>::value) return __float2half_rn(v);
  else return __float2bfloat16_rn(v);
}

// N consecutive elements (N * sizeof(T) bytes, aligned to that) as floats.
template <int N, class T>
__device__ __forceinline__ void load_vec(const T* p, float (&v)[N]) {
  struct alignas(N * sizeof(T)) Pack { T e[N]; };
  const Pack k = *reinterpret_cast<const Pack*>(p);
#pragma unroll
  for (int i = 0; i < N; ++i) v[i] = to_f32(k.e[i]);
}
template <int N, class T>
__device__ __forceinline__ void store_vec(T* p, const float (&v)[N]) {
  struct alignas(N * sizeof(T)) Pack { T e[N]; } k;
#pragma unroll
  for (int i = 0; i < N; ++i) k.e[i] = from_f32<T>(v[i]);
  *reinterpret_cast<Pack*>(p) = k;
}

// Eight consecutive weights (16-byte aligned) of a bank's type.
__device__ __forceinline__ void load_weights8(const void* base, int64_t at, int wtype, float (&v)[8]) {
  if (wtype == kDtF32) {
    const float4* p = reinterpret_cast<const float4*>(static_cast<const float*>(base) + at);
    const float4 a = p[0], b = p[1];
    v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w, v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
  } else if (wtype == kDtF16) {
    load_vec<8>(static_cast<const __half*>(base) + at, v);
  } else {
    load_vec<8>(static_cast<const __nv_bfloat16*>(base) + at, v);
  }
}

// ---------------------------------------------------------------------------
// Low-rank adapters on CUDA cores
// ---------------------------------------------------------------------------
// A cluster of eight CTAs takes one tile: CTA c sums its eighth of the input
// channels into partial t = x A^T (16 rows at a time), the partials meet
// through distributed shared memory, every CTA adds them in the same order
// (results do not depend on timing), and each finishes its eighth of the
// output channels. One launch with no workspace: a single row's latency is two
// short dependent loads (A, then B) instead of one SM walking both weights.
constexpr int kSmallCtas = 8, kSmallThreads = 256, kSmallWarps = kSmallThreads / 32;
constexpr int kSmallChunk = 128;  // input channels staged at a time, 4 per lane

template <class XT, class YT>
__global__ void __cluster_dims__(kSmallCtas, 1, 1) __launch_bounds__(kSmallThreads)
    lowrank_small_kernel(LowRankBank bank, AdapterPlanDev plan, LowRankArgs a) {
  constexpr int R = kAdapterSmallRows;
  __shared__ __align__(16) float s_x[R][kSmallChunk];
  __shared__ __align__(16) float s_part[kLowRankMaxRank][R];
  __shared__ __align__(16) float s_t[kLowRankMaxRank][R];
  __shared__ int32_t s_row[R];
  __shared__ float s_scale[R];
  cg::cluster_group cluster = cg::this_cluster();
  const int rank_id = (int)cluster.block_rank();
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int n_tiles = plan.counts[1];
  const XT* x = static_cast<const XT*>(a.x);
  const YT* base = static_cast<const YT*>(a.base);
  YT* y = static_cast<YT*>(a.y);
  // this CTA's input and output channels
  const int kper = (bank.ka / 32 + kSmallCtas - 1) / kSmallCtas * 32;
  const int k0 = min(bank.k_in, rank_id * kper), k1 = min(bank.k_in, k0 + kper);
  const int nper = (bank.n_out + kSmallCtas - 1) / kSmallCtas;
  const int n0 = min(bank.n_out, rank_id * nper), n1 = min(bank.n_out, n0 + nper);

  for (int tile = (int)(blockIdx.x / kSmallCtas); tile < n_tiles; tile += (int)(gridDim.x / kSmallCtas)) {
    const AdapterTile tl = plan.small[tile];
    LowRankAdapter ad{};
    if (tl.adapter >= 0 && tl.adapter < bank.n_adapters) ad = bank.adapters[tl.adapter];
    if (ad.rank == 0 && a.base == a.y && a.ldb == a.ldy) continue;  // in place and nothing to add (the whole cluster)
    for (int sub = 0; sub < tl.rows; sub += R) {
      const int rows = min(R, tl.rows - sub);
      if (tid < R) {
        const int p = tl.pos0 + sub + min(tid, rows - 1);
        s_row[tid] = plan.pos_row[p];
        float sc = ad.scale;
        if (a.absmax) sc = __fmul_rn(sc, __fdiv_rn(__uint_as_float(a.absmax[a.per_seq ? plan.pos_seq[p] : 0]), 127.0f));
        s_scale[tid] = sc;
      }
      __syncthreads();
      if (ad.rank > 0) {
        // partial t of this CTA's input channels: a warp per rank row j, its
        // lanes four channels each, 16 rows of x from shared memory
        for (int j0 = 0; j0 < ad.rank; j0 += kSmallWarps * 4) {
          float acc[4][R];
#pragma unroll
          for (int u = 0; u < 4; ++u)
#pragma unroll
            for (int i = 0; i < R; ++i) acc[u][i] = 0.0f;
          for (int kc = k0; kc < k1; kc += kSmallChunk) {
            const int kn = min(kSmallChunk, k1 - kc);
            __syncthreads();
            for (int i = tid; i < R * kSmallChunk; i += kSmallThreads) {
              const int r = i / kSmallChunk, c = i % kSmallChunk;
              s_x[r][c] = r < rows && c < kn ? to_f32(x[(int64_t)s_row[r] * a.ldx + kc + c]) : 0.0f;
            }
            __syncthreads();
#pragma unroll
            for (int u = 0; u < 4; ++u) {
              const int j = j0 + warp + u * kSmallWarps;
              if (j >= ad.rank || kc + lane * 4 >= bank.ka) continue;  // A's rows end at ka (zeros behind k_in)
              float w[4];
              const int64_t at = (int64_t)j * bank.ka + kc + lane * 4;
              if (bank.wtype == kDtF32) load_vec<4>(static_cast<const float*>(ad.a) + at, w);
              else if (bank.wtype == kDtF16) load_vec<4>(static_cast<const __half*>(ad.a) + at, w);
              else load_vec<4>(static_cast<const __nv_bfloat16*>(ad.a) + at, w);
              if (lane * 4 >= kn) w[0] = w[1] = w[2] = w[3] = 0.0f;  // the next CTA's channels
#pragma unroll
              for (int i = 0; i < R; ++i) {
                const float4 v = *reinterpret_cast<const float4*>(&s_x[i][lane * 4]);
                acc[u][i] = fmaf(v.x, w[0], fmaf(v.y, w[1], fmaf(v.z, w[2], fmaf(v.w, w[3], acc[u][i]))));
              }
            }
          }
#pragma unroll
          for (int u = 0; u < 4; ++u) {
            const int j = j0 + warp + u * kSmallWarps;
            if (j >= ad.rank) continue;
#pragma unroll
            for (int i = 0; i < R; ++i) {
              float v = acc[u][i];
#pragma unroll
              for (int o = 16; o > 0; o >>= 1) v = __fadd_rn(v, __shfl_xor_sync(0xffffffffu, v, o));
              if (lane == i) s_part[j][i] = v;
            }
          }
        }
        cluster.sync();
        for (int i = tid; i < ad.rank * R; i += kSmallThreads) {
          float v = 0.0f;
#pragma unroll
          for (int c = 0; c < kSmallCtas; ++c)
            v = __fadd_rn(v, *cluster.map_shared_rank(&s_part[0][0] + i, c));
          (&s_t[0][0])[i] = __fmul_rn(v, s_scale[i % R]);
        }
        cluster.sync();  // the partials are free for the next 16 rows
      }
      // this CTA's output channels: a thread per (channel, half of the rows)
      constexpr int H = R / 2;
      const int half = tid & 1;
      for (int n = n0 + (tid >> 1); n < n1; n += kSmallThreads / 2) {
        float acc[H];
#pragma unroll
        for (int i = 0; i < H; ++i) acc[i] = 0.0f;
        for (int j = 0; j < ad.rank; j += 8) {  // B's columns end at rp, zeros behind the rank
          float w[8];
          load_weights8(ad.b, (int64_t)n * ad.rp + j, bank.wtype, w);
#pragma unroll
          for (int u = 0; u < 8; ++u) {
            if (j + u >= ad.rank) break;
#pragma unroll
            for (int i = 0; i < H; i += 4) {
              const float4 t = *reinterpret_cast<const float4*>(&s_t[j + u][half * H + i]);
              acc[i] = fmaf(t.x, w[u], acc[i]);
              acc[i + 1] = fmaf(t.y, w[u], acc[i + 1]);
              acc[i + 2] = fmaf(t.z, w[u], acc[i + 2]);
              acc[i + 3] = fmaf(t.w, w[u], acc[i + 3]);
            }
          }
        }
#pragma unroll
        for (int i = 0; i < H; ++i) {
          const int r = half * H + i;
          if (r >= rows) continue;
          const float b = base ? to_f32(base[(int64_t)s_row[r] * a.ldb + n]) : 0.0f;
          y[(int64_t)s_row[r] * a.ldy + n] = from_f32<YT>(__fadd_rn(b, acc[i]));
        }
      }
      __syncthreads();
    }
  }
}

// ---------------------------------------------------------------------------
// Block norm
// ---------------------------------------------------------------------------
// TPR threads hold one row in registers, NC chunks of VEC elements each, so o
// and h are read once and h_out and y written once; the two sums of squares
// are float32 partial sums joined by a fixed tree. Bound by HBM.
constexpr int kNormThreads = 128;

template <int TPR>
__device__ __forceinline__ float row_sum(float v, float* s_red, int slot) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = __fadd_rn(v, __shfl_xor_sync(0xffffffffu, v, o));
  if constexpr (TPR > 32) {  // one row per CTA
    const int warp = threadIdx.x >> 5;
    float* red = s_red + slot * (TPR / 32);
    if ((threadIdx.x & 31) == 0) red[warp] = v;
    __syncthreads();
    v = red[0];
#pragma unroll
    for (int w = 1; w < TPR / 32; ++w) v = __fadd_rn(v, red[w]);
  }
  return v;
}

template <class OT, class HT, int TPR, int VEC, int NC>
__global__ void __launch_bounds__(TPR > kNormThreads ? TPR : kNormThreads) block_norm_kernel(BlockNormArgs a) {
  constexpr int kRows = TPR >= kNormThreads ? 1 : kNormThreads / TPR;  // rows per CTA
  __shared__ float s_red[TPR > 32 ? 2 * (TPR / 32) : 1];
  const int t = (int)threadIdx.x % TPR;
  const int64_t row = (int64_t)blockIdx.x * kRows + (int)threadIdx.x / TPR;
  if (row >= a.rows) return;  // whole warps (TPR 32), no row for a whole CTA otherwise: the grid covers the rows
  const OT* o = static_cast<const OT*>(a.o) + row * a.ldo;
  const HT* h = static_cast<const HT*>(a.h) + row * a.ldh;
  HT* ho = static_cast<HT*>(a.h_out) + row * a.ldho;
  float vo[NC][VEC], vh[NC][VEC];
#pragma unroll
  for (int c = 0; c < NC; ++c) {
    const int e = (c * TPR + t) * VEC;
    if (e < a.dim) {
      load_vec<VEC>(o + e, vo[c]);
      load_vec<VEC>(h + e, vh[c]);
    } else {
#pragma unroll
      for (int i = 0; i < VEC; ++i) vo[c][i] = vh[c][i] = 0.0f;
    }
  }
  int ad = a.row_adapter ? a.row_adapter[row] : 0;
  if (ad >= a.n_adapters) ad = -1;
  const float* gate = ad >= 0 && a.gates ? a.gates + (int64_t)ad * a.dim : nullptr;
  const float scale = ad >= 0 && a.scales ? a.scales[ad] : 1.0f;
  if (a.post) {
    float s = 0.0f;
#pragma unroll
    for (int c = 0; c < NC; ++c)
#pragma unroll
      for (int i = 0; i < VEC; ++i) s = fmaf(vo[c][i], vo[c][i], s);
    s = row_sum<TPR>(s, s_red, 0);
    const float inv = __frcp_rn(__fsqrt_rn(__fadd_rn(__fdiv_rn(s, (float)a.dim), a.eps)));
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      const int e = (c * TPR + t) * VEC;
      if (e >= a.dim) continue;
      float w[VEC];
      load_vec<VEC>(a.post + e, w);
#pragma unroll
      for (int i = 0; i < VEC; ++i) vo[c][i] = __fmul_rn(__fmul_rn(vo[c][i], inv), w[i]);
    }
  }
  float s = 0.0f;
#pragma unroll
  for (int c = 0; c < NC; ++c) {
    const int e = (c * TPR + t) * VEC;
    if (e >= a.dim) continue;
    if (gate) {
      float g[VEC];
      load_vec<VEC>(gate + e, g);
#pragma unroll
      for (int i = 0; i < VEC; ++i) vo[c][i] = __fmul_rn(vo[c][i], g[i]);
    }
#pragma unroll
    for (int i = 0; i < VEC; ++i) vh[c][i] = fmaf(scale, vh[c][i], vo[c][i]);
    store_vec<VEC>(ho + e, vh[c]);
#pragma unroll
    for (int i = 0; i < VEC; ++i) s = fmaf(vh[c][i], vh[c][i], s);
  }
  if (!a.pre) return;
  s = row_sum<TPR>(s, s_red, 1);
  const float inv = __frcp_rn(__fsqrt_rn(__fadd_rn(__fdiv_rn(s, (float)a.dim), a.eps)));
  OT* y = static_cast<OT*>(a.y) + row * a.ldy;
  float top = 0.0f;
#pragma unroll
  for (int c = 0; c < NC; ++c) {
    const int e = (c * TPR + t) * VEC;
    if (e >= a.dim) continue;
    float w[VEC], v[VEC];
    load_vec<VEC>(a.pre + e, w);
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
      v[i] = __fmul_rn(__fmul_rn(vh[c][i], inv), w[i]);
      top = fmaxf(top, fabsf(v[i]));
    }
    store_vec<VEC>(y + e, v);
  }
  if (a.absmax) {
    top = warp_max(top);
    if ((threadIdx.x & 31) == 0) atomicMax(a.absmax + (a.row_seq ? a.row_seq[row] : 0), __float_as_uint(top));
  }
}

template <class OT, class HT, int TPR, int VEC>
cudaError_t norm_chunks(const BlockNormArgs& a, cudaStream_t st) {
  constexpr int kThreads = TPR > kNormThreads ? TPR : kNormThreads;
  constexpr int kRows = kThreads / TPR, kMost = 32 / VEC;  // 32 elements per thread at most
  const int64_t grid = (a.rows + kRows - 1) / kRows;
  const int nc = ((a.dim + VEC - 1) / VEC + TPR - 1) / TPR;
  if (nc > kMost || grid > 0x7fffffff) return cudaErrorInvalidValue;
  if constexpr (VEC == 1) {
    block_norm_kernel<OT, HT, TPR, 1, kMost><<<(unsigned)grid, kThreads, 0, st>>>(a);
  } else {
    constexpr int q = kMost / 4;
    if (nc <= q) block_norm_kernel<OT, HT, TPR, VEC, q><<<(unsigned)grid, kThreads, 0, st>>>(a);
    else if (nc <= 2 * q) block_norm_kernel<OT, HT, TPR, VEC, 2 * q><<<(unsigned)grid, kThreads, 0, st>>>(a);
    else if (nc <= 3 * q) block_norm_kernel<OT, HT, TPR, VEC, 3 * q><<<(unsigned)grid, kThreads, 0, st>>>(a);
    else block_norm_kernel<OT, HT, TPR, VEC, kMost><<<(unsigned)grid, kThreads, 0, st>>>(a);
  }
  return cudaGetLastError();
}

bool aligned16(const void* p, int64_t ld, int size) {
  return (reinterpret_cast<uintptr_t>(p) & 15) == 0 && (ld * size) % 16 == 0;
}

template <class OT, class HT>
cudaError_t norm_types(const BlockNormArgs& a, cudaStream_t st) {
  constexpr int VEC = 16 / (sizeof(OT) > sizeof(HT) ? sizeof(OT) : sizeof(HT));
  const bool vec = a.dim % VEC == 0 && aligned16(a.o, a.ldo, sizeof(OT)) && aligned16(a.h, a.ldh, sizeof(HT)) &&
                   aligned16(a.h_out, a.ldho, sizeof(HT)) && (!a.y || aligned16(a.y, a.ldy, sizeof(OT)));
  if (a.dim <= 1024) return vec ? norm_chunks<OT, HT, 32, VEC>(a, st) : norm_chunks<OT, HT, 32, 1>(a, st);
  if (a.dim <= 4096) return vec ? norm_chunks<OT, HT, 128, VEC>(a, st) : norm_chunks<OT, HT, 128, 1>(a, st);
  return vec ? norm_chunks<OT, HT, 512, VEC>(a, st) : norm_chunks<OT, HT, 512, 1>(a, st);
}

template <class XT, class YT>
cudaError_t small_types(const LowRankBank& bank, const AdapterPlanDev& plan, int n_tiles, const LowRankArgs& a,
                        cudaStream_t st) {
  const int clusters = n_tiles < 4096 ? n_tiles : 4096;
  lowrank_small_kernel<XT, YT><<<clusters * kSmallCtas, kSmallThreads, 0, st>>>(bank, plan, a);
  return cudaGetLastError();
}

}  // namespace

cudaError_t launch_adapter_plan(const int32_t* pos, const int32_t* row0, const int32_t* seq, const int32_t* adapter,
                                int32_t n_seqs, int32_t rows, int32_t* pos_row, int32_t* pos_seq,
                                int32_t* row_adapter, cudaStream_t stream) {
  if (rows <= 0) return cudaSuccess;
  adapter_plan_kernel<<<(unsigned)(((int64_t)rows + 255) / 256), 256, 0, stream>>>(pos, row0, seq, adapter, n_seqs,
                                                                                   rows, pos_row, pos_seq, row_adapter);
  return cudaGetLastError();
}

cudaError_t launch_lowrank_small(const LowRankBank& bank, const AdapterPlanDev& plan, int n_tiles,
                                 const LowRankArgs& a, cudaStream_t st) {
  if (n_tiles <= 0) return cudaSuccess;
  if (a.xtype == kDtF32 && a.ytype == kDtF32) return small_types<float, float>(bank, plan, n_tiles, a, st);
  if (a.xtype == kDtF16 && a.ytype == kDtF16)
    return small_types<__half, __half>(bank, plan, n_tiles, a, st);
  if (a.xtype == kDtF16 && a.ytype == kDtF32)
    return small_types<__half, float>(bank, plan, n_tiles, a, st);
  if (a.xtype == kDtBF16 && a.ytype == kDtBF16)
    return small_types<__nv_bfloat16, __nv_bfloat16>(bank, plan, n_tiles, a, st);
  if (a.xtype == kDtBF16 && a.ytype == kDtF32)
    return small_types<__nv_bfloat16, float>(bank, plan, n_tiles, a, st);
  return cudaErrorInvalidValue;
}

cudaError_t launch_block_norm(const BlockNormArgs& a, cudaStream_t st) {
  if (a.rows <= 0) return cudaSuccess;
  if (a.dtype == kDtF32 && a.htype == kDtF32) return norm_types<float, float>(a, st);
  if (a.dtype == kDtF16 && a.htype == kDtF16) return norm_types<__half, __half>(a, st);
  if (a.dtype == kDtF16 && a.htype == kDtF32) return norm_types<__half, float>(a, st);
  if (a.dtype == kDtBF16 && a.htype == kDtBF16) return norm_types<__nv_bfloat16, __nv_bfloat16>(a, st);
  if (a.dtype == kDtBF16 && a.htype == kDtF32) return norm_types<__nv_bfloat16, float>(a, st);
  return cudaErrorInvalidValue;
}

}  // namespace sem
