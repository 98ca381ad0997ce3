// Adapters of many requests (sm_100a): the plan's row maps, the low-rank
// adapters of small calls on CUDA cores, and the block norm with its gate and
// residual scale. The tensor-core kernel is lowrank_tc.cu.
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

// Eight consecutive weights (16-byte aligned) in two steps, so that the loads are on their way while other work
// is done: the bytes, then the values. WT: float, or any 16-bit type (bf16 or
// fp16 by wtype).
template <class WT>
struct RawWeights8 {
  uint4 q[sizeof(WT) == 4 ? 2 : 1];
};
template <class WT>
__device__ __forceinline__ void fetch_weights8(const void* base, int64_t at, RawWeights8<WT>& r) {
  const uint4* p = reinterpret_cast<const uint4*>(static_cast<const WT*>(base) + at);
  r.q[0] = p[0];
  if constexpr (sizeof(WT) == 4) r.q[1] = p[1];
}
template <class WT>
__device__ __forceinline__ void weights8(const RawWeights8<WT>& r, int wtype, float (&v)[8]) {
  if constexpr (sizeof(WT) == 4) {
    const uint32_t w[8] = {r.q[0].x, r.q[0].y, r.q[0].z, r.q[0].w, r.q[1].x, r.q[1].y, r.q[1].z, r.q[1].w};
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = __uint_as_float(w[i]);
  } else {
    const uint32_t w[4] = {r.q[0].x, r.q[0].y, r.q[0].z, r.q[0].w};
    if (wtype == kDtBF16) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        v[2 * i] = __uint_as_float(w[i] << 16);
        v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
      }
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
        v[2 * i] = f.x;
        v[2 * i + 1] = f.y;
      }
    }
  }
}

// ---------------------------------------------------------------------------
// Low-rank adapters on CUDA cores
// ---------------------------------------------------------------------------
// A unit is up to 16 rows of one adapter. A cluster of two, four or eight CTAs
// takes it: each CTA sums its share of the input channels into a partial t =
// x A^T and writes it to every CTA of the cluster (distributed shared memory);
// after one cluster barrier each adds the partials in the same order and
// finishes its share of the output channels. One launch, no workspace, and two
// short dependent load phases (A, then B, which is fetched before the barrier
// with base) where one SM would walk both weights: what a few rows cost is
// latency. The shares do not go by the batch (a row's sums are the same for
// any cluster size: the input channels are cut in eight, and a CTA of a
// smaller cluster sums several of the eight one after the other). Float32 FMA
// throughout. Bound by that latency (per call of a CUDA graph): 12 float32 rows,
// 768 x 768, rank 8, 5.5 us. One fp16 unit of rank 16 takes 6.3 us at 768 x 256,
// 7.4 at 768 x 1280, 8.6 at 768 x 2304 (a thread's second and third round of
// output channels wait for base and B), 48 at once 7.9, 10.0 and 12.3. 48
// sequences of 1 to 24 fp16 rows, each with an adapter of its own, 768 x 1280,
// rank to 16, 12.9 us: 63 units, more than clusters of eight fit.
constexpr int kSmallParts = 8, kSmallThreads = 256, kSmallWarps = kSmallThreads / 32;
constexpr int kSmallChunk = 128, kSmallLd = kSmallChunk + 4;  // input channels staged at a time, padded (banks)
constexpr int kSmallRows = kAdapterSmallRows;
static_assert(kSmallRows == 16, "a thread's row is its lane modulo 16");

inline __host__ __device__ constexpr int small_smem_floats(int max_rank) {  // x, A, the partials of two units in turn, t
  return (kSmallRows + max_rank) * kSmallLd + 2 * kSmallParts * kSmallRows * max_rank + kSmallRows * ((max_rank + 7) & ~7);
}

// Eight consecutive values, of which those from `n` on are zero; `vec`: 16-byte
// aligned in memory (all of it is read then only if n >= 8).
template <class T>
__device__ __forceinline__ void load_row8(const T* p, int n, bool vec, float (&v)[8]) {
  if (vec && n >= 8) {
    if constexpr (sizeof(T) == 4) {
      const float4 a = *reinterpret_cast<const float4*>(p), b = *reinterpret_cast<const float4*>(p + 4);
      v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w, v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
    } else {
      load_vec<8>(p, v);
    }
  } else {
    T e[8];  // all loads first: a condition or conversion in between would make each wait for the one before
#pragma unroll
    for (int i = 0; i < 8; ++i) e[i] = p[min(i, n - 1)];
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = i < n ? to_f32(e[i]) : 0.0f;
  }
}

// RU: ranks per warp at most (ranks up to 8 RU).
template <class XT, class YT, class WT, int RU>
__global__ void __launch_bounds__(kSmallThreads, RU <= 4 ? 3 : 2)
    lowrank_small_kernel(LowRankBank bank, AdapterPlanDev plan, LowRankArgs a, int x_vec) {
  extern __shared__ __align__(16) float smem[];
  float* s_x = smem;                                   // [16][kSmallLd]
  float* s_a = s_x + kSmallRows * kSmallLd;            // [rank][kSmallLd]
  float* s_part = s_a + bank.max_rank * kSmallLd;      // [2][eighth][16 * rank]
  float* s_t = s_part + 2 * kSmallParts * kSmallRows * bank.max_rank;  // [rank][16]
  __shared__ int32_t s_row[kSmallRows];
  __shared__ float s_scale[kSmallRows];
  cg::cluster_group cluster = cg::this_cluster();
  const int cta = (int)cluster.block_rank(), ctas = (int)cluster.num_blocks(), tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const XT* x = static_cast<const XT*>(a.x);
  const YT* base = static_cast<const YT*>(a.base);
  YT* y = static_cast<YT*>(a.y);
  // an eighth of the input channels (a multiple of 8), this CTA's output channels (an even number)
  const int kper = ((bank.k_in + kSmallParts - 1) / kSmallParts + 7) & ~7;
  const int nper = ((bank.n_out + ctas - 1) / ctas + 1) & ~1;
  const int n0 = min(bank.n_out, cta * nper), n1 = min(bank.n_out, n0 + nper);
  constexpr int kSubs = kAdapterTileRows / kSmallRows;  // units of a large tile
  const bool in_place = a.base == a.y && a.ldb == a.ldy;
  int set = 0;
  bool started = false;  // every CTA of the cluster runs: its shared memory can be written
  cluster.barrier_arrive();
  const AdapterTile first = plan.small[min((int)(blockIdx.x / ctas), plan.max_seqs)];  // without waiting for the count
  const int n_small = plan.counts[1], n_units = n_small + plan.counts[0] * kSubs;

  for (int u = (int)(blockIdx.x / ctas); u < n_units; u += (int)(gridDim.x / ctas)) {
    AdapterTile tl = first;
    int sub = 0;
    if (u >= n_small) {
      tl = plan.large[(u - n_small) / kSubs];
      sub = (u - n_small) % kSubs * kSmallRows;
    } else if (u != (int)(blockIdx.x / ctas)) {
      tl = plan.small[u];
    }
    const int rows = min(kSmallRows, tl.rows - sub);
    if (rows <= 0) continue;  // the whole cluster
    LowRankAdapter ad{};
    if (tl.adapter >= 0 && tl.adapter < bank.n_adapters) ad = bank.adapters[tl.adapter];
    if (ad.rank == 0 && in_place) continue;  // nothing to add (the whole cluster)
    __syncthreads();  // the previous unit's rows, scales and t are read
    if (tid < kSmallRows) {
      const int r = sub + min(tid, rows - 1);  // rows behind the last one repeat it and are not stored
      s_row[tid] = tl.row0 >= 0 ? tl.row0 + r : plan.pos_row[tl.pos0 + r];
      float sc = ad.scale;
      if (a.absmax)
        sc = __fmul_rn(sc, __fdiv_rn(__uint_as_float(a.absmax[a.per_seq ? plan.pos_seq[tl.pos0 + r] : 0]), 127.0f));
      s_scale[tid] = sc;
    }
    __syncthreads();
    if (ad.rank == 0) {  // base as it is: adding a zero would change the sign of a zero and the bits of a NaN
      for (int r = warp; r < rows; r += kSmallWarps) {
        const int64_t row = s_row[r];
        for (int c = n0 + lane; c < n1; c += 128) {  // four loads in flight
          YT v[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) v[i] = base ? base[row * a.ldb + min(c + 32 * i, n1 - 1)] : from_f32<YT>(0.0f);
#pragma unroll
          for (int i = 0; i < 4; ++i)
            if (c + 32 * i < n1) y[row * a.ldy + c + 32 * i] = v[i];
        }
      }
      continue;  // the whole cluster
    }
    float* part = s_part + set * kSmallParts * kSmallRows * bank.max_rank;
    const int size = ad.rank * kSmallRows;
    // a thread: four rows of a pair of output channels; base and the first ranks of B are on their way while t is summed
    const int items = (n1 - n0 + 1) / 2 * (kSmallRows / 4);
    const int q = tid & 3;  // its rows 4 q ..
    YT b[2][4];
    RawWeights8<WT> w[2];
    auto fetch = [&](int item) {
      const int ch = n0 + item / 4 * 2;
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int c = min(ch + e, n1 - 1);
#pragma unroll
        for (int i = 0; i < 4; ++i)
          b[e][i] = base ? base[(int64_t)s_row[q * 4 + i] * a.ldb + c] : from_f32<YT>(0.0f);
        fetch_weights8(ad.b, (int64_t)c * ad.rp, w[e]);
      }
    };
    if (tid < items) fetch(tid);
    // a thread: one row (lane % 16), half of each chunk's channels (lane / 16), every eighth rank
    for (int eighth = cta; eighth < kSmallParts; eighth += ctas) {
      const int k0 = min(bank.k_in, eighth * kper), k1 = min(bank.k_in, k0 + kper);
      float acc[RU];
#pragma unroll
      for (int i = 0; i < RU; ++i) acc[i] = 0.0f;
      for (int kc = k0; kc < k1; kc += kSmallChunk) {
        const int kn = min(kSmallChunk, k1 - kc), oct = (kn + 7) / 8;
        if (eighth != cta || kc > k0) __syncthreads();
        auto put = [&](int r, int c, const float (&v)[8]) {
          float4* d = reinterpret_cast<float4*>(s_x + r * kSmallLd + c);
          d[0] = make_float4(v[0], v[1], v[2], v[3]);
          d[1] = make_float4(v[4], v[5], v[6], v[7]);
        };
        // x is one piece per thread at most; the first of A's is loaded before it is waited for
        const int r = tid / oct, c = tid % oct * 8;
        float vx[8], va[8];
        auto load_a = [&](int j, int ca) {  // zeros behind k_in
          RawWeights8<WT> raw;
          fetch_weights8(ad.a, (int64_t)j * bank.ka + kc + ca, raw);
          weights8(raw, bank.wtype, va);
        };
        if (r < kSmallRows) load_row8(x + (int64_t)s_row[r] * a.ldx + kc + c, kn - c, x_vec != 0, vx);
        if (r < ad.rank) load_a(r, c);
        if (r < kSmallRows) put(r, c, vx);
        if (r < ad.rank) put(kSmallRows + r, c, va);
        for (int i = tid + kSmallThreads; i < ad.rank * oct; i += kSmallThreads) {
          load_a(i / oct, i % oct * 8);
          put(kSmallRows + i / oct, i % oct * 8, va);
        }
        __syncthreads();
        const float* xr = s_x + (lane & 15) * kSmallLd;
#pragma unroll 4
        for (int c = (lane >> 4) * 4; c < oct * 8; c += 8) {
          const float4 v = *reinterpret_cast<const float4*>(xr + c);
#pragma unroll
          for (int i = 0; i < RU; ++i) {  // ranks there are not: the last one again
            const float4 w4 = *reinterpret_cast<const float4*>(s_a + min(warp + i * kSmallWarps, ad.rank - 1) * kSmallLd + c);
            acc[i] = fmaf(v.x, w4.x, fmaf(v.y, w4.y, fmaf(v.z, w4.z, fmaf(v.w, w4.w, acc[i]))));
          }
        }
      }
      if (!started) cluster.barrier_wait();
      started = true;
#pragma unroll
      for (int i = 0; i < RU; ++i) {
        const int j = warp + i * kSmallWarps;
        if (j >= ad.rank) break;
        const float v = __fadd_rn(acc[i], __shfl_xor_sync(0xffffffffu, acc[i], 16));
        // both halves of the lanes hold the sum: each sends it to half of the CTAs
        float* mine = part + eighth * size + j * kSmallRows + (lane & 15);
        for (int d = lane >> 4; d < ctas; d += 2) *cluster.map_shared_rank(mine, d) = v;
      }
    }
    cluster.sync();
    // The sets of partials take turns over the units that have this barrier: a set is written again only behind the
    // next such unit's barrier, which every CTA reaches with its sums below done. (A unit of rank 0 must not count:
    // the third unit's partials would land in a set that a slower CTA still sums.)
    set ^= 1;
    for (int i = tid; i < ad.rp * kSmallRows; i += kSmallThreads) {
      float v = 0.0f;
      if (i < size) {
#pragma unroll
        for (int c = 0; c < kSmallParts; ++c) v = __fadd_rn(v, part[c * size + i]);
        v = __fmul_rn(v, s_scale[i & 15]);
      }
      s_t[i] = v;  // zeros for the columns of B behind the rank
    }
    __syncthreads();
    for (int item = tid; item < items; item += kSmallThreads) {
      if (item != tid) fetch(item);
      const int ch = n0 + item / 4 * 2;
      float o[2][4];
#pragma unroll
      for (int i = 0; i < 4; ++i) o[0][i] = o[1][i] = 0.0f;
      for (int j = 0; j < ad.rp; j += 8) {
        RawWeights8<WT> nw[2];
        if (j + 8 < ad.rp) {
#pragma unroll
          for (int e = 0; e < 2; ++e)
            fetch_weights8(ad.b, (int64_t)min(ch + e, n1 - 1) * ad.rp + j + 8, nw[e]);
        }
        float f[2][8];
        weights8(w[0], bank.wtype, f[0]);
        weights8(w[1], bank.wtype, f[1]);
#pragma unroll
        for (int v = 0; v < 8; ++v) {
          const float4 t = *reinterpret_cast<const float4*>(s_t + (j + v) * kSmallRows + q * 4);
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            o[e][0] = fmaf(t.x, f[e][v], o[e][0]);
            o[e][1] = fmaf(t.y, f[e][v], o[e][1]);
            o[e][2] = fmaf(t.z, f[e][v], o[e][2]);
            o[e][3] = fmaf(t.w, f[e][v], o[e][3]);
          }
        }
        w[0] = nw[0], w[1] = nw[1];
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if (q * 4 + i >= rows) break;
        YT* d = y + (int64_t)s_row[q * 4 + i] * a.ldy + ch;
        d[0] = from_f32<YT>(__fadd_rn(to_f32(b[0][i]), o[0][i]));
        if (ch + 1 < n1) d[1] = from_f32<YT>(__fadd_rn(to_f32(b[1][i]), o[1][i]));
      }
    }
  }
  if (!started) cluster.barrier_wait();
  cluster.sync();  // no CTA leaves while another may still write to it
}

// ---------------------------------------------------------------------------
// Block norm
// ---------------------------------------------------------------------------
// TPR threads hold one row in registers, NC chunks of VEC elements each, so o
// and h are read once and h_out and y written once; the two sums of squares
// are float32 partial sums joined by a fixed tree. Bound by HBM: 131072 float32
// rows of 768 take 240 us, the rate of a plain copy; fp16 or bf16 rows over a
// float32 residual 191 us (184 at that rate), over a 16-bit one 155 us (123).
// Rows without alignment go by single elements: 10599 rows of 1153, fp16 over a
// float32 residual, 32 us (18.6 at the copy's rate).
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

// A warp per row: gate and up read once, h written once, bound by HBM.
__global__ void __launch_bounds__(128) gelu_up_kernel(const float* __restrict__ gu, int64_t rows, int F,
                                                      const int32_t* __restrict__ row_seq, float* __restrict__ h,
                                                      uint32_t* __restrict__ absmax) {
  const int64_t row = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 5);
  if (row >= rows) return;
  const float* g = gu + row * 2 * F;
  float top = 0.0f;
  for (int c = (threadIdx.x & 31) * 4; c < F; c += 128) {  // F is a multiple of 128
    float a[4], b[4];
    load_vec<4>(g + c, a);
    load_vec<4>(g + F + c, b);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      a[i] = __fmul_rn(gelu_quick_ref(a[i]), b[i]);
      top = fmaxf(top, fabsf(a[i]));
    }
    store_vec<4>(h + row * F + c, a);
  }
  top = warp_max(top);
  if ((threadIdx.x & 31) == 0) atomicMax(absmax + row_seq[row], __float_as_uint(top));
}

template <class OT, class HT, int TPR, int VEC>
cudaError_t norm_chunks(const BlockNormArgs& a, cudaStream_t st) {
  constexpr int kThreads = TPR > kNormThreads ? TPR : kNormThreads;
  constexpr int kRows = kThreads / TPR;
  constexpr int kMost = (VEC == 1 && TPR < 512 ? 16 : 32) / VEC;  // elements per thread at most: 32, or 16 single ones
  const int64_t grid = (a.rows + kRows - 1) / kRows;
  const int nc = ((a.dim + VEC - 1) / VEC + TPR - 1) / TPR;
  if (nc > kMost || grid > 0x7fffffff) return cudaErrorInvalidValue;
  constexpr int q = kMost / 4;
  if (nc <= q) block_norm_kernel<OT, HT, TPR, VEC, q><<<(unsigned)grid, kThreads, 0, st>>>(a);
  else if (nc <= 2 * q) block_norm_kernel<OT, HT, TPR, VEC, 2 * q><<<(unsigned)grid, kThreads, 0, st>>>(a);
  else if (nc <= 3 * q) block_norm_kernel<OT, HT, TPR, VEC, 3 * q><<<(unsigned)grid, kThreads, 0, st>>>(a);
  else block_norm_kernel<OT, HT, TPR, VEC, kMost><<<(unsigned)grid, kThreads, 0, st>>>(a);
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
  if (vec) {
    if (a.dim <= 1024) return norm_chunks<OT, HT, 32, VEC>(a, st);
    if (a.dim <= 4096) return norm_chunks<OT, HT, 128, VEC>(a, st);
    return norm_chunks<OT, HT, 512, VEC>(a, st);
  }
  if (a.dim <= 512) return norm_chunks<OT, HT, 32, 1>(a, st);
  if (a.dim <= 2048) return norm_chunks<OT, HT, 128, 1>(a, st);
  return norm_chunks<OT, HT, 512, 1>(a, st);
}

template <class XT, class YT, class WT, int RU>
cudaError_t small_ranks(const LowRankBank& bank, const AdapterPlanDev& plan, int n_units,
                        const LowRankArgs& a, cudaStream_t st) {
  const int smem = small_smem_floats(bank.max_rank) * 4;
  // The function's limit is set to the same value whatever the bank (its largest rank's need): another thread may set
  // it between this call's setting and its launch.
  constexpr int kMost = small_smem_floats(RU * kSmallWarps) * 4;
  if constexpr (kMost > 48 * 1024) {
    const cudaError_t e =
        cudaFuncSetAttribute(lowrank_small_kernel<XT, YT, WT, RU>, cudaFuncAttributeMaxDynamicSharedMemorySize, kMost);
    if (e != cudaSuccess) return e;
  }
  // The largest clusters that are all on the device at once. CTAs per SM: three, two at ranks above 32, one where their
  // shared memory is above half of an SM's (ranks above 65). By these, 15, 33 or 48 clusters of eight run at once, and
  // 33 per CTA and SM of four (a cluster leaves some of a processing cluster's SMs unused). One more unit, float32
  // rows, 768 x 768, on eights in two waves / on fours: 49 of rank 16 13.3 / 10.7 us,
  // 16 of rank 128 33.8 / 30.1, 33 of rank 128 50.7 / 31.0. One less on eights: 48 of rank 16 8.6, 33 of rank 64 16.1,
  // 15 of rank 128 18.0 us.
  constexpr int kEights[3] = {15, 33, 48};
  const int fit = 227 * 1024 / (smem + 1024), most = RU <= 4 ? 3 : 2, per_sm = fit < most ? fit : most;
  const int ctas = n_units <= kEights[per_sm - 1] ? 8 : n_units <= 33 * per_sm ? 4 : 2;
  const int clusters = n_units < 2048 ? n_units : 2048;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)(clusters * ctas));
  cfg.blockDim = dim3(kSmallThreads);
  cfg.dynamicSmemBytes = (size_t)smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = (unsigned)ctas;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, lowrank_small_kernel<XT, YT, WT, RU>, bank, plan, a,
                            aligned16(a.x, a.ldx, sizeof(XT)) ? 1 : 0);
}
template <class XT, class YT>
cudaError_t small_types(const LowRankBank& bank, const AdapterPlanDev& plan, int n_units,
                        const LowRankArgs& a, cudaStream_t st) {
  auto pick = [&](auto w) {
    using WT = decltype(w);
    if (bank.max_rank <= 16) return small_ranks<XT, YT, WT, 2>(bank, plan, n_units, a, st);
    if (bank.max_rank <= 32) return small_ranks<XT, YT, WT, 4>(bank, plan, n_units, a, st);
    return small_ranks<XT, YT, WT, 16>(bank, plan, n_units, a, st);
  };
  return bank.wtype == kDtF32 ? pick(float()) : pick(uint16_t());
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

cudaError_t launch_lowrank_small(const LowRankBank& bank, const AdapterPlanDev& plan, int n_large, int n_small,
                                 const LowRankArgs& a, cudaStream_t st) {
  const int64_t units = (int64_t)n_small + (int64_t)n_large * (kAdapterTileRows / kSmallRows);
  if (units <= 0) return cudaSuccess;
  const int n = units < 0x7fffffff ? (int)units : 0x7fffffff;
  if (a.xtype == kDtF32 && a.ytype == kDtF32) return small_types<float, float>(bank, plan, n, a, st);
  if (a.xtype == kDtF16 && a.ytype == kDtF16) return small_types<__half, __half>(bank, plan, n, a, st);
  if (a.xtype == kDtF16 && a.ytype == kDtF32) return small_types<__half, float>(bank, plan, n, a, st);
  if (a.xtype == kDtBF16 && a.ytype == kDtBF16)
    return small_types<__nv_bfloat16, __nv_bfloat16>(bank, plan, n, a, st);
  if (a.xtype == kDtBF16 && a.ytype == kDtF32)
    return small_types<__nv_bfloat16, float>(bank, plan, n, a, st);
  return cudaErrorInvalidValue;
}

cudaError_t launch_gelu_up(const float* gu, int64_t rows, int F, const int32_t* row_seq, float* h, uint32_t* absmax,
                           cudaStream_t st) {
  if (rows <= 0) return cudaSuccess;
  if (F % 128 || (rows + 3) / 4 > 0x7fffffff) return cudaErrorInvalidValue;
  gelu_up_kernel<<<(unsigned)((rows + 3) / 4), 128, 0, st>>>(gu, rows, F, row_seq, h, absmax);
  return cudaGetLastError();
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
