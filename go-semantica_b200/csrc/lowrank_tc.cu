// Low-rank adapters on the sm_100a tensor cores.
//
//   y[row] = base[row] + s (x[row] A^T) B^T
//
// A unit is up to RT rows of one adapter (and a share of the output channels
// when there are few rows). The shrink t = x A^T has the rows on the M lanes
// and the ranks on N; the expand D = B t^T has output channels on the lanes
// and the rows on N, so that the epilogue's threads read base and write y
// along the channels of a row, coalesced. Two expand accumulators hold the
// even and the odd channels of 256: a thread owns two neighbours.
//
// Numbers. Every value goes in as the parts that give at least 21 bits (22 of a
// float32's 24), and the products of parts (all but those below 2^-22) are
// accumulated in float32 in TMEM. Shrink of float32 rows: tf32 (11
// bits), x and float32 weights as hi + lo. Shrink of 16-bit rows (and INT8
// codes held as fp16): kind::f16 on the rows as they are, A in x's type: one
// part where the types are the same, else two bf16 parts of fp16, three bf16
// parts of float32, or two fp16 parts of a rank's weights scaled by a power of
// two (undone in t). Expand: tf32, t as hi + lo, B as stored or hi + lo. The
// tensor core cuts its sums instead of rounding them, which is most of the error:
// float32 rows of 768 values, rank 4 to 104, 1.1e-7 to 2.9e-7 of y's size, where
// float32 products and sums with rounding (the CUDA-core kernel) are 4e-8 off.
//
// Bound by HBM at the ranks in use: a row moves k |x| + 2 n |y| bytes and
// needs 2 r (k + n) flops (r = 16, 768 x 768, float32: 9.2 KB against 49
// kflop, two products each: 0.02 of the tensor pipe). So the work is to keep
// loads in flight and every other role short:
//   - X warps (8): rows of x to where their operand goes, 128-byte swizzled:
//     by TMA where a whole unit's rows follow each other, by asynchronous
//     copies otherwise (any order and alignment); float32 is then split there;
//   - two copy threads: the adapter's A and B tiles, which the bank keeps in
//     the swizzled layout, a bulk copy per piece (and the TMA of float32 x);
//   - a shrink and an expand MMA thread, so that the shrink of later units
//     goes on while the epilogue holds up the expand of an earlier one;
//   - T warps (2): t from TMEM, scaled, split, to shared memory;
//   - a unit warp: what to do next, looked up ahead for all the others;
//   - epilogue warps (16): base by asynchronous copies into a ring per warp,
//     ahead of the accumulators and across units.
// One persistent CTA per SM. Per call (device time; bytes at 6.56 TB/s, the
// rate of a plain copy, in parentheses):
//   65536 float32 rows, 768 x 768, rank 16:             113 us (92)
//   196608 rows of codes, 1152 x 768, rank 32:          280 to 300 us (253)
//   110213 ragged bf16 rows, 768 x 2304, rank to 64:    287 us (181)
//   16384 fp16 rows, 768 x 1280, rank 128, f32 weights:  93 us (17)
//   6075 ragged float32 rows, 517 x 1001, rank to 23:    35 us (9)
// The first two are near the copy's rate. In the third a unit reads 0.6 MB of
// B from L2 beside its 0.7 MB of rows, in the fourth 1.7 beside 0.4: weights
// in wide planes for tiles of 64 rows are what larger ranks pay. The last has
// no TMA for its rows: copies of 4 bytes and single stores, in one unit per SM.
#include <cuda_bf16.h>

#include <type_traits>

#include "common.cuh"
#include "kernels.h"
#include "sm100.cuh"
#include "tmap.h"

namespace sem {

namespace {

constexpr int kXWarps = 8, kXGroups = 2, kEpiWarps = 16, kTWarps = 2;
constexpr int kWarpEpi = kXWarps, kWarpT = kWarpEpi + kEpiWarps, kWarpShrink = kWarpT + kTWarps;
constexpr int kWarpA = kWarpShrink + 1, kWarpExpand = kWarpA + 1, kWarpB = kWarpExpand + 1, kWarpUnits = kWarpB + 1;
constexpr int kThreads = (kXWarps + kEpiWarps + 8) * 32;  // the last warpgroups: T, MMA, copy and unit warps, one idle
// Registers: 1024 threads get 64 each at launch; the last two warpgroups (and
// the X warps of 16-bit rows, which split nothing) give some back to the
// epilogue's. The shared memory leaves the L1 too small for spills: with
// 12 to 60 bytes of them (72, 72 and 40 registers) 110213 bf16 rows,
// 768 x 2304, rank to 64, took 365 us and takes 306 without.
template <class XT>
struct Regs {
  static constexpr int x = sizeof(XT) == 4 ? 64 : 48, epi = sizeof(XT) == 4 ? 72 : 80, rest = 48;
  static_assert(kXWarps * x + kEpiWarps * epi + 8 * rest <= kThreads / 32 * 64, "register split");
};
static_assert(kThreads == 1024, "64 registers at launch");
static_assert(kWarpEpi % 4 == 0 && kWarpT % 4 == 0, "TMEM lane quarters go by warp index");
constexpr int KC = 32;   // tf32 per swizzled 128-byte row
constexpr int kRt = 64;  // rows per unit at most
static_assert(kRt == kAdapterTileRows && kRt <= kTWarps * 32, "a unit is a tile or a part of one");
constexpr int kMaxSlots = 8;
constexpr int kBPlane = 128 * 128;  // one plane of a slot of B: 128 channels x 128 bytes
constexpr int kMiscBytes = 1792;
constexpr int kMaxSmem = 232448;  // an MMA reads 128 rows from a slot's start: a short slot's run on into sW and sT

__device__ uint32_t g_lowrank_error;

// kind::tf32, both operands K-major, float32 accumulator.
__host__ __device__ constexpr uint32_t idesc_tf32(int M, int N) {
  return (1u << 4) | (2u << 7) | (2u << 10) | ((uint32_t)(N >> 3) << 17) | ((uint32_t)(M >> 4) << 24);
}
// One lane of a converged warp. Unlike a test of the lane number it tells the
// compiler that a single thread goes on, which the operands of an MMA or a TMA
// copy need: 30 instead of 110 cycles to issue an MMA.
__device__ __forceinline__ bool elect_lane() {
  uint32_t p;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "elect.sync _|p, 0xffffffff;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}\n"
      : "=r"(p));
  return p != 0;
}
// kind::f16, fp16 (0) or bf16 (1) operands.
__host__ __device__ constexpr uint32_t idesc_16(int fmt, int M, int N) {
  return (1u << 4) | ((uint32_t)fmt << 7) | ((uint32_t)fmt << 10) | ((uint32_t)(N >> 3) << 17) |
         ((uint32_t)(M >> 4) << 24);
}
__device__ __forceinline__ void umma_tf32(uint32_t d_tmem, uint64_t adesc, uint64_t bdesc, uint32_t idesc,
                                          uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::tf32 [%0], %1, %2, %3, p;\n\t}\n" ::"r"(d_tmem),
      "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate)
      : "memory");
}
// The low word of a K-major 128-byte-swizzled operand's descriptor at shared
// address `a`; its high word is the same for all. One thread issues every MMA,
// so its instructions per MMA set their rate: moving 32 bytes (one K step)
// along a row is + 2 on the low word.
__device__ __forceinline__ uint32_t desc_lo(uint32_t a) { return ((a & 0x3FFFFu) >> 4) | 1u << 16; }
constexpr uint32_t kDescHi = (1024u >> 4) | 1u << 14 | 2u << 29;
__device__ __forceinline__ uint64_t desc_at(uint32_t lo) { return pack2u(lo, kDescHi); }

// A position in a ring of slots: the slot and the parity of its use.
struct Ring {
  uint32_t slot = 0, parity = 0;
  __device__ __forceinline__ void next(uint32_t slots) {
    if (++slot == slots) slot = 0, parity ^= 1;
  }
};

// Contiguous copy global -> shared, completing as transaction bytes on bar.
// Both addresses and the size are multiples of 16 bytes.
__device__ __forceinline__ void bulk_load(void* dst, const void* src, uint32_t bytes, uint64_t* bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(
                   smem_u32(dst)),
               "l"(src), "r"(bytes), "r"(smem_u32(bar))
               : "memory");
}

// mbar_wait's contract (bounded, gives up when another thread has); the clock
// is the SM's own and read only once a wait is long.
constexpr long long kWaitCycles = 4000000000ll;  // 2 s at 2 GHz
__device__ __forceinline__ bool stage_wait(uint64_t* bar, uint32_t parity, volatile int* abort_flag, uint32_t* err,
                                           uint32_t code) {
  const uint32_t a = smem_u32(bar);
  long long t0 = 0;
  for (uint32_t n = 1; !mbar_try_wait(a, parity); ++n) {
    if (n & 255) continue;
    if (*abort_flag) return false;
    const long long t = clock64();
    if (!t0) t0 = t;
    if (t - t0 > kWaitCycles) {
      *abort_flag = 1;
      atomicOr(err, code);
      return false;
    }
  }
  return true;
}

// A whole warp's wait: the same answer in every lane (each lane's own wait is
// bounded), so that a warp leaves its loop as one.
__device__ __forceinline__ bool warp_wait(uint64_t* bar, uint32_t parity, volatile int* abort_flag, uint32_t* err,
                                          uint32_t code) {
  return __all_sync(0xffffffffu, stage_wait(bar, parity, abort_flag, err, code));
}

// Asynchronous copies global -> shared: 16 bytes of which the first `bytes`
// come from memory (the rest are zeros), or 4 bytes.
__device__ __forceinline__ void copy16(uint32_t dst, const void* src, int bytes) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void copy4(uint32_t dst, const void* src, int bytes) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
// All but the last n of this thread's copy groups are complete (n < 6).
__device__ __forceinline__ void copy_wait(int n) {
  switch (n) {
    case 0: cp_async_wait<0>(); break;
    case 1: cp_async_wait<1>(); break;
    case 2: cp_async_wait<2>(); break;
    case 3: cp_async_wait<3>(); break;
    case 4: cp_async_wait<4>(); break;
    default: cp_async_wait<5>(); break;
  }
}

// v = hi + lo: hi the upper 11 significant bits; lo's bits behind its own 11
// are cut too: an operand is a tf32 value. An infinite v is hi, and NaN in lo.
// (The sum makes a NaN a quiet one, which the cut cannot turn into an infinity.)
__device__ __forceinline__ void split_tf32(float v, float& hi, float& lo) {
  v = __fadd_rn(v, 0.0f);
  hi = __uint_as_float(__float_as_uint(v) & 0xffffe000u);
  lo = __uint_as_float(__float_as_uint(__fsub_rn(v, hi)) & 0xffffe000u);
}
// The same with lo = 0 for an infinite v (and a NaN).
__device__ __forceinline__ void split_tf32_lo_finite(float v, float& hi, float& lo) {
  split_tf32(v, hi, lo);
  lo = lo == lo ? lo : 0.0f;
}

template <class T>
__device__ __forceinline__ float as_f32(T v) {
  if constexpr (std::is_same<T, float>::value) return v;
  else if constexpr (std::is_same<T, __half>::value) return __half2float(v);
  else return __bfloat162float(v);
}
template <class T>
__device__ __forceinline__ T as_type(float v) {
  if constexpr (std::is_same<T, float>::value) return v;
  else if constexpr (std::is_same<T, __half>::value) return __float2half_rn(v);
  else return __float2bfloat16_rn(v);
}

template <class T>
__device__ __forceinline__ uint32_t raw_bits(T v) {
  if constexpr (sizeof(T) == 4) return __float_as_uint(v);
  else return *reinterpret_cast<const uint16_t*>(&v);
}
template <class T>
__device__ __forceinline__ T from_bits(uint32_t b) {
  if constexpr (sizeof(T) == 4) {
    return __uint_as_float(b);
  } else {
    const uint16_t h = (uint16_t)b;
    return *reinterpret_cast<const T*>(&h);
  }
}

// 32 lanes x 8 columns of TMEM.
__device__ __forceinline__ void tmem_ld8(uint32_t taddr, uint32_t (&r)[8]) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7])
               : "r"(taddr));
}
__device__ __forceinline__ void reg_barrier8(uint32_t (&r)[8]) {
  asm volatile(""
               : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7])
               :
               : "memory");
}

// The 256 TMEM columns of t's accumulators. The tensor core cuts every sum it
// forms, an error that grows with the number of sums into one accumulator and
// with its size; so the products run into up to four accumulators (the low
// parts into one of their own, the stages of k over the others), which the T
// warps add with rounding. Banks of ranks up to 64 have two sets in turn.
struct ShrinkAcc {
  int bufs, width, hi_parts, parts;
  __device__ __forceinline__ ShrinkAcc(int max_rank, int rank, bool low, int k_stages) {
    bufs = max_rank <= 64 ? 2 : 1;
    width = (rank + 15) & ~15;  // N of the product: a multiple of 16
    parts = min(4, 256 / bufs / width);
    hi_parts = min(low ? parts - 1 : parts, k_stages);
    parts = hi_parts + (low ? 1 : 0);
  }
};

// What a CTA does next. The unit warp looks it up (32 units at a time, so that
// the dependent loads of tile and adapter cost no role anything) and passes it
// on through a ring in shared memory; the last entry has no rows.
struct alignas(16) Unit {
  const uint8_t* ta;     // A's tiles for this x
  const uint8_t* tb;
  const float* unscale;  // factors of t's ranks, or null
  int32_t pos0, rows;  // positions
  int32_t row0;        // their rows follow each other from here, or -1
  int32_t c0, c1;      // chunks of 256 output channels
  int32_t rank, rp;    // rank 0: y = base
  float scale;
};
constexpr int kUnitSlots = 8;  // above the four units that an epilogue warp's copies can be ahead of its stores
constexpr int kUnitReaders = kXWarps + kEpiWarps + kTWarps + 4;

// Parts of A for x of type XT and weights of type wtype.
__host__ __device__ constexpr int a_parts(int xtype, int wtype) {
  return xtype == kDtF32 ? (wtype == kDtF32 ? 2 : 1) : xtype == wtype ? 1 : xtype == kDtBF16 && wtype == kDtF32 ? 3 : 2;
}
template <class XT>
__host__ __device__ constexpr int dtype_of() {
  return std::is_same<XT, float>::value ? kDtF32 : std::is_same<XT, __half>::value ? kDtF16 : kDtBF16;
}

// Rows per batch of base that an epilogue warp copies (its registers hold eight at a time).
template <class YT>
__host__ __device__ constexpr int epi_rows() { return sizeof(YT) == 4 ? 8 : 16; }

struct TcParams {
  CUtensorMap tm_x, tm_b;  // rows of x (boxes of rt rows x 128 bytes, swizzled) and of base (a batch x 64 channels)
  LowRankBank bank;
  AdapterPlanDev plan;
  LowRankArgs a;
  int32_t rt, splits;        // rows per unit (16, 32 or 64), shares of the output channels
  int32_t x_slots, a_slots, b_slots, t_bufs;  // ring depths
  int32_t epi_ring;  // bytes of an epilogue warp's ring: 2048 or 4096
  int32_t x_vec;   // rows of x start on 16 bytes (16-byte copies, TMA)
  int32_t x_four;  // rows of x start on 4 bytes
  int32_t b_copy;  // bytes of a copy that base's rows are aligned for: 16, 4 or 2 (none, element loads)
  int32_t y_pair;  // y's channels can be stored in pairs
  uint32_t* err;
};

// Units of the plan's tiles: large ones in parts of rt rows, parts of the same
// number together (so that those behind a tile's last row come last), then the
// small ones.
__device__ __forceinline__ int64_t count_units(const TcParams& p, int n_large, int n_small) {
  return ((int64_t)n_large * (kAdapterTileRows / p.rt) + n_small) * p.splits;
}
template <int XTYPE>
__device__ __forceinline__ Unit get_unit(const TcParams& p, int n_large, int64_t u) {
  Unit r;
  const int split = (int)(u % p.splits);
  const int64_t v = u / p.splits, small = v - (int64_t)n_large * (kAdapterTileRows / p.rt);
  const AdapterTile tl = small >= 0 ? p.plan.small[small] : p.plan.large[v % n_large];
  const int off = small >= 0 ? 0 : (int)(v / n_large) * p.rt;
  r.pos0 = tl.pos0 + off;
  r.rows = min(p.rt, tl.rows - off);
  r.row0 = tl.row0 < 0 ? -1 : tl.row0 + off;
  const int chunks = (p.bank.n_out + 255) / 256;
  r.c0 = chunks * split / p.splits;
  r.c1 = chunks * (split + 1) / p.splits;
  r.ta = r.tb = nullptr;
  r.unscale = nullptr;
  r.rank = r.rp = 0;
  r.scale = 0.0f;
  if (r.rows > 0 && tl.adapter >= 0 && tl.adapter < p.bank.n_adapters) {
    const LowRankAdapter ad = p.bank.adapters[tl.adapter];
    r.ta = ad.ta[XTYPE], r.tb = ad.tb, r.rank = ad.rank, r.rp = ad.rp, r.scale = ad.scale;
    if (XTYPE == kDtF16) r.unscale = ad.unscale;
  }
  return r;
}

// A role's position in the ring of units.
struct UnitCursor {
  Ring r;
  // The next unit into `un`; false at the end or when the kernel gives up. Called by a whole warp (WARP) or by one
  // thread of it. RELEASE: the entry is free as far as this reader goes.
  template <bool WARP, bool RELEASE>
  __device__ __forceinline__ bool next(Unit& un, const Unit* units, uint64_t* full, uint64_t* empty,
                                       volatile int* abort_flag, uint32_t* err) {
    const bool ok = WARP ? warp_wait(&full[r.slot], r.parity, abort_flag, err, 4096u)
                         : stage_wait(&full[r.slot], r.parity, abort_flag, err, 4096u);
    if (!ok) return false;
    un = units[r.slot];
    if (RELEASE) {
      if (WARP) __syncwarp();
      if (!WARP || (threadIdx.x & 31) == 0) mbar_arrive(&empty[r.slot]);
    }
    r.next(kUnitSlots);
    return un.rows > 0;
  }
};

template <class XT, class YT>
__global__ void __launch_bounds__(kThreads, 1) lowrank_tc_kernel(const __grid_constant__ TcParams p) {
  constexpr int XTYPE = dtype_of<XT>();
  constexpr int PX = XTYPE == kDtF32 ? 2 : 1;                 // planes of x
  constexpr int KS = 128 / sizeof(XT);                        // input channels per stage: a 128-byte row of x
  constexpr int XE = 16 / sizeof(XT);                         // elements of a 16-byte copy
  constexpr int XL = KS / XE;                                 // copies per row
  constexpr int XR = kXWarps / kXGroups * 32 / XL;            // rows per pass of a group of X warps
  constexpr int XV = kRt / XR;                                // passes
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = smem_raw + ((1024 - (smem_u32(smem_raw) & 1023)) & 1023);
  const int PW = p.bank.wtype == kDtF32 ? 2 : 1;  // planes of B
  const int PA = a_parts(XTYPE, p.bank.wtype);    // parts of A
  const int x_atom = p.rt * 128, x_slot = PX * x_atom;  // [plane][rt rows][128 B]
  const int a_slot = ((p.bank.max_rank + 15) & ~15) * 128;  // a piece of A: the ranks' 128-byte rows
  const int t_plane = p.rt * 128, t_chunks = (p.bank.max_rank + KC - 1) / KC;  // [chunk][hi, lo][rt rows][128 B]
  uint8_t* sX = smem;
  uint8_t* sA = sX + p.x_slots * x_slot;
  uint8_t* sB = sA + p.a_slots * a_slot;
  uint8_t* sT = sB + p.b_slots * kBPlane;
  const int t_buf = t_chunks * 2 * t_plane;
  uint8_t* sE = sT + p.t_bufs * t_buf;
  uint8_t* misc = sE + kEpiWarps * p.epi_ring;
  uint64_t* xfull = reinterpret_cast<uint64_t*>(misc);
  uint64_t* xempty = xfull + kMaxSlots;
  uint64_t* afull = xempty + kMaxSlots;   // weights of the shrink and of the expand
  uint64_t* aempty = afull + kMaxSlots;
  uint64_t* bfull = aempty + kMaxSlots;
  uint64_t* bempty = bfull + kMaxSlots;
  uint64_t* tafull = bempty + kMaxSlots;  // a shrink accumulator is complete / read
  uint64_t* taempty = tafull + 2;
  uint64_t* tfull = taempty + 2;          // t in shared memory is written / free
  uint64_t* tfree = tfull + 2;
  uint64_t* dfull = tfree + 2;            // an expand accumulator is complete / read
  uint64_t* dempty = dfull + 2;
  uint64_t* drain = dempty + 2;           // [2] the MMA threads' last MMAs
  uint64_t* ufull = drain + 2;            // the ring of units
  uint64_t* uempty = ufull + kUnitSlots;
  uint64_t* xraw = uempty + kUnitSlots;    // float32 rows have arrived
  uint64_t* efull = xraw + kMaxSlots;      // [epilogue warp][4] a batch of base has arrived
  uint32_t* s_tmem = reinterpret_cast<uint32_t*>(efull + kEpiWarps * 4);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(s_tmem + 1);
  Unit* units = reinterpret_cast<Unit*>(misc + 1280);
  static_assert((7 * kMaxSlots + 14 + 2 * kUnitSlots + kEpiWarps * 4) * 8 + 8 <= 1280 &&
                    1280 + sizeof(Unit) * kUnitSlots <= kMiscBytes, "barriers and units");
  uint32_t* err = p.err ? p.err : &g_lowrank_error;

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int i = 0; i < kMaxSlots; ++i) {
      mbar_init(&xfull[i], kXWarps / kXGroups);
      mbar_init(&xempty[i], 1);
      mbar_init(&afull[i], 1);
      mbar_init(&aempty[i], 1);
      mbar_init(&bfull[i], 1);
      mbar_init(&bempty[i], 1);
      mbar_init(&xraw[i], 1);
    }
    for (int i = 0; i < kEpiWarps * 4; ++i) mbar_init(&efull[i], 1);
    for (int i = 0; i < 2; ++i) {
      mbar_init(&tafull[i], 1);
      mbar_init(&taempty[i], kTWarps);
      mbar_init(&dfull[i], 1);
      mbar_init(&dempty[i], kEpiWarps);
      mbar_init(&tfull[i], kTWarps);
      mbar_init(&tfree[i], 1);
      mbar_init(&drain[i], 1);
    }
    for (int i = 0; i < kUnitSlots; ++i) {
      mbar_init(&ufull[i], 1);
      mbar_init(&uempty[i], kUnitReaders);
    }
    *abort_flag = 0;
    fence_mbar_init();
  }
  if (warp == kWarpShrink) tmem_alloc(s_tmem, 512);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *s_tmem;  // shrink accumulators at columns 0 and 128, expand at 256 and 384
  const int k_stages = p.bank.ka / KS;

  if (warp < kXWarps) {
    // ---------------- x: global -> swizzled shared memory; float32 split in place ----------------
    if constexpr (Regs<XT>::x < 64) asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(Regs<XT>::x));
    const int k = p.bank.k_in;
    // The two groups of warps take the stages in turn (counted over all units), so that one converts while the other
    // waits, fences and issues.
    const int group = warp / (kXWarps / kXGroups), first_warp = group * (kXWarps / kXGroups);
    const int tx = threadIdx.x - first_warp * 32, col = tx % XL * XE, r0 = tx / XL;
    const int full_stages = p.x_vec ? k / KS : 0;  // stages that 16-byte copies can take
    const XT* row[XV];
    // the cursor of the copies: a unit, its stage ks
    UnitCursor uc;
    int ks = group, passes = 0, tma_row = -1;
    auto open = [&]() -> bool {  // the unit of stage ks, which counts from the present unit's first
      Unit un;
      for (bool have = passes > 0; !have || ks >= k_stages; have = true) {
        if (have) ks -= k_stages;
        do {
          if (!uc.next<true, true>(un, units, ufull, uempty, abort_flag, err)) return false;
        } while (un.rank == 0);
        passes = (un.rows + XR - 1) / XR;  // later ones have no rows
      }
      tma_row = p.x_vec && un.rows == p.rt ? un.row0 : -1;  // a box holds rows of the unit only
#pragma unroll
      for (int i = 0; i < XV; ++i) {  // behind the last row: that row again
        const int r = min(r0 + i * XR, un.rows - 1);
        row[i] = static_cast<const XT*>(p.a.x) +
                 (int64_t)(un.row0 >= 0 ? un.row0 + r : p.plan.pos_row[un.pos0 + r]) * p.a.ldx + col;
      }
      return true;
    };
    // this thread's 16-byte piece of its first row in a slot (its other rows are multiples of 8 further)
    static_assert(XR % 8 == 0, "swizzle");
    const uint32_t at0 = r0 * 128 + ((col / XE) ^ (r0 & 7)) * 16;
    auto step = [&](Ring& r) {  // to this group's next stage
      for (int i = 0; i < kXGroups; ++i) r.next(p.x_slots);
    };
    Ring ir, xr;  // copies issued, stages done
    for (int i = 0; i < group; ++i) ir.next(p.x_slots), xr.next(p.x_slots);
    uint32_t by_tma = 0;  // slots on their way by TMA
    bool ok = true, more = open();
    int pending = 0;
    auto issue = [&]() {  // the cursor's stage, with one group of copies (an empty one by TMA, and at the end)
      if (more) {
        // float32 by TMA: the A thread loads it, the X warps take over when the bytes are there (xraw)
        if (PX == 1 || tma_row < 0) {
          ok = warp_wait(&xempty[ir.slot], ir.parity ^ 1, abort_flag, err, 1u);
          if (!ok) return;
        }
        uint8_t* dst = sX + ir.slot * x_slot;
        by_tma &= ~(1u << ir.slot);
        if (tma_row >= 0) {
          by_tma |= 1u << ir.slot;
          if (PX == 1 && elect_lane()) {  // 16-bit rows go straight to the MMAs
            if (warp == first_warp) {
              mbar_arrive_expect_tx(&xfull[ir.slot], x_atom);
              tma_load_2d(&p.tm_x, &xfull[ir.slot], dst, ks * KS, tma_row);
            } else {
              mbar_arrive(&xfull[ir.slot]);
            }
          }
        } else {
          if (PX == 2 && warp == first_warp && lane == 0) mbar_arrive(&xraw[ir.slot]);  // its phases count stages
          const int c = ks * KS + col;
#pragma unroll
          for (int i = 0; i < XV; ++i) {
            if (i >= passes || r0 + i * XR >= p.rt) break;
            const uint32_t d = smem_u32(dst) + at0 + i * XR * 128;
            if (ks < full_stages) {
              copy16(d, row[i] + ks * KS, 16);
            } else if (p.x_four && (ks + 1) * KS <= k) {
#pragma unroll
              for (int j = 0; j < 4; ++j) copy4(d + j * 4, row[i] + ks * KS + j * (4 / (int)sizeof(XT)), 4);
            } else if (p.x_four) {  // what lies behind k is zeros (that A's are zeros is not enough for a NaN)
              constexpr int E4 = 4 / sizeof(XT);
#pragma unroll
              for (int j = 0; j < 4; ++j) {
                const int bytes = max(0, min(4, (k - c - j * E4) * (int)sizeof(XT)));
                copy4(d + j * 4, row[i] + (bytes ? ks * KS + j * E4 : -col), bytes);
              }
            } else if constexpr (PX == 1) {  // odd 16-bit addresses: loads, clamped instead of conditional
              XT e[XE];
#pragma unroll
              for (int j = 0; j < XE; ++j) e[j] = row[i][min(c + j, k - 1) - col];
              uint32_t v[4];
              const uint16_t* h = reinterpret_cast<const uint16_t*>(e);
#pragma unroll
              for (int j = 0; j < 4; ++j)
                v[j] = (c + 2 * j < k ? h[2 * j] : 0u) | (c + 2 * j + 1 < k ? (uint32_t)h[2 * j + 1] << 16 : 0u);
              *reinterpret_cast<uint4*>(dst + at0 + i * XR * 128) = make_uint4(v[0], v[1], v[2], v[3]);
            }
          }
        }
        step(ir);
        ++pending;
        ks += kXGroups;
        if (ks >= k_stages) more = open();
      }
      cp_async_commit();
    };
    const int depth = max(1, p.x_slots / kXGroups - (PX == 2 ? 1 : 0));
    for (int d = 0; ok && d < depth; ++d) issue();
    while (ok && pending > 0) {
      copy_wait(depth - 1);  // the oldest stage of this thread's own copies has landed
      if (PX == 2) {
        ok = warp_wait(&xraw[xr.slot], xr.parity, abort_flag, err, 16384u);
        if (!ok) break;
        uint8_t* dst = sX + xr.slot * x_slot + at0;
        float4 v[XV];
#pragma unroll
        for (int i = 0; i < XV; ++i)
          if (r0 + i * XR < p.rt) v[i] = *reinterpret_cast<const float4*>(dst + i * XR * 128);
#pragma unroll
        for (int i = 0; i < XV; ++i) {
          if (r0 + i * XR >= p.rt) break;
          float4 hi, lo;
          split_tf32(v[i].x, hi.x, lo.x);
          split_tf32(v[i].y, hi.y, lo.y);
          split_tf32(v[i].z, hi.z, lo.z);
          split_tf32(v[i].w, hi.w, lo.w);
          *reinterpret_cast<float4*>(dst + i * XR * 128) = hi;
          *reinterpret_cast<float4*>(dst + x_atom + i * XR * 128) = lo;
        }
      }
      if (PX == 2 || !(by_tma >> xr.slot & 1)) {
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(&xfull[xr.slot]);
      }
      step(xr);
      --pending;
      issue();
    }
    cp_async_wait<0>();
    // given up: loads in flight land before the CTA's shared memory is released
    for (; !ok && pending > 0; --pending, step(xr))
      mbar_wait_drain(PX == 2 ? &xraw[xr.slot] : &xfull[xr.slot], xr.parity);
  } else if (warp < kWarpT) {
    // ---------------- epilogue: base + accumulators -> y ----------------
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(Regs<XT>::epi));
    struct alignas(2 * sizeof(YT)) Pair { YT e[2]; };
    constexpr int B = epi_rows<YT>(), RB = 64 * sizeof(YT);  // rows of a batch, bytes of one: this warp's 64 channels
    constexpr int S = 8;                                     // rows in registers
    const int nb = p.epi_ring / (B * RB);                 // batches: 1 to 4
    const YT* base = static_cast<const YT*>(p.a.base);
    YT* y = static_cast<YT*>(p.a.y);
    const int quarter = warp & 3, n_out = p.bank.n_out;
    const uint32_t ring = smem_u32(sE) + (warp - kWarpEpi) * p.epi_ring;
    // this warp's rows [i0, i1) of a unit: a fourth of them, eight at least
    const int per = max(S, p.rt / 4), i0 = ((warp - kWarpEpi) >> 2) * per;
    // Lane i has row i0 + i of the unit, or its group's last one; first_row is that of the group's first lane when its
    // n rows follow each other (they increase), else -1.
    auto my_row = [&](const Unit& un, int end) -> int {
      const int i = min(i0 + lane, end - 1);
      return un.row0 >= 0 ? un.row0 + i : p.plan.pos_row[un.pos0 + i];
    };
    auto first_row = [&](int row, int n) -> int {
      const int first = __shfl_sync(0xffffffffu, row, 0);
      return __shfl_sync(0xffffffffu, row, n - 1) - first == n - 1 ? first : -1;
    };
    // the cursor of the copies: a unit, chunk fc of [.., fc1), rows from fi; its lane's row and its first row
    UnitCursor fu, uc;
    int fc = 0, fc1 = 0, fi = 0, fi1 = 0, frow0 = 0, frow = 0;
    uint64_t* bars = efull + (warp - kWarpEpi) * 4;
    Ring fr, er;      // batches copied, batches used
    int ahead = 0;    // units that fu is ahead of uc: the ring holds kUnitSlots, and uc alone frees them
    int filled = 0;   // batches copied and not yet used
    bool more = false, end = base == nullptr;
    auto open = [&]() -> bool {
      while (!end && ahead < kUnitSlots - 2) {
        Unit un;
        if (!fu.next<true, false>(un, units, ufull, uempty, abort_flag, err)) {
          end = true;
          break;
        }
        ++ahead;
        fi1 = min(un.rows, i0 + per);
        if (un.rank == 0 || i0 >= fi1) continue;
        frow = my_row(un, fi1);
        frow0 = first_row(frow, fi1 - i0);
        fc = un.c0, fc1 = un.c1, fi = i0;
        return true;
      }
      return false;
    };
    auto fill = [&]() {  // the cursor's batch, if there is one, as one group of copies
      if (!more) more = open();
      if (more) {
        const int ch = fc * 256 + quarter * 64, in = min(64, n_out - ch);  // channels of this warp's there are
        auto off = [&](int r) -> int64_t {  // rows behind the group's last one: that one again
          return __shfl_sync(0xffffffffu, frow, fi - i0 + r) * p.a.ldb;
        };
        const uint32_t fslot = ring + fr.slot * (B * RB);
        const bool tma = p.b_copy == 16 && frow0 >= 0 && fi + B <= fi1;  // a box holds rows of the unit only
        if (elect_lane()) {
          if (tma) {
            mbar_arrive_expect_tx(&bars[fr.slot], B * RB);
            tma_load_2d(&p.tm_b, &bars[fr.slot], sE + (fslot - smem_u32(sE)), ch, frow0 + fi - i0);
          } else {
            mbar_arrive(&bars[fr.slot]);  // its phases count batches
          }
        }
        if (tma) {
        } else if (p.b_copy == 16) {
          constexpr int LPR = RB / 16, E16 = 16 / sizeof(YT), RPI = 32 / LPR;  // lanes per row, rows per instruction
          const int c = lane % LPR * E16, bytes = max(0, min(16, (in - c) * (int)sizeof(YT)));
          const uint32_t dst = fslot + lane / LPR * RB + c * sizeof(YT);
          const YT* col = base + (bytes ? ch + c : 0);
#pragma unroll
          for (int j = 0; j < B; j += RPI) copy16(dst + j * RB, col + off(j + lane / LPR), bytes);
        } else if (p.b_copy == 4) {
          constexpr int E4 = 4 / sizeof(YT), NC = 2 / E4;  // copies of a lane per row
          const YT* col[NC];
          int bytes[NC];
#pragma unroll
          for (int q = 0; q < NC; ++q) {
            const int c = lane * E4 + 32 * q;
            bytes[q] = max(0, min(4, (in - c) * (int)sizeof(YT)));
            col[q] = base + (bytes[q] ? ch + c : 0);
          }
          const uint32_t dst = fslot + lane * 4;
          if (frow0 >= 0 && fi + B <= fi1) {  // the usual case in few instructions: they bound unaligned rows
#pragma unroll
            for (int q = 0; q < NC; ++q) col[q] += ((int64_t)frow0 + fi - i0) * p.a.ldb;
#pragma unroll
            for (int r = 0; r < B; ++r)
#pragma unroll
              for (int q = 0; q < NC; ++q) {
                copy4(dst + r * RB + q * 128, col[q], bytes[q]);
                col[q] += p.a.ldb;
              }
          } else {
#pragma unroll 2
            for (int r = 0; r < B; ++r) {
              const int64_t o = off(r);
#pragma unroll
              for (int q = 0; q < NC; ++q) copy4(dst + r * RB + q * 128, col[q] + o, bytes[q]);
            }
          }
        } else if constexpr (sizeof(YT) == 2) {  // odd 16-bit addresses: loads, clamped instead of conditional
          const YT* c0 = base + min(ch + lane, n_out - 1);
          const YT* c1 = base + min(ch + lane + 32, n_out - 1);
          YT* dst = reinterpret_cast<YT*>(sE + (fslot - smem_u32(sE)));
#pragma unroll 1
          for (int r = 0; r < B; r += 2) {
            YT v0[2], v1[2];
#pragma unroll
            for (int j = 0; j < 2; ++j) {
              const int64_t o = off(r + j);
              v0[j] = c0[o], v1[j] = c1[o];
            }
#pragma unroll
            for (int j = 0; j < 2; ++j) dst[(r + j) * 64 + lane] = v0[j], dst[(r + j) * 64 + lane + 32] = v1[j];
          }
        }
        fr.next(nb);
        fi += B;
        if (fi >= fi1) {
          fi = i0;
          more = ++fc < fc1;
        }
        cp_async_commit();
        ++filled;
      }
    };
    for (int b = 0; b < nb; ++b) fill();
    uint32_t d = 0;
    bool ok = true;
    Unit un;
    while (ok) {
      if (!more) more = open();  // fu reads an entry before uc frees it
      if (!uc.next<true, true>(un, units, ufull, uempty, abort_flag, err)) break;
      --ahead;
      if (un.rank == 0) {
        // y = base, eight loads in flight per lane
        const int first = un.c0 * 256, cols = min(n_out, un.c1 * 256) - first;
        for (int r = warp - kWarpEpi; r < un.rows; r += kEpiWarps) {
          const int64_t row = un.row0 >= 0 ? un.row0 + r : p.plan.pos_row[un.pos0 + r];
          const YT* src = base ? base + row * p.a.ldb + first : nullptr;
          YT* dst = y + row * p.a.ldy + first;
          for (int c = lane; c < cols; c += 256) {
            YT v[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) v[j] = src ? src[min(c + 32 * j, cols - 1)] : as_type<YT>(0.0f);
#pragma unroll
            for (int j = 0; j < 8; ++j)
              if (c + 32 * j < cols) dst[c + 32 * j] = v[j];
          }
        }
        continue;
      }
      const int i1 = min(un.rows, i0 + per);
      const int row = i0 < i1 ? my_row(un, i1) : 0, row0 = first_row(row, i1 - i0);
      for (int c = un.c0; c < un.c1; ++c, ++d) {
        ok = warp_wait(&dfull[d & 1], (d >> 1) & 1, abort_flag, err, 2u);
        if (!ok) break;
        tc_fence_after();
        const int ch = c * 256 + quarter * 64 + lane * 2;
        const uint32_t acc = tmem + ((uint32_t)(quarter * 32) << 16) + 256u + (d & 1) * 128u;
        for (int i = i0; i < i1; i += S) {
          Pair b[S];
          const int sub = (i - i0) % B;  // rows of the batch before these
          if (base) {
            if (sub == 0) {
              if (!filled) fill();  // the cursor was at its limit
              copy_wait(filled - 1);
              ok = warp_wait(&bars[er.slot], er.parity, abort_flag, err, 32768u);
              if (!ok) break;
              __syncwarp();  // the other lanes' copies
            }
            const uint8_t* src = sE + (ring - smem_u32(sE)) + (er.slot * B + sub) * RB + lane * 2 * sizeof(YT);
#pragma unroll
            for (int j = 0; j < S; ++j) b[j] = *reinterpret_cast<const Pair*>(src + j * RB);
          } else {
#pragma unroll
            for (int j = 0; j < S; ++j) b[j].e[0] = b[j].e[1] = as_type<YT>(0.0f);
          }
          uint32_t v0[S], v1[S];
          tmem_ld8(acc + (uint32_t)i, v0);
          tmem_ld8(acc + (uint32_t)(p.rt + i), v1);
          tmem_wait_ld();
          reg_barrier8(v0);
          reg_barrier8(v1);
#pragma unroll
          for (int j = 0; j < S; ++j) {
            b[j].e[0] = as_type<YT>(__fadd_rn(as_f32(b[j].e[0]), __uint_as_float(v0[j])));
            b[j].e[1] = as_type<YT>(__fadd_rn(as_f32(b[j].e[1]), __uint_as_float(v1[j])));
          }
          // The slot's next copy: the sums hold its values, and the fence orders the loads before what TMA writes. (Right
          // behind the loads nothing makes a copy wait for them.)
          if (base && (sub + S == B || i + S >= i1)) {
            fence_proxy_async_smem();
            __syncwarp();
            er.next(nb);
            --filled;
            fill();
          }
          const bool whole = row0 >= 0 && i + S <= i1;  // the usual case in few instructions
          if (p.y_pair) {
            if (whole) {
              if (ch < n_out) {
                YT* dst = y + (int64_t)(row0 + i - i0) * p.a.ldy + ch;
#pragma unroll
                for (int j = 0; j < S; ++j, dst += p.a.ldy) *reinterpret_cast<Pair*>(dst) = b[j];
              }
            } else {
#pragma unroll
              for (int j = 0; j < S; ++j) {
                YT* dst = y + __shfl_sync(0xffffffffu, row, i - i0 + j) * p.a.ldy + ch;
                if (i + j < i1 && ch < n_out) *reinterpret_cast<Pair*>(dst) = b[j];
              }
            }
          } else {
            // single values: exchanged so that the lanes' channels follow each other, lane and lane + 32
            const int c0 = ch - lane;
            auto swap = [&](int from, const Pair& v) -> YT {
              if constexpr (sizeof(YT) == 2) {
                const uint32_t both = __shfl_sync(0xffffffffu, raw_bits(v.e[0]) | raw_bits(v.e[1]) << 16, from);
                return from_bits<YT>(lane & 1 ? both >> 16 : both);
              } else {
                const uint32_t bits = __shfl_sync(0xffffffffu, raw_bits(v.e[0]), from);
                const uint32_t odd = __shfl_sync(0xffffffffu, raw_bits(v.e[1]), from);
                return from_bits<YT>(lane & 1 ? odd : bits);
              }
            };
            const bool first = c0 < n_out, second = c0 + 32 < n_out;
            if (whole) {
              YT* dst = y + (int64_t)(row0 + i - i0) * p.a.ldy + c0;
#pragma unroll
              for (int j = 0; j < S; ++j, dst += p.a.ldy) {
                const YT lo = swap(lane >> 1, b[j]), hi = swap(16 + (lane >> 1), b[j]);
                if (first) dst[0] = lo;
                if (second) dst[32] = hi;
              }
            } else {
#pragma unroll
              for (int j = 0; j < S; ++j) {
                const YT lo = swap(lane >> 1, b[j]), hi = swap(16 + (lane >> 1), b[j]);
                YT* dst = y + __shfl_sync(0xffffffffu, row, i - i0 + j) * p.a.ldy + c0;
                if (first && i + j < i1) dst[0] = lo;
                if (second && i + j < i1) dst[32] = hi;
              }
            }
          }
        }
        if (!ok) break;
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&dempty[d & 1]);
      }
    }
    cp_async_wait<0>();
    for (; !ok && filled > 0; --filled, er.next(nb)) mbar_wait_drain(&bars[er.slot], er.parity);  // as above
  } else {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(Regs<XT>::rest));
    if (warp < kWarpShrink) {
    // ---------------- t: TMEM -> scaled, split -> shared memory ----------------
    const int quarter = warp & 3, row = quarter * 32 + lane;  // this lane's row of the unit
    uint32_t q = 0;
    Ring tr;
    bool ok = true;
    UnitCursor uc;
    Unit un;
    while (ok && uc.next<true, true>(un, units, ufull, uempty, abort_flag, err)) {
      if (un.rank == 0) continue;
      float sc = un.scale;
      if (p.a.absmax && row < un.rows)
        sc = __fmul_rn(sc, __fdiv_rn(__uint_as_float(p.a.absmax[p.a.per_seq ? p.plan.pos_seq[un.pos0 + row] : 0]),
                                     127.0f));
      const ShrinkAcc sa(p.bank.max_rank, un.rank, PX == 2 || PA > 1, k_stages);
      ok = warp_wait(&tafull[(q & (sa.bufs - 1))], (q >> (sa.bufs - 1)) & 1, abort_flag, err, 4u) &&
           warp_wait(&tfree[tr.slot], tr.parity ^ 1, abort_flag, err, 8u);
      if (!ok) break;
      tc_fence_after();
      if (quarter * 32 < un.rows) {
        const uint32_t acc = tmem + ((uint32_t)(quarter * 32) << 16) + ((q & (sa.bufs - 1))) * 128u;
        for (int j = 0; j < un.rp; j += 8) {  // eight ranks: two 16-byte pieces of each plane
          float t[8];
          {
            uint32_t v[8];
            tmem_ld8(acc + (uint32_t)j, v);
            tmem_wait_ld();
            reg_barrier8(v);
#pragma unroll
            for (int e = 0; e < 8; ++e) t[e] = __uint_as_float(v[e]);
          }
          for (int k = 1; k < sa.hi_parts; ++k) {
            uint32_t v[8];
            tmem_ld8(acc + (uint32_t)(k * sa.width + j), v);
            tmem_wait_ld();
            reg_barrier8(v);
#pragma unroll
            for (int e = 0; e < 8; ++e) t[e] = __fadd_rn(t[e], __uint_as_float(v[e]));
          }
          // The low parts. Where the sum so far is an infinity or NaN it is the result, since every factor is in it with
          // its sign: an infinity times a low part of zero is a NaN that the formula does not have.
          if (PX == 2 || PA > 1) {
            uint32_t v[8];
            tmem_ld8(acc + (uint32_t)(sa.hi_parts * sa.width + j), v);
            tmem_wait_ld();
            reg_barrier8(v);
#pragma unroll
            for (int e = 0; e < 8; ++e)
              if (fabsf(t[e]) < __uint_as_float(0x7f800000u)) t[e] = __fadd_rn(t[e], __uint_as_float(v[e]));
          }
          if (XTYPE == kDtF16 && un.unscale) {
#pragma unroll
            for (int e = 0; e < 8; ++e) t[e] = __fmul_rn(t[e], __ldg(un.unscale + j + e));
          }
          float hi[8], lo[8];
#pragma unroll
          for (int e = 0; e < 8; ++e)  // ranks behind the last one meet zero columns of B: they have to be finite
            split_tf32_lo_finite(j + e < un.rank ? __fmul_rn(t[e], sc) : 0.0f, hi[e], lo[e]);
          uint8_t* dst = sT + tr.slot * t_buf + (j / KC) * 2 * t_plane + row * 128;
          if (row >= p.rt) continue;  // lanes without a row of t (units of 16 rows)
          const int c0 = (j % KC) / 4, x = row & 7;
          *reinterpret_cast<float4*>(dst + ((c0 ^ x) * 16)) = make_float4(hi[0], hi[1], hi[2], hi[3]);
          *reinterpret_cast<float4*>(dst + (((c0 + 1) ^ x) * 16)) = make_float4(hi[4], hi[5], hi[6], hi[7]);
          *reinterpret_cast<float4*>(dst + t_plane + ((c0 ^ x) * 16)) = make_float4(lo[0], lo[1], lo[2], lo[3]);
          *reinterpret_cast<float4*>(dst + t_plane + (((c0 + 1) ^ x) * 16)) = make_float4(lo[4], lo[5], lo[6], lo[7]);
        }
      }
      fence_proxy_async_smem();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) {
        mbar_arrive(&taempty[(q & (sa.bufs - 1))]);
        mbar_arrive(&tfull[tr.slot]);
      }
      tr.next(p.t_bufs);
      ++q;
    }
  } else if (warp == kWarpShrink) {
    // ---------------- tensor cores: t^T accumulators from x and A ----------------
    if (elect_lane()) {
      Ring xr, ar;
      uint32_t q = 0;
      bool ok = true;
      UnitCursor uc;
      Unit un;
      while (ok && uc.next<false, true>(un, units, ufull, uempty, abort_flag, err)) {
        if (un.rank == 0) continue;
        const ShrinkAcc sa(p.bank.max_rank, un.rank, PX == 2 || PA > 1, k_stages);
        const uint32_t set = q & (sa.bufs - 1), id = XTYPE == kDtF32 ? idesc_tf32(128, sa.width) : idesc_16(XTYPE == kDtBF16, 128, sa.width);
        ok = stage_wait(&taempty[set], ((q >> (sa.bufs - 1)) & 1) ^ 1, abort_flag, err, 16u);
        tc_fence_after();
        const uint32_t acc0 = tmem + set * 128u, acc_lo = acc0 + (uint32_t)(sa.hi_parts * sa.width);
        int c = 0;
        for (int part = 0; ok && part < sa.hi_parts; ++part) {
          const uint32_t acc = acc0 + (uint32_t)(part * sa.width);
          const int end = k_stages * (part + 1) / sa.hi_parts;
          for (uint32_t more = 0; c < end; ++c) {
            ok = stage_wait(&xfull[xr.slot], xr.parity, abort_flag, err, 32u);
            tc_fence_after();
            const uint32_t x0 = desc_lo(smem_u32(sX) + xr.slot * x_slot);
            auto piece = [&](int part) {  // a part of A against x
              if (!ok) return;
              ok = stage_wait(&afull[ar.slot], ar.parity, abort_flag, err, 64u);
              if (!ok) return;
              tc_fence_after();
              const uint32_t w = desc_lo(smem_u32(sA) + ar.slot * a_slot);
#pragma unroll
              for (int s = 0; s < 4; ++s) {
                const uint64_t dx = desc_at(x0 + 2 * s), dw = desc_at(w + 2 * s);
                const uint32_t on = s > 0 || c > 0;  // the low parts' accumulator has something
                if (PX == 2) {
                  umma_tf32(part == 0 ? acc : acc_lo, dx, dw, id, part > 0 ? 1 : s > 0 ? 1 : more);
                  if (part == 0) umma_tf32(acc_lo, desc_at(x0 + (x_atom >> 4) + 2 * s), dw, id, on);
                } else {
                  umma_f16(part == 0 ? acc : acc_lo, dx, dw, id, part > 1 ? 1 : part == 1 ? on : s > 0 ? 1 : more);
                }
              }
              umma_commit(&aempty[ar.slot]);
              ar.next(p.a_slots);
            };
            piece(0);
            if (PA > 1) piece(1);
            if (PX == 1 && PA > 2) piece(2);
            more = 1;
            if (!ok) break;
            umma_commit(&xempty[xr.slot]);
            xr.next(p.x_slots);
          }
        }
        if (ok) umma_commit(&tafull[set]);
        ++q;
      }
      // every MMA and every commit's arrival is done before the CTA's memory goes
      umma_commit(&drain[0]);
      mbar_wait_drain(&drain[0], 0);
    }
  } else if (warp == kWarpExpand) {
    // ---------------- tensor cores: result accumulators from B and t ----------------
    if (elect_lane()) {
      const uint32_t id = idesc_tf32(128, p.rt);
      Ring br, tr;
      uint32_t d = 0;
      bool ok = true;
      UnitCursor uc;
      Unit un;
      while (ok && uc.next<false, true>(un, units, ufull, uempty, abort_flag, err)) {
        if (un.rank == 0) continue;
        ok = stage_wait(&tfull[tr.slot], tr.parity, abort_flag, err, 128u);
        tc_fence_after();
        for (int c = un.c0; ok && c < un.c1; ++c, ++d) {
          ok = stage_wait(&dempty[d & 1], ((d >> 1) & 1) ^ 1, abort_flag, err, 256u);
          tc_fence_after();
          for (int g = 0; ok && g < 2; ++g) {  // even, then odd channels
            const uint32_t acc = tmem + 256u + (d & 1) * 128u + (uint32_t)(g * p.rt);
            uint32_t t = desc_lo(smem_u32(sT) + tr.slot * t_buf), more = 0;
            for (int left = un.rp / 8; ok && left > 0; left -= KC / 8) {
              for (int pl = 0; pl < PW; ++pl) {
                ok = ok && stage_wait(&bfull[br.slot], br.parity, abort_flag, err, 1024u);
                if (!ok) break;
                tc_fence_after();
                const uint32_t w = desc_lo(smem_u32(sB) + br.slot * kBPlane);
#pragma unroll
                for (int s = 0; s < KC / 8; ++s) {
                  if (s >= left) break;
                  if (pl == 0) {
                    umma_tf32(acc, desc_at(w + 2 * s), desc_at(t + (t_plane >> 4) + 2 * s), id, more);
                    more = 1;
                  }
                  umma_tf32(acc, desc_at(w + 2 * s), desc_at(t + 2 * s), id, 1);
                }
                umma_commit(&bempty[br.slot]);
                br.next(p.b_slots);
              }
              t += 2 * t_plane >> 4;
            }
          }
          if (ok) umma_commit(&dfull[d & 1]);
        }
        if (ok) umma_commit(&tfree[tr.slot]);
        tr.next(p.t_bufs);
      }
      umma_commit(&drain[1]);
      mbar_wait_drain(&drain[1], 0);
    }
  } else if (warp == kWarpUnits) {
    // ---------------- units: looked up 32 at a time ----------------
    const int n_large = p.plan.counts[0];
    const int64_t n_units = count_units(p, n_large, p.plan.counts[1]);
    const bool in_place = p.a.base == p.a.y && p.a.ldb == p.a.ldy;  // nothing to do for rows without an adapter
    Ring r;
    bool ok = true;
    for (int64_t first = blockIdx.x; ok; first += 32 * (int64_t)gridDim.x) {
      const int64_t u = first + lane * (int64_t)gridDim.x;
      Unit un;
      un.rows = 0;
      if (u < n_units) un = get_unit<XTYPE>(p, n_large, u);
      uint32_t todo = __ballot_sync(0xffffffffu, un.rows > 0 && un.c1 > un.c0 && (un.rank > 0 || !in_place));
      const bool last = first + 32 * (int64_t)gridDim.x >= n_units;
      while (ok && (todo || last)) {
        const int from = todo ? __ffs(todo) - 1 : 0;  // without one left: the end, an entry without rows
        ok = warp_wait(&uempty[r.slot], r.parity ^ 1, abort_flag, err, 8192u);
        if (!ok) break;
        if (lane == from) {
          if (!todo) un.rows = 0;
          units[r.slot] = un;
          mbar_arrive(&ufull[r.slot]);
        }
        __syncwarp();
        r.next(kUnitSlots);
        if (!todo) break;
        todo &= todo - 1;
      }
      if (last) break;
    }
  } else if (warp <= kWarpB && elect_lane()) {
    // ---------------- weights: bulk copies of the bank's tiles (A's, or B's) ----------------
    const bool is_a = warp == kWarpA;
    uint8_t* ring = is_a ? sA : sB;
    const uint32_t slots = is_a ? p.a_slots : p.b_slots, slot = is_a ? a_slot : kBPlane;
    uint64_t *full = is_a ? afull : bfull, *empty = is_a ? aempty : bempty;
    Ring r, xr;
    uint32_t issued = 0, x_issued = 0;
    bool ok = true;
    UnitCursor uc;
    Unit un;
    while (ok && uc.next<false, true>(un, units, ufull, uempty, abort_flag, err)) {
      if (un.rank == 0) continue;
      const int rcs = (un.rp + KC - 1) / KC;
      const uint32_t bytes = is_a ? un.rank * 128 : kBPlane;  // of a piece
      const uint8_t* src = is_a ? un.ta : un.tb + (size_t)un.c0 * 2 * rcs * PW * kBPlane;
      const int pieces = is_a ? k_stages * PA : (un.c1 - un.c0) * 2 * rcs * PW;
      const bool load_x = PX == 2 && is_a && p.x_vec && un.rows == p.rt && un.row0 >= 0;  // as the X warps see it
      for (int n = 0; n < pieces; ++n, src += bytes) {
        if (PX == 2 && is_a && n % PA == 0) {  // a stage of float32 rows
          if (load_x) {
            ok = stage_wait(&xempty[xr.slot], xr.parity ^ 1, abort_flag, err, 1u);
            if (!ok) break;
            mbar_arrive_expect_tx(&xraw[xr.slot], x_atom);
            tma_load_2d(&p.tm_x, &xraw[xr.slot], sX + xr.slot * x_slot, n / PA * KS, un.row0);
          }
          xr.next(p.x_slots);
          ++x_issued;
        }
        ok = stage_wait(&empty[r.slot], r.parity ^ 1, abort_flag, err, is_a ? 512u : 2048u);
        if (!ok) break;
        mbar_arrive_expect_tx(&full[r.slot], bytes);
        bulk_load(ring + r.slot * slot, src, bytes, &full[r.slot]);
        r.next(slots);
        ++issued;
      }
    }
    // copies in flight land before the CTA's shared memory is released
    for (uint32_t i = issued > slots ? issued - slots : 0; i < issued; ++i)
      mbar_wait_drain(&full[i % slots], (i / slots) & 1);
    const uint32_t xs = p.x_slots;
    for (uint32_t i = x_issued > xs ? x_issued - xs : 0; i < x_issued; ++i)
      mbar_wait_drain(&xraw[i % xs], (i / xs) & 1);
  }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == kWarpShrink) tmem_dealloc(tmem, 512);
}

// The bank's weights as the kernel's tiles, tf32 planes (hi, and lo for float32
// weights) of rows of 32 values whose 16-byte pieces are swizzled by the row
// number; zeros outside. A: [32 channels][plane][rank rows]. B:
// [chunk of 256 channels][even, odd][32 ranks][plane][128 rows], row i of a
// chunk's tile g being channel 2 i + g.
template <class WT>
__global__ void lowrank_tiles_kernel(const LowRankAdapter* ads, int k_in, int n_out, int ka, int planes) {
  const LowRankAdapter ad = ads[blockIdx.y];
  if (ad.rank == 0) return;
  const int64_t na = (int64_t)ad.rank * ka;
  const int rcs = (ad.rp + KC - 1) / KC, tiles = (n_out + 255) / 256 * 2 * rcs;
  const int64_t nb = (int64_t)tiles * 128 * KC;
  for (int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i < na + nb; i += (int64_t)gridDim.x * blockDim.x) {
    float v = 0.0f;
    int row, c;
    uint8_t* tile;
    int64_t plane;  // bytes from the hi to the lo plane
    if (i < na) {
      row = (int)(i / ka);
      const int kk = (int)(i % ka);
      c = kk % KC;
      plane = (int64_t)ad.rank * 128;
      tile = const_cast<uint8_t*>(ad.ta[kDtF32]) + (int64_t)(kk / KC) * planes * plane;
      if (kk < k_in) v = as_f32(static_cast<const WT*>(ad.a)[i]);
    } else {
      const int64_t b = i - na, t = b / (128 * KC);
      row = (int)(b % (128 * KC)) / KC;
      c = (int)(b % KC);
      plane = kBPlane;
      tile = const_cast<uint8_t*>(ad.tb) + t * planes * plane;
      const int64_t n = t / (2 * rcs) * 256 + 2 * row + t / rcs % 2;
      const int j = (int)(t % rcs) * KC + c;
      if (n < n_out && j < ad.rank) v = as_f32(static_cast<const WT*>(ad.b)[n * ad.rp + j]);
    }
    float* dst = reinterpret_cast<float*>(tile + (int64_t)row * 128 + (((c >> 2) ^ (row & 7)) * 16) + (c & 3) * 4);
    if (planes == 2) {
      float hi, lo;
      split_tf32_lo_finite(v, hi, lo);
      // An infinite t times a low part of zero would be NaN: B's are at least 2^-126, with the weight's sign, where that
      // is nothing to the weight (A's low products have an accumulator that an infinite sum leaves out).
      if (i >= na && lo == 0.0f && fabsf(v) >= ldexpf(1.0f, -100)) lo = copysignf(ldexpf(1.0f, -126), v);
      dst[0] = hi;
      dst[plane / 4] = lo;
    } else {
      dst[0] = v;
    }
  }
}

// A's tiles for 16-bit x: [k stage][part][rank rows of 64 channels], swizzled
// the same way. A CTA per rank. fp16 parts of other types: the rank's weights
// times the power of two that brings the largest to [2^13, 2^14).
template <class WT>
__global__ void lowrank_tiles16_kernel(const LowRankAdapter* ads, int k_in, int ka, int parts_f16, int parts_bf16) {
  __shared__ float s_max[8];
  const LowRankAdapter ad = ads[blockIdx.y];
  const int j = blockIdx.x;
  if (j >= ad.rank) return;  // the whole CTA
  const WT* w = static_cast<const WT*>(ad.a) + (int64_t)j * ka;
  float top = 0.0f;
  for (int k = threadIdx.x; k < k_in; k += blockDim.x) top = fmaxf(top, fabsf(as_f32(w[k])));
  top = warp_max(top);
  if ((threadIdx.x & 31) == 0) s_max[threadIdx.x >> 5] = top;
  __syncthreads();
  for (int i = 0; i < (int)blockDim.x / 32; ++i) top = fmaxf(top, s_max[i]);
  int up = 0;
  if (ad.unscale && top > 0.0f && top < __uint_as_float(0x7f800000u)) up = min(13 - ilogbf(top), 100);
  if (ad.unscale && threadIdx.x == 0) const_cast<float*>(ad.unscale)[j] = ldexpf(1.0f, -up);
  auto put = [&](int xtype, int parts, int part, int k, uint16_t bits) {
    uint8_t* row = const_cast<uint8_t*>(ad.ta[xtype]) + ((int64_t)(k / 64 * parts + part) * ad.rank + j) * 128;
    const int c = k % 64;
    *reinterpret_cast<uint16_t*>(row + (((c >> 3) ^ (j & 7)) * 16) + (c & 7) * 2) = bits;
  };
  for (int k = threadIdx.x; k < ka; k += blockDim.x) {
    const float v = k < k_in ? as_f32(w[k]) : 0.0f;
    const float f = ldexpf(v, up);
    const __half h = __float2half_rn(f);
    put(kDtF16, parts_f16, 0, k, __half_as_ushort(h));
    if (parts_f16 > 1) {
      const float rest = __fsub_rn(f, __half2float(h));
      put(kDtF16, parts_f16, 1, k, __half_as_ushort(__float2half_rn(isfinite(rest) ? rest : 0.0f)));
    }
    float rest = v;
    for (int part = 0; part < parts_bf16; ++part) {  // cut, not rounded: no part overflows
      const uint32_t bits = __float_as_uint(rest) & 0xffff0000u;
      put(kDtBF16, parts_bf16, part, k, (uint16_t)(bits >> 16));
      const float less = __fsub_rn(rest, __uint_as_float(bits));
      rest = isfinite(less) ? less : 0.0f;
    }
  }
}

template <class XT, class YT>
cudaError_t tc_types(TcParams p, int n_large, int n_small, cudaStream_t st) {
  constexpr int XTYPE = dtype_of<XT>(), PX = XTYPE == kDtF32 ? 2 : 1;
  const int chunks = (p.bank.n_out + 255) / 256;
  int dev = 0, sms = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e == cudaSuccess) e = cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
  if (e != cudaSuccess) return e;
  p.rt = kRt;
  p.splits = 1;
  // Fewer rows per unit, then shares of the channels, while all units still run at once: a unit's time is mostly its
  // pipeline's latency (6075 ragged float32 rows, 512 x 1024, rank 23: 27.0 us in one round of 64-row units, 29.9 in
  // two rounds of 32).
  auto units = [&](int rt, int splits) { return ((int64_t)n_large * (kAdapterTileRows / rt) + n_small) * splits; };
  while (p.rt > 16 && units(p.rt / 2, 1) <= sms) p.rt /= 2;
  while (p.splits < chunks && units(p.rt, p.splits + 1) <= sms) ++p.splits;
  // Shared memory: the most rows that fit two slots of every ring, then what is left for more of them.
  const int t_chunks = (p.bank.max_rank + KC - 1) / KC, a_slot = (p.bank.max_rank + 15) / 16 * 16 * 128;
  int smem = 0;
  for (; p.rt >= 16; p.rt /= 2) {
    const int t_buf = t_chunks * 2 * p.rt * 128, x_slot = PX * p.rt * 128;
    int left = kMaxSmem - 1024 - kMiscBytes - kEpiWarps * 2048 - 2 * (kBPlane + a_slot + x_slot) - t_buf;
    if (left < 0) continue;
    p.t_bufs = 1, p.a_slots = p.b_slots = p.x_slots = 2, p.epi_ring = 2048;
    auto grow = [&](int32_t& n, int by, int most, int bytes) {
      if (n + by > most || left < bytes) return false;
      left -= bytes, n += by;
      return true;
    };
    // B first where it is most of what a unit moves: 16384 fp16 rows, 768 x 1280, rank 128, float32 weights: 95.5 us
    // with x first, 92.8 with B; of rank 16 and float32 x, 114 and 120.
    if (t_chunks * (p.bank.wtype == kDtF32 ? 2 : 1) > 2) {
      while (grow(p.b_slots, 1, 4, kBPlane)) {
      }
    }
    while (grow(p.x_slots, 2, 6, 2 * x_slot)) {
    }
    grow(p.epi_ring, 2048, 4096, kEpiWarps * 2048);
    for (bool any = true; any;) {
      any = grow(p.b_slots, 1, kMaxSlots, kBPlane);
      any |= grow(p.a_slots, 1, kMaxSlots, a_slot);
      any |= grow(p.x_slots, 2, kMaxSlots, 2 * x_slot);
      any |= grow(p.t_bufs, 1, 2, t_buf);
    }
    smem = kMaxSmem - left;
    break;
  }
  if (!smem) return cudaErrorInvalidValue;
  constexpr int64_t kMaxLd = 1ll << 37;  // a tensor map's strides are below 2^40 bytes (a single row can have any)
  p.x_vec = (reinterpret_cast<uintptr_t>(p.a.x) & 15) == 0 && (p.a.ldx * sizeof(XT)) % 16 == 0 && p.a.ldx <= kMaxLd;
  p.x_four = (reinterpret_cast<uintptr_t>(p.a.x) | (uint64_t)(p.a.ldx * sizeof(XT))) % 4 == 0;
  const uintptr_t base = reinterpret_cast<uintptr_t>(p.a.base);
  p.b_copy = (base | (uint64_t)(p.a.ldb * sizeof(YT))) % 16 == 0 && p.a.ldb <= kMaxLd ? 16
             : (base | (uint64_t)(p.a.ldb * sizeof(YT))) % 4 == 0 ? 4 : 2;
  p.y_pair = p.bank.n_out % 2 == 0 &&
             (reinterpret_cast<uintptr_t>(p.a.y) | (uint64_t)(p.a.ldy * sizeof(YT))) % (2 * sizeof(YT)) == 0;
  // maps over as many rows as a plan can have; a box is loaded only where a unit has all its rows
  auto map = [&](CUtensorMap* m, const void* at, int type, int64_t cols, int64_t ld, uint32_t bc, uint32_t br,
                 CUtensorMapSwizzle swz) {
    const uint64_t dims[2] = {(uint64_t)cols, (uint64_t)(p.plan.max_rows > 0 ? p.plan.max_rows : 1)};
    const uint64_t strides[1] = {(uint64_t)ld * (type == kDtF32 ? 4 : 2)};
    const uint32_t box[2] = {bc, br};
    return tmap_nd(m, type == kDtF32 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32
                      : type == kDtF16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16,
                   at, 2, dims, strides, box, swz);
  };
  if (p.x_vec)
    e = map(&p.tm_x, p.a.x, XTYPE, p.bank.k_in, p.a.ldx, 128 / sizeof(XT), p.rt, CU_TENSOR_MAP_SWIZZLE_128B);
  if (e == cudaSuccess && base && p.b_copy == 16)
    e = map(&p.tm_b, p.a.base, dtype_of<YT>(), p.bank.n_out, p.a.ldb, 64, epi_rows<YT>(), CU_TENSOR_MAP_SWIZZLE_NONE);
  if (e != cudaSuccess) return e;
  e = cudaFuncSetAttribute(lowrank_tc_kernel<XT, YT>, cudaFuncAttributeMaxDynamicSharedMemorySize, kMaxSmem);
  if (e != cudaSuccess) return e;
  const int64_t n = units(p.rt, p.splits);
  lowrank_tc_kernel<XT, YT><<<(unsigned)(n < sms ? n : sms), kThreads, smem, st>>>(p);
  return cudaGetLastError();
}

}  // namespace

size_t lowrank_tile_bytes_a(int rank, int ka, int wtype, int xtype) {
  return (size_t)(ka / (xtype == kDtF32 ? KC : 64)) * rank * 128 * a_parts(xtype, wtype);
}
size_t lowrank_tile_bytes_b(int rp, int n_out, int wtype) {
  return (size_t)((n_out + 255) / 256 * 2) * ((rp + KC - 1) / KC) * kBPlane * (wtype == kDtF32 ? 2 : 1);
}

cudaError_t launch_lowrank_tiles(const LowRankBank& bank, cudaStream_t st) {
  if (bank.max_rank <= 0) return cudaSuccess;
  const int planes = bank.wtype == kDtF32 ? 2 : 1, rp = (bank.max_rank + 7) & ~7;
  const int64_t n = (int64_t)bank.max_rank * bank.ka + (int64_t)((bank.n_out + 255) / 256 * 2) * ((rp + KC - 1) / KC) * 128 * KC;
  const int f16 = a_parts(kDtF16, bank.wtype), bf16 = a_parts(kDtBF16, bank.wtype);
  for (int at = 0; at < bank.n_adapters; at += 65535) {  // the grid's second dimension
    const unsigned count = (unsigned)(bank.n_adapters - at < 65535 ? bank.n_adapters - at : 65535);
    const dim3 grid((unsigned)((n + 1023) / 1024 < 256 ? (n + 1023) / 1024 : 256), count), grid16(bank.max_rank, count);
    const LowRankAdapter* ads = bank.adapters + at;
    if (bank.wtype == kDtF32) {
      lowrank_tiles_kernel<float><<<grid, 256, 0, st>>>(ads, bank.k_in, bank.n_out, bank.ka, planes);
      lowrank_tiles16_kernel<float><<<grid16, 256, 0, st>>>(ads, bank.k_in, bank.ka, f16, bf16);
    } else if (bank.wtype == kDtF16) {
      lowrank_tiles_kernel<__half><<<grid, 256, 0, st>>>(ads, bank.k_in, bank.n_out, bank.ka, planes);
      lowrank_tiles16_kernel<__half><<<grid16, 256, 0, st>>>(ads, bank.k_in, bank.ka, f16, bf16);
    } else {
      lowrank_tiles_kernel<__nv_bfloat16><<<grid, 256, 0, st>>>(ads, bank.k_in, bank.n_out, bank.ka, planes);
      lowrank_tiles16_kernel<__nv_bfloat16><<<grid16, 256, 0, st>>>(ads, bank.k_in, bank.ka, f16, bf16);
    }
    const cudaError_t e = cudaGetLastError();
    if (e != cudaSuccess) return e;
  }
  return cudaSuccess;
}

cudaError_t launch_lowrank_tc(const LowRankBank& bank, const AdapterPlanDev& plan, int n_large, int n_small,
                              const LowRankArgs& a, uint32_t* err, cudaStream_t st) {
  if (n_large <= 0 && n_small <= 0) return cudaSuccess;
  TcParams p{};
  p.bank = bank;
  p.plan = plan;
  p.a = a;
  p.err = err;
  if (a.xtype == kDtF32 && a.ytype == kDtF32) return tc_types<float, float>(p, n_large, n_small, st);
  if (a.xtype == kDtF16 && a.ytype == kDtF16) return tc_types<__half, __half>(p, n_large, n_small, st);
  if (a.xtype == kDtF16 && a.ytype == kDtF32) return tc_types<__half, float>(p, n_large, n_small, st);
  if (a.xtype == kDtBF16 && a.ytype == kDtBF16) return tc_types<__nv_bfloat16, __nv_bfloat16>(p, n_large, n_small, st);
  if (a.xtype == kDtBF16 && a.ytype == kDtF32) return tc_types<__nv_bfloat16, float>(p, n_large, n_small, st);
  return cudaErrorInvalidValue;
}

}  // namespace sem
