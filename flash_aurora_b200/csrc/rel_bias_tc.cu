// bf16 window attention with a learned relative position bias on the tensor cores (tcgen05 UMMAs,
// accumulators in TMEM), forward and backward. The formulas are in rel_bias.cu.
//
// Both kernels are persistent, one CTA per SM over a contiguous range of (head, window) tiles in
// head-major order, so that a head's bias is fetched once per CTA and head and then stays on chip in
// fp32, in registers of the softmax warps. A window has 144 query rows and an M = 128 UMMA covers 128;
// rows 128..143 go through an M = 64 UMMA over rows 88..151 (the tile at an 88-row offset; what lies
// past the tile only reaches accumulator rows that nobody reads), which puts rows 128..135 into the third
// and rows 136..143 into the fourth TMEM quarter. Warps 4..11 own 16 query rows each of 0..127, warps 2
// and 3 eight rows each of 128..143, so that no SM sub-partition has three full softmax warps. A row's
// 144 keys sit in four threads of one warp (16x256b TMEM shape): row maxima and sums take two shuffles.
// Registers are moved from warps 0..3 to 4..11 (setmaxnreg).
//
// Region-id masks go through the tensor cores: with the ids of a window ranked, a K = 16 step adds
//   sum_r onehot(rank of query)[r] * (-c (1 - onehot(rank of key)[r])),  c = 100 / scale,
// exactly 0 to the raw logit of a pair of one region and -c to the others. c is a sum of two bf16 numbers, each
// with a column per rank (the best product of two, 16 ranks a step, is off by up to 0.028 of the 100 at scales
// like 0.39); a window of R regions takes ceil(R / 8) steps (none for R = 1), whatever its ids are. Shifts
// of all three axes make 8 regions.
// The per-logit alternative (compare and add in the softmax warps) cost 110 us of 350 on half-masked
// windows of 144 tokens. Byte masks are applied per logit.
//
// UMMAs are issued by one elected lane of a converged warp from precomputed descriptors: with a lane-0
// branch and descriptors built in place an UMMA took 75 cycles to issue whatever its shape, against
// 51 (128 x 64 x 16), 26 (64 x 16 x 16) and 75 (128 x 144 x 16) this way.
//
// P (and dS) are rounded to bf16 as tensor-core operands, the one rounding besides the outputs';
// logits, softmax statistics, dS in the bias gradient, and all accumulators are fp32.
#include <cuda.h>

#include <string>

#include "ptx.cuh"
#include "rel_bias.cuh"

namespace fa {
namespace relb {
namespace {

using namespace ptx;
using attn::kGroups;
using attn::kMaskedLog2;
using attn::kMaskU8;
using attn::kMaxN;
using attn::kNoMask;
using attn::kTileBytes;
using attn::kTimeoutNs;

constexpr int kThreads = 384;
// Registers per thread: launched at 168 (384 threads), then split between warps 0..3 and 4..11.
constexpr uint32_t kRegsLaunch = 168;
constexpr uint32_t kTmemCols = 512;
constexpr int kPChunk = kTileBytes;     // 64 keys x 144 rows of bf16, 128-byte swizzle
constexpr int kRow32 = kMaxN * 32;      // 16 columns x 144 rows of bf16, 32-byte swizzle
constexpr int kPBytes = 2 * kPChunk + kRow32;
constexpr int kMaskOpBytes = 2 * kRow32;  // A (queries) and B (keys) of one mask step
constexpr int kRemRow = 88;             // first row of the M = 64 block
constexpr uint32_t kRemOff = kRemRow * 128, kRemOff32 = kRemRow * 32;
constexpr uint32_t kLaneHalf = 16u << 16;  // second lane half of an M = 64 accumulator

constexpr uint32_t kIdescS = make_idesc(1, 128, kMaxN, false, false);
constexpr uint32_t kIdescS2 = make_idesc(1, 64, kMaxN, false, false);
constexpr uint32_t kIdescO = make_idesc(1, 128, 64, false, true);
constexpr uint32_t kIdescO2 = make_idesc(1, 64, 64, false, true);

// A descriptor whose operand starts `bytes` further on (the start field counts 16-byte units).
__device__ __forceinline__ uint64_t at(uint64_t desc, uint32_t bytes) { return desc + (uint64_t)(bytes >> 4); }

__device__ __forceinline__ bool elect_one() {
  uint32_t e;
  asm volatile("{ .reg .pred p; elect.sync _|p, 0xffffffff; selp.u32 %0, 1, 0, p; }" : "=r"(e));
  return e != 0;
}

// A whole warp's bounded wait: every lane gets the same answer, so that the warp stays together.
__device__ __forceinline__ bool warp_wait(uint32_t bar, uint32_t parity, volatile int* abort, int* status, int code) {
  return __all_sync(0xffffffffu, mbar_wait(bar, parity, abort, status, code, kTimeoutNs));
}
__device__ __forceinline__ bool warp_test(uint32_t bar, uint32_t parity) {
  return __all_sync(0xffffffffu, mbar_test_wait(bar, parity));
}

__device__ __forceinline__ float2 f2(uint32_t a, uint32_t b) {
  return make_float2(__uint_as_float(a), __uint_as_float(b));
}

// ------------------------------------------------------------------------------------------
// Rows and keys of one thread of a softmax warp. Warps 4..11: rows ra and rb = ra + 8. Warps 2 and 3
// (kRem): one row, which is the rb of warp 2's TMEM lanes and the ra of warp 3's. A thread holds keys
// 8j + 2 t0 and 8j + 2 t0 + 1 of each of its rows, j = 0..17.
// ------------------------------------------------------------------------------------------
template <bool kRem>
struct Lane {
  static constexpr int kRows = kRem ? 1 : 2;
  int t0, t1, row[kRows];
  bool hi;        // kRem: the row is in the rb registers
  uint32_t addr;  // TMEM lane offset of the warp's 16 lanes
  __device__ __forceinline__ Lane(int warp, int lane) {
    t0 = lane & 3;
    t1 = lane >> 2;
    if constexpr (kRem) {
      hi = warp == 2;
      row[0] = (hi ? 128 : 136) + t1;
      addr = (uint32_t)(32 * warp) << 16;
    } else {
      hi = false;
      const int base = 32 * (warp & 3) + 16 * ((warp - 4) >> 2);
      row[0] = base + t1;
      row[1] = base + 8 + t1;
      addr = (uint32_t)base << 16;
    }
  }
  // The pair of row r in the four accumulator registers of an 8-key block.
  __device__ __forceinline__ float2 pick(const uint32_t* v, int r) const {
    if constexpr (kRem) return hi ? f2(v[2], v[3]) : f2(v[0], v[1]);
    else return f2(v[2 * r], v[2 * r + 1]);
  }
  // Row r is row[0] + 8 r and row[0] % 8 = t1, so that the swizzle terms of both rows are equal.
  // Two bf16 of row r, 8-key block j, into a P-shaped operand tile.
  __device__ __forceinline__ void store_p(uint32_t sP, int j, int r, uint32_t v) const {
    if (j < 16)
      st_shared_u32(sP + row[0] * 128 + 4 * t0 + (((j & 7) ^ t1) << 4) + (j >> 3) * kPChunk + r * 1024, v);
    else
      st_shared_u32(sP + row[0] * 32 + 4 * t0 + ((((j & 1) ^ (t1 >> 2)) & 1) << 4) + 2 * kPChunk + r * 256, v);
  }
  // Row r of a 64-wide accumulator block (32 registers, 16x256b), scaled, to a staged bf16 tile.
  __device__ __forceinline__ void stage(uint32_t stg, const uint32_t (&o)[32], int r, float scale) const {
    const float2 s2 = make_float2(scale, scale);
#pragma unroll
    for (int jd = 0; jd < 8; ++jd) {
      const float2 y = __fmul2_rn(pick(&o[4 * jd], r), s2);
      st_shared_u32(stg + row[0] * 128 + 4 * t0 + ((jd ^ t1) << 4) + r * 1024, pack_bf16x2(y.x, y.y));
    }
  }
};

// The bias of this thread's pairs (see bias_rows).
template <bool kRem>
struct Bias {
  float2 b[18][Lane<kRem>::kRows];
  __device__ __forceinline__ void fetch(const Params& p, int h, const Lane<kRem>& l, int lane) {
    const float4* src = bias_rows(p, h, l.row[0], lane);
#pragma unroll
    for (int j = 0; j < 18; ++j) {
      if constexpr (kRem) {
        b[j][0] = __ldg(reinterpret_cast<const float2*>(src + j * 32) + (l.row[0] >= 136 ? 1 : 0));
      } else {
        const float4 v = __ldg(src + j * 32);
        b[j][0] = make_float2(v.x, v.y);
        b[j][1] = make_float2(v.z, v.w);
      }
    }
  }
};

// A byte mask's row of this thread (global memory), null past N.
template <bool kRem>
struct ByteMask {
  const uint8_t* m[Lane<kRem>::kRows];
  __device__ __forceinline__ void begin(const Params& p, const Lane<kRem>& l, int w) {
    const uint8_t* base = p.mask + (int64_t)(w % p.nW) * p.N * p.N;
#pragma unroll
    for (int r = 0; r < l.kRows; ++r) m[r] = l.row[r] < p.N ? base + l.row[r] * p.N : nullptr;
  }
  // Adds -100 (log2 domain) to the masked logits of 8-key block j.
  __device__ __forceinline__ void apply(const Params& p, const Lane<kRem>& l, int j, int r, float2& x) const {
    const int key = 8 * j + 2 * l.t0;
    if (m[r] && key < p.N && __ldg(m[r] + key)) x.x += kMaskedLog2;
    if (m[r] && key + 1 < p.N && __ldg(m[r] + key + 1)) x.y += kMaskedLog2;
  }
};

// ------------------------------------------------------------------------------------------
// Region masks. The ranks of a window's ids (kMaxN bytes, kNoRank past N) come with the tile's loads;
// one warp builds the operands, lane holds tokens lane + 32 m.
// ------------------------------------------------------------------------------------------
struct Regions {
  static constexpr uint32_t kOnes = 0x3f803f80u;  // two bf16
  int rank[5];
  int steps;  // mask K-steps: 0 for one region
  __device__ __forceinline__ void read(const uint8_t* ranks, int lane) {
    uint32_t most = 0;
#pragma unroll
    for (int m = 0; m < 5; ++m) {
      rank[m] = lane + 32 * m < kMaxN ? (int)ranks[lane + 32 * m] : kNoRank;
      most = max(most, rank[m] == kNoRank ? 0u : (uint32_t)rank[m]);
    }
    most = __reduce_max_sync(0xffffffffu, most);
    steps = most > 0 ? (int)(most >> 3) + 1 : 0;
  }
  // The A and B operands of step `st` (ranks 8 st .. 8 st + 7, a column of the high and one of the low part each;
  // rows of 16 bf16, 32-byte swizzle) at shared address `op`.
  __device__ __forceinline__ void build(uint32_t op, int st, int lane, uint32_t hi_bits, uint32_t lo_bits) const {
    const uint32_t hi2 = hi_bits | (hi_bits << 16), lo2 = lo_bits | (lo_bits << 16);
#pragma unroll
    for (int m = 0; m < 5; ++m) {
      if (m == 4 && lane >= kMaxN - 128) break;
      const int r = lane + 32 * m, slot = rank[m] - 8 * st;
      const uint32_t row = op + (uint32_t)r * 32u, sw = (uint32_t)((r >> 2) & 1) << 4;
      const bool in = rank[m] != kNoRank;
      const uint32_t h = in ? hi2 : 0u, l = in ? lo2 : 0u, half = slot & 1 ? 0xffff0000u : 0x0000ffffu;
      uint32_t hot[4];  // the rank's column; past N, and outside this step, none
#pragma unroll
      for (int e = 0; e < 4; ++e) hot[e] = (slot >> 1) == e ? half : 0u;
      const uint32_t a0 = hot[0] & kOnes, a1 = hot[1] & kOnes, a2 = hot[2] & kOnes, a3 = hot[3] & kOnes;
      st_shared_v4(row, a0, a1, a2, a3);  // the halves are alike, whichever the swizzle puts first
      st_shared_v4(row + 16u, a0, a1, a2, a3);
      st_shared_v4(row + kRow32 + sw, h & ~hot[0], h & ~hot[1], h & ~hot[2], h & ~hot[3]);
      st_shared_v4(row + kRow32 + (sw ^ 16u), l & ~hot[0], l & ~hot[1], l & ~hot[2], l & ~hot[3]);
    }
    fence_proxy_async_shared();
    __syncwarp();
  }
};

// `bytes` (a multiple of 16, 16-byte aligned on both sides) global -> shared, counted on an mbarrier.
__device__ __forceinline__ void bulk_load(uint32_t dst, const void* src, uint32_t bytes, uint32_t bar) {
  asm volatile("cp.async.bulk.shared::cta.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst), "l"(src),
               "r"(bytes), "r"(bar)
               : "memory");
}
__device__ __forceinline__ void load_ranks(uint32_t dst, const Params& p, int w, uint32_t bar) {
  bulk_load(dst, p.ranks + (int64_t)(w % p.nW) * kMaxN, kMaxN, bar);
}

struct Ctx {
  uint32_t sbase, bar0, tmem;
  uint8_t* smem;
  volatile int* abort;
  volatile int* steps;  // mask steps of a tile, by slot
  int t_begin, n_local;
  __device__ __forceinline__ uint32_t bar(int i) const { return bar0 + 8u * (uint32_t)i; }
};

// ------------------------------------------------------------------------------------------
// Forward.
//   warp 0      TMA producer: Q and K, V, 3-slot rings, and the mask operands; the output of a tile is
//               staged in its V slot and stored before the slot's reuse;
//   warp 1      TMEM owner and UMMA issuer:  S = Q K^T (M=128 and M=64), O = P V (M=128 and M=64);
//   warps 2-11  x = S scale + bias, softmax in the log2 domain, P to shared memory in bf16, then the
//               previous tile's output rows.
// ------------------------------------------------------------------------------------------
namespace fwd {

constexpr int kStages = 3;
constexpr int kQKBytes = 2 * kTileBytes;
constexpr int kStageBytes = 3 * kTileBytes;
constexpr int kOffP = kStages * kStageBytes;
constexpr int kOffMask = kOffP + kPBytes;  // two mask steps in flight
constexpr int kOffRanks = kOffMask + 2 * kMaskOpBytes;
constexpr int kOffBars = kOffRanks + kStages * kMaxN;
constexpr int kInfoSlots = 4;  // tile i + 4's steps are written after S of tile i + 2 is done, which follows tile i's
enum { kFullQK = 0, kEmptyQK = 3, kFullV = 6, kStaged = 9, kSFull = 12, kSFree, kPFull, kPEmpty, kOFull = 16,
       kOFree = 18, kDone = 20, kMaskFull = 21, kMaskEmpty = 23, kInfo = 25, kNumBars = kInfo + kInfoSlots };
constexpr int kSmem = kOffBars + kNumBars * 8 + 64 + 1024;
static_assert(kSmem <= 227 * 1024, "shared memory budget");
constexpr uint32_t kColS = 0, kColS2 = 160, kColO0 = 320, kColO1 = 384, kColO2 = 448;
constexpr uint32_t kRegsSmall = 120, kRegsMain = 192;
static_assert(4 * kRegsSmall + 8 * kRegsMain <= 12 * kRegsLaunch, "register split");
constexpr int kSoftmaxWarps = 10;

template <bool kRem, int kMask>
__device__ __forceinline__ void softmax_warps(const Params& p, const Ctx& c, int warp, int lane) {
  const Lane<kRem> l(warp, lane);
  constexpr int R = Lane<kRem>::kRows;
  const uint32_t tS = c.tmem + l.addr + (kRem ? kColS2 : kColS);
  const uint32_t sP = c.sbase + kOffP;
  Bias<kRem> bias;
  int cur_h = -1, prev = -1;
  float l_prev[R];

  auto epilogue = [&](int j) -> bool {
    const int ob = j & 1;
    if (!warp_wait(c.bar(kOFull + ob), (uint32_t)((j >> 1) & 1), c.abort, p.status, 101)) return false;
    tc_fence_after();
    uint32_t o[32];
    tmem_ld_16x256b_r32(c.tmem + l.addr + (kRem ? kColO2 + (ob ? kLaneHalf : 0u) : (ob ? kColO1 : kColO0)), o);
    tmem_wait_ld();
    tc_fence_before();
    __syncwarp();
    if (lane == 0) mbar_arrive(c.bar(kOFree + ob));
#pragma unroll
    for (int r = 0; r < R; ++r) l.stage(c.sbase + (j % kStages) * kStageBytes + kQKBytes, o, r, 1.f / l_prev[r]);
    fence_proxy_async_shared();
    __syncwarp();
    if (lane == 0) mbar_arrive(c.bar(kStaged + j % kStages));
    return true;
  };

  const float2 c2 = make_float2(p.scale_log2, p.scale_log2);
  bool ok = true;
  for (int i = 0; i < c.n_local; ++i) {
    const int t = c.t_begin + i, h = t / p.Bwin, w = t - h * p.Bwin;
    if (h != cur_h) {
      cur_h = h;
      bias.fetch(p, h, l, lane);
    }
    if (!warp_wait(c.bar(kSFull), (uint32_t)(i & 1), c.abort, p.status, 102)) { ok = false; break; }
    tc_fence_after();
    float2 x[18][R];
    if constexpr (kRem) {
#pragma unroll
      for (int q = 0; q < 9; q += 3) {
        uint32_t a[3][8];
#pragma unroll
        for (int e = 0; e < 3; ++e) tmem_ld_16x256b_r8(tS + 16 * (q + e), a[e]);
        tmem_wait_ld();
#pragma unroll
        for (int e = 0; e < 6; ++e) x[2 * q + e][0] = l.pick(&a[e >> 1][4 * (e & 1)], 0);
      }
    } else {
      uint32_t a[64], b[8];
      tmem_ld_16x256b_r64(tS, a);
      tmem_ld_16x256b_r8(tS + 128, b);
      tmem_wait_ld();
#pragma unroll
      for (int j = 0; j < 18; ++j)
#pragma unroll
        for (int r = 0; r < R; ++r) x[j][r] = j < 16 ? l.pick(&a[4 * (j & 15)], r) : l.pick(&b[4 * (j & 1)], r);
    }
    tc_fence_before();
    __syncwarp();
    if (lane == 0) mbar_arrive(c.bar(kSFree));
#pragma unroll
    for (int j = 0; j < 18; ++j)
#pragma unroll
      for (int r = 0; r < R; ++r) x[j][r] = __ffma2_rn(x[j][r], c2, bias.b[j][r]);
    if constexpr (kMask == kMaskU8) {
      ByteMask<kRem> mask;
      mask.begin(p, l, w);
#pragma unroll
      for (int j = 0; j < 18; ++j)
#pragma unroll
        for (int r = 0; r < R; ++r) mask.apply(p, l, j, r, x[j][r]);
    }
    float mx[R], sum[R];
    uint32_t pk[18][R];
#pragma unroll
    for (int r = 0; r < R; ++r) {
      mx[r] = -INFINITY;
#pragma unroll
      for (int j = 0; j < 18; ++j) mx[r] = fmax3(mx[r], x[j][r].x, x[j][r].y);
    }
#pragma unroll
    for (int r = 0; r < R; ++r) mx[r] = fmaxf(mx[r], __shfl_xor_sync(0xffffffffu, mx[r], 1));
#pragma unroll
    for (int r = 0; r < R; ++r) mx[r] = fmaxf(mx[r], __shfl_xor_sync(0xffffffffu, mx[r], 2));
    float2 s2[R];
#pragma unroll
    for (int r = 0; r < R; ++r) s2[r] = make_float2(0.f, 0.f);
#pragma unroll
    for (int j = 0; j < 18; ++j)
#pragma unroll
      for (int r = 0; r < R; ++r) {
        const float2 y = __fadd2_rn(x[j][r], make_float2(-mx[r], -mx[r]));
        const float2 e = make_float2(ex2(y.x), ex2(y.y));
        s2[r] = __fadd2_rn(s2[r], e);
        pk[j][r] = pack_bf16x2(e.x, e.y);
      }
#pragma unroll
    for (int r = 0; r < R; ++r) sum[r] = s2[r].x + s2[r].y;
#pragma unroll
    for (int r = 0; r < R; ++r) sum[r] += __shfl_xor_sync(0xffffffffu, sum[r], 1);
#pragma unroll
    for (int r = 0; r < R; ++r) sum[r] += __shfl_xor_sync(0xffffffffu, sum[r], 2);
    if (!warp_wait(c.bar(kPEmpty), (uint32_t)((i & 1) ^ 1), c.abort, p.status, 103)) { ok = false; break; }
#pragma unroll
    for (int j = 0; j < 18; ++j)
#pragma unroll
      for (int r = 0; r < R; ++r) l.store_p(sP, j, r, pk[j][r]);
    fence_proxy_async_shared();
    __syncwarp();
    if (lane == 0) mbar_arrive(c.bar(kPFull));
    if (p.stats && l.t0 == 0) {
      float2* st = p.stats + ((int64_t)w * p.H + h) * kMaxN;
#pragma unroll
      for (int r = 0; r < R; ++r) st[l.row[r]] = make_float2(mx[r], log2f(sum[r]));
    }
    if (prev >= 0 && !epilogue(prev)) { ok = false; break; }
    prev = i;
#pragma unroll
    for (int r = 0; r < R; ++r) l_prev[r] = sum[r];
  }
  if (ok && prev >= 0) epilogue(prev);
}

template <int kMask>
__device__ __forceinline__ void producer(const Params& p, const Ctx& c, int lane, const CUtensorMap* tmq,
                                         const CUtensorMap* tmk, const CUtensorMap* tmv, const CUtensorMap* tmo) {
  const int n = c.n_local;
  if (lane == 0) {
    tma_prefetch_desc(tmq);
    tma_prefetch_desc(tmk);
    tma_prefetch_desc(tmv);
  }
  auto store_out = [&](int j) {
    const int t = c.t_begin + j, h = t / p.Bwin;
    tma_store_4d(tmo, c.sbase + (j % kStages) * kStageBytes + kQKBytes, 0, 0, h, t - h * p.Bwin);
    bulk_commit_group();
  };
  int qk_issued = 0, v_issued = 0, jobs = 0;
  // Step i loads Q, K and the ranks of tile i, then V of tile i - 1, whose slot is freed about as late,
  // and builds the mask of tile i - 1, whose ranks have landed meanwhile.
  for (int i = 0; i <= n; ++i) {
    int ok = 1;
    if (lane == 0 && i < n) {
      const int t = c.t_begin + i, h = t / p.Bwin, w = t - h * p.Bwin, s = i % kStages;
      ok = mbar_wait(c.bar(kEmptyQK + s), (uint32_t)(((i / kStages) & 1) ^ 1), c.abort, p.status, 105, kTimeoutNs);
      if (ok) {
        const uint32_t dst = c.sbase + s * kStageBytes;
        mbar_arrive_expect_tx(c.bar(kFullQK + s), kQKBytes + (kMask == kGroups ? kMaxN : 0));
        tma_load_4d(dst, tmq, c.bar(kFullQK + s), 0, 0, h, w);
        tma_load_4d(dst + kTileBytes, tmk, c.bar(kFullQK + s), 0, 0, h, w);
        if constexpr (kMask == kGroups) load_ranks(c.sbase + kOffRanks + s * kMaxN, p, w, c.bar(kFullQK + s));
        ++qk_issued;
      }
    }
    if (lane == 0 && ok && i > 0) {
      const int j = i - 1, t = c.t_begin + j, h = t / p.Bwin, s = j % kStages;
      if (j >= kStages) {
        // The slot still holds the output of tile j - 3: store it and wait until it has been read.
        ok = mbar_wait(c.bar(kStaged + s), (uint32_t)(((j - kStages) / kStages) & 1), c.abort, p.status, 107, kTimeoutNs);
        if (ok) {
          store_out(j - kStages);
          bulk_wait_group_read0();
        }
      }
      if (ok) {
        mbar_arrive_expect_tx(c.bar(kFullV + s), kTileBytes);
        tma_load_4d(c.sbase + s * kStageBytes + kQKBytes, tmv, c.bar(kFullV + s), 0, 0, h, t - h * p.Bwin);
        ++v_issued;
      }
    }
    if (!__shfl_sync(0xffffffffu, ok, 0)) break;
    if (kMask == kGroups && i > 0) {
      const int j = i - 1, s = j % kStages;
      if (!warp_wait(c.bar(kFullQK + s), (uint32_t)((j / kStages) & 1), c.abort, p.status, 113)) break;
      Regions reg;
      reg.read(c.smem + kOffRanks + s * kMaxN, lane);
      if (lane == 0) {
        c.steps[j % kInfoSlots] = reg.steps;
        mbar_arrive(c.bar(kInfo + j % kInfoSlots));
      }
      for (int st = 0; st < reg.steps; ++st, ++jobs) {
        const int b = jobs & 1;
        if (!warp_wait(c.bar(kMaskEmpty + b), (uint32_t)(((jobs >> 1) & 1) ^ 1), c.abort, p.status, 104)) { ok = 0; break; }
        reg.build(c.sbase + kOffMask + b * kMaskOpBytes, st, lane, p.mask_hi, p.mask_lo);
        if (lane == 0) mbar_arrive(c.bar(kMaskFull + b));
      }
      if (!ok) break;
    }
  }
  if (lane == 0) {
    // Never leave with copies in flight (bounded, also after an abort).
    int no_abort = 0;
    for (int j = qk_issued > kStages ? qk_issued - kStages : 0; j < qk_issued; ++j)
      mbar_wait(c.bar(kFullQK + j % kStages), (uint32_t)((j / kStages) & 1), &no_abort, p.status, 106, kTimeoutNs);
    for (int j = v_issued > kStages ? v_issued - kStages : 0; j < v_issued; ++j)
      mbar_wait(c.bar(kFullV + j % kStages), (uint32_t)((j / kStages) & 1), &no_abort, p.status, 108, kTimeoutNs);
    for (int j = n > kStages ? n - kStages : 0; j < n; ++j) {
      if (!mbar_wait(c.bar(kStaged + j % kStages), (uint32_t)((j / kStages) & 1), c.abort, p.status, 109, kTimeoutNs))
        break;
      store_out(j);
    }
    bulk_wait_group0();
  }
}

// S and PV in whatever order their inputs become ready.
template <int kMask>
__device__ __forceinline__ void issuer(const Params& p, const Ctx& c) {
  const int n = c.n_local;
  const bool leader = elect_one();
  const uint64_t dQ = desc_sw128(c.sbase, 16, 1024), dV = desc_sw128(c.sbase + kQKBytes, kTileBytes, 1024);
  const uint64_t dP = desc_sw128(c.sbase + kOffP, 16, 1024), dP32 = desc_sw32(c.sbase + kOffP + 2 * kPChunk, 256);
  const uint64_t dM = desc_sw32(c.sbase + kOffMask, 256);
  int ns = 0, npv = 0, jobs = 0;
  uint64_t t_last = cycles();
  uint32_t idle = 0;
  bool ok = true;
  while (ok && npv < n) {
    bool progressed = false;
    if (ns < n) {
      const int s = ns % kStages;
      bool ready = warp_test(c.bar(kFullQK + s), (uint32_t)((ns / kStages) & 1)) &&
                   warp_test(c.bar(kSFree), (uint32_t)((ns & 1) ^ 1));
      if constexpr (kMask == kGroups)
        ready = ready && warp_test(c.bar(kInfo + ns % kInfoSlots), (uint32_t)((ns / kInfoSlots) & 1));
      if (ready) {
        tc_fence_after();
        const uint64_t q = at(dQ, s * kStageBytes), k = at(q, kTileBytes);
        if (leader) {
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            umma_f16(c.tmem + kColS, at(q, e * 32), at(k, e * 32), kIdescS, e > 0 ? 1u : 0u);
            umma_f16(c.tmem + kColS2, at(q, kRemOff + e * 32), at(k, e * 32), kIdescS2, e > 0 ? 1u : 0u);
          }
        }
        if constexpr (kMask == kGroups) {
          for (int st = c.steps[ns % kInfoSlots]; st > 0; --st, ++jobs) {
            const int b = jobs & 1;
            ok = warp_wait(c.bar(kMaskFull + b), (uint32_t)((jobs >> 1) & 1), c.abort, p.status, 112);
            if (!ok) break;
            tc_fence_after();
            if (leader) {
              const uint64_t a = at(dM, b * kMaskOpBytes), bb = at(a, kRow32);
              umma_f16(c.tmem + kColS, a, bb, kIdescS, 1u);
              umma_f16(c.tmem + kColS2, at(a, kRemOff32), bb, kIdescS2, 1u);
              umma_commit(c.bar(kMaskEmpty + b));
            }
          }
          if (!ok) break;
        }
        if (leader) {
          umma_commit(c.bar(kSFull));
          umma_commit(c.bar(kEmptyQK + s));
        }
        ++ns;
        progressed = true;
      }
    }
    if (npv < ns) {
      const int s = npv % kStages, ob = npv & 1;
      if (warp_test(c.bar(kPFull), (uint32_t)(npv & 1)) && warp_test(c.bar(kFullV + s), (uint32_t)((npv / kStages) & 1)) &&
          warp_test(c.bar(kOFree + ob), (uint32_t)(((npv >> 1) & 1) ^ 1))) {
        tc_fence_after();
        if (leader) {
          const uint64_t v = at(dV, s * kStageBytes);
          const uint32_t o = c.tmem + (ob ? kColO1 : kColO0), o2 = c.tmem + kColO2 + (ob ? kLaneHalf : 0u);
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const uint32_t off = (e >> 2) * kPChunk + (e & 3) * 32;
            umma_f16(o, at(dP, off), at(v, e * 2048), kIdescO, e > 0 ? 1u : 0u);
            umma_f16(o2, at(dP, off + kRemOff), at(v, e * 2048), kIdescO2, e > 0 ? 1u : 0u);
          }
          umma_f16(o, dP32, at(v, 8 * 2048), kIdescO, 1u);  // keys 128..143
          umma_f16(o2, at(dP32, kRemOff32), at(v, 8 * 2048), kIdescO2, 1u);
          umma_commit(c.bar(kOFull + ob));
          umma_commit(c.bar(kPEmpty));
        }
        ++npv;
        progressed = true;
      }
    }
    if (progressed) {
      idle = 0;
      t_last = cycles();
    } else if ((++idle & 63u) == 0) {
      bool stop = *c.abort != 0;
      if (cycles() - t_last > ns_to_cycles(kTimeoutNs)) {
        atomicCAS(p.status, 0, 110);
        *c.abort = 1;
        stop = true;
      }
      if (__any_sync(0xffffffffu, stop)) break;
    }
  }
  if (leader) umma_commit(c.bar(kDone));
  int no_abort = 0;
  mbar_wait(c.bar(kDone), 0, &no_abort, p.status, 111, kTimeoutNs);
  __syncwarp();
}

template <int kMask>
__global__ void __launch_bounds__(kThreads, 1)
rel_bias_fwd_tc_kernel(const __grid_constant__ CUtensorMap tmq, const __grid_constant__ CUtensorMap tmk,
                       const __grid_constant__ CUtensorMap tmv, const __grid_constant__ CUtensorMap tmo,
                       const Params p) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + kOffBars);
  int* words = reinterpret_cast<int*>(bars + kNumBars);  // abort flag, TMEM address, mask steps
  Ctx c;
  c.smem = smem;
  c.sbase = smem_u32(smem);
  c.bar0 = smem_u32(bars);
  c.abort = words;
  c.steps = words + 4;
  c.t_begin = tile_begin(p.num_tiles);
  c.n_local = tile_end(p.num_tiles) - c.t_begin;
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    *words = 0;
    for (int b = 0; b < kNumBars; ++b) {
      const bool all = (b >= kStaged && b < kStaged + kStages) || b == kSFree || b == kPFull || b == kOFree || b == kOFree + 1;
      mbar_init(c.bar(b), all ? kSoftmaxWarps : 1);
    }
    fence_mbarrier_init();
  }
  if (warp == 1) {
    tmem_alloc(smem_u32(words + 1), kTmemCols);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  c.tmem = (uint32_t)*reinterpret_cast<volatile int*>(words + 1);

  if (warp >= 4) {
    warpgroup_reg_alloc<kRegsMain>();
    softmax_warps<false, kMask>(p, c, warp, lane);
  } else {
    warpgroup_reg_dealloc<kRegsSmall>();
    if (warp >= 2) softmax_warps<true, kMask>(p, c, warp, lane);
    else if (warp == 1) issuer<kMask>(p, c);
    else producer<kMask>(p, c, lane, &tmq, &tmk, &tmv, &tmo);
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(c.tmem, kTmemCols);
  }
}

}  // namespace fwd

// ------------------------------------------------------------------------------------------
// Backward. Per tile:
//   S = Q K^T, dP = dO V^T                     M=128 (rows 0..127) and M=64 (rows 88..151), N=144
//   pass 1   P = exp2(x - max - log2 sum) from the forward's row statistics; delta = sum_k P dP; P
//            replaces S in TMEM (fp32) and goes to shared memory in bf16
//   dV = P^T dO                                runs while pass 2 computes
//   pass 2   dS = P (dP - delta), added to the head's bias gradient (fp32, in registers: 72 of each
//            thread of warps 4..11), and to shared memory in bf16
//   dQ = dS K, dK = dS^T Q                     dV and dQ are drained meanwhile; then S and dP of the next tile,
//                                              while dK is drained. Rows 128..143, whose S comes last, are the
//                                              last K-step of dV and dK and no part of the M=128 dQ, so nothing
//                                              waits for them early
// dV, dK, dQ of keys / rows 0..127 are M=128 UMMAs (P and dS are read MN-major for dV and dK); those
// of 128..143 are computed transposed, (64 head dims) x (16 rows), as M=64, N=16 UMMAs, at half
// the cost of an M=64, N=64 block.
// TMEM columns: S / P 0..143, dP 144..287, the M=64 blocks of S and dP in the two lane halves of 288..431,
// dV 432..495, the transposed remainders of dV and dK in the lane halves of 496..511. Over S, once pass 2 of
// rows 0..127 has read it, dQ 0..63; over the M=64 blocks, once pass 2 of rows 128..143 has, dK 288..351 and
// dQ's transposed remainder 416..431.
// Outputs are staged in the tile's own slots (dV over V, dK over K, dQ over dO, which dV was the last to
// read) and stored by warp 0 before it loads the tile after next into them. Two input slots, P and dS fill shared memory (230 KB);
// the mask operands of a tile are built in the dS buffer, which is free between dK of the tile before and
// the tile's own pass 2.
// ------------------------------------------------------------------------------------------
namespace bwd {

constexpr int kStages = 2;
constexpr int kOffQ = 0, kOffK = kTileBytes, kOffV = 2 * kTileBytes, kOffG = 3 * kTileBytes;
constexpr int kStageBytes = 4 * kTileBytes;
// P, the small things in the gap before the next 1024-byte boundary, dS, the row statistics of one tile.
constexpr int kOffP = kStages * kStageBytes;
constexpr int kOffRanks = kOffP + kPBytes;
constexpr int kOffBars = kOffRanks + kStages * kMaxN;
constexpr int kOffDs = (kOffP + kPBytes + 1023) / 1024 * 1024;
constexpr int kOffStats = kOffDs + kPBytes, kStatsBytes = kMaxN * 8;
constexpr int kMaskSlots = 4;  // mask steps built at once in the dS buffer
static_assert(kMaskSlots * kMaskOpBytes <= kPBytes, "mask operands fit the dS buffer");
enum { kFull = 0, kStaged = 2, kSMain = 4, kSRem, kPMain, kPRem, kDvFull, kDsMain, kDsRem, kDqFull, kRemFull, kDkFull,
       kDqFree, kTFree, kStats, kInfo, kMaskMore, kMaskEmpty, kDone, kNumBars };
static_assert(kOffBars + kNumBars * 8 + 24 <= kOffDs, "barriers and words fit the gap");
constexpr int kSmem = kOffStats + kStatsBytes;  // no slack: the kernel checks the base's alignment
static_assert(kSmem <= 227 * 1024, "shared memory budget");
constexpr uint32_t kColS = 0, kColP = 144, kColS2 = 288, kColDv = 432, kColRem = 496;
constexpr uint32_t kColDq = kColS, kColDk = kColS2, kColDq2 = kColS2 + 128;
constexpr uint32_t kRegsSmall = 120, kRegsMain = 192;
static_assert(4 * kRegsSmall + 8 * kRegsMain <= 12 * kRegsLaunch, "register split");
constexpr uint32_t kIdescT = make_idesc(1, 128, 64, true, true);    // A and B MN-major: dV, dK
constexpr uint32_t kIdescRemT = make_idesc(1, 64, 16, true, true);  // (64 dims) x (16 keys)
constexpr uint32_t kIdescRemQ = make_idesc(1, 64, 16, true, false); // (64 dims) x (16 queries)

// A transposed remainder block, (64 head dims) x (rows 128..143), of this warp's TMEM quarter: 16
// head dims, scaled, into rows 128..143 of a staged bf16 tile.
__device__ __forceinline__ void stage_rem(uint32_t taddr, uint32_t stg, int warp, int lane, float scale) {
  const int quarter = warp & 3, t0 = lane & 3, t1 = lane >> 2;
  uint32_t r[8];
  tmem_ld_16x256b_r8(taddr + ((uint32_t)(32 * quarter) << 16), r);
  tmem_wait_ld();
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const int row = 128 + 8 * (e >> 2) + 2 * t0 + (e & 1);
    const int d = 16 * quarter + t1 + 8 * ((e >> 1) & 1);
    const __nv_bfloat16 v = __float2bfloat16_rn(__uint_as_float(r[e]) * scale);
    asm volatile("st.shared.u16 [%0], %1;" ::"r"(stg + (uint32_t)(row * 128 + (((d >> 3) ^ (row & 7)) << 4) + (d & 7) * 2)),
                 "h"(__bfloat16_as_ushort(v))
                 : "memory");
  }
}

// The blocks of two accumulators in turn: 8 columns with the next block's loads in flight for warps 4..11,
// 16 columns without for warps 2 and 3, which have half the rows and fewer registers.
template <bool kRem>
struct TmemBlocks {
  static constexpr int kRegs = kRem ? 8 : 4;
  uint32_t a, b;
  uint32_t va[kRegs], vb[kRegs];
  __device__ __forceinline__ TmemBlocks(uint32_t a_, uint32_t b_) : a(a_), b(b_) {
    if constexpr (!kRem) load(0);
  }
  __device__ __forceinline__ void load(int j) {
    if constexpr (kRem) {
      tmem_ld_16x256b_r8(a + 8 * j, va);
      tmem_ld_16x256b_r8(b + 8 * j, vb);
    } else {
      tmem_ld_16x256b_r4(a + 8 * j, va);
      tmem_ld_16x256b_r4(b + 8 * j, vb);
    }
  }
  // The registers of 8-key block j, j = 0..17 in order.
  __device__ __forceinline__ void next(int j, uint32_t (&ca)[4], uint32_t (&cb)[4]) {
    const int o = kRem ? 4 * (j & 1) : 0;
    if (kRem && (j & 1) == 0) load(j);
    if (!kRem || (j & 1) == 0) tmem_wait_ld();
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      ca[e] = va[o + e];
      cb[e] = vb[o + e];
    }
    if constexpr (!kRem) {
      if (j < 17) load(j + 1);
    }
  }
};

template <bool kRem, int kMask>
__device__ __forceinline__ void softmax_warps(const Params& p, const Ctx& c, int warp, int lane) {
  const Lane<kRem> l(warp, lane);
  constexpr int R = Lane<kRem>::kRows;
  const uint32_t tS = c.tmem + l.addr + (kRem ? kColS2 : kColS);
  const uint32_t tP = c.tmem + l.addr + (kRem ? kColS2 + kLaneHalf : kColP);
  const uint32_t sP = c.sbase + kOffP, sDs = c.sbase + kOffDs;
  const float2 c2 = make_float2(p.scale_log2, p.scale_log2);
  Bias<kRem> bias;
  float2 grad[18][R];  // the head's bias gradient of this thread's pairs
  int cur_h = -1;
  auto flush = [&](int h) {
    if (!p.slots) return;
    float4* slot = slot_rows(p, blockIdx.x + h, l.row[0], lane);
#pragma unroll
    for (int j = 0; j < 18; ++j) {
      if constexpr (kRem) reinterpret_cast<float2*>(slot + j * 32)[l.row[0] >= 136 ? 1 : 0] = grad[j][0];
      else slot[j * 32] = make_float4(grad[j][0].x, grad[j][0].y, grad[j][1].x, grad[j][1].y);
    }
  };
  int h = c.t_begin / p.Bwin, w = c.t_begin - h * p.Bwin;
  for (int i = 0; i < c.n_local; ++i, ++w) {
    const int s = i & 1;
    const uint32_t par = (uint32_t)(i & 1);
    const uint32_t slot = c.sbase + s * kStageBytes;
    if (w == p.Bwin) {
      w = 0;
      ++h;
    }
    if (h != cur_h) {
      if (cur_h >= 0) flush(cur_h);
      cur_h = h;
#pragma unroll
      for (int j = 0; j < 18; ++j)
#pragma unroll
        for (int r = 0; r < R; ++r) grad[j][r] = make_float2(0.f, 0.f);
      bias.fetch(p, h, l, lane);
    }
    // Row statistics; +inf past N makes the rows' P zero.
    float2 mx[R], lg[R], d2[R];
    if (!warp_wait(c.bar(kStats), par, c.abort, p.status, 120)) return;
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const float2 v = l.row[r] < p.N ? reinterpret_cast<const float2*>(c.smem + kOffStats)[l.row[r]]
                                      : make_float2(INFINITY, 0.f);
      mx[r] = make_float2(-v.x, -v.x);
      lg[r] = make_float2(-v.y, -v.y);
      d2[r] = make_float2(0.f, 0.f);
    }
    ByteMask<kRem> mask;
    if constexpr (kMask == kMaskU8) mask.begin(p, l, w);
    if (!warp_wait(c.bar(kRem ? kSRem : kSMain), par, c.abort, p.status, 121)) return;
    tc_fence_after();
    // Pass 1.
    TmemBlocks<kRem> blk(tS, tP);
#pragma unroll
    for (int j = 0; j < 18; ++j) {
      uint32_t cs[4], cg[4];
      blk.next(j, cs, cg);
#pragma unroll
      for (int r = 0; r < R; ++r) {
        float2 x = __ffma2_rn(l.pick(cs, r), c2, bias.b[j][r]);
        if constexpr (kMask == kMaskU8) mask.apply(p, l, j, r, x);
        x = __fadd2_rn(__fadd2_rn(x, mx[r]), lg[r]);
        const float2 pr = make_float2(ex2(x.x), ex2(x.y));
        d2[r] = __ffma2_rn(pr, l.pick(cg, r), d2[r]);
        l.store_p(sP, j, r, pack_bf16x2(pr.x, pr.y));
        cs[2 * r] = __float_as_uint(pr.x);
        cs[2 * r + 1] = __float_as_uint(pr.y);
        if constexpr (kRem) {  // the lanes' other row is nobody's
          cs[2] = cs[0];
          cs[3] = cs[1];
        }
      }
      tmem_st_16x256b_r4(tS + 8 * j, cs);
    }
    tmem_wait_st();
    fence_proxy_async_shared();
    __syncwarp();
    if (lane == 0) mbar_arrive(c.bar(kRem ? kPRem : kPMain));
#pragma unroll
    for (int r = 0; r < R; ++r) {
      float d = d2[r].x + d2[r].y;
      d += __shfl_xor_sync(0xffffffffu, d, 1);
      d += __shfl_xor_sync(0xffffffffu, d, 2);
      d2[r] = make_float2(-d, -d);
    }
    // Pass 2. The dS buffer held the tile's mask operands until the last product of S was done.
    if (kMask == kGroups && !kRem && !warp_wait(c.bar(kSRem), par, c.abort, p.status, 119)) return;
    TmemBlocks<kRem> blk2(tS, tP);
#pragma unroll
    for (int j = 0; j < 18; ++j) {
      uint32_t cs[4], cg[4];
      blk2.next(j, cs, cg);
#pragma unroll
      for (int r = 0; r < R; ++r) {
        const float2 g = __fmul2_rn(l.pick(cs, r), __fadd2_rn(l.pick(cg, r), d2[r]));
        grad[j][r] = __fadd2_rn(grad[j][r], g);
        l.store_p(sDs, j, r, pack_bf16x2(g.x, g.y));
      }
    }
    fence_proxy_async_shared();
    tc_fence_before();
    __syncwarp();
    if (lane == 0) mbar_arrive(c.bar(kRem ? kDsRem : kDsMain));
    if constexpr (!kRem) {
      uint32_t o[32];
      auto drain = [&](int bar, int code, uint32_t col, uint32_t stg, float scale) -> bool {
        if (!warp_wait(c.bar(bar), par, c.abort, p.status, code)) return false;
        tc_fence_after();
        tmem_ld_16x256b_r32(c.tmem + l.addr + col, o);
        tmem_wait_ld();
#pragma unroll
        for (int r = 0; r < R; ++r) l.stage(stg, o, r, scale);
        return true;
      };
      if (!drain(kDvFull, 122, kColDv, slot + kOffV, 1.f)) return;
      if (warp < 8) stage_rem(c.tmem + kColRem, slot + kOffV, warp, lane, 1.f);
      if (!drain(kDqFull, 123, kColDq, slot + kOffG, p.scale)) return;
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(c.bar(kDqFree));
      if (!warp_wait(c.bar(kRemFull), par, c.abort, p.status, 118)) return;
      tc_fence_after();
      // The remainders; the K tile's last reader was dQ's.
      if (warp >= 8) stage_rem(c.tmem + kColDq2, slot + kOffG, warp, lane, p.scale);
      else stage_rem(c.tmem + kColRem + kLaneHalf, slot + kOffK, warp, lane, p.scale);
      if (!drain(kDkFull, 124, kColDk, slot + kOffK, p.scale)) return;
      fence_proxy_async_shared();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) {
        mbar_arrive(c.bar(kTFree));
        mbar_arrive(c.bar(kStaged + s));
      }
    }
  }
  if (cur_h >= 0) flush(cur_h);
}

template <int kMask>
__device__ __forceinline__ void producer(const Params& p, const Ctx& c, int lane, const CUtensorMap* tmq,
                                         const CUtensorMap* tmk, const CUtensorMap* tmv, const CUtensorMap* tmg,
                                         const CUtensorMap* tmdq, const CUtensorMap* tmdk, const CUtensorMap* tmdv) {
  const int n = c.n_local;
  int issued = 0, stats_issued = 0, more = 0;
  auto load = [&](int i) {
    const int t = c.t_begin + i, h = t / p.Bwin, w = t - h * p.Bwin;
    const uint32_t bar = c.bar(kFull + (i & 1)), slot = c.sbase + (i & 1) * kStageBytes;
    mbar_arrive_expect_tx(bar, kStageBytes + (kMask == kGroups ? kMaxN : 0));
    tma_load_4d(slot + kOffQ, tmq, bar, 0, 0, h, w);
    tma_load_4d(slot + kOffK, tmk, bar, 0, 0, h, w);
    tma_load_4d(slot + kOffG, tmg, bar, 0, 0, h, w);
    tma_load_4d(slot + kOffV, tmv, bar, 0, 0, h, w);
    if constexpr (kMask == kGroups) load_ranks(c.sbase + kOffRanks + (i & 1) * kMaxN, p, w, bar);
    ++issued;
  };
  auto store = [&](int j) {
    const int t = c.t_begin + j, h = t / p.Bwin, w = t - h * p.Bwin;
    const uint32_t slot = c.sbase + (j & 1) * kStageBytes;
    tma_store_4d(tmdq, slot + kOffG, 0, 0, h, w);
    tma_store_4d(tmdk, slot + kOffK, 0, 0, h, w);
    tma_store_4d(tmdv, slot + kOffV, 0, 0, h, w);
    bulk_commit_group();
  };
  auto load_stats = [&](int i) {
    const int t = c.t_begin + i, h = t / p.Bwin;
    mbar_arrive_expect_tx(c.bar(kStats), kStatsBytes);
    bulk_load(c.sbase + kOffStats, p.stats + ((int64_t)(t - h * p.Bwin) * p.H + h) * kMaxN, kStatsBytes, c.bar(kStats));
    ++stats_issued;
  };
  if (lane == 0) {
    if (n > 0) load_stats(0);
    for (int i = 0; i < kStages && i < n; ++i) load(i);
  }
  for (int i = 0; i < n; ++i) {
    int ok = 1;
    if constexpr (kMask == kGroups) {
      if (!warp_wait(c.bar(kFull + (i & 1)), (uint32_t)((i >> 1) & 1), c.abort, p.status, 137)) break;
      Regions now;
      now.read(c.smem + kOffRanks + (i & 1) * kMaxN, lane);
      // The dS buffer is free once dK of the tile before is done.
      if (now.steps > 0 && i > 0 && !warp_wait(c.bar(kDkFull), (uint32_t)((i - 1) & 1), c.abort, p.status, 133)) break;
      for (int st = 0; st < now.steps && ok; ++st) {
        if (st > 0 && st % kMaskSlots == 0) {  // more than 32 regions: wait until the slots have been read
          if (lane == 0) {
            if (st == kMaskSlots) {
              c.steps[i & 1] = now.steps;
              mbar_arrive(c.bar(kInfo));
            } else {
              mbar_arrive(c.bar(kMaskMore));
            }
          }
          ok = warp_wait(c.bar(kMaskEmpty), (uint32_t)(more & 1), c.abort, p.status, 134);
          ++more;
        }
        if (ok) now.build(c.sbase + kOffDs + (st % kMaskSlots) * kMaskOpBytes, st, lane, p.mask_hi, p.mask_lo);
      }
      if (!ok) break;
      if (lane == 0) {
        if (now.steps <= kMaskSlots) {
          c.steps[i & 1] = now.steps;
          mbar_arrive(c.bar(kInfo));
        } else {
          mbar_arrive(c.bar(kMaskMore));
        }
      }
    }
    if (i > 0 && i + 1 < n) {
      // Tile i - 1's outputs leave its slot, tile i + 1's inputs enter it.
      if (lane == 0) {
        ok = mbar_wait(c.bar(kStaged + ((i - 1) & 1)), (uint32_t)(((i - 1) >> 1) & 1), c.abort, p.status, 125, kTimeoutNs);
        if (ok) {
          store(i - 1);
          bulk_wait_group_read0();
          load(i + 1);
        }
      }
      if (!__shfl_sync(0xffffffffu, ok, 0)) break;
    }
    if (i + 1 < n) {
      // Every softmax warp has read tile i's statistics once its P is there.
      if (lane == 0) {
        ok = mbar_wait(c.bar(kPMain), (uint32_t)(i & 1), c.abort, p.status, 138, kTimeoutNs) &&
             mbar_wait(c.bar(kPRem), (uint32_t)(i & 1), c.abort, p.status, 138, kTimeoutNs);
        if (ok) load_stats(i + 1);
      }
      if (!__shfl_sync(0xffffffffu, ok, 0)) break;
    }
  }
  if (lane == 0) {
    // Never leave with copies in flight (bounded, also after an abort).
    int no_abort = 0;
    if (stats_issued > 0) mbar_wait(c.bar(kStats), (uint32_t)((stats_issued - 1) & 1), &no_abort, p.status, 139, kTimeoutNs);
    for (int j = issued > kStages ? issued - kStages : 0; j < issued; ++j)
      mbar_wait(c.bar(kFull + (j & 1)), (uint32_t)((j >> 1) & 1), &no_abort, p.status, 126, kTimeoutNs);
    for (int j = n > kStages ? n - kStages : 0; j < n; ++j) {
      if (!mbar_wait(c.bar(kStaged + (j & 1)), (uint32_t)((j >> 1) & 1), c.abort, p.status, 127, kTimeoutNs)) break;
      store(j);
    }
    bulk_wait_group0();
  }
}

template <int kMask>
__device__ __forceinline__ void issuer(const Params& p, const Ctx& c) {
  const bool leader = elect_one();
  const uint32_t sP = c.sbase + kOffP, sDs = c.sbase + kOffDs;
  // K-major (row) and MN-major (column) views of the input tiles, P and dS; 32-byte-swizzled parts.
  const uint64_t row0 = desc_sw128(c.sbase, 16, 1024), col0 = desc_sw128(c.sbase, kTileBytes, 1024);
  const uint64_t pT = desc_sw128(sP, kPChunk, 1024), p32 = desc_sw32(sP + 2 * kPChunk, 256);
  const uint64_t dsT = desc_sw128(sDs, kPChunk, 1024), ds = desc_sw128(sDs, 16, 1024);
  const uint64_t ds32 = desc_sw32(sDs + 2 * kPChunk, 256), mask0 = desc_sw32(sDs, 256);
  int more = 0;
  for (int i = 0; i < c.n_local; ++i) {
    const int s = i & 1;
    const uint32_t par = (uint32_t)(i & 1), slot = s * kStageBytes;
    const uint64_t qr = at(row0, slot + kOffQ), kr = at(row0, slot + kOffK), vr = at(row0, slot + kOffV),
                   gr = at(row0, slot + kOffG);
    const uint64_t qc = at(col0, slot + kOffQ), kc = at(col0, slot + kOffK), gc = at(col0, slot + kOffG);
    // S and dP of rows 0..127 as soon as the inputs are there and dQ of the tile before has been drained
    // (pass 2 of that tile is done); the M=64 blocks once its dK has been.
    if (!warp_wait(c.bar(kFull + s), (uint32_t)((i >> 1) & 1), c.abort, p.status, 128)) break;
    if (!warp_wait(c.bar(kDqFree), par ^ 1u, c.abort, p.status, 115)) break;
    tc_fence_after();
    if (leader) {
#pragma unroll
      for (int e = 0; e < 4; ++e) umma_f16(c.tmem + kColS, at(qr, e * 32), at(kr, e * 32), kIdescS, e > 0 ? 1u : 0u);
#pragma unroll
      for (int e = 0; e < 4; ++e) umma_f16(c.tmem + kColP, at(gr, e * 32), at(vr, e * 32), kIdescS, e > 0 ? 1u : 0u);
    }
    int steps = 0;
    if constexpr (kMask == kGroups) {
      if (!warp_wait(c.bar(kInfo), par, c.abort, p.status, 135)) break;
      tc_fence_after();
      steps = c.steps[i & 1];
    }
    const bool together = steps > kMaskSlots;  // the operands come in rounds: both blocks take each
    if (leader && !together) {
      for (int st = 0; st < steps; ++st) {
        const uint64_t a = at(mask0, st * kMaskOpBytes);
        umma_f16(c.tmem + kColS, a, at(a, kRow32), kIdescS, 1u);
      }
      umma_commit(c.bar(kSMain));
    }
    if (!warp_wait(c.bar(kTFree), par ^ 1u, c.abort, p.status, 129)) break;
    tc_fence_after();
    if (leader) {
#pragma unroll
      for (int e = 0; e < 4; ++e)
        umma_f16(c.tmem + kColS2, at(qr, kRemOff + e * 32), at(kr, e * 32), kIdescS2, e > 0 ? 1u : 0u);
#pragma unroll
      for (int e = 0; e < 4; ++e)
        umma_f16(c.tmem + kColS2 + kLaneHalf, at(gr, kRemOff + e * 32), at(vr, e * 32), kIdescS2, e > 0 ? 1u : 0u);
    }
    if constexpr (kMask == kGroups) {
      bool ok = true;
      for (int st = 0; st < steps; ++st) {
        if (st > 0 && st % kMaskSlots == 0) {
          if (leader) umma_commit(c.bar(kMaskEmpty));
          ok = warp_wait(c.bar(kMaskMore), (uint32_t)(more & 1), c.abort, p.status, 136);
          ++more;
          if (!ok) break;
          tc_fence_after();
        }
        if (leader) {
          const uint64_t a = at(mask0, (st % kMaskSlots) * kMaskOpBytes), bb = at(a, kRow32);
          if (together) umma_f16(c.tmem + kColS, a, bb, kIdescS, 1u);
          umma_f16(c.tmem + kColS2, at(a, kRemOff32), bb, kIdescS2, 1u);
        }
      }
      if (!ok) break;
    }
    if (leader) {
      if (together) umma_commit(c.bar(kSMain));
      umma_commit(c.bar(kSRem));
    }
    // dV: queries 16e .. 16e + 15 at step e; those of warps 2 and 3 are the last step.
    auto dv_step = [&](int e) {
      umma_f16(c.tmem + kColDv, at(pT, e * 2048), at(gc, e * 2048), kIdescT, e > 0 ? 1u : 0u);
      umma_f16(c.tmem + kColRem, at(gc, e * 2048), at(p32, e * 512), kIdescRemT, e > 0 ? 1u : 0u);
    };
    if (!warp_wait(c.bar(kPMain), par, c.abort, p.status, 130)) break;
    tc_fence_after();
    if (leader) {
#pragma unroll
      for (int e = 0; e < 8; ++e) dv_step(e);
    }
    if (!warp_wait(c.bar(kPRem), par, c.abort, p.status, 117)) break;
    tc_fence_after();
    if (leader) {
      dv_step(8);
      umma_commit(c.bar(kDvFull));
    }
    // dQ of rows 0..127 needs only their dS; the transposed remainders and dK need all.
    if (!warp_wait(c.bar(kDsMain), par, c.abort, p.status, 131)) break;
    tc_fence_after();
    if (leader) {
#pragma unroll
      for (int e = 0; e < 9; ++e)  // keys 16e .. 16e + 15
        umma_f16(c.tmem + kColDq, e < 8 ? at(ds, (e >> 2) * kPChunk + (e & 3) * 32) : ds32, at(kc, e * 2048), kIdescO,
                 e > 0 ? 1u : 0u);
      umma_commit(c.bar(kDqFull));
    }
    if (!warp_wait(c.bar(kDsRem), par, c.abort, p.status, 116)) break;
    tc_fence_after();
    if (leader) {
#pragma unroll
      for (int e = 0; e < 9; ++e) {
        umma_f16(c.tmem + kColDq2, at(kc, e * 2048),
                 e < 8 ? at(ds, (e >> 2) * kPChunk + (e & 3) * 32 + 128 * 128) : at(ds32, 128 * 32), kIdescRemQ, e > 0 ? 1u : 0u);
        umma_f16(c.tmem + kColRem + kLaneHalf, at(qc, e * 2048), at(ds32, e * 512), kIdescRemT, e > 0 ? 1u : 0u);
      }
      umma_commit(c.bar(kRemFull));
#pragma unroll
      for (int e = 0; e < 9; ++e)
        umma_f16(c.tmem + kColDk, at(dsT, e * 2048), at(qc, e * 2048), kIdescT, e > 0 ? 1u : 0u);
      umma_commit(c.bar(kDkFull));
    }
  }
  if (leader) umma_commit(c.bar(kDone));
  int no_abort = 0;
  mbar_wait(c.bar(kDone), 0, &no_abort, p.status, 132, kTimeoutNs);
  __syncwarp();
}

template <int kMask>
__global__ void __launch_bounds__(kThreads, 1)
rel_bias_bwd_tc_kernel(const __grid_constant__ CUtensorMap tmq, const __grid_constant__ CUtensorMap tmk,
                       const __grid_constant__ CUtensorMap tmv, const __grid_constant__ CUtensorMap tmg,
                       const __grid_constant__ CUtensorMap tmdq, const __grid_constant__ CUtensorMap tmdk,
                       const __grid_constant__ CUtensorMap tmdv, const Params p) {
  extern __shared__ __align__(1024) uint8_t smem[];
  if (smem_u32(smem) & 1023u) {  // uniform; dynamic shared memory starts on such a boundary here
    if (threadIdx.x == 0) atomicCAS(p.status, 0, 140);
    return;
  }
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + kOffBars);
  int* words = reinterpret_cast<int*>(bars + kNumBars);  // abort flag, TMEM address, mask steps
  Ctx c;
  c.smem = smem;
  c.sbase = smem_u32(smem);
  c.bar0 = smem_u32(bars);
  c.abort = words;
  c.steps = words + 4;
  c.t_begin = tile_begin(p.num_tiles);
  c.n_local = tile_end(p.num_tiles) - c.t_begin;
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    *words = 0;
    for (int b = 0; b < kNumBars; ++b) {
      const bool main = b == kStaged || b == kStaged + 1 || b == kTFree || b == kDqFree || b == kPMain || b == kDsMain;
      mbar_init(c.bar(b), main ? 8 : b == kPRem || b == kDsRem ? 2 : 1);
    }
    fence_mbarrier_init();
  }
  if (warp == 1) {
    tmem_alloc(smem_u32(words + 1), kTmemCols);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  c.tmem = (uint32_t)*reinterpret_cast<volatile int*>(words + 1);

  if (warp >= 4) {
    warpgroup_reg_alloc<kRegsMain>();
    softmax_warps<false, kMask>(p, c, warp, lane);
  } else {
    warpgroup_reg_dealloc<kRegsSmall>();
    if (warp >= 2) softmax_warps<true, kMask>(p, c, warp, lane);
    else if (warp == 1) issuer<kMask>(p, c);
    else producer<kMask>(p, c, lane, &tmq, &tmk, &tmv, &tmg, &tmdq, &tmdk, &tmdv);
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(c.tmem, kTmemCols);
  }
}

}  // namespace bwd

template <int kMask>
int launch_fwd(const Params& p, int grid, cudaStream_t s) {
  CUtensorMap mq, mk, mv, mo;
  int rc;
  if ((rc = attn::make_map(&mq, p.q, false, p.Bwin, p.H, p.N, p.sq)) != FA_OK) return rc;
  if ((rc = attn::make_map(&mk, p.k, false, p.Bwin, p.H, p.N, p.sk)) != FA_OK) return rc;
  if ((rc = attn::make_map(&mv, p.v, false, p.Bwin, p.H, p.N, p.sv)) != FA_OK) return rc;
  if ((rc = attn::make_map(&mo, p.out, false, p.Bwin, p.H, p.N, p.so)) != FA_OK) return rc;
  auto kern = fwd::rel_bias_fwd_tc_kernel<kMask>;
  FA_CUDA(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, fwd::kSmem));
  kern<<<grid, kThreads, fwd::kSmem, s>>>(mq, mk, mv, mo, p);
  return check_launch("rel_bias_fwd_tc_kernel");
}

template <int kMask>
int launch_bwd(const Params& p, int grid, cudaStream_t s) {
  CUtensorMap mq, mk, mv, mg, mdq, mdk, mdv;
  int rc;
  if ((rc = attn::make_map(&mq, p.q, false, p.Bwin, p.H, p.N, p.sq)) != FA_OK) return rc;
  if ((rc = attn::make_map(&mk, p.k, false, p.Bwin, p.H, p.N, p.sk)) != FA_OK) return rc;
  if ((rc = attn::make_map(&mv, p.v, false, p.Bwin, p.H, p.N, p.sv)) != FA_OK) return rc;
  if ((rc = attn::make_map(&mg, p.dout, false, p.Bwin, p.H, p.N, p.so)) != FA_OK) return rc;
  if ((rc = attn::make_map(&mdq, p.dq, false, p.Bwin, p.H, p.N, p.sdq)) != FA_OK) return rc;
  if ((rc = attn::make_map(&mdk, p.dk, false, p.Bwin, p.H, p.N, p.sdk)) != FA_OK) return rc;
  if ((rc = attn::make_map(&mdv, p.dv, false, p.Bwin, p.H, p.N, p.sdv)) != FA_OK) return rc;
  auto kern = bwd::rel_bias_bwd_tc_kernel<kMask>;
  FA_CUDA(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, bwd::kSmem));
  kern<<<grid, kThreads, bwd::kSmem, s>>>(mq, mk, mv, mg, mdq, mdk, mdv, p);
  return check_launch("rel_bias_bwd_tc_kernel");
}

}  // namespace

int run_bf16_forward(const Params& p, int mask_kind, int grid, cudaStream_t s) {
  if (mask_kind == kMaskU8) return launch_fwd<kMaskU8>(p, grid, s);
  if (mask_kind == kGroups) return launch_fwd<kGroups>(p, grid, s);
  return launch_fwd<kNoMask>(p, grid, s);
}

int run_bf16_backward(const Params& p, int mask_kind, int grid, cudaStream_t s) {
  if (mask_kind == kMaskU8) return launch_bwd<kMaskU8>(p, grid, s);
  if (mask_kind == kGroups) return launch_bwd<kGroups>(p, grid, s);
  return launch_bwd<kNoMask>(p, grid, s);
}

}  // namespace relb
}  // namespace fa
