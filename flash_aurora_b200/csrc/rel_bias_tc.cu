// bf16 window attention with a learned relative position bias on the tensor cores (tcgen05 UMMAs,
// accumulators in TMEM), forward and backward. The formulas are in rel_bias.cu.
//
// Both kernels are persistent, one CTA per SM over a contiguous range of (head, window) tiles in
// head-major order, so that a head's bias is fetched from the table once per CTA and head and then
// stays on chip in fp32: 72 registers of each softmax warp thread. A window has 144 query rows and an
// M = 128 UMMA covers 128; rows 128..143 go through an M = 64 UMMA over rows 80..143 (the tile at an
// 80-row offset), whose last 16 rows are kept. Warps 4..11 own 16 query rows each of 0..127, warp 3 owns
// rows 128..143; a row's 144 keys sit in four threads of one warp (16x256b TMEM shape), so row
// maxima and sums take two shuffles. Registers are moved from warps 0..3 to 4..11 (setmaxnreg); warp
// 3, which is in the smaller group, keeps its 9 KB of bias in shared memory.
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
constexpr int kRow32 = kMaxN * 32;      // 16 keys x 144 rows of bf16, 32-byte swizzle
constexpr int kPBytes = 2 * kPChunk + kRow32;
constexpr int kIdBytes = 160;           // a tile's region ids and, at byte 144, whether they differ
constexpr int kRemBytes = 18 * 32 * 16; // one float4 per lane and 8-key block: warp 3's bias
constexpr uint32_t kRowOff80 = 80 * 128;
constexpr uint32_t kRowOff80_32 = 80 * 32;
constexpr uint32_t kLaneHalf = 16u << 16;  // second lane half of an M = 64 accumulator

constexpr uint32_t kIdescS = make_idesc(1, 128, kMaxN, false, false);
constexpr uint32_t kIdescS2 = make_idesc(1, 64, kMaxN, false, false);
constexpr uint32_t kIdescO = make_idesc(1, 128, 64, false, true);
constexpr uint32_t kIdescO2 = make_idesc(1, 64, 64, false, true);

__device__ __forceinline__ uint32_t sw32_offset(int r, int e) {
  return (uint32_t)(r * 32 + ((((e >> 3) ^ (r >> 2)) & 1) << 4) + (e & 7) * 2);
}

// Row pair (ra, rb) and key quad position of one thread of a softmax warp.
struct Lane {
  int t0, t1, ra, rb;
  uint32_t addr;  // TMEM lane offset of the warp's 16 rows
};

__device__ __forceinline__ Lane make_lane(int warp, int lane) {
  Lane l;
  l.t0 = lane & 3;
  l.t1 = lane >> 2;
  const int rbase = warp == 3 ? 128 : 32 * (warp & 3) + 16 * ((warp - 4) >> 2);
  l.ra = rbase + l.t1;
  l.rb = l.ra + 8;
  l.addr = warp == 3 ? (96u << 16) : ((uint32_t)rbase << 16);  // rows 48..63 of an M = 64 block
  return l;
}

// bf16 pairs of 8-key block j (0..17), rows ra and rb, into the P operand tile.
__device__ __forceinline__ void store_p(uint32_t sP, const Lane& l, int j, uint32_t a, uint32_t b) {
  if (j < 16) {
    const uint32_t off = sP + (j >> 3) * kPChunk + (uint32_t)(4 * l.t0);
    st_shared_u32(off + l.ra * 128 + (((j & 7) ^ (l.ra & 7)) << 4), a);
    st_shared_u32(off + l.rb * 128 + (((j & 7) ^ (l.rb & 7)) << 4), b);
  } else {
    st_shared_u32(sP + 2 * kPChunk + sw32_offset(l.ra, (j & 1) * 8 + 2 * l.t0), a);
    st_shared_u32(sP + 2 * kPChunk + sw32_offset(l.rb, (j & 1) * 8 + 2 * l.t0), b);
  }
}

// The bias of this thread's 72 (row, key) pairs, one float4 per 8-key block (see bias_rows). Warp 3
// keeps them in shared memory.
template <bool kRem>
struct Bias {
  float4 b[kRem ? 1 : 18];
  uint32_t smem;
  __device__ __forceinline__ void fetch(const Params& p, int h, const Lane& l, int lane) {
    const float4* src = bias_rows(p, h, l.ra - l.t1, lane);
#pragma unroll
    for (int j = 0; j < 18; ++j) {
      const float4 v = __ldg(src + j * 32);
      if constexpr (kRem)
        st_shared_v4(smem + j * 512, __float_as_uint(v.x), __float_as_uint(v.y), __float_as_uint(v.z),
                     __float_as_uint(v.w));
      else
        b[j] = v;
    }
  }
  __device__ __forceinline__ float4 get(int j) const {
    if constexpr (kRem) {
      uint32_t x, y, z, w;
      ld_shared_v4(smem + j * 512, x, y, z, w);
      return make_float4(__uint_as_float(x), __uint_as_float(y), __uint_as_float(z), __uint_as_float(w));
    } else {
      return b[j];
    }
  }
};

// Mask of one tile as the softmax warps apply it.
template <int kMask>
struct TileMask {
  bool on;
  uint32_t ta, tb;      // region ids of rows ra, rb
  const uint8_t* ids;   // shared memory
  const uint8_t *ma, *mb;  // byte-mask rows (global), null past N
  __device__ __forceinline__ void begin(const Params& p, const Lane& l, int w, const uint8_t* tile_ids) {
    if constexpr (kMask == kGroups) {
      on = tile_ids[kMaxN] != 0;
      ids = tile_ids;
      ta = tile_ids[l.ra];
      tb = tile_ids[l.rb];
    } else if constexpr (kMask == kMaskU8) {
      on = true;
      const uint8_t* base = p.mask + (int64_t)(w % p.nW) * p.N * p.N;
      ma = l.ra < p.N ? base + l.ra * p.N : nullptr;
      mb = l.rb < p.N ? base + l.rb * p.N : nullptr;
    } else {
      on = false;
    }
  }
  // Adds -100 (log2 domain) to the masked logits of 8-key block j.
  __device__ __forceinline__ void apply(const Params& p, const Lane& l, int j, float2& xa, float2& xb) const {
    const int key = 8 * j + 2 * l.t0;
    if constexpr (kMask == kGroups) {
      const uint32_t kk = *reinterpret_cast<const unsigned short*>(ids + key);
      const uint32_t k0 = kk & 0xffu, k1 = kk >> 8;
      xa.x += k0 != ta ? kMaskedLog2 : 0.f;
      xa.y += k1 != ta ? kMaskedLog2 : 0.f;
      xb.x += k0 != tb ? kMaskedLog2 : 0.f;
      xb.y += k1 != tb ? kMaskedLog2 : 0.f;
    } else if constexpr (kMask == kMaskU8) {
      if (key < p.N) {
        if (ma && __ldg(ma + key)) xa.x += kMaskedLog2;
        if (mb && __ldg(mb + key)) xb.x += kMaskedLog2;
      }
      if (key + 1 < p.N) {
        if (ma && __ldg(ma + key + 1)) xa.y += kMaskedLog2;
        if (mb && __ldg(mb + key + 1)) xb.y += kMaskedLog2;
      }
    }
  }
};

// Region ids of a window's tokens lane + 32 m, and the store of a tile's ids with their "differ" flag.
__device__ __forceinline__ void load_ids(const Params& p, int w, int lane, uint32_t (&id)[5]) {
  const uint8_t* g = p.mask + (int64_t)(w % p.nW) * p.N;
  const uint32_t first = __ldg(g);
#pragma unroll
  for (int m = 0; m < 5; ++m) id[m] = lane + 32 * m < p.N ? (uint32_t)__ldg(g + lane + 32 * m) : first;
}
__device__ __forceinline__ void store_ids(uint8_t* dst, int lane, const uint32_t (&id)[5]) {
  const uint32_t first = __shfl_sync(0xffffffffu, id[0], 0);
  bool differ = false;
#pragma unroll
  for (int m = 0; m < 5; ++m) {
    differ = differ || id[m] != first;
    if (lane + 32 * m < kMaxN) dst[lane + 32 * m] = (uint8_t)id[m];
  }
  differ = __any_sync(0xffffffffu, differ);
  if (lane == 0) dst[kMaxN] = differ ? 1 : 0;
  __syncwarp();
}

// A whole warp's bounded wait: every lane gets the same answer, so that the warp stays together.
__device__ __forceinline__ bool warp_wait(uint32_t bar, uint32_t parity, volatile int* abort, int* status, int code) {
  return __all_sync(0xffffffffu, mbar_wait(bar, parity, abort, status, code, kTimeoutNs));
}

__device__ __forceinline__ float2 f2(uint32_t a, uint32_t b) {
  return make_float2(__uint_as_float(a), __uint_as_float(b));
}

// Rows ra, rb of a 64-wide accumulator block (32 registers, 16x256b), scaled, to a staged bf16 tile.
__device__ __forceinline__ void stage_rows(uint32_t stg, const Lane& l, const uint32_t (&o)[32], float sa, float sb) {
  const float2 a2 = make_float2(sa, sa), b2 = make_float2(sb, sb);
#pragma unroll
  for (int jd = 0; jd < 8; ++jd) {
    const float2 ya = __fmul2_rn(f2(o[4 * jd], o[4 * jd + 1]), a2);
    const float2 yb = __fmul2_rn(f2(o[4 * jd + 2], o[4 * jd + 3]), b2);
    st_shared_u32(stg + (uint32_t)l.ra * 128u + (uint32_t)(((jd ^ (l.ra & 7)) & 7) << 4) + 4u * l.t0,
                  pack_bf16x2(ya.x, ya.y));
    st_shared_u32(stg + (uint32_t)l.rb * 128u + (uint32_t)(((jd ^ (l.rb & 7)) & 7) << 4) + 4u * l.t0,
                  pack_bf16x2(yb.x, yb.y));
  }
}

// ------------------------------------------------------------------------------------------
// Forward.
//   warps 0, 2  TMA producers: Q, K and the region ids (warp 0), V (warp 2), 3-slot rings; the output
//               of a tile is staged in its V slot and stored by warp 2 before the slot's reuse;
//   warp 1      TMEM owner and UMMA issuer:  S = Q K^T (M=128 and M=64), O = P V (M=128 and M=64);
//   warps 3-11  x = S scale + bias (+ mask), softmax in the log2 domain, P to shared memory in bf16,
//               then the previous tile's output rows.
// ------------------------------------------------------------------------------------------
namespace fwd {

constexpr int kStages = 3;
constexpr int kQKBytes = 2 * kTileBytes;
constexpr int kStageBytes = 3 * kTileBytes;
constexpr int kOffP = kStages * kStageBytes;
constexpr int kOffRem = kOffP + kPBytes;
constexpr int kOffIds = kOffRem + kRemBytes;
// Region ids have a ring of their own: slot i % kIdSlots is rewritten for tile i + kIdSlots once the S
// product of tile i + kIdSlots - 3 is done, which follows every softmax warp's load of S of tile
// i + kIdSlots - 4 >= i + 1, so its work on tile i.
constexpr int kIdSlots = 5;
constexpr int kOffBars = kOffIds + kIdSlots * kIdBytes;
enum { kFullQK = 0, kEmptyQK = 3, kFullV = 6, kStaged = 9, kSFull = 12, kSFree, kPFull, kPEmpty, kOFull = 16,
       kOFree = 18, kDone = 20, kIds = 21, kNumBars = kIds + kIdSlots };
constexpr int kSmem = kOffBars + kNumBars * 8 + 16 + 1024;
static_assert(kSmem <= 227 * 1024, "shared memory budget");
constexpr uint32_t kColS = 0, kColS2 = 160, kColO0 = 320, kColO1 = 384, kColO2 = 448;
constexpr uint32_t kRegsSmall = 120, kRegsMain = 192;
static_assert(4 * kRegsSmall + 8 * kRegsMain <= 12 * kRegsLaunch, "register split");

struct Ctx {
  uint32_t sbase, bar0, tmem;
  uint8_t* smem;
  volatile int* abort;
  int t_begin, n_local;
  __device__ __forceinline__ uint32_t bar(int i) const { return bar0 + 8u * (uint32_t)i; }
};

template <bool kRem, int kMask>
__device__ __forceinline__ void softmax_warps(const Params& p, const Ctx& c, int warp, int lane) {
  const Lane l = make_lane(warp, lane);
  const uint32_t s_col = kRem ? kColS2 : kColS;
  const uint32_t sP = c.sbase + kOffP;
  Bias<kRem> bias;
  bias.smem = c.sbase + kOffRem + lane * 16;
  int cur_h = -1, prev = -1;
  float la_prev = 1.f, lb_prev = 1.f;

  auto epilogue = [&](int j, float la, float lb) -> bool {
    const int ob = j & 1;
    if (!warp_wait(c.bar(kOFull + ob), (uint32_t)((j >> 1) & 1), c.abort, p.status, 101)) return false;
    tc_fence_after();
    uint32_t o[32];
    const uint32_t col = kRem ? kColO2 + (ob ? kLaneHalf : 0u) : (ob ? kColO1 : kColO0);
    tmem_ld_16x256b_r32(c.tmem + l.addr + col, o);
    tmem_wait_ld();
    tc_fence_before();
    __syncwarp();
    if (lane == 0) mbar_arrive(c.bar(kOFree + ob));
    stage_rows(c.sbase + (j % kStages) * kStageBytes + kQKBytes, l, o, 1.f / la, 1.f / lb);
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
    TileMask<kMask> mask;
    if constexpr (kMask == kGroups) {
      if (!warp_wait(c.bar(kIds + i % kIdSlots), (uint32_t)((i / kIdSlots) & 1), c.abort, p.status, 102)) {
        ok = false;
        break;
      }
    }
    mask.begin(p, l, w, c.smem + kOffIds + (i % kIdSlots) * kIdBytes);
    if (!warp_wait(c.bar(kSFull), (uint32_t)(i & 1), c.abort, p.status, 103)) { ok = false; break; }
    tc_fence_after();
    uint32_t v[72];
    {
      uint32_t a[64], b[8];
      tmem_ld_16x256b_r64(c.tmem + l.addr + s_col, a);
      tmem_ld_16x256b_r8(c.tmem + l.addr + s_col + 128, b);
      tmem_wait_ld();
#pragma unroll
      for (int k = 0; k < 64; ++k) v[k] = a[k];
#pragma unroll
      for (int k = 0; k < 8; ++k) v[64 + k] = b[k];
    }
    tc_fence_before();
    __syncwarp();
    if (lane == 0) mbar_arrive(c.bar(kSFree));
    // The mask has a loop of its own behind one branch: inside this loop its 18 branches keep the
    // compiler from interleaving the blocks, which doubled the kernel's time even where none is taken.
#pragma unroll
    for (int j = 0; j < 18; ++j) {
      const float4 b = bias.get(j);
      const float2 xa = __ffma2_rn(f2(v[4 * j], v[4 * j + 1]), c2, make_float2(b.x, b.y));
      const float2 xb = __ffma2_rn(f2(v[4 * j + 2], v[4 * j + 3]), c2, make_float2(b.z, b.w));
      v[4 * j] = __float_as_uint(xa.x);
      v[4 * j + 1] = __float_as_uint(xa.y);
      v[4 * j + 2] = __float_as_uint(xb.x);
      v[4 * j + 3] = __float_as_uint(xb.y);
    }
    if (kMask != kNoMask && mask.on) {
#pragma unroll
      for (int j = 0; j < 18; ++j) {
        float2 xa = f2(v[4 * j], v[4 * j + 1]), xb = f2(v[4 * j + 2], v[4 * j + 3]);
        mask.apply(p, l, j, xa, xb);
        v[4 * j] = __float_as_uint(xa.x);
        v[4 * j + 1] = __float_as_uint(xa.y);
        v[4 * j + 2] = __float_as_uint(xb.x);
        v[4 * j + 3] = __float_as_uint(xb.y);
      }
    }
    float mxa = -INFINITY, mxb = -INFINITY;
#pragma unroll
    for (int j = 0; j < 18; ++j) {
      mxa = fmax3(mxa, __uint_as_float(v[4 * j]), __uint_as_float(v[4 * j + 1]));
      mxb = fmax3(mxb, __uint_as_float(v[4 * j + 2]), __uint_as_float(v[4 * j + 3]));
    }
    mxa = fmaxf(mxa, __shfl_xor_sync(0xffffffffu, mxa, 1));
    mxa = fmaxf(mxa, __shfl_xor_sync(0xffffffffu, mxa, 2));
    mxb = fmaxf(mxb, __shfl_xor_sync(0xffffffffu, mxb, 1));
    mxb = fmaxf(mxb, __shfl_xor_sync(0xffffffffu, mxb, 2));
    const float2 ma2 = make_float2(-mxa, -mxa), mb2 = make_float2(-mxb, -mxb);
    float2 la2 = make_float2(0.f, 0.f), lb2 = make_float2(0.f, 0.f);
    uint32_t pa[18], pb[18];
#pragma unroll
    for (int j = 0; j < 18; ++j) {
      const float2 ya = __fadd2_rn(f2(v[4 * j], v[4 * j + 1]), ma2);
      const float2 yb = __fadd2_rn(f2(v[4 * j + 2], v[4 * j + 3]), mb2);
      const float2 ea = make_float2(ex2(ya.x), ex2(ya.y)), eb = make_float2(ex2(yb.x), ex2(yb.y));
      la2 = __fadd2_rn(la2, ea);
      lb2 = __fadd2_rn(lb2, eb);
      pa[j] = pack_bf16x2(ea.x, ea.y);
      pb[j] = pack_bf16x2(eb.x, eb.y);
    }
    float la = la2.x + la2.y, lb = lb2.x + lb2.y;
    la += __shfl_xor_sync(0xffffffffu, la, 1);
    la += __shfl_xor_sync(0xffffffffu, la, 2);
    lb += __shfl_xor_sync(0xffffffffu, lb, 1);
    lb += __shfl_xor_sync(0xffffffffu, lb, 2);
    if (!warp_wait(c.bar(kPEmpty), (uint32_t)((i & 1) ^ 1), c.abort, p.status, 104)) { ok = false; break; }
#pragma unroll
    for (int j = 0; j < 18; ++j) store_p(sP, l, j, pa[j], pb[j]);
    fence_proxy_async_shared();
    __syncwarp();
    if (lane == 0) mbar_arrive(c.bar(kPFull));
    if (p.stats && l.t0 == 0) {
      float2* st = p.stats + ((int64_t)w * p.H + h) * p.N;
      if (l.ra < p.N) st[l.ra] = make_float2(mxa, log2f(la));
      if (l.rb < p.N) st[l.rb] = make_float2(mxb, log2f(lb));
    }
    if (prev >= 0 && !epilogue(prev, la_prev, lb_prev)) { ok = false; break; }
    prev = i;
    la_prev = la;
    lb_prev = lb;
  }
  if (ok && prev >= 0) epilogue(prev, la_prev, lb_prev);
}

template <int kMask>
__global__ void __launch_bounds__(kThreads, 1)
rel_bias_fwd_tc_kernel(const __grid_constant__ CUtensorMap tmq, const __grid_constant__ CUtensorMap tmk,
                       const __grid_constant__ CUtensorMap tmv, const __grid_constant__ CUtensorMap tmo,
                       const Params p) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + kOffBars);
  uint32_t* tmem_holder = reinterpret_cast<uint32_t*>(bars + kNumBars);
  __shared__ int abort_flag;
  Ctx c;
  c.smem = smem;
  c.sbase = smem_u32(smem);
  c.bar0 = smem_u32(bars);
  c.abort = &abort_flag;
  c.t_begin = tile_begin(p.num_tiles);
  c.n_local = tile_end(p.num_tiles) - c.t_begin;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    abort_flag = 0;
    for (int s = 0; s < kStages; ++s) {
      mbar_init(c.bar(kFullQK + s), 1);
      mbar_init(c.bar(kEmptyQK + s), 1);
      mbar_init(c.bar(kFullV + s), 1);
      mbar_init(c.bar(kStaged + s), 9);
    }
    mbar_init(c.bar(kSFull), 1);
    mbar_init(c.bar(kSFree), 9);
    mbar_init(c.bar(kPFull), 9);
    mbar_init(c.bar(kPEmpty), 1);
    for (int b = 0; b < 2; ++b) {
      mbar_init(c.bar(kOFull + b), 1);
      mbar_init(c.bar(kOFree + b), 9);
    }
    mbar_init(c.bar(kDone), 1);
    for (int b = 0; b < kIdSlots; ++b) mbar_init(c.bar(kIds + b), 1);
    fence_mbarrier_init();
  }
  if (warp == 1) {
    tmem_alloc(smem_u32(tmem_holder), kTmemCols);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  c.tmem = *tmem_holder;
  const int n = c.n_local;

  if (warp >= 4) {
    warpgroup_reg_alloc<kRegsMain>();
    softmax_warps<false, kMask>(p, c, warp, lane);
  } else {
    warpgroup_reg_dealloc<kRegsSmall>();
    if (warp == 3) {
      softmax_warps<true, kMask>(p, c, warp, lane);
    } else if (warp == 0) {
      if (lane == 0) {
        tma_prefetch_desc(&tmq);
        tma_prefetch_desc(&tmk);
      }
      int last_par[kStages] = {-1, -1, -1};
      uint32_t id[5], next_id[5];
      if constexpr (kMask == kGroups) {
        if (n > 0) load_ids(p, c.t_begin % p.Bwin, lane, next_id);
      }
      for (int i = 0; i < n; ++i) {
        const int t = c.t_begin + i, h = t / p.Bwin, w = t - h * p.Bwin, s = i % kStages;
        const uint32_t ph = (uint32_t)((i / kStages) & 1);
        if constexpr (kMask == kGroups) {
#pragma unroll
          for (int m = 0; m < 5; ++m) id[m] = next_id[m];
          if (i + 1 < n) load_ids(p, (t + 1) % p.Bwin, lane, next_id);  // one tile ahead
        }
        int ok = 1;
        if (lane == 0) ok = mbar_wait(c.bar(kEmptyQK + s), ph ^ 1u, c.abort, p.status, 105, kTimeoutNs);
        if (!__shfl_sync(0xffffffffu, ok, 0)) break;
        if (lane == 0) {
          const uint32_t dst = c.sbase + s * kStageBytes;
          mbar_arrive_expect_tx(c.bar(kFullQK + s), kQKBytes);
          tma_load_4d(dst, &tmq, c.bar(kFullQK + s), 0, 0, h, w);
          tma_load_4d(dst + kTileBytes, &tmk, c.bar(kFullQK + s), 0, 0, h, w);
          last_par[s] = (int)ph;
        }
        if constexpr (kMask == kGroups) {
          store_ids(smem + kOffIds + (i % kIdSlots) * kIdBytes, lane, id);
          if (lane == 0) mbar_arrive(c.bar(kIds + i % kIdSlots));
        }
      }
      if (lane == 0) {
        // Never leave with copies in flight (bounded, also after an abort).
        int no_abort = 0;
        for (int s = 0; s < kStages; ++s)
          if (last_par[s] >= 0) mbar_wait(c.bar(kFullQK + s), (uint32_t)last_par[s], &no_abort, p.status, 106, kTimeoutNs);
      }
    } else if (warp == 2) {
      if (lane == 0) tma_prefetch_desc(&tmv);
      int last_par[kStages] = {-1, -1, -1};
      auto store_out = [&](int j) {
        const int t = c.t_begin + j, h = t / p.Bwin;
        tma_store_4d(&tmo, c.sbase + (j % kStages) * kStageBytes + kQKBytes, 0, 0, h, t - h * p.Bwin);
        bulk_commit_group();
      };
      for (int i = 0; i < n; ++i) {
        const int t = c.t_begin + i, h = t / p.Bwin, w = t - h * p.Bwin, s = i % kStages;
        int ok = 1;
        if (lane == 0 && i >= kStages) {
          // The slot still holds the output of tile i - 3: store it and wait until it has been read.
          ok = mbar_wait(c.bar(kStaged + s), (uint32_t)(((i - kStages) / kStages) & 1), c.abort, p.status, 107, kTimeoutNs);
          if (ok) {
            store_out(i - kStages);
            bulk_wait_group_read0();
          }
        }
        if (!__shfl_sync(0xffffffffu, ok, 0)) break;
        if (lane == 0) {
          mbar_arrive_expect_tx(c.bar(kFullV + s), kTileBytes);
          tma_load_4d(c.sbase + s * kStageBytes + kQKBytes, &tmv, c.bar(kFullV + s), 0, 0, h, w);
          last_par[s] = (i / kStages) & 1;
        }
      }
      if (lane == 0) {
        int no_abort = 0;
        for (int s = 0; s < kStages; ++s)
          if (last_par[s] >= 0) mbar_wait(c.bar(kFullV + s), (uint32_t)last_par[s], &no_abort, p.status, 108, kTimeoutNs);
        for (int j = n > kStages ? n - kStages : 0; j < n; ++j) {
          if (!mbar_wait(c.bar(kStaged + j % kStages), (uint32_t)((j / kStages) & 1), c.abort, p.status, 109, kTimeoutNs))
            break;
          store_out(j);
        }
        bulk_wait_group0();
      }
    } else if (lane == 0) {
      // UMMA issuer: S and PV in whatever order their inputs become ready (non-blocking tests).
      int ns = 0, npv = 0;
      uint64_t t_last = cycles();
      uint32_t idle = 0;
      const uint32_t sP = c.sbase + kOffP;
      while (npv < n) {
        bool progressed = false;
        if (ns < n) {
          const int s = ns % kStages;
          if (mbar_test_wait(c.bar(kFullQK + s), (uint32_t)((ns / kStages) & 1)) &&
              mbar_test_wait(c.bar(kSFree), (uint32_t)((ns & 1) ^ 1))) {
            tc_fence_after();
            const uint32_t sQ = c.sbase + s * kStageBytes, sK = sQ + kTileBytes;
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              const uint64_t b = desc_sw128(sK + k * 32, 16, 1024);
              umma_f16(c.tmem + kColS, desc_sw128(sQ + k * 32, 16, 1024), b, kIdescS, k > 0 ? 1u : 0u);
              umma_f16(c.tmem + kColS2, desc_sw128(sQ + kRowOff80 + k * 32, 16, 1024), b, kIdescS2, k > 0 ? 1u : 0u);
            }
            umma_commit(c.bar(kSFull));
            umma_commit(c.bar(kEmptyQK + s));
            ++ns;
            progressed = true;
          }
        }
        if (npv < ns) {
          const int j = npv, s = j % kStages, ob = j & 1;
          if (mbar_test_wait(c.bar(kPFull), (uint32_t)(j & 1)) &&
              mbar_test_wait(c.bar(kFullV + s), (uint32_t)((j / kStages) & 1)) &&
              mbar_test_wait(c.bar(kOFree + ob), (uint32_t)(((j >> 1) & 1) ^ 1))) {
            tc_fence_after();
            const uint32_t sV = c.sbase + s * kStageBytes + kQKBytes;
            const uint32_t dO = c.tmem + (ob ? kColO1 : kColO0);
            const uint32_t dO2 = c.tmem + kColO2 + (ob ? kLaneHalf : 0u);
#pragma unroll
            for (int k = 0; k < 8; ++k) {
              const uint32_t pa = sP + (k >> 2) * kPChunk + (k & 3) * 32;
              const uint64_t b = desc_sw128(sV + k * 2048, kTileBytes, 1024);
              umma_f16(dO, desc_sw128(pa, 16, 1024), b, kIdescO, k > 0 ? 1u : 0u);
              umma_f16(dO2, desc_sw128(pa + kRowOff80, 16, 1024), b, kIdescO2, k > 0 ? 1u : 0u);
            }
            const uint32_t pa = sP + 2 * kPChunk;  // keys 128..143
            const uint64_t b = desc_sw128(sV + 8 * 2048, kTileBytes, 1024);
            umma_f16(dO, desc_sw32(pa, 256), b, kIdescO, 1u);
            umma_f16(dO2, desc_sw32(pa + kRowOff80_32, 256), b, kIdescO2, 1u);
            umma_commit(c.bar(kOFull + ob));
            umma_commit(c.bar(kPEmpty));
            ++npv;
            progressed = true;
          }
        }
        if (progressed) {
          idle = 0;
          t_last = cycles();
        } else if ((++idle & 63u) == 0) {
          if (*c.abort) break;
          if (cycles() - t_last > ns_to_cycles(kTimeoutNs)) {
            atomicCAS(p.status, 0, 110);
            *c.abort = 1;
            break;
          }
        }
      }
      umma_commit(c.bar(kDone));
      int no_abort = 0;
      mbar_wait(c.bar(kDone), 0, &no_abort, p.status, 111, kTimeoutNs);
    }
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
//   S = Q K^T, dP = dO V^T                     M=128 (rows 0..127) and M=64 (rows 80..143), N=144
//   pass 1   P = exp2(x - max - log2 sum) from the forward's row statistics; delta = sum_k P dP; P
//            replaces S in TMEM (fp32) and goes to shared memory in bf16
//   dV = P^T dO                                runs while pass 2 computes
//   pass 2   dS = P (dP - delta), added to the head's bias gradient (fp32, 72 registers of each
//            thread), to shared memory in bf16 over P once dV is done
//   dK = dS^T Q, dQ = dS K
// dV, dK, dQ of keys / rows 0..127 are M=128 UMMAs (P and dS are read MN-major for dV and dK); those
// of 128..143 are computed transposed, (64 head dims) x (16 rows), as M=64, N=16 UMMAs, which costs
// a quarter of an M=64, N=64 block.
// TMEM columns: S / P 0..143, dP 144..287 (then dK 144..207 and dQ 208..271), the M=64 blocks of S
// and dP in the two lane halves of 288..431 (then dQ's transposed remainder 416..431), dV 432..495,
// the transposed remainders of dV and dK in the lane halves of 496..511.
// Outputs are staged in the tile's own slots (dV over V, dK over K, dQ over Q) and stored by warp 0
// before it loads the tile after next into them. Two input slots (147 KB) and one P / dS tile leave
// no room for a second tile in flight: the chain of a tile is serial, its loads are not.
// ------------------------------------------------------------------------------------------
namespace bwd {

constexpr int kStages = 2;
constexpr int kOffQ = 0, kOffK = kTileBytes, kOffV = 2 * kTileBytes, kOffG = 3 * kTileBytes;
constexpr int kStageBytes = 4 * kTileBytes;
constexpr int kOffP = kStages * kStageBytes;
constexpr int kOffRem = kOffP + kPBytes;          // warp 3's bias
constexpr int kOffRemAcc = kOffRem + kRemBytes;   // warp 3's bias gradient
constexpr int kOffIds = kOffRemAcc + kRemBytes;
constexpr int kOffBars = kOffIds + kStages * kIdBytes;
enum { kFull = 0, kStaged = 2, kSFull = 4, kPFull, kDvFull, kDsFull, kDkFull, kTFree, kDone, kNumBars };
constexpr int kSmem = kOffBars + kNumBars * 8 + 16 + 1024;
static_assert(kSmem <= 227 * 1024, "shared memory budget");
constexpr uint32_t kColS = 0, kColP = 144, kColS2 = 288, kColDv = 432, kColRem = 496;
constexpr uint32_t kColDk = kColP, kColDq = kColP + 64, kColDq2 = kColS2 + 128;
constexpr uint32_t kRegsSmall = 104, kRegsMain = 200;
static_assert(4 * kRegsSmall + 8 * kRegsMain <= 12 * kRegsLaunch, "register split");
constexpr uint32_t kIdescT = make_idesc(1, 128, 64, true, true);    // A and B MN-major: dV, dK
constexpr uint32_t kIdescRemT = make_idesc(1, 64, 16, true, true);  // (64 dims) x (16 keys)
constexpr uint32_t kIdescRemQ = make_idesc(1, 64, 16, true, false); // (64 dims) x (16 queries)

struct Ctx {
  uint32_t sbase, bar0, tmem;
  uint8_t* smem;
  volatile int* abort;
  int t_begin, n_local;
  __device__ __forceinline__ uint32_t bar(int i) const { return bar0 + 8u * (uint32_t)i; }
};

// The head's bias gradient of this thread's 72 pairs.
template <bool kRem>
struct Grad {
  float2 a[kRem ? 1 : 36];
  uint32_t smem;
  __device__ __forceinline__ void clear() {
    if constexpr (kRem) {
      for (int j = 0; j < 18; ++j) st_shared_v4(smem + j * 512, 0u, 0u, 0u, 0u);
    } else {
#pragma unroll
      for (int j = 0; j < 36; ++j) a[j] = make_float2(0.f, 0.f);
    }
  }
  __device__ __forceinline__ void add(int j, float2 ga, float2 gb) {
    if constexpr (kRem) {
      uint32_t x, y, z, w;
      ld_shared_v4(smem + j * 512, x, y, z, w);
      const float2 sa = __fadd2_rn(f2(x, y), ga), sb = __fadd2_rn(f2(z, w), gb);
      st_shared_v4(smem + j * 512, __float_as_uint(sa.x), __float_as_uint(sa.y), __float_as_uint(sb.x),
                   __float_as_uint(sb.y));
    } else {
      a[2 * j] = __fadd2_rn(a[2 * j], ga);
      a[2 * j + 1] = __fadd2_rn(a[2 * j + 1], gb);
    }
  }
  __device__ __forceinline__ void flush(const Params& p, int h, const Lane& l) const {
    if (!p.slots) return;
    float* slot = p.slots + (int64_t)(blockIdx.x + h) * p.N * p.N;
#pragma unroll
    for (int j = 0; j < 18; ++j) {
      float4 v;
      if constexpr (kRem) {
        uint32_t x, y, z, w;
        ld_shared_v4(smem + j * 512, x, y, z, w);
        v = make_float4(__uint_as_float(x), __uint_as_float(y), __uint_as_float(z), __uint_as_float(w));
      } else {
        v = make_float4(a[2 * j].x, a[2 * j].y, a[2 * j + 1].x, a[2 * j + 1].y);
      }
      const int key = 8 * j + 2 * l.t0;
      if (l.ra < p.N) {
        if (key < p.N) slot[l.ra * p.N + key] = v.x;
        if (key + 1 < p.N) slot[l.ra * p.N + key + 1] = v.y;
      }
      if (l.rb < p.N) {
        if (key < p.N) slot[l.rb * p.N + key] = v.z;
        if (key + 1 < p.N) slot[l.rb * p.N + key + 1] = v.w;
      }
    }
  }
};

// A transposed remainder block, (64 head dims) x (rows 128..143), of this warp's TMEM quarter: 16
// head dims, scaled, into rows 128..143 of a staged bf16 tile.
__device__ __forceinline__ void stage_rem(uint32_t taddr, uint32_t stg, int quarter, const Lane& l, float scale) {
  uint32_t r[8];
  tmem_ld_16x256b_r8(taddr + ((uint32_t)(32 * quarter) << 16), r);
  tmem_wait_ld();
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const int row = 128 + 8 * (e >> 2) + 2 * l.t0 + (e & 1);
    const int d = 16 * quarter + l.t1 + 8 * ((e >> 1) & 1);
    const __nv_bfloat16 v = __float2bfloat16_rn(__uint_as_float(r[e]) * scale);
    asm volatile("st.shared.u16 [%0], %1;" ::"r"(stg + (uint32_t)(row * 128 + (((d >> 3) ^ (row & 7)) << 4) + (d & 7) * 2)),
                 "h"(__bfloat16_as_ushort(v))
                 : "memory");
  }
}

template <bool kRem, int kMask>
__device__ __forceinline__ void pass1(const Params& p, const Lane& l, const TileMask<kMask>& mask, const Bias<kRem>& bias,
                                      uint32_t tS, uint32_t tP, uint32_t sP, float2 sta, float2 stb, float2& da2,
                                      float2& db2) {
  // Pass 1, 16 keys (two 8-key blocks) at a time, the next loads in flight.
  const float2 c2 = make_float2(p.scale_log2, p.scale_log2);
  const float2 ma2 = make_float2(-sta.x, -sta.x), mb2 = make_float2(-stb.x, -stb.x);
  const float2 na2 = make_float2(-sta.y, -sta.y), nb2 = make_float2(-stb.y, -stb.y);
  uint32_t sv[8], gv[8];
  tmem_ld_16x256b_r8(tS, sv);
  tmem_ld_16x256b_r8(tP, gv);
#pragma unroll
  for (int q = 0; q < 9; ++q) {
    tmem_wait_ld();
    uint32_t cs[8], cg[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      cs[e] = sv[e];
      cg[e] = gv[e];
    }
    if (q < 8) {
      tmem_ld_16x256b_r8(tS + 16 * (q + 1), sv);
      tmem_ld_16x256b_r8(tP + 16 * (q + 1), gv);
    }
#pragma unroll
    for (int e = 0; e < 8; e += 4) {
      const int j = 2 * q + (e >> 2);
      const float4 b = bias.get(j);
      float2 xa = __ffma2_rn(f2(cs[e], cs[e + 1]), c2, make_float2(b.x, b.y));
      float2 xb = __ffma2_rn(f2(cs[e + 2], cs[e + 3]), c2, make_float2(b.z, b.w));
      if (kMask != kNoMask) mask.apply(p, l, j, xa, xb);
      xa = __fadd2_rn(__fadd2_rn(xa, ma2), na2);
      xb = __fadd2_rn(__fadd2_rn(xb, mb2), nb2);
      const float2 ea = make_float2(ex2(xa.x), ex2(xa.y)), eb = make_float2(ex2(xb.x), ex2(xb.y));
      da2 = __ffma2_rn(ea, f2(cg[e], cg[e + 1]), da2);
      db2 = __ffma2_rn(eb, f2(cg[e + 2], cg[e + 3]), db2);
      store_p(sP, l, j, pack_bf16x2(ea.x, ea.y), pack_bf16x2(eb.x, eb.y));
      cs[e] = __float_as_uint(ea.x);
      cs[e + 1] = __float_as_uint(ea.y);
      cs[e + 2] = __float_as_uint(eb.x);
      cs[e + 3] = __float_as_uint(eb.y);
    }
    tmem_st_16x256b_r8(tS + 16 * q, cs);
  }
}

template <bool kRem, int kMask>
__device__ __forceinline__ void softmax_warps(const Params& p, const Ctx& c, int warp, int lane) {
  const Lane l = make_lane(warp, lane);
  const uint32_t tS = c.tmem + l.addr + (kRem ? kColS2 : kColS);
  const uint32_t tP = c.tmem + l.addr + (kRem ? kColS2 + kLaneHalf : kColP);
  const uint32_t sP = c.sbase + kOffP;
  Bias<kRem> bias;
  bias.smem = c.sbase + kOffRem + lane * 16;
  Grad<kRem> grad;
  grad.smem = c.sbase + kOffRemAcc + lane * 16;
  int cur_h = -1;
  for (int i = 0; i < c.n_local; ++i) {
    const int t = c.t_begin + i, h = t / p.Bwin, w = t - h * p.Bwin, s = i & 1;
    const uint32_t par = (uint32_t)(i & 1);
    const uint32_t slot = c.sbase + s * kStageBytes;
    if (h != cur_h) {
      if (cur_h >= 0) grad.flush(p, cur_h, l);
      cur_h = h;
      grad.clear();
      bias.fetch(p, h, l, lane);
    }
    // Row statistics; +inf past N makes the rows' P zero.
    const float2* st = p.stats + ((int64_t)w * p.H + h) * p.N;
    const float2 pad = make_float2(INFINITY, 0.f);
    const float2 sta = l.ra < p.N ? __ldg(st + l.ra) : pad, stb = l.rb < p.N ? __ldg(st + l.rb) : pad;
    TileMask<kMask> mask;
    if (!warp_wait(c.bar(kSFull), par, c.abort, p.status, 121)) return;
    if constexpr (kMask == kGroups) {  // the ids came with the tile's loads, long complete
      if (!warp_wait(c.bar(kFull + s), (uint32_t)((i >> 1) & 1), c.abort, p.status, 122)) return;
    }
    mask.begin(p, l, w, c.smem + kOffIds + s * kIdBytes);
    tc_fence_after();
    float2 da2 = make_float2(0.f, 0.f), db2 = make_float2(0.f, 0.f);
    // One branch for the tile, not one per block: see the forward kernel.
    if (kMask != kNoMask && mask.on)
      pass1<kRem, kMask>(p, l, mask, bias, tS, tP, sP, sta, stb, da2, db2);
    else
      pass1<kRem, kNoMask>(p, l, TileMask<kNoMask>(), bias, tS, tP, sP, sta, stb, da2, db2);
    tmem_wait_st();
    fence_proxy_async_shared();
    tc_fence_before();
    __syncwarp();
    if (lane == 0) mbar_arrive(c.bar(kPFull));
    float da = da2.x + da2.y, db = db2.x + db2.y;
    da += __shfl_xor_sync(0xffffffffu, da, 1);
    da += __shfl_xor_sync(0xffffffffu, da, 2);
    db += __shfl_xor_sync(0xffffffffu, db, 1);
    db += __shfl_xor_sync(0xffffffffu, db, 2);
    const float2 ea2 = make_float2(-da, -da), eb2 = make_float2(-db, -db);
    uint32_t sv[8], gv[8];
    tmem_ld_16x256b_r8(tS, sv);
    tmem_ld_16x256b_r8(tP, gv);
    if (!warp_wait(c.bar(kDvFull), par, c.abort, p.status, 123)) {
      tmem_wait_ld();
      return;
    }
    // Pass 2: dS over P in shared memory.
#pragma unroll
    for (int q = 0; q < 9; ++q) {
      tmem_wait_ld();
      uint32_t cs[8], cg[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        cs[e] = sv[e];
        cg[e] = gv[e];
      }
      if (q < 8) {
        tmem_ld_16x256b_r8(tS + 16 * (q + 1), sv);
        tmem_ld_16x256b_r8(tP + 16 * (q + 1), gv);
      }
#pragma unroll
      for (int e = 0; e < 8; e += 4) {
        const int j = 2 * q + (e >> 2);
        const float2 ga = __fmul2_rn(f2(cs[e], cs[e + 1]), __fadd2_rn(f2(cg[e], cg[e + 1]), ea2));
        const float2 gb = __fmul2_rn(f2(cs[e + 2], cs[e + 3]), __fadd2_rn(f2(cg[e + 2], cg[e + 3]), eb2));
        grad.add(j, ga, gb);
        store_p(sP, l, j, pack_bf16x2(ga.x, ga.y), pack_bf16x2(gb.x, gb.y));
      }
    }
    fence_proxy_async_shared();
    tc_fence_before();
    __syncwarp();
    if (lane == 0) mbar_arrive(c.bar(kDsFull));
    // dV while the dK and dQ products run, then those.
    const int quarter = warp & 3;
    uint32_t o[32];
    if constexpr (!kRem) {
      tc_fence_after();
      tmem_ld_16x256b_r32(c.tmem + l.addr + kColDv, o);
      tmem_wait_ld();
      stage_rows(slot + kOffV, l, o, 1.f, 1.f);
      if (warp < 8) stage_rem(c.tmem + kColRem, slot + kOffV, quarter, l, 1.f);
    }
    if (!warp_wait(c.bar(kDkFull), par, c.abort, p.status, 124)) return;
    if constexpr (!kRem) {
      tc_fence_after();
      tmem_ld_16x256b_r32(c.tmem + l.addr + kColDk, o);
      tmem_wait_ld();
      stage_rows(slot + kOffK, l, o, p.scale, p.scale);
      tmem_ld_16x256b_r32(c.tmem + l.addr + kColDq, o);
      tmem_wait_ld();
      stage_rows(slot + kOffQ, l, o, p.scale, p.scale);
      if (warp < 8) stage_rem(c.tmem + kColDq2, slot + kOffQ, quarter, l, p.scale);
      else stage_rem(c.tmem + kColRem + kLaneHalf, slot + kOffK, quarter, l, p.scale);
      fence_proxy_async_shared();
    }
    tc_fence_before();
    __syncwarp();
    if (lane == 0) {
      mbar_arrive(c.bar(kTFree));
      mbar_arrive(c.bar(kStaged + s));
    }
  }
  if (cur_h >= 0) grad.flush(p, cur_h, l);
}

template <int kMask>
__global__ void __launch_bounds__(kThreads, 1)
rel_bias_bwd_tc_kernel(const __grid_constant__ CUtensorMap tmq, const __grid_constant__ CUtensorMap tmk,
                       const __grid_constant__ CUtensorMap tmv, const __grid_constant__ CUtensorMap tmg,
                       const __grid_constant__ CUtensorMap tmdq, const __grid_constant__ CUtensorMap tmdk,
                       const __grid_constant__ CUtensorMap tmdv, const Params p) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + kOffBars);
  uint32_t* tmem_holder = reinterpret_cast<uint32_t*>(bars + kNumBars);
  __shared__ int abort_flag;
  Ctx c;
  c.smem = smem;
  c.sbase = smem_u32(smem);
  c.bar0 = smem_u32(bars);
  c.abort = &abort_flag;
  c.t_begin = tile_begin(p.num_tiles);
  c.n_local = tile_end(p.num_tiles) - c.t_begin;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    abort_flag = 0;
    for (int b = 0; b < kNumBars; ++b) {
      const bool nine = b == kStaged || b == kStaged + 1 || b == kPFull || b == kDsFull || b == kTFree;
      mbar_init(c.bar(b), nine ? 9 : 1);
    }
    fence_mbarrier_init();
  }
  if (warp == 1) {
    tmem_alloc(smem_u32(tmem_holder), kTmemCols);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  c.tmem = *tmem_holder;
  const int n = c.n_local;

  if (warp >= 4) {
    warpgroup_reg_alloc<kRegsMain>();
    softmax_warps<false, kMask>(p, c, warp, lane);
  } else {
    warpgroup_reg_dealloc<kRegsSmall>();
    if (warp == 3) {
      softmax_warps<true, kMask>(p, c, warp, lane);
    } else if (warp == 0) {
      // Loads, and the stores of finished tiles.
      int last_par[kStages] = {-1, -1};
      auto store_out = [&](int j) {
        const int t = c.t_begin + j, h = t / p.Bwin, w = t - h * p.Bwin;
        const uint32_t slot = c.sbase + (j & 1) * kStageBytes;
        tma_store_4d(&tmdq, slot + kOffQ, 0, 0, h, w);
        tma_store_4d(&tmdk, slot + kOffK, 0, 0, h, w);
        tma_store_4d(&tmdv, slot + kOffV, 0, 0, h, w);
        bulk_commit_group();
      };
      for (int i = 0; i < n; ++i) {
        const int t = c.t_begin + i, h = t / p.Bwin, w = t - h * p.Bwin, s = i & 1;
        uint32_t id[5];
        if constexpr (kMask == kGroups) load_ids(p, w, lane, id);
        int ok = 1;
        if (lane == 0 && i >= kStages) {
          ok = mbar_wait(c.bar(kStaged + s), (uint32_t)(((i - kStages) >> 1) & 1), c.abort, p.status, 125, kTimeoutNs);
          if (ok) {
            store_out(i - kStages);
            bulk_wait_group_read0();
          }
        }
        if (!__shfl_sync(0xffffffffu, ok, 0)) break;
        if constexpr (kMask == kGroups) store_ids(smem + kOffIds + s * kIdBytes, lane, id);
        if (lane == 0) {
          const uint32_t bar = c.bar(kFull + s), slot = c.sbase + s * kStageBytes;
          mbar_arrive_expect_tx(bar, kStageBytes);
          tma_load_4d(slot + kOffQ, &tmq, bar, 0, 0, h, w);
          tma_load_4d(slot + kOffK, &tmk, bar, 0, 0, h, w);
          tma_load_4d(slot + kOffV, &tmv, bar, 0, 0, h, w);
          tma_load_4d(slot + kOffG, &tmg, bar, 0, 0, h, w);
          last_par[s] = (i >> 1) & 1;
        }
      }
      if (lane == 0) {
        // Never leave with copies in flight (bounded, also after an abort).
        int no_abort = 0;
        for (int s = 0; s < kStages; ++s)
          if (last_par[s] >= 0) mbar_wait(c.bar(kFull + s), (uint32_t)last_par[s], &no_abort, p.status, 126, kTimeoutNs);
        for (int j = n > kStages ? n - kStages : 0; j < n; ++j) {
          if (!mbar_wait(c.bar(kStaged + (j & 1)), (uint32_t)((j >> 1) & 1), c.abort, p.status, 127, kTimeoutNs)) break;
          store_out(j);
        }
        bulk_wait_group0();
      }
    } else if (warp == 1 && lane == 0) {
      const uint32_t sP = c.sbase + kOffP;
      for (int i = 0; i < n; ++i) {
        const int s = i & 1;
        const uint32_t par = (uint32_t)(i & 1);
        const uint32_t slot = c.sbase + s * kStageBytes;
        const uint32_t sQ = slot + kOffQ, sK = slot + kOffK, sV = slot + kOffV, sG = slot + kOffG;
        if (!mbar_wait(c.bar(kFull + s), (uint32_t)((i >> 1) & 1), c.abort, p.status, 128, kTimeoutNs)) break;
        if (!mbar_wait(c.bar(kTFree), par ^ 1u, c.abort, p.status, 129, kTimeoutNs)) break;
        tc_fence_after();
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const uint64_t b = desc_sw128(sK + k * 32, 16, 1024);
          umma_f16(c.tmem + kColS, desc_sw128(sQ + k * 32, 16, 1024), b, kIdescS, k > 0 ? 1u : 0u);
          umma_f16(c.tmem + kColS2, desc_sw128(sQ + kRowOff80 + k * 32, 16, 1024), b, kIdescS2, k > 0 ? 1u : 0u);
        }
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const uint64_t b = desc_sw128(sV + k * 32, 16, 1024);
          umma_f16(c.tmem + kColP, desc_sw128(sG + k * 32, 16, 1024), b, kIdescS, k > 0 ? 1u : 0u);
          umma_f16(c.tmem + kColS2 + kLaneHalf, desc_sw128(sG + kRowOff80 + k * 32, 16, 1024), b, kIdescS2,
                   k > 0 ? 1u : 0u);
        }
        umma_commit(c.bar(kSFull));
        if (!mbar_wait(c.bar(kPFull), par, c.abort, p.status, 130, kTimeoutNs)) break;
        tc_fence_after();
#pragma unroll
        for (int k = 0; k < 9; ++k) {  // queries 16k .. 16k + 15
          const uint64_t g = desc_sw128(sG + k * 2048, kTileBytes, 1024);
          umma_f16(c.tmem + kColDv, desc_sw128(sP + k * 2048, kPChunk, 1024), g, kIdescT, k > 0 ? 1u : 0u);
          umma_f16(c.tmem + kColRem, g, desc_sw32(sP + 2 * kPChunk + k * 512, 256), kIdescRemT, k > 0 ? 1u : 0u);
        }
        umma_commit(c.bar(kDvFull));
        if (!mbar_wait(c.bar(kDsFull), par, c.abort, p.status, 131, kTimeoutNs)) break;
        tc_fence_after();
#pragma unroll
        for (int k = 0; k < 9; ++k) {
          const uint64_t q = desc_sw128(sQ + k * 2048, kTileBytes, 1024);
          umma_f16(c.tmem + kColDk, desc_sw128(sP + k * 2048, kPChunk, 1024), q, kIdescT, k > 0 ? 1u : 0u);
          umma_f16(c.tmem + kColRem + kLaneHalf, q, desc_sw32(sP + 2 * kPChunk + k * 512, 256), kIdescRemT,
                   k > 0 ? 1u : 0u);
        }
#pragma unroll
        for (int k = 0; k < 9; ++k) {  // keys 16k .. 16k + 15
          const uint64_t kd = desc_sw128(sK + k * 2048, kTileBytes, 1024);
          const uint32_t pa = k < 8 ? sP + (k >> 2) * kPChunk + (k & 3) * 32 : sP + 2 * kPChunk;
          umma_f16(c.tmem + kColDq, k < 8 ? desc_sw128(pa, 16, 1024) : desc_sw32(pa, 256), kd, kIdescO, k > 0 ? 1u : 0u);
          umma_f16(c.tmem + kColDq2, kd, k < 8 ? desc_sw128(pa + 128 * 128, 16, 1024) : desc_sw32(pa + 128 * 32, 256),
                   kIdescRemQ, k > 0 ? 1u : 0u);
        }
        umma_commit(c.bar(kDkFull));
      }
      umma_commit(c.bar(kDone));
      int no_abort = 0;
      mbar_wait(c.bar(kDone), 0, &no_abort, p.status, 132, kTimeoutNs);
    }
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
