// The norms before and after a residual block, fused with the block's gate and residual scale, and
// their gradients. With N(v) the layer norm (or RMS norm) of a row, without affine:
//
//   before   z = N(x) (c2 + s2) + t2                                       x -> the block's input
//   after    y = a r + g (N(x) (c + s) + t)                                the block's output x, residual r
//   between  y as in after, z = N(y) (c2 + s2) + t2                        one block's end, the next one's start
//
// s, t, g, a, s2, t2 are per channel, shared or one row per batch element. Everything is computed in
// fp32 and rounded once per output; z of `between` is computed from the unrounded y.
//
// Backward, with n = N(x), p = n (c + s) + t, m = N(y) and the row statistics the forward pass kept:
//   d = dy + rho2 (dm - mean(dm) - m mean(dm m)),  dm = dz (c2 + s2)       (no mean(dm) for RMS)
//   dr = a d,  dx = rho (dn - mean(dn) - n mean(dn n)),  dn = g d (c + s)
//   ds = sum g d n, dt = sum g d, dg = sum d p, da = sum d r, ds2 = sum dz m, dt2 = sum dz
// The sums over rows are kept in registers by the threads that own the columns, added over a block's
// row groups in shared memory, and over blocks by a second kernel in a fixed order (no atomics).
//
// A row is read once, by its group of `tpr` threads. Forward rows of whole 16-byte units with a residual are bound by
// memory where their width fills the group's threads (0.82 to 1.0 of the measured copy bandwidth at 512, 1024 and 2048
// columns; 0.58 and 0.70 for `between` at 520 and 1536, which leave half and a quarter of them idle). `before` is not
// (0.36 to 0.61): its blocks per SM are those of the forms with five parameter arrays. Rows that go element by element
// are bound by their instructions, the backward pass by the chain of its two reductions. Every thread copies the
// elements that it will itself work on into a ring of its own in shared memory, kStages rows ahead
// (cp.async: no registers, no barrier), so that loads run while rows are reduced; with loads into
// registers at the top of each row the backward pass of (32400, 2048) rows took 504 us and the forward
// pass 336 us. The variance is taken about the mean (two reductions), not as E[x^2] - mean^2.
#include "fa_common.cuh"

namespace fa {
namespace {

enum { kBefore = 0, kAfter = 1, kBetween = 2 };
enum { kPostScale = 0, kPostShift, kGate, kResScale, kPreScale, kPreShift, kParams };
constexpr int kMaxDim = 4096;
constexpr int kFwdThreads = 128;

__device__ __forceinline__ uint32_t smem_addr(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }
__device__ __forceinline__ uint32_t lds32(uint32_t a) {
  uint32_t v;
  asm volatile("ld.shared.u32 %0, [%1];" : "=r"(v) : "r"(a) : "memory");
  return v;
}
__device__ __forceinline__ uint2 lds64(uint32_t a) {
  uint2 v;
  asm volatile("ld.shared.v2.u32 {%0, %1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(a) : "memory");
  return v;
}
__device__ __forceinline__ uint4 lds128(uint32_t a) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(a) : "memory");
  return v;
}

struct NormArgs {
  const void *x, *r, *dy, *dz;
  void *y, *z, *dx, *dr;
  const float* par[kParams];
  int64_t par_stride[kParams];  // batch stride: 0 (shared) or D
  float scale_bias, pre_scale_bias, res_scale, eps, inv_d;
  int rms, D, tpr;
  int64_t L;
  int B;
  float4* stats;  // per row: mean and 1 / deviation of x, and of y
  float* ws;      // backward: (B, gridDim.x, sums, D) partial column sums
  int param_off;  // backward: byte offset of the parameters in shared memory
};

// ------------------------------------------------------------------------------------------
// A row's elements of one thread: kVec: 4 consecutive ones per unit, units tpr apart (so that a warp's
// accesses are whole consecutive sectors in fp32 and bf16); else single elements tpr apart. kN per thread.
// ------------------------------------------------------------------------------------------
template <bool kVec>
__device__ __forceinline__ int col_of(int t, int tpr, int k) {
  return kVec ? (t + tpr * (k >> 2)) * 4 + (k & 3) : t + tpr * k;
}

// One tensor's share of the ring: kN elements per thread and stage. Vector rows go a unit at a time (16
// or 8 bytes), other fp32 rows 4 bytes; other bf16 rows, which cp.async cannot copy, are read when used.
template <typename T, bool kVec, int kN>
struct Column {
  static constexpr bool kRing = kVec || sizeof(T) == 4;
  static constexpr int kBytes = kRing ? kN * (int)sizeof(T) : 0;  // per thread
  static __device__ __forceinline__ void fetch(uint32_t ring, int threads, const T* row, int t, int tpr, int D, bool on) {
    if constexpr (kRing) {
      constexpr int kEls = kVec ? 4 : 1, kUnit = kEls * (int)sizeof(T);
#pragma unroll
      for (int i = 0; i < kN / kEls; ++i) {
        const int c = col_of<kVec>(t, tpr, i * kEls);
        const bool in = on && c < D;  // out of range: zeros
        const uint32_t dst = ring + (uint32_t)(i * threads + threadIdx.x) * kUnit;
        const T* src = in ? row + c : row;
        if constexpr (kUnit == 16)
          asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(in ? 16 : 0) : "memory");
        else
          asm volatile("cp.async.ca.shared.global [%0], [%1], %3, %2;" ::"r"(dst), "l"(src), "r"(in ? kUnit : 0), "n"(kUnit)
                       : "memory");
      }
    }
  }
  // Elements u .. u + 7 of the thread.
  static __device__ __forceinline__ void get8(uint32_t ring, int threads, const T* row, int t, int tpr, int D, bool on, int u,
                                              float2* v) {
    if constexpr (!kRing) {
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const int c0 = col_of<false>(t, tpr, u + 2 * k), c1 = col_of<false>(t, tpr, u + 2 * k + 1);
        v[k] = make_float2(on && c0 < D ? to_f32(row[c0]) : 0.f, on && c1 < D ? to_f32(row[c1]) : 0.f);
      }
    } else if constexpr (!kVec) {
#pragma unroll
      for (int k = 0; k < 4; ++k)
        v[k] = make_float2(__uint_as_float(lds32(ring + (uint32_t)((u + 2 * k) * threads + threadIdx.x) * 4)),
                           __uint_as_float(lds32(ring + (uint32_t)((u + 2 * k + 1) * threads + threadIdx.x) * 4)));
    } else {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const uint32_t at = ring + (uint32_t)((u / 4 + i) * threads + threadIdx.x) * (4 * (int)sizeof(T));
        if constexpr (sizeof(T) == 4) {
          const uint4 q = lds128(at);
          v[2 * i] = make_float2(__uint_as_float(q.x), __uint_as_float(q.y));
          v[2 * i + 1] = make_float2(__uint_as_float(q.z), __uint_as_float(q.w));
        } else {
          const uint2 q = lds64(at);
          v[2 * i] = unpack_bf16x2(q.x);
          v[2 * i + 1] = unpack_bf16x2(q.y);
        }
      }
    }
  }
};

constexpr int kStages = 3, kBwdStages = 2;  // rows of a group in flight
__device__ __forceinline__ void ring_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int kDepth>
__device__ __forceinline__ void ring_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(kDepth - 1) : "memory");
}
__device__ __forceinline__ void ring_drain() { asm volatile("cp.async.wait_all;" ::: "memory"); }

template <typename T, bool kVec, int kP>
__device__ __forceinline__ void store_row(T* row, int t, int tpr, int D, bool on, const float2 (&v)[kP]) {
  if (!on) return;
#pragma unroll
  for (int k = 0; k < kP; k += 2) {
    if constexpr (kVec) {
      const int c = col_of<true>(t, tpr, 2 * k);
      if (c >= D) continue;
      if constexpr (sizeof(T) == 4)
        *reinterpret_cast<float4*>(row + c) = make_float4(v[k].x, v[k].y, v[k + 1].x, v[k + 1].y);
      else
        *reinterpret_cast<uint2*>(row + c) = make_uint2(pack_bf16x2(v[k].x, v[k].y), pack_bf16x2(v[k + 1].x, v[k + 1].y));
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int c = col_of<false>(t, tpr, 2 * k + e);
        if (c < D) row[c] = from_f32<T>(e & 1 ? v[k + (e >> 1)].y : v[k + (e >> 1)].x);
      }
    }
  }
}

// Columns u .. u+7 of this thread of a parameter row plus `add` (null: `fill`; past D: 0).
template <bool kVec>
__device__ __forceinline__ void param8(const float* p, int t, int tpr, int D, int u, float add, float fill, float2* v) {
#pragma unroll
  for (int k = 0; k < 4; k += 2) {
    float e[4];
    const int c0 = col_of<kVec>(t, tpr, u + 2 * k);
    if (!p) {
#pragma unroll
      for (int i = 0; i < 4; ++i) e[i] = fill;
    } else if constexpr (kVec) {
      const float4 q = c0 < D ? __ldg(reinterpret_cast<const float4*>(p + c0)) : make_float4(-add, -add, -add, -add);
      e[0] = q.x + add;
      e[1] = q.y + add;
      e[2] = q.z + add;
      e[3] = q.w + add;
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int c = col_of<false>(t, tpr, u + 2 * k + i);
        e[i] = c < D ? __ldg(p + c) + add : 0.f;
      }
    }
    v[k] = make_float2(e[0], e[1]);
    v[k + 1] = make_float2(e[2], e[3]);
  }
}

// ------------------------------------------------------------------------------------------
// Sums over the threads of a row: shuffles inside a warp (rows narrower than a warp share one), and
// one named barrier per sum across warps; `buf` alternates so that one barrier is enough.
// ------------------------------------------------------------------------------------------
struct Group {
  int tpr, id, t;  // threads per row, row group in the block, thread in the group
  float2* buf;     // two buffers of (tpr / 32) partial sums of this group, read in pairs
  int par;
};

template <int kVals>
__device__ __forceinline__ void group_sum(Group& g, float (&v)[kVals]) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    if (o < g.tpr) {
#pragma unroll
      for (int i = 0; i < kVals; ++i) v[i] += __shfl_xor_sync(0xffffffffu, v[i], o);
    }
  }
  if (g.tpr > 32) {
    const int warps = g.tpr >> 5;
    float* b = reinterpret_cast<float*>(g.buf) + g.par * kVals * warps;
    g.par ^= 1;
    if ((g.t & 31) == 0) {
#pragma unroll
      for (int i = 0; i < kVals; ++i) b[(g.t >> 5) * kVals + i] = v[i];
    }
    asm volatile("bar.sync %0, %1;" ::"r"(g.id + 1), "r"(g.tpr) : "memory");
    // Two partial sums (of one value) or one (of two) per 8-byte read, in the same order for every thread.
    const float2* b2 = reinterpret_cast<const float2*>(b);
    float2 s = b2[0];
    const int reads = warps * kVals / 2;
    for (int w = 1; w < reads; ++w) {
      const float2 e = b2[w];
      s.x += e.x;
      s.y += e.y;
    }
    if constexpr (kVals == 1) {
      v[0] = s.x + s.y;
    } else {
      v[0] = s.x;
      v[1] = s.y;
    }
  }
}

__device__ __forceinline__ float2 dup(float v) { return make_float2(v, v); }
__device__ __forceinline__ float total(float2 v) { return v.x + v.y; }

// 1 for each of the pair (2 k, 2 k + 1) of this thread's columns that lies in the row, 0 for the others.
// Vector rows are in or out 4 columns at a time.
template <bool kVec>
__device__ __forceinline__ float2 in_row(const Group& g, int D, int k) {
  if constexpr (kVec) return dup(col_of<true>(g.t, g.tpr, 2 * k) < D ? 1.f : 0.f);
  else
    return make_float2(col_of<false>(g.t, g.tpr, 2 * k) < D ? 1.f : 0.f,
                       col_of<false>(g.t, g.tpr, 2 * k + 1) < D ? 1.f : 0.f);
}

// Mean and 1 / deviation of a row held by a group; v becomes the normalised row (0 past D, where it
// must come in as 0).
template <bool kVec, int kP>
__device__ __forceinline__ float2 normalise(Group& g, const NormArgs& a, float2 (&v)[kP]) {
  float s[1] = {0.f};
  float mean = 0.f;
  if (!a.rms) {
    float2 t = v[0];
#pragma unroll
    for (int k = 1; k < kP; ++k) t = __fadd2_rn(t, v[k]);
    s[0] = total(t);
    group_sum<1>(g, s);
    mean = s[0] * a.inv_d;
    const float2 m2 = dup(-mean);
#pragma unroll
    for (int k = 0; k < kP; ++k) v[k] = __ffma2_rn(in_row<kVec>(g, a.D, k), m2, v[k]);
  }
  float2 q = make_float2(0.f, 0.f);
#pragma unroll
  for (int k = 0; k < kP; ++k) q = __ffma2_rn(v[k], v[k], q);
  s[0] = total(q);
  group_sum<1>(g, s);
  const float rstd = rsqrtf(fmaf(s[0], a.inv_d, a.eps));
  const float2 r2 = dup(rstd);
#pragma unroll
  for (int k = 0; k < kP; ++k) v[k] = __fmul2_rn(v[k], r2);
  return make_float2(mean, rstd);
}

// kVpt units of 8 elements per thread. YT: the type of r and y, or of z in the `before` form. The
// parameters of a thread's columns stay in registers over its rows: y = a r + (g s) n + (g t).
template <typename XT, typename YT, int kForm, bool kVec, int kVpt>
__global__ void __launch_bounds__(kFwdThreads, kVpt == 2 ? 3 : 2) block_norm_kernel(const NormArgs a) {
  constexpr int kN = 8 * kVpt;
  using ColX = Column<XT, kVec, kN>;
  using ColR = Column<YT, kVec, kN>;
  constexpr int kStage = (ColX::kBytes + (kForm == kBefore ? 0 : ColR::kBytes)) * kFwdThreads;
  extern __shared__ __align__(16) uint8_t ring_mem[];
  __shared__ float2 buf[kFwdThreads / 32];
  const uint32_t ring = smem_addr(ring_mem);
  Group g;
  g.tpr = a.tpr;
  g.id = threadIdx.x / a.tpr;
  g.t = threadIdx.x - g.id * a.tpr;
  g.buf = buf + (g.id * a.tpr >> 5);
  g.par = 0;
  const int groups = kFwdThreads / a.tpr, D = a.D;
  const int64_t step = (int64_t)gridDim.x * groups;
  for (int b = blockIdx.y; b < a.B; b += gridDim.y) {
    const int64_t first = (int64_t)blockIdx.x * groups + g.id, base = (int64_t)b * a.L;
    auto fetch = [&](int64_t i, int stage) {
      const int64_t row = first + i * step;
      const bool on = row < a.L;
      const int64_t off = (base + (on ? row : 0)) * D;
      ColX::fetch(ring + stage * kStage, kFwdThreads, reinterpret_cast<const XT*>(a.x) + off, g.t, g.tpr, D, on);
      if constexpr (kForm != kBefore)
        ColR::fetch(ring + stage * kStage + ColX::kBytes * kFwdThreads, kFwdThreads, reinterpret_cast<const YT*>(a.r) + off, g.t,
                    g.tpr, D, on);
      ring_commit();
    };
#pragma unroll
    for (int i = 0; i < kStages; ++i) fetch(i, i);
    constexpr int kP = kN / 2, kPost = kForm == kBefore ? 1 : kP, kPre = kForm == kAfter ? 1 : kP;
    float2 gs[kPost], gt[kPost], rs[kPost], s2[kPre], t2[kPre];
    auto par = [&](int i) { return a.par[i] ? a.par[i] + b * a.par_stride[i] : nullptr; };
#pragma unroll
    for (int u = 0; u < kP; u += 4) {
      if constexpr (kForm != kBefore) {
        float2 p[4];
        param8<kVec>(par(kGate), g.t, g.tpr, D, 2 * u, 0.f, 1.f, p);
        param8<kVec>(par(kPostScale), g.t, g.tpr, D, 2 * u, a.scale_bias, a.scale_bias, &gs[u]);
        param8<kVec>(par(kPostShift), g.t, g.tpr, D, 2 * u, 0.f, 0.f, &gt[u]);
        param8<kVec>(par(kResScale), g.t, g.tpr, D, 2 * u, 0.f, a.res_scale, &rs[u]);
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          gs[u + k] = __fmul2_rn(gs[u + k], p[k]);
          gt[u + k] = __fmul2_rn(gt[u + k], __fmul2_rn(p[k], in_row<kVec>(g, D, u + k)));
        }
      }
      if constexpr (kForm != kAfter) {
        param8<kVec>(par(kPreScale), g.t, g.tpr, D, 2 * u, a.pre_scale_bias, a.pre_scale_bias, &s2[u]);
        param8<kVec>(par(kPreShift), g.t, g.tpr, D, 2 * u, 0.f, 0.f, &t2[u]);
      }
    }
    int stage = 0;
    int64_t i = 0;
    for (int64_t row0 = (int64_t)blockIdx.x * groups; row0 < a.L; row0 += step, ++i) {
      const bool on = row0 + g.id < a.L;
      const int64_t row = base + row0 + g.id, off = row * D;
      const uint32_t at = ring + stage * kStage;
      ring_wait<kStages>();
      float2 v[kP];
#pragma unroll
      for (int u = 0; u < kP; u += 4)
        ColX::get8(at, kFwdThreads, reinterpret_cast<const XT*>(a.x) + off, g.t, g.tpr, D, on, 2 * u, &v[u]);
      float4 st = make_float4(0.f, 0.f, 0.f, 0.f);
      const float2 sx = normalise<kVec>(g, a, v);
      st.x = sx.x;
      st.y = sx.y;
      if constexpr (kForm != kBefore) {
#pragma unroll
        for (int u = 0; u < kP; u += 4) {
          float2 r[4];
          ColR::get8(at + ColX::kBytes * kFwdThreads, kFwdThreads, reinterpret_cast<const YT*>(a.r) + off, g.t, g.tpr, D, on,
                     2 * u, r);
#pragma unroll
          for (int k = 0; k < 4; ++k) v[u + k] = __ffma2_rn(v[u + k], gs[u + k], __ffma2_rn(rs[u + k], r[k], gt[u + k]));
        }
        store_row<YT, kVec>(reinterpret_cast<YT*>(a.y) + off, g.t, g.tpr, D, on, v);
        if constexpr (kForm == kBetween) {
          const float2 sy = normalise<kVec>(g, a, v);
          st.z = sy.x;
          st.w = sy.y;
        }
      }
      fetch(i + kStages, stage);  // this thread has read its part of the stage
      stage = stage + 1 == kStages ? 0 : stage + 1;
      if constexpr (kForm != kAfter) {
#pragma unroll
        for (int k = 0; k < kP; ++k) v[k] = __ffma2_rn(v[k], s2[k], t2[k]);
        using ZT = typename std::conditional<kForm == kBefore, YT, XT>::type;
        store_row<ZT, kVec>(reinterpret_cast<ZT*>(a.z) + off, g.t, g.tpr, D, on, v);
      }
      if (a.stats && on && g.t == 0) a.stats[row] = st;
    }
    ring_drain();
  }
}

// ------------------------------------------------------------------------------------------
// Backward: 8 elements per thread, tpr = 1 .. 512 threads per row.
// ------------------------------------------------------------------------------------------
template <int kForm> constexpr int kSums = kForm == kBefore ? 2 : kForm == kAfter ? 4 : 6;
constexpr int kBwdMaxThreads = 512;

template <typename XT, typename YT, int kForm, bool kVec>
__global__ void __launch_bounds__(kBwdMaxThreads, 1) block_norm_bwd_kernel(const NormArgs a) {
  constexpr int kS = kSums<kForm>;
  constexpr int kPost = 0, kPre = kForm == kBefore ? 0 : 4;  // first sum of each norm
  using ZT = typename std::conditional<kForm == kBefore, YT, XT>::type;
  using ColX = Column<XT, kVec, 8>;
  using ColY = Column<YT, kVec, 8>;
  using ColZ = Column<ZT, kVec, 8>;
  constexpr int kX = ColX::kBytes, kR = kForm == kBefore ? 0 : ColY::kBytes, kZ = kForm == kAfter ? 0 : ColZ::kBytes;
  extern __shared__ __align__(16) uint8_t ring_mem[];
  __shared__ float2 buf[2 * kBwdMaxThreads / 32];
  float* comb = reinterpret_cast<float*>(ring_mem);  // after the rows
  const uint32_t ring = smem_addr(ring_mem), stage_bytes = (kX + 2 * kR + kZ) * blockDim.x;
  // After the ring (or the sums, whichever is larger): the parameters.
  float4* params = reinterpret_cast<float4*>(ring_mem + a.param_off);
  Group g;
  g.tpr = a.tpr;
  g.id = threadIdx.x / a.tpr;
  g.t = threadIdx.x - g.id * a.tpr;
  g.buf = buf + 2 * (g.id * a.tpr >> 5);
  g.par = 0;
  const int groups = blockDim.x / a.tpr, D = a.D, threads = blockDim.x;
  const int64_t step = (int64_t)gridDim.x * groups;
  for (int b = blockIdx.y; b < a.B; b += gridDim.y) {
    const int64_t first = (int64_t)blockIdx.x * groups + g.id, base = (int64_t)b * a.L;
    auto fetch = [&](int64_t i, int stage) {
      const int64_t row = first + i * step;
      const bool on = row < a.L;
      const int64_t off = (base + (on ? row : 0)) * D;
      uint32_t at = ring + stage * stage_bytes;
      ColX::fetch(at, threads, reinterpret_cast<const XT*>(a.x) + off, g.t, g.tpr, D, on);
      at += kX * threads;
      if constexpr (kForm != kBefore) {
        ColY::fetch(at, threads, reinterpret_cast<const YT*>(a.r) + off, g.t, g.tpr, D, on);
        at += kR * threads;
        if (a.dy) ColY::fetch(at, threads, reinterpret_cast<const YT*>(a.dy) + off, g.t, g.tpr, D, on);
        at += kR * threads;
      }
      if (kForm != kAfter && a.dz) ColZ::fetch(at, threads, reinterpret_cast<const ZT*>(a.dz) + off, g.t, g.tpr, D, on);
      ring_commit();
    };
#pragma unroll
    for (int i = 0; i < kBwdStages; ++i) fetch(i, i);
    // The parameters that a row needs, once per batch element, into shared memory in the order in which the
    // group's threads read them (fetched from global memory row by row, 40 KB a row of 2048, they missed L1
    // and cost two thirds of the kernel's time).
    if (g.id == 0) {
      auto put = [&](int slot, int i, float add, float fill) {
        float2 v[4];
        param8<kVec>(a.par[i] ? a.par[i] + b * a.par_stride[i] : nullptr, g.t, g.tpr, D, 0, add, fill, v);
#pragma unroll
        for (int k = 0; k < 2; ++k)
          params[(2 * slot + k) * g.tpr + g.t] = make_float4(v[2 * k].x, v[2 * k].y, v[2 * k + 1].x, v[2 * k + 1].y);
      };
      if constexpr (kForm == kBefore) {
        put(0, kPreScale, a.pre_scale_bias, a.pre_scale_bias);
      } else {
        put(0, kPostScale, a.scale_bias, a.scale_bias);
        put(1, kPostShift, 0.f, 0.f);
        put(2, kGate, 0.f, 1.f);
        put(3, kResScale, 0.f, a.res_scale);
        if constexpr (kForm == kBetween) put(4, kPreScale, a.pre_scale_bias, a.pre_scale_bias);
      }
    }
    __syncthreads();
    auto pget = [&](int slot, float2 (&v)[4]) {
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        const float4 q = params[(2 * slot + k) * g.tpr + g.t];
        v[2 * k] = make_float2(q.x, q.y);
        v[2 * k + 1] = make_float2(q.z, q.w);
      }
    };
    float2 acc[kS][4];
#pragma unroll
    for (int i = 0; i < kS; ++i)
#pragma unroll
      for (int k = 0; k < 4; ++k) acc[i][k] = make_float2(0.f, 0.f);
    int stage = 0;
    int64_t it = 0;
    const float4 none = make_float4(0.f, 0.f, 0.f, 0.f);
    float4 next = first < a.L ? __ldg(a.stats + base + first) : none;
    for (int64_t row0 = (int64_t)blockIdx.x * groups; row0 < a.L; row0 += step, ++it) {
      const bool on = row0 + g.id < a.L;
      const int64_t row = base + row0 + g.id, off = row * D;
      const float4 st = next;
      next = row0 + step + g.id < a.L ? __ldg(a.stats + row + step) : none;
      ring_wait<kBwdStages>();
      const uint32_t at = ring + stage * stage_bytes;
      // Values that two phases need (r, the parameters) are read from shared memory in each: the sums take 48
      // registers, and what is held over a reduction comes on top.
      float2 n[4];  // x, then the normalised row
      ColX::get8(at, threads, reinterpret_cast<const XT*>(a.x) + off, g.t, g.tpr, D, on, 0, n);
      const uint32_t at_r = at + kX * threads, at_d = at_r + kR * threads, at_z = at_d + kR * threads;
      auto get_r = [&](float2 (&v)[4]) {
        ColY::get8(at_r, threads, reinterpret_cast<const YT*>(a.r) + off, g.t, g.tpr, D, on, 0, v);
      };
      // Columns past D come in as zeros and stay so: their 1 / deviation is 0.
      constexpr int kU = kVec ? 2 : 1;  // pairs per unit
      float2 rho[4 / kU];
#pragma unroll
      for (int k = 0; k < 4; k += kU) rho[k / kU] = __fmul2_rn(dup(st.y), in_row<kVec>(g, D, k));
      const float2 mean = dup(-st.x);
#pragma unroll
      for (int k = 0; k < 4; ++k) n[k] = __fmul2_rn(__fadd2_rn(n[k], mean), rho[k / kU]);
      auto get_p = [&](float2 (&v)[4]) {
        float2 s[4];
        pget(0, s);
        pget(1, v);
#pragma unroll
        for (int k = 0; k < 4; ++k) v[k] = __ffma2_rn(n[k], s[k], v[k]);
      };
      float2 z[4], dn[4];
      if constexpr (kForm != kAfter) {
        if (a.dz) {
          ColZ::get8(at_z, threads, reinterpret_cast<const ZT*>(a.dz) + off, g.t, g.tpr, D, on, 0, z);
        } else {
#pragma unroll
          for (int k = 0; k < 4; ++k) z[k] = make_float2(0.f, 0.f);
        }
      }
      if constexpr (kForm == kBefore) {
        float2 s2[4];
        pget(0, s2);
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          acc[kPre][k] = __ffma2_rn(z[k], n[k], acc[kPre][k]);
          acc[kPre + 1][k] = __fadd2_rn(acc[kPre + 1][k], z[k]);
          dn[k] = __fmul2_rn(z[k], s2[k]);
        }
      } else {
        if constexpr (kForm == kBetween) {
          float2 m[4], q0 = make_float2(0.f, 0.f), q1 = q0;
          {
            float2 r[4], e[4];
            get_p(m);
            pget(2, e);
#pragma unroll
            for (int k = 0; k < 4; ++k) m[k] = __fmul2_rn(m[k], e[k]);
            get_r(r);
            pget(3, e);
            const float2 mean2 = dup(-st.z), rstd2 = dup(st.w);
#pragma unroll
            for (int k = 0; k < 4; ++k)
              m[k] = __fmul2_rn(__fadd2_rn(__ffma2_rn(e[k], r[k], m[k]), mean2), __fmul2_rn(rstd2, in_row<kVec>(g, D, k)));
          }
          float2 s2[4];
          pget(4, s2);
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            acc[kPre][k] = __ffma2_rn(z[k], m[k], acc[kPre][k]);
            acc[kPre + 1][k] = __fadd2_rn(acc[kPre + 1][k], z[k]);
            z[k] = __fmul2_rn(z[k], s2[k]);  // dm
            q0 = __fadd2_rn(q0, z[k]);
            q1 = __ffma2_rn(z[k], m[k], q1);
          }
          float sum[2] = {total(q0), total(q1)};
          group_sum<2>(g, sum);
          const float2 c0 = dup(a.rms ? 0.f : -sum[0] * a.inv_d), c1 = dup(-sum[1] * a.inv_d), rstd2 = dup(st.w);
#pragma unroll
          for (int k = 0; k < 4; ++k)
            z[k] = __fmul2_rn(__fmul2_rn(rstd2, in_row<kVec>(g, D, k)), __ffma2_rn(m[k], c1, __fadd2_rn(z[k], c0)));
        }
        float2 d[4];
        if (a.dy) {
          ColY::get8(at_d, threads, reinterpret_cast<const YT*>(a.dy) + off, g.t, g.tpr, D, on, 0, d);
        } else {
#pragma unroll
          for (int k = 0; k < 4; ++k) d[k] = make_float2(0.f, 0.f);
        }
        if constexpr (kForm == kBetween) {
#pragma unroll
          for (int k = 0; k < 4; ++k) d[k] = __fadd2_rn(d[k], z[k]);
        }
        float2 e[4], f[4];
        get_r(e);
        pget(3, f);
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          acc[kPost + kResScale][k] = __ffma2_rn(d[k], e[k], acc[kPost + kResScale][k]);
          f[k] = __fmul2_rn(f[k], d[k]);
        }
        if (a.dr) store_row<YT, kVec>(reinterpret_cast<YT*>(a.dr) + off, g.t, g.tpr, D, on, f);
        get_p(e);
        pget(2, f);
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          acc[kPost + kGate][k] = __ffma2_rn(d[k], e[k], acc[kPost + kGate][k]);
          d[k] = __fmul2_rn(f[k], d[k]);  // dp
          acc[kPost + kPostScale][k] = __ffma2_rn(d[k], n[k], acc[kPost + kPostScale][k]);
          acc[kPost + kPostShift][k] = __fadd2_rn(acc[kPost + kPostShift][k], d[k]);
        }
        pget(0, f);
#pragma unroll
        for (int k = 0; k < 4; ++k) dn[k] = __fmul2_rn(d[k], f[k]);
      }
      if (a.dx) {
        float2 q0 = make_float2(0.f, 0.f), q1 = q0;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          q0 = __fadd2_rn(q0, dn[k]);
          q1 = __ffma2_rn(dn[k], n[k], q1);
        }
        float sum[2] = {total(q0), total(q1)};
        group_sum<2>(g, sum);
        const float2 c0 = dup(a.rms ? 0.f : -sum[0] * a.inv_d), c1 = dup(-sum[1] * a.inv_d);
#pragma unroll
        for (int k = 0; k < 4; ++k)
          dn[k] = __fmul2_rn(rho[k / kU], __ffma2_rn(n[k], c1, __fadd2_rn(dn[k], c0)));
        store_row<XT, kVec>(reinterpret_cast<XT*>(a.dx) + off, g.t, g.tpr, D, on, dn);
      }
      fetch(it + kBwdStages, stage);  // this thread is done with its part of the stage
      stage = stage + 1 == kBwdStages ? 0 : stage + 1;
    }
    ring_drain();
    // This block's column sums of batch element b: over its row groups in turn, then to the workspace.
    float* ws = a.ws + ((int64_t)b * gridDim.x + blockIdx.x) * kS * D;
    if (groups == 1) {
#pragma unroll
      for (int i = 0; i < kS; ++i)
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          const int c = col_of<kVec>(g.t, g.tpr, k);
          if (c < D) ws[(int64_t)i * D + c] = k & 1 ? acc[i][k >> 1].y : acc[i][k >> 1].x;
        }
    } else {
      for (int q = 0; q < groups; ++q) {
        __syncthreads();
        if (g.id == q) {
#pragma unroll
          for (int i = 0; i < kS; ++i)
#pragma unroll
            for (int k = 0; k < 8; ++k) {
              const int c = col_of<kVec>(g.t, g.tpr, k);
              const float e = k & 1 ? acc[i][k >> 1].y : acc[i][k >> 1].x;
              if (c < D) comb[i * D + c] = q == 0 ? e : comb[i * D + c] + e;
            }
        }
      }
      __syncthreads();
      for (int e = threadIdx.x; e < kS * D; e += blockDim.x) ws[e] = comb[e];
    }
    __syncthreads();  // the next batch element uses the ring and the parameters again
  }
}

// Column sums over blocks (and batch elements, for a shared parameter), in double; the partials are still in L2.
// Eight rows of threads: 9 us for 2 x 148 partials of 6 x 2048 columns (19 with 32 rows), 8 us for 296 of 4 x 771 (9).
struct SumArgs {
  const float* ws;
  float* out[kParams];
  int per_batch[kParams];
  int first;  // parameter of sum 0
  int sums, blocks, B, D;
};
constexpr int kSumRows = 8;

__global__ void __launch_bounds__(32 * kSumRows) block_norm_sum_kernel(const SumArgs a) {
  const int i = blockIdx.z, c = blockIdx.x * 32 + threadIdx.x;
  float* out = a.out[a.first + i];
  if (!out) return;
  const bool own = a.per_batch[a.first + i];
  for (int b = blockIdx.y; b < (own ? a.B : 1); b += gridDim.y) {
    const int64_t lo = own ? (int64_t)b * a.blocks : 0, hi = own ? lo + a.blocks : (int64_t)a.B * a.blocks;
    double s = 0.0;
    if (c < a.D) {
#pragma unroll 8
      for (int64_t e = lo + threadIdx.y; e < hi; e += kSumRows) s += (double)a.ws[(e * a.sums + i) * a.D + c];
    }
    __shared__ double part[kSumRows][32];
    __syncthreads();
    part[threadIdx.y][threadIdx.x] = s;
    __syncthreads();
    if (threadIdx.y == 0 && c < a.D) {
      for (int y = 1; y < kSumRows; ++y) s += part[y][threadIdx.x];
      out[(int64_t)b * a.D + c] = (float)s;
    }
  }
}

int pow2_at_least(int v) {
  int p = 1;
  while (p < v) p *= 2;
  return p;
}

int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

bool any_per_batch(const int64_t* strides) {
  for (int i = 0; i < kParams; ++i)
    if (strides[i]) return true;
  return false;
}

struct BwdShape {
  int tpr, threads;
  int64_t B, L, blocks;  // batch elements and rows as the kernel sees them, blocks per batch element
};

BwdShape bwd_shape(const int64_t* strides, int64_t B, int64_t L, int64_t D) {
  BwdShape s;
  s.tpr = pow2_at_least((int)ceil_div(D, 8));
  s.threads = s.tpr > 256 ? 512 : 256;
  const bool split = any_per_batch(strides);
  s.B = split ? B : 1;
  s.L = split ? L : B * L;
  const int64_t resident = (int64_t)num_sms() * (512 / s.threads);
  const int64_t most = ceil_div(s.L, s.threads / s.tpr);
  s.blocks = resident / (s.B > 0 ? s.B : 1);
  if (s.blocks > most) s.blocks = most;
  if (s.blocks < 1) s.blocks = 1;
  return s;
}

int sums_of(int form) { return form == kBefore ? 2 : form == kAfter ? 4 : 6; }

template <typename XT, typename YT, int kForm>
int launch_fwd(NormArgs& a, bool vec, cudaStream_t s) {
  // 16 elements per thread or 32 (fewer warps a reduction, fewer warps an SM). 64M bf16 elements with an fp32
  // residual, in us at 32 / 16:      520        768        1024       1536       2048 columns
  //   before                       114 / 134   82 / 92    68 / 74    92 / 113   74 / 89
  //   after                        111 / 131  124 / 107  121 / 120  120 / 119  125 / 103
  //   between                      216 / 244  157 / 171  142 / 138  179 / 205  150 / 165
  // so 32 above 512 columns, but for `after` below 768 only. Element-wise rows, bound by their instructions and with
  // spills at 32, keep 16 as long as a block covers a row (21003 fp32 rows of 771: 57 us against 103).
  const bool wide = a.D > (!vec || (kForm == kAfter && a.D >= 768) ? 16 * kFwdThreads : 512);
  a.tpr = pow2_at_least((int)ceil_div(a.D, wide ? 32 : 16));
  const int groups = kFwdThreads / a.tpr;
  auto kern = vec ? (wide ? block_norm_kernel<XT, YT, kForm, true, 4> : block_norm_kernel<XT, YT, kForm, true, 2>)
                  : (wide ? block_norm_kernel<XT, YT, kForm, false, 4> : block_norm_kernel<XT, YT, kForm, false, 2>);
  int64_t gx = (int64_t)num_sms() * (wide ? 2 : 3) / a.B;  // resident blocks, each walking its rows
  const int64_t most = ceil_div(a.L, groups);
  gx = gx > most ? most : gx;
  const int per_el = (vec || sizeof(XT) == 4 ? (int)sizeof(XT) : 0) +
                     (kForm != kBefore && (vec || sizeof(YT) == 4) ? (int)sizeof(YT) : 0);
  const int smem = kStages * kFwdThreads * (wide ? 32 : 16) * per_el;
  FA_CUDA(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
  kern<<<dim3((unsigned)(gx < 1 ? 1 : gx), (unsigned)(a.B < 65535 ? a.B : 65535)), kFwdThreads, smem, s>>>(a);
  return check_launch("block_norm_kernel");
}

template <typename XT, typename YT, int kForm>
int launch_bwd(NormArgs& a, const BwdShape& sh, bool vec, cudaStream_t s) {
  auto kern = vec ? block_norm_bwd_kernel<XT, YT, kForm, true> : block_norm_bwd_kernel<XT, YT, kForm, false>;
  constexpr int kY = (int)sizeof(YT), kX = (int)sizeof(XT), kZ = kForm == kBefore ? kY : kX;
  int per_el = vec || kX == 4 ? kX : 0;
  if (kForm != kBefore && (vec || kY == 4)) per_el += 2 * kY;
  if (kForm != kAfter && (vec || kZ == 4)) per_el += kZ;
  int smem = kBwdStages * sh.threads * 8 * per_el;
  const int combine = sh.threads > sh.tpr ? kSums<kForm> * a.D * 4 : 0;
  if (smem < combine) smem = (combine + 15) / 16 * 16;
  a.param_off = smem;
  smem += (kForm == kBefore ? 1 : kForm == kAfter ? 4 : 5) * 8 * sh.tpr * 4;
  FA_CUDA(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
  kern<<<dim3((unsigned)sh.blocks, (unsigned)(sh.B < 65535 ? sh.B : 65535)), sh.threads, smem, s>>>(a);
  return check_launch("block_norm_bwd_kernel");
}

int check_args(int form, int norm, const void* x, int x_dtype, const void* r, int y_dtype, const float* const* params,
               const int64_t* strides, int64_t B, int64_t L, int64_t D) {
  FA_REQUIRE(form >= kBefore && form <= kBetween, FA_ERR_INVALID, "form must be FA_NORM_BEFORE, _AFTER or _BETWEEN");
  FA_REQUIRE(norm == FA_NORM_LAYER || norm == FA_NORM_RMS, FA_ERR_INVALID, "norm must be FA_NORM_LAYER or FA_NORM_RMS");
  FA_REQUIRE((x_dtype == FA_F32 || x_dtype == FA_BF16) && (y_dtype == FA_F32 || y_dtype == FA_BF16), FA_ERR_INVALID,
             "dtype must be FA_F32 or FA_BF16");
  FA_REQUIRE(B >= 0 && L >= 0 && D >= 1 && B < ((int64_t)1 << 31), FA_ERR_INVALID, "invalid shape");
  FA_REQUIRE(D <= kMaxDim, FA_ERR_UNSUPPORTED, "block norms support D <= 4096");
  FA_REQUIRE(L == 0 || B <= (((int64_t)1 << 60) / kMaxDim) / L, FA_ERR_INVALID, "shape too large");
  FA_REQUIRE(params && strides, FA_ERR_INVALID, "null parameter array");
  FA_REQUIRE(B * L == 0 || (x && (form == kBefore || r)), FA_ERR_INVALID, "null tensor pointer");
  for (int i = 0; i < kParams; ++i)
    FA_REQUIRE(strides[i] == 0 || (strides[i] == D && params[i]), FA_ERR_INVALID,
               "a parameter's batch stride must be 0 or D");
  return FA_OK;
}

void fill(NormArgs& a, int norm, const void* x, const void* r, const float* const* params, const int64_t* strides,
          float scale_bias, float pre_scale_bias, float res_scale, float eps, int64_t B, int64_t L, int64_t D) {
  a.x = x; a.r = r;
  const bool split = any_per_batch(strides);
  for (int i = 0; i < kParams; ++i) {
    a.par[i] = params[i];
    a.par_stride[i] = strides[i];
  }
  a.scale_bias = scale_bias; a.pre_scale_bias = pre_scale_bias; a.res_scale = res_scale; a.eps = eps;
  a.inv_d = 1.f / (float)D;
  a.rms = norm == FA_NORM_RMS; a.D = (int)D;
  a.B = split ? (int)B : 1;
  a.L = split ? L : B * L;
}

bool params_aligned(const float* const* params) {
  for (int i = 0; i < kParams; ++i)
    if (!aligned16(params[i])) return false;
  return true;
}

#define FA_NORM_DISPATCH(LAUNCH, ...)                                                                             \
  if (x_dtype == FA_F32 && y_dtype == FA_F32) return LAUNCH(float, float, __VA_ARGS__);                             \
  if (x_dtype == FA_F32) return LAUNCH(float, __nv_bfloat16, __VA_ARGS__);                                          \
  if (y_dtype == FA_F32) return LAUNCH(__nv_bfloat16, float, __VA_ARGS__);                                          \
  return LAUNCH(__nv_bfloat16, __nv_bfloat16, __VA_ARGS__)

template <typename XT, typename YT>
int fwd_form(int form, NormArgs& a, bool vec, cudaStream_t s) {
  if (form == kBefore) return launch_fwd<XT, YT, kBefore>(a, vec, s);
  if (form == kAfter) return launch_fwd<XT, YT, kAfter>(a, vec, s);
  return launch_fwd<XT, YT, kBetween>(a, vec, s);
}
template <typename XT, typename YT>
int bwd_form(int form, NormArgs& a, const BwdShape& sh, bool vec, cudaStream_t s) {
  if (form == kBefore) return launch_bwd<XT, YT, kBefore>(a, sh, vec, s);
  if (form == kAfter) return launch_bwd<XT, YT, kAfter>(a, sh, vec, s);
  return launch_bwd<XT, YT, kBetween>(a, sh, vec, s);
}
#define FA_FWD(XT, YT, ...) fwd_form<XT, YT>(__VA_ARGS__)
#define FA_BWD(XT, YT, ...) bwd_form<XT, YT>(__VA_ARGS__)

int dispatch_fwd(int x_dtype, int y_dtype, int form, NormArgs& a, bool vec, cudaStream_t s) {
  FA_NORM_DISPATCH(FA_FWD, form, a, vec, s);
}
int dispatch_bwd(int x_dtype, int y_dtype, int form, NormArgs& a, const BwdShape& sh, bool vec, cudaStream_t s) {
  FA_NORM_DISPATCH(FA_BWD, form, a, sh, vec, s);
}

}  // namespace
}  // namespace fa

using namespace fa;

extern "C" int fa_block_norm(int form, int norm, const void* x, int x_dtype, const void* residual, int y_dtype,
                             const float* const params[6], const int64_t param_strides[6], float scale_bias,
                             float pre_scale_bias, float residual_scale, float eps, void* y, void* z, float* stats,
                             int64_t B, int64_t L, int64_t D, void* stream) {
  const int rc = check_args(form, norm, x, x_dtype, residual, y_dtype, params, param_strides, B, L, D);
  if (rc != FA_OK || B * L == 0) return rc;
  FA_REQUIRE((form == kBefore || y) && (form == kAfter || z), FA_ERR_INVALID, "null output pointer");
  FA_REQUIRE(aligned16(stats), FA_ERR_INVALID, "stats must be 16-byte aligned");
  NormArgs a{};
  fill(a, norm, x, residual, params, param_strides, scale_bias, pre_scale_bias, residual_scale, eps, B, L, D);
  a.y = y; a.z = z; a.stats = reinterpret_cast<float4*>(stats);
  const bool vec = D % 4 == 0 && aligned16(x) && aligned16(residual) && aligned16(y) && aligned16(z) &&
                   params_aligned(params);
  return dispatch_fwd(x_dtype, y_dtype, form, a, vec, (cudaStream_t)stream);
}

extern "C" int64_t fa_block_norm_workspace(int form, const int64_t param_strides[6], int64_t B, int64_t L, int64_t D) {
  if (form < kBefore || form > kBetween || !param_strides || B < 0 || L < 0 || D < 1 || D > kMaxDim ||
      B >= ((int64_t)1 << 31) || (L > 0 && B > (((int64_t)1 << 60) / kMaxDim) / L))
    return set_error(FA_ERR_INVALID, "invalid block norm shape");
  const BwdShape s = bwd_shape(param_strides, B, L, D);
  return s.B * s.blocks * sums_of(form) * D * 4;
}

extern "C" int fa_block_norm_backward(int form, int norm, const void* x, int x_dtype, const void* residual,
                                      int y_dtype, const float* const params[6], const int64_t param_strides[6],
                                      float scale_bias, float pre_scale_bias, float residual_scale, float eps,
                                      const void* dy, const void* dz, const float* stats, void* dx, void* dresidual,
                                      float* const dparams[6], int64_t B, int64_t L, int64_t D, void* workspace,
                                      int64_t workspace_bytes, void* stream) {
  const int rc = check_args(form, norm, x, x_dtype, residual, y_dtype, params, param_strides, B, L, D);
  if (rc != FA_OK) return rc;
  FA_REQUIRE(dparams, FA_ERR_INVALID, "null gradient array");
  FA_REQUIRE(B * L == 0 || (stats && aligned16(stats)), FA_ERR_INVALID, "stats must be given, 16-byte aligned");
  const int64_t need = fa_block_norm_workspace(form, param_strides, B, L, D);
  FA_REQUIRE(need == 0 || (workspace && workspace_bytes >= need), FA_ERR_INVALID, "workspace too small");
  cudaStream_t s = (cudaStream_t)stream;
  const BwdShape sh = bwd_shape(param_strides, B, L, D);
  if (B == 0) {
    // No batch element: per-batch gradients are empty, shared ones are zero.
    for (int i = 0; i < kParams; ++i)
      if (dparams[i] && param_strides[i] == 0) FA_CUDA(cudaMemsetAsync(dparams[i], 0, (size_t)D * 4, s));
    return FA_OK;
  }
  NormArgs a{};
  fill(a, norm, x, residual, params, param_strides, scale_bias, pre_scale_bias, residual_scale, eps, B, L, D);
  a.dy = dy; a.dz = dz; a.dx = dx; a.dr = dresidual;
  a.stats = const_cast<float4*>(reinterpret_cast<const float4*>(stats));
  a.ws = reinterpret_cast<float*>(workspace);
  a.tpr = sh.tpr;
  const bool vec = D % 4 == 0 && aligned16(x) && aligned16(residual) && aligned16(dy) && aligned16(dz) &&
                   aligned16(dx) && aligned16(dresidual) && params_aligned(params);
  const int rc2 = dispatch_bwd(x_dtype, y_dtype, form, a, sh, vec, s);
  if (rc2 != FA_OK) return rc2;
  SumArgs m{};
  m.ws = a.ws;
  m.first = form == kBefore ? kPreScale : kPostScale;
  m.sums = sums_of(form); m.blocks = (int)sh.blocks; m.B = (int)sh.B; m.D = (int)D;
  bool any = false, own = false;
  for (int i = 0; i < kParams; ++i) {
    m.out[i] = i >= m.first && i < m.first + m.sums ? dparams[i] : nullptr;
    m.per_batch[i] = param_strides[i] != 0;
    any = any || m.out[i];
    own = own || (m.out[i] && m.per_batch[i]);
  }
  if (!any) return FA_OK;
  const unsigned gy = own ? (unsigned)(sh.B < 65535 ? sh.B : 65535) : 1u;
  block_norm_sum_kernel<<<dim3((unsigned)ceil_div(D, 32), gy, (unsigned)m.sums), dim3(32, kSumRows), 0, s>>>(m);
  return check_launch("block_norm_sum_kernel");
}
