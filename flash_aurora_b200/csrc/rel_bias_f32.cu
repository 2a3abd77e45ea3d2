// fp32 window attention with a learned relative position bias, forward and backward, on warp-level
// tensor-core products (m16n8k8, 3xTF32). The formulas are in rel_bias.cu.
//
// Every operand is split as x = hi + lo, both tf32; a product accumulates lo hi + hi lo + hi hi in
// fp32, so it is good to about 2^-22 of its terms and the result is an fp32 one, as fp32 gradients need.
// The 5th-generation path is not used here: kind::tf32 takes K-major operands only, and the backward
// pass would have to transpose, split and store five operands a tile; at three products a term both
// paths are bound by their products, not by memory.
//
// A block holds a tile's operands in shared memory (144 rows of 68 floats: every fragment read hits 32
// banks at a constant offset from one lane address) and each of its 9 warps owns 16 rows.
//   forward   S, online softmax, O.
//   backward  queries by rows: S, dP, delta, dS, dQ and the bias gradient (one partial per block and head in
//             global memory, read and written in fragment order); keys by rows: S^T and dP^T again, from which
//             P^T and dS^T are at hand as A operands of dV = P^T dO and dK = dS^T Q. The two products computed
//             again cost 2 of 7 and save 83 KB of shared memory for P and dS, and all exchange between warps
//             but delta.
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

constexpr int kThreads = 32 * kMaxN / 16;
constexpr int kLd = 68;            // floats per row: fragment reads, 4 or 8 rows apart, hit 32 banks
constexpr int kTile = kMaxN * kLd;  // floats

// Rows 0..N-1 of a (token, 64) operand into shared memory.
__device__ __forceinline__ void load_tile(float* dst, const void* src, const int64_t* st, int w, int h, int N) {
  const float* base = reinterpret_cast<const float*>(src) + w * st[0] + h * st[1];
  for (int e = threadIdx.x; e < N * 16; e += kThreads) {
    const int row = e >> 4, c = e & 15;
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_u32(dst + row * kLd + c * 4)),
                 "l"(base + row * st[2] + c * 4)
                 : "memory");
  }
}
__device__ __forceinline__ void wait_loads() { asm volatile("cp.async.wait_all;" ::: "memory"); }

// x = hi + lo with hi rounded to tf32 (half away from zero) by integer arithmetic: the cvt that rounds to
// tf32 issues at a quarter of this rate and bound these kernels. lo gets half a step added, since the tensor
// core drops the bits that tf32 lacks.
__device__ __forceinline__ void split(float x, uint32_t& hi, uint32_t& lo) {
  hi = (__float_as_uint(x) + 0x1000u) & 0xffffe000u;
  lo = __float_as_uint(x - __uint_as_float(hi)) + 0x1000u;
}

// A 16 x 8 A operand, split.
struct FragA {
  uint32_t h[4], l[4];
  // Rows g and g + 8, columns q and q + 4 of the 16 x 8 block whose element (g, q) is at t.
  __device__ __forceinline__ void load(const float* t) {
    split(t[0], h[0], l[0]);
    split(t[8 * kLd], h[1], l[1]);
    split(t[4], h[2], l[2]);
    split(t[8 * kLd + 4], h[3], l[3]);
  }
  // An accumulator block (16 rows x 8) as the operand: its columns in the order 0, 2, 4, 6, 1, 3, 5, 7, which
  // acc_by_cols() follows.
  __device__ __forceinline__ void take(const float (&c)[4]) {
    split(c[0], h[0], l[0]);
    split(c[2], h[1], l[1]);
    split(c[1], h[2], l[2]);
    split(c[3], h[3], l[3]);
  }
};

// d = a b + c. Not volatile: the compiler interleaves independent products, whose latency is 24 cycles.
__device__ __forceinline__ void mma_tf32(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1, float c0, float c1,
                                         float c2, float c3) {
  asm("mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %11, %12, %13};"
      : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(c0), "f"(c1), "f"(c2), "f"(c3));
}

// c += a b, 8 columns deep. The three products are summed from zero and added to c in fp32: the tensor core
// truncates its accumulator at every product, which over the 24 products of a 64-long sum left errors of 1e-6.
__device__ __forceinline__ void mma3(float (&c)[4], const FragA& a, float b0, float b1) {
  uint32_t h0, l0, h1, l1;
  split(b0, h0, l0);
  split(b1, h1, l1);
  float d[4];
  mma_tf32(d, a.l, h0, h1, 0.f, 0.f, 0.f, 0.f);
  mma_tf32(d, a.h, l0, l1, d[0], d[1], d[2], d[3]);
  mma_tf32(d, a.h, h0, h1, d[0], d[1], d[2], d[3]);
#pragma unroll
  for (int e = 0; e < 4; ++e) c[e] += d[e];
}

// c (16 x 8 kJ) = x y^T over 64 columns; x: element (g, q) of the 16 rows, y: of the first of the 8 kJ rows.
template <int kJ>
__device__ __forceinline__ void rows_by_rows(float (&c)[kJ][4], const float* x, const float* y) {
#pragma unroll
  for (int j = 0; j < kJ; ++j) c[j][0] = c[j][1] = c[j][2] = c[j][3] = 0.f;
#pragma unroll 2
  for (int k = 0; k < 8; ++k) {
    FragA a;
    a.load(x + 8 * k);
#pragma unroll
    for (int j = 0; j < kJ; ++j) mma3(c[j], a, y[8 * j * kLd + 8 * k], y[8 * j * kLd + 8 * k + 4]);
  }
}

// o (16 x 64) += c (16 x 8 kJ, an accumulator) times 8 kJ rows of 64; y: element (2 q, g) of the first.
template <int kJ>
__device__ __forceinline__ void acc_by_cols(float (&o)[8][4], const float (&c)[kJ][4], const float* y) {
#pragma unroll
  for (int j = 0; j < kJ; ++j) {
    FragA a;
    a.take(c[j]);
#pragma unroll
    for (int d = 0; d < 8; ++d) mma3(o[d], a, y[8 * j * kLd + 8 * d], y[(8 * j + 1) * kLd + 8 * d]);
  }
}

// The mask of a tile: whether (query, key) is masked.
template <int kMask>
struct Mask {
  const uint8_t* m;
  int N;
  __device__ __forceinline__ Mask(const Params& p, int w) : N(p.N) {
    const int64_t mw = w % p.nW;
    m = kMask == kGroups ? p.mask + mw * N : kMask == kMaskU8 ? p.mask + mw * N * N : nullptr;
  }
  __device__ __forceinline__ float add(int i, int j) const {
    if (kMask == kNoMask || i >= N || j >= N) return 0.f;
    const bool off = kMask == kGroups ? __ldg(m + i) != __ldg(m + j) : __ldg(m + i * N + j) != 0;
    return off ? kMaskedLog2 : 0.f;
  }
};

// Logits (log2 domain) of an accumulator of rows r0 + g, + 8 and columns n0 + 8 j + 2 q, + 1, from the raw
// products and a bias in fragment order. kT: rows are keys.
template <int kMask, bool kT, int kJ>
__device__ __forceinline__ void logits(float (&c)[kJ][4], const float4* bias, float scale, const Mask<kMask>& mask, int r0,
                                       int n0, int g, int q) {
#pragma unroll
  for (int j = 0; j < kJ; ++j) {
    const float4 b = __ldg(bias + (n0 / 8 + j) * 32);
    const float bb[4] = {b.x, b.y, b.z, b.w};
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      c[j][e] = fmaf(c[j][e], scale, bb[e]);
      if (kMask != kNoMask) {
        const int r = r0 + g + 8 * (e >> 1), n = n0 + 8 * j + 2 * q + (e & 1);
        c[j][e] += kT ? mask.add(n, r) : mask.add(r, n);
      }
    }
  }
}

__device__ __forceinline__ float quad_max(float v) {
  v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 1));
  return fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 2));
}
__device__ __forceinline__ float quad_sum(float v) {
  v += __shfl_xor_sync(0xffffffffu, v, 1);
  return v + __shfl_xor_sync(0xffffffffu, v, 2);
}

// Rows r0 + g and r0 + g + 8 of a 16 x 64 accumulator, scaled, to global memory.
__device__ __forceinline__ void store_rows(void* dst, const int64_t* st, int w, int h, int N, int r0, int g, int q,
                                           const float (&o)[8][4], float sa, float sb) {
  float* base = reinterpret_cast<float*>(dst) + w * st[0] + h * st[1] + 2 * q;
#pragma unroll
  for (int hi = 0; hi < 2; ++hi) {
    const int r = r0 + g + 8 * hi;
    if (r >= N) continue;
    const float s = hi ? sb : sa;
#pragma unroll
    for (int d = 0; d < 8; ++d)
      *reinterpret_cast<float2*>(base + r * st[2] + 8 * d) = make_float2(o[d][2 * hi] * s, o[d][2 * hi + 1] * s);
  }
}

constexpr int kFwdSmem = 3 * kTile * 4;
constexpr int kChunk = 6;  // 8-key blocks at a time

template <int kMask>
__global__ void __launch_bounds__(kThreads, 1) rel_bias_fwd_f32_kernel(const Params p) {
  extern __shared__ __align__(16) float sm[];
  float *sQ = sm, *sK = sm + kTile, *sV = sm + 2 * kTile;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, q = lane & 3, r0 = 16 * warp;
  const int rc = g * kLd + q, cr = 2 * q * kLd + g;  // lane offsets of the two kinds of fragment
  for (int e = threadIdx.x; e < 3 * kTile; e += kThreads) sm[e] = 0.f;  // rows past N stay zero
  __syncthreads();
  const int t_end = tile_end(p.num_tiles);
  for (int t = tile_begin(p.num_tiles); t < t_end; ++t) {
    const int h = t / p.Bwin, w = t - h * p.Bwin;
    load_tile(sQ, p.q, p.sq, w, h, p.N);
    load_tile(sK, p.k, p.sk, w, h, p.N);
    load_tile(sV, p.v, p.sv, w, h, p.N);
    wait_loads();
    __syncthreads();
    if (r0 < p.N) {
      const float4* bias = bias_rows(p, h, r0, lane);
      const Mask<kMask> mask(p, w);
      float o[8][4];
#pragma unroll
      for (int d = 0; d < 8; ++d) o[d][0] = o[d][1] = o[d][2] = o[d][3] = 0.f;
      float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
#pragma unroll 1
      for (int n0 = 0; n0 < p.N; n0 += 8 * kChunk) {
        float c[kChunk][4];
        rows_by_rows<kChunk>(c, sQ + r0 * kLd + rc, sK + n0 * kLd + rc);
        logits<kMask, false, kChunk>(c, bias, p.scale_log2, mask, r0, n0, g, q);
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          float mx = m[i];
#pragma unroll
          for (int j = 0; j < kChunk; ++j) mx = fmax3(mx, c[j][2 * i], c[j][2 * i + 1]);
          mx = quad_max(mx);
          // A row without a finite logit so far keeps zero sums (no inf - inf).
          const float f = m[i] == -INFINITY ? 0.f : exp2f(m[i] - mx), base = mx == -INFINITY ? 0.f : mx;
          m[i] = mx;
          l[i] *= f;
#pragma unroll
          for (int d = 0; d < 8; ++d) {
            o[d][2 * i] *= f;
            o[d][2 * i + 1] *= f;
          }
#pragma unroll
          for (int j = 0; j < kChunk; ++j) {
            c[j][2 * i] = exp2f(c[j][2 * i] - base);
            c[j][2 * i + 1] = exp2f(c[j][2 * i + 1] - base);
            l[i] += c[j][2 * i] + c[j][2 * i + 1];
          }
        }
        acc_by_cols<kChunk>(o, c, sV + n0 * kLd + cr);
      }
      const float la = quad_sum(l[0]), lb = quad_sum(l[1]);
      store_rows(p.out, p.so, w, h, p.N, r0, g, q, o, 1.f / la, 1.f / lb);
      if (p.stats && q == 0) {
        float2* st = p.stats + ((int64_t)w * p.H + h) * kMaxN + r0 + g;
        st[0] = make_float2(m[0], log2f(la));
        st[8] = make_float2(m[1], log2f(lb));
      }
    }
    __syncthreads();
  }
}

// ... + per query: -(row maximum), -(log2 of the row sum), delta
constexpr int kBwdSmem = (4 * kTile + 3 * kMaxN) * 4;

template <int kMask>
__global__ void __launch_bounds__(kThreads, 1) rel_bias_bwd_f32_kernel(const Params p) {
  extern __shared__ __align__(16) float sm[];
  float *sQ = sm, *sK = sm + kTile, *sV = sm + 2 * kTile, *sG = sm + 3 * kTile;
  float *sMax = sm + 4 * kTile, *sLog = sMax + kMaxN, *sDelta = sLog + kMaxN;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, q = lane & 3, r0 = 16 * warp;
  const int rc = g * kLd + q, cr = 2 * q * kLd + g;  // lane offsets of the two kinds of fragment
  for (int e = threadIdx.x; e < 4 * kTile; e += kThreads) sm[e] = 0.f;  // rows past N stay zero
  __syncthreads();
  const int t_begin = tile_begin(p.num_tiles), t_end = tile_end(p.num_tiles);
  for (int t = t_begin; t < t_end; ++t) {
    const int h = t / p.Bwin, w = t - h * p.Bwin;
    load_tile(sQ, p.q, p.sq, w, h, p.N);
    load_tile(sK, p.k, p.sk, w, h, p.N);
    load_tile(sV, p.v, p.sv, w, h, p.N);
    load_tile(sG, p.dout, p.so, w, h, p.N);
    if (threadIdx.x < kMaxN) {  // rows past N: P = 0
      const float2 st = threadIdx.x < p.N ? __ldg(p.stats + ((int64_t)w * p.H + h) * kMaxN + threadIdx.x)
                                          : make_float2(INFINITY, 0.f);
      sMax[threadIdx.x] = -st.x;
      sLog[threadIdx.x] = -st.y;
    }
    wait_loads();
    __syncthreads();
    const Mask<kMask> mask(p, w);
    if (r0 < p.N) {
      // Queries by rows.
      float c[18][4], d[18][4];
      rows_by_rows<18>(c, sQ + r0 * kLd + rc, sK + rc);
      logits<kMask, false, 18>(c, bias_rows(p, h, r0, lane), p.scale_log2, mask, r0, 0, g, q);
      rows_by_rows<18>(d, sG + r0 * kLd + rc, sV + rc);
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const float mx = sMax[r0 + g + 8 * i], lg = sLog[r0 + g + 8 * i];
        float delta = 0.f;
#pragma unroll
        for (int j = 0; j < 18; ++j)
#pragma unroll
          for (int e = 2 * i; e < 2 * i + 2; ++e) {
            c[j][e] = exp2f(c[j][e] + mx + lg);
            delta = fmaf(c[j][e], d[j][e], delta);
          }
        delta = quad_sum(delta);
        if (q == 0) sDelta[r0 + g + 8 * i] = delta;
#pragma unroll
        for (int j = 0; j < 18; ++j)
#pragma unroll
          for (int e = 2 * i; e < 2 * i + 2; ++e) c[j][e] *= d[j][e] - delta;  // dS
      }
      if (p.slots) {
        float4* slot = slot_rows(p, blockIdx.x + h, r0, lane);
        const bool first = t == t_begin || w == 0;  // of this head in this block
#pragma unroll
        for (int j = 0; j < 18; ++j) {
          float4 s = first ? make_float4(0.f, 0.f, 0.f, 0.f) : slot[j * 32];
          s.x += c[j][0];
          s.y += c[j][1];
          s.z += c[j][2];
          s.w += c[j][3];
          slot[j * 32] = s;
        }
      }
      float o[8][4];
#pragma unroll
      for (int e = 0; e < 8; ++e) o[e][0] = o[e][1] = o[e][2] = o[e][3] = 0.f;
      acc_by_cols<18>(o, c, sK + cr);
      store_rows(p.dq, p.sdq, w, h, p.N, r0, g, q, o, p.scale, p.scale);
    }
    __syncthreads();
    if (r0 < p.N) {
      // Keys by rows.
      float gv[8][4], gk[8][4];
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        gv[e][0] = gv[e][1] = gv[e][2] = gv[e][3] = 0.f;
        gk[e][0] = gk[e][1] = gk[e][2] = gk[e][3] = 0.f;
      }
      const float4* bias = bias_rows(p, p.H + h, r0, lane);
#pragma unroll 1
      for (int n0 = 0; n0 < p.N; n0 += 8 * kChunk) {
        float c[kChunk][4], d[kChunk][4];
        rows_by_rows<kChunk>(c, sK + r0 * kLd + rc, sQ + n0 * kLd + rc);
        logits<kMask, true, kChunk>(c, bias, p.scale_log2, mask, r0, n0, g, q);
        rows_by_rows<kChunk>(d, sV + r0 * kLd + rc, sG + n0 * kLd + rc);
#pragma unroll
        for (int j = 0; j < kChunk; ++j)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const int n = n0 + 8 * j + 2 * q + e;  // queries past N: sMax is -inf, so P = dS = 0
            const float mxn = sMax[n], lgn = sLog[n], dln = n < p.N ? sDelta[n] : 0.f;
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              const float pr = exp2f(c[j][2 * i + e] + mxn + lgn);
              c[j][2 * i + e] = pr;
              d[j][2 * i + e] = pr * (d[j][2 * i + e] - dln);
            }
          }
        acc_by_cols<kChunk>(gv, c, sG + n0 * kLd + cr);
        acc_by_cols<kChunk>(gk, d, sQ + n0 * kLd + cr);
      }
      store_rows(p.dv, p.sdv, w, h, p.N, r0, g, q, gv, 1.f, 1.f);
      store_rows(p.dk, p.sdk, w, h, p.N, r0, g, q, gk, p.scale, p.scale);
    }
    __syncthreads();
  }
}

template <int kMask>
int launch_fwd(const Params& p, cudaStream_t s) {
  auto kern = rel_bias_fwd_f32_kernel<kMask>;
  FA_CUDA(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, kFwdSmem));
  const int grid = p.num_tiles < num_sms() ? p.num_tiles : num_sms();
  kern<<<grid, kThreads, kFwdSmem, s>>>(p);
  return check_launch("rel_bias_fwd_f32_kernel");
}

template <int kMask>
int launch_bwd(const Params& p, int grid, cudaStream_t s) {
  auto kern = rel_bias_bwd_f32_kernel<kMask>;
  FA_CUDA(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, kBwdSmem));
  kern<<<grid, kThreads, kBwdSmem, s>>>(p);
  return check_launch("rel_bias_bwd_f32_kernel");
}

}  // namespace

int run_f32_forward(const Params& p, int mask_kind, cudaStream_t s) {
  if (mask_kind == kMaskU8) return launch_fwd<kMaskU8>(p, s);
  if (mask_kind == kGroups) return launch_fwd<kGroups>(p, s);
  return launch_fwd<kNoMask>(p, s);
}

int run_f32_backward(const Params& p, int mask_kind, int grid, cudaStream_t s) {
  if (mask_kind == kMaskU8) return launch_bwd<kMaskU8>(p, grid, s);
  if (mask_kind == kGroups) return launch_bwd<kGroups>(p, grid, s);
  return launch_bwd<kNoMask>(p, grid, s);
}

}  // namespace relb
}  // namespace fa
