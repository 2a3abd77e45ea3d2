// fp32 window attention with a learned relative position bias, forward and backward, on warp-level
// tensor-core products (m16n8k16). The formulas are in rel_bias.cu.
//
// Every operand is a pair of halves: x 2^-e = hi + lo, with a power of two of its row that brings the row's largest
// finite magnitude to [2^14, 2^15). The pair holds 22 bits of every element down to 2^-18 of that magnitude, and
// below it 2^-40 of the magnitude; an infinity or NaN makes NaNs of the sums that it enters and of no others. A
// product is lo hi + hi lo + hi hi, summed in fp32, so it is good to about 2^-22 of its terms, as 3xTF32 is, at
// half the instructions (16 deep instead of 8). Scales of rows that are summed over (V in P V, K in dS K, Q and dO
// in the keys' sums) join the other operand, which lies in registers, before it is scaled and split itself: a row of
// any size, in a masked place for instance, costs the others nothing.
// Each group of three products is summed from zero and added in fp32: kept in the tensor core's accumulator,
// which truncates at every product, the sums had errors of 1e-6 where these kernels are at 1.7e-7 (forward) and
// 2.5e-7 (gradients) of the outputs' norm. That is why these are not UMMAs, whose accumulators stay in TMEM: every
// group would go through registers, or keep the truncated sums.
//
// A block scales and splits its tile's operands once, into shared memory (16-byte chunks permuted by row, so that
// the fragments' loads, plain and transposed, hit all banks once); each of its 9 warps owns 16 rows.
//   forward   S, online softmax, O.
//   backward  queries by rows: S, dP, delta, dS, dQ and the bias gradient (one partial per block and head in
//             global memory, read and written in fragment order); keys by rows: S^T and dP^T again, from which
//             P^T and dS^T are at hand as A operands of dV = P^T dO and dK = dS^T Q. The two products computed
//             again cost 2 of 7 and save 166 KB of shared memory for the pairs of P and dS, and all exchange between
//             warps but delta.
// 1024 tiles of 144 tokens take 120 us forward (two blocks an SM; 40 % of issue slots) and 300 us backward (one;
// 32 %), against 23 / 41 us of memory traffic and about 33 / 115 us of products: what bounds them is the latency of
// dependent instructions with the 9 or 18 warps that registers and shared memory allow.
#include <cuda_fp16.h>

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
constexpr uint32_t kPart = kMaxN * 128;   // bytes of an operand's high (or low) parts: 144 rows of 64 halves
constexpr uint32_t kOperand = 2 * kPart;

// x, y = hi + lo.
__device__ __forceinline__ void split2(float x, float y, uint32_t& hi, uint32_t& lo) {
  const __half2 h = __floats2half2_rn(x, y);
  const float2 f = __half22float2(h);
  const __half2 l = __floats2half2_rn(x - f.x, y - f.y);
  hi = *reinterpret_cast<const uint32_t*>(&h);
  lo = *reinterpret_cast<const uint32_t*>(&l);
}

// The powers of two that bring a row of largest magnitude m into fp16's upper range, [2^14, 2^15), and back.
// Rows below 2^-112 are scaled as if they reached it (both powers stay normal numbers).
struct Scale {
  float up, down;
  __device__ __forceinline__ explicit Scale(float m) {
    const uint32_t e = max(__float_as_uint(m) >> 23, 15u);
    up = __uint_as_float((268u - e) << 23);
    down = __uint_as_float((e - 14u) << 23);
  }
};

__device__ __forceinline__ float quad_max(float v) {
  v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 1));
  return fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 2));
}
__device__ __forceinline__ float quad_sum(float v) {
  v += __shfl_xor_sync(0xffffffffu, v, 1);
  return v + __shfl_xor_sync(0xffffffffu, v, 2);
}

// A thread's share of a (token, 64) operand: 16 columns of two rows, a row in four lanes. The rows of a half
// warp are 2 apart, so that its 8-byte stores hit all banks once.
struct Share {
  static constexpr int kRows = 8 * (kThreads / 32);  // of the block at a time; two times kRows = kMaxN
  float4 x[2][4];
  __device__ __forceinline__ static int row(int i) {
    const int lane = threadIdx.x & 31;
    return i * kRows + 8 * (threadIdx.x >> 5) + 2 * ((lane >> 2) & 3) + (lane >> 4);
  }
  __device__ __forceinline__ void fetch(const void* src, const int64_t* st, int w, int h, int N) {
    const float* base = reinterpret_cast<const float*>(src) + w * st[0] + h * st[1] + 4 * (threadIdx.x & 3);
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int c = 0; c < 4; ++c)
        x[i][c] = row(i) < N ? __ldg(reinterpret_cast<const float4*>(base + row(i) * st[2] + 16 * c))
                             : make_float4(0.f, 0.f, 0.f, 0.f);
  }
  // The largest finite magnitude. An infinity must not set its row's scale: it would make zeros of the row's other
  // columns, which a product over rows (P V, P^T dO) sums apart from it.
  __device__ __forceinline__ static float finite_max(const float4 (&v)[4]) {
    float m = 0.f;
#pragma unroll
    for (int c = 0; c < 4; ++c)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float a = fabsf(e == 0 ? v[c].x : e == 1 ? v[c].y : e == 2 ? v[c].z : v[c].w);
        m = fmaxf(m, a == INFINITY ? 0.f : a);  // a NaN is passed over
      }
    return m;
  }
  // Into shared memory, scaled and split; 16-byte chunk c of row r lies at c ^ (r & 7). Rows past N: zeros.
  __device__ __forceinline__ void put(uint32_t dst, float* down) const {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      float m = 0.f;
#pragma unroll
      for (int c = 0; c < 4; ++c)
        m = fmaxf(m, fmaxf(fmaxf(fabsf(x[i][c].x), fabsf(x[i][c].y)), fmaxf(fabsf(x[i][c].z), fabsf(x[i][c].w))));
      m = quad_max(m);
      if (__any_sync(0xffffffffu, m == INFINITY)) m = quad_max(finite_max(x[i]));  // rare
      const Scale s(m);
      const int r = row(i), part = threadIdx.x & 3;
      if (part == 0) down[r] = s.down;
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        uint32_t h0, l0, h1, l1;
        split2(x[i][c].x * s.up, x[i][c].y * s.up, h0, l0);
        split2(x[i][c].z * s.up, x[i][c].w * s.up, h1, l1);
        const uint32_t at = dst + r * 128 + ((((part >> 1) + 2 * c) ^ (r & 7)) << 4) + (part & 1) * 8;
        asm volatile("st.shared.v2.u32 [%0], {%1, %2};" ::"r"(at), "r"(h0), "r"(h1) : "memory");
        asm volatile("st.shared.v2.u32 [%0], {%1, %2};" ::"r"(at + kPart), "r"(l0), "r"(l1) : "memory");
      }
    }
  }
};

// A lane's part in the addresses of fragments: of rows as the A operand, of rows as the B operand of a product
// over columns, and of a product over rows (transposed). The 8 x 8 matrices of an x4 load are, in this order,
//   a     rows 0-7 and 8-15 of the first 8 columns, then of the next 8
//   b     columns 0-7 and 8-15 of 8 rows, high parts, then low parts
//   t     rows 0-7 and 8-15 of 8 columns, high parts, then low parts
struct Lanes {
  uint32_t a, b, t, xa, xb, xt;
  __device__ __forceinline__ Lanes() {
    const uint32_t lane = threadIdx.x & 31, m = lane >> 3, r = lane & 7;
    a = (8 * (m & 1) + r) * 128;
    b = (m >> 1) * kPart + r * 128;
    t = (m >> 1) * kPart + a;
    xa = ((m >> 1) ^ r) << 4;
    xb = ((m & 1) ^ r) << 4;
    xt = r << 4;
  }
};

__device__ __forceinline__ void ldmatrix4(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ void ldmatrix4_trans(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}

// A 16 x 16 A operand.
struct FragA {
  uint32_t h[4], l[4];
  // Two adjacent accumulator blocks (16 rows x 8 each), rows g and g + 8 scaled.
  __device__ __forceinline__ void take(const float (&x)[4], const float (&y)[4], float ua, float ub) {
    split2(x[0] * ua, x[1] * ua, h[0], l[0]);
    split2(x[2] * ub, x[3] * ub, h[1], l[1]);
    split2(y[0] * ua, y[1] * ua, h[2], l[2]);
    split2(y[2] * ub, y[3] * ub, h[3], l[3]);
  }
};

// d = a b + c. Not volatile: the compiler interleaves independent products, whose latency is 24 cycles.
__device__ __forceinline__ void mma_f16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1, float c0, float c1,
                                        float c2, float c3) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %11, %12, %13};"
      : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(c0), "f"(c1), "f"(c2), "f"(c3));
}

// d = a b, 16 deep, b: high parts, low parts. Summed from zero, for the caller to add in fp32: the tensor core
// truncates its accumulator at every product, which over all the products of a sum left errors of 1e-6.
__device__ __forceinline__ void mma3(float (&d)[4], const FragA& a, const uint32_t (&b)[4]) {
  mma_f16(d, a.l, b[0], b[1], 0.f, 0.f, 0.f, 0.f);
  mma_f16(d, a.h, b[2], b[3], d[0], d[1], d[2], d[3]);
  mma_f16(d, a.h, b[0], b[1], d[0], d[1], d[2], d[3]);
}

// c (16 x 8 kJ) = x y^T over 64 columns, scales left out; x: of the first of 16 rows, y: of the first of 8 kJ.
template <int kJ>
__device__ __forceinline__ void rows_by_rows(float (&c)[kJ][4], uint32_t x, uint32_t y, const Lanes& L) {
#pragma unroll
  for (int j = 0; j < kJ; ++j) c[j][0] = c[j][1] = c[j][2] = c[j][3] = 0.f;
#pragma unroll 1
  for (int k = 0; k < 4; ++k) {
    FragA a;
    ldmatrix4(a.h, x + L.a + ((32 * k) ^ L.xa));
    ldmatrix4(a.l, x + L.a + ((32 * k) ^ L.xa) + kPart);
#pragma unroll
    for (int j = 0; j < kJ; ++j) {
      uint32_t b[4];
      float d[4];
      ldmatrix4(b, y + L.b + ((32 * k) ^ L.xb) + 1024 * j);
      mma3(d, a, b);
#pragma unroll
      for (int e = 0; e < 4; ++e) c[j][e] += d[e];
    }
  }
}

// o (16 x 64) += c (16 x 8 kJ, an accumulator) times 8 kJ rows of 64 whose scales down[] are; y: of the first row.
// The scales join c, whose rows are then scaled themselves.
template <int kJ>
__device__ __forceinline__ void acc_by_cols(float (&o)[8][4], const float (&c)[kJ][4], uint32_t y, const float* down, const Lanes& L) {
  float u[kJ][4], m[2] = {0.f, 0.f};
#pragma unroll
  for (int j = 0; j < kJ; ++j) {
    const float2 s = *reinterpret_cast<const float2*>(down + 8 * j);
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      u[j][2 * i] = c[j][2 * i] * s.x;
      u[j][2 * i + 1] = c[j][2 * i + 1] * s.y;
      m[i] = fmax3(m[i], fabsf(u[j][2 * i]), fabsf(u[j][2 * i + 1]));
    }
  }
  const Scale sa(quad_max(m[0])), sb(quad_max(m[1]));
#pragma unroll
  for (int j = 0; j < kJ; j += 2) {
    FragA a;
    a.take(u[j], u[j + 1], sa.up, sb.up);
#pragma unroll
    for (int d = 0; d < 8; ++d) {
      uint32_t b[4];
      float t[4];
      ldmatrix4_trans(b, y + L.t + ((16 * d) ^ L.xt) + 1024 * j);
      mma3(t, a, b);
      o[d][0] = fmaf(t[0], sa.down, o[d][0]);
      o[d][1] = fmaf(t[1], sa.down, o[d][1]);
      o[d][2] = fmaf(t[2], sb.down, o[d][2]);
      o[d][3] = fmaf(t[3], sb.down, o[d][3]);
    }
  }
}

// The mask of a tile, as what it adds to a logit; id: region ids in shared memory, rows past N alike.
template <int kMask>
struct Mask {
  const uint8_t* m;
  const int* id;
  int N;
  __device__ __forceinline__ Mask(const Params& p, int w, const int* ids)
      : m(kMask == kMaskU8 ? p.mask + (w % p.nW) * (int64_t)p.N * p.N : nullptr), id(ids), N(p.N) {}
  __device__ __forceinline__ float add(int i, int j) const {  // kMaskU8
    return i < N && j < N && __ldg(m + i * N + j) != 0 ? kMaskedLog2 : 0.f;
  }
};
template <int kMask>
__device__ __forceinline__ void load_ids(const Params& p, int w, int* ids) {
  if (kMask == kGroups && threadIdx.x < kMaxN)
    ids[threadIdx.x] = threadIdx.x < p.N ? __ldg(p.mask + (w % p.nW) * (int64_t)p.N + threadIdx.x) : 0;
}

// Logits (log2 domain) of an accumulator of rows r0 + g, + 8 and columns n0 + 8 j + 2 q, + 1, from the raw
// products, the scales of the rows (times the logit scale) and of the columns, and a bias in fragment order.
// kT: rows are keys.
template <int kMask, bool kT, int kJ>
__device__ __forceinline__ void logits(float (&c)[kJ][4], const float4* bias, float ra, float rb, const float* down,
                                       const Mask<kMask>& mask, int r0, int n0, int g, int q) {
  int ia = 0, ib = 0;
  if (kMask == kGroups) {
    ia = mask.id[r0 + g];
    ib = mask.id[r0 + g + 8];
  }
#pragma unroll
  for (int j = 0; j < kJ; ++j) {
    const float4 b = __ldg(bias + (n0 / 8 + j) * 32);
    const int n = n0 + 8 * j + 2 * q;
    const float2 s = *reinterpret_cast<const float2*>(down + n);
    c[j][0] = fmaf(c[j][0] * s.x, ra, b.x);
    c[j][1] = fmaf(c[j][1] * s.y, ra, b.y);
    c[j][2] = fmaf(c[j][2] * s.x, rb, b.z);
    c[j][3] = fmaf(c[j][3] * s.y, rb, b.w);
    if (kMask == kGroups) {
      const int2 in = *reinterpret_cast<const int2*>(mask.id + n);
      if (ia != in.x) c[j][0] += kMaskedLog2;
      if (ia != in.y) c[j][1] += kMaskedLog2;
      if (ib != in.x) c[j][2] += kMaskedLog2;
      if (ib != in.y) c[j][3] += kMaskedLog2;
    }
    if (kMask == kMaskU8) {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int r = r0 + g + 8 * (e >> 1);
        c[j][e] += kT ? mask.add(n + (e & 1), r) : mask.add(r, n + (e & 1));
      }
    }
  }
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

constexpr int kChunk = 6;  // 8-key blocks at a time
static_assert(kMaxN % (8 * kChunk) == 0 && kChunk % 2 == 0);

// Q, K, V; their rows' scales and the region ids. Two blocks an SM: one's loads and softmax under the other's products.
constexpr int kFwdSmem = 3 * kOperand + 4 * kMaxN * 4;
static_assert(2 * (kFwdSmem + 1024) <= 228 * 1024, "two blocks an SM");

template <int kMask>
__global__ void __launch_bounds__(kThreads, 2) rel_bias_fwd_f32_kernel(const Params p) {
  extern __shared__ __align__(128) uint8_t sm[];
  const uint32_t sQ = smem_u32(sm), sK = sQ + kOperand, sV = sK + kOperand;
  float *dQ = reinterpret_cast<float*>(sm + 3 * kOperand), *dK = dQ + kMaxN, *dV = dK + kMaxN;
  int* ids = reinterpret_cast<int*>(dV + kMaxN);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, q = lane & 3, r0 = 16 * warp;
  const Lanes L;
  const int t_end = tile_end(p.num_tiles);
  for (int t = tile_begin(p.num_tiles); t < t_end; ++t) {
    const int h = t / p.Bwin, w = t - h * p.Bwin;
    {
      Share a, b;
      a.fetch(p.q, p.sq, w, h, p.N);
      b.fetch(p.k, p.sk, w, h, p.N);
      load_ids<kMask>(p, w, ids);
      a.put(sQ, dQ);
      b.put(sK, dK);
      a.fetch(p.v, p.sv, w, h, p.N);
      a.put(sV, dV);
    }
    __syncthreads();
    if (r0 < p.N) {
      const float4* bias = bias_rows(p, h, r0, lane);
      const Mask<kMask> mask(p, w, ids);
      const float ra = p.scale_log2 * dQ[r0 + g], rb = p.scale_log2 * dQ[r0 + g + 8];
      float o[8][4];
#pragma unroll
      for (int d = 0; d < 8; ++d) o[d][0] = o[d][1] = o[d][2] = o[d][3] = 0.f;
      float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
#pragma unroll 1
      for (int n0 = 0; n0 < p.N; n0 += 8 * kChunk) {
        float c[kChunk][4];
        rows_by_rows<kChunk>(c, sQ + r0 * 128, sK + n0 * 128, L);
        logits<kMask, false, kChunk>(c, bias, ra, rb, dK, mask, r0, n0, g, q);
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
        acc_by_cols<kChunk>(o, c, sV + n0 * 128, dV + n0 + 2 * q, L);
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

// Q, K, V, dO; their rows' scales; per query: -(row maximum), -(log2 of the row sum), delta; the region ids
constexpr int kBwdSmem = 4 * kOperand + 8 * kMaxN * 4;

template <int kMask>
__global__ void __launch_bounds__(kThreads, 1) rel_bias_bwd_f32_kernel(const Params p) {
  extern __shared__ __align__(128) uint8_t sm[];
  const uint32_t sQ = smem_u32(sm), sK = sQ + kOperand, sV = sK + kOperand, sG = sV + kOperand;
  float *dQ = reinterpret_cast<float*>(sm + 4 * kOperand), *dK = dQ + kMaxN, *dV = dK + kMaxN, *dG = dV + kMaxN;
  float *sMax = dG + kMaxN, *sLog = sMax + kMaxN, *sDelta = sLog + kMaxN;
  int* ids = reinterpret_cast<int*>(sDelta + kMaxN);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, q = lane & 3, r0 = 16 * warp;
  const Lanes L;
  const int t_begin = tile_begin(p.num_tiles), t_end = tile_end(p.num_tiles);
  for (int t = t_begin; t < t_end; ++t) {
    const int h = t / p.Bwin, w = t - h * p.Bwin;
    {
      Share a, b;
      a.fetch(p.q, p.sq, w, h, p.N);
      b.fetch(p.k, p.sk, w, h, p.N);
      load_ids<kMask>(p, w, ids);
      if (threadIdx.x < kMaxN) {  // rows past N: P = 0
        const float2 st = threadIdx.x < p.N ? __ldg(p.stats + ((int64_t)w * p.H + h) * kMaxN + threadIdx.x)
                                            : make_float2(INFINITY, 0.f);
        sMax[threadIdx.x] = -st.x;
        sLog[threadIdx.x] = -st.y;
      }
      a.put(sQ, dQ);
      a.fetch(p.v, p.sv, w, h, p.N);
      b.put(sK, dK);
      b.fetch(p.dout, p.so, w, h, p.N);
      a.put(sV, dV);
      b.put(sG, dG);
    }
    __syncthreads();
    const Mask<kMask> mask(p, w, ids);
    if (r0 < p.N) {
      // Queries by rows.
      float c[18][4], d[18][4];
      rows_by_rows<18>(c, sQ + r0 * 128, sK, L);
      logits<kMask, false, 18>(c, bias_rows(p, h, r0, lane), p.scale_log2 * dQ[r0 + g], p.scale_log2 * dQ[r0 + g + 8], dK,
                               mask, r0, 0, g, q);
      rows_by_rows<18>(d, sG + r0 * 128, sV, L);
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const float mx = sMax[r0 + g + 8 * i], lg = sLog[r0 + g + 8 * i], dg = dG[r0 + g + 8 * i];
        float delta = 0.f;
#pragma unroll
        for (int j = 0; j < 18; ++j) {
          const float2 s = *reinterpret_cast<const float2*>(dV + 8 * j + 2 * q);
#pragma unroll
          for (int e = 2 * i; e < 2 * i + 2; ++e) {
            c[j][e] = exp2f(c[j][e] + mx + lg);
            d[j][e] *= (e & 1 ? s.y : s.x) * dg;
            delta = fmaf(c[j][e], d[j][e], delta);
          }
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
      acc_by_cols<18>(o, c, sK, dK + 2 * q, L);
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
      const float ra = p.scale_log2 * dK[r0 + g], rb = p.scale_log2 * dK[r0 + g + 8];
      const float va = dV[r0 + g], vb = dV[r0 + g + 8];
#pragma unroll 1
      for (int n0 = 0; n0 < p.N; n0 += 8 * kChunk) {
        float c[kChunk][4], d[kChunk][4];
        rows_by_rows<kChunk>(c, sK + r0 * 128, sQ + n0 * 128, L);
        logits<kMask, true, kChunk>(c, bias, ra, rb, dQ, mask, r0, n0, g, q);
        rows_by_rows<kChunk>(d, sV + r0 * 128, sG + n0 * 128, L);
#pragma unroll
        for (int j = 0; j < kChunk; ++j)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const int n = n0 + 8 * j + 2 * q + e;  // queries past N: sMax is -inf, so P = dS = 0
            const float mxn = sMax[n], lgn = sLog[n], dgn = dG[n], dln = n < p.N ? sDelta[n] : 0.f;
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              const float pr = exp2f(c[j][2 * i + e] + mxn + lgn);
              c[j][2 * i + e] = pr;
              d[j][2 * i + e] = pr * (d[j][2 * i + e] * ((i ? vb : va) * dgn) - dln);
            }
          }
        acc_by_cols<kChunk>(gv, c, sG + n0 * 128, dG + n0 + 2 * q, L);
        acc_by_cols<kChunk>(gk, d, sQ + n0 * 128, dQ + n0 + 2 * q, L);
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
  const int grid = p.num_tiles < 2 * num_sms() ? p.num_tiles : 2 * num_sms();
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
