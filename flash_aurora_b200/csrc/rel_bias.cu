// Window attention with a learned relative position bias, and its gradients (N <= 144, head_dim 64).
//
//   x_ij = scale q_i . k_j + T[index_ij, h] + mask_ij        mask: -100 where masked
//   P = softmax_j(x),  o = P v
//   dV = P^T dO,  dP = dO V^T,  dS_ij = P_ij (dP_ij - sum_j' P_ij' dP_ij')
//   dQ = scale dS K,  dK = scale dS^T Q,  dT[b, h] = sum over windows and pairs with index_ij = b of dS_ij
//
// The backward pass recomputes P from q, k and the bias with the row statistics that the forward
// pass kept, so nothing of size N x N per window ever reaches memory. The bias gradient is summed
// over the windows of a head inside each block (one N x N partial per block and head), and a second
// kernel adds the partials and the pairs of a bucket in a fixed order: no atomics, so the same call
// gives the same bits.
#include <cuda_bf16.h>

#include <cmath>

#include "rel_bias.cuh"

namespace fa {
namespace relb {
namespace {

using attn::kGroups;
using attn::kMaskedLog2;
using attn::kMaskU8;
using attn::kMaxN;
using attn::kNoMask;

// The bias of (query i, key j) in the log2 domain; -inf for keys past N, 0 for query rows past N.
// A finite entry stays finite (the clamp), so that a row of the lowest values is still a row.
__device__ __forceinline__ float bias_log2(const void* table, int bf16, const int32_t* index, int H, int N, int h, int i,
                                           int j) {
  if (j >= N) return -INFINITY;
  if (i >= N) return 0.f;
  const int64_t e = (int64_t)__ldg(index + i * N + j) * H + h;
  const float b = bf16 ? __bfloat162float(reinterpret_cast<const __nv_bfloat16*>(table)[e])
                       : __ldg(reinterpret_cast<const float*>(table) + e);
  const float x = b * kLog2e;
  return isinf(x) && !isinf(b) ? copysignf(3.4028234e38f, b) : x;
}

// What the attention kernels read beside their tensors: every head's bias in fragment order (see
// bias_rows), one float4 per thread of the first blocks, and with region ids the rank of every token's id
// among the ids of its window, one warp per window of the others. The gathers hit L1 here; in the
// attention kernels, whose shared memory leaves no L1, they cost a block 30 us a head.
constexpr int kExpandThreads = 192;
constexpr int kExpandBlocks = kBiasVecs / kExpandThreads;  // per head
static_assert(kBiasVecs % kExpandThreads == 0, "whole blocks");

__device__ __forceinline__ void rank_window(const uint8_t* ids, int N, int lane, uint8_t* out) {
  uint32_t id[5];
  int rank[5];
#pragma unroll
  for (int m = 0; m < 5; ++m) {
    id[m] = lane + 32 * m < N ? (uint32_t)__ldg(ids + lane + 32 * m) : 256u;
    rank[m] = 0;
  }
#pragma unroll
  for (uint32_t k = 0; k < 8; ++k) {  // ids 32 k .. 32 k + 31
    uint32_t bits = 0;
#pragma unroll
    for (int m = 0; m < 5; ++m) bits |= (id[m] >> 5) == k ? 1u << (id[m] & 31) : 0u;
    bits = __reduce_or_sync(0xffffffffu, bits);
#pragma unroll
    for (int m = 0; m < 5; ++m)
      rank[m] += (id[m] >> 5) > k ? __popc(bits) : (id[m] >> 5) == k ? __popc(bits & ((1u << (id[m] & 31)) - 1u)) : 0;
  }
#pragma unroll
  for (int m = 0; m < 5; ++m)
    if (lane + 32 * m < kMaxN) out[lane + 32 * m] = (uint8_t)(id[m] < 256u ? rank[m] : kNoRank);
}

__global__ void __launch_bounds__(kExpandThreads)
expand_bias_kernel(const void* table, int bf16, const int32_t* index, int H, int copies, int N, float4* out,
                   const uint8_t* ids, int64_t nW, uint8_t* ranks) {
  if ((int64_t)blockIdx.x >= (int64_t)copies * H * kExpandBlocks) {
    const int64_t w = ((int64_t)blockIdx.x - (int64_t)copies * H * kExpandBlocks) * (kExpandThreads / 32) + (threadIdx.x >> 5);
    if (w < nW) rank_window(ids + w * N, N, threadIdx.x & 31, ranks + w * kMaxN);
    return;
  }
  const int hc = blockIdx.x / kExpandBlocks, e = (blockIdx.x % kExpandBlocks) * kExpandThreads + threadIdx.x;
  const int lane = e & 31, j = (e >> 5) % 18, blk = (e >> 5) / 18;
  const int i = 16 * blk + (lane >> 2), k = 8 * j + 2 * (lane & 3);
  const bool transposed = hc >= H;  // rows are keys
  const int h = transposed ? hc - H : hc;
  float v[4];
#pragma unroll
  for (int c = 0; c < 4; ++c) {
    const int row = i + 8 * (c >> 1), col = k + (c & 1);
    v[c] = transposed ? bias_log2(table, bf16, index, H, N, h, col, row) : bias_log2(table, bf16, index, H, N, h, row, col);
  }
  out[(int64_t)hc * kBiasVecs + e] = make_float4(v[0], v[1], v[2], v[3]);
}

// The blocks of a main kernel of `grid` blocks whose tile ranges meet head h: block c covers tiles
// [c T / G, (c + 1) T / G), head h tiles [h Bwin, (h + 1) Bwin).
__device__ __forceinline__ int2 blocks_of_head(int h, int Bwin, int num_tiles, int grid) {
  auto block_of = [&](int64_t tile) {
    int c = (int)(tile * grid / num_tiles);
    while (c > 0 && (int64_t)c * num_tiles / grid > tile) --c;
    while (c + 1 < grid && (int64_t)(c + 1) * num_tiles / grid <= tile) ++c;
    return c;
  };
  const int64_t lo = (int64_t)h * Bwin;
  return make_int2(block_of(lo), block_of(lo + Bwin - 1));
}

// Adds a head's partials, coalesced, into its first one, one thread per pair; without this pass the
// gather below reads a sector per pair and partial.
constexpr int kSumThreads = 128;
__global__ void __launch_bounds__(kSumThreads) sum_slots_kernel(float* slots, int H, int Bwin, int num_tiles, int grid) {
  const int e = blockIdx.x * kSumThreads + threadIdx.x;
  for (int h = blockIdx.y; h < H; h += gridDim.y) {
    const int2 c = blocks_of_head(h, Bwin, num_tiles, grid);
    float* p = slots + (int64_t)(c.x + h) * (4 * kBiasVecs) + e;
    float s = *p;
#pragma unroll 8
    for (int i = 1; i <= c.y - c.x; ++i) s += __ldg(p + (int64_t)i * (4 * kBiasVecs));
    *p = s;
  }
}
static_assert(4 * kBiasVecs % kSumThreads == 0, "whole blocks");

// dT[b, h] = sum over the pairs of bucket b (positions order[offsets[b]] .. in the N x N index) of the
// head's first partial (summed: it is the sum of all) or of each, by kPer threads, a warp or a block, each
// adding its share in a fixed order.
constexpr int kReduceThreads = 256;
template <int kPer>
__global__ void __launch_bounds__(kReduceThreads)
bias_grad_kernel(const float* slots, const int32_t* order, const int32_t* offsets, void* dtable, int dtable_bf16, int H,
                 int num_buckets, int N, int Bwin, int num_tiles, int grid, int summed) {
  const int b = blockIdx.x * (kReduceThreads / kPer) + threadIdx.x / kPer, t = threadIdx.x % kPer;
  if (b >= num_buckets) return;  // whole warps
  for (int h = blockIdx.y; h < H; h += gridDim.y) {
    float acc = 0.f;
    if (num_tiles > 0) {
      int2 c = blocks_of_head(h, Bwin, num_tiles, grid);
      if (summed) c.y = c.x;
      const int p1 = offsets[b + 1];
      for (int e = offsets[b] + t; e < p1; e += kPer) {
        const int pos = order[e], i = pos / N;
        const float* f = slots + (int64_t)(c.x + h) * (4 * kBiasVecs) + frag_index(i, pos - i * N);
        for (int k = 0; k <= c.y - c.x; ++k) acc += f[(int64_t)k * (4 * kBiasVecs)];
      }
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) acc += __shfl_xor_sync(0xffffffffu, acc, o);
    if constexpr (kPer > 32) {
      __shared__ float warp_acc[kPer / 32];
      __syncthreads();
      if ((t & 31) == 0) warp_acc[t >> 5] = acc;
      __syncthreads();
      acc = 0.f;
      for (int i = 0; i < kPer / 32; ++i) acc += warp_acc[i];
    }
    if (t == 0) {
      const int64_t e = (int64_t)b * H + h;
      if (dtable_bf16) reinterpret_cast<__nv_bfloat16*>(dtable)[e] = __float2bfloat16_rn(acc);
      else reinterpret_cast<float*>(dtable)[e] = acc;
    }
  }
}

// Bias copies in the state: the fp32 backward pass reads the transposed one too.
int bias_copies(int precision) { return precision == FA_ATTN_BF16 ? 1 : 2; }

int grid_of(int64_t tiles) { return (int)(tiles < num_sms() ? tiles : num_sms()); }

// Checks shared by both directions; strides are {window, head, token} triples.
int check_args(int precision, int64_t Bwin, int64_t H, int64_t N, int64_t Dh, const void* const* ptrs, int n_ptrs,
               const int64_t* strides, const void* state, bool u8, bool ids, int64_t nW, float scale) {
  FA_REQUIRE(precision == FA_ATTN_BF16 || precision == FA_ATTN_FP32_3XTF32, FA_ERR_INVALID,
             "precision must be FA_ATTN_BF16 or FA_ATTN_FP32_3XTF32");
  FA_REQUIRE(strides, FA_ERR_INVALID, "null stride pointer");
  FA_REQUIRE(Bwin >= 0 && H >= 1 && N >= 1, FA_ERR_INVALID, "invalid attention shape");
  FA_REQUIRE(Dh == 64, FA_ERR_UNSUPPORTED, "window attention supports head_dim 64");
  FA_REQUIRE(N <= kMaxN, FA_ERR_UNSUPPORTED, "window attention supports N <= 144 tokens");
  FA_REQUIRE(fabsf(scale) >= 1e-30f && fabsf(scale) <= 1e30f, FA_ERR_INVALID,
             "scale must be finite and at least 1e-30 in magnitude");
  FA_REQUIRE(!(u8 && ids), FA_ERR_INVALID, "pass at most one of mask_u8 / group_ids");
  FA_REQUIRE(!(u8 || ids) || nW >= 1, FA_ERR_INVALID, "nW must be >= 1 with a mask");
  FA_REQUIRE(nW < ((int64_t)1 << 31), FA_ERR_INVALID, "too many mask windows");
  FA_REQUIRE(Bwin < ((int64_t)1 << 31) && H < ((int64_t)1 << 31) && Bwin * H < ((int64_t)1 << 31), FA_ERR_INVALID,
             "too many (window, head) tiles");
  if (Bwin == 0) return FA_OK;
  FA_REQUIRE(state && aligned16(state), FA_ERR_INVALID, "the state buffer must be given, 16-byte aligned");
  const int64_t es = precision == FA_ATTN_FP32_3XTF32 ? 4 : 2;
  for (int i = 0; i < n_ptrs; ++i) {
    FA_REQUIRE(ptrs[i], FA_ERR_INVALID, "null tensor pointer");
    FA_REQUIRE(aligned16(ptrs[i]), FA_ERR_INVALID, "tensors must be 16-byte aligned");
    for (int j = 0; j < 3; ++j)
      FA_REQUIRE(strides[3 * i + j] > 0 && (strides[3 * i + j] * es) % 16 == 0, FA_ERR_INVALID,
                 "strides must be positive multiples of 16 bytes");
  }
  return FA_OK;
}

// Two bf16 numbers whose sum is -100 / scale to 2^-17 of it.
void split_mask_value(float scale, uint32_t* hi_bits, uint32_t* lo_bits) {
  const double want = -100.0 / (double)scale;
  const __nv_bfloat16 hi = __float2bfloat16((float)want);
  *hi_bits = __nv_bfloat16_raw(hi).x;
  *lo_bits = __nv_bfloat16_raw(__float2bfloat16((float)(want - (double)__bfloat162float(hi)))).x;
}

void copy3(int64_t* dst, const int64_t* src) {
  for (int i = 0; i < 3; ++i) dst[i] = src[i];
}

}  // namespace
}  // namespace relb
}  // namespace fa

using namespace fa;
using namespace fa::relb;

extern "C" int64_t fa_window_attention_rel_bias_state(int precision, int64_t H, int64_t nW_ids) {
  if ((precision != FA_ATTN_BF16 && precision != FA_ATTN_FP32_3XTF32) || H < 1 || H >= ((int64_t)1 << 31) || nW_ids < 0 ||
      nW_ids >= ((int64_t)1 << 31))
    return set_error(FA_ERR_INVALID, "invalid attention shape");
  return bias_copies(precision) * H * kBiasVecs * 16 + nW_ids * kMaxN;
}

extern "C" int64_t fa_window_attention_rel_bias_workspace(int64_t Bwin, int64_t H, int64_t N) {
  if (Bwin < 0 || H < 1 || N < 1 || N > kMaxN || Bwin >= ((int64_t)1 << 31) || H >= ((int64_t)1 << 31) ||
      Bwin * H >= ((int64_t)1 << 31))
    return set_error(FA_ERR_INVALID, "invalid attention shape");
  return (grid_of(Bwin * H) + H) * kBiasVecs * 16;
}

extern "C" int fa_window_attention_rel_bias(int precision, int64_t Bwin, int64_t H, int64_t N, int64_t Dh,
                                            const void* q, const void* k, const void* v, void* out,
                                            const int64_t strides[12], const void* table, int table_dtype,
                                            const int32_t* index, const uint8_t* mask_u8, const uint8_t* group_ids,
                                            int64_t nW, float scale, void* state, float* stats, void* stream) {
  const void* ptrs[4] = {q, k, v, out};
  int rc = check_args(precision, Bwin, H, N, Dh, ptrs, 4, strides, state, mask_u8 != nullptr, group_ids != nullptr, nW,
                      scale);
  FA_REQUIRE(rc != FA_OK || (table && index && (table_dtype == FA_F32 || table_dtype == FA_BF16)), FA_ERR_INVALID,
             "null bias table or index, or table dtype not FA_F32 or FA_BF16");
  if (rc != FA_OK || Bwin == 0) return rc;
  FA_REQUIRE(aligned16(stats), FA_ERR_INVALID, "the row statistics must be 16-byte aligned");
  Params p{};
  p.Bwin = (int)Bwin; p.H = (int)H; p.N = (int)N; p.nW = (int)(nW > 0 ? nW : 1);
  p.num_tiles = (int)(Bwin * H);
  p.scale = scale; p.scale_log2 = scale * kLog2e;
  p.q = q; p.k = k; p.v = v; p.out = out;
  copy3(p.sq, strides); copy3(p.sk, strides + 3); copy3(p.sv, strides + 6); copy3(p.so, strides + 9);
  p.bias = reinterpret_cast<const float4*>(state);
  p.ranks = reinterpret_cast<const uint8_t*>(p.bias + bias_copies(precision) * H * kBiasVecs);
  p.mask = mask_u8 ? mask_u8 : group_ids;
  if (group_ids) split_mask_value(scale, &p.mask_hi, &p.mask_lo);
  p.stats = reinterpret_cast<float2*>(stats);
  cudaStream_t s = (cudaStream_t)stream;
  const int copies = bias_copies(precision);
  const int64_t blocks = copies * H * kExpandBlocks + (group_ids ? (nW + kExpandThreads / 32 - 1) / (kExpandThreads / 32) : 0);
  FA_REQUIRE(blocks < ((int64_t)1 << 31), FA_ERR_INVALID, "too many heads or mask windows");
  expand_bias_kernel<<<(unsigned)blocks, kExpandThreads, 0, s>>>(table, table_dtype == FA_BF16, index, p.H, copies, p.N,
                                                                reinterpret_cast<float4*>(state), group_ids,
                                                                group_ids ? nW : 0, const_cast<uint8_t*>(p.ranks));
  if ((rc = check_launch("expand_bias_kernel")) != FA_OK) return rc;
  const int grid = grid_of(p.num_tiles);
  p.status = attn::status_ptr();
  FA_REQUIRE(p.status, FA_ERR_CUDA, "cannot resolve the attention status word");
  const int kind = mask_u8 ? kMaskU8 : group_ids ? kGroups : kNoMask;
  return precision == FA_ATTN_BF16 ? run_bf16_forward(p, kind, grid, s) : run_f32_forward(p, kind, s);
}

extern "C" int fa_window_attention_rel_bias_backward(
    int precision, int64_t Bwin, int64_t H, int64_t N, int64_t Dh, const void* q, const void* k, const void* v,
    const void* dout, void* dq, void* dk, void* dv, const int64_t strides[21], const uint8_t* mask_u8,
    const uint8_t* group_ids, int64_t nW, float scale, const void* state, const float* stats, const int32_t* order,
    const int32_t* offsets, int64_t num_buckets, void* dtable, int dtable_dtype, void* workspace,
    int64_t workspace_bytes, void* stream) {
  const void* ptrs[7] = {q, k, v, dout, dq, dk, dv};
  int rc = check_args(precision, Bwin, H, N, Dh, ptrs, 7, strides, state, mask_u8 != nullptr, group_ids != nullptr, nW,
                      scale);
  if (rc != FA_OK) return rc;
  FA_REQUIRE((stats && aligned16(stats)) || Bwin == 0, FA_ERR_INVALID,
             "the row statistics must be given, 16-byte aligned");
  FA_REQUIRE(!dtable || dtable_dtype == FA_F32 || dtable_dtype == FA_BF16, FA_ERR_INVALID,
             "table dtype must be FA_F32 or FA_BF16");
  FA_REQUIRE(!dtable || (order && offsets && num_buckets >= 1 && num_buckets < ((int64_t)1 << 31)),
             FA_ERR_INVALID, "a bias gradient needs the bucket lists");
  cudaStream_t s = (cudaStream_t)stream;
  const int64_t need = fa_window_attention_rel_bias_workspace(Bwin, H, N);
  FA_REQUIRE(Bwin == 0 || (workspace && workspace_bytes >= need), FA_ERR_INVALID, "workspace too small");
  FA_REQUIRE(Bwin == 0 || aligned16(workspace), FA_ERR_INVALID, "the workspace must be 16-byte aligned");
  const int grid = grid_of(Bwin * H);
  if (Bwin > 0) {
    Params p{};
    p.Bwin = (int)Bwin; p.H = (int)H; p.N = (int)N; p.nW = (int)(nW > 0 ? nW : 1);
    p.num_tiles = (int)(Bwin * H);
    p.scale = scale; p.scale_log2 = scale * kLog2e;
    p.q = q; p.k = k; p.v = v; p.dout = dout; p.dq = dq; p.dk = dk; p.dv = dv;
    copy3(p.sq, strides); copy3(p.sk, strides + 3); copy3(p.sv, strides + 6); copy3(p.so, strides + 9);
    copy3(p.sdq, strides + 12); copy3(p.sdk, strides + 15); copy3(p.sdv, strides + 18);
    p.bias = reinterpret_cast<const float4*>(state);
    p.ranks = reinterpret_cast<const uint8_t*>(p.bias + bias_copies(precision) * H * kBiasVecs);
    p.mask = mask_u8 ? mask_u8 : group_ids;
    if (group_ids) split_mask_value(scale, &p.mask_hi, &p.mask_lo);
    p.stats = const_cast<float2*>(reinterpret_cast<const float2*>(stats));
    p.slots = dtable ? reinterpret_cast<float*>(workspace) : nullptr;
    p.status = attn::status_ptr();
    FA_REQUIRE(p.status, FA_ERR_CUDA, "cannot resolve the attention status word");
    const int kind = mask_u8 ? kMaskU8 : group_ids ? kGroups : kNoMask;
    rc = precision == FA_ATTN_BF16 ? run_bf16_backward(p, kind, grid, s) : run_f32_backward(p, kind, grid, s);
    if (rc != FA_OK) return rc;
  }
  if (!dtable) return FA_OK;
  const unsigned heads = (unsigned)(H < 65535 ? H : 65535);
  // Up to about three partials a head are gathered directly: a second launch costs more than it saves.
  const bool sum = Bwin > 0 && grid > 2 * H;
  if (sum) {
    sum_slots_kernel<<<dim3(4 * kBiasVecs / kSumThreads, heads), kSumThreads, 0, s>>>(
        reinterpret_cast<float*>(workspace), (int)H, (int)Bwin, (int)(Bwin * H), grid);
    if ((rc = check_launch("sum_slots_kernel")) != FA_OK) return rc;
  }
  // A warp per bucket where buckets are small (the 3-D offsets of a window: 27 pairs each on average, 20 us
  // with a block each), a block where they are large (32 log-distance buckets: 18 us with two warps each).
  const bool small = N * N <= 64 * num_buckets;
  auto kern = small ? bias_grad_kernel<32> : bias_grad_kernel<kReduceThreads>;
  const unsigned per_block = small ? kReduceThreads / 32 : 1;
  kern<<<dim3(((unsigned)num_buckets + per_block - 1) / per_block, heads), kReduceThreads, 0, s>>>(
      reinterpret_cast<const float*>(workspace), order, offsets, dtable, dtable_dtype == FA_BF16, (int)H, (int)num_buckets,
      (int)N, (int)Bwin, (int)(Bwin * H), grid, sum ? 1 : 0);
  return check_launch("bias_grad_kernel");
}
