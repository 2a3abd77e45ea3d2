// Shared definitions of window attention with a learned relative position bias (rel_bias*.cu).
#pragma once

#include "attention.cuh"
#include "fa_common.cuh"

namespace fa {
namespace relb {

constexpr float kLog2e = 1.4426950408889634f;

constexpr int kNoRank = 255;

// Tiles are (head, window) pairs in head-major order: tile t = head t / Bwin, window t % Bwin. A
// persistent block takes a contiguous range, so it meets one head, or few, and keeps that head's
// bias (and, backward, that head's bias gradient) across its windows.
struct Params {
  int Bwin, H, N, nW;
  int num_tiles;
  float scale, scale_log2;  // softmax scale, and the same times log2(e)
  const void *q, *k, *v, *dout;
  void *out, *dq, *dk, *dv;
  int64_t sq[3], sk[3], sv[3], so[3];  // element strides of window, head, token; so: out or dout
  int64_t sdq[3], sdk[3], sdv[3];
  const float4* bias;        // the bias in fragment order, see expand_bias_kernel in rel_bias.cu
  const uint8_t* mask;       // (nW, N, N) bytes or (nW, N) region ids, by MaskKind
  const uint8_t* ranks;      // with region ids: (nW, 144) rank of each token's id in its window, kNoRank past N
  uint32_t mask_hi, mask_lo; // bf16 bits: mask_hi + mask_lo = -100 / scale (region masks, bf16 kernels)
  float2* stats;             // (Bwin, H, 144): row maximum and log2 of the row sum, log2 domain
  float* slots;              // backward: (gridDim.x + H - 1) partial bias gradients in fragment order
  int* status;
};

__device__ __forceinline__ int tile_begin(int num_tiles) {
  return (int)(((int64_t)blockIdx.x * num_tiles) / gridDim.x);
}
__device__ __forceinline__ int tile_end(int num_tiles) {
  return (int)(((int64_t)(blockIdx.x + 1) * num_tiles) / gridDim.x);
}

// The fragment order of a head's bias: the 144 x 144 pairs in 9 blocks of 16 rows, each as 18 blocks of 8
// keys, each as one float4 per lane: rows t1 and t1 + 8 (x, y and z, w), keys 2 t0 and 2 t0 + 1, with
// t0 = lane % 4 and t1 = lane / 4. It is the accumulator layout of both kinds of tensor-core kernel here,
// so a warp reads its rows with coalesced 16-byte loads.
constexpr int kBiasVecs = 9 * 18 * 32;  // float4 per head
__device__ __forceinline__ const float4* bias_rows(const Params& p, int h, int row0, int lane) {
  return p.bias + ((int64_t)h * 9 + (row0 >> 4)) * (18 * 32) + lane;
}

// The same rows of a partial bias gradient.
__device__ __forceinline__ float4* slot_rows(const Params& p, int slot, int row0, int lane) {
  return reinterpret_cast<float4*>(p.slots) + ((int64_t)slot * 9 + (row0 >> 4)) * (18 * 32) + lane;
}
// Float index of pair (i, j) in fragment order.
__device__ __forceinline__ int frag_index(int i, int j) {
  return (((i >> 4) * 18 + (j >> 3)) * 32 + ((i & 7) << 2 | (j & 7) >> 1)) * 4 + ((i & 8) >> 2 | (j & 1));
}

// The fp32 kernels (rel_bias_f32.cu). Their backward pass also reads the transposed bias: heads H .. 2H - 1
// of `bias` hold, in fragment order, the pairs with keys as rows.
int run_f32_forward(const Params& p, int mask_kind, cudaStream_t s);
int run_f32_backward(const Params& p, int mask_kind, int grid, cudaStream_t s);

// The bf16 kernels (rel_bias_tc.cu); mask_kind: attn::kNoMask, kGroups or kMaskU8.
int run_bf16_forward(const Params& p, int mask_kind, int grid, cudaStream_t s);
int run_bf16_backward(const Params& p, int mask_kind, int grid, cudaStream_t s);

}  // namespace relb
}  // namespace fa
