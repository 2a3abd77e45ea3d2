// Shared definitions of window attention with a learned relative position bias (rel_bias*.cu).
#pragma once

#include "attention.cuh"
#include "fa_common.cuh"

namespace fa {
namespace relb {

constexpr float kLog2e = 1.4426950408889634f;

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
  const void* table;         // (num_buckets, H)
  int table_bf16;
  const int32_t* index;      // (N, N) bucket of each (query, key)
  const uint8_t* mask;       // (nW, N, N) bytes or (nW, N) region ids, by MaskKind
  float2* stats;             // (Bwin, H, N): row maximum and log2 of the row sum, log2 domain
  float* slots;              // backward: (gridDim.x + H - 1) partial bias gradients (N, N)
  int* status;
};

__device__ __forceinline__ int tile_begin(int num_tiles) {
  return (int)(((int64_t)blockIdx.x * num_tiles) / gridDim.x);
}
__device__ __forceinline__ int tile_end(int num_tiles) {
  return (int)(((int64_t)(blockIdx.x + 1) * num_tiles) / gridDim.x);
}

// The bias of (query i, key j) in the log2 domain; -inf for keys past N, 0 for query rows past N.
// A finite entry stays finite (the clamp), so that a row of the lowest values is still a row.
__device__ __forceinline__ float bias_log2(const Params& p, int h, int i, int j) {
  if (j >= p.N) return -INFINITY;
  if (i >= p.N) return 0.f;
  const int64_t e = (int64_t)__ldg(p.index + i * p.N + j) * p.H + h;
  const float b = p.table_bf16 ? __bfloat162float(reinterpret_cast<const __nv_bfloat16*>(p.table)[e])
                               : __ldg(reinterpret_cast<const float*>(p.table) + e);
  const float x = b * kLog2e;
  return isinf(x) && !isinf(b) ? copysignf(3.4028234e38f, b) : x;
}

// The bf16 kernels (rel_bias_tc.cu); mask_kind: attn::kNoMask, kGroups or kMaskU8.
int run_bf16_forward(const Params& p, int mask_kind, int grid, cudaStream_t s);
int run_bf16_backward(const Params& p, int mask_kind, int grid, cudaStream_t s);

}  // namespace relb
}  // namespace fa
