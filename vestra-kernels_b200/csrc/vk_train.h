// vk_train.h -- launchers of the trainable block pieces (attention with row
// statistics and its backward pass, rotary positions over several axes, the
// residual step between two norms), shared between their kernel files and the
// C-ABI layer (vk_abi_train.cu).
#pragma once

#include <cuda_runtime.h>
#include <stddef.h>
#include <stdint.h>

namespace vk {

// Division of n < 2^31 by a constant: a few instructions where the general
// one takes a hundred, at every step.
struct FastDiv {
  uint32_t mul, shift;
  explicit FastDiv(uint32_t d) : mul(0), shift(0) {
    while ((uint64_t{1} << shift) < d) ++shift;
    mul = static_cast<uint32_t>((((uint64_t{1} << shift) - d) << 32) / d + 1);
  }
  __device__ __forceinline__ int operator()(int n) const {
    return static_cast<int>((__umulhi(static_cast<uint32_t>(n), mul) + static_cast<uint32_t>(n)) >> shift);
  }
};

// A [batch, heads, tokens, head_dim] tensor, strides in elements.
struct HeadsView {
  void* p = nullptr;
  int64_t sb = 0, sh = 0, st = 0;
};

struct AttnShape {
  int batch = 0, heads = 0, nq = 0, nk = 0, dim = 0;
  float scale = 0.0f;
  const int32_t* q_lens = nullptr;   // [batch] or null
  const int32_t* kv_lens = nullptr;  // [batch] or null
};

// Tokens of sequence b: the whole dimension, or its length clamped to it.
__device__ __forceinline__ int seq_len(const int32_t* lens, int b, int tokens) {
  if (lens == nullptr) return tokens;
  const int n = __ldg(lens + b);
  return n < 0 ? 0 : (n > tokens ? tokens : n);
}

// CUDA-core attention, f32 or bf16 elements, head_dim 8, 16, 32 or 64
// (vk_attention_grad.cu).  The forward pass takes bf16 of 64 for one query only.
cudaError_t attention_forward_simt(const AttnShape& a, bool bf16, HeadsView q, HeadsView k, HeadsView v, HeadsView out,
                                   float* lse, cudaStream_t s);
cudaError_t attention_backward_simt(const AttnShape& a, bool bf16, HeadsView q, HeadsView k, HeadsView v, HeadsView out,
                                    const float* lse, HeadsView d_out, HeadsView dq, HeadsView dk, HeadsView dv,
                                    float* delta, cudaStream_t s);
// The same on the tensor cores, bf16, head_dim 64 (vk_attention_grad_tc.cu).
cudaError_t attention_forward_tc(const AttnShape& a, HeadsView q, HeadsView k, HeadsView v, HeadsView out, float* lse,
                                 int* err, cudaStream_t s);
cudaError_t attention_backward_tc(const AttnShape& a, HeadsView q, HeadsView k, HeadsView v, HeadsView out,
                                  const float* lse, HeadsView d_out, HeadsView dq, HeadsView dk, HeadsView dv,
                                  float* delta, int* err, cudaStream_t s);
// Zeros over [batch, heads, tokens, dim] / one value over n floats.
cudaError_t zero_heads(HeadsView x, bool bf16, int batch, int heads, int tokens, int dim, cudaStream_t s);
cudaError_t fill_f32(float* x, size_t n, float value, cudaStream_t s);

// Rotary positions over several axes (vk_rope_axes.cu).  Pair i of a head
// turns elements lo[i] and hi[i] by position[axis[i]] * inv[i].
constexpr int ROPE_MAX_PAIRS = 128;
struct RopePairs {
  double inv[ROPE_MAX_PAIRS];
  int16_t lo[ROPE_MAX_PAIRS], hi[ROPE_MAX_PAIRS];
  int8_t axis[ROPE_MAX_PAIRS];
  int pairs;    // pairs in all sections
  int rotated;  // elements in all sections; the others are copied
  int vec;      // 8, 4, 2 or 1: consecutive pairs whose elements are consecutive too, a divisor of every half section
};
cudaError_t rope_axes(bool bf16, int batch, int heads, int tokens, int head_dim, int axes, const RopePairs& pairs,
                      bool inverse, const int64_t* positions, bool positions_per_batch, HeadsView q, HeadsView q_out,
                      HeadsView k, HeadsView k_out, cudaStream_t s);

// The residual step between two norms (vk_residual_norm.cu).
struct ResidualNorm {
  int groups = 0, rows_per_group = 0, cols = 0;
  float eps = 0.0f;
  const float *gamma = nullptr, *beta = nullptr, *scale = nullptr, *gate = nullptr, *post_gamma = nullptr,
              *post_beta = nullptr;
};
constexpr int RESIDUAL_NORM_MAX_COLS = 8192;
cudaError_t residual_norm_forward(const ResidualNorm& r, bool stream_bf16, bool branch_bf16, const void* x,
                                  const void* branch, void* h, void* y, float* stats, float* post_stats,
                                  cudaStream_t s);
struct ResidualNormGrads {
  void *d_x = nullptr, *d_branch = nullptr;
  float *d_gamma = nullptr, *d_beta = nullptr, *d_scale = nullptr, *d_gate = nullptr, *d_post_gamma = nullptr,
        *d_post_beta = nullptr;
};
size_t residual_norm_workspace(const ResidualNorm& r);
cudaError_t residual_norm_backward(const ResidualNorm& r, bool stream_bf16, bool branch_bf16, const void* d_h,
                                   const void* d_y, const void* h, const void* branch, const float* stats,
                                   const float* post_stats, const ResidualNormGrads& g, float* workspace,
                                   cudaStream_t s);

}  // namespace vk
