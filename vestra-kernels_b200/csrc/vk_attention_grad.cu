// vk_attention_grad.cu -- attention with row statistics and its backward
// pass on the CUDA cores: f32 elements (f32 arithmetic throughout), and bf16
// elements of the head sizes the tensor-core kernels do not take.
//
//   s_ij = scale q_i . k_j          lse_i = log sum_j exp s_ij
//   p_ij = exp(s_ij - lse_i)        out_i = sum_j p_ij v_j
//   delta_i = d_out_i . out_i       dp_ij = d_out_i . v_j
//   ds_ij = p_ij (dp_ij - delta_i)
//   dv_j = sum_i p_ij d_out_i       dk_j = scale sum_i ds_ij q_i
//   dq_i = scale sum_j ds_ij k_j
//
// A block owns 64 rows (queries for the forward pass and dq, keys for dk and
// dv) and streams the other side in tiles of 64, so every sum has one owner
// and a fixed order: no atomics, the same bits every time.  The price is that
// the backward pass computes s and dp twice (7 products instead of 5).
//
// 256 threads hold a 4 x 4 piece of each 64 x 64 product.  Tiles are f32 in
// shared memory with rows of D + 4 floats, which puts the 16 rows that a
// half-warp reads at once on different banks.
#include <cuda_bf16.h>

#include "vk_common.cuh"
#include "vk_internal.h"
#include "vk_train.h"

namespace vk {

namespace {
constexpr int GT = 64;         // rows and columns of a tile
constexpr int G_THREADS = 256; // 16 x 16
constexpr int LDP = GT + 4;    // row of a 64 x 64 tile

__device__ __forceinline__ float4 load4(const float* p) { return *reinterpret_cast<const float4*>(p); }
__device__ __forceinline__ float4 load4(const __nv_bfloat16* p) {
  const uint2 u = *reinterpret_cast<const uint2*>(p);
  const float2 a = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&u.x));
  const float2 b = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&u.y));
  return make_float4(a.x, a.y, b.x, b.y);
}
__device__ __forceinline__ void store1(float* p, float x) { *p = x; }
__device__ __forceinline__ void store1(__nv_bfloat16* p, float x) { *p = __float2bfloat16_rn(x); }

template <class T>
__device__ __forceinline__ T* head_of(const HeadsView& v, int b, int h) {
  return static_cast<T*>(v.p) + b * v.sb + h * v.sh;
}

// Rows [r0, r0 + 64) of one head into shared memory; rows from n on are zero.
template <class T, int D>
__device__ __forceinline__ void load_tile(float* dst, const T* src, int64_t st, int r0, int n) {
#pragma unroll
  for (int i = 0; i < GT * D / 4; i += G_THREADS) {
    const int idx = i + threadIdx.x;
    if (GT * D / 4 % G_THREADS != 0 && idx >= GT * D / 4) break;
    const int row = idx / (D / 4), c = idx % (D / 4) * 4;
    float4 x = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    if (r0 + row < n) x = load4(src + static_cast<int64_t>(r0 + row) * st + c);
    *reinterpret_cast<float4*>(dst + row * (D + 4) + c) = x;
  }
}

// s[i][j] = a[4 ty + i] . b[tx + 16 j]
template <int D>
__device__ __forceinline__ void product_rows(float (&s)[4][4], const float* a, const float* b, int ty, int tx) {
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) s[i][j] = 0.0f;
#pragma unroll 4
  for (int k = 0; k < D; k += 4) {
    float4 x[4], y[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = *reinterpret_cast<const float4*>(a + (4 * ty + i) * (D + 4) + k);
#pragma unroll
    for (int j = 0; j < 4; ++j) y[j] = *reinterpret_cast<const float4*>(b + (tx + 16 * j) * (D + 4) + k);
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        s[i][j] = fmaf(x[i].x, y[j].x, s[i][j]);
        s[i][j] = fmaf(x[i].y, y[j].y, s[i][j]);
        s[i][j] = fmaf(x[i].z, y[j].z, s[i][j]);
        s[i][j] = fmaf(x[i].w, y[j].w, s[i][j]);
      }
  }
}

// acc[i][c] += sum_j p[4 ty + i][j] b[j][CPT tx + c]
template <int D, int CPT>
__device__ __forceinline__ void product_sum(float (&acc)[4][CPT], const float* p, const float* b, int ty, int tx) {
  if (CPT * tx >= D) return;
#pragma unroll 4
  for (int j = 0; j < GT; j += 4) {
    float4 x[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = *reinterpret_cast<const float4*>(p + (4 * ty + i) * LDP + j);
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      float y[CPT];
      const float* row = b + (j + u) * (D + 4) + CPT * tx;
      if constexpr (CPT == 4) {
        const float4 v = *reinterpret_cast<const float4*>(row);
        y[0] = v.x, y[1] = v.y, y[2] = v.z, y[3] = v.w;
      } else if constexpr (CPT == 2) {
        const float2 v = *reinterpret_cast<const float2*>(row);
        y[0] = v.x, y[1] = v.y;
      } else {
        y[0] = *row;
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float pv = u == 0 ? x[i].x : u == 1 ? x[i].y : u == 2 ? x[i].z : x[i].w;
#pragma unroll
        for (int c = 0; c < CPT; ++c) acc[i][c] = fmaf(pv, y[c], acc[i][c]);
      }
    }
  }
}

__device__ __forceinline__ float half_warp_sum(float x) {
#pragma unroll
  for (int o = 8; o > 0; o >>= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
  return x;
}
__device__ __forceinline__ float half_warp_max(float x) {
#pragma unroll
  for (int o = 8; o > 0; o >>= 1) x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, o));
  return x;
}

template <int D>
constexpr int cols_per_thread = D >= 16 ? D / 16 : 1;
}  // namespace

template <class T, int D>
__global__ void __launch_bounds__(G_THREADS)
    k_attn_forward_simt(AttnShape a, HeadsView q, HeadsView k, HeadsView v, HeadsView out, float* __restrict__ lse) {
  extern __shared__ float sm[];
  constexpr int CPT = cols_per_thread<D>;
  float* sQ = sm;
  float* sK = sQ + GT * (D + 4);
  float* sV = sK + GT * (D + 4);
  float* sP = sV + GT * (D + 4);
  const int tiles = (a.nq + GT - 1) / GT;
  const int bh = blockIdx.x / tiles, r0 = (blockIdx.x - bh * tiles) * GT;
  const int b = bh / a.heads, h = bh - b * a.heads;
  const int nq = seq_len(a.q_lens, b, a.nq), nk = r0 < nq ? seq_len(a.kv_lens, b, a.nk) : 0;
  const int ty = threadIdx.x >> 4, tx = threadIdx.x & 15;
  const T* kp = head_of<T>(k, b, h);
  const T* vp = head_of<T>(v, b, h);
  load_tile<T, D>(sQ, head_of<T>(q, b, h), q.st, r0, nq);
  float m[4], l[4], acc[4][CPT];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    m[i] = -INFINITY;
    l[i] = 0.0f;
#pragma unroll
    for (int c = 0; c < CPT; ++c) acc[i][c] = 0.0f;
  }
  for (int c0 = 0; c0 < nk; c0 += GT) {
    __syncthreads();
    load_tile<T, D>(sK, kp, k.st, c0, nk);
    load_tile<T, D>(sV, vp, v.st, c0, nk);
    __syncthreads();
    float s[4][4];
    product_rows<D>(s, sQ, sK, ty, tx);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      float top = -INFINITY;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        s[i][j] = c0 + tx + 16 * j < nk ? s[i][j] * a.scale : -INFINITY;
        top = fmaxf(top, s[i][j]);
      }
      const float m_new = fmaxf(m[i], half_warp_max(top));
      const float ref = m_new == -INFINITY ? 0.0f : m_new;  // a row of -inf so far: exp(-inf - 0) = 0
      const float f = expf(m[i] - ref);
      m[i] = m_new;
      l[i] *= f;  // this thread's columns; joined over the row at the end
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float p = expf(s[i][j] - ref);
        l[i] += p;
        sP[(4 * ty + i) * LDP + tx + 16 * j] = p;
      }
#pragma unroll
      for (int c = 0; c < CPT; ++c) acc[i][c] *= f;
    }
    __syncthreads();
    product_sum<D, CPT>(acc, sP, sV, ty, tx);
  }
  T* op = head_of<T>(out, b, h);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int row = r0 + 4 * ty + i;
    const float sum = half_warp_sum(l[i]);
    if (row >= a.nq) continue;
    const bool live = row < nq && sum != 0.0f;
    const float inv = live ? 1.0f / sum : 0.0f;
    if (tx == 0) lse[static_cast<size_t>(bh) * a.nq + row] = live ? m[i] + logf(sum) : -INFINITY;
#pragma unroll
    for (int c = 0; c < CPT; ++c)
      if (CPT * tx + c < D) store1(op + row * out.st + CPT * tx + c, live ? acc[i][c] * inv : 0.0f);
  }
}

// dq and delta: a block owns 64 queries and streams the keys.
template <class T, int D>
__global__ void __launch_bounds__(G_THREADS)
    k_attn_dq_simt(AttnShape a, HeadsView q, HeadsView k, HeadsView v, HeadsView out, const float* __restrict__ lse,
                   HeadsView d_out, HeadsView dq, float* __restrict__ delta) {
  extern __shared__ float sm[];
  constexpr int CPT = cols_per_thread<D>;
  float* sQ = sm;
  float* sG = sQ + GT * (D + 4);
  float* sK = sG + GT * (D + 4);
  float* sV = sK + GT * (D + 4);
  float* sP = sV + GT * (D + 4);
  const int tiles = (a.nq + GT - 1) / GT;
  const int bh = blockIdx.x / tiles, r0 = (blockIdx.x - bh * tiles) * GT;
  const int b = bh / a.heads, h = bh - b * a.heads;
  const int nq = seq_len(a.q_lens, b, a.nq), nk = r0 < nq ? seq_len(a.kv_lens, b, a.nk) : 0;
  const int ty = threadIdx.x >> 4, tx = threadIdx.x & 15;
  const T* kp = head_of<T>(k, b, h);
  const T* vp = head_of<T>(v, b, h);
  load_tile<T, D>(sQ, head_of<T>(q, b, h), q.st, r0, nq);
  load_tile<T, D>(sG, head_of<T>(d_out, b, h), d_out.st, r0, nq);
  load_tile<T, D>(sK, head_of<T>(out, b, h), out.st, r0, nq);  // for delta only
  __syncthreads();
  float ref[4], dl[4], acc[4][CPT];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int row = r0 + 4 * ty + i;
    float x = 0.0f;
    for (int c = tx; c < D; c += 16) x = fmaf(sG[(4 * ty + i) * (D + 4) + c], sK[(4 * ty + i) * (D + 4) + c], x);
    dl[i] = half_warp_sum(x);
    const float e = row < nq ? lse[static_cast<size_t>(bh) * a.nq + row] : 0.0f;
    ref[i] = e == -INFINITY ? 0.0f : e;  // such a row has scores of -inf only: exp(-inf - 0) = 0
    if (tx == 0 && row < a.nq) delta[static_cast<size_t>(bh) * a.nq + row] = dl[i];
#pragma unroll
    for (int c = 0; c < CPT; ++c) acc[i][c] = 0.0f;
  }
  for (int c0 = 0; c0 < nk; c0 += GT) {
    __syncthreads();
    load_tile<T, D>(sK, kp, k.st, c0, nk);
    load_tile<T, D>(sV, vp, v.st, c0, nk);
    __syncthreads();
    float s[4][4], dp[4][4];
    product_rows<D>(s, sQ, sK, ty, tx);
    product_rows<D>(dp, sG, sV, ty, tx);
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float p = c0 + tx + 16 * j < nk ? expf(fmaf(s[i][j], a.scale, -ref[i])) : 0.0f;
        sP[(4 * ty + i) * LDP + tx + 16 * j] = p * (dp[i][j] - dl[i]);
      }
    __syncthreads();
    product_sum<D, CPT>(acc, sP, sK, ty, tx);
  }
  T* dqp = head_of<T>(dq, b, h);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int row = r0 + 4 * ty + i;
    if (row >= a.nq) continue;
#pragma unroll
    for (int c = 0; c < CPT; ++c)
      if (CPT * tx + c < D) store1(dqp + row * dq.st + CPT * tx + c, row < nq ? acc[i][c] * a.scale : 0.0f);
  }
}

// dk and dv: a block owns 64 keys and streams the queries.
template <class T, int D>
__global__ void __launch_bounds__(G_THREADS)
    k_attn_dkdv_simt(AttnShape a, HeadsView q, HeadsView k, HeadsView v, const float* __restrict__ lse, HeadsView d_out,
                     HeadsView dk, HeadsView dv, const float* __restrict__ delta) {
  extern __shared__ float sm[];
  constexpr int CPT = cols_per_thread<D>;
  float* sK = sm;
  float* sV = sK + GT * (D + 4);
  float* sQ = sV + GT * (D + 4);
  float* sG = sQ + GT * (D + 4);
  float* sP = sG + GT * (D + 4);
  float* sD = sP + GT * LDP;
  float* sRef = sD + GT * LDP;
  float* sDelta = sRef + GT;
  const int tiles = (a.nk + GT - 1) / GT;
  const int bh = blockIdx.x / tiles, r0 = (blockIdx.x - bh * tiles) * GT;
  const int b = bh / a.heads, h = bh - b * a.heads;
  const int nk = seq_len(a.kv_lens, b, a.nk), nq = r0 < nk ? seq_len(a.q_lens, b, a.nq) : 0;
  const int ty = threadIdx.x >> 4, tx = threadIdx.x & 15;
  const T* qp = head_of<T>(q, b, h);
  const T* gp = head_of<T>(d_out, b, h);
  load_tile<T, D>(sK, head_of<T>(k, b, h), k.st, r0, nk);
  load_tile<T, D>(sV, head_of<T>(v, b, h), v.st, r0, nk);
  float ak[4][CPT], av[4][CPT];
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int c = 0; c < CPT; ++c) ak[i][c] = av[i][c] = 0.0f;
  for (int c0 = 0; c0 < nq; c0 += GT) {
    __syncthreads();
    load_tile<T, D>(sQ, qp, q.st, c0, nq);
    load_tile<T, D>(sG, gp, d_out.st, c0, nq);
    if (threadIdx.x < GT) {
      const int row = c0 + threadIdx.x;
      const size_t at = static_cast<size_t>(bh) * a.nq + row;
      const float e = row < nq ? lse[at] : 0.0f;
      sRef[threadIdx.x] = e == -INFINITY ? 0.0f : e;
      sDelta[threadIdx.x] = row < nq ? delta[at] : 0.0f;
    }
    __syncthreads();
    float s[4][4], dp[4][4];
    product_rows<D>(s, sK, sQ, ty, tx);
    product_rows<D>(dp, sV, sG, ty, tx);
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int c = tx + 16 * j;
        const float p = c0 + c < nq ? expf(fmaf(s[i][j], a.scale, -sRef[c])) : 0.0f;
        sP[(4 * ty + i) * LDP + c] = p;
        sD[(4 * ty + i) * LDP + c] = p * (dp[i][j] - sDelta[c]);
      }
    __syncthreads();
    product_sum<D, CPT>(av, sP, sG, ty, tx);
    product_sum<D, CPT>(ak, sD, sQ, ty, tx);
  }
  T* dkp = head_of<T>(dk, b, h);
  T* dvp = head_of<T>(dv, b, h);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int row = r0 + 4 * ty + i;
    if (row >= a.nk) continue;
#pragma unroll
    for (int c = 0; c < CPT; ++c)
      if (CPT * tx + c < D) {
        store1(dkp + row * dk.st + CPT * tx + c, row < nk ? ak[i][c] * a.scale : 0.0f);
        store1(dvp + row * dv.st + CPT * tx + c, row < nk ? av[i][c] : 0.0f);
      }
  }
}

template <class T>
__global__ void k_zero_heads(HeadsView x, int heads, int tokens, int dim, int64_t n) {
  for (int64_t i = blockIdx.x * static_cast<int64_t>(blockDim.x) + threadIdx.x; i < n;
       i += static_cast<int64_t>(gridDim.x) * blockDim.x) {
    const int64_t row = i / dim, bh = row / tokens;
    const int64_t b = bh / heads, h = bh - b * heads;
    store1(static_cast<T*>(x.p) + b * x.sb + h * x.sh + (row - bh * tokens) * x.st + (i - row * dim), 0.0f);
  }
}
__global__ void k_fill_f32(float* x, size_t n, float value) {
  for (size_t i = blockIdx.x * static_cast<size_t>(blockDim.x) + threadIdx.x; i < n;
       i += static_cast<size_t>(gridDim.x) * blockDim.x)
    x[i] = value;
}

static int fill_grid(size_t n) {
  const size_t g = (n + 255) / 256, cap = static_cast<size_t>(num_sms()) * 8;
  return static_cast<int>(g < cap ? g : cap);
}

cudaError_t zero_heads(HeadsView x, bool bf16, int batch, int heads, int tokens, int dim, cudaStream_t s) {
  const int64_t n = static_cast<int64_t>(batch) * heads * tokens * dim;
  if (n == 0) return cudaSuccess;
  if (bf16)
    k_zero_heads<__nv_bfloat16><<<fill_grid(n), 256, 0, s>>>(x, heads, tokens, dim, n);
  else
    k_zero_heads<float><<<fill_grid(n), 256, 0, s>>>(x, heads, tokens, dim, n);
  return cudaGetLastError();
}

cudaError_t fill_f32(float* x, size_t n, float value, cudaStream_t s) {
  if (n == 0) return cudaSuccess;
  k_fill_f32<<<fill_grid(n), 256, 0, s>>>(x, n, value);
  return cudaGetLastError();
}

namespace {
template <int D>
constexpr int tile_bytes(int tiles, int squares, int rows) {
  return (tiles * GT * (D + 4) + squares * GT * LDP + rows * GT) * static_cast<int>(sizeof(float));
}

template <class T, int D>
cudaError_t forward(const AttnShape& a, HeadsView q, HeadsView k, HeadsView v, HeadsView out, float* lse,
                    cudaStream_t s) {
  constexpr int bytes = tile_bytes<D>(3, 1, 0);
  auto* fn = k_attn_forward_simt<T, D>;
  const cudaError_t e = ensure_smem_limit(reinterpret_cast<const void*>(fn), bytes);
  if (e != cudaSuccess) return e;
  fn<<<a.batch * a.heads * ((a.nq + GT - 1) / GT), G_THREADS, bytes, s>>>(a, q, k, v, out, lse);
  return cudaGetLastError();
}

template <class T, int D>
cudaError_t backward(const AttnShape& a, HeadsView q, HeadsView k, HeadsView v, HeadsView out, const float* lse,
                     HeadsView d_out, HeadsView dq, HeadsView dk, HeadsView dv, float* delta, cudaStream_t s) {
  constexpr int bytes_q = tile_bytes<D>(4, 1, 0), bytes_k = tile_bytes<D>(4, 2, 2);
  auto* fq = k_attn_dq_simt<T, D>;
  auto* fk = k_attn_dkdv_simt<T, D>;
  cudaError_t e = ensure_smem_limit(reinterpret_cast<const void*>(fq), bytes_q);
  if (e == cudaSuccess) e = ensure_smem_limit(reinterpret_cast<const void*>(fk), bytes_k);
  if (e != cudaSuccess) return e;
  fq<<<a.batch * a.heads * ((a.nq + GT - 1) / GT), G_THREADS, bytes_q, s>>>(a, q, k, v, out, lse, d_out, dq, delta);
  e = cudaGetLastError();
  if (e != cudaSuccess) return e;
  fk<<<a.batch * a.heads * ((a.nk + GT - 1) / GT), G_THREADS, bytes_k, s>>>(a, q, k, v, lse, d_out, dk, dv, delta);
  return cudaGetLastError();
}
}  // namespace

cudaError_t attention_forward_simt(const AttnShape& a, bool bf16, HeadsView q, HeadsView k, HeadsView v, HeadsView out,
                                   float* lse, cudaStream_t s) {
  switch (a.dim) {
    case 8: return bf16 ? forward<__nv_bfloat16, 8>(a, q, k, v, out, lse, s) : forward<float, 8>(a, q, k, v, out, lse, s);
    case 16: return bf16 ? forward<__nv_bfloat16, 16>(a, q, k, v, out, lse, s) : forward<float, 16>(a, q, k, v, out, lse, s);
    case 32: return bf16 ? forward<__nv_bfloat16, 32>(a, q, k, v, out, lse, s) : forward<float, 32>(a, q, k, v, out, lse, s);
    case 64: return bf16 ? forward<__nv_bfloat16, 64>(a, q, k, v, out, lse, s) : forward<float, 64>(a, q, k, v, out, lse, s);
  }
  return cudaErrorInvalidValue;
}

cudaError_t attention_backward_simt(const AttnShape& a, bool bf16, HeadsView q, HeadsView k, HeadsView v, HeadsView out,
                                    const float* lse, HeadsView d_out, HeadsView dq, HeadsView dk, HeadsView dv,
                                    float* delta, cudaStream_t s) {
#define VK_BACKWARD(D)                                                                                    \
  case D:                                                                                                 \
    return bf16 ? backward<__nv_bfloat16, D>(a, q, k, v, out, lse, d_out, dq, dk, dv, delta, s)           \
                : backward<float, D>(a, q, k, v, out, lse, d_out, dq, dk, dv, delta, s)
  switch (a.dim) {
    VK_BACKWARD(8);
    VK_BACKWARD(16);
    VK_BACKWARD(32);
    VK_BACKWARD(64);
  }
#undef VK_BACKWARD
  return cudaErrorInvalidValue;
}

}  // namespace vk
