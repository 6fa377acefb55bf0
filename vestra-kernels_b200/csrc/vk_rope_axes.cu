// vk_rope_axes.cu -- rotary positions over several axes.
//
// Pair i of a head turns its elements (lo, hi) by a = position[axis] * inv[i]:
//   lo' = lo cos a - hi sin a,  hi' = hi cos a + lo sin a
// (the inverse, which is the gradient, with -sin).  HBM-bound: each element is
// read and written once.  A block takes a few tokens, computes their pairs'
// sin and cos once into shared memory and applies them to every head of q and
// k, so the angles cost 1 / (2 heads) of an evaluation per element pair.
//
// Angles are formed and reduced by 2 pi in double precision: an f32 product
// would be off by 2^-24 of the angle itself (2e-4 radians at position 4096).
// The reduced angle is rounded to f32 for sincosf: 2^-24 * pi at most.
#include <cuda_bf16.h>

#include "vk_common.cuh"
#include "vk_internal.h"
#include "vk_train.h"

namespace vk {

namespace {
constexpr int RA_THREADS = 256;

template <int BYTES>
struct RawOf;
template <>
struct RawOf<16> {
  using type = uint4;
};
template <>
struct RawOf<8> {
  using type = uint2;
};
template <>
struct RawOf<4> {
  using type = uint32_t;
};
template <>
struct RawOf<2> {
  using type = uint16_t;
};

__device__ __forceinline__ float to_f32(float x) { return x; }
__device__ __forceinline__ float to_f32(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ void from_f32(float& d, float x) { d = x; }
__device__ __forceinline__ void from_f32(__nv_bfloat16& d, float x) { d = __float2bfloat16_rn(x); }
}  // namespace

template <class T, int VEC>
__global__ void __launch_bounds__(RA_THREADS)
    k_rope_axes(const __grid_constant__ RopePairs pr, HeadsView q, HeadsView qo, HeadsView k, HeadsView ko, int heads,
                int tokens, int head_dim, int axes, bool inverse, const int64_t* __restrict__ positions,
                bool positions_per_batch, int per_block) {
  extern __shared__ float2 turn[];  // [token][pair] (sin, cos)
  const int chunks = (tokens + per_block - 1) / per_block;
  const int b = blockIdx.x / chunks, t0 = (blockIdx.x - b * chunks) * per_block;
  const int nt = min(per_block, tokens - t0);
  const int64_t* pos = positions + (positions_per_batch ? static_cast<int64_t>(b) * tokens + t0 : t0) * axes;
  for (int i = threadIdx.x; i < nt * pr.pairs; i += RA_THREADS) {
    const int t = i / pr.pairs, p = i - t * pr.pairs;
    const double a = static_cast<double>(pos[t * axes + pr.axis[p]]) * pr.inv[p];
    const double n = rint(a * 0.15915494309189535);
    double r = fma(n, -6.283185307179586, a);       // 2 pi = 6.283185307179586 + 2.4492935982947064e-16
    r = fma(n, -2.4492935982947064e-16, r);
    float s, c;
    sincosf(static_cast<float>(r), &s, &c);
    turn[i] = make_float2(inverse ? -s : s, c);
  }
  __syncthreads();
  const HeadsView in = blockIdx.y == 0 ? q : k, out = blockIdx.y == 0 ? qo : ko;
  const T* src = static_cast<const T*>(in.p) + b * in.sb;
  T* dst = static_cast<T*>(out.p) + b * out.sb;
  using Raw = typename RawOf<VEC * sizeof(T)>::type;
  union Piece {
    Raw raw;
    T x[VEC];
    __device__ Piece() {}
  };
  const int units = pr.pairs / VEC;       // per head
  const bool head_inner = in.sh < in.st;  // consecutive threads along the closer rows
  for (int i = threadIdx.x; i < nt * heads * units; i += RA_THREADS) {
    const int row = i / units, p = (i - row * units) * VEC;
    int t, h;
    if (head_inner) {
      t = row / heads;
      h = row - t * heads;
    } else {
      h = row / nt;
      t = row - h * nt;
    }
    const T* s = src + h * in.sh + (t0 + t) * in.st;
    T* d = dst + h * out.sh + (t0 + t) * out.st;
    const int lo = pr.lo[p], hi = pr.hi[p];
    Piece a, c;
    a.raw = *reinterpret_cast<const Raw*>(s + lo);
    c.raw = *reinterpret_cast<const Raw*>(s + hi);
#pragma unroll
    for (int j = 0; j < VEC; ++j) {
      const float2 sc = turn[t * pr.pairs + p + j];
      const float x = to_f32(a.x[j]), y = to_f32(c.x[j]);
      from_f32(a.x[j], fmaf(x, sc.y, -y * sc.x));
      from_f32(c.x[j], fmaf(y, sc.y, x * sc.x));
    }
    *reinterpret_cast<Raw*>(d + lo) = a.raw;
    *reinterpret_cast<Raw*>(d + hi) = c.raw;
  }
  if (pr.rotated < head_dim && in.p != out.p) {
    const int rest = head_dim - pr.rotated;
    for (int i = threadIdx.x; i < nt * heads * rest; i += RA_THREADS) {
      const int row = i / rest, e = pr.rotated + i - row * rest;
      const int h = row / nt, t = row - h * nt;
      dst[h * out.sh + (t0 + t) * out.st + e] = src[h * in.sh + (t0 + t) * in.st + e];
    }
  }
}

template <class T>
static cudaError_t launch_rope(int batch, int heads, int tokens, int head_dim, int axes, const RopePairs& pr,
                               bool inverse, const int64_t* positions, bool per_batch, HeadsView q, HeadsView qo,
                               HeadsView k, HeadsView ko, cudaStream_t s) {
  const int per_block = 4;
  const dim3 grid(batch * ((tokens + per_block - 1) / per_block), k.p != nullptr ? 2 : 1);
  const size_t smem = static_cast<size_t>(per_block) * pr.pairs * sizeof(float2);
#define VK_ROPE(V)                                                                                                \
  k_rope_axes<T, V><<<grid, RA_THREADS, smem, s>>>(pr, q, qo, k, ko, heads, tokens, head_dim, axes, inverse, positions, \
                                                   per_batch, per_block)
  if constexpr (sizeof(T) == 2) {
    if (pr.vec == 8) {
      VK_ROPE(8);
      return cudaGetLastError();
    }
  }
  if (pr.vec >= 4)
    VK_ROPE(4);
  else if (pr.vec == 2)
    VK_ROPE(2);
  else
    VK_ROPE(1);
#undef VK_ROPE
  return cudaGetLastError();
}

cudaError_t rope_axes(bool bf16, int batch, int heads, int tokens, int head_dim, int axes, const RopePairs& pairs,
                      bool inverse, const int64_t* positions, bool positions_per_batch, HeadsView q, HeadsView q_out,
                      HeadsView k, HeadsView k_out, cudaStream_t s) {
  return bf16 ? launch_rope<__nv_bfloat16>(batch, heads, tokens, head_dim, axes, pairs, inverse, positions,
                                           positions_per_batch, q, q_out, k, k_out, s)
              : launch_rope<float>(batch, heads, tokens, head_dim, axes, pairs, inverse, positions, positions_per_batch,
                                   q, q_out, k, k_out, s);
}

}  // namespace vk
