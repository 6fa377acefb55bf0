// vk_rope_axes.cu -- rotary positions over several axes.
//
// Pair i of a head turns its elements (lo, hi) by a = position[axis] * inv[i]:
//   lo' = lo cos a - hi sin a,  hi' = hi cos a + lo sin a
// (the inverse, which is the gradient, with -sin).  HBM-bound: each element is
// read and written once, and an angle is computed once for all heads of q and
// k.  A thread keeps the angles of a few pairs of one token and goes along the
// heads, three at a time.  16 clips of 3457 tokens, 12 heads of 64 each for q
// and k in bf16: 64 us, 5.3 TB/s; with four heads at a time 68, with two 68,
// with blocks of 256 threads 65, with the angles of a few tokens in shared
// memory and the threads along the heads 123.
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
constexpr int RA_THREADS = 128;
constexpr int RA_BATCH = 3;

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

// The angles of one pair of one token: (sin, cos).
__device__ __forceinline__ float2 rope_turn(int64_t position, double inv, bool inverse) {
  const double a = static_cast<double>(position) * inv;
  const double n = rint(a * 0.15915494309189535);
  double r = fma(n, -6.283185307179586, a);  // 2 pi = 6.283185307179586 + 2.4492935982947064e-16
  r = fma(n, -2.4492935982947064e-16, r);
  float s, c;
  sincosf(static_cast<float>(r), &s, &c);
  return make_float2(inverse ? -s : s, c);
}

// A thread has VEC consecutive pairs of one token, keeps their sin and cos in
// registers and takes them through a share of the heads of q and of k.
template <class T, int VEC>
__global__ void __launch_bounds__(RA_THREADS)
    k_rope_axes(const __grid_constant__ RopePairs pr, HeadsView q, HeadsView qo, HeadsView k, HeadsView ko, int heads,
                int share, int64_t rows, int units, int head_dim, int axes, bool inverse,
                const int64_t* __restrict__ positions, bool positions_per_batch, FastDiv by_units, FastDiv by_tokens,
                int tokens) {
  using Raw = typename RawOf<VEC * sizeof(T)>::type;
  union Piece {
    Raw raw;
    T x[VEC];
    __device__ Piece() {}
  };
  const int64_t i = static_cast<int64_t>(blockIdx.x) * RA_THREADS + threadIdx.x;
  if (i >= rows * units) return;
  const int row = by_units(static_cast<int>(i)), p = (static_cast<int>(i) - row * units) * VEC;
  const int b = by_tokens(row), t = row - b * tokens;
  const int h0 = blockIdx.y * share, h1 = min(heads, h0 + share);
  float2 sc[VEC];
  if (p < pr.pairs) {
    const int64_t* pos = positions + (positions_per_batch ? static_cast<int64_t>(row) : t) * axes;
#pragma unroll
    for (int j = 0; j < VEC; ++j) sc[j] = rope_turn(pos[pr.axis[p + j]], pr.inv[p + j], inverse);
  }
  for (int which = 0; which < (k.p != nullptr ? 2 : 1); ++which) {
    const HeadsView &in = which ? k : q, &out = which ? ko : qo;
    const T* s = static_cast<const T*>(in.p) + b * in.sb + t * in.st + h0 * in.sh;
    T* d = static_cast<T*>(out.p) + b * out.sb + t * out.st + h0 * out.sh;
    if (p >= pr.pairs) {  // the units past the pairs copy what is not rotated
      if (in.p != out.p)
        for (int h = h0; h < h1; ++h, s += in.sh, d += out.sh)
          for (int e = pr.rotated + (p - pr.pairs) / VEC; e < head_dim; e += units - pr.pairs / VEC) d[e] = s[e];
      continue;
    }
    const int lo = pr.lo[p], hi = pr.hi[p];
    for (int h = h0; h < h1; h += RA_BATCH, s += RA_BATCH * in.sh, d += RA_BATCH * out.sh) {
      Piece x[RA_BATCH], y[RA_BATCH];
#pragma unroll
      for (int u = 0; u < RA_BATCH; ++u)
        if (h + u < h1) {
          x[u].raw = *reinterpret_cast<const Raw*>(s + u * in.sh + lo);
          y[u].raw = *reinterpret_cast<const Raw*>(s + u * in.sh + hi);
        }
#pragma unroll
      for (int u = 0; u < RA_BATCH; ++u)
        if (h + u < h1) {
#pragma unroll
          for (int j = 0; j < VEC; ++j) {
            const float a = to_f32(x[u].x[j]), c = to_f32(y[u].x[j]);
            from_f32(x[u].x[j], fmaf(a, sc[j].y, -c * sc[j].x));
            from_f32(y[u].x[j], fmaf(c, sc[j].y, a * sc[j].x));
          }
          *reinterpret_cast<Raw*>(d + u * out.sh + lo) = x[u].raw;
          *reinterpret_cast<Raw*>(d + u * out.sh + hi) = y[u].raw;
        }
    }
  }
}

template <class T>
static cudaError_t launch_rope(int batch, int heads, int tokens, int head_dim, int axes, const RopePairs& pr,
                               bool inverse, const int64_t* positions, bool per_batch, HeadsView q, HeadsView qo,
                               HeadsView k, HeadsView ko, cudaStream_t s) {
  const int64_t rows = static_cast<int64_t>(batch) * tokens;
  // (elements that are only copied get threads of their own, 8 each)
  const int units = pr.pairs / pr.vec + (head_dim - pr.rotated + 7) / 8;
  const int64_t blocks = (rows * units + RA_THREADS - 1) / RA_THREADS;
  // The heads are split over blocks until every SM has four: a split computes
  // its angles again.
  int splits = 1;
  while (splits * RA_BATCH < heads && blocks * splits < 4 * num_sms()) ++splits;
  const int share = (heads + splits - 1) / splits;
  const dim3 grid(static_cast<unsigned>(blocks), (heads + share - 1) / share);
  const FastDiv by_units(units), by_tokens(tokens);
#define VK_ROPE(V)                                                                                                     \
  k_rope_axes<T, V><<<grid, RA_THREADS, 0, s>>>(pr, q, qo, k, ko, heads, share, rows, units, head_dim, axes, inverse,  \
                                                positions, per_batch, by_units, by_tokens, tokens)
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
