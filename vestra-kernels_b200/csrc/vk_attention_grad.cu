// vk_attention_grad.cu -- attention with row statistics and its backward
// pass on the CUDA cores: f32 elements (f32 arithmetic throughout), and bf16
// elements of the head sizes the tensor-core kernels do not take, of one query
// and of gradients of a few scores.
//
//   s_ij = scale q_i . k_j          lse_i = log sum_j exp s_ij
//   p_ij = exp(s_ij - lse_i)        out_i = sum_j p_ij v_j
//   delta_i = d_out_i . out_i       dp_ij = d_out_i . v_j
//   ds_ij = p_ij (dp_ij - delta_i)
//   dv_j = sum_i p_ij d_out_i       dk_j = scale sum_i ds_ij q_i
//   dq_i = scale sum_j ds_ij k_j
//
// A block owns 16 RM rows (queries for the forward pass and dq, keys for dk
// and dv) and streams the other side in tiles of 64, so every sum has one owner
// and a fixed order: no atomics, the same bits every time.  The price is that
// the backward pass computes s and dp twice (7 products instead of 5).  A few
// queries go without tiles (the kernels named few).
//
// 16 x TX threads hold an RM x 64 / TX piece of each product.  Tiles are f32 in
// shared memory with rows of D + 4 floats, which puts the rows that a warp
// reads at once on different banks.
//
// What bounds it is what shared memory returns: 128 bytes a cycle whether or
// not lanes read the same word, so a thread's RM x CN piece costs RM + CN
// cycles of it for RM CN / 4 of the FMA pipe (4 x 4: 8 for 4, 8 x 8: 16 for
// 16).  Five times 12 heads of 865 x 865 x 64 in f32: forward 8 x 8 325 us
// (35 TFLOP/s of the 74 that the FMA pipe has), 4 x 4 368, 2 x 4 530; backward
// 4 x 4 1206 us (33 TFLOP/s), 4 x 8 in half the threads 1246.  An 8 x 8 piece
// of the backward pass does not leave room for two blocks on an SM.
#include <cuda_bf16.h>

#include <type_traits>

#include "vk_common.cuh"
#include "vk_internal.h"
#include "vk_train.h"

namespace vk {

namespace {
constexpr int GT = 64;          // rows of a streamed tile
constexpr int LDP = GT + 4;     // row of a tile of scores

// Two f32 products and sums in one instruction, each rounded as fmaf rounds.
// (It halves what an 8 x 8 piece issues: 443 us without it against 325.)
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
  return d;
}
__device__ __forceinline__ uint64_t pair(float lo, float hi) {
  uint64_t d;
  asm("mov.b64 %0, {%1, %2};" : "=l"(d) : "f"(lo), "f"(hi));
  return d;
}
__device__ __forceinline__ float2 unpair(uint64_t x) {
  float2 d;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(d.x), "=f"(d.y) : "l"(x));
  return d;
}

__device__ __forceinline__ float4 load4(const float* p) { return *reinterpret_cast<const float4*>(p); }
__device__ __forceinline__ float4 load4(const __nv_bfloat16* p) {
  const uint2 u = *reinterpret_cast<const uint2*>(p);
  const float2 a = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&u.x));
  const float2 b = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&u.y));
  return make_float4(a.x, a.y, b.x, b.y);
}
__device__ __forceinline__ void store1(float* p, float x) { *p = x; }
__device__ __forceinline__ void store4(float* p, float a, float b, float c, float d) {
  *reinterpret_cast<float4*>(p) = make_float4(a, b, c, d);
}
__device__ __forceinline__ void store4(__nv_bfloat16* p, float a, float b, float c, float d) {
  *reinterpret_cast<uint2*>(p) = make_uint2(pack_bf16x2(a, b), pack_bf16x2(c, d));
}
__device__ __forceinline__ void store1(__nv_bfloat16* p, float x) { *p = __float2bfloat16_rn(x); }

template <class T>
__device__ __forceinline__ T* head_of(const HeadsView& v, int b, int h) {
  return static_cast<T*>(v.p) + b * v.sb + h * v.sh;
}

// Rows [r0, r0 + ROWS) of one head into shared memory; rows from n on are zero.
template <class T, int D, int ROWS, int THREADS>
__device__ __forceinline__ void load_tile(float* dst, const T* src, int64_t st, int r0, int n) {
#pragma unroll
  for (int i = 0; i < ROWS * D / 4; i += THREADS) {
    const int idx = i + threadIdx.x;
    if (ROWS * D / 4 % THREADS != 0 && idx >= ROWS * D / 4) break;
    const int row = idx / (D / 4), c = idx % (D / 4) * 4;
    float4 x = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    if (r0 + row < n) x = load4(src + static_cast<int64_t>(r0 + row) * st + c);
    *reinterpret_cast<float4*>(dst + row * (D + 4) + c) = x;
  }
}

// s[i][j] = a[ty + 16 i] . b[tx + TX j]
template <int D, int RM, int TX>
__device__ __forceinline__ void product_rows(float (&s)[RM][GT / TX], const float* a, const float* b, int ty, int tx) {
  constexpr int CN = GT / TX;
#pragma unroll
  for (int i = 0; i < RM; ++i)
#pragma unroll
    for (int j = 0; j < CN; ++j) s[i][j] = 0.0f;
#pragma unroll(RM == 8 ? 2 : 4)
  for (int k = 0; k < D; k += 4) {
    float4 y[CN];
#pragma unroll
    for (int j = 0; j < CN; ++j) y[j] = load4(b + (tx + TX * j) * (D + 4) + k);
#pragma unroll
    for (int i = 0; i < RM; ++i) {
      const float4 x = load4(a + (ty + 16 * i) * (D + 4) + k);
#pragma unroll
      for (int j = 0; j < CN; ++j) {
        s[i][j] = fmaf(x.x, y[j].x, s[i][j]);
        s[i][j] = fmaf(x.y, y[j].y, s[i][j]);
        s[i][j] = fmaf(x.z, y[j].z, s[i][j]);
        s[i][j] = fmaf(x.w, y[j].w, s[i][j]);
      }
    }
  }
}

// A thread's columns of an output row: groups of up to four neighbours, the
// groups 4 TX apart (neighbouring threads read neighbouring addresses).
template <int D, int TX>
struct OutCols {
  static constexpr int N = D >= TX ? D / TX : 1, GROUP = N < 4 ? N : 4;
  float v[N];
  __device__ __forceinline__ static bool any(int tx) { return D >= TX || tx < D; }
  __device__ __forceinline__ static int column(int c, int tx) { return c / GROUP * GROUP * TX + GROUP * tx + c % GROUP; }
  __device__ __forceinline__ void zero() {
#pragma unroll
    for (int c = 0; c < N; ++c) v[c] = 0.0f;
  }
  __device__ __forceinline__ void scale(float f) {
#pragma unroll
    for (int c = 0; c < N; ++c) v[c] *= f;
  }
  template <class T>
  __device__ __forceinline__ void store(T* row, int tx, float f) const {
    if (!any(tx)) return;
#pragma unroll
    for (int g = 0; g < N; g += GROUP) {
      T* p = row + g * TX + GROUP * tx;
      if constexpr (GROUP == 4) {
        store4(p, v[g] * f, v[g + 1] * f, v[g + 2] * f, v[g + 3] * f);
      } else {
#pragma unroll
        for (int c = 0; c < GROUP; ++c) store1(p + c, v[c] * f);
      }
    }
  }
};

// acc[i] += sum_j p[ty + 16 i][j] b[j]
template <int D, int RM, int TX>
__device__ __forceinline__ void product_sum(OutCols<D, TX> (&acc)[RM], const float* p, const float* b, int ty, int tx) {
  using Cols = OutCols<D, TX>;
  if (!Cols::any(tx)) return;
  constexpr int PAIRS = Cols::N / 2;
  uint64_t a2[RM][PAIRS > 0 ? PAIRS : 1];
#pragma unroll
  for (int i = 0; i < RM; ++i)
#pragma unroll
    for (int c = 0; c < PAIRS; ++c) a2[i][c] = pair(acc[i].v[2 * c], acc[i].v[2 * c + 1]);
#pragma unroll(RM == 8 ? 2 : 4)
  for (int j = 0; j < GT; j += 4) {
    float4 x[RM];
#pragma unroll
    for (int i = 0; i < RM; ++i) x[i] = load4(p + (ty + 16 * i) * LDP + j);
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const float* row = b + (j + u) * (D + 4) + Cols::GROUP * tx;
      uint64_t y[PAIRS > 0 ? PAIRS : 1];
      if constexpr (Cols::GROUP == 4) {
#pragma unroll
        for (int g = 0; g < Cols::N; g += 4) {
          const ulonglong2 w = *reinterpret_cast<const ulonglong2*>(row + g * TX);
          y[g / 2] = w.x;
          y[g / 2 + 1] = w.y;
        }
      } else if constexpr (PAIRS == 1) {
        y[0] = *reinterpret_cast<const uint64_t*>(row);
      }
#pragma unroll
      for (int i = 0; i < RM; ++i) {
        const float w = u == 0 ? x[i].x : u == 1 ? x[i].y : u == 2 ? x[i].z : x[i].w;
        if constexpr (PAIRS == 0) {
          acc[i].v[0] = fmaf(w, *row, acc[i].v[0]);
        } else {
          const uint64_t ww = pair(w, w);
#pragma unroll
          for (int c = 0; c < PAIRS; ++c) a2[i][c] = fma2(ww, y[c], a2[i][c]);
        }
      }
    }
  }
#pragma unroll
  for (int i = 0; i < RM; ++i)
#pragma unroll
    for (int c = 0; c < PAIRS; ++c) {
      const float2 v = unpair(a2[i][c]);
      acc[i].v[2 * c] = v.x;
      acc[i].v[2 * c + 1] = v.y;
    }
}

// The streamed tiles a block takes: all, or its share of a cluster's.
struct Share {
  int rank, from, to;
  __device__ __forceinline__ Share(int split, int n) : rank(static_cast<int>(blockIdx.x % split)) {
    const int tiles = (n + GT - 1) / GT, each = (tiles + split - 1) / split;
    from = min(rank * each, tiles) * GT;
    to = min(from + each * GT, n);
  }
};
// The blocks of a cluster join what their shares gave: every thread leaves its
// values in its own block's memory, THREADS floats apart, and block `rank`
// takes up some of the threads' elements from all blocks.
constexpr int MAX_SPLIT = 8;
constexpr int FEW = 4, FEW_MAX = 12;  // queries of a block without tiles, and of a sequence that goes that way
__device__ __forceinline__ float left_by(const float* mine, int rank) {
  float x;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(x) : "r"(mapa_shared(mine, rank)));
  return x;
}
__device__ __forceinline__ void left_by_all(float (&x)[MAX_SPLIT], const float* mine, int split, float none) {
#pragma unroll
  for (int r = 0; r < MAX_SPLIT; ++r) x[r] = r < split ? left_by(mine, r) : none;
}
// Calls fn(i, column, sum) for the elements of this block, summed in the order of the blocks.
template <int D, int TX, int RM, class F>
__device__ __forceinline__ void join_shares(const OutCols<D, TX> (&acc)[RM], float* buf, int rank, int split, F&& fn) {
  using Cols = OutCols<D, TX>;
  constexpr int N = Cols::N, THREADS = 16 * TX;
  static_assert(RM * N * THREADS <= 2 * GT * (D + 4), "buf is two streamed tiles");
  const int tx = threadIdx.x % TX;
  __syncthreads();
  float* mine = buf + threadIdx.x;
#pragma unroll
  for (int e = 0; e < RM * N; ++e) mine[e * THREADS] = acc[e / N].v[e % N];
  cluster_sync();
  const int per = max(1, RM * N / split);
  if (Cols::any(tx))
    for (int e = rank * per; e < min((rank + 1) * per, RM * N); ++e) {
      float x[MAX_SPLIT], sum = 0.0f;
      left_by_all(x, mine + e * THREADS, split, 0.0f);
#pragma unroll
      for (int r = 0; r < MAX_SPLIT; ++r) sum += x[r];
      fn(e / N, Cols::column(e % N, tx), sum);
    }
  cluster_sync();  // until then the others read this block's memory
}

// over the TX threads of a row
template <int TX>
__device__ __forceinline__ float lanes_sum(float x) {
#pragma unroll
  for (int o = TX / 2; o > 0; o >>= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
  return x;
}
template <int TX>
__device__ __forceinline__ float lanes_max(float x) {
#pragma unroll
  for (int o = TX / 2; o > 0; o >>= 1) x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, o));
  return x;
}
}  // namespace

template <class T, int D, int RM, int TX>
__global__ void __launch_bounds__(16 * TX, 2)
    k_attn_forward_simt(AttnShape a, int split, HeadsView q, HeadsView k, HeadsView v, HeadsView out,
                        float* __restrict__ lse) {
  extern __shared__ float sm[];
  constexpr int ROWS = 16 * RM, THREADS = 16 * TX, CN = GT / TX;
  float* sQ = sm;
  float* sK = sQ + ROWS * (D + 4);
  float* sV = sK + GT * (D + 4);
  float* sP = sV + GT * (D + 4);
  const int tiles = (a.nq + ROWS - 1) / ROWS;
  const int tile = blockIdx.x / split, bh = tile / tiles, r0 = (tile - bh * tiles) * ROWS;
  const int b = bh / a.heads, h = bh - b * a.heads;
  const int nq = seq_len(a.q_lens, b, a.nq), nk = r0 < nq ? seq_len(a.kv_lens, b, a.nk) : 0;
  const int ty = threadIdx.x / TX, tx = threadIdx.x % TX;
  const T* kp = head_of<T>(k, b, h);
  const T* vp = head_of<T>(v, b, h);
  load_tile<T, D, ROWS, THREADS>(sQ, head_of<T>(q, b, h), q.st, r0, nq);
  float m[RM], l[RM];
  OutCols<D, TX> acc[RM];
#pragma unroll
  for (int i = 0; i < RM; ++i) {
    m[i] = -INFINITY;
    l[i] = 0.0f;
    acc[i].zero();
  }
  const Share share(split, nk);
  for (int c0 = share.from; c0 < share.to; c0 += GT) {
    __syncthreads();
    load_tile<T, D, GT, THREADS>(sK, kp, k.st, c0, nk);
    load_tile<T, D, GT, THREADS>(sV, vp, v.st, c0, nk);
    __syncthreads();
    float s[RM][CN];
    product_rows<D, RM, TX>(s, sQ, sK, ty, tx);
#pragma unroll
    for (int i = 0; i < RM; ++i) {
      float top = -INFINITY;
#pragma unroll
      for (int j = 0; j < CN; ++j) {
        s[i][j] = c0 + tx + TX * j < nk ? s[i][j] * a.scale : -INFINITY;
        top = fmaxf(top, s[i][j]);
      }
      const float m_new = fmaxf(m[i], lanes_max<TX>(top));
      const float ref = m_new == -INFINITY ? 0.0f : m_new;  // a row of -inf so far: exp(-inf - 0) = 0
      const float f = expf(m[i] - ref);
      m[i] = m_new;
      l[i] *= f;  // this thread's columns; joined over the row at the end
#pragma unroll
      for (int j = 0; j < CN; ++j) {
        const float p = expf(s[i][j] - ref);
        l[i] += p;
        sP[(ty + 16 * i) * LDP + tx + TX * j] = p;
      }
      acc[i].scale(f);
    }
    __syncthreads();
    product_sum<D, RM, TX>(acc, sP, sV, ty, tx);
  }
#pragma unroll
  for (int i = 0; i < RM; ++i) l[i] = lanes_sum<TX>(l[i]);
  T* op = head_of<T>(out, b, h);
  if constexpr (RM <= 4)
    if (split > 1) {
      // every block has its share's maximum, sum and result of each row
      using Cols = OutCols<D, TX>;
      constexpr int N = Cols::N, PER = N + 2;
      static_assert(RM * PER * THREADS <= 2 * GT * (D + 4) + ROWS * LDP, "fits the tiles");
      __syncthreads();
      float* mine = sK + threadIdx.x;
#pragma unroll
      for (int i = 0; i < RM; ++i) {
        mine[i * PER * THREADS] = m[i], mine[(i * PER + 1) * THREADS] = l[i];
#pragma unroll
        for (int c = 0; c < N; ++c) mine[(i * PER + 2 + c) * THREADS] = acc[i].v[c];
      }
      cluster_sync();
      const int per = max(1, RM * N / split);
      for (int e = share.rank * per; e < min((share.rank + 1) * per, RM * N); ++e) {
        const int i = e / N, c = e % N, row = r0 + ty + 16 * i;
        const float* at = mine + i * PER * THREADS;
        float ms[MAX_SPLIT], ls[MAX_SPLIT], x[MAX_SPLIT];
        left_by_all(ms, at, split, -INFINITY);
        left_by_all(ls, at + THREADS, split, 0.0f);
        left_by_all(x, at + (2 + c) * THREADS, split, 0.0f);
        float top = -INFINITY, sum = 0.0f, total = 0.0f;
#pragma unroll
        for (int r = 0; r < MAX_SPLIT; ++r) top = fmaxf(top, ms[r]);
        const float ref = top == -INFINITY ? 0.0f : top;
#pragma unroll
        for (int r = 0; r < MAX_SPLIT; ++r) {
          const float f = expf(ms[r] - ref);
          sum = fmaf(ls[r], f, sum);
          total = fmaf(x[r], f, total);
        }
        if (row >= a.nq) continue;
        const bool live = row < nq && sum != 0.0f;
        if (tx == 0 && c == 0) lse[static_cast<size_t>(bh) * a.nq + row] = live ? top + logf(sum) : -INFINITY;
        if (Cols::any(tx)) store1(op + row * out.st + Cols::column(c, tx), live ? total / sum : 0.0f);
      }
      cluster_sync();  // until then the others read this block's memory
      return;
    }
#pragma unroll
  for (int i = 0; i < RM; ++i) {
    const int row = r0 + ty + 16 * i;
    const float sum = l[i];
    if (row >= a.nq) continue;
    const bool live = row < nq && sum != 0.0f;
    const float inv = live ? 1.0f / sum : 0.0f;
    if (tx == 0) lse[static_cast<size_t>(bh) * a.nq + row] = live ? m[i] + logf(sum) : -INFINITY;
    if (!live) acc[i].zero();  // (a sum of 0 has no values, but 0 * inf)
    acc[i].store(op + row * out.st, tx, inv);
  }
}

// A few queries: nothing is reused but q, which stays in registers, so keys and
// values come straight from memory, D / L of a key's elements in each of L
// lanes.  Every group of L lanes keeps a running maximum, sum and result of its
// own keys; lanes, warps and the cluster's blocks join them in that order.
// Bound by HBM: 1536 heads of one query and 3457 keys, f32, 415 us, the copy
// rate (2618 in tiles of 64 rows); 96 heads 55 us (227).  Four queries a block
// take what the exponentials cost: 96 heads of 7 queries and 3000 keys 139 us
// (202), of 16 270 (204 in tiles, so 12 is the most).
template <class T, int D, int ROWS>
__global__ void __launch_bounds__(256)
    k_attn_forward_few(AttnShape a, int split, HeadsView q, HeadsView k, HeadsView v, HeadsView out,
                       float* __restrict__ lse) {
  constexpr int L = D >= 32 ? 8 : D / 4, V = D / (4 * L), KEYS = 32 / L, WARPS = 8;
  __shared__ float part[WARPS][ROWS][D + 2], whole[ROWS][D + 2];  // maximum, sum, result
  const int tiles = (a.nq + ROWS - 1) / ROWS, tile = blockIdx.x / split, rank = blockIdx.x - tile * split;
  const int bh = tile / tiles, r0 = (tile - bh * tiles) * ROWS, b = bh / a.heads, h = bh - b * a.heads;
  const int nq = min(max(seq_len(a.q_lens, b, a.nq) - r0, 0), ROWS), nk = nq > 0 ? seq_len(a.kv_lens, b, a.nk) : 0;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, lg = lane % L, kg = lane / L;
  const int each = (nk + split - 1) / split, from = min(rank * each, nk), to = min(from + each, nk);
  const T* qp = head_of<T>(q, b, h) + r0 * q.st;
  const T* kp = head_of<T>(k, b, h);
  const T* vp = head_of<T>(v, b, h);
  float4 qv[ROWS][V], acc[ROWS][V], kk[V], vv[V];
  float m[ROWS], l[ROWS];
#pragma unroll
  for (int r = 0; r < ROWS; ++r) {
    m[r] = -INFINITY, l[r] = 0.0f;
#pragma unroll
    for (int i = 0; i < V; ++i) {
      acc[r][i] = qv[r][i] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
      if (r < nq) qv[r][i] = load4(qp + r * q.st + (i * L + lg) * 4);
    }
  }
  auto fetch = [&](int key) {
#pragma unroll
    for (int i = 0; i < V; ++i) {
      kk[i] = vv[i] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
      if (key < to) {
        kk[i] = load4(kp + key * k.st + (i * L + lg) * 4);
        vv[i] = load4(vp + key * v.st + (i * L + lg) * 4);
      }
    }
  };
  fetch(from + warp * KEYS + kg);
  for (int k0 = from + warp * KEYS; k0 < to; k0 += WARPS * KEYS) {
    const bool on = k0 + kg < to;
    float4 kc[V], vc[V];
#pragma unroll
    for (int i = 0; i < V; ++i) kc[i] = kk[i], vc[i] = vv[i];
    fetch(k0 + WARPS * KEYS + kg);
#pragma unroll
    for (int r = 0; r < ROWS; ++r)
      if (r < nq) {
        float s = 0.0f;
#pragma unroll
        for (int i = 0; i < V; ++i)
          s = fmaf(qv[r][i].x, kc[i].x, fmaf(qv[r][i].y, kc[i].y, fmaf(qv[r][i].z, kc[i].z, fmaf(qv[r][i].w, kc[i].w, s))));
        s = lanes_sum<L>(s);
        s = on ? s * a.scale : -INFINITY;
        const float m_new = fmaxf(m[r], s), ref = m_new == -INFINITY ? 0.0f : m_new;
        const float f = expf(m[r] - ref), p = expf(s - ref);
        m[r] = m_new;
        l[r] = fmaf(l[r], f, p);
#pragma unroll
        for (int i = 0; i < V; ++i) {
          acc[r][i].x = fmaf(acc[r][i].x, f, p * vc[i].x), acc[r][i].y = fmaf(acc[r][i].y, f, p * vc[i].y);
          acc[r][i].z = fmaf(acc[r][i].z, f, p * vc[i].z), acc[r][i].w = fmaf(acc[r][i].w, f, p * vc[i].w);
        }
      }
  }
#pragma unroll
  for (int r = 0; r < ROWS; ++r) {
#pragma unroll
    for (int o = L; o < 32; o *= 2) {
      const float tm = __shfl_xor_sync(0xffffffffu, m[r], o), m_new = fmaxf(m[r], tm);
      const float ref = m_new == -INFINITY ? 0.0f : m_new, f = expf(m[r] - ref), tf = expf(tm - ref);
      m[r] = m_new;
      l[r] = l[r] * f + __shfl_xor_sync(0xffffffffu, l[r], o) * tf;
#pragma unroll
      for (int i = 0; i < V; ++i) {
        acc[r][i].x = acc[r][i].x * f + __shfl_xor_sync(0xffffffffu, acc[r][i].x, o) * tf;
        acc[r][i].y = acc[r][i].y * f + __shfl_xor_sync(0xffffffffu, acc[r][i].y, o) * tf;
        acc[r][i].z = acc[r][i].z * f + __shfl_xor_sync(0xffffffffu, acc[r][i].z, o) * tf;
        acc[r][i].w = acc[r][i].w * f + __shfl_xor_sync(0xffffffffu, acc[r][i].w, o) * tf;
      }
    }
    if (kg == 0) {
      float* mine = part[warp][r];
      if (lg == 0) mine[0] = m[r], mine[1] = l[r];
#pragma unroll
      for (int i = 0; i < V; ++i) {
        float* d = mine + 2 + (i * L + lg) * 4;
        d[0] = acc[r][i].x, d[1] = acc[r][i].y, d[2] = acc[r][i].z, d[3] = acc[r][i].w;
      }
    }
  }
  __syncthreads();
  const int r = threadIdx.x / D, d = threadIdx.x - r * D;
  float top = -INFINITY, sum = 0.0f, total = 0.0f;
  auto join = [&](const float (&ms)[8], const float (&ls)[8], const float (&xs)[8]) {
    top = -INFINITY, sum = total = 0.0f;
#pragma unroll
    for (int w = 0; w < 8; ++w) top = fmaxf(top, ms[w]);
    const float ref = top == -INFINITY ? 0.0f : top;
#pragma unroll
    for (int w = 0; w < 8; ++w) {
      const float f = expf(ms[w] - ref);
      sum = fmaf(ls[w], f, sum);
      total = fmaf(xs[w], f, total);
    }
  };
  static_assert(WARPS == 8 && MAX_SPLIT == 8 && ROWS * D <= 256, "an element per thread, eight parts each");
  if (r < ROWS) {
    float ms[8], ls[8], xs[8];
#pragma unroll
    for (int w = 0; w < 8; ++w) ms[w] = part[w][r][0], ls[w] = part[w][r][1], xs[w] = part[w][r][2 + d];
    join(ms, ls, xs);
    if (split > 1) {
      whole[r][2 + d] = total;
      if (d == 0) whole[r][0] = top, whole[r][1] = sum;
    }
  }
  if (split > 1) {
    cluster_sync();
    if (r < ROWS && rank == 0) {
      float ms[8], ls[8], xs[8];
      left_by_all(ms, &whole[r][0], split, -INFINITY);
      left_by_all(ls, &whole[r][1], split, 0.0f);
      left_by_all(xs, &whole[r][2 + d], split, 0.0f);
      join(ms, ls, xs);
    }
    cluster_sync();  // until then the others' memory is read
    if (rank != 0) return;
  }
  if (r >= ROWS || r0 + r >= a.nq) return;
  const bool live = r < nq && sum != 0.0f;
  store1(head_of<T>(out, b, h) + (r0 + r) * out.st + d, live ? total / sum : 0.0f);
  if (d == 0) lse[static_cast<size_t>(bh) * a.nq + r0 + r] = live ? top + logf(sum) : -INFINITY;
}

// dq and delta: a block owns 16 RM queries and streams the keys.
template <class T, int D, int RM, int TX>
__global__ void __launch_bounds__(16 * TX, 2)
    k_attn_dq_simt(AttnShape a, int split, HeadsView q, HeadsView k, HeadsView v, HeadsView out, const float* __restrict__ lse,
                   HeadsView d_out, HeadsView dq, float* __restrict__ delta) {
  extern __shared__ float sm[];
  constexpr int ROWS = 16 * RM, THREADS = 16 * TX, CN = GT / TX;
  float* sQ = sm;
  float* sG = sQ + ROWS * (D + 4);
  float* sK = sG + ROWS * (D + 4);
  float* sV = sK + GT * (D + 4);
  float* sP = sV + GT * (D + 4);
  const int tiles = (a.nq + ROWS - 1) / ROWS;
  const int tile = blockIdx.x / split, bh = tile / tiles, r0 = (tile - bh * tiles) * ROWS;
  const int b = bh / a.heads, h = bh - b * a.heads;
  const int nq = seq_len(a.q_lens, b, a.nq), nk = r0 < nq ? seq_len(a.kv_lens, b, a.nk) : 0;
  const int ty = threadIdx.x / TX, tx = threadIdx.x % TX;
  const T* kp = head_of<T>(k, b, h);
  const T* vp = head_of<T>(v, b, h);
  load_tile<T, D, ROWS, THREADS>(sQ, head_of<T>(q, b, h), q.st, r0, nq);
  load_tile<T, D, ROWS, THREADS>(sG, head_of<T>(d_out, b, h), d_out.st, r0, nq);
  load_tile<T, D, ROWS, THREADS>(sK, head_of<T>(out, b, h), out.st, r0, nq);  // for delta only
  __syncthreads();
  float ref[RM], dl[RM];
  OutCols<D, TX> acc[RM];
#pragma unroll
  for (int i = 0; i < RM; ++i) {
    const int row = r0 + ty + 16 * i;
    float x = 0.0f;
    for (int c = tx; c < D; c += TX) x = fmaf(sG[(ty + 16 * i) * (D + 4) + c], sK[(ty + 16 * i) * (D + 4) + c], x);
    dl[i] = lanes_sum<TX>(x);
    const float e = row < nq ? lse[static_cast<size_t>(bh) * a.nq + row] : 0.0f;
    ref[i] = e == -INFINITY ? 0.0f : e;  // such a row has scores of -inf only: exp(-inf - 0) = 0
    if (tx == 0 && row < a.nq && blockIdx.x % split == 0) delta[static_cast<size_t>(bh) * a.nq + row] = dl[i];
    acc[i].zero();
  }
  const Share share(split, nk);
  for (int c0 = share.from; c0 < share.to; c0 += GT) {
    __syncthreads();
    load_tile<T, D, GT, THREADS>(sK, kp, k.st, c0, nk);
    load_tile<T, D, GT, THREADS>(sV, vp, v.st, c0, nk);
    __syncthreads();
    float s[RM][CN], dp[RM][CN];
    product_rows<D, RM, TX>(s, sQ, sK, ty, tx);
    product_rows<D, RM, TX>(dp, sG, sV, ty, tx);
#pragma unroll
    for (int i = 0; i < RM; ++i)
#pragma unroll
      for (int j = 0; j < CN; ++j) {
        const float p = c0 + tx + TX * j < nk ? expf(fmaf(s[i][j], a.scale, -ref[i])) : 0.0f;
        sP[(ty + 16 * i) * LDP + tx + TX * j] = p * (dp[i][j] - dl[i]);
      }
    __syncthreads();
    product_sum<D, RM, TX>(acc, sP, sK, ty, tx);
  }
  T* dqp = head_of<T>(dq, b, h);
  if (split > 1) {
    join_shares(acc, sK, share.rank, split, [&](int i, int col, float sum) {
      const int row = r0 + ty + 16 * i;
      if (row < a.nq) store1(dqp + row * dq.st + col, row < nq ? sum * a.scale : 0.0f);
    });
    return;
  }
#pragma unroll
  for (int i = 0; i < RM; ++i) {
    const int row = r0 + ty + 16 * i;
    if (row >= a.nq) continue;
    if (row >= nq) acc[i].zero();
    acc[i].store(dqp + row * dq.st, tx, a.scale);
  }
}

// dk and dv: a block owns 16 RM keys and streams the queries.
template <class T, int D, int RM, int TX>
__global__ void __launch_bounds__(16 * TX, 2)
    k_attn_dkdv_simt(AttnShape a, int split, HeadsView q, HeadsView k, HeadsView v, const float* __restrict__ lse, HeadsView d_out,
                     HeadsView dk, HeadsView dv, const float* __restrict__ delta) {
  extern __shared__ float sm[];
  constexpr int ROWS = 16 * RM, THREADS = 16 * TX, CN = GT / TX;
  float* sK = sm;
  float* sV = sK + ROWS * (D + 4);
  float* sQ = sV + ROWS * (D + 4);
  float* sG = sQ + GT * (D + 4);
  float* sP = sG + GT * (D + 4);
  float* sD = sP + ROWS * LDP;
  float* sRef = sD + ROWS * LDP;
  float* sDelta = sRef + GT;
  const int tiles = (a.nk + ROWS - 1) / ROWS;
  const int tile = blockIdx.x / split, bh = tile / tiles, r0 = (tile - bh * tiles) * ROWS;
  const int b = bh / a.heads, h = bh - b * a.heads;
  const int nk = seq_len(a.kv_lens, b, a.nk), nq = r0 < nk ? seq_len(a.q_lens, b, a.nq) : 0;
  const int ty = threadIdx.x / TX, tx = threadIdx.x % TX;
  const T* qp = head_of<T>(q, b, h);
  const T* gp = head_of<T>(d_out, b, h);
  load_tile<T, D, ROWS, THREADS>(sK, head_of<T>(k, b, h), k.st, r0, nk);
  load_tile<T, D, ROWS, THREADS>(sV, head_of<T>(v, b, h), v.st, r0, nk);
  OutCols<D, TX> ak[RM], av[RM];
#pragma unroll
  for (int i = 0; i < RM; ++i)
    ak[i].zero(), av[i].zero();
  const Share share(split, nq);
  for (int c0 = share.from; c0 < share.to; c0 += GT) {
    __syncthreads();
    load_tile<T, D, GT, THREADS>(sQ, qp, q.st, c0, nq);
    load_tile<T, D, GT, THREADS>(sG, gp, d_out.st, c0, nq);
    if (threadIdx.x < GT) {
      const int row = c0 + threadIdx.x;
      const size_t at = static_cast<size_t>(bh) * a.nq + row;
      const float e = row < nq ? lse[at] : 0.0f;
      sRef[threadIdx.x] = e == -INFINITY ? 0.0f : e;
      sDelta[threadIdx.x] = row < nq ? delta[at] : 0.0f;
    }
    __syncthreads();
    float s[RM][CN], dp[RM][CN];
    product_rows<D, RM, TX>(s, sK, sQ, ty, tx);
    product_rows<D, RM, TX>(dp, sV, sG, ty, tx);
#pragma unroll
    for (int i = 0; i < RM; ++i)
#pragma unroll
      for (int j = 0; j < CN; ++j) {
        const int c = tx + TX * j;
        const float p = c0 + c < nq ? expf(fmaf(s[i][j], a.scale, -sRef[c])) : 0.0f;
        sP[(ty + 16 * i) * LDP + c] = p;
        sD[(ty + 16 * i) * LDP + c] = p * (dp[i][j] - sDelta[c]);
      }
    __syncthreads();
    product_sum<D, RM, TX>(av, sP, sG, ty, tx);
    product_sum<D, RM, TX>(ak, sD, sQ, ty, tx);
  }
  T* dkp = head_of<T>(dk, b, h);
  T* dvp = head_of<T>(dv, b, h);
  if (split > 1) {
    join_shares(ak, sQ, share.rank, split, [&](int i, int col, float sum) {
      const int row = r0 + ty + 16 * i;
      if (row < a.nk) store1(dkp + row * dk.st + col, row < nk ? sum * a.scale : 0.0f);
    });
    join_shares(av, sQ, share.rank, split, [&](int i, int col, float sum) {
      const int row = r0 + ty + 16 * i;
      if (row < a.nk) store1(dvp + row * dv.st + col, row < nk ? sum : 0.0f);
    });
    return;
  }
#pragma unroll
  for (int i = 0; i < RM; ++i) {
    const int row = r0 + ty + 16 * i;
    if (row >= a.nk) continue;
    if (row >= nk) ak[i].zero(), av[i].zero();
    ak[i].store(dkp + row * dk.st, tx, a.scale);
    av[i].store(dvp + row * dv.st, tx, 1.0f);
  }
}

// The gradients of a few queries, in one pass: a key's dk and dv belong to the
// lanes that read it, dq is the cluster's sum.  Bound by HBM as the forward
// form is: 1536 heads of one query and 3457 keys, f32, 968 us, 86% of the copy
// rate (8886 in tiles of 64 rows); 96 heads 110 (642); 96 heads of 4 queries and
// 3000 keys 161 (554).
template <class T, int D, int ROWS>
__global__ void __launch_bounds__(256)
    k_attn_backward_few(AttnShape a, int split, HeadsView q, HeadsView k, HeadsView v, HeadsView out,
                        const float* __restrict__ lse, HeadsView d_out, HeadsView dq, HeadsView dk, HeadsView dv,
                        float* __restrict__ delta) {
  constexpr int L = D >= 32 ? 8 : D / 4, V = D / (4 * L), KEYS = 32 / L, WARPS = 8;
  __shared__ float part[WARPS][ROWS][D], whole[ROWS][D];  // dq
  const int bh = blockIdx.x / split, rank = blockIdx.x - bh * split, b = bh / a.heads, h = bh - b * a.heads;
  const int nq = min(seq_len(a.q_lens, b, a.nq), ROWS), nk = nq > 0 ? seq_len(a.kv_lens, b, a.nk) : 0;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, lg = lane % L, kg = lane / L;
  const int each = (a.nk + split - 1) / split, from = min(rank * each, a.nk), to = min(from + each, a.nk), end = min(to, nk);
  const T* qp = head_of<T>(q, b, h);
  const T* gp = head_of<T>(d_out, b, h);
  const T* op = head_of<T>(out, b, h);
  const T* kp = head_of<T>(k, b, h);
  const T* vp = head_of<T>(v, b, h);
  T* dkp = head_of<T>(dk, b, h);
  T* dvp = head_of<T>(dv, b, h);
  auto dot = [](const float4 (&x)[V], const float4 (&y)[V]) {
    float s = 0.0f;
#pragma unroll
    for (int i = 0; i < V; ++i)
      s = fmaf(x[i].x, y[i].x, fmaf(x[i].y, y[i].y, fmaf(x[i].z, y[i].z, fmaf(x[i].w, y[i].w, s))));
    return lanes_sum<L>(s);
  };
  auto add = [](float4 (&x)[V], float w, const float4 (&y)[V]) {
#pragma unroll
    for (int i = 0; i < V; ++i) {
      x[i].x = fmaf(w, y[i].x, x[i].x), x[i].y = fmaf(w, y[i].y, x[i].y);
      x[i].z = fmaf(w, y[i].z, x[i].z), x[i].w = fmaf(w, y[i].w, x[i].w);
    }
  };
  float4 qv[ROWS][V], gv[ROWS][V], acc[ROWS][V], kk[V], vv[V];
  float ref[ROWS], dl[ROWS];
#pragma unroll
  for (int r = 0; r < ROWS; ++r) {
    float4 o[V];
    ref[r] = 0.0f;
#pragma unroll
    for (int i = 0; i < V; ++i) {
      acc[r][i] = qv[r][i] = gv[r][i] = o[i] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
      if (r < nq) {
        const int at = (i * L + lg) * 4;
        qv[r][i] = load4(qp + r * q.st + at);
        gv[r][i] = load4(gp + r * d_out.st + at);
        o[i] = load4(op + r * out.st + at);
      }
    }
    dl[r] = dot(gv[r], o);
    if (r < nq) {
      const float e = lse[static_cast<size_t>(bh) * a.nq + r];
      ref[r] = e == -INFINITY ? 0.0f : e;  // such a row has scores of -inf only: exp(-inf - 0) = 0
    }
    if (rank == 0 && threadIdx.x == 0 && r < a.nq) delta[static_cast<size_t>(bh) * a.nq + r] = dl[r];
  }
  auto fetch = [&](int key) {
#pragma unroll
    for (int i = 0; i < V; ++i) {
      kk[i] = vv[i] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
      if (key < end) {
        kk[i] = load4(kp + key * k.st + (i * L + lg) * 4);
        vv[i] = load4(vp + key * v.st + (i * L + lg) * 4);
      }
    }
  };
  fetch(from + warp * KEYS + kg);
  for (int k0 = from + warp * KEYS; k0 < to; k0 += WARPS * KEYS) {
    const int key = k0 + kg;
    float4 kc[V], vc[V], gk[V], gvv[V];
#pragma unroll
    for (int i = 0; i < V; ++i) {
      kc[i] = kk[i], vc[i] = vv[i];
      gk[i] = gvv[i] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    }
    fetch(key + WARPS * KEYS);
#pragma unroll
    for (int r = 0; r < ROWS; ++r)
      if (r < nq) {
        const float s = dot(qv[r], kc), dp = dot(gv[r], vc);
        // (As weights of 0, keys past the end would turn what is not finite in q
        // or d_out into NaN; so would zeros in the place of the next share's
        // keys, where exp(-lse) is infinite.)
        if (key < end) {
          const float p = expf(fmaf(s, a.scale, -ref[r])), ds = p * (dp - dl[r]);
          add(gvv, p, gv[r]);
          add(gk, ds, qv[r]);
          add(acc[r], ds, kc);
        }
      }
    if (key < to) {
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const int at = (i * L + lg) * 4;
        store4(dkp + key * dk.st + at, gk[i].x * a.scale, gk[i].y * a.scale, gk[i].z * a.scale, gk[i].w * a.scale);
        store4(dvp + key * dv.st + at, gvv[i].x, gvv[i].y, gvv[i].z, gvv[i].w);
      }
    }
  }
#pragma unroll
  for (int r = 0; r < ROWS; ++r)
#pragma unroll
    for (int i = 0; i < V; ++i) {
      float x[4] = {acc[r][i].x, acc[r][i].y, acc[r][i].z, acc[r][i].w};
#pragma unroll
      for (int e = 0; e < 4; ++e) {
#pragma unroll
        for (int o = L; o < 32; o *= 2) x[e] += __shfl_xor_sync(0xffffffffu, x[e], o);
        if (kg == 0) part[warp][r][(i * L + lg) * 4 + e] = x[e];
      }
    }
  __syncthreads();
  const int r = threadIdx.x / D, d = threadIdx.x - r * D;
  static_assert(ROWS * D <= 256, "an element per thread");
  float total = 0.0f;
  if (r < ROWS) {
#pragma unroll
    for (int w = 0; w < WARPS; ++w) total += part[w][r][d];
    whole[r][d] = total;
  }
  if (split > 1) {
    cluster_sync();
    if (r < ROWS && rank == 0) {
      float xs[MAX_SPLIT];
      left_by_all(xs, &whole[r][d], split, 0.0f);
      total = 0.0f;
#pragma unroll
      for (int w = 0; w < MAX_SPLIT; ++w) total += xs[w];
    }
    cluster_sync();  // until then the others' memory is read
    if (rank != 0) return;
  }
  if (r < ROWS && r < a.nq) store1(head_of<T>(dq, b, h) + r * dq.st + d, r < nq ? total * a.scale : 0.0f);
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
// `own` tiles of 16 RM rows, `streamed` ones of 64, `scores` of 16 RM x 64, `rows` vectors of 64
template <int D, int RM>
constexpr int tile_bytes(int own, int streamed, int scores, int rows) {
  return ((own * 16 * RM + streamed * GT) * (D + 4) + scores * 16 * RM * LDP + rows * GT) * static_cast<int>(sizeof(float));
}
int blocks_of(const AttnShape& a, int tokens, int rows) { return a.batch * a.heads * ((tokens + rows - 1) / rows); }

template <class... P, class... A>
cudaError_t launch(void (*fn)(P...), int tiles, int split, int threads, int bytes, cudaStream_t s, A... args) {
  cudaError_t e = ensure_smem_limit(reinterpret_cast<const void*>(fn), bytes);
  if (e != cudaSuccess) return e;
  cudaLaunchAttribute cluster{};
  cluster.id = cudaLaunchAttributeClusterDimension;
  cluster.val.clusterDim.x = split, cluster.val.clusterDim.y = cluster.val.clusterDim.z = 1;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(tiles * split);
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = bytes;
  cfg.stream = s;
  cfg.attrs = &cluster;
  cfg.numAttrs = split > 1 ? 1 : 0;
  e = cudaLaunchKernelEx(&cfg, fn, args...);
  const cudaError_t last = cudaGetLastError();
  return e == cudaSuccess ? last : e;
}

// How a product of `own` rows per head with `streamed` ones is laid out: 16 rm
// rows per block, the streamed rows split over a cluster of `split` blocks.
//
// 8 (forward only) where the SM with the most rows has no more of them than
// with 4: 36 heads of 865 tokens 214 against 247 us, but 12 heads of 3457, 1243
// against 1180.  With fewer blocks than SMs the streamed side is split: up to
// four blocks for three SMs (12 heads of 197 tokens backward 48 us split by 2,
// 43 by 4), and up to two an SM where a share still has two tiles (18 heads of
// 197 by 2, 49, by 4, 64) or where lengths make many blocks short (18 heads of
// up to 197, 48 and 43).  6 heads of 433 tokens forward 41 us in one piece, 24
// split by 4; 12 heads of 100 queries and 3000 keys, 231 and 58 by 8.  2 for a
// few rows: 8 heads of 20 queries and 3000 keys of 32, 147 us with 64 rows in
// one block, 20 with 32, split by 8.  With one to two blocks an SM the streamed
// side is split where that takes an eighth off the busiest SM's tiles: 12 heads
// of 865 tokens forward 124 and 105, backward 413 and 336, but 36 heads of 433
// (252 blocks) 64 and 85 if split.
struct Layout {
  int rm, split;
};
Layout layout_of(const AttnShape& a, int own, int streamed, bool wide) {
  const int sms = num_sms(), n8 = blocks_of(a, own, 128), n4 = blocks_of(a, own, 64);
  if (wide && n8 > sms && (n8 + sms - 1) / sms * 2 <= (n4 + sms - 1) / sms) return {8, 1};
  const int tiles = (streamed + GT - 1) / GT;
  int split = 1;
  if (n4 >= sms) {
    if (n4 < 2 * sms) {
      int most = 2 * tiles;  // tiles of the busiest SM
      for (int s = 2; s <= MAX_SPLIT && s <= tiles; s *= 2) {
        const int now = (n4 * s + sms - 1) / sms * ((tiles + s - 1) / s);
        if (now * 8 <= most * 7) split = s, most = now;
      }
    }
    return {4, split};
  }
  const int rm = own <= 32 ? 2 : 4;
  const bool lens = a.q_lens != nullptr || a.kv_lens != nullptr;
  while (split < MAX_SPLIT && split * 2 <= tiles &&
         (n4 * split * 2 <= sms + sms / 3 || (n4 * split <= sms && (lens || split * 4 <= tiles))))
    split *= 2;
  return {rm, split};
}

// Of a form without tiles: four blocks an SM, 64 keys a block at least.
int few_split(int tiles, int keys) {
  int split = 1;
  while (split < MAX_SPLIT && static_cast<int64_t>(tiles) * split * 2 <= 4 * num_sms() && split * 128 <= keys) split *= 2;
  return split;
}

template <class T, int D>
cudaError_t forward(const AttnShape& a, HeadsView q, HeadsView k, HeadsView v, HeadsView out, float* lse,
                    cudaStream_t s) {
  if (a.nq == 1) {
    const int tiles = blocks_of(a, 1, 1), split = few_split(tiles, a.nk);
    return launch(k_attn_forward_few<T, D, 1>, tiles, split, 256, 0, s, a, split, q, k, v, out, lse);
  }
  if constexpr (D == 64 && std::is_same_v<T, __nv_bfloat16>) {
    return cudaErrorInvalidValue;  // the tensor cores take them
  } else {
    if (a.nq <= FEW_MAX) {
      const int tiles = blocks_of(a, a.nq, FEW), split = few_split(tiles, a.nk);
      return launch(k_attn_forward_few<T, D, FEW>, tiles, split, 256, 0, s, a, split, q, k, v, out, lse);
    }
    const Layout l = layout_of(a, a.nq, a.nk, true);
    const int tiles = blocks_of(a, a.nq, 16 * l.rm);
    if (l.rm == 8)
      return launch(k_attn_forward_simt<T, D, 8, 8>, tiles, 1, 128, tile_bytes<D, 8>(1, 2, 1, 0), s, a, 1, q, k, v, out, lse);
    if (l.rm == 4)
      return launch(k_attn_forward_simt<T, D, 4, 16>, tiles, l.split, 256, tile_bytes<D, 4>(1, 2, 1, 0), s, a, l.split, q, k,
                    v, out, lse);
    return launch(k_attn_forward_simt<T, D, 2, 16>, tiles, l.split, 256, tile_bytes<D, 2>(1, 2, 1, 0), s, a, l.split, q, k, v,
                  out, lse);
  }
}

template <class T, int D, int RM>
cudaError_t backward_dq(int split, const AttnShape& a, HeadsView q, HeadsView k, HeadsView v, HeadsView out,
                        const float* lse, HeadsView d_out, HeadsView dq, float* delta, cudaStream_t s) {
  return launch(k_attn_dq_simt<T, D, RM, 16>, blocks_of(a, a.nq, 16 * RM), split, 256, tile_bytes<D, RM>(2, 2, 1, 0), s, a,
                split, q, k, v, out, lse, d_out, dq, delta);
}
template <class T, int D, int RM>
cudaError_t backward_dkdv(int split, const AttnShape& a, HeadsView q, HeadsView k, HeadsView v, const float* lse,
                          HeadsView d_out, HeadsView dk, HeadsView dv, const float* delta, cudaStream_t s) {
  return launch(k_attn_dkdv_simt<T, D, RM, 16>, blocks_of(a, a.nk, 16 * RM), split, 256, tile_bytes<D, RM>(2, 2, 2, 2), s,
                a, split, q, k, v, lse, d_out, dk, dv, delta);
}
template <class T, int D>
cudaError_t backward(const AttnShape& a, HeadsView q, HeadsView k, HeadsView v, HeadsView out, const float* lse,
                     HeadsView d_out, HeadsView dq, HeadsView dk, HeadsView dv, float* delta, cudaStream_t s) {
  if (a.nq <= FEW) {
    const int heads = a.batch * a.heads, split = few_split(heads, a.nk);
    return a.nq == 1 ? launch(k_attn_backward_few<T, D, 1>, heads, split, 256, 0, s, a, split, q, k, v, out, lse, d_out, dq,
                              dk, dv, delta)
                     : launch(k_attn_backward_few<T, D, FEW>, heads, split, 256, 0, s, a, split, q, k, v, out, lse, d_out, dq,
                              dk, dv, delta);
  }
  Layout l = layout_of(a, a.nq, a.nk, false);
  const cudaError_t e = l.rm == 4 ? backward_dq<T, D, 4>(l.split, a, q, k, v, out, lse, d_out, dq, delta, s)
                                  : backward_dq<T, D, 2>(l.split, a, q, k, v, out, lse, d_out, dq, delta, s);
  if (e != cudaSuccess) return e;
  l = layout_of(a, a.nk, a.nq, false);
  return l.rm == 4 ? backward_dkdv<T, D, 4>(l.split, a, q, k, v, lse, d_out, dk, dv, delta, s)
                   : backward_dkdv<T, D, 2>(l.split, a, q, k, v, lse, d_out, dk, dv, delta, s);
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
