// vk_residual_norm.cu -- the residual step between two norms and its
// gradients, each in one pass over the rows:
//   n = branch or LN(branch; post),  h = x + scale gate n,  y = LN(h)
// Backward, with y^ = (h - mean) rstd and t = d_y gamma:
//   dh = d_h + rstd (t - <t> - y^ <t y^>)          (<>: mean over the row)
//   d_x = dh,  d_n = dh scale gate,  d_branch = d_n or through the post norm
//   column sums: d_gamma = sum d_y y^, d_beta = sum d_y, P = sum dh n per
//   group (d_scale = sum_groups gate P, d_gate = scale P), and the post norm's.
// Both are HBM-bound: at 768 columns, f32 stream and bf16 branch, 9.2 KB a row
// forward and 13.8 KB backward.  Rows live in registers; sums are f32.  What
// holds them back is the load and store path (three quarters busy when the
// vectors of a row were read as 16-byte halves) and the wait for a row, so
// eight f32 move at once and the next row is fetched while this one is worked
// on.  55,360 rows of that kind: forward 134 us with neither, 125 with the
// fetch, 105 with both (4.9 TB/s); backward 176, 156, 146 (5.2 TB/s).
// Three rows on their way through shared memory took what L1 has for the
// vectors: 153 and 193 us.  The five [cols] vectors in shared memory, 107.
//
// The column sums are split over blocks that own consecutive rows of one
// group and join in a second small kernel in a fixed order: no atomics, the
// same bits every time.
#include <cuda_bf16.h>

#include <algorithm>
#include <initializer_list>

#include "vk_common.cuh"
#include "vk_internal.h"
#include "vk_train.h"

namespace vk {

namespace {
constexpr int RN_BLOCK = 256;
// Values a thread may have of a row for the next row to be fetched while this
// one is worked on: above it the registers run out.
constexpr int RN_AHEAD = 24;

__device__ __forceinline__ float warp_total(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// VEC (8 or 1) consecutive values as they lie in memory.  Eight f32 go as one
// 32-byte access: as two of 16, each would use half of the lines it touches.
template <class T, int VEC>
struct Lanes {
  static constexpr int WORDS = VEC * sizeof(T) >= 4 ? VEC * sizeof(T) / 4 : 1;
  uint32_t w[WORDS];
  __device__ __forceinline__ void load(const T* p) {
    if constexpr (WORDS == 8) {
      asm volatile("ld.global.v8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
                   : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]), "=r"(w[4]), "=r"(w[5]), "=r"(w[6]), "=r"(w[7])
                   : "l"(__cvta_generic_to_global(p)));
    } else if constexpr (WORDS == 4) {
      const uint4 u = *reinterpret_cast<const uint4*>(p);
      w[0] = u.x, w[1] = u.y, w[2] = u.z, w[3] = u.w;
    } else if constexpr (sizeof(T) == 4) {
      w[0] = __float_as_uint(*reinterpret_cast<const float*>(p));
    } else {
      w[0] = *reinterpret_cast<const uint16_t*>(p);
    }
  }
  __device__ __forceinline__ void get(float (&d)[VEC]) const {
    if constexpr (sizeof(T) == 4) {
#pragma unroll
      for (int i = 0; i < VEC; ++i) d[i] = __uint_as_float(w[i]);
    } else if constexpr (VEC == 8) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        d[2 * i] = __uint_as_float(w[i] << 16);
        d[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
      }
    } else {
      d[0] = __uint_as_float(w[0] << 16);
    }
  }
};
template <int VEC>
__device__ __forceinline__ void get(float (&d)[VEC], const float* p) {
  Lanes<float, VEC> l;
  l.load(p);
  l.get(d);
}
template <int VEC>
__device__ __forceinline__ void put(float* p, const float (&d)[VEC]) {
  if constexpr (VEC == 8) {
    asm volatile("st.global.v8.f32 [%8], {%0,%1,%2,%3,%4,%5,%6,%7};" ::"f"(d[0]), "f"(d[1]), "f"(d[2]), "f"(d[3]),
                 "f"(d[4]), "f"(d[5]), "f"(d[6]), "f"(d[7]), "l"(__cvta_generic_to_global(p))
                 : "memory");
  } else {
    *p = d[0];
  }
}
template <int VEC>
__device__ __forceinline__ void put(__nv_bfloat16* p, const float (&d)[VEC]) {
  if constexpr (VEC == 8) {
    *reinterpret_cast<uint4*>(p) = make_uint4(pack_bf16x2(d[0], d[1]), pack_bf16x2(d[2], d[3]), pack_bf16x2(d[4], d[5]),
                                              pack_bf16x2(d[6], d[7]));
  } else {
    *p = __float2bfloat16_rn(d[0]);
  }
}
}  // namespace

// T threads per row, RN_BLOCK / T rows per block, NV vectors of VEC columns
// per thread.
template <class XT, class BT, int VEC, int T, int NV>
__global__ void __launch_bounds__(RN_BLOCK)
    k_residual_norm(ResidualNorm r, unsigned rows, FastDiv by_group, const XT* x, const BT* __restrict__ branch, XT* h, BT* y,
                    float* __restrict__ stats, float* __restrict__ post_stats) {
  constexpr int ROWS = RN_BLOCK / T, WARPS = T / 32;
  constexpr bool AHEAD = VEC * NV <= RN_AHEAD;
  __shared__ float part[4][RN_BLOCK / 32];
  const int in_row = threadIdx.x % T, slot = threadIdx.x / T;
  // sum over the T threads of a row; `which` names a slot of its own per call
  auto row_total = [&](float v, int which) {
    v = warp_total(v);
    if constexpr (WARPS == 1) return v;
    if ((threadIdx.x & 31) == 0) part[which][threadIdx.x >> 5] = v;
    __syncthreads();
    float s = 0.0f;
#pragma unroll
    for (int w = 0; w < WARPS; ++w) s += part[which][slot * WARPS + w];
    return s;
  };
  const float inv_cols = 1.0f / static_cast<float>(r.cols);
  Lanes<XT, VEC> raw_x[NV];
  Lanes<BT, VEC> raw_b[NV];
  int col[NV];
#pragma unroll
  for (int j = 0; j < NV; ++j) col[j] = (j * T + in_row) * VEC;
  auto fetch = [&](unsigned row) {
#pragma unroll
    for (int j = 0; j < NV; ++j)
      if (row < rows && col[j] < r.cols) {
        raw_b[j].load(branch + static_cast<size_t>(row) * r.cols + col[j]);
        raw_x[j].load(x + static_cast<size_t>(row) * r.cols + col[j]);
      }
  };
  if (AHEAD) fetch(blockIdx.x * ROWS + slot);
  // (the rows of a block go in step: its sums meet in shared memory)
  for (unsigned row0 = blockIdx.x * ROWS; row0 < rows; row0 += gridDim.x * ROWS) {
    const unsigned row = row0 + slot;
    if (!AHEAD) fetch(row);
    const bool live = row < rows;
    const size_t base = static_cast<size_t>(live ? row : 0) * r.cols;
    const float* gate = r.gate != nullptr && live ? r.gate + static_cast<size_t>(by_group(row)) * r.cols : nullptr;
    float n[NV][VEC], v[NV][VEC];
    bool has[NV];
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      has[j] = live && col[j] < r.cols;
#pragma unroll
      for (int e = 0; e < VEC; ++e) n[j][e] = v[j][e] = 0.0f;
      if (has[j]) {
        raw_b[j].get(n[j]);
        raw_x[j].get(v[j]);
      }
    }
    if (AHEAD) fetch(row + gridDim.x * ROWS);
    auto mean_rstd = [&](float (&u)[NV][VEC], int which) {
      float s = 0.0f;
#pragma unroll
      for (int j = 0; j < NV; ++j)
#pragma unroll
        for (int e = 0; e < VEC; ++e) s += u[j][e];
      const float mean = row_total(s, which) * inv_cols;
      float q = 0.0f;
#pragma unroll
      for (int j = 0; j < NV; ++j)
        if (has[j])
#pragma unroll
          for (int e = 0; e < VEC; ++e) q = fmaf(u[j][e] - mean, u[j][e] - mean, q);
      const float var = row_total(q, which + 1) * inv_cols;
      return make_float2(mean, 1.0f / sqrtf(var + r.eps));
    };
    if (r.post_gamma != nullptr) {
      const float2 mr = mean_rstd(n, 0);
      if (live && in_row == 0) *reinterpret_cast<float2*>(post_stats + 2 * static_cast<size_t>(row)) = mr;
#pragma unroll
      for (int j = 0; j < NV; ++j)
        if (has[j]) {
          float g[VEC], b[VEC];
          get<VEC>(g, r.post_gamma + col[j]);
          get<VEC>(b, r.post_beta + col[j]);
#pragma unroll
          for (int e = 0; e < VEC; ++e) n[j][e] = fmaf((n[j][e] - mr.x) * mr.y, g[e], b[e]);
        }
    }
#pragma unroll
    for (int j = 0; j < NV; ++j)
      if (has[j]) {
        float f[VEC];
        if (r.scale != nullptr) {
          get<VEC>(f, r.scale + col[j]);
#pragma unroll
          for (int e = 0; e < VEC; ++e) n[j][e] *= f[e];
        }
        if (gate != nullptr) {
          get<VEC>(f, gate + col[j]);
#pragma unroll
          for (int e = 0; e < VEC; ++e) n[j][e] *= f[e];
        }
#pragma unroll
        for (int e = 0; e < VEC; ++e) v[j][e] += n[j][e];
        put<VEC>(h + base + col[j], v[j]);
      }
    const float2 mr = mean_rstd(v, 2);
    if (live && in_row == 0) *reinterpret_cast<float2*>(stats + 2 * static_cast<size_t>(row)) = mr;
#pragma unroll
    for (int j = 0; j < NV; ++j)
      if (has[j]) {
        float g[VEC], b[VEC];
        get<VEC>(g, r.gamma + col[j]);
        get<VEC>(b, r.beta + col[j]);
#pragma unroll
        for (int e = 0; e < VEC; ++e) v[j][e] = fmaf((v[j][e] - mr.x) * mr.y, g[e], b[e]);
        put<VEC>(y + base + col[j], v[j]);
      }
    if constexpr (WARPS > 1) __syncthreads();  // before the next row's sums
  }
}

namespace {
// How the rows split into the blocks of the backward pass: `per_group` blocks
// of `rows` consecutive rows in each of `groups` groups (one group when there
// is no gate: only its gradient needs them apart).
struct Chunks {
  int groups, group_rows, rows, per_group;
  __host__ __device__ int count() const { return groups * per_group; }
};
Chunks chunks_of(const ResidualNorm& r) {
  Chunks c;
  c.groups = r.gate != nullptr ? r.groups : 1;
  c.group_rows = r.gate != nullptr ? r.rows_per_group : r.groups * r.rows_per_group;
  // five blocks per SM, what is resident at 768 columns (at other widths and
  // with a gate some places stay empty or some blocks start late), but at least
  // four rows each: a chunk writes its column sums once however few rows it has
  const int64_t want = static_cast<int64_t>(num_sms()) * 5;
  const int64_t total = static_cast<int64_t>(c.groups) * c.group_rows;
  int64_t rows = (total + want - 1) / want;
  if (rows < 4) rows = 4;
  if (rows > c.group_rows) rows = c.group_rows;
  c.rows = static_cast<int>(rows);
  c.per_group = static_cast<int>((c.group_rows + rows - 1) / rows);
  return c;
}
// Quantities summed over rows: d_gamma, d_beta, then P and the post norm's two where needed.
struct Sums {
  int p, post, count;
};
Sums sums_of(const ResidualNorm& r) {
  Sums s{-1, -1, 2};
  if (r.scale != nullptr || r.gate != nullptr) s.p = s.count++;
  if (r.post_gamma != nullptr) {
    s.post = s.count;
    s.count += 2;
  }
  return s;
}
}  // namespace

size_t residual_norm_workspace(const ResidualNorm& r) {
  return static_cast<size_t>(chunks_of(r).count()) * sums_of(r).count * r.cols * sizeof(float);
}

// One block per chunk of rows, blockDim.x threads per row, one row at a time.
template <class XT, class BT, int VEC, int NV>
__global__ void __launch_bounds__(RN_BLOCK)
    k_residual_norm_backward(ResidualNorm r, Chunks ck, Sums sm, const XT* d_h, const BT* d_y,
                             const XT* __restrict__ h, const BT* __restrict__ branch, const float* __restrict__ stats,
                             const float* __restrict__ post_stats, XT* d_x, BT* d_branch, float* __restrict__ part) {
  __shared__ float2 red[2][RN_BLOCK / 32];
  const int T = blockDim.x, warps = T >> 5;
  const int group = blockIdx.x / ck.per_group, chunk = blockIdx.x - group * ck.per_group;
  const int64_t first = static_cast<int64_t>(group) * ck.group_rows + static_cast<int64_t>(chunk) * ck.rows;
  const int nrows = min(ck.rows, ck.group_rows - chunk * ck.rows);
  const float inv_cols = 1.0f / static_cast<float>(r.cols);
  int flip = 0;
  auto row_totals = [&](float a, float b) {  // (sum a, sum b) over the block
    a = warp_total(a);
    b = warp_total(b);
    if ((threadIdx.x & 31) == 0) red[flip][threadIdx.x >> 5] = make_float2(a, b);
    __syncthreads();
    float2 s = make_float2(0.0f, 0.0f);
    for (int w = 0; w < warps; ++w) {
      s.x += red[flip][w].x;
      s.y += red[flip][w].y;
    }
    flip ^= 1;  // the next write goes to the other slot: one barrier per sum
    return s;
  };
  float sg[NV][VEC], sb[NV][VEC], sp[NV][VEC], spg[NV][VEC], spb[NV][VEC];
  float fac[NV][VEC];  // scale * gate of this group
  int col[NV];
  bool has[NV];
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    col[j] = (j * T + threadIdx.x) * VEC;
    has[j] = col[j] < r.cols;
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
      sg[j][e] = sb[j][e] = sp[j][e] = spg[j][e] = spb[j][e] = 0.0f;
      fac[j][e] = 1.0f;
    }
    if (has[j]) {
      float f[VEC];
      if (r.scale != nullptr) get<VEC>(fac[j], r.scale + col[j]);
      if (r.gate != nullptr) {
        get<VEC>(f, r.gate + static_cast<size_t>(group) * r.cols + col[j]);
#pragma unroll
        for (int e = 0; e < VEC; ++e) fac[j][e] *= f[e];
      }
    }
  }
  Lanes<BT, VEC> raw_t[NV], raw_n[NV];
  Lanes<XT, VEC> raw_h[NV], raw_d[NV];
  float2 mr_next = make_float2(0.0f, 0.0f), pr_next = mr_next;
  auto fetch = [&](int i) {
    if (i >= nrows) return;
    const size_t row = static_cast<size_t>(first + i), base = row * r.cols;
#pragma unroll
    for (int j = 0; j < NV; ++j)
      if (has[j]) {
        raw_t[j].load(d_y + base + col[j]);
        raw_h[j].load(h + base + col[j]);
        raw_n[j].load(branch + base + col[j]);
        if (d_h != nullptr) raw_d[j].load(d_h + base + col[j]);
      }
    mr_next = *reinterpret_cast<const float2*>(stats + 2 * row);
    if (sm.post >= 0) pr_next = *reinterpret_cast<const float2*>(post_stats + 2 * row);
  };
  constexpr bool AHEAD = VEC * NV <= RN_AHEAD;
  if (AHEAD) fetch(0);
  for (int i = 0; i < nrows; ++i) {
    if (!AHEAD) fetch(i);
    const size_t row = static_cast<size_t>(first + i), base = row * r.cols;
    const float2 mr = mr_next, pr = pr_next;
    float t[NV][VEC], hat[NV][VEC], dh[NV][VEC], n[NV][VEC];
    float s0 = 0.0f, s1 = 0.0f;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
#pragma unroll
      for (int e = 0; e < VEC; ++e) t[j][e] = hat[j][e] = dh[j][e] = n[j][e] = 0.0f;
      if (has[j]) {
        raw_t[j].get(t[j]);
        raw_h[j].get(hat[j]);
        raw_n[j].get(n[j]);
        if (d_h != nullptr) raw_d[j].get(dh[j]);
      }
    }
    if (AHEAD) fetch(i + 1);
#pragma unroll
    for (int j = 0; j < NV; ++j)
      if (has[j]) {
        float g[VEC];
        get<VEC>(g, r.gamma + col[j]);
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
          hat[j][e] = (hat[j][e] - mr.x) * mr.y;
          sg[j][e] = fmaf(t[j][e], hat[j][e], sg[j][e]);
          sb[j][e] += t[j][e];
          t[j][e] *= g[e];
          s0 += t[j][e];
          s1 = fmaf(t[j][e], hat[j][e], s1);
        }
      }
    const float2 tot = row_totals(s0, s1);
    const float m0 = tot.x * inv_cols, m1 = tot.y * inv_cols;
    s0 = s1 = 0.0f;
#pragma unroll
    for (int j = 0; j < NV; ++j)
      if (has[j]) {
#pragma unroll
        for (int e = 0; e < VEC; ++e) dh[j][e] = fmaf(mr.y, t[j][e] - m0 - hat[j][e] * m1, dh[j][e]);
        put<VEC>(d_x + base + col[j], dh[j]);
        if (sm.post >= 0) {
          float g[VEC], b[VEC];
          get<VEC>(g, r.post_gamma + col[j]);
          get<VEC>(b, r.post_beta + col[j]);
#pragma unroll
          for (int e = 0; e < VEC; ++e) {
            n[j][e] = (n[j][e] - pr.x) * pr.y;  // b^
            sp[j][e] = fmaf(dh[j][e], fmaf(n[j][e], g[e], b[e]), sp[j][e]);
            const float d = dh[j][e] * fac[j][e];
            spg[j][e] = fmaf(d, n[j][e], spg[j][e]);
            spb[j][e] += d;
            t[j][e] = d * g[e];
            s0 += t[j][e];
            s1 = fmaf(t[j][e], n[j][e], s1);
          }
        } else {
#pragma unroll
          for (int e = 0; e < VEC; ++e) {
            sp[j][e] = fmaf(dh[j][e], n[j][e], sp[j][e]);
            t[j][e] = dh[j][e] * fac[j][e];
          }
          put<VEC>(d_branch + base + col[j], t[j]);
        }
      }
    if (sm.post >= 0) {
      const float2 pt = row_totals(s0, s1);
      const float p0 = pt.x * inv_cols, p1 = pt.y * inv_cols;
#pragma unroll
      for (int j = 0; j < NV; ++j)
        if (has[j]) {
#pragma unroll
          for (int e = 0; e < VEC; ++e) t[j][e] = pr.y * (t[j][e] - p0 - n[j][e] * p1);
          put<VEC>(d_branch + base + col[j], t[j]);
        }
    }
  }
  const size_t step = static_cast<size_t>(gridDim.x) * r.cols;  // part [sum][chunk][cols]
  float* mine = part + static_cast<size_t>(blockIdx.x) * r.cols;
#pragma unroll
  for (int j = 0; j < NV; ++j)
    if (has[j]) {
      put<VEC>(mine + col[j], sg[j]);
      put<VEC>(mine + step + col[j], sb[j]);
      if (sm.p >= 0) put<VEC>(mine + sm.p * step + col[j], sp[j]);
      if (sm.post >= 0) {
        put<VEC>(mine + sm.post * step + col[j], spg[j]);
        put<VEC>(mine + (sm.post + 1) * step + col[j], spb[j]);
      }
    }
}

// Joins the chunks' column sums: a block of 32 x 32 threads takes 32 columns
// of one quantity, each row of threads every 32nd chunk, then a fixed tree.
// Quantities past the sums are the groups of d_gate.
__global__ void __launch_bounds__(1024)
    k_residual_norm_join(ResidualNorm r, Chunks ck, Sums sm, const float* __restrict__ part, ResidualNormGrads g,
                         int col_blocks) {
  __shared__ float tree[32][33];
  const int what = blockIdx.x / col_blocks;
  const int lane = threadIdx.x & 31, lot = threadIdx.x >> 5;
  const int col = (blockIdx.x - what * col_blocks) * 32 + lane;
  const int count = ck.count();
  const bool of_group = what >= sm.count;
  const int q = of_group ? sm.p : what;
  const int from = of_group ? (what - sm.count) * ck.per_group : 0, to = of_group ? from + ck.per_group : count;
  const bool weighted = q == sm.p && !of_group && r.gate != nullptr;
  float s = 0.0f;
  if (col < r.cols) {
    const float* p = part + static_cast<size_t>(q) * count * r.cols + col;
    if (weighted) {
#pragma unroll 4
      for (int c = from + lot; c < to; c += 32)
        s = fmaf(p[static_cast<size_t>(c) * r.cols], r.gate[static_cast<size_t>(c / ck.per_group) * r.cols + col], s);
    } else {
#pragma unroll 8
      for (int c = from + lot; c < to; c += 32) s += p[static_cast<size_t>(c) * r.cols];
    }
  }
  tree[lot][lane] = s;
  __syncthreads();
  s = warp_total(tree[lane][lot]);  // column `lot` of this block
  const int c = (blockIdx.x - what * col_blocks) * 32 + lot;
  if (lane != 0 || c >= r.cols) return;
  if (of_group)
    g.d_gate[static_cast<size_t>(what - sm.count) * r.cols + c] = r.scale != nullptr ? s * r.scale[c] : s;
  else if (q == 0)
    g.d_gamma[c] = s;
  else if (q == 1)
    g.d_beta[c] = s;
  else if (q == sm.p) {
    if (g.d_scale != nullptr) g.d_scale[c] = s;
  } else if (q == sm.post)
    g.d_post_gamma[c] = s;
  else
    g.d_post_beta[c] = s;
}

namespace {
// (a row of f32 is read 32 bytes at a time)
bool aligned32(std::initializer_list<const void*> ps) {
  for (const void* p : ps)
    if (reinterpret_cast<uintptr_t>(p) % 32 != 0) return false;
  return true;
}

// Blocks that are resident at once, at most `want`.
template <class F>
int resident_grid(F* fn, int want) {
  int* per_sm = per_device_slot(reinterpret_cast<const void*>(fn));
  if (*per_sm == 0 && (cudaOccupancyMaxActiveBlocksPerMultiprocessor(per_sm, fn, RN_BLOCK, 0) != cudaSuccess || *per_sm < 1))
    *per_sm = 1;
  return std::min(want, *per_sm * num_sms());
}

template <class XT, class BT>
cudaError_t forward(const ResidualNorm& r, const void* x, const void* branch, void* h, void* y, float* stats,
                    float* post_stats, cudaStream_t s) {
  const int rows = r.groups * r.rows_per_group;
  const bool wide = r.cols % 8 == 0 && aligned32({x, branch, h, y, r.gamma, r.beta, r.scale, r.gate, r.post_gamma, r.post_beta});
#define VK_RN(VEC, T, NV)                                                                                          \
  k_residual_norm<XT, BT, VEC, T, NV>                                                                              \
      <<<resident_grid(k_residual_norm<XT, BT, VEC, T, NV>, (rows - 1) / (RN_BLOCK / T) + 1), RN_BLOCK, 0,           \
         s>>>(r, rows, FastDiv(r.rows_per_group), static_cast<const XT*>(x), static_cast<const BT*>(branch),       \
              static_cast<XT*>(h), static_cast<BT*>(y), stats, post_stats)
  if (wide) {
    const int v = r.cols / 8;
    if (v <= 32)
      VK_RN(8, 32, 1);
    else if (v <= 64)
      VK_RN(8, 32, 2);
    else if (v <= 96)
      VK_RN(8, 32, 3);
    else if (v <= 128)
      VK_RN(8, 32, 4);
    else if (v <= 256)
      VK_RN(8, 128, 2);
    else if (v <= 512)
      VK_RN(8, 128, 4);
    else
      VK_RN(8, 256, 4);
  } else if (r.cols <= 128) {
    VK_RN(1, 32, 4);
  } else if (r.cols <= 512) {
    VK_RN(1, 128, 4);
  } else if (r.cols <= 2048) {
    VK_RN(1, 128, 16);
  } else {
    VK_RN(1, 256, 32);
  }
#undef VK_RN
  return cudaGetLastError();
}

template <class XT, class BT>
cudaError_t backward(const ResidualNorm& r, const void* d_h, const void* d_y, const void* h, const void* branch,
                     const float* stats, const float* post_stats, const ResidualNormGrads& g, float* part,
                     cudaStream_t s) {
  const Chunks ck = chunks_of(r);
  const Sums sm = sums_of(r);
  const bool wide = r.cols % 8 == 0 && aligned32({d_h, d_y, h, branch, g.d_x, g.d_branch, r.gamma, r.scale, r.gate,
                                                  r.post_gamma, r.post_beta, part});
  const int vecs = wide ? r.cols / 8 : r.cols;
  const int threads = vecs >= RN_BLOCK ? RN_BLOCK : (vecs + 31) / 32 * 32;
  const int nv = (vecs + threads - 1) / threads;
#define VK_RNB(VEC, NV)                                                                                              \
  k_residual_norm_backward<XT, BT, VEC, NV><<<ck.count(), threads, 0, s>>>(                                          \
      r, ck, sm, static_cast<const XT*>(d_h), static_cast<const BT*>(d_y), static_cast<const XT*>(h),                \
      static_cast<const BT*>(branch), stats, post_stats, static_cast<XT*>(g.d_x), static_cast<BT*>(g.d_branch), part)
  if (wide) {
    if (nv == 1)
      VK_RNB(8, 1);
    else if (nv == 2)
      VK_RNB(8, 2);
    else
      VK_RNB(8, 4);
  } else if (nv == 1) {
    VK_RNB(1, 1);
  } else if (nv <= 4) {
    VK_RNB(1, 4);
  } else if (nv <= 8) {
    VK_RNB(1, 8);
  } else {
    VK_RNB(1, 32);
  }
#undef VK_RNB
  cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return e;
  const int col_blocks = (r.cols + 31) / 32;
  const int what = sm.count + (r.gate != nullptr ? r.groups : 0);
  k_residual_norm_join<<<col_blocks * what, 1024, 0, s>>>(r, ck, sm, part, g, col_blocks);
  return cudaGetLastError();
}
}  // namespace

cudaError_t residual_norm_forward(const ResidualNorm& r, bool stream_bf16, bool branch_bf16, const void* x,
                                  const void* branch, void* h, void* y, float* stats, float* post_stats,
                                  cudaStream_t s) {
  if (stream_bf16) return forward<__nv_bfloat16, __nv_bfloat16>(r, x, branch, h, y, stats, post_stats, s);
  return branch_bf16 ? forward<float, __nv_bfloat16>(r, x, branch, h, y, stats, post_stats, s)
                     : forward<float, float>(r, x, branch, h, y, stats, post_stats, s);
}

cudaError_t residual_norm_backward(const ResidualNorm& r, bool stream_bf16, bool branch_bf16, const void* d_h,
                                   const void* d_y, const void* h, const void* branch, const float* stats,
                                   const float* post_stats, const ResidualNormGrads& g, float* workspace,
                                   cudaStream_t s) {
  if (stream_bf16)
    return backward<__nv_bfloat16, __nv_bfloat16>(r, d_h, d_y, h, branch, stats, post_stats, g, workspace, s);
  return branch_bf16 ? backward<float, __nv_bfloat16>(r, d_h, d_y, h, branch, stats, post_stats, g, workspace, s)
                     : backward<float, float>(r, d_h, d_y, h, branch, stats, post_stats, g, workspace, s);
}

}  // namespace vk
