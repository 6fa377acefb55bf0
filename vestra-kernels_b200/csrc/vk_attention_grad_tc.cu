// vk_attention_grad_tc.cu -- bf16 attention with row statistics and its
// backward pass on the 5th-generation tensor cores, head_dim 64 (the formulas
// are in vk_attention_grad.cu).
//
// Three persistent kernels, one CTA per SM: the forward pass, dq (with delta),
// and dk / dv.  Each CTA owns tiles of 128 rows (queries, queries, keys) and
// streams the other side in blocks of 128 through a TMA ring, so every sum
// has one owner: no atomics, the same bits every time.  The backward pass
// computes s and dp in both of its kernels for that (7 products per block
// instead of 5).
//
//   warp 0       TMA producer
//   warp 1       TMEM owner; lane 0 issues the MMAs
//   warps 2..17  the elementwise work on S (and dP) in TMEM, one row per
//                thread, the columns of a tile split between warps of the
//                same lane quadrant
//
// S and dP are bf16 products in f32.  P and dS are rounded to bf16 for the
// second products (one rounding of 2^-8 at most, next to the one of the
// result); everything else is f32.  Rows and columns past a sequence's length
// never reach a product: scores are masked, and the tail of a streamed tile is
// zeroed in shared memory, because 0 * NaN would spread what lies there.
#include "vk_common.cuh"
#include "vk_internal.h"
#include "vk_train.h"

namespace vk {

namespace {
constexpr int TR = 128;                 // rows of a tile, columns of a block
constexpr int TILE_B = TR * 128;        // bytes of 128 rows of 64 bf16
constexpr int ST = 4;                   // streamed blocks in flight
constexpr int TC_THREADS = 18 * 32;
constexpr float LOG2E = 1.4426950408889634f, LN2 = 0.6931471805599453f;

__device__ __forceinline__ void tma_load_4d(void* dst, const void* desc, uint64_t* bar, int32_t y, int32_t z, int32_t w) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%2, %3, %4, %5}], [%6];" ::"r"(smem_u32(dst)),
      "l"(reinterpret_cast<uint64_t>(desc)), "r"(0), "r"(y), "r"(z), "r"(w), "r"(smem_u32(bar))
      : "memory");
}
__device__ __forceinline__ void tmem_ld16(uint32_t taddr, uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(taddr)
      : "memory");
}

// Zeroes rows [valid, 128) of two tiles that TMA wrote; all lanes of a warp,
// before its MMAs read them.  A swizzled row stays in its own 128 bytes.
__device__ __forceinline__ void zero_tail(uint8_t* a, uint8_t* b, int valid, int lane) {
  for (int i = valid * 8 + lane; i < TR * 8; i += 32) {
    reinterpret_cast<uint4*>(a)[i] = make_uint4(0, 0, 0, 0);
    reinterpret_cast<uint4*>(b)[i] = make_uint4(0, 0, 0, 0);
  }
  fence_proxy_async();
  __syncwarp();
}

__device__ __forceinline__ bool warp_wait(uint64_t* bar, uint32_t parity, int* err, int code) {
  return __all_sync(0xffffffffu, mbar_wait(bar, parity, err, code));
}

__device__ __forceinline__ void store_bf16x16(__nv_bfloat16* p, const float* x, float f) {
  uint4* d = reinterpret_cast<uint4*>(p);
#pragma unroll
  for (int i = 0; i < 2; ++i)
    d[i] = make_uint4(pack_bf16x2(x[8 * i] * f, x[8 * i + 1] * f), pack_bf16x2(x[8 * i + 2] * f, x[8 * i + 3] * f),
                      pack_bf16x2(x[8 * i + 4] * f, x[8 * i + 5] * f), pack_bf16x2(x[8 * i + 6] * f, x[8 * i + 7] * f));
}
__device__ __forceinline__ void store_zero32(__nv_bfloat16* p) {  // 32 bytes
  reinterpret_cast<uint4*>(p)[0] = reinterpret_cast<uint4*>(p)[1] = make_uint4(0, 0, 0, 0);
}

// A reference to subtract from scores of which `top` is the largest so far.
// Where they are all -inf any finite one will do: it keeps 2^(-inf) at 0.
__device__ __forceinline__ float finite_ref(float top) { return top == -INFINITY ? -1e30f : top; }

// 2^x for a pair of lanes: pair `i` of 16 goes to the FMA pipe where MASK says
// so, the others to MUFU.
template <uint32_t MASK>
__device__ __forceinline__ float2 exp2_pair(float2 x, int i) {
  return (MASK >> (i & 15)) & 1 ? exp2_poly2(x) : make_float2(ex2_approx(x.x), ex2_approx(x.y));
}
}  // namespace

// ------------------------------------------------------------------ forward
// TMEM per tile (256 columns): S, and P over it, at [0, 128), and two O
// accumulators at [128, 192) and [192, 256): one for the first 64 keys of
// every block and one for the last 64.  The warps of a key half keep their own
// running reference and sum, so the two halves of a row meet only at the end:
// out = (f0 O0 + f1 O1) / (f0 l0 + f1 l1) with f = 2^(m - max m).
namespace {
constexpr uint32_t F_MASK = 0x0u;
constexpr size_t F_SMEM = 1024 + TILE_B * (4 + 2 * ST) + 4096 + 512;
}

__global__ void __launch_bounds__(TC_THREADS, 1)
    k_attn_forward_tc(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK,
                      const __grid_constant__ CUtensorMap tmV, AttnShape a, HeadsView out, float* __restrict__ lse,
                      int items, int per_head, int tpi, int* err) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* sQ = smem;  // [item parity][tile]
  uint8_t* sK = smem + 4 * TILE_B;
  uint8_t* sV = sK + ST * TILE_B;
  float2* sX = reinterpret_cast<float2*>(sV + ST * TILE_B);  // [tile][half][row] (reference, sum)
  uint64_t* bars = reinterpret_cast<uint64_t*>(reinterpret_cast<uint8_t*>(sX) + 4096);
  uint64_t* q_full = bars;           // [2] item parity
  uint64_t* q_empty = q_full + 2;    // [2]
  uint64_t* kv_full = q_empty + 2;   // [ST]
  uint64_t* kv_empty = kv_full + ST; // [ST]
  uint64_t* s_full = kv_empty + ST;  // [2] tile: S(j) ready, every earlier product of the tile done
  uint64_t* p_full = s_full + 2;     // [2 tiles][2 halves]
  uint64_t* o_done = p_full + 4;     // [2] tile
  uint64_t* x_full = o_done + 2;     // [2] tile: references and sums of both halves written
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(x_full + 2);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  struct Item {
    int b, h, q0, tiles, nb, nq, nk;  // tiles: how many of its tiles have queries and keys
  };
  auto item_of = [&](int it) {
    Item r;
    const int bh = it / per_head;
    r.b = bh / a.heads;
    r.h = bh - r.b * a.heads;
    r.q0 = (it - bh * per_head) * tpi * TR;
    r.nq = seq_len(a.q_lens, r.b, a.nq);
    r.nk = seq_len(a.kv_lens, r.b, a.nk);
    r.nb = (r.nk + TR - 1) / TR;
    r.tiles = r.nb == 0 ? 0 : min(tpi, (r.nq - r.q0 + TR - 1) / TR);
    if (r.tiles < 0) r.tiles = 0;
    return r;
  };

  if (threadIdx.x == 0) {
    for (int i = 0; i < 2; ++i) {
      mbar_init(&q_full[i], 1);
      mbar_init(&q_empty[i], 1);
      mbar_init(&s_full[i], 1);
      mbar_init(&p_full[2 * i], 4);
      mbar_init(&p_full[2 * i + 1], 4);
      mbar_init(&o_done[i], 1);
      mbar_init(&x_full[i], 8);
    }
    for (int i = 0; i < ST; ++i) {
      mbar_init(&kv_full[i], 1);
      mbar_init(&kv_empty[i], 1);
    }
    fence_mbar_init();
  }
  if (warp == 1) {
    tmem_alloc(tmem_slot, 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;

  if (warp == 0) {
    if (lane == 0) {
      uint32_t g = 0;
      bool ok = true;
      for (int it = blockIdx.x, c = 0; it < items && ok; it += gridDim.x) {
        const Item I = item_of(it);
        if (I.tiles == 0) continue;
        const int qb = c & 1;
        if (c >= 2 && !mbar_wait(&q_empty[qb], ((c >> 1) - 1) & 1, err, VK_DEV_TIMEOUT_PRODUCER)) break;
        ++c;
        mbar_arrive_expect_tx(&q_full[qb], I.tiles * TILE_B);
        for (int t = 0; t < I.tiles; ++t) tma_load_4d(sQ + (qb * 2 + t) * TILE_B, &tmQ, &q_full[qb], I.q0 + t * TR, I.h, I.b);
        for (int j = 0; j < I.nb; ++j, ++g) {
          const uint32_t st = g % ST;
          if (!(ok = mbar_wait(&kv_empty[st], ((g / ST) & 1) ^ 1, err, VK_DEV_TIMEOUT_PRODUCER))) break;
          mbar_arrive_expect_tx(&kv_full[st], 2 * TILE_B);
          tma_load_4d(sK + st * TILE_B, &tmK, &kv_full[st], j * TR, I.h, I.b);
          tma_load_4d(sV + st * TILE_B, &tmV, &kv_full[st], j * TR, I.h, I.b);
        }
      }
    }
  } else if (warp == 1) {
    constexpr uint32_t idS = idesc_bf16(128, 128), idO = idesc_bf16_bmn(128, 64);
    uint32_t g = 0, sp[2] = {0u, 0u};
    bool ok = true;
    for (int it = blockIdx.x, c = 0; it < items && ok; it += gridDim.x) {
      const Item I = item_of(it);
      if (I.tiles == 0) continue;
      const int qb = c & 1;
      auto block_ready = [&](uint32_t gg, int j) {
        if (!warp_wait(&kv_full[gg % ST], (gg / ST) & 1, err, VK_DEV_TIMEOUT_MMA)) return false;
        const int valid = I.nk - j * TR;
        if (valid < TR && I.nk < a.nk) zero_tail(sK + gg % ST * TILE_B, sV + gg % ST * TILE_B, valid, lane);
        return true;
      };
      auto issue_s = [&](int t, uint32_t st) {
        const uint64_t qd = smem_desc_k_sw128(smem_u32(sQ + (qb * 2 + t) * TILE_B));
        const uint64_t kd = smem_desc_k_sw128(smem_u32(sK + st * TILE_B));
#pragma unroll
        for (int k = 0; k < 4; ++k) umma_f16(tmem + t * 256, qd + k * 2, kd + k * 2, idS, k > 0 ? 1u : 0u);
        umma_commit(&s_full[t]);
      };
      if (!(ok = warp_wait(&q_full[qb], (c >> 1) & 1, err, VK_DEV_TIMEOUT_MMA) && block_ready(g, 0))) break;
      ++c;
      tc_fence_after();
      if (lane == 0)
        for (int t = 0; t < I.tiles; ++t) issue_s(t, g % ST);
      for (int j = 0; j < I.nb && ok; ++j, ++g) {
        const bool more = j + 1 < I.nb;
        if (more && !(ok = block_ready(g + 1, j + 1))) break;
        for (int t = 0; t < I.tiles && ok; ++t) {
          const uint64_t vd = smem_desc_mn_sw128(smem_u32(sV + g % ST * TILE_B));
          const uint32_t par = sp[t] & 1;
          ++sp[t];
          // O is overwritten at an item's first block: both halves' warps
          // have read the last item's O of this tile once they hand over P
          if (!(ok = warp_wait(&p_full[2 * t], par, err, VK_DEV_TIMEOUT_MMA))) break;
          if (j == 0 && !(ok = warp_wait(&p_full[2 * t + 1], par, err, VK_DEV_TIMEOUT_MMA))) break;
          for (int h = 0; h < 2; ++h) {
            if (h == 1 && j > 0 && !(ok = warp_wait(&p_full[2 * t + 1], par, err, VK_DEV_TIMEOUT_MMA))) break;
            tc_fence_after();
            if (lane == 0) {
#pragma unroll
              for (int k = 0; k < 4; ++k)
                umma_f16_ts(tmem + t * 256 + 128 + h * 64, tmem + t * 256 + h * 64 + k * 8,
                            vd + static_cast<uint64_t>((h * 4 + k) * (2048 >> 4)), idO, (j | k) > 0 ? 1u : 0u);
            }
          }
          if (!ok) break;
          if (lane == 0) {
            if (more)
              issue_s(t, (g + 1) % ST);  // after the products that read P, which it overwrites
            else
              umma_commit(&o_done[t]);
          }
        }
        if (ok && lane == 0) umma_commit(&kv_empty[g % ST]);
      }
      if (ok && lane == 0) umma_commit(&q_empty[qb]);
    }
  } else {
    const int e = warp - 2, quad = warp & 3;
    const int t = e >> 3, h = (e >> 2) & 1;
    const uint32_t tb = tmem + t * 256 + (static_cast<uint32_t>(quad * 32) << 16);
    const uint32_t ts = tb + h * 64, to = tb + 128 + h * 64;
    const float sl2 = a.scale * LOG2E;
    const int trow = quad * 32 + lane;
    uint32_t sp = 0, ct = 0;
    bool ok = true;
    for (int it = blockIdx.x; it < items && ok; it += gridDim.x) {
      const Item I = item_of(it);
      if (t >= tpi) break;
      const int row = I.q0 + t * TR + trow;
      __nv_bfloat16* op = static_cast<__nv_bfloat16*>(out.p) + I.b * out.sb + I.h * out.sh + row * out.st + h * 32;
      float* lp = lse + (static_cast<size_t>(I.b) * a.heads + I.h) * a.nq + row;
      if (t >= I.tiles) {  // no queries here, or no keys
        if (row < a.nq) {
          store_zero32(op);
          store_zero32(op + 16);
          if (h == 0) *lp = -INFINITY;
        }
        continue;
      }
      float m_ref = -INFINITY, l_run = 0.0f;
      for (int j = 0; j < I.nb; ++j, ++sp) {
        if (!warp_wait(&s_full[t], sp & 1, err, VK_DEV_TIMEOUT_EPILOGUE)) {
          ok = false;
          break;
        }
        tc_fence_after();
        const int valid = I.nk - j * TR - h * 64;  // of this half's 64 keys
        const bool full = valid >= 64;
        auto half_max = [&]() {
          float pm[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            uint32_t r[32];
            tmem_ld32(ts + c * 32, r);
            tmem_wait_ld();
#pragma unroll
            for (int i = 0; i < 32; ++i)
              if (full || c * 32 + i < valid) pm[i & 3] = fmaxf(pm[i & 3], __uint_as_float(r[i]));
          }
          return fmaxf(fmaxf(pm[0], pm[1]), fmaxf(pm[2], pm[3])) * sl2;
        };
        uint32_t pk[32];
        // p = 2^(s scale log2e - m), packed; returns the row's sum.  At the
        // first block m is the maximum of these 64 keys.
        auto exp_pass = [&](bool set_ref) {
          uint32_t r[64];
          tmem_ld32(ts, *reinterpret_cast<uint32_t(*)[32]>(&r[0]));
          tmem_ld32(ts + 32, *reinterpret_cast<uint32_t(*)[32]>(&r[32]));
          tmem_wait_ld();
          if (set_ref) {
            float pm[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
            if (full) {
#pragma unroll
              for (int i = 0; i < 64; i += 2)
                pm[(i >> 1) & 3] = max3f(pm[(i >> 1) & 3], __uint_as_float(r[i]), __uint_as_float(r[i + 1]));
            } else {
#pragma unroll
              for (int i = 0; i < 64; ++i)
                if (i < valid) pm[i & 3] = fmaxf(pm[i & 3], __uint_as_float(r[i]));
            }
            m_ref = fmaxf(fmaxf(pm[0], pm[1]), fmaxf(pm[2], pm[3])) * sl2;
          }
          // (where nothing but -inf came so far, the first finite score overflows the check below)
          const float m = finite_ref(m_ref);
          const float2 scale2 = make_float2(sl2, sl2), shift2 = make_float2(-m, -m);
          float2 ps[2] = {make_float2(0.0f, 0.0f), make_float2(0.0f, 0.0f)};
#pragma unroll
          for (int i = 0; i < 32; ++i) {
            float2 p = exp2_pair<F_MASK>(
                ffma2(make_float2(__uint_as_float(r[2 * i]), __uint_as_float(r[2 * i + 1])), scale2, shift2), i);
            if (!full) {
              p.x = 2 * i < valid ? p.x : 0.0f;
              p.y = 2 * i + 1 < valid ? p.y : 0.0f;
            }
            ps[i & 1] = fadd2(ps[i & 1], p);
            pk[i] = pack_bf16x2(p.x, p.y);
          }
          return (ps[0].x + ps[0].y) + (ps[1].x + ps[1].y);
        };
        // One pass against the running reference.  The final quotient does not
        // depend on it, so p may exceed 1; a row whose sum reaches 2^20 is done
        // again against the block's own maximum, with O and the sum rescaled
        // (the earlier products are complete: S(j) was issued after them, and
        // at the first block O is overwritten anyway).
        float l_blk = exp_pass(j == 0);
        if (__any_sync(0xffffffffu, !(l_blk < 1048576.0f))) {
          const float m_new = fmaxf(m_ref, half_max());
          const float f = ex2_approx(m_ref - finite_ref(m_new));
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            uint32_t o[32];
            tmem_ld32(to + c * 32, o);
            tmem_wait_ld();
#pragma unroll
            for (int d = 0; d < 32; ++d) o[d] = __float_as_uint(__uint_as_float(o[d]) * f);
            tmem_st32(to + c * 32, o);
          }
          l_run *= f;
          m_ref = m_new;
          l_blk = exp_pass(false);
        }
        tmem_st32(ts, pk);
        tmem_wait_st();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&p_full[2 * t + h]);
        l_run += l_blk;
      }
      if (!ok) break;
      sX[(t * 2 + h) * TR + trow] = make_float2(m_ref, l_run);
      __syncwarp();
      if (lane == 0) mbar_arrive(&x_full[t]);
      if (!warp_wait(&x_full[t], ct & 1, err, VK_DEV_TIMEOUT_EPILOGUE) ||
          !warp_wait(&o_done[t], ct & 1, err, VK_DEV_TIMEOUT_EPILOGUE)) {
        ok = false;
        break;
      }
      ++ct;
      tc_fence_after();
      const float2 x0 = sX[t * 2 * TR + trow], x1 = sX[(t * 2 + 1) * TR + trow];
      const float top = finite_ref(fmaxf(x0.x, x1.x));
      const float f0 = ex2_approx(x0.x - top), f1 = ex2_approx(x1.x - top);
      const float sum = f0 * x0.y + f1 * x1.y;
      uint32_t o0[32], o1[32];  // this warp's half of the 64 output columns
      tmem_ld32(tb + 128 + h * 32, o0);
      tmem_ld32(tb + 192 + h * 32, o1);
      tmem_wait_ld();
      tc_fence_before();
      if (row < a.nq) {
        const bool live = row < I.nq && sum != 0.0f;
        const float inv = 1.0f / sum, g0 = f0 * inv, g1 = f1 * inv;
        float o[32];
#pragma unroll
        for (int d = 0; d < 32; ++d) o[d] = live ? fmaf(__uint_as_float(o0[d]), g0, __uint_as_float(o1[d]) * g1) : 0.0f;
        store_bf16x16(op, o, 1.0f);
        store_bf16x16(op + 16, o + 16, 1.0f);
        if (h == 0) *lp = live ? fmaf(top, LN2, logf(sum)) : -INFINITY;
      }
    }
  }
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

// ------------------------------------------------------------------ backward
// Both backward kernels run one pipeline.  A CTA walks its items (tiles of
// 128 own rows) and the blocks of 128 streamed rows of each as one sequence of
// blocks n = 0, 1, ...; TMEM holds S twice ([0, 128), [128, 256)), dP once
// ([256, 384)) and the accumulators ([384, 512)).  Per block:
//   MMA  S(n+2) = own1 . streamed1     after the products that read P/dS(n)
//        dP(n+1) = own2 . streamed2    as soon as block n's dP has been read
//   warps p = 2^(S scale log2e - lse log2e), then dS = p (dP - delta), written
//        as bf16 over the columns of S they read
// so the exponentials of a block start while its dP is still being computed,
// and the products on P/dS(n) run under the elementwise work of n + 1.
// Each of the 16 warps has 32 rows and 32 of the 128 columns.
namespace {
constexpr uint32_t B_MASK = 0x0u;
constexpr uint32_t COL_DP = 256, COL_ACC = 384;
constexpr size_t B_STATS = ST * 2 * TR * sizeof(float);  // dk/dv: (-lse log2e, delta) of the streamed rows; dq: delta's parts
constexpr size_t B_SMEM = 1024 + TILE_B * (4 + 2 * ST) + B_STATS + 512;

// One block of the walk.
struct Blk {
  int it, j, nb, c;  // item, block of the item and their number, ordinal of the item among those with work
  int b, h, r0;      // sequence, head, first own row
  int own, len;      // own and streamed rows of the sequence
  bool ok;
};
}  // namespace

// DQ: own rows are queries (own1 = q, own2 = d_out), streamed ones keys
// (k, v), acc = dq.  Otherwise own rows are keys (k, v), streamed ones queries
// (q, d_out), acc = dv, dk.
template <bool DQ>
__global__ void __launch_bounds__(TC_THREADS, 1)
    k_attn_backward_tc(const __grid_constant__ CUtensorMap tmO1, const __grid_constant__ CUtensorMap tmO2,
                       const __grid_constant__ CUtensorMap tmS1, const __grid_constant__ CUtensorMap tmS2, AttnShape a,
                       HeadsView out, HeadsView d_out, const float* __restrict__ lse, float* delta, HeadsView g1,
                       HeadsView g2, int items, int per_head, int* err) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* sOwn = smem;  // [item parity][own1, own2]
  uint8_t* s1 = smem + 4 * TILE_B;
  uint8_t* s2 = s1 + ST * TILE_B;
  float* sStat = reinterpret_cast<float*>(s2 + ST * TILE_B);
  uint64_t* bars = reinterpret_cast<uint64_t*>(reinterpret_cast<uint8_t*>(sStat) + B_STATS);
  uint64_t* own_full = bars;           // [2]
  uint64_t* own_empty = own_full + 2;  // [2]
  uint64_t* st_full = own_empty + 2;   // [ST]
  uint64_t* st_empty = st_full + ST;   // [ST]
  uint64_t* s_full = st_empty + ST;    // [2]
  uint64_t* dp_full = s_full + 2;
  uint64_t* ds_full = dp_full + 1;     // P and dS of a block written, its dP read
  uint64_t* acc_full = ds_full + 1;    // the item's last products done
  uint64_t* part_full = acc_full + 1;  // dq: delta's parts written
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(part_full + 1);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int total_own = DQ ? a.nq : a.nk, total_len = DQ ? a.nk : a.nq;
  auto load_item = [&](Blk& k) {
    const int bh = k.it / per_head;
    k.b = bh / a.heads;
    k.h = bh - k.b * a.heads;
    k.r0 = (k.it - bh * per_head) * TR;
    const int nq = seq_len(a.q_lens, k.b, a.nq), nk = seq_len(a.kv_lens, k.b, a.nk);
    k.own = DQ ? nq : nk;
    k.len = DQ ? nk : nq;
    k.nb = k.r0 < k.own ? (k.len + TR - 1) / TR : 0;
  };
  // skipped(k) sees the items without work
  auto seek = [&](Blk& k, auto skipped) {
    k.j = 0;
    while ((k.ok = k.it < items)) {
      load_item(k);
      if (k.nb > 0) break;
      skipped(k);
      k.it += gridDim.x;
    }
  };
  auto nothing = [](const Blk&) {};
  auto first = [&](auto skipped) {
    Blk k{};
    k.it = blockIdx.x;
    seek(k, skipped);
    return k;
  };
  auto next = [&](Blk k, auto skipped) {
    if (k.ok && ++k.j == k.nb) {
      k.it += gridDim.x;
      ++k.c;
      seek(k, skipped);
    }
    return k;
  };

  if (threadIdx.x == 0) {
    for (int i = 0; i < 2; ++i) {
      mbar_init(&own_full[i], 1);
      mbar_init(&own_empty[i], 1);
      mbar_init(&s_full[i], 1);
    }
    for (int i = 0; i < ST; ++i) {
      mbar_init(&st_full[i], 1);
      mbar_init(&st_empty[i], 1);
    }
    mbar_init(dp_full, 1);
    mbar_init(ds_full, 16);
    mbar_init(acc_full, 1);
    mbar_init(part_full, 16);
    fence_mbar_init();
  }
  if (warp == 1) {
    tmem_alloc(tmem_slot, 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;

  if (warp == 0) {
    uint32_t n = 0;
    for (Blk k = first(nothing); k.ok; k = next(k, nothing), ++n) {
      const int ob = k.c & 1;
      if (k.j == 0) {
        if (k.c >= 2 && !warp_wait(&own_empty[ob], ((k.c >> 1) - 1) & 1, err, VK_DEV_TIMEOUT_PRODUCER)) break;
        if (lane == 0) {
          mbar_arrive_expect_tx(&own_full[ob], 2 * TILE_B);
          tma_load_4d(sOwn + (2 * ob) * TILE_B, &tmO1, &own_full[ob], k.r0, k.h, k.b);
          tma_load_4d(sOwn + (2 * ob + 1) * TILE_B, &tmO2, &own_full[ob], k.r0, k.h, k.b);
        }
      }
      const uint32_t st = n % ST;
      if (!warp_wait(&st_empty[st], ((n / ST) & 1) ^ 1, err, VK_DEV_TIMEOUT_PRODUCER)) break;
      if constexpr (!DQ) {
        // the streamed rows' statistics; a row past the length gets -inf: its p is 2^-inf = 0
        const size_t at = (static_cast<size_t>(k.b) * a.heads + k.h) * a.nq;
        float l[4], d[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int row = k.j * TR + i * 32 + lane;
          const bool in = row < k.len;
          l[i] = in ? lse[at + row] : INFINITY;
          d[i] = in ? delta[at + row] : 0.0f;
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          // lse = -inf: a row of scores of -inf only, whose p is 2^(-inf - 0) = 0
          sStat[st * 2 * TR + i * 32 + lane] = l[i] == -INFINITY ? 0.0f : -l[i] * LOG2E;
          sStat[st * 2 * TR + TR + i * 32 + lane] = d[i];
        }
        __syncwarp();
      }
      if (lane == 0) {
        mbar_arrive_expect_tx(&st_full[st], 2 * TILE_B);
        tma_load_4d(s1 + st * TILE_B, &tmS1, &st_full[st], k.j * TR, k.h, k.b);
        tma_load_4d(s2 + st * TILE_B, &tmS2, &st_full[st], k.j * TR, k.h, k.b);
      }
    }
  } else if (warp == 1) {
    constexpr uint32_t idS = idesc_bf16(128, 128), idA = idesc_bf16_bmn(128, 64);
    // waits for a block's operands and clears what lies past the length
    auto ready = [&](const Blk& k, uint32_t n) {
      if (k.j == 0 && !warp_wait(&own_full[k.c & 1], (k.c >> 1) & 1, err, VK_DEV_TIMEOUT_MMA)) return false;
      if (!warp_wait(&st_full[n % ST], (n / ST) & 1, err, VK_DEV_TIMEOUT_MMA)) return false;
      const int valid = k.len - k.j * TR;
      if (valid < TR && k.len < total_len) zero_tail(s1 + n % ST * TILE_B, s2 + n % ST * TILE_B, valid, lane);
      tc_fence_after();
      return true;
    };
    auto product = [&](uint32_t col, const uint8_t* own, const uint8_t* streamed) {
      const uint64_t od = smem_desc_k_sw128(smem_u32(own)), sd = smem_desc_k_sw128(smem_u32(streamed));
#pragma unroll
      for (int k = 0; k < 4; ++k) umma_f16(tmem + col, od + k * 2, sd + k * 2, idS, k > 0 ? 1u : 0u);
    };
    auto issue_s = [&](const Blk& k, uint32_t n) {
      if (lane == 0) {
        product((n & 1) * TR, sOwn + (k.c & 1) * 2 * TILE_B, s1 + n % ST * TILE_B);
        umma_commit(&s_full[n & 1]);
      }
    };
    auto issue_dp = [&](const Blk& k, uint32_t n) {
      if (lane == 0) {
        product(COL_DP, sOwn + ((k.c & 1) * 2 + 1) * TILE_B, s2 + n % ST * TILE_B);
        umma_commit(dp_full);
        if (k.j + 1 == k.nb) umma_commit(&own_empty[k.c & 1]);  // its S was issued before
      }
    };
    // acc += A . streamed, A = bf16 columns `col` + 32 (k / 2) + 8 (k % 2) of TMEM
    auto sum = [&](uint32_t acc, uint32_t col, const uint8_t* streamed, bool fresh) {
      const uint64_t sd = smem_desc_mn_sw128(smem_u32(streamed));
#pragma unroll
      for (int k = 0; k < 8; ++k)
        umma_f16_ts(tmem + acc, tmem + col + (k >> 1) * 32 + (k & 1) * 8, sd + static_cast<uint64_t>(k * (2048 >> 4)), idA,
                    fresh && k == 0 ? 0u : 1u);
    };
    Blk b0 = first(nothing), b1 = next(b0, nothing), b2 = next(b1, nothing);
    bool ok = true;
    if (b0.ok && (ok = ready(b0, 0))) {
      issue_s(b0, 0);
      issue_dp(b0, 0);
    }
    if (ok && b1.ok && (ok = ready(b1, 1))) issue_s(b1, 1);
    for (uint32_t n = 0; ok && b0.ok; ++n) {
      if (!(ok = warp_wait(ds_full, n & 1, err, VK_DEV_TIMEOUT_MMA))) break;
      tc_fence_after();
      if (b1.ok) issue_dp(b1, n + 1);
      if (lane == 0) {
        const uint32_t col = (n & 1) * TR;
        if constexpr (DQ) {
          sum(COL_ACC, col, s1 + n % ST * TILE_B, b0.j == 0);  // dq += dS k
        } else {
          sum(COL_ACC, col, s2 + n % ST * TILE_B, b0.j == 0);            // dv += P^T d_out
          sum(COL_ACC + 64, col + 16, s1 + n % ST * TILE_B, b0.j == 0);  // dk += dS^T q
        }
        umma_commit(&st_empty[n % ST]);
        if (b0.j + 1 == b0.nb) umma_commit(acc_full);
      }
      if (b2.ok) {
        if (!(ok = ready(b2, n + 2))) break;
        issue_s(b2, n + 2);  // after the products that read the P/dS it overwrites
      }
      b0 = b1;
      b1 = b2;
      b2 = next(b2, nothing);
    }
  } else {
    const int quad = warp & 3, part = (warp - 2) >> 2;  // columns [32 part, 32 part + 32)
    const uint32_t lanes = static_cast<uint32_t>(quad * 32) << 16;
    const float sl2 = a.scale * LOG2E;
    const int trow = quad * 32 + lane;
    // this thread's piece of its own row: dq columns [16 part, +16); dv (parts
    // 0, 1) or dk (parts 2, 3) columns [32 (part & 1), +32)
    auto piece = [&](const Blk& k) {
      const HeadsView& v = DQ || part < 2 ? g1 : g2;
      return static_cast<__nv_bfloat16*>(v.p) + k.b * v.sb + k.h * v.sh + static_cast<int64_t>(k.r0 + trow) * v.st +
             (DQ ? part * 16 : (part & 1) * 32);
    };
    auto skipped = [&](const Blk& k) {  // no own rows, or nothing to stream
      if (k.r0 + trow >= total_own) return;
      __nv_bfloat16* p = piece(k);
      store_zero32(p);
      if constexpr (DQ) {
        if (part == 0) delta[(static_cast<size_t>(k.b) * a.heads + k.h) * a.nq + k.r0 + trow] = 0.0f;
      } else {
        store_zero32(p + 16);
      }
    };
    // own row statistics (dq): lse, and this thread's 16 of the 64 products of delta
    float lse_next = 0.0f;
    uint4 o_next[2], d_next[2];
    auto fetch = [&](const Blk& k) {
      const int row = k.r0 + trow;
      lse_next = 0.0f;
      o_next[0] = o_next[1] = d_next[0] = d_next[1] = make_uint4(0, 0, 0, 0);
      if (!k.ok || row >= k.own) return;
      lse_next = lse[(static_cast<size_t>(k.b) * a.heads + k.h) * a.nq + row];
      const uint4* op = reinterpret_cast<const uint4*>(static_cast<const __nv_bfloat16*>(out.p) + k.b * out.sb +
                                                       k.h * out.sh + row * out.st + part * 16);
      const uint4* dp = reinterpret_cast<const uint4*>(static_cast<const __nv_bfloat16*>(d_out.p) + k.b * d_out.sb +
                                                       k.h * d_out.sh + row * d_out.st + part * 16);
      o_next[0] = op[0];
      o_next[1] = op[1];
      d_next[0] = dp[0];
      d_next[1] = dp[1];
    };
    auto partial_delta = [&]() {
      const uint32_t* o = reinterpret_cast<const uint32_t*>(o_next);
      const uint32_t* d = reinterpret_cast<const uint32_t*>(d_next);
      float x = 0.0f, y = 0.0f;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        x = fmaf(__uint_as_float(o[i] << 16), __uint_as_float(d[i] << 16), x);
        y = fmaf(__uint_as_float(o[i] & 0xffff0000u), __uint_as_float(d[i] & 0xffff0000u), y);
      }
      return x + y;
    };
    auto finish = [&](const Blk& k, uint32_t c) {  // the item's accumulators to memory
      if (!warp_wait(acc_full, c & 1, err, VK_DEV_TIMEOUT_EPILOGUE)) return false;
      tc_fence_after();
      const int row = k.r0 + trow;
      if constexpr (DQ) {
        uint32_t r[16];
        tmem_ld16(tmem + COL_ACC + lanes + part * 16, r);
        tmem_wait_ld();
        tc_fence_before();
        if (row < k.own)
          store_bf16x16(piece(k), reinterpret_cast<const float*>(r), a.scale);
        else if (row < total_own)
          store_zero32(piece(k));
      } else {
        uint32_t r[32];
        tmem_ld32(tmem + COL_ACC + lanes + part * 32, r);
        tmem_wait_ld();
        tc_fence_before();
        if (row < k.own) {
          const float f = part < 2 ? 1.0f : a.scale;
          store_bf16x16(piece(k), reinterpret_cast<const float*>(r), f);
          store_bf16x16(piece(k) + 16, reinterpret_cast<const float*>(r) + 16, f);
        } else if (row < total_own) {
          store_zero32(piece(k));
          store_zero32(piece(k) + 16);
        }
      }
      return true;
    };
    Blk k = first(skipped), done{};
    bool pending = false, ok = true;
    float shift = 0.0f, dl = 0.0f;
    if constexpr (DQ) fetch(k);
    for (uint32_t n = 0; k.ok; ++n) {
      const uint32_t st = n % ST, ts = tmem + (n & 1) * TR + part * 32 + lanes;
      if (DQ && k.j == 0) shift = lse_next == -INFINITY ? 0.0f : -lse_next * LOG2E;
      const int valid = DQ ? k.len - k.j * TR - part * 32 : 32;  // of this warp's columns (dk/dv: by the statistics)
      if (!(ok = warp_wait(&s_full[n & 1], (n >> 1) & 1, err, VK_DEV_TIMEOUT_EPILOGUE))) break;
      tc_fence_after();
      float p[32];
      {
        if constexpr (!DQ) {  // the statistics came with the block
          if (!(ok = warp_wait(&st_full[st], (n / ST) & 1, err, VK_DEV_TIMEOUT_EPILOGUE))) break;
        }
        uint32_t r[32];
        tmem_ld32(ts, r);
        tmem_wait_ld();
        const float4* sl = reinterpret_cast<const float4*>(sStat + st * 2 * TR + part * 32);
#pragma unroll
        for (int i = 0; i < 16; i += 2) {
          float2 h0 = make_float2(shift, shift), h1 = h0;
          if constexpr (!DQ) {
            const float4 v = sl[i / 2];
            h0 = make_float2(v.x, v.y);
            h1 = make_float2(v.z, v.w);
          }
          const float2 e0 = exp2_pair<B_MASK>(
              ffma2(make_float2(__uint_as_float(r[2 * i]), __uint_as_float(r[2 * i + 1])), make_float2(sl2, sl2), h0), i);
          const float2 e1 = exp2_pair<B_MASK>(
              ffma2(make_float2(__uint_as_float(r[2 * i + 2]), __uint_as_float(r[2 * i + 3])), make_float2(sl2, sl2), h1), i + 1);
          p[2 * i] = e0.x, p[2 * i + 1] = e0.y, p[2 * i + 2] = e1.x, p[2 * i + 3] = e1.y;
        }
        if (DQ && valid < 32) {
#pragma unroll
          for (int i = 0; i < 32; ++i)
            if (i >= valid) p[i] = 0.0f;
        }
      }
      if constexpr (!DQ) {
        uint32_t pk[16];
#pragma unroll
        for (int i = 0; i < 16; ++i) pk[i] = pack_bf16x2(p[2 * i], p[2 * i + 1]);
        tmem_st16(ts, pk);
      }
      if (k.j == 0) {
        if (pending && !(ok = finish(done, done.c))) break;
        pending = false;
        if constexpr (DQ) {
          float* mine = sStat + (k.c & 1) * 4 * TR;
          mine[part * TR + trow] = partial_delta();
          __syncwarp();
          if (lane == 0) mbar_arrive(part_full);
          if (!(ok = warp_wait(part_full, k.c & 1, err, VK_DEV_TIMEOUT_EPILOGUE))) break;
          dl = (mine[trow] + mine[TR + trow]) + (mine[2 * TR + trow] + mine[3 * TR + trow]);
          if (part == 0 && k.r0 + trow < total_own)
            delta[(static_cast<size_t>(k.b) * a.heads + k.h) * a.nq + k.r0 + trow] = dl;
        }
      }
      const Blk after = next(k, skipped);
      if constexpr (DQ) {
        if (k.j + 1 == k.nb) fetch(after);
      }
      if (!(ok = warp_wait(dp_full, n & 1, err, VK_DEV_TIMEOUT_EPILOGUE))) break;
      tc_fence_after();
      {
        uint32_t r[32], pk[16];
        tmem_ld32(tmem + COL_DP + part * 32 + lanes, r);
        tmem_wait_ld();
        const float4* sd = reinterpret_cast<const float4*>(sStat + st * 2 * TR + TR + part * 32);
#pragma unroll
        for (int i = 0; i < 16; i += 2) {
          float2 h0 = make_float2(dl, dl), h1 = h0;
          if constexpr (!DQ) {
            const float4 v = sd[i / 2];
            h0 = make_float2(v.x, v.y);
            h1 = make_float2(v.z, v.w);
          }
          const float2 d0 = fmul2(fsub2(make_float2(__uint_as_float(r[2 * i]), __uint_as_float(r[2 * i + 1])), h0),
                                  make_float2(p[2 * i], p[2 * i + 1]));
          const float2 d1 = fmul2(fsub2(make_float2(__uint_as_float(r[2 * i + 2]), __uint_as_float(r[2 * i + 3])), h1),
                                  make_float2(p[2 * i + 2], p[2 * i + 3]));
          pk[i] = pack_bf16x2(d0.x, d0.y);
          pk[i + 1] = pack_bf16x2(d1.x, d1.y);
        }
        tmem_st16(DQ ? ts : ts + 16, pk);
      }
      tmem_wait_st();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(ds_full);
      if (k.j + 1 == k.nb) {
        done = k;
        pending = true;
      }
      k = after;
    }
    if (ok && pending) finish(done, done.c);
  }
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

// ------------------------------------------------------------------ launches
namespace {
bool heads_map(CUtensorMap* m, const HeadsView& v, int batch, int heads, int tokens) {
  const uint64_t dims[4] = {64, static_cast<uint64_t>(tokens), static_cast<uint64_t>(heads), static_cast<uint64_t>(batch)};
  const uint64_t strides[3] = {static_cast<uint64_t>(v.st) * 2, static_cast<uint64_t>(v.sh) * 2, static_cast<uint64_t>(v.sb) * 2};
  const uint32_t box[4] = {64, TR, 1, 1};
  return make_tmap_nd(m, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, v.p, 4, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_128B);
}
}  // namespace

cudaError_t attention_forward_tc(const AttnShape& a, HeadsView q, HeadsView k, HeadsView v, HeadsView out, float* lse,
                                 int* err, cudaStream_t s) {
  CUtensorMap mq, mk, mv;
  if (!heads_map(&mq, q, a.batch, a.heads, a.nq) || !heads_map(&mk, k, a.batch, a.heads, a.nk) ||
      !heads_map(&mv, v, a.batch, a.heads, a.nk))
    return cudaErrorInvalidValue;
  const void* fn = reinterpret_cast<const void*>(k_attn_forward_tc);
  const cudaError_t e = ensure_smem_limit(fn, static_cast<int>(F_SMEM));
  if (e != cudaSuccess) return e;
  // Two query tiles share each K / V block; one where pairs would leave SMs idle.
  const int nt = (a.nq + TR - 1) / TR, bh = a.batch * a.heads;
  const int tpi = (nt + 1) / 2 * bh < num_sms() ? 1 : 2;
  const int per_head = (nt + tpi - 1) / tpi, items = per_head * bh;
  const int grid = items < num_sms() ? items : num_sms();
  k_attn_forward_tc<<<grid, TC_THREADS, F_SMEM, s>>>(mq, mk, mv, a, out, lse, items, per_head, tpi, err);
  return cudaGetLastError();
}

cudaError_t attention_backward_tc(const AttnShape& a, HeadsView q, HeadsView k, HeadsView v, HeadsView out,
                                  const float* lse, HeadsView d_out, HeadsView dq, HeadsView dk, HeadsView dv,
                                  float* delta, int* err, cudaStream_t s) {
  CUtensorMap mq, mk, mv, mg;
  if (!heads_map(&mq, q, a.batch, a.heads, a.nq) || !heads_map(&mk, k, a.batch, a.heads, a.nk) ||
      !heads_map(&mv, v, a.batch, a.heads, a.nk) || !heads_map(&mg, d_out, a.batch, a.heads, a.nq))
    return cudaErrorInvalidValue;
  cudaError_t e = ensure_smem_limit(reinterpret_cast<const void*>(k_attn_backward_tc<true>), static_cast<int>(B_SMEM));
  if (e == cudaSuccess) e = ensure_smem_limit(reinterpret_cast<const void*>(k_attn_backward_tc<false>), static_cast<int>(B_SMEM));
  if (e != cudaSuccess) return e;
  const int bh = a.batch * a.heads, sms = num_sms();
  const int qt = (a.nq + TR - 1) / TR, kt = (a.nk + TR - 1) / TR;
  k_attn_backward_tc<true><<<qt * bh < sms ? qt * bh : sms, TC_THREADS, B_SMEM, s>>>(mq, mg, mk, mv, a, out, d_out, lse, delta,
                                                                                    dq, dq, qt * bh, qt, err);
  e = cudaGetLastError();
  if (e != cudaSuccess) return e;
  k_attn_backward_tc<false><<<kt * bh < sms ? kt * bh : sms, TC_THREADS, B_SMEM, s>>>(mk, mv, mq, mg, a, out, d_out, lse, delta,
                                                                                     dv, dk, kt * bh, kt, err);
  return cudaGetLastError();
}

}  // namespace vk
