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
//   warp 1       TMEM owner; one thread issues MMAs
//   warp 2       with lengths: clears the tails of streamed tiles
//   warp 3       one thread issues MMAs
//   warps 4..7   backward: delta, and the results on their way to memory
//   the others   the elementwise work on S (and dP) in TMEM: two groups of four
//                warps, a row of 128 columns per thread.  (16 warps with 64
//                or 32 columns each spent half of their instructions on
//                waits and hand-overs, and most of their time in step.)
//
// S and dP are bf16 products in f32.  P and dS are rounded to bf16 for the
// second products (one rounding of 2^-8 at most, next to the one of the
// result); everything else is f32.  Rows and columns past a sequence's length
// never reach a product: scores are masked, and the tail of a streamed tile is
// zeroed in shared memory, because 0 * NaN would spread what lies there.
#include <limits.h>

#include "vk_common.cuh"
#include "vk_internal.h"
#include "vk_train.h"

namespace vk {

namespace {
constexpr int TR = 128;                 // rows of a tile, columns of a block
constexpr int TILE_B = TR * 128;        // bytes of 128 rows of 64 bf16
constexpr int ST = 4;                   // streamed blocks in flight
constexpr int EXT_B = TR * 32;          // bytes of 128 rows of 16 bf16
constexpr int F_THREADS = 12 * 32, B_THREADS = 16 * 32;
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

__device__ __forceinline__ void tmem_st8(uint32_t taddr, const uint32_t (&r)[8]) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"r"(taddr), "r"(r[0]),
               "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7])
               : "memory");
}

// Zeroes rows [valid, 128) of two tiles that TMA wrote, before MMAs read them;
// all lanes of a warp.  A swizzled row stays in its own 128 bytes.
__device__ __forceinline__ void zero_tail(uint8_t* a, uint8_t* b, int valid, int lane) {
  for (int i = valid * 8 + lane; i < TR * 8; i += 32) {
    reinterpret_cast<uint4*>(a)[i] = make_uint4(0, 0, 0, 0);
    reinterpret_cast<uint4*>(b)[i] = make_uint4(0, 0, 0, 0);
  }
  fence_proxy_async();
  __syncwarp();
}

// Register shares of the warps with the elementwise work and of the others.
// Forward: 256 * 208 + 128 * 88 = 384 * 168, the launch's.  Backward:
// 256 * 184 + 256 * 72 = 512 * 128.
template <int N>
__device__ __forceinline__ void regs_inc() {
  asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N));
}
template <int N>
__device__ __forceinline__ void regs_dec() {
  asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N));
}

// K-major operand of 16 columns without swizzle: 8 x 16-byte pieces of 128
// bytes, the two of a row 128 bytes apart, the next 8 rows 256.
__device__ __forceinline__ uint64_t smem_desc_k16(uint32_t saddr) {
  return static_cast<uint64_t>((saddr >> 4) & 0x3FFFu) | static_cast<uint64_t>(128u >> 4) << 16 |
         static_cast<uint64_t>(256u >> 4) << 32 | static_cast<uint64_t>(1u) << 46;
}
// Piece k of row r of such a tile.
__device__ __forceinline__ uint4* ext_piece(uint8_t* s, int r, int k) {
  return reinterpret_cast<uint4*>(s + (r >> 3) * 256 + k * 128 + (r & 7) * 16);
}
// x = hi + mid + lo in bf16, 24 bits of it; not finite: hi alone.
__device__ __forceinline__ void split3(float x, float& hi, float& mid, float& lo) {
  hi = __bfloat162float(__float2bfloat16_rn(x));
  const float rest = isfinite(x) ? x - hi : 0.0f;
  mid = __bfloat162float(__float2bfloat16_rn(rest));
  lo = rest - mid;
}

// True in one lane of a converged warp.  The MMA loops run under it: the
// compiler knows that a single thread is active and keeps the operands in
// uniform registers (under `lane == 0` each MMA took 115 cycles to issue), and
// that thread's waits need no vote of the warp.
__device__ __forceinline__ bool elect_one() {
  uint32_t p;
  asm volatile("{\n\t.reg .pred e;\n\telect.sync _|e, 0xffffffff;\n\tselp.u32 %0, 1, 0, e;\n\t}" : "=r"(p));
  return p != 0;
}

// After a wait ran out: the copies and products that are still under way must
// not outlive the block's shared and tensor memory.  Waits for a phase whatever
// the error word says, a tenth of a second at most.
__device__ __forceinline__ void drain(uint64_t* bar, uint32_t parity) {
  const uint64_t t0 = globaltimer();
  while (!mbar_try_wait(smem_u32(bar), parity) && globaltimer() - t0 < 100000000ull) {
  }
}

// One thread's wait for a phase; false (and `code` in the error word) when it
// ran out.  The clock and the error word are looked at every 1024 tries only.
__device__ __forceinline__ bool thread_wait(uint64_t* bar, uint32_t parity, int* err, int code) {
  const uint32_t a = smem_u32(bar);
  uint64_t t0 = 0;
  for (uint32_t it = 1; !mbar_try_wait(a, parity); ++it) {
    if ((it & 1023u) != 0) continue;
    const uint64_t t = globaltimer();
    if (t0 == 0) t0 = t;
    if (*reinterpret_cast<volatile int*>(err) != 0 || t - t0 > VK_WAIT_NS) {
      record_error(err, code);
      return false;
    }
  }
  return true;
}
// The same for a warp: one outcome for all lanes.  (A phase that is over
// already, the usual case, costs no loop: 64 images backward 612 and 603 us.)
__device__ __forceinline__ bool warp_wait(uint64_t* bar, uint32_t parity, int* err, int code) {
  if (__all_sync(0xffffffffu, mbar_try_wait(smem_u32(bar), parity))) return true;
  return __all_sync(0xffffffffu, thread_wait(bar, parity, err, code));
}

__device__ __forceinline__ void tma_store_4d(const void* desc, const void* src, int32_t y, int32_t z, int32_t w) {
  asm volatile("cp.async.bulk.tensor.4d.global.shared::cta.tile.bulk_group [%0, {%2, %3, %4, %5}], [%1];" ::"l"(
                   reinterpret_cast<uint64_t>(desc)),
               "r"(smem_u32(src)), "r"(0), "r"(y), "r"(z), "r"(w)
               : "memory");
}

// 16-byte piece c of row `lane` of a warp's output staging, 32 rows of 64 bf16
// in the order of TMA's 128-byte swizzle.  Rows leave through TMA because a thread's own stores, one row
// each, would touch 32 lines per instruction: 2000 cycles of address work per
// tile where an item has about 15000.
__device__ __forceinline__ uint4* staged(uint8_t* s, int lane, int c) {
  return reinterpret_cast<uint4*>(s + lane * 128 + ((c ^ lane) & 7) * 16);
}
__device__ __forceinline__ uint4 pack8(const float* x, float f) {
  return make_uint4(pack_bf16x2(x[0] * f, x[1] * f), pack_bf16x2(x[2] * f, x[3] * f), pack_bf16x2(x[4] * f, x[5] * f),
                    pack_bf16x2(x[6] * f, x[7] * f));
}
// The staged rows are on their way when this returns; the warp's lane 0 waits
// for them (bulk_wait_read) before the staging is used again.
__device__ __forceinline__ void send_rows(const void* desc, const uint8_t* s, int y, int rows, int z, int w, int lane) {
  fence_proxy_async();
  __syncwarp();
  if (lane == 0) {
    if (y < rows) tma_store_4d(desc, s, y, z, w);
    bulk_commit();
  }
}
__device__ __forceinline__ void store_zeros(__nv_bfloat16* p) {  // a row
  for (int i = 0; i < 64; i += 8) *reinterpret_cast<uint4*>(p + i) = make_uint4(0, 0, 0, 0);
}
// A row of 64 accumulator columns, times f, into the staging (zeros if not live).
__device__ __forceinline__ void stage_row(uint8_t* s, int lane, uint32_t taddr, float f, bool live) {
#pragma unroll
  for (int d0 = 0; d0 < 64; d0 += 32) {
    uint32_t r[32];
    tmem_ld32(taddr + d0, r);
    tmem_wait_ld();
    float x[32];
#pragma unroll
    for (int d = 0; d < 32; ++d) x[d] = live ? __uint_as_float(r[d]) : 0.0f;
#pragma unroll
    for (int c = 0; c < 4; ++c) *staged(s, lane, d0 / 8 + c) = pack8(x + 8 * c, f);
  }
}
// 128 columns of a row.
__device__ __forceinline__ void tmem_ld128(uint32_t taddr, uint32_t (&r)[128]) {
#pragma unroll
  for (int c = 0; c < 4; ++c) tmem_ld32(taddr + c * 32, *reinterpret_cast<uint32_t(*)[32]>(&r[c * 32]));
  tmem_wait_ld();
}

// A reference to subtract from scores of which `top` is the largest so far.
// Where they are all -inf any finite one will do: it keeps 2^(-inf) at 0.
__device__ __forceinline__ float finite_ref(float top) { return top == -INFINITY ? -1e30f : top; }

// Scores of columns from `valid` on become -inf.
__device__ __forceinline__ void mask_columns(uint32_t (&r)[128], int valid) {
  asm volatile("" ::: "memory");  // (a branch, not selects in every block)
#pragma unroll
  for (int i = 0; i < 128; ++i)
    if (i >= valid) r[i] = 0xff800000u;
}

// 2^x, by MUFU.  (A quarter of the pairs as a polynomial on the FMA pipe: of
// degree 4, 230 us against 238 for the forward pass of 64 images, but 2.7e-6
// off, which the row sums carry into lse; of degree 5, 2e-7 off, 240 us.)
__device__ __forceinline__ float2 exp2_pair(float2 x) { return make_float2(ex2_approx(x.x), ex2_approx(x.y)); }
}  // namespace

// ------------------------------------------------------------------ items
// Without lengths a CTA takes every gridDim.x-th item: all are alike.
//
// Of a padded batch (LENS) each CTA lays out its items once in shared memory,
// and its warps walk that list.  Those with work come first, sequences with the
// most blocks in front, then the others (rows that only get zeros); they go
// there and back over the CTAs, so that the one with the longest item of a
// round has the shortest of the next.  In the batch's own order the shares
// differ: of four sequences of 3457, 1729, 2283 and 829 tokens some CTAs had 160
// blocks of dq where the mean is 110.  That batch: forward 148 us in the
// batch's order, 109 this way, backward 332 and 296; 16 images of 865 to 115
// tokens forward 51 and 43.  (Batches without lengths only lose by the list: 64
// images backward 612 us and 650, so each form is a kernel of its own.)
// The steps are written out where they are taken: with named integers the
// kernels without lengths came out 3 to 5% slower.
namespace {
constexpr int LIST_MAX = 128;   // items of a CTA in a launch
constexpr int ORDER_MAX = 128;  // sequences that are ordered; more of them even out by themselves
template <bool LENS>
struct ItemList {
  int4 item[LIST_MAX];
  short2 len[ORDER_MAX];       // a sequence's items with work per head, and its blocks
  int first[2][ORDER_MAX];     // by rank: ordinal of a sequence's first item with work / without
  short2 sequence[ORDER_MAX];  // by rank: the sequence, its items with work per head
  int live;                    // items with work

  // `rows` own rows per item, `per_head` items per head, `count` of them from
  // `base` on in this launch; make((sequence, head), item of the head) gives
  // an entry.  Returns the length of the list.
  template <class F>
  __device__ __forceinline__ int build(const AttnShape& a, const int32_t* own_lens, int own, const int32_t* other_lens,
                                       int other, int rows, int per_head, int base, int count, F make) {
    const bool ordered = a.batch <= ORDER_MAX && per_head <= SHRT_MAX && other <= SHRT_MAX * TR;
    const int i = threadIdx.x;
    if (ordered) {
      if (i < a.batch) {
        const int nb = (seq_len(other_lens, i, other) + TR - 1) / TR;
        len[i] = make_short2(nb == 0 ? 0 : (seq_len(own_lens, i, own) + rows - 1) / rows, nb);
      }
      __syncthreads();
      if (i < a.batch) {
        const short2 mine = len[i];
        int rank = 0, with = 0, without = 0;
        for (int j = 0; j < a.batch; ++j) {
          const short2 o = len[j];
          if (o.y > mine.y || (o.y == mine.y && j < i)) {
            ++rank;
            with += o.x;
            without += per_head - o.x;
          }
        }
        first[0][rank] = with * a.heads;
        first[1][rank] = without * a.heads;
        sequence[rank] = make_short2(i, mine.x);
        if (rank == a.batch - 1) live = (with + mine.x) * a.heads;
      }
      __syncthreads();
    }
    const int g = gridDim.x, c = blockIdx.x, rounds = count / g;
    const int mine = rounds + ((rounds & 1 ? g - 1 - c : c) < count - rounds * g ? 1 : 0);
    for (int k = i; k < mine; k += blockDim.x) {
      const int it = base + k * g + (k & 1 ? g - 1 - c : c);
      int bh = it / per_head, n = it - bh * per_head;
      if (ordered) {
        const bool rest = it >= live;
        const int* f = first[rest];
        const int x = rest ? it - live : it;
        int r = 0;  // the last rank whose first item is not past x
        for (int left = a.batch; left > 1;) {
          const int half = left / 2;
          if (f[r + half] <= x) r += half;
          left -= half;
        }
        const short2 s = sequence[r];
        const int each = rest ? per_head - s.y : s.y, h = (x - f[r]) / each;
        bh = s.x * a.heads + h;
        n = x - f[r] - h * each + (rest ? s.y : 0);
      }
      item[k] = make(bh, n);
    }
    return mine;
  }
};
template <>
struct ItemList<false> {};
}  // namespace

// ------------------------------------------------------------------ forward
// An item is two query tiles, each with its own group of four warps, that
// share the K / V blocks of their head (one tile where pairs would leave SMs
// idle).  Without lengths, the last tiles of heads with an odd number of tiles
// pair up across heads; such an item streams two K / V sequences in turn.
// (865 tokens are 7 tiles: 19 items a CTA instead of 21 at 64 images.)  TMEM: S of the tiles [0, 128) and
// [128, 256), P as bf16 [256, 320) and [320, 384), O [384, 448) and [448, 512).
// S is handed back as soon as it is in registers, so that the next block's is
// there when the warps ask for it: they are bound by their exponentials.
//
// The columns past a sequence's end get their -inf from the tensor core: one
// more MMA in the last block, a column of ones against a column of 0 and -inf.
// (As selects in the warps it took as long as the block's exponentials.)
//
// 64 images of 865 tokens, 12 heads: 242 us in a replayed graph, 610 TFLOP/s
// (259 once the card is at its power limit, 1.77 GHz; 261 from the caller).
// MUFU needs 124 of them, the products 91; the two tiles' hand-overs take the
// rest.
namespace {
constexpr uint32_t F_P = 256, F_O = 384;
constexpr size_t F_SMEM = 1024 + TILE_B * (4 + 2 * ST) + (ST + 1) * EXT_B + 512;
}  // namespace

template <bool LENS>
__global__ void __launch_bounds__(F_THREADS, 1)
    k_attn_forward_tc(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK,
                      const __grid_constant__ CUtensorMap tmV, const __grid_constant__ CUtensorMap tmO, AttnShape a,
                      HeadsView out, float* __restrict__ lse, int items, int per_head, int mixed_from, FastDiv by_head,
                      FastDiv by_batch, int tpi, int* err) {
  extern __shared__ uint8_t smem_raw[];
  __shared__ ItemList<LENS> list;
  // LENS: the launch has `items` items from `mixed_from` on (there is no mixing), `mine` of them are this CTA's
  [[maybe_unused]] int mine = 0;
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* sQ = smem;  // [item parity][tile], then the tile's output on its way out
  uint8_t* sK = smem + 4 * TILE_B;
  uint8_t* sV = sK + ST * TILE_B;
  uint8_t* sMask = sV + ST * TILE_B;  // [ST] the keys' column of 0 and -inf (without lengths the first serves all), then the ones
  uint64_t* bars = reinterpret_cast<uint64_t*>(sMask + (ST + 1) * EXT_B);
  uint64_t* q_full = bars;             // [2 item parities][2 tiles]
  uint64_t* q_empty = q_full + 4;      // [2 item parities][2 tiles]
  uint64_t* kv_full = q_empty + 4;     // [ST]
  uint64_t* kv_empty = kv_full + ST;   // [ST]
  uint64_t* kv_clean = kv_empty + ST;  // [ST] with lengths: what lies past them is zero
  uint64_t* s_full = kv_clean + ST;    // [2] tile
  uint64_t* s_free = s_full + 2;       // [2] tile: S read
  uint64_t* p_full = s_free + 2;       // [2] tile: P written
  uint64_t* p_free = p_full + 2;       // [2] tile: P used, O complete up to its block
  uint64_t* started = p_free + 2;      // tile 0 has read its first S
  uint64_t* stopped = started + 1;     // [2] every product of the tile done, after an error
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(stopped + 2);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  struct Item {
    int bh[2], q0[2];  // (sequence, head) and first query of its tiles
    int tiles;         // how many of its tiles have queries and keys
    int kvs;           // K / V sequences that it streams
    int nb, nq, nk;    // blocks of a sequence, its queries and keys
  };
  auto item_of = [&](int it) {
    Item r;
    r.kvs = 1;
    if constexpr (LENS) {
      const int4 e = list.item[it];
      r.bh[0] = r.bh[1] = e.x;
      r.q0[0] = e.y;
      r.q0[1] = r.q0[0] + TR;
      r.nq = e.z;
      r.nk = e.w;
      r.nb = (r.nk + TR - 1) / TR;
      r.tiles = r.nb == 0 || r.q0[0] >= r.nq ? 0 : tpi == 2 && r.q0[1] < r.nq ? 2 : 1;
      return r;
    }
    if (it < mixed_from) {
      r.bh[0] = r.bh[1] = by_head(it);
      r.q0[0] = (it - r.bh[0] * per_head) * tpi * TR;
      r.q0[1] = r.q0[0] + TR;
    } else {
      r.bh[0] = 2 * (it - mixed_from);
      r.bh[1] = r.bh[0] + 1;
      r.q0[0] = r.q0[1] = (a.nq - 1) / TR * TR;
      if (r.bh[1] < a.batch * a.heads)
        r.kvs = 2;
      else
        r.q0[1] = a.nq;  // the last head of an odd number
    }
    const int b = by_batch(r.bh[0]);  // (one length for all where two sequences meet)
    r.nq = seq_len(a.q_lens, b, a.nq);
    r.nk = seq_len(a.kv_lens, b, a.nk);
    r.nb = (r.nk + TR - 1) / TR;
    r.tiles = r.nb == 0 || r.q0[0] >= r.nq ? 0 : tpi == 2 && r.q0[1] < r.nq ? 2 : 1;
    return r;
  };

  if (threadIdx.x == 0) {
    for (int i = 0; i < 2; ++i) {
      mbar_init(&q_full[2 * i], 1);
      mbar_init(&q_full[2 * i + 1], 1);
      mbar_init(&q_empty[2 * i], 4);  // the tile's warps, once their output has left the buffer
      mbar_init(&q_empty[2 * i + 1], 4);
      mbar_init(&s_full[i], 1);
      mbar_init(&s_free[i], 4);
      mbar_init(&p_full[i], 4);
      mbar_init(&p_free[i], 1);
    }
    for (int i = 0; i < ST; ++i) {
      mbar_init(&kv_full[i], 1);
      mbar_init(&kv_empty[i], tpi);
      mbar_init(&kv_clean[i], 1);
    }
    mbar_init(started, 4);
    mbar_init(&stopped[0], 1);
    mbar_init(&stopped[1], 1);
    fence_mbar_init();
  }
  for (int i = threadIdx.x; i < (ST + 1) * TR * 2; i += F_THREADS) {
    const int tile = i / (TR * 2), r = i / 2 % TR;
    uint4 v = make_uint4(0, 0, 0, 0);
    if ((i & 1) == 0 && tile == ST) v.x = 0x3f80u;                                                      // 1
    if ((i & 1) == 0 && tile == 0 && a.kv_lens == nullptr && r >= (a.nk - 1) % TR + 1) v.x = 0xff80u;   // -inf
    *ext_piece(sMask + tile * EXT_B, r, i & 1) = v;
  }
  fence_proxy_async();
  if (warp == 1) {
    tmem_alloc(tmem_slot, 512);
    tmem_relinquish();
  }
  if constexpr (LENS)
    mine = list.build(a, a.q_lens, a.nq, a.kv_lens, a.nk, tpi * TR, per_head, mixed_from, items, [&](int bh, int n) {
      const int b = bh / a.heads;
      return make_int4(bh, n * tpi * TR, seq_len(a.q_lens, b, a.nq), seq_len(a.kv_lens, b, a.nk));
    });
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  constexpr uint32_t tmem = 0;  // all 512 columns are ours: they start at 0

  if (warp < 4) regs_dec<88>();
  if (warp == 0) {
    if (elect_one()) {
      uint32_t g = 0, c = 0;                   // blocks, items with work
      uint32_t used[2][2] = {{0, 0}, {0, 0}};  // [parity][tile]
      bool ok = true;
      for (int it = LENS ? 0u : blockIdx.x; it < (LENS ? mine : items) && ok; it += (LENS ? 1u : gridDim.x)) {
        const Item I = item_of(it);
        if (I.tiles == 0) continue;
        const int qb = c & 1;
        // a tile's buffer is handed back by the warps of that tile, for the items in which it had work
#pragma unroll
        for (int t = 0; t < 2; ++t)
          if (ok && t < I.tiles) {
            uint32_t& u = qb ? used[1][t] : used[0][t];
            if (u > 0) ok = thread_wait(&q_empty[qb * 2 + t], (u - 1) & 1, err, VK_DEV_TIMEOUT_PRODUCER);
            ++u;
          }
        if (!ok) break;
        ++c;
        const int b0 = by_batch(I.bh[0]), h0 = I.bh[0] - b0 * a.heads, b1 = by_batch(I.bh[1]), h1 = I.bh[1] - b1 * a.heads;
        mbar_arrive_expect_tx(&q_full[qb * 2], TILE_B);
        tma_load_4d(sQ + qb * 2 * TILE_B, &tmQ, &q_full[qb * 2], I.q0[0], h0, b0);
        if (I.tiles > 1) {
          mbar_arrive_expect_tx(&q_full[qb * 2 + 1], TILE_B);
          tma_load_4d(sQ + (qb * 2 + 1) * TILE_B, &tmQ, &q_full[qb * 2 + 1], I.q0[1], h1, b1);
        }
        for (int j = 0; j < I.nb * I.kvs; ++j, ++g) {
          const uint32_t st = g % ST;
          if (!(ok = thread_wait(&kv_empty[st], ((g / ST) & 1) ^ 1, err, VK_DEV_TIMEOUT_PRODUCER))) break;
          const bool second = I.kvs == 2 && (j & 1);
          const int y = (I.kvs == 2 ? j >> 1 : j) * TR, h = second ? h1 : h0, b = second ? b1 : b0;
          mbar_arrive_expect_tx(&kv_full[st], 2 * TILE_B);
          tma_load_4d(sK + st * TILE_B, &tmK, &kv_full[st], y, h, b);
          tma_load_4d(sV + st * TILE_B, &tmV, &kv_full[st], y, h, b);
        }
      }
      if (*reinterpret_cast<volatile int*>(err) != 0) {
        for (uint32_t i = g > ST ? g - ST : 0; i < g; ++i) drain(&kv_full[i % ST], (i / ST) & 1);
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (used[i >> 1][i & 1] > 0) drain(&q_full[i], (used[i >> 1][i & 1] - 1) & 1);
      }
    }
  } else if (warp == 1 || (warp == 3 && tpi > 1)) {
    // Each tile's MMAs come from a thread of their own, S a block ahead of P V:
    // one thread for both would have to wait for their hand-overs in a fixed
    // order.
    if (elect_one()) {
      constexpr uint32_t idS = idesc_bf16(128, 128), idO = idesc_bf16_bmn(128, 64);
      const int t = warp == 1 ? 0 : 1;
      uint64_t* kv_ready = a.kv_lens != nullptr ? kv_clean : kv_full;
      // One slot of the K / V ring: slot j of the c-th item with work, `mine` if
      // this tile uses it.
      struct Slot {
        int it, tiles, kvs, j, nb;
        uint32_t c, g;  // ordinals of the item and of the slot
        bool mine, ragged;  // ragged: the sequence's last block is not full
      };
      auto load = [&](Slot k) {
        for (; k.it < (LENS ? mine : items); k.it += (LENS ? 1u : gridDim.x)) {
          const Item I = item_of(k.it);
          k.tiles = I.tiles;
          k.kvs = I.kvs;
          k.nb = I.nb * I.kvs;
          k.ragged = I.nk % TR != 0;
          if (I.tiles > 0) break;
        }
        k.j = 0;
        k.mine = k.kvs == 2 ? t == 0 : t < k.tiles;
        return k;
      };
      auto next = [&](Slot k) {
        ++k.g;
        if (++k.j < k.nb) {
          if (k.kvs == 2) k.mine = !k.mine;
          return k;
        }
        k.it += (LENS ? 1u : gridDim.x);
        ++k.c;
        return load(k);
      };
      bool ok = true;
      auto wait = [&](uint64_t* bar, uint32_t parity) { return ok = ok && thread_wait(bar, parity & 1, err, VK_DEV_TIMEOUT_MMA); };
      // Lets slots of the other tile go (each is waited for, so that no phase is missed).
      auto skip = [&](Slot& k) {
        while (k.it < (LENS ? mine : items) && !k.mine && wait(&kv_ready[k.g % ST], k.g / ST)) {
          umma_commit(&kv_empty[k.g % ST]);
          k = next(k);
        }
      };
      // S of this tile's n-th block, once its last S has been read
      uint32_t uses[2] = {0, 0};  // of the tile's two query buffers
      auto issue_s = [&](const Slot& k, uint32_t n) {
        if (k.it >= (LENS ? mine : items) || !wait(&kv_ready[k.g % ST], k.g / ST)) return;
        if (k.j < k.kvs) wait(&q_full[(k.c & 1) * 2 + t], k.c & 1 ? uses[1]++ : uses[0]++);
        if (n > 0) wait(&s_free[t], n - 1);
        if (!ok) return;
        tc_fence_after();
        const uint64_t qd = smem_desc_k_sw128(smem_u32(sQ + ((k.c & 1) * 2 + t) * TILE_B));
        const uint64_t kd = smem_desc_k_sw128(smem_u32(sK + k.g % ST * TILE_B));
#pragma unroll
        for (int i = 0; i < 4; ++i) umma_f16(tmem + t * TR, qd + i * 2, kd + i * 2, idS, i > 0 ? 1u : 0u);
        if (k.ragged && k.j + k.kvs >= k.nb)
          umma_f16(tmem + t * TR, smem_desc_k16(smem_u32(sMask + ST * EXT_B)),
                   smem_desc_k16(smem_u32(sMask + (a.kv_lens != nullptr ? k.g % ST : 0) * EXT_B)), idS, 1u);
        umma_commit(&s_full[t]);
      };
      Slot k = load(Slot{static_cast<int>(LENS ? 0u : blockIdx.x), 0, 1, 0, 0, 0, 0, false, false});
      // Tile 1 starts when tile 0 is about to take its exponentials: half a
      // block apart, the two share MUFU in turn (in step they took 3600 cycles
      // for a block of both, 2048 of them MUFU's).
      if (t == 1 && k.it < (LENS ? mine : items)) wait(started, 0);
      skip(k);
      issue_s(k, 0);
      for (uint32_t n = 0; ok && k.it < (LENS ? mine : items); ++n) {
        // The next S goes first where it needs at most the slot after the next:
        // further on, the ring would wait for this block's.
        Slot b = next(k);
        const bool near = b.it < (LENS ? mine : items) && (b.mine || b.kvs == 2);
        if (near) {
          skip(b);
          issue_s(b, n + 1);
        }
        if (!wait(&p_full[t], n)) break;
        tc_fence_after();
        const uint64_t vd = smem_desc_mn_sw128(smem_u32(sV + k.g % ST * TILE_B));
        // (an item's first product overwrites O: its warps read the last item's before they hand over P)
#pragma unroll
        for (int i = 0; i < 8; ++i)
          umma_f16_ts(tmem + F_O + t * 64, tmem + F_P + t * 64 + i * 8, vd + static_cast<uint64_t>(i * (2048 >> 4)), idO,
                      k.j < k.kvs && i == 0 ? 0u : 1u);
        umma_commit(&p_free[t]);
        umma_commit(&kv_empty[k.g % ST]);
        if (!near) {
          skip(b);
          issue_s(b, n + 1);
        }
        k = b;
      }
      if (!ok) {
        umma_commit(&stopped[t]);
        drain(&stopped[t], 0);
      }
    }
  } else if (warp == 2 && a.kv_lens != nullptr) {
    uint32_t g = 0;
    bool ok = true;
    for (int it = LENS ? 0u : blockIdx.x; it < (LENS ? mine : items) && ok; it += (LENS ? 1u : gridDim.x)) {
      const Item I = item_of(it);
      if (I.tiles == 0) continue;
      for (int j = 0; j < I.nb; ++j, ++g) {  // (with lengths, an item streams one sequence)
        if (!(ok = warp_wait(&kv_full[g % ST], (g / ST) & 1, err, VK_DEV_TIMEOUT_OTHER))) break;
        const int valid = I.nk - j * TR;
        if (valid < TR) {
          for (int r = lane; r < TR; r += 32)
            *ext_piece(sMask + g % ST * EXT_B, r, 0) = make_uint4(r < valid ? 0u : 0xff80u, 0, 0, 0);
          zero_tail(sK + g % ST * TILE_B, sV + g % ST * TILE_B, valid, lane);
        }
        if (lane == 0) mbar_arrive(&kv_clean[g % ST]);
      }
    }
  } else if (warp >= 4) {
    regs_inc<208>();
    const int t = (warp - 4) >> 2, quad = warp & 3;
    const uint32_t lanes = static_cast<uint32_t>(quad * 32) << 16;
    const uint32_t ts = tmem + t * TR + lanes, tp = tmem + F_P + t * 64 + lanes, to = tmem + F_O + t * 64 + lanes;
    const float sl2 = a.scale * LOG2E;
    const int trow = quad * 32 + lane;
    uint32_t n = 0, c = 0;  // blocks of this tile, items with work
    int owed = -1;          // the Q buffer whose staged output is still leaving
    auto settle = [&]() {
      if (owed >= 0 && lane == 0) {
        bulk_wait_read<0>();
        mbar_arrive(&q_empty[owed * 2 + t]);
      }
      owed = -1;
    };
    bool ok = true;
    for (int it = LENS ? 0u : blockIdx.x; it < (LENS ? mine : items) && ok && t < tpi; it += (LENS ? 1u : gridDim.x)) {
      const Item I = item_of(it);
      const int bh = t ? I.bh[1] : I.bh[0], q0 = t ? I.q0[1] : I.q0[0], row = q0 + trow;
      const int b = by_batch(bh), h = bh - b * a.heads;
      float* lp = lse + static_cast<size_t>(bh) * a.nq + row;
      const int qb = c & 1;
      if (I.tiles > 0) ++c;
      if (t >= I.tiles) {  // no queries here, or no keys
        if (row < a.nq) {
          store_zeros(static_cast<__nv_bfloat16*>(out.p) + b * out.sb + h * out.sh + row * out.st);
          *lp = -INFINITY;
        }
        settle();
        continue;
      }
      float m_ref = 0.0f, l_run = 0.0f;
      for (int j = 0; j < I.nb; ++j, ++n) {
        if (!(ok = warp_wait(&s_full[t], n & 1, err, VK_DEV_TIMEOUT_EPILOGUE))) break;
        tc_fence_after();
        uint32_t r[128];
        tmem_ld128(ts, r);
        tc_fence_before();
        float pm[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
        for (int i = 0; i < 128; i += 2)
          pm[(i >> 1) & 3] = max3f(pm[(i >> 1) & 3], __uint_as_float(r[i]), __uint_as_float(r[i + 1]));
        const float top = fmaxf(fmaxf(pm[0], pm[1]), fmaxf(pm[2], pm[3])) * sl2;
        if (j == 0) m_ref = finite_ref(top);
        // p = 2^(s scale log2e - m) against a reference that stays while no
        // score is more than 2^20 over it: the quotient O / l does not depend
        // on it.  Then O (complete once P(n-1) is used) and l are rescaled.
        // A row without values in the block comes here too: an infinite query
        // makes NaN of the zeroed keys past the end, which the tensor core's
        // -inf cannot mask.  (Looked for in a branch of its own: 2% slower.)
        if (__any_sync(0xffffffffu, top > m_ref + 20.0f || top == -INFINITY)) {
          if (I.nk - j * TR < TR) mask_columns(r, I.nk - j * TR);
          if (j > 0) {
            if (!(ok = warp_wait(&p_free[t], (n - 1) & 1, err, VK_DEV_TIMEOUT_EPILOGUE))) break;
            tc_fence_after();
            const float m_new = fmaxf(m_ref, top), f = ex2_approx(m_ref - m_new);
#pragma unroll
            for (int d0 = 0; d0 < 64; d0 += 16) {
              uint32_t o[16];
              tmem_ld16(to + d0, o);
              tmem_wait_ld();
#pragma unroll
              for (int d = 0; d < 16; ++d) o[d] = __float_as_uint(__uint_as_float(o[d]) * f);
              tmem_st16(to + d0, o);
            }
            l_run *= f;
            m_ref = m_new;
          }
        }
        __syncwarp();
        if (lane == 0) {
          mbar_arrive(&s_free[t]);
          if (t == 0 && n == 0) mbar_arrive(started);
        }
        const float2 scale2 = make_float2(sl2, sl2), shift2 = make_float2(-m_ref, -m_ref);
        float2 ps[2] = {make_float2(0.0f, 0.0f), make_float2(0.0f, 0.0f)};
#pragma unroll
        for (int i = 0; i < 64; ++i) {
          const float2 p = exp2_pair(
              ffma2(make_float2(__uint_as_float(r[2 * i]), __uint_as_float(r[2 * i + 1])), scale2, shift2));
          ps[i & 1] = fadd2(ps[i & 1], p);
          r[i] = pack_bf16x2(p.x, p.y);  // (over scores that are done with)
        }
        l_run += (ps[0].x + ps[0].y) + (ps[1].x + ps[1].y);
        if (n > 0 && !(ok = warp_wait(&p_free[t], (n - 1) & 1, err, VK_DEV_TIMEOUT_EPILOGUE))) break;
        tc_fence_after();
        tmem_st32(tp, *reinterpret_cast<uint32_t(*)[32]>(&r[0]));
        tmem_st32(tp + 32, *reinterpret_cast<uint32_t(*)[32]>(&r[32]));
        tmem_wait_st();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&p_full[t]);
        if (j == 0) settle();
      }
      if (!ok || !(ok = warp_wait(&p_free[t], (n - 1) & 1, err, VK_DEV_TIMEOUT_EPILOGUE))) break;
      tc_fence_after();
      // staged over the tile's queries (every product is done with them)
      const bool live = row < I.nq && l_run != 0.0f;
      uint8_t* stage = sQ + (qb * 2 + t) * TILE_B + quad * 4096;
      stage_row(stage, lane, to, live ? 1.0f / l_run : 0.0f, live);
      tc_fence_before();
      send_rows(&tmO, stage, q0 + quad * 32, a.nq, h, b, lane);
      owed = qb;
      if (row < a.nq) *lp = live ? fmaf(m_ref, LN2, logf(l_run)) : -INFINITY;
    }
    if (lane == 0) bulk_wait<0>();
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
// blocks n = 0, 1, ...  The two groups of warps take the even
// and the odd blocks; for each a warp
//   reads S and hands it back   -> MMA: the next block's S = own1 . streamed1
//   p = 2^(S scale log2e - lse log2e); dk/dv: writes P
//                               -> MMA: dv += P^T . streamed2
//   reads dP and hands it back  -> MMA: the next block's dP = own2 . streamed2
//   dS = p (dP - delta); writes dS
//                               -> MMA: dk (dq) += dS . streamed1
// S and dP are handed back as soon as they are in registers, so the other
// group's are there before it asks, and one group's exponentials (MUFU, 16 a
// clock) run beside the other's products and TMEM traffic.
// dk/dv: the streamed rows' lse and delta belong to columns there, and reading
// them back from shared memory for every row would take more of its bandwidth
// than the operands do.  They enter the products instead, as three more
// columns each (bf16 hi + mid + lo, 24 bits) against ones: S becomes
// S - lse / scale and dP becomes dP - delta for two more MMAs a block.
//
// 64 images of 865 tokens, 12 heads: 599 us for both kernels in a replayed
// graph, 614 TFLOP/s of five products (860 of the seven that run); 693 once the
// card is at its power limit, 1.65 GHz, and 696 from the caller.  MUFU is 42 to 55% busy, the
// tensor pipe 41 to 45%: with one S, P and dS in tensor memory, which is full,
// the groups wait for one another.
namespace {
// TMEM: S [0, 128); dq: dP twice [128, 384), dS [384, 448), dq [448, 512);
// dk/dv: dP [128, 256), P [256, 320), dS [320, 384), dv [384, 448), dk [448, 512)
constexpr uint32_t COL_DP = 128, COL_P = 256, COL_ACC = 384;
constexpr int B_EXTRA = (ST + 2) * EXT_B;     // dk/dv: lse and delta of the streamed blocks, ones; dq: the tile of `out`, delta
constexpr size_t B_SMEM = 1024 + TILE_B * (4 + 2 * ST) + B_EXTRA + 512;
}  // namespace

// DQ: own rows are queries (own1 = q, own2 = d_out), streamed ones keys
// (k, v), acc = dq.  Otherwise own rows are keys (k, v), streamed ones queries
// (q, d_out), acc = dv, dk.
template <bool DQ, bool LENS>
__global__ void __launch_bounds__(B_THREADS, 1)
    k_attn_backward_tc(const __grid_constant__ CUtensorMap tmO1, const __grid_constant__ CUtensorMap tmO2,
                       const __grid_constant__ CUtensorMap tmS1, const __grid_constant__ CUtensorMap tmS2,
                       const __grid_constant__ CUtensorMap tmOut, const __grid_constant__ CUtensorMap tmG1,
                       const __grid_constant__ CUtensorMap tmG2, AttnShape a, const float* __restrict__ lse, float* delta,
                       HeadsView g1, HeadsView g2, int base, int count, int per_head, FastDiv by_head, FastDiv by_batch,
                       int* err) {
  extern __shared__ uint8_t smem_raw[];
  __shared__ ItemList<LENS> list;
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* sOwn = smem;  // [item parity][own1, own2], then the item's output on its way out
  uint8_t* s1 = smem + 4 * TILE_B;
  uint8_t* s2 = s1 + ST * TILE_B;
  uint8_t* sExt = s2 + ST * TILE_B;                             // dk/dv: [ST] lse and delta, then the ones of S and of dP
  uint8_t* sOut = sExt;                                         // dq: the item's tile of `out`, for delta
  float2* sRow = reinterpret_cast<float2*>(sOut + TILE_B);      // dq: [item parity][row] (-lse log2e, delta)
  uint64_t* bars = reinterpret_cast<uint64_t*>(sExt + B_EXTRA);
  uint64_t* own_full = bars;            // [2] item parity
  uint64_t* own_empty = own_full + 2;   // [2]
  uint64_t* st_full = own_empty + 2;    // [ST]
  uint64_t* st_empty = st_full + ST;    // [ST]
  uint64_t* st_clean = st_empty + ST;   // [ST] with lengths: what lies past them is zero
  uint64_t* s_full = st_clean + ST;     // [2] group
  uint64_t* dp_full = s_full + 2;       // [2] group
  uint64_t* ds_full = dp_full + 2;      // [2] group: dS written
  uint64_t* p_free = ds_full + 2;       // [2] group, dk/dv: its P used
  uint64_t* ds_free = p_free + 2;       // [2] group: its dS used
  uint64_t* acc_full = ds_free + 2;     // [2] item parity: the item's last products done
  uint64_t* part_full = acc_full + 2;   // [2] item parity, dq: delta written, the item's tile of `out` read
  uint64_t* dp_free = part_full + 2;    // [2] group: dP read
  uint64_t* s_free = dp_free + 2;       // S read
  uint64_t* p_full = s_free + 1;       // dk/dv: P written
  uint64_t* acc_free = p_full + 1;      // the item's accumulators read
  uint64_t* stopped = acc_free + 1;     // [2] every product of a thread done, after an error
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(stopped + 2);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int total_own = DQ ? a.nq : a.nk;
  // An item: 128 own rows of one (sequence, head), and what it streams.
  struct Item {
    int it, bh, r0, own, len, nb;  // own and streamed rows of the sequence, blocks
  };
  // This CTA's items are the list's, or every gridDim.x-th one below `items`.
  // seek: the one from `it` on that has own rows and something to stream
  // (it >= items: none); skipped(I) sees those before it.
  int items = count;
  auto seek = [&](int it, auto skipped) {
    Item I{};
    for (; it < items; it += (LENS ? 1u : gridDim.x)) {
      if constexpr (LENS) {
        const int4 e = list.item[it];
        I.bh = e.x;
        I.r0 = e.y;
        I.own = e.z;
        I.len = e.w;
      } else {
        I.bh = by_head(it);
        I.r0 = (it - I.bh * per_head) * TR;
        const int b = by_batch(I.bh);
        const int nq = seq_len(a.q_lens, b, a.nq), nk = seq_len(a.kv_lens, b, a.nk);
        I.own = DQ ? nq : nk;
        I.len = DQ ? nk : nq;
      }
      I.nb = I.r0 < I.own ? (I.len + TR - 1) / TR : 0;
      if (I.nb > 0) break;
      skipped(I);
    }
    I.it = it;
    return I;
  };
  auto nothing = [](const Item&) {};

  if (threadIdx.x == 0) {
    for (int i = 0; i < 2; ++i) {
      mbar_init(&own_full[i], 1);
      mbar_init(&own_empty[i], 4);
      mbar_init(&s_full[i], 1);
      mbar_init(&dp_full[i], 1);
      mbar_init(&ds_full[i], 4);
      mbar_init(&p_free[i], 1);
      mbar_init(&ds_free[i], 1);
      mbar_init(&acc_full[i], 1);
      mbar_init(&part_full[i], 4);
      mbar_init(&dp_free[i], 4);
      mbar_init(&stopped[i], 1);
    }
    mbar_init(s_free, 4);
    mbar_init(p_full, 4);
    mbar_init(acc_free, 4);
    for (int i = 0; i < ST; ++i) {
      mbar_init(&st_full[i], 1);
      mbar_init(&st_empty[i], 1);
      mbar_init(&st_clean[i], 1);
    }
    fence_mbar_init();
  }
  if constexpr (!DQ) {
    // 16-byte piece of row r: the first holds the columns that count, the second stays zero
    for (int i = threadIdx.x; i < (ST + 2) * TR * 2; i += B_THREADS) {
      const int tile = i / (TR * 2), r = i / 2 % TR, k = i & 1;
      uint4 v = make_uint4(0, 0, 0, 0);
      if (k == 0 && tile == ST) v = make_uint4(0x3f803f80u, 0x00003f80u, 0, 0);          // 1 1 1 0 0 0 0 0
      if (k == 0 && tile == ST + 1) v = make_uint4(0, 0x3f800000u, 0x3f803f80u, 0);      // 0 0 0 1 1 1 0 0
      *ext_piece(sExt + tile * EXT_B, r, k) = v;
    }
    fence_proxy_async();
  }
  if (warp == 1) {
    tmem_alloc(tmem_slot, 512);
    tmem_relinquish();
  }
  if constexpr (LENS) {
    const int32_t *own_lens = DQ ? a.q_lens : a.kv_lens, *other_lens = DQ ? a.kv_lens : a.q_lens;
    const int total_other = DQ ? a.nk : a.nq;
    items = list.build(a, own_lens, total_own, other_lens, total_other, TR, per_head, base, count, [&](int bh, int n) {
      const int b = bh / a.heads;
      return make_int4(bh, n * TR, seq_len(own_lens, b, total_own), seq_len(other_lens, b, total_other));
    });
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  constexpr uint32_t tmem = 0;  // all 512 columns are ours: they start at 0

  if (warp < 8) regs_dec<72>();
  if (warp == 0) {
    uint32_t n = 0, c = 0;        // blocks, items
    uint32_t sent = 0, owns = 0;  // how many of them are loaded or on their way
    bool ok = true;
    const float inv_scale = 1.0f / a.scale;
    for (Item I = seek(LENS ? 0u : blockIdx.x, nothing); ok && I.it < items; I = seek(I.it + (LENS ? 1u : gridDim.x), nothing), ++c) {
      const uint32_t ob = c & 1;
      const int b = by_batch(I.bh), h = I.bh - b * a.heads;
      if (c >= 2 && !(ok = warp_wait(&own_empty[ob], ((c >> 1) - 1) & 1, err, VK_DEV_TIMEOUT_PRODUCER))) break;
      if (DQ && c >= 1 && !(ok = warp_wait(&part_full[(c - 1) & 1], ((c - 1) >> 1) & 1, err, VK_DEV_TIMEOUT_PRODUCER))) break;
      if (lane == 0) {
        mbar_arrive_expect_tx(&own_full[ob], (DQ ? 3 : 2) * TILE_B);
        tma_load_4d(sOwn + (2 * ob) * TILE_B, &tmO1, &own_full[ob], I.r0, h, b);
        tma_load_4d(sOwn + (2 * ob + 1) * TILE_B, &tmO2, &own_full[ob], I.r0, h, b);
        if constexpr (DQ) tma_load_4d(sOut, &tmOut, &own_full[ob], I.r0, h, b);
      }
      owns = c + 1;
      for (int j = 0; j < I.nb; ++j, ++n) {
        const uint32_t st = n % ST;
        float l[4], d[4];
        if constexpr (!DQ) {
          // the streamed rows' -lse / scale and -delta.  Rows past the length
          // are zeros in q and d_out, so their p counts nothing; lse = -inf is
          // a row of scores of -inf only, whose p is 2^-inf without it too.
          const size_t at = static_cast<size_t>(I.bh) * a.nq;
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int row = j * TR + i * 32 + lane;
            l[i] = row < I.len ? lse[at + row] : 0.0f;
            d[i] = row < I.len ? -delta[at + row] : 0.0f;
            l[i] = l[i] == -INFINITY ? 0.0f : -l[i] * inv_scale;
          }
        }
        if (!(ok = warp_wait(&st_empty[st], ((n / ST) & 1) ^ 1, err, VK_DEV_TIMEOUT_PRODUCER))) break;
        if constexpr (!DQ) {
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int r = i * 32 + lane;
            float x[6];
            split3(l[i], x[0], x[1], x[2]);
            split3(d[i], x[3], x[4], x[5]);
            *ext_piece(sExt + st * EXT_B, r, 0) =
                make_uint4(pack_bf16x2(x[0], x[1]), pack_bf16x2(x[2], x[3]), pack_bf16x2(x[4], x[5]), 0u);
          }
          fence_proxy_async();
          __syncwarp();
        }
        if (lane == 0) {
          mbar_arrive_expect_tx(&st_full[st], 2 * TILE_B);
          tma_load_4d(s1 + st * TILE_B, &tmS1, &st_full[st], j * TR, h, b);
          tma_load_4d(s2 + st * TILE_B, &tmS2, &st_full[st], j * TR, h, b);
        }
        sent = n + 1;
      }
    }
    if (*reinterpret_cast<volatile int*>(err) != 0) {
      for (uint32_t i = sent > ST ? sent - ST : 0; i < sent; ++i) drain(&st_full[i % ST], (i / ST) & 1);
      for (uint32_t i = owns > 2 ? owns - 2 : 0; i < owns; ++i) drain(&own_full[i & 1], (i >> 1) & 1);
    }
  } else if (warp == 1 || warp == 3) {
    // Two threads issue the MMAs, one S and dP, one the sums: their hand-overs
    // come in no fixed order.
    if (elect_one()) {
      constexpr uint32_t idS = idesc_bf16(128, 128), idA = idesc_bf16_bmn(128, 64);
      uint64_t* st_ready = (DQ ? a.kv_lens : a.q_lens) != nullptr ? st_clean : st_full;
      // One block of the walk: block j of nb of the c-th item with work.
      struct Blk {
        int it, j, nb;
        uint32_t c;
        bool ok;
      };
      auto load = [&](int it, uint32_t c) {
        const Item I = seek(it, nothing);
        return Blk{I.it, 0, I.nb, c, I.it < items};
      };
      auto next = [&](Blk k) {
        if (k.ok && ++k.j == k.nb) k = load(k.it + (LENS ? 1u : gridDim.x), k.c + 1);
        return k;
      };
      bool ok = true;
      auto wait = [&](uint64_t* bar, uint32_t parity) { return ok = ok && thread_wait(bar, parity & 1, err, VK_DEV_TIMEOUT_MMA); };
      Blk b0 = load(LENS ? 0u : blockIdx.x, 0);
      if (warp == 1) {
        auto product = [&](uint32_t col, const uint8_t* own, const uint8_t* streamed, uint32_t st, int ones) {
          tc_fence_after();
          const uint64_t od = smem_desc_k_sw128(smem_u32(own)), sd = smem_desc_k_sw128(smem_u32(streamed));
#pragma unroll
          for (int k = 0; k < 4; ++k) umma_f16(tmem + col, od + k * 2, sd + k * 2, idS, k > 0 ? 1u : 0u);
          if constexpr (!DQ)
            umma_f16(tmem + col, smem_desc_k16(smem_u32(sExt + (ST + ones) * EXT_B)), smem_desc_k16(smem_u32(sExt + st * EXT_B)),
                     idS, 1u);
        };
        // S of block n, once block n - 1's has been read
        auto issue_s = [&](const Blk& k, uint32_t n) {
          if (k.j == 0) wait(&own_full[k.c & 1], k.c >> 1);
          if (!wait(&st_ready[n % ST], n / ST) || (n > 0 && !wait(s_free, n - 1))) return;
          product(0, sOwn + (k.c & 1) * 2 * TILE_B, s1 + n % ST * TILE_B, n % ST, 0);
          umma_commit(&s_full[n & 1]);
        };
        auto issue_dp = [&](const Blk& k, uint32_t n) {
          // (dq has two of them)
          if (DQ ? n > 1 && !wait(&dp_free[n & 1], (n >> 1) - 1) : n > 0 && !wait(&dp_free[(n - 1) & 1], (n - 1) >> 1)) return;
          product(COL_DP + (DQ ? (n & 1) * TR : 0), sOwn + ((k.c & 1) * 2 + 1) * TILE_B, s2 + n % ST * TILE_B, n % ST, 1);
          umma_commit(&dp_full[n & 1]);
        };
        if constexpr (DQ) {
          for (uint32_t n = 0; ok && b0.ok; ++n, b0 = next(b0)) {
            issue_s(b0, n);
            if (ok) issue_dp(b0, n);
          }
        } else {
          Blk b1 = next(b0), b2 = next(b1);
          if (b0.ok) {
            issue_s(b0, 0);
            if (ok) issue_dp(b0, 0);
          }
          if (ok && b1.ok) issue_s(b1, 1);
          for (uint32_t n = 0; ok && b1.ok; ++n) {
            // S(n+2) early -- unless its item takes over the tiles of block n's
            const bool late = b2.c >= b0.c + 2;
            if (b2.ok && !late) issue_s(b2, n + 2);
            if (ok) issue_dp(b1, n + 1);
            if (ok && b2.ok && late) issue_s(b2, n + 2);
            b0 = b1;
            b1 = b2;
            b2 = next(b2);
          }
        }
      } else {
        // acc += A . streamed, A = 64 columns of TMEM from `col` on
        auto sum = [&](uint32_t acc, uint32_t col, const uint8_t* streamed, bool fresh) {
          tc_fence_after();
          const uint64_t sd = smem_desc_mn_sw128(smem_u32(streamed));
#pragma unroll
          for (int k = 0; k < 8; ++k)
            umma_f16_ts(tmem + acc, tmem + col + k * 8, sd + static_cast<uint64_t>(k * (2048 >> 4)), idA, fresh && k == 0 ? 0u : 1u);
        };
        auto acc_ready = [&](const Blk& k) {  // the last item's accumulators have been read
          return k.j > 0 || k.c == 0 || wait(acc_free, k.c - 1);
        };
        for (uint32_t n = 0; b0.ok; ++n) {
          if constexpr (!DQ) {
            if (!wait(p_full, n) || !acc_ready(b0)) break;
            sum(COL_ACC, COL_P, s2 + n % ST * TILE_B, b0.j == 0);  // dv += P^T d_out
            umma_commit(&p_free[n & 1]);
          }
          if (!wait(&ds_full[n & 1], n >> 1) || (DQ && !acc_ready(b0))) break;
          if constexpr (DQ)
            sum(COL_ACC + 64, COL_ACC, s1 + n % ST * TILE_B, b0.j == 0);  // dq += dS k
          else
            sum(COL_ACC + 64, COL_P + 64, s1 + n % ST * TILE_B, b0.j == 0);  // dk += dS^T q
          umma_commit(&ds_free[n & 1]);
          umma_commit(&st_empty[n % ST]);
          if (b0.j + 1 == b0.nb) umma_commit(&acc_full[b0.c & 1]);
          b0 = next(b0);
        }
      }
      if (!ok) {
        umma_commit(&stopped[warp >> 1]);
        drain(&stopped[warp >> 1], 0);
      }
    }
  } else if (warp == 2 && (DQ ? a.kv_lens : a.q_lens) != nullptr) {
    uint32_t n = 0;
    bool ok = true;
    for (Item I = seek(LENS ? 0u : blockIdx.x, nothing); ok && I.it < items; I = seek(I.it + (LENS ? 1u : gridDim.x), nothing))
      for (int j = 0; j < I.nb; ++j, ++n) {
        if (!(ok = warp_wait(&st_full[n % ST], (n / ST) & 1, err, VK_DEV_TIMEOUT_OTHER))) break;
        if (I.len - j * TR < TR) zero_tail(s1 + n % ST * TILE_B, s2 + n % ST * TILE_B, I.len - j * TR, lane);
        if (lane == 0) mbar_arrive(&st_clean[n % ST]);
      }
  } else if (warp >= 4 && warp < 8) {
    const int quad = warp & 3, trow = quad * 32 + lane;
    const uint32_t lanes = static_cast<uint32_t>(quad * 32) << 16;
    auto skipped = [&](const Item& I) {  // no own rows, or nothing to stream: zeros
      const int row = I.r0 + trow;
      if (row >= total_own) return;
      const int b = by_batch(I.bh), h = I.bh - b * a.heads;
      store_zeros(static_cast<__nv_bfloat16*>(g1.p) + b * g1.sb + h * g1.sh + row * g1.st);
      if constexpr (DQ)
        delta[static_cast<size_t>(I.bh) * a.nq + row] = 0.0f;
      else
        store_zeros(static_cast<__nv_bfloat16*>(g2.p) + b * g2.sb + h * g2.sh + row * g2.st);
    };
    // dq: the rows' -lse log2e and delta (from the tiles of out and d_out), a
    // row per thread, an item ahead of the warps that use them
    auto row_delta = [&](const Item& I, uint32_t c) {
      const int row = I.r0 + trow;
      const size_t at = static_cast<size_t>(I.bh) * a.nq + row;
      const float e = row < I.own ? lse[at] : 0.0f;
      if (!warp_wait(&own_full[c & 1], (c >> 1) & 1, err, VK_DEV_TIMEOUT_EPILOGUE)) return false;
      const uint8_t* og = sOwn + ((c & 1) * 2 + 1) * TILE_B;
      float x[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int at = trow * 128 + ((i ^ trow) & 7) * 16;
        const uint4 ov = *reinterpret_cast<const uint4*>(sOut + at), gv = *reinterpret_cast<const uint4*>(og + at);
        const uint32_t o[4] = {ov.x, ov.y, ov.z, ov.w}, g[4] = {gv.x, gv.y, gv.z, gv.w};
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          x[u & 1] = fmaf(__uint_as_float(o[u] << 16), __uint_as_float(g[u] << 16), x[u & 1]);
          x[2 + (u & 1)] = fmaf(__uint_as_float(o[u] & 0xffff0000u), __uint_as_float(g[u] & 0xffff0000u), x[2 + (u & 1)]);
        }
      }
      const float dl = (x[0] + x[1]) + (x[2] + x[3]);
      // lse = -inf: a row of scores of -inf only, whose p is 2^(-inf - 0) = 0
      sRow[(c & 1) * TR + trow] = make_float2(e == -INFINITY ? 0.0f : -e * LOG2E, dl);
      __syncwarp();
      if (lane == 0) mbar_arrive(&part_full[c & 1]);
      if (row < total_own) delta[at] = row < I.own ? dl : 0.0f;
      return true;
    };
    Item I = seek(LENS ? 0u : blockIdx.x, skipped);
    bool ok = !DQ || I.it >= items || row_delta(I, 0);
    for (uint32_t c = 0; ok && I.it < items; ++c) {
      const Item N = seek(I.it + (LENS ? 1u : gridDim.x), skipped);
      if (DQ && N.it < items && !(ok = row_delta(N, c + 1))) break;
      // the item's accumulators to memory, staged over its own tiles (every product is done with them)
      if (!(ok = warp_wait(&acc_full[c & 1], (c >> 1) & 1, err, VK_DEV_TIMEOUT_EPILOGUE))) break;
      tc_fence_after();
      const bool live = I.r0 + trow < I.own;
      const int b = by_batch(I.bh), h = I.bh - b * a.heads, y = I.r0 + quad * 32;
      uint8_t* stage = sOwn + (c & 1) * 2 * TILE_B + quad * 4096;
      stage_row(stage, lane, tmem + COL_ACC + (DQ ? 64 : 0) + lanes, DQ ? a.scale : 1.0f, live);
      if constexpr (!DQ) stage_row(stage + TILE_B, lane, tmem + COL_ACC + 64 + lanes, a.scale, live);
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(acc_free);
      send_rows(&tmG1, stage, y, total_own, h, b, lane);
      if constexpr (!DQ) send_rows(&tmG2, stage + TILE_B, y, total_own, h, b, lane);
      if (lane == 0) {
        bulk_wait_read<0>();
        mbar_arrive(&own_empty[c & 1]);
      }
      I = N;
    }
    if (lane == 0) bulk_wait<0>();
  } else if (warp >= 8) {
    regs_inc<184>();
    const int quad = warp & 3, grp = (warp - 8) >> 2;
    const uint32_t lanes = static_cast<uint32_t>(quad * 32) << 16;
    const uint32_t ts = tmem + lanes;
    const uint32_t tp = tmem + COL_P + lanes, td = tmem + (DQ ? COL_ACC : COL_P + 64) + lanes;
    const uint32_t tdp = tmem + COL_DP + (DQ ? grp * TR : 0) + lanes;
    const float sl2 = a.scale * LOG2E;
    const int trow = quad * 32 + lane;
    Item I = seek(LENS ? 0u : blockIdx.x, nothing);
    uint32_t n0 = 0, c = 0;  // blocks and items before this one
    bool ok = true;
    for (; ok && I.it < items; n0 += I.nb, ++c, I = seek(I.it + (LENS ? 1u : gridDim.x), nothing)) {
      float2 shift2 = make_float2(0.0f, 0.0f), delta2 = shift2;
      bool fresh = true;  // this group has had no block of the item yet
      for (int j = (n0 ^ grp) & 1; j < I.nb; j += 2) {
        const uint32_t n = n0 + j;
        if (DQ && fresh) {
          if (!(ok = warp_wait(&part_full[c & 1], (c >> 1) & 1, err, VK_DEV_TIMEOUT_EPILOGUE))) break;
          const float2 x = sRow[(c & 1) * TR + trow];
          shift2 = make_float2(x.x, x.x);
          delta2 = make_float2(x.y, x.y);
          fresh = false;
        }
        if (!(ok = warp_wait(&s_full[grp], (n >> 1) & 1, err, VK_DEV_TIMEOUT_EPILOGUE))) break;
        tc_fence_after();
        float p[128];
        {
          uint32_t r[128];
          tmem_ld128(ts, r);
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(s_free);
          // Streamed rows past the end are zeros: whatever finite P and dS a
          // score of 0 gives there count nothing.  They stay finite unless the
          // row's lse is far below 0 (dq) or an own row is infinite.
          if (I.len - j * TR < TR && __any_sync(0xffffffffu, !(shift2.x < 60.0f) || __uint_as_float(r[127]) != 0.0f))
            mask_columns(r, I.len - j * TR);
#pragma unroll
          for (int i = 0; i < 64; ++i) {
            const float2 s = make_float2(__uint_as_float(r[2 * i]), __uint_as_float(r[2 * i + 1])), f = make_float2(sl2, sl2);
            const float2 e = exp2_pair(DQ ? ffma2(s, f, shift2) : fmul2(s, f));
            p[2 * i] = e.x, p[2 * i + 1] = e.y;
          }
        }
        if constexpr (!DQ) {
          if (n > 0 && !(ok = warp_wait(&p_free[(n - 1) & 1], ((n - 1) >> 1) & 1, err, VK_DEV_TIMEOUT_EPILOGUE))) break;
          tc_fence_after();
#pragma unroll
          for (int q = 0; q < 8; ++q) {
            uint32_t pk[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) pk[i] = pack_bf16x2(p[q * 16 + 2 * i], p[q * 16 + 2 * i + 1]);
            tmem_st8(tp + q * 8, pk);
          }
          tmem_wait_st();
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(p_full);
        }
        if (!(ok = warp_wait(&dp_full[grp], (n >> 1) & 1, err, VK_DEV_TIMEOUT_EPILOGUE))) break;
        tc_fence_after();
        uint32_t r[2][16];
        tmem_ld16(tdp, r[0]);
#pragma unroll
        for (int q = 0; q < 8; ++q) {
          tmem_wait_ld();
          if (q < 7) tmem_ld16(tdp + (q + 1) * 16, r[(q + 1) & 1]);
          if (q == 7) {
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&dp_free[grp]);
          }
          const uint32_t(&d)[16] = r[q & 1];
          uint32_t pk[8];
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            float2 dp = make_float2(__uint_as_float(d[2 * i]), __uint_as_float(d[2 * i + 1]));
            if constexpr (DQ) dp = fsub2(dp, delta2);
            const float2 ds = fmul2(dp, make_float2(p[q * 16 + 2 * i], p[q * 16 + 2 * i + 1]));
            pk[i] = pack_bf16x2(ds.x, ds.y);
          }
          if (q == 0 && n > 0) {
            if (!(ok = warp_wait(&ds_free[(n - 1) & 1], ((n - 1) >> 1) & 1, err, VK_DEV_TIMEOUT_EPILOGUE))) break;
            tc_fence_after();
          }
          tmem_st8(td + q * 8, pk);
        }
        if (!ok) break;
        tmem_wait_st();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&ds_full[grp]);
      }
    }
  }
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

// ------------------------------------------------------------------ launches
namespace {
bool heads_map(CUtensorMap* m, const HeadsView& v, int batch, int heads, int tokens, uint32_t rows = TR) {
  const uint64_t dims[4] = {64, static_cast<uint64_t>(tokens), static_cast<uint64_t>(heads), static_cast<uint64_t>(batch)};
  const uint64_t strides[3] = {static_cast<uint64_t>(v.st) * 2, static_cast<uint64_t>(v.sh) * 2, static_cast<uint64_t>(v.sb) * 2};
  const uint32_t box[4] = {64, rows, 1, 1};
  return make_tmap_nd(m, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, v.p, 4, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_128B);
}
// One CTA per SM; with lengths a launch takes as many items as the lists hold.
template <class F>
cudaError_t over_items(int items, bool lens, F launch) {
  const int sms = num_sms(), most = lens ? sms * LIST_MAX : items;
  for (int base = 0; base < items; base += most) {
    const int count = items - base < most ? items - base : most;
    launch(base, count, count < sms ? count : sms);
    const cudaError_t e = cudaGetLastError();
    if (e != cudaSuccess) return e;
  }
  return cudaSuccess;
}
}  // namespace

cudaError_t attention_forward_tc(const AttnShape& a, HeadsView q, HeadsView k, HeadsView v, HeadsView out, float* lse,
                                 int* err, cudaStream_t s) {
  CUtensorMap mq, mk, mv, mo;
  if (!heads_map(&mq, q, a.batch, a.heads, a.nq) || !heads_map(&mk, k, a.batch, a.heads, a.nk) ||
      !heads_map(&mv, v, a.batch, a.heads, a.nk) || !heads_map(&mo, out, a.batch, a.heads, a.nq, 32))
    return cudaErrorInvalidValue;
  const bool lens = a.q_lens != nullptr || a.kv_lens != nullptr;
  auto kernel = lens ? k_attn_forward_tc<true> : k_attn_forward_tc<false>;
  const cudaError_t e = ensure_smem_limit(reinterpret_cast<const void*>(kernel), static_cast<int>(F_SMEM));
  if (e != cudaSuccess) return e;
  // Two query tiles share each K / V block; one where pairs would leave SMs idle.
  const int nt = (a.nq + TR - 1) / TR, bh = a.batch * a.heads;
  const int tpi = (nt + 1) / 2 * bh < num_sms() ? 1 : 2;
  int per_head = (nt + tpi - 1) / tpi, items = per_head * bh, mixed_from = items;
  if (tpi == 2 && nt % 2 == 1 && !lens) {
    per_head = nt / 2;
    mixed_from = per_head * bh;
    items = mixed_from + (bh + 1) / 2;
  }
  const FastDiv by_head(per_head > 0 ? per_head : 1), by_batch(a.heads);
  return over_items(items, lens, [&](int base, int count, int grid) {
    kernel<<<grid, F_THREADS, F_SMEM, s>>>(mq, mk, mv, mo, a, out, lse, count, per_head, lens ? base : mixed_from, by_head,
                                           by_batch, tpi, err);
  });
}

cudaError_t attention_backward_tc(const AttnShape& a, HeadsView q, HeadsView k, HeadsView v, HeadsView out,
                                  const float* lse, HeadsView d_out, HeadsView dq, HeadsView dk, HeadsView dv,
                                  float* delta, int* err, cudaStream_t s) {
  CUtensorMap mq, mk, mv, mg, mo, mdq, mdk, mdv;
  if (!heads_map(&mq, q, a.batch, a.heads, a.nq) || !heads_map(&mk, k, a.batch, a.heads, a.nk) ||
      !heads_map(&mv, v, a.batch, a.heads, a.nk) || !heads_map(&mg, d_out, a.batch, a.heads, a.nq) ||
      !heads_map(&mo, out, a.batch, a.heads, a.nq) || !heads_map(&mdq, dq, a.batch, a.heads, a.nq, 32) ||
      !heads_map(&mdk, dk, a.batch, a.heads, a.nk, 32) || !heads_map(&mdv, dv, a.batch, a.heads, a.nk, 32))
    return cudaErrorInvalidValue;
  const bool lens = a.q_lens != nullptr || a.kv_lens != nullptr;
  const int bh = a.batch * a.heads, qt = (a.nq + TR - 1) / TR, kt = (a.nk + TR - 1) / TR;
  const FastDiv by_batch(a.heads);
  auto dq_kernel = lens ? k_attn_backward_tc<true, true> : k_attn_backward_tc<true, false>;
  auto dkdv_kernel = lens ? k_attn_backward_tc<false, true> : k_attn_backward_tc<false, false>;
  cudaError_t e = ensure_smem_limit(reinterpret_cast<const void*>(dq_kernel), static_cast<int>(B_SMEM));
  if (e == cudaSuccess) e = ensure_smem_limit(reinterpret_cast<const void*>(dkdv_kernel), static_cast<int>(B_SMEM));
  if (e == cudaSuccess)
    e = over_items(qt * bh, lens, [&](int base, int count, int grid) {
      dq_kernel<<<grid, B_THREADS, B_SMEM, s>>>(mq, mg, mk, mv, mo, mdq, mdq, a, lse, delta, dq, dq, base, count, qt,
                                                FastDiv(qt), by_batch, err);
    });
  if (e != cudaSuccess) return e;
  return over_items(kt * bh, lens, [&](int base, int count, int grid) {
    dkdv_kernel<<<grid, B_THREADS, B_SMEM, s>>>(mk, mv, mq, mg, mo, mdv, mdk, a, lse, delta, dv, dk, base, count, kt,
                                                FastDiv(kt), by_batch, err);
  });
}

}  // namespace vk
