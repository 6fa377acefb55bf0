// vk_abi_train.cu -- the C ABI of the trainable block pieces: argument checks
// and launches.  Nothing here allocates or synchronises, so every call can be
// captured into a CUDA graph.
#include <math.h>

#include <algorithm>
#include <cmath>

#include "vestra_b200.h"
#include "vk_abi_internal.h"
#include "vk_internal.h"
#include "vk_train.h"

using namespace vk;

namespace {

// The context's device for one call; the caller's device comes back after it.
class DeviceGuard {
 public:
  explicit DeviceGuard(int device) {
    if (cudaGetDevice(&before_) != cudaSuccess) before_ = device;
    if (before_ != device) cudaSetDevice(device);
    changed_ = before_ != device;
  }
  ~DeviceGuard() {
    if (changed_) cudaSetDevice(before_);
  }

 private:
  int before_ = 0;
  bool changed_ = false;
};

// A C entry point throws nothing: the only exceptions below are the standard
// library's, out of host memory.
template <class F>
int guarded(vk_ctx* ctx, const char* name, F body) {
  if (ctx == nullptr) return vk_fail(VK_ERR_INVALID_ARGUMENT, "%s: NULL context", name);
  try {
    DeviceGuard device(ctx->device);
    return body();
  } catch (...) {
    return VK_ERR_OUT_OF_MEMORY;
  }
}

int dtype_ok(const char* name, int dtype) {
  if (dtype == VK_DTYPE_F32 || dtype == VK_DTYPE_BF16) return VK_OK;
  return vk_fail(VK_ERR_INVALID_ARGUMENT, "%s: unknown element type %d", name, dtype);
}

// Checks one tensor [batch, heads, tokens, dim] and returns its view; strides
// of dimensions of one element do not matter and become those of a packed
// tensor.  `align`: bytes that the base and the strides are multiples of.
int heads_view(const char* name, const char* what, const vk_heads* x, int dtype, size_t batch, size_t heads,
               size_t tokens, size_t dim, size_t align, HeadsView* out) {
  if (x == nullptr || x->data == nullptr) return vk_fail(VK_ERR_INVALID_ARGUMENT, "%s: %s is NULL", name, what);
  const int64_t size = dtype == VK_DTYPE_F32 ? 4 : 2;
  const size_t count[3] = {tokens, heads, batch};
  int64_t stride[3] = {x->token_stride, x->head_stride, x->batch_stride};
  const int64_t packed[3] = {static_cast<int64_t>(dim), static_cast<int64_t>(dim * tokens),
                             static_cast<int64_t>(dim * tokens * heads)};
  if (reinterpret_cast<uintptr_t>(x->data) % align != 0)
    return vk_fail(VK_ERR_INVALID_ARGUMENT, "%s: %s is not aligned to %zu bytes", name, what, align);
  int order[3], n = 0;
  for (int i = 0; i < 3; ++i) {
    if (count[i] <= 1) {
      stride[i] = packed[i];
      continue;
    }
    if (stride[i] <= 0 || stride[i] > (int64_t{1} << 38))  // 2^38 elements: below the 2^40 bytes of a tensor map
      return vk_fail(VK_ERR_INVALID_ARGUMENT, "%s: %s has a stride of %lld", name, what, (long long)stride[i]);
    if (stride[i] * size % static_cast<int64_t>(align) != 0)
      return vk_fail(VK_ERR_INVALID_ARGUMENT, "%s: a stride of %s is not a multiple of %zu bytes", name, what, align);
    order[n++] = i;
  }
  std::sort(order, order + n, [&](int a, int b) { return stride[a] < stride[b]; });
  int64_t extent = static_cast<int64_t>(dim);
  for (int i = 0; i < n; ++i) {
    const int d = order[i];
    if (stride[d] < extent) return vk_fail(VK_ERR_INVALID_ARGUMENT, "%s: %s overlaps itself", name, what);
    extent = (static_cast<int64_t>(count[d]) - 1) * stride[d] + extent;
  }
  out->p = x->data;
  out->st = stride[0];
  out->sh = stride[1];
  out->sb = stride[2];
  return VK_OK;
}

int attention_shape(const char* name, const vk_attention_shape* s, AttnShape* a) {
  if (s == nullptr) return vk_fail(VK_ERR_INVALID_ARGUMENT, "%s: shape is NULL", name);
  VK_TRY(dtype_ok(name, s->dtype));
  VK_TRY(vk_dims_fit(name, {s->batch, s->heads, s->q_tokens, s->kv_tokens, s->head_dim}));
  if (s->head_dim != 8 && s->head_dim != 16 && s->head_dim != 32 && s->head_dim != 64)
    return vk_fail(VK_UNSUPPORTED_SHAPE, "%s: head_dim %zu (supported: 8, 16, 32, 64)", name, s->head_dim);
  // tiles of 64 rows are counted in an int
  const size_t tiles = std::max(s->q_tokens, s->kv_tokens) / 64 + 1;
  if (tiles > (1 << 24) || (s->batch != 0 && s->heads > static_cast<size_t>(INT_MAX) / s->batch / tiles))
    return vk_fail(VK_UNSUPPORTED_SHAPE, "%s: more than 2^30 tokens or 2^31 tiles", name);
  if (!(std::isfinite(s->scale) && s->scale > 0.0f))
    return vk_fail(VK_ERR_INVALID_ARGUMENT, "%s: scale must be finite and positive", name);
  if (reinterpret_cast<uintptr_t>(s->q_lens) % 4 != 0 || reinterpret_cast<uintptr_t>(s->kv_lens) % 4 != 0)
    return vk_fail(VK_ERR_INVALID_ARGUMENT, "%s: lengths are not aligned", name);
  a->batch = static_cast<int>(s->batch);
  a->heads = static_cast<int>(s->heads);
  a->nq = static_cast<int>(s->q_tokens);
  a->nk = static_cast<int>(s->kv_tokens);
  a->dim = static_cast<int>(s->head_dim);
  a->scale = s->scale;
  a->q_lens = s->q_lens;
  a->kv_lens = s->kv_lens;
  return VK_OK;
}

int floats_ok(const char* name, const char* what, const float* p, size_t align = 4) {
  if (p == nullptr) return vk_fail(VK_ERR_INVALID_ARGUMENT, "%s: %s is NULL", name, what);
  if (reinterpret_cast<uintptr_t>(p) % align != 0)
    return vk_fail(VK_ERR_INVALID_ARGUMENT, "%s: %s is not aligned to %zu bytes", name, what, align);
  return VK_OK;
}

// Outputs that start where an input or another output does would be written
// while they are read.  (NULL: not there.)
int apart(const char* name, std::initializer_list<const void*> outs, std::initializer_list<const void*> ins) {
  for (const void* const* o = outs.begin(); o != outs.end(); ++o) {
    if (*o == nullptr) continue;
    for (const void* i : ins)
      if (*o == i) return vk_fail(VK_ERR_INVALID_ARGUMENT, "%s: an output is one of the inputs", name);
    for (const void* const* p = outs.begin(); p != o; ++p)
      if (*o == *p) return vk_fail(VK_ERR_INVALID_ARGUMENT, "%s: two outputs are the same", name);
  }
  return VK_OK;
}

}  // namespace

// ------------------------------------------------------------------ attention
extern "C" int vk_attention_forward(vk_ctx* ctx, const vk_attention_shape* shape, const vk_heads* q, const vk_heads* k,
                                    const vk_heads* v, const vk_heads* out, float* lse) {
  static const char* name = "vk_attention_forward";
  return guarded(ctx, name, [&]() -> int {
    AttnShape a;
    VK_TRY(attention_shape(name, shape, &a));
    const size_t B = shape->batch, H = shape->heads, D = shape->head_dim;
    if (B == 0 || H == 0 || a.nq == 0) return VK_OK;
    const bool bf16 = shape->dtype == VK_DTYPE_BF16;
    HeadsView vq, vk_, vv, vo;
    VK_TRY(heads_view(name, "out", out, shape->dtype, B, H, a.nq, D, 16, &vo));
    VK_TRY(floats_ok(name, "lse", lse));
    if (a.nk == 0) {
      VK_TRY_CUDA(zero_heads(vo, bf16, a.batch, a.heads, a.nq, a.dim, ctx->stream), name);
      return vk_cuda_status(fill_f32(lse, B * H * a.nq, -INFINITY, ctx->stream), name);
    }
    VK_TRY(heads_view(name, "q", q, shape->dtype, B, H, a.nq, D, 16, &vq));
    VK_TRY(heads_view(name, "k", k, shape->dtype, B, H, a.nk, D, 16, &vk_));
    VK_TRY(heads_view(name, "v", v, shape->dtype, B, H, a.nk, D, 16, &vv));
    VK_TRY(apart(name, {vo.p, lse}, {vq.p, vk_.p, vv.p}));
    // One query alone needs no tile: 12 heads of 3457 keys 61 us from the caller
    // (90 as a tile of 128 rows on the tensor cores), 1536 heads 372 (379).  Of
    // two queries the exponentials count already: 1536 heads 886 (371).
    if (bf16 && a.dim == 64 && a.nq > 1)
      return vk_cuda_status(attention_forward_tc(a, vq, vk_, vv, vo, lse, ctx->d_err, ctx->stream), name);
    return vk_cuda_status(attention_forward_simt(a, bf16, vq, vk_, vv, vo, lse, ctx->stream), name);
  });
}

extern "C" int vk_attention_backward(vk_ctx* ctx, const vk_attention_shape* shape, const vk_heads* q, const vk_heads* k,
                                     const vk_heads* v, const vk_heads* out, const float* lse, const vk_heads* d_out,
                                     const vk_heads* dq, const vk_heads* dk, const vk_heads* dv, float* delta) {
  static const char* name = "vk_attention_backward";
  return guarded(ctx, name, [&]() -> int {
    AttnShape a;
    VK_TRY(attention_shape(name, shape, &a));
    const size_t B = shape->batch, H = shape->heads, D = shape->head_dim;
    if (B == 0 || H == 0 || (a.nq == 0 && a.nk == 0)) return VK_OK;
    const bool bf16 = shape->dtype == VK_DTYPE_BF16;
    cudaStream_t s = ctx->stream;
    HeadsView vq, vk_, vv, vo, vg, vdq, vdk, vdv;
    if (a.nq != 0) VK_TRY(heads_view(name, "dq", dq, shape->dtype, B, H, a.nq, D, 16, &vdq));
    if (a.nk != 0) {
      VK_TRY(heads_view(name, "dk", dk, shape->dtype, B, H, a.nk, D, 16, &vdk));
      VK_TRY(heads_view(name, "dv", dv, shape->dtype, B, H, a.nk, D, 16, &vdv));
    }
    if (a.nq == 0) {  // no queries: nothing depends on k and v
      VK_TRY(apart(name, {vdk.p, vdv.p}, {}));
      VK_TRY_CUDA(zero_heads(vdk, bf16, a.batch, a.heads, a.nk, a.dim, s), name);
      return vk_cuda_status(zero_heads(vdv, bf16, a.batch, a.heads, a.nk, a.dim, s), name);
    }
    VK_TRY(floats_ok(name, "delta", delta));
    if (a.nk == 0) {  // no keys: out is zero whatever q is
      VK_TRY_CUDA(zero_heads(vdq, bf16, a.batch, a.heads, a.nq, a.dim, s), name);
      return vk_cuda_status(fill_f32(delta, B * H * a.nq, 0.0f, s), name);
    }
    VK_TRY(heads_view(name, "q", q, shape->dtype, B, H, a.nq, D, 16, &vq));
    VK_TRY(heads_view(name, "k", k, shape->dtype, B, H, a.nk, D, 16, &vk_));
    VK_TRY(heads_view(name, "v", v, shape->dtype, B, H, a.nk, D, 16, &vv));
    VK_TRY(heads_view(name, "out", out, shape->dtype, B, H, a.nq, D, 16, &vo));
    VK_TRY(heads_view(name, "d_out", d_out, shape->dtype, B, H, a.nq, D, 16, &vg));
    VK_TRY(floats_ok(name, "lse", lse));
    VK_TRY(apart(name, {vdq.p, vdk.p, vdv.p, delta}, {vq.p, vk_.p, vv.p, vo.p, vg.p, lse}));
    // The tensor cores take P and dS rounded to bf16.  That makes a gradient's
    // error 1.41 to 1.45 times the one of its own rounding as a root mean square,
    // of 2 keys (865 queries, 96 heads) as of 865, of 2 queries as of many.  In a
    // call of a few scores the largest of the few errors is up to 2.6 times the
    // largest rounding.  Such calls are launch latency either way (1 x 61 x 61 14
    // us on the device there, 23 here, 22 from the caller), so they keep f32
    // throughout.  One query alone
    // takes no tiles either: 12 heads of 3457 keys 44 us from the caller (78 on
    // the tensor cores), 1536 heads 813 (1177).
    const bool few = static_cast<int64_t>(a.batch) * a.heads * a.nq <= 8192 / a.nk;
    // There lse / scale is an operand: below this scale it could pass f32's range.
    const bool tiny_scale = a.scale < 0x1p-100f;
    if (bf16 && a.dim == 64 && a.nq > 1 && !few && !tiny_scale)
      return vk_cuda_status(attention_backward_tc(a, vq, vk_, vv, vo, lse, vg, vdq, vdk, vdv, delta, ctx->d_err, s), name);
    return vk_cuda_status(attention_backward_simt(a, bf16, vq, vk_, vv, vo, lse, vg, vdq, vdk, vdv, delta, s), name);
  });
}

// ------------------------------------------------------------------ rotary positions
extern "C" int vk_rope_axes(vk_ctx* ctx, const vk_rope_axes_shape* shape, const vk_heads* q, const vk_heads* k,
                            const int64_t* positions, const vk_heads* q_out, const vk_heads* k_out) {
  static const char* name = "vk_rope_axes";
  return guarded(ctx, name, [&]() -> int {
    if (shape == nullptr) return vk_fail(VK_ERR_INVALID_ARGUMENT, "%s: shape is NULL", name);
    const vk_rope_axes_shape& r = *shape;
    VK_TRY(dtype_ok(name, r.dtype));
    VK_TRY(vk_dims_fit(name, {r.batch, r.heads, r.tokens, r.head_dim}));
    if (r.head_dim == 0 || r.head_dim > 2 * ROPE_MAX_PAIRS)
      return vk_fail(VK_UNSUPPORTED_SHAPE, "%s: head_dim %zu (supported: 1 to %d)", name, r.head_dim, 2 * ROPE_MAX_PAIRS);
    if (r.axes == 0 || r.axes > VK_ROPE_MAX_AXES)
      return vk_fail(VK_ERR_INVALID_ARGUMENT, "%s: %zu axes (supported: 1 to %d)", name, r.axes, VK_ROPE_MAX_AXES);
    if (!(std::isfinite(r.freq) && r.freq > 0.0f))
      return vk_fail(VK_ERR_INVALID_ARGUMENT, "%s: freq must be finite and positive", name);
    if ((k == nullptr) != (k_out == nullptr)) return vk_fail(VK_ERR_INVALID_ARGUMENT, "%s: k without k_out", name);
    RopePairs p{};
    size_t at = 0;
    int vec = r.dtype == VK_DTYPE_F32 ? 4 : 8;
    for (size_t a = 0; a < r.axes; ++a) {
      const size_t w = r.sections[a];
      if (w % 2 != 0 || w > r.head_dim - at)
        return vk_fail(VK_ERR_INVALID_ARGUMENT, "%s: section %zu of %zu elements (even, together at most head_dim)", name, a, w);
      for (size_t i = 0; i < w / 2; ++i) {
        p.lo[p.pairs] = static_cast<int16_t>(at + i);
        p.hi[p.pairs] = static_cast<int16_t>(at + w / 2 + i);
        p.axis[p.pairs] = static_cast<int8_t>(a);
        p.inv[p.pairs] = std::pow(static_cast<double>(r.freq), -2.0 * static_cast<double>(i) / static_cast<double>(w));
        ++p.pairs;
      }
      while (w / 2 % vec != 0) vec /= 2;
      at += w;
    }
    p.rotated = static_cast<int>(at);
    if (r.batch == 0 || r.heads == 0 || r.tokens == 0) return VK_OK;
    // the pieces of all tokens are counted in an int, and so are the heads' splits in a grid dimension
    if (r.heads > 65535 * 4 || r.batch > static_cast<size_t>(INT_MAX) / (2 * ROPE_MAX_PAIRS) / r.tokens)
      return vk_fail(VK_UNSUPPORTED_SHAPE, "%s: too many heads or tokens", name);
    if (positions == nullptr || reinterpret_cast<uintptr_t>(positions) % 8 != 0)
      return vk_fail(VK_ERR_INVALID_ARGUMENT, "%s: positions are NULL or not aligned", name);
    const size_t size = r.dtype == VK_DTYPE_F32 ? 4 : 2;
    HeadsView vq, vqo, vk_, vko;
    VK_TRY(heads_view(name, "q", q, r.dtype, r.batch, r.heads, r.tokens, r.head_dim, size, &vq));
    VK_TRY(heads_view(name, "q_out", q_out, r.dtype, r.batch, r.heads, r.tokens, r.head_dim, size, &vqo));
    if (k != nullptr) {
      VK_TRY(heads_view(name, "k", k, r.dtype, r.batch, r.heads, r.tokens, r.head_dim, size, &vk_));
      VK_TRY(heads_view(name, "k_out", k_out, r.dtype, r.batch, r.heads, r.tokens, r.head_dim, size, &vko));
      VK_TRY(apart(name, {vqo.p, vko.p}, {}));
      if (vqo.p == vk_.p || vko.p == vq.p) return vk_fail(VK_ERR_INVALID_ARGUMENT, "%s: an output is the other's input", name);
    }
    for (int i = 0; i < (k != nullptr ? 2 : 1); ++i) {
      const HeadsView &in = i ? vk_ : vq, &out = i ? vko : vqo;
      if (in.p == out.p && (in.sb != out.sb || in.sh != out.sh || in.st != out.st))
        return vk_fail(VK_ERR_INVALID_ARGUMENT, "%s: in place with other strides", name);
    }
    // the widest piece that every address is aligned to
    for (const HeadsView* v : {&vq, &vqo, &vk_, &vko}) {
      const uint64_t bits = reinterpret_cast<uintptr_t>(v->p) | static_cast<uint64_t>(v->sb | v->sh | v->st) * size;
      while (bits % (vec * size) != 0) vec /= 2;
    }
    p.vec = vec;
    return vk_cuda_status(rope_axes(r.dtype == VK_DTYPE_BF16, static_cast<int>(r.batch), static_cast<int>(r.heads),
                                    static_cast<int>(r.tokens), static_cast<int>(r.head_dim), static_cast<int>(r.axes), p,
                                    r.inverse != 0, positions, r.positions_per_batch != 0, vq, vqo, vk_, vko, ctx->stream),
                          name);
  });
}

// ------------------------------------------------------------------ residual step between two norms
namespace {
int norm_shape(const char* name, const vk_residual_norm_shape* s, ResidualNorm* r) {
  if (s == nullptr) return vk_fail(VK_ERR_INVALID_ARGUMENT, "%s: shape is NULL", name);
  VK_TRY(dtype_ok(name, s->stream_dtype));
  VK_TRY(dtype_ok(name, s->branch_dtype));
  if (s->stream_dtype == VK_DTYPE_BF16 && s->branch_dtype == VK_DTYPE_F32)
    return vk_fail(VK_UNSUPPORTED_SHAPE, "%s: an f32 branch on a bf16 stream", name);
  VK_TRY(vk_dims_fit(name, {s->groups, s->rows_per_group, s->cols}));
  if (s->cols > static_cast<size_t>(RESIDUAL_NORM_MAX_COLS))
    return vk_fail(VK_UNSUPPORTED_SHAPE, "%s: %zu columns (at most %d)", name, s->cols, RESIDUAL_NORM_MAX_COLS);
  // rows, and the 32-column pieces of d_gate, are counted in an int
  if (s->groups != 0 && (s->rows_per_group > static_cast<size_t>(INT_MAX) / s->groups ||
                         s->cols / 32 + 1 > static_cast<size_t>(INT_MAX) / (s->groups + 8)))
    return vk_fail(VK_UNSUPPORTED_SHAPE, "%s: more than 2^31 rows", name);
  if (!(std::isfinite(s->eps) && s->eps >= 0.0f))
    return vk_fail(VK_ERR_INVALID_ARGUMENT, "%s: eps must be finite and not negative", name);
  if (s->groups != 0 && s->rows_per_group != 0 && s->cols != 0) {
    VK_TRY(floats_ok(name, "gamma", s->gamma));
    VK_TRY(floats_ok(name, "beta", s->beta));
  }
  if ((s->post_gamma == nullptr) != (s->post_beta == nullptr))
    return vk_fail(VK_ERR_INVALID_ARGUMENT, "%s: post_gamma and post_beta go together", name);
  for (const float* p : {s->scale, s->gate, s->post_gamma, s->post_beta})
    if (reinterpret_cast<uintptr_t>(p) % 4 != 0) return vk_fail(VK_ERR_INVALID_ARGUMENT, "%s: a vector is not aligned", name);
  r->groups = static_cast<int>(s->groups);
  r->rows_per_group = static_cast<int>(s->rows_per_group);
  r->cols = static_cast<int>(s->cols);
  r->eps = s->eps;
  r->gamma = s->gamma;
  r->beta = s->beta;
  r->scale = s->scale;
  r->gate = s->gate;
  r->post_gamma = s->post_gamma;
  r->post_beta = s->post_beta;
  return VK_OK;
}

int matrix_ok(const char* name, const char* what, const void* p, int dtype) {
  if (p == nullptr) return vk_fail(VK_ERR_INVALID_ARGUMENT, "%s: %s is NULL", name, what);
  if (reinterpret_cast<uintptr_t>(p) % (dtype == VK_DTYPE_F32 ? 4 : 2) != 0)
    return vk_fail(VK_ERR_INVALID_ARGUMENT, "%s: %s is not aligned", name, what);
  return VK_OK;
}
}  // namespace

extern "C" int vk_residual_norm_forward(vk_ctx* ctx, const vk_residual_norm_shape* shape, const void* x,
                                        const void* branch, void* h, void* y, float* stats, float* post_stats) {
  static const char* name = "vk_residual_norm_forward";
  return guarded(ctx, name, [&]() -> int {
    ResidualNorm r;
    VK_TRY(norm_shape(name, shape, &r));
    if (r.groups == 0 || r.rows_per_group == 0 || r.cols == 0) return VK_OK;
    VK_TRY(matrix_ok(name, "x", x, shape->stream_dtype));
    VK_TRY(matrix_ok(name, "h", h, shape->stream_dtype));
    VK_TRY(matrix_ok(name, "branch", branch, shape->branch_dtype));
    VK_TRY(matrix_ok(name, "y", y, shape->branch_dtype));
    VK_TRY(floats_ok(name, "stats", stats, 8));
    if (r.post_gamma != nullptr) VK_TRY(floats_ok(name, "post_stats", post_stats, 8));
    VK_TRY(apart(name, {h, y, stats, r.post_gamma != nullptr ? post_stats : nullptr},
                 {branch, r.gamma, r.beta, r.scale, r.gate, r.post_gamma, r.post_beta}));
    if (y == x) return vk_fail(VK_ERR_INVALID_ARGUMENT, "%s: y is x", name);
    return vk_cuda_status(residual_norm_forward(r, shape->stream_dtype == VK_DTYPE_BF16, shape->branch_dtype == VK_DTYPE_BF16,
                                                x, branch, h, y, stats, post_stats, ctx->stream),
                          name);
  });
}

extern "C" int vk_residual_norm_workspace(vk_ctx* ctx, const vk_residual_norm_shape* shape, size_t* bytes) {
  static const char* name = "vk_residual_norm_workspace";
  return guarded(ctx, name, [&]() -> int {
    if (bytes == nullptr) return vk_fail(VK_ERR_INVALID_ARGUMENT, "%s: bytes is NULL", name);
    ResidualNorm r;
    VK_TRY(norm_shape(name, shape, &r));
    *bytes = r.groups == 0 || r.rows_per_group == 0 || r.cols == 0 ? 0 : residual_norm_workspace(r);
    return VK_OK;
  });
}

extern "C" int vk_residual_norm_backward(vk_ctx* ctx, const vk_residual_norm_shape* shape, const void* d_h,
                                         const void* d_y, const void* h, const void* branch, const float* stats,
                                         const float* post_stats, const vk_residual_norm_grads* grads, void* workspace,
                                         size_t workspace_bytes) {
  static const char* name = "vk_residual_norm_backward";
  return guarded(ctx, name, [&]() -> int {
    ResidualNorm r;
    VK_TRY(norm_shape(name, shape, &r));
    if (grads == nullptr) return vk_fail(VK_ERR_INVALID_ARGUMENT, "%s: grads is NULL", name);
    if (r.cols == 0) return VK_OK;
    VK_TRY(floats_ok(name, "d_gamma", grads->d_gamma));
    VK_TRY(floats_ok(name, "d_beta", grads->d_beta));
    if ((grads->d_scale == nullptr) != (r.scale == nullptr) || (grads->d_gate == nullptr) != (r.gate == nullptr) ||
        (grads->d_post_gamma == nullptr) != (r.post_gamma == nullptr) ||
        (grads->d_post_beta == nullptr) != (r.post_gamma == nullptr))
      return vk_fail(VK_ERR_INVALID_ARGUMENT, "%s: d_scale, d_gate, d_post_gamma and d_post_beta are given exactly where their vectors are", name);
    for (const float* p : {grads->d_scale, grads->d_gate, grads->d_post_gamma, grads->d_post_beta})
      if (reinterpret_cast<uintptr_t>(p) % 4 != 0) return vk_fail(VK_ERR_INVALID_ARGUMENT, "%s: a gradient is not aligned", name);
    cudaStream_t s = ctx->stream;
    if (r.groups == 0 || r.rows_per_group == 0) {  // no rows: sums of nothing
      for (float* p : {grads->d_gamma, grads->d_beta, grads->d_scale, grads->d_post_gamma, grads->d_post_beta})
        if (p != nullptr) VK_TRY_CUDA(fill_f32(p, r.cols, 0.0f, s), name);
      if (grads->d_gate != nullptr) VK_TRY_CUDA(fill_f32(grads->d_gate, static_cast<size_t>(r.groups) * r.cols, 0.0f, s), name);
      return VK_OK;
    }
    VK_TRY(matrix_ok(name, "d_y", d_y, shape->branch_dtype));
    VK_TRY(matrix_ok(name, "h", h, shape->stream_dtype));
    VK_TRY(matrix_ok(name, "branch", branch, shape->branch_dtype));
    VK_TRY(matrix_ok(name, "d_x", grads->d_x, shape->stream_dtype));
    VK_TRY(matrix_ok(name, "d_branch", grads->d_branch, shape->branch_dtype));
    if (reinterpret_cast<uintptr_t>(d_h) % (shape->stream_dtype == VK_DTYPE_F32 ? 4 : 2) != 0)
      return vk_fail(VK_ERR_INVALID_ARGUMENT, "%s: d_h is not aligned", name);
    VK_TRY(floats_ok(name, "stats", stats, 8));
    if (r.post_gamma != nullptr) VK_TRY(floats_ok(name, "post_stats", post_stats, 8));
    const size_t need = residual_norm_workspace(r);
    if (workspace == nullptr || reinterpret_cast<uintptr_t>(workspace) % 16 != 0 || workspace_bytes < need)
      return vk_fail(VK_ERR_INVALID_ARGUMENT, "%s: workspace of %zu bytes, 16-byte aligned, is needed (got %zu)", name, need, workspace_bytes);
    VK_TRY(apart(name, {grads->d_x, grads->d_branch, workspace, grads->d_gamma, grads->d_beta, grads->d_scale, grads->d_gate,
                        grads->d_post_gamma, grads->d_post_beta},
                 {h, branch, stats, r.gamma, r.scale, r.gate, r.post_gamma, r.post_beta}));
    if (grads->d_x == d_y || grads->d_branch == d_h)
      return vk_fail(VK_ERR_INVALID_ARGUMENT, "%s: d_x may be d_h and d_branch d_y, not the other way round", name);
    ResidualNormGrads g;
    g.d_x = grads->d_x;
    g.d_branch = grads->d_branch;
    g.d_gamma = grads->d_gamma;
    g.d_beta = grads->d_beta;
    g.d_scale = grads->d_scale;
    g.d_gate = grads->d_gate;
    g.d_post_gamma = grads->d_post_gamma;
    g.d_post_beta = grads->d_post_beta;
    return vk_cuda_status(residual_norm_backward(r, shape->stream_dtype == VK_DTYPE_BF16, shape->branch_dtype == VK_DTYPE_BF16,
                                                 d_h, d_y, h, branch, stats, post_stats, g, static_cast<float*>(workspace), s),
                          name);
  });
}
