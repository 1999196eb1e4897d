// C ABI of the attention operators (s14_attn_*.hip): argument checks and
// launches.  Everything that a kernel takes from the host as an address or a
// size is checked here; what it reads from device memory it checks itself.
#include <hip/hip_runtime_api.h>

#include <cmath>
#include <type_traits>

#include "s14_attn.hpp"
#include "s14_attn_share.h"
#include "s14_internal.hpp"

using s14::fail;

namespace {

// Launches go to the context's device, whatever device is current.
class OnDevice {
 public:
  explicit OnDevice(int device) {
    err_ = hipGetDevice(&before_);
    if (err_ == hipSuccess && before_ != device) {
      err_ = hipSetDevice(device);
      moved_ = err_ == hipSuccess;
    }
  }
  ~OnDevice() {
    if (moved_) (void)hipSetDevice(before_);
  }
  hipError_t error() const { return err_; }

 private:
  int before_ = 0;
  bool moved_ = false;
  hipError_t err_;
};

int hip_fail(hipError_t e, const char *what) { return fail(S14_ERR_HIP, "%s: %s", what, hipGetErrorString(e)); }

int check_ctx(const s14_ctx *ctx) { return ctx ? S14_OK : fail(S14_ERR_INVALID, "NULL context"); }

int require(const s14_buffer &b, uint64_t bytes, uint32_t align, const char *label) {
  if (!b.ptr) return fail(S14_ERR_INVALID, "%s buffer is NULL", label);
  if (b.bytes < bytes)
    return fail(S14_ERR_CAPACITY, "%s buffer is %llu B, requires at least %llu B", label, (unsigned long long)b.bytes,
                (unsigned long long)bytes);
  if (reinterpret_cast<uintptr_t>(b.ptr) % align) return fail(S14_ERR_SHAPE, "%s buffer is not %u-byte aligned", label, align);
  return S14_OK;
}

bool head_dim(uint32_t dim) { return dim == 64 || dim == 128 || dim == 256 || dim == 512; }

constexpr uint64_t kMaxStride = 1ull << 24;  // elements; a key tile's rows stay inside 32-bit offsets
constexpr uint32_t kMaxTokens = 1u << 30, kMaxGrid = 65535;
constexpr uint32_t kMaxNorm = 65536;  // values of a norm's row: 64 a thread of a workgroup
constexpr uint64_t kMaxBlocks = 1u << 24;  // of 256 threads: a launch has below 2^32 in one dimension

// A packed [tokens][heads][dim] operand: dtype, strides, and that its last
// value lies inside the buffer.
int check_rows(const s14_rows *r, uint32_t tokens, uint32_t dim, bool bf16_only, const char *label) {
  if (!r) return fail(S14_ERR_INVALID, "NULL %s rows", label);
  if (r->dtype != S14_X_F32 && r->dtype != S14_X_BF16) return fail(S14_ERR_INVALID, "unknown %s dtype %d", label, r->dtype);
  if (bf16_only && r->dtype != S14_X_BF16) return fail(S14_ERR_INVALID, "%s must be bf16", label);
  if (!r->heads || r->heads > kMaxGrid) return fail(S14_ERR_SHAPE, "%s has %u heads, 1 to %u are allowed", label, r->heads, kMaxGrid);
  if (r->token_stride % 8 || r->head_stride % 8 || r->token_stride > kMaxStride || r->head_stride > kMaxStride)
    return fail(S14_ERR_SHAPE, "%s strides %llu and %u must be multiples of 8 elements, at most %llu", label,
                (unsigned long long)r->token_stride, r->head_stride, (unsigned long long)kMaxStride);
  // rows of a token, and tokens, do not overlap
  if ((r->heads > 1 && r->head_stride < dim) || (tokens > 1 && r->token_stride < dim))
    return fail(S14_ERR_SHAPE, "%s strides %llu and %u are below the head size %u", label,
                (unsigned long long)r->token_stride, r->head_stride, dim);
  if (!tokens) return S14_OK;
  const uint64_t last = uint64_t(tokens - 1) * r->token_stride + uint64_t(r->heads - 1) * r->head_stride + dim;
  return require(r->buf, last * (r->dtype == S14_X_F32 ? 4 : 2), 16, label);
}

int check_out(const s14_rows *out, const s14_rows *like, uint32_t tokens, uint32_t dim, const char *label) {
  if (int rc = check_rows(out, tokens, dim, false, label)) return rc;
  if (out->heads != like->heads) return fail(S14_ERR_SHAPE, "%s has %u heads, its input %u", label, out->heads, like->heads);
  // no two rows of an output share a place
  if (out->heads > 1 && tokens > 1) {
    const uint64_t all = uint64_t(out->heads - 1) * out->head_stride + dim;
    const uint64_t over = uint64_t(tokens - 1) * out->token_stride + dim;
    if (out->token_stride < all && out->head_stride < over)
      return fail(S14_ERR_SHAPE, "%s strides %llu and %u let rows overlap", label, (unsigned long long)out->token_stride,
                  out->head_stride);
  }
  return S14_OK;
}

s14::RowBytes bytes_of(const s14_rows *r, uint32_t dim) {
  const uint64_t size = r->dtype == S14_X_F32 ? 4 : 2;
  return {reinterpret_cast<uintptr_t>(r->buf.ptr), r->token_stride * size, r->head_stride * size, dim * size, r->heads};
}

// An output's rows lie apart from another operand's, but for each its own
// input's place: workgroups write while others read.
int check_apart(const s14_rows *out, const s14_rows *other, uint32_t tokens, uint32_t dim, bool own, const char *label) {
  if (!tokens || !s14::rows_share(bytes_of(out, dim), bytes_of(other, dim), tokens, own)) return S14_OK;
  return fail(S14_ERR_INVALID, "%s shares memory with %s rows", label, own ? "other" : "another operand's");
}

int check_rope(const s14_rope *r, uint32_t dim, s14::RopeArgs *out) {
  *out = s14::RopeArgs{};
  if (!r || !r->table.ptr) return S14_OK;
  if (r->layout != S14_ROPE_HALF && r->layout != S14_ROPE_INTERLEAVED)
    return fail(S14_ERR_INVALID, "unknown rotation layout %d", r->layout);
  if (!r->rot || r->rot % 8 || r->start % 8 || uint64_t(r->start) + r->rot > dim)
    return fail(S14_ERR_SHAPE, "rotation of %u dimensions at %u: multiples of 8 inside the head's %u are required", r->rot,
                r->start, dim);
  if (!r->positions) return fail(S14_ERR_SHAPE, "rotation table has no positions");
  if (int rc = require(r->table, uint64_t(r->positions) * r->rot * 4, 16, "rotation table")) return rc;
  *out = {static_cast<const float *>(r->table.ptr), r->positions, r->rot, r->start, r->layout == S14_ROPE_INTERLEAVED};
  return S14_OK;
}

int check_weight(const s14_buffer &w, uint32_t dim, float eps, const char *label) {
  if (!w.ptr) return S14_OK;
  if (!(eps >= 0.0f) || std::isinf(eps)) return fail(S14_ERR_INVALID, "norm eps %g must be finite and >= 0", double(eps));
  return require(w, 4ull * dim, 16, label);
}

// Shape of either cache.
template <class Cache>
int check_pages(const Cache *c) {
  if (!c) return fail(S14_ERR_INVALID, "NULL cache");
  if (!head_dim(c->dim)) return fail(S14_ERR_SHAPE, "cache head size %u is not 64, 128, 256 or 512", c->dim);
  if (c->page_tokens != 16 && c->page_tokens != 32 && c->page_tokens != 64 && c->page_tokens != 128)
    return fail(S14_ERR_SHAPE, "cache pages of %u tokens: 16, 32, 64 or 128 are required", c->page_tokens);
  if (!c->pages || !c->heads || c->heads > kMaxGrid / 2 || c->pages > uint32_t(INT32_MAX))
    return fail(S14_ERR_SHAPE, "cache of %u pages and %u heads", c->pages, c->heads);
  return S14_OK;
}

// Its buffers: bytes of codes and of scales of a (page, head), and the scales' alignment.
template <class Cache>
int check_codes(const Cache *c, uint64_t codes, uint64_t k_scales, uint64_t v_scales, uint32_t align, s14::CacheArgs *out) {
  const uint64_t places = uint64_t(c->pages) * c->heads;
  if (int rc = require(c->k, places * codes, 16, "k codes")) return rc;
  if (int rc = require(c->v, places * codes, 16, "v codes")) return rc;
  if (int rc = require(c->k_scale, places * k_scales, align, "k scales")) return rc;
  if (int rc = require(c->v_scale, places * v_scales, align, "v scales")) return rc;
  *out = {static_cast<uint8_t *>(c->k.ptr), static_cast<uint8_t *>(c->v.ptr), static_cast<uint8_t *>(c->k_scale.ptr),
          static_cast<uint8_t *>(c->v_scale.ptr), c->pages, c->heads, c->page_tokens, c->dim};
  return S14_OK;
}

int check_cache(const s14_kv_cache *c, s14::CacheArgs *out) {
  if (int rc = check_pages(c)) return rc;
  return check_codes(c, uint64_t(c->page_tokens) * c->dim, 1, 1, 1, out);
}

int check_cache(const s14_kv4_cache *c, s14::CacheArgs *out) {
  if (int rc = check_pages(c)) return rc;
  const uint64_t slots = c->page_tokens;
  return check_codes(c, slots * (c->dim / 2), slots * (c->dim / 32), slots * (c->dim < 128 ? 1 : c->dim / 128), 16, out);
}

int check_counts(uint32_t tokens, uint32_t seqs, uint32_t most) {
  if (tokens > kMaxTokens || seqs > kMaxGrid)
    return fail(S14_ERR_SHAPE, "%u tokens in %u sequences: at most %u and %u", tokens, seqs, kMaxTokens, kMaxGrid);
  if (most > tokens) return fail(S14_ERR_INVALID, "a longest count of %u among %u tokens", most, tokens);
  return S14_OK;
}

int check_table(const s14_buffer &cu, const s14_buffer &len, const s14_buffer &table, uint32_t seqs, uint32_t width,
                const char *len_label) {
  if (int rc = require(cu, 4 * (uint64_t(seqs) + 1), 4, "cu")) return rc;
  if (int rc = require(len, 4ull * seqs, 4, len_label)) return rc;
  if (!width || width > (1u << 24)) return fail(S14_ERR_SHAPE, "page table of %u pages a sequence", width);
  return require(table, 4ull * seqs * width, 4, "page table");
}

s14::AttnRows rows_of(const s14_rows *r) {
  return {r->buf.ptr, r->dtype == S14_X_BF16, r->heads, r->token_stride, r->head_stride};
}
s14::AttnOut out_of(const s14_rows *r) { return {r->buf.ptr, r->dtype == S14_X_BF16, r->token_stride, r->head_stride}; }

int check_scale(float scale) {
  return std::isfinite(scale) && scale > 0.0f
             ? S14_OK
             : fail(S14_ERR_INVALID, "attention scale %g must be finite and above 0", double(scale));
}

// Group size of q heads over key heads, and the optional lse.
int check_heads(const s14_rows *q, uint32_t kv, uint32_t tokens, const s14_buffer &lse) {
  if (q->heads % kv) return fail(S14_ERR_SHAPE, "%u query heads do not divide over %u key heads", q->heads, kv);
  if (!lse.ptr) return S14_OK;
  return require(lse, 4ull * tokens * q->heads, 4, "lse");
}

}  // namespace

extern "C" int s14_rope_table(s14_ctx *ctx, void *stream, uint32_t positions, uint32_t rot, double theta,
                              const s14_rope_scaling *scaling, s14_buffer table) {
  if (int rc = check_ctx(ctx)) return rc;
  if (!positions || positions > kMaxTokens || !rot || rot % 8 || rot > 512)
    return fail(S14_ERR_SHAPE, "rotation table of %u positions and %u dimensions", positions, rot);
  if (!(theta > 1.0) || std::isinf(theta)) return fail(S14_ERR_INVALID, "rotation base %g must be above 1", theta);
  s14::RopeTableArgs a{positions, rot, theta, 1.0, 0.0, 0.0, 0.0, 1.0, static_cast<float *>(table.ptr)};
  if (scaling) {
    const s14_rope_scaling &s = *scaling;
    if (!(s.factor > 0.0) || std::isinf(s.factor) || !std::isfinite(s.amplitude) || !(s.original >= 0.0) ||
        std::isinf(s.original))
      return fail(S14_ERR_INVALID, "rotation scaling factor %g, original %g, amplitude %g", s.factor, s.original, s.amplitude);
    if (s.original > 0.0 && !(s.beta_slow > 0.0 && s.beta_fast >= s.beta_slow && std::isfinite(s.beta_fast)))
      return fail(S14_ERR_INVALID, "rotation scaling turns %g to %g", s.beta_slow, s.beta_fast);
    a.factor = s.factor, a.original = s.original, a.fast = s.beta_fast, a.slow = s.beta_slow, a.amplitude = s.amplitude;
  }
  if (int rc = require(table, uint64_t(positions) * rot * 4, 16, "rotation table")) return rc;
  if ((uint64_t(positions) * (rot / 2) + 255) / 256 >= kMaxBlocks)
    return fail(S14_ERR_SHAPE, "rotation table of %u positions and %u dimensions exceeds one launch", positions, rot);
  const OnDevice on(s14::ctx_device(ctx));
  if (on.error() != hipSuccess) return hip_fail(on.error(), "hipSetDevice");
  const hipError_t e = s14::launch_rope_table(reinterpret_cast<hipStream_t>(stream), a);
  return e == hipSuccess ? S14_OK : hip_fail(e, "rope_table launch");
}

extern "C" int s14_qk_norm_rope(s14_ctx *ctx, void *stream, uint32_t tokens, uint32_t dim, const s14_rows *q,
                                const s14_rows *k, const s14_rows *q_out, const s14_rows *k_out, s14_buffer q_weight,
                                s14_buffer k_weight, float eps, const s14_rope *rope, s14_buffer positions) {
  if (int rc = check_ctx(ctx)) return rc;
  if (!head_dim(dim)) return fail(S14_ERR_SHAPE, "head size %u is not 64, 128, 256 or 512", dim);
  if (tokens > kMaxTokens) return fail(S14_ERR_SHAPE, "%u tokens, at most %u", tokens, kMaxTokens);
  if (!k) return fail(S14_ERR_INVALID, "NULL k rows");
  if (int rc = check_rows(q, tokens, dim, false, "q")) return rc;
  if (int rc = check_out(q_out, q, tokens, dim, "q output")) return rc;
  if (k->heads) {
    if (int rc = check_rows(k, tokens, dim, false, "k")) return rc;
    if (int rc = check_out(k_out, k, tokens, dim, "k output")) return rc;
  }
  if (int rc = check_weight(q_weight, dim, eps, "q norm weight")) return rc;
  if (int rc = check_weight(k_weight, dim, eps, "k norm weight")) return rc;
  s14::NormRopeArgs a{};
  if (int rc = check_rope(rope, dim, &a.rope)) return rc;
  if (a.rope.table && tokens)
    if (int rc = require(positions, 4ull * tokens, 4, "positions")) return rc;
  const uint64_t per = 2048 / dim;  // rows of a workgroup
  if ((uint64_t(tokens) * q->heads + per - 1) / per + (uint64_t(tokens) * k->heads + per - 1) / per >= kMaxBlocks)
    return fail(S14_ERR_SHAPE, "%u tokens of %u heads exceed one launch", tokens, q->heads + k->heads);
  if (!tokens) return S14_OK;
  if (int rc = check_apart(q_out, q, tokens, dim, true, "q output")) return rc;
  if (k->heads) {
    if (int rc = check_apart(k_out, k, tokens, dim, true, "k output")) return rc;
    if (int rc = check_apart(q_out, k, tokens, dim, false, "q output")) return rc;
    if (int rc = check_apart(k_out, q, tokens, dim, false, "k output")) return rc;
    if (s14::rows_share(bytes_of(q_out, dim), bytes_of(k_out, dim), tokens, false))
      return fail(S14_ERR_INVALID, "the q and k outputs share memory");
  }
  a.tokens = tokens, a.dim = dim;
  a.in[0] = rows_of(q), a.out[0] = out_of(q_out);
  if (k->heads) a.in[1] = rows_of(k), a.out[1] = out_of(k_out);
  a.weight[0] = static_cast<const float *>(q_weight.ptr), a.weight[1] = static_cast<const float *>(k_weight.ptr);
  a.eps = eps;
  a.positions = static_cast<const int32_t *>(positions.ptr);
  a.status = s14::ctx_status(ctx);
  const OnDevice on(s14::ctx_device(ctx));
  if (on.error() != hipSuccess) return hip_fail(on.error(), "hipSetDevice");
  const hipError_t e = s14::launch_norm_rope(reinterpret_cast<hipStream_t>(stream), a);
  return e == hipSuccess ? S14_OK : hip_fail(e, "qk_norm_rope launch");
}

// A row operand of add_rms_norm: one head of k values.
static int check_flat(const s14_rows *r, uint32_t rows, uint32_t k, const char *label) {
  if (r && r->heads != 1) return fail(S14_ERR_SHAPE, "%s has %u heads, one is required", label, r->heads);
  return check_rows(r, rows, k, false, label);
}

extern "C" int s14_add_rms_norm(s14_ctx *ctx, void *stream, uint32_t rows, uint32_t k, const s14_rows *x,
                                const s14_rows *residual, const s14_rows *residual_out, const s14_rows *y,
                                s14_buffer weight, float eps, uint32_t group, s14_buffer q, s14_buffer scales) {
  if (int rc = check_ctx(ctx)) return rc;
  if (rows > kMaxTokens) return fail(S14_ERR_SHAPE, "%u rows, at most %u", rows, kMaxTokens);
  if (!k || k % 8 || k > kMaxNorm) return fail(S14_ERR_SHAPE, "rows of %u values: multiples of 8, at most %u, are required", k, kMaxNorm);
  if (group && group != 32 && group != 64 && group != 128) return fail(S14_ERR_SHAPE, "scale group %u is not 32, 64 or 128", group);
  if (group && k % group) return fail(S14_ERR_SHAPE, "rows of %u values are not whole groups of %u", k, group);
  if (!y && !group) return fail(S14_ERR_INVALID, "neither y nor codes are asked for");
  if (int rc = check_flat(x, rows, k, "x")) return rc;
  const s14_rows *outs[2] = {residual_out, y};
  const char *const labels[2] = {"residual output", "y"};
  if (residual)
    if (int rc = check_flat(residual, rows, k, "residual")) return rc;
  for (int i = 0; i < 2; ++i)
    if (outs[i])
      if (int rc = check_flat(outs[i], rows, k, labels[i])) return rc;
  if (!weight.ptr) return fail(S14_ERR_INVALID, "norm weight buffer is NULL");
  if (int rc = check_weight(weight, k, eps, "norm weight")) return rc;
  if (!rows) return S14_OK;
  // a thread for eight values at most
  if (uint64_t(rows) * ((k / 8 + 63) / 64 * 64) >= kMaxBlocks * 256)
    return fail(S14_ERR_SHAPE, "%u rows of %u values exceed one launch", rows, k);
  const uint64_t values = uint64_t(rows) * k, n_scales = group ? values / group : 0;
  if (group) {
    if (int rc = require(q, values, 8, "codes")) return rc;
    if (int rc = require(scales, n_scales, 1, "scales")) return rc;
  }
  // rows may be written in their input's place; nothing else is shared
  const auto touch = [&](const s14_rows *r, const void *p, uint64_t bytes) {
    return r && s14::rows_touch(bytes_of(r, k), reinterpret_cast<uintptr_t>(p), bytes, rows);
  };
  for (int i = 0; i < 2; ++i) {
    if (!outs[i]) continue;
    if (int rc = check_apart(outs[i], x, rows, k, true, labels[i])) return rc;
    if (residual)
      if (int rc = check_apart(outs[i], residual, rows, k, true, labels[i])) return rc;
    if (touch(outs[i], weight.ptr, 4ull * k)) return fail(S14_ERR_INVALID, "%s shares memory with the norm weight", labels[i]);
  }
  if (residual_out && y && s14::rows_share(bytes_of(residual_out, k), bytes_of(y, k), rows, false))
    return fail(S14_ERR_INVALID, "the residual output and y share memory");
  if (group) {
    const s14::RowBytes codes{reinterpret_cast<uintptr_t>(q.ptr), 0, 0, values, 1};
    const s14::RowBytes byte_scales{reinterpret_cast<uintptr_t>(scales.ptr), 0, 0, n_scales, 1};
    bool shared = s14::rows_touch(codes, byte_scales.at, n_scales, 1);
    for (const s14::RowBytes &made : {codes, byte_scales}) {
      shared |= s14::rows_touch(made, reinterpret_cast<uintptr_t>(weight.ptr), 4ull * k, 1);
      for (const s14_rows *r : {x, residual, residual_out, y})
        shared |= touch(r, reinterpret_cast<const void *>(made.at), made.row);
    }
    if (shared) return fail(S14_ERR_INVALID, "codes or scales share memory with another operand");
  }
  s14::AddNormArgs a{};
  a.rows = rows, a.k = k;
  a.x = rows_of(x);
  if (residual) a.residual = rows_of(residual);
  if (residual_out) a.residual_out = out_of(residual_out);
  if (y) a.y = out_of(y);
  a.weight = static_cast<const float *>(weight.ptr), a.eps = eps, a.group = group;
  a.q = static_cast<uint8_t *>(q.ptr), a.scales = static_cast<uint8_t *>(scales.ptr);
  const OnDevice on(s14::ctx_device(ctx));
  if (on.error() != hipSuccess) return hip_fail(on.error(), "hipSetDevice");
  const hipError_t e = s14::launch_add_norm(reinterpret_cast<hipStream_t>(stream), a);
  return e == hipSuccess ? S14_OK : hip_fail(e, "add_rms_norm launch");
}

// Both caches' appends and attentions: the same checks, and a kernel file each.
template <class Cache>
static int append_to(hipError_t (*launch)(hipStream_t, const s14::AppendArgs &), s14_ctx *ctx, void *stream,
                     const Cache *cache, uint32_t tokens, uint32_t seqs, uint32_t max_new, const s14_rows *k,
                     const s14_rows *v, s14_buffer page_table, uint32_t table_width, s14_buffer cu, s14_buffer past,
                     s14_buffer k_weight, float eps, const s14_rope *rope) {
  if (int rc = check_ctx(ctx)) return rc;
  s14::AppendArgs a{};
  if (int rc = check_cache(cache, &a.cache)) return rc;
  if (int rc = check_counts(tokens, seqs, max_new)) return rc;
  if (int rc = check_rows(k, tokens, cache->dim, false, "k")) return rc;
  if (int rc = check_rows(v, tokens, cache->dim, false, "v")) return rc;
  if (k->heads != cache->heads || v->heads != cache->heads)
    return fail(S14_ERR_SHAPE, "k and v have %u and %u heads, the cache %u", k->heads, v->heads, cache->heads);
  if (int rc = check_weight(k_weight, cache->dim, eps, "k norm weight")) return rc;
  if (int rc = check_rope(rope, cache->dim, &a.rope)) return rc;
  if (!tokens || !seqs || !max_new) return S14_OK;
  if (int rc = check_table(cu, past, page_table, seqs, table_width, "past")) return rc;
  // 16 slots of D / 8 lanes a workgroup, and for each sequence two blocks that it may share
  if (std::is_same_v<Cache, s14_kv4_cache> && (uint64_t(tokens) / 16 + 2ull * seqs + 1) * 2 * cache->dim >= kMaxBlocks * 256)
    return fail(S14_ERR_SHAPE, "%u tokens of %u sequences exceed one launch", tokens, seqs);
  a.tokens = tokens, a.seqs = seqs, a.max_new = max_new, a.table_width = table_width;
  a.in[0] = rows_of(k), a.in[1] = rows_of(v);
  a.k_weight = static_cast<const float *>(k_weight.ptr), a.eps = eps;
  a.page_table = static_cast<const int32_t *>(page_table.ptr);
  a.cu = static_cast<const int32_t *>(cu.ptr), a.past = static_cast<const int32_t *>(past.ptr);
  a.status = s14::ctx_status(ctx);
  const OnDevice on(s14::ctx_device(ctx));
  if (on.error() != hipSuccess) return hip_fail(on.error(), "hipSetDevice");
  const hipError_t e = launch(reinterpret_cast<hipStream_t>(stream), a);
  return e == hipSuccess ? S14_OK : hip_fail(e, "append launch");
}

extern "C" int s14_kv_append(s14_ctx *ctx, void *stream, const s14_kv_cache *cache, uint32_t tokens, uint32_t seqs,
                             uint32_t max_new, const s14_rows *k, const s14_rows *v, s14_buffer page_table,
                             uint32_t table_width, s14_buffer cu, s14_buffer past, s14_buffer k_weight, float eps,
                             const s14_rope *rope) {
  return append_to(s14::launch_kv_append, ctx, stream, cache, tokens, seqs, max_new, k, v, page_table, table_width, cu,
                   past, k_weight, eps, rope);
}

extern "C" int s14_kv4_append(s14_ctx *ctx, void *stream, const s14_kv4_cache *cache, uint32_t tokens, uint32_t seqs,
                              uint32_t max_new, const s14_rows *k, const s14_rows *v, s14_buffer page_table,
                              uint32_t table_width, s14_buffer cu, s14_buffer past, s14_buffer k_weight, float eps,
                              const s14_rope *rope) {
  return append_to(s14::launch_kv4_append, ctx, stream, cache, tokens, seqs, max_new, k, v, page_table, table_width, cu,
                   past, k_weight, eps, rope);
}

template <class Cache>
static int attend_over(hipError_t (*launch)(hipStream_t, const s14::PagedArgs &, const s14::PagedPlan &, float *),
                       s14_ctx *ctx, void *stream, const s14_rows *q, const Cache *cache, uint32_t tokens, uint32_t seqs,
                       uint32_t max_new, uint32_t max_len, s14_buffer page_table, uint32_t table_width, s14_buffer cu,
                       s14_buffer lens, const s14_rows *out, s14_buffer lse, float scale, uint32_t window) {
  if (int rc = check_ctx(ctx)) return rc;
  s14::PagedArgs a{};
  if (int rc = check_cache(cache, &a.cache)) return rc;
  if (int rc = check_counts(tokens, seqs, max_new)) return rc;
  if (int rc = check_rows(q, tokens, cache->dim, true, "q")) return rc;
  if (int rc = check_out(out, q, tokens, cache->dim, "out")) return rc;
  if (int rc = check_heads(q, cache->heads, tokens, lse)) return rc;
  if (int rc = check_scale(scale)) return rc;
  if (max_len > uint32_t(INT32_MAX)) return fail(S14_ERR_SHAPE, "longest sequence of %u tokens", max_len);
  if (!tokens || !seqs || !max_new) return S14_OK;
  if (int rc = check_table(cu, lens, page_table, seqs, table_width, "lens")) return rc;
  // positions, and those of the steps ahead, stay in 31 bits
  if (uint64_t(table_width) * cache->page_tokens > (1ull << 31) - (1u << 16))
    return fail(S14_ERR_SHAPE, "page table of %u pages of %u tokens: past %llu positions", table_width, cache->page_tokens,
                (1ull << 31) - (1u << 16));
  a.tokens = tokens, a.seqs = seqs, a.heads = q->heads, a.max_new = max_new, a.max_len = max_len;
  a.table_width = table_width;
  a.q = static_cast<const uint16_t *>(q->buf.ptr), a.q_token = q->token_stride, a.q_head = q->head_stride;
  a.page_table = static_cast<const int32_t *>(page_table.ptr);
  a.cu = static_cast<const int32_t *>(cu.ptr), a.len = static_cast<const int32_t *>(lens.ptr);
  a.out = out_of(out), a.lse = static_cast<float *>(lse.ptr);
  a.scale = scale, a.window = window;
  const s14::PagedPlan p = s14::paged_plan(
      {seqs, a.heads, cache->heads, cache->dim, max_new, max_len, window, table_width * cache->page_tokens, std::is_same_v<Cache, s14_kv4_cache>});
  if (p.blocks >= kMaxBlocks || uint64_t(max_new) * q->heads >= (1ull << 31))
    return fail(S14_ERR_SHAPE, "%u new tokens of %u sequences exceed one launch", max_new, seqs);
  if (int rc = check_apart(out, q, tokens, cache->dim, true, "out")) return rc;
  a.status = s14::ctx_status(ctx), a.count = s14::ctx_attn_counters(ctx);
  const OnDevice on(s14::ctx_device(ctx));
  if (on.error() != hipSuccess) return hip_fail(on.error(), "hipSetDevice");
  float *part = nullptr;
  if (p.chunks > 1)
    if (int rc = s14::ctx_attn_workspace(ctx, s14::kPagedPartFloats * sizeof(float), &part)) return rc;
  const hipError_t e = launch(reinterpret_cast<hipStream_t>(stream), a, p, part);
  return e == hipSuccess ? S14_OK : hip_fail(e, "paged_attention launch");
}

extern "C" int s14_paged_attention(s14_ctx *ctx, void *stream, const s14_rows *q, const s14_kv_cache *cache,
                                   uint32_t tokens, uint32_t seqs, uint32_t max_new, uint32_t max_len,
                                   s14_buffer page_table, uint32_t table_width, s14_buffer cu, s14_buffer lens,
                                   const s14_rows *out, s14_buffer lse, float scale, uint32_t window) {
  return attend_over(s14::launch_paged_attention, ctx, stream, q, cache, tokens, seqs, max_new, max_len, page_table,
                     table_width, cu, lens, out, lse, scale, window);
}

extern "C" int s14_paged4_attention(s14_ctx *ctx, void *stream, const s14_rows *q, const s14_kv4_cache *cache,
                                    uint32_t tokens, uint32_t seqs, uint32_t max_new, uint32_t max_len,
                                    s14_buffer page_table, uint32_t table_width, s14_buffer cu, s14_buffer lens,
                                    const s14_rows *out, s14_buffer lse, float scale, uint32_t window) {
  return attend_over(s14::launch_paged4_attention, ctx, stream, q, cache, tokens, seqs, max_new, max_len, page_table,
                     table_width, cu, lens, out, lse, scale, window);
}

extern "C" int s14_prompt_attention(s14_ctx *ctx, void *stream, uint32_t dim, const s14_rows *q, const s14_rows *k,
                                    const s14_rows *v, uint32_t tokens, uint32_t seqs, s14_buffer cu,
                                    const s14_rows *out, s14_buffer lse, float scale, uint32_t window) {
  if (int rc = check_ctx(ctx)) return rc;
  if (dim != 64 && dim != 128 && dim != 256) return fail(S14_ERR_SHAPE, "prompt head size %u is not 64, 128 or 256", dim);
  if (int rc = check_counts(tokens, seqs, 0)) return rc;
  if (int rc = check_rows(q, tokens, dim, true, "q")) return rc;
  if (int rc = check_rows(k, tokens, dim, true, "k")) return rc;
  if (int rc = check_rows(v, tokens, dim, true, "v")) return rc;
  if (k->heads != v->heads) return fail(S14_ERR_SHAPE, "k has %u heads, v %u", k->heads, v->heads);
  if (int rc = check_out(out, q, tokens, dim, "out")) return rc;
  if (int rc = check_heads(q, k->heads, tokens, lse)) return rc;
  if (int rc = check_scale(scale)) return rc;
  if (!tokens || !seqs) return S14_OK;
  if (int rc = require(cu, 4 * (uint64_t(seqs) + 1), 4, "cu")) return rc;
  if ((uint64_t(tokens) * (q->heads / k->heads) / 128 + seqs + 1) * k->heads >= kMaxBlocks)
    return fail(S14_ERR_SHAPE, "%u tokens of %u heads exceed one launch", tokens, q->heads);
  if (int rc = check_apart(out, q, tokens, dim, true, "out")) return rc;
  if (int rc = check_apart(out, k, tokens, dim, false, "out")) return rc;
  if (int rc = check_apart(out, v, tokens, dim, false, "out")) return rc;
  s14::PromptArgs a{};
  a.tokens = tokens, a.seqs = seqs, a.heads = q->heads, a.kv_heads = k->heads, a.dim = dim;
  a.q = static_cast<const uint16_t *>(q->buf.ptr), a.q_token = q->token_stride, a.q_head = q->head_stride;
  a.k = static_cast<const uint16_t *>(k->buf.ptr), a.k_token = k->token_stride, a.k_head = k->head_stride;
  a.v = static_cast<const uint16_t *>(v->buf.ptr), a.v_token = v->token_stride, a.v_head = v->head_stride;
  // a single row's stride is never taken, but bounds the rows behind it
  if (tokens == 1) a.k_token = a.v_token = dim;
  a.cu = static_cast<const int32_t *>(cu.ptr);
  a.out = out_of(out), a.lse = static_cast<float *>(lse.ptr);
  a.scale = scale, a.window = window;
  const OnDevice on(s14::ctx_device(ctx));
  if (on.error() != hipSuccess) return hip_fail(on.error(), "hipSetDevice");
  const hipError_t e = s14::launch_prompt_attention(reinterpret_cast<hipStream_t>(stream), a);
  return e == hipSuccess ? S14_OK : hip_fail(e, "prompt_attention launch");
}
