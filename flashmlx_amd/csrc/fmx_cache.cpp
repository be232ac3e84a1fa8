// fmx_cache.cpp -- C-ABI of the KV cache's long-context operators
// (include/fmx_cache.h): argument checks, workspaces and launches.
#include <hip/hip_runtime.h>

#include <cmath>

#include "../../include/fmx_cache.h"
#include "fmx_cache_kernels.hpp"
#include "fmx_checks.hpp"

using namespace fmx;

namespace {

constexpr int64_t kMaxRows = FMX_CACHE_MAX_ROWS;
constexpr int64_t kMaxHeads = 65535;
// of the positions that attention reads: 64 rows' byte offsets within 32 bits
constexpr int64_t kMaxKeyStride = int64_t{1} << 24;
// (sequence, kv head) pairs of an eviction: a workgroup of 1024 threads each
constexpr int64_t kMaxEvictRows = int64_t{1} << 22;

int check_counts(int64_t batch, int64_t seq_len, int64_t n_heads, int64_t n_kv_heads) {
  if (batch < 0 || seq_len < 0 || batch > kMaxRows || seq_len > kMaxRows || batch * seq_len > kMaxRows)
    return fail(FMX_ERR_SHAPE, "batch %lld, seq_len %lld (at most 2^24 rows)", (long long)batch, (long long)seq_len);
  if (n_heads < 1 || n_heads > kMaxHeads || n_kv_heads < 1 || n_kv_heads > kMaxHeads)
    return fail(FMX_ERR_SHAPE, "n_heads %lld, n_kv_heads %lld", (long long)n_heads, (long long)n_kv_heads);
  return FMX_OK;
}

int check_key_stride(const fmx_heads& k, const fmx_heads& v, const char* name) {
  if (k.token_stride > kMaxKeyStride || v.token_stride > kMaxKeyStride)
    return fail(FMX_ERR_UNSUPPORTED, "%s: token strides above 2^24", name);
  return FMX_OK;
}

// Keys and values, both written: rows that overlap where the layouts are alike
// (they may well lie among each other, as in [slot, position, 2, head, element]).
int check_apart(const fmx_heads& k, const fmx_heads& v, const char* name, int64_t hd, int es) {
  const uintptr_t a = reinterpret_cast<uintptr_t>(k.data), b = reinterpret_cast<uintptr_t>(v.data);
  const bool alike =
      k.batch_stride == v.batch_stride && k.token_stride == v.token_stride && k.head_stride == v.head_stride;
  if (a == b || (alike && (a < b ? b - a : a - b) < static_cast<uintptr_t>(hd * es)))
    return fail(FMX_ERR_ARG, "%s: keys and values overlap", name);
  return FMX_OK;
}

int check_angles(const fmx_rope_angles* a, int64_t head_dim) {
  if (!a) return fail(FMX_ERR_ARG, "angles is NULL");
  if (head_dim < 2 || head_dim > kRopeMaxHd || a->dims < 2 || a->dims % 2 || a->dims > head_dim)
    return fail(FMX_ERR_SHAPE, "dims %lld of head_dim %lld (even, head_dim at most %d)", (long long)a->dims,
                (long long)head_dim, kRopeMaxHd);
  if (!std::isfinite(a->factor)) return fail(FMX_ERR_ARG, "factor not finite");
  return FMX_OK;
}

int check_pool(int64_t n_slots, int64_t max_seq) {
  if (n_slots < 0 || n_slots > kMaxRows || max_seq < 0 || max_seq > kMaxRows)
    return fail(FMX_ERR_SHAPE, "n_slots %lld, max_seq %lld (at most 2^24)", (long long)n_slots, (long long)max_seq);
  return FMX_OK;
}

int check_attention(const fmx_attention_shape* s, int64_t prefix_len, int64_t max_seq) {
  if (!s) return fail(FMX_ERR_ARG, "shape is NULL");
  if (s->dtype != FMX_BF16 && s->dtype != FMX_F16)
    return fail(FMX_ERR_DTYPE, "dtype %d (bf16 or float16)", s->dtype);
  FMX_RC(check_counts(s->batch, s->seq_len, s->n_heads, s->n_kv_heads));
  if (s->n_heads % s->n_kv_heads) return fail(FMX_ERR_SHAPE, "n_heads not a multiple of n_kv_heads");
  if (s->head_dim < 1) return fail(FMX_ERR_SHAPE, "head_dim %lld", (long long)s->head_dim);
  if (s->head_dim % 8 || s->head_dim > kCacheMaxHd)
    return fail(FMX_ERR_UNSUPPORTED, "head_dim %lld (a multiple of 8, at most %d)", (long long)s->head_dim,
                kCacheMaxHd);
  if (!std::isfinite(s->scale) || !(s->scale > 0.0f)) return fail(FMX_ERR_ARG, "scale must be finite and positive");
  if (prefix_len < 0 || prefix_len > kMaxRows || max_seq < 0 || max_seq > kMaxRows)
    return fail(FMX_ERR_SHAPE, "prefix_len %lld, max_seq %lld (at most 2^24)", (long long)prefix_len,
                (long long)max_seq);
  if (s->batch * s->seq_len * s->n_heads > (int64_t{1} << 30))
    return fail(FMX_ERR_UNSUPPORTED, "more than 2^30 query rows");
  if (s->batch * max_seq > (int64_t{1} << 36)) return fail(FMX_ERR_UNSUPPORTED, "more than 2^36 own positions");
  return FMX_OK;
}

// what is written against what is read after parts of it may have been
// written, and against each other
int check_out(const CacheAttnArgs& a) {
  const auto at = [&](const HeadsView& v, int64_t nb, int64_t nt, int64_t nh) {
    const fmx_heads h{v.p, v.bs, v.ts, v.hs};
    return v.p ? span(&h, nb, nt, nh, a.hd, 2) : Span{0, 0};
  };
  const Span out = at(a.out, a.B, a.L, a.nh);
  const Span lse = flat(a.lse, static_cast<int64_t>(a.B) * a.L * a.nh);
  const Span w = flat(a.w_out, a.n_slots * a.nkv * a.S);
  for (const Span& i : {at(a.q, a.B, a.L, a.nh), at(a.kp, 1, a.P, a.nkv), at(a.vp, 1, a.P, a.nkv),
                        at(a.kc, a.n_slots, a.S, a.nkv), at(a.vc, a.n_slots, a.S, a.nkv)}) {
    if (overlap(out, i)) return fail(FMX_ERR_ARG, "out overlaps q, the prefix or a cache");
    if (overlap(lse, i)) return fail(FMX_ERR_ARG, "lse overlaps q, the prefix or a cache");
    if (overlap(w, i)) return fail(FMX_ERR_ARG, "weights_out overlaps q or a cache");
  }
  if (overlap(out, lse) || overlap(out, w)) return fail(FMX_ERR_ARG, "out overlaps lse or weights_out");
  if (overlap(out, flat(a.w_in, a.n_slots * a.nkv * a.S))) return fail(FMX_ERR_ARG, "out overlaps weights_in");
  const fmx_heads o{a.out.p, a.out.bs, a.out.ts, a.out.hs};
  return check_written(o, "out", a.B, a.L, a.nh);
}

// Rows of q turned in place, and new keys or values that are among them (they
// may well lie between them, as in a fused row of q, k and v).
int check_not_among(const fmx_heads& k, const fmx_heads& q, const char* name, int64_t n_heads, int64_t hd, int es) {
  if (k.batch_stride != q.batch_stride || k.token_stride != q.token_stride) return FMX_OK;
  const int64_t d = (static_cast<const uint8_t*>(k.data) - static_cast<const uint8_t*>(q.data)) / es;
  const int64_t hs = q.head_stride;
  const bool among = (d < 0 ? -d : d) < hd || (hs > 0 && d > 0 && d % hs == 0 && d / hs < n_heads);
  return among ? fail(FMX_ERR_ARG, "q_out overlaps %s", name) : FMX_OK;
}

int check_launches(const CacheAttnArgs& a) {
  return cache_attn_fits(a) ? FMX_OK : fail(FMX_ERR_UNSUPPORTED, "more work than launches of fewer than 2^32 threads");
}

CacheAttnArgs attention_args(const fmx_attention_shape* s, int64_t prefix_len, int64_t max_seq, bool weights) {
  CacheAttnArgs a{};
  a.B = static_cast<int>(s->batch);
  a.L = static_cast<int>(s->seq_len);
  a.nh = static_cast<int>(s->n_heads);
  a.nkv = static_cast<int>(s->n_kv_heads);
  a.rep = a.nh / a.nkv;
  a.hd = static_cast<int>(s->head_dim);
  a.scale = s->scale;
  a.P = prefix_len;
  a.S = max_seq;
  static float mark;  // any address: the size queries only ask whether weights are wanted
  a.w_out = weights ? &mark : nullptr;
  return a;
}

}  // namespace

extern "C" {

int fmx_rope_frequencies(const fmx_rope_config* cfg, double* freqs, double* attention_factor) {
  if (!cfg || !freqs || !attention_factor) return fail(FMX_ERR_ARG, "NULL argument");
  const int64_t n = cfg->dims / 2;
  if (cfg->dims < 2 || cfg->dims % 2 || cfg->dims > kRopeMaxHd)
    return fail(FMX_ERR_SHAPE, "dims %lld (even, 2 .. %d)", (long long)cfg->dims, kRopeMaxHd);
  const int kind = cfg->scaling;
  const double s = cfg->factor;
  if (kind < FMX_ROPE_NONE || kind > FMX_ROPE_YARN) return fail(FMX_ERR_ARG, "scaling %d", kind);
  if (!std::isfinite(cfg->base) || !(cfg->base > 1.0)) return fail(FMX_ERR_ARG, "base must be above 1");
  if (kind != FMX_ROPE_NONE && (!std::isfinite(s) || !(s >= 1.0))) return fail(FMX_ERR_ARG, "factor below 1");
  if (kind == FMX_ROPE_NTK && cfg->dims < 4) return fail(FMX_ERR_SHAPE, "NTK scaling takes dims of at least 4");
  if (!std::isfinite(cfg->attention_factor) || cfg->attention_factor < 0.0)
    return fail(FMX_ERR_ARG, "attention_factor negative or not finite");
  const double two_pi = 6.283185307179586476925;
  const double dims = static_cast<double>(cfg->dims);
  double lo = 0.0, hi = 0.0;
  if (kind == FMX_ROPE_PARTS || kind == FMX_ROPE_YARN) {
    if (cfg->original_max < 1) return fail(FMX_ERR_ARG, "original_max below 1");
    if (!std::isfinite(cfg->high) || !(cfg->low > 0.0) || !(cfg->high > cfg->low))
      return fail(FMX_ERR_ARG, "turns: 0 < low < high");
    // the pair that turns r times over original_max:
    // original_max base^(-2 i / dims) = 2 pi r
    const double len = static_cast<double>(cfg->original_max), lb = std::log(cfg->base);
    lo = std::fmax(std::floor(dims * std::log(len / (cfg->high * two_pi)) / (2.0 * lb)), 0.0);
    hi = std::fmin(std::ceil(dims * std::log(len / (cfg->low * two_pi)) / (2.0 * lb)), dims - 1.0);
  }
  for (int64_t i = 0; i < n; ++i) {
    const double e = -2.0 * static_cast<double>(i) / dims;
    const double g = std::pow(cfg->base, e);
    double f = g;
    if (kind == FMX_ROPE_LINEAR) {
      f = g / s;
    } else if (kind == FMX_ROPE_NTK) {
      f = std::pow(cfg->base * std::pow(s, dims / (dims - 2.0)), e);
    } else if (kind == FMX_ROPE_PARTS || kind == FMX_ROPE_YARN) {
      double t;
      if (kind == FMX_ROPE_PARTS) {
        const double turns = static_cast<double>(cfg->original_max) * g / two_pi;
        t = (turns - cfg->low) / (cfg->high - cfg->low);
      } else {
        t = 1.0 - (static_cast<double>(i) - lo) / std::fmax(hi - lo, 1e-3);
      }
      t = std::fmin(std::fmax(t, 0.0), 1.0);
      f = t * g + (1.0 - t) * g / s;
    }
    freqs[i] = f;
  }
  *attention_factor = cfg->attention_factor > 0.0 ? cfg->attention_factor
                      : kind == FMX_ROPE_YARN     ? 0.1 * std::log(s) + 1.0
                                                  : 1.0;
  return ok();
}

int fmx_rope(const fmx_rope_angles* angles, int dtype, int64_t batch, int64_t seq_len, int64_t n_heads,
             int64_t head_dim, const fmx_heads* x, const int32_t* positions, int inverse, const fmx_heads* out,
             fmx_stream stream) {
  if (dtype != FMX_BF16 && dtype != FMX_F16 && dtype != FMX_F32)
    return fail(FMX_ERR_DTYPE, "dtype %d (bf16, float16 or float32)", dtype);
  FMX_RC(check_counts(batch, seq_len, n_heads, 1));
  FMX_RC(check_angles(angles, head_dim));
  if (batch * seq_len == 0) return ok();
  if (!angles->freqs || !positions) return fail(FMX_ERR_ARG, "NULL freqs or positions");
  const int es = elem_size(dtype);
  fmx_heads x_v, out_v;
  FMX_RC(check_view(x, "x", batch, seq_len, n_heads, es, 1, &x_v));
  FMX_RC(check_view(out, "out", batch, seq_len, n_heads, es, 1, &out_v));
  FMX_RC(check_written(out_v, "out", batch, seq_len, n_heads));
  x = &x_v;
  out = &out_v;
  if (!same(x, out) && overlap(span(x, batch, seq_len, n_heads, head_dim, es),
                               span(out, batch, seq_len, n_heads, head_dim, es)))
    return fail(FMX_ERR_ARG, "out overlaps x with other strides or another start");
  RotateArgs a{};
  a.freqs = angles->freqs;
  a.dims = static_cast<int>(angles->dims);
  a.factor = static_cast<float>(angles->factor);
  a.interleaved = angles->interleaved != 0;
  a.inverse = inverse != 0;
  a.B = static_cast<int>(batch);
  a.L = static_cast<int>(seq_len);
  a.nh = static_cast<int>(n_heads);
  a.hd = static_cast<int>(head_dim);
  a.q = view(x);
  a.q_out = view(out);
  a.pos = positions;
  FMX_HIP(launch_rotate(a, es, dtype == FMX_F16, static_cast<hipStream_t>(stream)));
  return ok();
}

int fmx_rope_append(const fmx_rope_angles* angles, int dtype, int64_t batch, int64_t seq_len, int64_t n_heads,
                    int64_t n_kv_heads, int64_t head_dim, const fmx_heads* q, const fmx_heads* k, const fmx_heads* v,
                    const int32_t* positions, const int32_t* offsets, const int32_t* slots, int64_t n_slots,
                    int64_t max_seq, const fmx_heads* q_out, const fmx_heads* k_cache, const fmx_heads* v_cache,
                    fmx_stream stream) {
  if (dtype != FMX_BF16 && dtype != FMX_F16 && dtype != FMX_F32)
    return fail(FMX_ERR_DTYPE, "dtype %d (bf16, float16 or float32)", dtype);
  FMX_RC(check_counts(batch, seq_len, n_heads, n_kv_heads));
  FMX_RC(check_angles(angles, head_dim));
  FMX_RC(check_pool(n_slots, max_seq));
  if (!slots && n_slots < batch) return fail(FMX_ERR_SHAPE, "n_slots below batch without slots");
  if (batch * seq_len == 0) return ok();
  if (!angles->freqs || !positions || !offsets) return fail(FMX_ERR_ARG, "NULL freqs, positions or offsets");
  const int es = elem_size(dtype);
  fmx_heads q_v, k_v, v_v, qo_v, kc_v, vc_v;
  FMX_RC(check_view(q, "q", batch, seq_len, n_heads, es, 1, &q_v));
  FMX_RC(check_view(k, "k", batch, seq_len, n_kv_heads, es, 1, &k_v));
  FMX_RC(check_view(v, "v", batch, seq_len, n_kv_heads, es, 1, &v_v));
  FMX_RC(check_view(q_out, "q_out", batch, seq_len, n_heads, es, 1, &qo_v));
  FMX_RC(check_view(k_cache, "k_cache", n_slots, max_seq, n_kv_heads, es, 1, &kc_v));
  FMX_RC(check_view(v_cache, "v_cache", n_slots, max_seq, n_kv_heads, es, 1, &vc_v));
  FMX_RC(check_written(qo_v, "q_out", batch, seq_len, n_heads));
  FMX_RC(check_written(kc_v, "k_cache", n_slots, max_seq, n_kv_heads));
  FMX_RC(check_written(vc_v, "v_cache", n_slots, max_seq, n_kv_heads));
  FMX_RC(check_apart(kc_v, vc_v, "caches", head_dim, es));
  q = &q_v;
  k = &k_v;
  v = &v_v;
  q_out = &qo_v;
  k_cache = &kc_v;
  v_cache = &vc_v;
  const Span ins[3] = {span(q, batch, seq_len, n_heads, head_dim, es),
                       span(k, batch, seq_len, n_kv_heads, head_dim, es),
                       span(v, batch, seq_len, n_kv_heads, head_dim, es)};
  const Span outs[3] = {span(q_out, batch, seq_len, n_heads, head_dim, es),
                        span(k_cache, n_slots, max_seq, n_kv_heads, head_dim, es),
                        span(v_cache, n_slots, max_seq, n_kv_heads, head_dim, es)};
  for (int c = 1; c < 3; ++c)  // caches against the inputs and q_out
    for (const Span& i : {ins[0], ins[1], ins[2], outs[0]})
      if (overlap(outs[c], i)) return fail(FMX_ERR_ARG, "a cache overlaps q, k, v or q_out");
  if (same(q, q_out)) {
    FMX_RC(check_not_among(*k, *q, "k", n_heads, head_dim, es));
    FMX_RC(check_not_among(*v, *q, "v", n_heads, head_dim, es));
  } else {
    for (const Span& i : ins)
      if (overlap(outs[0], i)) return fail(FMX_ERR_ARG, "q_out overlaps q, k or v and is not q itself");
  }
  RotateArgs a{};
  a.freqs = angles->freqs;
  a.dims = static_cast<int>(angles->dims);
  a.factor = static_cast<float>(angles->factor);
  a.interleaved = angles->interleaved != 0;
  a.B = static_cast<int>(batch);
  a.L = static_cast<int>(seq_len);
  a.nh = static_cast<int>(n_heads);
  a.nkv = static_cast<int>(n_kv_heads);
  a.hd = static_cast<int>(head_dim);
  a.q = view(q);
  a.k = view(k);
  a.v = view(v);
  a.q_out = view(q_out);
  a.kc = view(k_cache);
  a.vc = view(v_cache);
  a.pos = positions;
  a.offs = offsets;
  a.slots = slots;
  a.n_slots = n_slots;
  a.max_seq = max_seq;
  FMX_HIP(launch_rotate(a, es, dtype == FMX_F16, static_cast<hipStream_t>(stream)));
  return ok();
}

size_t fmx_attention_shared_prefix_workspace_size(const fmx_attention_shape* shape, int64_t prefix_len,
                                                  int64_t max_seq) {
  if (check_attention(shape, prefix_len, max_seq) != FMX_OK || shape->batch * shape->seq_len == 0) return 0;
  return cache_attn_workspace(attention_args(shape, prefix_len, max_seq, false));
}

int fmx_attention_shared_prefix(const fmx_attention_shape* shape, const fmx_heads* q, const fmx_heads* k_prefix,
                                const fmx_heads* v_prefix, int64_t prefix_len, const fmx_heads* k_cache,
                                const fmx_heads* v_cache, int64_t n_slots, int64_t max_seq, const int32_t* offsets,
                                const int32_t* slots, const fmx_heads* out, float* lse, void* workspace,
                                size_t workspace_bytes, fmx_stream stream_) {
  FMX_RC(check_attention(shape, prefix_len, max_seq));
  FMX_RC(check_pool(n_slots, max_seq));
  CacheAttnArgs a = attention_args(shape, prefix_len, max_seq, false);
  if (max_seq > 0 && !slots && n_slots < shape->batch)
    return fail(FMX_ERR_SHAPE, "n_slots below batch without slots");
  if (shape->batch * shape->seq_len == 0) return ok();
  fmx_heads q_v, out_v, kp_v, vp_v, kc_v, vc_v;
  FMX_RC(check_view(q, "q", shape->batch, shape->seq_len, shape->n_heads, 16, 8, &q_v));
  FMX_RC(check_view(out, "out", shape->batch, shape->seq_len, shape->n_heads, 16, 8, &out_v));
  if (prefix_len > 0) {
    FMX_RC(check_view(k_prefix, "k_prefix", 1, prefix_len, shape->n_kv_heads, 16, 8, &kp_v));
    FMX_RC(check_view(v_prefix, "v_prefix", 1, prefix_len, shape->n_kv_heads, 16, 8, &vp_v));
    FMX_RC(check_key_stride(kp_v, vp_v, "prefix"));
    a.kp = view(&kp_v);
    a.vp = view(&vp_v);
  }
  if (max_seq > 0) {
    FMX_RC(check_view(k_cache, "k_cache", n_slots, max_seq, shape->n_kv_heads, 16, 8, &kc_v));
    FMX_RC(check_view(v_cache, "v_cache", n_slots, max_seq, shape->n_kv_heads, 16, 8, &vc_v));
    FMX_RC(check_key_stride(kc_v, vc_v, "caches"));
    a.kc = view(&kc_v);
    a.vc = view(&vc_v);
    a.offs = offsets;
    a.slots = slots;
    a.n_slots = n_slots;
    if (!offsets) return fail(FMX_ERR_ARG, "offsets is NULL");
  }
  if (!aligned(lse, 4)) return fail(FMX_ERR_ARG, "lse not 4-byte aligned");
  hipStream_t stream = static_cast<hipStream_t>(stream_);
  a.q = view(&q_v);
  a.out = view(&out_v);
  a.lse = lse;
  FMX_RC(check_out(a));
  FMX_RC(check_launches(a));
  Workspace ws;
  FMX_RC(ws.bind(workspace, workspace_bytes, cache_attn_workspace(a), stream));
  FMX_HIP(launch_cache_attn(a, shape->dtype == FMX_F16, ws.p, stream));
  return ok();
}

size_t fmx_attention_scored_workspace_size(const fmx_attention_shape* shape, int64_t max_seq) {
  if (check_attention(shape, 0, max_seq) != FMX_OK || shape->batch * shape->seq_len == 0) return 0;
  return cache_attn_workspace(attention_args(shape, 0, max_seq, true));
}

int fmx_attention_scored(const fmx_attention_shape* shape, const fmx_heads* q, const fmx_heads* k_cache,
                         const fmx_heads* v_cache, int64_t n_slots, int64_t max_seq, const int32_t* offsets,
                         const int32_t* slots, const float* weights_in, float* weights_out, const fmx_heads* out,
                         void* workspace, size_t workspace_bytes, fmx_stream stream_) {
  FMX_RC(check_attention(shape, 0, max_seq));
  FMX_RC(check_pool(n_slots, max_seq));
  if (max_seq < 1) return fail(FMX_ERR_SHAPE, "max_seq below 1");
  CacheAttnArgs a = attention_args(shape, 0, max_seq, true);
  if (!slots && n_slots < shape->batch) return fail(FMX_ERR_SHAPE, "n_slots below batch without slots");
  if (shape->batch == 0) return ok();
  if (!aligned(weights_in, 4) || !aligned(weights_out, 4)) return fail(FMX_ERR_ARG, "weights not 4-byte aligned");
  if (weights_in && weights_in != weights_out) {
    const uintptr_t n = static_cast<uintptr_t>(n_slots) * static_cast<uintptr_t>(a.nkv) *
                        static_cast<uintptr_t>(max_seq) * 4;
    const uintptr_t i = reinterpret_cast<uintptr_t>(weights_in), o = reinterpret_cast<uintptr_t>(weights_out);
    if (overlap({i, i + n}, {o, o + n})) return fail(FMX_ERR_ARG, "weights_out overlaps weights_in in part");
  }
  hipStream_t stream = static_cast<hipStream_t>(stream_);
  a.slots = slots;
  a.n_slots = n_slots;
  a.w_in = weights_in;
  a.w_out = weights_out;
  if (shape->seq_len == 0) {  // no weights to add
    if (!weights_out || weights_out == weights_in) return ok();
    FMX_RC(check_launches(a));
    FMX_HIP(launch_cache_weights_kept(a, stream));
    return ok();
  }
  fmx_heads q_v, out_v, kc_v, vc_v;
  FMX_RC(check_view(q, "q", shape->batch, shape->seq_len, shape->n_heads, 16, 8, &q_v));
  FMX_RC(check_view(out, "out", shape->batch, shape->seq_len, shape->n_heads, 16, 8, &out_v));
  FMX_RC(check_view(k_cache, "k_cache", n_slots, max_seq, shape->n_kv_heads, 16, 8, &kc_v));
  FMX_RC(check_view(v_cache, "v_cache", n_slots, max_seq, shape->n_kv_heads, 16, 8, &vc_v));
  FMX_RC(check_key_stride(kc_v, vc_v, "caches"));
  if (!offsets || !weights_out) return fail(FMX_ERR_ARG, "NULL offsets or weights_out");
  a.q = view(&q_v);
  a.out = view(&out_v);
  a.kc = view(&kc_v);
  a.vc = view(&vc_v);
  a.offs = offsets;
  FMX_RC(check_out(a));
  FMX_RC(check_launches(a));
  Workspace ws;
  FMX_RC(ws.bind(workspace, workspace_bytes, cache_attn_workspace(a), stream));
  FMX_HIP(launch_cache_attn(a, shape->dtype == FMX_F16, ws.p, stream));
  return ok();
}

size_t fmx_cache_evict_workspace_size(int64_t batch, int64_t n_kv_heads, int64_t budget) {
  if (batch < 0 || batch > kMaxRows || n_kv_heads < 1 || n_kv_heads > kMaxHeads || budget < 1 || budget > kMaxRows ||
      batch * n_kv_heads >= kMaxEvictRows)
    return 0;
  return static_cast<size_t>(align_up(batch * n_kv_heads * budget * 4, 256));
}

int fmx_cache_evict(int dtype, int64_t batch, int64_t n_kv_heads, int64_t head_dim, const fmx_heads* k_cache,
                    const fmx_heads* v_cache, float* weights, int64_t n_slots, int64_t max_seq,
                    const int32_t* lengths, const int32_t* slots, int64_t budget, int64_t sinks, int64_t recent,
                    const fmx_heads* k_out, const fmx_heads* v_out, float* weights_out, int64_t out_max_seq,
                    int32_t* lengths_out, int32_t* kept, void* workspace, size_t workspace_bytes,
                    fmx_stream stream_) {
  if (dtype != FMX_BF16 && dtype != FMX_F16) return fail(FMX_ERR_DTYPE, "dtype %d (bf16 or float16)", dtype);
  FMX_RC(check_counts(batch, 1, 1, n_kv_heads));
  if (batch * n_kv_heads >= kMaxEvictRows) return fail(FMX_ERR_UNSUPPORTED, "2^22 rows of weights or more");
  FMX_RC(check_pool(n_slots, max_seq));
  if (max_seq < 1) return fail(FMX_ERR_SHAPE, "max_seq below 1");
  if (head_dim < 1 || head_dim > kRopeMaxHd)
    return fail(FMX_ERR_SHAPE, "head_dim %lld (1 .. %d)", (long long)head_dim, kRopeMaxHd);
  if (budget < 1 || budget > kMaxRows || sinks < 0 || recent < 0 || sinks > budget || recent > budget - sinks)
    return fail(FMX_ERR_SHAPE, "budget %lld, sinks %lld, recent %lld", (long long)budget, (long long)sinks,
                (long long)recent);
  const bool in_place = !k_out && !v_out && !weights_out;
  if (!in_place && (!k_out || !v_out || !weights_out))
    return fail(FMX_ERR_ARG, "k_out, v_out and weights_out: all of them or none");
  if (!in_place && (out_max_seq > kMaxRows || out_max_seq < (budget < max_seq ? budget : max_seq)))
    return fail(FMX_ERR_SHAPE, "out_max_seq %lld", (long long)out_max_seq);
  if (!slots && n_slots < batch) return fail(FMX_ERR_SHAPE, "n_slots below batch without slots");
  if (batch == 0) return ok();
  fmx_heads kc_v, vc_v, ko_v, vo_v;
  FMX_RC(check_view(k_cache, "k_cache", n_slots, max_seq, n_kv_heads, 2, 1, &kc_v));
  FMX_RC(check_view(v_cache, "v_cache", n_slots, max_seq, n_kv_heads, 2, 1, &vc_v));
  k_cache = &kc_v;
  v_cache = &vc_v;
  if (!weights || !lengths || !lengths_out) return fail(FMX_ERR_ARG, "NULL weights, lengths or lengths_out");
  if (!aligned(weights, 4) || !aligned(weights_out, 4)) return fail(FMX_ERR_ARG, "weights not 4-byte aligned");
  if (!in_place) {
    FMX_RC(check_view(k_out, "k_out", n_slots, out_max_seq, n_kv_heads, 2, 1, &ko_v));
    FMX_RC(check_view(v_out, "v_out", n_slots, out_max_seq, n_kv_heads, 2, 1, &vo_v));
    k_out = &ko_v;
    v_out = &vo_v;
  } else {
    k_out = k_cache;
    v_out = v_cache;
    weights_out = weights;
    out_max_seq = max_seq;
  }
  FMX_RC(check_written(*k_out, "keys", n_slots, out_max_seq, n_kv_heads));
  FMX_RC(check_written(*v_out, "values", n_slots, out_max_seq, n_kv_heads));
  FMX_RC(check_apart(*k_out, *v_out, in_place ? "caches" : "outputs", head_dim, 2));
  const Span ins[3] = {span(k_cache, n_slots, max_seq, n_kv_heads, head_dim, 2),
                       span(v_cache, n_slots, max_seq, n_kv_heads, head_dim, 2),
                       flat(weights, n_slots * n_kv_heads * max_seq)};
  const Span outs[3] = {span(k_out, n_slots, out_max_seq, n_kv_heads, head_dim, 2),
                        span(v_out, n_slots, out_max_seq, n_kv_heads, head_dim, 2),
                        flat(weights_out, n_slots * n_kv_heads * out_max_seq)};
  if (!in_place)
    for (const Span& o : outs)
      for (const Span& i : ins)
        if (overlap(o, i)) return fail(FMX_ERR_ARG, "an output overlaps an input");
  if (overlap(outs[2], outs[0]) || overlap(outs[2], outs[1])) return fail(FMX_ERR_ARG, "weights overlap a cache");
  // kept and lengths_out, against everything but lengths_out that is lengths
  const Span kept_s = flat(kept, batch * n_kv_heads * budget), lens_s = flat(lengths, batch);
  const Span lens_out_s = flat(lengths_out, batch), slots_s = flat(slots, slots ? batch : 0);
  for (const Span& o : {kept_s, lens_out_s}) {
    for (const Span& i : {ins[0], ins[1], ins[2], outs[0], outs[1], outs[2], slots_s})
      if (overlap(o, i)) return fail(FMX_ERR_ARG, "kept or lengths_out overlaps another array");
    if (overlap(o, lens_s) && lengths_out != lengths) return fail(FMX_ERR_ARG, "kept or lengths_out overlaps lengths");
  }
  if (overlap(kept_s, lens_s) || overlap(kept_s, lens_out_s))
    return fail(FMX_ERR_ARG, "kept overlaps lengths or lengths_out");
  hipStream_t stream = static_cast<hipStream_t>(stream_);
  EvictArgs a{};
  a.B = static_cast<int>(batch);
  a.nkv = static_cast<int>(n_kv_heads);
  a.row_bytes = head_dim * 2;
  a.k = static_cast<const uint8_t*>(k_cache->data);
  a.v = static_cast<const uint8_t*>(v_cache->data);
  a.k_bs = 2 * k_cache->batch_stride;
  a.k_ts = 2 * k_cache->token_stride;
  a.k_hs = 2 * k_cache->head_stride;
  a.v_bs = 2 * v_cache->batch_stride;
  a.v_ts = 2 * v_cache->token_stride;
  a.v_hs = 2 * v_cache->head_stride;
  a.k_out = static_cast<uint8_t*>(k_out->data);
  a.v_out = static_cast<uint8_t*>(v_out->data);
  a.ko_bs = 2 * k_out->batch_stride;
  a.ko_ts = 2 * k_out->token_stride;
  a.ko_hs = 2 * k_out->head_stride;
  a.vo_bs = 2 * v_out->batch_stride;
  a.vo_ts = 2 * v_out->token_stride;
  a.vo_hs = 2 * v_out->head_stride;
  a.w = weights;
  a.w_out = weights_out;
  a.n_slots = n_slots;
  a.S = max_seq;
  a.S_out = out_max_seq;
  a.lens = lengths;
  a.slots = slots;
  a.budget = budget;
  a.sinks = sinks;
  a.recent = recent;
  a.lens_out = lengths_out;
  a.in_place = in_place;
  if (!evict_fits(a)) return fail(FMX_ERR_UNSUPPORTED, "more rows than launches of fewer than 2^32 threads move");
  Workspace ws;
  if (!kept) {
    FMX_RC(ws.bind(workspace, workspace_bytes, fmx_cache_evict_workspace_size(batch, n_kv_heads, budget), stream));
    kept = static_cast<int32_t*>(ws.p);
  }
  a.kept = kept;
  FMX_HIP(launch_evict(a, stream));
  return ok();
}

}  // extern "C"
