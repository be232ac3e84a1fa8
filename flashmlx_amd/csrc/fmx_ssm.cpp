// fmx_ssm.cpp -- C-ABI of the state space layer's operators
// (include/fmx_ssm.h): argument checks, workspaces and launches.
#include <hip/hip_runtime.h>

#include <cmath>

#include "../../include/fmx_ssm.h"
#include "fmx_checks.hpp"
#include "fmx_ssm_kernels.hpp"

using namespace fmx;

namespace {

constexpr int64_t kMaxRows = FMX_CACHE_MAX_ROWS;
constexpr int64_t kMaxChannels = int64_t{1} << 20;
constexpr int64_t kMaxHeads = 65535;

int check_rows(int64_t batch, int64_t seq_len, int64_t n_slots) {
  if (batch < 0 || seq_len < 0 || batch > kMaxRows || seq_len > kMaxRows || batch * seq_len > kMaxRows)
    return fail(FMX_ERR_SHAPE, "batch %lld, seq_len %lld (at most 2^24 rows)", (long long)batch, (long long)seq_len);
  if (n_slots < 0 || n_slots > kMaxRows) return fail(FMX_ERR_SHAPE, "n_slots %lld (at most 2^24)", (long long)n_slots);
  return FMX_OK;
}

int element(int dtype, bool f32) {
  return dtype == FMX_BF16 ? kElBf16 : dtype == FMX_F16 ? kElF16 : f32 && dtype == FMX_F32 ? kElF32 : -1;
}

Span bytes(const void* p, int64_t n) {
  const uintptr_t lo = reinterpret_cast<uintptr_t>(p);
  return {lo, p ? lo + static_cast<uintptr_t>(n) : lo};
}

// an array that a call reads or writes, for the checks of what overlaps
struct Named {
  const char* name;
  Span at;
};

// `out` against everything else
template <int N>
int check_clear(const Named& out, const Named (&others)[N]) {
  for (const Named& o : others)
    if (overlap(out.at, o.at)) return fail(FMX_ERR_ARG, "%s overlaps %s", out.name, o.name);
  return FMX_OK;
}

int check_aligned(const void* p, const char* name, size_t align) {
  return aligned(p, align) ? FMX_OK : fail(FMX_ERR_ARG, "%s: not %zu-byte aligned", name, align);
}

// heads, groups and dimensions of a layer
int check_dims(int64_t nh, int64_t hd, int64_t groups, int64_t N) {
  if (nh < 1 || nh > kMaxHeads || groups < 1 || nh % groups)
    return fail(FMX_ERR_SHAPE, "n_heads %lld, n_groups %lld (heads in whole groups)", (long long)nh, (long long)groups);
  if (hd < 1 || N < 1) return fail(FMX_ERR_SHAPE, "head_dim %lld, state_dim %lld", (long long)hd, (long long)N);
  if (hd % 8 || hd > kScanMaxDim || N % 8 || N > kScanMaxDim)
    return fail(FMX_ERR_UNSUPPORTED, "head_dim %lld, state_dim %lld (multiples of 8, at most %d)", (long long)hd,
                (long long)N, kScanMaxDim);
  return FMX_OK;
}

int check_limits(float lo, float hi) {
  if (!std::isfinite(lo) || std::isnan(hi) || lo > hi) return fail(FMX_ERR_ARG, "dt_min %g, dt_max %g", lo, hi);
  return FMX_OK;
}

int check_scan_shape(const fmx_ssm_shape* s, int64_t n_slots) {
  if (!s) return fail(FMX_ERR_ARG, "shape is NULL");
  if (element(s->dtype, false) < 0) return fail(FMX_ERR_DTYPE, "dtype %d (bf16 or float16)", s->dtype);
  FMX_RC(check_rows(s->batch, s->seq_len, n_slots));
  FMX_RC(check_dims(s->n_heads, s->head_dim, s->n_groups, s->state_dim));
  return check_limits(s->dt_min, s->dt_max);
}

ScanArgs scan_args(const fmx_ssm_shape* s) {
  ScanArgs a{};
  a.B = static_cast<int>(s->batch);
  a.L = static_cast<int>(s->seq_len);
  a.nh = static_cast<int>(s->n_heads);
  a.hd = static_cast<int>(s->head_dim);
  a.groups = static_cast<int>(s->n_groups);
  a.N = static_cast<int>(s->state_dim);
  a.rep = a.nh / a.groups;
  a.softplus = s->dt_softplus != 0;
  a.dt_min = s->dt_min;
  a.dt_max = s->dt_max;
  return a;
}

int check_layer(const fmx_ssm_layer* l, int64_t batch, int64_t n_slots) {
  if (!l) return fail(FMX_ERR_ARG, "layer is NULL");
  if (element(l->dtype, false) < 0) return fail(FMX_ERR_DTYPE, "dtype %d (bf16 or float16)", l->dtype);
  FMX_RC(check_rows(batch, 1, n_slots));
  FMX_RC(check_dims(l->n_heads, l->head_dim, l->n_groups, l->state_dim));
  if (l->taps < 2 || l->taps > kMaxTaps) return fail(FMX_ERR_SHAPE, "taps %lld (2 .. %d)", (long long)l->taps, kMaxTaps);
  if (l->activation != FMX_ACT_NONE && l->activation != FMX_ACT_SILU)
    return fail(FMX_ERR_ARG, "activation %d", l->activation);
  if (l->n_heads * l->head_dim + 2 * l->n_groups * l->state_dim > kMaxChannels)
    return fail(FMX_ERR_SHAPE, "more than 2^20 channels");
  if (l->norm_groups < 1 || l->n_heads * l->head_dim % l->norm_groups)
    return fail(FMX_ERR_SHAPE, "norm_groups %lld of %lld channels", (long long)l->norm_groups,
                (long long)(l->n_heads * l->head_dim));
  if (!std::isfinite(l->eps) || !(l->eps > 0.0f)) return fail(FMX_ERR_ARG, "eps must be finite and positive");
  return check_limits(l->dt_min, l->dt_max);
}

StepArgs step_args(const fmx_ssm_layer* l, int64_t batch) {
  StepArgs a{};
  a.B = static_cast<int>(batch);
  a.nh = static_cast<int>(l->n_heads);
  a.hd = static_cast<int>(l->head_dim);
  a.groups = static_cast<int>(l->n_groups);
  a.N = static_cast<int>(l->state_dim);
  a.rep = a.nh / a.groups;
  a.taps = static_cast<int>(l->taps);
  a.silu = l->activation == FMX_ACT_SILU;
  a.C = a.nh * a.hd + 2 * a.groups * a.N;
  a.conv_w = l->conv_weight;
  a.conv_b = l->conv_bias;
  a.a = l->a;
  a.d = l->d;
  a.dt_bias = l->dt_bias;
  a.softplus = l->dt_softplus != 0;
  a.dt_min = l->dt_min;
  a.dt_max = l->dt_max;
  a.norm_w = l->norm_weight;
  a.norm_groups = static_cast<int>(l->norm_groups);
  a.eps = l->eps;
  a.gate_first = l->gate_first != 0;
  return a;
}

int too_much() { return fail(FMX_ERR_UNSUPPORTED, "more work than launches of fewer than 2^32 threads"); }

// Each call's checks: what its kernels are handed, and whether there is
// anything to run. Nothing is launched or allocated.
int plan_conv(int dtype, int64_t batch, int64_t seq_len, int64_t channels, int64_t taps, int activation,
              const fmx_heads* x, const void* weight, const void* bias, const void* state_in, void* state_out,
              int64_t n_slots, const int32_t* lengths, const int32_t* slots, const fmx_heads* out, ConvArgs* plan,
              bool* run) {
  *run = false;
  if (element(dtype, true) < 0) return fail(FMX_ERR_DTYPE, "dtype %d (bf16, float16 or float32)", dtype);
  FMX_RC(check_rows(batch, seq_len, n_slots));
  if (channels < 1 || channels > kMaxChannels) return fail(FMX_ERR_SHAPE, "channels %lld (1 .. 2^20)", (long long)channels);
  if (taps < 1 || taps > kMaxTaps) return fail(FMX_ERR_SHAPE, "taps %lld (1 .. %d)", (long long)taps, kMaxTaps);
  if (activation != FMX_ACT_NONE && activation != FMX_ACT_SILU) return fail(FMX_ERR_ARG, "activation %d", activation);
  if (taps == 1) state_in = state_out = nullptr;
  if (batch == 0 || (seq_len == 0 && (!state_out || state_out == state_in))) return FMX_OK;
  const int es = elem_size(dtype);
  fmx_heads x_v{}, out_v{};
  // (the kernel reads the weights whatever the lengths are)
  if (!weight) return fail(FMX_ERR_ARG, "weight is NULL");
  if (seq_len > 0) {
    FMX_RC(check_view(x, "x", batch, seq_len, 1, es, 1, &x_v));
    FMX_RC(check_view(out, "out", batch, seq_len, 1, es, 1, &out_v));
    FMX_RC(check_written(out_v, "out", batch, seq_len, 1));
  }
  const struct { const void* p; const char* name; } arrays[] = {
      {weight, "weight"}, {bias, "bias"}, {state_in, "state_in"}, {state_out, "state_out"}};
  for (const auto& r : arrays) FMX_RC(check_aligned(r.p, r.name, es));
  const int64_t state = n_slots * (taps - 1) * channels * es;
  const Named o{"out", span(&out_v, batch, seq_len, 1, channels, es)};
  const Named so{"state_out", bytes(state_out, state)}, si{"state_in", bytes(state_in, state)};
  const Named xs{"x", span(&x_v, batch, seq_len, 1, channels, es)};
  const Named ws{"weight", bytes(weight, channels * taps * es)}, bs{"bias", bytes(bias, channels * es)};
  const Named ls{"lengths", flat(lengths, batch)}, ss{"slots", flat(slots, batch)};
  FMX_RC(check_clear(o, {xs, ws, bs, si, so, ls, ss}));
  FMX_RC(check_clear(so, {xs, ws, bs, ls, ss}));
  if (state_out != state_in) FMX_RC(check_clear(so, {si}));
  ConvArgs& a = *plan;
  a = ConvArgs{};
  a.B = static_cast<int>(batch);
  a.L = static_cast<int>(seq_len);
  a.C = static_cast<int>(channels);
  a.taps = static_cast<int>(taps);
  a.silu = activation == FMX_ACT_SILU;
  a.x = view(&x_v);
  a.out = view(&out_v);
  a.w = weight;
  a.bias = bias;
  a.s_in = state_in;
  a.s_out = state_out;
  a.n_slots = n_slots;
  a.lens = lengths;
  a.slots = slots;
  if (!conv_fits(a, element(dtype, true))) return too_much();
  *run = true;
  return FMX_OK;
}

int plan_scan(const fmx_ssm_shape* shape, const fmx_heads* x, const fmx_heads* dt, const float* a, const fmx_heads* b,
              const fmx_heads* c, const float* d, const float* dt_bias, const float* state_in, float* state_out,
              int64_t n_slots, const int32_t* lengths, const int32_t* slots, const fmx_heads* out, ScanArgs* plan,
              bool* run) {
  *run = false;
  FMX_RC(check_scan_shape(shape, n_slots));
  const int64_t B = shape->batch, L = shape->seq_len, nh = shape->n_heads, hd = shape->head_dim;
  const int64_t G = shape->n_groups, N = shape->state_dim;
  if (B == 0 || (L == 0 && (!state_out || state_out == state_in))) return FMX_OK;
  ScanArgs& s = *plan;
  s = scan_args(shape);
  fmx_heads x_v{}, dt_v{}, b_v{}, c_v{}, out_v{};
  if (!a) return fail(FMX_ERR_ARG, "a is NULL");
  if (L > 0) {
    FMX_RC(check_view(x, "x", B, L, nh, 16, 8, &x_v));
    FMX_RC(check_view(dt, "dt", B, L, nh, 2, 1, &dt_v));
    FMX_RC(check_view(b, "b", B, L, G, 16, 8, &b_v));
    FMX_RC(check_view(c, "c", B, L, G, 16, 8, &c_v));
    FMX_RC(check_view(out, "out", B, L, nh, 16, 8, &out_v));
    FMX_RC(check_written(out_v, "out", B, L, nh));
  }
  for (const float* p : {a, d, dt_bias}) FMX_RC(check_aligned(p, "a, d or dt_bias", 4));
  FMX_RC(check_aligned(state_in, "state_in", 16));
  FMX_RC(check_aligned(state_out, "state_out", 16));
  const int64_t state = n_slots * nh * hd * N;
  const Named o{"out", span(&out_v, B, L, nh, hd, 2)};
  const Named so{"state_out", flat(state_out, state)}, si{"state_in", flat(state_in, state)};
  const Named xs{"x", span(&x_v, B, L, nh, hd, 2)}, ds{"dt", span(&dt_v, B, L, nh, 1, 2)};
  const Named bs{"b", span(&b_v, B, L, G, N, 2)}, cs{"c", span(&c_v, B, L, G, N, 2)};
  const Named as{"a", flat(a, nh)}, dd{"d", flat(d, nh)}, db{"dt_bias", flat(dt_bias, nh)};
  const Named ls{"lengths", flat(lengths, B)}, ss{"slots", flat(slots, B)};
  FMX_RC(check_clear(o, {xs, ds, bs, cs, as, dd, db, si, so, ls, ss}));
  FMX_RC(check_clear(so, {xs, ds, bs, cs, as, dd, db, ls, ss}));
  if (state_out != state_in) FMX_RC(check_clear(so, {si}));
  s.x = view(&x_v);
  s.dt = view(&dt_v);
  s.b = view(&b_v);
  s.c = view(&c_v);
  s.out = view(&out_v);
  s.a = a;
  s.d = d;
  s.dt_bias = dt_bias;
  s.s_in = state_in;
  s.s_out = state_out;
  s.n_slots = n_slots;
  s.lens = lengths;
  s.slots = slots;
  if (!scan_fits(s)) return too_much();
  *run = true;
  return FMX_OK;
}

int plan_norm(int dtype, int64_t batch, int64_t seq_len, int64_t channels, int64_t n_groups, float eps, int gate_first,
              const fmx_heads* x, const fmx_heads* z, const void* weight, const int32_t* lengths, const fmx_heads* out,
              GatedNormArgs* plan, bool* run) {
  *run = false;
  if (element(dtype, true) < 0) return fail(FMX_ERR_DTYPE, "dtype %d (bf16, float16 or float32)", dtype);
  FMX_RC(check_rows(batch, seq_len, 0));
  if (channels < 1 || channels > kMaxChannels || n_groups < 1 || channels % n_groups)
    return fail(FMX_ERR_SHAPE, "channels %lld (1 .. 2^20) in %lld groups", (long long)channels, (long long)n_groups);
  if (!std::isfinite(eps) || !(eps > 0.0f)) return fail(FMX_ERR_ARG, "eps must be finite and positive");
  if (batch * seq_len == 0) return FMX_OK;
  const int es = elem_size(dtype);
  fmx_heads x_v{}, z_v{}, out_v{};
  FMX_RC(check_view(x, "x", batch, seq_len, 1, es, 1, &x_v));
  if (z) FMX_RC(check_view(z, "z", batch, seq_len, 1, es, 1, &z_v));
  FMX_RC(check_view(out, "out", batch, seq_len, 1, es, 1, &out_v));
  FMX_RC(check_written(out_v, "out", batch, seq_len, 1));
  FMX_RC(check_aligned(weight, "weight", es));
  const Named o{"out", span(&out_v, batch, seq_len, 1, channels, es)};
  if (!same(&out_v, &x_v)) FMX_RC(check_clear(o, {{"x", span(&x_v, batch, seq_len, 1, channels, es)}}));
  if (z && !same(&out_v, &z_v)) FMX_RC(check_clear(o, {{"z", span(&z_v, batch, seq_len, 1, channels, es)}}));
  FMX_RC(check_clear(o, {{"weight", bytes(weight, channels * es)}, {"lengths", flat(lengths, batch)}}));
  GatedNormArgs& a = *plan;
  a = GatedNormArgs{};
  a.B = static_cast<int>(batch);
  a.L = static_cast<int>(seq_len);
  a.C = static_cast<int>(channels);
  a.groups = static_cast<int>(n_groups);
  a.eps = eps;
  a.gate_first = gate_first != 0;
  a.x = view(&x_v);
  if (z) a.z = view(&z_v);
  a.out = view(&out_v);
  a.w = weight;
  a.lens = lengths;
  if (!gated_norm_fits(a, element(dtype, true))) return too_much();
  *run = true;
  return FMX_OK;
}

}  // namespace

extern "C" {

int fmx_causal_conv(int dtype, int64_t batch, int64_t seq_len, int64_t channels, int64_t taps, int activation,
                    const fmx_heads* x, const void* weight, const void* bias, const void* state_in, void* state_out,
                    int64_t n_slots, const int32_t* lengths, const int32_t* slots, const fmx_heads* out,
                    fmx_stream stream) {
  ConvArgs a;
  bool run;
  FMX_RC(plan_conv(dtype, batch, seq_len, channels, taps, activation, x, weight, bias, state_in, state_out, n_slots,
                   lengths, slots, out, &a, &run));
  if (run) FMX_HIP(launch_conv(a, element(dtype, true), static_cast<hipStream_t>(stream)));
  return ok();
}

size_t fmx_ssm_scan_workspace_size(const fmx_ssm_shape* shape) {
  if (check_scan_shape(shape, 0) || shape->batch == 0) return 0;
  return scan_workspace(scan_args(shape));
}

int fmx_ssm_scan(const fmx_ssm_shape* shape, const fmx_heads* x, const fmx_heads* dt, const float* a,
                 const fmx_heads* b, const fmx_heads* c, const float* d, const float* dt_bias, const float* state_in,
                 float* state_out, int64_t n_slots, const int32_t* lengths, const int32_t* slots, const fmx_heads* out,
                 void* workspace, size_t workspace_bytes, fmx_stream stream) {
  ScanArgs s;
  bool run;
  FMX_RC(plan_scan(shape, x, dt, a, b, c, d, dt_bias, state_in, state_out, n_slots, lengths, slots, out, &s, &run));
  if (!run) return ok();
  const hipStream_t st = static_cast<hipStream_t>(stream);
  Workspace ws;
  FMX_RC(ws.bind(workspace, workspace_bytes, scan_workspace(s), st));
  FMX_HIP(launch_scan(s, shape->dtype == FMX_F16, ws.p, st));
  return ok();
}

int fmx_gated_norm(int dtype, int64_t batch, int64_t seq_len, int64_t channels, int64_t n_groups, float eps,
                   int gate_first, const fmx_heads* x, const fmx_heads* z, const void* weight, const int32_t* lengths,
                   const fmx_heads* out, fmx_stream stream) {
  GatedNormArgs a;
  bool run;
  FMX_RC(plan_norm(dtype, batch, seq_len, channels, n_groups, eps, gate_first, x, z, weight, lengths, out, &a, &run));
  if (run) FMX_HIP(launch_gated_norm(a, element(dtype, true), static_cast<hipStream_t>(stream)));
  return ok();
}

int fmx_ssm_prompt_check(const fmx_ssm_layer* layer, int64_t batch, int64_t seq_len, const fmx_heads* xbc,
                         const fmx_heads* dt, const fmx_heads* z, void* conv_rows, void* scan_rows, void* conv_state,
                         int64_t conv_slots, float* state, int64_t n_slots, const int32_t* lengths,
                         const int32_t* slots, const fmx_heads* out) {
  if (!layer) return fail(FMX_ERR_ARG, "layer is NULL");
  const fmx_ssm_layer& l = *layer;
  const fmx_ssm_shape shape{l.dtype, batch, seq_len, l.n_heads, l.head_dim, l.n_groups, l.state_dim, l.dt_softplus,
                            l.dt_min, l.dt_max};
  FMX_RC(check_scan_shape(&shape, n_slots));
  const int64_t d = l.n_heads * l.head_dim, n = l.n_groups * l.state_dim, C = d + 2 * n;
  uint16_t* v = static_cast<uint16_t*>(conv_rows);
  const fmx_heads v_rows{v, seq_len * C, C, 0}, y_rows{scan_rows, seq_len * d, d, 0};
  const fmx_heads x{v, seq_len * C, C, l.head_dim}, b{v ? v + d : v, seq_len * C, C, l.state_dim},
      c{v ? v + d + n : v, seq_len * C, C, l.state_dim}, y{scan_rows, seq_len * d, d, l.head_dim};
  ConvArgs conv;
  ScanArgs scan;
  GatedNormArgs norm;
  bool run;
  FMX_RC(plan_conv(l.dtype, batch, seq_len, C, l.taps, l.activation, xbc, l.conv_weight, l.conv_bias, conv_state,
                   conv_state, conv_slots, lengths, slots, &v_rows, &conv, &run));
  FMX_RC(plan_scan(&shape, &x, dt, l.a, &b, &c, l.d, l.dt_bias, state, state, n_slots, lengths, slots, &y, &scan, &run));
  FMX_RC(plan_norm(l.dtype, batch, seq_len, d, l.norm_groups, l.eps, l.gate_first, &y_rows, z, l.norm_weight, lengths,
                   out, &norm, &run));
  if (!run) return ok();
  // each call has looked at its own arrays: here one's outputs against those of the others
  const int64_t rows = batch * seq_len;
  const Named cs{"conv_state", bytes(l.taps > 1 ? conv_state : nullptr, conv_slots * (l.taps - 1) * C * 2)};
  const Named ss{"state", flat(state, n_slots * d * l.state_dim)};
  const Named vs{"conv_rows", bytes(v, rows * C * 2)}, ys{"scan_rows", bytes(scan_rows, rows * d * 2)};
  const fmx_heads dt_v{scan.dt.p, scan.dt.bs, scan.dt.ts, scan.dt.hs}, z_v{norm.z.p, norm.z.bs, norm.z.ts, 0};
  const fmx_heads out_v{norm.out.p, norm.out.bs, norm.out.ts, 0};
  const Named ds{"dt", span(&dt_v, batch, seq_len, l.n_heads, 1, 2)};
  const Named zs{"z", z ? span(&z_v, batch, seq_len, 1, d, 2) : Span{0, 0}};
  const Named as{"a", flat(l.a, l.n_heads)}, dd{"d", flat(l.d, l.n_heads)}, db{"dt_bias", flat(l.dt_bias, l.n_heads)};
  const Named nw{"norm_weight", bytes(l.norm_weight, 2 * d)}, ls{"lengths", flat(lengths, batch)};
  const Named cw{"conv_weight", bytes(l.conv_weight, 2 * C * l.taps)}, cb{"conv_bias", bytes(l.conv_bias, 2 * C)};
  FMX_RC(check_clear(cs, {ss, vs, ys, ds, zs, as, dd, db, nw}));
  FMX_RC(check_clear(ss, {vs, ys, zs, nw, cw, cb}));
  FMX_RC(check_clear(vs, {ys, ds, zs, as, dd, db, nw}));
  FMX_RC(check_clear(ys, {zs, nw, cw, cb, ls}));
  FMX_RC(check_clear(Named{"out", span(&out_v, batch, seq_len, 1, d, 2)}, {cs, ss, cw, cb, as, dd, db}));
  return ok();
}

size_t fmx_ssm_step_workspace_size(const fmx_ssm_layer* layer, int64_t batch) {
  if (check_layer(layer, batch, 0)) return 0;
  return step_workspace(step_args(layer, batch));
}

int fmx_ssm_step(const fmx_ssm_layer* layer, int64_t batch, const fmx_heads* xbc, const fmx_heads* dt,
                 const fmx_heads* z, void* conv_state, float* state, int64_t n_slots, const int32_t* slots,
                 const fmx_heads* out, void* workspace, size_t workspace_bytes, fmx_stream stream) {
  FMX_RC(check_layer(layer, batch, n_slots));
  if (batch == 0) return ok();
  StepArgs a = step_args(layer, batch);
  const int64_t d = a.nh * static_cast<int64_t>(a.hd);
  if (!a.conv_w || !a.a) return fail(FMX_ERR_ARG, "conv_weight or a is NULL");
  if (n_slots > 0 && (!conv_state || !state)) return fail(FMX_ERR_ARG, "conv_state or state is NULL");
  fmx_heads x_v{}, dt_v{}, z_v{}, out_v{};
  FMX_RC(check_view(xbc, "xbc", batch, 1, 1, 2, 1, &x_v));
  FMX_RC(check_view(dt, "dt", batch, 1, a.nh, 2, 1, &dt_v));
  if (z) FMX_RC(check_view(z, "z", batch, 1, 1, 2, 1, &z_v));
  FMX_RC(check_view(out, "out", batch, 1, 1, 2, 1, &out_v));
  FMX_RC(check_written(out_v, "out", batch, 1, 1));
  const struct { const void* p; const char* name; size_t align; } arrays[] = {
      {a.conv_w, "conv_weight", 2}, {a.conv_b, "conv_bias", 2}, {a.norm_w, "norm_weight", 2}, {a.a, "a", 4},
      {a.d, "d", 4}, {a.dt_bias, "dt_bias", 4}, {conv_state, "conv_state", 16}, {state, "state", 16}};
  for (const auto& r : arrays) FMX_RC(check_aligned(r.p, r.name, r.align));
  const Named o{"out", span(&out_v, batch, 1, 1, d, 2)};
  const Named cs{"conv_state", bytes(conv_state, n_slots * (a.taps - 1) * a.C * 2)};
  const Named st{"state", flat(state, n_slots * d * a.N)};
  const Named in[] = {{"xbc", span(&x_v, batch, 1, 1, a.C, 2)}, {"dt", span(&dt_v, batch, 1, a.nh, 1, 2)},
                      {"z", z ? span(&z_v, batch, 1, 1, d, 2) : Span{0, 0}},
                      {"conv_weight", bytes(a.conv_w, int64_t{2} * a.C * a.taps)}, {"conv_bias", bytes(a.conv_b, int64_t{2} * a.C)},
                      {"a", flat(a.a, a.nh)}, {"d", flat(a.d, a.nh)}, {"dt_bias", flat(a.dt_bias, a.nh)},
                      {"norm_weight", bytes(a.norm_w, 2 * d)}, {"slots", flat(slots, batch)}};
  for (const Named& w : {o, cs, st}) FMX_RC(check_clear(w, in));
  FMX_RC(check_clear(o, {cs, st}));
  FMX_RC(check_clear(cs, {st}));
  a.xbc = view(&x_v);
  a.dt = view(&dt_v);
  if (z) a.z = view(&z_v);
  a.out = view(&out_v);
  a.conv_state = conv_state;
  a.state = state;
  a.n_slots = n_slots;
  a.slots = slots;
  if (!step_fits(a)) return too_much();
  const hipStream_t s = static_cast<hipStream_t>(stream);
  Workspace ws;
  FMX_RC(ws.bind(workspace, workspace_bytes, step_workspace(a), s));
  FMX_HIP(launch_step(a, layer->dtype == FMX_F16, ws.p, s));
  return ok();
}

}  // extern "C"
