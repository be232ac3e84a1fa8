// fmx_checks.hpp -- argument checks and workspaces that the C entry points on
// strided views share (fmx_cache.cpp, fmx_ssm.cpp; library-internal).
#pragma once

#include <hip/hip_runtime.h>

#include <cstdarg>
#include <cstdio>

#include "../../include/fmx_cache.h"
#include "fmx_cache_kernels.hpp"

namespace fmx {

int set_error(int status, const char* msg);
void clear_error();

namespace {

inline int fail(int status, const char* fmt, ...) {
  char buf[512];
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(buf, sizeof(buf), fmt, ap);
  va_end(ap);
  return set_error(status, buf);
}

inline int ok() {
  clear_error();
  return FMX_OK;
}

inline bool aligned(const void* p, size_t a) { return (reinterpret_cast<uintptr_t>(p) % a) == 0; }

#define FMX_HIP(expr)                                                              \
  do {                                                                             \
    hipError_t e_ = (expr);                                                        \
    if (e_ != hipSuccess)                                                          \
      return fail(FMX_ERR_HIP, "%s: %s", #expr, hipGetErrorString(e_));            \
  } while (0)

#define FMX_RC(expr)        \
  do {                      \
    int rc_ = (expr);       \
    if (rc_) return rc_;    \
  } while (0)

// The caller's workspace, or one of the call's own (stream-ordered).
struct Workspace {
  void* p = nullptr;
  bool owned = false;
  hipStream_t stream = nullptr;
  ~Workspace() {
    if (owned) (void)hipFreeAsync(p, stream);
  }
  int bind(void* ws, size_t ws_bytes, size_t need, hipStream_t s) {
    if (need == 0) return FMX_OK;
    if (ws) {
      if (ws_bytes < need) return fail(FMX_ERR_WORKSPACE, "workspace %zu bytes, need %zu", ws_bytes, need);
      if (!aligned(ws, 256)) return fail(FMX_ERR_ARG, "workspace not 256-byte aligned");
      p = ws;
      return FMX_OK;
    }
    FMX_HIP(hipMallocAsync(&p, need, s));
    owned = true;
    stream = s;
    return FMX_OK;
  }
};

// strides: element offsets, and sums of a few of them, stay within 63 bits
// whatever the rows' count
constexpr int64_t kMaxStride = int64_t{1} << 34;

// A view of [nb, nt, nh] rows into *out (strides of axes with one entry are
// never used and taken as 0). data: aligned to `align` bytes (the element's
// size, or 16 with strides in whole 8s).
inline int check_view(const fmx_heads* v, const char* name, int64_t nb, int64_t nt, int64_t nh, size_t align,
               int stride_mult, fmx_heads* out) {
  if (!v || !v->data) return fail(FMX_ERR_ARG, "%s is NULL", name);
  if (!aligned(v->data, align)) return fail(FMX_ERR_ARG, "%s: data not %zu-byte aligned", name, align);
  if (v->batch_stride < 0 || v->token_stride < 0 || v->head_stride < 0)
    return fail(FMX_ERR_SHAPE, "%s: negative stride", name);
  *out = fmx_heads{v->data, nb > 1 ? v->batch_stride : 0, nt > 1 ? v->token_stride : 0, nh > 1 ? v->head_stride : 0};
  for (int64_t s : {out->batch_stride, out->token_stride, out->head_stride}) {
    if (s > kMaxStride) return fail(FMX_ERR_SHAPE, "%s: stride %lld", name, (long long)s);
    if (s % stride_mult) return fail(FMX_ERR_UNSUPPORTED, "%s: strides must be multiples of %d", name, stride_mult);
  }
  return FMX_OK;
}

inline HeadsView view(const fmx_heads* v) {
  return v ? HeadsView{v->data, v->batch_stride, v->token_stride, v->head_stride} : HeadsView{nullptr, 0, 0, 0};
}

inline bool same(const fmx_heads* a, const fmx_heads* b) {
  return a->data == b->data && a->batch_stride == b->batch_stride && a->token_stride == b->token_stride &&
         a->head_stride == b->head_stride;
}

// bytes from a view's first element to behind its last
struct Span {
  uintptr_t lo, hi;
};
inline Span span(const fmx_heads* v, int64_t nb, int64_t nt, int64_t nh, int64_t hd, int es) {
  const uintptr_t lo = reinterpret_cast<uintptr_t>(v->data);
  if (nb < 1 || nt < 1 || nh < 1) return {lo, lo};
  return {lo, lo + static_cast<uintptr_t>(((nb - 1) * v->batch_stride + (nt - 1) * v->token_stride +
                                           (nh - 1) * v->head_stride + hd) * es)};
}
inline bool overlap(const Span& a, const Span& b) { return a.lo < b.hi && b.lo < a.hi; }
inline Span flat(const void* p, int64_t n) {  // n elements of 4 bytes
  const uintptr_t lo = reinterpret_cast<uintptr_t>(p);
  return {lo, p ? lo + static_cast<uintptr_t>(n) * 4 : lo};
}

// A written view's rows of hd elements: two that are one row (a broadcast axis).
inline int check_written(const fmx_heads& v, const char* name, int64_t nb, int64_t nt, int64_t nh) {
  if ((nb > 1 && v.batch_stride == 0) || (nt > 1 && v.token_stride == 0) || (nh > 1 && v.head_stride == 0))
    return fail(FMX_ERR_ARG, "%s: written, with a stride of 0", name);
  return FMX_OK;
}

inline int elem_size(int dtype) { return dtype == FMX_F32 ? 4 : 2; }

}  // namespace

}  // namespace fmx
