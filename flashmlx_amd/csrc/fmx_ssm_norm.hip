// fmx_ssm_norm.hip -- the RMS norm of groups with its gate (the mixer's gated
// norm, server/src/nemotron_h.cpp):
//   gate first: u = x silu(z), u / rms(u) w;  otherwise x / rms(x) w silu(z)
//
// Bound by HBM: x and z are read and the result is written once. A group is
// taken whole by 2 to 64 neighbouring lanes or by a workgroup, which keep its
// products in registers between the sum and the division; longer groups are
// read a second time.
#include <algorithm>

#include "fmx_ssm_kernels.hpp"

namespace fmx {

namespace {

constexpr int kGateThreads = 256;

struct NormPlan {
  uint32_t items;     // (row, group) pairs
  int vecs;           // vectors of a group
};

template <int DT, int VEC>
__device__ inline Pack<typename El<DT>::T, VEC> norm_load(const void* p, int64_t at) {
  typedef typename El<DT>::T T;
  return *reinterpret_cast<const Pack<T, VEC>*>(static_cast<const T*>(p) + at);
}

// LN lanes per group (a workgroup for 256), NV vectors per lane kept (0: read
// again)
template <int DT, int VEC, int LN, int NV>
__global__ __launch_bounds__(kGateThreads) void gated_norm_kernel(GatedNormArgs a, NormPlan pl) {
  typedef typename El<DT>::T T;
  typedef Pack<T, VEC> V;
  __shared__ float s_sum[kGateThreads / kWave];
  constexpr int kPer = kGateThreads / LN;  // groups of a workgroup
  const uint32_t item = blockIdx.x * kPer + threadIdx.x / LN;
  const int j = threadIdx.x % LN;
  const uint32_t row = item / static_cast<uint32_t>(a.groups);
  const int g = static_cast<int>(item - row * a.groups);
  const int b = static_cast<int>(row / a.L), l = static_cast<int>(row % a.L);
  const bool live = item < pl.items && l < seq_length(a.lens, a.L, min(b, a.B - 1));
  if (LN == kGateThreads && !live) return;  // (a workgroup's threads agree)
  const int size = a.C / a.groups;
  const int64_t xo = b * a.x.bs + l * a.x.ts + static_cast<int64_t>(g) * size;
  const int64_t zo = b * a.z.bs + l * a.z.ts + static_cast<int64_t>(g) * size;
  const int64_t oo = b * a.out.bs + l * a.out.ts + static_cast<int64_t>(g) * size;
  const bool gate = a.z.p != nullptr;

  auto value = [&](const V& x, const V& z, int e) {
    const float v = El<DT>::ld(x.e[e]);
    return gate && a.gate_first ? v * silu_f32(El<DT>::ld(z.e[e])) : v;
  };
  auto store = [&](int i, const float* u, const V& z, float f) {
    V y;
    V w{};
    if (a.w) w = norm_load<DT, VEC>(a.w, static_cast<int64_t>(g) * size + i * VEC);
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
      float v = u[e] * f;
      if (a.w) v *= El<DT>::ld(w.e[e]);
      if (gate && !a.gate_first) v *= silu_f32(El<DT>::ld(z.e[e]));
      y.e[e] = El<DT>::st(v);
    }
    *reinterpret_cast<V*>(static_cast<T*>(a.out.p) + oo + i * VEC) = y;
  };

  constexpr int kKeep = NV ? NV : 1;
  V x[kKeep], z[kKeep];
  float sum = 0.0f;
  if (NV) {
#pragma unroll
    for (int i = 0; i < kKeep; ++i) {
      x[i] = V{};
      z[i] = V{};
      if (live && j + i * LN < pl.vecs) {
        x[i] = norm_load<DT, VEC>(a.x.p, xo + (j + i * LN) * VEC);
        if (gate) z[i] = norm_load<DT, VEC>(a.z.p, zo + (j + i * LN) * VEC);
      }
    }
  }
  float u[kKeep][VEC];
  auto add = [&](const V& x, const V& z, float* u) {
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
      u[e] = value(x, z, e);
      sum = __builtin_fmaf(u[e], u[e], sum);
    }
  };
  if (NV) {
#pragma unroll
    for (int i = 0; i < kKeep; ++i)
      if (j + i * LN < pl.vecs) add(x[i], z[i], u[i]);
  } else if (live) {
    for (int i = j; i < pl.vecs; i += LN) {
      const V xv = norm_load<DT, VEC>(a.x.p, xo + static_cast<int64_t>(i) * VEC);
      const V zv = gate ? norm_load<DT, VEC>(a.z.p, zo + static_cast<int64_t>(i) * VEC) : V{};
      add(xv, zv, u[0]);
    }
  }
  if (LN == kGateThreads) {
#pragma unroll
    for (int m = 1; m < kWave; m *= 2) sum += __shfl_xor(sum, m);
    if (threadIdx.x % kWave == 0) s_sum[threadIdx.x / kWave] = sum;
    __syncthreads();
    sum = 0.0f;
#pragma unroll
    for (int i = 0; i < kGateThreads / kWave; ++i) sum += s_sum[i];
  } else {
#pragma unroll
    for (int m = 1; m < LN; m *= 2) sum += __shfl_xor(sum, m);
  }
  if (!live) return;
  const float f = 1.0f / sqrtf(sum / static_cast<float>(size) + a.eps);
  if (NV) {
#pragma unroll
    for (int i = 0; i < kKeep; ++i)
      if (j + i * LN < pl.vecs) store(j + i * LN, u[i], z[i], f);
  } else {
    for (int i = j; i < pl.vecs; i += LN) {
      const V xv = norm_load<DT, VEC>(a.x.p, xo + static_cast<int64_t>(i) * VEC);
      const V zv = gate ? norm_load<DT, VEC>(a.z.p, zo + static_cast<int64_t>(i) * VEC) : V{};
#pragma unroll
      for (int e = 0; e < VEC; ++e) u[0][e] = value(xv, zv, e);
      store(i, u[0], zv, f);
    }
  }
}

// lanes of a group of so many vectors
int norm_lanes(int vecs) {
  if (vecs > 128) return kGateThreads;
  int n = 4;
  while (n < vecs && n < kWave) n *= 4;
  return n;
}

int64_t norm_items(const GatedNormArgs& a) { return static_cast<int64_t>(a.B) * a.L * a.groups; }

template <int DT, int VEC>
hipError_t gated_norm(const GatedNormArgs& a, hipStream_t stream) {
  const int64_t items = norm_items(a);
  if (items == 0) return hipSuccess;
  NormPlan pl{static_cast<uint32_t>(items), a.C / a.groups / VEC};
  const int ln = norm_lanes(pl.vecs), per = kGateThreads / ln;
  const dim3 grid(static_cast<uint32_t>((items + per - 1) / per)), wg(kGateThreads);
#define FMX_NORM(LN, NV) hipLaunchKernelGGL((gated_norm_kernel<DT, VEC, LN, NV>), grid, wg, 0, stream, a, pl)
  if (ln == 4) FMX_NORM(4, 1);
  else if (ln == 16) FMX_NORM(16, 1);
  else if (ln == 64 && pl.vecs <= 64) FMX_NORM(64, 1);
  else if (ln == 64) FMX_NORM(64, 2);
  else if (pl.vecs <= 256) FMX_NORM(256, 1);
  else if (pl.vecs <= 512) FMX_NORM(256, 2);
  else if (pl.vecs <= 1024) FMX_NORM(256, 4);
  else FMX_NORM(256, 0);
#undef FMX_NORM
  return hipGetLastError();
}

}  // namespace

bool gated_norm_fits(const GatedNormArgs& a) { return norm_items(a) <= max_blocks(kGateThreads); }

hipError_t launch_gated_norm(const GatedNormArgs& a, int dt, hipStream_t stream) {
  // 16-byte vectors where every row and group falls on them, single elements otherwise
  const int es = dt == kElF32 ? 4 : 2, vec = 16 / es;
  bool wide = a.C / a.groups % vec == 0 && reinterpret_cast<uintptr_t>(a.w) % 16 == 0;
  for (const HeadsView* v : {&a.x, &a.z, &a.out}) wide = wide && on_vectors(*v, es, vec);
  if (dt == kElF32) return wide ? gated_norm<kElF32, 4>(a, stream) : gated_norm<kElF32, 1>(a, stream);
  if (dt == kElF16) return wide ? gated_norm<kElF16, 8>(a, stream) : gated_norm<kElF16, 1>(a, stream);
  return wide ? gated_norm<kElBf16, 8>(a, stream) : gated_norm<kElBf16, 1>(a, stream);
}

}  // namespace fmx
