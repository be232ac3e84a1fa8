// fmx_ssm_norm.hip -- the RMS norm of groups with its gate (the mixer's gated
// norm, server/src/nemotron_h.cpp):
//   gate first: u = x silu(z), u / rms(u) w;  otherwise x / rms(x) w silu(z)
//
// Bound by HBM: x and z are read and the result is written once. A group is
// taken whole by 4 to 64 neighbouring lanes or by a workgroup, which keep its
// products in registers between the sum and the division; groups of more than
// 1024 vectors are read a second time. 8192 rows of 8 groups of 512 in bf16: 45
// us, 4.5 TB/s.
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
// again), GR groups loaded before the first one's sum. (A vector and its gate's
// are loaded in a branch, which waits for both before the next pair.)
template <int DT, int VEC, int LN, int NV, int GR>
__global__ __launch_bounds__(kGateThreads) void gated_norm_kernel(GatedNormArgs a, NormPlan pl) {
  typedef typename El<DT>::T T;
  typedef Pack<T, VEC> V;
  static_assert(GR == 1 || (NV && LN < kGateThreads), "several groups: kept, within a wave");
  __shared__ float s_sum[kGateThreads / kWave];
  constexpr int kPer = kGateThreads / LN;  // groups of a workgroup at once
  const int j = threadIdx.x % LN, size = a.C / a.groups;
  const bool gate = a.z.p != nullptr;

  auto value = [&](const V& x, const V& z, int e) {
    const float v = El<DT>::ld(x.e[e]);
    return gate && a.gate_first ? v * silu_f32(El<DT>::ld(z.e[e])) : v;
  };
  int64_t xo[GR], zo[GR], oo[GR], wo[GR];
  bool live[GR];
#pragma unroll
  for (int r = 0; r < GR; ++r) {
    const uint32_t item = (blockIdx.x * GR + r) * kPer + threadIdx.x / LN;
    const uint32_t row = item / static_cast<uint32_t>(a.groups);
    const int g = static_cast<int>(item - row * a.groups);
    const int b = static_cast<int>(row / a.L), l = static_cast<int>(row % a.L);
    live[r] = item < pl.items && l < seq_length(a.lens, a.L, min(b, a.B - 1));
    wo[r] = static_cast<int64_t>(g) * size;
    xo[r] = b * a.x.bs + l * a.x.ts + wo[r];
    zo[r] = b * a.z.bs + l * a.z.ts + wo[r];
    oo[r] = b * a.out.bs + l * a.out.ts + wo[r];
  }
  if (LN == kGateThreads && !live[0]) return;  // (a workgroup's threads agree)

  auto store = [&](int r, int i, const float* u, const V& z, float f) {
    V y;
    V w{};
    if (a.w) w = norm_load<DT, VEC>(a.w, wo[r] + i * VEC);
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
      float v = u[e] * f;
      if (a.w) v *= El<DT>::ld(w.e[e]);
      if (gate && !a.gate_first) v *= silu_f32(El<DT>::ld(z.e[e]));
      y.e[e] = El<DT>::st(v);
    }
    *reinterpret_cast<V*>(static_cast<T*>(a.out.p) + oo[r] + i * VEC) = y;
  };

  constexpr int kKeep = NV ? NV : 1;
  V x[GR][kKeep], z[GR][kKeep];
  if (NV) {
#pragma unroll
    for (int r = 0; r < GR; ++r)
#pragma unroll
      for (int i = 0; i < kKeep; ++i) {
        x[r][i] = V{};
        z[r][i] = V{};
        if (live[r] && j + i * LN < pl.vecs) {
          x[r][i] = norm_load<DT, VEC>(a.x.p, xo[r] + (j + i * LN) * VEC);
          if (gate) z[r][i] = norm_load<DT, VEC>(a.z.p, zo[r] + (j + i * LN) * VEC);
        }
      }
  }
#pragma unroll
  for (int r = 0; r < GR; ++r) {
    float u[kKeep][VEC];
    float sum = 0.0f;
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
        if (j + i * LN < pl.vecs) add(x[r][i], z[r][i], u[i]);
    } else {
      for (int i = j; i < pl.vecs; i += LN) {
        const V xv = norm_load<DT, VEC>(a.x.p, xo[r] + static_cast<int64_t>(i) * VEC);
        const V zv = gate ? norm_load<DT, VEC>(a.z.p, zo[r] + static_cast<int64_t>(i) * VEC) : V{};
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
    if (!live[r]) continue;
    const float f = 1.0f / sqrtf(sum / static_cast<float>(size) + a.eps);
    if (NV) {
#pragma unroll
      for (int i = 0; i < kKeep; ++i)
        if (j + i * LN < pl.vecs) store(r, j + i * LN, u[i], z[r][i], f);
    } else {
      for (int i = j; i < pl.vecs; i += LN) {
        const V xv = norm_load<DT, VEC>(a.x.p, xo[r] + static_cast<int64_t>(i) * VEC);
        const V zv = gate ? norm_load<DT, VEC>(a.z.p, zo[r] + static_cast<int64_t>(i) * VEC) : V{};
#pragma unroll
        for (int e = 0; e < VEC; ++e) u[0][e] = value(xv, zv, e);
        store(r, i, u[0], zv, f);
      }
    }
  }
}

// Lanes of a group of so many vectors: up to three vectors a lane rather than
// more lanes with some idle (8192 rows of 16 groups of 256 in bf16: 16 lanes 45
// us, 64 72; of 8 groups of 512, four a lane: 53, 64 lanes 49).
int norm_lanes(int vecs) {
  if (vecs > 128) return kGateThreads;
  int n = 4;
  while (3 * n < vecs && n < kWave) n *= 4;
  return n;
}

int64_t norm_items(const GatedNormArgs& a) { return static_cast<int64_t>(a.B) * a.L * a.groups; }

// Two groups at a time where there are enough for it: 8192 rows of 8
// groups of 512 50.4 us in a graph, one 52.3, four 60.6. (Of several vectors
// a lane one group's are enough: 16 groups of 256 45, two at once 51.)
constexpr int norm_most_rounds(int vec) { return vec > 1 ? 2 : 1; }
int norm_rounds(const GatedNormArgs& a, int vec) {
  const int vecs = a.C / a.groups / vec, ln = norm_lanes(vecs);
  const bool enough = norm_items(a) >= int64_t{4096} * (kGateThreads / ln);
  return ln < kGateThreads && (vecs <= ln || ln == kWave) && enough ? norm_most_rounds(vec) : 1;
}
int64_t norm_blocks(const GatedNormArgs& a, int vec) {
  const int at_once = kGateThreads / norm_lanes(a.C / a.groups / vec) * norm_rounds(a, vec);
  return (norm_items(a) + at_once - 1) / at_once;
}

template <int DT, int VEC>
hipError_t gated_norm(const GatedNormArgs& a, hipStream_t stream) {
  const int64_t items = norm_items(a);
  if (items == 0) return hipSuccess;
  NormPlan pl{static_cast<uint32_t>(items), a.C / a.groups / VEC};
  constexpr int kRounds = norm_most_rounds(VEC);
  const int ln = norm_lanes(pl.vecs), rounds = norm_rounds(a, VEC);
  const dim3 grid(static_cast<uint32_t>(norm_blocks(a, VEC))), wg(kGateThreads);
#define FMX_NORM(LN, NV, GR) hipLaunchKernelGGL((gated_norm_kernel<DT, VEC, LN, NV, GR>), grid, wg, 0, stream, a, pl)
#define FMX_NORM_FEW(LN, NV)                        \
  do {                                              \
    if (rounds > 1)                                 \
      FMX_NORM(LN, NV, kRounds);                    \
    else                                            \
      FMX_NORM(LN, NV, 1);                          \
  } while (0)
  if (ln == 4 && pl.vecs <= 4) FMX_NORM_FEW(4, 1);
  else if (ln == 4 && pl.vecs <= 8) FMX_NORM(4, 2, 1);
  else if (ln == 4) FMX_NORM(4, 3, 1);
  else if (ln == 16 && pl.vecs <= 16) FMX_NORM_FEW(16, 1);
  else if (ln == 16 && pl.vecs <= 32) FMX_NORM(16, 2, 1);
  else if (ln == 16) FMX_NORM(16, 3, 1);
  else if (ln == 64 && pl.vecs <= 64) FMX_NORM_FEW(64, 1);
  else if (ln == 64) FMX_NORM_FEW(64, 2);
  else if (pl.vecs <= 256) FMX_NORM(256, 1, 1);
  else if (pl.vecs <= 512) FMX_NORM(256, 2, 1);
  else if (pl.vecs <= 1024) FMX_NORM(256, 4, 1);
  else FMX_NORM(256, 0, 1);
#undef FMX_NORM_FEW
#undef FMX_NORM
  return hipGetLastError();
}

// 16 bytes at once where every row starts on a word and groups are whole
// vectors (19143 rows of 3 groups of 320 in f16, the gate's 4440 bytes apart:
// 35 us, by elements 102), single elements otherwise
bool norm_wide(const GatedNormArgs& a, int dt) {
  const int es = dt == kElF32 ? 4 : 2, vec = 16 / es;
  bool wide = a.C / a.groups % vec == 0 && on_words(a.w);
  for (const HeadsView* v : {&a.x, &a.z, &a.out}) wide = wide && on_words(*v, es);
  return wide;
}

}  // namespace

// (max_blocks of up to 64 groups twice are fewer than 2^32: the kernel counts them in 32 bits)
bool gated_norm_fits(const GatedNormArgs& a, int dt) {
  return norm_blocks(a, norm_wide(a, dt) ? (dt == kElF32 ? 4 : 8) : 1) <= max_blocks(kGateThreads);
}

hipError_t launch_gated_norm(const GatedNormArgs& a, int dt, hipStream_t stream) {
  const bool wide = norm_wide(a, dt);
  if (dt == kElF32) return wide ? gated_norm<kElF32, 4>(a, stream) : gated_norm<kElF32, 1>(a, stream);
  if (dt == kElF16) return wide ? gated_norm<kElF16, 8>(a, stream) : gated_norm<kElF16, 1>(a, stream);
  return wide ? gated_norm<kElBf16, 8>(a, stream) : gated_norm<kElBf16, 1>(a, stream);
}

}  // namespace fmx
