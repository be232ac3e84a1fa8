// fmx_ssm_step.hip -- one decoded token of the state space layer: convolution,
// scan and gated norm in two launches (the mixer's cached step,
// server/src/nemotron_h.cpp).
//
//   step_kernel       a workgroup per part of a head's state: the
//                     convolution of its x, b and c channels (the heads of a
//                     group form theirs anew: taps products a channel), then
//                     one update of the state; y in fp32 to the workspace
//   step_norm_kernel  the gated norm of y, and the convolution's state moved
//                     on (only now: the first launch reads it in many places)
//
// Bound by HBM: the state is read and written once (256 sequences of 64 heads of
// 64 rows, 128 columns: 239 us, 4.6 TB/s, of which the second launch, in whose
// place nothing else runs, takes 17; one sequence 8.1, two launches of one chain
// of loads each).
#include <algorithm>

#include "fmx_ssm_kernels.hpp"

namespace fmx {

namespace {

constexpr int kStepThreads = 256;

// Channel ch of the convolution of sequence b, before anything is rounded. K:
// the taps, whose weights and state rows are then loaded before the first product
// (behind the row's own element and the bias); 0: a.taps of them, one by one.
template <bool F16, int K>
__device__ inline float step_conv(const StepArgs& a, int b, int64_t slot, int ch) {
  const int taps = K ? K : a.taps;
  const uint16_t* w = static_cast<const uint16_t*>(a.conv_w) + static_cast<int64_t>(ch) * taps;
  const uint16_t* s = static_cast<const uint16_t*>(a.conv_state) + slot * (taps - 1) * a.C + ch;
  const uint16_t x = (static_cast<const uint16_t*>(a.xbc.p) + b * a.xbc.bs)[ch];
  float v = a.conv_b ? Act<F16>::ld(static_cast<const uint16_t*>(a.conv_b)[ch]) : 0.0f;
  if (slot >= 0) {
    if (K) {
      uint16_t wk[K ? K : 1], sk[K ? K : 1];
#pragma unroll
      for (int k = 0; k < K - 1; ++k) {
        wk[k] = w[k];
        sk[k] = s[static_cast<int64_t>(k) * a.C];
      }
#pragma unroll
      for (int k = 0; k < K - 1; ++k) v = __builtin_fmaf(Act<F16>::ld(wk[k]), Act<F16>::ld(sk[k]), v);
    } else {
      for (int k = 0; k < taps - 1; ++k)
        v = __builtin_fmaf(Act<F16>::ld(w[k]), Act<F16>::ld(s[static_cast<int64_t>(k) * a.C]), v);
    }
  }
  v = __builtin_fmaf(Act<F16>::ld(w[taps - 1]), Act<F16>::ld(x), v);
  return a.silu ? silu_f32(v) : v;
}

template <bool F16, int LN, int RP, int K>
__global__ __launch_bounds__(kStepThreads) void step_kernel(StepArgs a, int parts, float* y_out) {
  constexpr int kRows = kStepThreads / LN * RP;
  constexpr int kCols = 4 * LN;
  __shared__ float s_x[kRows];
  __shared__ f32x4_t s_b[LN], s_c[LN];
  const int tid = threadIdx.x, col = tid % LN, sub = tid / LN;
  uint32_t id = blockIdx.x;
  const int row0 = static_cast<int>(id % parts) * kRows;
  id /= parts;
  const int h = static_cast<int>(id % a.nh), b = static_cast<int>(id / a.nh);
  const int g = h / a.rep;
  const int64_t slot = seq_slot(a.slots, a.n_slots, b);
  const int rows = min(kRows, a.hd - row0);
  float* state = a.state + ((slot * a.nh + h) * a.hd + row0) * a.N + 4 * col;

  StateRows<LN, RP> st;
#pragma unroll
  for (int i = 0; i < RP; ++i) {
    const int r = sub + i * (kStepThreads / LN);
    st.s[i] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
    if (slot >= 0 && r < rows && 4 * col < a.N)
      st.s[i] = *reinterpret_cast<const f32x4_t*>(state + static_cast<int64_t>(r) * a.N);
  }
  const int d = a.nh * a.hd, n = a.groups * a.N;
  for (int i = tid; i < kRows + 2 * kCols; i += kStepThreads) {
    if (i < kRows) {
      s_x[i] = i < rows ? step_conv<F16, K>(a, b, slot, h * a.hd + row0 + i) : 0.0f;
    } else {
      const bool second = i >= kRows + kCols;
      const int j = i - kRows - (second ? kCols : 0);
      const float v = j < a.N ? step_conv<F16, K>(a, b, slot, d + (second ? n : 0) + g * a.N + j) : 0.0f;
      reinterpret_cast<float*>(second ? s_c : s_b)[j] = v;
    }
  }
  const float dt = time_step(Act<F16>::ld((static_cast<const uint16_t*>(a.dt.p) + b * a.dt.bs)[h * a.dt.hs]), a.dt_bias,
                             h, a.softplus, a.dt_min, a.dt_max);
  const float decay = expf(dt * a.a[h]), skip = a.d ? a.d[h] : 0.0f;
  __syncthreads();
  float u[RP], xs[RP], y[RP];
#pragma unroll
  for (int i = 0; i < RP; ++i) {
    xs[i] = s_x[sub + i * (kStepThreads / LN)];
    u[i] = dt * xs[i];
  }
  st.step(decay, u, s_b[col], s_c[col], y);
#pragma unroll
  for (int i = 0; i < RP; ++i) {
    const int r = sub + i * (kStepThreads / LN);
    if (r >= rows) continue;
    if (slot >= 0 && 4 * col < a.N) *reinterpret_cast<f32x4_t*>(state + static_cast<int64_t>(r) * a.N) = st.s[i];
    if (col == LN - 1) y_out[static_cast<int64_t>(b) * d + h * a.hd + row0 + r] = a.d ? y[i] + skip * xs[i] : y[i];
  }
}

// Workgroups [0, norms): a sequence's group each, its products kept in
// registers (NV vectors of VEC a thread; 0: formed again); the others:
// vectors of channels' states, whose rows, as many as there are taps at run time,
// go through private memory where they are vectors of 8.
template <bool F16, int VEC, int NV>
__global__ __launch_bounds__(kStepThreads) void step_norm_kernel(StepArgs a, uint32_t norms, const float* y_in) {
  typedef Pack<uint16_t, VEC> V;
  typedef Pack<float, VEC> Y;
  __shared__ float s_sum[kStepThreads / kWave];
  const int tid = threadIdx.x;
  if (blockIdx.x >= norms) {
    const uint32_t vecs = a.C / VEC, per = (vecs + kStepThreads - 1) / kStepThreads, id = blockIdx.x - norms;
    const int b = static_cast<int>(id / per), v = static_cast<int>(id % per) * kStepThreads + tid;
    const int64_t slot = seq_slot(a.slots, a.n_slots, b);
    if (slot < 0 || v >= static_cast<int>(vecs)) return;
    uint16_t* s = static_cast<uint16_t*>(a.conv_state) + slot * (a.taps - 1) * a.C + v * VEC;
    V rows[kMaxTaps - 1];
#pragma unroll
    for (int k = 1; k < kMaxTaps; ++k) {
      if (k < a.taps - 1) rows[k - 1] = *reinterpret_cast<const V*>(s + static_cast<int64_t>(k) * a.C);
      if (k == a.taps - 1) rows[k - 1] = *reinterpret_cast<const V*>(static_cast<const uint16_t*>(a.xbc.p) + b * a.xbc.bs + v * VEC);
    }
#pragma unroll
    for (int k = 0; k < kMaxTaps - 1; ++k)
      if (k < a.taps - 1) *reinterpret_cast<V*>(s + static_cast<int64_t>(k) * a.C) = rows[k];
    return;
  }
  const int d = a.nh * a.hd, size = d / a.norm_groups, vecs = size / VEC;
  const int b = static_cast<int>(blockIdx.x / a.norm_groups), at = static_cast<int>(blockIdx.x % a.norm_groups) * size;
  const float* y = y_in + static_cast<int64_t>(b) * d + at;
  const uint16_t* z = a.z.p ? static_cast<const uint16_t*>(a.z.p) + b * a.z.bs + at : nullptr;
  const uint16_t* w = a.norm_w ? static_cast<const uint16_t*>(a.norm_w) + at : nullptr;
  uint16_t* out = static_cast<uint16_t*>(a.out.p) + b * a.out.bs + at;
  const bool first = z && a.gate_first;
  constexpr int kKeep = NV ? NV : 1;
  Y yv[kKeep];
  V zv[kKeep], wv[kKeep];
  auto read = [&](int k, int i) {
    yv[k] = *reinterpret_cast<const Y*>(y + i * VEC);
    zv[k] = z ? *reinterpret_cast<const V*>(z + i * VEC) : V{};
    wv[k] = w ? *reinterpret_cast<const V*>(w + i * VEC) : V{};
  };
  float sum = 0.0f;
  auto form = [&](int k) {
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
      if (first) yv[k].e[e] *= silu_f32(Act<F16>::ld(zv[k].e[e]));
      sum = __builtin_fmaf(yv[k].e[e], yv[k].e[e], sum);
    }
  };
  auto store = [&](int k, int i, float f) {
    V o;
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
      float v = yv[k].e[e] * f;
      if (w) v *= Act<F16>::ld(wv[k].e[e]);
      if (z && !first) v *= silu_f32(Act<F16>::ld(zv[k].e[e]));
      o.e[e] = Act<F16>::st(v);
    }
    *reinterpret_cast<V*>(out + i * VEC) = o;
  };
  if (NV) {
#pragma unroll
    for (int k = 0; k < kKeep; ++k)
      if (tid + k * kStepThreads < vecs) read(k, tid + k * kStepThreads);
#pragma unroll
    for (int k = 0; k < kKeep; ++k)
      if (tid + k * kStepThreads < vecs) form(k);
  } else {
    for (int i = tid; i < vecs; i += kStepThreads) {
      read(0, i);
      form(0);
    }
  }
#pragma unroll
  for (int m = 1; m < kWave; m *= 2) sum += __shfl_xor(sum, m);
  if (tid % kWave == 0) s_sum[tid / kWave] = sum;
  __syncthreads();
  sum = 0.0f;
#pragma unroll
  for (int i = 0; i < kStepThreads / kWave; ++i) sum += s_sum[i];
  const float f = 1.0f / sqrtf(sum / static_cast<float>(size) + a.eps);
  if (NV) {
#pragma unroll
    for (int k = 0; k < kKeep; ++k)
      if (tid + k * kStepThreads < vecs) store(k, tid + k * kStepThreads, f);
  } else {
    for (int i = tid; i < vecs; i += kStepThreads) {
      read(0, i);
      form(0);
      store(0, i, f);
    }
  }
}

int step_lanes(int N) {
  int n = 2;
  while (4 * n < N) n *= 2;
  return n;
}
// Rows per lane: as many as a head has, up to 8. (One sequence's 64 heads in
// 64 to 512 workgroups: 12.4 us and 13 to 14.)
int step_rows(int hd, int ln) {
  int r = 1;
  while (r < 8 && kStepThreads / ln * r < hd) r *= 2;
  return r;
}

// workgroups of a head
int step_parts(const StepArgs& a, int ln) {
  const int rows = kStepThreads / ln * step_rows(a.hd, ln);
  return (a.hd + rows - 1) / rows;
}

template <bool F16, int LN, int K>
hipError_t step_scan(const StepArgs& a, float* y, hipStream_t stream) {
  const int rp = step_rows(a.hd, LN), parts = step_parts(a, LN);
  const dim3 grid(static_cast<uint32_t>(static_cast<int64_t>(a.B) * a.nh * parts)), wg(kStepThreads);
#define FMX_STEP(RP) hipLaunchKernelGGL((step_kernel<F16, LN, RP, K>), grid, wg, 0, stream, a, parts, y)
  if (rp == 1) FMX_STEP(1);
  else if (rp == 2) FMX_STEP(2);
  else if (rp == 4) FMX_STEP(4);
  else FMX_STEP(8);
#undef FMX_STEP
  return hipGetLastError();
}
template <bool F16, int LN>
hipError_t step_scan(const StepArgs& a, float* y, hipStream_t stream) {
  return a.taps == 4 ? step_scan<F16, LN, 4>(a, y, stream) : step_scan<F16, LN, 0>(a, y, stream);
}

int64_t step_shifts(const StepArgs& a, int vec) {
  return static_cast<int64_t>(a.B) * ((a.C / vec + kStepThreads - 1) / kStepThreads);
}

template <bool F16, int VEC>
hipError_t step_norm(const StepArgs& a, float* y, hipStream_t stream) {
  const uint32_t norms = static_cast<uint32_t>(a.B * a.norm_groups);
  const dim3 grid(norms + static_cast<uint32_t>(step_shifts(a, VEC))), wg(kStepThreads);
  const int vecs = a.nh * a.hd / a.norm_groups / VEC;
  if (vecs <= kStepThreads)
    hipLaunchKernelGGL((step_norm_kernel<F16, VEC, 1>), grid, wg, 0, stream, a, norms, y);
  else if (vecs <= 4 * kStepThreads)
    hipLaunchKernelGGL((step_norm_kernel<F16, VEC, 4>), grid, wg, 0, stream, a, norms, y);
  else
    hipLaunchKernelGGL((step_norm_kernel<F16, VEC, 0>), grid, wg, 0, stream, a, norms, y);
  return hipGetLastError();
}

// vectors of 8 where every row starts on a word
bool step_wide(const StepArgs& a) {
  bool wide = a.C % 8 == 0 && a.nh * a.hd / a.norm_groups % 8 == 0 && on_words(a.norm_w);
  for (const HeadsView* v : {&a.xbc, &a.z, &a.out}) wide = wide && on_words(*v, 2);
  return wide;
}

template <bool F16>
hipError_t step(const StepArgs& a, float* y, hipStream_t stream) {
  hipError_t e;
  switch (step_lanes(a.N)) {
    case 2: e = step_scan<F16, 2>(a, y, stream); break;
    case 4: e = step_scan<F16, 4>(a, y, stream); break;
    case 8: e = step_scan<F16, 8>(a, y, stream); break;
    case 16: e = step_scan<F16, 16>(a, y, stream); break;
    case 32: e = step_scan<F16, 32>(a, y, stream); break;
    default: e = step_scan<F16, 64>(a, y, stream); break;
  }
  if (e != hipSuccess) return e;
  return step_wide(a) ? step_norm<F16, 8>(a, y, stream) : step_norm<F16, 1>(a, y, stream);
}

}  // namespace

size_t step_workspace(const StepArgs& a) { return static_cast<size_t>(a.B) * a.nh * a.hd * sizeof(float); }

bool step_fits(const StepArgs& a) {
  return static_cast<int64_t>(a.B) * a.nh * step_parts(a, step_lanes(a.N)) <= max_blocks(kStepThreads) &&
         static_cast<int64_t>(a.B) * a.norm_groups + step_shifts(a, step_wide(a) ? 8 : 1) <= max_blocks(kStepThreads);
}

hipError_t launch_step(const StepArgs& a, bool f16, void* ws, hipStream_t stream) {
  float* y = static_cast<float*>(ws);
  return f16 ? step<true>(a, y, stream) : step<false>(a, y, stream);
}

}  // namespace fmx
