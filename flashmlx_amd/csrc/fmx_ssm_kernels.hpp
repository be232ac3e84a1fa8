// fmx_ssm_kernels.hpp -- argument blocks, launchers and shared device code of
// the state space layer's operators (fmx_ssm_conv.hip, fmx_ssm_scan.hip,
// fmx_ssm_step.hip, fmx_ssm_norm.hip; library-internal).
#pragma once

#include "fmx_cache_kernels.hpp"
#include "fmx_dev.hpp"

namespace fmx {

enum { kElBf16 = 0, kElF16 = 1, kElF32 = 2 };

// an element type's loads and stores
template <int DT>
struct El {
  typedef uint16_t T;
  static __device__ inline float ld(T v) { return Act<DT == kElF16>::ld(v); }
  static __device__ inline T st(float f) { return Act<DT == kElF16>::st(f); }
};
template <>
struct El<kElF32> {
  typedef float T;
  static __device__ inline float ld(T v) { return v; }
  static __device__ inline T st(float f) { return f; }
};

// N elements that one instruction moves: on whole words, which is all that the
// memory instructions of up to four words ask for
template <typename T, int N>
struct alignas(sizeof(T) * N < 4 ? sizeof(T) * N : 4) Pack {
  T e[N];
};

// v sigmoid(v), the argument of the exponential rounded once, hardware
// exponential and reciprocal: off by (|v| + 4) 2^-23 of itself at most where v is
// negative, by 4 2^-23 elsewhere; 0 from about -87 down, where the reciprocal is
// no normal number
__device__ inline float silu_f32(float v) {
  return v * __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(-v * 1.4426950408889634f));
}

// whether an array, or a view's rows, of elements of es bytes start on words
inline bool on_words(const void* p) { return reinterpret_cast<uintptr_t>(p) % 4 == 0; }
inline bool on_words(const HeadsView& v, int es) {
  return !v.p || (on_words(v.p) && v.bs * es % 4 == 0 && v.ts * es % 4 == 0);
}

__device__ inline int seq_length(const int32_t* lens, int L, int b) {
  return lens ? min(max(lens[b], 0), L) : L;
}

// ------------------------------------------------------------------ convolution

constexpr int kMaxTaps = 8;

struct ConvArgs {
  int B, L, C, taps, silu;
  HeadsView x, out;
  const void* w;
  const void* bias;
  const void* s_in;
  void* s_out;
  int64_t n_slots;
  const int32_t* lens;
  const int32_t* slots;
};
// (of all of these: whether the launches that a call makes are within max_blocks)
bool conv_fits(const ConvArgs& a, int dt);
hipError_t launch_conv(const ConvArgs& a, int dt, hipStream_t stream);

// ------------------------------------------------------------------ scan

constexpr int kScanMaxDim = 256;  // of a head, and of its state

struct ScanArgs {
  int B, L, nh, hd, groups, N, rep;
  HeadsView x, dt, b, c, out;
  const float* a;
  const float* d;
  const float* dt_bias;
  int softplus;
  float dt_min, dt_max;
  const float* s_in;
  float* s_out;
  int64_t n_slots;
  const int32_t* lens;
  const int32_t* slots;
};
size_t scan_workspace(const ScanArgs& a);
bool scan_fits(const ScanArgs& a);
hipError_t launch_scan(const ScanArgs& a, bool f16, void* ws, hipStream_t stream);

// ln(1 + e^-t), t >= 0, to 8 steps of 2^-24: e = e^-t with the product's rest,
// ln(1 + e) = 2 atanh(e / (2 + e)) by its series, whose argument is at most 1/3
// (the ninth term 2^-29)
__device__ inline float log1p_exp_minus(float t) {
  t = fminf(t, 126.0f);
  const float p = t * -1.44269504f, rest = __builtin_fmaf(t, -1.44269504f, -p) + t * -1.925963e-8f;
  float e = __builtin_amdgcn_exp2f(p);
  e = __builtin_fmaf(e, rest * 0.6931472f, e);
  const float d = 2.0f + e;
  float r = __builtin_amdgcn_rcpf(d);
  r = __builtin_fmaf(__builtin_fmaf(-d, r, 1.0f), r, r);
  const float s = e * r, q = s * s;
  float f = 1.0f / 15;
#pragma unroll
  for (int k = 13; k > 0; k -= 2) f = __builtin_fmaf(f, q, 1.0f / k);
  return 2.0f * s * f;
}

// the time step: ln(1 + e^v) = max(v, 0) + ln(1 + e^-|v|), which loses nothing
// where e^v is small; comparisons that leave a NaN one
__device__ inline float time_step(float raw, const float* bias, int h, int softplus, float lo, float hi) {
  float v = bias ? raw + bias[h] : raw;
  if (softplus) v = (v > 0.0f ? v : v == v ? 0.0f : v) + log1p_exp_minus(fabsf(v));
  return v < lo ? lo : v > hi ? hi : v;
}

// ------------------------------------------------------------------ one token

struct StepArgs {
  int B, nh, hd, groups, N, rep, taps, silu, C;
  HeadsView xbc, dt, z, out;
  const void* conv_w;
  const void* conv_b;
  const float* a;
  const float* d;
  const float* dt_bias;
  int softplus;
  float dt_min, dt_max;
  const void* norm_w;
  int norm_groups;
  float eps;
  int gate_first;
  void* conv_state;
  float* state;
  int64_t n_slots;
  const int32_t* slots;
};
size_t step_workspace(const StepArgs& a);
bool step_fits(const StepArgs& a);
hipError_t launch_step(const StepArgs& a, bool f16, void* ws, hipStream_t stream);

// ------------------------------------------------------------------ norm

struct GatedNormArgs {
  int B, L, C, groups;
  float eps;
  int gate_first;
  HeadsView x, z, out;
  const void* w;
  const int32_t* lens;
};
bool gated_norm_fits(const GatedNormArgs& a, int dt);
hipError_t launch_gated_norm(const GatedNormArgs& a, int dt, hipStream_t stream);

// ------------------------------------------------------------------ a state's rows

// Rows of a head's state in registers: lane j of LN neighbouring ones holds
// columns 4 j .. 4 j + 3 of RP rows. One token:
//   s = decay s + u b;  y = sum over the columns of c s, in the lanes' last one
template <int LN, int RP>
struct StateRows {
  f32x4_t s[RP];

  __device__ inline void step(float decay, const float* u, f32x4_t b, f32x4_t c, float* y) {
#pragma unroll
    for (int i = 0; i < RP; ++i) {
      s[i] = s[i] * decay + u[i] * b;
      const f32x4_t p = s[i] * c;
      y[i] = tree_to_last<LN>((p[0] + p[1]) + (p[2] + p[3]), 0.0f, [](float a, float b) { return a + b; });
    }
  }
};

}  // namespace fmx
