// fmx_ssm_conv.hip -- the short causal convolution of the state space layer
// (the mixer's conv1d, server/src/nemotron_h.cpp):
//   out[t] = act(bias + sum over k of w[k] x[t - taps + 1 + k])  per channel
//
// Bound by HBM: every element is read and written once (8191 tokens of 6144
// channels in fp32 79 us, 5.1 TB/s, a copy's rate; 2048 in bf16 15 us, 3.3 TB/s,
// one round of workgroups that wait for their loads). A thread takes one
// vector of channels over a run of tokens, whose taps - 1 rows before it it
// reads again (from the caches); neighbouring threads take neighbouring
// channels. In fp32 a run's loads are all in flight at once; 16-bit rows are
// unpacked in the branch that loads them, which waits for each before the next.
// The thread of a sequence's first run also keeps the state, so that
// state_out may be state_in: nobody else reads it.
#include "fmx_ssm_kernels.hpp"

namespace fmx {

namespace {

constexpr int kConvThreads = 256;
// Tokens of a run: at least taps - 1, so that only a sequence's first run
// reaches into the state. 8, or 4 where 8 make fewer threads than kConvFew: 7
// ragged sequences of up to 777 tokens of 1792 channels take 12.7 us in a graph
// for 15.0, 2048 of 6144 17.8 for 17.0, 8191 of 6144 in fp32 87.5 for 81.4 (16
// tokens: 18.6, 20.8, 83.3).
constexpr int kConvRun = 8, kConvShort = 4;
static_assert(kConvRun >= kMaxTaps - 1, "a run's rows before it are one run's");
constexpr int64_t kConvFew = 160 * 1024;

template <int DT, int VEC, int K, int R>
__global__ __launch_bounds__(kConvThreads) void conv_kernel(ConvArgs a, uint32_t per_seq, uint32_t total) {
  typedef typename El<DT>::T T;
  typedef Pack<T, VEC> V;
  const uint32_t id = blockIdx.x * kConvThreads + threadIdx.x;
  if (id >= total) return;
  const uint32_t cvs = static_cast<uint32_t>(a.C) / VEC;
  const int b = static_cast<int>(id / per_seq);
  const uint32_t rest = id - b * per_seq;
  const int t0 = static_cast<int>(rest / cvs) * R;
  const int ch = static_cast<int>(rest % cvs) * VEC;
  const int len = seq_length(a.lens, a.L, b);
  if (t0 >= len && t0 > 0) return;
  const int64_t slot = K > 1 ? seq_slot(a.slots, a.n_slots, b) : -1;
  const T* x = static_cast<const T*>(a.x.p) + b * a.x.bs + ch;
  T* out = static_cast<T*>(a.out.p) + b * a.out.bs + ch;
  const int64_t state0 = slot * (K - 1) * a.C + ch;
  const T* s_in = slot >= 0 && a.s_in ? static_cast<const T*>(a.s_in) + state0 : nullptr;
  V zero{};

  V rows[R + K - 1];
#pragma unroll
  for (int i = 0; i < R + K - 1; ++i) {
    const int t = t0 - (K - 1) + i;
    rows[i] = zero;
    if (t < 0) {
      if (s_in) rows[i] = *reinterpret_cast<const V*>(s_in + static_cast<int64_t>(i) * a.C);
    } else if (t < len) {
      rows[i] = *reinterpret_cast<const V*>(x + t * a.x.ts);
    }
  }
  V w[K], bias = zero;  // [channel][tap], in a row
#pragma unroll
  for (int k = 0; k < K; ++k)
    w[k] = *reinterpret_cast<const V*>(static_cast<const T*>(a.w) + static_cast<int64_t>(ch) * K + k * VEC);
  if (a.bias) bias = *reinterpret_cast<const V*>(static_cast<const T*>(a.bias) + ch);

#pragma unroll
  for (int r = 0; r < R; ++r) {
    if (t0 + r >= len) break;
    V y;
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
      float acc = El<DT>::ld(bias.e[e]);
#pragma unroll
      for (int k = 0; k < K; ++k)
        acc = __builtin_fmaf(El<DT>::ld(w[(e * K + k) / VEC].e[(e * K + k) % VEC]), El<DT>::ld(rows[r + k].e[e]), acc);
      y.e[e] = El<DT>::st(a.silu ? silu_f32(acc) : acc);
    }
    *reinterpret_cast<V*>(out + (t0 + r) * a.out.ts) = y;
  }

  if (K > 1 && t0 == 0 && slot >= 0 && a.s_out) {
    T* s_out = static_cast<T*>(a.s_out) + state0;
    // rows of the old state move to lower places only: in order, none is lost
    for (int j = 0; j < K - 1; ++j) {
      const int t = len - (K - 1) + j;
      V v = zero;
      if (t >= 0)
        v = *reinterpret_cast<const V*>(x + t * a.x.ts);
      else if (s_in)
        v = *reinterpret_cast<const V*>(s_in + static_cast<int64_t>(t + K - 1) * a.C);
      *reinterpret_cast<V*>(s_out + static_cast<int64_t>(j) * a.C) = v;
    }
  }
}

int64_t conv_threads(const ConvArgs& a, int vec, int run) {
  const int64_t runs = std::max<int64_t>(1, (static_cast<int64_t>(a.L) + run - 1) / run);
  return a.B * runs * (a.C / vec);
}

template <int DT, int VEC, int R>
hipError_t conv(const ConvArgs& a, hipStream_t stream) {
  const int64_t total = conv_threads(a, VEC, R);
  if (total == 0) return hipSuccess;
  const dim3 grid(static_cast<uint32_t>((total + kConvThreads - 1) / kConvThreads)), wg(kConvThreads);
  const uint32_t per_seq = static_cast<uint32_t>(total / a.B), n = static_cast<uint32_t>(total);
#define FMX_CONV(K) hipLaunchKernelGGL((conv_kernel<DT, VEC, K, R>), grid, wg, 0, stream, a, per_seq, n)
  switch (a.taps) {
    case 1: FMX_CONV(1); break;
    case 2: FMX_CONV(2); break;
    case 3: FMX_CONV(3); break;
    case 4: FMX_CONV(4); break;
    case 5: FMX_CONV(5); break;
    default:
      if constexpr (R == kConvRun) {
        if (a.taps == 6) FMX_CONV(6);
        if (a.taps == 7) FMX_CONV(7);
        if (a.taps == 8) FMX_CONV(8);
        break;
      }
      return hipErrorInvalidValue;
  }
#undef FMX_CONV
  return hipGetLastError();
}

int conv_run(const ConvArgs& a, int vec) {
  return a.taps - 1 <= kConvShort && conv_threads(a, vec, kConvRun) < kConvFew ? kConvShort : kConvRun;
}

template <int DT, int VEC>
hipError_t conv(const ConvArgs& a, hipStream_t stream) {
  return conv_run(a, VEC) == kConvShort ? conv<DT, VEC, kConvShort>(a, stream) : conv<DT, VEC, kConvRun>(a, stream);
}

// 16 bytes at once where every row starts on a word (9 sequences of 2127 rows
// of 1248 channels, 4440 bytes apart, 33 us, by elements 36), single elements
// otherwise
bool conv_wide(const ConvArgs& a, int dt) {
  const int es = dt == kElF32 ? 4 : 2, vec = 16 / es;
  bool wide = a.C % vec == 0 && on_words(a.x, es) && on_words(a.out, es);
  for (const void* p : {a.w, a.bias, a.s_in, static_cast<const void*>(a.s_out)})
    wide = wide && on_words(p);
  return wide;
}

}  // namespace

bool conv_fits(const ConvArgs& a, int dt) {
  const int vec = conv_wide(a, dt) ? (dt == kElF32 ? 4 : 8) : 1;
  return conv_threads(a, vec, conv_run(a, vec)) <= max_blocks(kConvThreads) * kConvThreads;
}

hipError_t launch_conv(const ConvArgs& a, int dt, hipStream_t stream) {
  const bool wide = conv_wide(a, dt);
  if (dt == kElF32) return wide ? conv<kElF32, 4>(a, stream) : conv<kElF32, 1>(a, stream);
  if (dt == kElF16) return wide ? conv<kElF16, 8>(a, stream) : conv<kElF16, 1>(a, stream);
  return wide ? conv<kElBf16, 8>(a, stream) : conv<kElBf16, 1>(a, stream);
}

}  // namespace fmx
