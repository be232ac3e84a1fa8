// fmx_ssm_scan.hip -- the selective scan of the state space layer (the
// mixer's ssm_kernel, server/src/nemotron_h.cpp:608-653), per sequence and head:
//   S[p, n] = exp(dt a) S[p, n] + dt x[p] b[n];  out[p] = sum_n c[n] S[p, n] + d x[p]
//
// scan_few_kernel walks the tokens one by one with the state in registers.
#include <algorithm>

#include "fmx_ssm_kernels.hpp"

namespace fmx {

namespace {

constexpr int kFewThreads = 256;
constexpr int kFewTokens = 8;  // staged together

// A workgroup takes 256 / LN * RP rows of a head's state.
template <bool F16, int LN, int RP>
__global__ __launch_bounds__(kFewThreads) void scan_few_kernel(ScanArgs a, int parts) {
  constexpr int kRows = kFewThreads / LN * RP;
  constexpr int kCols = 4 * LN;
  __shared__ float s_x[kFewTokens][kRows];
  __shared__ f32x4_t s_b[kFewTokens][LN];
  __shared__ f32x4_t s_c[kFewTokens][LN];
  __shared__ float s_dt[kFewTokens], s_decay[kFewTokens];
  const int tid = threadIdx.x, col = tid % LN, sub = tid / LN;
  uint32_t id = blockIdx.x;
  const int row0 = static_cast<int>(id % parts) * kRows;
  id /= parts;
  const int h = static_cast<int>(id % a.nh), b = static_cast<int>(id / a.nh);
  const int g = h / a.rep;
  const int len = seq_length(a.lens, a.L, b);
  const int64_t slot = seq_slot(a.slots, a.n_slots, b);
  const int rows = min(kRows, a.hd - row0);
  const uint16_t* x = static_cast<const uint16_t*>(a.x.p) + b * a.x.bs + h * a.x.hs + row0;
  const uint16_t* bp = static_cast<const uint16_t*>(a.b.p) + b * a.b.bs + g * a.b.hs;
  const uint16_t* cp = static_cast<const uint16_t*>(a.c.p) + b * a.c.bs + g * a.c.hs;
  const uint16_t* dtp = static_cast<const uint16_t*>(a.dt.p) + b * a.dt.bs + h * a.dt.hs;
  uint16_t* out = static_cast<uint16_t*>(a.out.p) + b * a.out.bs + h * a.out.hs + row0;
  const int64_t state0 = ((slot * a.nh + h) * a.hd + row0) * a.N + 4 * col;

  StateRows<LN, RP> st;
#pragma unroll
  for (int i = 0; i < RP; ++i) {
    const int r = sub + i * (kFewThreads / LN);
    st.s[i] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
    if (a.s_in && slot >= 0 && r < rows && 4 * col < a.N)
      st.s[i] = *reinterpret_cast<const f32x4_t*>(a.s_in + state0 + static_cast<int64_t>(r) * a.N);
  }
  const float rate = a.a[h], skip = a.d ? a.d[h] : 0.0f;

  for (int t0 = 0; t0 < len; t0 += kFewTokens) {
    const int nt = min(kFewTokens, len - t0);
    for (int i = tid; i < nt * kRows; i += kFewThreads) {
      const int t = i / kRows, r = i % kRows;
      s_x[t][r] = r < rows ? Act<F16>::ld(x[(t0 + t) * a.x.ts + r]) : 0.0f;
    }
    for (int i = tid; i < nt * kCols; i += kFewThreads) {
      const int t = i / kCols, n = i % kCols;
      const bool in = n < a.N;
      reinterpret_cast<float*>(s_b[t])[n] = in ? Act<F16>::ld(bp[(t0 + t) * a.b.ts + n]) : 0.0f;
      reinterpret_cast<float*>(s_c[t])[n] = in ? Act<F16>::ld(cp[(t0 + t) * a.c.ts + n]) : 0.0f;
    }
    if (tid < nt) {
      const float dt = time_step(Act<F16>::ld(dtp[(t0 + tid) * a.dt.ts]), a.dt_bias, h, a.softplus, a.dt_min, a.dt_max);
      s_dt[tid] = dt;
      s_decay[tid] = expf(dt * rate);
    }
    __syncthreads();
    for (int t = 0; t < nt; ++t) {
      float u[RP], xs[RP], y[RP];
#pragma unroll
      for (int i = 0; i < RP; ++i) {
        xs[i] = s_x[t][sub + i * (kFewThreads / LN)];
        u[i] = s_dt[t] * xs[i];
      }
      st.step(s_decay[t], u, s_b[t][col], s_c[t][col], y);
      if (col == LN - 1) {
#pragma unroll
        for (int i = 0; i < RP; ++i) {
          const int r = sub + i * (kFewThreads / LN);
          if (r < rows) out[(t0 + t) * a.out.ts + r] = Act<F16>::st(a.d ? y[i] + skip * xs[i] : y[i]);
        }
      }
    }
    __syncthreads();
  }
  if (a.s_out && slot >= 0 && 4 * col < a.N) {
#pragma unroll
    for (int i = 0; i < RP; ++i) {
      const int r = sub + i * (kFewThreads / LN);
      if (r < rows) *reinterpret_cast<f32x4_t*>(a.s_out + state0 + static_cast<int64_t>(r) * a.N) = st.s[i];
    }
  }
}

// lanes of a state row: whole vectors of 4 columns
int state_lanes(int N) {
  int n = 2;
  while (4 * n < N) n *= 2;
  return n;
}
// rows per lane: as many as a head has, up to 8
int state_rows(int hd, int ln) {
  int r = 1;
  while (r < 8 && kFewThreads / ln * r < hd) r *= 2;
  return r;
}

template <bool F16, int LN>
hipError_t scan_few(const ScanArgs& a, hipStream_t stream) {
  const int rp = state_rows(a.hd, LN), rows = kFewThreads / LN * rp;
  const int parts = (a.hd + rows - 1) / rows;
  const dim3 grid(static_cast<uint32_t>(static_cast<int64_t>(a.B) * a.nh * parts)), wg(kFewThreads);
#define FMX_FEW(RP) hipLaunchKernelGGL((scan_few_kernel<F16, LN, RP>), grid, wg, 0, stream, a, parts)
  if (rp == 1) FMX_FEW(1);
  else if (rp == 2) FMX_FEW(2);
  else if (rp == 4) FMX_FEW(4);
  else FMX_FEW(8);
#undef FMX_FEW
  return hipGetLastError();
}

template <bool F16>
hipError_t scan_few(const ScanArgs& a, hipStream_t stream) {
  switch (state_lanes(a.N)) {
    case 2: return scan_few<F16, 2>(a, stream);
    case 4: return scan_few<F16, 4>(a, stream);
    case 8: return scan_few<F16, 8>(a, stream);
    case 16: return scan_few<F16, 16>(a, stream);
    case 32: return scan_few<F16, 32>(a, stream);
    default: return scan_few<F16, 64>(a, stream);
  }
}

}  // namespace

size_t scan_workspace(const ScanArgs&) { return 0; }

bool scan_fits(const ScanArgs& a) {
  // (a part has at least 4 rows)
  return static_cast<int64_t>(a.B) * a.nh * ((a.hd + 3) / 4) <= max_blocks(kFewThreads);
}

hipError_t launch_scan(const ScanArgs& a, bool f16, void*, hipStream_t stream) {
  if (a.B == 0) return hipSuccess;
  return f16 ? scan_few<true>(a, stream) : scan_few<false>(a, stream);
}

}  // namespace fmx
