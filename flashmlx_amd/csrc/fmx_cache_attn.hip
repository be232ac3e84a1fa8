// fmx_cache_attn.hip -- attention of a batch over a shared prefix and its
// sequences' own caches, and over own caches with the keys' weights added up
// (no counterpart in the reference; mx::fast::scaled_dot_product_attention,
// server/src/model.cpp:879-882, at their place).
//
// One workgroup per (query row, head): keys in tiles of 256, a thread per
// key's score, the running maximum and sum of the softmax in fp32, a thread
// per dimension for the values. The weights: a thread per key of a (sequence,
// kv head), over the rows that see it, from the rows' ln sum exp.
#include "fmx_cache_kernels.hpp"

namespace fmx {

namespace {

constexpr int kRowThreads = 256;

template <bool F16>
__device__ inline float dot8(const float* q, const uint16_t* k, int hd) {
  float s = 0.0f;
  for (int c = 0; c < hd; c += 8) {
    const u32x4_t w = *reinterpret_cast<const u32x4_t*>(k + c);
#pragma unroll
    for (int m = 0; m < 4; ++m) {
      s = __builtin_fmaf(q[c + 2 * m], Act<F16>::lo(w[m]), s);
      s = __builtin_fmaf(q[c + 2 * m + 1], Act<F16>::hi(w[m]), s);
    }
  }
  return s;
}

__device__ inline float block_reduce(float v, bool is_max, float* s_red) {
  for (int o = 32; o >= 1; o >>= 1) {
    const float w = __shfl_xor(v, o);
    v = is_max ? fmaxf(v, w) : v + w;
  }
  __syncthreads();
  if ((threadIdx.x & 63) == 0) s_red[threadIdx.x >> 6] = v;
  __syncthreads();
  v = s_red[0];
  for (int w = 1; w < kRowThreads / kWave; ++w) v = is_max ? fmaxf(v, s_red[w]) : v + s_red[w];
  return v;
}

template <bool F16>
__global__ __launch_bounds__(kRowThreads) void attn_rows_kernel(CacheAttnArgs a, float* lse) {
  __shared__ float s_q[kCacheMaxHd], s_p[kRowThreads], s_red[kRowThreads / kWave];
  const int tid = threadIdx.x;
  const int t = blockIdx.x, h = blockIdx.y, b = t / a.L, l = t - b * a.L, g = h / a.rep;
  const uint16_t* q = static_cast<const uint16_t*>(a.q.p) + b * a.q.bs + l * a.q.ts + h * a.q.hs;
  if (tid < a.hd) s_q[tid] = Act<F16>::ld(q[tid]);
  const int64_t slot = a.S > 0 ? seq_slot(a.slots, a.n_slots, b) : -1;
  const int64_t own = a.S > 0 ? own_keys(a, slot, a.offs[b], l) : 0;
  float m = -__builtin_huge_valf(), z = 0.0f, o = 0.0f;
  for (int part = 0; part < 2; ++part) {
    const int64_t n = part ? own : a.P;
    if (n == 0) continue;
    const HeadsView& kv = part ? a.kc : a.kp;
    const HeadsView& vv = part ? a.vc : a.vp;
    const uint16_t* kb = static_cast<const uint16_t*>(kv.p) + (part ? slot * kv.bs : 0) + g * kv.hs;
    const uint16_t* vb = static_cast<const uint16_t*>(vv.p) + (part ? slot * vv.bs : 0) + g * vv.hs;
    for (int64_t j0 = 0; j0 < n; j0 += kRowThreads) {
      __syncthreads();
      const int64_t j = j0 + tid;
      const float s = j < n ? dot8<F16>(s_q, kb + j * kv.ts, a.hd) * a.scale : -__builtin_huge_valf();
      const float mt = fmaxf(m, block_reduce(s, true, s_red));
      const float mu = mt == -__builtin_huge_valf() ? 0.0f : mt;
      const float p = j < n ? expf(s - mu) : 0.0f;
      s_p[tid] = p;
      const float f = expf(m - mu);
      z = z * f + block_reduce(p, false, s_red);
      o *= f;
      m = mt;
      const int c = static_cast<int>(n - j0 < kRowThreads ? n - j0 : kRowThreads);
      if (tid < a.hd)
        for (int i = 0; i < c; ++i) o = __builtin_fmaf(s_p[i], Act<F16>::ld(vb[(j0 + i) * vv.ts + tid]), o);
    }
  }
  uint16_t* out = static_cast<uint16_t*>(a.out.p) + b * a.out.bs + l * a.out.ts + h * a.out.hs;
  if (tid < a.hd) out[tid] = Act<F16>::st(z == 0.0f ? 0.0f : o / z);
  if (tid == 0 && lse) lse[static_cast<int64_t>(t) * a.nh + h] = z == 0.0f ? -__builtin_huge_valf() : m + logf(z);
}

template <bool F16>
__global__ __launch_bounds__(kRowThreads) void attn_weights_kernel(CacheAttnArgs a, const float* lse) {
  __shared__ float s_q[kCacheMaxHd];
  const int tid = threadIdx.x;
  const int b = blockIdx.y / a.nkv, g = blockIdx.y % a.nkv;
  const int64_t slot = seq_slot(a.slots, a.n_slots, b);
  if (slot < 0) return;
  const int64_t j = static_cast<int64_t>(blockIdx.x) * kRowThreads + tid;
  const uint16_t* kb = static_cast<const uint16_t*>(a.kc.p) + slot * a.kc.bs + g * a.kc.hs;
  const int off = a.offs[b];
  float sum = 0.0f;
  for (int l = 0; l < a.L; ++l) {
    const int64_t n = own_keys(a, slot, off, l);
    for (int r = 0; r < a.rep; ++r) {
      const int h = g * a.rep + r;
      const uint16_t* q = static_cast<const uint16_t*>(a.q.p) + b * a.q.bs + l * a.q.ts + h * a.q.hs;
      __syncthreads();
      if (tid < a.hd) s_q[tid] = Act<F16>::ld(q[tid]);
      __syncthreads();
      if (j < n)
        sum += expf(dot8<F16>(s_q, kb + j * a.kc.ts, a.hd) * a.scale -
                    lse[(static_cast<int64_t>(b) * a.L + l) * a.nh + h]);
    }
  }
  if (j < a.S) {
    const int64_t w = (slot * a.nkv + g) * a.S + j;
    a.w_out[w] = (a.w_in ? a.w_in[w] : 0.0f) + sum;
  }
}

}  // namespace

size_t cache_attn_workspace(const CacheAttnArgs& a) {
  return a.w_out ? static_cast<size_t>(align_up(static_cast<int64_t>(a.B) * a.L * a.nh * 4, 256)) : 0;
}

hipError_t launch_cache_attn(const CacheAttnArgs& a, bool f16, void* ws, hipStream_t stream) {
  float* lse = a.w_out ? static_cast<float*>(ws) : a.lse;
  const dim3 grid(static_cast<uint32_t>(a.B * a.L), static_cast<uint32_t>(a.nh));
  if (f16)
    hipLaunchKernelGGL(attn_rows_kernel<true>, grid, dim3(kRowThreads), 0, stream, a, lse);
  else
    hipLaunchKernelGGL(attn_rows_kernel<false>, grid, dim3(kRowThreads), 0, stream, a, lse);
  if (a.w_out) {
    const dim3 wg(static_cast<uint32_t>((a.S + kRowThreads - 1) / kRowThreads), static_cast<uint32_t>(a.B * a.nkv));
    if (f16)
      hipLaunchKernelGGL(attn_weights_kernel<true>, wg, dim3(kRowThreads), 0, stream, a, lse);
    else
      hipLaunchKernelGGL(attn_weights_kernel<false>, wg, dim3(kRowThreads), 0, stream, a, lse);
  }
  return hipGetLastError();
}

}  // namespace fmx
