// fmx_evict.hip -- eviction of cached keys by accumulated attention weight
// (no counterpart in the reference).
//
//   evict_select_kernel  one workgroup per (sequence, kv head): the
//                        (budget - sinks - recent)-th largest weight of the
//                        middle positions by three rounds of digits (11, 11
//                        and 10 bits of an order-preserving image of the
//                        float), each a histogram in LDS; then the kept
//                        positions in order, and the weights moved
//   evict_move_kernel    the kept keys and values, into another cache
//   evict_shift_kernel   the same within one cache
#include "fmx_cache_kernels.hpp"

namespace fmx {

namespace {

constexpr int kSelThreads = 1024;
constexpr int kSelWaves = kSelThreads / kWave;
constexpr int kSelBins = 2048;

// unsigned image of a weight: larger weight, larger image; -0 as 0, any NaN
// above infinity
__device__ inline uint32_t weight_key(float f) {
  const uint32_t u = __float_as_uint(f + 0.0f);
  if ((u & 0x7fffffffu) > 0x7f800000u) return 0xffffffffu;
  return u ^ (u >> 31 ? 0xffffffffu : 0x80000000u);
}

// inclusive scan over the workgroup's threads
__device__ inline uint64_t block_scan(uint64_t v, uint64_t* s_tmp) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
  for (int d = 1; d < kWave; d <<= 1) {
    const uint64_t o = __shfl_up(v, d);
    if (lane >= d) v += o;
  }
  __syncthreads();
  if (lane == kWave - 1) s_tmp[wave] = v;
  __syncthreads();
  for (int w = 0; w < wave; ++w) v += s_tmp[w];
  return v;
}

__global__ __launch_bounds__(kSelThreads) void evict_select_kernel(EvictArgs a) {
  __shared__ uint32_t s_bin[kSelBins];
  __shared__ uint64_t s_tmp[kSelWaves];
  __shared__ uint32_t s_digit, s_above;
  const int tid = threadIdx.x;
  const int b = blockIdx.x / a.nkv, g = blockIdx.x % a.nkv;
  int32_t* kept = a.kept + static_cast<int64_t>(blockIdx.x) * a.budget;
  const int64_t slot = seq_slot(a.slots, a.n_slots, b);
  const int64_t len = slot < 0 ? 0 : a.lens[b];
  const int n = static_cast<int>(len < 0 ? 0 : (len > a.S ? a.S : len));
  const int budget = static_cast<int>(a.budget);
  const int cnt = min(n, budget);
  for (int i = cnt + tid; i < budget; i += kSelThreads) kept[i] = -1;
  if (slot < 0) return;
  const float* w = a.w + (slot * a.nkv + g) * a.S;
  float* wo = a.w_out + (slot * a.nkv + g) * a.S_out;
  const bool move_w = wo != w;
  if (n <= budget) {
    for (int i = tid; i < n; i += kSelThreads) kept[i] = i;
    for (int64_t i = move_w ? tid : n + tid; i < a.S_out; i += kSelThreads) wo[i] = i < n ? w[i] : 0.0f;
    return;
  }
  // middle positions [lo, hi), `need` of them kept
  const int lo = static_cast<int>(a.sinks), hi = n - static_cast<int>(a.recent);
  uint32_t need = static_cast<uint32_t>(budget - a.sinks - a.recent);
  uint32_t found = 0;  // digits of the need-th largest image, from the top
  int shift = 32;
  for (int round = 0; round < 3 && need > 0; ++round) {
    const int bits = round < 2 ? 11 : 10;
    shift -= bits;
    for (int i = tid; i < kSelBins; i += kSelThreads) s_bin[i] = 0;
    __syncthreads();
    for (int i = lo + tid; i < hi; i += kSelThreads) {
      const uint32_t u = weight_key(w[i]);
      if (round == 0 || u >> (shift + bits) == found >> (shift + bits))
        atomicAdd(&s_bin[u >> shift & ((1u << bits) - 1)], 1u);
    }
    __syncthreads();
    // from the largest digit down: thread t has digits top - 2 t, top - 2 t - 1
    const int top = (1 << bits) - 1;
    const uint32_t c0 = 2 * tid <= top ? s_bin[top - 2 * tid] : 0;
    const uint32_t c1 = 2 * tid + 1 <= top ? s_bin[top - 2 * tid - 1] : 0;
    const uint32_t end = static_cast<uint32_t>(block_scan(c0 + c1, s_tmp));
    const uint32_t start = end - c0 - c1;
    if (start < need && need <= end) {
      const bool first = need <= start + c0;
      s_digit = static_cast<uint32_t>(top - 2 * tid - (first ? 0 : 1));
      s_above = first ? start : start + c0;
    }
    __syncthreads();
    found |= s_digit << shift;
    need -= s_above;
    __syncthreads();
  }
  // kept: images above `found`, and the first `need` equal to it. Thread t
  // has a run of positions; counts of both kinds are scanned together.
  const bool some = budget > a.sinks + a.recent;
  const int run = (n + kSelThreads - 1) / kSelThreads;
  const int i0 = min(tid * run, n), i1 = min(i0 + run, n);
  uint64_t mine = 0;  // sure ones | equal ones << 32
  for (int i = i0; i < i1; ++i) {
    if (i < lo || i >= hi) {
      ++mine;
    } else if (some) {
      const uint32_t u = weight_key(w[i]);
      mine += (u > found ? 1ull : 0ull) + (u == found ? 1ull << 32 : 0ull);
    }
  }
  const uint64_t before = block_scan(mine, s_tmp) - mine;
  uint32_t eq = static_cast<uint32_t>(before >> 32);
  uint32_t at = static_cast<uint32_t>(before) + min(eq, need);
  for (int i = i0; i < i1; ++i) {
    bool keep = i < lo || i >= hi;
    if (!keep && some) {
      const uint32_t u = weight_key(w[i]);
      keep = u > found;
      if (u == found) keep = eq++ < need;
    }
    if (keep) kept[at++] = i;
  }
  __threadfence_block();
  __syncthreads();
  // the weights in order: position i comes from kept[i] >= i, so a tile's
  // reads are behind every earlier tile's writes
  for (int64_t i0w = 0; i0w < a.S_out; i0w += kSelThreads) {
    const int64_t i = i0w + tid;
    const float v = i < cnt ? w[kept[i]] : 0.0f;
    __syncthreads();
    if (i < a.S_out) wo[i] = v;
  }
}

__global__ __launch_bounds__(256) void evict_move_kernel(EvictArgs a) {
  const int b = blockIdx.y / a.nkv, g = blockIdx.y % a.nkv;
  const int64_t slot = seq_slot(a.slots, a.n_slots, b);
  const int32_t* kept = a.kept + static_cast<int64_t>(blockIdx.y) * a.budget;
  const int64_t per = a.row_bytes / 2, total = a.budget * per;
  for (int64_t i = blockIdx.x * 256ll + threadIdx.x; i < total && slot >= 0; i += gridDim.x * 256ll) {
    const int64_t row = i / per, e = i % per;
    const int32_t s = kept[row];
    if (s < 0) break;
    const int64_t ko = slot * a.ko_bs + g * a.ko_hs + row * a.ko_ts, ki = slot * a.k_bs + g * a.k_hs + s * a.k_ts;
    const int64_t vo = slot * a.vo_bs + g * a.vo_hs + row * a.vo_ts, vi = slot * a.v_bs + g * a.v_hs + s * a.v_ts;
    reinterpret_cast<uint16_t*>(a.k_out + ko)[e] = reinterpret_cast<const uint16_t*>(a.k + ki)[e];
    reinterpret_cast<uint16_t*>(a.v_out + vo)[e] = reinterpret_cast<const uint16_t*>(a.v + vi)[e];
  }
  if (blockIdx.x == 0 && g == 0 && threadIdx.x == 0) {
    int n = 0;
    if (slot >= 0) {
      int lo = 0, hi = static_cast<int>(a.budget);  // kept's entries from here on are -1
      while (lo < hi) {
        const int mid = (lo + hi) / 2;
        if (kept[mid] >= 0) lo = mid + 1; else hi = mid;
      }
      n = lo;
    }
    a.lens_out[b] = n;
  }
}

// One workgroup per (sequence, kv head, keys or values), rows in order: row i
// comes from row kept[i] >= i, so what a step reads lies behind all that
// earlier steps wrote, and what it writes is read by no later step.
__global__ __launch_bounds__(256) void evict_shift_kernel(EvictArgs a) {
  const int b = blockIdx.y / a.nkv, g = blockIdx.y % a.nkv;
  const int64_t slot = seq_slot(a.slots, a.n_slots, b);
  const int32_t* kept = a.kept + static_cast<int64_t>(blockIdx.y) * a.budget;
  const bool isv = blockIdx.x != 0;
  uint8_t* base = isv ? a.v_out + slot * a.v_bs + g * a.v_hs : a.k_out + slot * a.k_bs + g * a.k_hs;
  const int64_t ts = isv ? a.v_ts : a.k_ts;
  const int per = static_cast<int>(a.row_bytes / 2);
  int64_t n = 0;
  if (slot >= 0)
    for (int64_t row = 0; row < a.budget; ++row) {
      const int32_t s = kept[row];
      if (s < 0) break;
      ++n;
      if (s == row) continue;
      for (int e = threadIdx.x; e < per; e += 256)
        reinterpret_cast<uint16_t*>(base + row * ts)[e] = reinterpret_cast<const uint16_t*>(base + s * ts)[e];
    }
  if (!isv && g == 0 && threadIdx.x == 0) a.lens_out[b] = static_cast<int32_t>(n);
}

}  // namespace

hipError_t launch_evict(const EvictArgs& a, hipStream_t stream) {
  const uint32_t heads = static_cast<uint32_t>(a.B) * static_cast<uint32_t>(a.nkv);
  hipLaunchKernelGGL(evict_select_kernel, dim3(heads), dim3(kSelThreads), 0, stream, a);
  if (a.in_place) {
    hipLaunchKernelGGL(evict_shift_kernel, dim3(2, heads), dim3(256), 0, stream, a);
  } else {
    hipLaunchKernelGGL(evict_move_kernel, dim3(64, heads), dim3(256), 0, stream, a);
  }
  return hipGetLastError();
}

}  // namespace fmx
