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
#include <algorithm>

#include "fmx_cache_kernels.hpp"
#include "fmx_dev.hpp"

namespace fmx {

namespace {

constexpr int kSelThreads = 1024;
constexpr int kSelWaves = kSelThreads / kWave;
constexpr int kSelBins = 2048;
// copies of a long row's first histogram, lanes in turn: weights crowd in few
// digits, and a wave's additions to one address come one after the other
constexpr int kSelCopies = 8;
// positions whose images a thread keeps in registers (position tid + 1024 i)
constexpr int kSelKeep = 16;

// unsigned image of a weight: larger weight, larger image; -0 as 0, any NaN
// above infinity
__device__ inline uint32_t weight_key(float f) {
  const uint32_t u = __float_as_uint(f + 0.0f);
  if ((u & 0x7fffffffu) > 0x7f800000u) return 0xffffffffu;
  return u ^ (u >> 31 ? 0xffffffffu : 0x80000000u);
}

// inclusive scan over the workgroup's threads
__device__ inline uint32_t block_scan(uint32_t v, uint32_t* s_tmp) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  v = tree_to_last<64>(v, 0u, [](uint32_t a, uint32_t b) { return a + b; });  // (an inclusive scan)
  __syncthreads();
  if (lane == kWave - 1) s_tmp[wave] = v;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kSelWaves; ++w) v += w < wave ? s_tmp[w] : 0;
  return v;
}

struct SelShared {
  __attribute__((aligned(16))) uint32_t bin[kSelBins * kSelCopies];
  uint32_t tmp[kSelWaves];
  uint32_t digit, above;
  uint32_t cnt[kSelKeep * kSelWaves];
};

// One round: bins of the digit at `shift` of the images that agree with
// `found` above it, then the digit of the need-th largest, from the top.
template <int COPIES, typename F>
__device__ inline void select_round(SelShared& s, int shift, int bits, uint32_t& found, uint32_t& need,
                                    F&& each) {
  const int tid = threadIdx.x;
  u32x4_t* quads = reinterpret_cast<u32x4_t*>(s.bin);
#pragma unroll
  for (int i = 0; i < kSelBins * COPIES / 4; i += kSelThreads)
    if (i + tid < kSelBins * COPIES / 4) quads[i + tid] = u32x4_t{0, 0, 0, 0};
  __syncthreads();
  each([&](uint32_t u) {
    if (shift + bits == 32 || u >> (shift + bits) == found >> (shift + bits))
      atomicAdd(&s.bin[(u >> shift & ((1u << bits) - 1)) * COPIES + tid % COPIES], 1u);
  });
  __syncthreads();
  // from the largest digit down: thread t has digits top - 2 t, top - 2 t - 1
  const int top = (1 << bits) - 1;
  auto count = [&](int digit) {
    if (digit < 0) return 0u;
    uint32_t c = 0;
    if constexpr (COPIES == 1) {
      c = s.bin[digit];
    } else {
#pragma unroll
      for (int i = 0; i < COPIES / 4; ++i) {
        const u32x4_t x = quads[digit * (COPIES / 4) + i];
        c += x[0] + x[1] + x[2] + x[3];
      }
    }
    return c;
  };
  const uint32_t c0 = count(top - 2 * tid), c1 = count(top - 2 * tid - 1);
  const uint32_t end = block_scan(c0 + c1, s.tmp);
  const uint32_t start = end - c0 - c1;
  if (start < need && need <= end) {
    const bool first = need <= start + c0;
    s.digit = static_cast<uint32_t>(top - 2 * tid - (first ? 0 : 1));
    s.above = first ? start : start + c0;
  }
  __syncthreads();
  found |= s.digit << shift;
  need -= s.above;
  __syncthreads();
}

// A row of n > budget weights: the kept positions in order, and their weights.
// KEEP: so many positions per thread are kept in registers (n <= 1024 KEEP),
// 0: every round reads the weights again.
template <int KEEP, int COPIES>
__device__ void cut_row(const EvictArgs& a, SelShared& s, const float* w, float* wo, int32_t* kept, int n) {
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  // middle positions [lo, hi), `need` of them kept
  const int lo = static_cast<int>(a.sinks), hi = n - static_cast<int>(a.recent);
  uint32_t need = static_cast<uint32_t>(a.budget - a.sinks - a.recent);
  uint32_t found = 0;  // the need-th largest image, from its top digit down
  float v[KEEP ? KEEP : 1];
#pragma unroll
  for (int i = 0; i < KEEP; ++i) {
    const int p = tid + i * kSelThreads;
    v[i] = p < n ? w[p] : 0.0f;
  }
  if (need > 0) {
    auto all = [&](auto&& f) {
#pragma unroll
      for (int i = 0; i < KEEP; ++i) {
        const int p = tid + i * kSelThreads;
        if (p >= lo && p < hi) f(weight_key(v[i]));
      }
      if (KEEP == 0)
        for (int p = lo + tid; p < hi; p += kSelThreads) f(weight_key(w[p]));
    };
    select_round<COPIES>(s, 21, 11, found, need, all);
    // (few weights agree in the first digit: no crowds)
    select_round<1>(s, 10, 11, found, need, all);
    select_round<1>(s, 0, 10, found, need, all);
  } else {
    found = 0xffffffffu;  // nothing above it, none of its equals wanted
  }
  // In order: images above `found` and the first `need` equal to it go behind
  // those before them. In place a weight moves to a position <= its own, all
  // weights up to which have been read by then.
  const uint64_t below = lanes_below(lane);
  auto kinds = [&](int p, float x, bool* sure, bool* same) {
    const bool mid = p >= lo && p < hi;
    const uint32_t u = weight_key(x);
    *sure = p < n && (!mid || u > found);
    *same = mid && u == found;
  };
  auto put = [&](int p, float x, bool sure, bool same, uint32_t at, uint32_t eq) {
    // at, eq: sure and equal ones before p
    if (sure || (same && eq < need)) {
      const uint32_t pos = at + min(eq, need);
      kept[pos] = p;
      wo[pos] = x;
    }
  };
  if constexpr (KEEP > 0) {
    // counts of (1024 positions, wave), sure ones | equal ones << 16, scanned
    // in the positions' order
    static_assert(KEEP * kSelWaves <= kSelThreads && KEEP <= kSelKeep, "one thread per count, sums in 16 bits");
#pragma unroll
    for (int i = 0; i < KEEP; ++i) {
      bool sure, same;
      kinds(tid + i * kSelThreads, v[i], &sure, &same);
      const uint32_t c = static_cast<uint32_t>(__popcll(__ballot(sure)) | __popcll(__ballot(same)) << 16);
      if (lane == 0) s.cnt[i * kSelWaves + wave] = c;
    }
    __syncthreads();
    const uint32_t c = tid < KEEP * kSelWaves ? s.cnt[tid] : 0;
    const uint32_t before = block_scan(c, s.tmp) - c;
    if (tid < KEEP * kSelWaves) s.cnt[tid] = before;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < KEEP; ++i) {
      const int p = tid + i * kSelThreads;
      bool sure, same;
      kinds(p, v[i], &sure, &same);
      const uint64_t ms = __ballot(sure), me = __ballot(same);
      const uint32_t base = s.cnt[i * kSelWaves + wave];
      put(p, v[i], sure, same, (base & 0xffffu) + static_cast<uint32_t>(__popcll(ms & below)),
          (base >> 16) + static_cast<uint32_t>(__popcll(me & below)));
    }
  } else {
    uint32_t at = 0, eq = 0;  // of earlier positions
    for (int p0 = 0; p0 < n; p0 += kSelThreads) {
      const int p = p0 + tid;
      const float x = p < n ? w[p] : 0.0f;
      bool sure, same;
      kinds(p, x, &sure, &same);
      const uint64_t ms = __ballot(sure), me = __ballot(same);
      if (lane == 0) s.cnt[wave] = static_cast<uint32_t>(__popcll(ms) | __popcll(me) << 16);
      __syncthreads();
      uint32_t base = 0, sum = 0;
#pragma unroll
      for (int q = 0; q < kSelWaves; ++q) {
        base += q < wave ? s.cnt[q] : 0;
        sum += s.cnt[q];
      }
      put(p, x, sure, same, at + (base & 0xffffu) + static_cast<uint32_t>(__popcll(ms & below)),
          eq + (base >> 16) + static_cast<uint32_t>(__popcll(me & below)));
      at += sum & 0xffffu;
      eq += sum >> 16;
      __syncthreads();
    }
  }
}

// Bound by its chain of rounds: the weights are read once (up to 16384
// positions: kept in registers), a round is an LDS histogram and a scan. 64
// rows of up to 1152 weights 6.7 us, 64 rows of up to 16384 16 us (32 us with
// one copy of the histogram and every round reading them again).
__global__ __launch_bounds__(kSelThreads) void evict_select_kernel(EvictArgs a) {
  __shared__ SelShared s;
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
  if (n <= budget) {
    for (int i = tid; i < n; i += kSelThreads) kept[i] = i;
    for (int64_t i = wo != w ? tid : n + tid; i < a.S_out; i += kSelThreads) wo[i] = i < n ? w[i] : 0.0f;
    return;
  }
  if (n <= 2 * kSelThreads)
    cut_row<2, 1>(a, s, w, wo, kept, n);
  else if (n <= kSelKeep * kSelThreads)
    cut_row<kSelKeep, kSelCopies>(a, s, w, wo, kept, n);
  else
    cut_row<0, kSelCopies>(a, s, w, wo, kept, n);
  for (int64_t i = cnt + tid; i < a.S_out; i += kSelThreads) wo[i] = 0.0f;
}

// ------------------------------------------------------------------ keys and values

constexpr int kMoveThreads = 256;
constexpr int kMoveUnits = 4;  // of a thread, keys and values each: loads in flight

template <int VB>
struct Unit;
template <>
struct Unit<16> {
  typedef u32x4_t T;
};
template <>
struct Unit<2> {
  typedef uint16_t T;
};

// Bound by HBM: kept rows are read and written once, in kept order, so reads
// are runs of rows. 16 bytes per lane where rows and strides allow. 16
// sequences of 4 kv heads cut to 4000 rows of 128: 55 us for 250 MB, 4.5 TB/s
// (4.9 is a large copy's).
template <int VB>
__global__ __launch_bounds__(kMoveThreads) void evict_move_kernel(EvictArgs a, int chunks, int chunk_rows) {
  typedef typename Unit<VB>::T T;
  const int bg = blockIdx.x / chunks, chunk = blockIdx.x % chunks;
  const int b = bg / a.nkv, g = bg % a.nkv;
  const int64_t slot = seq_slot(a.slots, a.n_slots, b);
  const int32_t* kept = a.kept + static_cast<int64_t>(bg) * a.budget;
  const int per = static_cast<int>(a.row_bytes / VB);
  const int r0 = chunk * chunk_rows, r1 = min(static_cast<int>(a.budget), r0 + chunk_rows);
  if (slot >= 0) {
    const uint8_t* k = a.k + slot * a.k_bs + g * a.k_hs;
    const uint8_t* v = a.v + slot * a.v_bs + g * a.v_hs;
    uint8_t* ko = a.k_out + slot * a.ko_bs + g * a.ko_hs;
    uint8_t* vo = a.v_out + slot * a.vo_bs + g * a.vo_hs;
    const int units = (r1 - r0) * per;
    for (int u0 = threadIdx.x; u0 < units; u0 += kMoveThreads * kMoveUnits) {
      T kv[kMoveUnits], vv[kMoveUnits];
      int src[kMoveUnits], row[kMoveUnits], e[kMoveUnits];
#pragma unroll
      for (int i = 0; i < kMoveUnits; ++i) {
        const int u = u0 + i * kMoveThreads;
        row[i] = r0 + u / per;
        e[i] = u % per * VB;
        src[i] = u < units ? kept[row[i]] : -1;
      }
#pragma unroll
      for (int i = 0; i < kMoveUnits; ++i)
        if (src[i] >= 0) {
          kv[i] = *reinterpret_cast<const T*>(k + src[i] * a.k_ts + e[i]);
          vv[i] = *reinterpret_cast<const T*>(v + src[i] * a.v_ts + e[i]);
        }
#pragma unroll
      for (int i = 0; i < kMoveUnits; ++i)
        if (src[i] >= 0) {
          *reinterpret_cast<T*>(ko + row[i] * a.ko_ts + e[i]) = kv[i];
          *reinterpret_cast<T*>(vo + row[i] * a.vo_ts + e[i]) = vv[i];
        }
    }
  }
  if (chunk == 0 && g == 0 && threadIdx.x == 0) {
    const int64_t len = slot < 0 ? 0 : a.lens[b];
    const int64_t n = len < 0 ? 0 : (len > a.S ? a.S : len);
    a.lens_out[b] = static_cast<int32_t>(n < a.budget ? n : a.budget);
  }
}

// One workgroup per (sequence, kv head, keys or values, slice of the row), a
// block of rows after the other. Row i comes from row kept[i] >= i, so what a
// block reads lies behind all that earlier blocks wrote, and what it writes is
// read by no later block: only a block's own reads have to end before its
// writes begin. Bound by that chain of blocks, so rows are sliced until 512
// workgroups run: 79 us for 16 sequences of up to 16384 cut to
// 4000 positions, the selection included; one of 16384 cut to 8192, 57 us, 32
// workgroups for what a copy moves in 7.
template <int VB>
__global__ __launch_bounds__(kMoveThreads) void evict_shift_kernel(EvictArgs a, int slices, int slice_units) {
  typedef typename Unit<VB>::T T;
  constexpr int kUnits = 8;
  int item = blockIdx.x;
  const int slice = item % slices;
  item /= slices;
  const bool isv = item & 1;
  const int bg = item >> 1, b = bg / a.nkv, g = bg % a.nkv;
  const int64_t slot = seq_slot(a.slots, a.n_slots, b);
  const int32_t* kept = a.kept + static_cast<int64_t>(bg) * a.budget;
  if (slot >= 0) {
    uint8_t* base = (isv ? a.v_out + slot * a.v_bs + g * a.v_hs : a.k_out + slot * a.k_bs + g * a.k_hs) +
                    static_cast<int64_t>(slice) * slice_units * VB;
    const int64_t ts = isv ? a.v_ts : a.k_ts;
    const int per = min(slice_units, static_cast<int>(a.row_bytes / VB) - slice * slice_units);
    // lanes beyond the whole rows of a block idle
    const int rows = kMoveThreads / per, r = threadIdx.x / per, e = threadIdx.x % per * VB;
    const int budget = static_cast<int>(a.budget);
    for (int r0 = 0; r0 < budget; r0 += rows * kUnits) {
      if (kept[r0] < 0) break;
      T x[kUnits];
      int src[kUnits];
#pragma unroll
      for (int i = 0; i < kUnits; ++i) {
        const int row = r0 + i * rows + r;
        src[i] = r < rows && row < budget ? kept[row] : -1;
        if (src[i] == row) src[i] = -1;
      }
#pragma unroll
      for (int i = 0; i < kUnits; ++i) {
        x[i] = T{};
        if (src[i] >= 0) x[i] = *reinterpret_cast<const T*>(base + src[i] * ts + e);
      }
#pragma unroll
      for (int i = 0; i < kUnits; ++i) asm volatile("" : "+v"(x[i]));  // in registers, not on their way
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
      __syncthreads();
#pragma unroll
      for (int i = 0; i < kUnits; ++i)
        if (src[i] >= 0) *reinterpret_cast<T*>(base + (r0 + i * rows + r) * ts + e) = x[i];
    }
  }
  if (slice == 0 && !isv && g == 0 && threadIdx.x == 0) {
    // as many as are kept (lens may be lens_out, but nothing else reads it here)
    const int64_t len = slot < 0 ? 0 : a.lens[b];
    const int64_t n = len < 0 ? 0 : (len > a.S ? a.S : len);
    a.lens_out[b] = static_cast<int32_t>(n < a.budget ? n : a.budget);
  }
}

// the second launch
struct MoveGrid {
  int vb;             // bytes of a unit
  int slices, units;  // in place: slices of a row, units of a slice
  int64_t chunks;     // else: chunks of `rows` kept positions per (sequence, kv head)
  int rows;
  int64_t blocks;
};

MoveGrid move_grid(const EvictArgs& a) {
  int64_t all = a.row_bytes;
  for (int64_t s : {a.k_bs, a.k_ts, a.k_hs, a.v_bs, a.v_ts, a.v_hs,
                    a.ko_bs, a.ko_ts, a.ko_hs, a.vo_bs, a.vo_ts, a.vo_hs})
    all |= s;
  for (const void* p : {static_cast<const void*>(a.k), static_cast<const void*>(a.v),
                        static_cast<const void*>(a.k_out), static_cast<const void*>(a.v_out)})
    all |= static_cast<int64_t>(reinterpret_cast<uintptr_t>(p) & 15);
  MoveGrid m{};
  m.vb = all % 16 == 0 ? 16 : 2;
  const int64_t heads = static_cast<int64_t>(a.B) * a.nkv;
  const int per = static_cast<int>(a.row_bytes / m.vb);
  if (a.in_place) {
    // slices of a row, each at least 64 bytes, until 512 workgroups are busy
    int slices = 1;
    while (slices * 2 * 64 <= a.row_bytes && heads * 2 * slices < 512 && per % (slices * 2) == 0) slices *= 2;
    // (and no longer than a block of threads)
    while ((per + slices - 1) / slices > kMoveThreads) ++slices;
    m.units = (per + slices - 1) / slices;
    m.slices = (per + m.units - 1) / m.units;
    m.blocks = heads * 2 * m.slices;
  } else {
    // rows of a workgroup: about two rounds of its threads
    m.rows = std::max(1, 2 * kMoveThreads * kMoveUnits / per);
    m.chunks = (std::min(a.budget, a.S) + m.rows - 1) / m.rows;
    m.blocks = m.chunks * heads;
  }
  return m;
}

template <int VB>
hipError_t move_rows(const EvictArgs& a, const MoveGrid& m, hipStream_t stream) {
  const dim3 gr(static_cast<uint32_t>(m.blocks)), wg(kMoveThreads);
  if (a.in_place)
    hipLaunchKernelGGL(evict_shift_kernel<VB>, gr, wg, 0, stream, a, m.slices, m.units);
  else
    hipLaunchKernelGGL(evict_move_kernel<VB>, gr, wg, 0, stream, a, static_cast<int>(m.chunks), m.rows);
  return hipGetLastError();
}

}  // namespace

bool evict_fits(const EvictArgs& a) {
  return static_cast<int64_t>(a.B) * a.nkv <= max_blocks(kSelThreads) && move_grid(a).blocks <= max_blocks(kMoveThreads);
}

hipError_t launch_evict(const EvictArgs& a, hipStream_t stream) {
  const uint32_t heads = static_cast<uint32_t>(a.B) * static_cast<uint32_t>(a.nkv);
  hipLaunchKernelGGL(evict_select_kernel, dim3(heads), dim3(kSelThreads), 0, stream, a);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return e;
  const MoveGrid m = move_grid(a);
  return m.vb == 16 ? move_rows<16>(a, m, stream) : move_rows<2>(a, m, stream);
}

}  // namespace fmx
