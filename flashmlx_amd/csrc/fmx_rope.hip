// fmx_rope.hip -- rotary positions of any layout, and with them the caches'
// append (mx::fast::rope, server/src/model.cpp:875-876, and the cache update
// of :877-878).
//
// For a token at position p, pair i of its rotated heads turns by p f_i:
//   (a, b) -> m (a cos - b sin, a sin + b cos)
// The angle is formed in fp64 and reduced to a turn in [-1/2, 1/2] there (p
// f_i / 2 pi minus its nearest integer: 2^-53 of the angle, about 2^-32 turns
// at p = 2^21), its cosine and sine in fp32, the products in fp32, rounded
// once.
//
// Bound by HBM: every element is read and written once. A workgroup takes
// the rows of one or a few tokens (or a part of one token's), its loads are
// issued first, then its threads form the tokens' cosines and sines once for
// all heads in LDS while the loads are in flight; only as much LDS as those
// take (16 KB for every workgroup: 18.1 us for the 15.5 below). 4099 tokens of
// 32 heads of 128, half of each turned, fp16: 15.5 us alone for 67 MB, 4.3
// TB/s, and 14.1 a call among others, 4.8 (4.9 is a large copy's); 2 x 777
// tokens of 16 heads in fp32: 7.6 us for 25 MB. Eight decoded tokens take 4.6
// us, a launch and one chain of loads, fp64 products and stores.
#include <algorithm>

#include "fmx_cache_kernels.hpp"

namespace fmx {

namespace {

constexpr int kRotThreads = 256;
constexpr int kRotUnits = 2;       // units of a thread: pairs of vectors in flight
constexpr int kRotTable = 2048;    // (cos, sin) of a workgroup at most: 16 KB of LDS
constexpr double kInv2Pi = 0.15915494309189533577;

template <int ES, bool F16>
struct Elem;
template <bool F16>
struct Elem<2, F16> {
  typedef uint16_t T;
  static __device__ inline float ld(T v) { return Act<F16>::ld(v); }
  static __device__ inline T st(float f) { return Act<F16>::st(f); }
};
template <bool F16>
struct Elem<4, F16> {
  typedef float T;
  static __device__ inline float ld(T v) { return v; }
  static __device__ inline T st(float f) { return f; }
};

template <typename T, int N>
struct alignas(sizeof(T) * N) Vec {
  T e[N];
};

// the tokens of a workgroup and its part of a token's units
struct RotPlan {
  int tokens;      // per workgroup
  int parts;       // workgroups per token (tokens == 1)
  int units_rot;   // units of a rotated head: turned ones first, then copied ones
  int units_turn;
  int units_copy;  // of a v head
  int units;       // of a token
  int first;       // the launch's first token
};

// VEC elements per load; a turned unit is a pair of vectors (half layout), a
// vector of VEC / 2 pairs (interleaved), or one pair (VEC == 1)
template <int ES, bool F16, int VEC, bool INTER>
__global__ __launch_bounds__(kRotThreads) void rotate_kernel(RotateArgs a, RotPlan pl) {
  typedef Elem<ES, F16> E;
  typedef typename E::T T;
  typedef Vec<T, VEC> V;
  extern __shared__ float2 s_cs[];  // (cos, sin) of the tokens' pairs
  const int tid = threadIdx.x;
  const int half = a.dims / 2;
  const int rows = a.B * a.L;
  const int t0 = pl.first + static_cast<int>(blockIdx.x / pl.parts) * pl.tokens;
  const int part = static_cast<int>(blockIdx.x % pl.parts);
  const int nt = min(pl.tokens, rows - t0);

  const T* src[kRotUnits];
  T* dst[kRotUnits];
  int ib[kRotUnits];     // second vector of a turned unit (half layout, single pairs), else -1
  int cs[kRotUnits];     // its first cosine, or -1: copied
  V x0[kRotUnits], x1[kRotUnits];
#pragma unroll
  for (int u = 0; u < kRotUnits; ++u) {
    src[u] = nullptr;
    cs[u] = -1;
    ib[u] = -1;
    dst[u] = nullptr;
    int i = tid + u * kRotThreads + part * (kRotThreads * kRotUnits);
    const int tt = i / pl.units;
    if (pl.parts == 1 ? tt >= nt : i >= pl.units) continue;
    i -= tt * pl.units;
    const int t = t0 + tt;
    const int b = t / a.L, l = t - b * a.L;
    const int rot = (a.nh + a.nkv) * pl.units_rot;
    int h, e;  // head (q, k, v in a row) and the unit's first element
    if (i < rot) {
      h = i / pl.units_rot;
      const int w = i - h * pl.units_rot;
      if (w < pl.units_turn) {
        if (VEC == 1 || INTER) {
          const int pair = VEC == 1 ? w : w * (VEC / 2);
          e = INTER ? 2 * pair : pair;
          if (VEC == 1) ib[u] = INTER ? 1 : half;
          cs[u] = tt * half + pair;
        } else {
          e = w * VEC;
          ib[u] = half;
          cs[u] = tt * half + e;
        }
      } else {
        e = a.dims + (w - pl.units_turn) * VEC;
      }
    } else {
      h = a.nh + a.nkv + (i - rot) / pl.units_copy;
      e = (i - rot) % pl.units_copy * VEC;
    }
    const HeadsView* in = &a.q;
    const HeadsView* out = &a.q_out;
    int64_t ob = b, ol = l;
    if (h >= a.nh) {  // a cache row
      const bool isv = h >= a.nh + a.nkv;
      h -= isv ? a.nh + a.nkv : a.nh;
      in = isv ? &a.v : &a.k;
      out = isv ? &a.vc : &a.kc;
      ob = seq_slot(a.slots, a.n_slots, b);
      ol = static_cast<int64_t>(a.offs[b]) + l;
      if (ob < 0 || ol < 0 || ol >= a.max_seq) continue;
    }
    src[u] = static_cast<const T*>(in->p) + b * in->bs + l * in->ts + h * in->hs + e;
    dst[u] = static_cast<T*>(out->p) + ob * out->bs + ol * out->ts + h * out->hs + e;
    x0[u] = *reinterpret_cast<const V*>(src[u]);
    if (ib[u] >= 0) x1[u] = *reinterpret_cast<const V*>(src[u] + ib[u]);
  }

  for (int i = tid; i < nt * half; i += kRotThreads) {
    const int tt = i / half;
    const double turns = static_cast<double>(a.pos[t0 + tt]) * (a.freqs[i - tt * half] * kInv2Pi);
    const float r = static_cast<float>(2.0 * (turns - rint(turns)));
    float s, c;
    sincospif(r, &s, &c);
    s_cs[i] = make_float2(c * a.factor, (a.inverse ? -s : s) * a.factor);
  }
  __syncthreads();

#pragma unroll
  for (int u = 0; u < kRotUnits; ++u) {
    if (!src[u]) continue;
    if (cs[u] >= 0) {
      if (INTER && VEC > 1) {
#pragma unroll
        for (int j = 0; j < VEC / 2; ++j) {
          const float2 t = s_cs[cs[u] + j];
          const float p = E::ld(x0[u].e[2 * j]), q = E::ld(x0[u].e[2 * j + 1]);
          x0[u].e[2 * j] = E::st(p * t.x - q * t.y);
          x0[u].e[2 * j + 1] = E::st(p * t.y + q * t.x);
        }
      } else {
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
          const float2 t = s_cs[cs[u] + j];
          const float p = E::ld(x0[u].e[j]), q = E::ld(x1[u].e[j]);
          x0[u].e[j] = E::st(p * t.x - q * t.y);
          x1[u].e[j] = E::st(p * t.y + q * t.x);
        }
        *reinterpret_cast<V*>(dst[u] + ib[u]) = x1[u];
      }
    }
    *reinterpret_cast<V*>(dst[u]) = x0[u];
  }
}

template <int ES, bool F16, int VEC>
hipError_t rotate(const RotateArgs& a, hipStream_t stream) {
  RotPlan pl{};
  const int half = a.dims / 2;
  pl.units_turn = VEC == 1 ? half : a.interleaved ? a.dims / VEC : half / VEC;
  pl.units_rot = pl.units_turn + (a.hd - a.dims) / VEC;
  pl.units_copy = a.hd / VEC;
  const int64_t units = static_cast<int64_t>(a.nh + a.nkv) * pl.units_rot + static_cast<int64_t>(a.nkv) * pl.units_copy;
  if (units > (1 << 30)) return hipErrorInvalidValue;
  pl.units = static_cast<int>(units);
  constexpr int kPer = kRotThreads * kRotUnits;
  const int64_t rows = static_cast<int64_t>(a.B) * a.L;
  pl.parts = (pl.units + kPer - 1) / kPer;
  pl.tokens = pl.parts > 1 ? 1 : std::max(1, std::min(kPer / pl.units, kRotTable / half));
  const dim3 wg(kRotThreads);
  const size_t lds = static_cast<size_t>(pl.tokens) * half * sizeof(float2);
  const int64_t per = max_blocks(kRotThreads) / pl.parts * pl.tokens;  // tokens of a launch
  for (int64_t first = 0; first < rows; first += per) {
    pl.first = static_cast<int>(first);
    const int64_t grid = (std::min(per, rows - first) + pl.tokens - 1) / pl.tokens * pl.parts;
    const dim3 gr(static_cast<uint32_t>(grid));
    if (a.interleaved)
      hipLaunchKernelGGL((rotate_kernel<ES, F16, VEC, true>), gr, wg, lds, stream, a, pl);
    else
      hipLaunchKernelGGL((rotate_kernel<ES, F16, VEC, false>), gr, wg, lds, stream, a, pl);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
  }
  return hipSuccess;
}

bool vec_view(const HeadsView& v, int es, int vec) {
  return !v.p || (reinterpret_cast<uintptr_t>(v.p) % (es * vec) == 0 && v.bs % vec == 0 && v.ts % vec == 0 &&
                  v.hs % vec == 0);
}

}  // namespace

hipError_t launch_rotate(const RotateArgs& a, int es, bool f16, hipStream_t stream) {
  // 16-byte vectors where every row's start, the halves and the copied rest
  // fall on them, single elements otherwise
  const int vec = 16 / es;
  bool wide = a.hd % vec == 0 && a.dims % vec == 0 && (a.interleaved || (a.dims / 2) % vec == 0);
  for (const HeadsView* v : {&a.q, &a.k, &a.v, &a.q_out, &a.kc, &a.vc}) wide = wide && vec_view(*v, es, vec);
  if (es == 4) return wide ? rotate<4, false, 4>(a, stream) : rotate<4, false, 1>(a, stream);
  if (f16) return wide ? rotate<2, true, 8>(a, stream) : rotate<2, true, 1>(a, stream);
  return wide ? rotate<2, false, 8>(a, stream) : rotate<2, false, 1>(a, stream);
}

}  // namespace fmx
