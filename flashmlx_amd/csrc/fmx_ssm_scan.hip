// fmx_ssm_scan.hip -- the selective scan of the state space layer (the
// mixer's ssm_kernel, server/src/nemotron_h.cpp:608-653), per sequence and head:
//   S[p, n] = exp(dt a) S[p, n] + dt x[p] b[n];  out[p] = sum_n c[n] S[p, n] + d x[p]
//
// scan_few_kernel walks the tokens one by one with the state in registers: the
// state is read and written once, and that is its time while tokens are few (32
// sequences of 5 tokens, 32 heads of 128 rows and 64 columns: 18.7 us in a
// graph, 4.93 TB/s of a copy would be 14.2; each further token 0.75 us of
// staging, a chain of adds across lanes and a barrier).
//
// scan_chunk_kernel takes chunks of 64 tokens on the matrix cores. With f(s, t)
// the product of the decays of the tokens s + 1 .. t, the chunk's outputs are
//   out[t] = f(start, t) c[t] S + sum over s <= t of (c[t] . b[s]) f(s, t) dt[s] x[s]
// and its last state f(start, end) S + sum over s of f(s, end) dt[s] x[s] b[s],
// three products of matrices and one for the dots, which the heads of a group
// share. A wave has 16 rows of a head's state in accumulators, whose layout is
// an operand's as it is; only the weights of x cross waves, through LDS. fp32
// operands go in as sums of three numbers of bf16, all of their 24 bits; those
// of float16 that meet b and c as sums of two of float16, scaled, to 2^-23.
// (With weights, and bf16's state in outputs, in two bf16 numbers, 16 bits, 8192
// tokens took 116 us for 124, but where terms cancelled outputs were off by
// hundreds of what a walk of the same tokens is.) Long sequences are cut into
// segments: a first launch forms each segment's state from 0, a second starts
// each segment from the sum of those before it.
// 8192 tokens of 64 heads of 64 rows, 128 columns, 8 groups: 124 us (a walk of
// the tokens 7888).
// Measured and no faster, before the weights had a third part: four waves per
// SIMD with one buffer, 32 rows per wave without weights through LDS (157 us for
// 140 then), steps in a launch of their own, the SIMD's two waves in opposite
// phases (104 for 96), one item to a workgroup and two of those to a CU (142 in
// a graph for 134), groups of instructions interleaved by hand.
#include <algorithm>
#include <cstddef>

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

// workgroups of a head
int few_parts(const ScanArgs& a, int ln) {
  const int rows = kFewThreads / ln * state_rows(a.hd, ln);
  return (a.hd + rows - 1) / rows;
}

template <bool F16, int LN>
hipError_t scan_few(const ScanArgs& a, hipStream_t stream) {
  const int rp = state_rows(a.hd, LN), parts = few_parts(a, LN);
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

// ------------------------------------------------------------------ chunks on the matrix cores

constexpr int kChunk = 64;       // tokens
constexpr int kTileRows = 64;    // of a head, taken by four waves
constexpr int kSlotThreads = 256;

typedef short s16x4_t __attribute__((ext_vector_type(4)));
typedef short s16x8_t __attribute__((ext_vector_type(8)));

// 4 x 16 elements across 16 lanes: lane i gets element i % 4 of the lanes i / 4 + 4 e
__device__ inline s16x4_t read_tr(const uint8_t* p) {
  return __builtin_amdgcn_ds_read_tr16_b64_v4i16(
      (__attribute__((address_space(3))) s16x4_t*)const_cast<uint8_t*>(p));
}

__device__ inline f32x4_t mfma_bf16(s16x8_t a, s16x8_t b, f32x4_t c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, a), __builtin_bit_cast(bf16x8_t, b), c, 0, 0, 0);
}
__device__ inline f32x4_t mfma_f16(s16x8_t a, s16x8_t b, f32x4_t c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8_t, a), __builtin_bit_cast(f16x8_t, b), c, 0, 0, 0);
}
template <bool F16>
__device__ inline f32x4_t mfma_in(s16x8_t a, s16x8_t b, f32x4_t c) {
  return F16 ? mfma_f16(a, b, c) : mfma_bf16(a, b, c);
}

// Rows of CH 16-byte chunks in LDS, chunk c of row r at place c ^ swizzle(r):
// 16 lanes that read one chunk each of 16 rows, and 16 lanes that read four
// neighbouring halves each of four rows, meet in no bank.
template <int CH>
__device__ inline int swizzle(int row) {
  if (CH == 4) return row >> 2 & 3;
  if (CH == 8) return (row >> 1 & 1) << 2 | (row >> 2 & 3);
  return (row & 3) << 2 | (row >> 2 & 3);
}
template <int CH>
__device__ inline int chunk_at(int row, int c) {
  return (row * CH + (c ^ swizzle<CH>(row))) * 16;
}

// two floats as bf16, rounded, in one word
__device__ inline uint32_t pack_bf16(float a, float b) {
  typedef float f32x2_t __attribute__((ext_vector_type(2)));
  typedef __bf16 bf16x2_t __attribute__((ext_vector_type(2)));
  return __builtin_bit_cast(uint32_t, __builtin_convertvector(f32x2_t{a, b}, bf16x2_t));
}
__device__ inline float hi_bf16(uint32_t v) { return __uint_as_float(v & 0xffff0000u); }

template <bool F16>
__device__ inline uint32_t pack_in(float a, float b) {
  return F16 ? __builtin_bit_cast(uint32_t, f16x2_t{static_cast<_Float16>(a), static_cast<_Float16>(b)}) : pack_bf16(a, b);
}

// Values as a sum of PARTS numbers of bf16, in order: the first ones cut to 8
// bits (an AND, which is the float as well as what is packed; a conversion and
// its way back take 14 cycles a pair for 12), the last of two rounded. Three
// are exact, and so are two of a float16.
template <int PARTS>
__device__ inline void split_bf16(const float* v, s16x8_t* part) {
  float rest[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) rest[j] = v[j];
#pragma unroll
  for (int k = 0; k < PARTS; ++k) {
    u32x4_t w;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if (k + 1 == PARTS && PARTS < 3) {
        w[j] = pack_bf16(rest[2 * j], rest[2 * j + 1]);
      } else {
        const uint32_t lo = __float_as_uint(rest[2 * j]), hi = __float_as_uint(rest[2 * j + 1]);
        w[j] = __builtin_amdgcn_perm(hi, lo, 0x07060302u);
        if (k + 1 < PARTS) {
          rest[2 * j] -= __uint_as_float(lo & 0xffff0000u);
          rest[2 * j + 1] -= __uint_as_float(hi & 0xffff0000u);
        }
      }
    }
    part[k] = __builtin_bit_cast(s16x8_t, w);
  }
}
// as a sum of two of float16, each rounded: off by 2^-23 of the value or by
// 2^-25, whichever is more, of values within 2^15
__device__ inline void split_f16(const float* v, s16x8_t* part) {
  typedef float f32x2_t __attribute__((ext_vector_type(2)));
  u32x4_t h, l;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const f16x2_t a = __builtin_convertvector((f32x2_t{v[2 * j], v[2 * j + 1]}), f16x2_t);
    const f16x2_t b = __builtin_convertvector(
        (f32x2_t{v[2 * j] - static_cast<float>(a[0]), v[2 * j + 1] - static_cast<float>(a[1])}), f16x2_t);
    h[j] = __builtin_bit_cast(uint32_t, a);
    l[j] = __builtin_bit_cast(uint32_t, b);
  }
  part[0] = __builtin_bit_cast(s16x8_t, h);
  part[1] = __builtin_bit_cast(s16x8_t, l);
}

// The power of two that brings `most` to 2^13 .. 2^14 (0 and tiny values: 2^126
// at most), and its inverse
__device__ inline float scale_of(float most, float* inverse) {
  int k = 140 - static_cast<int>(__float_as_uint(most) >> 23);
  k = k > 126 ? 126 : k;
  *inverse = __uint_as_float(static_cast<uint32_t>(127 - k) << 23);
  return __uint_as_float(static_cast<uint32_t>(127 + k) << 23);
}

// The sequences cut into segments of whole chunks, each taken by workgroups of
// SLOTS (head, 64 rows) items of one group.
struct ChunkPlan {
  int tiles;        // 64-row tiles of a head
  int pairs;        // workgroups of a group
  int segs;         // segments of the longest sequence
  int seg_chunks;   // chunks of a segment
  int first_segs;   // segments of this launch
  int run;          // neighbouring workgroups on one XCD
  uint32_t total;   // workgroups with work
  int keep_first;   // state_in is copied (state_out is the same array)
};

// 16 bytes of each lane, at base + offset, to LDS, lane i's at byte `to` + 16 i;
// masked lanes' stay.
// (The builtin makes every later read of LDS wait for all loads in flight,
// also of the buffer that no load writes: here the wait is the caller's. The
// compiler sets m0 right before the instructions that it uses it for.)
__device__ inline void to_lds16(const void* base, uint32_t offset, uint32_t to) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"(to), "v"(offset), "s"(base)
               : "memory");
}
// a value that the compiler takes to be another one here, so that what is
// formed from it is formed again rather than kept through a loop
__device__ inline int afresh(int v) {
  asm volatile("" : "+v"(v));
  return v;
}
// keeps what is read from LDS above it above it
__device__ inline void read_first() { asm volatile("" ::: "memory"); }

// What a chunk's tokens need, per slot. Sums of log2 e dt a are formed in 64
// bits; from the chunk's start as two floats, whose differences are exact to
// 2^-24 of themselves however far the sums have run.
template <bool STATES>
struct ChunkSteps {
  float in[kChunk];         // dt times the decay from the token to the chunk's end
  float decay, pad[3];      // of the whole chunk
  float dt[kChunk];
  float sum[kChunk], rest[kChunk];
  float out[kChunk];        // the decay from the chunk's start to the token
  float near[kChunk];       // the decay from the token before its 16 to the token
  float far[16 + 32 + 48];  // dt times the decay from the token to the end of the 16 before 16 k: k = 1, 2, 3
};
template <>
struct ChunkSteps<true> {
  float in[kChunk];
  float decay, pad[3];
};
__device__ inline int far_at(int k) { return 8 * k * (k - 1); }

constexpr int kRound = 4;  // chunks whose steps are formed together, one by each wave of a slot
// Places for them: a round is formed in the middle of the one before it, of
// which the second half is still needed.
constexpr int kRing = kRound + kRound / 2;
constexpr int kWeightParts = 3;  // of bf16: all of the weights' 24 bits

template <int NK, int SLOTS, bool STATES>
struct ChunkLds {
  static constexpr int kRow = NK * 64;  // bytes of a token's b or c
  static constexpr int kBufs = NK > 4 && !STATES ? 1 : 2;
  __attribute__((aligned(16))) uint8_t b[kBufs][kChunk * kRow];
  __attribute__((aligned(16))) uint8_t x[kBufs][SLOTS][kChunk * kTileRows * 2];
  __attribute__((aligned(16))) uint8_t c[STATES ? 1 : kBufs][STATES ? 16 : kChunk * kRow];
  // weights of the tokens s for token t, in parts: rows t < 32 of 32 tokens,
  // the others of 64
  __attribute__((aligned(16))) uint8_t m[STATES ? 1 : SLOTS][STATES ? 1 : kWeightParts][STATES ? 16 : 32 * 64 + 32 * 128];
  ChunkSteps<STATES> steps[kRing][SLOTS];
};

__device__ inline int weight_at(int t, int chunk) {
  return t < 32 ? chunk_at<4>(t, chunk) : 32 * 64 + chunk_at<8>(t - 32, chunk);
}

// NK: 32-column steps of a state row. STATES: the first pass over segments,
// which forms their states alone.
template <bool F16, int NK, int SLOTS, bool STATES>
__global__ __launch_bounds__(kSlotThreads* SLOTS, 2) void scan_chunk_kernel(ScanArgs a, ChunkPlan pl, float* seg_states,
                                                                         float* seg_decays) {
  typedef ChunkLds<NK, SLOTS, STATES> Lds;
  constexpr int kThreads = kSlotThreads * SLOTS, kWaves = 4 * SLOTS;
  constexpr int kBufs = Lds::kBufs;
  constexpr int CH = NK * 4;
  constexpr int NT = 2 * NK;  // 16-column tiles of a state row
  __shared__ Lds lds;
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int slot = wave >> 2, w4 = wave & 3;
  const int i16 = lane & 15, g4 = lane >> 4;

  // ---- the item: neighbouring workgroups read one group's b and c, in one XCD's L2
  const uint32_t r = blockIdx.x / 8;
  uint32_t id = (r / pl.run * 8 + blockIdx.x % 8) * pl.run + r % pl.run;
  if (id >= pl.total) return;
  const int pair = static_cast<int>(id % pl.pairs);
  id /= pl.pairs;
  const int grp = static_cast<int>(id % a.groups);
  id /= a.groups;
  const int seg = static_cast<int>(id % pl.first_segs), b = static_cast<int>(id / pl.first_segs);
  const int len = seq_length(a.lens, a.L, b);
  const int seg_len = pl.seg_chunks * kChunk;
  const int t_first = seg * seg_len;
  if (STATES ? t_first + seg_len >= len : seg > 0 && t_first >= len) return;
  const int t_end = min(len, t_first + seg_len);
  const int chunks = (t_end - t_first + kChunk - 1) / kChunk;
  const int items = a.rep * pl.tiles;
  const int n_slots = min(SLOTS, items - pair * SLOTS);
  const int item = min(pair * SLOTS + slot, items - 1);
  const bool live = slot < n_slots;
  const int h = grp * a.rep + item / pl.tiles, row0 = item % pl.tiles * kTileRows;
  const int64_t pool = seq_slot(a.slots, a.n_slots, b);

  // ---- a chunk's rows straight to LDS, each wave a few KB of each (a wave's
  // loads of an array are kStep rows apart; their columns differ by what that
  // changes in the swizzle)
  constexpr int kBi = NK * 4 > kWaves ? NK * 4 / kWaves : 1;
  constexpr int kStep = kWaves * 64 / CH;
  static_assert(kBi == 1 || kStep % 8 == 0, "rows of a wave's loads");
  const int b_row = (wave * 64 + lane) / CH, b_col = (lane % CH ^ swizzle<CH>(b_row)) * 8;
  const int x_row = w4 * 16 + lane / 8, x_col = (lane % 8 ^ swizzle<8>(x_row)) * 8;
  const uint16_t* bp = static_cast<const uint16_t*>(a.b.p) + b * a.b.bs + grp * a.b.hs;
  const uint16_t* cp = STATES ? nullptr : static_cast<const uint16_t*>(a.c.p) + b * a.c.bs + grp * a.c.hs;
  const uint16_t* xp = static_cast<const uint16_t*>(a.x.p) + b * a.x.bs + h * a.x.hs + row0;
  uint16_t* op = STATES ? nullptr : static_cast<uint16_t*>(a.out.p) + b * a.out.bs + h * a.out.hs + row0;
  const uint32_t lds_at = static_cast<uint32_t>(reinterpret_cast<uintptr_t>((__attribute__((address_space(3))) Lds*)&lds));
  bp += t_first * a.b.ts;
  if (!STATES) cp += t_first * a.c.ts;
  xp += t_first * a.x.ts;
  if (!STATES) op += t_first * a.out.ts;
  const uint32_t b_off = static_cast<uint32_t>(b_row * static_cast<int>(a.b.ts)) * 2;
  const uint32_t c_off = STATES ? 0 : static_cast<uint32_t>(b_row * static_cast<int>(a.c.ts)) * 2;
  const uint32_t x_off = static_cast<uint32_t>(x_row * static_cast<int>(a.x.ts)) * 2;
  // (pointers go on by a chunk with each load)
  auto load_rows = [&](const uint16_t* from, uint32_t off, int64_t ts, int t0, uint32_t to, auto whole) {  // of b or c
#pragma unroll
    for (int k = 0; k < kBi; ++k) {
      const int col = b_col ^ (k * kStep / 4 % 4 * 8);
      if ((NK * 4 >= kWaves || wave < NK * 4) && (whole() || (t0 + b_row + k * kStep < t_end && col < a.N)))
        to_lds16(from + k * kStep * ts, off + col * 2, to + (wave + k * kWaves) * 1024);
    }
  };
  auto load_all = [&](int t0, int buf, auto whole) {
    load_rows(bp, b_off, a.b.ts, t0, lds_at + offsetof(Lds, b) + buf * sizeof(lds.b[0]), whole);
    if (!STATES) load_rows(cp, c_off, a.c.ts, t0, lds_at + offsetof(Lds, c) + buf * sizeof(lds.c[0]), whole);
    if (!live) return;
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const int col = x_col ^ (k * 16);
      if (whole() || (t0 + x_row + k * 8 < t_end && row0 + col < a.hd))
        to_lds16(xp + k * 8 * a.x.ts, x_off + col * 2,
                 lds_at + offsetof(Lds, x) + (buf * SLOTS + slot) * sizeof(lds.x[0][0]) + (w4 * 2 + k) * 1024);
    }
  };
  const bool wide = a.N == 32 * NK && a.hd % kTileRows == 0;
  auto load = [&](int t0, int buf) {
    if (wide && t0 + kChunk <= t_end)
      load_all(t0, buf, [] { return true; });  // (no lane masked: 40 instructions fewer)
    else
      load_all(t0, buf, [] { return false; });
    bp += kChunk * a.b.ts;
    if (!STATES) cp += kChunk * a.c.ts;
    xp += kChunk * a.x.ts;
  };

  // ---- the tokens' steps
  const float rate = a.a[h], bias = a.dt_bias ? a.dt_bias[h] : 0.0f;
  const float skip = !STATES && a.d ? a.d[h] : 0.0f;
  const uint16_t* dtp = static_cast<const uint16_t*>(a.dt.p) + b * a.dt.bs + h * a.dt.hs;
  uint16_t vdt = 0;
  auto load_dt = [&](int ck) {
    const int t = t_first + ck * kChunk + lane;
    vdt = t < t_end ? dtp[t * a.dt.ts] : 0;
  };
  auto steps = [&](int ck) {
    const bool in = t_first + ck * kChunk + lane < t_end;
    const float dt = in ? time_step(Act<F16>::ld(vdt) + bias, nullptr, 0, a.softplus, a.dt_min, a.dt_max) : 0.0f;
    const double own = in ? static_cast<double>(dt) * static_cast<double>(rate) * 1.4426950408889634074 : 0.0;
    const double sum = tree_to_last<64>(own, 0.0, [](double x, double y) { return x + y; });  // (an inclusive scan)
    const double all = readlane_f64(sum, 63);
    auto power = [](double e) { return __builtin_amdgcn_exp2f(static_cast<float>(e)); };
    ChunkSteps<STATES>& s = lds.steps[ck % kRing][slot];
    s.in[lane] = in ? dt * power(all - sum) : 0.0f;
    if (lane == 0) s.decay = power(all);
    if constexpr (!STATES) {
      const double at[3] = {readlane_f64(sum, 15), readlane_f64(sum, 31), readlane_f64(sum, 47)};
      const float lead = static_cast<float>(sum);
      s.dt[lane] = dt;
      s.sum[lane] = lead;
      s.rest[lane] = static_cast<float>(sum - static_cast<double>(lead));
      s.out[lane] = __builtin_amdgcn_exp2f(lead);
      s.near[lane] = power(lane < 16 ? sum : sum - at[max(g4, 1) - 1]);
#pragma unroll
      for (int k = 1; k < 4; ++k)
        if (lane < 16 * k) s.far[far_at(k) + lane] = dt * power(at[k - 1] - sum);
    }
  };
  if (live && w4 < chunks) load_dt(w4);
  const u32x4_t zero{0, 0, 0, 0};
  // What no load writes is 0, or of earlier tokens of the sequence: finite, or
  // of a row that is NaN by now.
  if (t_end - t_first < kBufs * kChunk || a.N < 32 * NK || a.hd % kTileRows != 0) {
    for (int i = tid; i < static_cast<int>(sizeof(lds.b) / 16); i += kThreads) reinterpret_cast<u32x4_t*>(lds.b)[i] = zero;
    for (int i = tid; i < static_cast<int>(sizeof(lds.x) / 16); i += kThreads) reinterpret_cast<u32x4_t*>(lds.x)[i] = zero;
    if (!STATES)
      for (int i = tid; i < static_cast<int>(sizeof(lds.c) / 16); i += kThreads) reinterpret_cast<u32x4_t*>(lds.c)[i] = zero;
  }
  if (!STATES) {  // tokens behind t in a step that t's own are in
    for (int v = tid; v < SLOTS * kWeightParts * 16 * 2; v += kThreads) {
      const int c = v % 2, t = v / 2 % 16, part = v / 32 % kWeightParts, q = v / 32 / kWeightParts;
      *reinterpret_cast<u32x4_t*>(lds.m[q][part] + weight_at(t, 2 + c)) = zero;
      *reinterpret_cast<u32x4_t*>(lds.m[q][part] + weight_at(32 + t, 6 + c)) = zero;
    }
  }
  lds_barrier();
  asm volatile("" : "+v"(vdt));  // (waited for here, so that the steps need not wait for the rows)
  if (chunks > 0) load(t_first, 0);

  // ---- the state: lane i16 has row i16 of its wave's 16; of tile nt columns
  // 32 (nt / 2) + 8 g4 + 4 (nt % 2) .. + 3, so that two tiles are 8 columns in
  // a row, as an operand takes them
  f32x4_t S[NT];
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) S[nt] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
  const int p_row = row0 + 16 * w4 + i16;
  const int64_t state0 = ((pool * a.nh + h) * a.hd + p_row) * a.N;
  auto column = [&](int nt) { return 32 * (nt >> 1) + 8 * g4 + 4 * (nt & 1); };
  const int64_t head = (static_cast<int64_t>(b) * a.nh + h) * pl.tiles + item % pl.tiles;
  constexpr int kBlock = kTileRows * NK * 32;
  auto seg_state = [&](int s, int nt) {
    return reinterpret_cast<f32x4_t*>(seg_states + (head * pl.segs + s) * kBlock + ((nt * 4 + w4) * 64 + lane) * 4);
  };
  if (live) {
    if (seg == 0) {
      if (!STATES && pl.keep_first && t_first + seg_len < len) {
        // (copied by the first pass; the array itself may have moved on)
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) S[nt] = *seg_state(pl.segs - 1, nt);
      } else if (a.s_in && pool >= 0 && p_row < a.hd) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
          if (column(nt) < a.N) S[nt] = *reinterpret_cast<const f32x4_t*>(a.s_in + state0 + column(nt));
      }
      if (STATES && pl.keep_first) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) *seg_state(pl.segs - 1, nt) = S[nt];
      }
    } else if (!STATES) {
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) S[nt] = *seg_state(0, nt);
      for (int s = 1; s < seg; ++s) {
        const float f = seg_decays[head * pl.segs + s];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) S[nt] = S[nt] * f + *seg_state(s, nt);
      }
    }
  }
  if (live && w4 < chunks) steps(w4);
  float seg_decay = 1.0f;

  // ---- operands' places in LDS, from a buffer's start; a few registers, of
  // which the others differ by a constant, added or (columns, swizzled) exclusive
  const int e4 = i16 >> 2, c4 = i16 & 3;
  const int row_base = chunk_at<CH>(i16, g4);               // 16 rows, one each lane: columns 8 g4 .. + 7
  const int col_base0 = chunk_at<CH>(8 * g4 + e4, c4);      // columns 8 c4 .. + 3 of row 8 g4 + e4
  const int col_base1 = chunk_at<CH>(8 * g4 + 4 + e4, c4);  // and of the row 4 behind it
  const int x_base0 = chunk_at<8>(8 * g4 + e4, 2 * w4 + (c4 >> 1)) + (c4 & 1) * 8;
  const int x_base1 = chunk_at<8>(8 * g4 + 4 + e4, 2 * w4 + (c4 >> 1)) + (c4 & 1) * 8;
  const int own_base = chunk_at<8>(i16, 2 * w4 + (g4 >> 1)) + (g4 & 1) * 8;  // rows 4 g4 .. + 3 of token i16
  const int m_base0 = weight_at(i16, g4), m_base1 = weight_at(32 + i16, g4);

  // The weights' 10 tiles of 16 tokens s and 16 tokens t: six below the diagonal
  // and the diagonal's four, which take longer, two to three a wave, or one for
  // both slots and, for four waves, another for one slot
  constexpr uint32_t kTileT = 0x6e4bf, kTileS = 0x1e424;  // two bits each
  constexpr int kTiles = 10, kTurns = SLOTS == 2 ? 2 : 3;

  wait_vmcnt0();
  for (int ck = 0; ck < chunks; ++ck) {
    const int t0 = t_first + ck * kChunk, nt_live = min(kChunk, t_end - t0);
    const int buf = kBufs == 2 ? ck & 1 : 0;
    const bool more = ck + 1 < chunks;
    lds_barrier();  // the chunk's rows have landed, and every wave is done with the one before it
    const int next = ck - ck % kRound + kRound + w4;  // of the next round, this wave's
    if (live && ck % kRound == 0 && next < chunks) load_dt(next);
    if (kBufs == 2 && more) load(t0 + kChunk, buf ^ 1);
    const uint8_t* bs = lds.b[buf];
    const uint8_t* xs = lds.x[buf][slot];
    const ChunkSteps<STATES>* round = lds.steps[ck % kRing];
    const ChunkSteps<STATES>& st = round[slot];
    f32x4_t y[4];
    // float16's operands are scaled, each row by its own power of two: a row
    // much smaller than its neighbours keeps its bits
    auto row_max = [](float v) {
      v = fmaxf(v, __shfl_xor(v, 16));
      return fmaxf(v, __shfl_xor(v, 32));
    };
    float most_s = 0.0f;  // of the row's magnitudes, NaN aside
    if (F16 && live) {
      auto largest = [&]() {
        most_s = 0.0f;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int i = 0; i < 4; ++i) most_s = fmaxf(most_s, fabsf(S[nt][i]));
        most_s = row_max(most_s);
      };
      largest();
      if (__any(__float_as_uint(most_s) >= 0x7f800000u)) {  // (no scale takes an infinity)
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) S[nt] += S[nt] * 0.0f;
        largest();
      }
    }

    if constexpr (!STATES) {
      const uint8_t* cs = lds.c[buf];
      const int row_at = afresh(row_base);
      // ---- what the state before the chunk gives: rows p, columns t
      if (live) {
#pragma unroll
        for (int tt = 0; tt < 4; ++tt) y[tt] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
        float back = 1.0f;
        const float scale = F16 ? scale_of(most_s, &back) : 1.0f;
#pragma unroll
        for (int kk = 0; kk < NK; ++kk) {
          s16x8_t fc[4];
#pragma unroll
          for (int tt = 0; tt < 4; ++tt)
            fc[tt] = *reinterpret_cast<const s16x8_t*>(cs + (row_at ^ 64 * kk) + tt * 16 * Lds::kRow);
          float v[8];
#pragma unroll
          for (int i = 0; i < 8; ++i) v[i] = F16 ? S[2 * kk + i / 4][i % 4] * scale : S[2 * kk + i / 4][i % 4];
          constexpr int kParts = F16 ? 2 : 3;
          s16x8_t part[kParts];
          if constexpr (F16)
            split_f16(v, part);
          else
            split_bf16<3>(v, part);
          read_first();
#pragma unroll
          for (int k = 0; k < kParts; ++k)
#pragma unroll
            for (int tt = 0; tt < 4; ++tt) y[tt] = mfma_in<F16>(part[k], fc[tt], y[tt]);
        }
        f32x4_t backs{1.0f, 1.0f, 1.0f, 1.0f};  // of the rows that the products are in
        if (F16) {
#pragma unroll
          for (int i = 0; i < 4; ++i) backs[i] = __shfl(back, 4 * g4 + i);
        }
#pragma unroll
        for (int tt = 0; tt < 4; ++tt) {
          y[tt] *= st.out[16 * tt + i16];
          if (F16) y[tt] *= backs;
        }
      }
      // ---- weights of the chunk's tokens: (c . b) times decay and step
      for (int turn = 0; turn < kTurns; ++turn) {
        const bool both = SLOTS == 1 || turn == 0;
        const int k = both ? wave + 4 * turn : 8 + (wave >> 1);
        if (k >= kTiles) break;
        const int tt = kTileT >> 2 * k & 3, ss = kTileS >> 2 * k & 3;
        f32x4_t dot{0.0f, 0.0f, 0.0f, 0.0f};
        s16x8_t fb[NK], fc[NK];
#pragma unroll
        for (int kk = 0; kk < NK; ++kk) {
          fb[kk] = *reinterpret_cast<const s16x8_t*>(bs + (row_at ^ 64 * kk) + ss * 16 * Lds::kRow);
          fc[kk] = *reinterpret_cast<const s16x8_t*>(cs + (row_at ^ 64 * kk) + tt * 16 * Lds::kRow);
        }
        read_first();
#pragma unroll
        for (int kk = 0; kk < NK; ++kk) dot = mfma_in<F16>(fb[kk], fc[kk], dot);
        const int t = 16 * tt + i16, s = 16 * ss + 4 * g4;
#pragma unroll
        for (int q = 0; q < SLOTS; ++q) {
          if (q >= n_slots || (!both && q != (wave & 1))) continue;
          const ChunkSteps<STATES>& sq = round[q];
          float m[4];
          if (ss < tt) {
            const f32x4_t far = *reinterpret_cast<const f32x4_t*>(sq.far + far_at(tt) + s);
            const float near = sq.near[t];
#pragma unroll
            for (int i = 0; i < 4; ++i) m[i] = dot[i] * (far[i] * near);
          } else {
            const f32x4_t sum = *reinterpret_cast<const f32x4_t*>(sq.sum + s);
            const f32x4_t rest = *reinterpret_cast<const f32x4_t*>(sq.rest + s);
            const f32x4_t dt = *reinterpret_cast<const f32x4_t*>(sq.dt + s);
            const float sum_t = sq.sum[t], rest_t = sq.rest[t];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const float f = __builtin_amdgcn_exp2f((sum_t - sum[i]) + (rest_t - rest[i]));
              // (by its bits: tokens behind t may hold anything)
              m[i] = __uint_as_float(__float_as_uint(dot[i] * (f * dt[i])) & (s + i <= t ? 0xffffffffu : 0u));
            }
          }
          const int at = weight_at(t, 2 * ss + (g4 >> 1)) + (g4 & 1) * 8;
#pragma unroll
          for (int k = 0; k < kWeightParts; ++k) {  // cut to 8 bits each
            *reinterpret_cast<u32x2_t*>(lds.m[q][k] + at) =
                u32x2_t{__builtin_amdgcn_perm(__float_as_uint(m[1]), __float_as_uint(m[0]), 0x07060302u),
                        __builtin_amdgcn_perm(__float_as_uint(m[3]), __float_as_uint(m[2]), 0x07060302u)};
#pragma unroll
            for (int i = 0; i < 4; ++i) m[i] -= hi_bf16(__float_as_uint(m[i]));
          }
        }
      }
      lds_barrier();  // the weights are in LDS
    }

    if (live) {
      // ---- the chunk's rows of x: lane i16 has row p, tokens 32 ks + 8 g4 + j
      const int x_at0 = afresh(x_base0), x_at1 = afresh(x_base1);
      s16x8_t fx[2];
#pragma unroll
      for (int ks = 0; ks < 2; ++ks) {
        const s16x4_t lo = read_tr(xs + x_at0 + ks * 32 * 128), hi = read_tr(xs + x_at1 + ks * 32 * 128);
        fx[ks] = __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
      }
      uint32_t odd = 0;
      constexpr uint32_t kUnit = F16 ? 0x04000400u : 0x00800080u;  // carries an exponent of ones into the sign
#pragma unroll
      for (int ks = 0; ks < 2; ++ks) {
        const u32x4_t w = __builtin_bit_cast(u32x4_t, fx[ks]);
#pragma unroll
        for (int j = 0; j < 4; ++j) odd |= (w[j] & 0x7fff7fffu) + kUnit;
      }
      int from = kChunk;  // the token from which row i16 is NaN
      float poison = 0.0f;  // added to its state's decay (a branch that changes the state costs a copy of it)
      const bool spoiled = __any((odd & 0x80008000u) != 0);
      if (spoiled) {
        // Values that are not finite, which the products would carry to the
        // tokens before theirs as 0 times infinity: taken out, and their row
        // NaN from their token on.
#pragma unroll
        for (int ks = 0; ks < 2; ++ks) {
          u32x4_t w = __builtin_bit_cast(u32x4_t, fx[ks]);
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const uint32_t is = ((w[j] & 0x7fff7fffu) + kUnit) >> 15 & 0x00010001u;
            w[j] &= ~((is << 16) - is);
            const int t = 32 * ks + 8 * g4 + 2 * j;
            from = min(from, t + kChunk - kChunk * static_cast<int>(is & 1));
            from = min(from, t + 1 + kChunk - kChunk * static_cast<int>(is >> 16));
          }
          fx[ks] = __builtin_bit_cast(s16x8_t, w);
        }
        from = min(from, __shfl_xor(from, 16));
        from = min(from, __shfl_xor(from, 32));
        poison = from < kChunk ? __builtin_nanf("") : 0.0f;
      }
      float u[8];  // what tokens 32 ks + 8 g4 + j bring
      auto incoming = [&](int ks) {
        const f32x4_t in0 = *reinterpret_cast<const f32x4_t*>(st.in + 32 * ks + 8 * g4);
        const f32x4_t in1 = *reinterpret_cast<const f32x4_t*>(st.in + 32 * ks + 8 * g4 + 4);
        const u32x4_t w = __builtin_bit_cast(u32x4_t, fx[ks]);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const float x = j % 2 ? Act<F16>::hi(w[j / 2]) : Act<F16>::lo(w[j / 2]);
          u[j] = (j < 4 ? in0[j] : in1[j - 4]) * x;
        }
      };
      float unscale = 1.0f, scale = 1.0f;
      if constexpr (F16) {
        float most = 0.0f;
#pragma unroll
        for (int ks = 0; ks < 2; ++ks) {
          incoming(ks);
#pragma unroll
          for (int j = 0; j < 8; ++j) most = fmaxf(most, fabsf(u[j]));
        }
        most = row_max(most);
        if (__float_as_uint(most) >= 0x7f800000u) {  // a step without end
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) S[nt] = f32x4_t{most, most, most, most} * 0.0f;
          most = 0.0f;
        }
        scale = scale_of(fmaxf(most, most_s * st.decay), &unscale);
      }
      if constexpr (!STATES) {
        // ---- what the chunk's own tokens give
        const int m_at0 = afresh(m_base0), m_at1 = afresh(m_base1);
#pragma unroll
        for (int ks = 0; ks < 2; ++ks) {
          s16x8_t fm[4][kWeightParts];
#pragma unroll
          for (int tt = 2 * ks; tt < 4; ++tt)
#pragma unroll
            for (int k = 0; k < kWeightParts; ++k)
              fm[tt][k] = *reinterpret_cast<const s16x8_t*>(
                  lds.m[slot][k] + (tt < 2 ? m_at0 + tt * 1024 : (m_at1 ^ 64 * ks) + (tt - 2) * 2048));
          read_first();
          s16x8_t xq[2] = {fx[ks], fx[ks]};
          if (F16) {
            const u32x4_t w = __builtin_bit_cast(u32x4_t, fx[ks]);
            float v[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) v[j] = j % 2 ? Act<F16>::hi(w[j / 2]) : Act<F16>::lo(w[j / 2]);
            split_bf16<2>(v, xq);
          }
#pragma unroll
          for (int k = 0; k < (F16 ? 2 : 1) * kWeightParts; ++k)
#pragma unroll
            for (int tt = 2 * ks; tt < 4; ++tt)
              y[tt] = mfma_bf16(xq[k / kWeightParts], fm[tt][k % kWeightParts], y[tt]);
        }
      }
      // ---- the state behind the chunk
      {
        const int col_at0 = afresh(col_base0), col_at1 = afresh(col_base1);
        const float f = F16 ? (st.decay + poison) * scale : st.decay + poison;
        if (STATES) seg_decay *= st.decay;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) S[nt] *= f;
#pragma unroll
        for (int ks = 0; ks < 2; ++ks) {
          constexpr int kParts = F16 ? 2 : 3, kAhead = NT < 4 ? NT : 4;
          s16x8_t part[kParts];
          incoming(ks);
          if constexpr (F16) {
#pragma unroll
            for (int j = 0; j < 8; ++j) u[j] *= scale;
            split_f16(u, part);
          } else {
            split_bf16<3>(u, part);
          }
#pragma unroll
          for (int first = 0; first < NT; first += kAhead) {
            s16x8_t fb[kAhead];
#pragma unroll
            for (int k = 0; k < kAhead; ++k) {
              const uint8_t* at = bs + ks * 32 * Lds::kRow;
              const int nt = first + k, flip = 64 * (nt >> 1), half = 8 * (nt & 1);
              const s16x4_t lo = read_tr(at + (col_at0 ^ flip) + half), hi = read_tr(at + (col_at1 ^ flip) + half);
              fb[k] = __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
            }
            read_first();
#pragma unroll
            for (int k = 0; k < kParts; ++k)
#pragma unroll
              for (int j = 0; j < kAhead; ++j) S[first + j] = mfma_in<F16>(fb[j], part[k], S[first + j]);
          }
        }
        if (F16) {
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) S[nt] *= unscale;
        }
      }
      // ---- the skip, and out: lane i16 has token t, rows 4 g4 .. + 3
      if constexpr (!STATES) {
        const int own_at = afresh(own_base);
        u32x2_t v[4];
#pragma unroll
        for (int tt = 0; tt < 4; ++tt) {
          const u32x2_t w = *reinterpret_cast<const u32x2_t*>(xs + own_at + tt * 2048);
          v[tt][0] = pack_in<F16>(__builtin_fmaf(skip, Act<F16>::lo(w[0]), y[tt][0]),
                                  __builtin_fmaf(skip, Act<F16>::hi(w[0]), y[tt][1]));
          v[tt][1] = pack_in<F16>(__builtin_fmaf(skip, Act<F16>::lo(w[1]), y[tt][2]),
                                  __builtin_fmaf(skip, Act<F16>::hi(w[1]), y[tt][3]));
        }
        if (kBufs == 2) wait_vmcnt0();  // (before the stores, which nobody waits for)
        const uint32_t to = static_cast<uint32_t>(i16 * static_cast<int>(a.out.ts) + 16 * w4 + 4 * g4);
#pragma unroll
        for (int tt = 0; tt < 4; ++tt)
          if (16 * tt + i16 < nt_live && row0 + 16 * w4 + 4 * g4 < a.hd)
            *reinterpret_cast<u32x2_t*>(op + 16 * tt * a.out.ts + to) = v[tt];
        if (spoiled) {
          wait_vmcnt0();
          for (int t = from + g4; t < nt_live; t += 4)
            if (p_row < a.hd) op[t * a.out.ts + 16 * w4 + i16] = F16 ? 0x7e00u : 0x7fc0u;
        }
        op += kChunk * a.out.ts;
      }
    }
    if (live && ck % kRound == kRound / 2 && next < chunks) steps(next);
    if (kBufs == 2 && (STATES || !live)) wait_vmcnt0();
    if (kBufs == 1 && more) {
      lds_barrier();
      load(t0 + kChunk, 0);
      wait_vmcnt0();
    }
  }

  if (!live) return;
  if (STATES) {
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) *seg_state(seg, nt) = S[nt];
    if (w4 == 0 && lane == 0) seg_decays[head * pl.segs + seg] = seg_decay;
  } else if (a.s_out && pool >= 0 && p_row < a.hd && seg == (len > 0 ? (len - 1) / seg_len : 0)) {
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
      if (column(nt) < a.N) *reinterpret_cast<f32x4_t*>(a.s_out + state0 + column(nt)) = S[nt];
  }
}

// ------------------------------------------------------------------ launches

int chunk_steps(int N) { return N <= 32 ? 1 : N <= 64 ? 2 : N <= 128 ? 4 : 8; }

// Tokens that the walk takes. One sequence of 64 heads of 64 rows and 128
// columns, in a graph: 8 tokens 9.9 us, 9 11.3, 12 13.1, 16 15.8, a chunk 9.9; 16
// of them 20, 22, 27, 32 and 25; 16 of 24 heads 8 13.0, 12 16.8, 16 19.8 and 12.7.
constexpr int kFewMost = 8;
constexpr int kFullGrid = 256;    // workgroups that fill the CUs (one each, by its LDS)
// Chunks of a segment up to which a workgroup takes one item rather than two
// (which halve the reads of b and c and half hide each other's latencies), in a
// graph: 64 heads of 200 tokens 20.4 us for 22.8, of 768 (3 chunks, 2 by two)
// 29.7 for 34.9, of 1024 (4, 2) 34.3 for 34.7; 4 sequences of 200 (4, 2) 23.0 for
// 29.9.
constexpr int kAloneChunks = 4;

struct ScanPlan {
  ChunkPlan ck;
  int slots, nk;
  size_t states;  // floats of the segments' states
  size_t bytes;
};

// Workgroups of `slots` items; as many segments as leave no CU without one and
// none with two, of 2 chunks at least. (8192 tokens of 64 heads in a graph: whole
// 584 us, in 2 segments 408, in 4 215, in 6 152, in 8 121, in 16 135; 16 ragged
// sequences of 24 heads, 192 workgroups: whole 125, in 2 152, in 4 130, in 6 117,
// in 8 144.)
ScanPlan scan_plan(const ScanArgs& a, int slots) {
  ScanPlan p{};
  ChunkPlan& c = p.ck;
  c.tiles = (a.hd + kTileRows - 1) / kTileRows;
  p.slots = slots;
  p.nk = chunk_steps(a.N);
  c.pairs = (a.rep * c.tiles + slots - 1) / slots;
  const int64_t base = static_cast<int64_t>(a.B) * a.groups * c.pairs;
  const int chunks = (a.L + kChunk - 1) / kChunk;
  const int want = static_cast<int>(std::min<int64_t>(kFullGrid / std::max<int64_t>(base, 1), 32));
  const int segs = std::max(1, std::min(want, chunks / 2));
  c.seg_chunks = (chunks + segs - 1) / segs;
  c.segs = (chunks + c.seg_chunks - 1) / c.seg_chunks;
  if (c.segs > 1) {
    const size_t heads = static_cast<size_t>(a.B) * a.nh * c.tiles * c.segs;
    p.states = heads * kTileRows * p.nk * 32;
    p.bytes = (p.states + heads) * sizeof(float);
  }
  return p;
}
ScanPlan scan_plan(const ScanArgs& a) {
  const ScanPlan p = scan_plan(a, 1);
  const bool alone = static_cast<int64_t>(a.B) * a.groups * p.ck.pairs <= kFullGrid && p.ck.seg_chunks <= kAloneChunks;
  return alone || a.rep * p.ck.tiles == 1 ? p : scan_plan(a, 2);
}

// a launch over `segs` segments: workgroups with work, neighbours on one XCD, and the grid
struct ChunkGrid {
  int64_t total, run, blocks;
};
ChunkGrid chunk_grid(const ScanArgs& a, const ChunkPlan& c, int segs) {
  ChunkGrid g;
  g.total = static_cast<int64_t>(a.B) * segs * a.groups * c.pairs;
  g.run = std::max<int64_t>(1, std::min<int64_t>(c.pairs, g.total / 64));
  g.blocks = (g.total + 8 * g.run - 1) / (8 * g.run) * (8 * g.run);
  return g;
}

template <bool F16, int NK, int SLOTS>
hipError_t scan_chunks(const ScanArgs& a, ScanPlan p, float* ws, hipStream_t stream) {
  ChunkPlan& c = p.ck;
  c.keep_first = a.s_in && a.s_in == a.s_out;
  float* decays = ws + p.states;
  for (int pass = c.segs > 1 ? 0 : 1; pass < 2; ++pass) {
    c.first_segs = pass ? c.segs : c.segs - 1;
    const ChunkGrid g = chunk_grid(a, c, c.first_segs);
    c.total = static_cast<uint32_t>(g.total);
    c.run = static_cast<int>(g.run);
    const dim3 grid(static_cast<uint32_t>(g.blocks)), wg(kSlotThreads * SLOTS);
    if (pass)
      hipLaunchKernelGGL((scan_chunk_kernel<F16, NK, SLOTS, false>), grid, wg, 0, stream, a, c, ws, decays);
    else
      hipLaunchKernelGGL((scan_chunk_kernel<F16, NK, SLOTS, true>), grid, wg, 0, stream, a, c, ws, decays);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
  }
  return hipSuccess;
}

template <bool F16>
hipError_t scan_chunks(const ScanArgs& a, float* ws, hipStream_t stream) {
  const ScanPlan p = scan_plan(a);
#define FMX_CHUNKS(NK) \
  p.slots == 2 ? scan_chunks<F16, NK, 2>(a, p, ws, stream) : scan_chunks<F16, NK, 1>(a, p, ws, stream)
  switch (p.nk) {
    case 1: return FMX_CHUNKS(1);
    case 2: return FMX_CHUNKS(2);
    case 4: return FMX_CHUNKS(4);
    default: return FMX_CHUNKS(8);
  }
#undef FMX_CHUNKS
}

// (the chunks' lanes address 64 rows by 32-bit offsets)
bool scan_in_chunks(const ScanArgs& a) {
  constexpr int64_t kMost = int64_t{1} << 24;
  return a.L > kFewMost && a.x.ts < kMost && a.b.ts < kMost && a.c.ts < kMost && a.out.ts < kMost;
}

}  // namespace

size_t scan_workspace(const ScanArgs& a) { return scan_in_chunks(a) ? scan_plan(a).bytes : 0; }

bool scan_fits(const ScanArgs& a) {
  if (!scan_in_chunks(a))
    return static_cast<int64_t>(a.B) * a.nh * few_parts(a, state_lanes(a.N)) <= max_blocks(kFewThreads);
  const ScanPlan p = scan_plan(a);
  return chunk_grid(a, p.ck, p.ck.segs).blocks <= max_blocks(kSlotThreads * p.slots);
}

hipError_t launch_scan(const ScanArgs& a, bool f16, void* ws, hipStream_t stream) {
  if (a.B == 0) return hipSuccess;
  if (scan_in_chunks(a))
    return f16 ? scan_chunks<true>(a, static_cast<float*>(ws), stream)
               : scan_chunks<false>(a, static_cast<float*>(ws), stream);
  return f16 ? scan_few<true>(a, stream) : scan_few<false>(a, stream);
}

}  // namespace fmx
