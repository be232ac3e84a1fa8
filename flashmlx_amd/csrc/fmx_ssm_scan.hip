// fmx_ssm_scan.hip -- the selective scan of the state space layer (the
// mixer's ssm_kernel, server/src/nemotron_h.cpp:608-653), per sequence and head:
//   S[p, n] = exp(dt a) S[p, n] + dt x[p] b[n];  out[p] = sum_n c[n] S[p, n] + d x[p]
//
// scan_few_kernel walks the tokens one by one with the state in registers.
//
// scan_chunk_kernel takes chunks of 64 tokens on the matrix cores. With f(s, t)
// the product of the decays of the tokens s + 1 .. t, the chunk's outputs are
//   out[t] = f(start, t) c[t] S + sum over s <= t of (c[t] . b[s]) f(s, t) dt[s] x[s]
// and its last state f(start, end) S + sum over s of f(s, end) dt[s] x[s] b[s],
// three products of matrices and one for the dots, which the heads of a group
// share. A wave has 16 rows of a head's state in accumulators, whose layout is
// an operand's as it is; only the weights of x cross waves, through LDS. fp32
// operands go in as sums of numbers of 8 (bf16) or 11 bits: three of them (24
// bits) where the state takes them in, two where outputs do, which are rounded
// to 8 or 11 bits. Long sequences are cut into segments: a first launch forms
// each segment's state from 0, a second starts each segment from the sum of
// those before it.
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
  return static_cast<uint32_t>(f32_to_bf16(a)) | static_cast<uint32_t>(f32_to_bf16(b)) << 16;
}
__device__ inline float lo_bf16(uint32_t v) { return __uint_as_float(v << 16); }
__device__ inline float hi_bf16(uint32_t v) { return __uint_as_float(v & 0xffff0000u); }

// Values as a sum of PARTS numbers of bf16 (8 bits each), in order
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
      w[j] = pack_bf16(rest[2 * j], rest[2 * j + 1]);
      if (k + 1 < PARTS) {
        rest[2 * j] -= lo_bf16(w[j]);
        rest[2 * j + 1] -= hi_bf16(w[j]);
      }
    }
    part[k] = __builtin_bit_cast(s16x8_t, w);
  }
}
// as a sum of two of float16 (22 bits), of values within 2^15
__device__ inline void split_f16(const float* v, s16x8_t* part) {
  u32x4_t h, l;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const auto a = __builtin_amdgcn_cvt_pkrtz(v[2 * j], v[2 * j + 1]);
    const auto b = __builtin_amdgcn_cvt_pkrtz(v[2 * j] - static_cast<float>(a[0]), v[2 * j + 1] - static_cast<float>(a[1]));
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

// What a chunk's tokens need, per slot and buffer. Sums of log2 e dt a from the
// chunk's start as two floats: their differences are exact to 2^-24 of
// themselves, however far the sums have run.
struct ChunkSteps {
  float sum[kChunk], rest[kChunk], dt[kChunk];
  float in[kChunk];    // dt times the decay from the token to the chunk's end
  float out[kChunk];   // the decay from the chunk's start to the token
  float decay;         // of the whole chunk
  float pad[3];
};

template <int NK, int SLOTS, bool STATES>
struct ChunkLds {
  static constexpr int kRow = NK * 64;  // bytes of a token's b or c
  __attribute__((aligned(16))) uint8_t b[kChunk * kRow];
  __attribute__((aligned(16))) uint8_t c[STATES ? 16 : kChunk * kRow];
  __attribute__((aligned(16))) uint8_t x[SLOTS][kChunk * kTileRows * 2];
  // weights of the tokens s for token t, in two parts: rows t < 32 of 32
  // tokens, the others of 64
  __attribute__((aligned(16))) uint8_t m[STATES ? 1 : SLOTS][STATES ? 1 : 2][STATES ? 16 : 32 * 64 + 32 * 128];
  ChunkSteps steps[2][SLOTS];
};

__device__ inline int weight_at(int t, int chunk) {
  return t < 32 ? chunk_at<4>(t, chunk) : 32 * 64 + chunk_at<8>(t - 32, chunk);
}

// NK: 32-column steps of a state row. STATES: the first pass over segments,
// which forms their states alone.
template <bool F16, int NK, int SLOTS, bool STATES>
__global__ __launch_bounds__(kSlotThreads* SLOTS, NK > 4 ? 2 : 4) void scan_chunk_kernel(ScanArgs a, ChunkPlan pl, float* seg_states, float* seg_decays) {
  typedef ChunkLds<NK, SLOTS, STATES> Lds;
  constexpr int kThreads = kSlotThreads * SLOTS;
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

  // ---- loads of a chunk to registers, and from there to LDS
  constexpr int kBc = NK > SLOTS ? NK / SLOTS : 1;  // vectors of a thread, of b and c each
  constexpr int kBcVecs = kChunk * CH;
  u32x4_t vb[kBc], vc[kBc], vx[2];
  uint16_t vdt = 0;
  const uint16_t* bp = static_cast<const uint16_t*>(a.b.p) + b * a.b.bs + grp * a.b.hs;
  const uint16_t* cp = STATES ? nullptr : static_cast<const uint16_t*>(a.c.p) + b * a.c.bs + grp * a.c.hs;
  const uint16_t* xp = static_cast<const uint16_t*>(a.x.p) + b * a.x.bs + h * a.x.hs + row0;
  const uint16_t* dtp = static_cast<const uint16_t*>(a.dt.p) + b * a.dt.bs + h * a.dt.hs;
  const u32x4_t zero{0, 0, 0, 0};
  const bool steps_wave = live && w4 == 3;
  auto load = [&](int t0) {
#pragma unroll
    for (int k = 0; k < kBc; ++k) {
      const int v = tid + k * kThreads, row = v / CH, col = v % CH * 8;
      vb[k] = zero;
      vc[k] = zero;
      if (v < kBcVecs && t0 + row < t_end && col < a.N) {
        vb[k] = *reinterpret_cast<const u32x4_t*>(bp + (t0 + row) * a.b.ts + col);
        if (!STATES) vc[k] = *reinterpret_cast<const u32x4_t*>(cp + (t0 + row) * a.c.ts + col);
      }
    }
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const int v = (tid & 255) + k * kSlotThreads, row = v / 8, col = v % 8 * 8;
      vx[k] = zero;
      if (live && t0 + row < t_end && row0 + col < a.hd)
        vx[k] = *reinterpret_cast<const u32x4_t*>(xp + (t0 + row) * a.x.ts + col);
    }
    if (steps_wave) vdt = t0 + lane < t_end ? dtp[(t0 + lane) * a.dt.ts] : 0;
  };
  auto stage = [&]() {
#pragma unroll
    for (int k = 0; k < kBc; ++k) {
      // columns 8 m .. 8 m + 7 of a 32-column step in the order in which an
      // accumulator's rows come: 4 g + i beside 16 + 4 g + i
      const int v = tid + k * kThreads, row = v / CH, m = v % 4, step = v % CH / 4;
      if (v >= kBcVecs) continue;
      const int half = (m >> 1) * 8;
      const int at0 = chunk_at<CH>(row, step * 4 + 2 * (m & 1)) + half;
      const int at1 = chunk_at<CH>(row, step * 4 + 2 * (m & 1) + 1) + half;
      *reinterpret_cast<u32x2_t*>(lds.b + at0) = u32x2_t{vb[k][0], vb[k][1]};
      *reinterpret_cast<u32x2_t*>(lds.b + at1) = u32x2_t{vb[k][2], vb[k][3]};
      if (!STATES) {
        *reinterpret_cast<u32x2_t*>(lds.c + at0) = u32x2_t{vc[k][0], vc[k][1]};
        *reinterpret_cast<u32x2_t*>(lds.c + at1) = u32x2_t{vc[k][2], vc[k][3]};
      }
    }
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const int v = (tid & 255) + k * kSlotThreads;
      *reinterpret_cast<u32x4_t*>(lds.x[slot] + chunk_at<8>(v / 8, v % 8)) = vx[k];
    }
  };

  // ---- the tokens' steps, formed by one wave of a slot: sums and their
  // differences in 64 bits
  const float rate = a.a[h], skip = a.d ? a.d[h] : 0.0f;
  double seg_sum = 0.0;
  auto steps = [&](int t0, int buf) {
    const bool in = t0 + lane < t_end;
    const float dt = in ? time_step(Act<F16>::ld(vdt), a.dt_bias, h, a.softplus, a.dt_min, a.dt_max) : 0.0f;
    double sum = in ? static_cast<double>(dt) * static_cast<double>(rate) * 1.4426950408889634074 : 0.0;
    sum = tree_to_last<64>(sum, 0.0, [](double x, double y) { return x + y; });
    const double all = readlane_f64(sum, 63);
    ChunkSteps& s = lds.steps[buf][slot];
    const float lead = static_cast<float>(sum);
    s.sum[lane] = lead;
    s.rest[lane] = static_cast<float>(sum - static_cast<double>(lead));
    s.dt[lane] = dt;
    s.in[lane] = in ? dt * __builtin_amdgcn_exp2f(static_cast<float>(all - sum)) : 0.0f;
    s.out[lane] = __builtin_amdgcn_exp2f(lead);
    if (lane == 0) s.decay = __builtin_amdgcn_exp2f(static_cast<float>(all));
    seg_sum += all;
  };

  // ---- the state: lane i16 has row i16 of its wave's 16, of the 16-column
  // tile nt columns 16 nt + 4 g4 .. + 3
  f32x4_t S[NT];
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) S[nt] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
  const int p_row = row0 + 16 * w4 + i16;
  const int64_t state0 = ((pool * a.nh + h) * a.hd + p_row) * a.N + 4 * g4;
  const int64_t head = (static_cast<int64_t>(b) * a.nh + h) * pl.tiles + item % pl.tiles;
  constexpr int kBlock = kTileRows * NK * 32;
  auto seg_state = [&](int s, int nt) {
    return reinterpret_cast<f32x4_t*>(seg_states + (head * pl.segs + s) * kBlock + ((nt * 4 + w4) * 64 + lane) * 4);
  };
  bool begun = false;  // whether the state may be other than 0
  if (live) {
    if (seg == 0) {
      const bool copied = !STATES && pl.keep_first && pl.segs > 1;
      if (copied ? t_first + seg_len < len : false) {
        // (written by the first pass; the array itself may have moved on)
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) S[nt] = *seg_state(pl.segs - 1, nt);
        begun = true;
      } else if (a.s_in && pool >= 0) {
        begun = true;
        if (p_row < a.hd) {
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
            if (16 * nt + 4 * g4 < a.N) S[nt] = *reinterpret_cast<const f32x4_t*>(a.s_in + state0 + 16 * nt);
        }
      }
      if (STATES && pl.keep_first) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) *seg_state(pl.segs - 1, nt) = S[nt];
      }
    } else if (!STATES) {
      begun = true;
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) S[nt] = *seg_state(0, nt);
      for (int s = 1; s < seg; ++s) {
        const float f = seg_decays[head * pl.segs + s];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) S[nt] = S[nt] * f + *seg_state(s, nt);
      }
    }
  }

  // ---- operands' places in LDS
  int row_at[NK];  // 16 rows, one each lane: chunk 4 step + g4
#pragma unroll
  for (int kk = 0; kk < NK; ++kk) row_at[kk] = chunk_at<CH>(i16, 4 * kk + g4);
  const int e4 = i16 >> 2, c4 = i16 & 3;
  int col_at[NK][2];  // columns of 4 rows by 4: rows 8 g4 + e4, and 4 behind them
#pragma unroll
  for (int kk = 0; kk < NK; ++kk)
#pragma unroll
    for (int u = 0; u < 2; ++u) col_at[kk][u] = chunk_at<CH>(8 * g4 + 4 * u + e4, 4 * kk + c4);
  int x_at[2];
#pragma unroll
  for (int u = 0; u < 2; ++u)
    x_at[u] = chunk_at<8>(8 * g4 + 4 * u + e4, 2 * w4 + (c4 >> 1)) + (c4 & 1) * 8;
  const uint8_t* xs = lds.x[slot];

  // weights' tiles (tokens s, token t) of this wave, rows of t from the longest on
  const int tile0 = SLOTS == 2 ? (wave < 2 ? 2 * wave : wave + 2) : (wave < 2 ? 2 * wave : 3 * wave - 2);
  const int tile1 = SLOTS == 2 ? (wave < 2 ? tile0 + 2 : tile0 + 1) : (wave < 2 ? tile0 + 2 : tile0 + 3);

  if (!STATES) {  // tokens behind t in a step that t's own are in
    for (int v = tid; v < SLOTS * 2 * 16 * 2; v += kThreads) {
      const int c = v % 2, t = v / 2 % 16, part = v / 32 % 2, q = v / 64;
      *reinterpret_cast<u32x4_t*>(lds.m[q][part] + weight_at(t, 2 + c)) = zero;
      *reinterpret_cast<u32x4_t*>(lds.m[q][part] + weight_at(32 + t, 6 + c)) = zero;
    }
  }

  if (chunks > 0) {
    load(t_first);
    if (steps_wave) steps(t_first, 0);
    stage();
  }
  lds_barrier();

  for (int ck = 0; ck < chunks; ++ck) {
    const int t0 = t_first + ck * kChunk, nt_live = min(kChunk, t_end - t0);
    const bool more = ck + 1 < chunks;
    const ChunkSteps& st = lds.steps[ck & 1][slot];
    if (more) load(t0 + kChunk);
    f32x4_t y[4];
    float most_s = 0.0f;  // of the state's magnitudes (float16)
    if (F16 && live && begun) {
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int i = 0; i < 4; ++i) most_s = fmaxf(most_s, fabsf(S[nt][i]));
      most_s = wave_max_f32(most_s);
    }
    bool slow = F16 && __float_as_uint(most_s) >= 0x7f800000u;

    if constexpr (!STATES) {
      // ---- weights of the chunk's tokens: (c . b) times decay and step
      for (int k = tile0; k < tile1; ++k) {
        const int tt = k < 4 ? 3 : k < 7 ? 2 : k < 9 ? 1 : 0;
        const int ss = k < 4 ? k : k < 7 ? k - 4 : k < 9 ? k - 7 : 0;
        if (16 * tt >= nt_live) continue;
        f32x4_t dot{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int kk = 0; kk < NK; ++kk) {
          const s16x8_t fb = *reinterpret_cast<const s16x8_t*>(lds.b + row_at[kk] + ss * 16 * Lds::kRow);
          const s16x8_t fc = *reinterpret_cast<const s16x8_t*>(lds.c + row_at[kk] + tt * 16 * Lds::kRow);
          dot = mfma_in<F16>(fb, fc, dot);
        }
        const int t = 16 * tt + i16, s = 16 * ss + 4 * g4;
#pragma unroll
        for (int q = 0; q < SLOTS; ++q) {
          if (q >= n_slots) break;
          const ChunkSteps& sq = lds.steps[ck & 1][q];
          const f32x4_t sum = *reinterpret_cast<const f32x4_t*>(sq.sum + s);
          const f32x4_t rest = *reinterpret_cast<const f32x4_t*>(sq.rest + s);
          const f32x4_t dt = *reinterpret_cast<const f32x4_t*>(sq.dt + s);
          const float sum_t = sq.sum[t], rest_t = sq.rest[t];
          float m[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float f = __builtin_amdgcn_exp2f((sum_t - sum[i]) + (rest_t - rest[i]));
            m[i] = s + i <= t ? dot[i] * (f * dt[i]) : 0.0f;
          }
          const uint32_t h0 = pack_bf16(m[0], m[1]), h1 = pack_bf16(m[2], m[3]);
          const uint32_t l0 = pack_bf16(m[0] - lo_bf16(h0), m[1] - hi_bf16(h0));
          const uint32_t l1 = pack_bf16(m[2] - lo_bf16(h1), m[3] - hi_bf16(h1));
          const int at = weight_at(t, 2 * ss + (g4 >> 1)) + (g4 & 1) * 8;
          *reinterpret_cast<u32x2_t*>(lds.m[q][0] + at) = u32x2_t{h0, h1};
          *reinterpret_cast<u32x2_t*>(lds.m[q][1] + at) = u32x2_t{l0, l1};
        }
      }
      // ---- what the state before the chunk gives: rows p, columns t
#pragma unroll
      for (int tt = 0; tt < 4; ++tt) y[tt] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
      if (live && begun) {
        float back = 1.0f;
        const float scale = F16 ? scale_of(most_s, &back) : 1.0f;
#pragma unroll
        for (int kk = 0; kk < NK; ++kk) {
          float v[8];
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            v[i] = F16 ? S[2 * kk][i] * scale : S[2 * kk][i];
            v[4 + i] = F16 ? S[2 * kk + 1][i] * scale : S[2 * kk + 1][i];
          }
          s16x8_t part[2];
          if (F16)
            split_f16(v, part);
          else
            split_bf16<2>(v, part);
#pragma unroll
          for (int tt = 0; tt < 4; ++tt) {
            if (16 * tt >= nt_live) break;
            const s16x8_t fc = *reinterpret_cast<const s16x8_t*>(lds.c + row_at[kk] + tt * 16 * Lds::kRow);
            y[tt] = mfma_in<F16>(part[0], fc, y[tt]);
            y[tt] = mfma_in<F16>(part[1], fc, y[tt]);
          }
        }
#pragma unroll
        for (int tt = 0; tt < 4; ++tt) {
          const float f = st.out[16 * tt + i16];
          y[tt] *= F16 ? f * back : f;
        }
      }
      lds_barrier();  // the weights are in LDS
    }

    if (live) {
      // ---- the chunk's rows of x: lane i16 has row p, tokens 32 ks + 8 g4 + j
      s16x8_t fx[2];
      uint32_t odd = 0;  // values that are not finite
#pragma unroll
      for (int ks = 0; ks < 2; ++ks) {
        const s16x4_t lo = read_tr(xs + x_at[0] + ks * 32 * 128), hi = read_tr(xs + x_at[1] + ks * 32 * 128);
        fx[ks] = __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
        const u32x4_t w = __builtin_bit_cast(u32x4_t, fx[ks]);
        const uint32_t unit = F16 ? 0x04000400u : 0x00800080u;
#pragma unroll
        for (int j = 0; j < 4; ++j) odd |= (w[j] & 0x7fff7fffu) + unit;
      }
      slow = slow || ((!STATES || F16) && __any((odd & 0x80008000u) != 0));
      float u[2][8];
      float most_u = 0.0f;
      auto incoming = [&](int ks) {
        const f32x4_t in0 = *reinterpret_cast<const f32x4_t*>(st.in + 32 * ks + 8 * g4);
        const f32x4_t in1 = *reinterpret_cast<const f32x4_t*>(st.in + 32 * ks + 8 * g4 + 4);
        const u32x4_t w = __builtin_bit_cast(u32x4_t, fx[ks]);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const float x = j % 2 ? Act<F16>::hi(w[j / 2]) : Act<F16>::lo(w[j / 2]);
          u[ks][j] = (j < 4 ? in0[j] : in1[j - 4]) * x;
        }
      };
      float unscale = 1.0f, scale = 1.0f;
      if constexpr (F16) {
#pragma unroll
        for (int ks = 0; ks < 2; ++ks) {
          incoming(ks);
#pragma unroll
          for (int j = 0; j < 8; ++j) most_u = fmaxf(most_u, fabsf(u[ks][j]));
        }
        most_u = wave_max_f32(most_u);
        const float most = fmaxf(most_u, most_s * st.decay);
        slow = slow || __float_as_uint(most) >= 0x7f800000u;
        scale = scale_of(most, &unscale);
      }
      if (!slow) {
        if constexpr (!STATES) {
          // ---- what the chunk's own tokens give
          s16x8_t xh[2], xl[2];
          if (F16) {
#pragma unroll
            for (int ks = 0; ks < 2; ++ks) {
              const u32x4_t w = __builtin_bit_cast(u32x4_t, fx[ks]);
              float v[8];
#pragma unroll
              for (int j = 0; j < 8; ++j) v[j] = j % 2 ? Act<F16>::hi(w[j / 2]) : Act<F16>::lo(w[j / 2]);
              s16x8_t part[2];
              split_bf16<2>(v, part);
              xh[ks] = part[0];
              xl[ks] = part[1];
            }
          } else {
#pragma unroll
            for (int ks = 0; ks < 2; ++ks) xh[ks] = fx[ks];
          }
#pragma unroll
          for (int tt = 0; tt < 4; ++tt) {
            if (16 * tt >= nt_live) break;
#pragma unroll
            for (int ks = 0; ks <= tt / 2; ++ks) {
              const int at = weight_at(16 * tt + i16, 4 * ks + g4);
              const s16x8_t mh = *reinterpret_cast<const s16x8_t*>(lds.m[slot][0] + at);
              const s16x8_t ml = *reinterpret_cast<const s16x8_t*>(lds.m[slot][1] + at);
              y[tt] = mfma_bf16(xh[ks], mh, y[tt]);
              y[tt] = mfma_bf16(xh[ks], ml, y[tt]);
              if (F16) y[tt] = mfma_bf16(xl[ks], mh, y[tt]);
            }
          }
          // ---- the skip, and out: lane i16 has token t, rows 4 g4 .. + 3
          const int p = 16 * w4 + 4 * g4;
#pragma unroll
          for (int tt = 0; tt < 4; ++tt) {
            const int t = 16 * tt + i16;
            const u32x2_t w = *reinterpret_cast<const u32x2_t*>(xs + chunk_at<8>(t, 2 * w4 + (g4 >> 1)) + (g4 & 1) * 8);
            float v[4] = {y[tt][0], y[tt][1], y[tt][2], y[tt][3]};
            if (a.d) {
              v[0] = __builtin_fmaf(skip, Act<F16>::lo(w[0]), v[0]);
              v[1] = __builtin_fmaf(skip, Act<F16>::hi(w[0]), v[1]);
              v[2] = __builtin_fmaf(skip, Act<F16>::lo(w[1]), v[2]);
              v[3] = __builtin_fmaf(skip, Act<F16>::hi(w[1]), v[3]);
            }
            if (t < nt_live && row0 + p < a.hd) {
              uint16_t* to = static_cast<uint16_t*>(a.out.p) + b * a.out.bs + (t0 + t) * a.out.ts + h * a.out.hs + row0 + p;
              *reinterpret_cast<u32x2_t*>(to) =
                  u32x2_t{static_cast<uint32_t>(Act<F16>::st(v[0])) | static_cast<uint32_t>(Act<F16>::st(v[1])) << 16,
                          static_cast<uint32_t>(Act<F16>::st(v[2])) | static_cast<uint32_t>(Act<F16>::st(v[3])) << 16};
            }
          }
        }
        // ---- the state behind the chunk
        const float f = F16 ? st.decay * scale : st.decay;
        if (begun) {
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) S[nt] *= f;
        }
#pragma unroll
        for (int ks = 0; ks < 2; ++ks) {
          if (32 * ks >= nt_live) break;
          s16x8_t part[3];
          if constexpr (F16) {
#pragma unroll
            for (int j = 0; j < 8; ++j) u[ks][j] *= scale;
            split_f16(u[ks], part);
          } else {
            incoming(ks);
            split_bf16<3>(u[ks], part);
          }
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
            const uint8_t* at = lds.b + ks * 32 * Lds::kRow + (nt & 1) * 8;
            const s16x4_t lo = read_tr(at + col_at[nt >> 1][0]), hi = read_tr(at + col_at[nt >> 1][1]);
            const s16x8_t fb = __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
            S[nt] = mfma_in<F16>(fb, part[0], S[nt]);
            S[nt] = mfma_in<F16>(fb, part[1], S[nt]);
            if (!F16) S[nt] = mfma_in<F16>(fb, part[2], S[nt]);
          }
        }
        if (F16) {
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) S[nt] *= unscale;
        }
      } else {
        // ---- values that are not finite: token by token, so that they reach
        // no other row and no earlier token
        for (int t = 0; t < nt_live; ++t) {
          const float s1 = st.sum[t], r1 = st.rest[t];
          const float f = __builtin_amdgcn_exp2f(t ? (s1 - st.sum[t - 1]) + (r1 - st.rest[t - 1]) : s1 + r1);
          const int pl_row = 16 * w4 + i16;
          const float x = Act<F16>::ld(
              *reinterpret_cast<const uint16_t*>(xs + chunk_at<8>(t, pl_row >> 3) + (pl_row & 7) * 2));
          const float ux = st.dt[t] * x;
          float sum = 0.0f;
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
            const int at = chunk_at<CH>(t, (nt >> 1) * 4 + g4) + (nt & 1) * 8;
            const u32x2_t wb = *reinterpret_cast<const u32x2_t*>(lds.b + at);
            const float vb4[4] = {Act<F16>::lo(wb[0]), Act<F16>::hi(wb[0]), Act<F16>::lo(wb[1]), Act<F16>::hi(wb[1])};
#pragma unroll
            for (int i = 0; i < 4; ++i) S[nt][i] = S[nt][i] * f + ux * vb4[i];
            if constexpr (!STATES) {
              const u32x2_t wc = *reinterpret_cast<const u32x2_t*>(lds.c + at);
              const float vc4[4] = {Act<F16>::lo(wc[0]), Act<F16>::hi(wc[0]), Act<F16>::lo(wc[1]), Act<F16>::hi(wc[1])};
              // (columns behind the state's end would make 0 times infinity)
              if (16 * nt + 4 * g4 < a.N) {
#pragma unroll
                for (int i = 0; i < 4; ++i) sum = __builtin_fmaf(S[nt][i], vc4[i], sum);
              }
            }
          }
          if constexpr (!STATES) {
            sum += __shfl_xor(sum, 16);
            sum += __shfl_xor(sum, 32);
            if (a.d) sum = __builtin_fmaf(skip, x, sum);
            if (g4 == 0 && row0 + pl_row < a.hd)
              (static_cast<uint16_t*>(a.out.p) + b * a.out.bs + (t0 + t) * a.out.ts + h * a.out.hs)[row0 + pl_row] =
                  Act<F16>::st(sum);
          }
        }
      }
      begun = true;
    }
    if (more) {
      if (steps_wave) steps(t0 + kChunk, (ck + 1) & 1);
      lds_barrier();  // every wave is done with this chunk
      stage();
      lds_barrier();
    }
  }

  if (!live) return;
  if (STATES) {
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) *seg_state(seg, nt) = S[nt];
    if (steps_wave && lane == 0) seg_decays[head * pl.segs + seg] = __builtin_amdgcn_exp2f(static_cast<float>(seg_sum));
  } else if (a.s_out && pool >= 0 && p_row < a.hd && seg == (len > 0 ? (len - 1) / seg_len : 0)) {
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
      if (16 * nt + 4 * g4 < a.N) *reinterpret_cast<f32x4_t*>(a.s_out + state0 + 16 * nt) = S[nt];
  }
}

// ------------------------------------------------------------------ launches

int chunk_steps(int N) { return N <= 32 ? 1 : N <= 64 ? 2 : N <= 128 ? 4 : 8; }

constexpr int kFewMost = 16;      // tokens that the walk takes
constexpr int kFullGrid = 512;    // workgroups that fill the CUs

struct ScanPlan {
  ChunkPlan ck;
  int slots, nk;
  size_t states;  // floats of the segments' states
  size_t bytes;
};

ScanPlan scan_plan(const ScanArgs& a) {
  ScanPlan p{};
  ChunkPlan& c = p.ck;
  c.tiles = (a.hd + kTileRows - 1) / kTileRows;
  const int items = a.rep * c.tiles;
  p.slots = items > 1 ? 2 : 1;
  p.nk = chunk_steps(a.N);
  c.pairs = (items + p.slots - 1) / p.slots;
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

template <bool F16, int NK, int SLOTS>
hipError_t scan_chunks(const ScanArgs& a, ScanPlan p, float* ws, hipStream_t stream) {
  ChunkPlan& c = p.ck;
  c.keep_first = a.s_in && a.s_in == a.s_out;
  float* decays = ws + p.states;
  for (int pass = c.segs > 1 ? 0 : 1; pass < 2; ++pass) {
    c.first_segs = pass ? c.segs : c.segs - 1;
    c.total = static_cast<uint32_t>(static_cast<int64_t>(a.B) * c.first_segs * a.groups * c.pairs);
    c.run = std::max(1, std::min<int>(c.pairs, c.total / 64));
    const uint32_t round = 8 * c.run;
    const dim3 grid((c.total + round - 1) / round * round), wg(kSlotThreads * SLOTS);
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

bool scan_in_chunks(const ScanArgs& a) { return a.L > kFewMost; }

}  // namespace

size_t scan_workspace(const ScanArgs& a) { return scan_in_chunks(a) ? scan_plan(a).bytes : 0; }

bool scan_fits(const ScanArgs& a) {
  // (a part of the walk has at least 4 rows; workgroups of chunks have 512
  // threads, as many as items, segments and a round to fill at most)
  return static_cast<int64_t>(a.B) * a.nh * ((a.hd + 3) / 4) <= max_blocks(kFewThreads) &&
         static_cast<int64_t>(a.B) * a.nh * ((a.hd + kTileRows - 1) / kTileRows) + kFullGrid + 8 * 65536 * 4 <=
             max_blocks(2 * kSlotThreads);
}

hipError_t launch_scan(const ScanArgs& a, bool f16, void* ws, hipStream_t stream) {
  if (a.B == 0) return hipSuccess;
  if (scan_in_chunks(a))
    return f16 ? scan_chunks<true>(a, static_cast<float*>(ws), stream)
               : scan_chunks<false>(a, static_cast<float*>(ws), stream);
  return f16 ? scan_few<true>(a, stream) : scan_few<false>(a, stream);
}

}  // namespace fmx
