// fmx_cache_attn.hip -- attention of a batch over a shared prefix and its
// sequences' own caches, and over own caches with the keys' weights added up
// (no counterpart in the reference; mx::fast::scaled_dot_product_attention,
// server/src/model.cpp:879-882, at their place).
//
// The rows of one kv head (its query heads of every query) are taken
// together, so keys and values are read once for all of them: the prefix for
// the rows of the whole batch, a cache slot for the rows of its sequence.
// Long axes of keys are cut into pieces; a piece leaves, for each row, the
// largest score m, the sum l of exp2(t - m) and the values' sum o with the
// same weights (t: score times log2 e), all fp32, and attn_join_kernel adds
// the pieces of a row: sum of exp2(m_i - M) o_i over that of exp2(m_i - M) l_i.
//
//   attn_narrow_kernel   tiles of 16 or 32 rows, keys straight to registers
//   attn_wide_kernel     tiles of 128 rows, keys and values staged in LDS
//   attn_both_kernel     both in one grid
//   attn_join_kernel     a row's pieces to its output; weights of the keys
//                        from stored scores
//   attn_weights_kernel, attn_weights_sum_kernel
//                        weights of the keys of many rows, scores formed again
#include <algorithm>

#include "fmx_cache_kernels.hpp"
#include "fmx_dev.hpp"

namespace fmx {

namespace {

constexpr int kThreads = 256;
constexpr int kWaves = kThreads / kWave;
constexpr int kStep = 32;                // keys of a wave's step
constexpr int kPiece = kPieceKeys;
static_assert(kPiece == kStep * kWaves, "a unit is one step of every wave");
// up to so many rows of a kv head run in narrow tiles
constexpr int kNarrowRows = 32;
constexpr float kLog2e = 1.44269504088896340736f;
constexpr float kLn2 = 0.69314718055994530942f;

__device__ inline float neg_inf() { return -__builtin_huge_valf(); }

// The fragments are in registers from here on: a load still counted as on its
// way at a loop's entry would make every round wait for the loads that it has
// just issued.
template <typename T, int N>
__device__ inline void settle(T (&f)[N]) {
#pragma unroll
  for (int i = 0; i < N; ++i) {
    u32x4_t w = __builtin_bit_cast(u32x4_t, f[i]);
    asm volatile("" : "+v"(w));
    f[i] = __builtin_bit_cast(T, w);
  }
}

// 16 or 4 bytes of every lane straight to LDS, lane after lane from `to` on
__device__ inline void load_to_lds16(const void* from, void* to) {
  __builtin_amdgcn_global_load_lds(from, (__attribute__((address_space(3))) void*)to, 16, 0, 0);
}
__device__ inline void load_to_lds4(const void* from, void* to) {
  __builtin_amdgcn_global_load_lds(from, (__attribute__((address_space(3))) void*)to, 4, 0, 0);
}

// of the four lanes i16 + 16 j: their maximum, their sum, in each
__device__ inline float quad_max(float v) {
  auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  v = fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
  a = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
}
__device__ inline float quad_sum(float v) {
  auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  v = __uint_as_float(a[0]) + __uint_as_float(a[1]);
  a = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return __uint_as_float(a[0]) + __uint_as_float(a[1]);
}

// What a forward's launches agree on.
struct Plan {
  int R;                // rows of a sequence and kv head: L * rep
  // the prefix: rows of all sequences, row b * R + l * rep + (head in group)
  int p_tiles, p_splits;
  int p_keys;           // of a split
  float* p_o;           // [split][nkv][B R][hd]
  float2* p_ml;         // [split][nkv][B R]
  // own keys: o_grid pieces over all sequences, or (wide tiles) o_splits
  // pieces of every row tile's keys, [split][B][nkv][R]
  bool p_wide, o_wide;
  int o_tiles, o_grid, o_splits;
  float* o_o;           // [piece][nkv][R][hd]
  float2* o_ml;         // [piece][nkv][R]
  int2* table;          // [B] (first piece, pieces) of a sequence
  // weights from stored scores: [B][nkv][R][s_ld] scores times log2 e
  float* scores;
  int64_t s_ld;
  float* lse;           // [B, L, nh]: the caller's, or null
  // weights of many rows: ln sum exp by log2 e of [B, nkv, R], and sums over
  // every w_parts-th block of kSumRows rows, [w_parts][B][nkv][S]
  float* lse2;
  float* w_part;
  int w_parts;
  bool direct;          // one piece per row: the wide tiles write the output
};

// Pieces of the own keys, found by every workgroup from the device's lengths:
// sequence b has u_b = ceil(keys / kPiece) units and ceil(u_b / c) pieces of c
// units, c the smallest that keeps all pieces within the grid: sum u_b / (grid
// - B) rounded up, or all of the longest possible sequence's. Lengths may
// differ as they like: all pieces but each sequence's last are equally long.
// Returns the sequence of piece w (-1: none), its piece number in *k and c in
// *units; workgroup 0 leaves the table.
struct PieceLds {
  uint32_t tmp[kWaves + 1];
  int seq, k;
};
__device__ int find_piece(const CacheAttnArgs& a, const Plan& pl, int w, bool write_table, int* k, int* units,
                          PieceLds& s) {
  const int tid = threadIdx.x;
  auto units_of = [&](int b) {
    const int64_t n = own_keys(a, seq_slot(a.slots, a.n_slots, b), a.offs[b], a.L - 1);
    return static_cast<uint32_t>((n + kPiece - 1) / kPiece);
  };
  uint32_t mine = 0;
  for (int b = tid; b < a.B; b += kThreads) mine += units_of(b);
  uint32_t total;
  block_exclusive_scan<kThreads>(mine, s.tmp, &total);
  const uint32_t room = static_cast<uint32_t>(pl.o_grid - a.B);
  const uint32_t c = max(1u, piece_units(total, room, a.S));
  if (tid == 0) s.seq = -1;
  uint32_t base = 0;
  for (int b0 = 0; b0 < a.B; b0 += kThreads) {
    const int b = b0 + tid;
    const uint32_t n = b < a.B ? (units_of(b) + c - 1) / c : 0;
    uint32_t sum;
    const uint32_t first = base + block_exclusive_scan<kThreads>(n, s.tmp, &sum);
    if (static_cast<uint32_t>(w) >= first && static_cast<uint32_t>(w) < first + n) {
      s.seq = b;
      s.k = w - static_cast<int>(first);
    }
    if (write_table && b < a.B) pl.table[b] = make_int2(static_cast<int>(first), static_cast<int>(n));
    base += sum;
  }
  __syncthreads();
  *k = s.k;
  *units = static_cast<int>(c);
  return s.seq;
}

// ------------------------------------------------------------------ narrow tiles
//
// One workgroup per (16 RT rows, piece of keys); each of its four waves takes
// every fourth step of 32 keys, and they join in LDS at the end.
//
// S^T = K Q^T by v_mfma_f32_16x16x32: a lane's A operand is 16 bytes of key
// i16 (+ 16), its B operand the row i16's query, which stays in registers.
// The result leaves lane (i16, j) with row i16's scores of keys 4j + r (+ 16):
// after exp2 the B operand of O^T += V^T P^T as it stands, if key 4j + r is
// slot 8j + r and key 16 + 4j + r slot 8j + 4 + r of the 32. Its A operand
// wants the same keys' values of one dimension: a lane loads VPL consecutive
// dimensions of each of its eight keys (1 KB of four rows per load of a
// wave), and pairs of keys are put together by v_perm. Nothing passes through
// LDS and no load is narrower than a cache line's half.
//
// The weights go into the value product as two numbers of the inputs' type,
// their leading bits and the rest (2^-16 or 2^-22 of a weight is lost at most):
// only the output is rounded. The matrix cores have time to spare here.
//
// Bound by HBM: every key and value is read once, 512 bytes (heads of 128) for
// 16 bytes of partial results per 128 keys and row. 16 sequences of up to
// 16001 keys, 32 heads over 4, fp16,
// scores stored: 59 us for 271 MB, 4.6 TB/s (6.2 is a large read's); one row
// per workgroup and head took 6.6 ms, the same values read for every head and
// queried one after the other. Short calls are bound by the chain of a
// workgroup (a piece's address, its loads, two products): 4 sequences of up to
// 64 keys behind 512 shared ones, 16 kv heads, 5 MB, take 6.7 us.
template <int HD>
struct Narrow {
  static constexpr int KC = HD / 32;            // 32-dimension steps of a score
  static constexpr int DT = HD / 16;            // 16-dimension tiles of the output
  static constexpr int VPL = HD / 16;           // dimensions of a key per lane
  static constexpr int VW = VPL / 2;            // 32-bit words of them
};

template <int RT>
struct NarrowLds {
  float m[kWaves][16 * RT], l[kWaves][16 * RT];
  int left[kWaves];
  PieceLds piece;
};

// where four dimensions from d on of a row's sums lie in LDS (rows one after
// the other: shifted against each other by the row, for the banks)
template <int HD>
__device__ inline f32x4_t* sums_at(float* o, int row, int d) {
  return reinterpret_cast<f32x4_t*>(o + row * HD + ((d >> 2) ^ (row & 7)) * 4);
}

// dimension of A row `row`, tile dt (runs of up to 8 per lane)
template <int HD>
__device__ inline int out_dim(int row, int dt) {
  constexpr int V8 = HD / 16 < 8 ? HD / 16 : 8;
  return dt / V8 * (16 * V8) + row * V8 + dt % V8;
}

typedef uint16_t u16x2_t __attribute__((ext_vector_type(2)));

// the larger exponent field, half by half
template <bool F16>
__device__ inline u16x2_t top_exp(u16x2_t m, uint32_t w) {
  return __builtin_elementwise_max(m, __builtin_bit_cast(u16x2_t, w & (F16 ? 0x7c007c00u : 0x7f807f80u)));
}
template <bool F16>
__device__ inline bool is_top(u16x2_t m) {
  constexpr uint16_t e = F16 ? 0x7c00 : 0x7f80;
  return m[0] == e || m[1] == e;
}

template <bool PAST, typename T>
__device__ inline T load(const T* p) {
  if constexpr (PAST) return __builtin_nontemporal_load(p);
  return *p;
}

// the halves of w that are infinite or NaN made 0
template <bool F16>
__device__ inline uint32_t word_finite(uint32_t w) {
  constexpr uint32_t e = F16 ? 0x7c00u : 0x7f80u;
  if ((w & e) == e) w &= 0xffff0000u;
  if ((w & (e << 16)) == e << 16) w &= 0xffffu;
  return w;
}

// The infinite and NaN values of keys [lo, hi), four dimensions at v, added
// to a row's sums
template <bool F16>
__device__ __attribute__((noinline)) void add_left_out(f32x4_t& acc, const uint16_t* v, int64_t ts, int lo, int hi) {
  for (int k = lo; k < hi; ++k)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float x = Act<F16>::ld(v[k * ts + i]);
      if (!(fabsf(x) < -neg_inf())) acc[i] += x;
    }
}

// PAST: loads go past the caches. ANY: hd may be below HD (chunks behind it
// read as zeros), and the rows of a tile may see different keys (several
// queries per sequence)
template <bool F16, int HD, int RT, bool PAST, bool ANY>
__device__ __attribute__((always_inline)) void narrow_item(const CacheAttnArgs& a, const Plan& pl, int n_prefix,
                                                           int block, float* o0, float* o1,
                                                           NarrowLds<RT>& s) {
  using N = Narrow<HD>;
  constexpr int KC = N::KC, DT = N::DT, VW = N::VW, VPL = N::VPL;
  typedef act8_t<F16> frag_t;
  // exp2's results are kept up to 2^10 for fp16 products, so that its
  // smallest normal number is 2^-24 of the largest weight; bf16 needs none
  constexpr float kBias = F16 ? 10.0f : 0.0f;
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int i16 = lane & 15, j = lane >> 4;

  // ---- the item: rows, keys
  const bool prefix = block < n_prefix;
  const int tiles = prefix ? pl.p_tiles : pl.o_tiles;
  int item = prefix ? block : block - n_prefix;
  const int tile = item % tiles;
  item /= tiles;
  const int g = item % a.nkv;
  const int piece = item / a.nkv;
  int seq = 0, k0, k1;
  const uint16_t* kb;
  const uint16_t* vb;
  int64_t kts, vts;
  int off = 0;
  int64_t slot = 0;
  if (prefix) {
    k0 = piece * pl.p_keys;
    k1 = static_cast<int>(min(a.P, static_cast<int64_t>(k0) + pl.p_keys));
    kb = static_cast<const uint16_t*>(a.kp.p) + g * a.kp.hs;
    vb = static_cast<const uint16_t*>(a.vp.p) + g * a.vp.hs;
    kts = a.kp.ts;
    vts = a.vp.ts;
  } else {
    int k, units;
    seq = find_piece(a, pl, piece, piece == 0 && g == 0 && tile == 0, &k, &units, s.piece);
    if (seq < 0) return;
    seq = __builtin_amdgcn_readfirstlane(seq);
    slot = seq_slot(a.slots, a.n_slots, seq);
    off = a.offs[seq];
    piece_keys(k, units, own_keys(a, slot, off, a.L - 1), &k0, &k1);
    k0 = __builtin_amdgcn_readfirstlane(k0);
    k1 = __builtin_amdgcn_readfirstlane(k1);
    kb = static_cast<const uint16_t*>(a.kc.p) + slot * a.kc.bs + g * a.kc.hs;
    vb = static_cast<const uint16_t*>(a.vc.p) + slot * a.vc.bs + g * a.vc.hs;
    kts = a.kc.ts;
    vts = a.vc.ts;
  }
  const int rows = prefix ? a.B * pl.R : pl.R;
  const int row0 = tile * 16 * RT;

  // ---- queries, and how many keys a row may see
  frag_t qf[RT][KC];
  int limit[RT];
#pragma unroll
  for (int rt = 0; rt < RT; ++rt) {
    const int m = min(row0 + rt * 16 + i16, rows - 1);
    const int b = prefix ? m / pl.R : seq;
    const int r = prefix ? m - b * pl.R : m;
    const int l = r / a.rep, h = g * a.rep + r - l * a.rep;
    const uint16_t* q = static_cast<const uint16_t*>(a.q.p) + b * a.q.bs + l * a.q.ts + h * a.q.hs;
#pragma unroll
    for (int t = 0; t < KC; ++t) {
      u32x4_t w = {0, 0, 0, 0};
      if (!ANY || 32 * t + 8 * j < a.hd) w = *reinterpret_cast<const u32x4_t*>(q + 32 * t + 8 * j);
      qf[rt][t] = __builtin_bit_cast(frag_t, w);
    }
    limit[rt] = prefix ? k1 : static_cast<int>(min(own_keys(a, slot, off, l), static_cast<int64_t>(k1)));
  }
  // keys below this are seen by every row of the tile
  const int all =
      prefix ? k1 : static_cast<int>(min(own_keys(a, slot, off, row0 / a.rep), static_cast<int64_t>(k1)));

  f32x4_t o[RT][DT];
  float mref[RT], lsum[RT];
#pragma unroll
  for (int rt = 0; rt < RT; ++rt) {
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) o[rt][dt] = f32x4_t{0, 0, 0, 0};
    mref[rt] = neg_inf();
    lsum[rt] = 0.0f;
  }
  const float c = a.scale * kLog2e;
  float* sc_out[RT];
#pragma unroll
  for (int rt = 0; rt < RT; ++rt)
    sc_out[rt] = pl.scores && !prefix && row0 + rt * 16 + i16 < rows
                     ? pl.scores + ((static_cast<int64_t>(seq) * a.nkv + g) * pl.R + row0 + rt * 16 + i16) * pl.s_ld
                     : nullptr;

  // rows behind the piece's last are read as its last
  u32x4_t kw[2][KC];
  uint32_t vw[8][VW];
  // (a lane's 64-bit row products are formed once; a step adds a scalar one)
  const int kk0 = k0 + wave * kStep;
  const uint16_t* kp0 = kb + min(kk0 + i16, k1 - 1) * kts + 8 * j;
  const uint16_t* vp0 = vb + min(kk0 + 4 * j, k1 - 1) * vts + (VPL == 4 ? 4 : 8) * i16;
  auto load_k = [&](int kk) {
    const bool whole = kk + kStep <= k1;
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      const uint16_t* p = whole ? kp0 + (kk - kk0 + 16 * x) * kts : kb + min(kk + 16 * x + i16, k1 - 1) * kts + 8 * j;
#pragma unroll
      for (int t = 0; t < KC; ++t)
        if (!ANY || 32 * t + 8 * j < a.hd)
          kw[x][t] = load<PAST>(reinterpret_cast<const u32x4_t*>(p + 32 * t));
        else
          kw[x][t] = u32x4_t{0, 0, 0, 0};
    }
  };
  auto load_v = [&](int kk) {
    const bool whole = kk + kStep <= k1;
#pragma unroll
    for (int sl = 0; sl < 8; ++sl) {
      const int row = 16 * (sl >> 2) + (sl & 3);
      const uint16_t* p = whole ? vp0 + (kk - kk0 + row) * vts
                                : vb + min(kk + row + 4 * j, k1 - 1) * vts + (VPL == 4 ? 4 : 8) * i16;
      if constexpr (VPL == 4) {
        u32x2_t w = {0, 0};
        if (!ANY || 4 * i16 < a.hd) w = load<PAST>(reinterpret_cast<const u32x2_t*>(p));
        vw[sl][0] = w[0];
        vw[sl][1] = w[1];
      } else {
#pragma unroll
        for (int q = 0; q < VPL / 8; ++q) {
          u32x4_t w = {0, 0, 0, 0};
          if (!ANY || 128 * q + 8 * i16 < a.hd)
            w = load<PAST>(reinterpret_cast<const u32x4_t*>(p + 128 * q));
#pragma unroll
          for (int i = 0; i < 4; ++i) vw[sl][4 * q + i] = w[i];
        }
      }
    }
  };
  // A operand of dimension tile dt from words w(slot)
  auto v_frag = [&](int dt, auto&& word) {
    u32x4_t f;
#pragma unroll
    for (int i = 0; i < 4; ++i)
      f[i] = __builtin_amdgcn_perm(word(2 * i + 1, dt / 2), word(2 * i, dt / 2), dt % 2 ? 0x07060302u : 0x05040100u);
    return __builtin_bit_cast(frag_t, f);
  };

  bool left_out = false;
  int kk = kk0;
  if (kk < k1) load_k(kk);
  for (; kk < k1; kk += kPiece) {
    load_v(kk);
    f32x4_t sc[RT][2];
#pragma unroll
    for (int rt = 0; rt < RT; ++rt)
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        sc[rt][x] = f32x4_t{0, 0, 0, 0};
#pragma unroll
        for (int t = 0; t < KC; ++t) sc[rt][x] = mfma16(__builtin_bit_cast(frag_t, kw[x][t]), qf[rt][t], sc[rt][x]);
      }
    if (kk + kPiece < k1) load_k(kk + kPiece);
    const bool part = kk + kStep > all;  // some row does not see all of the step
    frag_t ph[RT], pw[RT];               // weights: their leading bits and the rest
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
      float mt = neg_inf();
#pragma unroll
      for (int x = 0; x < 2; ++x)
#pragma unroll
        for (int r = 0; r < 4; ++r) sc[rt][x][r] *= c;
      if (sc_out[rt]) {
#pragma unroll
        for (int x = 0; x < 2; ++x)
          *reinterpret_cast<f32x4_t*>(sc_out[rt] + kk + 16 * x + 4 * j) = sc[rt][x];
      }
      if (part) {
#pragma unroll
        for (int x = 0; x < 2; ++x)
#pragma unroll
          for (int r = 0; r < 4; ++r)
            if (kk + 16 * x + 4 * j + r >= limit[rt]) sc[rt][x][r] = neg_inf();
      }
#pragma unroll
      for (int x = 0; x < 2; ++x)
#pragma unroll
        for (int r = 0; r < 4; ++r) mt = fmaxf(mt, sc[rt][x][r]);
      mt = quad_max(mt) - kBias;
      if (__any(mt > mref[rt])) {
        const float mn = fmaxf(mt, mref[rt]);
        const float f = __builtin_amdgcn_exp2f(mref[rt] - (mn == neg_inf() ? 0.0f : mn));
        mref[rt] = mn;
        lsum[rt] *= f;
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) o[rt][dt] *= f;
      }
      const float ms = mref[rt] == neg_inf() ? 0.0f : mref[rt];
#pragma unroll
      for (int x = 0; x < 2; ++x)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const float p = __builtin_amdgcn_exp2f(sc[rt][x][r] - ms);
          lsum[rt] += p;
          typedef typename std::conditional<F16, _Float16, __bf16>::type half_t;
          const half_t hi = static_cast<half_t>(p);
          ph[rt][4 * x + r] = hi;
          pw[rt][4 * x + r] = static_cast<half_t>(p - static_cast<float>(hi));
        }
    }
    if (part) {
      // values behind the piece count nothing, whatever they hold
      u16x2_t top = {0, 0};
#pragma unroll
      for (int sl = 0; sl < 8; ++sl) {
        const bool in = kk + 16 * (sl >> 2) + 4 * j + (sl & 3) < k1;
#pragma unroll
        for (int w = 0; w < VW; ++w) {
          vw[sl][w] = in ? vw[sl][w] : 0u;
          if (ANY && a.L > 1) top = top_exp<F16>(top, vw[sl][w]);
        }
      }
      if (ANY && __any(is_top<F16>(top))) {
        // infinite or NaN values that some rows see and others do not, whose
        // weight of 0 makes no 0 of them: left out here, added to the rows
        // that see them at the end
        left_out = true;
#pragma unroll
        for (int sl = 0; sl < 8; ++sl)
#pragma unroll
          for (int w = 0; w < VW; ++w) vw[sl][w] = word_finite<F16>(vw[sl][w]);
      }
    }
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) {
      const frag_t f = v_frag(dt, [&](int sl, int w) { return vw[sl][w]; });
#pragma unroll
      for (int rt = 0; rt < RT; ++rt) {
        o[rt][dt] = mfma16(f, ph[rt], o[rt][dt]);
        o[rt][dt] = mfma16(f, pw[rt], o[rt][dt]);
      }
    }
  }

  if (ANY && lane == 0) s.left[wave] = left_out;
  // ---- the waves' sums together: waves 0 and 1 leave theirs, 2 and 3 add
#pragma unroll
  for (int rt = 0; rt < RT; ++rt) {
    const float l = quad_sum(lsum[rt]);
    if (j == 0) {
      s.m[wave][rt * 16 + i16] = mref[rt];
      s.l[wave][rt * 16 + i16] = l;
    }
  }
  __syncthreads();
#pragma unroll
  for (int rt = 0; rt < RT; ++rt) {
    float m = s.m[0][rt * 16 + i16];
#pragma unroll
    for (int w = 1; w < kWaves; ++w) m = fmaxf(m, s.m[w][rt * 16 + i16]);
    const float f = __builtin_amdgcn_exp2f(mref[rt] - (m == neg_inf() ? 0.0f : m));
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) o[rt][dt] *= f;
  }
  auto leave = [&](bool add) {
#pragma unroll
    for (int rt = 0; rt < RT; ++rt)
#pragma unroll
      for (int r = 0; r < 4; ++r)
#pragma unroll
        for (int d4 = 0; d4 < DT; d4 += 4) {
          f32x4_t* p = sums_at<HD>(wave & 1 ? o1 : o0, rt * 16 + i16, out_dim<HD>(4 * j + r, d4));
          f32x4_t v = {o[rt][d4][r], o[rt][d4 + 1][r], o[rt][d4 + 2][r], o[rt][d4 + 3][r]};
          *p = add ? *p + v : v;
        }
  };
  if (wave < 2) leave(false);
  __syncthreads();
  if (wave >= 2) leave(true);
  __syncthreads();

  const int64_t first = prefix ? (static_cast<int64_t>(piece) * a.nkv + g) * rows + row0
                               : (static_cast<int64_t>(piece) * a.nkv + g) * pl.R + row0;
  const int nr = min(16 * RT, rows - row0);
  float* po = (prefix ? pl.p_o : pl.o_o) + first * a.hd;
  const int h4 = a.hd / 4;
  for (int i = tid; i < nr * h4; i += kThreads) {
    const int r = i / h4, d = (i - r * h4) * 4;
    f32x4_t v = *sums_at<HD>(o0, r, d) + *sums_at<HD>(o1, r, d);
    if (ANY && (s.left[0] | s.left[1] | s.left[2] | s.left[3]))
      add_left_out<F16>(v, vb + d, vts, max(k0, all / kStep * kStep),
                        prefix ? k1
                               : static_cast<int>(min(own_keys(a, slot, off, (row0 + r) / a.rep),
                                                      static_cast<int64_t>(k1))));
    *reinterpret_cast<f32x4_t*>(po + static_cast<int64_t>(i) * 4) = v;
  }
  if (tid < nr) {
    float m = s.m[0][tid];
#pragma unroll
    for (int w = 1; w < kWaves; ++w) m = fmaxf(m, s.m[w][tid]);
    float l = 0.0f;
#pragma unroll
    for (int w = 0; w < kWaves; ++w)
      l += s.l[w][tid] * __builtin_amdgcn_exp2f(s.m[w][tid] - (m == neg_inf() ? 0.0f : m));
    (prefix ? pl.p_ml : pl.o_ml)[first + tid] = make_float2(m, l);
  }
}

template <bool F16, int HD, int RT, bool PAST, bool ANY>
__global__ __launch_bounds__(kThreads) __attribute__((amdgpu_waves_per_eu(2)))
void attn_narrow_kernel(CacheAttnArgs a, Plan pl, int n_prefix) {
  __shared__ __attribute__((aligned(16))) float s_o[2][16 * RT * HD];
  __shared__ NarrowLds<RT> s;
  narrow_item<F16, HD, RT, PAST, ANY>(a, pl, n_prefix, blockIdx.x, s_o[0], s_o[1], s);
}

// ------------------------------------------------------------------ wide tiles
//
// One workgroup per (128 rows, piece of keys): 32 rows per wave, the keys and
// values of KT positions staged in LDS for all four.
//
// S^T = K Q^T and O^T += V^T P^T by v_mfma_f32_32x32x16. Register 8u + 4v + r
// of a lane (row c of the 32, half h) is the score of key 16u + 8v + 4h + r:
// after exp2 the B operand of the value product over those 16 keys, if key 16u
// + 8v + 4h + r is its slot 8h + 4v + r. Its A operand is the same keys' values of
// one dimension, which two transposing LDS reads of four keys each deliver.
// Keys and values come to LDS past the registers, in two buffers: the next
// positions are on their way while these are multiplied.
//
// The weights go into the value product as two numbers of the inputs' type, as
// in narrow tiles, so that a row's precision does not hang on how many rows its
// call has. That is half of all matrix work again (59 -> 71 us for the prompt
// below, 126 -> 145 us a call of 128 sequences behind 32768 positions; the
// figures given for choices further down are from before), but one number
// alone, off by up to 2^-8 or 2^-11 of the weight, moves a row with one
// dominating key by a step of the output. The maximum is only raised when a
// score lies more than kLazy above it: the weights reach 2^kLazy times kBias'
// 2^8 at most, in fp16 2^14 of 65504.
//
// Bound by a wave's own chain: by the cycle counter a step of 64 keys took it
// about 3000 cycles before the second product (issuing the next loads 500,
// scores 900, maximum 300, weights and values 1300, of which the matrix cores
// worked 1000), and a tile some 14000 before its first and after its last step
// (queries from HBM, outputs). The longest tile of a causal grid alone is two
// thirds of the kernel's time; keys dealt to two halves of a workgroup, or long
// and short tiles one after the other, gained nothing. A prompt of 2000 tokens,
// 32 heads over 4: 71 us, 0.46 PFLOP/s of the causal half (1.4 is a large
// library product's).
constexpr int kWideRows = 32 * kWaves;
constexpr int kCus = 256;
constexpr float kLazy = 6.0f;

__device__ inline f32x16_t mfma32(const bf16x8_t& a, const bf16x8_t& b, const f32x16_t& c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
}
__device__ inline f32x16_t mfma32(const f16x8_t& a, const f16x8_t& b, const f32x16_t& c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
}

// of the two lanes c and c + 32
__device__ inline float half_max(float v) {
  const auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
}
__device__ inline float half_sum(float v) {
  const auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return __uint_as_float(a[0]) + __uint_as_float(a[1]);
}

// what a wide launch goes over: pairs (of keys: piece, kv head [, sequence])
// times row tiles. Blocks go to the 8 XCDs in turn; with the pairs a divisor
// or a multiple of 8 a pair's tiles meet in one L2.
struct WideGrid {
  bool prefix;
  int pairs, padded, tiles, splits;
};

// Arrays of their own, so that the compiler can tell the buffers that loads are
// on their way to from those being read (it would wait for the loads before
// every read otherwise).
template <int HD>
struct WideLds {
  uint16_t *k0, *k1, *v0, *v1;  // KT * HD each
  int* left;
};
#define FMX_WIDE_LDS(HD, KT, name)                                             \
  __shared__ __attribute__((aligned(16))) uint16_t name##_k0[KT * HD];         \
  __shared__ __attribute__((aligned(16))) uint16_t name##_k1[KT * HD];         \
  __shared__ __attribute__((aligned(16))) uint16_t name##_v0[KT * HD];         \
  __shared__ __attribute__((aligned(16))) uint16_t name##_v1[KT * HD];         \
  __shared__ int name##_left;                                                  \
  const WideLds<HD> name{name##_k0, name##_k1, name##_v0, name##_v1, &name##_left}

// Rows of both arrays lie one after the other, their 16-byte chunks in an
// order of the row's own, so that the lanes that LDS serves together fall on
// different banks: a key's chunk c at c ^ swz_k (16 rows' same chunk), a
// value's 32-byte segment at segment ^ swz_v (four rows' two segments).
template <int HD>
__device__ inline int swz_k(int row) {
  return HD == 64 ? row >> 1 & 7 : row & 15;
}
template <int HD>
__device__ inline int swz_v(int row) {
  return HD == 64 ? row & 2 : (row & 3) * 2;
}

typedef short s16x4_t __attribute__((ext_vector_type(4)));
// 4 x 16 elements across 16 lanes: lane i gets element i % 4 of the lanes i / 4 + 4 e
__device__ inline s16x4_t lds_read_tr(const uint16_t* p) {
  return __builtin_amdgcn_ds_read_tr16_b64_v4i16(
      (__attribute__((address_space(3))) s16x4_t*)const_cast<uint16_t*>(p));
}

template <bool F16, int HD, int KT, bool ANY>
__device__ __attribute__((always_inline)) void wide_item(const CacheAttnArgs& a, const Plan& pl, const WideGrid& wg,
                                                         int block, const WideLds<HD>& sh) {
  typedef act8_t<F16> frag_t;
  constexpr int KS = HD / 16;              // score steps
  constexpr int DT = HD / 32;              // dimension tiles
  constexpr int kRowChunks = HD / 8;
  constexpr int kDmaRows = kWave / kRowChunks;             // rows of a wave's load
  constexpr int kWaveRows = KT / kWaves;
  constexpr int NL = kWaveRows / kDmaRows;                 // loads of a wave per array
  constexpr float kBias = F16 ? 8.0f : 0.0f;
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int c32 = lane & 31, h2 = lane >> 5;

  // ---- the item
  const int pair = block % wg.padded;
  if (pair >= wg.pairs || block >= wg.padded * wg.tiles) return;
  // Rows that see the most keys first; of the tiles that one round of the CUs
  // takes, every other round's in reverse, so that a CU's tiles are long and
  // short ones.
  int tile = block / wg.padded;
  {
    const int per = max(kCus / wg.padded, 1), round = tile / per;
    if (round & 1) tile = round * per + min(per, wg.tiles - round * per) - 1 - (tile - round * per);
  }
  tile = wg.tiles - 1 - tile;
  const int g = pair % a.nkv;
  const int split = wg.prefix ? pair / a.nkv : pair / a.nkv % wg.splits;
  const int seq = wg.prefix ? 0 : pair / a.nkv / wg.splits;
  const int rows = wg.prefix ? a.B * pl.R : pl.R;
  const int row0 = tile * kWideRows;
  int64_t slot = 0;
  int off = 0, k0, k1, all;
  const uint16_t* kb;
  const uint16_t* vb;
  int64_t kts, vts;
  if (wg.prefix) {
    k0 = split * pl.p_keys;
    k1 = static_cast<int>(min(a.P, static_cast<int64_t>(k0) + pl.p_keys));
    all = k1;
    kb = static_cast<const uint16_t*>(a.kp.p) + g * a.kp.hs;
    vb = static_cast<const uint16_t*>(a.vp.p) + g * a.vp.hs;
    kts = a.kp.ts;
    vts = a.vp.ts;
  } else {
    slot = seq_slot(a.slots, a.n_slots, seq);
    off = a.offs[seq];
    const int n = static_cast<int>(own_keys(a, slot, off, (min(row0 + kWideRows, rows) - 1) / a.rep));
    const int per = (n + wg.splits * KT - 1) / (wg.splits * KT) * KT;
    k0 = min(split * per, n);
    k1 = min(k0 + per, n);
    all = min(k1, static_cast<int>(own_keys(a, slot, off, row0 / a.rep)));
    kb = static_cast<const uint16_t*>(a.kc.p) + (slot < 0 ? 0 : slot) * a.kc.bs + g * a.kc.hs;
    vb = static_cast<const uint16_t*>(a.vc.p) + (slot < 0 ? 0 : slot) * a.vc.bs + g * a.vc.hs;
    kts = a.kc.ts;
    vts = a.vc.ts;
  }
  k0 = __builtin_amdgcn_readfirstlane(k0);
  k1 = __builtin_amdgcn_readfirstlane(k1);
  all = __builtin_amdgcn_readfirstlane(all);
  if (ANY && tid == 0) *sh.left = 0;

  // ---- this lane's row
  const int m = row0 + wave * 32 + c32;
  const int mr = min(m, rows - 1);
  const int b = wg.prefix ? mr / pl.R : seq;
  const int r = wg.prefix ? mr - b * pl.R : mr;
  const int l = r / a.rep, h = g * a.rep + r - l * a.rep;
  const int limit = wg.prefix ? k1 : min(k1, static_cast<int>(own_keys(a, slot, off, l)));
  // of the wave's rows: the fewest and the most keys one sees
  const int w_all = wg.prefix ? k1 : __builtin_amdgcn_readfirstlane(limit);
  const int w_end = wg.prefix ? k1 : __builtin_amdgcn_readlane(limit, 31);
  frag_t qf[KS];
  {
    const uint16_t* q = static_cast<const uint16_t*>(a.q.p) + b * a.q.bs + l * a.q.ts + h * a.q.hs;
#pragma unroll
    for (int t = 0; t < KS; ++t) {
      u32x4_t w = {0, 0, 0, 0};
      if (!ANY || 16 * t + 8 * h2 < a.hd) w = *reinterpret_cast<const u32x4_t*>(q + 16 * t + 8 * h2);
      qf[t] = __builtin_bit_cast(frag_t, w);
    }
  }

  // ---- staging: straight to LDS, a quarter of both arrays' rows per wave
  const int lr = lane / kRowChunks, lc = lane % kRowChunks;
  auto k_chunk = [&](int i) { return lc ^ swz_k<HD>(wave * kWaveRows + i * kDmaRows + lr); };
  auto v_chunk = [&](int i) { return lc ^ swz_v<HD>(wave * kWaveRows + i * kDmaRows + lr) << 1; };
  uint32_t ko[NL], vo[NL];  // byte offsets from the first position's row
#pragma unroll
  for (int i = 0; i < NL; ++i) {
    const uint32_t row = wave * kWaveRows + i * kDmaRows + lr;
    ko[i] = (row * static_cast<uint32_t>(kts) + 8 * k_chunk(i)) * 2;
    vo[i] = (row * static_cast<uint32_t>(vts) + 8 * v_chunk(i)) * 2;
  }
  auto dma = [&](const uint16_t* base, int64_t ts, const uint32_t (&off_b)[NL], bool keys, int kt, uint16_t* to) {
    const uint8_t* at = reinterpret_cast<const uint8_t*>(base + kt * ts);
    if (kt + KT <= k1 && (!ANY || a.hd == HD)) {
#pragma unroll
      for (int i = 0; i < NL; ++i) load_to_lds16(at + off_b[i], to + (wave * kWaveRows + i * kDmaRows) * HD);
      return;
    }
#pragma nounroll
    for (int i = 0; i < NL; ++i) {
      const int row = wave * kWaveRows + i * kDmaRows + lr, ch = keys ? k_chunk(i) : v_chunk(i);
      // rows behind the piece's last are read as its last
      const uint32_t o = (static_cast<uint32_t>(min(row, k1 - 1 - kt)) * static_cast<uint32_t>(ts) + 8 * ch) * 2;
      if (!ANY || 8 * ch < a.hd) load_to_lds16(at + o, to + (wave * kWaveRows + i * kDmaRows) * HD);
    }
  };
  auto load_k = [&](int kt, int buf) { dma(kb, kts, ko, true, kt, buf ? sh.k1 : sh.k0); };
  auto load_v = [&](int kt, int buf) { dma(vb, vts, vo, false, kt, buf ? sh.v1 : sh.v0); };
  // Values behind the piece count nothing, whatever they hold; infinite and
  // NaN ones that not all rows see are left out and added at the end.
  auto clean_v = [&](int kt, int buf) {
    for (int x = tid; x < KT * kRowChunks; x += kThreads) {
      u32x4_t* at = reinterpret_cast<u32x4_t*>(buf ? sh.v1 : sh.v0) + x;
      u32x4_t w = *at;
      u16x2_t top = {0, 0};
      const bool in = kt + x / kRowChunks < k1;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        w[i] = in ? w[i] : 0u;
        if (a.L > 1) top = top_exp<F16>(top, w[i]);
      }
      const bool bad = is_top<F16>(top);
      if (bad) {
        *sh.left = 1;
#pragma unroll
        for (int i = 0; i < 4; ++i) w[i] = word_finite<F16>(w[i]);
      }
      if (bad || !in) *at = w;
    }
    __syncthreads();
  };

  // ---- operands in LDS, in elements from a buffer's start
  int ka[KS], va[DT];
#pragma unroll
  for (int t = 0; t < KS; ++t) ka[t] = c32 * HD + ((2 * t + h2) ^ swz_k<HD>(c32)) * 8;
  {
    const int row = 4 * h2 + (lane & 15) / 4;
#pragma unroll
    for (int dt = 0; dt < DT; ++dt)
      va[dt] = row * HD + ((2 * dt + (lane >> 4 & 1)) ^ swz_v<HD>(row)) * 16 + (lane & 3) * 4;
  }

  f32x16_t o[DT];
#pragma unroll
  for (int dt = 0; dt < DT; ++dt)
#pragma unroll
    for (int i = 0; i < 16; ++i) o[dt][i] = 0.0f;
  float mref = neg_inf(), lsum = 0.0f;
  const float sc = a.scale * kLog2e;

  // operands from LDS: of score step t, and of dimension tile dt with 16 keys,
  // of part x (32) of the keys
  auto k_frag = [&](int t, int x, int buf) {
    return *reinterpret_cast<const frag_t*>((buf ? sh.k1 : sh.k0) + ka[t] + 32 * x * HD);
  };
  auto v_frag = [&](int t, int dt, int x, int buf) {
    typedef short s16x8_t __attribute__((ext_vector_type(8)));
    const uint16_t* v = (buf ? sh.v1 : sh.v0) + va[dt] + (32 * x + 16 * t) * HD;
    const s16x4_t lo = lds_read_tr(v), hi = lds_read_tr(v + 8 * HD);
    const s16x8_t w = __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
    return __builtin_bit_cast(frag_t, w);
  };
  auto scores = [&](auto&& frag) {
    f32x16_t s;
#pragma unroll
    for (int i = 0; i < 16; ++i) s[i] = 0.0f;
#pragma unroll
    for (int t = 0; t < KS; ++t) s = mfma32(frag(t), qf[t], s);
    return s;
  };
  // those that the row sees, and the maximum raised to them
  auto raise = [&](f32x16_t& s, int kx) {
    if (kx + 32 > w_all) {
#pragma unroll
      for (int i = 0; i < 16; ++i)
        if (kx + 8 * (i >> 2) + 4 * h2 + (i & 3) >= limit) s[i] = neg_inf();
    }
    float mt = s[0];
#pragma unroll
    for (int i = 1; i < 16; ++i) mt = fmaxf(mt, s[i]);
    mt = half_max(mt) * sc - kBias;
    if (__any(mt > mref + kLazy)) {
      const float mn = fmaxf(mt, mref);
      const float f = __builtin_amdgcn_exp2f(mref - (mn == neg_inf() ? 0.0f : mn));
      mref = mn;
      lsum *= f;
#pragma unroll
      for (int dt = 0; dt < DT; ++dt) o[dt] *= f;
    }
  };
  // the half's weights, and the values' sums with them
  auto values = [&](const f32x16_t& s, auto&& frag) {
    const float ms = mref == neg_inf() ? 0.0f : mref;
    float ls[2] = {0.0f, 0.0f};
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      frag_t ph, pw;  // their leading bits and the rest
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float p = __builtin_amdgcn_exp2f(__builtin_fmaf(s[8 * t + i], sc, -ms));
        ls[i & 1] += p;
        typedef typename std::conditional<F16, _Float16, __bf16>::type half_t;
        const half_t hi = static_cast<half_t>(p);
        ph[i] = hi;
        pw[i] = static_cast<half_t>(p - static_cast<float>(hi));
      }
      if constexpr (KT == 32) {
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) {
          const frag_t f = frag(t, dt);
          o[dt] = mfma32(f, ph, o[dt]);
          o[dt] = mfma32(f, pw, o[dt]);
        }
      } else {  // (no product waits for the one before it)
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) o[dt] = mfma32(frag(t, dt), ph, o[dt]);
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) o[dt] = mfma32(frag(t, dt), pw, o[dt]);
      }
    }
    lsum += ls[0] + ls[1];
  };
  // The keys at kt, in buffers buf. With 64 of them, the second 32's scores are
  // formed among the first's exponentials, so that a wave's matrix and vector
  // instructions overlap (the scheduler is told to deal them out in turn), and
  // operands are read before the branch ahead of their use (read there, a
  // product each time waits for LDS: 65 us for a prompt of 2000 tokens, 59 so).
  // With 32 there are no registers for that.
  auto step = [&](int kt, int buf) {
    // these keys and values have landed, and every wave is done with the
    // other buffers
    wait_vmcnt0();
    wait_lgkmcnt0();
    lds_dma_barrier();
    if (kt + KT < k1) {
      load_k(kt + KT, buf ^ 1);
      load_v(kt + KT, buf ^ 1);
    }
    if (kt + KT > all) clean_v(kt, buf);
    if (kt >= w_end) return;
    if constexpr (KT == 32) {
      f32x16_t s0 = scores([&](int t) { return k_frag(t, 0, buf); });
      raise(s0, kt);
      values(s0, [&](int t, int dt) { return v_frag(t, dt, 0, buf); });
    } else {
      frag_t kf[2][KS], vf[2][2][DT];
      auto read_k = [&](int x) {
#pragma unroll
        for (int t = 0; t < KS; ++t) kf[x][t] = k_frag(t, x, buf);
      };
      auto read_v = [&](int x) {
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
          for (int dt = 0; dt < DT; ++dt) vf[x][t][dt] = v_frag(t, dt, x, buf);
      };
      read_k(0);
      f32x16_t s0 = scores([&](int t) { return kf[0][t]; });
      read_k(1);
      asm volatile("" ::: "memory");  // (not to be moved behind the branch)
      raise(s0, kt);
      read_v(0);
      f32x16_t s1 = scores([&](int t) { return kf[1][t]; });
      values(s0, [&](int t, int dt) { return vf[0][t][dt]; });
      __builtin_amdgcn_sched_group_barrier(0x100, 4 * DT, 0);  // LDS reads
#pragma unroll
      for (int i = 0; i < KS; ++i) {
        __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);  // a matrix instruction
        __builtin_amdgcn_sched_group_barrier(0x002, 10, 0);  // vector ones
      }
#pragma unroll
      for (int i = 0; i < 4 * DT; ++i) {
        __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
        __builtin_amdgcn_sched_group_barrier(0x002, 3, 0);
      }
      read_v(1);
      asm volatile("" ::: "memory");
      raise(s1, kt + 32);
      values(s1, [&](int t, int dt) { return vf[1][t][dt]; });
    }
  };

  if (ANY && a.hd < HD) {  // chunks behind the heads' end, which no load writes
    for (uint16_t* buf : {sh.k0, sh.k1, sh.v0, sh.v1})
      for (int i = tid; i < KT * kRowChunks; i += kThreads)
        reinterpret_cast<u32x4_t*>(buf)[i] = u32x4_t{0, 0, 0, 0};
    __syncthreads();
  }
  if (k0 < k1) {
    load_k(k0, 0);
    load_v(k0, 0);
  }
  settle(qf);
  for (int kt = k0; kt < k1;) {
    step(kt, 0);
    kt += KT;
    if (kt >= k1) break;
    step(kt, 1);
    kt += KT;
  }
  __syncthreads();

  if (m >= rows) return;
  if (ANY && *sh.left) {
    const int lo = max(k0, k0 + (max(all, k0) - k0) / KT * KT);
#pragma unroll
    for (int dt = 0; dt < DT; ++dt)
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const int d = 32 * dt + 8 * q + 4 * h2;
        if (d >= a.hd) continue;
        f32x4_t v = {o[dt][4 * q], o[dt][4 * q + 1], o[dt][4 * q + 2], o[dt][4 * q + 3]};
        add_left_out<F16>(v, vb + d, vts, lo, limit);
#pragma unroll
        for (int i = 0; i < 4; ++i) o[dt][4 * q + i] = v[i];
      }
  }
  const float z = half_sum(lsum);
  if (pl.direct) {
    const float inv = z == 0.0f ? 0.0f : 1.0f / z;
    uint16_t* out = static_cast<uint16_t*>(a.out.p) + b * a.out.bs + l * a.out.ts + h * a.out.hs;
#pragma unroll
    for (int dt = 0; dt < DT; ++dt)
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const int d = 32 * dt + 8 * q + 4 * h2;
        u32x2_t w;
#pragma unroll
        for (int i = 0; i < 2; ++i)
          w[i] = Act<F16>::st(o[dt][4 * q + 2 * i] * inv) |
                 static_cast<uint32_t>(Act<F16>::st(o[dt][4 * q + 2 * i + 1] * inv)) << 16;
        if (!ANY || d < a.hd) *reinterpret_cast<u32x2_t*>(out + d) = w;
      }
    if (h2 == 0) {
      const float l2 = z == 0.0f ? neg_inf() : mref + __log2f(z);
      if (pl.lse) pl.lse[(static_cast<int64_t>(b) * a.L + l) * a.nh + h] = l2 * kLn2;
      if (pl.lse2) pl.lse2[(static_cast<int64_t>(b) * a.nkv + g) * pl.R + r] = l2;
    }
    return;
  }
  const int64_t at = wg.prefix ? (static_cast<int64_t>(split) * a.nkv + g) * rows + m
                               : ((static_cast<int64_t>(split) * a.B + seq) * a.nkv + g) * pl.R + m;
  float* po = (wg.prefix ? pl.p_o : pl.o_o) + at * a.hd;
#pragma unroll
  for (int dt = 0; dt < DT; ++dt)
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const int d = 32 * dt + 8 * q + 4 * h2;
      if (!ANY || d < a.hd)
        *reinterpret_cast<f32x4_t*>(po + d) =
            f32x4_t{o[dt][4 * q], o[dt][4 * q + 1], o[dt][4 * q + 2], o[dt][4 * q + 3]};
    }
  if (h2 == 0) (wg.prefix ? pl.p_ml : pl.o_ml)[at] = make_float2(mref, z);
}

// keys of a step: 64 (a prompt of 2000 tokens took 64.5 us so and 73 with 32),
// beyond heads of 128 as many as registers hold operands of
template <bool F16, int HD, bool ANY>
__global__ __launch_bounds__(kThreads) __attribute__((amdgpu_waves_per_eu(HD > 128 ? 1 : 2)))
void attn_wide_kernel(CacheAttnArgs a, Plan pl, WideGrid pg, WideGrid og, int n_prefix) {
  constexpr int KT = HD > 128 ? 32 : 64;
  FMX_WIDE_LDS(HD, KT, s);
  // (the prefix's blocks, then the own keys')
  const bool prefix = static_cast<int>(blockIdx.x) < n_prefix;
  wide_item<F16, HD, KT, ANY>(a, pl, prefix ? pg : og, prefix ? blockIdx.x : blockIdx.x - n_prefix, s);
}

// A prefix in wide tiles and own keys in narrow ones in one grid: the former
// keep the matrix cores busy, the latter HBM, as workgroups end at different
// times. With 32 keys per step both fit three times on a CU (narrow tiles of
// two row sets do not: then 64 keys, twice). 128 sequences behind 32768 shared
// positions: 90 + 65 us as two grids, 116 us so; 140 us with 64 keys.
template <bool F16, int HD, int RT, bool PAST, bool ANY>
__global__ __launch_bounds__(kThreads) __attribute__((amdgpu_waves_per_eu(RT == 1 ? 3 : 2)))
void attn_both_kernel(CacheAttnArgs a, Plan pl, WideGrid wg, int n_wide, int n_narrow) {
  constexpr int KT = RT == 1 ? 32 : 64;
  FMX_WIDE_LDS(HD, KT, s);
  static_assert(16 * RT * HD * 4 <= KT * HD * 2 && sizeof(NarrowLds<RT>) <= KT * HD * 2, "narrow tiles' LDS");
  const int base = (n_wide + 7) / 8 * 8;
  if (static_cast<int>(blockIdx.x) < base) {
    if (static_cast<int>(blockIdx.x) < n_wide) wide_item<F16, HD, KT, ANY>(a, pl, wg, blockIdx.x, s);
  } else {
    if (static_cast<int>(blockIdx.x) - base < n_narrow)
      narrow_item<F16, HD, RT, PAST, ANY>(a, pl, 0, blockIdx.x - base, reinterpret_cast<float*>(s.k0),
                                    reinterpret_cast<float*>(s.k1), *reinterpret_cast<NarrowLds<RT>*>(s.v0));
  }
}

// ------------------------------------------------------------------ join

// (m, l) of piece i of a row: the prefix's splits first, then its own pieces
struct RowPieces {
  const CacheAttnArgs& a;
  const Plan& pl;
  int64_t p_at, o_at, p_stride, o_stride;  // rows
  int np, n;
  __device__ RowPieces(const CacheAttnArgs& a_, const Plan& pl_, int b, int g, int r) : a(a_), pl(pl_) {
    p_stride = static_cast<int64_t>(a.nkv) * a.B * pl.R;
    o_stride = static_cast<int64_t>(a.nkv) * pl.R;
    np = pl.p_splits;
    p_at = (static_cast<int64_t>(g) * a.B + b) * pl.R + r;
    int2 t = make_int2(0, 0);
    if (pl.o_wide) {
      t = make_int2(b, pl.o_splits);
    } else if (pl.o_grid) {
      t = pl.table[b];
    }
    o_at = t.x * o_stride + static_cast<int64_t>(g) * pl.R + r;
    if (pl.o_wide) o_stride *= a.B;
    n = np + t.y;
  }
  __device__ float2 ml(int i) const {
    return i < np ? pl.p_ml[p_at + i * p_stride] : pl.o_ml[o_at + (i - np) * o_stride];
  }
  __device__ const float* o(int i) const {
    return (i < np ? pl.p_o + (p_at + i * p_stride) * a.hd : pl.o_o + (o_at + (i - np) * o_stride) * a.hd);
  }
};

constexpr int kWeightKeys = 1024;  // of a weights workgroup: four per thread
constexpr int kWeightAhead = 8;    // rows whose scores are loaded ahead

// M and 1 / sum of a row from its pieces' (m, l), a lane each; one wave. f:
// this lane's piece's factor, where there are no more than 64.
__device__ inline void row_stats(const RowPieces& ps, int lane, float* m_out, float* z_out, float* f) {
  float m = neg_inf(), z = 0.0f;
  float2 mine = make_float2(neg_inf(), 0.0f);
  for (int i = lane; i < ps.n; i += kWave) {
    mine = ps.ml(i);
    m = fmaxf(m, mine.x);
  }
  m = wave_max_f32(m);
  const float ms = m == neg_inf() ? 0.0f : m;
  *f = __builtin_amdgcn_exp2f(mine.x - ms);
  if (ps.n <= kWave) {
    z = mine.y * *f;
  } else {
    for (int i = lane; i < ps.n; i += kWave) {
      const float2 ml = ps.ml(i);
      z += ml.y * __builtin_amdgcn_exp2f(ml.x - ms);
    }
  }
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1) z += __shfl_xor(z, o);
  *m_out = ms;
  *z_out = z;
}

// Workgroups below n_join: one row each. The pieces' (m, l) are read a lane
// each and their values' sums dealt to the four waves, so a row waits for two
// or three rounds of loads, whatever its number of pieces (34 pieces of 1024
// rows: 27 us with 32 threads per row that walk them one by one, 18 us with a
// wave per row, 8 us so). PER_WAVE: four rows each, where there are rows
// enough to fill the card. The others: the weights of kWeightKeys keys of a (sequence,
// kv head) from the stored scores, a thread's loads issued before the rows'
// statistics are there.
template <bool F16, bool PER_WAVE>
__global__ __launch_bounds__(kThreads) void attn_join_kernel(CacheAttnArgs a, Plan pl, int n_join, int w_tiles) {
  __shared__ float s_acc[kWaves][kCacheMaxHd];
  __shared__ float2 s_row[kNarrowRows];
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  if (static_cast<int>(blockIdx.x) < n_join) {
    const int64_t row = PER_WAVE ? static_cast<int64_t>(blockIdx.x) * kWaves + wave : blockIdx.x;
    if (PER_WAVE && row >= static_cast<int64_t>(a.B) * a.L * a.nh) return;
    const int t = static_cast<int>(row / a.nh), h = static_cast<int>(row % a.nh);
    const int b = t / a.L, l = t - b * a.L, g = h / a.rep;
    const RowPieces ps(a, pl, b, g, l * a.rep + h - g * a.rep);
    float ms, z, f;
    row_stats(ps, lane, &ms, &z, &f);
    float acc[4] = {0, 0, 0, 0};
    const int vd = a.hd > 128 ? 4 : 2;  // dimensions of a lane
    const int d = lane * vd;
    const int at = d < a.hd ? d : 0;    // lanes behind the row keep nothing
    auto add = [&](int i, float fi) {
      const float* o = ps.o(i) + at;
      if (vd == 2) {
        const float2 v = *reinterpret_cast<const float2*>(o);
        acc[0] = __builtin_fmaf(v.x, fi, acc[0]);
        acc[1] = __builtin_fmaf(v.y, fi, acc[1]);
      } else {
        const f32x4_t v = *reinterpret_cast<const f32x4_t*>(o);
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[e] = __builtin_fmaf(v[e], fi, acc[e]);
      }
    };
    constexpr int kStride = PER_WAVE ? 1 : kWaves;
    for (int i0 = 0; i0 < ps.n; i0 += kWave) {
      // 64 pieces' factors, a lane each
      if (ps.n > kWave) f = i0 + lane < ps.n ? __builtin_amdgcn_exp2f(ps.ml(i0 + lane).x - ms) : 0.0f;
      const int c = min(kWave, ps.n - i0);
#pragma unroll 8
      for (int i = PER_WAVE ? 0 : wave; i < c; i += kStride)
        add(i0 + i, __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(f), i)));
    }
    const float inv = z == 0.0f ? 0.0f : 1.0f / z;
    uint16_t* out = static_cast<uint16_t*>(a.out.p) + b * a.out.bs + l * a.out.ts + h * a.out.hs;
    const auto pair = [&](float x, float y) {
      return Act<F16>::st(x * inv) | static_cast<uint32_t>(Act<F16>::st(y * inv)) << 16;
    };
    if constexpr (PER_WAVE) {
      if (d < a.hd) {
        if (vd == 2)
          *reinterpret_cast<uint32_t*>(out + d) = pair(acc[0], acc[1]);
        else
          *reinterpret_cast<u32x2_t*>(out + d) = u32x2_t{pair(acc[0], acc[1]), pair(acc[2], acc[3])};
      }
    } else {
      if (d < a.hd)
        for (int e = 0; e < vd; ++e) s_acc[wave][d + e] = acc[e];
      __syncthreads();
      if (2 * tid < a.hd) {
        float v[2];
#pragma unroll
        for (int e = 0; e < 2; ++e)
          v[e] = s_acc[0][2 * tid + e] + s_acc[1][2 * tid + e] + (s_acc[2][2 * tid + e] + s_acc[3][2 * tid + e]);
        reinterpret_cast<uint32_t*>(out)[tid] = pair(v[0], v[1]);
      }
    }
    if (PER_WAVE ? lane == 0 : tid == 0) {
      const float l2 = z == 0.0f ? neg_inf() : ms + __log2f(z);
      if (pl.lse) pl.lse[row] = l2 * kLn2;
      if (pl.lse2) pl.lse2[(static_cast<int64_t>(b) * a.nkv + g) * pl.R + l * a.rep + h - g * a.rep] = l2;
    }
    return;
  }
  int item = static_cast<int>(blockIdx.x) - n_join;
  const int64_t j = static_cast<int64_t>(item % w_tiles) * kWeightKeys + 4 * tid;
  item /= w_tiles;
  const int g = item % a.nkv, b = item / a.nkv;
  const int64_t slot = seq_slot(a.slots, a.n_slots, b);
  if (slot < 0) return;
  const int off = a.offs[b];
  const int64_t n = own_keys(a, slot, off, a.L - 1);
  const bool some = j - 4 * tid < n;  // of the workgroup's keys are seen
  // rows of scores are multiples of 32 long: four at a time stay within
  const float* sc = pl.scores + (static_cast<int64_t>(b) * a.nkv + g) * pl.R * pl.s_ld + j;
  f32x4_t ahead[kWeightAhead];
#pragma unroll
  for (int r = 0; r < kWeightAhead; ++r)
    if (j < n && r < pl.R) ahead[r] = *reinterpret_cast<const f32x4_t*>(sc + r * pl.s_ld);
  if (some) {
    for (int r = wave; r < pl.R; r += kWaves) {
      float ms, z, f;
      row_stats(RowPieces(a, pl, b, g, r), lane, &ms, &z, &f);
      if (lane == 0) s_row[r] = make_float2(ms, z == 0.0f ? 0.0f : 1.0f / z);
    }
    __syncthreads();
  }
  f32x4_t w = {0, 0, 0, 0};
  if (j < n) {
    auto add = [&](int r, const f32x4_t& v) {
      const int64_t lim = own_keys(a, slot, off, r / a.rep);
      const float2 st = s_row[r];
#pragma unroll
      for (int e = 0; e < 4; ++e)
        w[e] += j + e < lim ? __builtin_amdgcn_exp2f(v[e] - st.x) * st.y : 0.0f;
    };
#pragma unroll
    for (int r = 0; r < kWeightAhead; ++r)
      if (r < pl.R) add(r, ahead[r]);
    for (int r = kWeightAhead; r < pl.R; ++r) add(r, *reinterpret_cast<const f32x4_t*>(sc + r * pl.s_ld));
  }
  const int64_t at = (slot * a.nkv + g) * a.S + j;
#pragma unroll
  for (int e = 0; e < 4; ++e)
    if (j + e < a.S && (j + e < n || a.w_in != a.w_out))
      a.w_out[at + e] = (a.w_in ? a.w_in[at + e] : 0.0f) + w[e];
}

// ------------------------------------------------------------------ weights, scores formed again
//
// One workgroup per (128 keys, part of the rows): a wave keeps 32 keys as the
// B operand of S = Q K^T and goes over the rows, kSumRows at a time, which
// come straight to LDS (three buffers, loads two ahead) with their ln sum exp
// and how many keys they see. A lane then has 16 rows' scores of one key:
// exp2(t - lse) added up in the lane, over rows in order, in sums of kSumRows
// rows that are added to the total (a thousand rows' sum is off by tens of
// roundings, not by a thousand). A part is every w_parts-th block of rows, so
// that all parts of a causal triangle are equally long (parts of consecutive
// rows left some XCDs with 2.4 times the work of others: 64 us for a prompt of
// 2000 tokens, 32 heads over 4, which takes 37 us so). The parts' sums are added by
// attn_weights_sum_kernel, in order. Workgroups over one part's rows run on
// one XCD.
constexpr int kSumRows = 64;
constexpr int kSumKeys = 32 * kWaves;

template <bool F16, int HD, bool ANY>
__global__ __launch_bounds__(kThreads) void attn_weights_kernel(CacheAttnArgs a, Plan pl, int pairs, int padded) {
  typedef act8_t<F16> frag_t;
  constexpr int KS = HD / 16;
  constexpr int kRowChunks = HD / 8;
  constexpr int kDmaRows = kWave / kRowChunks;
  constexpr int NL = kSumRows / kWaves / kDmaRows;
  __shared__ __attribute__((aligned(16))) uint16_t s_q0[kSumRows * HD], s_q1[kSumRows * HD], s_q2[kSumRows * HD];
  __shared__ __attribute__((aligned(16))) float s_lse0[kSumRows], s_lse1[kSumRows], s_lse2[kSumRows];
  __shared__ __attribute__((aligned(16))) int s_lim0[kSumRows], s_lim1[kSumRows], s_lim2[kSumRows];
  uint16_t* const s_q[3] = {s_q0, s_q1, s_q2};
  float* const s_lse[3] = {s_lse0, s_lse1, s_lse2};
  int* const s_lim[3] = {s_lim0, s_lim1, s_lim2};

  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int c32 = lane & 31, h2 = lane >> 5;
  int item = static_cast<int>(blockIdx.x % padded);
  if (item >= pairs) return;
  const int tile = static_cast<int>(blockIdx.x / padded);
  const int part = item % pl.w_parts;
  item /= pl.w_parts;
  const int g = item % a.nkv, b = item / a.nkv;
  const int64_t slot = seq_slot(a.slots, a.n_slots, b);
  if (slot < 0) return;
  const int off = a.offs[b];
  const int key0 = tile * kSumKeys;
  const int n = static_cast<int>(own_keys(a, slot, off, a.L - 1));
  // the part's blocks of rows from the one with the first row that sees the
  // tile's first key
  const int64_t l0 = max(static_cast<int64_t>(key0) - off, static_cast<int64_t>(0));
  if (key0 >= n || l0 >= a.L) return;
  const int first = static_cast<int>(l0) * a.rep / kSumRows;
  const int r0 = (first + (part - first % pl.w_parts + pl.w_parts) % pl.w_parts) * kSumRows;
  const int r1 = pl.R, stride = kSumRows * pl.w_parts;
  if (r0 >= r1) return;

  const int key = key0 + wave * 32 + c32;
  frag_t kf[KS];
  {
    const uint16_t* k = static_cast<const uint16_t*>(a.kc.p) + slot * a.kc.bs + g * a.kc.hs + min(key, n - 1) * a.kc.ts;
#pragma unroll
    for (int t = 0; t < KS; ++t) {
      u32x4_t w = {0, 0, 0, 0};
      if (!ANY || 16 * t + 8 * h2 < a.hd) w = *reinterpret_cast<const u32x4_t*>(k + 16 * t + 8 * h2);
      kf[t] = __builtin_bit_cast(frag_t, w);
    }
  }
  // A lane's rows' addresses, moved on to the next block: dl queries and dr
  // heads, one query more where that passes the group's last head.
  const int lr = lane / kRowChunks, lc = lane % kRowChunks;
  const int dl = stride / a.rep, dr = stride % a.rep;
  const int64_t move = dl * a.q.ts + dr * a.q.hs, carry = a.q.ts - a.rep * a.q.hs;
  const uint16_t* qp[NL];
  int qh[NL];
#pragma unroll
  for (int i = 0; i < NL; ++i) {
    const int row = wave * 16 + i * kDmaRows + lr, l = (r0 + row) / a.rep;
    qh[i] = (r0 + row) % a.rep;
    qp[i] = static_cast<const uint16_t*>(a.q.p) + b * a.q.bs + l * a.q.ts + (g * a.rep + qh[i]) * a.q.hs +
            8 * (lc ^ swz_k<HD>(i * kDmaRows + lr));
  }
  int ml = (r0 + tid) / a.rep, mh = (r0 + tid) % a.rep;
  const float* lb = pl.lse2 + (static_cast<int64_t>(b) * a.nkv + g) * pl.R;
  // (rows behind the last are not loaded: no key counts for them, whatever the
  // buffer holds)
  auto load = [&](int r, int buf) {
#pragma unroll
    for (int i = 0; i < NL; ++i) {
      if (r + wave * 16 + i * kDmaRows + lr < r1 && (!ANY || 8 * (lc ^ swz_k<HD>(i * kDmaRows + lr)) < a.hd))
        load_to_lds16(qp[i], s_q[buf] + (wave * 16 + i * kDmaRows) * HD);
      qh[i] += dr;
      const bool over = qh[i] >= a.rep;
      qh[i] -= over ? a.rep : 0;
      qp[i] += over ? move + carry : move;
    }
    // (all waves: the same values, and the same number of loads in each)
    if (r + lane < r1) load_to_lds4(lb + r + lane, s_lse[buf]);
    if (tid < kSumRows) {
      s_lim[buf][tid] = r + tid < r1 ? static_cast<int>(own_keys(a, slot, off, ml)) : 0;
      ml += dl;
      mh += dr;
      if (mh >= a.rep) {
        mh -= a.rep;
        ++ml;
      }
    }
  };
  int qa[KS];
#pragma unroll
  for (int t = 0; t < KS; ++t) qa[t] = c32 * HD + ((2 * t + h2) ^ swz_k<HD>(c32)) * 8;
  const float c = a.scale * kLog2e;
  float total = 0.0f;
  if (ANY && a.hd < HD) {  // chunks behind the heads' end, which no load writes
    for (uint16_t* q : s_q)
      for (int i = tid; i < kSumRows * kRowChunks; i += kThreads)
        reinterpret_cast<u32x4_t*>(q)[i] = u32x4_t{0, 0, 0, 0};
    __syncthreads();
  }
  settle(kf);
  load(r0, 0);
  if (r0 + stride < r1) load(r0 + stride, 1);
  auto step = [&](int r, int buf) {
    // these rows have landed (the next ones, NL + 1 loads where they are
    // whole, may be on their way), and every wave is done with the third
    // buffer
    if (r + stride + kSumRows <= r1)
      wait_vmcnt<NL + 1>();
    else
      wait_vmcnt0();
    wait_lgkmcnt0();
    lds_dma_barrier();
    if (r + 2 * stride < r1) load(r + 2 * stride, (buf + 2) % 3);
    // whether a row of these may not see all of the keys: the first sees the
    // fewest (one of the buffer's limits, the same in every thread)
    const bool some = r + kSumRows > r1 || __builtin_amdgcn_readfirstlane(s_lim[buf][0]) < key0 + kSumKeys;
    f32x16_t s[kSumRows / 32];
#pragma unroll
    for (int x = 0; x < kSumRows / 32; ++x)
#pragma unroll
      for (int i = 0; i < 16; ++i) s[x][i] = 0.0f;
#pragma unroll
    for (int t = 0; t < KS; ++t)
#pragma unroll
      for (int x = 0; x < kSumRows / 32; ++x)
        s[x] = mfma32(*reinterpret_cast<const frag_t*>(s_q[buf] + qa[t] + 32 * x * HD), kf[t], s[x]);
    float sum = 0.0f;
#pragma unroll
    for (int x = 0; x < kSumRows / 32; ++x)
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const f32x4_t z = *reinterpret_cast<const f32x4_t*>(s_lse[buf] + 32 * x + 8 * q + 4 * h2);
        f32x4_t p;
#pragma unroll
        for (int i = 0; i < 4; ++i) p[i] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[x][4 * q + i], c, -z[i]));
        if (some) {
#pragma unroll
          for (int i = 0; i < 4; ++i)
            if (key >= s_lim[buf][32 * x + 8 * q + 4 * h2 + i]) p[i] = 0.0f;
        }
        sum += (p[0] + p[1]) + (p[2] + p[3]);
      }
    total += sum;
  };
  for (int r = r0;;) {
    step(r, 0);
    if ((r += stride) >= r1) break;
    step(r, 1);
    if ((r += stride) >= r1) break;
    step(r, 2);
    if ((r += stride) >= r1) break;
  }
  total = half_sum(total);
  if (h2 == 0 && key < n)
    pl.w_part[((static_cast<int64_t>(part) * a.B + b) * a.nkv + g) * a.S + key] = total;
}

__global__ __launch_bounds__(kThreads) void attn_weights_sum_kernel(CacheAttnArgs a, Plan pl, int tiles) {
  const int64_t j = static_cast<int64_t>(blockIdx.x % tiles) * kThreads + threadIdx.x;
  const int bg = blockIdx.x / tiles, b = bg / a.nkv, g = bg % a.nkv;
  const int64_t slot = seq_slot(a.slots, a.n_slots, b);
  if (slot < 0 || j >= a.S) return;
  float w = 0.0f;
  const int off = a.L > 0 ? a.offs[b] : 0;
  const bool seen = a.L > 0 && j < own_keys(a, slot, off, a.L - 1);
  if (seen) {
    // the parts with a block from the first row on that sees the tile's first
    // key have left a sum
    const int64_t l0 = max(j / kSumKeys * kSumKeys - off, static_cast<int64_t>(0));
    const int first = static_cast<int>(l0) * a.rep / kSumRows, last = (pl.R - 1) / kSumRows;
    const float* at = pl.w_part + (static_cast<int64_t>(b) * a.nkv + g) * a.S + j;
    const int64_t step = static_cast<int64_t>(a.B) * a.nkv * a.S;
    constexpr int kAhead = 8;  // loads on their way
    for (int p0 = 0; p0 < pl.w_parts; p0 += kAhead) {
      float v[kAhead];
#pragma unroll
      for (int i = 0; i < kAhead; ++i) {
        const int p = p0 + i;
        v[i] = p < pl.w_parts && last - (last - p) % pl.w_parts >= first ? at[p * step] : 0.0f;
      }
#pragma unroll
      for (int i = 0; i < kAhead; ++i) w += v[i];
    }
  }
  const int64_t at = (slot * a.nkv + g) * a.S + j;
  if (seen || a.w_in != a.w_out) a.w_out[at] = (a.w_in ? a.w_in[at] : 0.0f) + w;
}

// ------------------------------------------------------------------ plan

// workgroups that fill the card: three of 256 threads per CU
constexpr int64_t kFill = 768;
// and of wide tiles: two
constexpr int64_t kWideFill = 512;
// Narrow tiles load past the caches where prefix and cache slots are more than
// the 256 MB that the last of them holds. The rule goes by room (lengths are on
// the device): it gains where much of the room is in use, and loses where
// little is, so that what calls in turn read would have stayed. A call through
// them and past them, two sets of caches in turn: 16 sequences, 4 kv heads of
// 128, 16384 positions: 16000 each 99.8 and 89.1 us, 1000 16.7 and 15.1; 64
// sequences, 8 kv heads, 4096 positions: 2000 each 107.7 and 104.6 us, 500
// 32.6 and 37.9, 100 17.1 and 16.5.
constexpr int64_t kPastBytes = int64_t{256} << 20;
// rows from which a wave of the join takes one of its own: 32 waves per CU
constexpr int64_t kJoinWaves = 8192;
// keys of a wide tile's piece at least: shorter ones cost more in the join
// than they gain (own keys in one piece need none). Own pieces go by room too:
// 40 queries of 32 heads over 4 after 160 keys take 14.5 us in a cache of 512
// positions and 25 in one of 16384, after 3960 keys 26.8 in 4096 and 27.9.
constexpr int64_t kWidePrefixKeys = 256;
constexpr int64_t kWideOwnKeys = 512;
// workgroups for a prompt's weights, twice what runs at a time, as those of
// late keys have few rows (40 us with 768 for 37); a part has at least 256 rows
// or so
constexpr int64_t kSumFill = 1536;

struct Layout {
  Plan pl;
  int rt;
  size_t bytes;
};

Layout make_plan(const CacheAttnArgs& a, char* ws) {
  Layout y{};
  Plan& pl = y.pl;
  size_t used = 0;
  auto take = [&](int64_t n) {
    char* p = ws ? ws + used : nullptr;
    used = static_cast<size_t>(align_up(static_cast<int64_t>(used) + n, 256));
    return p;
  };
  pl.R = a.L * a.rep;
  const int64_t rows_p = static_cast<int64_t>(a.B) * pl.R;
  pl.p_wide = a.P > 0 && rows_p > kNarrowRows;
  pl.o_wide = a.S > 0 && pl.R > kNarrowRows;
  const int64_t rt_rows =
      std::max<int64_t>(a.P > 0 && !pl.p_wide ? rows_p : 0, a.S > 0 && !pl.o_wide ? pl.R : 0);
  // (heads beyond 128: two tiles' sums leave no registers for the keys)
  y.rt = rt_rows > 16 && a.hd <= 128 ? 2 : 1;
  const int tr = 16 * y.rt;
  if (a.P > 0) {
    const int rows = pl.p_wide ? kWideRows : tr;
    pl.p_tiles = static_cast<int>((rows_p + rows - 1) / rows);
    const int64_t units = (a.P + kPiece - 1) / kPiece;
    // (beside narrow tiles of two row sets a CU takes one wide workgroup)
    const int64_t fill = !pl.p_wide ? kFill : a.S > 0 && !pl.o_wide && y.rt == 2 ? kWideFill / 2 : kWideFill;
    int64_t splits = std::max<int64_t>(1, fill / (static_cast<int64_t>(pl.p_tiles) * a.nkv));
    splits = std::min(splits, pl.p_wide ? (a.P + kWidePrefixKeys - 1) / kWidePrefixKeys : units);
    const int64_t per = (units + splits - 1) / splits;
    pl.p_keys = static_cast<int>(per * kPiece);
    pl.p_splits = static_cast<int>((units + per - 1) / per);
  }
  if (a.S > 0) {
    const int64_t units = (a.S + kPiece - 1) / kPiece;
    if (pl.o_wide) {
      pl.o_tiles = (pl.R + kWideRows - 1) / kWideRows;
      const int64_t fill = kWideFill / (static_cast<int64_t>(pl.o_tiles) * a.nkv * a.B);
      pl.o_splits = static_cast<int>(std::max<int64_t>(1, std::min(fill, a.S / kWideOwnKeys)));
    } else {
      pl.o_tiles = (pl.R + tr - 1) / tr;
      // no more pieces than units of 128 keys, and the table's room
      const int64_t fill = std::max<int64_t>(1, kFill / (static_cast<int64_t>(pl.o_tiles) * a.nkv));
      pl.o_grid = static_cast<int>(a.B + std::min<int64_t>(fill, a.B * units));
      pl.table = reinterpret_cast<int2*>(take(static_cast<int64_t>(a.B) * 8));
    }
  }
  pl.direct = (pl.o_wide && pl.o_splits == 1 && a.P == 0) || (pl.p_wide && pl.p_splits == 1 && a.S == 0);
  if (a.P > 0 && !pl.direct) {
    pl.p_o = reinterpret_cast<float*>(take(pl.p_splits * rows_p * a.nkv * a.hd * 4));
    pl.p_ml = reinterpret_cast<float2*>(take(pl.p_splits * rows_p * a.nkv * 8));
  }
  if (a.S > 0 && !pl.direct) {
    const int64_t pieces = pl.o_wide ? static_cast<int64_t>(pl.o_splits) * a.B : pl.o_grid;
    pl.o_o = reinterpret_cast<float*>(take(pieces * a.nkv * pl.R * a.hd * 4));
    pl.o_ml = reinterpret_cast<float2*>(take(pieces * a.nkv * pl.R * 8));
  }
  if (a.w_out) {
    if (!pl.o_wide) {
      pl.s_ld = align_up(a.S, kStep);
      pl.scores = reinterpret_cast<float*>(take(rows_p * a.nkv * pl.s_ld * 4));
    } else {
      pl.lse2 = reinterpret_cast<float*>(take(rows_p * a.nkv * 4));
      const int64_t tiles = (a.S + kSumKeys - 1) / kSumKeys * a.nkv * a.B;
      pl.w_parts = static_cast<int>(std::max<int64_t>(1, std::min<int64_t>(kSumFill / tiles, (pl.R + 255) / 256)));
      pl.w_part = reinterpret_cast<float*>(take(pl.w_parts * static_cast<int64_t>(a.B) * a.nkv * a.S * 4));
    }
  } else {
    pl.lse = a.lse;
  }
  y.bytes = used;
  return y;
}

// blocks of a launch over wide tiles
int64_t wide_grid(const CacheAttnArgs& a, const Plan& pl, bool prefix, WideGrid* wg) {
  wg->prefix = prefix;
  wg->splits = prefix ? pl.p_splits : pl.o_splits;
  wg->tiles = prefix ? pl.p_tiles : pl.o_tiles;
  const int64_t pairs = static_cast<int64_t>(wg->splits) * a.nkv * (prefix ? 1 : a.B);
  const int64_t padded = pairs <= 8 ? pairs : align_up(pairs, 8);
  wg->pairs = static_cast<int>(pairs);
  wg->padded = static_cast<int>(padded);
  return padded * wg->tiles;
}

// A call's launches, in blocks of kThreads.
struct Grids {
  WideGrid pg, og;           // over wide tiles of the prefix and of own keys,
  int64_t p_wide, o_wide;    // their blocks,
  int64_t p_narrow, narrow;  // those over narrow tiles of the prefix, and of both
  bool per_wave;             // the join: rows, then weights from stored scores
  int64_t join, w_tiles, join_all;
  int64_t w_pairs, w_padded, w_grid, w_sum_tiles, w_sum;  // weights of many rows
  bool fits;
};

Grids make_grids(const CacheAttnArgs& a, const Plan& pl) {
  Grids gr{};
  if (pl.p_wide) gr.p_wide = wide_grid(a, pl, true, &gr.pg);
  if (pl.o_wide) gr.o_wide = wide_grid(a, pl, false, &gr.og);
  gr.p_narrow = pl.p_wide ? 0 : static_cast<int64_t>(pl.p_splits) * a.nkv * pl.p_tiles;
  gr.narrow = gr.p_narrow + (pl.o_wide ? 0 : static_cast<int64_t>(pl.o_grid) * a.nkv * pl.o_tiles);
  const int64_t rows = static_cast<int64_t>(a.B) * a.L * a.nh, bg = static_cast<int64_t>(a.B) * a.nkv;
  gr.per_wave = rows > kJoinWaves;
  gr.join = pl.direct ? 0 : gr.per_wave ? (rows + kWaves - 1) / kWaves : rows;
  gr.w_tiles = a.w_out && !pl.o_wide ? (a.S + kWeightKeys - 1) / kWeightKeys : 0;
  gr.join_all = gr.join + gr.w_tiles * bg;
  if (a.w_out && pl.o_wide) {
    gr.w_pairs = pl.w_parts * bg;
    gr.w_padded = gr.w_pairs <= 8 ? gr.w_pairs : align_up(gr.w_pairs, 8);
    gr.w_grid = (a.S + kSumKeys - 1) / kSumKeys * gr.w_padded;
    gr.w_sum_tiles = (a.S + kThreads - 1) / kThreads;
    gr.w_sum = gr.w_sum_tiles * bg;
  }
  // (wide and narrow ones may share a launch)
  const int64_t most = max_blocks(kThreads);
  gr.fits = gr.p_wide + gr.o_wide + gr.narrow + 16 <= most && gr.join_all <= most && gr.w_grid <= most &&
            gr.w_sum <= most;
  return gr;
}

template <bool F16, int HD, int RT, bool PAST, bool ANY>
hipError_t launch_tiles(const CacheAttnArgs& a, const Plan& pl, const Grids& gr, hipStream_t stream) {
  const int np = static_cast<int>(gr.p_wide), no = static_cast<int>(gr.o_wide), n = static_cast<int>(gr.narrow);
  const dim3 wg(kThreads);
  // (heads beyond 128: a wide workgroup takes all registers of a CU, and so
  // would narrow ones in its grid)
  if (HD <= 128 && pl.p_wide && n > 0) {
    const int groups = (np + 7) / 8 + (n + 7) / 8;
    if constexpr (HD <= 128)
      hipLaunchKernelGGL((attn_both_kernel<F16, HD, RT, PAST, ANY>), dim3(static_cast<uint32_t>(groups) * 8), wg, 0,
                         stream, a, pl, gr.pg, np, n);
    return hipGetLastError();
  }
  hipError_t e = hipSuccess;
  if (np + no) {
    const int first = static_cast<int>(align_up(np, 8));  // (own blocks start on the first XCD)
    hipLaunchKernelGGL((attn_wide_kernel<F16, HD, ANY>), dim3(first + no), wg, 0, stream, a, pl, gr.pg, gr.og, first);
    e = hipGetLastError();
  }
  if (e == hipSuccess && n) {
    hipLaunchKernelGGL((attn_narrow_kernel<F16, HD, RT, PAST, ANY>), dim3(static_cast<uint32_t>(n)), wg, 0, stream, a,
                       pl, static_cast<int>(gr.p_narrow));
    e = hipGetLastError();
  }
  return e;
}

template <bool F16, int HD, bool ANY>
hipError_t launch_parts(const CacheAttnArgs& a, const Plan& pl, const Grids& gr, int rt, hipStream_t stream) {
  const bool past = (a.P + static_cast<int64_t>(a.B) * a.S) * a.nkv * a.hd * 4 > kPastBytes;
  if constexpr (HD <= 128) {
    if (rt == 2)
      return past ? launch_tiles<F16, HD, 2, true, ANY>(a, pl, gr, stream)
                  : launch_tiles<F16, HD, 2, false, ANY>(a, pl, gr, stream);
  }
  return past ? launch_tiles<F16, HD, 1, true, ANY>(a, pl, gr, stream)
              : launch_tiles<F16, HD, 1, false, ANY>(a, pl, gr, stream);
}

template <bool F16, int HD>
void launch_weight_parts(const CacheAttnArgs& a, const Plan& pl, const Grids& gr, hipStream_t stream) {
  const dim3 grid(static_cast<uint32_t>(gr.w_grid)), wg(kThreads);
  const int pairs = static_cast<int>(gr.w_pairs), padded = static_cast<int>(gr.w_padded);
  if (a.hd == HD)
    hipLaunchKernelGGL((attn_weights_kernel<F16, HD, false>), grid, wg, 0, stream, a, pl, pairs, padded);
  else
    hipLaunchKernelGGL((attn_weights_kernel<F16, HD, true>), grid, wg, 0, stream, a, pl, pairs, padded);
}

template <bool F16>
hipError_t launch_weights(const CacheAttnArgs& a, const Plan& pl, const Grids& gr, hipStream_t stream) {
  if (a.hd <= 64)
    launch_weight_parts<F16, 64>(a, pl, gr, stream);
  else if (a.hd <= 128)
    launch_weight_parts<F16, 128>(a, pl, gr, stream);
  else
    launch_weight_parts<F16, 256>(a, pl, gr, stream);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return e;
  hipLaunchKernelGGL(attn_weights_sum_kernel, dim3(static_cast<uint32_t>(gr.w_sum)), dim3(kThreads), 0, stream, a, pl,
                     static_cast<int>(gr.w_sum_tiles));
  return hipGetLastError();
}

template <bool F16>
hipError_t launch(const CacheAttnArgs& a, void* ws, hipStream_t stream) {
  const Layout y = make_plan(a, static_cast<char*>(ws));
  const Plan& pl = y.pl;
  const Grids gr = make_grids(a, pl);
  hipError_t e;
  const bool any = a.L > 1;
  if (a.hd <= 64)
    e = a.hd == 64 && !any ? launch_parts<F16, 64, false>(a, pl, gr, y.rt, stream)
                           : launch_parts<F16, 64, true>(a, pl, gr, y.rt, stream);
  else if (a.hd <= 128)
    e = a.hd == 128 && !any ? launch_parts<F16, 128, false>(a, pl, gr, y.rt, stream)
                            : launch_parts<F16, 128, true>(a, pl, gr, y.rt, stream);
  else
    e = a.hd == 256 && !any ? launch_parts<F16, 256, false>(a, pl, gr, y.rt, stream)
                            : launch_parts<F16, 256, true>(a, pl, gr, y.rt, stream);
  if (e != hipSuccess) return e;
  if (gr.join_all > 0) {
    const dim3 grid(static_cast<uint32_t>(gr.join_all)), wg(kThreads);
    const int join = static_cast<int>(gr.join), w_tiles = static_cast<int>(gr.w_tiles);
    if (gr.per_wave)
      hipLaunchKernelGGL((attn_join_kernel<F16, true>), grid, wg, 0, stream, a, pl, join, w_tiles);
    else
      hipLaunchKernelGGL((attn_join_kernel<F16, false>), grid, wg, 0, stream, a, pl, join, w_tiles);
    e = hipGetLastError();
  }
  if (e == hipSuccess && a.w_out && pl.o_wide) e = launch_weights<F16>(a, pl, gr, stream);
  return e;
}

}  // namespace

size_t cache_attn_workspace(const CacheAttnArgs& a) { return make_plan(a, nullptr).bytes; }

// no queries: one launch over the weights' rows
static int64_t kept_tiles(const CacheAttnArgs& a) { return (a.S + kThreads - 1) / kThreads; }

bool cache_attn_fits(const CacheAttnArgs& a) {
  if (a.L == 0) return kept_tiles(a) * a.nkv * a.B <= max_blocks(kThreads);
  return make_grids(a, make_plan(a, nullptr).pl).fits;
}

hipError_t launch_cache_weights_kept(const CacheAttnArgs& a, hipStream_t stream) {
  const dim3 grid(static_cast<uint32_t>(kept_tiles(a) * a.nkv * a.B));
  hipLaunchKernelGGL(attn_weights_sum_kernel, grid, dim3(kThreads), 0, stream, a, Plan{},
                     static_cast<int>(kept_tiles(a)));
  return hipGetLastError();
}

hipError_t launch_cache_attn(const CacheAttnArgs& a, bool f16, void* ws, hipStream_t stream) {
  return f16 ? launch<true>(a, ws, stream) : launch<false>(a, ws, stream);
}

}  // namespace fmx
