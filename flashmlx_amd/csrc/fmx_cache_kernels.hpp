// fmx_cache_kernels.hpp -- argument blocks and launchers of the KV cache's
// long-context operators (fmx_rope.hip, fmx_cache_attn.hip, fmx_evict.hip;
// library-internal).
#pragma once

#include "fmx_common.hpp"

namespace fmx {

// workgroups of a launch: HIP takes fewer than 2^32 threads
constexpr int64_t max_blocks(int threads) { return ((int64_t{1} << 32) - 1) / threads; }

// strided rows of heads, as fmx_heads
struct HeadsView {
  void* p;
  int64_t bs, ts, hs;
};

// slot of sequence b, or -1 (a slot outside the cache)
__device__ inline int64_t seq_slot(const int32_t* slots, int64_t n_slots, int b) {
  if (!slots) return b < n_slots ? b : -1;
  const int s = slots[b];
  return s >= 0 && s < n_slots ? s : -1;
}

// ------------------------------------------------------------------ rope

constexpr int kRopeMaxHd = 1024;

struct RotateArgs {
  const double* freqs;
  int dims;
  float factor;
  int interleaved, inverse;
  int B, L, nh, nkv, hd;  // rotated heads: nh of q, then nkv of k; then nkv copied of v
  HeadsView q, k, v, q_out, kc, vc;
  const int32_t* pos;
  // null (q alone), or the caches' rows of sequence b: slots[b], offs[b] + l
  const int32_t* offs;
  const int32_t* slots;
  int64_t n_slots, max_seq;
};
// es: bytes of an element (2 or 4), f16: of a 2-byte one
hipError_t launch_rotate(const RotateArgs& a, int es, bool f16, hipStream_t stream);

// ------------------------------------------------------------------ attention

constexpr int kCacheMaxHd = 256;

struct CacheAttnArgs {
  int B, L, nh, nkv, rep, hd;
  float scale;
  HeadsView q, out, kp, vp, kc, vc;
  int64_t P;              // prefix positions
  int64_t n_slots, S;     // own caches
  const int32_t* offs;
  const int32_t* slots;
  float* lse;             // [B, L, nh] or null
  const float* w_in;      // [n_slots, nkv, S] or null
  float* w_out;           // or null: no weights
};
size_t cache_attn_workspace(const CacheAttnArgs& a);
// whether all of its launches are within max_blocks
bool cache_attn_fits(const CacheAttnArgs& a);
hipError_t launch_cache_attn(const CacheAttnArgs& a, bool f16, void* ws, hipStream_t stream);
// no queries (L 0): w_out's rows of the sequences' slots from w_in, or 0
hipError_t launch_cache_weights_kept(const CacheAttnArgs& a, hipStream_t stream);

// own keys that query l of sequence b sees (slot: of that sequence, or -1)
__device__ inline int64_t own_keys(const CacheAttnArgs& a, int64_t slot, int off, int l) {
  if (slot < 0) return 0;
  const int64_t n = static_cast<int64_t>(off) + l + 1;
  return n < 0 ? 0 : (n > a.S ? a.S : n);
}

// Own keys in pieces of whole units of kPieceKeys keys.
constexpr int kPieceKeys = 128;

// Units of a piece, the fewest that keep `total` units of all sequences within
// `room` pieces beside one per sequence: never more than a sequence of max_seq
// positions has, so that a piece's keys count within 32 bits.
__host__ __device__ inline uint32_t piece_units(uint32_t total, uint32_t room, int64_t max_seq) {
  const uint32_t c = total / room + (total % room != 0);
  const uint32_t most = static_cast<uint32_t>((max_seq + kPieceKeys - 1) / kPieceKeys);
  return c < most ? c : most;
}

// Keys [k0, k1) of piece k of a sequence of n keys.
__host__ __device__ inline void piece_keys(int k, int units, int64_t n, int* k0, int* k1) {
  *k0 = k * units * kPieceKeys;
  const int64_t end = *k0 + static_cast<int64_t>(units) * kPieceKeys;
  *k1 = static_cast<int>(n < end ? n : end);
}

// ------------------------------------------------------------------ eviction

struct EvictArgs {
  int B, nkv;
  int64_t row_bytes;      // of a position's keys of one head
  const uint8_t* k;       // strides in bytes
  const uint8_t* v;
  int64_t k_bs, k_ts, k_hs, v_bs, v_ts, v_hs;
  uint8_t* k_out;
  uint8_t* v_out;
  int64_t ko_bs, ko_ts, ko_hs, vo_bs, vo_ts, vo_hs;
  float* w;               // [n_slots, nkv, S]
  float* w_out;           // [n_slots, nkv, S_out] (w when in place)
  int64_t n_slots, S, S_out;
  const int32_t* lens;
  const int32_t* slots;
  int64_t budget, sinks, recent;
  int32_t* lens_out;
  int32_t* kept;          // [B, nkv, budget]
  bool in_place;
};
// whether both of its launches are within max_blocks
bool evict_fits(const EvictArgs& a);
hipError_t launch_evict(const EvictArgs& a, hipStream_t stream);

}  // namespace fmx
