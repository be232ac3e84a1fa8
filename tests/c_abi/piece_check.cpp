// Host check of how own keys are dealt to pieces (csrc/fmx_cache_kernels.hpp):
// for batches up to the operators' limits, every sequence's pieces cover its
// keys once and in order, and all pieces fit the grid. Prints what differs.
#include <cstdint>
#include <cstdio>
#include <vector>

#include "../../flashmlx_amd/csrc/fmx_cache_kernels.hpp"

using namespace fmx;

// n sequences of `keys` keys each
struct Run {
  int64_t n, keys;
};

static int check(const char* what, const std::vector<Run>& runs, int64_t max_seq, int64_t room) {
  int64_t total = 0;
  auto units_of = [](int64_t keys) { return (keys + kPieceKeys - 1) / kPieceKeys; };
  for (const Run& r : runs) total += r.n * units_of(r.keys);
  int64_t c = piece_units(static_cast<uint32_t>(total), static_cast<uint32_t>(room), max_seq);
  if (c < 1) c = 1;
  int64_t pieces = 0, batch = 0;
  for (const Run& r : runs) {
    const int64_t n = (units_of(r.keys) + c - 1) / c;
    pieces += r.n * n;
    batch += r.n;
    int64_t at = 0;
    for (int64_t k = 0; k < n; ++k) {
      int k0, k1;
      piece_keys(static_cast<int>(k), static_cast<int>(c), r.keys, &k0, &k1);
      if (k0 != at || k1 <= k0 || k1 > r.keys) {
        std::printf("%s: piece %lld of %lld keys is [%d, %d)\n", what, (long long)k, (long long)r.keys, k0, k1);
        return 1;
      }
      at = k1;
    }
    if (at != r.keys) {
      std::printf("%s: %lld of %lld keys\n", what, (long long)at, (long long)r.keys);
      return 1;
    }
  }
  if (pieces > batch + room) {
    std::printf("%s: %lld pieces for a grid of %lld\n", what, (long long)pieces, (long long)(batch + room));
    return 1;
  }
  return 0;
}

int main() {
  int bad = 0;
  for (int64_t room : {1, 2, 24, 191, 768}) {
    bad += check("one", {{1, 1}}, 1, room);
    bad += check("none", {{5, 0}}, 100, room);
    bad += check("ragged", {{1, 16384}, {3, 1}, {2, 0}, {1, 129}, {7, 5000}}, 16384, room);
    bad += check("longest", {{1, 1 << 24}}, 1 << 24, room);
    bad += check("longest and many", {{4095, 1 << 24}, {1, 1}}, 1 << 24, room);
    // 2^36 own positions, the most of one call
    bad += check("2^18 of 2^18", {{1 << 18, 1 << 18}}, 1 << 18, room);
    bad += check("2^24 of 2^12", {{1 << 24, 1 << 12}}, 1 << 12, room);
    bad += check("2^24 of 1", {{1 << 24, 1}}, 1, room);
  }
  if (!bad) std::printf("pieces ok\n");
  return bad != 0;
}
