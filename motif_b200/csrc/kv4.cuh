// The 4-bit paged key / value cache: storage layout and the arithmetic of one stored value.
//
// A pool is [pages, Hkv, page_size / 16, unit] bytes.  A unit holds 16 consecutive tokens of one
// kv head:
//   K codes [16][D / 2] | V codes [16][D / 2] | K pairs [D / DG][16] | V pairs [D / DG][16]
// DG = min(D, 64) neighbouring dims of one token form a group with a pair (scale s, centre m) in
// bf16, s in the low half of a 32-bit word; dim 2i of a row sits in the low nibble of byte i.  A
// code c in 0..15 stands for m + s (c - 8): s has 8 significant bits and |c - 8| <= 8, so
// s (c - 8) is exact in fp32 and the sum is rounded once.
//
// The page of 16 P tokens is P consecutive units whatever P is, so a kernel that walks units needs
// no page-size variants, a page of one head is one contiguous run (72 bytes a token for D = 64),
// and every unit starts on a 128-byte boundary.
#pragma once

#include "common.cuh"

namespace mb {
namespace kv4 {

constexpr int kUnit = 16;  // tokens of one unit

template <int D>
struct Layout {
  static_assert(D == 32 || D == 64 || D == 128, "head dims of the 4-bit cache");
  static constexpr int DG = D < 64 ? D : 64;   // dims of one group
  static constexpr int NG = D / DG;            // groups of one row
  static constexpr int kRow = D / 2;           // code bytes of one row
  static constexpr int kV = kUnit * kRow;      // V codes
  static constexpr int kKp = 2 * kUnit * kRow; // K pairs
  static constexpr int kVp = kKp + 4 * NG * kUnit;
  static constexpr int kBytes = kVp + 4 * NG * kUnit;
};

__host__ __device__ constexpr int64_t unit_bytes(int64_t D) { return kUnit * D + 8 * kUnit * (D < 64 ? 1 : D / 64); }

__device__ __forceinline__ float pair_scale(uint32_t w) { return __uint_as_float(w << 16); }
__device__ __forceinline__ float pair_centre(uint32_t w) { return __uint_as_float(w & 0xffff0000u); }

}  // namespace kv4
}  // namespace mb
