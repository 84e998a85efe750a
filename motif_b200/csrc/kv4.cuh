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

#include <atomic>
#include <type_traits>
#include <utility>

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

// Everything before this kernel in the stream has ended and its writes are there.
__device__ __forceinline__ void wait_for_previous() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

__device__ __forceinline__ float pair_scale(uint32_t w) { return __uint_as_float(w << 16); }
__device__ __forceinline__ float pair_centre(uint32_t w) { return __uint_as_float(w & 0xffff0000u); }

// x / P for 0 <= x < 2^31 and P = 16 UP, UP <= 64: (x / 16) ceil(2^33 / UP) / 2^33 is exact.
struct PageDiv {
  uint64_t m;
  int P;
  __device__ __forceinline__ int operator()(int x) const { return (int)(((uint64_t)((uint32_t)x >> 4) * m) >> 33); }
};
inline PageDiv page_div(int64_t P) {
  const uint64_t up = (uint64_t)P / kUnit;
  return {((1ull << 33) + up - 1) / up, (int)P};
}

// ------------------------------------------------------------------ host side
template <typename F>
int dispatch_dim(int64_t D, F&& f) {
  switch (D) {
    case 32: return f(std::integral_constant<int, 32>());
    case 64: return f(std::integral_constant<int, 64>());
    case 128: return f(std::integral_constant<int, 128>());
  }
  return set_error(MB_ERR_UNSUPPORTED, "kv4: head dim %lld (32, 64 or 128)", (long long)D);
}
template <typename F>
int dispatch(int dtype, int64_t D, F&& f) {
  switch (dtype) {
    case MB_F32: return dispatch_dim(D, [&](auto d) { return f(float(), d); });
    case MB_F16: return dispatch_dim(D, [&](auto d) { return f(__half(), d); });
    case MB_BF16: return dispatch_dim(D, [&](auto d) { return f(__nv_bfloat16(), d); });
  }
  return set_error(MB_ERR_DTYPE, "kv4: unsupported dtype %d", dtype);
}

// Launch that may begin while the kernel before it in the stream ends: every kernel launched so starts
// with wait_for_previous(), before it touches memory, and lets the next one begin early in turn.
template <typename... P, typename... A>
void launch(void (*kernel)(P...), dim3 grid, int threads, int smem, void* stream, A&&... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = (cudaStream_t)stream;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  cudaLaunchKernelEx(&cfg, kernel, std::forward<A>(args)...);
}

// SMs of the current device (0: the query failed).
inline int sm_count() {
  static std::atomic<int> known[64];
  int dev = 0, n = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return 0;
  if (dev < 64 && (n = known[dev].load(std::memory_order_relaxed)) > 0) return n;
  if (cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess) return 0;
  if (dev < 64) known[dev].store(n, std::memory_order_relaxed);
  return n;
}

inline int check_paging(const char* who, int64_t B, int64_t columns, int64_t ts, int64_t P) {
  MB_REQUIRE(B >= 0 && B <= (1 << 20), MB_ERR_SHAPE, "%s: %lld requests (0 .. 2^20)", who, (long long)B);
  MB_REQUIRE(columns >= 1 && ts >= columns, MB_ERR_SHAPE, "%s: block table of %lld columns, row stride %lld", who,
             (long long)columns, (long long)ts);
  MB_REQUIRE(P >= kUnit && P <= 1024 && P % kUnit == 0, MB_ERR_ARG, "%s: page size %lld (a multiple of 16, at most 1024)",
             who, (long long)P);
  // the attention's 32-bit token numbers run up to a tile past the last one
  MB_REQUIRE(columns <= (1 << 27) && columns * P <= (1ll << 31) - 1024, MB_ERR_SHAPE,
             "%s: a request could hold %lld pages of %lld tokens (fewer than 2^31 - 1023 tokens)", who, (long long)columns,
             (long long)P);
  return MB_OK;
}
inline int check_pool(const char* who, const void* pool, int64_t pages, int64_t Hkv, int64_t P) {
  MB_REQUIRE(pool, MB_ERR_ARG, "%s: null pointer", who);
  MB_REQUIRE(reinterpret_cast<uintptr_t>(pool) % 16 == 0, MB_ERR_ALIGN, "%s: the pool must be 16-byte aligned", who);
  MB_REQUIRE(pages >= 1 && Hkv >= 1 && Hkv <= 65535, MB_ERR_SHAPE, "%s: %lld pages, %lld kv heads", who,
             (long long)pages, (long long)Hkv);
  MB_REQUIRE(pages * P < (1ll << 31), MB_ERR_SHAPE, "%s: %lld slots (fewer than 2^31)", who, (long long)(pages * P));
  return MB_OK;
}
inline int check_rows16(const char* who, const void* p, const int64_t* s, int64_t esize) {
  bool ok = reinterpret_cast<uintptr_t>(p) % 16 == 0;
  for (int i = 0; i < 3; ++i) ok = ok && s[i] * esize % 16 == 0;
  MB_REQUIRE(ok, MB_ERR_ALIGN, "%s: rows must start on 16-byte boundaries", who);
  return MB_OK;
}


}  // namespace kv4
}  // namespace mb
