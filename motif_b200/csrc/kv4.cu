// What a serving loop needs beside the attention over its paged 4-bit cache (kv4_attention.cu): the
// reservation of cache slots from request lengths, the quantising append, and the read-back of
// cached prefixes.  Layout and value of a stored code: kv4.cuh.
#include <math.h>

#include "common.cuh"
#include "kv4.cuh"

namespace mb {
namespace {

using kv4::kUnit;
using kv4::Layout;
using kv4::PageDiv;

// ------------------------------------------------------------------ slot reservation
// need_b = ceil((len_b + new_b) / P) - ceil(len_b / P) fresh pages.  Requests are served in order:
// request b gets its pages when they fit its table row, its tokens fit the slot map, and the pages
// asked for up to and including it do not exceed the free count; the i-th fresh page is the i-th
// from the top of the free list.
//
// A block of THREADS requests at a time: every CTA scans the block's tokens and pages by itself, then
// the threads of all CTAs share the writing.  Where lens_out is lens (or the free counts are one) the
// CTAs are a cluster, whose barrier keeps the writes behind everybody's reads.  A new token's page is an
// old table entry or comes straight from the free list, so nobody waits for the fresh entries to be
// written.  Bound by latency (the bytes take 0.1 us): one scan and two dependent loads.  3.3 us for one
// token of each of 64 requests (one CTA of four warps), 4.4 for 32 prompts of 4096 tokens, 5.7 for 517
// ragged chunks (in place, on a cluster of 8, 7.6 and 9.0); on one CTA the latter two took 43.9 and 35.2.
constexpr int kClusterCtas = 8;  // the most a cluster holds everywhere
constexpr int kReserveCtas = 64;

__device__ __forceinline__ int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

// Sums of whole numbers 0 .. 2^31 - 1 that stop at 2^31 - 1 (which is past every limit compared with).
__device__ __forceinline__ int add_to_most(int a, int b) { return (int)min((uint32_t)a + (uint32_t)b, 0x7fffffffu); }

__device__ __forceinline__ int warp_scan(int v) {  // inclusive
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int u = __shfl_up_sync(0xffffffffu, v, o);
    if ((int)(threadIdx.x & 31) >= o) v = add_to_most(v, u);
  }
  return v;
}

// Inclusive scan over the block's threads; `part` holds one value per warp.
template <int THREADS>
__device__ __forceinline__ int block_scan(int v, int* part) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  v = warp_scan(v);
  if (lane == 31) part[warp] = v;
  __syncthreads();
  // every warp scans the warps' sums for itself
  const int sums = warp_scan(lane < THREADS / 32 ? part[lane] : 0);
  const int before = __shfl_sync(0xffffffffu, sums, max(warp - 1, 0));
  return warp ? add_to_most(v, before) : v;
}

template <int THREADS>
__global__ void __launch_bounds__(THREADS) paged_reserve_kernel(
    const int32_t* lens, const int32_t* __restrict__ new_lens, int32_t* table, int64_t ts,
    const int32_t* __restrict__ free_pages, const int32_t* free_count, int32_t* lens_out, int32_t* free_out,
    int32_t* __restrict__ slots, bool vector, bool in_place, int total, int B, int columns, int cap, PageDiv by) {
  // of each request of the block: end of its tokens and of its fresh pages, both counted over all
  __shared__ int s_end[THREADS], s_pages[THREADS];
  __shared__ int s_len[THREADS], s_new[THREADS];  // new: -1 - new where it is not served
  __shared__ int part[2][32];
  __shared__ int s_taken;
  allow_dependent_launch();
  kv4::wait_for_previous();
  const int tid = threadIdx.x, lane = tid & 31, P = by.P;
  const int ranks = gridDim.x, rank = blockIdx.x;
  const int me = rank * THREADS + tid, all_threads = ranks * THREADS;
  auto pages = [&](int n) { return by(n) + (by(n) * P < n ? 1 : 0); };
  const int avail = min(max(*free_count, 0), cap);
  if (tid == 0) s_taken = 0;
  int tokens = 0, used = 0;  // of the blocks before
  for (int b0 = 0; b0 < B; b0 += THREADS) {
    const int b = b0 + tid, n = min(THREADS, B - b0);
    int half = THREADS / 2;
    while (half >= n && half > 1) half >>= 1;
    int len = 0, fresh = 0;
    if (b < B) {
      len = max(lens[b], 0);
      fresh = max(new_lens[b], 0);
    }
    const int end = add_to_most(tokens, block_scan<THREADS>(fresh, part[0]));
    const int full = add_to_most(len, fresh);
    const bool possible = b < B && full <= columns * P && end <= total;
    const int need = possible ? pages(full) - pages(len) : 0;
    const int upto = add_to_most(used, block_scan<THREADS>(need, part[1]));
    const bool ok = possible && (need == 0 || upto <= avail);
    s_end[tid] = end;
    s_pages[tid] = upto;
    s_len[tid] = len;
    s_new[tid] = ok ? fresh : -1 - fresh;
    // those that were served and took pages come first: the last of them says how many were taken
    const int taken = __reduce_max_sync(0xffffffffu, ok && need ? upto : 0);
    if (lane == 0 && taken) atomicMax(&s_taken, taken);
    if (in_place && ranks > 1) asm volatile("barrier.cluster.arrive.aligned;\nbarrier.cluster.wait.aligned;" ::: "memory");
    else __syncthreads();
    if (rank == 0 && b < B) lens_out[b] = ok ? full : len;
    // the first request of the block whose running sum (tokens or pages) passes x
    auto find = [&](const int* sums, int x) {
      int r = 0;
      for (int step = half; step; step >>= 1)
        if (r + step < n && sums[r + step - 1] <= x) r += step;
      return r;
    };
    // fresh table entries: the i-th from the top of the free list (past `avail` nobody is served)
    for (int i = used + me; i < min(s_pages[n - 1], avail); i += all_threads) {
      const int r = find(s_pages, i);
      if (s_new[r] < 0) continue;
      const int want = pages(s_len[r] + s_new[r]);
      table[(int64_t)(b0 + r) * ts + want - (s_pages[r] - i)] = free_pages[avail - 1 - i];
    }
    // slots: a run of neighbouring tokens per thread, whole groups of four where there are many; a
    // page is looked up once for the tokens of the run that lie in it
    const int stop = min(s_end[n - 1], total);
    const int run = stop - tokens <= all_threads ? 1 : ((stop - tokens + 3) / all_threads + 4) / 4 * 4;
    const int from = (run == 1 ? tokens : tokens & ~3) + me * run;  // groups of four start at multiples of 4
    int token = max(from, tokens);
    const int last = min(from + run, stop);
    if (from < stop && token < last) {
      int r = find(s_end, token);
      while (token < last) {
        while (s_end[r] <= token) ++r;
        int until = min(last, s_end[r]), v = -1, up = 0;
        if (s_new[r] >= 0) {
          const int pos = s_len[r] + token - (s_end[r] - s_new[r]), at = by(pos), off = pos - at * P;
          const int have = pages(s_len[r]), want = pages(s_len[r] + s_new[r]);
          const int page = at < have ? table[(int64_t)(b0 + r) * ts + at]
                                     : free_pages[avail - 1 - (s_pages[r] - (want - at))];
          v = page * P + off;
          up = 1;
          until = min(until, token + P - off);
        }
        while (token < until) {
          if ((token & 3) == 0 && token + 4 <= until && vector) {
            *reinterpret_cast<int4*>(slots + token) = make_int4(v, v + up, v + 2 * up, v + 3 * up);
            token += 4, v += 4 * up;
          } else {
            slots[token] = v;
            ++token, v += up;
          }
        }
      }
    }
    tokens = s_end[THREADS - 1];
    used = s_pages[THREADS - 1];
    __syncthreads();
  }
  for (int64_t i = (int64_t)tokens + me; i < total; i += all_threads) slots[i] = -1;
  if (rank == 0 && tid == 0) *free_out = avail - s_taken;
}

// Finished requests give their pages back: onto the top of the free list in request order, their
// table rows become -1 and their lengths 0.  One CTA, whose warps copy rows: 64 requests of 128 pages 4.9
// us, 512 of 128 19.8, 512 of 512 67 (the bytes take 0.02 to 0.5); once in a request's life.
constexpr int kReleaseThreads = 1024;

__global__ void __launch_bounds__(kReleaseThreads) paged_release_kernel(
    const uint8_t* __restrict__ done, int32_t* __restrict__ lens, int32_t* __restrict__ table, int64_t ts,
    int32_t* __restrict__ free_pages, int32_t* __restrict__ free_count, int B, int columns, int64_t cap, int P) {
  __shared__ int part[32];
  __shared__ int s_at[kReleaseThreads], s_held[kReleaseThreads];
  allow_dependent_launch();
  kv4::wait_for_previous();
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  int top = max(*free_count, 0);
  for (int b0 = 0; b0 < B; b0 += kReleaseThreads) {
    const int b = b0 + tid;
    int held = 0;
    if (b < B && done[b]) {
      held = (int)min(ceil_div(max(lens[b], 0), P), (int64_t)columns);
      lens[b] = 0;
    }
    const int upto = add_to_most(top, block_scan<kReleaseThreads>(held, part));
    s_at[tid] = upto - held;
    s_held[tid] = held;
    __syncthreads();
    for (int r = warp; r < min(kReleaseThreads, B - b0); r += kReleaseThreads / 32) {
      int32_t* row = table + (int64_t)(b0 + r) * ts;
      for (int j = lane; j < s_held[r]; j += 32) {
        if (s_at[r] + j < cap) free_pages[s_at[r] + j] = row[j];
        row[j] = -1;
      }
    }
    top = s_at[kReleaseThreads - 1] + s_held[kReleaseThreads - 1];
    __syncthreads();
  }
  if (tid == 0) *free_count = (int32_t)min((int64_t)top, cap);
}

// ------------------------------------------------------------------ append
template <typename I>
struct Strides12 {
  I s[12];  // k(b,h,t) v(b,h,t) k_out(b,h,t) v_out(b,h,t); 32-bit ones make each product one instruction
  __device__ __forceinline__ int64_t at(int i, int b, int h, int t) const {
    return (int64_t)b * s[i] + (int64_t)h * s[i + 1] + (int64_t)t * s[i + 2];
  }
};

__device__ __forceinline__ float fmax_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float fmin_nan(float a, float b) {
  float r;
  asm("min.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

template <typename T> struct Pair;
template <> struct Pair<__half> { using type = __half2; };
template <> struct Pair<__nv_bfloat16> { using type = __nv_bfloat162; };

// Eight consecutive elements at a 16-byte aligned address, and for 16-bit types as they lie there.
template <typename T>
__device__ __forceinline__ void load8(const T* p, float* x, uint4& raw) {
  if constexpr (sizeof(T) == 4) {
    const float4 a = *reinterpret_cast<const float4*>(p), b = *reinterpret_cast<const float4*>(p + 4);
    x[0] = a.x, x[1] = a.y, x[2] = a.z, x[3] = a.w, x[4] = b.x, x[5] = b.y, x[6] = b.z, x[7] = b.w;
  } else {
    raw = *reinterpret_cast<const uint4*>(p);
    const T* h = reinterpret_cast<const T*>(&raw);
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = to_f(h[i]);
  }
}
template <typename T>
__device__ __forceinline__ void store8(T* p, const float* x) {
  if constexpr (sizeof(T) == 4) {
    *reinterpret_cast<float4*>(p) = make_float4(x[0], x[1], x[2], x[3]);
    *reinterpret_cast<float4*>(p + 4) = make_float4(x[4], x[5], x[6], x[7]);
  } else {
    *reinterpret_cast<uint4*>(p) =
        make_uint4(pack2<T>(x[0], x[1]), pack2<T>(x[2], x[3]), pack2<T>(x[4], x[5]), pack2<T>(x[6], x[7]));
  }
}

__device__ __forceinline__ __half2 lows(__half2 a, __half2 b) { return __lows2half2(a, b); }
__device__ __forceinline__ __half2 highs(__half2 a, __half2 b) { return __highs2half2(a, b); }
__device__ __forceinline__ __nv_bfloat162 lows(__nv_bfloat162 a, __nv_bfloat162 b) { return __lows2bfloat162(a, b); }
__device__ __forceinline__ __nv_bfloat162 highs(__nv_bfloat162 a, __nv_bfloat162 b) { return __highs2bfloat162(a, b); }

// Largest and smallest of the group that LANES neighbouring lanes hold, 8 E values each (a NaN
// anywhere: both NaN).  16-bit values keep (max, -min) as a packed pair of their own type, so one
// packed maximum per step reduces both.
template <typename T, int LANES, int E>
__device__ __forceinline__ void extremes(const uint4* raw, const float* x, float& hi, float& lo) {
  if constexpr (sizeof(T) == 4) {
    hi = lo = x[0];
#pragma unroll
    for (int i = 1; i < 8 * E; ++i) hi = fmax_nan(hi, x[i]), lo = fmin_nan(lo, x[i]);
#pragma unroll
    for (int d = 1; d < LANES; d <<= 1) {
      hi = fmax_nan(hi, __shfl_xor_sync(0xffffffffu, hi, d));
      lo = fmin_nan(lo, __shfl_xor_sync(0xffffffffu, lo, d));
    }
  } else {
    using T2 = typename Pair<T>::type;
    const T2* v = reinterpret_cast<const T2*>(raw);
    T2 a = v[0], c = v[0];
#pragma unroll
    for (int i = 1; i < 4 * E; ++i) a = __hmax2_nan(a, v[i]), c = __hmin2_nan(c, v[i]);
    const T2 n = __hneg2(c);
    // (largest, -smallest) of the two halves
    T2 both = __hmax2_nan(lows(a, n), highs(a, n));
#pragma unroll
    for (int d = 1; d < LANES; d <<= 1) {
      const uint32_t u = __shfl_xor_sync(0xffffffffu, *reinterpret_cast<const uint32_t*>(&both), d);
      both = __hmax2_nan(both, *reinterpret_cast<const T2*>(&u));
    }
    hi = to_f(both.x);
    lo = -to_f(both.y);
  }
}

// The group's pair and this thread's 8 E codes, a word for eight; y becomes the values they stand for.
//
// The code is the nearest whole number to RN(d / s), d = RN(x - m), ties to even.  With r = RN(1 / s),
// q = RN(d r) and the exact residual e = d - q s (one fma), RN(q + e r) is RN(d / s) (Markstein 1990:
// a correctly rounded reciprocal and a quotient within one unit give the correctly rounded quotient),
// at a multiplication and two fmas a value, in packed pairs; so is range / 15.  Scales below 2^-100,
// where r or e could leave the range, divide, as do groups whose codes could.  Adding 1.5 2^23 + 8
// rounds to a whole number, ties to even, and leaves c + 8 in the low bits, so the word is a sum of
// shifted sums less a constant.
template <int E>
__device__ __forceinline__ void quantise(const float* x, float hi, float lo, float* y, uint32_t* word, uint32_t& pair) {
  const float range = __fsub_rn(hi, lo);
  constexpr float r15 = 1.0f / 15.0f;
  const float q15 = __fmul_rn(range, r15);
  float step = __fmaf_rn(__fmaf_rn(-q15, 15.0f, range), r15, q15);
  // ranges whose scale is below 2^-100 divide; 0 and NaN are among them
  bool odd = !(range >= 1.2e-29f);
  if (odd) step = __fdiv_rn(range, 15.0f);
  float s = __bfloat162float(__float2bfloat16_rn(step));
  float m = __bfloat162float(__float2bfloat16_rn(__fmaf_rn(8.0f, s, lo)));  // 8 s is exact: one rounding
  if (!(range <= 3.4028234e38f)) s = m = __uint_as_float(0x7fc00000u);  // a NaN or an infinity: all NaN
  // the extremes lie on -8 and 7 but for the rounding of s and m: only where that is large (a centre
  // far from 0) can a code leave the range
  odd = odd || lo - m < -8.49f * s || hi - m > 7.49f * s;
  constexpr float kRound = 12582912.f + 8.f;
  uint32_t sum[E] = {};
  if (!odd) {
    const float r = __frcp_rn(s);
    const float2 m2 = make_float2(-m, -m), r2 = make_float2(r, r), s2 = make_float2(s, s), n2 = make_float2(-s, -s);
#pragma unroll
    for (int i = 0; i < 4 * E; ++i) {
      const float2 d = fadd2(make_float2(x[2 * i], x[2 * i + 1]), m2), q0 = fmul2(d, r2);
      const float2 t = fadd2(ffma2(ffma2(n2, q0, d), r2, q0), make_float2(kRound, kRound));
      sum[i / 4] += __float_as_uint(t.x) * (1u << (8 * (i % 4))) + __float_as_uint(t.y) * (16u << (8 * (i % 4)));
      const float2 v = ffma2(s2, fadd2(t, make_float2(-kRound, -kRound)), make_float2(m, m));
      y[2 * i] = v.x, y[2 * i + 1] = v.y;
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8 * E; ++i) {
      const float q = s > 0.f ? __fdiv_rn(__fsub_rn(x[i], m), s) : 0.f;
      const float t = __fadd_rn(fminf(fmaxf(q, -8.f), 7.f), kRound);
      sum[i / 8] += __float_as_uint(t) << (4 * (i % 8));
      y[i] = fmaf(s, __fsub_rn(t, kRound), m);
    }
  }
  // the bits of 1.5 2^23 in every term
#pragma unroll
  for (int e = 0; e < E; ++e) word[e] = sum[e] - 0x4b400000u * 0x11111111u;
  pair = (__float_as_uint(m) & 0xffff0000u) | (__float_as_uint(s) >> 16);
}

// A thread takes E chunks of eight dims of one group, the same ones of K and V of one token and head:
// DG / 8 E neighbouring lanes make a group, the rows of a warp are neighbouring tokens of one head
// (blockIdx.y), whose codes and pairs lie next to each other.  What a group needs once (its pair, the
// reciprocal, the addresses: more than half of the instructions at E = 1) is shared by 8 E values a
// lane.  131072 tokens of 3 bf16 heads of 64 with the stored values given back: 40.4 us at E = 2, 5.7
// TB/s or 87 % of the copy rate (E = 1 50.7; E = 4 as slow, of too few warps; IEEE divisions at E = 1
// 128.6).  A call that does not fill the GPU is a chain of latencies, which E = 1 makes shorter: one
// token of 64 requests 1.8 us against 2.1.  fp32 is at the copy rate at E = 1: 5003 tokens of 8 heads
// of 128 11.7 us (15.1 with inputs that were not in L2 before).  CTAs that stay and fetch their next rows early measured slower (60.5 us where E = 1
// took 51.0: the registers cost more warps than the early loads hide).
template <typename T, int D, int E, typename I>
__global__ void __launch_bounds__(256) kv4_append_kernel(const T* __restrict__ k, const T* __restrict__ v,
                                                         const int32_t* __restrict__ slots,
                                                         uint8_t* __restrict__ pool, T* __restrict__ k_out,
                                                         T* __restrict__ v_out, Strides12<I> st, int N, int T_, int Hkv,
                                                         int nslots, PageDiv by) {
  using L = Layout<D>;
  constexpr int LANES = L::DG / (8 * E), W = D / (8 * E);  // threads of a group, of a row
  const int w = threadIdx.x % W, h = blockIdx.y;
  const int64_t at = (int64_t)blockIdx.x * (256 / W) + threadIdx.x / W;
  const bool live = at < N;  // whole groups of lanes: W divides the warp
  const int n = live ? (int)at : 0;
  const int b = T_ == N ? 0 : n / T_, t = n - b * T_;
  allow_dependent_launch();
  kv4::wait_for_previous();
  const int slot = live ? slots[n] : -1;
  const int g = w / LANES, c0 = g * (L::DG / 8) + w % LANES;  // chunks c0, c0 + LANES, ... of eight dims
  float x[2][8 * E], y[2][8 * E], hi, lo;
  uint4 raw[2][E];
#pragma unroll
  for (int e = 0; e < E; ++e) {
    load8(k + st.at(0, b, h, t) + 8 * (c0 + LANES * e), x[0] + 8 * e, raw[0][e]);
    load8(v + st.at(3, b, h, t) + 8 * (c0 + LANES * e), x[1] + 8 * e, raw[1][e]);
  }
  uint32_t word[2][E], pair[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    extremes<T, LANES, E>(raw[i], x[i], hi, lo);
    quantise<E>(x[i], hi, lo, y[i], word[i], pair[i]);
  }
  if (!live) return;
  if (slot >= 0 && slot < nslots) {
    const int page = by(slot), off = slot - page * by.P, r = off % kUnit;
    uint8_t* u = pool + (((int64_t)page * Hkv + h) * (by.P / kUnit) + off / kUnit) * L::kBytes;
#pragma unroll
    for (int e = 0; e < E; ++e) {
      *reinterpret_cast<uint32_t*>(u + r * L::kRow + 4 * (c0 + LANES * e)) = word[0][e];
      *reinterpret_cast<uint32_t*>(u + L::kV + r * L::kRow + 4 * (c0 + LANES * e)) = word[1][e];
    }
    if (w % LANES == 0) {
      *reinterpret_cast<uint32_t*>(u + L::kKp + (g * kUnit + r) * 4) = pair[0];
      *reinterpret_cast<uint32_t*>(u + L::kVp + (g * kUnit + r) * 4) = pair[1];
    }
  }
  if (k_out) {
#pragma unroll
    for (int e = 0; e < E; ++e) {
      store8(k_out + st.at(6, b, h, t) + 8 * (c0 + LANES * e), y[0] + 8 * e);
      store8(v_out + st.at(9, b, h, t) + 8 * (c0 + LANES * e), y[1] + 8 * e);
    }
  }
}

// ------------------------------------------------------------------ gather
// Eight values of one word: a code in the last bits of 2^23 is a float 2^23 + c; taking 2^23 + 8 off is
// exact, and s (c - 8) + m is rounded once.
__device__ __forceinline__ void values8(uint32_t word, uint32_t pair, float* x) {
  const float2 s = make_float2(kv4::pair_scale(pair), kv4::pair_scale(pair));
  const float2 m = make_float2(kv4::pair_centre(pair), kv4::pair_centre(pair));
#pragma unroll
  for (int i = 0; i < 8; i += 2) {
    const float2 c = make_float2(__uint_as_float(((word >> (4 * i)) & 15u) | 0x4b000000u),
                                 __uint_as_float(((word >> (4 * i + 4)) & 15u) | 0x4b000000u));
    const float2 v = ffma2(fadd2(c, make_float2(-8388616.f, -8388616.f)), s, m);
    x[i] = v.x, x[i + 1] = v.y;
  }
}

// A thread reads E words of codes of K and of V of one token and group and writes eight values of each;
// D / 8 E neighbouring lanes make a row, a warp neighbouring tokens of one head.  Tokens at or past the
// request's length, and those of pages outside the pool, become zeros.  32 prefixes of up to 4096 tokens,
// 3 bf16 heads of 64 (115 MB, most of it written): 19.3 us at E = 2, where the bytes take 17.6; 20.4 at
// E = 1, whose length, page and pair serve half as many values (64-bit indexes and conversions from
// integers: 26.6).
template <typename T, int D, int E>
__global__ void __launch_bounds__(256) kv4_gather_kernel(const uint8_t* __restrict__ pool,
                                                         const int32_t* __restrict__ table, int64_t ts,
                                                         const int32_t* __restrict__ lens, T* __restrict__ k_out,
                                                         T* __restrict__ v_out, int blocks, int Hkv, int S, int pages,
                                                         int columns, PageDiv by) {
  using L = Layout<D>;
  constexpr int LANES = L::DG / (8 * E), W = D / (8 * E);  // threads of a group, of a row
  const int b = blockIdx.x / blocks, h = blockIdx.y, w = threadIdx.x % W;
  const int64_t token = (int64_t)(blockIdx.x - b * blocks) * (256 / W) + threadIdx.x / W;
  allow_dependent_launch();
  kv4::wait_for_previous();
  if (token >= S) return;
  const int j = (int)token;
  const int g = w / LANES, c0 = g * (L::DG / 8) + w % LANES;  // chunks c0, c0 + LANES, ... of eight dims
  const int64_t to = (((int64_t)b * Hkv + h) * S + j) * D + 8 * c0;
  bool there = false;
  uint32_t kc[E], vc[E], kp, vp;
  if (j < min(lens[b], columns * by.P)) {
    const int column = by(j), off = j - column * by.P, page = table[b * ts + column];
    if (page >= 0 && page < pages) {
      const uint8_t* u = pool + (((int64_t)page * Hkv + h) * (by.P / kUnit) + off / kUnit) * L::kBytes;
      const int r = off % kUnit;
      there = true;
#pragma unroll
      for (int e = 0; e < E; ++e) {
        kc[e] = *reinterpret_cast<const uint32_t*>(u + r * L::kRow + 4 * (c0 + LANES * e));
        vc[e] = *reinterpret_cast<const uint32_t*>(u + L::kV + r * L::kRow + 4 * (c0 + LANES * e));
      }
      kp = *reinterpret_cast<const uint32_t*>(u + L::kKp + (g * kUnit + r) * 4);
      vp = *reinterpret_cast<const uint32_t*>(u + L::kVp + (g * kUnit + r) * 4);
    }
  }
#pragma unroll
  for (int e = 0; e < E; ++e) {
    float kx[8] = {}, vx[8] = {};
    if (there) values8(kc[e], kp, kx), values8(vc[e], vp, vx);
    store8(k_out + to + 8 * LANES * e, kx);
    store8(v_out + to + 8 * LANES * e, vx);
  }
}

}  // namespace
}  // namespace mb

using namespace mb;
using namespace mb::kv4;

extern "C" int motif_b200_paged_reserve(const int32_t* lens, const int32_t* new_lens, int32_t* block_table,
                                        int64_t table_stride, const int32_t* free_pages, const int32_t* free_count,
                                        int32_t* lens_out, int32_t* free_count_out, int32_t* slots, int64_t total_new,
                                        int64_t B, int64_t max_pages, int64_t free_capacity, int64_t page_size,
                                        void* stream) {
  MB_REQUIRE(((lens && new_lens && block_table && lens_out) || B == 0) && free_pages && free_count &&
                 free_count_out && (slots || total_new == 0),
             MB_ERR_ARG, "paged_reserve: null pointer");
  if (int rc = check_paging("paged_reserve", B, max_pages, table_stride, page_size)) return rc;
  // the kernel counts tokens in 32 bits and looks up to a page, and up to eight tokens a thread, ahead
  MB_REQUIRE(total_new >= 0 && total_new <= (1ll << 31) - (1 << 20), MB_ERR_SHAPE,
             "paged_reserve: %lld new tokens (0 .. 2^31 - 2^20)", (long long)total_new);
  MB_REQUIRE(free_capacity >= 1 && free_capacity * page_size < (1ll << 31), MB_ERR_SHAPE,
             "paged_reserve: free list of %lld pages", (long long)free_capacity);
  // every CTA reads the lengths, and some write: where the outputs are not the inputs themselves, whose
  // writes wait for all reads, they share nothing with them
  auto meet = [](const int32_t* p, int64_t n, const int32_t* q, int64_t m) { return p < q + m && q < p + n; };
  MB_REQUIRE((lens_out == lens || !meet(lens_out, B, lens, B)) && !meet(lens_out, B, new_lens, B) &&
                 !meet(slots, total_new, lens, B) && !meet(slots, total_new, new_lens, B) &&
                 !meet(slots, total_new, lens_out, B) && !meet(free_count_out, 1, new_lens, B) &&
                 !meet(free_count_out, 1, lens, B) && !meet(free_count_out, 1, lens_out, B),
             MB_ERR_ARG, "paged_reserve: lens_out, slots and free_count_out overlap each other or the lengths");
  const PageDiv by = page_div(page_size);
  const bool vector = reinterpret_cast<uintptr_t>(slots) % 16 == 0;
  const bool in_place = lens_out == lens || free_count_out == free_count;
  auto go = [&](auto kernel, int threads, bool many) {
    const int ctas = !many ? 1 : in_place ? kClusterCtas : kReserveCtas;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(ctas);
    cfg.blockDim = dim3(threads);
    cfg.stream = (cudaStream_t)stream;
    cudaLaunchAttribute at[2];
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    at[1].id = cudaLaunchAttributeClusterDimension;
    at[1].val.clusterDim.x = ctas;
    at[1].val.clusterDim.y = at[1].val.clusterDim.z = 1;
    cfg.attrs = at;
    cfg.numAttrs = in_place && ctas > 1 ? 2 : 1;
    cudaLaunchKernelEx(&cfg, kernel, lens, new_lens, block_table, table_stride, free_pages, free_count, lens_out,
                       free_count_out, slots, vector, in_place, (int)total_new, (int)B, (int)max_pages,
                       (int)free_capacity, by);
  };
  // a decode step's worth of requests and tokens: four warps scan faster than 16; many tokens: many
  // CTAs share the writing, from where their cost (nothing, or a cluster's barrier) is made up for:
  // 16384 tokens take 3.8 us on 64 CTAs, 4.4 on a cluster of 8, 4096 tokens 4.7 on one
  const bool many = total_new > (in_place ? 4096 : 1024);
  if (B <= 128 && total_new <= 1024) go(paged_reserve_kernel<128>, 128, false);
  else if (B <= 512) go(paged_reserve_kernel<512>, 512, many);
  else go(paged_reserve_kernel<1024>, 1024, many);
  return check_launch("paged_reserve");
}

extern "C" int motif_b200_paged_release(const uint8_t* done, int32_t* lens, int32_t* block_table, int64_t table_stride,
                                        int32_t* free_pages, int32_t* free_count, int64_t B, int64_t max_pages,
                                        int64_t free_capacity, int64_t page_size, void* stream) {
  MB_REQUIRE(((done && lens && block_table) || B == 0) && free_pages && free_count, MB_ERR_ARG,
             "paged_release: null pointer");
  if (int rc = check_paging("paged_release", B, max_pages, table_stride, page_size)) return rc;
  MB_REQUIRE(free_capacity >= 1 && free_capacity * page_size < (1ll << 31), MB_ERR_SHAPE,
             "paged_release: free list of %lld pages", (long long)free_capacity);
  if (B == 0) return MB_OK;
  launch(paged_release_kernel, dim3(1), kReleaseThreads, 0, stream, done, lens, block_table, table_stride, free_pages,
         free_count, (int)B, (int)max_pages, free_capacity, (int)page_size);
  return check_launch("paged_release");
}

extern "C" int64_t motif_b200_kv4_unit_bytes(int64_t D) { return D == 32 || D == 64 || D == 128 ? kv4::unit_bytes(D) : 0; }

extern "C" int motif_b200_kv4_append(const void* k, const void* v, const int32_t* slots, void* pool, void* k_out,
                                     void* v_out, const int64_t* strides, int64_t B, int64_t T, int64_t Hkv, int64_t D,
                                     int64_t num_pages, int64_t page_size, int dtype, void* stream) {
  MB_REQUIRE(strides && ((k && v && slots) || B * T == 0), MB_ERR_ARG, "kv4_append: null pointer");
  MB_REQUIRE((k_out == nullptr) == (v_out == nullptr), MB_ERR_ARG, "kv4_append: k_out and v_out go together");
  MB_REQUIRE(B >= 0 && T >= 0 && B * T < (1ll << 31), MB_ERR_SHAPE, "kv4_append: B %lld, T %lld", (long long)B,
             (long long)T);
  if (int rc = check_paging("kv4_append", B, 1, 1, page_size)) return rc;
  if (int rc = check_pool("kv4_append", pool, num_pages, Hkv, page_size)) return rc;
  return dispatch(dtype, D, [&](auto t, auto d) -> int {
    using E = decltype(t);
    constexpr int DD = decltype(d)::value;
    if (B * T == 0) return MB_OK;
    const void* ptrs[4] = {k, v, k_out, v_out};
    for (int i = 0; i < 4; ++i)
      if (ptrs[i])
        if (int rc = check_rows16("kv4_append", ptrs[i], strides + 3 * i, sizeof(E))) return rc;
    // 16-bit rows: two chunks a thread unless one makes at most two CTAs an SM.  Measured in CTAs of the
    // one-chunk form, one against two: 96 CTAs 2.05 us / 2.21, 192 2.91 / 2.77, 256 3.00 / 3.22 (4 heads
    // of 32) and 3.07 / 3.32 (8 of 128), 384 3.31 / 2.78, 512 3.29 / 3.49 and 3.32 / 3.45, 1024 5.90 / 4.68
    // and 5.93 / 4.71.  fp32 (one): 12.34 us / 12.54 for 4096 tokens of 8 heads of 128.
    auto go = [&](auto width, auto chunks) {
      using I = decltype(width);
      constexpr int C = decltype(chunks)::value;
      constexpr int64_t per_cta = 256 / (DD / (8 * C));
      Strides12<I> st;
      for (int i = 0; i < 12; ++i) st.s[i] = (I)strides[i];
      launch(kv4_append_kernel<E, DD, C, I>, dim3((unsigned)((B * T + per_cta - 1) / per_cta), (unsigned)Hkv), 256, 0, stream,
             (const E*)k, (const E*)v, slots, (uint8_t*)pool, (E*)k_out, (E*)v_out, st, (int)(B * T), (int)T, (int)Hkv,
             (int)(num_pages * page_size), page_div(page_size));
    };
    bool fits = true;
    for (int i = 0; i < 12; ++i) fits = fits && strides[i] >= 0 && strides[i] < (1ll << 31);
    auto go_width = [&](auto chunks) {
      if (fits) go(int32_t(), chunks);
      else go(int64_t(), chunks);
    };
    using One = std::integral_constant<int, 1>;
    using Two = std::integral_constant<int, 2>;
    if constexpr (sizeof(E) == 2) {
      if ((B * T + 2048 / DD - 1) / (2048 / DD) * Hkv > 2 * sm_count()) go_width(Two());
      else go_width(One());
    } else {
      go_width(One());
    }
    return check_launch("kv4_append");
  });
}

extern "C" int motif_b200_kv4_gather(const void* pool, const int32_t* block_table, int64_t table_stride,
                                     const int32_t* lens, void* k_out, void* v_out, int64_t B, int64_t Hkv, int64_t S,
                                     int64_t D, int64_t num_pages, int64_t page_size, int64_t max_pages, int dtype,
                                     void* stream) {
  MB_REQUIRE((block_table && lens && k_out && v_out) || B * S == 0, MB_ERR_ARG, "kv4_gather: null pointer");
  if (int rc = check_paging("kv4_gather", B, max_pages, table_stride, page_size)) return rc;
  if (int rc = check_pool("kv4_gather", pool, num_pages, Hkv, page_size)) return rc;
  MB_REQUIRE(S >= 0 && S < (1ll << 31), MB_ERR_SHAPE, "kv4_gather: length %lld", (long long)S);
  return dispatch(dtype, D, [&](auto t, auto d) -> int {
    using E = decltype(t);
    constexpr int DD = decltype(d)::value;
    if (B * S == 0) return MB_OK;
    const int64_t none[3] = {0, 0, 0};
    if (int rc = check_rows16("kv4_gather", k_out, none, 1)) return rc;
    if (int rc = check_rows16("kv4_gather", v_out, none, 1)) return rc;
    MB_REQUIRE(B * ((S + 2048 / DD - 1) / (2048 / DD)) < (1ll << 31), MB_ERR_SHAPE, "kv4_gather: %lld rows",
               (long long)(B * Hkv * S));
    auto go = [&](auto chunks) {
      constexpr int C = decltype(chunks)::value;
      constexpr int64_t per_cta = 256 / (DD / (8 * C));
      const int64_t blocks = (S + per_cta - 1) / per_cta;
      launch(kv4_gather_kernel<E, DD, C>, dim3((unsigned)(B * blocks), (unsigned)Hkv), 256, 0, stream,
             (const uint8_t*)pool, block_table, table_stride, lens, (E*)k_out, (E*)v_out, (int)blocks, (int)Hkv,
             (int)S, (int)num_pages, (int)max_pages, page_div(page_size));
    };
    // Two chunks a thread unless one would have all of its CTAs running at once (eight an SM).  Measured
    // in CTAs of the one-chunk form, one against two: 512 2.51 us / 3.63 (fp16, 8 heads of 128) and 2.60 /
    // 3.71 (bf16, 4 of 32), 768 3.22 / 2.74 (bf16, 3 of 64), 1024 3.87 / 4.24 and 3.89 / 4.23, 2048 6.45 /
    // 5.19, 32768 69.8 / 54.2; fp32, 8 heads of 128: 1024 7.50 / 9.17, 4096 20.6 / 19.7, 32768 144.6 / 133.1.
    if (B * ((S + 2048 / DD - 1) / (2048 / DD)) * Hkv > 8 * sm_count()) go(std::integral_constant<int, 2>());
    else go(std::integral_constant<int, 1>());
    return check_launch("kv4_gather");
  });
}
