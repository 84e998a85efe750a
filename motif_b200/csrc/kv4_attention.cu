// Chord attention of the newest tokens of every request over its paged 4-bit cache (kv4.cuh).
//
//   logit(r, j) = (scale q_r . k_j - alpha (|j - pos_r - mu| + eps)^beta) ssmax log(pos_r + 1),  j <= pos_r
//
// with k_j = m_j + s_j (c_j - 8) per group of dims, so
//   q . k_j          = sum_groups  s_j (q . (c_j - 8)) + m_j sum(q)
//   sum_j p_j v_j    = sum_j (p_j s_j)(c_j - 8)        + sum_j p_j m_j
// and both products run on whole numbers -8 .. 7 that every 16-bit float holds exactly: the codes
// become matrix operands without a scale, the scales are applied in fp32 to the 16 x 8 results (K)
// and to the weights (V).  The other operand is split into two 16-bit parts (q, after a power-of-two
// normalisation of its row, into fp16 high + low, 22 bits; p s into bf16 high + low, 16 bits), and
// the parts are two neighbouring columns of one MMA: with the keys on the M side a tile of 4 query
// rows fills N = 8, a thread's two accumulator columns are the two parts of ONE query row, and their
// sum is the product to fp32 accuracy at no further instruction.  The score tile [keys x (row, part)]
// is the transpose of what the second product wants: one movmatrix per 8 keys.
//
// Work is cut by tiles of 64 keys (32 for D = 128), not by requests: every warp of the grid is a
// worker and takes an equal run of the tiles of all (request, row tile, kv head) segments in order,
// so requests of any lengths load the GPU evenly, and the lengths may change on the device between
// replays of a CUDA graph.  A segment inside one worker's run is written out by it; one that spans
// workers leaves a partial (o, m, l) per worker, which the merge kernel joins in worker order.
//
// Each warp owns a ring of tiles in shared memory that lane 0 fills with bulk copies (one per tile
// where a tile lies in one page); nothing is shared between warps.
#include <math.h>

#include "common.cuh"
#include "kv4.cuh"

namespace mb {
namespace {

using kv4::kUnit;
using kv4::Layout;

__device__ unsigned int g_kv4_wait_timeouts = 0;

constexpr int kWarps = 4;
constexpr int kStages = 3;
constexpr uint32_t kWaitLimit = 1u << 20;
constexpr float kLog2e = 1.4426950408889634f;

struct Strides6 {
  int64_t s[6];  // q(b,h,t) out(b,h,t)
};

struct Args {
  const uint8_t* pool;
  const int32_t* table;
  int64_t ts;
  const int32_t* lens;
  const int32_t* q_lens;
  const float *alpha, *beta, *mu, *ssmax;
  float* ws;
  Strides6 st;
  int B, H, Hkv, T, G, Z;   // Z: row tiles of the G T query rows of one (request, kv head)
  int P, columns;
  int64_t pages;
  int workers;
  float scale, eps;
};

template <int D>
struct Tile {
  static constexpr int kUnits = D == 128 ? 2 : 4;
  static constexpr int kKeys = kUnits * kUnit;
  static constexpr int kBytes = kUnits * Layout<D>::kBytes;
};

// ------------------------------------------------------------------ the cut into workers
// Lengths are clamped to what the table can name; a request without query rows has no tiles.
__device__ __forceinline__ int length_of(const Args& a, int b) {
  return (int)max((int64_t)0, min((int64_t)a.lens[b], (int64_t)a.columns * a.P));
}
__device__ __forceinline__ int queries_of(const Args& a, int b) {
  return a.q_lens ? min(max(a.q_lens[b], 0), a.T) : a.T;
}
template <int KT>
__device__ __forceinline__ int tiles_of(const Args& a, int b) {
  return queries_of(a, b) > 0 ? (length_of(a, b) + KT - 1) / KT : 0;
}

// Exclusive prefix of the requests' tiles at each thread's run of requests (pre[0 .. threads]).
template <int KT, int THREADS>
__device__ __forceinline__ void scan_requests(const Args& a, int64_t* pre) {
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int run = (a.B + THREADS - 1) / THREADS;
  __shared__ int64_t part[THREADS / 32];
  int64_t v = 0;
  for (int b = tid * run; b < min(a.B, (tid + 1) * run); ++b) v += tiles_of<KT>(a, b);
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int64_t u = __shfl_up_sync(0xffffffffu, v, o);
    if (lane >= o) v += u;
  }
  if (lane == 31) part[warp] = v;
  __syncthreads();
  for (int w = 0; w < warp; ++w) v += part[w];
  pre[tid + 1] = v;
  if (tid == 0) pre[0] = 0;
  __syncthreads();
}

// First tile of worker w, and the worker of tile x, of `total` tiles over `n` workers.
__device__ __forceinline__ int64_t worker_start(int64_t total, int n, int64_t w) {
  return total >= n ? total * w / n : min(w, total);
}
__device__ __forceinline__ int64_t worker_of(int64_t total, int n, int64_t x) {
  return total >= n ? ((x + 1) * n - 1) / total : x;
}

// A place in the order of tiles: request, segment of it (z * Hkv + kv head), tile of the segment.
struct Cursor {
  int b, seg, k, nt;
};

template <int KT, int THREADS>
__device__ __forceinline__ Cursor locate(const Args& a, const int64_t* pre, int64_t x) {
  const int zh = a.Z * a.Hkv, lane = threadIdx.x & 31;
  const int run = (a.B + THREADS - 1) / THREADS;
  int c = 0;  // last run of requests that starts at or before x (empty ones share a start)
#pragma unroll
  for (int i = 0; i < THREADS / 32; ++i)
    c += __popc(__ballot_sync(0xffffffffu, pre[i * 32 + lane + 1] * zh <= x));
  int64_t left = x - pre[c] * zh;
  Cursor u;
  u.b = c * run;
  while (true) {
    u.nt = tiles_of<KT>(a, u.b);
    if (left < (int64_t)u.nt * zh || u.b + 1 >= a.B) break;
    left -= (int64_t)u.nt * zh;
    ++u.b;
  }
  u.seg = (int)(left / max(u.nt, 1));
  u.k = (int)(left % max(u.nt, 1));
  return u;
}
template <int KT>
__device__ __forceinline__ void advance(const Args& a, Cursor& u) {
  if (++u.k < u.nt) return;
  u.k = 0;
  if (++u.seg < a.Z * a.Hkv) return;
  u.seg = 0;
  do {
    if (++u.b >= a.B) return;
    u.nt = tiles_of<KT>(a, u.b);
  } while (u.nt == 0);
}

// ------------------------------------------------------------------ small device helpers
__device__ __forceinline__ uint32_t lop_and_or(uint32_t a, uint32_t b, uint32_t c) {  // (a & b) | c
  uint32_t r;
  asm("lop3.b32 %0, %1, %2, %3, 0xEA;" : "=r"(r) : "r"(a), "r"(b), "r"(c));
  return r;
}
__device__ __forceinline__ uint32_t hadd2(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("add.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}
__device__ __forceinline__ uint32_t hfma2(uint32_t a, uint32_t b, uint32_t c) {
  uint32_t r;
  asm("fma.rn.f16x2 %0, %1, %2, %3;" : "=r"(r) : "r"(a), "r"(b), "r"(c));
  return r;
}
__device__ __forceinline__ uint32_t badd2(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("add.rn.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}
__device__ __forceinline__ uint32_t transpose8x8(uint32_t a) {
  uint32_t r;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(a));
  return r;
}

// Codes of eight dims as four fp16 pairs c - 8: pair i holds dims (i, i + 4).  0x6400 is 1024, whose
// last mantissa bit is 1: OR-ing a nibble into bits 0..3 adds it, into bits 4..7 adds 16 times it.
__device__ __forceinline__ void codes_f16(uint32_t w, uint32_t* h) {
  const uint32_t v = w >> 8;
  h[0] = hadd2(lop_and_or(w, 0x000f000fu, 0x64006400u), 0xe408e408u);                // - 1032
  h[1] = hfma2(lop_and_or(w, 0x00f000f0u, 0x64006400u), 0x2c002c00u, 0xd480d480u);   // / 16 - 72
  h[2] = hadd2(lop_and_or(v, 0x000f000fu, 0x64006400u), 0xe408e408u);
  h[3] = hfma2(lop_and_or(v, 0x00f000f0u, 0x64006400u), 0x2c002c00u, 0xd480d480u);
}
// Four codes of two keys (low halves of the pair: one key, high: the other) as bf16 pairs c - 8
// (0x4300 is 128, last mantissa bit 1).
__device__ __forceinline__ void codes_bf16(uint32_t x, uint32_t* h) {
#pragma unroll
  for (int i = 0; i < 4; ++i) h[i] = badd2(lop_and_or(x >> (4 * i), 0x000f000fu, 0x43004300u), 0xc308c308u);  // - 136
}

// Place of row r of a group of 8 keys: rows 2t, 2t + 1 are keys t, t + 4, so that the four lanes of a
// V load take neighbouring keys (128 consecutive bytes of shared memory per load).
__device__ __forceinline__ int key_of_row(int r) { return (r >> 1) + 4 * (r & 1); }

// ------------------------------------------------------------------ the worker kernel
template <typename T, int D, int NT>
__global__ void __launch_bounds__(32 * kWarps) kv4_attention_kernel(const T* __restrict__ q, T* __restrict__ out,
                                                                    const Args a) {
  using L = Layout<D>;
  constexpr int TU = Tile<D>::kUnits, KT = Tile<D>::kKeys;
  constexpr int NG = L::NG, DG = L::DG;
  constexpr int KW = DG / 32;        // 32-bit words of K codes of a thread per row and group
  constexpr int MT = DG / 16;        // 16-dim output tiles of a group
  constexpr int RT = 4 * NT;         // query rows of a row tile
  constexpr int THREADS = 32 * kWarps;
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ int64_t pre[THREADS + 1];
  __shared__ __align__(8) uint64_t bars[kWarps][kStages];

  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int g8 = lane >> 2, t4 = lane & 3;
  uint8_t* ring = smem + warp * (kStages * Tile<D>::kBytes);
  uint64_t* bar = bars[warp];
  if (lane == 0) {
    for (int s = 0; s < kStages; ++s) mbar_init(&bar[s], 1);
    mbar_init_fence();
  }
  scan_requests<KT, THREADS>(a, pre);
  allow_dependent_launch();  // the merge may take its place; it waits for this grid to end

  const int zh = a.Z * a.Hkv;
  const int64_t total = pre[THREADS] * zh;
  // worker numbers run over the CTAs first: few tiles spread over all SMs
  const int worker = warp * gridDim.x + blockIdx.x;
  const int64_t first = worker_start(total, a.workers, worker);
  const int64_t count = worker_start(total, a.workers, worker + 1) - first;
  if (count <= 0) return;
  Cursor cur = locate<KT, THREADS>(a, pre, first);
  Cursor ahead = cur;

  const int UP = a.P / kUnit;
  const bool one_copy = UP % TU == 0;  // a tile's units lie in one page, next to each other
  // Page of this lane's unit (lane & 3, where it is one) of the tile at `ahead`, -1: none.
  int pid = -1, usub = 0, useg = 0;
  auto look = [&]() {
    const int u = ahead.k * TU + lane;
    pid = -1;
    useg = ahead.seg;
    if (lane < TU && u * kUnit < length_of(a, ahead.b)) {
      pid = a.table[(int64_t)ahead.b * a.ts + u / UP];
      usub = u % UP;
    }
  };
  uint32_t valid = 0;  // bits of the units of the tiles in the ring, TU per stage
  auto issue = [&](int s) {
    const bool ok = pid >= 0 && pid < a.pages;
    const uint32_t mask = __ballot_sync(0xffffffffu, ok);
    valid = (valid & ~(((1u << TU) - 1) << (TU * s))) | (mask << (TU * s));
    const uint32_t bytes = __popc(mask) * L::kBytes;
    if (lane == 0) mbar_arrive_expect_tx(&bar[s], bytes);
    __syncwarp();
    if (ok && (lane == 0 || !one_copy)) {
      const uint8_t* src = a.pool + (((int64_t)pid * a.Hkv + useg % a.Hkv) * UP + usub) * (int64_t)L::kBytes;
      bulk_load(ring + s * Tile<D>::kBytes + lane * L::kBytes, src, one_copy ? bytes : L::kBytes, &bar[s]);
    }
  };
  for (int s = 0; s < kStages; ++s) {
    if (s >= count) break;
    if (s) advance<KT>(a, ahead);
    look();
    issue(s);
  }
  int64_t looked = min((int64_t)kStages, count);  // tiles issued; the next one's page is read one tile early
  if (looked < count) {
    advance<KT>(a, ahead);
    look();
  }

  // state of the current segment
  uint32_t qf[NT][NG][2 * KW][2];
  float sq[NT][NG], qsc[NT], rc[NT], al[NT], be[NT], mh[NT];
  int pos[NT];
  float o[NT][NG][MT][4], m[NT], l[NT], pm[NT][NG];
  int lo_pos = 0;  // smallest position of a row that sees keys

  bool fresh = true, from_start = true;
  for (int64_t i = 0; i < count; ++i) {
    if (fresh) {
      fresh = false;
      from_start = cur.k == 0;
      const int hk = cur.seg % a.Hkv, z = cur.seg / a.Hkv;
      const int nq = queries_of(a, cur.b), base = length_of(a, cur.b) - nq;
      const int rows = a.G * a.T;
      lo_pos = max(0, base + z * RT / a.G);
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        // the query row whose scores this thread holds
        const int r = min(z * RT + n * 4 + t4, rows - 1);
        const int h = hk * a.G + r % a.G;
        pos[n] = max(0, base + min(r / a.G, nq - 1));
        rc[n] = a.ssmax[h] * logf((float)pos[n] + 1.f) * kLog2e;
        al[n] = -a.alpha[h];
        be[n] = a.beta[h];
        mh[n] = a.mu[h];
        // the query row of this thread's B fragments: column g8 = (row g8 / 2, part g8 & 1)
        const int r2 = min(z * RT + n * 4 + (g8 >> 1), rows - 1);
        const T* qp = q + cur.b * a.st.s[0] + (hk * a.G + r2 % a.G) * a.st.s[1] + (r2 / a.G) * a.st.s[2];
        float x[NG][8 * KW], top = 0.f;
#pragma unroll
        for (int g = 0; g < NG; ++g)
#pragma unroll
          for (int e = 0; e < 8 * KW; ++e) {
            x[g][e] = to_f(qp[g * DG + t4 * 8 * KW + e]);
            top = fmaxf(top, fabsf(x[g][e]));
          }
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
        // power of two that brings the row's largest value to 2^13 .. 2^14 (fp16 ends at 2^16)
        const int ex = min(max((int)(__float_as_uint(top) >> 23) - 127, -112), 127);
        const float up = __uint_as_float((uint32_t)(13 - ex + 127) << 23);
        const float down = __uint_as_float((uint32_t)(ex - 13 + 127) << 23);
#pragma unroll
        for (int g = 0; g < NG; ++g) {
          float sum = 0.f, part[8 * KW];
#pragma unroll
          for (int e = 0; e < 8 * KW; ++e) {
            const float y = x[g][e] * up, hi = __half2float(__float2half_rn(y));
            part[e] = (g8 & 1) ? __half2float(__float2half_rn(y - hi)) : hi;
            sum += part[e];
          }
#pragma unroll
          for (int w = 0; w < KW; ++w)
#pragma unroll
            for (int p = 0; p < 2; ++p) {
              qf[n][g][2 * w + p][0] = pack2<__half>(part[8 * w + 2 * p], part[8 * w + 2 * p + 4]);
              qf[n][g][2 * w + p][1] = pack2<__half>(part[8 * w + 2 * p + 1], part[8 * w + 2 * p + 5]);
            }
          sum += __shfl_xor_sync(0xffffffffu, sum, 1);
          sum += __shfl_xor_sync(0xffffffffu, sum, 2);
          sum += __shfl_xor_sync(0xffffffffu, sum, 4);
          sq[n][g] = __shfl_sync(0xffffffffu, sum, 8 * t4);
        }
        qsc[n] = a.scale * __shfl_sync(0xffffffffu, down, 8 * t4);
        m[n] = -INFINITY;
        l[n] = 0.f;
#pragma unroll
        for (int g = 0; g < NG; ++g) {
          pm[n][g] = 0.f;
#pragma unroll
          for (int t = 0; t < MT; ++t) o[n][g][t][0] = o[n][g][t][1] = o[n][g][t][2] = o[n][g][t][3] = 0.f;
        }
      }
    }

    const int s = (int)(i % kStages);
    if (!__all_sync(0xffffffffu, mbar_wait_bounded(&bar[s], (uint32_t)((i / kStages) & 1), kWaitLimit))) {
      // never expected: the error is counted, copies in flight are waited for, the rows stay unwritten
      if (lane == 0) atomicAdd(&g_kv4_wait_timeouts, 1u);
      for (int64_t j = i + 1; j < looked; ++j)
        mbar_wait_bounded(&bar[j % kStages], (uint32_t)((j / kStages) & 1), kWaitLimit);
      return;
    }
    const uint8_t* tile = ring + s * Tile<D>::kBytes;
    const uint32_t units = (valid >> (TU * s)) & ((1u << TU) - 1);
    const int k0 = cur.k * KT;
    // every key of the tile is there and visible to every row
    const bool whole = units == (1u << TU) - 1 && k0 + KT - 1 <= lo_pos;

    float x[NT][TU][2];
    float top[NT];
#pragma unroll
    for (int n = 0; n < NT; ++n) top[n] = -INFINITY;
#pragma unroll
    for (int u = 0; u < TU; ++u) {
      const uint8_t* unit = tile + u * L::kBytes;
      float dot[NT][2];
#pragma unroll
      for (int n = 0; n < NT; ++n) dot[n][0] = dot[n][1] = 0.f;
      const int r0 = key_of_row(g8);
#pragma unroll
      for (int g = 0; g < NG; ++g) {
        uint32_t w0[KW], w1[KW];
        const uint8_t* at = unit + r0 * L::kRow + g * (DG / 2) + t4 * (4 * KW);
        if constexpr (KW == 2) {
          const uint2 y0 = *reinterpret_cast<const uint2*>(at), y1 = *reinterpret_cast<const uint2*>(at + 8 * L::kRow);
          w0[0] = y0.x, w0[1] = y0.y, w1[0] = y1.x, w1[1] = y1.y;
        } else {
          w0[0] = *reinterpret_cast<const uint32_t*>(at);
          w1[0] = *reinterpret_cast<const uint32_t*>(at + 8 * L::kRow);
        }
        float acc[NT][4];
#pragma unroll
        for (int n = 0; n < NT; ++n) acc[n][0] = acc[n][1] = acc[n][2] = acc[n][3] = 0.f;
#pragma unroll
        for (int w = 0; w < KW; ++w) {
          uint32_t c0[4], c1[4];
          codes_f16(w0[w], c0);
          codes_f16(w1[w], c1);
#pragma unroll
          for (int p = 0; p < 2; ++p) {
            const uint32_t af[4] = {c0[2 * p], c1[2 * p], c0[2 * p + 1], c1[2 * p + 1]};
#pragma unroll
            for (int n = 0; n < NT; ++n) mma_16816<__half>(acc[n], af, qf[n][g][2 * w + p]);
          }
        }
        const uint32_t* kp = reinterpret_cast<const uint32_t*>(unit + L::kKp) + g * kUnit + r0;
        const uint32_t p0 = kp[0], p1 = kp[8];
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          dot[n][0] = fmaf(kv4::pair_scale(p0), acc[n][0] + acc[n][1], fmaf(kv4::pair_centre(p0), sq[n][g], dot[n][0]));
          dot[n][1] = fmaf(kv4::pair_scale(p1), acc[n][2] + acc[n][3], fmaf(kv4::pair_centre(p1), sq[n][g], dot[n][1]));
        }
      }
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int key = u * kUnit + r0 + 8 * e;
          const float dist = fabsf((float)(k0 + key - pos[n]) - mh[n]) + a.eps;
          float bias;
          if constexpr (sizeof(T) == 4) {
            bias = al[n] * powf(dist, be[n]);
          } else {
            bias = al[n] * ex2f_(be[n] * __log2f(dist));
          }
          float y = fmaf(dot[n][e], qsc[n], bias) * rc[n];
          if (!whole && (!((units >> u) & 1u) || k0 + key > pos[n])) y = -INFINITY;
          x[n][u][e] = y;
          top[n] = fmaxf(top[n], y);
        }
    }

#pragma unroll
    for (int n = 0; n < NT; ++n) {
#pragma unroll
      for (int d = 4; d < 32; d <<= 1) top[n] = fmaxf(top[n], __shfl_xor_sync(0xffffffffu, top[n], d));
      const float mn = fmaxf(m[n], top[n]);
      const float shift = mn == -INFINITY ? 0.f : mn;
      const float f = exp2f(m[n] - shift);
      m[n] = mn;
      l[n] *= f;
#pragma unroll
      for (int g = 0; g < NG; ++g) {
        pm[n][g] *= f;
#pragma unroll
        for (int t = 0; t < MT; ++t)
#pragma unroll
          for (int e = 0; e < 4; ++e) o[n][g][t][e] *= f;
      }
#pragma unroll
      for (int u = 0; u < TU; ++u)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const float p = sizeof(T) == 4 ? exp2f(x[n][u][e] - shift) : ex2f_(x[n][u][e] - shift);
          x[n][u][e] = p;
          l[n] += p;
        }
    }

#pragma unroll
    for (int u = 0; u < TU; ++u) {
      const uint8_t* unit = tile + u * L::kBytes;
      const int r0 = key_of_row(g8);
#pragma unroll
      for (int g = 0; g < NG; ++g) {
        const uint32_t* vp = reinterpret_cast<const uint32_t*>(unit + L::kVp) + g * kUnit + r0;
        uint32_t pr[2] = {vp[0], vp[8]};
        uint32_t bf[NT][2];
#pragma unroll
        for (int e = 0; e < 2; ++e)
#pragma unroll
          for (int n = 0; n < NT; ++n) {
            // a key that is not there may have any pair: its weight is 0, its product must be too
            const bool there = whole || x[n][u][e] != 0.f;
            const float ps = there ? x[n][u][e] * kv4::pair_scale(pr[e]) : 0.f;
            pm[n][g] = there ? fmaf(x[n][u][e], kv4::pair_centre(pr[e]), pm[n][g]) : pm[n][g];
            const float hi = __bfloat162float(__float2bfloat16_rn(ps));
            bf[n][e] = transpose8x8(pack2<__nv_bfloat16>(hi, ps - hi));
          }
        const uint8_t* at = unit + L::kV + t4 * L::kRow + g * (DG / 2) + (KW == 2 ? 4 * g8 : 4 * (g8 >> 1));
        uint32_t w[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) w[j] = *reinterpret_cast<const uint32_t*>(at + 4 * j * L::kRow);
#pragma unroll
        for (int hf = 0; hf < KW; ++hf) {  // halves of a word: four dims each
          const uint32_t sel = KW == 2 ? (hf ? 0x7632u : 0x5410u) : ((g8 & 1) ? 0x7632u : 0x5410u);
          uint32_t c0[4], c1[4];
          codes_bf16(__byte_perm(w[0], w[1], sel), c0);
          codes_bf16(__byte_perm(w[2], w[3], sel), c1);
#pragma unroll
          for (int p = 0; p < 2; ++p) {
            const uint32_t af[4] = {c0[2 * p], c0[2 * p + 1], c1[2 * p], c1[2 * p + 1]};
#pragma unroll
            for (int n = 0; n < NT; ++n) mma_16816<__nv_bfloat16>(o[n][g][2 * hf + p], af, bf[n]);
          }
        }
      }
    }

    __syncwarp();  // every lane is done with the stage
    if (looked < count) {
      fence_proxy_async_smem();
      issue(s);
      if (++looked < count) {
        advance<KT>(a, ahead);
        look();
      }
    }

    const bool ends = cur.k + 1 == cur.nt;
    if (ends || i + 1 == count) {
      const int hk = cur.seg % a.Hkv, z = cur.seg / a.Hkv;
      const int nq = queries_of(a, cur.b), base = length_of(a, cur.b) - nq;
      const bool direct = ends && from_start;
      // partial slot: 0 where the segment began before this worker's run, 1 where it began in it
      float* part = a.ws + ((int64_t)worker * 2 + (from_start ? 1 : 0)) * RT * (D + 4);
#pragma unroll
      for (int n = 0; n < NT; ++n) {
#pragma unroll
        for (int d = 4; d < 32; d <<= 1) {
          l[n] += __shfl_xor_sync(0xffffffffu, l[n], d);
#pragma unroll
          for (int g = 0; g < NG; ++g) pm[n][g] += __shfl_xor_sync(0xffffffffu, pm[n][g], d);
        }
        const int r = z * RT + n * 4 + t4;
        const int t = r / a.G;
        const bool sees = t < nq && base + t >= 0;
        const float inv = direct ? (sees && l[n] != 0.f ? 1.f / l[n] : 0.f) : 1.f;
        if (r < a.G * a.T) {
#pragma unroll
          for (int g = 0; g < NG; ++g) {
            float y[2 * MT];
#pragma unroll
            for (int j = 0; j < MT; ++j) {
              y[2 * j] = (o[n][g][j][0] + o[n][g][j][1] + pm[n][g]) * inv;
              y[2 * j + 1] = (o[n][g][j][2] + o[n][g][j][3] + pm[n][g]) * inv;
            }
            const int d0 = g * DG + g8 * 2 * MT;
            if (direct) {
              T* dst = out + cur.b * a.st.s[3] + (hk * a.G + r % a.G) * a.st.s[4] + t * a.st.s[5] + d0;
#pragma unroll
              for (int j = 0; j < 2 * MT; ++j) dst[j] = from_f<T>(sees ? y[j] : 0.f);
            } else {
              float* dst = part + (n * 4 + t4) * (D + 4) + d0;
#pragma unroll
              for (int j = 0; j < 2 * MT; j += 4)
                *reinterpret_cast<float4*>(dst + j) = make_float4(y[j], y[j + 1], y[j + 2], y[j + 3]);
            }
          }
          if (!direct && g8 == 0) {
            part[(n * 4 + t4) * (D + 4) + D] = m[n];
            part[(n * 4 + t4) * (D + 4) + D + 1] = l[n];
          }
        }
      }
      fresh = true;
    }
    advance<KT>(a, cur);
  }
}

// ------------------------------------------------------------------ merge
// One CTA per (request, row tile, kv head): joins the workers' partials of a segment that spans
// several, in worker order, and zeroes the rows of a segment without tiles.  A warp takes every
// fourth row, its lanes D / 32 dims.
template <typename T, int D, int NT>
__global__ void __launch_bounds__(128) kv4_merge_kernel(T* __restrict__ out, const Args a) {
  constexpr int KT = Tile<D>::kKeys, RT = 4 * NT, E = D / 32;
  __shared__ int64_t pre[129];
  scan_requests<KT, 128>(a, pre);
  const int zh = a.Z * a.Hkv, run = (a.B + 127) / 128;
  const int b = blockIdx.x / zh, seg = blockIdx.x % zh;
  const int hk = seg % a.Hkv, z = seg / a.Hkv;
  int64_t before = pre[b / run];
  for (int i = b / run * run; i < b; ++i) before += tiles_of<KT>(a, i);
  const int64_t total = pre[128] * zh;
  const int nt = tiles_of<KT>(a, b);
  const int64_t x0 = before * zh + (int64_t)seg * nt;
  int64_t w0 = 0, w1 = 0;
  if (nt > 0) {
    w0 = worker_of(total, a.workers, x0);
    w1 = worker_of(total, a.workers, x0 + nt - 1);
  }
  // every CTA waits, also those without work: what follows this grid must find the workers' done
  asm volatile("griddepcontrol.wait;" ::: "memory");
  if (nt > 0 && w0 == w1) return;  // written by its worker
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int nq = queries_of(a, b), base = length_of(a, b) - nq;
  for (int rr = warp; rr < RT; rr += 4) {
    const int r = z * RT + rr;
    if (r >= a.G * a.T) break;
    const int t = r / a.G;
    T* dst = out + b * a.st.s[3] + (hk * a.G + r % a.G) * a.st.s[4] + t * a.st.s[5] + lane * E;
    float acc[E], mx = -INFINITY, den = 0.f;
#pragma unroll
    for (int e = 0; e < E; ++e) acc[e] = 0.f;
    if (nt > 0 && t < nq && base + t >= 0) {
      // the first worker's slot 1 where the segment began in its run, every other one's slot 0
      auto slot = [&](int64_t w) { return a.ws + ((w * 2 + (w == w0 ? 1 : 0)) * RT + rr) * (D + 4); };
      for (int64_t w = w0 + lane; w <= w1; w += 32) mx = fmaxf(mx, slot(w)[D]);
      mx = warp_max(mx);
      if (mx == -INFINITY) mx = 0.f;
      for (int64_t wb = w0; wb <= w1; wb += 32) {
        float f = 0.f;
        if (wb + lane <= w1) {
          f = exp2f(slot(wb + lane)[D] - mx);
          den = fmaf(f, slot(wb + lane)[D + 1], den);
        }
        const int n = (int)min((int64_t)32, w1 - wb + 1);
#pragma unroll 8
        for (int i = 0; i < n; ++i) {
          const float fi = __shfl_sync(0xffffffffu, f, i);
          const float* src = slot(wb + i) + lane * E;
#pragma unroll
          for (int e = 0; e < E; ++e) acc[e] = fmaf(fi, src[e], acc[e]);
        }
      }
      den = warp_sum(den);
    }
    const float inv = den != 0.f ? 1.f / den : 0.f;
#pragma unroll
    for (int e = 0; e < E; ++e) dst[e] = from_f<T>(acc[e] * inv);
  }
}

// ------------------------------------------------------------------ host side
// Rows of one row tile: 4, 8 or 16 query rows (NT score columns per thread); 8 at most for D = 128,
// whose output tile is twice as wide.
int row_tile(int64_t rows, int64_t D) {
  if (rows <= 4) return 1;
  return rows <= 8 || D == 128 ? 2 : 4;
}

int sm_count() {
  int dev = 0, n = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return 0;
  if (cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess) return 0;
  return n;
}

constexpr int kCtasPerSm = 4;

template <typename T, int D, int NT>
int launch(const void* q, void* out, Args a, cudaStream_t stream) {
  constexpr int smem = kWarps * kStages * Tile<D>::kBytes;
  const void* fn = reinterpret_cast<const void*>(&kv4_attention_kernel<T, D, NT>);
  if (int rc = ensure_smem_attr(fn, smem)) return rc;
  kv4_attention_kernel<T, D, NT><<<a.workers / kWarps, 32 * kWarps, smem, stream>>>((const T*)q, (T*)out, a);
  if (int rc = check_launch("kv4_chord_attention")) return rc;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)((int64_t)a.B * a.Z * a.Hkv));
  cfg.blockDim = dim3(128);
  cfg.stream = stream;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  cudaLaunchKernelEx(&cfg, kv4_merge_kernel<T, D, NT>, (T*)out, (const Args)a);
  return check_launch("kv4_chord_attention (merge)");
}

}  // namespace

int read_and_clear_kv4_timeouts(unsigned int* count) {
  unsigned int v = 0, zero = 0;
  if (cudaMemcpyFromSymbol(&v, g_kv4_wait_timeouts, sizeof(v)) != cudaSuccess ||
      cudaMemcpyToSymbol(g_kv4_wait_timeouts, &zero, sizeof(zero)) != cudaSuccess)
    return set_error(MB_ERR_CUDA, "wait_timeouts: %s", cudaGetErrorString(cudaGetLastError()));
  *count = v;
  return MB_OK;
}

}  // namespace mb

using namespace mb;
using namespace mb::kv4;

extern "C" int64_t motif_b200_kv4_attention_workspace_bytes(int64_t H, int64_t Hkv, int64_t T, int64_t D) {
  if (Hkv < 1 || H < Hkv || T < 1) return 0;
  return (int64_t)sm_count() * kCtasPerSm * kWarps * 2 * 4 * row_tile(H / Hkv * T, D) * (D + 4) * 4;
}

extern "C" int motif_b200_kv4_chord_attention(const void* q, const void* pool, const int32_t* block_table,
                                              int64_t table_stride, const int32_t* lens, const int32_t* q_lens,
                                              const float* alpha, const float* beta, const float* mu,
                                              const float* ssmax, void* out, const int64_t* strides, int64_t B,
                                              int64_t H, int64_t Hkv, int64_t T, int64_t D, int64_t num_pages,
                                              int64_t page_size, int64_t max_pages, float scale, float eps,
                                              void* workspace, int64_t workspace_bytes, int dtype, void* stream) {
  MB_REQUIRE(strides && alpha && beta && mu && ssmax && ((q && out && block_table && lens) || B * T == 0), MB_ERR_ARG,
             "kv4_chord_attention: null pointer");
  if (int rc = check_paging("kv4_chord_attention", B, max_pages, table_stride, page_size)) return rc;
  if (int rc = check_pool("kv4_chord_attention", pool, num_pages, Hkv, page_size)) return rc;
  MB_REQUIRE(H >= 1 && H % Hkv == 0, MB_ERR_SHAPE, "kv4_chord_attention: %lld heads not divisible by %lld kv heads",
             (long long)H, (long long)Hkv);
  MB_REQUIRE(T >= 0 && H * T < (1ll << 24) && B * H * T < (1ll << 31), MB_ERR_SHAPE,
             "kv4_chord_attention: B %lld, H %lld, T %lld", (long long)B, (long long)H, (long long)T);
  return dispatch(dtype, D, [&](auto t, auto d) -> int {
    using E = decltype(t);
    constexpr int DD = decltype(d)::value;
    if (B * T == 0) return MB_OK;
    const int64_t need = motif_b200_kv4_attention_workspace_bytes(H, Hkv, T, D);
    MB_REQUIRE(need > 0 && workspace && workspace_bytes >= need, MB_ERR_ARG,
               "kv4_chord_attention: workspace of %lld bytes, %lld given", (long long)need,
               (long long)(workspace ? workspace_bytes : 0));
    MB_REQUIRE(reinterpret_cast<uintptr_t>(workspace) % 16 == 0, MB_ERR_ALIGN,
               "kv4_chord_attention: the workspace must be 16-byte aligned");
    Args a;
    a.pool = (const uint8_t*)pool;
    a.table = block_table;
    a.ts = table_stride;
    a.lens = lens;
    a.q_lens = q_lens;
    a.alpha = alpha, a.beta = beta, a.mu = mu, a.ssmax = ssmax;
    a.ws = (float*)workspace;
    for (int i = 0; i < 6; ++i) a.st.s[i] = strides[i];
    a.B = (int)B, a.H = (int)H, a.Hkv = (int)Hkv, a.T = (int)T, a.G = (int)(H / Hkv);
    a.P = (int)page_size, a.columns = (int)max_pages, a.pages = num_pages;
    a.scale = scale, a.eps = eps;
    const int nt = row_tile((int64_t)a.G * T, D);
    a.Z = (int)(((int64_t)a.G * T + 4 * nt - 1) / (4 * nt));
    a.workers = sm_count() * kCtasPerSm * kWarps;
    MB_REQUIRE((int64_t)a.B * a.Z * a.Hkv < (1ll << 31), MB_ERR_SHAPE, "kv4_chord_attention: too many rows");
    if (nt == 1) return launch<E, DD, 1>(q, out, a, (cudaStream_t)stream);
    if constexpr (DD < 128)
      if (nt == 4) return launch<E, DD, 4>(q, out, a, (cudaStream_t)stream);
    return launch<E, DD, 2>(q, out, a, (cudaStream_t)stream);
  });
}
