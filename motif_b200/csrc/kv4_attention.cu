// Chord attention of the newest tokens of every request over its paged 4-bit cache (kv4.cuh).
//
//   logit(r, j) = (scale q_r . k_j - alpha (|j - pos_r - mu| + eps)^beta) ssmax log(pos_r + 1),  j <= pos_r
//
// with k_j = m_j + s_j (c_j - 8) per group of dims, so
//   q . k_j          = sum_groups  s_j (q . c_j - 8 sum(q)) + m_j sum(q)
//   sum_j p_j v_j    = sum_j (p_j s_j) c_j                  + sum_j p_j (m_j - 8 s_j)
// and both products run on the codes themselves.  A code in bits 0..3 of an fp16 IS the number
// c 2^-24, in bits 4..7 c 2^-20 (subnormal, exact, and the tensor cores take them as they are), so a
// packed word becomes matrix operands with one AND per pair and no conversion; the powers of two are
// undone in fp32.  The other operand is split into two fp16 parts of 11 bits each (q after a
// power-of-two normalisation of its row, p s against the largest scale so far), and the parts are
// two neighbouring columns of one MMA: with the keys on the M side a tile of 4 query rows fills
// N = 8, a thread's two accumulator columns are the two parts of ONE query row, and their sum is the
// product to 22 bits at no further instruction.  The score tile [keys x (row, part)] is the transpose
// of what the second product wants: one movmatrix per 8 keys.
//
// Work is cut by tiles of 64 keys (32 for D = 128), not by requests: the tiles of all (request, row
// tile, kv head) segments in order are dealt out in equal runs to the CTAs and within them to the
// warps, so requests of any lengths load the GPU evenly, and the lengths may change on the device
// between replays of a CUDA graph.  A segment inside one warp's run is written out by it; one that
// spans warps is joined in shared memory, one that spans CTAs leaves a partial (o, m, l) per CTA,
// which the merge kernel joins in CTA order.
//
// Each warp owns a ring of tiles in shared memory that its first lanes fill with bulk copies (one per
// tile where a tile lies in one page).
#include <math.h>

#include "common.cuh"
#include "kv4.cuh"

namespace mb {
namespace {

using kv4::kUnit;
using kv4::Layout;

__device__ unsigned int g_kv4_wait_timeouts = 0;

constexpr int kWarps = 4;
constexpr int kStages = 2;
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
  int ctas;
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

// `total` tiles over at most `n` CTAs, at least one tile per warp: the number of CTAs that work, the
// first tile of CTA c of `m` working ones, and the CTA of tile x.
__device__ __forceinline__ int64_t working_ctas(int64_t total, int n) {
  return min((int64_t)n, (total + kWarps - 1) / kWarps);
}
__device__ __forceinline__ int64_t cta_start(int64_t total, int64_t m, int64_t c) { return total * c / m; }
__device__ __forceinline__ int64_t cta_of(int64_t total, int64_t m, int64_t x) { return ((x + 1) * m - 1) / total; }

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
__device__ __forceinline__ bool advance(const Args& a, Cursor& u) {  // true: another segment
  if (++u.k < u.nt) return false;
  u.k = 0;
  if (++u.seg < a.Z * a.Hkv) return true;
  u.seg = 0;
  do {
    if (++u.b >= a.B) return true;
    u.nt = tiles_of<KT>(a, u.b);
  } while (u.nt == 0);
  return true;
}

// ------------------------------------------------------------------ small device helpers
__device__ __forceinline__ uint32_t transpose8x8(uint32_t a) {
  uint32_t r;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(a));
  return r;
}
__device__ __forceinline__ float lg2_(float x) {
  float y;
  asm("lg2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float pow2(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }  // -126 .. 127

// D = A B + C on fp16 operands with C in registers of its own.
__device__ __forceinline__ void mma_f16(float* d, const uint32_t* a, const uint32_t* b, float c0, float c1, float c2,
                                        float c3) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
      "{%10,%11,%12,%13};\n"
      : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b[0]), "r"(b[1]), "f"(c0), "f"(c1), "f"(c2), "f"(c3));
}

// The nibbles of w as four fp16 pairs: nibbles (0, 4) and (2, 6) times 2^-24, (1, 5) and (3, 7) times 2^-20.
__device__ __forceinline__ void codes(uint32_t w, uint32_t* h) {
  const uint32_t v = w >> 8;
  h[0] = w & 0x000f000fu;
  h[1] = w & 0x00f000f0u;
  h[2] = v & 0x000f000fu;
  h[3] = v & 0x00f000f0u;
}

// Place of row r of a group of 8 keys: rows 2t, 2t + 1 are keys t, t + 4, so that the four lanes of a
// V load take neighbouring keys (128 consecutive bytes of shared memory per load).
__device__ __forceinline__ int key_of_row(int r) { return (r >> 1) + 4 * (r & 1); }

// ------------------------------------------------------------------ the worker kernel
// An unfinished piece of a segment at the end of a warp's run: [RT rows][D + 4] floats (o, m, l), its
// segment (request * Z * Hkv + seg, -1: none) and whether it holds the segment's first / last tile.
struct Piece {
  int64_t segment;
  int begins, ends;
};
template <int D, int NT>
constexpr int piece_floats() {
  return 4 * NT * (D + 4);
}
// A warp's last piece takes its ring's place, which is free by then; one that a segment from before
// the run leaves on the way needs its own.
template <int D, int NT>
constexpr int attention_smem() {
  static_assert(piece_floats<D, NT>() * 4 <= kStages * Tile<D>::kBytes, "a piece fits the ring");
  return kWarps * (kStages * Tile<D>::kBytes + piece_floats<D, NT>() * 4);
}

// CTAs per SM of the worker kernel, by the registers its output tile leaves.
__host__ __device__ constexpr int ctas_per_sm(int nt, int D) { return nt == 1 ? (D <= 64 ? 4 : 3) : nt == 2 && D <= 64 ? 3 : 2; }

template <typename T, int D, int NT>
__global__ void __launch_bounds__(32 * kWarps, ctas_per_sm(NT, D)) kv4_attention_kernel(const T* __restrict__ q, T* __restrict__ out,
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
  __shared__ Piece pieces[kWarps][2];

  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int g8 = lane >> 2, t4 = lane & 3;
  uint8_t* ring = smem + warp * (kStages * Tile<D>::kBytes);
  auto piece_at = [&](int w, int which) {
    return reinterpret_cast<float*>(which ? smem + w * (kStages * Tile<D>::kBytes)
                                          : smem + kWarps * (kStages * Tile<D>::kBytes) + w * piece_floats<D, NT>() * 4);
  };
  uint64_t* bar = bars[warp];
  if (lane == 0) {
    for (int s = 0; s < kStages; ++s) mbar_init(&bar[s], 1);
    mbar_init_fence();
    pieces[warp][0].segment = pieces[warp][1].segment = -1;
  }
  scan_requests<KT, THREADS>(a, pre);
  allow_dependent_launch();  // the merge may take its place; it waits for this grid to end

  const int zh = a.Z * a.Hkv;
  const int64_t total = pre[THREADS] * zh;
  const int64_t working = working_ctas(total, gridDim.x);
  if (blockIdx.x >= working) return;
  const int64_t cta_first = cta_start(total, working, blockIdx.x);
  const int cta_count = (int)(cta_start(total, working, blockIdx.x + 1) - cta_first);
  const int run0 = (int)((int64_t)cta_count * warp / kWarps);
  const int count = (int)((int64_t)cta_count * (warp + 1) / kWarps) - run0;

  bool failed = false;
  if (count > 0) {
    Cursor cur = locate<KT, THREADS>(a, pre, cta_first + run0);

    // The tile to be copied next: its page of this lane's unit (lanes 0 .. TU - 1) is looked up one
    // tile before the copy is issued.
    const int UP = a.P / kUnit;
    const bool one_copy = UP % TU == 0;  // a tile's units lie in one page, next to each other
    const int step_page = TU / UP, step_sub = TU % UP, page0 = lane / UP, sub0 = lane % UP;
    Cursor ahead = cur;
    int a_len = length_of(a, ahead.b), a_head = ahead.seg % a.Hkv;
    int a_page = (ahead.k * TU + lane) / UP, a_sub = (ahead.k * TU + lane) % UP;
    const int32_t* a_row = a.table + (int64_t)ahead.b * a.ts;
    int pid = -1;
    auto look = [&]() {
      pid = -1;
      if (lane < TU && (ahead.k * TU + lane) * kUnit < a_len) pid = a_row[a_page];
    };
    auto step = [&]() {
      if (advance<KT>(a, ahead)) {
        a_head = ahead.seg % a.Hkv;
        a_len = length_of(a, ahead.b);
        a_row = a.table + (int64_t)ahead.b * a.ts;
        a_page = page0, a_sub = sub0;
      } else {
        a_page += step_page, a_sub += step_sub;
        if (a_sub >= UP) a_sub -= UP, ++a_page;
      }
      look();
    };
    uint32_t valid = 0;  // units that are there, TU bits per stage
    auto issue = [&](int s) {
      const bool ok = pid >= 0 && pid < a.pages;
      const uint32_t mask = __ballot_sync(0xffffffffu, ok);
      valid = (valid & ~(((1u << TU) - 1) << (TU * s))) | (mask << (TU * s));
      const uint32_t bytes = __popc(mask) * L::kBytes;
      if (lane == 0) mbar_arrive_expect_tx(&bar[s], bytes);
      __syncwarp();
      if (ok && (lane == 0 || !one_copy))
        bulk_load(ring + s * Tile<D>::kBytes + lane * L::kBytes,
                  a.pool + (((int64_t)pid * a.Hkv + a_head) * UP + a_sub) * (int64_t)L::kBytes,
                  one_copy ? bytes : L::kBytes, &bar[s]);
    };
    look();
    int looked = 0;  // tiles issued
    while (true) {
      issue(looked);
      ++looked;
      if (looked < count) step();
      if (looked >= min(kStages, count)) break;
    }

    // state of the current segment
    uint32_t qf[NT][NG][2 * KW][2];
    float sq[NT][NG], qr[NT], ar[NT], be[NT], mh[NT];
    int pos[NT];
    float o[NT][NG][MT][4], m[NT], l[NT], pm[NT][NG];
    int ve = 0;        // o holds p s 2^(14 - ve): the exponent of the largest V scale so far
    int lo_pos = 0;    // smallest position of a row that sees keys
    int nq = 0, base = 0, len = 0;
    const float kf = (float)key_of_row(g8);

    bool fresh = true, from_start = true;
    int s = 0, phase = 0;
    for (int i = 0; i < count; ++i) {
      if (fresh) {
        fresh = false;
        from_start = cur.k == 0;
        const int hk = cur.seg % a.Hkv, z = cur.seg / a.Hkv;
        len = length_of(a, cur.b);
        nq = queries_of(a, cur.b);
        base = len - nq;
        ve = -110;
        const int rows = a.G * a.T;
        lo_pos = max(0, base + z * RT / a.G);
#pragma unroll
        for (int n = 0; n < NT; ++n) {
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
          const float up = pow2(13 - ex);
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
                // the codes of these dims are 16 times as large
                qf[n][g][2 * w + p][1] = pack2<__half>(part[8 * w + 2 * p + 1] * 0.0625f, part[8 * w + 2 * p + 5] * 0.0625f);
              }
            sum += __shfl_xor_sync(0xffffffffu, sum, 1);
            sum += __shfl_xor_sync(0xffffffffu, sum, 2);
            sum += __shfl_xor_sync(0xffffffffu, sum, 4);
            sq[n][g] = __shfl_sync(0xffffffffu, sum, 8 * t4) * pow2(-24);
          }
          const int exr = __shfl_sync(0xffffffffu, ex, 8 * t4);
          // the query row whose scores this thread holds; logits in units of log 2
          const int r = min(z * RT + n * 4 + t4, rows - 1);
          const int h = hk * a.G + r % a.G;
          pos[n] = max(0, base + min(r / a.G, nq - 1));
          const float rc = a.ssmax[h] * logf((float)pos[n] + 1.f) * kLog2e;
          qr[n] = a.scale * rc * 2048.f * pow2(exr);
          ar[n] = -a.alpha[h] * rc;
          be[n] = a.beta[h];
          mh[n] = -a.mu[h];
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

      if (!__all_sync(0xffffffffu, mbar_wait_bounded(&bar[s], (uint32_t)phase, kWaitLimit))) {
        // never expected: the error is counted, copies in flight are waited for, the rows stay unwritten
        if (lane == 0) atomicAdd(&g_kv4_wait_timeouts, 1u);
        for (int j = i + 1; j < looked; ++j)
          mbar_wait_bounded(&bar[j % kStages], (uint32_t)((j / kStages) & 1), kWaitLimit);
        failed = true;
        break;
      }
      const uint8_t* tile = ring + s * Tile<D>::kBytes;
      const uint32_t units = (valid >> (TU * s)) & ((1u << TU) - 1);
      const int k0 = cur.k * KT;

      // W: every key of the tile is there and visible to every row
      auto attend = [&](auto whole) {
        constexpr bool W = decltype(whole)::value;
        const int r0 = key_of_row(g8);
        float2 x[NT][TU];
        float top[NT], dk[NT];
        uint32_t vp[TU][NG][2];
        float big = 0.f;
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          top[n] = -INFINITY;
          dk[n] = (float)(k0 - pos[n]) + kf;
        }
#pragma unroll
        for (int u = 0; u < TU; ++u) {
          const uint8_t* unit = tile + u * L::kBytes;
          float2 dot[NT];
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
            for (int w = 0; w < KW; ++w) {
              uint32_t c0[4], c1[4];
              codes(w0[w], c0);
              codes(w1[w], c1);
#pragma unroll
              for (int p = 0; p < 2; ++p) {
                const uint32_t af[4] = {c0[2 * p], c1[2 * p], c0[2 * p + 1], c1[2 * p + 1]};
#pragma unroll
                for (int n = 0; n < NT; ++n) {
                  const float start = -8.f * sq[n][g];
                  if (w == 0 && p == 0) mma_f16(acc[n], af, qf[n][g][0], start, 0.f, start, 0.f);
                  else mma_16816<__half>(acc[n], af, qf[n][g][2 * w + p]);
                }
              }
            }
            const uint32_t* kp = reinterpret_cast<const uint32_t*>(unit + L::kKp) + g * kUnit + r0;
            const uint32_t p0 = kp[0], p1 = kp[8];
            const uint32_t* vq = reinterpret_cast<const uint32_t*>(unit + L::kVp) + g * kUnit + r0;
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              vp[u][g][e] = vq[8 * e];
              // what lies in a slot that holds no token may be any pair
              if (!W && (!((units >> u) & 1u) || k0 + u * kUnit + r0 + 8 * e >= len)) vp[u][g][e] = 0u;
              big = fmaxf(big, kv4::pair_scale(vp[u][g][e]));
            }
            const float2 ks = make_float2(kv4::pair_scale(p0), kv4::pair_scale(p1));
            const float2 km = make_float2(kv4::pair_centre(p0), kv4::pair_centre(p1));
#pragma unroll
            for (int n = 0; n < NT; ++n) {
              const float2 s2 = make_float2(sq[n][g], sq[n][g]);
              const float2 both = fadd2(make_float2(acc[n][0], acc[n][2]), make_float2(acc[n][1], acc[n][3]));
              dot[n] = g ? ffma2(ks, both, ffma2(km, s2, dot[n])) : ffma2(ks, both, fmul2(km, s2));
            }
          }
#pragma unroll
          for (int n = 0; n < NT; ++n) {
            // key - pos is a whole number: exact; -mu, |.| + eps round as in the formula
            const float2 gap = fadd2(make_float2(dk[n], dk[n]), make_float2(u * 16.f, u * 16.f + 8.f));
            const float2 off = fadd2(gap, make_float2(mh[n], mh[n]));
            const float2 dist = make_float2(fabsf(off.x) + a.eps, fabsf(off.y) + a.eps);
            float2 pw;
            if constexpr (sizeof(T) == 4) {
              pw = make_float2(powf(dist.x, be[n]), powf(dist.y, be[n]));
            } else {
              const float2 ln = fmul2(make_float2(lg2_(dist.x), lg2_(dist.y)), make_float2(be[n], be[n]));
              pw = make_float2(ex2f_(ln.x), ex2f_(ln.y));
            }
            float2 y = ffma2(dot[n], make_float2(qr[n], qr[n]), fmul2(pw, make_float2(ar[n], ar[n])));
            if (!W) {
              const bool there = (units >> u) & 1u;
              if (!there || gap.x > 0.f) y.x = -INFINITY;
              if (!there || gap.y > 0.f) y.y = -INFINITY;
            }
            x[n][u] = y;
            top[n] = fmax3(top[n], y.x, y.y);
          }
        }

        // o is kept against the largest V scale so far: p s 2^(14 - ve) stays below fp16's end
        const uint32_t bits = __reduce_max_sync(0xffffffffu, __float_as_uint(big));
        const int vn = max(ve, (int)(bits >> 23) - 127);
        const float vdown = pow2(max(ve - vn, -126)), vup = pow2(14 - vn);
        ve = vn;
#pragma unroll
        for (int n = 0; n < NT; ++n) {
#pragma unroll
          for (int d = 4; d < 32; d <<= 1) top[n] = fmaxf(top[n], __shfl_xor_sync(0xffffffffu, top[n], d));
          const float mn = fmaxf(m[n], top[n]);
          const float shift = mn == -INFINITY ? 0.f : mn;
          const float f = exp2f(m[n] - shift);
          m[n] = mn;
          if (__any_sync(0xffffffffu, f * vdown != 1.f)) {
            l[n] *= f;
#pragma unroll
            for (int g = 0; g < NG; ++g) {
              pm[n][g] *= f;
#pragma unroll
              for (int t = 0; t < MT; ++t)
#pragma unroll
                for (int e = 0; e < 4; ++e) o[n][g][t][e] *= f * vdown;
            }
          }
#pragma unroll
          for (int u = 0; u < TU; ++u) {
            const float2 y = fadd2(x[n][u], make_float2(-shift, -shift));
            x[n][u] = sizeof(T) == 4 ? make_float2(exp2f(y.x), exp2f(y.y)) : make_float2(ex2f_(y.x), ex2f_(y.y));
            l[n] += x[n][u].x + x[n][u].y;
          }
        }

#pragma unroll
        for (int u = 0; u < TU; ++u) {
          const uint8_t* unit = tile + u * L::kBytes;
#pragma unroll
          for (int g = 0; g < NG; ++g) {
            const float2 vs = make_float2(kv4::pair_scale(vp[u][g][0]), kv4::pair_scale(vp[u][g][1]));
            const float2 vm = ffma2(vs, make_float2(-8.f, -8.f),
                                    make_float2(kv4::pair_centre(vp[u][g][0]), kv4::pair_centre(vp[u][g][1])));
            const float2 vn2 = fmul2(vs, make_float2(vup, vup));
            uint32_t bf[NT][2];
#pragma unroll
            for (int n = 0; n < NT; ++n) {
              float2 ps = fmul2(x[n][u], vn2);
              float2 pc = fmul2(x[n][u], vm);
              if (!W) {  // a weight of 0 leaves out even a NaN (a later token of the same request)
                if (x[n][u].x == 0.f) ps.x = pc.x = 0.f;
                if (x[n][u].y == 0.f) ps.y = pc.y = 0.f;
              }
              pm[n][g] += pc.x + pc.y;
              // 11 bits each: the high part is cut off, exactly a number of fp16
              const float2 hi = make_float2(__uint_as_float(__float_as_uint(ps.x) & 0xffffe000u),
                                            __uint_as_float(__float_as_uint(ps.y) & 0xffffe000u));
              bf[n][0] = transpose8x8(pack2<__half>(hi.x, ps.x - hi.x));
              bf[n][1] = transpose8x8(pack2<__half>(hi.y, ps.y - hi.y));
            }
            const uint8_t* at = unit + L::kV + t4 * L::kRow + g * (DG / 2) + (KW == 2 ? 4 * g8 : 4 * (g8 >> 1));
            uint32_t w[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) w[j] = *reinterpret_cast<const uint32_t*>(at + 4 * j * L::kRow);
#pragma unroll
            for (int hf = 0; hf < KW; ++hf) {  // halves of a word: four dims each
              const uint32_t sel = KW == 2 ? (hf ? 0x7632u : 0x5410u) : ((g8 & 1) ? 0x7632u : 0x5410u);
              uint32_t c0[4], c1[4];
              codes(__byte_perm(w[0], w[1], sel), c0);
              codes(__byte_perm(w[2], w[3], sel), c1);
#pragma unroll
              for (int p = 0; p < 2; ++p) {
                const uint32_t af[4] = {c0[2 * p], c0[2 * p + 1], c1[2 * p], c1[2 * p + 1]};
#pragma unroll
                for (int n = 0; n < NT; ++n) mma_16816<__half>(o[n][g][2 * hf + p], af, bf[n]);
              }
            }
          }
        }
      };
      if (units == (1u << TU) - 1 && k0 + KT - 1 <= lo_pos) attend(std::true_type());
      else attend(std::false_type());

      __syncwarp();  // every lane is done with the stage
      if (looked < count) {
        fence_proxy_async_smem();
        issue(s);
        if (++looked < count) step();
      }
      if (++s == kStages) s = 0, phase ^= 1;

      const bool ends = cur.k + 1 == cur.nt;
      if (ends || i + 1 == count) {
        const int hk = cur.seg % a.Hkv, z = cur.seg / a.Hkv;
        const bool direct = ends && from_start;
        // the run's last piece goes where the ring was
        const int which = i + 1 == count ? 1 : 0;
        float* part = piece_at(warp, which);
        if (!direct && lane == 0) {
          pieces[warp][which].segment = (int64_t)cur.b * zh + cur.seg;
          pieces[warp][which].begins = from_start;
          pieces[warp][which].ends = ends;
        }
        const float back = pow2(min(ve, 127));  // and 2^10
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
#pragma unroll
          for (int g = 0; g < NG; ++g) {
            float y[2 * MT];
#pragma unroll
            for (int j = 0; j < MT; ++j) {
              y[2 * j] = fmaf((o[n][g][j][0] + o[n][g][j][1]) * 1024.f, back, pm[n][g]) * inv;
              y[2 * j + 1] = fmaf((o[n][g][j][2] + o[n][g][j][3]) * 64.f, back, pm[n][g]) * inv;
            }
            const int d0 = g * DG + g8 * 2 * MT;
            if (direct) {
              if (r < a.G * a.T) {
                T* dst = out + cur.b * a.st.s[3] + (hk * a.G + r % a.G) * a.st.s[4] + t * a.st.s[5] + d0;
#pragma unroll
                for (int j = 0; j < 2 * MT; ++j) dst[j] = from_f<T>(sees ? y[j] : 0.f);
              }
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
        fresh = true;
      }
      advance<KT>(a, cur);
    }
  }

  // The CTA's pieces in tile order: neighbours of one segment are joined, and written out where the
  // CTA holds all of the segment, else left to the merge (slot 0 where the segment began before this
  // CTA's run, 1 where it began in it).
  if (__syncthreads_or(failed)) return;
  for (int first = 0; first < 2 * kWarps;) {
    const Piece head = pieces[first >> 1][first & 1];
    if (head.segment < 0) {
      ++first;
      continue;
    }
    uint32_t members = 1u << first;
    int ends = head.ends, next = first + 1;
    for (; next < 2 * kWarps; ++next) {
      const Piece& p = pieces[next >> 1][next & 1];
      if (p.segment < 0) continue;
      if (p.segment != head.segment) break;
      members |= 1u << next;
      ends = p.ends;
    }
    const bool direct = head.begins && ends;
    const int b = (int)(head.segment / zh), seg = (int)(head.segment % zh);
    const int hk = seg % a.Hkv, z = seg / a.Hkv;
    const int nq = queries_of(a, b), base = length_of(a, b) - nq;
    float* part = a.ws + ((int64_t)blockIdx.x * 2 + (head.begins ? 1 : 0)) * piece_floats<D, NT>();
    for (int v = threadIdx.x; v < RT * (D / 4); v += THREADS) {
      const int rr = v / (D / 4), d = v % (D / 4) * 4;
      float mx = -INFINITY;
      for (uint32_t w = members; w; w &= w - 1) {
        const int i = __ffs(w) - 1;
        mx = fmaxf(mx, piece_at(i >> 1, i & 1)[rr * (D + 4) + D]);
      }
      const float shift = mx == -INFINITY ? 0.f : mx;
      float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
      float den = 0.f;
      for (uint32_t w = members; w; w &= w - 1) {
        const int i = __ffs(w) - 1;
        const float* src = piece_at(i >> 1, i & 1) + rr * (D + 4);
        const float f = exp2f(src[D] - shift);
        const float4 y = *reinterpret_cast<const float4*>(src + d);
        acc.x = fmaf(f, y.x, acc.x), acc.y = fmaf(f, y.y, acc.y);
        acc.z = fmaf(f, y.z, acc.z), acc.w = fmaf(f, y.w, acc.w);
        den = fmaf(f, src[D + 1], den);
      }
      if (direct) {
        const int r = z * RT + rr, t = r / a.G;
        if (r < a.G * a.T) {
          const float inv = t < nq && base + t >= 0 && den != 0.f ? 1.f / den : 0.f;
          T* dst = out + b * a.st.s[3] + (hk * a.G + r % a.G) * a.st.s[4] + t * a.st.s[5] + d;
          const bool sees = t < nq && base + t >= 0;
          dst[0] = from_f<T>(sees ? acc.x * inv : 0.f), dst[1] = from_f<T>(sees ? acc.y * inv : 0.f);
          dst[2] = from_f<T>(sees ? acc.z * inv : 0.f), dst[3] = from_f<T>(sees ? acc.w * inv : 0.f);
        }
      } else {
        *reinterpret_cast<float4*>(part + rr * (D + 4) + d) = acc;
        if (d == 0) {
          part[rr * (D + 4) + D] = mx;
          part[rr * (D + 4) + D + 1] = den;
        }
      }
    }
    first = next;
  }
}

// ------------------------------------------------------------------ merge
// One CTA per segment: joins the CTAs' partials of a segment that spans several, in a fixed order
// (each group of D RT / 4 threads takes every n-th partial, the groups are summed in order), and
// zeroes the rows of a segment without tiles.
constexpr int kMergeThreads = 512;

template <typename T, int D, int NT>
__global__ void __launch_bounds__(kMergeThreads) kv4_merge_kernel(T* __restrict__ out, const Args a) {
  constexpr int KT = Tile<D>::kKeys, RT = 4 * NT, NV = RT * D / 4, PL = kMergeThreads / NV;
  static_assert(NV <= kMergeThreads && kMergeThreads % NV == 0, "whole groups of threads");
  __shared__ int64_t pre[kMergeThreads + 1];
  __shared__ float s_shift[RT], s_den[RT];
  __shared__ float4 s_acc[PL][NV];
  scan_requests<KT, kMergeThreads>(a, pre);
  const int zh = a.Z * a.Hkv, run = (a.B + kMergeThreads - 1) / kMergeThreads;
  const int b = blockIdx.x / zh, seg = blockIdx.x % zh;
  const int hk = seg % a.Hkv, z = seg / a.Hkv;
  int64_t before = pre[b / run];
  for (int i = b / run * run; i < b; ++i) before += tiles_of<KT>(a, i);
  const int64_t total = pre[kMergeThreads] * zh;
  const int nt = tiles_of<KT>(a, b);
  const int64_t x0 = before * zh + (int64_t)seg * nt;
  int64_t c0 = 0;
  int n = 0;  // partials
  if (nt > 0) {
    const int64_t working = working_ctas(total, a.ctas);
    c0 = cta_of(total, working, x0);
    n = (int)(cta_of(total, working, x0 + nt - 1) - c0) + 1;
  }
  // every CTA waits, also those without work: what follows this grid must find the workers' done
  asm volatile("griddepcontrol.wait;" ::: "memory");
  if (n == 1) return;  // written by its CTA
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  // the first CTA's slot 1 (the segment began in its run), every other one's slot 0
  auto slot = [&](int i) { return a.ws + ((c0 + i) * 2 + (i == 0 ? 1 : 0)) * piece_floats<D, NT>(); };
  if (n > 0) {
    for (int rr = warp; rr < RT; rr += kMergeThreads / 32) {
      float mx = -INFINITY, den = 0.f;
      for (int i = lane; i < n; i += 32) mx = fmaxf(mx, slot(i)[rr * (D + 4) + D]);
      mx = warp_max(mx);
      if (mx == -INFINITY) mx = 0.f;
      for (int i = lane; i < n; i += 32)
        den = fmaf(exp2f(slot(i)[rr * (D + 4) + D] - mx), slot(i)[rr * (D + 4) + D + 1], den);
      den = warp_sum(den);
      if (lane == 0) s_shift[rr] = mx, s_den[rr] = den;
    }
  }
  __syncthreads();
  const int v = tid % NV, pl = tid / NV, rr = v / (D / 4), d = v % (D / 4) * 4;
  float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
  if (n > 0) {
    const float shift = s_shift[rr];
#pragma unroll 4
    for (int i = pl; i < n; i += PL) {
      const float* src = slot(i) + rr * (D + 4);
      const float f = exp2f(src[D] - shift);
      const float4 y = *reinterpret_cast<const float4*>(src + d);
      acc.x = fmaf(f, y.x, acc.x), acc.y = fmaf(f, y.y, acc.y);
      acc.z = fmaf(f, y.z, acc.z), acc.w = fmaf(f, y.w, acc.w);
    }
  }
  s_acc[pl][v] = acc;
  __syncthreads();
  if (pl) return;
  for (int i = 1; i < PL; ++i) {
    const float4 y = s_acc[i][v];
    acc.x += y.x, acc.y += y.y, acc.z += y.z, acc.w += y.w;
  }
  const int nq = queries_of(a, b), base = length_of(a, b) - nq;
  const int r = z * RT + rr, t = r / a.G;
  if (r >= a.G * a.T) return;
  const bool sees = n > 0 && t < nq && base + t >= 0 && s_den[rr] != 0.f;
  const float inv = sees ? 1.f / s_den[rr] : 0.f;
  T* dst = out + b * a.st.s[3] + (hk * a.G + r % a.G) * a.st.s[4] + t * a.st.s[5] + d;
  dst[0] = from_f<T>(sees ? acc.x * inv : 0.f), dst[1] = from_f<T>(sees ? acc.y * inv : 0.f);
  dst[2] = from_f<T>(sees ? acc.z * inv : 0.f), dst[3] = from_f<T>(sees ? acc.w * inv : 0.f);
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

template <typename T, int D, int NT>
int launch(const void* q, void* out, Args a, cudaStream_t stream) {
  constexpr int smem = attention_smem<D, NT>();
  const void* fn = reinterpret_cast<const void*>(&kv4_attention_kernel<T, D, NT>);
  if (int rc = ensure_smem_attr(fn, smem)) return rc;
  kv4_attention_kernel<T, D, NT><<<a.ctas, 32 * kWarps, smem, stream>>>((const T*)q, (T*)out, a);
  if (int rc = check_launch("kv4_chord_attention")) return rc;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)((int64_t)a.B * a.Z * a.Hkv));
  cfg.blockDim = dim3(kMergeThreads);
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
  const int nt = row_tile(H / Hkv * T, D);
  return (int64_t)sm_count() * ctas_per_sm(nt, (int)D) * 2 * 4 * nt * (D + 4) * 4;
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
    a.ctas = sm_count() * ctas_per_sm(nt, (int)D);
    MB_REQUIRE((int64_t)a.B * a.Z * a.Hkv < (1ll << 31), MB_ERR_SHAPE, "kv4_chord_attention: too many rows");
    if (nt == 1) return launch<E, DD, 1>(q, out, a, (cudaStream_t)stream);
    if constexpr (DD < 128)
      if (nt == 4) return launch<E, DD, 4>(q, out, a, (cudaStream_t)stream);
    return launch<E, DD, 2>(q, out, a, (cudaStream_t)stream);
  });
}
