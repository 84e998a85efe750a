// RMSNorm, GatedRMSNorm and SwiGLU for training: their forward with one rounding, and their
// gradients.
//
// Per row of N values x, with r = (mean(x^2) + eps)^(-1/2), weight w, gate g and act = g sig(g):
//   y  = x r w [act]                                 (motif/ops/rms_norm.py:419-553)
//   u  = dy [act] w
//   dx = r (u - x r^2 mean(u x))
//   dw = sum over the rows of dy [act] x r
//   dg = dy (x r w) sig(g) (1 + g (1 - sig(g)))
// and SwiGLU, y = v act: dv = dy act, dg = dy v sig(g) (1 + g (1 - sig(g))).
// All of it in fp32, each output rounded once.  (The kernels that run where nothing needs a
// gradient, norms.cu, keep the eager reference's rounding of every intermediate result.)
//
// Memory bounds these: every tensor is read or written once.  A row is held by a group of G threads
// (a part of a warp, a warp, or the CTA) as NV 16-byte vectors a thread, so r is recomputed in the
// backward pass from values that are there anyway instead of stored (4 bytes a row each way: 3 % of
// the traffic of rows of 64).  The weight's gradient is a sum over all rows: each thread keeps its
// columns' sums in registers over the rows that its group walks, the CTA adds its groups in order
// and leaves one row of partial sums, and a second kernel adds those in order (both in 64 bits): no
// atomics, the same bits every time.
#include <algorithm>
#include <type_traits>

#include "common.cuh"

namespace mb {
namespace {

constexpr int kThreads = 256;
constexpr int kCtasPerSm = 2;      // resident CTAs: each walks its share of the rows

// A 16-byte vector of a row, as it is in memory and as numbers.
template <typename T> struct Row16 {
  static constexpr int E = 16 / (int)sizeof(T);
  __device__ static uint4 load(const T* p) { return *reinterpret_cast<const uint4*>(p); }
  __device__ static void numbers(const uint4& u, float (&v)[E]) {
    const T* e = reinterpret_cast<const T*>(&u);
#pragma unroll
    for (int i = 0; i < E; ++i) v[i] = to_f(e[i]);
  }
  __device__ static void pairs(const uint4& u, float2 (&v)[E / 2]) {
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
    if constexpr (sizeof(T) == 4) {
      v[0] = make_float2(__uint_as_float(w[0]), __uint_as_float(w[1]));
      v[1] = make_float2(__uint_as_float(w[2]), __uint_as_float(w[3]));
    } else if constexpr (std::is_same<T, __half>::value) {
#pragma unroll
      for (int i = 0; i < 4; ++i) v[i] = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) v[i] = make_float2(__uint_as_float(w[i] << 16), __uint_as_float(w[i] & 0xffff0000u));
    }
  }
  __device__ static void store_pairs(T* p, const float2 (&v)[E / 2]) {
    uint4 u;
    if constexpr (sizeof(T) == 4)
      u = make_uint4(__float_as_uint(v[0].x), __float_as_uint(v[0].y), __float_as_uint(v[1].x), __float_as_uint(v[1].y));
    else
      u = make_uint4(pack2<T>(v[0].x, v[0].y), pack2<T>(v[1].x, v[1].y), pack2<T>(v[2].x, v[2].y), pack2<T>(v[3].x, v[3].y));
    *reinterpret_cast<uint4*>(p) = u;
  }
  __device__ static void store(T* p, const float (&v)[E]) {
    __align__(16) T e[E];
#pragma unroll
    for (int i = 0; i < E; ++i) e[i] = from_f<T>(v[i]);
    *reinterpret_cast<uint4*>(p) = *reinterpret_cast<const uint4*>(e);
  }
};

__device__ __forceinline__ float load_as(const void* p, int dtype, int64_t i) {
  return dtype == MB_F32    ? reinterpret_cast<const float*>(p)[i]
         : dtype == MB_BF16 ? to_f(reinterpret_cast<const __nv_bfloat16*>(p)[i])
                            : to_f(reinterpret_cast<const __half*>(p)[i]);
}
__device__ __forceinline__ void store_as(void* p, int dtype, int64_t i, float v) {
  if (dtype == MB_F32)
    reinterpret_cast<float*>(p)[i] = v;
  else if (dtype == MB_BF16)
    reinterpret_cast<__nv_bfloat16*>(p)[i] = from_f<__nv_bfloat16>(v);
  else
    reinterpret_cast<__half*>(p)[i] = from_f<__half>(v);
}

// sig(g) with the MUFU exponential and reciprocal: a few units of 2^-23, and |g| of 2^-24 from the rounded exponent
__device__ __forceinline__ float sig_(float g) { return rcpf_(1.0f + ex2f_(g * kNegLog2e)); }

struct NormArgs {
  const void* x;      // rows of N (plain) or N values then N gates (gated)
  const void* w;      // [N] of w_dtype, or null
  const void* dy;     // backward: rows of N
  void* out;          // forward: y; backward: dx (laid out as x)
  float* part;        // backward: [parts][N] partial sums of dw, or null
  int64_t M, xs, ds, os;  // rows; row strides of x, dy and out
  int N, w_dtype;
  float eps;
};

// Sums over the G threads of a row (BOTH: of two values, else of the first).  G > 32: over the CTA,
// through `red` (two slots in turn, so one barrier a row is enough).
template <int G, bool BOTH>
__device__ __forceinline__ float2 row_sum(float2 v, float2 (*red)[kThreads / 32], int& slot) {
#pragma unroll
  for (int o = (G < 32 ? G : 32) / 2; o > 0; o >>= 1) {
    v.x += __shfl_xor_sync(0xffffffffu, v.x, o);
    if constexpr (BOTH) v.y += __shfl_xor_sync(0xffffffffu, v.y, o);
  }
  if constexpr (G > 32) {
    float2* r = red[slot];
    slot ^= 1;
    if ((threadIdx.x & 31) == 0) r[threadIdx.x >> 5] = v;
    __syncthreads();
    v = r[0];
#pragma unroll
    for (int i = 1; i < kThreads / 32; ++i) {
      v.x += r[i].x;
      v.y += r[i].y;
    }
  }
  return v;
}

// Rows whose length is a multiple of the vector and whose addresses are 16-byte aligned.  Every thread
// copies the vectors that it will use itself into its own places of a ring in shared memory
// (cp.async), rows ahead: no barrier, and no registers held by what is under way.
//
// Two CTAs an SM with six 4 KB pieces each (16 bytes of every thread) under way, 48 KB an SM, are enough for
// the memory's latency; more cost time (393216 gated rows of 128, forward: 49.4 us with 24 KB a CTA, 53.4
// with 40, 55.6 with 56; backward 96.6 us with 12, 90.3 with 24, 99.0 with 36).
//
// The backward pass over four vectors a thread (gated: three) needs more than the 128 registers that two
// CTAs leave it: one CTA then, with twice as much under way (98304 rows of 1024: 233 us with spills, 106
// without; 65536 gated rows of 768: 131 and 88).
template <int NV, bool GATED, bool BWD>
__host__ __device__ constexpr int resident() {
  return BWD && NV > (GATED ? 2 : 3) ? 1 : kCtasPerSm;
}
template <int NV, bool GATED, bool BWD>
__host__ __device__ constexpr int stages() {
  constexpr int each = (1 + GATED + BWD) * NV, ahead = 6 * kCtasPerSm / resident<NV, GATED, BWD>();
  return 1 + ((ahead + each / 2) / each > 1 ? (ahead + each / 2) / each : 1);
}
template <typename T, int G, int NV, bool GATED, bool BWD>
__global__ void __launch_bounds__(kThreads, resident<NV, GATED, BWD>()) norm_rows_kernel(const NormArgs a) {
  constexpr int E = Row16<T>::E, H = E / 2;
  constexpr int kGroups = kThreads / G;
  constexpr int kTensors = 1 + GATED + BWD, S = stages<NV, GATED, BWD>();
  // the weight, and sig(g) from the first pass over a row to the second, stay in registers while there
  // is room (two CTAs an SM: 128); else the weight lies in shared memory and sig(g) is computed twice
  constexpr bool kKeep = NV < 3;
  __shared__ float2 red[2][kThreads / 32];
  __shared__ float4 w_all[kKeep ? 1 : E / 4][kKeep ? 1 : NV * G];
  extern __shared__ uint4 ring[];  // [S][tensor][NV][threads]; in the end BWD's partial sums
  const int lane = threadIdx.x % G, group = threadIdx.x / G;
  const int N = a.N;
  int slot = 0;
  float2 w[kKeep ? NV : 1][H], dw[BWD ? NV : 1][H];
  auto weight_at = [&](int c) { return c < N ? (a.w ? load_as(a.w, a.w_dtype, c) : 1.0f) : 0.0f; };
#pragma unroll
  for (int v = 0; v < NV; ++v)
#pragma unroll
    for (int h = 0; h < H; ++h) {
      const int c = (v * G + lane) * E + 2 * h;
      if constexpr (kKeep) w[v][h] = make_float2(weight_at(c), weight_at(c + 1));
      if constexpr (BWD) dw[v][h] = make_float2(0.f, 0.f);
    }
  if constexpr (!kKeep) {
    for (int i = threadIdx.x; i < NV * G * E; i += kThreads)
      reinterpret_cast<float*>(&w_all[i % E / 4][i / E])[i % 4] = weight_at(i);
    __syncthreads();
  }
  auto weights = [&](int v, float2 (&o)[H]) {
#pragma unroll
    for (int h = 0; h < H; ++h) {
      if constexpr (kKeep) {
        o[h] = w[v][h];
      } else if (h % 2 == 0) {
        const float4 q = w_all[h / 2][v * G + lane];
        o[h] = make_float2(q.x, q.y);
        o[h + 1] = make_float2(q.z, q.w);
      }
    }
  };
  const float inv_n = 1.0f / (float)N;
  const int64_t step = (int64_t)gridDim.x * kGroups;
  int64_t row = (int64_t)blockIdx.x * kGroups + group, ahead = row;  // computed; requested
  const int64_t x_step = step * a.xs, d_step = step * a.ds, o_step = step * a.os;
  const T* xp = reinterpret_cast<const T*>(a.x) + row * a.xs + lane * E;
  const T* dp = reinterpret_cast<const T*>(a.dy) + row * a.ds + lane * E;
  T* op = reinterpret_cast<T*>(a.out) + row * a.os + lane * E;
  uint4* const places = ring + threadIdx.x;
  auto request = [&](int stage) {
    uint4* at = places + stage * (kTensors * NV * kThreads);
    const bool there = ahead < a.M;  // zeros elsewhere; a row that is not there is not addressed
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      const bool in = there && (v * G + lane) * E < N;
      cp_async16(at + v * kThreads, in ? xp + v * G * E : reinterpret_cast<const T*>(a.x), in);
      if constexpr (GATED) cp_async16(at + (NV + v) * kThreads, in ? xp + N + v * G * E : reinterpret_cast<const T*>(a.x), in);
      if constexpr (BWD)
        cp_async16(at + ((kTensors - 1) * NV + v) * kThreads, in ? dp + v * G * E : reinterpret_cast<const T*>(a.dy), in);
    }
    cp_async_commit();
    ahead += step;
    xp += x_step;
    if constexpr (BWD) dp += d_step;
  };
#pragma unroll
  for (int i = 0; i < S - 1; ++i) request(i);
  int stage = 0;
  // every thread of the CTA makes the same number of rounds: the row sums are taken together
  for (; row - group < a.M; row += step, op += o_step) {
    cp_async_wait<S - 2>();
    request(stage == 0 ? S - 1 : stage - 1);  // into the place of the row before, whose values have been used
    const uint4* at = places + stage * (kTensors * NV * kThreads);
    stage = stage + 1 == S ? 0 : stage + 1;
    float2 sig[GATED && kKeep ? NV : 1][H];
    float2 sx = make_float2(0.f, 0.f), sy = sx;
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      float2 x[H], g[H], d[H], wv[H];
      if constexpr (BWD) weights(v, wv);
      Row16<T>::pairs(at[v * kThreads], x);
      if constexpr (GATED) Row16<T>::pairs(at[(NV + v) * kThreads], g);
      if constexpr (BWD) Row16<T>::pairs(at[((kTensors - 1) * NV + v) * kThreads], d);
#pragma unroll
      for (int h = 0; h < H; ++h) {
        sx = ffma2(x[h], x[h], sx);
        float2 t = make_float2(0.f, 0.f);
        if constexpr (BWD) t = fmul2(d[h], wv[h]);
        if constexpr (GATED && (BWD || kKeep)) {
          const float2 sg = make_float2(sig_(g[h].x), sig_(g[h].y));
          if constexpr (kKeep) sig[v][h] = sg;
          if constexpr (BWD) t = fmul2(t, fmul2(g[h], sg));
        }
        if constexpr (BWD) sy = ffma2(t, x[h], sy);
      }
    }
    const float2 s = row_sum<G, BWD>(make_float2(sx.x + sx.y, sy.x + sy.y), red, slot);
    const bool live = row < a.M;
    const float r = live ? rsqrtf(s.x * inv_n + a.eps) : 0.f;
    const float k = -s.y * inv_n * r * r;
    const float2 r2 = make_float2(r, r), k2 = make_float2(k, k), one = make_float2(1.f, 1.f);
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      float2 x[H], g[H], d[H], o[H], og[H], wv[H];
      weights(v, wv);
      Row16<T>::pairs(at[v * kThreads], x);
      if constexpr (GATED) Row16<T>::pairs(at[(NV + v) * kThreads], g);
      if constexpr (BWD) Row16<T>::pairs(at[((kTensors - 1) * NV + v) * kThreads], d);
#pragma unroll
      for (int h = 0; h < H; ++h) {
        const float2 xh = fmul2(x[h], r2);
        float2 sg = one;
        if constexpr (GATED && kKeep) sg = sig[v][h];
        if constexpr (GATED && !kKeep) sg = make_float2(sig_(g[h].x), sig_(g[h].y));
        if constexpr (BWD) {
          float2 dn = d[h];
          if constexpr (GATED) {
            const float2 act = fmul2(g[h], sg);
            dn = fmul2(d[h], act);
            // sig (1 + g (1 - sig)) = sig + act (1 - sig)
            const float2 slope = ffma2(act, ffma2(sg, make_float2(-1.f, -1.f), one), sg);
            og[h] = fmul2(fmul2(d[h], fmul2(xh, wv[h])), slope);
          }
          dw[v][h] = ffma2(dn, xh, dw[v][h]);
          o[h] = fmul2(r2, ffma2(x[h], k2, fmul2(dn, wv[h])));
        } else {
          o[h] = fmul2(xh, wv[h]);
          if constexpr (GATED) o[h] = fmul2(o[h], fmul2(g[h], sg));
        }
      }
      if (live && (v * G + lane) * E < N) {
        Row16<T>::store_pairs(op + v * G * E, o);
        if constexpr (BWD && GATED) Row16<T>::store_pairs(op + N + v * G * E, og);
      }
    }
  }
  if constexpr (BWD) {
    allow_dependent_launch();  // the weight's kernel may take its place (it waits for this one's end)
    if (a.part == nullptr) return;
    float* pr = a.part + (int64_t)blockIdx.x * N;
    if constexpr (G == kThreads) {
#pragma unroll
      for (int v = 0; v < NV; ++v)
#pragma unroll
        for (int e = 0; e < E; ++e)
          if ((v * G + lane) * E < N) pr[(v * G + lane) * E + e] = e % 2 ? dw[v][e / 2].y : dw[v][e / 2].x;
    } else {
      constexpr int W = G * NV * E;
      float* acc = reinterpret_cast<float*>(ring);  // [kGroups][W]
      cp_async_wait<0>();  // (of rows that are not there)
      __syncthreads();
#pragma unroll
      for (int v = 0; v < NV; ++v)
#pragma unroll
        for (int e = 0; e < E; ++e) acc[group * W + (v * G + lane) * E + e] = e % 2 ? dw[v][e / 2].y : dw[v][e / 2].x;
      __syncthreads();
      for (int c = threadIdx.x; c < N; c += kThreads) {
        double t = 0.0;
#pragma unroll 4
        for (int i = 0; i < kGroups; ++i) t += acc[i * W + c];
        pr[c] = (float)t;
      }
    }
  }
}

// Other lengths and alignments: V elements at a time (two where the addresses allow it), L elements a thread
// at most; the row is read twice, the second time from the L1.  dw's sums stay in registers (in memory, as
// a row of `part` that is read and written for every row of x, 200000 rows of 250 took 207 us backward; 75).
template <typename T, int V>
__device__ __forceinline__ void load_some(const T* p, float (&v)[V]) {
  if constexpr (V == 1) {
    v[0] = to_f(*p);
  } else if constexpr (sizeof(T) == 4) {
    const float2 u = *reinterpret_cast<const float2*>(p);
    v[0] = u.x;
    v[1] = u.y;
  } else {
    const uint32_t u = *reinterpret_cast<const uint32_t*>(p);
    const T* e = reinterpret_cast<const T*>(&u);
    v[0] = to_f(e[0]);
    v[1] = to_f(e[1]);
  }
}
template <typename T, int V>
__device__ __forceinline__ void store_some(T* p, const float (&v)[V]) {
  if constexpr (V == 1)
    *p = from_f<T>(v[0]);
  else if constexpr (sizeof(T) == 4)
    *reinterpret_cast<float2*>(p) = make_float2(v[0], v[1]);
  else
    *reinterpret_cast<uint32_t*>(p) = pack2<T>(v[0], v[1]);
}
template <typename T, int G, int L, int V, bool GATED, bool BWD>
__global__ void __launch_bounds__(kThreads) norm_some_kernel(const NormArgs a) {
  constexpr int kGroups = kThreads / G, K = L / V;
  __shared__ float2 red[2][kThreads / 32];
  extern __shared__ float sums[];  // BWD, several groups: [group][N] at the end
  const int lane = threadIdx.x % G, group = threadIdx.x / G;
  const int N = a.N;
  int slot = 0;
  const float inv_n = 1.0f / (float)N;
  float w[K][V], dw[BWD ? K : 1][V];
#pragma unroll
  for (int i = 0; i < K; ++i)
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const int c = (i * G + lane) * V + j;
      w[i][j] = c < N && a.w ? load_as(a.w, a.w_dtype, c) : 1.0f;
      if constexpr (BWD) dw[i][j] = 0.f;
    }
  const int64_t step = (int64_t)gridDim.x * kGroups;
  for (int64_t row0 = (int64_t)blockIdx.x * kGroups; row0 < a.M; row0 += step) {
    const int64_t row = row0 + group;
    const bool live = row < a.M;
    const T* xr = reinterpret_cast<const T*>(a.x) + row * a.xs + lane * V;
    const T* dr = reinterpret_cast<const T*>(a.dy) + row * a.ds + lane * V;
    float2 s = make_float2(0.f, 0.f);
#pragma unroll
    for (int i = 0; i < K; ++i)
      if (live && (i * G + lane) * V < N) {
        float x[V], g[V], d[V];
        load_some<T, V>(xr + i * G * V, x);
        if constexpr (GATED && BWD) load_some<T, V>(xr + N + i * G * V, g);
        if constexpr (BWD) load_some<T, V>(dr + i * G * V, d);
#pragma unroll
        for (int j = 0; j < V; ++j) {
          s.x = fmaf(x[j], x[j], s.x);
          if constexpr (BWD) {
            float t = d[j] * w[i][j];
            if constexpr (GATED) t *= g[j] * sig_(g[j]);
            s.y = fmaf(t, x[j], s.y);
          }
        }
      }
    s = row_sum<G, BWD>(s, red, slot);
    if (!live) continue;
    const float r = rsqrtf(s.x * inv_n + a.eps);
    const float k = s.y * inv_n * r * r;
    T* outr = reinterpret_cast<T*>(a.out) + row * a.os + lane * V;
#pragma unroll
    for (int i = 0; i < K; ++i)
      if ((i * G + lane) * V < N) {
        float x[V], g[V], d[V], o[V], og[V];
        load_some<T, V>(xr + i * G * V, x);
        if constexpr (GATED) load_some<T, V>(xr + N + i * G * V, g);
        if constexpr (BWD) load_some<T, V>(dr + i * G * V, d);
#pragma unroll
        for (int j = 0; j < V; ++j) {
          const float xh = x[j] * r;
          float act = 1.0f, sg = 0.f;
          if constexpr (GATED) {
            sg = sig_(g[j]);
            act = g[j] * sg;
          }
          if constexpr (BWD) {
            const float dn = GATED ? d[j] * act : d[j];
            dw[i][j] = fmaf(dn, xh, dw[i][j]);
            o[j] = r * (dn * w[i][j] - x[j] * k);
            if constexpr (GATED) og[j] = d[j] * (xh * w[i][j]) * (sg + act * (1.0f - sg));
          } else {
            o[j] = GATED ? xh * w[i][j] * act : xh * w[i][j];
          }
        }
        store_some<T, V>(outr + i * G * V, o);
        if constexpr (BWD && GATED) store_some<T, V>(outr + N + i * G * V, og);
      }
  }
  if constexpr (BWD) {
    allow_dependent_launch();
    if (a.part == nullptr) return;
    float* pr = a.part + (int64_t)blockIdx.x * N;
    float* to = kGroups == 1 ? pr : sums + group * N;
#pragma unroll
    for (int i = 0; i < K; ++i)
#pragma unroll
      for (int j = 0; j < V; ++j)
        if ((i * G + lane) * V + j < N) to[(i * G + lane) * V + j] = dw[i][j];
    if constexpr (kGroups > 1) {
      __syncthreads();
      for (int c = threadIdx.x; c < N; c += kThreads) {
        double t = 0.0;
#pragma unroll
        for (int i = 0; i < kGroups; ++i) t += sums[i * N + c];
        pr[c] = (float)t;
      }
    }
  }
}

// Longer rows than the kernels above hold: a CTA a row, element by element, dw's sums in its row of `part`.
template <typename T, bool GATED, bool BWD>
__global__ void __launch_bounds__(kThreads) norm_long_kernel(const NormArgs a) {
  __shared__ float2 red[2][kThreads / 32];
  const int N = a.N;
  int slot = 0;
  const float inv_n = 1.0f / (float)N;
  float* pr = BWD && a.part ? a.part + (int64_t)blockIdx.x * N : nullptr;
  if (pr)
    for (int c = threadIdx.x; c < N; c += kThreads) pr[c] = 0.f;
  for (int64_t row = blockIdx.x; row < a.M; row += gridDim.x) {
    const T* xr = reinterpret_cast<const T*>(a.x) + row * a.xs;
    const T* dr = reinterpret_cast<const T*>(a.dy) + row * a.ds;
    float2 s = make_float2(0.f, 0.f);
    for (int c = threadIdx.x; c < N; c += kThreads) {
      const float x = to_f(xr[c]);
      s.x = fmaf(x, x, s.x);
      if constexpr (BWD) {
        float t = to_f(dr[c]);
        if (a.w) t *= load_as(a.w, a.w_dtype, c);
        if constexpr (GATED) {
          const float g = to_f(xr[N + c]);
          t *= g * sig_(g);
        }
        s.y = fmaf(t, x, s.y);
      }
    }
    s = row_sum<kThreads, BWD>(s, red, slot);
    const float r = rsqrtf(s.x * inv_n + a.eps);
    const float k = s.y * inv_n * r * r;
    T* outr = reinterpret_cast<T*>(a.out) + row * a.os;
    for (int c = threadIdx.x; c < N; c += kThreads) {
      const float x = to_f(xr[c]), xh = x * r;
      const float w = a.w ? load_as(a.w, a.w_dtype, c) : 1.0f;
      float act = 1.0f, sg = 0.f, g = 0.f;
      if constexpr (GATED) {
        g = to_f(xr[N + c]);
        sg = sig_(g);
        act = g * sg;
      }
      if constexpr (BWD) {
        const float d = to_f(dr[c]), dn = GATED ? d * act : d;
        if (pr) pr[c] = fmaf(dn, xh, pr[c]);
        outr[c] = from_f<T>(r * (dn * w - x * k));
        if constexpr (GATED) outr[N + c] = from_f<T>(d * (xh * w) * (sg + act * (1.0f - sg)));
      } else {
        outr[c] = from_f<T>(GATED ? xh * w * act : xh * w);
      }
    }
  }
}

// dw[c] = the sum of part[0 .. parts)[c], in that order within each of 32 runs, the runs in order; in 64 bits, as where a
// CTA's groups are added: a sum of a few hundred rows is off by its terms' roundings and its own alone (512 x 256 in
// fp32: 6.8e-8, 1.3e-7 with 32).
__global__ void __launch_bounds__(1024) norm_dw_kernel(const float* __restrict__ part, int parts, int N,
                                                       void* __restrict__ dw, int w_dtype) {
  __shared__ double sums[32][33];
  asm volatile("griddepcontrol.wait;\n" ::: "memory");
  const int cx = threadIdx.x & 31, py = threadIdx.x >> 5, c = blockIdx.x * 32 + cx;
  const int run = (parts + 31) / 32, p1 = min(parts, (py + 1) * run);
  double t = 0.0;
  if (c < N)
#pragma unroll 8
    for (int p = py * run; p < p1; ++p) t += part[(int64_t)p * N + c];
  sums[py][cx] = t;
  __syncthreads();
  if (py == 0 && c < N) {
    t = 0.0;
#pragma unroll
    for (int i = 0; i < 32; ++i) t += sums[i][cx];
    store_as(dw, w_dtype, c, (float)t);
  }
}

// SwiGLU: one thread a vector of values and gates (backward: and gradients), or an element of each.
template <typename T, bool VEC, bool BWD>
__global__ void __launch_bounds__(kThreads) swiglu_rows_kernel(const T* __restrict__ x, const T* __restrict__ dy,
                                                               T* __restrict__ out, int64_t M, int N, int64_t xs,
                                                               int64_t ds, int64_t os) {
  constexpr int E = VEC ? Row16<T>::E : 1;
  const int nv = N / E;
  const int64_t total = M * nv;
  for (int64_t i = (int64_t)blockIdx.x * kThreads + threadIdx.x; i < total; i += (int64_t)gridDim.x * kThreads) {
    const int64_t row = i / nv;
    const int c = (int)(i - row * nv) * E;
    float v[E], g[E], d[E];
    if constexpr (VEC) {
      const uint4 vr = Row16<T>::load(x + row * xs + c), gr = Row16<T>::load(x + row * xs + N + c);
      if constexpr (BWD) Row16<T>::numbers(Row16<T>::load(dy + row * ds + c), d);
      Row16<T>::numbers(vr, v);
      Row16<T>::numbers(gr, g);
    } else {
      v[0] = to_f(x[row * xs + c]);
      g[0] = to_f(x[row * xs + N + c]);
      if constexpr (BWD) d[0] = to_f(dy[row * ds + c]);
    }
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const float sg = sig_(g[e]);
      if constexpr (BWD) {
        const float dv = d[e] * (g[e] * sg);
        g[e] = d[e] * v[e] * (sg * (1.0f + g[e] * (1.0f - sg)));
        v[e] = dv;
      } else {
        v[e] *= g[e] * sg;
      }
    }
    T* o = out + row * os + c;
    if constexpr (VEC) {
      Row16<T>::store(o, v);
      if constexpr (BWD) Row16<T>::store(o + N, g);
    } else {
      o[0] = from_f<T>(v[0]);
      if constexpr (BWD) o[N] = from_f<T>(g[0]);
    }
  }
}

template <typename F>
int by_dtype(int dtype, const char* what, F&& f) {
  if (dtype == MB_F32) return f(0.f);
  if (dtype == MB_BF16) return f(__nv_bfloat16{});
  if (dtype == MB_F16) return f(__half{});
  return set_error(MB_ERR_DTYPE, "%s: unsupported dtype code %d", what, dtype);
}

// How a call is cut: by 16-byte vectors, by elements or pairs of them, or a CTA a row; the threads of a row,
// vectors (elements) a thread, CTAs.
enum { kByVectors, kByElements, kByRows };
struct Plan {
  int way, g, n, grid;
};
Plan norm_plan(int64_t M, int64_t N, int elem_bytes, bool aligned, bool gated, bool bwd) {
  const int e = 16 / elem_bytes;
  Plan p = {};
  const int64_t vecs = N / e;
  int64_t each = 8;  // resident CTAs an SM
  if (aligned && N % e == 0 && vecs <= kThreads * 4) {
    p.way = kByVectors;
    p.g = vecs <= 8 ? 8 : vecs <= 16 ? 16 : vecs <= 128 ? 32 : kThreads;
    p.n = (int)((vecs + p.g - 1) / p.g);
    if (p.g == kThreads && p.n == 3) p.n = 4;
    each = bwd && p.n > (gated ? 2 : 3) ? 1 : kCtasPerSm;
  } else if (N <= 1024 || (bwd && N <= 32 * kThreads)) {  // forward, nothing is kept over the rows of long ones
    p.way = kByElements;
    p.g = N <= 1024 ? 32 : kThreads;
    p.n = N <= 8 * p.g ? 8 : N <= 16 * p.g ? 16 : 32;
    each = p.n == 8 ? 4 : p.n == 16 ? 3 : 2;
  } else {
    p.way = kByRows;
    p.g = kThreads;
  }
  const int64_t groups = kThreads / p.g, sms = multiprocessors();
  // one wave of CTAs; for very long rows dw's partial sums stay below 128 MB, or one row of them an SM
  const int64_t most = std::max<int64_t>(sms, std::min<int64_t>(sms * each, (1LL << 25) / N));
  p.grid = (int)std::min<int64_t>((M + groups - 1) / groups, most);
  return p;
}
// every row of the call begins at a multiple of `bytes`
bool norm_aligned(const NormArgs& a, int elem_bytes, bool bwd, int bytes) {
  const int64_t e = bytes / elem_bytes;
  uintptr_t at = (uintptr_t)a.x | (uintptr_t)a.out;
  int64_t strides = a.xs | a.os;
  if (bwd) {
    at |= (uintptr_t)a.dy;
    strides |= a.ds;
  }
  return at % bytes == 0 && strides % e == 0 && a.N % e == 0;
}

template <typename T, bool GATED, bool BWD>
int launch_norm(const NormArgs& a, const Plan& p, cudaStream_t st) {
  auto rows = [&](auto g, auto nv) {
    constexpr int G = decltype(g)::value, NV = decltype(nv)::value;
    constexpr int kTensors = 1 + GATED + BWD;
    // the ring; the groups' sums at the end (NV E floats a thread) fit in it: two stages of two tensors
    // are as large for 16-bit rows
    constexpr int smem = kThreads * 16 * NV * kTensors * stages<NV, GATED, BWD>();
    static_assert(smem >= kThreads * NV * Row16<T>::E * 4 || !BWD, "the sums fit");
    auto kern = norm_rows_kernel<T, G, NV, GATED, BWD>;
    if (int e = ensure_smem_attr((const void*)kern, smem)) return e;
    kern<<<p.grid, kThreads, smem, st>>>(a);
    return (int)MB_OK;
  };
  const bool two = norm_aligned(a, sizeof(T), BWD, 2 * sizeof(T));
  auto some = [&](auto g, auto l) {
    constexpr int G = decltype(g)::value, L = decltype(l)::value;
    auto kern = two ? norm_some_kernel<T, G, L, 2, GATED, BWD> : norm_some_kernel<T, G, L, 1, GATED, BWD>;
    kern<<<p.grid, kThreads, BWD && G < kThreads ? kThreads / G * a.N * 4 : 0, st>>>(a);
    return (int)MB_OK;
  };
  using std::integral_constant;
  int rc = MB_OK;
  integral_constant<int, 8> c8;
  integral_constant<int, 16> c16;
  integral_constant<int, 32> c32;
  integral_constant<int, kThreads> all;
  integral_constant<int, 1> n1;
  integral_constant<int, 2> n2;
  integral_constant<int, 3> n3;
  integral_constant<int, 4> n4;
  if (p.way == kByRows)
    norm_long_kernel<T, GATED, BWD><<<p.grid, kThreads, 0, st>>>(a);
  else if (p.way == kByElements && p.g == 32)
    rc = p.n == 8 ? some(c32, c8) : p.n == 16 ? some(c32, c16) : some(c32, c32);
  else if (p.way == kByElements) {
    if constexpr (BWD)  // (longer rows go forward a CTA at a time)
      rc = p.n == 8 ? some(all, c8) : p.n == 16 ? some(all, c16) : some(all, c32);
  }
  else if (p.g == 8)
    rc = rows(c8, n1);
  else if (p.g == 16)
    rc = rows(c16, n1);
  else if (p.g == 32)
    rc = p.n == 1 ? rows(c32, n1) : p.n == 2 ? rows(c32, n2) : p.n == 3 ? rows(c32, n3) : rows(c32, n4);
  else
    rc = p.n == 1 ? rows(all, n1) : p.n == 2 ? rows(all, n2) : rows(all, n4);
  if (rc) return rc;
  return check_launch(BWD ? "rms_norm_backward" : "rms_norm_train");
}

template <bool BWD>
int launch_swiglu(const char* what, const void* x, const void* dy, void* out, int64_t M, int64_t N, int64_t xs,
                  int64_t ds, int64_t os, int dtype, void* stream) {
  MB_REQUIRE(M == 0 || (x && out && (dy || !BWD)), MB_ERR_ARG, "%s: null pointer", what);
  MB_REQUIRE(M >= 0 && M < (1LL << 38) && N > 0 && N <= (1 << 24), MB_ERR_SHAPE, "%s: bad shape M=%lld N=%lld", what,
             (long long)M, (long long)N);
  return by_dtype(dtype, what, [&](auto t) {
    using T = decltype(t);
    constexpr int E = Row16<T>::E;
    const bool vec = N % E == 0 && (xs | ds | os) % E == 0 && ((uintptr_t)x | (uintptr_t)dy | (uintptr_t)out) % 16 == 0;
    const int64_t work = M * (vec ? N / E : N);
    if (M == 0) return (int)MB_OK;
    const unsigned grid = (unsigned)std::min<int64_t>((work + kThreads - 1) / kThreads, (int64_t)multiprocessors() * 32);
    auto kern = vec ? swiglu_rows_kernel<T, true, BWD> : swiglu_rows_kernel<T, false, BWD>;
    kern<<<grid, kThreads, 0, (cudaStream_t)stream>>>((const T*)x, (const T*)dy, (T*)out, M, (int)N, xs, ds, os);
    return check_launch(what);
  });
}

int elem_bytes(int dtype) { return dtype == MB_F32 ? 4 : 2; }

int check_norm(const char* what, int64_t M, int64_t N, int dtype, int w_dtype) {
  MB_REQUIRE(dtype == MB_F32 || dtype == MB_F16 || dtype == MB_BF16, MB_ERR_DTYPE, "%s: unsupported dtype code %d", what,
             dtype);
  MB_REQUIRE(w_dtype == MB_F32 || w_dtype == MB_F16 || w_dtype == MB_BF16, MB_ERR_DTYPE,
             "%s: unsupported weight dtype code %d", what, w_dtype);
  MB_REQUIRE(M >= 0 && M < (1LL << 40) && N > 0 && N <= (1 << 20), MB_ERR_SHAPE, "%s: bad shape M=%lld N=%lld", what,
             (long long)M, (long long)N);
  return MB_OK;
}

}  // namespace
}  // namespace mb

extern "C" int motif_b200_rms_norm_train(const void* x, const void* w, int w_dtype, void* y, int64_t M, int64_t N,
                                         int64_t xs, int64_t ys, int gated, float eps, int dtype, void* stream) {
  using namespace mb;
  MB_REQUIRE(M == 0 || (x && y), MB_ERR_ARG, "rms_norm_train: null pointer");
  if (int e = check_norm("rms_norm_train", M, N, dtype, w_dtype)) return e;
  if (M == 0) return MB_OK;
  NormArgs a = {};
  a.x = x;
  a.w = w;
  a.out = y;
  a.M = M;
  a.N = (int)N;
  a.xs = xs;
  a.os = ys;
  a.w_dtype = w_dtype;
  a.eps = eps;
  const Plan p = norm_plan(M, N, elem_bytes(dtype), norm_aligned(a, elem_bytes(dtype), false, 16), gated, false);
  return by_dtype(dtype, "rms_norm_train", [&](auto t) {
    using T = decltype(t);
    return gated ? launch_norm<T, true, false>(a, p, (cudaStream_t)stream)
                 : launch_norm<T, false, false>(a, p, (cudaStream_t)stream);
  });
}

extern "C" int64_t motif_b200_rms_norm_backward_workspace_bytes(int64_t M, int64_t N, int dtype) {
  using namespace mb;
  if (check_norm("rms_norm_backward_workspace_bytes", M, N, dtype, MB_F32)) return -1;
  // the most of all ways of cutting a call of these sizes (by the alignment of its tensors, and gated or not)
  int64_t parts = 1;
  for (int i = 0; i < 4; ++i)
    parts = std::max<int64_t>(parts, norm_plan(M, N, elem_bytes(dtype), i & 1, i & 2, true).grid);
  return parts * N * 4;
}

extern "C" int motif_b200_rms_norm_backward(const void* x, const void* w, int w_dtype, const void* dy, void* dx,
                                            void* dw, int64_t M, int64_t N, int64_t xs, int64_t ds, int64_t os,
                                            int gated, float eps, void* workspace, int64_t workspace_bytes, int dtype,
                                            void* stream) {
  using namespace mb;
  MB_REQUIRE(M == 0 || (x && dy && dx), MB_ERR_ARG, "rms_norm_backward: null pointer");
  if (int e = check_norm("rms_norm_backward", M, N, dtype, w_dtype)) return e;
  MB_REQUIRE(!dw || w, MB_ERR_ARG, "rms_norm_backward: the gradient of a weight that is not there");
  MB_REQUIRE(!dw || (workspace && workspace_bytes >= motif_b200_rms_norm_backward_workspace_bytes(M, N, dtype)), MB_ERR_ARG,
             "rms_norm_backward: workspace of %lld bytes is too small", (long long)workspace_bytes);
  cudaStream_t st = (cudaStream_t)stream;
  NormArgs a = {};
  a.x = x;
  a.w = w;
  a.dy = dy;
  a.out = dx;
  a.part = dw ? (float*)workspace : nullptr;
  a.M = M;
  a.N = (int)N;
  a.xs = xs;
  a.ds = ds;
  a.os = os;
  a.w_dtype = w_dtype;
  a.eps = eps;
  const Plan p = norm_plan(M, N, elem_bytes(dtype), norm_aligned(a, elem_bytes(dtype), true, 16), gated, true);
  if (M > 0) {
    const int rc = by_dtype(dtype, "rms_norm_backward", [&](auto t) {
      using T = decltype(t);
      return gated ? launch_norm<T, true, true>(a, p, st) : launch_norm<T, false, true>(a, p, st);
    });
    if (rc) return rc;
  }
  if (!dw) return MB_OK;
  const int parts = p.grid;  // 0 for no rows: dw is zero
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.gridDim = dim3((unsigned)((N + 31) / 32));
  cfg.blockDim = dim3(1024);
  cfg.stream = st;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  cudaLaunchKernelEx(&cfg, norm_dw_kernel, (const float*)workspace, parts, (int)N, dw, w_dtype);
  return check_launch("rms_norm_backward (weight)");
}

extern "C" int motif_b200_swiglu_train(const void* x, void* y, int64_t M, int64_t N, int64_t xs, int64_t ys, int dtype,
                                       void* stream) {
  return mb::launch_swiglu<false>("swiglu_train", x, nullptr, y, M, N, xs, 0, ys, dtype, stream);
}

extern "C" int motif_b200_swiglu_backward(const void* x, const void* dy, void* dx, int64_t M, int64_t N, int64_t xs,
                                          int64_t ds, int64_t os, int dtype, void* stream) {
  return mb::launch_swiglu<true>("swiglu_backward", x, dy, dx, M, N, xs, ds, os, dtype, stream);
}
