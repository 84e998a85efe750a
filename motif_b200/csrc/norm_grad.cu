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
// and leaves one row of partial sums, and a second kernel adds those in order: no atomics, the same
// bits every time.
#include <algorithm>

#include "common.cuh"

namespace mb {
namespace {

constexpr int kThreads = 256;
constexpr int kCtasPerSm = 4;      // partial sums are written once a CTA, so the grid stays this small

template <typename T> struct Row16 {
  static constexpr int E = 16 / (int)sizeof(T);  // elements of a 16-byte vector
  __device__ static void load(const T* p, float (&v)[E]) {
    const uint4 u = *reinterpret_cast<const uint4*>(p);
    const T* e = reinterpret_cast<const T*>(&u);
#pragma unroll
    for (int i = 0; i < E; ++i) v[i] = to_f(e[i]);
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

// sig(g) with the MUFU exponential and reciprocal (relative error a few 1e-7)
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

// Sum of (a, b) over the G threads of a row.  G > 32: over the CTA, through `red` (two slots in
// turn, so one barrier a row is enough).
template <int G>
__device__ __forceinline__ float2 row_sum(float2 v, float2 (*red)[kThreads / 32], int& slot) {
#pragma unroll
  for (int o = (G < 32 ? G : 32) / 2; o > 0; o >>= 1) {
    v.x += __shfl_xor_sync(0xffffffffu, v.x, o);
    v.y += __shfl_xor_sync(0xffffffffu, v.y, o);
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

// Rows whose length is a multiple of the vector and whose addresses are 16-byte aligned.
template <typename T, int G, int NV, bool GATED, bool BWD>
__global__ void __launch_bounds__(kThreads) norm_rows_kernel(const NormArgs a) {
  constexpr int E = Row16<T>::E;
  constexpr int kGroups = kThreads / G;
  __shared__ float2 red[2][kThreads / 32];
  extern __shared__ float acc[];  // BWD, G < kThreads: [kGroups][G * NV * E] at the end
  const int lane = threadIdx.x % G, group = threadIdx.x / G;
  const int N = a.N;
  int slot = 0;
  float w[NV][E], dw[NV][E];
#pragma unroll
  for (int v = 0; v < NV; ++v) {
    const int c = (v * G + lane) * E;
#pragma unroll
    for (int e = 0; e < E; ++e) {
      w[v][e] = c < N ? (a.w ? load_as(a.w, a.w_dtype, c + e) : 1.0f) : 0.0f;
      dw[v][e] = 0.0f;
    }
  }
  const float inv_n = 1.0f / (float)N;
  const int64_t step = (int64_t)gridDim.x * kGroups;
  // every thread of the CTA makes the same number of rounds: the row sums are taken together
  for (int64_t row0 = (int64_t)blockIdx.x * kGroups; row0 < a.M; row0 += step) {
    const int64_t row = row0 + group;
    const bool live = row < a.M;
    const T* xr = reinterpret_cast<const T*>(a.x) + row * a.xs;
    const T* dr = reinterpret_cast<const T*>(a.dy) + row * a.ds;
    float x[NV][E], g[GATED ? NV : 1][E], d[BWD ? NV : 1][E];
    float2 s = make_float2(0.f, 0.f);
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      const int c = (v * G + lane) * E;
      const bool in = live && c < N;
      if (in) {
        Row16<T>::load(xr + c, x[v]);
        if constexpr (GATED) Row16<T>::load(xr + N + c, g[v]);
        if constexpr (BWD) Row16<T>::load(dr + c, d[v]);
      } else {
#pragma unroll
        for (int e = 0; e < E; ++e) {
          x[v][e] = 0.f;
          if constexpr (GATED) g[v][e] = 0.f;
          if constexpr (BWD) d[v][e] = 0.f;
        }
      }
    }
#pragma unroll
    for (int v = 0; v < NV; ++v)
#pragma unroll
      for (int e = 0; e < E; ++e) {
        s.x = fmaf(x[v][e], x[v][e], s.x);
        if constexpr (BWD) {
          float t = d[v][e] * w[v][e];
          if constexpr (GATED) t *= g[v][e] * sig_(g[v][e]);
          s.y = fmaf(t, x[v][e], s.y);
        }
      }
    s = row_sum<G>(s, red, slot);
    const float r = rsqrtf(s.x * inv_n + a.eps);
    const float k = s.y * inv_n * r * r;
    T* outr = reinterpret_cast<T*>(a.out) + row * a.os;
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      const int c = (v * G + lane) * E;
      if (!live || c >= N) continue;
      float o[E], og[GATED ? E : 1];
#pragma unroll
      for (int e = 0; e < E; ++e) {
        const float xh = x[v][e] * r;
        float act = 1.0f, sg = 0.f;
        if constexpr (GATED) {
          sg = sig_(g[v][e]);
          act = g[v][e] * sg;
        }
        if constexpr (BWD) {
          const float dn = GATED ? d[v][e] * act : d[v][e];
          dw[v][e] = fmaf(dn, xh, dw[v][e]);
          o[e] = r * (dn * w[v][e] - x[v][e] * k);
          if constexpr (GATED) og[e] = d[v][e] * (xh * w[v][e]) * (sg * (1.0f + g[v][e] * (1.0f - sg)));
        } else {
          o[e] = xh * w[v][e];
          if constexpr (GATED) o[e] *= act;
        }
      }
      Row16<T>::store(outr + c, o);
      if constexpr (BWD && GATED) Row16<T>::store(outr + N + c, og);
    }
  }
  if constexpr (BWD) {
    if (a.part == nullptr) return;
    float* pr = a.part + (int64_t)blockIdx.x * N;
    if constexpr (G == kThreads) {
#pragma unroll
      for (int v = 0; v < NV; ++v)
#pragma unroll
        for (int e = 0; e < E; ++e)
          if ((v * G + lane) * E < N) pr[(v * G + lane) * E + e] = dw[v][e];
    } else {
      constexpr int W = G * NV * E;
#pragma unroll
      for (int v = 0; v < NV; ++v)
#pragma unroll
        for (int e = 0; e < E; ++e) acc[group * W + (v * G + lane) * E + e] = dw[v][e];
      __syncthreads();
      for (int c = threadIdx.x; c < N; c += kThreads) {
        float t = 0.f;
#pragma unroll 4
        for (int i = 0; i < kGroups; ++i) t += acc[i * W + c];
        pr[c] = t;
      }
    }
  }
}

// Any length and alignment: one row at a time per group of G threads (a warp, or the CTA for long
// rows), element by element, the row read twice (the second time from the L1).  A group's partial
// sums of dw live in its own row of `part`, each column always touched by the same thread.
template <typename T, int G, bool GATED, bool BWD>
__global__ void __launch_bounds__(kThreads) norm_any_kernel(const NormArgs a) {
  constexpr int kGroups = kThreads / G;
  __shared__ float2 red[2][kThreads / 32];
  const int lane = threadIdx.x % G, group = threadIdx.x / G;
  const int N = a.N;
  int slot = 0;
  const float inv_n = 1.0f / (float)N;
  const int64_t step = (int64_t)gridDim.x * kGroups;
  float* pr = BWD && a.part ? a.part + ((int64_t)blockIdx.x * kGroups + group) * N : nullptr;
  if (pr)
    for (int c = lane; c < N; c += G) pr[c] = 0.f;
  for (int64_t row0 = (int64_t)blockIdx.x * kGroups; row0 < a.M; row0 += step) {
    const int64_t row = row0 + group;
    const bool live = row < a.M;
    const T* xr = reinterpret_cast<const T*>(a.x) + row * a.xs;
    const T* dr = reinterpret_cast<const T*>(a.dy) + row * a.ds;
    float2 s = make_float2(0.f, 0.f);
    if (live)
      for (int c = lane; c < N; c += G) {
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
    s = row_sum<G>(s, red, slot);
    if (!live) continue;
    const float r = rsqrtf(s.x * inv_n + a.eps);
    const float k = s.y * inv_n * r * r;
    T* outr = reinterpret_cast<T*>(a.out) + row * a.os;
    for (int c = lane; c < N; c += G) {
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
        if constexpr (GATED) outr[N + c] = from_f<T>(d * (xh * w) * (sg * (1.0f + g * (1.0f - sg))));
      } else {
        outr[c] = from_f<T>(GATED ? xh * w * act : xh * w);
      }
    }
  }
}

// dw[c] = the sum of part[0 .. parts)[c], in that order within each of 32 runs, the runs in order.
__global__ void __launch_bounds__(1024) norm_dw_kernel(const float* __restrict__ part, int parts, int N,
                                                       void* __restrict__ dw, int w_dtype) {
  __shared__ float sums[32][33];
  const int cx = threadIdx.x & 31, py = threadIdx.x >> 5, c = blockIdx.x * 32 + cx;
  const int run = (parts + 31) / 32, p1 = min(parts, (py + 1) * run);
  float t = 0.f;
  if (c < N)
#pragma unroll 8
    for (int p = py * run; p < p1; ++p) t += part[(int64_t)p * N + c];
  sums[py][cx] = t;
  __syncthreads();
  if (py == 0 && c < N) {
    t = 0.f;
#pragma unroll
    for (int i = 0; i < 32; ++i) t += sums[i][cx];
    store_as(dw, w_dtype, c, t);
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
      Row16<T>::load(x + row * xs + c, v);
      Row16<T>::load(x + row * xs + N + c, g);
      if constexpr (BWD) Row16<T>::load(dy + row * ds + c, d);
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

// How a call is cut: threads of a row, vectors a thread (0: element by element), CTAs.
struct Plan {
  int g, nv, grid;
};
Plan norm_plan(int64_t M, int64_t N, int elem_bytes, bool aligned) {
  const int e = 16 / elem_bytes;
  Plan p = {};
  const int64_t vecs = N / e;
  if (!aligned || N % e != 0 || vecs > kThreads * 4) {
    p.g = N > 1024 ? kThreads : 32;
  } else if (vecs <= 32) {
    p.g = vecs <= 8 ? 8 : vecs <= 16 ? 16 : 32;
    p.nv = 1;
  } else if (vecs <= 128) {
    p.g = 32;
    p.nv = (int)((vecs + 31) / 32);
  } else {
    p.g = kThreads;
    p.nv = vecs <= kThreads ? 1 : vecs <= 2 * kThreads ? 2 : 4;
  }
  const int64_t groups = kThreads / p.g;
  // very long rows: the partial sums of dw stay below 128 MB, or one row of them an SM
  const int64_t most = std::max<int64_t>(148, std::min<int64_t>(148 * kCtasPerSm, (1LL << 25) / N));
  p.grid = (int)std::min<int64_t>((M + groups - 1) / groups, most);
  return p;
}
// rows of partial sums that a call leaves
int64_t norm_parts(const Plan& p) { return p.nv ? p.grid : (int64_t)p.grid * (kThreads / p.g); }
bool norm_aligned(const NormArgs& a, int elem_bytes, bool bwd) {
  const int64_t e = 16 / elem_bytes;
  uintptr_t at = (uintptr_t)a.x | (uintptr_t)a.out;
  int64_t strides = a.xs | a.os;
  if (bwd) {
    at |= (uintptr_t)a.dy;
    strides |= a.ds;
  }
  return at % 16 == 0 && strides % e == 0;
}

template <typename T, bool GATED, bool BWD>
int launch_norm(const NormArgs& a, const Plan& p, cudaStream_t st) {
  auto rows = [&](auto g, auto nv) {
    constexpr int G = decltype(g)::value, NV = decltype(nv)::value;
    const int smem = BWD && G < kThreads ? kThreads * NV * Row16<T>::E * 4 : 0;
    norm_rows_kernel<T, G, NV, GATED, BWD><<<p.grid, kThreads, smem, st>>>(a);
  };
  using std::integral_constant;
  if (p.nv == 0) {
    if (p.g == 32)
      norm_any_kernel<T, 32, GATED, BWD><<<p.grid, kThreads, 0, st>>>(a);
    else
      norm_any_kernel<T, kThreads, GATED, BWD><<<p.grid, kThreads, 0, st>>>(a);
  } else if (p.g == 8) {
    rows(integral_constant<int, 8>{}, integral_constant<int, 1>{});
  } else if (p.g == 16) {
    rows(integral_constant<int, 16>{}, integral_constant<int, 1>{});
  } else if (p.g == 32) {
    if (p.nv == 1) rows(integral_constant<int, 32>{}, integral_constant<int, 1>{});
    if (p.nv == 2) rows(integral_constant<int, 32>{}, integral_constant<int, 2>{});
    if (p.nv == 3) rows(integral_constant<int, 32>{}, integral_constant<int, 3>{});
    if (p.nv == 4) rows(integral_constant<int, 32>{}, integral_constant<int, 4>{});
  } else {
    if (p.nv == 1) rows(integral_constant<int, kThreads>{}, integral_constant<int, 1>{});
    if (p.nv == 2) rows(integral_constant<int, kThreads>{}, integral_constant<int, 2>{});
    if (p.nv == 4) rows(integral_constant<int, kThreads>{}, integral_constant<int, 4>{});
  }
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
    const unsigned grid = (unsigned)std::min<int64_t>((work + kThreads - 1) / kThreads, 148LL * 32);
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
  const Plan p = norm_plan(M, N, elem_bytes(dtype), norm_aligned(a, elem_bytes(dtype), false));
  return by_dtype(dtype, "rms_norm_train", [&](auto t) {
    using T = decltype(t);
    return gated ? launch_norm<T, true, false>(a, p, (cudaStream_t)stream)
                 : launch_norm<T, false, false>(a, p, (cudaStream_t)stream);
  });
}

extern "C" int64_t motif_b200_rms_norm_backward_workspace_bytes(int64_t M, int64_t N, int dtype) {
  using namespace mb;
  if (check_norm("rms_norm_backward_workspace_bytes", M, N, dtype, MB_F32)) return -1;
  // the more of both ways of cutting a call of these sizes (by the alignment of its tensors)
  const int64_t parts = std::max(norm_parts(norm_plan(M, N, elem_bytes(dtype), true)),
                                 norm_parts(norm_plan(M, N, elem_bytes(dtype), false)));
  return std::max<int64_t>(parts, 1) * N * 4;
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
  const Plan p = norm_plan(M, N, elem_bytes(dtype), norm_aligned(a, elem_bytes(dtype), true));
  if (M > 0) {
    const int rc = by_dtype(dtype, "rms_norm_backward", [&](auto t) {
      using T = decltype(t);
      return gated ? launch_norm<T, true, true>(a, p, st) : launch_norm<T, false, true>(a, p, st);
    });
    if (rc) return rc;
  }
  if (!dw) return MB_OK;
  const int parts = (int)norm_parts(p);  // 0 for no rows: dw is zero
  norm_dw_kernel<<<(unsigned)((N + 31) / 32), 1024, 0, st>>>((const float*)workspace, parts, (int)N, dw, w_dtype);
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
