// The vocabulary loss (vocab_loss.cu has the formulas) of at most 16 fp32 tokens, on the CUDA cores.
//
// So few tokens leave the weight's bytes as the bound, 4 a weight for the loss and 12 with its gradients (W twice, dW
// once).  Splitting W into three bf16 parts for the tensor cores moves 16 and 30 instead.  Loss and loss with gradients,
// us, here and there:
//   tokens x d x words     8 x 1952 x 107248    16 x 1952 x 107248    8 x 768 x 32000    16 x 64 x 300
//   here                   178, 588             252, 737              35, 105            12, 25
//   on the tensor cores    865, 1648            871, 1661             115, 247           22, 51
// The first is 4.7 and 4.3 TB/s of W's and dW's bytes.  From 16 tokens on fp32 products are the bound, 4 N of them to
// each 4 bytes of W, and the tensor cores gain on them: hence the limit.
//
//   scores   x in shared memory; a warp takes four rows of W at a time, so that a value of x serves four products, and
//            leaves the logits [V][R] (64 bytes a word at most, a part of what W has) with a running maximum and
//            sum of exponentials for each lane's tokens.
//   grads    a thread keeps four columns of all tokens' x (or dx) in registers and walks words: dW's row is a
//            sum over the tokens, dx gains a multiple of W's row.  The CTAs' sums of dx are added in order.
#include <algorithm>

#include "vocab_few.cuh"

namespace mb {
namespace {

constexpr int kMost = 16;  // tokens
constexpr int kThreads = 256;
constexpr int kScoreThreads = 512;
constexpr float kLog2e = 1.4426950408889634f;
constexpr int64_t kMostDim = 3200;  // 16 rows of x in shared memory

struct Few {
  const float *x, *w;
  int64_t xs, ws;
  const int64_t* labels;
  int64_t ignore;
  int N, V, d, dp;      // dp: d rounded up to four
  int reduction, ctas;  // of the scores
  float* rows;          // [R][dp], zeros behind the tokens
  float* s;             // [V][R]
  float2* seg;          // [ctas][R]
  float* target;        // [R]
  float2* stat;         // [R]: largest logit, 1 / sum
  int* place;           // [N]
  int* index;           // [R]
  int* label;           // [R]
  int* count;
  float* loss;
  const float* up;
  int64_t up_stride;
  float *dx, *dw, *part;  // part: [grads' CTAs][R][dp]
};

__device__ __forceinline__ void wait_for_previous() { asm volatile("griddepcontrol.wait;\n" ::: "memory"); }

// Four columns of a row of d, zeros behind it.
__device__ __forceinline__ float4 load4(const float* p, int c, int d, bool aligned) {
  if (aligned && c + 4 <= d) return *reinterpret_cast<const float4*>(p + c);
  float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
  if (c < d) v.x = p[c];
  if (c + 1 < d) v.y = p[c + 1];
  if (c + 2 < d) v.z = p[c + 2];
  if (c + 3 < d) v.w = p[c + 3];
  return v;
}
__device__ __forceinline__ bool rows_aligned(const float* p, int64_t stride) {
  return (reinterpret_cast<uintptr_t>(p) & 15) == 0 && stride % 4 == 0;
}

// Every CTA finds the tokens that have a loss, the first one writes what it finds; each copies its part of x.
template <int R>
__global__ void __launch_bounds__(kThreads) few_pack_kernel(const Few a) {
  __shared__ int from[R];
  allow_dependent_launch();
  wait_for_previous();
  const int tid = threadIdx.x;
  if (tid < 32) {
    const int64_t label = tid < a.N ? a.labels[tid] : a.ignore;
    const bool live = tid < a.N && label != a.ignore;
    const unsigned vote = __ballot_sync(0xffffffffu, live);
    const int at = __popc(vote & ((1u << tid) - 1u));
    if (tid < R) from[tid] = -1;
    __syncwarp();
    if (live) from[at] = tid;
    if (blockIdx.x == 0) {
      if (live) {
        a.index[at] = tid;
        a.label[at] = label >= 0 && label < a.V ? (int)label : -1;
      }
      if (tid < a.N) {
        a.place[tid] = live ? at : -1;
        if (!live && a.reduction == 0) a.loss[tid] = 0.f;
      }
      if (tid == 0) *a.count = __popc(vote);
    }
  }
  __syncthreads();
  for (int i = blockIdx.x * kThreads + tid; i < R * a.dp; i += gridDim.x * kThreads) {
    const int r = i / a.dp, c = i - r * a.dp;
    a.rows[i] = from[r] >= 0 && c < a.d ? a.x[from[r] * a.xs + c] : 0.f;
  }
}

__device__ __forceinline__ void add_to(float& top, float& sum, float s) {
  if (s > top) {
    sum *= ex2f_((top - s) * kLog2e);
    top = s;
  }
  sum += ex2f_((s - (top == -INFINITY ? 0.f : top)) * kLog2e);
}
__device__ __forceinline__ void join(float& top, float& sum, float t2, float s2) {
  const float now = fmaxf(top, t2), ref = now == -INFINITY ? 0.f : now;
  sum = sum * ex2f_((top - ref) * kLog2e) + s2 * ex2f_((t2 - ref) * kLog2e);
  top = now;
}

template <int R>
__global__ void __launch_bounds__(kScoreThreads, 1) few_scores_kernel(const Few a) {
  constexpr int kWords = 4, kHeld = kWords * R / 32;  // sums that a lane ends with
  extern __shared__ float4 xs[];                      // [R][dp / 4]
  __shared__ float2 runs[kScoreThreads / 32][kWords * R];
  allow_dependent_launch();
  wait_for_previous();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = kScoreThreads / 32;
  const int dq = a.dp / 4;
  for (int i = threadIdx.x; i < R * dq; i += kScoreThreads) xs[i] = reinterpret_cast<const float4*>(a.rows)[i];
  const bool aligned = rows_aligned(a.w, a.ws);
  float top[kHeld], sum[kHeld];
  int label[kHeld];
#pragma unroll
  for (int i = 0; i < kHeld; ++i) {
    const int r = (lane * kHeld + i) % R;
    top[i] = -INFINITY;
    sum[i] = 0.f;
    label[i] = r < *a.count ? a.label[r] : -1;
  }
  __syncthreads();
  for (int v0 = (blockIdx.x * warps + warp) * kWords; v0 < a.V; v0 += gridDim.x * warps * kWords) {
    float acc[kWords * R];
#pragma unroll
    for (int i = 0; i < kWords * R; ++i) acc[i] = 0.f;
    const float* w = a.w + (int64_t)v0 * a.ws;
    for (int q0 = lane; q0 < dq; q0 += 64) {
      float4 wq[2][kWords];
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int k = 0; k < kWords; ++k)
          wq[h][k] = v0 + k < a.V && q0 + 32 * h < dq ? load4(w + k * a.ws, 4 * (q0 + 32 * h), a.d, aligned)
                                                      : make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        if (q0 + 32 * h >= dq) break;
#pragma unroll
        for (int r = 0; r < R; ++r) {
          const float4 x = xs[r * dq + q0 + 32 * h];
#pragma unroll
          for (int k = 0; k < kWords; ++k) {
            float& t = acc[k * R + r];
            t = fmaf(x.x, wq[h][k].x, t);
            t = fmaf(x.y, wq[h][k].y, t);
            t = fmaf(x.z, wq[h][k].z, t);
            t = fmaf(x.w, wq[h][k].w, t);
          }
        }
      }
    }
    // the warp's sums: each step hands half of the values over, so a lane ends with its own few of all
#pragma unroll
    for (int o = 16, n = kWords * R / 2; o > 0; o >>= 1, n >>= 1) {
      const bool upper = lane & o;
#pragma unroll
      for (int i = 0; i < kWords * R / 2; ++i)
        if (i < n) {
          const float give = upper ? acc[i] : acc[i + n], keep = upper ? acc[i + n] : acc[i];
          acc[i] = keep + __shfl_xor_sync(0xffffffffu, give, o);
        }
    }
#pragma unroll
    for (int i = 0; i < kHeld; ++i) {
      const int at = lane * kHeld + i, v = v0 + at / R;
      if (v < a.V) {
        a.s[(int64_t)v0 * R + at] = acc[i];
        add_to(top[i], sum[i], acc[i]);
        if (label[i] == v) a.target[at % R] = acc[i];
      }
    }
  }
#pragma unroll
  for (int i = 0; i < kHeld; ++i) runs[warp][lane * kHeld + i] = make_float2(top[i], sum[i]);
  __syncthreads();
  if (threadIdx.x < R) {
    float t = -INFINITY, s = 0.f;
    for (int i = 0; i < warps; ++i)
      for (int k = 0; k < kWords; ++k) join(t, s, runs[i][k * R + threadIdx.x].x, runs[i][k * R + threadIdx.x].y);
    a.seg[blockIdx.x * R + threadIdx.x] = make_float2(t, s);
  }
}

// One CTA, a warp a token.
template <int R>
__global__ void __launch_bounds__(32 * R) few_join_kernel(const Few a) {
  __shared__ double losses[R];
  allow_dependent_launch();
  wait_for_previous();
  const int lane = threadIdx.x & 31, r = threadIdx.x >> 5, live = *a.count;
  float top = -INFINITY, sum = 0.f;
  for (int i = lane; i < a.ctas; i += 32) {
    const float2 v = a.seg[i * R + r];
    join(top, sum, v.x, v.y);
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const float t2 = __shfl_down_sync(0xffffffffu, top, o), s2 = __shfl_down_sync(0xffffffffu, sum, o);
    join(top, sum, t2, s2);
  }
  if (lane == 0) {
    const float nan = __int_as_float(0x7fffffff), ref = top == -INFINITY ? 0.f : top;
    const bool known = r < live && a.label[r] >= 0;  // a label that is no word: NaN, in the gradients too
    a.stat[r] = make_float2(ref, known ? 1.0f / sum : nan);
    const float one = known ? (ref - a.target[r]) + logf(sum) : nan;
    losses[r] = r < live ? (double)one : 0.0;
    if (a.reduction == 0 && r < live) a.loss[a.index[r]] = one;
  }
  __syncthreads();
  if (threadIdx.x == 0 && a.reduction != 0) {
    double loss = 0.0;
    for (int i = 0; i < R; ++i) loss += losses[i];
    *a.loss = (float)(a.reduction == 1 ? loss / (double)live : loss);  // no tokens: 0 / 0, as it is
  }
}

__device__ __forceinline__ float few_scale(const Few& a) {
  const int live = *a.count;
  if (a.reduction == 0) return 1.0f;
  if (live <= 0) return 0.0f;
  return (a.up ? *a.up : 1.0f) * (a.reduction == 1 ? 1.0f / (float)live : 1.0f);
}

// A CTA has 1024 columns (blockIdx.y) and a run of words; T threads share a row's columns, the groups of T take
// words in turn.  DX: partial sums of dx; else dW's rows.
template <int R, bool DX>
__global__ void __launch_bounds__(kThreads, 2) few_grads_kernel(const Few a, int T, int words) {
  constexpr int kTile = 64;
  __shared__ float4 g[kTile][R / 4];
  __shared__ float4 turn[kThreads];
  allow_dependent_launch();
  wait_for_previous();
  const int groups = kThreads / T, group = threadIdx.x / T, c = blockIdx.y * 1024 + 4 * (threadIdx.x % T);
  const bool mine = c < a.dp && 4 * (threadIdx.x % T) < 1024;
  const int live = *a.count, begin = blockIdx.x * words, end = min(a.V, begin + words);
  const bool aligned = DX ? rows_aligned(a.w, a.ws) : rows_aligned(a.dw, a.d);
  const float scale = few_scale(a);
  float4 v[R];  // DX: the sums of dx; else x
#pragma unroll
  for (int r = 0; r < R; ++r) {
    v[r] = make_float4(0.f, 0.f, 0.f, 0.f);
    if (!DX && mine) v[r] = *reinterpret_cast<const float4*>(a.rows + r * a.dp + c);
  }
  for (int v0 = begin; v0 < end; v0 += kTile) {
    __syncthreads();
    for (int i = threadIdx.x; i < kTile * R; i += kThreads) {
      const int word = v0 + i / R, r = i % R;
      float p = 0.f;
      if (word < end && r < live) {
        const float2 st = a.stat[r];
        p = ex2f_((a.s[(int64_t)word * R + r] - st.x) * kLog2e) * st.y;
        if (a.label[r] == word) p -= 1.0f;
        if (a.reduction == 0) p *= a.up[a.index[r] * a.up_stride];
      }
      reinterpret_cast<float*>(&g[i / R][0])[r] = p;
    }
    __syncthreads();
    const int n = min(kTile, end - v0);
    if (DX) {
      for (int k0 = group; k0 < n; k0 += 4 * groups) {
        float4 w[4];
#pragma unroll
        for (int h = 0; h < 4; ++h)
          if (mine && k0 + h * groups < n)
            w[h] = load4(a.w + (int64_t)(v0 + k0 + h * groups) * a.ws, c, a.d, aligned);
#pragma unroll
        for (int h = 0; h < 4; ++h)
          if (mine && k0 + h * groups < n) {
#pragma unroll
            for (int q = 0; q < R / 4; ++q) {
              const float4 p = g[k0 + h * groups][q];
              const float e[4] = {p.x, p.y, p.z, p.w};
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                float4& t = v[4 * q + i];
                t.x = fmaf(e[i], w[h].x, t.x);
                t.y = fmaf(e[i], w[h].y, t.y);
                t.z = fmaf(e[i], w[h].z, t.z);
                t.w = fmaf(e[i], w[h].w, t.w);
              }
            }
          }
      }
    } else if (mine) {
      for (int k = group; k < n; k += groups) {
        float4 t = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int q = 0; q < R / 4; ++q) {
          const float4 p = g[k][q];
          const float e[4] = {p.x, p.y, p.z, p.w};
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            t.x = fmaf(e[i], v[4 * q + i].x, t.x);
            t.y = fmaf(e[i], v[4 * q + i].y, t.y);
            t.z = fmaf(e[i], v[4 * q + i].z, t.z);
            t.w = fmaf(e[i], v[4 * q + i].w, t.w);
          }
        }
        float* out = a.dw + (int64_t)(v0 + k) * a.d + c;
        if (aligned && c + 4 <= a.d) {
          *reinterpret_cast<float4*>(out) = make_float4(t.x * scale, t.y * scale, t.z * scale, t.w * scale);
        } else {
          if (c < a.d) out[0] = t.x * scale;
          if (c + 1 < a.d) out[1] = t.y * scale;
          if (c + 2 < a.d) out[2] = t.z * scale;
          if (c + 3 < a.d) out[3] = t.w * scale;
        }
      }
    }
  }
  if (DX) {
#pragma unroll
    for (int r = 0; r < R; ++r) {
      turn[threadIdx.x] = v[r];
      __syncthreads();
      if (group == 0 && mine) {
        float4 t = turn[threadIdx.x];
        for (int i = 1; i < groups; ++i) {
          const float4 o = turn[threadIdx.x + i * T];
          t.x += o.x;
          t.y += o.y;
          t.z += o.z;
          t.w += o.w;
        }
        *reinterpret_cast<float4*>(a.part + ((int64_t)blockIdx.x * R + r) * a.dp + c) = t;
      }
      __syncthreads();
    }
  }
}

// dx of token blockIdx.x: the CTAs' sums, in runs of eight that are added in order; zeros without a loss.
template <int R>
__global__ void __launch_bounds__(256) few_dx_kernel(const Few a, int parts) {
  __shared__ float sums[8][33];
  allow_dependent_launch();
  wait_for_previous();
  const int r = a.place[blockIdx.x], cx = threadIdx.x & 31, py = threadIdx.x >> 5, c = blockIdx.y * 32 + cx;
  float t = 0.f;
  if (r >= 0 && c < a.d) {
    const int run = (parts + 7) / 8, end = min(parts, (py + 1) * run);
#pragma unroll 8
    for (int p = py * run; p < end; ++p) t += a.part[((int64_t)p * R + r) * a.dp + c];
  }
  sums[py][cx] = t;
  __syncthreads();
  if (py != 0 || c >= a.d) return;
  t = 0.f;
#pragma unroll
  for (int i = 0; i < 8; ++i) t += sums[i][cx];
  a.dx[(int64_t)blockIdx.x * a.d + c] = r >= 0 ? t * few_scale(a) : 0.f;
}

int64_t up_to(int64_t n, int64_t m) { return (n + m - 1) / m * m; }
int few_rows(int64_t N) { return N <= 8 ? 8 : kMost; }
int few_ctas() { return std::max(1, multiprocessors()); }       // of the scores
int few_parts() { return 2 * std::max(4, multiprocessors()); }  // of dx's sums, at most

struct Layout {
  int64_t rows, s, stat, place, index, label, count, state;
  int64_t seg, target, forward, part, backward;
};
Layout layout_of(int64_t N, int64_t V, int64_t d) {
  Layout l = {};
  const int64_t R = few_rows(N), dp = up_to(d, 4);
  auto take = [](int64_t& total, int64_t bytes) {
    const int64_t at = total;
    total = up_to(total + bytes, 256);
    return at;
  };
  l.rows = take(l.state, R * dp * 4);
  l.s = take(l.state, V * R * 4);
  l.stat = take(l.state, R * 8);
  l.place = take(l.state, kMost * 4);
  l.index = take(l.state, R * 4);
  l.label = take(l.state, R * 4);
  l.count = take(l.state, 4);
  l.seg = take(l.forward, few_ctas() * R * 8);
  l.target = take(l.forward, R * 4);
  l.part = take(l.backward, few_parts() * R * dp * 4);
  return l;
}

template <typename K, typename... A>
int launch(const char* what, K kern, dim3 grid, int threads, int smem, cudaStream_t st, A... args) {
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.gridDim = grid;
  cfg.blockDim = dim3((unsigned)threads);
  cfg.dynamicSmemBytes = (size_t)smem;
  cfg.stream = st;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  cudaLaunchKernelEx(&cfg, kern, args...);
  return check_launch(what);
}

Few few_of(const FewCall& c) {
  const Layout l = layout_of(c.N, c.V, c.d);
  Few a = {};
  a.x = c.x;
  a.w = c.w;
  a.xs = c.xs;
  a.ws = c.ws;
  a.labels = c.labels;
  a.ignore = c.ignore;
  a.N = (int)c.N;
  a.V = (int)c.V;
  a.d = (int)c.d;
  a.dp = (int)up_to(c.d, 4);
  a.reduction = c.reduction;
  a.ctas = few_ctas();
  a.rows = reinterpret_cast<float*>(c.state + l.rows);
  a.s = reinterpret_cast<float*>(c.state + l.s);
  a.stat = reinterpret_cast<float2*>(c.state + l.stat);
  a.place = reinterpret_cast<int*>(c.state + l.place);
  a.index = reinterpret_cast<int*>(c.state + l.index);
  a.label = reinterpret_cast<int*>(c.state + l.label);
  a.count = reinterpret_cast<int*>(c.state + l.count);
  a.seg = reinterpret_cast<float2*>(c.work + l.seg);
  a.target = reinterpret_cast<float*>(c.work + l.target);
  a.part = reinterpret_cast<float*>(c.work + l.part);
  a.loss = c.loss;
  a.up = c.up;
  a.up_stride = c.up_stride;
  a.dx = c.dx;
  a.dw = c.dw;
  return a;
}

template <int R>
int forward(const FewCall& c) {
  const Few a = few_of(c);
  int rc = launch("linear_cross_entropy (few: pack)", few_pack_kernel<R>, dim3((unsigned)((R * a.dp + 2 * kThreads - 1) / (2 * kThreads))), kThreads, 0, c.st, a);
  const int smem = R * a.dp * 4;
  if (!rc) rc = ensure_smem_attr((const void*)few_scores_kernel<R>, kMost * (int)kMostDim * 4);
  if (!rc) rc = launch("linear_cross_entropy (few: scores)", few_scores_kernel<R>, dim3(a.ctas), kScoreThreads, smem, c.st, a);
  if (!rc) rc = launch("linear_cross_entropy (few: join)", few_join_kernel<R>, dim3(1), 32 * R, 0, c.st, a);
  return rc;
}

template <int R>
int backward(const FewCall& c) {
  const Few a = few_of(c);
  const int columns = std::min(1024, a.dp), blocks = (a.dp + 1023) / 1024;
  int T = 8;
  while (4 * T < columns) T *= 2;
  // two CTAs an SM in all, each with a run of words
  const int runs = std::max(1, std::min(few_parts() / blocks, (a.V + 63) / 64)), words = (a.V + runs - 1) / runs;
  const dim3 grid((unsigned)((a.V + words - 1) / words), (unsigned)blocks);
  int rc = MB_OK;
  if (a.dx && a.N > 0) {
    rc = launch("linear_cross_entropy (few: dx)", few_grads_kernel<R, true>, grid, kThreads, 0, c.st, a, T, words);
    if (!rc)
      rc = launch("linear_cross_entropy (few: dx join)", few_dx_kernel<R>, dim3((unsigned)a.N, (unsigned)((a.d + 31) / 32)),
                  256, 0, c.st, a, (int)grid.x);
  }
  if (a.dw && !rc)
    rc = launch("linear_cross_entropy (few: dw)", few_grads_kernel<R, false>, grid, kThreads, 0, c.st, a, T, words);
  return rc;
}

}  // namespace

bool few_tokens(int64_t N, int64_t d, int dtype) { return dtype == MB_F32 && N <= kMost && d <= kMostDim; }

void few_sizes(int64_t N, int64_t V, int64_t d, int64_t* state, int64_t* forward_bytes, int64_t* backward_bytes) {
  const Layout l = layout_of(N, V, d);
  *state = l.state;
  *forward_bytes = l.forward;
  *backward_bytes = l.backward;
}

int few_forward(const FewCall& c) { return few_rows(c.N) == 8 ? forward<8>(c) : forward<kMost>(c); }
int few_backward(const FewCall& c) { return few_rows(c.N) == 8 ? backward<8>(c) : backward<kMost>(c); }

}  // namespace mb
