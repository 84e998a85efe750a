// Softmax cross entropy of a linear head over a large vocabulary, without its logits.
//
//   s = x W^T (x [N, d], W [V, d]),  loss_n = log sum_v exp(s_nv) - s_n,t(n)
//   G_nv = g_n (exp(s_nv) / sum - [v = t(n)]),  dx = G W,  dW = G^T x
// (g_n: the gradient that arrives at loss_n.)  Tokens whose label is `ignore_index` are left out of all
// of it: the rows that have a loss are packed together first, so they cost no arithmetic, and a NaN
// or an infinity in a padded row reaches nothing.
//
// Everything that is a product runs on the tensor cores of CTA pairs (tcgen05 cta_group::2, tiles of
// 256 x 256, operands by TMA, fp32 sums in TMEM):
//   scores   a tile of s per step.  For the loss alone a thread owns a row and keeps its running maximum and sum
//            of exponentials across all vocabulary tiles that its pair walks; the logits are never written.
//   product  dx += G W and dW += G^T x.  W, x and (for dW) G are read with the summed dimension along the
//            rows (MN-major operands), so nothing is transposed.
// Two ways to the gradients:
//   at once  (mean and sum; bf16, fp32) the scores leave E = exp(s - s_t) for a run of rows, 0.5 GB at a time, with
//            the rows' sums L; G = E / L - [v = t], where the label's place is patched, dx's rows are divided
//            at the end and dW sums E times x / L.  6 N V d flops.
//   again    (per-token gradients, which arrive later; fp16, whose range is too small for E) the forward pass
//            keeps each row's maximum and sum, the backward pass computes the scores once more and leaves G for a
//            piece of the vocabulary and a run of rows, 0.25 GB at a time.  8 N V d flops.
// Without the pieces the logits of 131072 tokens and 32000 words would be 8.4 GB in bf16, 16.8 in fp32.
//
// The tensor cores bound it: 32768 x 768 x 32000 in bf16 takes 3.9 ms for 4.83 TFLOP (1230 TFLOP/s, 74 % of the
// measured burst rate; scores 1140 to 1180, products 1360), and 4.5 ms when it runs without a pause, where the power cap
// sets the clock (the three bare library products of these shapes take 4.0 ms then).  Tensor pipe 69 % in the scores,
// 81 % in the products; shared memory, which the operands fill and empty once for each use, is what is nearest
// to its limit beside it.  0.5 GB of E at a time against 0.25 and 1: 3924, 4175 and 3844 us.
//
// Types.  16-bit operands enter as they are.  At once: E is rounded to bf16 once, x / L once; again: G once
// (2^-9 or 2^-12, what the last rounding of dx and dW makes as well).  There G is kept between -1 and 1 (times 2^15 in
// fp16, whose smallest normal number is 2^-14: a probability keeps its bits down to 2^-29), and what g_n has beyond
// is multiplied in at the end.  fp32 operands are split into three bf16 parts each (24 bits), and the six products
// of parts that matter are summed, the small ones first: the rate of these is a sixth, still three times plain fp32's.
// 16 fp32 tokens or less are bound by W's bytes instead and go to vocab_few.cu.
//
// Every wait is bounded; a CTA whose wait runs out counts itself (motif_b200_wait_timeouts), lets what
// it issued land, and leaves NaN in the tiles that it owes.
#include <algorithm>
#include <type_traits>

#include "common.cuh"
#include "pair.cuh"
#include "vocab_few.cuh"

namespace mb {

__device__ unsigned int g_vocab_wait_timeouts = 0;

namespace {

constexpr int kTile = 256;               // rows and columns of a pair's tile
constexpr int kBK = 64;                  // summed elements of a stage
constexpr int kOperand = 128 * kBK * 2;  // bytes of one operand's stage in one CTA: 128 rows or columns
constexpr int kStage = 2 * kOperand;
constexpr int kStages = 6;
constexpr int kEnders = 8;               // warps of the tile's end: two for each quarter of the TMEM lanes
constexpr int kThreads = 64 + 32 * kEnders;  // a copying warp, an issuing warp, and those
constexpr int kEnd = kEnders * 4096;     // a buffer for each
constexpr int kSmem = kStages * kStage + kEnd + 256 + 1024;
constexpr uint32_t kWait = 1u << 22;
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kHalfScale = 32768.0f;   // of G in fp16

// Which parts of the two operands a step multiplies: one part, or the six products of three parts whose
// size is 2^-16 of the whole and more, the small ones first (each sum then rounds at its own size).
template <int P> struct Parts;
template <> struct Parts<1> {
  static constexpr int n = 1;
  __device__ static int a(int) { return 0; }
  __device__ static int b(int) { return 0; }
};
template <> struct Parts<3> {
  static constexpr int n = 6;
  __device__ static int a(int i) { return (0x201100 >> (4 * (5 - i))) & 15; }
  __device__ static int b(int i) { return (0x021010 >> (4 * (5 - i))) & 15; }
};
// The type of operands in shared memory: 16-bit tensors' own, bf16 for the parts of fp32.
template <typename T> using Op = typename std::conditional<std::is_same<T, float>::value, __nv_bfloat16, T>::type;
template <typename T> constexpr int kParts = std::is_same<T, float>::value ? 3 : 1;

struct RowStat {
  float top, inv;  // the largest logit; 1 / sum of exp(s - top)
};

// ------------------------------------------------------------------------------- the pair's pipeline
struct Smem {
  unsigned char* ring;
  unsigned char* end;
  uint64_t *full, *empty, *tfull, *tempty, *mdone;
  uint32_t* tmem;
};
__device__ __forceinline__ Smem carve(unsigned char* raw) {
  Smem s;
  s.ring = raw + ((1024u - (smem_u32(raw) & 1023u)) & 1023u);
  s.end = s.ring + kStages * kStage;
  s.full = reinterpret_cast<uint64_t*>(s.end + kEnd);
  s.empty = s.full + kStages;
  s.tfull = s.empty + kStages;
  s.tempty = s.tfull + 2;
  s.mdone = s.tempty + 2;
  s.tmem = reinterpret_cast<uint32_t*>(s.mdone + 1);
  return s;
}
// Waits for the kernel before this one in the stream (these kernels begin while it ends).
__device__ __forceinline__ void wait_for_previous() { asm volatile("griddepcontrol.wait;\n" ::: "memory"); }

__device__ __forceinline__ uint32_t pair_begin(const Smem& s) {
  allow_dependent_launch();
  if (threadIdx.x < 32) tmem_alloc_pair(s.tmem, 512);
  if (threadIdx.x == 32) {
    for (int i = 0; i < kStages; ++i) {
      mbar_init(&s.full[i], 1);
      mbar_init(&s.empty[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&s.tfull[i], 1);
      mbar_init(&s.tempty[i], 2 * kEnders);  // both CTAs' warps
    }
    mbar_init(s.mdone, 1);
    mbar_init_fence();
  }
  tc_fence_before();
  __syncthreads();
  cluster_sync2();  // both CTAs' barriers exist before a copy or an arrival crosses the pair
  tc_fence_after();
  wait_for_previous();
  return *s.tmem;
}
__device__ __forceinline__ void pair_end(uint32_t tmem) {
  tc_fence_before();
  __syncthreads();
  cluster_sync2();  // every MMA, copy and arrival of the pair is done
  if (threadIdx.x < 32) {
    tc_fence_after();
    tmem_dealloc_pair(tmem, 512);
  }
}

// The copying thread: `it` counts stages over the kernel's life.  Returns the stage's memory, or null
// when the wait for it ran out.  `bytes`: of both CTAs' copies.
__device__ __forceinline__ unsigned char* stage_begin(const Smem& s, int it, bool leader, uint32_t bytes, uint32_t& bar) {
  const int st = it % kStages;
  if (!mbar_wait_bounded(&s.empty[st], (uint32_t)(((it / kStages) & 1) ^ 1), kWait)) return nullptr;
  bar = map_rank(smem_u32(&s.full[st]), 0);
  if (leader) mbar_arrive_expect_tx(&s.full[st], bytes);
  return s.ring + st * kStage;
}
// A left operand whose last tile is not full: boxes of 32 rows, as many as hold rows of it.  (What else lies
// in the stage reaches only rows of the sums that nobody reads.)
__device__ __forceinline__ int boxes_of(int rows, uint32_t rank) { return min(max((rows - 128 * (int)rank + 31) / 32, 0), 4); }
__device__ __forceinline__ void load_rows(unsigned char* st, const CUtensorMap* whole, const CUtensorMap* box, int boxes, int x,
                                          int y, uint32_t bar) {
  if (boxes == 4) {
    tma_load_2d_pair(st, whole, x, y, bar);
  } else {
    for (int i = 0; i < boxes; ++i) tma_load_2d_pair(st + i * 4096, box, x, y + 32 * i, bar);
  }
}
__device__ __forceinline__ void copies_failed(const Smem& s, int it, bool leader) {
  atomicAdd(&g_vocab_wait_timeouts, 1u);
  if (leader)  // what was issued lands before the CTA leaves
    for (int u = max(0, it - kStages); u < it; ++u)
      mbar_wait_bounded(&s.full[u % kStages], (uint32_t)((u / kStages) & 1), kWait);
}

// The leader's issuing thread: one tile's MMAs over `steps` stages.  MN-major operands keep 64 rows of
// the summed dimension for each block of 64 rows or columns: 2 KB further for 16 of them, 8 KB for the
// next block.
template <bool A_MN, bool B_MN>
__device__ __forceinline__ bool issue_tile(const Smem& s, uint32_t d, uint32_t idesc, int steps, int& it) {
  for (int i = 0; i < steps; ++i, ++it) {
    const int st = it % kStages;
    if (!mbar_wait_bounded(&s.full[st], (uint32_t)((it / kStages) & 1), kWait)) return false;
    tc_fence_after();
    const uint32_t a = smem_u32(s.ring + st * kStage), b = a + kOperand;
#pragma unroll
    for (int k = 0; k < kBK / 16; ++k)
      umma_pair(d, A_MN ? umma_desc_sw128(a + k * 2048, 8192, 1024) : umma_desc_sw128(a + k * 32, 16, 1024),
                B_MN ? umma_desc_sw128(b + k * 2048, 8192, 1024) : umma_desc_sw128(b + k * 32, 16, 1024), idesc,
                (i > 0 || k > 0) ? 1u : 0u);
    const uint32_t e = smem_u32(&s.empty[st]);
    umma_commit_pair(e);
    umma_commit_pair(map_rank(e, 1));
  }
  return true;
}
// BUFS: tiles of TMEM that take turns.
template <int BUFS>
__device__ __forceinline__ bool tile_free(const Smem& s, int done) {
  const bool ok = mbar_wait_bounded(&s.tempty[done % BUFS], (uint32_t)(((done / BUFS) & 1) ^ 1), kWait);
  tc_fence_after();
  return ok;
}
template <int BUFS>
__device__ __forceinline__ void tile_issued(const Smem& s, int done) {
  const uint32_t f = smem_u32(&s.tfull[done % BUFS]);
  umma_commit_pair(f);
  umma_commit_pair(map_rank(f, 1));
}
__device__ __forceinline__ void issue_end(const Smem& s, bool failed) {
  umma_commit_pair(smem_u32(s.mdone));  // every MMA issued, after a failure too
  if (!mbar_wait_bounded(s.mdone, 0, kWait) || failed) atomicAdd(&g_vocab_wait_timeouts, 1u);
}
// A warp of the tile's end: the tile's sums are there (false: never; `lost` then stays set).
template <int BUFS>
__device__ __forceinline__ void tile_ready(const Smem& s, int done, bool& lost) {
  if (lost) return;
  const bool ok = mbar_wait_bounded(&s.tfull[done % BUFS], (uint32_t)((done / BUFS) & 1), kWait);
  if (__any_sync(0xffffffffu, !ok)) {
    lost = true;
    if ((threadIdx.x & 31) == 0) atomicAdd(&g_vocab_wait_timeouts, 1u);
  }
  tc_fence_after();
}
template <int BUFS>
__device__ __forceinline__ void tile_read(const Smem& s, int done, bool lost, bool leader) {
  tc_fence_before();
  __syncwarp();
  if ((threadIdx.x & 31) == 0 && !lost) {
    if (leader)
      mbar_arrive(&s.tempty[done % BUFS]);
    else
      mbar_arrive_remote(map_rank(smem_u32(&s.tempty[done % BUFS]), 0));
  }
}
// 32 columns of this thread's row; NaN where the tile never came.
__device__ __forceinline__ void read32(uint32_t taddr, bool lost, uint32_t (&r)[32]) {
  if (!lost) {
    tmem_ld32(taddr, r);
    return;
  }
#pragma unroll
  for (int i = 0; i < 32; ++i) r[i] = 0x7fffffffu;
}
__device__ __forceinline__ void read32_wait(bool lost, uint32_t (&r)[32]) {
  if (!lost) tmem_wait_ld(r);
}

// fp32: a sum leaves the tensor cores every 512 terms, since they cut each partial sum off at 24 bits; what has left
// adds up in the other half of the TMEM (dx of 512 tokens, 1024 features and 32000 words: error 4.4e-6 with 3556 terms
// at a time, 6.8e-7; a logit of 16384 positive products: 6.8e-5 of it all at once, 4.6e-7).
constexpr int kFlush = 8;  // stages
__device__ __forceinline__ void tmem_st32(uint32_t taddr, const float (&v)[32]) {
  const uint32_t* r = reinterpret_cast<const uint32_t*>(v);
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32};\n" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
      "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]),
      "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]),
      "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31])
      : "memory");
}

// A warp of the tile's end: a part of the sum that is not its last, for the columns first, first + step, .. < end (32 at
// a time) of the warp's lanes.  `more`: parts have left before.
__device__ __forceinline__ void keep_part(const Smem& s, int done, bool& lost, bool leader, uint32_t lanes, int first, int end,
                                          int step, bool more) {
  tile_ready<1>(s, done, lost);
#pragma unroll 1
  for (int col = first; col < end; col += step) {
    uint32_t r[32], o[32];
    read32(lanes + col, lost, r);
    if (more) read32(lanes + kTile + col, lost, o);
    read32_wait(lost, r);
    if (more) read32_wait(lost, o);
    float v[32];
#pragma unroll
    for (int i = 0; i < 32; ++i) v[i] = __uint_as_float(r[i]) + (more ? __uint_as_float(o[i]) : 0.f);
    if (!lost) tmem_st32(lanes + kTile + col, v);
  }
  asm volatile("tcgen05.wait::st.sync.aligned;\n" ::: "memory");
  tile_read<1>(s, done, lost, leader);
}
// 32 columns of the last part with what has left before.
__device__ __forceinline__ void add_parts(uint32_t lanes, int col, bool lost, uint32_t (&r)[32]) {
  uint32_t o[32];
  read32(lanes + kTile + col, lost, o);
  read32_wait(lost, o);
#pragma unroll
  for (int i = 0; i < 32; ++i) r[i] = __float_as_uint(__uint_as_float(r[i]) + __uint_as_float(o[i]));
}

// ------------------------------------------------------------------------------- packing
struct PackArgs {
  const void* x;           // [N, d], rows xs apart
  const int64_t* labels;   // [N]
  int64_t N, xs, ignore;
  int V, d, dp;            // dp: row length of the packed operand
  int64_t rows;            // packed rows of a part (N rounded up to a tile)
  void* packed;            // [parts][rows][dp]
  int* count;              // tokens that have a loss
  int* ticket;             // zeroed here for the joining kernel
  const int* group;        // tokens with a loss in each run of 256, or null: the labels are read instead
  int* label;              // [rows]: of the packed rows, -1 where it is not one of V
  int* index;              // [rows]: of the packed rows, where they came from
  int* place;              // [N]: the packed row of a token, -1 without one
  float* loss;             // per-token losses: 0 is written for tokens without one (null: no such output)
  const void* w;           // with `ref`: [V, d], rows ws apart
  int64_t ws;
  float* ref;              // [rows]: the label's logit of the packed rows, or null
  int* flags;              // [runs]: zeroed here for the scores
  int runs;
  int tokens;              // of a CTA, a divisor of 256
};

__global__ void __launch_bounds__(256) group_count_kernel(const int64_t* __restrict__ labels, int64_t N, int64_t ignore,
                                                          int* __restrict__ group) {
  allow_dependent_launch();
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int n = __syncthreads_count(i < N && labels[i] != ignore);
  if (threadIdx.x == 0) group[blockIdx.x] = n;
}

// x as the sum of three bf16 numbers (exact but for what lies below 2^-24 of x).
__device__ __forceinline__ void split3(float x, __nv_bfloat16 (&p)[3]) {
  p[0] = __float2bfloat16_rn(x);
  if (__hisinf(p[0])) {
    p[1] = p[2] = __float2bfloat16_rn(0.f);
    if (isinf(x)) return;  // an infinity stays one: its remainder would be a NaN
    p[0] = __float2bfloat16_rz(x);  // beyond bf16's largest number: from below
  }
  const float r1 = x - __bfloat162float(p[0]);
  p[1] = __float2bfloat16_rn(r1);
  p[2] = __float2bfloat16_rn(r1 - __bfloat162float(p[1]));
}
// Eight elements from column c of a row of d, zeros behind its end.
template <typename T> struct Eight {
  uint4 u[sizeof(T) / 2];
  __device__ void load(const T* src, int c, int d, bool aligned) {
    if (aligned && c + 8 <= d) {
#pragma unroll
      for (int i = 0; i < (int)sizeof(T) / 2; ++i) u[i] = reinterpret_cast<const uint4*>(src + c)[i];
    } else {
      T* e = reinterpret_cast<T*>(u);
#pragma unroll
      for (int i = 0; i < 8; ++i) e[i] = c + i < d ? src[c + i] : from_f<T>(0.f);
    }
  }
  __device__ void store(Op<T>* dst, int c, int64_t part) const {
    if constexpr (kParts<T> == 1) {
      *reinterpret_cast<uint4*>(dst + c) = u[0];
    } else {
      const float* e = reinterpret_cast<const float*>(u);
      __align__(16) __nv_bfloat16 o[3][8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        __nv_bfloat16 p[3];
        split3(e[i], p);
#pragma unroll
        for (int k = 0; k < 3; ++k) o[k][i] = p[k];
      }
#pragma unroll
      for (int k = 0; k < 3; ++k) *reinterpret_cast<uint4*>(dst + k * part + c) = *reinterpret_cast<const uint4*>(o[k]);
    }
  }
};
// One row of d elements into its parts, zeros behind it up to dp (a multiple of 8); a warp, four requests at a
// time.
template <typename T>
__device__ __forceinline__ void pack_row(const T* src, int d, Op<T>* dst, int dp, int64_t part, int lane) {
  const bool aligned = (reinterpret_cast<uintptr_t>(src) & 15) == 0;
  for (int c0 = lane * 8; c0 < dp; c0 += 1024) {
    Eight<T> v[4];
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (c0 + 256 * i < dp) v[i].load(src, c0 + 256 * i, d, aligned);
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (c0 + 256 * i < dp) v[i].store(dst, c0 + 256 * i, part);
  }
}
template <typename T>
__device__ __forceinline__ void zero_row(Op<T>* dst, int dp, int64_t part, int lane) {
  for (int p = 0; p < kParts<T>; ++p)
    for (int c = lane * 8; c < dp; c += 256) *reinterpret_cast<uint4*>(dst + p * part + c) = make_uint4(0, 0, 0, 0);
}

// Sum of the products of two rows, in fp32; a warp.
template <typename T>
__device__ __forceinline__ float dot_rows(const T* x, const T* w, int d, int lane) {
  const bool ax = (reinterpret_cast<uintptr_t>(x) & 15) == 0, aw = (reinterpret_cast<uintptr_t>(w) & 15) == 0;
  float t[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
  for (int c0 = lane * 8; c0 < d; c0 += 512) {
    Eight<T> u[2], v[2];
#pragma unroll
    for (int i = 0; i < 2; ++i)
      if (c0 + 256 * i < d) {
        u[i].load(x, c0 + 256 * i, d, ax);
        v[i].load(w, c0 + 256 * i, d, aw);
      }
#pragma unroll
    for (int i = 0; i < 2; ++i)
      if (c0 + 256 * i < d) {
        const T *p = reinterpret_cast<const T*>(u[i].u), *q = reinterpret_cast<const T*>(v[i].u);
#pragma unroll
        for (int e = 0; e < 8; ++e) t[e] = fmaf(to_f(p[e]), to_f(q[e]), t[e]);
      }
  }
  return warp_sum(((t[0] + t[1]) + (t[2] + t[3])) + ((t[4] + t[5]) + (t[6] + t[7])));
}

template <typename T>
__global__ void __launch_bounds__(256) pack_kernel(const PackArgs a) {
  __shared__ int part[8], before[8], place[256];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int64_t first = (int64_t)blockIdx.x * a.tokens, run = first / 256 * 256;
  allow_dependent_launch();
  wait_for_previous();
  const int64_t mine = run + tid;
  const int64_t label = mine < a.N ? a.labels[mine] : a.ignore;
  // tokens with a loss in the runs before this one
  int n = 0;
  if (a.group) {
    for (int64_t i = tid; i < run / 256; i += 256) n += a.group[i];
  } else {
    for (int64_t i = tid; i < run; i += 256) n += a.labels[i] != a.ignore;
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) n += __shfl_xor_sync(0xffffffffu, n, o);
  const bool live = label != a.ignore;
  const unsigned vote = __ballot_sync(0xffffffffu, live);
  if (lane == 0) {
    before[warp] = n;
    part[warp] = __popc(vote);
  }
  __syncthreads();
  int at = 0, total = 0;
  for (int w = 0; w < 8; ++w) {
    at += before[w];
    total += before[w] + part[w];
    if (w < warp) at += part[w];
  }
  at += __popc(vote & ((1u << lane) - 1u));
  place[tid] = live ? at : -1;
  if (mine >= first && mine < first + a.tokens && mine < a.N) {
    a.place[mine] = live ? at : -1;
    if (live) {
      a.label[at] = label >= 0 && label < a.V ? (int)label : -1;
      a.index[at] = (int)mine;
    } else if (a.loss) {
      a.loss[mine] = 0.f;
    }
  }
  __syncthreads();
  const T* x = reinterpret_cast<const T*>(a.x);
  Op<T>* out = reinterpret_cast<Op<T>*>(a.packed);
  const int64_t plane = a.rows * a.dp;
  for (int i = warp; i < a.tokens; i += 8) {
    const int64_t token = first + i;
    if (token >= a.N) break;
    const int to = place[token - run];
    if (to < 0) continue;
    pack_row<T>(x + token * a.xs, a.d, out + (int64_t)to * a.dp, a.dp, plane, lane);
    if (a.ref) {
      const int64_t word = a.labels[token];
      const bool known = word >= 0 && word < a.V;
      const float s = known ? dot_rows<T>(x + token * a.xs, reinterpret_cast<const T*>(a.w) + word * a.ws, a.d, lane) : 0.f;
      if (lane == 0) a.ref[to] = s;
    }
  }
  // the last CTA sees all tokens: it leaves their number, and zeros up to the end of the last 64 rows (what the
  // products sum over together)
  if (first + a.tokens >= a.N) {
    const int64_t end = min(a.rows, (int64_t)(total + kBK - 1) / kBK * kBK);
    for (int64_t r = total + warp; r < end; r += 8) zero_row<T>(out + r * a.dp, a.dp, plane, lane);
    if (tid == 0) {
      *a.count = total;
      *a.ticket = 0;
    }
    if (a.flags)
      for (int i = tid; i < a.runs; i += 256) a.flags[i] = 0;
  }
}

// The weight as an operand, where it cannot be one itself: fp32, or rows that are not 16-byte aligned.
template <typename T>
__global__ void __launch_bounds__(256) pack_weight_kernel(const T* __restrict__ w, int64_t ws, int V, int d, int dp,
                                                          int64_t rows, Op<T>* __restrict__ out) {
  allow_dependent_launch();
  wait_for_previous();
  const int lane = threadIdx.x & 31;
  const int64_t plane = rows * dp;
  for (int64_t r = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5); r < rows; r += (int64_t)gridDim.x * 8) {
    if (r < V)
      pack_row<T>(w + r * ws, d, out + r * dp, dp, plane, lane);
    else
      zero_row<T>(out + r * dp, dp, plane, lane);
  }
}

// ------------------------------------------------------------------------------- scores
// What becomes of a tile of logits:
//   kLoss   nothing but its rows' maxima and sums of exponentials
//   kAgain  G, from the rows' maxima and sums
//   kOnce   E = exp(s - s_t) (0 at the label): the gradients' exponentials before their sum is known, with that
//           sum.  s_t, the label's logit, is known before, and is near the largest one unless the loss is
//           large: exp(66) fits all types here.  A row with a larger logit raises the run's flag; its sum goes
//           on from there, and kAgain computes the run's G instead.
enum { kLoss, kAgain, kOnce };
constexpr float kFar = 66.0f;

struct ScoreArgs {
  const int* count;         // tokens with a loss
  int row0, rows;           // this call's packed rows: row0 .. row0 + rows
  int v0, nv;               // its vocabulary: v0 .. v0 + nv
  int kblocks;
  int64_t x_part, w_part;   // rows from one part of an operand to the next
  const int* label;         // [rows of the packed operand]
  float2* seg;              // kLoss, kOnce: (reference, sum) of each row of half a pair's run through a row tile
  float* target;            // kLoss, kOnce: the label's logit
  const float* ref;         // kOnce: the label's logit, known before (to a rounding or two)
  int* flag;                // kOnce: set where a logit is far above it; kAgain: works only if set (null: always)
  const RowStat* stat;      // kAgain
  const int* index;         // kAgain: packed row -> token
  const float* up;          // kAgain: per-token gradients (null: 1)
  int64_t up_stride;
  const float* scale;       // kAgain: [1] = what `up` is multiplied by (a power of two); with `up` only
  int64_t g_part;           // rows from one part of G or E to the next
};

// Pair p of np (as many as there are, or as there are tiles) walks the tiles [p T / np, (p + 1) T / np) of the
// row tiles times nt vocabulary tiles, the vocabulary fastest.  A run through one row tile has the number
// p + (row tile), which no other has.
__host__ __device__ __forceinline__ int64_t range_start(int64_t p, int64_t tiles, int64_t np) { return p * tiles / np; }
__host__ __device__ __forceinline__ int64_t range_owner(int64_t t, int64_t tiles, int64_t np) {
  return ((t + 1) * np - 1) / tiles;
}

// 16-bit operands' exponentials are 2^(s log2 e - m), one multiply-add each, with m = top log2 e rounded: what that
// rounding takes off is the same for a whole row, and is put back where the row's sum or divisor leaves.  (Left out, a
// loss is off by half a unit of m: 4e-5 for logits near 1000.)  From 2^29 on (a label masked with the type's lowest value),
// where m loses more than 32 or is not finite, neighbouring numbers are 64 apart: next to the largest logit nothing
// counts, in any base, and in base 2 the exponent s - top is exact.
constexpr float kFarTop = 536870912.0f;
__device__ __forceinline__ float lost_of(float top) {
  return fabsf(top) < kFarTop ? fmaf(top, kLog2e, -__fmul_rn(top, kLog2e)) : 0.f;
}

// LONG (fp32, more than 512 features): the sums leave the tensor cores in parts, so one tile has all of the TMEM and the
// next one waits for its end (4096 x 768 x 32000, loss 914 -> 964 us, with gradients 2905 -> 2973; the losses' error 3.7e-7 ->
// 2.0e-7, at 4096 features 2.3e-6 -> 2.3e-7).
template <typename T, int MODE, bool LONG>
__global__ void __launch_bounds__(kThreads, 1) scores_kernel(const __grid_constant__ CUtensorMap tmX,
                                                             const __grid_constant__ CUtensorMap tmX32,
                                                             const __grid_constant__ CUtensorMap tmW,
                                                             const __grid_constant__ CUtensorMap tmG,
                                                             const ScoreArgs a) {
  using O = Op<T>;
  constexpr int P = kParts<T>;
  static_assert(!LONG || P > 1, "16-bit operands' sums stay in the tensor cores");
  constexpr int kBufs = LONG ? 1 : 2, kTake = LONG ? kFlush : 1 << 30;
  extern __shared__ unsigned char raw[];
  const Smem s = carve(raw);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = cluster_rank2();
  const bool leader = rank == 0;
  if (MODE == kAgain && a.flag) {
    allow_dependent_launch();
    wait_for_previous();
    if (*a.flag == 0) return;  // both CTAs of a pair read the same
  }
  const uint32_t tmem = pair_begin(s);
  const int np = gridDim.x >> 1, pair = blockIdx.x >> 1;
  const int live = min(max(*a.count - a.row0, 0), a.rows);
  const int mt = (live + kTile - 1) / kTile, nt = (a.nv + kTile - 1) / kTile;
  const int64_t tiles = (int64_t)mt * nt;
  const int64_t walkers = min((int64_t)np, tiles);
  const int64_t t0 = pair < walkers ? range_start(pair, tiles, walkers) : 0;
  const int64_t t1 = pair < walkers ? range_start(pair + 1, tiles, walkers) : 0;

  if (warp == 0) {
    if (lane == 0) {
      int it = 0;
      bool failed = false;
      for (int64_t t = t0; t < t1 && !failed; ++t) {
        const int m = (int)(t / nt), n = (int)(t - (int64_t)m * nt);
        const int xr = a.row0 + m * kTile + 128 * (int)rank, wr = a.v0 + n * kTile + 128 * (int)rank;
        const int rows = live - m * kTile, boxes = boxes_of(rows, rank);
        const uint32_t bytes = 4096 * (boxes_of(rows, 0) + boxes_of(rows, 1)) + 2 * kOperand;
        for (int k0 = 0; k0 < a.kblocks && !failed; k0 += kTake)
        for (int p = 0; p < Parts<P>::n && !failed; ++p)
          for (int kb = k0; kb < min(a.kblocks, k0 + kTake); ++kb, ++it) {
            uint32_t bar;
            unsigned char* st = stage_begin(s, it, leader, bytes, bar);
            if (!st) {
              failed = true;
              break;
            }
            load_rows(st, &tmX, &tmX32, boxes, kb * kBK, xr + (int)(Parts<P>::a(p) * a.x_part), bar);
            tma_load_2d_pair(st + kOperand, &tmW, kb * kBK, wr + (int)(Parts<P>::b(p) * a.w_part), bar);
          }
      }
      if (failed) copies_failed(s, it, leader);
    }
    __syncwarp();
  } else if (warp == 1) {
    if (lane == 0 && leader) {
      constexpr uint32_t idesc =
          umma_idesc_f16(std::is_same<O, __nv_bfloat16>::value ? 1u : 0u, kTile, kTile, 0, 0);
      int it = 0, done = 0;
      bool failed = false;
      for (int64_t t = t0; t < t1 && !failed; ++t)
        for (int k0 = 0; k0 < a.kblocks && !failed; k0 += kTake, ++done) {
          failed = !tile_free<kBufs>(s, done) ||
                   !issue_tile<false, false>(s, tmem + (uint32_t)(done % kBufs * kTile), idesc,
                                             Parts<P>::n * min(kTake, a.kblocks - k0), it);
          if (!failed) tile_issued<kBufs>(s, done);
        }
      issue_end(s, failed);
    }
    __syncwarp();
  } else {
    const int q = warp & 3, half = (warp - 2) >> 2;  // the TMEM lanes that this warp can read; its columns
    const int in_tile = (int)rank * 128 + q * 32 + lane, c0 = half * (kTile / 2);
    unsigned char* buf = s.end + (warp - 2) * 4096;
    // what leaves is larger than the L2 and read next by another kernel: it should not push the weight out
    uint64_t policy;
    asm volatile("createpolicy.fractional.L2::evict_first.b64 %0, 1.0;\n" : "=l"(policy));
    int done = 0, m_now = -1, label = -1;
    bool lost = false, mine = false;
    float top = 0.f, sum = 0.f;  // kLoss, kOnce: of the run so far; kAgain: the row's largest logit
    float inv = 0.f, g = 0.f;    // kAgain
    // 64 columns from column c of the tile: `at` is the label's, `valid` columns are words.  64 at a time, so that
    // each of the few warps has enough independent work (32 at a time took twice as long a tile).
    auto block = [&](uint32_t (&r0)[32], uint32_t (&r1)[32], int c, int at, int valid, int row, int x, int y) {
      float z[64];
#pragma unroll
      for (int i = 0; i < 32; ++i) {
        z[i] = __uint_as_float(r0[i]);
        z[32 + i] = __uint_as_float(r1[i]);
      }
      const bool here = __any_sync(0xffffffffu, (unsigned)(at - c) < 64u);
      if constexpr (MODE != kAgain) {
        if (valid < c + 64) {
#pragma unroll
          for (int i = 0; i < 64; ++i)
            if (c + i >= valid) z[i] = -INFINITY;
        }
        if (here) {
          float own = 0.f;
#pragma unroll
          for (int i = 0; i < 64; ++i) {
            const bool it = at == c + i;
            own = it ? z[i] : own;
            if (MODE == kOnce) z[i] = it ? -INFINITY : z[i];  // its part is added when the row is settled
          }
          if ((unsigned)(at - c) < 64u) a.target[row] = own;
        }
        float t8[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          t8[j] = fmax3(z[8 * j], z[8 * j + 1], z[8 * j + 2]);
          t8[j] = fmax3(t8[j], z[8 * j + 3], z[8 * j + 4]);
          t8[j] = fmax3(t8[j], z[8 * j + 5], z[8 * j + 6]);
          t8[j] = fmaxf(t8[j], z[8 * j + 7]);
        }
        const float now = fmax3(fmax3(t8[0], t8[1], t8[2]), fmax3(t8[3], t8[4], t8[5]), fmaxf(t8[6], t8[7]));
        // (from a million on m loses bits that exponentials of 66 have no room for)
        const float reach = P == 1 && fabsf(top) >= 1048576.0f ? 0.f : kFar;
        const bool raise = MODE == kLoss ? now > top : mine && now > top + reach;  // (rows behind the last hold anything)
        if (__any_sync(0xffffffffu, raise) && raise) {
          sum *= ex2f_((top - now) * kLog2e + (P == 1 ? lost_of(now) - lost_of(top) : 0.f));  // 0 from -inf
          top = now;
          if (MODE == kOnce) *a.flag = 1;
        }
      }
      // (s - top) log2 e: for 16-bit operands as one multiply-add (`lost_of`)
      const float ref = MODE != kAgain && top == -INFINITY ? 0.f : top;  // (kOnce: the label's logit may be -inf)
      const float c1 = P == 1 && fabsf(ref) >= kFarTop ? 1.f : kLog2e, m = -ref * c1;
      const float2 c2 = make_float2(c1, c1), n2 = make_float2(-ref, -ref);
      const float2 m2 = make_float2(m, m), i2 = make_float2(inv, inv);
      float2 acc[4] = {};
#pragma unroll
      for (int i = 0; i < 64; i += 2) {
        const float2 v = make_float2(z[i], z[i + 1]);
        const float2 e = P == 1 ? ffma2(v, c2, m2) : fmul2(fadd2(v, n2), c2);
        float2 w = make_float2(ex2f_(e.x), ex2f_(e.y));
        if constexpr (MODE == kAgain)
          w = fmul2(w, i2);
        else
          acc[i / 2 % 4] = fadd2(acc[i / 2 % 4], w);
        z[i] = w.x;
        z[i + 1] = w.y;
      }
      if constexpr (MODE != kAgain) {
        const float2 all = fadd2(fadd2(acc[0], acc[1]), fadd2(acc[2], acc[3]));
        sum += all.x + all.y;
      } else if (here) {
#pragma unroll
        for (int i = 0; i < 64; ++i)
          if (at == c + i) z[i] -= g;
      }
      if constexpr (MODE != kLoss) {
        if (!mine || valid < c + 64) {
#pragma unroll
          for (int i = 0; i < 64; ++i)
            if (!mine || c + i >= valid) z[i] = 0.f;
        }
#pragma unroll
        for (int p = 0; p < P; ++p) {
          uint32_t w[32];
#pragma unroll
          for (int i = 0; i < 32; ++i) {
            w[i] = pack2<O>(z[2 * i], z[2 * i + 1]);
            if (p + 1 < P) {
              const float2 back = round2<O>(z[2 * i], z[2 * i + 1]);
              z[2 * i] -= back.x;
              z[2 * i + 1] -= back.y;
            }
          }
          // 32 rows x 128 bytes in the 128-byte swizzle of the tensor map, once the block before has left
          if (lane == 0) asm volatile("cp.async.bulk.wait_group.read 0;\n" ::: "memory");
          __syncwarp();
#pragma unroll
          for (int u = 0; u < 8; ++u)
            *reinterpret_cast<uint4*>(buf + lane * 128 + ((u ^ (lane & 7)) << 4)) =
                make_uint4(w[4 * u], w[4 * u + 1], w[4 * u + 2], w[4 * u + 3]);
          fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0) {
            asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.bulk_group.L2::cache_hint [%0, {%1, %2}], [%3], %4;\n" ::"l"(
                             reinterpret_cast<uint64_t>(&tmG)),
                         "r"(x + c), "r"((int)(p * a.g_part) + y), "r"(smem_u32(buf)), "l"(policy)
                         : "memory");
            asm volatile("cp.async.bulk.commit_group;\n" ::: "memory");
          }
        }
      }
    };
    auto run_ends = [&] {
      a.seg[((int64_t)(pair + m_now) * 2 + half) * kTile + in_tile] =
          make_float2(top, P == 1 ? sum * ex2f_(-lost_of(top)) : sum);
    };
    for (int64_t t = t0; t < t1; ++t, ++done) {
      const int m = (int)(t / nt), n = (int)(t - (int64_t)m * nt);
      const int row = a.row0 + m * kTile + in_tile;
      if (m != m_now) {
        if (MODE != kAgain && m_now >= 0) run_ends();
        m_now = m;
        mine = m * kTile + in_tile < live;
        label = mine ? a.label[row] : -1;
        sum = 0.f;
        if constexpr (MODE == kLoss) top = -INFINITY;
        if constexpr (MODE == kOnce) top = mine ? a.ref[row] : 0.f;
        if constexpr (MODE == kAgain) {
          if (mine) {
            const RowStat st = a.stat[row];
            g = a.up ? a.up[a.index[row] * a.up_stride] * a.scale[1] : 1.0f;
            if constexpr (std::is_same<T, __half>::value) g *= kHalfScale;
            top = st.top;
            inv = P == 1 ? st.inv * g * ex2f_(-lost_of(top)) : st.inv * g;
          }
        }
      }
      const int at = label - (a.v0 + n * kTile);  // the label's column, if it is in this tile
      const int valid = a.nv - n * kTile;         // columns of the tile that are words
      const int x = n * kTile, y = m * kTile + (int)rank * 128 + q * 32;
      const uint32_t lanes = tmem + ((uint32_t)(q * 32) << 16);
      if constexpr (LONG)
        for (int k0 = 0; k0 + kTake < a.kblocks; k0 += kTake, ++done)
          keep_part(s, done, lost, leader, lanes, c0, c0 + kTile / 2, 32, k0 > 0);
      const uint32_t taddr = lanes + (uint32_t)(done % kBufs * kTile);
      tile_ready<kBufs>(s, done, lost);
#pragma unroll 1
      for (int h = 0; h < 2; ++h) {
        uint32_t r0[32], r1[32];
        read32(taddr + c0 + 64 * h, lost, r0);
        read32(taddr + c0 + 64 * h + 32, lost, r1);
        read32_wait(lost, r0);
        read32_wait(lost, r1);
        if constexpr (LONG) {  // (there has been a part before: more features than one holds)
          add_parts(lanes, c0 + 64 * h, lost, r0);
          add_parts(lanes, c0 + 64 * h + 32, lost, r1);
        }
        if (h == 1) tile_read<kBufs>(s, done, lost, leader);  // the tile is in registers: the next one may come
        block(r0, r1, c0 + 64 * h, at, valid, row, x, y);
      }
    }
    if constexpr (MODE != kLoss) {
      if (lane == 0) asm volatile("cp.async.bulk.wait_group 0;\n" ::: "memory");
      __syncwarp();
    }
    if (MODE != kAgain && m_now >= 0) run_ends();
  }
  pair_end(tmem);
}

// ------------------------------------------------------------------------------- the loss
struct JoinArgs {
  const int* count;
  int* ticket;
  const float2* seg;
  const float* target;
  const int* label;
  const int* index;
  RowStat* stat;
  float* loss;       // [N] or one value
  double* partial;   // one a CTA
  int nt, np;        // of the scores
  int reduction;     // 0 none, 1 mean, 2 sum
};

// The sum of a CTA's losses to partial[cta]; the last CTA of all adds those, in one order whoever it is.
template <int N>
__device__ __forceinline__ void add_losses(double* sums, int cta, int ctas, double* partial, int* ticket, bool mean, int live,
                                           float* out) {
  __shared__ int last;
  __shared__ double warps[8];
  double loss = 0.0;
  if (threadIdx.x == 0) {
    for (int i = 0; i < N; ++i) loss += sums[i];
    partial[cta] = loss;
    __threadfence();
    last = atomicAdd(ticket, 1) == ctas - 1;
  }
  __syncthreads();
  if (!last) return;
  __threadfence();
  loss = 0.0;
  for (int i = threadIdx.x; i < ctas; i += 256) loss += __ldcg(partial + i);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) loss += __shfl_xor_sync(0xffffffffu, loss, o);
  if ((threadIdx.x & 31) == 0) warps[threadIdx.x >> 5] = loss;
  __syncthreads();
  if (threadIdx.x == 0) {
    loss = 0.0;
    for (int i = 0; i < 8; ++i) loss += warps[i];
    *out = (float)(mean ? loss / (double)live : loss);  // no tokens: 0 / 0, as it is
  }
}

constexpr int kJoinRows = 8;  // of a CTA: a warp a row

// (reference, sum) pairs of a row's runs s0 .. s1, joined over a warp: exponentials relative to the largest reference.
__device__ __forceinline__ void join_runs(const float2* seg, int s0, int s1, int in_tile, float& top, float& sum) {
  const int lane = threadIdx.x & 31;
#pragma unroll 4
  for (int i = s0 + lane; i < s1; i += 32) {
    const float2 v = seg[(int64_t)i * kTile + in_tile];
    const float now = fmaxf(top, v.x), ref = now == -INFINITY ? 0.f : now;
    sum = sum * ex2f_((top - ref) * kLog2e) + v.y * ex2f_((v.x - ref) * kLog2e);
    top = now;
  }
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {  // the two sides of an exchange add in the same order
    const float t2 = __shfl_xor_sync(0xffffffffu, top, o), s2 = __shfl_xor_sync(0xffffffffu, sum, o);
    const float now = fmaxf(top, t2), ref = now == -INFINITY ? 0.f : now;
    const float mine = sum * ex2f_((top - ref) * kLog2e), other = s2 * ex2f_((t2 - ref) * kLog2e);
    sum = (lane & o) ? other + mine : mine + other;
    top = now;
  }
}

__global__ void __launch_bounds__(32 * kJoinRows) join_kernel(const JoinArgs a) {
  __shared__ double sums[kJoinRows];
  allow_dependent_launch();
  wait_for_previous();
  const int live = *a.count, r = threadIdx.x >> 5, j = threadIdx.x & 31, row = blockIdx.x * kJoinRows + r;
  const int mt = (live + kTile - 1) / kTile, ctas = max((live + kJoinRows - 1) / kJoinRows, 1);
  if (blockIdx.x >= ctas) return;  // the first CTA is there for a call without tokens, too
  float top = -INFINITY, sum = 0.f;
  if (row < live) {
    const int m = row / kTile;
    const int64_t tiles = (int64_t)mt * a.nt, walkers = min((int64_t)a.np, tiles);
    const int s0 = 2 * ((int)range_owner((int64_t)m * a.nt, tiles, walkers) + m);
    const int s1 = 2 * ((int)range_owner((int64_t)(m + 1) * a.nt - 1, tiles, walkers) + m) + 2;
    join_runs(a.seg, s0, s1, row % kTile, top, sum);
  }
  double loss = 0.0;
  if (row < live && j == 0) {
    const float ref = top == -INFINITY ? 0.f : top;
    const bool known = a.label[row] >= 0;
    const float nan = __int_as_float(0x7fffffff);
    RowStat st;
    st.top = ref;
    st.inv = known ? 1.0f / sum : nan;  // a label that is no word: NaN, in the gradients too
    a.stat[row] = st;
    const float one = known ? (ref - a.target[row]) + logf(sum) : nan;
    if (a.reduction == 0) a.loss[a.index[row]] = one;
    loss = one;
  }
  if (a.reduction == 0) return;
  if (j == 0) sums[r] = loss;
  __syncthreads();
  add_losses<kJoinRows>(sums, blockIdx.x, ctas, a.partial, a.ticket, a.reduction == 1, live, a.loss);
}

// kOnce's rows: their loss, and what turns exponentials into gradients.  G L = E - L [v = t] with L the whole
// sum, so the label's place gets -(the sum of the others), which loses nothing however near to 1 its
// probability is; dx's rows are divided by L at the end, and dW sums E times x / L.  The label's part of L comes
// from the tiles, like the others' (the tensor cores cut sums off, which moves large logits by 4e-7 of
// themselves; between logits of one size it cancels).  In bf16 the divisor also takes back the rounding of the
// label's place, the largest part of G: without that, the error of dx was 1.4 times as large.  (The row's other words, which
// are as much together but less each, carry it instead, on top of the rounding of their own.)  A warp a row.
struct SettleArgs {
  const int* count;
  int* ticket;
  const float2* seg;
  const float* ref;
  const float* target;
  const int* label;
  RowStat* stat;
  const int* flag;       // the run's exponentials are G (kAgain computes them next): nothing is left to divide
  float* row_scale;      // [rows of the run]
  float* loss;
  double* partial;
  int nt, np, mean;
  int row0, rows;        // the run
  const void* x;         // [parts][x_part][dp]
  int64_t x_part;
  void* weighed;         // [parts][w_part][dp]: x / L of the run's rows, zeros up to the end of 64
  int64_t w_part;
  int dp;
  void* e;               // [parts][w_part][ld]
  int64_t ld;
};
constexpr int kSettleRows = 8;

template <typename T>
__global__ void __launch_bounds__(32 * kSettleRows) settle_kernel(const SettleArgs a) {
  using O = Op<T>;
  constexpr int P = kParts<T>;
  __shared__ double sums[kSettleRows];
  allow_dependent_launch();
  wait_for_previous();
  const int all = *a.count, live = min(max(all - a.row0, 0), a.rows), flagged = *a.flag;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, r = blockIdx.x * kSettleRows + warp, row = a.row0 + r;
  const int cta = a.row0 / kSettleRows + blockIdx.x, ctas = max((all + kSettleRows - 1) / kSettleRows, 1);
  O* weighed = reinterpret_cast<O*>(a.weighed) + (int64_t)r * a.dp;
  const int64_t w_plane = a.w_part * a.dp, x_plane = a.x_part * a.dp;
  double loss = 0.0;
  if (r < live) {
    const int mt = (live + kTile - 1) / kTile, m = r / kTile, in_tile = r % kTile;
    const int64_t tiles = (int64_t)mt * a.nt, walkers = min((int64_t)a.np, tiles);
    const int s0 = 2 * ((int)range_owner((int64_t)m * a.nt, tiles, walkers) + m);
    const int s1 = 2 * ((int)range_owner((int64_t)(m + 1) * a.nt - 1, tiles, walkers) + m) + 2;
    const float ref = a.ref[row];
    float top = ref, sum = 0.f;
    join_runs(a.seg, s0, s1, in_tile, top, sum);
    const int label = a.label[row];
    const float nan = __int_as_float(0x7fffffff);
    const float target = label >= 0 ? a.target[row] : nan;  // a label that is no word: NaN, in the gradients too
    const float own = ex2f_((target - top) * kLog2e);       // 1 to a rounding but for far logits
    const float inv = 1.0f / (sum + own);
    loss = own > 0.5f ? log1pf(sum / own) : (top - target) + logf(sum + own);
    float scale = flagged && label >= 0 ? 1.0f : inv;
    float others = sum;  // as E holds them
    if (P == 1 && !flagged) {
      const float lost = lost_of(ref);
      others *= ex2f_(lost);
      scale *= ex2f_(-lost);
      if (sum > 1e-30f && sum < 1e30f) scale *= others / to_f(from_f<O>(others));
    }
    if (lane == 0) {
      RowStat st;
      st.top = top;
      st.inv = inv;
      a.stat[row] = st;
      a.row_scale[r] = scale;
      if (!flagged && label >= 0) {
        O* e = reinterpret_cast<O*>(a.e) + (int64_t)r * a.ld + label;
        if constexpr (P == 1) {
          *e = from_f<O>(-others);
        } else {
          __nv_bfloat16 p[3];
          split3(-others, p);
          for (int i = 0; i < 3; ++i) e[i * a.w_part * a.ld] = p[i];
        }
      }
    }
    const O* x = reinterpret_cast<const O*>(a.x) + (int64_t)row * a.dp;
    for (int c = lane * 8; c < a.dp; c += 256) {
      Eight<T> v;
      T* o = reinterpret_cast<T*>(v.u);
      float f[8];
      uint4 u[P];
#pragma unroll
      for (int p = 0; p < P; ++p) u[p] = *reinterpret_cast<const uint4*>(x + p * x_plane + c);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        f[i] = to_f(reinterpret_cast<const O*>(&u[P - 1])[i]);
        for (int p = P - 2; p >= 0; --p) f[i] += to_f(reinterpret_cast<const O*>(&u[p])[i]);
        o[i] = from_f<T>(f[i] * scale);
      }
      v.store(weighed, c, w_plane);
    }
  } else if (r < (live + kBK - 1) / kBK * kBK) {
    zero_row<T>(weighed, a.dp, w_plane, lane);
  }
  if (cta >= ctas || (r - warp >= live && cta > 0)) return;  // (the first CTA is there for a call without tokens, too)
  if (lane == 0) sums[warp] = loss;
  __syncthreads();
  add_losses<kSettleRows>(sums, cta, ctas, a.partial, a.ticket, a.mean, all, a.loss);
}

// dst = src * *scale, for up to two arrays: the gradients of a loss that another one follows.  In place there is nothing
// to do where that is 1.
template <typename T>
__global__ void __launch_bounds__(256) scale_out_kernel(const T* a, T* ao, int64_t na, const T* b, T* bo, int64_t nb,
                                                        const float* __restrict__ scale) {
  const float s = *scale;
  const int64_t step = (int64_t)gridDim.x * 256, first = (int64_t)blockIdx.x * 256 + threadIdx.x;
  constexpr int E = 16 / (int)sizeof(T);
#pragma unroll
  for (int which = 0; which < 2; ++which) {
    const T* src = which ? b : a;
    T* dst = which ? bo : ao;
    const int64_t n = which ? nb : na, vecs = n / E;
    if (src == dst && s == 1.0f) continue;
#pragma unroll 4
    for (int64_t i = first; i < vecs; i += step) {
      const uint4 u = reinterpret_cast<const uint4*>(src)[i];
      const T* e = reinterpret_cast<const T*>(&u);
      __align__(16) T o[E];
#pragma unroll
      for (int k = 0; k < E; ++k) o[k] = from_f<T>(to_f(e[k]) * s);
      reinterpret_cast<uint4*>(dst)[i] = *reinterpret_cast<const uint4*>(o);
    }
    for (int64_t i = vecs * E + first; i < n; i += step) dst[i] = from_f<T>(to_f(src[i]) * s);
  }
}

// For per-token gradients.  scale[0]: what dx and dW are multiplied by at the end; scale[1]: what the
// per-token gradients are multiplied by before (a power of two that brings the largest to 1 / 2 .. 1).
__global__ void __launch_bounds__(1024) scale_kernel(const float* __restrict__ up, int64_t up_stride, int64_t N,
                                                     const int* __restrict__ place, float* __restrict__ scale) {
  __shared__ float tops[32];
  allow_dependent_launch();
  wait_for_previous();
  float top = 0.f;
#pragma unroll 4
  for (int64_t i = threadIdx.x; i < N; i += 1024)
    if (place[i] >= 0) top = fmaxf(top, fabsf(up[i * up_stride]));
  top = warp_max(top);
  if ((threadIdx.x & 31) == 0) tops[threadIdx.x >> 5] = top;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int i = 1; i < 32; ++i) top = fmaxf(top, tops[i]);
    int e = 0;
    if (top > 0.f && top <= 3.4e38f) frexpf(top, &e);
    e = max(-126, min(126, e));
    scale[0] = ldexpf(1.0f, e);
    scale[1] = ldexpf(1.0f, -e);
  }
}

// ------------------------------------------------------------------------------- products
constexpr int kMostWaves = 3;

struct ProductArgs {
  const int* count;
  int by_rows;              // 1: dx (tile rows are tokens, the sum runs over words); 0: dW (the other way)
  int row0, rows;           // the packed rows of this call
  int v0, nv;               // its vocabulary
  int d;
  int steps;                // products of parts a stage of the sum takes
  int64_t a_part, b_part;   // rows from one part of an operand to the next
  float4* slots;            // [kMostWaves pairs][256 / 4][256]: tiles whose sum is split
  float* acc;               // [rows or nv][ld] fp32, or null
  int64_t ld;
  int first, last;          // first: acc holds nothing yet; last: the result leaves as T
  int g0;                   // column of G where the piece begins
  int b_row0;               // dW: the right operand's first row
  const float* row_scale;   // dx: [rows], or null
  const float* scale;       // [0] (per-token gradients), or null:
  const float* up;          // the one gradient (null: 1),
  int mean;                 // over the tokens with a loss
  void* out;                // dx (rows by `index`) or dW
  const int* index;
  const int* place;         // dx, first call: [N], the tokens without a loss (-1) get zeros
  int64_t N;
  struct Cut* cut;          // left here for the join: dividing again in each of its threads took most of its time
};
template <typename T>
__device__ __forceinline__ float last_scale(const ProductArgs& a) {
  if (!a.last) return 1.0f;
  const float fold = std::is_same<T, __half>::value ? 1.0f / kHalfScale : 1.0f;
  if (a.scale) return a.scale[0] * fold;
  if (*a.count <= 0) return 0.0f;  // no token has a loss: the gradients are zero, whatever 0 / 0 says
  return (a.up ? *a.up : 1.0f) * (a.mean ? 1.0f / (float)*a.count : 1.0f) * fold;
}
struct Cut {  // how a product's tiles are spread over the pairs
  int mt, nt, width, kb, full, split, units;  // width: columns of a tile
};
// Columns are cut evenly, in steps of 32.  Whole waves of tiles keep their sum in one pair; of the rest each
// tile's sum is cut into equal parts: one wave of them, or, where the sums are long, two or three waves if that ends
// more than a tenth sooner (48 tiles on 74 pairs: three parts each, two waves of a third).  (Dealing the rest's stages
// out evenly instead, so that a pair works on two neighbouring tiles, balances better but lets the pairs read
// different rows of W at a time: 16384 x 768 x 32000 1883 -> 1920 us, 3277 rows 442 -> 466.)  Not so where it saves less
// than the parts' way through memory costs (6 us; a stage of a tile is 0.28 us).
__host__ __device__ __forceinline__ Cut cut_product(const ProductArgs& a, int live, int np) {
  Cut c;
  const int m = a.by_rows ? live : a.nv, k = a.by_rows ? (live > 0 ? a.nv : 0) : live;
  c.mt = (m + kTile - 1) / kTile;
  c.nt = (a.d + kTile - 1) / kTile;
  c.width = ((a.d + c.nt - 1) / c.nt + 31) & ~31;
  c.kb = (k + kBK - 1) / kBK;
  const int tiles = c.mt * c.nt, rem = tiles % np;
  c.full = tiles - rem;
  c.split = rem > 0 ? np / rem : 1;
  if (rem > 0 && c.kb * a.steps >= 128)
    for (int waves = 2, best = 1; waves <= kMostWaves; ++waves)
      if (waves * np / rem * 9 * best > c.split * 10 * waves) {
        c.split = waves * np / rem;
        best = waves;
      }
  c.split = min(c.split, c.kb);
  if (c.split <= 1 || c.kb * a.steps * (c.split - 1) < 20 * c.split) {
    c.split = 1;
    c.full = tiles;
  }
  c.units = c.full + (tiles - c.full) * c.split;
  return c;
}
__device__ __forceinline__ int product_live(const ProductArgs& a) { return min(max(*a.count - a.row0, 0), a.rows); }
struct Unit {
  int m, n, k0, k1, slot;  // slot < 0: a whole tile
};
__device__ __forceinline__ Unit unit_at(const Cut& c, int u) {
  Unit r;
  int tile = u;
  r.k0 = 0;
  r.k1 = c.kb;
  r.slot = -1;
  if (u >= c.full) {
    const int j = u - c.full, part = j % c.split;
    tile = c.full + j / c.split;
    r.k0 = (int)((int64_t)part * c.kb / c.split);
    r.k1 = (int)((int64_t)(part + 1) * c.kb / c.split);
    r.slot = j;
  }
  r.m = tile / c.nt;
  r.n = tile - r.m * c.nt;
  return r;
}
__device__ __forceinline__ int64_t row_out(const ProductArgs& a, int row) {
  return (a.by_rows ? (int64_t)a.index[a.row0 + row] : (int64_t)(a.v0 + row)) * a.d;
}
// 32 columns of each of a warp's 32 rows (a thread has a row's): what earlier calls left is added; the sum
// stays in fp32 or leaves as T.  It goes out by way of shared memory, so that a store instruction writes whole
// 64-byte (fp32: 128-byte) runs of rows instead of 16 bytes of each.
template <typename T>
__device__ __forceinline__ void finish32(const ProductArgs& a, int row, int rows, int col, int end, float (&v)[32],
                                         float scale, unsigned char* buf) {
  const int n = min(32, end - col), lane = threadIdx.x & 31;
  if (!a.first && row < rows) {
    const float* p = a.acc + (int64_t)row * a.ld + col;
#pragma unroll
    for (int i = 0; i < 32; i += 4)
      if (i < n) {  // rows are padded to fours
        const float4 o = *reinterpret_cast<const float4*>(p + i);
        v[i] += o.x;
        v[i + 1] += o.y;
        v[i + 2] += o.z;
        v[i + 3] += o.w;
      }
  }
  // rows that do not begin at 16 bytes leave in single elements, a warp a row's 32 (an element of 32 rows at a time
  // instead: bf16 loss with gradients of 4096 x 767 x 32000 675 us, here 531)
  const bool odd = a.last && (a.d % (16 / (int)sizeof(T)) != 0 || (reinterpret_cast<uintptr_t>(a.out) & 15) != 0);
  const bool wide = odd || !a.last || sizeof(T) == 4;  // 128 bytes of a row, or 64
  if (a.last) {
#pragma unroll
    for (int i = 0; i < 32; ++i) v[i] *= scale;
  }
  const int64_t mine = a.last && row < rows ? row_out(a, row) : (int64_t)row * a.ld;
  __syncwarp();  // the chunk before has been read
  if (wide) {
#pragma unroll
    for (int u = 0; u < 8; ++u)
      *reinterpret_cast<float4*>(buf + lane * 128 + ((u ^ (lane & 7)) << 4)) =
          make_float4(v[4 * u], v[4 * u + 1], v[4 * u + 2], v[4 * u + 3]);
  } else if constexpr (sizeof(T) == 2) {
#pragma unroll
    for (int u = 0; u < 4; ++u)
      *reinterpret_cast<uint4*>(buf + lane * 64 + ((u ^ ((lane >> 1) & 3)) << 4)) =
          make_uint4(pack2<T>(v[8 * u], v[8 * u + 1]), pack2<T>(v[8 * u + 2], v[8 * u + 3]),
                     pack2<T>(v[8 * u + 4], v[8 * u + 5]), pack2<T>(v[8 * u + 6], v[8 * u + 7]));
  }
  __syncwarp();
  const int row0 = row - lane;
  if (odd) {
    T* out = reinterpret_cast<T*>(a.out);
#pragma unroll 8
    for (int r = 0; r < 32; ++r) {
      const int64_t at = __shfl_sync(0xffffffffu, mine, r);
      if (row0 + r < rows && lane < n)
        out[at + col + lane] =
            from_f<T>(*reinterpret_cast<const float*>(buf + r * 128 + (((lane >> 2) ^ (r & 7)) << 4) + (lane & 3) * 4));
    }
  } else if (wide) {
    char* out = reinterpret_cast<char*>(a.last ? reinterpret_cast<float*>(a.out) : a.acc);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int r = 4 * i + (lane >> 3), u = lane & 7;
      const int64_t at = __shfl_sync(0xffffffffu, mine, r);
      if (row0 + r < rows && 4 * u < n)
        *reinterpret_cast<float4*>(out + (at + col + 4 * u) * 4) =
            *reinterpret_cast<const float4*>(buf + r * 128 + ((u ^ (r & 7)) << 4));
    }
  } else {
    T* out = reinterpret_cast<T*>(a.out);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int r = 8 * i + (lane >> 2), u = lane & 3;
      const int64_t at = __shfl_sync(0xffffffffu, mine, r);
      if (row0 + r < rows && 8 * u < n)
        *reinterpret_cast<uint4*>(out + at + col + 8 * u) =
            *reinterpret_cast<const uint4*>(buf + r * 64 + ((u ^ ((r >> 1) & 3)) << 4));
    }
  }
}

// A_MN: the left operand's summed dimension runs along its rows (dW); the right one's always does.
template <typename T, bool A_MN>
__global__ void __launch_bounds__(kThreads, 1) product_kernel(const __grid_constant__ CUtensorMap tmA,
                                                              const __grid_constant__ CUtensorMap tmA32,
                                                              const __grid_constant__ CUtensorMap tmB,
                                                              const ProductArgs a) {
  using O = Op<T>;
  constexpr int P = kParts<T>;
  constexpr int kBufs = P == 1 ? 2 : 1, kTake = P == 1 ? 1 << 30 : kFlush;
  extern __shared__ unsigned char raw[];
  const Smem s = carve(raw);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = cluster_rank2();
  const bool leader = rank == 0;
  const uint32_t tmem = pair_begin(s);
  const int np = gridDim.x >> 1, pair = blockIdx.x >> 1;
  const int live = product_live(a);
  const Cut c = cut_product(a, live, np);
  if (blockIdx.x == 0 && threadIdx.x == 0) *a.cut = c;

  if (warp == 0) {
    if (lane == 0) {
      int it = 0;
      bool failed = false;
      for (int u = pair; u < c.units && !failed; u += np) {
        const Unit w = unit_at(c, u);
        const int cols = (min(c.width, a.d - w.n * c.width) + 31) & ~31;
        const int ar = w.m * kTile + 128 * (int)rank, bc = w.n * c.width + (int)rank * (cols / 2);
        const int rows = A_MN ? kTile : live - w.m * kTile, boxes = boxes_of(rows, rank);
        const uint32_t bytes = 4096 * (boxes_of(rows, 0) + boxes_of(rows, 1)) + 2 * kOperand;
        // the right operand's rows: words of this piece, or this call's tokens
        const int br = a.by_rows ? a.v0 : a.b_row0;
        for (int k0 = w.k0; k0 < w.k1 && !failed; k0 += kTake)
        for (int p = 0; p < Parts<P>::n && !failed; ++p)
          for (int kb = k0; kb < min(w.k1, k0 + kTake); ++kb, ++it) {
            uint32_t bar;
            unsigned char* st = stage_begin(s, it, leader, bytes, bar);
            if (!st) {
              failed = true;
              break;
            }
            const int pa = (int)(Parts<P>::a(p) * a.a_part), pb = (int)(Parts<P>::b(p) * a.b_part);
            if constexpr (A_MN) {
              tma_load_2d_pair(st, &tmA, a.g0 + ar, pa + kb * kBK, bar);
              tma_load_2d_pair(st + 8192, &tmA, a.g0 + ar + 64, pa + kb * kBK, bar);
            } else {
              load_rows(st, &tmA, &tmA32, boxes, a.g0 + kb * kBK, pa + ar, bar);
            }
            tma_load_2d_pair(st + kOperand, &tmB, bc, pb + br + kb * kBK, bar);
            tma_load_2d_pair(st + kOperand + 8192, &tmB, bc + 64, pb + br + kb * kBK, bar);
          }
      }
      if (failed) copies_failed(s, it, leader);
    }
    __syncwarp();
  } else if (warp == 1) {
    if (lane == 0 && leader) {
      int it = 0, done = 0;
      bool failed = false;
      for (int u = pair; u < c.units && c.kb > 0 && !failed; u += np) {
        const Unit w = unit_at(c, u);
        const int cols = (min(c.width, a.d - w.n * c.width) + 31) & ~31;
        const uint32_t idesc =
            umma_idesc_f16(std::is_same<O, __nv_bfloat16>::value ? 1u : 0u, kTile, cols, A_MN ? 1u : 0u, 1u);
        for (int k0 = w.k0; k0 < w.k1 && !failed; k0 += kTake, ++done) {
          failed = !tile_free<kBufs>(s, done) ||
                   !issue_tile<A_MN, true>(s, tmem + (uint32_t)(done % kBufs * kTile), idesc,
                                           Parts<P>::n * min(kTake, w.k1 - k0), it);
          if (!failed) tile_issued<kBufs>(s, done);
        }
      }
      issue_end(s, failed);
    }
    __syncwarp();
  } else {
    const int q = warp & 3, half = (warp - 2) >> 2;
    const int in_tile = (int)rank * 128 + q * 32 + lane;
    unsigned char* buf = s.end + (warp - 2) * 4096;
    const float scale = last_scale<T>(a);
    if (a.place) {  // while the first tile is on its way: zeros for the tokens without a loss
      T* dx = reinterpret_cast<T*>(a.out);
      for (int64_t n = (int64_t)blockIdx.x * kEnders + warp - 2; n < a.N; n += (int64_t)gridDim.x * kEnders)
        if (a.place[n] < 0)
          for (int c = lane; c < a.d; c += 32) dx[n * a.d + c] = from_f<T>(0.f);
    }
    int done = 0;
    bool lost = false;
    for (int u = pair; u < c.units; u += np, ++done) {
      const Unit w = unit_at(c, u);
      const int row = w.m * kTile + in_tile, rows = a.by_rows ? live : a.nv;
      const int cols = min(c.width, a.d - w.n * c.width);
      const uint32_t lanes = tmem + ((uint32_t)(q * 32) << 16);
      bool more = false;  // parts of this sum have left before
      if constexpr (P > 1)
        for (int k0 = w.k0; k0 + kTake < w.k1; k0 += kTake, ++done) {
          keep_part(s, done, lost, leader, lanes, half * 32, cols, 64, more);
          more = true;
        }
      const uint32_t taddr = lanes + (uint32_t)(done % kBufs * kTile);
      if (c.kb > 0) tile_ready<kBufs>(s, done, lost);
#pragma unroll 1
      for (int col = half * 32; col < cols; col += 64) {
        uint32_t r[32];
        if (c.kb > 0) {
          read32(taddr + col, lost, r);
          read32_wait(lost, r);
        } else {  // nothing to sum: the result is what earlier calls left, or zero
#pragma unroll
          for (int i = 0; i < 32; ++i) r[i] = 0u;
        }
        if (P > 1 && more) add_parts(lanes, col, lost, r);
        float v[32];
#pragma unroll
        for (int i = 0; i < 32; ++i) v[i] = __uint_as_float(r[i]);
        if (w.slot >= 0) {  // [slot][four columns][row]: the warp's rows lie next to each other
          float4* p = a.slots + ((int64_t)w.slot * (kTile / 4) + col / 4) * kTile + in_tile;
#pragma unroll
          for (int i = 0; i < 8; ++i) p[i * kTile] = make_float4(v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3]);
        } else {
          const float own = a.last && a.row_scale && row < rows ? scale * a.row_scale[row] : scale;
          finish32<T>(a, row, rows, w.n * c.width + col, w.n * c.width + cols, v, own, buf);
        }
      }
      if (c.kb > 0) tile_read<kBufs>(s, done, lost, leader);
    }
  }
  pair_end(tmem);
}

// The tiles whose sum was split: their parts are added in order.  A CTA takes 32 rows x 32 columns of a tile: a
// warp adds four columns of the rows, then the block of sums is turned so that rows leave in runs.
template <typename T>
__global__ void __launch_bounds__(256) join_product_kernel(const ProductArgs a) {
  __shared__ float4 turn[32][9];
  allow_dependent_launch();
  wait_for_previous();
  const Cut c = *a.cut;
  const int live = product_live(a), j = blockIdx.x / 64, tile = c.full + j;
  if (tile >= c.mt * c.nt) return;
  const int m = tile / c.nt, n = tile - m * c.nt, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int r0 = (blockIdx.x >> 3 & 7) * 32, c0 = (blockIdx.x & 7) * 32;
  const int rows = a.by_rows ? live : a.nv;
  const int end = min(a.d, (n + 1) * c.width);
  if (m * kTile + r0 >= rows || n * c.width + c0 >= end) return;
  const float4* src = a.slots + ((int64_t)j * c.split * (kTile / 4) + c0 / 4 + warp) * kTile + r0 + lane;
  float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 8
  for (int p = 0; p < c.split; ++p) {
    const float4 o = src[(int64_t)p * (kTile / 4) * kTile];
    v.x += o.x;
    v.y += o.y;
    v.z += o.z;
    v.w += o.w;
  }
  turn[lane][warp] = v;
  __syncthreads();
  const int row = m * kTile + r0 + (threadIdx.x >> 3), col = n * c.width + c0 + 4 * (threadIdx.x & 7);
  if (row >= rows || col >= end) return;
  v = turn[threadIdx.x >> 3][threadIdx.x & 7];
  float4* acc = reinterpret_cast<float4*>(a.acc + (int64_t)row * a.ld + col);  // rows are padded to fours
  if (!a.first) {
    const float4 o = *acc;
    v.x += o.x;
    v.y += o.y;
    v.z += o.z;
    v.w += o.w;
  }
  if (!a.last) {
    *acc = v;
    return;
  }
  const float scale = last_scale<T>(a) * (a.row_scale ? a.row_scale[row] : 1.0f);
  T* p = reinterpret_cast<T*>(a.out) + row_out(a, row) + col;
  const float e[4] = {v.x * scale, v.y * scale, v.z * scale, v.w * scale};
  if (a.d % 4 == 0 && (reinterpret_cast<uintptr_t>(a.out) & 15) == 0) {
    if constexpr (sizeof(T) == 4)
      *reinterpret_cast<float4*>(p) = make_float4(e[0], e[1], e[2], e[3]);
    else
      *reinterpret_cast<uint2*>(p) = make_uint2(pack2<T>(e[0], e[1]), pack2<T>(e[2], e[3]));
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (col + i < end) p[i] = from_f<T>(e[i]);
  }
}

// ------------------------------------------------------------------------------- host
int64_t up_to(int64_t n, int64_t m) { return (n + m - 1) / m * m; }

// What the forward pass leaves for the backward one, and what each pass needs besides.
struct Sizes {
  int parts;
  int64_t rows, dp, vrows;  // packed rows, row length, packed words
  // offsets of the state
  int64_t x, w, label, index, place, stat, count, ticket, state_bytes;
  // forward workspace
  int64_t group, seg, target, partial, forward_bytes;
  // backward: rows of a run, words of a piece, and the workspace
  int64_t run, piece, g, slots, dx_acc, dw_acc, scale, cut, backward_bytes;
};
// Elements of G that are there at once (16-bit; fp32 keeps three parts of a third as many).
constexpr int64_t kPiece = 1LL << 27;
constexpr int64_t kRun = 8192;
Sizes sizes_of(int64_t N, int64_t V, int64_t d, bool pack_w, int dtype, int np) {
  Sizes s = {};
  s.parts = dtype == MB_F32 ? 3 : 1;
  s.rows = up_to(std::max<int64_t>(N, 1), kTile);
  s.dp = up_to(d, 8);
  s.vrows = up_to(V, kTile);
  auto take = [](int64_t& total, int64_t bytes) {
    const int64_t at = total;
    total = up_to(total + bytes, 256);
    return at;
  };
  s.x = take(s.state_bytes, s.parts * s.rows * s.dp * 2);
  s.label = take(s.state_bytes, s.rows * 4);
  s.index = take(s.state_bytes, s.rows * 4);
  s.place = take(s.state_bytes, N * 4);
  s.stat = take(s.state_bytes, s.rows * (int64_t)sizeof(RowStat));
  s.count = take(s.state_bytes, 4);
  s.ticket = take(s.state_bytes, 4);
  s.w = take(s.state_bytes, pack_w ? s.parts * s.vrows * s.dp * 2 : 0);  // last: nothing's place depends on it
  const int64_t mt = s.rows / kTile;
  s.group = take(s.forward_bytes, up_to(N, 256) / 256 * 4);
  s.seg = take(s.forward_bytes, (np + mt) * 2 * kTile * (int64_t)sizeof(float2));
  s.target = take(s.forward_bytes, s.rows * 4);
  s.partial = take(s.forward_bytes, s.rows / kJoinRows * 8);
  // a run of rows and a piece of the vocabulary: G of both together stays below kPiece elements
  const int64_t most = kPiece / s.parts;
  s.run = std::min(s.rows, s.parts == 3 ? kRun / 2 : kRun);
  s.piece = std::min(s.vrows, std::max<int64_t>(kTile, most / s.run / kTile * kTile));
  s.run = std::min(s.rows, std::max(s.run, most / s.piece / kTile * kTile));
  s.g = take(s.backward_bytes, s.parts * s.run * s.piece * 2);
  s.slots = take(s.backward_bytes, (int64_t)kMostWaves * np * kTile * kTile * 4);
  s.dx_acc = take(s.backward_bytes, s.piece < s.vrows ? s.run * up_to(d, 4) * 4 : 0);
  s.dw_acc = take(s.backward_bytes, s.run < s.rows ? V * up_to(d, 4) * 4 : 0);
  s.scale = take(s.backward_bytes, 8);
  s.cut = take(s.backward_bytes, sizeof(Cut));
  return s;
}

// The loss and its gradients at once: everything lies in the workspace.
struct OnceSizes {
  int parts;
  int64_t rows, dp, vrows, run, runs, piece;
  int64_t x, w, label, index, place, stat, ref, target, row_scale, count, ticket, flags, group, seg, partial;
  int64_t e, weighed, slots, dx_acc, dw_acc, cut, bytes;
};
// Elements of E that are there at once: a run of rows with the whole vocabulary (fp32: three parts of a third
// as many), or 256 rows of a vocabulary so large that they have more.
constexpr int64_t kOnceElements = 1LL << 28;
// 16-bit: terms that are added within the tensor cores, which cut each partial sum off at 24 bits (2^16 / 16
// of them: 2^-12 of the result at most, half a unit of bf16 being 2^-9).
constexpr int64_t kLongRun = 1LL << 16;

OnceSizes once_sizes_of(int64_t N, int64_t V, int64_t d, bool pack_w, int dtype, int np) {
  OnceSizes s = {};
  s.parts = dtype == MB_F32 ? 3 : 1;
  s.rows = up_to(std::max<int64_t>(N, 1), kTile);
  s.dp = up_to(d, 8);
  s.vrows = up_to(V, kTile);
  s.run = std::min(s.rows, std::max<int64_t>(kTile, kOnceElements / s.parts / s.vrows / kTile * kTile));
  s.run = std::min(s.run, kLongRun);
  s.runs = (s.rows + s.run - 1) / s.run;
  s.piece = std::min(s.vrows, s.parts == 1 ? kLongRun : s.vrows);  // dx's sums run over the words of a piece
  auto take = [&](int64_t bytes) {
    const int64_t at = s.bytes;
    s.bytes = up_to(s.bytes + bytes, 256);
    return at;
  };
  s.x = take(s.parts * s.rows * s.dp * 2);
  s.w = take(pack_w ? s.parts * s.vrows * s.dp * 2 : 0);
  s.label = take(s.rows * 4);
  s.index = take(s.rows * 4);
  s.place = take(N * 4);
  s.stat = take(s.rows * (int64_t)sizeof(RowStat));
  s.ref = take(s.rows * 4);
  s.target = take(s.rows * 4);
  s.row_scale = take(s.run * 4);
  s.count = take(4);
  s.ticket = take(4);
  s.flags = take(s.runs * 4);
  s.group = take(up_to(N, 256) / 256 * 4);
  s.seg = take((np + s.run / kTile) * 2 * kTile * (int64_t)sizeof(float2));
  s.partial = take(s.rows / kSettleRows * 8);
  s.e = take(s.parts * s.run * s.vrows * 2);
  s.weighed = take(s.parts * s.run * s.dp * 2);
  s.slots = take((int64_t)kMostWaves * np * kTile * kTile * 4);
  s.dx_acc = take(s.piece < s.vrows ? s.run * up_to(d, 4) * 4 : 0);
  s.dw_acc = take(s.runs > 1 ? V * up_to(d, 4) * 4 : 0);
  s.cut = take(sizeof(Cut));
  return s;
}

// Launches that may begin while the kernel before them ends (all of these wait for it before they touch memory).
template <typename K, typename... A>
int launch(const char* what, K kern, int64_t grid, int threads, cudaStream_t st, int smem, int cluster, A... args) {
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute at[2];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  at[1].id = cudaLaunchAttributeClusterDimension;
  at[1].val.clusterDim.x = (unsigned)cluster;
  at[1].val.clusterDim.y = 1;
  at[1].val.clusterDim.z = 1;
  cfg.gridDim = dim3((unsigned)grid);
  cfg.blockDim = dim3((unsigned)threads);
  cfg.dynamicSmemBytes = (size_t)smem;
  cfg.stream = st;
  cfg.attrs = at;
  cfg.numAttrs = cluster > 1 ? 2 : 1;
  cudaLaunchKernelEx(&cfg, kern, args...);
  return check_launch(what);
}
template <typename K, typename... A>
int launch_pairs(const char* what, K kern, int np, cudaStream_t st, A... args) {
  if (int e = ensure_smem_attr((const void*)kern, kSmem)) return e;
  return launch(what, kern, 2 * np, kThreads, st, kSmem, 2, args...);
}

struct Call {
  const void *x, *w;
  int64_t xs, ws;
  const int64_t* labels;
  int64_t ignore, N, V, d;
  int reduction, dtype;
  unsigned char *state, *work;
  cudaStream_t st;
  bool pack_w;
  Sizes s;
  int np;
};
template <typename T> T* at(unsigned char* base, int64_t off) { return reinterpret_cast<T*>(base + off); }

// The scores' kernel of a call.
template <typename T, int MODE>
int launch_scores(const char* what, int np, cudaStream_t st, const CUtensorMap& x, const CUtensorMap& x32, const CUtensorMap& w,
                  const CUtensorMap& g, const ScoreArgs& a) {
  if constexpr (kParts<T> > 1)
    if (a.kblocks > kFlush) return launch_pairs(what, scores_kernel<T, MODE, true>, np, st, x, x32, w, g, a);
  return launch_pairs(what, scores_kernel<T, MODE, false>, np, st, x, x32, w, g, a);
}

// The weight as rows for the tensor maps: itself, or its packed copy.
void weight_rows(const Call& c, const void** base, int64_t* rows, int64_t* stride, int64_t* cols) {
  *base = c.pack_w ? c.state + c.s.w : c.w;
  *rows = c.pack_w ? c.s.parts * c.s.vrows : c.V;
  *stride = c.pack_w ? c.s.dp : c.ws;
  *cols = c.pack_w ? c.s.dp : c.d;
}

// The rows that have a loss, packed, and the weight where it has to be.
template <typename T>
int pack(const Call& c, PackArgs& p, int* group, void* packed_w, int64_t vrows) {
  if (c.N > 8192) {  // below that a CTA reads the labels before its own
    group_count_kernel<<<(unsigned)((c.N + 255) / 256), 256, 0, c.st>>>(c.labels, c.N, c.ignore, group);
    if (int e = check_launch("linear_cross_entropy (count)")) return e;
    p.group = group;
  }
  p.x = c.x;
  p.labels = c.labels;
  p.N = c.N;
  p.xs = c.xs;
  p.ignore = c.ignore;
  p.V = (int)c.V;
  p.d = (int)c.d;
  // a warp takes one token (48 x 768 x 32000, ten calls in a row from C with the mean of the losses: 27.8 us; two tokens
  // 29.2), or two where that were more CTAs than SMs
  p.tokens = c.N <= 8 * multiprocessors() ? 8 : 16;
  int rc = launch("linear_cross_entropy (pack)", pack_kernel<T>,
                  std::max<int64_t>(1, (c.N + p.tokens - 1) / p.tokens), 256, c.st, 0, 1, p);
  if (!rc && c.pack_w)
    rc = launch("linear_cross_entropy (pack weight)", pack_weight_kernel<T>,
                std::min<int64_t>((vrows + 7) / 8, multiprocessors() * 16), 256, c.st, 0, 1, (const T*)c.w, c.ws,
                (int)c.V, (int)c.d, p.dp, vrows, (Op<T>*)packed_w);
  return rc;
}

template <typename T>
int forward(const Call& c, float* loss) {
  const Sizes& s = c.s;
  PackArgs p = {};
  p.dp = (int)s.dp;
  p.rows = s.rows;
  p.packed = c.state + s.x;
  p.count = at<int>(c.state, s.count);
  p.ticket = at<int>(c.state, s.ticket);
  p.label = at<int>(c.state, s.label);
  p.index = at<int>(c.state, s.index);
  p.place = at<int>(c.state, s.place);
  p.loss = c.reduction == 0 ? loss : nullptr;
  int rc = pack<T>(c, p, at<int>(c.work, s.group), c.state + s.w, s.vrows);
  if (rc) return rc;
  CUtensorMap tmX, tmX32, tmW;
  const void* wb;
  int64_t wr, wst, wc;
  weight_rows(c, &wb, &wr, &wst, &wc);
  rc = encode_tile_map_2d(&tmX, c.state + s.x, 2, s.dp, s.parts * s.rows, s.dp * 2, kBK, 128, 128);
  if (!rc) rc = encode_tile_map_2d(&tmX32, c.state + s.x, 2, s.dp, s.parts * s.rows, s.dp * 2, kBK, 32, 128);
  if (!rc) rc = encode_tile_map_2d(&tmW, wb, 2, wc, wr, wst * 2, kBK, 128, 128);
  if (rc) return rc;
  ScoreArgs a = {};
  a.count = p.count;
  a.rows = (int)s.rows;
  a.nv = (int)c.V;
  a.kblocks = (int)((c.d + kBK - 1) / kBK);
  a.x_part = s.rows;
  a.w_part = s.vrows;
  a.label = p.label;
  a.seg = at<float2>(c.work, s.seg);
  a.target = at<float>(c.work, s.target);
  rc = launch_scores<T, kLoss>("linear_cross_entropy (scores)", c.np, c.st, tmX, tmX32, tmW, tmX, a);
  if (rc) return rc;
  JoinArgs j = {};
  j.count = p.count;
  j.ticket = p.ticket;
  j.seg = a.seg;
  j.target = a.target;
  j.label = p.label;
  j.index = p.index;
  j.stat = at<RowStat>(c.state, s.stat);
  j.loss = loss;
  j.partial = at<double>(c.work, s.partial);
  j.nt = (int)((c.V + kTile - 1) / kTile);
  j.np = c.np;
  j.reduction = c.reduction;
  return launch("linear_cross_entropy (join)", join_kernel, s.rows / kJoinRows, 32 * kJoinRows, c.st, 0, 1, j);
}

template <typename T>
int backward(const Call& c, const float* up, int64_t up_stride, void* dx, void* dw) {
  const Sizes& s = c.s;
  const int* count = at<int>(c.state, s.count);
  const int* place = at<int>(c.state, s.place);
  const int* index = at<int>(c.state, s.index);
  float* scale = at<float>(c.work, s.scale);
  int rc = MB_OK;
  if (c.reduction == 0) {
    rc = launch("linear_cross_entropy_backward (scale)", scale_kernel, 1, 1024, c.st, 0, 1, up, up_stride, c.N, place, scale);
    if (rc) return rc;
  }
  const void* wb;
  int64_t wr, wst, wc;
  weight_rows(c, &wb, &wr, &wst, &wc);
  CUtensorMap tmX, tmX32, tmW, tmG, tmXk, tmWk, tmGa, tmGa32, tmGt;
  unsigned char* g = c.work + s.g;
  rc = encode_tile_map_2d(&tmX, c.state + s.x, 2, s.dp, s.parts * s.rows, s.dp * 2, kBK, 128, 128);
  if (!rc) rc = encode_tile_map_2d(&tmW, wb, 2, wc, wr, wst * 2, kBK, 128, 128);
  if (!rc) rc = encode_tile_map_2d(&tmX32, c.state + s.x, 2, s.dp, s.parts * s.rows, s.dp * 2, kBK, 32, 128);
  if (!rc) rc = encode_tile_map_2d(&tmXk, c.state + s.x, 2, s.dp, s.parts * s.rows, s.dp * 2, 64, kBK, 128);
  if (!rc) rc = encode_tile_map_2d(&tmWk, wb, 2, wc, wr, wst * 2, 64, kBK, 128);
  if (!rc) rc = encode_tile_map_2d(&tmG, g, 2, s.piece, s.parts * s.run, s.piece * 2, 64, 32, 128);   // stored
  if (!rc) rc = encode_tile_map_2d(&tmGa, g, 2, s.piece, s.parts * s.run, s.piece * 2, kBK, 128, 128);  // tokens x words
  if (!rc) rc = encode_tile_map_2d(&tmGa32, g, 2, s.piece, s.parts * s.run, s.piece * 2, kBK, 32, 128);
  if (!rc) rc = encode_tile_map_2d(&tmGt, g, 2, s.piece, s.parts * s.run, s.piece * 2, 64, kBK, 128);   // words x tokens
  if (rc) return rc;
  for (int64_t r0 = 0; r0 < s.rows; r0 += s.run)
    for (int64_t v0 = 0; v0 < c.V; v0 += s.piece) {
      ScoreArgs a = {};
      a.count = count;
      a.row0 = (int)r0;
      a.rows = (int)std::min(s.run, s.rows - r0);
      a.v0 = (int)v0;
      a.nv = (int)std::min(s.piece, c.V - v0);
      a.kblocks = (int)((c.d + kBK - 1) / kBK);
      a.x_part = s.rows;
      a.w_part = s.vrows;
      a.label = at<int>(c.state, s.label);
      a.stat = at<RowStat>(c.state, s.stat);
      a.index = index;
      a.up = c.reduction == 0 ? up : nullptr;
      a.up_stride = up_stride;
      a.scale = scale;
      a.g_part = s.run;
      rc = launch_scores<T, kAgain>("linear_cross_entropy_backward (scores)", c.np, c.st, tmX, tmX32, tmW, tmG, a);
      if (rc) return rc;
      ProductArgs p = {};
      p.steps = Parts<kParts<T>>::n;
      p.count = count;
      p.row0 = a.row0;
      p.rows = a.rows;
      p.v0 = a.v0;
      p.nv = a.nv;
      p.d = (int)c.d;
      p.a_part = s.run;
      p.slots = at<float4>(c.work, s.slots);
      p.ld = up_to(c.d, 4);
      p.cut = at<Cut>(c.work, s.cut);
      p.scale = c.reduction == 0 ? scale : nullptr;
      p.up = up;
      p.mean = c.reduction == 1;
      p.b_row0 = p.row0;
      p.index = index;
      p.N = c.N;
      if (dx) {
        p.by_rows = 1;
        p.b_part = s.vrows;
        p.acc = at<float>(c.work, s.dx_acc);
        p.first = v0 == 0;
        p.last = v0 + s.piece >= c.V;
        p.out = dx;
        p.place = r0 == 0 && v0 == 0 ? place : nullptr;
        rc = launch_pairs("linear_cross_entropy_backward (dx)", product_kernel<T, false>, c.np, c.st, tmGa, tmGa32, tmWk,
                          p);
        // how many tiles are split the device knows: at most all, and fewer than there are pairs
        const int64_t most = std::min<int64_t>(c.np - 1, up_to(p.rows, kTile) / kTile * ((c.d + kTile - 1) / kTile));
        if (!rc && most > 0)
          rc = launch("linear_cross_entropy_backward (dx join)", join_product_kernel<T>, 64 * most, 256, c.st, 0, 1, p);
        if (rc) return rc;
      }
      if (dw) {
        p.by_rows = 0;
        p.b_part = s.rows;
        p.acc = at<float>(c.work, s.dw_acc) + v0 * p.ld;
        p.first = r0 == 0;
        p.last = r0 + s.run >= s.rows;
        p.out = dw;
        p.place = nullptr;
        rc = launch_pairs("linear_cross_entropy_backward (dw)", product_kernel<T, true>, c.np, c.st, tmGt, tmGt, tmXk, p);
        const int64_t rest = up_to(p.nv, kTile) / kTile * ((c.d + kTile - 1) / kTile) % c.np;
        if (!rc && rest > 0 && c.N > kBK)  // (a sum of one stage is not split)
          rc = launch("linear_cross_entropy_backward (dw join)", join_product_kernel<T>, 64 * rest, 256, c.st, 0, 1, p);
        if (rc) return rc;
      }
    }
  return MB_OK;
}

// Loss and gradients, run by run: E, its rows' sums, then both products.
template <typename T>
int once(const Call& c, const OnceSizes& s, float* loss, void* dx, void* dw) {
  unsigned char* ws = c.work;
  PackArgs p = {};
  p.dp = (int)s.dp;
  p.rows = s.rows;
  p.packed = ws + s.x;
  p.count = at<int>(ws, s.count);
  p.ticket = at<int>(ws, s.ticket);
  p.label = at<int>(ws, s.label);
  p.index = at<int>(ws, s.index);
  p.place = at<int>(ws, s.place);
  p.w = c.w;
  p.ws = c.ws;
  p.ref = at<float>(ws, s.ref);
  p.flags = at<int>(ws, s.flags);
  p.runs = (int)s.runs;
  int rc = pack<T>(c, p, at<int>(ws, s.group), ws + s.w, s.vrows);
  if (rc) return rc;
  const void* wb = c.pack_w ? ws + s.w : c.w;
  const int64_t wr = c.pack_w ? s.parts * s.vrows : c.V, wst = c.pack_w ? s.dp : c.ws, wc = c.pack_w ? s.dp : c.d;
  CUtensorMap tmX, tmX32, tmW, tmWk, tmE, tmEa, tmEa32, tmEt, tmXk;
  unsigned char* e = ws + s.e;
  rc = encode_tile_map_2d(&tmX, ws + s.x, 2, s.dp, s.parts * s.rows, s.dp * 2, kBK, 128, 128);
  if (!rc) rc = encode_tile_map_2d(&tmX32, ws + s.x, 2, s.dp, s.parts * s.rows, s.dp * 2, kBK, 32, 128);
  if (!rc) rc = encode_tile_map_2d(&tmW, wb, 2, wc, wr, wst * 2, kBK, 128, 128);
  if (!rc) rc = encode_tile_map_2d(&tmWk, wb, 2, wc, wr, wst * 2, 64, kBK, 128);
  if (!rc) rc = encode_tile_map_2d(&tmXk, ws + s.weighed, 2, s.dp, s.parts * s.run, s.dp * 2, 64, kBK, 128);
  if (!rc) rc = encode_tile_map_2d(&tmE, e, 2, s.vrows, s.parts * s.run, s.vrows * 2, 64, 32, 128);      // stored
  if (!rc) rc = encode_tile_map_2d(&tmEa, e, 2, s.vrows, s.parts * s.run, s.vrows * 2, kBK, 128, 128);   // tokens x words
  if (!rc) rc = encode_tile_map_2d(&tmEa32, e, 2, s.vrows, s.parts * s.run, s.vrows * 2, kBK, 32, 128);
  if (!rc) rc = encode_tile_map_2d(&tmEt, e, 2, s.vrows, s.parts * s.run, s.vrows * 2, 64, kBK, 128);    // words x tokens
  if (rc) return rc;
  for (int64_t i = 0; i < s.runs; ++i) {
    ScoreArgs a = {};
    a.count = p.count;
    a.row0 = (int)(i * s.run);
    a.rows = (int)std::min(s.run, s.rows - i * s.run);
    a.nv = (int)c.V;
    a.kblocks = (int)((c.d + kBK - 1) / kBK);
    a.x_part = s.rows;
    a.w_part = s.vrows;
    a.label = p.label;
    a.seg = at<float2>(ws, s.seg);
    a.ref = p.ref;
    a.target = at<float>(ws, s.target);
    a.flag = p.flags + i;
    a.stat = at<RowStat>(ws, s.stat);
    a.index = p.index;
    a.g_part = s.run;
    rc = launch_scores<T, kOnce>("linear_cross_entropy_train (scores)", c.np, c.st, tmX, tmX32, tmW, tmE, a);
    if (rc) return rc;
    SettleArgs b = {};
    b.count = p.count;
    b.ticket = p.ticket;
    b.seg = a.seg;
    b.ref = p.ref;
    b.target = a.target;
    b.label = p.label;
    b.stat = at<RowStat>(ws, s.stat);
    b.flag = a.flag;
    b.row_scale = at<float>(ws, s.row_scale);
    b.loss = loss;
    b.partial = at<double>(ws, s.partial);
    b.nt = (int)((c.V + kTile - 1) / kTile);
    b.np = c.np;
    b.mean = c.reduction == 1;
    b.row0 = a.row0;
    b.rows = a.rows;
    b.x = ws + s.x;
    b.x_part = s.rows;
    b.weighed = ws + s.weighed;
    b.w_part = s.run;
    b.dp = (int)s.dp;
    b.e = e;
    b.ld = s.vrows;
    rc = launch("linear_cross_entropy_train (settle)", settle_kernel<T>, a.rows / kSettleRows, 32 * kSettleRows, c.st, 0, 1, b);
    if (!rc)
      rc = launch_scores<T, kAgain>("linear_cross_entropy_train (again)", c.np, c.st, tmX, tmX32, tmW, tmE, a);
    if (rc) return rc;
    ProductArgs q = {};
    q.steps = Parts<kParts<T>>::n;
    q.count = p.count;
    q.row0 = a.row0;
    q.rows = a.rows;
    q.d = (int)c.d;
    q.a_part = s.run;
    q.slots = at<float4>(ws, s.slots);
    q.ld = up_to(c.d, 4);
    q.cut = at<Cut>(ws, s.cut);
    q.mean = c.reduction == 1;
    q.index = p.index;
    q.N = c.N;
    const int64_t nt = (c.d + kTile - 1) / kTile;
    for (int64_t v0 = 0; dx && v0 < c.V; v0 += s.piece) {
      q.by_rows = 1;
      q.v0 = (int)v0;
      q.g0 = (int)v0;
      q.nv = (int)std::min(s.piece, c.V - v0);
      q.b_part = s.vrows;
      q.acc = at<float>(ws, s.dx_acc);
      q.row_scale = b.row_scale;
      q.first = v0 == 0;
      q.last = v0 + s.piece >= c.V;
      q.out = dx;
      q.place = i == 0 && v0 == 0 ? p.place : nullptr;
      rc = launch_pairs("linear_cross_entropy_train (dx)", product_kernel<T, false>, c.np, c.st, tmEa, tmEa32, tmWk, q);
      // how many tiles are split the device knows: at most all, and fewer than there are pairs
      const int64_t most = std::min<int64_t>(c.np - 1, a.rows / kTile * nt);
      if (!rc && most > 0)
        rc = launch("linear_cross_entropy_train (dx join)", join_product_kernel<T>, 64 * most, 256, c.st, 0, 1, q);
      if (rc) return rc;
    }
    if (dw) {
      q.by_rows = 0;
      q.v0 = 0;
      q.g0 = 0;
      q.nv = (int)c.V;
      q.b_part = s.run;
      q.b_row0 = 0;
      q.acc = at<float>(ws, s.dw_acc);
      q.row_scale = nullptr;
      q.first = i == 0;
      q.last = i + 1 == s.runs;
      q.out = dw;
      q.place = nullptr;
      rc = launch_pairs("linear_cross_entropy_train (dw)", product_kernel<T, true>, c.np, c.st, tmEt, tmEt, tmXk, q);
      const int64_t rest = s.vrows / kTile * nt % c.np;
      if (!rc && rest > 0 && c.N > kBK)  // (a sum of one stage is not split)
        rc = launch("linear_cross_entropy_train (dw join)", join_product_kernel<T>, 64 * rest, 256, c.st, 0, 1, q);
      if (rc) return rc;
    }
  }
  return MB_OK;
}

// 16-bit weights whose rows the tensor maps can describe are operands themselves.
bool must_pack(const void* w, int64_t ws, int64_t d, int dtype) {
  return dtype == MB_F32 || (uintptr_t)w % 16 != 0 || ws % 8 != 0 || ws < d;
}

int check_sizes(const char* what, int64_t N, int64_t V, int64_t d, int dtype) {
  MB_REQUIRE(dtype == MB_F32 || dtype == MB_F16 || dtype == MB_BF16, MB_ERR_DTYPE, "%s: unsupported dtype code %d", what,
             dtype);
  MB_REQUIRE(N >= 0 && N < (1LL << 29) && V > 0 && V < (1LL << 29) && d > 0 && d < (1LL << 24), MB_ERR_SHAPE,
             "%s: bad sizes N=%lld V=%lld d=%lld", what, (long long)N, (long long)V, (long long)d);
  return MB_OK;
}
// `state_bytes`: the backward pass's, which is laid out as the forward pass chose (0: this is that pass).  Where the
// weight lies and how its rows are strided may have changed in between, so neither tells: the state's size does.
int make_call(const char* what, Call& c, int64_t state_bytes = 0) {
  if (int e = check_sizes(what, c.N, c.V, c.d, c.dtype)) return e;
  MB_REQUIRE(c.reduction >= 0 && c.reduction <= 2, MB_ERR_ARG, "%s: unknown reduction %d", what, c.reduction);
  MB_REQUIRE(c.w && c.state && c.work, MB_ERR_ARG, "%s: null pointer", what);
  MB_REQUIRE(((uintptr_t)c.state | (uintptr_t)c.work) % 256 == 0, MB_ERR_ALIGN,
             "%s: state and workspace must be 256-byte aligned", what);
  c.np = std::max(1, multiprocessors() / 2);
  c.pack_w = must_pack(c.w, c.ws, c.d, c.dtype);
  c.s = sizes_of(c.N, c.V, c.d, c.pack_w, c.dtype, c.np);
  if (few_tokens(c.N, c.d, c.dtype)) {
    few_sizes(c.N, c.V, c.d, &c.s.state_bytes, &c.s.forward_bytes, &c.s.backward_bytes);
  } else if (state_bytes && c.dtype != MB_F32) {  // (fp32 weights are always packed)
    const Sizes other = sizes_of(c.N, c.V, c.d, !c.pack_w, c.dtype, c.np);
    if (state_bytes == other.state_bytes) {
      MB_REQUIRE(!c.pack_w, MB_ERR_ALIGN,
                 "%s: the forward pass read the weight where it was, so its rows must begin at 16-byte boundaries here, too",
                 what);
      c.pack_w = true;
      c.s = other;
    }
    MB_REQUIRE(state_bytes == c.s.state_bytes, MB_ERR_ARG,
               "%s: a state of %lld bytes is none that a forward pass of these sizes left (%lld or %lld)", what,
               (long long)state_bytes, (long long)c.s.state_bytes, (long long)other.state_bytes);
  }
  return MB_OK;
}
// The call as the kernels of a few fp32 tokens take it.
FewCall few_call(const Call& c) {
  FewCall f = {};
  f.x = (const float*)c.x;
  f.w = (const float*)c.w;
  f.xs = c.xs;
  f.ws = c.ws;
  f.labels = c.labels;
  f.ignore = c.ignore;
  f.N = c.N;
  f.V = c.V;
  f.d = c.d;
  f.reduction = c.reduction;
  f.state = c.state;
  f.work = c.work;
  f.st = c.st;
  return f;
}

}  // namespace

int read_and_clear_vocab_timeouts(unsigned int* count) {
  unsigned int v = 0, zero = 0;
  if (cudaMemcpyFromSymbol(&v, g_vocab_wait_timeouts, sizeof(v)) != cudaSuccess ||
      cudaMemcpyToSymbol(g_vocab_wait_timeouts, &zero, sizeof(zero)) != cudaSuccess)
    return set_error(MB_ERR_CUDA, "wait_timeouts: %s", cudaGetErrorString(cudaGetLastError()));
  *count = v;
  return MB_OK;
}

}  // namespace mb

extern "C" int motif_b200_linear_cross_entropy_bytes(const void* w, int64_t ws, int64_t N, int64_t V, int64_t d, int dtype,
                                                     int64_t* bytes) {
  using namespace mb;
  MB_REQUIRE(bytes, MB_ERR_ARG, "linear_cross_entropy_bytes: null pointer");
  if (int e = check_sizes("linear_cross_entropy_bytes", N, V, d, dtype)) return e;
  if (few_tokens(N, d, dtype)) {
    few_sizes(N, V, d, bytes, bytes + 1, bytes + 2);
    return MB_OK;
  }
  const Sizes s = sizes_of(N, V, d, must_pack(w, ws, d, dtype), dtype, std::max(1, multiprocessors() / 2));
  bytes[0] = s.state_bytes;
  bytes[1] = s.forward_bytes;
  bytes[2] = s.backward_bytes;
  return MB_OK;
}

extern "C" int motif_b200_linear_cross_entropy(const void* x, int64_t xs, const void* w, int64_t ws, const int64_t* labels,
                                               int64_t ignore_index, int reduction, float* loss, int64_t N, int64_t V,
                                               int64_t d, void* state, int64_t state_bytes, void* workspace,
                                               int64_t workspace_bytes, int dtype, void* stream) {
  using namespace mb;
  Call c = {};
  c.x = x;
  c.xs = xs;
  c.w = w;
  c.ws = ws;
  c.labels = labels;
  c.ignore = ignore_index;
  c.reduction = reduction;
  c.N = N;
  c.V = V;
  c.d = d;
  c.dtype = dtype;
  c.state = (unsigned char*)state;
  c.work = (unsigned char*)workspace;
  c.st = (cudaStream_t)stream;
  if (int e = make_call("linear_cross_entropy", c)) return e;
  MB_REQUIRE((N == 0 || (x && labels)) && (loss || (N == 0 && reduction == 0)), MB_ERR_ARG,
             "linear_cross_entropy: null pointer");
  MB_REQUIRE(state_bytes >= c.s.state_bytes && workspace_bytes >= c.s.forward_bytes, MB_ERR_ARG,
             "linear_cross_entropy: %lld and %lld bytes of state and workspace needed, got %lld and %lld",
             (long long)c.s.state_bytes, (long long)c.s.forward_bytes, (long long)state_bytes,
             (long long)workspace_bytes);
  if (few_tokens(N, d, dtype)) {
    FewCall f = few_call(c);
    f.loss = loss;
    return few_forward(f);
  }
  if (dtype == MB_F32) return forward<float>(c, loss);
  return dtype == MB_BF16 ? forward<__nv_bfloat16>(c, loss) : forward<__half>(c, loss);
}

extern "C" int motif_b200_linear_cross_entropy_backward(const void* w, int64_t ws, const float* grad_loss,
                                                        int64_t grad_stride, int reduction, void* dx, void* dw, int64_t N,
                                                        int64_t V, int64_t d, void* state, int64_t state_bytes,
                                                        void* workspace, int64_t workspace_bytes, int dtype,
                                                        void* stream) {
  using namespace mb;
  Call c = {};
  c.w = w;
  c.ws = ws;
  c.reduction = reduction;
  c.N = N;
  c.V = V;
  c.d = d;
  c.dtype = dtype;
  c.state = (unsigned char*)state;
  c.work = (unsigned char*)workspace;
  c.st = (cudaStream_t)stream;
  if (int e = make_call("linear_cross_entropy_backward", c, std::max<int64_t>(1, state_bytes))) return e;
  MB_REQUIRE(grad_loss || (N == 0 && reduction == 0), MB_ERR_ARG, "linear_cross_entropy_backward: null pointer");
  MB_REQUIRE(state_bytes >= c.s.state_bytes && workspace_bytes >= c.s.backward_bytes, MB_ERR_ARG,
             "linear_cross_entropy_backward: %lld and %lld bytes of state and workspace needed, got %lld and %lld",
             (long long)c.s.state_bytes, (long long)c.s.backward_bytes, (long long)state_bytes,
             (long long)workspace_bytes);
  if (!dx && !dw) return MB_OK;
  if (few_tokens(N, d, dtype)) {
    FewCall f = few_call(c);
    f.up = grad_loss;
    f.up_stride = grad_stride;
    f.dx = (float*)dx;
    f.dw = (float*)dw;
    return few_backward(f);
  }
  if (dtype == MB_F32) return backward<float>(c, grad_loss, grad_stride, dx, dw);
  return dtype == MB_BF16 ? backward<__nv_bfloat16>(c, grad_loss, grad_stride, dx, dw)
                          : backward<__half>(c, grad_loss, grad_stride, dx, dw);
}

extern "C" int64_t motif_b200_linear_cross_entropy_train_workspace_bytes(const void* w, int64_t ws, int64_t N, int64_t V,
                                                                         int64_t d, int dtype) {
  using namespace mb;
  if (check_sizes("linear_cross_entropy_train_workspace_bytes", N, V, d, dtype)) return -1;
  if (few_tokens(N, d, dtype)) {
    int64_t state, forward_bytes, backward_bytes;
    few_sizes(N, V, d, &state, &forward_bytes, &backward_bytes);
    return state + std::max(forward_bytes, backward_bytes);
  }
  return once_sizes_of(N, V, d, must_pack(w, ws, d, dtype), dtype, std::max(1, multiprocessors() / 2)).bytes;
}

extern "C" int motif_b200_linear_cross_entropy_train(const void* x, int64_t xs, const void* w, int64_t ws,
                                                     const int64_t* labels, int64_t ignore_index, int reduction,
                                                     float* loss, void* dx, void* dw, int64_t N, int64_t V, int64_t d,
                                                     void* workspace, int64_t workspace_bytes, int dtype, void* stream) {
  using namespace mb;
  Call c = {};
  c.x = x;
  c.xs = xs;
  c.w = w;
  c.ws = ws;
  c.labels = labels;
  c.ignore = ignore_index;
  c.reduction = reduction;
  c.N = N;
  c.V = V;
  c.d = d;
  c.dtype = dtype;
  c.state = c.work = (unsigned char*)workspace;
  c.st = (cudaStream_t)stream;
  if (int e = make_call("linear_cross_entropy_train", c)) return e;
  MB_REQUIRE(dtype != MB_F16, MB_ERR_UNSUPPORTED,
             "linear_cross_entropy_train: fp16 has too small a range for exponentials without their sum");
  MB_REQUIRE(reduction == 1 || reduction == 2, MB_ERR_ARG, "linear_cross_entropy_train: reduction must be 1 or 2, got %d",
             reduction);
  MB_REQUIRE((N == 0 || (x && labels)) && loss, MB_ERR_ARG, "linear_cross_entropy_train: null pointer");
  if (few_tokens(N, d, dtype)) {
    MB_REQUIRE(workspace_bytes >= c.s.state_bytes + std::max(c.s.forward_bytes, c.s.backward_bytes), MB_ERR_ARG,
               "linear_cross_entropy_train: %lld bytes of workspace needed, got %lld",
               (long long)(c.s.state_bytes + std::max(c.s.forward_bytes, c.s.backward_bytes)), (long long)workspace_bytes);
    FewCall f = few_call(c);
    f.loss = loss;
    f.dx = (float*)dx;
    f.dw = (float*)dw;
    f.work = c.work + c.s.state_bytes;
    if (int e = few_forward(f)) return e;
    return dx || dw ? few_backward(f) : MB_OK;
  }
  const OnceSizes s = once_sizes_of(N, V, d, c.pack_w, dtype, c.np);
  MB_REQUIRE(workspace_bytes >= s.bytes, MB_ERR_ARG, "linear_cross_entropy_train: %lld bytes of workspace needed, got %lld",
             (long long)s.bytes, (long long)workspace_bytes);
  return dtype == MB_F32 ? once<float>(c, s, loss, dx, dw) : once<__nv_bfloat16>(c, s, loss, dx, dw);
}

extern "C" int motif_b200_scale_gradients(const void* a, void* a_out, int64_t a_n, const void* b, void* b_out, int64_t b_n,
                                          const float* scale, int dtype, void* stream) {
  using namespace mb;
  MB_REQUIRE(scale && a_n >= 0 && b_n >= 0 && (a_n == 0 || (a && a_out)) && (b_n == 0 || (b && b_out)), MB_ERR_ARG,
             "scale_gradients: null pointer or bad size");
  MB_REQUIRE(((uintptr_t)a | (uintptr_t)a_out | (uintptr_t)b | (uintptr_t)b_out) % 16 == 0, MB_ERR_ALIGN,
             "scale_gradients: arrays must be 16-byte aligned");
  MB_REQUIRE(dtype == MB_F32 || dtype == MB_F16 || dtype == MB_BF16, MB_ERR_DTYPE,
             "scale_gradients: unsupported dtype code %d", dtype);
  if (a_n + b_n == 0) return MB_OK;
  const int64_t most = std::max(a_n, b_n) / 8 / 256 + 1;
  const unsigned grid = (unsigned)std::min<int64_t>(most, multiprocessors() * 8);
  auto go = [&](auto t) {
    using T = decltype(t);
    scale_out_kernel<T><<<grid, 256, 0, (cudaStream_t)stream>>>((const T*)a, (T*)a_out, a_n, (const T*)b, (T*)b_out, b_n,
                                                               scale);
    return check_launch("scale_gradients");
  };
  return dtype == MB_F32 ? go(0.f) : dtype == MB_BF16 ? go(__nv_bfloat16{}) : go(__half{});
}
