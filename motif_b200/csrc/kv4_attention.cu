// Chord attention of the newest tokens of every request over its paged 4-bit cache (kv4.cuh).
//
//   logit(r, j) = (scale q_r . k_j - alpha (|j - pos_r - mu| + eps)^beta) ssmax log(pos_r + 1),  j <= pos_r
//
// with k_j = m_j + s_j (c_j - 8) per group of dims, so
//   q . k_j          = sum_groups  s_j (q . c_j - 8 sum(q)) + m_j sum(q)
//   sum_j p_j v_j    = sum_j (p_j s_j) c_j                  + sum_j p_j (m_j - 8 s_j)
// and both products run on the codes themselves.  A code in bits 6..9 of an fp16 IS the number c 2^-18
// (subnormal, exact, and the tensor cores take it as it is), so a packed word becomes matrix operands with
// a shift and an AND per pair and no conversion; the power of two is undone in fp32.  The other operand is
// split into two fp16 parts of 11 bits each (q after a power-of-two normalisation of its row, p s against
// the largest scales that have weight), and the parts are two neighbouring columns of one MMA: with the
// keys on the M side a tile of 4 query rows fills N = 8, a thread's two accumulator columns are the two
// parts of ONE query row, and their sum is the product to 22 bits at no further instruction.  (16-bit
// queries are one part; the sums of the products are the tensor cores', which cut below 24 bits of the
// largest term: see codes().)  The score tile [keys x (row, part)] is the transpose of what the second
// product wants: one movmatrix per 8 keys.  mma.sync and not tcgen05: a kv head has 4 to 16 query rows,
// the operand that comes from memory must be unpacked in registers, and the tensor pipe is busy for a
// fifth of the time as it is.
//
// Work is cut by tiles of 64 keys (128 for D = 32), not by requests: the tiles of all (request, row tile,
// kv head) segments in order are dealt out in equal runs to the CTAs (one per SM) and within them to the
// warps, so requests of any lengths load the GPU evenly, and the lengths may change on the device between
// replays of a CUDA graph.  A segment inside one warp's run is written out by it; one that spans warps is
// joined in shared memory, one that spans CTAs leaves a partial (o, m, l) per CTA, which the merge kernel
// joins in CTA order once it has waited for the workers.  Each warp owns a ring of two tiles in shared
// memory that its first lanes fill with bulk copies (one per tile where a tile lies in one page).
//
// What bounds it: neither the memory nor a pipe, but latency that three warps a scheduler do not hide, each
// of which waits for a tile, scores it, weighs it and takes the second product one after the other.  64
// requests of 8192 tokens (12 / 3 heads of 64, 113 MB): 36.2 us on the GPU, 3.1 TB/s, where the bytes alone
// would take 17.4; 197 warp instructions a unit of 16 keys in all, issue slots 54 % busy, the half-rate
// integer pipe that isolates the codes 51 %, the tensor pipe 18 %.  8 requests, where a warp has one or two
// tiles: 11.5 us.  12 warps of 147 registers: 8 warps 40.5 us; 16 warps 35.7, but 12.5 against 11.5 for 8
// requests; 128-key tiles on 8 warps 38.7.  48 ragged requests of up to 5000 tokens, 4 new ones each, 16
// query rows on 4 fp16 kv heads of 128 (54 MB): 46.1 us, in two passes of 8 rows.
#include <math.h>

#include "common.cuh"
#include "kv4.cuh"

namespace mb {
namespace {

using kv4::kUnit;
using kv4::Layout;

__device__ unsigned int g_kv4_wait_timeouts = 0;

constexpr int kStages = 2;
constexpr uint32_t kWaitLimit = 1u << 20;
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kSlack = 4.f;  // log 2 units
constexpr int kLift = 60;       // the most that a row's weights are lifted by, log 2

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
  kv4::PageDiv by;
  int most;                 // tokens that a row of the table can name
  int64_t pages;
  int ctas;
  bool fail;                // a test: the waits of every third CTA run out at once
  float scale, eps;
};

// 64 keys: a tile's independent chains are what hides latency beside two or three warps a scheduler.
// D = 128 on 32 keys and 12 warps 46.2 us against 42.3 on 64 keys and 8 (32 requests of 8192 tokens, 4 kv
// heads); D = 32 on 64 keys 29.1 against 27.0 on 128 (64 requests of 8192, 3 kv heads).
template <int D>
struct Tile {
  static constexpr int kUnits = D == 32 ? 8 : 4;
  static constexpr int kKeys = kUnits * kUnit;
  static constexpr int kBytes = kUnits * Layout<D>::kBytes;
};

// ------------------------------------------------------------------ the cut into workers
// Lengths are clamped to what the table can name; a request without query rows has no tiles.
__device__ __forceinline__ int length_of(const Args& a, int b) { return max(0, min(a.lens[b], a.most)); }
__device__ __forceinline__ int queries_of(const Args& a, int b) {
  return a.q_lens ? min(max(a.q_lens[b], 0), a.T) : a.T;
}
template <int KT>
__device__ __forceinline__ int tiles_of(const Args& a, int b) {
  return queries_of(a, b) > 0 ? (int)((uint32_t)(length_of(a, b) + KT - 1) / KT) : 0;
}

// The requests' tiles, by one warp: lane i counts those of the i-th run of `run` requests.
struct Requests {
  int run;
  int upto;   // tiles of this lane's run and the ones before it
  int mine;
  int total;  // tiles of all segments (the host keeps this below 2^31)
};
__device__ __forceinline__ int warp_scan(int v) {  // inclusive
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int u = __shfl_up_sync(0xffffffffu, v, o);
    if ((int)(threadIdx.x & 31) >= o) v += u;
  }
  return v;
}
template <int KT>
__device__ __forceinline__ Requests scan_requests(const Args& a) {
  Requests q;
  const int lane = threadIdx.x & 31;
  q.mine = 0;
  if (a.B <= 128) {
    q.run = (a.B + 31) / 32;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int b = lane * q.run + i;
      if (i < q.run && b < a.B) q.mine += tiles_of<KT>(a, b);
    }
  } else {
    // 32 neighbouring requests at a time (a lane reading a run of its own would spread every load over
    // as many lines): the sum of a group goes to the lane whose run it lies in
    const int groups = (a.B + 31) / 32, each = (groups + 31) / 32;
    q.run = 32 * each;
    for (int i0 = 0; i0 < groups; i0 += 8) {
      int len[8], nq[8];  // asked for together
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int b = 32 * (i0 + i) + lane;
        len[i] = b < a.B ? a.lens[b] : 0;
        nq[i] = a.q_lens && b < a.B ? a.q_lens[b] : a.T;
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const uint32_t t = nq[i] > 0 ? (uint32_t)(max(0, min(len[i], a.most)) + KT - 1) / KT : 0u;
        const int sum = (int)__reduce_add_sync(0xffffffffu, t);
        if ((i0 + i) / each == lane) q.mine += sum;
      }
    }
  }
  q.upto = warp_scan(q.mine);
  q.total = __shfl_sync(0xffffffffu, q.upto, 31) * a.Z * a.Hkv;
  return q;
}

// `total` tiles over at most `n` CTAs, at least four each (one for a warp of every scheduler): the
// first CTAs take one more than the others.
struct Cut {
  int working, each, more;
  __device__ __forceinline__ Cut(int total, int n) {
    working = min(n, (total + 3) / 4);
    each = working ? total / working : 0;
    more = total - each * working;
  }
  __device__ __forceinline__ int start(int c) const { return each * c + min(c, more); }
  __device__ __forceinline__ int cta_of(int x) const {
    const int wide = more * (each + 1);
    return x < wide ? x / (each + 1) : more + (x - wide) / each;
  }
};

// A place in the order of tiles: request, segment of it (z * Hkv + kv head), tile of the segment.
struct Cursor {
  int b, seg, k, nt;
};

template <int KT>
__device__ __forceinline__ Cursor locate(const Args& a, const Requests& q, int x) {
  const int zh = a.Z * a.Hkv, lane = threadIdx.x & 31;
  // the first run whose tiles reach past x
  const int c = __popc(__ballot_sync(0xffffffffu, q.upto * zh <= x));
  int left = x - __shfl_sync(0xffffffffu, q.upto - q.mine, c) * zh;
  Cursor u;
  u.b = c;
  u.nt = __shfl_sync(0xffffffffu, q.mine, c);
  if (q.run > 1) {
    for (int i0 = 0; i0 < q.run; i0 += 32) {
      const int b = c * q.run + i0 + lane;
      const int t = i0 + lane < q.run && b < a.B ? tiles_of<KT>(a, b) : 0;
      const int upto = warp_scan(t);
      const int n = __popc(__ballot_sync(0xffffffffu, upto * zh <= left));
      if (n < 32) {
        left -= __shfl_sync(0xffffffffu, upto - t, n) * zh;
        u.b = c * q.run + i0 + n;
        u.nt = __shfl_sync(0xffffffffu, t, n);
        break;
      }
      left -= __shfl_sync(0xffffffffu, upto, 31) * zh;
    }
  }
  u.seg = left / u.nt;
  u.k = left - u.seg * u.nt;
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

// The row tile and kv head of a segment, and the new token and head (within the kv head's group) of
// query row r.
__device__ __forceinline__ void split_segment(const Args& a, int seg, int& z, int& hk) {
  z = a.Z == 1 ? 0 : seg / a.Hkv;
  hk = seg - z * a.Hkv;
}
__device__ __forceinline__ void split_row(const Args& a, int r, int& t, int& gi) {
  t = a.T == 1 ? 0 : r / a.G;
  gi = r - t * a.G;
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

// x^b, b != 0, for fp32 tensors: log2 x as a whole number e and log2 f of f = x 2^-e in 0.75 .. 1.5, b e
// with its rounding error kept, and 2^(b log2 x) from the fraction of b e, so that the fast logarithm's
// and power's errors (2^-22 absolute and relative) are all there is, however large log2 x.  At x = 0 (no
// eps, a key at mu) it is 0 or, for b < 0, infinite.
__device__ __forceinline__ float power(float x, float b) {
  const int e = (int)(__float_as_uint(x) - 0x3f400000u) >> 23;
  const float f = __uint_as_float(__float_as_uint(x) - ((uint32_t)e << 23)), fe = (float)e;
  const float t = b * fe, lost = fmaf(b, fe, -t);
  const float n = rintf(t);
  const float y = ex2f_((t - n) + fmaf(b, lg2_(f), lost));
  return x == 0.f ? (b > 0.f ? 0.f : INFINITY) : y * pow2((int)fminf(fmaxf(n, -126.f), 127.f));
}

// D = A B + C on fp16 operands with C in registers of its own.
__device__ __forceinline__ void mma_f16(float* d, const uint32_t* a, const uint32_t* b, float c0, float c1, float c2,
                                        float c3) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
      "{%10,%11,%12,%13};\n"
      : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b[0]), "r"(b[1]), "f"(c0), "f"(c1), "f"(c2), "f"(c3));
}

// The nibbles of w as four fp16 pairs, nibbles (0, 4), (1, 5), (2, 6) and (3, 7) times U (or kOdd U).  For 16-bit
// tensors they stay the subnormal numbers that the masked bits are (U = 2^-18).  The tensor cores align
// the products of a step by their operands' exponent fields and cut below 24 bits; a subnormal's field
// stands for its bit 9, so the codes are shifted to end there, which leaves the sums all but the bits of
// 8 sum(q) against q . c.  In bits 0..3 and 4..7, without most of the shifts, the sums kept 17 bits and 64
// requests of 8192 took 33.0 us where they took 35.2; distance from 64 bits before the last rounding (16
// requests of 8192, fp16) 2.0e-5 there, 9.5e-7 here, and 1.1e-6 for elementary operations in fp32.  fp32
// tensors make them normal numbers c - 8 (U = 1: the bits of 1024 or-ed in, 1024 + 8 U taken off; where
// they lie in the word does not matter then, and the odd nibbles come out 16 times as large) at one more
// instruction a pair, and need the sums less 8 no more; for 16-bit ones that took 39.5 us.  Nearly all of
// the distance is the second product's; the first one's shows where logits are sharp (ten times as large, D
// = 32: 8.7e-6 against 5.6e-7 with its codes in bits 0..3 and 4..7, at 35.3 us; fp32 operations 4.8e-7).
template <bool EXACT>
__device__ __forceinline__ void codes(uint32_t w, uint32_t* h) {
  if constexpr (EXACT) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t v = (i < 2 ? w : w >> 8) & (i & 1 ? 0x00f000f0u : 0x000f000fu);
      asm("add.rn.f16x2 %0, %1, %2;" : "=r"(h[i]) : "r"(v | 0x64006400u), "r"(i & 1 ? 0xe480e480u : 0xe408e408u));
    }
  } else {
    constexpr uint32_t kBits = 0x03c003c0u;
    h[0] = (w << 6) & kBits;
    h[1] = (w << 2) & kBits;
    h[2] = (w >> 2) & kBits;
    h[3] = (w >> 6) & kBits;
  }
}

// Eight consecutive elements at a 16-byte aligned address.
template <typename T>
__device__ __forceinline__ void load8(const T* p, float* x) {
  if constexpr (sizeof(T) == 4) {
    const float4 a = *reinterpret_cast<const float4*>(p), b = *reinterpret_cast<const float4*>(p + 4);
    x[0] = a.x, x[1] = a.y, x[2] = a.z, x[3] = a.w, x[4] = b.x, x[5] = b.y, x[6] = b.z, x[7] = b.w;
  } else {
    const uint4 a = *reinterpret_cast<const uint4*>(p);
    const T* h = reinterpret_cast<const T*>(&a);
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = to_f(h[i]);
  }
}
// Four neighbouring outputs y f (zeros where the row sees no key); the host asks for rows of out on
// 16-byte boundaries.
template <typename T>
__device__ __forceinline__ void store4(T* p, float4 y, float f, bool sees) {
  const float4 v = sees ? make_float4(y.x * f, y.y * f, y.z * f, y.w * f) : make_float4(0.f, 0.f, 0.f, 0.f);
  if constexpr (sizeof(T) == 4) *reinterpret_cast<float4*>(p) = v;
  else *reinterpret_cast<uint2*>(p) = make_uint2(pack2<T>(v.x, v.y), pack2<T>(v.z, v.w));
}

// Place of row r of a group of 8 keys: rows 2t, 2t + 1 are keys t, t + 4, so that the four lanes of a
// V load take neighbouring keys (128 consecutive bytes of shared memory per load).
__device__ __forceinline__ int key_of_row(int r) { return (r >> 1) + 4 * (r & 1); }

// Zeroes the rows of every n-th request without tiles.
template <typename T, int D>
__device__ __forceinline__ void zero_rows(T* out, const Args& a) {
  for (int e = blockIdx.x; e < a.B; e += gridDim.x) {
    if (tiles_of<Tile<D>::kKeys>(a, e) > 0) continue;
    for (int i = threadIdx.x; i < a.H * a.T * (D / 4); i += blockDim.x) {
      const int row = i / (D / 4), h = row / a.T;
      store4(out + e * a.st.s[3] + h * a.st.s[4] + (row - h * a.T) * a.st.s[5] + i % (D / 4) * 4,
             make_float4(0.f, 0.f, 0.f, 0.f), 0.f, false);
    }
  }
}

// ------------------------------------------------------------------ the worker kernel
// Warps of the one CTA an SM runs, by the registers and the ring that the output tile leaves them (8 query
// rows of D = 128 on 12 warps and 32 keys spill: 53.3 us against 46.1; so do 16 rows of D = 64: 113
// against 77).
__host__ __device__ constexpr int warps_of(int nt, int D) { return nt <= 2 && D <= 64 ? 12 : 8; }

// An unfinished piece of a segment at the end of a warp's run: [RT rows][D + 4] floats (o, m, l), its
// segment, whether it holds the segment's first / last tile, the tiles that follow it in the segment, and
// the new tokens and first position of the request.
struct Piece {
  int b, seg;  // b < 0: none
  int begins, ends, more, nq, base;
};
// What a worker CTA leaves to the merge beside its partials: the segment that begins in its run and goes
// on in the next ones, in how many CTAs it lies, and the new tokens and first position of its request.
struct alignas(16) Open {
  int parts, b, seg, nq, base;  // parts 0: none
  int pad[3];
};
__host__ __device__ constexpr int piece_floats(int nt, int64_t D) { return 4 * nt * ((int)D + 4); }
template <int D, int NT>
__host__ __device__ constexpr int piece_floats() {
  return piece_floats(NT, D);
}
// The workspace: two partials of every CTA, then an Open of each.
template <int D, int NT>
__device__ __forceinline__ Open* open_of(const Args& a, int cta) {
  return reinterpret_cast<Open*>(a.ws + (int64_t)a.ctas * 2 * piece_floats<D, NT>()) + cta;
}
// A warp's last piece takes its ring's place, which is free by then; one that a segment from before
// the run leaves on the way needs its own.
template <int D, int NT>
constexpr int attention_smem() {
  static_assert(piece_floats<D, NT>() * 4 <= kStages * Tile<D>::kBytes, "a piece fits the ring");
  return warps_of(NT, D) * (kStages * Tile<D>::kBytes + piece_floats<D, NT>() * 4);
}

// A CTA's `count` tiles over its W warps: warp w's run starts at tile run_start(count, w).  Fewer
// tiles than warps go to the first ones, one of each scheduler in turn.
template <int W>
__device__ __forceinline__ int run_start(int count, int w) {
  return count <= W ? min(w, count) : (int)((int64_t)count * w / W);
}

template <typename T, int D, int NT>
__global__ void __launch_bounds__(32 * warps_of(NT, D), 1)
    kv4_attention_kernel(const T* __restrict__ q, T* __restrict__ out, const Args a) {
  constexpr int kWarps = warps_of(NT, D);
  using L = Layout<D>;
  constexpr int TU = Tile<D>::kUnits, KT = Tile<D>::kKeys;
  constexpr int NG = L::NG, DG = L::DG;
  constexpr int KW = DG / 32;        // 32-bit words of K codes of a thread per row and group
  constexpr int MT = DG / 16;        // 16-dim output tiles of a group
  constexpr int RT = 4 * NT;         // query rows of a row tile
  constexpr bool EXACT = sizeof(T) == 4;
  constexpr int kUnitBits = EXACT ? 0 : 18;  // codes enter the products times 2^-kUnitBits,
  constexpr float kOdd = EXACT ? 16.f : 1.f;  // those of odd nibbles times kOdd as well
  // 16-bit queries have no low part: with 8 rows or more every column of the first product is a row,
  // a thread holding rows 2 t4 and 2 t4 + 1 of each 8; else row t4 of each 4, its parts in two columns
  constexpr bool WIDE = !EXACT && NT > 1;
  constexpr int QT = WIDE ? NT / 2 : NT;  // column tiles of the first product
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ __align__(8) uint64_t bars[kWarps][kStages];
  __shared__ Piece pieces[kWarps][2];
  __shared__ int s_total;

  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int g8 = lane >> 2, t4 = lane & 3;
  auto row_of = [&](int n) { return WIDE ? (n >> 1) * 8 + 2 * t4 + (n & 1) : n * 4 + t4; };  // in the row tile
  uint8_t* ring = smem + warp * (kStages * Tile<D>::kBytes);
  auto piece_at = [&](int w, int which) {
    return reinterpret_cast<float*>(which ? smem + w * (kStages * Tile<D>::kBytes)
                                          : smem + kWarps * (kStages * Tile<D>::kBytes) + w * piece_floats<D, NT>() * 4);
  };
  uint64_t* bar = bars[warp];
  if (lane == 0) {
    for (int s = 0; s < kStages; ++s) mbar_init(&bar[s], 1);
    mbar_init_fence();
    pieces[warp][0].b = pieces[warp][1].b = -1;
  }
  kv4::wait_for_previous();
  allow_dependent_launch();  // the merge, which waits for the end of this grid before it touches memory
  const Requests reqs = scan_requests<KT>(a);
  const Cut cut(reqs.total, gridDim.x);
  if ((int)blockIdx.x >= cut.working) {
    if (threadIdx.x == 0) open_of<D, NT>(a, blockIdx.x)->parts = 0;
    zero_rows<T, D>(out, a);
    return;
  }
  if (threadIdx.x == 0) s_total = reqs.total;
  const int cta_first = cut.start(blockIdx.x), cta_count = cut.each + ((int)blockIdx.x < cut.more ? 1 : 0);
  const int run0 = run_start<kWarps>(cta_count, warp);
  const int count = run_start<kWarps>(cta_count, warp + 1) - run0;

  bool failed = false;
  const uint32_t polls = a.fail && blockIdx.x % 3 == 1 ? 0 : kWaitLimit;
  if (count > 0) {
    Cursor cur = locate<KT>(a, reqs, cta_first + run0);

    // The tile to be copied next: its page of this lane's unit (lanes 0 .. TU - 1) is looked up one
    // tile before the copy is issued.
    const int UP = a.by.P / kUnit;
    const bool one_copy = UP % TU == 0;  // a tile's units lie in one page, next to each other
    const int step_page = a.by(KT), step_sub = TU - step_page * UP;
    const int page0 = a.by(lane * kUnit), sub0 = lane - page0 * UP;
    Cursor ahead = cur;
    int a_len = length_of(a, ahead.b), a_z, a_head;
    split_segment(a, ahead.seg, a_z, a_head);
    int a_page = a.by((ahead.k * TU + lane) * kUnit), a_sub = ahead.k * TU + lane - a_page * UP;
    const int32_t* a_row = a.table + (int64_t)ahead.b * a.ts;
    struct Look {
      int pid, head, sub;  // pid -1: no such unit
    };
    auto look = [&]() {
      Look f = {-1, a_head, a_sub};
      if (lane < TU && (ahead.k * TU + lane) * kUnit < a_len) f.pid = a_row[a_page];
      return f;
    };
    auto step = [&]() {
      if (advance<KT>(a, ahead)) {
        split_segment(a, ahead.seg, a_z, a_head);
        a_len = length_of(a, ahead.b);
        a_row = a.table + (int64_t)ahead.b * a.ts;
        a_page = page0, a_sub = sub0;
      } else {
        a_page += step_page, a_sub += step_sub;
        if (a_sub >= UP) a_sub -= UP, ++a_page;
      }
      return look();
    };
    uint32_t valid = 0;  // units that are there, TU bits per stage
    auto issue = [&](int s, const Look& f) {
      const bool ok = f.pid >= 0 && f.pid < a.pages;
      const uint32_t mask = __ballot_sync(0xffffffffu, ok);
      valid = (valid & ~(((1u << TU) - 1) << (TU * s))) | (mask << (TU * s));
      const uint32_t bytes = __popc(mask) * L::kBytes;
      if (lane == 0) mbar_arrive_expect_tx(&bar[s], bytes);
      __syncwarp();
      if (ok && (lane == 0 || !one_copy))
        bulk_load(ring + s * Tile<D>::kBytes + lane * L::kBytes,
                  a.pool + (((int64_t)f.pid * a.Hkv + f.head) * UP + f.sub) * (int64_t)L::kBytes,
                  one_copy ? bytes : L::kBytes, &bar[s]);
    };
    Look next = look();
    int looked = 0;  // tiles issued

    // state of the current segment
    uint32_t qf[QT][NG][2 * KW][2];
    float sq[NT][NG], qr[NT], ar[NT], be[NT], mh[NT];
    int pos[NT];
    // weights are taken against a reference that a row's logits exceed by limit[n] at most, kSlack more
    // than the row's lift: it moves when a tile goes beyond that, not with every new maximum
    float o[NT][NG][MT][4], ref[NT], limit[NT];
    float2 l[NT], pm[NT][NG];  // of the thread's keys of rows 0 .. 7 and 8 .. 15 of the units
    // o holds p s 2^(10 - ve), ve the exponent of the largest V scale so far.  Where the keys that have
    // weight have scales more than 2^12 below it, the row's weights are all 2^lift larger, so that the
    // fp16 parts of p s keep their 22 bits; a tile whose scales reach vtop looks again
    int ve = 0;
    float vup = 0.f, vtop = 0.f;  // 2^(10 - ve), the least 2^(ve + 1 - lift) (0: no tile yet)
    int lo_pos = 0;    // smallest position of a row that sees keys
    int nq = 0, base = 0, len = 0;
    const float kf = (float)key_of_row(g8);

    bool fresh = true, from_start = true;
    int s = 0, phase = 0;
    for (int i = 0; i < count; ++i) {
      if (fresh) {
        fresh = false;
        from_start = cur.k == 0;
        int z, hk;
        split_segment(a, cur.seg, z, hk);
        len = length_of(a, cur.b);
        nq = queries_of(a, cur.b);
        base = len - nq;
        ve = -110;
        vup = pow2(120);
        vtop = 0.f;
        const int rows = a.G * a.T;
        int t, gi;
        split_row(a, z * RT, t, gi);
        lo_pos = max(0, base + t);
        float x[QT][NG][8 * KW];
#pragma unroll
        for (int n = 0; n < QT; ++n) {
          // the query row of this thread's B fragments: column g8 = row g8, or (row g8 / 2, part g8 & 1)
          split_row(a, min(z * RT + (WIDE ? n * 8 + g8 : n * 4 + (g8 >> 1)), rows - 1), t, gi);
          const T* qp = q + cur.b * a.st.s[0] + (hk * a.G + gi) * a.st.s[1] + t * a.st.s[2];
#pragma unroll
          for (int g = 0; g < NG; ++g)
#pragma unroll
            for (int w = 0; w < KW; ++w) load8(qp + g * DG + t4 * 8 * KW + 8 * w, x[n][g] + 8 * w);
        }
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          // the query row whose scores this thread holds; logits in units of log 2
          split_row(a, min(z * RT + row_of(n), rows - 1), t, gi);
          const int h = hk * a.G + gi;
          pos[n] = max(0, base + min(t, nq - 1));
          qr[n] = a.ssmax[h];
          ar[n] = a.alpha[h];
          be[n] = a.beta[h];
          mh[n] = be[n] == 0.f ? 0.5f : -a.mu[h];  // x^0 is 1 for x = 0 too (no eps): any other place will do
        }
        if (i == 0) {
          // the first copies go out after the loads above, which would wait behind every warp's copies
          issue(0, next);
          looked = 1;
          if (count > 1) next = step();
        }
        float sums[QT][NG];
        int exps[QT];
#pragma unroll
        for (int n = 0; n < QT; ++n) {
          float top = 0.f;
#pragma unroll
          for (int g = 0; g < NG; ++g)
#pragma unroll
            for (int e = 0; e < 8 * KW; e += 2) top = fmax3(top, fabsf(x[n][g][e]), fabsf(x[n][g][e + 1]));
          top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
          top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
          // power of two that brings the row's largest value to 2^13 .. 2^14 (fp16 ends at 2^16)
          exps[n] = min(max((int)(__float_as_uint(top) >> 23) - 127, -112), 127);
          const float up = pow2(13 - exps[n]);
#pragma unroll
          for (int g = 0; g < NG; ++g) {
            float2 sum = make_float2(0.f, 0.f);
#pragma unroll
            for (int w = 0; w < KW; ++w)
#pragma unroll
              for (int p = 0; p < 4; ++p) {
                const float2 y = fmul2(make_float2(x[n][g][8 * w + p], x[n][g][8 * w + p + 4]), make_float2(up, up));
                sum = fadd2(sum, y);
                const float2 v = p & 1 ? fmul2(y, make_float2(1.f / kOdd, 1.f / kOdd)) : y;
                uint32_t f = pack2<__half>(v.x, v.y);
                if (!WIDE && (g8 & 1)) {  // the low part; values of 16 bits have none
                  const float2 hi = __half22float2(*reinterpret_cast<__half2*>(&f));
                  f = EXACT ? pack2<__half>(v.x - hi.x, v.y - hi.y) : 0u;
                }
                qf[n][g][2 * w + (p >> 1)][p & 1] = f;
              }
            sums[n][g] = sum.x + sum.y;
            sums[n][g] += __shfl_xor_sync(0xffffffffu, sums[n][g], 1);
            sums[n][g] += __shfl_xor_sync(0xffffffffu, sums[n][g], 2);
          }
        }
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          const int qt = WIDE ? n >> 1 : n, from = WIDE ? 4 * (2 * t4 + (n & 1)) : 8 * t4;
#pragma unroll
          for (int g = 0; g < NG; ++g) sq[n][g] = __shfl_sync(0xffffffffu, sums[qt][g], from) * pow2(-kUnitBits);
          const int exr = __shfl_sync(0xffffffffu, exps[qt], from);
          const float rc = qr[n] * logf((float)pos[n] + 1.f) * kLog2e;
          qr[n] = a.scale * rc * pow2(kUnitBits - 13) * pow2(exr);
          ar[n] *= -rc;
          ref[n] = 0.f;
          limit[n] = -INFINITY;
          l[n] = make_float2(0.f, 0.f);
#pragma unroll
          for (int g = 0; g < NG; ++g) {
            pm[n][g] = make_float2(0.f, 0.f);
#pragma unroll
            for (int t = 0; t < MT; ++t) o[n][g][t][0] = o[n][g][t][1] = o[n][g][t][2] = o[n][g][t][3] = 0.f;
          }
        }
      }

      if (i == 0 && count > 1) {
        issue(1, next);
        looked = 2;
        if (count > 2) next = step();
      }
      // never expected to run out: nothing more is asked for then, and what is on its way may still land
      if (__any_sync(0xffffffffu, !mbar_wait_bounded(&bar[s], (uint32_t)phase, polls))) {
        failed = true;
        mbar_wait_bounded(&bar[s], (uint32_t)phase, kWaitLimit);
        static_assert(kStages == 2, "one other stage");
        if (looked > i + 1) mbar_wait_bounded(&bar[s ^ 1], (uint32_t)(phase ^ s), kWaitLimit);
        break;
      }
      const uint8_t* tile = ring + s * Tile<D>::kBytes;
      const uint32_t units = (valid >> (TU * s)) & ((1u << TU) - 1);
      const int k0 = cur.k * KT;

      {
        const int r0 = key_of_row(g8);
        float2 x[NT][TU];
        float2 gap[NT];  // key - pos: a whole number, exact
        float top[NT];
        uint32_t vp[TU][NG][2];
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          const float d = (float)(k0 - pos[n]) + kf;
          gap[n] = make_float2(d, d + 8.f);
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
            float acc[QT][4];
#pragma unroll
            for (int w = 0; w < KW; ++w) {
              uint32_t c0[4], c1[4];
              codes<EXACT>(w0[w], c0);
              codes<EXACT>(w1[w], c1);
#pragma unroll
              for (int p = 0; p < 2; ++p) {
                const uint32_t af[4] = {c0[2 * p], c1[2 * p], c0[2 * p + 1], c1[2 * p + 1]};
#pragma unroll
                for (int n = 0; n < QT; ++n) {
                  if (w == 0 && p == 0) {
                    const float s0 = EXACT ? 0.f : -8.f * sq[WIDE ? 2 * n : n][g];
                    const float s1 = WIDE ? -8.f * sq[WIDE ? 2 * n + 1 : n][g] : 0.f;
                    mma_f16(acc[n], af, qf[n][g][0], s0, s1, s0, s1);
                  } else {
                    mma_16816<__half>(acc[n], af, qf[n][g][2 * w + p]);
                  }
                }
              }
            }
            const uint32_t* kp = reinterpret_cast<const uint32_t*>(unit + L::kKp) + g * kUnit + r0;
            const uint32_t p0 = kp[0], p1 = kp[8];
            const uint32_t* vq = reinterpret_cast<const uint32_t*>(unit + L::kVp) + g * kUnit + r0;
            vp[u][g][0] = vq[0], vp[u][g][1] = vq[8];
            const float2 ks = make_float2(kv4::pair_scale(p0), kv4::pair_scale(p1));
            const float2 km = make_float2(kv4::pair_centre(p0), kv4::pair_centre(p1));
#pragma unroll
            for (int n = 0; n < NT; ++n) {
              const float2 s2 = make_float2(sq[n][g], sq[n][g]);
              const float* c = acc[WIDE ? n >> 1 : n];
              const float2 both = WIDE ? make_float2(c[n & 1], c[2 + (n & 1)]) : make_float2(c[0] + c[1], c[2] + c[3]);
              dot[n] = g ? ffma2(ks, both, ffma2(km, s2, dot[n])) : ffma2(ks, both, fmul2(km, s2));
            }
          }
#pragma unroll
          for (int n = 0; n < NT; ++n) {
            const float2 off = fadd2(gap[n], make_float2(mh[n], mh[n]));
            if (u + 1 < TU) gap[n] = fadd2(gap[n], make_float2(16.f, 16.f));
            const float2 dist = make_float2(fabsf(off.x) + a.eps, fabsf(off.y) + a.eps);
            float2 pw;
            if constexpr (sizeof(T) == 4) {
              pw = make_float2(power(dist.x, be[n]), power(dist.y, be[n]));
            } else {
              const float2 ln = fmul2(make_float2(lg2_(dist.x), lg2_(dist.y)), make_float2(be[n], be[n]));
              pw = make_float2(ex2f_(ln.x), ex2f_(ln.y));
            }
            x[n][u] = ffma2(dot[n], make_float2(qr[n], qr[n]),
                            ffma2(pw, make_float2(ar[n], ar[n]), make_float2(-ref[n], -ref[n])));
          }
        }
        if (units != (1u << TU) - 1 || k0 + KT - 1 > lo_pos) {
          // keys that a row does not see weigh nothing; a slot that holds no token may hold any pair,
          // which must not meet the weight 0
          float all = 0.f;
#pragma unroll
          for (int u = 0; u < TU; ++u)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              const int key = k0 + u * kUnit + r0 + 8 * e;
              const bool there = (units >> u) & 1u;
#pragma unroll
              for (int n = 0; n < NT; ++n)
                if (!there || key > pos[n]) (e ? x[n][u].y : x[n][u].x) = -INFINITY;
#pragma unroll
              for (int g = 0; g < NG; ++g) {
                if (!there || key >= len) vp[u][g][e] = 0u;
                all += kv4::pair_scale(vp[u][g][e]) + kv4::pair_centre(vp[u][g][e]);
              }
            }
          if (!(fabsf(all) < INFINITY)) {
            // nor may the pair of a group that is no number: it goes by itself to the sums of the rows that
            // see its key
#pragma unroll
            for (int u = 0; u < TU; ++u)
#pragma unroll
              for (int e = 0; e < 2; ++e)
#pragma unroll
                for (int g = 0; g < NG; ++g) {
                  const float any = kv4::pair_scale(vp[u][g][e]) + kv4::pair_centre(vp[u][g][e]);
                  if (fabsf(any) < INFINITY) continue;
                  vp[u][g][e] = 0u;
#pragma unroll
                  for (int n = 0; n < NT; ++n)
                    if (k0 + u * kUnit + r0 + 8 * e <= pos[n]) (e ? pm[n][g].y : pm[n][g].x) += any;
                }
          }
        }
        float big = 0.f;
#pragma unroll
        for (int u = 0; u < TU; ++u)
#pragma unroll
          for (int g = 0; g < NG; ++g) big = fmax3(big, kv4::pair_scale(vp[u][g][0]), kv4::pair_scale(vp[u][g][1]));
        bool beyond = big >= vtop;
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          top[n] = -INFINITY;
#pragma unroll
          for (int u = 0; u < TU; ++u) top[n] = fmax3(top[n], x[n][u].x, x[n][u].y);
          beyond = beyond || top[n] > limit[n];
        }
        if (__any_sync(0xffffffffu, beyond)) {
          // p s 2^(10 - ve) stays below 2^(kSlack + 11), weights and what they are multiplied with in range
          const int most = (int)(__reduce_max_sync(0xffffffffu, __float_as_uint(big)) >> 23) - 127;
          const int vn = max(ve, most);
          const float vdown = pow2(max(ve - vn, -126));
          float small = INFINITY, lifted = kSlack;
#pragma unroll
          for (int u = 0; u < TU; ++u)
#pragma unroll
            for (int g = 0; g < NG; ++g)
              small = fminf(small, fminf(kv4::pair_scale(vp[u][g][0]), kv4::pair_scale(vp[u][g][1])));
#pragma unroll
          for (int n = 0; n < NT; ++n) {
            lifted = fmaxf(lifted, limit[n]);
#pragma unroll
            for (int d = 4; d < 32; d <<= 1) top[n] = fmaxf(top[n], __shfl_xor_sync(0xffffffffu, top[n], d));
          }
          auto move = [&](int n, float up) {
            const float f = limit[n] == -INFINITY ? 1.f : exp2f(-up);  // the first keys: the sums are still 0
            ref[n] += up;
            const float2 f2 = make_float2(f, f), fo = make_float2(f * vdown, f * vdown);
            l[n] = fmul2(l[n], f2);
#pragma unroll
            for (int g = 0; g < NG; ++g) {
              pm[n][g] = fmul2(pm[n][g], f2);
#pragma unroll
              for (int t = 0; t < MT; ++t)
#pragma unroll
                for (int e = 0; e < 4; e += 2) {
                  const float2 y = fmul2(make_float2(o[n][g][t][e], o[n][g][t][e + 1]), fo);
                  o[n][g][t][e] = y.x, o[n][g][t][e + 1] = y.y;
                }
            }
#pragma unroll
            for (int u = 0; u < TU; ++u) x[n][u] = fadd2(x[n][u], make_float2(-up, -up));
          };
          // scales within 2^12 of each other need no lift, whatever the weights
          const bool apart = small * 4096.f < pow2(min(vn, 127)) || lifted > kSlack || (vn > ve && vtop > 0.f);
          if (!__any_sync(0xffffffffu, apart)) {
            vtop = pow2(min(vn, 126) + 1);
#pragma unroll
            for (int n = 0; n < NT; ++n) {
              move(n, top[n] > limit[n] ? top[n] : 0.f);
              if (top[n] > limit[n]) limit[n] = kSlack;
            }
          } else {
            vtop = pow2(min(vn, 126) + 1);
#pragma unroll
            for (int n = 0; n < NT; ++n) {
              const bool first = limit[n] == -INFINITY, moves = top[n] > limit[n];
              const float was = first ? 0.f : limit[n] - kSlack, at = moves ? top[n] : was;
              float heavy = 0.f;  // the largest weighted scale of this tile
#pragma unroll
              for (int u = 0; u < TU; ++u) {
                float2 vs = make_float2(kv4::pair_scale(vp[u][0][0]), kv4::pair_scale(vp[u][0][1]));
                if constexpr (NG == 2)
                  vs = make_float2(fmaxf(vs.x, kv4::pair_scale(vp[u][1][0])),
                                   fmaxf(vs.y, kv4::pair_scale(vp[u][1][1])));
                heavy = fmax3(heavy, ex2f_(x[n][u].x - at) * vs.x, ex2f_(x[n][u].y - at) * vs.y);
              }
#pragma unroll
              for (int d = 4; d < 32; d <<= 1) heavy = fmaxf(heavy, __shfl_xor_sync(0xffffffffu, heavy, d));
              // the exponent that the row needs, which falls no faster than its sums do
              int need = heavy > 0.f ? min(most, (int)(__float_as_uint(heavy) >> 23) - 127 + 12) : first ? vn : -127;
              if (!first) need = max(need, ve - (int)was - (int)fminf(at - was, 256.f));
              const int lift = vn > 100 || (first && !moves) ? 0 : min(max(vn - need, 0), kLift);
              vtop = fminf(vtop, pow2(min(vn - lift, 126) + 1));
              move(n, first && !moves ? 0.f : at - (float)lift);
              if (!first || moves) limit[n] = kSlack + (float)lift;
            }
          }
          ve = vn;
          vup = pow2(10 - vn);
        }
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int u = 0; u < TU; ++u) {
            const float2 y = x[n][u];
            x[n][u] = sizeof(T) == 4 ? make_float2(exp2f(y.x), exp2f(y.y)) : make_float2(ex2f_(y.x), ex2f_(y.y));
            l[n] = fadd2(l[n], x[n][u]);
          }

#pragma unroll
        for (int u = 0; u < TU; ++u) {
          const uint8_t* unit = tile + u * L::kBytes;
#pragma unroll
          for (int g = 0; g < NG; ++g) {
            const float2 vs = make_float2(kv4::pair_scale(vp[u][g][0]), kv4::pair_scale(vp[u][g][1]));
            const float2 vc = make_float2(kv4::pair_centre(vp[u][g][0]), kv4::pair_centre(vp[u][g][1]));
            const float2 vm = EXACT ? vc : ffma2(vs, make_float2(-8.f, -8.f), vc);
            const float2 vn2 = fmul2(vs, make_float2(vup, vup));
            uint32_t bf[NT][2];
#pragma unroll
            for (int n = 0; n < NT; ++n) {
              const float2 ps = fmul2(x[n][u], vn2);
              pm[n][g] = ffma2(x[n][u], vm, pm[n][g]);
              // 11 bits each: the high part is cut off, exactly a number of fp16
              const float2 hi = make_float2(__uint_as_float(__float_as_uint(ps.x) & 0xffffe000u),
                                            __uint_as_float(__float_as_uint(ps.y) & 0xffffe000u));
              const float2 lo = ffma2(hi, make_float2(-1.f, -1.f), ps);
              bf[n][0] = transpose8x8(pack2<__half>(hi.x, lo.x));
              bf[n][1] = transpose8x8(pack2<__half>(hi.y, lo.y));
            }
            const uint8_t* at = unit + L::kV + t4 * L::kRow + g * (DG / 2) + (KW == 2 ? 4 * g8 : 4 * (g8 >> 1));
            uint32_t w[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) w[j] = *reinterpret_cast<const uint32_t*>(at + 4 * j * L::kRow);
#pragma unroll
            for (int hf = 0; hf < KW; ++hf) {  // halves of a word: four dims each
              const uint32_t sel = KW == 2 ? (hf ? 0x7632u : 0x5410u) : ((g8 & 1) ? 0x7632u : 0x5410u);
              uint32_t c0[4], c1[4];
              codes<EXACT>(__byte_perm(w[0], w[1], sel), c0);
              codes<EXACT>(__byte_perm(w[2], w[3], sel), c1);
#pragma unroll
              for (int p = 0; p < 2; ++p) {
                const uint32_t af[4] = {c0[2 * p], c0[2 * p + 1], c1[2 * p], c1[2 * p + 1]};
#pragma unroll
                for (int n = 0; n < NT; ++n) mma_16816<__half>(o[n][g][2 * hf + p], af, bf[n]);
              }
            }
          }
        }
      }

      __syncwarp();  // every lane is done with the stage
      if (looked < count) {
        fence_proxy_async_smem();
        issue(s, next);
        if (++looked < count) next = step();
      }
      if (++s == kStages) s = 0, phase ^= 1;

      const bool ends = cur.k + 1 == cur.nt;
      if (ends || i + 1 == count) {
        int z, hk;
        split_segment(a, cur.seg, z, hk);
        const bool direct = ends && from_start;
        // the run's last piece goes where the ring was
        const int which = i + 1 == count ? 1 : 0;
        float* part = piece_at(warp, which);
        if (!direct && lane == 0) {
          pieces[warp][which].b = cur.b;
          pieces[warp][which].seg = cur.seg;
          pieces[warp][which].begins = from_start;
          pieces[warp][which].ends = ends;
          pieces[warp][which].more = cur.nt - 1 - cur.k;
          pieces[warp][which].nq = nq;
          pieces[warp][which].base = base;
        }
        const float back = pow2(min(ve, 127));  // and 2^(kUnitBits - 10)
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          float ln = l[n].x + l[n].y, pn[NG];
#pragma unroll
          for (int g = 0; g < NG; ++g) pn[g] = pm[n][g].x + pm[n][g].y;
#pragma unroll
          for (int d = 4; d < 32; d <<= 1) {
            ln += __shfl_xor_sync(0xffffffffu, ln, d);
#pragma unroll
            for (int g = 0; g < NG; ++g) pn[g] += __shfl_xor_sync(0xffffffffu, pn[g], d);
          }
          const int r = z * RT + row_of(n);
          int t, gi;
          split_row(a, r, t, gi);
          const bool sees = t < nq && base + t >= 0;
          const float inv = direct ? (sees && ln != 0.f ? 1.f / ln : 0.f) : 1.f;
#pragma unroll
          for (int g = 0; g < NG; ++g) {
            float y[2 * MT];
#pragma unroll
            for (int j = 0; j < MT; ++j) {
              y[2 * j] = fmaf((o[n][g][j][0] + o[n][g][j][1]) * pow2(kUnitBits - 10), back, pn[g]) * inv;
              y[2 * j + 1] = fmaf((o[n][g][j][2] + o[n][g][j][3]) * (pow2(kUnitBits - 10) / kOdd), back, pn[g]) * inv;
            }
            const int d0 = g * DG + g8 * 2 * MT;
            if (direct) {
              if (r < a.G * a.T) {
                T* dst = out + cur.b * a.st.s[3] + (hk * a.G + gi) * a.st.s[4] + t * a.st.s[5] + d0;
#pragma unroll
                for (int j = 0; j < 2 * MT; j += 4)
                  store4(dst + j, make_float4(y[j], y[j + 1], y[j + 2], y[j + 3]), 1.f, sees);
              }
            } else {
              float* dst = part + row_of(n) * (D + 4) + d0;
#pragma unroll
              for (int j = 0; j < 2 * MT; j += 4)
                *reinterpret_cast<float4*>(dst + j) = make_float4(y[j], y[j + 1], y[j + 2], y[j + 3]);
            }
          }
          if (!direct && g8 == 0) {
            part[row_of(n) * (D + 4) + D] = limit[n] == -INFINITY ? -INFINITY : ref[n];
            part[row_of(n) * (D + 4) + D + 1] = ln;
          }
        }
        fresh = true;
      }
      advance<KT>(a, cur);
    }
  }

  zero_rows<T, D>(out, a);  // while other warps are still at work

  // The CTA's pieces in tile order: neighbours of one segment are joined, and written out where the
  // CTA holds all of the segment, else left to the merge (slot 0 where the segment began before this
  // CTA's run, 1 where it began in it).
  if (__syncthreads_or(failed)) {
    // the copies that were on their way had a second wait; what depends on this CTA's tiles becomes NaN,
    // here for the segments within its run and by the merge for those that reach beyond
    if (threadIdx.x == 0) atomicAdd(&g_kv4_wait_timeouts, 1u);
    float* part = a.ws + (int64_t)blockIdx.x * 2 * piece_floats<D, NT>();
    for (int i = threadIdx.x; i < 2 * piece_floats<D, NT>(); i += 32 * kWarps) part[i] = NAN;
    const Requests all = scan_requests<KT>(a);
    const Cut again(all.total, gridDim.x);
    const int first = again.start(blockIdx.x), last = again.start(blockIdx.x + 1);
    Cursor u = locate<KT>(a, all, first);
    if (threadIdx.x == 0) open_of<D, NT>(a, blockIdx.x)->parts = 0;
    for (int x = first - u.k; x < last;) {
      const int nq = queries_of(a, u.b), base = length_of(a, u.b) - nq;
      int z, hk, t, gi;
      split_segment(a, u.seg, z, hk);
      for (int i = threadIdx.x; i < RT * (D / 4) && x >= first && x + u.nt <= last; i += 32 * kWarps) {
        const int r = z * RT + i / (D / 4);
        split_row(a, r, t, gi);
        if (r < a.G * a.T)
          store4(out + u.b * a.st.s[3] + (hk * a.G + gi) * a.st.s[4] + t * a.st.s[5] + i % (D / 4) * 4,
                 make_float4(NAN, NAN, NAN, NAN), 1.f, t < nq && base + t >= 0);
      }
      if (threadIdx.x == 0 && x >= first && x + u.nt > last)
        *open_of<D, NT>(a, blockIdx.x) = {again.cta_of(x + u.nt - 1) - (int)blockIdx.x + 1, u.b, u.seg, nq, base, {}};
      x += u.nt;
      u.k = u.nt - 1;
      advance<KT>(a, u);
    }
    return;
  }
  constexpr int SLOTS = 2 * kWarps, LV = D / 4, H = 32 / LV;
  static_assert(SLOTS <= 32, "a lane per slot");
  Piece mine = {-1, 0, 0, 0, 0, 0, 0};
  if (lane < SLOTS) mine = pieces[lane >> 1][lane & 1];
  const uint32_t present = __ballot_sync(0xffffffffu, mine.b >= 0);
  uint32_t group = __match_any_sync(0xffffffffu, ((uint64_t)(uint32_t)mine.b << 32) | (uint32_t)mine.seg) & present;
  const uint32_t heads = __ballot_sync(0xffffffffu, mine.b >= 0 && lane == __ffs(group) - 1);
  const uint32_t ending = __ballot_sync(0xffffffffu, mine.b >= 0 && mine.ends);
  const uint32_t open = __ballot_sync(0xffffffffu, ((heads >> lane) & 1u) && mine.begins && !(group & ending));
  const int more = __shfl_sync(0xffffffffu, mine.more, 31 - __clz(group | 1u));  // of the group's last piece
  if (warp == kWarps - 1 && lane == max(__ffs(open) - 1, 0)) {  // at most one; the last warp has the fewest items
    const Cut all(s_total, gridDim.x);  // the open segment holds the CTA's last tile
    const int parts = open ? all.cta_of(all.start(blockIdx.x + 1) - 1 + more) - (int)blockIdx.x + 1 : 0;
    *open_of<D, NT>(a, blockIdx.x) = {parts, mine.b, mine.seg, mine.nq, mine.base, {}};
  }
  // an item is one row of one group; H members at a time, D / 4 lanes each
  for (int item = warp; item < __popc(heads) * RT; item += kWarps) {
    const int rr = item % RT;
    uint32_t rest = heads;
    for (int i = item / RT; i > 0; --i) rest &= rest - 1;
    const int head = __ffs(rest) - 1;
    uint32_t members = __shfl_sync(0xffffffffu, group, head);
    const bool begins = __shfl_sync(0xffffffffu, mine.begins, head), direct = begins && (members & ending);
    const int b = __shfl_sync(0xffffffffu, mine.b, head), seg = __shfl_sync(0xffffffffu, mine.seg, head);
    float2 ml = make_float2(-INFINITY, 0.f);
    if ((members >> lane) & 1u) ml = *reinterpret_cast<const float2*>(piece_at(lane >> 1, lane & 1) + rr * (D + 4) + D);
    const float mx = warp_max(ml.x), shift = mx == -INFINITY ? 0.f : mx;
    const float f = exp2f(ml.x - shift);
    const float den = warp_sum(f * ml.y);
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
    while (members) {
      int i = -1;
#pragma unroll
      for (int h = 0; h < H; ++h) {
        if (h == lane / LV) i = __ffs(members) - 1;
        members &= members - 1;
      }
      const float fi = __shfl_sync(0xffffffffu, f, max(i, 0));
      if (i >= 0) {
        const float4 y = *reinterpret_cast<const float4*>(piece_at(i >> 1, i & 1) + rr * (D + 4) + lane % LV * 4);
        acc.x = fmaf(fi, y.x, acc.x), acc.y = fmaf(fi, y.y, acc.y);
        acc.z = fmaf(fi, y.z, acc.z), acc.w = fmaf(fi, y.w, acc.w);
      }
    }
#pragma unroll
    for (int h = LV; h < 32; h <<= 1) {
      acc.x += __shfl_xor_sync(0xffffffffu, acc.x, h), acc.y += __shfl_xor_sync(0xffffffffu, acc.y, h);
      acc.z += __shfl_xor_sync(0xffffffffu, acc.z, h), acc.w += __shfl_xor_sync(0xffffffffu, acc.w, h);
    }
    if (lane >= LV) continue;
    const int d = lane * 4;
    if (direct) {
      int z, hk, t, gi;
      split_segment(a, seg, z, hk);
      const int r = z * RT + rr;
      split_row(a, r, t, gi);
      if (r < a.G * a.T) {
        const int nq = queries_of(a, b), base = length_of(a, b) - nq;
        const bool sees = t < nq && base + t >= 0 && den != 0.f;
        store4(out + b * a.st.s[3] + (hk * a.G + gi) * a.st.s[4] + t * a.st.s[5] + d, acc, sees ? 1.f / den : 0.f, sees);
      }
    } else {
      float* part = a.ws + ((int64_t)blockIdx.x * 2 + (begins ? 1 : 0)) * piece_floats<D, NT>() + rr * (D + 4);
      *reinterpret_cast<float4*>(part + d) = acc;
      if (d == 0) *reinterpret_cast<float2*>(part + D) = make_float2(mx, den);
    }
  }
}

// ------------------------------------------------------------------ merge
// Merge CTA c joins the partials of the segment that begins in worker CTA c's run and goes on in the next
// one's, if there is one (the worker has left beside them which).  Thread group i of D RT / 4 threads
// takes partials i, i + PL, ... in one pass with a running maximum; the groups are joined in order.  256
// threads of 40 registers find room beside the worker CTAs, so the merge is there when they end.
constexpr int kMergeThreads = 256;

template <typename T, int D, int NT>
__global__ void __launch_bounds__(kMergeThreads, 6) kv4_merge_kernel(T* __restrict__ out, const Args a) {
  constexpr int KT = Tile<D>::kKeys, RT = 4 * NT, NV = RT * D / 4, PL = kMergeThreads / NV;
  static_assert(NV <= kMergeThreads && kMergeThreads % NV == 0, "whole groups of threads");
  __shared__ float s_m[PL][RT], s_l[PL][RT];
  __shared__ float4 s_acc[PL][NV];
  allow_dependent_launch();  // a projection that follows may start fetching its weights
  // no memory is touched before; every CTA waits, also those without work: what follows this grid must
  // find the workers' done
  kv4::wait_for_previous();
  const int tid = threadIdx.x, c0 = blockIdx.x;
  const int v = tid % NV, pl = tid / NV, rr = v / (D / 4), d = v % (D / 4) * 4;
  const Open u = *open_of<D, NT>(a, c0);
  const int n = min(u.parts, a.ctas - c0);
  float4 y = make_float4(0.f, 0.f, 0.f, 0.f), acc = y;
  float2 ml = make_float2(-INFINITY, 0.f);
  float m = -INFINITY, l = 0.f;
  auto fetch = [&](int i) {
    // the first CTA's slot 1 (the segment began in its run), every other one's slot 0
    const float* src = a.ws + ((int64_t)(c0 + i) * 2 + (i == 0 ? 1 : 0)) * piece_floats<D, NT>() + rr * (D + 4);
    y = *reinterpret_cast<const float4*>(src + d);
    ml = *reinterpret_cast<const float2*>(src + D);
  };
  if (c0 + pl < a.ctas) fetch(pl);  // together with the number of them
  int z, hk, t, gi;
  split_segment(a, u.seg, z, hk);
  const int r = z * RT + rr;
  split_row(a, r, t, gi);
#pragma unroll 4
  for (int i = pl; i < n; i += PL) {
    if (i > pl) fetch(i);
    const float mn = fmaxf(m, ml.x), shift = mn == -INFINITY ? 0.f : mn;
    const float f = exp2f(m - shift), fi = exp2f(ml.x - shift);
    acc.x = fmaf(fi, y.x, acc.x * f), acc.y = fmaf(fi, y.y, acc.y * f);
    acc.z = fmaf(fi, y.z, acc.z * f), acc.w = fmaf(fi, y.w, acc.w * f);
    l = fmaf(fi, ml.y, l * f);
    m = mn;
  }
  if (n) {  // the same for all threads
    s_acc[pl][v] = acc;
    if (d == 0) s_m[pl][rr] = m, s_l[pl][rr] = l;
    __syncthreads();
  }
  if (n && pl == 0 && r < a.G * a.T) {
    m = -INFINITY;
#pragma unroll
    for (int i = 0; i < PL; ++i) m = fmaxf(m, s_m[i][rr]);
    const float shift = m == -INFINITY ? 0.f : m;
    acc = make_float4(0.f, 0.f, 0.f, 0.f);
    l = 0.f;
#pragma unroll
    for (int i = 0; i < PL; ++i) {
      const float f = exp2f(s_m[i][rr] - shift);
      y = s_acc[i][v];
      acc.x = fmaf(f, y.x, acc.x), acc.y = fmaf(f, y.y, acc.y);
      acc.z = fmaf(f, y.z, acc.z), acc.w = fmaf(f, y.w, acc.w);
      l = fmaf(f, s_l[i][rr], l);
    }
    const bool sees = t < u.nq && u.base + t >= 0 && l != 0.f;
    store4(out + u.b * a.st.s[3] + (hk * a.G + gi) * a.st.s[4] + t * a.st.s[5] + d, acc, sees ? 1.f / l : 0.f, sees);
  }
}

// ------------------------------------------------------------------ host side
// Score columns per thread of a row tile: tiles of 4, 8 or 16 query rows.  D = 128 stops at 8: with 16
// the output tile alone takes half the registers, and the spills cost more than the second pass over
// the cache saves (48 ragged requests of up to 5000 tokens, 16 rows: a fifth slower).
int row_tile(int64_t rows, int64_t D) {
  if (rows <= 4) return 1;
  return rows <= 8 || D == 128 ? 2 : 4;
}

// Both kernels ask for the same split of an SM's memory, so that merge CTAs may start beside workers.
int prepare_kernel(const void* fn, int smem) {
  if (smem && cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, smem) != cudaSuccess)
    return check_launch("cudaFuncSetAttribute (dynamic shared memory)");
  if (cudaFuncSetAttribute(fn, cudaFuncAttributePreferredSharedMemoryCarveout, cudaSharedmemCarveoutMaxShared) !=
      cudaSuccess)
    return check_launch("cudaFuncSetAttribute (carveout)");
  return MB_OK;
}

template <typename T, int D, int NT>
int launch(const void* q, void* out, Args a, cudaStream_t stream) {
  constexpr int smem = attention_smem<D, NT>();
  const void* fn = reinterpret_cast<const void*>(&kv4_attention_kernel<T, D, NT>);
  if (int rc = once_per_device(fn, prepare_kernel, smem)) return rc;
  const void* merge = reinterpret_cast<const void*>(&kv4_merge_kernel<T, D, NT>);
  if (int rc = once_per_device(merge, prepare_kernel, 0)) return rc;
  kv4::launch(kv4_attention_kernel<T, D, NT>, dim3(a.ctas), 32 * warps_of(NT, D), smem, stream, (const T*)q, (T*)out,
              (const Args)a);
  if (int rc = check_launch("kv4_chord_attention")) return rc;
  kv4::launch(kv4_merge_kernel<T, D, NT>, dim3(a.ctas), kMergeThreads, 0, stream, (T*)out, (const Args)a);
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
  return (int64_t)sm_count() * (2 * piece_floats(row_tile(H / Hkv * T, D), D) * (int64_t)sizeof(float) + sizeof(Open));
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
    a.by = page_div(page_size), a.most = (int)(max_pages * page_size), a.pages = num_pages;
    a.scale = scale, a.eps = eps;
    a.fail = forced(MB_FORCE_KV4_WAIT_FAILS);
    if (int rc = check_rows16("kv4_chord_attention", q, strides, sizeof(E))) return rc;
    if (int rc = check_rows16("kv4_chord_attention", out, strides + 3, sizeof(E))) return rc;
    const int nt = row_tile((int64_t)a.G * T, D);
    a.Z = (int)(((int64_t)a.G * T + 4 * nt - 1) / (4 * nt));
    a.ctas = kv4::sm_count();
    const int64_t tiles = (max_pages * page_size + Tile<DD>::kKeys - 1) / Tile<DD>::kKeys;
    MB_REQUIRE((int64_t)a.B * a.Z * a.Hkv * tiles < (1ll << 31), MB_ERR_SHAPE,
               "kv4_chord_attention: B * Hkv * row tiles * key tiles = %lld (fewer than 2^31)",
               (long long)((int64_t)a.B * a.Z * a.Hkv * tiles));
    if (nt == 1) return launch<E, DD, 1>(q, out, a, (cudaStream_t)stream);
    if constexpr (DD < 128)
      if (nt == 4) return launch<E, DD, 4>(q, out, a, (cudaStream_t)stream);
    return launch<E, DD, 2>(q, out, a, (cudaStream_t)stream);
  });
}
