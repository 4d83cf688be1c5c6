// Attention of one token over the compressed key-value cache.
//
// With q' = Rk q and the packed rows' centroids c, the score of token j is
//   s_j = scale * kn_j * sum_i q'_i c[kcode_ji]
// and the output Rv^T (sum_j p_j vn_j c[vcode_j]), p = softmax(s): neither side
// of the cache is turned back, only the query and the output.
//
// Three launches, each let in early by the one before it (programmatic
// dependent launch):
//  1. kv_query_kernel turns the queries (f32), splits each into f16 hi + lo
//     planes of a power-of-two scale and one block sums up the sequences' units
//     of work.
//  2. kv_attend_kernel: persistent blocks take equal runs of units (a unit: one
//     step of all warps of one key-value head and up to eight of its query heads),
//     so ragged batches and single long sequences fill the GPU alike.  One pass
//     with running maximum and sum; a block leaves one partial result for every
//     head that its run touches.
//  3. kv_join_kernel puts a head's partials together in order (no atomics: the
//     same call gives the same bits) and turns the output back.
// With `accumulate`, 2 also leaves the scores and a fourth kernel turns them
// into softmax weights.
//
// The step.  A warp takes 16 tokens at a time through mma.m16n8k16: keys are
// the A operand (16 tokens x 16 coordinates), the eight queries B, so S^T has
// tokens in rows; values transposed are A (16 coordinates x 16 tokens) and P^T
// is B, made from S^T's registers by movmatrix.  Operand registers are made in
// place from the packed codes: every lane's 16-byte load of a row holds the
// coordinates of its own operand registers, because the order of coordinates
// is free as long as the queries have the same one.  A packed byte is decoded
// by one shared-memory lookup that gives both of its centroids as an f16 pair
// (4 bits; at 8 bits one centroid as f16 hi + lo, at 2 bits four centroids as two
// pairs), from a table with a copy for each lane (at 2 bits each lane of half a
// warp): no bank conflicts, and the address is one dp4a.
//
// What bounds it: issued instructions and shared memory.  At 4 bits and d = 128
// sixteen tokens of a head are 2.2 KB and, for bf16 outputs, some 470 instructions,
// 96 of them lookups (an SM's shared memory does one a cycle) and 32 matrix products.
// 16 sequences of 0 to 32768 tokens, 8 heads, 32 query heads, bf16: the kernel
// 100 us, 2.6 TB/s of rows (the call 106, a copy's rate 40); issue slots 57 % taken,
// shared memory 63 %, the matrix pipe 31 %, three warps a scheduler.  tcgen05 would
// relieve the matrix pipe, which is not the limit, and have the decoded rows, four
// times the codes for each of hi and lo, written to shared or tensor memory first.
//
// Roundings.  Centroids and queries are taken times powers of two that put the
// largest at 2^13; f16 hi has 11 bits, hi + lo 22.  Softmax weights times value
// norms (times a scale that follows the largest product so far) are rounded to
// f16 for the product.
//   Scores are products of hi + lo for every type: what a score is off by, its
//   softmax weight is off by, times the score, so that 11 bits lose 0.4 % of a
//   weight at |q||k| / sqrt(d) = 100 and bf16 outputs were off by 1.2 times their
//   own rounding at scores of 200, 1.6 times at 900.
//   Values and their weights are hi alone for bf16 outputs: errors of 2^-12 in the
//   mean next to the output's 2^-9, whatever the values and scores.
//   For f16 and f32 outputs (FINE) they are hi + lo as well.  (f16 with the
//   centroids' hi alone had up to 3.4 times the error of the output's own
//   rounding: all tokens share the few centroids' errors, nothing averages.)
// Maxima, sums and accumulators are f32.  The tensor cores' sums are cut off, not
// rounded, and a chain of them drifts: scores are four sums put together in f32,
// and FINE adds every group's values to the output in f32.
#include <float.h>

#include "kv.cuh"

namespace pqb {
namespace kv {

constexpr int kHeadsPer = 8;    // query heads of one block: the width of an mma
constexpr int kMaxWorkers = 384;  // blocks of the attention kernel
constexpr int kLeastUnit = 64;     // tokens of the smallest unit of any shape
constexpr int kSegmentCost = 768;  // what taking up a segment costs, in tokens
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;
// Softmax weights relative to the running maximum of the scores reach 2^3 before
// that follows.  A value's weight, that times its norm, is held relative to a
// reference of its own for each query head, near the largest such product so far:
// a long value that is not attended to takes no bits from the others.  It is taken
// times 2^10 and reaches 2^5 of its reference before that follows: at most 2^15 in
// f16, with 11 bits down to 2^-23 of the largest.
constexpr float kRescale = 3.f;
constexpr float kWeightScale = 1024.f;
constexpr float kMostWeight = 32768.f;
constexpr float kMostUp = 0x1p100f;  // (products below 2^-90 lose bits)

__device__ __forceinline__ void pdl_wait() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void pdl_next() {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
}

__device__ __forceinline__ void mma16816(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2,
                                         uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
      "{%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

__device__ __forceinline__ uint32_t transpose8(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}

__device__ __forceinline__ uint32_t pack_half2(float a, float b) {
  const __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}

__device__ __forceinline__ float2 unpack_half2(uint32_t x) {
  return __half22float2(*reinterpret_cast<const __half2*>(&x));
}

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// B bytes (2, 4, 8 or 16) at a shared-memory address.
template <int B>
__device__ __forceinline__ void shared_bytes(uint32_t at, uint32_t* w) {
  if constexpr (B == 16)
    asm volatile("ld.shared.v4.b32 {%0,%1,%2,%3}, [%4];"
                 : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3])
                 : "r"(at));
  else if constexpr (B == 8)
    asm volatile("ld.shared.v2.b32 {%0,%1}, [%2];" : "=r"(w[0]), "=r"(w[1]) : "r"(at));
  else if constexpr (B == 4)
    asm volatile("ld.shared.b32 %0, [%1];" : "=r"(w[0]) : "r"(at));
  else
    asm volatile("{\n\t.reg .b16 h;\n\tld.shared.b16 h, [%1];\n\tcvt.u32.u16 %0, h;\n\t}"
                 : "=r"(w[0])
                 : "r"(at));
}

__device__ __forceinline__ float shared_float(uint32_t at) {
  float x;
  asm volatile("ld.shared.f32 %0, [%1];" : "=f"(x) : "r"(at));
  return x;
}

__device__ __forceinline__ void copy16(uint32_t to, const void* from) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to), "l"(from) : "memory");
}
__device__ __forceinline__ void copy_commit() {
  asm volatile("cp.async.commit_group;" ::: "memory");
}
template <int N>
__device__ __forceinline__ void copy_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

// How a row of D coordinates is dealt to L lanes: lane i holds bytes
// [u * L * UB + i * UB, + UB) of it for each unit u, CU codes a unit.
template <int D, int BITS, int L>
struct Deal {
  static constexpr int row = D * BITS / 8;  // bytes of a row of D coordinates
  static constexpr int bytes = row / L;
  static constexpr int UB = bytes < 16 ? bytes : 16;
  static constexpr int units = bytes / UB;
  static constexpr int words = (bytes + 3) / 4;
  static constexpr int CU = UB * 8 / BITS;
  // Coordinate of the lane's code n.
  static __device__ __forceinline__ int dim(int lane, int n) {
    return (n / CU) * L * CU + lane * CU + n % CU;
  }
};

// Sixteen rows lie in shared memory one after another, each with the room of D
// coordinates, their 16-byte pieces exchanged so that a warp's loads meet no bank
// twice: keys are read by 8 rows x 4 pieces, values by 4 rows (2t and 2t + 1
// alternating) x 8 lanes.  Where piece n of the sixteen rows lies:
template <int ROW>
__device__ __forceinline__ int key_piece(int n) {
  return ROW >= 128 ? n ^ ((n / (ROW / 16) & 1) << 2) : n;
}
template <int ROW>
__device__ __forceinline__ int value_piece(int n) {
  return ROW >= 128 ? n ^ ((n / (ROW / 16) >> 1 & 3) << 1)
         : ROW >= 32 ? n ^ ((n / (ROW / 16) >> 2 & 1) << 1)
                     : n;
}

// Decoding.  A side's table has 256 entries of 128 bytes, a copy of the entry's
// word for every lane (2 bits: of its two words for every lane of half a warp);
// keys' first, values' behind them, then the lo tables of the sides that have one
// (2 and 4 bits; at 8 an entry holds both parts): keys', then with FINE values'.
// `base` is the lane's place in entry 0 as a shared-memory address; one dp4a adds
// 128 times a byte of the packed word to it.  AT: where the table lies from there.
constexpr uint32_t kTableBytes = 32768;

template <int BITS>
__device__ __forceinline__ uint32_t lane_place(int lane) {
  return BITS == 2 ? (lane & 15) * 8 : lane * 4;
}

template <int AT>
__device__ __forceinline__ uint32_t lookup(uint32_t base, uint32_t w, int byte) {
  const uint32_t at = __dp4a(w, 128u << (8 * byte), base);
  uint32_t x;
  asm("ld.shared.b32 %0, [%1+%2];" : "=r"(x) : "r"(at), "n"(AT));
  return x;
}

template <int AT>
__device__ __forceinline__ uint2 lookup2(uint32_t base, uint32_t w, int byte) {
  const uint32_t at = __dp4a(w, 128u << (8 * byte), base);
  uint2 x;
  asm("ld.shared.v2.b32 {%0,%1}, [%2+%3];"
      : "=r"(x.x), "=r"(x.y)
      : "r"(at), "n"(AT));
  return x;
}

// The four codes that a lane gives to one K step: pairs a (first operand
// register) and b (third), hi and lo.
constexpr int kKeyLo = 2 * (int)kTableBytes;

template <int BITS, int W>
__device__ __forceinline__ void decode_key(const uint32_t (&w)[W], int s, uint32_t base,
                                           uint32_t& ah, uint32_t& bh, uint32_t& al, uint32_t& bl) {
  if constexpr (BITS == 4) {
    const uint32_t x = w[s >> 1];
    const int b = (s & 1) * 2;
    ah = lookup<0>(base, x, b);
    bh = lookup<0>(base, x, b + 1);
    al = lookup<kKeyLo>(base, x, b);
    bl = lookup<kKeyLo>(base, x, b + 1);
  } else if constexpr (BITS == 8) {
    const uint32_t x = w[s];
    const uint32_t e0 = lookup<0>(base, x, 0), e1 = lookup<0>(base, x, 1);
    const uint32_t e2 = lookup<0>(base, x, 2), e3 = lookup<0>(base, x, 3);
    ah = __byte_perm(e0, e1, 0x5410);
    bh = __byte_perm(e2, e3, 0x5410);
    al = __byte_perm(e0, e1, 0x7632);
    bl = __byte_perm(e2, e3, 0x7632);
  } else {
    const uint2 e = lookup2<0>(base, w[s >> 2], s & 3);
    ah = e.x;
    bh = e.y;
    const uint2 f = lookup2<kKeyLo>(base, w[s >> 2], s & 3);
    al = f.x;
    bl = f.y;
  }
}

// Codes 2m, 2m + 1 (and 2m + 2, 2m + 3) of two tokens' rows: of each code the pair
// (x's, y's), even ones in `e`, odd ones in `o`.  LO: with lo parts, their table AT.
template <int BITS, bool LO, int AT, int W>
__device__ __forceinline__ void decode_value(const uint32_t (&x)[W], const uint32_t (&y)[W], int m,
                                             uint32_t base, uint32_t (&eh)[2], uint32_t (&oh)[2],
                                             uint32_t (&el)[2], uint32_t (&ol)[2]) {
  if constexpr (BITS == 4) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int n = m + i;
      const uint32_t p = lookup<0>(base, x[n >> 2], n & 3), q = lookup<0>(base, y[n >> 2], n & 3);
      eh[i] = __byte_perm(p, q, 0x5410);
      oh[i] = __byte_perm(p, q, 0x7632);
      if constexpr (LO) {
        const uint32_t r = lookup<AT>(base, x[n >> 2], n & 3), t = lookup<AT>(base, y[n >> 2], n & 3);
        el[i] = __byte_perm(r, t, 0x5410);
        ol[i] = __byte_perm(r, t, 0x7632);
      }
    }
  } else if constexpr (BITS == 8) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int n = m + i, b = 2 * (n & 1);
      const uint32_t p0 = lookup<0>(base, x[n >> 1], b), p1 = lookup<0>(base, x[n >> 1], b + 1);
      const uint32_t q0 = lookup<0>(base, y[n >> 1], b), q1 = lookup<0>(base, y[n >> 1], b + 1);
      eh[i] = __byte_perm(p0, q0, 0x5410);
      oh[i] = __byte_perm(p1, q1, 0x5410);
      if constexpr (LO) {
        el[i] = __byte_perm(p0, q0, 0x7632);
        ol[i] = __byte_perm(p1, q1, 0x7632);
      }
    }
  } else {
    const int n = m >> 1;  // byte of the row
    const uint2 p = lookup2<0>(base, x[n >> 2], n & 3), q = lookup2<0>(base, y[n >> 2], n & 3);
    eh[0] = __byte_perm(p.x, q.x, 0x5410);
    oh[0] = __byte_perm(p.x, q.x, 0x7632);
    eh[1] = __byte_perm(p.y, q.y, 0x5410);
    oh[1] = __byte_perm(p.y, q.y, 0x7632);
    if constexpr (LO) {
      const uint2 r = lookup2<AT>(base, x[n >> 2], n & 3), t = lookup2<AT>(base, y[n >> 2], n & 3);
      el[0] = __byte_perm(r.x, t.x, 0x5410);
      ol[0] = __byte_perm(r.x, t.x, 0x7632);
      el[1] = __byte_perm(r.y, t.y, 0x5410);
      ol[1] = __byte_perm(r.y, t.y, 0x7632);
    }
  }
}

// ---------------------------------------------------------------------------
// Work: the units of all (sequence, key-value head, block of query heads), in
// that order; segment = the units of one of them.
// ---------------------------------------------------------------------------

struct Work {
  const int32_t* table;
  int64_t table_stride;
  int table_width;
  const int32_t* lengths;
  int batch, heads, group, blocks;  // blocks of query heads per key-value head
  int unit;                         // tokens of a unit
  const int* first;                 // [batch + 1] first unit of each sequence

  int empty;                        // units without tokens, a segment's first

  // A segment's units: first as many without tokens as taking it up costs a block
  // (4 us at D = 128, 7 us at D = 256, as much as some 768 tokens).  Without
  // them, the block that gets a batch's short sequences ends last (16 sequences
  // of 0 to 32768 tokens: 24 % of the time of the other SMs).
  __device__ int units_of(int len) const { return len ? empty + (len + unit - 1) / unit : 0; }
};

// Worker of a unit: worker w of n takes units [w * total / n, (w + 1) * total / n).
__device__ __forceinline__ int worker_of(int64_t u, int n, int total) {
  return (int)(((u + 1) * n - 1) / total);
}

struct QueryOut {
  __half *hi, *lo;  // [segment][8][D]
  float* factor;    // [segment][8]: score = factor * key norm * product, in log2
};

// Turning rows by a D x D matrix: kRotParts threads a column share its products.
// A thread's first elements of the matrix (64 KB from L2 at D = 128) are loaded
// ahead, where the kernel still waits for the rows; x comes in 16-byte loads, as
// one load for each product bounds the block by shared memory (D = 256: 11 us).
constexpr int kRotParts = 4;
constexpr int kRotAhead = 16;

template <int D>
struct Turn {
  float r[kRotAhead];
  const float* m;
  int d, j, i0;

  __device__ __forceinline__ void ahead(const float* M, int d_, int j_, int part) {
    m = M;
    d = d_;
    j = j_;
    i0 = part * (D / kRotParts);
#pragma unroll
    for (int i = 0; i < kRotAhead; ++i) r[i] = at(i0 + i);
  }
  __device__ __forceinline__ float at(int i) const {
    return i < d && j < d ? __ldg(m + i * d + j) : 0.f;
  }
  // acc[g] = sum over this thread's rows i of x[g][i] * M[i][j].
  __device__ __forceinline__ void run(const float (&x)[kHeadsPer][D], float (&acc)[kHeadsPer]) {
#pragma unroll
    for (int g = 0; g < kHeadsPer; ++g) acc[g] = 0.f;
#pragma unroll 1
    for (int i = i0; i < i0 + D / kRotParts; i += kRotAhead) {
      float w[kRotAhead];
#pragma unroll
      for (int k = 0; k < kRotAhead; ++k) w[k] = r[k];
      if (i + kRotAhead < i0 + D / kRotParts) {
#pragma unroll
        for (int k = 0; k < kRotAhead; ++k) r[k] = at(i + kRotAhead + k);
      }
#pragma unroll
      for (int k = 0; k < kRotAhead; k += 4)
#pragma unroll
        for (int g = 0; g < kHeadsPer; ++g) {
          const float4 v = *reinterpret_cast<const float4*>(&x[g][i + k]);
          acc[g] = fmaf(v.x, w[k], acc[g]);
          acc[g] = fmaf(v.y, w[k + 1], acc[g]);
          acc[g] = fmaf(v.z, w[k + 2], acc[g]);
          acc[g] = fmaf(v.w, w[k + 3], acc[g]);
        }
    }
  }
};

template <class T, int D>
__global__ void __launch_bounds__(kRotParts * D)
kv_query_kernel(const T* __restrict__ q, int64_t sb, int64_t sh, int d, int page_size,
                const float* __restrict__ RT, const int* __restrict__ exponent, float scale,
                Work wk, QueryOut out, int* __restrict__ first) {
  constexpr int threads = kRotParts * D, warps = threads / 32;
  __shared__ __align__(16) float sq[kHeadsPer][D];
  __shared__ float red[kRotParts][kHeadsPer][D];
  __shared__ int s_part[warps];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  pdl_next();
  const int per = wk.heads * wk.blocks;
  if (blockIdx.x == wk.batch * per) {
    // First units: a running sum over the sequences.
    int base = 0;
    for (int b0 = 0; b0 < wk.batch; b0 += threads) {
      const int b = b0 + tid;
      const int n = b < wk.batch
                        ? per * wk.units_of(clamp_length(wk.lengths[b], wk.table_width, page_size))
                        : 0;
      int v = n;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int y = __shfl_up_sync(0xffffffffu, v, o);
        if (lane >= o) v += y;
      }
      if (lane == 31) s_part[warp] = v;
      __syncthreads();
      int before = 0, all = 0;
      for (int i = 0; i < warps; ++i) {
        if (i < warp) before += s_part[i];
        all += s_part[i];
      }
      if (b < wk.batch) first[b] = base + before + v - n;
      base += all;
      __syncthreads();
    }
    if (tid == 0) first[wk.batch] = base;
    return;
  }
  const int b = blockIdx.x / per, h = blockIdx.x % per / wk.blocks, hb = blockIdx.x % wk.blocks;
  const int ng = min(kHeadsPer, wk.group - hb * kHeadsPer);
  const T* src = q + b * sb + ((int64_t)h * wk.group + hb * kHeadsPer) * sh;
  const int j = tid % D, part = tid / D;
  Turn<D> turn;
  turn.ahead(RT, d, j, part);
#pragma unroll
  for (int g = part; g < kHeadsPer; g += kRotParts)
    sq[g][j] = g < ng && j < d ? to_f32<T>(src[g * sh + j]) : 0.f;
  __syncthreads();
  float acc[kHeadsPer];
  turn.run(sq, acc);
#pragma unroll
  for (int g = 0; g < kHeadsPer; ++g) red[part][g][j] = acc[g];
  __syncthreads();
  // A warp per head: scale to a largest of [2^13, 2^14) and split.
  if (warp >= kHeadsPer) return;
  float y[D / 32], mx = 0.f;
#pragma unroll
  for (int i = 0; i < D / 32; ++i) {
    y[i] = 0.f;
#pragma unroll
    for (int p = 0; p < kRotParts; ++p) y[i] += red[p][warp][lane + 32 * i];
    mx = fmaxf(mx, fabsf(y[i]));
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
  const int e = mx > 0.f && mx < INFINITY ? max(-100, min(100, 13 - ilogbf(mx))) : 0;
  const int64_t row = (int64_t)blockIdx.x * kHeadsPer + warp;
  const float up = ldexpf(1.f, e);
#pragma unroll
  for (int i = 0; i < D / 32; ++i) {
    const float v = y[i] * up;
    const __half hi = __float2half_rn(v);
    out.hi[row * D + lane + 32 * i] = hi;
    out.lo[row * D + lane + 32 * i] = __float2half_rn(v - __half2float(hi));
  }
  if (lane == 0) out.factor[row] = ldexpf(scale * kLog2e, -e - *exponent);
}

struct Parts {
  float* o;    // [slot][8][D], times 2^(exponent of the values' centroids - 14)
  float2* ml;  // [slot][8]: maximum (log2), sum
};

template <int D, int KB, int VB, bool FINE>
struct AttendShape {
  static constexpr bool k_lo = KB != 8, v_lo = FINE && VB != 8;  // sides with a lo table
  static constexpr int table_bytes = (2 + k_lo + v_lo) * (int)kTableBytes;
  static constexpr int ostride = D + 8;  // of a partial result's head in shared memory
  // A warp has two stages, a step's rows and norms each; a stage also holds the
  // warp's partial result at a segment's end, while the next segment's first
  // step comes into the other.
  static constexpr int stage_of(int mt) {
    const int step = 16 * mt * (D * KB / 8 + D * VB / 8 + 8);
    const int part = kHeadsPer * ostride * 4;
    return step > part ? step : part;
  }
  static constexpr int room = 224 * 1024 - table_bytes;
  static constexpr int fit(int mt) { return room / (2 * stage_of(mt)) / 2 * 2; }
  // Registers allow 12 warps up to D = 128 (16 of bf16 outputs spill: 113 us instead
  // of 100 of the case above) and 8 at D = 256, where shared memory leaves 8, 6 or 4
  // warps beside two, three or four tables.
  static constexpr int most = D <= 128 ? 12 : 8;
  // A warp's step is two groups of 16 tokens at D = 64, one above.  (4 bits, bf16, 16
  // sequences of 0 to 32768 tokens, 8 heads of 4 query heads, D = 64: 65 us next to 71
  // with one; at D = 128, 0 to 16384 tokens: 67 with one next to 66 with two, which
  // needs as many registers more as spill with hi + lo values; 8 + 4 bits 52 and 52.)
  static constexpr int MT = D == 64 ? 2 : 1;
  static constexpr int stage = stage_of(MT);
  static constexpr int warps = fit(MT) < most ? fit(MT) : most;
  static constexpr int threads = 32 * warps;
  static constexpr int unit = warps * 16 * MT;
  static constexpr int smem = table_bytes + 2 * warps * stage;
};

template <int D, int KB, int VB, bool FINE>
__global__ void __launch_bounds__(AttendShape<D, KB, VB, FINE>::threads, 1)
kv_attend_kernel(Side sk, Side sv, int pages, int page_shift, Work wk, QueryOut qo, Parts parts,
                 float* __restrict__ scores, int64_t score_width) {
  using Shape = AttendShape<D, KB, VB, FINE>;
  constexpr int MT = Shape::MT, NW = Shape::warps;
  constexpr int VLO_AT = (Shape::k_lo ? 2 : 1) * (int)kTableBytes;  // from the values' table
  using KD = Deal<D, KB, 4>;
  using VD = Deal<D, VB, 8>;
  constexpr int KS = D / 16;  // K steps of a score, and pairs of coordinates of a value
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ float s_m[NW][kHeadsPer], s_l[NW][kHeadsPer], s_f[NW][kHeadsPer];
  __shared__ int s_b;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;

  // Tables, from the codec's entries (set-up data: not written by the kernel
  // before).  A thread copies an entry to the 32 lanes' places.
#pragma unroll
  for (int table = 0; table < Shape::table_bytes / (int)kTableBytes; ++table) {
    const bool lo = table >= 2, value = table == 1 || (lo && (!Shape::k_lo || table == 3));
    const Codec& c = value ? sv.c : sk.c;
    for (int n = tid; n < 256; n += Shape::threads) {
      const uint2 e = c.pairs[(lo ? 256 : 0) + n];
      const uint4 v = make_uint4(e.x, e.y, e.x, e.y);
#pragma unroll
      for (int i = 0; i < 8; ++i)
        *reinterpret_cast<uint4*>(smem + table * kTableBytes + n * 128 + ((i + n) & 7) * 16) = v;
    }
  }
  const uint32_t table0 = (uint32_t)__cvta_generic_to_shared(smem);
  const uint32_t kbase = table0 + lane_place<KB>(lane);
  const uint32_t vbase = table0 + kTableBytes + lane_place<VB>(lane);

  // A stage: MT times sixteen rows of keys, of values, sixteen norms of either.
  constexpr int values_at = 16 * KD::row, norms_at = 16 * (KD::row + VD::row);
  constexpr int group = norms_at + 128;
  const uint32_t kld = (uint32_t)sk.ldb, vld = (uint32_t)sv.ldb;
  const uint32_t stage0 = (uint32_t)__cvta_generic_to_shared(smem) + Shape::table_bytes +
                          warp * 2 * Shape::stage;
  // Row r of the scores (lane: r = g and g + 8) is token r ^ (r >> 1 & 1), so that
  // the tokens of lane (g, t)'s value operands, those of rows 2t, 2t + 1 (+ 8),
  // alternate between even and odd rows of shared memory over t.
  const int tok_k = g ^ (g >> 1 & 1), tok_v = 2 * t + (t & 1);
  // The lane's places in a group.  (Where a row is shorter than D coordinates,
  // what lies behind it meets zeros in the queries and is dropped from the
  // values; any bytes decode to finite centroids.)
  uint32_t kat[KD::units], vat[2][VD::units];
#pragma unroll
  for (int u = 0; u < KD::units; ++u) {
    const int at = tok_k * KD::row + (u * 4 + t) * KD::UB;
    kat[u] = key_piece<KD::row>(at / 16) * 16 + at % 16;
  }
#pragma unroll
  for (int e = 0; e < 2; ++e)
#pragma unroll
    for (int u = 0; u < VD::units; ++u) {
      const int at = (tok_v ^ e) * VD::row + (u * 8 + g) * VD::UB;
      vat[e][u] = values_at + value_piece<VD::row>(at / 16) * 16 + at % 16;
    }
  const uint32_t norm_at = norms_at + 4 * tok_k;
  // Copies: the lane's pieces of a group (piece n of the pool's sixteen rows is
  // piece n % (ld / 16) of row n / (ld / 16)), and where they come from.
  constexpr int KJ = (KD::row + 31) / 32, VJ = (VD::row + 31) / 32;
  uint32_t kto[KJ], vto[VJ];
#pragma unroll
  for (int j = 0; j < KJ; ++j) {
    const int n = lane + 32 * j, per_row = kld / 16;
    kto[j] = 16 * key_piece<KD::row>(n / per_row * (KD::row / 16) + n % per_row);
  }
#pragma unroll
  for (int j = 0; j < VJ; ++j) {
    const int n = lane + 32 * j, per_row = vld / 16;
    vto[j] = values_at + 16 * value_piece<VD::row>(n / per_row * (VD::row / 16) + n % per_row);
  }
  const uint8_t *kfrom = sk.rows + lane * 16, *vfrom = sv.rows + lane * 16;
  const float* nfrom = (lane & 4 ? sv.norms : sk.norms) + (lane & 3) * 4;
  const uint32_t nto = norms_at + 16 * lane;
  pdl_wait();
  pdl_next();

  const int per = wk.heads * wk.blocks;
  const int total = wk.first[wk.batch];
  const int n = min((int)gridDim.x, total);
  if ((int)blockIdx.x >= n) return;
  int u = (int)((int64_t)blockIdx.x * total / n);
  const int uend = (int)(((int64_t)blockIdx.x + 1) * total / n);
  for (int i = tid; i < wk.batch; i += Shape::threads)
    if (wk.first[i] <= u && u < wk.first[i + 1]) s_b = i;
  __syncthreads();

  constexpr int stride = Shape::unit;
  // A segment and the block's share of it, tokens [t0, t1).  Those of a warp's
  // segment and its next one wait in shared memory: the loop has no registers to
  // spare for them.
  struct Segment {
    int b, seg, hb, h, t0, t1;
    int pid[MT];  // pages of the warp's first step's groups; -1 for none
  };
  __shared__ Segment s_segment[2][NW];
  auto page_of = [&](const int32_t* row, int t1, int base, int i) {
    const int tok = base + 16 * i;
    int p = -1;
    if (tok < t1) {
      p = __ldg(row + (tok >> page_shift));
      if (p >= pages) p = -1;
    }
    return p;
  };
  // The segment of unit u, from sequence b on; u moves behind it.
  auto take = [&](int which, int b) {
    Segment x;
    x.t0 = x.t1 = 0;
    x.b = b;
    x.seg = x.hb = x.h = 0;
#pragma unroll
    for (int i = 0; i < MT; ++i) x.pid[i] = -1;
    while (u < uend) {
      while (u >= wk.first[x.b + 1]) ++x.b;
      const int len = clamp_length(wk.lengths[x.b], wk.table_width, 1 << page_shift);
      const int nu = wk.units_of(len);
      const int r = u - wk.first[x.b], in = r / nu, from = r % nu, u0 = max(from, wk.empty);
      const int u1 = min(nu, from + (uend - u));
      u += u1 - from;
      if (u1 <= u0) continue;  // empty units alone, at the end of the run
      x.h = in / wk.blocks;
      x.hb = in % wk.blocks;
      x.seg = x.b * per + in;
      x.t0 = (u0 - wk.empty) * stride;
      x.t1 = min(len, (u1 - wk.empty) * stride);
#pragma unroll
      for (int i = 0; i < MT; ++i)
        x.pid[i] = page_of(wk.table + x.b * wk.table_stride, x.t1, x.t0 + warp * 16 * MT, i);
      break;
    }
    if (lane == 0) s_segment[which][warp] = x;
    __syncwarp();
  };
  // Copies the step at `base`, its groups on pages pid, to a stage.  Groups without a page read page 0:
  // what tokens that are not there decode to is finite, and meets a weight of 0.
  // (A pool has fewer than 2^32 rows.)
  auto fetch = [&](const int (&pid)[MT], int h, int base, uint32_t stage) {
#pragma unroll
    for (int i = 0; i < MT; ++i) {
      const uint32_t row = ((uint32_t)(max(pid[i], 0) * wk.heads + h) << page_shift) +
                           (uint32_t)((base + 16 * i) & ((1 << page_shift) - 1));
      const uint8_t* kp = kfrom + (uint64_t)row * kld;
      const uint8_t* vp = vfrom + (uint64_t)row * vld;
#pragma unroll
      for (int j = 0; j < KJ; ++j)
        if (lane + 32 * j < (int)kld) copy16(stage + i * group + kto[j], kp + 512 * j);
#pragma unroll
      for (int j = 0; j < VJ; ++j)
        if (lane + 32 * j < (int)vld) copy16(stage + i * group + vto[j], vp + 512 * j);
      if (lane < 8) copy16(stage + i * group + nto, nfrom + row);
    }
    copy_commit();
  };

  take(0, s_b);
  int p = 0;  // stage of the step to come
  {
    const Segment& x = s_segment[0][warp];
    if (x.t0 + warp * 16 * MT < x.t1) fetch(x.pid, x.h, x.t0 + warp * 16 * MT, stage0);
  }
#pragma unroll 1
  for (int which = 0;; which ^= 1) {
    const Segment& seg = s_segment[which][warp];
    const int t1 = seg.t1, h = seg.h;
    if (seg.t0 >= t1) break;
    const int32_t* prow = wk.table + seg.b * wk.table_stride;
    int base = seg.t0 + warp * 16 * MT;
    int pid[MT], pid1[MT];  // pages of the step to come and of the one after it
#pragma unroll
    for (int i = 0; i < MT; ++i) {
      pid[i] = seg.pid[i];
      pid1[i] = page_of(prow, t1, base + stride, i);
    }

    // The queries as B operands: lane (g, t) holds head g.
    uint32_t qh[KS][2], ql[KS][2];
    {
      const __half* hi = qo.hi + ((int64_t)seg.seg * kHeadsPer + g) * D;
      const __half* lo = qo.lo + ((int64_t)seg.seg * kHeadsPer + g) * D;
#pragma unroll
      for (int s = 0; s < KS; ++s) {
        const int dim = KD::dim(t, 4 * s);
        uint2 x = *reinterpret_cast<const uint2*>(hi + dim);
        qh[s][0] = x.x;
        qh[s][1] = x.y;
        x = *reinterpret_cast<const uint2*>(lo + dim);
        ql[s][0] = x.x;
        ql[s][1] = x.y;
      }
    }
    const float f0 = qo.factor[(int64_t)seg.seg * kHeadsPer + 2 * t];
    const float f1 = qo.factor[(int64_t)seg.seg * kHeadsPer + 2 * t + 1];
    take(which ^ 1, seg.b);  // (while the queries come)

    float o[KS][4];
#pragma unroll
    for (int m = 0; m < KS; ++m) o[m][0] = o[m][1] = o[m][2] = o[m][3] = 0.f;
    float m0 = -FLT_MAX, m1 = -FLT_MAX, l0 = 0.f, l1 = 0.f;
    float up0 = kMostUp, up1 = kMostUp;  // what value weights are taken times

#pragma unroll 1
    for (; base < t1; base += stride) {
      const uint32_t st = stage0 + p * Shape::stage;
      bool there = base + 16 * MT <= t1;
      uint32_t gone = 0;  // groups without a page
#pragma unroll
      for (int i = 0; i < MT; ++i) {
        if (pid[i] < 0) gone |= 1u << i;
        pid[i] = pid1[i];
      }
      there = there && gone == 0;
      p ^= 1;
      if (base + stride < t1) {
        fetch(pid, h, base + stride, stage0 + p * Shape::stage);
#pragma unroll
        for (int i = 0; i < MT; ++i) pid1[i] = page_of(prow, t1, base + 2 * stride, i);
        copy_wait<1>();
      } else {
        copy_wait<0>();
      }
      __syncwarp();

      // Scores: S^T, tokens of rows g and g + 8, heads 2t and 2t + 1.
      float s[MT][4];
#pragma unroll
      for (int i = 0; i < MT; ++i) {
        uint32_t kw[2][KD::words];
#pragma unroll
        for (int e = 0; e < 2; ++e)
#pragma unroll
          for (int un = 0; un < KD::units; ++un)
            shared_bytes<KD::UB>(st + kat[un] + (i * group + e * 8 * KD::row),
                                 &kw[e][un * KD::UB / 4]);
        s[i][0] = s[i][1] = s[i][2] = s[i][3] = 0.f;
        float more[3][4] = {};
#pragma unroll
        for (int k = 0; k < KS; ++k) {
          uint32_t a0, a1, a2, a3, c0, c1, c2, c3;
          decode_key<KB>(kw[0], k, kbase, a0, a2, c0, c2);
          decode_key<KB>(kw[1], k, kbase, a1, a3, c1, c3);
          mma16816(k % 2 ? more[0] : s[i], a0, a1, a2, a3, qh[k][0], qh[k][1]);
          mma16816(more[1], a0, a1, a2, a3, ql[k][0], ql[k][1]);
          mma16816(more[2], c0, c1, c2, c3, qh[k][0], qh[k][1]);
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) s[i][e] += more[0][e] + (more[1][e] + more[2][e]);
      }
      float mx0 = -FLT_MAX, mx1 = -FLT_MAX, vn[MT][2];
#pragma unroll
      for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const uint32_t at = st + norm_at + (i * group + 32 * e);
          const float kn = shared_float(at);
          vn[i][e] = shared_float(at + 64);
          s[i][2 * e] *= kn * f0;
          s[i][2 * e + 1] *= kn * f1;
        }
      if (!there) {
#pragma unroll
        for (int i = 0; i < MT; ++i)
#pragma unroll
          for (int e = 0; e < 2; ++e)
            if ((gone >> i & 1) || base + 16 * i + tok_k + 8 * e >= t1) {
              s[i][2 * e] = s[i][2 * e + 1] = -INFINITY;
              vn[i][e] = 0.f;
            }
      }
#pragma unroll
      for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const float x = s[i][2 * e], y = s[i][2 * e + 1];
          if (scores) {
            const int tok = base + 16 * i + tok_k + 8 * e;
            if (tok < t1) {
              float* to = scores +
                          (((int64_t)seg.b * wk.heads + h) * score_width + tok) * wk.group +
                          seg.hb * kHeadsPer + 2 * t;
              if (seg.hb * kHeadsPer + 2 * t < wk.group) to[0] = x;
              if (seg.hb * kHeadsPer + 2 * t + 1 < wk.group) to[1] = y;
            }
          }
          mx0 = fmaxf(mx0, x);
          mx1 = fmaxf(mx1, y);
        }

      auto scale_output = [&](float e0, float e1) {
#pragma unroll
        for (int m = 0; m < KS; ++m) {
          o[m][0] *= e0;
          o[m][1] *= e1;
          o[m][2] *= e0;
          o[m][3] *= e1;
        }
      };
      if (__any_sync(0xffffffffu, mx0 > m0 + kRescale || mx1 > m1 + kRescale)) {
#pragma unroll
        for (int w = 4; w < 32; w <<= 1) {
          mx0 = fmaxf(mx0, __shfl_xor_sync(0xffffffffu, mx0, w));
          mx1 = fmaxf(mx1, __shfl_xor_sync(0xffffffffu, mx1, w));
        }
        mx0 = fmaxf(mx0, m0);
        mx1 = fmaxf(mx1, m1);
        l0 *= ex2(m0 - mx0);
        l1 *= ex2(m1 - mx1);
        // Products so far count for as much less: that much larger is their scale.
        up0 *= ex2(mx0 - m0);
        up1 *= ex2(mx1 - m1);
        if (up0 > kMostUp || up1 > kMostUp) {
          scale_output(up0 > kMostUp ? kMostUp / up0 : 1.f, up1 > kMostUp ? kMostUp / up1 : 1.f);
          up0 = fminf(up0, kMostUp);
          up1 = fminf(up1, kMostUp);
        }
        m0 = mx0;
        m1 = mx1;
      }
      // Softmax weights times value norms, in place of the scores.
      float y0 = 0.f, y1 = 0.f;
#pragma unroll
      for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const float p0 = ex2(s[i][2 * e] - m0), p1 = ex2(s[i][2 * e + 1] - m1);
          l0 += p0;
          l1 += p1;
          s[i][2 * e] = p0 * vn[i][e];
          s[i][2 * e + 1] = p1 * vn[i][e];
          y0 = fmaxf(y0, s[i][2 * e]);
          y1 = fmaxf(y1, s[i][2 * e + 1]);
        }
      if (__any_sync(0xffffffffu, y0 * up0 > kMostWeight || y1 * up1 > kMostWeight)) {
#pragma unroll
        for (int w = 4; w < 32; w <<= 1) {
          y0 = fmaxf(y0, __shfl_xor_sync(0xffffffffu, y0, w));
          y1 = fmaxf(y1, __shfl_xor_sync(0xffffffffu, y1, w));
        }
        // (a power of two: the largest product comes below kWeightScale)
        auto follow = [](float y, float up) {
          return y * up > kMostWeight
                     ? ldexpf(kWeightScale, -min(ilogbf(fminf(y, FLT_MAX)) + 1, 110)) : up;
        };
        const float n0 = follow(y0, up0), n1 = follow(y1, up1);
        scale_output(n0 / up0, n1 / up1);
        up0 = n0;
        up1 = n1;
      }
      // P^T as B operands: tokens of rows 2t, 2t + 1 (and + 8), head g.
      uint32_t ph[MT][2], pl[MT][2];
#pragma unroll
      for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const float x = s[i][2 * e] * up0, y = s[i][2 * e + 1] * up1;
          const uint32_t hi = pack_half2(x, y);
          ph[i][e] = transpose8(hi);
          if constexpr (FINE) {
            const float2 f = unpack_half2(hi);
            pl[i][e] = transpose8(pack_half2(x - f.x, y - f.y));
          }
        }
#pragma unroll
      for (int i = 0; i < MT; ++i) {
        uint32_t vw[4][VD::words];
#pragma unroll
        for (int e = 0; e < 4; ++e)
#pragma unroll
          for (int un = 0; un < VD::units; ++un)
            shared_bytes<VD::UB>(st + vat[e & 1][un] + (i * group + (e >> 1) * 8 * VD::row),
                                 &vw[e][un * VD::UB / 4]);
#pragma unroll
        for (int m = 0; m < KS; m += 2) {
          uint32_t a0[2], a1[2], a2[2], a3[2], c0[2], c1[2], c2[2], c3[2];
          decode_value<VB, FINE, VLO_AT>(vw[0], vw[1], m, vbase, a0, a1, c0, c1);
          decode_value<VB, FINE, VLO_AT>(vw[2], vw[3], m, vbase, a2, a3, c2, c3);
#pragma unroll
          for (int z = 0; z < 2; ++z) {
            if constexpr (FINE) {
              float sum[4] = {};
              mma16816(sum, a0[z], a1[z], a2[z], a3[z], pl[i][0], pl[i][1]);
              mma16816(sum, c0[z], c1[z], c2[z], c3[z], ph[i][0], ph[i][1]);
              mma16816(sum, a0[z], a1[z], a2[z], a3[z], ph[i][0], ph[i][1]);
#pragma unroll
              for (int e = 0; e < 4; ++e) o[m + z][e] += sum[e];
            } else {
              mma16816(o[m + z], a0[z], a1[z], a2[z], a3[z], ph[i][0], ph[i][1]);
            }
          }
        }
      }
      __syncwarp();
    }

    // The next segment's first step comes while this one's partial results are
    // joined, warps in order, by way of each warp's other stage.
    {
      const Segment& x = s_segment[which ^ 1][warp];
      if (x.t0 + warp * 16 * MT < x.t1)
        fetch(x.pid, x.h, x.t0 + warp * 16 * MT, stage0 + p * Shape::stage);
    }
#pragma unroll
    for (int w = 4; w < 32; w <<= 1) {
      l0 += __shfl_xor_sync(0xffffffffu, l0, w);
      l1 += __shfl_xor_sync(0xffffffffu, l1, w);
    }
    if (g == 0) {
      s_m[warp][2 * t] = m0;
      s_m[warp][2 * t + 1] = m1;
      s_l[warp][2 * t] = l0;
      s_l[warp][2 * t + 1] = l1;
      // (2^-14 for the centroids' scale: sums of values of norms up to 2^100 fit f32)
      s_f[warp][2 * t] = 0x1p-14f / up0;
      s_f[warp][2 * t + 1] = 0x1p-14f / up1;
    }
    const int active = min(NW, (t1 - seg.t0 + 16 * MT - 1) / (16 * MT));
    uint8_t* own = smem + Shape::table_bytes + (warp * 2 + (p ^ 1)) * Shape::stage;
    __shared__ const float* s_part[NW];
    if (lane == 0) s_part[warp] = reinterpret_cast<const float*>(own);
    if (warp < active) {
      float* dst = reinterpret_cast<float*>(own) + 2 * t * Shape::ostride;
#pragma unroll
      for (int m = 0; m < KS; ++m) {
        const int dim = VD::dim(g, 2 * m);
        *reinterpret_cast<float2*>(dst + dim) = make_float2(o[m][0], o[m][2]);
        *reinterpret_cast<float2*>(dst + Shape::ostride + dim) = make_float2(o[m][1], o[m][3]);
      }
    }
    __syncthreads();
    const int64_t slot = (int64_t)blockIdx.x + seg.seg;
    const int ng = min(kHeadsPer, wk.group - seg.hb * kHeadsPer);
    for (int hd = warp; hd < kHeadsPer; hd += NW) {
      const bool in = lane < active;
      const float m = in ? s_m[lane][hd] : -FLT_MAX;
      float mm = m;
#pragma unroll
      for (int w = 16; w > 0; w >>= 1) mm = fmaxf(mm, __shfl_xor_sync(0xffffffffu, mm, w));
      const float f = ex2(m - mm);
      float l = in ? s_l[lane][hd] * f : 0.f;
#pragma unroll
      for (int w = 16; w > 0; w >>= 1) l += __shfl_xor_sync(0xffffffffu, l, w);
      if (in) s_f[lane][hd] *= f;
      if (lane == 0) parts.ml[slot * kHeadsPer + hd] = make_float2(mm, l);
    }
    __syncthreads();
    for (int i = tid; i < ng * D; i += Shape::threads) {
      const int hd = i / D, j = i % D;
      float sum = 0.f;
#pragma unroll 4
      for (int w = 0; w < active; ++w)
        sum = fmaf(s_part[w][hd * Shape::ostride + j], s_f[w][hd], sum);
      parts.o[slot * kHeadsPer * D + i] = sum;
    }
    __syncthreads();
  }
}

// One block per segment: its partials in order, 1 / sum, the values' scale,
// and the rotation back.
template <class T, int D>
__global__ void __launch_bounds__(kRotParts * D)
kv_join_kernel(Parts parts, Work wk, int workers, int d, int page_size,
               const float* __restrict__ R, const int* __restrict__ exponent, T* __restrict__ out,
               float* __restrict__ lse, float* __restrict__ lse2) {
  __shared__ __align__(16) float so[kHeadsPer][D];
  __shared__ float s_l[kHeadsPer];
  // The partials' factors [worker][head], then the parts' sums [part][head][D].
  constexpr int room = kRotParts > kMaxWorkers / D ? kRotParts : kMaxWorkers / D;
  __shared__ float red[room][kHeadsPer][D];
  float* fac = &red[0][0][0];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, j = tid % D, part = tid / D;
  const int per = wk.heads * wk.blocks, seg = blockIdx.x;
  const int b = seg / per, seg_in = seg % per, h = seg_in / wk.blocks, hb = seg_in % wk.blocks;
  const int ng = min(kHeadsPer, wk.group - hb * kHeadsPer);
  const int64_t row0 = ((int64_t)b * wk.heads + h) * wk.group + hb * kHeadsPer;
  const float vscale = ldexpf(0x1p14f, -*exponent);
  pdl_next();
  // (The kernel before lets this one in after the queries' kernel has ended: what
  // that one left, in L2, can be read before the wait for the partial results.)
  Turn<D> turn;
  turn.ahead(R, d, j, part);
  const int len = clamp_length(wk.lengths[b], wk.table_width, page_size);
  const int nu = wk.units_of(len), total = __ldcg(wk.first + wk.batch);
  int w0 = 0, nw = 0;
  if (nu) {
    const int n = min(workers, total);
    const int64_t u0 = __ldcg(wk.first + b) + (int64_t)seg_in * nu;
    w0 = worker_of(u0 + wk.empty, n, total);
    nw = worker_of(u0 + nu - 1, n, total) - w0 + 1;
  }
  const int64_t slot0 = (int64_t)w0 + seg;
  pdl_wait();
  if (warp < kHeadsPer) {
    float m = -FLT_MAX, l = 0.f;
    for (int w = lane; w < nw; w += 32)
      m = fmaxf(m, parts.ml[(slot0 + w) * kHeadsPer + warp].x);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
    for (int w = lane; w < nw; w += 32) {
      const float2 ml = parts.ml[(slot0 + w) * kHeadsPer + warp];
      const float f = ex2(ml.x - m);
      l = fmaf(ml.y, f, l);
      fac[w * kHeadsPer + warp] = f;
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) l += __shfl_xor_sync(0xffffffffu, l, o);
    if (lane == 0) {
      s_l[warp] = l;
      if (warp < ng) {
        const float l2 = l == 0.f ? -INFINITY : m + log2f(l);
        if (lse) lse[row0 + warp] = l2 * kLn2;
        if (lse2) lse2[row0 + warp] = l2;
      }
    }
  }
  __syncthreads();
  float acc[kHeadsPer];
#pragma unroll
  for (int g = 0; g < kHeadsPer; ++g) acc[g] = 0.f;
#pragma unroll 4
  for (int w = part; w < nw; w += kRotParts) {
    const float* o = parts.o + (slot0 + w) * kHeadsPer * D + j;
#pragma unroll
    for (int g = 0; g < kHeadsPer; ++g)
      if (g < ng) acc[g] = fmaf(o[g * D], fac[w * kHeadsPer + g], acc[g]);
  }
  __syncthreads();
#pragma unroll
  for (int g = 0; g < kHeadsPer; ++g) red[part][g][j] = acc[g];
  __syncthreads();
  for (int g = part; g < kHeadsPer; g += kRotParts) {
    float x = 0.f;
#pragma unroll
    for (int p = 0; p < kRotParts; ++p) x += red[p][g][j];
    so[g][j] = g >= ng || s_l[g] == 0.f ? 0.f : x / s_l[g] * vscale;
  }
  __syncthreads();
  turn.run(so, acc);
#pragma unroll
  for (int g = 0; g < kHeadsPer; ++g) red[part][g][j] = acc[g];
  __syncthreads();
  if (j < d)
    for (int g = part; g < ng; g += kRotParts) {
      float y = 0.f;
#pragma unroll
      for (int p = 0; p < kRotParts; ++p) y += red[p][g][j];
      out[(row0 + g) * d + j] = from_f32<T>(y);
    }
}

// weights += sum over the key-value head's queries of 2^(score - lse2).
__global__ void __launch_bounds__(256)
kv_weights_kernel(const float* __restrict__ scores, const float* __restrict__ lse2, Work wk,
                  int pages, int page_size, int64_t width, float* __restrict__ weights) {
  const int64_t bh = blockIdx.y + (int64_t)blockIdx.z * gridDim.y;
  if (bh >= (int64_t)wk.batch * wk.heads) return;
  const int b = (int)(bh / wk.heads), h = (int)(bh % wk.heads);
  pdl_wait();
  const int len = clamp_length(wk.lengths[b], wk.table_width, page_size);
  for (int t = blockIdx.x * blockDim.x + threadIdx.x; t < len; t += gridDim.x * blockDim.x) {
    const int pg = wk.table[b * wk.table_stride + t / page_size];
    if (pg < 0 || pg >= pages) continue;
    const float* s = scores + (bh * width + t) * wk.group;
    const float* l = lse2 + bh * wk.group;
    float w = 0.f;
    for (int g = 0; g < wk.group; ++g) w += ex2(s[g] - __ldg(l + g));
    atomicAdd(weights + ((int64_t)pg * wk.heads + h) * page_size + t % page_size, w);
  }
}

// ---------------------------------------------------------------------------
// Host
// ---------------------------------------------------------------------------

struct AttendPlan {
  int D, blocks, segments, workers;
  int64_t rows, width;
  size_t bytes;
  QueryOut q;
  Parts parts;
  int* first;
  float *lse2, *scores;
};

inline AttendPlan attend_plan(const pq_kv_cache& c, int batch, int q_heads, int table_width,
                              int accumulate, void* ws, size_t ws_bytes) {
  AttendPlan p;
  p.D = padded_d(c.d);
  const int group = q_heads / c.heads;
  p.blocks = (group + kHeadsPer - 1) / kHeadsPer;
  p.rows = (int64_t)batch * q_heads;
  p.width = (int64_t)table_width * c.page_size;
  const int64_t segments = (int64_t)batch * c.heads * p.blocks;
  p.segments = (int)segments;
  // A block per SM, never more than the units (of at least kLeastUnit tokens, and
  // a segment's empty ones) that the table has room for.
  const int64_t units = segments * ((kSegmentCost + p.width) / kLeastUnit + 2);
  p.workers = (int)max((int64_t)1, min(units, (int64_t)min(num_sms(), kMaxWorkers)));
  Carve cv(ws, ws_bytes);
  p.q.hi = cv.take<__half>(segments * kHeadsPer * p.D);
  p.q.lo = cv.take<__half>(segments * kHeadsPer * p.D);
  p.q.factor = cv.take<float>(segments * kHeadsPer);
  p.first = cv.take<int>(batch + 1);
  p.parts.o = cv.take<float>((segments + p.workers) * kHeadsPer * p.D);
  p.parts.ml = cv.take<float2>((segments + p.workers) * kHeadsPer);
  p.lse2 = cv.take<float>(p.rows);
  p.scores = accumulate ? cv.take<float>(p.rows * p.width) : nullptr;
  p.bytes = cv.off;
  return p;
}

template <class... KArgs, class... Args>
inline int launch_pdl(void (*kernel)(KArgs...), dim3 grid, int threads, size_t smem,
                      cudaStream_t st, bool early, Args... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute at;
  at.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &at;
  cfg.numAttrs = early ? 1 : 0;
  PQ_CUDA_TRY(cudaLaunchKernelEx(&cfg, kernel, KArgs(args)...));
  PQ_LAUNCH_CHECK("kv attend");
  return PQ_OK;
}

template <int D, int KB, int VB, bool FINE>
int launch_attend(const pq_kv_cache& c, Work wk, const AttendPlan& p, int workers,
                  cudaStream_t st) {
  using Shape = AttendShape<D, KB, VB, FINE>;
  auto kern = kv_attend_kernel<D, KB, VB, FINE>;
  const int page_shift = page_shift_of(c);
  static_assert(Shape::warps >= 4 && Shape::unit >= kLeastUnit, "too little shared memory");
  const int rc = allow_smem<kv_attend_kernel<D, KB, VB, FINE>>(Shape::smem);
  if (rc) return rc;
  return launch_pdl(kern, dim3(workers), Shape::threads, Shape::smem, st, true, side_k(c),
                    side_v(c), c.pages, page_shift, wk, p.q, p.parts, p.scores, p.width);
}

// Calls f with the kernel's template arguments.
template <int D, int KB, int VB, class F>
int with_fine(bool fine, F f) {
  return fine ? f.template operator()<D, KB, VB, true>() : f.template operator()<D, KB, VB, false>();
}
template <int D, int KB, class F>
int with_v(int vb, bool fine, F f) {
  return vb == 2 ? with_fine<D, KB, 2>(fine, f)
                 : vb == 4 ? with_fine<D, KB, 4>(fine, f) : with_fine<D, KB, 8>(fine, f);
}
template <int D, class F>
int with_k(int kb, int vb, bool fine, F f) {
  return kb == 2 ? with_v<D, 2>(vb, fine, f)
                 : kb == 4 ? with_v<D, 4>(vb, fine, f) : with_v<D, 8>(vb, fine, f);
}
template <class F>
int with_shape(int D, int kb, int vb, bool fine, F f) {
  return D == 64 ? with_k<64>(kb, vb, fine, f)
                 : D == 128 ? with_k<128>(kb, vb, fine, f) : with_k<256>(kb, vb, fine, f);
}

struct UnitOf {
  template <int D, int KB, int VB, bool FINE>
  int operator()() const {
    return AttendShape<D, KB, VB, FINE>::unit;
  }
};
struct LaunchAttend {
  const pq_kv_cache& c;
  Work wk;
  const AttendPlan& p;
  int workers;
  cudaStream_t st;
  template <int D, int KB, int VB, bool FINE>
  int operator()() const {
    return launch_attend<D, KB, VB, FINE>(c, wk, p, workers, st);
  }
};

template <class T, int D>
int launch_query(const pq_kv_cache& c, const void* q, int64_t sb, int64_t sh, float scale, Work wk,
                 const AttendPlan& p, cudaStream_t st) {
  const Codec k = codec_of(c.k_codec, c.d);
  return launch_pdl(kv_query_kernel<T, D>, dim3(p.segments + 1), kRotParts * D, 0, st, false, (const T*)q, sb,
                    sh, c.d, c.page_size, k.RT, k.exponent, scale, wk, p.q, p.first);
}

template <class T, int D>
int launch_join(const pq_kv_cache& c, Work wk, const AttendPlan& p, int workers, void* out,
                float* lse, int accumulate, cudaStream_t st) {
  const Codec v = codec_of(c.v_codec, c.d);
  return launch_pdl(kv_join_kernel<T, D>, dim3(p.segments), kRotParts * D, 0, st, true, p.parts, wk, workers,
                    c.d, c.page_size, v.R, v.exponent, (T*)out, lse,
                    accumulate ? p.lse2 : (float*)nullptr);
}

}  // namespace kv
}  // namespace pqb

using namespace pqb;

extern "C" {

size_t pq_kv_attend_workspace_bytes(const pq_kv_cache* cache, int batch, int q_heads,
                                    int table_width, int accumulate) {
  if (!cache || batch <= 0 || q_heads <= 0 || table_width < 0 || cache->heads <= 0) return 256;
  return kv::attend_plan(*cache, batch, q_heads, table_width, accumulate, nullptr, 0).bytes;
}

int pq_kv_attend(const pq_kv_cache* cache, const void* q, int dtype, int64_t q_stride_b,
                 int64_t q_stride_h, const int32_t* table, int64_t table_stride, int table_width,
                 const int32_t* lengths, int batch, int q_heads, float scale, void* out,
                 float* lse, int accumulate, void* ws, size_t ws_bytes, void* stream) {
  int rc = kv::check_cache(cache);
  if (rc) return rc;
  rc = kv::check_dtype(dtype);
  if (rc) return rc;
  const pq_kv_cache& c = *cache;
  rc = kv::check_sequences(table, table_width, lengths, batch, c.page_size);
  if (rc) return rc;
  PQ_CHECK_ARG(q_heads >= 1 && q_heads % c.heads == 0,
               "q_heads must be a multiple of the cache's %d (got %d)", c.heads, q_heads);
  PQ_CHECK_ARG(isfinite(scale), "scale must be finite");
  if (batch == 0) return PQ_OK;
  PQ_CHECK_ARG(q && out, "null pointer argument");
  const int64_t widest =
      (kv::kSegmentCost + (int64_t)table_width * c.page_size) / kv::kLeastUnit + 2;
  PQ_CHECK_ARG((int64_t)batch * q_heads < (1ll << 28) &&
                   (int64_t)batch * q_heads * widest < (1ll << 31),
               "a call takes fewer than 2^28 query rows and 2^31 pieces of 64 tokens");
  const kv::AttendPlan p =
      kv::attend_plan(c, batch, q_heads, table_width, accumulate, ws, ws_bytes);
  if (!ws || ws_bytes < p.bytes)
    return fail(PQ_ERR_WORKSPACE, "pq_kv_attend needs %zu workspace bytes, got %zu", p.bytes,
                ws_bytes);
  const cudaStream_t st = (cudaStream_t)stream;
  const bool fine = dtype != PQ_KV_BF16;
  kv::Work wk;
  wk.table = table;
  wk.table_stride = table_stride;
  wk.table_width = c.pages ? table_width : 0;  // without a pool every sequence is empty
  wk.lengths = lengths;
  wk.batch = batch;
  wk.heads = c.heads;
  wk.group = q_heads / c.heads;
  wk.blocks = p.blocks;
  wk.first = p.first;
  wk.unit = kv::with_shape(p.D, c.k_bits, c.v_bits, fine, kv::UnitOf{});
  wk.empty = (kv::kSegmentCost + wk.unit - 1) / wk.unit;
  const int workers = p.workers;
  PQ_KV_DISPATCH_T(dtype, {
    rc = p.D == 64 ? kv::launch_query<T_, 64>(c, q, q_stride_b, q_stride_h, scale, wk, p, st)
                   : p.D == 128
                         ? kv::launch_query<T_, 128>(c, q, q_stride_b, q_stride_h, scale, wk, p, st)
                         : kv::launch_query<T_, 256>(c, q, q_stride_b, q_stride_h, scale, wk, p, st);
  });
  if (rc) return rc;
  rc = kv::with_shape(p.D, c.k_bits, c.v_bits, fine, kv::LaunchAttend{c, wk, p, workers, st});
  if (rc) return rc;
  PQ_KV_DISPATCH_T(dtype, {
    rc = p.D == 64 ? kv::launch_join<T_, 64>(c, wk, p, workers, out, lse, accumulate, st)
                   : p.D == 128
                         ? kv::launch_join<T_, 128>(c, wk, p, workers, out, lse, accumulate, st)
                         : kv::launch_join<T_, 256>(c, wk, p, workers, out, lse, accumulate, st);
  });
  if (rc) return rc;
  if (accumulate && p.width) {
    const int64_t bh = (int64_t)batch * c.heads;
    const int gy = (int)min(bh, (int64_t)32768);
    const int64_t gx = min((p.width + 255) / 256, max((int64_t)1, (int64_t)16 * num_sms() / bh));
    rc = kv::launch_pdl(kv::kv_weights_kernel, dim3((unsigned)gx, gy, (unsigned)((bh + gy - 1) / gy)),
                        256, 0, st, true, p.scores, p.lse2, wk, c.pages, c.page_size, p.width,
                        c.weights);
    if (rc) return rc;
  }
  return PQ_OK;
}

}  // extern "C"
