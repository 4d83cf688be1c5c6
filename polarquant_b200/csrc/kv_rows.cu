// Rows of the compressed key-value cache: the codec's tables, writing tokens
// (norm, rotation, Lloyd-Max codes, packing, scatter into the pages) and
// reading slots back as vectors.
#include "kv.cuh"
#include "tc.cuh"

#include <type_traits>

namespace pqb {
namespace kv {

// ---------------------------------------------------------------------------
// The codec's tables
// ---------------------------------------------------------------------------

// Entry of a cell, for cells of [i - 1/2, i + 1/2) / scale + lo widened by `slack`:
// the boundary in it and the number of boundaries below that.  A cell without a
// boundary has one at 1e30, a cell with several NaN: their coordinates are
// recomputed exactly.
__device__ uint2 cell_entry(const float* bounds, int count, int i, int cells, float lo, float width,
                            float slack) {
  const float from = i == 0 ? -INFINITY : lo + (i - 0.5f) * width - slack;
  const float to = i == cells - 1 ? INFINITY : lo + (i + 0.5f) * width + slack;
  int below = 0, in = 0;
  for (int k = 0; k < count; ++k) {
    if (bounds[k] < from)
      ++below;
    else if (bounds[k] <= to)
      ++in;
  }
  const float b = in == 0 ? 1e30f : in == 1 ? bounds[below] : __int_as_float(0x7fc00000);
  return make_uint2(__float_as_uint(b), (uint32_t)below);
}

__global__ void prepare_codec_kernel(const float* __restrict__ R, const float* __restrict__ bounds,
                                     const float* __restrict__ cent, int d, int bits, int D,
                                     Codec out) {
  const int t = blockIdx.x * blockDim.x + threadIdx.x, threads = gridDim.x * blockDim.x;
  const int levels = 1 << bits;
  for (int i = t; i < d * d; i += threads) {
    const float v = R[i];
    const_cast<float*>(out.R)[i] = v;
    const_cast<float*>(out.RT)[(i % d) * d + i / d] = v;
  }
  // Planes: operand register r of lane (g, t) for columns of tile n and step s.
  for (int i = t; i < D / 8 * (D / 16) * 32; i += threads) {
    const int lane = i & 31, s = (i >> 5) % (D / 16), n = (i >> 5) / (D / 16);
    const int g = lane >> 2, tt = lane & 3;
    const int col = (g >> 1) * (D / 4) + (n >> 2) * 8 + 2 * (n & 3) + (g & 1);
    __half hi[4], lo[4];
    for (int k = 0; k < 4; ++k) {
      const int row = tt * (D / 4) + 4 * s + k;
      const float v = col < d && row < d ? R[col * d + row] * 16384.f : 0.f;
      hi[k] = __float2half_rn(v);
      lo[k] = __float2half_rn(v - __half2float(hi[k]));
    }
    uint2* p = const_cast<uint2*>(out.planes);
    p[i] = make_uint2(__half_as_ushort(hi[0]) | (uint32_t)__half_as_ushort(hi[1]) << 16,
                      __half_as_ushort(hi[2]) | (uint32_t)__half_as_ushort(hi[3]) << 16);
    p[D / 8 * (D / 16) * 32 + i] =
        make_uint2(__half_as_ushort(lo[0]) | (uint32_t)__half_as_ushort(lo[1]) << 16,
                   __half_as_ushort(lo[2]) | (uint32_t)__half_as_ushort(lo[3]) << 16);
  }
  // The same, row by row.
  for (int i = t; i < D * D; i += threads) {
    const int col = i / D, row = i % D;
    const float v = col < d && row < d ? R[col * d + row] * 16384.f : 0.f;
    const __half hi = __float2half_rn(v);
    __half* p = const_cast<__half*>(out.rows);
    p[i] = hi;
    p[D * D + i] = __float2half_rn(v - __half2float(hi));
  }
  // Cells between the first and the last boundary.
  {
    const int cells = bits == 8 ? kCells : kFewCells;
    const float lo = bounds[0], hi = bounds[levels - 2];
    float width = (hi - lo) / (cells - 1);
    if (!(width > 1e-30f && width < 1e30f)) width = 0.f;  // one cell for all
    const float scale = width > 0.f ? 1.f / (hi - lo) : 0.f;
    for (int i = t; i < cells; i += threads)
      const_cast<uint2*>(out.cells)[i] =
          width > 0.f ? cell_entry(bounds, levels - 1, i, cells, lo, width, 0.01f * width + 1e-5f)
                      : make_uint2(0x7fc00000u, 0u);
    if (t == 0) {
      const_cast<float*>(out.range)[0] = scale;
      const_cast<float*>(out.range)[1] = width > 0.f ? -lo * scale : 0.f;
    }
  }
  if (blockIdx.x) return;
  if (t < 256) {
    const_cast<float*>(out.bounds)[t] = t < levels - 1 ? bounds[t] : INFINITY;
    const_cast<float*>(out.cent)[t] = t < levels ? cent[t] : 0.f;
  }
  __shared__ uint32_t s_half[256];  // hi | lo << 16
  __shared__ int s_mx;
  if (threadIdx.x == 0) s_mx = 0;
  __syncthreads();
  const float c = threadIdx.x < levels ? cent[threadIdx.x] : 0.f;
  atomicMax(&s_mx, __float_as_int(fabsf(c)));  // ordered as the floats are
  __syncthreads();
  const float mx = __int_as_float(s_mx);
  const int e = mx > 0.f ? max(-100, min(100, 13 - ilogbf(mx))) : 0;
  const float x = ldexpf(c, e);
  const __half hi = __float2half_rn(x), lo = __float2half_rn(x - __half2float(hi));
  s_half[threadIdx.x] = __half_as_ushort(hi) | (uint32_t)__half_as_ushort(lo) << 16;
  __syncthreads();
  const int i = threadIdx.x;
  uint2 p0, p1;
  if (bits == 8) {
    p0 = make_uint2(s_half[i], s_half[i]);
    p1 = make_uint2(0u, 0u);
  } else {
    // The byte's codes: two at 4 bits, four at 2.
    uint32_t c[4];
    for (int k = 0; k < 4; ++k)
      c[k] = s_half[bits == 4 ? (k & 1 ? i & 15 : i >> 4) : i >> (6 - 2 * k) & 3];
    p0 = make_uint2(__byte_perm(c[0], c[1], 0x5410), __byte_perm(c[2], c[3], 0x5410));
    p1 = make_uint2(__byte_perm(c[0], c[1], 0x7632), __byte_perm(c[2], c[3], 0x7632));
  }
  const_cast<uint2*>(out.pairs)[i] = p0;
  const_cast<uint2*>(out.pairs)[256 + i] = p1;
  if (i == 0) *const_cast<int*>(out.exponent) = e;
}

// ---------------------------------------------------------------------------
// Append
//
// x -> norm = f32(sqrt(sum_f64 x^2)), u = x / max(norm, 1e-8) in f32, code_j =
// #{boundaries < sum_i u_i R_ji}, exactly.
//
// The rotation runs on the tensor cores in f16 operands and f32 sums: a row's x
// times a power of two is f16 hi (exact for 16-bit inputs but for elements below
// 2^-28 of the largest) or hi + lo (f32), R * 2^14 is hi + lo, and hi*hi + hi*lo
// (+ lo*hi) are summed; the scales and 1 / max(norm, 1e-8) come after.  That is
// within (steps + 8) * 2^-23 of the exact product (each of the sum's `steps`
// additions loses at most 2^-23 of a partial sum, which is at most |u||R_j| = 1;
// operands lose 2^-22): coordinates that near a boundary are recomputed by a
// warp in f64.  So codes do not depend on how the product was taken.
//
// Counting boundaries takes one table lookup: cells narrower than the gaps
// between boundaries hold at most one (from a copy for each lane at 2 and 4
// bits, with the code in the low four bits of the boundary).
//
// Two kernels.  Calls of few rows (kv_append_few_kernel, mma.m16n8k16): a block
// takes 16 rows, its warps 32 columns each, planes of R from L2.  Which column
// and which element stands where in the operands is free, so a lane (g, t) loads
// a quarter of row g from its t-th run of d / 4 elements and gets coordinates of
// the same run back.  Others (kv_append_kernel, tcgen05): below.
// ---------------------------------------------------------------------------

__device__ __forceinline__ void mma_rows(float (&c)[4], const uint32_t (&a)[4], uint2 b) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
      "{%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b.x), "r"(b.y));
}

struct AppendArgs {
  const void *k, *v;
  int64_t k_sn, k_sh, v_sn, v_sh;
  uint32_t rows, heads, first_tile;
  int64_t slots_end;
  int d, page_shift;
  bool k_vec, v_vec;  // rows can be read 16 bytes at a time
  Side sk, sv;
  const int64_t* slots;
  const int32_t* positions;
  const float* weights;
  int32_t* out_pos;
  float* out_w;

  // Index of row r (token r / heads, head r % heads) in the pool; -1 for none.
  __device__ int64_t place(uint32_t r) const {
    const int64_t slot = slots[r / heads];
    if (slot < 0 || slot >= slots_end) return -1;
    const uint32_t s = (uint32_t)slot;
    return ((int64_t)(s >> page_shift) * heads + r % heads << page_shift) +
           (s & ((1u << page_shift) - 1u));
  }
  // What a token holds besides codes, by one thread of a row.
  __device__ void write_token(const Side& sd, bool is_v, uint32_t r, int64_t at,
                              float norm) const {
    sd.norms[at] = norm;
    if (!is_v) {
      out_pos[at] = positions[r / heads];
      out_w[at] = weights ? weights[r] : 0.f;
    }
  }
};

constexpr int kCellWords = 2 * kCells > 32 * kFewCells ? 2 * kCells : 32 * kFewCells;

template <class T, int D>
struct FewShape {
  static constexpr bool wide = sizeof(T) == 4;  // x is hi + lo
  static constexpr int rows = 16;
  static constexpr int steps = D / 16;
  static constexpr int warps = D / 32;          // 32 columns each, 8 a lane
};

// 16 bytes of x as f32.
template <class T>
__device__ __forceinline__ void widen16(const uint4& w, float* f) {
  if constexpr (sizeof(T) == 4) {
    f[0] = __uint_as_float(w.x);
    f[1] = __uint_as_float(w.y);
    f[2] = __uint_as_float(w.z);
    f[3] = __uint_as_float(w.w);
  } else {
    const T* e = reinterpret_cast<const T*>(&w);
#pragma unroll
    for (int k = 0; k < 8; ++k) f[k] = to_f32<T>(e[k]);
  }
}

// The table of cells (kCellWords) and the boundaries in shared memory, by all
// threads of the block.
template <int BITS>
__device__ __forceinline__ void fill_cells(const Codec& cd, uint32_t* s_cell, float* s_bounds) {
  for (int i = threadIdx.x; i < 256; i += blockDim.x) s_bounds[i] = cd.bounds[i];
  if constexpr (BITS == 8) {
    for (int i = threadIdx.x; i < kCells; i += blockDim.x)
      reinterpret_cast<uint2*>(s_cell)[i] = cd.cells[i];
  } else {
    for (int i = threadIdx.x; i < kFewCells * 32; i += blockDim.x) {
      const uint2 c = cd.cells[i >> 5];
      s_cell[i] = (c.x & ~15u) | c.y;
    }
  }
}

// Coding of a product x (a sum of the operands as they are scaled): y = x * inv.
template <int BITS>
struct Coder {
  uint32_t base;  // the lane's place in the table, less what the bits of 2^23 come to in it
  float scale, offset;
  static constexpr int cells = BITS == 8 ? kCells : kFewCells;

  __device__ __forceinline__ Coder(const Codec& cd, const uint32_t* s_cell)
      : base((uint32_t)__cvta_generic_to_shared(s_cell) +
             (BITS == 8 ? 0u : (threadIdx.x & 31) * 4u) - 0x4b000000u * (BITS == 8 ? 8u : 128u)),
        scale(cd.range[0]),
        offset(cd.range[1]) {}

  // Number of boundaries below y, right unless `off`, the distance to the cell's
  // boundary, is within the band or NaN.
  __device__ __forceinline__ uint32_t code(float x, float inv, float& off) const {
    const float cell =
        fmaf(__saturatef(fmaf(x, inv * scale, offset)), (float)(cells - 1), 8388608.f);
    uint32_t e, c;
    if constexpr (BITS == 8) {
      asm("ld.shared.v2.b32 {%0,%1}, [%2];"
          : "=r"(e), "=r"(c)
          : "r"(__float_as_uint(cell) * 8u + base));
    } else {
      asm("ld.shared.b32 %0, [%1];" : "=r"(e) : "r"(__float_as_uint(cell) * 128u + base));
      c = e & 15u;
    }
    off = fmaf(x, inv, -__uint_as_float(e));
    return c + (off > 0.f ? 1u : 0u);
  }
};

// A word of codes of 0.
template <int BITS>
__device__ __noinline__ uint32_t zero_codes(const float* s_bounds) {
  uint32_t code = 0;
#pragma unroll
  for (int step = 1 << (BITS - 1); step > 0; step >>= 1)
    if (0.f > s_bounds[code + step - 1]) code += step;
  return code * (BITS == 8 ? 0x01010101u : BITS == 4 ? 0x11111111u : 0x55555555u);
}

// A boundary below 1 with its low four bits taken loses 15 * 2^-24 < 1e-6.
__host__ __device__ constexpr float band_of(int products, int bits) {
  return (products + 8) * 1.1920929e-7f + (bits == 8 ? 0.f : 1e-6f);
}

// The code of column `col` of the row at x by the exact product, by eight
// neighbouring lanes (all lanes of the warp call it; `valid` ones have a row).
//
// First sum_i x_i R_ji / den in f64: rounding x_i / den to f32 first moves that by
// at most 2^-24 sum |u_i R_ji| <= 2^-24, so only within 1e-7 of a boundary the
// divisions are taken one by one.  All of a lane's loads of 128 coordinates come
// before their use (a loop of one after another made 13 us of an event).
template <class T, int BITS>
__device__ __noinline__ uint32_t exact_code(const T* x, float den, const float* rr,
                                            const float* s_bounds, int d, bool vec, bool valid) {
  const int lane = threadIdx.x & 31;
  constexpr int E = 16 / sizeof(T);
  double y = 0.0;
  if (valid) {
#pragma unroll 1
    for (int j0 = (lane & 7) * 8; j0 < d; j0 += 128) {
      uint4 w[2][8 / E];
      float4 m[2][2];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int j = j0 + 64 * h;
        if (vec && d % 8 == 0 && j < d) {
#pragma unroll
          for (int k = 0; k < 8 / E; ++k) w[h][k] = *reinterpret_cast<const uint4*>(x + j + k * E);
          m[h][0] = __ldg(reinterpret_cast<const float4*>(rr + j));
          m[h][1] = __ldg(reinterpret_cast<const float4*>(rr + j + 4));
        } else {
#pragma unroll
          for (int k = 0; k < 8 / E; ++k) {
            __align__(16) T e[E];
#pragma unroll
            for (int z = 0; z < E; ++z)
              e[z] = j + k * E + z < d ? x[j + k * E + z] : from_f32<T>(0.f);
            w[h][k] = *reinterpret_cast<const uint4*>(e);
          }
          float r[8];
#pragma unroll
          for (int k = 0; k < 8; ++k) r[k] = j + k < d ? __ldg(rr + j + k) : 0.f;
          m[h][0] = make_float4(r[0], r[1], r[2], r[3]);
          m[h][1] = make_float4(r[4], r[5], r[6], r[7]);
        }
      }
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        float f[8];
#pragma unroll
        for (int k = 0; k < 8 / E; ++k) widen16<T>(w[h][k], f + k * E);
        const float r[8] = {m[h][0].x, m[h][0].y, m[h][0].z, m[h][0].w,
                            m[h][1].x, m[h][1].y, m[h][1].z, m[h][1].w};
#pragma unroll
        for (int k = 0; k < 8; ++k) y = fma((double)f[k], (double)r[k], y);
      }
    }
  }
#pragma unroll
  for (int o = 4; o > 0; o >>= 1) y += __shfl_xor_sync(0xffffffffu, y, o);
  y /= (double)den;
  auto count = [&](double v) {
    uint32_t code = 0;
#pragma unroll
    for (int step = 1 << (BITS - 1); step > 0; step >>= 1)
      if (v > (double)s_bounds[code + step - 1]) code += step;
    return code;
  };
  uint32_t code = count(y);
  // (or the sum is not finite, of a row whose norm overflows)
  if (__any_sync(0xffffffffu, valid && !(count(y - 1e-7) == count(y + 1e-7) && isfinite(y)))) {
    y = 0.0;
    if (valid)
      for (int j = lane & 7; j < d; j += 8)
        y = fma((double)__fdiv_rn(to_f32<T>(x[j]), den), (double)__ldg(rr + j), y);
#pragma unroll
    for (int o = 4; o > 0; o >>= 1) y += __shfl_xor_sync(0xffffffffu, y, o);
    code = count(y);
  }
  return code;
}

// Replaces a stored row's code (of a word whose other codes may be replaced at the
// same time).
template <int BITS>
__device__ __forceinline__ void replace_code(uint8_t* row, int col, uint32_t code) {
  const int bit = col * BITS, shift = (bit & 24) + 8 - BITS - (bit & 7);
  uint32_t* word = reinterpret_cast<uint32_t*>(row) + (bit >> 5);
  atomicAnd(word, ~(((1u << BITS) - 1u) << shift));
  atomicOr(word, code << shift);
}

// Replaces the codes of flagged coordinates, four at a time.  `near`: the lane's
// flags; where(from, n, ...) gives the row, column and divisor of lane `from`'s
// flag n; patch(n, code) is called on the lane that had the flag.
template <class T, int BITS, class Where, class Patch>
__device__ __forceinline__ void recompute(uint32_t near, const float* R, const float* s_bounds,
                                          int d, bool vec, Where where, Patch patch) {
  const int lane = threadIdx.x & 31;
  uint32_t pend = __ballot_sync(0xffffffffu, near != 0u);
#pragma unroll 1
  while (pend) {
    int from[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      from[i] = pend ? __ffs(pend) - 1 : -1;
      pend &= pend - 1;
    }
    const int mine = lane < 8 ? from[0] : lane < 16 ? from[1] : lane < 24 ? from[2] : from[3];
    const uint32_t flags = __shfl_sync(0xffffffffu, near, max(mine, 0));
    const int n = max(__ffs(flags) - 1, 0);
    const T* x;
    int col;
    float den;
    where(max(mine, 0), n, x, col, den);
    const uint32_t code =
        exact_code<T, BITS>(x, den, R + (int64_t)col * d, s_bounds, d, vec, mine >= 0);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t c = __shfl_sync(0xffffffffu, code, 8 * i);
      if (lane == from[i]) {
        patch(__ffs(near) - 1, c);
        near &= near - 1;
      }
    }
    if (!pend) pend = __ballot_sync(0xffffffffu, near != 0u);
  }
}

// The same for coordinates of each lane's row at x whose codes are stored already
// (at `to`): flags left[32 * i] for the 32 coordinates from col0 + 32 * i on.
template <class T, int BITS>
__device__ __noinline__ void recompute_stored(const uint32_t* left, int chunks, const T* x,
                                              float den, int col0, const float* R,
                                              const float* s_bounds, int d, bool vec, uint8_t* to) {
#pragma unroll 1
  for (int i = 0; i < chunks; ++i, col0 += 32)
    recompute<T, BITS>(
        left[32 * i], R, s_bounds, d, vec,
        [&](int from, int k, const T*& row, int& col, float& dn) {
          row = reinterpret_cast<const T*>(
              __shfl_sync(0xffffffffu, reinterpret_cast<unsigned long long>(x), from));
          col = min(col0 + k, d - 1);
          dn = __shfl_sync(0xffffffffu, den, from);
        },
        [&](int k, uint32_t code) { replace_code<BITS>(to, col0 + k, code); });
}

// A quarter of a row, from x on (the row's coordinate k0): D / 4 elements.
template <class T, int D>
__device__ __forceinline__ void load_quarter(const T* x, int k0, int d, bool vec,
                                             uint4 (&w)[D / 4 * sizeof(T) / 16]) {
  constexpr int E = 16 / sizeof(T), N = D / 4 / E;
  if (vec) {
#pragma unroll
    for (int j = 0; j < N; ++j)
      w[j] = k0 + j * E < d ? *reinterpret_cast<const uint4*>(x + j * E) : make_uint4(0u, 0u, 0u, 0u);
  } else {
#pragma unroll
    for (int j = 0; j < N; ++j) {
      uint32_t v[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        if constexpr (sizeof(T) == 4) {
          v[k] = k0 + j * E + k < d ? __float_as_uint(to_f32<T>(x[j * E + k])) : 0u;
        } else {
          const uint16_t* p = reinterpret_cast<const uint16_t*>(x) + j * E + 2 * k;
          const int at = k0 + j * E + 2 * k;
          v[k] = (at < d ? p[0] : 0u) | (uint32_t)(at + 1 < d ? p[1] : 0u) << 16;
        }
      }
      w[j] = make_uint4(v[0], v[1], v[2], v[3]);
    }
  }
}

// A row's norm, and the power of two for its f16 planes.  The row is in four
// neighbouring lanes, a quarter each.
struct RowScale {
  float norm, den, up, inv;  // inv: of a sum of scaled operands, to the unit vector's coordinate
};

template <class T, int N>
__device__ __forceinline__ RowScale scale_row(const uint4 (&w)[N]) {
  double s4[4] = {0.0, 0.0, 0.0, 0.0};  // four chains
  float mx = 0.f;
#pragma unroll
  for (int j = 0; j < N; ++j) {
    float f[16 / sizeof(T)];
    widen16<T>(w[j], f);
#pragma unroll
    for (int k = 0; k < 16 / (int)sizeof(T); ++k) {
      s4[k & 3] = fma((double)f[k], (double)f[k], s4[k & 3]);
      mx = fmaxf(mx, fabsf(f[k]));
    }
  }
  double ss = (s4[0] + s4[1]) + (s4[2] + s4[3]);
#pragma unroll
  for (int o = 1; o < 4; o <<= 1) {
    ss += __shfl_xor_sync(0xffffffffu, ss, o);
    mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
  }
  RowScale r;
  r.norm = __double2float_rn(__dsqrt_rn(ss));
  r.den = fmaxf(r.norm, 1e-8f);
  // max |x| * 2^e in [2^14, 2^15): f16's range, and sums of at most 2^29 sqrt(d)
  const int e = mx > 0.f && mx < INFINITY ? max(-126, min(126, 14 - ilogbf(mx))) : 0;
  r.up = __int_as_float((127 + e) << 23);
  r.inv = __int_as_float((127 - e) << 23) / 16384.f / r.den;
  return r;
}

template <class T, int D, int BITS>
__device__ __forceinline__ void append_few(const AppendArgs& a, uint32_t* s_cell, float* s_bounds) {
  using S = FewShape<T, D>;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const bool is_v = blockIdx.y != 0;
  const Side& sd = is_v ? a.sv : a.sk;
  const Codec& cd = sd.c;
  const T* src = reinterpret_cast<const T*>(is_v ? a.v : a.k);
  const int64_t sn = is_v ? a.v_sn : a.k_sn, sh = is_v ? a.v_sh : a.k_sh;
  const int d = a.d;
  const uint32_t rows = a.rows, heads = a.heads, row0 = blockIdx.x * S::rows;
  fill_cells<BITS>(cd, s_cell, s_bounds);
  __syncthreads();
  const Coder<BITS> coder(cd, s_cell);
  constexpr float band = band_of(S::steps * (S::wide ? 3 : 2), BITS);

  // Rows g and g + 8: registers 0 and 2 of the A operand hold the first, 1 and 3
  // the second.
  uint32_t ah[S::steps][4], al[S::wide ? S::steps : 1][4];
  float inv[2], den[2];
  bool zero[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const uint32_t r = min(row0 + g + 8 * i, rows - 1);
    const T* x = src + (int64_t)(r / heads) * sn + (r % heads) * sh + t * (D / 4);
    constexpr int E = 16 / sizeof(T), N = D / 4 / E;
    uint4 w[N];
    load_quarter<T, D>(x, t * (D / 4), d, is_v ? a.v_vec : a.k_vec, w);
    const RowScale rs = scale_row<T>(w);
    inv[i] = rs.inv;
    den[i] = rs.den;
    zero[i] = rs.norm == 0.f;
    if (t == 0 && warp == 0 && row0 + g + 8 * i < rows) {
      const int64_t at = a.place(r);
      if (at >= 0) a.write_token(sd, is_v, r, at, rs.norm);
    }
#pragma unroll
    for (int j = 0; j < N; ++j) {
      float f[E];
      widen16<T>(w[j], f);
#pragma unroll
      for (int k = 0; k < E; k += 2) {
        const int n = j * E + k, s = n >> 2, h = (n >> 1) & 1;
        const __half2 hi = __floats2half2_rn(f[k] * rs.up, f[k + 1] * rs.up);
        ah[s][2 * h + i] = *reinterpret_cast<const uint32_t*>(&hi);
        if constexpr (S::wide) {
          const float2 b = __half22float2(hi);
          const __half2 lo = __floats2half2_rn(f[k] * rs.up - b.x, f[k + 1] * rs.up - b.y);
          al[s][2 * h + i] = *reinterpret_cast<const uint32_t*>(&lo);
        }
      }
    }
  }
  float acc[4][4];
#pragma unroll
  for (int q = 0; q < 4; ++q) acc[q][0] = acc[q][1] = acc[q][2] = acc[q][3] = 0.f;
  const uint2* bp = cd.planes + warp * 4 * S::steps * 32 + lane;
#pragma unroll
  for (int s = 0; s < S::steps; ++s)
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const uint2 bh = __ldg(bp + (q * S::steps + s) * 32);
      const uint2 bl = __ldg(bp + (D / 8 + q) * S::steps * 32 + s * 32);
      mma_rows(acc[q], ah[s], bh);
      mma_rows(acc[q], ah[s], bl);
      if constexpr (S::wide) mma_rows(acc[q], al[s], bh);
    }
  // Codes of columns t * D / 4 + warp * 8 + k: packed, the first code highest in
  // its byte, and which of them are next to a boundary.
  constexpr int cw = BITS == 8 ? 2 : 1;
  const int col0 = t * (D / 4) + warp * 8;
  uint32_t packed[2][cw], near = 0;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
#pragma unroll
    for (int w = 0; w < cw; ++w) packed[i][w] = 0u;
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      float off;
      uint32_t code = coder.code(acc[k >> 1][2 * i + (k & 1)], inv[i], off);
      if (col0 + k >= d) code = 0u;
      if (!(fabsf(off) >= band) && col0 + k < d && row0 + g + 8 * i < rows)
        near |= 1u << (8 * i + k);
      const int bit = k * BITS;
      packed[i][bit >> 5] |= code << ((bit & 24) + 8 - BITS - (bit & 7));
    }
    if (zero[i]) {  // all coordinates 0, which may be next to a boundary
      near &= ~(255u << (8 * i));
      const uint32_t word = zero_codes<BITS>(s_bounds);
#pragma unroll
      for (int w = 0; w < cw; ++w) packed[i][w] = 0u;
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const int bit = k * BITS;
        if (col0 + k < d)
          packed[i][bit >> 5] |=
              word & ((1u << BITS) - 1u) << ((bit & 24) + 8 - BITS - (bit & 7));
      }
    }
  }
  recompute<T, BITS>(
      near, cd.R, s_bounds, d, is_v ? a.v_vec : a.k_vec,
      [&](int from, int n, const T*& x, int& col, float& dn) {
        const uint32_t r = min(row0 + (from >> 2) + 8 * (n >> 3), rows - 1);
        x = src + (int64_t)(r / heads) * sn + (r % heads) * sh;
        col = min((from & 3) * (D / 4) + warp * 8 + (n & 7), d - 1);
        const float d0 = __shfl_sync(0xffffffffu, den[0], from);
        const float d1 = __shfl_sync(0xffffffffu, den[1], from);
        dn = n >> 3 ? d1 : d0;
      },
      [&](int n, uint32_t code) {
        const int bit = (n & 7) * BITS, shift = (bit & 24) + 8 - BITS - (bit & 7);
#pragma unroll
        for (int z = 0; z < 2; ++z)
#pragma unroll
          for (int w = 0; w < cw; ++w)
            if (z == n >> 3 && w == bit >> 5)
              packed[z][w] = (packed[z][w] & ~(((1u << BITS) - 1u) << shift)) | code << shift;
      });
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const uint32_t r = row0 + g + 8 * i;
    if (r >= rows) break;
    const int64_t at = a.place(r);
    const int off = col0 * BITS / 8;
    if (at < 0 || off >= sd.ldb) continue;
    uint8_t* to = sd.rows + at * sd.ldb + off;
    if constexpr (BITS == 8)
      *reinterpret_cast<uint2*>(to) = make_uint2(packed[i][0], packed[i][1]);
    else if constexpr (BITS == 4)
      *reinterpret_cast<uint32_t*>(to) = packed[i][0];
    else
      *reinterpret_cast<uint16_t*>(to) = (uint16_t)packed[i][0];
  }
}

template <class T, int D>
__global__ void __launch_bounds__(32 * FewShape<T, D>::warps, 1)
kv_append_few_kernel(AppendArgs a) {
  __shared__ __align__(16) uint32_t s_cell[kCellWords];
  __shared__ float s_bounds[256];
  const int bits = blockIdx.y ? a.sv.bits : a.sk.bits;
  if (bits == 2)
    append_few<T, D, 2>(a, s_cell, s_bounds);
  else if (bits == 4)
    append_few<T, D, 4>(a, s_cell, s_bounds);
  else
    append_few<T, D, 8>(a, s_cell, s_bounds);
}

// ---------------------------------------------------------------------------
// Append of many rows.  A persistent block per SM takes one side (at D = 256 a
// part of its columns too), with R's planes resident in shared memory, and tiles
// of 128 rows: sixteen warps load rows (four lanes a row; the next tile's are on
// their way while this one's are scaled) and split them into 128-byte-swizzled
// K-major f16 tiles; one thread issues the tcgen05.mma (M = 128, N = the block's
// columns) into one of two TMEM accumulators; eight other warps read an accumulator, a
// lane per row, code, pack and store it.  The three run on different tiles.
//
// Bound by the two ends' instructions and the waits between them: 196608 rows of
// either side, bf16, d = 128, 4 bits, take 101 us, 1.3 TB/s of 6.4; 50 % of the
// issue slots, 34 % of the ALUs and 12 % of the tensor pipe are taken.  768 threads
// leave 80 registers each, and all but the 16-bit kernels of D = 64 spill (268 bytes
// of stores a thread here, 1000 at D = 256): the longest waits are for local memory
// and rows alike (long scoreboard 4.8 of 11 cycles between a warp's instructions).
// ---------------------------------------------------------------------------

// tc::mbar_wait that sleeps: the waiting warps would otherwise issue as many
// instructions as the working ones (10 us).
__device__ __forceinline__ bool wait(uint32_t bar, uint32_t parity, volatile int* abort, int err) {
  if (tc::mbar_try_wait(bar, parity)) return true;
  const long long t0 = clock64();
  while (true) {
    __nanosleep(20);
    if (tc::mbar_try_wait(bar, parity)) return true;
    if (*abort) return false;
    if (clock64() - t0 > tc::kWaitCycles) {
      *abort = err;
      device_fail(err);
      return false;
    }
  }
}

template <class T, int D>
struct ManyShape {
  static constexpr bool wide = sizeof(T) == 4;
  static constexpr int planes = wide ? 2 : 1;
  static constexpr int cols = D <= 128 ? D : wide ? 64 : 128;  // of a block
  static constexpr int parts = D / cols;
  static constexpr int kblocks = D / 64;                      // of 64 elements, 128 bytes a row
  static constexpr int a_bytes = planes * kblocks * 128 * 128;
  static constexpr int b_bytes = 2 * kblocks * cols * 128;
  static constexpr int buffers = D <= 64 || (D == 128 && !wide) ? 2 : 1;
  // Coordinates to recompute that a block lists, and the tiles it takes in a
  // launch: about half to three quarters of the list at 8 bits and normal data.
  static constexpr int listed = D <= 128 ? 2048 : 1024;
  static constexpr int most_tiles = D <= 128 ? 24 : 8;
  static constexpr int tmem = 2 * cols;
  // (8 * 2 * cols: flags of what does not fit the list, eight warps' cols / 2 words.)
  static constexpr int smem = 1024 + b_bytes + buffers * a_bytes + 4 * kCellWords + 1024 + 9 * listed +
                              8 * 2 * cols;
};
constexpr int kCodeWarps = 8, kLoadWarps = 16;
constexpr int kManyThreads = 32 * (kCodeWarps + kLoadWarps);

template <class T, int D, int BITS>
__device__ __forceinline__ void append_many(const AppendArgs& a, uint8_t* smem, float (*s_inv)[128],
                                            float (*s_norm)[128], uint32_t bars, uint32_t tmem,
                                            volatile int* abort, int* s_listed) {
  using S = ManyShape<T, D>;
  constexpr int NB = S::buffers;
  uint8_t* s_b = smem;
  uint8_t* s_a = smem + S::b_bytes;
  uint32_t* s_cell = reinterpret_cast<uint32_t*>(smem + S::b_bytes + NB * S::a_bytes);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const bool is_v = blockIdx.y & 1;
  const int part = blockIdx.y >> 1;
  const Side& sd = is_v ? a.sv : a.sk;
  const Codec& cd = sd.c;
  const T* src = reinterpret_cast<const T*>(is_v ? a.v : a.k);
  const int64_t sn = is_v ? a.v_sn : a.k_sn, sh = is_v ? a.v_sh : a.k_sh;
  const int d = a.d;
  const uint32_t rows = a.rows, heads = a.heads;
  const uint32_t first = blockIdx.x + a.first_tile;

  // R's planes: [plane][kblock][column][64], 16-byte pieces exchanged by row & 7.
  for (int i = threadIdx.x; i < 2 * S::cols * (D / 8); i += kManyThreads) {
    const int piece = i % (D / 8), col = i / (D / 8) % S::cols, plane = i / (D / 8) / S::cols;
    const uint4 v = *reinterpret_cast<const uint4*>(cd.rows + (size_t)plane * D * D +
                                                    (size_t)(part * S::cols + col) * D + piece * 8);
    const int kb = piece >> 3, c = piece & 7;
    *reinterpret_cast<uint4*>(s_b + ((plane * S::kblocks + kb) * S::cols + col) * 128 +
                              ((c ^ (col & 7)) << 4)) = v;
  }
  float* s_bounds = reinterpret_cast<float*>(s_cell + kCellWords);
  float* l_den = s_bounds + 256;  // the list: divisor, row, column
  uint32_t* l_row = reinterpret_cast<uint32_t*>(l_den + S::listed);
  uint8_t* l_col = reinterpret_cast<uint8_t*>(l_row + S::listed);
  fill_cells<BITS>(cd, s_cell, s_bounds);
  asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  __syncthreads();

  const uint32_t AFULL = bars, AEMPTY = bars + 16, TFULL = bars + 32, TEMPTY = bars + 48,
                 DRAIN = bars + 64;
  const uint32_t tiles = min((rows + 127) / 128, a.first_tile + gridDim.x * S::most_tiles);
  if (warp >= kCodeWarps) {
    // ---- rows into A tiles: 8 rows a warp, four lanes a row ----
    const int t = lane & 3, lr = (warp - kCodeWarps) * 8 + (lane >> 2);  // row of the tile
    const bool vec = is_v ? a.v_vec : a.k_vec;
    constexpr int E = 16 / sizeof(T), N = D / 4 / E;
    constexpr bool AHEAD = N <= 2;  // registers for two tiles' rows (D = 64; above, spills cost more)
    uint4 w[N], w1[AHEAD ? N : 1];
    auto load = [&](uint32_t tile, uint4 (&to)[N]) {
      const uint32_t r = min(tile * 128 + lr, rows - 1);
      const T* x = src + (int64_t)(r / heads) * sn + (r % heads) * sh + t * (D / 4);
      load_quarter<T, D>(x, t * (D / 4), d, vec, to);
    };
    // The products of the block's n-th tile, by one thread of the first of these
    // warps, once all of them have brought their rows.
    auto multiply = [&](uint32_t n) {
      bool ok = true;
      if (lane == 0) {
        const int buf = n % NB, acc = n & 1;
        ok = wait(TEMPTY + 8 * acc, ((n >> 1) & 1) ^ 1, abort, tc::kErrWaitAccEmpty) &&
             wait(AFULL + 8 * buf, (n / NB) & 1, abort, tc::kErrWaitTmaFull);
        if (ok) {
          tc::tc_fence_after();
          const uint32_t idesc = tc::idesc_f16_f32(128, S::cols);
          const uint32_t a0 = tc::smem_u32(s_a) + buf * S::a_bytes, b0 = tc::smem_u32(s_b);
          const uint32_t dt = tmem + acc * S::cols;
#pragma unroll 1
          for (int kb = 0; kb < S::kblocks; ++kb) {
            const uint32_t ah = a0 + kb * 128 * 128, bh = b0 + kb * S::cols * 128;
            const uint32_t al = ah + S::kblocks * 128 * 128, bl = bh + S::kblocks * S::cols * 128;
#pragma unroll
            for (int kk = 0; kk < 4; ++kk) {
              const uint32_t off = kk * 32;
              tc::mma_f16(dt, tc::sw128_desc(ah + off), tc::sw128_desc(bh + off), idesc,
                          (kb | kk) != 0);
              tc::mma_f16(dt, tc::sw128_desc(ah + off), tc::sw128_desc(bl + off), idesc, 1);
              if constexpr (S::wide)
                tc::mma_f16(dt, tc::sw128_desc(al + off), tc::sw128_desc(bh + off), idesc, 1);
            }
          }
          tc::mma_commit(AEMPTY + 8 * buf);
          tc::mma_commit(TFULL + 8 * acc);
          tc::mbar_arrive(TFULL + 8 * acc);  // hands on what the loading warps wrote besides
        }
      }
      return __shfl_sync(0xffffffffu, (int)ok, 0) != 0;
    };
    uint32_t n = 0;
    if (first < tiles) load(first, w);
    for (uint32_t tile = first; tile < tiles; tile += gridDim.x, ++n) {
      const int buf = n % NB;
      const bool more = tile + gridDim.x < tiles;
      if constexpr (AHEAD)
        if (more) load(tile + gridDim.x, w1);
      const RowScale rs = scale_row<T>(w);
      if (!wait(AEMPTY + 8 * buf, ((n / NB) & 1) ^ 1, abort, tc::kErrWaitStageEmpty)) break;
      uint8_t* dst = s_a + buf * S::a_bytes;
      if (t == 0) {
        s_inv[n & 3][lr] = rs.inv;
        s_norm[n & 3][lr] = rs.norm;
      }
      // Pieces of eight f16.
#pragma unroll
      for (int p = 0; p < D / 32; ++p) {
        uint32_t hi[4], lo[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          float f[E];
          widen16<T>(w[(8 * p + 2 * k) / E], f);
          const float x0 = f[(8 * p + 2 * k) % E] * rs.up, x1 = f[(8 * p + 2 * k) % E + 1] * rs.up;
          const __half2 h = __floats2half2_rn(x0, x1);
          hi[k] = *reinterpret_cast<const uint32_t*>(&h);
          if constexpr (S::wide) {
            const float2 b = __half22float2(h);
            const __half2 l = __floats2half2_rn(x0 - b.x, x1 - b.y);
            lo[k] = *reinterpret_cast<const uint32_t*>(&l);
          }
        }
        const int piece = t * (D / 32) + p, kb = piece >> 3, c = piece & 7;
        uint8_t* to = dst + (kb * 128 + lr) * 128 + ((c ^ (lr & 7)) << 4);
        *reinterpret_cast<uint4*>(to) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
        if constexpr (S::wide)
          *reinterpret_cast<uint4*>(to + S::kblocks * 128 * 128) =
              make_uint4(lo[0], lo[1], lo[2], lo[3]);
      }
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      __syncwarp();
      if (lane == 0) tc::mbar_arrive(AFULL + 8 * buf);
      if (warp == kCodeWarps && !multiply(n)) break;
      if constexpr (AHEAD) {
#pragma unroll
        for (int j = 0; j < N; ++j) w[j] = w1[j];
      } else {
        if (more) load(tile + gridDim.x, w);
      }
    }
    if (warp == kCodeWarps && lane == 0) {
      // Before the block ends, every product that was issued has completed.
      tc::mma_commit(DRAIN);
      volatile int never = 0;
      wait(DRAIN, 0, &never, tc::kErrWaitAccFull);
    }
    __syncwarp();
  } else {
    // ---- accumulators into codes: warps w and w + 4 the halves of the columns ----
    const int q = warp & 3, half = warp >> 2;
    const Coder<BITS> coder(cd, s_cell);
    constexpr float band = band_of(S::kblocks * 4 * (S::wide ? 3 : 2), BITS);
    // Flags behind the list's end: chunks of 32 columns, a word a lane.
    constexpr int chunks = S::cols / 64;
    uint32_t* s_left = reinterpret_cast<uint32_t*>(l_col + S::listed) + warp * (S::cols / 2);
    uint32_t n = 0;
    auto place = [&](uint32_t tile) {
      const uint32_t r = tile * 128 + q * 32 + lane;
      return tile < tiles && r < rows ? a.place(r) : (int64_t)-1;
    };
    int64_t next = place(first);
    for (uint32_t tile = first; tile < tiles; tile += gridDim.x, ++n) {
      const int acc = n & 1;
      if (!wait(TFULL + 8 * acc, (n >> 1) & 1, abort, tc::kErrWaitAccFull)) break;
      tc::tc_fence_after();
      const uint32_t row = tile * 128 + q * 32 + lane;
      const float inv = s_inv[n & 3][q * 32 + lane], norm = s_norm[n & 3][q * 32 + lane];
      const float den = fmaxf(norm, 1e-8f);
      const int64_t at = next;
      next = place(tile + gridDim.x);
      if (half == 0 && part == 0 && at >= 0) a.write_token(sd, is_v, row, at, norm);
      uint8_t* to = sd.rows + at * sd.ldb;
      uint32_t over = 0;
#pragma unroll 1
      for (int c = half * (S::cols / 2); c < (half + 1) * (S::cols / 2); c += 32) {
        uint32_t v[32];
        __syncwarp();
        tc::tmem_ld32(tmem + ((uint32_t)(32 * q) << 16) + acc * S::cols + c, v);
        tc::tmem_ld_wait(v);
        const int col0 = part * S::cols + c, left = d - col0;
        if (left <= 0) {
          // Columns behind the row's end: zeros up to its padded length.
          s_left[(c % (S::cols / 2)) + lane] = 0u;
          const int off = col0 * BITS / 8;
          if (at >= 0)
            for (int j = off; j < min(off + 4 * BITS, (int)sd.ldb); j += 4)
              *reinterpret_cast<uint32_t*>(to + j) = 0u;
          continue;
        }
        uint32_t packed[BITS], near = 0;
#pragma unroll
        for (int w = 0; w < BITS; ++w) {
          constexpr int per = 32 / BITS;
          uint32_t x = 0;
#pragma unroll
          for (int k = 0; k < per; ++k) {
            float off;
            const uint32_t code = coder.code(__uint_as_float(v[w * per + k]), inv, off);
            if (!(fabsf(off) >= band)) near |= 1u << (w * per + k);
            if constexpr (BITS == 8)
              x |= code << (8 * k);
            else
              x = (x << BITS) + code;
          }
          packed[w] = BITS == 8 ? x : __byte_perm(x, 0u, 0x0123);
        }
        if (left < 32) near &= (1u << left) - 1u;
        if (at < 0) near = 0u;
        if (near && norm == 0.f) {  // all coordinates 0, next to a boundary
          near = 0u;
          const uint32_t word = zero_codes<BITS>(s_bounds);
#pragma unroll
          for (int w = 0; w < BITS; ++w) packed[w] = word;
        }
        if (left < 32) {
#pragma unroll
          for (int w = 0; w < BITS; ++w) {
            const int keep = min(max(left * BITS - 32 * w, 0), 32);  // bits, from the first code on
            const uint32_t m = keep >= 32 ? 0xffffffffu : ~(0xffffffffu >> keep);
            packed[w] &= __byte_perm(m, 0u, 0x0123);
          }
        }
        // Coordinates next to a boundary go to the list.  Those behind its end (of many
        // equal rows, say) are recomputed after the tile: in this loop the call would
        // cost it registers (120 us instead of 104).
        if (near) {
          const int cnt = __popc(near);
          int i = atomicAdd(s_listed, cnt);
#pragma unroll 1
          while (near && i < S::listed) {
            l_den[i] = den;
            l_row[i] = row;
            l_col[i] = (uint8_t)(col0 + __ffs(near) - 1);
            near &= near - 1;
            ++i;
          }
        }
        s_left[(c % (S::cols / 2)) + lane] = near;
        over |= near;
        if (at >= 0) {
          const int off = col0 * BITS / 8;
          if constexpr (BITS == 2) {
            if (off < sd.ldb) *reinterpret_cast<uint2*>(to + off) = make_uint2(packed[0], packed[1]);
          } else {
#pragma unroll
            for (int w = 0; w < BITS; w += 4)
              if (off + 4 * w < sd.ldb)
                *reinterpret_cast<uint4*>(to + off + 4 * w) =
                    make_uint4(packed[w], packed[w + 1], packed[w + 2], packed[w + 3]);
          }
        }
      }
      tc::tc_fence_before();
      __syncwarp();
      if (lane == 0) tc::mbar_arrive(TEMPTY + 8 * acc);
      if (__any_sync(0xffffffffu, over != 0u)) {
        const uint32_t r = min(row, rows - 1);
        recompute_stored<T, BITS>(s_left + lane, chunks,
                                  src + (int64_t)(r / heads) * sn + (r % heads) * sh, den,
                                  part * S::cols + half * (S::cols / 2), cd.R, s_bounds, d,
                                  is_v ? a.v_vec : a.k_vec, to);
      }
    }
  }

  // The listed coordinates, by all warps, into the rows as they are stored (codes
  // of one word may be replaced at the same time: by atomics on their own bits).
  __syncthreads();
  const int listed = min(*s_listed, S::listed);
#pragma unroll 1
  for (int e0 = warp * 4; e0 < listed; e0 += kManyThreads / 32 * 4) {
    const int e = min(e0 + (lane >> 3), listed - 1);
    const bool valid = e0 + (lane >> 3) < listed;
    const uint32_t r = l_row[e];
    const int col = l_col[e];
    const uint32_t code = exact_code<T, BITS>(
        src + (int64_t)(r / heads) * sn + (r % heads) * sh, l_den[e], cd.R + (int64_t)col * d,
        s_bounds, d, is_v ? a.v_vec : a.k_vec, valid);
    if (valid && (lane & 7) == 0) {
      replace_code<BITS>(sd.rows + a.place(r) * sd.ldb, col, code);
    }
  }
}

template <class T, int D>
__global__ void __launch_bounds__(kManyThreads, 1) kv_append_kernel(AppendArgs a) {
  using S = ManyShape<T, D>;
  extern __shared__ __align__(16) uint8_t smem_raw[];
  __shared__ float s_inv[4][128], s_norm[4][128];
  __shared__ __align__(8) uint64_t s_bar[9];
  __shared__ uint32_t s_tmem;
  __shared__ int s_abort, s_listed;
  const uint32_t raw = tc::smem_u32(smem_raw);
  uint8_t* smem = smem_raw + (((raw + 1023u) & ~1023u) - raw);
  const uint32_t bars = tc::smem_u32(s_bar);
  if (threadIdx.x == 0) {
    for (int i = 0; i < 2; ++i) {
      tc::mbar_init(bars + 8 * i, kLoadWarps);       // AFULL: the loading warps
      tc::mbar_init(bars + 16 + 8 * i, 1);           // AEMPTY: a commit
      tc::mbar_init(bars + 32 + 8 * i, 2);           // TFULL: a commit and the thread itself
      tc::mbar_init(bars + 48 + 8 * i, kCodeWarps);  // TEMPTY: the coding warps
    }
    tc::mbar_init(bars + 64, 1);
    s_abort = s_listed = 0;
    tc::fence_barrier_init();
  }
  if (threadIdx.x >> 5 == kCodeWarps) tc::tmem_alloc(tc::smem_u32(&s_tmem), S::tmem);
  tc::tc_fence_before();
  __syncthreads();
  tc::tc_fence_after();
  const uint32_t tmem = s_tmem;
  const int bits = blockIdx.y & 1 ? a.sv.bits : a.sk.bits;
  if (bits == 2)
    append_many<T, D, 2>(a, smem, s_inv, s_norm, bars, tmem, &s_abort, &s_listed);
  else if (bits == 4)
    append_many<T, D, 4>(a, smem, s_inv, s_norm, bars, tmem, &s_abort, &s_listed);
  else
    append_many<T, D, 8>(a, smem, s_inv, s_norm, bars, tmem, &s_abort, &s_listed);
  tc::tc_fence_before();
  __syncthreads();
  if (threadIdx.x >> 5 == kCodeWarps) {
    tc::tc_fence_after();
    tc::tmem_dealloc(tmem, S::tmem);
  }
}

template <class T, int D>
int launch_append(const AppendArgs& a, cudaStream_t st) {
  // Few rows, one wave of blocks of 16 on either side of the cache: R's planes from
  // L2 (bf16, D = 128, 4 bits: 256 rows in 9.8 us next to 14.9 by the other kernel,
  // 2368 in 10.3 next to 15.4; 4736 would take 17.9).
  if (a.rows <= 16u * num_sms()) {
    using S = FewShape<T, D>;
    kv_append_few_kernel<T, D>
        <<<dim3((a.rows + S::rows - 1) / S::rows, 2), 32 * S::warps, 0, st>>>(a);
    PQ_LAUNCH_CHECK("kv_append_few_kernel");
    return PQ_OK;
  }
  using S = ManyShape<T, D>;
  auto kern = kv_append_kernel<T, D>;
  const int rc = allow_smem<kv_append_kernel<T, D>>(S::smem);
  if (rc) return rc;
  const uint32_t tiles = (a.rows + 127) / 128;
  const dim3 grid(min(tiles, (uint32_t)max(1, num_sms() / (2 * S::parts))), 2 * S::parts);
  AppendArgs part = a;
  for (part.first_tile = 0; part.first_tile < tiles; part.first_tile += grid.x * S::most_tiles) {
    kern<<<grid, kManyThreads, S::smem, st>>>(part);
    PQ_LAUNCH_CHECK("kv_append_kernel");
  }
  return PQ_OK;
}

// ---------------------------------------------------------------------------
// Read: norm * centroid[code], rounded once.
//
// A lane takes 16 codes of a row; a warp 32 such pieces of one token.  2 x 196608
// rows of d = 128, 4 bits, to bf16: 33 us, 4.0 TB/s of codes read and vectors written,
// 0.62 of a copy's rate.  Bound by the wait for codes, of which a warp has one task's
// on the way (long scoreboard 6.5 of 18 cycles between a warp's instructions), and by
// instructions (58 % of the issue slots).  The lookups are from tables with a copy
// for each lane (or each pair of lanes half a warp apart, for 64-bit entries): an
// f32 centroid at 8 bits, both of a byte's at 4, both of a nibble's at 2.
// ---------------------------------------------------------------------------

struct ReadArgs {
  Side sk, sv;
  const int64_t* slots;
  int64_t slots_end;
  uint32_t tasks;
  int heads, d, page_shift, pieces, per_token;  // 16-code pieces of a row, warps of a token
  bool vec;                                    // rows of the output are 16-byte aligned
  void *k, *v;
};

constexpr int kReadThreads = 512;

template <class T, int BITS>
__device__ __forceinline__ void read_rows(const ReadArgs& a, uint32_t* table) {
  const bool is_v = blockIdx.y != 0;
  const Side& s = is_v ? a.sv : a.sk;
  T* out = reinterpret_cast<T*>(is_v ? a.v : a.k);
  const int lane = threadIdx.x & 31;
  constexpr int entries = BITS == 2 ? 16 : 256;  // of 128 bytes
  for (int i = threadIdx.x; i < entries * 32; i += kReadThreads) {
    const int e = i >> 5;
    float c;
    if (BITS == 8)
      c = s.c.cent[e];
    else
      c = s.c.cent[i & 1 ? e & ((1 << BITS) - 1) : e >> BITS];
    table[i] = __float_as_uint(c);
  }
  __syncthreads();
  const uint32_t base = (uint32_t)__cvta_generic_to_shared(table) +
                        (BITS == 8 ? lane * 4 : (lane & 15) * 8);
  // A task is a warp's 32 pieces of a token; the next task's codes are on their way
  // while this one's are decoded.
  struct Piece {
    uint32_t x[BITS == 8 ? 4 : BITS == 4 ? 2 : 1];
    float norm;
    bool there;    // a slot of the pool
    int left;      // codes of the row from here on; 0 for no piece
    int64_t to;
  };
  const uint32_t step = gridDim.x * (kReadThreads / 32);
  auto fetch = [&](uint32_t w) {
    Piece p;
    p.there = false;
    p.left = 0;
    p.norm = 0.f;
    p.to = 0;
    if (w >= a.tasks) return p;
    const uint32_t tok = a.per_token == 1 ? w : w / (uint32_t)a.per_token;
    const uint32_t unit = (w - tok * a.per_token) * 32 + lane, h = unit / (uint32_t)a.pieces,
                   piece = unit - h * a.pieces;
    if (h >= (uint32_t)a.heads) return p;
    const int64_t slot = a.slots[tok];
    p.left = a.d - (int)piece * 16;
    p.to = ((int64_t)tok * a.heads + h) * a.d + piece * 16;
    p.there = slot >= 0 && slot < a.slots_end;
    if (p.there) {
      const uint32_t sl = (uint32_t)slot;
      const uint32_t at = (((sl >> a.page_shift) * a.heads + h) << a.page_shift) +
                          (sl & ((1u << a.page_shift) - 1u));
      const uint8_t* row = s.rows + (uint64_t)at * (uint32_t)s.ldb + piece * (2 * BITS);
      if constexpr (BITS == 8)
        *reinterpret_cast<uint4*>(p.x) = *reinterpret_cast<const uint4*>(row);
      else if constexpr (BITS == 4)
        *reinterpret_cast<uint2*>(p.x) = *reinterpret_cast<const uint2*>(row);
      else
        p.x[0] = *reinterpret_cast<const uint32_t*>(row);
      p.norm = s.norms[at];
    }
    return p;
  };
  uint32_t w = blockIdx.x * (kReadThreads / 32) + (threadIdx.x >> 5);
  Piece next = fetch(w);
#pragma unroll 1
  for (; w < a.tasks; w += step) {
    const Piece p = next;
    next = fetch(w + step);
    if (p.left <= 0) continue;
    constexpr int E = 16 / sizeof(T);
    uint4 y[16 / E];
    if (p.there) {
      float f[16];
#pragma unroll
      for (int i = 0; i < (BITS == 8 ? 16 : 8); ++i) {
        if constexpr (BITS == 8) {
          asm("ld.shared.f32 %0, [%1];"
              : "=f"(f[i])
              : "r"(__dp4a(p.x[i >> 2], 128u << (8 * (i & 3)), base)));
        } else {
          uint32_t at;
          if constexpr (BITS == 4) {
            at = __dp4a(p.x[i >> 2], 128u << (8 * (i & 3)), base);
          } else {
            // nibble i, the high one of a byte first
            const int low = (i >> 1) * 8 + (i & 1 ? 0 : 4);
            at = base + ((p.x[0] >> low) & 15u) * 128u;
          }
          asm("ld.shared.v2.f32 {%0,%1}, [%2];" : "=f"(f[2 * i]), "=f"(f[2 * i + 1]) : "r"(at));
        }
      }
      uint32_t* o = reinterpret_cast<uint32_t*>(y);
#pragma unroll
      for (int i = 0; i < 16; i += 2) {
        const float v0 = __fmul_rn(p.norm, f[i]), v1 = __fmul_rn(p.norm, f[i + 1]);
        if constexpr (sizeof(T) == 4) {
          o[i] = __float_as_uint(v0);
          o[i + 1] = __float_as_uint(v1);
        } else if constexpr (std::is_same<T, __half>::value) {
          const __half2 v = __floats2half2_rn(v0, v1);
          o[i >> 1] = *reinterpret_cast<const uint32_t*>(&v);
        } else {
          const __nv_bfloat162 v = __floats2bfloat162_rn(v0, v1);
          o[i >> 1] = *reinterpret_cast<const uint32_t*>(&v);
        }
      }
    } else {
#pragma unroll
      for (int i = 0; i < 16 / E; ++i) y[i] = make_uint4(0u, 0u, 0u, 0u);
    }
    T* to = out + p.to;
    if (a.vec) {
#pragma unroll
      for (int i = 0; i < 16 / E; ++i)
        if (i * E < p.left) *reinterpret_cast<uint4*>(to + i * E) = y[i];
    } else {
      const T* e = reinterpret_cast<const T*>(y);
#pragma unroll
      for (int i = 0; i < 16; ++i)
        if (i < p.left) to[i] = e[i];
    }
  }
}

template <class T>
__global__ void __launch_bounds__(kReadThreads) kv_read_kernel(ReadArgs a) {
  __shared__ uint32_t table[256 * 32];
  const int bits = blockIdx.y ? a.sv.bits : a.sk.bits;
  if (bits == 2)
    read_rows<T, 2>(a, table);
  else if (bits == 4)
    read_rows<T, 4>(a, table);
  else
    read_rows<T, 8>(a, table);
}

}  // namespace kv
}  // namespace pqb

using namespace pqb;

extern "C" {

size_t pq_kv_codec_bytes(int d, int bits) {
  if (d < 1 || d > PQ_KV_MAX_D || !kv::bits_ok(bits)) return 0;
  return kv::codec_bytes(d, bits);
}

int pq_kv_prepare_codec(const float* R, const float* boundaries, const float* centroids, int d,
                        int bits, void* codec, size_t codec_bytes, void* stream) {
  PQ_CHECK_ARG(d >= 1 && d <= PQ_KV_MAX_D, "d must be in [1, %d] (got %d)", PQ_KV_MAX_D, d);
  PQ_CHECK_ARG(kv::bits_ok(bits), "bits must be 2, 4 or 8 (got %d)", bits);
  PQ_CHECK_ARG(R && boundaries && centroids && codec, "null pointer argument");
  if (codec_bytes < kv::codec_bytes(d, bits))
    return fail(PQ_ERR_WORKSPACE, "pq_kv_prepare_codec needs %zu bytes, got %zu",
                kv::codec_bytes(d, bits), codec_bytes);
  kv::prepare_codec_kernel<<<64, 256, 0, (cudaStream_t)stream>>>(
      R, boundaries, centroids, d, bits, kv::padded_d(d), kv::codec_of(codec, d));
  PQ_LAUNCH_CHECK("prepare_codec_kernel");
  return PQ_OK;
}

int pq_kv_append(const pq_kv_cache* cache, const void* k, const void* v, int dtype, int64_t n,
                 int64_t k_stride_n, int64_t k_stride_h, int64_t v_stride_n, int64_t v_stride_h,
                 const int64_t* slots, const int32_t* positions, const float* weights,
                 void* stream) {
  int rc = kv::check_cache(cache);
  if (rc) return rc;
  rc = kv::check_dtype(dtype);
  if (rc) return rc;
  PQ_CHECK_ARG(n >= 0 && n * cache->heads < (1ll << 31), "a call takes fewer than 2^31 rows");
  if (n == 0) return PQ_OK;
  PQ_CHECK_ARG(k && v && slots && positions, "null pointer argument");
  kv::AppendArgs a;
  a.k = k;
  a.v = v;
  a.k_sn = k_stride_n;
  a.k_sh = k_stride_h;
  a.v_sn = v_stride_n;
  a.v_sh = v_stride_h;
  a.rows = (uint32_t)(n * cache->heads);
  a.first_tile = 0;
  a.slots_end = (int64_t)cache->pages * cache->page_size;
  a.heads = cache->heads;
  a.d = cache->d;
  a.page_shift = kv::page_shift_of(*cache);
  const int size = dtype == PQ_KV_F32 ? 4 : 2;
  auto vec = [&](const void* p, int64_t sn, int64_t sh) {
    return (uintptr_t)p % 16 == 0 && sn * size % 16 == 0 && sh * size % 16 == 0 &&
           cache->d * size % 16 == 0;
  };
  a.k_vec = vec(k, k_stride_n, k_stride_h);
  a.v_vec = vec(v, v_stride_n, v_stride_h);
  a.sk = kv::side_k(*cache);
  a.sv = kv::side_v(*cache);
  a.slots = slots;
  a.positions = positions;
  a.weights = weights;
  a.out_pos = cache->positions;
  a.out_w = cache->weights;
  const int D = kv::padded_d(cache->d);
  const cudaStream_t st = (cudaStream_t)stream;
  PQ_KV_DISPATCH_T(dtype, {
    rc = D == 64 ? kv::launch_append<T_, 64>(a, st)
                 : D == 128 ? kv::launch_append<T_, 128>(a, st)
                            : kv::launch_append<T_, 256>(a, st);
  });
  return rc;
}

int pq_kv_read(const pq_kv_cache* cache, const int64_t* slots, int64_t n, void* k, void* v,
               int dtype, void* stream) {
  int rc = kv::check_cache(cache);
  if (rc) return rc;
  rc = kv::check_dtype(dtype);
  if (rc) return rc;
  PQ_CHECK_ARG(n >= 0 && n * cache->heads < (1ll << 31), "a call takes fewer than 2^31 rows");
  if (n == 0) return PQ_OK;
  PQ_CHECK_ARG(slots && k && v, "null pointer argument");
  kv::ReadArgs a;
  a.sk = kv::side_k(*cache);
  a.sv = kv::side_v(*cache);
  a.slots = slots;
  a.slots_end = (int64_t)cache->pages * cache->page_size;
  a.heads = cache->heads;
  a.d = cache->d;
  a.page_shift = kv::page_shift_of(*cache);
  a.pieces = (cache->d + 15) / 16;
  a.per_token = (int)(((int64_t)cache->heads * a.pieces + 31) / 32);
  a.tasks = (uint32_t)(n * a.per_token);
  a.k = k;
  a.v = v;
  a.vec = cache->d * (dtype == PQ_KV_F32 ? 4 : 2) % 16 == 0 && (uintptr_t)k % 16 == 0 &&
          (uintptr_t)v % 16 == 0;
  const int64_t blocks = ((int64_t)a.tasks + kv::kReadThreads / 32 - 1) / (kv::kReadThreads / 32);
  // Three blocks an SM, those that fit, over both sides.
  const dim3 grid((unsigned)min(blocks, (int64_t)3 * num_sms() / 2), 2);
  PQ_KV_DISPATCH_T(dtype, {
    kv::kv_read_kernel<T_><<<grid, kv::kReadThreads, 0, (cudaStream_t)stream>>>(a);
  });
  PQ_LAUNCH_CHECK("kv_read_kernel");
  return PQ_OK;
}

}  // extern "C"
