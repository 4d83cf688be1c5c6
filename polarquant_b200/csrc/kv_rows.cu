// Rows of the compressed key-value cache: the codec's tables, writing tokens
// (norm, rotation, Lloyd-Max codes, packing, scatter into the pages) and
// reading slots back as vectors.
#include "kv.cuh"

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
  uint32_t p0, p1;
  if (bits == 4) {
    const uint32_t a = s_half[i >> 4], b = s_half[i & 15];
    p0 = __byte_perm(a, b, 0x5410);
    p1 = __byte_perm(a, b, 0x7632);
  } else if (bits == 8) {
    p0 = s_half[i];
    p1 = 0u;
  } else {
    p0 = p1 = 0u;
    if (i < 4)  // byte i of the four 32-bit hi | lo words
      for (int k = 0; k < 4; ++k) p0 |= ((s_half[k] >> (8 * i)) & 255u) << (8 * k);
  }
  const_cast<uint32_t*>(out.pairs)[i] = p0;
  const_cast<uint32_t*>(out.pairs)[256 + i] = p1;
  if (i == 0) *const_cast<int*>(out.exponent) = e;
}

// ---------------------------------------------------------------------------
// Append
//
// x -> norm = f32(sqrt(sum_f64 x^2)), u = x / max(norm, 1e-8) in f32, code_j =
// #{boundaries < sum_i u_i R_ji}, exactly.
//
// The rotation runs on mma.m16n8k16 (f16 operands, f32 sums): a row's x times a
// power of two is f16 hi (exact for 16-bit inputs but for elements below 2^-28
// of the largest) or hi + lo (f32), R * 2^14 is hi + lo, and hi*hi + hi*lo (+
// lo*hi) are summed; the scales and 1 / max(norm, 1e-8) come after.  That is
// within (steps + 8) * 2^-23 of the exact product (each of the sum's `steps`
// additions loses at most 2^-23 of a partial sum, which is at most |u||R_j| = 1;
// operands lose 2^-22): coordinates that near a boundary are recomputed by the
// warp in f64.  So codes do not depend on how the product was taken.
//
// Which column and which element stands where in the operands is free, so a
// lane (g, t) loads a quarter of row g from its t-th run of d / 4 elements, and
// gets the coordinates of the same run back: it packs whole words.  Counting
// boundaries takes one table lookup: cells narrower than the gaps between
// boundaries hold at most one (from a copy for each lane at 2 and 4 bits, with
// the code in the low four bits of the boundary).
//
// A warp takes `ROWS` rows (32: the planes' operands, read from shared memory,
// serve two of them) through all columns with the planes of a side resident in
// shared memory; a call of few rows instead spreads the columns over the warps
// and reads the planes from L2.
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
  uint32_t rows, heads;
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
};

constexpr int kCellWords = 2 * kCells > 32 * kFewCells ? 2 * kCells : 32 * kFewCells;

template <class T, int D, bool SMALL>
struct AppendShape {
  static constexpr bool wide = sizeof(T) == 4;  // x is hi + lo
  static constexpr int MT = SMALL || wide || D == 256 ? 1 : 2;
  static constexpr int rows = 16 * MT;
  static constexpr int steps = D / 16;
  static constexpr int chunks = D / 32;                      // of 8 columns a lane
  static constexpr int per = SMALL ? 1 : (D == 256 ? 4 : chunks);  // chunks of a warp
  static constexpr int parts = SMALL ? 1 : chunks / per;     // blocks that share a row's columns
  static constexpr int warps = SMALL ? chunks : (D == 64 ? 16 : 12);
  static constexpr int groups = SMALL ? 1 : warps;           // row groups of a block at a time
  static constexpr int run = per * 8;                        // columns of a lane in a row
  static constexpr int plane = D / 8 / parts * steps * 32;   // uint2 of a plane in the block
  static constexpr int plane_bytes = SMALL ? 0 : 2 * plane * 8;
  static constexpr int smem = plane_bytes + 4 * kCellWords + warps * 2 * MT * 8 * 128;
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

template <class T, int D, int BITS, bool SMALL>
__device__ __forceinline__ void append_rows(const AppendArgs& a, uint8_t* smem) {
  using S = AppendShape<T, D, SMALL>;
  constexpr int MT = S::MT;
  constexpr int run_bytes = S::run * BITS / 8, words = (run_bytes + 3) / 4;
  constexpr int cells = BITS == 8 ? kCells : kFewCells;
  uint2* s_plane = reinterpret_cast<uint2*>(smem);
  uint32_t* s_cell = reinterpret_cast<uint32_t*>(smem + S::plane_bytes);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  // The lane's packed runs, one of each of its rows: word w of row i.
  uint32_t* s_run = s_cell + kCellWords + warp * (2 * MT * 8 * 32) + lane;
  // blockIdx.y: the part of the columns and, lowest, the side.
  const bool is_v = blockIdx.y & 1;
  const int part = blockIdx.y >> 1;
  const Side& sd = is_v ? a.sv : a.sk;
  const Codec& cd = sd.c;
  const T* src = reinterpret_cast<const T*>(is_v ? a.v : a.k);
  const int64_t sn = is_v ? a.v_sn : a.k_sn, sh = is_v ? a.v_sh : a.k_sh;
  const bool vec = is_v ? a.v_vec : a.k_vec;
  const int d = a.d;
  const uint32_t rows = a.rows, heads = a.heads;

  if constexpr (!SMALL) {
    const uint2* p = cd.planes + part * S::plane;
    for (int i = threadIdx.x; i < S::plane; i += blockDim.x) {
      s_plane[i] = p[i];
      s_plane[S::plane + i] = p[D / 8 * S::steps * 32 + i];
    }
  }
  if constexpr (BITS == 8) {
    for (int i = threadIdx.x; i < cells; i += blockDim.x)
      reinterpret_cast<uint2*>(s_cell)[i] = cd.cells[i];
  } else {
    for (int i = threadIdx.x; i < cells * 32; i += blockDim.x) {
      const uint2 c = cd.cells[i >> 5];
      s_cell[i] = (c.x & ~15u) | c.y;
    }
  }
  __syncthreads();
  const float cs = cd.range[0], co = cd.range[1];
  // (a boundary below 1 with its low four bits taken loses 15 * 2^-24 < 1e-6)
  constexpr float band =
      (S::steps * (S::wide ? 3 : 2) + 8) * 1.1920929e-7f + (BITS == 8 ? 0.f : 1e-6f);

  const uint32_t groups = (rows + S::rows - 1) / S::rows;
#pragma unroll 1
  for (uint32_t gr = blockIdx.x * S::groups + (SMALL ? 0 : warp); gr < groups;
       gr += gridDim.x * S::groups) {
    // x of rows g, g + 8 (, g + 16, g + 24) in f32, a quarter of each a lane.
    const uint32_t row0 = gr * S::rows;
    uint32_t ah[MT][S::steps][4], al[S::wide ? MT : 1][S::wide ? S::steps : 1][4];
    float inv[2 * MT], den[2 * MT];
#pragma unroll
    for (int i = 0; i < 2 * MT; ++i) {
      const uint32_t r = min(row0 + g + 8 * i, rows - 1);
      const T* x = src + (int64_t)(r / heads) * sn + (r % heads) * sh + t * (D / 4);
      float f[D / 4];
      constexpr int E = 16 / sizeof(T);
      if (vec) {
        uint4 w[D / 4 / E];
#pragma unroll
        for (int j = 0; j < D / 4 / E; ++j)
          w[j] = t * (D / 4) + j * E < d ? *reinterpret_cast<const uint4*>(x + j * E)
                                         : make_uint4(0u, 0u, 0u, 0u);
#pragma unroll
        for (int j = 0; j < D / 4 / E; ++j) widen16<T>(w[j], f + j * E);
      } else {
#pragma unroll
        for (int j = 0; j < D / 4; ++j) f[j] = t * (D / 4) + j < d ? to_f32<T>(x[j]) : 0.f;
      }
      double ss = 0.0;
      float mx = 0.f;
#pragma unroll
      for (int j = 0; j < D / 4; ++j) {
        ss = fma((double)f[j], (double)f[j], ss);
        mx = fmaxf(mx, fabsf(f[j]));
      }
#pragma unroll
      for (int o = 1; o < 4; o <<= 1) {
        ss += __shfl_xor_sync(0xffffffffu, ss, o);
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
      }
      const float nrm = __double2float_rn(__dsqrt_rn(ss));
      den[i] = fmaxf(nrm, 1e-8f);
      if (t == 0 && part == 0 && (!SMALL || warp == 0) && row0 + g + 8 * i < rows) {
        const int64_t at = a.place(r);
        if (at >= 0) {
          sd.norms[at] = nrm;
          if (!is_v) {
            a.out_pos[at] = a.positions[r / heads];
            a.out_w[at] = a.weights ? a.weights[r] : 0.f;
          }
        }
      }
      // max |x| * 2^e in [2^14, 2^15): f16's range, and sums of at most 2^29 sqrt(d)
      const int e =
          mx > 0.f && mx < INFINITY ? max(-126, min(126, 14 - ilogbf(mx))) : 0;
      const float up = __int_as_float((127 + e) << 23);
      inv[i] = __int_as_float((127 - e) << 23) / 16384.f / den[i];
      // Registers 0 and 2 of the A operand hold row g, 1 and 3 row g + 8.
#pragma unroll
      for (int s = 0; s < S::steps; ++s)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const float x0 = f[4 * s + 2 * h] * up, x1 = f[4 * s + 2 * h + 1] * up;
          const __half2 hi = __floats2half2_rn(x0, x1);
          ah[i >> 1][s][2 * h + (i & 1)] = *reinterpret_cast<const uint32_t*>(&hi);
          if constexpr (S::wide) {
            const float2 b = __half22float2(hi);
            const __half2 lo = __floats2half2_rn(x0 - b.x, x1 - b.y);
            al[i >> 1][s][2 * h + (i & 1)] = *reinterpret_cast<const uint32_t*>(&lo);
          }
        }
    }

    // Eight columns a lane at a time.  (One body for all: unrolled over the
    // chunks the code does not fit the instruction cache.)
#pragma unroll 1
    for (int c = 0; c < S::per; ++c) {
      const int chunk = SMALL ? warp : part * S::per + c;
      float acc[MT][4][4];
#pragma unroll
      for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int q = 0; q < 4; ++q) acc[m][q][0] = acc[m][q][1] = acc[m][q][2] = acc[m][q][3] = 0.f;
      const uint2* bp = SMALL ? cd.planes + chunk * 4 * S::steps * 32 + lane
                              : s_plane + c * 4 * S::steps * 32 + lane;
      constexpr int lo_at = SMALL ? D / 8 * S::steps * 32 : S::plane;
#pragma unroll
      for (int s = 0; s < S::steps; ++s)
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const uint2 bh = bp[(q * S::steps + s) * 32], bl = bp[lo_at + (q * S::steps + s) * 32];
#pragma unroll
          for (int m = 0; m < MT; ++m) {
            mma_rows(acc[m][q], ah[m][s], bh);
            mma_rows(acc[m][q], ah[m][s], bl);
            if constexpr (S::wide) mma_rows(acc[m][q], al[m][s], bh);
          }
        }
      // Codes of rows g + 8i, columns t * D / 4 + chunk * 8 + k: packed, the first
      // code highest in its byte, and which of them are next to a boundary.
      constexpr int cw = BITS == 8 ? 2 : 1;
      uint32_t packed[2 * MT][cw], near = 0;
      const int left = min(8, d - (t * (D / 4) + chunk * 8));  // columns that there are
#pragma unroll
      for (int i = 0; i < 2 * MT; ++i) {
#pragma unroll
        for (int w = 0; w < cw; ++w) packed[i][w] = 0u;
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          const float y = acc[i >> 1][k >> 1][2 * (i & 1) + (k & 1)] * inv[i];
          const float cell = fmaf(__saturatef(fmaf(y, cs, co)), (float)(cells - 1), 8388608.f);
          float b;
          uint32_t code;
          if constexpr (BITS == 8) {
            const uint2 e =
                reinterpret_cast<const uint2*>(s_cell)[__float_as_uint(cell) & (cells - 1)];
            b = __uint_as_float(e.x);
            code = e.y;
          } else {
            const uint32_t e = s_cell[(__float_as_uint(cell) & (cells - 1)) * 32 + lane];
            b = __uint_as_float(e);
            code = e & 15u;
          }
          const float off = y - b;
          if (off > 0.f) ++code;
          if (!(fabsf(off) >= band)) near |= 1u << (8 * i + k);
          const int bit = k * BITS;
          packed[i][bit >> 5] |= code << ((bit & 24) + 8 - BITS - (bit & 7));
        }
      }
      if (left < 8) {
        // Bits of the columns behind the row's end are 0.
#pragma unroll
        for (int i = 0; i < 2 * MT; ++i)
#pragma unroll
          for (int k = 0; k < 8; ++k)
            if (k >= left) {
              const int bit = k * BITS;
              packed[i][bit >> 5] &=
                  ~(((1u << BITS) - 1u) << ((bit & 24) + 8 - BITS - (bit & 7)));
              near &= ~(1u << (8 * i + k));
            }
      }
#pragma unroll
      for (int i = 0; i < 2 * MT; ++i)
        if (row0 + g + 8 * i >= rows) near &= ~(255u << (8 * i));
      // Coordinates next to a boundary, by the whole warp.
      uint32_t pend = __ballot_sync(0xffffffffu, near != 0u);
#pragma unroll 1
      while (pend) {
        const int from = __ffs(pend) - 1;
        pend &= pend - 1;
        uint32_t mask = __shfl_sync(0xffffffffu, near, from);
#pragma unroll 1
        while (mask) {
          const int n = __ffs(mask) - 1, i = n >> 3, k = n & 7;
          mask &= mask - 1;
          float dn = den[0];
#pragma unroll
          for (int z = 1; z < 2 * MT; ++z)
            if (z == i) dn = den[z];
          dn = __shfl_sync(0xffffffffu, dn, from);
          const uint32_t r = row0 + (from >> 2) + 8 * i;
          const T* x = src + (int64_t)(r / heads) * sn + (r % heads) * sh;
          const float* rr = cd.R + ((from & 3) * (D / 4) + chunk * 8 + k) * d;
          double y = 0.0;
          for (int j = lane; j < d; j += 32)
            y = fma((double)__fdiv_rn(to_f32<T>(x[j]), dn), (double)__ldg(rr + j), y);
#pragma unroll
          for (int o = 16; o > 0; o >>= 1) y += __shfl_xor_sync(0xffffffffu, y, o);
          uint32_t code = 0;
#pragma unroll
          for (int step = 1 << (BITS - 1); step > 0; step >>= 1)
            if (y > (double)__ldg(cd.bounds + code + step - 1)) code += step;
          const int bit = k * BITS, shift = (bit & 24) + 8 - BITS - (bit & 7);
          if (lane == from) {
#pragma unroll
            for (int z = 0; z < 2 * MT; ++z)
#pragma unroll
              for (int w = 0; w < cw; ++w)
                if (z == i && w == bit >> 5)
                  packed[z][w] = (packed[z][w] & ~(((1u << BITS) - 1u) << shift)) | code << shift;
          }
        }
      }
#pragma unroll
      for (int i = 0; i < 2 * MT; ++i) {
        if constexpr (BITS == 2) {
          uint16_t* to = reinterpret_cast<uint16_t*>(s_run + (i * 8 + (c >> 1)) * 32) + (c & 1);
          *to = (uint16_t)packed[i][0];
        } else {
#pragma unroll
          for (int w = 0; w < cw; ++w) s_run[(i * 8 + c * cw + w) * 32] = packed[i][w];
        }
      }
    }

#pragma unroll 1
    for (int i = 0; i < 2 * MT; ++i) {
      const uint32_t r = row0 + g + 8 * i;
      if (r >= rows) break;
      const int64_t at = a.place(r);
      if (at < 0) continue;
      const int off = (t * (D / 4) + (SMALL ? warp : part * S::per) * 8) * BITS / 8;
      uint8_t* to = sd.rows + at * sd.ldb + off;
      const uint32_t* w = s_run + i * 8 * 32;
      if constexpr (run_bytes >= 16) {
#pragma unroll
        for (int j = 0; j < words; j += 4)
          if (off + 4 * j < sd.ldb)
            *reinterpret_cast<uint4*>(to + 4 * j) =
                make_uint4(w[j * 32], w[(j + 1) * 32], w[(j + 2) * 32], w[(j + 3) * 32]);
      } else if (off < sd.ldb) {
        if constexpr (run_bytes == 8)
          *reinterpret_cast<uint2*>(to) = make_uint2(w[0], w[32]);
        else if constexpr (run_bytes == 4)
          *reinterpret_cast<uint32_t*>(to) = w[0];
        else
          *reinterpret_cast<uint16_t*>(to) = (uint16_t)w[0];
      }
    }
  }
}

template <class T, int D, bool SMALL>
__global__ void __launch_bounds__(32 * AppendShape<T, D, SMALL>::warps, 1)
kv_append_kernel(AppendArgs a) {
  extern __shared__ __align__(16) uint8_t smem[];
  const int bits = blockIdx.y & 1 ? a.sv.bits : a.sk.bits;
  if (bits == 2)
    append_rows<T, D, 2, SMALL>(a, smem);
  else if (bits == 4)
    append_rows<T, D, 4, SMALL>(a, smem);
  else
    append_rows<T, D, 8, SMALL>(a, smem);
}

template <class T, int D, bool SMALL>
int launch_append(const AppendArgs& a, cudaStream_t st) {
  using S = AppendShape<T, D, SMALL>;
  constexpr int smem = S::smem;
  auto kern = kv_append_kernel<T, D, SMALL>;
  PQ_CUDA_TRY(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
  const int64_t groups = ((int64_t)a.rows + S::rows - 1) / S::rows;
  const int64_t blocks = (groups + S::groups - 1) / S::groups;
  const int64_t most = SMALL ? 1 << 20 : max(1, num_sms() / (2 * S::parts));
  kern<<<dim3((unsigned)min(blocks, most), 2 * S::parts), 32 * S::warps, smem, st>>>(a);
  PQ_LAUNCH_CHECK("kv_append_kernel");
  return PQ_OK;
}

template <class T, int D>
int launch_append_rows(const AppendArgs& a, cudaStream_t st) {
  // Few rows: as many blocks of 16 rows as there are, each reading the planes
  // from L2; more than two waves of them: resident planes.
  if (a.rows <= 16u * num_sms()) return launch_append<T, D, true>(a, st);
  return launch_append<T, D, false>(a, st);
}

// ---------------------------------------------------------------------------
// Read: norm * centroid[code], rounded once.
//
// A lane takes 16 codes of a row; a warp 32 such pieces of one token.  Bound by
// the bytes written; the lookups are from tables with a copy for each lane (or
// each pair of lanes half a warp apart, for 64-bit entries): an f32 centroid at
// 8 bits, both of a byte's at 4, both of a nibble's at 2.
// ---------------------------------------------------------------------------

struct ReadArgs {
  Side sk, sv;
  const int64_t* slots;
  int64_t n, slots_end;
  int heads, d, page_size, pieces, per_token;  // 16-code pieces of a row, warps of a token
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
  const int64_t tasks = a.n * a.per_token;
  const int64_t step = (int64_t)gridDim.x * (kReadThreads / 32);
  for (int64_t w = (int64_t)blockIdx.x * (kReadThreads / 32) + (threadIdx.x >> 5); w < tasks;
       w += step) {
    const int64_t tok = a.per_token == 1 ? w : w / a.per_token;
    const int unit = (int)(w - tok * a.per_token) * 32 + lane;
    const int h = unit / a.pieces, piece = unit - h * a.pieces;
    if (h >= a.heads) continue;
    const int64_t slot = a.slots[tok];
    const bool in = slot >= 0 && slot < a.slots_end;
    uint32_t x[4] = {0u, 0u, 0u, 0u};
    float nrm = 0.f;
    if (in) {
      const int64_t at =
          (((int64_t)((uint32_t)slot / (uint32_t)a.page_size)) * a.heads + h) * a.page_size +
          (uint32_t)slot % (uint32_t)a.page_size;
      const uint8_t* row = s.rows + at * s.ldb + piece * (2 * BITS);
      if (BITS == 8)
        *reinterpret_cast<uint4*>(x) = *reinterpret_cast<const uint4*>(row);
      else if (BITS == 4)
        *reinterpret_cast<uint2*>(x) = *reinterpret_cast<const uint2*>(row);
      else
        x[0] = *reinterpret_cast<const uint32_t*>(row);
      nrm = s.norms[at];
    }
    float f[16];
#pragma unroll
    for (int i = 0; i < (BITS == 8 ? 16 : 8); ++i) {
      if constexpr (BITS == 8) {
        asm("ld.shared.f32 %0, [%1];"
            : "=f"(f[i])
            : "r"(__dp4a(x[i >> 2], 128u << (8 * (i & 3)), base)));
      } else {
        uint32_t at;
        if constexpr (BITS == 4) {
          at = __dp4a(x[i >> 2], 128u << (8 * (i & 3)), base);
        } else {
          // nibble i, the high one of a byte first
          const int low = (i >> 1) * 8 + (i & 1 ? 0 : 4);
          at = base + ((x[0] >> low) & 15u) * 128u;
        }
        asm("ld.shared.v2.f32 {%0,%1}, [%2];" : "=f"(f[2 * i]), "=f"(f[2 * i + 1]) : "r"(at));
      }
    }
    __align__(16) T y[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) y[i] = from_f32<T>(in ? __fmul_rn(nrm, f[i]) : 0.f);
    T* to = out + ((tok * a.heads + h) * a.d + piece * 16);
    const int left = a.d - piece * 16;
    if (a.vec) {
      constexpr int E = 16 / sizeof(T);
#pragma unroll
      for (int i = 0; i < 16; i += E)
        if (i < left) *reinterpret_cast<uint4*>(to + i) = *reinterpret_cast<const uint4*>(y + i);
    } else {
#pragma unroll
      for (int i = 0; i < 16; ++i)
        if (i < left) to[i] = y[i];
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
    rc = D == 64 ? kv::launch_append_rows<T_, 64>(a, st)
                 : D == 128 ? kv::launch_append_rows<T_, 128>(a, st)
                            : kv::launch_append_rows<T_, 256>(a, st);
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
  a.n = n;
  a.slots_end = (int64_t)cache->pages * cache->page_size;
  a.heads = cache->heads;
  a.d = cache->d;
  a.page_size = cache->page_size;
  a.pieces = (cache->d + 15) / 16;
  a.per_token = (int)(((int64_t)cache->heads * a.pieces + 31) / 32);
  a.k = k;
  a.v = v;
  a.vec = cache->d * (dtype == PQ_KV_F32 ? 4 : 2) % 16 == 0 && (uintptr_t)k % 16 == 0 &&
          (uintptr_t)v % 16 == 0;
  const int64_t blocks = (n * a.per_token + kv::kReadThreads / 32 - 1) / (kv::kReadThreads / 32);
  const dim3 grid((unsigned)min(blocks, (int64_t)2 * num_sms()), 2);
  PQ_KV_DISPATCH_T(dtype, {
    kv::kv_read_kernel<T_><<<grid, kv::kReadThreads, 0, (cudaStream_t)stream>>>(a);
  });
  PQ_LAUNCH_CHECK("kv_read_kernel");
  return PQ_OK;
}

}  // extern "C"
