// Rows of the compressed key-value cache: the codec's tables, writing tokens
// (norm, rotation, Lloyd-Max codes, packing, scatter into the pages) and
// reading slots back as vectors.
#include "kv.cuh"

namespace pqb {
namespace kv {

__global__ void prepare_codec_kernel(const float* __restrict__ R, const float* __restrict__ bounds,
                                     const float* __restrict__ cent, int d, int bits,
                                     float* __restrict__ oR, float* __restrict__ oRT,
                                     float* __restrict__ ob, float* __restrict__ oc,
                                     uint32_t* __restrict__ pairs, int* __restrict__ exponent) {
  const int t = blockIdx.x * blockDim.x + threadIdx.x;
  for (int i = t; i < d * d; i += gridDim.x * blockDim.x) {
    const float v = R[i];
    oR[i] = v;
    oRT[(i % d) * d + i / d] = v;
  }
  if (t < 256) {
    ob[t] = t < (1 << bits) - 1 ? bounds[t] : INFINITY;
    oc[t] = t < (1 << bits) ? cent[t] : 0.f;
  }
  if (blockIdx.x) return;
  __shared__ uint32_t s_half[256];  // hi | lo << 16
  __shared__ int s_mx;
  if (threadIdx.x == 0) s_mx = 0;
  __syncthreads();
  const float c = threadIdx.x < (1 << bits) ? cent[threadIdx.x] : 0.f;
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
  pairs[i] = p0;
  pairs[256 + i] = p1;
  if (i == 0) *exponent = e;
}

// Append.  x -> norm = f32(sqrt(sum_f64 x^2)), u = x / max(norm, 1e-8) in f32,
// code_j = #{boundaries < sum_i u_i R_ji}, the sum in f64.  One warp per row;
// lane l holds columns l, l + 32, ...
constexpr int kAppendWarps = 8;

template <class T>
__global__ void __launch_bounds__(32 * kAppendWarps)
append_kernel(const T* __restrict__ k, const T* __restrict__ v, int64_t k_sn, int64_t k_sh,
              int64_t v_sn, int64_t v_sh, int64_t n, int heads, int d, int64_t slots_end,
              int page_size, Side sk, Side sv, const int64_t* __restrict__ slots,
              const int32_t* __restrict__ positions, const float* __restrict__ weights,
              int32_t* __restrict__ out_pos, float* __restrict__ out_w) {
  __shared__ float su[kAppendWarps][PQ_KV_MAX_D];
  __shared__ uint8_t sc[kAppendWarps][PQ_KV_MAX_D];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const bool is_v = blockIdx.y != 0;
  const Side& s = is_v ? sv : sk;
  const int64_t r = (int64_t)blockIdx.x * kAppendWarps + warp;
  if (r >= n * heads) return;
  const int64_t tok = r / heads;
  const int h = (int)(r % heads);
  const int64_t slot = slots[tok];
  if (slot < 0 || slot >= slots_end) return;
  const T* x = is_v ? v + tok * v_sn + h * v_sh : k + tok * k_sn + h * k_sh;
  double ss = 0.0;
  for (int i = lane; i < d; i += 32) {
    const float f = to_f32<T>(x[i]);
    su[warp][i] = f;
    ss = fma((double)f, (double)f, ss);
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
  const float nrm = __double2float_rn(__dsqrt_rn(ss));
  const float den = fmaxf(nrm, 1e-8f);
  for (int i = lane; i < d; i += 32) su[warp][i] = __fdiv_rn(su[warp][i], den);
  __syncwarp();
  const int levels = 1 << s.bits;
  for (int j = lane; j < PQ_KV_MAX_D; j += 32) {
    uint32_t code = 0;
    if (j < d) {
      double y = 0.0;
      for (int i = 0; i < d; ++i) y = fma((double)su[warp][i], (double)s.c.RT[i * d + j], y);
      for (int step = levels >> 1; step > 0; step >>= 1)
        if (y > (double)s.c.bounds[code + step - 1]) code += step;
    }
    sc[warp][j] = (uint8_t)code;
  }
  __syncwarp();
  const int64_t at = ((slot / page_size) * heads + h) * page_size + slot % page_size;
  uint8_t* row = s.rows + at * s.ldb;
  const int per = 8 / s.bits;
  for (int b = lane; b < s.ldb; b += 32) {
    uint32_t w = 0;
    for (int t = 0; t < per; ++t) {
      const int j = b * per + t;
      w = (w << s.bits) | (j < PQ_KV_MAX_D ? sc[warp][j] : 0u);
    }
    row[b] = (uint8_t)w;
  }
  if (lane == 0) {
    s.norms[at] = nrm;
    if (!is_v) {
      out_pos[at] = positions[tok];
      out_w[at] = weights ? weights[r] : 0.f;
    }
  }
}

// Read: one warp per row, norm * centroid[code].
template <class T>
__global__ void __launch_bounds__(256)
read_kernel(Side sk, Side sv, const int64_t* __restrict__ slots, int64_t n, int heads, int d,
            int64_t slots_end, int page_size, T* __restrict__ ok, T* __restrict__ ov) {
  __shared__ float cent[256];
  const Side& s = blockIdx.y ? sv : sk;
  T* out = blockIdx.y ? ov : ok;
  if (threadIdx.x < 256) cent[threadIdx.x] = s.c.cent[threadIdx.x];
  __syncthreads();
  const int lane = threadIdx.x & 31;
  const int64_t r = (int64_t)blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5);
  if (r >= n * heads) return;
  const int64_t slot = slots[r / heads];
  const bool in = slot >= 0 && slot < slots_end;
  const int64_t at =
      in ? ((slot / page_size) * heads + r % heads) * page_size + slot % page_size : 0;
  const float nrm = in ? s.norms[at] : 0.f;
  for (int j = lane; j < d; j += 32)
    out[r * d + j] =
        from_f32<T>(in ? __fmul_rn(nrm, cent[code_at(s.rows + at * s.ldb, j, s.bits)]) : 0.f);
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
  const kv::Codec c = kv::codec_of(codec, d);
  kv::prepare_codec_kernel<<<64, 256, 0, (cudaStream_t)stream>>>(
      R, boundaries, centroids, d, bits, (float*)c.R, (float*)c.RT, (float*)c.bounds,
      (float*)c.cent, (uint32_t*)c.pairs, (int*)c.exponent);
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
  const int64_t rows = n * cache->heads;
  const dim3 grid((unsigned)((rows + kv::kAppendWarps - 1) / kv::kAppendWarps), 2);
  PQ_KV_DISPATCH_T(dtype, {
    kv::append_kernel<T_><<<grid, 32 * kv::kAppendWarps, 0, (cudaStream_t)stream>>>(
        (const T_*)k, (const T_*)v, k_stride_n, k_stride_h, v_stride_n, v_stride_h, n,
        cache->heads, cache->d, (int64_t)cache->pages * cache->page_size, cache->page_size,
        kv::side_k(*cache), kv::side_v(*cache), slots, positions, weights, cache->positions,
        cache->weights);
  });
  PQ_LAUNCH_CHECK("kv::append_kernel");
  return PQ_OK;
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
  const dim3 grid((unsigned)((n * cache->heads + 7) / 8), 2);
  PQ_KV_DISPATCH_T(dtype, {
    kv::read_kernel<T_><<<grid, 256, 0, (cudaStream_t)stream>>>(
        kv::side_k(*cache), kv::side_v(*cache), slots, n, cache->heads, cache->d,
        (int64_t)cache->pages * cache->page_size, cache->page_size, (T_*)k, (T_*)v);
  });
  PQ_LAUNCH_CHECK("kv::read_kernel");
  return PQ_OK;
}

}  // extern "C"
