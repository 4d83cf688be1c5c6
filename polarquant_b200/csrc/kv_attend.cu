// Attention of one token over the compressed key-value cache.
//
// With q' = Rk q and the packed rows' centroids c, the score of token j is
//   s_j = scale * kn_j * sum_i q'_i c[kcode_ji]
// and the output Rv^T (sum_j p_j vn_j c[vcode_j]), p = softmax(s): neither side
// of the cache is turned back, only the query and the output.
//
// rotate_kernel turns the queries; attend_kernel takes kSplit tokens of one
// key-value head and up to eight of its query heads and leaves their maximum,
// sum and unnormalised output; join_kernel puts a row's splits together and
// turns the output back; weights_kernel adds the softmax weights.
#include "kv.cuh"

namespace pqb {
namespace kv {

constexpr int kSplit = 512;   // tokens of one block
constexpr int kTile = 32;     // tokens dequantised at a time
constexpr int kHeadsPer = 8;  // query heads of one block
constexpr float kLog2e = 1.4426950408889634f;

// Queries in rotated coordinates, times scale * log2(e) (scores are powers of 2).
template <class T>
__global__ void __launch_bounds__(PQ_KV_MAX_D)
rotate_kernel(const T* __restrict__ q, int64_t sb, int64_t sh, int hq, int d,
              const float* __restrict__ RT, float scale, float* __restrict__ out) {
  __shared__ float sq[PQ_KV_MAX_D];
  const int b = blockIdx.x / hq, h = blockIdx.x % hq, j = threadIdx.x;
  if (j < d) sq[j] = to_f32<T>(q[b * sb + h * sh + j]);
  __syncthreads();
  if (j >= d) return;
  float y = 0.f;
  for (int i = 0; i < d; ++i) y = fmaf(sq[i], RT[i * d + j], y);
  out[(int64_t)blockIdx.x * d + j] = y * (scale * kLog2e);
}

__global__ void __launch_bounds__(128)
attend_kernel(Side sk, Side sv, int heads, int group, int d, int pages, int page_size,
              const float* __restrict__ qrot, const int32_t* __restrict__ table,
              int64_t table_stride, int table_width, const int32_t* __restrict__ lengths,
              int splits, float* __restrict__ part_o, float2* __restrict__ part_ml,
              float* __restrict__ scores, int64_t score_width) {
  extern __shared__ float sm[];
  float* sq = sm;                            // kHeadsPer x d
  float* tile = sq + kHeadsPer * d;          // kTile x (d + 1)
  float* sp = tile + kTile * (d + 1);        // kHeadsPer x kTile
  float* cent_k = sp + kHeadsPer * kTile;    // 256
  float* cent_v = cent_k + 256;              // 256
  __shared__ float s_m[kHeadsPer], s_l[kHeadsPer], s_c[kHeadsPer];
  const int split = blockIdx.x, b = blockIdx.y / heads, h = blockIdx.y % heads;
  const int hq = heads * group, g0 = blockIdx.z * kHeadsPer, ng = min(kHeadsPer, group - g0);
  const int len = clamp_length(lengths[b], table_width, page_size);
  const int t0 = split * kSplit, t1 = min(len, t0 + kSplit);
  const int64_t row0 = (int64_t)b * hq + (int64_t)h * group + g0;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  if (t0 >= t1) {
    if (tid < ng) part_ml[(row0 + tid) * splits + split] = make_float2(-INFINITY, 0.f);
    return;
  }
  for (int i = tid; i < ng * d; i += blockDim.x) sq[i] = qrot[row0 * d + i];
  for (int i = tid; i < 256; i += blockDim.x) {
    cent_k[i] = sk.c.cent[i];
    cent_v[i] = sv.c.cent[i];
  }
  if (tid < kHeadsPer) {
    s_m[tid] = -INFINITY;
    s_l[tid] = 0.f;
  }
  float acc[2][kHeadsPer];
#pragma unroll
  for (int g = 0; g < kHeadsPer; ++g) acc[0][g] = acc[1][g] = 0.f;
  for (int base = t0; base < t1; base += kTile) {
    // Each thread's token of the tile, for norms and rows.
    auto place = [&](int i, bool& in) -> int64_t {
      const int t = base + i;
      in = t < t1;
      const int pg = in ? table[b * table_stride + t / page_size] : -1;
      in = pg >= 0 && pg < pages;
      return in ? ((int64_t)pg * heads + h) * page_size + t % page_size : 0;
    };
    for (int side = 0; side < 2; ++side) {
      const Side& s = side ? sv : sk;
      const float* cent = side ? cent_v : cent_k;
      __syncthreads();
      for (int i = warp; i < kTile; i += 4) {
        bool in;
        const int64_t at = place(i, in);
        const float nrm = in ? s.norms[at] : 0.f;
        for (int j = lane; j < d; j += 32)
          tile[i * (d + 1) + j] = in ? nrm * cent[code_at(s.rows + at * s.ldb, j, s.bits)] : 0.f;
      }
      __syncthreads();
      if (side == 0) {
        bool in;
        place(lane, in);
        for (int g = warp; g < ng; g += 4) {
          float y = 0.f;
          for (int j = 0; j < d; ++j) y = fmaf(sq[g * d + j], tile[lane * (d + 1) + j], y);
          if (!in) y = -INFINITY;
          if (scores && base + lane < t1)
            scores[(row0 + g) * score_width + base + lane] = y;
          float mx = y;
#pragma unroll
          for (int o = 16; o > 0; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
          const float m = fmaxf(s_m[g], mx);
          const float mm = m == -INFINITY ? 0.f : m;
          const float p = exp2f(y - mm);
          float l = p;
#pragma unroll
          for (int o = 16; o > 0; o >>= 1) l += __shfl_xor_sync(0xffffffffu, l, o);
          sp[g * kTile + lane] = p;
          __syncwarp();
          if (lane == 0) {
            s_c[g] = exp2f(s_m[g] - mm);
            s_l[g] = s_l[g] * s_c[g] + l;
            s_m[g] = m;
          }
        }
      } else {
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          const int j = tid + 128 * u;
          if (j >= d) continue;
#pragma unroll
          for (int g = 0; g < kHeadsPer; ++g) {
            if (g >= ng) break;
            float a = acc[u][g] * s_c[g];
            for (int i = 0; i < kTile; ++i) a = fmaf(sp[g * kTile + i], tile[i * (d + 1) + j], a);
            acc[u][g] = a;
          }
        }
      }
    }
  }
  __syncthreads();
#pragma unroll
  for (int u = 0; u < 2; ++u)
#pragma unroll
    for (int g = 0; g < kHeadsPer; ++g)
      if (g < ng && tid + 128 * u < d)
        part_o[((row0 + g) * splits + split) * d + tid + 128 * u] = acc[u][g];
  if (tid < ng) part_ml[(row0 + tid) * splits + split] = make_float2(s_m[tid], s_l[tid]);
}

template <class T>
__global__ void __launch_bounds__(PQ_KV_MAX_D)
join_kernel(const float* __restrict__ part_o, const float2* __restrict__ part_ml, int splits, int d,
            const float* __restrict__ R, T* __restrict__ out, float* __restrict__ lse,
            float* __restrict__ lse2) {
  __shared__ float so[PQ_KV_MAX_D];
  const int64_t row = blockIdx.x;
  const int j = threadIdx.x;
  float m = -INFINITY;
  for (int s = 0; s < splits; ++s) m = fmaxf(m, part_ml[row * splits + s].x);
  const float mm = m == -INFINITY ? 0.f : m;
  float l = 0.f, o = 0.f;
  for (int s = 0; s < splits; ++s) {
    const float2 ml = part_ml[row * splits + s];
    if (ml.y == 0.f) continue;
    const float c = exp2f(ml.x - mm);
    l = fmaf(ml.y, c, l);
    if (j < d) o = fmaf(part_o[(row * splits + s) * d + j], c, o);
  }
  if (j < d) so[j] = l > 0.f ? o / l : (l == 0.f ? 0.f : l);
  __syncthreads();
  if (j == 0) {
    const float l2 = l > 0.f ? mm + log2f(l) : (l == 0.f ? -INFINITY : l);
    if (lse) lse[row] = l2 / kLog2e;
    if (lse2) lse2[row] = l2;
  }
  if (j >= d) return;
  float y = 0.f;
  for (int i = 0; i < d; ++i) y = fmaf(so[i], R[i * d + j], y);
  out[row * d + j] = from_f32<T>(y);
}

__global__ void __launch_bounds__(256)
weights_kernel(const float* __restrict__ scores, const float* __restrict__ lse2, int heads,
               int group, int pages, int page_size, const int32_t* __restrict__ table,
               int64_t table_stride, int table_width, const int32_t* __restrict__ lengths,
               int64_t width, float* __restrict__ weights) {
  const int b = blockIdx.y / heads, h = blockIdx.y % heads;
  const int len = clamp_length(lengths[b], table_width, page_size);
  const int t = blockIdx.x * blockDim.x + threadIdx.x;
  if (t >= len) return;
  const int pg = table[b * table_stride + t / page_size];
  if (pg < 0 || pg >= pages) return;
  const int64_t row0 = ((int64_t)b * heads + h) * group;
  float w = 0.f;
  for (int g = 0; g < group; ++g) w += exp2f(scores[(row0 + g) * width + t] - lse2[row0 + g]);
  atomicAdd(weights + ((int64_t)pg * heads + h) * page_size + t % page_size, w);
}

struct AttendPlan {
  int splits;
  int64_t rows, width;
  size_t bytes;
  float *qrot, *part_o, *lse2, *scores;
  float2* part_ml;
};

inline AttendPlan attend_plan(const pq_kv_cache& c, int batch, int q_heads, int table_width,
                              int accumulate, void* ws, size_t ws_bytes) {
  AttendPlan p;
  p.rows = (int64_t)batch * q_heads;
  p.width = (int64_t)table_width * c.page_size;
  p.splits = (int)max((int64_t)1, (p.width + kSplit - 1) / kSplit);
  Carve cv(ws, ws_bytes);
  p.qrot = cv.take<float>(p.rows * c.d);
  p.part_o = cv.take<float>(p.rows * p.splits * c.d);
  p.part_ml = cv.take<float2>(p.rows * p.splits);
  p.lse2 = cv.take<float>(p.rows);
  p.scores = accumulate ? cv.take<float>(p.rows * p.width) : nullptr;
  p.bytes = cv.off;
  return p;
}

}  // namespace kv
}  // namespace pqb

using namespace pqb;

extern "C" {

size_t pq_kv_attend_workspace_bytes(const pq_kv_cache* cache, int batch, int q_heads,
                                    int table_width, int accumulate) {
  if (!cache || batch <= 0 || q_heads <= 0 || table_width < 0) return 256;
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
  PQ_CHECK_ARG((int64_t)batch * q_heads < 65536, "batch * q_heads must be below 65536");
  const kv::AttendPlan p =
      kv::attend_plan(c, batch, q_heads, table_width, accumulate, ws, ws_bytes);
  if (!ws || ws_bytes < p.bytes)
    return fail(PQ_ERR_WORKSPACE, "pq_kv_attend needs %zu workspace bytes, got %zu", p.bytes,
                ws_bytes);
  const cudaStream_t st = (cudaStream_t)stream;
  const kv::Side sk = kv::side_k(c), sv = kv::side_v(c);
  const int group = q_heads / c.heads;
  PQ_KV_DISPATCH_T(dtype, {
    kv::rotate_kernel<T_><<<(unsigned)p.rows, PQ_KV_MAX_D, 0, st>>>(
        (const T_*)q, q_stride_b, q_stride_h, q_heads, c.d, sk.c.RT, scale, p.qrot);
  });
  PQ_LAUNCH_CHECK("kv::rotate_kernel");
  const size_t smem = sizeof(float) * ((size_t)kv::kHeadsPer * c.d + kv::kTile * (c.d + 1) +
                                       kv::kHeadsPer * kv::kTile + 512);
  const dim3 grid(p.splits, batch * c.heads, (group + kv::kHeadsPer - 1) / kv::kHeadsPer);
  kv::attend_kernel<<<grid, 128, smem, st>>>(sk, sv, c.heads, group, c.d, c.pages, c.page_size,
                                             p.qrot, table, table_stride, table_width, lengths,
                                             p.splits, p.part_o, p.part_ml, p.scores, p.width);
  PQ_LAUNCH_CHECK("kv::attend_kernel");
  PQ_KV_DISPATCH_T(dtype, {
    kv::join_kernel<T_><<<(unsigned)p.rows, PQ_KV_MAX_D, 0, st>>>(
        p.part_o, p.part_ml, p.splits, c.d, sv.c.R, (T_*)out, lse, p.lse2);
  });
  PQ_LAUNCH_CHECK("kv::join_kernel");
  if (accumulate && p.width) {
    const dim3 wg((unsigned)((p.width + 255) / 256), batch * c.heads);
    kv::weights_kernel<<<wg, 256, 0, st>>>(p.scores, p.lse2, c.heads, group, c.pages, c.page_size,
                                           table, table_stride, table_width, lengths, p.width,
                                           c.weights);
    PQ_LAUNCH_CHECK("kv::weights_kernel");
  }
  return PQ_OK;
}

}  // extern "C"
