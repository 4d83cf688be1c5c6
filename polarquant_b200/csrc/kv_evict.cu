// Eviction from the compressed key-value cache.
//
// For every sequence and head: the `budget` first tokens by (protected, weight
// descending, slot ascending) stay.  A radix selection on a monotone 32-bit key
// of the weight finds the key of the last one that stays and how many of its
// equals do; then the evicted tokens before the budget (holes) and the kept
// ones behind it (movers), equally many, are listed in slot order and
// move_kernel copies the j-th mover to the j-th hole.  Sources lie behind the
// budget and destinations before it, so the copies do not depend on each other.
#include "kv.cuh"

namespace pqb {
namespace kv {

constexpr int kEvictThreads = 1024;

struct EvictArgs {
  Side sk, sv;
  int heads, pages, page_size, table_width, budget, recent, sinks;
  const int32_t* table;
  int64_t table_stride;
  const int32_t* lengths;
  const float* prompt;  // or null
  int64_t prompt_sb, prompt_sh;
  int prompt_width;
  int32_t* positions;
  float* weights;
  int32_t* new_lengths;
  int32_t* lists;  // [batch * heads][2][width of lists]: holes, movers
  int32_t* counts;
  int64_t list_width;

  __device__ int length(int b) const {
    const int len = clamp_length(lengths[b], table_width, page_size);
    return prompt ? min(len, prompt_width) : len;
  }
  // Index of token t in the pools of one value a token; -1 without a page.
  __device__ int64_t at(int b, int h, int t) const {
    const int pg = table[b * table_stride + t / page_size];
    return pg >= 0 && pg < pages ? ((int64_t)pg * heads + h) * page_size + t % page_size : -1;
  }
  __device__ int position(int64_t at, int t) const {
    return prompt ? t : (at < 0 ? INT32_MIN : positions[at]);
  }
  __device__ float weight(int b, int h, int64_t at, int t) const {
    return prompt ? prompt[b * prompt_sb + h * prompt_sh + t] : (at < 0 ? -INFINITY : weights[at]);
  }
};

// Monotone in the weight; -0 as 0, NaN below everything; protected as +inf.
__device__ __forceinline__ uint32_t weight_key(float w, bool safe) {
  if (safe) return 0xff800000u;
  if (isnan(w)) return 0u;
  const uint32_t u = __float_as_uint(w == 0.f ? 0.f : w);
  return (u >> 31) ? ~u : (u | 0x80000000u);
}

// Exclusive prefix sum over the block; `total` gets the sum.
__device__ __forceinline__ int block_scan(int x, int* s_warp, int& total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int v = x;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int y = __shfl_up_sync(0xffffffffu, v, o);
    if (lane >= o) v += y;
  }
  __syncthreads();
  if (lane == 31) s_warp[warp] = v;
  __syncthreads();
  if (warp == 0) {
    int w = s_warp[lane];
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int y = __shfl_up_sync(0xffffffffu, w, o);
      if (lane >= o) w += y;
    }
    s_warp[lane] = w;
  }
  __syncthreads();
  total = s_warp[31];
  return v - x + (warp ? s_warp[warp - 1] : 0);
}

__global__ void __launch_bounds__(kEvictThreads) select_kernel(EvictArgs a) {
  __shared__ int s_hist[256], s_warp[32], s_max, s_digit, s_need;
  const int b = blockIdx.x / a.heads, h = blockIdx.x % a.heads, tid = threadIdx.x;
  const int len = a.length(b);
  if (h == 0 && tid == 0) a.new_lengths[b] = min(len, a.budget);
  int32_t* holes = a.lists + (int64_t)blockIdx.x * 2 * a.list_width;
  int32_t* movers = holes + a.list_width;
  if (len <= a.budget) {
    if (tid == 0) a.counts[blockIdx.x] = 0;
    if (a.prompt)
      for (int t = tid; t < len; t += kEvictThreads) {
        const int64_t at = a.at(b, h, t);
        if (at >= 0) {
          a.weights[at] = a.weight(b, h, at, t);
          a.positions[at] = t;
        }
      }
    return;
  }
  // The largest position.
  if (tid == 0) s_max = INT32_MIN;
  __syncthreads();
  int mx = INT32_MIN;
  if (a.prompt)
    mx = len - 1;
  else
    for (int t = tid; t < len; t += kEvictThreads) mx = max(mx, a.position(a.at(b, h, t), t));
  atomicMax(&s_max, mx);
  __syncthreads();
  const int64_t recent_from = (int64_t)s_max - a.recent;
  auto key = [&](int t) {
    const int64_t at = a.at(b, h, t);
    if (at < 0) return 0u;
    const int pos = a.position(at, t);
    return weight_key(a.weight(b, h, at, t),
                      pos < a.sinks || (int64_t)pos > recent_from);
  };
  // The key of the last token that stays, eight bits at a time.
  uint32_t prefix = 0, mask = 0;
  int need = a.budget;
  for (int shift = 24; shift >= 0 && need > 0; shift -= 8) {
    if (tid < 256) s_hist[tid] = 0;
    __syncthreads();
    for (int t = tid; t < len; t += kEvictThreads) {
      const uint32_t k = key(t);
      if ((k & mask) == prefix) atomicAdd(&s_hist[(k >> shift) & 255u], 1);
    }
    __syncthreads();
    if (tid == 0) {
      int dgt = 255, left = need;
      while (dgt > 0 && s_hist[dgt] < left) left -= s_hist[dgt--];
      s_digit = dgt;
      s_need = left;
    }
    __syncthreads();
    prefix |= (uint32_t)s_digit << shift;
    mask |= 255u << shift;
    need = s_need;
    __syncthreads();
  }
  // Tokens above `prefix` and the first `need` of its equals stay.  In slot
  // order: ties taken, holes and movers so far.
  int ties = 0, nh = 0, nm = 0;
  for (int t0 = 0; t0 < len; t0 += kEvictThreads) {
    const int t = t0 + tid;
    const uint32_t k = t < len ? key(t) : 0u;
    const bool tie = t < len && k == prefix;
    int total;
    const int rank = block_scan(tie, s_warp, total) + ties;
    ties += total;
    const bool kept = t < len && a.budget > 0 && (k > prefix || (tie && rank < need));
    const bool hole = t < min(len, a.budget) && !kept, mover = kept && t >= a.budget;
    const int both = block_scan((hole ? 1 : 0) | (mover ? 1 << 16 : 0), s_warp, total);
    if (hole) holes[nh + (both & 0xffff)] = t;
    if (mover) movers[nm + (both >> 16)] = t;
    nh += total & 0xffff;
    nm += total >> 16;
    if (a.prompt && kept && !mover) {
      const int64_t at = a.at(b, h, t);
      if (at >= 0) {
        a.weights[at] = a.weight(b, h, at, t);
        a.positions[at] = t;
      }
    }
  }
  if (tid == 0) a.counts[blockIdx.x] = min(nh, nm);
}

// One warp per moved token.
__global__ void __launch_bounds__(256) move_kernel(EvictArgs a) {
  const int b = blockIdx.y / a.heads, h = blockIdx.y % a.heads, lane = threadIdx.x & 31;
  const int n = a.counts[blockIdx.y];
  const int32_t* holes = a.lists + (int64_t)blockIdx.y * 2 * a.list_width;
  const int32_t* movers = holes + a.list_width;
  const int warps = gridDim.x * (blockDim.x >> 5);
  for (int i = blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5); i < n; i += warps) {
    const int ts = movers[i];
    const int64_t to = a.at(b, h, holes[i]), from = a.at(b, h, ts);
    if (to < 0 || from < 0) continue;
    const int nk = (int)(a.sk.ldb / 16), nv = (int)(a.sv.ldb / 16);
    const uint4* ks = reinterpret_cast<const uint4*>(a.sk.rows + from * a.sk.ldb);
    const uint4* vs = reinterpret_cast<const uint4*>(a.sv.rows + from * a.sv.ldb);
    uint4* kd = reinterpret_cast<uint4*>(a.sk.rows + to * a.sk.ldb);
    uint4* vd = reinterpret_cast<uint4*>(a.sv.rows + to * a.sv.ldb);
    for (int j = lane; j < nk + nv; j += 32) {
      if (j < nk)
        kd[j] = ks[j];
      else
        vd[j - nk] = vs[j - nk];
    }
    if (lane == 0) {
      a.sk.norms[to] = a.sk.norms[from];
      a.sv.norms[to] = a.sv.norms[from];
      a.positions[to] = a.position(from, ts);
      a.weights[to] = a.weight(b, h, from, ts);
    }
  }
}

inline int64_t evict_list_width(const pq_kv_cache& c, int table_width, int budget) {
  const int64_t width = (int64_t)table_width * c.page_size;
  return max((int64_t)0, min((int64_t)budget, width - budget));
}

inline size_t evict_bytes(const pq_kv_cache& c, int batch, int table_width, int budget,
                          EvictArgs* a, void* ws, size_t ws_bytes) {
  const int64_t rows = (int64_t)batch * c.heads, w = evict_list_width(c, table_width, budget);
  Carve cv(ws, ws_bytes);
  int32_t* counts = cv.take<int32_t>(rows);
  int32_t* lists = cv.take<int32_t>(rows * 2 * w);
  if (a) {
    a->counts = counts;
    a->lists = lists;
    a->list_width = w;
  }
  return cv.off;
}

}  // namespace kv
}  // namespace pqb

using namespace pqb;

extern "C" {

size_t pq_kv_evict_workspace_bytes(const pq_kv_cache* cache, int batch, int table_width,
                                   int budget) {
  if (!cache || batch <= 0 || table_width < 0 || budget < 0) return 256;
  return kv::evict_bytes(*cache, batch, table_width, budget, nullptr, nullptr, 0);
}

int pq_kv_evict(const pq_kv_cache* cache, const int32_t* table, int64_t table_stride,
                int table_width, const int32_t* lengths, int batch, int budget, int recent,
                int sinks, const float* prompt_weights, int64_t prompt_stride_b,
                int64_t prompt_stride_h, int prompt_width, int32_t* new_lengths, void* ws,
                size_t ws_bytes, void* stream) {
  int rc = kv::check_cache(cache);
  if (rc) return rc;
  const pq_kv_cache& c = *cache;
  rc = kv::check_sequences(table, table_width, lengths, batch, c.page_size);
  if (rc) return rc;
  PQ_CHECK_ARG(budget >= 0 && recent >= 0 && sinks >= 0,
               "budget, recent and sinks must be at least 0");
  PQ_CHECK_ARG(prompt_width >= 0, "prompt_width must be at least 0");
  if (batch == 0) return PQ_OK;
  PQ_CHECK_ARG(new_lengths, "null pointer argument");
  PQ_CHECK_ARG((int64_t)batch * c.heads < 65536, "batch * heads must be below 65536");
  kv::EvictArgs a;
  const size_t need = kv::evict_bytes(c, batch, table_width, budget, &a, ws, ws_bytes);
  if (!ws || ws_bytes < need)
    return fail(PQ_ERR_WORKSPACE, "pq_kv_evict needs %zu workspace bytes, got %zu", need,
                ws_bytes);
  a.sk = kv::side_k(c);
  a.sv = kv::side_v(c);
  a.heads = c.heads;
  a.pages = c.pages;
  a.page_size = c.page_size;
  a.table_width = table_width;
  a.budget = budget;
  a.recent = recent;
  a.sinks = sinks;
  a.table = table;
  a.table_stride = table_stride;
  a.lengths = lengths;
  a.prompt = prompt_weights;
  a.prompt_sb = prompt_stride_b;
  a.prompt_sh = prompt_stride_h;
  a.prompt_width = prompt_width;
  a.positions = c.positions;
  a.weights = c.weights;
  a.new_lengths = new_lengths;
  const cudaStream_t st = (cudaStream_t)stream;
  const int rows = batch * c.heads;
  kv::select_kernel<<<rows, kv::kEvictThreads, 0, st>>>(a);
  PQ_LAUNCH_CHECK("kv::select_kernel");
  if (a.list_width) {
    const int64_t per = (a.list_width + 7) / 8;
    const dim3 grid((unsigned)min(per, (int64_t)max(1, 8 * num_sms() / rows)), rows);
    kv::move_kernel<<<grid, 256, 0, st>>>(a);
    PQ_LAUNCH_CHECK("kv::move_kernel");
  }
  return PQ_OK;
}

}  // extern "C"
