// Eviction from the compressed key-value cache.
//
// For every sequence and head: the `budget` first tokens by (protected, weight
// descending, slot ascending) stay.  A radix selection on a monotone 32-bit key
// of the weight (11, 11 and 10 bits) finds the key of the last one that stays
// and how many of its equals do; then the evicted tokens before the budget
// (holes) and the kept ones behind it (movers), equally many (tokens on pages
// outside the pool are neither), are listed in slot order and kv_move_kernel
// copies the j-th mover to the j-th hole.  Sources lie behind the budget and
// destinations before it, so the copies do not depend on each other, and what
// does not have to move stays: at a constant budget a step moves as many rows as
// it evicts.
//
// A sequence and head is one block or a cluster of eight, whose blocks have an
// eighth of the tokens each and add their counts to the first one's histogram
// through distributed shared memory.  A block keeps its tokens' keys in shared
// memory (up to kKeep; beyond that weights and positions are read again).
//
// Bound by latency, of passes and barriers alike: 48 heads of 0 to 65536 tokens with
// a cluster each take 44 us, of which weights and the table are 2 us at DRAM's rate;
// 47 % of the issue slots are taken, and of the 13 cycles between a warp's
// instructions loads from memory take 2.7, barriers 2.5 and fixed latencies 2.3.
// Eight heads of 65536 tokens, moves included, take 34 us, of 131072 52; beyond that
// keys no longer fit the cluster's shared memory and are read again: 262144 188 us.
#include <cooperative_groups.h>

#include "kv.cuh"

namespace pqb {
namespace kv {

namespace cg = cooperative_groups;

constexpr int kEvictThreads = 512;
constexpr int kKeep = 16384;  // keys of a block in shared memory
constexpr int kBins = 2048;

struct EvictArgs {
  Side sk, sv;
  int heads, pages, page_shift, table_width, budget, recent, sinks;
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
    const int len = clamp_length(lengths[b], table_width, 1 << page_shift);
    return prompt ? min(len, prompt_width) : len;
  }
  // Index of token t in the pools of one value a token; -1 without a page.
  __device__ int64_t at(int b, int h, int t) const {
    const int pg = __ldg(table + b * table_stride + (t >> page_shift));
    return pg >= 0 && pg < pages
               ? (((int64_t)pg * heads + h) << page_shift) + (t & ((1 << page_shift) - 1))
               : -1;
  }
};

// Monotone in the weight; -0 as 0, NaN below everything, protected above +inf.
// (0 is the key of a token on a page outside the pool.)
__device__ __forceinline__ uint32_t weight_key(float w, bool safe) {
  if (safe) return 0xffffffffu;
  if (isnan(w)) return 1u;
  const uint32_t u = __float_as_uint(w == 0.f ? 0.f : w);
  return (u >> 31) ? ~u : (u | 0x80000000u);
}

// Exclusive prefix sum over the block's kEvictThreads; `total` gets the sum.
__device__ __forceinline__ int block_scan(int x, int* s_warp, int& total) {
  constexpr int warps = kEvictThreads / 32;
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
  int before = 0;
  total = 0;
#pragma unroll
  for (int i = 0; i < warps; ++i) {
    const int y = s_warp[i];
    if (i < warp) before += y;
    total += y;
  }
  return v - x + before;
}

// (Three blocks an SM: with registers for one, 48 clusters of eight took turns,
// 70 us instead of 44.)
template <int CL>
__global__ void __launch_bounds__(kEvictThreads, 3) kv_select_kernel(EvictArgs a) {
  extern __shared__ uint32_t s_key[];
  __shared__ int s_hist[kBins], s_warp[32], s_rank[3][CL], s_max, s_digit, s_left, s_missing;
  auto cluster = cg::this_cluster();
  const int rank = CL > 1 ? (int)cluster.block_rank() : 0;
  const int row = blockIdx.x / CL, b = row / a.heads, h = row % a.heads, tid = threadIdx.x;
  auto sync = [&] {
    if constexpr (CL > 1)
      cluster.sync();
    else
      __syncthreads();
  };
  // A shared variable of block r of the cluster.
  auto of = [&](int* p, int r) {
    if constexpr (CL > 1)
      return cluster.map_shared_rank(p, r);
    else
      return p;
  };
  const int len = a.length(b);
  const int chunk = (len + CL - 1) / CL, begin = min(rank * chunk, len),
            end = min(begin + chunk, len);
  if (h == 0 && rank == 0 && tid == 0) a.new_lengths[b] = min(len, a.budget);
  const float* given = a.prompt ? a.prompt + b * a.prompt_sb + h * a.prompt_sh : nullptr;
  if (len <= a.budget) {  // the same for the whole cluster
    if (rank == 0 && tid == 0) a.counts[row] = 0;
    if (given)
      for (int t = begin + tid; t < end; t += kEvictThreads) {
        const int64_t at = a.at(b, h, t);
        if (at >= 0) {
          a.weights[at] = given[t];
          a.positions[at] = t;
        }
      }
    return;
  }
  // Nothing stays, nothing is written, and no block of the cluster needs another:
  // what follows reaches into the others' shared memory only behind a barrier of
  // the cluster, and the radix passes, which have them, are for budgets above 0.
  if (a.budget == 0) {
    if (rank == 0 && tid == 0) a.counts[row] = 0;
    return;
  }

  // The largest position.
  int64_t recent_from = (int64_t)(len - 1) - a.recent;
  if (!given) {
    int mx = INT32_MIN;
    if (a.recent > 0)
      for (int t = begin + tid; t < end; t += kEvictThreads) {
        const int64_t at = a.at(b, h, t);
        if (at >= 0) mx = max(mx, a.positions[at]);
      }
    if (tid == 0) s_max = INT32_MIN;
    sync();
    mx = __reduce_max_sync(0xffffffffu, mx);
    if ((tid & 31) == 0 && mx != INT32_MIN)
      for (int r = 0; r < CL; ++r) atomicMax(of(&s_max, r), mx);
    sync();
    recent_from = a.recent > 0 ? (int64_t)s_max - a.recent : INT64_MAX;
  } else if (a.recent == 0) {
    recent_from = INT64_MAX;
  }
  auto read_key = [&](int t) {
    const int64_t at = a.at(b, h, t);
    if (at < 0) return 0u;
    const int pos = given ? t : (a.sinks > 0 || a.recent > 0 ? a.positions[at] : INT32_MAX);
    const bool safe = pos < a.sinks || (int64_t)pos > recent_from;
    return weight_key(given ? __ldg(given + t) : a.weights[at], safe);
  };
  // Key i lies at i + i / 32, so that threads that walk runs of them meet
  // different banks.
  {
    const int kept = min(end - begin, kKeep);
    for (int i0 = tid; i0 < kept; i0 += 4 * kEvictThreads) {
      uint32_t k[4];
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const int i = i0 + u * kEvictThreads;
        k[u] = read_key(begin + min(i, kept - 1));
      }
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const int i = i0 + u * kEvictThreads;
        if (i < kept) s_key[i + (i >> 5)] = k[u];
      }
    }
  }
  auto key = [&](int t) {
    const int i = t - begin;
    return i < kKeep ? s_key[i + (i >> 5)] : read_key(t);
  };

  // The key of the last token that stays, and how many of its equals do.  A token
  // on a page outside the pool cannot stay, and one before the budget is a place
  // that no other can take: as many fewer stay.
  uint32_t prefix = 0, mask = 0;
  int need = a.budget;
#pragma unroll 1
  for (int pass = 0; pass < 3; ++pass) {
    const int shift = pass == 0 ? 21 : pass == 1 ? 10 : 0, bits = pass == 2 ? 10 : 11;
    for (int i = tid; i < kBins; i += kEvictThreads) s_hist[i] = 0;
    if (pass == 0 && tid == 0) s_missing = 0;
    sync();
    int missing = 0;
    for (int t = begin + tid; t < end; t += kEvictThreads) {
      const uint32_t k = key(t);
      missing += k == 0u && t < a.budget;
      if ((k & mask) == prefix) atomicAdd(&s_hist[(k >> shift) & ((1u << bits) - 1u)], 1);
    }
    if (pass == 0) {
      missing = __reduce_add_sync(0xffffffffu, missing);
      if ((tid & 31) == 0 && missing) atomicAdd(of(&s_missing, 0), missing);
    }
    if constexpr (CL > 1) {
      __syncthreads();
      if (rank) {
        int* first = of(s_hist, 0);
        for (int i = tid; i < kBins; i += kEvictThreads)
          if (s_hist[i]) atomicAdd(first + i, s_hist[i]);
      }
    }
    sync();
    if (rank == 0) {
      if (pass == 0) need -= s_missing;
      if (need == 0 && tid == 0)  // no place at all: no key is above the last digits
        for (int r = 0; r < CL; ++r) {
          *of(&s_digit, r) = (1 << bits) - 1;
          *of(&s_left, r) = 0;
        }
      // Four bins a thread from the highest down: where the count reaches `need`.
      constexpr int each = kBins / kEvictThreads;
      int c[each], sum = 0, total;
#pragma unroll
      for (int i = 0; i < each; ++i) {
        c[i] = s_hist[kBins - 1 - (tid * each + i)];
        sum += c[i];
      }
      int before = block_scan(sum, s_warp, total);
#pragma unroll
      for (int i = 0; i < each; ++i) {
        if (before < need && before + c[i] >= need)
          for (int r = 0; r < CL; ++r) {
            *of(&s_digit, r) = kBins - 1 - (tid * each + i);
            *of(&s_left, r) = need - before;
          }
        before += c[i];
      }
    }
    sync();
    prefix |= (uint32_t)s_digit << shift;
    mask |= ((1u << bits) - 1u) << shift;
    need = s_left;
  }

  // Tokens above `prefix` and the first `need` of its equals stay.  A thread takes
  // a run of the block's tokens: it counts its equals, then its holes and movers,
  // and lists them behind those of the threads and blocks before it.
  const int budget = a.budget;
  __syncthreads();
  const int run = (end - begin + kEvictThreads - 1) / kEvictThreads;
  const int from = min(begin + tid * run, end), to = min(from + run, end);
  int ties = 0;
  for (int t = from; t < to; ++t) ties += key(t) == prefix;
  int total;
  int tie = block_scan(ties, s_warp, total);
  if constexpr (CL > 1) {
    if (tid == 0)
      for (int r = 0; r < CL; ++r) *of(&s_rank[0][rank], r) = total;
    cluster.sync();
    for (int r = 0; r < rank; ++r) tie += s_rank[0][r];
  }
  auto stays = [&](uint32_t k, int& tie) {
    if (k < prefix) return false;
    return k > prefix || tie++ < need;
  };
  int holes_n = 0, movers_n = 0, tie1 = tie;
  for (int t = from; t < to; ++t) {
    const uint32_t k = key(t);
    const bool kept = stays(k, tie1);
    holes_n += t < budget && !kept && k;
    movers_n += t >= budget && kept;
  }
  // (counts of a block are below 2^30: two scans, as one word holds only one)
  int block_holes, block_movers;
  int at_hole = block_scan(holes_n, s_warp, block_holes);
  int at_mover = block_scan(movers_n, s_warp, block_movers);
  if constexpr (CL > 1) {
    if (tid == 0)
      for (int r = 0; r < CL; ++r) {
        *of(&s_rank[1][rank], r) = block_holes;
        *of(&s_rank[2][rank], r) = block_movers;
      }
    cluster.sync();
    for (int r = 0; r < rank; ++r) {
      at_hole += s_rank[1][r];
      at_mover += s_rank[2][r];
    }
    block_holes = block_movers = 0;
    for (int r = 0; r < CL; ++r) {
      block_holes += s_rank[1][r];
      block_movers += s_rank[2][r];
    }
  }
  if (rank == 0 && tid == 0) a.counts[row] = min(block_holes, block_movers);
  int32_t* holes = a.lists + (int64_t)row * 2 * a.list_width;
  int32_t* movers = holes + a.list_width;
  for (int t = from; t < to; ++t) {
    const uint32_t k = key(t);
    const bool kept = stays(k, tie);
    if (t < budget && !kept && k) holes[at_hole++] = t;
    if (t >= budget && kept) movers[at_mover++] = t;
  }
  if (given && begin < budget) {
    // A kept token of a prompt that stays in its place gets its weight and position:
    // every token before the budget does, and a hole's are overwritten by its mover's.
    for (int t = begin + tid; t < min(end, budget); t += kEvictThreads) {
      const int64_t at = a.at(b, h, t);
      if (at >= 0) {
        a.weights[at] = given[t];
        a.positions[at] = t;
      }
    }
  }
}

// A warp takes 32 pairs: a lane each for the addresses, then the rows' 16-byte
// pieces one after another.
__global__ void __launch_bounds__(256) kv_move_kernel(EvictArgs a) {
  const int lane = threadIdx.x & 31;
  const int row = blockIdx.y, b = row / a.heads, h = row % a.heads;
  const int n = a.counts[row];
  const int32_t* holes = a.lists + (int64_t)row * 2 * a.list_width;
  const int32_t* movers = holes + a.list_width;
  const int warps = gridDim.x * (blockDim.x >> 5);
  const int nk = (int)(a.sk.ldb / 16), pieces = nk + (int)(a.sv.ldb / 16);
  for (int i0 = (blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5)) * 32; i0 < n;
       i0 += warps * 32) {
    const int i = i0 + lane;
    int64_t to = -1, from = -1;
    if (i < n) {
      const int ts = movers[i];
      to = a.at(b, h, holes[i]);
      from = a.at(b, h, ts);
      if (to < 0 || from < 0) {
        to = from = -1;
      } else {
        a.sk.norms[to] = a.sk.norms[from];
        a.sv.norms[to] = a.sv.norms[from];
        a.positions[to] = a.prompt ? ts : a.positions[from];
        a.weights[to] =
            a.prompt ? a.prompt[b * a.prompt_sb + h * a.prompt_sh + ts] : a.weights[from];
      }
    }
    // Four loads before their stores.
    for (int j0 = 0; j0 < pieces; j0 += 4) {
      uint4 w[4];
      uint4* dst[4];
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const int j = lane + 32 * (j0 + u), pair = min(j / pieces, 31), piece = j % pieces;
        const int64_t x = __shfl_sync(0xffffffffu, from, pair);
        const int64_t y = __shfl_sync(0xffffffffu, to, pair);
        dst[u] = nullptr;
        if (j0 + u < pieces && x >= 0) {
          const uint8_t* src = piece < nk ? a.sk.rows + x * a.sk.ldb + piece * 16
                                          : a.sv.rows + x * a.sv.ldb + (piece - nk) * 16;
          dst[u] = reinterpret_cast<uint4*>(piece < nk
                                                ? a.sk.rows + y * a.sk.ldb + piece * 16
                                                : a.sv.rows + y * a.sv.ldb + (piece - nk) * 16);
          w[u] = *reinterpret_cast<const uint4*>(src);
        }
      }
#pragma unroll
      for (int u = 0; u < 4; ++u)
        if (dst[u]) *dst[u] = w[u];
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

template <int CL>
int launch_select(const EvictArgs& a, int rows, int64_t width, cudaStream_t st) {
  const int keep = (int)min((int64_t)kKeep, (width + CL - 1) / CL);
  // (and the gaps between every 32 of them)
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)rows * CL);
  cfg.blockDim = dim3(kEvictThreads);
  cfg.dynamicSmemBytes = (size_t)(keep + keep / 32 + 1) * 4;
  cfg.stream = st;
  cudaLaunchAttribute at;
  at.id = cudaLaunchAttributeClusterDimension;
  at.val.clusterDim.x = CL;
  at.val.clusterDim.y = at.val.clusterDim.z = 1;
  cfg.attrs = &at;
  cfg.numAttrs = 1;
  const int rc = allow_smem<kv_select_kernel<CL>>((kKeep + kKeep / 32 + 1) * 4);
  if (rc) return rc;
  PQ_CUDA_TRY(cudaLaunchKernelEx(&cfg, kv_select_kernel<CL>, a));
  PQ_LAUNCH_CHECK("kv_select_kernel");
  return PQ_OK;
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
  PQ_CHECK_ARG(new_lengths + batch <= lengths || lengths + batch <= new_lengths,
               "new_lengths must not overlap lengths");
  a.sk = kv::side_k(c);
  a.sv = kv::side_v(c);
  a.heads = c.heads;
  a.pages = c.pages;
  a.page_shift = kv::page_shift_of(c);
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
  const int64_t width = (int64_t)table_width * c.page_size;
  // A cluster for long rows, unless there are more than fit at once (three blocks
  // an SM) and a block can keep all keys.  One block next to a cluster, us:
  //   8 rows of 4096 tokens 18.6, 15.4; of 16384 50, 20; 48 rows of 4096 19.5, 23.6;
  //   of 8192 28, 26; of 16384 50, 30; 128 rows of 8192 28, 60; of 16384 51, 70;
  //   of 65536 438, 149; 512 rows of 8192 65, 214; of 32768 485, 366
  const bool apart = width > kv::kKeep || (width > 4096 && rows * 8 <= 3 * num_sms());
  rc = apart ? kv::launch_select<8>(a, rows, width, st) : kv::launch_select<1>(a, rows, width, st);
  if (rc) return rc;
  if (a.list_width) {
    const int64_t per = (a.list_width + 255) / 256;
    const dim3 grid((unsigned)min(per, (int64_t)max(1, 8 * num_sms() / rows)), rows);
    kv::kv_move_kernel<<<grid, 256, 0, st>>>(a);
    PQ_LAUNCH_CHECK("kv_move_kernel");
  }
  return PQ_OK;
}

}  // extern "C"
