// Shared parts of the compressed key-value cache's kernels: argument checks,
// the tables of a codec, and the addresses of a page's rows.
#pragma once
#include <cuda_bf16.h>

#include <atomic>

#include "common.cuh"
#include "context.cuh"

namespace pqb {
namespace kv {

// One side's tables as pq_kv_prepare_codec lays them out.
struct Codec {
  const float* R;         // d x d
  const float* RT;        // its transpose
  const float* bounds;    // 2^bits - 1, then infinity
  const float* cent;      // 2^bits
  const uint2* pairs;     // [2][256] centroids * 2^exponent as f16, what a byte decodes to
                          // 4 bits: its two, twice; hi parts, then lo parts
                          // 2 bits: its first two and last two; hi, then lo
                          // 8 bits: hi and lo part, twice; then nothing
  const int* exponent;    // the largest centroid * 2^exponent lies in [2^13, 2^14)
  const float* range;     // cell of y = saturate(y * range[0] + range[1]) * (cells - 1), rounded
  const uint2* cells;     // [2048]: the cell's boundary (f32) and the code below it
  const uint2* planes;    // [2][D / 8][D / 16][32]: R * 2^14 as f16 hi and lo, in the order
                          // of mma.m16n8k16's B operand (kv_rows.cu)
  const __half* rows;     // [2][D][D]: the same planes row by row
};

constexpr int kCells = 2048;      // of a codec of 8 bits
constexpr int kFewCells = 64;     // of one of 2 or 4 bits
inline int padded_d(int d) { return d <= 64 ? 64 : d <= 128 ? 128 : 256; }

inline size_t codec_bytes(int d, int /*bits*/) {
  const size_t D = padded_d(d);
  return (size_t)2 * align_up((size_t)d * d * sizeof(float), 256) + 6 * 1024 + 256 +
         kCells * sizeof(uint2) + 2 * 2 * D * D * sizeof(__half);
}

inline Codec codec_of(const void* tables, int d) {
  const char* b = (const char*)tables;
  const size_t m = align_up((size_t)d * d * sizeof(float), 256);
  Codec c;
  c.R = (const float*)b;
  c.RT = (const float*)(b + m);
  b += 2 * m;
  c.bounds = (const float*)b;
  c.cent = (const float*)(b + 1024);
  c.pairs = (const uint2*)(b + 2048);
  c.exponent = (const int*)(b + 6144);
  c.range = (const float*)(b + 6144 + 64);
  c.cells = (const uint2*)(b + 6144 + 256);
  c.planes = c.cells + kCells;
  const int D = padded_d(d);
  c.rows = (const __half*)(c.planes + D * D / 2);
  return c;
}

// One side of the pool.
struct Side {
  uint8_t* rows;
  float* norms;
  int64_t ldb;
  int bits;
  Codec c;
};

inline Side side_k(const pq_kv_cache& c) {
  return Side{c.k_rows, c.k_norms, c.k_ldb, c.k_bits, codec_of(c.k_codec, c.d)};
}
inline Side side_v(const pq_kv_cache& c) {
  return Side{c.v_rows, c.v_norms, c.v_ldb, c.v_bits, codec_of(c.v_codec, c.d)};
}

inline int page_shift_of(const pq_kv_cache& c) {
  int s = 4;
  while ((1 << s) < c.page_size) ++s;
  return s;
}

inline bool bits_ok(int b) { return b == 2 || b == 4 || b == 8; }

inline int check_cache(const pq_kv_cache* c) {
  PQ_CHECK_ARG(c, "null cache");
  PQ_CHECK_ARG(c->d >= 1 && c->d <= PQ_KV_MAX_D, "d must be in [1, %d] (got %d)", PQ_KV_MAX_D,
               c->d);
  PQ_CHECK_ARG(bits_ok(c->k_bits) && bits_ok(c->v_bits),
               "k_bits and v_bits must be 2, 4 or 8 (got %d and %d)", c->k_bits, c->v_bits);
  PQ_CHECK_ARG(c->heads >= 1, "heads must be at least 1 (got %d)", c->heads);
  PQ_CHECK_ARG(c->pages >= 0, "pages must be at least 0 (got %d)", c->pages);
  PQ_CHECK_ARG(c->page_size >= 16 && c->page_size <= 1024 &&
                   (c->page_size & (c->page_size - 1)) == 0,
               "page_size must be a power of two from 16 to 1024 (got %d)", c->page_size);
  PQ_CHECK_ARG((int64_t)c->pages * c->page_size < (1ll << 31) &&
                   (int64_t)c->pages * c->heads * c->page_size < (1ll << 32) &&
                   (int64_t)c->pages * c->heads < (1ll << 31),
               "a pool has fewer than 2^31 slots and 2^32 rows");
  PQ_CHECK_ARG(c->k_ldb == (int64_t)align_up(row_bytes(c->d, c->k_bits), 16) &&
                   c->v_ldb == (int64_t)align_up(row_bytes(c->d, c->v_bits), 16),
               "k_ldb and v_ldb must be a row's packed bytes rounded up to 16 (got %lld and %lld)",
               (long long)c->k_ldb, (long long)c->v_ldb);
  PQ_CHECK_ARG(c->k_codec && c->v_codec, "null codec");
  PQ_CHECK_ARG(c->pages == 0 || (c->k_rows && c->v_rows && c->k_norms && c->v_norms &&
                                 c->positions && c->weights),
               "null pool pointer");
  PQ_CHECK_ARG(((uintptr_t)c->k_rows | (uintptr_t)c->v_rows | (uintptr_t)c->k_norms |
                (uintptr_t)c->v_norms | (uintptr_t)c->positions | (uintptr_t)c->weights) % 16 == 0,
               "the pool's arrays must be 16-byte aligned");
  return PQ_OK;
}

inline int check_dtype(int dtype) {
  PQ_CHECK_ARG(dtype == PQ_KV_F32 || dtype == PQ_KV_F16 || dtype == PQ_KV_BF16,
               "dtype must be 0 (f32), 1 (f16) or 2 (bf16) (got %d)", dtype);
  return PQ_OK;
}

inline int check_sequences(const int32_t* table, int table_width, const int32_t* lengths,
                           int batch, int page_size) {
  PQ_CHECK_ARG(table_width >= 0 && (int64_t)table_width * page_size <= (1ll << 30),
               "a sequence has at most 2^30 tokens");
  PQ_CHECK_ARG((table || table_width == 0) && lengths, "null table or lengths");
  PQ_CHECK_ARG(batch >= 0, "batch must be at least 0");
  return PQ_OK;
}

// Lets a kernel take more than 48 KB of dynamic shared memory, once in each
// context of a device (the runtime's call costs 1 us; a device's number above 63
// asks anew).  K is the kernel itself, so that each has ids of its own.
template <auto K>
inline int allow_smem(int bytes) {
  static std::atomic<unsigned long long> done[64];
  int dev = 0;
  PQ_CUDA_TRY(cudaGetDevice(&dev));
  const unsigned long long id = current_ctx_id();
  if (id && dev < 64 && done[dev].load(std::memory_order_relaxed) == id) return PQ_OK;
  PQ_CUDA_TRY(cudaFuncSetAttribute(K, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes));
  // (the call above made the context current, where there was none)
  if (dev < 64) done[dev].store(current_ctx_id(), std::memory_order_relaxed);
  return PQ_OK;
}

template <class T>
__device__ __forceinline__ float to_f32(T x);
template <>
__device__ __forceinline__ float to_f32<float>(float x) { return x; }
template <>
__device__ __forceinline__ float to_f32<__half>(__half x) { return __half2float(x); }
template <>
__device__ __forceinline__ float to_f32<__nv_bfloat16>(__nv_bfloat16 x) {
  return __bfloat162float(x);
}

template <class T>
__device__ __forceinline__ T from_f32(float x);
template <>
__device__ __forceinline__ float from_f32<float>(float x) { return x; }
template <>
__device__ __forceinline__ __half from_f32<__half>(float x) { return __float2half_rn(x); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float x) {
  return __float2bfloat16_rn(x);
}

// Runs the statement with T_ as the element type of `dtype`.
#define PQ_KV_DISPATCH_T(dtype, ...)      \
  do {                                    \
    if ((dtype) == PQ_KV_F32) {           \
      using T_ = float;                   \
      __VA_ARGS__;                        \
    } else if ((dtype) == PQ_KV_F16) {    \
      using T_ = __half;                  \
      __VA_ARGS__;                        \
    } else {                              \
      using T_ = __nv_bfloat16;           \
      __VA_ARGS__;                        \
    }                                     \
  } while (0)

__device__ __forceinline__ int clamp_length(int len, int table_width, int page_size) {
  return max(0, min(len, table_width * page_size));
}

}  // namespace kv
}  // namespace pqb
