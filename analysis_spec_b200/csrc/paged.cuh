// Paged KV cache: pools of pages (page, kv_head, position in page, dim), strided with unit
// stride on dim, and a table whose entry [b][i] is the pool page of positions
// [i * page_size, (i + 1) * page_size) of sequence b. Shared by the append and the attention.
#pragma once

#include "common.cuh"

#include <cuda_bf16.h>
#include <cuda_fp16.h>

namespace speckv {

template <typename T> __device__ __forceinline__ float load_f(T x);
template <> __device__ __forceinline__ float load_f<float>(float x) { return x; }
template <> __device__ __forceinline__ float load_f<__nv_bfloat16>(__nv_bfloat16 x) { return __bfloat162float(x); }
template <> __device__ __forceinline__ float load_f<__half>(__half x) { return __half2float(x); }
template <typename T> __device__ __forceinline__ T store_f(float x);
template <> __device__ __forceinline__ float store_f<float>(float x) { return x; }
template <> __device__ __forceinline__ __nv_bfloat16 store_f<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }
template <> __device__ __forceinline__ __half store_f<__half>(float x) { return __float2half_rn(x); }

struct PageTable {
  const int64_t* entries;
  long long stride;      // entries between two sequences
  long long width;       // entries of one sequence
  long long num_pages;   // pages of the pools
  long long page_size;   // positions of a page

  // Pool page of table entry i of sequence b; -1, reported once, when it is not a page of the pools.
  __device__ __forceinline__ long long page(long long b, long long i, unsigned long long* err) const {
    const long long p = entries[b * stride + i];
    if (p < 0 || p >= num_pages) {
      record_error(err, SPECKV_DERR_PAGE_TABLE, p);
      return -1;
    }
    return p;
  }
};

// Host checks that both paged entries share.
inline int check_pages(const char* fn, const int64_t* table, int64_t table_stride, int64_t table_pages,
                       int64_t num_pages, int64_t page_size, int64_t batch) {
  if (page_size < 1 || page_size > (1 << 20) || num_pages < 1 || num_pages > (1ll << 31) || table_pages < 1 ||
      table_pages > (1ll << 31))
    return fail(SPECKV_EINVAL, "%s: bad page geometry (%lld pages of %lld positions, table of %lld)", fn,
                (long long)num_pages, (long long)page_size, (long long)table_pages);
  if (table_pages * page_size > (1ll << 31))
    return fail(SPECKV_ENOSUPPORT, "%s: a sequence of more than 2^31 positions", fn);
  if (table == nullptr || (batch > 1 && table_stride < table_pages))
    return fail(SPECKV_EINVAL, "%s: page table rows overlap or are missing", fn);
  return SPECKV_OK;
}

// Strides of dimensions of one entry are never taken: they count as 0, so that an odd one does not cost a call
// its aligned kernel (4000 keys of 8 q / 1 KV heads x 128 in bf16 with a head stride of 7: 12.5 us, 420 before).
inline void drop_unused_strides(long long* strides, std::initializer_list<int64_t> sizes) {
  for (const int64_t n : sizes) {
    if (n == 1) *strides = 0;
    ++strides;
  }
}

inline int check_strides(const char* fn, const int64_t* strides, int n) {
  for (int i = 0; i < n; ++i)
    if (strides[i] < 0) return fail(SPECKV_EINVAL, "%s: negative stride %lld", fn, (long long)strides[i]);
  return SPECKV_OK;
}

}  // namespace speckv
