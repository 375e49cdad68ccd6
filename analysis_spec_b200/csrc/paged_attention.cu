// Attention of one new token per sequence over a paged KV cache.
//
//   out[b][0][hq][:] = sum_c softmax_c(scale q[b][hq] . k_c) v_c,   c < lengths[b]
// with k_c / v_c the rows of KV head hq / g (g = q_heads / kv_heads) that the page table names.
// A sequence of length 0 gives zeros. Scores, softmax statistics and output sums in fp32.
#include "paged.cuh"

namespace speckv {
namespace {

struct PagedArgs {
  const void* q;
  const void* k;
  const void* v;
  void* out;
  long long qs[2], ks[3], vs[3];
  PageTable table;
  const int64_t* lengths;
  long long batch, q_heads, kv_heads, dim;
  float scale_log2;  // scale * log2(e): the softmax runs in powers of two
  unsigned long long* err;
};

// Positions of sequence b: its length, cut to what the table can name (reported).
__device__ __forceinline__ long long live_length(const PagedArgs& a, long long b) {
  long long n = a.lengths[b];
  const long long most = a.table.width * a.table.page_size;
  if (n > most) {
    record_error(a.err, SPECKV_DERR_PAGE_TABLE, n);
    n = most;
  }
  return n < 0 ? 0 : n;
}

constexpr int kScalarWarps = 8;
constexpr int kScalarDims = 8;  // dims per lane: head dims to 256

// CTA per (sequence, query head), a key per warp and step: any head dim to 256, stride, alignment.
template <typename T>
__global__ void __launch_bounds__(kScalarWarps * 32) paged_attention_scalar_kernel(PagedArgs a) {
  const long long b = blockIdx.x / a.q_heads, hq = blockIdx.x % a.q_heads;
  const long long hk = hq / (a.q_heads / a.kv_heads);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, D = (int)a.dim;
  const T* q = static_cast<const T*>(a.q) + b * a.qs[0] + hq * a.qs[1];
  const long long n = live_length(a, b);
  float qr[kScalarDims], o[kScalarDims], m = -INFINITY, l = 0.f;
#pragma unroll
  for (int j = 0; j < kScalarDims; ++j) {
    qr[j] = lane + 32 * j < D ? load_f<T>(q[lane + 32 * j]) : 0.f;
    o[j] = 0.f;
  }
  for (long long c = warp; c < n; c += kScalarWarps) {
    const long long index = c / a.table.page_size, row = c - index * a.table.page_size;
    const long long page = a.table.page(b, index, a.err);
    if (page < 0) continue;
    const T* k = static_cast<const T*>(a.k) + page * a.ks[0] + hk * a.ks[1] + row * a.ks[2];
    const T* v = static_cast<const T*>(a.v) + page * a.vs[0] + hk * a.vs[1] + row * a.vs[2];
    float s = 0.f;
#pragma unroll
    for (int j = 0; j < kScalarDims; ++j)
      if (lane + 32 * j < D) s = fmaf(qr[j], load_f<T>(k[lane + 32 * j]), s);
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) s += __shfl_xor_sync(0xffffffffu, s, off);
    s *= a.scale_log2;
    const float top = fmaxf(m, s);
    const float base = top == -INFINITY ? 0.f : top;
    const float keep = exp2f(m - base), p = exp2f(s - base);
    l = l * keep + p;
    m = top;
#pragma unroll
    for (int j = 0; j < kScalarDims; ++j)
      if (lane + 32 * j < D) o[j] = fmaf(p, load_f<T>(v[lane + 32 * j]), o[j] * keep);
  }
  __shared__ float sm[kScalarWarps], sl[kScalarWarps], so[kScalarWarps][kScalarDims * 32];
  if (lane == 0) {
    sm[warp] = m;
    sl[warp] = l;
  }
#pragma unroll
  for (int j = 0; j < kScalarDims; ++j) so[warp][lane + 32 * j] = o[j];
  __syncthreads();
  float top = -INFINITY;
  for (int w = 0; w < kScalarWarps; ++w) top = fmaxf(top, sm[w]);
  const float base = top == -INFINITY ? 0.f : top;
  for (int d = threadIdx.x; d < D; d += kScalarWarps * 32) {
    float sum = 0.f, total = 0.f;
    for (int w = 0; w < kScalarWarps; ++w) {
      const float f = exp2f(sm[w] - base);
      total = fmaf(sl[w], f, total);
      sum = fmaf(so[w][d], f, sum);
    }
    // NaN sums pass through: only a sequence with nothing to see divides by zero
    static_cast<T*>(a.out)[(b * a.q_heads + hq) * a.dim + d] = store_f<T>(total == 0.f ? 0.f : sum / total);
  }
}

template <typename T>
int launch_paged(const PagedArgs& a, cudaStream_t s) {
  paged_attention_scalar_kernel<T><<<(unsigned)(a.batch * a.q_heads), kScalarWarps * 32, 0, s>>>(a);
  return check_launch("speckv_paged_attention");
}

}  // namespace
}  // namespace speckv

using namespace speckv;

extern "C" int speckv_paged_attention(const void* query, const void* key_pages, const void* value_pages,
                                      const int64_t* strides, const int64_t* page_table, int64_t table_stride,
                                      int64_t table_pages, int64_t num_pages, int64_t page_size,
                                      const int64_t* lengths, void* out, int64_t batch, int64_t q_heads,
                                      int64_t kv_heads, int64_t dim, float scale, int32_t dtype, void* stream) {
  const char* fn = "speckv_paged_attention";
  if (batch < 0 || q_heads < 1 || kv_heads < 1 || dim < 1) return fail(SPECKV_EINVAL, "%s: bad sizes", fn);
  if (q_heads % kv_heads != 0)
    return fail(SPECKV_EINVAL, "%s: %lld query heads not a multiple of %lld kv heads", fn, (long long)q_heads,
                (long long)kv_heads);
  if (dtype != SPECKV_F32 && dtype != SPECKV_BF16 && dtype != SPECKV_F16)
    return fail(SPECKV_EINVAL, "%s: unsupported dtype %d", fn, dtype);
  int st = check_pages(fn, page_table, table_stride, table_pages, num_pages, page_size, batch);
  if (st) return st;
  if (dim > 256) return fail(SPECKV_ENOSUPPORT, "%s: head dim %lld above 256", fn, (long long)dim);
  if (batch == 0) return SPECKV_OK;
  if (batch > (1 << 20) || q_heads > 1024 || batch * q_heads >= (1ll << 31))
    return fail(SPECKV_ENOSUPPORT, "%s: more than 2^20 sequences or 1024 query heads", fn);
  if (!query || !key_pages || !value_pages || !strides || !lengths || !out)
    return fail(SPECKV_EINVAL, "%s: null pointer", fn);
  st = check_current_device(fn, {query, key_pages, page_table, out});
  if (st) return st;
  PagedArgs a;
  a.q = query;
  a.k = key_pages;
  a.v = value_pages;
  a.out = out;
  a.qs[0] = strides[0];
  a.qs[1] = strides[1];
  for (int i = 0; i < 3; ++i) {
    a.ks[i] = strides[2 + i];
    a.vs[i] = strides[5 + i];
  }
  a.table = {page_table, table_stride, table_pages, num_pages, page_size};
  a.lengths = lengths;
  a.batch = batch;
  a.q_heads = q_heads;
  a.kv_heads = kv_heads;
  a.dim = dim;
  a.scale_log2 = scale * 1.4426950408889634f;
  a.err = device_error_word();
  if (a.err == nullptr) return fail(SPECKV_ECUDA, "%s: no error word on device", fn);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  switch (dtype) {
    case SPECKV_F32: return launch_paged<float>(a, s);
    case SPECKV_BF16: return launch_paged<__nv_bfloat16>(a, s);
    default: return launch_paged<__half>(a, s);
  }
}
