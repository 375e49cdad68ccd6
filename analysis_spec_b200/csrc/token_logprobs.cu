// Log-probabilities of given tokens under rows of logits, with the entropy of each row and its
// top alternatives, and their gradient.
//
//   z = x / T,  lse = log sum_i exp(z_i),  p_i = exp(z_i - lse)
//   logprob = z_token - lse        entropy = lse - sum_i p_i z_i
//   top_ids: the k largest x, equal ones by the lower index (-0 equals 0, NaN below every
//   number); top_logprobs = z_id - lse
//   dx_i = 1/T [ g_lp (d_i,token - p_i) - g_H p_i (log p_i + entropy) + sum_j g_j (d_i,id_j - p_i) ]
// Statistics in fp32 whatever the logits' type. A row whose token (or source row) is negative is
// skipped: not read, zeros out, ids -1, gradient 0. A row of -inf alone has nothing to choose
// from: logprob -inf, entropy 0, gradient 0. NaN or +inf in a row makes its numbers NaN.
#include "paged.cuh"

namespace speckv {
namespace {

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;

struct ScoreArgs {
  const void* logits;
  long long sb, sr;          // element strides of (sequence, row); unit stride on the vocabulary
  const int64_t* tokens;     // may be null
  long long tb, tr;
  const int64_t* rows;       // source row of each output row; may be null (its own)
  long long rb, rr;
  long long batch, per, source_rows, vocab;
  float inv_t;
  int top;
  float* logprobs;
  float* entropy;
  float* lse;
  float* top_logprobs;
  int64_t* top_ids;
  unsigned long long* err;
  // gradient
  const float* g_logprobs;
  const float* g_entropy;
  const float* g_top;
  void* grad;                // (batch * per, vocab) contiguous
};

// Source element offset and token of output row n; false when the row is skipped.
__device__ __forceinline__ bool score_row(const ScoreArgs& a, long long n, long long& offset, long long& token) {
  const long long b = n / a.per, r = n - b * a.per;
  token = -1;
  if (a.tokens != nullptr) {
    token = a.tokens[b * a.tb + r * a.tr];
    if (token < 0) return false;
    if (token >= a.vocab) {
      record_error(a.err, SPECKV_DERR_TOKEN_INDEX, token);
      return false;
    }
  }
  long long src = r;
  if (a.rows != nullptr) {
    src = a.rows[b * a.rb + r * a.rr];
    if (src < 0) return false;
    if (src >= a.source_rows) {
      record_error(a.err, SPECKV_DERR_TOKEN_INDEX, src);
      return false;
    }
  }
  offset = b * a.sb + src * a.sr;
  return true;
}

// Order of the logits as unsigned integers: NaN 0, -0 and 0 alike.
__device__ __forceinline__ uint32_t order_key(float x) {
  if (x != x) return 0u;
  const uint32_t u = __float_as_uint(x + 0.f);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}

constexpr int kScoreThreads = 256;

template <typename F> __device__ __forceinline__ float block_reduce(float x, float* buf, F f) {
  for (int off = 16; off > 0; off >>= 1) x = f(x, __shfl_xor_sync(0xffffffffu, x, off));
  __syncthreads();
  if ((threadIdx.x & 31) == 0) buf[threadIdx.x >> 5] = x;
  __syncthreads();
  x = buf[0];
  for (int w = 1; w < kScoreThreads / 32; ++w) x = f(x, buf[w]);
  return x;
}

__device__ __forceinline__ void write_skipped(const ScoreArgs& a, long long n) {
  if (threadIdx.x == 0) {
    if (a.logprobs != nullptr) a.logprobs[n] = 0.f;
    a.entropy[n] = 0.f;
    a.lse[n] = 0.f;
  }
  for (int j = threadIdx.x; j < a.top; j += blockDim.x) {
    a.top_logprobs[n * a.top + j] = 0.f;
    a.top_ids[n * a.top + j] = -1;
  }
}

// CTA per row: the maximum, then the sums, then k scans for the alternatives.
template <typename T>
__global__ void __launch_bounds__(kScoreThreads) token_logprobs_kernel(ScoreArgs a) {
  __shared__ float buf[kScoreThreads / 32];
  __shared__ unsigned long long best;
  const long long n = blockIdx.x;
  long long offset = 0, token = -1;
  if (!score_row(a, n, offset, token)) {
    write_skipped(a, n);
    return;
  }
  const T* x = static_cast<const T*>(a.logits) + offset;
  float m = -INFINITY;
  bool nan = false;
  for (long long i = threadIdx.x; i < a.vocab; i += kScoreThreads) {
    const float z = load_f<T>(x[i]);
    nan |= z != z || z == INFINITY;
    m = fmaxf(m, z);
  }
  nan = __syncthreads_or(nan);
  m = block_reduce(m, buf, [](float u, float v) { return fmaxf(u, v); });
  const float base = m == -INFINITY ? 0.f : m;
  float s = 0.f, t = 0.f;
  for (long long i = threadIdx.x; i < a.vocab; i += kScoreThreads) {
    const float y = (load_f<T>(x[i]) - base) * a.inv_t;
    const float e = expf(y);
    s += e;
    t += e > 0.f ? e * y : 0.f;
  }
  s = block_reduce(s, buf, [](float u, float v) { return u + v; });
  t = block_reduce(t, buf, [](float u, float v) { return u + v; });
  const bool empty = m == -INFINITY && !nan;
  const float log_s = logf(s);
  const float lse = nan ? NAN : empty ? -INFINITY : base * a.inv_t + log_s;
  if (threadIdx.x == 0) {
    if (a.logprobs != nullptr) {
      const float y = (load_f<T>(x[token]) - base) * a.inv_t;
      a.logprobs[n] = nan ? NAN : empty ? -INFINITY : y - log_s;
    }
    a.entropy[n] = nan ? NAN : empty ? 0.f : log_s - t / s;
    a.lse[n] = lse;
  }
  unsigned long long last = ~0ull;
  for (int j = 0; j < a.top; ++j) {
    __syncthreads();
    if (threadIdx.x == 0) best = 0ull;
    __syncthreads();
    unsigned long long mine = 0ull;
    for (long long i = threadIdx.x; i < a.vocab; i += kScoreThreads) {
      const unsigned long long key = (unsigned long long)order_key(load_f<T>(x[i])) << 32 | (0xffffffffu - (uint32_t)i);
      if (key < last && key > mine) mine = key;
    }
    atomicMax(&best, mine);
    __syncthreads();
    last = best;
    if (threadIdx.x == 0) {
      const long long id = 0xffffffffu - (uint32_t)last;
      a.top_ids[n * a.top + j] = id;
      const float y = (load_f<T>(x[id]) - base) * a.inv_t;
      a.top_logprobs[n * a.top + j] = nan ? NAN : empty ? -INFINITY : y - log_s;
    }
  }
}

// CTA per row, elements one by one.
template <typename T>
__global__ void __launch_bounds__(kScoreThreads) token_logprobs_backward_kernel(ScoreArgs a) {
  const long long n = blockIdx.x;
  T* g = static_cast<T*>(a.grad) + n * a.vocab;
  long long offset = 0, token = -1;
  const bool live = score_row(a, n, offset, token) && a.lse[n] != -INFINITY;
  if (!live) {
    for (long long i = threadIdx.x; i < a.vocab; i += kScoreThreads) g[i] = store_f<T>(0.f);
    return;
  }
  const T* x = static_cast<const T*>(a.logits) + offset;
  const float ga = a.g_logprobs != nullptr ? a.g_logprobs[n] : 0.f;
  const float gh = a.g_entropy != nullptr ? a.g_entropy[n] : 0.f;
  const float lse = a.lse[n], entropy = a.entropy[n];
  float all = ga;
  if (a.g_top != nullptr)
    for (int j = 0; j < a.top; ++j) all += a.g_top[n * a.top + j];
  for (long long i = threadIdx.x; i < a.vocab; i += kScoreThreads) {
    const float logp = load_f<T>(x[i]) * a.inv_t - lse;
    const float p = expf(logp);
    float d = p == 0.f ? 0.f : -p * (all + gh * (logp + entropy));
    if (i == token) d += ga;
    if (a.g_top != nullptr)
      for (int j = 0; j < a.top; ++j)
        if (a.top_ids[n * a.top + j] == i) d += a.g_top[n * a.top + j];
    g[i] = store_f<T>(d * a.inv_t);
  }
}

int check_scores(const char* fn, const void* logits, int32_t dtype, const int64_t* tokens, int64_t batch, int64_t per,
                 int64_t source_rows, int64_t vocab, float inv_temperature, int32_t top) {
  if (batch < 0 || per < 0 || source_rows < 0 || vocab < 1) return fail(SPECKV_EINVAL, "%s: bad sizes", fn);
  if (dtype != SPECKV_F32 && dtype != SPECKV_BF16 && dtype != SPECKV_F16)
    return fail(SPECKV_EINVAL, "%s: unsupported dtype %d", fn, dtype);
  if (!(inv_temperature > 0.f) || !(inv_temperature <= 3.0e38f))
    return fail(SPECKV_EINVAL, "%s: 1 / temperature must be positive and finite", fn);
  if (top < 0 || top > SPECKV_MAX_TOP || top > vocab)
    return fail(SPECKV_EINVAL, "%s: %d alternatives of %lld (at most %d)", fn, top, (long long)vocab, SPECKV_MAX_TOP);
  if (vocab >= (1ll << 31) || batch > (1ll << 31) || per > (1ll << 31) || batch * per >= (1ll << 31))
    return fail(SPECKV_ENOSUPPORT, "%s: 2^31 rows or entries or more", fn);
  return SPECKV_OK;
}

}  // namespace
}  // namespace speckv

using namespace speckv;

extern "C" int speckv_token_logprobs(const void* logits, int32_t dtype, int64_t stride_b, int64_t stride_r,
                                     const int64_t* tokens, int64_t tokens_stride_b, int64_t tokens_stride_r,
                                     const int64_t* rows, int64_t rows_stride_b, int64_t rows_stride_r,
                                     int64_t batch, int64_t per_batch, int64_t source_rows, int64_t vocab,
                                     float inv_temperature, int32_t top, float* logprobs, float* entropy, float* lse,
                                     float* top_logprobs, int64_t* top_ids, void* stream) {
  const char* fn = "speckv_token_logprobs";
  int st = check_scores(fn, logits, dtype, tokens, batch, per_batch, source_rows, vocab, inv_temperature, top);
  if (st || batch == 0 || per_batch == 0) return st;
  if (rows == nullptr && source_rows != per_batch)
    return fail(SPECKV_EINVAL, "%s: %lld rows of logits for %lld", fn, (long long)source_rows, (long long)per_batch);
  if (logits == nullptr || entropy == nullptr || lse == nullptr || (tokens == nullptr) != (logprobs == nullptr) ||
      (top > 0 && (top_logprobs == nullptr || top_ids == nullptr)))
    return fail(SPECKV_EINVAL, "%s: null pointer", fn);
  st = check_current_device(fn, {logits, tokens, entropy});
  if (st) return st;
  ScoreArgs a{};
  a.logits = logits;
  a.sb = stride_b;
  a.sr = stride_r;
  a.tokens = tokens;
  a.tb = tokens_stride_b;
  a.tr = tokens_stride_r;
  a.rows = rows;
  a.rb = rows_stride_b;
  a.rr = rows_stride_r;
  a.batch = batch;
  a.per = per_batch;
  a.source_rows = source_rows;
  a.vocab = vocab;
  a.inv_t = inv_temperature;
  a.top = top;
  a.logprobs = logprobs;
  a.entropy = entropy;
  a.lse = lse;
  a.top_logprobs = top_logprobs;
  a.top_ids = top_ids;
  a.err = device_error_word();
  if (a.err == nullptr) return fail(SPECKV_ECUDA, "%s: no error word on device", fn);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const unsigned grid = (unsigned)(batch * per_batch);
  switch (dtype) {
    case SPECKV_F32: token_logprobs_kernel<float><<<grid, kScoreThreads, 0, s>>>(a); break;
    case SPECKV_BF16: token_logprobs_kernel<__nv_bfloat16><<<grid, kScoreThreads, 0, s>>>(a); break;
    default: token_logprobs_kernel<__half><<<grid, kScoreThreads, 0, s>>>(a); break;
  }
  return check_launch(fn);
}

extern "C" int speckv_token_logprobs_backward(const void* logits, int32_t dtype, int64_t stride_b, int64_t stride_r,
                                              const int64_t* tokens, int64_t tokens_stride_b, int64_t tokens_stride_r,
                                              int64_t batch, int64_t per_batch, int64_t vocab, float inv_temperature,
                                              int32_t top, const float* entropy, const float* lse,
                                              const int64_t* top_ids, const float* grad_logprobs,
                                              const float* grad_entropy, const float* grad_top_logprobs,
                                              void* grad_logits, void* stream) {
  const char* fn = "speckv_token_logprobs_backward";
  int st = check_scores(fn, logits, dtype, tokens, batch, per_batch, per_batch, vocab, inv_temperature, top);
  if (st || batch == 0 || per_batch == 0) return st;
  if (logits == nullptr || entropy == nullptr || lse == nullptr || grad_logits == nullptr ||
      (grad_logprobs != nullptr && tokens == nullptr) ||
      (grad_top_logprobs != nullptr && (top < 1 || top_ids == nullptr)))
    return fail(SPECKV_EINVAL, "%s: null pointer", fn);
  st = check_current_device(fn, {logits, tokens, grad_logits});
  if (st) return st;
  ScoreArgs a{};
  a.logits = logits;
  a.sb = stride_b;
  a.sr = stride_r;
  a.tokens = tokens;
  a.tb = tokens_stride_b;
  a.tr = tokens_stride_r;
  a.batch = batch;
  a.per = per_batch;
  a.source_rows = per_batch;
  a.vocab = vocab;
  a.inv_t = inv_temperature;
  a.top = top;
  a.entropy = const_cast<float*>(entropy);
  a.lse = const_cast<float*>(lse);
  a.top_ids = const_cast<int64_t*>(top_ids);
  a.g_logprobs = grad_logprobs;
  a.g_entropy = grad_entropy;
  a.g_top = grad_top_logprobs;
  a.grad = grad_logits;
  a.err = device_error_word();
  if (a.err == nullptr) return fail(SPECKV_ECUDA, "%s: no error word on device", fn);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const unsigned grid = (unsigned)(batch * per_batch);
  switch (dtype) {
    case SPECKV_F32: token_logprobs_backward_kernel<float><<<grid, kScoreThreads, 0, s>>>(a); break;
    case SPECKV_BF16: token_logprobs_backward_kernel<__nv_bfloat16><<<grid, kScoreThreads, 0, s>>>(a); break;
    default: token_logprobs_backward_kernel<__half><<<grid, kScoreThreads, 0, s>>>(a); break;
  }
  return check_launch(fn);
}
