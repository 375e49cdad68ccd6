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
#include "cluster.cuh"
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
  float* stats;              // (rows, 2): reference r, log2 of the sum of 2^((x - r) log2(e) / T)
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

__device__ __forceinline__ float order_value(uint32_t key) {
  return __uint_as_float(key & 0x80000000u ? key & 0x7fffffffu : ~key);
}

__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Maximum of two numbers; NaN when one of them is.
__device__ __forceinline__ float max_nan(float x, float y) {
  float z;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(z) : "f"(x), "f"(y));
  return z;
}

// Two fp32 numbers in one register pair, as the packed fp32 instructions take them.
typedef unsigned long long Two;
__device__ __forceinline__ Two two(float x, float y) {
  Two r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(x), "f"(y));
  return r;
}
__device__ __forceinline__ void parts(Two v, float& x, float& y) { asm("mov.b64 {%0, %1}, %2;" : "=f"(x), "=f"(y) : "l"(v)); }
__device__ __forceinline__ Two add2(Two x, Two y) {
  Two r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(x), "l"(y));
  return r;
}
__device__ __forceinline__ Two mul2(Two x, Two y) {
  Two r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(x), "l"(y));
  return r;
}
__device__ __forceinline__ Two fma2(Two x, Two y, Two z) {
  Two r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(x), "l"(y), "l"(z));
  return r;
}

// 32 bytes of logits, one load.
struct Bytes32 {
  uint32_t w[8];
};
__device__ __forceinline__ Bytes32 load_stream(const void* p) {
  Bytes32 r;
  asm volatile("ld.global.nc.L1::no_allocate.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
               : "=r"(r.w[0]), "=r"(r.w[1]), "=r"(r.w[2]), "=r"(r.w[3]), "=r"(r.w[4]), "=r"(r.w[5]), "=r"(r.w[6]),
                 "=r"(r.w[7])
               : "l"(p));
  return r;
}
__device__ __forceinline__ Bytes32 from_pieces(const uint4& a, const uint4& b) {
  return Bytes32{{a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w}};
}
__device__ __forceinline__ void store_stream(void* p, const Bytes32& v) {
  asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "r"(v.w[0]), "r"(v.w[1]),
               "r"(v.w[2]), "r"(v.w[3]), "r"(v.w[4]), "r"(v.w[5]), "r"(v.w[6]), "r"(v.w[7])
               : "memory");
}

__device__ __forceinline__ void copy_async(void* to, const void* from) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"((uint32_t)__cvta_generic_to_shared(to)), "l"(from)
               : "memory");
}

// The logits of one 32-bit word, their largest (NaN when one is), and what the fast sums take
// for them: kLow stands for anything lower, so that -inf has a weight of 0 and a finite distance.
template <typename T> struct Word;
template <> struct Word<float> {
  static constexpr int N = 1;
  static constexpr float kLow = -INFINITY;  // the distance is cut instead
  static constexpr uint32_t kNone = 0xff800000u;  // -inf
  static __device__ __forceinline__ uint32_t top(uint32_t x, uint32_t y) {
    return __float_as_uint(max_nan(__uint_as_float(x), __uint_as_float(y)));
  }
  static __device__ __forceinline__ float largest(uint32_t x) { return __uint_as_float(x); }
  static __device__ __forceinline__ uint32_t cut(uint32_t x) { return x; }
};
template <> struct Word<__nv_bfloat16> {
  static constexpr int N = 2;
  static constexpr float kLow = -1e30f;
  static constexpr uint32_t kNone = 0xff80ff80u;
  static __device__ __forceinline__ __nv_bfloat162 pair(uint32_t u) { return *reinterpret_cast<__nv_bfloat162*>(&u); }
  static __device__ __forceinline__ uint32_t bits(__nv_bfloat162 h) { return *reinterpret_cast<uint32_t*>(&h); }
  static __device__ __forceinline__ uint32_t top(uint32_t x, uint32_t y) { return bits(__hmax2_nan(pair(x), pair(y))); }
  static __device__ __forceinline__ void values(uint32_t u, float& x, float& y) {  // the upper half of an fp32
    x = __uint_as_float(u << 16);
    y = __uint_as_float(u & 0xffff0000u);
  }
  static __device__ __forceinline__ float largest(uint32_t u) {
    float x, y;
    values(u, x, y);
    return max_nan(x, y);
  }
  static __device__ __forceinline__ uint32_t cut(uint32_t u) {
    return bits(__hmax2(pair(u), pair(0xf149f149u)));  // -9.97e29
  }
  static __device__ __forceinline__ uint32_t pack(float x, float y) { return bits(__floats2bfloat162_rn(x, y)); }
};
template <> struct Word<__half> {
  static constexpr int N = 2;
  static constexpr float kLow = -65504.f;
  static constexpr uint32_t kNone = 0xfc00fc00u;
  static __device__ __forceinline__ __half2 pair(uint32_t u) { return *reinterpret_cast<__half2*>(&u); }
  static __device__ __forceinline__ uint32_t bits(__half2 h) { return *reinterpret_cast<uint32_t*>(&h); }
  static __device__ __forceinline__ uint32_t top(uint32_t x, uint32_t y) { return bits(__hmax2_nan(pair(x), pair(y))); }
  static __device__ __forceinline__ void values(uint32_t u, float& x, float& y) {
    const float2 f = __half22float2(pair(u));
    x = f.x;
    y = f.y;
  }
  static __device__ __forceinline__ float largest(uint32_t u) {
    float x, y;
    values(u, x, y);
    return max_nan(x, y);
  }
  static __device__ __forceinline__ uint32_t cut(uint32_t u) {
    return bits(__hmax2(pair(u), pair(0xfbfffbffu)));
  }
  static __device__ __forceinline__ uint32_t pack(float x, float y) { return bits(__floats2half2_rn(x, y)); }
};

// Two neighbouring logits of a vector (fp32: words 2 i and 2 i + 1; else word i).
template <typename T> __device__ __forceinline__ void pair_values(const Bytes32& v, int i, bool cut, float& x, float& y) {
  if constexpr (Word<T>::N == 1) {
    x = __uint_as_float(v.w[2 * i]);
    y = __uint_as_float(v.w[2 * i + 1]);
  } else {
    Word<T>::values(cut ? Word<T>::cut(v.w[i]) : v.w[i], x, y);
  }
}
template <typename T> __device__ __forceinline__ float vector_top(const Bytes32& v) {
  typedef Word<T> W;
  return W::largest(W::top(W::top(W::top(v.w[0], v.w[1]), W::top(v.w[2], v.w[3])),
                           W::top(W::top(v.w[4], v.w[5]), W::top(v.w[6], v.w[7]))));
}

// A row as single entries up to the first boundary of BYTES, whole pieces of that size, and
// single entries.
template <int BYTES> struct RowSplit {
  int head, pieces, tail;  // entries, pieces, entries
  __device__ __forceinline__ RowSplit(const void* row, int vocab, int size) {
    const int n = BYTES / size;
    head = min(vocab, (int)((BYTES - (reinterpret_cast<uintptr_t>(row) & (BYTES - 1))) & (BYTES - 1)) / size);
    pieces = (vocab - head) / n;
    tail = vocab - head - pieces * n;
  }
};

constexpr float kEmpty = -150.f;   // 2^-150 is 0 in fp32: where distances to the reference end
constexpr float kSlack = 10.f;     // a distance may pass the reference by 2^10 before it moves
constexpr float kWide = 1048576.f; // references to 2^20 take the fused product

// Sums of a thread over its entries, by a reference r (one of its entries) that stays within
// 2^kSlack of their maximum: y = (x - r) c, c = log2(e) / T, s = sum 2^y, t = sum 2^y y.
// y is one fused product x c - rc with rc = r c rounded; what that rounding left out is put back once
// at the end. References whose product is so large that the rounding would matter before that
// (a row of a mask's lowest value, say) take the difference first, vector by vector (wide).
template <typename T> struct Running {
  float r = -INFINITY, rc = 0.f, limit = NAN;  // a vector that is not below `limit` looks at the reference first
  Two s = 0ull, t = 0ull;  // of the even and the odd entries
  bool bad = false, wide = false;  // bad: NaN or +inf seen

  __device__ __forceinline__ void move(float top, float c, float wide_at) {
    if (top != top || top == INFINITY) {
      bad = true;
      return;
    }
    if (top > r) {
      const float to = top * c;
      const bool is_wide = !(fabsf(to) <= wide_at);
      // between the references the sums are by: r c itself where wide, else its rounding
      float d = rc - to;
      if (wide || is_wide) {
        d = (r - top) * c;
        if (!is_wide) d += fmaf(top, c, -to);
        if (!wide) d -= fmaf(r, c, -rc);
      }
      if (r == -INFINITY || d <= kEmpty) {
        s = t = 0ull;
      } else {
        const float f = exp2_fast(d);
        t = mul2(two(f, f), fma2(two(d, d), s, t));
        s = mul2(two(f, f), s);
      }
      r = top;
      rc = to;
      wide = is_wide;
      limit = wide ? NAN : top + fminf(kSlack / c, 1e30f);
    }
  }
  __device__ __forceinline__ void add(float y0, float y1) {
    const Two e = two(exp2_fast(y0), exp2_fast(y1));
    s = add2(s, e);
    t = fma2(e, two(y0, y1), t);
  }
  __device__ __forceinline__ void add_vector(const Bytes32& v, float c) {
#pragma unroll
    for (int i = 0; i < 16 / (int)sizeof(T); ++i) {
      float x0, x1, y0, y1;
      pair_values<T>(v, i, true, x0, x1);
      parts(fma2(two(x0, x1), two(c, c), two(-rc, -rc)), y0, y1);
      if (sizeof(T) == 4) {
        y0 = fmaxf(y0, kEmpty);
        y1 = fmaxf(y1, kEmpty);
      }
      add(y0, y1);
    }
  }
  __device__ __forceinline__ void add_wide(float x0, float x1, float c) {
    add(fmaxf((x0 - r) * c, kEmpty), fmaxf((x1 - r) * c, kEmpty));
  }
  __device__ __forceinline__ void vector(const Bytes32& v, float top, float c, float wide_at) {
    if (!(top <= limit)) {
      move(top, c, wide_at);
      if (wide) {
#pragma unroll
        for (int i = 0; i < 16 / (int)sizeof(T); ++i) {
          float x0, x1;
          pair_values<T>(v, i, false, x0, x1);
          add_wide(x0, x1, c);
        }
        return;
      }
      // No entry above -inf yet: nothing to add. What stands for -inf has a finite distance from a reference
      // that takes the fused product only; from none it would pass fp32's range at c above 3e8 (0 x inf).
      if (r == -INFINITY) return;
    }
    add_vector(v, c);
  }
  __device__ __forceinline__ void single(float x, float c, float wide_at) {
    if (!(x <= limit)) move(x, c, wide_at);
    if (wide)
      add_wide(x, -INFINITY, c);
    else
      add(fmaxf(fmaf(x, c, -rc), kEmpty), kEmpty);
  }
  // The sums by r itself.
  __device__ __forceinline__ void finish(float c, float& s1, float& t1) {
    float s2, t2;
    parts(s, s1, s2);
    parts(t, t1, t2);
    s1 += s2;
    t1 += t2;
    if (!wide && r != -INFINITY) {
      const float d = fmaf(r, c, -rc), f = exp2_fast(-d);
      t1 = f * fmaf(-d, s1, t1);
      s1 *= f;
    }
  }
};

// Joins the sums of two references.
__device__ __forceinline__ void join_sums(float& r, float& s, float& t, float r2, float s2, float t2, float c) {
  const float to = fmaxf(r, r2);  // -inf for both: no entry, sums of 0
  const float d = fmaxf((r - to) * c, kEmpty), d2 = fmaxf((r2 - to) * c, kEmpty);
  const float f = exp2_fast(d), f2 = exp2_fast(d2);
  t = f * fmaf(d, s, t) + f2 * fmaf(d2, s2, t2);
  s = f * s + f2 * s2;
  r = to;
}

__device__ __forceinline__ void write_skipped(const ScoreArgs& a, long long n) {
  if (threadIdx.x == 0) {
    if (a.logprobs != nullptr) a.logprobs[n] = 0.f;
    a.entropy[n] = 0.f;
    if (a.stats != nullptr) a.stats[2 * n] = a.stats[2 * n + 1] = 0.f;
  }
  for (int j = threadIdx.x; j < a.top; j += blockDim.x) {
    a.top_logprobs[n * a.top + j] = 0.f;
    a.top_ids[n * a.top + j] = -1;
  }
}

// References that take the fused product: its rounding stays below 2^-4, and what stands for -inf
// keeps a weight of 0.
template <typename T> __device__ __forceinline__ float widest(float c) {
  if (!(c >= 1e-20f && c <= 1e8f)) return -1.f;
  return fminf(kWide, -Word<T>::kLow * c + kEmpty - kSlack);
}

// A cluster of CTAs per row, an equal run of its vectors each (one CTA for many rows). A vector is two
// 16-byte pieces half a warp's kilobyte apart, so that each copy of a warp is one run of memory.
//
// One pass over the logits. For the alternatives each thread also keeps the largest entry of each
// of kRuns runs of its vectors. A search over the threads' largest entries (a count over the CTA a
// step) finds a threshold that at least k of them reach and few more; the runs that reach it, and
// only those (about k kRuns' share of a thread each), are read again, and all their entries that
// reach it are ranked by (value, index). Those are all of the row's: so if they are k or more, the
// k first of them are the row's. If not (or if they are too many, or NaN is among the logits),
// k scans of the row find them, entry by entry. That costs: with five finite logits a row and ten alternatives
// (a masked vocabulary) 3904 x 151680 bf16 take 6.6 ms and 4 x 151644 fp32 73 us; ties that fill more than
// kRunList runs (3904 x 32000 whole numbers) 0.93 ms instead of 70 us. In a cluster it is the run of a CTA that
// has to hold k finite logits.
//
// 3904 x 151680 bf16 with ten alternatives takes 205 to 243 us, from GPU to GPU (0.75 to 0.9 of the copy
// bandwidth measured on one), 179 to 201 without (0.9 or more): an exponential and the products around it keep
// the issue slots two thirds busy, and what follows a row's last logit is hidden by the SM's other CTAs in part
// only. 4 x 151644 fp32: 12.3 us, 8.3 to 9.1 without alternatives.
constexpr int kRuns = 8, kRunList = 128;

template <typename T, int THREADS, bool TOP>
__global__ void __launch_bounds__(THREADS, 1024 / THREADS) token_logprobs_kernel(ScoreArgs a) {
  constexpr int WARPS = THREADS / 32, P = 16 / sizeof(T), AHEAD = 4;  // P: entries of a piece
  // bits of the order that every logit of the type has alike
  constexpr int SHIFT = sizeof(T) == 4 ? 0 : Word<T>::kLow == -65504.f ? 13 : 16;
  __shared__ uint4 s_ring[AHEAD][2][THREADS];
  __shared__ float s_r[WARPS], s_most[WARPS], s_s[WARPS], s_t[WARPS], s_part[3];
  __shared__ int s_bad, s_count, s_runs;
  __shared__ float s_run[TOP ? kRuns : 1][TOP ? THREADS : 1];
  __shared__ int s_runlist[TOP ? kRunList : 1];
  __shared__ unsigned long long s_list[TOP ? THREADS : 1], s_result[TOP ? SPECKV_MAX_TOP : 1], s_best;
  const uint32_t ctas = cluster_size(), rank = cluster_rank();
  const long long n = blockIdx.x / ctas;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, vocab = (int)a.vocab;
  long long offset = 0, token = -1;
  if (!score_row(a, n, offset, token)) {
    if (rank == 0) write_skipped(a, n);
    return;  // every CTA of the cluster returns here
  }
  const T* x = static_cast<const T*>(a.logits) + offset;
  const float given = tid == 0 && token >= 0 ? load_f<T>(x[token]) : 0.f;
  const RowSplit<16> row(x, vocab, sizeof(T));
  const int blocks = (row.pieces + 63) / 64;  // 32 vectors each, the last one perhaps in part
  const int lo = 32 * (int)((long long)blocks * rank / ctas), hi = 32 * (int)((long long)blocks * (rank + 1) / ctas);
  const int own = (hi - lo + THREADS - 1) / THREADS, run = max(1, (own + kRuns - 1) / kRuns);  // vectors of a thread, of a run
  const T* pieces = x + row.head;
  auto no_second = [](Bytes32& v) {
    v.w[4] = v.w[5] = v.w[6] = v.w[7] = Word<T>::kNone;
  };
  auto piece_of = [](int i, int h) { return (i >> 5) * 64 + h * 32 + (i & 31); };
  const float c = a.inv_t * kLog2e, wide_at = widest<T>(c);
  if (tid == 0) s_bad = s_count = s_runs = 0;

  Running<T> w;
  float best = -INFINITY, most = -INFINITY;  // of the run, of the thread
  int run_at = 0;                            // the run
  auto single = [&](int i) {
    const float v = load_f<T>(x[i]);
    w.single(v, c, wide_at);
    best = fmaxf(best, v);
  };
  if (rank == 0 && tid < row.head) single(tid);
  {
    // Each thread's vectors pass through its own slots of shared memory, AHEAD of them under way: no
    // registers wait for memory, and no thread waits for another.
    auto fetch = [&](int u, int i) {
      if (i < hi) {
#pragma unroll
        for (int h = 0; h < 2; ++h)
          if (piece_of(i, h) < row.pieces) copy_async(&s_ring[u][h][tid], pieces + (long long)piece_of(i, h) * P);
      }
      asm volatile("cp.async.commit_group;" ::: "memory");
    };
    int i = lo + tid, end = run;
#pragma unroll
    for (int u = 0; u < AHEAD; ++u) fetch(u, i + u * THREADS);
    for (int j = 0; j < own; j += AHEAD, i += AHEAD * THREADS)
#pragma unroll
      for (int u = 0; u < AHEAD; ++u) {
        if (TOP && j + u == end && end < own) {
          s_run[run_at++][tid] = best;
          most = fmaxf(most, best);
          best = -INFINITY;
          end += run;
        }
        asm volatile("cp.async.wait_group %0;" ::"n"(AHEAD - 1) : "memory");
        const int at = i + u * THREADS;
        if (at < hi && piece_of(at, 0) < row.pieces) {
          Bytes32 v = from_pieces(s_ring[u][0][tid], s_ring[u][1][tid]);
          if (piece_of(at, 1) >= row.pieces) no_second(v);
          const float top = vector_top<T>(v);
          fetch(u, at + AHEAD * THREADS);
          if (TOP) best = fmaxf(best, top);
          w.vector(v, top, c, wide_at);
        }
      }
  }
  if (rank == ctas - 1 && tid < row.tail) single(row.head + row.pieces * P + tid);
  if (TOP) {
    s_run[run_at][tid] = best;
    most = fmaxf(most, best);
  }

  // sums of the CTA, by its largest reference
  float s, t, r = w.r, peak = most;
  w.finish(c, s, t);
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) {
    r = fmaxf(r, __shfl_xor_sync(0xffffffffu, r, off));
    if (TOP) peak = fmaxf(peak, __shfl_xor_sync(0xffffffffu, peak, off));
  }
  if (lane == 0) {
    s_r[warp] = r;
    s_most[warp] = peak;
  }
  __syncthreads();
  if (w.bad) s_bad = 1;
#pragma unroll
  for (int v = 0; v < WARPS; ++v) {
    r = fmaxf(r, s_r[v]);
    if (TOP) peak = fmaxf(peak, s_most[v]);
  }
  {
    const float d = fmaxf((w.r - r) * c, kEmpty), f = exp2_fast(d);  // no entry above -inf: s = t = 0
    t = f * fmaf(d, s, t);
    s *= f;
  }
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) {
    s += __shfl_xor_sync(0xffffffffu, s, off);
    t += __shfl_xor_sync(0xffffffffu, t, off);
  }
  if (lane == 0) {
    s_s[warp] = s;
    s_t[warp] = t;
  }
  if (TOP) {
    const int k = a.top;
    const uint32_t mine = order_key(most) >> SHIFT, first = order_key(peak) >> SHIFT;
    // down from the largest entry in growing steps, then halving: k to k + 6 threads
    uint32_t above = first + 1, level = first, step = 1u << (19 - SHIFT);
    int reach = 0;
    for (;;) {
      level = first > step ? first - step : 0u;
      reach = __syncthreads_count(mine >= level);
      if (reach >= k || level == 0u) break;
      above = level;
      step *= 4u;
      if (step >= (1u << 30)) step = 0xffffffffu;
    }
    while (reach > k + 6 && above - level > 1u) {
      const uint32_t middle = level + (above - level) / 2;
      const int count = __syncthreads_count(mine >= middle);
      if (count >= k) {
        level = middle;
        reach = count;
      } else {
        above = middle;
      }
    }
    if (mine >= level)
      for (int i = 0; i <= run_at; ++i)
        if (order_key(s_run[i][tid]) >> SHIFT >= level) {
          const int place = atomicAdd(&s_runs, 1);
          if (place < kRunList) s_runlist[place] = i << 16 | tid;
        }
    if (tid < SPECKV_MAX_TOP) s_result[tid] = 0ull;
    __syncthreads();
    const int runs = s_runs;
    auto key_of = [](float v, int i) { return (unsigned long long)order_key(v) << 32 | (0xffffffffu - (uint32_t)i); };
    auto keep = [&](float v, int i) {
      if (order_key(v) >> SHIFT >= level) {
        const int place = atomicAdd(&s_count, 1);
        if (place < THREADS) s_list[place] = key_of(v, i);
      }
    };
    if (runs <= kRunList) {
      for (int item = tid; item < runs * run; item += THREADS) {
        const int entry = s_runlist[item / run], part = item % run, owner = entry & 0xffff, number = entry >> 16;
        if (part == 0 && number == 0 && rank == 0 && owner < row.head) keep(load_f<T>(x[owner]), owner);
        if (part == 0 && number == run_at && rank == ctas - 1 && owner < row.tail) {
          const int i = row.head + row.pieces * P + owner;
          keep(load_f<T>(x[i]), i);
        }
        const int i = lo + owner + (number * run + part) * THREADS;
        if (i < hi && piece_of(i, 0) < row.pieces) {
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const int piece = piece_of(i, h);
            if (piece < row.pieces) {
              const uint4 raw = __ldg(reinterpret_cast<const uint4*>(pieces + (long long)piece * P));
              const Bytes32 v{{raw.x, raw.y, raw.z, raw.w}};
#pragma unroll
              for (int e = 0; e < P / 2; ++e) {
                float f0, f1;
                pair_values<T>(v, e, false, f0, f1);
                keep(f0, row.head + piece * P + 2 * e);
                keep(f1, row.head + piece * P + 2 * e + 1);
              }
            }
          }
        }
      }
    }
    __syncthreads();
    const int count = s_count;
    if (!s_bad && runs <= kRunList && count >= k && count <= THREADS) {
      if (tid < count) {
        const unsigned long long key = s_list[tid];
        int before = 0;
        for (int i = 0; i < count; ++i) before += s_list[i] > key;
        if (before < k) s_result[before] = key;
      }
    } else {
      unsigned long long last = ~0ull;
      for (int j = 0; j < k; ++j) {
        __syncthreads();
        if (tid == 0) s_best = 0ull;
        __syncthreads();
        unsigned long long found = 0ull;
        auto scan = [&](int i) {
          const unsigned long long key = key_of(load_f<T>(x[i]), i);
          if (key < last && key > found) found = key;
        };
        if (rank == 0 && tid < row.head) scan(tid);
        for (int i = lo * 2 * P + tid; i < min(hi * 2, row.pieces) * P; i += THREADS) scan(row.head + i);
        if (rank == ctas - 1 && tid < row.tail) scan(row.head + row.pieces * P + tid);
        if (found) atomicMax(&s_best, found);
        __syncthreads();
        last = s_best;
        if (tid == 0) s_result[j] = last;
        if (last == 0ull) break;
      }
    }
  }
  __syncthreads();
  bool bad = s_bad;
  s = t = 0.f;
#pragma unroll
  for (int v = 0; v < WARPS; ++v) {
    s += s_s[v];
    t += s_t[v];
  }
  if (ctas > 1) {
    if (tid == 0) {
      s_part[0] = r;
      s_part[1] = s;
      s_part[2] = t;
    }
    cluster_sync();
    if (rank == 0) {
      float r2[8], s2[8], t2[8];
      int bad2[8];
#pragma unroll
      for (uint32_t o = 1; o < 8; ++o)
        if (o < ctas) {
          r2[o] = remote_float(&s_part[0], o);
          s2[o] = remote_float(&s_part[1], o);
          t2[o] = remote_float(&s_part[2], o);
          bad2[o] = __float_as_int(remote_float(&s_bad, o));
        }
#pragma unroll
      for (uint32_t o = 1; o < 8; ++o)
        if (o < ctas) {
          join_sums(r, s, t, r2[o], s2[o], t2[o], c);
          bad |= bad2[o] != 0;
        }
    }
  }
  if (rank == 0) {
    const float log_s = log2f(s);
    const bool empty = r == -INFINITY && !bad;
    auto logprob = [&](float v) { return bad ? NAN : empty ? -INFINITY : (v - r) * a.inv_t - log_s * kLn2; };
    if (tid == 0) {
      if (a.logprobs != nullptr) a.logprobs[n] = logprob(given);
      a.entropy[n] = bad ? NAN : empty ? 0.f : fmaxf(log_s - t / s, 0.f) * kLn2;
      if (a.stats != nullptr) {
        a.stats[2 * n] = bad ? NAN : r;
        a.stats[2 * n + 1] = bad ? NAN : empty ? -INFINITY : log_s;
      }
    }
    if (TOP) {
      const int k = a.top;
      auto emit = [&](int place, unsigned long long key) {
        const long long at = n * k + place;
        a.top_ids[at] = 0xffffffffu - (uint32_t)key;
        a.top_logprobs[at] = logprob(order_value((uint32_t)(key >> 32)));
      };
      if (ctas == 1) {
        if (tid < k) emit(tid, s_result[tid]);
      } else {
        // the CTAs' alternatives, ranked
        const int all = (int)ctas * k;
        if (tid < all) s_list[tid] = remote_u64(&s_result[tid % k], tid / k);
        __syncthreads();
        if (tid < all) {
          const unsigned long long key = s_list[tid];
          int before = 0;
          for (int o = 0; o < all; ++o) before += s_list[o] > key;
          if (key != 0ull && before < k) emit(before, key);
        }
      }
    }
  }
  if (ctas > 1) cluster_sync();  // the other CTAs' shared memory is read until here
}

constexpr int kGradThreads = 256;
constexpr int kGradSpan = 4;  // 32-byte vectors a thread handles

// CTA per (row, run of vectors). One exponential and one product chain an entry:
//   dx = p (u + v y) with y = log2 p, p = 2^y, u = -(sum of gradients + g_H H) / T,
//   v = -g_H ln(2) / T; the token and the alternatives add their own gradient afterwards.
// Bound by memory: forward and gradient of 4096 x 151644 bf16 take 559 to 608 us (0.9 to 0.98 of the
// copy bandwidth measured on one GPU), of 1024 x 151644 fp32 297 us (0.97).
template <typename T>
__global__ void __launch_bounds__(kGradThreads) token_logprobs_backward_kernel(ScoreArgs a, int runs) {
  constexpr int N = 32 / sizeof(T);
  const long long n = blockIdx.x / runs;
  const int part = (int)(blockIdx.x - n * runs), tid = threadIdx.x, vocab = (int)a.vocab;
  T* g = static_cast<T*>(a.grad) + n * a.vocab;
  const RowSplit<32> row(g, vocab, sizeof(T));
  const int lo = part * kGradThreads * kGradSpan, hi = min(row.pieces, lo + kGradThreads * kGradSpan);
  const int e_lo = part == 0 ? 0 : row.head + lo * N, e_hi = part == runs - 1 ? vocab : row.head + hi * N;
  long long offset = 0, token = -1;
  if (!score_row(a, n, offset, token) || a.stats[2 * n] == -INFINITY) {
    const Bytes32 zero{};
    for (int i = lo + tid; i < hi; i += kGradThreads) store_stream(g + row.head + (long long)i * N, zero);
    if (part == 0 && tid < row.head) g[tid] = store_f<T>(0.f);
    if (part == runs - 1 && tid < row.tail) g[row.head + row.pieces * N + tid] = store_f<T>(0.f);
    return;
  }
  const T* x = static_cast<const T*>(a.logits) + offset;
  // The gradient's vectors are aligned; the logits' lie alike, or (a view such as logits[:, :-1]) only
  // their words do, or (of an odd offset) lie across two words each: 1024 x 151643 bf16 in a pitch of
  // 151644 with its forward 189 to 209 us, 164 to 190 where they lie alike, 546 entry by entry.
  const uintptr_t apart = (reinterpret_cast<uintptr_t>(x) ^ reinterpret_cast<uintptr_t>(g)) & 31;
  Bytes32 in[kGradSpan];
#pragma unroll
  for (int k = 0; k < kGradSpan; ++k) {
    const int i = lo + tid + k * kGradThreads;
    if (i < hi) {
      const T* from = x + row.head + (long long)i * N;
      if (apart == 0) {
        in[k] = load_stream(from);
      } else if ((apart & 3) == 0) {
#pragma unroll
        for (int e = 0; e < 8; ++e) in[k].w[e] = __ldg(reinterpret_cast<const uint32_t*>(from) + e);
      } else if constexpr (sizeof(T) == 2) {
        const unsigned short* half = reinterpret_cast<const unsigned short*>(from);
        uint32_t before = (uint32_t)__ldg(half) << 16;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const uint32_t w = e < 7 ? __ldg(reinterpret_cast<const uint32_t*>(half + 1) + e) : __ldg(half + 15);
          in[k].w[e] = __funnelshift_r(before, w, 16);
          before = w;
        }
      }
    }
  }
  const float ga = a.g_logprobs != nullptr ? a.g_logprobs[n] : 0.f;
  const float gh = a.g_entropy != nullptr ? a.g_entropy[n] : 0.f;
  float all = ga;
  if (a.g_top != nullptr)
    for (int j = 0; j < a.top; ++j) all += a.g_top[n * a.top + j];
  const float c = a.inv_t * kLog2e, r = a.stats[2 * n], log_s = a.stats[2 * n + 1];
  const float u = -a.inv_t * (all + gh * a.entropy[n]), v = -a.inv_t * gh * kLn2;  // NaN rows: u is NaN
  auto slope = [&](float z) {
    const float y = fmaxf(fmaf(z - r, c, -log_s), kEmpty);  // -inf: weight 0, not 0 x inf
    return exp2_fast(y) * fmaf(v, y, u);
  };
#pragma unroll
  for (int k = 0; k < kGradSpan; ++k) {
    const int i = lo + tid + k * kGradThreads;
    if (i < hi) {
      Bytes32 out;
#pragma unroll
      for (int e = 0; e < N / 2; ++e) {
        float x0, x1, y0, y1;
        pair_values<T>(in[k], e, false, x0, x1);
        parts(fma2(add2(two(x0, x1), two(-r, -r)), two(c, c), two(-log_s, -log_s)), y0, y1);
        y0 = fmaxf(y0, kEmpty);
        y1 = fmaxf(y1, kEmpty);
        parts(mul2(two(exp2_fast(y0), exp2_fast(y1)), fma2(two(v, v), two(y0, y1), two(u, u))), x0, x1);
        if constexpr (sizeof(T) == 4) {
          out.w[2 * e] = __float_as_uint(x0);
          out.w[2 * e + 1] = __float_as_uint(x1);
        } else {
          out.w[e] = Word<T>::pack(x0, x1);
        }
      }
      store_stream(g + row.head + (long long)i * N, out);
    }
  }
  if (part == 0 && tid < row.head) g[tid] = store_f<T>(slope(load_f<T>(x[tid])));
  if (part == runs - 1 && tid < row.tail) {
    const int i = row.head + row.pieces * N + tid;
    g[i] = store_f<T>(slope(load_f<T>(x[i])));
  }
  // the entries that have a gradient of their own, each written once more, whole
  const int extra = a.g_top != nullptr ? a.top : 0;
  if (extra == 0 && ga == 0.f) return;
  __syncthreads();
  for (int j = tid; j <= extra; j += kGradThreads) {
    long long id = token;
    float own = ga;
    if (j < extra) {
      id = a.top_ids[n * a.top + j];
      own = a.g_top[n * a.top + j] + (id == token ? ga : 0.f);
    } else {
      for (int k = 0; k < extra; ++k)
        if (a.top_ids[n * a.top + k] == token) id = -1;  // counted with that alternative
    }
    if (id >= e_lo && id < e_hi) g[id] = store_f<T>(fmaf(own, a.inv_t, slope(load_f<T>(x[id]))));
  }
}

template <typename T, int THREADS, bool TOP>
int launch_scores_as(const char* fn, const ScoreArgs& a, int ctas, cudaStream_t s) {
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = ctas;
  attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(a.batch * a.per * ctas));
  cfg.blockDim = dim3(THREADS);
  cfg.stream = s;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, token_logprobs_kernel<T, THREADS, TOP>, a);
  if (e != cudaSuccess) return fail(SPECKV_ECUDA, "%s: launch failed: %s", fn, cudaGetErrorString(e));
  return SPECKV_OK;
}

template <typename T>
int launch_scores(const char* fn, const ScoreArgs& a, cudaStream_t s) {
  const long long rows = a.batch * a.per, vectors = a.vocab * sizeof(T) / 32;
  const int sms = sm_count();
  if (sms == 0) return fail(SPECKV_ECUDA, "%s: no SM count", fn);
  // A cluster per row while that makes no more than two CTAs an SM (four fit, but clusters do not pack:
  // 148 x 151680 bf16 18.6 to 20.0 us, 28.7 with twice the CTAs) and leaves each thread a vector.
  int ctas = 1;
  while (ctas < 8 && rows * ctas <= sms && vectors / (ctas * 2) >= 256) ctas *= 2;
  if (rows * ctas >= (1ll << 31)) return fail(SPECKV_ENOSUPPORT, "%s: too many rows", fn);
  // What follows a row's last logit takes a CTA 2 to 6 us: at vocabularies to 128 K entries of 16 bits
  // twice the CTAs of half the threads hide more of it (3904 x 32000 bf16, ten alternatives: 71 us
  // instead of 86), longer rows want the wider CTA (900 x 151644 fp32: 102 to 106 us, 123 with 128 threads).
  if (ctas == 1 && vectors <= 8192)
    return a.top > 0 ? launch_scores_as<T, 128, true>(fn, a, 1, s) : launch_scores_as<T, 128, false>(fn, a, 1, s);
  return a.top > 0 ? launch_scores_as<T, 256, true>(fn, a, ctas, s) : launch_scores_as<T, 256, false>(fn, a, ctas, s);
}

template <typename T>
int launch_gradient(const char* fn, const ScoreArgs& a, cudaStream_t s) {
  const long long vectors = a.vocab * (long long)sizeof(T) / 32, span = kGradThreads * kGradSpan;
  const long long runs = vectors <= span ? 1 : (vectors + span - 1) / span;
  if (a.batch * a.per * runs >= (1ll << 31)) return fail(SPECKV_ENOSUPPORT, "%s: too many rows", fn);
  token_logprobs_backward_kernel<T><<<(unsigned)(a.batch * a.per * runs), kGradThreads, 0, s>>>(a, (int)runs);
  return check_launch(fn);
}

int check_scores(const char* fn, const void* logits, int32_t dtype, const int64_t* tokens, int64_t batch, int64_t per,
                 int64_t source_rows, int64_t vocab, float inv_temperature, int32_t top) {
  if (batch < 0 || per < 0 || source_rows < 0 || vocab < 1) return fail(SPECKV_EINVAL, "%s: bad sizes", fn);
  if (dtype != SPECKV_F32 && dtype != SPECKV_BF16 && dtype != SPECKV_F16)
    return fail(SPECKV_EINVAL, "%s: unsupported dtype %d", fn, dtype);
  if (!(inv_temperature >= 1e-30f) || !(inv_temperature <= 1e30f))
    return fail(SPECKV_EINVAL, "%s: 1 / temperature must lie in [1e-30, 1e30]", fn);
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
                                     float inv_temperature, int32_t top, float* logprobs, float* entropy, float* stats,
                                     float* top_logprobs, int64_t* top_ids, void* stream) {
  const char* fn = "speckv_token_logprobs";
  int st = check_scores(fn, logits, dtype, tokens, batch, per_batch, source_rows, vocab, inv_temperature, top);
  if (st || batch == 0 || per_batch == 0) return st;
  if (rows == nullptr && source_rows != per_batch)
    return fail(SPECKV_EINVAL, "%s: %lld rows of logits for %lld", fn, (long long)source_rows, (long long)per_batch);
  if (logits == nullptr || entropy == nullptr || (tokens == nullptr) != (logprobs == nullptr) ||
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
  a.stats = stats;
  a.top_logprobs = top_logprobs;
  a.top_ids = top_ids;
  a.err = device_error_word();
  if (a.err == nullptr) return fail(SPECKV_ECUDA, "%s: no error word on device", fn);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  switch (dtype) {
    case SPECKV_F32: return launch_scores<float>(fn, a, s);
    case SPECKV_BF16: return launch_scores<__nv_bfloat16>(fn, a, s);
    default: return launch_scores<__half>(fn, a, s);
  }
}

extern "C" int speckv_token_logprobs_backward(const void* logits, int32_t dtype, int64_t stride_b, int64_t stride_r,
                                              const int64_t* tokens, int64_t tokens_stride_b, int64_t tokens_stride_r,
                                              int64_t batch, int64_t per_batch, int64_t vocab, float inv_temperature,
                                              int32_t top, const float* entropy, const float* stats,
                                              const int64_t* top_ids, const float* grad_logprobs,
                                              const float* grad_entropy, const float* grad_top_logprobs,
                                              void* grad_logits, void* stream) {
  const char* fn = "speckv_token_logprobs_backward";
  int st = check_scores(fn, logits, dtype, tokens, batch, per_batch, per_batch, vocab, inv_temperature, top);
  if (st || batch == 0 || per_batch == 0) return st;
  if (logits == nullptr || entropy == nullptr || stats == nullptr || grad_logits == nullptr ||
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
  a.stats = const_cast<float*>(stats);
  a.top_ids = const_cast<int64_t*>(top_ids);
  a.g_logprobs = grad_logprobs;
  a.g_entropy = grad_entropy;
  a.g_top = grad_top_logprobs;
  a.grad = grad_logits;
  a.err = device_error_word();
  if (a.err == nullptr) return fail(SPECKV_ECUDA, "%s: no error word on device", fn);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  switch (dtype) {
    case SPECKV_F32: return launch_gradient<float>(fn, a, s);
    case SPECKV_BF16: return launch_gradient<__nv_bfloat16>(fn, a, s);
    default: return launch_gradient<__half>(fn, a, s);
  }
}
