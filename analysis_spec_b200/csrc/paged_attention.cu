// Attention of one new token per sequence over a paged KV cache.
//
//   out[b][0][hq][:] = sum_c softmax_c(scale q[b][hq] . k_c) v_c,   c < lengths[b]
// with k_c / v_c the rows of KV head hq / g (g = q_heads / kv_heads) that the page table names.
// A sequence of length 0 gives zeros. Scores, softmax statistics and output sums in fp32.
#include "cluster.cuh"
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

// CTA per (sequence, query head), a key per warp and step: head dims and views off 16-byte boundaries. Reads
// the cache once per query head and waits for each key: 20 to 34 times the time of the kernels below (4000 keys of
// 8 / 1 heads x 128: 420 us in bf16, 414 in fp32).
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

// ---- tensor-core kernels: head dims to 64 / 128 / 256 ----------------------------------------------
//
// Scores are K q^T (16 keys x 8 heads per matrix instruction), outputs V^T p^T (16 dims x 8
// heads): the group's heads are the narrow side, so keys are never padded to 128 rows, as the
// tcgen05 shapes would want. At 2 to 8 flops a byte the tensor pipe is a tenth busy either way; what
// counts is the cache's bytes in flight, so every warp streams its own blocks of 16 keys and waits
// for no other warp until an item ends.

__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

__device__ __forceinline__ uint4 load_stream(const void* p) {
  uint4 r;
  asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];"
               : "=r"(r.x), "=r"(r.y), "=r"(r.z), "=r"(r.w)
               : "l"(p));
  return r;
}

// 16 bytes to shared memory; zeros when `live` is false (nothing is read then).
__device__ __forceinline__ void copy_row(uint32_t to, const void* from, bool live) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to), "l"(from), "r"(live ? 16 : 0) : "memory");
}

__device__ __forceinline__ void load_matrices(uint32_t at, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(at)
               : "memory");
}
__device__ __forceinline__ uint32_t load_word(uint32_t at) {
  uint32_t r;
  asm volatile("ld.shared.u32 %0, [%1];" : "=r"(r) : "r"(at) : "memory");
  return r;
}

__device__ __forceinline__ void mma(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                    uint32_t b1, __nv_bfloat16) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
               "{%0, %1, %2, %3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
               : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                    uint32_t b1, __half) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
               "{%0, %1, %2, %3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
               : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

__device__ __forceinline__ void mma_tf32(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
               "{%0, %1, %2, %3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// An fp32 number as two tf32 parts: hi is x rounded (off by 2^-11 of x at most), lo the rest, at most 12 bits,
// of which the product takes 11: x = hi + lo up to 2^-23 of x. The rounding is two whole-number instructions:
// cvt.rna, which shares a slower pipe, made 64 x 256..2048 49.9 us instead of 47.5. Numbers within 2^-12 of fp32's
// largest round to infinity, and what is infinite has no rest (NaN).
__device__ __forceinline__ void split(uint32_t x, uint32_t& hi, uint32_t& lo) {
  hi = (x + 0x1000u) & 0xffffe000u;
  lo = __float_as_uint(__uint_as_float(x) - __uint_as_float(hi));
}
// The same, not moved out of its loop: the parts of all queries would not fit the registers.
__device__ __forceinline__ void split_here(uint32_t x, uint32_t& hi, uint32_t& lo) {
  asm volatile("{\n\t.reg .u32 r;\n\tadd.u32 r, %1, 0x1000;\n\tand.b32 %0, r, 0xffffe000;\n\t}" : "=r"(hi) : "r"(x));
  lo = __float_as_uint(__uint_as_float(x) - __uint_as_float(hi));
}
__device__ __forceinline__ void split4(const uint32_t (&x)[4], uint32_t (&hi)[4], uint32_t (&lo)[4]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) split(x[i], hi[i], lo[i]);
}
// A product of fp32 operands is the three products above 2^-22: ah bh, and the small ones al bh + ah bl. The
// matrix instructions cut their sums toward zero, about 2^-24 of what they hold each time: sums kept in them over a
// sequence came out low by up to 2.5e-6. So sums of ah bh are kept there over a few instructions only and go on in
// rounded fp32 additions; the small products are 2^-11 of them, and so is what is cut from theirs.

// Transpose of an 8 x 8 matrix of 16-bit elements held as a matrix fragment.
__device__ __forceinline__ uint32_t transpose8(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}

// x and y as a pair of 16-bit values, and what that rounding left out as another.
__device__ __forceinline__ void split_pair(float x, float y, uint32_t& hi, uint32_t& lo, __nv_bfloat16) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(x, y);
  const __nv_bfloat162 l = __floats2bfloat162_rn(x - __low2float(h), y - __high2float(h));
  hi = *reinterpret_cast<const uint32_t*>(&h);
  lo = *reinterpret_cast<const uint32_t*>(&l);
}
__device__ __forceinline__ void split_pair(float x, float y, uint32_t& hi, uint32_t& lo, __half) {
  const __half2 h = __floats2half2_rn(x, y);
  const __half2 l = __floats2half2_rn(x - __low2float(h), y - __high2float(h));
  hi = *reinterpret_cast<const uint32_t*>(&h);
  lo = *reinterpret_cast<const uint32_t*>(&l);
}

// 4 x 12000 keys, 16 q / 2 KV heads: 18.1 us at one tile and at two (half the parts), 20.3 at six.
constexpr int kMinTiles = 2;         // a CTA's share is at least this many tiles
constexpr int kCluster = 8;          // CTAs of a cluster at most
// One launch beats two where the work is small (1 x 200 keys 8.3 us, 12.8 as shares) and still where a
// CTA has 11 tiles (64 x 256..2048 23.7 us, 24.0); at 21 uneven lengths cost more (64 x 256..4000 37.9, 33.7).
constexpr int kClusterTiles = 12;    // tiles of a cluster's CTA at most

// Weights are 2^(score - reference). The reference need not be the maximum: any value near it keeps the
// weights and sums well inside fp32, and the sums are divided by the total at the end. So it moves only
// when a score passes it by more than kSlack, to kLow below that score. fp16 weights enter the
// tensor cores in two parts above the type's smallest step, 2^-24: they are taken near the type's upper
// end, 2^11 to 2^15, and what a weight loses is 2^-36 of the largest (2^-25 at a reference of the maximum:
// 5000 keys of weight 2^-26 beside one of 1 came out 1.6 % low). bf16 and tf32 parts have fp32's range.
template <typename T> struct Reference {
  static constexpr float kLow = 0.f, kSlack = 8.f;
};
template <> struct Reference<__half> {
  static constexpr float kLow = 11.f, kSlack = 15.f;
};

// Warps of a CTA, CTAs per SM (by registers in 16 bits, by the rings in fp32) and shared memory. WIDE:
// 16 bits, twice the warps.
template <typename T, int D, int NT, bool WIDE = false> struct Shape {
  static constexpr bool kHalf = sizeof(T) == 2;
  static constexpr int kRow = D * (int)sizeof(T);      // bytes of a key row
  static constexpr int kStages = 3;                    // fp32: blocks of K or V under way per warp
  static constexpr int kWarps = (kHalf && !WIDE) || (!kHalf && D == 256) ? 4 : 8;
  static constexpr int kRing = kHalf ? 0 : kWarps * kStages * 16 * kRow;
  static constexpr int kSums = kWarps * 8 * (D + 4) * 4;
  static constexpr int kShared = kRing > kSums ? kRing : kSums;
  static constexpr int kResident = WIDE ? 1 : !kHalf ? (D == 64 ? 2 : 1)
                                   : D == 64 ? (NT == 1 ? 4 : 3) : D == 128 && NT == 1 ? 3 : 2;
  static constexpr int kTile = 16 * kWarps;            // keys of a tile: a block a warp
};

// An item is (sequence, KV head, up to 8 NT of its query heads). All items' tiles, in order, are
// cut into equal shares, one per CTA; a share that begins or ends inside an item leaves its part
// of that item in the workspace, and the CTA in whose share the item begins describes it for
// the join.
struct Join {
  int b, h, slot, count;  // count 0: nothing to join; parts at `slot` of share slot / 2, then at slot 0 of each next share
};

struct PlanArgs {
  float* parts;   // (2 * CTAs) x [8 NT][dim + 2]: sums, reference, total
  Join* joins;    // one per item where there are fewer items than CTAs (by_item), else one per CTA
  int chunks;     // items per (sequence, KV head)
  int by_item;
};

// What a CTA's warps leave of an item, beside their sums.
template <int W, int NT> struct Parts {
  float m[W][8 * NT], l[W][8 * NT];
  float top[8 * NT], all[8 * NT];  // of all warps
};

// Four outputs: sums over their total, zeros where there is nothing to see.
template <typename T> __device__ __forceinline__ void store_four(T* to, const float4& sum, float all) {
  const float x[4] = {sum.x, sum.y, sum.z, sum.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) to[i] = store_f<T>(all == 0.f ? 0.f : x[i] / all);
}

// Joins the warps' parts of an item: own(u, e, f, to) writes the lane's sums of head 8 u + 2 t + e,
// times f, to that head's row; emit(head of the item, dim, sums of four dims, reference, total) gets
// the outcome.
template <int D, int NT, int W, typename Own, typename Emit>
__device__ __forceinline__ void join_warps(unsigned char* shared, Parts<W, NT>& sm, float (&m)[NT][2], float (&l)[NT][2],
                                           int heads, Own own, Emit emit) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
#pragma unroll
  for (int u = 0; u < NT; ++u)
#pragma unroll
    for (int e = 0; e < 2; ++e) {
#pragma unroll
      for (int off = 4; off < 32; off <<= 1) l[u][e] += __shfl_xor_sync(0xffffffffu, l[u][e], off);
      if (g == 0) {
        sm.m[warp][u * 8 + 2 * t + e] = m[u][e];
        sm.l[warp][u * 8 + 2 * t + e] = l[u][e];
      }
    }
  __syncthreads();  // the rings, over which the sums lie, are idle from here on
  float(*sums)[8][D + 4] = reinterpret_cast<float(*)[8][D + 4]>(shared);  // [W]
  if (threadIdx.x < 8 * NT) {
    const int head = threadIdx.x;
    float top = sm.m[0][head], all = 0.f;
#pragma unroll
    for (int w = 1; w < W; ++w) top = fmaxf(top, sm.m[w][head]);
    const float ref = top == -INFINITY ? 0.f : top;
#pragma unroll
    for (int w = 0; w < W; ++w) all = fmaf(sm.l[w][head], exp2f(sm.m[w][head] - ref), all);
    sm.top[head] = top;
    sm.all[head] = all;
  }
#pragma unroll
  for (int u = 0; u < NT; ++u) {
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int head = u * 8 + 2 * t + e;
      float top = sm.m[0][head];
#pragma unroll
      for (int w = 1; w < W; ++w) top = fmaxf(top, sm.m[w][head]);
      const float f = top == -INFINITY ? 1.f : exp2f(m[u][e] - top);
      own(u, e, f, sums[warp][2 * t + e]);
    }
    __syncthreads();
    for (int i = threadIdx.x; i < 2 * D; i += W * 32) {  // four dims each
      const int head = 4 * i / D, d = 4 * i - head * D;
      if (u * 8 + head >= heads) break;
      float4 sum = *reinterpret_cast<const float4*>(&sums[0][head][d]);
#pragma unroll
      for (int w = 1; w < W; ++w) {
        const float4 more = *reinterpret_cast<const float4*>(&sums[w][head][d]);
        sum.x += more.x, sum.y += more.y, sum.z += more.z, sum.w += more.w;
      }
      emit(u * 8 + head, d, sum, sm.top[u * 8 + head], sm.all[u * 8 + head]);
    }
    __syncthreads();
  }
}

// 16-bit caches. Operands come straight from memory into registers: the dims of a product may be
// taken in any order, so a lane's 16-byte chunks of its key rows are its fragments as they are, and
// two keys' chunks of V give theirs by byte permutes. 8 KB a warp are under way, 12 warps on an SM.
// (Copied ahead through shared memory instead, 8 warps, 256 x 512..6144 took 293 us, 275 so.)
// WHOLE: pages hold a multiple of 16 positions, so that a block lies in one, and the head dim is D. Else
// each row is looked up by itself and cut to its dims (256 x 512..6144, 28 / 4 heads, fp16: pages of 24
// positions 358 us, dim 96 349 us, 273 us where WHOLE holds).
// One CTA's part of an item: tiles [t0, ...) of its keys up to position `end`.
template <typename T, int D, int NT, bool WHOLE, bool WIDE, typename Emit>
__device__ __forceinline__ void attend_part16(const PagedArgs& a, unsigned char* shared,
                                              Parts<Shape<T, D, NT, WIDE>::kWarps, NT>& sm, long long b, int hk, int h0,
                                              int heads, int t0, long long end, Emit emit) {
  typedef Shape<T, D, NT, WIDE> S;
  typedef Reference<T> R;
  constexpr int KC = D / 32;  // 16-byte chunks of a key row per lane
  constexpr int VC = D / 64;  // 16-byte chunks of a value row per lane
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const long long group = a.q_heads / a.kv_heads;
  const T* kbase = static_cast<const T*>(a.k) + hk * a.ks[1];
  const T* vbase = static_cast<const T*>(a.v) + hk * a.vs[1];
  const uint32_t P = (uint32_t)a.table.page_size;
  const int dim = WHOLE ? D : (int)a.dim;  // dims from there to D are zeros, not read

  uint4 kreg[2][KC], vreg[4][VC];
  // block i of this warp: keys [16 (W t0 + warp + W i), + 16)
  const long long key0 = (long long)t0 * S::kTile + warp * 16;
  const int count = key0 < end ? (int)((end - key0 + S::kTile - 1) / S::kTile) : 0;
  // this lane's first row and chunk of a block: key rows g and g + 8, value rows 2t, 2t + 1, 2t + 8, 2t + 9
  const T* klane = kbase + g * a.ks[2] + t * 8;
  const T* vlane = vbase + 2 * t * a.vs[2] + g * 8;

  // A block lies in one page (WHOLE). Each lane finds the place of one block in 32.
  long long k_places = -1, v_places = -1, k_at = -1, v_at = -1;  // element offsets; -1: no such block or page
  int live = 0;  // keys of the block being loaded
  uint32_t seen = 0;  // bit 0 / 1: key rows g and g + 8 of the block in kreg are live
  auto place = [&](int i) {
    if (WHOLE) {
      if ((i & 31) == 0) {
        const long long key = key0 + (long long)(i + lane) * S::kTile;
        k_places = v_places = -1;
        if (key < end) {
          const uint32_t index = (uint32_t)key / P, row = (uint32_t)key - index * P;
          const long long page = a.table.page(b, index, a.err);
          if (page >= 0) {
            k_places = page * a.ks[0] + row * a.ks[2];
            v_places = page * a.vs[0] + row * a.vs[2];
          }
        }
      }
      k_at = __shfl_sync(0xffffffffu, k_places, i & 31);
      v_at = __shfl_sync(0xffffffffu, v_places, i & 31);
      live = k_at < 0 ? 0 : (int)min(16ll, end - key0 - (long long)i * S::kTile);
    }
  };
  auto row_ptr = [&](const T* from, const long long* st, long long key) -> const T* {
    if (key >= end) return nullptr;
    const uint32_t index = (uint32_t)key / P;
    const long long p = a.table.page(b, index, a.err);
    return p < 0 ? nullptr : from + p * st[0] + (long long)((uint32_t)key - index * P) * st[2];
  };
  auto load_k = [&](int i) {
    if (WHOLE && live == 16) {
      const T* p = klane + k_at;
#pragma unroll
      for (int j = 0; j < KC; ++j) {
        kreg[0][j] = load_stream(p + 32 * j);
        kreg[1][j] = load_stream(p + 8 * a.ks[2] + 32 * j);
      }
      seen = 3u;
      return;
    }
    const long long key = key0 + (long long)i * S::kTile;
    const T* p[2];
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      if (WHOLE)
        p[x] = g + 8 * x < live ? klane + k_at + 8 * x * a.ks[2] : nullptr;
      else
        p[x] = row_ptr(kbase + t * 8, a.ks, key + g + 8 * x);
#pragma unroll
      for (int j = 0; j < KC; ++j)
        kreg[x][j] = p[x] != nullptr && (WHOLE || t * 8 + 32 * j < dim) ? load_stream(p[x] + 32 * j) : make_uint4(0, 0, 0, 0);
    }
    seen = (p[0] != nullptr ? 1u : 0u) | (p[1] != nullptr ? 2u : 0u);
  };
  auto load_v = [&](int i) {
    if (WHOLE && live == 16) {
      const T* p = vlane + v_at;
#pragma unroll
      for (int x = 0; x < 4; ++x)
#pragma unroll
        for (int c = 0; c < VC; ++c) vreg[x][c] = load_stream(p + ((x & 1) + (x >> 1) * 8) * a.vs[2] + 64 * c);
      return;
    }
    const long long key = key0 + (long long)i * S::kTile;
#pragma unroll
    for (int x = 0; x < 4; ++x) {
      const int k = 2 * t + (x & 1) + (x >> 1) * 8;
      const T* p;
      if (WHOLE)
        p = k < live ? vlane + v_at + ((x & 1) + (x >> 1) * 8) * a.vs[2] : nullptr;
      else
        p = row_ptr(vbase + g * 8, a.vs, key + k);
      // rows that are not there may hold anything: 0 x NaN is NaN
#pragma unroll
      for (int c = 0; c < VC; ++c)
        vreg[x][c] = p != nullptr && (WHOLE || g * 8 + 64 * c < dim) ? load_stream(p + 64 * c) : make_uint4(0, 0, 0, 0);
    }
  };

  if (count > 0) {
    place(0);
    load_k(0);
    load_v(0);
  }
  // queries as the second operand: lane (g, t) holds head g, the same dims as its key chunks
  uint4 q[NT][KC];
#pragma unroll
  for (int u = 0; u < NT; ++u)
#pragma unroll
    for (int j = 0; j < KC; ++j) {
      q[u][j] = make_uint4(0, 0, 0, 0);
      if (u * 8 + g < heads && (WHOLE || (t + 4 * j) * 8 < dim)) {
        const T* p = static_cast<const T*>(a.q) + b * a.qs[0] + (hk * group + h0 + u * 8 + g) * a.qs[1] +
                     (t + 4 * j) * 8;
        q[u][j] = *reinterpret_cast<const uint4*>(p);
      }
    }
  float o[NT][VC][4][4], m[NT][2], l[NT][2];
#pragma unroll
  for (int u = 0; u < NT; ++u) {
#pragma unroll
    for (int c = 0; c < VC; ++c)
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[u][c][i][e] = 0.f;
    m[u][0] = m[u][1] = -INFINITY;
    l[u][0] = l[u][1] = 0.f;
  }

  for (int i = 0; i < count; ++i) {
    // scores of 16 keys x 8 heads: rows keys g, g + 8, columns heads 2t, 2t + 1
    float s[NT][4];
#pragma unroll
    for (int u = 0; u < NT; ++u) {
      float s2[4] = {0.f, 0.f, 0.f, 0.f};
      s[u][0] = s[u][1] = s[u][2] = s[u][3] = 0.f;
#pragma unroll
      for (int j = 0; j < KC; ++j) {
        mma(s[u], kreg[0][j].x, kreg[1][j].x, kreg[0][j].y, kreg[1][j].y, q[u][j].x, q[u][j].y, T());
        mma(s2, kreg[0][j].z, kreg[1][j].z, kreg[0][j].w, kreg[1][j].w, q[u][j].z, q[u][j].w, T());
      }
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        s[u][e] = (s[u][e] + s2[e]) * a.scale_log2;
        if (!(seen >> (e >> 1) & 1u)) s[u][e] = -INFINITY;
      }
    }
    if (i + 1 < count) {
      place(i + 1);
      load_k(i + 1);
    }
    uint32_t ph[NT][2], pl[NT][2];
#pragma unroll
    for (int u = 0; u < NT; ++u) {
      float t0m = fmaxf(s[u][0], s[u][2]), t1m = fmaxf(s[u][1], s[u][3]);
      if (__any_sync(0xffffffffu, t0m > m[u][0] + R::kSlack || t1m > m[u][1] + R::kSlack)) {  // the first block, from -inf
#pragma unroll
        for (int off = 4; off < 32; off <<= 1) {
          t0m = fmaxf(t0m, __shfl_xor_sync(0xffffffffu, t0m, off));
          t1m = fmaxf(t1m, __shfl_xor_sync(0xffffffffu, t1m, off));
        }
        const float n0 = fmaxf(m[u][0], t0m - R::kLow), n1 = fmaxf(m[u][1], t1m - R::kLow);
        const float f0 = n0 == -INFINITY ? 1.f : exp2f(m[u][0] - n0);
        const float f1 = n1 == -INFINITY ? 1.f : exp2f(m[u][1] - n1);
        m[u][0] = n0;
        m[u][1] = n1;
        l[u][0] *= f0;
        l[u][1] *= f1;
#pragma unroll
        for (int c = 0; c < VC; ++c)
#pragma unroll
          for (int x = 0; x < 4; ++x) {
            o[u][c][x][0] *= f0;
            o[u][c][x][1] *= f1;
            o[u][c][x][2] *= f0;
            o[u][c][x][3] *= f1;
          }
      }
      const float r0 = m[u][0] == -INFINITY ? 0.f : m[u][0], r1 = m[u][1] == -INFINITY ? 0.f : m[u][1];
      const float p0 = exp2_fast(s[u][0] - r0), p1 = exp2_fast(s[u][1] - r1), p2 = exp2_fast(s[u][2] - r0),
                  p3 = exp2_fast(s[u][3] - r1);
      l[u][0] += p0 + p2;
      l[u][1] += p1 + p3;
      // weights to (key pairs, heads) fragments, in two 16-bit parts: the tensor pipe has room
      // for a second product, and one of 8 bits alone would lose more than the output's rounding
      split_pair(p0, p1, ph[u][0], pl[u][0], T());
      split_pair(p2, p3, ph[u][1], pl[u][1], T());
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        ph[u][x] = transpose8(ph[u][x]);
        pl[u][x] = transpose8(pl[u][x]);
      }
    }
#pragma unroll
    for (int c = 0; c < VC; ++c)
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        const uint32_t v0 = (&vreg[0][c].x)[x], v1 = (&vreg[1][c].x)[x];
        const uint32_t v2 = (&vreg[2][c].x)[x], v3 = (&vreg[3][c].x)[x];
        // pairs of keys of one dim: dims 2x (row g) and 2x + 1 (row g + 8) of the lane's chunk
        const uint32_t a0 = __byte_perm(v0, v1, 0x5410), a1 = __byte_perm(v0, v1, 0x7632);
        const uint32_t a2 = __byte_perm(v2, v3, 0x5410), a3 = __byte_perm(v2, v3, 0x7632);
#pragma unroll
        for (int u = 0; u < NT; ++u) {
          mma(o[u][c][x], a0, a1, a2, a3, ph[u][0], ph[u][1], T());
          mma(o[u][c][x], a0, a1, a2, a3, pl[u][0], pl[u][1], T());
        }
      }
    if (i + 1 < count) load_v(i + 1);
  }

  join_warps<D, NT, S::kWarps>(shared, sm, m, l, heads, [&](int u, int e, float f, float* to) {
#pragma unroll
    for (int c = 0; c < VC; ++c)
#pragma unroll
      for (int x = 0; x < 4; ++x)
        *reinterpret_cast<float2*>(to + (g + 8 * c) * 8 + 2 * x) = make_float2(o[u][c][x][e] * f, o[u][c][x][2 + e] * f);
  }, emit);
}

// fp32 caches. Twice the bytes a key and six instructions a product: K and V rows are copied ahead
// through a ring of shared memory per warp (blocks of K and of V in turn, 16 bytes a lane and copy),
// which leaves the registers to the products. Products are three of tf32 parts. Against 64 bits the outputs are
// off by 1.9e-7 to 2.9e-7 (rms, normal inputs, 200 to 130000 keys), plain fp32 operations by 3.0e-7 to 9.3e-7.
template <int D, int NT, bool WHOLE, typename Emit>
__device__ __forceinline__ void attend_part32(const PagedArgs& a, unsigned char* shared,
                                              Parts<Shape<float, D, NT>::kWarps, NT>& sm, long long b, int hk, int h0,
                                              int heads, int t0, long long end, Emit emit) {
  typedef Shape<float, D, NT> S;
  typedef Reference<float> R;
  constexpr int CHUNKS = S::kRow / 16, E = 4, BLOCK = 16 * S::kRow;
  constexpr int STEPS = D / (2 * E);      // products of a score: 8 dims each
  constexpr int kChain = 4;               // of them whose large products are summed in the matrix instructions
  constexpr int ROWS = 32 / CHUNKS > 0 ? 32 / CHUNKS : 1;  // rows that one copy of a warp covers
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const long long group = a.q_heads / a.kv_heads;
  const float* kbase = static_cast<const float*>(a.k) + hk * a.ks[1];
  const float* vbase = static_cast<const float*>(a.v) + hk * a.vs[1];
  const uint32_t P = (uint32_t)a.table.page_size;
  const int dim = WHOLE ? D : (int)a.dim;  // dims from there to D are zeros, not read
  const uint32_t mine = (uint32_t)__cvta_generic_to_shared(shared) + warp * S::kStages * BLOCK;
  // Chunk c of row r lies at c ^ swizzle(r): the 8 rows of a matrix, and the 4 rows that a
  // transposed operand takes, are in different banks.
  auto swizzle = [](int r) { return ((r & 3) << 1) | ((r >> 2) & 1); };

  // block i of this warp: keys [16 (W t0 + warp + W i), + 16)
  const long long key0 = (long long)t0 * S::kTile + warp * 16;
  const int count = key0 < end ? (int)((end - key0 + S::kTile - 1) / S::kTile) : 0;

  // Each lane finds the place of one block in 32 (a block lies in one page where WHOLE) or of one row
  // of a block, as element offsets; -1: no such block or row, or no page of the pools.
  long long k_places = -1, v_places = -1;
  bool missing = false;  // a page of this item is not one of the pools'
  auto find = [&](long long key) {
    k_places = v_places = -1;
    bool bad = false;
    if (key < end) {
      const uint32_t index = (uint32_t)key / P, row = (uint32_t)key - index * P;
      const long long page = a.table.page(b, index, a.err);
      bad = page < 0;
      if (!bad) {
        k_places = page * a.ks[0] + row * a.ks[2];
        v_places = page * a.vs[0] + row * a.vs[2];
      }
    }
    missing = __any_sync(0xffffffffu, bad) || missing;
  };
  // piece 2 i: the keys of block i, piece 2 i + 1: its values
  auto copy_piece = [&](int piece, int stage) {
    const int i = piece >> 1;
    const bool values = piece & 1;
    const uint32_t to = mine + stage * BLOCK;
    const long long key = key0 + (long long)i * S::kTile;
    if (!values) {
      if (WHOLE) {
        if ((i & 31) == 0) find(key + (long long)lane * S::kTile);
      } else {
        find(lane < 16 ? key + lane : end);
      }
    }
    const long long place = values ? v_places : k_places, block = __shfl_sync(0xffffffffu, place, i & 31);
    const float* base = values ? vbase : kbase;
    const long long stride = values ? a.vs[2] : a.ks[2];
    const int rows = block < 0 ? 0 : (int)min(16ll, end - key);
    const int r0 = lane / CHUNKS, chunk = lane % CHUNKS;
#pragma unroll
    for (int r = 0; r < 16; r += ROWS) {
      const long long row = WHOLE ? block + (r + r0) * stride : __shfl_sync(0xffffffffu, place, r + r0);
      const bool live = WHOLE ? r + r0 < rows : row >= 0;
#pragma unroll
      for (int c = chunk; c < CHUNKS; c += 32) {
        const bool there = live && (WHOLE || c * E < dim);
        copy_row(to + (r + r0) * S::kRow + ((c ^ swizzle(r + r0)) << 4), there ? base + row + c * E : base, there);
      }
    }
  };
  // bits 0 and 1: whether keys g and g + 8 of block i count
  auto counted = [&](int i) -> uint32_t {
    uint32_t live = 0;
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      const long long key = key0 + (long long)i * S::kTile + g + 8 * x;
      if (key < end) {
        const long long page = a.table.entries[b * a.table.stride + (uint32_t)key / P];
        if (page >= 0 && page < a.table.num_pages) live |= 1u << x;
      }
    }
    return live;
  };

#pragma unroll
  for (int i = 0; i < S::kStages; ++i) {
    if (i < 2 * count) copy_piece(i, i);
    asm volatile("cp.async.commit_group;" ::: "memory");
  }
  // queries as the second operand: head g, the dims of this lane's k
  uint32_t q[NT][STEPS][2];
#pragma unroll
  for (int u = 0; u < NT; ++u) {
    const bool there = u * 8 + g < heads;
    const float* p = static_cast<const float*>(a.q) + b * a.qs[0] + (hk * group + h0 + (there ? u * 8 + g : 0)) * a.qs[1] +
                 t;
#pragma unroll
    for (int i = 0; i < STEPS; ++i)
#pragma unroll
      for (int x = 0; x < 2; ++x)
        q[u][i][x] = there && (WHOLE || (2 * i + x) * E < dim) ? *reinterpret_cast<const uint32_t*>(p + (2 * i + x) * E) : 0u;
  }
  float o[NT][D / 16][4], m[NT][2], l[NT][2];
#pragma unroll
  for (int u = 0; u < NT; ++u) {
#pragma unroll
    for (int i = 0; i < D / 16; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e) o[u][i][e] = 0.f;
    m[u][0] = m[u][1] = -INFINITY;
    l[u][0] = l[u][1] = 0.f;
  }
  const int k_lane = (lane & 15) * S::kRow, k_swizzle = swizzle(lane & 15), k_chunk = lane >> 4;
  int stage = 0;
  auto next_piece = [&](int piece) {  // the current one is read; its slot takes the piece kStages on
    __syncwarp();
    if (piece + S::kStages < 2 * count) copy_piece(piece + S::kStages, stage);
    asm volatile("cp.async.commit_group;" ::: "memory");
    stage = stage + 1 == S::kStages ? 0 : stage + 1;
    asm volatile("cp.async.wait_group %0;" ::"n"(S::kStages - 1) : "memory");
    __syncwarp();  // the other lanes' copies too
  };
  asm volatile("cp.async.wait_group %0;" ::"n"(S::kStages - 1) : "memory");
  __syncwarp();

  for (int i = 0; i < count; ++i) {
    const uint32_t k_at = mine + stage * BLOCK;
    // scores of 16 keys x 8 heads: rows keys g, g + 8, columns heads 2t, 2t + 1
    float s[NT][4], large[NT][4], small[NT][2][4];
#pragma unroll
    for (int u = 0; u < NT; ++u)
#pragma unroll
      for (int e = 0; e < 4; ++e) s[u][e] = small[u][0][e] = small[u][1][e] = 0.f;
#pragma unroll
    for (int j = 0; j < STEPS; ++j) {
      uint32_t k[4], kh[4], kl[4];
      load_matrices(k_at + k_lane + (((2 * j + k_chunk) ^ k_swizzle) << 4), k);
      split4(k, kh, kl);
#pragma unroll
      for (int u = 0; u < NT; ++u) {
        uint32_t qh[2], ql[2];
        split_here(q[u][j][0], qh[0], ql[0]);
        split_here(q[u][j][1], qh[1], ql[1]);
        if (j % kChain == 0)
#pragma unroll
          for (int e = 0; e < 4; ++e) large[u][e] = 0.f;
        mma_tf32(large[u], kh, qh[0], qh[1]);
        mma_tf32(small[u][0], kl, qh[0], qh[1]);
        mma_tf32(small[u][1], kh, ql[0], ql[1]);
        if (j % kChain == kChain - 1)
#pragma unroll
          for (int e = 0; e < 4; ++e) s[u][e] += large[u][e];
      }
    }
    // parts of infinite or huge keys may cancel (inf - inf): such a block's scores are summed term by term
    bool lost = false;
#pragma unroll
    for (int u = 0; u < NT; ++u)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        s[u][e] += small[u][0][e] + small[u][1][e];
        lost |= s[u][e] != s[u][e];
      }
    if (__any_sync(0xffffffffu, lost)) {
#pragma unroll
      for (int u = 0; u < NT; ++u)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int row = g + 8 * (e >> 1), head = u * 8 + 2 * t + (e & 1);
          s[u][e] = 0.f;
          if (head < heads) {
            const float* p = static_cast<const float*>(a.q) + b * a.qs[0] + (hk * group + h0 + head) * a.qs[1];
            for (int d = 0; d < dim; ++d)
              s[u][e] = fmaf(p[d], __uint_as_float(load_word(k_at + row * S::kRow + (((d >> 2) ^ swizzle(row)) << 4) + (d & 3) * 4)),
                             s[u][e]);
          }
        }
    }
    const bool part = missing || end - key0 - (long long)i * S::kTile < 16;
    const uint32_t live = part ? counted(i) : 3u;
    next_piece(2 * i);
    const uint32_t v_at = mine + stage * BLOCK;
    uint32_t ph[NT][2][2], pl[NT][2][2];  // weights as the second operand: keys t and t + 4 of each half, head g
#pragma unroll
    for (int u = 0; u < NT; ++u) {
      float(&z)[4] = s[u];
#pragma unroll
      for (int e = 0; e < 4; ++e) z[e] = part && !(live >> (e >> 1) & 1u) ? -INFINITY : z[e] * a.scale_log2;
      float top0 = fmaxf(z[0], z[2]), top1 = fmaxf(z[1], z[3]);
      if (__any_sync(0xffffffffu, top0 > m[u][0] + R::kSlack || top1 > m[u][1] + R::kSlack)) {
#pragma unroll
        for (int off = 4; off < 32; off <<= 1) {
          top0 = fmaxf(top0, __shfl_xor_sync(0xffffffffu, top0, off));
          top1 = fmaxf(top1, __shfl_xor_sync(0xffffffffu, top1, off));
        }
        const float n0 = fmaxf(m[u][0], top0 - R::kLow), n1 = fmaxf(m[u][1], top1 - R::kLow);
        const float f0 = n0 == -INFINITY ? 1.f : exp2f(m[u][0] - n0);
        const float f1 = n1 == -INFINITY ? 1.f : exp2f(m[u][1] - n1);
        m[u][0] = n0;
        m[u][1] = n1;
        l[u][0] *= f0;
        l[u][1] *= f1;
#pragma unroll
        for (int x = 0; x < D / 16; ++x) {
          o[u][x][0] *= f0;
          o[u][x][1] *= f1;
          o[u][x][2] *= f0;
          o[u][x][3] *= f1;
        }
      }
      const float r0 = m[u][0] == -INFINITY ? 0.f : m[u][0], r1 = m[u][1] == -INFINITY ? 0.f : m[u][1];
      float p[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        // the weight that the products take: what they cut from the low part is not in the total either
        uint32_t hi, lo;
        split(__float_as_uint(exp2_fast(z[e] - (e & 1 ? r1 : r0))), hi, lo);
        p[e] = __uint_as_float(hi) + __uint_as_float(lo & 0xffffe000u);
      }
      l[u][0] += p[0] + p[2];
      l[u][1] += p[1] + p[3];
#pragma unroll
      for (int x = 0; x < 2; ++x)
#pragma unroll
        for (int y = 0; y < 2; ++y) {
          const int from = (t + 4 * y) * 4 + (g >> 1);
          const float even = __shfl_sync(0xffffffffu, p[2 * x], from), odd = __shfl_sync(0xffffffffu, p[2 * x + 1], from);
          split(__float_as_uint(g & 1 ? odd : even), ph[u][x][y], pl[u][x][y]);
        }
    }
#pragma unroll
    for (int j = 0; j < D / 16; ++j) {
      uint32_t vh[2][4], vl[2][4];
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        uint32_t v[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {  // dims 16 j + g (+ 8), keys 8 x + t (+ 4)
          const int row = 8 * x + t + 4 * (e >> 1);
          v[e] = load_word(v_at + row * S::kRow + (((4 * j + (g >> 2) + 2 * (e & 1)) ^ swizzle(row)) << 4) + (g & 3) * 4);
        }
        split4(v, vh[x], vl[x]);
      }
#pragma unroll
      for (int u = 0; u < NT; ++u) {
        float sum[4] = {0.f, 0.f, 0.f, 0.f};  // of the block: the small products first
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          mma_tf32(sum, vl[x], ph[u][x][0], ph[u][x][1]);
          mma_tf32(sum, vh[x], pl[u][x][0], pl[u][x][1]);
        }
#pragma unroll
        for (int x = 0; x < 2; ++x) mma_tf32(sum, vh[x], ph[u][x][0], ph[u][x][1]);
#pragma unroll
        for (int e = 0; e < 4; ++e) o[u][j][e] += sum[e];
      }
    }
    next_piece(2 * i + 1);
  }
  asm volatile("cp.async.wait_all;" ::: "memory");

  join_warps<D, NT, S::kWarps>(shared, sm, m, l, heads, [&](int u, int e, float f, float* to) {
#pragma unroll
    for (int j = 0; j < D / 16; ++j) {
      to[16 * j + g] = o[u][j][e] * f;
      to[16 * j + g + 8] = o[u][j][2 + e] * f;
    }
  }, emit);
}

template <typename T, int D, int NT, bool WHOLE, bool WIDE, typename Emit>
__device__ __forceinline__ void attend_part(const PagedArgs& a, unsigned char* shared,
                                            Parts<Shape<T, D, NT, WIDE>::kWarps, NT>& sm, long long b, int hk, int h0, int heads,
                                            int t0, long long end, Emit emit) {
  if constexpr (sizeof(T) == 2)
    attend_part16<T, D, NT, WHOLE, WIDE>(a, shared, sm, b, hk, h0, heads, t0, end, emit);
  else
    attend_part32<D, NT, WHOLE>(a, shared, sm, b, hk, h0, heads, t0, end, emit);
}

__device__ __forceinline__ long long tiles_of(const PagedArgs& a, long long b, int tile) {
  return (live_length(a, b) + tile - 1) / tile;
}

// Equal shares of all sequences' tiles, one per resident CTA: no CTA waits for a longer sequence, and a
// long cache is split as finely as the GPU is wide. Bound by memory: 256 sequences of 512 to 6144
// positions (28 q / 4 KV heads x 128, fp16) 267 to 283 us, 2 of 100001 to 130000 (40 / 8, bf16) 144 to
// 150 us, 0.96 or more of the copy bandwidth measured on this GPU; the first in fp32 609 to 664 us (0.82 to 0.89).
template <typename T, int D, int NT, bool WHOLE>
__global__ void __launch_bounds__(Shape<T, D, NT>::kWarps * 32, Shape<T, D, NT>::kResident)
    paged_attention_share_kernel(PagedArgs a, PlanArgs plan) {
  constexpr int W = Shape<T, D, NT>::kWarps, kTile = Shape<T, D, NT>::kTile;
  constexpr int PART = 8 * NT * (D + 2);
  asm volatile("griddepcontrol.launch_dependents;");
  extern __shared__ __align__(128) unsigned char shared[];
  __shared__ Parts<W, NT> sm;
  __shared__ long long s_scan[W], s_find[2];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const long long group = a.q_heads / a.kv_heads, per_seq = a.kv_heads * plan.chunks;
  const int G = gridDim.x, cta = blockIdx.x, dim = WHOLE ? D : (int)a.dim;

  // sequences with nothing to see
  for (long long b = cta; b < a.batch; b += G)
    if (live_length(a, b) == 0) {
      if (plan.by_item)
        for (long long i = threadIdx.x; i < per_seq; i += W * 32) plan.joins[b * per_seq + i] = Join{0, 0, 0, 0};
      for (long long i = threadIdx.x; i < a.q_heads * dim; i += W * 32)
        static_cast<T*>(a.out)[b * a.q_heads * dim + i] = store_f<T>(0.f);
    }

  // tiles before each thread's run of sequences, and in all
  const long long run = (a.batch + W * 32 - 1) / (W * 32);
  const long long b_lo = min(a.batch, (long long)threadIdx.x * run), b_hi = min(a.batch, b_lo + run);
  long long mine = 0;
  for (long long b = b_lo; b < b_hi; ++b) mine += tiles_of(a, b, kTile);
  long long upto = mine;
#pragma unroll
  for (int off = 1; off < 32; off <<= 1) {
    const long long x = __shfl_up_sync(0xffffffffu, upto, off);
    if (lane >= off) upto += x;
  }
  if (lane == 31) s_scan[warp] = upto;
  if (threadIdx.x < 2) s_find[threadIdx.x] = 0;
  __syncthreads();
  long long total = 0;
#pragma unroll
  for (int w = 0; w < W; ++w) {
    if (w < warp) upto += s_scan[w];
    total += s_scan[w];
  }
  total *= per_seq;
  const long long shares = max(1ll, min((long long)G, (total + kMinTiles - 1) / kMinTiles));
  const long long lo = cta < shares ? cta * total / shares : total;
  const long long hi = cta < shares ? (cta + 1) * total / shares : total;
  if (lo >= hi) {
    if (threadIdx.x == 0 && !plan.by_item) plan.joins[cta] = Join{0, 0, 0, 0};
    return;
  }
  // the sequence of tile `lo`
  if (mine > 0 && lo >= (upto - mine) * per_seq && lo < upto * per_seq) {
    long long before = (upto - mine) * per_seq, b = b_lo;
    for (; b + 1 < b_hi; ++b) {
      const long long n = tiles_of(a, b, kTile) * per_seq;
      if (lo < before + n) break;
      before += n;
    }
    s_find[0] = b;
    s_find[1] = before;
  }
  __syncthreads();
  long long b = s_find[0], base = s_find[1], at = lo;  // base: first tile of sequence b
  Join join{0, 0, 0, 0};
  bool first_segment = true;

  while (at < hi && b < a.batch) {
    const long long n = live_length(a, b), nb = (n + kTile - 1) / kTile;
    if (nb == 0 || at >= base + nb * per_seq) {
      base += nb * per_seq;
      ++b;
      continue;
    }
    const int h = (int)((at - base) / nb);
    const long long item = base + h * nb;  // first tile of the item
    const int t0 = (int)(at - item), t1 = (int)min(nb, hi - item);
    const int hk = h / plan.chunks, h0 = (h - hk * plan.chunks) * 8 * NT;  // first query head in its group
    const int heads = min((int)group - h0, 8 * NT);
    const long long end = min(n, (long long)t1 * kTile);

    const bool whole = t0 == 0 && t1 == nb;
    const int slot = 2 * cta + (first_segment ? 0 : 1);
    float* part = plan.parts + (long long)slot * PART;
    if (t0 == 0 && t1 < nb) {
      const long long last = ((item + nb) * shares - 1) / total;  // the share that holds the item's last tile
      join = Join{(int)b, h, slot, (int)(last - cta) + 1};
    }
    if (t0 == 0 && plan.by_item && threadIdx.x == 0) plan.joins[b * per_seq + h] = t1 < nb ? join : Join{0, 0, 0, 0};
    T* out = static_cast<T*>(a.out) + (b * a.q_heads + hk * group + h0) * dim;
    attend_part<T, D, NT, WHOLE, false>(a, shared, sm, b, hk, h0, heads, t0, end, [&](int head, int d, const float4& sum, float top, float all) {
      if (whole) {
        if (WHOLE || d < dim) store_four(out + head * dim + d, sum, all);
      } else {
        *reinterpret_cast<float4*>(part + head * D + d) = sum;
        if (d == 0) {
          part[8 * NT * D + head] = top;
          part[8 * NT * (D + 1) + head] = all;
        }
      }
    });
    at = item + t1;
    first_segment = false;
  }
  if (threadIdx.x == 0 && !plan.by_item) plan.joins[cta] = join;
}

// Few items: a cluster of CTAs each, an equal run of its tiles per CTA, joined through the cluster's
// shared memory. One launch, no workspace. Where each of its CTAs has an SM to itself, eight warps share
// the work (WIDE): one warp per scheduler leaves most of the issue slots empty. Bound by latency: 64
// sequences of 256 to 2048 positions (16 / 2 heads, bf16) 23.8 to 24.1 us: a block of 16 keys a warp costs 1.3 us
// of dependent loads and products (11 of them in the longest sequence's CTAs), the rest is launch,
// length, page and joins; one of 200 positions 8.2 us a call, 6.3 in a captured graph.
template <typename T, int D, int NT, bool WHOLE, bool WIDE>
__global__ void __launch_bounds__(Shape<T, D, NT, WIDE>::kWarps * 32, Shape<T, D, NT, WIDE>::kResident)
    paged_attention_cluster_kernel(PagedArgs a, PlanArgs plan) {
  constexpr int W = Shape<T, D, NT, WIDE>::kWarps, kTile = Shape<T, D, NT, WIDE>::kTile;
  extern __shared__ __align__(128) unsigned char shared[];
  __shared__ Parts<W, NT> sm;
  __shared__ __align__(16) float s_sum[8 * NT][D];
  __shared__ float s_top[8 * NT], s_all[8 * NT];
  const uint32_t ctas = cluster_size(), rank = cluster_rank();
  const long long group = a.q_heads / a.kv_heads, per_seq = a.kv_heads * plan.chunks;
  const uint32_t index = blockIdx.x / ctas;
  const long long b = index / (uint32_t)per_seq;
  const int h = (int)(index - b * per_seq);
  const int hk = h / plan.chunks, h0 = (h - hk * plan.chunks) * 8 * NT, heads = min((int)group - h0, 8 * NT);
  const long long n = live_length(a, b), nb = (n + kTile - 1) / kTile;
  const int t0 = (int)(nb * rank / ctas), t1 = (int)(nb * (rank + 1) / ctas);
  attend_part<T, D, NT, WHOLE, WIDE>(a, shared, sm, b, hk, h0, heads, t0, min(n, (long long)t1 * kTile),
                                [&](int head, int d, const float4& sum, float top, float all) {
                                  *reinterpret_cast<float4*>(&s_sum[head][d]) = sum;
                                  if (d == 0) {
                                    s_top[head] = top;
                                    s_all[head] = all;
                                  }
                                });
  cluster_sync();
  // each CTA joins its share of the outputs
  const int dim = WHOLE ? D : (int)a.dim;
  T* out = static_cast<T*>(a.out) + (b * a.q_heads + hk * group + h0) * dim;
  for (int i = rank * W * 32 + threadIdx.x; i < heads * D / 4; i += ctas * W * 32) {
    const int head = 4 * i / D, d = 4 * i - head * D;
    float top[kCluster], all[kCluster], ref = -INFINITY;
    float4 sum[kCluster];
#pragma unroll
    for (int r = 0; r < kCluster; ++r)
      if (r < ctas) {
        top[r] = remote_float(&s_top[head], r);
        all[r] = remote_float(&s_all[head], r);
        sum[r] = remote_float4(&s_sum[head][d], r);
      }
#pragma unroll
    for (int r = 0; r < kCluster; ++r)
      if (r < ctas) ref = fmaxf(ref, top[r]);
    if (ref == -INFINITY) ref = 0.f;
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
    float total = 0.f;
#pragma unroll
    for (int r = 0; r < kCluster; ++r)
      if (r < ctas) {
        const float f = exp2f(top[r] - ref);
        total = fmaf(all[r], f, total);
        o.x = fmaf(sum[r].x, f, o.x), o.y = fmaf(sum[r].y, f, o.y);
        o.z = fmaf(sum[r].z, f, o.z), o.w = fmaf(sum[r].w, f, o.w);
      }
    if (WHOLE || d < dim) store_four(out + head * dim + d, o, total);
  }
  cluster_sync();  // the other CTAs' shared memory is read until here
}

// Joins the parts of the items that more than one share holds, in the order of the shares: CTA per
// (entry of the joins, query head of its item); its WARPS warps take every WARPS-th part each.
template <typename T, int D, int NT, int WARPS>
__global__ void __launch_bounds__(WARPS * 32) paged_attention_join_kernel(PagedArgs a, PlanArgs plan) {
  constexpr int PART = 8 * NT * (D + 2), E = D / 32, BATCH = 4;
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const Join j = plan.joins[blockIdx.x];
  const int group = (int)(a.q_heads / a.kv_heads), head = blockIdx.y;
  const int hk = j.h / plan.chunks, h0 = (j.h - hk * plan.chunks) * 8 * NT;
  if (j.count == 0 || h0 + head >= group) return;
  __shared__ float s_top[WARPS], s_all[WARPS], s_sum[WARPS][D];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  auto part = [&](int k) {
    return plan.parts + (long long)(k == 0 ? j.slot : 2 * (j.slot / 2 + k)) * PART;
  };
  float top = -INFINITY, all = 0.f, sum[E];
#pragma unroll
  for (int e = 0; e < E; ++e) sum[e] = 0.f;
  for (int k0 = warp; k0 < j.count; k0 += WARPS * BATCH) {
    float m[BATCH], l[BATCH], v[BATCH][E];
#pragma unroll
    for (int i = 0; i < BATCH; ++i) {
      const int k = k0 + WARPS * i;
      m[i] = -INFINITY;
      if (k < j.count) {
        const float* p = part(k);
        m[i] = p[8 * NT * D + head];
        l[i] = p[8 * NT * (D + 1) + head];
#pragma unroll
        for (int e = 0; e < E; ++e) v[i][e] = p[head * D + lane + 32 * e];
      }
    }
    float next = top;
#pragma unroll
    for (int i = 0; i < BATCH; ++i) next = fmaxf(next, m[i]);
    const float ref = next == -INFINITY ? 0.f : next, keep = exp2f(top - ref);
    all *= keep;
#pragma unroll
    for (int e = 0; e < E; ++e) sum[e] *= keep;
#pragma unroll
    for (int i = 0; i < BATCH; ++i)
      if (k0 + WARPS * i < j.count) {
        const float f = exp2f(m[i] - ref);
        all = fmaf(l[i], f, all);
#pragma unroll
        for (int e = 0; e < E; ++e) sum[e] = fmaf(v[i][e], f, sum[e]);
      }
    top = next;
  }
  if (lane == 0) {
    s_top[warp] = top;
    s_all[warp] = all;
  }
#pragma unroll
  for (int e = 0; e < E; ++e) s_sum[warp][lane + 32 * e] = sum[e];
  __syncthreads();
  top = s_top[0];
#pragma unroll
  for (int w = 1; w < WARPS; ++w) top = fmaxf(top, s_top[w]);
  const float ref = top == -INFINITY ? 0.f : top;
  float f[WARPS], total = 0.f;
#pragma unroll
  for (int w = 0; w < WARPS; ++w) {
    f[w] = exp2f(s_top[w] - ref);
    total = fmaf(s_all[w], f[w], total);
  }
  T* out = static_cast<T*>(a.out) + (j.b * a.q_heads + hk * group + h0 + head) * a.dim;
  for (int d = threadIdx.x; d < a.dim; d += WARPS * 32) {
    float o = 0.f;
#pragma unroll
    for (int w = 0; w < WARPS; ++w) o = fmaf(s_sum[w][d], f[w], o);
    out[d] = store_f<T>(total == 0.f ? 0.f : o / total);
  }
}

template <typename T> void shape_of(int64_t dim, int nt, int& resident, int& tile) {
  if (dim == 64) resident = nt == 1 ? Shape<T, 64, 1>::kResident : Shape<T, 64, 2>::kResident, tile = Shape<T, 64, 1>::kTile;
  else if (dim == 128) resident = nt == 1 ? Shape<T, 128, 1>::kResident : Shape<T, 128, 2>::kResident, tile = Shape<T, 128, 1>::kTile;
  else resident = Shape<T, 256, 1>::kResident, tile = Shape<T, 256, 1>::kTile;
}

// Query heads of an item: the tensor instruction takes 8, two of them share the key and value
// registers where those leave room (head dims to 128): 256 x 512..6144 with 32 q / 2 KV heads x 128
// 177 us, 268 with every key read twice.
int head_tiles(int64_t dim, int64_t group) { return group > 8 && dim <= 128 ? 2 : 1; }

// Head dim that the kernels are built for: rows of whole 16-byte pieces are read as the next one's, with
// zeros behind them (64 x 256..2048, dim 96, bf16 32 us, 542 with the kernel for any dim); 0: none.
template <typename T> int64_t built_dim(int64_t dim) {
  if (dim > 256 || dim * sizeof(T) % 16 != 0) return 0;
  return dim <= 64 ? 64 : dim <= 128 ? 128 : 256;
}

// CTAs of a cluster per item, 0 for equal shares: clusters where they all run at once and the
// longest sequence that the table can hold leaves each CTA few tiles.
int cluster_ctas(long long items, long long tiles, int full) {
  if (items > full) return 0;
  const long long ctas = min(min((long long)kCluster, full / items), tiles);
  return tiles <= ctas * kClusterTiles ? (int)ctas : 0;
}

// How a tensor shape is launched, from sizes that the host knows.
struct Launch {
  int sms, tiles8, chunks, full, cluster;  // SMs; NT; items per (sequence, KV head); CTAs resident; CTAs per item or 0
  long long items, tiles;             // tiles of the longest sequence that the table can hold
  int64_t dim, workspace;             // dim: the kernels'
};

template <typename T>
Launch plan_launch(int64_t batch, int64_t q_heads, int64_t kv_heads, int64_t head_dim, int64_t positions, int sms) {
  Launch l;
  l.sms = sms;
  const int64_t dim = l.dim = built_dim<T>(head_dim);
  const int64_t group = q_heads / kv_heads;
  l.tiles8 = head_tiles(dim, group);
  int resident, tile;
  shape_of<T>(dim, l.tiles8, resident, tile);
  l.chunks = (int)((group + 8 * l.tiles8 - 1) / (8 * l.tiles8));
  l.full = sms * resident;
  l.items = batch * kv_heads * l.chunks;
  l.tiles = (positions + tile - 1) / tile;
  l.cluster = cluster_ctas(l.items, l.tiles, l.full);
  l.workspace = l.cluster > 0 ? 0 : (int64_t)l.full * (2 * 8 * l.tiles8 * (dim + 2) * sizeof(float) + sizeof(Join));
  return l;
}

// Lets `kernel` have its shared memory, once per device.
template <typename K> cudaError_t allow_shared(K kernel, int bytes, bool (&done)[64]) {
  if (bytes <= 32768) return cudaSuccess;  // within what every kernel has
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess || dev < 0 || dev >= 64 || done[dev]) return e;
  e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
  if (e == cudaSuccess) done[dev] = true;
  return e;
}

int launch_failed(cudaError_t e) {
  return fail(SPECKV_ECUDA, "speckv_paged_attention: launch failed: %s", cudaGetErrorString(e));
}

template <typename T, int D, int NT, bool WHOLE>
int launch_shares(const PagedArgs& a, const PlanArgs& plan, int ctas, cudaStream_t s) {
  typedef Shape<T, D, NT> S;
  static bool done[64] = {false};
  auto kernel = paged_attention_share_kernel<T, D, NT, WHOLE>;
  cudaError_t e = allow_shared(kernel, S::kShared, done);
  if (e != cudaSuccess) return launch_failed(e);
  kernel<<<ctas, S::kWarps * 32, S::kShared, s>>>(a, plan);
  if ((e = cudaGetLastError()) != cudaSuccess) return launch_failed(e);
  // starts while the first kernel ends (programmatic dependent launch), waits for it before it reads
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg = {};
  const int entries = plan.by_item ? (int)(a.batch * a.kv_heads * plan.chunks) : ctas;
  // Few items of many parts: 16 warps join them faster (1 x 130000, 2 items, 32.5 us, 38.0 with 4),
  // else 4 do (64 x 512..6144, 256 items, 78 us, 83 with 16).
  const bool many = ctas > 16 * entries;
  cfg.gridDim = dim3(entries, (unsigned)min((int)(a.q_heads / a.kv_heads), 8 * NT));
  cfg.blockDim = dim3(many ? 512 : 128);
  cfg.stream = s;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  e = many ? cudaLaunchKernelEx(&cfg, paged_attention_join_kernel<T, D, NT, 16>, a, plan)
           : cudaLaunchKernelEx(&cfg, paged_attention_join_kernel<T, D, NT, 4>, a, plan);
  return e == cudaSuccess ? SPECKV_OK : launch_failed(e);
}

template <typename T, int D, int NT, bool WHOLE, bool WIDE>
int launch_clusters(const PagedArgs& a, const PlanArgs& plan, int items, int ctas, cudaStream_t s) {
  typedef Shape<T, D, NT, WIDE> S;
  static bool done[64] = {false};
  auto kernel = paged_attention_cluster_kernel<T, D, NT, WHOLE, WIDE>;
  cudaError_t e = allow_shared(kernel, S::kShared, done);
  if (e != cudaSuccess) return launch_failed(e);
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = ctas;
  attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(items * ctas));
  cfg.blockDim = dim3(S::kWarps * 32);
  cfg.dynamicSmemBytes = S::kShared;
  cfg.stream = s;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  e = cudaLaunchKernelEx(&cfg, kernel, a, plan);
  return e == cudaSuccess ? SPECKV_OK : launch_failed(e);
}

template <typename T, int D, int NT>
int launch_tensor(const PagedArgs& a, const Launch& l, void* workspace, cudaStream_t s) {
  PlanArgs plan;
  plan.chunks = l.chunks;
  plan.by_item = 0;
  plan.joins = static_cast<Join*>(workspace);
  plan.parts = reinterpret_cast<float*>(plan.joins + l.full);
  const bool whole = a.table.page_size % 16 == 0 && a.dim == D;
  // Wide CTAs have an SM each, and clusters of eight do not fill all of them: at 96 CTAs or fewer they
  // all run at once (12.4 us instead of 15.3, 6 x 4000 keys of 16 / 2 heads), 128 took two turns (19.4, 15.8).
  constexpr bool can = sizeof(T) == 2;
  if (l.cluster > 0 && can && l.items * l.cluster * 3 <= l.sms * 2)
    return whole ? launch_clusters<T, D, NT, true, can>(a, plan, (int)l.items, l.cluster, s)
                  : launch_clusters<T, D, NT, false, can>(a, plan, (int)l.items, l.cluster, s);
  if (l.cluster > 0)
    return whole ? launch_clusters<T, D, NT, true, false>(a, plan, (int)l.items, l.cluster, s)
                  : launch_clusters<T, D, NT, false, false>(a, plan, (int)l.items, l.cluster, s);
  // no more CTAs than shares of the longest sequences possible
  const double most = (double)l.items * (double)l.tiles / kMinTiles;
  const int ctas = most < l.full ? (int)most + 1 : l.full;
  plan.by_item = l.items < ctas;
  return whole ? launch_shares<T, D, NT, true>(a, plan, ctas, s) : launch_shares<T, D, NT, false>(a, plan, ctas, s);
}

template <typename T>
int launch_paged(const PagedArgs& a, void* workspace, int64_t bytes, cudaStream_t s) {
  // 16-byte loads need aligned rows; other views take the scalar kernel
  const size_t es = sizeof(T);
  bool aligned = built_dim<T>(a.dim) > 0;
  const void* bases[4] = {a.q, a.k, a.v, a.out};
  for (const void* p : bases) aligned = aligned && reinterpret_cast<uintptr_t>(p) % 16 == 0;
  for (int i = 0; i < 3; ++i) aligned = aligned && a.ks[i] * es % 16 == 0 && a.vs[i] * es % 16 == 0;
  for (int i = 0; i < 2; ++i) aligned = aligned && a.qs[i] * es % 16 == 0;
  if (!aligned) {
    paged_attention_scalar_kernel<T><<<(unsigned)(a.batch * a.q_heads), kScalarWarps * 32, 0, s>>>(a);
    return check_launch("speckv_paged_attention");
  }
  const int sms = sm_count();
  if (sms == 0) return fail(SPECKV_ECUDA, "speckv_paged_attention: no SM count");
  const Launch l = plan_launch<T>(a.batch, a.q_heads, a.kv_heads, a.dim, a.table.width * a.table.page_size, sms);
  if (l.workspace > 0 && (workspace == nullptr || bytes < l.workspace || reinterpret_cast<uintptr_t>(workspace) % 16))
    return fail(SPECKV_EINVAL, "speckv_paged_attention: workspace of %lld bytes, %lld needed (16-byte aligned)",
                (long long)bytes, (long long)l.workspace);
  if (l.dim == 64)
    return l.tiles8 == 1 ? launch_tensor<T, 64, 1>(a, l, workspace, s) : launch_tensor<T, 64, 2>(a, l, workspace, s);
  if (l.dim == 128)
    return l.tiles8 == 1 ? launch_tensor<T, 128, 1>(a, l, workspace, s) : launch_tensor<T, 128, 2>(a, l, workspace, s);
  return launch_tensor<T, 256, 1>(a, l, workspace, s);
}

}  // namespace
}  // namespace speckv

using namespace speckv;

extern "C" int speckv_paged_attention(const void* query, const void* key_pages, const void* value_pages,
                                      const int64_t* strides, const int64_t* page_table, int64_t table_stride,
                                      int64_t table_pages, int64_t num_pages, int64_t page_size,
                                      const int64_t* lengths, void* out, int64_t batch, int64_t q_heads,
                                      int64_t kv_heads, int64_t dim, float scale, int32_t dtype, void* workspace,
                                      int64_t workspace_bytes, void* stream) {
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
  st = check_strides(fn, strides, 8);
  if (st) return st;
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
  drop_unused_strides(a.qs, {batch, q_heads});
  drop_unused_strides(a.ks, {num_pages, kv_heads, page_size});
  drop_unused_strides(a.vs, {num_pages, kv_heads, page_size});
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
    case SPECKV_F32: return launch_paged<float>(a, workspace, workspace_bytes, s);
    case SPECKV_BF16: return launch_paged<__nv_bfloat16>(a, workspace, workspace_bytes, s);
    default: return launch_paged<__half>(a, workspace, workspace_bytes, s);
  }
}

extern "C" int64_t speckv_paged_attention_workspace(int64_t batch, int64_t q_heads, int64_t kv_heads, int64_t dim,
                                                    int64_t table_pages, int64_t page_size, int32_t dtype) {
  if (batch < 1 || q_heads < 1 || kv_heads < 1 || q_heads % kv_heads != 0 || table_pages < 1 || page_size < 1 ||
      table_pages > (1ll << 31) / page_size || (dtype == SPECKV_F32 ? built_dim<float>(dim) : built_dim<__half>(dim)) == 0)
    return 0;
  const int64_t positions = table_pages * page_size;
  return dtype == SPECKV_F32 ? plan_launch<float>(batch, q_heads, kv_heads, dim, positions, sm_count()).workspace
                             : plan_launch<__half>(batch, q_heads, kv_heads, dim, positions, sm_count()).workspace;
}
