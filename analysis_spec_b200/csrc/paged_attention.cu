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

// ---- tensor-core kernel: head dims 64 / 128 / 256 in bf16 / fp16 -------------------------------

__device__ __forceinline__ uint4 load_stream(const void* p) {
  uint4 r;
  asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];"
               : "=r"(r.x), "=r"(r.y), "=r"(r.z), "=r"(r.w)
               : "l"(p));
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

constexpr int kWarps = 4;
constexpr int kTile = 16 * kWarps;   // keys of a tile: 16 a warp
constexpr int kMinTiles = 2;         // a CTA's share is at least this many tiles
constexpr int kCluster = 8;          // CTAs of a cluster at most
constexpr int kClusterTiles = 8;     // tiles of a cluster's CTA at most
constexpr float kSlack = 8.f;        // scores may pass the running reference by 2^8 before it moves

// An item is (sequence, KV head, up to 8 NT of its query heads). All items' tiles, in order, are
// cut into equal shares, one per CTA; a share that begins or ends inside an item leaves its part
// of that item in the workspace, and the CTA in whose share the item begins describes it for
// the join.
struct Join {
  int b, h, slot, count;  // count 0: nothing to join; parts at `slot`, then slots 2 (c + 1), 2 (c + 2), ...
};

struct PlanArgs {
  float* parts;   // (2 * CTAs) x [8 NT][dim + 2]: sums, reference, total
  Join* joins;    // one per CTA
  int chunks;     // items per (sequence, KV head)
};

__device__ __forceinline__ long long tiles_of(const PagedArgs& a, long long b) {
  return (live_length(a, b) + kTile - 1) / kTile;
}

// Shared memory of a CTA: its warps' parts of an item.
template <int D, int NT> struct Parts {
  float o[kWarps][8][D + 4];
  float m[kWarps][8 * NT], l[kWarps][8 * NT];
};

// One CTA's part of an item: tiles [t0, ...) of its keys up to position `end`. Calls
// emit(head of the item, dim, sum, reference, total) for each of its heads and dims.
template <typename T, int D, int NT, bool PAGE16, typename Emit>
__device__ __forceinline__ void attend_part(const PagedArgs& a, Parts<D, NT>& sm, long long b, int hk, int h0, int heads,
                                            int t0, long long end, Emit emit) {
  constexpr int KC = D / 32;  // 16-byte chunks of a key row per lane
  constexpr int VC = D / 64;  // 16-byte chunks of a value row per lane
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const long long group = a.q_heads / a.kv_heads;
  const T* kbase = static_cast<const T*>(a.k) + hk * a.ks[1];
  const T* vbase = static_cast<const T*>(a.v) + hk * a.vs[1];
  const int64_t* table = a.table.entries + b * a.table.stride;
  const uint32_t P = (uint32_t)a.table.page_size;

  uint4 kreg[2][KC], vreg[4][VC];
  uint32_t seen = 0;  // bit 0 / 1: key rows g and g + 8 of the block in kreg are live
  long long pages = -1;
  // block i of this warp: keys [16 (4 t0 + warp + 4 i), + 16)
  const long long key0 = (long long)t0 * kTile + warp * 16;
  const int count = key0 < end ? (int)((end - key0 + kTile - 1) / kTile) : 0;

  // rows of block i: PAGE16: one page for all; else a page per row
  long long page = -1;
  uint32_t row = 0;
  auto place = [&](int i) {
    if (PAGE16) {
      if ((i & 31) == 0) {
        const long long key = key0 + (long long)(i + lane) * kTile;
        pages = -1;
        if (key < end) pages = a.table.page(b, (uint32_t)key / P, a.err);
      }
      page = __shfl_sync(0xffffffffu, pages, i & 31);
      row = (uint32_t)(key0 + (long long)i * kTile) % P;
    }
  };
  auto row_ptr = [&](const T* from, const long long* st, long long key) -> const T* {
    if (key >= end) return nullptr;
    const uint32_t index = (uint32_t)key / P;
    const long long p = a.table.page(b, index, a.err);
    return p < 0 ? nullptr : from + p * st[0] + (long long)((uint32_t)key - index * P) * st[2];
  };
  auto load_k = [&](int i) {
    const long long key = key0 + (long long)i * kTile;
    const T* p0;
    const T* p1;
    if (PAGE16) {
      const int live = page < 0 ? 0 : (int)min(16ll, end - key);
      p0 = kbase + page * a.ks[0] + (long long)(row + g) * a.ks[2];
      p1 = g + 8 < live ? p0 + 8 * a.ks[2] : nullptr;
      if (g >= live) p0 = nullptr;
    } else {
      p0 = row_ptr(kbase, a.ks, key + g);
      p1 = row_ptr(kbase, a.ks, key + g + 8);
    }
    seen = (p0 != nullptr ? 1u : 0u) | (p1 != nullptr ? 2u : 0u);
#pragma unroll
    for (int j = 0; j < KC; ++j) {
      kreg[0][j] = kreg[1][j] = make_uint4(0, 0, 0, 0);
      if (p0 != nullptr) kreg[0][j] = load_stream(p0 + (t + 4 * j) * 8);
      if (p1 != nullptr) kreg[1][j] = load_stream(p1 + (t + 4 * j) * 8);
    }
  };
  auto load_v = [&](int i) {
    const long long key = key0 + (long long)i * kTile;
#pragma unroll
    for (int x = 0; x < 4; ++x) {
      const int k = 2 * t + (x & 1) + (x >> 1) * 8;  // keys 2t, 2t + 1, 2t + 8, 2t + 9
      const T* p;
      if (PAGE16) {
        const int live = page < 0 ? 0 : (int)min(16ll, end - key);
        p = k < live ? vbase + page * a.vs[0] + (long long)(row + k) * a.vs[2] : nullptr;
      } else {
        p = row_ptr(vbase, a.vs, key + k);
      }
#pragma unroll
      for (int c = 0; c < VC; ++c) {
        vreg[x][c] = make_uint4(0, 0, 0, 0);  // rows that are not there may hold anything: 0 x NaN is NaN
        if (p != nullptr) vreg[x][c] = load_stream(p + (g + 8 * c) * 8);
      }
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
      if (u * 8 + g < heads) {
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
      // The reference need not be the maximum: any value within 2^8 of it keeps every weight and
      // sum well inside fp32, and the sums are divided by the total at the end. So it moves only
      // when a score passes it by more than that (the first block moves it from -inf).
      if (__any_sync(0xffffffffu, t0m > m[u][0] + kSlack || t1m > m[u][1] + kSlack)) {
#pragma unroll
        for (int off = 4; off < 32; off <<= 1) {
          t0m = fmaxf(t0m, __shfl_xor_sync(0xffffffffu, t0m, off));
          t1m = fmaxf(t1m, __shfl_xor_sync(0xffffffffu, t1m, off));
        }
        const float n0 = fmaxf(m[u][0], t0m), n1 = fmaxf(m[u][1], t1m);
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
      const float p0 = exp2f(s[u][0] - r0), p1 = exp2f(s[u][1] - r1), p2 = exp2f(s[u][2] - r0),
                  p3 = exp2f(s[u][3] - r1);
      l[u][0] += p0 + p2;
      l[u][1] += p1 + p3;
      // weights to (key pairs, heads) fragments, in two 16-bit parts: the tensor pipe has room
      // for a second product, and one 8-bit weight alone would lose more than the output's rounding
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


  // the warps' parts, joined
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
  __syncthreads();
#pragma unroll
  for (int u = 0; u < NT; ++u) {
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int head = u * 8 + 2 * t + e;
      float top = sm.m[0][head];
#pragma unroll
      for (int w = 1; w < kWarps; ++w) top = fmaxf(top, sm.m[w][head]);
      const float f = top == -INFINITY ? 1.f : exp2f(m[u][e] - top);
#pragma unroll
      for (int c = 0; c < VC; ++c) {
        float* to = &sm.o[warp][2 * t + e][(g + 8 * c) * 8];
#pragma unroll
        for (int x = 0; x < 4; ++x)
          *reinterpret_cast<float2*>(to + 2 * x) = make_float2(o[u][c][x][e] * f, o[u][c][x][2 + e] * f);
      }
    }
    __syncthreads();
    for (int i = threadIdx.x; i < 8 * D; i += kWarps * 32) {
      const int head = i / D, d = i - head * D;
      if (u * 8 + head >= heads) break;
      float top = sm.m[0][u * 8 + head];
#pragma unroll
      for (int w = 1; w < kWarps; ++w) top = fmaxf(top, sm.m[w][u * 8 + head]);
      const float ref = top == -INFINITY ? 0.f : top;
      float sum = 0.f, all = 0.f;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) {
        sum += sm.o[w][head][d];
        all = fmaf(sm.l[w][u * 8 + head], exp2f(sm.m[w][u * 8 + head] - ref), all);
      }
      emit(u * 8 + head, d, sum, top, all);
    }
    __syncthreads();
  }
}

// CTAs per SM of the tensor-core kernels.
template <int D, int NT> constexpr int resident() { return D == 64 ? (NT == 1 ? 4 : 3) : D == 128 ? (NT == 1 ? 3 : 2) : 2; }

template <typename T, int D, int NT, bool PAGE16>
__global__ void __launch_bounds__(kWarps * 32, resident<D, NT>()) paged_attention_mma_kernel(PagedArgs a, PlanArgs plan) {
  constexpr int PART = 8 * NT * (D + 2);
  asm volatile("griddepcontrol.launch_dependents;");
  __shared__ Parts<D, NT> sm;
  __shared__ long long s_scan[kWarps], s_find[2];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const long long group = a.q_heads / a.kv_heads, per_seq = a.kv_heads * plan.chunks;
  const int G = gridDim.x, cta = blockIdx.x;

  // sequences with nothing to see
  for (long long b = cta; b < a.batch; b += G)
    if (live_length(a, b) == 0)
      for (long long i = threadIdx.x; i < a.q_heads * D; i += kWarps * 32)
        static_cast<T*>(a.out)[b * a.q_heads * D + i] = store_f<T>(0.f);

  // tiles before each thread's run of sequences, and in all
  const long long run = (a.batch + kWarps * 32 - 1) / (kWarps * 32);
  const long long b_lo = min(a.batch, (long long)threadIdx.x * run), b_hi = min(a.batch, b_lo + run);
  long long mine = 0;
  for (long long b = b_lo; b < b_hi; ++b) mine += tiles_of(a, b);
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
  for (int w = 0; w < kWarps; ++w) {
    if (w < warp) upto += s_scan[w];
    total += s_scan[w];
  }
  total *= per_seq;
  const long long shares = max(1ll, min((long long)G, (total + kMinTiles - 1) / kMinTiles));
  const long long lo = cta < shares ? cta * total / shares : total;
  const long long hi = cta < shares ? (cta + 1) * total / shares : total;
  if (lo >= hi) {
    if (threadIdx.x == 0) plan.joins[cta] = Join{0, 0, 0, 0};
    return;
  }
  // the sequence of tile `lo`
  if (mine > 0 && lo >= (upto - mine) * per_seq && lo < upto * per_seq) {
    long long before = (upto - mine) * per_seq, b = b_lo;
    for (; b + 1 < b_hi; ++b) {
      const long long n = tiles_of(a, b) * per_seq;
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
    T* out = static_cast<T*>(a.out) + (b * a.q_heads + hk * group + h0) * D;
    attend_part<T, D, NT, PAGE16>(a, sm, b, hk, h0, heads, t0, end, [&](int head, int d, float sum, float top, float all) {
      if (whole) {
        out[head * D + d] = store_f<T>(all == 0.f ? 0.f : sum / all);
      } else {
        part[head * D + d] = sum;
        if (d == 0) {
          part[8 * NT * D + head] = top;
          part[8 * NT * (D + 1) + head] = all;
        }
      }
    });
    at = item + t1;
    first_segment = false;
  }
  if (threadIdx.x == 0) plan.joins[cta] = join;
}

// Few items: a cluster of CTAs each, an equal run of its tiles per CTA, joined through the
// cluster's shared memory. One launch, no workspace.
template <typename T, int D, int NT, bool PAGE16>
__global__ void __launch_bounds__(kWarps * 32, resident<D, NT>())
    paged_attention_cluster_kernel(PagedArgs a, PlanArgs plan) {
  __shared__ Parts<D, NT> sm;
  __shared__ float s_sum[8 * NT][D], s_top[8 * NT], s_all[8 * NT];
  const uint32_t ctas = cluster_size(), rank = cluster_rank();
  const long long group = a.q_heads / a.kv_heads, per_seq = a.kv_heads * plan.chunks;
  const uint32_t index = blockIdx.x / ctas;
  const long long b = index / (uint32_t)per_seq;
  const int h = (int)(index - b * per_seq);
  const int hk = h / plan.chunks, h0 = (h - hk * plan.chunks) * 8 * NT, heads = min((int)group - h0, 8 * NT);
  const long long n = live_length(a, b), nb = (n + kTile - 1) / kTile;
  const int t0 = (int)(nb * rank / ctas), t1 = (int)(nb * (rank + 1) / ctas);
  attend_part<T, D, NT, PAGE16>(a, sm, b, hk, h0, heads, t0, min(n, (long long)t1 * kTile),
                                [&](int head, int d, float sum, float top, float all) {
                                  s_sum[head][d] = sum;
                                  if (d == 0) {
                                    s_top[head] = top;
                                    s_all[head] = all;
                                  }
                                });
  cluster_sync();
  // each CTA joins its share of the outputs
  T* out = static_cast<T*>(a.out) + (b * a.q_heads + hk * group + h0) * D;
  for (int i = rank * kWarps * 32 + threadIdx.x; i < heads * D; i += ctas * kWarps * 32) {
    const int head = i / D, d = i - head * D;
    float top[kCluster], all[kCluster], sum[kCluster], ref = -INFINITY;
#pragma unroll
    for (int r = 0; r < kCluster; ++r)
      if (r < ctas) {
        top[r] = remote_float(&s_top[head], r);
        all[r] = remote_float(&s_all[head], r);
        sum[r] = remote_float(&s_sum[head][d], r);
      }
#pragma unroll
    for (int r = 0; r < kCluster; ++r)
      if (r < ctas) ref = fmaxf(ref, top[r]);
    if (ref == -INFINITY) ref = 0.f;
    float o = 0.f, total = 0.f;
#pragma unroll
    for (int r = 0; r < kCluster; ++r)
      if (r < ctas) {
        const float f = exp2f(top[r] - ref);
        total = fmaf(all[r], f, total);
        o = fmaf(sum[r], f, o);
      }
    out[i] = store_f<T>(total == 0.f ? 0.f : o / total);
  }
  cluster_sync();  // the other CTAs' shared memory is read until here
}

// Joins the parts of the items that more than one share holds, in the order of the shares: CTA per
// (share, query head of the item that begins in it); its warps take every fourth part each.
template <typename T, int D, int NT>
__global__ void __launch_bounds__(128) paged_attention_join_kernel(PagedArgs a, PlanArgs plan) {
  constexpr int PART = 8 * NT * (D + 2), E = D / 32, BATCH = 4;
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const Join j = plan.joins[blockIdx.x];
  const int group = (int)(a.q_heads / a.kv_heads), head = blockIdx.y;
  const int hk = j.h / plan.chunks, h0 = (j.h - hk * plan.chunks) * 8 * NT;
  if (j.count == 0 || h0 + head >= group) return;
  __shared__ float s_top[4], s_all[4], s_sum[4][D];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  // part 0 is at its own slot, part k >= 1 the first of share blockIdx.x + k
  auto part = [&](int k) {
    return plan.parts + (long long)(k == 0 ? j.slot : 2 * ((int)blockIdx.x + k)) * PART;
  };
  float top = -INFINITY, all = 0.f, sum[E];
#pragma unroll
  for (int e = 0; e < E; ++e) sum[e] = 0.f;
  for (int k0 = warp; k0 < j.count; k0 += 4 * BATCH) {
    float m[BATCH], l[BATCH], v[BATCH][E];
#pragma unroll
    for (int i = 0; i < BATCH; ++i) {
      const int k = k0 + 4 * i;
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
      if (k0 + 4 * i < j.count) {
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
  top = fmaxf(fmaxf(s_top[0], s_top[1]), fmaxf(s_top[2], s_top[3]));
  const float ref = top == -INFINITY ? 0.f : top;
  float f[4], total = 0.f;
#pragma unroll
  for (int w = 0; w < 4; ++w) {
    f[w] = exp2f(s_top[w] - ref);
    total = fmaf(s_all[w], f[w], total);
  }
  T* out = static_cast<T*>(a.out) + (j.b * a.q_heads + hk * group + h0 + head) * D;
  for (int d = threadIdx.x; d < D; d += 128) {
    float o = 0.f;
#pragma unroll
    for (int w = 0; w < 4; ++w) o = fmaf(s_sum[w][d], f[w], o);
    out[d] = store_f<T>(total == 0.f ? 0.f : o / total);
  }
}

int sm_count() {
  static int counts[64] = {0};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return 0;
  if (counts[dev] == 0 && cudaDeviceGetAttribute(&counts[dev], cudaDevAttrMultiProcessorCount, dev) != cudaSuccess)
    return 0;
  return counts[dev];
}

int ctas_per_sm(int64_t dim, int nt) {
  return dim == 64 ? (nt == 1 ? resident<64, 1>() : resident<64, 2>())
                   : dim == 128 ? (nt == 1 ? resident<128, 1>() : resident<128, 2>()) : resident<256, 1>();
}

// Query heads of an item: the tensor instruction takes 8, two of them share the key and value
// registers where those leave room (head dims to 128).
int head_tiles(int64_t dim, int64_t group) { return group > 8 && dim <= 128 ? 2 : 1; }

bool tensor_shape(int64_t dim, int32_t dtype) {
  return dtype != SPECKV_F32 && (dim == 64 || dim == 128 || dim == 256);
}

// CTAs of a cluster per item, 0 for equal shares: clusters where they all run at once and the
// longest sequence that the table can hold leaves each CTA few tiles.
int cluster_ctas(long long items, long long tiles, int full) {
  int ctas = 1;
  while (ctas < kCluster && ctas < tiles && items * ctas * 2 <= full) ctas *= 2;
  return items * ctas <= full && tiles <= (long long)ctas * kClusterTiles ? ctas : 0;
}

// How a tensor shape is launched, from sizes that the host knows.
struct Launch {
  int tiles8, chunks, full, cluster;  // NT; items per (sequence, KV head); CTAs resident; CTAs per item or 0
  long long items, tiles;             // tiles of the longest sequence that the table can hold
  int64_t workspace;
};

Launch plan_launch(int64_t batch, int64_t q_heads, int64_t kv_heads, int64_t dim, int64_t positions, int sms) {
  Launch l;
  const int64_t group = q_heads / kv_heads;
  l.tiles8 = head_tiles(dim, group);
  l.chunks = (int)((group + 8 * l.tiles8 - 1) / (8 * l.tiles8));
  l.full = sms * ctas_per_sm(dim, l.tiles8);
  l.items = batch * kv_heads * l.chunks;
  l.tiles = (positions + kTile - 1) / kTile;
  l.cluster = cluster_ctas(l.items, l.tiles, l.full);
  l.workspace = l.cluster > 0 ? 0 : (int64_t)l.full * (2 * 8 * l.tiles8 * (dim + 2) * sizeof(float) + sizeof(Join));
  return l;
}

template <typename T, int D, int NT>
int launch_shares(const PagedArgs& a, const PlanArgs& plan, int ctas, cudaStream_t s) {
  if (a.table.page_size % 16 == 0)
    paged_attention_mma_kernel<T, D, NT, true><<<ctas, kWarps * 32, 0, s>>>(a, plan);
  else
    paged_attention_mma_kernel<T, D, NT, false><<<ctas, kWarps * 32, 0, s>>>(a, plan);
  int st = check_launch("speckv_paged_attention");
  if (st) return st;
  // starts while the first kernel ends (programmatic dependent launch), waits for it before it reads
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(ctas, (unsigned)min((int)(a.q_heads / a.kv_heads), 8 * NT));
  cfg.blockDim = dim3(128);
  cfg.stream = s;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, paged_attention_join_kernel<T, D, NT>, a, plan);
  if (e != cudaSuccess) return fail(SPECKV_ECUDA, "speckv_paged_attention: launch failed: %s", cudaGetErrorString(e));
  return SPECKV_OK;
}

template <typename T, int D, int NT>
int launch_clusters(const PagedArgs& a, const PlanArgs& plan, int items, int ctas, cudaStream_t s) {
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = ctas;
  attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(items * ctas));
  cfg.blockDim = dim3(kWarps * 32);
  cfg.stream = s;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  const cudaError_t e = a.table.page_size % 16 == 0
                            ? cudaLaunchKernelEx(&cfg, paged_attention_cluster_kernel<T, D, NT, true>, a, plan)
                            : cudaLaunchKernelEx(&cfg, paged_attention_cluster_kernel<T, D, NT, false>, a, plan);
  if (e != cudaSuccess) return fail(SPECKV_ECUDA, "speckv_paged_attention: launch failed: %s", cudaGetErrorString(e));
  return SPECKV_OK;
}

template <typename T, int D, int NT>
int launch_tensor(const PagedArgs& a, const Launch& l, void* workspace, cudaStream_t s) {
  PlanArgs plan;
  plan.chunks = l.chunks;
  plan.joins = static_cast<Join*>(workspace);
  plan.parts = reinterpret_cast<float*>(plan.joins + l.full);
  if (l.cluster > 0) return launch_clusters<T, D, NT>(a, plan, (int)l.items, l.cluster, s);
  // no more CTAs than shares of the longest sequences possible
  const double most = (double)l.items * (double)l.tiles / kMinTiles;
  return launch_shares<T, D, NT>(a, plan, most < l.full ? (int)most + 1 : l.full, s);
}

template <typename T>
int launch_paged(const PagedArgs& a, int32_t dtype, void* workspace, int64_t bytes, cudaStream_t s) {
  // 16-byte loads need aligned rows; other views take the scalar kernel
  const size_t es = sizeof(T);
  bool aligned = tensor_shape(a.dim, dtype);
  const void* bases[4] = {a.q, a.k, a.v, a.out};
  for (const void* p : bases) aligned = aligned && reinterpret_cast<uintptr_t>(p) % 16 == 0;
  for (int i = 0; i < 3; ++i) aligned = aligned && a.ks[i] * es % 16 == 0 && a.vs[i] * es % 16 == 0;
  for (int i = 0; i < 2; ++i) aligned = aligned && a.qs[i] * es % 16 == 0;
  if (!aligned) {
    paged_attention_scalar_kernel<T><<<(unsigned)(a.batch * a.q_heads), kScalarWarps * 32, 0, s>>>(a);
    return check_launch("speckv_paged_attention");
  }
  if constexpr (sizeof(T) == 2) {
    const int sms = sm_count();
    if (sms == 0) return fail(SPECKV_ECUDA, "speckv_paged_attention: no SM count");
    const Launch l = plan_launch(a.batch, a.q_heads, a.kv_heads, a.dim, a.table.width * a.table.page_size, sms);
    if (l.workspace > 0 && (workspace == nullptr || bytes < l.workspace || reinterpret_cast<uintptr_t>(workspace) % 16))
      return fail(SPECKV_EINVAL, "speckv_paged_attention: workspace of %lld bytes, %lld needed (16-byte aligned)",
                  (long long)bytes, (long long)l.workspace);
    if (a.dim == 64)
      return l.tiles8 == 1 ? launch_tensor<T, 64, 1>(a, l, workspace, s) : launch_tensor<T, 64, 2>(a, l, workspace, s);
    if (a.dim == 128)
      return l.tiles8 == 1 ? launch_tensor<T, 128, 1>(a, l, workspace, s) : launch_tensor<T, 128, 2>(a, l, workspace, s);
    return launch_tensor<T, 256, 1>(a, l, workspace, s);
  }
  return SPECKV_OK;
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
    case SPECKV_F32: return launch_paged<float>(a, dtype, workspace, workspace_bytes, s);
    case SPECKV_BF16: return launch_paged<__nv_bfloat16>(a, dtype, workspace, workspace_bytes, s);
    default: return launch_paged<__half>(a, dtype, workspace, workspace_bytes, s);
  }
}

extern "C" int64_t speckv_paged_attention_workspace(int64_t batch, int64_t q_heads, int64_t kv_heads, int64_t dim,
                                                    int64_t table_pages, int64_t page_size, int32_t dtype) {
  if (batch < 1 || q_heads < 1 || kv_heads < 1 || q_heads % kv_heads != 0 || table_pages < 1 || page_size < 1 ||
      table_pages > (1ll << 31) / page_size || !tensor_shape(dim, dtype))
    return 0;
  return plan_launch(batch, q_heads, kv_heads, dim, table_pages * page_size, sm_count()).workspace;
}
