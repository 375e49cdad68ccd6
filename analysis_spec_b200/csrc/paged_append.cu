// Append of new K / V rows to a paged cache, with the rotary position rotation applied to K on
// the way and to the queries in the same launch.
//
//   slot = starts[b] + t, page = table[b][slot / P], row = slot mod P
//   key_pages[page][h][row][:]   = rotate(key[b][h][t], position)
//   value_pages[page][h][row][:] = value[b][h][t]
//   query_out[b][h][t]           = rotate(query[b][h][t], position)
// with, for j < r / 2, c = cos[position][j], s = sin[position][j] and the pair (x, y) of
// elements (j, j + r / 2) or, interleaved, (2j, 2j + 1): x' = x c - y s, y' = y c + x s.
// Products in fp32, one rounding on the way out.
#include "paged.cuh"

namespace speckv {
namespace {

struct AppendArgs {
  const void* key;
  const void* value;
  const void* query;   // may be null
  void* query_out;
  void* key_pages;
  void* value_pages;
  long long ks[3], vs[3], qs[3], os[3], kps[3], vps[3];
  PageTable table;
  const int64_t* starts;
  const int64_t* counts;     // may be null: every row of every sequence is live
  const int64_t* positions;  // may be null: the slot
  long long pos_b, pos_t;
  const float* cos;          // (positions, rot / 2); null: no rotation
  const float* sin;
  long long rot_positions;
  int rot, interleaved;
  long long batch, q_heads, kv_heads, rows, dim;
  unsigned long long* err;
};

// Where a token goes: pool page (-1: it is padding or refused), row of the page, rotation row.
struct Place {
  long long page, row, position;
};

__device__ __forceinline__ Place place_token(const AppendArgs& a, long long b, long long t) {
  Place p{-1, 0, 0};
  if (a.counts != nullptr && t >= a.counts[b]) return p;
  const long long slot = a.starts[b] + t;
  if (slot < 0 || slot >= a.table.width * a.table.page_size) {
    record_error(a.err, SPECKV_DERR_PAGE_TABLE, slot);
    return p;
  }
  p.position = a.positions != nullptr ? a.positions[b * a.pos_b + t * a.pos_t] : slot;
  if (a.cos != nullptr && (p.position < 0 || p.position >= a.rot_positions)) {
    record_error(a.err, SPECKV_DERR_ROTATION_INDEX, p.position);
    return p;
  }
  const long long index = slot / a.table.page_size;
  p.row = slot - index * a.table.page_size;
  p.page = a.table.page(b, index, a.err);
  return p;
}

constexpr int kAppendThreads = 64;

// One CTA per token; elements one by one: any head dim, rotation width, stride and alignment (8
// prompts to 4001 tokens, as below: 405 us).
template <typename T>
__global__ void __launch_bounds__(kAppendThreads) paged_append_scalar_kernel(AppendArgs a) {
  const long long b = blockIdx.x / a.rows, t = blockIdx.x % a.rows;
  __shared__ Place shared;
  if (threadIdx.x == 0) shared = place_token(a, b, t);
  __syncthreads();
  const Place p = shared;
  const long long q_heads = a.query != nullptr ? a.q_heads : 0;
  const int half = a.cos != nullptr ? a.rot / 2 : 0;
  // item of a head: the `half` pairs, then the elements that are copied
  const int items = (int)a.dim - half;
  const long long total = (q_heads + 2 * a.kv_heads) * items;
  for (long long i = threadIdx.x; i < total; i += kAppendThreads) {
    long long h = i / items;
    const int j = (int)(i - h * items);
    const T* src;
    T* dst;
    bool turn = j < half;
    if (h < q_heads) {
      src = static_cast<const T*>(a.query) + b * a.qs[0] + h * a.qs[1] + t * a.qs[2];
      dst = static_cast<T*>(a.query_out) + b * a.os[0] + h * a.os[1] + t * a.os[2];
    } else if (p.page < 0) {
      continue;
    } else if (h < q_heads + a.kv_heads) {
      h -= q_heads;
      src = static_cast<const T*>(a.key) + b * a.ks[0] + h * a.ks[1] + t * a.ks[2];
      dst = static_cast<T*>(a.key_pages) + p.page * a.kps[0] + h * a.kps[1] + p.row * a.kps[2];
    } else {
      h -= q_heads + a.kv_heads;
      src = static_cast<const T*>(a.value) + b * a.vs[0] + h * a.vs[1] + t * a.vs[2];
      dst = static_cast<T*>(a.value_pages) + p.page * a.vps[0] + h * a.vps[1] + p.row * a.vps[2];
      turn = false;
      if (j < half) {  // the two elements a pair of this index holds
        dst[j] = src[j];
        dst[j + half] = src[j + half];
        continue;
      }
    }
    const int x = turn ? (a.interleaved ? 2 * j : j) : j + half;
    if (!turn) {
      dst[x] = p.page < 0 ? store_f<T>(0.f) : src[x];
      continue;
    }
    const int y = a.interleaved ? x + 1 : x + half;
    float u = 0.f, v = 0.f;
    if (p.page >= 0) {
      const float c = a.cos[p.position * half + j], s = a.sin[p.position * half + j];
      const float fx = load_f<T>(src[x]), fy = load_f<T>(src[y]);
      u = fx * c - fy * s;
      v = fy * c + fx * s;
    }
    dst[x] = store_f<T>(u);
    dst[y] = store_f<T>(v);
  }
}

// 16 bytes of a row: their elements as pairs of fp32 numbers.
template <typename T> struct Piece;
template <> struct Piece<float> {
  static constexpr int N = 4;
  static __device__ __forceinline__ void get(const uint4& r, float (&x)[4]) {
    x[0] = __uint_as_float(r.x), x[1] = __uint_as_float(r.y), x[2] = __uint_as_float(r.z), x[3] = __uint_as_float(r.w);
  }
  static __device__ __forceinline__ uint4 put(const float (&x)[4]) {
    return make_uint4(__float_as_uint(x[0]), __float_as_uint(x[1]), __float_as_uint(x[2]), __float_as_uint(x[3]));
  }
};
template <> struct Piece<__nv_bfloat16> {
  static constexpr int N = 8;
  static __device__ __forceinline__ void get(const uint4& r, float (&x)[8]) {
    const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {  // a bf16 is the upper half of an fp32
      x[2 * i] = __uint_as_float(w[i] << 16);
      x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    }
  }
  static __device__ __forceinline__ uint32_t pair(float x, float y) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(x, y);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
  static __device__ __forceinline__ uint4 put(const float (&x)[8]) {
    return make_uint4(pair(x[0], x[1]), pair(x[2], x[3]), pair(x[4], x[5]), pair(x[6], x[7]));
  }
};
template <> struct Piece<__half> {
  static constexpr int N = 8;
  static __device__ __forceinline__ void get(const uint4& r, float (&x)[8]) {
    const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
      x[2 * i] = f.x;
      x[2 * i + 1] = f.y;
    }
  }
  static __device__ __forceinline__ uint32_t pair(float x, float y) {
    const __half2 h = __floats2half2_rn(x, y);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
  static __device__ __forceinline__ uint4 put(const float (&x)[8]) {
    return make_uint4(pair(x[0], x[1]), pair(x[2], x[3]), pair(x[4], x[5]), pair(x[6], x[7]));
  }
};

// x' = x c - y s, y' = y c + x s of the pairs of two 16-byte pieces of a row: element i of one with
// element i of the other, or neighbours within each.
template <typename T, bool INTERLEAVED, int N>
__device__ __forceinline__ void rotate(uint4& px, uint4& py, const float (&c)[N], const float (&s)[N]) {
  float x[N], y[N];
  Piece<T>::get(px, x);
  Piece<T>::get(py, y);
#pragma unroll
  for (int i = 0; i < N; ++i) {
    float& first = INTERLEAVED ? (i < N / 2 ? x[2 * i] : y[2 * i - N]) : x[i];
    float& second = INTERLEAVED ? (i < N / 2 ? x[2 * i + 1] : y[2 * i - N + 1]) : y[i];
    const float u = first, v = second;
    first = u * c[i] - v * s[i];
    second = v * c[i] + u * s[i];
  }
  px = Piece<T>::put(x);
  py = Piece<T>::put(y);
}

// CTA per token. A thread keeps one slice of the token's cos / sin row in registers and turns that
// pair of 16-byte pieces in kHeads heads at a time, all loaded before the first is stored; then the
// pieces that are copied. Needs 16-byte aligned rows and rotation_dim / 2 a multiple of 16 bytes.
// A token's work is two dependent rounds of loads (where it goes; its page, angles and rows), so
// the CTA is small and its registers are held to 64: 16 tokens of an SM (32 where a warp does for a
// token) are in such rounds at once.
// Memory bound where tokens are many: 8 prompts to 4001 tokens, 40 q / 8 KV heads x 128 in fp16,
// 113 to 116 us (0.94 or more of the copy bandwidth measured on this GPU; in fp32 219, 0.99); latency bound
// below: 64 x 61 rows of 16 / 2 heads 10.3 us (0.63), one row each of 256 sequences 6.6 us, the cost of the
// host call.
constexpr int kHeads = 3;

template <typename T, bool INTERLEAVED, int THREADS>
__global__ void __launch_bounds__(THREADS, 1024 / THREADS) paged_append_kernel(AppendArgs a) {
  constexpr int N = Piece<T>::N;
  const uint32_t b = blockIdx.x / (uint32_t)a.rows, t = blockIdx.x - b * (uint32_t)a.rows;
  const int q_heads = a.query != nullptr ? (int)a.q_heads : 0, kv_heads = (int)a.kv_heads, dim = (int)a.dim;
  const long long live = a.counts != nullptr ? a.counts[b] : a.rows, slot = a.starts[b] + t;
  const long long position = a.positions != nullptr ? a.positions[b * a.pos_b + t * a.pos_t] : slot;
  const T* q = static_cast<const T*>(a.query) + b * a.qs[0] + t * a.qs[2];
  T* qo = static_cast<T*>(a.query_out) + b * a.os[0] + t * a.os[2];
  bool stored = t < live;
  if (stored && (slot < 0 || slot >= a.table.width * a.table.page_size)) {
    record_error(a.err, SPECKV_DERR_PAGE_TABLE, slot);
    stored = false;
  }
  if (stored && a.cos != nullptr && (position < 0 || position >= a.rot_positions)) {
    record_error(a.err, SPECKV_DERR_ROTATION_INDEX, position);
    stored = false;
  }
  const uint32_t size = (uint32_t)a.table.page_size, index = stored ? (uint32_t)slot / size : 0u;
  const long long page = stored ? a.table.entries[b * a.table.stride + index] : 0;  // checked below

  const int half = a.rot / 2, slices = half / N;  // slices <= THREADS
  const T* k = static_cast<const T*>(a.key) + b * a.ks[0] + t * a.ks[2];
  const T* v = static_cast<const T*>(a.value) + b * a.vs[0] + t * a.vs[2];
  const int slice = slices > 0 ? threadIdx.x % slices : 0, h0 = slices > 0 ? threadIdx.x / slices : 0;
  const int step = slices > 0 ? THREADS / slices : 1, heads = slices > 0 && h0 < step ? q_heads + kv_heads : 0;
  const int x = INTERLEAVED ? 2 * slice * N : slice * N, y = INTERLEAVED ? x + N : x + half;
  uint4 px[kHeads], py[kHeads];
  auto load = [&](int h) {
#pragma unroll
    for (int i = 0; i < kHeads; ++i) {
      const int hi = h + i * step;
      if (hi < heads) {
        const T* row = hi < q_heads ? q + hi * a.qs[1] : k + (hi - q_heads) * a.ks[1];
        px[i] = *reinterpret_cast<const uint4*>(row + x);
        py[i] = *reinterpret_cast<const uint4*>(row + y);
      }
    }
  };
  float c[N], s[N];
  if (stored && heads > 0) {
    load(h0);
    const float4* cr = reinterpret_cast<const float4*>(a.cos + position * half + slice * N);
    const float4* sr = reinterpret_cast<const float4*>(a.sin + position * half + slice * N);
#pragma unroll
    for (int i = 0; i < N / 4; ++i) {
      const float4 cc = __ldg(cr + i), ss = __ldg(sr + i);
      c[4 * i] = cc.x, c[4 * i + 1] = cc.y, c[4 * i + 2] = cc.z, c[4 * i + 3] = cc.w;
      s[4 * i] = ss.x, s[4 * i + 1] = ss.y, s[4 * i + 2] = ss.z, s[4 * i + 3] = ss.w;
    }
  }
  if (stored && (page < 0 || page >= a.table.num_pages)) {
    record_error(a.err, SPECKV_DERR_PAGE_TABLE, page);
    stored = false;
  }
  if (!stored) {  // padding: its queries are zeros
    const int pieces = dim / N;
    for (int i = threadIdx.x; i < q_heads * pieces; i += THREADS)
      *reinterpret_cast<uint4*>(qo + (i / pieces) * a.os[1] + (i % pieces) * N) = make_uint4(0, 0, 0, 0);
    return;
  }
  const long long row = slot - (long long)index * size;
  T* kp = static_cast<T*>(a.key_pages) + page * a.kps[0] + row * a.kps[2];
  T* vp = static_cast<T*>(a.value_pages) + page * a.vps[0] + row * a.vps[2];
  for (int h = h0; h < heads; h += kHeads * step) {
    if (h != h0) load(h);
#pragma unroll
    for (int i = 0; i < kHeads; ++i) {
      const int hi = h + i * step;
      if (hi < heads) {
        T* to = hi < q_heads ? qo + hi * a.os[1] : kp + (hi - q_heads) * a.kps[1];
        rotate<T, INTERLEAVED>(px[i], py[i], c, s);
        *reinterpret_cast<uint4*>(to + x) = px[i];
        *reinterpret_cast<uint4*>(to + y) = py[i];
      }
    }
  }
  // V, then what lies past the rotation in K and Q
  const int whole = dim / N, rest = (dim - a.rot) / N;
  const int v_items = kv_heads * whole, items = v_items + (rest > 0 ? (q_heads + kv_heads) * rest : 0);
  for (int i = threadIdx.x; i < items; i += THREADS) {
    const T* from;
    T* to;
    if (i < v_items) {
      const int h = i / whole, e = (i - h * whole) * N;
      from = v + h * a.vs[1] + e;
      to = vp + h * a.vps[1] + e;
    } else {
      const int j = i - v_items, h = j / rest, e = a.rot + (j - h * rest) * N;
      from = h < q_heads ? q + h * a.qs[1] + e : k + (h - q_heads) * a.ks[1] + e;
      to = h < q_heads ? qo + h * a.os[1] + e : kp + (h - q_heads) * a.kps[1] + e;
    }
    *reinterpret_cast<uint4*>(to) = *reinterpret_cast<const uint4*>(from);
  }
}

// Whether every row begins on a 16-byte boundary and the rotation splits into whole pieces.
template <typename T> bool in_pieces(const AppendArgs& a) {
  const int64_t n = 16 / sizeof(T);
  bool ok = a.dim % n == 0 && a.rot / 2 % n == 0 && a.rot / 2 / n <= kAppendThreads;
  for (const void* p : {a.key, a.value, a.query, (const void*)a.query_out, (const void*)a.key_pages,
                        (const void*)a.value_pages, (const void*)a.cos, (const void*)a.sin})
    ok = ok && reinterpret_cast<uintptr_t>(p) % 16 == 0;
  for (int i = 0; i < 3; ++i)
    ok = ok && a.ks[i] % n == 0 && a.vs[i] % n == 0 && a.qs[i] % n == 0 && a.os[i] % n == 0 && a.kps[i] % n == 0 &&
         a.vps[i] % n == 0;
  return ok;
}

template <typename T, int THREADS> void launch_pieces(const AppendArgs& a, unsigned tokens, cudaStream_t s) {
  if (a.interleaved)
    paged_append_kernel<T, true, THREADS><<<tokens, THREADS, 0, s>>>(a);
  else
    paged_append_kernel<T, false, THREADS><<<tokens, THREADS, 0, s>>>(a);
}

template <typename T>
int launch_append(const AppendArgs& a, cudaStream_t s) {
  const unsigned tokens = (unsigned)(a.batch * a.rows);
  const int sms = sm_count();
  if (sms == 0) return fail(SPECKV_ECUDA, "speckv_paged_append: no SM count");
  // More tokens than CTAs of 64 run at once, and at most five pairs of pieces a lane: a warp does for a
  // token, twice as many are under way (16 q / 2 KV heads x 128 bf16, 64 x 61 rows 12.0 -> 10.3 us, 8 x 4001
  // 63.4 -> 57.5). With 28 / 4 heads, eight pairs a lane, it does not (64 x 61 rows 16.6 us, 17.4).
  const int64_t slices = a.rot / 2 * (int64_t)sizeof(T) / 16, heads = a.kv_heads + (a.query != nullptr ? a.q_heads : 0);
  if (!in_pieces<T>(a))
    paged_append_scalar_kernel<T><<<tokens, kAppendThreads, 0, s>>>(a);
  else if (tokens > 16u * (unsigned)sms && slices > 0 && slices <= 32 && slices * heads <= 5 * 32)
    launch_pieces<T, 32>(a, tokens, s);
  else
    launch_pieces<T, kAppendThreads>(a, tokens, s);
  return check_launch("speckv_paged_append");
}

}  // namespace
}  // namespace speckv

using namespace speckv;

extern "C" int speckv_paged_append(const void* key, const void* value, const void* query, void* query_out,
                                   void* key_pages, void* value_pages, const int64_t* strides,
                                   const int64_t* page_table, int64_t table_stride, int64_t table_pages,
                                   int64_t num_pages, int64_t page_size, const int64_t* starts,
                                   const int64_t* counts, const int64_t* positions, int64_t positions_stride_b,
                                   int64_t positions_stride_t, const float* cos, const float* sin,
                                   int64_t rotation_positions, int64_t rotation_dim, int32_t interleaved,
                                   int64_t batch, int64_t q_heads, int64_t kv_heads, int64_t rows, int64_t dim,
                                   int32_t dtype, void* stream) {
  const char* fn = "speckv_paged_append";
  if (batch < 0 || rows < 0 || kv_heads < 1 || dim < 1 || dim > 1024 || kv_heads > 65535)
    return fail(SPECKV_EINVAL, "%s: bad sizes", fn);
  if (dtype != SPECKV_F32 && dtype != SPECKV_BF16 && dtype != SPECKV_F16)
    return fail(SPECKV_EINVAL, "%s: unsupported dtype %d", fn, dtype);
  if (query != nullptr && (q_heads < 1 || q_heads > 65535 || query_out == nullptr))
    return fail(SPECKV_EINVAL, "%s: query without heads or output", fn);
  if ((cos == nullptr) != (sin == nullptr)) return fail(SPECKV_EINVAL, "%s: cos and sin come together", fn);
  if (cos != nullptr && (rotation_dim < 2 || rotation_dim % 2 || rotation_dim > dim || rotation_positions < 1))
    return fail(SPECKV_EINVAL, "%s: rotation of %lld of %lld dims over %lld positions", fn, (long long)rotation_dim,
                (long long)dim, (long long)rotation_positions);
  if (interleaved < 0 || interleaved > 1) return fail(SPECKV_EINVAL, "%s: interleaved is 0 or 1", fn);
  int st = check_pages(fn, page_table, table_stride, table_pages, num_pages, page_size, batch);
  if (st) return st;
  if (batch == 0 || rows == 0) return SPECKV_OK;
  if (batch > (1ll << 31) || rows > (1ll << 31) || batch * rows >= (1ll << 31))
    return fail(SPECKV_ENOSUPPORT, "%s: 2^31 tokens or more", fn);
  if (!key || !value || !key_pages || !value_pages || !strides || !starts)
    return fail(SPECKV_EINVAL, "%s: null pointer", fn);
  st = check_strides(fn, strides, 18);
  if (st) return st;
  st = check_current_device(fn, {key, key_pages, page_table, query_out});
  if (st) return st;
  AppendArgs a;
  a.key = key;
  a.value = value;
  a.query = query;
  a.query_out = query_out;
  a.key_pages = key_pages;
  a.value_pages = value_pages;
  for (int i = 0; i < 3; ++i) {
    a.ks[i] = strides[i];
    a.vs[i] = strides[3 + i];
    a.qs[i] = strides[6 + i];
    a.os[i] = strides[9 + i];
    a.kps[i] = strides[12 + i];
    a.vps[i] = strides[15 + i];
  }
  drop_unused_strides(a.ks, {batch, kv_heads, rows});
  drop_unused_strides(a.vs, {batch, kv_heads, rows});
  drop_unused_strides(a.qs, {batch, q_heads, rows});
  drop_unused_strides(a.os, {batch, q_heads, rows});
  drop_unused_strides(a.kps, {num_pages, kv_heads, page_size});
  drop_unused_strides(a.vps, {num_pages, kv_heads, page_size});
  a.table = {page_table, table_stride, table_pages, num_pages, page_size};
  a.starts = starts;
  a.counts = counts;
  a.positions = positions;
  a.pos_b = positions_stride_b;
  a.pos_t = positions_stride_t;
  a.cos = cos;
  a.sin = sin;
  a.rot_positions = rotation_positions;
  a.rot = cos != nullptr ? (int)rotation_dim : 0;
  a.interleaved = interleaved;
  a.batch = batch;
  a.q_heads = q_heads;
  a.kv_heads = kv_heads;
  a.rows = rows;
  a.dim = dim;
  a.err = device_error_word();
  if (a.err == nullptr) return fail(SPECKV_ECUDA, "%s: no error word on device", fn);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  switch (dtype) {
    case SPECKV_F32: return launch_append<float>(a, s);
    case SPECKV_BF16: return launch_append<__nv_bfloat16>(a, s);
    default: return launch_append<__half>(a, s);
  }
}
