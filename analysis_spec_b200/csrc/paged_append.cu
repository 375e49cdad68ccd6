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

constexpr int kAppendThreads = 128;

// One CTA per token; elements one by one: any head dim, rotation width, stride and alignment.
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

// 16 bytes of rows: N elements.
template <typename T> struct Pack {
  static constexpr int N = 16 / sizeof(T);
  union {
    uint4 raw;
    T e[N];
  };
};

// x' = x c - y s, y' = y c + x s of the pairs of two 16-byte pieces of a row: element i of one with
// element i of the other, or neighbours within each.
template <typename T, bool INTERLEAVED>
__device__ __forceinline__ void rotate(Pack<T>& x, Pack<T>& y, const float (&c)[Pack<T>::N],
                                       const float (&s)[Pack<T>::N]) {
  constexpr int N = Pack<T>::N;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    T& first = INTERLEAVED ? (i < N / 2 ? x.e[2 * i] : y.e[2 * i - N]) : x.e[i];
    T& second = INTERLEAVED ? (i < N / 2 ? x.e[2 * i + 1] : y.e[2 * i - N + 1]) : y.e[i];
    const float u = load_f<T>(first), v = load_f<T>(second);
    first = store_f<T>(u * c[i] - v * s[i]);
    second = store_f<T>(v * c[i] + u * s[i]);
  }
}

// CTA per token. A thread keeps one slice of the token's cos / sin row in registers and turns that
// pair of 16-byte pieces in kHeads heads at a time, all loaded before the first is stored; then the
// pieces that are copied. Needs 16-byte aligned rows and rotation_dim / 2 a multiple of 16 bytes.
constexpr int kHeads = 4;

template <typename T, bool INTERLEAVED>
__global__ void __launch_bounds__(kAppendThreads) paged_append_kernel(AppendArgs a) {
  constexpr int N = Pack<T>::N;
  const uint32_t b = blockIdx.x / (uint32_t)a.rows, t = blockIdx.x - b * (uint32_t)a.rows;
  const Place p = place_token(a, b, t);
  const int q_heads = a.query != nullptr ? (int)a.q_heads : 0, kv_heads = (int)a.kv_heads, dim = (int)a.dim;
  const T* q = static_cast<const T*>(a.query) + b * a.qs[0] + t * a.qs[2];
  T* qo = static_cast<T*>(a.query_out) + b * a.os[0] + t * a.os[2];
  if (p.page < 0) {  // padding: its queries are zeros
    const int pieces = dim / N;
    for (int i = threadIdx.x; i < q_heads * pieces; i += kAppendThreads)
      *reinterpret_cast<uint4*>(qo + (i / pieces) * a.os[1] + (i % pieces) * N) = make_uint4(0, 0, 0, 0);
    return;
  }
  const T* k = static_cast<const T*>(a.key) + b * a.ks[0] + t * a.ks[2];
  const T* v = static_cast<const T*>(a.value) + b * a.vs[0] + t * a.vs[2];
  T* kp = static_cast<T*>(a.key_pages) + p.page * a.kps[0] + p.row * a.kps[2];
  T* vp = static_cast<T*>(a.value_pages) + p.page * a.vps[0] + p.row * a.vps[2];

  const int half = a.rot / 2, slices = half / N;  // slices <= 128
  if (slices > 0) {
    const int slice = threadIdx.x % slices, h0 = threadIdx.x / slices, step = kAppendThreads / slices;
    if (h0 < step) {
      const int x = INTERLEAVED ? 2 * slice * N : slice * N, y = INTERLEAVED ? x + N : x + half;
      float c[N], s[N];
      const float4* cr = reinterpret_cast<const float4*>(a.cos + p.position * half + slice * N);
      const float4* sr = reinterpret_cast<const float4*>(a.sin + p.position * half + slice * N);
#pragma unroll
      for (int i = 0; i < N / 4; ++i) {
        const float4 cc = __ldg(cr + i), ss = __ldg(sr + i);
        c[4 * i] = cc.x, c[4 * i + 1] = cc.y, c[4 * i + 2] = cc.z, c[4 * i + 3] = cc.w;
        s[4 * i] = ss.x, s[4 * i + 1] = ss.y, s[4 * i + 2] = ss.z, s[4 * i + 3] = ss.w;
      }
      const int heads = q_heads + kv_heads;
      for (int h = h0; h < heads; h += kHeads * step) {
        Pack<T> px[kHeads], py[kHeads];
#pragma unroll
        for (int i = 0; i < kHeads; ++i) {
          const int hi = h + i * step;
          if (hi < heads) {
            const T* row = hi < q_heads ? q + hi * a.qs[1] : k + (hi - q_heads) * a.ks[1];
            px[i].raw = *reinterpret_cast<const uint4*>(row + x);
            py[i].raw = *reinterpret_cast<const uint4*>(row + y);
          }
        }
#pragma unroll
        for (int i = 0; i < kHeads; ++i) {
          const int hi = h + i * step;
          if (hi < heads) {
            T* row = hi < q_heads ? qo + hi * a.os[1] : kp + (hi - q_heads) * a.kps[1];
            rotate<T, INTERLEAVED>(px[i], py[i], c, s);
            *reinterpret_cast<uint4*>(row + x) = px[i].raw;
            *reinterpret_cast<uint4*>(row + y) = py[i].raw;
          }
        }
      }
    }
  }
  // V, then what lies past the rotation in K and Q
  const int whole = dim / N, rest = (dim - a.rot) / N;
  const int v_items = kv_heads * whole, items = v_items + (rest > 0 ? (q_heads + kv_heads) * rest : 0);
  for (int i = threadIdx.x; i < items; i += kAppendThreads) {
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

template <typename T>
int launch_append(const AppendArgs& a, cudaStream_t s) {
  const unsigned tokens = (unsigned)(a.batch * a.rows);
  if (!in_pieces<T>(a))
    paged_append_scalar_kernel<T><<<tokens, kAppendThreads, 0, s>>>(a);
  else if (a.interleaved)
    paged_append_kernel<T, true><<<tokens, kAppendThreads, 0, s>>>(a);
  else
    paged_append_kernel<T, false><<<tokens, kAppendThreads, 0, s>>>(a);
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
