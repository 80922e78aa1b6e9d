// kv8_cache.hip -- the paged 8-bit K/V cache: quantize-on-write and reading back.
#include "kv8.hpp"

#include <algorithm>

namespace csahca {
namespace {

constexpr int kThreads = 256;

// ---------------------------------------------------------------------------
// Write
// ---------------------------------------------------------------------------
template <typename T>
struct WriteArgs {
  const T* x[2];
  int64_t sb[2], sh[2], sn[2];
  Kv8Cache c;
  const int32_t* start;
  const int32_t* counts;
  int32_t pages_per;  // pages that new_tokens can touch
  int32_t new_tokens;
};

// N consecutive elements as they are stored; kVec: at an address of N * sizeof(T).
template <typename T, int N>
struct Packed {
  static constexpr int kWords = N * sizeof(T) / 4;
  uint32_t w[kWords];
  template <bool kVec>
  __device__ __forceinline__ void load(const T* p) {
    if constexpr (kVec) {
      constexpr int kPer = kWords < 4 ? kWords : 4;
      using V = uint32_t __attribute__((ext_vector_type(kPer)));
#pragma unroll
      for (int i = 0; i < kWords; i += kPer) {
        const V v = load_global_raw<V>(reinterpret_cast<const uint32_t*>(p) + i);
        __builtin_memcpy(w + i, &v, sizeof(V));
      }
    } else {
      T e[N];
#pragma unroll
      for (int i = 0; i < N; ++i) e[i] = load_global_elem(p + i);
      __builtin_memcpy(w, e, sizeof(w));
    }
  }
  __device__ __forceinline__ float at(int i) const {
    if constexpr (sizeof(T) == 4) {
      return __uint_as_float(w[i]);
    } else {
      const uint32_t half = i % 2 ? w[i / 2] >> 16 : w[i / 2] & 0xffffu;
      if constexpr (std::is_same_v<T, bf16>) return __uint_as_float(i % 2 ? w[i / 2] & 0xffff0000u : half << 16);
      return static_cast<float>(__builtin_bit_cast(_Float16, static_cast<uint16_t>(half)));
    }
  }
  // max(m, the finite magnitudes)
  __device__ __forceinline__ float max_finite(float m) const {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const float v = fabsf(at(i));
      m = fmaxf(m, v < __builtin_inff() ? v : 0.f);
    }
    return m;
  }
};

// Four values to four bytes.
template <typename F>
__device__ __forceinline__ uint32_t encode4(float a, float b, float c, float d) {
  const float x[4] = {a, b, c, d};
  float y[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    y[i] = fminf(fmaxf(x[i], -F::kMax), F::kMax);
    if constexpr (std::is_same_v<F, E4m3>) y[i] = x[i] != x[i] ? x[i] : y[i];
    else y[i] = x[i] != x[i] ? 0.f : rintf(y[i]);
  }
  if constexpr (std::is_same_v<F, E4m3>) {
    const int lo = __builtin_amdgcn_cvt_pk_fp8_f32(y[0], y[1], 0, false);
    return static_cast<uint32_t>(__builtin_amdgcn_cvt_pk_fp8_f32(y[2], y[3], lo, true));
  } else {
    return (static_cast<uint32_t>(static_cast<int>(y[0])) & 0xffu) |
           (static_cast<uint32_t>(static_cast<int>(y[1])) & 0xffu) << 8 |
           (static_cast<uint32_t>(static_cast<int>(y[2])) & 0xffu) << 16 |
           static_cast<uint32_t>(static_cast<int>(y[3])) << 24;
  }
}

// Four stored bytes rounded anew at a larger scale.
template <typename F>
__device__ __forceinline__ uint32_t rescale4(uint32_t w, float ratio) {
  return encode4<F>(kv8_decode<F, 0>(w) * ratio, kv8_decode<F, 1>(w) * ratio, kv8_decode<F, 2>(w) * ratio,
                    kv8_decode<F, 3>(w) * ratio);
}

// Where a workgroup's page lies among its sequence's new tokens.
struct Span {
  int32_t page;   // physical; -1: nothing to write
  int32_t lo, hi; // rows that get new tokens; those before lo are live
  int64_t token;  // new token of row lo
};

template <typename T>
__device__ __forceinline__ Span span_of(const WriteArgs<T>& a, int64_t b, int32_t j) {
  const Kv8Cache& c = a.c;
  const int64_t start = a.start[b];
  const int64_t count = a.counts ? min(max(a.counts[b], 0), a.new_tokens) : a.new_tokens;
  Span s{-1, 0, 0, 0};
  if (start < 0) return s;
  const int64_t block = static_cast<uint32_t>(start) / static_cast<uint32_t>(c.page_size) + j;
  const int64_t first = block * c.page_size;
  s.lo = static_cast<int32_t>(max(start - first, static_cast<int64_t>(0)));
  s.hi = static_cast<int32_t>(min(start + count - first, static_cast<int64_t>(c.page_size)));
  s.token = first + s.lo - start;
  if (s.hi > s.lo) s.page = kv8_page(c, b, block);
  return s;
}

// The scale of a tile whose new values reach amax (in every thread), and where
// it grew, old / new (else 0).
template <typename F>
__device__ __forceinline__ float new_scale(float amax, int lo, const float* scale, float* ratio) {
  const float s = kv8_scale_for<F>(amax);
  *ratio = 0.f;
  if (lo == 0) return s;
  const float old = *scale;
  if (!(s > old)) return old;
  *ratio = old / s;
  return s;
}

__device__ __forceinline__ float group_max(float v, float* lds) {
#pragma unroll
  for (int off = 32; off >= 1; off >>= 1) v = fmaxf(v, xor_lanes(v, off));
  if (blockDim.x == kWave) return v;
  if (threadIdx.x % kWave == 0) lds[threadIdx.x / kWave] = v;
  __syncthreads();
  for (int i = 0; i < kThreads / kWave; ++i) v = fmaxf(v, lds[i]);
  return v;
}

// K: eight dimensions of a row at a time.
template <typename T, typename F, bool kVec>
__device__ __forceinline__ void write_k(const WriteArgs<T>& a, int64_t b, int32_t h, const Span s, float* lds) {
  constexpr int kKept = 4;  // of a thread's pieces, those that stay in registers between the two passes
  const int D8 = a.c.head_dim / 8, n = (s.hi - s.lo) * D8;
  const T* x = a.x[0] + b * a.sb[0] + h * a.sh[0] + s.token * a.sn[0];
  uint8_t* tile = a.c.k + kv8_tile(a.c, s.page, h);
  float* scale = a.c.k_scale + static_cast<int64_t>(s.page) * a.c.kv_heads + h;
  const auto fetch = [&](int i) {
    Packed<T, 8> p;
    const uint32_t row = static_cast<uint32_t>(i) / static_cast<uint32_t>(D8);
    p.template load<kVec>(x + row * a.sn[0] + (i - row * D8) * 8);
    return p;
  };
  Packed<T, 8> kept[kKept];
  float amax = 0.f;
#pragma unroll
  for (int k = 0; k < kKept; ++k) {
    const int i = threadIdx.x + k * blockDim.x;
    if (i < n) kept[k] = fetch(i);
  }
#pragma unroll
  for (int k = 0; k < kKept; ++k)
    if (threadIdx.x + k * blockDim.x < n) amax = kept[k].max_finite(amax);
  for (int i = threadIdx.x + kKept * blockDim.x; i < n; i += blockDim.x) amax = fetch(i).max_finite(amax);
  amax = group_max(amax, lds);
  float ratio;
  const float sc = new_scale<F>(amax, s.lo, scale, &ratio), inv = 1.0f / sc;
  if (ratio > 0.f) {
    for (int i = threadIdx.x; i < s.lo * D8; i += blockDim.x) {
      uint2* p = reinterpret_cast<uint2*>(tile) + i;
      const uint2 w = *p;
      *p = make_uint2(rescale4<F>(w.x, ratio), rescale4<F>(w.y, ratio));
    }
  }
  uint2* out = reinterpret_cast<uint2*>(tile) + s.lo * D8;
  const auto put = [&](int i, const Packed<T, 8>& p) {
    out[i] = make_uint2(encode4<F>(p.at(0) * inv, p.at(1) * inv, p.at(2) * inv, p.at(3) * inv),
                        encode4<F>(p.at(4) * inv, p.at(5) * inv, p.at(6) * inv, p.at(7) * inv));
  };
#pragma unroll
  for (int k = 0; k < kKept; ++k) {
    const int i = threadIdx.x + k * blockDim.x;
    if (i < n) put(i, kept[k]);
  }
  for (int i = threadIdx.x + kKept * blockDim.x; i < n; i += blockDim.x) put(i, fetch(i));
  if (blockDim.x > kWave) __syncthreads();  // every thread has read the old scale
  if (threadIdx.x == 0) *scale = sc;
}

// V: two dimensions of a group of 16 tokens at a time, which are 32 bytes.
template <typename T, typename F, bool kVec>
__device__ __forceinline__ void write_v(const WriteArgs<T>& a, int64_t b, int32_t h, const Span s, float* lds) {
  const int D2 = a.c.head_dim / 2, g0 = s.lo / kKv8Group, g1 = (s.hi + kKv8Group - 1) / kKv8Group, n = (g1 - g0) * D2;
  const T* x = a.x[1] + b * a.sb[1] + h * a.sh[1] + s.token * a.sn[1];
  uint8_t* tile = a.c.v + kv8_tile(a.c, s.page, h);
  float* scale = a.c.v_scale + static_cast<int64_t>(s.page) * a.c.kv_heads + h;
  struct Piece {
    Packed<T, 2> t[kKv8Group];
  };
  // Piece i: rows outside [lo, hi) repeat the nearest one inside.
  const auto fetch = [&](int i) {
    Piece p;
    const int g = static_cast<uint32_t>(i) / static_cast<uint32_t>(D2), d = (i - g * D2) * 2;
#pragma unroll
    for (int t = 0; t < kKv8Group; ++t) {
      const int row = min(max((g0 + g) * kKv8Group + t, s.lo), s.hi - 1);
      p.t[t].template load<kVec>(x + (row - s.lo) * a.sn[1] + d);
    }
    return p;
  };
  const auto most = [&](const Piece& p, float m) {
#pragma unroll
    for (int t = 0; t < kKv8Group; ++t) m = p.t[t].max_finite(m);
    return m;
  };
  Piece kept;
  float amax = 0.f;
  if (threadIdx.x < n) {
    kept = fetch(threadIdx.x);
    amax = most(kept, amax);
  }
  for (int i = threadIdx.x + blockDim.x; i < n; i += blockDim.x) amax = most(fetch(i), amax);
  amax = group_max(amax, lds);
  float ratio;
  const float sc = new_scale<F>(amax, s.lo, scale, &ratio), inv = 1.0f / sc;
  uint4* out = reinterpret_cast<uint4*>(tile);
  if (ratio > 0.f) {  // groups of live tokens alone
    for (int i = threadIdx.x; i < g0 * a.c.head_dim; i += blockDim.x) {
      const uint4 w = out[i];
      out[i] = make_uint4(rescale4<F>(w.x, ratio), rescale4<F>(w.y, ratio), rescale4<F>(w.z, ratio),
                          rescale4<F>(w.w, ratio));
    }
  }
  const auto put = [&](int i, const Piece& p) {
    const int g = static_cast<uint32_t>(i) / static_cast<uint32_t>(D2), d = (i - g * D2) * 2;
    const int first = (g0 + g) * kKv8Group;
    uint4* at = out + (g0 + g) * a.c.head_dim + d;
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      uint32_t w[4];
#pragma unroll
      for (int k = 0; k < 4; ++k)
        w[k] = encode4<F>(p.t[4 * k].at(e) * inv, p.t[4 * k + 1].at(e) * inv, p.t[4 * k + 2].at(e) * inv,
                          p.t[4 * k + 3].at(e) * inv);
      if (first < s.lo || first + kKv8Group > s.hi) {  // tokens before and behind keep their bytes, or are rescaled
        const uint4 o = at[e];
        const uint32_t old[4] = {o.x, o.y, o.z, o.w};
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          uint32_t fresh = 0, live = 0;
#pragma unroll
          for (int t = 0; t < 4; ++t) {
            const int row = first + 4 * k + t;
            fresh |= row >= s.lo && row < s.hi ? 0xffu << (8 * t) : 0u;
            live |= row < s.lo ? 0xffu << (8 * t) : 0u;
          }
          uint32_t was = old[k];
          if (ratio > 0.f) was = (rescale4<F>(was, ratio) & live) | (was & ~live);
          w[k] = (w[k] & fresh) | (was & ~fresh);
        }
      }
      at[e] = make_uint4(w[0], w[1], w[2], w[3]);
    }
  };
  if (threadIdx.x < n) put(threadIdx.x, kept);
  for (int i = threadIdx.x + blockDim.x; i < n; i += blockDim.x) put(i, fetch(i));
  if (blockDim.x > kWave) __syncthreads();  // every thread has read the old scale
  if (threadIdx.x == 0) *scale = sc;
}

// One workgroup (or, for few tokens, wavefront) owns K or V of one (sequence,
// page, head): the largest new value, the scale, and the bytes, with the values
// kept in registers between (a 64 x 128 page whole; of larger ones the rest is
// read again).  Nothing that it reads or writes is another's, so no order between
// workgroups shows in the result.  Bound by memory: 4 x 8192 tokens, 8 heads of 128
// in bf16, 201 MB, 41.3 us (4.9 TB/s, as a copy); reading one value a thread twice
// took 165.  32 single tokens 4.5 us, the latency of three dependent loads.
template <typename T, typename F, bool kVec>
__global__ __launch_bounds__(kThreads) void kv8_write_kernel(const WriteArgs<T> a) {
  __shared__ float lds[kThreads / kWave];
  uint32_t i = blockIdx.x;
  const uint32_t h = i % a.c.kv_heads;
  i /= a.c.kv_heads;
  const bool v = i & 1;
  i /= 2;
  const int32_t j = i % a.pages_per;
  const int64_t b = i / a.pages_per;
  const Span s = span_of(a, b, j);
  if (s.page < 0) return;
  if (v) {
    write_v<T, F, kVec>(a, b, h, s, lds);
  } else {
    write_k<T, F, kVec>(a, b, h, s, lds);
  }
}

// ---------------------------------------------------------------------------
// Read
// ---------------------------------------------------------------------------
template <typename T>
struct ReadArgs {
  Kv8Cache c;
  const int32_t* start;
  const int32_t* lengths;
  T* out[2];
  int32_t max_tokens;
  int32_t groups;  // aligned groups of 16 positions that a sequence's span can touch
  uint32_t threads;
};

// 16 bytes of values; kStream: past the caches.
template <typename T, int N, bool kStream>
__device__ __forceinline__ void store_vec(T* p, const float* v) {
  uint32_t w[N * sizeof(T) / 4];
  static_assert(sizeof(w) == 16, "16-byte stores");
  if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int i = 0; i < N; ++i) w[i] = __float_as_uint(v[i]);
  } else {
#pragma unroll
    for (int i = 0; i < N; i += 2) {
      const T a = from_f32<T>(v[i]), b = from_f32<T>(v[i + 1]);
      w[i / 2] = __builtin_bit_cast(uint16_t, a) | static_cast<uint32_t>(__builtin_bit_cast(uint16_t, b)) << 16;
    }
  }
  const u32x4_t out = {w[0], w[1], w[2], w[3]};
  if constexpr (kStream) {
    __builtin_nontemporal_store(out, reinterpret_cast<u32x4_t*>(p));
  } else {
    *reinterpret_cast<u32x4_t*>(p) = out;
  }
}

// A thread reads N dimensions (16 bytes of output) of a group of 16 positions,
// K and V: both are 16 N bytes, V already in the order of a row once its bytes
// are taken across.  All 32 N bytes are in flight before any is used.  Bound by
// memory: 4 x 8192 tokens, 8 heads of 128 to bf16, 201 MB, 45.2 us, 42.6 with
// streaming stores (4.7 TB/s; a copy reaches 4.9).
template <typename T, typename F, bool kStream>
__global__ __launch_bounds__(kThreads) void kv8_read_kernel(const ReadArgs<T> a) {
  constexpr int N = 16 / sizeof(T);
  const Kv8Cache& c = a.c;
  const uint32_t at = blockIdx.x * kThreads + threadIdx.x;
  if (at >= a.threads) return;
  const uint32_t per = c.head_dim / N, unit = at / per;
  const int d = (at - unit * per) * N;
  const uint32_t bh = unit / a.groups, b = bh / c.kv_heads;
  const int32_t h = bh - b * c.kv_heads;
  const int64_t start = a.start ? a.start[b] : 0;
  // groups are counted from the one that holds position `start` (which may be negative)
  const int64_t first = (start & ~static_cast<int64_t>(kKv8Group - 1)) + static_cast<int64_t>(unit - bh * a.groups) * kKv8Group;
  const int64_t row = first - start;  // output row of the group's first position
  if (row >= a.max_tokens) return;
  const int64_t len = a.lengths[b];
  int32_t page = -1;
  if (first >= 0 && first < len) page = kv8_page(c, b, first / c.page_size);
  float ks = 0.f, vs = 0.f;
  uint32_t kw[kKv8Group][N / 4], vw[N][4];
#pragma unroll
  for (int t = 0; t < kKv8Group; ++t)
#pragma unroll
    for (int i = 0; i < N / 4; ++i) kw[t][i] = 0;
#pragma unroll
  for (int e = 0; e < N; ++e)
#pragma unroll
    for (int i = 0; i < 4; ++i) vw[e][i] = 0;
  if (page >= 0) {
    const int64_t tile = static_cast<int64_t>(page) * c.kv_heads + h;
    const int64_t off = (tile * c.page_size + first % c.page_size) * c.head_dim;
    ks = c.k_scale[tile];
    vs = c.v_scale[tile];
    const uint8_t* k = c.k + off + d;
    const uint8_t* v = c.v + off + d * kKv8Group;
#pragma unroll
    for (int t = 0; t < kKv8Group; ++t)
#pragma unroll
      for (int i = 0; i < N / 4; ++i) kw[t][i] = *reinterpret_cast<const uint32_t*>(k + t * c.head_dim + 4 * i);
#pragma unroll
    for (int e = 0; e < N; ++e) {
      const uint4 w = *reinterpret_cast<const uint4*>(v + e * kKv8Group);
      vw[e][0] = w.x;
      vw[e][1] = w.y;
      vw[e][2] = w.z;
      vw[e][3] = w.w;
    }
  }
#pragma unroll
  for (int t = 0; t < kKv8Group; ++t) {
    if (row + t < 0 || row + t >= a.max_tokens) continue;
    const bool in = page >= 0 && first + t < len;
    float x[N], y[N];
#pragma unroll
    for (int e = 0; e < N; ++e) {
      x[e] = in ? kv8_decode<F, 0>(kw[t][e / 4] >> (8 * (e % 4))) * ks : 0.f;
      y[e] = in ? kv8_decode<F, 0>(vw[e][t / 4] >> (8 * (t % 4))) * vs : 0.f;
    }
    const int64_t to = (static_cast<int64_t>(bh) * a.max_tokens + row + t) * c.head_dim + d;
    store_vec<T, N, kStream>(a.out[0] + to, x);
    store_vec<T, N, kStream>(a.out[1] + to, y);
  }
}

}  // namespace
}  // namespace csahca

using namespace csahca;

extern "C" int csahca_kv8_write(const void* k, const void* v, int dtype, int64_t k_stride_batch,
                                int64_t k_stride_head, int64_t k_stride_token, int64_t v_stride_batch,
                                int64_t v_stride_head, int64_t v_stride_token, void* k_cache, void* v_cache,
                                float* k_scale, float* v_scale, int format, int64_t num_pages, int64_t page_size,
                                const int32_t* block_table, int64_t blocks, int64_t table_stride,
                                const int32_t* start, const int32_t* counts, int64_t batch, int64_t kv_heads,
                                int64_t new_tokens, int64_t head_dim, void* stream) {
  clear_error();
  CSAHCA_REQUIRE(kv8_value_dtype(dtype), "unsupported dtype");
  CSAHCA_REQUIRE(batch >= 0 && new_tokens >= 0, "negative dimension");
  Kv8Cache c{static_cast<uint8_t*>(k_cache), static_cast<uint8_t*>(v_cache), k_scale, v_scale, block_table, table_stride,
             static_cast<int32_t>(num_pages), static_cast<int32_t>(blocks), static_cast<int32_t>(page_size),
             static_cast<int32_t>(kv_heads), static_cast<int32_t>(head_dim)};
  if (const int rc = kv8_check_cache(c, format, num_pages, blocks, page_size, kv_heads, head_dim)) return rc;
  CSAHCA_REQUIRE(batch <= INT32_MAX && new_tokens <= INT32_MAX, "too many tokens in one call");
  if (batch == 0 || kv_heads == 0 || new_tokens == 0 || num_pages == 0 || blocks == 0) return CSAHCA_OK;
  if (const int rc = kv8_check_pointers(c)) return rc;
  CSAHCA_REQUIRE(k && v && start, "null tensor pointer");
  const int64_t pages_per = (new_tokens + page_size - 2) / page_size + 1;
  CSAHCA_REQUIRE(batch * pages_per <= UINT32_MAX / kThreads / (2 * kv_heads), "too many tokens in one call");
  const int64_t grid = 2 * kv_heads * pages_per * batch;
  return dispatch_kv8_dtype(dtype, [&](auto tag) {
    using T = decltype(tag);
    return dispatch_kv8(format, [&](auto fmt) {
      using F = decltype(fmt);
      WriteArgs<T> a{{static_cast<const T*>(k), static_cast<const T*>(v)},
                     {k_stride_batch, v_stride_batch},
                     {k_stride_head, v_stride_head},
                     {k_stride_token, v_stride_token},
                     c,
                     start,
                     counts,
                     static_cast<int32_t>(pages_per),
                     static_cast<int32_t>(new_tokens)};
      // Eight K values and two V values a load, where every row begins on such a border.
      const auto whole = [](const void* p, int64_t n, int64_t s0, int64_t s1, int64_t s2) {
        return reinterpret_cast<uintptr_t>(p) % std::min<size_t>(16, n * sizeof(T)) == 0 && s0 % n == 0 && s1 % n == 0 &&
               s2 % n == 0;
      };
      const bool vec = whole(k, 8, k_stride_batch, k_stride_head, k_stride_token) &&
                       whole(v, 2, v_stride_batch, v_stride_head, v_stride_token);
      // A wavefront alone needs no barrier (32 sequences' single tokens 5.3 us, in four 6.0),
      // but a page takes several (64 tokens 9.2 us in one, 4.5 in four).
      const dim3 threads(std::min(new_tokens, page_size) * head_dim <= 2048 ? kWave : kThreads);
      return launch("kv8_write_kernel", vec ? kv8_write_kernel<T, F, true> : kv8_write_kernel<T, F, false>,
                    dim3(static_cast<uint32_t>(grid)), threads, 0, static_cast<hipStream_t>(stream), a);
    });
  });
}

extern "C" int csahca_kv8_read(const void* k_cache, const void* v_cache, const float* k_scale, const float* v_scale,
                               int format, int64_t num_pages, int64_t page_size, const int32_t* block_table,
                               int64_t blocks, int64_t table_stride, const int32_t* start, const int32_t* lengths,
                               void* k_out, void* v_out, int dtype, int64_t batch, int64_t kv_heads,
                               int64_t max_tokens, int64_t head_dim, void* stream) {
  clear_error();
  CSAHCA_REQUIRE(kv8_value_dtype(dtype), "unsupported dtype");
  CSAHCA_REQUIRE(batch >= 0 && max_tokens >= 0, "negative dimension");
  Kv8Cache c{static_cast<uint8_t*>(const_cast<void*>(k_cache)), static_cast<uint8_t*>(const_cast<void*>(v_cache)),
             const_cast<float*>(k_scale), const_cast<float*>(v_scale), block_table, table_stride,
             static_cast<int32_t>(num_pages), static_cast<int32_t>(blocks), static_cast<int32_t>(page_size),
             static_cast<int32_t>(kv_heads), static_cast<int32_t>(head_dim)};
  if (const int rc = kv8_check_cache(c, format, num_pages, blocks, page_size, kv_heads, head_dim)) return rc;
  CSAHCA_REQUIRE(batch <= INT32_MAX && max_tokens <= INT32_MAX, "too many tokens in one call");
  if (batch == 0 || kv_heads == 0 || max_tokens == 0) return CSAHCA_OK;
  CSAHCA_REQUIRE(k_out && v_out && lengths, "null tensor pointer");
  if (num_pages == 0) c.blocks = 0;  // an empty pool reads as zeros
  if (c.blocks > 0) {
    if (const int rc = kv8_check_pointers(c)) return rc;
  }
  CSAHCA_REQUIRE(reinterpret_cast<uintptr_t>(k_out) % 16 == 0 && reinterpret_cast<uintptr_t>(v_out) % 16 == 0,
                 "outputs must be 16-byte aligned");
  const int64_t groups = ceil_div(max_tokens, kKv8Group) + (start ? 1 : 0);
  const int64_t per = head_dim / (dtype == CSAHCA_F32 ? 4 : 8);
  CSAHCA_REQUIRE(batch <= UINT32_MAX / kv_heads && batch * kv_heads <= UINT32_MAX / 2 / per / groups,
                 "too many tokens in one call");
  const int64_t threads = batch * kv_heads * groups * per;
  return dispatch_kv8_dtype(dtype, [&](auto tag) {
    using T = decltype(tag);
    return dispatch_kv8(format, [&](auto fmt) {
      using F = decltype(fmt);
      // Outputs that the caches (8 x 4 MiB) cannot hold for their reader go past them.
      const bool stream_out = 2 * batch * kv_heads * max_tokens * head_dim * static_cast<int64_t>(sizeof(T)) > (32 << 20);
      ReadArgs<T> a{c,
                    start,
                    lengths,
                    {static_cast<T*>(k_out), static_cast<T*>(v_out)},
                    static_cast<int32_t>(max_tokens),
                    static_cast<int32_t>(groups),
                    static_cast<uint32_t>(threads)};
      return launch("kv8_read_kernel", stream_out ? kv8_read_kernel<T, F, true> : kv8_read_kernel<T, F, false>,
                    dim3(static_cast<uint32_t>(ceil_div(threads, kThreads))), dim3(kThreads), 0,
                    static_cast<hipStream_t>(stream), a);
    });
  });
}
