// kv8_cache.hip -- the paged 8-bit K/V cache: quantize-on-write and reading back.
#include "kv8.hpp"

namespace csahca {
namespace {

constexpr int kThreads = 256;

__device__ __forceinline__ float block_max(float v, float* lds) {
#pragma unroll
  for (int off = 32; off >= 1; off >>= 1) v = fmaxf(v, xor_lanes(v, off));
  if (threadIdx.x % kWave == 0) lds[threadIdx.x / kWave] = v;
  __syncthreads();
  for (int i = 0; i < kThreads / kWave; ++i) v = fmaxf(v, lds[i]);
  return v;
}

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

// Byte offset of (token row, dimension d) in a (page, head) tile.
template <bool kV>
__device__ __forceinline__ int tile_at(int row, int d, int D) {
  return kV ? (row / kKv8Group * D + d) * kKv8Group + row % kKv8Group : row * D + d;
}

// One workgroup owns K or V of one (sequence, page, head): nothing it reads or
// writes is another's.
template <typename T, typename F, bool kV>
__device__ void write_tile(const WriteArgs<T>& a, int64_t b, int32_t j, int32_t h, float* lds) {
  const Kv8Cache& c = a.c;
  const int64_t start = a.start[b];
  const int64_t count = a.counts ? min(max(a.counts[b], 0), a.new_tokens) : a.new_tokens;
  if (start < 0) return;
  const int64_t block = start / c.page_size + j;
  const int64_t first = block * c.page_size;
  const int lo = static_cast<int>(max(start - first, static_cast<int64_t>(0)));
  const int hi = static_cast<int>(min(start + count - first, static_cast<int64_t>(c.page_size)));
  if (hi <= lo) return;
  const int32_t page = kv8_page(c, b, block);
  if (page < 0) return;
  const int D = c.head_dim, n = (hi - lo) * D;
  const T* x = a.x[kV] + b * a.sb[kV] + h * a.sh[kV] + (first + lo - start) * a.sn[kV];
  uint8_t* tile = (kV ? c.v : c.k) + kv8_tile(c, page, h);
  float* scale = (kV ? c.v_scale : c.k_scale) + static_cast<int64_t>(page) * c.kv_heads + h;

  float amax = 0.f;
  for (int i = threadIdx.x; i < n; i += kThreads) {
    const float v = fabsf(to_f32(x[i / D * a.sn[kV] + i % D]));
    if (v < __builtin_inff()) amax = fmaxf(amax, v);
  }
  amax = block_max(amax, lds);
  float s = kv8_scale_for<F>(amax);
  if (lo > 0) {
    const float old = *scale;
    if (s > old) {
      const float ratio = old / s;
      for (int i = threadIdx.x; i < lo * D; i += kThreads) {
        uint8_t* p = tile + tile_at<kV>(i / D, i % D, D);
        *p = static_cast<uint8_t>(kv8_encode<F>(kv8_decode<F, 0>(*p) * ratio));
      }
    } else {
      s = old;
    }
  }
  const float inv = 1.0f / s;
  for (int i = threadIdx.x; i < n; i += kThreads)
    tile[tile_at<kV>(lo + i / D, i % D, D)] =
        static_cast<uint8_t>(kv8_encode<F>(to_f32(x[i / D * a.sn[kV] + i % D]) * inv));
  __syncthreads();  // every thread has read the old scale
  if (threadIdx.x == 0) *scale = s;
}

template <typename T, typename F>
__global__ __launch_bounds__(kThreads) void kv8_write_kernel(const WriteArgs<T> a) {
  __shared__ float lds[kThreads / kWave];
  uint32_t i = blockIdx.x;
  const bool v = i & 1;
  i /= 2;
  const int32_t h = i % a.c.kv_heads;
  i /= a.c.kv_heads;
  const int32_t j = i % a.pages_per;
  const int64_t b = i / a.pages_per;
  if (v) {
    write_tile<T, F, true>(a, b, j, h, lds);
  } else {
    write_tile<T, F, false>(a, b, j, h, lds);
  }
}

template <typename T>
struct ReadArgs {
  Kv8Cache c;
  const int32_t* start;
  const int32_t* lengths;
  T* out[2];
  int32_t max_tokens;
};

template <typename T, typename F>
__global__ __launch_bounds__(kThreads) void kv8_read_kernel(const ReadArgs<T> a) {
  const Kv8Cache& c = a.c;
  const int64_t row = blockIdx.x;  // (batch, head, token)
  const int64_t n = row % a.max_tokens, bh = row / a.max_tokens;
  const int64_t b = bh / c.kv_heads;
  const int32_t h = static_cast<int32_t>(bh % c.kv_heads);
  const int64_t pos = (a.start ? a.start[b] : 0) + n;
  int32_t page = -1;
  if (pos >= 0 && pos < a.lengths[b]) page = kv8_page(c, b, pos / c.page_size);
  const int D = c.head_dim;
  for (int i = threadIdx.x; i < 2 * D; i += kThreads) {
    const bool v = i >= D;
    const int d = v ? i - D : i;
    float x = 0.f;
    if (page >= 0) {
      const int r = static_cast<int>(pos % c.page_size);
      const uint8_t* tile = (v ? c.v : c.k) + kv8_tile(c, page, h);
      const float s = (v ? c.v_scale : c.k_scale)[static_cast<int64_t>(page) * c.kv_heads + h];
      x = kv8_decode<F, 0>(tile[v ? tile_at<true>(r, d, D) : tile_at<false>(r, d, D)]) * s;
    }
    a.out[v][row * D + d] = from_f32<T>(x);
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
  CSAHCA_REQUIRE(batch * pages_per <= INT32_MAX / (2 * kv_heads), "too many tokens in one call");
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
      return launch("kv8_write_kernel", kv8_write_kernel<T, F>, dim3(static_cast<uint32_t>(grid)), dim3(kThreads), 0,
                    static_cast<hipStream_t>(stream), a);
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
  CSAHCA_REQUIRE(max_tokens <= INT32_MAX / (batch * kv_heads), "too many tokens in one call");
  const int64_t rows = batch * kv_heads * max_tokens;
  return dispatch_kv8_dtype(dtype, [&](auto tag) {
    using T = decltype(tag);
    return dispatch_kv8(format, [&](auto fmt) {
      using F = decltype(fmt);
      ReadArgs<T> a{c, start, lengths, {static_cast<T*>(k_out), static_cast<T*>(v_out)},
                    static_cast<int32_t>(max_tokens)};
      return launch("kv8_read_kernel", kv8_read_kernel<T, F>, dim3(static_cast<uint32_t>(rows)), dim3(kThreads), 0,
                    static_cast<hipStream_t>(stream), a);
    });
  });
}
