// kv8_attend.hip -- attention over the paged 8-bit K/V cache.
#include "kv8.hpp"

#include <cfloat>

namespace csahca {
namespace {

constexpr int kThreads = 256;

template <typename T>
struct AttendArgs {
  Kv8Cache c;
  const T* q;
  T* out;
  const int32_t* lengths;
  const void* ids;  // listed chunks, or null: all tokens
  int64_t chunk;
  int32_t top_k;
  int32_t ids64;
  int32_t queries;
  int32_t group;  // query heads of a K/V head
  float scale_log2;
};

__device__ __forceinline__ float block_max(float v, float* lds) {
  v = fmaxf(v, xor_lanes(v, 32));
#pragma unroll
  for (int off = 16; off >= 1; off >>= 1) v = fmaxf(v, xor_lanes(v, off));
  __syncthreads();
  if (threadIdx.x % kWave == 0) lds[threadIdx.x / kWave] = v;
  __syncthreads();
  for (int i = 0; i < kThreads / kWave; ++i) v = fmaxf(v, lds[i]);
  return v;
}

// One workgroup per query row (batch, query, head): kThreads token slots at a
// time, a thread a token for the scores and a thread a dimension for the sum.
template <typename T, typename F>
__global__ __launch_bounds__(kThreads) void kv8_attend_row_kernel(const AttendArgs<T> a) {
  __shared__ float q[kKv8MaxHeadDim], p[kThreads], red[kThreads / kWave];
  __shared__ int64_t at[kThreads];
  const Kv8Cache& c = a.c;
  const int D = c.head_dim, heads = c.kv_heads * a.group;
  const int64_t row = blockIdx.x;
  const int32_t head = static_cast<int32_t>(row % heads), h = head / a.group;
  const int32_t i = static_cast<int32_t>(row / heads % a.queries);
  const int64_t b = row / heads / a.queries;
  const int64_t cap = static_cast<int64_t>(c.blocks) * c.page_size;
  int64_t n = min(max(static_cast<int64_t>(a.lengths[b]), static_cast<int64_t>(0)), cap);
  n = n - a.queries + 1 + i;
  const int64_t slots = a.ids ? a.top_k * a.chunk : n;
  for (int d = threadIdx.x; d < D; d += kThreads) q[d] = to_f32(a.q[row * D + d]);
  __syncthreads();
  float m = -FLT_MAX, l = 0.f, o = 0.f;  // a finite start: scores that are all NaN still reach the sums
  for (int64_t t0 = 0; t0 < slots; t0 += kThreads) {
    const int64_t slot = t0 + threadIdx.x;
    int64_t pos = slot;
    if (a.ids && slot < slots) {
      const int64_t list = (b * c.kv_heads + h) * a.top_k + slot / a.chunk;
      const int64_t id = a.ids64 ? static_cast<const int64_t*>(a.ids)[list] : static_cast<const int32_t*>(a.ids)[list];
      pos = id < 0 || id > cap / a.chunk ? -1 : id * a.chunk + slot % a.chunk;
    }
    int32_t page = -1;
    if (slot < slots && pos >= 0 && pos < n) page = kv8_page(c, b, pos / c.page_size);
    float s = -__builtin_inff(), vs = 0.f;
    int64_t base = -1;
    if (page >= 0) {
      const int r = static_cast<int>(pos % c.page_size);
      const int64_t tile = kv8_tile(c, page, h);
      const uint4* kp = reinterpret_cast<const uint4*>(c.k + tile + static_cast<int64_t>(r) * D);
      float dot = 0.f;
      for (int u = 0; u < D / 16; ++u) {
        const uint4 w = kp[u];
        const uint32_t ww[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          dot = fmaf(kv8_decode<F, 0>(ww[e]), q[16 * u + 4 * e], dot);
          dot = fmaf(kv8_decode<F, 1>(ww[e]), q[16 * u + 4 * e + 1], dot);
          dot = fmaf(kv8_decode<F, 2>(ww[e]), q[16 * u + 4 * e + 2], dot);
          dot = fmaf(kv8_decode<F, 3>(ww[e]), q[16 * u + 4 * e + 3], dot);
        }
      }
      const int64_t sc = static_cast<int64_t>(page) * c.kv_heads + h;
      s = dot * c.k_scale[sc] * a.scale_log2;
      vs = c.v_scale[sc];
      base = tile + static_cast<int64_t>(r / kKv8Group) * D * kKv8Group + r % kKv8Group;
    }
    const float top = fmaxf(m, block_max(s, red));
    {
      const float w = base >= 0 ? fast_exp2(s - top) : 0.f;
      const float fix = fast_exp2(m - top);
      p[threadIdx.x] = w * vs;
      at[threadIdx.x] = base;
      l = l * fix + w;  // this thread's slots only; the threads' sums are joined at the end
      o *= fix;
      m = top;
      __syncthreads();
      if (threadIdx.x < D) {
        const int most = static_cast<int>(min(slots - t0, static_cast<int64_t>(kThreads)));
        for (int t = 0; t < most; ++t)
          if (at[t] >= 0) o = fmaf(p[t], kv8_decode<F, 0>(c.v[at[t] + threadIdx.x * kKv8Group]), o);
      }
    }
  }
  l = wave_sum(l);
  __syncthreads();
  if (threadIdx.x % kWave == 0) red[threadIdx.x / kWave] = l;
  __syncthreads();
  l = 0.f;
  for (int w = 0; w < kThreads / kWave; ++w) l += red[w];
  if (threadIdx.x < D) a.out[row * D + threadIdx.x] = from_f32<T>(l != 0.f ? o / l : 0.f);
}

int attend(const Kv8Cache& c, const void* q, void* out, int dtype, int format, int64_t batch, int64_t queries,
           int64_t heads, const int32_t* lengths, const void* ids, int index_dtype, int64_t top_k, int64_t chunk,
           double softmax_scale, hipStream_t stream) {
  CSAHCA_REQUIRE(queries <= INT32_MAX / (batch * heads), "too many query rows in one call");
  return dispatch_kv8_dtype(dtype, [&](auto tag) {
    using T = decltype(tag);
    return dispatch_kv8(format, [&](auto fmt) {
      using F = decltype(fmt);
      AttendArgs<T> a{c,
                      static_cast<const T*>(q),
                      static_cast<T*>(out),
                      lengths,
                      ids,
                      chunk,
                      static_cast<int32_t>(top_k),
                      index_dtype == CSAHCA_I64,
                      static_cast<int32_t>(queries),
                      static_cast<int32_t>(heads / c.kv_heads),
                      static_cast<float>(softmax_scale * 1.4426950408889634)};
      return launch("kv8_attend_row_kernel", kv8_attend_row_kernel<T, F>,
                    dim3(static_cast<uint32_t>(batch * queries * heads)), dim3(kThreads), 0, stream, a);
    });
  });
}

int check(const Kv8Cache& c, int dtype, int format, int64_t batch, int64_t queries, int64_t heads, int64_t kv_heads,
          int64_t head_dim, int64_t num_pages, int64_t page_size, int64_t blocks) {
  CSAHCA_REQUIRE(kv8_value_dtype(dtype), "unsupported dtype");
  CSAHCA_REQUIRE(batch >= 0 && queries >= 0 && heads >= 0, "negative dimension");
  if (const int rc = kv8_check_cache(c, format, num_pages, blocks, page_size, kv_heads, head_dim)) return rc;
  CSAHCA_REQUIRE(heads == 0 || (kv_heads > 0 && heads % kv_heads == 0), "q heads must be a multiple of the cache's heads");
  CSAHCA_REQUIRE(batch <= INT32_MAX && queries <= INT32_MAX && heads <= 65535, "too many query rows in one call");
  return CSAHCA_OK;
}

Kv8Cache cache_of(const void* k_cache, const void* v_cache, const float* k_scale, const float* v_scale,
                  int64_t num_pages, int64_t page_size, const int32_t* block_table, int64_t blocks,
                  int64_t table_stride, int64_t kv_heads, int64_t head_dim) {
  return Kv8Cache{static_cast<uint8_t*>(const_cast<void*>(k_cache)), static_cast<uint8_t*>(const_cast<void*>(v_cache)),
                  const_cast<float*>(k_scale), const_cast<float*>(v_scale), block_table, table_stride,
                  static_cast<int32_t>(num_pages), static_cast<int32_t>(blocks), static_cast<int32_t>(page_size),
                  static_cast<int32_t>(kv_heads), static_cast<int32_t>(head_dim)};
}

}  // namespace
}  // namespace csahca

using namespace csahca;

extern "C" size_t csahca_kv8_decode_workspace_bytes(int64_t batch, int64_t queries, int64_t heads, int64_t kv_heads,
                                                    int64_t head_dim, int64_t page_size, int64_t blocks) {
  return 0;
}

extern "C" int csahca_kv8_decode_forward(const void* q, void* out, int dtype, int64_t batch, int64_t queries,
                                         int64_t heads, int64_t kv_heads, int64_t head_dim, const void* k_cache,
                                         const void* v_cache, const float* k_scale, const float* v_scale, int format,
                                         int64_t num_pages, int64_t page_size, const int32_t* block_table,
                                         int64_t blocks, int64_t table_stride, const int32_t* lengths,
                                         double softmax_scale, void* workspace, size_t workspace_bytes,
                                         void* stream) {
  clear_error();
  Kv8Cache c = cache_of(k_cache, v_cache, k_scale, v_scale, num_pages, page_size, block_table, blocks,
                        table_stride, kv_heads, head_dim);
  if (const int rc = check(c, dtype, format, batch, queries, heads, kv_heads, head_dim, num_pages, page_size, blocks))
    return rc;
  if (batch == 0 || queries == 0 || heads == 0) return CSAHCA_OK;
  CSAHCA_REQUIRE(q && out && lengths, "null tensor pointer");
  if (num_pages == 0) c.blocks = 0;  // an empty pool: nothing to attend to
  if (c.blocks > 0) {
    if (const int rc = kv8_check_pointers(c)) return rc;
  }
  return attend(c, q, out, dtype, format, batch, queries, heads, lengths, nullptr, CSAHCA_I32, 0, 1, softmax_scale,
                static_cast<hipStream_t>(stream));
}

extern "C" size_t csahca_kv8_csa_decode_workspace_bytes(int64_t batch, int64_t heads, int64_t kv_heads,
                                                        int64_t head_dim, int64_t top_k, int64_t chunk_size) {
  return 0;
}

extern "C" int csahca_kv8_csa_decode_forward(const void* q, void* out, int dtype, int64_t batch, int64_t heads,
                                             int64_t kv_heads, int64_t head_dim, const void* k_cache,
                                             const void* v_cache, const float* k_scale, const float* v_scale,
                                             int format, int64_t num_pages, int64_t page_size,
                                             const int32_t* block_table, int64_t blocks, int64_t table_stride,
                                             const int32_t* lengths, const void* chunk_indices, int index_dtype,
                                             int64_t top_k, int64_t chunk_size, double softmax_scale,
                                             void* workspace, size_t workspace_bytes, void* stream) {
  clear_error();
  Kv8Cache c = cache_of(k_cache, v_cache, k_scale, v_scale, num_pages, page_size, block_table, blocks,
                        table_stride, kv_heads, head_dim);
  if (const int rc = check(c, dtype, format, batch, 1, heads, kv_heads, head_dim, num_pages, page_size, blocks))
    return rc;
  CSAHCA_REQUIRE(index_dtype == CSAHCA_I32 || index_dtype == CSAHCA_I64, "chunk_indices must be int32 or int64");
  CSAHCA_REQUIRE(chunk_size > 0, "chunk_size must be positive");
  CSAHCA_REQUIRE(top_k >= 0 && chunk_size <= INT32_MAX && top_k <= INT32_MAX, "negative dimension");
  if (batch == 0 || heads == 0) return CSAHCA_OK;
  CSAHCA_REQUIRE(q && out && lengths && (chunk_indices || top_k == 0), "null tensor pointer");
  if (num_pages == 0) c.blocks = 0;  // an empty pool: nothing to attend to
  if (c.blocks > 0) {
    if (const int rc = kv8_check_pointers(c)) return rc;
  }
  // an empty list: a list of no chunks, told from "all tokens" by its pointer
  return attend(c, q, out, dtype, format, batch, 1, heads, lengths, chunk_indices ? chunk_indices : lengths, index_dtype,
                chunk_indices ? top_k : 0, chunk_size, softmax_scale, static_cast<hipStream_t>(stream));
}
