// kv8.hpp -- the paged 8-bit K/V cache: formats, page lookup, argument checks.
//
// A cache is num_pages pages of page_size tokens (a multiple of 16), each with
// kv_heads heads of head_dim values:
//   k_cache [num_pages, kv_heads, page_size, head_dim]
//   v_cache [num_pages, kv_heads, page_size / 16, head_dim, 16]
// one byte a value, and an fp32 scale for each (page, head) of K and of V; a
// value is byte * scale.  V is transposed in groups of 16 tokens so that the
// attention's second product reads 16 consecutive tokens of one dimension with
// one 16-byte load, as its matrix operand wants them.
#pragma once

#include "common.hpp"

namespace csahca {

constexpr int kKv8Group = 16;        // tokens that v_cache holds together
constexpr int kKv8MaxPage = 256;     // tokens of a page, at most
constexpr int kKv8MaxHeadDim = 256;  // a multiple of 32
constexpr int kKv8LeastExp = -120;   // scales are 2^-120 .. 2^120

// The two formats: the largest magnitude, and as kTop 2^kTopExp with kTop in
// [0.5, 1).
struct E4m3 {
  static constexpr float kMax = 448.0f, kTop = 0.875f;
  static constexpr int kTopExp = 9;
};
struct Int8 {
  static constexpr float kMax = 127.0f, kTop = 0.9921875f;
  static constexpr int kTopExp = 7;
};

// Byte `Sel` of a word as fp32.
template <typename F, int Sel>
__device__ __forceinline__ float kv8_decode(uint32_t w) {
  if constexpr (std::is_same_v<F, E4m3>) {
    return __builtin_amdgcn_cvt_f32_fp8(static_cast<int>(w), Sel);
  } else {
    return static_cast<float>(static_cast<int8_t>(w >> (8 * Sel)));
  }
}

// The scale that holds values up to amax: the least power of two s with
// amax <= kMax s, within 2^-120 .. 2^120 (amax = 0: 2^-120).
template <typename F>
__device__ __forceinline__ float kv8_scale_for(float amax) {
  int e;
  const float m = frexpf(amax, &e);  // amax = m 2^e, m in [0.5, 1)
  e = m <= F::kTop ? e - F::kTopExp : e - F::kTopExp + 1;
  if (!(amax > 0.f) || e < kKv8LeastExp) e = kKv8LeastExp;
  if (e > -kKv8LeastExp) e = -kKv8LeastExp;
  return __builtin_ldexpf(1.0f, e);
}

// A paged cache as the kernels take it.
struct Kv8Cache {
  uint8_t* k;
  uint8_t* v;
  float* k_scale;
  float* v_scale;
  const int32_t* table;  // [batch, blocks], rows table_stride apart
  int64_t table_stride;
  int32_t num_pages;
  int32_t blocks;
  int32_t page_size;
  int32_t kv_heads;
  int32_t head_dim;
};

// Physical page of a sequence's logical page, or -1 where there is none.
__device__ __forceinline__ int32_t kv8_page(const Kv8Cache& c, int64_t batch, int64_t block) {
  if (block < 0 || block >= c.blocks) return -1;
  const int32_t id = c.table[batch * c.table_stride + block];
  return id >= 0 && id < c.num_pages ? id : -1;
}

// Bytes before (page, head) in k_cache and in v_cache.
__device__ __forceinline__ int64_t kv8_tile(const Kv8Cache& c, int32_t page, int32_t head) {
  return (static_cast<int64_t>(page) * c.kv_heads + head) * c.page_size * c.head_dim;
}

inline int kv8_check_cache(const Kv8Cache& c, int format, int64_t num_pages, int64_t blocks, int64_t page_size,
                           int64_t kv_heads, int64_t head_dim) {
  CSAHCA_REQUIRE(format == CSAHCA_KV8_E4M3 || format == CSAHCA_KV8_INT8, "k_cache must be float8_e4m3fn or int8");
  CSAHCA_REQUIRE(num_pages >= 0 && blocks >= 0 && kv_heads >= 0, "negative dimension");
  CSAHCA_REQUIRE(page_size > 0 && page_size <= kKv8MaxPage && page_size % kKv8Group == 0,
                 "page_size must be a multiple of 16, at most 256");
  CSAHCA_REQUIRE(head_dim > 0 && head_dim <= kKv8MaxHeadDim && head_dim % 32 == 0,
                 "head_dim must be a multiple of 32, at most 256");
  CSAHCA_REQUIRE(num_pages <= INT32_MAX && blocks <= INT32_MAX / kKv8MaxPage && kv_heads <= 65535,
                 "cache dimension too large");
  CSAHCA_REQUIRE(c.table_stride >= blocks, "block_table rows overlap");
  return CSAHCA_OK;
}

inline int kv8_check_pointers(const Kv8Cache& c) {
  CSAHCA_REQUIRE(c.k && c.v && c.k_scale && c.v_scale && c.table, "null tensor pointer");
  CSAHCA_REQUIRE(reinterpret_cast<uintptr_t>(c.k) % 16 == 0 && reinterpret_cast<uintptr_t>(c.v) % 16 == 0,
                 "k_cache and v_cache must be 16-byte aligned");
  return CSAHCA_OK;
}

// Dispatch a callable templated on the format.
template <typename F>
int dispatch_kv8(int format, F&& f) {
  return format == CSAHCA_KV8_E4M3 ? f(E4m3{}) : f(Int8{});
}

// f32, f16 and bf16: the value types of these operators.
inline bool kv8_value_dtype(int dt) { return dt == CSAHCA_F32 || dt == CSAHCA_F16 || dt == CSAHCA_BF16; }

template <typename F>
int dispatch_kv8_dtype(int dtype, F&& f) {
  switch (dtype) {
    case CSAHCA_BF16: return f(bf16{});
    case CSAHCA_F16: return f(f16{});
    default: return f(float{});
  }
}

}  // namespace csahca
