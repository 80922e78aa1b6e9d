// kv8_attend.hip -- attention over the paged 8-bit K/V cache: the split, the join
// of its parts, and the entry points.  The kernel is in kv8_attend.hpp.
#include "kv8_attend.hpp"

#include <algorithm>

namespace csahca {
namespace {

// The rows (batch, K/V head, row) of sequences that have several parts:
// out = 2^(M - S) sum_p 2^(m_p - M) O_p / sum_p 2^(s_p - S) l_p, M = max m_p, S = max
// s_p, the maxima of the parts' numerators and sums.  A thread
// takes four dimensions of a row and every join_lanes-th part; a row's parts are
// in flight together, up to four a thread (a wavefront a row and four parts a
// round trip took 22 us for the 32 parts of 8192 tokens of 8 heads, this 4.6).
// The order of the sums is fixed by the split alone.
__global__ __launch_bounds__(kKv8Threads) void kv8_join_kernel(const Kv8Attend a) {
  __shared__ f32x4_t sums[kKv8Threads];
  __shared__ float tops[kKv8Threads], stops[kKv8Threads], totals[kKv8Threads];
  const int32_t D = a.c.head_dim, wide = D / 4, lanes = kKv8Threads / wide;
  const int32_t per = lanes / a.join_lanes;  // rows of a workgroup, all of one sequence
  const int64_t brows = static_cast<int64_t>(a.c.kv_heads) * a.rows, groups = (brows + per - 1) / per;
  const int64_t b = blockIdx.x / groups;
  const int32_t d = threadIdx.x % wide * 4, unit = threadIdx.x / wide, lane = unit % a.join_lanes;
  const int64_t hr = blockIdx.x % groups * per + unit / a.join_lanes;
  int32_t count = 0, first = 0;
  kv8_parts_of(a, static_cast<int32_t>(b), &count, &first);
  if (count <= 1) return;
  const bool mine = unit < per * a.join_lanes && hr < brows;
  const int32_t h = static_cast<int32_t>(hr / a.rows), r = static_cast<int32_t>(hr % a.rows);
  const int64_t step = static_cast<int64_t>(a.c.kv_heads) * a.rows;
  const int64_t slot0 = (static_cast<int64_t>(first) * a.c.kv_heads + h) * a.rows + r;
  float top = -FLT_MAX, stop = -FLT_MAX, total = 0.f;
  f32x4_t acc{0.f, 0.f, 0.f, 0.f};
  const auto add = [&](float m, float ms, float l, f32x4_t o) {
    const float up = fmaxf(top, m), sup = fmaxf(stop, ms);
    total = total * fast_exp2(stop - sup) + l * fast_exp2(ms - sup);
    acc = acc * fast_exp2(top - up) + o * fast_exp2(m - up);
    top = up;
    stop = sup;
  };
  if (mine) {
    for (int p0 = lane; p0 < count; p0 += 4 * a.join_lanes) {
      float4 ml[4];
      f32x4_t o[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {  // behind the last part: that part again, unused
        const int64_t slot = slot0 + min(p0 + i * a.join_lanes, count - 1) * step;
        ml[i] = reinterpret_cast<const float4*>(a.part_ml)[slot];
        o[i] = *reinterpret_cast<const f32x4_t*>(a.part_o + slot * D + d);
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if (p0 + i * a.join_lanes >= count) break;
        add(ml[i].x, ml[i].y, ml[i].z, o[i]);
      }
    }
  }
  tops[threadIdx.x] = top;
  stops[threadIdx.x] = stop;
  totals[threadIdx.x] = total;
  sums[threadIdx.x] = acc;
  __syncthreads();
  if (!mine || lane > 0) return;
  for (int i = 1; i < a.join_lanes; ++i) {
    const int at = i * wide + threadIdx.x;
    add(tops[at], stops[at], totals[at], sums[at]);
  }
  const int64_t heads = static_cast<int64_t>(a.c.kv_heads) * a.group;
  kv8_store4(a, ((b * a.queries + r / a.group) * heads + h * a.group + r % a.group) * D + d,
             kv8_result(acc, total, top - stop));
}

// How a call is laid out over workgroups, from its sizes alone.
struct Split {
  int tiles;       // row tiles (16 rows) of a wavefront, 1 or 2; 0: the kernel of many rows
  int row_waves;   // wavefronts of a workgroup over the rows, 1, 2, 4 or (many rows) 8
  int row_groups;
  int round;       // wavefronts over the tokens
  int min_tiles;   // 64-token tiles of a part, at least (a list: exactly)
  int even_log2, ragged_log2;  // workgroups over the tokens, at most about: lengths alike, ragged
  int64_t parts;   // parts over the batch, at most
  bool joined;     // whether a sequence may have several
};

// Each threshold with both sides measured (us; heads of 128 in bf16 unless said;
// kernel + join where there is one):
//   * more than 64 rows go to the kernel of many rows: 96 rows over 4 x 8192 tokens
//     38 + 7 there, 43 + 9 with 32 rows a wavefront; 160 rows 46 + 9 / 67 + 6; up to
//     64 they fit a workgroup of the other at 30 + 7.  (Heads of 64, 128 rows: 27 / 25.)
//   * two row tiles a wavefront for 17 rows on, up to heads of 192: 32 rows over
//     8 x 16384 tokens 54 / 58 with one, 64 rows 68 / 87, 64 rows of 192 97 / 122; of
//     256, where the registers spill, 304 / 183.
//   * up to four rounds of a workgroup's wavefronts go undivided, without the join:
//     512 tokens 11.4 / 8.9 + 4.2, 1024 tokens 14 / 10.5 + 4.5, 2048 tokens 20 / 10 + 4.3.
//   * lengths that are alike are divided among 2^8 workgroups, one a CU (32 rows over
//     8 x 16384 tokens 64 + 4 with 2^8, 70 + 6 with 2^9, 82 + 8 with 2^10; single rows
//     differ by 2), so 2^9 for lists too costs the join (27 + 4 / 28); ragged ones
//     (uniform up to 32768) among 2^10, of a batch of 16 with 4 rows 74 + 6, 84 + 5
//     with 2^9, 100 with 2^8; of more rows, whose partial results weigh more, 2^9 (32
//     rows 62 + 5, 67 + 8 with 2^10) and in the kernel of many rows 2^8 (512 rows
//     53 + 12, 82 + 41 with 2^10).
Split split_of(int dtype, int64_t batch, int64_t rows, int64_t kv_heads, int64_t head_dim, int64_t tiles, bool list) {
  Split s;
  const int64_t row_tiles = ceil_div(rows, 16);
  if (rows > 64 && dtype != CSAHCA_F32) {  // the kernel of many rows, 32 a wavefront
    s.tiles = 0;
    s.row_waves = kv8_rows_waves(head_dim);
    s.row_groups = static_cast<int>(ceil_div(row_tiles, 2 * s.row_waves));
    s.round = 1;
  } else {
    s.tiles = row_tiles <= 1 || dtype == CSAHCA_F32 || head_dim > kKv8TwoTilesDim ? 1 : 2;
    const int64_t waves = ceil_div(row_tiles, s.tiles);
    s.row_waves = waves <= 1 ? 1 : waves <= 2 ? 2 : 4;
    s.row_groups = static_cast<int>(ceil_div(waves, s.row_waves));
    s.round = kKv8Waves / s.row_waves;
  }
  s.even_log2 = 8;
  s.ragged_log2 = s.tiles == 0 ? 8 : rows <= 16 ? 10 : 9;
  const int round = s.round;
  s.min_tiles = tiles <= 4 * round ? std::max(static_cast<int>(ceil_div(tiles, round)), 1) * round : round;
  const int64_t target = int64_t{1} << (list ? s.even_log2 : s.ragged_log2);
  const int64_t lanes = kv_heads * s.row_groups;
  if (list) {
    const int64_t per = batch * lanes >= target ? tiles : ceil_div(tiles * batch * lanes, target);
    s.min_tiles = static_cast<int>(ceil_div(std::max<int64_t>(per, s.min_tiles), round) * round);
    s.parts = batch * ceil_div(tiles, s.min_tiles);
  } else {
    s.parts = std::min(target / lanes + batch, batch * std::max<int64_t>(ceil_div(tiles, s.min_tiles), 1));
  }
  s.joined = s.parts > batch;
  return s;
}

size_t workspace_of(const Split& s, int64_t kv_heads, int64_t rows, int64_t head_dim) {
  return s.joined ? static_cast<size_t>(s.parts * kv_heads * rows * (head_dim + 4)) * sizeof(float) : 0;
}

int attend(Kv8Attend a, int format, int64_t tiles, void* workspace, size_t workspace_bytes, hipStream_t stream) {
  const Split s = split_of(a.dtype, a.batch, a.rows, a.c.kv_heads, a.c.head_dim, tiles, a.ids != nullptr);
  CSAHCA_REQUIRE(s.parts <= INT32_MAX / a.c.kv_heads / s.row_groups &&
                     a.rows <= INT32_MAX / a.c.kv_heads / a.batch,
                 "too many query rows in one call");
  if (s.joined && (workspace == nullptr || workspace_bytes < workspace_of(s, a.c.kv_heads, a.rows, a.c.head_dim)))
    return fail(CSAHCA_ERR_WORKSPACE, "workspace too small for kv8 decode");
  CSAHCA_REQUIRE(!s.joined || reinterpret_cast<uintptr_t>(workspace) % 16 == 0, "workspace must be 16-byte aligned");
  const int64_t brows = int64_t{a.rows} * a.c.kv_heads, lanes = kKv8Threads / (a.c.head_dim / 4);
  a.join_lanes = static_cast<int32_t>(std::min(lanes, ceil_div(s.parts / a.batch, 4)));
  const int64_t join_grid = ceil_div(brows, lanes / a.join_lanes) * a.batch;
  CSAHCA_REQUIRE(!s.joined || join_grid <= UINT32_MAX / kKv8Threads, "too many query rows in one call");
  a.row_groups = s.row_groups;
  a.row_waves = s.row_waves;
  a.round = s.round;
  a.parts = static_cast<int32_t>(s.parts);
  a.min_tiles = s.min_tiles;
  a.even_log2 = s.even_log2;
  a.ragged_log2 = s.ragged_log2;
  a.part_o = static_cast<float*>(workspace);
  a.part_ml = a.part_o + s.parts * a.c.kv_heads * a.rows * a.c.head_dim;
  const int rc = format == CSAHCA_KV8_E4M3 ? kv8_attend_launch_e4m3(a, s.tiles, stream)
                                           : kv8_attend_launch_int8(a, s.tiles, stream);
  if (rc != CSAHCA_OK || !s.joined) return rc;
  return launch("kv8_join_kernel", kv8_join_kernel, dim3(static_cast<uint32_t>(join_grid)), dim3(kKv8Threads), 0, stream,
                a);
}

int check(const Kv8Cache& c, int dtype, int format, int64_t batch, int64_t queries, int64_t heads, int64_t kv_heads,
          int64_t head_dim, int64_t num_pages, int64_t page_size, int64_t blocks) {
  CSAHCA_REQUIRE(kv8_value_dtype(dtype), "unsupported dtype");
  CSAHCA_REQUIRE(batch >= 0 && queries >= 0 && heads >= 0, "negative dimension");
  if (const int rc = kv8_check_cache(c, format, num_pages, blocks, page_size, kv_heads, head_dim)) return rc;
  CSAHCA_REQUIRE(heads == 0 || (kv_heads > 0 && heads % kv_heads == 0), "q heads must be a multiple of the cache's heads");
  CSAHCA_REQUIRE(batch <= INT32_MAX && heads <= 65535 && (heads == 0 || queries <= INT32_MAX / heads),
                 "too many query rows in one call");
  CSAHCA_REQUIRE(num_pages <= INT32_MAX / (page_size / kKv8Group) / std::max<int64_t>(kv_heads, 1),
                 "cache dimension too large");  // the kernel counts groups of 16 tokens in 32 bits
  return CSAHCA_OK;
}

Kv8Attend args_of(const Kv8Cache& c, const void* q, void* out, int dtype, int64_t batch, int64_t queries, int64_t heads,
                  const int32_t* lengths, double softmax_scale) {
  Kv8Attend a{};
  a.c = c;
  a.q = q;
  a.out = out;
  a.lengths = lengths;
  a.chunk = 1;
  a.dtype = dtype;
  a.batch = static_cast<int32_t>(batch);
  a.queries = static_cast<int32_t>(queries);
  a.group = static_cast<int32_t>(heads / c.kv_heads);
  a.rows = static_cast<int32_t>(queries * a.group);
  a.page_groups = static_cast<uint32_t>(c.page_size / kKv8Group);
  a.page_magic = a.page_groups == 1 ? 0u : static_cast<uint32_t>(((uint64_t{1} << 32) + a.page_groups - 1) / a.page_groups);
  a.scale_log2 = static_cast<float>(softmax_scale * 1.4426950408889634);
  return a;
}

// Sub-blocks (aligned groups of 16 tokens) that a chunk of this size can touch.
int64_t chunk_subs(int64_t chunk) { return chunk % kKv8Group == 0 ? chunk / kKv8Group : (chunk + 14) / kKv8Group + 1; }

Kv8Cache cache_of(const void* k_cache, const void* v_cache, const float* k_scale, const float* v_scale,
                  int64_t num_pages, int64_t page_size, const int32_t* block_table, int64_t blocks,
                  int64_t table_stride, int64_t kv_heads, int64_t head_dim) {
  return Kv8Cache{static_cast<uint8_t*>(const_cast<void*>(k_cache)), static_cast<uint8_t*>(const_cast<void*>(v_cache)),
                  const_cast<float*>(k_scale), const_cast<float*>(v_scale), block_table, table_stride,
                  static_cast<int32_t>(num_pages), static_cast<int32_t>(blocks), static_cast<int32_t>(page_size),
                  static_cast<int32_t>(kv_heads), static_cast<int32_t>(head_dim)};
}

// The page range of a call: an empty pool holds nothing to attend to.
int check_pool(Kv8Cache& c, const void* q, const void* out, const int32_t* lengths) {
  CSAHCA_REQUIRE(q && out && lengths, "null tensor pointer");
  CSAHCA_REQUIRE(reinterpret_cast<uintptr_t>(q) % 16 == 0 && reinterpret_cast<uintptr_t>(out) % 16 == 0,
                 "q and out must be 16-byte aligned");
  if (c.num_pages == 0) c.blocks = 0;
  return c.blocks > 0 ? kv8_check_pointers(c) : static_cast<int>(CSAHCA_OK);
}

}  // namespace
}  // namespace csahca

using namespace csahca;

extern "C" size_t csahca_kv8_decode_workspace_bytes(int dtype, int64_t batch, int64_t queries, int64_t heads,
                                                    int64_t kv_heads, int64_t head_dim, int64_t page_size,
                                                    int64_t blocks) {
  if (batch <= 0 || queries <= 0 || heads <= 0 || kv_heads <= 0 || head_dim <= 0 || page_size <= 0 || blocks < 0) return 0;
  if (batch > INT32_MAX || heads > 65535 || queries > INT32_MAX / heads || head_dim > kKv8MaxHeadDim ||
      page_size > kKv8MaxPage || blocks > INT32_MAX / kKv8MaxPage)
    return 0;  // refused by the call
  const int64_t rows = queries * (heads / kv_heads);
  return workspace_of(split_of(dtype, batch, rows, kv_heads, head_dim, ceil_div(blocks * page_size, kKv8Tile), false),
                      kv_heads, rows, head_dim);
}

extern "C" int csahca_kv8_decode_forward(const void* q, void* out, int dtype, int64_t batch, int64_t queries,
                                         int64_t heads, int64_t kv_heads, int64_t head_dim, const void* k_cache,
                                         const void* v_cache, const float* k_scale, const float* v_scale, int format,
                                         int64_t num_pages, int64_t page_size, const int32_t* block_table,
                                         int64_t blocks, int64_t table_stride, const int32_t* lengths,
                                         double softmax_scale, void* workspace, size_t workspace_bytes,
                                         void* stream) {
  clear_error();
  Kv8Cache c = cache_of(k_cache, v_cache, k_scale, v_scale, num_pages, page_size, block_table, blocks, table_stride,
                        kv_heads, head_dim);
  if (const int rc = check(c, dtype, format, batch, queries, heads, kv_heads, head_dim, num_pages, page_size, blocks))
    return rc;
  if (batch == 0 || queries == 0 || heads == 0) return CSAHCA_OK;
  if (const int rc = check_pool(c, q, out, lengths)) return rc;
  return attend(args_of(c, q, out, dtype, batch, queries, heads, lengths, softmax_scale), format,
                ceil_div(blocks * page_size, kKv8Tile), workspace, workspace_bytes, static_cast<hipStream_t>(stream));
}

extern "C" size_t csahca_kv8_csa_decode_workspace_bytes(int dtype, int64_t batch, int64_t heads, int64_t kv_heads,
                                                        int64_t head_dim, int64_t top_k, int64_t chunk_size) {
  if (batch <= 0 || heads <= 0 || kv_heads <= 0 || head_dim <= 0 || top_k <= 0 || chunk_size <= 0) return 0;
  if (batch > INT32_MAX || heads > 65535 || head_dim > kKv8MaxHeadDim || chunk_size > INT32_MAX ||
      top_k > INT32_MAX / kKv8Group / chunk_subs(chunk_size))
    return 0;  // refused by the call
  const int64_t rows = heads / kv_heads;
  return workspace_of(split_of(dtype, batch, rows, kv_heads, head_dim, ceil_div(top_k * chunk_subs(chunk_size), 4), true),
                      kv_heads, rows, head_dim);
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
  Kv8Cache c = cache_of(k_cache, v_cache, k_scale, v_scale, num_pages, page_size, block_table, blocks, table_stride,
                        kv_heads, head_dim);
  if (const int rc = check(c, dtype, format, batch, 1, heads, kv_heads, head_dim, num_pages, page_size, blocks))
    return rc;
  CSAHCA_REQUIRE(index_dtype == CSAHCA_I32 || index_dtype == CSAHCA_I64, "chunk_indices must be int32 or int64");
  CSAHCA_REQUIRE(chunk_size > 0, "chunk_size must be positive");
  CSAHCA_REQUIRE(top_k >= 0, "negative dimension");
  CSAHCA_REQUIRE(chunk_size <= INT32_MAX && top_k <= INT32_MAX / kKv8Group / chunk_subs(chunk_size),
                 "too many listed tokens in one call");
  if (batch == 0 || heads == 0) return CSAHCA_OK;
  CSAHCA_REQUIRE(chunk_indices || top_k == 0, "null tensor pointer");
  if (const int rc = check_pool(c, q, out, lengths)) return rc;
  Kv8Attend a = args_of(c, q, out, dtype, batch, 1, heads, lengths, softmax_scale);
  const int64_t subs = chunk_subs(chunk_size), tiles = ceil_div(top_k * subs, 4);
  if (c.blocks > 0 && top_k > 0) {
    a.ids = chunk_indices;
    a.ids64 = index_dtype == CSAHCA_I64;
    a.chunk = static_cast<int32_t>(chunk_size);
    a.top_k = static_cast<int32_t>(top_k);
    a.subs = static_cast<int32_t>(subs);
    a.list_tiles = static_cast<int32_t>(tiles);
  } else {
    a.c.blocks = 0;  // nothing listed: as over an empty cache
  }
  return attend(a, format, a.ids ? tiles : 0, workspace, workspace_bytes, static_cast<hipStream_t>(stream));
}
