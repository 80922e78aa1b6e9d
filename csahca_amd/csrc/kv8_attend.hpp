// kv8_attend.hpp -- attention over the paged 8-bit K/V cache: the kernel.
//
// out = softmax(c q K^T) V for R = queries * group rows of a K/V head, over the
// tokens of a sequence or of listed chunks.  Both products are matrix
// instructions (16x16x32, f16 operands, fp32 sums) on transposed operands:
//
//   S^T [64 tokens x 16 rows] = K Q^T      O^T [D x 16 rows] += V^T P^T
//
// so that no value changes lanes between them.  A wavefront takes 64 tokens at
// a time, as four groups ("sub-blocks") of 16 consecutive ones.  Lane l holds
// row n = l % 16 of the result and, for its quarter g = l / 16:
//   * S^T: the accumulator of K tile t (t = 0..3) holds its rows 4g..4g+3.  Rows
//     of a K tile may be any tokens, so row 4g + i of tile t is token 4t + i of
//     sub-block g: a lane's 16 scores are the 16 tokens of its sub-block.
//   * P^T: as the second product's operand a lane supplies 8 tokens an
//     instruction: its sub-block's first 8 and last 8, as they stand.
//   * V^T: the matching operand is 16 consecutive tokens of dimension
//     16 dt + n: one 16-byte load, because the cache keeps V that way.
//   * K: 16 bytes of a token's row a load; the order of dimensions in the sum is
//     free, so a lane's 16 bytes feed two instructions, with q loaded alike.
//
// Beside 16-bit values the operands are f16, in which a byte is exact and so is
// q, its rows scaled by a power of two to below 2^15 (bf16 has the wider range).
// A page's K scale and the row's factor go into the score; its V scale goes into
// the exponent: p = 2^(s + log2 vs - m) with m the running maximum of that sum,
// so p V is in units of the largest p vs so far whatever the scales are, and the
// softmax's sum takes p / vs (by a third small product, as if V's byte were 1,
// whose rows keep the sub-blocks apart).  p is rounded to f16's 11 bits.  It is
// held times 2^12; m is an integer (so that differences of such maxima are exact) and
// moves only when a score passes it by 3: the sums are rarely rescaled, p stays at
// most 2^15, and what is lost of a weight for want of exponent is at most 2^-36 of
// the largest p vs.  For the sum that is 2^-36 of its largest weight times the ratio
// of two V scales.  Where those of a part differ by more than 2^10 (a page of zeros
// has the least scale there is), or are so small that p / vs would overflow, the sum
// is taken by 16 more exponentials a lane and tile, beside a maximum of the scores
// alone; sums and their maxima are kept and joined apart from the numerators'
// (which costs the rest 0.3 us a call).
//
// Beside f32 values the operands are bf16, as wide as f32: q and p as three bf16
// each, 24 bits, of which nothing is lost.  Rows of q beyond 2^60 are scaled to
// that, so that products with bytes do not overflow before K's scale is applied.
#pragma once

#include <cfloat>

#include "kv8.hpp"

namespace csahca {

constexpr int kKv8Threads = 256;
constexpr int kKv8Waves = kKv8Threads / kWave;
constexpr int kKv8Tile = 64;      // tokens a wavefront takes at a time
constexpr int kKv8SegTiles = 256;  // tiles whose pages a workgroup looks up at once
constexpr int kKv8Lookups = kKv8SegTiles * 4 / kKv8Threads;  // sub-blocks of a segment a thread
constexpr int kKv8GridRows = 32768;   // of a launch: its y dimension, the rest in z
constexpr int kKv8TwoTilesDim = 192;  // head sizes up to which a wavefront's registers hold two row tiles
constexpr float kKv8PShift = 12.0f;  // a weight is held times 2^12 ...
constexpr float kKv8Slack = 3.0f;    // ... and may pass the running maximum by 2^3
constexpr float kKv8Near = 3.0f;     // V scales of a wavefront's look-up are near within 2^3 of one of them ...
constexpr float kKv8NearRefs = 4.0f;   // ... and those of a part if those ones are within 2^4 of each other
constexpr float kKv8NearLeast = -80.0f;  // and none is below 2^-80, where the sum of weights / scale would overflow

typedef _Float16 half2_t __attribute__((ext_vector_type(2)));
typedef _Float16 half8_t __attribute__((ext_vector_type(8)));
typedef __bf16 bhalf8_t __attribute__((ext_vector_type(8)));
typedef float f32x4_t __attribute__((ext_vector_type(4)));

struct Kv8Attend {
  Kv8Cache c;
  const void* q;
  void* out;
  const int32_t* lengths;
  const void* ids;  // listed chunks [batch, kv_heads, top_k]; null: all tokens
  int32_t chunk;
  int32_t ids64;
  int32_t top_k;
  int32_t subs;        // sub-blocks of a chunk, at most
  int32_t list_tiles;  // tiles of a list
  int32_t dtype;
  int32_t batch;
  int32_t queries;
  int32_t group;
  int32_t rows;        // queries * group
  int32_t row_groups;  // workgroups over the rows
  int32_t row_waves;   // wavefronts of a workgroup over the rows; the others split the tokens
  int32_t parts;       // parts of all sequences, at most
  int32_t round;       // wavefronts over the tokens, a power of two: a part has a multiple of as many tiles
  int32_t min_tiles;   // tiles of a part, at least
  int32_t even_log2;   // workgroups over the tokens, at most about, where lengths are alike ...
  int32_t ragged_log2; // ... and where they are not
  int32_t join_lanes;  // of a joining workgroup, thread groups that share a row's parts
  uint32_t page_groups;  // groups of 16 tokens of a page, 1 to 16 ...
  uint32_t page_magic;   // ... and 2^32 / that, rounded up
  float scale_log2;
  float* part_ml;      // [parts, kv_heads, rows, 4]: m, the sum's maximum, the sum, unused
  float* part_o;       // [parts, kv_heads, rows, D]
};

// Where part `part` lies: its sequence, its tiles, and how many parts the
// sequence has (`count`, from index `first` on).
struct Kv8Part {
  int32_t batch, begin, end, count, first;
};

__device__ __forceinline__ int32_t kv8_length(const Kv8Attend& a, int64_t b) {
  const int32_t cap = a.c.blocks * a.c.page_size;
  return min(max(a.lengths[b], 0), cap);
}

// Inclusive prefix sum over the lanes (rows of 16 shifted by 1, 2, 4, 8, then the
// last lanes of rows and halves passed on).
__device__ __forceinline__ int32_t kv8_wave_scan(int32_t v) {
  v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xf, 0xf, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xf, 0xf, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xf, 0xf, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xf, 0xf, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xa, 0xf, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xc, 0xf, false);
  return v;
}

__device__ __forceinline__ int32_t kv8_wave_sum(int32_t v) { return __builtin_amdgcn_readlane(kv8_wave_scan(v), kWave - 1); }

__device__ __forceinline__ int32_t kv8_tiles(const Kv8Attend& a, int32_t b) {
  return b < a.batch ? (kv8_length(a, b) + kKv8Tile - 1) / kKv8Tile : 0;
}

// Tiles of a part: one size for all sequences, from the lengths on the device, in
// whole rounds of the wavefronts that split the tokens.  Lengths that are alike
// are divided among 2^even_log2 workgroups, which run at once; ragged ones among
// 2^ragged_log2, so that the last to run are short.  Every wavefront works it out
// by itself, a lane a sequence; `mine` is the lane's tiles of the last 64
// sequences (of all, where the batch is not larger).
__device__ __forceinline__ int32_t kv8_part_size(const Kv8Attend& a, int32_t* mine) {
  const int lane = threadIdx.x % kWave;
  int64_t total = 0;
  int32_t most = 0;
  for (int base = 0; base < a.batch; base += kWave) {
    *mine = kv8_tiles(a, base + lane);
    total += kv8_wave_sum(*mine);
    most = max(most, *mine);
  }
#pragma unroll
  for (int d = 32; d >= 1; d /= 2) most = max(most, __float_as_int(xor_lanes(__int_as_float(most), d)));
  const int log2 = static_cast<int64_t>(most) * a.batch <= total + total / 8 ? a.even_log2 : a.ragged_log2;
  const int64_t per = (total * a.c.kv_heads * a.row_groups + (int64_t{1} << log2) - 1) >> log2;
  return (max(a.min_tiles, static_cast<int32_t>(min(per, int64_t{1} << 30))) + a.round - 1) & -a.round;
}

// The part of index `part` over all sequences, each of which has at least one
// (batch -1: there are fewer).
__device__ __forceinline__ Kv8Part kv8_locate(const Kv8Attend& a, int32_t part) {
  if (a.ids) {
    const int32_t count = (a.list_tiles + a.min_tiles - 1) / a.min_tiles, j = part % count;
    return {part / count, j * a.min_tiles, min((j + 1) * a.min_tiles, a.list_tiles), count, part - j};
  }
  const int lane = threadIdx.x % kWave;
  int32_t tiles = 0, first = 0;
  const int32_t size = kv8_part_size(a, &tiles);
  for (int base = 0; base < a.batch; base += kWave) {
    if (a.batch > kWave) tiles = kv8_tiles(a, base + lane);
    const int32_t count = base + lane < a.batch ? max((tiles + size - 1) / size, 1) : 0;
    const int32_t upto = kv8_wave_scan(count);
    const uint64_t hit = __ballot(first + upto > part);
    if (hit) {
      const int at = __ffsll(static_cast<unsigned long long>(hit)) - 1;
      const int32_t n = __builtin_amdgcn_readlane(count, at), from = first + __builtin_amdgcn_readlane(upto, at) - n;
      const int32_t j = part - from;
      return {base + at, j * size, min((j + 1) * size, __builtin_amdgcn_readlane(tiles, at)), n, from};
    }
    first += __builtin_amdgcn_readlane(upto, kWave - 1);
  }
  return {-1, 0, 0, 0, 0};
}

// How many parts sequence b has, and the index of its first.
__device__ __forceinline__ void kv8_parts_of(const Kv8Attend& a, int32_t b, int32_t* count, int32_t* first) {
  if (a.ids) {
    *count = (a.list_tiles + a.min_tiles - 1) / a.min_tiles;
    *first = b * *count;
    return;
  }
  const int lane = threadIdx.x % kWave;
  int32_t tiles = 0;
  const int32_t size = kv8_part_size(a, &tiles);
  *first = 0;
  for (int base = 0; base <= b; base += kWave) {
    if (a.batch > kWave) tiles = kv8_tiles(a, base + lane);
    const int32_t mine = base + lane <= b ? max((tiles + size - 1) / size, 1) : 0;
    *first += kv8_wave_sum(mine);
    *count = __builtin_amdgcn_readlane(mine, b % kWave);
  }
  *first -= *count;
}

// A sub-block: its index in the caches (bytes / (16 D)), its valid tokens
// [lo, hi), and the index of its scales (-1: no valid token).
struct Kv8Sub {
  uint32_t at;
  uint32_t lohi;
  int32_t scale;
};
constexpr uint32_t kKv8Whole = 16u << 8;

// Sub-block u of sequence b (n tokens) or, with a list, of its chunks.
__device__ __forceinline__ Kv8Sub kv8_resolve(const Kv8Attend& a, int32_t b, int32_t h, int32_t n, uint32_t u) {
  const Kv8Cache& c = a.c;
  uint32_t group = u;  // of 16 tokens, within the sequence
  int32_t lo = 0, hi = 0;
  if (a.ids) {
    const uint32_t j = u / static_cast<uint32_t>(a.subs);
    if (j < static_cast<uint32_t>(a.top_k)) {
      const int64_t at = (static_cast<int64_t>(b) * c.kv_heads + h) * a.top_k + j;
      const int64_t id = a.ids64 ? static_cast<const int64_t*>(a.ids)[at] : static_cast<const int32_t*>(a.ids)[at];
      if (id >= 0 && id <= static_cast<uint32_t>(n) / static_cast<uint32_t>(a.chunk)) {  // so that its first token is at most n
        const int32_t from = static_cast<int32_t>(id) * a.chunk, to = from + min(a.chunk, n - from);
        group = from / kKv8Group + (u - j * a.subs);
        lo = max(from - static_cast<int32_t>(group) * kKv8Group, 0);
        hi = max(min(to - static_cast<int32_t>(group) * kKv8Group, kKv8Group), 0);
      }
    }
  } else {
    hi = max(min(n - static_cast<int32_t>(u) * kKv8Group, kKv8Group), 0);
  }
  Kv8Sub s{0u, 0u, -1};
  if (hi > lo) {
    // group / (groups of a page): exact, as group < 2^27 and the divisor is at most 16
    const uint32_t block = a.page_groups == 1 ? group : __umulhi(group, a.page_magic);
    const int32_t page = kv8_page(c, b, block);
    if (page >= 0) {
      s.scale = page * c.kv_heads + h;
      s.at = static_cast<uint32_t>(s.scale) * a.page_groups + (group - block * a.page_groups);
      s.lohi = static_cast<uint32_t>(lo) | static_cast<uint32_t>(hi) << 8;
    }
  }
  return s;
}

// The upper halves of two fp32 values: bf16, cut off.
__device__ __forceinline__ uint32_t kv8_upper_halves(float lo, float hi) {
  return __builtin_amdgcn_perm(__float_as_uint(hi), __float_as_uint(lo), 0x07060302u);
}

// An address as the compiler cannot see through it (loads from it stay where
// they are), and a load at a constant offset from one.
__device__ __forceinline__ uint64_t kv8_opaque(const void* p) {
  uint64_t a = reinterpret_cast<uint64_t>(p);
  asm volatile("" : "+v"(a));
  return a;
}
template <typename V, bool kStream>
__device__ __forceinline__ V kv8_load(uint64_t base, int offset) {
  const auto* p = reinterpret_cast<const __attribute__((address_space(1))) V*>(base + offset);
  if constexpr (kStream) return __builtin_nontemporal_load(p);
  return *p;
}

// The larger of three in one instruction (fmaxf twice also quiets each operand).
__device__ __forceinline__ float kv8_max3(float a, float b, float c) {
  float r;
  asm("v_max3_f32 %0, %1, %2, %3" : "=v"(r) : "v"(a), "v"(b), "v"(c));
  return r;
}

// log2 of V scales, of a lane's sub-blocks or a part's: the least and the largest.
struct Kv8Range {
  float lo = FLT_MAX, hi = -FLT_MAX;
};

// One of a wavefront's, +inf where they are not near that one, NaN where there are none.
__device__ __forceinline__ float kv8_scale_ref(const Kv8Range& lane) {
  const uint64_t has = __ballot(lane.hi > -FLT_MAX);
  if (has == 0) return __builtin_nanf("");
  const float ref = __int_as_float(
      __builtin_amdgcn_readlane(__float_as_int(lane.hi), __ffsll(static_cast<unsigned long long>(has)) - 1));
  const bool far = lane.lo < fmaxf(ref - kKv8Near, kKv8NearLeast) || lane.hi > ref + kKv8Near;
  return __ballot(far) ? __builtin_inff() : ref;
}

// Whether the V scales of a part are far apart, with the refs of N more wavefronts.
template <int N>
__device__ __forceinline__ bool kv8_far_scales(const float* refs, Kv8Range* part) {
#pragma unroll
  for (int i = 0; i < N; i += 4) {
    const f32x4_t ref = *reinterpret_cast<const f32x4_t*>(refs + i);
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      part->lo = fminf(part->lo, ref[k]);
      part->hi = fmaxf(part->hi, ref[k]);
    }
  }
  return __ballot(part->hi - part->lo > kKv8NearRefs) != 0;
}

// 0x80 in each byte that is an e4m3 NaN.
__device__ __forceinline__ uint32_t kv8_nan_bytes(uint32_t w) { return ((w & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u; }

// Eight bytes as eight f16 (kF32: bf16), which is exact.
template <typename F, bool kF32>
__device__ __forceinline__ u32x4_t kv8_operand(uint32_t lo, uint32_t hi) {
  u32x4_t r;
  if constexpr (std::is_same_v<F, E4m3> && !kF32) {
    r[0] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(lo, 1.0f, false));
    r[1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(lo, 1.0f, true));
    r[2] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(hi, 1.0f, false));
    r[3] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(hi, 1.0f, true));
  } else if constexpr (std::is_same_v<F, E4m3>) {
    r[0] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, 1.0f, false));
    r[1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, 1.0f, true));
    r[2] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, 1.0f, false));
    r[3] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, 1.0f, true));
  } else if constexpr (!kF32) {
    // b + 128 under the exponent of 1024 is the f16 1152 + b
    const half2_t off = {static_cast<_Float16>(1152.0f), static_cast<_Float16>(1152.0f)};
    const uint32_t w[2] = {lo ^ 0x80808080u, hi ^ 0x80808080u};
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      r[2 * i] = __builtin_bit_cast(
          uint32_t, __builtin_bit_cast(half2_t, __builtin_amdgcn_perm(0x64646464u, w[i], 0x04010400u)) - off);
      r[2 * i + 1] = __builtin_bit_cast(
          uint32_t, __builtin_bit_cast(half2_t, __builtin_amdgcn_perm(0x64646464u, w[i], 0x04030402u)) - off);
    }
  } else {
    const uint32_t w[2] = {lo, hi};
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      r[2 * i] = kv8_upper_halves(kv8_decode<Int8, 0>(w[i]), kv8_decode<Int8, 1>(w[i]));
      r[2 * i + 1] = kv8_upper_halves(kv8_decode<Int8, 2>(w[i]), kv8_decode<Int8, 3>(w[i]));
    }
  }
  return r;
}

template <bool kF32>
__device__ __forceinline__ f32x4_t kv8_mfma(u32x4_t a, u32x4_t b, f32x4_t c) {
  if constexpr (kF32) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bhalf8_t, a), __builtin_bit_cast(bhalf8_t, b), c, 0,
                                                   0, 0);
  } else {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(half8_t, a), __builtin_bit_cast(half8_t, b), c, 0, 0,
                                                  0);
  }
}

// Eight fp32 values as operands: one f16 each, or three bf16 that add up to it
// (the upper 8 bits, those of what is left, and the last ones).
template <bool kF32, int NP>
__device__ __forceinline__ void kv8_split(const float (&v)[8], u32x4_t (&out)[NP]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (kF32) {
      float x = v[2 * i], y = v[2 * i + 1];
#pragma unroll
      for (int p = 0; p < NP; ++p) {
        out[p][i] = kv8_upper_halves(x, y);
        x -= __uint_as_float(__float_as_uint(x) & 0xffff0000u);
        y -= __uint_as_float(__float_as_uint(y) & 0xffff0000u);
      }
    } else {
      const half2_t h = {static_cast<_Float16>(v[2 * i]), static_cast<_Float16>(v[2 * i + 1])};
      out[0][i] = __builtin_bit_cast(uint32_t, h);
    }
  }
}

// Four values to the output, rounded to its type.
__device__ __forceinline__ void kv8_store4(const Kv8Attend& a, int64_t at, f32x4_t y) {
  if (a.dtype == CSAHCA_F32) {
    *reinterpret_cast<f32x4_t*>(static_cast<float*>(a.out) + at) = y;
  } else {
    uint16_t r[4];
#pragma unroll
    for (int e = 0; e < 4; ++e)
      r[e] = a.dtype == CSAHCA_F16 ? __builtin_bit_cast(uint16_t, static_cast<f16>(y[e])) : float_to_bf16_bits(y[e]);
    *reinterpret_cast<uint2*>(static_cast<uint16_t*>(a.out) + at) =
        make_uint2(r[0] | static_cast<uint32_t>(r[1]) << 16, r[2] | static_cast<uint32_t>(r[3]) << 16);
  }
}

// The sums 2^up acc / total, 0 where there are none.
__device__ __forceinline__ f32x4_t kv8_result(f32x4_t acc, float total, float up) {
  acc *= total != 0.f ? 1.0f / total : 0.f;
#pragma unroll
  for (int i = 0; i < 4; ++i) acc[i] = __builtin_ldexpf(acc[i], static_cast<int>(up));
  return acc;
}

// Workgroups of a CU: two while a wavefront's registers (K, V, the sums, q, scores
// and weights, counted in the second line) fit 256 beside some 70 others: 64 rows of
// 96 over 8 x 16384 tokens 51 us, one workgroup 58; of 128, which do not fit, 88 / 68;
// 64 rows of 192 one by one 126 / 122.  In between are f32 rows of 128: 16 rows
// 53 / 50, 32 rows, which share the loads, 34 / 38.
template <int D, int NP, int NT, bool kStream>
constexpr int kKv8Blocks =
    D / 4 * (2 + NT) + NP * NT * D / 8 + 16 * NT + 8 * NP * NT <= (kStream ? 180 : 190) ? 2 : 1;

// Bound by the read stream where there are tokens enough: 32 x 32768 tokens, 8 heads of
// 128, 2.15 GB, 322 us (6.7 TB/s); 16 ragged ones of 4 rows 75 (5.7).  A wavefront keeps a
// tile's K and V (16 KB at heads of 128) in flight while it works on the one before, two
// workgroups a CU 128 KB.  1 x 8192 tokens take 9 us: lengths, table, scales and the tile,
// a round trip each.
//
// kStream: no other wavefront reads a tile (one over the rows), and its loads go
// past the caches: 32 x 32768 tokens 370 us without and 344 with (6.2 TB/s), 16 ragged
// 78.6 / 73.4, 32 rows over 8 x 16384 tokens 59 / 54, of 192 84 / 77 (of 64 27 / 28);
// where wavefronts share tiles it costs (heads of 256 in 4 wavefronts of 16 rows:
// 57.7 / 81.3).
template <int D, typename F, bool kF32, int NT, bool kStream>
__global__ __launch_bounds__(kKv8Threads, (kKv8Blocks<D, kF32 ? 3 : 1, NT, kStream>)) void kv8_attend_kernel(const Kv8Attend a) {
  constexpr int NP = kF32 ? 3 : 1;         // operands that make up a value of q or a weight
  constexpr int kSteps = D / 32;           // matrix instructions over D
  constexpr int kWide = D / 64;            // 16-byte loads of a K row
  constexpr bool kTail = D % 64 != 0;      // and one of 8 bytes
  constexpr int kDTiles = D / 16;
  constexpr int kRowPad = D + 4;
  constexpr size_t kMergeBytes = sizeof(float) * kKv8Waves * 16 * kRowPad;
  constexpr size_t kSubBytes = 20 * kKv8SegTiles * 4;
  __shared__ __attribute__((aligned(16))) char lds[kMergeBytes > kSubBytes ? kMergeBytes : kSubBytes];
  __shared__ float4 lds_ml[kKv8Waves][16];  // the maximum, the sum's maximum, the sum
  __shared__ float lds_ms[kKv8Waves][NT * 16];  // where V scales are far apart, the sums' maxima
  __shared__ __attribute__((aligned(16))) float refs[kKv8Waves];  // of a segment's V scales
  uint2* sub_at = reinterpret_cast<uint2*>(lds);                          // index, valid tokens
  float2* sub_scale = reinterpret_cast<float2*>(lds) + kKv8SegTiles * 4;  // K scale, log2 of the V scale
  float* sub_inv = reinterpret_cast<float*>(lds) + kKv8SegTiles * 16;     // 1 / V scale

  const int lane = threadIdx.x % kWave, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int n = lane % 16, g = lane / 16;
  // Workgroups in order of heads (which lie next to each other in memory), row
  // groups and parts.
  const int32_t h = blockIdx.x, at_part = blockIdx.z * kKv8GridRows + blockIdx.y;
  const int32_t part_index = a.row_groups == 1 ? at_part : at_part / a.row_groups, rg = at_part - part_index * a.row_groups;
  if (part_index >= a.parts) return;
  const Kv8Part part = kv8_locate(a, part_index);
  if (part.batch < 0) return;  // fewer parts than the launch allows for
  const int32_t b = part.batch;
  const int32_t len = kv8_length(a, b);
  const int32_t token_waves = kKv8Waves / a.row_waves;
  const int32_t row0 = (rg * a.row_waves + wave / token_waves) * (NT * 16);
  const int32_t heads = a.c.kv_heads * a.group;

  // The lane's dimensions of row n of each row tile, as they are stored.
  constexpr int kRaw = kF32 ? 2 : 1;  // 16-byte loads of eight values
  u32x4_t raw[NT][kSteps][kRaw];
  int32_t limit[NT];  // tokens the row sees
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    const int32_t r = min(row0 + nt * 16 + n, a.rows - 1);
    const int32_t qi = a.queries == 1 ? 0 : r / a.group;
    const int64_t at = ((static_cast<int64_t>(b) * a.queries + qi) * heads + h * a.group + (r - qi * a.group)) * D;
    limit[nt] = max(len - a.queries + 1 + qi, 0);
#pragma unroll
    for (int k = 0; k < kSteps; ++k) {
      const int d = kTail && k == kSteps - 1 ? kWide * 64 + g * 8 : k / 2 * 64 + g * 16 + k % 2 * 8;
#pragma unroll
      for (int p = 0; p < kRaw; ++p)
        raw[nt][k][p] = load_global_raw<u32x4_t>(static_cast<const uint8_t*>(a.q) + (at + d) * 2 * kRaw + 16 * p);
    }
  }

  int32_t end = part.end;
  if (!a.ids) {  // the last row of the workgroup sees the most
    const int32_t last = min((rg + 1) * a.row_waves * NT * 16, a.rows) - 1;
    end = min(end, (max(len - a.queries + 1 + last / a.group, 0) + kKv8Tile - 1) / kKv8Tile);
  }
  const int32_t least = len - a.queries + 1 + row0 / a.group;  // the wavefront's first row sees the least
  const uint8_t* kbase = a.c.k + (lane % 4) * D + g * 16;
  const uint8_t* ktail = a.c.k + (lane % 4) * D + kWide * 64 + g * 8;
  const uint8_t* vbase = a.c.v + n * kKv8Group;

  u32x4_t kw[4][kWide > 0 ? kWide : 1];
  u32x2_t kt[4];
  u32x4_t vw[kDTiles];
  const auto load_k = [&](uint32_t at) {
    const int64_t off = static_cast<int64_t>(at) * (kKv8Group * D);
    const uint64_t wide = kv8_opaque(kbase + off), tail = kv8_opaque(ktail + off);
#pragma unroll
    for (int t = 0; t < 4; ++t) {
#pragma unroll
      for (int w = 0; w < kWide; ++w) kw[t][w] = kv8_load<u32x4_t, kStream>(wide, 4 * t * D + 64 * w);
      if constexpr (kTail) kt[t] = kv8_load<u32x2_t, kStream>(tail, 4 * t * D);
    }
  };
  const auto load_v = [&](uint32_t at) {
    const uint64_t base = kv8_opaque(vbase + static_cast<int64_t>(at) * (kKv8Group * D));
#pragma unroll
    for (int dt = 0; dt < kDTiles; ++dt) vw[dt] = kv8_load<u32x4_t, kStream>(base, dt * 16 * kKv8Group);
  };

  // The pages of the segment's sub-blocks, then this wavefront's first loads and
  // the sub-blocks' scales, which only the scores wait for.
  float ks[kKv8Lookups], vs[kKv8Lookups];  // vs 0: none
  const int32_t first = wave % token_waves;
  const auto look_up = [&](int32_t seg, int32_t tiles) {
#pragma unroll
    for (int i = 0; i < kKv8Lookups; ++i) {
      const int at = i * kKv8Threads + threadIdx.x;
      ks[i] = 0.f;
      vs[i] = 0.f;
      if (at < tiles * 4) {
        const Kv8Sub sub = kv8_resolve(a, b, h, len, static_cast<uint32_t>(seg) * 4 + at);
        sub_at[at] = make_uint2(sub.at, sub.lohi);
        if (sub.scale >= 0) {
          ks[i] = a.c.k_scale[sub.scale];
          vs[i] = fmaxf(a.c.v_scale[sub.scale], FLT_MIN);
        }
      }
    }
    lds_barrier();
    if (first < tiles) {
      load_k(sub_at[first * 4 + n / 4].x);
      load_v(sub_at[first * 4 + g].x);
    }
  };
  // Before q is converted, where there are registers to hold both.
  constexpr bool kEarly = NT == 1 && D <= 128;
  if constexpr (kEarly) look_up(part.begin, min(end - part.begin, kKv8SegTiles));

  // q as operands, in f16 its rows scaled to below 2^15
  u32x4_t q[NT][kSteps][NP];
  float rc[NT], m[NT], l[NT];
  f32x4_t o[NT][kDTiles];
  const float sign = a.scale_log2 < 0.f ? -1.f : 1.f;
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    float v[kSteps][8], top = 0.f;
#pragma unroll
    for (int k = 0; k < kSteps; ++k) {
      const u32x4_t w = raw[nt][k][0];
      if constexpr (kF32) {
        const u32x4_t w1 = raw[nt][k][1];
        widen16<float>(make_uint4(w[0], w[1], w[2], w[3]), v[k]);
        widen16<float>(make_uint4(w1[0], w1[1], w1[2], w1[3]), v[k] + 4);
      } else if (a.dtype == CSAHCA_F16) {
        widen16<f16>(make_uint4(w[0], w[1], w[2], w[3]), v[k]);
      } else {
        widen16<bf16>(make_uint4(w[0], w[1], w[2], w[3]), v[k]);
      }
    }
    // times 2^down: 16-bit rows to below 2^15, f32 rows beyond 2^60 to that, so that no product overflows
#pragma unroll
    for (int k = 0; k < kSteps; ++k)
#pragma unroll
      for (int e = 0; e < 8; ++e) top = fmaxf(top, fabsf(v[k][e]));
    top = fmaxf(top, xor_lanes(top, 16));
    top = fmaxf(top, xor_lanes(top, 32));
    int e2 = 15;
    if (top > 0.f && top < __builtin_inff()) (void)frexpf(top, &e2);
    const int down = kF32 ? min(60 - e2, 0) : 15 - e2;
#pragma unroll
    for (int k = 0; k < kSteps; ++k) {
#pragma unroll
      for (int e = 0; e < 8; ++e) v[k][e] = __builtin_ldexpf(v[k][e] * sign, down);
      kv8_split<kF32>(v[k], q[nt][k]);
    }
    rc[nt] = __builtin_ldexpf(fabsf(a.scale_log2), -down);
    m[nt] = -FLT_MAX;  // finite: a row of NaN scores still reaches the sums
    l[nt] = 0.f;
#pragma unroll
    for (int dt = 0; dt < kDTiles; ++dt) o[nt][dt] = f32x4_t{0.f, 0.f, 0.f, 0.f};
  }
  // The weights' sums by sub-block: row r < 4 of the product takes those of quarter r.
  u32x4_t ones;
#pragma unroll
  for (int i = 0; i < 4; ++i) ones[i] = n != g ? 0u : kF32 ? 0x3f803f80u : 0x3c003c00u;
  if constexpr (!kEarly) look_up(part.begin, min(end - part.begin, kKv8SegTiles));

  bool far = false;
  Kv8Range scales;
  for (int32_t seg = part.begin; seg < end;) {
    const int32_t seg_end = min(end - seg, kKv8SegTiles);
    Kv8Range range;
#pragma unroll
    for (int i = 0; i < kKv8Lookups; ++i) {
      if (i * kKv8Threads >= seg_end * 4) break;
      const int at = i * kKv8Threads + threadIdx.x;
      const float lv = __builtin_amdgcn_logf(vs[i]);
      if (vs[i] > 0.f) range = {fminf(range.lo, lv), fmaxf(range.hi, lv)};
      if (at < seg_end * 4) {
        sub_scale[at] = make_float2(ks[i], vs[i] > 0.f ? lv : 0.f);
        sub_inv[at] = vs[i] > 0.f ? fast_exp2(-lv) : 0.f;
      }
    }
    const float ref = kv8_scale_ref(range);
    if (lane == 0) refs[wave] = ref;
    lds_barrier();
    if (kv8_far_scales<kKv8Waves>(refs, &scales) && !far) {
      far = true;
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) lds_ms[wave][nt * 16 + n] = m[nt];
    }

    // One tile; its successor's K and V are loaded as its own are done with.
    const auto tile_step = [&](int32_t tile, auto more) {
      const uint32_t lohi = sub_at[tile * 4 + g].y;
      const float2 scale = sub_scale[tile * 4 + g];
      uint32_t next_k = 0u, next_v = 0u;
      if constexpr (more.value) {
        next_k = sub_at[(tile + token_waves) * 4 + n / 4].x;
        next_v = sub_at[(tile + token_waves) * 4 + g].x;
      }

      f32x4_t s[NT][4];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int t = 0; t < 4; ++t) s[nt][t] = f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int k = 0; k < kSteps; ++k)
#pragma unroll
        for (int t0 = 0; t0 < 4; t0 += 2) {
          u32x4_t ka[2];
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            const int t = t0 + j;
            if (kTail && k == kSteps - 1) {
              ka[j] = kv8_operand<F, kF32>(kt[t][0], kt[t][1]);
            } else if (k % 2 == 0) {
              ka[j] = kv8_operand<F, kF32>(kw[t][k / 2][0], kw[t][k / 2][1]);
            } else {
              ka[j] = kv8_operand<F, kF32>(kw[t][k / 2][2], kw[t][k / 2][3]);
            }
          }
#pragma unroll
          for (int p = 0; p < NP; ++p)
#pragma unroll
            for (int j = 0; j < 2; ++j)
#pragma unroll
              for (int nt = 0; nt < NT; ++nt) s[nt][t0 + j] = kv8_mfma<kF32>(ka[j], q[nt][k][p], s[nt][t0 + j]);
        }
      if constexpr (more.value) load_k(next_k);

      const int32_t lo = lohi & 0xff, hi = lohi >> 8;
      const bool edge = __ballot(lohi != kKv8Whole) != 0 || (!a.ids && (seg + tile + 1) * kKv8Tile > least);
      if (edge) {
        const int32_t token = (seg + tile) * kKv8Tile + g * kKv8Group;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          const int32_t to = a.ids ? hi : min(hi, limit[nt] - token);
#pragma unroll
          for (int i = 0; i < 16; ++i)
            s[nt][i / 4][i % 4] = i >= lo && i < to ? s[nt][i / 4][i % 4] : -__builtin_inff();
        }
        // bytes behind the sequence may be NaN, which a weight of 0 does not hide
        uint32_t keep[4];
#pragma unroll
        for (int w = 0; w < 4; ++w) {
          keep[w] = 0;
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (4 * w + e >= lo && 4 * w + e < hi) keep[w] |= 0xffu << (8 * e);
        }
#pragma unroll
        for (int dt = 0; dt < kDTiles; ++dt)
#pragma unroll
          for (int w = 0; w < 4; ++w) vw[dt][w] &= keep[w];
        if (std::is_same_v<F, E4m3> && !a.ids && a.queries > 1) {
          // A token that later queries see may hold NaN too: it is taken out, and the
          // sums of the rows that do see it are made NaN by a product of ones.
          uint32_t any = 0;
#pragma unroll
          for (int dt = 0; dt < kDTiles; ++dt)
#pragma unroll
            for (int w = 0; w < 4; ++w) any |= kv8_nan_bytes(vw[dt][w]);
          if (__builtin_expect(__ballot(any != 0) != 0, 0)) {
            u32x4_t seen[NT][2];
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
              const int32_t to = min(hi, limit[nt] - token);
#pragma unroll
              for (int i = 0; i < 8; ++i) {
                const uint32_t one = kF32 ? 0x3f80u : 0x3c00u;
                seen[nt][i / 4][i % 4] = (2 * i >= lo && 2 * i < to ? one : 0u) |
                                         (2 * i + 1 >= lo && 2 * i + 1 < to ? one << 16 : 0u);
              }
            }
#pragma unroll
            for (int dt = 0; dt < kDTiles; ++dt) {
              uint32_t nan[4];
#pragma unroll
              for (int w = 0; w < 4; ++w) {
                nan[w] = kv8_nan_bytes(vw[dt][w]) >> 7;
                vw[dt][w] &= ~(nan[w] * 0xffu);
                nan[w] *= 0x38u;  // 1.0
              }
#pragma unroll
              for (int nt = 0; nt < NT; ++nt) {
                f32x4_t hit{0.f, 0.f, 0.f, 0.f};
                hit = kv8_mfma<kF32>(kv8_operand<F, kF32>(nan[0], nan[1]), seen[nt][0], hit);
                hit = kv8_mfma<kF32>(kv8_operand<F, kF32>(nan[2], nan[3]), seen[nt][1], hit);
#pragma unroll
                for (int i = 0; i < 4; ++i) o[nt][dt][i] = hit[i] > 0.f ? __builtin_nanf("") : o[nt][dt][i];
              }
            }
          }
        }
      }

      // The factor of a lane's scores is not negative, so their maximum is that of
      // the products (and not 0, so that a masked one stays -inf).
      float c[NT], top[NT];
      bool up = false;
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        c[nt] = fmaxf(scale.x * rc[nt], FLT_MIN);
        float most = s[nt][3][3];
#pragma unroll
        for (int i = 0; i < 14; i += 2) most = kv8_max3(most, s[nt][i / 4][i % 4], s[nt][(i + 1) / 4][(i + 1) % 4]);
        most = fmaxf(most, s[nt][3][2]);
        most = fmaf(most, c[nt], scale.y);
        most = fmaxf(most, xor_lanes(most, 16));
        top[nt] = fmaxf(most, xor_lanes(most, 32));
        up = up || top[nt] > m[nt] + kKv8Slack;
      }
      if (__ballot(up)) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          top[nt] = ceilf(fmaxf(top[nt], m[nt]));
          const float fix = fast_exp2(m[nt] - top[nt]);
          if (!far) l[nt] *= fix;
#pragma unroll
          for (int dt = 0; dt < kDTiles; ++dt) o[nt][dt] *= fix;
          m[nt] = top[nt];
        }
      }
      if (__builtin_expect(far, 0)) {
        // The weights for the sum by themselves, beside their own maximum.
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          float most = -FLT_MAX;
#pragma unroll
          for (int i = 0; i < 16; ++i) most = fmaxf(most, s[nt][i / 4][i % 4] * c[nt]);
          most = fmaxf(most, xor_lanes(most, 16));
          most = fmaxf(most, xor_lanes(most, 32));
          const float was = lds_ms[wave][nt * 16 + n], up = fmaxf(was, ceilf(most));
          float sum = 0.f;
#pragma unroll
          for (int i = 0; i < 16; ++i) sum += fast_exp2(fmaf(s[nt][i / 4][i % 4], c[nt], kKv8PShift - up));
          l[nt] = fmaf(l[nt], fast_exp2(was - up), sum);
          lds_ms[wave][nt * 16 + n] = up;
        }
      }
      const f32x4_t inv_vs = *reinterpret_cast<const f32x4_t*>(sub_inv + tile * 4);
      u32x4_t pa[NT][2][NP];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        const float base = scale.y - m[nt] + kKv8PShift;
        f32x4_t sum{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          float p[8];
#pragma unroll
          for (int e = 0; e < 8; ++e) p[e] = fast_exp2(fmaf(s[nt][2 * half + e / 4][e % 4], c[nt], base));
          kv8_split<kF32>(p, pa[nt][half]);
#pragma unroll
          for (int i = 0; i < NP; ++i) sum = kv8_mfma<kF32>(ones, pa[nt][half][i], sum);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) l[nt] = fmaf(sum[i], far ? 0.f : inv_vs[i], l[nt]);
      }
#pragma unroll
      for (int dt = 0; dt < kDTiles; dt += 2) {
        u32x4_t va[2][2];
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          va[j][0] = kv8_operand<F, kF32>(vw[dt + j][0], vw[dt + j][1]);
          va[j][1] = kv8_operand<F, kF32>(vw[dt + j][2], vw[dt + j][3]);
        }
#pragma unroll
        for (int half = 0; half < 2; ++half)
#pragma unroll
          for (int i = 0; i < NP; ++i)
#pragma unroll
            for (int j = 0; j < 2; ++j)
#pragma unroll
              for (int nt = 0; nt < NT; ++nt) o[nt][dt + j] = kv8_mfma<kF32>(va[j][half], pa[nt][half][i], o[nt][dt + j]);
      }
      if constexpr (more.value) load_v(next_v);
    };
    int32_t tile = first;
    for (; tile + token_waves < seg_end; tile += token_waves) tile_step(tile, std::true_type{});
    if (tile < seg_end) tile_step(tile, std::false_type{});
    seg += kKv8SegTiles;
    if (seg < end) {
      lds_barrier();  // the segment's entries are done with
      look_up(seg, min(end - seg, kKv8SegTiles));
    }
  }

  // The wavefronts that split the tokens are joined, a row tile at a time.
  float* merge = reinterpret_cast<float*>(lds);
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    float sum = l[nt];
    sum += xor_lanes(sum, 16);
    sum += xor_lanes(sum, 32);
    __syncthreads();
#pragma unroll
    for (int dt = 0; dt < kDTiles; ++dt)
      *reinterpret_cast<f32x4_t*>(merge + (wave * 16 + n) * kRowPad + dt * 16 + g * 4) = o[nt][dt];
    if (g == 0) {
      lds_ml[wave][n] = make_float4(m[nt], far ? lds_ms[wave][nt * 16 + n] : m[nt], sum, 0.f);
    }
    __syncthreads();
    // thread: (row wavefront, row, four dimensions)
    for (int i = threadIdx.x; i < a.row_waves * 16 * (D / 4); i += kKv8Threads) {
      const int d = i % (D / 4) * 4, row = i / (D / 4) % 16, w0 = i / (D / 4 * 16) * token_waves;
      const int32_t r = (rg * a.row_waves + w0 / token_waves) * (NT * 16) + nt * 16 + row;
      if (r >= a.rows) continue;
      float top = -FLT_MAX, stop = -FLT_MAX, total = 0.f;
      for (int w = 0; w < token_waves; ++w) {
        top = fmaxf(top, lds_ml[w0 + w][row].x);
        stop = fmaxf(stop, lds_ml[w0 + w][row].y);
      }
      f32x4_t acc{0.f, 0.f, 0.f, 0.f};
      for (int w = 0; w < token_waves; ++w) {
        const float4 ml = lds_ml[w0 + w][row];
        total = fmaf(ml.z, fast_exp2(ml.y - stop), total);
        acc += *reinterpret_cast<const f32x4_t*>(merge + ((w0 + w) * 16 + row) * kRowPad + d) * fast_exp2(ml.x - top);
      }
      if (part.count > 1) {
        const int64_t slot = (static_cast<int64_t>(part_index) * a.c.kv_heads + h) * a.rows + r;
        *reinterpret_cast<f32x4_t*>(a.part_o + slot * D + d) = acc;
        if (d == 0) *reinterpret_cast<float4*>(a.part_ml + 4 * slot) = make_float4(top, stop, total, 0.f);
      } else {
        const int32_t qi = a.queries == 1 ? 0 : r / a.group;
        const int64_t at =
            ((static_cast<int64_t>(b) * a.queries + qi) * heads + h * a.group + (r - qi * a.group)) * D + d;
        kv8_store4(a, at, kv8_result(acc, total, top - stop));
      }
    }
  }
}

// ---------------------------------------------------------------------------
// Many rows (prompt chunks): 32 rows a wavefront, eight wavefronts a workgroup
// (four above 128 dimensions).
//
// A matrix instruction keeps its SIMD from vector instructions for half its time
// and those behind it in its wavefront wait with it: beside a 16x16x32 product
// about two vector instructions are free and each further one costs its time,
// beside a 32x32x16 (as many operands, twice the work) six are.  So this kernel
// takes 32x32x16 and sets six vector instructions behind each: the weights of a
// tile beside the scores of the next, and beside the sums the maximum of the next
// and the operands of tiles to come.  Those a workgroup's wavefronts make
// together, each converting its share of a tile's bytes once and passing it on
// through LDS (two tiles of K and of V, one barrier a tile).  Measured, 2 x 512
// queries over 16384 tokens, heads 32 / 8 of 128, 271 GFLOP: the kernel above with
// 32 rows a wavefront 329 us; 32x32x16 and shared operands, phase after phase, 337;
// interleaved 313; eight wavefronts instead of four 278 (972 TFLOP/s; a library
// product of 8192^3 in f16 reaches 1250); NaN bytes and scales far apart 284.  By
// counters a SIMD's matrix instructions take 124 us and its vector instructions 146,
// with little overlap.  Taken out one at a time, writing operands to LDS is 47 us,
// reading them 20, the loads 22, exponentials 20.
//
// Lane l holds row n = l % 32; its half g = l / 32 the tokens of sub-block g of
// each 32 of a tile: row 8b + 4g + j of a K tile is token 4b + j of sub-block g,
// so the lane's scores are its sub-block's 16 tokens, and its weights the second
// product's operand, first 8 and last 8.
// ---------------------------------------------------------------------------
typedef float f32x16_t __attribute__((ext_vector_type(16)));

__device__ __forceinline__ f32x16_t kv8_mfma32(u32x4_t a, u32x4_t b, f32x16_t c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(half8_t, a), __builtin_bit_cast(half8_t, b), c, 0, 0, 0);
}

// Wavefronts of a workgroup: two a SIMD while a wavefront's registers fit 256.
constexpr int kv8_rows_waves(int64_t head_dim) { return head_dim <= 128 ? 8 : 4; }

template <int D, typename F>
__global__ __launch_bounds__(kv8_rows_waves(D) * kWave) void kv8_attend_rows_kernel(const Kv8Attend a) {
  constexpr int kWaves = kv8_rows_waves(D);
  constexpr int kTiles = kWaves * kWave / 4;  // tiles whose pages are looked up at once: a sub-block a thread
  constexpr int kSteps = D / 16;   // products over D
  constexpr int kChunks = D / 32;  // 16-byte loads of a K row by a lane; 32-row tiles of the output
  constexpr int kPieces = (D / 16 + kWaves - 1) / kWaves;  // of a tile's D / 16 loads of K, those of a wavefront
  // operands of two tiles, of 64 lanes: load p gives operands 2 p and 2 p + 1
  __shared__ u32x4_t kops[2][D / 8][kWave], vops[2][D / 8][kWave];
  __shared__ uint2 sub_at[2][kTiles * 4];      // index, valid tokens
  __shared__ float4 sub_scale[2][kTiles * 4];  // K scale, log2 of the V scale, 1 / V scale
  __shared__ uint64_t sub_cut[2][kWaves];          // sub-blocks that are not whole, a bit each
  __shared__ uint16_t nans[2][D][4];               // tokens of a sub-block whose V is NaN ...
  __shared__ uint32_t nan_at[2][kWaves];           // ... and whether a wavefront found any
  __shared__ float lds_ms[kWaves][32];  // where V scales are far apart, the sums' maxima
  __shared__ __attribute__((aligned(16))) float refs[2][kWaves];  // of a segment's V scales

  const int lane = threadIdx.x % kWave, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int n = lane % 32, g = lane / 32;
  const int32_t h = blockIdx.x, at_part = blockIdx.z * kKv8GridRows + blockIdx.y;
  const int32_t part_index = at_part / a.row_groups, rg = at_part - part_index * a.row_groups;
  if (part_index >= a.parts) return;
  const Kv8Part part = kv8_locate(a, part_index);
  if (part.batch < 0) return;  // fewer parts than the launch allows for
  const int32_t b = part.batch, len = kv8_length(a, b);
  const int32_t row0 = (rg * kWaves + wave) * 32;
  const int32_t heads = a.c.kv_heads * a.group;
  const int32_t r = min(row0 + n, a.rows - 1), qi = r / a.group;
  const int64_t q_at = ((static_cast<int64_t>(b) * a.queries + qi) * heads + h * a.group + (r - qi * a.group)) * D;
  const int32_t limit = max(len - a.queries + 1 + qi, 0);      // tokens the row sees
  const int32_t least = len - a.queries + 1 + row0 / a.group;  // and the wavefront's first row
  // The first row of all waves sees the tokens before this tile.
  const int32_t all_see =
      a.ids ? INT32_MAX : max(len - a.queries + 1 + rg * kWaves * 32 / a.group, 0) / kKv8Tile - part.begin;
  int32_t end = part.end;
  if (!a.ids) {  // the workgroup's last row sees the most
    const int32_t last = min((rg + 1) * kWaves * 32, a.rows) - 1;
    end = min(end, (max(len - a.queries + 1 + last / a.group, 0) + kKv8Tile - 1) / kKv8Tile);
  }

  // q in f16, its row scaled to below 2^15: dimension 32 c + 16 g + 8 half + e
  u32x4_t q[kSteps];
  float rc;
  {
    float v[kSteps][8], top = 0.f;
#pragma unroll
    for (int k = 0; k < kSteps; ++k) {
      const int64_t at = q_at + k / 2 * 32 + g * 16 + k % 2 * 8;
      if (a.dtype == CSAHCA_F16) {
        load16(static_cast<const f16*>(a.q) + at, v[k]);
      } else {
        load16(static_cast<const bf16*>(a.q) + at, v[k]);
      }
#pragma unroll
      for (int e = 0; e < 8; ++e) top = fmaxf(top, fabsf(v[k][e]));
    }
    top = fmaxf(top, xor_lanes(top, 32));
    int e2 = 15;
    if (top > 0.f && top < __builtin_inff()) (void)frexpf(top, &e2);
    const float sign = a.scale_log2 < 0.f ? -1.f : 1.f;
#pragma unroll
    for (int k = 0; k < kSteps; ++k) {
#pragma unroll
      for (int e = 0; e < 8; ++e) v[k][e] = __builtin_ldexpf(v[k][e] * sign, 15 - e2);
      u32x4_t one[1];
      kv8_split<false>(v[k], one);
      q[k] = one[0];
    }
    rc = __builtin_ldexpf(fabsf(a.scale_log2), e2 - 15);
  }
  float m = -FLT_MAX, l = 0.f;
  f32x16_t o[kChunks];
#pragma unroll
  for (int dt = 0; dt < kChunks; ++dt)
#pragma unroll
    for (int i = 0; i < 16; ++i) o[dt][i] = 0.f;

  // Sub-blocks of 64 tiles from tile `seg` on, into buffer `buf`.
  const auto look_up = [&](int32_t seg, int buf) {
    const Kv8Sub sub = kv8_resolve(a, b, h, len, static_cast<uint32_t>(seg) * 4 + threadIdx.x);
    sub_at[buf][threadIdx.x] = make_uint2(sub.at, sub.lohi);
    const uint64_t cut = __ballot(sub.lohi != kKv8Whole);
    if (lane == 0) sub_cut[buf][wave] = cut;
    float ks = 0.f, lv = 0.f;
    Kv8Range range;
    if (sub.scale >= 0) {
      ks = a.c.k_scale[sub.scale];
      lv = __builtin_amdgcn_logf(fmaxf(a.c.v_scale[sub.scale], FLT_MIN));
      range = {lv, lv};
    }
    sub_scale[buf][threadIdx.x] = make_float4(ks, lv, fast_exp2(-lv), 0.f);
    const float ref = kv8_scale_ref(range);
    if (lane == 0) refs[buf][wave] = ref;
  };
  // Entry of a tile's sub-block s (tiles are counted from the part's first).
  const auto entry = [](int32_t tile, int s) { return tile % kTiles * 4 + s; };

  // This wavefront's loads of a tile's K and of its V (behind the last one it
  // repeats that), and their operands into LDS.
  u32x4_t kpiece[kPieces], vpiece[kPieces];
  const auto piece_of = [&](int i) { return min(wave + kWaves * i, D / 16 - 1); };
  const auto k_at = [&](int32_t tile, int i) {
    return sub_at[tile / kTiles % 2][entry(tile, 2 * (piece_of(i) / kChunks) + n / 4 % 2)].x;
  };
  const auto v_at = [&](int32_t tile, int i) {
    return sub_at[tile / kTiles % 2][entry(tile, 2 * (piece_of(i) / kChunks) + g)].x;
  };
  const uint8_t* kbase = a.c.k + (n / 8 * 4 + n % 4) * D + g * 16;
  const uint8_t* vbase = a.c.v + n * kKv8Group;
  const auto fetch_k = [&](int i, uint32_t at) {
    kpiece[i] = load_global_raw<u32x4_t>(kbase + (static_cast<int64_t>(at) * (kKv8Group * D) + piece_of(i) % kChunks * 32));
  };
  const auto fetch_v = [&](int i, uint32_t at) {
    vpiece[i] = load_global_raw<u32x4_t>(
        vbase + (static_cast<int64_t>(at) * (kKv8Group * D) + piece_of(i) % kChunks * 32 * kKv8Group));
  };
  const auto pass_k = [&](int32_t tile, int i, int half) {
    kops[tile % 2][2 * piece_of(i) + half][lane] = kv8_operand<F, false>(kpiece[i][2 * half], kpiece[i][2 * half + 1]);
  };
  const auto pass_v = [&](int32_t tile, int i, int half) {
    vops[tile % 2][2 * piece_of(i) + half][lane] = kv8_operand<F, false>(vpiece[i][2 * half], vpiece[i][2 * half + 1]);
  };
  // Masks a tile's scores, and its bytes of V on the way to LDS: those behind the
  // sequence may be NaN, which a weight of 0 does not hide.
  const auto cut_of = [&](int32_t tile) {
    return reinterpret_cast<const uint8_t*>(sub_cut[tile / kTiles % 2])[tile % kTiles / 2] >> (tile % 2 * 4) & 15;
  };
  const auto mask = [&](int32_t tile, uint32_t cut, f32x16_t (&s)[2]) {
    if (__builtin_amdgcn_readfirstlane(cut) != 0 || (!a.ids && (part.begin + tile + 1) * kKv8Tile > least)) {
      uint32_t lohi[2];
#pragma unroll
      for (int u = 0; u < 2; ++u) lohi[u] = sub_at[tile / kTiles % 2][entry(tile, 2 * u + g)].y;
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const int32_t lo = lohi[u] & 0xff, hi = lohi[u] >> 8;
        const int32_t to = a.ids ? hi : min(hi, limit - ((part.begin + tile) * kKv8Tile + (2 * u + g) * kKv8Group));
#pragma unroll
        for (int i = 0; i < 16; ++i) s[u][i] = i >= lo && i < to ? s[u][i] : -__builtin_inff();
      }
#pragma unroll
      for (int i = 0; i < kPieces; ++i) {
        const uint32_t own = piece_of(i) / kChunks ? lohi[1] : lohi[0];
        const int32_t lo = own & 0xff, hi = own >> 8;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          uint32_t keep = 0;
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (4 * k + e >= lo && 4 * k + e < hi) keep |= 0xffu << (8 * e);
          vpiece[i][k] &= keep;
        }
      }
    }
    if (std::is_same_v<F, E4m3> && tile >= all_see) {
      // A token that later queries see may hold NaN too: it is taken out and noted.
      uint32_t any = 0;
#pragma unroll
      for (int i = 0; i < kPieces; ++i) {
        uint32_t bits = 0;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const uint32_t nan = kv8_nan_bytes(vpiece[i][k]) >> 7;
          vpiece[i][k] &= ~(nan * 0xffu);
          bits |= ((nan * 0x10204080u) >> 28) << (4 * k);  // the four bytes' bits together
        }
        nans[tile % 2][piece_of(i) % kChunks * 32 + n][2 * (piece_of(i) / kChunks) + g] = static_cast<uint16_t>(bits);
        any |= bits;
      }
      const bool found = __ballot(any != 0) != 0;
      if (lane == 0) nan_at[tile % 2][wave] = found;
    }
  };
  // The sums of the rows that see a token whose V is NaN become NaN.
  const auto spread_nans = [&](int32_t tile) {
    uint32_t any = 0;
    for (int w = 0; w < kWaves; ++w) any |= nan_at[tile % 2][w];
    if (__builtin_amdgcn_readfirstlane(any) == 0) return;
    const int32_t sees = limit - (part.begin + tile) * kKv8Tile;
    const uint64_t seen = sees >= kKv8Tile ? ~uint64_t{0} : sees <= 0 ? 0u : (uint64_t{1} << sees) - 1;
#pragma unroll
    for (int dt = 0; dt < kChunks; ++dt)
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const uint64_t has = *reinterpret_cast<const uint64_t*>(nans[tile % 2][dt * 32 + i / 4 * 8 + 4 * g + i % 4]);
        if (has & seen) o[dt][i] = __builtin_nanf("");
      }
  };
  const auto scores = [&](int32_t tile, f32x16_t (&s)[2]) {
#pragma unroll
    for (int u = 0; u < 2; ++u)
#pragma unroll
      for (int i = 0; i < 16; ++i) s[u][i] = 0.f;
#pragma unroll
    for (int k = 0; k < kSteps; ++k)
#pragma unroll
      for (int u = 0; u < 2; ++u) s[u] = kv8_mfma32(kops[tile % 2][u * kSteps + k][lane], q[k], s[u]);
  };

  // Of a tile: the factor of a lane's scores, log2 of the V scale and 1 / that.
  struct Scale {
    float c[2], lv[2], inv[2];
  };
  const auto scale_of = [&](int32_t tile) {
    Scale x;
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const float4 e = sub_scale[tile / kTiles % 2][entry(tile, 2 * u + g)];
      x.c[u] = fmaxf(e.x * rc, FLT_MIN);  // not 0, so that a masked score stays -inf
      x.lv[u] = e.y;
      x.inv[u] = e.z;
    }
    return x;
  };
  const auto top_of = [&](const Scale& x, const float (&most)[2]) {
    const float top = fmaxf(fmaf(most[0], x.c[0], x.lv[0]), fmaf(most[1], x.c[1], x.lv[1]));
    return fmaxf(top, xor_lanes(top, 32));
  };

  // Tile `tile`, whose scores are in `s`, and the next one's scores into `t`.  A
  // product waits for the one before it and everything behind it waits with it,
  // so each is followed by the vector instructions that it hides.
  const int32_t tiles = end - part.begin;
  Scale now;
  float top = 0.f;  // of the tile's scores
  bool far = false;
  Kv8Range scales;
  const auto step = [&](int32_t tile, f32x16_t (&s)[2], f32x16_t (&t)[2]) {
    if (tile % kTiles == 0) {
      if (kv8_far_scales<kWaves>(refs[tile / kTiles % 2], &scales) && !far) {
        far = true;
        lds_ms[wave][n] = m;
      }
      if (tile + kTiles < tiles) look_up(part.begin + tile + kTiles, tile / kTiles % 2 ^ 1);
    }
    const int32_t next = min(tile + 1, tiles - 1);
    const uint32_t cut = cut_of(next);
    constexpr int kAhead = 3;  // operands read ahead of their product
    const u32x4_t(*kop)[kWave] = kops[(tile + 1) % 2];
    const u32x4_t(*vop)[kWave] = vops[tile % 2];
    u32x4_t ready[kAhead];
    const auto k_operand = [&](int i) { return kop[i % 2 * kSteps + i / 2][lane]; };
#pragma unroll
    for (int i = 0; i < kAhead; ++i) ready[i] = k_operand(i);
    if (__ballot(top > m + kKv8Slack)) {
      top = ceilf(fmaxf(top, m));
      const float fix = fast_exp2(m - top);
      if (!far) l *= fix;
#pragma unroll
      for (int dt = 0; dt < kChunks; ++dt) o[dt] *= fix;
      m = top;
    }

    if (__builtin_expect(far, 0)) {
      // The weights for the sum by themselves, beside their own maximum.
      float most = -FLT_MAX;
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int i = 0; i < 16; ++i) most = fmaxf(most, s[u][i] * now.c[u]);
      most = fmaxf(most, xor_lanes(most, 32));
      const float was = lds_ms[wave][n], up = fmaxf(was, ceilf(most));
      float own = 0.f;
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int i = 0; i < 16; ++i) own += fast_exp2(fmaf(s[u][i], now.c[u], kKv8PShift - up));
      l = fmaf(l, fast_exp2(was - up), own);
      lds_ms[wave][n] = up;
      now.inv[0] = now.inv[1] = 0.f;  // and none of these
    }

    // the weights, beside the next tile's scores
    u32x4_t pa[2][2];
    const float base[2] = {now.lv[0] - m + kKv8PShift, now.lv[1] - m + kKv8PShift};
    float sum[2] = {0.f, 0.f};
#pragma unroll
    for (int u = 0; u < 2; ++u)
#pragma unroll
      for (int i = 0; i < 16; ++i) t[u][i] = 0.f;
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int i = 0; i < 2 * kSteps; ++i) {
      t[i % 2] = kv8_mfma32(ready[i % kAhead], q[i / 2], t[i % 2]);
      __builtin_amdgcn_sched_barrier(0);
      if (i + kAhead < 2 * kSteps) {
        ready[i % kAhead] = k_operand(i + kAhead);
      } else {
        ready[i % kAhead] = vop[i + kAhead - 2 * kSteps][lane];
      }
#pragma unroll
      for (int w = i * 8 / kSteps; w < (i + 1) * 8 / kSteps; ++w) {  // its share of the 16 pairs of scores
        const int v = w / 8, e = w % 8;
        const half2_t p = {static_cast<_Float16>(fast_exp2(fmaf(s[v][2 * e], now.c[v], base[v]))),
                           static_cast<_Float16>(fast_exp2(fmaf(s[v][2 * e + 1], now.c[v], base[v])))};
        sum[v] = __builtin_amdgcn_fdot2(p, half2_t{static_cast<_Float16>(1.f), static_cast<_Float16>(1.f)}, sum[v], false);
        uint32_t bits = __builtin_bit_cast(uint32_t, p);
        asm volatile("" : "+v"(bits), "+v"(sum[v]));  // here, not behind the next branch
        pa[v][e / 4][e % 4] = bits;
      }
      __builtin_amdgcn_sched_barrier(0);
    }
    l = fmaf(sum[0], now.inv[0], fmaf(sum[1], now.inv[1], l));
    mask(next, cut, t);

    // the sums, beside the operands and the loads of tiles to come and the next maximum
    constexpr int kProducts = 4 * kChunks, kOperands = 4 * kPieces;
    float most[2] = {t[0][15], t[1][15]};
    uint32_t at = 0;  // where the next load begins
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int i = 0; i < kProducts; ++i) {  // operand i: 32 tokens u, dimensions dt, tokens 8 half .. of each lane
      const int u = i / (2 * kChunks), dt = i / 2 % kChunks, half = i % 2;
      o[dt] = kv8_mfma32(ready[(2 * kSteps + i) % kAhead], pa[u][half], o[dt]);
      __builtin_amdgcn_sched_barrier(0);
      if (i + kAhead < kProducts) ready[(2 * kSteps + i) % kAhead] = vop[i + kAhead][lane];
      if (i == 0) {
        now = scale_of(next);
        at = v_at(min(tile + 2, tiles - 1), 0);
      }
      // its share of the 16 maxima, and of the operands: V of tile + 1, then K of
      // tile + 2, in the buffer of this one; behind a load's second operand the next load
#pragma unroll
      for (int w = i * 16 / kProducts; w < (i + 1) * 16 / kProducts; ++w)
        most[w / 8] = w % 8 < 7 ? kv8_max3(most[w / 8], t[w / 8][w % 8 * 2], t[w / 8][w % 8 * 2 + 1])
                                : fmaxf(most[w / 8], t[w / 8][14]);
#pragma unroll
      for (int w = i * kOperands / kProducts; w < (i + 1) * kOperands / kProducts; ++w) {
        if (w < kOperands / 2) {
          pass_v(tile + 1, w / 2, w % 2);
          if (w % 2) {
            fetch_v(w / 2, at);
            at = w / 2 + 1 < kPieces ? v_at(min(tile + 2, tiles - 1), w / 2 + 1) : k_at(min(tile + 3, tiles - 1), 0);
          }
        } else {
          pass_k(tile, w / 2 - kPieces, w % 2);
          if (w % 2) {
            fetch_k(w / 2 - kPieces, at);
            if (w + 1 < kOperands) at = k_at(min(tile + 3, tiles - 1), w / 2 - kPieces + 1);
          }
        }
      }
      __builtin_amdgcn_sched_barrier(0);
    }
    top = top_of(now, most);
    if (std::is_same_v<F, E4m3> && tile >= all_see) spread_nans(tile);
    lds_barrier();
  };

  if (tiles > 0) {
    f32x16_t s0[2], s1[2];
    look_up(part.begin, 0);
    lds_barrier();
#pragma unroll
    for (int i = 0; i < kPieces; ++i) {
      fetch_k(i, k_at(0, i));
      fetch_v(i, v_at(0, i));
    }
#pragma unroll
    for (int i = 0; i < 2 * kPieces; ++i) pass_k(0, i / 2, i % 2);
#pragma unroll
    for (int i = 0; i < kPieces; ++i) fetch_k(i, k_at(min(1, tiles - 1), i));
    lds_barrier();
    scores(0, s0);
    mask(0, cut_of(0), s0);
    now = scale_of(0);
    float most[2];
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      most[u] = s0[u][0];
#pragma unroll
      for (int i = 1; i < 16; ++i) most[u] = fmaxf(most[u], s0[u][i]);
    }
    top = top_of(now, most);
#pragma unroll
    for (int i = 0; i < 2 * kPieces; ++i) {
      pass_v(0, i / 2, i % 2);
      pass_k(1, i / 2, i % 2);
    }
#pragma unroll
    for (int i = 0; i < kPieces; ++i) {
      fetch_v(i, v_at(min(1, tiles - 1), i));
      fetch_k(i, k_at(min(2, tiles - 1), i));
    }
    lds_barrier();
    if (row0 < a.rows) {
      for (int32_t tile = 0; tile < tiles; tile += 2) {
        step(tile, s0, s1);
        if (tile + 1 < tiles) step(tile + 1, s1, s0);
      }
    } else {  // no rows: the operands alone
      for (int32_t tile = 0; tile < tiles; ++tile) {
        if (tile % kTiles == 0 && tile + kTiles < tiles) look_up(part.begin + tile + kTiles, tile / kTiles % 2 ^ 1);
        mask(min(tile + 1, tiles - 1), cut_of(min(tile + 1, tiles - 1)), s0);
#pragma unroll
        for (int i = 0; i < kPieces; ++i) {
          pass_v(tile + 1, i, 0);
          pass_v(tile + 1, i, 1);
          fetch_v(i, v_at(min(tile + 2, tiles - 1), i));
          pass_k(tile, i, 0);
          pass_k(tile, i, 1);
          fetch_k(i, k_at(min(tile + 3, tiles - 1), i));
        }
        lds_barrier();
      }
    }
  }

  l += xor_lanes(l, 32);
  const float ms = far ? lds_ms[wave][n] : m;
  if (row0 + n >= a.rows) return;
  if (part.count > 1) {
    const int64_t slot = (static_cast<int64_t>(part_index) * a.c.kv_heads + h) * a.rows + r;
#pragma unroll
    for (int dt = 0; dt < kChunks; ++dt)
#pragma unroll
      for (int i = 0; i < 4; ++i)
        *reinterpret_cast<f32x4_t*>(a.part_o + slot * D + dt * 32 + 8 * i + 4 * g) =
            f32x4_t{o[dt][4 * i], o[dt][4 * i + 1], o[dt][4 * i + 2], o[dt][4 * i + 3]};
    if (g == 0) *reinterpret_cast<float4*>(a.part_ml + 4 * slot) = make_float4(m, ms, l, 0.f);
  } else {
#pragma unroll
    for (int dt = 0; dt < kChunks; ++dt)
#pragma unroll
      for (int i = 0; i < 4; ++i)
        kv8_store4(a, q_at + dt * 32 + 8 * i + 4 * g,
                   kv8_result(f32x4_t{o[dt][4 * i], o[dt][4 * i + 1], o[dt][4 * i + 2], o[dt][4 * i + 3]}, l, m - ms));
  }
}

// Launch for one format; `tiles` row tiles (16 rows) a wavefront, 0: the kernel of
// many rows.
template <typename F>
int kv8_attend_launch(const Kv8Attend& a, int tiles, hipStream_t stream) {
  const int64_t over = static_cast<int64_t>(a.parts) * a.row_groups;
  const dim3 grid(static_cast<uint32_t>(a.c.kv_heads), static_cast<uint32_t>(over < kKv8GridRows ? over : kKv8GridRows),
                  static_cast<uint32_t>(ceil_div(over, kKv8GridRows)));
  const auto go = [&](auto kernel) {
    return launch("kv8_attend_kernel", kernel, grid, dim3(kKv8Threads), 0, stream, a);
  };
  const bool alone = a.row_waves == 1;
  const auto by_tiles = [&](auto dim) {
    constexpr int D = decltype(dim)::value;
    if (a.dtype == CSAHCA_F32)
      return alone ? go(kv8_attend_kernel<D, F, true, 1, true>) : go(kv8_attend_kernel<D, F, true, 1, false>);
    if (tiles == 0)
      return launch("kv8_attend_rows_kernel", kv8_attend_rows_kernel<D, F>, grid, dim3(kv8_rows_waves(D) * kWave), 0, stream,
                    a);
    if constexpr (D <= kKv8TwoTilesDim) {
      if (tiles == 2)
        return alone ? go(kv8_attend_kernel<D, F, false, 2, true>) : go(kv8_attend_kernel<D, F, false, 2, false>);
    } else {
      if (!alone) return go(kv8_attend_kernel<D, F, false, 1, false>);
    }
    return go(kv8_attend_kernel<D, F, false, 1, true>);
  };
  switch (a.c.head_dim / 32) {
    case 1: return by_tiles(std::integral_constant<int, 32>{});
    case 2: return by_tiles(std::integral_constant<int, 64>{});
    case 3: return by_tiles(std::integral_constant<int, 96>{});
    case 4: return by_tiles(std::integral_constant<int, 128>{});
    case 5: return by_tiles(std::integral_constant<int, 160>{});
    case 6: return by_tiles(std::integral_constant<int, 192>{});
    case 7: return by_tiles(std::integral_constant<int, 224>{});
    default: return by_tiles(std::integral_constant<int, 256>{});
  }
}

int kv8_attend_launch_e4m3(const Kv8Attend& a, int tiles, hipStream_t stream);
int kv8_attend_launch_int8(const Kv8Attend& a, int tiles, hipStream_t stream);

}  // namespace csahca
