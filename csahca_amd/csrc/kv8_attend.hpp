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
// held times 2^11 and m moves only when a score passes it by 4: the sums are
// rarely rescaled, p stays at most 2^15, and what is lost of a weight for want of
// exponent is at most 2^-36 of the largest weight.
//
// Beside f32 values the operands are bf16, as wide as f32: q and p as three bf16
// each, 24 bits, of which nothing is lost.
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
constexpr float kKv8PShift = 11.0f;  // a weight is held times 2^11 ...
constexpr float kKv8Slack = 4.0f;    // ... and may pass the running maximum by 2^4

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
  int32_t min_tiles;   // tiles of a part, at least
  int32_t target_log2; // about 2^target_log2 workgroups over all
  int32_t join_lanes;  // of a joining workgroup, thread groups that share a row's parts
  uint32_t page_groups;  // groups of 16 tokens of a page, 1 to 16 ...
  uint32_t page_magic;   // ... and 2^32 / that, rounded up
  float scale_log2;
  float* part_ml;      // [parts, kv_heads, rows, 2]
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

// Tiles of a part: one size for all sequences, from the lengths on the device,
// so that ragged lengths spread evenly over about 2^target_log2 workgroups.
// Whole rounds of the wavefronts that split the tokens.  Every wavefront works
// it out by itself, a lane a sequence; `mine` is the lane's tiles of the last
// 64 sequences (of all, where the batch is not larger).
__device__ __forceinline__ int32_t kv8_part_size(const Kv8Attend& a, int32_t* mine) {
  const int lane = threadIdx.x % kWave;
  int64_t total = 0;
  for (int base = 0; base < a.batch; base += kWave) {
    *mine = kv8_tiles(a, base + lane);
    total += kv8_wave_sum(*mine);
  }
  const int64_t per = (total * a.c.kv_heads * a.row_groups) >> a.target_log2;
  const int32_t round = kKv8Waves / a.row_waves;  // a power of two
  return (max(a.min_tiles, static_cast<int32_t>(per) + 1) + round - 1) & -round;
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
template <typename V>
__device__ __forceinline__ V kv8_load(uint64_t base, int offset) {
  return *reinterpret_cast<const __attribute__((address_space(1))) V*>(base + offset);
}

// The larger of three in one instruction (fmaxf twice also quiets each operand).
__device__ __forceinline__ float kv8_max3(float a, float b, float c) {
  float r;
  asm("v_max3_f32 %0, %1, %2, %3" : "=v"(r) : "v"(a), "v"(b), "v"(c));
  return r;
}

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

// Workgroups of a CU: two while a wavefront's registers (K, V, the sums, q, scores
// and weights) fit 256.
template <int D, int NP, int NT>
constexpr int kKv8Blocks = D / 4 * (2 + NT) + NP * NT * D / 8 + 16 * NT + 8 * NP * NT <= 216 ? 2 : 1;

template <int D, typename F, bool kF32, int NT>
__global__ __launch_bounds__(kKv8Threads, (kKv8Blocks<D, kF32 ? 3 : 1, NT>)) void kv8_attend_kernel(const Kv8Attend a) {
  constexpr int NP = kF32 ? 3 : 1;         // operands that make up a value of q or a weight
  constexpr int kSteps = D / 32;           // matrix instructions over D
  constexpr int kWide = D / 64;            // 16-byte loads of a K row
  constexpr bool kTail = D % 64 != 0;      // and one of 8 bytes
  constexpr int kDTiles = D / 16;
  constexpr int kRowPad = D + 4;
  constexpr size_t kMergeBytes = sizeof(float) * kKv8Waves * 16 * kRowPad;
  constexpr size_t kSubBytes = 20 * kKv8SegTiles * 4;
  __shared__ __attribute__((aligned(16))) char lds[kMergeBytes > kSubBytes ? kMergeBytes : kSubBytes];
  __shared__ float lds_ml[kKv8Waves][16][2];
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
      for (int w = 0; w < kWide; ++w) kw[t][w] = kv8_load<u32x4_t>(wide, 4 * t * D + 64 * w);
      if constexpr (kTail) kt[t] = kv8_load<u32x2_t>(tail, 4 * t * D);
    }
  };
  const auto load_v = [&](uint32_t at) {
    const uint64_t base = kv8_opaque(vbase + static_cast<int64_t>(at) * (kKv8Group * D));
#pragma unroll
    for (int dt = 0; dt < kDTiles; ++dt) vw[dt] = kv8_load<u32x4_t>(base, dt * 16 * kKv8Group);
  };

  // The pages of the segment's sub-blocks, then this wavefront's first loads and
  // the sub-blocks' scales, which only the scores wait for.
  float ks[kKv8Lookups], vs[kKv8Lookups];
  const int32_t first = wave % token_waves;
  const auto look_up = [&](int32_t seg, int32_t tiles) {
#pragma unroll
    for (int i = 0; i < kKv8Lookups; ++i) {
      const int at = i * kKv8Threads + threadIdx.x;
      ks[i] = 0.f;
      vs[i] = 1.f;
      if (at < tiles * 4) {
        const Kv8Sub sub = kv8_resolve(a, b, h, len, static_cast<uint32_t>(seg) * 4 + at);
        sub_at[at] = make_uint2(sub.at, sub.lohi);
        if (sub.scale >= 0) {
          ks[i] = a.c.k_scale[sub.scale];
          vs[i] = a.c.v_scale[sub.scale];
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
    int e2 = 15;
    if constexpr (!kF32) {
#pragma unroll
      for (int k = 0; k < kSteps; ++k)
#pragma unroll
        for (int e = 0; e < 8; ++e) top = fmaxf(top, fabsf(v[k][e]));
      top = fmaxf(top, xor_lanes(top, 16));
      top = fmaxf(top, xor_lanes(top, 32));
      if (top > 0.f && top < __builtin_inff()) (void)frexpf(top, &e2);
    }
#pragma unroll
    for (int k = 0; k < kSteps; ++k) {
#pragma unroll
      for (int e = 0; e < 8; ++e) v[k][e] = kF32 ? v[k][e] * sign : __builtin_ldexpf(v[k][e] * sign, 15 - e2);
      kv8_split<kF32>(v[k], q[nt][k]);
    }
    rc[nt] = __builtin_ldexpf(fabsf(a.scale_log2), e2 - 15);
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

  for (int32_t seg = part.begin; seg < end;) {
    const int32_t seg_end = min(end - seg, kKv8SegTiles);
#pragma unroll
    for (int i = 0; i < kKv8Lookups; ++i) {
      const int at = i * kKv8Threads + threadIdx.x;
      if (at < seg_end * 4) {
        const float lv = __builtin_amdgcn_logf(fmaxf(vs[i], FLT_MIN));
        sub_scale[at] = make_float2(ks[i], lv);
        sub_inv[at] = fast_exp2(-lv);
      }
    }
    lds_barrier();

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
      }

      // The factor of a lane's scores is not negative, so their maximum is that of
      // the products (and not 0, so that a masked one stays -inf).
      float c[NT], top[NT];
      bool up = false;
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        c[nt] = fmaxf(scale.x * rc[nt], 1e-30f);
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
          top[nt] = fmaxf(top[nt], m[nt]);
          const float fix = fast_exp2(m[nt] - top[nt]);
          l[nt] *= fix;
#pragma unroll
          for (int dt = 0; dt < kDTiles; ++dt) o[nt][dt] *= fix;
          m[nt] = top[nt];
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
        for (int i = 0; i < 4; ++i) l[nt] = fmaf(sum[i], inv_vs[i], l[nt]);
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
      lds_ml[wave][n][0] = m[nt];
      lds_ml[wave][n][1] = sum;
    }
    __syncthreads();
    // thread: (row wavefront, row, four dimensions)
    for (int i = threadIdx.x; i < a.row_waves * 16 * (D / 4); i += kKv8Threads) {
      const int d = i % (D / 4) * 4, row = i / (D / 4) % 16, w0 = i / (D / 4 * 16) * token_waves;
      const int32_t r = (rg * a.row_waves + w0 / token_waves) * (NT * 16) + nt * 16 + row;
      if (r >= a.rows) continue;
      float top = -FLT_MAX, total = 0.f;
      for (int w = 0; w < token_waves; ++w) top = fmaxf(top, lds_ml[w0 + w][row][0]);
      f32x4_t acc{0.f, 0.f, 0.f, 0.f};
      for (int w = 0; w < token_waves; ++w) {
        const float fix = fast_exp2(lds_ml[w0 + w][row][0] - top);
        total = fmaf(lds_ml[w0 + w][row][1], fix, total);
        acc += *reinterpret_cast<const f32x4_t*>(merge + ((w0 + w) * 16 + row) * kRowPad + d) * fix;
      }
      if (part.count > 1) {
        const int64_t slot = (static_cast<int64_t>(part_index) * a.c.kv_heads + h) * a.rows + r;
        *reinterpret_cast<f32x4_t*>(a.part_o + slot * D + d) = acc;
        if (d == 0) *reinterpret_cast<float2*>(a.part_ml + 2 * slot) = make_float2(top, total);
      } else {
        const float inv = total != 0.f ? 1.0f / total : 0.f;
        const int32_t qi = a.queries == 1 ? 0 : r / a.group;
        const int64_t at =
            ((static_cast<int64_t>(b) * a.queries + qi) * heads + h * a.group + (r - qi * a.group)) * D + d;
        kv8_store4(a, at, acc * inv);
      }
    }
  }
}

// Launch for one format; `tiles` row tiles (16 rows) a wavefront.
template <typename F>
int kv8_attend_launch(const Kv8Attend& a, int tiles, hipStream_t stream) {
  const int64_t over = static_cast<int64_t>(a.parts) * a.row_groups;
  const dim3 grid(static_cast<uint32_t>(a.c.kv_heads), static_cast<uint32_t>(over < kKv8GridRows ? over : kKv8GridRows),
                  static_cast<uint32_t>(ceil_div(over, kKv8GridRows)));
  const auto go = [&](auto kernel) {
    return launch("kv8_attend_kernel", kernel, grid, dim3(kKv8Threads), 0, stream, a);
  };
  const auto by_tiles = [&](auto dim) {
    constexpr int D = decltype(dim)::value;
    if (a.dtype == CSAHCA_F32) return go(kv8_attend_kernel<D, F, true, 1>);
    if constexpr (D <= kKv8TwoTilesDim) {
      if (tiles == 2) return go(kv8_attend_kernel<D, F, false, 2>);
    }
    return go(kv8_attend_kernel<D, F, false, 1>);
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
