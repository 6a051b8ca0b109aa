// What the two forms of the prompt and differential attention share: the launch's
// parameters, the search for a row tile's sequence, splits, and cache rows on
// their way to LDS as fp16.
#ifndef PA_PREFILL_COMMON_H_
#define PA_PREFILL_COMMON_H_

#include <hip/hip_runtime.h>
#include <stdint.h>

#include <type_traits>

#include "kv_math.h"
#include "launch_math.h"
#include "pa_errors.h"
#include "pagedattn.h"

// A checked call (build() in paged_prefill.hip).
struct PParams {
  const uint8_t *q;
  const uint8_t *k;
  const uint8_t *v;
  const uint8_t *ks;
  const uint8_t *vs;
  uint8_t *out;
  float *part_out;  // [num_splits, num_tokens, num_q_heads, DV]
  float *part_lse;  // [num_splits, num_tokens, num_q_heads]
  const int32_t *bt;
  const int32_t *seq_lens;
  const int32_t *start;  // [batch + 1] row offsets, or NULL: one row a sequence
  const float *lam;      // differential: [num_q_heads / 2]
  const float *norm;     // differential: [DV] or NULL
  int32_t batch, num_tokens, units, group, num_q_heads;
  int32_t num_blocks, max_tokens, log2_page, num_splits;
  int32_t chunks;        // > 0: chunks wanted of all row tiles of a unit together
  int32_t tiles;         // row tiles of the launch
  int32_t sqt, sqh, sot, soh;  // elements
  uint32_t skn, skt, skh, ssn, sst;  // bytes
  int32_t sbtb, slam;    // elements
  float qk_scale;        // sm_scale * log2(e)
  float norm_eps, out_scale;
  int32_t io_bf16;
  Div by_units, by_splits, by_tiles, by_group, by_seq_tiles, by_heads;
};

// The form for few rows a sequence (paged_stream.hip), its merge included.
PA_HIDDEN hipError_t launch_streams(const PParams &p, const pa_prefill_args *a, int maps, hipStream_t st);

namespace {

typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));

constexpr int kWaves = 4;
constexpr int kRowsPerWave = 32;
// P is 2^kTopLog2 at the running maximum, which moves only when a score passes it by
// kRescaleLog2: P stays below 2^15, in fp16's range, and what is far below the maximum
// stays out of its subnormals for longer. (The sums hold the same factor.)
constexpr float kTopLog2 = 7.0f;
constexpr float kRescaleLog2 = 8.0f;
constexpr int kSplitUnit = 128;  // splits are multiples of this many tokens
// A lane offset past every buffer (page_rsrc's -1 leaves all others in range):
// the load returns zeros.
constexpr uint32_t kOutside = 0xfffffff0u;
constexpr int kRsrcBytes = (int)kOutside;

// x with what DPP control CTRL hands the lanes of ROWS (the others: `none`).
template <int CTRL, int ROWS>
__device__ __forceinline__ int dpp(int x, int none) {
  return __builtin_amdgcn_update_dpp(none, x, CTRL, ROWS, 0xf, false);
}

// The wave's lanes combined, for every lane; `none` changes nothing.
template <typename OP>
__device__ __forceinline__ int wave_join(int x, int none, OP op) {
  x = op(x, dpp<0x111, 0xf>(x, none));  // row_shr:1
  x = op(x, dpp<0x112, 0xf>(x, none));
  x = op(x, dpp<0x114, 0xf>(x, none));
  x = op(x, dpp<0x118, 0xf>(x, none));
  x = op(x, dpp<0x142, 0xa>(x, none));  // row_bcast:15 into rows 1 and 3
  x = op(x, dpp<0x143, 0xc>(x, none));  // row_bcast:31 into rows 2 and 3
  return __builtin_amdgcn_readlane(x, 63);
}

__device__ __forceinline__ int wave_sum(int x) {
  return wave_join(x, 0, [](int a, int b) { return a + b; });
}

__device__ __forceinline__ int wave_max(int x) {
  return wave_join(x, INT32_MIN, [](int a, int b) { return max(a, b); });
}

// x combined with the value of the other half of the wave (lane ^ 32).
__device__ __forceinline__ float half_max(float x) {
  const uint32_t u = __float_as_uint(x);
  const auto a = __builtin_amdgcn_permlane32_swap(u, u, false, false);
  return fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
}

__device__ __forceinline__ float half_sum(float x) {
  const uint32_t u = __float_as_uint(x);
  const auto a = __builtin_amdgcn_permlane32_swap(u, u, false, false);
  return __uint_as_float(a[0]) + __uint_as_float(a[1]);
}

// x combined over the 64 / COLS lanes that share a column.
template <int COLS>
__device__ __forceinline__ float column_max(float x) {
  if constexpr (COLS == 16) {
    const uint32_t u = __float_as_uint(x);
    const auto a = __builtin_amdgcn_permlane16_swap(u, u, false, false);
    x = fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
  }
  return half_max(x);
}

template <int COLS>
__device__ __forceinline__ float column_sum(float x) {
  if constexpr (COLS == 16) {
    const uint32_t u = __float_as_uint(x);
    const auto a = __builtin_amdgcn_permlane16_swap(u, u, false, false);
    x = __uint_as_float(a[0]) + __uint_as_float(a[1]);
  }
  return half_sum(x);
}

// Token (in its tile) of a lane's score e: four neighbouring tokens a lane group.
template <int COLS>
__device__ __forceinline__ int score_token(int e, int grp) {
  return 256 / COLS * (e / 4) + 4 * grp + e % 4;
}

// int8: scores times their tokens' K scales (in LDS); multiply(e, k) takes k to score e.
template <int COLS, int N, typename MULTIPLY>
__device__ __forceinline__ void scale_scores(MULTIPLY multiply, const float *scales, int grp) {
#pragma unroll
  for (int e = 0; e < N; e += 4) {
    const f32x4 k4 = *reinterpret_cast<const f32x4 *>(scales + score_token<COLS>(e, grp));
#pragma unroll
    for (int j = 0; j < 4; ++j) multiply(e + j, k4[j]);
  }
}

// int8: V's scale as P meets it before its rounding to fp16. Tokens that a row does
// not see may have any scale and their P is 0: infinities and NaN become the largest
// float, whose product with 0 is 0 and with any other P is fp16's infinity.
__device__ __forceinline__ float finite_scale(float s) {
  constexpr float kMost = 3.4028234663852886e38f;
  return fminf(fmaxf(s, -kMost), kMost);
}

// So that neither large nor small products leave fp16's range they are divided by a
// power of two, `limit` (0 before the first), which follows the largest product of
// the lane's row so far, `top`, with room for 2^7 times that; the accumulators are in
// units of it. Moves the limit up where `top` has passed its room, and returns what
// the accumulators have to be multiplied by; nothing to do when no lane had to (`any`
// false).
template <int COLS>
__device__ __forceinline__ float raise_limit(float &limit, float top, bool &any) {
  top = column_max<COLS>(fminf(top, 0x1p100f));  // (an infinity makes the row's result one, at any limit)
  const bool need = top > limit * 32768.f;
  any = __builtin_amdgcn_ballot_w64(need) != 0;
  if (__builtin_expect(!any, 1)) return 1.f;
  const uint32_t e = max(__float_as_uint(top) >> 23, 30u);
  const float f = need ? limit * __uint_as_float((261 - e) << 23) : 1.f;
  if (need) limit = __uint_as_float((e - 7) << 23);
  return f;
}

// 1 / limit, a power of two (0 where the row has met no product).
__device__ __forceinline__ float inverse_limit(float limit) {
  return limit > 0.f ? __uint_as_float((254u << 23) - __float_as_uint(limit)) : 0.f;
}

// First row of sequence b among the packed rows, kept inside them whatever the
// device's offsets hold.
__device__ __forceinline__ int row_start(const PParams &p, int b) {
  return p.start ? min(max(ro(p.start)[b], 0), p.num_tokens) : b;
}

// The sequence whose key(start, b) is the last at or below x, for a key that
// grows with b: 64 probes at a time.
template <typename KEY>
__device__ __forceinline__ int find_sequence(const PParams &p, int x, int lane, KEY key) {
  int lo = 0, n = p.batch;
  for (;;) {
    const int step = (n + 63) / 64;
    const int b = lo + lane * step;
    bool below = false;
    if (lane * step < n) below = key(row_start(p, b), b) <= x;
    const uint64_t m = __builtin_amdgcn_ballot_w64(below);
    const int count = m == ~0ull ? 64 : __builtin_ctzll(~m);
    lo += max(count - 1, 0) * step;
    if (step == 1) return __builtin_amdgcn_readfirstlane(lo);
    n = min(step, p.batch - lo);
  }
}

// A row tile: its sequence, its first row there, and the tokens that its rows see.
struct RowTile {
  int b, row0, rows;  // rows: n_b * group (row0 >= rows: no such tile)
  int token0;         // first packed row of the sequence
  int first;          // tokens before the sequence's new ones (negative: fewer than n_b in all)
  int len;            // T_b
  int hi;             // tokens seen by the last row of the tile
};

// `index` of the sequence's tiles of ROWS rows.
template <int ROWS>
__device__ __forceinline__ RowTile tile_at(const PParams &p, int b, int index) {
  RowTile t;
  t.b = b;
  t.token0 = row_start(p, b);
  const int n = p.start ? max(row_start(p, b + 1) - t.token0, 0) : 1;
  t.rows = n * p.group;
  t.row0 = index * ROWS;
  t.len = max(0, min(ro(p.seq_lens)[b], p.max_tokens));
  t.first = t.len - n;
  const int last = min(n - 1, (int)div_by((uint32_t)(t.row0 + ROWS - 1), p.by_group));
  t.hi = max(0, t.first + last + 1);
  return t;
}

// The most units of a split (kSplitUnit tokens each) with p.chunks: the num_splits'th
// part of the longest sequence, and what gives p.chunks over all row tiles of ROWS
// rows together, so a ragged batch's long sequences take many and its short ones one.
// Every workgroup sums the lengths itself, two loads a lane for 64 sequences, and the
// merge comes to the same. 0 without p.chunks.
template <int ROWS>
__device__ __forceinline__ uint32_t split_units(const PParams &p, int lane) {
  if (p.chunks == 0) return 0;
  int longest = 0, total = 0;  // total: units; a lane's stops at 2^24
  for (int b = lane; b < p.batch; b += 64) {
    const int n = p.start ? max(row_start(p, b + 1) - row_start(p, b), 0) : 1;
    if (n == 0) continue;
    const int len = max(0, min(ro(p.seq_lens)[b], p.max_tokens));
    longest = max(longest, len);
    const uint32_t tiles = ((uint32_t)(n * p.group) + ROWS - 1) / ROWS;
    const uint32_t units = (uint32_t)(max(len - n / 2, 0) + kSplitUnit - 1) / kSplitUnit;
    total = (int)min((uint64_t)total + (uint64_t)tiles * units, (uint64_t)1 << 24);
  }
  const uint32_t most = div_by(((uint32_t)wave_max(longest) + kSplitUnit - 1) / kSplitUnit + p.num_splits - 1, p.by_splits);
  return max(max(most, ((uint32_t)wave_sum(total) + p.chunks - 1) / p.chunks), 1u);
}

// Tokens of a split of a row tile that sees `hi`: equal shares of at most `most`
// units, or (0) the num_splits'th part.
__device__ __forceinline__ int split_tokens(const PParams &p, int hi, uint32_t most) {
  const uint32_t units = ((uint32_t)hi + kSplitUnit - 1) / kSplitUnit;
  if (most == 0) return (int)div_by(units + p.num_splits - 1, p.by_splits) * kSplitUnit;
  const uint32_t pieces = max((units + most - 1) / most, 1u);
  return (int)((units + pieces - 1) / pieces) * kSplitUnit;
}

template <int POLICY, int WORDS>
__device__ __forceinline__ void load_piece(uint32_t (&w)[WORDS], __amdgpu_buffer_rsrc_t r, uint32_t off) {
  if constexpr (WORDS == 4) {
    const u32x4 x = __builtin_amdgcn_raw_buffer_load_b128(r, off, 0, POLICY);
    w[0] = x.x; w[1] = x.y; w[2] = x.z; w[3] = x.w;
  } else {
    const u32x2 x = __builtin_amdgcn_raw_buffer_load_b64(r, off, 0, POLICY);
    w[0] = x.x; w[1] = x.y;
  }
}

template <int SC>
__device__ __forceinline__ uint32_t load_scale(__amdgpu_buffer_rsrc_t r, uint32_t off) {
  if constexpr (SC == PA_SCALE_FP32) return __builtin_amdgcn_raw_buffer_load_b32(r, off, 0, 0);
  else return __builtin_amdgcn_raw_buffer_load_b16(r, off, 0, 0);
}

// A piece's elements as fp16 words (two elements each). int8 values come as they are,
// exactly; their scales meet the scores and P (below), so no product is rounded to
// fp16 on the way in.
template <int KV, int WORDS>
__device__ __forceinline__ void to_halves(uint32_t *h, const uint32_t (&w)[WORDS]) {
  if constexpr (KV == PA_KV_FP16) {
#pragma unroll
    for (int i = 0; i < WORDS; ++i) h[i] = w[i];
  } else if constexpr (KV == PA_KV_BF16) {
#pragma unroll
    for (int i = 0; i < WORDS; ++i) h[i] = bf16x2_to_f16x2(w[i]);
  } else if constexpr (KV == PA_KV_FP8_E5M2) {
#pragma unroll
    for (int i = 0; i < WORDS; ++i) {
      h[2 * i] = bytes_to_halves<KV>(w[i], w[i], pair_sel<KV>(0, 1));
      h[2 * i + 1] = bytes_to_halves<KV>(w[i], w[i], pair_sel<KV>(2, 3));
    }
  } else {
    // x + 128 under the exponent byte 0x64 is 1024 + (x + 128)
#pragma unroll
    for (int i = 0; i < WORDS; ++i) {
      const uint32_t x = w[i] ^ kInt8Sign;
      const f16x2 a = __builtin_bit_cast(f16x2, perm(kF16Exp1024, x, 0x04010400u));
      const f16x2 b = __builtin_bit_cast(f16x2, perm(kF16Exp1024, x, 0x04030402u));
      const f16x2 c = {(_Float16)1152.0f, (_Float16)1152.0f};
      h[2 * i] = __builtin_bit_cast(uint32_t, a - c);
      h[2 * i + 1] = __builtin_bit_cast(uint32_t, b - c);
    }
  }
}

template <int SC>
__device__ __forceinline__ float scale_value(uint32_t bits) {
  if constexpr (SC == PA_SCALE_FP32) return __uint_as_float(bits);
  else return (float)__builtin_bit_cast(_Float16, (uint16_t)bits);
}

// Whether a half of the word is an infinity or NaN.
__device__ __forceinline__ bool has_wild(uint32_t w) {
  return (w & 0x7c00u) == 0x7c00u || (w & 0x7c000000u) == 0x7c000000u;
}

// Infinities and NaN of the word's halves to zeros; whether there was one.
__device__ __forceinline__ bool tame_word(uint32_t &w) {
  if (__builtin_expect(!has_wild(w), 1)) return false;
  if ((w & 0x7c00u) == 0x7c00u) w &= 0xffff0000u;
  if ((w & 0x7c000000u) == 0x7c000000u) w &= 0xffffu;
  return true;
}

// Four neighbouring elements of a result row.
__device__ __forceinline__ void store4(uint8_t *dst, float a, float b, float c, float d, bool bf16) {
  u32x2 w;
  if (bf16) {
    w = u32x2{f32_to_bf16_bits(a) | (f32_to_bf16_bits(b) << 16), f32_to_bf16_bits(c) | (f32_to_bf16_bits(d) << 16)};
  } else {
    w = u32x2{cvt_pk_f16(a, b), cvt_pk_f16(c, d)};
  }
  *reinterpret_cast<u32x2 *>(dst) = w;
}

// Eight elements of one column of V, for a product over V^T: each 16 lanes read two
// blocks of four rows by 16 columns (`a`: this lane's eight bytes of the first; the
// second `step` bytes on) and get a column each.
__device__ __forceinline__ f16x8 read_columns(const uint8_t *a, int step) {
  typedef __attribute__((address_space(3))) s16x4 lds_s16x4;
  const s16x4 x = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4 *)a);
  const s16x4 y = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4 *)(a + step));
  const u32x2 xa = __builtin_bit_cast(u32x2, x), ya = __builtin_bit_cast(u32x2, y);
  return as_f16x8(xa.x, xa.y, ya.x, ya.y);
}

// A lane's share of a result row: with COLS columns (rows of the result) in the 64
// lanes, lanes of column c hold four neighbouring elements each from 256 / COLS * g
// + 4 * (lane / COLS) on, g = 0, 1, ...; `get(e)` is element e % 4 of group e / 4.
// Times f, and with `normed` times the norm's weight if there is one.
template <int W, int COLS, typename GET>
__device__ __forceinline__ void store_rows(const PParams &p, GET get, float f, bool normed, int packed, int out_head,
                                           int lane) {
  uint8_t *dst = p.out + 2 * ((int64_t)packed * p.sot + (int64_t)out_head * p.soh);
  const float *norm = normed ? p.norm : nullptr;
#pragma unroll
  for (int e = 0; e < W * COLS / 64; e += 4) {
    const int d = 64 / COLS * e + 4 * (lane / COLS);
    f32x4 y = {get(e) * f, get(e + 1) * f, get(e + 2) * f, get(e + 3) * f};
    if (norm) y *= *reinterpret_cast<const f32x4 *>(norm + d);
    store4(dst + 2 * d, y.x, y.y, y.z, y.w, p.io_bf16);
  }
}

// The same as a partial: normalised, and its log2-sum-exp.
template <int W, int COLS, typename GET>
__device__ __forceinline__ void store_partial(const PParams &p, GET get, float m, float l, int split, int packed,
                                              int head, int lane) {
  const int64_t at = ((int64_t)split * p.num_tokens + packed) * p.num_q_heads + head;
  const float inv = l == 0.f ? 0.f : 1.0f / l;
  float *dst = p.part_out + at * W;
#pragma unroll
  for (int e = 0; e < W * COLS / 64; e += 4)
    *reinterpret_cast<f32x4 *>(dst + 64 / COLS * e + 4 * (lane / COLS)) =
        f32x4{get(e) * inv, get(e + 1) * inv, get(e + 2) * inv, get(e + 3) * inv};
  if (lane < COLS) p.part_lse[at] = l == 0.f ? -INFINITY : m + __log2f(l);
}

// Joins the partials of a split launch: one wave an output row, W / 64 elements a
// lane (W = 32: the upper half of the wave idles), up to four splits' loads at once.
// Bound by latency for few rows (5 us), by the partials' bytes for many (25,700 rows of
// two maps and 128 elements, two splits: 14 us). Several rows a wave, or weights found
// one a lane, took 18-21 us there. Row tiles of one split are done;
// empty splits were not written and are not read.
template <int W, int MAPS, int ROWS>
__global__ void __launch_bounds__(256) prefill_merge_kernel(const PParams p) {
  constexpr int E = W >= 64 ? W / 64 : 1;
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const uint32_t out_heads = p.num_q_heads / MAPS;
  const uint32_t x = blockIdx.x * 4u + wave;  // row * out_heads + head
  if (x >= (uint32_t)p.num_tokens * out_heads) return;
  const int packed = div_by(x, p.by_heads);
  const int out_head = x - packed * out_heads;
  int b = packed;
  if (p.start) {
    b = find_sequence(p, packed, lane, [](int start, int) { return start; });
    const int s0 = row_start(p, b), s1 = row_start(p, b + 1);
    if (packed < s0 || packed >= s1) return;  // a row of no sequence
  }
  const int token = packed - row_start(p, b);
  const int in_group = out_head % p.group;
  const RowTile rt = tile_at<ROWS>(p, b, (token * p.group + in_group) / ROWS);
  const int chunk = split_tokens(p, rt.hi, split_units<ROWS>(p, lane));
  if (rt.hi <= chunk) return;  // written by its one workgroup
  const int n = (rt.hi - 1) / chunk + 1;
  const bool sees = rt.first + token >= 0;

  const int d0 = E * lane;
  const bool mine = d0 < W;
  const int64_t at = (int64_t)packed * p.num_q_heads + MAPS * out_head;
  const int64_t step = (int64_t)p.num_tokens * p.num_q_heads;
  float m[MAPS], sum[MAPS] = {}, acc[MAPS][E] = {};
#pragma unroll
  for (int map = 0; map < MAPS; ++map) m[map] = -INFINITY;
  // `ahead` splits, their loads on the way together; one that saw nothing of the row
  // (-inf) is left out whatever it holds
  auto join = [&](int s, auto ahead) {
    constexpr int kAhead = decltype(ahead)::value;
    float lse[kAhead][MAPS], o[kAhead][MAPS][E] = {};
#pragma unroll
    for (int i = 0; i < kAhead; ++i)
#pragma unroll
      for (int map = 0; map < MAPS; ++map) {
        lse[i][map] = p.part_lse[at + map + (s + i) * step];
        if (mine) {
#pragma unroll
          for (int e = 0; e < E; ++e) o[i][map][e] = p.part_out[(at + map + (s + i) * step) * W + d0 + e];
        }
      }
#pragma unroll
    for (int map = 0; map < MAPS; ++map) {
      float top = m[map];
#pragma unroll
      for (int i = 0; i < kAhead; ++i) top = fmaxf(top, lse[i][map]);
      const float base = top == -INFINITY ? 0.f : top;
      const float old = __builtin_amdgcn_exp2f(m[map] - base);
      sum[map] *= old;
#pragma unroll
      for (int e = 0; e < E; ++e) acc[map][e] *= old;
#pragma unroll
      for (int i = 0; i < kAhead; ++i) {
        const float w = __builtin_amdgcn_exp2f(lse[i][map] - base);
        sum[map] += w;
#pragma unroll
        for (int e = 0; e < E; ++e) acc[map][e] += lse[i][map] == -INFINITY ? 0.f : w * o[i][map][e];
      }
      m[map] = top;
    }
  };
  int s = 0;
  for (; s + 4 <= n; s += 4) join(s, std::integral_constant<int, 4>());
  if (s + 2 <= n) {
    join(s, std::integral_constant<int, 2>());
    s += 2;
  }
  if (s < n) join(s, std::integral_constant<int, 1>());
  float y[E] = {};
#pragma unroll
  for (int map = 0; map < MAPS; ++map) {
    const float inv = sees ? 1.0f / sum[map] : 0.f;
    const float f = map == 1 ? -inv * p.lam[(int64_t)out_head * p.slam] : inv;
#pragma unroll
    for (int e = 0; e < E; ++e) y[e] += acc[map][e] * f;
  }
  if constexpr (MAPS == 2) {
    if (p.norm) {
      float sq = 0.f;
#pragma unroll
      for (int e = 0; e < E; ++e) sq += y[e] * y[e];
#pragma unroll
      for (int o = 1; o < 64; o *= 2) sq += __shfl_xor(sq, o);
      const float f = __builtin_amdgcn_rsqf(sq * (1.0f / W) + p.norm_eps) * p.out_scale;
#pragma unroll
      for (int e = 0; e < E; ++e) y[e] *= f * (mine ? p.norm[d0 + e] : 0.f);
    }
  }
  if (!mine) return;
  uint16_t *dst = reinterpret_cast<uint16_t *>(p.out) + (int64_t)packed * p.sot + (int64_t)out_head * p.soh + d0;
#pragma unroll
  for (int e = 0; e < E; ++e)
    dst[e] = p.io_bf16 ? (uint16_t)f32_to_bf16_bits(y[e]) : __builtin_bit_cast(uint16_t, (_Float16)y[e]);
}

template <int W, int MAPS, int ROWS>
void launch_merge(const PParams &p, hipStream_t st) {
  const dim3 rows(((uint32_t)p.num_tokens * (uint32_t)(p.num_q_heads / MAPS) + 3) / 4);
  hipLaunchKernelGGL((prefill_merge_kernel<W, MAPS, ROWS>), rows, dim3(256), 0, st, p);
}

}  // namespace

#endif  // PA_PREFILL_COMMON_H_
