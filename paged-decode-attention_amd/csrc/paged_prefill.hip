// Causal attention of several new tokens of each sequence over the paged KV
// cache, and differential attention of one or several, for MI355X (gfx950).
//
// Sequence b holds T_b tokens, the last n_b of them new (n_b from the start
// offsets of the packed query rows; one each without them). With g query heads
// a kv head, the rows of one (sequence, kv head) are the n_b * g pairs (token,
// head of the group), token-major, so a tile of rows shares every K/V byte and
// its causal edge is a few tokens wide. Row r of token i sees the tokens t <= T_b
// - n_b + i; a row that sees none is zeros.
//
// Differential attention takes heads in pairs: query heads 2i, 2i + 1 are the
// two maps of output head i, kv heads 2j, 2j + 1 hold the keys of maps 1 and 2
// and the two halves of the value, which is twice as wide:
//   o_i = softmax(s q_2i K_2j^T) V_j - lambda_i softmax(s q_2i+1 K_2j+1^T) V_j
// and, with a weight w, o_i * rsqrt(mean(o_i^2) + eps) * w * out_scale. Each map
// is a row of its own in the kernel; neighbouring waves hold the two maps of the
// same rows and meet once, at the end.
//
// A workgroup of four waves takes 128 rows, 32 a wave. K and V of a tile of
// tokens go through registers (where 1-byte and bf16 caches become the fp16
// values that the decode attends over) into LDS, double-buffered: the next
// tile's loads are in flight while this one is computed.
//   S^T[tok, row] = K . Q^T     v_mfma_f32_32x32x16_f16, a lane's column is its row
//   O^T[d, row]  += V^T . P^T   the same; P^T comes straight from the S
//                               accumulators, V^T from LDS by transposing reads
// The softmax runs in the log2 domain over one pass; the running maximum moves
// only when a tile exceeds it by kRescaleLog2, which keeps P below 2^8 and
// leaves most tiles without a rescale. P is rounded to fp16 for its product
// (half a unit in 2^-11, the same rounding as the cache's rows); scores,
// maxima, sums and outputs stay in fp32 until the one rounding of the result.
//
// Where rows are few and sequences long, the tokens are cut into num_splits
// chunks; each writes a normalised fp32 partial and its log2-sum-exp, and a
// second kernel joins them.

#include <hip/hip_runtime.h>
#include <stdint.h>

#include <algorithm>

#include "kv_math.h"
#include "launch_math.h"
#include "pa_errors.h"
#include "pagedattn.h"

namespace {

typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));

constexpr int kWaves = 4;
constexpr int kRowsPerWave = 32;
constexpr float kRescaleLog2 = 8.0f;
constexpr int kSplitUnit = 128;  // splits are multiples of this many tokens
// A lane offset past every buffer (page_rsrc's -1 leaves all others in range):
// the load returns zeros.
constexpr uint32_t kOutside = 0xfffffff0u;
constexpr int kRsrcBytes = (int)kOutside;

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
  int32_t max_seq_len;   // > 0: chunks no shorter than those of a sequence this long
  int32_t tiles;         // row tiles of the launch
  int32_t sqt, sqh, sot, soh;  // elements
  uint32_t skn, skt, skh, ssn, sst;  // bytes
  int32_t sbtb, slam;    // elements
  float qk_scale;        // sm_scale * log2(e)
  float norm_eps, out_scale;
  int32_t io_bf16;
  Div by_units, by_splits, by_group, by_seq_tiles, by_heads;
};

// Compile-time geometry: MAPS maps of head_dim D each, a cache row of W = MAPS *
// D elements, which is also the width of the value.
template <int KV, int D, int MAPS>
struct PGeo {
  static constexpr int W = D * MAPS;
  static constexpr int kElem = (KV == PA_KV_FP16 || KV == PA_KV_BF16) ? 2 : 1;
  static constexpr int BN = W <= 128 ? 64 : 32;         // tokens of a tile
  static constexpr int kPieceBytes = W * kElem >= 64 ? 16 : 8;  // of a lane's load
  static constexpr int kPieceElems = kPieceBytes / kElem;
  static constexpr int kPieceWords = kPieceBytes / 4;
  static constexpr int kPPR = W / kPieceElems;          // pieces of a row: 4 .. 32
  static constexpr int kIter = BN * kPPR / (64 * kWaves);
  // Rows padded so that 16 lanes reading 16 bytes of 16 rows (K), or four rows
  // of 64 bytes read transposed (V), use all 64 banks once.
  static constexpr int kKStride = W * 2 + 16;
  static constexpr int kVStride = W == 32 ? 64 : W * 2 + 64;
  static constexpr int kKBytes = BN * kKStride;
  static constexpr int kBufBytes = kKBytes + BN * kVStride;
  static constexpr int kRowTile = kRowsPerWave * kWaves / MAPS;
  static constexpr int kKSteps = D / 16;
  static constexpr int kDB = W / 32;  // 32-element blocks of the value
  static constexpr int kWavesPerEU = W == 256 ? 1 : 2;
  static_assert(64 / kPPR <= 16 && BN * kPPR % (64 * kWaves) == 0, "a wave's load lies in one page");
};

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

// Tokens of a split of a row tile that sees `hi`, a multiple of UNIT: the tile's own
// chunk, or that of a tile that sees max_seq_len if it is larger (ragged batches:
// long sequences take all splits, short ones few).
template <int UNIT>
__device__ __forceinline__ int split_tokens(const PParams &p, int hi) {
  const uint32_t units = ((uint32_t)max(hi, p.max_seq_len) + UNIT - 1) / UNIT;
  return (int)div_by(units + p.num_splits - 1, p.by_splits) * UNIT;
}

template <int KV, int SC, int D, int MAPS>
struct Staged {
  using G = PGeo<KV, D, MAPS>;
  uint32_t k[G::kIter][G::kPieceWords];
  uint32_t v[G::kIter][G::kPieceWords];
  uint32_t ks[KV == PA_KV_INT8 ? G::kIter : 1];  // int8: scale bits
  uint32_t vs[KV == PA_KV_INT8 ? G::kIter : 1];
};

// The pages of a tile that a wave loads from, by piece.
template <int N>
struct Pages {
  int id[N];
};

// What a lane loads, the same in every tile.
struct LaneAddr {
  uint32_t off;   // bytes from the load's first row
  uint32_t soff;  // int8: of its scale
  int row[4];     // the row in the tile of piece i
};

// First of the 64 / kPPR rows of the tile that a wave's load i covers.
template <int KV, int D, int MAPS>
__device__ __forceinline__ int first_row(int wave, int i) {
  using G = PGeo<KV, D, MAPS>;
  return (64 * wave + 64 * kWaves * i) / G::kPPR;
}

template <int WORDS>
__device__ __forceinline__ void load_piece(uint32_t (&w)[WORDS], __amdgpu_buffer_rsrc_t r, uint32_t off) {
  if constexpr (WORDS == 4) {
    const u32x4 x = __builtin_amdgcn_raw_buffer_load_b128(r, off, 0, 0);
    w[0] = x.x; w[1] = x.y; w[2] = x.z; w[3] = x.w;
  } else {
    const u32x2 x = __builtin_amdgcn_raw_buffer_load_b64(r, off, 0, 0);
    w[0] = x.x; w[1] = x.y;
  }
}

template <int SC>
__device__ __forceinline__ uint32_t load_scale(__amdgpu_buffer_rsrc_t r, uint32_t off) {
  if constexpr (SC == PA_SCALE_FP32) return __builtin_amdgcn_raw_buffer_load_b32(r, off, 0, 0);
  else return __builtin_amdgcn_raw_buffer_load_b16(r, off, 0, 0);
}

// The pages of the tile at n0 that this wave loads from. Rows past the sequence
// take the last token's page (and are read as zeros).
template <int KV, int D, int MAPS>
__device__ __forceinline__ void load_pages(Pages<PGeo<KV, D, MAPS>::kIter> &page, const PParams &p,
                                           const ro_i32 *bt_row, int n0, int len, int wave) {
#pragma unroll
  for (int i = 0; i < PGeo<KV, D, MAPS>::kIter; ++i) {
    const int t = min(n0 + first_row<KV, D, MAPS>(wave, i), len - 1);
    page.id[i] = bt_row[(uint32_t)t >> p.log2_page];
  }
}

// Issue the loads of the tile at n0. Rows at or past `len` read as zeros, so
// what a page holds past the sequence's end never meets a product.
template <int KV, int SC, int D, int MAPS>
__device__ __forceinline__ void load_tile(Staged<KV, SC, D, MAPS> &st, const PParams &p, const uint8_t *kbase,
                                          const uint8_t *vbase, const uint8_t *ksbase, const uint8_t *vsbase,
                                          const Pages<PGeo<KV, D, MAPS>::kIter> &page, const LaneAddr &la, int n0,
                                          int len, int wave) {
  using G = PGeo<KV, D, MAPS>;
#pragma unroll
  for (int i = 0; i < G::kIter; ++i) {
    const int t0 = n0 + first_row<KV, D, MAPS>(wave, i);
    const uint32_t blk = (uint32_t)min(max(page.id[i], 0), p.num_blocks - 1);
    const uint32_t in_page = (uint32_t)t0 & ((1u << p.log2_page) - 1u);
    const uint64_t row0 = (uint64_t)blk * p.skn + in_page * p.skt;
    const bool inside = n0 + la.row[i] < len;
    const uint32_t off = inside ? la.off : kOutside;
    load_piece(st.k[i], page_rsrc(kbase + row0, kRsrcBytes), off);
    load_piece(st.v[i], page_rsrc(vbase + row0, kRsrcBytes), off);
    if constexpr (KV == PA_KV_INT8) {
      const uint64_t srow0 = (uint64_t)blk * p.ssn + in_page * p.sst;
      const uint32_t soff = inside ? la.soff : kOutside;
      st.ks[i] = load_scale<SC>(page_rsrc(ksbase + srow0, kRsrcBytes), soff);
      st.vs[i] = load_scale<SC>(page_rsrc(vsbase + srow0, kRsrcBytes), soff);
    }
  }
}

// A piece's elements as fp16 words (two elements each).
template <int KV, int SC, int WORDS>
__device__ __forceinline__ void to_halves(uint32_t *h, const uint32_t (&w)[WORDS], uint32_t scale_bits) {
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
  } else if constexpr (SC == PA_SCALE_FP16) {
    const uint32_t s2 = scale_bits | (scale_bits << 16);
#pragma unroll
    for (int i = 0; i < WORDS; ++i) {
      h[2 * i] = i8pair_fp16_scale(w[i] ^ kInt8Sign, 0, 1, s2);
      h[2 * i + 1] = i8pair_fp16_scale(w[i] ^ kInt8Sign, 2, 3, s2);
    }
  } else {
    const float s = __uint_as_float(scale_bits) * kInt8Unit, c = s * (-1.0f / 131072.0f);
#pragma unroll
    for (int i = 0; i < WORDS; ++i) {
      const uint32_t x = w[i] ^ kInt8Sign;
      h[2 * i] = i8pair_fp32_scale(perm(x, x, pair_sel<KV>(0, 1)), s, c, s, c);
      h[2 * i + 1] = i8pair_fp32_scale(perm(x, x, pair_sel<KV>(2, 3)), s, c, s, c);
    }
  }
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

// The staged tile into an LDS buffer (K rows, then V rows). With `tame`,
// infinities and NaN of V become zeros, and the result tells whether this lane
// had one.
template <int KV, int SC, int D, int MAPS>
__device__ __forceinline__ bool store_tile(uint8_t *buf, const Staged<KV, SC, D, MAPS> &st, const LaneAddr &la,
                                           int col, bool tame) {
  using G = PGeo<KV, D, MAPS>;
  constexpr int kHalves = G::kPieceElems / 2;  // words
  bool wild = false;
#pragma unroll
  for (int i = 0; i < G::kIter; ++i) {
    uint32_t h[kHalves];
    to_halves<KV, SC>(h, st.k[i], KV == PA_KV_INT8 ? st.ks[KV == PA_KV_INT8 ? i : 0] : 0);
    uint8_t *kd = buf + la.row[i] * G::kKStride + col * 2;
#pragma unroll
    for (int w = 0; w < kHalves; w += 4) *reinterpret_cast<u32x4 *>(kd + 4 * w) = u32x4{h[w], h[w + 1], h[w + 2], h[w + 3]};
    to_halves<KV, SC>(h, st.v[i], KV == PA_KV_INT8 ? st.vs[KV == PA_KV_INT8 ? i : 0] : 0);
    if (tame) {
#pragma unroll
      for (int w = 0; w < kHalves; ++w) wild |= tame_word(h[w]);
    }
    uint8_t *vd = buf + G::kKBytes + la.row[i] * G::kVStride + col * 2;
#pragma unroll
    for (int w = 0; w < kHalves; w += 4) *reinterpret_cast<u32x4 *>(vd + 4 * w) = u32x4{h[w], h[w + 1], h[w + 2], h[w + 3]};
  }
  return wild;
}

// The V^T operand of tokens 16 kb .. + 15 and value elements 32 db .. + 31: lane
// (row d = lane & 31, half h) holds tokens 16 kb + 8 (j / 4) + 4 h + j % 4. Every 16
// lanes read four rows of 16 elements and get a column each.
template <int VSTRIDE>
__device__ __forceinline__ f16x8 read_v(const uint8_t *v, int kb, int db, uint32_t lane_off) {
  typedef __attribute__((address_space(3))) s16x4 lds_s16x4;
  const uint8_t *a = v + 16 * kb * VSTRIDE + 64 * db + lane_off;
  const s16x4 x = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4 *)a);
  const s16x4 y = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4 *)(a + 8 * VSTRIDE));
  const u32x2 xa = __builtin_bit_cast(u32x2, x), ya = __builtin_bit_cast(u32x2, y);
  return as_f16x8(xa.x, xa.y, ya.x, ya.y);
}

template <int D, int W>
struct RowState {
  f16x8 q[D / 16];
  f32x16 acc[W / 32];
  float m;  // running maximum (log2 domain), -inf before the first visible score
  float l;  // sum over this lane's tokens
};

// Scores of a tile's tokens: lane (row = lane & 31, half h) holds those of tokens
// 32 b + 8 (i / 4) + 4 h + i % 4 in s[b][i]. `k`: this lane's K operand in LDS.
template <int KSTEPS, int STRIDE, int NB>
__device__ __forceinline__ void scores_of(f32x16 (&s)[NB], const f16x8 *q, const uint8_t *k) {
#pragma unroll
  for (int b = 0; b < NB; ++b) {
    s[b] = f32x16{};
#pragma unroll
    for (int ks = 0; ks < KSTEPS; ++ks) {
      const f16x8 kop = *reinterpret_cast<const f16x8 *>(k + 32 * b * STRIDE + 32 * ks);
      s[b] = __builtin_amdgcn_mfma_f32_32x32x16_f16(kop, q[ks], s[b], 0, 0, 0);
    }
  }
}

// Scores of tokens that the lane's row does not see (past `lim`) become -inf.
template <int NB>
__device__ __forceinline__ void mask(f32x16 (&s)[NB], int n0, int lim, int h) {
#pragma unroll
  for (int b = 0; b < NB; ++b)
#pragma unroll
    for (int i = 0; i < 16; ++i)
      if (n0 + 32 * b + 8 * (i / 4) + 4 * h + i % 4 > lim) s[b][i] = -INFINITY;
}

// The largest score of the lane's row, in the log2 domain.
template <int NB>
__device__ __forceinline__ float top_score(const f32x16 (&s)[NB], float qk_scale) {
  float top = s[0][0];
#pragma unroll
  for (int b = 0; b < NB; ++b)
#pragma unroll
    for (int i = 0; i < 16; ++i) top = fmaxf(top, s[b][i]);
  return half_max(top) * qk_scale;
}

// Moves the running maximum to `top` where that is far above it.
template <int D, int W>
__device__ __forceinline__ void rescale(RowState<D, W> &st, float top) {
  const bool need = top > st.m + kRescaleLog2;
  if (__builtin_expect(__builtin_amdgcn_ballot_w64(need) != 0, 0)) {
    const float m_new = need ? top : st.m;
    const float alpha = need ? __builtin_amdgcn_exp2f(st.m - m_new) : 1.0f;
    st.l *= alpha;
#pragma unroll
    for (int d = 0; d < W / 32; ++d) st.acc[d] *= alpha;
    st.m = m_new;
  }
}

// Scores to P, and O^T += V^T P^T.
template <int VSTRIDE, int D, int W, int NB>
__device__ __forceinline__ void accumulate(RowState<D, W> &st, f32x16 (&s)[NB], const uint8_t *v, uint32_t v_lane,
                                           float qk_scale) {
  // (a row that has seen nothing yet: every score is -inf and P is 0)
  const float m = st.m == -INFINITY ? 0.f : st.m;
  float sum[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int b = 0; b < NB; ++b)
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      s[b][i] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[b][i], qk_scale, -m));
      sum[i & 3] += s[b][i];
    }
  st.l += (sum[0] + sum[1]) + (sum[2] + sum[3]);
#pragma unroll
  for (int kb = 0; kb < 2 * NB; ++kb) {
    uint32_t w[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const f16x2 two = {(_Float16)s[kb / 2][8 * (kb & 1) + 2 * j], (_Float16)s[kb / 2][8 * (kb & 1) + 2 * j + 1]};
      w[j] = __builtin_bit_cast(uint32_t, two);
    }
    const f16x8 pop = as_f16x8(w[0], w[1], w[2], w[3]);
#pragma unroll
    for (int d = 0; d < W / 32; ++d)
      st.acc[d] = __builtin_amdgcn_mfma_f32_32x32x16_f16(read_v<VSTRIDE>(v, kb, d, v_lane), pop, st.acc[d], 0, 0, 0);
  }
}

// The infinities and NaN of V in a masked tile. A product with P = 0 would hand
// them to rows that do not see their token, so the tile had zeros in their
// place; here they are added to the rows that see them, as they are: whatever P
// above zero they meet, the sum is what it would be.
template <int BN, int VSTRIDE, int D, int W>
__device__ __forceinline__ void add_wild(RowState<D, W> &st, const uint8_t *v, int n0, int lim, int lane) {
  for (int t = 0; t < BN; ++t) {
    const uint8_t *row = v + t * VSTRIDE + 8 * (lane >> 5);
#pragma unroll
    for (int d = 0; d < W / 32; ++d)
#pragma unroll
      for (int i = 0; i < 16; i += 4) {
        const u32x2 w = *reinterpret_cast<const u32x2 *>(row + 64 * d + 4 * i);
        if (n0 + t <= lim && (has_wild(w.x) || has_wild(w.y))) {
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const uint32_t bits = e & 1 ? w[e / 2] >> 16 : w[e / 2] & 0xffffu;
            if ((bits & 0x7c00u) == 0x7c00u) st.acc[d][i + e] += (float)__builtin_bit_cast(_Float16, (uint16_t)bits);
          }
        }
      }
  }
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

// A lane's accumulators (elements 32 d + 2 i + 4 h .. + 3 in acc[d][i .. i + 3], i a
// multiple of 4) as an output row: times f, and with `normed` times the norm's
// weight if there is one.
template <int W>
__device__ __forceinline__ void store_rows(const PParams &p, const f32x16 *acc, float f, bool normed, int packed,
                                           int out_head, int h) {
  uint8_t *dst = p.out + 2 * ((int64_t)packed * p.sot + (int64_t)out_head * p.soh + 4 * h);
  const float *norm = normed ? p.norm : nullptr;
#pragma unroll
  for (int d = 0; d < W / 32; ++d)
#pragma unroll
    for (int i = 0; i < 16; i += 4) {
      f32x4 y = {acc[d][i] * f, acc[d][i + 1] * f, acc[d][i + 2] * f, acc[d][i + 3] * f};
      if (norm) y *= *reinterpret_cast<const f32x4 *>(norm + 32 * d + 2 * i + 4 * h);
      store4(dst + 2 * (32 * d + 2 * i), y.x, y.y, y.z, y.w, p.io_bf16);
    }
}

// The same as a partial: normalised, and its log2-sum-exp.
template <int W>
__device__ __forceinline__ void store_partial(const PParams &p, const f32x16 *acc, float m, float l, int split,
                                              int packed, int head, int h) {
  const int64_t at = ((int64_t)split * p.num_tokens + packed) * p.num_q_heads + head;
  const float inv = l == 0.f ? 0.f : 1.0f / l;
  float *dst = p.part_out + at * W + 4 * h;
#pragma unroll
  for (int d = 0; d < W / 32; ++d)
#pragma unroll
    for (int i = 0; i < 16; i += 4)
      *reinterpret_cast<f32x4 *>(dst + 32 * d + 2 * i) =
          f32x4{acc[d][i] * inv, acc[d][i + 1] * inv, acc[d][i + 2] * inv, acc[d][i + 3] * inv};
  if (h == 0) p.part_lse[at] = l == 0.f ? -INFINITY : m + __log2f(l);
}

template <int KV, int SC, int D, int MAPS>
__global__ void __launch_bounds__(64 * kWaves) __attribute__((amdgpu_waves_per_eu(PGeo<KV, D, MAPS>::kWavesPerEU)))
paged_prefill_kernel(const PParams p) {
  using G = PGeo<KV, D, MAPS>;
  constexpr int W = G::W;
  __shared__ __attribute__((aligned(16))) uint8_t sm[2 * G::kBufBytes];
  __shared__ int sm_wild;  // V holds an infinity or NaN in a masked tile

  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int h = lane >> 5;
  const int map = MAPS == 2 ? wave & 1 : 0;
  const int wave_row = kRowsPerWave * (wave / MAPS);

  // blockIdx = (tile * num_splits + split) * units + unit: the units (kv heads)
  // of the same tokens run together, and with 8 of them each XCD keeps one
  // head's K/V in its L2. Tiles go from the last, which see the most tokens.
  const uint32_t x1 = div_by(blockIdx.x, p.by_units);
  const int unit = blockIdx.x - x1 * p.units;
  const uint32_t x2 = div_by(x1, p.by_splits);
  const int split = x1 - x2 * p.num_splits;
  const int tile = p.tiles - 1 - (int)x2;

  int b, index;
  if (p.start) {
    // sequence b's tiles are numbered from start_b * group / rows + b on: at
    // least as many as it needs
    auto key = [&](int start, int seq) { return (int)((uint32_t)(start * p.group) / G::kRowTile) + seq; };
    b = find_sequence(p, tile, lane, key);
    index = tile - key(row_start(p, b), b);
    if (index < 0) return;
  } else {
    b = div_by(tile, p.by_seq_tiles);
    index = tile - b * p.by_seq_tiles.d;
  }
  const RowTile rt = tile_at<G::kRowTile>(p, b, index);
  if (rt.row0 >= rt.rows) return;

  int lo = 0, hi = rt.hi;
  bool direct = true;  // the row tile is this workgroup's alone: no partials
  if (p.num_splits > 1) {
    const int chunk = split_tokens<kSplitUnit>(p, rt.hi);
    if (split > 0 && (int64_t)split * chunk >= rt.hi) return;  // empty
    lo = split * chunk;
    hi = min(rt.hi, lo + chunk);
    direct = rt.hi <= chunk;
  }

  // this lane's row: its token, its head, the last token it sees
  const int row = rt.row0 + wave_row + (lane & 31);
  const bool live = row < rt.rows;
  const int r = min(row, rt.rows - 1);
  const int token = div_by((uint32_t)r, p.by_group);
  const int head = MAPS * (unit * p.group + (r - token * p.group)) + map;  // query head
  const int lim = rt.first + token;
  // the fewest tokens that a row of the wave sees
  const int least = rt.first + (int)div_by((uint32_t)min(rt.row0 + wave_row, rt.rows - 1), p.by_group) + 1;
  const int least_all = rt.first + (int)div_by((uint32_t)rt.row0, p.by_group) + 1;

  RowState<D, W> st;
  st.m = -INFINITY;
  st.l = 0.f;
#pragma unroll
  for (int d = 0; d < G::kDB; ++d) st.acc[d] = f32x16{};
  {
    const uint16_t *qrow = reinterpret_cast<const uint16_t *>(p.q) + (int64_t)(rt.token0 + token) * p.sqt +
                           (int64_t)head * p.sqh + 8 * h;
#pragma unroll
    for (int ks = 0; ks < G::kKSteps; ++ks) {
      const u32x4 w = *reinterpret_cast<const u32x4 *>(qrow + 16 * ks);
      st.q[ks] = p.io_bf16 ? bf16x8_to_f16x8(w) : __builtin_bit_cast(f16x8, w);
    }
  }

  if (lo < hi) {
    LaneAddr la;
    const int piece = lane % G::kPPR;
    const int col = piece * G::kPieceElems;
#pragma unroll
    for (int i = 0; i < G::kIter; ++i) la.row[i] = (64 * kWaves * i + (int)threadIdx.x) / G::kPPR;
    const uint32_t in_load = (uint32_t)lane / G::kPPR;
    const uint32_t part = (uint32_t)col / D;  // the differential cache row's half
    la.off = in_load * p.skt + part * p.skh + ((uint32_t)col - part * D) * G::kElem;
    la.soff = in_load * p.sst + part * (SC == PA_SCALE_FP32 ? 4 : 2);
    const int64_t head_off = (int64_t)unit * MAPS * p.skh;
    const int64_t scale_off = (int64_t)unit * MAPS * (SC == PA_SCALE_FP32 ? 4 : 2);
    const uint8_t *kbase = p.k + head_off, *vbase = p.v + head_off;
    const uint8_t *ksbase = p.ks + scale_off, *vsbase = p.vs + scale_off;
    const ro_i32 *bt_row = ro(p.bt) + (int64_t)rt.b * p.sbtb;

    Staged<KV, SC, D, MAPS> staged;
    Pages<G::kIter> page;
    auto load = [&](int n0) {
      load_tile<KV, SC, D, MAPS>(staged, p, kbase, vbase, ksbase, vsbase, page, la, n0, rt.len, wave);
    };
    if (threadIdx.x == 0) sm_wild = 0;
    load_pages<KV, D, MAPS>(page, p, bt_row, lo, rt.len, wave);
    load(lo);
    load_pages<KV, D, MAPS>(page, p, bt_row, lo + G::BN, rt.len, wave);
    __syncthreads();  // (sm_wild)
    if (store_tile<KV, SC, D, MAPS>(sm, staged, la, col, lo + G::BN > least_all)) sm_wild = 1;
    __syncthreads();
    const uint32_t k_lane = (lane & 31) * G::kKStride + map * D * 2 + 16 * h;
    const uint32_t v_lane = (4 * h + ((lane & 15) >> 2)) * G::kVStride + 32 * ((lane >> 4) & 1) + 8 * (lane & 3);
    int cur = 0;
    for (int n0 = lo; n0 < hi; n0 += G::BN) {
      const bool more = n0 + G::BN < hi;
      if (more) {
        load(n0 + G::BN);
        load_pages<KV, D, MAPS>(page, p, bt_row, n0 + 2 * G::BN, rt.len, wave);
      }
      const uint8_t *buf = sm + cur * G::kBufBytes;
      f32x16 s[G::BN / 32];
      scores_of<G::kKSteps, G::kKStride>(s, st.q, buf + k_lane);
      if (n0 + G::BN > least) {
        asm volatile("");  // a branch: as selects these would run on every tile
        mask(s, n0, lim, h);
      }
      rescale(st, top_score(s, p.qk_scale));
      accumulate<G::kVStride>(st, s, buf + G::kKBytes, v_lane, p.qk_scale);
      if (more && store_tile<KV, SC, D, MAPS>(sm + (cur ^ 1) * G::kBufBytes, staged, la, col, n0 + 2 * G::BN > least_all))
        sm_wild = 1;
      __syncthreads();
      cur ^= 1;
    }
    if (__builtin_expect(sm_wild, 0)) {
      // the masked tiles once more, with V as it is
      const int from = max(lo, max(least_all - 1, 0) / G::BN * G::BN);
      for (int n0 = from; n0 < hi; n0 += G::BN) {
        load_pages<KV, D, MAPS>(page, p, bt_row, n0, rt.len, wave);
        load(n0);
        store_tile<KV, SC, D, MAPS>(sm, staged, la, col, false);
        __syncthreads();
        if (n0 + G::BN > least_all) add_wild<G::BN, G::kVStride>(st, sm + G::kKBytes, n0, lim, lane);
        __syncthreads();
      }
    }
  }

  const float l = half_sum(st.l);
  if (!direct) {
    if (live) store_partial<W>(p, st.acc, st.m, l, split, rt.token0 + token, head, h);
    return;
  }
  // (a row that sees nothing is zeros; one whose visible scores are all -inf is 0 / 0)
  float inv = lim < 0 ? 0.f : 1.0f / l;
  if constexpr (MAPS == 1) {
    if (live) store_rows<W>(p, st.acc, inv, false, rt.token0 + token, head, h);
  } else {
    float *other = reinterpret_cast<float *>(sm) + (wave / 2) * (W / 2) * 64;
    __syncthreads();  // every wave is done with the tiles
    if (map == 1) {
      inv *= p.lam[(int64_t)(head / 2) * p.slam];
#pragma unroll
      for (int d = 0; d < G::kDB; ++d)
#pragma unroll
        for (int i = 0; i < 16; ++i) other[(16 * d + i) * 64 + lane] = st.acc[d][i] * inv;
    }
    __syncthreads();
    if (map == 1) return;
    float sq = 0.f;
#pragma unroll
    for (int d = 0; d < G::kDB; ++d)
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        st.acc[d][i] = st.acc[d][i] * inv - other[(16 * d + i) * 64 + lane];
        sq += st.acc[d][i] * st.acc[d][i];
      }
    sq = half_sum(sq);
    if (!live) return;
    const float f = p.norm ? __builtin_amdgcn_rsqf(sq * (1.0f / W) + p.norm_eps) * p.out_scale : 1.0f;
    store_rows<W>(p, st.acc, f, true, rt.token0 + token, head / 2, h);
  }
}

// ----------------------------------------------------------------------------
// Few rows: 32 columns of S^T hold all rows of a (sequence, kv head), or of 16 of
// its (token, head) pairs with both maps (columns 0-15 and 16-31). Then the four
// waves of a workgroup share rows, not tokens: wave w takes the 32-token tiles w,
// w + 4, ... of the workgroup's range, through LDS of its own, with no barrier
// until the end, where the four are joined as splits are. What bounds it is the
// stream of K and V: a wave's next tile is in flight while it computes one.
//
// The maps of a differential row differ in the half of the K row they meet: each
// half's products are summed on their own, with q zero in the other map's
// columns, and a lane keeps its column's sum (what the other half holds,
// infinities too, stays out of it).
// ----------------------------------------------------------------------------

template <int KV, int D, int MAPS>
struct SGeo {
  static constexpr int W = D * MAPS;
  static constexpr int kElem = (KV == PA_KV_FP16 || KV == PA_KV_BF16) ? 2 : 1;
  static constexpr int kPieceBytes = W * kElem >= 64 ? 16 : 8;
  static constexpr int kPieceElems = kPieceBytes / kElem;
  static constexpr int kPieceWords = kPieceBytes / 4;
  static constexpr int kPPR = W / kPieceElems;     // 4 .. 32
  static constexpr int kIter = 32 * kPPR / 64;     // loads of K (and of V) a tile
  static constexpr int kKStride = W * 2 + 16;
  static constexpr int kVStride = W == 32 ? 64 : W * 2 + 64;
  static constexpr int kSlot = 32 * (kKStride + kVStride);  // LDS of a wave
  static constexpr int kKSteps = W / 16;
  static constexpr int kDB = W / 32;
  static constexpr int kRowTile = 32 / MAPS;
  static constexpr int kWavesPerEU = W == 256 ? 1 : 2;
  // Rows of 512 bytes: K and V take turns in the same registers (both at once, with
  // accumulators and q, do not fit 512); a wave then has 16 KB in flight as others do.
  static constexpr bool kTurns = W * kElem > 256;
};

// K or V of a tile on its way to LDS.
template <int KV, int D, int MAPS>
struct StreamHalf {
  using G = SGeo<KV, D, MAPS>;
  uint32_t w[G::kIter][G::kPieceWords];
  uint32_t scale[KV == PA_KV_INT8 ? G::kIter : 1];
};

template <int KV, int SC, int D, int MAPS>
__global__ void __launch_bounds__(64 * kWaves) __attribute__((amdgpu_waves_per_eu(SGeo<KV, D, MAPS>::kWavesPerEU)))
paged_stream_kernel(const PParams p) {
  using G = SGeo<KV, D, MAPS>;
  constexpr int W = G::W;
  constexpr int kAccBytes = (kWaves - 1) * (W / 2) * 64 * 4;
  constexpr int kBytes = kWaves * G::kSlot > kAccBytes ? kWaves * G::kSlot : kAccBytes;
  __shared__ __attribute__((aligned(16))) uint8_t sm[kBytes];
  __shared__ float sm_m[kWaves][32], sm_l[kWaves][32];

  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int col = lane & 31, h = lane >> 5;
  const int map = MAPS == 2 ? col >> 4 : 0;

  // blockIdx = (tile * num_splits + split) * units + unit
  const uint32_t x1 = div_by(blockIdx.x, p.by_units);
  const int unit = blockIdx.x - x1 * p.units;
  const uint32_t x2 = div_by(x1, p.by_splits);
  const int split = x1 - x2 * p.num_splits;
  const int tile = (int)x2;
  int b, index;
  if (p.start) {
    auto key = [&](int start, int seq) { return (int)((uint32_t)(start * p.group) / G::kRowTile) + seq; };
    b = find_sequence(p, tile, lane, key);
    index = tile - key(row_start(p, b), b);
    if (index < 0) return;
  } else {
    b = div_by(tile, p.by_seq_tiles);
    index = tile - b * p.by_seq_tiles.d;
  }
  const RowTile rt = tile_at<G::kRowTile>(p, b, index);
  if (rt.row0 >= rt.rows) return;
  int lo = 0, hi = rt.hi;
  bool direct = true;
  if (p.num_splits > 1) {
    const int chunk = split_tokens<kSplitUnit>(p, rt.hi);
    if (split > 0 && (int64_t)split * chunk >= rt.hi) return;
    lo = split * chunk;
    hi = min(rt.hi, lo + chunk);
    direct = rt.hi <= chunk;
  }

  const int row = rt.row0 + (MAPS == 2 ? col & 15 : col);
  const bool live = row < rt.rows;
  const int r = min(row, rt.rows - 1);
  const int token = div_by((uint32_t)r, p.by_group);
  const int head = MAPS * (unit * p.group + (r - token * p.group)) + map;
  const int lim = rt.first + token;
  const int least = rt.first + (int)div_by((uint32_t)rt.row0, p.by_group) + 1;  // tokens that the first row sees

  RowState<W, W> st;
  st.m = -INFINITY;
  st.l = 0.f;
#pragma unroll
  for (int d = 0; d < G::kDB; ++d) st.acc[d] = f32x16{};
  {
    const uint16_t *qrow = reinterpret_cast<const uint16_t *>(p.q) + (int64_t)(rt.token0 + token) * p.sqt +
                           (int64_t)head * p.sqh + 8 * h;
#pragma unroll
    for (int ks = 0; ks < D / 16; ++ks) {
      const u32x4 w = *reinterpret_cast<const u32x4 *>(qrow + 16 * ks);
      const f16x8 x = p.io_bf16 ? bf16x8_to_f16x8(w) : __builtin_bit_cast(f16x8, w);
      if constexpr (MAPS == 1) {
        st.q[ks] = x;
      } else {
        st.q[ks] = map == 0 ? x : f16x8{};
        st.q[D / 16 + ks] = map == 1 ? x : f16x8{};
      }
    }
  }

  // this lane's piece of a load: row (of 64 / kPPR), element
  const int row_in = lane / G::kPPR;
  const int ecol = lane % G::kPPR * G::kPieceElems;
  const uint32_t part = (uint32_t)ecol / D;
  const uint32_t off = row_in * p.skt + part * p.skh + ((uint32_t)ecol - part * D) * G::kElem;
  const uint32_t soff = row_in * p.sst + part * (SC == PA_SCALE_FP32 ? 4 : 2);
  const int64_t head_off = (int64_t)unit * MAPS * p.skh;
  const int64_t scale_off = (int64_t)unit * MAPS * (SC == PA_SCALE_FP32 ? 4 : 2);
  const ro_i32 *bt_row = ro(p.bt) + (int64_t)rt.b * p.sbtb;
  uint8_t *slot = sm + wave * G::kSlot;

  // tile at n0 (a multiple of 32: a 16-token half lies in one page)
  auto pages = [&](int n0, int (&pg)[2]) {
#pragma unroll
    for (int u = 0; u < 2; ++u) pg[u] = bt_row[(uint32_t)min(n0 + 16 * u, rt.len - 1) >> p.log2_page];
  };
  StreamHalf<KV, D, MAPS> first_half, second_half;
  auto &tk = first_half;
  auto &tv = G::kTurns ? first_half : second_half;
  auto load = [&](StreamHalf<KV, D, MAPS> &t, const uint8_t *base, const uint8_t *sbase, int n0, const int (&pg)[2]) {
#pragma unroll
    for (int i = 0; i < G::kIter; ++i) {
      const int r0 = i * (64 / G::kPPR);  // first row of the load
      const uint32_t blk = (uint32_t)min(max(pg[r0 / 16], 0), p.num_blocks - 1);
      const uint32_t in_page = (uint32_t)(n0 + r0) & ((1u << p.log2_page) - 1u);
      const bool inside = n0 + r0 + row_in < rt.len;
      load_piece(t.w[i], page_rsrc(base + head_off + (uint64_t)blk * p.skn + in_page * p.skt, kRsrcBytes),
                 inside ? off : kOutside);
      if constexpr (KV == PA_KV_INT8)
        t.scale[i] = load_scale<SC>(page_rsrc(sbase + scale_off + (uint64_t)blk * p.ssn + in_page * p.sst, kRsrcBytes),
                                    inside ? soff : kOutside);
    }
  };
  auto load_k = [&](int n0, const int (&pg)[2]) { load(tk, p.k, p.ks, n0, pg); };
  auto load_v = [&](int n0, const int (&pg)[2]) { load(tv, p.v, p.vs, n0, pg); };
  // into the wave's slot; with `tame` as store_tile does for V
  auto store = [&](const StreamHalf<KV, D, MAPS> &t, uint8_t *dst, int stride, bool tame) {
    bool wild = false;
#pragma unroll
    for (int i = 0; i < G::kIter; ++i) {
      constexpr int kHalves = G::kPieceElems / 2;
      uint32_t x[kHalves];
      to_halves<KV, SC>(x, t.w[i], KV == PA_KV_INT8 ? t.scale[KV == PA_KV_INT8 ? i : 0] : 0);
      if (tame) {
#pragma unroll
        for (int w = 0; w < kHalves; ++w) wild |= tame_word(x[w]);
      }
      uint8_t *d = dst + (i * (64 / G::kPPR) + row_in) * stride + ecol * 2;
#pragma unroll
      for (int w = 0; w < kHalves; w += 4) *reinterpret_cast<u32x4 *>(d + 4 * w) = u32x4{x[w], x[w + 1], x[w + 2], x[w + 3]};
    }
    return wild;
  };
  auto store_k = [&] { store(tk, slot, G::kKStride, false); };
  auto store_v = [&](bool tame) { return store(tv, slot + 32 * G::kKStride, G::kVStride, tame); };
  auto sync_slot = [] {
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
  };

  const uint8_t *k_lane = slot + col * G::kKStride + 16 * h;
  const uint8_t *v_slot = slot + 32 * G::kKStride;
  const uint32_t v_lane = (4 * h + ((lane & 15) >> 2)) * G::kVStride + 32 * ((lane >> 4) & 1) + 8 * (lane & 3);
  const int n_first = lo + 32 * wave;
  bool wild = false;
  if (n_first < hi) {
    int pg[2];
    pages(n_first, pg);
    load_k(n_first, pg);
    if constexpr (G::kTurns) store_k();
    load_v(n_first, pg);
    pages(n_first + 32 * kWaves, pg);
    for (int n0 = n_first; n0 < hi; n0 += 32 * kWaves) {
      const bool masked = n0 + 32 > least;
      const int next = n0 + 32 * kWaves;
      if constexpr (!G::kTurns) {
        store_k();
        wild |= store_v(masked);
      }
      sync_slot();
      if (!G::kTurns && next < hi) {
        load_k(next, pg);
        load_v(next, pg);
        pages(next + 32 * kWaves, pg);
      }
      f32x16 s[1];
      if constexpr (MAPS == 1) {
        scores_of<G::kKSteps, G::kKStride>(s, st.q, k_lane);
      } else {
        f32x16 s2[1];
        scores_of<G::kKSteps / 2, G::kKStride>(s, st.q, k_lane);
        scores_of<G::kKSteps / 2, G::kKStride>(s2, st.q + G::kKSteps / 2, k_lane + 2 * D);
#pragma unroll
        for (int i = 0; i < 16; ++i) s[0][i] = map == 1 ? s2[0][i] : s[0][i];
      }
      if (masked) {
        asm volatile("");  // a branch
        mask(s, n0, lim, h);
      }
      rescale(st, top_score(s, p.qk_scale));
      if constexpr (G::kTurns) {
        wild |= store_v(masked);
        sync_slot();
        if (next < hi) load_k(next, pg);
      }
      accumulate<G::kVStride>(st, s, v_slot, v_lane, p.qk_scale);
      sync_slot();
      if (G::kTurns && next < hi) {
        store_k();
        load_v(next, pg);
        pages(next + 32 * kWaves, pg);
      }
    }
    if (__builtin_expect(__builtin_amdgcn_ballot_w64(wild) != 0, 0)) {
      for (int n0 = n_first; n0 < hi; n0 += 32 * kWaves) {
        if (n0 + 32 <= least) continue;
        pages(n0, pg);
        load_v(n0, pg);
        store_v(false);
        sync_slot();
        add_wild<32, G::kVStride>(st, v_slot, n0, lim, lane);
        sync_slot();
      }
    }
  }

  // join the waves
  const float lw = half_sum(st.l);
  if (h == 0) {
    sm_m[wave][col] = st.m;
    sm_l[wave][col] = lw;
  }
  __syncthreads();  // (and every wave is done with its slot)
  float m = -INFINITY;
#pragma unroll
  for (int w = 0; w < kWaves; ++w) m = fmaxf(m, sm_m[w][col]);
  float l = 0.f;
#pragma unroll
  for (int w = 0; w < kWaves; ++w) {
    const float mw = sm_m[w][col];
    // (a wave that saw nothing of the row has a sum of zero)
    l += mw == -INFINITY ? sm_l[w][col] : sm_l[w][col] * __builtin_amdgcn_exp2f(mw - m);
  }
  const float f = st.m == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(st.m - m);
  float *others = reinterpret_cast<float *>(sm);
  if (wave > 0) {
#pragma unroll
    for (int d = 0; d < G::kDB; ++d)
#pragma unroll
      for (int i = 0; i < 16; ++i) others[((wave - 1) * (W / 2) + 16 * d + i) * 64 + lane] = st.acc[d][i] * f;
  }
  __syncthreads();
  if (wave > 0) return;
#pragma unroll
  for (int d = 0; d < G::kDB; ++d)
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      float a = st.acc[d][i] * f;
#pragma unroll
      for (int w = 1; w < kWaves; ++w) a += others[((w - 1) * (W / 2) + 16 * d + i) * 64 + lane];
      st.acc[d][i] = a;
    }
  if (!direct) {
    if (live) store_partial<W>(p, st.acc, m, l, split, rt.token0 + token, head, h);
    return;
  }
  float inv = lim < 0 ? 0.f : 1.0f / l;
  if constexpr (MAPS == 1) {
    if (live) store_rows<W>(p, st.acc, inv, false, rt.token0 + token, head, h);
  } else {
    // columns c and c + 16 (lanes apart by 16) hold the maps of a row
    if (map == 1) inv *= p.lam[(int64_t)(head / 2) * p.slam];
    float sq = 0.f;
#pragma unroll
    for (int d = 0; d < G::kDB; ++d)
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const uint32_t x = __float_as_uint(st.acc[d][i] * inv);
        const auto two = __builtin_amdgcn_permlane16_swap(x, x, false, false);
        const float y = __uint_as_float(two[0]) - __uint_as_float(two[1]);
        st.acc[d][i] = y;
        sq += y * y;
      }
    sq = half_sum(sq);
    if (live && map == 0) {
      const float scale = p.norm ? __builtin_amdgcn_rsqf(sq * (1.0f / W) + p.norm_eps) * p.out_scale : 1.0f;
      store_rows<W>(p, st.acc, scale, true, rt.token0 + token, head / 2, h);
    }
  }
}

// Joins the partials of a split launch: one wave an output row, W / 64 elements a
// lane (W = 32: the upper half of the wave idles). Row tiles of one split are done;
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
  const int chunk = split_tokens<kSplitUnit>(p, rt.hi);
  if (rt.hi <= chunk) return;  // written by its one workgroup
  const int n = (rt.hi - 1) / chunk + 1;
  const bool sees = rt.first + token >= 0;

  float y[E] = {};
  const int d0 = E * lane;
  const bool mine = d0 < W;
#pragma unroll
  for (int map = 0; map < MAPS; ++map) {
    const int64_t at = (int64_t)packed * p.num_q_heads + MAPS * out_head + map;
    const int64_t step = (int64_t)p.num_tokens * p.num_q_heads;
    float m = -INFINITY, sum = 0.f, acc[E] = {};
    for (int s = 0; s < n; ++s) {
      const float lse = p.part_lse[at + s * step];
      float o[E] = {};
      if (mine) {
#pragma unroll
        for (int e = 0; e < E; ++e) o[e] = p.part_out[(at + s * step) * W + d0 + e];
      }
      if (lse == -INFINITY) continue;
      const float m_new = lse > m ? lse : m;
      const float old = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m - m_new);
      const float w = __builtin_amdgcn_exp2f(lse - m_new);
      sum = sum * old + w;
#pragma unroll
      for (int e = 0; e < E; ++e) acc[e] = acc[e] * old + w * o[e];
      m = m_new;
    }
    const float inv = sees ? 1.0f / sum : 0.f;
    const float f = map == 1 ? -inv * p.lam[(int64_t)out_head * p.slam] : inv;
#pragma unroll
    for (int e = 0; e < E; ++e) y[e] += acc[e] * f;
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

bool fits_i32(int64_t x) { return x >= 0 && x < (int64_t(1) << 31); }

int build(const pa_prefill_args *a, int maps, PParams *out) {
  if (a == nullptr) return pa_fail(PA_ERR_INVALID, "args is NULL");
  if (!a->q || !a->k_cache || !a->v_cache || !a->out || !a->block_table || !a->seq_lens)
    return pa_fail(PA_ERR_INVALID, "q, k_cache, v_cache, out, block_table and seq_lens must be non-NULL");
  if (a->batch < 0 || a->num_tokens < 0) return pa_fail(PA_ERR_INVALID, "batch %d and num_tokens %d must not be negative", a->batch, a->num_tokens);
  if (a->num_q_heads <= 0 || a->num_kv_heads <= 0 || a->num_q_heads % a->num_kv_heads)
    return pa_fail(PA_ERR_INVALID, "num_q_heads %d must be a multiple of num_kv_heads %d", a->num_q_heads, a->num_kv_heads);
  if (a->num_blocks <= 0 || a->max_blocks <= 0)
    return pa_fail(PA_ERR_INVALID, "num_blocks %d and max_blocks %d must be positive", a->num_blocks, a->max_blocks);
  const int d = a->head_dim;
  if (d != 32 && d != 64 && d != 128 && (d != 256 || maps == 2))
    return pa_fail(PA_ERR_UNSUPPORTED, "head_dim %d not in %s", d, maps == 2 ? "(32, 64, 128)" : "(32, 64, 128, 256)");
  const int bs = a->block_size;
  if (bs < 16 || bs > 256 || (bs & (bs - 1)))
    return pa_fail(PA_ERR_UNSUPPORTED, "block_size %d is not a power of two in [16, 256]", bs);
  if (a->kv_dtype != PA_KV_FP16 && a->kv_dtype != PA_KV_FP8_E5M2 && a->kv_dtype != PA_KV_INT8 && a->kv_dtype != PA_KV_BF16)
    return pa_fail(PA_ERR_INVALID, "kv_dtype %d unknown", a->kv_dtype);
  if (a->io_dtype != PA_IO_FP16 && a->io_dtype != PA_IO_BF16) return pa_fail(PA_ERR_INVALID, "io_dtype %d unknown", a->io_dtype);
  if (!(a->sm_scale > 0.0f) || a->sm_scale * kLog2e > 3.0e38f)
    return pa_fail(PA_ERR_INVALID, "sm_scale must be positive and finite");
  if (a->num_splits < 1 || a->num_splits > PA_MAX_SPLITS)
    return pa_fail(PA_ERR_INVALID, "num_splits %d not in [1, %d]", a->num_splits, PA_MAX_SPLITS);
  if (a->num_splits > 1 && (!a->part_out || !a->part_lse))
    return pa_fail(PA_ERR_INVALID, "num_splits %d needs part_out and part_lse", a->num_splits);
  if (a->max_seq_len < 0) return pa_fail(PA_ERR_INVALID, "max_seq_len %d < 0", a->max_seq_len);
  if (a->form != PA_FORM_TILES && a->form != PA_FORM_STREAMS) return pa_fail(PA_ERR_INVALID, "form %d unknown", a->form);
  if (!a->query_start_loc && a->num_tokens != a->batch)
    return pa_fail(PA_ERR_INVALID, "without query_start_loc num_tokens (%d) must be batch (%d)", a->num_tokens, a->batch);
  const int64_t elem = (a->kv_dtype == PA_KV_FP16 || a->kv_dtype == PA_KV_BF16) ? 2 : 1;
  const int64_t strides[] = {a->stride_qt, a->stride_qh, a->stride_kn, a->stride_kt, a->stride_kh,
                             a->stride_ot, a->stride_oh, a->stride_btb};
  for (int64_t s : strides)
    if (s < 0) return pa_fail(PA_ERR_INVALID, "strides must be non-negative");
  if (!pa_aligned(a->q, 16) || a->stride_qt % 8 || a->stride_qh % 8)
    return pa_fail(PA_ERR_INVALID, "q and its strides must be 16-byte aligned");
  if (!pa_aligned(a->out, 16) || a->stride_ot % 8 || a->stride_oh % 8)
    return pa_fail(PA_ERR_INVALID, "out and its strides must be 16-byte aligned");
  if (!pa_aligned(a->k_cache, 16) || !pa_aligned(a->v_cache, 16) || a->stride_kn * elem % 16 ||
      a->stride_kt * elem % 16 || a->stride_kh * elem % 16)
    return pa_fail(PA_ERR_INVALID, "k_cache, v_cache and their strides must be 16-byte aligned");
  if (a->num_splits > 1 && (!pa_aligned(a->part_out, 16) || !pa_aligned(a->part_lse, 4)))
    return pa_fail(PA_ERR_INVALID, "part_out must be 16-byte aligned, part_lse 4-byte");
  int64_t sb = 0;
  if (a->kv_dtype == PA_KV_INT8) {
    if (a->scale_dtype != PA_SCALE_FP16 && a->scale_dtype != PA_SCALE_FP32)
      return pa_fail(PA_ERR_INVALID, "int8 KV needs scale_dtype fp16 or fp32, got %d", a->scale_dtype);
    if (!a->k_scale || !a->v_scale) return pa_fail(PA_ERR_INVALID, "int8 KV needs k_scale and v_scale");
    if (a->stride_sn < 0 || a->stride_st < 0) return pa_fail(PA_ERR_INVALID, "scale strides must be non-negative");
    sb = a->scale_dtype == PA_SCALE_FP32 ? 4 : 2;
    if (!pa_aligned(a->k_scale, (int)sb) || !pa_aligned(a->v_scale, (int)sb))
      return pa_fail(PA_ERR_INVALID, "scale pointers must be %d-byte aligned", (int)sb);
  } else if (a->scale_dtype != PA_SCALE_NONE) {
    return pa_fail(PA_ERR_INVALID, "scale_dtype must be PA_SCALE_NONE for kv_dtype %d", a->kv_dtype);
  }
  if (maps == 2) {
    if (a->num_kv_heads % 2) return pa_fail(PA_ERR_INVALID, "differential attention takes kv heads in pairs, got %d", a->num_kv_heads);
    if (!a->lam || !pa_aligned(a->lam, 4) || !fits_i32(a->stride_lam)) return pa_fail(PA_ERR_INVALID, "lam must be non-NULL and 4-byte aligned, its stride non-negative");
    if (a->norm_weight && !pa_aligned(a->norm_weight, 16)) return pa_fail(PA_ERR_INVALID, "norm_weight must be 16-byte aligned");
  }
  const int64_t gib = int64_t(1) << 30;
  if ((int64_t)a->max_blocks * bs >= 2 * gib) return pa_fail(PA_ERR_UNSUPPORTED, "max_blocks * block_size must be below 2^31 tokens");
  if ((int64_t)std::max(a->batch, 1) * a->stride_btb >= 2 * gib) return pa_fail(PA_ERR_UNSUPPORTED, "batch * stride_btb must be below 2^31");
  if (bs * a->stride_kt * elem >= 2 * gib || a->stride_kn * elem >= 4 * gib || a->stride_kh * elem >= 2 * gib ||
      bs * a->stride_st * sb >= 2 * gib || a->stride_sn * sb >= 4 * gib)
    return pa_fail(PA_ERR_UNSUPPORTED, "a page must be under 2 GiB, page strides under 4 GiB, the kv-head stride under 2 GiB");
  if (16 * a->stride_kt * elem + (maps - 1) * a->stride_kh * elem >= 4 * gib - 4096)
    return pa_fail(PA_ERR_UNSUPPORTED, "a pair of kv heads must lie within 4 GiB");
  if (!fits_i32(a->stride_qt) || !fits_i32(a->stride_qh) || !fits_i32(a->stride_ot) || !fits_i32(a->stride_oh))
    return pa_fail(PA_ERR_UNSUPPORTED, "q and out strides must be below 2^31 elements");
  const int group = a->num_q_heads / a->num_kv_heads;
  const int units = a->num_kv_heads / maps;
  if ((int64_t)a->num_tokens * a->num_q_heads >= 2 * gib) return pa_fail(PA_ERR_UNSUPPORTED, "num_tokens * num_q_heads must be below 2^31");
  const int row_tile = a->form == PA_FORM_STREAMS ? kRowsPerWave / maps : kRowsPerWave * kWaves / maps;
  const int seq_tiles = (group + row_tile - 1) / row_tile;
  const int64_t tiles = a->query_start_loc ? (int64_t)a->num_tokens * group / row_tile + a->batch
                                           : (int64_t)a->batch * seq_tiles;
  if (tiles * units * a->num_splits >= 2 * gib) return pa_fail(PA_ERR_UNSUPPORTED, "too many workgroups");

  PParams p = {};
  p.q = static_cast<const uint8_t *>(a->q);
  p.k = static_cast<const uint8_t *>(a->k_cache);
  p.v = static_cast<const uint8_t *>(a->v_cache);
  p.ks = static_cast<const uint8_t *>(a->k_scale);
  p.vs = static_cast<const uint8_t *>(a->v_scale);
  p.out = static_cast<uint8_t *>(a->out);
  p.part_out = a->part_out;
  p.part_lse = a->part_lse;
  p.bt = a->block_table;
  p.seq_lens = a->seq_lens;
  p.start = a->query_start_loc;
  p.lam = a->lam;
  p.norm = maps == 2 ? a->norm_weight : nullptr;
  p.batch = a->batch;
  p.num_tokens = a->num_tokens;
  p.units = units;
  p.group = group;
  p.num_q_heads = a->num_q_heads;
  p.num_blocks = a->num_blocks;
  p.max_tokens = a->max_blocks * bs;
  p.log2_page = __builtin_ctz((unsigned)bs);
  p.num_splits = a->num_splits;
  p.max_seq_len = std::min(a->max_seq_len, p.max_tokens);
  p.tiles = (int32_t)tiles;
  p.sqt = (int32_t)a->stride_qt;
  p.sqh = (int32_t)a->stride_qh;
  p.sot = (int32_t)a->stride_ot;
  p.soh = (int32_t)a->stride_oh;
  p.skn = (uint32_t)(a->stride_kn * elem);
  p.skt = (uint32_t)(a->stride_kt * elem);
  p.skh = (uint32_t)(a->stride_kh * elem);
  p.ssn = (uint32_t)(a->stride_sn * sb);
  p.sst = (uint32_t)(a->stride_st * sb);
  p.sbtb = (int32_t)a->stride_btb;
  p.slam = (int32_t)a->stride_lam;
  p.qk_scale = a->sm_scale * kLog2e;
  p.norm_eps = a->norm_eps;
  p.out_scale = a->out_scale;
  p.io_bf16 = a->io_dtype == PA_IO_BF16;
  p.by_units = make_div(units);
  p.by_splits = make_div(a->num_splits);
  p.by_group = make_div(group);
  p.by_seq_tiles = make_div(seq_tiles);
  p.by_heads = make_div(a->num_q_heads / maps);
  *out = p;
  return PA_OK;
}

template <int KV, int SC, int D, int MAPS>
hipError_t launch(const PParams &p, bool streams, hipStream_t st) {
  constexpr int W = D * MAPS;
  const dim3 grid((uint32_t)(p.tiles * p.units * p.num_splits)), threads(64 * kWaves);
  if (streams)
    hipLaunchKernelGGL((paged_stream_kernel<KV, SC, D, MAPS>), grid, threads, 0, st, p);
  else
    hipLaunchKernelGGL((paged_prefill_kernel<KV, SC, D, MAPS>), grid, threads, 0, st, p);
  if (p.num_splits > 1) {
    const dim3 rows(((uint32_t)p.num_tokens * (uint32_t)(p.num_q_heads / MAPS) + 3) / 4);
    if (streams)
      hipLaunchKernelGGL((prefill_merge_kernel<W, MAPS, SGeo<KV, D, MAPS>::kRowTile>), rows, dim3(256), 0, st, p);
    else
      hipLaunchKernelGGL((prefill_merge_kernel<W, MAPS, PGeo<KV, D, MAPS>::kRowTile>), rows, dim3(256), 0, st, p);
  }
  return hipGetLastError();
}

template <int KV, int SC>
hipError_t launch_kv(const PParams &p, int d, int maps, bool streams, hipStream_t st) {
  if (maps == 1) {
    switch (d) {
      case 32: return launch<KV, SC, 32, 1>(p, streams, st);
      case 64: return launch<KV, SC, 64, 1>(p, streams, st);
      case 128: return launch<KV, SC, 128, 1>(p, streams, st);
      default: return launch<KV, SC, 256, 1>(p, streams, st);
    }
  }
  switch (d) {
    case 32: return launch<KV, SC, 32, 2>(p, streams, st);
    case 64: return launch<KV, SC, 64, 2>(p, streams, st);
    default: return launch<KV, SC, 128, 2>(p, streams, st);
  }
}

int attend(const pa_prefill_args *a, int maps, void *stream) {
  PParams p;
  const int rc = build(a, maps, &p);
  if (rc != PA_OK) return rc;
  if (p.tiles == 0 || p.num_tokens == 0) return pa_ok();
  hipStream_t st = static_cast<hipStream_t>(stream);
  const int d = a->head_dim;
  const bool streams = a->form == PA_FORM_STREAMS;
  hipError_t e;
  if (a->kv_dtype == PA_KV_FP16) e = launch_kv<PA_KV_FP16, PA_SCALE_NONE>(p, d, maps, streams, st);
  else if (a->kv_dtype == PA_KV_BF16) e = launch_kv<PA_KV_BF16, PA_SCALE_NONE>(p, d, maps, streams, st);
  else if (a->kv_dtype == PA_KV_FP8_E5M2) e = launch_kv<PA_KV_FP8_E5M2, PA_SCALE_NONE>(p, d, maps, streams, st);
  else if (a->scale_dtype == PA_SCALE_FP32) e = launch_kv<PA_KV_INT8, PA_SCALE_FP32>(p, d, maps, streams, st);
  else e = launch_kv<PA_KV_INT8, PA_SCALE_FP16>(p, d, maps, streams, st);
  if (e != hipSuccess) return pa_fail(PA_ERR_HIP, "launch failed: %s", hipGetErrorString(e));
  return pa_ok();
}

}  // namespace

extern "C" {

int pa_prefill(const pa_prefill_args *a, void *stream) {
  if (a && !a->query_start_loc) return pa_fail(PA_ERR_INVALID, "query_start_loc must be non-NULL");
  return attend(a, 1, stream);
}

int pa_diff_prefill(const pa_prefill_args *a, void *stream) {
  if (a && !a->query_start_loc) return pa_fail(PA_ERR_INVALID, "query_start_loc must be non-NULL");
  return attend(a, 2, stream);
}

int pa_diff_decode(const pa_prefill_args *a, void *stream) {
  if (a && a->query_start_loc) return pa_fail(PA_ERR_INVALID, "query_start_loc must be NULL: one query token a sequence");
  return attend(a, 2, stream);
}

}  // extern "C"
