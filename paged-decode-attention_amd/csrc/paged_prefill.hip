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
// A workgroup takes 32 rows a wave, 128 or 256 in all. K and V of a tile of tokens go
// through registers (where 1-byte and bf16 caches become fp16; int8 values exactly,
// their scales meet the scores and P) into LDS, double-buffered: the next tile's loads
// are in flight while this one is computed.
//   S^T[tok, row] = K . Q^T     v_mfma_f32_32x32x16_f16, a lane's column is its row
//   O^T[d, row]  += V^T . P^T   the same; P^T comes straight from the S
//                               accumulators, V^T from LDS by transposing reads
// The softmax runs in the log2 domain over one pass; the running maximum moves
// only when a tile exceeds it by kRescaleLog2, which leaves most tiles without a
// rescale. P is rounded to fp16 for its product (half a step of 2^-10: 1.3 times the
// error that the result's own rounding makes, see the streams for two products);
// scores, maxima, sums and outputs stay in fp32 until the one rounding of the result.
//
// What bounds it: a long prompt the card's power (16,384 tokens, 32 q / 8 kv heads of
// 128, fp16: 2,210-2,300 us, 960-990 TFLOP/s; with all inputs zero 1,855, and a library
// product of 8192^3 runs at 1,140-1,350 on data, 1,810 on zeros); in between, the
// softmax's VALU instructions, about as long as the products that they alternate with;
// small launches the latency of the chain length -> page -> K. Tried and slower or equal:
// K a tile ahead of V with its products between the softmax's instructions, three
// waves a SIMD on 32-token tiles, s_setprio around the products, block-table entries in
// lanes instead of scalar loads.
//
// Where rows are few and sequences long, the tokens are cut into num_splits
// chunks; each writes a normalised fp32 partial and its log2-sum-exp, and a
// second kernel joins them. Fewer rows still: paged_stream.hip.

#include <hip/hip_runtime.h>
#include <stdint.h>

#include <algorithm>

#include "pa_errors.h"
#include "pagedattn.h"
#include "prefill_common.h"

namespace {

// Waves of a workgroup, two on a SIMD. Rows of 128 elements on: eight of one
// workgroup, which share the loads, the staging registers and the LDS of a tile
// (against two workgroups of four: a prompt of 16,384 tokens, 32 q / 8 kv heads
// 2,380 -> 2,235 us; pairs of 128-element heads do not fit two waves otherwise, 505
// -> 270 us for 4,096 tokens). Heads of 256: four, their accumulators and q take a
// SIMD's registers.
template <int D, int MAPS> constexpr int kTileWaves = D * MAPS >= 128 && D < 256 ? 8 : 4;

// Compile-time geometry: MAPS maps of head_dim D each, a cache row of W = MAPS *
// D elements, which is also the width of the value.
template <int KV, int D, int MAPS>
struct PGeo {
  static constexpr int W = D * MAPS;
  static constexpr int kElem = (KV == PA_KV_FP16 || KV == PA_KV_BF16) ? 2 : 1;
  static constexpr int kNW = kTileWaves<D, MAPS>;       // waves of a workgroup
  static constexpr int BN = W <= 128 ? 64 : 32;         // tokens of a tile
  static constexpr int kPieceBytes = W * kElem >= 64 ? 16 : 8;  // of a lane's load
  static constexpr int kPieceElems = kPieceBytes / kElem;
  static constexpr int kPieceWords = kPieceBytes / 4;
  static constexpr int kPPR = W / kPieceElems;          // pieces of a row: 4 .. 32
  static constexpr int kIter = BN * kPPR / (64 * kNW);
  // Rows padded so that 16 lanes reading 16 bytes of 16 rows (K), or four rows
  // of 64 bytes read transposed (V), use all 64 banks once.
  static constexpr int kKStride = W * 2 + 16;
  static constexpr int kVStride = W == 32 ? 64 : W * 2 + 64;
  static constexpr int kKBytes = BN * kKStride;
  static constexpr int kBufBytes = kKBytes + BN * kVStride;
  static constexpr int kRowTile = kRowsPerWave * kNW / MAPS;
  static constexpr int kKSteps = D / 16;
  static constexpr int kDB = W / 32;  // 32-element blocks of the value
  static constexpr int kWavesPerEU = D == 256 ? 1 : 2;
  static_assert(64 / kPPR <= 16 && BN * kPPR % (64 * kNW) == 0, "a wave's load lies in one page");
};

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
  return (64 * wave + 64 * G::kNW * i) / G::kPPR;
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
    load_piece<0>(st.k[i], page_rsrc(kbase + row0, kRsrcBytes), off);
    load_piece<0>(st.v[i], page_rsrc(vbase + row0, kRsrcBytes), off);
    if constexpr (KV == PA_KV_INT8) {
      const uint64_t srow0 = (uint64_t)blk * p.ssn + in_page * p.sst;
      const uint32_t soff = inside ? la.soff : kOutside;
      st.ks[i] = load_scale<SC>(page_rsrc(ksbase + srow0, kRsrcBytes), soff);
      st.vs[i] = load_scale<SC>(page_rsrc(vsbase + srow0, kRsrcBytes), soff);
    }
  }
}

// The staged tile into an LDS buffer (K rows, then V rows). With `tame`,
// infinities and NaN of V become zeros, and the result tells whether this lane
// had one. int8: the scales of K's MAPS heads, then V's, into `scales`.
template <int KV, int SC, int D, int MAPS>
__device__ __forceinline__ bool store_tile(uint8_t *buf, const Staged<KV, SC, D, MAPS> &st, const LaneAddr &la,
                                           int col, bool tame, float *scales) {
  using G = PGeo<KV, D, MAPS>;
  constexpr int kHalves = G::kPieceElems / 2;  // words
  bool wild = false;
#pragma unroll
  for (int i = 0; i < G::kIter; ++i) {
    uint32_t h[kHalves];
    to_halves<KV>(h, st.k[i]);
    uint8_t *kd = buf + la.row[i] * G::kKStride + col * 2;
#pragma unroll
    for (int w = 0; w < kHalves; w += 4) *reinterpret_cast<u32x4 *>(kd + 4 * w) = u32x4{h[w], h[w + 1], h[w + 2], h[w + 3]};
    to_halves<KV>(h, st.v[i]);
    if (KV != PA_KV_INT8 && tame) {
#pragma unroll
      for (int w = 0; w < kHalves; ++w) wild |= tame_word(h[w]);
    }
    uint8_t *vd = buf + G::kKBytes + la.row[i] * G::kVStride + col * 2;
#pragma unroll
    for (int w = 0; w < kHalves; w += 4) *reinterpret_cast<u32x4 *>(vd + 4 * w) = u32x4{h[w], h[w + 1], h[w + 2], h[w + 3]};
    if constexpr (KV == PA_KV_INT8) {
      if (col % D == 0) {
        scales[col / D * G::BN + la.row[i]] = scale_value<SC>(st.ks[i]);
        scales[(MAPS + col / D) * G::BN + la.row[i]] = finite_scale(scale_value<SC>(st.vs[i]));
      }
    }
  }
  return wild;
}

template <int D, int W>
struct RowState {
  f16x8 q[D / 16];
  f32x16 acc[W / 32];
  float m;  // running maximum - kTopLog2 (log2 domain), -inf before the first visible score
  float l;  // sum over this lane's tokens
  float limit;  // int8: the accumulators' unit (raise_limit)
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
  const bool need = top > st.m + (kTopLog2 + kRescaleLog2);
  if (__builtin_expect(__builtin_amdgcn_ballot_w64(need) != 0, 0)) {
    const float m_new = need ? top - kTopLog2 : st.m;
    const float alpha = need ? __builtin_amdgcn_exp2f(st.m - m_new) : 1.0f;
    st.l *= alpha;
#pragma unroll
    for (int d = 0; d < W / 32; ++d) st.acc[d] *= alpha;
    st.m = m_new;
  }
}

// Scores to P, and O^T += V^T P^T, 16 tokens a product: lane (row d = lane & 31, half
// h) holds tokens 16 kb + 8 (j / 4) + 4 h + j % 4 of V^T, as the scores lie.
// int8 (PARTS > 0: heads of a value row): times V's scales in `vs`, over the limit.
template <int VSTRIDE, int PARTS, int D, int W, int NB>
__device__ __forceinline__ void accumulate(RowState<D, W> &st, f32x16 (&s)[NB], const uint8_t *v, uint32_t v_lane,
                                           float qk_scale, const float *vs, int h) {
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
  constexpr int kHeads = PARTS > 0 ? PARTS : 1;
  float inv = 1.f;
  if constexpr (PARTS > 0) {
    float top = 0.f;
#pragma unroll
    for (int part = 0; part < PARTS; ++part)
#pragma unroll
      for (int e = 0; e < 16 * NB; e += 4) {
        const f32x4 v4 = *reinterpret_cast<const f32x4 *>(vs + 32 * NB * part + score_token<32>(e, h));
#pragma unroll
        for (int j = 0; j < 4; ++j) top = fmaxf(top, fabsf(s[e / 16][e % 16 + j] * v4[j]));
      }
    bool any;
    const float f = raise_limit<32>(st.limit, top, any);
    if (__builtin_expect(any, 0)) {
#pragma unroll
      for (int d = 0; d < W / 32; ++d) st.acc[d] *= f;
    }
    inv = inverse_limit(st.limit);
  }
#pragma unroll
  for (int kb = 0; kb < 2 * NB; ++kb) {
    f16x8 pop[kHeads];
#pragma unroll
    for (int part = 0; part < kHeads; ++part) {
      uint32_t w[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int i = 8 * (kb & 1) + 2 * j;
        float a = s[kb / 2][i], b = s[kb / 2][i + 1];
        if constexpr (PARTS > 0) {
          const float *at = vs + 32 * NB * part + score_token<32>(8 * kb + 2 * j, h);
          a = a * at[0] * inv;  // (in this order: 0 times the largest scale is 0)
          b = b * at[1] * inv;
        }
        const f16x2 two = {(_Float16)a, (_Float16)b};
        w[j] = __builtin_bit_cast(uint32_t, two);
      }
      pop[part] = as_f16x8(w[0], w[1], w[2], w[3]);
    }
#pragma unroll
    for (int d = 0; d < W / 32; ++d)
      st.acc[d] = __builtin_amdgcn_mfma_f32_32x32x16_f16(
          read_columns(v + 16 * kb * VSTRIDE + 64 * d + v_lane, 8 * VSTRIDE), pop[d * kHeads / (W / 32)], st.acc[d], 0, 0, 0);
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

// The row tile of this rank, longest first: a launch of a few rounds of workgroups
// otherwise ends with whatever long tiles come last, alone on their CUs. Tile i of
// sequence b sees about o_b + i row tiles' worth of tokens, o_b those before its new
// ones, so count(x) = sum_b clamp(o_b + c_b - x, 0, c_b) tiles see x or more, and a
// search over x finds the rank's level, one sequence a lane. Beyond 64 sequences:
// in reverse order, so each sequence's longest come first. False: no such tile.
template <int ROWS>
__device__ __forceinline__ bool pick_tile(const PParams &p, int rank, int lane, int &b, int &index) {
  if (!p.start) {
    b = div_by(rank, p.by_seq_tiles);
    index = rank - b * p.by_seq_tiles.d;
    return true;
  }
  if (p.batch > 64) {
    // sequence b's tiles are numbered from start_b * group / rows + b on: at
    // least as many as it needs
    auto key = [&](int start, int seq) { return (int)((uint32_t)(start * p.group) / ROWS) + seq; };
    const int tile = p.tiles - 1 - rank;
    b = find_sequence(p, tile, lane, key);
    index = tile - key(row_start(p, b), b);
    return index >= 0;
  }
  int c = 0, o = 0;
  if (lane < p.batch) {
    const int n = max(row_start(p, lane + 1) - row_start(p, lane), 0);
    c = (n * p.group + ROWS - 1) / ROWS;
    const int len = max(0, min(ro(p.seq_lens)[lane], p.max_tokens));
    o = (int)min((int64_t)max(len - n, 0) * p.group / ROWS, (int64_t)1 << 24);
  }
  if (rank >= wave_sum(c)) return false;
  // count(lo) > rank >= count(hi) = above, hi the first power of two past all tiles
  int lo = 0, hi = 1, above = 0;
  while (__builtin_amdgcn_ballot_w64(c > 0 && o + c > hi)) hi *= 2;
  while (hi - lo > 1) {
    const int mid = lo + (hi - lo) / 2;
    const int n = wave_sum(min(max(o + c - mid, 0), c));
    if (n > rank) {
      lo = mid;
    } else {
      hi = mid;
      above = n;
    }
  }
  uint64_t m = __builtin_amdgcn_ballot_w64(c > 0 && o <= lo && lo < o + c);
  for (int k = rank - above; k > 0; --k) m &= m - 1;
  b = __builtin_ctzll(m | (1ull << 63));
  b = __builtin_amdgcn_readfirstlane(b);
  index = lo - __builtin_amdgcn_readlane(o, b);
  return true;
}

template <int KV, int SC, int D, int MAPS>
__global__ void __launch_bounds__((64 * kTileWaves<D, MAPS>))
    __attribute__((amdgpu_waves_per_eu(PGeo<KV, D, MAPS>::kWavesPerEU)))
paged_prefill_kernel(const PParams p) {
  using G = PGeo<KV, D, MAPS>;
  constexpr int W = G::W;
  __shared__ __attribute__((aligned(16))) uint8_t sm[2 * G::kBufBytes];
  constexpr bool kInt8 = KV == PA_KV_INT8;
  constexpr int kTileScales = 2 * MAPS * G::BN;  // of K's heads, then of V's
  __shared__ __attribute__((aligned(16))) float sm_sc[kInt8 ? 2 * kTileScales : 4];
  __shared__ int sm_wild;  // V holds an infinity or NaN in a masked tile

  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int h = lane >> 5;
  const int map = MAPS == 2 ? wave & 1 : 0;
  const int wave_row = kRowsPerWave * (wave / MAPS);

  // blockIdx = (split * tiles + tile) * units + unit: the units (kv heads) of the
  // same tokens run together, and with 8 of them each XCD keeps one head's K/V in
  // its L2. Row tiles go from those that see the most tokens on. Splits are
  // outermost: the later ones hold tokens of the longest sequences only, and a CU
  // that the round-robin gave always the same split would have all or no work
  // (24 sequences of 500-8,000 tokens in 4 splits 85.7 us, in 3 65.1).
  const uint32_t x1 = div_by(blockIdx.x, p.by_units);
  const int unit = blockIdx.x - x1 * p.units;
  const int split = div_by(x1, p.by_tiles);
  const int rank = x1 - (uint32_t)split * p.tiles;
  int b, index;
  if (!pick_tile<G::kRowTile>(p, rank, lane, b, index)) return;
  const RowTile rt = tile_at<G::kRowTile>(p, b, index);
  if (rt.row0 >= rt.rows) return;

  int lo = 0, hi = rt.hi;
  bool direct = true;  // the row tile is this workgroup's alone: no partials
  if (p.num_splits > 1) {
    const int chunk = split_tokens(p, rt.hi, split_units<G::kRowTile>(p, lane));
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
  const bool busy = rt.row0 + wave_row < rt.rows;  // the wave has rows; otherwise it only helps to load
  // the fewest tokens that a row of the wave sees
  const int least = rt.first + (int)div_by((uint32_t)min(rt.row0 + wave_row, rt.rows - 1), p.by_group) + 1;
  const int least_all = rt.first + (int)div_by((uint32_t)rt.row0, p.by_group) + 1;

  RowState<D, W> st;
  st.m = -INFINITY;
  st.l = 0.f;
  st.limit = 0.f;
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
    for (int i = 0; i < G::kIter; ++i) la.row[i] = (64 * G::kNW * i + (int)threadIdx.x) / G::kPPR;
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
    if (store_tile<KV, SC, D, MAPS>(sm, staged, la, col, lo + G::BN > least_all, sm_sc)) sm_wild = 1;
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
      if (busy) {
        const uint8_t *buf = sm + cur * G::kBufBytes;
        f32x16 s[G::BN / 32];
        scores_of<G::kKSteps, G::kKStride>(s, st.q, buf + k_lane);
        const float *scales = sm_sc + (kInt8 ? cur * kTileScales : 0);
        const bool masked = n0 + G::BN > least;
        if constexpr (kInt8)
          scale_scores<32, G::BN / 2>([&](int e, float k) { s[e / 16][e % 16] *= k; }, scales + map * G::BN, h);
        if (masked) {
          asm volatile("");  // a branch: as selects these would run on every tile
          mask(s, n0, lim, h);
        }
        rescale(st, top_score(s, p.qk_scale));
        accumulate<G::kVStride, kInt8 ? MAPS : 0>(st, s, buf + G::kKBytes, v_lane, p.qk_scale, scales + MAPS * G::BN, h);
      }
      if (more && store_tile<KV, SC, D, MAPS>(sm + (cur ^ 1) * G::kBufBytes, staged, la, col, n0 + 2 * G::BN > least_all,
                                              sm_sc + (kInt8 ? (cur ^ 1) * kTileScales : 0)))
        sm_wild = 1;
      __syncthreads();
      cur ^= 1;
    }
    if (!kInt8 && __builtin_expect(sm_wild, 0)) {
      // the masked tiles once more, with V as it is
      const int from = max(lo, max(least_all - 1, 0) / G::BN * G::BN);
      for (int n0 = from; n0 < hi; n0 += G::BN) {
        load_pages<KV, D, MAPS>(page, p, bt_row, n0, rt.len, wave);
        load(n0);
        store_tile<KV, SC, D, MAPS>(sm, staged, la, col, false, sm_sc);
        __syncthreads();
        if (busy && n0 + G::BN > least_all) add_wild<G::BN, G::kVStride>(st, sm + G::kKBytes, n0, lim, lane);
        __syncthreads();
      }
    }
  }

  const float l = half_sum(st.l);
  if constexpr (kInt8) {
#pragma unroll
    for (int d = 0; d < G::kDB; ++d) st.acc[d] *= st.limit;
  }
  auto element = [&](int e) { return st.acc[e / 16][e % 16]; };
  if (!direct) {
    if (live) store_partial<W, 32>(p, element, st.m, l, split, rt.token0 + token, head, lane);
    return;
  }
  // (a row that sees nothing is zeros; one whose visible scores are all -inf is 0 / 0)
  float inv = lim < 0 ? 0.f : 1.0f / l;
  // Results leave through LDS: lanes hold eight bytes of 32 different rows, and
  // stored so every 64 bytes of a row would be written in pieces.
  auto store_result = [&](float f, bool normed) {
    constexpr int kStride = W * 2 + 16, kLanes = W / 8, kRows = 64 / kLanes;
    static_assert(G::kNW / MAPS * 32 * kStride <= 2 * G::kBufBytes, "the rows fit the tiles' LDS");
    uint8_t *rows = sm + (wave / MAPS) * 32 * kStride;
    const float *norm = normed ? p.norm : nullptr;
#pragma unroll
    for (int e = 0; e < W / 2; e += 4) {
      const int d = 2 * e + 4 * h;
      f32x4 y = {element(e) * f, element(e + 1) * f, element(e + 2) * f, element(e + 3) * f};
      if (norm) y *= *reinterpret_cast<const f32x4 *>(norm + d);
      store4(rows + (lane & 31) * kStride + 2 * d, y.x, y.y, y.z, y.w, p.io_bf16);
    }
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
#pragma unroll
    for (int i = 0; i < 32 / kRows; ++i) {
      const int in_wave = i * kRows + lane / kLanes, at = rt.row0 + wave_row + in_wave;
      if (at < rt.rows) {
        const int tok = div_by((uint32_t)at, p.by_group), out_head = unit * p.group + (at - tok * p.group);
        const u32x4 x = *reinterpret_cast<const u32x4 *>(rows + in_wave * kStride + 16 * (lane % kLanes));
        *reinterpret_cast<u32x4 *>(p.out + 2 * ((int64_t)(rt.token0 + tok) * p.sot + (int64_t)out_head * p.soh) +
                                   16 * (lane % kLanes)) = x;
      }
    }
  };
  if constexpr (MAPS == 1) {
    store_result(inv, false);
  } else {
    // the second map's waves hand theirs over, as many registers at a time as LDS holds
    constexpr int kRegs = W / 2, kRounds = kRegs * G::kNW / 2 * 256 > 2 * G::kBufBytes ? 2 : 1, kPart = kRegs / kRounds;
    static_assert(kPart * G::kNW / 2 * 256 <= 2 * G::kBufBytes, "a part fits the tiles' LDS");
    float *other = reinterpret_cast<float *>(sm) + (wave / 2) * kPart * 64 + lane;
    if (map == 1) inv *= p.lam[(int64_t)(head / 2) * p.slam];
    float sq = 0.f;
#pragma unroll
    for (int part = 0; part < kRounds; ++part) {
      __syncthreads();  // every wave is done with the tiles, or with the part before
      if (map == 1) {
#pragma unroll
        for (int e = 0; e < kPart; ++e) other[e * 64] = element(part * kPart + e) * inv;
      }
      __syncthreads();
      if (map == 0) {
#pragma unroll
        for (int e = 0; e < kPart; ++e) {
          const int i = part * kPart + e;
          const float x = st.acc[i / 16][i % 16] * inv - other[e * 64];
          st.acc[i / 16][i % 16] = x;
          sq += x * x;
        }
      }
    }
    __syncthreads();
    if (map == 1) return;
    sq = half_sum(sq);
    const float f = p.norm ? __builtin_amdgcn_rsqf(sq * (1.0f / W) + p.norm_eps) * p.out_scale : 1.0f;
    store_result(f, true);
  }
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
  if (a->chunks < 0) return pa_fail(PA_ERR_INVALID, "chunks %d < 0", a->chunks);
  if (a->form < PA_FORM_TILES || a->form > PA_FORM_STREAMS16) return pa_fail(PA_ERR_INVALID, "form %d unknown", a->form);
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
  const int waves = a->form == PA_FORM_TILES && d * maps >= 128 && d < 256 ? 8 : kWaves;
  const int columns = a->form == PA_FORM_TILES ? kRowsPerWave * waves : a->form == PA_FORM_STREAMS ? 32 : 16;
  const int row_tile = columns / maps;
  const int seq_tiles = (group + row_tile - 1) / row_tile;
  const int64_t tiles = a->query_start_loc ? (int64_t)a->num_tokens * group / row_tile + a->batch
                                           : (int64_t)a->batch * seq_tiles;
  // a launch holds fewer than 2^32 threads (the merge: a wave an output row)
  if (tiles * units >= 2 * gib || tiles * units * a->num_splits * waves >= 4 * gib / 64 ||
      (a->num_splits > 1 && (int64_t)a->num_tokens * (a->num_q_heads / maps) >= 4 * gib / 64 - 4))
    return pa_fail(PA_ERR_UNSUPPORTED, "too many rows and splits for one launch: 2^26 waves at most");

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
  p.chunks = std::min(a->chunks, 1 << 30);
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
  p.by_tiles = make_div((uint32_t)std::max<int64_t>(tiles, 1));
  p.by_group = make_div(group);
  p.by_seq_tiles = make_div(seq_tiles);
  p.by_heads = make_div(a->num_q_heads / maps);
  *out = p;
  return PA_OK;
}

template <int KV, int SC, int D, int MAPS>
hipError_t launch(const PParams &p, hipStream_t st) {
  using G = PGeo<KV, D, MAPS>;
  hipLaunchKernelGGL((paged_prefill_kernel<KV, SC, D, MAPS>), dim3((uint32_t)(p.tiles * p.units * p.num_splits)),
                     dim3(64 * G::kNW), 0, st, p);
  if (p.num_splits > 1) launch_merge<G::W, MAPS, G::kRowTile>(p, st);
  return hipGetLastError();
}

template <int KV, int SC>
hipError_t launch_kv(const PParams &p, int d, int maps, hipStream_t st) {
  if (maps == 1) {
    switch (d) {
      case 32: return launch<KV, SC, 32, 1>(p, st);
      case 64: return launch<KV, SC, 64, 1>(p, st);
      case 128: return launch<KV, SC, 128, 1>(p, st);
      default: return launch<KV, SC, 256, 1>(p, st);
    }
  }
  switch (d) {
    case 32: return launch<KV, SC, 32, 2>(p, st);
    case 64: return launch<KV, SC, 64, 2>(p, st);
    default: return launch<KV, SC, 128, 2>(p, st);
  }
}

int attend(const pa_prefill_args *a, int maps, void *stream) {
  PParams p;
  const int rc = build(a, maps, &p);
  if (rc != PA_OK) return rc;
  if (p.batch == 0 || p.num_tokens == 0) return pa_ok();  // (the searches need a sequence)
  hipStream_t st = static_cast<hipStream_t>(stream);
  const int d = a->head_dim;
  hipError_t e;
  if (a->form != PA_FORM_TILES) e = launch_streams(p, a, maps, st);
  else if (a->kv_dtype == PA_KV_FP16) e = launch_kv<PA_KV_FP16, PA_SCALE_NONE>(p, d, maps, st);
  else if (a->kv_dtype == PA_KV_BF16) e = launch_kv<PA_KV_BF16, PA_SCALE_NONE>(p, d, maps, st);
  else if (a->kv_dtype == PA_KV_FP8_E5M2) e = launch_kv<PA_KV_FP8_E5M2, PA_SCALE_NONE>(p, d, maps, st);
  else if (a->scale_dtype == PA_SCALE_FP32) e = launch_kv<PA_KV_INT8, PA_SCALE_FP32>(p, d, maps, st);
  else e = launch_kv<PA_KV_INT8, PA_SCALE_FP16>(p, d, maps, st);
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
