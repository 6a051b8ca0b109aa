// Prompt and differential attention where a (sequence, kv head) has few rows: a few
// speculative tokens, or the one new token of a decode step.
//
// COLS (16 or 32) columns of the score products hold all rows of a row tile, or half
// as many (token, head) pairs with both maps: map 1 in the lower half of the
// columns, map 2 in the upper. The four waves of a workgroup share the rows and
// split the tokens: wave w takes the 32-token tiles w, w + 4, ... of the
// workgroup's range through LDS of its own, with no barrier until the end, where the
// four are joined as splits are.
//   S^T[tok, col] = K . Q^T   16 columns: v_mfma_f32_16x16x32_f16, 32 columns:
//   O^T[d, col] += V^T . P^T  v_mfma_f32_32x32x16_f16; a lane's column is its row
// The maps of a differential row differ in the half of the K row they meet: every
// column meets both halves, in sums of their own, and a lane keeps its map's.
//
// What bounds it is the stream of K and V. They take turns in a wave's registers and
// in its LDS slot: V is on its way during K's products and the softmax, the next
// tile's K during V's. Half the registers and LDS so hold twice the waves, which keeps
// as many bytes in flight as both at once and measured faster (160 int8 sequences of
// 100 to 8,000 tokens 57 -> 52 us).
// The loads are non-temporal: a step reads each byte once (64 sequences of 4,096
// tokens, pairs of 128-element heads, fp16: 203 us with plain loads, 180 with these).
// 16 columns where they hold the rows: the accumulators, the softmax and the
// products are half those of 32. That case now takes 164-176 us, 6.1-6.6 TB/s of K and
// V, 156 us at the best rate of a read of them here.
//
// Ragged batches: chunks sized by the batch's lengths, which the kernel finds, so that
// they fill the chip once (split_units in prefill_common.h; 160 int8 sequences of 100
// to 8,000 tokens 57 -> 49 us, 24 of up to 8,000 with 5 new tokens 74 -> 64).

#include "prefill_common.h"

namespace {

// For a lane of map 1, its value minus that of the same row's map 2, COLS / 2 lanes on.
template <int COLS>
__device__ __forceinline__ float minus_other_map(float x) {
  const uint32_t u = __float_as_uint(x);
  if constexpr (COLS == 32) {
    const auto two = __builtin_amdgcn_permlane16_swap(u, u, false, false);
    return __uint_as_float(two[0]) - __uint_as_float(two[1]);
  } else {
    // row_ror:8: the lane 8 on in the 16
    const int other = __builtin_amdgcn_update_dpp(0, (int)u, 0x128, 0xf, 0xf, false);
    return x - __int_as_float(other);
  }
}

template <int KV, int D, int MAPS, int COLS>
struct SGeo {
  static constexpr int W = D * MAPS;
  static constexpr int kElem = (KV == PA_KV_FP16 || KV == PA_KV_BF16) ? 2 : 1;
  static constexpr int kPieceBytes = W * kElem >= 64 ? 16 : 8;  // of a lane's load
  static constexpr int kPieceElems = kPieceBytes / kElem;
  static constexpr int kPieceWords = kPieceBytes / 4;
  static constexpr int kPPR = W / kPieceElems;     // pieces of a row: 4 .. 32
  static constexpr int kIter = 32 * kPPR / 64;     // loads of K or V of a tile
  // Rows padded so that 16 lanes reading 16 bytes of 16 rows (K), or the rows of a
  // transposed read (V: four of 64 bytes, or eight of 32), use all banks once.
  static constexpr int kKStride = W * 2 + 16;
  static constexpr int kVStride = COLS == 16 ? W * 2 + 32 : W == 32 ? 64 : W * 2 + 64;
  static constexpr int kSlot = 32 * (kKStride > kVStride ? kKStride : kVStride);  // LDS of a wave
  static constexpr int kRowTile = COLS / MAPS;
  static constexpr int kScores = COLS / 2;         // of a lane and tile
  static constexpr int kAcc = W * COLS / 64;       // accumulator floats of a lane
  static constexpr int kSteps = D * COLS / 512;    // score products of a map (16 or 32 elements each)
  static constexpr int kWavesPerEU = COLS == 16 ? (W == 256 ? 2 : 3) : W == 256 ? 1 : 2;
};

template <int COLS>
struct Block;  // a product's accumulators
template <>
struct Block<32> {
  typedef f32x16 type;
  static constexpr int kFloats = 16;
  static __device__ __forceinline__ f32x16 product(f16x8 a, f16x8 b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
  }
};
template <>
struct Block<16> {
  typedef f32x4 type;
  static constexpr int kFloats = 4;
  static __device__ __forceinline__ f32x4 product(f16x8 a, f16x8 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
  }
};

// K or V of a tile on its way to LDS.
template <int KV, int N, int WORDS>
struct Half {
  uint32_t w[N][WORDS];
  uint32_t scale[KV == PA_KV_INT8 ? N : 1];
};

__device__ __forceinline__ void sync_slot() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

template <int KV, int SC, int D, int MAPS, int COLS>
__global__ void __launch_bounds__(64 * kWaves)
    __attribute__((amdgpu_waves_per_eu(SGeo<KV, D, MAPS, COLS>::kWavesPerEU)))
paged_stream_kernel(const PParams p) {
  using G = SGeo<KV, D, MAPS, COLS>;
  using B = Block<COLS>;
  constexpr int W = G::W;
  constexpr int kGroups = 64 / COLS;  // lanes of a column
  constexpr int kAccBytes = (kWaves - 1) * G::kAcc * 64 * 4;
  constexpr int kBytes = kWaves * G::kSlot > kAccBytes ? kWaves * G::kSlot : kAccBytes;
  __shared__ __attribute__((aligned(16))) uint8_t sm[kBytes];
  __shared__ float sm_m[kWaves][COLS], sm_l[kWaves][COLS];
  constexpr bool kInt8 = KV == PA_KV_INT8;
  __shared__ __attribute__((aligned(16))) float sm_sc[kInt8 ? kWaves * 2 * MAPS * 32 : 4];

  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int col = lane % COLS, grp = lane / COLS;
  const int map = MAPS == 2 ? col / (COLS / 2) : 0;

  // blockIdx = (split * tiles + tile) * units + unit, as the form for many rows
  const uint32_t x1 = div_by(blockIdx.x, p.by_units);
  const int unit = blockIdx.x - x1 * p.units;
  const int split = div_by(x1, p.by_tiles);
  const int tile = x1 - (uint32_t)split * p.tiles;
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
  bool direct = true;  // the row tile is this workgroup's alone: no partials
  if (p.num_splits > 1) {
    const int chunk = split_tokens(p, rt.hi, split_units<G::kRowTile>(p, lane));
    if (split > 0 && (int64_t)split * chunk >= rt.hi) return;  // empty
    lo = split * chunk;
    hi = min(rt.hi, lo + chunk);
    direct = rt.hi <= chunk;
  }

  // this lane's row: its token, its head, the last token it sees
  const int row = rt.row0 + col % G::kRowTile;
  const bool live = row < rt.rows;
  const int r = min(row, rt.rows - 1);
  const int token = div_by((uint32_t)r, p.by_group);
  const int head = MAPS * (unit * p.group + (r - token * p.group)) + map;
  const int lim = rt.first + token;
  const int least = rt.first + (int)div_by((uint32_t)rt.row0, p.by_group) + 1;  // tokens that the first row sees

  // this lane's piece of a load: row (of 64 / kPPR), element
  const int row_in = lane / G::kPPR;
  const int ecol = lane % G::kPPR * G::kPieceElems;
  const uint32_t part = (uint32_t)ecol / D;  // the differential cache row's half
  const uint32_t off = row_in * p.skt + part * p.skh + ((uint32_t)ecol - part * D) * G::kElem;
  const uint32_t soff = row_in * p.sst + part * (SC == PA_SCALE_FP32 ? 4 : 2);
  const int64_t head_off = (int64_t)unit * MAPS * p.skh;
  const int64_t scale_off = (int64_t)unit * MAPS * (SC == PA_SCALE_FP32 ? 4 : 2);
  const ro_i32 *bt_row = ro(p.bt) + (int64_t)rt.b * p.sbtb;
  uint8_t *slot = sm + wave * G::kSlot;
  float *k_scales = sm_sc + (kInt8 ? wave * 2 * MAPS * 32 : 0), *v_scales = k_scales + (kInt8 ? MAPS * 32 : 0);

  // the pages of the tile at n0 (a multiple of 32: each 16-token half lies in one)
  auto pages = [&](int n0, int (&pg)[2]) {
#pragma unroll
    for (int u = 0; u < 2; ++u) pg[u] = bt_row[(uint32_t)min(n0 + 16 * u, rt.len - 1) >> p.log2_page];
  };
  typedef Half<KV, G::kIter, G::kPieceWords> HalfTile;
  HalfTile t;
  // rows at or past the sequence's end read as zeros
  auto load = [&](const uint8_t *base, const uint8_t *sbase, int n0, const int (&pg)[2]) {
#pragma unroll
    for (int i = 0; i < G::kIter; ++i) {
      const int r0 = i * (64 / G::kPPR);  // first row of the load
      const uint32_t blk = (uint32_t)min(max(pg[r0 / 16], 0), p.num_blocks - 1);
      const uint32_t in_page = (uint32_t)(n0 + r0) & ((1u << p.log2_page) - 1u);
      const bool inside = n0 + r0 + row_in < rt.len;
      load_piece<kLoadNT>(t.w[i], page_rsrc(base + head_off + (uint64_t)blk * p.skn + in_page * p.skt, kRsrcBytes),
                          inside ? off : kOutside);
      if constexpr (KV == PA_KV_INT8)
        t.scale[i] = load_scale<SC>(page_rsrc(sbase + scale_off + (uint64_t)blk * p.ssn + in_page * p.sst, kRsrcBytes),
                                    inside ? soff : kOutside);
    }
  };
  // into the wave's slot; with `tame`, infinities and NaN become zeros, and the
  // result tells whether this lane had one
  auto store = [&](int stride, bool tame, float *scales) {
    bool wild = false;
#pragma unroll
    for (int i = 0; i < G::kIter; ++i) {
      constexpr int kHalves = G::kPieceElems / 2;
      uint32_t x[kHalves];
      to_halves<KV>(x, t.w[i]);
      if (!kInt8 && tame) {
#pragma unroll
        for (int w = 0; w < kHalves; ++w) wild |= tame_word(x[w]);
      }
      uint8_t *d = slot + (i * (64 / G::kPPR) + row_in) * stride + ecol * 2;
#pragma unroll
      for (int w = 0; w < kHalves; w += 4) *reinterpret_cast<u32x4 *>(d + 4 * w) = u32x4{x[w], x[w + 1], x[w + 2], x[w + 3]};
      if constexpr (kInt8) {
        const float sc = scale_value<SC>(t.scale[i]);
        if (ecol % D == 0) scales[part * 32 + i * (64 / G::kPPR) + row_in] = scales == v_scales ? finite_scale(sc) : sc;
      }
    }
    return wild;
  };

  constexpr int kBlocks = G::kAcc / B::kFloats;  // of the value's elements
  typename B::type acc[kBlocks] = {};
  auto element = [&](int e) -> float { return acc[e / B::kFloats][e % B::kFloats]; };
  float m = -INFINITY;  // running maximum - kTopLog2 (log2 domain)
  float l = 0.f;        // sum over this lane's tokens
  float limit = 0.f;    // int8: the accumulators' unit (raise_limit)
  f16x8 q[G::kSteps];
  bool wild = false;
  const int n_first = lo + 32 * wave;
  if (n_first < hi) {
    int pg[2];
    pages(n_first, pg);
    load(p.k, p.ks, n_first, pg);
    const uint16_t *qrow = reinterpret_cast<const uint16_t *>(p.q) + (int64_t)(rt.token0 + token) * p.sqt +
                           (int64_t)head * p.sqh + 8 * grp;
#pragma unroll
    for (int ks = 0; ks < G::kSteps; ++ks) {
      const u32x4 w = *reinterpret_cast<const u32x4 *>(qrow + 8 * kGroups * ks);
      q[ks] = p.io_bf16 ? bf16x8_to_f16x8(w) : __builtin_bit_cast(f16x8, w);
    }
    store(G::kKStride, false, k_scales);
    load(p.v, p.vs, n_first, pg);
    pages(n_first + 32 * kWaves, pg);
    const uint8_t *k_lane = slot + col * G::kKStride + 16 * grp;
    // V: 16 lanes take four rows (4 * group on) of 16 columns
    const uint32_t v_lane = (4 * grp + ((lane & 15) >> 2)) * G::kVStride + (COLS == 32 ? 32 * ((lane >> 4) & 1) : 0) +
                            8 * (lane & 3);

    for (int n0 = n_first; n0 < hi; n0 += 32 * kWaves) {
      const bool masked = n0 + 32 > least;
      const int next = n0 + 32 * kWaves;
      sync_slot();
      float s[G::kScores];
#pragma unroll
      for (int u = 0; u < 32 / COLS; ++u) {
        typename B::type one = {}, two = {};
#pragma unroll
        for (int ks = 0; ks < G::kSteps; ++ks) {
          const uint8_t *a = k_lane + COLS * u * G::kKStride + 16 * kGroups * ks;
          one = B::product(*reinterpret_cast<const f16x8 *>(a), q[ks], one);
          if constexpr (MAPS == 2) two = B::product(*reinterpret_cast<const f16x8 *>(a + 2 * D), q[ks], two);
        }
#pragma unroll
        for (int i = 0; i < B::kFloats; ++i) s[B::kFloats * u + i] = MAPS == 2 && map == 1 ? two[i] : one[i];
      }
      if constexpr (kInt8) scale_scores<COLS, G::kScores>([&](int e, float k) { s[e] *= k; }, k_scales + 32 * map, grp);
      if (masked) {
        asm volatile("");  // a branch: as selects these would run on every tile
#pragma unroll
        for (int e = 0; e < G::kScores; ++e)
          if (n0 + score_token<COLS>(e, grp) > lim) s[e] = -INFINITY;
      }
      float top = s[0];
#pragma unroll
      for (int e = 1; e < G::kScores; ++e) top = fmaxf(top, s[e]);
      top = column_max<COLS>(top) * p.qk_scale;
      const bool need = top > m + (kTopLog2 + kRescaleLog2);
      if (__builtin_expect(__builtin_amdgcn_ballot_w64(need) != 0, 0)) {
        const float m_new = need ? top - kTopLog2 : m;
        const float alpha = need ? __builtin_amdgcn_exp2f(m - m_new) : 1.0f;
        l *= alpha;
#pragma unroll
        for (int d = 0; d < G::kAcc / B::kFloats; ++d) acc[d] *= alpha;
        m = m_new;
      }
      // (a row that has seen nothing yet: every score is -inf and P is 0)
      const float base = m == -INFINITY ? 0.f : m;
      float sum[2] = {0.f, 0.f};
#pragma unroll
      for (int e = 0; e < G::kScores; ++e) {
        s[e] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[e], p.qk_scale, -base));
        sum[e & 1] += s[e];
      }
      l += sum[0] + sum[1];
      sync_slot();
      wild |= store(G::kVStride, masked, v_scales);
      sync_slot();
      if (next < hi) load(p.k, p.ks, next, pg);
      // P as product operands; int8: by head of the value row, times V's scales.
      // Differential rows, whose difference can be far smaller than its terms, take P as
      // two fp16 values, cut to 11 bits and what that leaves: the stream has time for
      // the second product, and P's rounding stays out of the result.
      constexpr int kHeads = kInt8 ? MAPS : 1;
      constexpr bool kTwice = MAPS == 2;
      uint32_t cut[kHeads][G::kScores / 2], left[kHeads][G::kScores / 2];
      float inv = 1.f;
      if constexpr (kInt8) {
        float top = 0.f;
#pragma unroll
        for (int part = 0; part < kHeads; ++part)
#pragma unroll
          for (int e = 0; e < G::kScores; e += 4) {
            const f32x4 v4 = *reinterpret_cast<const f32x4 *>(v_scales + 32 * part + score_token<COLS>(e, grp));
#pragma unroll
            for (int j = 0; j < 4; ++j) top = fmaxf(top, fabsf(s[e + j] * v4[j]));
          }
        bool any;
        const float f = raise_limit<COLS>(limit, top, any);
        if (__builtin_expect(any, 0)) {
#pragma unroll
          for (int d = 0; d < kBlocks; ++d) acc[d] *= f;
        }
        inv = inverse_limit(limit);
      }
#pragma unroll
      for (int part = 0; part < kHeads; ++part)
#pragma unroll
        for (int e = 0; e < G::kScores; e += 2) {
          float a = s[e], c = s[e + 1];
          if constexpr (kInt8) {
            const float *at = v_scales + 32 * part + score_token<COLS>(e, grp);
            a = a * at[0] * inv;  // (in this order: 0 times the largest scale is 0)
            c = c * at[1] * inv;
          }
          if constexpr (kTwice) {
            cut[part][e / 2] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_pkrtz(a, c));
            const f16x2 h = __builtin_bit_cast(f16x2, cut[part][e / 2]);
            const f16x2 r = {(_Float16)(a - (float)h[0]), (_Float16)(c - (float)h[1])};
            left[part][e / 2] = __builtin_bit_cast(uint32_t, r);
          } else {
            const f16x2 h = {(_Float16)a, (_Float16)c};
            cut[part][e / 2] = __builtin_bit_cast(uint32_t, h);
          }
        }
#pragma unroll
      for (int kb = 0; kb < G::kScores / 8; ++kb) {
        f16x8 pop[kHeads], rest[kHeads];
#pragma unroll
        for (int part = 0; part < kHeads; ++part) {
          pop[part] = as_f16x8(cut[part][4 * kb], cut[part][4 * kb + 1], cut[part][4 * kb + 2], cut[part][4 * kb + 3]);
          if constexpr (kTwice)
            rest[part] = as_f16x8(left[part][4 * kb], left[part][4 * kb + 1], left[part][4 * kb + 2], left[part][4 * kb + 3]);
        }
        // 32 columns: tokens 16 kb + 8 (j / 4) + 4 grp + j % 4; 16: 16 (j / 4) + 4 grp + j % 4
#pragma unroll
        for (int d = 0; d < kBlocks; ++d) {
          const f16x8 v = read_columns(slot + 16 * kb * G::kVStride + 2 * COLS * d + v_lane, 256 / COLS * G::kVStride);
          acc[d] = B::product(v, pop[d * kHeads / kBlocks], acc[d]);
          if constexpr (kTwice) acc[d] = B::product(v, rest[d * kHeads / kBlocks], acc[d]);
        }
      }
      sync_slot();
      if (next < hi) {
        store(G::kKStride, false, k_scales);
        load(p.v, p.vs, next, pg);
        pages(next + 32 * kWaves, pg);
      }
    }
    if (!kInt8 && __builtin_expect(__builtin_amdgcn_ballot_w64(wild) != 0, 0)) {
      // V's infinities and NaN in masked tiles, added to the rows that see them
      for (int n0 = n_first; n0 < hi; n0 += 32 * kWaves) {
        if (n0 + 32 <= least) continue;
        pages(n0, pg);
        load(p.v, p.vs, n0, pg);
        store(G::kVStride, false, v_scales);
        sync_slot();
        for (int t1 = 0; t1 < 32; ++t1) {
          const uint8_t *vrow = slot + t1 * G::kVStride + 8 * grp;
#pragma unroll
          for (int e = 0; e < G::kAcc; e += 4) {
            const u32x2 x = *reinterpret_cast<const u32x2 *>(vrow + 2 * (64 / COLS) * e);
            if (n0 + t1 <= lim && (has_wild(x.x) || has_wild(x.y))) {
#pragma unroll
              for (int j = 0; j < 4; ++j) {
                const uint32_t bits = j & 1 ? x[j / 2] >> 16 : x[j / 2] & 0xffffu;
                if ((bits & 0x7c00u) == 0x7c00u)
                  acc[(e + j) / B::kFloats][(e + j) % B::kFloats] += (float)__builtin_bit_cast(_Float16, (uint16_t)bits);
              }
            }
          }
        }
        sync_slot();
      }
    }
  }

  if constexpr (kInt8) {
#pragma unroll
    for (int d = 0; d < kBlocks; ++d) acc[d] *= limit;
  }
  // join the waves
  const float lw = column_sum<COLS>(l);
  if (grp == 0) {
    sm_m[wave][col] = m;
    sm_l[wave][col] = lw;
  }
  __syncthreads();  // (and every wave is done with its slot)
  float all_m = -INFINITY;
#pragma unroll
  for (int w = 0; w < kWaves; ++w) all_m = fmaxf(all_m, sm_m[w][col]);
  float all_l = 0.f;
#pragma unroll
  for (int w = 0; w < kWaves; ++w) {
    const float mw = sm_m[w][col];
    // (a wave that saw nothing of the row has a sum of zero)
    all_l += mw == -INFINITY ? sm_l[w][col] : sm_l[w][col] * __builtin_amdgcn_exp2f(mw - all_m);
  }
  const float f = m == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(m - all_m);
  float *others = reinterpret_cast<float *>(sm);
  if (wave > 0) {
#pragma unroll
    for (int e = 0; e < G::kAcc; ++e) others[((wave - 1) * G::kAcc + e) * 64 + lane] = element(e) * f;
  }
  __syncthreads();
  if (wave > 0) return;
#pragma unroll
  for (int e = 0; e < G::kAcc; ++e) {
    float a = element(e) * f;
#pragma unroll
    for (int w = 1; w < kWaves; ++w) a += others[((w - 1) * G::kAcc + e) * 64 + lane];
    acc[e / B::kFloats][e % B::kFloats] = a;
  }
  if (!direct) {
    if (live) store_partial<W, COLS>(p, element, all_m, all_l, split, rt.token0 + token, head, lane);
    return;
  }
  // (a row that sees nothing is zeros; one whose visible scores are all -inf is 0 / 0)
  float inv = lim < 0 ? 0.f : 1.0f / all_l;
  if constexpr (MAPS == 1) {
    if (live) store_rows<W, COLS>(p, element, inv, false, rt.token0 + token, head, lane);
  } else {
    if (map == 1) inv *= p.lam[(int64_t)(head / 2) * p.slam];
    float sq = 0.f;
#pragma unroll
    for (int e = 0; e < G::kAcc; ++e) {
      const float y = minus_other_map<COLS>(element(e) * inv);
      acc[e / B::kFloats][e % B::kFloats] = y;
      sq += y * y;
    }
    sq = column_sum<COLS>(sq);
    if (live && map == 0) {
      const float scale = p.norm ? __builtin_amdgcn_rsqf(sq * (1.0f / W) + p.norm_eps) * p.out_scale : 1.0f;
      store_rows<W, COLS>(p, element, scale, true, rt.token0 + token, head / 2, lane);
    }
  }
}

template <int KV, int SC, int D, int MAPS, int COLS>
hipError_t launch_cols(const PParams &p, hipStream_t st) {
  using G = SGeo<KV, D, MAPS, COLS>;
  hipLaunchKernelGGL((paged_stream_kernel<KV, SC, D, MAPS, COLS>), dim3((uint32_t)(p.tiles * p.units * p.num_splits)),
                     dim3(64 * kWaves), 0, st, p);
  if (p.num_splits > 1) launch_merge<G::W, MAPS, G::kRowTile>(p, st);
  return hipGetLastError();
}

template <int KV, int SC, int D, int MAPS>
hipError_t launch(const PParams &p, int form, hipStream_t st) {
  return form == PA_FORM_STREAMS16 ? launch_cols<KV, SC, D, MAPS, 16>(p, st) : launch_cols<KV, SC, D, MAPS, 32>(p, st);
}

template <int KV, int SC>
hipError_t launch_kv(const PParams &p, int d, int maps, int form, hipStream_t st) {
  if (maps == 1) {
    switch (d) {
      case 32: return launch<KV, SC, 32, 1>(p, form, st);
      case 64: return launch<KV, SC, 64, 1>(p, form, st);
      case 128: return launch<KV, SC, 128, 1>(p, form, st);
      default: return launch<KV, SC, 256, 1>(p, form, st);
    }
  }
  switch (d) {
    case 32: return launch<KV, SC, 32, 2>(p, form, st);
    case 64: return launch<KV, SC, 64, 2>(p, form, st);
    default: return launch<KV, SC, 128, 2>(p, form, st);
  }
}

}  // namespace

PA_HIDDEN hipError_t launch_streams(const PParams &p, const pa_prefill_args *a, int maps, hipStream_t st) {
  const int d = a->head_dim, form = a->form;
  if (a->kv_dtype == PA_KV_FP16) return launch_kv<PA_KV_FP16, PA_SCALE_NONE>(p, d, maps, form, st);
  if (a->kv_dtype == PA_KV_BF16) return launch_kv<PA_KV_BF16, PA_SCALE_NONE>(p, d, maps, form, st);
  if (a->kv_dtype == PA_KV_FP8_E5M2) return launch_kv<PA_KV_FP8_E5M2, PA_SCALE_NONE>(p, d, maps, form, st);
  if (a->scale_dtype == PA_SCALE_FP32) return launch_kv<PA_KV_INT8, PA_SCALE_FP32>(p, d, maps, form, st);
  return launch_kv<PA_KV_INT8, PA_SCALE_FP16>(p, d, maps, form, st);
}
