// A serving step's tables for MI355X (gfx950): block table, slot map, positions,
// lengths and start offsets from each row's new tokens, with the pages taken from
// (and, for finished rows, returned to) a stack of free pages on the device.
//
// With L_b tokens in the cache (0 for a finished row, whose pages are pushed
// first), n_b new ones and P tokens a page, row b takes the pages
//   ceil(L_b / P) .. ceil((L_b + n_b) / P) - 1
// from the top of the stack, rows in order, and its token i goes to slot
//   table[b, (L_b + i) / P] * P + (L_b + i) % P.
// Everything is a prefix sum over rows: pages pushed, tokens asked for, pages
// needed, tokens given. Rows that do not fit get nothing: a row that its own
// table row does not hold; from the first row on that max_tokens does not hold,
// every row that asks for tokens; from the first row on that the stack does not
// hold, every row that needs a page. The sums run over what was asked, so no row
// overtakes an earlier one, and no atomics: the same inputs give the same tables.
//
// One workgroup sums the rows, a chunk of its threads at a time. A row that moves
// few pages and gets few tokens is written by its own thread, which has all it needs
// in registers (the decode step: no search, three dependent loads in all); the
// others go on a list in LDS that the waves share, a row a wave, so a long prompt
// does not hold up a lane. With more than kSlotsInline tokens the slots are written
// by a second launch over the whole chip, a binary search of the offsets each. What
// bounds it is latency: the launch, the chain of loads, the prefix sums (three, by
// DPP inside a wave). As a graph's node, 64 rows of one new token 4.3 us (2.9 in the
// kernel; 7.3 with rows and slots in two launches and sums through LDS), 512 rows, 48
// of them prompts of 200 to 4,000 tokens, 13.6 (21.9).

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "launch_math.h"
#include "pa_errors.h"
#include "pagedattn.h"

namespace {

constexpr int kSlotsInline = 16384;
constexpr int kSlotThreads = 256;
constexpr int kSearchRows = 4096;  // offsets that the slots' launch holds in LDS
constexpr int kFew = 4;            // pages, tokens that a row's own thread writes

struct TParams {
  int32_t *table;
  const int32_t *lens;
  const int32_t *fresh;
  const uint8_t *finished;
  int32_t *stack;
  const int32_t *count;
  int32_t *lens_out;
  int32_t *count_out;
  int32_t *start;
  int64_t *slots;
  int64_t *positions;
  int32_t rows, blocks, page, stack_size, max_tokens;
  int64_t stride;
  Div by_page;
};

__device__ __forceinline__ int pages_of(const TParams &p, int tokens) {
  return (int)div_by((uint32_t)tokens + (uint32_t)p.page - 1u, p.by_page);
}

// x plus the value that DPP control CTRL hands the lanes of ROWS.
template <int CTRL, int ROWS>
__device__ __forceinline__ int64_t dpp_add(int64_t x) {
  const int lo = __builtin_amdgcn_update_dpp(0, (int)x, CTRL, ROWS, 0xf, false);
  const int hi = __builtin_amdgcn_update_dpp(0, (int)(x >> 32), CTRL, ROWS, 0xf, false);
  return x + (int64_t)(((uint64_t)(uint32_t)hi << 32) | (uint32_t)lo);
}

__device__ __forceinline__ int64_t lane_value(int64_t x, int lane) {
  const uint32_t lo = __builtin_amdgcn_readlane((int)x, lane), hi = __builtin_amdgcn_readlane((int)(x >> 32), lane);
  return (int64_t)((uint64_t)hi << 32 | lo);
}

// Exclusive prefix sums over the workgroup's threads; `total` gets the sum. Two
// 32-bit sums fit one value, the upper one's addends shifted.
template <int THREADS>
__device__ __forceinline__ int64_t block_scan(int64_t x, int64_t *wave_sums, int64_t &total) {
  constexpr int kWaves = THREADS / 64;
  static_assert(kWaves <= 16, "the waves' sums are added across a row of 16 lanes");
  int64_t s = x;
  s = dpp_add<0x111, 0xf>(s);  // row_shr:1
  s = dpp_add<0x112, 0xf>(s);
  s = dpp_add<0x114, 0xf>(s);
  s = dpp_add<0x118, 0xf>(s);
  s = dpp_add<0x142, 0xa>(s);  // row_bcast:15 into rows 1 and 3
  s = dpp_add<0x143, 0xc>(s);  // row_bcast:31 into rows 2 and 3
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  __syncthreads();  // (an earlier scan's sums have been read)
  if (lane == 63) wave_sums[wave] = s;
  __syncthreads();
  int64_t w = lane < kWaves ? wave_sums[lane] : 0;
  w = dpp_add<0x111, 0xf>(w);
  w = dpp_add<0x112, 0xf>(w);
  w = dpp_add<0x114, 0xf>(w);
  w = dpp_add<0x118, 0xf>(w);
  total = lane_value(w, kWaves - 1);
  return (wave > 0 ? lane_value(w, wave - 1) : 0) + s - x;
}

// The last of n ascending values (the first at or below x) that is at or below x.
template <typename PTR>
__device__ __forceinline__ int last_at_or_below(PTR v, int n, int x) {
  int lo = 0, len = n;
  while (len > 1) {
    const int half = len / 2;
    if (v[lo + half] <= x) {
      lo += half;
      len -= half;
    } else {
      len = half;
    }
  }
  return lo;
}

__device__ __forceinline__ void write_slot(const TParams &p, int64_t i, int page, int pos, int blk) {
  p.slots[i] = (int64_t)page * p.page + (pos - blk * p.page);
  if (p.positions) p.positions[i] = pos;
}

__device__ __forceinline__ void write_pad(const TParams &p, int i) {
  p.slots[i] = -1;
  if (p.positions) p.positions[i] = 0;
}

// A row that waves work on: its columns from `have` on take stack[from - 0, 1, ...]
// (finished rows: give theirs to stack[from + 0, 1, ...]), its tokens go to packed
// places from `begin` on.
struct Job {
  int32_t row, len, n, begin, have, need, from;
};

template <int THREADS, bool SLOTS>
__global__ void __launch_bounds__(THREADS) step_rows_kernel(const TParams p) {
  constexpr int kWaves = THREADS / 64;
  __shared__ int64_t sums[kWaves];
  __shared__ Job jobs[THREADS];
  __shared__ int job_count;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  int top = max(0, min(*p.count, p.stack_size));
  const int most = (int)min((int64_t)p.blocks * p.page, (int64_t)0x7fffffff);
  if (tid == 0) job_count = 0;  // (the scans' barriers come before its first use)

  if (p.finished) {
    for (int base = 0; base < p.rows; base += THREADS) {
      const int b = base + tid;
      int push = 0;
      if (b < p.rows && p.finished[b]) push = min(pages_of(p, min(max(p.lens[b], 0), most)), p.blocks);
      int64_t total;
      const int first = (int)block_scan<THREADS>(push, sums, total);
      if (push > 0) jobs[atomicAdd(&job_count, 1)] = Job{b, 0, 0, 0, 0, push, first};
      __syncthreads();
      const int count = job_count;
      for (int k = wave; k < count; k += kWaves) {
        const Job j = jobs[k];
        for (int c = lane; c < j.need; c += 64) {
          const int64_t to = (int64_t)top + j.from + c;
          if (to < p.stack_size) p.stack[to] = p.table[j.row * p.stride + c];
        }
      }
      __syncthreads();  // (also: what is pushed is seen by the pops below)
      if (tid == 0) job_count = 0;
      top = (int)min((int64_t)top + total, (int64_t)p.stack_size);
    }
  }

  int64_t asked = 0;                     // tokens asked for before this chunk
  int needed = 0, given = 0, taken = 0;  // pages needed, tokens given, pages taken before it
  for (int base = 0; base < p.rows; base += THREADS) {
    const int b = base + tid;
    int len = 0, n = 0, last = 0;
    if (b < p.rows) {
      len = p.finished && p.finished[b] ? 0 : max(p.lens[b], 0);
      n = max(p.fresh[b], 0);
      // the page that the row's next token may share with its last
      if constexpr (SLOTS) last = p.table[b * p.stride + min((int)div_by((uint32_t)min(len, most), p.by_page), p.blocks - 1)];
    }
    if ((int64_t)len + n > most) n = 0;
    int64_t total;
    const int64_t tokens_before = asked + block_scan<THREADS>(n, sums, total);
    asked += total;
    if (tokens_before + n > p.max_tokens) n = 0;
    const int have = pages_of(p, min(len, most));
    int need = pages_of(p, min(len, most) + n) - have;
    const int pages_before = needed + (int)block_scan<THREADS>(need, sums, total);
    needed += (int)total;
    if (need > 0 && pages_before + need > top) n = need = 0;
    const int64_t both = block_scan<THREADS>((int64_t)need << 32 | n, sums, total);
    const int begin = given + (int)both;
    const int from = top - 1 - taken - (int)(both >> 32);
    if (b < p.rows) {
      p.start[b] = begin;
      p.lens_out[b] = len + n;
      if (b == p.rows - 1) p.start[p.rows] = begin + n;
    }
    if (need > kFew || (SLOTS && n > kFew)) {
      jobs[atomicAdd(&job_count, 1)] = Job{b, len, n, begin, have, need, from};
    } else if (need > 0 || n > 0) {
      int page[kFew];
#pragma unroll
      for (int c = 0; c < kFew; ++c)
        if (c < need) page[c] = p.stack[from - c];
#pragma unroll
      for (int c = 0; c < kFew; ++c)
        if (c < need) p.table[b * p.stride + have + c] = page[c];
      if constexpr (SLOTS) {
#pragma unroll
        for (int i = 0; i < kFew; ++i)
          if (i < n) {
            const int pos = len + i, blk = (int)div_by((uint32_t)pos, p.by_page);
            int pg = last;
#pragma unroll
            for (int c = 0; c < kFew; ++c)
              if (blk == have + c) pg = page[c];
            write_slot(p, begin + i, pg, pos, blk);
          }
      }
    }
    __syncthreads();
    const int count = job_count;
    for (int k = wave; k < count; k += kWaves) {
      const Job j = jobs[k];
      int32_t *row = p.table + j.row * p.stride;
      for (int c = lane; c < j.need; c += 64) row[j.have + c] = p.stack[j.from - c];
      if constexpr (SLOTS) {
        for (int i = lane; i < j.n; i += 64) {
          const int pos = j.len + i, blk = (int)div_by((uint32_t)pos, p.by_page);
          write_slot(p, j.begin + i, blk < j.have ? row[blk] : p.stack[j.from - (blk - j.have)], pos, blk);
        }
      }
    }
    given += (int)total;
    taken += (int)(total >> 32);
    __syncthreads();
    if (tid == 0) job_count = 0;
  }
  if (tid == 0) {
    *p.count_out = top - taken;
    if (p.rows == 0) p.start[0] = 0;
  }
  if constexpr (SLOTS) {
    for (int i = given + tid; i < p.max_tokens; i += THREADS) write_pad(p, i);
  }
}

__global__ void __launch_bounds__(kSlotThreads) step_slots_kernel(const TParams p) {
  __shared__ int32_t starts[kSearchRows];
  const int i = blockIdx.x * kSlotThreads + threadIdx.x;
  const bool in_lds = p.rows <= kSearchRows;
  if (in_lds) {
    for (int b = threadIdx.x; b < p.rows; b += kSlotThreads) starts[b] = p.start[b];
    __syncthreads();
  }
  if (i >= p.max_tokens) return;
  if (i >= p.start[p.rows]) {
    write_pad(p, i);
    return;
  }
  const int b = in_lds ? last_at_or_below(starts, p.rows, i) : last_at_or_below(p.start, p.rows, i);
  const int begin = p.start[b];
  const int pos = p.lens_out[b] - (p.start[b + 1] - begin) + (i - begin);
  const int blk = (int)div_by((uint32_t)pos, p.by_page);
  write_slot(p, i, p.table[b * p.stride + blk], pos, blk);
}

}  // namespace

extern "C" int pa_step_tables(const pa_step_tables_args *a, void *stream) {
  if (a == nullptr) return pa_fail(PA_ERR_INVALID, "args is NULL");
  if (a->batch < 0 || a->max_tokens < 0 || a->free_capacity < 0)
    return pa_fail(PA_ERR_INVALID, "batch %d, max_tokens %d and free_capacity %d must not be negative", a->batch,
                   a->max_tokens, a->free_capacity);
  if (a->max_blocks <= 0 || a->block_size <= 0)
    return pa_fail(PA_ERR_INVALID, "max_blocks %d and block_size %d must be positive", a->max_blocks, a->block_size);
  if (!a->free_count || !a->free_count_out || !a->query_start_loc)
    return pa_fail(PA_ERR_INVALID, "free_count, free_count_out and query_start_loc must be non-NULL");
  if (a->batch > 0 && (!a->block_table || !a->seq_lens || !a->new_lens || !a->seq_lens_out))
    return pa_fail(PA_ERR_INVALID, "block_table, seq_lens, new_lens and seq_lens_out must be non-NULL");
  if (a->max_tokens > 0 && !a->slot_mapping) return pa_fail(PA_ERR_INVALID, "slot_mapping must be non-NULL");
  if (a->free_capacity > 0 && !a->free_pages) return pa_fail(PA_ERR_INVALID, "free_pages must be non-NULL");
  const void *words[] = {a->block_table, a->seq_lens, a->new_lens, a->free_pages, a->free_count,
                         a->seq_lens_out, a->free_count_out, a->query_start_loc};
  for (const void *w : words)
    if (!pa_aligned(w, 4)) return pa_fail(PA_ERR_INVALID, "int32 pointers must be 4-byte aligned");
  if (!pa_aligned(a->slot_mapping, 8) || !pa_aligned(a->positions, 8))
    return pa_fail(PA_ERR_INVALID, "slot_mapping and positions must be 8-byte aligned");
  if (a->stride_btb < a->max_blocks && a->batch > 1)
    return pa_fail(PA_ERR_INVALID, "stride_btb %lld is below max_blocks %d: rows overlap", (long long)a->stride_btb, a->max_blocks);
  const int64_t lim = int64_t(1) << 31;
  // (one page and one table row above the last token: sums of pages stay in 32 bits)
  if ((int64_t)a->max_blocks * a->block_size >= lim - a->block_size || (int64_t)a->batch * a->max_blocks >= lim ||
      a->batch >= (1 << 30) || a->max_tokens >= (1 << 30))
    return pa_fail(PA_ERR_UNSUPPORTED, "max_blocks * block_size and batch * max_blocks must be below 2^31, batch and max_tokens below 2^30");
  TParams p;
  p.table = a->block_table;
  p.lens = a->seq_lens;
  p.fresh = a->new_lens;
  p.finished = a->finished;
  p.stack = a->free_pages;
  p.count = a->free_count;
  p.lens_out = a->seq_lens_out;
  p.count_out = a->free_count_out;
  p.start = a->query_start_loc;
  p.slots = a->slot_mapping;
  p.positions = a->positions;
  p.rows = a->batch;
  p.blocks = a->max_blocks;
  p.page = a->block_size;
  p.stack_size = a->free_capacity;
  p.max_tokens = a->max_tokens;
  p.stride = a->stride_btb;
  p.by_page = make_div((uint32_t)a->block_size);
  hipStream_t st = static_cast<hipStream_t>(stream);
  // few rows: few waves to add up
  const bool small = p.rows <= 256, inlined = p.max_tokens <= kSlotsInline;
  if (small && inlined) hipLaunchKernelGGL((step_rows_kernel<256, true>), dim3(1), dim3(256), 0, st, p);
  else if (inlined) hipLaunchKernelGGL((step_rows_kernel<1024, true>), dim3(1), dim3(1024), 0, st, p);
  else if (small) hipLaunchKernelGGL((step_rows_kernel<256, false>), dim3(1), dim3(256), 0, st, p);
  else hipLaunchKernelGGL((step_rows_kernel<1024, false>), dim3(1), dim3(1024), 0, st, p);
  if (!inlined)
    hipLaunchKernelGGL(step_slots_kernel, dim3((p.max_tokens + kSlotThreads - 1) / kSlotThreads), dim3(kSlotThreads), 0, st, p);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return pa_fail(PA_ERR_HIP, "launch failed: %s", hipGetErrorString(e));
  return pa_ok();
}
