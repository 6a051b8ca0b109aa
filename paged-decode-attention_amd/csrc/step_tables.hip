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
// One workgroup sums the rows, 1,024 at a time, and moves the pages: page j of
// all that move belongs to the row whose range of the sums holds j (a binary
// search in LDS), so one long prompt does not hold up a lane. Slots are
// independent of each other: a second launch writes them over the whole chip, or,
// up to kSlotsInline of them, the same workgroup, which saves that launch.

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "launch_math.h"
#include "pa_errors.h"
#include "pagedattn.h"

namespace {

constexpr int kThreads = 1024;
constexpr int kWaves = kThreads / 64;
constexpr int kSlotsInline = 4096;
constexpr int kSlotThreads = 256;

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

// Exclusive prefix sums over the workgroup's threads; `total` gets the sum.
template <typename T>
__device__ __forceinline__ T block_scan(T x, T *wave_sums, T &total) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  T s = x;
#pragma unroll
  for (int o = 1; o < 64; o *= 2) {
    const T y = __shfl_up(s, o);
    if (lane >= o) s += y;
  }
  __syncthreads();  // (an earlier scan's sums have been read)
  if (lane == 63) wave_sums[wave] = s;
  __syncthreads();
  T before = 0;
  total = 0;
#pragma unroll
  for (int w = 0; w < kWaves; ++w) {
    const T t = wave_sums[w];
    if (w < wave) before += t;
    total += t;
  }
  return before + s - x;
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

// Slot and position of packed token i of row b.
__device__ __forceinline__ void write_slot(const TParams &p, int i, int b, int row_start, int row_end) {
  const int pos = p.lens_out[b] - (row_end - row_start) + (i - row_start);
  const int blk = (int)div_by((uint32_t)pos, p.by_page);
  p.slots[i] = (int64_t)p.table[b * p.stride + blk] * p.page + (pos - blk * p.page);
  if (p.positions) p.positions[i] = pos;
}

__device__ __forceinline__ void write_pad(const TParams &p, int i) {
  p.slots[i] = -1;
  if (p.positions) p.positions[i] = 0;
}

template <bool SLOTS>
__global__ void __launch_bounds__(kThreads) step_rows_kernel(const TParams p) {
  __shared__ int32_t sums[kWaves];
  __shared__ int64_t wide_sums[kWaves];
  __shared__ int32_t first[kThreads];  // this chunk's pages moved before row i
  __shared__ int32_t at[kThreads];     // and the first column that they go to
  const int tid = threadIdx.x;
  int top = max(0, min(*p.count, p.stack_size));
  const int most = (int)min((int64_t)p.blocks * p.page, (int64_t)0x7fffffff);

  if (p.finished) {
    for (int base = 0; base < p.rows; base += kThreads) {
      const int b = base + tid;
      int push = 0;
      if (b < p.rows && p.finished[b]) push = min(pages_of(p, min(max(p.lens[b], 0), most)), p.blocks);
      int total;
      first[tid] = block_scan(push, sums, total);
      __syncthreads();
      for (int j = tid; j < total; j += kThreads) {
        const int r = last_at_or_below(first, kThreads, j);
        const int64_t to = (int64_t)top + j;
        if (to < p.stack_size) p.stack[to] = p.table[(base + r) * p.stride + (j - first[r])];
      }
      top = (int)min((int64_t)top + total, (int64_t)p.stack_size);
      __syncthreads();
    }
  }

  int64_t asked = 0;          // tokens asked for before this chunk
  int needed = 0, given = 0, taken = 0;  // pages needed, tokens given, pages taken before it
  for (int base = 0; base < p.rows; base += kThreads) {
    const int b = base + tid;
    int len = 0, n = 0;
    if (b < p.rows) {
      len = p.finished && p.finished[b] ? 0 : max(p.lens[b], 0);
      n = max(p.fresh[b], 0);
    }
    if ((int64_t)len + n > most) n = 0;
    int64_t all;
    const int64_t tokens_before = asked + block_scan<int64_t>(n, wide_sums, all);
    asked += all;
    if (tokens_before + n > p.max_tokens) n = 0;
    const int have = pages_of(p, min(len, most));
    int need = pages_of(p, min(len, most) + n) - have;
    int total;
    const int pages_before = needed + block_scan(need, sums, total);
    needed += total;
    if (need > 0 && pages_before + need > top) n = need = 0;
    const int begin = given + block_scan(n, sums, total);
    given += total;
    if (b < p.rows) {
      p.start[b] = begin;
      p.lens_out[b] = len + n;
      if (b == p.rows - 1) p.start[p.rows] = begin + n;
    }
    first[tid] = block_scan(need, sums, total);
    at[tid] = have;
    __syncthreads();
    for (int j = tid; j < total; j += kThreads) {
      const int r = last_at_or_below(first, kThreads, j);
      p.table[(base + r) * p.stride + at[r] + (j - first[r])] = p.stack[top - 1 - taken - j];
    }
    taken += total;
    __syncthreads();
  }
  if (tid == 0) {
    *p.count_out = top - taken;
    if (p.rows == 0) p.start[0] = 0;
  }
  if constexpr (SLOTS) {
    // (the barrier above ends the writes of start, lens_out and table by this workgroup)
    for (int i = tid; i < p.max_tokens; i += kThreads) {
      if (i < given) {
        const int b = last_at_or_below(p.start, p.rows, i);
        write_slot(p, i, b, p.start[b], p.start[b + 1]);
      } else {
        write_pad(p, i);
      }
    }
  }
}

__global__ void __launch_bounds__(kSlotThreads) step_slots_kernel(const TParams p) {
  const int i = blockIdx.x * kSlotThreads + threadIdx.x;
  if (i >= p.max_tokens) return;
  if (i < p.start[p.rows]) {
    const int b = last_at_or_below(p.start, p.rows, i);
    write_slot(p, i, b, p.start[b], p.start[b + 1]);
  } else {
    write_pad(p, i);
  }
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
  if (p.max_tokens <= kSlotsInline) {
    hipLaunchKernelGGL((step_rows_kernel<true>), dim3(1), dim3(kThreads), 0, st, p);
  } else {
    hipLaunchKernelGGL((step_rows_kernel<false>), dim3(1), dim3(kThreads), 0, st, p);
    hipLaunchKernelGGL(step_slots_kernel, dim3((p.max_tokens + kSlotThreads - 1) / kSlotThreads), dim3(kSlotThreads), 0, st, p);
  }
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return pa_fail(PA_ERR_HIP, "launch failed: %s", hipGetErrorString(e));
  return pa_ok();
}
