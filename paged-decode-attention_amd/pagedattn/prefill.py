"""Attention of prompts over the paged cache, and differential attention (HIP).

`paged_prefill_hip` attends several new tokens of each sequence over the cache
that already holds them (write them with `reshape_and_cache` first): prompts,
chunks of prompts, a few speculative tokens. `paged_diff_prefill_hip` and
`paged_diff_decode_hip` are the differential forms, for several tokens and for
one. Launches go through the C ABI (include/pagedattn.h); there is no CPU path.
Split partials are allocated per call from torch's caching allocator, on the
current stream, so calls on different streams and captured graphs share nothing.
"""

from __future__ import annotations

import torch

from . import _abi
from .cache import PagedKVCache
from .hip_decode import _IO_CODE, _KV_CODE, _SCALE_CODE, _STORE_DTYPE, _cu_count, _launch

# Columns of a workgroup's score products, by form (csrc/paged_prefill.hip,
# csrc/paged_stream.hip): rows, a row being a new token and a head of its kv head's
# group; the differential forms take two columns a row, one for each map. Tiles
# have 256 where a cache row (of a pair, in the differential forms) has 128 elements
# or more, unless a head has 256.
_COLUMNS = {_abi.PA_FORM_TILES: 128, _abi.PA_FORM_STREAMS: 32, _abi.PA_FORM_STREAMS16: 16}
WIDE_TILE_COLUMNS = 256
# Workgroups that a CU holds at once, by form and elements of a cache row (2 elsewhere).
_PER_CU = {_abi.PA_FORM_TILES: {256: 1, 128: 1}, _abi.PA_FORM_STREAMS: {256: 1},
           _abi.PA_FORM_STREAMS16: {256: 2, 128: 4}}
# A split is a multiple of this many tokens; fewer than MIN_SPLIT_TOKENS are not
# worth a partial and its share of the merge.
MIN_SPLIT_TOKENS = 256
# How many times the average sequence's chunks the longest may take.
UNEVEN = {_abi.PA_FORM_TILES: 1, _abi.PA_FORM_STREAMS: 3, _abi.PA_FORM_STREAMS16: 3}
# Launches with less than this share of the chip's workgroups are split.
SPLIT_BELOW = 0.85


def _plan(rows: int, batch: int, units: int, longest: int, cus: int, width: int, maps: int) -> tuple[int, int]:
    """(form, num_splits) from shapes alone: `rows` (token, head) rows in all
    for each of `units` kv heads (pairs of them in the differential forms), cache rows
    of `width` elements. Sequences whose rows a stream's columns hold on average
    stream. Splits fill the chip (`_chunks`), and a sequence longer than the average may
    take more of them than its share."""
    form = _abi.PA_FORM_TILES
    for few in (_abi.PA_FORM_STREAMS16, _abi.PA_FORM_STREAMS):
        if rows * maps <= _COLUMNS[few] * batch:
            form = few
            break
    columns = _COLUMNS[form]
    if form == _abi.PA_FORM_TILES and width >= 128 and width // maps < 256:
        columns = WIDE_TILE_COLUMNS
    work = max(1, max(batch, rows * maps // columns) * units)
    slots = _PER_CU[form].get(width, 2) * cus
    splits = 1
    if work < SPLIT_BELOW * slots:
        uneven = min(batch, UNEVEN[form])
        splits = max(1, min(-(-slots // work) * uneven, -(-longest // MIN_SPLIT_TOKENS), _abi.PA_MAX_SPLITS))
    return form, splits


def _chunks(form: int, units: int, cus: int, width: int) -> int:
    """Chunks of a split launch for each unit; 0: every tile by itself. They fill 3/4 of
    the chip: a sequence's chunks are more than its share by half a one on average, and
    a few more than the chip holds take a round of their own (24 int8 sequences of up to
    8,000 tokens, 5 new: 0.6 67 us, 0.75 63, 0.8 76). (Tiles' chunks come longest first, which balances as well, and
    sizing them by the batch's lengths gave more partials: 12 prompts of 60 to 700
    tokens after up to 3,000, pairs of 64-element heads, 86 against 96 us.)"""
    return 0 if form == _abi.PA_FORM_TILES else max(1, _PER_CU[form].get(width, 2) * cus * 3 // (4 * units))


# Checked argument structs by the geometry they were checked for: shapes, strides,
# types and devices of every tensor and the call's numbers, nothing of a tensor's
# identity or address. A call of a known geometry copies its struct and sets the
# pointers (the C side checks every call again).
_CHECKED: dict[tuple, tuple] = {}
_CHECKED_MAX = 512
_copy_args = _abi.PaPrefillArgs.from_buffer_copy


def _attend(fn_name, maps, q, cache, start, out, sm_scale, num_splits, max_seq_len, lam=None, norm_weight=None,
            norm_eps=0.0, out_scale=1.0):
    """Check a call's tensors (once per geometry), fill pa_prefill_args and launch."""
    k, v, ks, vs, bt, sl = (cache.k_cache, cache.v_cache, cache.k_scale, cache.v_scale, cache.block_table,
                            cache.seq_lens)
    shape = cache.shape
    # (numbers by value: a tensor given as one would be a key by its identity)
    sm_scale = None if sm_scale is None else float(sm_scale)
    num_splits = None if num_splits is None else int(num_splits)
    # (the plan's unit, so a serving loop's growing length is not a geometry every step)
    longest = None if max_seq_len is None else max(0, -(-int(max_seq_len) // MIN_SPLIT_TOKENS)) * MIN_SPLIT_TOKENS
    norm_eps, out_scale = float(norm_eps), float(out_scale)
    key = (fn_name, q.shape, q.stride(), q.dtype, q.get_device(), k.shape, k.stride(), k.dtype, k.get_device(),
           v.shape, v.stride(), v.dtype, v.get_device(), bt.shape, bt.stride(), bt.dtype, bt.get_device(),
           sl.shape, sl.stride(), sl.dtype, sl.get_device(), cache.kv_dtype, cache.block_size, shape.num_q_heads,
           shape.num_kv_heads, shape.head_dim, sm_scale, num_splits, longest, norm_eps, out_scale)
    for t in (start, out, lam, norm_weight, ks, vs):
        key += (None,) if t is None else (t.shape, t.stride(), t.dtype, t.get_device())
    hit = _CHECKED.get(key)
    if hit is None:
        hit = _check(maps, q, cache, start, out, sm_scale, num_splits, longest, lam, norm_weight, norm_eps,
                     out_scale)
        if len(_CHECKED) >= _CHECKED_MAX:
            _CHECKED.clear()
        _CHECKED[key] = hit
    args, out_shape, part_out, part = hit
    if out is None:
        out = torch.empty(out_shape, dtype=q.dtype, device=q.device)
    if args is None:  # no rows
        return out
    a = _copy_args(args)
    a.q, a.k_cache, a.v_cache, a.out = q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr()
    a.block_table, a.seq_lens = bt.data_ptr(), sl.data_ptr()
    if start is not None:
        a.query_start_loc = start.data_ptr()
    if lam is not None:
        a.lam = lam.data_ptr()
        if norm_weight is not None:
            a.norm_weight = norm_weight.data_ptr()
    if cache.kv_dtype == "int8":
        a.k_scale, a.v_scale = ks.data_ptr(), vs.data_ptr()
    if part:
        partials = torch.empty((part,), dtype=torch.float32, device=q.device)
        a.part_out = partials.data_ptr()
        a.part_lse = a.part_out + part_out
    rc = _launch(q, getattr(_abi.load(), fn_name), a)
    if rc:
        _abi.check(rc, fn_name)
    return out


def _check(maps, q, cache, start, out, sm_scale, num_splits, longest, lam, norm_weight, norm_eps, out_scale):
    """(struct without pointers or None where there are no rows, the result's shape,
    bytes of part_out, floats of all partials) of a call, or the error of a wrong one."""
    if q.dim() != 3:
        raise ValueError(f"q {tuple(q.shape)} is not [tokens, heads, head_dim]")
    n, hq, d = q.shape
    shape, kv_dtype = cache.shape, cache.kv_dtype
    hkv = shape.num_kv_heads
    if kv_dtype not in _KV_CODE:
        raise NotImplementedError(f"kv_dtype {kv_dtype!r} is not supported by the HIP kernel")
    if q.dtype not in _IO_CODE:
        raise NotImplementedError(f"q dtype {q.dtype}: float16 or bfloat16")
    if hq != shape.num_q_heads or d != shape.head_dim:
        raise ValueError(f"q has {hq} heads of {d}, cache shape expects {shape.num_q_heads} of {shape.head_dim}")
    if hkv <= 0 or hq % hkv or hkv % maps:
        raise ValueError(f"{hq} query heads and {hkv} kv heads do not group" + (" in pairs" if maps == 2 else ""))
    k, v, bt, sl = cache.k_cache, cache.v_cache, cache.block_table, cache.seq_lens
    out_shape = (n, hq // maps, maps * d)
    if out is not None and (out.shape != out_shape or out.dtype != q.dtype):
        raise ValueError(f"out {out.dtype} {tuple(out.shape)} is not {q.dtype} {out_shape}")
    dev = q.get_device()
    for name, t in (("k_cache", k), ("v_cache", v), ("out", out), ("block_table", bt), ("seq_lens", sl),
                    ("query_start_loc", start), ("lam", lam), ("norm_weight", norm_weight)):
        if t is not None and t.get_device() != dev:
            raise ValueError(f"{name} is on {t.device}, q on {q.device}")
    if k.dtype != _STORE_DTYPE[kv_dtype] or v.dtype != k.dtype:
        raise ValueError(f"k/v cache dtype {k.dtype}/{v.dtype} does not match kv_dtype {kv_dtype}")
    kst, qst = k.stride(), q.stride()
    ost = (out_shape[1] * out_shape[2], out_shape[2], 1) if out is None else out.stride()
    if k.dim() != 4 or tuple(k.shape[1:]) != (cache.block_size, hkv, d) or v.shape != k.shape or v.stride() != kst:
        raise ValueError(f"k_cache {tuple(k.shape)} is not [NB, {cache.block_size}, {hkv}, {d}], or v_cache differs")
    if kst[3] != 1 or (qst[2] != 1 and n) or (ost[2] != 1 and n):
        raise ValueError("head_dim must be the contiguous (stride-1) dimension of q, out and the caches")
    if bt.dtype != torch.int32 or sl.dtype != torch.int32 or bt.dim() != 2 or sl.dim() != 1:
        raise ValueError("block_table [B, max_blocks] and seq_lens [B] must be int32")
    b, blocks = bt.shape
    if sl.shape[0] != b or (b > 1 and sl.stride(0) != 1) or (blocks > 1 and bt.stride(1) != 1):
        raise ValueError(f"block_table {tuple(bt.shape)} / seq_lens {tuple(sl.shape)}: [B, n] and [B], rows contiguous")
    if start is None:
        if n != b:
            raise ValueError(f"q has {n} rows for {b} sequences")
    elif start.dtype != torch.int32 or start.shape != (b + 1,) or (b and start.stride(0) != 1):
        raise ValueError(f"query_start_loc must be contiguous int32 [{b + 1}]")
    sst, scale_code = (0, 0), _abi.PA_SCALE_NONE
    if kv_dtype == "int8":
        ks, vs = cache.k_scale, cache.v_scale
        if ks is None or vs is None or ks.dtype not in _SCALE_CODE or vs.dtype != ks.dtype:
            raise ValueError("int8 cache needs float16 or float32 k_scale/v_scale")
        sst = ks.stride()
        if ks.shape != k.shape[:3] or vs.shape != ks.shape or vs.stride() != sst or sst[2] != 1:
            raise ValueError("k_scale/v_scale must be [NB, block_size, H_kv] with equal strides and a contiguous "
                             "head dimension")
        if ks.get_device() != dev or vs.get_device() != dev:
            raise ValueError("scales must live on q's device")
        scale_code = _SCALE_CODE[ks.dtype]
    lam_stride = 0
    if maps == 2:
        if lam.dtype != torch.float32 or lam.shape != (hq // 2,):
            raise ValueError(f"lam must be float32 [{hq // 2}], got {lam.dtype} {tuple(lam.shape)}")
        lam_stride = lam.stride(0)
        if norm_weight is not None and (norm_weight.dtype != torch.float32 or norm_weight.shape != (2 * d,)
                                        or norm_weight.stride(0) != 1):
            raise ValueError(f"norm_weight must be contiguous float32 [{2 * d}]")
    if not q.is_cuda:
        raise ValueError(f"q is on {q.device}: the HIP kernel needs GPU tensors")
    if n == 0 or b == 0:
        return None, out_shape, 0, 0
    capacity = blocks * cache.block_size
    longest = capacity if longest is None else min(longest, capacity)
    form, planned = _plan(n * (hq // hkv), b, hkv // maps, longest, _cu_count(q.device), maps * d, maps)
    chunks = 0
    if num_splits is None:
        num_splits, chunks = planned, _chunks(form, hkv // maps, _cu_count(q.device), maps * d)
    rows = num_splits * n * hq if num_splits > 1 else 0
    args = _abi.PaPrefillArgs()
    args.batch, args.num_tokens, args.num_q_heads, args.num_kv_heads, args.head_dim = b, n, hq, hkv, d
    args.block_size, args.num_blocks, args.max_blocks = cache.block_size, k.shape[0], blocks
    args.num_splits, args.chunks, args.form = num_splits, chunks, form
    args.stride_qt, args.stride_qh = qst[0], qst[1]
    args.stride_kn, args.stride_kt, args.stride_kh = kst[0], kst[1], kst[2]
    args.stride_sn, args.stride_st = sst[0], sst[1]
    args.stride_ot, args.stride_oh = ost[0], ost[1]
    args.stride_btb, args.stride_lam = bt.stride(0) if b > 1 else blocks, lam_stride
    args.kv_dtype, args.scale_dtype, args.io_dtype = _KV_CODE[kv_dtype], scale_code, _IO_CODE[q.dtype]
    args.sm_scale = d ** -0.5 if sm_scale is None else sm_scale
    args.norm_eps, args.out_scale = norm_eps, out_scale
    return args, out_shape, 4 * rows * maps * d, rows * (maps * d + 1)


def paged_prefill_hip(
    q: torch.Tensor,
    cache: PagedKVCache,
    query_start_loc: torch.Tensor,
    out: torch.Tensor | None = None,
    sm_scale: float | None = None,
    num_splits: int | None = None,
    max_seq_len: int | None = None,
) -> torch.Tensor:
    """Causal paged GQA attention of several new tokens of each sequence.

    q [tokens, Hq, D] fp16 or bf16 holds the sequences' new tokens packed one
    sequence after the other: sequence b's are rows query_start_loc[b] ..
    query_start_loc[b + 1] - 1 (int32 [B + 1] on the device, not decreasing).
    cache.seq_lens counts the tokens in the cache, the new ones included, so
    row i of n_b sees tokens 0 .. T_b - n_b + i. A row that sees none is zeros.
    Rows of no sequence (padding behind the last) are left as they are in `out`.

    `num_splits` cuts the longest sequence's tokens into at most that many chunks, and
    the others' into chunks no longer, joined by a second kernel. None plans them from
    the shapes alone, with no device sync: the kernel itself sizes the chunks by the
    lengths it finds, so that they fill the chip evenly. `max_seq_len` (a host int;
    None: what the block table can hold) is what that plans by. Results do not depend
    on either beyond rounding, and longer sequences are attended whole.
    """
    return _attend("pa_prefill", 1, q, cache, query_start_loc, out, sm_scale, num_splits, max_seq_len)


def paged_diff_prefill_hip(
    q: torch.Tensor,
    cache: PagedKVCache,
    query_start_loc: torch.Tensor,
    lam: torch.Tensor,
    out: torch.Tensor | None = None,
    norm_weight: torch.Tensor | None = None,
    norm_eps: float = 1e-5,
    out_scale: float = 1.0,
    sm_scale: float | None = None,
    num_splits: int | None = None,
    max_seq_len: int | None = None,
) -> torch.Tensor:
    """Differential attention of several new tokens of each sequence.

    Heads come in pairs: query heads 2i and 2i + 1 of q [tokens, Hq, D] are the
    two maps of output head i, kv heads 2j and 2j + 1 of the cache (j = i //
    group) the keys of the maps and the two halves of the value:
        out[:, i] = softmax(q_2i K_2j) V_j - lam[i] * softmax(q_2i+1 K_2j+1) V_j
    out is [tokens, Hq / 2, 2 D]. `lam` float32 [Hq / 2] (one for the layer:
    `lam.expand(Hq // 2)`). With `norm_weight` float32 [2 D] each head's row is
    normalised by its root mean square (plus norm_eps) and scaled by norm_weight
    * out_scale. Rows and the other arguments as in `paged_prefill_hip`.
    """
    return _attend("pa_diff_prefill", 2, q, cache, query_start_loc, out, sm_scale, num_splits, max_seq_len, lam,
                   norm_weight, norm_eps, out_scale)


def paged_diff_decode_hip(
    q: torch.Tensor,
    cache: PagedKVCache,
    lam: torch.Tensor,
    out: torch.Tensor | None = None,
    norm_weight: torch.Tensor | None = None,
    norm_eps: float = 1e-5,
    out_scale: float = 1.0,
    sm_scale: float | None = None,
    num_splits: int | None = None,
    max_seq_len: int | None = None,
) -> torch.Tensor:
    """Differential attention of one new token of each sequence: q [B, Hq, D] ->
    [B, Hq / 2, 2 D]. Arguments as in `paged_diff_prefill_hip`; a sequence of
    length 0 yields zeros."""
    return _attend("pa_diff_decode", 2, q, cache, None, out, sm_scale, num_splits, max_seq_len, lam, norm_weight,
                   norm_eps, out_scale)


__all__ = ["paged_prefill_hip", "paged_diff_prefill_hip", "paged_diff_decode_hip"]
