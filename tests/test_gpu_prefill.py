"""Prompt attention over the paged cache against the float64 oracle, on the GPU."""

from __future__ import annotations

import dataclasses

import pytest
import torch

import prompt_oracle as po
from pagedattn import (LLAMA3_8B, MHA_DEBUG, QWEN25_05B, ModelShape, _abi, allocate, paged_decode_hip,
                       paged_prefill_hip, prefill)

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True, params=["planned", "tiles", "streams", "streams16"])
def form(request, monkeypatch):
    """Every test as the plan has it, and in the form for many rows and the two for few."""
    if request.param != "planned":
        plan = prefill._plan
        code = {"tiles": _abi.PA_FORM_TILES, "streams": _abi.PA_FORM_STREAMS,
                "streams16": _abi.PA_FORM_STREAMS16}[request.param]
        monkeypatch.setattr(prefill, "_plan", lambda *a: (code, plan(*a)[1]))
    monkeypatch.setattr(prefill, "_CHECKED", {})  # (what is kept there has its form)
    return request.param

WIDE = ModelShape(4, 1, 256, "wide")
THIN = ModelShape(6, 2, 32, "thin")
MQA = ModelShape(71, 1, 64, "mqa")
SEVENTEEN = ModelShape(34, 2, 64, "g17")


def packed(new):
    start = [0]
    for n in new:
        start.append(start[-1] + n)
    return start


def case(shape, new, total, kv="fp16", sdt=torch.float16, io=torch.float16, page=16, seed=0, pad=0):
    """q (with `pad` more rows behind the last sequence), cache, offsets."""
    c = allocate(shape, len(new), total, block_size=page, kv_dtype=kv, seed=seed, scale_dtype=sdt, device="cuda",
                 slack_blocks=3)
    g = torch.Generator().manual_seed(100 + seed)
    start = packed(new)
    q = torch.randn((start[-1] + pad, shape.num_q_heads, shape.head_dim), generator=g).to(io).cuda()
    size = torch.linspace(0.5, 2.5, shape.num_q_heads)[None, :, None].to(io).cuda()
    return q * size, c, start


def offsets(start):
    return torch.tensor(start, dtype=torch.int32, device="cuda")


def check(q, c, start, **kw):
    print(f"{c.shape.name} {c.kv_dtype} page {c.block_size} start {start[:8]} lens {c.seq_lens.tolist()[:8]} {kw}",
          flush=True)
    got = paged_prefill_hip(q, c, offsets(start), **kw)
    torch.cuda.synchronize()
    want, bound = po.attend(q, c, start, sm_scale=kw.get("sm_scale"))
    share = po.worst(got[:start[-1]], want[:start[-1]], bound[:start[-1]])
    assert share < 1, share
    return got


KV = [("fp16", torch.float16), ("bf16", torch.float16), ("fp8_e5m2", torch.float16), ("int8", torch.float16),
      ("int8", torch.float32)]


@pytest.mark.parametrize("kv,sdt", KV, ids=["fp16", "bf16", "fp8", "int8h", "int8s"])
@pytest.mark.parametrize("shape", [LLAMA3_8B, QWEN25_05B, MHA_DEBUG, WIDE, THIN], ids=lambda s: s.name)
def test_ragged_prompts(shape, kv, sdt):
    """Whole prompts and chunks, one token to past two row tiles, in one launch."""
    new, total = [1, 33, 64, 7], [1, 33, 150, 100]
    io = torch.bfloat16 if kv == "bf16" else torch.float16
    q, c, start = case(shape, new, total, kv, sdt, io, seed=1)
    check(q, c, start)


@pytest.mark.parametrize("page", [16, 32, 64, 128, 256])
@pytest.mark.parametrize("kv,sdt", [KV[0], KV[4]], ids=["fp16", "int8s"])
def test_pages(page, kv, sdt):
    """Pages that end inside a tile, and tiles that end inside a page."""
    q, c, start = case(QWEN25_05B, [17, 5, 40], [17, 261, 333], kv, sdt, page=page, seed=2)
    check(q, c, start)


@pytest.mark.parametrize("shape", [MQA, SEVENTEEN, ModelShape(1, 1, 128, "one"), ModelShape(16, 16, 64, "mha")],
                         ids=lambda s: s.name)
def test_groups(shape):
    """Groups that do not divide the row tile, wider than it, and of one head."""
    q, c, start = case(shape, [3, 19, 2], [3, 70, 90], seed=3)
    check(q, c, start)


@pytest.mark.parametrize("io", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("scale", [None, 0.03])
def test_io_types_and_scale(io, scale):
    q, c, start = case(LLAMA3_8B, [9, 20], [40, 20], "fp8_e5m2", io=io, seed=4)
    check(q, c, start, sm_scale=scale)


def test_rows_that_see_nothing():
    """A sequence with fewer tokens in all than new ones, one with none, and one without new tokens."""
    q, c, start = case(LLAMA3_8B, [12, 5, 0, 3, 1], [4, 0, 50, 30, 0], seed=5)
    for splits in (1, 3):
        got = check(q, c, start, num_splits=splits)
        assert bool((got[:8] == 0).all()) and bool((got[12:17] == 0).all()) and bool((got[-1] == 0).all())


def test_rows_of_no_sequence_are_left():
    q, c, start = case(LLAMA3_8B, [5, 8], [30, 8], seed=6, pad=11)
    for splits in (1, 4):
        out = torch.full_like(q, 7.0)
        check(q, c, start, out=out, num_splits=splits)
        assert bool((out[start[-1]:] == 7.0).all())
    shifted = [3, 8, 16]  # nor do the first three rows belong to one
    out = torch.full_like(q, 7.0)
    paged_prefill_hip(q, c, offsets(shifted), out=out)
    want, bound = po.attend(q, c, shifted)
    assert bool((out[:3] == 7.0).all()) and po.worst(out[3:16], want[3:16], bound[3:16]) < 1


@pytest.mark.parametrize("splits", [1, 2, 3, 7, 40, None])
@pytest.mark.parametrize("longest", [None, 500, 1500, 5000])
@pytest.mark.parametrize("shape", [LLAMA3_8B, QWEN25_05B, WIDE], ids=lambda s: s.name)
def test_splits(shape, splits, longest):
    """Few rows over long sequences, more splits than tiles among them; the longest length given or
    not, right or wrong."""
    q, c, start = case(shape, [2, 5, 1], [1500, 3, 64], "int8", torch.float32, seed=7)
    check(q, c, start, num_splits=splits, max_seq_len=longest)


@pytest.mark.parametrize("batch", [2, 9, 70])
@pytest.mark.parametrize("long", [900, 5000])
def test_ragged_splits(batch, long):
    """Planned splits, sized by the lengths that the launch finds: one long sequence among short and
    empty ones, then another as long, all with the same plan."""
    total = [long if i == 1 else 17 * (i % 6) for i in range(batch)]
    new = [min(1 + i % 3, n) for i, n in enumerate(total)]
    q, c, start = case(QWEN25_05B, new, total, seed=23)
    check(q, c, start, max_seq_len=long)
    c.seq_lens[1] = long // 3
    check(q, c, start, max_seq_len=long)
    check(q, c, start, max_seq_len=300)  # shorter than the longest: attended whole all the same


@pytest.mark.parametrize("batch", [63, 64, 65, 130, 4200])
def test_many_sequences(batch):
    """The search for a tile's sequence, at one, two and three rounds of 64 probes."""
    new = [(3 * i) % 4 for i in range(batch)]
    total = [n + (i % 5) for i, n in enumerate(new)]
    if batch > 200:  # a few rows only are compared
        new = [1 if i % 7 == 0 else 0 for i in range(batch)]
        total = [n + (i % 5) for i, n in enumerate(new)]
    q, c, start = case(THIN, new, total, seed=8)
    check(q, c, start, num_splits=1)
    check(q, c, start, num_splits=2)


def test_one_token_rows_equal_the_decode():
    q, c, start = case(LLAMA3_8B, [1] * 5, [1, 700, 33, 128, 2049], "int8", torch.float16, seed=9)
    got = check(q, c, start)
    ref = paged_decode_hip(q, c)
    _, bound = po.attend(q, c, start)
    # both are within their bounds of the exact result: twice the bound apart at most, and two roundings
    assert bool(((got - ref).abs().double() <= 2 * bound + 2 ** -10 * ref.abs().double() + 2 ** -20).all())


def test_long_prompt_rows():
    """A prompt of many row tiles: the first, some inner and the last rows."""
    q, c, start = case(QWEN25_05B, [2500], [2700], seed=10)
    got = paged_prefill_hip(q, c, offsets(start))
    k, v = po.dense_rows(c, 0)
    for i in (0, 1, 17, 18, 1023, 1300, 2499):
        for h in (0, 6, 7, 13):
            want, bound = po.one_map(q[i:i + 1, h].double(), k[:, h // 7], v[:, h // 7], 200 + i, 64 ** -0.5)
            assert po.worst(got[i:i + 1, h], want, bound) < 1, (i, h)


@pytest.mark.parametrize("kv,sdt", [KV[0], KV[2]], ids=["fp16", "fp8"])
@pytest.mark.parametrize("splits", [1, 3])
def test_what_pages_hold_past_the_end(kv, sdt, splits):
    """NaN and infinities behind the sequences' ends and in the pages of nobody change nothing."""
    q, c, start = case(LLAMA3_8B, [6, 21], [37, 21], kv, sdt, seed=11)
    want = paged_prefill_hip(q, c, offsets(start), num_splits=splits).clone()
    used = torch.zeros(c.k_cache.shape[:2], dtype=torch.bool, device="cuda")
    for b, t in enumerate(c.seq_lens.tolist()):
        pos = torch.arange(t, device="cuda")
        used[c.block_table[b].long()[pos // 16], pos % 16] = True
    for junk in (float("nan"), float("inf")):
        for store in (c.k_cache, c.v_cache):
            flat = store.view(torch.uint8) if kv == "fp8_e5m2" else store
            flat[~used] = (0x7f if junk != junk else 0x7c) if kv == "fp8_e5m2" else junk
        assert torch.equal(paged_prefill_hip(q, c, offsets(start), num_splits=splits), want)


@pytest.mark.parametrize("junk", [float("inf"), float("-inf"), float("nan")])
@pytest.mark.parametrize("which", ["k", "v"])
@pytest.mark.parametrize("splits", [1, 2])
def test_infinities_reach_only_the_rows_that_see_them(junk, which, splits):
    """An infinity or NaN in a new token's K or V: rows before it are what they were."""
    q, c, start = case(LLAMA3_8B, [150], [170], seed=12)
    before = paged_prefill_hip(q, c, offsets(start), num_splits=splits).clone()
    t = 20 + 77  # row 77's token
    store = c.k_cache if which == "k" else c.v_cache
    store[c.block_table[0, t // 16].long(), t % 16, :, 5] = junk
    got = paged_prefill_hip(q, c, offsets(start), num_splits=splits)
    assert torch.equal(got[:77], before[:77])
    if which == "v":
        hit = got[77:, :, 5].float()
        # (a P that rounds to zero makes 0 * inf, NaN)
        assert bool((torch.isnan(hit) | (hit == junk)).all())
        others = [e for e in range(128) if e != 5]
        assert torch.equal(got[77:, :, others], before[77:, :, others])
    elif junk != junk:
        assert bool(torch.isnan(got[77:].float()).all())
    # (an infinite K makes a score of +inf, NaN after the softmax, or of -inf, by the sign of q)


@pytest.mark.parametrize("splits", [1, 3])
@pytest.mark.parametrize("sdt", [torch.float16, torch.float32])
def test_int8_scales_of_any_size(sdt, splits):
    """Scales far apart, all tiny, all large, beyond what fp16 holds: P * scale stays in range."""
    for seed, factors in enumerate(([1e-3, 1.0, 300.0], [1e-4], [2000.0], [0.0, 1.0])):
        q, c, start = case(LLAMA3_8B, [9, 40], [600, 70], "int8", sdt, seed=60 + seed)
        r = torch.Generator().manual_seed(seed)
        pick = torch.tensor(factors)[torch.randint(len(factors), c.v_scale.shape, generator=r)].cuda()
        c.v_scale.copy_(c.v_scale * pick)
        check(q, c, start, num_splits=splits)
    if sdt == torch.float32:
        c.v_scale.mul_(1e7)
        got = paged_prefill_hip(q.bfloat16(), c, offsets(start), num_splits=splits)
        want, bound = po.attend(q.bfloat16(), c, start)
        assert po.worst(got, want, bound) < 1


@pytest.mark.parametrize("junk", [float("inf"), float("nan"), 1e30])
@pytest.mark.parametrize("which", ["k", "v"])
@pytest.mark.parametrize("splits", [1, 2])
def test_int8_scales_reach_only_the_rows_that_see_them(junk, which, splits):
    q, c, start = case(LLAMA3_8B, [150], [170], "int8", torch.float32, seed=70)
    before = paged_prefill_hip(q, c, offsets(start), num_splits=splits).clone()
    t = 20 + 77  # row 77's token
    (c.k_scale if which == "k" else c.v_scale)[c.block_table[0, t // 16].long(), t % 16] = junk
    got = paged_prefill_hip(q, c, offsets(start), num_splits=splits)
    assert torch.equal(got[:77], before[:77])
    if which == "v":
        hit = got[77:].float()  # (a value of 0, or a P that rounds to it, may meet the scale)
        assert float((~torch.isfinite(hit)).float().mean()) > 0.9


def test_strides():
    """q cut out of packed q/k/v rows, out inside a wider buffer, the cache with heads outermost in the page."""
    shape = LLAMA3_8B
    q, c, start = case(shape, [30, 9], [64, 9], seed=13)
    want = paged_prefill_hip(q, c, offsets(start))
    wide = torch.zeros((39, 48, 128), dtype=torch.float16, device="cuda")
    wide[:, 8:40] = q
    out = torch.zeros((39, 40, 136), dtype=torch.float16, device="cuda")
    hnd = dataclasses.replace(c, k_cache=c.k_cache.permute(0, 2, 1, 3).contiguous().permute(0, 2, 1, 3),
                              v_cache=c.v_cache.permute(0, 2, 1, 3).contiguous().permute(0, 2, 1, 3))
    table = torch.zeros((2, 99), dtype=torch.int32, device="cuda")
    table[:, 3:3 + c.block_table.shape[1]] = c.block_table
    hnd = dataclasses.replace(hnd, block_table=table[:, 3:3 + c.block_table.shape[1]])
    paged_prefill_hip(wide[:, 8:40], hnd, offsets(start), out=out[:, 4:36, :128])
    assert torch.equal(out[:, 4:36, :128], want)
    assert bool((out[:, :4] == 0).all()) and bool((out[:, 36:] == 0).all()) and bool((out[..., 128:] == 0).all())


def test_pool_past_4_gib():
    """Pages more than 4 GiB past the base."""
    shape = LLAMA3_8B
    q, c, start = case(shape, [20], [50], seed=14)
    want = paged_prefill_hip(q, c, offsets(start))
    blocks = (5 << 30) // (16 * 8 * 128 * 2)
    k = torch.empty((blocks, 16, 8, 128), dtype=torch.float16, device="cuda")
    v = torch.empty_like(k)
    far = torch.tensor([blocks - 1, blocks - 9, 3, blocks // 2 + 70000], dtype=torch.int32, device="cuda")
    k[far.long()] = c.k_cache[c.block_table[0].long()]
    v[far.long()] = c.v_cache[c.block_table[0].long()]
    big = dataclasses.replace(c, k_cache=k, v_cache=v, block_table=far[None, :])
    assert torch.equal(paged_prefill_hip(q, big, offsets(start)), want)


@pytest.mark.parametrize("splits", [1, 4, None])
def test_graph_replays_follow_the_lengths(splits):
    """Captured once, replayed with other lengths, offsets and q between eager work."""
    q, c, start = case(LLAMA3_8B, [5, 9], [90, 40], seed=15, pad=2)
    st, out = offsets(start), torch.zeros_like(q)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        paged_prefill_hip(q, c, st, out=out, num_splits=splits)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        paged_prefill_hip(q, c, st, out=out, num_splits=splits)
    for lens, to in (([90, 40], [0, 5, 14]), ([61, 33], [0, 9, 16]), ([7, 48], [0, 0, 3]), ([90, 40], [0, 5, 14])):
        c.seq_lens.copy_(torch.tensor(lens, dtype=torch.int32))
        st.copy_(torch.tensor(to, dtype=torch.int32))
        q.mul_(-1)
        out.fill_(3.0)
        graph.replay()
        torch.cuda.synchronize()
        eager = paged_prefill_hip(q, c, st, out=torch.full_like(q, 3.0), num_splits=splits)
        assert torch.equal(out, eager)
        want, bound = po.attend(q, c, to)
        assert po.worst(out[:to[-1]], want[:to[-1]], bound[:to[-1]]) < 1


def test_streams_at_once_and_bit_stability():
    """Split calls on two streams at once, each with partials of its own; the same bits every time."""
    q, c, start = case(LLAMA3_8B, [4], [3000], seed=16)
    q2, c2, _ = case(LLAMA3_8B, [4], [2500], seed=17)
    st = offsets(start)
    want = paged_prefill_hip(q, c, st, num_splits=9).clone()
    want2 = paged_prefill_hip(q2, c2, st, num_splits=9).clone()
    torch.cuda.synchronize()
    a, b = torch.cuda.Stream(), torch.cuda.Stream()
    for _ in range(10):
        with torch.cuda.stream(a):
            x = paged_prefill_hip(q, c, st, num_splits=9)
        with torch.cuda.stream(b):
            y = paged_prefill_hip(q2, c2, st, num_splits=9)
        torch.cuda.synchronize()
        assert torch.equal(x, want) and torch.equal(y, want2)


def test_device_values_out_of_range_stay_in_bounds():
    """Block-table entries outside the pool are clamped into it, lengths past the table to the table,
    offsets past the rows to the rows."""
    q, c, start = case(LLAMA3_8B, [6, 5], [40, 30], seed=18)
    bad = dataclasses.replace(c, block_table=c.block_table.clone(), seq_lens=c.seq_lens.clone())
    bad.block_table[0, 0], bad.block_table[1, 1] = -5, 1 << 30
    fixed = dataclasses.replace(bad, block_table=bad.block_table.clamp(0, c.num_blocks - 1))
    assert torch.equal(paged_prefill_hip(q, bad, offsets(start)), paged_prefill_hip(q, fixed, offsets(start)))
    bad.seq_lens[1] = 1 << 30
    fixed.seq_lens[1] = c.block_table.shape[1] * 16
    assert torch.equal(paged_prefill_hip(q, bad, offsets(start)), paged_prefill_hip(q, fixed, offsets(start)))
    out = torch.zeros_like(q)
    paged_prefill_hip(q, c, offsets([-4, 6, 5000]), out=out)
    torch.cuda.synchronize()
    assert torch.equal(out, paged_prefill_hip(q, c, offsets(start)))


def test_empty_calls():
    q, c, start = case(LLAMA3_8B, [0, 0], [5, 0], seed=19)
    assert paged_prefill_hip(q, c, offsets(start)).shape == (0, 32, 128)
