"""Differential attention over the paged cache against the float64 oracle, on the GPU."""

from __future__ import annotations

import dataclasses

import pytest
import torch

import prompt_oracle as po
from pagedattn import (LLAMA3_8B, MHA_DEBUG, QWEN25_05B, ModelShape, _abi, paged_diff_decode_hip,
                       paged_diff_prefill_hip, paged_prefill_hip, prefill)
from test_gpu_prefill import KV, case, offsets

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

THIN = ModelShape(12, 4, 32, "thin")
WIDE_GROUP = ModelShape(142, 2, 64, "g71")


def weights(shape, seed, norm=True):
    g = torch.Generator().manual_seed(500 + seed)
    lam = (0.6 + 0.3 * torch.randn((shape.num_q_heads // 2,), generator=g)).cuda()
    w = (1.0 + 0.2 * torch.randn((2 * shape.head_dim,), generator=g)).cuda() if norm else None
    return lam, w


def check(q, c, start, lam, w, **kw):
    print(f"{c.shape.name} {c.kv_dtype} page {c.block_size} start {start[:8]} lens {c.seq_lens.tolist()[:8]} "
          f"norm {w is not None} {kw}", flush=True)
    decode = start == list(range(len(start)))
    more = {"norm_weight": w, "norm_eps": 1e-5, "out_scale": 0.4} if w is not None else {}
    got = paged_diff_prefill_hip(q, c, offsets(start), lam, **more, **kw)
    torch.cuda.synchronize()
    want, bound = po.attend(q, c, start, lam=lam, **more)
    n = start[-1]
    assert po.worst(got[:n], want[:n], bound[:n]) < 1
    if decode:
        one = paged_diff_decode_hip(q, c, lam, **more, **kw)
        torch.cuda.synchronize()
        assert po.worst(one, want, bound) < 1
        return one
    return got


@pytest.mark.parametrize("kv,sdt", KV, ids=["fp16", "bf16", "fp8", "int8h", "int8s"])
@pytest.mark.parametrize("shape", [LLAMA3_8B, QWEN25_05B, MHA_DEBUG, THIN], ids=lambda s: s.name)
@pytest.mark.parametrize("new,total", [([1, 1, 1, 1], [1, 300, 31, 64]), ([1, 20, 40], [1, 75, 40])],
                         ids=["decode", "prefill"])
def test_types_and_shapes(shape, kv, sdt, new, total):
    io = torch.bfloat16 if kv == "bf16" else torch.float16
    q, c, start = case(shape, new, total, kv, sdt, io, seed=21)
    lam, w = weights(shape, 21)
    check(q, c, start, lam, w)
    check(q, c, start, lam, None, num_splits=1)


@pytest.mark.parametrize("splits", [1, 2, 5, 33, None])
@pytest.mark.parametrize("new", [[1, 1, 1], [3, 1, 2]], ids=["decode", "prefill"])
def test_splits(splits, new):
    for shape, page in ((QWEN25_05B, 32), (LLAMA3_8B, 16)):
        q, c, start = case(shape, new, [1200, 3, 64], "int8", torch.float32, page=page, seed=22)
        lam, w = weights(shape, 22)
        check(q, c, start, lam, w, num_splits=splits)
        check(q, c, start, lam, w, num_splits=splits, max_seq_len=1200)


def test_ragged_splits():
    """Planned splits, sized by the lengths that the launch finds."""
    total = [0, 3000, 5, 40, 1, 700] + [30] * 70
    q, c, start = case(QWEN25_05B, [1] * len(total), total, "int8", torch.float32, page=32, seed=29)
    lam, w = weights(QWEN25_05B, 29)
    check(q, c, start, lam, w)
    check(q, c, start, lam, w, max_seq_len=3000)


@pytest.mark.parametrize("splits", [1, 3])
def test_empty_rows_and_sequences(splits):
    q, c, start = case(QWEN25_05B, [1, 1, 1], [0, 40, 0], seed=23)
    lam, w = weights(QWEN25_05B, 23)
    got = check(q, c, start, lam, w, num_splits=splits)
    assert bool((got[0] == 0).all()) and bool((got[2] == 0).all())
    q, c, start = case(QWEN25_05B, [9, 0, 4], [5, 30, 2], seed=24, pad=3)
    out = torch.full((16, 7, 128), 7.0, dtype=torch.float16, device="cuda")
    got = check(q, c, start, lam, w, num_splits=splits, out=out)
    assert bool((got[:4] == 0).all()) and bool((got[13:] == 7.0).all())


def test_wide_group():
    """More pairs a kv pair than a row tile holds."""
    lam, w = weights(WIDE_GROUP, 25)
    for new in ([1, 1], [3, 2]):
        q, c, start = case(WIDE_GROUP, new, [50, 33], seed=25)
        check(q, c, start, lam, w)


def test_one_lambda_for_all_and_zero():
    """A stride of zero; lambda 0 leaves the first map."""
    q, c, start = case(QWEN25_05B, [5, 3], [60, 3], seed=26)
    lam = torch.tensor([0.35], device="cuda").expand(7)
    check(q, c, start, lam, None)
    first = check(q, c, start, torch.zeros(7, device="cuda"), None)
    # V's first half alone is what a plain attention with the first map's queries and keys gives; each
    # is within its bound of that (they may sum in another order)
    half = dataclasses.replace(c, shape=ModelShape(7, 1, 64, "half"), k_cache=c.k_cache[:, :, :1],
                               v_cache=c.v_cache[:, :, :1])
    plain = paged_prefill_hip(q[:, 0::2].contiguous(), half, offsets(start))
    want, bound = po.attend(q[:, 0::2], half, start)
    assert po.worst(first[..., :64], want, bound) < 1 and po.worst(plain, want, bound) < 1


def test_strided_heads():
    """Heads outermost in the page: the two heads of a pair lie apart."""
    q, c, start = case(LLAMA3_8B, [12, 4], [64, 9], "int8", torch.float32, seed=27)
    lam, w = weights(LLAMA3_8B, 27)
    want = paged_diff_prefill_hip(q, c, offsets(start), lam, norm_weight=w)
    apart = [t.permute(0, 2, 1, 3).contiguous().permute(0, 2, 1, 3) for t in (c.k_cache, c.v_cache)]
    hnd = dataclasses.replace(c, k_cache=apart[0], v_cache=apart[1])
    out = torch.zeros((16, 20, 264), dtype=torch.float16, device="cuda")
    paged_diff_prefill_hip(q, hnd, offsets(start), lam, norm_weight=w, out=out[:, 2:18, :256])
    assert torch.equal(out[:, 2:18, :256], want)
    assert bool((out[:, :2] == 0).all()) and bool((out[..., 256:] == 0).all())
    qd = q[:2].contiguous()
    assert torch.equal(paged_diff_decode_hip(qd, hnd, lam, norm_weight=w),
                       paged_diff_decode_hip(qd, c, lam, norm_weight=w))


@pytest.mark.parametrize("junk", [float("inf"), float("nan")])
def test_infinities_reach_only_the_rows_that_see_them(junk):
    q, c, start = case(LLAMA3_8B, [90], [100], seed=28)
    lam, _ = weights(LLAMA3_8B, 28)
    before = paged_diff_prefill_hip(q, c, offsets(start), lam).clone()
    t = 10 + 41
    c.v_cache[c.block_table[0, t // 16].long(), t % 16, 2, 9] = junk
    got = paged_diff_prefill_hip(q, c, offsets(start), lam)
    assert torch.equal(got[:41], before[:41])
    # head 2 is the first half of pair 1's value: output heads 4 .. 7, element 9, inf - lambda inf
    assert bool(torch.isnan(got[41:, 4:8, 9].float()).all())
    keep = torch.ones((16, 256), dtype=torch.bool, device="cuda")
    keep[4:8, 9] = False
    assert torch.equal(got[:, keep], before[:, keep])


@pytest.mark.parametrize("splits", [1, 4])
def test_graph_replays(splits):
    q, c, _ = case(QWEN25_05B, [1, 1, 1], [200, 150, 90], "fp8_e5m2", seed=29)
    lam, w = weights(QWEN25_05B, 29)
    out = torch.zeros((3, 7, 128), dtype=torch.float16, device="cuda")
    call = lambda o: paged_diff_decode_hip(q, c, lam, out=o, norm_weight=w, num_splits=splits)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        call(out)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call(out)
    for lens in ([200, 150, 90], [0, 3, 64], [129, 1, 17]):
        c.seq_lens.copy_(torch.tensor(lens, dtype=torch.int32))
        q.mul_(-1)
        out.fill_(3.0)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, call(torch.zeros_like(out)))
