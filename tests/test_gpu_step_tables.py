"""A step's tables on the GPU against the rules in plain Python, and a serving run of all of it."""

from __future__ import annotations

import random

import pytest
import torch

import prompt_oracle as po
from pagedattn import (PagedKVCache, QWEN25_05B, build_step_tables, paged_decode_hip, paged_prefill_hip,
                       reshape_and_cache)

pytestmark = pytest.mark.gpu


def oracle(table, lens, new, stack, count, page, max_tokens, finished=None):
    """The rules, row by row. Lists in, (start, slots, positions, lens, count, table, stack) out."""
    table, stack = [list(r) for r in table], list(stack)
    limit = len(table[0]) * page if table else 0
    lens = [max(0, x) for x in lens]
    new = [max(0, x) for x in new]
    for b, gone in enumerate(finished or []):
        if gone:
            for c in range(-(-lens[b] // page)):
                stack[count] = table[b][c]
                count += 1
            lens[b] = 0
    pool, asked, needed = count, 0, 0
    start, slots, positions = [0], [], []
    for b, n in enumerate(new):
        have = -(-lens[b] // page)
        if lens[b] + n > limit:
            n = 0
        asked += n
        if asked > max_tokens:
            n = 0
        need = -(-(lens[b] + n) // page) - have
        needed += need
        if need and needed > pool:
            n = need = 0
        for c in range(have, have + need):
            count -= 1
            table[b][c] = stack[count]
        for pos in range(lens[b], lens[b] + n):
            slots.append(table[b][pos // page] * page + pos % page)
            positions.append(pos)
        lens[b] += n
        start.append(start[-1] + n)
    pad = max_tokens - len(slots)
    return start, slots + [-1] * pad, positions + [0] * pad, lens, count, table, stack


def on_gpu(values, dtype=torch.int32):
    return torch.tensor(values, dtype=dtype, device="cuda")


def check(table, lens, new, stack, count, page, max_tokens, finished=None, in_place=False, stride=None):
    t = on_gpu(table)
    if stride:
        wide = torch.full((len(table), stride), -9, dtype=torch.int32, device="cuda")
        wide[:, :t.shape[1]] = t
        t = wide[:, :t.shape[1]]
    d_lens, d_stack, d_count = on_gpu(lens), on_gpu(stack), on_gpu([count])
    kw = {} if in_place else {"seq_lens_out": torch.full_like(d_lens, -7), "free_count_out": on_gpu([-7])}
    got = build_step_tables(t, d_lens, on_gpu(new), d_stack, d_count, page, max_tokens,
                            finished=None if finished is None else on_gpu(finished, torch.bool), **kw)
    torch.cuda.synchronize()
    want = oracle(table, lens, new, stack, count, page, max_tokens, finished)
    have = (got.query_start_loc, got.slot_mapping, got.positions, got.seq_lens, got.free_count, t, d_stack)
    names = ("query_start_loc", "slot_mapping", "positions", "seq_lens", "free_count", "block_table", "free_pages")
    for name, x, y in zip(names, have, want):
        assert x.tolist() == ([y] if name == "free_count" else y), name
    if in_place:
        assert d_lens.tolist() == want[3] and d_count.tolist() == [want[4]]
    else:
        assert d_lens.tolist() == list(lens) and d_count.tolist() == [count]
    if stride:
        assert bool((wide[:, len(table[0]):] == -9).all())
    return got


def scene(rows, page, blocks, seed, prompts=0.2, done=0.2, free=400):
    """Rows that grow, enter and finish, with pages dealt from one shuffled pool."""
    r = random.Random(seed)
    lens = [r.randint(0, page * blocks // 2) for _ in range(rows)]
    pool = list(range(sum(-(-x // page) for x in lens) + free))
    r.shuffle(pool)
    table = []
    for x in lens:
        n = -(-x // page)
        table.append([pool.pop() for _ in range(n)] + [0] * (blocks - n))
    new = [r.randint(2, page * blocks // 3) if r.random() < prompts else r.choice([0, 1, 1, 1]) for _ in range(rows)]
    gone = [r.random() < done for _ in range(rows)]
    size = sum(-(-x // page) for x in lens) + free
    return table, lens, new, pool + [0] * (size - len(pool)), len(pool), gone


@pytest.mark.parametrize("rows", [1, 2, 63, 64, 65, 500, 1023, 1024, 1025, 2500])
@pytest.mark.parametrize("max_tokens", [3000, 20000], ids=["one_launch", "two_launches"])
def test_rows(rows, max_tokens):
    table, lens, new, stack, count, gone = scene(rows, 16, 12, rows, prompts=0.05, free=2000)
    check(table, lens, new, stack, count, 16, max_tokens)
    check(table, lens, new, stack, count, 16, max_tokens, gone, in_place=True)


@pytest.mark.parametrize("page", [1, 3, 16, 32, 64, 256])
def test_page_sizes_and_strides(page):
    table, lens, new, stack, count, gone = scene(40, page, 9, page)
    check(table, lens, new, stack, count, page, 6000, gone, stride=13)


@pytest.mark.parametrize("free,max_tokens", [(0, 5000), (3, 5000), (20, 5000), (400, 0), (400, 1), (400, 200)])
def test_rows_that_do_not_fit(free, max_tokens):
    """The stack, or the token capacity, gives out in the middle of the rows."""
    for seed in range(4):
        table, lens, new, stack, count, gone = scene(50, 16, 10, 70 + seed, free=free)
        check(table, lens, new, stack, count, 16, max_tokens)
        check(table, lens, new, stack, count, 16, max_tokens, gone)


def test_edges_of_a_row():
    """Exactly full rows and pages, negative values, a table row one token too short, huge requests."""
    table = [[5, 6], [7, 0], [8, 9], [0, 0], [10, 0], [0, 0]]
    stack = [20, 21, 22, 23, 24, 25, 26]
    check(table, [31, 16, 32, 0, 15, 0], [1, 16, 1, 33, 1, 32], stack, 7, 16, 100)
    check(table, [17, 16, 32, -3, 15, 0], [15, -4, 0, 0, 2, -1], stack, 7, 16, 100, [False] * 5 + [True])
    big = 2 ** 31 - 1
    check(table, [17, 16, 32, 0, 15, 0], [big, 1, big, big, big, 2], stack, 7, 16, 100)


def test_a_finished_row_is_used_again_at_once():
    table = [[3, 1, 0], [4, 0, 0]]
    got = check(table, [20, 16], [18, 1], [0, 2, 0, 0, 0], 2, 16, 64, [True, False])
    assert got.slot_mapping[0].item() == 1 * 16  # the last page pushed is the first taken


def test_long_rows():
    """A prompt of hundreds of pages beside rows of one token, and its pages returned."""
    lens, new = [1, 9000, 0, 5], [1, 0, 12345, 1]
    pages = [-(-x // 16) for x in lens]
    pool = list(range(sum(pages) + 900))
    random.Random(5).shuffle(pool)
    table = [[pool.pop() for _ in range(n)] + [0] * (800 - n) for n in pages]
    size = sum(pages) + 900
    stack = pool + [0] * (size - len(pool))
    check(table, lens, new, stack, len(pool), 16, 16384)
    check(table, lens, new, stack, len(pool), 16, 16384, [False, True, False, False], in_place=True)


def test_empty():
    t = torch.zeros((0, 4), dtype=torch.int32, device="cuda")
    e = torch.zeros((0,), dtype=torch.int32, device="cuda")
    got = build_step_tables(t, e, e, on_gpu([1, 2]), on_gpu([2]), 16, 5)
    assert got.query_start_loc.tolist() == [0] and got.slot_mapping.tolist() == [-1] * 5
    assert got.free_count.tolist() == [2]


def test_serving_run():
    """Prompts enter, are written and attended, decode as replays of one graph, finish; new ones take
    their rows and pages. Every step's attention against the oracle over the tokens written so far."""
    shape, page, rows, blocks, pool = QWEN25_05B, 16, 4, 6, 20
    dev = "cuda"
    table = torch.zeros((rows, blocks), dtype=torch.int32, device=dev)
    lens = torch.zeros((rows,), dtype=torch.int32, device=dev)
    free = torch.randperm(pool, generator=torch.Generator().manual_seed(1)).to(torch.int32).to(dev)
    count = on_gpu([pool])
    k = torch.zeros((pool, page, 2, 64), dtype=torch.float16, device=dev)
    cache = PagedKVCache(shape, page, "fp16", k, torch.zeros_like(k), None, None, table, lens)
    g = torch.Generator().manual_seed(2)
    rand = lambda n, h: torch.randn((n, h, 64), generator=g).half().to(dev)
    new, done = torch.zeros_like(lens), torch.zeros((rows,), dtype=torch.bool, device=dev)
    said = [[] for _ in range(rows)]  # (k, v) of every token of each row

    def verify(got, q, start):
        for b in range(rows):
            if start[b] == start[b + 1]:
                continue
            kk = torch.stack([x for x, _ in said[b]]).double()
            vv = torch.stack([x for _, x in said[b]]).double()
            assert int(lens[b]) == len(said[b])
            first = len(said[b]) - (start[b + 1] - start[b])
            for h in (0, 13):
                rows_b = slice(start[b], start[b + 1])
                want, bound = po.one_map(q[rows_b, h].double(), kk[:, h // 7], vv[:, h // 7], first, 0.125)
                assert po.worst(got[rows_b, h], want, bound) < 1, (b, h)

    def prompt_step(add, gone):
        new.copy_(on_gpu(add))
        done.copy_(on_gpu(gone, torch.bool))
        step = build_step_tables(table, lens, new, free, count, page, 128, finished=done)
        q, kk, vv = rand(128, 14), rand(128, 2), rand(128, 2)
        reshape_and_cache(kk, vv, cache, step.slot_mapping)
        got = paged_prefill_hip(q, cache, step.query_start_loc)
        start = step.query_start_loc.tolist()
        for b in range(rows):
            said[b] = ([] if gone[b] else said[b]) + [(kk[i], vv[i]) for i in range(start[b], start[b + 1])]
        verify(got, q, start)

    prompt_step([30, 17, 0, 1], [False] * 4)
    # a decode step as a graph: every row that holds something grows by one token
    q, kk, vv = rand(rows, 14), rand(rows, 2), rand(rows, 2)
    out = torch.zeros_like(q)
    nobody = torch.zeros_like(done)
    buffers = dict(query_start_loc=torch.zeros((rows + 1,), dtype=torch.int32, device=dev),
                   slot_mapping=torch.zeros((rows,), dtype=torch.int64, device=dev),
                   positions=torch.zeros((rows,), dtype=torch.int64, device=dev))
    new.fill_(1)

    def decode_step():
        step = build_step_tables(table, lens, new, free, count, page, rows, finished=nobody, **buffers)
        reshape_and_cache(kk, vv, cache, step.slot_mapping)
        paged_decode_hip(q, cache, out=out, num_splits=1)

    def replayed(replay):
        for t in (q, kk, vv):
            t.copy_(rand(*t.shape[:2]))
        replay()
        torch.cuda.synchronize()
        for b in range(rows):
            said[b].append((kk[b].clone(), vv[b].clone()))
        verify(out, q, list(range(rows + 1)))

    replayed(decode_step)  # eager once: every library path is loaded before the capture
    graph = torch.cuda.CUDAGraph()
    keep = [t.clone() for t in (table, lens, free, count, cache.k_cache, cache.v_cache)]
    with torch.cuda.graph(graph):
        decode_step()
    for t, x in zip((table, lens, free, count, cache.k_cache, cache.v_cache), keep):
        assert torch.equal(t, x)  # a capture runs nothing
    for _ in range(18):
        replayed(graph.replay)
    prompt_step([25, 0, 4, 40], [True, False, False, True])
    new.fill_(1)
    for _ in range(5):
        replayed(graph.replay)
    held = sum(-(-len(x) // page) for x in said)
    assert int(count) == pool - held
    owned = [p for b in range(rows) for p in table[b, :-(-len(said[b]) // page)].tolist()]
    assert sorted(owned + free[:int(count)].tolist()) == list(range(pool))


@pytest.mark.parametrize("rows", [3, 257, 1500])
@pytest.mark.parametrize("max_tokens", [16384, 16385, 40000])
def test_between_one_launch_and_two(rows, max_tokens):
    """Rows of one to a few pages and of many, in turn, around the size that takes a second launch."""
    r = random.Random(rows + max_tokens)
    lens = [r.choice([0, 1, 15, 16, 17, 100, 900]) for _ in range(rows)]
    new = [r.choice([0, 1, 2, 4, 5, 16, 64, 65, 81, 130]) for _ in range(rows)]
    pages = [-(-x // 16) for x in lens]
    pool = list(range(sum(pages) + sum(new) // 8 + rows))
    r.shuffle(pool)
    size = len(pool)
    table = [[pool.pop() for _ in range(n)] + [0] * (70 - n) for n in pages]
    stack = pool + [0] * (size - len(pool))
    gone = [r.random() < 0.3 for _ in range(rows)]
    check(table, lens, new, stack, len(pool), 16, max_tokens)
    check(table, lens, new, stack, len(pool), 16, max_tokens, gone, in_place=True)
