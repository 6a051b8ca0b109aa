"""Prompt attention, differential attention and step tables, as cases that can be timed and compared.

Four kinds of call:

  prefill       causal attention of several new tokens of each sequence over the paged cache that
                already holds them: whole prompts, chunks of prompts, a few speculative tokens.
  diff_decode   differential attention of one new token of each sequence over the paged cache.
  diff_prefill  the same for several new tokens.
  tables        a serving step's block table, slot map, positions and lengths, built on the device
                from the sequences' new token counts and a stack of free pages.

With `own` false, `run` computes them from elementary torch operations in 32 bits (whole numbers for
the tables); with `own` true it calls `pagedattn`. `exact` computes them in 64 bits, from the
definitions.

Shapes are the library's presets (a differential layer takes their heads in pairs); lengths follow
its benchmark and tests. K and V are N(0, 1) rows stored in the cache's type; the query heads'
magnitudes run from 0.5 to 2.5, so some heads attend widely and some to few tokens.
"""

from __future__ import annotations

import math
import pathlib
import random
import sys

import torch

own = False

DEV = "cuda"
# (query heads, kv heads, head dim)
SHAPES = {
    "llama3-8b": (32, 8, 128),
    "llama3-70b": (64, 8, 128),
    "qwen2.5-0.5b": (14, 2, 64),
    "mha-debug": (8, 8, 128),
}
STORE = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp8_e5m2": torch.float8_e5m2, "int8": torch.int8}
SCALES = {"fp16": torch.float16, "fp32": torch.float32}
EPS = 1e-5
LAMBDA_INIT = 0.8 - 0.6 * math.exp(-0.3 * 11)  # a middle layer's

# bounds of a drawn case: those of the largest listed ones
MOST_FLOPS = 4.0 * 128 * 32 * (16384 * 16385 // 2)
MOST_KV_BYTES = 64 * 4096 * 4096
MOST_ROWS = 1024
MOST_TABLE_TOKENS = 131072


# ---------------------------------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------------------------------

def listed():
    def attend(name, kind, shape, kv, io, batch, new, ctx, scale="", page=16, norm=False):
        return {"name": name, "kind": kind, "shape": shape, "kv": kv, "scale": scale, "io": io, "page": page,
                "batch": batch, "new_lo": new[0], "new_hi": new[1], "ctx_lo": ctx[0], "ctx_hi": ctx[1],
                "norm": norm}

    def tables(name, rows, page, blocks, grow, prompts, lo, hi, finished, ctx, capacity):
        return {"name": name, "kind": "tables", "rows": rows, "page": page, "blocks": blocks, "grow": grow,
                "prompts": prompts, "lo": lo, "hi": hi, "finished": finished, "ctx": ctx, "capacity": capacity}

    return [
        # one short question to a small model: bound by latency
        attend("short_prompt_bf16", "prefill", "qwen2.5-0.5b", "bf16", "bf16", 1, (37, 37), (0, 0)),
        # a batch of chat prompts of different lengths
        attend("chat_prompts_fp16", "prefill", "llama3-8b", "fp16", "fp16", 6, (150, 1500), (0, 0)),
        # one whole long prompt: the largest
        attend("long_prompt_fp16", "prefill", "llama3-8b", "fp16", "fp16", 1, (16384, 16384), (0, 0)),
        # chunks of long prompts beside what the fp8 cache holds of them, a large model
        attend("chunked_fp8", "prefill", "llama3-70b", "fp8_e5m2", "bf16", 4, (512, 512), (1000, 12000)),
        # five speculative tokens of each of two dozen sequences, int8 cache with fp32 scales
        attend("verify_int8", "prefill", "llama3-8b", "int8", "fp16", 24, (5, 5), (500, 8000), scale="fp32"),
        # two dozen chats with short contexts on a small differential model
        attend("diff_chat_fp16", "diff_decode", "qwen2.5-0.5b", "fp16", "fp16", 24, (1, 1), (31, 191), norm=True),
        # a full batch of 4K contexts
        attend("diff_batch_fp16", "diff_decode", "llama3-8b", "fp16", "fp16", 64, (1, 1), (4095, 4095), norm=True),
        # ragged contexts in an int8 cache with fp16 scales, pages of 32 tokens
        attend("diff_ragged_int8", "diff_decode", "qwen2.5-0.5b", "int8", "fp16", 160, (1, 1), (100, 8000),
               scale="fp16", page=32, norm=True),
        # a whole prompt of a differential model
        attend("diff_prompt_bf16", "diff_prefill", "llama3-8b", "bf16", "bf16", 1, (4096, 4096), (0, 0), norm=True),
        # chunks of a small differential model's prompts, fp8 cache, no norm
        attend("diff_chunks_fp8", "diff_prefill", "qwen2.5-0.5b", "fp8_e5m2", "fp16", 12, (60, 700), (0, 3000)),
        # a decode step's tables: every sequence grows by one token
        tables("tables_decode_step", 64, 16, 512, 64, 0, 0, 0, 0, 4096, 64),
        # a mixed step: sequences that grow, some that finish, prompts that enter
        tables("tables_mixed_step", 512, 16, 1024, 440, 48, 200, 4000, 24, 8000, 131072),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _token_bytes(case):
    """K and V bytes of one token of one layer, scales included."""
    _, hkv, d = SHAPES[case["shape"]]
    per = d * torch.empty((), dtype=STORE[case["kv"]]).element_size()
    return 2 * hkv * (per + {"": 0, "fp16": 2, "fp32": 4}[case["scale"]])


def draw(rng):
    kind = rng.choices(["prefill", "diff_decode", "diff_prefill", "tables"], [3, 3, 2, 2])[0]
    if kind == "tables":
        rows = _log_int(rng, 1, MOST_ROWS)
        prompts = rng.choice([0, 0, _log_int(rng, 1, max(1, rows // 4))]) if rows > 3 else 0
        finished = rng.choice([0, _log_int(rng, 1, max(1, rows // 8))]) if rows > 3 else 0
        hi = max(2, min(4000, MOST_TABLE_TOKENS // (2 * max(1, prompts))))
        page = rng.choice([16, 16, 32, 64])
        ctx = _log_int(rng, 16, 8000)
        blocks = -(-(ctx + hi + 1) // page) + rng.randint(0, 64)
        capacity = rows + prompts * hi + rng.randint(0, 300)
        return {"kind": kind, "rows": rows, "page": page, "blocks": blocks, "grow": rows - prompts - finished,
                "prompts": prompts, "lo": max(1, hi // 16), "hi": hi, "finished": finished, "ctx": ctx,
                "capacity": capacity}
    kv = rng.choice(["fp16", "bf16", "fp8_e5m2", "int8"])
    case = {"kind": kind, "shape": rng.choice(sorted(SHAPES)), "kv": kv,
            "scale": rng.choice(["fp16", "fp32"]) if kv == "int8" else "",
            "io": "bf16" if kv == "bf16" else rng.choice(["fp16", "bf16"]),
            "page": rng.choice([16, 16, 16, 32, 64]), "norm": kind != "prefill" and rng.random() < 0.7}
    case["batch"] = _log_int(rng, 1, 192 if kind == "diff_decode" else 32)
    if kind == "diff_decode":
        case["new_lo"] = case["new_hi"] = 1
        hi = _log_int(rng, 32, 65536)
    else:
        case["new_hi"] = _log_int(rng, 2, 8192)
        case["new_lo"] = max(1, case["new_hi"] // rng.choice([1, 1, 8]))
        hi = rng.choice([0, _log_int(rng, 16, 32768)])
    case["ctx_hi"] = hi
    case["ctx_lo"] = hi // rng.choice([1, 16])
    while (work(case)["flops"] > 0.95 * MOST_FLOPS
           or case["batch"] * (case["ctx_hi"] + case["new_hi"]) * _token_bytes(case) > 0.95 * MOST_KV_BYTES):
        if case["batch"] > 1:
            case["batch"] = case["batch"] * 3 // 4
        else:
            case["ctx_hi"], case["ctx_lo"] = case["ctx_hi"] * 3 // 4, case["ctx_lo"] * 3 // 4
            case["new_hi"] = max(1, case["new_hi"] * 7 // 8)
            case["new_lo"] = min(case["new_lo"], case["new_hi"])
    return case


def lengths(case):
    """(new tokens, tokens before them) of each sequence. They belong to the case, not to the seed."""
    r = random.Random(f"{case['batch']} {case['new_lo']} {case['new_hi']} {case['ctx_lo']} {case['ctx_hi']}")
    n = case["batch"]
    return ([r.randint(case["new_lo"], case["new_hi"]) for _ in range(n)],
            [r.randint(case["ctx_lo"], case["ctx_hi"]) for _ in range(n)])


def table_rows(case):
    """(tokens before, new tokens, finished) of each row of a tables case."""
    r = random.Random(f"{case['rows']} {case['ctx']} {case['hi']} {case['prompts']} {case['finished']}")
    kinds = ["grow"] * case["grow"] + ["prompt"] * case["prompts"] + ["finished"] * case["finished"]
    r.shuffle(kinds)
    before, new = [], []
    for kind in kinds:
        before.append(0 if kind == "prompt" else r.randint(1, case["ctx"]))
        new.append({"grow": 1, "prompt": r.randint(max(1, case["lo"]), max(1, case["hi"])), "finished": 0}[kind])
    return before, new, [kind == "finished" for kind in kinds]


def work(case):
    if case["kind"] == "tables":
        before, new, done = table_rows(case)
        p = case["page"]
        pages = sum(-(-(b + n) // p) - -(-b // p) for b, n, d in zip(before, new, done) if not d)
        freed = sum(-(-b // p) for b, d in zip(before, done) if d)
        tokens = sum(new)
        # lengths in and out, start offsets; pages moved; slots and positions
        return {"bytes": 16 * case["rows"] + 8 * (pages + freed) + 16 * case["capacity"], "flops": 4 * tokens}
    hq, hkv, d = SHAPES[case["shape"]]
    new, ctx = lengths(case)
    rows = sum(new)
    pairs = sum(n * c + n * (n + 1) // 2 for n, c in zip(new, ctx))
    tokens = sum(new) + sum(ctx)
    per_pair = (4 if case["kind"] == "prefill" else 6) * d * hq
    pages = sum(-(-(n + c) // case["page"]) for n, c in zip(new, ctx))
    return {"bytes": tokens * _token_bytes(case) + 2 * rows * hq * d * 2 + 4 * pages, "flops": per_pair * pairs}


# ---------------------------------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------------------------------

def _fill(g, shape, kv, scale):
    """N(0, 1) rows of `shape` [NB, P, H, D] in the cache's type, and their scales (int8: absolute
    maximum / 127 per token and head)."""
    store = torch.empty(shape, dtype=STORE[kv], device=DEV)
    sc = torch.empty(shape[:3], dtype=SCALES[scale], device=DEV) if kv == "int8" else None
    per = shape[1] * shape[2] * shape[3]
    step = max(1, (1 << 26) // per)
    for i in range(0, shape[0], step):
        x = torch.randn((min(step, shape[0] - i), *shape[1:]), generator=g, device=DEV, dtype=torch.float32)
        if kv != "int8":
            store[i:i + step] = x.to(torch.float16).to(STORE[kv]) if kv == "fp8_e5m2" else x.to(STORE[kv])
            continue
        s = (x.abs().amax(-1) / 127.0).to(SCALES[scale])
        sc[i:i + step] = s
        store[i:i + step] = (x / s.float()[..., None]).round().clamp(-127, 127).to(torch.int8)
    return store, sc


def _ints(values, dtype=torch.int32):
    return torch.tensor(values, dtype=dtype, device=DEV)


def _starts(new):
    cu = [0]
    for n in new:
        cu.append(cu[-1] + n)
    return cu


def prepare(case, seed):
    if case["kind"] == "tables":
        return _prepare_tables(case, seed)
    g = torch.Generator(device=DEV).manual_seed(seed)
    hq, hkv, d = SHAPES[case["shape"]]
    new, ctx = lengths(case)
    total = [n + c for n, c in zip(new, ctx)]
    p = case["page"]
    pages = [-(-t // p) for t in total]
    pool = sum(pages) + 7
    order = torch.randperm(pool, generator=torch.Generator().manual_seed(seed)).to(torch.int32)
    table = torch.zeros((len(new), max(pages)), dtype=torch.int32)
    at = 0
    for b, n in enumerate(pages):
        table[b, :n] = order[at:at + n]
        at += n
    k, ks = _fill(g, (pool, p, hkv, d), case["kv"], case["scale"])
    v, vs = _fill(g, (pool, p, hkv, d), case["kv"], case["scale"])
    io = torch.bfloat16 if case["io"] == "bf16" else torch.float16
    size = torch.linspace(0.5, 2.5, hq, device=DEV)[:, None]
    q = (torch.randn((sum(new), hq, d), generator=g, device=DEV) * size).to(io)
    state = {"case": case, "q": q, "k": k, "v": v, "ks": ks, "vs": vs, "table": table.to(DEV), "new": new,
             "total": total, "lens": _ints(total), "start": _ints(_starts(new)), "longest": max(total)}
    if case["kind"] != "prefill":
        # exp of two learned dot products and the layer's constant, once a layer
        w = torch.randn((4, hq // 2, d), generator=g, device=DEV) * 0.1
        state["lam"] = (w[0] * w[1]).sum(-1).exp() - (w[2] * w[3]).sum(-1).exp() + LAMBDA_INIT
        state["norm"] = (1.0 + 0.2 * torch.randn((2 * d,), generator=g, device=DEV)) if case["norm"] else None
    if own:
        pkg = str(pathlib.Path(__file__).resolve().parent.parent / "paged-decode-attention_amd")
        if pkg not in sys.path:
            sys.path.insert(0, pkg)
        from pagedattn import ModelShape, PagedKVCache

        state["cache"] = PagedKVCache(ModelShape(hq, hkv, d, case["shape"]), p, case["kv"], k, v, ks, vs,
                                      state["table"], state["lens"])
    return state


def _prepare_tables(case, seed):
    before, new, done = table_rows(case)
    p = case["page"]
    held = [-(-b // p) for b in before]
    need = sum(-(-(b + n) // p) - h for b, n, h, d in zip(before, new, held, done) if not d)
    pool = sum(held) + need + 64
    order = torch.randperm(pool, generator=torch.Generator().manual_seed(seed)).to(torch.int32)
    table = torch.zeros((case["rows"], case["blocks"]), dtype=torch.int32)
    at = 0
    for b, n in enumerate(held):
        table[b, :n] = order[at:at + n]
        at += n
    free = torch.zeros((pool,), dtype=torch.int32)  # room for every page of the pool
    free[:pool - at] = order[at:]
    state = {"case": case, "table": table.to(DEV), "lens": _ints(before), "new": _ints(new), "free": free.to(DEV),
             "count": _ints([pool - at]), "done": _ints(done, torch.bool) if any(done) else None,
             "lens_out": torch.empty((case["rows"],), dtype=torch.int32, device=DEV),
             "count_out": torch.empty((1,), dtype=torch.int32, device=DEV)}
    if own:
        pkg = str(pathlib.Path(__file__).resolve().parent.parent / "paged-decode-attention_amd")
        if pkg not in sys.path:
            sys.path.insert(0, pkg)
        import pagedattn  # noqa: F401
    return state


# ---------------------------------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------------------------------

def run(state):
    kind = state["case"]["kind"]
    if kind == "tables":
        return _run_tables(state)
    if not own:
        return _plain(state)
    import pagedattn

    if kind == "prefill":
        return pagedattn.paged_prefill_hip(state["q"], state["cache"], state["start"], max_seq_len=state["longest"])
    more = {"max_seq_len": state["longest"]}
    if state["norm"] is not None:
        more.update(norm_weight=state["norm"], norm_eps=EPS, out_scale=1.0 - LAMBDA_INIT)
    if kind == "diff_decode":
        return pagedattn.paged_diff_decode_hip(state["q"], state["cache"], state["lam"], **more)
    return pagedattn.paged_diff_prefill_hip(state["q"], state["cache"], state["start"], state["lam"], **more)


def _run_tables(state):
    page, capacity = state["case"]["page"], state["case"]["capacity"]
    if own:
        import pagedattn

        step = pagedattn.build_step_tables(state["table"], state["lens"], state["new"], state["free"], state["count"],
                                           page, capacity, finished=state["done"], seq_lens_out=state["lens_out"],
                                           free_count_out=state["count_out"])
        return (step.query_start_loc, step.slot_mapping, step.positions, step.seq_lens, step.free_count,
                state["table"], state["free"])
    return _plain_tables(state, page, capacity)


def _rows(store, scale, pages):
    """The cache rows of some pages, [tokens, heads, D] in 32 bits."""
    x = store[pages].to(torch.float32)
    if scale is not None:
        x = x * scale[pages].to(torch.float32)[..., None]
    return x.flatten(0, 1)


def _softmax_values(q, k, v, first, scale):
    """q [n, H, D], k [T, G, D], v [T, G, E] -> [n, H, E]; row i sees tokens 0 .. first + i."""
    n, h, d = q.shape
    t, g = k.shape[:2]
    per = h // g
    out = torch.empty((n, h, v.shape[2]), dtype=q.dtype, device=q.device)
    hidden = torch.arange(t, device=q.device)[None, :] > first + torch.arange(n, device=q.device)[:, None]
    step = max(1, int(2 ** 30 // max(1, n * t * per)))  # kv heads at a time
    for j in range(0, g, step):
        w = min(step, g - j)
        qq = q[:, j * per:(j + w) * per].reshape(n, w, per, d).permute(1, 2, 0, 3).reshape(w, per * n, d)
        s = torch.matmul(qq, k[:, j:j + w].permute(1, 2, 0).contiguous()).view(w, per, n, t)
        s *= scale
        s.masked_fill_(hidden, -math.inf)
        s -= s.amax(-1, keepdim=True)
        s.exp_()
        o = torch.matmul(s.view(w, per * n, t), v[:, j:j + w].permute(1, 0, 2).contiguous()).view(w, per, n, -1)
        o /= s.sum(-1, keepdim=True)
        out[:, j * per:(j + w) * per] = o.permute(2, 0, 1, 3).reshape(n, w * per, -1)
    return out


def _plain(state):
    case = state["case"]
    q = state["q"].to(torch.float32)
    hq, hkv, d = SHAPES[case["shape"]]
    diff = case["kind"] != "prefill"
    scale = d ** -0.5
    out = torch.empty((q.shape[0], hq // 2, 2 * d) if diff else tuple(q.shape), dtype=torch.float32, device=DEV)
    at = 0
    for b, (n, total) in enumerate(zip(state["new"], state["total"])):
        pages = state["table"][b, :-(-total // case["page"])].long()
        k = _rows(state["k"], state["ks"], pages)[:total]
        v = _rows(state["v"], state["vs"], pages)[:total]
        x = q[at:at + n]
        if diff:
            v = v.reshape(total, hkv // 2, 2 * d)
            one = _softmax_values(x[:, 0::2], k[:, 0::2], v, total - n, scale)
            two = _softmax_values(x[:, 1::2], k[:, 1::2], v, total - n, scale)
            out[at:at + n] = one - state["lam"][:, None] * two
        else:
            out[at:at + n] = _softmax_values(x, k, v, total - n, scale)
        at += n
    if diff and state["norm"] is not None:
        out *= (out.square().mean(-1, keepdim=True) + EPS).rsqrt()
        out *= state["norm"] * (1.0 - LAMBDA_INIT)
    return out.to(state["q"].dtype)


def _plain_tables(state, page, capacity):
    table, free, count = state["table"], state["free"], state["count"]
    rows, blocks = table.shape
    col = torch.arange(blocks, device=DEV)[None, :]
    lens = state["lens"].long().clamp_min(0)
    new = state["new"].long().clamp_min(0)
    held = (lens + page - 1) // page
    size = free.shape[0]
    top = count.long()
    if state["done"] is not None:
        # finished rows push their pages, one row after the other
        push = torch.where(state["done"], held, 0)
        to = top + (push.cumsum(0) - push)[:, None] + col
        to = torch.where(col < push[:, None], to, size).clamp(0, size)
        spare = torch.cat([free, free[:1]])
        spare.scatter_(0, to.flatten(), table.flatten())
        free.copy_(spare[:size])
        top = top + push.sum()
        lens = torch.where(state["done"], 0, lens)
        held = torch.where(state["done"], 0, held)
    # rows that do not fit get nothing: their table row, the token capacity, the pages left
    fits = lens + new <= blocks * page
    asked = torch.where(fits, new, 0)
    fits &= (asked == 0) | (asked.cumsum(0) <= capacity)
    asked = torch.where(fits, asked, 0)
    need = (lens + asked + page - 1) // page - held
    fits &= (need == 0) | (need.cumsum(0) <= top)
    given = torch.where(fits, asked, 0)
    need = torch.where(fits, need, 0)
    first = need.cumsum(0) - need
    take = (top - 1 - first[:, None] - (col - held[:, None])).clamp(0, size - 1)
    added = (col >= held[:, None]) & (col < (held + need)[:, None])
    table.copy_(torch.where(added, free[take], table))
    start = torch.zeros((rows + 1,), dtype=torch.int64, device=DEV)
    start[1:] = given.cumsum(0)
    i = torch.arange(capacity, device=DEV)
    b = torch.searchsorted(start, i, right=True).sub_(1).clamp_(0, rows - 1)
    pos = i - start[b] + lens[b]
    live = i < start[-1]
    slot = table[b, (pos // page).clamp(0, blocks - 1)].long() * page + pos % page
    slot = torch.where(live, slot, -1)
    pos = torch.where(live, pos, 0)
    state["lens_out"].copy_(lens + given)
    state["count_out"].copy_(top - need.sum())
    return start.to(torch.int32), slot, pos, state["lens_out"], state["count_out"], table, free


# ---------------------------------------------------------------------------------------------------
# the definitions in 64 bits
# ---------------------------------------------------------------------------------------------------

def exact(case, seed):
    state = prepare(case, seed)
    if case["kind"] == "tables":
        return _exact_tables(case, state)
    new, ctx = lengths(case)
    hq, hkv, d = SHAPES[case["shape"]]
    pairs = 1 if case["kind"] == "prefill" else 2  # heads that make one output head
    kv_heads = hkv // pairs
    group = hq // hkv
    result = torch.zeros((sum(new), hq // pairs, pairs * d), dtype=torch.float64, device=DEV)

    def token_rows(store, scales, where, head):
        blk, off = where
        x = store[blk, off, head].to(torch.float64)
        return x if scales is None else x * scales[blk, off, head].to(torch.float64)[:, None]

    row = 0
    for b in range(case["batch"]):
        total = new[b] + ctx[b]
        t = torch.arange(total, device=DEV)
        where = (state["table"][b].long()[t // case["page"]], t % case["page"])
        for j in range(kv_heads):
            keys = [token_rows(state["k"], state["ks"], where, pairs * j + m) for m in range(pairs)]
            value = torch.cat([token_rows(state["v"], state["vs"], where, pairs * j + m) for m in range(pairs)], 1)
            for h in range(j * group, (j + 1) * group):
                for lo in range(0, new[b], 8192):
                    hi = min(new[b], lo + 8192)
                    seen = t[None, :] <= torch.arange(ctx[b] + lo, ctx[b] + hi, device=DEV)[:, None]
                    maps = []
                    for m in range(pairs):
                        x = state["q"][row + lo:row + hi, pairs * h + m].to(torch.float64)
                        logit = (x @ keys[m].t()) / math.sqrt(d)
                        weight = torch.where(seen, logit, -math.inf)
                        maps.append(torch.exp(weight - torch.logsumexp(weight, 1, keepdim=True)))
                    p = maps[0] if pairs == 1 else maps[0] - state["lam"][h].to(torch.float64) * maps[1]
                    y = p @ value
                    if pairs == 2 and state["norm"] is not None:
                        y = y / torch.sqrt((y * y).mean(1, keepdim=True) + EPS)
                        y = y * state["norm"].to(torch.float64) * (1.0 - LAMBDA_INIT)
                    result[row + lo:row + hi, h] = y
        row += new[b]
    return result


def _exact_tables(case, state):
    before, new, done = table_rows(case)
    page, capacity, blocks = case["page"], case["capacity"], case["blocks"]
    table = state["table"].tolist()
    count = int(state["count"])
    stack = state["free"].tolist()
    size = len(stack)
    for b, gone in enumerate(done):
        if gone:
            for c in range(-(-before[b] // page)):
                stack[count] = table[b][c]
                count += 1
    after, start, slots, positions = [], [0], [], []
    pool, asked, needed = count, 0, 0
    for b, n in enumerate(new):
        length = 0 if done[b] else before[b]
        have, want = -(-length // page), -(-(length + n) // page)
        # served in row order: from the first row that the capacity (or the pool) does not hold, no row
        # gets tokens (or pages); a row that its own table row does not hold counts for neither
        if length + n > blocks * page:
            n, want = 0, have
        asked += n
        if n > 0 and asked > capacity:
            n, want = 0, have
        needed += want - have
        if want > have and needed > pool:
            n, want = 0, have
        for c in range(have, want):
            count -= 1
            table[b][c] = stack[count]
        for x in range(length, length + n):
            positions.append(x)
            slots.append(table[b][x // page] * page + x % page)
        after.append(length + n)
        start.append(start[-1] + n)
    pad = capacity - len(slots)
    assert len(stack) == size
    return (_ints(start), _ints(slots + [-1] * pad, torch.int64), _ints(positions + [0] * pad, torch.int64),
            _ints(after), _ints([count]), _ints(table), _ints(stack))
