"""CPU tests of the prompt attention, differential attention and step tables: the C ABI's layout and
refusals, the wrappers' refusals, and the plan. Nothing here launches a kernel."""

from __future__ import annotations

import ctypes
import dataclasses
import pathlib
import re
import subprocess

import pytest
import torch

from pagedattn import (LLAMA3_8B, QWEN25_05B, ModelShape, _abi, allocate, build_step_tables, paged_diff_decode_hip,
                       paged_diff_prefill_hip, paged_prefill_hip, prefill)

ROOT = pathlib.Path(__file__).resolve().parent.parent
HEADER = ROOT / "include" / "pagedattn.h"
cpu_only = pytest.mark.skipif(torch.cuda.is_available(), reason="fake-pointer validation runs on CPU hosts only")
FAKE = 0x10000  # 16-byte aligned, never dereferenced


def _lib():
    if not _abi.lib_path().exists():
        import __graft_entry__

        __graft_entry__.build()
    return _abi.load()


def test_struct_layout_matches_header(tmp_path):
    structs = (("pa_prefill_args", _abi.PaPrefillArgs), ("pa_step_tables_args", _abi.PaStepTablesArgs))
    lines = ['#include <stddef.h>', '#include <stdio.h>', '#include "pagedattn.h"', 'int main(void){']
    for cname, cls in structs:
        lines.append(f'printf("{cname} sizeof %zu\\n", sizeof({cname}));')
        for f, _ in cls._fields_:
            lines.append(f'printf("{cname} {f} %zu\\n", offsetof({cname}, {f}));')
    lines.append("return 0;}")
    src, exe = tmp_path / "layout.c", tmp_path / "layout"
    src.write_text("\n".join(lines))
    subprocess.run(["gcc", "-std=c11", f"-I{ROOT / 'include'}", str(src), "-o", str(exe)], check=True)
    table = {tuple(x.split()[:2]): int(x.split()[2])
             for x in subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.splitlines()}
    for cname, cls in structs:
        assert table[(cname, "sizeof")] == ctypes.sizeof(cls)
        for f, _ in cls._fields_:
            assert table[(cname, f)] == getattr(cls, f).offset, (cname, f)


def test_form_constants_match_header():
    text = HEADER.read_text()
    for name in ("PA_FORM_TILES", "PA_FORM_STREAMS", "PA_FORM_STREAMS16"):
        assert int(re.search(rf"#define {name} (\d+)", text).group(1)) == getattr(_abi, name)


def _args(diff=False, **over):
    a = _abi.PaPrefillArgs()
    a.q = a.k_cache = a.v_cache = a.out = a.block_table = a.seq_lens = a.query_start_loc = FAKE
    a.batch, a.num_tokens, a.num_q_heads, a.num_kv_heads, a.head_dim = 2, 0, 32, 8, 128
    a.block_size, a.num_blocks, a.max_blocks, a.num_splits = 16, 64, 8, 1
    a.stride_qt, a.stride_qh = 32 * 128, 128
    a.stride_kn, a.stride_kt, a.stride_kh = 16 * 8 * 128, 8 * 128, 128
    a.stride_ot, a.stride_oh = 32 * 128, 256 if diff else 128
    a.stride_btb = 8
    a.kv_dtype, a.scale_dtype, a.io_dtype = _abi.PA_KV_FP16, _abi.PA_SCALE_NONE, _abi.PA_IO_FP16
    a.sm_scale = 0.1
    if diff:
        a.lam, a.stride_lam = FAKE, 1
    for name, value in over.items():
        setattr(a, name, value)
    return a


INVALID, UNSUPPORTED = _abi.PA_ERR_INVALID, _abi.PA_ERR_UNSUPPORTED
NAN, INF = float("nan"), float("inf")
BAD = [
    *[({p: None}, INVALID) for p in ("q", "k_cache", "v_cache", "out", "block_table", "seq_lens")],
    ({"batch": -1}, INVALID), ({"num_tokens": -1}, INVALID), ({"num_q_heads": 0}, INVALID),
    ({"num_kv_heads": 0}, INVALID), ({"num_kv_heads": 6}, INVALID), ({"num_blocks": 0}, INVALID),
    ({"max_blocks": 0}, INVALID), ({"head_dim": 96}, UNSUPPORTED), ({"block_size": 8}, UNSUPPORTED),
    ({"block_size": 48}, UNSUPPORTED), ({"block_size": 512}, UNSUPPORTED), ({"kv_dtype": 7}, INVALID),
    ({"io_dtype": 2}, INVALID), ({"sm_scale": 0.0}, INVALID), ({"sm_scale": -1.0}, INVALID),
    ({"sm_scale": NAN}, INVALID), ({"sm_scale": INF}, INVALID), ({"num_splits": 0}, INVALID),
    ({"num_splits": 5000}, INVALID), ({"num_splits": 2}, INVALID), ({"chunks": -1}, INVALID),
    ({"form": 3}, INVALID), ({"form": -1}, INVALID), ({"stride_qt": -8}, INVALID), ({"stride_kn": -8}, INVALID),
    ({"stride_btb": -1}, INVALID), ({"q": FAKE + 8}, INVALID), ({"stride_qh": 132}, INVALID),
    ({"out": FAKE + 2}, INVALID), ({"stride_oh": 129}, INVALID), ({"k_cache": FAKE + 4}, INVALID),
    ({"stride_kh": 4}, INVALID), ({"kv_dtype": _abi.PA_KV_INT8}, INVALID),
    ({"kv_dtype": _abi.PA_KV_INT8, "scale_dtype": _abi.PA_SCALE_FP32}, INVALID),
    ({"scale_dtype": _abi.PA_SCALE_FP16}, INVALID),
    ({"kv_dtype": _abi.PA_KV_INT8, "scale_dtype": _abi.PA_SCALE_FP32, "k_scale": FAKE + 2, "v_scale": FAKE}, INVALID),
    ({"max_blocks": 1 << 28}, UNSUPPORTED), ({"batch": 1 << 20, "stride_btb": 1 << 12}, UNSUPPORTED),
    ({"stride_kt": 1 << 27}, UNSUPPORTED), ({"stride_kn": 1 << 31}, UNSUPPORTED), ({"stride_kh": 1 << 30}, UNSUPPORTED),
    ({"stride_qt": 1 << 31}, UNSUPPORTED), ({"stride_ot": 1 << 31}, UNSUPPORTED),
    ({"num_tokens": 1 << 26}, UNSUPPORTED),
    ({"num_tokens": 1 << 25, "num_splits": 4096, "part_out": FAKE, "part_lse": FAKE}, UNSUPPORTED),
    ({"num_tokens": 1 << 24, "num_splits": 2, "part_out": FAKE, "part_lse": FAKE}, UNSUPPORTED),
    ({"num_tokens": 1 << 23, "num_splits": 64, "part_out": FAKE, "part_lse": FAKE}, UNSUPPORTED),
    ({"num_splits": 2, "part_out": FAKE + 4, "part_lse": FAKE}, INVALID),
]


@cpu_only
@pytest.mark.parametrize("over,code", BAD, ids=[",".join(o) + f"{i}" for i, (o, _) in enumerate(BAD)])
def test_c_refusals(over, code):
    lib = _lib()
    for fn, diff in ((lib.pa_prefill, False), (lib.pa_diff_prefill, True)):
        assert fn(ctypes.byref(_args(diff, **over)), None) == code, lib.pa_last_error()
        assert lib.pa_last_error()
        assert fn(ctypes.byref(_args(diff)), None) == _abi.PA_OK  # (no rows: nothing is launched)


@cpu_only
def test_c_refusals_of_one_form():
    lib = _lib()
    for fn in (lib.pa_prefill, lib.pa_diff_prefill, lib.pa_diff_decode):
        assert fn(None, None) == INVALID
    for fn in (lib.pa_prefill, lib.pa_diff_prefill):
        assert fn(ctypes.byref(_args(True, query_start_loc=None, num_tokens=2)), None) == INVALID
    decode = dict(query_start_loc=None, num_tokens=0, batch=0)
    assert lib.pa_diff_decode(ctypes.byref(_args(True, **decode)), None) == _abi.PA_OK
    assert lib.pa_diff_decode(ctypes.byref(_args(True)), None) == INVALID
    assert lib.pa_diff_decode(ctypes.byref(_args(True, query_start_loc=None, num_tokens=5)), None) == INVALID
    for over, code in (({"lam": None}, INVALID), ({"lam": FAKE + 2}, INVALID), ({"stride_lam": -1}, INVALID),
                       ({"norm_weight": FAKE + 4}, INVALID), ({"head_dim": 256}, UNSUPPORTED),
                       ({"num_q_heads": 9, "num_kv_heads": 3}, INVALID)):
        assert lib.pa_diff_prefill(ctypes.byref(_args(True, **over)), None) == code, over
    assert lib.pa_prefill(ctypes.byref(_args(head_dim=256)), None) == _abi.PA_OK
    # rows of no sequence: nothing to do (before any HIP call)
    for form in (_abi.PA_FORM_TILES, _abi.PA_FORM_STREAMS, _abi.PA_FORM_STREAMS16):
        assert lib.pa_prefill(ctypes.byref(_args(batch=0, num_tokens=500, form=form)), None) == _abi.PA_OK


def _table_args(**over):
    a = _abi.PaStepTablesArgs()
    for name, kind in a._fields_:
        if kind is ctypes.c_void_p and name != "finished":
            setattr(a, name, FAKE)
    a.batch, a.max_blocks, a.block_size, a.free_capacity, a.max_tokens, a.stride_btb = 4, 16, 16, 64, 32, 16
    for name, value in over.items():
        setattr(a, name, value)
    return a


@cpu_only
@pytest.mark.parametrize("over,code", [
    ({"batch": -1}, INVALID), ({"max_tokens": -1}, INVALID), ({"free_capacity": -1}, INVALID),
    ({"max_blocks": 0}, INVALID), ({"block_size": 0}, INVALID), ({"free_count": None}, INVALID),
    ({"free_count_out": None}, INVALID), ({"query_start_loc": None}, INVALID), ({"block_table": None}, INVALID),
    ({"seq_lens": None}, INVALID), ({"new_lens": None}, INVALID), ({"seq_lens_out": None}, INVALID),
    ({"slot_mapping": None}, INVALID), ({"free_pages": None}, INVALID), ({"seq_lens": FAKE + 2}, INVALID),
    ({"slot_mapping": FAKE + 4}, INVALID), ({"positions": FAKE + 4}, INVALID), ({"stride_btb": 15}, INVALID),
    ({"max_blocks": 1 << 27, "stride_btb": 1 << 27}, UNSUPPORTED),
    ({"batch": 1 << 20, "max_blocks": 1 << 12, "stride_btb": 1 << 12}, UNSUPPORTED),
    ({"max_tokens": 1 << 30}, UNSUPPORTED),
])
def test_table_refusals(over, code):
    lib = _lib()
    assert lib.pa_step_tables(ctypes.byref(_table_args(**over)), None) == code, lib.pa_last_error()
    assert lib.pa_step_tables(None, None) == INVALID


def _call(shape=LLAMA3_8B, kv="fp16", **cache_over):
    c = allocate(shape, 2, [20, 5], kv_dtype=kv, device="cpu", scale_dtype=torch.float32)
    c = dataclasses.replace(c, **cache_over)
    q = torch.zeros((6, shape.num_q_heads, shape.head_dim), dtype=torch.float16)
    return q, c, torch.tensor([0, 4, 6], dtype=torch.int32)


def test_wrapper_refusals():
    """Every check that comes before the one for the device."""
    q, c, st = _call()
    lam = torch.zeros(16)
    with pytest.raises(ValueError, match="GPU"):
        paged_prefill_hip(q, c, st)
    with pytest.raises(ValueError, match="GPU"):
        paged_diff_prefill_hip(q, c, st, lam)
    with pytest.raises(ValueError, match="GPU"):
        paged_diff_decode_hip(q[:2], c, lam)
    bad = [
        (ValueError, lambda: paged_prefill_hip(q[0], c, st)),
        (NotImplementedError, lambda: paged_prefill_hip(q.float(), c, st)),
        (ValueError, lambda: paged_prefill_hip(q[:, :8], c, st)),
        (ValueError, lambda: paged_prefill_hip(q[..., :64], c, st)),
        (ValueError, lambda: paged_prefill_hip(q.transpose(0, 2).contiguous().transpose(0, 2), c, st)),
        (ValueError, lambda: paged_prefill_hip(q, c, st, out=q[:5])),
        (ValueError, lambda: paged_prefill_hip(q, c, st, out=q.bfloat16())),
        (ValueError, lambda: paged_prefill_hip(q, c, st.long())),
        (ValueError, lambda: paged_prefill_hip(q, c, st[:2])),
        (NotImplementedError, lambda: paged_prefill_hip(q, dataclasses.replace(c, kv_dtype="int4"), st)),
        (ValueError, lambda: paged_prefill_hip(q, dataclasses.replace(c, kv_dtype="bf16"), st)),
        (ValueError, lambda: paged_prefill_hip(q, dataclasses.replace(c, block_size=32), st)),
        (ValueError, lambda: paged_prefill_hip(q, dataclasses.replace(c, v_cache=c.v_cache[:, :8]), st)),
        (ValueError, lambda: paged_prefill_hip(q, dataclasses.replace(c, k_cache=c.k_cache[0]), st)),
        (ValueError, lambda: paged_prefill_hip(q, dataclasses.replace(c, block_table=c.block_table.long()), st)),
        (ValueError, lambda: paged_prefill_hip(q, dataclasses.replace(c, block_table=c.block_table[0]), st)),
        (ValueError, lambda: paged_prefill_hip(q, dataclasses.replace(c, seq_lens=c.seq_lens[:1]), st)),
        (ValueError, lambda: paged_diff_decode_hip(q, c, lam)),
        (ValueError, lambda: paged_diff_prefill_hip(q, c, st, lam[:8])),
        (ValueError, lambda: paged_diff_prefill_hip(q, c, st, lam.half())),
        (ValueError, lambda: paged_diff_prefill_hip(q, c, st, lam, norm_weight=torch.ones(128))),
        (ValueError, lambda: paged_diff_prefill_hip(q, c, st, lam, norm_weight=torch.ones(512)[::2])),
    ]
    for error, call in bad:
        with pytest.raises(error) as e:
            call()
        assert "needs GPU tensors" not in str(e.value)
    q8, c8, _ = _call(kv="int8")
    for over in ({"k_scale": None}, {"v_scale": c8.v_scale.half()}, {"k_scale": c8.k_scale[:, :8]}):
        with pytest.raises(ValueError, match="scale"):
            paged_prefill_hip(q8, dataclasses.replace(c8, **over), st)
    odd = ModelShape(9, 3, 64, "odd")
    q3, c3, _ = _call(odd)
    with pytest.raises(ValueError, match="pairs"):
        paged_diff_prefill_hip(q3, c3, st, torch.zeros(4))


def test_table_wrapper_refusals():
    i32 = torch.int32
    good = dict(block_table=torch.zeros((3, 8), dtype=i32), seq_lens=torch.zeros(3, dtype=i32),
                new_lens=torch.zeros(3, dtype=i32), free_pages=torch.zeros(9, dtype=i32),
                free_count=torch.zeros(1, dtype=i32), block_size=16, max_tokens=5)
    with pytest.raises(ValueError, match="GPU"):
        build_step_tables(**good)
    for over in ({"block_table": torch.zeros((3, 8))}, {"block_table": torch.zeros(3, dtype=i32)},
                 {"block_table": torch.zeros((8, 3), dtype=i32).t()}, {"block_table": torch.zeros((3, 0), dtype=i32)},
                 {"seq_lens": torch.zeros(2, dtype=i32)}, {"seq_lens": torch.zeros(3)},
                 {"new_lens": torch.zeros(6, dtype=i32)[::2]}, {"free_count": torch.zeros(2, dtype=i32)},
                 {"free_pages": torch.zeros((3, 3), dtype=i32)}, {"finished": torch.zeros(3, dtype=i32)},
                 {"slot_mapping": torch.zeros(5, dtype=i32)}, {"slot_mapping": torch.zeros(4, dtype=torch.int64)},
                 {"positions": torch.zeros(6, dtype=torch.int64)}, {"query_start_loc": torch.zeros(3, dtype=i32)},
                 {"seq_lens_out": torch.zeros(4, dtype=i32)}, {"max_tokens": -1}):
        with pytest.raises(ValueError) as e:
            build_step_tables(**{**good, **over})
        assert "built on the GPU" not in str(e.value), over


def test_plan():
    """The form by average rows, the splits by what is left of the chip."""
    tiles, streams, streams16 = _abi.PA_FORM_TILES, _abi.PA_FORM_STREAMS, _abi.PA_FORM_STREAMS16
    plan = prefill._plan
    # rows, batch, units, longest, CUs, row width, maps
    assert plan(16384 * 4, 1, 8, 16384, 256, 128, 1) == (tiles, 1)
    assert plan(24 * 5 * 4, 24, 8, 8000, 256, 128, 1)[0] == streams
    assert plan(24 * 4 * 4, 24, 8, 8000, 256, 128, 1)[0] == streams16
    assert plan(24 * 9 * 4, 24, 8, 8000, 256, 128, 1)[0] == tiles
    assert plan(64 * 4, 64, 4, 4096, 256, 256, 2)[0] == streams16   # 8 columns: 4 pairs, two maps
    assert plan(64 * 12, 64, 4, 4096, 256, 256, 2)[0] == streams
    assert plan(64 * 17, 64, 4, 4096, 256, 256, 2)[0] == tiles
    # splits: none that would hold fewer than 256 tokens, none for a full chip
    assert plan(24 * 7, 24, 1, 192, 256, 128, 2) == (streams16, 1)
    assert plan(4, 1, 8, 100_000, 256, 128, 1)[1] == 128
    assert plan(4, 1, 8, 1024, 256, 128, 1)[1] == 4
    assert plan(4000 * 4, 4000, 8, 8192, 256, 128, 1)[1] == 1


def test_presets_take_pairs():
    for shape in (LLAMA3_8B, QWEN25_05B):
        assert shape.num_kv_heads % 2 == 0 and shape.num_q_heads % 2 == 0
