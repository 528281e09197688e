"""CPU-side checks of the operators over a cache in 4 bits, the beams and the pages: the ctypes structures have the header's layout, and what the C ABI and the host layer refuse is
refused before any launch."""

import ctypes
import os
import subprocess

import numpy as np
import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

import fp4_model as fp4
from conftest import ROOT

NULL, SHAPE, DTYPE, ALIGN, WORKSPACE, UNSUPPORTED = -1, -2, -3, -4, -5, -6
P = 1 << 20  # a pointer that nothing follows


def test_struct_layout_matches_the_c_compiler(tmp_path):
    from tpa import _dispatch as d

    fields = {n: getattr(d, n) for n in ("TpaFp4RowsArgs", "TpaDecodeFp4Args", "TpaBeamSelectArgs", "TpaPool", "TpaPagesForkArgs", "TpaPagesCompactArgs")}
    lines = ["#include <stdio.h>", "#include <stddef.h>", '#include "tpa_abi.h"', "int main(void) {"]
    for name, cls in fields.items():
        lines.append(f'printf("{name} %zu\\n", sizeof({name}));')
        lines += [f'printf("{name}.{f} %zu\\n", offsetof({name}, {f}));' for f, _ in cls._fields_]
    (tmp_path / "layout.c").write_text("\n".join(lines + ["return 0; }"]))
    subprocess.run(["gcc", "-I", os.path.join(ROOT, "include"), str(tmp_path / "layout.c"), "-o", str(tmp_path / "layout")], check=True)
    got = dict(line.split() for line in subprocess.run([str(tmp_path / "layout")], check=True, capture_output=True, text=True).stdout.splitlines())
    for name, cls in fields.items():
        assert int(got[name]) == ctypes.sizeof(cls)
        assert all(int(got[f"{name}.{f}"]) == getattr(cls, f).offset for f, _ in cls._fields_), name


def test_row_bytes():
    from tpa import tpa

    assert tpa.fp4_row_bytes(32, 128) == 88 and tpa.fp4_row_bytes(1, 1) == 4 and tpa.fp4_row_bytes(0, 64) == 0
    assert all(tpa.fp4_row_bytes(h, d) == fp4.row_bytes(h, d) for h in (1, 5, 8, 31, 32, 33, 64) for d in (1, 2, 63, 64, 65, 128))


def test_the_model_of_the_format():
    """The definition in numpy on values that can be worked out by hand."""
    codes, scale = fp4.quantise([7.25, 1.0, -0.25, 0.26, 5.0, -3.5])
    assert scale == 127 and (codes & 7).tolist() == [7, 2, 0, 1, 6, 6] and (codes >> 3).tolist() == [0, 0, 1, 0, 0, 1]
    assert fp4.quantise([7.2500001])[1] == 128 and fp4.quantise([0.0])[1] == 2 and fp4.quantise([np.inf])[1] == 255
    a, b = fp4.read_rows(np.maximum(fp4.write_row(np.arange(1, 7), np.full(33, -0.75)), 0), 6, 33)
    assert a.tolist() == [1, 2, 3, 4, 4, 6] and b.tolist() == [-0.75] * 33


def rows(read=False, **changed):
    from tpa import _dispatch as d

    f = lambda w: d.TpaFactor(P, 4 * 2 * w, 2 * w, w)
    a = d.TpaFp4RowsArgs(ka=f(8), kb=f(64), va=f(8), vb=f(64), k_cache=f(40), v_cache=f(40), slots=P, page_size=4, num_slots=16, B=2, l=4, H=8, dk=64, dv=64, rk=2, dtype=1)
    for k, v in changed.items():
        if k in ("ka", "vb", "k_cache"):
            getattr(a, k).ptr = v
        else:
            setattr(a, k, v)
    lib = d.load_library()
    return (lib.tpa_cache_read_fp4 if read else lib.tpa_cache_write_fp4)(ctypes.byref(a), None)


@pytest.mark.parametrize("read", [False, True])
@pytest.mark.parametrize(
    "code,changed",
    [(SHAPE, {k: 0}) for k in ("B", "l", "H", "dk", "dv", "rk", "page_size")]
    + [(SHAPE, dict(num_slots=-4)), (SHAPE, dict(num_slots=15)), (SHAPE, dict(B=1 << 16, l=1 << 16)), (SHAPE, dict(rk=1 << 15)), (DTYPE, dict(dtype=2)), (NULL, dict(ka=None)), (NULL, dict(vb=None)),
       (NULL, dict(k_cache=None)), (NULL, dict(slots=None))],
)
def test_rows_refuse(read, code, changed):
    assert rows(read, **changed) == code


def decode(size=False, **changed):
    from tpa import _dispatch as d

    f = lambda w, n: d.TpaFactor(P, n * 2 * w, 2 * w, w)
    a = d.TpaDecodeFp4Args(qa=f(8, 1), qb=f(64, 1), k_cache=f(40, 50), v_cache=f(40, 50), o=P, lse=P, B=2, lq=1, lk=50, H=8, dk=64, dv=64, rq=2, rk=2, dtype=1, sm_scale=1.0, workspace=P, workspace_bytes=1 << 30)
    for k, v in changed.items():
        if k in ("qa", "v_cache"):
            getattr(a, k).ptr = v
        elif k == "stride":
            a.k_cache.stride_r = v
        else:
            setattr(a, k, v)
    lib = d.load_library()
    return lib.tpa_decode_fp4_workspace_bytes(ctypes.byref(a)) if size else lib.tpa_decode_fp4(ctypes.byref(a), None)


@pytest.mark.parametrize(
    "code,changed",
    [(SHAPE, {k: 0}) for k in ("B", "lq", "lk", "H", "dk", "dv", "rq", "rk")]
    + [(SHAPE, dict(dk=257)), (SHAPE, dict(dv=300)), (SHAPE, dict(B=1 << 20, lq=64)), (SHAPE, dict(lk=1 << 30, rk=4)), (DTYPE, dict(dtype=-1)), (UNSUPPORTED, dict(causal=3)), (UNSUPPORTED, dict(kernel=3)),
       (UNSUPPORTED, dict(kernel=2, H=12)), (UNSUPPORTED, dict(kernel=2, rk=3)), (UNSUPPORTED, dict(kernel=2, dk=128)), (UNSUPPORTED, dict(kernel=2, stride=42)), (NULL, dict(qa=None)), (NULL, dict(v_cache=None)), (NULL, dict(o=None)),
       (SHAPE, dict(page_table=P, page_size=0, pages_per_seq=9, num_pages=9)), (SHAPE, dict(page_table=P, page_size=7, pages_per_seq=7, num_pages=9)), (SHAPE, dict(page_table=P, page_size=10, pages_per_seq=5)),
       (WORKSPACE, dict(workspace=None)), (WORKSPACE, dict(workspace_bytes=1000)), (ALIGN, dict(workspace=P + 16)), (ALIGN, dict(o=P + 8))],
)
def test_decode_refuses(code, changed):
    assert decode(**changed) == code


def test_decode_workspace():
    assert decode(True) > 0 and decode(True, kernel=1) == 0 and decode(True, rk=3) == 0 and decode(True, B=0) == 0 and decode(True, kernel=2, rk=3) == 0
    # the size it names is the size it needs
    need = decode(True)
    assert decode(workspace_bytes=need - 1) == WORKSPACE
    # more columns than a grid has sets of: the vector units, which need no workspace
    assert decode(size=True, B=1, lq=262140, kernel=2) > 0 and decode(size=True, B=1, lq=262141) == 0 and decode(B=1, lq=262141, kernel=2) == UNSUPPORTED


def beams(**changed):
    from tpa import _dispatch as d

    a = d.TpaBeamSelectArgs(logits=P, stride_b=400, stride_n=100, scores=P, finished=P, new_scores=P, parents=P, tokens=P, new_finished=P, B=2, beams=4, vocab=100, num_out=4, eos_token=3, dtype=0,
                            workspace=P, workspace_bytes=1 << 30)
    for k, v in changed.items():
        setattr(a, k, v)
    return d.load_library().tpa_beam_select(ctypes.byref(a), None)


@pytest.mark.parametrize(
    "code,changed",
    [(SHAPE, {k: 0}) for k in ("B", "beams", "vocab", "num_out")]
    + [(SHAPE, dict(beams=65)), (SHAPE, dict(num_out=65)), (SHAPE, dict(beams=1, vocab=3, num_out=4, eos_token=-1)), (SHAPE, dict(beams=64, vocab=1 << 25)), (SHAPE, dict(beams=1, vocab=(1 << 30) + 1, num_out=1)), (SHAPE, dict(eos_token=100)),
       (SHAPE, dict(eos_token=-2)), (UNSUPPORTED, dict(eos_token=-1)), (DTYPE, dict(dtype=5)), (WORKSPACE, dict(workspace=None)), (WORKSPACE, dict(workspace_bytes=8)), (ALIGN, dict(workspace=P + 8))]
    + [(NULL, {k: None}) for k in ("logits", "scores", "new_scores", "parents", "tokens", "new_finished")],
)
def test_beam_select_refuses(code, changed):
    assert beams(**changed) == code


def pages(fork, pool=None, **changed):
    from tpa import _dispatch as d

    pools = (d.TpaPool * 1)(d.TpaPool(*(pool or (P, 4 * 88, 88))))
    at = iter(range(2, 40))
    cls = d.TpaPagesForkArgs if fork else d.TpaPagesCompactArgs
    a = cls(**{n: next(at) * P for n, t in cls._fields_ if t is ctypes.c_void_p}, pools=pools, num_pools=1, B=3, pages_per_seq=5, page_size=4, num_pages=20, num_free=9, workspace_bytes=1 << 30)
    if fork:
        a.M = 4
    for k, v in changed.items():
        setattr(a, k, getattr(a, v) if isinstance(v, str) else v)
    lib = d.load_library()
    return (lib.tpa_pages_fork if fork else lib.tpa_pages_compact)(ctypes.byref(a), None)


@pytest.mark.parametrize("fork", [True, False])
@pytest.mark.parametrize(
    "code,changed",
    [(SHAPE, {k: 0}) for k in ("pages_per_seq", "page_size", "num_pages")]
    + [(SHAPE, {k: -1}) for k in ("B", "num_free", "num_pools")]
    + [(SHAPE, dict(B=8193)), (SHAPE, dict(pages_per_seq=1 << 30)), (SHAPE, dict(num_pages=1 << 30)), (SHAPE, dict(pool=(P, 4 * 88, 0))), (SHAPE, dict(pool=(P, 1 << 40, 1 << 30))), (UNSUPPORTED, dict(pool=(P, 4 * 88 - 1, 88))),
       (NULL, dict(pool=(None, 400, 88))), (WORKSPACE, dict(num_pages=9000, workspace=None)), (WORKSPACE, dict(num_pages=9000, workspace_bytes=64)), (ALIGN, dict(num_pages=9000, workspace=P + 4)), (UNSUPPORTED, dict(new_page_table="page_table")),
       (UNSUPPORTED, dict(new_page_shares="page_shares")), (UNSUPPORTED, dict(new_free_start="free_start")), (UNSUPPORTED, dict(new_free_pages="new_page_shares"))]
    + [(NULL, {k: None}) for k in ("page_table", "kv_lengths", "page_shares", "free_pages", "new_page_table", "new_page_shares", "new_free_pages", "new_free_start")],
)
def test_pages_refuse(fork, code, changed):
    assert pages(fork, **changed) == code


def test_pages_workspace():
    from tpa import _dispatch as d

    size = d.load_library().tpa_pages_workspace_bytes
    assert size(2048, 2048, 8192, 96) == 0 and size(8192, 0, 8192, 96) == 0
    for b, m, total in ((2049, 1, 100), (1, 2049, 100), (1, 1, 8193), (1, 0, 8193)):  # the size it names is the size it needs
        need = size(b, m, total, 1)
        assert need > 0 and pages(m > 0, B=b, num_pages=total, workspace_bytes=need - 1, **({"M": m} if m else {})) == WORKSPACE
    assert size(1, 1, 8192, 97) > 0
    assert size(1, -1, 9000, 1) == 0 and size(1, 1, 0, 1) == 0


def test_pages_refuse_what_only_one_call_has():
    assert pages(True, M=8193) == SHAPE and pages(True, M=-1) == SHAPE and pages(True, parents=None) == NULL and pages(True, new_kv_lengths=None) == NULL
    assert pages(False, num_pages=(1 << 20) + 1) == SHAPE and pages(False, moved=None) == NULL


def test_the_host_layer_refuses_operands_that_do_not_fit():
    """Shape-only tensors that claim to live on a GPU reach the checks and nothing behind them."""
    from tpa import tpa

    with FakeTensorMode():
        new = lambda *s, dtype=torch.bfloat16, on="cuda": torch.empty(s, device=on, dtype=dtype)
        u8, i32 = dict(dtype=torch.uint8), dict(dtype=torch.int32)
        k, cache, slots = new(1, 6, 2, 72), new(5, 4, 2, 40, **u8), new(1, 6, **i32)
        for bad in (
            lambda: tpa.tpa_cache_write_fp4(k, k, 8, new(5, 4, 2, 44, **u8), cache, slots),
            lambda: tpa.tpa_cache_write_fp4(k, k, 8, cache, cache, new(1, 5, **i32)),
            lambda: tpa.tpa_cache_write_fp4(k, k, 8, cache, cache, new(1, 6, on="cuda:1", **i32)),
            lambda: tpa.tpa_cache_write_fp4(k[0], k, 8, cache, cache, slots),
            lambda: tpa.tpa_cache_read_fp4(cache, cache, 8, slots, head_dim=128),
            lambda: tpa.tpa_cache_read_fp4(cache, cache, 8, slots[0], head_dim=64),
            lambda: tpa.tpa_cache_read_fp4(cache, cache, 8, slots, head_dim=0),
            lambda: tpa.tpa_decode_fp4(k[..., :8], k[..., 8:], cache, new(5, 4, 2, 44, **u8)),
            lambda: tpa.tpa_beam_select(new(2, 3, 9)[0], new(2, 3)),
            lambda: tpa.tpa_beam_select(new(2, 3, 9), new(2, 4)),
            lambda: tpa.tpa_beam_select(new(2, 3, 9), new(2, 3), num_out=28),
            lambda: tpa.tpa_beam_select(new(2, 3, 9), new(2, 3), num_out=0),
            lambda: tpa.tpa_beam_select(new(2, 3, 9), new(2, 3), eos_token=9),
            lambda: tpa.tpa_beam_select(new(2, 3, 9), new(2, 3), finished=new(2, 3, dtype=torch.bool)),
            lambda: tpa.tpa_pages_fork(new(2, 4, **i32), new(3, **i32), new(2, **i32), new(9, **i32), new(4, **i32), [], page_size=4),
            lambda: tpa.tpa_pages_fork(new(2, 4, **i32), new(2, **i32), new(2, **i32), new(9, **i32), new(4, **i32), [new(9, 5, 2)], page_size=4),
            lambda: tpa.tpa_pages_fork(new(2, 4, **i32), new(2, **i32), new(2, **i32), new(9, **i32), new(4, **i32), [new(9, 4, 2)[:, :, :1]], page_size=4),
            lambda: tpa.tpa_pages_compact(new(2, 4, **i32), new(2, **i32), new(0, **i32), new(4, **i32), [], page_size=4),
            lambda: tpa.tpa_pages_compact(new(2, 4, **i32), new(2, **i32), new(9, **i32), new(4, **i32), [], page_size=0),
        ):
            with pytest.raises(ValueError):
                bad()
        for bad in (
            lambda: tpa.tpa_cache_write_fp4(k, k, 8, new(5, 4, 2, 40), cache, slots),
            lambda: tpa.tpa_cache_write_fp4(k, k, 8, new(5, 4, 2, 40, on="cpu", **u8), cache, slots),
            lambda: tpa.tpa_cache_write_fp4(k, new(1, 6, 2, 72, dtype=torch.float32), 8, cache, cache, slots),
            lambda: tpa.tpa_cache_write_fp4(new(1, 6, 2, 72, dtype=torch.float16), new(1, 6, 2, 72, dtype=torch.float16), 8, cache, cache, slots),
            lambda: tpa.tpa_cache_read_fp4(cache, cache, 8, slots, head_dim=64, dtype=torch.float16),
            lambda: tpa.tpa_beam_select(new(2, 3, 9), new(2, 3), finished=new(2, 3), eos_token=1),
            lambda: tpa.tpa_beam_select(new(2, 3, 9), new(2, 3, **i32)),
            lambda: tpa.tpa_beam_select(new(2, 3, 9, **i32), new(2, 3)),
            lambda: tpa.tpa_pages_compact(new(2, 4, **i32), new(2, **i32), new(9, **i32), new(4, **i32), [new(9, 4, 2, on="cpu")], page_size=4),
            lambda: tpa.tpa_pages_compact(new(2, 4, **i32), new(2, **i32), new(9, **i32), new(4, **i32), 7, page_size=4),
        ):
            with pytest.raises(TypeError):
                bad()
        with pytest.raises(AssertionError):
            tpa.tpa_cache_write_fp4(k, new(1, 5, 2, 72), 8, cache, cache, slots)
        with pytest.raises(AssertionError):
            tpa.tpa_cache_write_fp4(k, k, 72, cache, cache, slots)
