"""CPU-side checks of tpa_page_tables, tpa_norm_rope(_bwd) and tpa_decode_shared: the ctypes structures have the header's layout, and what the
C ABI and the host layer refuse is refused before any launch."""

import ctypes
import itertools
import os
import subprocess

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

from conftest import ROOT

NULL, SHAPE, DTYPE, ALIGN, WORKSPACE, UNSUPPORTED = -1, -2, -3, -4, -5, -6
P = 1 << 20  # a pointer that nothing follows


def test_struct_layout_matches_the_c_compiler(tmp_path):
    from tpa import _dispatch as d

    fields = {"TpaPageTablesArgs": d.TpaPageTablesArgs, "TpaNormRopeArgs": d.TpaNormRopeArgs, "TpaNormRopeBwdArgs": d.TpaNormRopeBwdArgs}
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


def page_tables(**changed):
    from tpa import _dispatch as d

    a = d.TpaPageTablesArgs(kv_lengths=P, new_tokens=2 * P, page_table=3 * P, free_pages=4 * P, free_start=5 * P, slots=6 * P, positions=7 * P, starts=8 * P,
                            new_kv_lengths=9 * P, new_free_start=10 * P, B=4, pages_per_seq=8, page_size=16, num_free=9, num_tokens=7)
    for k, v in changed.items():
        setattr(a, k, v)
    return d.load_library().tpa_page_tables(ctypes.byref(a), None)


@pytest.mark.parametrize(
    "code,changed",
    [(SHAPE, dict(B=0)), (SHAPE, dict(B=8193)), (SHAPE, dict(page_size=0)), (SHAPE, dict(pages_per_seq=-1)), (SHAPE, dict(num_tokens=-1)), (SHAPE, dict(num_free=-1)),
     (SHAPE, dict(pages_per_seq=1 << 20, page_size=1 << 11)), (UNSUPPORTED, dict(new_kv_lengths=P)), (UNSUPPORTED, dict(new_kv_lengths=P + 12)), (UNSUPPORTED, dict(new_free_start=5 * P))]
    + [(NULL, {f: None}) for f in ("kv_lengths", "new_tokens", "page_table", "free_pages", "slots", "positions", "starts", "new_kv_lengths", "new_free_start")],
)
def test_page_tables_refuses(code, changed):
    assert page_tables(**changed) == code


def norm_rope(bwd=False, **changed):
    from tpa import _dispatch as d

    cls = d.TpaNormRopeBwdArgs if bwd else d.TpaNormRopeArgs
    names = [n for n, t in cls._fields_ if t is d.TpaFactor]
    a = cls(**{n: d.TpaFactor(P, 1440, 144, 144) for n in names}, rope_cos=P, rope_sin=P, n_axes=1, B=1, l=4, H=16, D=128, rq=6, rk=2, rope_len=9, dtype=1, weight_dtype=0,
            normalize=1, eps=1e-6)
    a.sections[0] = 64
    if bwd:
        a.dq_weight, a.workspace, a.workspace_bytes = P, P, 1 << 30
    for k, v in changed.items():
        if k == "sections":
            for i, x in enumerate(v):
                a.sections[i] = x
        elif k in names:
            getattr(a, k).ptr = v
        else:
            setattr(a, k, v)
    fn = d.load_library().tpa_norm_rope_bwd if bwd else d.load_library().tpa_norm_rope
    return fn(ctypes.byref(a), None)


@pytest.mark.parametrize("bwd", [False, True])
@pytest.mark.parametrize(
    "code,changed",
    [(SHAPE, {k: 0}) for k in ("B", "l", "H", "D", "rq", "rk", "rope_len", "n_axes")]
    + [(SHAPE, dict(D=127)), (SHAPE, dict(D=258)), (SHAPE, dict(n_axes=5)), (SHAPE, dict(sections=[65])), (SHAPE, dict(sections=[-1])), (SHAPE, dict(n_axes=2, sections=[40, 25])),
       (SHAPE, dict(B=1 << 16, l=1 << 16)), (SHAPE, dict(H=4096, rq=64, kernel=1)), (DTYPE, dict(dtype=2)), (DTYPE, dict(weight_dtype=-1)), (UNSUPPORTED, dict(kernel=3)),
       (UNSUPPORTED, dict(kernel=2, D=96, sections=[48])), (UNSUPPORTED, dict(kernel=2, H=12)), (UNSUPPORTED, dict(kernel=2, rq=17)), (NULL, dict(rope_cos=None)), (NULL, dict(rope_sin=None)),
       (NULL, dict(qa=None)), (NULL, dict(kb=None))],
)
def test_norm_rope_refuses(bwd, code, changed):
    assert norm_rope(bwd, **changed) == code


def test_norm_rope_refuses_what_only_one_direction_has():
    assert norm_rope(qb_out=None) == NULL
    assert norm_rope(slots=P, page_size=0, num_slots=64) == SHAPE
    assert norm_rope(slots=P, page_size=16, num_slots=40) == SHAPE
    assert norm_rope(slots=P, page_size=16, num_slots=64, va_out=None) == NULL
    assert norm_rope(True, dqb=None) == NULL
    assert norm_rope(True, workspace=None) == WORKSPACE
    assert norm_rope(True, workspace_bytes=100) == WORKSPACE
    assert norm_rope(True, workspace=P + 4) == ALIGN


def shared(prefix=4, **changed):
    from tpa import _dispatch as d

    f = lambda w: d.TpaFactor(P, 40 * 2 * w, 2 * w, w)
    a = d.TpaFwdArgs(qa=f(8), qb=f(64), ka=f(8), kb=f(64), va=f(8), vb=f(64), o=P, lse=P, B=2, lq=1, lk=40, H=8, dk=64, dv=64, rq=2, rk=2, dtype=1, sm_scale=1.0)
    for k, v in changed.items():
        if k in ("qa", "vb"):
            getattr(a, k).ptr = v
        else:
            setattr(a, k, v)
    return d.load_library().tpa_decode_shared(ctypes.byref(a), prefix, None)


@pytest.mark.parametrize(
    "code,changed",
    [(SHAPE, dict(prefix=-1)), (SHAPE, dict(prefix=41)), (SHAPE, dict(B=0)), (SHAPE, dict(dk=300)), (DTYPE, dict(dtype=7)), (NULL, dict(o=None)), (NULL, dict(vb=None)),
     (UNSUPPORTED, dict(num_splits=3)), (UNSUPPORTED, dict(nomat=1)), (UNSUPPORTED, dict(q_segment_ids=P, kv_segment_ids=P)), (UNSUPPORTED, dict(causal=3)), (UNSUPPORTED, dict(kernel=5)),
     (SHAPE, dict(page_table=P, page_size=0, pages_per_seq=3)), (SHAPE, dict(page_table=P, page_size=16, pages_per_seq=2)), (UNSUPPORTED, dict(kernel=2, H=9)), (UNSUPPORTED, dict(kernel=2, rk=3)),
     (SHAPE, dict(B=1 << 20, lq=1 << 10)), (SHAPE, dict(B=1 << 18, lq=8))],
)
def test_decode_shared_refuses(code, changed):
    assert shared(**changed) == code


@pytest.mark.parametrize("h,dk", [(8, 64), (24, 128), (32, 64), (64, 128)])
@pytest.mark.parametrize("dtype", [0, 1])
def test_the_workspace_holds_whole_ranges(dtype, h, dk):
    """For every split of a cache into prefix and own keys: parts of D + 2 numbers a row and head, no more ranges than blocks of 32 rows."""
    from tpa import _dispatch as d

    lib = d.load_library()
    f = lambda w: d.TpaFactor(P, 1 << 20, 8 * w, w)
    for b, lq, rk, lk in itertools.product((1, 2, 37, 300), (1, 5, 64), (1, 2, 8), (1, 31, 200, 5000, 70000)):
        for prefix in sorted({0, 1, lk // 2, lk - 1, lk}):
            a = d.TpaFwdArgs(qa=f(h), qb=f(dk), ka=f(h), kb=f(dk), va=f(h), vb=f(dk), B=b, lq=lq, lk=lk, H=h, dk=dk, dv=dk, rq=6, rk=rk, dtype=dtype, sm_scale=1.0)
            for name in ("ka", "kb", "va", "vb"):
                w = getattr(a, name).stride_r
                getattr(a, name).stride_l = rk * w
            size = lib.tpa_decode_shared_workspace_bytes(ctypes.byref(a), prefix)
            of_range = 4 * b * lq * h * (dk + 2)
            assert size % of_range == 0 and 1 <= size // of_range <= (prefix * rk + 31) // 32 + ((lk - prefix) * rk + 63) // 32 + 1, (b, lq, rk, lk, prefix, size)


def test_the_host_layer_refuses_operands_that_do_not_fit():
    """Shape-only tensors that claim to live on a GPU reach the checks and nothing behind them."""
    from tpa import tpa

    with FakeTensorMode():
        new = lambda *s, dtype=torch.bfloat16, on="cuda": torch.empty(s, device=on, dtype=dtype)
        q, k, cos = new(2, 6, 6, 72), new(2, 6, 2, 72), new(9, 32, dtype=torch.float32)
        with pytest.raises(ValueError):
            tpa.tpa_norm_rope(q[0], k, 8, cos, cos)
        with pytest.raises(AssertionError):
            tpa.tpa_norm_rope(q, new(2, 5, 2, 72), 8, cos, cos)
        with pytest.raises(TypeError):
            tpa.tpa_norm_rope(q, new(2, 6, 2, 72, dtype=torch.float32), 8, cos, cos)
        with pytest.raises(TypeError):
            tpa.tpa_norm_rope(new(2, 6, 6, 72, dtype=torch.float16), new(2, 6, 2, 72, dtype=torch.float16), 8, cos, cos)
        with pytest.raises(ValueError):
            tpa.tpa_norm_rope(q, k, 8, cos, cos, sections=[])
        with pytest.raises(TypeError):
            tpa.tpa_norm_rope(q, k, 8, cos, cos, sections=[8, 2.5])
        i32 = dict(dtype=torch.int32)
        with pytest.raises(ValueError):
            tpa.tpa_page_tables(new(2, **i32), new(2, **i32), new(2, 4), new(9, **i32), page_size=4, num_tokens=2)
        with pytest.raises(ValueError):
            tpa.tpa_page_tables(new(2, **i32), new(2, **i32), new(2, 4, **i32), new(9, **i32), page_size=4, num_tokens=2, free_start=new(2, **i32))
        with pytest.raises(ValueError):  # a second device
            tpa.tpa_page_tables(new(2, **i32), new(2, on="cuda:1", **i32), new(2, 4, **i32), new(9, **i32), page_size=4, num_tokens=2)
