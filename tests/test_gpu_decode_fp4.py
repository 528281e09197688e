"""tpa_decode_fp4 against softmax attention in 64 bits over the numbers that the rows stand for.

Tolerances, before the first run.  With L the largest sum of the magnitudes in a logit and A the output's sum of the magnitudes p |V|: for bf16 queries both Q and a
weight p a_v stand as two bf16 numbers (off by 2^-17 of themselves), for fp32 ones they are held to 2^-24; fp32 sums of n
terms are off by n 2^-24 of the magnitudes, an exponential by 2^-22 and the 2^-23 of its argument.  So a logit is off by
  delta = (2^-17 or 2^-24, and (D + 2 rk + rq + 8) 2^-24) L + 2^-22
  |lse - exact| <= 2 delta + 2^-20 (|lse| + 1);  |o - exact| <= (2 delta + weight + (keys + 64) 2^-24) A + |o| half a step of its type + keys 2^-126 max |V|:
a weight below 2^-126 is no number of 32 bits any more, in A it is one (a sum that the first run met: 2e-64 where every other term is 0).
"""

import itertools

import numpy as np
import pytest
import torch

import fp4_model as fp4
from tpa import tpa

pytestmark = pytest.mark.gpu
NONE, TOP_LEFT, BOTTOM_RIGHT = False, True, tpa.CAUSAL_BOTTOM_RIGHT


def problem(seed, b, lq, h, d, rq, rk, tokens, dtype, page=None, dv=None, scales=(125, 130)):
    """Queries, caches (pools and a table with `page`) on the host."""
    rng = np.random.default_rng(seed)
    dv = dv or d
    q = torch.from_numpy(rng.standard_normal((b, lq, rq, h + d), np.float32)).to(dtype)
    if page is None:
        shape, table = (b, tokens), None
    else:
        per_seq = -(-tokens // page)
        shape = (b * per_seq + 2, page)
        table = rng.permutation(b * per_seq + 2)[: b * per_seq].reshape(b, per_seq).astype(np.int32)
    return q, fp4.random_rows(rng, (*shape, rk), h, d, scales), fp4.random_rows(rng, (*shape, rk), h, dv, scales), table


def keys_of(lengths, causal, offset, lq, tokens, i, row):
    n = tokens if lengths is None else min(max(int(lengths[i]), 0), tokens)
    if causal is NONE:
        return n
    return max(0, min(n, row + offset + 1 + (n - lq if causal == BOTTOM_RIGHT and causal is not True else 0)))


def exact(q, kc, vc, table, h, d, dv, scale, lengths, causal, offset):
    q = q.double().numpy()
    b, lq, rq, _ = q.shape
    tokens = kc.shape[1] if table is None else table.shape[1] * kc.shape[1]
    o, a = np.full((2, b, lq, h, dv), np.nan)
    lse, big, lost = np.full((b, h, lq), -np.inf), np.zeros((b, h, lq)), 0.0
    for i in range(b):
        rows = [c[i] if table is None else c[table[i]].reshape(tokens, *c.shape[2:]) for c in (kc, vc)]
        (ka, kb), (va, vb) = fp4.read_rows(rows[0], h, d), fp4.read_rows(rows[1], h, dv)
        for row in range(lq):
            n = keys_of(lengths, causal, offset, lq, tokens, i, row)
            if n == 0:
                continue
            Q = np.einsum("rh,rd->hd", q[i, row, :, :h], q[i, row, :, h:]) / rq
            Qm = np.einsum("rh,rd->hd", abs(q[i, row, :, :h]), abs(q[i, row, :, h:])) / rq
            K, V = np.einsum("trh,trd->htd", ka[:n], kb[:n]) / ka.shape[1], np.einsum("trh,trd->htd", va[:n], vb[:n]) / ka.shape[1]
            Km, Vm = np.einsum("trh,trd->htd", abs(ka[:n]), abs(kb[:n])) / ka.shape[1], np.einsum("trh,trd->htd", abs(va[:n]), abs(vb[:n])) / ka.shape[1]
            lost = max(lost, n * 2.0**-126 * Vm.max())
            x = np.einsum("hd,htd->ht", Q, K) * scale
            most = x.max(-1, keepdims=True)
            p = np.exp(x - most)
            lse[i, :, row] = np.log(p.sum(-1)) + most[:, 0]
            p /= p.sum(-1, keepdims=True)
            o[i, row], a[i, row] = np.einsum("ht,htd->hd", p, V), np.einsum("ht,htd->hd", p, Vm)
            big[i, :, row] = (np.einsum("hd,htd->ht", Qm, Km) * abs(scale)).max(-1)
    return o, lse, a, big, tokens, lost


def compare(got, want, d, rq, rk, dtype):
    o, lse, a, big, keys, lost = want
    go, gl = got[0].double().cpu().numpy(), got[1].double().cpu().numpy()
    assert got[0].dtype == dtype and np.array_equal(np.isnan(go), np.isnan(o)) and np.array_equal(np.isinf(gl), np.isinf(lse))
    bf16 = dtype == torch.bfloat16
    delta = ((2.0**-17 if bf16 else 2.0**-24) + (d + 2 * rk + rq + 8) * 2.0**-24) * big + 2.0**-22
    with np.errstate(invalid="ignore"):
        assert not (abs(gl - lse) > 2 * delta + 2.0**-20 * (abs(lse) + 1)).any()
        t = (2 * delta.transpose(0, 2, 1)[..., None] + (2.0**-17 if bf16 else 2.0**-24) + (keys + 64) * 2.0**-24) * a + abs(o) * torch.finfo(dtype).eps / 2 + lost
        assert not (abs(go - o) > t).any(), np.nanmax(abs(go - o) / t)


def check(gpu, seed, b, lq, h, d, rq, rk, tokens, dtype, page=None, dv=None, lengths=None, causal=NONE, offset=0, scale=None, **options):
    q, kc, vc, table = problem(seed, b, lq, h, d, rq, rk, tokens, dtype, page, dv)
    scale = d**-0.5 if scale is None else scale
    dev = lambda x: None if x is None else torch.as_tensor(x).to(gpu)
    got = tpa.tpa_decode_fp4(dev(q[..., :h]), dev(q)[..., h:], dev(kc), dev(vc), scale, kv_lengths=None if lengths is None else dev(np.array(lengths, np.int32)),
                             page_table=dev(table), causal=causal, causal_offset=offset, v_head_dim=dv, **options)
    compare(got, exact(q, kc, vc, table, h, d, dv or d, scale, lengths, causal, offset), d, rq, rk, dtype)


BOTH = pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])


@BOTH
@pytest.mark.parametrize("rk", [1, 2, 4, 8])
@pytest.mark.parametrize("h,d", [(8, 64), (16, 128), (32, 128), (24, 64), (40, 128), (64, 64)])
def test_head_layouts_and_ranks(gpu, h, d, rk, dtype):
    check(gpu, h + rk, 3, 1, h, d, 6, rk, 200, dtype, page=64, lengths=[200, 1, 77])


@BOTH
@pytest.mark.parametrize("page", [1, 5, 16, 48, 64, 300])
def test_pages_of_any_size(gpu, page, dtype):
    check(gpu, page, 2, 2, 16, 64, 3, 2, 301, dtype, page=page, lengths=[301, 149], causal=BOTTOM_RIGHT)


@BOTH
@pytest.mark.parametrize("lq,h", [(1, 8), (3, 8), (4, 8), (5, 8), (2, 24), (7, 16), (4, 64), (64, 8)])
@pytest.mark.parametrize("causal,offset", [(NONE, 0), (TOP_LEFT, 0), (TOP_LEFT, 90), (BOTTOM_RIGHT, 0), (BOTTOM_RIGHT, -3), (TOP_LEFT, -2), (TOP_LEFT, 2**31 - 1), (BOTTOM_RIGHT, -(2**31))])
def test_rows_and_masks(gpu, lq, h, causal, offset, dtype):
    check(gpu, lq, 3, lq, h, 64, 6, 2, 131, dtype, lengths=[131, 0, lq + 1], causal=causal, offset=offset)


@BOTH
@pytest.mark.parametrize("tokens,lengths", [(1, None), (1, [0]), (2, [1]), (15, None), (16, None), (17, [-4]), (64, [99]), (129, None), (5000, None), (5000, [4999])])
def test_lengths_of_one_sequence(gpu, tokens, lengths, dtype):
    check(gpu, tokens, 1, 1, 8, 128, 6, 2, tokens, dtype, lengths=lengths)


@BOTH
def test_many_sequences_of_all_lengths(gpu, dtype):
    """More sequences than threads deal out, most of them shorter than a share, empty ones between and at both ends."""
    lengths = [(i * 37) % 90 if i % 5 else 0 for i in range(600)] + [0, 0]
    check(gpu, 0, len(lengths), 1, 8, 64, 1, 2, 90, dtype, page=16, lengths=lengths)


@BOTH
@pytest.mark.parametrize("h,d,dv,rk,rq", [(5, 33, 20, 3, 2), (1, 1, 1, 1, 1), (12, 64, 64, 2, 6), (16, 64, 128, 2, 6), (8, 96, 96, 6, 16), (3, 256, 255, 2, 1), (16, 64, 64, 16, 6)])
def test_other_shapes_on_the_vector_units(gpu, h, d, dv, rk, rq, dtype):
    check(gpu, h, 2, 3, h, d, rq, rk, 270, dtype, page=7, dv=dv, lengths=[270, 100], causal=BOTTOM_RIGHT)
    check(gpu, h, 2, 1, h, d, rq, rk, 270, dtype, dv=dv, lengths=[1, 0])


@BOTH
@pytest.mark.parametrize("scale", [0.0, -0.3, 2.0])
def test_scales(gpu, scale, dtype):
    check(gpu, 3, 2, 2, 16, 64, 40, 2, 100, dtype, scale=scale)
    check(gpu, 3, 2, 2, 16, 64, 40, 2, 100, dtype, scale=scale, kernel=1)


@BOTH
def test_numbers_that_are_not_finite(gpu, dtype):
    """NaN in a token that a row sees gives NaN; behind the lengths it is not read."""
    h, d, rk, tokens = 32, 64, 2, 150
    q, kc, vc, table = problem(5, 4, 1, h, d, 6, rk, tokens, dtype)
    at = d // 2 + h // 2
    kc[0, 120:, :, at:], vc[0, 120:, :, at:] = 255, 255   # behind the length
    kc[1, 40, 1, at] = 255                                # a block of b of K: every head's logit
    vc[2, 149, 0, at + 1] = 255                           # numbers 32 .. 63 of V
    kc[3, :, :, at:] = 255                                # every logit
    dev = lambda x: torch.as_tensor(x).to(gpu)
    lengths = np.array([120, 150, 150, 150], np.int32)
    for kernel in (0, 1):
        o, lse = tpa.tpa_decode_fp4(dev(q[..., :h]), dev(q[..., h:]), dev(kc), dev(vc), 0.1, kv_lengths=dev(lengths), kernel=kernel)
        o, lse = o.float().cpu(), lse.cpu()
        assert torch.isfinite(o[0]).all() and torch.isfinite(lse[0]).all()
        assert o[1].isnan().all() and lse[1].isnan().all() and o[3].isnan().all() and lse[3].isnan().all()
        assert torch.isfinite(o[2, ..., :32]).all() and o[2, ..., 32:].isnan().all() and torch.isfinite(lse[2]).all()


# heads of a few, of whole sets of 32 and of any number, whose rows a block has one behind the other
LAYOUTS = pytest.mark.parametrize("h,d,rk", [(8, 64, 2), (8, 128, 4), (16, 128, 1), (32, 64, 8), (32, 128, 2), (64, 64, 4), (64, 128, 1), (96, 128, 2), (128, 128, 2), (24, 64, 2), (40, 128, 8), (96, 64, 1), (160, 128, 2)])


@BOTH
@LAYOUTS
@pytest.mark.parametrize("page", [64, None])
def test_what_is_behind_the_last_token(gpu, h, d, rk, page, dtype):
    """The rest of a block, a page and a pool holds bytes that stand for NaN."""
    lengths, tokens = [1, 77, 192, 0, 33], 192
    q, kc, vc, table = problem(h, 5, 2, h, d, 6, rk, tokens, dtype, page)
    for i, n in enumerate(lengths):
        for t in range(n, tokens):
            at = (i, t) if page is None else (table[i, t // page], t % page)
            kc[at], vc[at] = 255, 255
    if page:
        for unused in set(range(len(kc))) - set(table.ravel()):
            kc[unused], vc[unused] = 255, 255
    dev = lambda x: None if x is None else torch.as_tensor(x).to(gpu)
    got = tpa.tpa_decode_fp4(dev(q[..., :h]), dev(q)[..., h:], dev(kc), dev(vc), 0.1, kv_lengths=dev(np.array(lengths, np.int32)), page_table=dev(table), causal=BOTTOM_RIGHT)
    compare(got, exact(q, kc, vc, table, h, d, d, 0.1, lengths, BOTTOM_RIGHT, 0), d, 6, rk, dtype)


@BOTH
@LAYOUTS
def test_every_scale_that_is_no_number(gpu, h, d, rk, dtype):
    """One scale byte of a row at a time, of K in one call and of V in another: what it belongs to is NaN and nothing else (the last sequence has none);
    scales far apart in V."""
    page, tokens, lq = 32, 128, 2
    first, scales = (d + 1) // 2 + h // 2, d // 32 + -(-h // 32)
    q, kc, vc, table = problem(h + 1, scales + 1, lq, h, d, 6, rk, tokens, dtype, page)
    vc = fp4.random_rows(np.random.default_rng(h + d), vc.shape[:-1], h, d, (90, 165))
    dev = lambda x: torch.as_tensor(x).to(gpu)
    for which in (0, 1):
        caches = [kc.copy(), vc.copy()]
        for i in range(scales):
            t = (31 * i + 5) % tokens
            caches[which][table[i, t // page], t % page, i % rk, first + i] = 255
        got = tpa.tpa_decode_fp4(dev(q[..., :h]), dev(q)[..., h:], dev(caches[0]), dev(caches[1]), 0.1, page_table=dev(table))
        want = exact(q, *caches, table, h, d, d, 0.1, None, NONE, 0)
        assert np.isnan(want[0]).any() and not np.isnan(want[0]).all()
        assert np.array_equal(np.isnan(got[1].cpu().numpy()), np.isnan(want[1]))
        compare(got, want, d, 6, rk, dtype)


@BOTH
@LAYOUTS
def test_rows_with_room_between_them(gpu, h, d, rk, dtype):
    """Rows of a wider array, one behind the other, at 4 bytes behind a 16-byte place."""
    q, kc, vc, table = problem(h + 2, 2, 3, h, d, 5, rk, 160, dtype, 32)
    dev = lambda x: torch.as_tensor(x).to(gpu)
    n = kc.shape[-1]
    wide = [torch.full((*c.shape[:-1], n + 20), 255, dtype=torch.uint8, device=gpu) for c in (kc, vc)]
    for x, c in zip(wide, (kc, vc)):
        x[..., 4 : 4 + n] = dev(c)
    got = tpa.tpa_decode_fp4(dev(q[..., :h]), dev(q)[..., h:], *(x[..., 4 : 4 + n] for x in wide), 0.1, kv_lengths=dev(np.array([160, 95], np.int32)), page_table=dev(table), causal=TOP_LEFT, causal_offset=120)
    compare(got, exact(q, kc, vc, table, h, d, d, 0.1, [160, 95], TOP_LEFT, 120), d, 5, rk, dtype)


@BOTH
@pytest.mark.parametrize("seed", range(24))
def test_shapes_that_nobody_picked(gpu, seed, dtype):
    rng = np.random.default_rng(1000 + seed)
    pick = lambda *x: x[int(rng.integers(len(x)))]
    h, d, rk, rq, lq, b = pick(8, 16, 24, 32, 40, 48, 56, 64, 96, 128, 7), pick(64, 128, 128, 64, 80), pick(1, 2, 2, 4, 8, 3), pick(1, 2, 6, 17), pick(1, 1, 2, 3, 6), int(rng.integers(1, 9))
    tokens, page = int(np.exp(rng.uniform(0, np.log(600)))), pick(None, 1, 3, 8, 16, 32, 64, 100)
    causal, offset = pick((NONE, 0), (TOP_LEFT, 40), (BOTTOM_RIGHT, 0), (BOTTOM_RIGHT, 2))
    check(gpu, seed, b, lq, h, d, rq, rk, tokens, dtype, page=page, lengths=rng.integers(-1, tokens + 2, b).tolist(), causal=causal, offset=offset, scale=float(rng.uniform(0.02, 0.3)))


@BOTH
def test_tables_with_pages_outside_the_pools(gpu, dtype):
    """They are read as the nearest page, and other sequences are not touched by them."""
    h, d, rk, page = 16, 64, 2, 8
    q, kc, vc, table = problem(6, 2, 1, h, d, 6, rk, 40, dtype, page)
    bad = table.copy()
    bad[1, 2], bad[1, 4] = -7, 2**31 - 1
    near = table.copy()
    near[1, 2], near[1, 4] = 0, len(kc) - 1
    dev = lambda x: torch.as_tensor(x).to(gpu)
    for kernel in (0, 1):
        got, want = (tpa.tpa_decode_fp4(dev(q[..., :h]), dev(q[..., h:]), dev(kc), dev(vc), 0.1, page_table=dev(t), kernel=kernel) for t in (bad, near))
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


@BOTH
def test_strides_and_odd_places(gpu, dtype):
    """Caches inside a wider array, ranks apart, rows at places that are no multiple of 4 (the vector units), queries at odd places."""
    b, h, d, rk, rq, tokens = 2, 16, 64, 2, 3, 70
    q, kc, vc, _ = problem(7, b, 2, h, d, rq, rk, tokens, dtype)
    want = exact(q, kc, vc, None, h, d, d, 0.125, None, BOTTOM_RIGHT, 0)
    n = kc.shape[-1]
    wide_q = torch.zeros(b, 2, rq + 1, h + d + 5, dtype=dtype, device=gpu)
    wide_q[:, :, 1:, 3 : 3 + h + d] = q.to(gpu)
    for first, step in ((4, 2 * n + 8), (1, 2 * n + 3)):
        wide = torch.zeros(tokens, rk, b, step, dtype=torch.uint8, device=gpu)
        k, v = (wide.permute(2, 0, 1, 3)[..., at : at + n] for at in (first, first + n + (0 if step % 4 else 4)))
        k.copy_(torch.from_numpy(kc))
        v.copy_(torch.from_numpy(vc))
        got = tpa.tpa_decode_fp4(wide_q[:, :, 1:, 3 : 3 + h], wide_q[:, :, 1:, 3 + h : 3 + h + d], k, v, 0.125, causal=BOTTOM_RIGHT)
        compare(got, want, d, rq, rk, dtype)


def test_the_same_whatever_the_neighbours_are(gpu):
    """Shares of the rounds change with the other sequences; results stay within their tolerance, and a call gives the same bits every time."""
    for b, lengths in itertools.product((1, 5), ([700], [700, 3, 0, 650, 1])):
        if len(lengths) == b:
            check(gpu, 11, b, 1, 32, 128, 6, 2, 700, torch.bfloat16, page=64, lengths=lengths)
    q, kc, vc, table = problem(12, 5, 1, 32, 128, 6, 2, 900, torch.bfloat16, 64)
    dev = lambda x: torch.as_tensor(x).to(gpu)
    args = (dev(q[..., :32]), dev(q[..., 32:]), dev(kc), dev(vc), 0.1)
    runs = [tpa.tpa_decode_fp4(*args, page_table=dev(table)) for _ in range(3)]
    assert all(torch.equal(x, y) for r in runs[1:] for x, y in zip(r, runs[0]))


def test_captured_with_its_own_workspace_and_another_stream(gpu):
    h, d, rk = 16, 64, 2
    q, kc, vc, table = problem(13, 3, 2, h, d, 6, rk, 130, torch.bfloat16, 16)
    dev = lambda x: torch.as_tensor(x).to(gpu)
    q, kc, vc, table, lengths = dev(q), dev(kc), dev(vc), dev(table), dev(np.array([130, 5, 64], np.int32))
    need = tpa.decode_fp4_workspace_bytes(q[..., :h], q[..., h:], kc, vc, page_table=table)
    ws = torch.zeros(need, dtype=torch.uint8, device=gpu)
    call = lambda: tpa.tpa_decode_fp4(q[..., :h], q[..., h:], kc, vc, 0.1, workspace=ws, kv_lengths=lengths, page_table=table, causal=BOTTOM_RIGHT)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        call()
    torch.cuda.current_stream().wait_stream(stream)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call()
    for i in range(4):
        lengths.copy_(torch.tensor([130 - 7 * i, 5 + i, 0 if i == 2 else 64], dtype=torch.int32))
        want = tpa.tpa_decode_fp4(q[..., :h], q[..., h:], kc, vc, 0.1, kv_lengths=lengths, page_table=table, causal=BOTTOM_RIGHT)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(x.nan_to_num(7), y.nan_to_num(7)) for x, y in zip(out, want))


def test_offsets_past_32_bits(gpu):
    """A pool of more than 4 GB, with the sequence's pages at both of its ends."""
    h, d, rk, page = 32, 128, 2, 64
    n = fp4.row_bytes(h, d)
    pages = (5 << 30) // (page * rk * n)
    rng = np.random.default_rng(1)
    small = [fp4.random_rows(rng, (4, page, rk), h, d) for _ in range(2)]
    pools = [torch.empty(pages, page, rk, n, dtype=torch.uint8, device=gpu) for _ in range(2)]
    at = np.array([0, pages - 1, pages // 2, pages - 2])
    for pool, rows in zip(pools, small):
        pool[torch.from_numpy(at).to(gpu)] = torch.from_numpy(rows).to(gpu)
    q = torch.from_numpy(rng.standard_normal((1, 1, 6, h + d), np.float32)).to(torch.bfloat16)
    got = tpa.tpa_decode_fp4(q[..., :h].to(gpu), q[..., h:].to(gpu), *pools, 0.1, page_table=torch.from_numpy(at[None].astype(np.int32)).to(gpu))
    compare(got, exact(q, *small, np.arange(4)[None], h, d, d, 0.1, None, NONE, 0), d, 6, rk, torch.bfloat16)
    # writing and reading at those ends
    k = torch.randn(1, 4, rk, h + d, generator=torch.Generator().manual_seed(2)).to(gpu)
    slots = torch.tensor([[5, pages * page - 1, (pages // 2) * page + 9, (pages - 2) * page]], dtype=torch.int32, device=gpu)
    tpa.tpa_cache_write_fp4(k, k, h, *pools, slots)
    rows = np.stack([fp4.write_row(r[:h], r[h:]) for r in k.reshape(-1, h + d).cpu().numpy()])
    want = np.concatenate(fp4.read_rows(np.maximum(rows, 0), h, d), -1).reshape(k.shape)
    for x in tpa.tpa_cache_read_fp4(*pools, h, slots, head_dim=d, dtype=torch.float32):
        assert np.array_equal(x.double().cpu().numpy(), want)


def test_empty_calls(gpu):
    rows = fp4.row_bytes(8, 64)
    kc = torch.zeros(2, 0, 2, rows, dtype=torch.uint8, device=gpu)
    q = torch.ones(2, 3, 1, 72, device=gpu)
    o, lse = tpa.tpa_decode_fp4(q[..., :8], q[..., 8:], kc, kc, 1.0)
    assert o.shape == (2, 3, 8, 64) and o.isnan().all() and (lse == -float("inf")).all()
    kc = torch.zeros(0, 4, 2, rows, dtype=torch.uint8, device=gpu)
    o, lse = tpa.tpa_decode_fp4(q[:0, ..., :8], q[:0, ..., 8:], kc, kc, 1.0)
    assert o.shape == (0, 3, 8, 64) and lse.shape == (0, 8, 3)
