"""tpa_cache_write_fp4 and tpa_cache_read_fp4 against the definition.  Both are exact arithmetic: bytes and numbers have to be equal."""

import numpy as np
import pytest
import torch

import fp4_model as fp4
from tpa import tpa

pytestmark = pytest.mark.gpu

SIZES = [(8, 64, 64), (32, 128, 128), (24, 128, 64), (64, 64, 64), (16, 40, 72), (5, 33, 7), (1, 1, 1), (33, 96, 31)]


def write(gpu, k, v, h, slots, pages, page, seed=0):
    """Pools of random bytes after the call, and before it."""
    rng = np.random.default_rng(seed)
    rk, dk, dv = k.shape[2], k.shape[3] - h, v.shape[3] - h
    before = [rng.integers(0, 256, (pages, page, rk, fp4.row_bytes(h, d)), dtype=np.uint8) for d in (dk, dv)]
    pools = [torch.from_numpy(x.copy()).to(gpu) for x in before]
    assert tpa.tpa_cache_write_fp4(k, v, h, *pools, torch.as_tensor(slots, device=gpu)) is None
    return [x.cpu().numpy() for x in pools], before


def check_written(after, before, x, h, slots):
    want = before.astype(np.int64)
    page = before.shape[1]
    written = np.zeros(before.shape[:2], bool)
    x = x.float().cpu().numpy()
    for b, i in np.ndindex(slots.shape):
        s = int(slots[b, i])
        if 0 <= s < before.shape[0] * page:
            written[s // page, s % page] = True
            for r in range(x.shape[2]):
                row = fp4.write_row(x[b, i, r, :h], x[b, i, r, h:])
                want[s // page, s % page, r] = np.where(row < 0, after[s // page, s % page, r], row)
    assert np.array_equal(after, want)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("h,dk,dv", SIZES)
def test_rows_are_the_definitions(gpu, h, dk, dv, dtype):
    g = torch.Generator().manual_seed(h + dk)
    b, l, rk, pages, page = 2, 7, 3, 5, 6
    k, v = (torch.randn(b, l, rk, h + d, generator=g).mul(torch.exp(3 * torch.randn(b, l, rk, 1, generator=g))).to(dtype).to(gpu) for d in (dk, dv))
    slots = torch.randperm(pages * page, generator=g)[: b * l].view(b, l).to(torch.int32).numpy()
    slots[0, 2], slots[1, 0], slots[1, 6] = -1, pages * page, 2**31 - 1  # none, behind the pools
    after, before = write(gpu, k, v, h, slots, pages, page)
    for a, was, x in zip(after, before, (k, v)):
        check_written(a, was, x, h, slots)
    got = tpa.tpa_cache_read_fp4(*(torch.from_numpy(a).to(gpu) for a in after), h, torch.from_numpy(slots).to(gpu), head_dim=dk, v_head_dim=dv, dtype=dtype)
    for a, x, d in zip(after, got, (dk, dv)):
        assert x.dtype == dtype
        flat = np.concatenate([a.reshape(-1, *a.shape[2:]), np.zeros_like(a[:1, 0])])
        want = np.concatenate(fp4.read_rows(flat[np.where((slots >= 0) & (slots < pages * page), slots, -1)], h, d), -1)
        assert np.array_equal(x.double().cpu().numpy(), want)


def test_borders_of_the_levels(gpu):
    """Values on and beside every border, at scales from the smallest to the largest, both signs."""
    borders = np.concatenate([(fp4.LEVELS[1:] + fp4.LEVELS[:-1]) / 2, fp4.LEVELS[1:], [7.25, 7.5]]).astype(np.float32)
    near = np.concatenate([np.nextafter(borders, np.float32(0)), borders, np.nextafter(borders, np.float32(99))])
    blocks = []
    for e in (-149, -126, -125, -3, 0, 1, 60, 124, 125):
        for x in near:
            with np.errstate(under="ignore", over="ignore"):
                blocks.append(np.resize(np.concatenate([[x], near[near <= x]]), 32).astype(np.float32) * np.float32(2.0) ** np.float32(e))
    x = np.stack(blocks)
    x = x[np.isfinite(x).all(-1)]
    x[::2] *= -1
    n = len(x)
    k = torch.from_numpy(np.concatenate([x, x], -1)).view(1, n, 1, 64).to(gpu)  # h = d = 32
    slots = np.arange(n, dtype=np.int32)[None]
    after, before = write(gpu, k, k, 32, slots, n, 1)
    check_written(after[0], before[0], k, 32, slots)
    assert np.array_equal(after[0][..., :34], after[1][..., :34])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_zeros_and_numbers_that_are_not_finite(gpu, dtype):
    h, d = 40, 64
    k = torch.randn(1, 6, 2, h + d, generator=torch.Generator().manual_seed(1)).to(dtype)
    k[0, 0, 0] = 0
    k[0, 1, 0, 3] = float("nan")       # the first block of a
    k[0, 2, 1, 39] = float("inf")      # the second, short one
    k[0, 3, 0, h + 33] = -float("inf")  # the second of b
    k = k.to(gpu)
    slots = np.arange(6, dtype=np.int32)[None]
    after, before = write(gpu, k, k, h, slots, 2, 3)
    check_written(after[0], before[0], k, h, slots)
    got, _ = tpa.tpa_cache_read_fp4(*(torch.from_numpy(a).to(gpu) for a in after), h, torch.from_numpy(slots).to(gpu), head_dim=d, dtype=dtype)
    nan = got.isnan().cpu()
    want = torch.zeros_like(nan)
    want[0, 1, 0, :32] = want[0, 2, 1, 32:40] = want[0, 3, 0, h + 32 : h + 64] = True
    assert torch.equal(nan, want) and got[0, 0, 0].abs().max() == 0


def test_strided_factors_and_pools_other_integers_other_streams(gpu):
    h, d, rk = 16, 64, 2
    base = torch.randn(2, 9, 2 * rk, h + d + 3, generator=torch.Generator().manual_seed(2)).to(gpu)
    k, v = base[:, 1:8, ::2, 1 : 1 + h + d], base[:, 1:8, 1::2, 3:]  # rows at odd places
    wide = torch.zeros(4, 7, rk, 2 * fp4.row_bytes(h, d) + 1, dtype=torch.uint8, device=gpu)
    kc, vc = wide[..., : fp4.row_bytes(h, d)], wide[..., fp4.row_bytes(h, d) : 2 * fp4.row_bytes(h, d)]
    slots = torch.randperm(28, generator=torch.Generator().manual_seed(3))[:14].view(2, 7).to(gpu)  # int64
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        tpa.tpa_cache_write_fp4(k, v, h, kc, vc, slots)
        got = tpa.tpa_cache_read_fp4(kc, vc, h, slots, head_dim=d, dtype=torch.float32)
    torch.cuda.current_stream().wait_stream(stream)
    for x, y in zip(got, (k, v)):
        rows = np.stack([fp4.write_row(r[:h], r[h:]) for r in y.reshape(-1, h + d).cpu().numpy()])
        want = np.concatenate(fp4.read_rows(np.maximum(rows, 0), h, d), -1).reshape(y.shape)
        assert np.array_equal(x.double().cpu().numpy(), want)
    assert wide[..., -1].max() == 0


def test_no_tokens_and_no_pages(gpu):
    rows = fp4.row_bytes(8, 64)
    empty, none = torch.empty(1, 0, 2, 72, device=gpu), torch.empty(1, 0, dtype=torch.int32, device=gpu)
    pools = [torch.zeros(2, 4, 2, rows, dtype=torch.uint8, device=gpu) for _ in range(2)]
    tpa.tpa_cache_write_fp4(empty, empty, 8, *pools, none)
    assert tpa.tpa_cache_read_fp4(*pools, 8, none, head_dim=64)[0].shape == (1, 0, 2, 72)
    no_pages = [p[:0] for p in pools]
    k, slot = torch.ones(1, 1, 2, 72, device=gpu), torch.zeros(1, 1, dtype=torch.int32, device=gpu)
    tpa.tpa_cache_write_fp4(k, k, 8, *no_pages, slot)
    assert tpa.tpa_cache_read_fp4(*no_pages, 8, slot, head_dim=64)[0].abs().max() == 0
