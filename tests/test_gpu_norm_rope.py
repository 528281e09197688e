"""tpa_norm_rope, its gradients and its form that writes into a paged cache, against the formulas in 64 bits on dense head vectors.

Tolerances.  One rounding to the result's type is off by half a step: 2^-8 (bf16) or 2^-24 (fp32) of the value.  Before it, sums in
32 bits (64 for the norms of fp32 factors) are off by at most their length times 2^-24 of the sum of their terms' sizes:
  b':  three roundings of |w| (|b0| + |b1|) under the rotation.
  a':  s = n^-1/2 carries half the relative error of n = |X_h|^2 / D + eps: `kappa`, the sum of the terms' sizes over n, times
       (D + R^2) 2^-25, and six more roundings.
  db:  M = sum_h w_h a a^T and the mixture of the b rows: H + R + 3 (relative error of s) + 16 roundings of the sum of the terms' sizes; the
       matrix-core kernel splits M and w a into two bf16 numbers, 2^-16 each of the same sum.
  da:  the same with the sum over the ranks in place of the heads.
  d weight: chains of at most 128 terms.
"""

import numpy as np
import pytest
import torch

from tpa import tpa

pytestmark = pytest.mark.gpu
U = 2.0**-24


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def rope(rope_len, d):
    ang = torch.arange(rope_len, dtype=torch.float64)[:, None] * 10000.0 ** (-torch.arange(0, d, 2, dtype=torch.float64) / d)
    return ang.cos().float(), ang.sin().float()


def turned(x, cos, sin):
    a, b = x[..., 0::2], x[..., 1::2]
    return torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)


def angles(positions, sections, cos, sin, d):
    """cos, sin [b, l, 1, d/2] in 64 bits: pair j by its axis' position, pairs past the last section by none."""
    n = cos.shape[0]
    c, s = torch.ones((*positions.shape[:2], d // 2), dtype=torch.float64), torch.zeros((*positions.shape[:2], d // 2), dtype=torch.float64)
    j = 0
    for axis, count in enumerate(sections):
        at = positions[..., axis].long().clamp(0, n - 1)
        c[..., j : j + count], s[..., j : j + count] = cos.double()[at][..., j : j + count], sin.double()[at][..., j : j + count]
        j += count
    return c[:, :, None], s[:, :, None]


def side(x, h, weight, c, s, eps, normalize, dy=None):
    """Results and tolerances' ingredients of one side; x[b, l, r, h + d] in 64 bits."""
    r, d = x.shape[2], x.shape[3] - h
    a, b = x[..., :h], x[..., h:]
    dense = torch.matmul(a.transpose(2, 3), b) / r
    n = dense.square().mean(-1) + eps
    scale = n.rsqrt() if normalize else torch.ones_like(n)
    sizes = torch.matmul(a.abs().transpose(2, 3), b.abs()) / r  # [.., h, d]
    kappa = (sizes.square().mean(-1) + eps) / n if normalize else torch.zeros_like(n)
    out = torch.cat([a * scale[:, :, None], turned(b * weight, c, s)], -1)
    size = turned((b * weight).abs(), c.abs(), -s.abs())
    even, odd = (b * weight).abs()[..., 0::2], (b * weight).abs()[..., 1::2]
    size = torch.stack([even * c.abs() + odd * s.abs(), odd * c.abs() + even * s.abs()], -1).flatten(-2)
    rel_s = (d + r * r) * U / 2 * kappa + 6 * U
    slack = torch.cat([(a * scale[:, :, None]).abs() * rel_s[:, :, None], 4 * U * size], -1)
    if dy is None:
        return out, slack
    da, e = dy[..., :h], turned(dy[..., h:], c, -s)
    even, odd = dy[..., h:].abs()[..., 0::2], dy[..., h:].abs()[..., 1::2]
    e_size = torch.stack([even * c.abs() + odd * s.abs(), odd * c.abs() + even * s.abs()], -1).flatten(-2)
    u = (da * a).sum(2)
    w = -(scale**3) * u / (d * r * r) if normalize else torch.zeros_like(u)
    w_size = scale**3 * (da * a).abs().sum(2) / (d * r * r) if normalize else torch.zeros_like(u)
    g, g_size = torch.matmul(b, b.transpose(2, 3)), torch.matmul(b.abs(), b.abs().transpose(2, 3))
    m, m_size = torch.matmul(a * w[:, :, None], a.transpose(2, 3)), torch.matmul(a.abs() * w_size[:, :, None], a.abs().transpose(2, 3))
    grad = torch.cat([da * scale[:, :, None] + w[:, :, None] * torch.matmul(g, a), e * weight + torch.matmul(m, b)], -1)
    worst = rel_s.amax(-1)[:, :, None, None]
    split = 2 * 2.0**-16
    g_slack = torch.cat([(da * scale[:, :, None]).abs() * (rel_s[:, :, None] + U) + w_size[:, :, None] * torch.matmul(g_size, a.abs()) * (3 * worst + (d + 2 * r + 16) * U),
                         4 * U * e_size * weight.abs() + torch.matmul(m_size, b.abs()) * (3 * worst + (h + 2 * r + 16) * U + split)], -1)
    return out, slack, grad, g_slack, (e * b).sum((0, 1, 2)), 128 * U * (e_size * b.abs()).sum((0, 1, 2))


def make(seed, b, l, h, d, rq, rk, dtype, axes=1, weights=torch.float32, rope_len=97):
    g = torch.Generator().manual_seed(seed)
    n = lambda *s: torch.randn(s, generator=g)
    x = {k: n(b, l, r, h + d).to(dtype) for k, r in (("q", rq), ("k", rk), ("v", rk), ("dq", rq), ("dk", rk))}
    x["wq"], x["wk"] = ((1 + 0.3 * n(d)).to(weights) for _ in range(2))
    x["pos"] = torch.randint(-3, rope_len + 3, (b, l, axes), generator=g).to(torch.int32)
    x["cos"], x["sin"] = rope(rope_len, d)
    return x


def near(got, want, slack, dtype, name):
    got = got.detach().cpu().double()
    tol = half_step(dtype) * want.abs() + slack * (1 + half_step(dtype)) + 1e-37
    bad = (got - want).abs() > tol
    assert got.shape == want.shape and not bad.any(), (name, int(bad.sum()), (got - want).abs()[bad].max().item(), (tol[bad]).min().item())


SHAPES = [
    # b, l, h, d, rq, rk, sections
    (1, 1, 8, 64, 6, 2, None),              # one token
    (3, 37, 16, 128, 6, 2, None),           # an odd number of tokens
    (2, 19, 32, 128, 1, 1, None),           # sixteen tokens to a tile of rows
    (1, 70, 24, 64, 3, 4, [8, 12, 12]),     # three axes
    (2, 9, 64, 64, 16, 8, [8, 12, 8]),      # ranks that fill the tile; four pairs that do not turn
    (1, 33, 40, 128, 5, 7, [16, 24, 16, 8]),  # four axes, ranks between the kernels' own
    (1, 3, 72, 128, 9, 12, [64]),           # more heads than lanes
    (2, 5, 8, 128, 2, 6, [0, 64]),          # an axis without pairs
    (1, 2, 8, 64, 16, 16, []),
]
ANY = [
    (2, 7, 3, 10, 5, 2, [2, 1]),            # odd heads, a head size of no kernel
    (1, 4, 8, 64, 17, 20, None),            # ranks past a tile
    (1, 5, 16, 128, 6, 2, [15, 24, 25]),    # axes that end inside a chunk of pairs
    (1, 2, 1, 2, 1, 1, None),
    (1, 2, 130, 256, 24, 30, None),         # the most LDS
]
CASES = [(s, 0) for s in SHAPES] + [(s, 1) for s in SHAPES] + [(s, 0) for s in ANY]


def call(x, h, sections, gpu, **more):
    axes = sections or [x["cos"].shape[1]]
    pos = x["pos"].to(gpu)
    return dict(num_heads=h, rope_cos=x["cos"].to(gpu), rope_sin=x["sin"].to(gpu), q_weight=x["wq"].to(gpu), k_weight=x["wk"].to(gpu),
                positions=pos if len(axes) > 1 else pos[..., 0], sections=sections or None, **more)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("shape,kernel", CASES)
def test_forward_and_gradients(gpu, dtype, shape, kernel):
    b, l, h, d, rq, rk, sections = shape
    x = make(b * 1000 + l, b, l, h, d, rq, rk, dtype, axes=len(sections or [0]))
    kw = call(x, h, sections, gpu, kernel=kernel)
    q, k = (x[n].to(gpu).requires_grad_() for n in ("q", "k"))
    kw["q_weight"].requires_grad_()
    kw["k_weight"].requires_grad_()
    got = tpa.tpa_norm_rope(q, k, **kw)
    grads = torch.autograd.grad(got, (q, k, kw["q_weight"], kw["k_weight"]), (x["dq"].to(gpu), x["dk"].to(gpu)))
    c, s = angles(x["pos"], sections or [d // 2], x["cos"], x["sin"], d)
    for i, n in enumerate("qk"):
        out, slack, grad, g_slack, dw, w_slack = side(x[n].double(), h, x["w" + n].double(), c, s, 1e-6, True, x["d" + n].double())
        near(got[i], out, slack, dtype, n)
        near(grads[i], grad, g_slack, dtype, "d" + n)
        near(grads[2 + i], dw, w_slack, torch.float32, "dw" + n)
    direct = tpa.tpa_norm_rope_bwd(q.detach(), k.detach(), dq_out=x["dq"].to(gpu), dk_out=x["dk"].to(gpu), **kw)
    assert all(torch.equal(g, w) for g, w in zip(direct, grads))


@pytest.mark.parametrize("kernel", [0, 1])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_without_norms_weights_or_positions(gpu, dtype, kernel):
    """No weights are ones, no positions are 0 .. l - 1, without norms the head factors pass through untouched; bf16 weights."""
    b, l, h, d, rq, rk = 2, 21, 16, 64, 6, 2
    x = make(7, b, l, h, d, rq, rk, dtype, weights=torch.bfloat16)
    cos, sin = x["cos"].to(gpu), x["sin"].to(gpu)
    q, k = x["q"].to(gpu), x["k"].to(gpu)
    x["pos"] = torch.arange(l, dtype=torch.int32)[None, :, None].expand(b, l, 1)
    c, s = angles(x["pos"], [d // 2], x["cos"], x["sin"], d)
    ones = torch.ones(d, dtype=torch.float64)
    for normalize in (False, True):
        got = tpa.tpa_norm_rope(q, k, h, cos, sin, normalize=normalize, kernel=kernel)
        for i, n in enumerate("qk"):
            out, slack = side(x[n].double(), h, ones, c, s, 1e-6, normalize)
            near(got[i], out, slack, dtype, (n, normalize))
            if not normalize:
                assert torch.equal(got[i][..., :h].cpu(), x[n][..., :h])
    got = tpa.tpa_norm_rope_bwd(q, k, h, cos, sin, x["dq"].to(gpu), x["dk"].to(gpu), q_weight=x["wq"].to(gpu), normalize=False, kernel=kernel)
    _, _, grad, g_slack, dw, w_slack = side(x["q"].double(), h, x["wq"].double(), c, s, 1e-6, False, x["dq"].double())
    near(got[0], grad, g_slack, dtype, "dq")
    near(got[2], dw, w_slack, torch.bfloat16, "dw")
    assert got[3] is None and got[2].dtype == torch.bfloat16
    near(got[1], *side(x["k"].double(), h, ones, c, s, 1e-6, False, x["dk"].double())[2:4], dtype, "dk")


def test_gradients_against_differences(gpu):
    """The gradient along a direction is the difference quotient of a loss in fp32: (f(x + t v) - f(x - t v)) / 2 t, off by t^2 times the third
    derivative along v and by the roundings of f over t; with t = 1/64 and unit directions both are below 2^-9 of the sizes here."""
    b, l, h, d, rq, rk = 1, 12, 8, 64, 6, 2
    x = make(3, b, l, h, d, rq, rk, torch.float32)
    cos, sin, pos = x["cos"].to(gpu), x["sin"].to(gpu), x["pos"][..., 0].to(gpu)
    leaves = [x[n].to(gpu).requires_grad_() for n in ("q", "k", "wq", "wk")]
    up = [x[n].to(gpu).double() for n in ("dq", "dk")]

    def loss(q, k, wq, wk):
        out = tpa.tpa_norm_rope(q, k, h, cos, sin, wq, wk, pos)
        return sum((o.double() * u).sum() for o, u in zip(out, up))

    grads = torch.autograd.grad(loss(*leaves), leaves)
    g = torch.Generator().manual_seed(9)
    for i, leaf in enumerate(leaves):
        v = torch.randn(leaf.shape, generator=g).to(gpu)
        v /= v.norm()
        t = 1 / 64
        moved = [[y.detach() + (sign * t * v if j == i else 0) for j, y in enumerate(leaves)] for sign in (1, -1)]
        quotient = (loss(*moved[0]) - loss(*moved[1])).item() / (2 * t)
        want = (grads[i].double() * v.double()).sum().item()
        assert abs(quotient - want) <= 2.0**-9 * grads[i].double().norm().item() + 1e-3, (i, quotient, want)


@pytest.mark.parametrize("kernel", [0, 1])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("shape", [(1, 1, 32, 128, 6, 2), (1, 45, 16, 64, 6, 4), (3, 11, 8, 64, 1, 1), (1, 30, 64, 64, 16, 8), (1, 6, 24, 128, 3, 5)])
def test_write_into_a_paged_cache(gpu, dtype, kernel, shape):
    """K and V factors land in their slots, bit for bit what tpa_norm_rope gives; slots outside the pools are dropped, nothing else is touched."""
    b, l, h, d, rq, rk = shape
    x = make(11, b, l, h, d, rq, rk, dtype)
    kw = call(x, h, None, gpu, kernel=kernel)
    page, pages = 16, b * l // 16 + 3
    slots = torch.randperm(pages * page, generator=torch.Generator().manual_seed(5))[: b * l].view(b, l)
    dropped = torch.arange(b * l).view(b, l) % 5 == 4
    slots[dropped] = torch.tensor([-1, pages * page, -(2**31), 2**31 - 1]).repeat(b * l)[: int(dropped.sum())]
    pools = [torch.full((pages, page, rk, w), float("nan"), dtype=dtype, device=gpu) for w in (h, d, h, d)]
    q, k, v = (x[n].to(gpu) for n in "qkv")
    got = tpa.tpa_norm_rope_write(q, k, v, h, kw["rope_cos"], kw["rope_sin"], *pools, slots.to(gpu), kw["q_weight"], kw["k_weight"], kw["positions"], kernel=kernel)
    want_q, want_k = tpa.tpa_norm_rope(q, k, **kw)
    assert torch.equal(got, want_q)
    at = slots[~dropped].to(gpu)
    for pool, want in zip(pools, (want_k[..., :h], want_k[..., h:], v[..., :h], v[..., h:])):
        flat = pool.flatten(0, 1)
        assert torch.equal(flat[at], want[~dropped.to(gpu)])
        rest = torch.ones(pages * page, dtype=torch.bool, device=gpu)
        rest[at] = False
        assert flat[rest].isnan().all()


def test_contiguous_cache_as_pool_and_views(gpu):
    """Pages may be the batch entries of a contiguous cache, arrays may be views with gaps; inputs may be expanded."""
    b, l, h, d, rq, rk, cache = 2, 5, 8, 64, 6, 2, 12
    x = make(13, b, l, h, d, rq, rk, torch.bfloat16)
    kw = call(x, h, None, gpu)
    wide = torch.zeros((b, cache + 2, rk, 2 * (h + d) + 16), dtype=torch.bfloat16, device=gpu)[:, 1:-1]
    pools = [wide[..., :h], wide[..., h : h + d], wide[..., h + d : 2 * h + d], wide[..., 2 * h + d : 2 * (h + d)]]
    slots = torch.arange(l, device=gpu)[None] + cache * torch.arange(b, device=gpu)[:, None] + 3
    q = x["q"].to(gpu)[:, :, :1].expand(b, l, rq, h + d)
    k = torch.zeros((b, 2 * l, rk + 1, h + d + 8), dtype=torch.bfloat16, device=gpu)[:, ::2, 1:, 8:]
    k.copy_(x["k"].to(gpu))
    got = tpa.tpa_norm_rope_write(q, k, x["v"].to(gpu), h, kw["rope_cos"], kw["rope_sin"], *pools, slots, kw["q_weight"], kw["k_weight"], kw["positions"])
    want_q, want_k = tpa.tpa_norm_rope(q.contiguous(), k.contiguous(), **kw)
    assert torch.equal(got, want_q)
    assert torch.equal(torch.cat([pools[0], pools[1]], -1)[:, 3 : 3 + l], want_k) and torch.equal(torch.cat([pools[2], pools[3]], -1)[:, 3 : 3 + l], x["v"].to(gpu))
    assert not wide[:, :3].any() and not wide[:, 3 + l :].any() and not wide[..., 2 * (h + d) :].any()


@pytest.mark.parametrize("kernel", [0, 1])
def test_special_values_stay_in_their_token(gpu, kernel):
    """Zeros, infinities and NaN in one token: its own results follow the formula, the other tokens of its tile do not change."""
    b, l, h, d, rq, rk = 1, 8, 8, 64, 2, 2
    x = make(17, b, l, h, d, rq, rk, torch.bfloat16)
    kw = call(x, h, None, gpu, kernel=kernel)
    q, k = x["q"].clone(), x["k"]
    want = tpa.tpa_norm_rope(q.to(gpu), k.to(gpu), **kw)[0]
    q[0, 2] = 0
    q[0, 4, 1, h + 3] = float("inf")
    q[0, 6, 0, 1] = float("nan")
    got = tpa.tpa_norm_rope(q.to(gpu), k.to(gpu), **kw)[0]
    for t in (0, 1, 3, 5, 7):
        assert torch.equal(got[0, t], want[0, t])
    assert not got[0, 2].any()
    assert got[0, 6, :, 1].isnan().all() and torch.equal(got[0, 6, :, 2:], want[0, 6, :, 2:])
    assert torch.equal(got[0, 4, 0, h:], want[0, 4, 0, h:])
    dq = x["dq"].to(gpu)
    _, _, dw, _ = clean = tpa.tpa_norm_rope_bwd(x["q"].to(gpu), k.to(gpu), dq_out=dq, dk_out=x["dk"].to(gpu), **kw)
    got = tpa.tpa_norm_rope_bwd(q.to(gpu), k.to(gpu), dq_out=dq, dk_out=x["dk"].to(gpu), **kw)
    for t in (0, 1, 3, 5, 7):
        assert torch.equal(got[0][0, t], clean[0][0, t])
    assert torch.equal(got[1], clean[1]) and torch.equal(got[3], clean[3])


def test_no_tokens_and_gradients_of_one_output(gpu):
    h, d = 8, 64
    x = make(19, 2, 6, h, d, 6, 2, torch.bfloat16)
    kw = call(x, h, None, gpu)
    none = dict(kw, positions=kw["positions"][:, :0])
    q0, k0 = x["q"].to(gpu)[:, :0], x["k"].to(gpu)[:, :0]
    assert [t.shape for t in tpa.tpa_norm_rope(q0, k0, **none)] == [q0.shape, k0.shape]
    w = kw["q_weight"].clone().requires_grad_()
    out = tpa.tpa_norm_rope(q0, k0, **dict(none, q_weight=w))
    assert not torch.autograd.grad(out[0].sum() + out[1].sum(), w)[0].any()
    q, k = (x[n].to(gpu).requires_grad_() for n in "qk")
    whole = tpa.tpa_norm_rope_bwd(q.detach(), k.detach(), dq_out=x["dq"].to(gpu), dk_out=x["dk"].to(gpu), **kw)
    out = tpa.tpa_norm_rope(q, k, **kw)
    got = torch.autograd.grad(out[1], (q, k), x["dk"].to(gpu), allow_unused=True)
    assert got[0] is None and torch.equal(got[1], whole[1])
    # an expanded gradient, as a sum gives it, and a broadcast input, whose gradient is summed
    g = torch.autograd.grad(tpa.tpa_norm_rope(q, k, **kw)[0].sum(), q)[0]
    assert torch.equal(g, tpa.tpa_norm_rope_bwd(q.detach(), k.detach(), dq_out=torch.ones_like(q), dk_out=x["dk"].to(gpu), **kw)[0])
    one = x["q"].to(gpu)[:1].float().requires_grad_()
    kw32 = dict(kw, positions=kw["positions"][:1].expand(2, 6).contiguous())
    g = torch.autograd.grad(tpa.tpa_norm_rope(one.expand(2, -1, -1, -1), k.detach().float(), **kw32)[0], one, x["dq"].to(gpu).float())[0]
    parts = tpa.tpa_norm_rope_bwd(one.detach().expand(2, -1, -1, -1), k.detach().float(), dq_out=x["dq"].to(gpu).float(), dk_out=x["dk"].to(gpu).float(), **kw32)[0]
    assert torch.equal(g, parts.sum(0, keepdim=True))


def test_replays_from_a_graph(gpu):
    """Forward and backward calls captured once and replayed, with eager work between, give the eager results bit for bit."""
    h, d = 16, 128
    x = make(23, 2, 50, h, d, 6, 2, torch.bfloat16)
    kw = call(x, h, None, gpu)
    q, k, dq, dk = (x[n].to(gpu) for n in ("q", "k", "dq", "dk"))
    pools = [torch.zeros((8, 16, 2, w), dtype=torch.bfloat16, device=gpu) for w in (h, d, h, d)]
    slots = torch.arange(100, dtype=torch.int32, device=gpu).view(2, 50)

    def work():
        return (*tpa.tpa_norm_rope(q, k, **kw), *tpa.tpa_norm_rope_bwd(q, k, dq_out=dq, dk_out=dk, **kw),
                tpa.tpa_norm_rope_write(q, k, k, h, kw["rope_cos"], kw["rope_sin"], *pools, slots, kw["q_weight"], kw["k_weight"], kw["positions"]))

    eager = [t.clone() for t in (*work(), *pools)]
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        work()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            captured = work()
    for _ in range(3):
        for t in (*captured, *pools):
            t.zero_()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(g, w) for g, w in zip((*captured, *pools), eager))


@pytest.mark.parametrize("given", [(), ("wq",), ("wk",), ("wq", "wk")])
def test_autograd_with_and_without_weights(gpu, given):
    """torch.autograd gives the backward call's gradients, to the weights that are there and no others."""
    h, d = 8, 64
    x = make(37, 2, 9, h, d, 6, 2, torch.bfloat16)
    kw = dict(call(x, h, None, gpu), q_weight=None, k_weight=None, positions=None)
    for n in given:
        kw[n[1] + "_weight"] = x[n].to(gpu)
    q, k, dq, dk = (x[n].to(gpu) for n in ("q", "k", "dq", "dk"))
    want = [g for g in tpa.tpa_norm_rope_bwd(q, k, dq_out=dq, dk_out=dk, **kw) if g is not None]
    leaves = [t.requires_grad_() for t in (q, k, kw["q_weight"], kw["k_weight"]) if t is not None]
    got = torch.autograd.grad(tpa.tpa_norm_rope(q, k, **kw), leaves, (dq, dk))
    assert len(got) == len(want) == 2 + len(given) and all(torch.equal(a, b) for a, b in zip(got, want))
    for i in range(len(leaves)):  # one at a time
        for j, t in enumerate(leaves):
            t.requires_grad_(j == i)
        assert torch.equal(torch.autograd.grad(tpa.tpa_norm_rope(q, k, **kw), leaves[i], (dq, dk), allow_unused=True)[0] if i > 1 else
                           torch.autograd.grad(tpa.tpa_norm_rope(q, k, **kw)[i], leaves[i], (dq, dk)[i])[0], want[i])


@pytest.mark.parametrize("kernel", [1, 2])
@pytest.mark.parametrize("dtype,h,d,rq,rk", [(torch.bfloat16, 64, 64, 16, 8), (torch.bfloat16, 16, 128, 6, 2), (torch.float32, 24, 64, 3, 1)])
def test_results_over_the_inputs(gpu, dtype, h, d, rq, rk, kernel):
    """The C entry point takes the inputs' own memory for its results: bit for bit what it writes elsewhere."""
    import ctypes

    from tpa import _dispatch as dispatch

    x = make(41, 3, 37, h, d, rq, rk, dtype)
    kw = call(x, h, None, gpu)
    q, k = x["q"].to(gpu), x["k"].to(gpu)
    want = tpa.tpa_norm_rope(q, k, kernel=kernel, **kw)
    positions = kw["positions"].contiguous()
    f = {n + "a": dispatch.factor(t[..., :h]) for n, t in (("q", q), ("k", k))} | {n + "b": dispatch.factor(t[..., h:]) for n, t in (("q", q), ("k", k))}
    args = dispatch.TpaNormRopeArgs(
        **f, **{n + "_out": t for n, t in f.items()}, positions=positions.data_ptr(), rope_cos=kw["rope_cos"].data_ptr(), rope_sin=kw["rope_sin"].data_ptr(),
        q_weight=kw["q_weight"].data_ptr(), k_weight=kw["k_weight"].data_ptr(), n_axes=1, sections=(ctypes.c_int32 * 4)(d // 2), B=3, l=37, H=h, D=d, rq=rq, rk=rk, rope_len=len(kw["rope_cos"]),
        dtype=dispatch.dtype_code(dtype), weight_dtype=dispatch.dtype_code(kw["q_weight"].dtype), kernel=kernel, normalize=1, eps=kw.get("eps", 1e-6))
    torch.cuda.synchronize()
    assert dispatch.load_library().tpa_norm_rope(ctypes.byref(args), torch.cuda.current_stream().cuda_stream) == 0
    torch.cuda.synchronize()
    assert torch.equal(q, want[0]) and torch.equal(k, want[1])


def test_a_backward_pass_in_a_graph(gpu):
    """Captured with its gradients while nothing eager of the leaves lives; refused, before any of it is recorded, while something does."""
    h, d = 16, 64
    x = make(29, 2, 40, h, d, 6, 2, torch.bfloat16)
    kw = call(x, h, None, gpu)
    q, k, dq, dk = (x[n].to(gpu) for n in ("q", "k", "dq", "dk"))
    want = tpa.tpa_norm_rope_bwd(q, k, dq_out=dq, dk_out=dk, **kw)
    leaves = [q.requires_grad_(), k.requires_grad_()]
    work = lambda: torch.autograd.grad(tpa.tpa_norm_rope(q, k, **kw), leaves, (dq, dk))
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        work()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        got = work()
    for _ in range(3):
        for t in got:
            t.zero_()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    alive = tpa.tpa_norm_rope(q, k, **kw)
    torch.cuda.synchronize()
    refused = torch.cuda.CUDAGraph()
    with torch.cuda.graph(refused, stream=stream):
        with pytest.raises(RuntimeError, match="eager graph"):
            tpa.tpa_norm_rope(q, k, **kw)
        kept = tpa.tpa_norm_rope(q.detach(), k.detach(), **kw)
    refused.replay()
    torch.cuda.synchronize()
    assert torch.equal(kept[0], alive[0]) and torch.equal(kept[1], alive[1])


def test_slots_and_positions_of_64_bits(gpu):
    """Numbers that 32 bits do not hold are outside the pools and behind the last position, not some other place."""
    h, d = 8, 64
    x = make(31, 1, 4, h, d, 6, 2, torch.bfloat16)
    kw = call(x, h, None, gpu)
    q, k = x["q"].to(gpu), x["k"].to(gpu)
    pools = [torch.zeros((2, 4, 2, w), dtype=torch.bfloat16, device=gpu) for w in (h, d, h, d)]
    slots = torch.tensor([[1, 2**32 + 3, -(2**32) + 2, 6]], device=gpu)
    write = lambda s, p: tpa.tpa_norm_rope_write(q, k, k, h, kw["rope_cos"], kw["rope_sin"], *pools, s, kw["q_weight"], kw["k_weight"], p)
    write(slots, kw["positions"])
    used = pools[1].flatten(0, 1).flatten(1).any(1)
    assert used.tolist() == [i in (1, 6) for i in range(8)]
    last = kw["rope_cos"].shape[0] - 1
    far, end = (tpa.tpa_norm_rope(q, k, **dict(kw, positions=torch.tensor([[0, 1, p, 2]], device=gpu))) for p in (2**40, last))
    assert torch.equal(far[0], end[0]) and torch.equal(far[1], end[1])
    for bad in (slots.float(), slots > 0):
        with pytest.raises(TypeError):
            write(bad, kw["positions"])
        with pytest.raises(TypeError):
            write(slots, bad)


def test_refusals(gpu):
    h, d = 8, 64
    x = make(29, 2, 6, h, d, 6, 2, torch.bfloat16)
    q, k, v = (x[n].to(gpu) for n in "qkv")
    cos, sin = x["cos"].to(gpu), x["sin"].to(gpu)
    for bad in (dict(sections=[40]), dict(sections=[8] * 5), dict(sections=[-1, 8]), dict(positions=x["pos"].to(gpu)[:1]), dict(sections=[8, 8], positions=x["pos"].to(gpu))):
        with pytest.raises(ValueError):
            tpa.tpa_norm_rope(q, k, h, cos, sin, **bad)
    for args in ((q, k[:1], h, cos, sin), (q, k, 0, cos, sin), (q, k, h, cos[:, 1:], sin), (q, k, h + 2, cos, sin)):
        with pytest.raises(AssertionError):
            tpa.tpa_norm_rope(*args)
    with pytest.raises(AssertionError):
        tpa.tpa_norm_rope(q, k, h, cos, sin, q_weight=cos[0])
    with pytest.raises(TypeError):
        tpa.tpa_norm_rope(q, k.float(), h, cos, sin)
    with pytest.raises(TypeError):
        tpa.tpa_norm_rope(q, k, h, cos, sin, q_weight=x["wq"].to(gpu), k_weight=x["wk"].to(gpu).bfloat16())
    pools = [torch.zeros((2, 16, 2, w), dtype=torch.bfloat16, device=gpu) for w in (h, d, h, d)]
    slots = torch.arange(12, device=gpu).view(2, 6)
    with pytest.raises(TypeError):
        tpa.tpa_norm_rope_write(q, k, v, h, cos, sin, *(p.cpu() for p in pools), slots)
    with pytest.raises(ValueError):
        tpa.tpa_norm_rope_write(q, k, v, h, cos, sin, *pools, slots[:1])
    with pytest.raises(AssertionError):
        tpa.tpa_norm_rope_write(q, k, v, h, cos, sin, pools[1], *pools[1:], slots)
    with pytest.raises(TypeError):
        tpa.tpa_norm_rope_write(q, k, v, h, cos, sin, *(p.float() for p in pools), slots)
    r = q.clone().requires_grad_()
    out = tpa.tpa_norm_rope(r, k, h, cos, sin)[0]
    with pytest.raises(RuntimeError, match="second derivative"):
        torch.autograd.grad(out.float().square().sum(), r, create_graph=True)


@pytest.mark.parametrize("write", ["positions", "cos", "sin"])
def test_arrays_written_again_before_the_backward(gpu, write):
    """The gradients turn by the forward's positions: where these have been written over, torch says so.  What the call has converted is its own."""
    h, d = 8, 64
    x = make(43, 2, 9, h, d, 6, 2, torch.bfloat16)
    kw = call(x, h, None, gpu)
    q = x["q"].to(gpu).requires_grad_()
    k, dq = x["k"].to(gpu), x["dq"].to(gpu)
    arrays = dict(positions=kw["positions"].contiguous(), cos=kw["rope_cos"], sin=kw["rope_sin"])
    kw.update(positions=arrays["positions"])
    want = torch.autograd.grad(tpa.tpa_norm_rope(q, k, **kw)[0], q, dq)[0]
    out = tpa.tpa_norm_rope(q, k, **kw)[0]
    arrays[write].add_(0)
    with pytest.raises(RuntimeError, match="inplace operation"):
        torch.autograd.grad(out, q, dq)
    wide = dict(positions=kw["positions"].long(), rope_cos=kw["rope_cos"].double(), rope_sin=kw["rope_sin"].double(), q_weight=kw["q_weight"], k_weight=kw["k_weight"], num_heads=h)
    out = tpa.tpa_norm_rope(q, k, **wide)[0]
    for n in ("positions", "rope_cos", "rope_sin"):
        wide[n].zero_()
    assert torch.equal(torch.autograd.grad(out, q, dq)[0], want)


def test_tables_of_inference_and_tables_that_ask_for_gradients(gpu):
    h, d = 8, 64
    x = make(47, 2, 9, h, d, 6, 2, torch.bfloat16)
    kw = call(x, h, None, gpu)
    q = x["q"].to(gpu).requires_grad_()
    k, dq = x["k"].to(gpu), x["dq"].to(gpu)
    want = torch.autograd.grad(tpa.tpa_norm_rope(q, k, **kw)[0], q, dq)[0]
    with torch.inference_mode():
        made = {n: kw[n] + 0 for n in ("positions", "rope_cos", "rope_sin")}
    assert torch.equal(torch.autograd.grad(tpa.tpa_norm_rope(q, k, **dict(kw, **made))[0], q, dq)[0], want)
    for n in ("rope_cos", "rope_sin"):
        asks = dict(kw, **{n: kw[n].clone().requires_grad_()})
        with pytest.raises(NotImplementedError):
            tpa.tpa_norm_rope(q, k, **asks)
        with torch.no_grad():
            tpa.tpa_norm_rope(q, k, **asks)


def first_power(x, h, weight, c, s, eps, dy):
    """`side`'s results with the slack of norms that are summed over the head vectors themselves: with kappa as the sum of the terms' sizes over
    their sum, an element of X_h is off by 2 R U of its terms' sizes, the norm by kappa^(1/2) of that, and by D + 16 roundings of its own.  fp32
    factors have their norms in 64 bits, within the same."""
    r, d = x.shape[2], x.shape[3] - h
    a, b = x[..., :h], x[..., h:]
    dense, sizes = torch.matmul(a.transpose(2, 3), b) / r, torch.matmul(a.abs().transpose(2, 3), b.abs()) / r
    n = dense.square().mean(-1) + eps
    scale = n.rsqrt()
    rel_s = (2 * r * ((sizes.square().mean(-1) + eps) / n).sqrt() + d + 16) * U
    out, _, grad, _, dw, _ = side(x, h, weight, c, s, eps, True, dy)
    da = dy[..., :h]
    w = scale**3 * (da * a).abs().sum(2) / (d * r * r)
    m_size = torch.matmul(a.abs() * w[:, :, None], a.abs().transpose(2, 3))
    worst = rel_s.amax(-1)[:, :, None, None]
    # w comes from the norm and the sum over the ranks of da a; the gradients of a from G a, those of b from the mixture, each a sum of terms that cancel
    # to the first power: G, M and w a are within 4 U of what they stand for
    g_size = torch.matmul(b.abs(), b.abs().transpose(2, 3))
    g_slack = torch.cat([(da * scale[:, :, None]).abs() * (rel_s[:, :, None] + 2 * U) + (w * 3 * rel_s)[:, :, None] * torch.matmul(b, dense.transpose(2, 3)).abs() * r
                         + w[:, :, None] * torch.matmul(g_size, a.abs()) * (d + 3 * r + 20) * U,
                         8 * U * dy[..., h:].abs().amax(-1, keepdim=True) * weight.abs() * 2 + torch.matmul((a.abs() * (3 * rel_s * w)[:, :, None]), dense.abs()) * r
                         + torch.matmul(m_size, b.abs()) * (h + 3 * r + 24) * U], -1)
    return out[..., :h], (a * scale[:, :, None]).abs() * rel_s[:, :, None], grad, g_slack


def cancelling(apart, b, l, h, d, rq, rk, dtype):
    """`make`'s arrays, every second rank the one before it with the other sign of a and a b that is off by 2^-apart: head vectors 2^apart smaller than
    their terms."""
    x = make(apart, b, l, h, d, rq, rk, torch.float32)
    g = torch.Generator().manual_seed(apart)
    for n in "qk":
        y = x[n].to(torch.bfloat16).float()
        y[:, :, 1::2, :h] = -y[:, :, ::2, :h]
        y[:, :, 1::2, h:] = (y[:, :, ::2, h:] * (1 + 2.0**-apart * torch.randn(y[:, :, ::2, h:].shape, generator=g))).to(torch.bfloat16).float()
        x[n] = y.to(dtype)
        x["d" + n] = x["d" + n].to(dtype)
    return x


@pytest.mark.parametrize("kernel", [1, 2])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("h,d,rq,rk", [(16, 128, 2, 6), (32, 64, 4, 16), (8, 64, 8, 2)])
@pytest.mark.parametrize("apart", [5, 7, 9])
def test_ranks_that_cancel(gpu, dtype, h, d, rq, rk, apart, kernel):
    """The norms of head vectors that are far smaller than their terms are as near as if the vectors had been formed; a token's do not depend on
    the tokens beside it."""
    x = cancelling(apart, 2, 21, h, d, rq, rk, dtype)
    kw = call(x, h, None, gpu, kernel=kernel)
    got = tpa.tpa_norm_rope(x["q"].to(gpu), x["k"].to(gpu), **kw)
    c, s = angles(x["pos"], [d // 2], x["cos"], x["sin"], d)
    others = make(apart, 2, 21, h, d, rq, rk, dtype)
    for i, n in enumerate("qk"):
        out, slack, _, _ = first_power(x[n].double(), h, x["w" + n].double(), c, s, 1e-6, x["d" + n].double())
        near(got[i][..., :h], out, slack, dtype, n)
        others[n][:, ::3] = x[n][:, ::3]
    beside = tpa.tpa_norm_rope(others["q"].to(gpu), others["k"].to(gpu), **kw)
    assert all(torch.equal(a[:, ::3], b[:, ::3]) for a, b in zip(got, beside))


@pytest.mark.parametrize("kernel", [1, 2])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("h,d,rq,rk", [(16, 128, 2, 6), (32, 64, 4, 16), (8, 64, 8, 2)])
@pytest.mark.parametrize("apart", [5, 7, 9])
def test_gradients_of_ranks_that_cancel(gpu, dtype, h, d, rq, rk, apart, kernel):
    """The same of the gradients, which hold the cube of the norm and sums over the ranks that cancel."""
    x = cancelling(apart, 2, 21, h, d, rq, rk, dtype)
    kw = call(x, h, None, gpu, kernel=kernel)
    grads = tpa.tpa_norm_rope_bwd(x["q"].to(gpu), x["k"].to(gpu), dq_out=x["dq"].to(gpu), dk_out=x["dk"].to(gpu), **kw)
    c, s = angles(x["pos"], [d // 2], x["cos"], x["sin"], d)
    for i, n in enumerate("qk"):
        _, _, grad, g_slack = first_power(x[n].double(), h, x["w" + n].double(), c, s, 1e-6, x["d" + n].double())
        near(grads[i], grad, g_slack, dtype, "d" + n)


@pytest.mark.parametrize("dtype,h,d,rq,rk", [(torch.bfloat16, 192, 64, 1, 1), (torch.bfloat16, 192, 128, 1, 2), (torch.float32, 128, 64, 1, 1), (torch.float32, 128, 128, 2, 1), (torch.bfloat16, 512, 128, 1, 1)])
def test_many_heads_at_rank_one(gpu, dtype, h, d, rq, rk):
    """Sixteen tokens to a wave, each with a number for every head in LDS: the matrix-core kernels take them in both directions, weights at any address too."""
    x = make(h, 2, 21, h, d, rq, rk, dtype)
    kw = call(x, h, None, gpu, kernel=2)
    for n in ("q_weight", "k_weight"):
        kw[n] = torch.cat([kw[n].new_zeros(1), kw[n]])[1:]
    q, k = (x[n].to(gpu) for n in "qk")
    got = tpa.tpa_norm_rope(q, k, **kw)
    grads = tpa.tpa_norm_rope_bwd(q, k, dq_out=x["dq"].to(gpu), dk_out=x["dk"].to(gpu), **kw)
    c, s = angles(x["pos"], [d // 2], x["cos"], x["sin"], d)
    for i, n in enumerate("qk"):
        out, slack, grad, g_slack, dw, w_slack = side(x[n].double(), h, x["w" + n].double(), c, s, 1e-6, True, x["d" + n].double())
        near(got[i], out, slack, dtype, n)
        near(grads[i], grad, g_slack, dtype, "d" + n)
        near(grads[2 + i], dw, w_slack, torch.float32, "dw" + n)


@pytest.mark.parametrize("gone", ["q", "k", "qk"])
def test_a_side_without_a_gradient_is_not_looked_at(gpu, gone):
    """The C entry point with one side's gradient, the other side's fields left as anything."""
    import ctypes

    from tpa import _dispatch as dispatch

    h, d, rq, rk = 16, 64, 6, 2
    x = make(53, 2, 37, h, d, rq, rk, torch.bfloat16)
    kw = call(x, h, None, gpu)
    arrays = {n: x[n].to(gpu) for n in ("q", "k", "dq", "dk")}
    want = tpa.tpa_norm_rope_bwd(arrays["q"], arrays["k"], dq_out=arrays["dq"], dk_out=arrays["dk"], kernel=2, **kw)
    grads, d_weights, fields = {}, {}, {}
    for n in "qk":
        grads[n], d_weights[n] = torch.zeros_like(arrays[n]), torch.zeros(d, device=gpu)
        for part, at in (("a", slice(0, h)), ("b", slice(h, None))):
            for name, t in ((n + part, arrays[n]), (f"d{n}{part}_out", arrays["d" + n]), (f"d{n}{part}", grads[n])):
                fields[name] = dispatch.factor(t[..., at]) if n not in gone else dispatch.TpaFactor(None if name.endswith("a_out") else 6, 3, -5, 7)
    ws = torch.empty(1 << 22, dtype=torch.uint8, device=gpu)
    positions = kw["positions"].contiguous()
    args = dispatch.TpaNormRopeBwdArgs(
        **fields, dq_weight=d_weights["q"].data_ptr(), dk_weight=d_weights["k"].data_ptr(), positions=positions.data_ptr(), rope_cos=kw["rope_cos"].data_ptr(),
        rope_sin=kw["rope_sin"].data_ptr(), q_weight=3 if "q" in gone else kw["q_weight"].data_ptr(), k_weight=3 if "k" in gone else kw["k_weight"].data_ptr(), n_axes=1,
        sections=(ctypes.c_int32 * 4)(d // 2), B=2, l=37, H=h, D=d, rq=-1 if "q" in gone else rq, rk=99 if "k" in gone else rk, rope_len=len(kw["rope_cos"]),
        dtype=1, weight_dtype=0, kernel=2, normalize=1, eps=1e-6, workspace=ws.data_ptr(), workspace_bytes=ws.numel())
    torch.cuda.synchronize()
    assert dispatch.load_library().tpa_norm_rope_bwd(ctypes.byref(args), torch.cuda.current_stream().cuda_stream) == 0
    torch.cuda.synchronize()
    for i, n in enumerate("qk"):
        assert torch.equal(grads[n], torch.zeros_like(grads[n]) if n in gone else want[i])
        assert torch.equal(d_weights[n], torch.zeros_like(d_weights[n]) if n in gone else want[2 + i])


@pytest.mark.parametrize("kernel", [1, 2])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_small_head_vectors_without_eps(gpu, dtype, kernel):
    """Head vectors of about 2^-43 and eps 0: the cube of 2^43 is no number of 32 bits, the gradients are."""
    h, d = 8, 128
    x = make(59, 1, 11, h, d, 16, 15, dtype)
    for n in "qk":
        x[n][..., h:] *= 2.0**-41
    kw = call(x, h, None, gpu, kernel=kernel, eps=0.0)
    grads = tpa.tpa_norm_rope_bwd(x["q"].to(gpu), x["k"].to(gpu), dq_out=x["dq"].to(gpu), dk_out=x["dk"].to(gpu), **kw)
    c, s = angles(x["pos"], [d // 2], x["cos"], x["sin"], d)
    for i, n in enumerate("qk"):
        _, _, grad, g_slack, _, _ = side(x[n].double(), h, x["w" + n].double(), c, s, 0.0, True, x["d" + n].double())
        near(grads[i], grad, g_slack, dtype, "d" + n)


@pytest.mark.parametrize(
    "b,l,h,d,rq,rk,dtype,kernel,sections",
    [
        (3, 7001, 16, 128, 6, 2, torch.bfloat16, 2, None),          # several groups of tokens to a wave of the backward, unequal shares
        (2, 9003, 64, 64, 16, 8, torch.bfloat16, 2, [8, 12, 12]),   # and, past 16384 groups, of the forward
        (1, 20011, 8, 64, 6, 2, torch.float32, 2, None),
        (1, 17003, 32, 128, 9, 3, torch.float32, 2, None),
        (1, 5003, 8, 64, 6, 2, torch.bfloat16, 1, None),            # more tokens than workgroups of the plain kernels
        (5, 1009, 3, 10, 5, 2, torch.float32, 0, None),
    ],
)
def test_many_tokens(gpu, b, l, h, d, rq, rk, dtype, kernel, sections):
    """Waves and workgroups that serve several groups of tokens.  A sum of a weight's gradient is a chain of what a lane or thread meets and 76 more."""
    x = make(l, b, l, h, d, rq, rk, dtype, axes=len(sections or [0]))
    kw = call(x, h, sections, gpu, kernel=kernel)
    q, k = (x[n].to(gpu) for n in "qk")
    got = tpa.tpa_norm_rope(q, k, **kw)
    grads = tpa.tpa_norm_rope_bwd(q, k, dq_out=x["dq"].to(gpu), dk_out=x["dk"].to(gpu), **kw)
    again = tpa.tpa_norm_rope_bwd(q, k, dq_out=x["dq"].to(gpu), dk_out=x["dk"].to(gpu), **kw)
    assert all(torch.equal(g, w) for g, w in zip(grads, again))
    with torch.device(gpu):
        c, s = angles(x["pos"].to(gpu), sections or [d // 2], x["cos"].to(gpu), x["sin"].to(gpu), d)
        for i, n in enumerate("qk"):
            r = (rq, rk)[i]
            chain = -(-b * l // 768) * r + 76  # at most: a workgroup of the plain kernels has every 768th token, a lane of the others fewer rows
            ingredients = side(x[n].to(gpu).double(), h, x["w" + n].to(gpu).double(), c, s, 1e-6, True, x["d" + n].to(gpu).double())
            out, slack, grad, g_slack, dw, w_slack = (t.cpu() for t in ingredients)
            near(got[i], out, slack, dtype, n)
            near(grads[i], grad, g_slack, dtype, "d" + n)
            near(grads[2 + i], dw, w_slack * (chain / 128), torch.float32, "dw" + n)


@pytest.mark.parametrize("h,d,rq,rk", [(16, 128, 2, 6), (32, 64, 4, 16), (8, 64, 8, 2), (24, 128, 16, 4)])
def test_ranks_that_cancel_in_a_cache_and_beside_values_that_are_not_finite(gpu, h, d, rq, rk):
    """Written into a cache bit for bit what tpa_norm_rope gives; infinities and NaN of some tokens, a zero token, and tokens that do not cancel stay
    with themselves, in both directions."""
    x = cancelling(8, 2, 21, h, d, rq, rk, torch.bfloat16)
    plain = make(61, 2, 21, h, d, rq, rk, torch.bfloat16)
    for n in "qk":
        x[n][:, 1::4] = plain[n][:, 1::4]
    kw = call(x, h, None, gpu)
    q, k, v, dq, dk = (x[n].to(torch.bfloat16).to(gpu) for n in ("q", "k", "v", "dq", "dk"))
    want = tpa.tpa_norm_rope(q, k, kernel=2, **kw)
    grads = tpa.tpa_norm_rope_bwd(q, k, dq_out=dq, dk_out=dk, kernel=2, **kw)
    pools = [torch.zeros((4, 16, rk, w), dtype=torch.bfloat16, device=gpu) for w in (h, d, h, d)]
    slots = torch.randperm(64, generator=torch.Generator().manual_seed(2))[:42].view(2, 21).to(gpu)
    got = tpa.tpa_norm_rope_write(q, k, v, h, kw["rope_cos"], kw["rope_sin"], *pools, slots, kw["q_weight"], kw["k_weight"], kw["positions"], kernel=2)
    assert torch.equal(got, want[0])
    for pool, part in zip(pools, (want[1][..., :h], want[1][..., h:], v[..., :h], v[..., h:])):
        assert torch.equal(pool.flatten(0, 1)[slots], part)
    for y in (q, k):
        y[0, 2, -1, h + 1], y[0, 5, 0, h + d - 1], y[1, 11, -1, 0], y[1, 14] = float("inf"), float("nan"), float("-inf"), 0
    others = torch.ones(2, 21, dtype=torch.bool, device=gpu)
    others[0, [2, 5]] = others[1, [11, 14]] = False
    again = tpa.tpa_norm_rope(q, k, kernel=2, **kw)
    again_grads = tpa.tpa_norm_rope_bwd(q, k, dq_out=dq, dk_out=dk, kernel=2, **kw)
    for a, b in zip((*again, *again_grads[:2]), (*want, *grads[:2])):
        assert torch.equal(a[others], b[others]) and not torch.equal(a, b)


def test_the_most_heads(gpu):
    """As many heads at rank 1 as the header names for every type and head size; one block more is the plain kernel's, or refused."""
    for h, kernel in ((504, 2), (512, 0)):
        x = make(h, 1, 17, h, 128, 1, 1, torch.float32)
        kw = call(x, h, None, gpu, kernel=kernel)
        q, k = (x[n].to(gpu) for n in "qk")
        grads = tpa.tpa_norm_rope_bwd(q, k, dq_out=x["dq"].to(gpu), dk_out=x["dk"].to(gpu), **kw)
        c, s = angles(x["pos"], [64], x["cos"], x["sin"], 128)
        for i, n in enumerate("qk"):
            _, _, grad, g_slack, _, _ = side(x[n].double(), h, x["w" + n].double(), c, s, 1e-6, True, x["d" + n].double())
            near(grads[i], grad, g_slack, torch.float32, "d" + n)
    with pytest.raises(RuntimeError):
        tpa.tpa_norm_rope_bwd(q, k, dq_out=x["dq"].to(gpu), dk_out=x["dk"].to(gpu), **dict(kw, kernel=2))
