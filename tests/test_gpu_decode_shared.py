"""tpa_decode_shared (decode of a batch that shares its first tokens) against dense attention in 64 bits.

Tolerances, with P = sum_k p_k (1/R) sum_r |va_r||vb_r| the sum of the sizes of an output's terms and X = sm_scale |Q||K| that of a
logit's (Q and K with the sizes of their factors):
  one rounding of the output: 2^-8 (bf16) or 2^-24 (fp32) of it;
  the matrix-core kernel for bf16 rounds the weights p va to bf16: 2^-8 P, and keeps Q as two bf16 numbers: 2^-16 X on a logit;
  sums in 32 bits: a logit (2 D + R Rq) 2^-24 X, the sums over n keys n 2^-24 P;
  a logit that is off by x moves the output by at most 2 x P and the logsumexp by x.
"""

import math

import pytest
import torch

from tpa import tpa

pytestmark = pytest.mark.gpu
U = 2.0**-24


def oracle(qa, qb, caches, prefix, lengths, scale, causal, offset):
    """caches: the four arrays [b, lk, rk, x], already with entry 0's prefix; results and their tolerances' ingredients, all in 64 bits."""
    f = [t.double() for t in (qa, qb, *caches)]
    dense = lambda a, b: torch.matmul(a.transpose(2, 3), b) / a.shape[2]  # [b, l, h, d]
    q, k, v = (dense(f[i], f[i + 1]) for i in (0, 2, 4))
    qs, ks, vs = (dense(f[i].abs(), f[i + 1].abs()) for i in (0, 2, 4))
    b, lq, h, _ = q.shape
    lk = k.shape[1]
    x = scale * torch.einsum("blhd,bthd->bhlt", q, k)
    xs = scale * torch.einsum("blhd,bthd->bhlt", qs, ks)
    t = torch.arange(lk)
    sees = lengths[:, None].expand(b, lq).clone()
    if causal:
        last = torch.arange(lq)[None] + offset + 1 + ((lengths[:, None] - lq) if causal == 2 else 0)
        sees = torch.minimum(sees, last.clamp(min=0))
    hidden = t >= sees[:, None, :, None]
    x = x.masked_fill(hidden, -math.inf)
    lse = torch.logsumexp(x, -1)
    p = torch.exp(x - lse[..., None])
    o = torch.einsum("bhlt,bthd->blhd", p, v)
    size = torch.einsum("bhlt,bthd->blhd", p, vs)
    return o, lse, size, xs.masked_fill(hidden, 0).amax(-1)


def check(gpu, b, lq, prefix, own, h, d, rq, rk, dtype, kernel, page=0, causal=0, offset=0, lengths=None, seed=0, sharp=1.0, dv=None):
    g = torch.Generator().manual_seed(seed + 7 * b + prefix)
    lk = prefix + own
    dv = dv or d
    if page:
        lk = -(-lk // page) * page
    n = lambda *s: torch.randn(s, generator=g)
    qa, qb = (sharp * rq**0.5 * n(b, lq, rq, h)).to(dtype), n(b, lq, rq, d).to(dtype)
    caches = [(n(b, lk, rk, w) * (rk**0.5 if i == 0 else 1)).to(dtype) for i, w in enumerate((h, d, h, dv))]
    for c in caches:
        c[:, :prefix] = c[:1, :prefix]
    length = torch.full((b,), prefix + own) if lengths is None else torch.tensor(lengths)
    scale = d**-0.5
    o, lse, size, xs = oracle(qa, qb, caches, prefix, length, scale, causal, offset)
    dev = [t.to(gpu) for t in (qa, qb)]
    more = {}
    if page:  # pools with the prefix's whole pages once, everything else NaN where no token is
        pages, whole = lk // page, prefix // page
        ids = torch.randperm(whole + b * (pages - whole), generator=g).to(torch.int32)
        table = torch.empty((b, pages), dtype=torch.int32)
        table[:, :whole] = ids[:whole]
        table[:, whole:] = ids[whole:].view(b, -1)
        pools = [torch.full((len(ids), page, rk, c.shape[3]), float("nan"), dtype=dtype) for c in caches]
        for pool, c in zip(pools, caches):
            for i in range(b):
                for j in range(pages):
                    tokens = max(0, min(page, int(length[i]) - j * page))
                    pool[table[i, j], :tokens] = c[i, j * page : j * page + tokens]
        more["page_table"] = table.to(gpu)
        dev += [p.to(gpu) for p in pools]
    else:
        for c in caches[0:]:
            for i in range(b):
                c[i, int(length[i]) :] = float("nan")
                if i:
                    c[i, :prefix] = float("nan")  # only entry 0's prefix is read
        dev += [c.to(gpu) for c in caches]
        if int(length[0]) < min(prefix, int(length.max())):
            pytest.fail("entry 0 holds the prefix")
    got, got_lse = tpa.tpa_decode_shared(*dev, prefix_length=prefix, sm_scale=scale, kernel=kernel, kv_lengths=None if lengths is None and not page else length.to(gpu),
                                         causal=causal, causal_offset=offset, **more)
    got, got_lse = got.cpu().double(), got_lse.cpu().double()
    empty = lse == -math.inf
    assert got.isnan().any(-1).transpose(1, 2).equal(empty) and (got_lse[empty] == -math.inf).all()
    half = torch.finfo(dtype).eps / 2
    split = 2.0**-16 if dtype == torch.bfloat16 else 0
    logit = (split + (2 * d + rk * rq) * U) * xs
    keep = ~empty
    slack = 2 * logit.transpose(1, 2)[..., None] * size + (half if dtype == torch.bfloat16 else 0) * size + (lk + 16) * U * size
    assert ((got_lse - lse).abs()[keep] <= (logit + (lk + 8) * U + 4 * U * lse.abs())[keep]).all(), (got_lse - lse).abs()[keep].max()
    bad = ((got - o).abs() > half * o.abs() + slack * (1 + half)) & keep.transpose(1, 2)[..., None]
    assert not bad.any(), ((got - o).abs()[bad].max(), int(bad.sum()))


KERNELS = [0, 1]
BF, F32 = torch.bfloat16, torch.float32


@pytest.mark.parametrize("kernel", KERNELS)
@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize(
    "b,lq,prefix,own,h,d,rq,rk",
    [
        (1, 1, 1, 1, 8, 64, 1, 1),          # one token of each
        (3, 1, 200, 17, 16, 128, 6, 2),
        (2, 1, 0, 40, 8, 64, 6, 2),         # no prefix
        (5, 1, 300, 0, 32, 128, 6, 2),      # nothing but the prefix
        (9, 1, 130, 70, 32, 64, 6, 4),      # more columns than a workgroup takes
        (4, 2, 65, 33, 64, 64, 16, 8),      # two blocks of heads, rank 8
        (40, 1, 64, 5, 24, 128, 3, 1),      # 24 heads
        (2, 5, 31, 9, 40, 64, 2, 2),        # 40 heads, blocks of 8
        (1, 70, 90, 70, 8, 128, 6, 2),      # many rows
        (2, 1, 1000, 1, 8, 64, 6, 2),
    ],
)
def test_contiguous(gpu, b, lq, prefix, own, h, d, rq, rk, dtype, kernel):
    check(gpu, b, lq, prefix, own, h, d, rq, rk, dtype, kernel)


@pytest.mark.parametrize("kernel", KERNELS)
@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize(
    "prefix,page,lengths,lq",
    [
        (128, 64, [128, 190, 129, 300, 256], 1),   # nothing of its own, the middle of a page, a page's first and last token
        (150, 64, [200, 151, 150, 320], 1),        # the prefix ends inside a page
        (96, 32, [100, 40, 0, 96, 160], 1),        # shorter than the prefix, empty
        (64, 32, [67, 64 + 33, 70], 3),            # speculated tokens
        (320, 64, [321] * 12, 1),
    ],
)
def test_paged_and_ragged(gpu, prefix, page, lengths, lq, dtype, kernel):
    own = max(max(lengths) - prefix, 0)
    for causal in (0, 2):
        check(gpu, len(lengths), lq, prefix, own, 16, 128, 6, 2, dtype, kernel, page=page, causal=causal, lengths=lengths)


@pytest.mark.parametrize("kernel", KERNELS)
@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("causal,offset", [(1, 0), (1, 40), (1, -1), (2, 0), (2, -3), (2, 5)])
def test_masks(gpu, dtype, kernel, causal, offset):
    """The mask's border in the prefix, behind it, before the first key (rows that see nothing)."""
    check(gpu, 3, 6, 50, 20, 8, 64, 6, 2, dtype, kernel, causal=causal, offset=offset)
    check(gpu, 2, 6, 33, 2, 8, 128, 2, 4, dtype, kernel, causal=causal, offset=offset, lengths=[35, 34])


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("h,d,rk,dv,page", [(3, 10, 3, 7, 0), (8, 64, 16, 64, 0), (5, 64, 2, 64, 16), (8, 256, 2, 256, 5), (8, 64, 3, 64, 7)])
def test_shapes_of_no_matrix_core_kernel(gpu, dtype, h, d, rk, dv, page):
    check(gpu, 3, 2, 21, 30, h, d, 5, rk, dtype, 0, dv=dv, page=page)


@pytest.mark.parametrize("kernel", KERNELS)
@pytest.mark.parametrize("dtype", [BF, F32])
def test_sharp_logits(gpu, dtype, kernel):
    """Logits with a standard deviation of 12: the maximum grows along the keys and between the prefix and the rest."""
    check(gpu, 4, 1, 700, 300, 16, 64, 6, 2, dtype, kernel, sharp=12.0)


def test_equals_decode_over_a_replicated_prefix(gpu):
    """The call is tpa_decode's over the same arrays, within both kernels' tolerances (3 roundings of 2^-8 each of P <= max |V|)."""
    b, h, d, prefix, own = 6, 32, 128, 1500, 100
    g = torch.Generator().manual_seed(1)
    n = lambda *s: torch.randn(s, generator=g).to(BF).to(gpu)
    qa, qb = n(b, 1, 6, h), n(b, 1, 6, d)
    caches = [n(b, prefix + own, 2, w) for w in (h, d, h, d)]
    for c in caches:
        c[:, :prefix] = c[:1, :prefix]
    lengths = torch.tensor([1600, 1500, 1550, 1599, 1501, 1570], dtype=torch.int32, device=gpu)
    got, lse = tpa.tpa_decode_shared(qa, qb, *caches, prefix_length=prefix, sm_scale=d**-0.5, kv_lengths=lengths)
    want, want_lse = tpa.tpa_decode(qa, qb, *caches, sm_scale=d**-0.5, kv_lengths=lengths)
    assert (got.float() - want.float()).abs().max() <= 2.0**-6 and (lse - want_lse).abs().max() <= 2.0**-8


def test_a_serving_step(gpu):
    """Page tables, norms with rotation into the cache, decode over the shared prefix: three calls of a step, twice in a row, against the
    same sequences attended to in 64 bits.  The logits' tolerance is the kernel's (see above) over the cached bf16 factors."""
    b, h, d, rq, rk, page, prefix, pages = 5, 16, 64, 6, 2, 32, 96, 8
    g = torch.Generator().manual_seed(4)
    n = lambda *s: torch.randn(s, generator=g).to(BF).to(gpu)
    ang = torch.arange(512, dtype=torch.float64)[:, None] * 10000.0 ** (-torch.arange(0, d, 2, dtype=torch.float64) / d)
    cos, sin = ang.cos().float().to(gpu), ang.sin().float().to(gpu)
    table = torch.full((b, pages), -7, dtype=torch.int32, device=gpu)
    free = torch.randperm(60, generator=g).to(torch.int32).to(gpu)
    pools = [torch.full((60, page, rk, w), float("nan"), dtype=BF, device=gpu) for w in (h, d, h, d)]
    # the prompt that all share goes into the first pages
    zero, start = torch.zeros(1, dtype=torch.int32, device=gpu), None
    row = table[:1].clone()
    slots, positions, _, _, start = tpa.tpa_page_tables(zero, zero + prefix, row, free, page_size=page, num_tokens=prefix)
    x = [n(1, prefix, r, h + d) for r in (rq, rk, rk)]
    tpa.tpa_norm_rope_write(*x, h, cos, sin, *pools, slots[None], positions=positions[None])
    history_v = [[x[2][0]] for _ in range(b)]
    _, k = tpa.tpa_norm_rope(x[0], x[1], h, cos, sin)
    history_k = [[k[0]] for _ in range(b)]
    table[:] = row
    lengths = torch.full((b,), prefix, dtype=torch.int32, device=gpu)
    for news in ([3, 1, 2, 40, 1], [1, 1, 1, 1, 1]):
        total = sum(news)
        new = torch.tensor(news, dtype=torch.int32, device=gpu)
        slots, positions, starts, lengths, start = tpa.tpa_page_tables(lengths, new, table, free, page_size=page, num_tokens=total + 3, free_start=start)
        q, k, v = (n(1, total + 3, r, h + d) for r in (rq, rk, rk))
        q_new = tpa.tpa_norm_rope_write(q, k, v, h, cos, sin, *pools, slots[None], positions=positions[None])
        k_new = tpa.tpa_norm_rope(q, k, h, cos, sin, positions=positions[None])[1]
        for i, (first, count) in enumerate(zip(starts.tolist(), news)):
            history_k[i].append(k_new[0, first : first + count])
            history_v[i].append(v[0, first : first + count])
        last = q_new[0, starts[1:].long() - 1][:, None]
        o, lse = tpa.tpa_decode_shared(last[..., :h], last[..., h:], *pools, prefix_length=prefix, sm_scale=d**-0.5, kv_lengths=lengths, page_table=table)
        for i in range(b):
            kv = [torch.cat(t)[None].cpu() for t in (history_k[i], history_v[i])]
            assert int(lengths[i]) == kv[0].shape[1]
            caches = [kv[0][..., :h], kv[0][..., h:], kv[1][..., :h], kv[1][..., h:]]
            qi = last[i : i + 1].cpu()
            want, want_lse, size, xs = oracle(qi[..., :h], qi[..., h:], caches, prefix, torch.tensor([kv[0].shape[1]]), d**-0.5, 0, 0)
            logit = (2.0**-16 + 2 * d * U) * xs.transpose(1, 2)[..., None]
            err = (o[i : i + 1].cpu().double() - want).abs()
            assert (err <= 2.0**-8 * want.abs() + (2.0**-8 + 2 * logit + 400 * U) * size * 1.01).all()


def test_replays_from_a_graph_and_two_streams(gpu):
    """A captured call follows lengths that change between replays; two calls at once on two streams have workspaces of their own."""
    b, h, d, prefix = 4, 32, 128, 900
    g = torch.Generator().manual_seed(2)
    n = lambda *s: torch.randn(s, generator=g).to(BF).to(gpu)
    qa, qb = n(b, 1, 6, h), n(b, 1, 6, d)
    caches = [n(b, 1200, 2, w) for w in (h, d, h, d)]
    lengths = torch.tensor([900, 1000, 1100, 1200], dtype=torch.int32, device=gpu)
    call = lambda: tpa.tpa_decode_shared(qa, qb, *caches, prefix_length=prefix, sm_scale=d**-0.5, kv_lengths=lengths)
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        call()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            captured = call()
    for shift in (0, 1, 2):
        lengths.copy_(torch.tensor([900, 1000, 1100, 1200], dtype=torch.int32).roll(shift))
        want = call()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(captured, want))
    others = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for s in others:
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            got.append([call() for _ in range(3)])
    torch.cuda.synchronize()
    assert all(torch.equal(x, y) for r in got for one in r for x, y in zip(one, want))


def test_a_captured_serving_step(gpu):
    """The three calls of a step in one graph that advances its own lengths: every replay gives what the eager step gives, pages opened on the way."""
    b, h, d, rq, rk, page, prefix, pages, steps = 4, 8, 64, 6, 2, 32, 64, 5, 5
    g = torch.Generator().manual_seed(9)
    ang = torch.arange(256, dtype=torch.float64)[:, None] * 10000.0 ** (-torch.arange(0, d, 2, dtype=torch.float64) / d)
    cos, sin = ang.cos().float().to(gpu), ang.sin().float().to(gpu)
    new = [[torch.randn((1, b, r, h + d), generator=g).to(BF).to(gpu) for r in (rq, rk, rk)] for _ in range(steps)]
    pools = [torch.randn((24, page, rk, w), generator=g).to(BF) for w in (h, d, h, d)]
    table = torch.full((b, pages), -1, dtype=torch.int32)
    table[:, :2], table[:, 2] = torch.tensor([5, 3]), torch.tensor([7, 8, -1, 9])
    lengths = torch.tensor([prefix + 30, prefix + 31, prefix, prefix + 5], dtype=torch.int32)

    class State:
        def __init__(self):
            self.pools, self.table, self.lengths = [p.to(gpu) for p in pools], table.to(gpu), lengths.to(gpu)
            self.free, self.start, self.ones = torch.arange(10, 20, dtype=torch.int32, device=gpu), torch.zeros(1, dtype=torch.int32, device=gpu), torch.ones(b, dtype=torch.int32, device=gpu)
            self.x = [t.clone() for t in new[0]]

        def step(self):
            slots, positions, starts, after, start = tpa.tpa_page_tables(self.lengths, self.ones, self.table, self.free, page_size=page, num_tokens=b, free_start=self.start)
            q = tpa.tpa_norm_rope_write(*self.x, h, cos, sin, *self.pools, slots[None], positions=positions[None]).transpose(0, 1)
            out = tpa.tpa_decode_shared(q[..., :h], q[..., h:], *self.pools, prefix_length=prefix, sm_scale=d**-0.5, kv_lengths=after, page_table=self.table)
            self.lengths.copy_(after)
            self.start.copy_(start)
            return out

    State().step()  # the kernels' first launches
    eager, state = State(), State()
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        captured = state.step()
    for x in new:
        for to, t in zip(state.x + eager.x, x + x):
            to.copy_(t)
        want = eager.step()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert not want[0].isnan().any()
        assert all(torch.equal(y, z) for y, z in zip(captured, want))
        assert all(torch.equal(y, z) for y, z in zip([state.table, state.lengths, state.start, *state.pools], [eager.table, eager.lengths, eager.start, *eager.pools]))
    assert eager.lengths.tolist() == [n + steps for n in lengths.tolist()] and int(eager.start) == 3


def test_the_plan_s_borders(gpu):
    """Ranges of one block, of two, of whole tiles that end inside a tile; waves side by side from one to eight, and sharing blocks."""
    for b, lq, prefix, own, h, d, rk in ((1, 1, 17, 16, 8, 64, 2), (1, 2, 33, 31, 8, 128, 1), (2, 1, 2000, 700, 16, 64, 2), (16, 1, 500, 3, 8, 128, 4), (3, 4, 129, 260, 24, 64, 8), (70, 1, 257, 20, 16, 64, 1)):
        for dtype in (BF, F32):
            check(gpu, b, lq, prefix, own, h, d, 3, rk, dtype, 2)
            check(gpu, b, lq, prefix // 32 * 32 + 32, own, h, d, 17, rk, dtype, 2, page=32)


def test_a_row_that_is_not_finite_stays_with_itself(gpu):
    """Infinite and NaN queries of one sequence, in the column sets of others, and non-finite own keys."""
    for dtype, h in ((BF, 8), (BF, 32), (F32, 16)):
        g = torch.Generator().manual_seed(3)
        n = lambda *s: torch.randn(s, generator=g).to(dtype).to(gpu)
        qa, qb, caches = n(6, 1, 5, h), n(6, 1, 5, 64), [n(6, 150, 2, w) for w in (h, 64, h, 64)]
        call = lambda: tpa.tpa_decode_shared(qa, qb, *caches, prefix_length=100, sm_scale=0.125, kernel=2)
        want, want_lse = call()
        qa[1, 0, 2], qb[3, 0, 4, 7], caches[1][4, 120, 1, 3] = math.inf, math.nan, math.nan
        got, lse = call()
        for i in (0, 2, 5):
            assert torch.equal(got[i], want[i]) and torch.equal(lse[i], want_lse[i])
        assert all(got[i].isnan().any() for i in (1, 3, 4))


def test_refusals(gpu):
    n = lambda *s: torch.zeros(s, dtype=BF, device=gpu)
    qa, qb, caches = n(2, 1, 6, 8), n(2, 1, 6, 64), [n(2, 20, 2, w) for w in (8, 64, 8, 64)]
    for prefix in (-1, 21):
        with pytest.raises(ValueError):
            tpa.tpa_decode_shared(qa, qb, *caches, prefix_length=prefix)
    with pytest.raises(ValueError):
        tpa.tpa_decode_shared(qa, qb, *caches, prefix_length=4, kv_lengths=torch.zeros(3, dtype=torch.int32, device=gpu))
    with pytest.raises(ValueError):
        tpa.tpa_decode_shared(qa, qb, *caches, prefix_length=4, causal=3)
    with pytest.raises(AssertionError):
        tpa.tpa_decode_shared(qa, qb[:1], *caches, prefix_length=4)
    with pytest.raises(TypeError):
        tpa.tpa_decode_shared(qa, qb, *(c.float() for c in caches), prefix_length=4)
    need = tpa.decode_shared_workspace_bytes(qa, qb, *caches, prefix_length=4)
    o, _ = tpa.tpa_decode_shared(qa, qb, *caches, prefix_length=4, workspace=torch.empty(need, dtype=torch.uint8, device=gpu))
    assert not o.any()
    with pytest.raises(ValueError):
        tpa.tpa_decode_shared(qa, qb, *caches, prefix_length=4, workspace=torch.empty(1, dtype=torch.uint8, device=gpu).expand(need))


def ranges_of(b, lq, prefix, lk, h, d, rk, qa, qb, caches, table=None):
    """Key ranges that the call's plan has (parts of D + 2 numbers a row and head), and blocks of 32 rows (token, rank) in all."""
    size = tpa.decode_shared_workspace_bytes(qa, qb, *caches, prefix_length=prefix, page_table=table, kernel=2) - 256
    of_block = 32 // rk
    return size // (4 * b * lq * h * (d + 2)), -(-prefix // of_block) + -(-(lk - prefix // of_block * of_block) // of_block)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("where", ["own key", "block of the prefix", "prefix", "query", "query of the first"])
def test_nan_is_not_taken_for_no_key(gpu, dtype, where):
    """NaN where a row sees nothing else in a range of keys: the row's output and lse are NaN, as the formula has it; rows that do not see it keep
    their results, one that sees no key its NaN and -inf."""
    b, h, d, prefix, lk = 5, 16, 64, 160, 200
    g = torch.Generator().manual_seed(11)
    n = lambda *s: torch.randn(s, generator=g).to(dtype).to(gpu)
    qa, qb, caches = n(b, 1, 5, h), n(b, 1, 5, d), [n(b, lk, 2, w) for w in (h, d, h, d)]
    lengths = torch.tensor([161, 200, 160, 0, 40], dtype=torch.int32, device=gpu)
    assert len(set(ranges_of(b, 1, prefix, lk, h, d, 2, qa, qb, caches))) == 1  # every block is a range of its own
    call = lambda kernel: tpa.tpa_decode_shared(qa, qb, *caches, prefix_length=prefix, sm_scale=d**-0.5, kv_lengths=lengths, kernel=kernel)
    clean = {kernel: call(kernel) for kernel in (1, 2)}
    if where == "own key":
        caches[1][0, 160], hit = math.nan, [0]  # the only one behind the prefix
    elif where == "block of the prefix":
        caches[1][0, 48:64], hit = math.nan, [0, 1, 2]
    elif where == "prefix":
        caches[0][0, :160], hit = math.nan, [0, 1, 2, 4]
    elif where == "query":
        qb[1, 0, 3, 7], hit = math.nan, [1]
    else:
        qa[0], hit = math.nan, [0]
    for kernel in (1, 2):
        o, lse = call(kernel)
        for i in range(b):
            if i in hit:
                assert o[i].isnan().all() and lse[i].isnan().all(), (kernel, i)
            elif i == 3:
                assert o[i].isnan().all() and (lse[i] == -math.inf).all(), kernel
            else:
                assert torch.equal(o[i], clean[kernel][0][i]) and torch.equal(lse[i], clean[kernel][1][i]), (kernel, i)


@pytest.mark.parametrize(
    "b,lq,prefix,own,h,d,rk,dtype,page",
    [
        (64, 1, 6000, 40, 32, 128, 2, BF, 64),      # eight waves of columns over the prefix
        (64, 1, 5000, 40, 32, 128, 2, BF, 0),
        (64, 2, 70, 3000, 32, 128, 2, BF, 64),      # own keys
        (24, 4, 500, 2500, 64, 64, 4, BF, 32),      # two blocks of heads, rank 4
        (100, 4, 500, 1500, 8, 128, 8, BF, 0),      # rank 8, a set of four rows
        (33, 3, 1200, 2500, 24, 64, 1, BF, 64),     # 24 heads, rank 1
        (64, 1, 4000, 40, 32, 128, 2, F32, 64),
        (64, 1, 300, 1600, 16, 128, 2, F32, 0),
        (70, 2, 1500, 1500, 32, 64, 4, F32, 48),
    ],
)
def test_ranges_of_many_tiles(gpu, b, lq, prefix, own, h, d, rk, dtype, page):
    """Workgroups that go round the two tile buffers several times, over the prefix and over own keys of all lengths."""
    rq, lk, scale = 6, prefix + own, d**-0.5
    if page:
        lk = -(-lk // page) * page
    g = torch.Generator(device=gpu).manual_seed(b + prefix)
    n = lambda *s: torch.randn(s, generator=g, device=gpu)
    qa, qb = (rq**0.5 * n(b, lq, rq, h)).to(dtype), n(b, lq, rq, d).to(dtype)
    length = prefix + lq + torch.arange(b) * 7919 % (own - lq + 1)
    length[b // 2] = prefix + own
    if page:  # a pool in which nothing but the prefix and the rows' own tokens is a number
        pages, whole = lk // page, prefix // page
        ids = torch.randperm(whole + b * (pages - whole), generator=g, device=gpu)
        table = torch.cat([ids[:whole].expand(b, whole), ids[whole:].view(b, -1)], 1)
        caches = [torch.full((len(ids), page, rk, w), math.nan, dtype=dtype, device=gpu) for w in (h, d, h, d)]
        place = lambda i, t: (table[i, t // page], t % page)
    else:
        table = None
        caches = [torch.full((b, lk, rk, w), math.nan, dtype=dtype, device=gpu) for w in (h, d, h, d)]
        place = lambda i, t: (torch.full_like(t, i), t)
    first = torch.arange(prefix, device=gpu)
    for x, c in enumerate(caches):
        c[place(0, first)] = (n(prefix, rk, c.shape[3]) * (rk**0.5 if x == 0 else 1)).to(dtype)
        for i in range(b):
            t = torch.arange(prefix, int(length[i]), device=gpu)
            c[place(i, t)] = (n(len(t), rk, c.shape[3]) * (rk**0.5 if x == 0 else 1)).to(dtype)
    more = {} if table is None else dict(page_table=table.to(torch.int32).contiguous())
    ranges, blocks = ranges_of(b, lq, prefix, lk, h, d, rk, qa, qb, caches, more.get("page_table"))
    assert blocks >= 3 * (4 if dtype == BF else 2) * ranges
    call = lambda: tpa.tpa_decode_shared(qa, qb, *caches, prefix_length=prefix, sm_scale=scale, kernel=2, kv_lengths=length.to(gpu), causal=2, **more)
    got, got_lse = call()
    assert all(torch.equal(x, y) for x, y in zip(call(), (got, got_lse)))
    assert not got.isnan().any() and not got_lse.isnan().any()
    half, split = torch.finfo(dtype).eps / 2, 2.0**-16 if dtype == BF else 0
    for i in sorted({0, 1, b // 3, b // 2, b - 1}):
        t = torch.arange(prefix, int(length[i]), device=gpu)
        kv = [torch.cat([c[place(0, first)], c[place(i, t)]])[None] for c in caches]
        with torch.device(gpu):
            o, lse, size, xs = oracle(qa[i : i + 1], qb[i : i + 1], kv, prefix, length[i : i + 1].to(gpu), scale, 2, 0)
        logit = (split + (2 * d + rk * rq) * U) * xs
        slack = 2 * logit.transpose(1, 2)[..., None] * size + (half if dtype == BF else 0) * size + (lk + 16) * U * size
        assert ((got_lse[i].double() - lse[0]).abs() <= (logit + (lk + 8) * U + 4 * U * lse.abs())[0]).all(), i
        assert ((got[i].double() - o[0]).abs() <= (half * o.abs() + slack * (1 + half))[0]).all(), i


@pytest.mark.parametrize("dtype", [BF, F32])
def test_pages_whose_rows_are_no_power_of_two(gpu, dtype):
    """Pages of 48 and 80 tokens at rank 2, of 24 at rank 4, of 96 at rank 1: whole blocks of rows, of which a page holds 3 or 5."""
    for page, rk, prefix, lengths in ((48, 2, 200, [230, 480, 201, 192, 300]), (80, 2, 160, [161, 400, 240]), (24, 4, 100, [180, 101, 144]), (96, 1, 96, [97, 300, 96])):
        check(gpu, len(lengths), 1, prefix, max(lengths) - prefix, 16, 64, 6, rk, dtype, 2, page=page, lengths=lengths)
        check(gpu, len(lengths), 3, prefix, max(lengths) - prefix, 8, 128, 6, rk, dtype, 2, page=page, lengths=lengths, causal=2)
