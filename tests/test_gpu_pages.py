"""tpa_pages_fork and tpa_pages_compact against plain walks over the sequences, and a run of a beam search's step.  All results are whole numbers and bytes and have to be equal."""

import numpy as np
import pytest
import torch

import fp4_model as fp4
from tpa import tpa

pytestmark = pytest.mark.gpu


def walk_fork(table, lengths, parents, shares, free, start, pools, page):
    b, per_row = table.shape
    total = len(shares)
    start = max(0, min(start, len(free)))
    inside = lambda p: 0 <= p < total
    lengths = np.clip(lengths, 0, per_row * page)
    shares = np.maximum(shares, 0)
    children = [[i for i, s in enumerate(parents) if s == old] for old in range(b)]
    count, new_table, new_len = shares.copy(), np.zeros((len(parents), per_row), np.int64), np.zeros(len(parents), np.int64)
    at = start
    copies = []
    for i, s in enumerate(parents):
        if not 0 <= s < b:
            continue
        full, tail = divmod(int(lengths[s]), page)
        new_table[i, :full] = table[s, :full]
        new_len[i] = full * page
        if not tail:
            continue
        last = table[s, full]
        if not inside(last) or (children[s][0] == i and shares[last] == 0):
            new_table[i, full], new_len[i] = last, lengths[s]
        else:
            got = free[at] if at < len(free) else -1
            at = min(at + 1, len(free))
            if inside(got):
                copies.append((last, got, tail))
                new_table[i, full], new_len[i] = got, lengths[s]
    for s in range(b):
        full, tail = divmod(int(lengths[s]), page)
        for p in table[s, :full]:
            if inside(p):
                count[p] += len(children[s]) - 1
        if tail and inside(table[s, full]) and not (children[s] and shares[table[s, full]] == 0):
            count[table[s, full]] -= 1
    released = np.nonzero(count < 0)[0]
    new_free = free.copy()
    for j, p in enumerate(released):
        if at - len(released) + j >= 0:
            new_free[at - len(released) + j] = p
    after = [x.copy() for x in pools]
    for x, old in zip(after, pools):
        for src, dst, tail in copies:
            x[dst, :tail] = old[src, :tail]
    return new_table, new_len, np.maximum(count, 0), new_free, np.array([max(0, at - len(released))]), after


def walk_compact(table, lengths, shares, free, start, pools, page):
    total = len(shares)
    start = max(0, min(start, len(free)))
    is_free = np.zeros(total, bool)
    for p in free[start:]:
        if 0 <= p < total:
            is_free[p] = True
    n = total - is_free.sum()
    moved = np.arange(total)
    holes, movers = np.nonzero(is_free[:n])[0], n + np.nonzero(~is_free[n:])[0]
    moved[movers] = holes
    after = [x.copy() for x in pools]
    for x in after:
        x[holes] = x[movers]
    count = np.zeros_like(shares)
    count[moved[~is_free]] = shares[~is_free]
    new_free = free.copy()
    new_free[len(free) - (total - n) :] = np.arange(n, total)
    new_table = np.zeros_like(table)
    for b, length in enumerate(np.clip(lengths, 0, table.shape[1] * page)):
        for e in range(-(-int(length) // page)):
            new_table[b, e] = moved[table[b, e]] if 0 <= table[b, e] < total else table[b, e]
    return new_table, count, new_free, np.array([len(free) - (total - n)]), moved, after


def make_pools(rng, total, page, shapes):
    return [rng.integers(0, 256, (total, page, *s), dtype=np.uint8) for s in shapes]


def dev(gpu, x, dtype=torch.int32):
    return torch.as_tensor(np.asarray(x)).to(dtype).to(gpu)


def check_fork(gpu, table, lengths, parents, shares, free, start, page, shapes=((2, 20),), seed=0, dtype=torch.int32):
    rng = np.random.default_rng(seed)
    table, lengths, shares, free = (np.array(x, np.int64) for x in (table, lengths, shares, free))
    pools = make_pools(rng, len(shares), page, shapes)
    want = walk_fork(table, lengths, parents, shares, free, start or 0, pools, page)
    on_gpu = [torch.from_numpy(x.copy()).to(gpu) for x in pools]
    args = [dev(gpu, x, dtype) for x in (table, lengths, parents, shares, free)]
    kept = [x.clone() for x in args]
    for _ in range(2):  # the same again: nothing that it reads was changed
        got = tpa.tpa_pages_fork(*args, on_gpu, page_size=page, free_start=None if start is None else dev(gpu, [start]))
        for name, g, w in zip(("table", "lengths", "shares", "free", "start"), got, want):
            assert g.dtype == torch.int32 and np.array_equal(g.cpu().numpy(), w), name
        assert all(np.array_equal(g.cpu().numpy(), w) for g, w in zip(on_gpu, want[5]))
        assert all(torch.equal(x, y) for x, y in zip(args, kept))


@pytest.mark.parametrize(
    "table,lengths,parents,shares,free,start,page",
    [
        ([[0]], [1], [0], [0, 0], [0, 1], 1, 1),                                          # the smallest: nothing changes
        ([[3, 1]], [5], [0, 0, 0], [0] * 6, [3, 1, 2, 0, 4, 5], 2, 4),                     # one goes on three times: a page kept, two copied
        ([[3, 1], [0, 5]], [8, 7], [1, 1], [0] * 6, [3, 1, 0, 5, 2, 4], 4, 4),             # one is dropped: whole pages come back
        ([[3, 1], [0, 5]], [8, 7], [], [0] * 6, [3, 1, 0, 5, 2, 4], 4, 4),                 # all are
        ([[3, 1], [0, 5]], [8, 7], [-1, 1, 2, 0, -1], [0] * 6, [3, 1, 0, 5, 2, 4], 4, 4),  # empty rows, other rows
        ([[2, 1], [2, 4]], [6, 7], [0, 0], [0, 0, 1, 0, 0], [2, 1, 4, 0, 3], 3, 4),        # a shared page whose holder is dropped
        ([[2, 1], [2, 4]], [6, 7], [-1, -1], [0, 0, 1, 0, 0], [2, 1, 4, 0, 3], 3, 4),      # and both of its holders
        ([[2, 1]], [6], [0], [0, 1, 0, 0], [2, 1, 0, 3], 2, 4),                            # a last page that somebody else holds: copied even for one
        ([[2, 1]], [6], [0, 0], [0, 0, 0], [2, 1, 0], 3, 4),                               # no page left
        ([[2, 1]], [6], [0, 0, 0], [0, 0, 0], [2, 1, 0], 2, 4),                            # one page left for two
        ([[2, 1]], [6], [0, 0, 0], [0, 0, 0], [2, 1, 99, 0], 2, 4),                        # a page of the list outside the pools
        ([[2, -1], [7, 0]], [8, 3], [0, 0, 1, 1], [0, 0, 0], [1], 0, 4),                   # entries outside the pools
        ([[2, 1]], [99], [0, 0], [0, 0, 0], [0], 0, 4),                                    # a length past the row
        ([[2, 1]], [-3], [0, 0], [0, 0, 0], [0], 0, 4),
        ([[2, 1]], [5], [-1], [0, 0, 0], [], None, 4),                                     # no list: nowhere to put them
        ([[2, 1]], [5], [-1], [0, 0, -9], [0, 0, 0], 1, 4),                                # room for one of two; a count below zero
        ([[2, 1]], [5], [0, 0], [0, 0, 0], [0], -5, 4),                                    # a start outside the list
    ],
)
def test_fork(gpu, table, lengths, parents, shares, free, start, page):
    check_fork(gpu, table, lengths, parents, shares, free, start, page)


@pytest.mark.parametrize("seed,b,m,pages,page,extra,shapes", [
    (0, 40, 40, 9, 4, 30, ((2, 20), (3,))),           # rows of 40 and of 3 bytes
    (1, 300, 500, 3, 16, 300, ((1, 32), (2, 8, 5))),
    (2, 7, 2000, 2, 5, 900, ((4,),)),
    (3, 1200, 1100, 30, 2, 50, ((16,),)),             # pages in several ranges of the count
    (4, 3, 3, 2, 300, 3, ((2, 88), (7,))),            # pages of several chunks
])
def test_fork_of_many(gpu, seed, b, m, pages, page, extra, shapes):
    """Sequences that share pages at several places, in the order of a real search: forked, grown, forked again."""
    rng = np.random.default_rng(seed)
    total = b * pages + extra
    ids = rng.permutation(total)
    table = ids[: b * pages].reshape(b, pages).copy()
    lengths = rng.integers(0, pages * page + 1, b)
    shares = np.zeros(total, np.int64)
    for s in range(1, b):
        if rng.random() < 0.5:  # the first pages are those of the sequence before
            n = int(min(lengths[s], lengths[s - 1]) // page * rng.random())
            table[s, :n] = table[s - 1, :n]
    used = np.arange(pages) < (-(-lengths // page))[:, None]
    np.add.at(shares, table[used], 1)
    shares = np.maximum(shares - 1, 0)
    parents = rng.integers(-1, b, m)
    check_fork(gpu, table, lengths, parents, shares, np.concatenate([ids]), b * pages, page, shapes, seed, torch.int64)


def test_more_pools_than_a_launch_takes(gpu):
    check_fork(gpu, [[3, 1], [0, 5]], [6, 7], [1, 1, 0], [0] * 6, [3, 1, 0, 5, 2, 4], 4, 4, ((1, 8),) * 200)


def check_compact(gpu, table, lengths, shares, free, start, page, shapes=((2, 20),), seed=0):
    rng = np.random.default_rng(seed)
    table, lengths, shares, free = (np.array(x, np.int64) for x in (table, lengths, shares, free))
    pools = make_pools(rng, len(shares), page, shapes)
    want = walk_compact(table, lengths, shares, free, start or 0, pools, page)
    on_gpu = [torch.from_numpy(x.copy()).to(gpu) for x in pools]
    args = [dev(gpu, x) for x in (table, lengths, shares, free)]
    for _ in range(2):
        got = tpa.tpa_pages_compact(*args, on_gpu, page_size=page, free_start=None if start is None else dev(gpu, [start]))
        for name, g, w in zip(("table", "shares", "free", "start", "moved"), got, want):
            assert g.dtype == torch.int32 and np.array_equal(g.cpu().numpy(), w), name
        assert all(np.array_equal(g.cpu().numpy(), w) for g, w in zip(on_gpu, want[5]))


@pytest.mark.parametrize(
    "table,lengths,shares,free,start,page",
    [
        ([[0]], [1], [4], [0], 1, 1),                                   # one page, in use
        ([[0]], [0], [0], [0], 0, 1),                                   # one page, free
        ([[5, 3], [4, 0]], [6, 4], [9, 0, 0, 1, 2, 3], [5, 3, 4, 0, 1, 2], 4, 4),
        ([[5, 3], [4, 0]], [6, 4], [9, 0, 0, 1, 2, 3], [], None, 4),     # no page is free
        ([[0, 1]], [8], [1, 2, 3, 4], [0, 1, 3, 2], 2, 4),               # nothing to move
        ([[3, 9], [-1, 2]], [8, 8], [1, 2, 3, 4], [0, 1, 1, 77, -5], 0, 4),  # a list with a page twice and pages outside; entries outside
        ([[3, 2]], [100], [1, 2, 3, 4], [1, 0], -3, 4),
    ],
)
def test_compact(gpu, table, lengths, shares, free, start, page):
    check_compact(gpu, table, lengths, shares, free, start, page)


@pytest.mark.parametrize("seed,total,holes,page,shapes", [(0, 33, 0.5, 4, ((3,), (2, 16))), (1, 5000, 0.3, 2, ((20,),)), (2, 40000, 0.9, 1, ((16,),)), (3, 40001, 0.02, 1, ((5,),)), (4, 40, 0.4, 300, ((2, 88),))])
def test_compact_of_many(gpu, seed, total, holes, page, shapes):
    rng = np.random.default_rng(seed)
    ids = rng.permutation(total)
    n = int(total * (1 - holes))
    per_row = max(1, n // 50)
    table = ids[: n // per_row * per_row].reshape(-1, per_row)
    check_compact(gpu, table, rng.integers(0, per_row * page + 1, len(table)), rng.integers(0, 5, total), ids, n, page, shapes, seed)


def test_types_strides_and_what_is_refused(gpu):
    total, page = 6, 4
    wide = torch.arange(total * 2 * page * 3, dtype=torch.float32, device=gpu).view(total, 2, page, 3)
    pool = wide[:, 1]  # pages apart
    table, lengths, parents = dev(gpu, [[3, 1]]), dev(gpu, [6]), dev(gpu, [0, 0])
    shares, free = dev(gpu, [0] * total), dev(gpu, [3, 1, 0, 2, 4, 5])
    before = wide.clone()
    out = tpa.tpa_pages_fork(table, lengths, parents.view(1, 2), shares, free, (pool, torch.zeros(total, page, 0, device=gpu)), page_size=page, free_start=dev(gpu, [2]))
    before[0, 1, :2] = before[1, 1, :2]
    assert torch.equal(wide, before) and out[0].tolist() == [[3, 1], [3, 0]] and out[1].tolist() == [6, 6]
    ok = dict(page_size=page)
    with pytest.raises(ValueError):
        tpa.tpa_pages_fork(table, lengths, parents, shares, free, [wide.transpose(1, 2)], **ok)  # tokens in pieces
    with pytest.raises(ValueError):
        tpa.tpa_pages_fork(table, lengths, parents, shares, free, [wide[:1, 1].expand(total, page, 3)], **ok)  # one page for all
    with pytest.raises(ValueError):
        tpa.tpa_pages_compact(table, lengths, shares, free, [pool[:5]], **ok)
    with pytest.raises(TypeError):
        tpa.tpa_pages_compact(table, lengths, shares, free, [pool.cpu()], **ok)
    with pytest.raises(TypeError):
        tpa.tpa_pages_compact(table, lengths, shares.float(), free, [pool], **ok)


def test_captured(gpu):
    rng = np.random.default_rng(0)
    total, page = 40, 4
    table, lengths = dev(gpu, rng.permutation(total)[:24].reshape(4, 6)), dev(gpu, [22, 9, 13, 24])
    shares, free, start = dev(gpu, [0] * total), dev(gpu, np.arange(total)), dev(gpu, [24])
    parents = dev(gpu, [0, 0, 1, 3])
    pool = torch.from_numpy(rng.integers(0, 256, (total, page, 8), dtype=np.uint8)).to(gpu)
    calls = (lambda p: tpa.tpa_pages_fork(table, lengths, parents, shares, free, [p], page_size=page, free_start=start),
             lambda p: tpa.tpa_pages_compact(table, lengths, shares, free, [p], page_size=page, free_start=start))
    for call in calls:
        call(pool.clone())
        torch.cuda.synchronize()
        mine = pool.clone()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got = call(mine)
        for i in range(4):
            parents.copy_(dev(gpu, rng.integers(-1, 4, 4)))
            mine.copy_(pool)
            other = pool.clone()
            want = call(other)
            torch.cuda.synchronize()
            graph.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(x, y) for x, y in zip(got, want)) and torch.equal(mine, other)


@pytest.mark.parametrize("beams,page", [(3, 4), (4, 16)])
def test_a_search_over_a_cache_in_4_bits(gpu, beams, page):
    """Prompts, then steps of selection, pages, new tokens and attention; every sequence's cache is at all times what its own history of tokens would have written, and its
    attention is that over a contiguous cache of this history."""
    rng = np.random.default_rng(beams)
    b, h, d, rq, rk, vocab, steps, per_row, total = 2, 8, 64, 3, 2, 50, 12, 12, 140
    rows, n = b * beams, fp4.row_bytes(h, d)
    pools = [torch.zeros(total, page, rk, n, dtype=torch.uint8, device=gpu) for _ in range(2)]
    factors = torch.from_numpy(rng.standard_normal((2, 400, vocab, rk, h + d), np.float32)).to(gpu)  # of a token at a position
    table, lengths = dev(gpu, np.zeros((rows, per_row))), dev(gpu, [0] * rows)
    shares, free, start = dev(gpu, [0] * total), dev(gpu, rng.permutation(total)), dev(gpu, [0])
    scores = torch.full((b, beams), -float("inf"), device=gpu)
    scores[:, 0] = 0
    finished = torch.zeros(b, beams, dtype=torch.bool, device=gpu)
    history = [[] for _ in range(rows)]

    def append(tokens):
        nonlocal lengths, start
        news = dev(gpu, [len(t) for t in tokens])
        count = sum(len(t) for t in tokens)
        slots, positions, _, lengths, start = tpa.tpa_page_tables(lengths, news, table, free, page_size=page, num_tokens=count + 3, free_start=start)
        flat = torch.tensor([t for seq in tokens for t in seq] + [0] * 3, device=gpu)
        k, v = (f[positions.long(), flat] for f in factors)
        tpa.tpa_cache_write_fp4(k[None], v[None], h, *pools, slots[None])
        for seq, t in zip(history, tokens):
            seq.extend(t)

    append([rng.integers(0, vocab, 7 if i < beams else 3).tolist() if i % beams == 0 else [] for i in range(rows)])
    # the other beams start as copies of the first
    table, lengths, shares, free, start = tpa.tpa_pages_fork(table, lengths, dev(gpu, [i // beams * beams for i in range(rows)]), shares, free, pools, page_size=page, free_start=start)
    history = [list(history[i // beams * beams]) for i in range(rows)]
    for step in range(steps):
        logits = torch.from_numpy(rng.standard_normal((b, beams, vocab), np.float32)).to(gpu)
        scores, parents, tokens, finished = tpa.tpa_beam_select(logits, scores, finished=finished, eos_token=0)
        table, lengths, shares, free, start = tpa.tpa_pages_fork(table, lengths, parents, shares, free, pools, page_size=page, free_start=start)
        history = [list(history[i]) for i in parents.flatten().tolist()]
        if step == 7:
            table, shares, free, start, moved = tpa.tpa_pages_compact(table, lengths, shares, free, pools, page_size=page, free_start=start)
            in_use = int(start)
            assert sorted(set(table[torch.arange(per_row, device=gpu) < ((lengths + page - 1) // page)[:, None]].tolist())) == list(range(in_use))
        append([[t] for t in tokens.flatten().tolist()])
        assert lengths.tolist() == [len(x) for x in history]
        # pages: as many holders as the counts say
        used = table[torch.arange(per_row, device=gpu) < ((lengths + page - 1) // page)[:, None]]
        holders = torch.bincount(used, minlength=total)
        assert torch.equal((holders - 1).clamp(min=0).int(), shares) and int(start) == int((holders > 0).sum())
        q = torch.from_numpy(rng.standard_normal((rows, 1, rq, h + d), np.float32)).to(gpu)
        got = tpa.tpa_decode_fp4(q[..., :h], q[..., h:], *pools, 0.1, kv_lengths=lengths, page_table=table)
        most = max(len(x) for x in history)
        flat = [torch.zeros(rows, most, rk, n, dtype=torch.uint8, device=gpu) for _ in range(2)]
        slots = torch.full((rows, most), -1, dtype=torch.int32)
        ids = torch.zeros(rows, most, dtype=torch.long)
        for i, seq in enumerate(history):
            slots[i, : len(seq)] = i * most + torch.arange(len(seq), dtype=torch.int32)
            ids[i, : len(seq)] = torch.tensor(seq)
        k, v = (f[torch.arange(most, device=gpu), ids.to(gpu)] for f in factors)
        tpa.tpa_cache_write_fp4(k, v, h, *flat, slots.to(gpu))
        want = tpa.tpa_decode_fp4(q[..., :h], q[..., h:], *flat, 0.1, kv_lengths=lengths)
        assert all(torch.equal(x, y) for x, y in zip(got, want))
