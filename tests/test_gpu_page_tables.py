"""tpa_page_tables (page tables, slots and positions of a step's new tokens) against a plain walk over the requests, and its refusals.
All results are whole numbers and have to be equal."""

import numpy as np
import pytest
import torch

from tpa import tpa

pytestmark = pytest.mark.gpu


def walk(lengths, news, table, free, page, rows, start):
    """The definition, request by request and token by token."""
    table = table.copy()
    cap = table.shape[1] * page
    slots, positions = np.full(rows, -1, np.int32), np.zeros(rows, np.int32)
    starts, after, row, at = [0], [], 0, max(0, min(start, len(free)))
    for b, (length, new) in enumerate(zip(lengths, news)):
        length, new = max(0, min(length, cap)), min(max(new, 0), rows - row)
        have = -(-length // page)
        want = -(-min(length + new, cap) // page) - have
        got = min(want, len(free) - at)
        table[b, have : have + got] = free[at : at + got]
        end = min(length + new, cap) if got == want else (have + got) * page
        for i in range(new):
            positions[row + i] = length + i
            if length + i < end:
                slots[row + i] = table[b, (length + i) // page] * page + (length + i) % page
        at += got
        row += new
        starts.append(row)
        after.append(end)
    return slots, positions, np.array(starts), np.array(after), np.array([at]), table


def check(gpu, lengths, news, pages, page, rows, n_free, start, seed=0):
    rng = np.random.default_rng(seed)
    ids = rng.permutation(len(lengths) * pages + n_free).astype(np.int32)
    table, free = ids[: len(lengths) * pages].reshape(len(lengths), pages).copy(), ids[len(lengths) * pages :].copy()
    want = walk(lengths, news, table, free, page, rows, start or 0)
    dev = lambda x: torch.tensor(np.asarray(x), dtype=torch.int32, device=gpu)
    t = dev(table)
    got = tpa.tpa_page_tables(dev(lengths), dev(news), t, dev(free), page_size=page, num_tokens=rows, free_start=None if start is None else dev([start]))
    for name, g, w in zip(("slots", "positions", "starts", "new_kv_lengths", "new_free_start", "page_table"), (*got, t), want):
        assert g.dtype == torch.int32 and g.cpu().tolist() == w.tolist(), name


@pytest.mark.parametrize(
    "lengths,news,pages,page,rows,n_free,start",
    [
        ([0], [1], 1, 1, 1, 1, None),                        # the smallest step
        ([5], [0], 2, 4, 0, 3, 0),                           # no new token, no row
        ([0, 3, 4, 7], [1, 1, 1, 1], 2, 4, 4, 9, 2),         # first page, inside a page, at a page's end
        ([0, 0, 0], [0, 9, 0], 4, 4, 16, 4, 1),              # requests without tokens beside one with three pages, padding
        ([6, 2], [5, 9], 2, 4, 14, 9, 0),                    # past the end of the table's row
        ([3, 3, 3], [6, 6, 6], 4, 4, 18, 4, 1),              # the free list runs out inside the second request
        ([4, 4], [4, 4], 4, 4, 8, 0, None),                  # no free page at all
        ([1, 1], [3, 3], 4, 4, 8, 5, 99),                    # start behind the list's end; no page is needed
        ([-2, 50, 2], [-1, 3, 2], 3, 8, 6, 5, -4),           # lengths, counts and a start outside their ranges
        ([0, 0], [7, 7], 4, 4, 10, 9, 0),                    # more tokens than rows: the rest has none
        ([2147483647, 0], [2147483647, 2147483647], 4, 4, 20, 9, 0),
    ],
)
def test_steps(gpu, lengths, news, pages, page, rows, n_free, start):
    check(gpu, lengths, news, pages, page, rows, n_free, start)


@pytest.mark.parametrize("b,most,page,pages", [(64, 1, 64, 8), (255, 40, 16, 9), (256, 3, 1, 12), (257, 700, 16, 60), (1031, 5, 7, 11), (8192, 2, 32, 3)])
@pytest.mark.parametrize("scarce", [False, True])
def test_many_requests(gpu, b, most, page, pages, scarce):
    rng = np.random.default_rng(b)
    lengths, news = rng.integers(0, pages * page, b).tolist(), rng.integers(0, most + 1, b).tolist()
    rows = sum(news) + (0 if scarce else 77)
    check(gpu, lengths, news, pages, page, rows, b * pages // (8 if scarce else 1) + 3, 3, seed=b)


def test_numpy_lengths_and_int64(gpu):
    t = torch.zeros((2, 4), dtype=torch.int32, device=gpu)
    got = tpa.tpa_page_tables(np.array([0, 5]), torch.tensor([2, 1], device=gpu), t, torch.arange(10, 20, device=gpu), page_size=4, num_tokens=3)
    assert got[0].tolist() == [40, 41, 1] and t.tolist() == [[10, 0, 0, 0], [0, 0, 0, 0]]


def test_replays_from_a_graph_and_on_another_stream(gpu):
    """Three decode steps captured once: the lengths, the table and the free list's start go from step to step on the GPU."""
    b, page, pages = 5, 4, 6
    lengths0 = torch.tensor([0, 3, 4, 9, 15], dtype=torch.int32, device=gpu)
    news, free = torch.ones(b, dtype=torch.int32, device=gpu), torch.arange(40, 70, dtype=torch.int32, device=gpu)
    table0 = torch.arange(b * pages, dtype=torch.int32, device=gpu).view(b, pages)
    lengths, table, start = lengths0.clone(), table0.clone(), torch.zeros(1, dtype=torch.int32, device=gpu)

    def step():
        slots, _, _, after, at = tpa.tpa_page_tables(lengths, news, table, free, page_size=page, num_tokens=b, free_start=start)
        lengths.copy_(after)
        start.copy_(at)
        return slots

    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        step()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            captured = step()
    torch.cuda.synchronize()
    lengths.copy_(lengths0)
    table.copy_(table0)
    start.zero_()
    at, t, n = 0, table0.cpu().numpy(), lengths0.tolist()
    for _ in range(6):
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        want = walk(n, [1] * b, t, free.cpu().numpy(), page, b, at)
        t, n, at = want[5], want[3].tolist(), int(want[4][0])
        assert captured.tolist() == want[0].tolist() and table.cpu().tolist() == t.tolist() and lengths.tolist() == n and start.tolist() == [at]


def test_refusals(gpu):
    t = torch.zeros((2, 4), dtype=torch.int32, device=gpu)
    n = torch.zeros(2, dtype=torch.int32, device=gpu)
    with pytest.raises(TypeError):
        tpa.tpa_page_tables(n, n, t.cpu(), n, page_size=4, num_tokens=2)
    for bad in (t.long(), t.T, t[0]):
        with pytest.raises(ValueError):
            tpa.tpa_page_tables(n, n, bad, n, page_size=4, num_tokens=2)
    with pytest.raises(ValueError):
        tpa.tpa_page_tables(n[:1], n, t, n, page_size=4, num_tokens=2)
    with pytest.raises(ValueError):
        tpa.tpa_page_tables(n, n, t, n, page_size=0, num_tokens=2)
    with pytest.raises(ValueError):
        tpa.tpa_page_tables(n, n, t, n, page_size=4, num_tokens=-1)
    with pytest.raises(ValueError):
        tpa.tpa_page_tables(n, n, t, n, page_size=4, num_tokens=1, free_start=n)


def test_under_inference_mode(gpu):
    with torch.inference_mode():
        table = torch.full((2, 4), -1, dtype=torch.int32, device=gpu)
        free = torch.arange(5, 13, dtype=torch.int32, device=gpu)
        slots, positions, starts, after, start = tpa.tpa_page_tables(torch.tensor([0, 0], device=gpu), torch.tensor([3, 9], device=gpu), table, free, page_size=4, num_tokens=14)
        after = after + 1
    assert slots.tolist() == [20, 21, 22, 24, 25, 26, 27, 28, 29, 30, 31, 32, -1, -1] and starts.tolist() == [0, 3, 12]
    assert after.tolist() == [4, 10] and int(start) == 4 and table.tolist() == [[5, -1, -1, -1], [6, 7, 8, -1]] and positions[:3].tolist() == [0, 1, 2]


@pytest.mark.parametrize("rows", [2**31 - 1, 2**31 - 300])
def test_the_most_rows(gpu, rows):
    """As many rows as 31 bits hold: the padding behind the tokens ends with the arrays."""
    table, free = torch.zeros((2, 4), dtype=torch.int32, device=gpu), torch.arange(9, dtype=torch.int32, device=gpu)
    slots, positions, starts, after, start = tpa.tpa_page_tables(torch.tensor([0, 3], device=gpu), torch.tensor([2, 1], device=gpu), table, free, page_size=4, num_tokens=rows)
    assert slots[:3].tolist() == [0, 1, 3] and positions[:3].tolist() == [0, 1, 3] and starts.tolist() == [0, 2, 3] and after.tolist() == [2, 4] and start.tolist() == [1]
    for first in range(3, rows, 2**28):
        assert (slots[first : first + 2**28] == -1).all() and not positions[first : first + 2**28].any()
    assert len(slots) == len(positions) == rows


def test_pages_whose_slots_31_bits_do_not_hold(gpu):
    """A page so far back, or no page at all (-1, or anything below zero), gives no slot, never another page's."""
    far = 2**31 // 16
    table = torch.tensor([[far, 3], [-1, 3], [-far - 1, 3], [far - 1, 3]], dtype=torch.int32, device=gpu)
    free = torch.tensor([far * 2, -5, far + 7, far - 2], dtype=torch.int32, device=gpu)
    got = tpa.tpa_page_tables(torch.tensor([2, 2, 2, 2], device=gpu), torch.ones(4, dtype=torch.int32, device=gpu), table, free, page_size=16, num_tokens=4)
    assert got[0].tolist() == [-1, -1, -1, (far - 1) * 16 + 2] and got[1].tolist() == [2] * 4
    got = tpa.tpa_page_tables(torch.tensor([16, 16, 16, 16], device=gpu), torch.ones(4, dtype=torch.int32, device=gpu), table, free, page_size=16, num_tokens=4)
    assert got[0].tolist() == [-1, -1, -1, (far - 2) * 16] and got[4].tolist() == [4]


@pytest.mark.parametrize("page,pages", [(2**31 - 1, 1), (2**30, 1), (2**30 - 1, 2), (2**29 + 5, 3)])
def test_the_largest_pages(gpu, page, pages):
    """Pages whose sizes 31 bits just hold, request by request in Python's integers; a slot past 31 bits is none, a position past them is their end."""
    cap, n_free, rows, most = page * pages, 9, 23, 2**31 - 1
    lengths, news = [0, 1, 2, cap - 3, cap, page, page - 1, cap - 1], [3, 1, 4, 9, 2, 1, 2, 1]
    ids = list(range(len(lengths) * pages + n_free))
    table, free = [ids[i * pages : (i + 1) * pages] for i in range(len(lengths))], ids[len(lengths) * pages :]
    dev = lambda x: torch.tensor(x, dtype=torch.int32, device=gpu)
    got_table = dev(table)
    got = tpa.tpa_page_tables(dev(lengths), dev(news), got_table, dev(free), page_size=page, num_tokens=rows, free_start=dev([1]))
    slots, positions, starts, after, at = [], [], [0], [], 1
    for row, length, new in zip(table, lengths, news):
        have = -(-length // page)
        opened = max(0, -(-min(length + new, cap) // page) - have)
        row[have : have + opened] = free[at : at + opened]
        at += opened
        for position in range(length, length + new):
            slot = row[position // page] * page + position % page if position < cap else -1
            slots.append(slot if slot <= most else -1)
            positions.append(min(position, most))
        starts.append(len(slots))
        after.append(min(length + new, cap))
    assert len(slots) == rows and at <= n_free
    for name, g, w in zip(("slots", "positions", "starts", "new_kv_lengths", "new_free_start", "page_table"), (*got, got_table), (slots, positions, starts, after, [at], table)):
        assert g.tolist() == w, name


def test_no_requests(gpu):
    """A step in which nothing runs: rows of padding, no page taken; the free list's start inside the list."""
    none = torch.zeros(0, dtype=torch.int32, device=gpu)
    table, free = torch.zeros((0, 4), dtype=torch.int32, device=gpu), torch.arange(9, dtype=torch.int32, device=gpu)
    for rows, start, want in ((5, None, 0), (0, 3, 3), (700, 99, 9), (1, -2, 0)):
        got = tpa.tpa_page_tables(none, none, table, free, page_size=4, num_tokens=rows, free_start=None if start is None else torch.tensor([start], device=gpu))
        assert [t.tolist() for t in got] == [[-1] * rows, [0] * rows, [0], [], [want]] and all(t.dtype == torch.int32 for t in got)
