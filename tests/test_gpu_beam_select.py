"""tpa_beam_select against its definition in 64 bits.  Whole numbers have to be equal; a score is off by half a step of fp32 and what the logarithm of the sum is off by
(exponentials right to 2^-22 of themselves, sums of no more than 512 terms in a row in fp32: 2^-15 at the very most, 2^-21 allowed here for numbers of one size)."""

import numpy as np
import pytest
import torch

from tpa import tpa

pytestmark = pytest.mark.gpu


def definition(logits, scores, k, finished, eos):
    x = logits.double().cpu().numpy()
    s = scores.double().cpu().numpy()
    b, n, vocab = x.shape
    with np.errstate(all="ignore"):
        most = x.max(-1, keepdims=True)
        value = s[..., None] + (x - most - np.log(np.exp(x - most).sum(-1, keepdims=True)))
    done = np.zeros((b, n), bool) if finished is None else finished.cpu().numpy()
    value[done] = -np.inf
    if done.any():
        value[..., eos] = np.where(done, s, value[..., eos])
    value[np.isnan(value) | np.isposinf(value)] = -np.inf
    value = value.reshape(b, -1)
    at = np.argsort(-value, axis=1, kind="stable")[:, :k]
    beam, token = at // vocab, at % vocab
    out = np.take_along_axis(value, at, 1)
    return out, beam + n * np.arange(b)[:, None], token, np.take_along_axis(done, beam, 1) | (token == (-1 if eos is None else eos))


def check(logits, scores, k=None, finished=None, eos=None):
    want = definition(logits, scores, k or logits.shape[1], finished, eos)
    got = tpa.tpa_beam_select(logits, scores, num_out=k, finished=finished, eos_token=eos)
    assert [x.dtype for x in got] == [torch.float32, torch.int32, torch.int32, torch.bool]
    for g, w in zip(got[1:], want[1:]):
        assert np.array_equal(g.cpu().numpy(), w)
    g, w = got[0].double().cpu().numpy(), want[0]
    assert np.array_equal(np.isinf(g), np.isinf(w))
    fine = np.isfinite(w)
    assert (abs(g[fine] - w[fine]) <= 2.0**-24 * abs(w[fine]) + 2.0**-21).all()


def inputs(gpu, seed, b, n, vocab, dtype, spread=2.5):
    g = torch.Generator().manual_seed(seed)
    return (spread * torch.randn(b, n, vocab, generator=g)).to(dtype).to(gpu), (-10 * torch.rand(b, n, generator=g)).to(gpu)


BOTH = pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])


@BOTH
@pytest.mark.parametrize("vocab", [1, 2, 63, 511, 512, 513, 1024, 1025, 5000, 33000])
@pytest.mark.parametrize("b,n", [(1, 1), (2, 3), (5, 4)])
def test_sizes(gpu, b, n, vocab, dtype):
    check(*inputs(gpu, vocab, b, n, vocab, dtype), k=min(n, n * vocab))


@BOTH
@pytest.mark.parametrize("n,k", [(1, 1), (1, 64), (2, 4), (5, 10), (16, 16), (64, 64), (3, 1)])
def test_widths(gpu, n, k, dtype):
    check(*inputs(gpu, k, 3, n, 1500, dtype), k=k)


@BOTH
def test_a_large_vocabulary(gpu, dtype):
    check(*inputs(gpu, 1, 24, 8, 60000, dtype))


@BOTH
@pytest.mark.parametrize("b,n,k,vocab", [(1, 16, 16, 160000), (2, 64, 64, 5000), (1, 64, 8, 70001), (3, 5, 64, 20000)])
def test_many_beams_with_many_continuations(gpu, b, n, k, vocab, dtype):
    """More candidates than the second launch copies, in more lists than it copies the first of, and lists that hold most of what wins."""
    logits, scores = inputs(gpu, 11, b, n, vocab, dtype)
    check(logits, scores, k=k)
    logits[:, 0, 100:100 + k] += 20.0
    check(logits, scores, k=k)
    check(torch.zeros_like(logits), torch.zeros_like(scores), k=k)


@BOTH
def test_ties_go_to_the_lower_index(gpu, dtype):
    for b, n, vocab, levels in ((2, 1, 3000, 3), (1, 1, 2100, 1), (2, 4, 700, 2)):
        x = torch.randint(0, levels, (b, 1, vocab), generator=torch.Generator().manual_seed(vocab)).to(dtype).to(gpu).expand(b, n, vocab)
        check(x, torch.zeros(b, n, device=gpu), k=min(16, n * vocab))  # beams that are alike: ties between them too
    zeros = torch.zeros(1, 2, 600, device=gpu, dtype=dtype)
    zeros[0, 0, 10:20] = -0.0
    check(zeros, torch.zeros(1, 2, device=gpu), k=32)
    rising = torch.arange(2048, device=gpu).to(dtype)[None, None] / 64  # every logit goes in
    check(rising, torch.zeros(1, 1, device=gpu), k=40)


@BOTH
def test_finished_beams(gpu, dtype):
    logits, scores = inputs(gpu, 4, 6, 4, 1100, dtype)
    finished = torch.rand(6, 4, generator=torch.Generator().manual_seed(5)) < 0.4
    finished[0], finished[1] = True, False
    scores[2] = -0.5  # a finished beam's score beats what the others can reach
    logits[3, :, 7] = 30.0  # and so does the end of one that goes on
    check(logits, scores, finished=finished.to(gpu), eos=7)
    check(logits, scores, k=9, finished=finished.to(gpu), eos=7)
    check(logits, scores, eos=7)


@BOTH
def test_masked_logits_and_dead_beams(gpu, dtype):
    inf = float("inf")
    logits, scores = inputs(gpu, 6, 7, 3, 1300, dtype)
    logits[0, :, 5:] = -inf              # fewer tokens than continuations
    logits[1] = -inf                     # none at all: the lowest indices
    logits[2, 0, 17] = float("nan")       # a beam that is no number
    logits[3, 1, 3] = inf
    scores[4, 1:] = -inf                 # the first step: one beam
    scores[5, 0], scores[6, 2] = float("nan"), inf
    check(logits, scores, k=20)
    logits[2, :, 40] = float("nan")
    check(logits, scores, k=3)
    check(logits[:, :, :4], scores, k=12)


@BOTH
def test_logits_far_apart(gpu, dtype):
    """Chunks of which one holds all of the sum, in either order, and large magnitudes."""
    logits, scores = inputs(gpu, 8, 2, 2, 4000, dtype, spread=1.0)
    logits[0, 0, :1024] -= 30000
    logits[0, 1, 1024:] -= 30000
    logits[1] *= 1000
    check(logits, scores, k=6)


@BOTH
def test_strides_and_types(gpu, dtype):
    g = torch.Generator().manual_seed(9)
    base = torch.randn(3, 2, 5, 1201, generator=g).to(dtype).to(gpu)
    scores = -torch.rand(3, 2, generator=g).to(gpu)
    check(base[:, :, 2, 1:1100], scores)                     # rows at odd places
    check(base[:, :, 0, ::3], scores)                        # a strided vocabulary
    check(base[:, :1, 1].expand(3, 2, 1201), scores)         # one row for all beams
    check(base[:, :, 3], scores.double())
    check(base[:, :, 3].transpose(0, 1).contiguous().transpose(0, 1), scores)


def test_empty_and_other_streams_and_graphs(gpu):
    out = tpa.tpa_beam_select(torch.empty(0, 4, 100, device=gpu), torch.empty(0, 4, device=gpu))
    assert [tuple(x.shape) for x in out] == [(0, 4)] * 4
    logits, scores = inputs(gpu, 10, 3, 4, 3000, torch.float32)
    finished = torch.zeros(3, 4, dtype=torch.bool, device=gpu)
    call = lambda: tpa.tpa_beam_select(logits, scores, finished=finished, eos_token=2)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        got = call()
    torch.cuda.current_stream().wait_stream(stream)
    assert all(torch.equal(x, y) for x, y in zip(got, call()))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = call()
    for i in range(4):
        logits.copy_(inputs(gpu, 20 + i, 3, 4, 3000, torch.float32)[0])
        finished[:, i] = True
        want = call()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(got, want))
