"""tpa_beam_select where logits are masked by large finite numbers, against its definition in 64 bits.

Whole numbers have to be equal.  A score is off by half a step of fp32 and by the logarithm of the sum.  With d a logit's distance from the beam's largest: a term is
exp2 of a product whose factors and result are rounded (2 |d| 2^-24 of the term, along the whole way to the beam's largest), the hardware's exponential is off by 2^-23, and
a lane has at most 16 batches: 18 exponentials one behind the other (36 2^-24) and 16 + 3 sums in fp32 (19 2^-24), the rest is in 64 bits.  The mean of |d| over the
softmax's weights is the entropy less the logarithm of the sum, at most ln(vocab).  So the logarithm is off by (2 ln(vocab) + 60) 2^-24.
"""

import math

import numpy as np
import pytest
import torch

from test_gpu_beam_select import definition, inputs
from tpa import tpa

pytestmark = pytest.mark.gpu
BOTH = pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
LOWEST = "lowest"


def check(logits, scores, k, **options):
    vocab = logits.shape[-1]
    want = definition(logits, scores, k, options.get("finished"), options.get("eos_token"))
    got = tpa.tpa_beam_select(logits, scores, num_out=k, **options)
    for name, g, w in zip(("parents", "tokens", "finished"), got[1:], want[1:]):
        assert np.array_equal(g.cpu().numpy(), w), name
    g, w = got[0].double().cpu().numpy(), want[0]
    assert np.array_equal(np.isinf(g), np.isinf(w))
    fine = np.isfinite(w)
    assert (abs(g[fine] - w[fine]) <= 2.0**-24 * abs(w[fine]) + (2 * math.log(vocab) + 60) * 2.0**-24).all()


def mask(logits, value):
    """In each request another part of the vocabulary; the last request has whole beams."""
    value = torch.finfo(logits.dtype).min if value == LOWEST else value
    keep = logits[1, :, [3, 700, 701, 2500, 4999]].clone()
    logits[0, :, 4000:] = value             # a tail: whole chunks and a part of one
    logits[1] = value                       # all but a few tokens
    logits[1, :, [3, 700, 701, 2500, 4999]] = keep
    logits[2, :, 8:16] = value              # eight neighbours, in a chunk's first batch
    logits[2, 0, 1024 : 1024 + 512] = value  # a whole first batch
    logits[3, :, 40:48] = value             # eight neighbours in both batches of a chunk
    logits[3, :, 512 + 40 : 512 + 48] = value
    logits[4, :, ::2] = value               # every other one
    logits[4, 1, : 4096] = value
    logits[5, :2] = value                   # two whole beams of three
    logits[6] = value                       # and all
    return logits


@BOTH
@pytest.mark.parametrize("value", [-1e5, -1e9, -1e10, -1e11, -1e12, -1e18, -1e20, -1e24, -1e30, -1e32, -1e35, -1e37, -1e38, -2e38, LOWEST])
def test_large_finite_masks(gpu, value, dtype):
    logits, scores = inputs(gpu, 31, 7, 3, 5000, dtype)
    mask(logits, value)
    for k in (3, 40):
        check(logits, scores, k)
    finished = torch.zeros(7, 3, dtype=torch.bool, device=gpu)
    finished[:, 1] = True
    check(logits, scores, 6, finished=finished, eos_token=4000)


@BOTH
def test_masks_of_several_values(gpu, dtype):
    """Masked twice, by values far apart, beside -inf; beams that have nothing but masks of two values."""
    logits, scores = inputs(gpu, 32, 4, 3, 5000, dtype)
    logits[0, :, 1000:3000], logits[0, :, 2000:] = -1e10, -1e30
    logits[1], logits[1, :, 100:200] = -1e30, -1e10
    logits[2], logits[2, :, 100:200] = -float("inf"), -1e30
    logits[3, 0], logits[3, 0, 4990:] = torch.finfo(dtype).min, -1e20
    for k in (3, 64):
        check(logits, scores, k)


@BOTH
@pytest.mark.parametrize("value", [-1e10, -1e30, LOWEST])
def test_masks_in_long_chunks(gpu, value, dtype):
    """Chunks of eight and sixteen batches."""
    logits, scores = inputs(gpu, 33, 24, 8, 131072, dtype)
    value = torch.finfo(dtype).min if value == LOWEST else value
    logits[:, :, 128000:] = value
    logits[:, 0, 64:72], logits[:, 1, 8192 : 2 * 8192], logits[:, 2], logits[:, 3, 4096 : 4096 + 3584] = value, value, value, value
    check(logits, scores, 8)
