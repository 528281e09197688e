"""tpa_beam_select where different logits have the same value in 64 bits: equal values go to the lower index all the same.

Beside a logit of 1e30 all others are -1e30, beside a score of -5 logits of 1e-30 are none.  The logarithm of the sum is 0 in these cases, or what it is off by is lost in the
values, so the definition's values are equal where the operator's are.
"""

import pytest
import torch

from test_gpu_beam_masks import check
from test_gpu_beam_select import inputs

pytestmark = pytest.mark.gpu
BOTH = pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])


@BOTH
@pytest.mark.parametrize("value", [1e8, 1e10, 1e12, 1e20, 1e30, 3e38])
@pytest.mark.parametrize("k", [1, 2, 5, 64])
def test_a_token_that_is_forced(gpu, k, value, dtype):
    logits, scores = inputs(gpu, 41, 3, 2, 5000, dtype)
    logits[0, :, 37] = value
    logits[1, 1, 4990] = value
    logits[2, 0, 2000], logits[2, 1, 0] = value, value
    check(logits, scores, k)


@BOTH
@pytest.mark.parametrize("b,n,vocab,k", [(2, 3, 5000, 20), (1, 2, 70001, 64), (2, 64, 1500, 64), (1, 1, 3, 3), (40, 8, 60000, 8)])
def test_logits_that_no_value_shows(gpu, b, n, vocab, k, dtype):
    logits, scores = inputs(gpu, 42, b, n, vocab, dtype)
    logits *= 1e-30
    scores[0] = -5.0
    check(logits, scores, k)
    logits[:, :, : vocab - vocab // 3] = -50.0  # all of them far behind
    check(logits, scores, k)


@BOTH
def test_ties_with_finished_beams(gpu, dtype):
    """A finished beam whose score is the value that all but one of the others' tokens have."""
    logits, scores = inputs(gpu, 43, 3, 3, 5000, dtype)
    logits[:, :, 4000] = 1e30
    finished = torch.tensor([[True, False, False], [False, True, False], [False, False, True]], device=gpu)
    scores[finished] = -logits[0, 0, 4000].float()
    for k in (1, 3, 30):
        check(logits, scores, k, finished=finished, eos_token=7)
