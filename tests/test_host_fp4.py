"""Arguments that the host layer of the operators over a cache in 4 bits and of the beam selection refuses, without a GPU."""

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

from tpa import _dispatch, tpa


def on_gpu(*shape, dtype=torch.bfloat16):
    return torch.empty(shape, device="cuda", dtype=dtype)


@pytest.mark.parametrize("n", [-1, -5, -(2**40)])
def test_sizes_below_zero_are_not_the_default(n):
    with FakeTensorMode():
        with pytest.raises(ValueError):
            tpa.tpa_beam_select(on_gpu(2, 3, 9), on_gpu(2, 3), num_out=n)
        cache = on_gpu(2, 4, 2, 40, dtype=torch.uint8)
        with pytest.raises(_dispatch.TpaError):
            tpa.tpa_decode_fp4(on_gpu(2, 1, 2, 8), on_gpu(2, 1, 2, 64), cache, cache, v_head_dim=n)
