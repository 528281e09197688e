"""Sizes that a launch or 64 bits do not hold, which the operators over a cache in 4 bits and the beam selection refuse before any launch."""

from test_abi_fp4 import SHAPE, WORKSPACE, beams, decode


def test_decode_one_row_more_than_a_launch_takes():
    for columns in (dict(B=1 << 20, lq=2), dict(B=1 << 21, lq=1), dict(B=2, lq=1 << 20)):
        assert decode(**columns, kernel=1) == SHAPE and decode(True, **columns, kernel=1) == 0
    assert decode(B=2, lq=1 << 20) == SHAPE  # (too many columns for the matrix-core kernel)
    assert decode(True, B=1 << 21, lq=1) > 0 and decode(B=1 << 21, lq=1, workspace_bytes=8) == WORKSPACE


def test_decode_sizes_whose_product_passes_64_bits():
    """2^64 and 2^65: zero in 64 bits."""
    for columns in (dict(B=1 << 22, lq=1 << 21, H=1 << 21), dict(B=1 << 22, lq=1 << 21, H=1 << 22), dict(B=1 << 30, lq=1 << 30, H=1 << 4)):
        for kernel in (0, 1):
            assert decode(**columns, kernel=kernel) == SHAPE and decode(True, **columns, kernel=kernel) == 0


def test_beam_select_more_than_a_launch_takes():
    from tpa import _dispatch as d

    size = d.load_library().tpa_beam_select_workspace_bytes
    # a wave for each chunk of a beam, a workgroup for each request; fewer than 2^32 work-items
    for refused, taken in ((dict(B=1 << 24, beams=1, vocab=5), dict(B=(1 << 24) - 1, beams=1, vocab=5)), (dict(B=1 << 20, beams=64, vocab=64), dict(B=(1 << 20) - 1, beams=64, vocab=64)),
                           (dict(B=1 << 12, beams=1, vocab=1 << 29), dict(B=(1 << 12) - 1, beams=1, vocab=1 << 25))):
        assert beams(**refused, num_out=1, eos_token=0) == SHAPE and size(*refused.values(), 1, 0) == 0
        assert beams(**taken, num_out=1, eos_token=0, workspace_bytes=8) == WORKSPACE and size(*taken.values(), 1, 0) > 8
    # sizes whose products pass 64 bits
    for sizes in ((2**31 - 1, 64, 2**31 - 1), (2**31 - 1, 2, 1 << 30)):
        assert size(*sizes, 1, 0) == 0
