"""Counters under capture: as many parts of an attention over pages as without, by the sizes alone.  No GPU needed."""
import pytest


@pytest.mark.parametrize("D", [64, 128])
def test_captured_launches_are_cut_like_eager_ones(D):
    from ditango_amd import _hip
    nbytes = int(_hip.load_library().dt_attn_workspace_bytes())
    few, many = 32 * (D + 2) * 4, 256 * (D + 2) * 4          # bytes of a part: sums, a maximum and a sum of weights a row
    most = nbytes // 2 // few
    assert most <= _hip.CAPTURED_COUNTERS // 2 <= _hip.KEPT_COUNTERS // 2
    for n in range(most + 1):                                # parts of few rows that a launch may have
        assert (nbytes - n * few) // many <= (_hip.CAPTURED_COUNTERS - n) // 8
