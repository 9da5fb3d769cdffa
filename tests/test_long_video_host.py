"""What the operators of long videos do on the host.  No GPU needed."""
import copy
import pickle

import pytest
import torch


def test_a_pair_has_no_place_for_scales():
    """``merge_any`` and ``load_block`` give ``(out, lse)``: of 8 bits that would be elements without their scales."""
    from ditango_amd.core.cache import STATE_FORMATS, BlockState, merge_any, proCache
    x, lse = torch.zeros(1, 4, 2, 64, dtype=torch.bfloat16), torch.zeros(1, 2, 4)
    for fmt, dtype in STATE_FORMATS.items():
        with pytest.raises(ValueError, match="scales"):
            merge_any([(x, lse), (x, lse)], dst_dtype=dtype)
        cache = proCache(8, 0, state_format=fmt)
        state = BlockState.empty(x.shape, fmt, "cpu")
        cache.out_block_cache[0], cache.lse_block_cache[0] = state, state.lse
        with pytest.raises(ValueError, match="scales"):
            cache.load_block(0, dtype)


@pytest.mark.parametrize("again", [copy.copy, copy.deepcopy, lambda x: pickle.loads(pickle.dumps(x))], ids=["copy", "deepcopy", "pickle"])
def test_axes_that_have_been_used_are_copied(again):
    """A model that holds its axes is deep-copied, saved and sent to other processes after its first call as before it."""
    from ditango_amd.producer import RotaryAxes
    axes = RotaryAxes(dims=(64, 32, 32), base=(10000.0, 500.0, 500.0), pairing="rotate_half")
    turns, table = axes.turns, axes.table
    other = again(axes)
    assert other == axes and hash(other) == hash(axes) and other.turns == turns and other.sections == axes.sections
    assert type(other.table) is type(table)
    module = torch.nn.Module()
    module.axes = axes
    assert again(module).axes == axes and axes.table is table
