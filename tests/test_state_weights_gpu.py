"""Merges of states that hold undefined values where they have no weight.  Bounds: those of ``test_block_states_gpu``."""
import math

import pytest
import torch

from oracle import long_video as L
from tests.test_block_states_gpu import DEV, FORMATS, _check_merge, _state

pytestmark = pytest.mark.gpu


def _any_bytes(g, B, S, H, D, fmt):
    """An 8-bit state as it may lie in memory that nobody has written: every element and scale byte, among them e4m3's own undefined 0x7f and 0xff."""
    from ditango_amd.core.cache import STATE_FORMATS, BlockState
    elements = torch.randint(0, 256, (B, S, H, D), generator=g, dtype=torch.uint8)
    elements[..., 5], elements[..., D - 7] = 0x7f, 0xff
    scales = torch.arange(B * S * H * D // 32, dtype=torch.int64).remainder(256).to(torch.uint8).view(B, S, H, D // 32)
    return BlockState(elements.to(DEV).view(STATE_FORMATS[fmt]), scales.to(DEV), torch.full((B, H, S), -math.inf, device=DEV))


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("n", [2, 7])
@pytest.mark.parametrize("B, S, H", [(1, 5, 3), (2, 37, 8), (1, 300, 24)])       # rows one by one, and in tiles
def test_memory_that_nobody_wrote_adds_nothing_without_weight(hip, B, S, H, n, D, fmt):
    from ditango_amd.core.cache import merge_any, quantized
    g = torch.Generator().manual_seed(S + n)
    unwritten = _any_bytes(g, B, S, H, D, fmt)
    given = [_state(g, B, S, H, D, t, 0.3) for t in [torch.bfloat16, torch.float32, torch.float16, torch.bfloat16, torch.float32, torch.bfloat16][:n - 1]]
    out, lse = merge_any([unwritten] + given, dst_dtype=torch.float32)
    _check_merge(out, lse, [(o.cpu(), l.cpu()) for o, l in given], torch.float32)
    # rows that are there in the 8-bit state and rows that are not
    o, l = _state(g, B, S, H, D, torch.float32, 0.3)
    some = quantized(o, l, fmt)
    written = torch.rand(B, S, H, generator=g).to(DEV) < 0.5
    written[0, 0, 0], written[0, 1, 0] = True, False
    blank = ~written
    some.elements.view(torch.uint8)[blank] = unwritten.elements.view(torch.uint8)[blank]
    some.scales[blank] = unwritten.scales[blank]
    some.lse.copy_(torch.where(written, l.transpose(1, 2), torch.full((), -math.inf, device=DEV)).transpose(1, 2))
    values = L.value(torch.where(blank[..., None], torch.zeros((), device=DEV), some.elements.float()).cpu(),
                     torch.where(blank[..., None], torch.zeros((), dtype=torch.int32, device=DEV), some.scales.int() - 127).cpu())
    out, lse = merge_any(given + [some], dst_dtype=torch.bfloat16)
    _check_merge(out, lse, [(o.cpu(), l.cpu()) for o, l in given] + [(values, some.lse.cpu())], torch.bfloat16)
