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


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("D, H", [(64, 8), (128, 8), (64, 3)])        # in tiles (heads of 128 from six states on), and row by row
@pytest.mark.parametrize("behind", [0.0, 40.0, 90.0, 120.0, 400.0])
def test_undefined_values_are_seen_in_any_order(hip, behind, D, H, fmt):
    """One state of many holds an infinity and a NaN and lies ``behind`` the others in its lse, beyond what fp32 has a weight for: wherever it comes among them,
    these elements are not finite and all others are what they are without it."""
    from ditango_amd.core.cache import BlockState, merge_any, quantized
    g = torch.Generator().manual_seed(int(behind) + D)
    B, S = 1, 18
    for kind in (fmt, "bf16", "f32"):
        for n in (1, 5, 9, 66):
            others = [_state(g, B, S, H, D, (torch.bfloat16, torch.float32)[i % 2], 0.3) for i in range(n)]
            others = [(o, l + 3.0 * i) for i, (o, l) in enumerate(others)]      # the largest lse comes late
            others = [quantized(o, l, fmt) if i % 3 == 2 else (o, l) for i, (o, l) in enumerate(others)]
            o, l = _state(g, B, S, H, D, torch.float32, 0.3)
            l = torch.stack([s.lse if isinstance(s, BlockState) else s[1] for s in others]).amax(0) - behind
            o[0, 3, 1, 7], o[0, 11, 2, D - 1] = math.inf, math.nan
            odd = quantized(o, l, fmt) if kind in FORMATS else (o.to(dict(bf16=torch.bfloat16, f32=torch.float32)[kind]), l)
            bad = ~o.isfinite()
            if kind in FORMATS:                                # the whole block reads as NaN
                bad = bad.unflatten(-1, (-1, 32)).any(-1, keepdim=True).expand(-1, -1, -1, -1, 32).flatten(-2)
            clean = torch.where(bad, torch.zeros_like(o), o)
            clean = quantized(clean, l, fmt) if kind in FORMATS else (clean.to(odd[0].dtype), l)
            for at in sorted({0, n // 2, n}):
                put = lambda s: others[:at] + [s] + others[at:]
                got, lse = merge_any(put(odd), dst_dtype=torch.float32)
                want, want_lse = merge_any(put(clean), dst_dtype=torch.float32)
                assert torch.equal(got.isfinite(), ~bad), (kind, n, at)
                assert torch.equal(got[~bad], want[~bad]) and torch.equal(lse, want_lse)
