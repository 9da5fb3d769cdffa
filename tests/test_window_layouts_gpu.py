"""``window_attention`` over tensors whose rows lie apart: any token and head stride that is a multiple of 8 elements, a base that starts 8
elements behind another, K, V and q each in a layout of its own.  What lies between the rows is NaN, so that one 16-byte chunk read
from the wrong place shows.  Bounds: those of ``test_window_gpu``."""
import math

import pytest
import torch

from tests.test_window_gpu import DEV, _check, _run

pytestmark = pytest.mark.gpu


def _apart(t, token, head, offset):
    """``t`` ``[B,S,H,D]`` in storage with these strides (elements) behind ``offset`` elements, NaN all round it."""
    B, S, H, D = t.shape
    one = max((S - 1) * token, 0) + (H - 1) * head + D + 24
    room = torch.full((offset + B * one + 64,), math.nan, dtype=t.dtype, device=t.device)
    view = room[offset:].as_strided((B, S, H, D), (one, token, head, 1))
    view.copy_(t)
    return view


def _layouts(H, S, D):
    """(token stride, head stride, offset): padded rows, one more head in between, heads in front of tokens, a base that is off a line."""
    return [(H * (D + 8), D + 8, 8), (H * (D + 32), D + 32, 0), (H * D + 8, D, 24), (H * D + 72, D, 40), ((H + 1) * (D + 40), D + 40, 16),
            (D + 8, S * (D + 8) + 8, 8), (D + 64, S * (D + 64) + 16, 32), (1000, 1000 * S + 8, 56)]


# few rows with 8 and with 4 wavefronts, whole and in parts; workgroups of 256 rows, whole and (the last, heads of 128) with a last round in parts:
# tests/test_window_launches.py
SIZES = [(1, 8, 517, 8, 2, dict(left=63, right=0, sinks=1)), (2, 1, 4001, 4, 1, dict(left=1500, right=0, sinks=64)),
         (1, 300, 640, 6, 3, dict(left=100, right=30, sinks=5, q_begin=200)), (1, 65, 30, 3, 1, dict(left=20, right=None)),
         (2, 700, 900, 32, 16, dict(left=1, right=0, frame=128, sinks=70, q_begin=190)), (1, 1200, 1200, 36, 36, dict(left=None, right=0)),
         (1, 600, 1500, 40, 20, dict(left=None, right=0))]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("size", range(len(SIZES)))
@pytest.mark.parametrize("layout", range(8))
def test_rows_that_lie_apart(hip, layout, size, D, dtype):
    B, Sq, Sk, H, Hk, w = SIZES[size]
    g = torch.Generator(device=DEV).manual_seed(8 * size + layout)
    mk = lambda S, heads, sigma: (torch.randn(B, S, heads, D, generator=g, device=DEV) * sigma).to(dtype)
    q, k, v = mk(Sq, H, 1.5), mk(Sk, Hk, 1.5), mk(Sk, Hk, 1.0)
    at = [_layouts(t.shape[2], t.shape[1], D)[(layout + i) % 8] for t, i in ((q, 5), (k, 0), (v, 3))]
    apart = [_apart(t, *a) for t, a in zip((q, k, v), at)]
    got = _run(*apart, **w)
    _check(*got, q, k, v, **w)
    want = _run(q, k, v, **w)                 # and, the arithmetic being the same, bit for bit what dense rows give
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("pad", [8, 24, 32, 56, 64, 72, 120, 136, 872])
def test_one_head_beside_other_columns(hip, pad, D):
    """``buf[..., :D]`` of a cache of one head with some columns more, and the columns' last D: every remainder that a token stride can leave."""
    g = torch.Generator(device=DEV).manual_seed(pad)
    buf = torch.full((2, 2, 410, 1, D + pad), math.nan, dtype=torch.bfloat16, device=DEV)
    k, v = buf[0, ..., :D], buf[1, ..., pad:]
    for t in (k, v):
        t.copy_(torch.randn(t.shape, generator=g, device=DEV))
    for Sq, H in ((1, 4), (400, 48)):
        q = torch.randn(2, Sq, H, D, generator=g, device=DEV).bfloat16()
        w = dict(left=150, right=0, sinks=7)
        _check(*_run(q, k, v, **w), q, k.contiguous(), v.contiguous(), **w)
