"""``window_attention`` against its definition in float64.

Bound.  A score is a sum of D products in fp32: off by at most (D + 8) 2^-24 sum |q_i k_i| scale, and a probability by that much relative
(the exponential itself: 2^-20).  P is rounded to the tensors' 16 bits (half a step, u), the result once more, the sums are fp32:
  |out - o| <= u |o| + (u + e) sum_j w_j |v_j|,   |lse - l| <= e + 2^-21 |l|,   e = (D + 8) 2^-24 max sum |q k| scale + 2^-18.
fp16 probabilities below 2^-14 lose no more than 2^-25 each, next to a sum of at least 1: + Sk 2^-25 max |v|.
"""
import math

import pytest
import torch

from oracle import long_video as L

pytestmark = pytest.mark.gpu

DEV = "cuda:0"


def _tensors(B, Sq, Sk, H, Hk, D, dtype, seed=0, sigma=1.5):
    g = torch.Generator(device=DEV).manual_seed(seed)
    mk = lambda *s: torch.randn(*s, generator=g, device=DEV)
    return (mk(B, Sq, H, D) * sigma).to(dtype), (mk(B, Sk, Hk, D) * sigma).to(dtype), mk(B, Sk, Hk, D).to(dtype)


def _check(out, lse, q, k, v, **w):
    o, l, weight, top = L.window_attention(q, k, v, **w)
    u = torch.finfo(q.dtype).eps / 2
    e = (q.shape[-1] + 8) * 2.0 ** -24 * top + 2.0 ** -18
    tol = u * o.abs() + (u + e) * weight
    if q.dtype is torch.float16 and k.shape[1]:
        tol = tol + k.shape[1] * 2.0 ** -25 * torch.nan_to_num(v.double(), posinf=0.0, neginf=0.0).abs().max()
    same = (out.double() == o) | (out.isnan() & o.isnan())
    assert bool((same | ((out.double() - o).abs() <= tol + 1e-30)).all()), float(((out.double() - o).abs() - tol).nan_to_num().max())
    empty = l == -math.inf
    assert bool((lse[empty] == -math.inf).all()) and bool((out.transpose(1, 2)[empty] == 0).all())
    d = (lse.double() - l)[~empty]
    assert bool((d.abs() <= e + 2.0 ** -21 * l[~empty].abs()).all()), float(d.abs().max())


def _run(q, k, v, **w):
    from ditango_amd.window import window_attention
    out, lse = window_attention(q, k, v, **w)
    torch.cuda.synchronize()
    assert out.shape == q.shape and out.dtype == q.dtype and lse.shape == (q.shape[0], q.shape[2], q.shape[1])
    return out, lse


CASES = [
    # B, Sq, Sk, H, Hk, window
    (1, 1, 1, 1, 1, dict(right=0)),
    (1, 1, 700, 3, 3, dict(left=99, right=0, sinks=4)),
    (2, 1, 4001, 4, 1, dict(left=1500, right=0, sinks=64)),
    (1, 8, 517, 8, 2, dict(left=63, right=0, sinks=1)),
    (1, 130, 130, 2, 2, dict(left=0, right=0)),
    (1, 257, 257, 2, 1, dict(left=31, right=32)),
    (2, 100, 333, 3, 3, dict(left=17, right=0, sinks=65, q_begin=7)),
    (1, 150, 150, 2, 2, dict(left=1, right=0, frame=37, sinks=11, q_begin=0)),
    (1, 60, 400, 6, 2, dict(left=2, right=1, frame=50, sinks=13, q_begin=300)),
    (1, 40, 100, 1, 1, dict(left=5, right=0, q_begin=90)),            # the last rows stand behind every key
    (1, 40, 100, 1, 1, dict(left=5, right=0, q_begin=200)),           # all of them
    (1, 40, 100, 1, 1, dict(left=5, right=0, sinks=3, q_begin=2000)),  # ... but for the sinks
    (1, 70, 33, 2, 2, dict(left=4, right=0)),                         # the first rows stand before every key
    (1, 65, 300, 2, 2, dict()),
    (1, 65, 300, 2, 2, dict(left=None, right=0)),
    (1, 65, 300, 2, 2, dict(left=10, right=None, sinks=300)),
    (1, 64, 64, 1, 1, dict(left=2, right=0, frame=1 << 29, sinks=0)),
    (1, 33, 97, 1, 1, dict(left=(1 << 31) - 1, right=(1 << 31) - 1, frame=1 << 29)),
    (2, 1030, 1030, 32, 32, dict(left=99, right=20, sinks=6)),        # enough rows for workgroups of 256
    (2, 700, 900, 32, 16, dict(left=1, right=0, frame=128, sinks=70, q_begin=190)),
    (3, 600, 777, 40, 40, dict(left=None, right=0, sinks=0)),
    (1, 1500, 1600, 64, 8, dict(left=2, right=2, frame=100, sinks=100, q_begin=100)),
    (1, 2100, 2100, 66, 66, dict(left=None, right=0)),                # ... with a last round that is cut along the keys
    (1, 2100, 2300, 70, 70, dict(left=9, right=3, frame=100, sinks=150, q_begin=200)),
]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("case", range(len(CASES)))
def test_matches_the_definition(hip, case, D, dtype):
    B, Sq, Sk, H, Hk, w = CASES[case]
    q, k, v = _tensors(B, Sq, Sk, H, Hk, D, dtype, seed=case)
    _check(*_run(q, k, v, **w), q, k, v, **w)


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("Sq, H", [(1, 4), (5, 24), (400, 64)])
def test_lengths_on_the_gpu(hip, D, Sq, H):
    """Samples of unequal length; behind the length stands what must not count."""
    lens = torch.tensor([0, 1, 63, 64, 65, 400, 777, 9999, -5], dtype=torch.int32, device=DEV)
    B, Sk = lens.numel(), 777
    q, k, v = _tensors(B, Sq, Sk, H, H // 4, D, torch.bfloat16, seed=Sq)
    for b, n in enumerate(lens.clamp(0, Sk).tolist()):
        k[b, n:] = float("nan")
        v[b, n:] = float("inf")
    for w in (dict(left=200, right=0, sinks=3), dict(left=None, right=None), dict(left=30, right=0, q_begin=10)):
        _check(*_run(q, k, v, kv_lens=lens, **w), q, k, v, kv_lens=lens, **w)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("Sq, H, Hk, left", [(48, 2, 1, 6), (700, 64, 1, 6), (2100, 66, 66, 6), (2100, 66, 66, 1500)])
def test_masked_values_add_nothing(hip, Sq, H, Hk, left, dtype):
    """Infinities and NaN in values and keys that some rows see and others do not."""
    q, k, v = _tensors(1, Sq, Sq, H, Hk, 64, dtype, seed=1)
    v[0, 20, 0, 5] = float("inf")
    v[0, 33, 0, 7] = float("nan")
    v[0, 2, 0, 9] = float("-inf")
    k[0, 41] = float("nan")
    w = dict(left=left, right=0, sinks=1)
    out, lse = _run(q, k, v, **w)
    seen = L.visible(Sq, Sq, Sq, left, 0, 1, 1, None)
    hurt = seen[:, 41]
    assert bool(out[0, hurt.to(DEV), 0].isnan().all()) and bool(lse[0, 0, hurt.to(DEV)].isnan().all())
    out, q, k, v = out[:, :, :2], q[:, :, :2], k[:, :, :1 if Hk == 1 else 2], v[:, :, :1 if Hk == 1 else 2]      # (the others have nothing special)
    keep = (~hurt).nonzero()[:, 0].to(DEV)
    o, l, weight, top = L.window_attention(q, k, v, **w)
    got, want = out[0, keep].double(), o[0, keep]
    assert torch.equal(got.isfinite(), want.isfinite())
    fine = want.isfinite()
    u = torch.finfo(dtype).eps / 2
    e = 72 * 2.0 ** -24 * top + 2.0 ** -18
    tol = u * want.abs() + (u + e) * weight[0, keep] + Sq * 2.0 ** -25 * 6
    assert bool(((got - want).abs() <= tol)[fine].all())


@pytest.mark.parametrize("D", [64, 128])
def test_strided_inputs(hip, D):
    """k and v as slices of one projection, q with heads in front of tokens, a batch that is broadcast."""
    g = torch.Generator(device=DEV).manual_seed(4)
    kv = torch.randn(1, 300, 3, 2, D, generator=g, device=DEV).bfloat16()
    k, v = kv[:, :, :, 0].expand(2, 300, 3, D), kv[:, :, :, 1].expand(2, 300, 3, D)
    q = torch.randn(2, 6, 100, D, generator=g, device=DEV).bfloat16().transpose(1, 2)
    w = dict(left=70, right=0, sinks=2)
    _check(*_run(q, k, v, **w), q, k, v, **w)


@pytest.mark.parametrize("Sq, H", [(3, 1), (20000, 4)])
def test_offsets_beyond_32_bits(hip, Sq, H):
    """A cache whose last keys lie 5 GB behind its first."""
    Sk, stride = 2500, 1 << 20
    room = torch.empty(2, Sk * stride, dtype=torch.bfloat16, device=DEV)
    k, v = (room[i].as_strided((1, Sk, 1, 64), (0, stride, 64, 1)) for i in range(2))
    q, k0, v0 = _tensors(1, Sq, Sk, H, 1, 64, torch.bfloat16, seed=5)
    k.copy_(k0)
    v.copy_(v0)
    w = dict(left=100, right=0, sinks=2, q_begin=Sk - 50 if Sq > 50 else None)
    out, lse = _run(q, k, v, **w)
    n = min(Sq, 50)
    rows = slice(0, n)
    _check(out[:, rows], lse[:, :, rows], q[:, rows], k0, v0, **{**w, "q_begin": Sk - n})


def test_large_scores_and_a_late_maximum(hip):
    """Scores whose maximum comes late and is far above the first tile's: the running reference has to move."""
    q, k, v = _tensors(1, 300, 900, 2, 2, 128, torch.bfloat16, seed=6, sigma=6.0)
    k = k * torch.linspace(0.05, 2.0, 900, device=DEV).view(1, -1, 1, 1).to(k.dtype)
    w = dict(left=None, right=0)
    _check(*_run(q, k, v, **w), q, k, v, **w)


def test_same_result_again_and_rows_outside_stay(hip):
    """Bit for bit the same at every call, destinations of the caller's, and nothing is written around them."""
    q, k, v = _tensors(1, 5, 5000, 4, 4, 128, torch.bfloat16, seed=7)
    room = torch.full((3, 5, 4, 128), 7.0, dtype=torch.bfloat16, device=DEV)
    room_l = torch.full((3, 4, 5), 7.0, device=DEV)
    first = _run(q, k, v, left=4000, right=0, sinks=10)
    again = _run(q, k, v, left=4000, right=0, sinks=10, out=room[1:2], lse=room_l[1:2])
    assert torch.equal(first[0], again[0]) and torch.equal(first[1], again[1])
    assert bool((room[0] == 7).all()) and bool((room[2] == 7).all()) and bool((room_l[::2] == 7).all())


def test_no_tokens(hip):
    q, k, v = _tensors(2, 3, 0, 4, 2, 64, torch.bfloat16)
    out, lse = _run(q, k, v, left=3, right=0)
    assert bool((out == 0).all()) and bool((lse == -math.inf).all())
    out, lse = _run(q[:, :0], k, v)
    assert out.shape == (2, 0, 4, 64) and lse.shape == (2, 4, 0)


@pytest.mark.parametrize("Sq, H", [(1, 4), (300, 128)])
def test_captured_launch_follows_the_lengths(hip, Sq, H):
    q, k, v = _tensors(2, Sq, 2000, H, 4, 64, torch.bfloat16, seed=8)
    lens = torch.tensor([900, 1400], dtype=torch.int32, device=DEV)
    from ditango_amd.window import window_attention
    w = dict(left=1000, right=0, sinks=5)
    window_attention(q, k, v, kv_lens=lens, **w)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out, lse = window_attention(q, k, v, kv_lens=lens, **w)
    for step in range(4):
        lens.add_(step * 37)
        graph.replay()
        torch.cuda.synchronize()
        eager = window_attention(q, k, v, kv_lens=lens, **w)
        assert torch.equal(out, eager[0]) and torch.equal(lse, eager[1])


def test_two_streams_at_once(hip):
    """Launches that are cut into parts on two streams: each has a workspace of its own."""
    from ditango_amd.window import window_attention
    sets = [_tensors(1, 2, 30000, 2, 2, 128, torch.bfloat16, seed=s) for s in (1, 2)]
    want = [window_attention(*t, left=None, right=0) for t in sets]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in sets]
    got = [[], []]
    for _ in range(10):
        for i, (s, t) in enumerate(zip(streams, sets)):
            with torch.cuda.stream(s):
                got[i].append(window_attention(*t, left=None, right=0))
    torch.cuda.synchronize()
    for i in range(2):
        for o, l in got[i]:
            assert torch.equal(o, want[i][0]) and torch.equal(l, want[i][1])


def test_windows_that_part_the_keys_merge_to_the_whole(hip):
    """States of two key ranges, merged, are the state of both (what the operator returns them for)."""
    from ditango_amd.core.cache import merge_any
    q, k, v = _tensors(1, 90, 600, 2, 2, 64, torch.bfloat16, seed=9)
    near = _run(q, k[:, 300:], v[:, 300:], left=50, right=0)
    far = _run(q, k[:, :300], v[:, :300])
    out, lse = merge_any([near, far], dst_dtype=torch.float32)
    o1, l1, w1, t1 = L.window_attention(q, k[:, 300:], v[:, 300:], left=50, right=0)
    o2, l2, w2, t2 = L.window_attention(q, k[:, :300], v[:, :300])
    o, l = L.merge([(o1, l1), (o2, l2)])
    assert float((lse.double() - l).abs().max()) < 1e-4
    # each state is off by u |o| + (u + e) w in bf16, u = 2^-8; their merge by the weighted sum, at most the larger of the two
    tol = torch.maximum(2.0 ** -8 * o1.abs() + (2.0 ** -8 + 1e-4) * w1, 2.0 ** -8 * o2.abs() + (2.0 ** -8 + 1e-4) * w2) + 1e-4
    assert bool(((out.double() - o).abs() <= tol).all())


def test_the_step_adapter_hands_it_out(hip):
    from ditango_amd.core import config, parallel_state
    from ditango_amd.executor.step.attentions import Attention
    config.init_config(None)
    parallel_state.init_local_groups(1, 0)
    try:
        layer = Attention(0)
        q, k, v = _tensors(1, 64, 256, 2, 2, 128, torch.bfloat16, seed=10)
        got = layer.attn_processor("window")(q, k, v, causal=True, left=1, frame=64, sinks=64)
        want, _ = _run(q, k, v, left=1, right=0, frame=64, sinks=64)
        assert torch.equal(got, want)
        with pytest.raises(ValueError, match="causal"):
            layer.attn_processor("window")(q, k, v, causal=True, right=1)
    finally:
        parallel_state.destroy_local_groups()


@pytest.mark.parametrize("captured", [False, True])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("Sq, Sk, H, Hk, left", [(1, 30000, 2, 2, None), (3, 40, 4, 2, 11), (70, 5000, 2, 2, 3000), (700, 900, 64, 1, 150), (2100, 2100, 66, 66, 1500)])
def test_undefined_scores_stay_undefined(hip, Sq, Sk, H, Hk, left, D, captured):
    """A query that holds a NaN, and the queries that see a key that does, become NaN, in the lse as well, however the keys are shared out; no other does."""
    from ditango_amd.window import window_attention
    q, k, v = _tensors(1, Sq, Sk, H, Hk, D, torch.bfloat16, seed=12)
    w = dict(left=left, right=0)
    query, key = (0, 0), (Sk - 1 - Sq // 2, Hk - 1)
    q2, k2 = q.clone(), k.clone()
    q2[0, query[0], query[1], D - 3] = math.nan
    k2[0, key[0], key[1], 7] = math.nan
    window_attention(q2, k2, v, **w)
    if captured:
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out, lse = window_attention(q2, k2, v, **w)
        graph.replay()
        torch.cuda.synchronize()
    else:
        out, lse = _run(q2, k2, v, **w)
    at = torch.arange(Sq, device=DEV) + Sk - Sq
    sees = (at >= key[0]) & (at - (Sk if left is None else left) <= key[0])
    nan = torch.zeros(1, H, Sq, dtype=torch.bool, device=DEV)
    nan[0, key[1] * (H // Hk):(key[1] + 1) * (H // Hk)] = sees
    nan[0, query[1], query[0]] = True
    assert torch.equal(lse.isnan(), nan) and torch.equal(out.isnan(), nan.transpose(1, 2)[..., None].expand_as(out))
    _check(torch.where(out.isnan(), L.window_attention(q, k, v, **w)[0].to(out.dtype), out), torch.where(nan, L.window_attention(q, k, v, **w)[1].float(), lse), q, k, v, **w)


@pytest.mark.parametrize("Sq, Sk, H, Hk, w", [(1, 3000, 4, 2, dict(left=1000, right=0, sinks=70)), (700, 900, 64, 1, dict(left=150, right=3, sinks=5)),
                                              (2100, 2100, 66, 66, dict(left=2, right=1, frame=300, sinks=100, q_begin=0)), (2100, 2100, 66, 66, dict(left=None, right=0))])
def test_undefined_values_where_rows_do_and_do_not_see_them(hip, Sq, Sk, H, Hk, w):
    """Heads of 128: values without a finite magnitude in tiles that are seen whole, in part and not at all, in every key head."""
    q, k, v = _tensors(1, Sq, Sk, H, Hk, 128, torch.bfloat16, seed=13, sigma=1.0)
    for i in range(Hk):
        v[0, (37 * i + 1) % Sk, i, i % 128] = float("nan")
        v[0, (911 * i + 500) % Sk, i, (i + 64) % 128] = float("inf")
        v[0, Sk - 1 - i % 3, i, (i + 9) % 128] = float("-inf")
    _check(*_run(q, k, v, **w), q, k, v, **w)


def test_keys_that_batches_and_heads_share_by_stride(hip):
    """Expanded tensors: strides of 0 along the batch, the heads and (one key) the tokens."""
    q, k, v = _tensors(3, 50, 200, 4, 1, 64, torch.bfloat16, seed=14)
    k, v = k[:1].expand(3, -1, 4, -1), v[:1].expand(3, -1, 4, -1)
    got = _run(q, k, v, left=70, right=0, sinks=3)
    want = _run(q, k.contiguous(), v.contiguous(), left=70, right=0, sinks=3)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    one = (k[:, :1].expand(-1, 90, -1, -1), v[:, :1].expand(-1, 90, -1, -1))
    got, want = _run(q, *one, left=20, right=5), _run(q, *(t.contiguous() for t in one), left=20, right=5)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_results_over_the_queries(hip):
    """``out`` may be q: a row is read before anything of it is written, also where several workgroups share it."""
    from ditango_amd.window import window_attention
    for Sq, Sk, H in ((1, 9000, 2), (40, 9000, 2), (2100, 2100, 66)):
        q, k, v = _tensors(1, Sq, Sk, H, H, 64, torch.bfloat16, seed=15)
        want = _run(q, k, v, left=None, right=0)
        out, lse = window_attention(q, k, v, left=None, right=0, out=q)
        torch.cuda.synchronize()
        assert out.data_ptr() == q.data_ptr() and torch.equal(q, want[0]) and torch.equal(lse, want[1])
