"""``prepare_qk_axes`` against its definition in float64.

Bound.  fp32 throughout, one rounding to 16 bits (half a step, u).  Statistics are sums of 64 or 128 terms in chains of at most 12 roundings,
a root and a division; an element then sees 4 more, an angle's sine and cosine are right to 2^-22: together below 32 roundings of 2^-24
of the larger of the pair's two elements, and of the row's largest magnitude times the row's scale where a mean is taken off.
  |y - o| <= u |o| + 32 2^-24 (|v_a| + |v_b| + max |x| rs |w|)
"""
import pytest
import torch

from oracle import long_video as L

pytestmark = pytest.mark.gpu

DEV = "cuda:0"

AXES = [
    dict(dims=(16, 24, 24), base=10000.0),
    dict(dims=(16, 56, 56), base=256.0),
    dict(dims=(64, 32, 32), base=10000.0, pairing="rotate_half"),
    dict(dims=(32, 16, 16), base=(100.0, 5000.0, 1.5), pairing="rotate_half"),
    dict(dims=(32, 48, 48), base=1000000.0, pairing="rotate_half", halves="head"),
    dict(dims=(2, 62), base=77.0),
    dict(dims=(128,), base=10000.0, pairing="rotate_half"),
]


def _reference(x, positions, axes, norm, weight, bias):
    base = axes["base"] if isinstance(axes["base"], tuple) else (axes["base"],) * len(axes["dims"])
    n = L.norm(x.cpu(), norm, None if weight is None else weight.cpu(), None if bias is None else bias.cpu())
    return n, L.rotate(n, positions.cpu(), axes["dims"], base, axes.get("pairing", "interleaved"), axes.get("halves", "axis"))


def _check(y, x, positions, axes, norm=None, weight=None, bias=None, scale=1.0):
    n, o = _reference(x, positions, axes, norm, weight, bias)
    partner = torch.empty_like(n)
    for a, b, _, _ in L.pairs(axes["dims"], axes.get("pairing", "interleaved"), axes.get("halves", "axis")):
        partner[..., a], partner[..., b] = n[..., b], n[..., a]
    spread = 0.0
    if norm is not None:
        xd = x.cpu().double()
        c = xd - xd.mean(-1, keepdim=True) if norm == "layer_norm" else xd
        spread = xd.abs().amax(-1, keepdim=True) / (c.pow(2).mean(-1, keepdim=True) + 1e-6).sqrt() * (1 if weight is None else float(weight.abs().max()))
        if bias is not None:
            spread = spread + float(bias.abs().max())
    u = torch.finfo(y.dtype).eps / 2
    tol = u * (o * scale).abs() + 32 * 2.0 ** -24 * scale * (n.abs() + partner.abs() + spread)
    if y.dtype is torch.float16:
        tol = tol + 2.0 ** -25           # half a step of its smallest numbers
    err = (y.cpu().double() - o * scale).abs()
    assert bool((err <= tol).all()), float((err - tol).max())


def _positions(g, shape, far):
    return torch.randint(-far, far + 1, shape, generator=g).to(torch.int32).to(DEV)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("norm", [None, "rms", "layer_norm"])
@pytest.mark.parametrize("axes", range(len(AXES)))
def test_matches_the_definition(hip, axes, norm, dtype):
    from ditango_amd.producer import RotaryAxes, prepare_qk_axes
    spec = AXES[axes]
    D = sum(spec["dims"])
    g = torch.Generator().manual_seed(axes)
    for B, S, H, Hk, far in ((1, 1, 1, 1, 3), (2, 37, 5, 5, 60), (1, 19, 12, 4, 100000), (3, 7, 9, 1, 2 ** 31 - 1)):
        q = (torch.randn(B, S, H, D, generator=g) * 2 + 0.3).to(dtype).to(DEV)
        k = (torch.randn(B, S, Hk, D, generator=g) * 2).to(dtype).to(DEV)
        w = [(torch.rand(D, generator=g) + 0.5).to(dtype).to(DEV) for _ in range(2)] if norm else [None, None]
        b = [(torch.randn(D, generator=g) * 0.1).to(DEV) for _ in range(2)] if norm == "layer_norm" else [None, None]
        pos = _positions(g, (B, S, len(spec["dims"])) if S % 2 else (S, len(spec["dims"])), far)
        if far > 2 ** 24:     # a float64 angle of such a position is off by 2^31 2^-53 turns of 2 pi at most: 2^-19, above the bound
            pos = pos.clamp(-2 ** 24, 2 ** 24)
        qy, ky = prepare_qk_axes(q, k, pos, RotaryAxes(**spec), norm=norm, q_weight=w[0], q_bias=b[0], k_weight=w[1], k_bias=b[1])
        assert qy.is_contiguous() and ky.is_contiguous() and qy.dtype == ky.dtype == dtype
        _check(qy, q, pos, spec, norm, w[0], b[0])
        _check(ky, k, pos, spec, norm, w[1], b[1])


def test_every_position_turns_exactly(hip):
    """Positions to both ends of 32 bits, against whole-number arithmetic: the angle of n is n times the angle of one, modulo a turn."""
    from decimal import Decimal, localcontext
    import math
    from ditango_amd.producer import RotaryAxes, prepare_qk_axes
    axes = RotaryAxes(dims=(64,), base=10000.0)
    n = torch.tensor([[-2 ** 31], [2 ** 31 - 1], [-1], [1], [0], [123456789], [-987654321]], dtype=torch.int32, device=DEV)
    q = torch.zeros(1, n.numel(), 1, 64, device=DEV).half()
    q[..., 0::2] = 1.0
    y, none = prepare_qk_axes(q, None, n, axes)
    assert none is None
    pi = Decimal("3.14159265358979323846264338327950288419716939937510582097494459")
    with localcontext() as ctx:
        ctx.prec = 60
        for i, p in enumerate(n[:, 0].tolist()):
            for j in range(32):
                turn = (Decimal(p) * Decimal(10000) ** (Decimal(-2 * j) / 64) / (2 * pi)) % 1
                a = 2 * math.pi * float(turn)
                # sine and cosine to 2^-22, rounded to fp16
                assert abs(float(y[0, i, 0, 2 * j]) - math.cos(a)) <= 2.0 ** -11 * abs(math.cos(a)) + 2.0 ** -22
                assert abs(float(y[0, i, 0, 2 * j + 1]) - math.sin(a)) <= 2.0 ** -11 * abs(math.sin(a)) + 2.0 ** -22


def test_text_at_the_origin_is_left_alone_and_the_grid_is_the_clips(hip):
    from ditango_amd.producer import RotaryAxes, grid_positions, prepare_qk_axes
    pos = grid_positions(2, 3, 4, text=5, first_frame=7, device=DEV)
    assert pos.shape == (29, 3) and pos[:5].eq(0).all() and pos[5].tolist() == [7, 0, 0] and pos[-1].tolist() == [8, 2, 3]
    q = torch.randn(1, 29, 2, 64, device=DEV).bfloat16()
    y, _ = prepare_qk_axes(q, None, pos, RotaryAxes(dims=(16, 24, 24)))
    assert torch.equal(y[:, :5], q[:, :5]) and not torch.equal(y[:, 5:], q[:, 5:])


def test_reads_slices_of_a_projection_and_writes_in_place(hip):
    from ditango_amd.producer import RotaryAxes, prepare_qk_axes
    g = torch.Generator().manual_seed(3)
    spec = AXES[2]
    qkv = torch.randn(2, 50, 8 + 2 * 2, 128, generator=g).bfloat16().to(DEV)
    q, k = qkv[:, :, :8], qkv[:, :, 8:10]
    pos = _positions(g, (50, 3), 500)
    want = prepare_qk_axes(q, k, pos, RotaryAxes(**spec), norm="rms")
    _check(want[0], q, pos, spec, "rms")
    qc, kc = q.contiguous(), k.contiguous()
    got = prepare_qk_axes(qc, kc, pos, RotaryAxes(**spec), norm="rms", out=(qc, kc))
    assert got[0].data_ptr() == qc.data_ptr() and torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_agrees_with_the_tables(hip):
    """The same rotation through ``prepare_qk`` and fp32 tables: two roundings of tables that differ by 2^-23 at most."""
    from ditango_amd.producer import RotaryAxes, grid_positions, prepare_qk, prepare_qk_axes
    pos = grid_positions(3, 4, 5, device=DEV)
    dims = (16, 56, 56)
    ang = torch.cat([pos[:, i:i + 1].double() * 256.0 ** (-torch.arange(0, d, 2, device=DEV).double() / d) for i, d in enumerate(dims)], -1)
    cos, sin = (t.float().repeat_interleave(2, -1).contiguous() for t in (ang.cos(), ang.sin()))
    q = torch.randn(1, 60, 6, 128, device=DEV).bfloat16()
    w = torch.rand(128, device=DEV) + 0.5
    a = prepare_qk(q, norm="rms", weight=w, rope="interleaved", freqs_cis=(cos, sin), fold_softmax_scale=0.0)
    b, _ = prepare_qk_axes(q, None, pos, RotaryAxes(dims=dims, base=256.0), norm="rms", q_weight=w, fold_softmax_scale=0.0)
    d = (a.float() - b.float()).abs()
    assert bool((d <= 2.0 ** -7 * a.float().abs() + 1e-6).all()) and float((d > 0).float().mean()) < 0.01


def test_replayed_from_a_graph(hip):
    from ditango_amd.producer import RotaryAxes, prepare_qk_axes
    axes = RotaryAxes(dims=(16, 24, 24))
    q, k = torch.randn(1, 40, 6, 64, device=DEV).half(), torch.randn(1, 40, 2, 64, device=DEV).half()
    pos = torch.zeros(40, 3, dtype=torch.int32, device=DEV)
    prepare_qk_axes(q, k, pos, axes, norm="rms")
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = prepare_qk_axes(q, k, pos, axes, norm="rms")
    for step in range(4):
        pos.add_(step + 1)
        graph.replay()
        torch.cuda.synchronize()
        want = prepare_qk_axes(q, k, pos, axes, norm="rms")
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_no_tokens(hip):
    from ditango_amd.producer import RotaryAxes, prepare_qk_axes
    q = torch.empty(2, 0, 4, 64, dtype=torch.bfloat16, device=DEV)
    y, k = prepare_qk_axes(q, q[:, :, :2], torch.empty(0, 3, dtype=torch.int32, device=DEV), RotaryAxes(dims=(16, 24, 24)))
    assert y.shape == (2, 0, 4, 64) and k.shape == (2, 0, 2, 64)


def test_more_than_2_to_the_31_elements(hip):
    """The end of a sequence of 2.3 billion elements, against the same tokens on their own."""
    from ditango_amd.producer import RotaryAxes, grid_positions, prepare_qk_axes
    S, H, D, n = 140_001, 128, 128, 37
    q = torch.empty(1, S, H, D, dtype=torch.bfloat16, device=DEV).normal_(generator=torch.Generator(device=DEV).manual_seed(4))
    axes, pos = RotaryAxes(dims=(16, 56, 56), base=256.0), grid_positions(1, 140_001, 1, device=DEV)
    k = q[:, :, :2]
    got = prepare_qk_axes(q, k, pos, axes, norm="rms")
    for at in (slice(0, n), slice(S - n, S)):
        want = prepare_qk_axes(q[:, at], k[:, at], pos[at].contiguous(), axes, norm="rms")
        assert torch.equal(got[0][:, at], want[0]) and torch.equal(got[1][:, at], want[1])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("norm", [None, "rms", "layer_norm"])
@pytest.mark.parametrize("axes", range(len(AXES)))
def test_a_long_sequence_is_its_pieces(hip, axes, norm, dtype):
    """Long launches give a lane group eight heads, short ones four: the same bits, q with and without k, also where heads do not fill a group."""
    from ditango_amd.producer import RotaryAxes, prepare_qk_axes
    g = torch.Generator().manual_seed(40 + axes)
    axes = RotaryAxes(**AXES[axes])
    D, n = sum(axes.dims), 50
    w, b = (torch.randn(D, generator=g).to(dtype).to(DEV) for _ in range(2))
    p = dict(norm=norm, q_weight=w, k_weight=b, q_bias=b if norm == "layer_norm" else None, fold_softmax_scale=0.3)
    for B, S, H, Hk in ((2, 2401, 24, 8), (1, 5003, 22, 5), (1, 3001, 45, None)):
        q = torch.randn(B, S, H, D, generator=g).to(dtype).to(DEV)
        k = None if Hk is None else torch.randn(B, S, Hk, D, generator=g).to(dtype).to(DEV)
        pos = _positions(g, (B, S, len(axes.dims)), 3000)
        whole = prepare_qk_axes(q, k, pos, axes, **p)
        for at in (slice(0, n), slice(S // 2, S // 2 + n), slice(S - n, S)):
            piece = prepare_qk_axes(q[:, at], None if k is None else k[:, at], pos[:, at], axes, **p)
            assert torch.equal(whole[0][:, at], piece[0]) and (k is None or torch.equal(whole[1][:, at], piece[1]))
