"""8-bit attention states against their definition in float64: elements and scales are exact, whatever arithmetic makes them; a merge is off
by its fp32 sums (n + 8 roundings and an exponential, 2^-20, of sum_i w_i |out_i|) and one rounding of the result."""
import math

import pytest
import torch

from oracle import long_video as L

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
FORMATS = ["e4m3", "int8"]


def _state(g, B, S, H, D, dtype=torch.float32, sigma=1.0):
    out = torch.randn(B, S, H, D, generator=g) * torch.exp(sigma * torch.randn(B, S, H, 1, generator=g))
    return out.to(dtype).to(DEV), (torch.randn(B, H, S, generator=g) * 3).to(DEV)


def _exact(state, out):
    elements, exponents = L.quantize(out.cpu(), "int8" if state.elements.dtype is torch.int8 else "e4m3")
    assert torch.equal(state.elements.cpu().double(), elements)
    assert torch.equal(state.scales.cpu().double(), exponents + 127)


@pytest.mark.parametrize("bsh", [False, True])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("fmt", FORMATS)
def test_store_and_load(hip, fmt, D, dtype, bsh):
    from ditango_amd.core.cache import proCache
    g = torch.Generator().manual_seed(D)
    for B, S, H in ((1, 1, 1), (2, 37, 3), (1, 300, 5), (3, 5, 8)):
        out, lse = _state(g, B, S, H, D, dtype, 2.0)
        lse[0, 0, 0] = -math.inf
        cache = proCache(8, 0, state_format=fmt)
        cache.store_block(2, out, lse.transpose(1, 2).unsqueeze(-1).contiguous() if bsh else lse)
        state, l = cache.get_block(2)
        assert state.lse is l and torch.equal(l, lse) and state.shape == (B, S, H, D)
        _exact(state, out)
        for dst in (torch.float32, torch.bfloat16):
            o, l = cache.load_block(2, dst)
            assert torch.equal(l.squeeze(-1).transpose(1, 2), lse) and o.dtype == dst
            # 7 significant bits at most: exact in bf16 too
            assert torch.equal(o.cpu().double(), L.value(state.elements.cpu(), state.scales.cpu().int() - 127))


@pytest.mark.parametrize("D, S", [(128, 2741), (64, 5481)])
@pytest.mark.parametrize("fmt", FORMATS)
def test_a_large_state_is_its_pieces(hip, fmt, D, S):
    """More rows than a launch of the small form: the same bits as piece by piece, and back, in every type."""
    from ditango_amd.core.cache import BlockState, merge_any, quantized
    g = torch.Generator().manual_seed(S)
    for dtype in (torch.float32, torch.bfloat16):
        out, lse = _state(g, 1, S, 12, D, dtype)
        state = quantized(out, lse, fmt)
        assert torch.equal(state.lse, lse)
        for a in range(0, S, 700):
            piece = quantized(out[:, a:a + 700].contiguous(), lse[:, :, a:a + 700].contiguous(), fmt)
            assert torch.equal(piece.elements.view(torch.uint8), state.elements[:, a:a + 700].contiguous().view(torch.uint8))
            assert torch.equal(piece.scales, state.scales[:, a:a + 700])
        for dst in (torch.float32, torch.bfloat16):
            back, l = merge_any([state], dst_dtype=dst, dst_lse_bsh=True)
            assert torch.equal(l.squeeze(-1).transpose(1, 2), lse)
            want = state.elements.float().unflatten(-1, (-1, 32)) * torch.exp2(state.scales.float() - 127).unsqueeze(-1)
            assert torch.equal(back.float(), want.flatten(-2))


@pytest.mark.parametrize("fmt", FORMATS)
def test_rows_at_the_ends_of_the_range(hip, fmt):
    from ditango_amd.core.cache import BlockState, merge_any
    x = torch.randn(1, 12, 1, 64)
    x[0, 0] = 0.0
    x[0, 1] *= 1e-38
    x[0, 2] *= 1e-41                                  # below the normal numbers
    x[0, 3] = x[0, 3].clamp(-1, 1) * 3e38
    x[0, 4, 0, :32], x[0, 4, 0, 32:] = 448.0, 448.0000305       # at the border, and just above it
    x[0, 5, 0, :32], x[0, 5, 0, 32:] = 127.0, 127.0000076
    x[0, 6] = 2.0 ** -126
    x[0, 7] = torch.arange(64) - 31.5                 # ties
    x[0, 8, 0, 3], x[0, 8, 0, 40] = math.inf, 1.0
    x[0, 9, 0, 50] = math.nan
    x[0, 10] = -0.0
    x[0, 11] = 2.0 ** -149
    state = BlockState.empty(x.shape, fmt, DEV)
    lse = torch.zeros(1, 1, 12, device=DEV)
    merge_any([(x.to(DEV), lse)], dst=state)
    bad = ~x.unflatten(-1, (2, 32)).isfinite().all(-1)
    clean = torch.where(bad.repeat_interleave(32, -1), torch.zeros_like(x), x)
    elements, exponents = L.quantize(clean, fmt)
    assert torch.equal(state.elements.cpu().double(), elements)
    assert torch.equal(state.scales.cpu().double(), torch.where(bad, 255.0, exponents + 127))
    back, _ = merge_any([state], dst_dtype=torch.float32)
    assert torch.equal(back.cpu().isnan(), bad.repeat_interleave(32, -1))
    assert torch.equal(back.cpu().double()[~back.cpu().isnan()], L.value(elements, exponents)[~back.cpu().isnan()])


def _check_merge(out, lse, states, dtype):
    """states: float64 (out, lse)."""
    o, l = L.merge(states)
    weight, _ = L.merge([(s.abs(), x) for s, x in states])
    e = (len(states) + 8) * 2.0 ** -24 + 2.0 ** -20 * 4
    tol = (torch.finfo(dtype).eps / 2) * o.abs() + e * weight
    if dtype is torch.float16:
        tol = tol + 2.0 ** -25
    assert bool(((out.cpu().double() - o).abs() <= tol).all()), float(((out.cpu().double() - o).abs() - tol).max())
    none = l == -math.inf
    assert bool((lse.cpu()[none] == -math.inf).all())
    assert bool(((lse.cpu().double() - l)[~none].abs() <= 2.0 ** -20 + 2.0 ** -22 * l[~none].abs()).all())


@pytest.mark.parametrize("out", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("kinds", ["e4m3", "int8 int8", "e4m3 bf16", "int8 fp16 f32", "e4m3 int8 e4m3 int8 e4m3 bf16 bf16 bf16 bf16 bf16 f32 f32",
                                   " ".join(["int8"] * 70 + ["bf16"] * 69)])
def test_merge(hip, kinds, D, out):
    from ditango_amd.core.cache import BlockState, merge_any
    g = torch.Generator().manual_seed(len(kinds))
    types = {"bf16": torch.bfloat16, "fp16": torch.float16, "f32": torch.float32}
    for B, S, H in ((1, 1, 1), (2, 37, 3)):
        states, want = [], []
        for i, kind in enumerate(kinds.split()):
            o, l = _state(g, B, S, H, D, types.get(kind, torch.float32), 0.3)
            if i % 3 == 1:
                l[0, 0] = -math.inf
            if S > 1:
                l[:, :, 5] = -math.inf                # a row without a key in any state
            if kind in FORMATS:
                state = BlockState.empty((B, S, H, D), kind, DEV)
                merge_any([(o, l)], dst=state)
                states.append(state)
                want.append((L.value(state.elements.cpu(), state.scales.cpu().int() - 127), l.cpu()))
            else:
                states.append((o, l) if i % 2 else (o, l.transpose(1, 2).unsqueeze(-1).contiguous()))
                want.append((o.cpu(), l.cpu()))
        if len(states) == 1:
            continue      # a copy
        got, lse = merge_any(states, dst_dtype=out, dst_lse_bsh=True)
        assert got.dtype == out and lse.shape == (B, S, H, 1)
        _check_merge(got, lse.squeeze(-1).transpose(1, 2), want, out)


@pytest.mark.parametrize("fmt", FORMATS)
def test_a_state_without_weight_is_left_out_whatever_it_holds(hip, fmt):
    from ditango_amd.core.cache import BlockState, merge_any
    g = torch.Generator().manual_seed(1)
    bad, none = _state(g, 1, 4, 2, 64)
    bad[:] = math.nan
    none[:] = -math.inf
    state = BlockState.empty(bad.shape, fmt, DEV)
    merge_any([(bad, none)], dst=state)
    assert bool((state.scales == 255).all())
    o, l = _state(g, 1, 4, 2, 64, torch.bfloat16)
    out, lse = merge_any([state, (o, l), (bad, none)], dst_dtype=torch.bfloat16)
    assert torch.equal(out, o) and torch.equal(lse, l)
    # and with weight it is seen
    out, lse = merge_any([BlockState(state.elements, state.scales, torch.zeros_like(none)), (o, l)])
    assert bool(out.isnan().all()) and bool(lse.isfinite().all())


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("D", [64, 128])
def test_coarsening_in_place(hip, fmt, D):
    """``_merge_blocks``: neighbours merged into the first one's memory, quantised again."""
    from ditango_amd.core.cache import proCache
    g = torch.Generator().manual_seed(2)
    cache = proCache(8, 0, state_format=fmt)
    values = []
    for b in range(8):
        o, l = _state(g, 2, 33, 3, D, torch.bfloat16, 0.3)
        if b == 5:
            values.append(None)
            continue
        cache.store_block(b, o, l)
        s = cache.out_block_cache[b]
        values.append((L.value(s.elements.cpu(), s.scales.cpu().int() - 127), l.cpu()))
    where = [None if s is None else s.elements.data_ptr() for s in cache.out_block_cache]
    cache._merge_blocks(4)
    for b in range(4):
        s = cache.out_block_cache[b]
        members = [v for v in values[2 * b:2 * b + 2] if v is not None]
        assert s.elements.data_ptr() == where[2 * b]
        if len(members) == 1:
            assert torch.equal(L.value(s.elements.cpu(), s.scales.cpu().int() - 127), members[0][0])
            continue
        o, l = L.merge(members)
        assert bool(((s.lse.cpu().double() - l).abs() <= 2.0 ** -20 + 2.0 ** -22 * l.abs()).all())
        # half a step of the block's largest element (int8) or of the value (e4m3, above its smallest), and the fp32 merge
        got = L.value(s.elements.cpu(), s.scales.cpu().int() - 127)
        scale = torch.ldexp(torch.ones(1, dtype=torch.float64), s.scales.cpu().int() - 127).repeat_interleave(32, -1)
        half = scale / 2 if fmt == "int8" else torch.maximum(o.abs() * 2.0 ** -4, scale * 2.0 ** -10)
        assert bool(((got - o).abs() <= half * (1 + 2.0 ** -10) + 1e-5).all())


@pytest.mark.parametrize("fmt", FORMATS)
def test_replayed_from_a_graph(hip, fmt):
    from ditango_amd.core.cache import BlockState, merge_any
    g = torch.Generator().manual_seed(3)
    o, l = _state(g, 1, 50, 4, 64, torch.bfloat16)
    state = BlockState.empty(o.shape, fmt, DEV)

    def step():
        merge_any([(o, l)], dst=state)
        return merge_any([state, (o, l)], dst_dtype=torch.bfloat16)
    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for i in range(4):
        o.add_(0.5)
        l.mul_(1.1)
        graph.replay()
        torch.cuda.synchronize()
        kept = state.elements.clone()
        want = step()
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1]) and torch.equal(kept.view(torch.uint8), state.elements.view(torch.uint8))


def test_no_rows(hip):
    from ditango_amd.core.cache import BlockState, merge_any
    o, l = torch.empty(1, 0, 4, 64, device=DEV), torch.empty(1, 4, 0, device=DEV)
    state = BlockState.empty(o.shape, "int8", DEV)
    assert merge_any([(o, l)], dst=state) is state and merge_any([state])[0].shape == (1, 0, 4, 64)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("fmt", FORMATS)
def test_merged_into_one_of_the_states_and_with_itself(hip, fmt, dtype):
    """The destination is a 16- or 32-bit state among 8-bit ones; a state that appears twice counts twice."""
    from ditango_amd.core.cache import merge_any, quantized
    g = torch.Generator().manual_seed(21)
    for B, S, H, D in ((1, 3, 1, 64), (2, 411, 5, 128)):
        o, l = _state(g, B, S, H, D, dtype, 0.3)
        state = quantized(*_state(g, B, S, H, D, torch.float32, 0.3), fmt)
        want = merge_any([state, (o, l), state], dst_dtype=dtype)
        own = (L.value(state.elements.cpu(), state.scales.cpu().int() - 127), state.lse.cpu())
        _check_merge(want[0], want[1], [own, (o.cpu(), l.cpu()), own], dtype)
        got = merge_any([state, (o, l), state], dst=(o, l))
        assert got[0] is o and torch.equal(o, want[0]) and torch.equal(l, want[1])


@pytest.mark.parametrize("fmt", FORMATS)
def test_more_than_2_to_the_31_elements(hip, fmt):
    """A state of 2.3 billion elements, stored, merged and loaded, against pieces of its end on their own."""
    from ditango_amd.core.cache import BlockState, merge_any, quantized
    S, H, D, n = 140_001, 128, 128, 33
    out = torch.empty(1, S, H, D, dtype=torch.bfloat16, device=DEV).normal_(generator=torch.Generator(device=DEV).manual_seed(3))
    lse = torch.randn(1, H, S, device=DEV)
    state = quantized(out, lse, fmt)
    ends = [slice(0, n), slice(S - n, S)]
    for at in ends:
        o, l = out[:, at].contiguous(), lse[:, :, at].contiguous()
        piece = quantized(o, l, fmt)
        part = BlockState(state.elements[:, at], state.scales[:, at], state.lse[:, :, at])
        assert torch.equal(part.elements.view(torch.uint8), piece.elements.view(torch.uint8)) and torch.equal(part.scales, piece.scales)
        assert torch.equal(part.lse, piece.lse)
    both = merge_any([state, (out, lse)], dst_dtype=torch.bfloat16)
    back = merge_any([state], dst_dtype=torch.bfloat16)
    for at in ends:
        o, l = out[:, at].contiguous(), lse[:, :, at].contiguous()
        piece = quantized(o, l, fmt)
        for whole, want in ((both, merge_any([piece, (o, l)], dst_dtype=torch.bfloat16)), (back, merge_any([piece], dst_dtype=torch.bfloat16))):
            assert torch.equal(whole[0][:, at], want[0]) and torch.equal(whole[1][:, :, at], want[1])


@pytest.mark.parametrize("bsh", [False, True])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("kinds", ["e4m3 int8", "int8 bf16 f32 e4m3 int8 fp16", " ".join(["int8", "bf16", "e4m3"] * 13), " ".join(["e4m3"] * 64), " ".join(["f32"] * 7 + ["int8"] * 60)],
                         ids=["two", "six", "39", "64", "67"])
def test_merge_of_heads_in_tiles(hip, kinds, D, bsh):
    """Heads and queries in tiles, whose lse come together: queries that do not fill the last one, lse in both layouts, more states than a launch takes."""
    from ditango_amd.core.cache import BlockState, merge_any
    g = torch.Generator().manual_seed(len(kinds) + D)
    types = {"bf16": torch.bfloat16, "fp16": torch.float16, "f32": torch.float32}
    for B, S, H in ((2, 37, 8), (1, 18, 24), (3, 16, 16)):
        states, want = [], []
        for i, kind in enumerate(kinds.split()):
            o, l = _state(g, B, S, H, D, types.get(kind, torch.float32), 0.3)
            if i % 3 == 1:
                l[0, 0] = -math.inf
            l[:, :, 5] = -math.inf
            if kind in FORMATS:
                state = BlockState.empty((B, S, H, D), kind, DEV)
                merge_any([(o, l)], dst=state)
                states.append(state)
                want.append((L.value(state.elements.cpu(), state.scales.cpu().int() - 127), l.cpu()))
            else:
                states.append((o, l) if i % 2 else (o, l.transpose(1, 2).unsqueeze(-1).contiguous()))
                want.append((o.cpu(), l.cpu()))
        got, lse = merge_any(states, dst_dtype=torch.bfloat16, dst_lse_bsh=bsh)
        _check_merge(got, lse.squeeze(-1).transpose(1, 2) if bsh else lse, want, torch.bfloat16)
        if isinstance(states[0], BlockState):
            first = states[0]
            again, again_lse = merge_any(states, dst_dtype=torch.float32)
            merge_any(states, dst=first)
            assert torch.equal(first.lse, again_lse)
            _exact(first, again)
