"""``plan_pages``, ``append_pages`` and ``prepare_qkv_pages`` against their definitions: whole numbers and copied values exactly, rotated keys and
queries as ``prepare_qk_axes`` computes them, bit for bit (its own tests hold that to float64)."""
import random

import pytest
import torch

from oracle import pages as P

pytestmark = pytest.mark.gpu

DEV = "cuda:0"


def _i32(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


def _plan(tables, lens, new, n_tokens, n_pages, page, in_place=False):
    from ditango_amd.pages import plan_pages
    width = len(tables[0])
    t = _i32(tables) if width else torch.empty(len(tables), 0, dtype=torch.int32, device=DEV)
    before = _i32(lens)
    plan = plan_pages(t, before, _i32(new), n_tokens, n_pages=n_pages, page_size=page, in_place=in_place)
    torch.cuda.synchronize()
    assert (plan.lens.data_ptr() == before.data_ptr()) == in_place
    assert plan.slots.dtype is torch.int64 and plan.served.dtype is torch.bool
    return t.tolist(), plan.lens.tolist(), plan.cu_seqlens.tolist(), plan.slots.tolist(), plan.served.tolist()


def _case(rng, B, page, width, n_pages, most_new, wild=False):
    """Tables of distinct pages in any order and what may stand behind them; with `wild`, lengths and entries that nobody should hand over."""
    ids = list(range(n_pages))
    rng.shuffle(ids)
    tables, lens, new = [], [], []
    for _ in range(B):
        held = min(rng.randint(0, width), len(ids))
        row = [ids.pop() for _ in range(held)]
        tables.append(row + [rng.choice([-1, 0, rng.randint(0, 2 ** 31 - 1), max(n_pages - 1, 0)]) for _ in range(width - held)])
        lens.append(rng.randint(max(0, (held - 1) * page + 1), held * page) if held else 0)
        new.append(rng.choice([0, 1, rng.randint(0, most_new)]))
        if wild:
            lens[-1] = rng.choice([lens[-1], -5, -2 ** 31, 2 ** 31 - 1, width * page + 3])
            new[-1] = rng.choice([new[-1], -1, 2 ** 31 - 1, -2 ** 31])
    return tables, lens, new


@pytest.mark.parametrize("B, page, width, n_pages, most_new", [
    (1, 16, 1, 1, 16), (1, 16, 4, 0, 3), (3, 16, 8, 40, 50), (8, 64, 40, 200, 1), (17, 48, 20, 333, 300), (64, 16, 30, 1200, 100),
    (300, 32, 5, 1000, 30), (1, 16, 3000, 4000, 20000), (2, 256, 300, 700, 30000), (1025, 16, 3, 2500, 9), (2048, 16, 2, 4095, 40)])
def test_plan_matches_the_definition(hip, B, page, width, n_pages, most_new):
    rng = random.Random(B * 1000 + page)
    for turn in range(4):
        tables, lens, new = _case(rng, B, page, width, n_pages, most_new)
        total = sum(new)
        for n_tokens in (total, total + 7, total // 2):
            want = P.plan(tables, lens, new, n_tokens, n_pages, page)
            got = _plan(tables, lens, new, n_tokens, n_pages, page, in_place=turn == 1)
            assert list(got) == list(want)


@pytest.mark.parametrize("B", [1, 5, 70, 2000])
def test_plan_of_lengths_that_cannot_be(hip, B):
    rng = random.Random(B)
    for _ in range(6):
        width = rng.choice([0, 1, 3, 17])
        n_pages = rng.choice([0, 1, 31, 32, 33, 50])
        tables, lens, new = _case(rng, B, 16, width, n_pages, 40, wild=True)
        for n_tokens in (0, 1, 500, 5000):
            assert list(_plan(tables, lens, new, n_tokens, n_pages, 16)) == list(P.plan(tables, lens, new, n_tokens, n_pages, 16))


def test_plan_of_the_largest_pool(hip):
    """2^20 pages, nearly all of them held by 2048 requests, some of them by several."""
    B, width, page, n_pages = 2048, 520, 16, 1 << 20
    g = torch.Generator(device=DEV).manual_seed(5)
    tables = torch.randperm(n_pages, generator=g, device=DEV)[:B * 511].view(B, 511).to(torch.int32)
    tables = torch.cat((tables, torch.full((B, width - 511), -1, dtype=torch.int32, device=DEV)), 1).contiguous()
    tables[7, :100] = tables[8, :100]
    lens = torch.randint(500 * page, 511 * page, (B,), generator=g, device=DEV, dtype=torch.int32)
    new = torch.randint(0, 60, (B,), generator=g, device=DEV, dtype=torch.int32)
    total = int(new.sum())
    want = P.plan(tables.tolist(), lens.tolist(), new.tolist(), total, n_pages, page)
    got = _plan(tables.tolist(), lens.tolist(), new.tolist(), total, n_pages, page)
    assert list(got) == list(want)


def test_plan_hands_out_pages_in_order_and_says_who_got_none(hip):
    tables = [[5, 7, -1, -1], [-1] * 4, [2, -1, -1, -1], [7, -1, -1, -1]]
    # free: 0, 1, 3, 4, 6 of 8 pages.  0: 20 tokens + 12 fit its two pages; 1: 32 tokens, two pages; 2: 16 + 33 tokens, three; 3: has room in its own
    got = _plan(tables, [20, 0, 16, 3], [12, 32, 33, 2], 79, 8, 16)
    assert got[0] == [[5, 7, -1, -1], [0, 1, -1, -1], [2, 3, 4, 6], [7, -1, -1, -1]]
    assert got[1] == [32, 32, 49, 5] and got[2] == [0, 12, 44, 77, 79] and got[4] == [True] * 4
    assert got[3] == list(range(7 * 16 + 4, 8 * 16)) + list(range(32)) + list(range(48, 80)) + [96] + [7 * 16 + 3, 7 * 16 + 4]
    # of 6 pages (7 is none of them) 0, 1, 3, 4 are free: two are left for 2, one too few
    got = _plan(tables, [20, 0, 16, 3], [12, 32, 33, 2], 79, 6, 16)
    assert got[0] == [[5, 7, -1, -1], [0, 1, -1, -1], [2, -1, -1, -1], [7, -1, -1, -1]]
    assert got[1] == [32, 32, 16, 5] and got[2] == [0, 12, 44, 77, 79] and got[4] == [True, True, False, True]
    assert got[3] == [-1] * 12 + list(range(32)) + [-1] * 35


def test_tables_with_rows_apart(hip):
    from ditango_amd.pages import plan_pages
    wide = torch.full((3, 50), 9, dtype=torch.int32, device=DEV)
    plan_pages(wide[:, 4:8], _i32([0, 16, 0]), _i32([40, 1, 5]), 46, n_pages=20, page_size=16)
    assert wide[:, 4:8].tolist() == [[0, 1, 2, 9], [9, 3, 9, 9], [4, 9, 9, 9]] and bool((wide[:, :4] == 9).all()) and bool((wide[:, 8:] == 9).all())


def _pools(g, n_pages, page, Hk, D, dtype, layout):
    """Pages as they may lie in memory: dense, heads outermost in a page, keys and values of a page side by side, in a larger pool."""
    mk = lambda *s: torch.randn(*s, generator=g, device=DEV).to(dtype)
    if layout == "dense":
        return mk(n_pages, page, Hk, D), mk(n_pages, page, Hk, D)
    if layout == "heads first":
        return mk(n_pages, Hk, page, D).transpose(1, 2), mk(n_pages, Hk, page, D).transpose(1, 2)
    if layout == "together":
        both = mk(n_pages, page, Hk, 2, D)
        return both[..., 0, :], both[..., 1, :]
    both = mk(n_pages, 2, page, Hk + 1, D + 8)
    return both[:, 0, :, :Hk, :D], both[:, 1, :, 1:, 8:]


LAYOUTS = ["dense", "heads first", "together", "apart"]


@pytest.mark.parametrize("layout", LAYOUTS)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("T, Hk, D, page", [(1, 1, 64, 16), (5, 3, 128, 48), (77, 12, 64, 16), (1000, 5, 128, 256), (2049, 24, 64, 32)])
def test_append_writes_its_slots_and_nothing_else(hip, T, Hk, D, page, dtype, layout):
    from ditango_amd.pages import append_pages
    g = torch.Generator(device=DEV).manual_seed(T)
    n_pages = T // page + 3
    kp, vp = _pools(g, n_pages, page, Hk, D, dtype, layout)
    slots = torch.randperm(n_pages * page, generator=g, device=DEV)[:T]
    slots[torch.rand(T, generator=g, device=DEV) < 0.1] = -1
    slots[T // 2] = n_pages * page                       # behind the pool
    if T > 3:
        slots[0], slots[1], slots[2] = -2 ** 63, 2 ** 63 - 1, 2 ** 32 + 5
    kv = torch.randn(T, 2 * Hk, D, generator=g, device=DEV).to(dtype)
    k, v = kv[:, :Hk], kv[:, Hk:]
    want = []
    there = (slots >= 0) & (slots < n_pages * page)
    for pool, x in ((kp, k), (vp, v)):
        rows = pool.clone().reshape(n_pages * page, Hk, D)
        rows[slots[there]] = x[there]
        want.append(rows.view(n_pages, page, Hk, D))
    append_pages(k, v, kp, vp, slots)
    assert torch.equal(kp, want[0]) and torch.equal(vp, want[1])


AXES = [dict(dims=(16, 24, 24), base=10000.0), dict(dims=(16, 56, 56), base=256.0), dict(dims=(64, 32, 32), pairing="rotate_half"),
        dict(dims=(32, 16, 16), pairing="rotate_half", base=(100.0, 5000.0, 1.5)), dict(dims=(64, 64), pairing="rotate_half", halves="head")]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("norm", [None, "rms", "layer_norm"])
@pytest.mark.parametrize("axes", range(len(AXES)))
def test_prepare_is_the_producer_and_the_append(hip, axes, norm, dtype):
    from ditango_amd.pages import append_pages, prepare_qkv_pages
    from ditango_amd.producer import RotaryAxes, prepare_qk_axes
    spec = RotaryAxes(**AXES[axes])
    D = sum(spec.dims)
    g = torch.Generator(device=DEV).manual_seed(axes)
    for T, H, Hk, page, layout in ((1, 1, 1, 16, "dense"), (37, 5, 5, 16, "heads first"), (200, 12, 3, 48, "together"), (1500, 24, 8, 64, "apart"), (900, 48, 48, 128, "dense")):
        n_pages = T // page + 2
        kp, vp = _pools(g, n_pages, page, Hk, D, dtype, layout)
        slots = torch.randperm(n_pages * page, generator=g, device=DEV)[:T]
        slots[torch.rand(T, generator=g, device=DEV) < 0.1] = -1
        slots[0] = n_pages * page
        qkv = (torch.randn(T, H + 2 * Hk, D, generator=g, device=DEV) * 2 + 0.2).to(dtype)
        q, k, v = qkv[:, :H], qkv[:, H:H + Hk], qkv[:, H + Hk:]
        w = [(torch.rand(D, generator=g, device=DEV) + 0.5).to(dtype) for _ in range(2)] if norm else [None, None]
        b = [torch.randn(D, generator=g, device=DEV) * 0.1 for _ in range(2)] if norm == "layer_norm" else [None, None]
        pos = torch.randint(-1000, 100000, (T, len(spec.dims)), generator=g, device=DEV, dtype=torch.int32)
        kw = dict(norm=norm, q_weight=w[0], k_weight=w[1], q_bias=b[0], k_bias=b[1])
        want_q, want_k = prepare_qk_axes(q[None], k[None], pos, spec, **kw)
        want = kp.clone(), vp.clone()
        append_pages(want_k[0], v, want[0], want[1], slots)
        y = prepare_qkv_pages(q, k, v, pos, spec, kp, vp, slots, **kw)
        assert y.is_contiguous() and torch.equal(y, want_q[0]) and torch.equal(kp, want[0]) and torch.equal(vp, want[1])
        packed = q.contiguous()
        assert prepare_qkv_pages(packed, k, v, pos, spec, kp, vp, slots, out=packed, **kw).data_ptr() == packed.data_ptr()
        assert torch.equal(packed, want_q[0]) and torch.equal(kp, want[0])


def test_nothing_to_do(hip):
    from ditango_amd.pages import append_pages, paged_attention, plan_pages, prepare_qkv_pages
    from ditango_amd.producer import RotaryAxes
    pages = torch.zeros(2, 16, 3, 64, device=DEV).bfloat16()
    none = torch.empty(0, 3, 64, device=DEV).bfloat16()
    slots = torch.empty(0, dtype=torch.int64, device=DEV)
    append_pages(none, none, pages, pages, slots)
    y = prepare_qkv_pages(none, none, none, torch.empty(0, 3, dtype=torch.int32, device=DEV), RotaryAxes(dims=(16, 24, 24)), pages, pages, slots)
    assert y.shape == (0, 3, 64)
    plan = plan_pages(_i32([[0], [1]]), _i32([3, 16]), _i32([0, 0]), 0, n_pages=2, page_size=16)
    assert plan.lens.tolist() == [3, 16] and plan.served.tolist() == [True, True] and plan.slots.numel() == 0
    out, lse = paged_attention(none, pages, pages, _i32([[0], [1]]), plan.lens, plan.cu_seqlens)
    assert out.shape == (0, 3, 64) and lse.shape == (3, 0)
    torch.cuda.synchronize()
