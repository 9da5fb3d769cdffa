"""The operators of a cache of pages at the ends of what they take: no pages, no entries, one huge page, as many requests as there may be, and the launches that
cut their work in every way there is, with undefined values in masked and in visible places."""
import pytest
import torch

from tests.test_paged_attention_gpu import _check, _i32, _run, _setup

pytestmark = pytest.mark.gpu

DEV = "cuda:0"


def test_the_step_adapter_hands_it_out(hip):
    from ditango_amd.core import config, parallel_state
    from ditango_amd.executor.step.attentions import Attention
    from ditango_amd.pages import plan_pages
    config.init_config(None)
    parallel_state.init_local_groups(1, 0)
    try:
        attend = Attention(0).attn_processor("paged")
        before, new, Hk, D, page = [130, 64], [70, 3], 2, 128, 32
        q, kp, vp, tables, cu = _setup(before, new, 4, Hk, D, page, torch.bfloat16, spare=9)
        width = len(tables[0]) + 3
        rows = _i32([t + [-1] * (width - len(t)) for t in tables])
        plan = plan_pages(rows, _i32(before), _i32(new), q.shape[0], n_pages=kp.shape[0], page_size=page)
        k, v = (torch.randn(q.shape[0], Hk, D, device=DEV).bfloat16() for _ in range(2))
        got = attend(q, k, v, kp, vp, rows, plan, causal=True, left=1, frame=64, sinks=64)
        lens = [a + b for a, b in zip(before, new)]
        assert plan.lens.tolist() == lens
        want, lse = _run(q, kp, vp, rows.tolist(), lens, cu, left=1, right=0, frame=64, sinks=64)
        assert torch.equal(got, want)
        _check(want, lse, q, kp, vp, rows.tolist(), lens, cu, left=1, right=0, frame=64, sinks=64)
        with pytest.raises(ValueError, match="causal"):
            attend(q, k, v, kp, vp, rows, plan, causal=True, right=1)
    finally:
        parallel_state.destroy_local_groups()


@pytest.mark.parametrize("rows", [3, 300])
@pytest.mark.parametrize("D", [64, 128])
def test_no_pages_and_no_entries(hip, D, rows):
    from ditango_amd.pages import append_pages, paged_attention, plan_pages
    q = torch.randn(rows, 2, D, device=DEV).bfloat16()
    none = torch.empty(0, 16, 2, D, device=DEV, dtype=torch.bfloat16)
    some = torch.randn(4, 16, 2, D, device=DEV).bfloat16()
    for pages, width, lens in ((none, 0, 500), (some, 0, 500), (some, 3, 0)):
        tables = torch.zeros(2, width, device=DEV, dtype=torch.int32)
        out, lse = paged_attention(q, pages, pages, tables, _i32([lens, lens]), _i32([0, rows - 1, rows]), right=0)
        assert bool((out == 0).all()) and bool((lse == -float("inf")).all())
    # entries but no page: keys and values of zeros
    out, lse = paged_attention(q, none, none, torch.zeros(2, 40, device=DEV, dtype=torch.int32), _i32([600, 50]), _i32([0, rows - 1, rows]))
    assert bool((out == 0).all())
    assert float((lse[:, :-1].double() - torch.tensor(600.0).double().log()).abs().max()) < 2.0 ** -18
    assert float((lse[:, -1].double() - torch.tensor(50.0).double().log()).abs().max()) < 2.0 ** -18
    append_pages(q, q, none, none, torch.zeros(rows, device=DEV, dtype=torch.int64))
    for n_pages, width in ((0, 5), (5, 0), (0, 0)):
        tables = torch.full((3, width), 7, device=DEV, dtype=torch.int32)
        plan = plan_pages(tables, _i32([0, 0, 0]), _i32([0, rows, 0]), rows, n_pages=n_pages, page_size=16)
        assert plan.lens.tolist() == [0, 0, 0] and plan.served.tolist() == [True, False, True] and bool((plan.slots == -1).all())
        assert bool((tables == 7).all())


@pytest.mark.parametrize("D", [64, 128])
def test_one_huge_page(hip, D):
    lens, new = [9000, 401], [300, 2]
    q, kp, vp, tables, cu = _setup(lens, new, 4, 2, D, 9008, torch.bfloat16, spare=0)
    for w in (dict(right=0), dict(left=900, right=0, sinks=33)):
        out, lse = _run(q, kp, vp, tables, lens, cu, **w)
        _check(out, lse, q, kp, vp, tables, lens, cu, **w)


@pytest.mark.parametrize("most", [1, 200])
def test_as_many_requests_as_there_may_be(hip, most):
    B = 2048
    new = [b % 3 == 0 for b in range(B)]
    new = [int(n) for n in new]
    new[7], new[2047] = most, most
    lens = [n + b % 41 for b, n in enumerate(new)]
    lens[2047] += 3000
    q, kp, vp, tables, cu = _setup(lens, new, 2, 1, 64, 16, torch.float16, junk=float("inf"), behind=2)
    out, lse = _run(q, kp, vp, tables, lens, cu, most, right=0)
    _check(out, lse, q, kp, vp, tables, lens, cu, right=0)


CUTS = {      # lens, new, H, Hk
    "rows of three tiles, keys in parts": ([8000, 5001, 700], [40, 37, 40], 12, 6),
    "little work, all of it in tiles of 32": ([2400, 300], [139, 5], 8, 8),
    "all tiles of 256 rows in parts": ([9000, 60], [250, 1], 9, 9),
    "the last round of tiles of 256 rows in parts": ([2000, 3000, 900], [1500, 256, 1], 42, 42),
}


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("name", CUTS)
def test_undefined_values_however_the_work_is_cut(hip, name, D):
    """Infinities behind every request; visible infinite values, each seen by some rows and not by others; then a key that one row sees."""
    lens, new, H, Hk = CUTS[name]
    q, kp, vp, tables, cu = _setup(lens, new, H, Hk, D, 64, torch.bfloat16, junk=float("inf"), seed=len(name))
    w = dict(right=0)
    out, lse = _run(q, kp, vp, tables, lens, cu, max(new), **w)
    _check(out, lse, q, kp, vp, tables, lens, cu, **w)
    j = lens[0] - new[0] // 2
    vp[tables[0][j // 64], j % 64, Hk - 1, D - 3] = float("inf")
    vp[tables[0][1], 5, 0, 1] = -float("inf")
    for w in (dict(right=0), dict(left=lens[0] - new[0] // 3 - 70, right=0)):
        out, lse = _run(q, kp, vp, tables, lens, cu, max(new), **w)
        _check(out, lse, q, kp, vp, tables, lens, cu, **w)

    i = lens[1] - 1
    defined = kp.clone()
    kp[tables[1][i // 64], i % 64, 0, 7] = float("nan")
    hurt = torch.zeros(q.shape[0], H, 1, device=DEV, dtype=torch.bool)
    hurt[cu[2] - 1, :H // Hk] = True
    got = _run(q, kp, vp, tables, lens, cu, max(new), **w)
    assert bool((got[0].isnan() == (out.isnan() | hurt)).all()) and bool((got[1].isnan() == hurt[..., 0].t()).all())
    # (the rows beside it stay within their bound, not the same bits: its tile is computed once more, from exact maxima)
    _check(torch.where(hurt, out, got[0]), torch.where(hurt[..., 0].t(), lse, got[1]), q, defined, vp, tables, lens, cu, **w)


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("rows", [65, 97, 128, 129, 161, 225, 256, 257, 353])
def test_tiles_that_are_not_full(hip, rows, D):
    """Wavefronts of a tile of 256 rows that have none, beside others: with one part and with many, on short lists of tiles and on long ones."""
    for B, len_, H, Hk, w in ((3, 9000, 2, 2, dict(right=0)), (40, 500, 8, 8, dict(right=0)), (5, 420, 20, 20, dict(left=30, right=0, sinks=7)), (66, rows, 4, 4, dict(right=0))):
        lens, new = [len_ + b for b in range(B)], [rows] + [1] * (B - 2) + [rows]
        q, kp, vp, tables, cu = _setup(lens, new, H, Hk, D, 32, torch.bfloat16, junk=float("inf"), seed=rows)
        vp[tables[0][0], 3, 0, 0] = float("inf")
        out, lse = _run(q, kp, vp, tables, lens, cu, rows, **w)
        _check(out, lse, q, kp, vp, tables, lens, cu, **w)


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("len_, rows, H, Hk", [(38000, 617, 2, 2), (20000, 255, 1, 1), (9000, 140, 6, 3), (60000, 300, 4, 1)])
def test_many_parts_meet(hip, len_, rows, H, Hk, D):
    """Tiles of 256 rows whose keys are cut into many parts, which meet in groups: within their bound, the same bits each time, counters left at zero."""
    q, kp, vp, tables, cu = _setup([len_, 300], [rows, 1], H, Hk, D, 64, torch.bfloat16, junk=float("inf"), seed=rows)
    out, lse = _run(q, kp, vp, tables, [len_, 300], cu, rows, right=0)
    _check(out, lse, q, kp, vp, tables, [len_, 300], cu, right=0)
    for _ in range(5):
        again = _run(q, kp, vp, tables, [len_, 300], cu, rows, right=0)
        assert torch.equal(again[0], out) and torch.equal(again[1], lse)
    for counters in hip._counters.values():
        assert not bool(counters.any())
    vp[tables[0][0], 5, 0, 1] = -float("inf")
    j = len_ - rows // 2
    vp[tables[0][j // 64], j % 64, Hk - 1, D - 3] = float("inf")
    out, lse = _run(q, kp, vp, tables, [len_, 300], cu, rows, right=0)
    _check(out, lse, q, kp, vp, tables, [len_, 300], cu, right=0)
