"""``paged_attention`` against its definition in float64; the bound is that of ``tests/test_window_gpu.py``:
  |out - o| <= u |o| + (u + e) sum_j w_j |v_j|,   |lse - l| <= e + 2^-21 |l|,   e = (D + 8) 2^-24 max sum |q k| scale + 2^-18,
and for fp16, whose probabilities below 2^-14 lose no more than 2^-25 each, + keys 2^-25 max |v|.
"""
import math
import random

import pytest
import torch

from oracle import pages as P

pytestmark = pytest.mark.gpu

DEV = "cuda:0"


def _i32(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


def _cu(new):
    cu = [0]
    for n in new:
        cu.append(cu[-1] + n)
    return cu


def _setup(lens, new, H, Hk, D, page, dtype, seed=0, sigma=1.5, junk=float("nan"), behind=0, spare=2):
    """Requests on pages in any order; every place that no request's token has holds `junk`, entries behind a request's last one are no pages."""
    g = torch.Generator(device=DEV).manual_seed(seed)
    held = [-(-n // page) for n in lens]
    n_pages = sum(held) + spare
    ids = torch.randperm(n_pages, generator=g, device=DEV).tolist()
    width = max(held + [1]) + 1
    tables = []
    for h in held:
        tables.append([ids.pop() for _ in range(h)] + [random.Random(seed).choice([-1, n_pages, 2 ** 31 - 1, -2 ** 31])] * (width - h))
    kp = torch.full((n_pages, page, Hk, D), junk, device=DEV, dtype=dtype)
    vp = torch.full((n_pages, page, Hk, D), junk, device=DEV, dtype=dtype)
    for row, n in zip(tables, lens):
        for i in range(-(-n // page)):
            m = min(page, n - i * page)
            kp[row[i], :m] = (torch.randn(m, Hk, D, generator=g, device=DEV) * sigma).to(dtype)
            vp[row[i], :m] = torch.randn(m, Hk, D, generator=g, device=DEV).to(dtype)
    q = (torch.randn(sum(new) + behind, H, D, generator=g, device=DEV) * sigma).to(dtype)
    return q, kp, vp, tables, _cu(new)


def _check(out, lse, q, kp, vp, tables, lens, cu, **w):
    o, l, weight, top = P.attention(q, kp, vp, tables, lens, cu, **w)
    u = torch.finfo(q.dtype).eps / 2
    e = (q.shape[-1] + 8) * 2.0 ** -24 * top + 2.0 ** -18
    tol = u * o.abs() + (u + e) * weight
    if q.dtype is torch.float16:
        tol = tol + max([min(max(n, 0), 1 << 30) for n in lens]) * 2.0 ** -25 * torch.nan_to_num(vp.double(), posinf=0.0, neginf=0.0).abs().max()
    same = (out.double() == o) | (out.isnan() & o.isnan())
    assert bool((same | ((out.double() - o).abs() <= tol + 1e-30)).all()), float(((out.double() - o).abs() - tol).nan_to_num().max())
    empty = l == -math.inf
    assert bool((lse[empty] == -math.inf).all()) and bool((out.transpose(0, 1)[empty] == 0).all())
    known = ~empty & ~l.isnan()
    assert bool(lse[l.isnan()].isnan().all())
    d = (lse.double() - l)[known]
    assert bool((d.abs() <= e + 2.0 ** -21 * l[known].abs()).all()), float(d.abs().max())


def _run(q, kp, vp, tables, lens, cu, most=None, **w):
    from ditango_amd.pages import paged_attention
    out, lse = paged_attention(q, kp, vp, _i32(tables), _i32(lens), _i32(cu), max_seqlen_q=most, **w)
    torch.cuda.synchronize()
    assert out.shape == q.shape and out.dtype == q.dtype and lse.shape == (q.shape[1], q.shape[0]) and lse.dtype is torch.float32
    return out, lse


CASES = [
    # lens, new, H, Hk, page, window
    ([1], [1], 1, 1, 16, dict(right=0)),
    ([700], [1], 3, 3, 16, dict(left=99, right=0, sinks=4)),
    ([4001, 17, 260], [1, 1, 1], 4, 1, 64, dict(left=1500, right=0, sinks=64)),
    ([517, 3, 64, 65], [8, 3, 1, 2], 8, 2, 32, dict(right=0)),
    ([130], [130], 2, 2, 48, dict(left=0, right=0)),
    ([257, 300], [257, 20], 2, 1, 144, dict(left=31, right=32)),
    ([333, 90, 0], [100, 90, 0], 3, 3, 16, dict(left=17, right=0, sinks=65)),
    ([150, 400], [150, 37], 2, 2, 256, dict(left=1, right=0, frame=37, sinks=11)),
    ([460, 400], [60, 50], 6, 2, 16, dict(left=2, right=1, frame=50, sinks=13)),
    ([2000, 33, 1], [600, 1, 1], 4, 2, 64, dict()),
    ([5000, 4000], [40, 3], 16, 2, 16, dict(right=0)),
    ([700, 1], [513, 1], 2, 2, 1024, dict(right=0)),
    ([64, 128, 63, 65, 32, 31, 33], [1, 2, 1, 1, 32, 31, 33], 2, 1, 32, dict(right=0)),
    ([90, 20], [90, 20], 33, 1, 16, dict(right=0)),
    ([1100], [300], 40, 5, 80, dict(left=200, right=0)),
    ([20, 9], [40, 9], 2, 2, 16, dict(right=0)),                 # more rows than tokens: the first ones stand in front of every key
]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("case", range(len(CASES)))
def test_matches_the_definition(hip, case, D, dtype):
    lens, new, H, Hk, page, w = CASES[case]
    q, kp, vp, tables, cu = _setup(lens, new, H, Hk, D, page, dtype, seed=case)
    for most in (None, max(new)):
        out, lse = _run(q, kp, vp, tables, lens, cu, most, **w)
        _check(out, lse, q, kp, vp, tables, lens, cu, **w)


@pytest.mark.parametrize("most", [1, 40, 1000])
def test_the_hint_of_rows_changes_no_result(hip, most):
    lens, new = [900, 300, 40, 2000, 77], [500, 1, 40, 2, 60]
    q, kp, vp, tables, cu = _setup(lens, new, 4, 2, 128, 16, torch.bfloat16, behind=9)
    out, lse = _run(q, kp, vp, tables, lens, cu, most, right=0)
    _check(out, lse, q, kp, vp, tables, lens, cu, right=0)


def test_many_requests(hip):
    rng = random.Random(1)
    for B, most in ((64, 300), (65, 3), (200, 40), (1030, 2)):
        new = [rng.choice([0, 1, rng.randint(1, most)]) for _ in range(B)]
        lens = [n + rng.choice([0, 1, rng.randint(0, 200)]) for n in new]
        q, kp, vp, tables, cu = _setup(lens, new, 2, 1, 64, 16, torch.bfloat16, seed=B)
        out, lse = _run(q, kp, vp, tables, lens, cu, max(new), right=0, left=90, sinks=3)
        _check(out, lse, q, kp, vp, tables, lens, cu, right=0, left=90, sinks=3)


@pytest.mark.parametrize("seed", range(24))
def test_random_requests(hip, seed):
    rng = random.Random(seed)
    B = rng.choice([1, 2, 3, 5, 9])
    Hk = rng.choice([1, 2, 3, 8])
    H = Hk * rng.choice([1, 1, 2, 3, 7, 16])
    page = rng.choice([16, 32, 48, 64, 112, 128])
    new = [rng.choice([0, 1, rng.randint(1, 8), rng.randint(1, 400)]) for _ in range(B)]
    lens = [max(0, n + rng.choice([0, rng.randint(0, 60), rng.randint(0, 3000)])) for n in new]
    frame = rng.choice([1, 1, rng.randint(2, 200)])
    reach = rng.randint(0, 5) if frame > 1 else rng.randint(0, 600)
    w = dict(left=rng.choice([None, reach]), right=rng.choice([0, 0, None, reach]), frame=frame, sinks=rng.choice([0, 1, rng.randint(0, 150)]))
    D, dtype = rng.choice([64, 128]), rng.choice([torch.bfloat16, torch.float16])
    if sum(new) == 0:
        new[0], lens[0] = 1, lens[0] + 1
    q, kp, vp, tables, cu = _setup(lens, new, H, Hk, D, page, dtype, seed=seed, behind=rng.choice([0, 1, 40]))
    out, lse = _run(q, kp, vp, tables, lens, cu, **w)
    _check(out, lse, q, kp, vp, tables, lens, cu, **w)


@pytest.mark.parametrize("D", [64, 128])
def test_large_launches(hip, D):
    """Every form of the launch with work for the whole GPU: long caches of few rows, many rows, and both together."""
    for lens, new, H, Hk, w in (([9000, 30011, 517], [1, 1, 1], 8, 8, dict(right=0)),
                                ([20011], [2], 16, 1, dict(right=0)),
                                ([3000, 2999], [2500, 1200], 8, 4, dict(right=0)),
                                ([6000, 700, 5000, 44], [1000, 1, 3, 1], 8, 8, dict(right=0, left=3, frame=256, sinks=77))):
        q, kp, vp, tables, cu = _setup(lens, new, H, Hk, D, 64, torch.bfloat16, junk=float("inf"))
        out, lse = _run(q, kp, vp, tables, lens, cu, max(new), **w)
        _check(out, lse, q, kp, vp, tables, lens, cu, **w)


def test_rows_of_no_request(hip):
    """In front of the first boundary, behind the last one, between none."""
    lens, new = [100, 50], [30, 5]
    for D in (64, 128):
        q, kp, vp, tables, cu = _setup(lens, new, 3, 3, D, 16, torch.bfloat16, behind=70)
        cu = [c + 20 for c in cu]
        out, lse = torch.full_like(q, 7.0), torch.full((3, q.shape[0]), 7.0, device=DEV)
        got = _run(q, kp, vp, tables, lens, cu, right=0, out=out, lse=lse)
        assert got[0].data_ptr() == out.data_ptr() and got[1].data_ptr() == lse.data_ptr()
        _check(out, lse, q, kp, vp, tables, lens, cu, right=0)
        assert bool((out[:20] == 0).all()) and bool((out[55:] == 0).all())


@pytest.mark.parametrize("rows", [1, 3, 300])
def test_boundaries_and_lengths_that_cannot_be(hip, rows):
    """Clamped to what is there: nothing is read or written out of place."""
    q, kp, vp, tables, cu = _setup([100, 60], [rows, 4], 2, 2, 64, 16, torch.bfloat16, junk=0.25)
    width = len(tables[0])
    for lens, cu in (([10 ** 9, 60], cu), ([-5, -2 ** 31], cu), ([100, 60], [0, rows, 10 ** 9]), ([100, 60], [0, rows, -3]), ([100, 60], [-7, rows, rows + 4]),
                     ([2 ** 31 - 1, 2 ** 31 - 1], [0, 2 ** 31 - 1, 2 ** 31 - 1])):
        out, lse = _run(q, kp, vp, tables, lens, cu, right=0)
        _check(out, lse, q, kp, vp, tables, [min(n, width * 16) for n in lens], cu, right=0)


def test_overlapping_requests_end(hip):
    """Boundaries that fall: more rows in all than there are.  What comes out is not said, but the launch ends and touches nothing else."""
    q, kp, vp, tables, _ = _setup([100] * 200, [3] * 200, 2, 1, 64, 16, torch.bfloat16, junk=0.25)
    for cu in ([0, 600] * 100 + [0], [600, 0] * 100 + [600]):
        guard = torch.full((602, 2, 64), 5.0, device=DEV).bfloat16()
        out = guard[1:601]
        from ditango_amd.pages import paged_attention
        paged_attention(q, kp, vp, _i32(tables), _i32([100] * 200), _i32(cu), right=0, out=out)
        torch.cuda.synchronize()
        assert bool((guard[0] == 5).all()) and bool((guard[601] == 5).all())


@pytest.mark.parametrize("new", [1, 200])
def test_entries_that_are_no_pages_read_as_zeros(hip, new):
    lens = [333, 200]
    q, kp, vp, tables, cu = _setup(lens, [new, 1], 2, 2, 128, 16, torch.bfloat16)
    for i, bad in ((0, -1), (5, kp.shape[0]), (20, 2 ** 31 - 1), (11, -2 ** 31)):
        tables[0][i] = bad
    out, lse = _run(q, kp, vp, tables, lens, cu, right=0)
    _check(out, lse, q, kp, vp, tables, lens, cu, right=0)


def test_pages_of_the_past_may_go(hip):
    """Entries in front of every window are never looked at."""
    lens, new = [900, 700], [3, 260]
    for D in (64, 128):
        q, kp, vp, tables, cu = _setup(lens, new, 2, 2, D, 16, torch.float16)
        want = _run(q, kp, vp, tables, lens, cu, left=127, right=0, sinks=16)
        for b, n in enumerate(new):
            for i in range(1, (lens[b] - n - 127) // 16):
                kp[tables[b][i]] = float("nan")
                vp[tables[b][i]] = float("inf")
                tables[b][i] = -1
        got = _run(q, kp, vp, tables, lens, cu, left=127, right=0, sinks=16)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


@pytest.mark.parametrize("new", [1, 4, 300])
def test_undefined_values_stay_with_the_rows_that_see_them(hip, new):
    """Masked places hold infinities and NaN; visible ones too, and then the rows that see them, and no others, are undefined."""
    lens = [800, 333]
    for D, Hk in ((64, 1), (128, 2)):
        q, kp, vp, tables, cu = _setup(lens, [new, 2], 2, Hk, D, 16, torch.bfloat16)
        j = 800 - new // 2 - 1                       # seen by the later rows only
        vp[tables[0][j // 16], j % 16, 0, 3] = float("inf")
        vp[tables[0][1], 2, 0, 5] = float("nan")     # behind the window of most
        for w in (dict(right=0), dict(right=0, left=781), dict(right=0, left=40)):
            out, lse = _run(q, kp, vp, tables, lens, cu, **w)
            _check(out, lse, q, kp, vp, tables, lens, cu, **w)


def test_layouts(hip):
    """Pages and queries wherever they lie: heads first in a page, keys and values side by side, q a slice of a projection, rows of tables apart."""
    from ditango_amd.pages import paged_attention
    lens, new = [300, 77], [70, 1]
    for D in (64, 128):
        q, kp, vp, tables, cu = _setup(lens, new, 6, 3, D, 32, torch.bfloat16, junk=float("inf"))
        wide = torch.randn(q.shape[0], 20, D + 8, device=DEV).bfloat16()
        wide[:, 2:8, :D] = q
        want = _run(q, kp, vp, tables, lens, cu, right=0)
        both = torch.stack((kp, vp), 3).flatten(3)                                   # [pages, page, Hk, 2 D]
        apart = _i32([[9] * 3 + t + [5] for t in tables])
        for x, a, b in ((q, kp.transpose(1, 2).contiguous().transpose(1, 2), vp), (wide[:, 2:8, :D], both[..., :D], both[..., D:]),
                        (q, torch.cat((vp, kp), 1)[:, 32:], torch.cat((vp, kp), 1)[:, :32])):
            out, lse = paged_attention(x, a, b, apart[:, 3:-1], _i32(lens), _i32(cu), right=0)
            assert torch.equal(out, want[0]) and torch.equal(lse, want[1])
        same = q.clone()
        out, lse = paged_attention(same, kp, vp, _i32(tables), _i32(lens), _i32(cu), right=0, out=same)
        assert torch.equal(same, want[0]) and torch.equal(lse, want[1])


def test_shared_pages(hip):
    """Requests with one beginning, and one page at two places."""
    lens, new = [200, 180], [5, 60]
    q, kp, vp, tables, cu = _setup(lens, new, 2, 2, 64, 16, torch.bfloat16)
    tables[1][:6] = tables[0][:6]
    tables[0][7] = tables[0][3]
    out, lse = _run(q, kp, vp, tables, lens, cu, right=0)
    _check(out, lse, q, kp, vp, tables, lens, cu, right=0)


def test_scales_and_large_scores(hip):
    for D in (64, 128):
        lens, new = [500, 60], [90, 2]
        q, kp, vp, tables, cu = _setup(lens, new, 2, 2, D, 16, torch.bfloat16, sigma=6.0)
        for scale in (0.0, 0.02, 1.0):
            out, lse = _run(q, kp, vp, tables, lens, cu, right=0, softmax_scale=scale)
            _check(out, lse, q, kp, vp, tables, lens, cu, right=0, scale=scale or None)


def test_the_largest_offsets(hip):
    """A pool of more than 2^32 bytes, of which the last pages are read."""
    n_pages, page, Hk, D = 70000, 16, 24, 128        # 6.9 GB each
    kp = torch.zeros(n_pages, page, Hk, D, device=DEV, dtype=torch.bfloat16)
    vp = torch.zeros_like(kp)
    small_k, small_v = (torch.randn(40, page, Hk, D, device=DEV).bfloat16() for _ in range(2))
    at = torch.arange(n_pages - 40, n_pages, device=DEV)
    kp[at], vp[at] = small_k, small_v
    q = torch.randn(203, Hk, D, device=DEV).bfloat16()
    tables = torch.randperm(40, device=DEV).view(2, 20).to(torch.int32)
    lens, cu = [310, 320], [0, 200, 203]
    want = _run(q, small_k, small_v, tables.tolist(), lens, cu, right=0)
    got = _run(q, kp, vp, (tables + n_pages - 40).tolist(), lens, cu, right=0)
    assert torch.equal(want[0], got[0]) and torch.equal(want[1], got[1])
    _check(want[0], want[1], q, small_k, small_v, tables.tolist(), lens, cu, right=0)
    from ditango_amd.pages import append_pages
    new_k, new_v = (torch.randn(3, Hk, D, device=DEV).bfloat16() for _ in range(2))
    slots = torch.tensor([n_pages * page - 1, 0, (n_pages - 30) * page + 5], device=DEV)
    append_pages(new_k, new_v, kp, vp, slots)
    rows = kp.view(-1, Hk, D), vp.view(-1, Hk, D)
    assert torch.equal(rows[0][slots], new_k) and torch.equal(rows[1][slots], new_v)
