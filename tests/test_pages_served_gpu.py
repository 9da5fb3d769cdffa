"""Requests that a plan of pages refuses, in the attention behind it: their rows are in ``cu_seqlens``, but have neither keys nor a place, and get 0 and an lse of
-inf like rows of no request.  The bounds are those of ``tests/test_paged_attention_gpu.py``, of lengths that are 0 where a request is not served."""
import math

import pytest
import torch

from tests.test_paged_attention_gpu import _check, _i32, _setup

pytestmark = pytest.mark.gpu

DEV = "cuda:0"


def _refused(before, new, H, Hk, D, page, dtype, **kw):
    """(q, k pages, v pages, tables, plan): the pool has no page left, so that who needs one is refused."""
    from ditango_amd.pages import plan_pages
    q, kp, vp, tables, _ = _setup(before, new, H, Hk, D, page, dtype, spare=0, **kw)
    tables = _i32([t + [-1] * 20 for t in tables])
    return q, kp, vp, tables, plan_pages(tables, _i32(before), _i32(new), q.shape[0], n_pages=kp.shape[0], page_size=page)


def _seen(plan):
    return [n if s else 0 for n, s in zip(plan.lens.tolist(), plan.served.tolist())]


def _nothing(out, lse, plan):
    cu = plan.cu_seqlens.tolist()
    for b, served in enumerate(plan.served.tolist()):
        rows = slice(cu[b], cu[b + 1])
        assert served or bool((out[rows] == 0).all()) and (lse is None or bool((lse[:, rows] == -math.inf).all()))


def test_the_step_adapter(hip):
    from ditango_amd.core import config, parallel_state
    from ditango_amd.executor.step.attentions import Attention
    config.init_config(None)
    parallel_state.init_local_groups(1, 0)
    try:
        attend = Attention(0).attn_processor("paged")
        q, kp, vp, tables, plan = _refused([70, 200, 90], [10, 40, 4], 4, 2, 128, 32, torch.bfloat16)
        assert plan.served.tolist() == [True, False, True] and plan.lens.tolist() == [80, 200, 94]
        k, v = (torch.randn(q.shape[0], 2, 128, device=DEV).bfloat16() for _ in range(2))
        got = attend(q, k, v, kp, vp, tables, plan, causal=True)
        _nothing(got, None, plan)
        from ditango_amd.pages import paged_attention
        want = paged_attention(q, kp, vp, tables, _i32(_seen(plan)), plan.cu_seqlens, right=0)
        assert torch.equal(got, want[0])
    finally:
        parallel_state.destroy_local_groups()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("before, new, H, Hk", [
    ([60, 800, 33], [4, 1, 2], 4, 2),                    # few rows
    ([60, 3000, 9000], [4, 40, 7], 8, 2),                # ... in parts
    ([70, 900, 600], [10, 330, 300], 2, 2),              # tiles of 256 rows, the refused ones' among them
    ([16] * 70, [20 + b % 7 * 30 for b in range(70)], 3, 1),
])
def test_refused_requests_have_no_keys(hip, before, new, H, Hk, D, dtype):
    from ditango_amd.pages import paged_attention
    q, kp, vp, tables, plan = _refused(before, new, H, Hk, D, 16, dtype, behind=3, junk=0.25)      # (new tokens' places as well)
    served = plan.served.tolist()
    assert False in served
    for s in (served, [not x for x in served], [False] * len(new), [True] * len(new)):
        mask = torch.tensor(s, device=DEV)
        seen = [n if x else 0 for n, x in zip(plan.lens.tolist(), s)]
        for w in (dict(right=0), dict(left=1, right=0, frame=50, sinks=9)):
            out, lse = paged_attention(q, kp, vp, tables, plan.lens, plan.cu_seqlens, served=mask, max_seqlen_q=max(new), **w)
            torch.cuda.synchronize()
            want = paged_attention(q, kp, vp, tables, _i32(seen), plan.cu_seqlens, max_seqlen_q=max(new), **w)
            assert torch.equal(out, want[0]) and torch.equal(lse, want[1])
            if s == served:
                _nothing(out, lse, plan)
                _check(out, lse, q, kp, vp, tables.tolist(), seen, plan.cu_seqlens.tolist(), **w)
    out, lse = paged_attention(q, kp, vp, tables, plan.lens, plan.cu_seqlens, right=0)
    want = paged_attention(q, kp, vp, tables, plan.lens, plan.cu_seqlens, right=0, served=torch.ones(len(new), dtype=torch.bool, device=DEV))
    assert torch.equal(out, want[0]) and torch.equal(lse, want[1])


@pytest.mark.parametrize("new", [[5, 3], [40, 90]])
def test_a_captured_step_whose_pool_runs_dry(hip, new):
    """Nobody reads ``served`` on the host: replays go on, and once there is no page left the rows of who needs one are 0."""
    from ditango_amd.pages import append_pages, paged_attention, plan_pages
    H, D, page, n_pages = 2, 128, 16, 2 * sum(new) // 16 + 3
    g = torch.Generator(device=DEV).manual_seed(0)
    kp, vp = (torch.zeros(n_pages, page, H, D, device=DEV, dtype=torch.bfloat16) for _ in range(2))
    tables, lens, more = torch.full((2, 40), -1, dtype=torch.int32, device=DEV), _i32([0, 0]), _i32(new)
    q, k, v = (torch.randn(sum(new), H, D, generator=g, device=DEV).bfloat16() for _ in range(3))

    def step():
        plan = plan_pages(tables, lens, more, q.shape[0], n_pages=n_pages, page_size=page, in_place=True)
        append_pages(k, v, kp, vp, plan.slots)
        return plan, paged_attention(q, kp, vp, tables, plan.lens, plan.cu_seqlens, served=plan.served, right=0)

    step()
    torch.cuda.synchronize()
    lens.zero_()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        plan, (out, lse) = step()
    refused = 0
    for turn in range(12):          # (60 and 36 tokens need 7 pages of the 4, 480 and 1080 98 of the 19)
        for x in (q, k, v):
            x.copy_(torch.randn(sum(new), H, D, generator=g, device=DEV))
        graph.replay()
        torch.cuda.synchronize()
        _check(out, lse, q, kp, vp, tables.tolist(), _seen(plan), plan.cu_seqlens.tolist(), right=0)
        _nothing(out, lse, plan)
        refused += plan.served.tolist().count(False)
        want = paged_attention(q, kp, vp, tables, _i32(_seen(plan)), plan.cu_seqlens, right=0)
        assert torch.equal(out, want[0]) and torch.equal(lse, want[1])
    assert refused


def test_what_served_may_be(hip):
    from ditango_amd import _hip
    from ditango_amd.pages import paged_attention
    q, pages = torch.zeros(4, 2, 64, device=DEV).bfloat16(), torch.zeros(3, 16, 2, 64, device=DEV).bfloat16()
    tables, lens, cu = _i32([[0], [1]]), _i32([4, 4]), _i32([0, 2, 4])
    yes = torch.ones(2, dtype=torch.bool, device=DEV)
    for bad in (yes[:1], yes[None], yes.cpu(), torch.ones(4, dtype=torch.bool, device=DEV)[::2]):
        with pytest.raises(_hip.DitangoHipError, match="served"):
            paged_attention(q, pages, pages, tables, lens, cu, served=bad)
    out, lse = paged_attention(q, pages, pages, tables, lens, cu, served=torch.tensor([True, False], device=DEV))
    assert bool((out == 0).all()) and bool((lse[:, 2:] == -math.inf).all()) and float((lse[:, :2].double() - math.log(4)).abs().max()) < 2.0 ** -18
