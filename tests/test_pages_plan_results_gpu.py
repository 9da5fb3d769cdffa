"""The results of a plan of pages are parts of one allocation: tensors like any others, in inference mode and on other streams too."""
import io

import pytest
import torch

from oracle import pages as P

pytestmark = pytest.mark.gpu

DEV = "cuda:0"


def _i32(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


def _plan(new, tables, lens, **kw):
    from ditango_amd.pages import plan_pages
    return plan_pages(tables, lens, _i32(new), sum(new) + 1, n_pages=20, page_size=16, **kw)


@pytest.mark.parametrize("B", [1, 2, 3])
@pytest.mark.parametrize("mode", [torch.no_grad, torch.inference_mode, torch.enable_grad])
def test_tensors_like_any_others(hip, B, mode):
    with mode():
        tables, lens = torch.full((B, 6), -1, dtype=torch.int32, device=DEV), _i32([0] * B)
        for turn in range(3):                     # a plan's lengths are the next one's
            new = [5 + turn + b for b in range(B)]
            want = P.plan(tables.tolist(), lens.tolist(), new, sum(new) + 1, 20, 16)
            plan = _plan(new, tables, lens)
            assert [tables.tolist(), *(x.tolist() for x in plan)] == list(want)
            parts = [(x.data_ptr(), x.data_ptr() + x.numel() * x.element_size()) for x in plan]
            for x, (lo, hi) in zip(plan, parts):
                assert lo % x.element_size() == 0 and x.is_contiguous() and not x.requires_grad
                assert sum(a < hi and lo < b for a, b in parts) == 1
            lens = plan.lens
        plan.lens.add_(1)                         # writes to one change no other
        assert [x.tolist() for x in plan[1:]] == list(want)[2:] and plan.lens.tolist() == [n + 1 for n in want[1]]


def test_saved_as_clones(hip):
    plan = _plan([5, 17], torch.full((2, 6), -1, dtype=torch.int32, device=DEV), _i32([0, 0]))
    file = io.BytesIO()
    torch.save([x.clone() for x in plan], file)
    file.seek(0)
    assert all(torch.equal(a, b) for a, b in zip(plan, torch.load(file, weights_only=True)))
    lens = plan.lens.clone()
    assert lens.untyped_storage().nbytes() == 8


def test_kept_on_another_stream(hip):
    """The allocation goes back once the streams that it is recorded on are through with it, whichever of its parts is recorded."""
    side = torch.cuda.Stream()
    tables, lens = torch.full((2, 6), -1, dtype=torch.int32, device=DEV), _i32([0, 0])
    for part in range(4):
        plan = _plan([5, 17], tables, lens)
        want = [x.tolist() for x in plan]
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            torch.cuda._sleep(20_000_000)
            got = [x.clone() for x in plan]
        plan[part].record_stream(side)
        del plan
        for _ in range(8):                        # would take its place
            _plan([5, 17], tables, lens, in_place=False)[2].fill_(-5)
        torch.cuda.synchronize()
        assert [x.tolist() for x in got] == want
        tables.fill_(-1)
