"""Which kernels the windowed attention launches, and in which order, without a GPU (tests/window_log.py)."""
import pytest

from tests.test_window_layouts_gpu import SIZES
from tests.window_log import record


def test_the_gpu_tests_of_layouts_reach_every_form(tmp_path):
    calls = [dict(kind="window", B=B, Sq=Sq, Sk=Sk, H=H, Hk=Hk, D=D, **w) for D in (64, 128) for B, Sq, Sk, H, Hk, w in SIZES]
    names = [[k for _, k in kernels] for kernels in record(tmp_path, calls)]
    for D in (64, 128):
        for form in (f"attn_window_kernelILi{D}E", f"attn_window_few_kernelILi{D}ELb0ELi8E", f"attn_window_few_kernelILi{D}ELb0ELi4E"):
            assert any(form in ks[0] for ks in names), form
    assert any("fold_kernelILi128E" in ks[-1] for ks in names) and any(len(ks) == 1 for ks in names)


# launches whose parts a fold kernel reads: workgroups of 256 rows, and of 32 without counters; of 32 rows with counters, whose last part reads the others; and one of the
# attention of whole chunks, with the same workspace
SHARED = dict(kind="window", B=1, Sq=2100, Sk=2100, H=66, Hk=66, D=128, right=0)
FEW = dict(kind="window", B=1, Sq=2, Sk=30000, H=2, Hk=2, D=128, counters=False)
MEETING = dict(FEW, counters=True)
CHUNK = dict(kind="chunk", B=1, Sq=900, Sk=2600, H=2, D=128)


@pytest.mark.parametrize("call", [SHARED, FEW, CHUNK])
@pytest.mark.parametrize("other", [SHARED, FEW, MEETING, CHUNK])
def test_no_parts_come_between_parts_and_their_fold(tmp_path, call, other):
    """Two threads on one stream share its workspace: behind a launch whose parts a fold kernel reads comes that kernel, and no other launch."""
    alone, pair, both = record(tmp_path, [call, other], [call, other], 15)
    assert len(alone) == 2 and "fold" in alone[1][1]
    assert len(pair) == (1 if other is MEETING else 2)
    assert len(both) == 15 * (len(alone) + len(pair)) and len({t for t, _ in both}) == 2
    parts_of = {}
    for kernels in (alone, pair):
        if len(kernels) == 2:
            parts_of.setdefault(kernels[1][1], set()).add(kernels[0][1])
    for (t0, k0), (t1, k1) in zip(both, both[1:]):
        if k1 in parts_of:
            assert t0 == t1 and k0 in parts_of[k1]
