"""Which kernels the windowed attention launches, and in which order, without a GPU (tests/window_log.py)."""
from tests.test_window_layouts_gpu import SIZES
from tests.window_log import record


def test_the_gpu_tests_of_layouts_reach_every_form(tmp_path):
    calls = [dict(kind="window", B=B, Sq=Sq, Sk=Sk, H=H, Hk=Hk, D=D, **w) for D in (64, 128) for B, Sq, Sk, H, Hk, w in SIZES]
    names = [[k for _, k in kernels] for kernels in record(tmp_path, calls)]
    for D in (64, 128):
        for form in (f"attn_window_kernelILi{D}E", f"attn_window_few_kernelILi{D}ELb0ELi8E", f"attn_window_few_kernelILi{D}ELb0ELi4E"):
            assert any(form in ks[0] for ks in names), form
    assert any("fold_kernelILi128E" in ks[-1] for ks in names) and any(len(ks) == 1 for ks in names)
