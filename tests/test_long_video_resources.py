"""Register, scratch and occupancy budget of the operators for long videos, from the build's record.  No GPU needed.

A copy of the argument tables in scratch, or a spilled register in the windowed attention's loop (whose reload waits for every tile load under way), changes
no result and costs a multiple of the time."""
import json

import pytest


@pytest.fixture(scope="module")
def resources():
    from ditango_amd import build
    if not build.RESOURCES_PATH.exists() or not build.LIB_PATH.exists():
        build.build_lib()
    flat = {}
    for per_file in json.loads(build.RESOURCES_PATH.read_text()).values():
        flat.update(per_file)
    return flat


def _kernels(resources, fragment, n):
    found = {k: v for k, v in resources.items() if fragment in k}
    assert len(found) == n, (fragment, sorted(found))
    return found


def test_windowed_attention(resources):
    for name, r in _kernels(resources, "attn_window_kernel", 4).items():
        assert r["ScratchSize [bytes/lane]"] == 0 and r["VGPRs Spill"] == 0, (name, r)
        assert r["Occupancy [waves/SIMD]"] == (2 if "ILi128E" in name else 4), (name, r)
    for name, r in _kernels(resources, "attn_window_few_kernel", 8).items():
        # heads of 64: some registers around the loop, none within it
        assert r["ScratchSize [bytes/lane]"] <= (0 if "ILi128E" in name else 40), (name, r)
        assert r["Occupancy [waves/SIMD]"] == (2 if "ILi128E" in name else 4), (name, r)


@pytest.mark.parametrize("fragment, n", [("attn_window_fold_kernel", 4), ("merge_blocks_kernel", 4), ("copy_blocks_kernel", 12), ("qk_norm_rope_axes_kernel", 32)])
def test_streaming_kernels_use_no_scratch(resources, fragment, n):
    for name, r in _kernels(resources, fragment, n).items():
        assert r["ScratchSize [bytes/lane]"] == 0 and r["VGPRs Spill"] == 0, (name, r)
