"""Register, scratch and occupancy budget of the operators for a cache of pages, and which kernels a call launches.  No GPU needed.

A copy of the argument tables in scratch, or a spilled register in the attention's loop, changes no result and costs a multiple of the time."""
import json
import subprocess
import sys

import pytest

from tests.launch_log import LIB, _RUNTIME


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


def test_paged_attention(resources):
    for fragment, n in (("attn_pages_kernel", 4), ("attn_pages_few_kernel", 8)):
        for name, r in _kernels(resources, fragment, n).items():
            # heads of 64: some registers around the few rows' loop, none within it
            assert r["ScratchSize [bytes/lane]"] <= (0 if "ILi128E" in name else 40), (name, r)
            assert r["Occupancy [waves/SIMD]"] >= (2 if "ILi128E" in name else 4), (name, r)


@pytest.mark.parametrize("fragment, n", [("plan_pages_kernel", 1), ("plan_slots_kernel", 1), ("append_pages_kernel", 1), ("prepare_pages_kernel", 32)])
def test_the_others_use_no_scratch(resources, fragment, n):
    for name, r in _kernels(resources, fragment, n).items():
        assert r["ScratchSize [bytes/lane]"] == 0 and r["VGPRs Spill"] == 0, (name, r)


_PROCESS = r"""
import ctypes, json, sys
runtime = ctypes.CDLL(sys.argv[1], mode=ctypes.RTLD_GLOBAL)
runtime.log_text.restype = ctypes.c_char_p
lib = ctypes.CDLL(sys.argv[2])
i32, i64, vp, f32 = ctypes.c_int32, ctypes.c_int64, ctypes.c_void_p, ctypes.c_float
lib.dt_attn_workspace_bytes.restype = i64
lib.dt_last_error.restype = ctypes.c_char_p
AT = 1 << 20   # any aligned address

class Window(ctypes.Structure):
    _fields_ = [(n, i32) for n in ("left", "right", "frame", "sinks", "q_begin")] + [("kv_lens", vp)]
class Pool(ctypes.Structure):
    _fields_ = [("k", vp), ("v", vp), ("ks", i64 * 3), ("vs", i64 * 3), ("n_pages", i32), ("page_size", i32)]

def attend(T, B, H, Hk, D, most):
    s = (i64 * 3)(16 * Hk * D, Hk * D, D)
    pool, w = Pool(AT, AT, s, s, 100, 16), Window(-1, 0, 1, 0, -1, None)
    return lib.dt_attn_pages_fwd(vp(AT), (i64 * 2)(H * D, D), vp(AT), vp(AT), *[i32(x) for x in (T, H, Hk, D)], ctypes.byref(pool), vp(AT), i64(64), i32(64), i32(B),
                                 vp(AT), vp(AT), i32(most), ctypes.byref(w), f32(0), i32(0), vp(AT), i64(lib.dt_attn_workspace_bytes()), vp(AT), i64(1 << 18), vp(0))

def plan(B, T):
    return lib.dt_plan_pages(vp(AT), i64(64), i32(64), vp(AT), vp(AT), i32(B), i32(1000), i32(16), i32(T), vp(AT), vp(AT), vp(AT), vp(AT), vp(0))

answer = []
for kind, *args in json.loads(sys.stdin.read()):
    runtime.log_clear()
    rc = {"attend": attend, "plan": plan}[kind](*args)
    assert rc == 0, lib.dt_last_error()
    answer.append([line.split(" ", 1)[1] for line in runtime.log_text().decode().splitlines()])
print(json.dumps(answer))
"""


def _record(tmp_path, calls):
    source, runtime, script = tmp_path / "runtime.cpp", tmp_path / "runtime.so", tmp_path / "process.py"
    source.write_text(_RUNTIME)
    subprocess.run(["g++", "-shared", "-fPIC", "-O1", "-o", str(runtime), str(source)], check=True)
    script.write_text(_PROCESS)
    run = subprocess.run([sys.executable, str(script), str(runtime), LIB], input=json.dumps(calls), capture_output=True, text=True, timeout=100)
    assert run.returncode == 0, run.stderr[-2000:]
    return json.loads(run.stdout)


def test_which_kernels_run(tmp_path):
    """One launch an attention call: few rows with four wavefronts or eight, or both forms; a plan of many tokens finds their slots behind it."""
    calls = [("attend", 8, 8, 24, 24, 128, 1), ("attend", 2, 2, 8, 8, 64, 1), ("attend", 2000, 8, 24, 24, 128, 1900), ("attend", 300, 3, 8, 1, 64, 100),
             ("plan", 8, 8), ("plan", 8, 5000)]
    kernels = _record(tmp_path, calls)
    assert [len(k) for k in kernels] == [1, 1, 1, 1, 1, 2]
    for k, fragment in zip(kernels, ("attn_pages_few_kernelILi128ELb0ELi4E", "attn_pages_few_kernelILi64ELb0ELi8E", "attn_pages_kernelILi128E", "attn_pages_kernelILi64E",
                                     "plan_pages_kernel", "plan_pages_kernel")):
        assert fragment in k[0]
    assert "plan_slots_kernel" in kernels[-1][1]
