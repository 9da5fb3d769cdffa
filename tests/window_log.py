"""Which kernels the windowed attention launches, without a GPU: ``tests/launch_log.py`` for ``dt_attn_window_fwd``."""
import json
import subprocess
import sys

from tests.launch_log import LIB, _RUNTIME

_PROCESS = r"""
import ctypes, json, sys, threading
runtime = ctypes.CDLL(sys.argv[1], mode=ctypes.RTLD_GLOBAL)
runtime.log_text.restype = ctypes.c_char_p
lib = ctypes.CDLL(sys.argv[2])
i32, i64, vp, f32 = ctypes.c_int32, ctypes.c_int64, ctypes.c_void_p, ctypes.c_float
lib.dt_attn_workspace_bytes.restype = i64
lib.dt_last_error.restype = ctypes.c_char_p
AT = 1 << 20   # any aligned address

class Window(ctypes.Structure):
    _fields_ = [(n, i32) for n in ("left", "right", "frame", "sinks", "q_begin")] + [("kv_lens", vp)]

def window(B, Sq, Sk, H, Hk, D, left=None, right=None, frame=1, sinks=0, q_begin=None, counters=True):
    strides = lambda S, heads: (i64 * 3)(S * heads * D, heads * D, D)
    limit = lambda x: -1 if x is None else x
    w = Window(limit(left), limit(right), frame, sinks, limit(q_begin), None)
    rc = lib.dt_attn_window_fwd(*[vp(AT)] * 5, *[i32(x) for x in (B, Sq, Sk, H, Hk, D)], strides(Sq, H), strides(Sk, Hk), strides(Sk, Hk), ctypes.byref(w), f32(0),
                                i32(0), vp(AT), i64(lib.dt_attn_workspace_bytes()), vp(AT if counters else 0), i64(1 << 18 if counters else 0), vp(0))
    assert rc == 0, lib.dt_last_error()

def chunk(B, Sq, Sk, H, D):
    # the attention launch of one chunk, split, with the workspace of the windowed launches
    at = (vp * 1)(AT)
    rc = lib.dt_attn_seg_jobs_ws_fwd(vp(AT), i32(B), i32(Sq), i32(H), i32(D), i64(Sq * H * D), i64(H * D), i64(D), i32(1), at, at, (i32 * 1)(Sk), (i64 * 1)(Sk * H * D),
                                     i64(H * D), i64(D), i32(1), (i32 * 2)(0, 1), (i32 * 1)(0), vp(0), vp(0), vp(0), vp(0), at, at, f32(0), i32(0), vp(AT),
                                     i64(lib.dt_attn_workspace_bytes()), vp(0))
    assert rc == 0, lib.dt_last_error()

def call(kind, **kw): {"window": window, "chunk": chunk}[kind](**kw)

asked = json.loads(sys.stdin.read())
answer = []
for calls in asked["in turn"]:
    runtime.log_clear()
    call(**calls)
    answer.append([line.split(" ", 1) for line in runtime.log_text().decode().splitlines()])
if asked["together"]:
    runtime.log_clear()
    runtime.log_wait(2000)
    start = threading.Barrier(len(asked["together"]))
    def work(c):
        start.wait()
        for _ in range(asked["times"]): call(**c)
    threads = [threading.Thread(target=work, args=(c,)) for c in asked["together"]]
    for t in threads: t.start()
    for t in threads: t.join()
    answer.append([line.split(" ", 1) for line in runtime.log_text().decode().splitlines()])
print(json.dumps(answer))
"""


def record(tmp_path, in_turn=(), together=(), times=0):
    """As ``tests.launch_log.record``; a call is ``dict(kind="window" or "chunk", ...)`` with the arguments of the functions above."""
    source, runtime = tmp_path / "runtime.cpp", tmp_path / "runtime.so"
    source.write_text(_RUNTIME)
    subprocess.run(["g++", "-shared", "-fPIC", "-O1", "-o", str(runtime), str(source)], check=True)
    script = tmp_path / "process.py"
    script.write_text(_PROCESS)
    asked = json.dumps({"in turn": list(in_turn), "together": list(together), "times": times})
    run = subprocess.run([sys.executable, str(script), str(runtime), LIB], input=asked, capture_output=True, text=True, timeout=100)
    assert run.returncode == 0, run.stderr[-2000:]
    return json.loads(run.stdout)
