"""What the operators of long videos refuse, on the host, before any launch."""
import ctypes

import pytest
import torch

from ditango_amd import _hip


def _err(lib, rc, code=-1):
    assert rc == code, (rc, lib.dt_last_error())
    return lib.dt_last_error().decode()


class Window(ctypes.Structure):
    _fields_ = [(n, ctypes.c_int32) for n in ("left", "right", "frame", "sinks", "q_begin")] + [("kv_lens", ctypes.c_void_p)]


class State(ctypes.Structure):
    _fields_ = [("out", ctypes.c_void_p), ("scales", ctypes.c_void_p), ("lse", ctypes.c_void_p), ("dtype", ctypes.c_int32), ("lse_layout", ctypes.c_int32)]


class Rows(ctypes.Structure):
    _fields_ = [("x", ctypes.c_void_p), ("stride_b", ctypes.c_int64), ("stride_s", ctypes.c_int64), ("stride_h", ctypes.c_int64), ("y", ctypes.c_void_p),
                ("weight", ctypes.c_void_p), ("bias", ctypes.c_void_p), ("H", ctypes.c_int32), ("out_scale", ctypes.c_float)]


def test_window_arguments():
    lib = _hip.load_library()
    ok = dict(q=4096, k=4096, v=4096, out=4096, lse=4096, B=1, Sq=4, Sk=4, H=4, Hk=2, D=64, qs=(512, 128, 64), ks=(512, 128, 64), vs=(512, 128, 64),
              left=1, right=0, frame=1, sinks=0, q_begin=-1, flags=0, ws=None, bytes=0, counters=None, n=0)

    def call(**kw):
        a = {**ok, **kw}
        s = [None if a[n] is None else (ctypes.c_int64 * 3)(*a[n]) for n in ("qs", "ks", "vs")]
        w = Window(a["left"], a["right"], a["frame"], a["sinks"], a["q_begin"], None)
        return lib.dt_attn_window_fwd(a["q"], a["k"], a["v"], a["out"], a["lse"], a["B"], a["Sq"], a["Sk"], a["H"], a["Hk"], a["D"], *s,
                                      ctypes.cast(ctypes.pointer(w), ctypes.c_void_p), 0.0, a["flags"], a["ws"], a["bytes"], a["counters"], a["n"], None)

    for kw in (dict(B=0), dict(Sq=0), dict(Sk=-1), dict(H=0), dict(Hk=0), dict(Hk=3)):
        assert "must be positive" in _err(lib, call(**kw))
    assert "head dim" in _err(lib, call(D=96), -2)
    for kw in (dict(q=None), dict(k=None), dict(v=None), dict(out=None), dict(lse=None), dict(qs=None), dict(q=4104), dict(k=4104), dict(out=4104)):
        assert "non-null" in _err(lib, call(**kw))
    for name in ("qs", "ks", "vs"):
        assert "multiples of 8" in _err(lib, call(**{name: (512, 129, 64)}))
    for name in ("ks", "vs"):
        for stride in (-128, (1 << 23) + 8):
            assert "token strides" in _err(lib, call(**{name: (512, stride, 64)}))
    for kw in (dict(left=-2), dict(right=-2), dict(frame=0), dict(sinks=-1), dict(q_begin=-2)):
        assert "window" in _err(lib, call(**kw))
    for kw in (dict(Sq=(1 << 29) + 1), dict(Sk=(1 << 29) + 1), dict(frame=(1 << 29) + 1), dict(sinks=(1 << 29) + 1), dict(q_begin=(1 << 29) + 1)):
        assert "2^29" in _err(lib, call(**kw), -2)
    for flags in (1, 3, 4):
        assert "flags" in _err(lib, call(flags=flags))
    for kw in (dict(ws=4104, bytes=1024), dict(ws=4096, bytes=-1)):
        assert "workspace" in _err(lib, call(**kw))
    for kw in (dict(counters=4098, n=4), dict(counters=4096, n=-1)):
        assert "counters" in _err(lib, call(**kw))
    assert "too many" in _err(lib, call(Sq=1 << 29, H=64, Hk=2))


def test_state_arguments():
    lib = _hip.load_library()
    good = State(4096, 4096, 4096, 4, 0)

    def call(n=1, states=good, dst=good, B=1, Sq=4, H=2, D=64):
        arr = (State * max(n, 1))(*([states] * max(n, 1)))
        return lib.dt_merge_block_states(n, ctypes.cast(arr, ctypes.c_void_p), ctypes.cast(ctypes.pointer(dst), ctypes.c_void_p) if dst else None, B, Sq, H, D,
                                         None)

    for n in (0, -1, 65):
        assert "need 1..64" in _err(lib, call(n=n))
    assert "destination" in _err(lib, call(dst=None))
    for kw in (dict(B=0), dict(Sq=0), dict(H=-1)):
        assert "must be positive" in _err(lib, call(**kw))
    assert "head dim" in _err(lib, call(D=32), -2)
    assert "too many rows" in _err(lib, call(B=1 << 20, Sq=1 << 20, H=1 << 20))
    for bad in (State(4096, 4096, 4096, 5, 0), State(4096, 4096, 4096, -1, 0), State(4096, 4096, 4096, 1, 2)):
        assert "bad dtype" in _err(lib, call(states=bad)) and "bad dtype" in _err(lib, call(dst=bad))
    for bad in (State(None, 4096, 4096, 3, 0), State(4104, 4096, 4096, 0, 0), State(4096, None, 4096, 3, 0), State(4096, 4096, None, 1, 0)):
        assert "non-null" in _err(lib, call(states=bad)) and "non-null" in _err(lib, call(dst=bad))


def test_rotary_arguments():
    lib = _hip.load_library()

    def call(n=1, B=1, S=4, D=64, norm=1, positions=4096, n_axes=3, axis=0, rope=1, sections=(), rounding=0, stride=0, turns=True, **row):
        a = {**dict(x=4096, stride_b=512, stride_s=128, stride_h=64, y=4096, weight=None, bias=None, H=2, out_scale=1.0), **row}
        rows = (Rows * 2)(*[Rows(**a)] * 2)
        return lib.dt_qk_norm_rope_axes(ctypes.cast(rows, ctypes.c_void_p), n, B, S, D, norm, 1e-6, positions, stride, n_axes,
                                        (ctypes.c_uint64 * 64)() if turns else None, (ctypes.c_uint8 * 64)(*[axis] * 64), rope,
                                        (ctypes.c_int32 * max(len(sections), 1))(*sections), len(sections), rounding, None)

    for kw in (dict(n=0), dict(n=3), dict(B=0), dict(S=-1)):
        assert "one or two tensors" in _err(lib, call(**kw))
    assert "head dim" in _err(lib, call(D=256), -2)
    for kw in (dict(norm=3), dict(rope=0), dict(rope=3), dict(rounding=1), dict(rounding=2)):
        assert "bad norm" in _err(lib, call(**kw))
    for kw in (dict(positions=None), dict(n_axes=0), dict(n_axes=9), dict(turns=False), dict(stride=-1)):
        assert "axes" in _err(lib, call(**kw))
    assert "axis 3 of 3" in _err(lib, call(axis=3))
    for s in ((32, 16), (60, 4), (64, 64), (-64, 128), (0, 64)):
        assert "section" in _err(lib, call(rope=2, sections=s))
    assert "0..8 sections" in _err(lib, call(rope=2, sections=(8,) * 9))
    for kw in (dict(x=None), dict(y=None), dict(x=4100), dict(stride_s=129), dict(H=0)):
        assert "tensor 0" in _err(lib, call(**kw))
    for scale in (0.0, -1.0, float("inf"), float("nan")):
        assert "out_scale" in _err(lib, call(out_scale=scale))
    assert "16-byte" in _err(lib, call(weight=4100))
    assert "too many rows" in _err(lib, call(B=1 << 16, S=1 << 16))


def test_python_arguments():
    from ditango_amd.core.cache import BlockState, merge_any, proCache
    from ditango_amd.producer import RotaryAxes, prepare_qk_axes
    from ditango_amd.window import window_attention
    q = torch.zeros(1, 4, 2, 64, dtype=torch.bfloat16)
    with pytest.raises(_hip.DitangoHipError, match="must live on the GPU"):
        window_attention(q, q, q)
    for kw in (dict(left=-1), dict(right=1.5), dict(sinks=-1), dict(frame=0), dict(q_begin=-3), dict(left=True), dict(left=1 << 31),
               dict(kv_lens=torch.zeros(1, dtype=torch.int64))):
        with pytest.raises(ValueError):
            window_attention(q, q, q, **kw)
    axes = RotaryAxes(dims=(16, 24, 24))
    pos = torch.zeros(4, 3, dtype=torch.int32)
    with pytest.raises(_hip.DitangoHipError, match="must live on the GPU"):
        prepare_qk_axes(q, q, pos, axes)
    for bad in (pos.long(), pos.float(), pos[:, :2], pos[0], pos.view(1, 1, 4, 3)):
        with pytest.raises(ValueError):
            prepare_qk_axes(q, q, bad, axes)
    with pytest.raises(ValueError):
        prepare_qk_axes(q, q, pos, axes, norm="batch")
    for kw in (dict(dims=(16, 24)), dict(dims=(15, 49)), dict(dims=()), dict(dims=(64,), base=1.0), dict(dims=(64,), base=(2.0, 3.0)), dict(dims=(64,), base=float("inf")),
               dict(dims=(64,), pairing="halves"), dict(dims=(20, 44), pairing="rotate_half"), dict(dims=(64,), halves="row"), dict(dims=(4,) * 16)):
        with pytest.raises(ValueError):
            RotaryAxes(**kw)
    with pytest.raises(ValueError, match="state_format"):
        proCache(8, 0, state_format="fp4")
    with pytest.raises(_hip.DitangoHipError, match="must live on the GPU"):
        merge_any([(q, torch.zeros(1, 2, 4))])
    with pytest.raises(_hip.DitangoHipError, match="must live on the GPU"):
        merge_any([BlockState.empty(q.shape, "int8", "cpu")])
    with pytest.raises(ValueError, match="at least one state"):
        merge_any([])


def test_frequencies_are_whole_fractions_of_a_turn():
    """Each to half a unit of 2^-64 turns, from exact arithmetic; axes share out the pairs in order."""
    import math
    from ditango_amd.producer import RotaryAxes
    axes = RotaryAxes(dims=(16, 56, 56), base=(256.0, 256.0, 10000.0))
    turns, axis = axes.turns
    assert axis == [0] * 8 + [1] * 28 + [2] * 28 and turns[0] == turns[8] == turns[36] \
        == (int("28be60db9391054a7f09d5f47d4d377036d8a5664f10e4107f9458eaf7aef158", 16) + 2 ** 191) >> 192      # 1 / (2 pi) in units of 2^-256
    for t, (i, j) in zip(turns, [(i, j) for i, d in enumerate(axes.dims) for j in range(d // 2)]):
        f = axes.base[i] ** (-2.0 * j / axes.dims[i]) / (2 * math.pi) * 2.0 ** 64
        assert abs(t - f) <= f * 2.0 ** -49


def test_memory_of_a_cached_row():
    from ditango_amd.core.cache import BlockState, proCache
    x = torch.empty(1, 8, 2, 128, dtype=torch.bfloat16)
    assert proCache(8, 0).set_block_size_mb(x) * 2 ** 20 == 16 * 260
    assert proCache(8, 0, state_format="int8").set_block_size_mb(x) * 2 ** 20 == 16 * 136
    assert BlockState.empty(x.shape, "e4m3", "cpu").nbytes == 16 * 136


def test_grids_beyond_the_launchers_are_refused():
    """A grid holds fewer than 2^32 lanes: more rows than that are refused before the launch, not by it."""
    lib = _hip.load_library()
    strides = (ctypes.c_int64 * 3)(0, 128, 64)
    w = Window(1, 0, 1, 0, -1, None)
    for B, Sq in ((1 << 23, 1), (1 << 13, 1 << 18)):
        assert "too many query rows" in _err(lib, lib.dt_attn_window_fwd(4096, 4096, 4096, 4096, 4096, B, Sq, 4, 2, 2, 64, strides, strides, strides,
                                                                         ctypes.cast(ctypes.pointer(w), ctypes.c_void_p), 0.0, 0, None, 0, None, 0, None))
    rows = (Rows * 1)(Rows(4096, 0, 0, 0, 4096, None, None, 1, 1.0))
    for D, S in ((64, 1 << 15), (128, 1 << 14)):
        assert "too many rows" in _err(lib, lib.dt_qk_norm_rope_axes(ctypes.cast(rows, ctypes.c_void_p), 1, 1 << 14, S, D, 1, 1e-6, 4096, 0, 3,
                                                                     (ctypes.c_uint64 * 64)(), (ctypes.c_uint8 * 64)(), 1, None, 0, 0, None))
