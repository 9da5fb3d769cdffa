"""What the operators of a cache of pages refuse, on the host, before any launch; the oracle's plan has what a plan has to have."""
import ctypes
import random

import pytest
import torch

from ditango_amd import _hip
from oracle import pages as P
from tests.test_long_video_refusals import Rows, Window, _err

I64x3 = ctypes.c_int64 * 3


class PagePool(ctypes.Structure):
    _fields_ = [("k", ctypes.c_void_p), ("v", ctypes.c_void_p), ("k_strides", I64x3), ("v_strides", I64x3), ("n_pages", ctypes.c_int32),
                ("page_size", ctypes.c_int32)]


def _pool(k=4096, v=4096, ks=(2048, 128, 64), vs=(2048, 128, 64), n_pages=4, page_size=16):
    return PagePool(k, v, I64x3(*ks), I64x3(*vs), n_pages, page_size)


def _ref(x):
    return None if x is None else ctypes.cast(ctypes.pointer(x), ctypes.c_void_p)


def _pair(s):
    return None if s is None else (ctypes.c_int64 * 2)(*s)


BAD_POOLS = [(dict(n_pages=-1), "multiple of 16", -1), (dict(page_size=0), "multiple of 16", -1), (dict(page_size=24), "multiple of 16", -1),
             (dict(page_size=-16), "multiple of 16", -1), (dict(n_pages=1 << 27), "2^31", -2), (dict(k=None), "non-null", -1), (dict(v=4104), "aligned", -1),
             (dict(ks=(2048, 129, 64)), "multiples of 8", -1), (dict(vs=(2049, 128, 64)), "multiples of 8", -1), (dict(vs=(2048, 128, 60)), "multiples of 8", -1),
             (dict(ks=(2048, -128, 64)), "token strides", -1), (dict(vs=(2048, (1 << 23) + 8, 64)), "token strides", -1)]


def test_plan_arguments():
    lib = _hip.load_library()
    ok = dict(tables=4096, stride=8, width=8, lens=4096, new=4096, B=2, n_pages=16, page=16, n=4, lens_out=4096, cu=4096, slots=4096, served=4096)

    def call(**kw):
        a = {**ok, **kw}
        return lib.dt_plan_pages(a["tables"], a["stride"], a["width"], a["lens"], a["new"], a["B"], a["n_pages"], a["page"], a["n"], a["lens_out"], a["cu"],
                                 a["slots"], a["served"], None)

    for kw in (dict(B=0), dict(B=-1), dict(width=-1), dict(n_pages=-1), dict(n=-1), dict(page=0), dict(page=8), dict(page=-16), dict(page=40)):
        assert "must be positive" in _err(lib, call(**kw))
    for kw in (dict(tables=None), dict(lens=None), dict(new=None), dict(lens_out=None), dict(cu=None), dict(slots=None), dict(served=None), dict(stride=7)):
        assert "non-null" in _err(lib, call(**kw))
    for kw in (dict(B=2049), dict(n_pages=(1 << 20) + 1), dict(width=1 << 26, stride=1 << 26), dict(n=(1 << 30) + 1), dict(n_pages=1 << 20, page=2048)):
        assert "not supported" in _err(lib, call(**kw), -2)


def test_append_arguments():
    lib = _hip.load_library()
    ok = dict(k=4096, v=4096, ks=(128, 64), vs=(128, 64), T=4, Hk=2, D=64, pool=_pool(), slots=4096)

    def call(**kw):
        a = {**ok, **kw}
        return lib.dt_append_pages(a["k"], a["v"], _pair(a["ks"]), _pair(a["vs"]), a["T"], a["Hk"], a["D"], _ref(a["pool"]), a["slots"], None)

    for kw in (dict(T=0), dict(T=-1), dict(Hk=0)):
        assert "must be positive" in _err(lib, call(**kw))
    assert "head dim" in _err(lib, call(D=96), -2)
    for kw in (dict(k=None), dict(v=None), dict(ks=None), dict(vs=None), dict(slots=None), dict(k=4100), dict(v=4104)):
        assert "non-null" in _err(lib, call(**kw))
    for kw in (dict(ks=(129, 64)), dict(vs=(128, 4))):
        assert "multiples of 8" in _err(lib, call(**kw))
    assert "pages must be given" in _err(lib, call(pool=None))
    for kw, text, code in BAD_POOLS:
        assert text in _err(lib, call(pool=_pool(**kw)), code)
    assert "too many rows" in _err(lib, call(T=1 << 28, Hk=2))


def test_prepare_arguments():
    lib = _hip.load_library()

    def call(T=4, D=64, norm=1, positions=4096, n_axes=3, axis=0, rope=1, sections=(), rounding=0, turns=True, v=4096, vs=(128, 64), slots=4096, pool=_pool(),
             rows=True, second=None, **row):
        a = {**dict(x=4096, stride_b=512, stride_s=128, stride_h=64, y=4096, weight=None, bias=None, H=2, out_scale=1.0), **row}
        r = (Rows * 2)(Rows(**a), Rows(**{**a, "y": None, **(second or {})}))
        return lib.dt_prepare_pages(ctypes.cast(r, ctypes.c_void_p) if rows else None, v, _pair(vs), T, D, norm, 1e-6, positions, n_axes,
                                    (ctypes.c_uint64 * 64)() if turns else None, (ctypes.c_uint8 * 64)(*[axis] * 64), rope,
                                    (ctypes.c_int32 * max(len(sections), 1))(*sections), len(sections), rounding, _ref(pool), slots, None)

    for kw in (dict(T=0), dict(T=-4), dict(rows=False)):
        assert "need q, k" in _err(lib, call(**kw))
    assert "head dim" in _err(lib, call(D=256), -2)
    assert "pages must be given" in _err(lib, call(pool=None))
    for kw, text, code in BAD_POOLS:
        assert text in _err(lib, call(pool=_pool(**kw)), code)
    for kw in (dict(norm=3), dict(rope=0), dict(rounding=1)):
        assert "bad norm" in _err(lib, call(**kw))
    for kw in (dict(positions=None), dict(n_axes=0), dict(n_axes=9), dict(turns=False)):
        assert "axes" in _err(lib, call(**kw))
    assert "axis 3 of 3" in _err(lib, call(axis=3))
    assert "section" in _err(lib, call(rope=2, sections=(60, 4)))
    for kw in (dict(x=None), dict(y=None), dict(x=4100), dict(stride_s=129), dict(H=0)):
        assert "tensor 0" in _err(lib, call(**kw))
    assert "tensor 1" in _err(lib, call(second=dict(x=None)))
    assert "out_scale" in _err(lib, call(out_scale=0.0))
    assert "16-byte" in _err(lib, call(weight=4100))
    for kw in (dict(v=None), dict(v=4104), dict(vs=None), dict(slots=None), dict(vs=(129, 64)), dict(vs=(128, 63))):
        assert "v, its strides" in _err(lib, call(**kw))
    assert "too many rows" in _err(lib, call(T=1 << 30, H=8))


def test_attention_arguments():
    lib = _hip.load_library()
    ok = dict(q=4096, qs=(256, 64), out=4096, lse=4096, T=4, H=4, Hk=2, D=64, pool=_pool(), tables=4096, stride=8, width=8, B=2, lens=4096, cu=4096, most=4,
              left=1, right=0, frame=1, sinks=0, window=True, flags=0, ws=None, bytes=0, counters=None, n=0)

    def call(**kw):
        a = {**ok, **kw}
        w = Window(a["left"], a["right"], a["frame"], a["sinks"], -1, None)
        return lib.dt_attn_pages_fwd(a["q"], _pair(a["qs"]), a["out"], a["lse"], a["T"], a["H"], a["Hk"], a["D"], _ref(a["pool"]), a["tables"], a["stride"],
                                     a["width"], a["B"], a["lens"], a["cu"], a["most"], _ref(w) if a["window"] else None, 0.0, a["flags"], a["ws"], a["bytes"],
                                     a["counters"], a["n"], None)

    for kw in (dict(T=0), dict(B=0), dict(H=0), dict(Hk=0), dict(Hk=3), dict(T=-1)):
        assert "must be positive" in _err(lib, call(**kw))
    assert "head dim" in _err(lib, call(D=96), -2)
    assert "pages must be given" in _err(lib, call(pool=None))
    for kw, text, code in BAD_POOLS:
        assert text in _err(lib, call(pool=_pool(**kw)), code)
    for kw in (dict(q=None), dict(out=None), dict(lse=None), dict(qs=None), dict(q=4104), dict(out=4104), dict(lens=None), dict(cu=None), dict(window=False),
               dict(tables=None)):
        assert "non-null" in _err(lib, call(**kw))
    for kw in (dict(qs=(257, 64)), dict(qs=(256, 4))):
        assert "multiples of 8" in _err(lib, call(**kw))
    for kw in (dict(width=-1), dict(stride=7)):
        assert "width" in _err(lib, call(**kw))
    for kw in (dict(left=-2), dict(right=-2), dict(frame=0), dict(sinks=-1)):
        assert "window" in _err(lib, call(**kw))
    for kw in (dict(width=1 << 26, stride=1 << 26), dict(T=(1 << 29) + 1), dict(frame=(1 << 29) + 1), dict(sinks=(1 << 29) + 1)):
        assert "2^29" in _err(lib, call(**kw), -2)
    for flags in (1, 3, 4):
        assert "flags" in _err(lib, call(flags=flags))
    for kw in (dict(ws=4104, bytes=1024), dict(ws=4096, bytes=-1)):
        assert "workspace" in _err(lib, call(**kw))
    for kw in (dict(counters=4098, n=4), dict(counters=4096, n=-1)):
        assert "counters" in _err(lib, call(**kw))
    assert "too many" in _err(lib, call(T=1 << 29, H=64, Hk=2))


def test_python_arguments():
    from ditango_amd.pages import append_pages, paged_attention, plan_pages, prepare_qkv_pages
    from ditango_amd.producer import RotaryAxes
    q = torch.zeros(4, 2, 64, dtype=torch.bfloat16)
    pages = torch.zeros(2, 16, 2, 64, dtype=torch.bfloat16)
    i32 = lambda *s: torch.zeros(*s, dtype=torch.int32)
    slots, pos, axes = torch.zeros(4, dtype=torch.int64), i32(4, 3), RotaryAxes(dims=(16, 24, 24))
    on_gpu = pytest.raises(_hip.DitangoHipError, match="must live on the GPU")
    with on_gpu:
        plan_pages(i32(1, 4), i32(1), i32(1), 4, n_pages=2, page_size=16)
    with on_gpu:
        append_pages(q, q, pages, pages, slots)
    with on_gpu:
        prepare_qkv_pages(q, q, q, pos, axes, pages, pages, slots)
    with on_gpu:
        paged_attention(q, pages, pages, i32(1, 2), i32(1), i32(2))
    for bad in ((i32(1, 4).long(), i32(1), i32(1)), (i32(1, 4), i32(1).long(), i32(1)), (i32(1, 4), i32(1), i32(1).float())):
        with pytest.raises(ValueError, match="int32"):
            plan_pages(*bad, 4, n_pages=2, page_size=16)
    for bad in ((i32(1, 2).long(), i32(1), i32(2)), (i32(1, 2), i32(1).long(), i32(2)), (i32(1, 2), i32(1), i32(2).long())):
        with pytest.raises(ValueError, match="int32"):
            paged_attention(q, pages, pages, *bad)
    for kw in (dict(left=-1), dict(right=1.5), dict(sinks=-1), dict(frame=0), dict(left=True), dict(max_seqlen_q=-4), dict(max_seqlen_q=1 << 31)):
        with pytest.raises(ValueError):
            paged_attention(q, pages, pages, i32(1, 2), i32(1), i32(2), **kw)
    for bad in (pos.long(), pos[:, :2], pos[0], pos[None]):
        with pytest.raises(ValueError):
            prepare_qkv_pages(q, q, q, bad, axes, pages, pages, slots)
    with pytest.raises(ValueError, match="norm"):
        prepare_qkv_pages(q, q, q, pos, axes, pages, pages, slots, norm="batch")


def test_the_oracles_plan_gives_no_page_twice():
    rng = random.Random(3)
    for _ in range(200):
        page, width, n_pages, B = 16, rng.randint(1, 6), rng.randint(0, 20), rng.randint(1, 6)
        tables, lens = [[-1] * width for _ in range(B)], [0] * B
        for _ in range(5):
            new = [rng.randint(0, 40) for _ in range(B)]
            before = lens
            tables, lens, cu, slots, served = P.plan(tables, lens, new, sum(new), n_pages, page)
            held = [p for row, n in zip(tables, lens) for p in row[:-(-n // page)]]
            assert len(set(held)) == len(held) and all(0 <= p < n_pages for p in held)
            used = [s for s in slots if s >= 0]
            assert len(set(used)) == len(used) == sum(lens) - sum(before)
            for b in range(B):
                assert lens[b] == before[b] + (new[b] if served[b] else 0)
            gone = rng.randrange(B)
            lens[gone] = 0
