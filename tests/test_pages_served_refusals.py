"""What paged attention refuses of ``served``, on the host."""
import pytest
import torch

from ditango_amd import _hip
from tests.test_long_video_refusals import Window, _err
from tests.test_pages_refusals import _pair, _pool, _ref


def test_python_arguments():
    from ditango_amd.pages import paged_attention
    q, pages = torch.zeros(4, 2, 64, dtype=torch.bfloat16), torch.zeros(2, 16, 2, 64, dtype=torch.bfloat16)
    i32 = lambda *s: torch.zeros(*s, dtype=torch.int32)
    for bad in (i32(1), torch.zeros(1), torch.zeros(1, dtype=torch.uint8)):
        with pytest.raises(ValueError, match="bool"):
            paged_attention(q, pages, pages, i32(1, 2), i32(1), i32(2), served=bad)


def test_the_c_entry_refuses_what_the_other_one_does():
    lib = _hip.load_library()
    ok = dict(q=4096, T=4, D=64, lens=4096, cu=4096, flags=0, stride=8)

    def call(**kw):
        a = {**ok, **kw}
        w = Window(1, 0, 1, 0, -1, None)
        return lib.dt_attn_pages_served_fwd(a["q"], _pair((256, 64)), 4096, 4096, a["T"], 4, 2, a["D"], _ref(_pool()), 4096, a["stride"], 8, 2, a["lens"], None, a["cu"],
                                            4, _ref(w), 0.0, a["flags"], None, 0, None, 0, None)

    assert "must be positive" in _err(lib, call(T=0))
    assert "head dim" in _err(lib, call(D=96), -2)
    for kw in (dict(q=None), dict(lens=None), dict(cu=None)):
        assert "non-null" in _err(lib, call(**kw))
    assert "width" in _err(lib, call(stride=7))
    assert "flags" in _err(lib, call(flags=1))
