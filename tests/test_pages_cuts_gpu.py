"""How paged attention cuts the keys of its tiles of 256 rows, each way with cases that take it: parts of one length that meet in groups, a last round in parts behind one
or two whole ones, more requests than a wavefront has lanes; with room for all parts, for some and for none; captured, on several streams, from several threads.

Which way a launch goes is seen from what it leaves in a workspace of the test's own: the slots of its parts.  ``_room`` knows where they lie, which the
slots bear out (a part's sums and its maxima lie in different places and have to agree)."""
import ctypes
import threading

import pytest
import torch

from tests.test_long_video_refusals import Window
from tests.test_paged_attention_gpu import _check, _i32, _setup
from tests.test_pages_refusals import I64x3, PagePool

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
WORDS = 1 << 14
FP16 = 2               # DT_ATTN_FP16
GUARD = 1 << 16       # bytes behind the workspace


def _room(T, H, Hk, D, B, most, most_len, nbytes, words):
    """Slots that a launch has for parts of 256 rows and of few, the latter first in the workspace."""
    cus = torch.cuda.get_device_properties(0).multi_processor_count
    group = H // Hk
    rows, requests = T * group, min(B, T)
    few = 96 if D == 64 else 64
    as_few = Hk * (rows // 32 + requests)
    assert min(most * group, rows) > (few if as_few > cus else 96), "few rows only"
    uncut = Hk * (rows // 256 + min(requests, rows // (few + 1)) + min(rows // 32 + requests, requests * (few // 32)))
    slots = cus * (2 if D == 64 else 1)
    groups = uncut + min(3 * slots // 2, uncut * min(most_len // 512, 63))
    if B <= 64 and as_few <= slots:
        groups = max(groups, as_few + slots)
    bytes_of = [rows * (D + 2) * 4 for rows in (256, 32)]
    n_few = min(nbytes // 2 // bytes_of[1], words // 2, groups)
    return min((nbytes - n_few * bytes_of[1]) // bytes_of[0], (words - n_few) // 8, groups), n_few


class Launch:
    """``dt_attn_pages_fwd`` with a workspace and counters of its own."""

    def __init__(self, hip, nbytes=None, words=WORDS):
        self.lib = hip.load_library()
        self.nbytes = int(self.lib.dt_attn_workspace_bytes()) if nbytes is None else nbytes
        self.words = words
        self.workspace = torch.empty(self.nbytes + GUARD, dtype=torch.uint8, device=DEV)
        self.counters = torch.zeros(words + 16, dtype=torch.int32, device=DEV)
        self.counters[words:] = 7

    def __call__(self, q, kp, vp, tables, lens, cu, most, left=-1, right=0, frame=1, sinks=0):
        """(out, lse, slots of parts of 256 rows, ... of few)"""
        T, H, D = q.shape
        Hk = kp.shape[2]
        tables, lens, cu = _i32(tables), _i32(lens), _i32(cu)
        out, lse = torch.full_like(q, 3.0), torch.full((H, T), 3.0, device=DEV)
        self.workspace.fill_(255)
        strides = [I64x3(*x.stride()[:3]) for x in (kp, vp)]
        pool, w = PagePool(kp.data_ptr(), vp.data_ptr(), *strides, kp.shape[0], kp.shape[1]), Window(left, right, frame, sinks, -1, None)
        ref = lambda x: ctypes.cast(ctypes.pointer(x), ctypes.c_void_p)
        rc = self.lib.dt_attn_pages_fwd(q.data_ptr(), (ctypes.c_int64 * 2)(*q.stride()[:2]), out.data_ptr(), lse.data_ptr(), T, H, Hk, D, ref(pool), tables.data_ptr(),
                                        tables.stride(0), tables.shape[1], lens.shape[0], lens.data_ptr(), cu.data_ptr(), most, ref(w), 0.0,
                                        FP16 if q.dtype is torch.float16 else 0, self.workspace.data_ptr() if self.nbytes else None, self.nbytes,
                                        self.counters.data_ptr() if self.words else None, self.words, torch.cuda.current_stream().cuda_stream)
        assert rc == 0, self.lib.dt_last_error()
        torch.cuda.synchronize()
        assert not bool(self.counters[:self.words].any()) and bool((self.counters[self.words:] == 7).all())
        assert bool((self.workspace[self.nbytes:] == 255).all())
        n_big, n_few = _room(T, H, Hk, D, lens.shape[0], most, tables.shape[1] * kp.shape[1], self.nbytes if self.words else 0, self.words if self.nbytes else 0)
        words = self.workspace[:self.nbytes // 4 * 4].view(torch.int32)
        slots, at = [], 0
        for n, rows in ((n_few, 32), (n_big, 256)):
            sums = words[at:at + n * rows * D].view(n, rows * D)
            maxima = words[at + n * rows * D:at + n * rows * (D + 2)].view(n, rows * 2)
            at += n * rows * (D + 2)
            used = (maxima != -1).any(1)
            assert torch.equal(used, (sums != -1).any(1))
            slots.append(used.nonzero()[:, 0].tolist())
        assert bool((words[at:] == -1).all())
        return out, lse, slots[1], slots[0]


# lens, new, H, Hk, heads of, slots of parts of 256 rows: (items that are cut, at least so many parts each)
TOKENS = [100 + b for b in range(65)]
CUTS = {
    "few items of many requests, D=64": ([38000] + TOKENS, [617] + [1] * 65, 2, 2, 64, (6, 9)),
    "few items of many requests, D=128": ([38000] + TOKENS, [617] + [1] * 65, 2, 2, 128, (6, 9)),
    "one item a key head, D=64": ([20000] + TOKENS, [255] + [1] * 65, 4, 1, 64, (4, 9)),
    "items of 8 heads beside tokens": ([6000, 700, 5000, 44], [1000, 1, 3, 1], 8, 8, 128, (32, 4)),
    "60 items, D=64": ([9000, 60], [300, 1], 60, 60, 64, (60, 4)),
    "four items behind a round, D=64": ([6000] * 3 + [300] * 2, [1000] * 3 + [1] * 2, 43, 43, 64, (4, 9)),
    "eight items behind a round, D=64": ([6000, 300, 300], [1000, 1, 1], 130, 130, 64, (8, 9)),
    "four items behind a round, D=128": ([9000] * 4 + [300] * 2, [1100] * 4 + [1] * 2, 13, 13, 128, (4, 9)),
    "four items behind two rounds, D=128": ([6000] * 3 + [300] * 2, [1000] * 3 + [1] * 2, 43, 43, 128, (4, 9)),
    "four items behind a round, 70 requests, D=128": ([3000] * 65 + [300] * 5, [230] * 65 + [1] * 5, 4, 4, 128, (4, 9)),
    "eight items behind a round, 70 requests, D=64": ([3000] * 65 + [300] * 5, [230] * 65 + [1] * 5, 8, 8, 64, (8, 9)),
}


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("name", CUTS)
def test_every_cut(hip, name, dtype):
    """Within the bound, the same bits each time, undefined values with the rows that see them."""
    lens, new, H, Hk, D, (items, ways) = CUTS[name]
    q, kp, vp, tables, cu = _setup(lens, new, H, Hk, D, 64, dtype, junk=float("inf"), seed=len(name))
    launch = Launch(hip)
    out, lse, big, few = launch(q, kp, vp, tables, lens, cu, max(new))
    assert len(big) % items == 0 and len(big) >= items * ways, (len(big), len(few))
    _check(out, lse, q, kp, vp, tables, lens, cu, right=0)
    for _ in range(3):
        again = launch(q, kp, vp, tables, lens, cu, max(new))
        assert torch.equal(again[0], out) and torch.equal(again[1], lse) and again[2:] == (big, few)
    from ditango_amd.pages import paged_attention
    own = paged_attention(q, kp, vp, _i32(tables), _i32(lens), _i32(cu), max_seqlen_q=max(new), right=0)
    assert torch.equal(own[0], out) and torch.equal(own[1], lse)
    # an infinite value that all rows see, one that half of the first request's do, and one of a request behind it
    vp[tables[0][0], 5, 0, 1] = -float("inf")
    j = lens[0] - new[0] // 2
    vp[tables[0][j // 64], j % 64, Hk - 1, D - 3] = float("inf")
    j = lens[-1] - 1
    vp[tables[-1][j // 64], j % 64, Hk // 2, 2] = float("inf")
    out, lse, big, few = launch(q, kp, vp, tables, lens, cu, max(new))
    assert len(big) >= items * ways
    _check(out, lse, q, kp, vp, tables, lens, cu, right=0)
    # ... and a key, for the last third of the first request's rows
    j = lens[0] - new[0] // 3
    kp[tables[0][j // 64], j % 64, 0, 7] = float("nan")
    out, lse, big, few = launch(q, kp, vp, tables, lens, cu, max(new))
    _check(out, lse, q, kp, vp, tables, lens, cu, right=0)


def _beside(seed, dtype=torch.bfloat16):
    lens, new = [6000, 700, 5000, 44], [1000, 1, 3, 1]
    return (*_setup(lens, new, 8, 8, 128, 64, dtype, seed=seed), lens, new)


def test_room_for_some_parts(hip):
    """32 items of 256 rows: without room for a part of each and one more they are not cut; with little they are cut less."""
    q, kp, vp, tables, cu, lens, new = _beside(1)
    whole = int(hip.load_library().dt_attn_workspace_bytes())
    some = 504 * 32 * 130 * 4 + 110 * 256 * 130 * 4          # 504 slots of few rows, 110 of 256
    for nbytes, words, parts in ((0, 0, 0), (whole, 0, 0), (0, WORDS, 0), (whole, 16, 0), (whole, 800, 0), (whole, 1400, 64), (some, WORDS, 64), (8 << 20, WORDS, 0),
                                 (whole, WORDS, 256)):
        launch = Launch(hip, nbytes, words)
        out, lse, big, few = launch(q, kp, vp, tables, lens, cu, max(new))
        assert len(big) == parts, (nbytes, words, len(big))
        _check(out, lse, q, kp, vp, tables, lens, cu, right=0)


def _attend(case, **w):
    from ditango_amd.pages import paged_attention
    q, kp, vp, tables, cu, lens, new = case
    return paged_attention(q, kp, vp, tables, lens, cu, max_seqlen_q=1000, right=0, **w)


def _three():
    cases = [_beside(s, dtype) for s, dtype in ((2, torch.bfloat16), (3, torch.float16), (4, torch.bfloat16))]
    on_gpu = [(q, kp, vp, _i32(tables), _i32(cu), _i32(lens), new) for q, kp, vp, tables, cu, lens, new in cases]
    want = [_attend(c) for c in on_gpu]
    torch.cuda.synchronize()
    for (out, lse), (q, kp, vp, tables, cu, lens, new) in zip(want, cases):
        _check(out, lse, q, kp, vp, tables, lens, cu, right=0)
    return on_gpu, want


def test_two_graphs_and_eager_launches(hip):
    cases, want = _three()
    assert len(Launch(hip)(*cases[0][:3], cases[0][3].tolist(), cases[0][5].tolist(), cases[0][4].tolist(), 1000)[2]) == 256      # tiles of 256 rows, in parts
    graphs, outs = [], []
    for c in cases[:2]:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(_attend(c))
        graphs.append(graph)
    streams = [torch.cuda.Stream() for _ in range(2)]
    for turn in range(5):
        for t in outs[0] + outs[1]:
            t.zero_()
        torch.cuda.synchronize()
        for graph, stream in zip(graphs if turn % 2 else graphs[::-1], streams):
            with torch.cuda.stream(stream):
                graph.replay()
        eager = _attend(cases[2])
        torch.cuda.synchronize()
        for got, ref in zip(outs + [eager], want):
            assert torch.equal(got[0], ref[0]) and torch.equal(got[1], ref[1])


def test_threads_and_streams(hip):
    cases, want = _three()
    bad = []

    def work(i, own_stream):
        stream = torch.cuda.Stream() if own_stream else torch.cuda.default_stream()
        with torch.cuda.stream(stream):
            for _ in range(15):
                out, lse = _attend(cases[i])
                stream.synchronize()
                if not (torch.equal(out, want[i][0]) and torch.equal(lse, want[i][1])):
                    bad.append(i)

    for own in (True, False):
        threads = [threading.Thread(target=work, args=(i, own)) for i in range(3)]
        for t in threads:
            t.start()
        for t in threads:
            t.join()
    assert not bad
    torch.cuda.synchronize()
    assert all(not bool(c.any()) for c in hip._counters.values())
