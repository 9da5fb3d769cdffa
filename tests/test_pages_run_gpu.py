"""The operators of a cache of pages as a server uses them, step after step: plan, keys and values into their pages, attention; eager and captured, on several
streams and threads.  A request's results are those of ``window_attention`` on a cache of its own, within the bounds of both."""
import random
import threading

import pytest
import torch

from oracle import pages as P
from tests.test_paged_attention_gpu import _check

pytestmark = pytest.mark.gpu

DEV = "cuda:0"


def _i32(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


def _step(q, k, v, positions, axes, kp, vp, tables, lens, new, window, in_place=False, most=None):
    from ditango_amd.pages import paged_attention, plan_pages, prepare_qkv_pages
    plan = plan_pages(tables, lens, new, q.shape[0], n_pages=kp.shape[0], page_size=kp.shape[1], in_place=in_place)
    q = prepare_qkv_pages(q, k, v, positions, axes, kp, vp, plan.slots, norm="rms")
    return plan, q, paged_attention(q, kp, vp, tables, plan.lens, plan.cu_seqlens, max_seqlen_q=most, **window)


@pytest.mark.parametrize("D, H, Hk, page, dtype", [(128, 4, 2, 16, torch.bfloat16), (64, 6, 6, 48, torch.float16), (128, 3, 3, 128, torch.bfloat16)])
def test_rollouts_step_by_step(hip, D, H, Hk, page, dtype):
    """Requests that come, grow at their own pace and go; pages of those that have gone are used again."""
    from ditango_amd.producer import RotaryAxes, prepare_qk_axes
    rng = random.Random(D + H)
    g = torch.Generator(device=DEV).manual_seed(page)
    axes = RotaryAxes(dims=(16, 56, 56), base=256.0) if D == 128 else RotaryAxes(dims=(16, 24, 24))
    B, width = 5, 900 // page + 1
    kp, vp = (torch.full((3 * width, page, Hk, D), float("nan"), device=DEV, dtype=dtype) for _ in range(2))
    tables, lens = torch.full((B, width), -1, dtype=torch.int32, device=DEV), _i32([0] * B)
    caches = [[torch.empty(0, Hk, D, device=DEV, dtype=dtype) for _ in range(2)] for _ in range(B)]
    for step in range(12):
        gone = rng.randrange(B)
        if step % 3 == 2:
            lens[gone] = 0
            caches[gone] = [c[:0] for c in caches[gone]]
        new = [rng.choice([0, 1, 1, rng.randint(2, 40), rng.randint(100, 260)]) for _ in range(B)]
        T = sum(new) + rng.choice([0, 9])
        qkv = torch.randn(max(T, 1), H + 2 * Hk, D, generator=g, device=DEV).to(dtype)
        q, k, v = qkv[:, :H], qkv[:, H:H + Hk], qkv[:, H + Hk:]
        pos = torch.randint(0, 500, (q.shape[0], 3), generator=g, device=DEV, dtype=torch.int32)
        window = rng.choice([dict(right=0), dict(left=60, right=0, sinks=9), dict(left=2, right=0, frame=50, sinks=16)])
        before = lens.tolist()
        want = P.plan(tables.tolist(), before, new, q.shape[0], kp.shape[0], page)
        plan, q, (out, lse) = _step(q, k, v, pos, axes, kp, vp, tables, lens, _i32(new), window)
        torch.cuda.synchronize()
        assert [tables.tolist(), plan.lens.tolist(), plan.cu_seqlens.tolist(), plan.slots.tolist(), plan.served.tolist()] == list(want)
        lens = plan.lens
        # what the pages hold is what each request has got
        want_q, want_k = prepare_qk_axes(qkv[None, :, :H], k[None], pos, axes, norm="rms")
        assert torch.equal(q, want_q[0])
        for b in range(B):
            lo, hi = plan.cu_seqlens[b:b + 2].tolist()
            if plan.served[b]:
                caches[b] = [torch.cat((c, x[lo:hi])) for c, x in zip(caches[b], (want_k[0], v))]
            for c, pages in zip(caches[b], (kp, vp)):
                assert torch.equal(P.gathered(pages, tables[b].tolist(), lens[b].item()), c)
        clean = [torch.where(torch.isnan(x), torch.zeros_like(x), x) for x in (kp, vp)]
        _check(out, lse, q, *clean, tables.tolist(), lens.tolist(), plan.cu_seqlens.tolist(), **window)


def test_the_same_as_a_cache_of_its_own(hip):
    """paged_attention beside window_attention on the same tokens: both within their bound of the same numbers, and states that merge."""
    from ditango_amd.core.cache import merge_any
    from ditango_amd.pages import append_pages, paged_attention, plan_pages
    from ditango_amd.window import window_attention
    g = torch.Generator(device=DEV).manual_seed(0)
    for D, H, Hk, n, L in ((128, 4, 4, 300, 1000), (64, 8, 2, 1, 2000)):
        k, v = (torch.randn(2, L, Hk, D, generator=g, device=DEV).bfloat16() for _ in range(2))
        q = torch.randn(2, n, H, D, generator=g, device=DEV).bfloat16()
        kp, vp = (torch.zeros(2 * (L // 64 + 1), 64, Hk, D, device=DEV, dtype=torch.bfloat16) for _ in range(2))
        tables = torch.full((2, L // 64 + 1), -1, dtype=torch.int32, device=DEV)
        plan = plan_pages(tables, _i32([0, 0]), _i32([L, L]), 2 * L, n_pages=kp.shape[0], page_size=64)
        append_pages(k.flatten(0, 1), v.flatten(0, 1), kp, vp, plan.slots)
        w = dict(left=500, right=0, sinks=20)
        out, lse = paged_attention(q.flatten(0, 1), kp, vp, tables, plan.lens, _i32([0, n, 2 * n]), **w)
        o, l = window_attention(q, k, v, **w)
        scale = float(o.float().abs().max())
        assert float((out.view_as(o).float() - o.float()).abs().max()) <= 2.0 ** -6 * scale
        assert float((lse.view(H, 2, n).transpose(0, 1) - l).abs().max()) <= 1e-3
        # a packed state is a state of one sample: merged with itself it stays what it is, half the weight each
        twice, lse2 = merge_any([(out[None], lse[None]), (out[None], lse[None])], dst_dtype=torch.float32)
        assert float((twice[0] - out.float()).abs().max()) <= 1e-6 * scale and float((lse2[0] - lse - 0.6931472).abs().max()) <= 1e-5


def _server(D=128, H=4, Hk=2, page=16, dtype=torch.bfloat16, B=3, seed=0, first=(200, 3, 77)):
    from ditango_amd.producer import RotaryAxes
    g = torch.Generator(device=DEV).manual_seed(seed)
    s = dict(axes=RotaryAxes(dims=(16, 56, 56), base=256.0) if D == 128 else RotaryAxes(dims=(16, 24, 24)), H=H, Hk=Hk, D=D, g=g, dtype=dtype, B=B)
    s["kp"], s["vp"] = (torch.randn(200, page, Hk, D, generator=g, device=DEV).to(dtype) for _ in range(2))
    width = 60
    s["tables"] = torch.full((B, width), -1, dtype=torch.int32, device=DEV)
    ids = torch.randperm(200, generator=g, device=DEV).to(torch.int32)
    for b, n in enumerate(first):
        h = -(-n // page)
        s["tables"][b, :h] = ids[:h]
        ids = ids[h:]
    s["lens"] = _i32(list(first))
    return s


def _inputs(s, T):
    qkv = torch.randn(T, s["H"] + 2 * s["Hk"], s["D"], generator=s["g"], device=DEV).to(s["dtype"])
    return qkv, torch.randint(0, 300, (T, 3), generator=s["g"], device=DEV, dtype=torch.int32)


def _run_step(s, qkv, pos, new, in_place, **kw):
    H, Hk = s["H"], s["Hk"]
    return _step(qkv[:, :H], qkv[:, H:H + Hk], qkv[:, H + Hk:], pos, s["axes"], s["kp"], s["vp"], s["tables"], s["lens"], new, dict(right=0), in_place, **kw)


@pytest.mark.parametrize("new", [[1, 1, 1], [40, 1, 130]])
@pytest.mark.parametrize("D", [64, 128])
def test_captured_steps_follow_the_lengths(hip, D, new):
    """A whole step in a graph, replayed: lengths, tables and caches grow, eager work of the same kind in between."""
    s, e = _server(D=D), _server(D=D)
    T = sum(new) + 5
    qkv, pos = _inputs(s, T)
    counts = _i32(new)
    warm = _server(D=D, seed=3)
    _run_step(warm, qkv, pos, counts, True, most=max(new))
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        plan, q, (out, lse) = _run_step(s, qkv, pos, counts, True, most=max(new))
    state = s["lens"].clone()
    assert state.tolist() == e["lens"].tolist()                   # (nothing ran under capture)
    for turn in range(4):
        x, p = _inputs(s, T)
        c = [max(0, n - turn) for n in new]
        qkv.copy_(x)
        pos.copy_(p)
        counts.copy_(_i32(c))
        graph.replay()
        eplan, eq, (eout, else_) = _run_step(e, x, p, _i32(c), True, most=max(new))
        torch.cuda.synchronize()
        for a, b in ((s["lens"], e["lens"]), (s["tables"], e["tables"]), (plan.slots, eplan.slots), (plan.cu_seqlens, eplan.cu_seqlens), (plan.served, eplan.served),
                     (s["kp"], e["kp"]), (s["vp"], e["vp"]), (q, eq), (out, eout), (lse, else_)):
            assert torch.equal(a, b)
    assert s["lens"].tolist() == [n + 4 * m - sum(min(m, t) for t in range(4)) for n, m in zip((200, 3, 77), new)]


def _attend(s, q, lens, cu, **w):
    from ditango_amd.pages import paged_attention
    return paged_attention(q, s["kp"], s["vp"], s["tables"], lens, cu, **w)


def _long(seed, new=(1, 2), lens=(3000, 2100)):
    """Requests whose keys are cut into parts."""
    g = torch.Generator(device=DEV).manual_seed(seed)
    s = dict(kp=torch.randn(400, 16, 2, 128, generator=g, device=DEV).bfloat16(), vp=torch.randn(400, 16, 2, 128, generator=g, device=DEV).bfloat16(),
             tables=torch.randperm(400, generator=g, device=DEV)[:380].view(2, 190).to(torch.int32))
    cu = [0, new[0], sum(new)]
    return s, torch.randn(sum(new), 2, 128, generator=g, device=DEV).bfloat16(), _i32(list(lens)), _i32(cu)


def test_two_graphs_and_eager_launches_share_nothing(hip):
    """Launches with parts, captured twice and eager, in any order and on two streams at once: the same results every time."""
    cases = [_long(0), _long(1, (300, 1)), _long(2)]
    want = [_attend(*c, right=0) for c in cases]
    torch.cuda.synchronize()
    graphs, outs = [], []
    for c in cases[:2]:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(_attend(*c, right=0))
        graphs.append(graph)
    streams = [torch.cuda.Stream() for _ in range(2)]
    for turn in range(4):
        for o in outs:
            for t in o:
                t.zero_()
        torch.cuda.synchronize()
        for graph, stream in zip(graphs if turn % 2 else graphs[::-1], streams):
            with torch.cuda.stream(stream):
                graph.replay()
        eager = _attend(*cases[2], right=0)
        torch.cuda.synchronize()
        for got, ref in zip(outs + [eager], want):
            assert torch.equal(got[0], ref[0]) and torch.equal(got[1], ref[1])


def test_threads_and_streams(hip):
    cases = [_long(i, (1 + 100 * (i % 3), 1 + i)) for i in range(4)]
    want = [_attend(*c, right=0) for c in cases]
    torch.cuda.synchronize()
    bad = []

    def work(i, own_stream):
        stream = torch.cuda.Stream() if own_stream else torch.cuda.default_stream()
        with torch.cuda.stream(stream):
            for _ in range(30):
                out, lse = _attend(*cases[i], right=0)
                stream.synchronize()
                if not (torch.equal(out, want[i][0]) and torch.equal(lse, want[i][1])):
                    bad.append(i)

    for own in (True, False):
        threads = [threading.Thread(target=work, args=(i, own)) for i in range(4)]
        for t in threads:
            t.start()
        for t in threads:
            t.join()
    assert not bad


def test_repeats_bit_for_bit_and_leaves_its_counters_at_zero(hip):
    from ditango_amd import _hip
    cases = [_long(5), _long(6, (700, 3)), _long(7, (1, 1), (3040, 3040)), _long(8, (90, 90), (3040, 100))]
    first = [_attend(*c, left=2500, right=0) for c in cases]
    for _ in range(5):
        for c, (o, l) in zip(cases, first):
            out, lse = _attend(*c, left=2500, right=0)
            assert torch.equal(out, o) and torch.equal(lse, l)
    torch.cuda.synchronize()
    kept = [c for c in _hip._counters.values()]
    assert kept and all(not bool(c.any()) for c in kept)


def test_without_scratch_and_with_little(hip):
    """The C entry point with no workspace, no counters, or room for a few parts only: the same numbers, cut differently."""
    import ctypes
    from tests.test_long_video_refusals import Window
    from tests.test_pages_refusals import PagePool, I64x3
    lib = hip.load_library()
    for new in ((1, 2), (300, 1)):
        s, q, lens, cu = _long(11, new)
        want = _attend(s, q, lens, cu, right=0)
        strides = I64x3(*s["kp"].stride()[:3])
        pool = PagePool(s["kp"].data_ptr(), s["vp"].data_ptr(), strides, strides, 400, 16)
        w = Window(-1, 0, 1, 0, -1, None)
        ws = torch.empty(4 << 20, dtype=torch.uint8, device=DEV)
        counters = torch.zeros(64, dtype=torch.int32, device=DEV)
        ref = lambda x: ctypes.cast(ctypes.pointer(x), ctypes.c_void_p)
        for nbytes, words in ((0, 0), (1 << 20, 0), (0, 64), (1 << 17, 64), (4 << 20, 5), (4 << 20, 64)):
            out, lse = torch.full_like(q, 3.0), torch.full((2, q.shape[0]), 3.0, device=DEV)
            rc = lib.dt_attn_pages_fwd(q.data_ptr(), (ctypes.c_int64 * 2)(*q.stride()[:2]), out.data_ptr(), lse.data_ptr(), q.shape[0], 2, 2, 128, ref(pool),
                                       s["tables"].data_ptr(), s["tables"].stride(0), 190, 2, lens.data_ptr(), cu.data_ptr(), max(new), ref(w), 0.0, 0,
                                       ws.data_ptr() if nbytes else None, nbytes, counters.data_ptr() if words else None, words,
                                       torch.cuda.current_stream().cuda_stream)
            assert rc == 0, lib.dt_last_error()
            torch.cuda.synchronize()
            assert float((out.float() - want[0].float()).abs().max()) <= 2.0 ** -7 and float((lse - want[1]).abs().max()) <= 1e-4
            assert not bool(counters.any())


def test_inputs_of_another_kind_are_refused(hip):
    from ditango_amd import _hip
    from ditango_amd.pages import append_pages, paged_attention, plan_pages, prepare_qkv_pages
    from ditango_amd.producer import RotaryAxes
    q, pages = torch.zeros(4, 2, 64, device=DEV).bfloat16(), torch.zeros(3, 16, 2, 64, device=DEV).bfloat16()
    tables, lens, cu = _i32([[0, 1]]), _i32([4]), _i32([0, 4])
    slots, pos, axes = torch.zeros(4, dtype=torch.int64, device=DEV), torch.zeros(4, 3, dtype=torch.int32, device=DEV), RotaryAxes(dims=(16, 24, 24))
    bad = pytest.raises(_hip.DitangoHipError)
    for args in ((q.float(), pages, pages), (q, pages.half(), pages), (q, pages, pages.half()), (q, pages[:, :, :1].expand(3, 16, 3, 64), pages),
                 (q[None], pages, pages), (q, pages[0], pages), (q.half(), pages, pages), (q, pages, pages[:2]), (q[..., :32], pages[..., :32], pages[..., :32])):
        with bad:
            paged_attention(*args, tables, lens, cu)
    for args in ((tables[0], lens, cu), (tables, _i32([4, 4]), cu), (tables, lens, lens), (tables.t(), lens, cu), (tables, lens.cpu(), cu), (tables.cpu(), lens, cu)):
        with bad:
            paged_attention(q, pages, pages, *args)
    for kw in (dict(out=q[:2]), dict(out=q.half()), dict(lse=torch.zeros(4, 2, device=DEV)), dict(lse=torch.zeros(2, 4, device=DEV).half()), dict(out=q.cpu())):
        with bad:
            paged_attention(q, pages, pages, tables, lens, cu, **kw)
    with bad:
        paged_attention(q, pages[:, :8], pages[:, :8], tables, lens, cu)                     # pages of 8 tokens
    for args in ((q, q, pages, pages, slots.int()), (q, q, pages, pages, slots[:3]), (q, q[:3], pages, pages, slots), (q, q, pages, pages.half(), slots),
                 (q, q, pages, pages[:, :, :1], slots), (q.float(), q.float(), pages, pages, slots), (q, q, pages, pages, slots.cpu())):
        with bad:
            append_pages(*args)
    for args in ((q, q, q, pos, axes, pages, pages, slots[:2]), (q, q[:2], q, pos, axes, pages, pages, slots), (q, q, q.half(), pos, axes, pages, pages, slots),
                 (q, q, q, pos[:3], axes, pages, pages, slots), (q, q, q, pos.cpu(), axes, pages, pages, slots),
                 (q, q, q, pos, RotaryAxes(dims=(16, 56, 56)), pages, pages, slots)):
        with bad:
            prepare_qkv_pages(*args)
    for kw in (dict(q_weight=torch.ones(32, device=DEV)), dict(out=q[:1]), dict(out=q.float())):
        with bad:
            prepare_qkv_pages(q, q, q, pos, axes, pages, pages, slots, norm="rms", **kw)
    for args, kw in (((tables, lens, lens, 4), dict(n_pages=3, page_size=12)), ((tables, lens, lens, -1), dict(n_pages=3, page_size=16)),
                     ((tables, _i32([1, 2]), lens, 4), dict(n_pages=3, page_size=16)), ((tables, lens, lens, 4), dict(n_pages=1 << 21, page_size=16)),
                     ((tables[:0], lens[:0], lens[:0], 4), dict(n_pages=3, page_size=16))):
        with bad:
            plan_pages(*args, **kw)
    torch.cuda.synchronize()
