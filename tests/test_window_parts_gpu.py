"""Windows that are cut into parts along the keys: launches from two threads, values that one part sees and the others do not."""
import math
import threading

import pytest
import torch

from tests.test_window_gpu import DEV, _tensors

pytestmark = pytest.mark.gpu


def test_threads_that_launch_on_one_stream_share_its_workspace(hip):
    """Launches with a fold kernel behind their parts, of every kind and of the attention of whole chunks, from two threads on one stream: bit for bit what one thread
    alone gets (tests/test_window_launches.py has the order of the launches)."""
    from ditango_amd import _hip
    few = _tensors(1, 2, 30000, 2, 2, 128, torch.bfloat16, seed=1)
    shared = _tensors(1, 2100, 2100, 66, 66, 128, torch.bfloat16, seed=2)
    chunk = _tensors(1, 900, 2600, 2, 2, 128, torch.bfloat16, seed=3)
    stream = lambda: _hip._stream_at(few[0], "q")
    window = lambda t, right, counters: _hip._host().attn_window(*t, -1, right, 1, 0, -1, None, 0.0, None, None, _hip.attn_workspace(DEV), counters, stream())
    runs = [lambda: window(few, -1, None), lambda: window(shared, 0, None), lambda: window(few, -1, _hip._stream_counters(few[0].device, 1)),
            lambda: hip.attn_states(chunk[0], [chunk[1]], [chunk[2]], [[0]], 32, hip.attn_workspace(DEV))[0]]
    want = [run() for run in runs]
    torch.cuda.synchronize()
    for pair in ((0, 1), (0, 2), (1, 2), (0, 3), (1, 3)):
        got, errors, start = [[], []], [], threading.Barrier(2)

        def work(i):
            try:
                start.wait()
                for _ in range(60):
                    got[i].append(runs[pair[i]]())
            except Exception as e:   # noqa: BLE001 (reported by the assertion below)
                errors.append(e)
        threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
        for t in threads:
            t.start()
        for t in threads:
            t.join()
        torch.cuda.synchronize()
        assert not errors
        for i in range(2):
            o0, l0 = want[pair[i]]
            assert len(got[i]) == 60 and all(torch.equal(o, o0) and torch.equal(l, l0) for o, l in got[i])


@pytest.mark.parametrize("captured", [False, True])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("Sq, Sk, H, Hk", [(1, 256, 4, 4), (33, 300, 2, 1), (1, 30000, 2, 2), (9, 4000, 4, 2), (400, 410, 48, 1), (2100, 2100, 66, 66)])
def test_undefined_values_of_keys_far_below_the_others_are_seen(hip, Sq, Sk, H, Hk, D, captured):
    """Keys whose weight fp32 has no number for beside the others': their infinite and undefined values are those of visible keys all the same, whichever wavefront or part
    has the keys, and no other element changes."""
    from ditango_amd.window import window_attention
    q, k, v = _tensors(1, Sq, Sk, H, Hk, D, torch.bfloat16, seed=31, sigma=0.5)
    q += 4.0
    k[:, :Sk // 2] -= 32.0                       # scores of -4 x 32 sqrt(D), beside some units
    odd = v.clone()
    odd[0, 5, 0, 3], odd[0, Sk // 2 - 1, Hk - 1, D - 2] = math.inf, math.nan
    run = lambda x: window_attention(q, k, x)
    clean, clean_lse = run(v)
    if captured:
        run(odd)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out, lse = run(odd)
        graph.replay()
    else:
        out, lse = run(odd)
    torch.cuda.synchronize()
    bad = torch.zeros(1, 1, H, D, dtype=torch.bool, device=DEV)
    bad[0, 0, :H // Hk, 3] = True
    bad[0, 0, H - H // Hk:, D - 2] = True
    assert torch.equal(out.isfinite(), (~bad).expand_as(out))
    if not captured:                             # (a captured launch adds its parts up in another order)
        assert torch.equal(lse, clean_lse) and torch.equal(out[:, :, ~bad[0, 0]], clean[:, :, ~bad[0, 0]])
