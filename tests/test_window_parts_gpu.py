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
