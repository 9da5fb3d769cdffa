"""Memory of layer calls with 8-bit states: what a call allocates beside the cache, where the budget has no room for the cache, and where it has little beside it."""
import numpy as np
import pytest
import torch

from tests.test_long_video_run_gpu import DEV, _bound, env  # noqa: F401 (a fixture)

pytestmark = pytest.mark.gpu

B, S, H, D = 1, 3000, 8, 128
STATE = S * H * (2 * D + 4)                      # bytes of a 16-bit state


def _inputs(C, dtype, seed=0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    mk = lambda n: torch.randn(B, n, H, D, generator=g, device=DEV).to(dtype)
    return mk(S), [mk(60 + 7 * c) for c in range(C)], [mk(60 + 7 * c) for c in range(C)]


def _peak(run):
    """(result, most bytes allocated during the call beyond what was there before it)."""
    torch.cuda.synchronize()
    before = torch.cuda.memory_allocated()
    torch.cuda.reset_peak_memory_stats()
    out = run()
    torch.cuda.synchronize()
    return out, torch.cuda.max_memory_allocated() - before


@pytest.mark.parametrize("varlen", ["no", "host", "gpu"])
@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
def test_a_layer_without_room_makes_no_state_of_each_chunk(env, fmt, varlen):  # noqa: F811
    """The 8-bit path without an arena takes the memory of the 16-bit one without, and gives its result bit for bit."""
    from ditango_amd.core.attention import proAttention
    from ditango_amd.core.parallel_state import get_usp_group
    from ditango_amd.utils import update_timestep
    C, diag = 8, 2
    rm = env(C, diag, 2, 1, state_format=fmt)
    rm.set_chunk_mask(np.zeros((2, 1, C), dtype=np.uint8), diag=diag)
    group = get_usp_group()
    small, plain = proAttention(0, group), proAttention(0, group)
    plain.cache = type(plain.cache)(C, 0)
    for x in (small, plain):
        x.cache.memory_constraint = 0.0
    q, ks, vs = _inputs(C, torch.bfloat16)
    if varlen == "no":
        group.set_kv_chunks(ks, vs)
        run = lambda x: x.attn(q, ks[diag], vs[diag])
    else:
        at = [[0, 30, 50 + 7 * c] for c in range(C)]
        cu, cu_q = ([torch.tensor(a, dtype=torch.int32, device=DEV) for a in at], torch.tensor([0, 1000, 2900], dtype=torch.int32, device=DEV)) \
            if varlen == "gpu" else (at, [0, 1000, 2900])
        group.set_kv_chunks(ks, vs, cu_seqlens_kv=cu)
        run = lambda x: x.varlen_attn(q[0], ks[diag][0], vs[diag][0], cu_q, cu[diag], S, S)
    for x in (plain, small):
        run(x)                                   # (the stream's workspace)
    for t in range(2):
        update_timestep(t)
        a, most_a = _peak(lambda: run(plain))
        b, most_b = _peak(lambda: run(small))
        n = S if varlen == "no" else 2900
        assert torch.equal(a.view(S, H, D)[:n], b.view(S, H, D)[:n]) and torch.equal(plain.last_lse[:, :n], small.last_lse[:, :n])
        assert most_b <= most_a + (1 << 20)
        assert most_b < 5 * STATE                # one state of 16 bits, the result of 32, its lse


def test_nor_in_exact_mode(env):  # noqa: F811
    from ditango_amd.core.attention import proAttention
    from ditango_amd.core.parallel_state import get_usp_group
    C = 40                                       # (more chunks than one launch addresses: two pieces)
    rm = env(C, 0, 1, 1, state_format="int8")
    rm.set_chunk_mask(np.zeros((1, 1, C), dtype=np.uint8), diag=0)
    group = get_usp_group()
    small, plain = proAttention(0, group), proAttention(0, group)
    plain.cache = type(plain.cache)(C, 0)
    for x in (small, plain):
        x.fp32_inputs, x.cache.memory_constraint = "exact", 0.0
    q, ks, vs = _inputs(C, torch.float32)
    group.set_kv_chunks(ks, vs)
    small.attn(q, ks[0], vs[0])
    a = plain.attn(q, ks[0], vs[0])
    for out_dtype in (torch.float32, torch.bfloat16):
        small.out_dtype = out_dtype
        b, most = _peak(lambda: small.attn(q, ks[0], vs[0]))
        assert b.dtype == out_dtype and most < 12 * STATE            # two pieces, their merge, the result
        # the same sums in another order: 8e-6 of values below 6 each way; then one rounding
        assert float((a - b.float()).abs().max()) <= 1e-4 + (0.0 if out_dtype is torch.float32 else 2.0 ** -8 * 6.0)
        assert float((plain.last_lse - small.last_lse).abs().max()) < 1e-5
