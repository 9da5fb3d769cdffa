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


@pytest.mark.parametrize("mode", ["no", "host", "gpu", "exact"])
@pytest.mark.parametrize("room", [1, 3])
@pytest.mark.parametrize("C", [8, 70])           # (and more chunks than one launch addresses)
def test_fresh_states_under_a_mask_stay_within_the_budget(env, C, room, mode):  # noqa: F811
    """A budget with room for ``room`` fresh states beside the arena: a call allocates no more, and gives what a call that has all of them at once gives."""
    from ditango_amd.core.attention import proAttention
    from ditango_amd.core.parallel_state import get_usp_group
    from ditango_amd.utils import update_timestep
    diag, T, dtype = 2, 3, torch.float32 if mode == "exact" else torch.bfloat16
    rm = env(C, diag, T, 1, state_format="int8")
    mask = (np.random.default_rng(C).random((T, 1, C)) < 0.5).astype(np.uint8)
    mask[0], mask[2] = 0, 1
    rm.set_chunk_mask(mask, diag=diag)
    group = get_usp_group()
    tight, easy = proAttention(0, group), proAttention(0, group)
    q, ks, vs = _inputs(C, dtype)
    if mode == "exact":
        tight.fp32_inputs = easy.fp32_inputs = "exact"
    if mode in ("no", "exact"):
        group.set_kv_chunks(ks, vs)
        run = lambda x: x.attn(q, ks[diag], vs[diag]).view(S, H, D)
        n = S
    else:
        at = [[0, 30, 50 + 7 * c] for c in range(C)]
        cu, cu_q = ([torch.tensor(a, dtype=torch.int32, device=DEV) for a in at], torch.tensor([0, 1000, 2900], dtype=torch.int32, device=DEV)) \
            if mode == "gpu" else (at, [0, 1000, 2900])
        group.set_kv_chunks(ks, vs, cu_seqlens_kv=cu)
        run = lambda x: x.varlen_attn(q[0], ks[diag][0], vs[diag][0], cu_q, cu[diag], S, S)
        n = 2900
    run(easy)                                    # (the stream's workspace)
    easy.cache.release()
    each, running, arena = S * H * (dtype.itemsize * D + 4), S * H * (4 * D + 4), C * S * H * (D + D // 32 + 4)
    for t in range(T):
        update_timestep(t)
        a, most_a = _peak(lambda: run(easy))
        here = torch.cuda.memory_allocated()
        tight.cache.memory_constraint = (here + (arena if t == 0 else 0) + running + room * each + 4096) / 2 ** 20
        b, most_b = _peak(lambda: run(tight))
        assert tight.cache.arena_out is not None and here + most_b <= tight.cache.memory_constraint * 2 ** 20 + (2 << 20)
        if t == 0:
            assert most_a > arena + C * each - (1 << 20)
        # both from states of the same bits but for how a launch shares its keys out: half a step of 16 bits here and there, and with it a step of the 8-bit cache
        assert float((a[:n] - b[:n]).abs().max()) <= _bound("int8", 6.0, 1)
        assert float((easy.last_lse[:, :n] - tight.last_lse[:, :n]).abs().max()) < 1e-4


@pytest.mark.parametrize("N, rank, col", [(8, 3, (1, 1, 4, 4, 2, 2, 1)), (4, 1, (1, 1, 2, 1, 4, 2, 1))])
@pytest.mark.parametrize("exact, out_dtype", [(False, torch.float32), (False, torch.bfloat16), (True, torch.float32)])
def test_fresh_states_under_the_stride_schedule_stay_within_the_budget(env, N, rank, col, exact, out_dtype):  # noqa: F811
    from ditango_amd.core.attention import proAttention
    from ditango_amd.core.parallel_state import get_usp_group
    from ditango_amd.utils import update_timestep
    rm = env(N, rank, len(col), 1, state_format="int8")
    rm.divider_map[:, 0] = torch.tensor(col)
    group = get_usp_group()
    tight, easy = proAttention(0, group), proAttention(0, group)
    tight.out_dtype = easy.out_dtype = out_dtype
    dtype = torch.bfloat16
    if exact:
        tight.fp32_inputs = easy.fp32_inputs = "exact"
        dtype = torch.float32
    each, running, slot = S * H * (dtype.itemsize * D + 4), S * H * (4 * D + 4), S * H * (D + D // 32 + 4)
    grouped = 0
    for t in range(len(col)):
        update_timestep(t)
        q, ks, vs = _inputs(N, dtype, seed=t)
        group.set_kv_chunks(ks, vs)
        a, most_a = _peak(lambda: easy.attn(q, ks[rank], vs[rank]))
        jobs, stores = len(easy.last_plan.launch[1]), len(easy.last_plan.stores)
        here = torch.cuda.memory_allocated()
        tight.cache.memory_constraint = (here + running + 2 * each + max(stores, N) * slot + 4096) / 2 ** 20      # (the schedule's own guard asks for N slots at most)
        b, most_b = _peak(lambda: tight.attn(q, ks[rank], vs[rank]))
        assert easy.last_plan == tight.last_plan and b.dtype == out_dtype
        result = S * H * (2 * D + 4) if out_dtype is torch.bfloat16 else 0
        assert here + most_b <= tight.cache.memory_constraint * 2 ** 20 + result + (2 << 20)
        grouped += running + jobs * each + stores * slot > running + 2 * each + max(stores, N) * slot
        assert float((a.float() - b.float()).abs().max()) <= _bound("int8", 6.0, 4)
        assert float((easy.last_lse - tight.last_lse).abs().max()) < 1e-4
    assert grouped
