"""The operators of long videos together, as a rollout and as a sampler use them."""
import numpy as np
import pytest
import torch

from oracle import long_video as L

pytestmark = pytest.mark.gpu

DEV = "cuda:0"


@pytest.fixture
def env(hip):
    from ditango_amd.core import config, parallel_state, redundancy_map as rmod
    from ditango_amd import utils

    def make(N, rank, T, L, **cfg):
        parallel_state.init_local_groups(N, rank)
        config.init_config(None, num_inference_steps=T, num_layers=L, **cfg)
        rmod.destroy_redundancy_map()
        rmod._redundancy_map = rmod.RedundancyMap(config.get_config())
        return rmod.get_redundancy_map()

    yield make
    rmod.destroy_redundancy_map()
    parallel_state.destroy_local_groups()
    utils.update_timestep(0)
    config.init_config(None)


@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
def test_a_rollout(hip, fmt):
    """Frame after frame: its q and k are normalised and rotated by their place, its keys join the ones before, it attends to the window and the
    first frame; the state against a prompt is kept in 8 bits at the first step and merged from there at every one."""
    from ditango_amd.core.cache import merge_any, proCache
    from ditango_amd.producer import RotaryAxes, grid_positions, prepare_qk_axes
    from ditango_amd.window import window_attention
    B, H, Hk, D, f, h, w, frames = 2, 4, 2, 128, 1, 6, 10, 5
    n = h * w
    spec = dict(dims=(16, 56, 56), base=256.0)
    axes, cache = RotaryAxes(**spec), proCache(frames, 0, state_format=fmt)
    g = torch.Generator(device=DEV).manual_seed(0)
    prompt = [torch.randn(B, 40, Hk, D, generator=g, device=DEV).bfloat16() for _ in range(2)]
    wq, wk = (torch.rand(D, generator=g, device=DEV) + 0.5 for _ in range(2))
    k_cache, v_cache = (torch.full((B, frames * n, Hk, D), float("nan"), dtype=torch.bfloat16, device=DEV) for _ in range(2))
    lens = torch.zeros(B, dtype=torch.int32, device=DEV)
    first = None
    for t in range(frames):
        q0, k0, v0 = (torch.randn(B, n, x, D, generator=g, device=DEV).bfloat16() for x in (H, Hk, Hk))
        pos = grid_positions(f, h, w, first_frame=t, device=DEV)
        q, k = prepare_qk_axes(q0, k0, pos, axes, norm="rms", q_weight=wq, k_weight=wk)
        for x, y, wt in ((q0, q, wq), (k0, k, wk)):
            o = L.rotate(L.norm(x.cpu(), "rms", wt.cpu()), pos.cpu(), spec["dims"], (256.0,) * 3, "interleaved")
            assert bool(((y.cpu().double() - o).abs() <= 2.0 ** -8 * o.abs() + 1e-4).all())
        k_cache[:, t * n:(t + 1) * n], v_cache[:, t * n:(t + 1) * n] = k, v0
        lens.add_(n)
        out, lse = window_attention(q, k_cache, v_cache, left=1, right=0, frame=n, sinks=n, kv_lens=lens)
        o, l, weight, _ = L.window_attention(q, k_cache[:, :(t + 1) * n], v_cache[:, :(t + 1) * n], left=1, right=0, frame=n, sinks=n)
        assert bool(((out.double() - o).abs() <= 2.0 ** -8 * o.abs() + (2.0 ** -8 + 1e-3) * weight).all()) and float((lse.double() - l).abs().max()) < 1e-3
        if first is None:
            first = window_attention(q, *prompt)
            cache.store_block(0, *first)
        state, _ = cache.get_block(0)
        whole, whole_lse = merge_any([state, (out, lse)], dst_dtype=torch.bfloat16, dst_lse_bsh=True)
        e, x = L.quantize(first[0].cpu(), fmt)
        want, want_l = L.merge([(L.value(e, x), first[1].cpu()), (out.cpu(), lse.cpu())])
        assert bool(((whole.cpu().double() - want).abs() <= 2.0 ** -8 * want.abs() + 1e-5).all())
        assert float((whole_lse.squeeze(-1).transpose(1, 2).cpu().double() - want_l).abs().max()) < 1e-5


def _bound(fmt, vmax, stores):
    """How far the 8-bit cache may take a result: a value is off by half a step of its block, at most max |v| / 127 (int8) or a 16th of it and
    a 2^-10 of the block's scale (e4m3), once for every time it is stored; 16-bit states by 2^-8 max |v| each way."""
    return vmax * (stores * (1 / 127 if fmt == "int8" else 2.0 ** -4) + 2.0 ** -7)


@pytest.mark.parametrize("exact", [False, True])
@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
@pytest.mark.parametrize("N, rank, col", [(8, 3, (1, 1, 1, 4, 4, 4, 2, 2, 2, 2, 1, 1)), (4, 1, (1, 1, 1, 2, 2, 2, 1, 4, 2, 2, 1, 1))])
def test_a_generation_under_the_stride_schedule(env, N, rank, col, fmt, exact):
    """Beside the same generation with 16-bit states: one schedule, states in 8 bits, results within the cache's steps."""
    from ditango_amd.core.attention import proAttention
    from ditango_amd.core.cache import BlockState
    from ditango_amd.core.parallel_state import get_usp_group
    from ditango_amd.utils import update_timestep
    B, H, S, D = 1, 2, 100, 64
    rm = env(N, rank, len(col), 1)
    rm.divider_map[:, 0] = torch.tensor(col)
    group = get_usp_group()
    plain, small = proAttention(0, group), proAttention(0, group)
    small.cache = type(small.cache)(N, 0, state_format=fmt)
    if exact:
        plain.fp32_inputs = small.fp32_inputs = "exact"
    g = torch.Generator(device=DEV).manual_seed(N)
    dtype = torch.float32 if exact else torch.bfloat16
    reused = 0
    for t in range(len(col)):
        update_timestep(t)
        q = torch.randn(B, S, H, D, generator=g, device=DEV).to(dtype)
        ks, vs = ([torch.randn(B, S, H, D, generator=g, device=DEV).to(dtype) for _ in range(N)] for _ in range(2))
        group.set_kv_chunks(ks, vs)
        a = plain.attn(q, ks[rank], vs[rank])
        b = small.attn(q, ks[rank], vs[rank])
        assert plain.last_plan == small.last_plan and a.shape == b.shape and a.dtype == b.dtype
        reused += len(small.last_plan.reuse_merged)
        assert all(o is None or isinstance(o, BlockState) for o in small.cache.out_block_cache)
        assert float((plain.last_lse - small.last_lse).abs().max()) < 1e-4
        assert float((a - b).abs().max()) <= _bound(fmt, 6.0, 4)       # 25 600 normal values: below 6; stored once, coarsened at most 3 times
        if not small.last_plan.reuse_merged:
            assert float((a - b).abs().max()) <= 2.0 ** -7 * 6.0       # nothing from the cache: the merges differ in their order only
    assert reused > 0


@pytest.mark.parametrize("varlen", ["no", "host", "gpu"])
@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
def test_a_generation_under_a_mask(env, fmt, varlen):
    from ditango_amd.core.attention import proAttention
    from ditango_amd.core.parallel_state import get_usp_group
    from ditango_amd.utils import update_timestep
    C, T, H, S, D = 6, 4, 3, 90, 128
    rm = env(C, 2, T, 1, state_format=fmt)
    mask = (np.random.default_rng(0).random((T, 1, C)) < 0.6).astype(np.uint8)
    mask[0] = 0
    mask[3] = 1
    rm.set_chunk_mask(mask, diag=2)
    group = get_usp_group()
    small, plain = proAttention(0, group), proAttention(0, group)
    assert small.cache.state_format == fmt
    plain.cache = type(plain.cache)(C, 0)
    g = torch.Generator(device=DEV).manual_seed(1)
    cu = [0, 70, 84]
    for t in range(T):
        update_timestep(t)
        q = torch.randn(1, S, H, D, generator=g, device=DEV).bfloat16()
        ks, vs = ([torch.randn(1, S, H, D, generator=g, device=DEV).bfloat16() for _ in range(C)] for _ in range(2))
        if varlen == "no":
            group.set_kv_chunks(ks, vs)
            a, b = (x.attn(q, ks[2], vs[2]) for x in (plain, small))
        else:
            c = torch.tensor(cu, dtype=torch.int32, device=DEV) if varlen == "gpu" else cu
            group.set_kv_chunks(ks, vs, cu_seqlens_kv=[c] * C)
            a, b = (x.varlen_attn(q[0], ks[2][0], vs[2][0], c, c, 90, 90) for x in (plain, small))
            assert bool((b[84:] == 0).all())
        n = S if varlen == "no" else 84
        assert float((plain.last_lse[:, :n] - small.last_lse[:, :n]).abs().max()) < 1e-4
        a, b = a.reshape(S, H, D), b.reshape(S, H, D)
        assert float((a - b).abs().max()) <= _bound(fmt, 6.0, 1)
        if mask[t].sum() and t:
            assert not torch.equal(a, b)
    assert small.cache.arena_out.element_size() == 1 and small.cache.diag_out is None
    small.cache.release()
    assert small.cache.arena_scales is None


def test_a_layer_without_room_for_its_arena_recomputes(env):
    from ditango_amd.core.attention import proAttention
    from ditango_amd.core.parallel_state import get_usp_group
    from ditango_amd.utils import update_timestep
    C, S, H, D = 4, 50, 2, 64
    rm = env(C, 0, 2, 1, state_format="int8")
    mask = np.zeros((2, 1, C), dtype=np.uint8)
    mask[1, 0, 1:] = 1
    rm.set_chunk_mask(mask, diag=0)
    group = get_usp_group()
    attn = proAttention(0, group)
    attn.cache.memory_constraint = 0.0
    q = torch.randn(1, S, H, D, device=DEV).bfloat16()
    ks, vs = ([torch.randn(1, S, H, D, device=DEV).bfloat16() for _ in range(C)] for _ in range(2))
    group.set_kv_chunks(ks, vs)
    outs = []
    for t in range(2):
        update_timestep(t)
        outs.append(attn.attn(q, ks[0], vs[0]))
    assert attn.cache.arena_out is None and torch.equal(outs[0], outs[1])


@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
def test_many_ragged_chunks_under_a_mask(env, fmt):
    """More chunks than one launch addresses, some without a key, some steps that compute nothing but the own chunk."""
    from ditango_amd.core.attention import proAttention
    from ditango_amd.core.parallel_state import get_usp_group
    from ditango_amd.utils import update_timestep
    C, T, H, S, D = 70, 3, 2, 40, 64
    rm = env(C, 5, T, 1, state_format=fmt)
    mask = (np.random.default_rng(1).random((T, 1, C)) < 0.5).astype(np.uint8)
    mask[0], mask[2] = 0, 1
    rm.set_chunk_mask(mask, diag=5)
    group = get_usp_group()
    small, plain = proAttention(0, group), proAttention(0, group)
    plain.cache = type(plain.cache)(C, 0)
    g = torch.Generator(device=DEV).manual_seed(2)
    lens = [0 if c % 11 == 3 else 1 + (c * 17) % 60 for c in range(C)]
    for t in range(T):
        update_timestep(t)
        q = torch.randn(2, S, H, D, generator=g, device=DEV).bfloat16()
        ks, vs = ([torch.randn(2, n, H, D, generator=g, device=DEV).bfloat16() for n in lens] for _ in range(2))
        group.set_kv_chunks(ks, vs)
        a, b = (x.attn(q, ks[5], vs[5]) for x in (plain, small))
        assert float((plain.last_lse - small.last_lse).abs().max()) < 1e-4
        assert float((a - b).abs().max()) <= _bound(fmt, 6.0, 1)
