"""What the memory guard counts under a state format.  No GPU needed."""
import torch

from ditango_amd.core.cache import proCache

B, Sq, H, D = 1, 1024, 8, 128
MB = B * Sq * H / 2 ** 20                        # bytes of a row in MB


def _cache(mb_free):
    cache = proCache(8, 0, state_format="int8")
    cache.memory_probe, cache.memory_constraint = (lambda: 1000.0), 1000.0 + mb_free
    return cache


def test_an_arena_needs_room_for_fresh_states_beside_it():
    """8 slots of 136 bytes a row, a fresh state of 260 (exact mode: 516), and the 516 of the result that it is merged into."""
    for fresh_bytes, fresh in ((2, 260), (4, 516)):
        need = MB * (8 * 136 + fresh + 516)
        assert _cache(need + 1e-3).ensure_arena(8, B, Sq, H, D, torch.device("cpu"), fresh_bytes=fresh_bytes)
        cache = _cache(need - 1e-3)
        assert not cache.ensure_arena(8, B, Sq, H, D, torch.device("cpu"), fresh_bytes=fresh_bytes) and cache.arena_out is None
    plain = proCache(8, 0)                       # 16 bits: nine states, as ever
    plain.memory_probe, plain.memory_constraint = (lambda: 1000.0), 1000.0 + MB * 9 * 260 + 1e-3
    assert plain.ensure_arena(8, B, Sq, H, D, torch.device("cpu"))


def test_how_many_fresh_states_there_may_be_at_once():
    at_once = lambda rows, n, element_bytes=2, kept=0: _cache(MB * rows + 1e-3).fresh_at_once(n, B, Sq, H, D, element_bytes, kept)
    assert at_once(516 + 8 * 260, 8) == 8 and at_once(516 + 9 * 260, 8) == 8
    assert at_once(516 + 8 * 260 - 1, 8) == 7
    assert at_once(516 + 3 * 260, 8) == 3 and at_once(516 + 3 * 260 - 1, 8) == 2
    assert at_once(516 + 3 * 260 + 5 * 136, 8, kept=5) == 3 and at_once(516 + 8 * 260 + 8 * 136, 8, kept=8) == 8
    assert at_once(516 + 3 * 516, 8, element_bytes=4) == 3
    assert at_once(0, 8) == 1 and _cache(-500.0).fresh_at_once(8, B, Sq, H, D, 2) == 1


def test_no_bound_and_no_rows():
    cache = _cache(0.0)
    cache.memory_constraint = float("inf")
    assert cache.fresh_at_once(8, B, Sq, H, D, 2) == 8 and cache.ensure_arena(8, B, Sq, H, D, torch.device("cpu"))
    cache.memory_constraint = float("-inf")
    assert cache.fresh_at_once(8, B, Sq, H, D, 2) == 1
    for free in (100.0, 0.0, -100.0):
        assert _cache(free).fresh_at_once(8, B, 0, H, D, 2) == 8
