"""What a cache in 8 bits takes in memory when nobody says how many sequences it is for, without a GPU."""
import pytest
import torch

from burn_lm_b200.cache import Cache, default_slots
from burn_lm_b200.engine.replay import cache_slots, cache_tokens
from burn_lm_b200.kernels import PAGE
from burn_lm_b200.parts.base import CacheNeed
from burn_lm_b200.plan import ScheduleEntry


def size(bits, tokens, dtype, dim):
    need = CacheNeed("kv", n_kv_heads=2, head_dim=dim, bits=bits)
    slots = default_slots([need, need, None], -(-tokens // PAGE))
    return Cache([need, need], [ScheduleEntry(0), ScheduleEntry(1)], tokens, slots, tokens, dtype, torch.device("cpu")).bytes()


@pytest.mark.parametrize("dim", [64, 80, 128])
@pytest.mark.parametrize("tokens", [256, 1000, 4096, 20000])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_it_is_smaller_than_one_in_the_compute_dtype(tokens, dim, dtype):
    assert size(8, tokens, dtype, dim) < 0.85 * size(0, tokens, dtype, dim)


def test_slots():
    kv = lambda bits: CacheNeed("kv", n_kv_heads=1, head_dim=16, bits=bits)  # noqa: E731
    for pages, plain, eight in ((1, 1, 1), (3, 3, 1), (64, 64, 16), (1024, 1024, 256), (10000, 1024, 1024)):
        assert default_slots([kv(0), None], pages) == plain
        assert default_slots([kv(0), (kv(0), kv(8))], pages) == eight
        assert default_slots([], pages) == plain


@pytest.mark.parametrize("tokens", [1, 64, 2048, 8192, 65536, 200000])
def test_a_replay_has_slots_for_the_requests_that_it_has_pages_for(tokens):
    """A page for each of 32 requests, or a quarter on top where that is more: so many requests may be live."""
    assert cache_slots(tokens, "compute") is None
    live = max(32, tokens // 4 // PAGE)
    assert live <= cache_slots(tokens, "int8") <= max(32, cache_tokens(tokens) // PAGE)
