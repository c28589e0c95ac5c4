"""A call that is broken off while answers are forked leaves nothing held (CPU)."""
import types

import pytest
import torch

from pico_engine.cache import Cache, CacheNeeds, KVNeed
from pico_engine.engine.engine import EngineBackend
from pico_engine.engine.generate import generate


@pytest.mark.parametrize("error", [KeyboardInterrupt, SystemExit, RuntimeError, MemoryError])
@pytest.mark.parametrize("where", ["choose", "begin"])
def test_answers_that_are_broken_off_are_closed(error, where):
    cache = Cache([CacheNeeds(kv=KVNeed(1, 16, None))], 4096, 8, torch.float32, "cpu", allocate=False)

    def broken(*a, **k):
        raise error

    def prompts(slots, ids, use_graph=None):
        for s, p in zip(slots, ids):
            cache.reserve(s, len(p))
            cache.advance(s, len(p))
        return torch.zeros(len(slots), 5)
    memory = types.SimpleNamespace(begin=broken if where == "begin" else lambda *a: None, rules=lambda *a: None)
    engine = types.SimpleNamespace(cache=cache, device=torch.device("cpu"), prefill_tokens_per_step=100, stepper=types.SimpleNamespace(step=prompts),
                                   rule_memory=lambda: memory, last_timing={"prefill_s": 0.0})
    backend = EngineBackend(engine, types.SimpleNamespace(params=types.SimpleNamespace(ruled=True), choose=broken), False)
    with pytest.raises(error):
        generate(backend, [[1] * 70, [2] * 3], 5, (), 8, 4096, answers=3)
    assert not cache.lengths and not cache.prefix and cache.slots.free_count == 8 and cache.groups[0].pages.free_count == cache.n_pages
    cache.check()
