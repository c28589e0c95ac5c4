"""A step that is refused leaves its sequences as they were (CPU)."""
import types

import pytest
import torch

from pico_engine.cache import Cache, CacheNeeds, KVNeed
from pico_engine.engine.step import StepError, Stepper


@pytest.mark.parametrize("lens,want,ids,more", [
    ([200, 1], None, [[1] * 199 + [100], [1]], {}),                       # a token outside the vocabulary
    ([200, 1], None, [[1] * 200, [-1]], {}),
    ([200, 1], None, [[1] * 199, [1]], {}),                               # fewer tokens than announced
    ([200, 1], [[0], [1]], [[1] * 200, [1]], {}),                         # a wanted place that the row does not have
    ([200, 1], [[-1], [0]], None, {}),
    ([200, 1], None, None, dict(n_tiles=(2, 1))),                         # more attention runs than the layout holds
    ([200, 1], None, None, dict(shared=True)),                            # shared pages in a step of several tokens a row
    ([300, 300], None, None, {}),                                         # beyond the longest sequence
    ([1, 0], None, None, {}),
])
def test_a_refused_step_takes_no_pages(lens, want, ids, more):
    needs = [CacheNeeds(kv=KVNeed(2, 16, None)), CacheNeeds(kv=KVNeed(2, 16, 32))]
    cache = Cache(needs, 2048, 4, torch.float32, "cpu", allocate=False)
    st = Stepper(types.SimpleNamespace(plan=types.SimpleNamespace(vocab_size=100), dtype=torch.float32), cache, 256)
    a, b = cache.open(), cache.open()
    cache.reserve(b, 3)
    cache.advance(b, 3)
    before = [{s: list(row) for s, row in g.table.items()} for g in cache.groups]
    with pytest.raises(StepError):
        st.describe([a, b], lens, want, ids, **more)
    assert [g.table for g in cache.groups] == before and cache.lengths == {a: 0, b: 3}
    lay, host, starts = st.describe([a, b], [1, 1], None, [[5], [6]])      # and the next one is laid out as if it had not been there
    assert starts == [0, 3] and [lay.widths, [len(g.table[a]) for g in cache.groups]] == [[1, 1], [1, 1]]
    cache.check()
