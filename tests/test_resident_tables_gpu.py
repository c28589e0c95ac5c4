"""Captured decode steps that lay themselves out, for sequences that hold more pages than the step needs: against steps whose tables come from the host."""
import pytest
import torch

from conftest import TINY, make_weights, write_model
from pico_engine.engine import graph as graph_module
from pico_engine.engine.step import StepError
from pico_engine.sampling import Sampler, SamplingParams

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def eng(tmp_path_factory):
    from pico_engine.engine.engine import Engine
    return Engine(write_model(tmp_path_factory.mktemp("m") / "A", dict(TINY["A"]), make_weights(TINY["A"], 1, sharp=True)), dtype="float32")


def needed(cache, g, slots, width):
    """The page table up to each row's newest token (its step has advanced by now)."""
    table = cache.page_table(g, slots, width)
    for row, s in zip(table, slots):
        row[-(-max(cache.length(s), 1) // 64):] = -1
    return table


def answers(eng, resident, steps=60):
    """The tokens of four sequences, of which one has met a refused step and two have pages reserved ahead, after a prompt of the last."""
    eng.ensure_cache(4096, 128, 8)
    cache, st = eng.cache, eng.stepper
    slots = [cache.open() for _ in range(4)]
    out = []
    try:
        with pytest.raises(StepError, match="vocabulary"):
            st.step([slots[0]], [[1] * 99 + [10 ** 6]])
        cache.reserve(slots[1], 128)
        cache.reserve(slots[2], 65)
        st.step([slots[3]], [[3] * 64])
        g = graph_module.GraphedDecode(st, Sampler(SamplingParams(temperature=0.0)), 4)
        assert (g.tables is not None) == resident
        tokens = [1, 2, 3, 4]
        for _ in range(steps):
            tokens = g.launch(slots, tokens, [0, 1, 2, 3], [0] * 4).tokens()
            out.append(list(tokens))
            if resident:
                for k, w in enumerate(g.layout.widths):
                    got = g.dev[g.layout.tables[k]: g.layout.tables[k] + 4 * w].view(4, w).cpu().numpy()
                    assert (got == needed(cache, k, slots, w)).all()
    finally:
        for s in slots:
            cache.close(s)
    return out


@torch.inference_mode()
def test_steps_of_sequences_with_pages_reserved_ahead(eng, monkeypatch):
    monkeypatch.setattr(graph_module, "RESIDENT_ROWS", 1000)
    want = answers(eng, False)
    monkeypatch.setattr(graph_module, "RESIDENT_ROWS", 4)
    assert answers(eng, True) == want


@torch.inference_mode()
def test_a_launch_that_fails_can_be_made_again(eng, monkeypatch):
    """The description of a step does not reach the device: the next launch sends its pages again."""
    eng.ensure_cache(4096, 128, 8)
    cache, st = eng.cache, eng.stepper
    prompts = [[7] * 20, [8] * 3, [9] * 64, [5] * 60]
    g = graph_module.GraphedDecode(st, Sampler(SamplingParams(temperature=0.0)), 4)
    plainly, got = st.upload, []
    for fails in (False, True):
        slots = [cache.open() for _ in prompts]
        try:
            st.step(slots, prompts)
            tokens, seen = [1, 2, 3, 4], []
            for i in range(60):
                if fails and i in (0, 4, 5, 44, 59):
                    def broken(host, dev=None):
                        raise MemoryError
                    monkeypatch.setattr(st, "upload", broken)
                    with pytest.raises(MemoryError):
                        g.launch(slots, tokens, [0] * 4, [0] * 4)
                    monkeypatch.setattr(st, "upload", plainly)
                tokens = g.launch(slots, tokens, [0] * 4, [0] * 4).tokens()
                seen.append(list(tokens))
            got.append(seen)
        finally:
            for s in slots:
                cache.close(s)
    assert got[0] == got[1]
