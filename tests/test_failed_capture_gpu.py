"""A captured step whose trial runs fail: the step runs kernel by kernel instead, from where it would have started."""
import warnings

import pytest
import torch

import kevelorn_models
from conftest import TINY, make_weights, write_model
from pico_engine.engine import graph as graph_module
from pico_engine.sampling import TokenAutomaton

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("name", ["A", "K1"])
@pytest.mark.parametrize("fails_at", [1, 2, 3])
def test_a_trial_run_that_fails_leaves_no_trace(tmp_path, monkeypatch, name, fails_at):
    """What the step before chose, a mixer's state, what the rules remember: counted once."""
    from pico_engine.engine.engine import Engine
    cfg, weights = (TINY["A"], make_weights(TINY["A"], 0, sharp=True)) if name == "A" else \
        (kevelorn_models.CONFIGS["K1"], kevelorn_models.make_weights(kevelorn_models.CONFIGS["K1"], 40, 8))
    eng = Engine(write_model(tmp_path / "m", dict(cfg), weights), dtype="float32")
    vocab = eng.model.plan.vocab_size
    g = torch.Generator().manual_seed(3)
    t = torch.randint(0, 4, (4, vocab), generator=g)
    t[torch.rand(4, vocab, generator=g) < 0.5] = -1
    t[:, 0] = 1
    prompts = [torch.randint(0, vocab, (n,), generator=g).tolist() for n in (9, 30, 4, 17, 20)]
    kw = dict(max_tokens=[3, 9, 12, 5, 12], temperature=0, stop_token_ids=(), frequency_penalty=3.0, repetition_penalty=1.2, grammar=TokenAutomaton(t))
    want = eng.generate(prompts, use_graph=False, **kw)
    plainly, runs = graph_module.GraphedDecode._forward, {}

    def forward(self):
        plainly(self)
        runs[id(self)] = runs.get(id(self), 0) + 1
        if runs[id(self)] == fails_at:
            raise RuntimeError("no room for a trial run")
    monkeypatch.setattr(graph_module.GraphedDecode, "_forward", forward)
    with warnings.catch_warnings(record=True) as said:
        warnings.simplefilter("always")
        got = eng.generate(prompts, use_graph=True, **kw)
    assert got == want
    assert any("no room" in str(w.message) for w in said) and all(g.graph is None for g in eng._graphs.values()) and len(runs) >= 3


def test_a_prompts_trial_run_that_fails_leaves_no_trace(tmp_path, monkeypatch):
    from pico_engine.engine.engine import Engine
    cfg = kevelorn_models.CONFIGS["K1"]
    eng = Engine(write_model(tmp_path / "m", dict(cfg), kevelorn_models.make_weights(cfg, 40, 8)), dtype="float32")
    assert eng.model.cache_needs() and any(n is not None and n.state_elems for n in eng.model.cache_needs())
    prompts = [[5, 6, 7, 8, 9, 10, 11] * 4, [3, 1, 2]]
    want = eng.generate(prompts, 10, temperature=0, stop_token_ids=())   # (the first prompt step of its sizes runs kernel by kernel)
    plainly, broken = graph_module.GraphedPrompt._forward, []

    def forward(self, ctx):
        plainly(self, ctx)
        if self.launches == 2 and not broken:
            broken.append(self)
            raise RuntimeError("no room for a trial run")
    monkeypatch.setattr(graph_module.GraphedPrompt, "_forward", forward)
    with pytest.warns(UserWarning, match="no room"):
        assert eng.generate(prompts, 10, temperature=0, stop_token_ids=()) == want
    assert broken and broken[0].graph is None
    assert eng.generate(prompts, 10, temperature=0, stop_token_ids=()) == want
