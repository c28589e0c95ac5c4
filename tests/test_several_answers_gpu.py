"""Several answers to a prompt, rules on what they may say, and page tables that stay on the device, through generation: against answers that
are generated one by one, and against the plain implementation with the rules written out in 64 bits."""
import random

import pytest
import torch

import kevelorn_models
import lefilorn_models
import plain_qwen2 as plain
import pupidra_models
from conftest import TINY, make_weights, write_model
from pico_engine.engine import graph as graph_module
from pico_engine.ops import kernels as K
from pico_engine.sampling import TokenAutomaton

pytestmark = pytest.mark.gpu

OTHERS = {"K1": (kevelorn_models.CONFIGS["K1"], lambda c: kevelorn_models.make_weights(c, 40, 8)),
          "K3": (kevelorn_models.CONFIGS["K3"], lambda c: kevelorn_models.make_weights(c, 42, 8)),
          "P4": (pupidra_models.CONFIGS["P4"], lambda c: pupidra_models.make_weights(c, 50)),
          "L3": (lefilorn_models.CONFIGS["L3"], lambda c: lefilorn_models.make_weights(c, 62))}
LENGTHS = [70, 5, 128, 64, 1, 100]


@pytest.fixture(scope="module")
def models(tmp_path_factory):
    """{(config, dtype): (engine, cfg, weights)}."""
    from pico_engine.engine.engine import Engine
    root, out = tmp_path_factory.mktemp("models"), {}
    for i, (name, cfg) in enumerate(TINY.items()):
        weights = make_weights(cfg, i, sharp=True)
        folder = write_model(root / name, cfg, weights)
        for dtype in ("float32", "bfloat16"):
            out[(name, dtype)] = (Engine(folder, dtype=dtype), dict(cfg), weights)
    for name, (cfg, weights) in OTHERS.items():
        out[(name, "float32")] = (Engine(write_model(root / name, cfg, weights(cfg)), dtype="float32"), cfg, None)
    return out


@pytest.fixture
def together(monkeypatch):
    """Shared pages are read together however short they are; counts the layers that do it."""
    calls = []
    plainly = K.attention_shared
    monkeypatch.setattr(K, "SHARING_PAYS_BYTES", 1)
    monkeypatch.setattr(K, "attention_shared", lambda *a, **kw: (calls.append(a[0].shape[0]), plainly(*a, **kw))[1])
    return calls


def prompts_of(cfg, lengths=LENGTHS, seed=5):
    g = torch.Generator().manual_seed(seed)
    vocab, longest = cfg.get("vocab_size") or cfg["vocab"], cfg.get("max_position_embeddings", 512) - 24
    return [torch.randint(0, vocab, (min(n, longest),), generator=g).tolist() for n in lengths]


def nothing_held(eng):
    eng.cache.check()
    assert not eng.cache.lengths and eng.cache.slots.free_count == eng.cache.max_seqs
    assert all(g.pages.free_count == eng.cache.n_pages for g in eng.cache.groups) and not eng.cache.prefix


@pytest.mark.parametrize("name", ["A", "B", "C", "K1", "K3", "P4", "L3"])
@pytest.mark.parametrize("use_graph", [False, True])
def test_answers_are_those_of_separate_requests(models, name, use_graph):
    eng, cfg, _ = models[(name, "float32")]
    prompts = prompts_of(cfg)
    kw = dict(max_tokens=20, temperature=0.9, top_p=1.0, seed=3, stop_token_ids=(7, 11), use_graph=use_graph)
    one_by_one = eng.generate([p for p in prompts for _ in range(3)], **kw)
    got = eng.generate(prompts, n=3, **kw)
    assert got == [one_by_one[i: i + 3] for i in range(0, len(one_by_one), 3)]
    assert len({tuple(o) for o in got[2]}) > 1                                  # each answer draws for itself
    nothing_held(eng)


def test_answers_of_one_prompt_of_none_and_over_several_batches(models):
    eng, cfg, w = models[("A", "float32")]
    prompts = prompts_of(cfg, [9, 64, 3])
    want = [plain.generate(cfg, w, p, 6) for p in prompts]
    assert eng.generate(prompts[0], 6, temperature=0, n=2) == [want[0]] * 2
    assert eng.generate(prompts[0], 6, temperature=0, n=1) == want[0]
    assert eng.generate([prompts[0], [], prompts[1]], 6, temperature=0, n=2) == [[want[0]] * 2, [[], []], [want[1]] * 2]
    assert eng.generate(prompts, [0, 1, 6], temperature=0, n=3) == [[[]] * 3, [want[1][:1]] * 3, [want[2]] * 3]
    old, eng.max_batch = eng.max_batch, 4                                       # families are cut: 3 + 1, 2 + 2, ..
    try:
        assert eng.generate(prompts, 6, temperature=0, n=3) == [[o] * 3 for o in want]
        assert eng.generate(prompts, 6, temperature=0, n=9) == [[o] * 9 for o in want]
    finally:
        eng.max_batch = old
    with pytest.raises(ValueError, match="at least one answer"):
        eng.generate(prompts, 6, n=0)
    nothing_held(eng)


@pytest.mark.parametrize("name", ["C", "P4"])
def test_a_cache_that_holds_a_familys_prompt_once(tmp_path, name):
    """No more pages than the prompt's and what the answers add: every batch runs, with the answers of a cache that is large enough for all."""
    from pico_engine.engine.engine import Engine
    cfg = TINY["C"] if name == "C" else OTHERS[name][0]
    weights = make_weights(cfg, 2, sharp=True) if name == "C" else OTHERS[name][1](cfg)
    folder = write_model(tmp_path / "m", dict(cfg), weights)
    prompts = prompts_of(cfg, [300, 40])
    kw = dict(max_tokens=20, temperature=0.9, top_p=1.0, seed=1, stop_token_ids=())
    want = Engine(folder, dtype="float32").generate([p for p in prompts for _ in range(6)], **kw)
    for tokens in (320 + 5 * 64 + 6 * 64, 320 + 5 * 64, 320 + 64, 320):          # all together; a family a batch; two answers; one
        eng = Engine(folder, dtype="float32", max_tokens_in_cache=tokens)
        assert eng.generate(prompts, n=6, **kw) == [want[:6], want[6:]]
        assert eng.cache.n_pages * 64 == tokens
        nothing_held(eng)


@pytest.mark.parametrize("name", ["A", "B", "C"])
def test_a_prompt_in_portions(models, name):
    eng, cfg, _ = models[(name, "float32")]
    prompts = prompts_of(cfg)
    want = eng.generate(prompts, 8, temperature=0, n=2)
    old, eng.prefill_tokens_per_step = eng.prefill_tokens_per_step, 48
    try:
        assert eng.generate(prompts, 8, temperature=0, n=2) == want
    finally:
        eng.prefill_tokens_per_step = old
    nothing_held(eng)


# ---------------------------------------------------------------------------- rules

def ruled(logits, prompt, out, params, grammar, state):
    """The logits of the next token under the rules, in 64 bits."""
    x = logits.double().clone()
    rep, presence, frequency = (params.get(k, d) for k, d in (("repetition_penalty", 1.0), ("presence_penalty", 0.0), ("frequency_penalty", 0.0)))
    for t in set(prompt) | set(out):
        x[t] = x[t] / rep if x[t] > 0 else x[t] * rep
    for t in set(out):
        x[t] -= presence + frequency * out.count(t)
    for t, v in dict(params.get("logit_bias", {})).items():
        x[t] += v
    if grammar is not None:
        x[grammar.transitions[state] < 0] = -float("inf")
    return x


def automaton(vocab, states, seed):
    """Every state allows a fifth of the tokens, and leads on to states of all kinds."""
    g = torch.Generator().manual_seed(seed)
    t = torch.randint(0, states, (states, vocab), generator=g)
    t[torch.rand(states, vocab, generator=g) < 0.8] = -1
    t[torch.arange(states), torch.randint(0, vocab, (states,), generator=g)] = 0
    return TokenAutomaton(t, start=1)


RULES = [dict(repetition_penalty=1.3), dict(presence_penalty=0.7, frequency_penalty=0.4), dict(logit_bias={3: 2.5, 250: -4.0, 17: -float("inf")}),
         dict(repetition_penalty=0.8, presence_penalty=-0.5, logit_bias=[(i, 0.01 * i) for i in range(1, 150)]), dict(grammar=True),
         dict(repetition_penalty=1.2, presence_penalty=0.3, frequency_penalty=0.2, logit_bias={5: 1.0}, grammar=True)]


@pytest.mark.parametrize("rules", range(len(RULES)))
@pytest.mark.parametrize("name,use_graph", [("A", True), ("A", False), ("C", True)])
def test_rules_float32(models, name, use_graph, rules):
    eng, cfg, w = models[(name, "float32")]
    params = dict(RULES[rules])
    grammar = automaton(cfg["vocab_size"], 5, rules) if params.pop("grammar", False) else None
    prompts = prompts_of(cfg, [9, 70, 3])
    got = eng.generate(prompts, 12, temperature=0, use_graph=use_graph, n=2, stop_token_ids=(), grammar=grammar, **params)
    again = eng.generate(prompts, 12, temperature=0, use_graph=use_graph, stop_token_ids=(), grammar=grammar, **params)
    changed = 0
    for p, answers, alone in zip(prompts, got, again):
        assert answers[0] == answers[1] == alone
        out, state = [], 1
        for tok in answers[0]:
            row = ruled(plain.forward(cfg, w, p + out)[-1], p, out, params, grammar, state)
            assert int(row.argmax()) == tok, (p[:3], out)
            out.append(tok)
            state = state if grammar is None else int(grammar.transitions[state, tok])
        changed += out != plain.generate(cfg, w, p, 12)
    assert changed                                                              # (the rules do something)
    nothing_held(eng)


def test_settings_of_rules_share_a_graph_and_forget(models):
    """Numbers are read at run time: calls that vary them capture nothing new, and nothing is left of the sequences that held a slot before."""
    eng, cfg, _ = models[("A", "float32")]
    prompts = prompts_of(cfg, [9, 30])
    kw = dict(max_tokens=10, temperature=0)
    eng.generate(prompts, repetition_penalty=1.5, logit_bias={1: 1.0}, **kw)
    before = set(eng._graphs)
    a = eng.generate(prompts, repetition_penalty=1.0, frequency_penalty=2.0, logit_bias={9: -3.0, 4: 1.0}, **kw)
    assert set(eng._graphs) == before
    assert a == eng.generate(prompts, frequency_penalty=2.0, logit_bias={9: -3.0, 4: 1.0}, use_graph=False, **kw)
    assert a == eng.generate(prompts, frequency_penalty=2.0, logit_bias={9: -3.0, 4: 1.0}, **kw)
    for bad in (dict(logit_bias={256: 1.0}), dict(grammar=automaton(255, 3, 0)), dict(repetition_penalty=0.0), dict(frequency_penalty=float("nan"))):
        with pytest.raises(ValueError):
            eng.generate(prompts, **kw, **bad)
    nothing_held(eng)


# ---------------------------------------------------------------------------- shared pages and tables on the device

@pytest.mark.parametrize("use_graph", [False, True])
def test_shared_pages_read_together_bfloat16(models, together, use_graph):
    """Each chosen token must be a (near) maximum of the plain logits for the answer's own prefix, as answers of requests on their own."""
    eng, cfg, w = models[("C", "bfloat16")]
    prompts = prompts_of(cfg, [130, 20, 300, 64])
    got = eng.generate(prompts, 12, temperature=0, n=5, use_graph=use_graph, stop_token_ids=())
    assert len(together) > 0
    exact = 0
    for p, answers in zip(prompts, got):
        for out in answers:
            logits = plain.forward(cfg, w, p + out)
            for i, tok in enumerate(out):
                row = logits[len(p) + i - 1]
                assert float(row.max() - row[tok]) <= 4e-2 * max(1.0, float(row.abs().max())), (i, tok)
                exact += int(row.argmax()) == tok
    assert exact >= 200
    nothing_held(eng)


@pytest.mark.parametrize("name,dtype", [("A", "float32"), ("A", "bfloat16"), ("K3", "float32")])
def test_tables_on_the_device_change_no_token(models, monkeypatch, name, dtype):
    """Requests of unequal lengths that end one by one and take over one another's slots, over page ends, with and without forks; after every step the
    tables of its buffer are those of the cache."""
    eng, cfg, _ = models[(name, dtype)]
    rng = random.Random(4)
    prompts = prompts_of(cfg, [60, 3, 64, 1, 90, 62, 20, 63, 5])
    budgets = [rng.choice([3, 9, 20]) for _ in prompts]
    kw = dict(temperature=0.8, top_p=1.0, seed=2, stop_token_ids=(5,))
    plainly = graph_module.GraphedDecode.launch
    seen = []

    def launch(self, slots, *a, **k):
        flight = plainly(self, slots, *a, **k)
        if self.tables is not None:
            seen.append(len(self._many))
            lay, cache = self.layout, eng.cache
            for g, w in enumerate(lay.widths):
                table = self.dev[lay.tables[g]: lay.tables[g] + self.B * w].view(self.B, w).cpu().numpy()
                assert (table == cache.page_table(g, self._slots, w)).all()
            assert self.dev[lay.pos: lay.pos + self.B].tolist() == self._starts
            assert self.dev[lay.row: lay.row + self.B].tolist() == list(range(self.B)) and self.dev[lay.first: lay.first + self.B + 1].tolist() == list(range(self.B + 1))
        return flight
    monkeypatch.setattr(graph_module.GraphedDecode, "launch", launch)
    old, eng.max_batch = eng.max_batch, 4
    try:
        monkeypatch.setattr(graph_module, "RESIDENT_ROWS", 1000)
        eng._graphs.clear()
        want = [eng.generate(prompts, budgets, n=n, **kw) for n in (1, 3)]
        assert not seen
        monkeypatch.setattr(graph_module, "RESIDENT_ROWS", 1)
        eng._graphs.clear()
        assert [eng.generate(prompts, budgets, n=n, **kw) for n in (1, 3)] == want
        rows = len(seen)
        assert rows > 20 and sum(seen) > 0 and 0 in seen
        monkeypatch.setattr(graph_module, "RESIDENT_ROWS", 3)                # some steps this way, some that
        eng._graphs.clear()
        assert [eng.generate(prompts, budgets, n=n, **kw) for n in (1, 3)] == want
        assert rows < len(seen) < 2 * rows
    finally:
        eng.max_batch = old
        eng._graphs.clear()
    nothing_held(eng)


def test_windowed_caches_keep_their_tables_on_the_host(models):
    eng, _, _ = models[("B", "float32")]
    eng.generate([1, 2, 3], 2, temperature=0)
    assert eng.stepper.resident_tables() is None


def test_everything_together(models, together, monkeypatch):
    """Answers that share pages, under penalties, biases and a grammar, with their tables on the device: what is chosen is (nearly) the best of the plain
    logits under the rules, and allowed.  The logits' tolerance of 4e-2 grows by the repetition penalty of 1.3 at most (it multiplies negative ones)."""
    monkeypatch.setattr(graph_module, "RESIDENT_ROWS", 1)
    cfg = dict(TINY["C"], use_sliding_window=False)
    from pico_engine.engine.engine import Engine
    import tempfile
    from pathlib import Path
    weights = make_weights(cfg, 9, sharp=True)
    with tempfile.TemporaryDirectory() as d:
        eng = Engine(write_model(Path(d) / "m", cfg, weights), dtype="bfloat16")
    grammar = automaton(cfg["vocab_size"], 7, 8)
    params = dict(repetition_penalty=1.3, presence_penalty=0.4, frequency_penalty=0.3, logit_bias={8: 1.5, 100: -2.0})
    prompts = prompts_of(cfg, [130, 20, 300, 64])
    greedy = eng.generate(prompts, 16, temperature=0, n=6, stop_token_ids=(), grammar=grammar, **params)
    drawn = eng.generate(prompts, 16, temperature=0.9, n=6, seed=4, stop_token_ids=(13,), grammar=grammar, **params)
    assert len(together) > 0 and any(g.shared and g.tables is not None and g.graph is not None for g in eng._graphs.values())
    for p, answers in zip(prompts, greedy):
        for out in answers:
            assert grammar.walk(out) >= 0 and len(out) == 16
            logits, state = plain.forward(cfg, weights, p + out), grammar.start
            for i, tok in enumerate(out):
                raw = logits[len(p) + i - 1]
                row = ruled(raw, p, out[:i], params, grammar, state)
                assert float(row.max() - row[tok]) <= 1.3 * 4e-2 * max(1.0, float(raw.abs().max())), (i, tok)
                state = int(grammar.transitions[state, tok])
    for answers in drawn:
        assert all(grammar.walk(out) >= 0 and 13 not in out for out in answers) and len({tuple(o) for o in answers}) > 1
    nothing_held(eng)


@pytest.mark.parametrize("name", ["C", "K3", "P4", "L3"])
def test_steps_with_and_without_shared_pages(models, together, tmp_path, name):
    """One step of a family and of sequences beside it, in bfloat16, its layers' attention one by one and together: two roundings of the same logits, each
    within the 4e-2 of the engine's comparisons with the plain implementation."""
    from pico_engine.engine.engine import Engine
    if name == "C":
        eng, cfg, _ = models[("C", "bfloat16")]
    else:
        cfg = OTHERS[name][0]
        eng = Engine(write_model(tmp_path / "m", cfg, OTHERS[name][1](cfg)), dtype="bfloat16")
    prompts = prompts_of(cfg, [200, 9, 150])
    logits = {}
    for least in (10 ** 12, 1):
        K.SHARING_PAYS_BYTES = least                                             # (put back by the fixture)
        eng.ensure_cache(4096, 480, 32)
        slots = [eng.cache.open() for _ in prompts]
        try:
            eng.stepper.step(slots, prompts)
            slots += eng.cache.fork(slots[0], 4) + eng.cache.fork(slots[2], 1)
            order = [slots[i] for i in (1, 0, 3, 4, 5, 6, 2, 7)]
            logits[least] = [eng.stepper.step(order, [[t + i] for i in range(8)]).clone() for t in (3, 20)]
        finally:
            for s in slots:
                eng.cache.close(s)
        assert (len(together) > 0) == (least == 1)
    for a, b in zip(*logits.values()):
        assert float((a - b).abs().max()) <= 8e-2 * float(a.abs().max())
        assert not torch.equal(a[1], a[2])


def test_command_line(models, tmp_path):
    import json
    import os
    import subprocess
    import sys
    eng, cfg, w = models[("A", "float32")]
    folder = write_model(tmp_path / "m", dict(TINY["A"]), w)
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    r = subprocess.run([sys.executable, "-m", "pico_engine", str(folder), "--prompt", "5,17,3", "--prompt", "9,9", "--max-tokens", "6", "--temperature", "0.8",
                        "--dtype", "float32", "--n", "2", "--repetition-penalty", "1.3", "--frequency-penalty", "0.5", "--logit-bias", "3:2.5,17:-1"],
                       cwd=root, capture_output=True, text=True)
    assert r.returncode == 0, r.stderr[-2000:]
    lines = [json.loads(line) for line in r.stdout.splitlines() if line.startswith("{")]
    want = eng.generate([[5, 17, 3], [9, 9]], 6, 0.8, n=2, repetition_penalty=1.3, frequency_penalty=0.5, logit_bias={3: 2.5, 17: -1.0})
    assert [(q["prompt"], q["output"]) for q in lines] == [(p, o) for p, answers in zip(([5, 17, 3], [9, 9]), want) for o in answers]
