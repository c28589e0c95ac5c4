"""The 4-bit cache through the attention part, the engine and the command line.

The attention part is compared with the plain form in 64 bits on its own products' rows (codes equal, results within ``plain_int4.attend``'s bound and the last product's).  An engine's logits are
compared with the plain model whose keys and values are what the codes stand for: the engine's are off by a bfloat16 rounding or two (some 2^-8 of a number that has up to 8 steps
to its middle), so a code in twenty or so lands a step from the plain one: as much again as a third of the coding itself.  0.1 of the logits' size."""
import pytest
import torch

import plain_int4
import plain_qwen2 as plain
from conftest import TINY_C, make_weights, write_model
from pico_engine.ops import kernels as K

pytestmark = pytest.mark.gpu

LONG = {**TINY_C, "max_position_embeddings": 2048, "use_sliding_window": False}
LENGTHS = [70, 5, 128, 64, 1, 300]


@pytest.fixture(scope="module")
def folders(tmp_path_factory):
    root, out = tmp_path_factory.mktemp("int4"), {}
    for i, (name, cfg) in enumerate({"window": TINY_C, "long": LONG}.items()):
        weights = make_weights(cfg, 7 + i, sharp=True)
        out[name] = (write_model(root / name, cfg, weights), dict(cfg), weights)
    return out


def prompts(cfg, lengths=LENGTHS, seed=3):
    g = torch.Generator().manual_seed(seed)
    return [torch.randint(0, cfg["vocab_size"], (n,), generator=g).tolist() for n in lengths]


def coded_logits(cfg, weights, tokens, monkeypatch):
    """The plain model over keys and values as a 4-bit cache holds them."""
    plainly = plain.attention
    with monkeypatch.context() as m:
        m.setattr(plain, "attention", lambda q, k, v, w: plainly(q, *(plain_int4.stands_for(x.bfloat16()).float() for x in (k, v)), w))
        return plain.forward(cfg, weights, tokens)


def near(got, want):
    return float((got.cpu().float() - want.float()).abs().max()) <= 0.1 * max(1.0, float(want.abs().max()))


# ---------------------------------------------------------------------------- the part

def part_of(nh, nkv, hd, window, rotary, H=96):
    from pico_engine.config import GQAAttentionSpec, NoPositionSpec, RotaryHalfSpec
    from pico_engine.parts import MIXERS, build_part
    g = torch.Generator().manual_seed(nh)
    names = (("q", nh * hd), ("k", nkv * hd), ("v", nkv * hd))
    tensors = {f"a.{n}_proj.weight": torch.randn(o, H, generator=g) * H ** -0.5 for n, o in names}
    tensors.update({f"a.{n}_proj.bias": torch.randn(o, generator=g) for n, o in names})
    tensors["a.o_proj.weight"] = torch.randn(H, nh * hd, generator=g) * (nh * hd) ** -0.5
    spec = GQAAttentionSpec(hidden=H, n_heads=nh, n_kv_heads=nkv, head_dim=hd, qkv_bias=True, window=window, scale=hd ** -0.5,
                            position=RotaryHalfSpec(hd, 5e4) if rotary else NoPositionSpec(), prefix="a.")
    part = build_part(MIXERS, "mixer", spec, torch.bfloat16, "cuda")
    part.take_tensors(lambda n: tensors[n].bfloat16().cuda())
    part.prepare(1024)
    return part


@pytest.mark.parametrize("nh,nkv,hd,window,rotary,keep", [(14, 2, 64, None, True, None), (8, 2, 128, 100, True, None), (4, 4, 64, None, False, 3), (28, 4, 128, None, True, 4)])
def test_the_part_over_prompts_and_tokens(nh, nkv, hd, window, rotary, keep):
    from types import SimpleNamespace
    from pico_engine.cache import Cache
    from pico_engine.engine.step import Stepper
    from pico_engine.ops import linear
    part = part_of(nh, nkv, hd, window, rotary)
    cache = Cache([part.cache_needs()], 64 * 40, 4, torch.bfloat16, "cuda", int4=True, bounds=keep is not None)
    assert cache.groups[0].int4 and cache.groups[0].v is None
    stepper = Stepper(SimpleNamespace(plan=SimpleNamespace(vocab_size=1 << 20), dtype=torch.bfloat16), cache, 1024, keep)
    slots = [cache.open() for _ in range(3)]
    keys, values = ([torch.zeros(0, nkv, hd, dtype=torch.float64, device="cuda") for _ in slots] for _ in range(2))
    for step, lens in enumerate([[330, 9, 63], [1, 1, 1], [40, 1, 2], [1, 1, 1], [1, 1, 1]]):
        lay, host, starts = stepper.describe(slots, lens, None, None)
        ctx = stepper.context(lay, stepper.upload(host), lens, starts, slots)
        h = torch.randn(sum(lens), 96, generator=torch.Generator(device="cuda").manual_seed(step), device="cuda").bfloat16()
        got = part._attend(h, ctx, 0, True).double().view(-1, nh, hd)
        for s, n in zip(slots, lens):
            cache.advance(s, n)
        rows = linear(h, part.w_qkv, part.b_qkv, out_dtype=torch.bfloat16).view(-1, nh + 2 * nkv, hd)
        at = 0
        for b, (start, n) in enumerate(zip(starts, lens)):
            x = rows[at:at + n].double()
            if rotary:
                c, s = (t.cuda().double()[start:start + n, None] for t in part._tables(ctx))
                lo, hi = x[:, :nh + nkv, :hd // 2], x[:, :nh + nkv, hd // 2:]
                x = torch.cat([torch.cat([lo * c - hi * s, lo * s + hi * c], -1), x[:, nh + nkv:]], 1)
            q = x[:, :nh].float().bfloat16()
            keys[b] = torch.cat([keys[b], plain_int4.stands_for(x[:, nh:nh + nkv].float().bfloat16())])
            values[b] = torch.cat([values[b], plain_int4.stands_for(x[:, nh + nkv:])])
            for i in sorted({0, n // 2, n - 1}):
                pos = start + i
                w, unit = rows_of(q[i], keys[b][:pos + 1], values[b][:pos + 1], hd ** -0.5, window, keep if all(m == 1 for m in lens) else None)
                # a query's own rounding (2^-8 of it) moves a score by 2^-8 of its terms, another two by the kernel's; weights and results in bfloat16
                assert (got[at + i] - w).abs().max() <= unit, (step, b, i)
            at += n


def rows_of(q, k, v, scale, window, keep):
    """(results of a token's heads in 64 bits, what they may be off by)."""
    nh, nkv, pos = q.shape[0], k.shape[1], k.shape[0] - 1
    out = []
    for h in range(nh):
        g = h * nkv // nh
        j = torch.arange(pos + 1, device="cuda")
        if window:
            j = j[j > pos - window]
        if keep is not None and pos // 64 + 1 > keep:
            qs = q.view(nkv, -1, q.shape[1])[g].double()
            pages = range(1, pos // 64)
            score = {p: float(torch.maximum(qs * k[p * 64:p * 64 + 64, g].amin(0).float().bfloat16().double(), qs * k[p * 64:p * 64 + 64, g].amax(0).float().bfloat16().double()).sum()) for p in pages}
            best = sorted(pages, key=lambda p: (-score[p], p))[:keep - 2] + [0, pos // 64]
            j = torch.cat([torch.arange(p * 64, min(p * 64 + 64, pos + 1), device="cuda") for p in sorted(best)])
        w = torch.softmax(k[j, g] @ q[h].double() * scale, 0)
        out.append(w @ v[j, g])
    # roundings: a query's 2^-8, keys' 2^-11, weights' and values' 2^-8 and another behind a step: of scores of up to 8 and values of up to 4 in size, as root mean squares over 64 terms
    return torch.stack(out), 2.0 ** -8 * 4 * 4


# ---------------------------------------------------------------------------- the engine

@pytest.mark.parametrize("name", ["window", "long"])
def test_logits_against_the_plain_model(folders, name, monkeypatch):
    from pico_engine import Engine
    folder, cfg, weights = folders[name]
    eng = Engine(folder, cache="int4", max_context=512)
    eng.ensure_cache(64 * 40, 512)
    texts = prompts(cfg)
    slots = [eng.cache.open() for _ in texts]
    out = eng.stepper.step(slots, texts)
    for i, t in enumerate(texts):
        assert near(out[i], coded_logits(cfg, weights, t, monkeypatch)[-1]), i
    for _ in range(3):                                                      # single tokens, then a few at once
        more = [[(7 * i + len(t)) % cfg["vocab_size"]] for i, t in enumerate(texts)]
        texts = [t + m for t, m in zip(texts, more)]
        out = eng.stepper.step(slots, more)
    for i, t in enumerate(texts):
        assert near(out[i], coded_logits(cfg, weights, t, monkeypatch)[-1]), i
    for s in slots:
        eng.cache.close(s)
    eng.cache.check()


@pytest.mark.parametrize("attend", [None, 4])
def test_generation_captured_or_not(folders, attend):
    from pico_engine import Engine
    folder, cfg, _ = folders["long"]
    eng = Engine(folder, cache="int4", attend_pages=attend, max_context=700)
    texts = prompts(cfg, [400, 30, 64, 129])
    got = eng.generate(texts, max_tokens=70, temperature=0.0, stop_token_ids=())
    assert got == eng.generate(texts, max_tokens=70, temperature=0.0, stop_token_ids=(), use_graph=False)
    assert got == eng.generate(texts, max_tokens=70, temperature=0.0, stop_token_ids=())
    several = eng.generate(texts[0], max_tokens=70, temperature=0.0, stop_token_ids=(), n=3)
    assert several[0] == several[1] == several[2]
    eng.cache.check()
    assert not eng.cache.lengths and eng.cache.groups[0].pages.free_count == eng.cache.n_pages


def test_selected_pages_that_are_all_change_nothing(folders):
    """A token that sees no more pages than it may attend to has the results of one that attends to all (other sums of the same terms)."""
    from pico_engine import Engine
    folder, cfg, _ = folders["long"]
    outs = []
    for attend in (None, 8):
        eng = Engine(folder, cache="int4", attend_pages=attend)
        eng.ensure_cache(64 * 30, 1500)
        text = prompts(cfg, [400])[0]
        slot = eng.cache.open()
        eng.stepper.step([slot], [text])
        eng.stepper.max_context = 1500
        if attend:
            lay, host, starts = eng.stepper.describe([slot], [1], None, [[5]])
            ctx = eng.stepper.context(lay, eng.stepper.upload(host), [1], starts, [slot])
            ctx.max_context = 1500                                           # as in a captured step: the choice is made, of all pages
            ids = torch.tensor([5], dtype=torch.int32, device="cuda")
            outs.append(eng.model.forward(ids, ctx, torch.zeros(1, dtype=torch.int32, device="cuda"))[0].clone())
        else:
            outs.append(eng.stepper.step([slot], [[5]])[0].clone())
    assert float((outs[0] - outs[1]).abs().max()) <= 2e-2 * float(outs[0].abs().max())


def test_memory_and_forked_bytes(folders):
    from pico_engine import Engine
    folder, cfg, _ = folders["long"]
    coded, whole = (Engine(folder, cache=c) for c in ("int4", None))
    for e in (coded, whole):
        e.ensure_cache(64 * 30, 1500)
    assert coded.cache.bytes() * 16 == whole.cache.bytes() * 5
    text = prompts(cfg, [100])[0]
    slot = coded.cache.open()
    coded.stepper.step([slot], [text])
    (other,) = coded.cache.fork(slot)
    g = coded.cache.groups[0]
    a, b = g.table[slot], g.table[other]
    assert a[0] == b[0] and a[1] != b[1] and torch.equal(g.k[:, a[1]], g.k[:, b[1]])
    one, two = coded.stepper.step([slot, other], [[9], [9]])
    assert torch.equal(one, two)


def test_what_engines_refuse(folders):
    from pico_engine import Engine
    folder, _, _ = folders["long"]
    for more, match in ((dict(cache="int8"), "cache must be"), (dict(attend_pages=4), "goes with"), (dict(cache="int4", attend_pages=0), "must be positive"),
                        (dict(cache="int4", dtype="float32"), "no layer of this model")):
        with pytest.raises(ValueError, match=match):
            Engine(folder, **more)


def test_command_line(folders, capsys):
    from pico_engine.__main__ import main
    folder, cfg, _ = folders["long"]
    main([str(folder), "--random-prompt", "200,5", "--max-tokens", "6", "--temperature", "0", "--cache", "int4", "--attend-pages", "2", "--stop-token-ids", ""])
    out = capsys.readouterr().out
    assert out.count('"output"') == 2 and "generated 12 tokens" in out
    with pytest.raises(SystemExit):
        main([str(folder), "--prompt", "1", "--attend-pages", "2"])
