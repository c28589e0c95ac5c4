"""What several answers to one prompt cost beside the decoder itself: attention over a shared prefix, the rules on what may be chosen next,
and the page tables of a step.

A case is a plain dict.  ``op`` says which operator it goes through:

* ``"attention"``: one token a row; the rows of a group share the pages of their prompt and hold the rest for themselves;
* ``"rules"``: penalties for repeated tokens, biases and a grammar's mask on the logits of a step;
* ``"note"``: the tokens of prompts marked in the table of seen tokens;
* ``"tables"``: positions, rows, places in the cache and page tables of a step, from the lengths of its requests.

``own`` false: elementary torch operations.  ``own`` true: the library's kernels.
"""
from __future__ import annotations

import math

import torch

own = False

DEVICE = "cuda"
PAGE = 64
VOCAB = 151936
# (query heads, key/value heads, head size) of qwen2.5-0.5b, of design_compare's middle size, of qwen2.5-7b
SMALL, MIDDLE, LARGE = (14, 2, 64), (16, 4, 128), (28, 4, 128)
LONGEST = 32768                     # positions of the largest configuration
NONE = float("-inf")


def _text(values):
    return ",".join(str(int(v)) for v in values)


def _ints(text):
    return [int(v) for v in text.split(",")]


def _attention(size, rows, shared, low, high, window=0, keep_first=0, sinks=False, slopes=False):
    heads, kv_heads, dim = size
    return dict(op="attention", heads=heads, kv_heads=kv_heads, dim=dim, rows=_text(rows), shared=_text(shared), low=low, high=high,
                window=window, keep_first=keep_first, sinks=sinks, slopes=slopes)


def _rules(rows, vocab, penalties, biases, masked, allowed=0.02):
    return dict(op="rules", rows=rows, vocab=vocab, penalties=penalties, biases=biases, masked=masked, allowed=allowed)


def listed():
    return [
        # four answers to a short prompt: nothing but latency
        dict(_attention(SMALL, [4], [576], 1, 90), name="answers_4"),
        # sixteen answers to the benchmark's context
        dict(_attention(SMALL, [16], [4032], 1, 500), name="answers_16"),
        # a full batch of answers to a document near the longest context
        dict(_attention(SMALL, [64], [31744], 1, 900), name="answers_64_long"),
        # the larger model: unequal groups on unequal prompts, one answer that is alone among them
        dict(_attention(LARGE, [16, 1, 9, 30, 8], [1984, 640, 6080, 3008, 192], 1, 700), name="answers_groups_large"),
        # a sliding window with kept first keys and a sink, answers that have left part of their prompt behind
        dict(_attention(MIDDLE, [24, 8], [2496, 960], 1, 1500, window=2000, keep_first=4, sinks=True), name="answers_window"),
        # one request under a repetition penalty
        dict(_rules(1, VOCAB, True, 0, False), name="rules_1"),
        # a full batch under all rules
        dict(_rules(64, VOCAB, True, 300, True), name="rules_64"),
        # many requests under a grammar alone, a vocabulary that is no multiple of 32
        dict(_rules(200, 50257, False, 0, True), name="rules_grammar_200"),
        # the prompts of a batch, noted before its first token is chosen
        dict(op="note", slots=64, vocab=VOCAB, tokens=16000, name="note_prompts"),
        # a decode step of a full batch, contexts up to the longest
        dict(op="tables", rows=64, width=512, low=20000, high=32700, new="1", name="tables_64"),
        # unequal prompts, a chunk of a longer one among them
        dict(op="tables", rows=5, width=512, low=0, high=300, new="5001,1807,700,33,8000", name="tables_prompts"),
        # a very large batch of short conversations
        dict(op="tables", rows=2000, width=128, low=100, high=8000, new="1", name="tables_2000"),
    ]


def draw(rng):
    log = lambda a, b: int(round(math.exp(rng.uniform(math.log(a), math.log(b)))))      # noqa: E731
    kind = rng.choice(["attention", "attention", "attention", "rules", "rules", "tables", "note"])
    if kind == "attention":
        size = rng.choice([SMALL, MIDDLE, LARGE])
        while True:
            rows = [log(1, 64) for _ in range(rng.choice([1, 1, 2, 3, 6]))]
            shared = [log(1, 496) * PAGE for _ in rows]
            high = log(1, 1000)
            # the plain form gathers every row's whole context
            if sum(rows) <= 128 and sum(rows) * (max(shared) + high) * size[1] * size[2] <= 64 * LONGEST * 128:
                break
        window = rng.choice([0, 0, rng.randint(100, 4000)])
        return _attention(size, rows, shared, 1, high, window, rng.choice([0, 4, 100]) if window else 0, rng.random() < 0.3, rng.random() < 0.2)
    if kind == "rules":
        vocab = rng.choice([VOCAB, 152064, 50257, rng.randint(300, 130000)])
        while True:
            penalties, biases, masked = rng.random() < 0.7, rng.choice([0, 0, log(1, 1000)]), rng.random() < 0.5
            if penalties or biases or masked:
                break
        return _rules(log(1, 64), vocab, penalties, min(biases, vocab), masked, rng.choice([0.0005, 0.02, 0.5]))
    if kind == "note":
        return dict(op="note", slots=log(1, 64), vocab=rng.choice([VOCAB, 50257, 32000]), tokens=log(1, 16000))
    rows = log(1, 2000)
    width = log(8, 512 if rows <= 500 else 128)
    if rng.random() < 0.5:
        return dict(op="tables", rows=rows, width=width, low=0, high=width * PAGE - 1, new="1")
    return dict(op="tables", rows=rows, width=width, low=0, high=width * PAGE // 2, new=str(log(1, min(width * PAGE // 2, max(1, 16000 // rows)))))


# ---------------------------------------------------------------------------- inputs

def _generator(seed):
    return torch.Generator(device=DEVICE).manual_seed(int(seed))


def _normal(g, *shape, dtype=torch.float32):
    return torch.randn(*shape, generator=g, device=DEVICE, dtype=torch.float32).to(dtype)


def _lengths(case):
    """(group, shared positions, own tokens with the one that this step brings) of every row."""
    out = []
    for i, (n, s) in enumerate(zip(_ints(case["rows"]), _ints(case["shared"]))):
        for j in range(n):
            out.append((i, s, case["low"] + (case["high"] - case["low"]) * ((j * 37 + 11 * i + 5) % (n + 2)) // (n + 1)))
    return out


def prepare(case, seed):
    g = _generator(seed)
    return {"attention": _prepare_attention, "rules": _prepare_rules, "note": _prepare_note, "tables": _prepare_tables}[case["op"]](case, g)


def _prepare_attention(case, g):
    H, G, D = case["heads"], case["kv_heads"], case["dim"]
    rows = _lengths(case)
    T = len(rows)
    own_pages = [-(-n // PAGE) for _, _, n in rows]
    width = max(s // PAGE + p for (_, s, _), p in zip(rows, own_pages))
    prompts = [s // PAGE for s in _ints(case["shared"])]
    total = sum(prompts) + sum(own_pages)
    order = torch.randperm(total + 3, generator=g, device=DEVICE).tolist()            # pages lie anywhere in the pool
    at, prompt_pages = 0, []
    for n in prompts:
        prompt_pages.append(order[at:at + n])
        at += n
    table = []
    for (i, _, _), p in zip(rows, own_pages):
        row = prompt_pages[i] + order[at:at + p]
        at += p
        table.append(row + [-1] * (width - len(row)))
    pos = [s + n - 1 for _, s, n in rows]
    groups = []
    for t, (i, s, _) in enumerate(rows):
        members = [u for u, r in enumerate(rows) if r[0] == i]
        groups.append([members[0], len(members), s, min(members, key=lambda u: pos[u])])
    qkv = _normal(g, T, (H + 2 * G) * D, dtype=torch.bfloat16) * 1.5                  # queries at the front of wider rows
    return dict(case=case, qkv=qkv, k=_normal(g, total + 3, G, PAGE, D, dtype=torch.bfloat16), v=_normal(g, total + 3, G, PAGE, D, dtype=torch.bfloat16),
                table=torch.tensor(table, dtype=torch.int32, device=DEVICE), pos=torch.tensor(pos, dtype=torch.int32, device=DEVICE),
                row=torch.arange(T, dtype=torch.int32, device=DEVICE), groups=torch.tensor(groups, dtype=torch.int32, device=DEVICE),
                longest=max(pos) + 1, scale=D ** -0.5,
                sinks=_normal(g, H) if case["sinks"] else None,
                slopes=torch.exp2(-8.0 * torch.arange(1, H + 1, device=DEVICE) / H).float() if case["slopes"] else None)


def _prepare_rules(case, g):
    B, V, n = case["rows"], case["vocab"], case["biases"]
    state = dict(case=case, logits=_normal(g, B, V) * 3.0, slots=torch.randperm(B + 2, generator=g, device=DEVICE)[:B].int(), history=None,
                 penalties=None, bias_range=None, bias_ids=None, bias_values=None, masks=None, mask_rows=None)
    if case["penalties"]:
        # a text's tokens: few of them often; some tokens of the vocabulary in the prompt
        common = torch.rand(B + 2, V, generator=g, device=DEVICE)
        counts = torch.where(common > 0.998, 1 + (common * 1e6).long() % 9, torch.zeros((), dtype=torch.long, device=DEVICE))
        prompt = torch.rand(B + 2, V, generator=g, device=DEVICE) > 0.995
        state["history"] = (counts - 32768 * prompt).to(torch.int16)
        state["penalties"] = torch.stack([1.0 + torch.rand(B, generator=g, device=DEVICE), torch.rand(B, generator=g, device=DEVICE),
                                          torch.rand(B, generator=g, device=DEVICE) * 0.5], dim=1).contiguous()
    if n:
        # two lists that the rows of two requests' answers share
        ids = torch.stack([torch.randperm(V, generator=g, device=DEVICE)[:n] for _ in range(2)])
        state["bias_ids"] = ids.reshape(-1).int()
        state["bias_values"] = _normal(g, 2 * n) * 5.0
        which = torch.arange(B, device=DEVICE) % 2
        state["bias_range"] = torch.stack([which * n, (which + 1) * n], dim=1).int().contiguous()
    if case["masked"]:
        M = 24                                                                            # states of a grammar
        allowed = torch.rand(M, V, generator=g, device=DEVICE) < case["allowed"]
        words = -(-V // 32)
        bits = torch.zeros(M, words * 32, dtype=torch.int64, device=DEVICE)
        bits[:, :V] = allowed
        packed = (bits.view(M, words, 32) << torch.arange(32, device=DEVICE)).sum(dim=2)
        state["masks"] = torch.where(packed >= 2 ** 31, packed - 2 ** 32, packed).int()
        rows = torch.randint(0, M, (B,), generator=g, device=DEVICE)
        rows[B // 2:: 7] = -1                                                             # some requests have no grammar
        if B == 1:
            rows[:] = 5
        state["mask_rows"] = rows.int()
    return state


def _prepare_note(case, g):
    S, V, n = case["slots"], case["vocab"], case["tokens"]
    counts = torch.randint(0, 3, (S, V), generator=g, device=DEVICE)
    # a text's tokens: the smaller the id, the more often
    tokens = (torch.rand(n, generator=g, device=DEVICE) ** 4 * V).int().clamp_(max=V - 1)
    return dict(case=case, history=counts.to(torch.int16), tokens=tokens, slots=torch.randint(0, S, (n,), generator=g, device=DEVICE).int())


def _prepare_tables(case, g):
    B, W = case["rows"], case["width"]
    new = _ints(case["new"])
    lens = torch.tensor([new[b % len(new)] for b in range(B)], dtype=torch.int32, device=DEVICE)
    room = W * PAGE - lens
    starts = torch.minimum(torch.randint(case["low"], case["high"] + 1, (B,), generator=g, device=DEVICE).int(), room.int())
    held = (starts + PAGE - 1) // PAGE
    need = (starts + lens + PAGE - 1) // PAGE
    n_slots = B + 3
    slots = torch.randperm(n_slots, generator=g, device=DEVICE)[:B].int()
    n_pages = n_slots * W
    order = torch.randperm(n_pages, generator=g, device=DEVICE).int()
    resident = torch.full((n_slots, W), -1, dtype=torch.int32, device=DEVICE)
    there = torch.arange(W, device=DEVICE)[None, :] < held[:, None]
    resident[slots.long()] = torch.where(there, order[:B * W].view(B, W), resident[slots.long()])
    fresh = order[B * W:][:int((need - held).sum())].contiguous()
    T = int(lens.sum())
    empty = lambda *shape: torch.full(shape, -7, dtype=torch.int32, device=DEVICE)       # noqa: E731
    return dict(case=case, slots=slots, starts=starts, lens=lens, held=held.int(), pages=fresh, resident=resident,
                out=(empty(T), empty(T), empty(B + 1), empty(T), empty(B, W)))


# ---------------------------------------------------------------------------- one pass

def run(state):
    if own:
        return _own(state)
    return {"attention": _plain_attention, "rules": _plain_rules, "note": _plain_note, "tables": _plain_tables}[state["case"]["op"]](state)


def _own(state):
    from pico_engine.ops import kernels
    s, c = state, state["case"]
    if c["op"] == "attention":
        return kernels.attention_shared(s["qkv"], s["qkv"].shape[1], c["heads"], c["kv_heads"], c["dim"], s["k"], s["v"], s["table"], s["table"].shape[1],
                                        s["pos"], s["row"], s["groups"], c["window"] or None, s["scale"], s["longest"], keep_first=c["keep_first"],
                                        slopes=s["slopes"], sinks=s["sinks"])
    if c["op"] == "rules":
        return kernels.adjust_logits(s["logits"], s["slots"], s["history"], s["penalties"], s["bias_range"], s["bias_ids"], s["bias_values"],
                                     s["masks"], s["mask_rows"])
    if c["op"] == "note":
        return kernels.note_tokens(s["history"], s["slots"], s["tokens"], prompt=True)
    return kernels.step_tables(s["slots"], s["starts"], s["lens"], s["held"], s["pages"], s["resident"], *s["out"]) + (s["resident"],)


def _plain_attention(s):
    c = s["case"]
    H, G, D, T = c["heads"], c["kv_heads"], c["dim"], s["pos"].shape[0]
    pages = s["table"].clamp(min=0).long()
    L = pages.shape[1] * PAGE
    keys = s["k"][pages].float().permute(0, 2, 1, 3, 4).reshape(T, G, L, D)
    values = s["v"][pages].float().permute(0, 2, 1, 3, 4).reshape(T, G, L, D)
    q = s["qkv"][:, :H * D].float().view(T, G, H // G, D)
    scores = (q @ keys.transpose(2, 3)) * s["scale"]                                     # [T, G, H / G, L]
    j, pos = torch.arange(L, device=DEVICE)[None, :], s["pos"].long()[:, None]
    seen = j <= pos
    if c["window"]:
        seen = seen & ((j > pos - c["window"]) | (j < c["keep_first"]))
    if s["slopes"] is not None:
        scores = scores - s["slopes"].view(1, G, H // G, 1) * (pos - j).float()[:, None, None, :]
    scores = torch.where(seen[:, None, None, :], scores, NONE)
    top = scores.amax(dim=3, keepdim=True)
    w = torch.exp(scores - top)
    total = w.sum(dim=3, keepdim=True)
    if s["sinks"] is not None:
        total = total + torch.exp(s["sinks"].view(1, G, H // G, 1) - top)
    out = (w @ values) / total
    return out.reshape(T, H * D).to(torch.bfloat16)


def _plain_rules(s):
    z, V = s["logits"], s["case"]["vocab"]
    if s["history"] is not None:
        h = s["history"][s["slots"].long()].int()
        count = h & 0x7FFF
        r, presence, frequency = (s["penalties"][:, i:i + 1] for i in range(3))
        z = torch.where(h != 0, torch.where(z > 0, z / r, z * r), z)
        z = torch.where(count > 0, z - (presence + count.float() * frequency), z)
    if s["bias_ids"] is not None:
        n = s["bias_ids"].shape[0] // 2
        lists = torch.zeros(2, V, device=DEVICE).scatter_add(1, s["bias_ids"].long().view(2, n), s["bias_values"].view(2, n))
        z = z + lists[(s["bias_range"][:, 0] // n).long()]
    if s["masks"] is not None:
        v = torch.arange(V, device=DEVICE)
        words = s["masks"][s["mask_rows"].clamp(min=0).long()][:, v // 32]
        allowed = ((words >> (v % 32)) & 1).bool() | (s["mask_rows"] < 0)[:, None]
        z = torch.where(allowed, z, NONE)
    return z


def _plain_note(s):
    V = s["history"].shape[1]
    at = s["slots"].long() * V + s["tokens"].long()
    flat = s["history"].view(-1)
    flat[at] = flat[at] | -32768
    return s["history"]


def _plain_tables(s):
    lens, starts, held, (B, W) = s["lens"].long(), s["starts"].long(), s["held"].long(), s["out"][4].shape
    T = s["out"][0].shape[0]
    first = torch.cumsum(lens, 0) - lens
    row = torch.repeat_interleave(torch.arange(B, device=DEVICE), lens, output_size=T)
    pos = starts[row] + torch.arange(T, device=DEVICE) - first[row]
    fresh = torch.clamp((starts + lens + PAGE - 1) // PAGE - held, min=0)
    before = torch.cumsum(fresh, 0) - fresh
    w = torch.arange(W, device=DEVICE)[None, :]
    taken = (w >= held[:, None]) & (w < (held + fresh)[:, None])
    at = (before[:, None] + w - held[:, None]).clamp(0, max(s["pages"].shape[0] - 1, 0))
    known = s["resident"][s["slots"].long()]
    table = torch.where(taken, s["pages"][at], known) if s["pages"].shape[0] else known
    s["resident"][s["slots"].long()] = table
    page = table[row, pos // PAGE]
    places = torch.where(page >= 0, page * PAGE + (pos % PAGE).int(), -1)
    there = w < (held + fresh)[:, None]
    row_first = torch.cat([first, lens.sum()[None]])
    return pos.int(), row.int(), row_first.int(), places.int(), torch.where(there, table, -1), s["resident"]


# ---------------------------------------------------------------------------- what a pass cannot do without

def work(case):
    if case["op"] == "attention":
        H, G, D = case["heads"], case["kv_heads"], case["dim"]
        rows, window, keep = _lengths(case), case["window"], case["keep_first"]
        pairs = keys = 0
        least = {}
        for i, s, n in rows:
            pos = s + n - 1
            lo = max(0, pos - window + 1) if window else 0
            kept = min(keep, lo)
            pairs += pos + 1 - lo + kept
            keys += pos + 1 - max(lo, s) + max(0, kept - s)                            # a row's own keys
            seen = max(0, s - lo) + min(kept, s)
            least[i] = max(least.get(i, 0), seen)
        keys += sum(least.values())                                                     # and each prompt's once
        return {"bytes": 4.0 * keys * G * D + 4.0 * len(rows) * H * D, "flops": 4.0 * pairs * H * D}
    if case["op"] == "rules":
        B, V = case["rows"], case["vocab"]
        a_row = 8.0 * V + (2.0 * V if case["penalties"] else 0.0)
        return {"bytes": B * a_row + 16.0 * case["biases"] + (min(B, 24) * V / 8.0 if case["masked"] else 0.0), "flops": float(B) * V}
    if case["op"] == "note":
        return {"bytes": case["tokens"] * (8.0 + 4.0), "flops": float(case["tokens"])}
    B, W, new = case["rows"], case["width"], _ints(case["new"])
    T = sum(new[b % len(new)] for b in range(B))
    return {"bytes": 20.0 * B + 12.0 * T + 8.0 * B * W, "flops": float(T)}


# ---------------------------------------------------------------------------- the definitions in 64 bits

def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "attention":
        return _exact_attention(s)
    if case["op"] == "rules":
        return _exact_rules(s)
    if case["op"] == "note":
        seen = torch.zeros(s["history"].shape, dtype=torch.bool, device=DEVICE)
        seen[s["slots"].long(), s["tokens"].long()] = True
        return (s["history"].long() - 32768 * seen).to(torch.int16)                      # counts alone before
    return _exact_tables(s)


def _exact_attention(s):
    c = s["case"]
    H, G, D = c["heads"], c["kv_heads"], c["dim"]
    out = []
    for t, pos in enumerate(s["pos"].tolist()):
        places = torch.arange(pos + 1, device=DEVICE)
        if c["window"]:
            places = places[(places > pos - c["window"]) | (places < c["keep_first"])]
        page = s["table"][t].long()[places // PAGE]
        k, v = (s[x][page, :, places % PAGE].double() for x in ("k", "v"))              # [n, G, D]
        for h in range(H):
            x = (k[:, h * G // H] @ s["qkv"][t, h * D:(h + 1) * D].double()) * s["scale"]
            if s["slopes"] is not None:
                x = x - s["slopes"][h].double() * (pos - places)
            if s["sinks"] is not None:
                x = torch.cat([x, s["sinks"][h].double()[None]])
            p = torch.softmax(x, 0)[:places.shape[0]]
            out.append(p @ v[:, h * G // H])
    return torch.cat(out).view(len(s["pos"]), H * D)


def _exact_rules(s):
    z = s["logits"].double()
    V = z.shape[1]
    for b in range(z.shape[0]):
        if s["history"] is not None:
            h = s["history"][int(s["slots"][b])].long()
            r, presence, frequency = s["penalties"][b].double().tolist()
            count = torch.where(h < 0, h + 32768, h)
            z[b] = torch.where(h == 0, z[b], torch.where(z[b] > 0, z[b] / r, z[b] * r))
            z[b] -= torch.where(count > 0, presence + count * frequency, torch.zeros((), device=DEVICE, dtype=torch.double))
        if s["bias_ids"] is not None:
            a, e = s["bias_range"][b].tolist()
            z[b].index_add_(0, s["bias_ids"][a:e].long(), s["bias_values"][a:e].double())
        if s["masks"] is not None and int(s["mask_rows"][b]) >= 0:
            words = s["masks"][int(s["mask_rows"][b])].long() & 0xFFFFFFFF
            bits = torch.stack([(words >> i) & 1 for i in range(32)], dim=1).reshape(-1)[:V]
            z[b][bits == 0] = NONE
    return z


def _exact_tables(s):
    pos, row, first, places = [], [], [0], []
    resident, pages = s["resident"].tolist(), s["pages"].tolist()
    width = s["out"][4].shape[1]
    tables = []
    for b, (slot, start, n, held) in enumerate(zip(*(s[k].tolist() for k in ("slots", "starts", "lens", "held")))):
        entries = resident[slot]
        for w in range(held, -(-(start + n) // PAGE)):
            entries[w] = pages.pop(0)
        for p in range(start, start + n):
            pos.append(p)
            row.append(b)
            places.append(entries[p // PAGE] * PAGE + p % PAGE)
        first.append(len(pos))
        have = max(held, -(-(start + n) // PAGE))
        tables.append(entries[:have] + [-1] * (width - have))
    return tuple(torch.tensor(x, dtype=torch.int32, device=DEVICE) for x in (pos, row, first, places, tables, resident))
