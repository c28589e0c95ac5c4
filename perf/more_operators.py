"""What a long context costs: keys and values appended to a cache of 4 bits with the position rotation on the way, attention over that cache
for single tokens and for prompts, the bounds of a page's keys, and attention over the pages that a cheap score selects.

A case is a plain dict.  ``op`` says which operator it goes through:

* ``"append"``: queries and keys rotated, keys and values stored in 4 bits (the outputs: the queries, and what the stored codes stand for);
* ``"decode"``: attention of one token a row over the cache;
* ``"prompt"``: attention of several tokens a row, which stand at the end of what the row holds;
* ``"bounds"``: the least and the greatest key, channel by channel, of the pages that a step has filled;
* ``"selected"``: the pages that a token's heads can score highest, and attention over these.

``own`` false: elementary torch operations.  ``own`` true: the library's kernels.

How a cache of 4 bits holds a head's row: its channels in groups of 32, x of a group (bfloat16) as a code c of 0 to 15 that stands for
mid + step * (c - 7.5), with mid = (max + min) / 2 and step = (max - min) / 15 rounded to bfloat16, c = floor((x - mid) / step) + 8 (8 where step is 0).
"""
from __future__ import annotations

import math

import torch

own = False

DEVICE = "cuda"
PAGE = 64
# (query heads, key/value heads, head size) of qwen2.5-0.5b, of design_compare's middle size, of qwen2.5-7b
SMALL, MIDDLE, LARGE = (14, 2, 64), (16, 4, 128), (28, 4, 128)
LONGEST = 32768                     # positions of the largest configuration
NONE = float("-inf")
CHUNK = 2048                        # blocks that are packed or unpacked at a time


def _text(values):
    return ",".join(str(int(v)) for v in values)


def _ints(text):
    return [int(v) for v in text.split(",")]


def _case(op, size, **more):
    heads, kv_heads, dim = size
    return dict(op=op, heads=heads, kv_heads=kv_heads, dim=dim, **more)


def listed():
    return [
        # the token of one conversation: nothing but latency
        dict(_case("append", SMALL, starts="1000", lens="1", rotated=True), name="append_1"),
        # the prompts of a batch, one of them the next piece of a longer one
        dict(_case("append", LARGE, starts="0,0,4071,0", lens="5001,1807,700,33", rotated=True), name="append_prompts"),
        # one conversation on the benchmark's context
        dict(_case("decode", SMALL, rows=1, low=4000, high=4096, window=0), name="decode_1"),
        # a full batch of conversations near the longest context
        dict(_case("decode", SMALL, rows=64, low=20000, high=32700, window=0), name="decode_64_long"),
        # the larger model, many conversations from short to long
        dict(_case("decode", LARGE, rows=200, low=1, high=6000, window=0), name="decode_200_large"),
        # a sliding window
        dict(_case("decode", MIDDLE, rows=32, low=100, high=8000, window=2000), name="decode_window"),
        # unequal prompts, one of them the next piece of a longer one
        dict(_case("prompt", LARGE, starts="0,0,4071,0", lens="5001,1807,700,33", window=0), name="prompts_large"),
        # a question behind a long document
        dict(_case("prompt", SMALL, starts="15937", lens="500", window=0), name="prompt_question"),
        # the pages that the prompts of a batch have filled
        dict(_case("bounds", LARGE, starts="0,0,4071,0", lens="5001,1807,700,33"), name="bounds_prompts"),
        # a decode step of which some rows end a page
        dict(_case("bounds", SMALL, starts=_text(1000 + 29 * b for b in range(64)), lens=_text([1] * 64)), name="bounds_64"),
        # one conversation on the longest context, 32 pages of about 510 read
        dict(_case("selected", SMALL, rows=1, low=32000, high=32700, keep=32), name="selected_1"),
        # a batch of the larger model, 64 pages of about 410 read
        dict(_case("selected", LARGE, rows=48, low=20000, high=32700, keep=64), name="selected_48"),
    ]


def draw(rng):
    log = lambda a, b: int(round(math.exp(rng.uniform(math.log(a), math.log(b)))))      # noqa: E731
    kind = rng.choice(["append", "append", "decode", "decode", "decode", "prompt", "prompt", "bounds", "selected", "selected"])
    size = rng.choice([SMALL, SMALL, MIDDLE, LARGE, LARGE, (8, 8, 64), (32, 2, 128), (24, 8, 128)])
    G, D = size[1], size[2]
    if kind in ("append", "prompt", "bounds"):
        if rng.random() < 0.5 and kind != "prompt":
            rows = log(1, 256)
            lens, starts = [1] * rows, [rng.randint(0, 2000) for _ in range(rows)]
        else:
            rows = rng.choice([1, 1, 2, 3, 5])
            lens = [log(2, 6000 // rows) for _ in range(rows)]
            starts = [rng.choice([0, 0, rng.randint(1, 8000)]) for _ in range(rows)]
        if kind == "append":
            return _case(kind, size, starts=_text(starts), lens=_text(lens), rotated=rng.random() < 0.8)
        if kind == "bounds":
            return _case(kind, size, starts=_text(starts), lens=_text(lens))
        return _case(kind, size, starts=_text(starts), lens=_text(lens), window=rng.choice([0, 0, log(10, 5000)]))
    rows, high = log(1, 64 if kind == "selected" else 256), log(64, 32700)
    while rows * high * G * D > 64 * LONGEST * 2 * 64:
        rows, high = max(1, rows - 1 - rows // 8), max(64, high - high // 16)
    low = rng.choice([1, max(1, high // 2)])
    if kind == "selected":
        return _case(kind, size, rows=rows, low=low, high=high, keep=log(2, 128))
    return _case(kind, size, rows=rows, low=low, high=high, window=rng.choice([0, 0, 0, log(10, 4000)]))


# ---------------------------------------------------------------------------- how a page lies in memory

def _turn(words, by):
    """32-bit words (int64) turned left."""
    return ((words << by) | (words >> (32 - by))) & 0xFFFFFFFF if by else words


def _to_words(codes):
    """codes [..., 4 (i), 2 (hi)] of 0 to 15 as int32 words [...]: an element's sign at bit 15 + 16 hi and its magnitude at bits 4 to 6 + 16 hi, turned left by 4 i."""
    k = torch.where(codes >= 8, codes - 8, 7 - codes)
    field = ((codes < 8).long() << 15) | (k << 4)
    pair = field[..., 0] | (field[..., 1] << 16)
    word = pair[..., 0]
    for i in range(1, 4):
        word = word | _turn(pair[..., i], 4 * i)
    return torch.where(word >= 2 ** 31, word - 2 ** 32, word).int()


def _from_words(words):
    """What the elements of int32 words [...] are, in steps from the middle: float32 [..., 4, 2]."""
    w = words.long() & 0xFFFFFFFF
    out = []
    for i in range(4):
        r = _turn(w, (32 - 4 * i) % 32)
        for hi in (0, 16):
            k = ((r >> (4 + hi)) & 7).float() + 0.5
            out.append(torch.where((r >> (15 + hi)) & 1 == 1, -k, k))
    return torch.stack(out, dim=-1).unflatten(-1, (4, 2))


def _code(x):
    """codes (int64), steps and middles (bfloat16) of rows x [..., D]."""
    x = x.float().unflatten(-1, (-1, 32))
    hi, lo = x.amax(dim=-1, keepdim=True), x.amin(dim=-1, keepdim=True)
    fifteen = torch.full((), 15.0, device=x.device)
    mid, step = ((hi + lo) * 0.5).to(torch.bfloat16), ((hi - lo) / fifteen).to(torch.bfloat16)
    c = torch.floor((x - mid.float()) / step.float()) + 8
    c = torch.where(step.float() == 0, torch.full((), 8.0, device=x.device), c).clamp(0, 15)
    return c.flatten(-2).long(), step[..., 0], mid[..., 0]


def _stands_for(codes, step, mid):
    c = codes.float().unflatten(-1, (-1, 32))
    return (mid.float()[..., None] + step.float()[..., None] * (c - 7.5)).flatten(-2)


def _pack(keys, values):
    """Blocks uint8 [n, 80 D] of keys and values [n, 64, D]."""
    n, _, D = keys.shape
    h, nb = D // 64, D // 32
    c, ks, km = _code(keys)
    kw = _to_words(c.view(n, 64, nb, 4, 4, 2).transpose(2, 3))
    c, vs, vm = _code(values)
    c = c.view(n, 4, 2, 4, 2, h, 2, 8, 2, 2)                                              # tile, half, t, hi; h, w2, g, w1, nib
    vw = _to_words(c.permute(0, 1, 5, 7, 3, 6, 8, 2, 9, 4).reshape(n, 4, h, 8, 4, 4, 4, 2))
    km = torch.stack([ks, km], dim=2)
    vm = torch.stack([x.view(n, 4, 2, 4, 2, nb).permute(0, 1, 5, 3, 2, 4) for x in (vs, vm)], dim=2)
    return torch.cat([x.contiguous().view(n, -1).view(torch.uint8) for x in (kw, vw, km, vm)], dim=1)


def _unpack(blocks):
    """What blocks [n, 80 D] hold: keys and values float32 [n, 64, D]."""
    n, D = blocks.shape[0], blocks.shape[1] // 80
    h, nb = D // 64, D // 32
    part = lambda a, b, t: blocks[:, a * D: b * D].contiguous().view(t)                   # noqa: E731
    k = _from_words(part(0, 32, torch.int32).view(n, 64, 4, nb)).transpose(2, 3).reshape(n, 64, nb, 32)
    v = _from_words(part(32, 64, torch.int32).view(n, 4, h, 8, 4, 2, 2)).unflatten(-2, (2, 2))   # tile, h, g, t, w2, w1, half, nib, hi
    v = v.permute(0, 1, 7, 4, 9, 2, 5, 3, 6, 8).reshape(n, 64, nb, 32)
    km = part(64, 72, torch.bfloat16).view(n, 64, 2, nb).float()
    vm = part(72, 80, torch.bfloat16).view(n, 4, 2, nb, 4, 2, 2).permute(0, 1, 5, 4, 6, 2, 3).reshape(n, 64, 2, nb).float()
    return tuple((m[:, :, 1, :, None] + m[:, :, 0, :, None] * x).reshape(n, 64, D) for x, m in ((k, km), (v, vm)))


# ---------------------------------------------------------------------------- inputs

def _generator(seed):
    return torch.Generator(device=DEVICE).manual_seed(int(seed))


def _normal(g, *shape, dtype=torch.float32):
    return torch.randn(*shape, generator=g, device=DEVICE, dtype=torch.float32).to(dtype)


def _spread(case):
    """The position of each row's token, from ``low`` to ``high`` tokens held."""
    n = case["rows"]
    return [case["low"] - 1 + (case["high"] - case["low"]) * ((j * 37 + 5) % (n + 2)) // (n + 1) for j in range(n)]


def _rows(case):
    """(first position, tokens) of every row."""
    if "rows" in case:
        return [(p, 1) for p in _spread(case)]
    return list(zip(_ints(case["starts"]), _ints(case["lens"])))


def _fill(g, pool, kv_heads, dim):
    """Keys with channels that stand out and pages that lie together, values of unit size."""
    offset = _normal(g, kv_heads, 1, dim) * (1.0 + 4.0 * (torch.arange(dim, device=DEVICE) % 16 == 3))
    flat = pool.view(-1, pool.shape[-1])
    for at in range(0, pool.shape[0], CHUNK // kv_heads):
        n = min(CHUNK // kv_heads, pool.shape[0] - at)
        keys = _normal(g, n, kv_heads, 64, dim) + 0.5 * _normal(g, n, kv_heads, 1, dim) + offset
        values = _normal(g, n, kv_heads, 64, dim)
        flat[at * kv_heads: (at + n) * kv_heads] = _pack(keys.to(torch.bfloat16).view(-1, 64, dim), values.to(torch.bfloat16).view(-1, 64, dim))


def _angles(dim, positions):
    inverse = 1.0 / (1e6 ** (torch.arange(0, dim, 2, dtype=torch.float32) / dim))
    angles = torch.arange(positions, dtype=torch.float32)[:, None] * inverse[None, :]
    return angles.cos().to(DEVICE).contiguous(), angles.sin().to(DEVICE).contiguous()


def _runs(rows, most=128):
    """Runs of at most 128 tokens of a row: row, first token, tokens, position; those that see most first."""
    out, at = [], 0
    for b, (start, n) in enumerate(rows):
        out.extend((b, at + off, min(most, n - off), start + off) for off in range(0, n, most))
        at += n
    return sorted(out, key=lambda r: -(r[3] + r[2]))


def prepare(case, seed):
    g = _generator(seed)
    op, H, G, D = case["op"], case["heads"], case["kv_heads"], case["dim"]
    rows = _rows(case)
    T = sum(n for _, n in rows)
    held = [-(-(s + n) // PAGE) for s, n in rows]
    total = sum(held) + 3
    order = torch.randperm(total, generator=g, device=DEVICE).int()                       # pages lie anywhere in the pool
    table = torch.full((len(rows), max(held)), -1, dtype=torch.int32)
    at, host = 0, order.cpu()
    for b, p in enumerate(held):
        table[b, :p] = host[at:at + p]
        at += p
    pos = torch.cat([torch.arange(s, s + n) for s, n in rows])
    row = torch.repeat_interleave(torch.arange(len(rows)), torch.tensor([n for _, n in rows]))
    pool = torch.zeros(total, G, 80 * D, dtype=torch.uint8, device=DEVICE)
    _fill(g, pool, G, D)
    state = dict(case=case, pool=pool, table=table.to(DEVICE), pos=pos.int().to(DEVICE), row=row.int().to(DEVICE), scale=D ** -0.5,
                 longest=max(s + n for s, n in rows))
    if op == "bounds":
        state["bounds"] = torch.zeros(total, G, 2, D, dtype=torch.bfloat16, device=DEVICE)
        return state
    qkv = _normal(g, T, (H + 2 * G) * D)
    if op == "append":
        offset = _normal(g, G * D) * (1.0 + 4.0 * (torch.arange(G * D, device=DEVICE) % 16 == 3))
        qkv[:, H * D: (H + G) * D] += offset                                              # keys with channels that stand out
        state["cos"], state["sin"] = _angles(D, state["longest"]) if case["rotated"] else (None, None)
    state["qkv"] = (qkv * 1.5).to(torch.bfloat16)                                         # queries at the front of wider rows
    if op == "prompt":
        state["runs"] = torch.tensor(_runs(rows), dtype=torch.int32, device=DEVICE)
    if op == "selected":
        bounds = torch.zeros(total, G, 2, D, dtype=torch.bfloat16, device=DEVICE)
        for i in range(0, total, CHUNK // G):
            k = _unpack(pool[i: i + CHUNK // G].flatten(0, 1))[0]
            bounds[i: i + CHUNK // G] = torch.stack([k.amin(dim=1), k.amax(dim=1)], dim=1).view(-1, G, 2, D).to(torch.bfloat16)
        state["bounds"] = bounds
    return state


# ---------------------------------------------------------------------------- one pass

def run(state):
    if own:
        return _own(state)
    return {"append": _plain_append, "decode": _plain_attention, "prompt": _plain_attention, "bounds": _plain_bounds,
            "selected": _plain_selected}[state["case"]["op"]](state)


def _own(s):
    from pico_engine.ops import kernels
    c = s["case"]
    H, G, D, W = c["heads"], c["kv_heads"], c["dim"], s["table"].shape[1]
    if c["op"] == "append":
        q = kernels.store_int4(s["qkv"], H, G, D, s["cos"], s["sin"], s["pos"], s["row"], s["pool"], s["table"], W)
        return (q,) + kernels.load_int4(s["pool"], G, D, s["pos"], s["row"], s["table"], W)
    if c["op"] == "decode":
        return kernels.attention_int4(s["qkv"], s["qkv"].shape[1], H, G, D, s["pool"], s["table"], W, s["pos"], s["row"], c["window"] or None,
                                      s["scale"], s["longest"])
    if c["op"] == "prompt":
        return kernels.attention_int4_prompt(s["qkv"], s["qkv"].shape[1], H, G, D, s["pool"], s["table"], W, s["runs"], s["pos"].shape[0],
                                             c["window"] or None, s["scale"])
    if c["op"] == "bounds":
        return kernels.page_bounds(s["pool"], G, D, s["pos"], s["row"], s["table"], W, s["bounds"])
    pages = kernels.select_pages(s["qkv"], s["qkv"].shape[1], H, G, D, s["bounds"], s["table"], W, s["pos"], s["row"], c["keep"], s["longest"])
    return (kernels.attention_int4_selected(s["qkv"], s["qkv"].shape[1], H, G, D, s["pool"], pages, s["scale"]), pages.table, pages.pos)


def _plain_append(s):
    c = s["case"]
    H, G, D = c["heads"], c["kv_heads"], c["dim"]
    T = s["qkv"].shape[0]
    x = s["qkv"].view(T, H + 2 * G, D)
    q, k, v = x[:, :H], x[:, H:H + G], x[:, H + G:]
    if s["cos"] is not None:
        cos, sin = s["cos"][s["pos"].long()][:, None], s["sin"][s["pos"].long()][:, None]

        def turned(x, cos, sin):
            a, b = x[..., :D // 2], x[..., D // 2:]
            return torch.cat([a * cos - b * sin, a * sin + b * cos], dim=-1).float().to(torch.bfloat16)

        q, k = turned(q.float(), cos, sin), turned(k.double(), cos.double(), sin.double())        # (64 bits next to a code's border)
    return (q.reshape(T, H * D).contiguous(),) + tuple(_stands_for(*_code(x)) for x in (k, v))


def _of_row(s, b, pages):
    """Keys and values float32 [kv heads, positions, D] of the pages ``pages`` of row b."""
    G, D = s["case"]["kv_heads"], s["case"]["dim"]
    k, v = _unpack(s["pool"][s["table"][b, pages].long()].flatten(0, 1))
    return tuple(x.view(-1, G, 64, D).transpose(0, 1).reshape(G, -1, D) for x in (k, v))


def _attend(q, k, v, at, j, scale, window):
    """q [n, H, D] at positions ``at``, keys and values [G, L, D] at positions ``j``: float32 [n, H, D]."""
    n, H, D = q.shape
    G = k.shape[0]
    scores = (q.view(n, G, H // G, D).permute(1, 2, 0, 3).reshape(G, -1, D) @ k.transpose(1, 2)).view(G, H // G, n, -1) * scale
    seen = j[None, :] <= at[:, None]
    if window:
        seen = seen & (j[None, :] > at[:, None] - window)
    scores = torch.where(seen, scores, NONE)
    w = torch.exp(scores - scores.amax(dim=3, keepdim=True))
    out = (w.view(G, -1, w.shape[3]) @ v).view(G, H // G, n, D) / w.sum(dim=3, keepdim=True)
    return out.permute(2, 0, 1, 3).reshape(n, H, D)


def _plain_attention(s):
    c = s["case"]
    H, D, window = c["heads"], c["dim"], c["window"]
    q = s["qkv"][:, :H * D].float().view(-1, H, D)
    out, at = [], 0
    for b, (start, n) in enumerate(_rows(c)):
        first = max(0, start - window + 1) // PAGE if window else 0
        pages = torch.arange(first, (start + n - 1) // PAGE + 1, device=DEVICE)
        k, v = _of_row(s, b, pages)
        j = (pages[:, None] * PAGE + torch.arange(PAGE, device=DEVICE)).flatten()
        for i in range(0, n, 256):
            m = min(256, n - i)
            out.append(_attend(q[at + i: at + i + m], k, v, s["pos"][at + i: at + i + m], j, s["scale"], window))
        at += n
    return torch.cat(out).reshape(-1, H * D).to(torch.bfloat16)


def _plain_bounds(s):
    c = s["case"]
    G, D = c["kv_heads"], c["dim"]
    ends = s["pos"] % PAGE == PAGE - 1
    pages = s["table"][s["row"][ends].long(), s["pos"][ends].long() // PAGE].long()
    if pages.shape[0]:
        k = _unpack(s["pool"][pages].flatten(0, 1))[0]
        s["bounds"][pages] = torch.stack([k.amin(dim=1), k.amax(dim=1)], dim=1).view(-1, G, 2, D).to(torch.bfloat16)
    return s["bounds"]


def _plain_selected(s):
    c = s["case"]
    H, G, D, keep = c["heads"], c["kv_heads"], c["dim"], c["keep"]
    q = s["qkv"][:, :H * D].view(-1, H, D)
    outs, tables, places = [], [], []
    for t, (p, _) in enumerate(_rows(c)):
        last = p // PAGE
        pages = torch.arange(last + 1, device=DEVICE)[None, :].expand(G, -1)
        if last + 1 > keep:
            x = q[t].view(G, H // G, D).double()                                          # (64 bits: scores of two pages may lie close together)
            up, down = x.clamp(min=0).sum(dim=1), x.clamp(max=0).sum(dim=1)
            lo, hi = s["bounds"][s["table"][t, 1:last].long()].double().unbind(dim=2)      # [pages, G, D]
            score = (up * hi + down * lo).sum(dim=2).t()
            best = torch.sort(score, dim=1, descending=True, stable=True)[1][:, :max(keep - 2, 0)] + 1
            ends = [torch.zeros(G, 1, dtype=torch.long, device=DEVICE)] if keep > 1 else []
            pages = torch.sort(torch.cat(ends + [best, torch.full((G, 1), last, device=DEVICE)], dim=1), dim=1)[0]
        n = pages.shape[1]
        physical = s["table"][t].long()[pages]                                            # [G, n]
        head = torch.arange(G, device=DEVICE)[:, None]
        k, v = (x.view(G, n * 64, D) for x in _unpack(s["pool"][physical, head].flatten(0, 1)))
        j = (pages[:, :, None] * PAGE + torch.arange(PAGE, device=DEVICE)).view(G, -1)
        scores = (q[t].float().view(G, H // G, D) @ k.transpose(1, 2)) * s["scale"]
        scores = torch.where((j <= p)[:, None, :], scores, NONE)
        w = torch.exp(scores - scores.amax(dim=2, keepdim=True))
        outs.append(((w @ v) / w.sum(dim=2, keepdim=True)).reshape(1, H * D))
        block = torch.full((G, keep), -1, dtype=torch.int32, device=DEVICE)
        block[:, :n] = (physical * G + head).int()
        tables.append(block)
        places.extend([(n - 1) * PAGE + p % PAGE] * G)
    return torch.cat(outs).to(torch.bfloat16), torch.cat(tables), torch.tensor(places, dtype=torch.int32, device=DEVICE)


# ---------------------------------------------------------------------------- what a pass cannot do without

def work(case):
    H, G, D = case["heads"], case["kv_heads"], case["dim"]
    rows = _rows(case)
    T = sum(n for _, n in rows)
    if case["op"] == "append":
        stored = 1.25 * T * G * D
        turned = 4.0 * D * len({p for s, n in rows for p in range(s, s + n)}) if case["rotated"] else 0.0
        return {"bytes": 2.0 * T * (H + 2 * G) * D + turned + 2.0 * T * H * D + 2 * stored + 8.0 * T * G * D, "flops": 3.0 * T * (H + G) * D}
    if case["op"] == "bounds":
        ended = sum((s + n) // PAGE - s // PAGE for s, n in rows)
        return {"bytes": 44.0 * D * ended * G + 8.0 * T, "flops": 128.0 * D * ended * G + T}          # (every token's position is looked at)
    if case["op"] == "selected":
        seen = [(min(p // PAGE + 1, case["keep"]), max(0, p // PAGE - 1) if p // PAGE + 1 > case["keep"] else 0) for p, _ in rows]
        keys = sum((n - 1) * PAGE + p % PAGE + 1 for (n, _), (p, _) in zip(seen, rows))
        return {"bytes": 1.25 * 2 * keys * G * D / 2 + 4.0 * D * G * sum(n for _, n in seen) + 4.0 * T * H * D,
                "flops": 4.0 * keys * H * D + 4.0 * D * G * sum(n for _, n in seen)}
    window = case["window"]
    pairs = keys = 0
    for s, n in rows:
        pairs += sum(min(p + 1, window) if window else p + 1 for p in range(s, s + n))
        keys += s + n - (max(0, s - window + 1) if window else 0)
    return {"bytes": 1.25 * keys * G * D + 4.0 * T * H * D, "flops": 4.0 * pairs * H * D}


# ---------------------------------------------------------------------------- the definitions in 64 bits

def exact(case, seed):
    s = prepare(case, seed)
    return {"append": _exact_append, "decode": _exact_attention, "prompt": _exact_attention, "bounds": _exact_bounds, "selected": _exact_selected}[case["op"]](s)


def _exact_group(x):
    """What a row x [D] of bfloat16 is stored as."""
    out = []
    for a in range(0, x.shape[-1], 32):
        y = x[..., a: a + 32].double()
        top, bottom = y.max(dim=-1, keepdim=True)[0], y.min(dim=-1, keepdim=True)[0]
        mid, step = ((top + bottom) / 2).to(torch.bfloat16).double(), ((top - bottom) / 15).to(torch.bfloat16).double()
        level = torch.floor((y - mid) / torch.where(step > 0, step, 1.0)).clamp(-8, 7) + 0.5
        out.append(mid + step * level)
    return torch.cat(out, dim=-1)


def _exact_append(s):
    c = s["case"]
    H, G, D = c["heads"], c["kv_heads"], c["dim"]
    x = s["qkv"].double().view(-1, H + 2 * G, D)
    if s["cos"] is not None:
        angle = torch.complex(s["cos"].double(), s["sin"].double())[s["pos"].long()][:, None]
        z = torch.complex(x[:, :H + G, :D // 2].contiguous(), x[:, :H + G, D // 2:].contiguous()) * angle
        x = torch.cat([torch.cat([z.real, z.imag], dim=-1), x[:, H + G:]], dim=1)
    keys = x[:, H:H + G].float().to(torch.bfloat16)                                       # the cache codes keys of the model's type
    return x[:, :H].reshape(-1, H * D), _exact_group(keys), _exact_group(x[:, H + G:])


def _places(D):
    """Where key and value of (position, channel) lie in a block: for each of the two the word, the bit of the sign, that of the magnitude, the index of
    the step and that of the middle (in bfloat16 numbers from the block's start), all [64, D]."""
    p, d = torch.arange(64)[:, None].expand(64, D), torch.arange(D)[None, :].expand(64, D)
    nb = D // 32
    b, c = d // 32, d % 32
    i, hi = c % 8 // 2, c % 2
    keys = (p * (D // 8) + c // 8 * nb + b, (16 * hi + 15 + 4 * i) % 32, (16 * hi + 4 + 4 * i) % 32, 32 * D + p * 2 * nb + b, 32 * D + p * 2 * nb + nb + b)
    tile, r = p // 16, p % 16
    half, t, hi = r // 8, r % 8 // 2, r % 2
    m = 2 * b + c % 4 // 2
    i = 2 * half + c % 2
    word = 8 * D + ((tile * (D // 64) + m // 4) * 32 + c // 4 * 4 + t) * 4 + m % 4
    step = 36 * D + (tile * 2 * nb + b) * 16 + 4 * t + 2 * half + hi
    values = (word, (16 * hi + 15 + 4 * i) % 32, (16 * hi + 4 + 4 * i) % 32, step, step + 16 * nb)
    return [[x.to(DEVICE) for x in side] for side in (keys, values)]


def _exact_unpack(blocks):
    """float64 keys and values [n, 64, D]."""
    D = blocks.shape[1] // 80
    words, numbers = blocks.contiguous().view(torch.int32).long(), blocks.contiguous().view(torch.bfloat16).double()
    out = []
    for word, sign, place, step, mid in _places(D):
        # a magnitude's three bits may pass the word's end
        k = sum((((words[:, word] >> ((place + j) % 32)) & 1) << j) for j in range(3))
        level = (k.double() + 0.5) * (1 - 2 * ((words[:, word] >> sign) & 1)).double()
        out.append(numbers[:, mid] + numbers[:, step] * level)
    return out


def _exact_row(s, b, last, first=0):
    G, D = s["case"]["kv_heads"], s["case"]["dim"]
    ks, vs = [], []
    for at in range(first, last + 1, 128):
        pages = s["table"][b, at: min(at + 128, last + 1)].long()
        k, v = _exact_unpack(s["pool"][pages].flatten(0, 1))
        ks.append(k.view(-1, G, 64, D))
        vs.append(v.view(-1, G, 64, D))
    return torch.cat(ks), torch.cat(vs)                                                   # [pages, G, 64, D]


def _exact_attention(s):
    c = s["case"]
    H, G, D = c["heads"], c["kv_heads"], c["dim"]
    q, at, out = s["qkv"][:, :H * D].double().view(-1, H, D), 0, []
    for b, (start, n) in enumerate(_rows(c)):
        first = max(0, start - c["window"] + 1) // PAGE if c["window"] else 0
        k, v = _exact_row(s, b, (start + n - 1) // PAGE, first)
        of = torch.empty(n, H, D, dtype=torch.float64, device=DEVICE)
        for h in range(H):
            kh, vh = k[:, h * G // H].reshape(-1, D), v[:, h * G // H].reshape(-1, D)
            for i in range(0, n, 512):
                x = q[at + i: at + min(n, i + 512), h] @ kh.t() * s["scale"]
                away = torch.arange(start + i, start + i + x.shape[0], device=DEVICE)[:, None] - torch.arange(first * PAGE, first * PAGE + kh.shape[0], device=DEVICE)
                x[(away < 0) | (away >= (c["window"] or 1 << 40))] = NONE
                of[i: i + 512, h] = torch.softmax(x, dim=1) @ vh
        out.append(of)
        at += n
    return torch.cat(out).view(-1, H * D)


def _exact_bounds(s):
    out = s["bounds"].double()
    for p, b in zip(s["pos"].tolist(), s["row"].tolist()):
        if p % PAGE == PAGE - 1:
            page = int(s["table"][b, p // PAGE])
            k = _exact_unpack(s["pool"][page])[0]
            out[page, :, 0], out[page, :, 1] = k.min(dim=1)[0], k.max(dim=1)[0]
    return out


def _exact_selected(s):
    c = s["case"]
    H, G, D, keep = c["heads"], c["kv_heads"], c["dim"], c["keep"]
    outs, tables, places = [], [], []
    for t, p in enumerate(s["pos"].tolist()):
        row, last = s["table"][t].tolist(), p // PAGE
        ends = s["bounds"][s["table"][t, :last].long()].double()                           # [pages, G, 2, D]
        for h in range(G):
            q = s["qkv"][t, h * (H // G) * D: (h + 1) * (H // G) * D].double().view(-1, D)
            pages = list(range(last + 1))
            if last + 1 > keep:
                # the most that a key between the bounds can score, added over the heads
                most = torch.maximum(q[:, None] * ends[None, :, h, 0], q[:, None] * ends[None, :, h, 1]).sum(dim=(0, 2)).tolist()
                middle = sorted(range(1, last), key=lambda j: (-most[j], j))[: max(keep - 2, 0)]
                pages = sorted(([0] if keep > 1 else []) + middle + [last])
            tables.append([row[j] * G + h for j in pages] + [-1] * (keep - len(pages)))
            places.append((len(pages) - 1) * PAGE + p % PAGE)
            blocks = s["pool"].view(-1, 80 * D)[torch.tensor(tables[-1][:len(pages)], device=DEVICE)]
            k, v = (x.reshape(-1, D)[: places[-1] + 1] for x in _exact_unpack(blocks))
            outs.append(torch.softmax(q @ k.t() * s["scale"], dim=1) @ v)
    return (torch.cat(outs).view(-1, H * D), torch.tensor(tables, dtype=torch.int32, device=DEVICE), torch.tensor(places, dtype=torch.int32, device=DEVICE))
