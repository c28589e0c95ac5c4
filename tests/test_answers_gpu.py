"""Several answers to one prompt: attention over shared pages, rules on logits and the tables of a step, each kernel alone against the plain
formulas in 64 bits.

Attention's bound, entry by entry: probabilities are rounded to bfloat16 for the product with the values (half a step, 2^-8 of each, so at most 2^-8 of
sum p |v|) and so is the result (2^-8 of |o|); what float32 adds (scores of up to 128 terms, 2^-24 each, times scores of at most 40: 3e-4 of a
probability in the worst case) is covered by the tenth that the bound leaves on top."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

PAGE = 64


@pytest.fixture(scope="module")
def K():
    from pico_engine.ops import kernels
    return kernels


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def randn(*shape, seed=0, scale=1.0):
    return torch.randn(*shape, generator=gen(seed), device="cuda") * scale


def ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


# ---------------------------------------------------------------------------- attention

class Answers:
    """Groups of rows with shared and own pages, scattered over a pool whose rows nobody has written hold ``rubbish``."""

    def __init__(self, nh, nkv, hd, groups, seed, rubbish=0.0, extra=24):
        """groups: [(shared positions, [own tokens of each row])]"""
        g = torch.Generator().manual_seed(seed)
        self.nh, self.nkv, self.hd = nh, nkv, hd
        need = sum(s // PAGE + sum(-(-n // PAGE) for n in own) for s, own in groups)
        order = torch.randperm(need + 5, generator=g).tolist()
        self.k = torch.full((need + 5, nkv, PAGE, hd), rubbish, dtype=torch.bfloat16, device="cuda")
        self.v = self.k.clone()
        table, self.pos, members = [], [], []
        for i, (s, own) in enumerate(groups):
            prompt = [order.pop() for _ in range(s // PAGE)]
            for n in own:
                table.append(prompt + [order.pop() for _ in range(-(-n // PAGE))])
                self.pos.append(s + n - 1)
            members.append((len(own), s, own.index(min(own))))
        for t, (row, p) in enumerate(zip(table, self.pos)):
            for w, page in enumerate(row):
                used = min(PAGE, p + 1 - w * PAGE)
                self.k[page, :, :used] = randn(nkv, used, hd, seed=seed * 7919 + page).bfloat16()
                self.v[page, :, :used] = randn(nkv, used, hd, seed=seed * 104729 + page).bfloat16()
        self.T, self.members = len(table), members
        self.width = max(len(r) for r in table) + 2
        self.table = ints([r + [-1] * (self.width - len(r)) for r in table])
        self.rows = randn(self.T, nh * hd + extra, seed=seed + 1, scale=1.5).bfloat16()      # queries inside wider rows
        self.sinks, self.slopes = randn(nh, seed=seed + 2), torch.exp2(-8.0 * torch.arange(1, nh + 1, device="cuda") / nh)

    def run(self, K, window=None, keep=0, sinks=False, slopes=False, groups=None, out=None, bound=None, together=True):
        return K.attention_shared(self.rows, self.rows.shape[1], self.nh, self.nkv, self.hd, self.k, self.v, self.table, self.width, ints(self.pos),
                                  torch.arange(self.T, dtype=torch.int32, device="cuda"), K.shared_groups(self.members, "cuda") if groups is None else groups,
                                  window, self.hd ** -0.5, bound or max(self.pos) + 1, out=out, keep_first=keep,
                                  slopes=self.slopes if slopes else None, sinks=self.sinks if sinks else None, together=together)

    def want(self, window=None, keep=0, sinks=False, slopes=False):
        """(result, sum p |v|) in 64 bits."""
        out, mass = [], []
        for t, pos in enumerate(self.pos):
            j = torch.arange(pos + 1, device="cuda")
            if window:
                j = j[(j > pos - window) | (j < keep)]
            page = self.table[t].long()[j // PAGE]
            k, v = (x[page, :, j % PAGE].double().repeat_interleave(self.nh // self.nkv, dim=1) for x in (self.k, self.v))      # [n, nh, hd]
            s = torch.einsum("hd,nhd->hn", self.rows[t, :self.nh * self.hd].double().view(self.nh, self.hd), k) * self.hd ** -0.5
            if slopes:
                s = s - self.slopes.double()[:, None] * (pos - j)
            if sinks:
                s = torch.cat([s, self.sinks.double()[:, None]], dim=1)
            p = torch.softmax(s, dim=1)[:, :len(j)]
            out.append(torch.einsum("hn,nhd->hd", p, v))
            mass.append(torch.einsum("hn,nhd->hd", p, v.abs()))
        return torch.stack(out).view(self.T, -1), torch.stack(mass).view(self.T, -1)


def agree(got, want, mass):
    assert torch.isfinite(got).all()
    over = (got.double() - want).abs() / (2.0 ** -8 * 1.1 * (want.abs() + mass) + 1e-30)
    assert float(over.max()) <= 1.0, float(over.max())


SHARED = [  # nh, nkv, hd, [(shared positions, own tokens)]
    (14, 2, 64, [(64, [1])]),                                                   # one row, one page
    (14, 2, 64, [(0, [1, 70, 64, 65])]),                                        # rows that share nothing
    (14, 2, 64, [(576, [1, 64, 65, 90])]),                                      # an odd number of pages
    (14, 2, 64, [(4096, [1 + 7 * i for i in range(40)])]),                      # several tiles of rows
    (28, 4, 128, [(192, [3, 1]), (0, [130]), (1024, [5, 700, 64, 1, 9]), (64, [2]), (1984, [1] * 20)]),
    (16, 4, 128, [(2048 + 64, [30] * 33)]),
    (3, 3, 64, [(640, [2] * 130), (64, [1])]),                                  # a query head a key head: 128 rows a tile, and two more
    (40, 1, 128, [(320, [4, 8, 100, 1])]),                                      # three rows a tile
    (128, 1, 64, [(128, [1, 66])]),                                             # one row a tile
    (5, 1, 128, [(20032, [9, 1, 1500])]),                                       # long
    (2, 2, 64, [(64 * (1 + i % 4), [1 + i % 3] * (1 + i % 5)) for i in range(70)]),      # many small groups
    (2, 1, 128, [(64 * (i % 4), [1 + i % 70] * (2 + i % 5)) for i in range(110)]),       # more than 320 rows
    (4, 4, 64, [(64, [3] * 300), (0, [40]), (192, [65] * 29)]),
]


@pytest.mark.parametrize("nh,nkv,hd,groups", SHARED)
@pytest.mark.parametrize("rubbish", [0.0, float("nan")])
def test_attention_shared(K, nh, nkv, hd, groups, rubbish):
    a = Answers(nh, nkv, hd, groups, seed=nh + hd, rubbish=rubbish)
    got = a.run(K)
    K.check_status("cuda")
    agree(got, *a.want())


MASKS = [  # window, keep_first, sinks, slopes
    (300, 0, False, False), (64, 0, False, False), (1, 0, True, False), (500, 4, True, False), (129, 200, False, True), (None, 0, True, True),
    (100000, 0, False, False), (700, 64, True, True),
]


@pytest.mark.parametrize("window,keep,sinks,slopes", MASKS)
@pytest.mark.parametrize("nh,nkv,hd,groups", [SHARED[2], SHARED[4], (4, 2, 64, [(1024, [1, 40, 200, 700]), (0, [300]), (128, [64, 63])])])
def test_attention_shared_under_masks(K, nh, nkv, hd, groups, window, keep, sinks, slopes):
    """Windows that leave some rows of a group nothing of the prompt, end inside a page, or let its first keys stand; sinks; distance slopes."""
    a = Answers(nh, nkv, hd, groups, seed=nh + hd)
    got = a.run(K, window, keep, sinks, slopes)
    K.check_status("cuda")
    agree(got, *a.want(window, keep, sinks, slopes))


def test_attention_shared_where_the_window_has_given_pages_back(K):
    """Prompt pages behind every row's window are no longer in the tables."""
    a = Answers(8, 2, 64, [(1024, [300, 310, 333])], seed=5)
    want = a.want(window=400)
    gone = (1024 + 300 - 1 - 400 + 1) // PAGE
    a.table[:, :gone] = -1
    agree(a.run(K, window=400), *want)
    K.check_status("cuda")


def test_attention_shared_scores_of_any_size(K):
    """Scores of about a hundred, whose maximum moves up and down from page to page."""
    for hd in (64, 128):
        a = Answers(14, 2, hd, [(2048, [1, 5, 64, 100, 7])], seed=hd)
        for w, page in enumerate(a.table[0, :32].tolist()):
            a.k[page] *= 1 + w % 7
        a.rows *= 3
        agree(a.run(K), *a.want())
    K.check_status("cuda")


def test_attention_shared_equals_each_row_alone(K):
    """Whether rows are read together or one by one makes no difference beyond the bound, and a repeated call none at all."""
    a = Answers(14, 2, 64, [(1280, [1, 30, 64, 65, 200]), (64, [5, 6])], seed=3)
    want = a.want()
    alone = K.shared_groups([(1, 0, 0)] * a.T, "cuda")
    agree(a.run(K, groups=alone), *want)
    first = a.run(K)
    for _ in range(3):
        assert torch.equal(a.run(K), first)
    agree(a.run(K, together=False), *want)                               # (the decode kernel, every row by itself)
    assert torch.equal(a.run(K, together=None), a.run(K, together=False))      # what little rows share here does not pay
    assert torch.equal(a.run(K, bound=30000), a.run(K, bound=30000))
    K.check_status("cuda")


@pytest.mark.parametrize("window,keep", [(2000, 4), (None, 0)])
def test_attention_shared_when_memory_is_slow(K, window, keep):
    """Keys and values that come from DRAM, late and in any order, call after call without a pause: the same bits every time.  (Such calls once
    had results of a tile that were taken before its last products were done.)"""
    a = Answers(32, 8, 128, [(2496, [1 + 61 * i % 1500 for i in range(24)]), (960, [1 + 97 * i % 700 for i in range(8)])], seed=6)
    want = a.want(window=window, keep=keep, sinks=True)
    flush = torch.empty(2 ** 28, dtype=torch.uint8, device="cuda")       # more than L2 holds
    first = a.run(K, window, keep, sinks=True)
    agree(first, *want)
    wrong = torch.zeros((), device="cuda")
    for _ in range(400):
        flush.zero_()
        for _ in range(2):
            wrong += (a.run(K, window, keep, sinks=True) != first).any()
    assert int(wrong) == 0
    K.check_status("cuda")


def test_attention_shared_reads_no_further_than_the_table(K):
    """Positions and shared pages beyond a row of the table: what the row names is read."""
    a = Answers(14, 2, 64, [(192, [64, 128]), (128, [64])], seed=8)
    want = a.want()
    a.table = a.table[:, :5].contiguous()                                # (the second row's pages fill it)
    a.width = 5
    a.pos[1] += 64 * 40
    a.pos[2] += 64 * 2 + 5
    agree(a.run(K), *want)
    groups = K.shared_groups(a.members, "cuda")
    groups[:2, 2] = 64 * 100                                             # the first group's rows name two pages of their own behind the three: those are not shared
    a.run(K, groups=groups)
    K.check_status("cuda")


@pytest.mark.parametrize("nh,nkv,hd", [(2, 1, 64), (4, 2, 128)])
def test_attention_shared_of_as_many_rows_as_it_takes(K, nh, nkv, hd):
    groups = [(64 * (1 + i % 3), [1 + (i + j) % 66 for j in range(16)]) for i in range(32)] + [(128, [1 + j % 5 for j in range(512)])]
    a = Answers(nh, nkv, hd, groups, seed=hd)
    assert a.T == K.SHARED_MAX_ROWS
    agree(a.run(K), *a.want())
    agree(a.run(K, window=90, keep=3), *a.want(window=90, keep=3))
    K.check_status("cuda")


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("value", [float("nan"), float("inf"), -float("inf")])
def test_attention_shared_of_what_is_no_number(K, hd, value):
    """A key that is no number in a group's prompt reaches all of its rows' heads of that key head, one in a row's own part that row's, a value its column;
    nothing else moves by a bit."""
    a = Answers(6, 2, hd, [(640, [3, 70, 130]), (192, [5, 9])], seed=hd)
    agree(a.run(K), *a.want())
    before = a.run(K).view(5, 2, 3, hd).clone()
    for pool, page, rows in ((a.k, a.table[0, 4], [0, 1, 2]), (a.k, a.table[1, 10], [1]), (a.v, a.table[3, 1], [3, 4]), (a.v, a.table[2, 12], [2])):
        keep = pool[page, 1].clone()
        pool[page, 1, 1] = value if pool is a.k else pool[page, 1, 1].index_fill(0, torch.tensor([5], device="cuda"), value)
        got = a.run(K).view(5, 2, 3, hd)
        pool[page, 1] = keep
        touched = torch.zeros(5, 2, 3, hd, dtype=torch.bool, device="cuda")
        touched[rows, 1] = True
        if pool is a.v:
            touched[..., :5] = touched[..., 6:] = False
        assert torch.equal(got[~touched], before[~touched])
        assert not torch.isfinite(got[touched]).any() if value != value or pool is a.v else True
    agree(a.run(K), *a.want())
    K.check_status("cuda")


def test_attention_shared_in_two_captured_graphs(K):
    """Two graphs captured one after the other and replayed in turn, on two streams at once, beside eager calls: each has scratch of its own."""
    a, b = (Answers(14, 2, 64, [(64 * n, [1 + 5 * i for i in range(m)])], seed=n) for n, m in ((30, 20), (100, 9)))
    outs, graphs = [], []
    args = []
    for x in (a, b):
        fixed = dict(groups=K.shared_groups(x.members, "cuda"))
        pos, row = ints(x.pos), torch.arange(x.T, dtype=torch.int32, device="cuda")
        call = lambda x=x, f=fixed, pos=pos, row=row: K.attention_shared(x.rows, x.rows.shape[1], x.nh, x.nkv, x.hd, x.k, x.v, x.table, x.width, pos, row,
                                                                       f["groups"], None, x.hd ** -0.5, max(x.pos) + 1, together=True)
        args.append(call)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            call()
        torch.cuda.current_stream().wait_stream(side)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(call())
        graphs.append(g)
    wants = [a.want(), b.want()]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    for _ in range(5):
        for s, g in zip(streams, graphs):
            with torch.cuda.stream(s):
                g.replay()
        eager = args[0]()
    torch.cuda.synchronize()
    for o, w in zip(outs + [eager], wants + [wants[0]]):
        agree(o, *w)
    K.check_status("cuda")


# ---------------------------------------------------------------------------- rules on logits

def rules_case(B, V, seed, history=True, biases=0, masks=True, twice=False):
    g = gen(seed)
    c = dict(logits=torch.randn(B, V, generator=g, device="cuda") * 4)
    if history:
        h = torch.randint(0, 4, (B + 3, V), generator=g, device="cuda") * (torch.rand(B + 3, V, generator=g, device="cuda") < 0.3)
        h[:, V // 2] = 32767
        h = h - 32768 * (torch.rand(B + 3, V, generator=g, device="cuda") < 0.2)
        c.update(history=h.to(torch.int16), slots=torch.randperm(B + 3, generator=g, device="cuda")[:B].int(),
                 penalties=torch.rand(B, 3, generator=g, device="cuda") + 0.3)
    if biases:
        ids = torch.randint(0, V, (3, biases), generator=g, device="cuda")
        if twice:
            ids[:, biases // 2:] = ids[:, :biases - biases // 2]
        c.update(bias_ids=ids.reshape(-1).int(), bias_values=torch.randn(3 * biases, generator=g, device="cuda"))
        which = torch.arange(B, device="cuda") % 4                       # every fourth row has none
        c["bias_range"] = torch.stack([which * biases, torch.where(which == 3, which, which + 1) * biases], dim=1).int().contiguous()
    if masks:
        allowed = torch.rand(5, V, generator=g, device="cuda") < 0.3
        allowed[3] = False                                               # leaves nothing
        allowed[4] = True
        c.update(masks=pack(allowed), mask_rows=(torch.arange(B, device="cuda") % 6 - 1).int())
        c["allowed"] = allowed
    return c


def pack(allowed):
    M, V = allowed.shape
    words = -(-V // 32)
    bits = torch.zeros(M, words * 32, dtype=torch.int64, device="cuda")
    bits[:, :V] = allowed
    w = (bits.view(M, words, 32) << torch.arange(32, device="cuda")).sum(dim=2)
    return torch.where(w >= 2 ** 31, w - 2 ** 32, w).int()


def rules_want(c):
    """The result in 64 bits and the size of the numbers that went into it."""
    z = c["logits"].double()
    size = z.abs()
    V = z.shape[1]
    if "history" in c:
        h = c["history"][c["slots"].long()].long()
        count = h % 32768
        r, presence, frequency = (c["penalties"][:, i:i + 1].double() for i in range(3))
        z = torch.where(h != 0, torch.where(z > 0, z / r, z * r), z)
        size = z.abs()
        off = torch.where(count > 0, presence + count * frequency, 0.0)
        z, size = z - off, size + off.abs()
    if "bias_ids" in c:
        for b, (a, e) in enumerate(c["bias_range"].tolist()):
            z[b].index_add_(0, c["bias_ids"][a:e].long(), c["bias_values"][a:e].double())
            size[b].index_add_(0, c["bias_ids"][a:e].long(), c["bias_values"][a:e].double().abs())
    if "masks" in c:
        rows = c["mask_rows"].long()
        z = torch.where(c["allowed"][rows.clamp(min=0)] | (rows < 0)[:, None], z, float("-inf"))
    return z, size


def adjust(K, c, **more):
    return K.adjust_logits(c["logits"], *(c.get(k) for k in ("slots", "history", "penalties", "bias_range", "bias_ids", "bias_values", "masks", "mask_rows")), **more)


def rules_agree(got, want, size):
    """A handful of float32 operations, each off by half a step (2^-24) of at most the size of its numbers: eight of them are more than there are
    (a quotient, a product and sum, a difference, and biases that come to no more than six)."""
    assert torch.equal(torch.isinf(got), torch.isinf(want)) and not torch.isnan(got).any()
    live = torch.isfinite(want)
    assert bool((((got.double() - want).abs() <= 8 * 2.0 ** -24 * size + 1e-37) | ~live).all())


@pytest.mark.parametrize("B,V", [(1, 1), (3, 31), (7, 33), (1, 4096), (2, 50257), (13, 2047), (5, 2049), (4, 8200), (64, 1000), (3, 151936)])
@pytest.mark.parametrize("kind", ["penalties", "masks", "biases", "twice", "all"])
def test_adjust_logits(K, B, V, kind):
    c = rules_case(B, V, seed=B + V, history=kind in ("penalties", "all"), masks=kind in ("masks", "all"),
                   biases=0 if kind in ("penalties", "masks") else min(V, 37), twice=kind == "twice")
    kept = c["logits"].clone()
    want, size = rules_want(c)
    got = adjust(K, c)
    rules_agree(got, want, size)
    assert torch.equal(c["logits"], kept)
    again = adjust(K, c, out=c["logits"])                                # in place: the same bits
    assert again is c["logits"] and torch.equal(again, got)


def test_adjust_logits_of_values_that_are_not_finite(K):
    """Infinities and numbers that are none: masked places are -inf, whatever stood there; others follow the formula."""
    c = rules_case(6, 300, seed=1, biases=5)
    c["logits"][:, ::7] = float("nan")
    c["logits"][:, 1::7] = float("inf")
    c["logits"][:, 2::7] = float("-inf")
    c["logits"][:, 3::7] = torch.finfo(torch.float32).min
    got = adjust(K, c)
    rows = c["mask_rows"].long()
    allowed = c["allowed"][rows.clamp(min=0)] | (rows < 0)[:, None]
    assert bool((got[~allowed] == float("-inf")).all())
    assert torch.equal(torch.isnan(got), torch.isnan(c["logits"]) & allowed)
    assert bool((got[:, 1::7][allowed[:, 1::7]] == float("inf")).all())


def test_adjust_logits_many_biases(K):
    """Lists as long as the vocabulary and longer, with tokens many times over, added in the list's order: the same bits every time."""
    V, n = 5000, 12000
    c = rules_case(3, V, seed=9, history=False, masks=False)
    c["bias_ids"] = (torch.rand(n, generator=gen(2), device="cuda") ** 3 * V).int().clamp_(max=V - 1)
    c["bias_values"] = randn(n, seed=3)
    c["bias_range"] = ints([[0, n], [100, 100], [5000, 5001]])
    got = adjust(K, c)
    z, size = rules_want(c)
    many = torch.zeros(3, V, device="cuda", dtype=torch.double)
    for b, (a, e) in enumerate(c["bias_range"].tolist()):
        many[b] = torch.bincount(c["bias_ids"][a:e].long(), minlength=V)
    assert bool(((got.double() - z).abs() <= (many + 2) * 2.0 ** -24 * size + 1e-37).all())
    for _ in range(3):
        assert torch.equal(adjust(K, c), got)


def test_adjust_logits_outside_the_tables(K):
    """Slots, mask rows and bias tokens that are outside the tables change nothing."""
    c = rules_case(4, 100, seed=4, biases=3)
    c["slots"][1] = 1000
    c["slots"][2] = -1
    c["mask_rows"][:] = ints([-1, 5, 99, -7])
    c["bias_ids"][:] = ints([100, -1, 2 ** 30] * 3)
    c["bias_range"][3] = ints([-5, 10 ** 9])
    got = adjust(K, c)
    assert torch.equal(got[1:3], c["logits"][1:3]) and torch.isfinite(got).all()


def test_adjust_logits_of_a_view(K):
    """Rows that start on a 4-byte boundary only."""
    for V in (1000, 1001):
        c = rules_case(3, V, seed=V, biases=8)
        want, size = rules_want(c)
        wide = torch.empty(3 * V + 1, device="cuda")
        logits, out = wide[1:].view(3, V), torch.empty(3 * V + 3, device="cuda")[3:].view(3, V)
        logits.copy_(c["logits"])
        c["logits"] = logits
        rules_agree(adjust(K, c, out=out), want, size)


def test_adjust_logits_by_an_automatons_states(K):
    """The mask of a slot's state in the place of one named by the row: the same results; states and slots outside the tables have no mask."""
    c = rules_case(9, 1234, seed=2, biases=20)
    states = ints([-1, 3, 0, 2, 5, 1, 4, 2, 0, 1, -7, 3])
    c["slots"] = ints([11, 0, 12, -1, 4, 7, 6, 10, 2])
    n = len(states)
    c["history"] = c["history"][:n] if c["history"].shape[0] >= n else None
    assert c["history"] is not None
    named = ints([int(states[s]) if 0 <= s < n else -1 for s in c["slots"].tolist()])
    want = K.adjust_logits(c["logits"], c["slots"], c["history"], c["penalties"], c["bias_range"], c["bias_ids"], c["bias_values"], c["masks"], named)
    got = K.adjust_logits(c["logits"], c["slots"], c["history"], c["penalties"], c["bias_range"], c["bias_ids"], c["bias_values"], c["masks"], states=states)
    assert torch.equal(got, want)
    alone = K.adjust_logits(c["logits"], c["slots"], masks=c["masks"], states=states)
    assert torch.equal(alone, K.adjust_logits(c["logits"], masks=c["masks"], mask_rows=named))


def test_rules_then_the_choice(K):
    """As a step runs them: tokens noted, rules applied, the next token chosen; a row that its mask leaves one token gets that token, greedy or drawn."""
    B, V = 6, 2500
    history = torch.zeros(B + 1, V, dtype=torch.int16, device="cuda")
    slots, base = torch.arange(B, dtype=torch.int32, device="cuda"), randn(B, V, seed=1)
    penalties = torch.tensor([[1.0, 100.0, 0.0]], device="cuda").repeat(B, 1)
    chosen = []
    for step in range(5):
        z = K.adjust_logits(base, slots, history, penalties)
        t = K.argmax(z)
        K.note_tokens(history, slots, t)
        chosen.append(t.long())
    order = base.argsort(dim=1, descending=True)[:, :5].T                # the five best, one after the other
    assert torch.equal(torch.stack(chosen), order)
    allowed = torch.zeros(1, V, dtype=torch.bool, device="cuda")
    allowed[0, 1234] = True
    z = K.adjust_logits(base, masks=pack(allowed), mask_rows=torch.zeros(B, dtype=torch.int32, device="cuda"))
    steps = torch.zeros(B, dtype=torch.int32, device="cuda")
    for t in (K.argmax(z), K.sample(z, 0.7, 0, 1.0, 3, slots, steps), K.sample(z, 0.7, 5, 0.9, 3, slots, steps)):
        assert (t == 1234).all()


@pytest.mark.parametrize("n,V,N", [(1, 7, 1), (3, 100, 1000), (64, 50257, 20000), (5, 151936, 4096)])
@pytest.mark.parametrize("prompt", [False, True])
def test_note_tokens(K, n, V, N, prompt):
    g = gen(n + N)
    history = torch.randint(-32768, 32768, (n, V), generator=g, device="cuda").to(torch.int16)
    slots = torch.randint(0, n, (N,), generator=g, device="cuda").int()
    tokens = (torch.rand(N, generator=g, device="cuda") ** 4 * V).int().clamp_(max=V - 1)          # many of them many times
    h = history.long().cpu()
    sign, count = h < 0, h % 32768
    add = torch.zeros(n * V, dtype=torch.long).index_add_(0, slots.cpu().long() * V + tokens.cpu().long(), torch.ones(N, dtype=torch.long)).view(n, V)
    want = (count - 32768 * (sign | (add > 0))) if prompt else (torch.clamp(count + add, max=32767) - 32768 * sign)
    assert K.note_tokens(history, slots, tokens, prompt=prompt) is history
    assert torch.equal(history.long().cpu(), want)


def test_note_tokens_outside_the_tables(K):
    history = torch.zeros(4, 50, dtype=torch.int16, device="cuda")
    K.note_tokens(history[1:3], ints([0, 1, 2, -1, 0, 1, 0]), ints([-1, 50, 3, 3, 2 ** 31 - 1, -2 ** 31, 7]))
    want = torch.zeros(4, 50, dtype=torch.int16)
    want[1, 7] = 1
    assert torch.equal(history.cpu(), want)


def test_note_tokens_moves_automata(K):
    """States follow their sequence's tokens in order, several in one call; what a state does not allow leads to -1, which stays."""
    S, V, n, N = 6, 40, 5, 300
    g = torch.Generator().manual_seed(1)
    transitions = torch.randint(-1, S, (S, V), generator=g).int()
    transitions[:, :30] = transitions[:, :30].clamp(min=0)
    states = torch.tensor([0, 3, -1, 5, 2], dtype=torch.int32)
    slots, tokens = torch.randint(0, n + 1, (N,), generator=g).int(), torch.randint(0, V, (N,), generator=g).int()
    for upto in (0, 1, 4, 40, N):
        want = states.tolist()
        for s, t in zip(slots[:upto].tolist(), tokens[:upto].tolist()):
            if s < n:
                want[s] = int(transitions[want[s], t]) if want[s] >= 0 else -1
        got = states.cuda()
        K.note_tokens(None, slots[:upto].cuda(), tokens[:upto].cuda(), states=got, transitions=transitions.cuda())
        assert got.tolist() == want, upto


# ---------------------------------------------------------------------------- the tables of a step

def tables_want(slots, starts, lens, held, pages, resident, width):
    pos, row, first, places, tables = [], [], [0], [], []
    resident, pages = [list(r) for r in resident], list(pages)
    for b, (s, start, n, h) in enumerate(zip(slots, starts, lens, held)):
        need = max(h, -(-(start + n) // PAGE))
        for w in range(h, need):
            resident[s][w] = pages.pop(0)
        for p in range(start, start + n):
            page = resident[s][p // PAGE]
            pos.append(p); row.append(b); places.append(page * PAGE + p % PAGE if page >= 0 else -1)
        first.append(len(pos))
        tables.append(resident[s][:need] + [-1] * (width - need))
    return pos, row, first, places, tables, resident


@pytest.mark.parametrize("B,width,lens", [
    (1, 1, [1]), (1, 8, [512]), (5, 9, [1]), (64, 40, [1]), (7, 40, [1, 64, 65, 0, 700, 63, 128]), (300, 16, [1, 3]), (2000, 4, [1]), (3, 600, [30000, 1, 5]),
])
@pytest.mark.parametrize("spare", [0, 3])
def test_step_tables(K, B, width, lens, spare):
    """Lengths of zero, one, whole pages and one more; rows that hold more pages than they need, and resident tables wider than the step's; what lies
    behind the last token stays as it was."""
    import random
    rng = random.Random(B + width + spare)
    lens = [lens[b % len(lens)] for b in range(B)]
    starts = [rng.choice([0, PAGE, rng.randint(0, width * PAGE)]) for _ in range(B)]
    starts = [min(s, width * PAGE - n) for s, n in zip(starts, lens)]
    held = [min(width, -(-s // PAGE) + rng.choice([0, 0, 1])) for s in starts]
    slots = rng.sample(range(B + 4), B)
    R = width + spare
    order = rng.sample(range((B + 4) * R), (B + 4) * R)
    resident = [[-1] * R for _ in range(B + 4)]
    for s, h in zip(slots, held):
        for w in range(h):
            resident[s][w] = order.pop() if rng.random() < 0.95 else -1            # (a window has given some back)
    fresh = [order.pop() for _ in range(sum(max(0, -(-(s + n) // PAGE) - h) for s, n, h in zip(starts, lens, held)))]
    want = tables_want(slots, starts, lens, held, fresh, resident, width)
    T = sum(lens)
    res = ints(resident)
    full = lambda *s: torch.full(s, -7, dtype=torch.int32, device="cuda")      # noqa: E731
    out = (full(T + spare), full(T + spare), full(B + 1), full(T + spare), full(B, width))
    got = K.step_tables(ints(slots), ints(starts), ints(lens), ints(held), ints(fresh), res, *out)
    assert all(a is b for a, b in zip(got, out))
    for name, a, w in zip(("pos", "row", "first", "places", "tables", "resident"), got + (res,), want):
        assert a[:len(w)].tolist() == w, name
    for a in (got[0], got[1], got[3]):
        assert a[T:].tolist() == [-7] * spare
    # the same step again, now with its pages in the resident table
    again = K.step_tables(ints(slots), ints(starts), ints(lens), ints([max(h, -(-(s + n) // PAGE)) for s, n, h in zip(starts, lens, held)]), ints([]), res,
                          *(full(*x.shape) for x in out))
    assert all(torch.equal(a, b) for a, b in zip(again, got)) and res.tolist() == want[5]


def test_step_tables_outside_the_tables(K):
    """Slots outside the resident table, rows longer than it, and too few pages give -1, and nothing else is written."""
    res = torch.arange(12, dtype=torch.int32, device="cuda").view(4, 3)
    full = lambda *s: torch.full(s, -7, dtype=torch.int32, device="cuda")      # noqa: E731
    out = K.step_tables(ints([0, 9, -1, 1]), ints([0, 0, 0, 150]), ints([1, 1, 1, 400]), ints([1, 1, 1, 2]), ints([77]), res[:2],
                        full(403), full(403), full(5), full(403), full(4, 3))
    assert out[3].tolist() == [0, -1, -1] + [77 * PAGE + p % PAGE for p in range(150, 192)] + [-1] * (550 - 192)
    assert out[4].tolist() == [[0, -1, -1], [-1, -1, -1], [-1, -1, -1], [3, 4, 77]]
    assert res.tolist() == [[0, 1, 2], [3, 4, 77], [6, 7, 8], [9, 10, 11]]
    assert out[2].tolist() == [0, 1, 2, 3, 403] and out[0][3:].tolist() == list(range(150, 550))
