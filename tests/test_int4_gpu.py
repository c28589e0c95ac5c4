"""A long context's cache: rows appended in 4 bits, attention over them, the bounds of pages and attention over selected ones, each kernel alone
against the plain form in 64 bits (``plain_int4``).

Codes, steps, middles and selected pages are equal to the plain form's.  Attention's bound, number by number (``plain_int4.attend``): a weight is rounded to bfloat16 for the product
(2^-8 of it at most, on |v|), its product with a value's step once more (2^-8, on the part of v that its code carries), and the result (2^-8 of it); a score's error moves its weight by as much."""
import pytest
import torch

import plain_int4 as plain

pytestmark = pytest.mark.gpu

PAGE = 64
HEADS = [(14, 2, 64), (28, 4, 128), (8, 8, 64), (32, 2, 128), (1, 1, 64), (20, 1, 128)]


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


class Paged:
    """Rows of ``lengths`` positions on pages anywhere in a pool, whose places that nobody has written hold ``rubbish``."""

    def __init__(self, H, G, D, lengths, seed, rubbish=None, extra=24):
        self.H, self.G, self.D, self.lengths = H, G, D, lengths
        held = [max(1, -(-n // PAGE)) for n in lengths]
        self.n_pages = sum(held) + 3
        order = torch.randperm(self.n_pages, generator=torch.Generator().manual_seed(seed)).tolist()
        self.width = max(held) + 2
        rows = []
        for p in held:
            rows.append([order.pop() for _ in range(p)])
        self.table = ints([r + [-1] * (self.width - len(r)) for r in rows])
        self.pages = rows
        keys = (randn(self.n_pages, G, 64, D, seed=seed + 1) + randn(G, 1, D, seed=seed + 2, scale=2.0)).bfloat16()
        values = randn(self.n_pages, G, 64, D, seed=seed + 3).bfloat16()
        if rubbish is not None:
            for r, n in zip(rows, lengths):
                if n % PAGE:
                    keys[r[-1], :, n % PAGE:] = rubbish
                    values[r[-1], :, n % PAGE:] = rubbish
        self.keys, self.values = keys, values
        self.pool = plain.pack(keys.view(-1, 64, D), values.view(-1, 64, D)).view(self.n_pages, G, 80 * D)
        self.q = randn(len(lengths), H * D + extra, seed=seed + 4, scale=1.5).bfloat16()
        self.scale = D ** -0.5

    def attention(self, K, pos, row, q=None, window=None, table=None, bound=None, out=None):
        q = self.q if q is None else q
        return K.attention_int4(q, q.shape[1], self.H, self.G, self.D, self.pool, self.table if table is None else table, self.width, ints(pos), ints(row), window,
                                self.scale, bound or max(max(pos), 0) + 1, out=out)

    def check(self, got, pos, row, q=None, window=None, table=None, halves=False):
        q = self.q if q is None else q
        table = self.table if table is None else table
        for t, (p, r) in enumerate(zip(pos, row)):
            n = p // PAGE + 1
            j = torch.arange(n * PAGE, device="cuda")
            seen = (j <= p) & ((j > p - window) if window else (j >= 0))
            there = table[r, :n] >= 0
            seen = seen & there.repeat_interleave(PAGE)
            blocks = self.pool[table[r, :n].clamp(min=0).long()]
            want, bound = plain.attend(q[t, :self.H * self.D].view(self.H, self.D), blocks, seen[None].expand(self.G, -1), self.scale, halves)
            off = (got[t].double().view(self.H, self.D) - want).abs()
            assert (off <= bound + 1e-30).all(), (t, p, float((off / (bound + 1e-30)).max()))


# ---------------------------------------------------------------------------- appending

def angles(D, n):
    a = torch.arange(n, dtype=torch.float32)[:, None] / 1e4 ** (torch.arange(0, D, 2, dtype=torch.float32) / D)
    return a.cos().cuda().contiguous(), a.sin().cuda().contiguous()


def append(K, p, qkv, starts, lens, cos=None, sin=None, pool=None, table=None):
    pos = [s + i for s, n in zip(starts, lens) for i in range(n)]
    row = [b for b, n in enumerate(lens) for _ in range(n)]
    q = K.store_int4(qkv, p.H, p.G, p.D, cos, sin, ints(pos), ints(row), p.pool if pool is None else pool, p.table if table is None else table, p.width)
    return q, pos, row


@pytest.mark.parametrize("H,G,D", HEADS)
@pytest.mark.parametrize("starts,lens", [([0], [1]), ([77], [1]), ([0, 15, 63, 100], [1, 1, 1, 1]), ([0, 5, 250], [130, 40, 17]), ([3], [700])])
def test_appended_rows(K, H, G, D, starts, lens):
    p = Paged(H, G, D, [s + n for s, n in zip(starts, lens)], 5)
    T, before = sum(lens), p.pool.clone()
    x = randn(T, H + 2 * G, D, seed=9, scale=1.3).bfloat16()
    cos, sin = angles(D, 1000)
    q, pos, row = append(K, p, x.view(T, -1), starts, lens, cos, sin)
    c, s = cos.double()[pos][:, None], sin.double()[pos][:, None]
    a, b = x[..., :D // 2].double(), x[..., D // 2:].double()
    turned, size = torch.cat([a * c - b * s, a * s + b * c], -1), torch.cat([(a * c).abs() + (b * s).abs(), (a * s).abs() + (b * c).abs()], -1)
    off = (q.double().view(T, H, D) - turned[:, :H]).abs()
    assert (off <= 2.0 ** -8 * turned[:, :H].abs() + 2.0 ** -22 * size[:, :H] + 1e-30).all()      # one rounding, and float32's
    want_k, want_v = plain.stands_for(turned[:, H:H + G].float().bfloat16()), plain.stands_for(x[:, H + G:])
    k, v = K.load_int4(p.pool, G, D, ints(pos), ints(row), p.table, p.width)
    assert torch.equal(k.double(), want_k.float().double()) and torch.equal(v.double(), want_v.float().double())
    # the plain form of the whole pool with these rows in it: nothing else has changed
    keys, values = plain.unpack(before.view(-1, 80 * D))[:2]
    after_k, after_v = (t.view(p.n_pages, G, 64, D) for t in plain.unpack(p.pool.view(-1, 80 * D))[:2])
    keys, values = keys.view(p.n_pages, G, 64, D).clone(), values.view(p.n_pages, G, 64, D).clone()
    for i, (at, r) in enumerate(zip(pos, row)):
        page = p.pages[r][at // PAGE]
        keys[page, :, at % PAGE], values[page, :, at % PAGE] = want_k[i], want_v[i]
    assert torch.equal(after_k, keys) and torch.equal(after_v, values)


@pytest.mark.parametrize("H,G,D", [(14, 2, 64), (4, 4, 128)])
def test_pieces_leave_the_same_bytes(K, H, G, D):
    n = 333
    p = Paged(H, G, D, [n], 3)
    x = randn(n, (H + 2 * G) * D, seed=1).bfloat16()
    cos, sin = angles(D, 400)
    whole, pieces = torch.zeros_like(p.pool), torch.zeros_like(p.pool)
    q, _, _ = append(K, p, x, [0], [n], cos, sin, whole)
    at, rows = 0, []
    for m in [1, 1, 13, 2, 16, 31, 1, 64, 100, 3, 101]:
        rows.append(append(K, p, x[at:at + m].contiguous(), [at], [m], cos, sin, pieces)[0])
        at += m
    assert at == n and torch.equal(whole, pieces) and torch.equal(q, torch.cat(rows))


@pytest.mark.parametrize("H,G,D", [(14, 2, 64), (4, 4, 128)])
def test_positions_with_gaps(K, H, G, D):
    """Tokens of a sequence whose positions leave some out: those of one word (positions two or one and eight apart of sixteen) stand anywhere in the call."""
    rows = [[4, 13], [4, 5, 12, 13, 20], [0, 1, 9], [3, 10, 11, 64, 66, 73, 75], list(range(0, 60, 3)), [5], [16, 18, 25, 27, 30]] * 6
    p = Paged(H, G, D, [80] * len(rows), 35)
    pos, row = [x for r in rows for x in r], [b for b, r in enumerate(rows) for _ in r]
    qkv = randn(len(pos), (H + 2 * G) * D, seed=36).bfloat16()
    want, got = p.pool.clone(), p.pool.clone()
    for i, (a, b) in enumerate(zip(pos, row)):
        K.store_int4(qkv[i:i + 1], H, G, D, None, None, ints([a]), ints([b]), want, p.table, p.width)
    for _ in range(3):
        K.store_int4(qkv, H, G, D, None, None, ints(pos), ints(row), got, p.table, p.width)
        assert torch.equal(got, want)
        got.copy_(p.pool)


def test_numbers_that_are_none_and_pages_that_are_not_there(K):
    H, G, D = 2, 2, 64
    p = Paged(H, G, D, [70, 70], 4)
    x = randn(4, H + 2 * G, D, seed=2).bfloat16()
    x[0, H, 3], x[1, H + G, 40], x[2, H + G + 1, 63] = float("nan"), float("inf"), float("-inf")
    x[1, H + 1, :32], x[1, H + 1, 0] = 3e38, -3e38                          # a spread that bfloat16 holds, a sum of the two that cancels
    x[2, H, :32], x[2, H, 5] = 3.3e38, 3.2e38                               # a sum that float32 does not hold
    x[3, H, 32:] = -2.5                                                     # all equal
    table = p.table.clone()
    table[1, 1] = -1
    before = p.pool.clone()
    q = K.store_int4(x.view(4, -1), H, G, D, None, None, ints([10, 11, 12, 66]), ints([0, 0, 0, 1]), p.pool, table, p.width)
    assert torch.equal(q.view(4, H, D), x[:, :H])
    k, v = K.load_int4(p.pool, G, D, ints([10, 11, 12, 66]), ints([0, 0, 0, 1]), table, p.width)
    assert torch.isnan(k[0, 0, :32]).all() and torch.isfinite(k[0, 0, 32:]).all()
    assert torch.isnan(v[1, 0, 32:]).all() and torch.isnan(v[2, 1, 32:]).all() and torch.isfinite(v[1, 0, :32]).all()
    assert torch.isnan(k[2, 0, :32]).all() and not torch.isnan(k[0, 1]).any()
    assert (k[3] == 0).all() and (v[3] == 0).all()                          # not stored: no page
    gone = p.pages[1][1]
    assert torch.equal(p.pool[gone], before[gone])
    q = K.store_int4(x.view(4, -1), H, G, D, None, None, ints([60, 61, 62, 63]), ints([0, 0, 0, 1]), p.pool, p.table, p.width)
    k, v = K.load_int4(p.pool, G, D, ints([63]), ints([1]), p.table, p.width)
    assert (k[0, 0, 32:] == -2.5).all()


# ---------------------------------------------------------------------------- attention

@pytest.mark.parametrize("H,G,D", HEADS)
@pytest.mark.parametrize("lengths", [[1], [2, 15, 16, 17, 63, 64, 65], [500, 1, 1029], [4100]])
def test_attention(K, H, G, D, lengths):
    p = Paged(H, G, D, lengths, 7 + H, rubbish=float("nan"))
    pos, row = [n - 1 for n in lengths], list(range(len(lengths)))
    p.check(p.attention(K, pos, row), pos, row)
    p.check(p.attention(K, pos, row, bound=1 << 21), pos, row)              # a launch for long contexts, whatever they are


@pytest.mark.parametrize("H,G,D", [(14, 2, 64), (16, 4, 128)])
@pytest.mark.parametrize("window", [1, 2, 63, 64, 65, 100, 1000])
def test_attention_under_a_window(K, H, G, D, window):
    lengths = [1, 64, 70, 300, 1300]
    p = Paged(H, G, D, lengths, 11)
    # what a window has left behind is no number, and pages of it are not there
    table = p.table.clone()
    for r, n in enumerate(lengths):
        table[r, :max(0, n - window) // PAGE] = -1
        first = max(0, n - window)
        if first % PAGE:
            page = p.pages[r][first // PAGE]
            p.keys[page, :, :first % PAGE] = float("inf")
            p.values[page, :, :first % PAGE] = float("nan")
    p.pool = plain.pack(p.keys.view(-1, 64, D), p.values.view(-1, 64, D)).view(p.n_pages, G, 80 * D)
    pos, row = [n - 1 for n in lengths], list(range(len(lengths)))
    for bound in (4000, 1 << 21):
        p.check(p.attention(K, pos, row, window=window, table=table, bound=bound), pos, row, window=window, table=table)


@pytest.mark.parametrize("H,G,D,rows,window", [(28, 4, 128, 48, 300), (14, 2, 64, 120, 1000), (20, 1, 128, 100, 130)])
def test_many_rows_under_a_window(K, H, G, D, rows, window):
    """Launches for as many pages as a window can lie on, short and long rows among them."""
    lengths = [1 + (b * 997) % 2600 for b in range(rows)]
    p = Paged(H, G, D, lengths, 13, rubbish=float("nan"))
    table = p.table.clone()
    for r, n in enumerate(lengths):
        table[r, :max(0, n - window) // PAGE] = -1
    pos, row, q = [n - 1 for n in lengths], list(range(rows)), p.q
    got = p.attention(K, pos, row, window=window, table=table)
    some = list(range(0, rows, 5))
    p.check(got[some], [pos[i] for i in some], some, q=q[some], window=window, table=table)


def test_several_tokens_of_a_row_and_rows_in_any_order(K):
    p = Paged(14, 2, 64, [300, 90, 700], 2)
    pos, row = [0, 299, 17, 89, 650, 5, 699], [2, 0, 1, 1, 2, 0, 2]
    q = randn(7, 14 * 64, seed=3).bfloat16()
    for bound in (700, 1 << 21):
        got = p.attention(K, pos, row, q=q, bound=bound)
        p.check(got, pos, row, q=q)
    alone = torch.cat([p.attention(K, [a], [b], q=q[i:i + 1].contiguous(), bound=700) for i, (a, b) in enumerate(zip(pos, row))])
    p.check(alone, pos, row, q=q)


def test_rows_that_see_nothing_and_groups_that_are_none(K):
    p = Paged(4, 2, 64, [200, 130, 64], 6)
    table = p.table.clone()
    table[0] = -1
    table[1, 1] = -1
    long = p.attention(K, [199, 129, 63], [0, 1, 2], table=table, bound=1 << 21)
    assert (long[0] == 0).all()
    p.check(long, [199, 129, 63], [0, 1, 2], table=table)
    out = p.attention(K, [199, 129, 63], [0, 1, 2], table=table)
    assert (out[0] == 0).all()
    p.check(out, [199, 129, 63], [0, 1, 2], table=table)
    keys = p.keys.clone()
    keys[p.pages[2][0], 1, 40, 7] = float("nan")                             # of one key head: its queries' results are none, the others as they were
    p.pool = plain.pack(keys.view(-1, 64, 64), p.values.view(-1, 64, 64)).view(p.n_pages, 2, -1)
    again = p.attention(K, [199, 129, 63], [0, 1, 2], table=table)
    assert torch.equal(again[:2], out[:2]) and torch.equal(again[2, :128], out[2, :128]) and torch.isnan(again[2, 128:]).all()


@pytest.mark.parametrize("size", [1e-3, 30.0])
def test_scores_and_values_of_any_size(K, size):
    p = Paged(8, 2, 128, [700], 8)
    p.keys, p.values = p.keys * (size if size > 1 else 1.0), p.values * size
    p.pool = plain.pack(p.keys.view(-1, 64, 128), p.values.view(-1, 64, 128)).view(p.n_pages, 2, -1)
    p.check(p.attention(K, [699], [0]), [699], [0])


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("q_up,k_up,v_up", [(-40, 40, 60), (40, -40, -40), (60, -60, 0), (0, 0, -40)])
def test_sizes_near_the_ends(K, D, q_up, k_up, v_up):
    """Powers of two change no code and no weight: results are the plain ones' times the values' power, bit for bit."""
    p = Paged(4, 2, D, [700, 90], 12)
    pos, row = [699, 89], [0, 1]
    want = p.attention(K, pos, row)
    p.pool = plain.pack((p.keys.double() * 2.0 ** k_up).bfloat16().view(-1, 64, D), (p.values.double() * 2.0 ** v_up).bfloat16().view(-1, 64, D)).view(p.n_pages, 2, -1)
    p.scale *= 2.0 ** -(q_up + k_up)
    got = p.attention(K, pos, row, q=(p.q.double() * 2.0 ** q_up).bfloat16())
    assert torch.equal(got.double(), want.double() * 2.0 ** v_up)


# ---------------------------------------------------------------------------- prompts

@pytest.mark.parametrize("H,G,D", [(14, 2, 64), (28, 4, 128), (2, 2, 64), (20, 1, 128)])
@pytest.mark.parametrize("starts,lens,window", [([0], [1], None), ([0], [128], None), ([0, 3, 64, 1000], [129, 1, 200, 77], None), ([500, 0], [300, 260], 100), ([0], [640], 64)])
def test_prompts(K, H, G, D, starts, lens, window):
    p = Paged(H, G, D, [s + n for s, n in zip(starts, lens)], 21, rubbish=float("nan"))
    T = sum(lens)
    q = randn(T + 3, H * D + 16, seed=4, scale=1.5).bfloat16()
    out = torch.full((T, H * D), 7.0, dtype=torch.bfloat16, device="cuda")
    got = K.attention_int4_prompt(q, q.shape[1], H, G, D, p.pool, p.table, p.width, K.prefill_tiles(lens, starts, "cuda", K.PREFILL_TILE_TCGEN05), T, window, p.scale, out=out)
    pos = [s + i for s, n in zip(starts, lens) for i in range(n)]
    row = [b for b, n in enumerate(lens) for _ in range(n)]
    some = sorted(set(list(range(0, T, 37)) + [0, T - 1, min(T - 1, 127), min(T - 1, 128)]))
    p.check(got[some], [pos[i] for i in some], [row[i] for i in some], q=q[some], window=window, halves=True)


def test_runs_that_are_not_listed_stay(K):
    p = Paged(4, 2, 64, [200, 200], 3)
    q = randn(400, 256, seed=5).bfloat16()
    out = torch.full((400, 256), 7.0, dtype=torch.bfloat16, device="cuda")
    K.attention_int4_prompt(q, 256, 4, 2, 64, p.pool, p.table, p.width, ints([[1, 230, 40, 30]]), 400, None, p.scale, out=out)
    assert (out[:230] == 7).all() and (out[270:] == 7).all()
    p.check(out[230:270], list(range(30, 70)), [1] * 40, q=q[230:270], halves=True)


# ---------------------------------------------------------------------------- bounds and selected pages

@pytest.mark.parametrize("H,G,D", [(14, 2, 64), (28, 4, 128)])
@pytest.mark.parametrize("starts,lens", [([63], [1]), ([0, 62, 127, 60], [1, 1, 1, 4]), ([0, 30], [300, 34]), ([5], [20])])
def test_bounds(K, H, G, D, starts, lens):
    p = Paged(H, G, D, [s + n for s, n in zip(starts, lens)], 31)
    p.keys[p.pages[0][0], 0, 3, 1] = float("nan")
    p.pool = plain.pack(p.keys.view(-1, 64, D), p.values.view(-1, 64, D)).view(p.n_pages, G, 80 * D)
    bounds = torch.full((p.n_pages, G, 2, D), 9.0, dtype=torch.bfloat16, device="cuda")
    pos = [s + i for s, n in zip(starts, lens) for i in range(n)]
    row = [b for b, n in enumerate(lens) for _ in range(n)]
    got = K.page_bounds(p.pool, G, D, ints(pos), ints(row), p.table, p.width, bounds)
    assert got is bounds
    want = torch.full_like(bounds, 9.0)
    keys = plain.unpack(p.pool.view(-1, 80 * D))[0].view(p.n_pages, G, 64, D)
    for a, b in zip(pos, row):
        if a % PAGE == PAGE - 1:
            page = p.pages[b][a // PAGE]
            want[page] = torch.stack([keys[page].amin(1), keys[page].amax(1)], 1).float().bfloat16()
    assert torch.equal(torch.nan_to_num(got, nan=5e4), torch.nan_to_num(want, nan=5e4))


def bounds_of(p):
    keys = plain.unpack(p.pool.view(-1, 80 * p.D))[0].view(p.n_pages, p.G, 64, p.D)
    return torch.stack([keys.amin(2), keys.amax(2)], 2).bfloat16()


def chosen(p, bounds, t, pos, row, keep):
    """Pages (in the order of the positions) of every head."""
    out, last = [], pos // PAGE
    for g in range(p.G):
        if last < keep:
            out.append(list(range(last + 1)))
            continue
        q = p.q[t, :p.H * p.D].double().view(p.G, -1, p.D)[g]
        b = bounds[p.table[row, :last + 1].long(), g].double()
        score = torch.maximum(q[:, None] * b[None, :, 0], q[:, None] * b[None, :, 1]).sum((0, 2)).nan_to_num(nan=float("inf")).tolist()
        best = sorted(range(1, last), key=lambda j: (-score[j], j))[:max(0, keep - 2)]
        out.append(sorted(([0] if keep > 1 else []) + best + [last]))
    return out


@pytest.mark.parametrize("H,G,D", HEADS[:4])
@pytest.mark.parametrize("keep", [1, 2, 3, 8, 40])
def test_selected_pages(K, H, G, D, keep):
    lengths = [1, 64, 65, 64 * 8, 64 * 8 + 1, 1500, 3000]
    p = Paged(H, G, D, lengths, 41, rubbish=float("nan"))
    bounds = bounds_of(p)
    pos, row = [n - 1 for n in lengths], list(range(len(lengths)))
    pages = K.select_pages(p.q, p.q.shape[1], H, G, D, bounds, p.table, p.width, ints(pos), ints(row), keep, 3000)
    got = K.attention_int4_selected(p.q, p.q.shape[1], H, G, D, p.pool, pages, p.scale)
    for t, n in enumerate(lengths):
        want = chosen(p, bounds, t, pos[t], t, keep)
        seen = torch.zeros(G, p.width * PAGE, dtype=torch.bool, device="cuda")
        for g, js in enumerate(want):
            ids = [p.pages[t][j] * G + g for j in js]
            assert pages.table[t * G + g].tolist() == ids + [-1] * (keep - len(ids))
            assert int(pages.pos[t * G + g]) == (len(js) - 1) * PAGE + pos[t] % PAGE
            for j in js:
                seen[g, j * PAGE: (j + 1) * PAGE] = True
        seen[:, pos[t] + 1:] = False
        w, bound = plain.attend(p.q[t, :H * D].view(H, D), p.pool[p.table[t].clamp(min=0).long()], seen, p.scale)
        assert ((got[t].double().view(H, D) - w).abs() <= bound + 1e-30).all()


@pytest.mark.parametrize("H,G,D,rows,keep", [(28, 4, 128, 38, 12), (14, 2, 64, 96, 40), (20, 1, 128, 150, 30)])
def test_selected_pages_of_many_rows(K, H, G, D, rows, keep):
    lengths = [1 + (b * 677) % (64 * 60) for b in range(rows)]
    p = Paged(H, G, D, lengths, 43, rubbish=float("nan"))
    bounds = bounds_of(p)
    pos, row = [n - 1 for n in lengths], list(range(rows))
    pages = K.select_pages(p.q, p.q.shape[1], H, G, D, bounds, p.table, p.width, ints(pos), ints(row), keep, max(lengths))
    got = K.attention_int4_selected(p.q, p.q.shape[1], H, G, D, p.pool, pages, p.scale)
    wide = K.SelectedPages(torch.cat([pages.table, torch.full((rows * G, 300 - keep), -1, dtype=torch.int32, device="cuda")], 1), pages.pos)      # a launch for more
    for out in (got, K.attention_int4_selected(p.q, p.q.shape[1], H, G, D, p.pool, wide, p.scale)):
        for t in range(0, rows, 7):
            seen = torch.zeros(G, p.width * PAGE, dtype=torch.bool, device="cuda")
            for g in range(G):
                for page in pages.table[t * G + g].tolist():
                    if page >= 0:
                        j = p.pages[t].index(page // G)
                        seen[g, j * PAGE: (j + 1) * PAGE] = True
            seen[:, pos[t] + 1:] = False
            w, bound = plain.attend(p.q[t, :H * D].view(H, D), p.pool[p.table[t].clamp(min=0).long()], seen, p.scale)
            assert ((out[t].double().view(H, D) - w).abs() <= bound + 1e-30).all()


def test_pages_that_score_alike_and_bounds_that_are_none(K):
    H, G, D = 4, 2, 64
    p = Paged(H, G, D, [64 * 30], 51)
    bounds = torch.zeros(p.n_pages, G, 2, D, dtype=torch.bfloat16, device="cuda")
    args = (p.q, p.q.shape[1], H, G, D, bounds, p.table, p.width, ints([64 * 30 - 1]), ints([0]), 5, 64 * 30)
    ids = lambda js, g: [p.pages[0][j] * G + g for j in js]                 # noqa: E731
    pages = K.select_pages(*args)
    assert pages.table.tolist() == [ids([0, 1, 2, 3, 29], g) for g in range(G)]     # all alike: the first ones
    bounds[p.pages[0][17], 1, 0, 5] = float("nan")
    bounds[p.pages[0][20], :, 1] = float("inf")
    pages = K.select_pages(*args)
    assert pages.table.tolist() == [ids([0, 1, 2, 20, 29], 0), ids([0, 1, 17, 20, 29], 1)]


@pytest.mark.parametrize("n_pages", [700, 1024, 1025, 1400])
@pytest.mark.parametrize("kind", ["close", "equal", "none"])
def test_scores_that_differ_by_little(K, n_pages, kind):
    """Scores closer to one another than their errors in float32, many and few of them; runs of equal ones; bounds that are no number, here and there and nearly everywhere."""
    H, G, D = 14, 2, 64
    p = Paged(H, G, D, [64 * n_pages - 5, 64 * 60], 53)
    g = gen(54)
    bounds = torch.zeros(p.n_pages, G, 2, D, dtype=torch.bfloat16, device="cuda")
    base = torch.randn(G, 1, D, generator=g, device="cuda") * 100
    bounds[:] = base.bfloat16()
    if kind == "close":                                                      # one channel of one row tells them apart, by less than the others' roundings
        bounds[:, :, :, 3] = (torch.randn(p.n_pages, G, 1, generator=g, device="cuda") * 1e-5).bfloat16()
    elif kind == "equal":
        bounds[:, :, 1, 9] += torch.randint(0, 3, (p.n_pages, G), generator=g, device="cuda") * 64.0
    else:
        few = torch.rand(p.n_pages, G, generator=g, device="cuda")
        bounds[:, 0, 0, 5] = torch.where(few[:, 0] < 0.02, float("nan"), bounds[:, 0, 0, 5].float()).bfloat16()
        bounds[:, 1, 1, 60] = torch.where(few[:, 1] < 0.97, float("nan"), bounds[:, 1, 1, 60].float()).bfloat16()
    pos = [64 * n_pages - 6, 64 * 60 - 1]
    for keep in (3, 30, 200, 650):
        pages = K.select_pages(p.q, p.q.shape[1], H, G, D, bounds, p.table, p.width, ints(pos), ints([0, 1]), keep, 64 * n_pages)
        for t in range(2):
            for h, js in enumerate(chosen(p, bounds, t, pos[t], t, keep)):
                assert pages.table[t * G + h].tolist() == [p.pages[t][j] * G + h for j in js] + [-1] * (keep - len(js)), (t, h, keep)


def test_tokens_that_see_nothing_and_positions_behind_the_table(K):
    H, G, D = 14, 2, 64
    p = Paged(H, G, D, [64 * 9, 64 * 9, 64 * 9, 700], 52)
    bounds = bounds_of(p)
    pos, row = [-1, 300, 300, 64 * p.width + 5, 575], [0, -1, 4, 3, 1]
    q = randn(5, H * D, seed=5).bfloat16()
    for keep in (2, 5, 40):
        pages = K.select_pages(q, H * D, H, G, D, bounds, p.table, p.width, ints(pos), ints(row), keep, 64 * p.width + 10)
        assert (pages.table[:3 * G] == -1).all() and (pages.pos[:3 * G] == -1).all()
        got = K.attention_int4_selected(q, H * D, H, G, D, p.pool, pages, p.scale)
        assert (got[:3] == 0).all()
        assert pages.pos[4 * G:].tolist() == [(min(keep, 9) - 1) * 64 + 63] * G
    assert torch.equal(pages.pos[3 * G: 4 * G], ints([64 * p.width - 1] * G))
    p.check(got[3:], [64 * p.width - 1, 575], [3, 1], q=q[3:])


def test_a_context_of_many_pages(K):
    H, G, D, n = 2, 1, 64, 64 * 2100
    p = Paged(H, G, D, [n, 64 * 1000 + 7], 61)
    bounds = bounds_of(p)
    for keep in (3, 100, 2000):
        pages = K.select_pages(p.q, p.q.shape[1], H, G, D, bounds, p.table, p.width, ints([n - 1, 64 * 1000 + 6]), ints([0, 1]), keep, n)
        for t, pos in enumerate((n - 1, 64 * 1000 + 6)):
            js = chosen(p, bounds, t, pos, t, keep)[0]
            assert pages.table[t].tolist() == [p.pages[t][j] for j in js] + [-1] * (keep - len(js))


# ---------------------------------------------------------------------------- all of it

@pytest.mark.parametrize("H,G,D", [(14, 2, 64), (28, 4, 128)])
def test_a_prompt_then_tokens(K, H, G, D):
    """A sequence as a model runs it: a prompt appended and attended to, its pages' bounds, then tokens one by one over all and over selected pages."""
    n, more, keep = 450, 70, 4
    p = Paged(H, G, D, [n + more], 71)
    p.pool.zero_()
    bounds = torch.zeros(p.n_pages, G, 2, D, dtype=torch.bfloat16, device="cuda")
    x = randn(n + more, (H + 2 * G) * D, seed=6, scale=1.2).bfloat16()
    cos, sin = angles(D, 1000)
    q, pos, row = append(K, p, x[:n].contiguous(), [0], [n], cos, sin)
    K.page_bounds(p.pool, G, D, ints(pos), ints(row), p.table, p.width, bounds)
    a = K.attention_int4_prompt(q, H * D, H, G, D, p.pool, p.table, p.width, K.prefill_tiles([n], [0], "cuda", K.PREFILL_TILE_TCGEN05), n, None, p.scale)
    some = [0, 100, n - 1]
    p.check(a[some], some, [0] * 3, q=q[some], halves=True)
    for i in range(n, n + more):
        q, _, _ = append(K, p, x[i:i + 1].contiguous(), [i], [1], cos, sin)
        K.page_bounds(p.pool, G, D, ints([i]), ints([0]), p.table, p.width, bounds)
        p.check(p.attention(K, [i], [0], q=q), [i], [0], q=q)
        pages = K.select_pages(q, H * D, H, G, D, bounds, p.table, p.width, ints([i]), ints([0]), keep, n + more)
        p.q = q
        want = chosen(p, bounds, 0, i, 0, keep)
        assert pages.table.tolist() == [[p.pages[0][j] * G + g for j in js] for g, js in enumerate(want)]
    done = (n + more) // PAGE
    assert torch.equal(bounds[p.pages[0][:done]], bounds_of(p)[p.pages[0][:done]])


def test_refusals(K):
    from pico_engine.ops import KernelError
    p = Paged(4, 2, 64, [100], 1)
    one, q = ints([5]), p.q
    ok = dict(window=None)
    bad = [lambda: K.attention_int4(q, q.shape[1], 4, 2, 64, p.pool[:, :1], p.table, p.width, one, ints([0]), None, 1.0, 100),
           lambda: K.attention_int4(q, q.shape[1], 4, 2, 64, p.pool.view(p.n_pages, 1, -1), p.table, p.width, one, ints([0]), None, 1.0, 100),
           lambda: K.attention_int4(q.float(), q.shape[1], 4, 2, 64, p.pool, p.table, p.width, one, ints([0]), None, 1.0, 100),
           lambda: K.attention_int4(q, 255, 4, 2, 64, p.pool, p.table, p.width, one, ints([0]), None, 1.0, 100),
           lambda: K.attention_int4(q, q.shape[1], 4, 2, 64, p.pool, p.table, p.width, ints([5, 6]), ints([0, 0]), None, 1.0, 100),
           lambda: K.attention_int4(q, q.shape[1], 4, 2, 64, p.pool, p.table, p.width + 1, one, ints([0]), None, 1.0, 100),
           lambda: K.attention_int4(q, q.shape[1], 4, 2, 64, p.pool, p.table, p.width, one, ints([0]), None, 1.0, 0),
           lambda: K.attention_int4(q, q.shape[1], 4, 2, 64, p.pool, p.table, p.width, one, ints([0]), -1, 1.0, 100),
           lambda: K.attention_int4(q, q.shape[1], 4, 2, 64, p.pool, p.table, p.width, one.long(), ints([0]), None, 1.0, 100),
           lambda: K.attention_int4_prompt(q, q.shape[1], 4, 2, 64, p.pool, p.table, p.width, ints([0, 0, 1, 0]), 1, None, 1.0),
           lambda: K.store_int4(q, 4, 2, 64, None, None, one, ints([0]), p.pool, p.table, p.width),
           lambda: K.store_int4(randn(1, 512).bfloat16(), 4, 2, 64, randn(9, 32), None, one, ints([0]), p.pool, p.table, p.width),
           lambda: K.store_int4(randn(1, 512).bfloat16(), 4, 2, 64, randn(9, 64), randn(9, 64), one, ints([0]), p.pool, p.table, p.width),
           lambda: K.load_int4(p.pool, 2, 128, one, ints([0]), p.table, p.width),
           lambda: K.page_bounds(p.pool, 2, 64, one, ints([0]), p.table, p.width, torch.zeros(p.n_pages, 2, 2, 32, dtype=torch.bfloat16, device="cuda")),
           lambda: K.select_pages(q, q.shape[1], 4, 2, 64, torch.zeros(p.n_pages, 2, 1, 64, dtype=torch.bfloat16, device="cuda"), p.table, p.width, one, ints([0]), 4, 100),
           lambda: K.select_pages(q, q.shape[1], 4, 2, 64, bounds_of(p), p.table, p.width, one, ints([0]), 0, 100),
           lambda: K.attention_int4_selected(q, q.shape[1], 4, 2, 64, p.pool, K.SelectedPages(ints([[1, 2]]), ints([3])), 1.0)]
    before = p.pool.clone()
    for call in bad:
        with pytest.raises(KernelError):
            call()
    assert torch.equal(before, p.pool)
    none = torch.empty(0, dtype=torch.int32, device="cuda")
    assert K.attention_int4(q[:0], q.shape[1], 4, 2, 64, p.pool, p.table, p.width, none, none, None, 1.0, 1).shape == (0, 256)
    assert K.load_int4(p.pool, 2, 64, none, none, p.table, p.width)[0].shape == (0, 2, 64)


def test_prompts_over_groups_that_are_none(K):
    """A value or key that is no number reaches the tokens that see it, and no other."""
    H, G, D, n = 4, 2, 64, 300
    p = Paged(H, G, D, [n], 81)
    q = randn(n, H * D, seed=7).bfloat16()
    tiles = K.prefill_tiles([n], [0], "cuda", K.PREFILL_TILE_TCGEN05)
    run = lambda: K.attention_int4_prompt(q, H * D, H, G, D, p.pool, p.table, p.width, tiles, n, None, p.scale)     # noqa: E731
    clean = run()
    keys, values = p.keys.clone(), p.values.clone()
    keys[p.pages[0][1], 0, 36, 3], values[p.pages[0][3], 1, 8, 40] = float("nan"), float("inf")                       # positions 100 and 200
    p.pool = plain.pack(keys.view(-1, 64, D), values.view(-1, 64, D)).view(p.n_pages, G, 80 * D)
    out = run().view(n, H, D)
    first, second = out[:, :2], out[:, 2:]
    assert torch.equal(first[:100], clean.view(n, H, D)[:100, :2]) and torch.isnan(first[100:]).all()
    assert torch.equal(second[:200], clean.view(n, H, D)[:200, 2:]) and torch.isnan(second[200:]).all()


def test_runs_and_pages_that_are_none_of_the_call(K):
    """Runs of rows, tokens or positions that the call does not have, and pages beyond the pool, read and write nothing."""
    H, G, D = 4, 2, 64
    p = Paged(H, G, D, [200], 91)
    q = randn(200, H * D, seed=8).bfloat16()
    out = torch.full((200, H * D), 7.0, dtype=torch.bfloat16, device="cuda")
    table = p.table.clone()
    table[0, 1] = p.n_pages + 5
    runs = [[0, 0, 40, 130], [1, 50, 10, 0], [-1, 50, 10, 0], [0, 190, 20, 0], [0, 60, 0, 0], [0, 70, 10, -5], [0, -3, 10, 0], [0, 90, 5, 64 * p.width + 1000]]
    K.attention_int4_prompt(q, H * D, H, G, D, p.pool, table, p.width, ints(runs), 200, None, p.scale, out=out)
    assert (out[40:90] == 7).all() and (out[95:] == 7).all()
    there = table.clone()
    there[0, 1] = -1
    p.check(out[:40], list(range(130, 170)), [0] * 40, q=q[:40], table=there, halves=True)
    got = p.attention(K, [180], [0], q=q, table=table)
    p.check(got, [180], [0], q=q, table=there)


@pytest.mark.parametrize("H,G,D", [(14, 2, 64), (4, 1, 128)])
@pytest.mark.parametrize("start,n", [(0, 300), (4000, 130)])
def test_prompts_over_pages_of_all_sizes(K, H, G, D, start, n):
    """Pages whose values differ by many powers of two, and queries and keys far from one."""
    total = start + n
    p = Paged(H, G, D, [total], 98)
    up = torch.randint(-25, 60, (p.n_pages, G, 1, 1), generator=gen(99), device="cuda")
    p.pool = plain.pack((p.keys.double() * 2.0 ** -20).bfloat16().view(-1, 64, D), (p.values.double() * 2.0 ** up).bfloat16().view(-1, 64, D)).view(p.n_pages, G, 80 * D)
    q = (randn(n, H * D, seed=100).double() * 2.0 ** 30).bfloat16()
    p.scale *= 2.0 ** -10
    got = K.attention_int4_prompt(q, H * D, H, G, D, p.pool, p.table, p.width, K.prefill_tiles([n], [start], "cuda", K.PREFILL_TILE_TCGEN05), n, None, p.scale)
    some = [0, n // 2, n - 1]
    p.check(got[some], [start + i for i in some], [0] * 3, q=q[some], halves=True)


@pytest.mark.parametrize("H,G,D,rows", [(4, 2, 64, 5000), (2, 1, 128, 17000)])
def test_prompts_of_many_rows(K, H, G, D, rows):
    lens = [1 + b % 3 for b in range(rows)]
    p = Paged(H, G, D, lens, 96)
    n = sum(lens)
    q = randn(n, H * D, seed=97).bfloat16()
    got = K.attention_int4_prompt(q, H * D, H, G, D, p.pool, p.table, p.width, K.prefill_tiles(lens, [0] * rows, "cuda", K.PREFILL_TILE_TCGEN05), n, None, p.scale)
    pos, row = [i for c in lens for i in range(c)], [b for b, c in enumerate(lens) for _ in range(c)]
    some = list(range(0, n, 997))
    p.check(got[some], [pos[i] for i in some], [row[i] for i in some], q=q[some], halves=True)


@pytest.mark.parametrize("H,G,D", [(14, 2, 64), (28, 4, 128)])
def test_rows_that_share_a_page_see_it_as_far_as_they_go(K, H, G, D):
    """One sequence on the pages of several rows, each with a part of the tokens, the last page's among them: as one row has it."""
    n, cuts = 64 * 20 + 50, [64 * 20, 64 * 20 + 1, 64 * 20 + 10, 64 * 20 + 33, 64 * 20 + 50]
    p = Paged(H, G, D, [n], 93)
    q = randn(n, H * D, seed=94).bfloat16()
    whole = K.attention_int4_prompt(q, H * D, H, G, D, p.pool, p.table, p.width, K.prefill_tiles([n], [0], "cuda", K.PREFILL_TILE_TCGEN05), n, None, p.scale)
    lens = [b - a for a, b in zip([0] + cuts, cuts)]
    table = p.table.expand(len(lens), -1).contiguous()
    for _ in range(5):
        got = K.attention_int4_prompt(q, H * D, H, G, D, p.pool, table, p.width, K.prefill_tiles(lens, [0] + cuts[:-1], "cuda", K.PREFILL_TILE_TCGEN05), n, None, p.scale)
        some = [c - 1 for c in cuts]
        p.check(got[some], some, [0] * len(some), q=q[some], halves=True)
        assert torch.equal(got[:64 * 20], whole[:64 * 20])


@pytest.mark.parametrize("H,G,D", [(14, 2, 64), (4, 1, 128)])
@pytest.mark.parametrize("start,n,window", [(4000, 200, None), (5000, 1, None), (3000, 130, 2500), (300, 100, None)])
def test_a_prompt_behind_a_long_context(K, H, G, D, start, n, window):
    """Few runs on many pages: their steps are shared by several CTAs."""
    p = Paged(H, G, D, [start + n, 70], 101)
    q = randn(n + 70, H * D, seed=9, scale=1.5).bfloat16()
    tiles = K.prefill_tiles([n, 70], [start, 0], "cuda", K.PREFILL_TILE_TCGEN05)
    got = K.attention_int4_prompt(q, H * D, H, G, D, p.pool, p.table, p.width, tiles, n + 70, window, p.scale)
    some = sorted({0, n // 2, n - 1, n, n + 33, n + 69})
    pos = [start + i if i < n else i - n for i in some]
    p.check(got[some], pos, [0 if i < n else 1 for i in some], q=q[some], window=window, halves=True)


# ---------------------------------------------------------------------------- large caches, streams, captured calls

def test_a_cache_beyond_four_gigabytes(K):
    """Pages behind the four billionth byte (and 16-bit pages behind it, in a prompt's scratch): the same as on a small pool."""
    H, G, D, n = 16, 8, 128, 1500
    p = Paged(H, G, D, [n], 101)
    far = 53000
    pool = K.int4_pool(far + p.n_pages, G, D, "cuda")
    assert pool.numel() > 1 << 32
    table = torch.where(p.table >= 0, p.table + far, p.table)
    x = randn(n, (H + 2 * G) * D, seed=102).bfloat16()
    bounds, near = [torch.zeros(m.shape[0], G, 2, D, dtype=torch.bfloat16, device="cuda") for m in (pool, p.pool)]
    outs = []
    for where, places, ends in ((pool, table, bounds), (p.pool.zero_(), p.table, near)):
        q, pos, row = append(K, p, x, [0], [n], pool=where, table=places)
        K.page_bounds(where, G, D, ints(pos), ints(row), places, p.width, ends)
        out = [q, *K.load_int4(where, G, D, ints(pos), ints(row), places, p.width)]
        tiles = K.prefill_tiles([n], [0], "cuda", K.PREFILL_TILE_TCGEN05)
        out.append(K.attention_int4_prompt(q, H * D, H, G, D, where, places, p.width, tiles, n, None, p.scale))
        for most in (n, 1 << 21):
            out.append(K.attention_int4(q[-40:], H * D, H, G, D, where, places, p.width, ints(pos[-40:]), ints(row[-40:]), None, p.scale, most))
        pages = K.select_pages(q[-40:], H * D, H, G, D, ends, places, p.width, ints(pos[-40:]), ints(row[-40:]), 6, n)
        out.append(K.attention_int4_selected(q[-40:], H * D, H, G, D, where, pages, p.scale))
        outs.append(out)
    assert torch.equal(pool[far:far + p.n_pages], p.pool) and torch.equal(bounds[far:far + p.n_pages], near) and not pool[:far].any()
    for a, b in zip(*outs):
        assert torch.equal(a, b)


def test_calls_on_two_streams_and_captured(K):
    """Two graphs, of calls with scratch of their own, replayed at the same time, many times over: every result as the eager call's."""
    cases = []
    for seed, (H, G, D) in ((111, (28, 4, 128)), (112, (14, 2, 64))):
        lengths = [3000 + 37 * b for b in range(48)]
        p = Paged(H, G, D, lengths, seed)
        bounds = bounds_of(p)
        pos, row, lens = ints([n - 1 for n in lengths]), ints(list(range(48))), [150, 1, 33]
        tiles = K.prefill_tiles(lens, [2000, 500, 2900], "cuda", K.PREFILL_TILE_TCGEN05)
        long = randn(184, H * D, seed=seed).bfloat16()

        def run(p=p, bounds=bounds, pos=pos, row=row, tiles=tiles, long=long, H=H, G=G, D=D):
            a = K.attention_int4(p.q, p.q.shape[1], H, G, D, p.pool, p.table, p.width, pos, row, None, p.scale, 1 << 21)
            pages = K.select_pages(p.q, p.q.shape[1], H, G, D, bounds, p.table, p.width, pos, row, 40, 5000)
            return [a, pages.table, pages.pos, K.attention_int4_selected(p.q, p.q.shape[1], H, G, D, p.pool, pages, p.scale),
                    K.attention_int4(p.q, p.q.shape[1], H, G, D, p.pool, p.table, p.width, pos, row, 500, p.scale, 5000),
                    K.attention_int4_prompt(long, H * D, H, G, D, p.pool, p.table, p.width, tiles, 184, None, p.scale)]
        cases.append((run, [x.clone() for x in run()]))
    torch.cuda.synchronize()
    graphs, streams = [], [torch.cuda.Stream(), torch.cuda.Stream()]
    for run, _ in cases:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = run()
        graphs.append((g, out))
    for _ in range(20):
        for out in (o for _, outs in graphs for o in outs):
            out.zero_()
        torch.cuda.synchronize()
        for (g, _), s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        for (_, outs), (_, want) in zip(graphs, cases):
            assert all(torch.equal(a, b) for a, b in zip(outs, want))
    for _ in range(20):
        got = []
        for (run, _), s in zip(cases, streams):
            with torch.cuda.stream(s):
                got.append(run())
        torch.cuda.synchronize()
        for outs, (_, want) in zip(got, cases):
            assert all(torch.equal(a, b) for a, b in zip(outs, want))
