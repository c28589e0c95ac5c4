"""The 4-bit cache where it can go wrong seldom or far from the ordinary: short prompts again and again, sizes at the ends of the types, arguments beyond 32 bits, calls of several threads.
Compared with the plain form in 64 bits (``plain_int4``) within the bounds that ``test_int4_gpu`` derives."""
import pytest
import torch

import plain_int4 as plain
from test_int4_gpu import HEADS, PAGE, Paged, append, bounds_of, gen, ints, randn       # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def K():
    from pico_engine.ops import kernels
    return kernels


# ---------------------------------------------------------------------------- prompts

@pytest.mark.parametrize("H,G,D", [(14, 2, 64), (8, 4, 128)])
def test_short_prompts_again_and_again(K, H, G, D):
    """Runs that see at most 128 keys, whose second half of softmax warps has no keys: queries are scaled by the largest number of the whole row, whichever half of the channels it is in."""
    lens = [1 + (7 * b) % 128 for b in range(300)]
    p = Paged(H, G, D, lens, 121)
    n = sum(lens)
    q = randn(n, H, D, seed=122)
    q[::2, :, D // 2:] *= 2.0 ** -9
    q[1::2, :, :D // 2] *= 2.0 ** -9
    q = q.bfloat16().view(n, H * D)
    tiles = K.prefill_tiles(lens, [0] * len(lens), "cuda", K.PREFILL_TILE_TCGEN05)
    run = lambda: K.attention_int4_prompt(q, H * D, H, G, D, p.pool, p.table, p.width, tiles, n, None, p.scale)     # noqa: E731
    first = run()
    pos, row = [i for c in lens for i in range(c)], [b for b, c in enumerate(lens) for _ in range(c)]
    some = list(range(0, n, 811))
    p.check(first[some], [pos[i] for i in some], [row[i] for i in some], q=q[some], halves=True)
    for _ in range(100):
        assert torch.equal(run(), first)


@pytest.mark.parametrize("H,G,D", [(14, 2, 64), (8, 2, 128)])
def test_prompts_over_pages_without_a_value(K, H, G, D):
    """Pages whose values are all zero beside pages of small ones: they weigh in the softmax and carry nothing, and the others keep their bits."""
    n = 500
    p = Paged(H, G, D, [n], 131)
    up = torch.full((p.n_pages, 1, 1, 1), 2.0 ** -30, device="cuda", dtype=torch.float64)
    up[p.pages[0][2]] = 0.0
    up[p.pages[0][5]] = 0.0
    p.pool = plain.pack(p.keys.view(-1, 64, D), (p.values.double() * up).bfloat16().view(-1, 64, D)).view(p.n_pages, G, 80 * D)
    q = randn(n, H * D, seed=132).bfloat16()
    got = K.attention_int4_prompt(q, H * D, H, G, D, p.pool, p.table, p.width, K.prefill_tiles([n], [0], "cuda", K.PREFILL_TILE_TCGEN05), n, None, p.scale)
    some = [0, 100, 200, 383, n - 1]
    p.check(got[some], some, [0] * len(some), q=q[some], halves=True)


@pytest.mark.parametrize("H,G,D", [(14, 2, 64), (28, 4, 128)])
@pytest.mark.parametrize("window", [None, 100])
def test_expanded_pages_lie_by_row_or_by_page(K, H, G, D, window):
    """A prompt on a pool of many pages expands what its rows can see, one on a wide table the pool's: results are the same, with a bound of the positions too."""
    starts, lens = [0, 700, 130], [300, 129, 1]
    p = Paged(H, G, D, [s + n for s, n in zip(starts, lens)], 181, rubbish=float("nan"))
    T, tiles = sum(lens), K.prefill_tiles(lens, starts, "cuda", K.PREFILL_TILE_TCGEN05)
    q = randn(T, H * D, seed=182).bfloat16()
    many = torch.cat([p.pool, torch.full((1500, G, 80 * D), 255, dtype=torch.uint8, device="cuda")])
    wide = torch.full((3, 900), -1, dtype=torch.int32, device="cuda")
    wide[:, :p.width] = p.table
    run = lambda pool, table, most=None: K.attention_int4_prompt(q, H * D, H, G, D, pool, table, table.shape[1], tiles, T, window, p.scale, max_context=most)     # noqa: E731
    by_page, by_row = run(p.pool, p.table), run(many, p.table)
    pos, row = [s + i for s, n in zip(starts, lens) for i in range(n)], [b for b, n in enumerate(lens) for _ in range(n)]
    some = sorted(set(range(0, T, 37)) | {T - 1, T - 2, 299, 300})
    for got in (by_page, by_row, run(p.pool, wide), run(many, wide), run(many, wide, 829), run(many, wide, 1 << 40)):
        p.check(got[some], [pos[i] for i in some], [row[i] for i in some], q=q[some], window=window, halves=True)
    assert torch.equal(run(many, wide, 829), by_row)


def test_a_short_prompt_on_a_large_cache_asks_for_little_memory(K):
    H, G, D = 4, 2, 64
    pool = K.int4_pool(20000, G, D, "cuda")
    q, table = randn(33, H * D, seed=1).bfloat16(), torch.full((1, 512), -1, dtype=torch.int32, device="cuda")
    table[0, 0] = 19999
    tiles = K.prefill_tiles([33], [0], "cuda", K.PREFILL_TILE_TCGEN05)
    K.attention_int4_prompt(q, H * D, H, G, D, pool, table, 512, tiles, 33, None, 1.0)
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    out = K.attention_int4_prompt(q, H * D, H, G, D, pool, table, 512, tiles, 33, None, 1.0, max_context=64)
    page = G * 64 * D * 4                                                    # of keys and values in 16 bits
    assert torch.cuda.max_memory_allocated() - before <= page + out.numel() * 2 + 16384
    before = torch.cuda.memory_allocated()
    torch.cuda.reset_peak_memory_stats()
    K.attention_int4_prompt(q, H * D, H, G, D, pool, table, 512, tiles, 33, None, 1.0)
    assert torch.cuda.max_memory_allocated() - before <= 600 * page


def test_expanded_pages_beyond_four_gigabytes(K):
    """A table of more places than the pool has pages: every page of the pool has its place in the scratch, those behind the four billionth byte too."""
    H, G, D, n = 16, 8, 128, 1500
    p = Paged(H, G, D, [n], 191)
    far = 40000
    pool = torch.cat([torch.zeros(far, G, 80 * D, dtype=torch.uint8, device="cuda"), p.pool])
    table = torch.full((2000, p.width), -1, dtype=torch.int32, device="cuda")
    table[1999] = torch.where(p.table[0] >= 0, p.table[0] + far, p.table[0])
    assert table.numel() > pool.shape[0] and pool.shape[0] * G * 64 * D * 2 > 1 << 32
    q, tiles = randn(n, H * D, seed=192).bfloat16(), K.prefill_tiles([n], [0], "cuda", K.PREFILL_TILE_TCGEN05)
    want = K.attention_int4_prompt(q, H * D, H, G, D, p.pool, p.table, p.width, tiles, n, None, p.scale)
    tiles[:, 0] = 1999
    assert torch.equal(K.attention_int4_prompt(q, H * D, H, G, D, pool, table, p.width, tiles, n, None, p.scale), want)


# ---------------------------------------------------------------------------- appending

@pytest.mark.parametrize("G,D", [(2, 64), (2, 128)])
def test_rows_whose_steps_are_subnormal(K, G, D):
    """Groups of numbers down to the smallest that bfloat16 has, whose steps are subnormal."""
    H, n = 2, 130
    p = Paged(H, G, D, [n], 141)
    x = torch.zeros(n, H + 2 * G, D, dtype=torch.float64, device="cuda")
    for i in range(n):
        x[i] = torch.randint(-200, 200, (H + 2 * G, D), generator=gen(i), device="cuda").double() * 2.0 ** (-133 + i % 13)
    x = x.bfloat16()
    append(K, p, x.view(n, -1), [0], [n])
    k, v = K.load_int4(p.pool, G, D, ints(list(range(n))), ints([0] * n), p.table, p.width)
    assert torch.equal(k.double(), plain.stands_for(x[:, H:H + G]).float().double()) and torch.equal(v.double(), plain.stands_for(x[:, H + G:]).float().double())


@pytest.mark.parametrize("G,D", [(2, 64), (2, 128)])
def test_numbers_next_to_a_border_of_two_codes(K, G, D):
    """Groups of a middle of one and steps of a quarter, and numbers so much smaller than the middle that their difference in float32 lies on a border, whichever side of it they are on."""
    H, n = 2, 64
    p = Paged(H, G, D, [n], 145)
    x = torch.randint(-4, 5, (n, H + 2 * G, D), generator=gen(146), device="cuda").double() * 0.25
    tiny = torch.rand(x.shape, generator=gen(147), device="cuda") < 0.5
    sign = torch.randint(0, 2, x.shape, generator=gen(148), device="cuda") * 2 - 1
    x = torch.where(tiny, sign * 2.0 ** -30, x)
    x[..., ::32], x[..., 1::32] = 2.875, -0.875
    x = (x * 2.0 ** torch.randint(-60, 60, (n, 1, 1), generator=gen(149), device="cuda")).bfloat16()
    append(K, p, x.view(n, -1), [0], [n])
    k, v = K.load_int4(p.pool, G, D, ints(list(range(n))), ints([0] * n), p.table, p.width)
    assert torch.equal(k.double(), plain.stands_for(x[:, H:H + G]).float().double()) and torch.equal(v.double(), plain.stands_for(x[:, H + G:]).float().double())


# ---------------------------------------------------------------------------- arguments

def test_windows_and_contexts_beyond_32_bits(K):
    """A window or a bound of positions that a 32-bit integer does not hold is one that leaves nothing out."""
    H, G, D = 14, 2, 64
    p = Paged(H, G, D, [1500, 300], 151)
    pos, row = [1499, 299], [0, 1]
    want = p.attention(K, pos, row)
    for window in (2 ** 31 - 1, 2 ** 31, 2 ** 32 + 5, 2 ** 40):
        assert torch.equal(p.attention(K, pos, row, window=window), want)
    q = randn(1800, H * D, seed=152).bfloat16()
    tiles = K.prefill_tiles([1500, 300], [0, 0], "cuda", K.PREFILL_TILE_TCGEN05)
    runs = [K.attention_int4_prompt(q, H * D, H, G, D, p.pool, p.table, p.width, tiles, 1800, w, p.scale) for w in (None, 2 ** 31 - 1, 2 ** 32 + 5, 2 ** 40)]
    assert all(torch.equal(runs[0], r) for r in runs[1:])
    for bound in (2 ** 31, 2 ** 32 + 100, 2 ** 40):
        p.check(p.attention(K, pos, row, bound=bound), pos, row)
    bounds = bounds_of(p)
    one, other = (K.select_pages(p.q, p.q.shape[1], H, G, D, bounds, p.table, p.width, ints(pos), ints(row), 5, most) for most in (1500, 2 ** 32 + 100))
    assert torch.equal(one.table, other.table) and torch.equal(one.pos, other.pos)


def test_rows_of_more_positions_than_an_integer_counts(K):
    from pico_engine.ops import KernelError
    p = Paged(2, 1, 64, [100], 155)
    wide = torch.full((1, 1 << 25), -1, dtype=torch.int32, device="cuda")
    wide[0, :2] = p.table[0, :2]
    for call in (lambda: K.attention_int4(p.q, p.q.shape[1], 2, 1, 64, p.pool, wide, 1 << 25, ints([99]), ints([0]), None, 1.0, 100),
                 lambda: K.attention_int4_selected(p.q, p.q.shape[1], 2, 1, 64, p.pool, K.SelectedPages(wide, ints([99])), 1.0)):
        with pytest.raises(KernelError, match="a row has at most"):
            call()
    narrow = wide[:, :(1 << 25) - 1].contiguous()
    got = K.attention_int4(p.q, p.q.shape[1], 2, 1, 64, p.pool, narrow, narrow.shape[1], ints([99]), ints([0]), None, p.scale, 100)
    assert torch.equal(got, p.attention(K, [99], [0]))


def test_calls_of_two_threads(K):
    """Calls that need little and much shared memory, from two threads at once: neither takes away what the other's launch needs."""
    from threading import Thread
    failed = []

    def select(pages, times):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                q, bounds = torch.zeros(1, 128, dtype=torch.bfloat16, device="cuda"), torch.zeros(1, 1, 2, 64, dtype=torch.bfloat16, device="cuda")
                table = torch.full((1, pages), -1, dtype=torch.int32, device="cuda")
                for _ in range(times):
                    K.select_pages(q, 128, 2, 1, 64, bounds, table, pages, ints([64 * pages - 1]), ints([0]), 4, 64 * pages)
        except Exception as e:                              # noqa: BLE001
            failed.append(e)

    def prompts(rows, times):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                q, pool = torch.zeros(1, 128, dtype=torch.bfloat16, device="cuda"), K.int4_pool(1, 1, 64, "cuda")
                table = torch.zeros(rows, 1, dtype=torch.int32, device="cuda")
                for _ in range(times):
                    K.attention_int4_prompt(q, 128, 2, 1, 64, pool, table, 1, ints([[rows - 1, 0, 1, 0]]), 1, None, 1.0)
        except Exception as e:                              # noqa: BLE001
            failed.append(e)

    for call, small, large in ((select, 2200, 9900), (prompts, 4000, 17900)):
        threads = [Thread(target=call, args=(n, 1500)) for n in (small, large, small)]
        for t in threads:
            t.start()
        for t in threads:
            t.join()
        torch.cuda.synchronize()
    assert not failed, failed[0]


@pytest.mark.parametrize("D", [64, 128])
def test_scales_and_products_at_the_ends(K, D):
    """Small queries against small keys under the largest scales, one token and prompts; scales that the kernels do not have are refused."""
    from pico_engine.ops import KernelError
    p = Paged(4, 2, D, [700, 90], 201)
    pos, row = [699, 89], [0, 1]
    p.pool = plain.pack((p.keys.double() * 2.0 ** -30).bfloat16().view(-1, 64, D), p.values.view(-1, 64, D)).view(p.n_pages, 2, -1)
    p.scale *= 2.0 ** 60
    q = (p.q.double() * 2.0 ** -30).bfloat16()
    for bound in (700, 1 << 21):
        p.check(p.attention(K, pos, row, q=q, bound=bound), pos, row, q=q)
    long = (randn(90, 4 * D, seed=202).double() * 2.0 ** -30).bfloat16()
    got = K.attention_int4_prompt(long, 4 * D, 4, 2, D, p.pool, p.table, p.width, K.prefill_tiles([0, 90], [0, 0], "cuda", K.PREFILL_TILE_TCGEN05), 90, None, p.scale)
    some = [0, 40, 89]
    p.check(got[some], some, [1] * 3, q=long[some], halves=True)
    args = (q, q.shape[1], 4, 2, D, p.pool)
    one = ints([3])
    for scale in (0.0, -1.0, 2.0 ** 60, float("inf"), float("nan")):
        for call in (lambda: K.attention_int4(*args, p.table, p.width, one, ints([0]), None, scale, 100), lambda: K.attention_int4_prompt(*args, p.table, p.width, ints([[0, 0, 1, 3]]), 1, None, scale),
                     lambda: K.attention_int4_selected(*args, K.SelectedPages(ints([[0], [1]]), ints([3, 3])), scale)):
            with pytest.raises(KernelError, match="scale must be positive and less than"):
                call()


# ---------------------------------------------------------------------------- tokens

@pytest.mark.parametrize("H,G,D", [(6, 2, 64), (14, 1, 128)])
@pytest.mark.parametrize("bound", [200, 1 << 21])
def test_sums_of_queries_keep_the_bits_of_float32(K, H, G, D, bound):
    """Scores that are the small difference of large products of middles with sums of queries: 128.25 and a few 2^-12 times 8,192, less 128.25 times 8,192."""
    p = Paged(H, G, D, [150, 70], 171)
    keys = torch.zeros_like(p.keys)
    keys[:, :, ::2, :32], keys[:, :, ::2, 32:64] = 8192.0, -8192.0
    if D == 128:
        keys[:, :, 1::2, 64:96], keys[:, :, 1::2, 96:] = -8192.0, 8192.0
    p.pool = plain.pack(keys.view(-1, 64, D), p.values.view(-1, 64, D)).view(p.n_pages, G, 80 * D)
    q = torch.zeros(2, H, D, device="cuda")
    for b in range(0, D, 32):
        q[..., b], q[..., b + 9] = 128.0, 0.25
    extra = torch.tensor([(1 + h % 3) * 2.0 ** -12 for h in range(H)], device="cuda")
    q[..., 17], q[1, :, D - 5] = extra, 2 * extra                             # in the first group, and in the last one's too
    q = q.bfloat16().view(2, H * D)
    got = K.attention_int4(q, H * D, H, G, D, p.pool, p.table, p.width, ints([149, 69]), ints([0, 1]), None, 0.5, bound).double().view(2, H, D)
    for t, n in enumerate((150, 70)):
        blocks = p.pool[p.table[t, :n // 64 + 1].long()]
        k, v, part, _ = (x.view(-1, G, 64, D).transpose(0, 1).reshape(G, -1, D)[:, :n] for x in plain.unpack(blocks.flatten(0, 1)))
        for h in range(H):
            g = h * G // H
            w = torch.softmax(k[g] @ q[t].double().view(H, D)[h] * 0.5, 0)
            # sums and scores have no rounding here; weights are rounded (on v), once more behind a step, and the result
            bound_of = 2.0 ** -8 * (w @ (v[g].abs() + part[g].abs()) + (w @ v[g]).abs()) + 2.0 ** -18
            assert ((got[t, h] - w @ v[g]).abs() <= bound_of).all(), (t, h)


@pytest.mark.parametrize("H,G,D", [(14, 2, 64), (28, 4, 128)])
@pytest.mark.parametrize("window", [None, 300])
@pytest.mark.parametrize("bound", [3100, 1 << 21])
def test_pages_read_early_or_late_are_the_same(K, H, G, D, window, bound):
    """``early_pages`` moves a wait, no result: behind an append of the tokens' own rows, one that ends a page and one that begins one among them."""
    lengths = [64 * 40 + 1, 64 * 7, 1, 3000, 65] * (1 if bound == 3100 else 30)
    p = Paged(H, G, D, lengths, 161)
    T = len(lengths)
    pos, row = ints([n - 1 for n in lengths]), ints(list(range(T)))
    cos, sin = (randn(4000, D // 2, seed=s) for s in (1, 2))
    for seed in range(6):
        x, outs, pools = randn(T, (H + 2 * G) * D, seed=163 + seed).bfloat16(), [], []
        for early in (True, False):
            pool = p.pool.clone()
            torch.cuda.synchronize()
            q = K.store_int4(x, H, G, D, cos, sin, pos, row, pool, p.table, p.width)
            outs.append(K.attention_int4(q, H * D, H, G, D, pool, p.table, p.width, pos, row, window, p.scale, bound, early_pages=early))
            pools.append(pool)
        assert torch.equal(*outs) and torch.equal(*pools)
    p.pool, some = pools[0], list(range(0, T, 7))
    p.check(outs[0][some], [lengths[i] - 1 for i in some], some, q=q[some], window=window)


# ---------------------------------------------------------------------------- the part and the engine

@pytest.fixture(scope="module")
def folder(tmp_path_factory):
    from conftest import make_weights, write_model
    from test_int4_engine_gpu import LONG
    return write_model(tmp_path_factory.mktemp("int4_edges") / "long", LONG, make_weights(LONG, 8, sharp=True)), LONG


def test_a_prompts_last_piece_of_one_token_attends_to_everything(folder):
    """However a prompt is cut, its tokens see all of it; decoded tokens see the pages that are selected."""
    from pico_engine import Engine
    from pico_engine.engine.engine import EngineBackend
    from pico_engine.sampling import Sampler, SamplingParams
    from test_int4_engine_gpu import prompts
    path, cfg = folder
    texts, logits = prompts(cfg, [6 * 64 + 1, 65, 700]), {}
    for attend in (None, 4):
        eng = Engine(path, cache="int4", attend_pages=attend, max_context=1500, max_tokens_in_cache=64 * 60)
        eng.ensure_cache(64 * 60, 1500)
        eng.prefill_tokens_per_step = 64
        slots = [eng.cache.open() for _ in texts]
        back = EngineBackend(eng, Sampler(SamplingParams(0.0, 0, 1.0, 0)), False)
        logits[attend] = [back._prompts(slots[:1], texts[:1])[0], *back._prompts(slots[1:], texts[1:])]
        logits[attend].append(eng.stepper.step(slots, [[3], [4], [5]]))
    for a, b in zip(logits[None][:3], logits[4][:3]):
        assert torch.equal(a, b)
    assert not torch.equal(logits[None][3], logits[4][3])


def test_selection_without_a_layer_that_selects_is_refused(tmp_path):
    from conftest import TINY_C, make_weights, write_model
    from pico_engine import Engine
    cfg = {**TINY_C, "max_position_embeddings": 512, "use_sliding_window": True, "sliding_window": 100, "max_window_layers": 0}
    path = write_model(tmp_path / "windows", cfg, make_weights(cfg, 5))
    Engine(path, cache="int4")
    with pytest.raises(ValueError, match="attend_pages"):
        Engine(path, cache="int4", attend_pages=4)


@pytest.mark.parametrize("attend", [None, 4])
def test_captured_steps_go_by_the_rows_they_have(folder, attend):
    """An engine set up for long contexts launches for the ones it has: no selection before a row has more pages than are kept, prompts with scratch for their own positions; and the
    results are those of steps that are not captured, across the borders."""
    from pico_engine import Engine
    from test_int4_engine_gpu import prompts
    path, cfg = folder
    eng = Engine(path, cache="int4", attend_pages=attend, max_context=2000)
    texts = prompts(cfg, [230, 30, 100])
    got = [eng.generate(texts, max_tokens=60, temperature=0.0, stop_token_ids=()) for _ in range(3)]
    contexts = {key[4] for key in eng._graphs}
    # (four rows of two key heads are few pairs, whose kernel changes at 15 pages: 512 positions have it as they do, 1,024 do not)
    assert contexts == ({512} if attend is None else {256, 2000}) and all(g.graph is not None for g in eng._graphs.values())
    assert {(key[1], key[2]) for key in eng.stepper._prompt_graphs} == {(384, 384)} and all(g.graph is not None for g in eng.stepper._prompt_graphs.values())
    plainly = eng.generate(texts, max_tokens=60, temperature=0.0, stop_token_ids=(), use_graph=False)
    assert got[0] == got[1] == got[2] == plainly
    short = next(iter(eng._graphs.values()))
    if attend is not None and short.max_context == 256:
        slot = eng.cache.open()
        eng.stepper.step([slot], [[1] * 256])
        with pytest.raises(ValueError, match="reaches further"):
            short.launch([slot], [1], [0], [1])
        eng.cache.close(slot)
    eng.cache.check()


def test_the_bound_of_a_captured_steps_positions(K):
    """The largest power of two whose kernels are those of the rows at hand."""
    from types import SimpleNamespace
    from pico_engine.cache import Cache
    from pico_engine.engine.step import Stepper
    from test_int4_engine_gpu import part_of
    part = part_of(14, 2, 64, None, True)
    cache = Cache([part.cache_needs()], 64 * 1200, 4, torch.bfloat16, "cuda", int4=True, bounds=True)
    model = SimpleNamespace(plan=SimpleNamespace(vocab_size=1 << 20), dtype=torch.bfloat16, int4_shapes=lambda *a: (part.int4_shape(*a),))
    slot = cache.open()
    for attend, rows, length, want in ((None, 64, 999, 16384), (None, 64, 16384, 32768), (None, 1, 500, 512), (None, 1, 3000, 32768), (None, 32, 1000, 32768), (64, 64, 1000, 4096),
                                       (64, 64, 4096, 32768), (64, 64, 4095, 4096), (100, 64, 5000, 6400), (100, 64, 6399, 6400),
                                       (100, 64, 6400, 32768)):
        stepper = Stepper(model, cache, 32768, attend)
        cache.lengths[slot] = length
        assert stepper.launch_context(rows, [slot]) == want, (attend, rows, length)
    cache.lengths[slot] = 0
    stepper = Stepper(model, cache, 32768, None)
    for tokens, start, n, want in ((128, 0, 100, 128), (2048, 0, 2000, 2048), (512, 9000, 400, 16384), (512, 0, 33, 512)):
        cache.lengths[slot] = start
        assert stepper.prompt_context(tokens, [slot], [n]) == want
    cache.lengths[slot] = 0


@pytest.mark.parametrize("nh,nkv,hd,keep", [(14, 2, 64, None), (8, 2, 128, 3)])
def test_a_part_that_reads_another_ones_cache(nh, nkv, hd, keep):
    """Keys and values are the owner's; the reader turns its own queries and stores nothing."""
    from types import SimpleNamespace
    from pico_engine.cache import Cache
    from pico_engine.engine.step import Stepper
    from pico_engine.ops import linear
    from test_int4_engine_gpu import part_of, rows_of
    owner, reader = part_of(nh, nkv, hd, None, True), part_of(nh, nkv, hd, None, True)
    reader.w_qkv.copy_(reader.w_qkv.flip(1))
    cache = Cache([owner.cache_needs()], 64 * 20, 2, torch.bfloat16, "cuda", int4=True, bounds=keep is not None)
    stepper = Stepper(SimpleNamespace(plan=SimpleNamespace(vocab_size=1 << 20), dtype=torch.bfloat16), cache, 1024, keep)
    slots = [cache.open() for _ in range(2)]
    keys, values = ([torch.zeros(0, nkv, hd, dtype=torch.float64, device="cuda") for _ in slots] for _ in range(2))
    for step, lens in enumerate([[300, 70], [1, 1], [1, 1]]):
        lay, host, starts = stepper.describe(slots, lens, None, None)
        ctx = stepper.context(lay, stepper.upload(host), lens, starts, slots)
        h = torch.randn(sum(lens), 96, generator=gen(step), device="cuda").bfloat16()
        owner._attend(h, ctx, 0, True)
        held, ends = cache.groups[0].k.clone(), None if keep is None else cache.groups[0].bounds.clone()
        got = reader._attend(h, ctx, 0, False).double().view(-1, nh, hd)
        assert torch.equal(held, cache.groups[0].k) and (keep is None or torch.equal(ends, cache.groups[0].bounds))
        for s, n in zip(slots, lens):
            cache.advance(s, n)
        rows = [linear(h, part.w_qkv, part.b_qkv, out_dtype=torch.bfloat16).view(-1, nh + 2 * nkv, hd).double() for part in (owner, reader)]
        at = 0
        for b, (start, n) in enumerate(zip(starts, lens)):
            c, s = (t.cuda().double()[start:start + n, None] for t in owner._tables(ctx))
            turned = []
            for x in rows:
                lo, hi = x[at:at + n, :nh + nkv, :hd // 2], x[at:at + n, :nh + nkv, hd // 2:]
                turned.append(torch.cat([lo * c - hi * s, lo * s + hi * c], -1).float().bfloat16())
            keys[b] = torch.cat([keys[b], plain.stands_for(turned[0][:, nh:])])
            values[b] = torch.cat([values[b], plain.stands_for(rows[0][at:at + n, nh + nkv:])])
            for i in sorted({0, n // 2, n - 1}):
                w, unit = rows_of(turned[1][i, :nh], keys[b][:start + i + 1], values[b][:start + i + 1], hd ** -0.5, None, keep if all(m == 1 for m in lens) else None)
                assert (got[at + i] - w).abs().max() <= unit, (step, b, i)
            at += n


@pytest.mark.parametrize("window,attend", [(False, None), (False, 3), (True, None)])
def test_every_call_that_a_generation_makes(tmp_path, monkeypatch, K, window, attend):
    """Prompts, tokens and selected pages of an engine, call by call: what is appended is what the codes of the call's own rows stand for, bit by bit, and attention is within its bounds of the plain
    form over the pool's bytes.  (Logits of a whole model allow for more: a bfloat16 rounding in front of a code moves the code.)"""
    from conftest import TINY_C, make_weights, write_model
    from pico_engine import Engine
    from test_int4_engine_gpu import LONG, prompts
    cfg = TINY_C if window else LONG
    eng = Engine(write_model(tmp_path / "model", cfg, make_weights(cfg, 9, sharp=True)), cache="int4", attend_pages=attend, max_context=512)
    calls = {"store": 0, "prompt": 0, "token": 0, "selected": 0}
    store, token, prompt, selected = K.store_int4, K.attention_int4, K.attention_int4_prompt, K.attention_int4_selected

    def blocks_of(pool, table, row, n):
        return pool[table[row, :n].clamp(min=0).long()]

    def rows_checked(got, q, H, G, D, pool, table, pos, row, window, scale, halves):
        for i in sorted({0, len(pos) // 3, len(pos) - 1}):
            n, j = pos[i] // PAGE + 1, torch.arange((pos[i] // PAGE + 1) * PAGE, device="cuda")
            seen = (j <= pos[i]) & ((j > pos[i] - window) if window else (j >= 0)) & (table[row[i], :n] >= 0).repeat_interleave(PAGE)
            want, bound = plain.attend(q[i].view(H, D), blocks_of(pool, table, row[i], n), seen[None].expand(G, -1), scale, halves)
            assert ((got[i].double().view(H, D) - want).abs() <= bound + 1e-30).all(), (pos[i], window)

    def stored(qkv, H, G, D, cos, sin, pos, row, pool, table, width, out=None):
        q = store(qkv, H, G, D, cos, sin, pos, row, pool, table, width, out)
        x = qkv.view(-1, H + 2 * G, D).double()
        c, s = (t.double()[pos.long()][:, None] for t in (cos, sin))
        a, b = x[:, :H + G, :D // 2], x[:, :H + G, D // 2:]
        turned = torch.cat([a * c - b * s, a * s + b * c], -1)
        k, v = K.load_int4(pool, G, D, pos, row, table, width)
        assert torch.equal(k.double(), plain.stands_for(turned[:, H:].float().bfloat16()).float().double()) and torch.equal(v.double(), plain.stands_for(x[:, H + G:]).float().double())
        size = torch.cat([(a * c).abs() + (b * s).abs(), (a * s).abs() + (b * c).abs()], -1)[:, :H]
        assert ((q.double().view(-1, H, D) - turned[:, :H]).abs() <= 2.0 ** -8 * turned[:, :H].abs() + 2.0 ** -22 * size + 1e-30).all()
        calls["store"] += 1
        return q

    def tokens(q, stride, H, G, D, pool, table, width, pos, row, window, scale, most, out=None, early_pages=False):
        got = token(q, stride, H, G, D, pool, table, width, pos, row, window, scale, most, out, early_pages)
        rows_checked(got, q, H, G, D, pool, table, pos.tolist(), row.tolist(), window, scale, False)
        calls["token"] += 1
        return got

    def prompted(q, stride, H, G, D, pool, table, width, tiles, n, window, scale, out=None, max_context=None):
        got = prompt(q, stride, H, G, D, pool, table, width, tiles, n, window, scale, out, max_context)
        where = {r[1] + i: (r[3] + i, r[0]) for r in tiles.tolist() for i in range(r[2])}
        assert sorted(where) == list(range(n))
        rows_checked(got, q, H, G, D, pool, table, [where[i][0] for i in range(n)], [where[i][1] for i in range(n)], window, scale, True)
        calls["prompt"] += 1
        return got

    def chosen_pages(q, stride, H, G, D, pool, pages, scale, out=None):
        got = selected(q, stride, H, G, D, pool, pages, scale, out)
        for i in range(q.shape[0]):
            for g in range(G):
                ids, at = pages.table[i * G + g].tolist(), int(pages.pos[i * G + g])
                ids = [x for x in ids if x >= 0]
                assert len(ids) <= attend and at < len(ids) * PAGE
                seen = torch.arange(len(ids) * PAGE, device="cuda") <= at
                part = q[i].view(G, -1, D)[g]
                want, bound = plain.attend(part, pool.flatten(0, 1)[ids][:, None], seen[None], scale)
                assert ((got[i].double().view(G, -1, D)[g] - want).abs() <= bound + 1e-30).all()
        calls["selected"] += 1
        return got

    for name, f in (("store_int4", stored), ("attention_int4", tokens), ("attention_int4_prompt", prompted), ("attention_int4_selected", chosen_pages)):
        monkeypatch.setattr(K, name, f)
    texts = prompts(cfg, [240, 30, 64, 129] if not window else [200, 30, 64, 129])
    eng.prefill_tokens_per_step = 150
    eng.generate(texts, max_tokens=20, temperature=0.0, stop_token_ids=(), use_graph=False)
    assert calls["store"] > 20 and calls["prompt"] >= 3 and (calls["selected"] if attend else calls["token"]) >= 19
