"""The page tables that stay on the device (CPU): what a step sends for them, laid out as the kernel does it, is what the cache holds."""
import random

import torch

from pico_engine.cache import Cache, CacheNeeds, KVNeed, PAGE, pages_for
from pico_engine.engine.tables import ResidentTables


def cache_of(max_tokens=4096, max_seqs=8, groups=1):
    needs = [CacheNeeds(kv=KVNeed(1 + g, 16, None)) for g in range(groups)]
    return Cache(needs, max_tokens, max_seqs, torch.float32, "cpu", allocate=False)


def lay_out(resident, slots, starts, held, pages):
    """The tables of a step of one token a row, by the kernel's contract: row b takes ceil((start + 1) / 64) - held of the numbers, in the rows' order."""
    at, tables = 0, []
    for s, start, h in zip(slots, starts, held):
        need = max(pages_for(start + 1), int(h))
        for w in range(int(h), need):
            resident[s, w] = pages[at]
            at += 1
        tables.append(resident[s, :need].tolist())
    assert at == len(pages)                                              # (numbers that no row takes would be the next row's)
    return tables


def step(tables, cache, slots):
    """One step of a token each; every row's table has to name the sequence's own pages."""
    for s in slots:
        cache.reserve(s, 1)
    for g in range(len(cache.groups)):
        held, pages, learned = tables.fresh(g, slots)
        got = lay_out(tables.tables[g], slots, [cache.length(s) for s in slots], held, pages)
        assert got == [cache.groups[g].table[s][:pages_for(cache.length(s) + 1)] for s in slots]
        tables.learn(g, learned)
    for s in slots:
        cache.advance(s, 1)


def test_a_sequence_that_holds_more_pages_than_a_step_needs():
    """Pages reserved ahead stay out of the step until its positions reach them; those of the rows behind are their own."""
    cache = cache_of(groups=2)
    tables = ResidentTables(cache, 512)
    a, b, c = (cache.open() for _ in range(3))
    cache.reserve(a, 200)
    cache.reserve(b, 65)
    for _ in range(2 * PAGE + 3):
        step(tables, cache, [a, b, c])
    cache.reserve(b, 5 * PAGE)
    step(tables, cache, [c, b, a])
    cache.close(b)
    b = cache.open()
    cache.reserve(b, 130)
    step(tables, cache, [b, a, c])


def test_a_step_that_is_not_launched_teaches_the_device_nothing():
    """Until its step has been launched, a page is sent again."""
    cache = cache_of()
    tables = ResidentTables(cache, 512)
    a, b = cache.open(), cache.open()
    step(tables, cache, [b])
    cache.reserve(a, 1)
    first = tables.fresh(0, [a, b, cache.idle_slot])
    again = tables.fresh(0, [a, b, cache.idle_slot])
    assert first[0].tolist() == again[0].tolist() == [0, 1, 1] and first[1] == again[1] == cache.groups[0].table[a] and first[2] == again[2]
    tables.learn(0, first[2])
    assert tables.fresh(0, [a, b])[1] == []


def test_sequences_that_come_go_fork_and_reserve_ahead():
    rng = random.Random(3)
    cache = cache_of(max_tokens=200 * PAGE, max_seqs=12)
    tables = ResidentTables(cache, 40 * PAGE)
    live = []
    for _ in range(400):
        what = rng.random()
        if what < 0.1 and len(live) < 10:
            live.append(cache.open())
            if rng.random() < 0.5:
                n = rng.randint(1, 300)
                cache.reserve(live[-1], n)
                cache.advance(live[-1], rng.choice([n, n, 0, n // 2]))
        elif what < 0.15 and live and len(live) < 10:
            live += cache.fork(rng.choice(live), rng.randint(1, 2))
        elif what < 0.2 and live:
            cache.close(live.pop(rng.randrange(len(live))))
        elif what < 0.3 and live:
            s = rng.choice(live)
            cache.reserve(s, min(rng.randint(1, 200), 40 * PAGE - cache.length(s)))
        rows = [s for s in rng.sample(live, rng.randint(0, len(live))) if cache.length(s) + 1 < 40 * PAGE]
        if rows:
            step(tables, cache, rows)
    cache.check()
