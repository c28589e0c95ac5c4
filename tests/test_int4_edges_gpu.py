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
