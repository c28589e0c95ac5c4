"""The 4-bit cache without a GPU: the plain form against itself, and what the entry points refuse before anything is launched."""
import pytest
import torch

import plain_int4 as plain
from pico_engine.ops import KernelError, kernels as K


@pytest.mark.parametrize("D", [64, 128])
def test_blocks_hold_what_rows_stand_for(D):
    g = torch.Generator().manual_seed(D)
    k, v = (torch.randn(3, 64, D, generator=g).bfloat16() * s for s in (2.0, 0.01))
    k[0, 5, :32] = 1.5                                   # equal numbers: held as they are
    v[1, 7, 32:64] = 0.0
    blocks = plain.pack(k, v)
    keys, values, _, _ = plain.unpack(blocks)
    assert blocks.shape == (3, K.int4_page_bytes(D))
    assert torch.equal(keys, plain.stands_for(k)) and torch.equal(values, plain.stands_for(v))
    assert (keys[0, 5, :32] == 1.5).all() and (values[1, 7, 32:64] == 0).all()
    for x, y in ((k, keys), (v, values)):
        a = x.double().unflatten(-1, (-1, 32))
        spread, middle = a.amax(-1) - a.amin(-1), (a.amax(-1) + a.amin(-1)).abs() / 2
        # half a step (spread / 30); the step is off by 2^-8 of itself at 7.5 steps, the middle by 2^-8
        off = (spread / 30) * (1 + 2.0 ** -8) + 7.5 * spread / 15 * 2.0 ** -8 + middle * 2.0 ** -8
        assert ((y - x.double()).abs().unflatten(-1, (-1, 32)) <= off[..., None] + 1e-30).all()


def test_every_bit_of_a_block_is_used_once():
    for D in (64, 128):
        seen = torch.zeros(20 * D, 32, dtype=torch.int64)
        for which in (False, True):
            word, sign, magnitude, _, _ = plain.places(D, which)
            for bit in [sign] + [(magnitude + j) % 32 for j in range(3)]:
                seen.index_put_((word.reshape(-1), bit.reshape(-1)), torch.ones(64 * D, dtype=torch.int64), accumulate=True)
        assert (seen[:16 * D] == 1).all() and (seen[16 * D:] == 0).all()
        numbers = torch.cat([torch.stack(plain.places(D, w)[3:]).reshape(-1) for w in (False, True)])
        assert numbers.unique().tolist() == list(range(32 * D, 40 * D))


def test_what_can_be_held():
    assert K.int4_takes(torch.bfloat16, 14, 2, 64) and K.int4_takes(torch.bfloat16, 28, 4, 128)
    assert not K.int4_takes(torch.float32, 14, 2, 64) and not K.int4_takes(torch.bfloat16, 14, 2, 96) and not K.int4_takes(torch.bfloat16, 14, 4, 64)


def test_heads_are_checked_before_tensors():
    t = torch.zeros(1)
    for call in (lambda h, g, d: K.store_int4(t, h, g, d, None, None, t, t, t, t, 1), lambda h, g, d: K.attention_int4(t, h * d, h, g, d, t, t, 1, t, t, None, 1.0, 1),
                 lambda h, g, d: K.attention_int4_prompt(t, h * d, h, g, d, t, t, 1, t, 1, None, 1.0), lambda h, g, d: K.select_pages(t, h * d, h, g, d, t, t, 1, t, t, 1, 1)):
        for heads in ((3, 2, 64), (4, 0, 64), (4, 2, 96), (0, 1, 64)):
            with pytest.raises(KernelError, match="4-bit caches take"):
                call(*heads)
        with pytest.raises(KernelError, match="must live on a CUDA device"):
            call(4, 2, 64)


def test_pages_of_codes_only_where_all_their_readers_take_them():
    from types import SimpleNamespace as N
    from pico_engine.cache import CacheNeeds
    from pico_engine.cache.needs import KVNeed
    from pico_engine.parts.model import DecoderModel
    takes, other = CacheNeeds(kv=KVNeed(2, 64, may_be_int4=True)), CacheNeeds(kv=KVNeed(2, 64))
    model = object.__new__(DecoderModel)
    model.layers = [N(cache_needs=lambda n=n: n) for n in (takes, takes, other, takes)]
    model.plan = N(embedding_pairs=None, schedule=[N(layer=0, cache_of=None), N(layer=1, cache_of=None), N(layer=2, cache_of=0), N(layer=3, cache_of=1), N(layer=3, cache_of=None)])
    assert model.cache_needs() == [other, takes, None, None, takes]
