"""Refusals of the operators for several answers to a prompt, found before anything is launched: on the CPU, with tensors that say they are on a device."""
import pytest
import torch

from pico_engine.ops import kernels as K
from pico_engine.ops.library import KernelError


class OnDevice(torch.Tensor):
    is_cuda = True


def there(t):
    return t.as_subclass(OnDevice)


def i32(*shape):
    return there(torch.zeros(*shape, dtype=torch.int32))


def f32(*shape):
    return there(torch.zeros(*shape))


def refused(call, what):
    with pytest.raises(KernelError, match=what):
        call()


# ---------------------------------------------------------------------------- attention

def attention(**change):
    bf = lambda *s: there(torch.zeros(*s, dtype=torch.bfloat16))         # noqa: E731
    a = dict(q=bf(3, 14 * 64 + 8), q_stride=14 * 64 + 8, n_heads=14, n_kv_heads=2, head_dim=64, k_pool=bf(9, 2, 64, 64), v_pool=bf(9, 2, 64, 64),
             block_table=i32(3, 4), table_stride=4, tok_pos=i32(3), tok_row=i32(3), groups=i32(3, 4), window=None, scale=0.125, max_context=256)
    a.update(change)
    return lambda: K.attention_shared(**a)


@pytest.mark.parametrize("change,what", [
    (dict(q=torch.zeros(3, 904, dtype=torch.bfloat16)), "q must live on a CUDA device"),
    (dict(q=f32(3, 904)), "q must be torch.bfloat16"),
    (dict(k_pool=there(torch.zeros(9, 2, 32, 64, dtype=torch.bfloat16)), v_pool=there(torch.zeros(9, 2, 32, 64, dtype=torch.bfloat16))), "cache pool must be"),
    (dict(v_pool=there(torch.zeros(8, 2, 64, 64, dtype=torch.bfloat16))), "v_pool must have shape"),
    (dict(head_dim=32), "head sizes"), (dict(scale=0.0), "positive scale"), (dict(n_heads=13), "query heads"), (dict(n_heads=258, q_stride=258 * 64), "at most 128 query heads"),
    (dict(q_stride=900), "multiple of 8"), (dict(q_stride=888), "rows of 896"), (dict(q_stride=2000), "rows of 896"),
    (dict(tok_pos=i32(1025)), "at most 1024 rows"), (dict(k_pool=there(torch.zeros(0, dtype=torch.bfloat16)), v_pool=there(torch.zeros(0, dtype=torch.bfloat16))), "cache pool must be"),
    (dict(tok_row=i32(2)), "tok_row must have shape"), (dict(groups=i32(2, 4)), "groups must have shape"),
    (dict(max_context=0), "max_context"), (dict(keep_first=-1), "not negative"), (dict(window=-4), "not negative"),
    (dict(sinks=f32(2)), "sinks must have shape"), (dict(slopes=f32(2)), "slopes must have shape"),
    (dict(out=there(torch.zeros(3, 64, dtype=torch.bfloat16))), "out must have shape"),
])
def test_attention_shared_refuses(change, what):
    refused(attention(**change), what)


def test_shared_groups():
    assert K.shared_group_rows([(2, 128, 1), (1, 0, 0), (3, 64, 0)]) == [(0, 2, 128, 1)] * 2 + [(2, 1, 0, 2)] + [(3, 3, 64, 3)] * 3
    assert K.shared_groups([], "cpu").shape == (0, 4)
    for bad in ((0, 64, 0), (2, 63, 0), (2, -64, 0), (2, 64, 2), (2, 64, -1)):
        refused(lambda: K.shared_group_rows([bad]), "whole pages")


# ---------------------------------------------------------------------------- rules on logits

def rules(**change):
    a = dict(logits=f32(4, 100), slots=i32(4), history=there(torch.zeros(6, 100, dtype=torch.int16)), penalties=f32(4, 3), bias_range=i32(4, 2), bias_ids=i32(9),
             bias_values=f32(9), masks=i32(2, 4), mask_rows=i32(4))
    a.update(change)
    return lambda: K.adjust_logits(**a)


@pytest.mark.parametrize("change,what", [
    (dict(logits=torch.zeros(4, 100)), "logits must live on a CUDA device"), (dict(logits=f32(100)), "rows, vocabulary"),
    (dict(logits=there(torch.zeros(4, 100, dtype=torch.bfloat16))), "logits must be torch.float32"),
    (dict(slots=None), "go together"), (dict(penalties=None), "go together"), (dict(history=None), "go together"),
    (dict(history=i32(6, 100)), "history must be torch.int16"), (dict(history=there(torch.zeros(6, 99, dtype=torch.int16))), "history must have shape"),
    (dict(penalties=f32(4, 2)), "penalties must have shape"), (dict(bias_range=None), "go together"), (dict(bias_values=f32(8)), "bias_values must have shape"),
    (dict(bias_range=i32(5, 2)), "bias_range must have shape"), (dict(masks=None), "go together"), (dict(masks=i32(2, 3)), "masks must have shape"),
    (dict(mask_rows=i32(3)), "mask_rows must have shape"), (dict(states=i32(6)), "go together"), (dict(mask_rows=None), "go together"),
    (dict(mask_rows=None, states=i32(5)), "a row a slot each"), (dict(mask_rows=None, states=i32(6, 1)), "states must have shape"),
    (dict(slots=i32(3)), "slots must have shape"), (dict(slots=None, history=None, penalties=None, mask_rows=None, states=i32(6)), "go together"), (dict(out=f32(4, 99)), "out must have shape"),
    (dict(logits=there(torch.zeros(100, 4).T)), "logits must be contiguous"),
])
def test_adjust_logits_refuses(change, what):
    refused(rules(**change), what)


def test_adjust_logits_refuses_too_many_rows():
    refused(lambda: K.adjust_logits(f32(65536, 1)), "65,535 rows")
    assert K.adjust_logits(f32(0, 5)).shape == (0, 5) and K.adjust_logits(f32(5, 0)).shape == (5, 0)


@pytest.mark.parametrize("change,what", [
    (dict(tokens=i32(3, 2)), "one row"), (dict(slots=i32(2)), "slots must have shape"), (dict(history=i32(4, 100)), "must be torch.int16"),
    (dict(history=None), "needs a history"), (dict(states=i32(4)), "needs a history"), (dict(states=i32(5), transitions=i32(3, 100)), "states must have shape"),
    (dict(states=i32(4), transitions=i32(3, 99)), "transitions must have shape"),
])
def test_note_tokens_refuses(change, what):
    a = dict(history=there(torch.zeros(4, 100, dtype=torch.int16)), slots=i32(3), tokens=i32(3))
    a.update(change)
    refused(lambda: K.note_tokens(**a), what)


# ---------------------------------------------------------------------------- the tables of a step

@pytest.mark.parametrize("change,what", [
    (dict(slots=i32(2)), "starts must have shape"), (dict(lens=f32(3)), "lens must be torch.int32"), (dict(resident=i32(12)), "page tables"),
    (dict(tables=i32(12)), "page tables"), (dict(tables=i32(4, 5)), "tables must have shape"), (dict(row_first=i32(3)), "row_first must have shape"),
    (dict(places=i32(6)), "places must have shape"), (dict(pages=i32(2, 2)), "pages must have shape"),
    (dict(slots=i32(0), starts=i32(0), lens=i32(0), held=i32(0), tables=i32(0, 5), row_first=i32(1)), "at least one row"),
])
def test_step_tables_refuses(change, what):
    a = dict(slots=i32(3), starts=i32(3), lens=i32(3), held=i32(3), pages=i32(4), resident=i32(6, 8), tok_pos=i32(7), tok_row=i32(7), row_first=i32(4),
             places=i32(7), tables=i32(3, 5))
    a.update(change)
    refused(lambda: K.step_tables(**a), what)


# ---------------------------------------------------------------------------- whether rows are read together

def test_shared_bytes_at_most():
    """What rows do not read again: nothing of one row, of others what the first reads, which a window and its kept keys bound."""
    assert K.shared_bytes_at_most(1, 2, 64, 10 ** 6) == 0 == K.shared_bytes_at_most(0, 2, 64, 10 ** 6)
    assert K.shared_bytes_at_most(16, 2, 64, 4096) == 15 * 4096 * 2 * 64 * 4
    assert K.shared_bytes_at_most(64, 4, 128, 30000, 100) == K.shared_bytes_at_most(64, 4, 128, 100) == 63 * 100 * 4 * 128 * 4
    assert K.shared_bytes_at_most(64, 4, 128, 30000, 100, 4) == 63 * 104 * 4 * 128 * 4
    assert K.shared_bytes_at_most(64, 4, 128, 90, 100, 4) == K.shared_bytes_at_most(64, 4, 128, 90) == K.shared_bytes_at_most(64, 4, 128, 90, 0, 4)
    assert not K.sharing_pays(K.shared_bytes_at_most(64, 4, 128, 30000, 100)) and K.sharing_pays(K.shared_bytes_at_most(64, 4, 128, 30000))
