"""Attention over shared pages and rules on logits where they can go wrong unseen: beside tests/test_answers_gpu.py, whose cases and oracle these use.

Attention over many keys, by rows: an entry's bound of 2^-8 of sum p |v| is far above a result in which random values cancel.  The roundings of the probabilities do
not hang together: an error sum_j d_j p_j v_j with |d_j| <= 2^-8 (half a step of bfloat16, each its own) has a root mean square of 2^-8 sqrt(sum p^2 v^2) at most, the result's
rounding 2^-8 of the result.  Over a row's entries (320 or more, in which values are their own) the root mean square of the error stays within the sum of
the two; uniform roundings come to 0.29 of it, and a page of 64 keys left out to 2.9 times it or more (both worked out for these cases in 64 bits)."""
import pytest
import torch

from test_answers_gpu import Answers, K, adjust, agree, gen, ints, rules_case, rules_want      # noqa: F401  (K: the fixture)

pytestmark = pytest.mark.gpu

PAGE = 64


# ---------------------------------------------------------------------------- attention

def visible(a, t, pos, window, keep):
    """The keys that row t sees, of those its row of the table names."""
    j = torch.arange(min(pos + 1, a.table.shape[1] * PAGE), device="cuda")
    return j[(j > pos - window) | (j < keep)] if window else j


def alone(a, t, pos, window=None, keep=0, sinks=False):
    """(result, sum p |v|, sum p^2 v^2) of row t in 64 bits; zeros where it sees nothing."""
    j = visible(a, t, pos, window, keep)
    j = j[a.table[t].long()[j // PAGE] >= 0]
    page = a.table[t].long()[j // PAGE]
    k, v = (x[page, :, j % PAGE].double().repeat_interleave(a.nh // a.nkv, dim=1) for x in (a.k, a.v))
    s = torch.einsum("hd,nhd->hn", a.rows[t, :a.nh * a.hd].double().view(a.nh, a.hd), k) * a.hd ** -0.5
    if sinks:
        s = torch.cat([s, a.sinks.double()[:, None]], dim=1)
    if s.shape[1] == 0:
        return (torch.zeros(a.nh * a.hd, dtype=torch.double, device="cuda"),) * 3
    p = torch.softmax(s, dim=1)[:, :len(j)]
    return tuple(torch.einsum("hn,nhd->hd", x, y).reshape(-1) for x, y in ((p, v), (p, v.abs()), (p ** 2, v ** 2)))


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("window,keep,sinks", [(100, 0, False), (100, 0, True), (64 * 9, 0, False), (100, 70, False), (100, 200, True), (1, 1, False)])
@pytest.mark.parametrize("beyond", [[0, 1, 2, 3, 4], [1], [4], [0, 2]])
def test_a_window_beyond_the_table(K, hd, window, keep, sinks, beyond):
    """Rows whose positions have left the table, and their windows with them, see the kept keys and no more, zeros where there are none; the others what they always do.  A table
    entry past the newest token's page is -1."""
    a = Answers(6, 2, hd, [(192, [64, 128, 3]), (0, [100]), (128, [70])], seed=hd)
    pos = list(a.pos)
    for t in beyond:
        a.pos[t] = a.width * PAGE + 2000 * (t + 1)
    want = [alone(a, t, p, window, keep, sinks) for t, p in enumerate(a.pos)]
    out = torch.full((a.T, a.nh * hd), 7.0, dtype=torch.bfloat16, device="cuda")
    groups = K.shared_groups([(3, 192, min(range(3), key=lambda i: a.pos[i])), (1, 0, 0), (1, 0, 0)], "cuda")
    got = a.run(K, window, keep, sinks, out=out, groups=groups, bound=a.width * PAGE)
    K.check_status("cuda")
    agree(got, torch.stack([w[0] for w in want]), torch.stack([w[1] for w in want]))
    assert any(float(want[t][0].abs().max()) == 0 for t in beyond) == (keep == 0)
    a.pos = pos
    agree(a.run(K, window, keep, sinks), *a.want(window, keep, sinks))


@pytest.mark.parametrize("window,keep", [(None, 0), (3000, 5)])
@pytest.mark.parametrize("nh,nkv,hd,groups", [
    (5, 1, 128, [(20032, [9, 1, 1500])]), (14, 2, 64, [(4096, [1 + 7 * i for i in range(40)])]), (8, 2, 128, [(4096, [70, 1]), (6016, [5, 64, 300])]),
    (14, 2, 64, [(31744, [1, 90])]),
])
def test_no_page_of_a_long_context_is_left_out(K, nh, nkv, hd, groups, window, keep):
    a = Answers(nh, nkv, hd, groups, seed=nh)
    got = a.run(K, window, keep).double()
    K.check_status("cuda")
    rms = lambda x: float(x.pow(2).mean().sqrt())                        # noqa: E731
    for t, pos in enumerate(a.pos):
        want, _, spread = alone(a, t, pos, window, keep)
        assert rms(got[t] - want) <= 2.0 ** -8 * (rms(want) + float(spread.mean().sqrt())), t


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("value", [float("inf"), -float("inf")])
@pytest.mark.parametrize("whole", [False, True])
def test_infinite_keys(K, hd, value, whole):
    """A score of +inf leaves a row no number, one of -inf no weight for its key; a key of infinities whose signs do not agree with the query's gives a score that is
    no number.  As in 64 bits.  (Read one by one, a row whose sum of weights is no number is zeros.)"""
    a = Answers(6, 2, hd, [(640, [3, 70, 130]), (192, [5, 9])], seed=hd)
    for page in (a.table[0, 4], a.table[1, 10], a.table[3, 1]):
        keep = a.k[page, 1].clone()
        a.k[page, 1, 1, slice(None) if whole else slice(7, 8)] = value
        want, mass = (torch.stack(x) for x in list(zip(*(alone(a, t, p) for t, p in enumerate(a.pos))))[:2])
        got, fine = a.run(K), torch.isfinite(want)
        assert torch.equal(torch.isfinite(got), fine)
        agree(torch.where(fine, got, 0.0), torch.where(fine, want, 0.0), torch.where(fine, mass, 0.0))
        a.k[page, 1] = keep
    agree(a.run(K), *a.want())
    K.check_status("cuda")


def test_shared_positions_beyond_the_table_move_no_other_group(K):
    a = Answers(14, 2, 64, [(192, [64, 128]), (128, [64])], seed=8)
    a.table = a.table[:, :5].contiguous()
    a.width = 5
    groups = K.shared_groups(a.members, "cuda")
    groups[:2, 2] = 64 * 100
    got, want, mass = a.run(K, groups=groups), *a.want()
    agree(got[2:], want[2:], mass[2:])
    K.check_status("cuda")


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("window,keep,sinks,slopes", [(None, 0, False, False), (500, 4, True, True)])
def test_pages_read_early_or_late_are_the_same(K, hd, window, keep, sinks, slopes):
    """``early_pages`` moves a wait, no result: rows that share pages, rows alone, more rows than the kernel takes at a time."""
    for groups in ([(1024, [5, 700, 64, 1, 9]), (0, [130])], [(64 * (1 + i % 3), [1 + i % 70] * 8) for i in range(60)]):
        a = Answers(8, 2, hd, groups, seed=hd)
        got = []
        for early in (True, False):
            got.append(K.attention_shared(a.rows, a.rows.shape[1], 8, 2, hd, a.k, a.v, a.table, a.width, ints(a.pos), torch.arange(a.T, dtype=torch.int32, device="cuda"),
                                          K.shared_groups(a.members, "cuda"), window, hd ** -0.5, max(a.pos) + 1, keep_first=keep, slopes=a.slopes if slopes else None,
                                          sinks=a.sinks if sinks else None, early_pages=early, together=True))
        agree(got[1], *a.want(window, keep, sinks, slopes))
        assert torch.equal(*got)
    K.check_status("cuda")


def test_a_direct_call_chooses_by_what_its_window_lets_rows_share(K):
    """Left to choose, a call reads rows one by one where a window leaves little to share, however long the context, and where it has one row."""
    a = Answers(14, 2, 64, [(640, [1, 30, 64, 65, 200]), (64, [5, 6])], seed=3)
    for window, keep in ((100, 0), (100, 70)):
        got = a.run(K, window, keep, bound=30000, together=None)
        assert torch.equal(got, a.run(K, window, keep, bound=30000, together=False))
        agree(got, *a.want(window, keep))
    assert torch.equal(a.run(K, bound=30000, together=None), a.run(K, bound=30000))
    b = Answers(14, 2, 64, [(4096, [9])], seed=4)
    assert torch.equal(b.run(K, bound=10 ** 6, together=None), b.run(K, bound=10 ** 6, together=False))
    K.check_status("cuda")


# ---------------------------------------------------------------------------- rules

@pytest.mark.parametrize("apart", [1, 100, 511, 512, 513, 1500, 4000])
def test_biases_of_a_token_are_added_up_before_they_meet_its_logit(K, apart):
    """Two that cancel leave the logit as it was, and the third alone counts, however far apart they stand in the list; so do masks and rows beside them."""
    V, n = 140000, apart + 700
    c = rules_case(3, V, seed=4, history=False, masks=False)
    ids = torch.randperm(V - 10, generator=gen(1), device="cuda")[:n].int()
    values = torch.randn(n, generator=gen(2), device="cuda")
    ids[::7] = (ids[::7].long() % 400 + 131072).int()                    # (tokens that lie 131,072 above others of the list)
    first = 20
    ids[[first, first + apart, first + apart + 600]] = V - 3
    values[first], values[first + apart], values[first + apart + 600] = 1e8, -1e8, 0.25
    c["bias_ids"], c["bias_values"], c["bias_range"] = ids, values, ints([[0, n], [0, first + apart + 300], [first + 1, n]])
    c["masks"], c["mask_rows"] = torch.full((1, (V + 31) // 32), -1, dtype=torch.int32, device="cuda"), ints([-1, 0, -1])
    got = adjust(K, c)
    x = c["logits"][:, V - 3]
    assert got[0, V - 3] == x[0] + 0.25 and got[1, V - 3] == x[1] and got[2, V - 3] == x[2] + (torch.tensor(-1e8, device="cuda") + 0.25)
    c.pop("masks"), c.pop("mask_rows")
    want, size = rules_want(c)
    others = torch.ones(V, dtype=torch.bool, device="cuda")
    others[V - 3] = False
    # of the others no token stands there more than 20 times
    times = torch.bincount(ids.long(), minlength=V)
    assert int(times[others].max()) <= 20
    assert bool(((got.double() - want).abs() <= 22 * 2.0 ** -24 * size)[:, others].all())
    for _ in range(3):
        assert torch.equal(adjust(K, c), got)
