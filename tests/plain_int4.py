"""A cache of 4-bit keys and values, bit by bit: what a block holds, in 64 bits, independent of the library."""
import torch

PAGE = 64


def quantise(x):
    """(levels 0..15, steps, middles) of rows x [..., D] (bfloat16 values); steps and middles float64 [..., D / 32]."""
    y = x.double().unflatten(-1, (-1, 32))
    top, low = y.amax(-1), y.amin(-1)
    mid, step = ((top + low) / 2).to(torch.bfloat16).double(), ((top - low) / 15).to(torch.bfloat16).double()
    none = ~(torch.isfinite(mid) & torch.isfinite(step))
    mid, step = torch.where(none, torch.nan, mid), torch.where(none, torch.nan, step)
    level = torch.floor((y - mid[..., None]) / step[..., None]) + 8
    level = torch.where(step[..., None] == 0, 8.0, level).nan_to_num(0.0).clamp(0, 15)
    return level.long().flatten(-2), step, mid


def stands_for(x):
    """What a cache keeps of rows x [..., D]: float64."""
    level, step, mid = quantise(x)
    return (mid[..., None] + step[..., None] * (level.unflatten(-1, (-1, 32)).double() - 7.5)).flatten(-2)


def places(D, values):
    """For every (position of a page, channel): the word, the bits of sign and magnitude in it, the places of step and middle (bfloat16 numbers), [64, D] each."""
    p, c = torch.arange(64)[:, None], torch.arange(D)[None, :]
    b, nb, zero = c // 32, D // 32, torch.zeros(64, D, dtype=torch.long)
    if values:
        f, t, e = p % 16 // 8, p % 8 // 2, p % 2
        m = 2 * b + c % 4 // 2
        i = 2 * f + c % 2
        word = 8 * D + ((p // 16 * (D // 64) + m // 4) * 32 + c % 32 // 4 * 4 + t) * 4 + m % 4
        step = 36 * D + (p // 16 * 2 * nb + b) * 16 + 4 * t + 2 * f + e
        mid = step + 16 * nb
    else:
        i, e = c % 8 // 2, c % 2
        word = p * (D // 8) + c % 32 // 8 * nb + b
        step = 32 * D + p * 2 * nb + b
        mid = step + nb
    return [x + zero for x in (word, (15 + 16 * e + 4 * i) % 32, (4 + 16 * e + 4 * i) % 32, step, mid)]


def pack(keys, values):
    """Blocks uint8 [n, 80 D] that hold keys and values [n, 64, D] (bfloat16)."""
    n, _, D = keys.shape
    words = torch.zeros(n, 20 * D, dtype=torch.int64, device=keys.device)
    numbers = torch.zeros(n, 40 * D, dtype=torch.bfloat16, device=keys.device)
    for x, which in ((keys, False), (values, True)):
        word, sign, magnitude, at_step, at_mid = (v.to(keys.device) for v in places(D, which))
        level, step, mid = quantise(x)
        k = torch.where(level >= 8, level - 8, 7 - level)
        bits = (level < 8).long() << sign
        for j in range(3):
            bits = bits + (((k >> j) & 1) << ((magnitude + j) % 32))
        words.scatter_add_(1, word.reshape(1, -1).expand(n, -1), bits.reshape(n, -1))
        for at, v in ((at_step, step), (at_mid, mid)):
            numbers.scatter_(1, at.reshape(1, -1).expand(n, -1), v.to(torch.bfloat16).repeat_interleave(32, dim=-1).reshape(n, -1))
    out = torch.where(words >= 2 ** 31, words - 2 ** 32, words).int().view(torch.uint8).clone()
    out[:, 64 * D:] = numbers.view(torch.uint8)[:, 64 * D:]
    return out


def unpack(blocks):
    """float64 (keys, values, steps times level of the values) [n, 64, D] of blocks [n, 80 D]."""
    D = blocks.shape[1] // 80
    words, numbers, out = blocks.contiguous().view(torch.int32).long(), blocks.contiguous().view(torch.bfloat16).double(), []
    for which in (False, True):
        word, sign, magnitude, at_step, at_mid = (v.to(blocks.device) for v in places(D, which))
        w = words[:, word]
        k = sum(((w >> ((magnitude + j) % 32)) & 1) << j for j in range(3)).double() + 0.5
        part = numbers[:, at_step] * torch.where((w >> sign) & 1 == 1, -k, k)
        out += [numbers[:, at_mid] + part, part, numbers[:, at_mid]]
    return out[0], out[3], out[4], out[2]


def attend(q, kept, seen, scale, halves=False):
    """q [H, D] over blocks of one row: ``kept`` [P, G, 80 D], ``seen`` bool [G, 64 P].  (result [H, D], its bound per number in halves of a bfloat16 step,
    see the tests) in 64 bits.  ``halves``: for a kernel that takes keys, values and weights as float16."""
    H, D = q.shape
    P, G, _ = kept.shape
    keys, values, part, mids = (x.view(P, G, 64, D).transpose(0, 1).reshape(G, P * 64, D) for x in unpack(kept.flatten(0, 1)))
    out, bound = [], []
    q = q.double()
    for h in range(H):
        g = h * G // H
        k, v, s = keys[g][seen[g]], values[g][seen[g]], part[g][seen[g]]
        if k.shape[0] == 0:
            out.append(torch.zeros(D, dtype=torch.float64, device=q.device)); bound.append(out[-1])
            continue
        x = k @ q[h] * scale
        w = torch.softmax(x, 0)
        o = w @ v
        # a score's error: the sums of a group's queries in two bfloat16 parts times its middle (2^-16), and float32 sums
        m, sums = mids[g][seen[g]], q[h].view(-1, 32).sum(1).abs().repeat_interleave(32)
        err = scale * (2.0 ** -16 * (m.abs() @ sums) / 32 + (D + 16) * 2.0 ** -23 * ((k.abs() + m.abs()) @ q[h].abs())) + 2.0 ** -20
        if halves:
            # half a step of float16, 2^-11, of every key; below 2^-14 of the page's largest times 2^14, a step of 2^-24 of that (page and query row are brought to 2^14 at most)
            err = scale * (2.0 ** -11 + (D + 16) * 2.0 ** -23) * (k.abs() @ q[h].abs()) + scale * 2.0 ** -37 * D * k.abs().max() * q[h].abs().max() + 2.0 ** -20
        out.append(o)
        # what scores are off moves weights by as much; the result is rounded
        moved = 2 * (w * err) @ (v - o).abs() + 2 * (w @ err) * (w @ (v - o).abs()) + 2.0 ** -8 * o.abs()
        if halves:
            # weights and values rounded to float16, 2^-11 each.  Of a page with values up to 2^f weights are held times 2^f, up to 2^14 for the largest of all pages (2^6 where the
            # reference point lags behind it): below 2^-14 their steps are 2^-24, 2^-30 of the largest; values below 2^-28 of 2^f are off by 2^-39 of it.
            most = values[g].nan_to_num(0.0).abs().view(P, -1).amax(1).repeat_interleave(64)[seen[g]] * 2
            moved = moved + 2 * 2.0 ** -11 * (w @ v.abs()) + k.shape[0] * 2.0 ** -30 * (w * most).max() + 2.0 ** -38 * (w @ most)
        else:
            # weights rounded (on v), and once more behind a step (on the part that the codes carry)
            moved = moved + 2.0 ** -8 * (w @ (v.abs() + s.abs()))
        bound.append(moved)
    return torch.stack(out), torch.stack(bound)
