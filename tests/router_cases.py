"""Plain 64-bit forms of the router's operators and of microscaled rows, and bounds on what the kernels may be off by.

Choices, counts, codes and scales have to be equal.  A softmax's exponentials are off by their arguments' rounding,
2^-24 of at most `depth` (the distance between a row's logits), and by the function's own 2^-22; a sum of n positive terms
by n 2^-24 of it.  The instruction for the exponential gives 0 below the least normal number, 2^-126 (TINY): what it is
multiplied by is off by as much.
"""
import torch

from rows_cases import SUM, rounding  # noqa: F401


TINY = 2.0 ** -126


def masked(logits, mask):
    x = logits.double()
    return x if mask is None else torch.where(mask.expand(x.shape), x, float('-inf'))


def share_error(x, dim=1):
    """The relative error of softmax's (and sigmoid's) values of rows x, [rows, 1]."""
    finite = torch.where(torch.isfinite(x), x, 0.0)
    depth = finite.abs().amax(dim, keepdim=True) * 2
    return depth * 2.0 ** -23 + 2.0 ** -20 + (x.shape[dim] + 8) * 2.0 ** -24


def plain_gate(logits, choices, bias, mask, score, normalize, scale, d_weights):
    """(expert, (weights, bound), (d_logits, bound)); NaN logits are not covered."""
    rows, experts = logits.shape
    x = masked(logits, mask)
    key = masked(logits.float() + (0 if bias is None else bias.float()), mask)
    ordered, order = torch.sort(key, dim=1, descending=True, stable=True)
    live = ~torch.isneginf(ordered[:, :choices])
    expert = torch.where(live, order[:, :choices], -1)
    taken = torch.zeros((rows, experts), dtype=torch.bool, device=x.device)
    taken.scatter_(1, order[:, :choices], live)
    g = torch.zeros((rows, experts), dtype=torch.float64, device=x.device)
    g.scatter_(1, order[:, :choices], torch.where(live, d_weights.double(), 0.0))
    if score == 'softmax':
        pool = torch.where(taken, x, float('-inf')) if normalize else x
        p = torch.nan_to_num(torch.softmax(pool, 1))  # (a row of nothing)
        own = torch.where(taken, p, 0.0)
    else:
        logs = torch.where(taken, torch.nn.functional.logsigmoid(x), float('-inf'))
        p = own = torch.nan_to_num(torch.softmax(logs, 1)) if normalize else torch.where(taken, torch.sigmoid(x), 0.0)
    error = share_error(x)
    inner, size = (own * g).sum(1, keepdim=True), (own * g).abs().sum(1, keepdim=True)
    if score == 'softmax':
        d, most = p * (g - inner), p * (g.abs() + size)
    elif normalize:
        d, most = p * torch.sigmoid(-x) * (g - inner), p * torch.sigmoid(-x) * (g.abs() + size)
    else:
        d, most = p * torch.sigmoid(-x) * g, p * torch.sigmoid(-x) * g.abs()
    d, most = scale * torch.where(torch.isneginf(x), 0.0, d), abs(scale) * torch.where(torch.isneginf(x), 0.0, most)
    weights = scale * torch.where(live, own.gather(1, order[:, :choices]), 0.0)
    d_bound = most * (4 * error + (choices + 8) * SUM) + abs(scale) * (g.abs() + size) * TINY
    return (expert, (weights, weights.abs() * error + abs(scale) * TINY),
            (d, d_bound + rounding(d.abs() + d_bound, logits.dtype) + TINY))


def plain_balance(logits, expert, mask, score, total, d_loss, d_z):
    """({loss, z}: (value, bound), counts, (d_logits, bound))."""
    rows, experts = logits.shape
    x = masked(logits, mask)
    live = ~torch.isneginf(x).all(1)
    n = int(live.sum())
    keys = expert.reshape(-1).long()
    counts = torch.bincount(keys[(keys >= 0) & (keys < experts)], minlength=experts)
    load = counts.double() if total is None else total.double()
    f = load / load.sum() if load.sum() > 0 else load
    x = torch.where(live[:, None], x, 0.0)
    lse = torch.logsumexp(x, 1)
    soft = torch.softmax(x, 1)
    logs = torch.nn.functional.logsigmoid(x)
    p = soft if score == 'softmax' else torch.softmax(logs, 1)
    slope = torch.ones_like(p) if score == 'softmax' else torch.sigmoid(-x)
    soft, p, lse = (torch.where(live[:, None], t, 0.0) for t in (soft, p, lse[:, None]))
    lse = lse[:, 0]
    error = share_error(x)
    # rows that one thread adds up, then warps, blocks (in 64 bits)
    adds = rows // (4 * 148) + 32
    per = 1 / n if n else 0.0
    loss, z = experts * (f * p.sum(0)).sum() * per, (lse * lse).sum() * per
    off = lse.abs() * 2.0 ** -22 + error[:, 0]  # of lse
    answer = dict(loss=(loss, loss * (error.max() if rows else 0) * 2 + loss * adds * 2.0 ** -24 + loss * 2.0 ** -22),
                  z=(z, (2 * lse.abs() * off + off * off).sum() * per + z * adds * 2.0 ** -23))
    inner = (p * f).sum(1, keepdim=True)
    a, b = d_loss * experts * per * p * slope, d_z * 2 * per * lse[:, None] * soft
    d = a * (f - inner) + b
    bound = a.abs() * (f + inner) * (6 * error + (experts + 16) * SUM) + b.abs() * (6 * error + 16 * SUM) + abs(d_z) * 2 * per * soft * off[:, None]
    bound = bound + (abs(d_loss) * experts * (f + inner) + abs(d_z) * 2 * lse.abs()[:, None] + 1) * TINY
    return answer, counts, (d, bound + rounding(d.abs() + bound, logits.dtype))


CODES = [0, 0.5, 1, 1.5, 2, 3, 4, 6]
E4M3 = [m * 2.0 ** -9 for m in range(8)] + [(8 + m) * 2.0 ** (p - 10) for p in range(1, 16) for m in range(8) if (p, m) != (15, 7)]


def nearest(table, v):
    """The entry of an ascending table next to v >= 0, ties to the even place, saturating; and its place."""
    table = torch.tensor(table, dtype=torch.float64, device=v.device)
    border = (table[1:] + table[:-1]) / 2
    low, high = torch.searchsorted(border, v), torch.searchsorted(border, v, right=True)
    place = torch.where((low != high) & (low % 2 == 1), high, low)
    return table[place], place


def least_power(v, most, least):
    """The least whole e >= least with v <= most 2^e, exact."""
    powers = torch.tensor([most * 2.0 ** e for e in range(least, 129)], dtype=torch.float64, device=v.device)
    return torch.searchsorted(powers, v) + least


def plain_micro(x, block):
    """(values in 64 bits, codes, scale bytes [rows, blocks], row scales) of x [rows, width]."""
    rows, width = x.shape
    blocks = -(-width // block)
    v = torch.nn.functional.pad(x.double(), (0, blocks * block - width)).view(rows, blocks, block)
    bad = ~torch.isfinite(v).all(2).all(1)
    v = torch.where(bad[:, None, None], 0.0, v)
    top = v.abs().amax(2)
    if block == 16:
        k = torch.where(top.amax(1) > 0, least_power(top.amax(1), 2688.0, -126), 0)
        outer = torch.ldexp(torch.ones_like(top[:, 0]), k)
        scale, byte = nearest(E4M3, top / (6 * outer[:, None]))
    else:
        outer = torch.ones_like(top[:, 0])
        e = least_power(top, 6.0, -127)
        scale, byte = torch.ldexp(torch.ones_like(top), e), torch.where(bad[:, None], 0, e + 127)
    whole = (scale * outer[:, None])[:, :, None]
    size, place = nearest(CODES, torch.where(whole > 0, v.abs() / torch.where(whole > 0, whole, 1.0), 0.0))
    values = (torch.sign(v) * size * whole).view(rows, -1)[:, :width]
    codes = (place + 8 * torch.signbit(v).long()).view(rows, -1)[:, :width]
    outer = torch.where(bad, float('nan'), outer)
    return torch.where(bad[:, None], float('nan'), values), codes, byte, outer


def unpacked(micro):
    """(codes [rows, padded width], scale bytes [rows, padded blocks]) of one group's Micro, from its layout."""
    low = micro.codes.reshape(-1, micro.codes.shape[-1]).long()
    codes = torch.stack([low & 15, low >> 4], 2).flatten(1)
    tiles, columns = micro.scales.shape[1:3]
    # tile [l][q][b]: row 32 q + l, block b
    scales = micro.scales[0].view(tiles, columns, 32, 4, 4).permute(0, 3, 2, 1, 4).reshape(tiles * 128, columns * 4)
    return codes, scales.long()
