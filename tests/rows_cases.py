"""Plain 64-bit forms of the routed-expert row operators, and bounds on what the kernels may be off by.

Rounding to a type is off by at most half a step: eps / 2 relative, or half the smallest subnormal.  An fp32 sum of
n terms is off by at most n 2^-23 times the sum of their magnitudes: every addition, rounded or cut, loses at most
2^-23 of a partial sum that is itself at most that sum.
"""
import math

import torch

TYPES = [torch.float16, torch.bfloat16, torch.float32]
SUM = 2.0 ** -23


def rounding(value, dtype):
    """Half a step of dtype at |value|."""
    info = torch.finfo(dtype)
    return value.abs() * (info.eps / 2) + info.smallest_normal * info.eps / 2


def within(got, want, bound, what):
    """|got - want| <= bound everywhere (want and bound in 64 bits); the same NaNs and infinities."""
    got = got.double()
    assert got.shape == want.shape, (what, got.shape, want.shape)
    finite = torch.isfinite(want)
    assert torch.equal(got.isnan(), want.isnan()), f'{what}: NaN in other places'
    assert torch.equal(got[got.isinf()], want[want.isinf()]), f'{what}: infinities differ'
    over = ((got - want).abs() - bound)[finite]
    if over.numel():
        assert over.max().item() <= 0, f'{what}: over its bound by {over.max().item():.3e} ({(over > 0).sum().item()} elements)'


def plain_order(expert, bins):
    """(order, slot, offsets) from the definition, on the host."""
    keys = expert.reshape(-1).tolist()
    kept = [(k, i) for i, k in enumerate(keys) if 0 <= k < bins]
    kept.sort()
    gone = [i for i, k in enumerate(keys) if not 0 <= k < bins]
    slot = [0] * len(keys)
    for place, (_, i) in enumerate(kept):
        slot[i] = place
    for place, i in enumerate(gone, len(kept)):
        slot[i] = ~place
    counts = [0] * (bins + 1)
    for k, _ in kept:
        counts[k + 1] += 1
    offsets = torch.tensor(counts).cumsum(0)
    return torch.tensor([i for _, i in kept] + [~i for i in gone]), torch.tensor(slot).reshape(expert.shape), offsets


def activated(z, name):
    """act(z), act'(z) in 64 bits."""
    if name == 'relu':
        return z.clamp(min=0), (z > 0).double()
    if name == 'silu':
        p = torch.sigmoid(z)
        return z * p, p * (1 + z * (1 - p))
    if name == 'gelu':
        p = torch.special.ndtr(z)
        return z * p, p + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)
    return z, torch.ones_like(z)


def plain_linear(x, weight, bias, residual, edges, activation, d_y):
    """{name: (value, bound)} of y and the gradients in 64 bits; edges: the groups' row ranges."""
    dtype = x.dtype
    x, d_y = x.double(), d_y.double()
    w = weight.double().view(-1, *weight.shape[-2:])
    rows, (outputs, inputs) = x.shape[0], w.shape[1:]
    b = None if bias is None else bias.double().view(-1, outputs)
    zeros = {'y': (rows, outputs), 'd_x': (rows, inputs), 'd_weight': tuple(w.shape), 'd_bias': (w.shape[0], outputs),
             'd_residual': (rows, outputs)}
    value = {k: torch.zeros(s, dtype=torch.float64, device=x.device) for k, s in zeros.items()}
    bound = {k: torch.zeros(s, dtype=torch.float64, device=x.device) for k, s in zeros.items()}
    # ReLU cases use whole numbers, whose sums are exact; the others have smooth slopes: |act'| < 1.13, |act''| < 0.8
    steep = 0.0 if activation in ('none', 'relu') else 0.8
    for g, (lo, hi) in enumerate(edges):
        z = x[lo:hi] @ w[g].t()
        off = (inputs + 1) * SUM * (x[lo:hi].abs() @ w[g].abs().t())
        if b is not None:
            z = z + b[g]
            off = off + 2.0 ** -24 * z.abs()
        a, slope = activated(z, activation)
        y = a if residual is None else a + residual[lo:hi].double()
        # the exponential's and error function's own errors: a few 2^-23 of act, its argument's rounding included
        own = 0.0 if steep == 0 else 2.0 ** -20 * (z.abs() + 1)
        value['y'][lo:hi] = y
        bound['y'][lo:hi] = 1.13 * off + own + 2.0 ** -24 * (a.abs() + y.abs()) + rounding(y, dtype)
        g_y = d_y[lo:hi]
        dz = g_y * slope
        code = 0.0 if activation in ('none', 'relu') else 2.0 ** -16
        slope_off = steep * off + own + code
        exact_off = g_y.abs() * slope_off + 2.0 ** -23 * dz.abs()  # before dz is rounded for the products
        dz_off = exact_off + (0 if activation == 'none' else rounding(dz.abs() + exact_off, dtype))
        value['d_x'][lo:hi] = dz @ w[g]
        bound['d_x'][lo:hi] = dz_off @ w[g].abs() + (outputs + 1) * SUM * (dz.abs() + dz_off) @ w[g].abs()
        value['d_weight'][g] = dz.t() @ x[lo:hi]
        bound['d_weight'][g] = dz_off.t() @ x[lo:hi].abs() + (hi - lo + 1) * SUM * (dz.abs() + dz_off).t() @ x[lo:hi].abs()
        value['d_bias'][g] = dz.sum(0)
        bound['d_bias'][g] = exact_off.sum(0) + (hi - lo + 1) * SUM * (dz.abs() + exact_off).sum(0)
        value['d_residual'][lo:hi] = g_y
    for k in ('d_x', 'd_weight', 'd_bias'):
        bound[k] = bound[k] + rounding(value[k].abs() + bound[k], dtype)
    value['d_weight'], bound['d_weight'] = (t['d_weight'].view(weight.shape) for t in (value, bound))
    if weight.dim() == 2:
        value['d_bias'], bound['d_bias'] = value['d_bias'][0], bound['d_bias'][0]
    return {k: (value[k], bound[k]) for k in value}
