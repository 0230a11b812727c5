"""The router's and the 4-bit operators of routed experts, as cases to be timed and compared.

Four operators of `odie_b200.experts`:

* `gate`: the experts of each row and their weights from the router's logits; training cases return d logits.
* `balance`: the balance loss, the mean square of the logits' log-sum-exp, and rows per expert; training cases return
  d logits.
* `quantize` and `dequantize`: rows as microscaled 4-bit floats and back.
* `linear4`: y = residual + act(q(x) W4^T + b), W4 kept in 4 bits, one matrix or one for each group of consecutive rows,
  x quantised on the way.

`own` false computes each operator from elementary torch operations in 32 bits (64 for quotients next to a rounding
border and for sums over many rows), rounded once; true calls the framework.
"""
import math

import torch

own = False

TYPES = {'f16': torch.float16, 'bf16': torch.bfloat16, 'f32': torch.float32}
BYTES = {'f16': 2, 'bf16': 2, 'f32': 4}


def listed():
    return [
        # one decoding step of a batch of 32 rows, two of 64 experts each: latency
        dict(name='gate-step', op='gate', rows=32, experts=64, choices=2, dtype='bf16', score='softmax', normalize=True,
             biased=False, padded=0.0, masked=0.0, train=False),
        # the routed-expert benchmark's step: 2^20 coordinates, 16 experts, top-1 by the softmax itself
        dict(name='gate-coords', op='gate', rows=1 << 20, experts=16, choices=1, dtype='f16', score='softmax',
             normalize=False, biased=False, padded=0.0, masked=0.0, train=True),
        # a long training batch with many experts, eight for each row, a load bias on the choice, padded rows
        dict(name='gate-batch', op='gate', rows=65536, experts=256, choices=8, dtype='bf16', score='sigmoid',
             normalize=True, biased=True, padded=0.03, masked=0.0, train=True),
        # the balance loss of the benchmark's step
        dict(name='balance-coords', op='balance', rows=1 << 20, experts=16, choices=1, dtype='f16', score='softmax',
             padded=0.0, masked=0.0, dropped=0.0, train=True),
        # nothing a multiple of anything, experts masked per row, padded rows, fp32
        dict(name='balance-odd', op='balance', rows=5003, experts=37, choices=3, dtype='f32', score='sigmoid',
             padded=0.05, masked=0.2, dropped=0.1, train=True),
        # a long batch of wide rows to 4 bits and back
        dict(name='quantize-batch', op='quantize', rows=16384, width=2048, dtype='bf16', block=16),
        # rows of no multiple of a block, powers of two as scales, fp32
        dict(name='quantize-odd', op='quantize', rows=5003, width=773, dtype='f32', block=32),
        # one row: the bytes of the weights
        dict(name='linear4-row', op='linear4', rows=1, inputs=4096, outputs=4096, groups=0, dtype='bf16', block=16,
             activation='gelu', bias=True, residual=True, tail=0),
        # a decoding batch
        dict(name='linear4-decode', op='linear4', rows=64, inputs=4096, outputs=4096, groups=0, dtype='bf16', block=32,
             activation='none', bias=False, residual=False, tail=0),
        # a long batch through one wide layer
        dict(name='linear4-batch', op='linear4', rows=16384, inputs=2048, outputs=8192, groups=0, dtype='bf16',
             block=16, activation='silu', bias=True, residual=True, tail=0),
        # rows sorted into 64 ragged experts, some rows behind the last one
        dict(name='linear4-experts', op='linear4', rows=32768, inputs=1024, outputs=2048, groups=64, dtype='bf16',
             block=16, activation='gelu', bias=True, residual=False, tail=100),
        # nothing a multiple of anything
        dict(name='linear4-odd', op='linear4', rows=1021, inputs=333, outputs=515, groups=0, dtype='f16', block=32,
             activation='silu', bias=True, residual=True, tail=0),
    ]


def _spread(rng, low, high):
    """A whole number of [low, high], even over its logarithm."""
    return min(high, max(low, round(math.exp(rng.uniform(math.log(low), math.log(high))))))


def draw(rng):
    op = rng.choice(['gate', 'balance', 'quantize', 'linear4', 'linear4'])
    if op in ('gate', 'balance'):
        experts = rng.choice([rng.randint(1, 300), 8, 16, 64, 128, 256])
        rows = _spread(rng, 1, min(1 << 20, (1 << 24) // experts))
        case = dict(op=op, rows=rows, experts=experts, choices=rng.randint(1, min(8, experts)),
                    dtype=rng.choice(['f16', 'bf16', 'f32']), score=rng.choice(['softmax', 'sigmoid']),
                    padded=rng.choice([0.0, 0.1]), masked=rng.choice([0.0, 0.3]))
        if op == 'gate':
            return dict(case, normalize=rng.random() < 0.5, biased=rng.random() < 0.5, train=rng.random() < 0.7)
        return dict(case, dropped=rng.choice([0.0, 0.1]), train=rng.random() < 0.7)
    if op == 'quantize':
        width = rng.choice([_spread(rng, 1, 8192), 32 * _spread(rng, 1, 256)])
        return dict(op=op, rows=_spread(rng, 1, min(1 << 20, (1 << 25) // width)), width=width,
                    dtype=rng.choice(['f16', 'bf16', 'f32']), block=rng.choice([16, 32]))
    inputs, outputs = (rng.choice([_spread(rng, 16, 4096), 64 * _spread(rng, 1, 64)]) for _ in range(2))
    groups = rng.choice([0, 0, rng.randint(1, 64)])
    rows = _spread(rng, 1, min(32768, (1 << 37) // (inputs * outputs)))
    return dict(op=op, rows=rows, inputs=inputs, outputs=outputs, groups=groups, dtype=rng.choice(['f16', 'bf16']),
                block=rng.choice([16, 32]), activation=rng.choice(['none', 'relu', 'silu', 'gelu']),
                bias=rng.random() < 0.5, residual=rng.random() < 0.5,
                tail=rng.randint(0, rows // 8) if groups else 0)


# ---------------------------------------------------------------- what a program has in hand
def prepare(case, seed):
    g = torch.Generator(device='cuda').manual_seed(seed)
    dtype = TYPES[case['dtype']]

    def normal(*shape, std=1.0, dtype=dtype):
        return (torch.randn(shape, generator=g, device='cuda') * std).to(dtype)

    def chance(p, *shape):
        return torch.rand(shape, generator=g, device='cuda') < p
    s = dict(case=case)
    if case['op'] in ('gate', 'balance'):
        n, e, k = case['rows'], case['experts'], case['choices']
        # a router's logits: some experts liked by all rows, and what each row likes
        s['logits'] = (normal(n, e, std=1.5, dtype=torch.float32) + normal(e, std=0.7, dtype=torch.float32)).to(dtype)
        s['mask'] = None
        if case['masked']:  # experts that a row may not take, and rows of padding
            s['mask'] = ~chance(case['masked'], n, e)
            if case['padded']:
                s['mask'] &= ~chance(case['padded'], n, 1)
        elif case['padded']:
            s['mask'] = ~chance(case['padded'], n, 1)
        if case['op'] == 'gate':
            s['bias'] = normal(e, std=0.2, dtype=torch.float32) if case['biased'] else None
            if case['train']:
                s['d_weights'] = normal(n, k, dtype=torch.float32)
        else:
            key = s['logits'].float()
            if s['mask'] is not None:
                key = torch.where(s['mask'], key, float('-inf'))
            top, expert = torch.topk(key, k, dim=1)
            gone = torch.isneginf(top)
            if case['dropped']:  # over the capacity of an expert
                gone |= chance(case['dropped'], n, k)
            s['expert'] = torch.where(gone, -1, expert).to(torch.int32)
            if case['train']:  # the loss's scale in fp16 training, times the two terms' coefficients
                s['d_loss'] = torch.tensor(2.0 ** 16 * 0.01, device='cuda')
                s['d_z'] = torch.tensor(2.0 ** 16 * 0.001, device='cuda')
        if case['train']:
            s['logits'].requires_grad_()
    elif case['op'] == 'quantize':
        # activations: columns of different sizes
        s['x'] = (normal(case['rows'], case['width'], dtype=torch.float32) *
                  torch.exp(normal(case['width'], dtype=torch.float32))).to(dtype)
    else:
        m, i, o, groups = case['rows'], case['inputs'], case['outputs'], case['groups']
        s['x'] = normal(m, i)
        weight = normal(*([groups] if groups else []), o, i, std=i ** -0.5)
        s['bias'] = normal(*([groups] if groups else []), o, std=0.1) if case['bias'] else None
        s['residual'] = normal(m, o) if case['residual'] else None
        s['offsets'] = s['edges'] = None
        if groups:
            cuts = torch.rand(groups - 1, generator=g, device='cuda').sort().values * (m - case['tail'])
            edges = [0] + [int(c) for c in cuts.cpu()] + [m - case['tail']]
            s['edges'] = edges
            s['offsets'] = torch.tensor(edges, dtype=torch.int32, device='cuda')
        if own:  # weights are laid out once
            from odie_b200.experts import quantize
            s['weight'] = quantize(weight, block=case['block'])
        else:
            s['weight'] = _quantized(weight, case['block'])
        s['raw weight'] = weight
    return s


# ---------------------------------------------------------------- one pass
def run(s):
    return {'gate': _gate, 'balance': _balance, 'quantize': _quantize, 'linear4': _linear4}[s['case']['op']](s)


def _masked(s, logits):
    return logits if s['mask'] is None else torch.where(s['mask'], logits, float('-inf'))


def _gate(s):
    case = s['case']
    if own:
        from odie_b200.experts import gate
        expert, weights = gate(s['logits'], case['choices'], bias=s['bias'], mask=s['mask'], score=case['score'],
                               normalize=case['normalize'], scale=1.5)
        answer = dict(expert=expert, weights=weights.detach())
        if case['train']:
            answer['d_logits'] = torch.autograd.grad(weights, s['logits'], s['d_weights'])[0]
        return answer
    logits = _masked(s, s['logits'].detach().float())
    key = logits if s['bias'] is None else logits + s['bias']
    key, expert = torch.sort(key, dim=1, descending=True, stable=True)
    key, expert = key[:, :case['choices']], expert[:, :case['choices']]
    live = ~torch.isneginf(key)
    chosen = torch.where(live, logits.gather(1, expert), float('-inf'))
    zero = torch.zeros((), device=logits.device)
    if case['score'] == 'softmax':
        pool = chosen if case['normalize'] else logits
        top = pool.max(1, keepdim=True).values
        top = torch.where(torch.isneginf(top), zero, top)
        total = torch.exp(pool - top).sum(1, keepdim=True)
        p = torch.where(live, torch.exp(chosen - top) / total, zero)
    else:
        p = torch.exp(-_softplus(-torch.where(live, chosen, zero)))  # the sigmoid
        p = torch.where(live, p, zero)
        if case['normalize']:
            total = p.sum(1, keepdim=True)
            p = torch.where(live, p / torch.where(total > 0, total, 1.0), zero)
    answer = dict(expert=torch.where(live, expert, -1).to(torch.int32), weights=1.5 * p)
    if case['train']:
        g = torch.where(live, 1.5 * s['d_weights'], zero)
        mean = (p * g).sum(1, keepdim=True)
        if case['score'] == 'softmax':
            d = p * (g - mean) if case['normalize'] else p * g
        else:
            complement = torch.exp(-_softplus(torch.where(live, chosen, zero)))
            d = p * complement * ((g - mean) if case['normalize'] else g)
        d_logits = torch.zeros_like(logits).scatter_add_(1, expert, torch.where(live, d, zero))
        if case['score'] == 'softmax' and not case['normalize']:
            d_logits -= torch.exp(logits - top) / torch.where(total > 0, total, 1.0) * mean
        answer['d_logits'] = d_logits.to(s['logits'].dtype)
    return answer


def _softplus(v):
    return v.clamp(min=0) + torch.log1p(torch.exp(-v.abs()))


def _balance(s):
    case = s['case']
    if own:
        from odie_b200.experts import balance
        loss, z, counts = balance(s['logits'], s['expert'], mask=s['mask'], score=case['score'])
        answer = dict(loss=loss.detach(), z=z.detach(), counts=counts)
        if case['train']:
            answer['d_logits'] = torch.autograd.grad([loss, z], s['logits'], [s['d_loss'], s['d_z']])[0]
        return answer
    e = case['experts']
    logits = _masked(s, s['logits'].detach().float())
    zero = torch.zeros((), device=logits.device)
    live = ~torch.isneginf(logits).all(1)
    rows = live.sum().clamp(min=1)
    expert = s['expert'].reshape(-1).long()
    counts = torch.zeros(e + 1, dtype=torch.int64, device=logits.device)
    counts.index_add_(0, torch.where((expert >= 0) & (expert < e), expert, e), torch.ones_like(expert))
    counts = counts[:e]
    top = torch.where(live, logits.max(1).values, zero)
    total = torch.where(live, torch.exp(logits - top[:, None]).sum(1), 1.0)
    soft = torch.exp(logits - top[:, None]) / total[:, None]
    lse = torch.where(live, top + torch.log(total), zero)
    p, slope = soft, torch.ones_like(soft)
    if case['score'] == 'sigmoid':
        sigmoid = torch.exp(-_softplus(-logits))
        p = sigmoid / torch.where(live, sigmoid.sum(1), 1.0)[:, None]
        slope = torch.exp(-_softplus(logits))
    f = counts.float() / counts.sum().clamp(min=1)
    loss = e * (f.double() * p.double().sum(0) / rows).sum()
    answer = dict(loss=loss.float(), z=(lse.double().square().sum() / rows).float(), counts=counts.to(torch.int32))
    if case['train']:
        d = (s['d_loss'] * e / rows) * p * slope * (f - (p * f).sum(1, keepdim=True))
        d = d + (s['d_z'] * 2 / rows) * lse[:, None] * soft
        answer['d_logits'] = d.to(s['logits'].dtype)
    return answer


def _quantized(x, block):
    """The values that x's microscaled form stands for: fp32, of x's shape.  A quotient decides on which side of a
    border a value rounds, so it is taken in 64 bits."""
    width = x.shape[-1]
    pad = -width % block
    v = torch.nn.functional.pad(x.detach().double(), (0, pad)).unflatten(-1, (-1, block))
    top = v.abs().amax(-1, keepdim=True)
    if block == 32:
        scale = _power(top, 6.0, -127)
    else:
        outer = _power(top.amax(-2, keepdim=True), 2688.0, -126)
        outer = torch.where(top.amax(-2, keepdim=True) > 0, outer, 1.0)
        t = top / (6 * outer)
        step = torch.ldexp(torch.ones_like(t), (torch.frexp(t).exponent - 4).clamp(min=-9))
        scale = torch.round(t / step) * step * outer
    q = torch.where(scale > 0, v / torch.where(scale > 0, scale, 1.0), 0.0)
    size = q.abs()
    step = torch.where(size < 2, 0.5, torch.where(size < 4, 1.0, 2.0))
    code = torch.sign(q) * (torch.round(size / step) * step).clamp(max=6)
    return (code * scale).flatten(-2)[..., :width].float()


def _power(v, most, least):
    """The least power of two p with v <= most p, and at least 2^least: exact, without a quotient."""
    mantissa, exponent = torch.frexp(v)
    most_mantissa, most_exponent = math.frexp(most)
    exponent = exponent - most_exponent + (mantissa > most_mantissa).to(exponent.dtype)
    exponent = torch.where(v > 0, exponent, least).clamp(min=least)
    return torch.ldexp(torch.ones_like(v), exponent)


def _quantize(s):
    case = s['case']
    if own:
        from odie_b200.experts import dequantize, quantize
        return dict(values=dequantize(quantize(s['x'], block=case['block']), dtype=s['x'].dtype))
    return dict(values=_quantized(s['x'], case['block']).to(s['x'].dtype))


def _activated(z, name):
    if name == 'relu':
        return z.clamp(min=0)
    if name == 'silu':
        return z / (1 + torch.exp(-z))
    if name == 'gelu':
        return 0.5 * z * torch.erfc(-z * math.sqrt(0.5))
    return z


def _linear4(s):
    case = s['case']
    if own:
        from odie_b200.experts import linear4
        return dict(y=linear4(s['x'], s['weight'], bias=s['bias'], residual=s['residual'],
                              activation=case['activation'], offsets=s['offsets']))
    x, weight = _quantized(s['x'], case['block']), s['weight']
    y = torch.zeros((case['rows'], case['outputs']), device=x.device)
    edges = s['edges'] or [0, case['rows']]
    for g, (low, high) in enumerate(zip(edges, edges[1:])):
        if low == high:
            continue
        z = x[low:high] @ (weight[g] if case['groups'] else weight).t()
        if s['bias'] is not None:
            z = z + (s['bias'][g] if case['groups'] else s['bias']).float()
        z = _activated(z, case['activation'])
        y[low:high] = z if s['residual'] is None else z + s['residual'][low:high].float()
    return dict(y=y.to(s['x'].dtype))


# ---------------------------------------------------------------- least work
def work(case):
    size = BYTES[case['dtype']]
    if case['op'] == 'gate':
        n, e, k = case['rows'], case['experts'], case['choices']
        mask = n * e if case['masked'] else n if case['padded'] else 0
        moved, flops = n * e * size + mask + n * k * 8, n * e * k
        if case['train']:  # d weights, the choices and weights, d logits; the logits too where all of them count
            dense = case['score'] == 'softmax' and not case['normalize']
            moved += n * k * 12 + n * e * size * (2 if dense else 1)
            flops += n * e
        return dict(bytes=moved, flops=flops)
    if case['op'] == 'balance':
        n, e, k = case['rows'], case['experts'], case['choices']
        mask = n * e if case['masked'] else n if case['padded'] else 0
        moved, flops = n * e * size + mask + n * k * 4 + 4 * e + 8, 5 * n * e
        if case['train']:
            moved += 2 * n * e * size + mask + 4 * e
            flops += 9 * n * e
        return dict(bytes=moved, flops=flops)
    if case['op'] == 'quantize':
        n, w = case['rows'], case['width']
        return dict(bytes=2 * n * w * size + n * w // 2 + n * w // case['block'], flops=3 * n * w)
    m, i, o, groups = case['rows'], case['inputs'], case['outputs'], max(1, case['groups'])
    moved = (m * i + m * o * (2 if case['residual'] else 1) + (groups * o if case['bias'] else 0)) * size
    moved += groups * o * (i // 2 + i // case['block'])
    return dict(bytes=moved, flops=2 * (m - case['tail']) * i * o)


# ---------------------------------------------------------------- the definitions in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    with torch.no_grad():
        return {'gate': _exact_gate, 'balance': _exact_balance, 'quantize': _exact_quantize,
                'linear4': _exact_linear4}[case['op']](s, case)


def _exact_gate(s, case):
    n, e, k = case['rows'], case['experts'], case['choices']
    logits = s['logits'].double()
    allowed = torch.ones((n, e), dtype=torch.bool, device='cuda') if s['mask'] is None else s['mask'].expand(n, e)
    key = logits if s['bias'] is None else (logits + s['bias'].double()).float().double()
    open_ = allowed & (key > float('-inf'))
    taken = torch.zeros_like(open_)
    experts = []
    place = torch.arange(e, device='cuda')
    for _ in range(k):  # the first of the highest, again and again
        left = open_ & ~taken
        best = torch.where(left, key, float('-inf')).amax(1, keepdim=True)
        first = torch.where(left & (key == best), place, e).amin(1)
        experts.append(first)
        taken |= place == first[:, None]
    expert = torch.stack(experts, 1)
    live = expert < e
    expert = torch.where(live, expert, -1)
    if case['score'] == 'softmax':
        pool = taken if case['normalize'] else allowed
        s_all = torch.exp(torch.where(pool, logits, float('-inf')) - torch.where(allowed, logits, float('-inf')).amax(1, keepdim=True))
        s_all = torch.nan_to_num(s_all, nan=0.0)
        total = s_all.sum(1, keepdim=True)
        p = s_all / torch.where(total > 0, total, 1.0)
    else:
        p = torch.sigmoid(logits) * taken
        if case['normalize']:
            p = p / p.sum(1, keepdim=True).clamp(min=1e-300)
    index = expert.clamp(min=0).long()
    answer = dict(expert=expert.to(torch.int32), weights=torch.where(live, 1.5 * p.gather(1, index), 0.0))
    if case['train']:
        g = torch.zeros((n, e), dtype=torch.float64, device='cuda')
        g.scatter_add_(1, index, torch.where(live, s['d_weights'].double() * 1.5, 0.0))
        inner = (p * g * taken).sum(1, keepdim=True)
        d = p * (g - inner) if case['score'] == 'softmax' or case['normalize'] else p * g
        answer['d_logits'] = d if case['score'] == 'softmax' else d * torch.sigmoid(-logits)
    return answer


def _exact_balance(s, case):
    n, e = case['rows'], case['experts']
    logits = s['logits'].double()
    if s['mask'] is not None:
        logits = logits.masked_fill(~s['mask'].expand(n, e), float('-inf'))
    live = (logits > float('-inf')).any(1)
    rows = max(1, int(live.sum()))
    counts = torch.stack([(s['expert'] == j).sum() for j in range(e)])
    f = counts.double() / max(1, int(counts.sum()))
    logits = logits[live]
    lse = torch.logsumexp(logits, 1)
    soft = torch.softmax(logits, 1)
    p = soft
    if case['score'] == 'sigmoid':
        p = torch.sigmoid(logits)
        p = p / p.sum(1, keepdim=True)
    answer = dict(loss=e * (f * p.sum(0)).sum() / rows, z=(lse * lse).sum() / rows, counts=counts.to(torch.int32))
    if case['train']:
        d = p * (f - (p @ f)[:, None]) * (s['d_loss'].double() * e / rows)
        if case['score'] == 'sigmoid':
            d = d * torch.sigmoid(-logits)
        d = d + soft * lse[:, None] * (s['d_z'].double() * 2 / rows)
        whole = torch.zeros((n, e), dtype=torch.float64, device='cuda')
        whole[live] = d
        answer['d_logits'] = whole
    return answer


def _exact_values(x, block):
    """The microscaled values of x [rows, width] from the tables of both formats, by the borders between neighbours."""
    device = x.device
    codes = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6], dtype=torch.float64, device=device)
    e4m3 = torch.tensor([m * 2.0 ** -9 for m in range(8)] +
                        [(8 + m) * 2.0 ** (p - 10) for p in range(1, 16) for m in range(8) if p < 15 or m < 7],
                        dtype=torch.float64, device=device)

    def nearest(table, v):  # ties to the even place
        border = (table[1:] + table[:-1]) / 2
        low, high = torch.searchsorted(border, v, right=False), torch.searchsorted(border, v, right=True)
        return table[torch.where((low != high) & (low % 2 == 1), high, low)]
    powers = torch.tensor([2.0 ** p for p in range(-149, 129)], dtype=torch.float64, device=device)
    out = torch.empty(x.shape, dtype=torch.float64, device=device)
    for begin in range(0, x.shape[0], 4096):
        rows = x[begin:begin + 4096].double()
        outer = torch.ones((rows.shape[0], 1), dtype=torch.float64, device=device)
        if block == 16:
            top = rows.abs().amax(1, keepdim=True)
            outer = torch.where(top > 0, powers[torch.searchsorted(2688 * powers[23:], top).clamp(max=240) + 23], 1.0)
        for first in range(0, x.shape[1], block):
            part = rows[:, first:first + block]
            top = part.abs().amax(1, keepdim=True)
            if block == 16:
                scale = nearest(e4m3, top / (6 * outer)) * outer
            else:
                scale = powers[torch.searchsorted(6 * powers[22:], top) + 22]
            size = nearest(codes, (part.abs() / scale.clamp(min=1e-300)))
            out[begin:begin + 4096, first:first + block] = torch.sign(part) * size * scale
    return out


def _exact_quantize(s, case):
    return dict(values=_exact_values(s['x'], case['block']))


def _exact_linear4(s, case):
    x = _exact_values(s['x'], case['block'])
    y = torch.zeros((case['rows'], case['outputs']), dtype=torch.float64, device='cuda')
    edges = s['edges'] or [0, case['rows']]
    for g, (low, high) in enumerate(zip(edges, edges[1:])):
        weight = _exact_values(s['raw weight'][g] if case['groups'] else s['raw weight'], case['block'])
        z = torch.nn.functional.linear(x[low:high], weight)
        if s['bias'] is not None:
            z += (s['bias'][g] if case['groups'] else s['bias']).double()
        z = {'none': lambda: z, 'relu': lambda: torch.relu(z), 'silu': lambda: z * torch.sigmoid(z),
             'gelu': lambda: z * torch.special.ndtr(z)}[case['activation']]()
        if s['residual'] is not None:
            z = z + s['residual'][low:high].double()
        y[low:high] = z
    return dict(y=y)
