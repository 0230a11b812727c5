"""The routed-expert row operators, as cases to be timed and compared.

Three operators of `odie_b200.experts`:

* `dispatch`: rows sorted by expert and back.  `sort_rows` orders the (row, choice) pairs by expert, `dispatch`
  copies every row to its places, `combine` brings the experts' results back as weighted sums.  Training cases
  return the gradients of rows, results and weights too.
* `linear`: y = residual + act(x W^T + b), one weight matrix or one for each group of consecutive rows.
* `embed`: rows of a learned table by integer id, times a scale; training cases return the table's gradient.

`own` false computes each operator from elementary torch operations in 32 bits (64 for the long sums of the
table's gradient), rounded once; true calls the framework.
"""
import math

import torch

own = False

TYPES = {'f16': torch.float16, 'bf16': torch.bfloat16, 'f32': torch.float32}
BYTES = {'f16': 2, 'bf16': 2, 'f32': 4}


def listed():
    return [
        # one decoding step of a batch of 32 rows, two of 64 experts each: latency of four launches
        dict(name='dispatch-step', op='dispatch', rows=32, choices=2, experts=64, width=1024, dtype='bf16',
             dropped=0.0, train=False),
        # the routed-expert benchmark's step: 2^20 coordinates, 16 experts, 32 features, top-1
        dict(name='dispatch-coords', op='dispatch', rows=1 << 20, choices=1, experts=16, width=32, dtype='f16',
             dropped=0.0, train=True),
        # a long training batch, four of 64 experts for each row
        dict(name='dispatch-batch', op='dispatch', rows=16384, choices=4, experts=64, width=2048, dtype='bf16',
             dropped=0.0, train=True),
        # nothing a multiple of anything, a tenth of the choices dropped (masked or over capacity), fp32
        dict(name='dispatch-odd', op='dispatch', rows=5003, choices=3, experts=37, width=773, dtype='f32',
             dropped=0.1, train=True),
        # a single row through a square layer: the weights' bytes are all that counts
        dict(name='linear-one', op='linear', rows=1, inputs=4096, outputs=4096, groups=0, dtype='bf16',
             activation='gelu', bias=True, residual=True, tail=0, train=False),
        # the decoder's first layer on a benchmark batch
        dict(name='linear-coords', op='linear', rows=1 << 20, inputs=32, outputs=64, groups=0, dtype='f16',
             activation='relu', bias=True, residual=False, tail=0, train=True),
        # a wide layer on a long batch, bound by the tensor cores
        dict(name='linear-wide', op='linear', rows=16384, inputs=2048, outputs=8192, groups=0, dtype='bf16',
             activation='silu', bias=True, residual=True, tail=0, train=True),
        # 64 experts' own layers on sorted rows, groups of very different sizes, 100 rows behind the last group
        dict(name='linear-experts', op='linear', rows=32768, inputs=1024, outputs=2048, groups=64, dtype='bf16',
             activation='gelu', bias=True, residual=False, tail=100, train=True),
        # odd in every size: rows that no 16-byte load can start on
        dict(name='linear-odd', op='linear', rows=1021, inputs=333, outputs=515, groups=0, dtype='f16',
             activation='silu', bias=True, residual=True, tail=0, train=True),
        # 48 ids of one serving step
        dict(name='embed-step', op='embed', ids=48, table=32768, width=1024, dtype='bf16', scale=32.0, skew=1.0,
             masked=0.0, train=False),
        # a training batch with a few very frequent ids
        dict(name='embed-batch', op='embed', ids=65536, table=65536, width=1024, dtype='bf16', scale=32.0, skew=3.0,
             masked=0.01, train=True),
        # a learned code for each 256 x 256 tile of the gigapixel image, looked up by 2^20 coordinates
        dict(name='embed-tiles', op='embed', ids=1 << 20, table=16384, width=32, dtype='f32', scale=1.0, skew=1.0,
             masked=0.0, train=True),
    ]


def _spread(rng, low, high):
    """A whole number spread evenly over the logarithm of [low, high]."""
    return min(high, max(low, round(math.exp(rng.uniform(math.log(low), math.log(high))))))


def draw(rng):
    op = rng.choice(['dispatch', 'linear', 'embed'])
    train = rng.random() < 0.6
    if op == 'dispatch':
        experts = _spread(rng, 1, 256)
        choices = min(experts, rng.choice([1, 1, 2, 3, 4, 8]))
        width = _spread(rng, 1, 4096)
        rows = _spread(rng, 1, min(1 << 20, (1 << 26) // (choices * width), (1 << 26) // experts))
        return dict(op=op, rows=rows, choices=choices, experts=experts, width=width,
                    dtype=rng.choice(['f16', 'bf16', 'f32']), dropped=rng.choice([0.0, 0.0, 0.1]), train=train)
    if op == 'linear':
        groups = rng.choice([0, 0, _spread(rng, 1, 64)])
        inputs, outputs = _spread(rng, 1, 4096), _spread(rng, 1, 8192)
        if rng.random() < 0.5:  # half the draws with rows that 16-byte loads can start on
            inputs, outputs = -(-inputs // 8) * 8, -(-outputs // 8) * 8
        if groups:  # the groups' weights together stay within the wide layer's few times over
            outputs = max(1, min(outputs, (1 << 27) // (groups * inputs)))
        rows = _spread(rng, 1, max(1, min(1 << 20, (1 << 37) // (inputs * outputs), (1 << 27) // max(inputs, outputs))))
        return dict(op=op, rows=rows, inputs=inputs, outputs=outputs, groups=groups, dtype=rng.choice(['f16', 'bf16']),
                    activation=rng.choice(['none', 'relu', 'silu', 'gelu']), bias=rng.random() < 0.7,
                    residual=rng.random() < 0.5, tail=rng.choice([0, rows // 7]) if groups else 0, train=train)
    width = _spread(rng, 1, 2048)
    table = _spread(rng, 1, min(1 << 17, (1 << 26) // width))
    ids = _spread(rng, 1, min(1 << 20, (1 << 26) // width))
    return dict(op=op, ids=ids, table=table, width=width, dtype=rng.choice(['f16', 'bf16', 'f32']),
                scale=rng.choice([1.0, 32.0, 0.5]), skew=rng.choice([1.0, 2.0, 4.0]), masked=rng.choice([0.0, 0.05]),
                train=train)


# ---------------------------------------------------------------- inputs
def _group_sizes(case, seed):
    """Rows of each group: exponential shares (some groups several times the mean, some near empty) of the rows
    before the tail, on the host."""
    g = torch.Generator().manual_seed(seed * 2 + 1)
    share = torch.rand(case['groups'], generator=g, dtype=torch.float64).clamp_(min=1e-12).log_().neg_()
    edges = torch.cumsum(share, 0)
    edges = (edges / edges[-1] * (case['rows'] - case['tail'])).round().to(torch.int64)
    return torch.diff(edges, prepend=torch.zeros(1, dtype=torch.int64))


def prepare(case, seed):
    g = torch.Generator(device='cuda').manual_seed(seed)
    dtype = TYPES[case['dtype']]

    def normal(*shape, std=1.0):
        return (torch.randn(shape, generator=g, device='cuda') * std).to(dtype)

    s = dict(case=case)
    if case['op'] == 'dispatch':
        n, k, e, w = case['rows'], case['choices'], case['experts'], case['width']
        # skewed, distinct choices: the top k of noise around a preference that differs among experts
        preference = torch.randn(e, generator=g, device='cuda')
        noise = -torch.rand((n, e), generator=g, device='cuda').clamp_(min=1e-20).log_().neg_().log_()
        logits = preference + noise
        top = torch.topk(logits, k, dim=1)
        expert = top.indices.to(torch.int32)
        if case['dropped']:
            gone = torch.rand((n, k), generator=g, device='cuda') < case['dropped']
            expert = torch.where(gone, torch.full_like(expert, -1), expert)
        weights = torch.softmax(logits, 1).gather(1, top.indices)
        s.update(expert=expert, weights=weights, x=normal(n, w), results=normal(n * k, w))
        if case['train']:
            s.update(d_rows=normal(n * k, w), d_out=normal(n, w))
            s['x'].requires_grad_(), s['results'].requires_grad_(), s['weights'].requires_grad_()
    elif case['op'] == 'linear':
        m, i, o, groups = case['rows'], case['inputs'], case['outputs'], case['groups']
        lead = (groups,) if groups else ()
        s.update(x=normal(m, i), weight=normal(*lead, o, i, std=i ** -0.5), bias=None, residual=None, offsets=None)
        if case['bias']:
            s['bias'] = normal(*lead, o, std=0.5)
        if case['residual']:
            s['residual'] = normal(m, o)
        if groups:
            sizes = _group_sizes(case, seed)
            offsets = torch.zeros(groups + 1, dtype=torch.int32)
            offsets[1:] = torch.cumsum(sizes, 0)
            s.update(offsets=offsets.cuda(), longest=max(1, int(sizes.max())))
        if case['train']:
            s['d_out'] = normal(m, o)
            s['leaves'] = [name for name in ('x', 'weight', 'bias', 'residual') if s[name] is not None]
            [s[name].requires_grad_() for name in s['leaves']]
    else:
        n, v, w = case['ids'], case['table'], case['width']
        rank = (torch.rand(n, generator=g, device='cuda', dtype=torch.float64) ** case['skew'] * v).long().clamp_(max=v - 1)
        ids = torch.randperm(v, generator=g, device='cuda')[rank]
        if case['masked']:
            ids = torch.where(torch.rand(n, generator=g, device='cuda') < case['masked'], torch.full_like(ids, -1), ids)
        s.update(ids=ids, table=normal(v, w, std=0.5))
        if case['train']:
            s['d_out'] = normal(n, w)
            s['table'].requires_grad_()
    return s


# ---------------------------------------------------------------- one pass
def run(s):
    return {'dispatch': _dispatch, 'linear': _linear, 'embed': _embed}[s['case']['op']](s)


def _dispatch(s):
    case = s['case']
    if own:
        from odie_b200.experts import combine, dispatch, sort_rows
        order = sort_rows(s['expert'], case['experts'])
        rows = dispatch(s['x'], order)
        out = combine(s['results'], order, s['weights'])
        answer = dict(offsets=order.offsets, rows=rows.detach(), out=out.detach())
        if case['train']:
            leaves = [s['x'], s['results'], s['weights']]
            answer.update(zip(('d_x', 'd_results', 'd_weights'),
                              torch.autograd.grad([rows, out], leaves, [s['d_rows'], s['d_out']])))
        return answer
    n, k, e, w = case['rows'], case['choices'], case['experts'], case['width']
    dtype = s['x'].dtype
    key = s['expert'].reshape(-1).long()
    dropped = (key < 0) | (key >= e)
    key = torch.where(dropped, e, key)
    ordered, order = torch.sort(key, stable=True)
    offsets = torch.searchsorted(ordered, torch.arange(e + 1, device=key.device)).to(torch.int32)
    slot = torch.empty_like(order)
    slot[order] = torch.arange(n * k, device=key.device)
    live = (~dropped).float()
    x, results, weights = s['x'].detach().float(), s['results'].detach().float(), s['weights'].detach().float()
    rows = x[order // k] * live[order][:, None]
    taken = results[slot].view(n, k, w) * live.view(n, k, 1)
    out = (taken * weights[:, :, None]).sum(1)
    answer = dict(offsets=offsets, rows=rows.to(dtype), out=out.to(dtype))
    if case['train']:
        d_rows, d_out = s['d_rows'].float(), s['d_out'].float()
        d_x = (d_rows[slot] * live[:, None]).view(n, k, w).sum(1)
        d_results = d_out[order // k] * (weights.reshape(-1) * live)[order][:, None]
        d_weights = (taken * d_out[:, None, :]).sum(2)
        answer.update(d_x=d_x.to(dtype), d_results=d_results.to(dtype), d_weights=d_weights)
    return answer


def _activated(z, name):
    """(act(z), act'(z)) from elementary operations."""
    if name == 'relu':
        on = (z > 0).to(z.dtype)
        return z * on, on
    if name == 'silu':
        p = torch.sigmoid(z)
        return z * p, p * (1 + z * (1 - p))
    if name == 'gelu':
        p = 0.5 * (1 + torch.erf(z * math.sqrt(0.5)))
        return z * p, p + z * torch.exp(-0.5 * z * z) * (1 / math.sqrt(2 * math.pi))
    return z, torch.ones_like(z)


def _linear(s):
    case = s['case']
    if own:
        from odie_b200.experts import linear
        y = linear(s['x'], s['weight'], bias=s['bias'], residual=s['residual'], activation=case['activation'],
                   offsets=s['offsets'])
        answer = dict(y=y.detach())
        if case['train']:
            grads = torch.autograd.grad(y, [s[name] for name in s['leaves']], s['d_out'])
            answer.update(zip(('d_' + name for name in s['leaves']), grads))
        return answer
    dtype = s['x'].dtype
    x, weight = s['x'].detach().float(), s['weight'].detach().float()
    bias = None if s['bias'] is None else s['bias'].detach().float()
    residual = None if s['residual'] is None else s['residual'].detach().float()
    if case['groups']:  # every group padded to the longest one, one batched product
        m, groups, longest = case['rows'], case['groups'], s['longest']
        position = torch.arange(m, device=x.device)
        edges = s['offsets'].long()
        group = torch.searchsorted(edges[1:], position, right=True)
        live = (group < groups).float()[:, None]
        group = group.clamp(max=groups - 1)
        place = (group, (position - edges[group]).clamp(max=longest - 1))

        def padded(rows):
            return torch.zeros((groups, longest, rows.shape[1]), device=x.device).index_put(place, rows * live, True)
        xp = padded(x)
        z = torch.bmm(xp, weight.transpose(1, 2))[place]
        z = z if bias is None else z + bias[group]
    else:
        live = 1.0
        z = x @ weight.t()
        z = z if bias is None else z + bias
    a, slope = _activated(z, case['activation'])
    y = a if residual is None else a + residual
    answer = dict(y=(y * live).to(dtype))
    if case['train']:
        d_out = s['d_out'].float() * live
        dz = d_out * slope
        if case['groups']:
            dzp = padded(dz)
            grads = dict(x=torch.bmm(dzp, weight)[place] * live, weight=torch.bmm(dzp.transpose(1, 2), xp),
                         bias=dzp.sum(1), residual=d_out)
        else:
            grads = dict(x=dz @ weight, weight=dz.t() @ x, bias=dz.sum(0), residual=d_out)
        answer.update({'d_' + name: grads[name].to(dtype) for name in s['leaves']})
    return answer


def _embed(s):
    case = s['case']
    if own:
        from odie_b200.experts import embed
        out = embed(s['ids'], s['table'], scale=case['scale'])
        answer = dict(out=out.detach())
        if case['train']:
            answer['d_table'] = torch.autograd.grad(out, s['table'], s['d_out'])[0]
        return answer
    table, dtype = s['table'].detach(), s['table'].dtype
    live = (s['ids'] >= 0) & (s['ids'] < case['table'])
    safe = torch.where(live, s['ids'], 0)
    out = table[safe].float() * (case['scale'] * live.float())[:, None]
    answer = dict(out=out.to(dtype))
    if case['train']:
        d = s['d_out'].double() * (case['scale'] * live.double())[:, None]
        total = torch.zeros(table.shape, dtype=torch.float64, device=table.device).index_add_(0, safe, d)
        answer['d_table'] = total.to(dtype)
    return answer


# ---------------------------------------------------------------- least work
def work(case):
    size = BYTES[case['dtype']]
    if case['op'] == 'dispatch':
        n, k, w = case['rows'], case['choices'], case['width']
        moved = (2 * n + 2 * n * k) * w * size + n * k * 8 + 4 * (case['experts'] + 1)  # x, rows, results, out
        flops = 2 * n * k * w
        if case['train']:  # d_rows, d_x, d_out, d_results; the results and weights again; d_weights
            moved += (2 * n + 3 * n * k) * w * size + n * k * 8
            flops += (1 + 1 + 2) * n * k * w
        return dict(bytes=moved, flops=flops)
    if case['op'] == 'linear':
        m, i, o, g = case['rows'], case['inputs'], case['outputs'], max(1, case['groups'])
        moved = m * i + g * o * i + m * o * (2 if case['residual'] else 1) + (g * o if case['bias'] else 0)
        flops = 2 * (m - case['tail']) * i * o
        if case['train']:  # d_out, x and the weights again; their gradients
            moved += m * o + m * i + g * o * i + m * i + g * o * i + (g * o if case['bias'] else 0)
            flops *= 3
        return dict(bytes=moved * size, flops=flops)
    n, v, w = case['ids'], case['table'], case['width']
    moved = n * 8 + (min(n, v) + n) * w * size
    flops = n * w
    if case['train']:
        moved += n * 8 + (n + v) * w * size
        flops += n * w
    return dict(bytes=moved, flops=flops)


# ---------------------------------------------------------------- the definitions in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    with torch.no_grad():
        return {'dispatch': _exact_dispatch, 'linear': _exact_linear, 'embed': _exact_embed}[case['op']](s, case)


def _exact_dispatch(s, case):
    n, k, e, w = case['rows'], case['choices'], case['experts'], case['width']
    expert = s['expert'].long().cpu().reshape(-1)
    groups = [torch.nonzero(expert == j).reshape(-1) for j in range(e)]
    sequence = torch.cat(groups)  # the pairs in their order, expert by expert, without the dropped ones
    count = sequence.numel()
    offsets = torch.zeros(e + 1, dtype=torch.int32)
    offsets[1:] = torch.cumsum(torch.tensor([len(q) for q in groups]), 0)
    sequence = sequence.cuda()
    token = sequence // k
    x, y, p = s['x'].double(), s['results'].double()[:count], s['weights'].double().reshape(-1)[sequence][:, None]
    rows = torch.zeros((n * k, w), dtype=torch.float64, device='cuda')
    rows[:count] = x[token]
    out = torch.zeros((n, w), dtype=torch.float64, device='cuda').index_add_(0, token, p * y)
    answer = dict(offsets=None, rows=rows, out=out)
    if case['train']:
        d_rows, d_out = s['d_rows'].double()[:count], s['d_out'].double()
        d_x = torch.zeros((n, w), dtype=torch.float64, device='cuda').index_add_(0, token, d_rows)
        d_results = torch.zeros((n * k, w), dtype=torch.float64, device='cuda')
        d_results[:count] = p * d_out[token]
        d_weights = torch.zeros(n * k, dtype=torch.float64, device='cuda')
        d_weights[sequence] = torch.einsum('rw,rw->r', y, d_out[token])
        answer.update(d_x=d_x, d_results=d_results, d_weights=d_weights.view(n, k))
    return answer


def _exact_linear(s, case):
    m, i, o = case['rows'], case['inputs'], case['outputs']
    edges = s['offsets'].tolist() if case['groups'] else [0, m]
    x, weight = s['x'].double(), s['weight'].double().view(-1, o, i)
    bias = None if s['bias'] is None else s['bias'].double().view(-1, o)
    y = torch.zeros((m, o), dtype=torch.float64, device='cuda')
    d = {name: torch.zeros(s[name].shape, dtype=torch.float64, device='cuda') for name in s.get('leaves', [])}
    for j, (a, b) in enumerate(zip(edges[:-1], edges[1:])):
        z = x[a:b] @ weight[j].t()
        if bias is not None:
            z += bias[j]
        name = case['activation']
        if name == 'silu':
            value, slope = z / (1 + torch.exp(-z)), (1 + torch.exp(-z) * (1 + z)) / (1 + torch.exp(-z)) ** 2
            far = z < -300  # exp(-z)^2 leaves the range: silu and its slope are zero there to any precision
            value, slope = value.masked_fill(far, 0), slope.masked_fill(far, 0)
        elif name == 'gelu':
            cdf = torch.special.ndtr(z)
            value, slope = z * cdf, cdf + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)
        elif name == 'relu':
            value, slope = z.clamp(min=0), (z > 0).double()
        else:
            value, slope = z, 1.0
        y[a:b] = value if s['residual'] is None else value + s['residual'][a:b].double()
        if case['train']:
            g = s['d_out'][a:b].double()
            dz = g * slope
            d['x'][a:b] = dz @ weight[j]
            d['weight'].view(-1, o, i)[j] = dz.t() @ x[a:b]
            if bias is not None:
                d['bias'].view(-1, o)[j] = dz.sum(0)
            if s['residual'] is not None:
                d['residual'][a:b] = g
    return dict(y=y, **{'d_' + name: value for name, value in d.items()})


def _exact_embed(s, case):
    ids, scale = s['ids'], case['scale']
    good = torch.nonzero((ids >= 0) & (ids < case['table'])).reshape(-1)
    out = torch.zeros((case['ids'], case['width']), dtype=torch.float64, device='cuda')
    out[good] = scale * s['table'].double()[ids[good]]
    answer = dict(out=out)
    if case['train']:
        ordered, back = torch.sort(ids[good], stable=True)
        sums = torch.zeros(s['table'].shape, dtype=torch.float64, device='cuda')
        # running sums of the rows in id order, a block of columns at a time, and their differences at the ids' ends
        edges = torch.searchsorted(ordered, torch.arange(case['table'] + 1, device=ids.device))
        for c in range(0, case['width'], 128):
            run_sum = torch.zeros((good.numel() + 1, min(128, case['width'] - c)), dtype=torch.float64, device='cuda')
            run_sum[1:] = torch.cumsum(s['d_out'][good][:, c:c + 128].double()[back], 0)
            sums[:, c:c + 128] = run_sum[edges[1:]] - run_sum[edges[:-1]]
        answer['d_table'] = scale * sums
    return answer
