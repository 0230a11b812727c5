"""The router's operators on the GPU (gate, balance of odie_b200.experts) against plain 64-bit forms."""
import pytest
import torch

from router_cases import plain_balance, plain_gate
from rows_cases import TYPES, within

pytestmark = pytest.mark.gpu

# rows, experts, choices
SIZES = [(1, 1, 1), (1, 64, 2), (3, 7, 7), (33, 8, 3), (257, 9, 2), (1000, 16, 1), (130, 37, 5), (65, 64, 64), (129, 100, 8), (77, 256, 8), (500, 200, 16), (300, 256, 4), (64, 130, 5),
         (50, 257, 4), (31, 512, 64), (9, 1000, 10), (17, 1024, 64), (5003, 16, 4)]


def made(rows, experts, dtype, seed, spread=2.0):
    g = torch.Generator(device='cuda').manual_seed(seed)
    logits = (torch.randn((rows, experts), generator=g, device='cuda') * spread).to(dtype)
    if rows > 2:
        logits[rows // 2] = logits[rows // 2, 0]  # a row of ties
    return g, logits


def masks(kind, g, rows, experts):
    if kind == 'none':
        return None
    if kind == 'experts':
        mask = torch.rand(experts, generator=g, device='cuda') < 0.7
        return mask
    if kind == 'rows':
        return torch.rand((rows, 1), generator=g, device='cuda') < 0.8
    mask = torch.rand((rows, experts), generator=g, device='cuda') < 0.5
    mask[0] = False  # nothing is left
    if kind == 'strided':
        return torch.stack([mask, ~mask], 2)[..., 0]
    return mask


@pytest.mark.parametrize('rows, experts, choices', SIZES)
@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('score, normalize', [('softmax', True), ('softmax', False), ('sigmoid', True), ('sigmoid', False)])
def test_gate(cuda, rows, experts, choices, dtype, score, normalize):
    from odie_b200.experts import gate
    for kind, biased, scale in (('none', False, 1.0), ('dense', True, 2.5), ('rows', False, -0.5), ('experts', True, 1.0), ('strided', False, 1.0)):
        g, logits = made(rows, experts, dtype, rows + experts)
        mask = masks(kind, g, rows, experts)
        bias = torch.randn(experts, generator=g, device='cuda') if biased else None
        d_weights = torch.randn((rows, choices), generator=g, device='cuda')
        logits.requires_grad_()
        expert, weights = gate(logits, choices, bias=bias, mask=mask, score=score, normalize=normalize, scale=scale)
        (d_logits,) = torch.autograd.grad(weights, logits, d_weights)
        want = plain_gate(logits.detach(), choices, bias, mask, score, normalize, scale, d_weights)
        assert expert.dtype == torch.int32 and torch.equal(expert.long(), want[0]), kind
        within(weights.detach(), *want[1], f'weights {kind}')
        assert d_logits.dtype == dtype
        within(d_logits, *want[2], f'd_logits {kind}')
        again = gate(logits.detach(), choices, bias=bias, mask=mask, score=score, normalize=normalize, scale=scale)
        assert torch.equal(again.expert, expert) and torch.equal(again.weights, weights.detach())


def test_gate_gradient_against_differences(cuda):
    """d weights / d logits by central differences in fp32: their rounding is 2^-24 of a weight over a step of 2^-6,
    their curvature at most the step's square."""
    from odie_b200.experts import gate
    _, logits = made(40, 12, torch.float32, 3, spread=1.0)
    g = torch.Generator(device='cuda').manual_seed(4)
    d_weights = torch.randn((40, 3), generator=g, device='cuda')
    for score, normalize in (('softmax', True), ('softmax', False), ('sigmoid', True), ('sigmoid', False)):
        leaf = logits.clone().requires_grad_()
        expert, weights = gate(leaf, 3, score=score, normalize=normalize)
        (d,) = torch.autograd.grad(weights, leaf, d_weights)
        step = 2.0 ** -6
        for e in range(12):
            ahead, behind = logits.clone(), logits.clone()
            ahead[:, e] += step
            behind[:, e] -= step
            sides = [gate(x, 3, score=score, normalize=normalize) for x in (ahead, behind)]
            same = (sides[0].expert == expert).all(1) & (sides[1].expert == expert).all(1)
            slope = ((sides[0].weights - sides[1].weights).double() * d_weights).sum(1) / (2 * step)
            error = (slope - d[:, e])[same].abs()
            assert same.sum() > 20 and error.max() <= d_weights.abs().sum(1).max() * (step ** 2 + 2.0 ** -24 * 64 / step)


@pytest.mark.parametrize('dtype', TYPES)
def test_gate_of_extreme_logits(cuda, dtype):
    """The type's lowest value as a mask, infinities, NaN behind a mask and before it, -0 beside 0, far negative rows."""
    from odie_b200.experts import gate
    low = torch.finfo(dtype).min
    inf, nan = float('inf'), float('nan')
    logits = torch.tensor([[low, low, low, low], [low, 1, low, 2], [-inf, 3, -inf, -inf], [-inf, -inf, -inf, -inf], [nan, 1, 2, 3],
                           [-0.0, 0.0, -1, -0.0], [-300, -200, -250, -201], [300, 200, 299, 298]], dtype=dtype, device='cuda')
    mask = torch.ones((8, 4), dtype=torch.bool, device='cuda')
    mask[4, 0] = False
    for score, normalize in (('softmax', True), ('softmax', False), ('sigmoid', True), ('sigmoid', False)):
        leaf = logits.clone().requires_grad_()
        expert, weights = gate(leaf, 2, mask=mask, score=score, normalize=normalize)
        assert expert.tolist() == [[0, 1], [3, 1], [1, -1], [-1, -1], [3, 2], [0, 1], [1, 3], [0, 2]]
        (d,) = torch.autograd.grad(weights, leaf, torch.ones_like(weights))
        assert torch.isfinite(weights).all() and torch.isfinite(d).all()
        clean = torch.where(mask, logits, 0.0)
        want = plain_gate(clean, 2, None, mask, score, normalize, 1.0, torch.ones_like(weights))
        if score == 'softmax' or normalize:
            pairs = slice(1, None)  # (the plain logsigmoid of the lowest double is not meant here)
        else:
            pairs = slice(0, None)
        within(weights.detach()[pairs], want[1][0][pairs], want[1][1][pairs], 'weights')
        within(d[pairs], want[2][0][pairs], want[2][1][pairs], 'd_logits')
        assert score == 'sigmoid' or abs(weights[0, 0].item() - (0.5 if normalize else 0.25)) < 2.0 ** -20
    # an open NaN is taken first, and its row's softmax is NaN; other rows are as they were
    expert, weights = gate(logits[4:6], 2)
    assert expert.tolist() == [[0, 3], [0, 1]] and weights[0].isnan().all() and torch.isfinite(weights[1]).all()
    # a bias of -inf closes an expert to all rows, without taking it out of the softmax
    closed = torch.tensor([0, 0, 0, -inf], device='cuda')
    expert, weights = gate(logits[5:], 4, bias=closed, normalize=False)
    assert (expert[:, 3] == -1).all() and not (expert == 3).any()
    # infinite logits: NaN weights, as a softmax has them
    assert gate(torch.tensor([[inf, 0.0]], dtype=dtype, device='cuda'), 1).weights.isnan().all()


def test_gate_rows_strides_and_streams(cuda):
    """No rows, logits that are a strided or unaligned view, another stream, a gradient that is broadcast."""
    from odie_b200.experts import gate
    none = torch.zeros((0, 8), device='cuda', requires_grad=True)
    expert, weights = gate(none, 2)
    assert expert.shape == weights.shape == (0, 2)
    assert torch.autograd.grad(weights.sum(), none)[0].shape == (0, 8)
    g, wide = made(60, 49, torch.bfloat16, 5)
    for view in (wide[:, 1:33], wide[::2], wide.t()[:40].t(), wide.reshape(-1)[3:3 + 48 * 50].view(50, 48)):
        a, b = gate(view, 3), gate(view.clone(memory_format=torch.contiguous_format), 3)
        assert torch.equal(a.expert, b.expert) and torch.equal(a.weights, b.weights)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = gate(wide, 3)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(other.weights, gate(wide, 3).weights)
    leaf = wide.float().requires_grad_()
    weights = gate(leaf, 3, normalize=False).weights
    (d,) = torch.autograd.grad(weights.sum(), leaf, retain_graph=True)  # an expanded gradient
    (same,) = torch.autograd.grad(weights, leaf, torch.ones_like(weights))
    assert torch.equal(d, same)


# ---------------------------------------------------------------- balance
@pytest.mark.parametrize('rows, experts, choices', SIZES + [(100000, 5, 2), (70001, 64, 2)])
@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('score', ['softmax', 'sigmoid'])
def test_balance(cuda, rows, experts, choices, dtype, score):
    from odie_b200.experts import balance
    for kind, ids in (('none', torch.int32), ('dense', torch.int64), ('rows', torch.int32), ('strided', torch.int32)):
        g, logits = made(rows, experts, dtype, rows + experts + 1)
        mask = masks(kind, g, rows, experts)
        expert = torch.randint(-1, experts + 1, (rows, choices), generator=g, device='cuda', dtype=ids)
        if ids == torch.int64:
            expert[0] = 1 << 40
        total = torch.randint(0, 1000, (experts,), generator=g, device='cuda', dtype=torch.int64) if kind == 'rows' else None
        logits.requires_grad_()
        loss, z, counts = balance(logits, expert, mask=mask, score=score, total=total)
        scale_loss, scale_z = float(rows), 0.25 * rows
        (d,) = torch.autograd.grad([loss, z], logits, [torch.tensor(scale_loss, device='cuda'), torch.tensor(scale_z, device='cuda')])
        want, want_counts, want_d = plain_balance(logits.detach(), expert, mask, score, total, scale_loss, scale_z)
        assert counts.dtype == torch.int32 and torch.equal(counts.long(), want_counts)
        within(loss.detach(), *want['loss'], f'loss {kind}')
        within(z.detach(), *want['z'], f'z {kind}')
        within(d, *want_d, f'd_logits {kind}')
        again = balance(logits, expert, mask=mask, score=score, total=total)
        assert all(torch.equal(a, b) for a, b in zip(again, (loss, z, counts)))


def test_balance_of_one_term(cuda):
    """Only the loss, or only z, is differentiated; an even load has a loss of 1; none has no gradient."""
    from odie_b200.experts import balance
    _, logits = made(96, 12, torch.float32, 7)
    expert = torch.arange(96, device='cuda', dtype=torch.int32) % 12
    leaf = logits.clone().requires_grad_()
    loss, z, counts = balance(leaf, expert)
    assert (counts == 8).all() and abs(loss.item() - 1) <= 2.0 ** -20 and not counts.requires_grad
    for out, scales in ((loss, (1.0, 0.0)), (z, (0.0, 1.0))):
        (d,) = torch.autograd.grad(out, leaf, retain_graph=True)
        within(d, *plain_balance(logits, expert, None, 'softmax', None, *scales)[2], 'one term')


def test_balance_of_nothing(cuda):
    """No rows; rows that are all masked; choices that are all dropped."""
    from odie_b200.experts import balance
    for rows, mask, key in ((0, None, 0), (5, torch.zeros((5, 1), dtype=torch.bool, device='cuda'), 1), (5, None, -1)):
        logits = torch.randn((rows, 6), device='cuda', requires_grad=True)
        loss, z, counts = balance(logits, torch.full((rows, 2), key, dtype=torch.int32, device='cuda'), mask=mask)
        (d,) = torch.autograd.grad(loss + z, logits)
        assert loss.item() == 0 and (z.item() == 0) == (key != -1) and torch.isfinite(d).all() and d.shape == (rows, 6)
        assert counts.tolist() == ([0] * 6 if rows == 0 or key < 0 else [0, 10, 0, 0, 0, 0])


@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('score', ['softmax', 'sigmoid'])
def test_balance_of_extreme_logits(cuda, dtype, score):
    from odie_b200.experts import balance
    low = torch.finfo(dtype).min
    inf = float('inf')
    logits = torch.tensor([[low, 1, low, 2], [-inf, 3, -inf, -inf], [-inf, -inf, -inf, -inf], [float('nan'), 1, 2, 3], [-300, -200, -250, -201],
                           [300, 200, 299, 298], [-100, 20, -90, 3]], dtype=dtype, device='cuda')
    mask = torch.ones((7, 4), dtype=torch.bool, device='cuda')
    mask[3, 0] = False
    expert = torch.tensor([[3, 1], [1, -1], [-1, -1], [3, 2], [1, 3], [0, 2], [1, 3]], dtype=torch.int32, device='cuda')
    leaf = logits.clone().requires_grad_()
    loss, z, counts = balance(leaf, expert, mask=mask, score=score)
    (d,) = torch.autograd.grad(loss + z, leaf)
    want, want_counts, want_d = plain_balance(torch.where(mask, logits, 0.0), expert, mask, score, None, 1.0, 1.0)
    assert counts.tolist() == want_counts.tolist() and torch.isfinite(d).all()
    within(loss.detach(), *want['loss'], 'loss')
    within(z.detach(), *want['z'], 'z')
    within(d, *want_d, 'd_logits')


def test_router_is_captured_and_replayed(cuda):
    """gate and balance with their gradients in one graph, replayed on other logits."""
    from odie_b200.experts import balance, gate
    _, logits = made(300, 24, torch.bfloat16, 9)
    _, others = made(300, 24, torch.bfloat16, 10)
    d_weights = torch.randn((300, 2), device='cuda')

    def step(leaf):
        routing = gate(leaf, 2, normalize=False)
        loss, z, counts = balance(leaf, routing.expert)
        (d,) = torch.autograd.grad((routing.weights * d_weights).sum() + loss + 0.1 * z, leaf)
        return [*routing, loss, z, counts, d]
    want = [[t.detach().clone() for t in step(x.clone().requires_grad_())] for x in (logits, others)]
    static = logits.clone().requires_grad_()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(static)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        results = step(static)
    for x, w in zip((logits, others, logits), (want[0], want[1], want[0])):
        with torch.no_grad():
            static.copy_(x)
        graph.replay()
        assert all(torch.equal(a.detach(), b) for a, b in zip(results, w))


def test_router_is_differentiable_once(cuda):
    from odie_b200.experts import balance, gate
    leaf = torch.randn((10, 6), device='cuda', requires_grad=True)
    expert, weights = gate(leaf, 2)
    (d,) = torch.autograd.grad(weights.square().sum(), leaf, create_graph=True)
    with pytest.raises(RuntimeError, match='differentiable once'):
        d.sum().backward()
    loss, z, _ = balance(leaf, expert)
    (d,) = torch.autograd.grad(loss * z, leaf, create_graph=True)
    with pytest.raises(RuntimeError, match='differentiable once'):
        d.sum().backward()
    import torch.autograd.forward_ad as forward
    with forward.dual_level():
        dual = forward.make_dual(leaf.detach(), torch.ones_like(leaf))
        for call in (lambda: gate(dual, 2), lambda: balance(dual, expert)):
            with pytest.raises(NotImplementedError, match='forward-mode'):
                call()
