"""The routed-expert row operators on the GPU (odie_b200.experts) at the ends of what they take: derivatives of other
kinds, the widest rows, values that are no numbers, far tails, waits that run out.  Bounds as in rows_cases."""
import pytest
import torch

from rows_cases import SUM, plain_linear, rounding, within

pytestmark = pytest.mark.gpu

HALVES = [torch.float16, torch.bfloat16]


def generator(seed):
    return torch.Generator(device='cuda').manual_seed(seed)


def normal(g, *shape, dtype=torch.float32, std=1.0):
    return (torch.randn(shape, generator=g, device='cuda') * std).to(dtype)


# ---------------------------------------------------------------- derivatives of other kinds
def differentiable_calls():
    """{name: (call, its differentiable arguments)} of every operator."""
    from odie_b200.experts import combine, dispatch, embed, linear, sort_rows
    g = generator(1)
    order = sort_rows(torch.randint(0, 3, (30, 2), generator=g, device='cuda'), 3)
    ids = torch.randint(0, 5, (30,), generator=g, device='cuda')
    weights = torch.rand((30, 2), generator=g, device='cuda')
    half = [normal(g, *s, dtype=torch.float16) for s in ((30, 16), (24, 16), (24,), (30, 24))]
    return {'linear': (lambda x, w, b, r: linear(x, w, b, r, 'silu'), half),
            'linear x.T': (lambda x, w: linear(x.t(), w), [half[0].t().contiguous(), half[1]]),
            'dispatch': (lambda x, p: dispatch(x, order, p), [normal(g, 30, 8), weights]),
            'combine': (lambda y, p: combine(y, order, p), [normal(g, 60, 8), weights]),
            'embed': (lambda table: embed(ids, table), [normal(g, 5, 16)])}


@pytest.mark.parametrize('name', ['linear', 'linear x.T', 'dispatch', 'combine', 'embed'])
@pytest.mark.parametrize('requires_grad', [False, True])
def test_forward_mode_is_refused(cuda, name, requires_grad):
    """A tangent is not dropped: of an argument, or of the gradient that a backward pass is given."""
    from torch.autograd import forward_ad
    call, arguments = differentiable_calls()[name]
    with forward_ad.dual_level():
        for i, t in enumerate(arguments):
            dual = forward_ad.make_dual(t.detach().clone().requires_grad_(requires_grad), torch.ones_like(t))
            for grad in (torch.enable_grad, torch.no_grad):
                with grad(), pytest.raises(RuntimeError, match='forward-mode'):
                    call(*arguments[:i], dual, *arguments[i + 1:])
        leaves = [t.detach().clone().requires_grad_() for t in arguments]
        y = call(*leaves)
        d = torch.ones_like(y)
        want = torch.autograd.grad(y, leaves, d, retain_graph=True)
        with pytest.raises(RuntimeError, match='forward-mode'):
            torch.autograd.grad(y, leaves, forward_ad.make_dual(d, torch.ones_like(d)), retain_graph=True)
        assert all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(y, leaves, d), want))


@pytest.mark.parametrize('name', ['linear', 'dispatch', 'combine', 'embed'])
def test_function_transforms_are_refused(cuda, name):
    call, arguments = differentiable_calls()[name]
    first, rest = arguments[0], arguments[1:]
    for transformed in (lambda: torch.func.vmap(lambda t: call(t, *rest))(first[None]),
                        lambda: torch.func.grad(lambda t: call(t, *rest).float().sum())(first),
                        lambda: torch.func.jvp(lambda t: call(t, *rest), (first,), (first,))):
        with pytest.raises(RuntimeError):
            transformed()


@pytest.mark.parametrize('activation', ['relu', 'silu', 'gelu'])
@pytest.mark.parametrize('inputs, outputs', [(16, 24), (80, 72)])
def test_second_derivatives_of_linear_are_refused(cuda, activation, inputs, outputs):
    """Also where the first derivative that is asked for keeps little: a smooth slope depends on x, weight and bias."""
    from odie_b200.experts import linear
    g = generator(1)
    arguments = [normal(g, *s, dtype=torch.float16) for s in ((30, inputs), (outputs, inputs), (outputs,), (30, outputs))]
    smooth = activation != 'relu'
    for wanted in ([0], [1], [2], [0, 1, 2, 3]):
        leaves = [t.detach().clone().requires_grad_(j in wanted) for j, t in enumerate(arguments)]
        y = linear(*leaves, activation)
        first = torch.autograd.grad(y, [leaves[i] for i in wanted], torch.ones_like(y), create_graph=True)
        for i, a in zip(wanted, first):
            for j in wanted:
                if (smooth and i < 3 and j < 3) or (i, j) in ((0, 1), (1, 0)):
                    with pytest.raises(RuntimeError, match='once'):
                        torch.autograd.grad(a.float().square().sum(), leaves[j], retain_graph=True, allow_unused=True)


@pytest.mark.parametrize('name', ['dispatch', 'combine'])
def test_second_derivatives_between_rows_and_weights_are_refused(cuda, name):
    call, arguments = differentiable_calls()[name]
    leaves = [t.detach().clone().requires_grad_() for t in arguments]
    y = call(*leaves)
    first = torch.autograd.grad(y, leaves, torch.ones_like(y), create_graph=True)
    for a, other in zip(first, leaves[::-1]):
        with pytest.raises(RuntimeError, match='once'):
            torch.autograd.grad(a.float().square().sum(), other, retain_graph=True, allow_unused=True)


# ---------------------------------------------------------------- the widest rows
@pytest.mark.parametrize('rows, inputs, outputs', [(3, 8, 1 << 20), (5, 16, (1 << 20) - 8), (2, 8, 1 << 20), (3, 1 << 20, 8), (3, 4, (1 << 20) - 3)])
def test_linear_of_the_most_inputs_and_outputs(cuda, rows, inputs, outputs):
    """Up to 2^20 of either, with every gradient."""
    from odie_b200.experts import linear
    g = generator(rows + inputs)
    case = [normal(g, *s, dtype=torch.bfloat16, std=std) for s, std in (((rows, inputs), 1), ((outputs, inputs), inputs ** -0.5), ((outputs,), 1),
                                                                        ((rows, outputs), 1), ((rows, outputs), 1))]
    leaves = [t.requires_grad_() for t in case[:4]]
    y = linear(*leaves, 'silu')
    grads = torch.autograd.grad(y, leaves, case[4])
    plain = plain_linear(*(t.detach() for t in case[:4]), [(0, rows)], 'silu', case[4])
    within(y.detach(), *plain['y'], 'y')
    for name, got in zip(('x', 'weight', 'bias', 'residual'), grads):
        within(got, *plain['d_' + name], 'd_' + name)


@pytest.mark.parametrize('dtype, width', [(torch.float16, 65535 * 256 + 1), (torch.float32, 65535 * 256 + 3)])
def test_embed_of_very_wide_rows(cuda, dtype, width):
    """More columns than one launch's second grid dimension holds."""
    from odie_b200.experts import embed
    g = generator(3)
    ids = torch.tensor([1, 0, 1, 5], device=cuda)
    table, d_out = normal(g, 3, width, dtype=dtype).requires_grad_(), normal(g, 4, width, dtype=dtype)
    out = embed(ids, table)
    assert torch.equal(out[:3], table[ids[:3]]) and (out[3] == 0).all()
    (grad,) = torch.autograd.grad(out, table, d_out)
    assert torch.equal(grad[0], d_out[1]) and (grad[2] == 0).all()
    assert torch.equal(grad[1], (d_out[0].float() + d_out[2].float()).to(dtype))  # one fp32 sum, rounded once
