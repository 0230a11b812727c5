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


# ---------------------------------------------------------------- what is no number, in other rows
def passing(x, weight, **kwargs):
    """[rows, outputs] bool: where linear's ReLU passes a gradient, one output at a time: d x is then a row of W or 0."""
    from odie_b200.experts import linear
    x = x.clone().requires_grad_()
    y = linear(x, weight, activation='relu', **kwargs)
    found = torch.empty(y.shape, dtype=torch.bool, device=y.device)
    for n in range(y.shape[1]):
        d_y = torch.zeros_like(y)
        d_y[:, n] = 1
        (d_x,) = torch.autograd.grad(y, x, d_y, retain_graph=True)
        found[:, n] = (d_x != 0).any(1)
    return found


@pytest.mark.parametrize('poison', [float('nan'), float('inf'), float('-inf')])
@pytest.mark.parametrize('inputs, outputs', [(32, 16), (64, 64), (24, 40)])
@pytest.mark.parametrize('dtype', HALVES)
def test_thin_relu_corner_beside_rows_of_no_numbers(cuda, poison, inputs, outputs, dtype):
    """A row's units go by its own fp32 chain in ascending order of the inputs (a unit of sum zero is off), whatever stands
    in the rows around it: sums that cancel to their last bits, with all their weight in even columns, and rows of zeros."""
    g = generator(inputs)
    rows = 4096
    x, w = normal(g, rows, inputs, dtype=dtype), normal(g, outputs, inputs, std=0.3, dtype=dtype)
    x[:, 1::2] = 0
    for level in range(3):  # the last even inputs cancel the sum of output 0 to 2^-24 of it
        k = inputs - 6 + 2 * level
        w[0, k] = 2.0 ** (-8 * level)
        x[:, k] = (-(x[:, :k].double() @ w[0, :k].double()) * 2.0 ** (8 * level)).to(dtype)
    x[::5] = 0
    hit = torch.rand(rows, generator=g, device=cuda) < 0.3
    x[hit, torch.randint(inputs // 2, (rows,), generator=g, device=cuda)[hit] * 2] = poison
    both = hit & (torch.rand(rows, generator=g, device=cuda) < 0.3)
    x[both] = poison
    chain = torch.zeros(rows, outputs, device=cuda)
    for k in range(inputs):
        chain = chain + x[:, k:k + 1].float() * w[:, k].float()
    found = passing(x, w)
    assert torch.equal(found[~hit], chain[~hit] > 0)


def relu_bits(x, weight, bias):
    """[rows, outputs] bool: the ReLU's bits that the C interface keeps for the gradient."""
    from odie_b200 import _lib
    (rows, inputs), outputs = x.shape, weight.shape[0]
    y, bits = x.new_empty(rows, outputs), torch.empty((rows, (outputs + 7) // 8, 1), device=x.device, dtype=torch.uint8)
    status = _lib.library().odie_linear(x.data_ptr(), weight.data_ptr(), bias.data_ptr(), None, rows, inputs, outputs, 1, None,
                                        int(x.dtype == torch.bfloat16), 1, y.data_ptr(), bits.data_ptr(), None, _lib.stream_handle())
    _lib.check(status, 'odie_linear')
    return (bits >> torch.arange(8, device=x.device, dtype=torch.uint8) & 1).view(rows, -1)[:, :outputs].bool()


@pytest.mark.parametrize('where', ['weight', 'bias'])
@pytest.mark.parametrize('poison', [float('nan'), float('inf')])
def test_thin_relu_corner_beside_units_of_no_numbers(cuda, where, poison):
    """The same beside another output whose weights or bias are no numbers."""
    g = generator(7)
    rows, inputs, outputs = 2000, 32, 24
    x, w, b = normal(g, rows, inputs).half(), normal(g, outputs, inputs, std=0.3).half(), torch.zeros(outputs, device=cuda).half()
    w[:, 1::2] = 0
    for level in range(3):
        k = inputs - 6 + 2 * level
        w[0, k] = 2.0 ** (-8 * level)
        x[:, k] = (-(x[:, :k].double() @ w[0, :k].double()) * 2.0 ** (8 * level)).half()
    x[::5], x[640:768] = 0, 0
    chain = torch.zeros(rows, outputs, device=cuda)
    for k in range(inputs):
        chain = chain + x[:, k:k + 1].float() * w[:, k].float()
    if where == 'weight':
        w[5, 2] = poison
    else:
        b[5] = poison
    found = relu_bits(x, w, b)  # (d x would hold 0 times the other unit's weight)
    others = torch.arange(outputs, device=cuda) != 5
    assert torch.equal(found[:, others], chain[:, others] > 0)


# ---------------------------------------------------------------- far tails
@pytest.mark.parametrize('rows, width', [(2000, 64), (2000, 72), (1, 64), (2, 72), (100, 1024)])
@pytest.mark.parametrize('dtype', HALVES)
def test_gelu_tails(cuda, rows, width, dtype):
    """z P(z) to half a step of its own size and 2^-15 of it, from z = -9 to 9 (z: the elements of x, by a product with
    the unit matrix, exact).

    What the fp32 arithmetic is off by, relative to the result: P(-u) = t (polynomial in t) e^(-u^2/2) is a fit to
    2^-14.5 = 4.3e-5 of P in the far tail; e^(-u^2/2) with u^2/2 log2 e <= 58.5
    rounded twice, 2 x 58.5 x 2^-24 ln 2 = 4.8e-6; the approximate exponential and inverse and eight roundings,
    12 x 2^-23 = 1.4e-6.  Together below 2^-14."""
    from odie_b200.experts import linear
    z = (torch.linspace(-9, 9, rows * width, device=cuda) if rows > 2 else torch.linspace(-9, -3, rows * width, device=cuda)).to(dtype).view(rows, width)
    y = linear(z, torch.eye(width, device=cuda, dtype=dtype), activation='gelu')
    want = z.double() * torch.special.erfc(z.double() * -(0.5 ** 0.5)) / 2  # (ndtr's tail has an absolute grain of 1e-16)
    off = 2.0 ** -14 * want.abs()
    within(y, want, off + rounding(want.abs() + off, dtype), 'gelu')


# ---------------------------------------------------------------- waits that run out
@pytest.fixture
def wait_limit(cuda):
    from odie_b200 import _lib
    yield lambda polls: _lib.check(_lib.library().odie_linear_wait_limit(polls), 'odie_linear_wait_limit')
    torch.cuda.synchronize()
    _lib.library().odie_linear_wait_limit(-1)


def linear_status():
    from odie_b200 import _lib
    status = torch.full((1,), -1, dtype=torch.int32, device='cuda')
    _lib.check(_lib.library().odie_linear_status(status.data_ptr(), _lib.stream_handle()), 'odie_linear_status')
    return status.item()


# single tiles, the sum over K cut, tiles of 64 and 128 columns, SM pairs, several experts, units of a long sum over rows
WAITS = [(100, 72, 72, 0), (40, 2048, 200, 0), (3000, 200, 136, 0), (4096, 520, 2048, 0), (2000, 136, 264, 3), (20000, 256, 264, 0)]


@pytest.mark.parametrize('case', WAITS)
def test_linear_after_waits_that_ran_out(cuda, wait_limit, case):
    """A kernel whose waits give up (at once, or while its copies and products are on their way) ends, says so, and
    leaves the next one as it was."""
    from odie_b200 import experts
    rows, inputs, outputs, groups = case
    g = generator(rows)
    lead = (groups,) if groups else ()
    leaves = [normal(g, *s, dtype=torch.bfloat16).requires_grad_() for s in ((rows, inputs), (*lead, outputs, inputs), (*lead, outputs))]
    offsets = torch.linspace(0, rows - 7, groups + 1, device=cuda).int() if groups else None
    d = normal(g, rows, outputs, dtype=torch.bfloat16)

    def forward():
        return experts.linear(*leaves, activation='silu', offsets=offsets)
    y = forward()

    def backward():
        return torch.autograd.grad(y, leaves, d, retain_graph=True)
    grads = backward()
    for polls in (0, 1, 2, 3, 5):
        for call in (forward, backward):
            wait_limit(polls)
            call()
            torch.cuda.synchronize()
            wait_limit(-1)
            status = linear_status()
            assert status in ((2,) if polls == 0 else (0, 2))
            if status:
                with pytest.raises(RuntimeError, match='incomplete'):
                    experts.check()
            assert torch.equal(forward(), y) and all(torch.equal(a, b) for a, b in zip(backward(), grads))


@pytest.mark.parametrize('case', [(100, 72, 72, 0), (4096, 520, 2048, 0)])
def test_linear_raises_after_a_wait_that_ran_out(cuda, wait_limit, case):
    """Once, at the next forward or backward call or check, whichever comes first; also for a replayed graph."""
    from odie_b200 import experts
    g = generator(1)
    rows, inputs, outputs, _ = case
    x, w = normal(g, rows, inputs).half().requires_grad_(), normal(g, outputs, inputs).half().requires_grad_()
    want = experts.linear(x, w, activation='relu')
    d = torch.ones_like(want)
    grads = torch.autograd.grad(want, [x, w], d, retain_graph=True)

    def fails():
        wait_limit(0)
        experts.linear(x.detach(), w.detach())
        torch.cuda.synchronize()
        wait_limit(-1)
    for call in (lambda: experts.linear(x, w), lambda: torch.autograd.grad(want, [x, w], d, retain_graph=True), experts.check):
        fails()
        with pytest.raises(RuntimeError, match='incomplete'):
            call()
        call()
        experts.check()
    assert linear_status() == 0
    assert torch.equal(experts.linear(x, w, activation='relu'), want)
    assert all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(want, [x, w], d), grads))
    wait_limit(0)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        experts.linear(x.detach(), w.detach())
    wait_limit(-1)
    experts.check()
    for _ in range(2):
        graph.replay()
        with pytest.raises(RuntimeError, match='incomplete'):
            experts.check()
    experts.check()


def test_linear_captured_first(cuda):
    """A graph may hold the process's first call."""
    import subprocess
    import sys
    program = """
import torch
from odie_b200.experts import linear, check
x, w = torch.randn(300, 80, device='cuda').half(), torch.randn(72, 80, device='cuda').half()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    y = linear(x, w)
graph.replay()
check()
assert torch.equal(y, linear(x, w))
print('the same')
"""
    from pathlib import Path
    run = subprocess.run([sys.executable, '-c', program], capture_output=True, text=True, timeout=300, cwd=Path(__file__).resolve().parents[1])
    assert run.returncode == 0 and 'the same' in run.stdout, run.stderr


# ---------------------------------------------------------------- memory
def peak(call):
    """(bytes that call takes beside its results, its results)."""
    call()
    torch.cuda.synchronize()
    before = torch.cuda.memory_allocated()
    torch.cuda.reset_peak_memory_stats()
    results = call()
    torch.cuda.synchronize()
    return torch.cuda.max_memory_allocated() - torch.cuda.memory_allocated(), results


@pytest.mark.parametrize('rows', [1, 2])
def test_few_rows_take_no_scratch(cuda, rows):
    """No padded copy of the weights, whose rows are no multiple of 16 bytes."""
    from odie_b200.experts import linear
    g = generator(rows)
    x, w = normal(g, rows, 1025, dtype=torch.float16), normal(g, 2000, 1025, dtype=torch.float16)
    taken, y = peak(lambda: linear(x, w))
    assert taken == 0
    want, off = x.double() @ w.double().t(), 1026 * SUM * (x.double().abs() @ w.double().abs().t())
    within(y, want, off + rounding(want.abs() + off, torch.float16), 'y')


@pytest.mark.parametrize('shift', [0, 1])
def test_thin_gradients_take_the_sums_of_the_weights_alone(cuda, shift):
    """Also where the residual starts on no 16-byte boundary and the forward pass leaves the thin kernel."""
    from odie_b200.experts import linear
    g = generator(9)
    rows, inputs, outputs = 1 << 17, 32, 64
    x, w, b = (normal(g, *s, dtype=torch.float16).requires_grad_() for s in ((rows, inputs), (outputs, inputs), (outputs,)))
    residual = normal(g, rows * outputs + 8, dtype=torch.float16)[shift:shift + rows * outputs].view(rows, outputs)
    y = linear(x, w, b, residual, 'silu')
    d = normal(g, rows, outputs, dtype=torch.float16)
    taken, grads = peak(lambda: torch.autograd.grad(y, [x, w, b], d, retain_graph=True))
    assert taken <= 4 << 20  # 412 units of 33 x 64 fp32 sums: 3.5 MB; dz would be 17 MB
    plain = plain_linear(x.detach(), w.detach(), b.detach(), residual, [(0, rows)], 'silu', d)
    within(y.detach(), *plain['y'], 'y')
    for name, got in zip(('x', 'weight', 'bias'), grads):
        within(got, *plain['d_' + name], 'd_' + name)
