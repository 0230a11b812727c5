"""The routed-expert row operators on the GPU (odie_b200.experts) against plain 64-bit forms, with the bounds of
rows_cases: half a step of the result's type for its rounding, 2^-23 of the summed magnitudes per fp32 addition."""
import pytest
import torch

from rows_cases import SUM, TYPES, activated, plain_linear, plain_order, rounding, within

pytestmark = pytest.mark.gpu

HALVES = [torch.float16, torch.bfloat16]


def generator(seed):
    return torch.Generator(device='cuda').manual_seed(seed)


def normal(g, *shape, dtype=torch.float32, std=1.0):
    return (torch.randn(shape, generator=g, device='cuda') * std).to(dtype)


# ---------------------------------------------------------------- order
SORTS = [(0, 1, 4), (1, 1, 1), (31, 1, 3), (4096, 1, 5), (4097, 1, 5), (257, 3, 64), (1000, 8, 1023), (3000, 2, 1024),
         (20000, 1, 1), (12345, 2, 200), (9000, 1, 70000), (5, 1, 70000), (50000, 1, (1 << 20) + 3),
         (16384, 1, 511), (16385, 1, 512), (8192, 2, 1 << 19), (4096, 1, 300), (70000, 1, 5), (262144, 1, 700),
         (262145, 1, 40), (300001, 1, 1500), (1100000, 1, 16)]


@pytest.mark.parametrize('rows, choices, bins', SORTS)
@pytest.mark.parametrize('dtype', [torch.int32, torch.int64])
def test_sort_rows(cuda, rows, choices, bins, dtype):
    from odie_b200.experts import sort_rows
    g = generator(rows + bins)
    # skewed keys, some of them outside on both sides
    keys = (torch.rand((rows, choices), generator=g, device=cuda) ** 2 * (bins + 2)).floor().to(dtype) - 1
    if rows > 2 and dtype == torch.int64:
        keys[1] = 1 << 40
        keys[2] = -(1 << 40)
    order = sort_rows(keys, bins)
    want = plain_order(keys.cpu(), bins)
    for got, w, name in zip(order, want, ('order', 'slot', 'offsets')):
        assert torch.equal(got.cpu().long(), w.long()), name
    strided = torch.stack([keys, keys + 1], -1)[..., 0]  # every other element
    again = sort_rows(strided, bins)
    assert all(torch.equal(a, b) for a, b in zip(order, again))


def test_sort_rows_all_dropped_and_all_equal(cuda):
    from odie_b200.experts import sort_rows
    for n in (100, 10000):
        order = sort_rows(torch.full((n,), -1, dtype=torch.int32, device=cuda), 7)
        assert (order.offsets == 0).all()
        assert torch.equal(order.order, ~torch.arange(n, dtype=torch.int32, device=cuda))
        assert torch.equal(order.slot.view(-1), ~torch.arange(n, dtype=torch.int32, device=cuda))
        order = sort_rows(torch.full((n,), 6, dtype=torch.int32, device=cuda), 7)
        assert torch.equal(order.order, torch.arange(n, dtype=torch.int32, device=cuda))
        assert order.offsets.tolist() == [0] * 7 + [n]


# ---------------------------------------------------------------- dispatch and combine
ROWS = [(1, 1, 1, 1), (3, 2, 2, 7), (33, 1, 4, 32), (100, 3, 7, 33), (257, 2, 64, 128), (65, 4, 16, 1030), (7, 5, 9, 4104),
        (2000, 8, 12, 24),
        # enough rows for a warp per several wide ones
        (16500, 1, 16, 520), (8300, 2, 16, 300), (16400, 1, 5, 131), (5600, 3, 6, 35), (4100, 4, 9, 100), (16384, 1, 3, 2048)]


@pytest.mark.parametrize('rows, choices, bins, width', ROWS)
@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('weighted', [False, True])
def test_dispatch_and_combine(cuda, rows, choices, bins, width, dtype, weighted):
    from odie_b200.experts import combine, dispatch, sort_rows
    g = generator(rows * 7 + width)
    expert = torch.randint(-1, bins, (rows, choices), generator=g, device=cuda, dtype=torch.int32)
    order = sort_rows(expert, bins)
    x, results = normal(g, rows, width, dtype=dtype).requires_grad_(), normal(g, rows * choices, width, dtype=dtype)
    live = int(order.offsets[-1])
    results[live:] = float('nan')  # behind the last group: never read
    results.requires_grad_()
    weights = None
    if weighted:
        weights = torch.rand((rows, choices), generator=g, device=cuda)
        weights[expert < 0] = float('nan')  # a dropped choice's weight is never read
        weights.requires_grad_()
    d_rows, d_out = normal(g, rows * choices, width, dtype=dtype), normal(g, rows, width, dtype=dtype)
    d_rows[live:] = float('nan')
    leaves = [x, results] + ([weights] if weighted else [])
    sent, out = dispatch(x, order, weights), combine(results, order, weights)
    first = torch.autograd.grad(sent, [x] + leaves[2:], d_rows, retain_graph=True)
    second = torch.autograd.grad(out, [results] + leaves[2:], d_out, retain_graph=True)

    pair = order.order[:live].long()
    t = pair // choices
    p = (weights.detach().double().view(-1)[pair] if weighted else torch.ones(live, dtype=torch.float64, device=cuda))[:, None]
    xd, yd, gd, od = x.detach().double(), results.detach().double()[:live], d_rows.double()[:live], d_out.double()

    def spread(values):  # [live] rows into [rows * choices], zero behind
        return torch.cat([values, torch.zeros((rows * choices - live, width), dtype=torch.float64, device=cuda)])

    def summed(values):
        return torch.zeros((rows, width), dtype=torch.float64, device=cuda).index_add_(0, t, values)

    def paired(values):  # one number per live pair into [rows, choices]
        full = torch.zeros(rows * choices, dtype=torch.float64, device=cuda)
        full[pair] = values
        return full.view(rows, choices)
    want = spread(p * xd[t])
    within(sent.detach(), want, (2.0 ** -24 * want.abs() if weighted else 0) + (rounding(want, dtype) if weighted else 0), 'dispatch')
    magnitude = choices * SUM
    for got, values, name in ((out.detach(), yd, 'combine'), (first[0], gd, 'd_x')):
        want = summed(p * values)
        bound = magnitude * summed(p * values.abs())
        within(got, want, bound + rounding(want.abs() + bound, dtype), name)
    want = spread(p * od[t])
    within(second[0], want, (2.0 ** -24 * want.abs() + rounding(want, dtype)) if weighted else 0 * want, 'd_results')
    if weighted:
        for got, a, b, name in ((first[1], xd[t], gd, 'dispatch d_weights'), (second[1], yd, od[t], 'combine d_weights')):
            within(got, paired((a * b).sum(1)), paired(width * SUM * (a * b).abs().sum(1)), name)
    # the same bits again
    assert torch.equal(sent, dispatch(x, order, weights)) and torch.equal(out, combine(results, order, weights))


def test_weights_of_other_types_and_shapes(cuda):
    from odie_b200.experts import combine, sort_rows
    g = generator(1)
    order = sort_rows(torch.randint(0, 4, (50,), generator=g, device=cuda), 4)
    y = normal(g, 50, 16, dtype=torch.bfloat16)
    weights = torch.rand(50, generator=g, device=cuda).to(torch.bfloat16).requires_grad_()
    out = combine(y, order, weights)
    (d,) = torch.autograd.grad(out, weights, torch.ones_like(out))
    assert d.shape == (50,) and d.dtype == torch.bfloat16
    want = y.double()[order.slot.view(-1).long()].sum(1)
    off = 16 * SUM * y.double()[order.slot.view(-1).long()].abs().sum(1)
    within(d, want, off + rounding(want.abs() + off, torch.bfloat16), 'bf16 weights')


def test_unaligned_and_strided_rows(cuda):
    """Rows that start off 16-byte boundaries, or are strided or transposed views."""
    from odie_b200.experts import combine, dispatch, sort_rows
    g = generator(2)
    order = sort_rows(torch.randint(0, 5, (40, 2), generator=g, device=cuda), 5)
    base = normal(g, 41 * 24 + 8, dtype=torch.float16)
    for x in (base[1:1 + 40 * 24].view(40, 24), base[2:2 + 40 * 24].view(40, 24), base[:40 * 24].view(24, 40).t(),
              base[:41 * 24].view(41, 24)[1:, ::2]):
        sent = dispatch(x, order)
        assert torch.equal(sent, x[order.order.long() // 2])
        assert torch.equal(combine(sent, order), (x.float() * 2).half())


# ---------------------------------------------------------------- linear
LINEARS = [(1, 1, 1), (1, 9000, 40), (2, 1024, 33), (4, 2050, 64), (3, 5001, 10), (16, 4096, 72), (100, 3000, 200), (40, 1100, 515), (1, 64, 128), (2, 7, 3), (3, 256, 260), (8, 136, 24), (17, 40, 1000), (5, 333, 515), (127, 64, 64),
           (128, 32, 64), (129, 256, 256), (300, 1000, 72), (1000, 72, 264), (257, 2048, 128), (640, 520, 776), (5000, 200, 48), (2500, 1030, 31),
           # up to 64 inputs and outputs: the layers that stay in registers
           (9, 8, 8), (200, 24, 32), (333, 64, 40), (3000, 40, 64), (5000, 64, 64), (1111, 32, 8)]


def linear_case(rows, inputs, outputs, dtype, activation, groups=None, seed=0, bias=True, residual=True):
    """Inputs of a case; whole numbers for ReLU, so that every sum is exact and none sits near its corner."""
    g = generator(seed + rows * 31 + inputs * 7 + outputs)
    lead = (groups,) if groups else ()

    def draw(*shape, std=1.0):
        if activation == 'relu':
            return torch.randint(-1, 2, shape, generator=g, device='cuda').to(dtype)
        return normal(g, *shape, dtype=dtype, std=std)
    return (draw(rows, inputs), draw(*lead, outputs, inputs, std=inputs ** -0.5), draw(*lead, outputs) if bias else None,
            draw(rows, outputs) if residual else None, draw(rows, outputs))


def check_linear(case, activation, edges=None, offsets=None):
    from odie_b200.experts import linear
    x, weight, bias, residual, d_y = case
    names = [n for n, t in zip(('x', 'weight', 'bias', 'residual'), case) if t is not None]
    leaves = [t.requires_grad_() for t in case[:4] if t is not None]
    y = linear(x, weight, bias, residual, activation, offsets)
    grads = torch.autograd.grad(y, leaves, d_y)
    plain = plain_linear(*(None if t is None else t.detach() for t in case[:4]), edges or [(0, x.shape[0])], activation, d_y)
    within(y.detach(), *plain['y'], 'y')
    for name, got in zip(names, grads):
        assert got.dtype == x.dtype
        within(got, *plain['d_' + name], 'd_' + name)
    with torch.no_grad():  # the path without gradients gives the same bits
        assert torch.equal(y, linear(x, weight, bias, residual, activation, offsets))
    return y, grads


@pytest.mark.parametrize('rows, inputs, outputs', LINEARS)
@pytest.mark.parametrize('dtype', HALVES)
@pytest.mark.parametrize('activation', ['none', 'relu', 'silu', 'gelu'])
def test_linear(cuda, rows, inputs, outputs, dtype, activation):
    plain = activation == 'none'  # without an activation: once with and once without bias and residual
    check_linear(linear_case(rows, inputs, outputs, dtype, activation), activation)
    if plain:
        check_linear(linear_case(rows, inputs, outputs, dtype, activation, bias=False, residual=False), activation)


GROUPS = [[0], [1], [5, 0, 3], [127, 128, 129], [0, 0, 300], [64, 1, 0, 63, 200], [1] * 33, [700, 2, 0, 130]]


@pytest.mark.parametrize('sizes', GROUPS)
@pytest.mark.parametrize('inputs, outputs', [(64, 128), (96, 40), (37, 21), (264, 520), (32, 64), (64, 40)])
@pytest.mark.parametrize('dtype, activation', [(torch.float16, 'relu'), (torch.bfloat16, 'gelu'), (torch.bfloat16, 'none')])
@pytest.mark.parametrize('tail', [0, 19])
def test_linear_groups(cuda, sizes, inputs, outputs, dtype, activation, tail):
    rows = sum(sizes) + tail
    if rows == 0:
        rows, tail = 3, 3
    case = linear_case(rows, inputs, outputs, dtype, activation, groups=len(sizes))
    offsets = torch.tensor([0] + sizes, device=cuda).cumsum(0).to(torch.int32)
    edges = [(int(a), int(b)) for a, b in zip(offsets[:-1], offsets[1:])]
    check_linear(case, activation, edges, offsets)


@pytest.mark.parametrize('inputs, outputs', [(72, 136), (32, 64), (33, 70)])
@pytest.mark.parametrize('poison', [float('nan'), float('inf')])
def test_linear_groups_keep_apart(cuda, poison, inputs, outputs):
    """NaN or infinity in one group's rows and weights, or behind the last group, reaches nothing of the others."""
    from odie_b200.experts import linear
    g = generator(5)
    sizes = [70, 50, 0, 90]
    offsets = torch.tensor([0] + sizes, device=cuda).cumsum(0).to(torch.int32)
    rows = sum(sizes) + 11
    x, w, b = normal(g, rows, inputs).half(), normal(g, 4, outputs, inputs, std=0.1).half(), normal(g, 4, outputs).half()
    d_y = normal(g, rows, outputs).half()
    clean = [t.clone() for t in (x, w, b, d_y)]
    x[70:120], d_y[70:120], x[210:], d_y[210:] = poison, poison, poison, poison
    w[2], b[2] = poison, poison  # the empty group's
    results = []
    for x_, w_, b_, d_ in ((x, w, b, d_y), clean):
        leaves = [t.requires_grad_() for t in (x_, w_, b_)]
        y = linear(x_, w_, b_, activation='gelu', offsets=offsets)
        results.append([y.detach(), *torch.autograd.grad(y, leaves, d_)])
    (y, dx, dw, db), (y0, dx0, dw0, db0) = results
    for got, want in ((y, y0), (dx, dx0)):
        assert torch.equal(got[:70], want[:70]) and torch.equal(got[120:210], want[120:210])
        assert (got[210:] == 0).all()
    for got, want in ((dw, dw0), (db, db0)):
        assert torch.equal(got[[0, 3]], want[[0, 3]]) and (got[2] == 0).all() and (want[2] == 0).all()
    assert not torch.isfinite(dw[1]).all()


def test_linear_infinities_and_nan_pass_through(cuda):
    """Infinite and NaN sums give what the activation gives, in the rows that hold them."""
    from odie_b200.experts import linear
    w = torch.eye(64, device=cuda).half()
    x = torch.zeros(130, 64, device=cuda).half()
    x[3, 5], x[4, 6] = float('inf'), float('nan')
    for activation in ('none', 'relu'):
        y = linear(x, w, activation=activation)
        # inf times the zeros of other columns is NaN in this row, as in any product
        assert y[3].isnan().sum() == 63 and y[3, 5] == float('inf') and y[4].isnan().all()
        rest = torch.cat([y[:3], y[5:]])
        assert (rest == 0).all()
    xs = x.clone()[4:5].requires_grad_()
    (d,) = torch.autograd.grad(linear(xs, w, activation='silu'), xs, torch.ones(1, 64, device=cuda).half())
    assert d.isnan().all()  # the kept slope holds NaN


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


@pytest.mark.parametrize('rows, inputs, outputs', [(1, 64, 128), (2, 5000, 33), (2, 40, 21), (17, 40, 72), (5, 333, 35), (40, 2048, 24), (300, 72, 264),
                                                   (3, 24, 32), (333, 64, 40), (200, 24, 8)])
@pytest.mark.parametrize('residual', [False, True])
def test_linear_relu_of_sums_too_small_for_y(cuda, rows, inputs, outputs, residual):
    """A ReLU is on where its fp32 sum is above zero, also where y holds 0 for it, or a residual hides it."""
    g = generator(rows + inputs + outputs)
    signs = torch.randint(-1, 2, (outputs, inputs), generator=g, device=cuda)
    signs[:, 0] += signs[:, 0] == 0  # (no row of W is zero)
    at = torch.randint(inputs, (rows,), generator=g, device=cuda)
    x = torch.zeros(rows, inputs, device=cuda, dtype=torch.float16)
    x[torch.arange(rows, device=cuda), at] = 2 ** -13
    r = normal(g, rows, outputs).half() if residual else None
    found = passing(x, signs * torch.tensor(2 ** -13, device=cuda, dtype=torch.float16), residual=r)  # sums of 2^-26, 0 and -2^-26
    assert torch.equal(found, signs.t()[at] > 0)


@pytest.mark.parametrize('rows, inputs, outputs', [(2000, 32, 64), (333, 64, 40), (500, 24, 8), (1, 32, 16), (900, 64, 64), (2, 64, 64)])
@pytest.mark.parametrize('dtype', HALVES)
def test_thin_relu_at_its_corner(cuda, rows, inputs, outputs, dtype):
    """Sums that cancel to the last bits: a layer of up to 64 inputs and outputs is on where the fp32 chain in ascending
    order of the inputs is above zero.  (The products of 16-bit values are exact in fp32, so a rounded product and sum
    are the fused step.)"""
    g = generator(rows + inputs)
    x, w = normal(g, rows, inputs, dtype=dtype), normal(g, outputs, inputs, std=0.3, dtype=dtype)
    for level in range(3):  # the last inputs cancel the sum of output 0 to 2^-24 of it
        k = inputs - 3 + level
        w[0, k] = 2.0 ** (-8 * level)
        x[:, k] = (-(x[:, :k].double() @ w[0, :k].double()) * 2.0 ** (8 * level)).to(dtype)
    chain = torch.zeros(rows, outputs, device=cuda)
    for k in range(inputs):
        chain = chain + x[:, k:k + 1].float() * w[:, k].float()
    assert torch.equal(passing(x, w), chain > 0)


@pytest.mark.parametrize('rows, inputs, outputs', [(1, 64, 16), (20, 72, 16), (20, 32, 16)])
def test_linear_relu_passes_gradients_of_nan(cuda, rows, inputs, outputs):
    """A NaN sum is not <= 0: its gradient passes, as torch.relu's does."""
    g = generator(rows)
    x, w = normal(g, rows, inputs).half(), normal(g, outputs, inputs).half()
    x[0, 3] = float('nan')
    found = passing(x, w)
    assert found[0].all() and torch.equal(found[1:], x[1:].double() @ w.double().t() > 0)


@pytest.mark.parametrize('rows, inputs, outputs', [(2, 40, 21), (2, 5000, 9), (300, 72, 264), (130, 64, 67), (40, 2048, 35), (333, 64, 40), (333, 32, 64)])
@pytest.mark.parametrize('shift', [0, 1])
def test_linear_relu_bits(cuda, rows, inputs, outputs, shift):
    """The C interface's slope of a ReLU: bit c % 8 of byte c / 8, at any address, read back by the gradient; nothing is
    written around it, nor anything without an activation.  Whole numbers, so that every sum is exact."""
    from odie_b200 import _lib
    lib = _lib.library()
    g = generator(rows + outputs)
    x = torch.randint(-2, 3, (rows, inputs), generator=g, device=cuda).half()
    w = torch.randint(-2, 3, (outputs, inputs), generator=g, device=cuda).half()
    z = x.double() @ w.double().t()
    pitch = (outputs + 7) // 8
    buffer = torch.full((rows * pitch + 16,), 0xa5, dtype=torch.uint8, device=cuda)
    y, d_x = torch.empty(rows, outputs, device=cuda).half(), torch.empty_like(x)
    sizes = (rows, inputs, outputs, 1)
    scratch = torch.empty(max(1, lib.odie_linear_scratch(*sizes), lib.odie_linear_backward_scratch(*sizes)), dtype=torch.uint8, device=cuda)
    stream = torch.cuda.current_stream().cuda_stream
    slope = buffer.data_ptr() + 8 + shift
    for activation in (0, 1):
        assert lib.odie_linear(x.data_ptr(), w.data_ptr(), None, None, *sizes, None, 0, activation, y.data_ptr(), slope, scratch.data_ptr(), stream) == 0
        if activation == 0:
            assert (buffer == 0xa5).all()
    bits = buffer[8 + shift:8 + shift + rows * pitch].view(rows, pitch, 1) >> torch.arange(8, device=cuda, dtype=torch.uint8) & 1
    assert torch.equal(bits.view(rows, pitch * 8)[:, :outputs].bool(), z > 0)
    assert (buffer[:8 + shift] == 0xa5).all() and (buffer[8 + shift + rows * pitch:] == 0xa5).all()
    d_y = torch.randint(-2, 3, (rows, outputs), generator=g, device=cuda).half()
    assert lib.odie_linear_backward(d_y.data_ptr(), slope, 1, x.data_ptr(), w.data_ptr(), *sizes, None, 0, d_x.data_ptr(), None, None, None,
                                    scratch.data_ptr(), stream) == 0
    want = (d_y.double() * (z > 0)) @ w.double()
    within(d_x, want, rounding(want, torch.float16), 'd_x')


def test_linear_shapes_and_strides(cuda):
    """Leading dimensions, no rows, transposed and misaligned operands, broadcast residual, expanded gradients."""
    from odie_b200.experts import linear
    g = generator(9)
    x = normal(g, 3, 5, 48).half()
    w, r = normal(g, 40, 48, std=0.2).half(), normal(g, 40).half()
    flat = x.reshape(15, 48)
    want = linear(flat, w, residual=r.expand(15, 40).contiguous())
    assert torch.equal(linear(x, w, residual=r), want.view(3, 5, 40))
    assert linear(x[:0], w).shape == (0, 5, 40)
    assert linear(x[0, 0], w).shape == (40,)
    assert torch.equal(linear(x.transpose(0, 1), w, residual=r), want.view(3, 5, 40).transpose(0, 1))
    assert torch.equal(linear(flat, w.t().contiguous().t(), residual=r), want)
    odd = torch.empty(15 * 48 + 1, device=cuda, dtype=torch.float16)[1:].view(15, 48)
    odd.copy_(flat)
    assert torch.equal(linear(odd, w, residual=r), want)
    w_odd = torch.empty(40 * 48 + 1, device=cuda, dtype=torch.float16)[1:].view(40, 48).copy_(w)
    assert torch.equal(linear(flat, w_odd, residual=r), want)
    # a broadcast gradient and a broadcast residual's gradient
    xs, rs, ws = flat.clone().requires_grad_(), r.clone().requires_grad_(), w.clone().requires_grad_()
    dx, dr, dw = torch.autograd.grad(linear(xs, ws, residual=rs).sum(), [xs, rs, ws])
    assert torch.equal(dr, torch.full_like(r, 15.0))
    ones = torch.ones(15, 40, device=cuda, dtype=torch.float16)
    within(dx, ones.double() @ w.double(), 41 * SUM * (ones.double() @ w.double().abs()) +
           rounding(1.001 * (ones.double() @ w.double().abs()), torch.float16), 'd_x of a sum')
    # no rows: zero gradients
    xe = flat[:0].clone().requires_grad_()
    be = normal(g, 40).half().requires_grad_()
    y = linear(xe, ws, be, activation='silu')
    d = torch.autograd.grad(y, [xe, ws, be], torch.empty_like(y))
    assert d[0].shape == (0, 48) and (d[1] == 0).all() and (d[2] == 0).all()


@pytest.mark.parametrize('activation', ['silu', 'gelu'])
def test_linear_gradient_against_differences(cuda, activation):
    """The kernel's gradient along random directions against central differences of the 64-bit formula."""
    case = linear_case(33, 40, 24, torch.bfloat16, activation)
    x, weight, bias, residual, d_y = case
    _, grads = check_linear(case, activation)
    plain = plain_linear(*(t.detach() for t in case[:4]), [(0, 33)], activation, d_y)
    p = [t.detach().double() for t in case[:4]]
    g = generator(77)
    along = [torch.randn(t.shape, generator=g, device=cuda, dtype=torch.float64) for t in p]
    h = 1e-5

    def value(step):
        a, b, c, r = (t + step * d for t, d in zip(p, along))
        return ((activated(a @ b.t() + c, activation)[0] + r) * d_y.double()).sum().item()
    slope = (value(h) - value(-h)) / (2 * h)
    got = sum((gr.double() * d).sum().item() for gr, d in zip(grads, along))
    bounds = [plain['d_' + n][1] for n in ('x', 'weight', 'bias', 'residual')]
    allowed = sum((b * d.abs()).sum().item() for b, d in zip(bounds, along)) + 1e-6 * abs(slope) + 1e-6
    assert abs(got - slope) <= allowed


@pytest.mark.parametrize('rows, inputs, outputs', [(40, 32, 64), (40, 64, 128), (5, 64, 64)])
@pytest.mark.parametrize('wanted', ['x', 'weight', 'bias', 'residual'])
def test_linear_single_gradients(cuda, rows, inputs, outputs, wanted):
    """Each gradient by itself, the others not asked for, has the bits of the whole backward pass."""
    from odie_b200.experts import linear
    case = linear_case(rows, inputs, outputs, torch.bfloat16, 'silu')
    offsets = torch.tensor([0, rows - 3], dtype=torch.int32, device=cuda)
    for grouped in (False, True):
        named = dict(zip(('x', 'weight', 'bias', 'residual'), (t.detach() for t in case[:4])))
        if grouped:
            named.update(weight=named['weight'][None], bias=named['bias'][None])
        more = dict(activation='silu', offsets=offsets if grouped else None)
        every = {k: v.clone().requires_grad_() for k, v in named.items()}
        want = torch.autograd.grad(linear(**every, **more), every[wanted], case[4])[0]
        one = {k: v.clone().requires_grad_(k == wanted) for k, v in named.items()}
        got = torch.autograd.grad(linear(**one, **more), one[wanted], case[4])[0]
        assert torch.equal(got, want)


def test_linear_waits_never_run_out(cuda):
    import odie_b200._lib as _lib
    status = torch.full((1,), -1, dtype=torch.int32, device=cuda)
    check_linear(linear_case(700, 520, 776, torch.bfloat16, 'gelu'), 'gelu')
    _lib.check(_lib.library().odie_linear_status(status.data_ptr(), _lib.stream_handle()), 'odie_linear_status')
    assert status.item() == 0


def test_linear_refusals(cuda):
    from odie_b200.experts import linear
    x, w = torch.zeros(4, 8, device=cuda).half(), torch.zeros(16, 8, device=cuda).half()
    off = torch.zeros(3, dtype=torch.int32, device=cuda)
    wg = torch.zeros(2, 16, 8, device=cuda).half()
    for bad in (dict(x=x.float()), dict(weight=w.bfloat16()), dict(weight=w[:, :7]), dict(weight=w[:0]), dict(bias=w[0]),
                dict(residual=torch.zeros(4, 16, device=cuda)), dict(activation='tanh'), dict(weight=wg),
                dict(weight=wg, offsets=off[:2]), dict(weight=wg, offsets=off.long()), dict(weight=wg, offsets=off.cpu()),
                dict(weight=w.cpu()), dict(x=x[None], weight=wg, offsets=off), dict(x=x[:, :0], weight=w[:, :0])):
        with pytest.raises(ValueError):
            linear(**{**dict(x=x, weight=w), **bad})
    wide = x[:1, :1].expand(1, (1 << 32) + 8)  # 8 in 32 bits
    for bad in (dict(x=wide, weight=wide), dict(weight=w[:1].expand((1 << 20) + 1, 8))):
        with pytest.raises(ValueError, match='2\\^20'):
            linear(**{**dict(x=x), **bad})
    with pytest.raises(RuntimeError):  # not broadcastable
        linear(x, w, residual=torch.zeros(3, 16, device=cuda).half())


def test_linear_offsets_out_of_range_stay_inside(cuda):
    """Offsets past the rows, or negative, are cut to them: nothing out of range is read or written."""
    from odie_b200.experts import linear
    g = generator(3)
    x, w = normal(g, 100, 64).half(), normal(g, 2, 64, 64).half()
    got = linear(x, w, offsets=torch.tensor([0, 60, 1000], dtype=torch.int32, device=cuda))
    assert torch.equal(got, linear(x, w, offsets=torch.tensor([0, 60, 100], dtype=torch.int32, device=cuda)))
    got = linear(x, w, offsets=torch.tensor([-5, -3, 40], dtype=torch.int32, device=cuda))
    assert torch.equal(got, linear(x, w, offsets=torch.tensor([0, 0, 40], dtype=torch.int32, device=cuda)))


@pytest.mark.parametrize('inputs, outputs', [(64, 64), (136, 72)])
def test_linear_offsets_running_backwards_stay_inside(cuda, inputs, outputs):
    """Offsets that run backwards make groups overlap, and more units of work than there is room for: what the results
    are is open, but the gradients' neighbours in memory keep their values and later calls work."""
    from odie_b200.experts import linear
    g = generator(6)
    rows = 6000
    x, w, b = (normal(g, *s).half().requires_grad_() for s in ((rows, inputs), (6, outputs, inputs), (6, outputs)))
    d = normal(g, rows, outputs).half()
    good = torch.arange(0, 7, dtype=torch.int32, device=cuda) * 1000
    bad = torch.tensor([0, 6000, 0, 6000, 10, 5990, 0], dtype=torch.int32, device=cuda)
    want = torch.autograd.grad(linear(x, w, b, activation='silu', offsets=good), [x, w, b], d)
    guards = [torch.full((1 << 20,), 7.0, device=cuda) for _ in range(8)]
    torch.autograd.grad(linear(x, w, b, activation='silu', offsets=bad), [x, w, b], d)
    torch.cuda.synchronize()
    assert all((t == 7.0).all() for t in guards)
    again = torch.autograd.grad(linear(x, w, b, activation='silu', offsets=good), [x, w, b], d)
    assert all(torch.equal(a, e) for a, e in zip(want, again))


# ---------------------------------------------------------------- embed
EMBEDS = [(1, 1, 1), (5, 3, 7), (64, 1, 32), (300, 2, 33), (129, 1000, 128), (4096, 50, 24), (5000, 5000, 16), (70000, 3, 8),
          (1000, 70000, 40), (200, 17, 2056), (20000, (1 << 20) + 5, 1),
          (16500, 3000, 130), (16384, 100, 520), (16384, 100, 257)]


@pytest.mark.parametrize('count, rows, width', EMBEDS)
@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('id_type', [torch.int32, torch.int64])
def test_embed(cuda, count, rows, width, dtype, id_type):
    from odie_b200.experts import embed
    g = generator(count + rows + width)
    ids = (torch.rand(count, generator=g, device=cuda, dtype=torch.float64) ** 3 * (rows + 2)).long() - 1
    ids[::7] = rows // 2
    ids = ids.to(id_type)
    table, d_out = normal(g, rows, width, dtype=dtype), normal(g, count, width, dtype=dtype)
    scale = 1.25
    live = (ids >= 0) & (ids < rows)
    d_out[~live] = float('nan')  # positions of ids outside the table are not read
    table.requires_grad_()
    out = embed(ids, table, scale)
    (grad,) = torch.autograd.grad(out, table, d_out, retain_graph=True)
    safe = ids.long().clamp(0, rows - 1)
    want = scale * table.detach().double()[safe] * live.double()[:, None]
    within(out.detach(), want, 2.0 ** -24 * want.abs() + rounding(want, dtype), 'embed')
    d = torch.where(live[:, None], d_out, torch.zeros_like(d_out)).double() * scale
    zero = torch.zeros((rows, width), dtype=torch.float64, device=cuda)
    want, size = zero.index_add(0, safe, d), zero.index_add(0, safe, d.abs())
    counts = torch.zeros(rows, dtype=torch.float64, device=cuda).index_add_(0, safe, live.double())
    bound = (counts[:, None] + 1) * SUM * size
    within(grad, want, bound + rounding(want.abs() + bound, dtype), 'd_table')
    assert (grad[counts == 0] == 0).all()
    assert torch.equal(grad, torch.autograd.grad(out, table, d_out)[0])  # the same bits again


@pytest.mark.parametrize('count', [63, 64, 65, 128, 4097, 40000])
def test_embed_one_id_takes_all(cuda, count):
    """One run over every chunk, beside runs that end on and around chunk borders."""
    from odie_b200.experts import embed
    ids = torch.full((count,), 3, device=cuda)
    ids[:count // 2:2] = 1
    table = torch.zeros(5, 12, device=cuda, requires_grad=True)
    ones = torch.ones(count, 12, device=cuda)
    (grad,) = torch.autograd.grad(embed(ids, table), table, ones)
    want = torch.bincount(ids, minlength=5).float()[:, None].expand(5, 12)  # whole numbers: exact
    assert torch.equal(grad, want)


def test_embed_shapes_and_empty(cuda):
    from odie_b200.experts import embed
    table = torch.randn(9, 6, device=cuda, requires_grad=True)
    ids = torch.tensor([[0, 8, 9], [-1, 4, 4]], device=cuda)
    out = embed(ids, table)
    assert out.shape == (2, 3, 6) and (out[0, 2] == 0).all() and torch.equal(out[1, 1], table[4])
    (grad,) = torch.autograd.grad(out.sum(), table)  # an expanded gradient
    assert torch.equal(grad[4], torch.full((6,), 2.0, device=cuda)) and (grad[1] == 0).all()
    none = embed(ids[:0], table)
    assert none.shape == (0, 3, 6)
    (grad,) = torch.autograd.grad(none, table, torch.empty_like(none))
    assert (grad == 0).all()
    strided = embed(ids.t(), table)
    assert torch.equal(strided, out.transpose(0, 1))
    for bad in (dict(ids=ids.float()), dict(ids=ids.to(torch.int16)), dict(ids=ids.cpu()), dict(table=table[0]),
                dict(table=table.double()), dict(table=table[:0]), dict(table=table[:, :0])):
        with pytest.raises(ValueError):
            embed(**{**dict(ids=ids, table=table), **bad})


def test_no_rows(cuda):
    from odie_b200.experts import combine, dispatch, sort_rows
    order = sort_rows(torch.empty((0, 2), dtype=torch.int32, device=cuda), 4)
    x = torch.empty((0, 8), device=cuda, requires_grad=True)
    weights = torch.empty((0, 2), device=cuda, requires_grad=True)
    sent = dispatch(x, order, weights)
    out = combine(sent, order, weights)
    assert sent.shape == (0, 8) and out.shape == (0, 8)
    d = torch.autograd.grad(out, [x, weights], torch.empty_like(out))
    assert d[0].shape == (0, 8) and d[1].shape == (0, 2)


def test_gradients_are_differentiable_once(cuda):
    """create_graph gives the same gradients; differentiating them again is an error, not a silent zero."""
    from odie_b200.experts import combine, dispatch, embed, linear, sort_rows
    g = generator(1)
    x, w = normal(g, 30, 16).half().requires_grad_(), normal(g, 16, 16).half().requires_grad_()
    table = normal(g, 5, 16).requires_grad_()
    order = sort_rows(torch.randint(0, 3, (30,), generator=g, device=cuda), 3)
    ids = torch.randint(0, 5, (30,), generator=g, device=cuda)
    for f, leaf in ((lambda: linear(x, w, activation='silu'), x), (lambda: dispatch(x, order), x),
                    (lambda: combine(x, order), x), (lambda: embed(ids, table), table)):
        y = f()
        d = torch.ones_like(y, requires_grad=True)
        (plain,) = torch.autograd.grad(y, leaf, torch.ones_like(y), retain_graph=True)
        (graph,) = torch.autograd.grad(y, leaf, d, create_graph=True)
        assert torch.equal(plain, graph)
        with pytest.raises(RuntimeError, match='once'):
            torch.autograd.grad(graph.sum(), d)


def test_leaves_of_modules_accumulate(cuda):
    """backward() twice accumulates into .grad, also through shared weights."""
    from odie_b200.experts import linear
    g = generator(4)
    x, w = normal(g, 20, 32).half(), normal(g, 32, 32, std=0.1).half().requires_grad_()
    y = linear(linear(x, w, activation='gelu'), w)
    d = normal(g, 20, 32).half()
    (once,) = torch.autograd.grad(y, w, d, retain_graph=True)
    y.backward(d, retain_graph=True)
    y.backward(d)
    assert torch.equal(w.grad, once + once)


def test_order_refusals(cuda):
    from odie_b200.experts import combine, dispatch, sort_rows
    ids = torch.zeros(6, 2, dtype=torch.int32, device=cuda)
    for bad in (dict(expert=ids.float()), dict(expert=ids[None]), dict(bins=0), dict(bins=1 << 30), dict(expert=ids[:, :0])):
        with pytest.raises(ValueError):
            sort_rows(**{**dict(expert=ids, bins=4), **bad})
    order = sort_rows(ids, 4)
    x = torch.zeros(6, 8, device=cuda)
    for call in (lambda: dispatch(x[:5], order), lambda: combine(x, order), lambda: dispatch(x.double(), order),
                 lambda: dispatch(x, tuple(order)), lambda: dispatch(x, order, x), lambda: dispatch(x, order, ids),
                 lambda: dispatch(x[:, :0], order)):
        with pytest.raises(ValueError):
            call()


# ---------------------------------------------------------------- together
def expert_mlp_reference(features, heads, expert, weights, ids):
    """ExpertHeads in 64 bits from its masters, expert by expert."""
    h0 = features.double()
    if ids is not None:
        h0 = h0 + heads.codes.double()[ids]
    out = 0
    for j in range(expert.shape[1]):
        per = torch.zeros((features.shape[0], heads.weights[-1].shape[1]), dtype=torch.float64, device=features.device)
        for e in range(heads.experts):
            rows = (expert[:, j] == e).nonzero().view(-1)
            h = h0[rows]
            for i, (w, b) in enumerate(zip(heads.weights, heads.biases)):
                h = h @ w[e].double().t() + b[e].double()
                h = h.clamp(min=0) if i + 1 < len(heads.weights) else h
            per = per.index_copy(0, rows, h)
        out = out + per * weights[:, j:j + 1].double()
    return out


@pytest.mark.parametrize('rows, choices, experts', [(1, 1, 4), (777, 1, 16), (500, 2, 8)])
def test_expert_heads_run_and_gradients(cuda, rows, choices, experts):
    """embed -> sort -> dispatch -> linear x 3 -> combine, and back, against the 64-bit model.

    Every layer rounds to fp16 (eps 2^-10): weights, inputs and results are each off by half a step, 2^-11, so a
    layer adds at most 3 x 2^-11 of its magnitude to the relative error; three layers, the code and the weighted
    sum stay within 12 x 2^-11 of the magnitudes' norms, and the backward pass as much again.  ReLU corners that
    the rounding moves (|z| below it) change single terms by no more than the rounding itself forward; backward
    they drop or add whole terms for a share of about 2^-9 of the units, a relative norm of 2^-4.5 at most."""
    from odie_b200.experts import ExpertHeads
    g = generator(rows)
    heads = ExpertHeads(32, 3, 64, 2, experts, seed=4, codes=10)
    with torch.no_grad():
        heads.codes.normal_(0, 0.5, generator=g)
        for b in heads.biases:
            b.normal_(0, 0.2, generator=g)
    features = normal(g, rows, 32).half().requires_grad_()
    expert = torch.randint(0, experts, (rows, choices), generator=g, device=cuda, dtype=torch.int32)
    expert[rows // 2:, -1] = -1 if choices > 1 else expert[rows // 2:, -1]
    weights = torch.rand((rows, choices), generator=g, device=cuda).requires_grad_()
    ids = torch.randint(0, 10, (rows,), generator=g, device=cuda)
    out = heads(features, expert, weights, ids)
    assert out.dtype == torch.float16 and out.shape == (rows, 3)
    want = expert_mlp_reference(features, heads, expert, weights, ids)
    assert (out.double() - want).norm() <= 12 * 2 ** -11 * want.norm()
    d = normal(g, rows, 3).half()
    leaves = [features, weights, *heads.parameters()]
    got, plain = torch.autograd.grad(out, leaves, d), torch.autograd.grad(want, leaves, d.double())
    for a, b in zip(got, plain):
        assert a.dtype == b.dtype and torch.isfinite(a).all()
        assert (a.double() - b.double()).norm() <= (2 ** -4.5 + 24 * 2 ** -11) * b.double().norm()


def test_routed_model_features_through_expert_heads(cuda):
    """The routed model's own routing and expert features, decoded by the experts' own heads instead of the shared one."""
    from odie_b200.experts import ExpertHeads
    from odie_b200.model import ExpertHashQuery, RoutedExperts
    from odie_b200.workloads import experts_config
    config = experts_config(experts=4, seed=5, batch=512,
                            encoding=dict(n_levels=16, n_features_per_level=2, log2_hashmap_size=9, base_resolution=4,
                                          per_level_scale=1.4),
                            router_encoding=dict(n_levels=16, n_features_per_level=2, log2_hashmap_size=7,
                                                 base_resolution=2, per_level_scale=1.2))
    config.update(grid_init=0.5, router_init=0.5)
    model = RoutedExperts(config)
    xy = torch.rand(1000, 2, generator=generator(1), device=cuda)
    expert, prob, _ = model.route(xy)
    features = ExpertHashQuery.apply(xy, model.grid, expert, model.expert_total, model.records, model.input_width)
    heads = ExpertHeads(32, 3, 64, 2, 4, seed=1)
    rgb = heads(features, expert, prob)
    rgb.float().square().mean().backward()
    want = expert_mlp_reference(features.detach(), heads, expert[:, None], prob[:, None], None)
    assert (rgb.double() - want).norm() <= 12 * 2 ** -11 * want.norm()
    for p in [model.grid, *heads.weights, *heads.biases]:
        assert p.grad is not None and torch.isfinite(p.grad).all() and p.grad.abs().sum() > 0


def everything(x, weight, bias, expert, weights, table, ids):
    from odie_b200.experts import combine, dispatch, embed, linear, sort_rows
    order = sort_rows(expert, weight.shape[0])
    h = linear(dispatch(x + embed(ids, table), order), weight, bias, activation='silu', offsets=order.offsets)
    return combine(h, order, weights)


def everything_inputs(seed, rows=300):
    g = generator(seed)
    leaves = [normal(g, rows, 64, dtype=torch.bfloat16), normal(g, 6, 64, 64, dtype=torch.bfloat16, std=0.1),
              normal(g, 6, 64, dtype=torch.bfloat16), torch.rand((rows, 2), generator=g, device='cuda'),
              normal(g, 40, 64, dtype=torch.bfloat16)]
    expert = torch.randint(-1, 6, (rows, 2), generator=g, device='cuda', dtype=torch.int32)
    ids = torch.randint(0, 40, (rows,), generator=g, device='cuda')
    return [t.requires_grad_() for t in leaves], expert, ids, normal(g, rows, 64, dtype=torch.bfloat16)


def pass_of(leaves, expert, ids, d):
    x, w, b, p, table = leaves
    out = everything(x, w, b, expert, p, table, ids)
    return [out.detach(), *torch.autograd.grad(out, leaves, d)]


def test_captured_and_replayed(cuda):
    """Forward and backward captured into a CUDA graph and replayed on new inputs, beside eager calls."""
    leaves, expert, ids, d = everything_inputs(1)
    other, expert2, ids2, d2 = everything_inputs(2)
    want = [pass_of(leaves, expert, ids, d), pass_of(other, expert2, ids2, d2)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        pass_of(leaves, expert, ids, d)
    torch.cuda.current_stream().wait_stream(side)
    graphs, results = [], []
    for _ in range(2):  # two graphs of the same leaves
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            results.append(pass_of(leaves, expert, ids, d))
        graphs.append(graph)
    for graph, result in zip(graphs, results):
        graph.replay()
        eager = pass_of(leaves, expert, ids, d)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(result, want[0]))
        assert all(torch.equal(a, b) for a, b in zip(eager, want[0]))
    with torch.no_grad():
        for a, b in zip([*leaves, expert, ids, d], [*other, expert2, ids2, d2]):
            a.copy_(b)
    for graph, result in zip(graphs, results):
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(result, want[1]))


def test_two_streams_at_once(cuda):
    """Calls in flight on two streams share nothing."""
    cases = [everything_inputs(s, rows) for s, rows in ((3, 3000), (4, 5000))]
    want = [pass_of(*c) for c in cases]
    streams = [torch.cuda.Stream() for _ in cases]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(5):
        for i, (stream, c) in enumerate(zip(streams, cases)):
            with torch.cuda.stream(stream):
                got[i] = pass_of(*c)
    torch.cuda.synchronize()
    for g, w in zip(got, want):
        assert all(torch.equal(a, b) for a, b in zip(g, w))
