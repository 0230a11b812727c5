"""The router's operators and microscaled rows at the ends of what they take: more elements than 32 bits count, derivatives and
transforms of other kinds, values that are no numbers, offsets that run backwards, tensors of other threads' streams."""
import pytest
import torch

from router_cases import plain_gate, plain_micro
from rows_cases import within

pytestmark = pytest.mark.gpu


def generator(seed):
    return torch.Generator(device='cuda').manual_seed(seed)


# ---------------------------------------------------------------- more than 2^31 elements
def test_gate_and_balance_of_many_rows(cuda):
    """2^31 + 2^21 logits: the last rows are those of a call of their own."""
    from odie_b200.experts import balance, gate
    rows, experts = (1 << 21) + (1 << 11), 1024
    logits = torch.empty((rows, experts), dtype=torch.float16, device='cuda').normal_(generator=generator(1))
    leaf = logits.requires_grad_()
    expert, weights = gate(leaf, 2, normalize=False)
    d_weights = torch.ones((rows, 2), device='cuda')
    (d,) = torch.autograd.grad(weights, leaf, d_weights)
    tail = slice(rows - 300, rows)
    own = leaf.detach()[tail].clone().requires_grad_()
    e, w = gate(own, 2, normalize=False)
    assert torch.equal(e, expert[tail]) and torch.equal(w, weights[tail])
    assert torch.equal(torch.autograd.grad(w, own, d_weights[tail])[0], d[tail])
    del d
    loss, z, counts = balance(leaf, expert)
    (d,) = torch.autograd.grad(loss, leaf, torch.tensor(float(rows), device='cuda'))
    assert counts.sum().item() == 2 * rows and 0.9 < loss.item() < 1.2  # (independent logits: near an even load)
    p = torch.softmax(own.detach().double(), 1)
    f = counts.double() / (2 * rows)
    want = experts * p * (f - p @ f[:, None])
    assert (d[tail].double() - want).norm() <= 2 ** -9 * want.norm()


def test_quantize_and_linear4_of_many_rows(cuda):
    """2^31 + 2^17 values, and as many results."""
    from odie_b200.experts import dequantize, linear4, quantize
    rows, width = (1 << 17) + 8, 1 << 14
    x = torch.empty((rows, width), dtype=torch.bfloat16, device='cuda').normal_(generator=generator(2))
    micro = quantize(x)
    tail = slice(rows - 130, rows)
    want = plain_micro(x[tail], 16)[0]
    y = dequantize(micro, torch.bfloat16)
    assert torch.equal(y[tail].double(), want)
    del y, micro
    weight = quantize(torch.empty((width, 64), device='cuda').normal_(generator=generator(3)))
    y = linear4(x[:, :64], weight)  # a strided view, one block of K
    own = linear4(x[tail, :64], weight)
    assert (y[tail].double() - own.double()).abs().max() <= 2 ** -8 * own.double().abs().max()
    assert torch.isfinite(y[0]).all() and y.shape == (rows, width)


# ---------------------------------------------------------------- derivatives of other kinds
def calls():
    from odie_b200.experts import balance, gate, linear4, quantize
    ids = torch.zeros((5, 2), dtype=torch.int32, device='cuda')
    weight = quantize(torch.randn((8, 6), device='cuda'))
    return {'gate': lambda x: gate(x, 2).weights, 'gate dense': lambda x: gate(x, 2, normalize=False).weights,
            'balance': lambda x: balance(x, ids).loss, 'quantize': lambda x: quantize(x).codes,
            'linear4': lambda x: linear4(x.half(), weight)}


@pytest.mark.parametrize('name', ['gate', 'gate dense', 'balance', 'quantize', 'linear4'])
def test_forward_mode_is_refused(cuda, name):
    from torch.autograd import forward_ad
    call, x = calls()[name], torch.randn((5, 6), device='cuda')
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(x, torch.ones_like(x))
        for grad in (torch.enable_grad, torch.no_grad):
            with grad(), pytest.raises(RuntimeError, match='forward-mode'):
                call(dual)
        if name not in ('quantize', 'linear4'):
            leaf = x.clone().requires_grad_()
            y = call(leaf)
            with pytest.raises(RuntimeError, match='forward-mode'):
                torch.autograd.grad(y, leaf, forward_ad.make_dual(torch.ones_like(y), torch.ones_like(y)))


@pytest.mark.parametrize('name', ['gate', 'gate dense', 'balance', 'quantize', 'linear4'])
def test_function_transforms_are_refused(cuda, name):
    call, x = calls()[name], torch.randn((5, 6), device='cuda')
    with pytest.raises(RuntimeError):
        torch.func.vmap(call)(torch.stack([x, x]))
    if name not in ('quantize', 'linear4'):
        with pytest.raises(RuntimeError):
            torch.func.grad(lambda t: call(t).sum())(x)
        with pytest.raises(RuntimeError):
            torch.func.jvp(call, (x,), (x,))
    assert torch.isfinite(call(x).float()).all()


def test_gate_hangs_by_what_its_gradient_depends_on(cuda):
    """A second derivative raises through the logits and through the gradient that the backward pass was given."""
    from odie_b200.experts import gate
    for normalize in (True, False):
        leaf = torch.randn((5, 6), device='cuda', requires_grad=True)
        weights = gate(leaf, 2, normalize=normalize).weights
        d = torch.ones_like(weights, requires_grad=True)
        (g,) = torch.autograd.grad(weights, leaf, d, create_graph=True)
        for t in (leaf, d):
            with pytest.raises(RuntimeError, match='once'):
                torch.autograd.grad(g.sum(), t, retain_graph=True)


def test_results_that_were_changed_are_not_used(cuda):
    """Weights or logits written over between the passes are an error, not another gradient."""
    from odie_b200.experts import balance, gate
    leaf = torch.randn((5, 6), device='cuda', requires_grad=True)
    x = leaf * 1
    expert, weights = gate(x, 2)
    total = weights.sum()
    weights.detach().mul_(2)
    with pytest.raises(RuntimeError, match='inplace'):
        total.backward()
    loss = balance(x, expert).loss
    x.detach().mul_(2)
    with pytest.raises(RuntimeError, match='inplace'):
        loss.backward()


# ---------------------------------------------------------------- values
@pytest.mark.parametrize('experts', [5, 30, 100, 256, 300, 1000])
def test_gate_of_no_numbers(cuda, experts):
    """A NaN among a row's logits, of either sign, is its first choice, and its softmax is NaN; rows beside it are not."""
    from odie_b200.experts import balance, gate
    g = generator(experts)
    logits = torch.randn((40, experts), generator=g, device='cuda')
    bad = logits.clone()
    places = torch.arange(40, device='cuda') * 7 % experts
    nan = torch.tensor([0x7fc00000, -4194304, 0x7f800001, -1], dtype=torch.int32, device='cuda').view(torch.float32)
    bad[torch.arange(0, 40, 2), places[::2]] = nan[torch.arange(20, device='cuda') % 4]
    for choices in (1, 4, min(experts, 17)):
        for normalize in (True, False):
            expert, weights = gate(bad, choices, normalize=normalize)
            want = gate(logits, choices, normalize=normalize)
            assert torch.equal(expert[::2, 0].long(), places[::2]) and weights[::2].isnan().all()
            assert torch.equal(expert[1::2], want.expert[1::2]) and torch.equal(weights[1::2], want.weights[1::2])
    mask = ~bad.isnan()
    expert, weights = gate(bad, 1, mask=mask)
    want = plain_gate(torch.where(mask, bad, 0.0), 1, None, mask, 'softmax', True, 1.0, torch.ones((40, 1), device='cuda'))
    assert torch.equal(expert.long(), want[0])
    leaf = bad.clone().requires_grad_()
    loss, z, _ = balance(leaf, expert, mask=mask)
    assert torch.isfinite(torch.autograd.grad(loss + z, leaf)[0]).all()


def test_gate_of_ties(cuda):
    """Rows whose highest logit many experts have: the lowest numbers, in ascending order."""
    from odie_b200.experts import gate
    for experts in (8, 20, 100, 256, 200, 512, 1024):
        logits = torch.zeros((6, experts), dtype=torch.bfloat16, device='cuda')
        logits[1] = -0.0
        logits[2, ::2] = -0.0
        logits[3, : experts // 2] = -1
        logits[4, ::3] = 1
        logits[5] = torch.finfo(torch.bfloat16).min
        for choices in (1, 2, 5, min(experts, 16), min(experts, 40)):
            for bias in (None, torch.zeros(experts, device='cuda')):
                expert = gate(logits, choices, bias=bias).expert
                want = torch.sort(logits.float() + 0.0, dim=1, descending=True, stable=True).indices[:, :choices]
                assert torch.equal(expert.long(), want)


def test_linear4_with_offsets_out_of_order(cuda):
    """Offsets that run backwards or out of range: rows of y may hold anything, but nothing else is touched."""
    from odie_b200.experts import linear4, quantize
    x = torch.randn((300, 96), device='cuda').half()
    weight = quantize(torch.randn((4, 200, 96), device='cuda'))
    for bad in ([0, 200, 100, 300, 50], [5, -7, 1 << 30, 20, 300], [300, 300, 300, 300, 300], [0, 0, 0, 0, 10000]):
        y = linear4(x, weight, offsets=torch.tensor(bad, dtype=torch.int32, device='cuda'))
        assert y.shape == (300, 200)
    good = torch.tensor([0, 100, 150, 150, 280], dtype=torch.int32, device='cuda')
    y = linear4(x, weight, offsets=good)
    assert torch.isfinite(y).all() and (y[280:] == 0).all()


def test_linear4_leaves_what_stands_beside_its_results(cuda):
    """Through the C interface: results of odd sizes within a larger buffer, the rest of which stays as it was."""
    from odie_b200 import _lib
    from odie_b200.experts import linear4, quantize
    lib = _lib.library()
    for rows, inputs, outputs, offset in ((3, 100, 77, 1), (5, 100, 77, 3), (200, 300, 130, 8), (700, 256, 515, 5), (3000, 96, 520, 8)):
        x = torch.randn((rows, inputs), device='cuda').bfloat16()
        micro = quantize(torch.randn((outputs, inputs), device='cuda'))
        want = linear4(x, micro, activation='relu')
        buffer = torch.full((rows * outputs + 64,), 7.0, device='cuda', dtype=torch.bfloat16)
        y = buffer[offset:offset + rows * outputs]
        work = torch.empty(lib.odie_linear4_scratch(rows, inputs, outputs, 1, 0, 16), dtype=torch.uint8, device='cuda')
        status = lib.odie_linear4(x.data_ptr(), micro.codes.data_ptr(), micro.scales.data_ptr(), micro.row_scales.data_ptr(), 16, None, None, rows,
                                  inputs, outputs, 1, None, 1, 1, y.data_ptr(), work.data_ptr() if work.numel() else None,
                                  torch.cuda.current_stream().cuda_stream)
        assert status == 0, _lib.error()
        assert torch.equal(y.view(rows, outputs), want)
        assert (buffer[:offset] == 7).all() and (buffer[offset + rows * outputs:] == 7).all()


def test_rows_do_not_depend_on_their_neighbours(cuda):
    """A row's 4-bit result is the same among many and among few, but for the order of its sum."""
    from odie_b200.experts import linear4, quantize
    g = generator(4)
    x = torch.randn((600, 1000), generator=g, device='cuda').half() * torch.logspace(-2, 2, 600, device='cuda').half()[:, None]
    weight = torch.randn((300, 1000), generator=g, device='cuda')
    micro = quantize(weight)
    y = linear4(x, micro)
    magnitude = plain_micro(x, 16)[0].abs() @ plain_micro(weight, 16)[0].abs().t()
    for part in (slice(0, 1), slice(7, 10), slice(100, 150), slice(300, 600)):
        own = linear4(x[part], micro)
        bound = 2 * 1001 * 2.0 ** -23 * magnitude[part]
        within(own, y[part].double(), bound + 2 * 2.0 ** -11 * (y[part].double().abs() + bound) + 2.0 ** -24, 'rows')


@pytest.mark.parametrize('rows, inputs, outputs', [(3, 8, 1 << 20), (5, 16, (1 << 20) - 8), (300, 40, (1 << 20) - 3), (3, 1 << 20, 8), (6, (1 << 20) - 3, 5)])
@pytest.mark.parametrize('block', [16, 32])
def test_linear4_of_the_most_inputs_and_outputs(cuda, rows, inputs, outputs, block):
    """Up to 2^20 of either; compared at some of many columns."""
    from odie_b200.experts import linear4, quantize
    g = generator(rows + block)
    x = torch.randn((rows, inputs), generator=g, device='cuda').bfloat16()
    weight = (torch.randn((outputs, inputs), generator=g, device='cuda') * inputs ** -0.5).bfloat16()
    y = linear4(x, quantize(weight, block=block), activation='silu')
    at = torch.tensor(sorted({0, 1, outputs // 2, outputs - 1, *torch.randint(0, outputs, (60,), generator=torch.Generator().manual_seed(1)).tolist()}), device='cuda')
    q, w = plain_micro(x, block)[0], plain_micro(weight[at], block)[0]
    z = q @ w.t()
    off = (inputs + 1) * 2.0 ** -23 * (q.abs() @ w.abs().t()) + 3 * 2.0 ** -24 * z.abs()
    want = z * torch.sigmoid(z)
    bound = 1.13 * off + 2.0 ** -20 * (z.abs() + 1)
    within(y[:, at], want, bound + 2.0 ** -8 * (want.abs() + bound), 'silu')


@pytest.mark.parametrize('dtype', [torch.float16, torch.float32])
@pytest.mark.parametrize('block', [16, 32])
def test_quantize_the_longest_rows(cuda, dtype, block):
    from odie_b200.experts import dequantize, quantize
    for width in (1 << 20, (1 << 20) - 5):
        x = torch.randn((3, width), generator=generator(5), device='cuda').to(dtype)
        assert torch.equal(dequantize(quantize(x, block=block)).double(), plain_micro(x, block)[0])


@pytest.mark.parametrize('up, down', [(100, -100), (-60, -50), (60, -110), (-110, 100), (110, -125)])
@pytest.mark.parametrize('rows, inputs, outputs', [(1, 300, 40), (3, 64, 200), (50, 2048, 130), (300, 256, 700)])
@pytest.mark.parametrize('block', [16, 32])
def test_linear4_of_far_rows_and_weights(cuda, up, down, rows, inputs, outputs, block):
    """Rows and weights of sizes whose product is far from either: no step on the way leaves the range that the result is in."""
    from odie_b200.experts import linear4, quantize
    g = generator(rows)
    x, weight = torch.randn((rows, inputs), generator=g, device='cuda'), torch.randn((outputs, inputs), generator=g, device='cuda')
    x, weight = (x.double() * 2.0 ** up).bfloat16(), (weight.double() * 2.0 ** down).bfloat16()
    y = linear4(x, quantize(weight, block=block))
    q, w = plain_micro(x, block)[0], plain_micro(weight, block)[0]
    want = q @ w.t()
    bound = (inputs + 1) * 2.0 ** -23 * (q.abs() @ w.abs().t()) + 3 * 2.0 ** -24 * want.abs()
    within(y, want, bound + 2.0 ** -8 * (want.abs() + bound) + 2.0 ** -134, 'y')


@pytest.mark.parametrize('groups', [31, 32, 255, 256, 257, 1023, 1024])
@pytest.mark.parametrize('spread', ['some empty', 'last only', 'none', 'one row each'])
def test_linear4_of_many_groups(cuda, groups, spread):
    """Each way of finding a tile's rows from the offsets, with rows of more than one tile and rows of no group."""
    from odie_b200.experts import linear4, quantize
    from test_gpu_micro import plain_linear4
    g = generator(groups)
    sizes = [0] * groups
    if spread == 'some empty':
        for i, n in ((0, 129), (groups // 3, 300), (groups - 2, 128), (groups - 1, 5)):
            sizes[i] = n
    elif spread == 'last only':
        sizes[-1] = 400
    elif spread == 'one row each':
        sizes = [1] * groups
    edges = [0]
    for n in sizes:
        edges.append(edges[-1] + n)
    rows = edges[-1] + 140
    x = torch.randn((rows, 48), generator=g, device='cuda').bfloat16()
    weight = (torch.randn((groups, 24, 48), generator=g, device='cuda') / 7).bfloat16()
    y = linear4(x, quantize(weight), offsets=torch.tensor(edges, dtype=torch.int32, device='cuda'))
    value, bound = plain_linear4(x, weight, None, None, list(zip(edges, edges[1:])), 'none', 16)
    within(y, value, bound, 'many groups')
    assert (y[edges[-1]:] == 0).all()


@pytest.mark.parametrize('groups', [256, 1024])
def test_linear4_of_many_groups_with_offsets_out_of_order(cuda, groups):
    from odie_b200.experts import linear4, quantize
    x = torch.randn((700, 48), device='cuda').half()
    weight = quantize(torch.randn((groups, 24, 48), device='cuda'))
    for step in (1, 2, 3):
        bad = torch.arange(groups + 1, dtype=torch.int32).remainder(step + 1).mul(900).sub(100).cuda()
        assert linear4(x, weight, offsets=bad).shape == (700, 24)
    y = linear4(x, weight, offsets=torch.full((groups + 1,), 700, dtype=torch.int32, device='cuda').mul_(torch.arange(groups + 1, device='cuda') > 0))
    assert torch.isfinite(y).all()
