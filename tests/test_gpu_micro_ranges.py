"""linear4 on rows and weights whose scales are far from 1, on each of its ways: one or two rows, parts of K, tiles of 128 and
of 256, groups.  No step on the way leaves a range that the result is in."""
import pytest
import torch

from router_cases import plain_micro
from test_gpu_micro import plain_linear4

pytestmark = pytest.mark.gpu

# rows, inputs, outputs, sizes of groups: one row, two, parts of K, tiles of 128, of 256, and both with groups
WAYS = [(1, 300, 40, None), (2, 256, 130, None), (64, 4096, 200, None), (3, 64, 200, None), (300, 256, 700, None), (3000, 256, 1000, None),
        (300, 256, 200, [100, 0, 150]), (3000, 256, 1000, [1000, 1500, 400])]


def made(rows, inputs, outputs, sizes, up, down, seed):
    """(x, weight, their exact product, the product of their magnitudes, offsets) of rows of 2^up and weights of 2^down."""
    from odie_b200.experts import quantize
    g = torch.Generator(device='cuda').manual_seed(seed)
    groups = len(sizes or [1])
    x = torch.randn((rows, inputs), generator=g, device='cuda')
    weight = torch.randn((groups, outputs, inputs), generator=g, device='cuda')
    x, weight = (x.double() * 2.0 ** up).bfloat16(), (weight.double() * 2.0 ** down).bfloat16()
    edges = [0]
    for n in sizes or [rows]:
        edges.append(edges[-1] + n)
    micro = quantize(weight if sizes else weight[0])
    offsets = torch.tensor(edges, dtype=torch.int32, device='cuda') if sizes else None
    return x, weight, micro, list(zip(edges, edges[1:])), offsets


def close(got, want, bound):
    """Within the bound, which counts in double; equal where fp32's range or bf16's has ended."""
    got, most = got.double(), torch.finfo(torch.bfloat16).max
    over = ((got - want).abs() > bound) & ~((got.isinf()) & (want.abs() + bound > most) & (got.sign() == want.sign()))
    assert not got.isnan().any() and not over.any(), f'{over.sum().item()} of {over.numel()} are off, {got.isinf().sum().item()} infinite'


@pytest.mark.parametrize('up, down', [(118, -118), (116, -110), (122, -120), (-118, 118), (-110, 122), (-66, -66), (-125, -4), (70, 50)])
@pytest.mark.parametrize('rows, inputs, outputs, sizes', WAYS)
def test_scales_of_rows_and_columns(cuda, rows, inputs, outputs, sizes, up, down):
    """Sums of `inputs` terms in fp32; a result below the least normal number is off by half a step of bf16 there, 2^-134, and
    of fp32 before it, 2^-150."""
    from odie_b200.experts import linear4
    x, weight, micro, edges, offsets = made(rows, inputs, outputs, sizes, up, down, rows + up)
    y = linear4(x, micro, offsets=offsets)
    q = plain_micro(x, 16)[0]
    want, size = (torch.zeros((rows, outputs), dtype=torch.float64, device='cuda') for _ in range(2))
    for i, (low, high) in enumerate(edges):
        w = plain_micro(weight[i], 16)[0]
        want[low:high], size[low:high] = q[low:high] @ w.t(), q[low:high].abs() @ w.abs().t()
    bound = (inputs + 1) * 2.0 ** -23 * size + 3 * 2.0 ** -24 * want.abs()
    close(y, want, bound + 2.0 ** -8 * (want.abs() + bound) + 2.0 ** -134 + 2.0 ** -149)


@pytest.mark.parametrize('rows, inputs, outputs, sizes', WAYS)
def test_an_epilogue_after_far_scales(cuda, rows, inputs, outputs, sizes):
    """Bias, activation and residual are what they are with ordinary scales: rows and weights times 2^110 and 2^-110 give the
    same bits, and so they do where some rows are far and some are not."""
    from odie_b200.experts import linear4, quantize
    x, weight, micro, edges, offsets = made(rows, inputs, outputs, sizes, 0, -3, rows)
    g = torch.Generator(device='cuda').manual_seed(1)
    bias = torch.randn(weight.shape[:2], generator=g, device='cuda').bfloat16()
    residual = torch.randn((rows, outputs), generator=g, device='cuda').bfloat16()
    far = quantize((weight.double() * 2.0 ** -110).bfloat16() if sizes else (weight[0].double() * 2.0 ** -110).bfloat16())
    b = bias if sizes else bias[0]
    for activation in ('none', 'relu', 'silu', 'gelu'):
        want = linear4(x, micro, bias=b, residual=residual, activation=activation, offsets=offsets)
        got = linear4((x.double() * 2.0 ** 110).bfloat16(), far, bias=b, residual=residual, activation=activation, offsets=offsets)
        assert torch.equal(got, want)
    value, bound = plain_linear4(x, weight, bias, residual, edges, 'gelu', 16)
    close(want, value, bound)
    part = torch.arange(rows, device='cuda') % 50 == 1
    mixed = torch.where(part[:, None], x.double() * 2.0 ** 90, x.double()).bfloat16()
    got = linear4(mixed, micro, offsets=offsets)
    want = linear4(x, micro, offsets=offsets)
    assert torch.equal(got[~part], want[~part]) and torch.equal(got[part].double(), want[part].double() * 2.0 ** 90)


@pytest.mark.parametrize('rows, inputs, outputs, sizes', WAYS)
def test_nothing_of_far_scales_is_nothing(cuda, rows, inputs, outputs, sizes):
    """Rows and weights without a value in common: 0, also where the product of their scales is infinite."""
    from odie_b200.experts import linear4, quantize
    x, weight, _, _, offsets = made(rows, inputs, outputs, sizes, 120, 30, rows)
    x[:, 1::2] = 0
    weight[..., ::2] = 0
    for block in (16, 32):
        y = linear4(x, quantize(weight if sizes else weight[0], block=block), offsets=offsets)
        assert (y == 0).all(), (block, y.isnan().sum().item())


@pytest.mark.parametrize('rows', [1, 2, 3, 300])
@pytest.mark.parametrize('inputs, at', [(32, 5), (2100, 2077)])
def test_scales_of_blocks(cuda, rows, inputs, at):
    """Blocks of 32: the scales of a row's block and a weight's are 2^124 and 2^4 (their largest values meet zeros), the one
    product 2^126; and with 2^-124 and 2^-4, 2^-130."""
    from odie_b200.experts import linear4, quantize
    block = at // 32 * 32
    for sign in (1, -1):
        x, w = (torch.zeros((n, inputs), dtype=torch.float64, device='cuda') for n in (rows, 40))
        x[:, block], x[:, at] = 2.0 ** (126 if sign > 0 else -122), 2.0 ** (123 if sign > 0 else -125)
        w[:, block + 1], w[:, at] = 2.0 ** (6 if sign > 0 else -2), 2.0 ** (3 if sign > 0 else -5)
        micro = quantize(w.bfloat16(), block=32)
        y = linear4(x.bfloat16(), micro)
        assert (y.double() == 2.0 ** (126 if sign > 0 else -130)).all(), y
