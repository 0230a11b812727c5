"""Microscaled 4-bit rows on the GPU (quantize, dequantize, linear4 of odie_b200.experts) against plain 64-bit forms."""
import pytest
import torch

from router_cases import plain_micro, unpacked
from rows_cases import SUM, TYPES, activated, rounding, within

pytestmark = pytest.mark.gpu

HALVES = [torch.float16, torch.bfloat16]
ROWS = [(1, 1), (1, 16), (3, 31), (128, 32), (129, 33), (5, 64), (300, 100), (257, 128), (7, 1000), (130, 2048), (64, 4096), (33, 5000), (3, 20001)]


def generator(seed):
    return torch.Generator(device='cuda').manual_seed(seed)


def values(g, *shape, dtype=torch.float32, std=1.0):
    """Columns of different sizes, some of them zero."""
    x = torch.randn(shape, generator=g, device='cuda') * torch.exp(2 * torch.randn(shape[-1:], generator=g, device='cuda'))
    return (x * std * (torch.rand(shape, generator=g, device='cuda') < 0.9)).to(dtype)


def check_micro(micro, x, block):
    want, codes, scales, outer = plain_micro(x, block)
    got_codes, got_scales = unpacked(micro)
    rows, width = x.shape
    assert micro.shape == x.shape
    within(micro.row_scales.reshape(-1), outer, torch.zeros_like(outer), 'row scales')
    live = ~outer.isnan()
    assert torch.equal(got_scales[:rows, :scales.shape[1]][live], scales[live])
    assert (got_scales[:rows, scales.shape[1]:] == 0).all() and (got_scales[rows:] == 0).all() and (got_codes[:, width:] == 0).all()
    differ = (got_codes[:, :width] != codes) & live[:, None] & ~((got_codes[:, :width] % 8 == 0) & (codes % 8 == 0))  # zeros of either sign
    assert not differ.any()
    return want


@pytest.mark.parametrize('rows, width', ROWS)
@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('block', [16, 32])
def test_quantize_and_dequantize(cuda, rows, width, dtype, block):
    from odie_b200.experts import dequantize, quantize
    x = values(generator(rows + width), rows, width, dtype=dtype, std=0.01 if dtype == torch.float16 else 1.0)
    if rows > 4:
        x[1] = 0
        x[2, 0] = float('inf')
        x[3, width - 1] = float('nan')
        x[4] *= 2.0 ** -12
    micro = quantize(x, block=block)
    want = check_micro(micro, x, block)
    for to in TYPES:
        within(dequantize(micro, to), want, rounding(want, to) if to == torch.float16 else torch.zeros_like(want), f'values in {to}')
    again = quantize(x, block=block)
    assert all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip(micro[:3], again[:3]))


@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('block', [16, 32])
def test_quantize_next_to_borders(cuda, dtype, block):
    """Values on the borders between codes and one step of the type beside them, for every block scale there can be."""
    from odie_b200.experts import quantize
    borders = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0], dtype=torch.float64)
    rows = []
    for mantissa in range(8, 16):
        for exponent in (-9, -2, 0, 3):
            scale = mantissa * 2.0 ** exponent
            for side in (0, 1, -1):
                v = (borders * scale).to(dtype)
                if side:
                    v = (v.view(torch.int32 if dtype == torch.float32 else torch.int16) + side).view(dtype)
                row = torch.zeros(64, dtype=dtype)
                row[0] = 6 * scale           # the block's largest: its scale is exact
                row[1:8], row[8:15] = v, -v
                row[40] = 2688 * 2.0 ** (exponent + 1)  # the row's
                rows.append(row)
    check_micro(quantize(torch.stack(rows).cuda(), block=block), torch.stack(rows).cuda(), block)


@pytest.mark.parametrize('block', [16, 32])
def test_quantize_far_numbers(cuda, block):
    """Rows of the largest and smallest fp32 and bf16 numbers, and blocks far below their row."""
    from odie_b200.experts import dequantize, quantize
    g = generator(3)
    for dtype in (torch.float32, torch.bfloat16):
        x = torch.randn((40, 96), generator=g, device='cuda')
        power = torch.linspace(-148, 124, 40, device='cuda').round().double()
        x = (x.double() * torch.ldexp(torch.ones_like(power), power.long())[:, None]).to(dtype)
        x[:, 32:64] = (x[:, 32:64].double() * 2.0 ** -14).to(dtype)
        x = torch.where(torch.isfinite(x), x, 0.0)
        want = check_micro(quantize(x, block=block), x, block)
        # (numbers below the least normal one may be cut to it in a product of scales)
        within(dequantize(quantize(x, block=block)), want, rounding(want, torch.float32), 'values')


def test_quantize_groups_views_and_nothing(cuda):
    from odie_b200.experts import dequantize, quantize
    g = generator(5)
    for rows in (5, 128, 200):
        x = values(g, 3, rows, 100, dtype=torch.bfloat16)
        micro = quantize(x, block=16)
        assert micro.shape == x.shape and micro.scales.shape == (3, -(-rows // 128), 2, 512)
        for i in range(3):
            one = quantize(x[i], block=16)
            assert torch.equal(one.codes, micro.codes[i]) and torch.equal(one.scales[0], micro.scales[i])
        assert torch.equal(dequantize(micro, torch.bfloat16)[1], dequantize(quantize(x[1], block=16), torch.bfloat16))
    x = values(g, 41, 77, dtype=torch.float16, std=0.01)
    for view in (x[:, 3:70], x[::2], x.t(), x.reshape(-1)[1:1 + 40 * 64].view(40, 64)):
        a, b = quantize(view, block=32), quantize(view.clone(memory_format=torch.contiguous_format), block=32)
        assert torch.equal(a.codes, b.codes) and torch.equal(a.scales, b.scales)
    none = quantize(x[:0], block=16)
    assert none.codes.shape == (0, 48) and dequantize(none).shape == (0, 77)


# ---------------------------------------------------------------- the product
def plain_linear4(x, weight, bias, residual, edges, activation, block):
    """(value, bound) in 64 bits; weight [groups, outputs, inputs]."""
    dtype = x.dtype
    q = plain_micro(x, block)[0]
    rows, outputs, inputs = x.shape[0], weight.shape[1], x.shape[1]
    value = torch.zeros((rows, outputs), dtype=torch.float64, device=x.device)
    bound = torch.zeros_like(value)
    for g, (lo, hi) in enumerate(edges):
        w = plain_micro(weight[g], block)[0]
        z = q[lo:hi] @ w.t()
        off = (inputs + 1) * SUM * (q[lo:hi].abs() @ w.abs().t()) + 3 * 2.0 ** -24 * z.abs()
        if bias is not None:
            z = z + bias[g].double()
            off = off + 2.0 ** -24 * z.abs()
        a, _ = activated(z, activation)
        y = a if residual is None else a + residual[lo:hi].double()
        own = 0.0 if activation in ('none', 'relu') else 2.0 ** -20 * (z.abs() + 1)
        value[lo:hi] = y
        b = 1.13 * off + own + 2.0 ** -24 * (a.abs() + y.abs())
        bound[lo:hi] = b + rounding(y.abs() + b, dtype)
    return value, bound


LAYERS = [(1, 1, 1), (1, 16, 8), (2, 64, 128), (1, 4096, 512), (3, 333, 515), (5, 256, 136), (64, 4096, 256), (100, 1000, 300), (128, 512, 128), (129, 257, 129),
          (300, 2048, 1024), (1021, 333, 515), (2, 5000, 77), (700, 544, 2000), (8, 16384, 40), (4000, 96, 520), (1, 20001, 33), (4, 2048, 1000),
          (2500, 1100, 1300)]


@pytest.mark.parametrize('rows, inputs, outputs', LAYERS)
@pytest.mark.parametrize('dtype', HALVES)
@pytest.mark.parametrize('block', [16, 32])
def test_linear4(cuda, rows, inputs, outputs, dtype, block):
    from odie_b200.experts import linear4, quantize
    g = generator(rows + inputs + outputs)
    x = torch.randn((rows, inputs), generator=g, device='cuda').to(dtype)
    weight = (torch.randn((outputs, inputs), generator=g, device='cuda') * inputs ** -0.5).to(dtype)
    micro = quantize(weight, block=block)
    for activation, biased, added in (('none', False, False), ('relu', True, False), ('silu', True, True), ('gelu', False, True)):
        bias = torch.randn(outputs, generator=g, device='cuda').to(dtype) if biased else None
        residual = torch.randn((rows, outputs), generator=g, device='cuda').to(dtype) if added else None
        y = linear4(x, micro, bias=bias, residual=residual, activation=activation)
        want = plain_linear4(x, weight[None], None if bias is None else bias[None], residual, [(0, rows)], activation, block)
        assert y.dtype == dtype
        within(y, *want, activation)
        assert torch.equal(y, linear4(x, micro, bias=bias, residual=residual, activation=activation))


# sizes of groups, rows behind the last one
GROUPS = [([5], 0), ([0, 1, 0, 2], 3), ([128, 256, 1, 127, 129], 0), ([1] * 40, 5), ([300, 0, 700, 513], 130), ([0, 0, 0], 17), ([2000, 3, 1500], 0)]


@pytest.mark.parametrize('sizes, tail', GROUPS)
@pytest.mark.parametrize('inputs, outputs', [(96, 40), (333, 515), (1024, 768)])
@pytest.mark.parametrize('block', [16, 32])
def test_linear4_of_groups(cuda, sizes, tail, inputs, outputs, block):
    from odie_b200.experts import linear4, quantize
    g = generator(len(sizes) + tail + inputs)
    rows, groups, dtype = sum(sizes) + tail, len(sizes), torch.bfloat16 if inputs == 333 else torch.float16
    x = torch.randn((rows, inputs), generator=g, device='cuda').to(dtype)
    if tail:
        x[-tail:] = float('nan')  # never read into a result
    weight = (torch.randn((groups, outputs, inputs), generator=g, device='cuda') * inputs ** -0.5).to(dtype)
    bias, residual = torch.randn((groups, outputs), generator=g, device='cuda').to(dtype), torch.randn((rows, outputs), generator=g, device='cuda').to(dtype)
    edges = [0]
    for n in sizes:
        edges.append(edges[-1] + n)
    offsets = torch.tensor(edges, dtype=torch.int32, device='cuda')
    micro = quantize(weight, block=block)
    y = linear4(x, micro, bias=bias, residual=residual, activation='silu', offsets=offsets)
    value, bound = plain_linear4(x, weight, bias, residual, list(zip(edges, edges[1:])), 'silu', block)
    within(y, value, bound, 'groups')
    assert (y[edges[-1]:] == 0).all()


def test_linear4_keeps_a_bad_row_to_itself(cuda):
    """A row or column with an infinity or NaN is NaN, and no other."""
    from odie_b200.experts import linear4, quantize
    g = generator(8)
    for rows, inputs, outputs in ((1, 200, 64), (3, 512, 200), (300, 512, 600)):
        x = torch.randn((rows, inputs), generator=g, device='cuda').bfloat16()
        weight = torch.randn((outputs, inputs), generator=g, device='cuda')
        weight[outputs // 2, 7] = float('inf')
        if rows > 1:
            x[1, inputs - 1] = float('nan')
        for block in (16, 32):
            bad = linear4(x, quantize(weight, block=block)).isnan()
            want = torch.zeros_like(bad)
            want[:, outputs // 2] = True
            if rows > 1:
                want[1] = True
            assert torch.equal(bad, want)


def test_linear4_shapes_views_and_streams(cuda):
    from odie_b200.experts import linear4, quantize
    g = generator(9)
    weight = torch.randn((72, 80), generator=g, device='cuda')
    micro = quantize(weight)
    x = torch.randn((4, 5, 80), generator=g, device='cuda').half()
    whole = linear4(x, micro, residual=x[..., :1])
    assert whole.shape == (4, 5, 72)
    assert torch.equal(whole.view(20, 72), linear4(x.view(20, 80), micro, residual=x.view(20, 80)[:, :1]))
    assert torch.equal(linear4(x[0, 0], micro), linear4(x[0, :1], micro)[0])
    assert linear4(x[:0], micro).shape == (0, 5, 72)
    odd = torch.randn(20 * 80 + 3, generator=g, device='cuda').half()[3:].view(20, 80)
    assert torch.equal(linear4(odd, micro), linear4(odd.clone(), micro))
    assert torch.equal(linear4(odd.t().contiguous().t(), micro), linear4(odd, micro))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = linear4(odd, micro)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(other, linear4(odd, micro))


def test_linear4_is_captured_and_replayed(cuda):
    """Two graphs of one layer, of a row and of a batch, replayed in turn on other rows."""
    from odie_b200.experts import linear4, quantize
    g = generator(10)
    micro = quantize(torch.randn((300, 520), generator=g, device='cuda'))
    inputs = [torch.randn((n, 520), generator=g, device='cuda').bfloat16() for n in (1, 400)]
    others = [torch.randn_like(x) for x in inputs]
    want = [[linear4(x, micro, activation='gelu') for x in xs] for xs in (inputs, others)]
    static, graphs, results = [x.clone() for x in inputs], [], []
    for x in static:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            results.append(linear4(x, micro, activation='gelu'))
        graphs.append(graph)
    for turn, xs in ((0, inputs), (1, others), (0, inputs)):
        for x, s in zip(xs, static):
            s.copy_(x)
        for graph in graphs:
            graph.replay()
        assert all(torch.equal(a, b) for a, b in zip(results, want[turn]))


def test_linear4_wait_that_runs_out(cuda):
    """A product whose waits may not poll at all ends, and the next call says so, once; then all is as before."""
    from odie_b200 import _lib
    from odie_b200.experts import check, linear4, quantize
    lib = _lib.library()
    g = generator(11)
    for rows, inputs, outputs in ((64, 4096, 256), (700, 544, 2000), (4000, 512, 2048)):
        x = torch.randn((rows, inputs), generator=g, device='cuda').bfloat16()
        micro = quantize(torch.randn((outputs, inputs), generator=g, device='cuda'))
        want = linear4(x, micro)
        torch.cuda.synchronize()
        assert lib.odie_linear_wait_limit(0) == 0
        try:
            linear4(x, micro)
            torch.cuda.synchronize()
        finally:
            assert lib.odie_linear_wait_limit(-1) == 0
        with pytest.raises(RuntimeError, match='ran out'):
            linear4(x, micro)
        check()
        assert torch.equal(linear4(x, micro), want)
