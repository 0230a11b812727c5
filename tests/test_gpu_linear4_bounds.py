"""linear4 writes its results and its scratch and nothing beside them, whatever the offsets; sums over K in parts of unequal
length; rows that are no numbers among rows of far scales; what a wait that ran out is called."""
import pytest
import torch

from test_gpu_micro import plain_linear4
from rows_cases import within

pytestmark = pytest.mark.gpu

GUARD = 4096  # bytes before and behind


def guarded(size):
    """(buffer, its inner `size` bytes on a 256-byte boundary); filled with 0x5a."""
    buffer = torch.full((size + 2 * GUARD,), 0x5a, dtype=torch.uint8, device='cuda')
    assert buffer.data_ptr() % 256 == 0
    return buffer, buffer[GUARD:GUARD + size]


BAD = {
    'backwards': lambda groups, rows: [rows - i * rows // groups for i in range(groups + 1)],
    'to and fro': lambda groups, rows: [0] + [(i * 7919) % (rows + 1) for i in range(1, groups + 1)],
    'far out': lambda groups, rows: [(-1) ** i * (1 << 30) + i for i in range(groups + 1)],
    'whole, again and again': lambda groups, rows: [i % 2 * rows for i in range(groups + 1)],
    'negative': lambda groups, rows: [-5] * (groups + 1),
    'none': lambda groups, rows: [0] * (groups + 1),
    'extremes': lambda groups, rows: [(1 << 31) - 1 if i % 3 else -(1 << 31) for i in range(groups + 1)],
}


@pytest.mark.parametrize('kind', list(BAD))
@pytest.mark.parametrize('groups, rows, inputs, outputs', [(4, 300, 96, 200), (3, 3000, 64, 1000), (40, 513, 48, 33), (256, 700, 48, 24), (1024, 2100, 32, 40)])
@pytest.mark.parametrize('block', [16, 32])
def test_offsets_out_of_order_touch_nothing_else(cuda, kind, groups, rows, inputs, outputs, block):
    from odie_b200 import _lib
    from odie_b200.experts import quantize
    lib = _lib.library()
    g = torch.Generator(device='cuda').manual_seed(groups)
    x = torch.randn((rows, inputs), generator=g, device='cuda').half()
    residual = torch.randn((rows, outputs), generator=g, device='cuda').half()
    micro = quantize(torch.randn((groups, outputs, inputs), generator=g, device='cuda'), block=block)
    offsets = torch.tensor(BAD[kind](groups, rows), dtype=torch.int32, device='cuda')
    kept = [t.clone() for t in (x, residual, *micro[:3], offsets)]
    y_buffer, y = guarded(rows * outputs * 2)
    work_buffer, work = guarded(lib.odie_linear4_scratch(rows, inputs, outputs, groups, 1, block))
    status = lib.odie_linear4(x.data_ptr(), micro.codes.data_ptr(), micro.scales.data_ptr(), micro.row_scales.data_ptr(), block, None,
                              residual.data_ptr(), rows, inputs, outputs, groups, offsets.data_ptr(), 0, 2, y.data_ptr(), work.data_ptr(),
                              torch.cuda.current_stream().cuda_stream)
    assert status == 0, _lib.error()
    for buffer in (y_buffer, work_buffer):
        assert (buffer[:GUARD] == 0x5a).all() and (buffer[-GUARD:] == 0x5a).all()
    assert all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip(kept, (x, residual, *micro[:3], offsets)))


# blocks of 256 inputs: 17 in parts of 5, 5, 5 and 2; 33 and 41 in seven parts; 9 in two
@pytest.mark.parametrize('inputs', [4200, 8300, 10500, 12400, 2100])
@pytest.mark.parametrize('rows, outputs', [(64, 300), (5, 100), (129, 130)])
@pytest.mark.parametrize('block', [16, 32])
def test_parts_of_unequal_length(cuda, inputs, rows, outputs, block):
    from odie_b200.experts import linear4, quantize
    g = torch.Generator(device='cuda').manual_seed(inputs + rows)
    x = torch.randn((rows, inputs), generator=g, device='cuda').bfloat16()
    weight = (torch.randn((outputs, inputs), generator=g, device='cuda') * inputs ** -0.5).bfloat16()
    residual = torch.randn((rows, outputs), generator=g, device='cuda').bfloat16()
    y = linear4(x, quantize(weight, block=block), residual=residual, activation='silu')
    within(y, *plain_linear4(x, weight[None], None, residual, [(0, rows)], 'silu', block), 'y')


@pytest.mark.parametrize('rows, inputs, outputs', [(1, 300, 40), (64, 4096, 200), (300, 256, 700), (3000, 256, 1000)])
def test_no_numbers_among_far_scales(cuda, rows, inputs, outputs):
    """A bad row or column is NaN and no other, also beside rows of 2^100 and of 2^-100."""
    from odie_b200.experts import linear4, quantize
    g = torch.Generator(device='cuda').manual_seed(rows)
    x = torch.randn((rows, inputs), generator=g, device='cuda') * torch.where(torch.arange(rows, device='cuda') % 2 == 0, 2.0 ** 100, 2.0 ** -100)[:, None]
    weight = torch.randn((outputs, inputs), generator=g, device='cuda')
    weight[outputs // 2, 7] = float('inf')
    if rows > 1:
        x[5, inputs - 1] = float('nan')
    bad = linear4(x.bfloat16(), quantize(weight)).isnan()
    want = torch.zeros_like(bad)
    want[:, outputs // 2] = True
    if rows > 1:
        want[5] = True
    assert torch.equal(bad, want)


def test_a_wait_that_ran_out_is_named(cuda):
    """What `linear` or `check` raise after a product in 4 bits does not send its reader to `linear` alone."""
    from odie_b200 import _lib
    from odie_b200.experts import check, linear, linear4, quantize
    lib = _lib.library()
    x = torch.randn((300, 512), device='cuda').half()
    micro = quantize(torch.randn((600, 512), device='cuda'))
    want = linear4(x, micro)
    for call in (check, lambda: linear(x, x[:8])):
        torch.cuda.synchronize()
        assert lib.odie_linear_wait_limit(0) == 0
        try:
            linear4(x, micro)
            torch.cuda.synchronize()
        finally:
            assert lib.odie_linear_wait_limit(-1) == 0
        with pytest.raises(RuntimeError, match='linear4'):
            call()
        call()
    assert torch.equal(linear4(x, micro), want)
