"""CPU: refusals of the routed-expert row operators, all of them on the host before any device work."""
import ctypes

import pytest
import torch

from odie_b200 import _lib, experts


@pytest.fixture(scope='module')
def lib():
    from odie_b200 import builder
    builder.build()
    return _lib.library()


def test_cpu_tensors_are_refused():
    x, ids = torch.zeros(4, 8), torch.zeros(4, dtype=torch.int32)
    with pytest.raises(ValueError, match='CUDA'):
        experts.sort_rows(ids, 4)
    with pytest.raises(ValueError, match='CUDA'):
        experts.linear(x.half(), torch.zeros(8, 8).half())
    with pytest.raises(ValueError, match='CUDA'):
        experts.embed(ids, x)
    order = experts.RowOrder(ids, ids.view(4, 1), torch.zeros(5, dtype=torch.int32))
    with pytest.raises(ValueError, match='CUDA'):
        experts.dispatch(x, order)
    with pytest.raises(ValueError, match='CUDA'):
        experts.combine(x, order)


# Non-null pointers that nothing reads: every call below fails its checks before it touches them.
SOME = ctypes.c_void_p(256)


@pytest.mark.parametrize('change, message', [
    (dict(key_bytes=2), 'int32 or int64'), (dict(n=-1), 'keys'), (dict(n=2 ** 31), 'keys'), (dict(bins=0), 'bins'),
    (dict(bins=1 << 30), 'bins'), (dict(keys=None), 'keys'), (dict(order=None), 'order'), (dict(offsets=None), 'offsets'),
    (dict(n=100000, scratch=None), 'scratch')])
def test_sort_rows_refuses(lib, change, message):
    a = dict(keys=SOME, key_bytes=4, n=8, bins=4, order=SOME, slot=SOME, offsets=SOME, scratch=None, stream=0)
    a.update(change)
    assert lib.odie_sort_rows(*a.values()) == -1
    assert message in _lib.error()


@pytest.mark.parametrize('change, message', [
    (dict(n=-1), 'pairs'), (dict(choices=0), 'pairs'), (dict(n=2 ** 30, choices=2), 'pairs'), (dict(width=0), 'elements'),
    (dict(dtype=3), 'element type'), (dict(dtype=-1), 'element type'), (dict(slot=None), 'is required'), (dict(rows=None), 'required'),
    (dict(out=None), 'required')])
def test_dispatch_and_combine_refuse(lib, change, message):
    a = dict(rows=SOME, n=8, choices=2, width=8, dtype=0, slot=SOME, weights=None, out=SOME, stream=0)
    a.update(change)
    assert lib.odie_combine(*a.values()) == -1
    assert message in _lib.error()
    a = dict(rows=SOME, n=8, choices=2, width=8, dtype=0, order=SOME, slot=SOME, weights=None, out=SOME, stream=0)
    a.update(change)
    assert lib.odie_dispatch(*a.values()) == -1
    assert message in _lib.error()


@pytest.mark.parametrize('change, message', [
    (dict(width=0), 'elements'), (dict(dtype=5), 'element type'), (dict(order=None), 'order'), (dict(slot=None), 'slot'), (dict(d_out=None), 'required'),
    (dict(rows=None), 'required')])
def test_combine_backward_refuses(lib, change, message):
    a = dict(d_out=SOME, rows=SOME, n=8, choices=2, width=8, dtype=0, order=SOME, slot=SOME, weights=None, d_rows=SOME, d_weights=SOME,
             stream=0)
    a.update(change)
    assert lib.odie_combine_backward(*a.values()) == -1
    assert message in _lib.error()


LINEAR = [(dict(rows=-1), 'rows'), (dict(rows=2 ** 31), 'rows'), (dict(inputs=0), 'inputs'), (dict(outputs=0), 'outputs'),
          (dict(inputs=(1 << 20) + 1), 'inputs'), (dict(groups=0), 'groups'), (dict(groups=1025, offsets=SOME), 'groups'),
          (dict(groups=2), 'offsets'), (dict(dtype=2), 'fp16'), (dict(x=None), 'required'), (dict(weight=None), 'required')]


@pytest.mark.parametrize('change, message', LINEAR + [
    (dict(activation=4), 'activation'), (dict(activation=-1), 'activation'), (dict(y=None), 'required')])
def test_linear_refuses(lib, change, message):
    a = dict(x=SOME, weight=SOME, bias=None, residual=None, rows=8, inputs=8, outputs=8, groups=1, offsets=None, dtype=0,
             activation=0, y=SOME, slope=None, scratch=SOME, stream=0)
    a.update(change)
    assert lib.odie_linear(*a.values()) == -1
    assert message in _lib.error()


@pytest.mark.parametrize('change, message', LINEAR + [(dict(d_y=None), 'required'), (dict(activation=1), 'slope'), (dict(activation=5), 'activation'),
                                                      (dict(scratch=ctypes.c_void_p(16)), '256-byte')])
def test_linear_backward_refuses(lib, change, message):
    a = dict(d_y=SOME, slope=None, activation=0, x=SOME, weight=SOME, rows=8, inputs=8, outputs=8, groups=1, offsets=None, dtype=0,
             d_x=SOME, d_weight=SOME, d_bias=None, d_residual=None, scratch=SOME, stream=0)
    a.update(change)
    assert lib.odie_linear_backward(*a.values()) == -1
    assert message in _lib.error()


EMBED = [(dict(id_bytes=2), 'int32 or int64'), (dict(n=-1), 'ids'), (dict(n=2 ** 31), 'ids'), (dict(rows=0), 'table'),
         (dict(rows=1 << 30), 'table'), (dict(width=0), 'elements'), (dict(dtype=7), 'element type')]


@pytest.mark.parametrize('change, message', EMBED + [
    (dict(ids=None), 'required'), (dict(table=None), 'required'), (dict(out=None), 'required')])
def test_embed_refuses(lib, change, message):
    a = dict(ids=SOME, id_bytes=4, n=8, table=SOME, rows=8, width=8, dtype=0, scale=1.0, out=SOME, stream=0)
    a.update(change)
    assert lib.odie_embed(*a.values()) == -1
    assert message in _lib.error()


@pytest.mark.parametrize('change, message', EMBED + [
    (dict(ids=None), 'required'), (dict(d_out=None), 'required'), (dict(d_table=None), 'required'),
    (dict(scratch=None), 'required')])
def test_embed_backward_refuses(lib, change, message):
    a = dict(ids=SOME, id_bytes=4, n=8, d_out=SOME, rows=8, width=8, dtype=0, scale=1.0, d_table=SOME, scratch=SOME, stream=0)
    a.update(change)
    assert lib.odie_embed_backward(*a.values()) == -1
    assert message in _lib.error()


def test_scratch_sizes_are_bounded_and_grow(lib):
    assert lib.odie_sort_rows_scratch(4096, 1 << 20) == 0  # one block
    assert 0 < lib.odie_sort_rows_scratch(4097, 16) < lib.odie_sort_rows_scratch(1 << 20, 16) <= 4 * (1 << 20)
    assert lib.odie_sort_rows_scratch(1 << 20, 1 << 16) >= 3 * 4 * (1 << 20)  # a pair buffer and the sorted keys
    assert lib.odie_embed_backward_scratch(1 << 16, 1 << 16, 1024) > lib.odie_embed_backward_scratch(1 << 16, 1 << 16, 32)
