"""CPU: refusals of the router's operators and of microscaled rows, all of them on the host before any device work, and the
sizes of their scratch."""
import ctypes

import pytest
import torch

from odie_b200 import _lib, experts


@pytest.fixture(scope='module')
def lib():
    from odie_b200 import builder
    builder.build()
    return _lib.library()


def test_cpu_tensors_and_names_are_refused(lib):
    x = torch.zeros(4, 8)
    micro = experts.Micro(torch.zeros(4, 16, dtype=torch.uint8), torch.zeros(1, 1, 1, 512, dtype=torch.uint8), torch.zeros(4), 8, 16)
    for call in (lambda: experts.gate(x, 2), lambda: experts.balance(x, torch.zeros(4, dtype=torch.int32)), lambda: experts.quantize(x),
                 lambda: experts.dequantize(micro), lambda: experts.linear4(x.half(), micro)):
        with pytest.raises(ValueError, match='CUDA'):
            call()
    with pytest.raises(ValueError, match='score'):
        experts.gate(x, 2, score='tanh')
    with pytest.raises(ValueError, match='score'):
        experts.balance(x, torch.zeros(4, dtype=torch.int32), score=None)
    with pytest.raises(ValueError, match='activation'):
        experts.linear4(x.half(), micro, activation='tanh')
    with pytest.raises(ValueError, match='Micro'):
        experts.linear4(x.half(), x)
    with pytest.raises(ValueError, match='Micro'):
        experts.dequantize(x)
    for block in (0, 8, 64):
        with pytest.raises(ValueError, match='block'):
            experts.quantize(x, block=block)


# Non-null pointers that nothing reads: every call below fails its checks before it touches them.
SOME = ctypes.c_void_p(256)
NAN, INF = float('nan'), float('inf')

LOGITS = [(dict(rows=-1), 'rows'), (dict(rows=2 ** 31), 'rows'), (dict(experts=0), 'experts'), (dict(experts=1025), 'experts'),
          (dict(dtype=3), 'element type'), (dict(score=2), 'score'), (dict(score=-1), 'score')]
GATE = LOGITS + [(dict(choices=0), 'choices'), (dict(choices=9), 'choices'), (dict(experts=100, choices=65), 'choices'),
                 (dict(rows=2 ** 30, choices=2), 'pairs'), (dict(scale=0.0), 'scale'), (dict(scale=NAN), 'scale'), (dict(scale=INF), 'scale'), (dict(scale=1e-40), 'scale'),
                 (dict(expert=None), 'required'), (dict(weights=None), 'required')]


@pytest.mark.parametrize('change, message', GATE + [(dict(logits=None), 'required')])
def test_gate_refuses(lib, change, message):
    a = dict(logits=SOME, rows=4, experts=8, dtype=0, bias=None, mask=None, row_step=0, expert_step=0, choices=2, score=0, normalize=1, scale=1.0,
             expert=SOME, weights=SOME, stream=0)
    a.update(change)
    assert lib.odie_gate(*a.values()) == -1
    assert message in _lib.error()


@pytest.mark.parametrize('change, message', GATE + [(dict(d_weights=None), 'required'), (dict(d_logits=None), 'required'),
                                                    (dict(logits=None, score=1), 'logits'), (dict(logits=None, normalize=0), 'logits')])
def test_gate_backward_refuses(lib, change, message):
    a = dict(d_weights=SOME, logits=SOME, rows=4, experts=8, dtype=0, mask=None, row_step=0, expert_step=0, expert=SOME, weights=SOME, choices=2,
             score=0, normalize=1, scale=1.0, d_logits=SOME, stream=0)
    a.update(change)
    assert lib.odie_gate_backward(*a.values()) == -1
    assert message in _lib.error()


@pytest.mark.parametrize('change, message', LOGITS + [
    (dict(key_bytes=2), 'int32 or int64'), (dict(pairs=-1), 'pairs'), (dict(pairs=2 ** 31), 'pairs'), (dict(logits=None), 'required'),
    (dict(expert=None), 'required'), (dict(rows=0), 'without rows'), (dict(loss=None), 'required'), (dict(z=None), 'required'),
    (dict(counts=None), 'required'), (dict(stats=None), 'required'), (dict(scratch=None), 'scratch'), (dict(scratch=ctypes.c_void_p(16)), '256-byte')])
def test_balance_refuses(lib, change, message):
    a = dict(logits=SOME, rows=4, experts=8, dtype=0, mask=None, row_step=0, expert_step=0, score=0, expert=SOME, key_bytes=4, pairs=8, total=None,
             loss=SOME, z=SOME, counts=SOME, stats=SOME, scratch=SOME, stream=0)
    a.update(change)
    assert lib.odie_balance(*a.values()) == -1
    assert message in _lib.error()


@pytest.mark.parametrize('change, message', LOGITS + [(dict(logits=None), 'required'), (dict(stats=None), 'required'), (dict(d_logits=None), 'required')])
def test_balance_backward_refuses(lib, change, message):
    a = dict(d_loss=SOME, d_z=SOME, logits=SOME, rows=4, experts=8, dtype=0, mask=None, row_step=0, expert_step=0, score=0, stats=SOME, d_logits=SOME,
             stream=0)
    a.update(change)
    assert lib.odie_balance_backward(*a.values()) == -1
    assert message in _lib.error()


MICRO = [(dict(groups=0), 'rows'), (dict(rows=-1), 'rows'), (dict(rows=2 ** 31), 'rows'), (dict(groups=2 ** 20, rows=2 ** 12), 'rows'),
         (dict(groups=2 ** 25, rows=1), 'tiles'), (dict(width=0), 'columns'), (dict(width=(1 << 20) + 1), 'columns'), (dict(dtype=3), 'element type'),
         (dict(block=64), 'block'), (dict(block=0), 'block'), (dict(codes=None), 'required'), (dict(scales=None), 'required'),
         (dict(row_scales=None), 'required'), (dict(codes=ctypes.c_void_p(8)), '16-byte'), (dict(scales=ctypes.c_void_p(8)), '16-byte')]


@pytest.mark.parametrize('change, message', MICRO + [(dict(x=None), 'required')])
def test_quantize_refuses(lib, change, message):
    a = dict(x=SOME, groups=1, rows=4, width=8, dtype=0, block=16, codes=SOME, scales=SOME, row_scales=SOME, stream=0)
    a.update(change)
    assert lib.odie_quantize(*a.values()) == -1
    assert message in _lib.error()


@pytest.mark.parametrize('change, message', MICRO + [(dict(out=None), 'required')])
def test_dequantize_refuses(lib, change, message):
    a = dict(codes=SOME, scales=SOME, row_scales=SOME, groups=1, rows=4, width=8, block=16, dtype=0, out=SOME, stream=0)
    a.update(change)
    assert lib.odie_dequantize(*a.values()) == -1
    assert message in _lib.error()


@pytest.mark.parametrize('change, message', [
    (dict(rows=-1), 'rows'), (dict(rows=2 ** 31), 'rows'), (dict(inputs=0), 'inputs'), (dict(outputs=0), 'outputs'), (dict(inputs=(1 << 20) + 1), 'inputs'),
    (dict(groups=0), 'groups'), (dict(groups=1025, offsets=SOME), 'groups'), (dict(groups=2), 'offsets'), (dict(dtype=2), 'fp16'), (dict(block=8), 'blocks'),
    (dict(activation=4), 'activation'), (dict(x=None), 'required'), (dict(codes=None), 'required'), (dict(scales=None), 'required'),
    (dict(row_scales=None), 'required'), (dict(y=None), 'required'), (dict(scratch=None), 'scratch'), (dict(scratch=ctypes.c_void_p(16)), '256-byte'),
    (dict(codes=ctypes.c_void_p(8)), '16-byte')])
def test_linear4_refuses(lib, change, message):
    a = dict(x=SOME, codes=SOME, scales=SOME, row_scales=SOME, block=16, bias=None, residual=None, rows=8, inputs=8, outputs=8, groups=1, offsets=None,
             dtype=0, activation=0, y=SOME, scratch=SOME, stream=0)
    a.update(change)
    assert lib.odie_linear4(*a.values()) == -1
    assert message in _lib.error()


def test_scratch_sizes(lib):
    assert lib.odie_balance_scratch(0, 8) == 0 and lib.odie_balance_scratch(-1, 8) == 0 and lib.odie_balance_scratch(8, 1025) == 0
    assert 0 < lib.odie_balance_scratch(1, 8) <= lib.odie_balance_scratch(1 << 20, 8) <= lib.odie_balance_scratch(2 ** 31 - 1, 8) < 1 << 22
    for block in (16, 32):
        for offsets in (0, 1):  # codes, scales and row scales of the rows, at least
            for rows, inputs in ((1, 1), (129, 333), (4096, 1024)):
                size = lib.odie_linear4_scratch(rows, inputs, 512, 1, offsets, block)
                if rows <= 2 and not offsets:  # one kernel, which keeps them to itself
                    assert size == 0
                    continue
                assert size >= rows * (-(-inputs // 32) * 16 + 4) + -(-rows // 128) * -(-inputs // (4 * block)) * 512
    assert lib.odie_linear4_scratch(2, 1 << 20, 512, 1, 0, 16) > 0  # too long for it
    assert lib.odie_linear4_scratch(8, 8, 8, 1, 0, 24) == 0 and lib.odie_linear4_scratch(8, 0, 8, 1, 0, 16) == 0
