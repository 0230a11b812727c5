"""CPU: what the row operators refuse, and how they are built, beyond test_rows.py."""
import pytest

from odie_b200 import _lib


@pytest.fixture(scope='module')
def lib():
    from odie_b200 import builder
    builder.build()
    return _lib.library()


def test_linear_wait_limit_refuses(lib):
    for polls in (-2, (1 << 22) + 1):
        assert lib.odie_linear_wait_limit(polls) == -1
        assert 'polls' in _lib.error()
    assert lib.odie_linear_wait_limit(0) == 0 and lib.odie_linear_wait_limit(-1) == 0


def test_linear_check_without_a_device(lib):
    import torch
    if not torch.cuda.is_available():  # an error, not an abort
        assert lib.odie_linear_check() == -1 and _lib.error()
