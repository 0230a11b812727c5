"""CPU: what the row operators refuse, and how they are built, beyond test_rows.py."""
import subprocess
import sys
from pathlib import Path

import pytest

from odie_b200 import _lib

ROOT = Path(__file__).resolve().parents[1]


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


WITHOUT_TORCH = """
import sys
class Hidden:
    def find_spec(self, name, path=None, target=None):
        if name.split('.')[0] == 'torch':
            raise ModuleNotFoundError(name)
sys.meta_path.insert(0, Hidden())
import odie_b200
from odie_b200 import builder
from pathlib import Path
builder.TORCH_OPS = Path(sys.argv[1]) / '_torch_ops.so'
assert odie_b200.build() == builder.LIBRARY and builder.LIBRARY.exists() and not builder.TORCH_OPS.exists()
odie_b200.library()
"""


def test_the_library_is_built_without_torch(lib, tmp_path):
    run = subprocess.run([sys.executable, '-c', WITHOUT_TORCH, str(tmp_path)], capture_output=True, text=True, cwd=ROOT)
    assert run.returncode == 0, run.stderr
    assert 'not built' in run.stderr


def test_the_library_is_built_without_torch_headers(lib, tmp_path, monkeypatch, capsys):
    from odie_b200 import builder
    assert builder.torch_headers()
    monkeypatch.setattr(builder, 'TORCH_OPS', tmp_path / '_torch_ops.so')
    monkeypatch.setattr(builder.sysconfig, 'get_paths', lambda: {'include': str(tmp_path)})
    assert builder.build() == builder.LIBRARY and not builder.TORCH_OPS.exists()
    assert 'not built' in capsys.readouterr().err


def test_torch_ops_of_another_torch_are_stale(lib, monkeypatch):
    """The file is built again after torch has changed, whatever the files' times say."""
    import importlib.metadata
    from odie_b200 import builder
    assert not builder.torch_ops_stale()
    with monkeypatch.context() as m:
        m.setattr(importlib.metadata, 'version', lambda name: '0.0.1')
        assert builder.torch_ops_stale()
        built = []
        m.setattr(builder, 'build_torch_ops', lambda: built.append(True))
        builder.build()
        assert built
    assert not builder.torch_ops_stale()


def test_linear_scratch_is_what_the_call_uses(lib):
    """Nothing for one or two rows without offsets, the weights' sums alone behind thin layers; at most the general size."""
    for rows, inputs, outputs, groups in ((1, 4097, 8192, 1), (2, 333, 515, 1), (1 << 20, 32, 64, 1), (1 << 20, 64, 64, 16), (700, 333, 72, 5),
                                          (64, 4096, 4096, 1)):
        most, most_back = lib.odie_linear_scratch(rows, inputs, outputs, groups), lib.odie_linear_backward_scratch(rows, inputs, outputs, groups)
        for offsets in (0, 1):
            for on_16 in (0, 1):
                size, back = lib.odie_linear_scratch_for(rows, inputs, outputs, groups, offsets, on_16), lib.odie_linear_backward_scratch_for(rows, inputs, outputs, groups, on_16)
                thin = on_16 and inputs <= 64 and outputs <= 64
                assert size == (0 if thin or (rows <= 2 and not offsets) else most)
                assert 0 < back <= most_back and (not thin or back <= 4 * (148 * 4 + groups + 1) * (inputs + 1) * outputs + 256)
    assert lib.odie_linear_scratch_for(8, 0, 8, 1, 0, 1) == 0 and lib.odie_linear_backward_scratch_for(8, 8, 8, 1025, 1) == 0
