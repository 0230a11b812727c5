"""Build the sm_100a shared library libodie_b200.so in-tree with nvcc, and _torch_ops.so, the torch functions over it.

The library is the product's compute path: every CUDA kernel plus the C-ABI
declared in include/odie_b200.h.  It is built next to this file so that it
travels with the repository snapshot; nothing is installed elsewhere.  The library needs no torch: where torch or its
headers are missing, it alone is built.
"""
from concurrent.futures import ThreadPoolExecutor
import importlib.metadata
import os
import subprocess
import sys
import sysconfig
from pathlib import Path

PACKAGE = Path(__file__).resolve().parent
ROOT = PACKAGE.parent
SOURCES = ['encode.cu', 'step.cu', 'mlp_tc.cu', 'router.cu', 'probe.cu', 'layout.cu', 'residual.cu', 'selection.cu',
           'synth.cu', 'hashgrid32.cu', 'sort.cu', 'dispatch.cu', 'embed.cu', 'thin.cu', 'linear.cu', 'gate.cu', 'balance.cu',
           'micro.cu', 'linear4.cu',
           'runtime.cu']
LIBRARY = PACKAGE / 'libodie_b200.so'
TORCH_OPS = PACKAGE / '_torch_ops.so'  # a Python extension module: odie_b200._torch_ops
ARCH = ['-gencode', 'arch=compute_100a,code=sm_100a']
FLAGS = ['-O3', '-std=c++17', '-lineinfo', '--expt-relaxed-constexpr', '-Xcompiler', '-fPIC',
         '-Xcompiler', '-fvisibility=hidden', '-diag-suppress', '177']


def nvcc():
    return str(Path(os.environ.get('CUDA_HOME', '/usr/local/cuda')) / 'bin' / 'nvcc')


def stale():
    if not LIBRARY.exists():
        return True
    built = LIBRARY.stat().st_mtime
    inputs = [p for p in (PACKAGE / 'csrc').glob('*') if p.suffix != '.cpp'] + [ROOT / 'include' / 'odie_b200.h', Path(__file__)]
    return any(p.stat().st_mtime > built for p in inputs)


def torch_key():
    """What _torch_ops.so is compiled against: the versions of this interpreter and of its torch (without importing it)."""
    try:
        torch = importlib.metadata.version('torch')
    except importlib.metadata.PackageNotFoundError:
        torch = 'unknown'
    return f'{sys.implementation.cache_tag} torch {torch}'


def torch_ops_key():
    """The file that says what TORCH_OPS was compiled against."""
    return PACKAGE / '_build' / (TORCH_OPS.stem + '.key')


def torch_ops_stale():
    if not TORCH_OPS.exists() or not torch_ops_key().exists() or torch_ops_key().read_text() != torch_key():
        return True
    built = TORCH_OPS.stat().st_mtime
    return any(p.stat().st_mtime > built for p in (PACKAGE / 'csrc' / 'torch_ops.cpp', ROOT / 'include' / 'odie_b200.h',
                                                   Path(__file__)))


def torch_headers():
    """Whether this interpreter can compile extensions of its torch."""
    try:
        import torch
    except ImportError:
        return False
    return ((Path(torch.__file__).parent / 'include' / 'torch' / 'extension.h').exists() and
            (Path(sysconfig.get_paths()['include']) / 'Python.h').exists())


def build_torch_ops():
    """g++ on csrc/torch_ops.cpp against this interpreter's torch; the library beside it is found by its folder."""
    import torch
    from torch.utils import cpp_extension
    include = [*cpp_extension.include_paths(), sysconfig.get_paths()['include'],
               str(Path(os.environ.get('CUDA_HOME', '/usr/local/cuda')) / 'include'), str(ROOT / 'include')]
    libs = Path(torch.__file__).parent / 'lib'
    tmp = TORCH_OPS.with_suffix('.so.tmp')
    command = ['g++', '-O2', '-std=c++17', '-shared', '-fPIC', '-fvisibility=hidden', '-DTORCH_EXTENSION_NAME=_torch_ops',
               f'-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}',
               *[flag for path in include for flag in ('-isystem', path)], str(PACKAGE / 'csrc' / 'torch_ops.cpp'), '-o', str(tmp),
               f'-L{libs}', '-lc10', '-lc10_cuda', '-ltorch', '-ltorch_cpu', '-ltorch_cuda', '-ltorch_python', f'-L{PACKAGE}',
               '-lodie_b200', '-Wl,-rpath,$ORIGIN', f'-Wl,-rpath,{libs}']
    subprocess.run(command, check=True)
    torch_ops_key().parent.mkdir(exist_ok=True)
    torch_ops_key().unlink(missing_ok=True)  # (none, rather than another file's, if this ends here)
    os.replace(tmp, TORCH_OPS)
    torch_ops_key().write_text(torch_key())


def build(force=False, verbose=False):
    if force or stale():
        build_library(verbose)
    if force or torch_ops_stale():
        if torch_headers():
            build_torch_ops()
        else:
            print(f'{TORCH_OPS.name} is not built: torch or its headers are missing', file=sys.stderr)
    return LIBRARY


def build_library(verbose=False):
    build_dir = PACKAGE / '_build'
    build_dir.mkdir(exist_ok=True)
    include = ['-I', str(PACKAGE / 'csrc'), '-I', str(ROOT / 'include')]

    def compile_source(source):
        obj = build_dir / (Path(source).stem + '.o')
        command = [nvcc(), *FLAGS, *ARCH, *include, '-c', str(PACKAGE / 'csrc' / source), '-o', str(obj)]
        if verbose:
            print(' '.join(command), file=sys.stderr)
        subprocess.run(command, check=True)
        return str(obj)
    with ThreadPoolExecutor(min(8, os.cpu_count() or 1)) as pool:  # each source is an nvcc of its own
        objects = list(pool.map(compile_source, SOURCES))
    tmp = LIBRARY.with_suffix('.so.tmp')
    subprocess.run([nvcc(), '-shared', *ARCH, *objects, '-o', str(tmp), '-lcudart'], check=True)
    os.replace(tmp, LIBRARY)


if __name__ == '__main__':
    print(build(force='--force' in sys.argv, verbose=True))
