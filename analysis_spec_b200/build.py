"""Builds libspeckv.so (all CUDA sources under csrc/) for sm_100a with nvcc, and the CPython
module _front.so (csrc/front.cpp, the torch front end of the decode-step operators) with g++.

Both are built in-tree next to this file so that they ship with the
package. A rebuild happens only when a source, header or flag changed (a hash
of them is kept beside the library).
"""
import hashlib
import os
import subprocess
import sys
from concurrent.futures import ThreadPoolExecutor
from pathlib import Path

HERE = Path(__file__).resolve().parent
CSRC = HERE / 'csrc'
INCLUDE = HERE.parent / 'include'
LIB = HERE / 'libspeckv.so'
FRONT = HERE / '_front.so'
OBJDIR = HERE / '_build'

CXX = os.environ.get('CXX', 'g++')
NVCC = os.environ.get('NVCC', '/usr/local/cuda/bin/nvcc')
ARCH = ['-gencode', 'arch=compute_100a,code=sm_100a']
FLAGS = ['-O3', '-std=c++17', '-lineinfo', '-Xcompiler', '-fPIC', '-Xcompiler', '-O2',
         '--expt-relaxed-constexpr', '-I', str(INCLUDE)]


def _sources():
    return sorted(CSRC.glob('*.cu'))


def _digest():
    h = hashlib.sha256()
    h.update(' '.join(ARCH + FLAGS).encode())
    for path in sorted([p for p in CSRC.glob('*') if p.suffix != '.cpp'] + list(INCLUDE.glob('*.h'))):
        if path.is_file():
            h.update(path.name.encode())
            h.update(path.read_bytes())
    return h.hexdigest()


def build(force=False, verbose=False):
    """Compile and link libspeckv.so and _front.so; returns the library's path."""
    stamp = LIB.with_suffix('.so.hash')
    digest = _digest()
    if not force and LIB.exists() and stamp.exists() and stamp.read_text() == digest:
        build_front(force, verbose)
        return LIB
    OBJDIR.mkdir(exist_ok=True)

    def compile_one(src):
        obj = OBJDIR / (src.stem + '.o')
        cmd = [NVCC, *ARCH, *FLAGS, '-c', str(src), '-o', str(obj)]
        if verbose:
            print(' '.join(cmd), file=sys.stderr)
        proc = subprocess.run(cmd, capture_output=True, text=True)
        if proc.returncode != 0:
            raise RuntimeError(f'nvcc failed on {src.name}:\n{proc.stdout}\n{proc.stderr}')
        return obj

    with ThreadPoolExecutor(max_workers=min(8, os.cpu_count() or 1)) as pool:
        objs = list(pool.map(compile_one, _sources()))
    tmp = LIB.with_suffix('.so.tmp')
    cmd = [NVCC, *ARCH, '-shared', '-o', str(tmp), *map(str, objs)]
    proc = subprocess.run(cmd, capture_output=True, text=True)
    if proc.returncode != 0:
        raise RuntimeError(f'nvcc link failed:\n{proc.stdout}\n{proc.stderr}')
    os.replace(tmp, LIB)
    stamp.write_text(digest)
    build_front(force, verbose)
    return LIB


def build_front(force=False, verbose=False):
    """Compile and link _front.so against the installed torch and libspeckv.so; returns its path."""
    import sysconfig

    import torch
    include = Path(torch.__file__).resolve().parent / 'include'
    libdir = Path(torch.__file__).resolve().parent / 'lib'
    src = CSRC / 'front.cpp'
    cmd = [CXX, '-std=c++17', '-O2', '-fPIC', '-shared', '-fvisibility=hidden', '-DTORCH_API_INCLUDE_EXTENSION_H',
           f'-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}', '-isystem', str(include), '-isystem',
           str(include / 'torch' / 'csrc' / 'api' / 'include'), '-isystem', str(Path(NVCC).parent.parent / 'include'),
           '-isystem', sysconfig.get_paths()['include'], str(src), '-o', str(FRONT.with_suffix('.so.tmp')),
           f'-L{libdir}', '-lc10', '-lc10_cuda', '-ltorch_cuda', '-ltorch_cpu', '-ltorch', '-ltorch_python', f'-L{HERE}',
           f'-l:{LIB.name}', '-Wl,-rpath,$ORIGIN']
    h = hashlib.sha256(' '.join(cmd + [torch.__version__]).encode())
    for path in (src, INCLUDE / 'speckv.h'):
        h.update(path.read_bytes())
    stamp = FRONT.with_suffix('.so.hash')
    if not force and FRONT.exists() and stamp.exists() and stamp.read_text() == h.hexdigest():
        return FRONT
    if verbose:
        print(' '.join(cmd), file=sys.stderr)
    proc = subprocess.run(cmd, capture_output=True, text=True)
    if proc.returncode != 0:
        raise RuntimeError(f'{CXX} failed on {src.name}:\n{proc.stdout}\n{proc.stderr}')
    os.replace(FRONT.with_suffix('.so.tmp'), FRONT)
    stamp.write_text(h.hexdigest())
    return FRONT


if __name__ == '__main__':
    print(build(force='--force' in sys.argv, verbose='-v' in sys.argv))
