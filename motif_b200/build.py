"""Build `libmotif_b200.so` (all CUDA kernels + the C ABI) in-tree for sm_100a, and `_paged_host.so`
(the compiled Python entry points of the paged cache, on the same C ABI) beside it.

    python -m motif_b200.build [--force] [--jobs N] [--lib-only]

Each `csrc/*.cu` is compiled to an object in `_build/` with
`-gencode arch=compute_100a,code=sm_100a`, then linked into
`motif_b200/libmotif_b200.so` next to this file.  Rebuilds only when a source or
header is newer than the library (the host module: its source or the C header).  A user of the C ABI
alone needs neither Python's headers nor a C++ compiler for torch's: `--lib-only` leaves the module out.
"""

import argparse
import concurrent.futures as cf
import glob
import os
import shutil
import subprocess
import sys
import sysconfig

HERE = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(HERE)
CSRC = os.path.join(HERE, 'csrc')
BUILD = os.path.join(ROOT, '_build')
LIB = os.path.join(HERE, 'libmotif_b200.so')
HOST_SRC = os.path.join(CSRC, 'paged_host.cpp')
HOST = os.path.join(HERE, '_paged_host.so')
HEADER = os.path.join(ROOT, 'include', 'motif_b200.h')

ARCH = ['-gencode', 'arch=compute_100a,code=sm_100a']
NVCC_FLAGS = ['-O3', '-std=c++17', '-lineinfo', '-Xcompiler', '-fPIC', '-Xcompiler', '-fvisibility=hidden',
              '--expt-relaxed-constexpr', f'-I{os.path.join(ROOT, "include")}']


def nvcc() -> str:
    for cand in (os.environ.get('NVCC'), shutil.which('nvcc'), '/usr/local/cuda/bin/nvcc'):
        if cand and os.path.exists(cand):
            return cand
    raise RuntimeError('nvcc not found: set NVCC or put the CUDA toolkit on PATH')


def sources():
    return sorted(glob.glob(os.path.join(CSRC, '*.cu')))


def _stale() -> bool:
    if not os.path.exists(LIB):
        return True
    t = os.path.getmtime(LIB)
    deps = sources() + glob.glob(os.path.join(CSRC, '*.cuh')) + [HEADER]
    return any(os.path.getmtime(p) > t for p in deps)


def _compile(src: str) -> str:
    obj = os.path.join(BUILD, os.path.basename(src) + '.o')
    cmd = [nvcc(), *ARCH, *NVCC_FLAGS, '-c', src, '-o', obj]
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f'nvcc failed on {src}:\n{r.stderr}')
    return obj


def _build_host(force: bool) -> None:
    """Compile `_paged_host.so` against torch's headers and link it to the library beside it."""
    deps = (HOST_SRC, HEADER)
    if not force and os.path.exists(HOST) and all(os.path.getmtime(p) <= os.path.getmtime(HOST) for p in deps):
        return
    import torch
    root = os.path.dirname(torch.__file__)
    cuda = os.path.dirname(os.path.dirname(nvcc()))
    include = [sysconfig.get_paths()['include'], os.path.join(root, 'include'),
               os.path.join(root, 'include', 'torch', 'csrc', 'api', 'include'), os.path.join(cuda, 'include')]
    tmp = HOST + '.tmp'
    cmd = [os.environ.get('CXX', 'g++'), '-O2', '-std=c++17', '-fPIC', '-shared', '-fvisibility=hidden',
           f'-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}', *[f'-I{p}' for p in include], HOST_SRC,
           '-o', tmp, f'-L{HERE}', '-l:libmotif_b200.so', '-Wl,-rpath,$ORIGIN', f'-L{os.path.join(root, "lib")}',
           '-ltorch_python', '-ltorch', '-ltorch_cpu', '-ltorch_cuda', '-lc10', '-lc10_cuda']
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f'{cmd[0]} failed on {HOST_SRC}:\n{r.stderr}')
    os.replace(tmp, HOST)


def build(force: bool = False, jobs: int = 0, verbose: bool = False, host: bool = True) -> str:
    """Compile every kernel and link the shared library and (with `host`) the host module; returns the
    library's path."""
    if force or _stale():
        _build_lib(jobs)
        if verbose:
            print(f'built {LIB}')
    if host:
        _build_host(force)
    return LIB


def _build_lib(jobs: int) -> None:
    os.makedirs(BUILD, exist_ok=True)
    srcs = sources()
    jobs = jobs or min(len(srcs), os.cpu_count() or 4)
    with cf.ThreadPoolExecutor(max_workers=jobs) as ex:
        objs = list(ex.map(_compile, srcs))
    tmp = LIB + '.tmp'
    cmd = [nvcc(), *ARCH, '-shared', '-Xcompiler', '-fPIC', *objs, '-o', tmp, '-lcudart']
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f'link failed:\n{r.stderr}')
    os.replace(tmp, LIB)


def main():
    ap = argparse.ArgumentParser()
    ap.add_argument('--force', action='store_true')
    ap.add_argument('--jobs', type=int, default=0)
    ap.add_argument('--lib-only', action='store_true')
    a = ap.parse_args()
    build(force=a.force, jobs=a.jobs, verbose=True, host=not a.lib_only)


if __name__ == '__main__':
    sys.exit(main())
