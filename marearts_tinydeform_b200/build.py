"""Build the native library in-tree: nvcc -> marearts_tinydeform_b200/_tinydeform.so (sm_100a only).

The library is a plain C-ABI shared object (include/tinydeform.h) with no torch headers; Python reaches it through
ctypes (``_native.py``). It is rebuilt when any source under csrc/ or the public header is newer than the .so.

    python -m marearts_tinydeform_b200.build [--force]
"""

import concurrent.futures
import os
import subprocess
import sys
import tempfile

HERE = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(HERE)
CSRC = os.path.join(HERE, 'csrc')
HEADER = os.path.join(ROOT, 'include', 'tinydeform.h')
LIB = os.path.join(HERE, '_tinydeform.so')
# the checked build: every corner token re-tested against [0, N) where a kernel reads or writes its row (tests only)
DEBUG_LIB = os.path.join(HERE, '_tinydeform_debug.so')
ARCH = ['-gencode', 'arch=compute_100a,code=sm_100a']


def _nvcc():
    for cand in (os.environ.get('NVCC'), '/usr/local/cuda/bin/nvcc'):
        if cand and os.path.exists(cand):
            return cand
    return 'nvcc'


def sources():
    return sorted(os.path.join(CSRC, f) for f in os.listdir(CSRC) if f.endswith(('.cu', '.cuh', '.h')))


def stale(lib=LIB):
    if not os.path.exists(lib):
        return True
    built = os.path.getmtime(lib)
    return any(os.path.getmtime(p) > built for p in sources() + [HEADER, __file__])


def _run(cmd):
    print(' '.join(cmd), file=sys.stderr)
    subprocess.run(cmd, check=True)


def build(force=False, verbose=False, debug=False):
    """Compile every csrc/*.cu, each a translation unit of its own, side by side, and link them into _tinydeform.so
    (debug: the checked _tinydeform_debug.so, -DTD_DEBUG_BOUNDS) if it is missing or stale; return the library path."""
    lib = DEBUG_LIB if debug else LIB
    if not force and not stale(lib):
        return lib
    flags = [*ARCH, '-O3', '-lineinfo', '-std=c++17', '--expt-relaxed-constexpr',
             '-Xcompiler', '-fPIC,-O3,-fvisibility=hidden', '-I' + os.path.join(ROOT, 'include')]
    if debug:
        flags.insert(0, '-DTD_DEBUG_BOUNDS')
    if verbose:
        flags.insert(0, '-Xptxas=-v')
    with tempfile.TemporaryDirectory() as objects:
        units = [p for p in sources() if p.endswith('.cu')]
        outs = [os.path.join(objects, os.path.basename(p)[:-3] + '.o') for p in units]
        with concurrent.futures.ThreadPoolExecutor(len(units)) as pool:
            list(pool.map(_run, [[_nvcc(), *flags, '-c', p, '-o', o] for p, o in zip(units, outs)]))
        tmp = lib + '.tmp'
        _run([_nvcc(), *ARCH, '-shared', *outs, '-o', tmp])
    os.replace(tmp, lib)
    return lib


if __name__ == '__main__':
    build(force='--force' in sys.argv, verbose='-v' in sys.argv)
    if '--debug' in sys.argv:
        build(force='--force' in sys.argv, verbose='-v' in sys.argv, debug=True)
