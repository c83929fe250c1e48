"""Builds ``libelx_hip.so`` (the optimizer step) and ``libelx_ops.so`` (the operators beside it) in-tree with hipcc for
gfx950, and ``_elx_torch.so`` (autograd over the latter, host code only) with g++ against the installed torch.

    python -m elixir_amd.build

-ffp-contract=off keeps the kernels' arithmetic to the fused multiply-adds that are written out;
packed fp32 instructions are switched off for the device pass.  The digest of the sources is compiled
in (``elx_source_sha``), so that a binding can tell a library built from other sources.
"""
import os
import shutil
import subprocess
import sys
import sysconfig

from . import _ops_abi, _torch_ext
from ._abi import LIB_PATH, built_source_sha, source_sha16

_HERE = os.path.dirname(os.path.abspath(__file__))
_ROOT = os.path.dirname(_HERE)
SOURCES = [os.path.join(_HERE, 'csrc', 'elx_kernels.hip'), os.path.join(_HERE, 'csrc', 'elx_host.cpp')]
HOST_SOURCE = os.path.join(_HERE, 'csrc', 'elx_host.cpp')
OUTPUT = LIB_PATH
OPS_SOURCES = [f for f in _ops_abi.source_files() if f.endswith(('.hip', '.cpp'))]
OPS_OUTPUT = _ops_abi.LIB_PATH

HIPCC_FLAGS = [
    '--offload-arch=gfx950', '-O3', '-std=c++17', '-fPIC', '-shared', '-ffp-contract=off', '-Xclang', '-target-feature',
    '-Xclang', '-packed-fp32-ops', '-Wno-unused-command-line-argument'
]


def hipcc_path() -> str:
    for cand in (shutil.which('hipcc'), '/opt/rocm/bin/hipcc'):
        if cand and os.path.exists(cand):
            return cand
    raise RuntimeError('hipcc not found: the HIP extension cannot be built')


def build(verbose: bool = True) -> str:
    """Compiles both libraries, side by side; returns the path of ``libelx_hip.so``."""
    head, include = [hipcc_path()] + HIPCC_FLAGS, ['-I', os.path.join(_ROOT, 'include')]
    cmds = [head + [f'-DELX_SOURCE_SHA="{source_sha16()}"'] + include + ['-o', OUTPUT] + SOURCES,
            head + [f'-DELX_OPS_SOURCE_SHA="{_ops_abi.source_sha16()}"'] + include + ['-o', OPS_OUTPUT] + OPS_SOURCES]
    procs = []
    for cmd in cmds:
        if verbose:
            print(' '.join(cmd), flush=True)
        procs.append(subprocess.Popen(cmd, stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True))
    failed = []
    for proc in procs:
        # the host pass does not know the device-only target feature and says so; that is harmless
        out = '\n'.join(l for l in proc.communicate()[0].splitlines() if 'packed-fp32-ops' not in l)
        if proc.returncode != 0:
            failed.append(f'hipcc failed ({proc.returncode}):\n{out}')
        elif verbose and out.strip():
            print(out)
    if failed:
        raise RuntimeError('\n'.join(failed))
    if torch_ext_buildable():
        build_torch_ext(verbose)
    else:    # the step with 32-bit moments does without; what needs it raises
        print('_elx_torch.so is not built: it takes g++ and the headers of torch.  layer_norm, embedding and reading 8-bit moments '
              'will raise.', file=sys.stderr, flush=True)
    return OUTPUT


def torch_ext_buildable() -> bool:
    """Whether the host compiler and the headers that the Python extension takes are here."""
    import torch
    return shutil.which('g++') is not None and os.path.isdir(os.path.join(os.path.dirname(torch.__file__), 'include'))


def build_torch_ext(verbose: bool = True) -> str:
    """The Python extension with the autograd functions; links ``libelx_ops.so`` beside it."""
    import torch
    home = os.path.dirname(torch.__file__)
    rocm = os.path.dirname(os.path.dirname(os.path.realpath(hipcc_path())))
    cmd = ['g++', '-std=c++17', '-O2', '-fPIC', '-shared', '-Wall', f'-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}',
           '-D__HIP_PLATFORM_AMD__=1', '-DUSE_ROCM', f'-DELX_TORCH_STAMP="{_torch_ext.stamp()}"',
           '-I', os.path.join(_ROOT, 'include'), '-I', sysconfig.get_paths()['include']]
    for path in (os.path.join(home, 'include'), os.path.join(home, 'include', 'torch', 'csrc', 'api', 'include'), os.path.join(rocm, 'include')):
        cmd += ['-isystem', path]
    cmd += ['-o', _torch_ext.LIB_PATH, _torch_ext.SOURCE, '-L', os.path.join(home, 'lib'), '-lc10', '-lc10_hip', '-ltorch', '-ltorch_cpu',
            '-ltorch_hip', '-ltorch_python', '-L', _HERE, '-lelx_ops', '-Wl,-rpath,$ORIGIN']
    if verbose:
        print(' '.join(cmd), flush=True)
    proc = subprocess.run(cmd, stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True)
    if proc.returncode != 0:
        raise RuntimeError(f'g++ failed ({proc.returncode}):\n{proc.stdout}')
    if verbose and proc.stdout.strip():
        print(proc.stdout)
    return _torch_ext.LIB_PATH


def build_host_checked(out_path: str, verbose: bool = False) -> str:
    """The host-only part of the library (table validators, unscale mode, LDS reservation) compiled alone
    by g++ with AddressSanitizer and UBSan, for the tests of the validators: what is accepted or refused
    there is decided by the same source file that is linked into ``libelx_hip.so``."""
    cmd = ['g++', '-std=c++17', '-O1', '-g', '-fPIC', '-shared', '-fno-omit-frame-pointer',
           '-fsanitize=address,undefined', '-fno-sanitize-recover=all', '-Wall', '-Wextra', '-Werror',
           '-I', os.path.join(_ROOT, 'include'), '-o', out_path, HOST_SOURCE]
    if verbose:
        print(' '.join(cmd), flush=True)
    subprocess.run(cmd, check=True)
    return out_path


def is_stale() -> bool:
    """A built library is missing, or was built from other sources than the ones beside it."""
    return (not os.path.exists(OUTPUT) or built_source_sha(OUTPUT) != source_sha16() or not os.path.exists(OPS_OUTPUT)
            or _ops_abi.built_source_sha(OPS_OUTPUT) != _ops_abi.source_sha16()
            or (_torch_ext.built_stamp(_torch_ext.LIB_PATH) != _torch_ext.stamp() and torch_ext_buildable()))


def ensure_built(verbose: bool = False) -> str:
    """For test runs, the smoke check and the benchmark: compiles the library when none is there or when
    the one that is there was built from other sources (an edited kernel must never be measured through
    an old binary); a library that matches its sources is loaded as it is.  The product itself never
    builds behind the caller's back: ``elixir_amd._abi.load`` raises when the library is missing or stale."""
    if is_stale():
        if os.path.exists(OUTPUT):
            print(f'{OUTPUT} was built from other sources: rebuilding', file=sys.stderr, flush=True)
        build(verbose=verbose)
    return OUTPUT


if __name__ == '__main__':
    build()
    sys.exit(0)
