"""Loads ``_elx_torch.so``: autograd of ``layer_norm`` and ``embedding`` over the C ABI of ``libelx_ops.so``, compiled against
the torch that is installed (``elixir_amd/csrc/torch/elx_torch.cpp``).  One that is missing, was built from other sources or
for another torch raises; there is no other implementation."""
import hashlib
import os
import re

import torch

_HERE = os.path.dirname(os.path.abspath(__file__))
LIB_PATH = os.path.join(_HERE, '_elx_torch.so')
SOURCE = os.path.join(_HERE, 'csrc', 'torch', 'elx_torch.cpp')


def source_files():
    """What the extension is made from, in the order of the digest: its source and the headers it calls through."""
    include = os.path.join(os.path.dirname(_HERE), 'include')
    return [SOURCE] + [os.path.join(include, f) for f in ('elx_ops.h', 'elx_abi.h')]


def stamp() -> str:
    """What a build carries: the digest of its sources, and the version of torch."""
    h = hashlib.sha256()
    for path in source_files():
        with open(path, 'rb') as f:
            h.update(f.read())
    return f'{h.hexdigest()[:16]} torch {torch.__version__}'


def built_stamp(path: str) -> str:
    """The stamp in a built file ('' when there is none), read without loading it."""
    try:
        with open(path, 'rb') as f:
            found = re.search(rb'elx_torch built from \[([^\]]*)\]', f.read())
    except OSError:
        return ''
    return found.group(1).decode() if found else ''


_ext = None


def load():
    global _ext
    if _ext is None:
        built, now = built_stamp(LIB_PATH), stamp()
        if built != now:
            raise RuntimeError(f'{LIB_PATH} is missing or was built from something else ({built or "nothing"}) than what is here '
                               f'({now}): run `python -m elixir_amd.build`')
        from . import _elx_torch
        _ext = _elx_torch
    return _ext
