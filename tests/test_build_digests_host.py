"""Builds: every header of this repository that a built file includes is part of the digest it carries, so that an edit makes the
build stale; without a host compiler the libraries of the step are built all the same."""
import os
import re

import pytest

from elixir_amd import _abi, _ops_abi, _torch_ext, build as B

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def included(path, seen):
    """The files of this repository that ``path`` includes, directly or not."""
    for name in re.findall(r'^\s*#include\s+"([^"]+)"', open(path).read(), re.M):
        for base in (os.path.dirname(path), os.path.join(ROOT, 'include')):
            at = os.path.normpath(os.path.join(base, name))
            if os.path.exists(at):
                if at not in seen:
                    seen.add(at)
                    included(at, seen)
                break
    return seen


@pytest.mark.parametrize('sources,digested', [(B.SOURCES, _abi.source_files), (B.OPS_SOURCES, _ops_abi.source_files),
                                              ([_torch_ext.SOURCE], _torch_ext.source_files)])
def test_the_digest_covers_every_source_and_header(sources, digested):
    files = {os.path.normpath(f) for f in digested()}
    for source in sources:
        assert os.path.normpath(source) in files
        assert included(source, set()) <= files, included(source, set()) - files


def test_an_edited_header_makes_the_extension_stale(monkeypatch, tmp_path):
    files = _torch_ext.source_files()
    assert not B.is_stale()
    for i, name in enumerate(files):
        copy = tmp_path / os.path.basename(name)
        copy.write_bytes(open(name, 'rb').read() + b'\n')
        monkeypatch.setattr(_torch_ext, 'source_files', lambda i=i, copy=str(copy): files[:i] + [copy] + files[i + 1:])
        assert B.is_stale()


def test_the_libraries_are_built_without_a_host_compiler(monkeypatch, capsys):
    """The step with 32-bit moments needs hipcc alone, as before there was an extension."""
    ran = []

    class Done:
        returncode = 0

        def __init__(self, cmd, **kw):
            ran.append(cmd[0])

        def communicate(self):
            return '', None

    monkeypatch.setattr(B.subprocess, 'Popen', Done)
    monkeypatch.setattr(B.subprocess, 'run', lambda cmd, **kw: ran.append(cmd[0]))
    which = B.shutil.which
    monkeypatch.setattr(B.shutil, 'which', lambda name: None if name == 'g++' else which(name))
    assert B.build(verbose=False) == B.OUTPUT
    assert len(ran) == 2 and 'g++' not in ran and 'layer_norm' in capsys.readouterr().err
    # nothing that could be built is stale; loading the extension is refused by itself
    monkeypatch.setattr(_torch_ext, 'stamp', lambda: 'other')
    assert not B.is_stale()
    monkeypatch.setattr(_torch_ext, '_ext', None)
    with pytest.raises(RuntimeError, match='missing or was built from something else'):
        _torch_ext.load()
