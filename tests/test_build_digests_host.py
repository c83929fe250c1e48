"""Every header of this repository that a built file includes is part of the digest it carries: an edit makes the build stale."""
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
