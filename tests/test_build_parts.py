"""The library can be built without the compiled Python module (no GPU, nothing is compiled)."""

import sys

import pytest

from motif_b200 import build


def test_library_alone_needs_no_python_headers(monkeypatch):
    def missing(force):
        raise RuntimeError('g++ failed: Python.h: No such file or directory')

    monkeypatch.setattr(build, '_stale', lambda: False)
    monkeypatch.setattr(build, '_build_host', missing)
    with pytest.raises(RuntimeError, match='Python.h'):   # never left out unasked
        build.build()
    assert build.build(host=False) == build.LIB
    monkeypatch.setattr(sys, 'argv', ['build', '--lib-only'])
    build.main()
