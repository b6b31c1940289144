"""CPU tests of the build: what it compiles, and what it does where a part fails."""
import os

import pytest

from ddq_b200 import build as b


def test_the_library_is_built_where_the_module_on_torch_does_not_build(monkeypatch, tmp_path):
    """A user of the C ABI needs no Python headers and no host compiler for torch's."""
    made = []
    monkeypatch.setattr(b, "is_stale", lambda: False)
    lib = b.LIB_PATH

    def broken(force=False):
        made.append(os.path.exists(lib))
        raise RuntimeError("no Python.h")
    b.build()
    monkeypatch.setattr(b, "build_torch", broken)
    with pytest.warns(RuntimeWarning, match="ddq_b200.paged is not available: no Python.h"):
        assert b.build() == lib
    assert made == [True]
