"""CPU tests of the build: what it compiles, and what it does where a part fails."""
import os
import sysconfig

import pytest
import torch

from ddq_b200 import _lib, build as b


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


@pytest.mark.parametrize("other", ["torch", "cuda", "source", "python"])
def test_a_module_of_another_torch_or_python_is_not_taken(monkeypatch, other):
    """The module is compiled on both's headers: it is neither fresh nor loaded elsewhere."""
    b.build_torch()
    here = b.torch_path()
    assert os.path.exists(here)
    if other == "torch":
        monkeypatch.setattr(torch, "__version__", "9.9.9+cu999")
    elif other == "cuda":
        monkeypatch.setattr(torch.version, "cuda", "99.9")
    elif other == "source":
        monkeypatch.setattr(torch.version, "git_version", "f" * 40)
    else:
        monkeypatch.setattr(sysconfig, "get_config_var", lambda name: ".cpython-999.so")
    assert b.torch_path() != here

    def compiler(cmd, **kw):
        raise OSError("the module would be compiled")
    monkeypatch.setattr(b.subprocess, "run", compiler)
    with pytest.raises(OSError, match="would be compiled"):
        b.build_torch()
    monkeypatch.setattr(_lib, "_paged", None)
    with pytest.raises(RuntimeError, match="not found; build it"):
        _lib.load_paged()


def test_the_reference_modules_need_a_whole_checkout_or_none(monkeypatch, tmp_path):
    """No checkout, or an empty one, is skipped; one that lacks a file is an error."""
    from oracle import build_ref as r
    monkeypatch.setattr(r, "REF_OUT", str(tmp_path / "out"))

    def no_build(*a, **kw):
        raise AssertionError("nothing is compiled here")
    monkeypatch.setattr(r.subprocess, "Popen", no_build)
    assert r.build(str(tmp_path / "absent")) == []
    some = tmp_path / "checkout"
    some.mkdir()
    assert r.build(str(some)) == []
    names = list(r.MODULES.values())
    (some / names[1]).write_text("")
    with pytest.raises(FileNotFoundError, match=names[0]):
        r.build(str(some))
