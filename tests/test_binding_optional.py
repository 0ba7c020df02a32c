"""A runtime does not need the compiled binding, and never loads one that was built for another torch or Python."""
import ctypes
import os
import sysconfig

import pytest
import torch


class Library:
    """The library with a runtime that needs no device and entry points that record."""

    def __init__(self, lib):
        self._lib, self.seen = lib, []

    def __getattr__(self, name):
        return getattr(self._lib, name)

    def pw_runtime_create(self, device, flags, out):
        out._obj.value = 0xBEEF
        return 0

    def pw_runtime_destroy(self, rt):
        return None


@pytest.mark.parametrize("content", [None, b"not an extension"])
def test_a_runtime_without_the_binding(monkeypatch, tmp_path, content):
    from mimo_prismwing_b200 import _lib
    from mimo_prismwing_b200.runtime import WideMoeRuntime
    path = tmp_path / ("_pw_torch" + sysconfig.get_config_var("EXT_SUFFIX"))
    if content:
        path.write_bytes(content)
    library = Library(_lib.load())
    monkeypatch.setattr(_lib, "load", lambda: library)
    monkeypatch.setattr(_lib, "BINDING_PATH", str(path))
    monkeypatch.setattr(_lib, "_binding", None)
    with pytest.warns(RuntimeWarning, match="longer on the host"):
        rt = WideMoeRuntime(0)
    assert rt._calls is None

    def record(*args):
        library.seen.append(args)
        return 0

    # an asynchronous call takes the way through ctypes (host tensors stand in for the device's)
    library.pw_linear, rt.device = record, -1
    monkeypatch.setattr(WideMoeRuntime, "_mem", staticmethod(lambda where, asynchronous: (3, None)))
    out = rt.linear(torch.zeros((2, 64), dtype=torch.bfloat16), torch.zeros((8, 64), dtype=torch.bfloat16),
                    asynchronous=True).output
    assert out.shape == (2, 8) and library.seen[0][0].value == 0xBEEF
    rt.close()


def test_a_runtime_with_the_binding(monkeypatch):
    from mimo_prismwing_b200 import _lib
    from mimo_prismwing_b200.runtime import WideMoeRuntime
    library = Library(_lib.load())
    monkeypatch.setattr(_lib, "load", lambda: library)
    rt = WideMoeRuntime(0)
    assert type(rt._calls).__name__ == "Calls"
    rt.close()


def test_the_bindings_name_is_of_this_torch_and_python():
    from mimo_prismwing_b200 import _lib, build
    name = os.path.basename(_lib.BINDING_PATH)
    assert torch.__version__ in name and name.endswith(sysconfig.get_config_var("EXT_SUFFIX"))
    assert build.BINDING_PATH == _lib.BINDING_PATH
    assert ctypes.sizeof(ctypes.c_void_p) == 8  # handles go to the binding as 64-bit integers
