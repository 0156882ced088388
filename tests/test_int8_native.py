"""The 8-bit operators' native parts fit each other (no GPU needed): declarations, prototypes and the extension's build."""
import ctypes
import re
from pathlib import Path

import pytest

from triton_client_amd import _build
from triton_client_amd.ops import _bind

HIP = Path(_build.CSRC) / "hip"

_C_TYPES = {"int": ctypes.c_int, "long long": ctypes.c_longlong, "double": ctypes.c_double, "float": ctypes.c_float}


def _declared():
    """``{name: (result, [arguments])}`` of the 8-bit operators' functions as kernels.h declares them, in ctypes' types."""
    text = re.sub(r"//[^\n]*", "", (HIP / "kernels.h").read_text())
    found = {}
    for result, name, args in re.findall(r"([\w ]+?)\s+(tca_int8_\w+)\(([^)]*)\);", text):
        types = []
        for arg in args.split(","):
            words = arg.replace("const ", "").strip()
            types.append(ctypes.c_void_p if "*" in words else _C_TYPES[words.rsplit(" ", 1)[0]])
        found[name] = (_C_TYPES[result.strip()], types)
    return found


class _Function:
    restype, argtypes = None, None


class _Library:
    """Takes the prototypes in the place of the loaded library."""

    def __init__(self):
        self.functions = {}

    def __getattr__(self, name):
        return self.functions.setdefault(name, _Function())


def test_prototypes_are_the_declared_ones():
    library = _Library()
    _bind.install(library)
    declared = _declared()
    assert len(declared) >= 5
    for name, (result, args) in declared.items():
        function = library.functions[name]
        assert function.restype is result and list(function.argtypes) == args, name


def test_the_extension_calls_what_is_declared():
    """No signature of its own, and built again when the declarations change."""
    source = (Path(_build.CSRC) / "capi" / "torch_ops.cc").read_text()
    assert '#include "kernels.h"' in source and "(*)(const void" not in source
    for name in _declared():
        if name in source:
            variable = re.search(rf"decltype\(&{name}\) (\w+);", source).group(1)
            assert f'{{"{name}", Set<{variable}>}}' in source  # the address of that name goes there


def test_the_extension_takes_all_addresses_or_none():
    pytest.importorskip("torch")
    from triton_client_amd import _native

    ops = _native.torch_ops()
    assert set(ops.launchers) <= set(_declared())
    with pytest.raises(TypeError):
        ops.use(*range(len(ops.launchers) - 1))
    with pytest.raises(TypeError):
        ops.use(*[0] * (len(ops.launchers) - 1), "address")


def test_the_extension_depends_on_the_declarations(monkeypatch):
    pytest.importorskip("torch")
    seen = []
    monkeypatch.setattr(_build, "_stale", lambda out, sources: seen.extend(sources))
    _build.build_torch()
    assert HIP / "kernels.h" in seen
