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


class _OtherTorch:
    """An extension that loads, built for another torch."""

    built_for = "1.0.0 0123456789"
    launchers = ("tca_int8_quantize_launch",)

    @staticmethod
    def use(*addresses):
        raise AssertionError("it must not be used")


@pytest.mark.parametrize("names_it", [True, False])
def test_an_extension_for_another_torch_is_left_alone(monkeypatch, names_it):
    torch = pytest.importorskip("torch")
    from triton_client_amd import _lib, _native
    from triton_client_amd.ops import int8

    if not names_it:
        monkeypatch.delattr(_OtherTorch, "built_for")
    monkeypatch.setattr(_native, "_torch_ops", None)
    monkeypatch.setattr(_lib, "_tca_torch", _OtherTorch, raising=False)
    with pytest.raises(ImportError, match="was built for torch"):
        _native.torch_ops()
    # the operators then go their general way
    monkeypatch.setattr(int8, "_plain", None)
    with pytest.warns(RuntimeWarning, match="was built for torch"), pytest.raises(ValueError, match="CUDA"):
        int8.quantize_int8(torch.zeros(2, 8))


def test_the_extension_is_built_again_for_another_torch(monkeypatch, tmp_path):
    """Also where its file is newer than that torch's."""
    torch = pytest.importorskip("torch")
    built = []
    monkeypatch.setattr(_build, "LIBDIR", tmp_path)
    monkeypatch.setattr(_build, "_compile_atomic", lambda cmd, out: (built.append(cmd), out.write_bytes(b"")))
    _build.build_torch()
    _build.build_torch()
    assert len(built) == 1 and f'-DTCA_TORCH="{torch.__version__} {torch.version.git_version}"' in built[0]
    (tmp_path / "_tca_torch.torch").write_text("1.0.0 0123456789")
    _build.build_torch()
    assert len(built) == 2
    (tmp_path / "_tca_torch.torch").unlink()
    _build.build_torch()
    assert len(built) == 3


def test_the_built_extension_names_its_torch():
    torch = pytest.importorskip("torch")
    from triton_client_amd import _native

    assert _native.torch_ops().built_for == f"{torch.__version__} {torch.version.git_version}"
