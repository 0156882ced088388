"""Refusals of the 8-bit integer operators (no GPU needed: every one of them comes before any launch)."""
import pytest
import torch

from triton_client_amd.ops import int8

H = torch.float16


def _x(*shape, dtype=H):
    return torch.zeros(shape, dtype=dtype)


@pytest.mark.parametrize("call,error", [
    (lambda: int8.quantize_int8(_x(2, 8, dtype=torch.int32)), TypeError),
    (lambda: int8.quantize_int8(_x(2, 8, dtype=torch.float64)), TypeError),
    (lambda: int8.quantize_int8(_x()), ValueError),
    (lambda: int8.quantize_int8(_x(2, 0)), ValueError),
    (lambda: int8.quantize_int8(_x(2, 8)), ValueError),  # not on a GPU
    (lambda: int8.silu_mul_int8(_x(2, 7)), ValueError),
    (lambda: int8.silu_mul_int8(_x(2, 8)), ValueError),
    (lambda: int8.rms_norm_int8(_x(2, 8), _x(8, dtype=torch.bfloat16)), TypeError),
    (lambda: int8.rms_norm_int8(_x(2, 8), _x(7)), ValueError),
    (lambda: int8.rms_norm_int8(_x(2, 8), _x(16)[::2]), ValueError),
    (lambda: int8.rms_norm_int8(_x(2, 8), _x(8), eps=0.0), ValueError),
    (lambda: int8.rms_norm_int8(_x(2, 8), _x(8), eps=float("nan")), ValueError),
    (lambda: int8.rms_norm_int8(_x(2, 8), _x(8), eps=float("inf")), ValueError),
    (lambda: int8.rms_norm_int8(_x(2, 8), _x(8), sum_out=_x(2, 8)), ValueError),
    (lambda: int8.rms_norm_int8(_x(2, 8), _x(8), residual=_x(2, 8, dtype=torch.float32)), ValueError),
    (lambda: int8.rms_norm_int8(_x(2, 8), _x(8), residual=_x(1, 8)), ValueError),
    (lambda: int8.dequantize_int8(_x(2, 8), torch.ones(2)), TypeError),
    (lambda: int8.dequantize_int8(_x(2, 8, dtype=torch.int8), torch.ones(2, dtype=H)), TypeError),
    (lambda: int8.dequantize_int8(_x(2, 8, dtype=torch.int8), torch.ones(3)), ValueError),
    (lambda: int8.dequantize_int8(_x(2, 8, dtype=torch.int8), torch.ones(2), dtype=torch.int8), TypeError),
    (lambda: int8.dequantize_int8(_x(2, 0, dtype=torch.int8), torch.ones(2)), ValueError),
    (lambda: int8.dequantize_int8(_x(2, 8, dtype=torch.int8), torch.ones(2)), ValueError),
])
def test_row_refusals(call, error):
    with pytest.raises(error):
        call()


def _linear(m=3, n=4, k=16, **changes):
    args = {"x": _x(m, k, dtype=torch.int8), "x_scale": torch.ones(m), "weight": _x(n, k, dtype=torch.int8),
            "weight_scale": torch.ones(n)}
    args.update(changes)
    return int8.linear_int8(**args)


@pytest.mark.parametrize("changes,error", [
    ({}, ValueError),  # not on a GPU
    ({"x": _x(3, 16, dtype=torch.uint8)}, TypeError),
    ({"weight": _x(4, 16)}, TypeError),
    ({"x_scale": torch.ones(3, dtype=torch.float64)}, TypeError),
    ({"weight_scale": torch.ones(4, dtype=H)}, TypeError),
    ({"x_scale": torch.ones(4)}, ValueError),
    ({"x_scale": torch.ones(3, 1)}, ValueError),
    ({"weight_scale": torch.ones(3)}, ValueError),
    ({"weight": _x(4, 15, dtype=torch.int8)}, ValueError),
    ({"weight": _x(16, dtype=torch.int8), "weight_scale": torch.ones(())}, ValueError),
    ({"weight": _x(2, 4, 16, dtype=torch.int8), "weight_scale": torch.ones(2, 4)}, ValueError),
    ({"bias": _x(4, dtype=torch.float32)}, ValueError),
    ({"bias": _x(3)}, ValueError),
    ({"bias": _x(8)[::2]}, ValueError),
    ({"residual": _x(3, 5)}, ValueError),
    ({"residual": _x(1, 4)}, ValueError),
    ({"residual": _x(3, 4, dtype=torch.bfloat16)}, ValueError),
    ({"dtype": torch.int32}, TypeError),
    ({"k": 0}, ValueError),
    ({"k": int8.MAX_K + 1}, ValueError),
])
def test_linear_refusals(changes, error):
    with pytest.raises(error):
        _linear(**changes)


def test_gradients_are_refused():
    x = torch.ones(2, 8, requires_grad=True)
    for call in (lambda: int8.quantize_int8(x), lambda: int8.silu_mul_int8(x),
                 lambda: int8.rms_norm_int8(x, torch.ones(8)),
                 lambda: int8.rms_norm_int8(x.detach(), torch.ones(8, requires_grad=True)),
                 lambda: _linear(dtype=torch.float32, bias=torch.ones(4, requires_grad=True)),
                 lambda: _linear(x_scale=torch.ones(3, requires_grad=True))):
        with pytest.raises(ValueError, match="no gradient"):
            call()
        with torch.no_grad(), pytest.raises(ValueError, match="CUDA"):
            call()


@pytest.mark.parametrize("out,error", [
    (lambda: torch.zeros(3, 4, dtype=torch.float32), "shape"),
    (lambda: torch.zeros(3, 5, dtype=H), "shape"),
    (lambda: torch.zeros(4, 3, dtype=H).t(), "contiguous rows"),
    (lambda: torch.zeros(1, 4, dtype=H).expand(3, 4), "contiguous rows"),
    (lambda: torch.zeros(3, 8, dtype=H)[:, ::2], "contiguous rows"),
    (lambda: torch.zeros(12, dtype=H).as_strided((3, 4), (3, 1)), "contiguous rows"),
])
def test_destinations_are_checked(out, error):
    with pytest.raises(ValueError, match=error):
        int8._out_rows(out(), (3, 4), H, torch.device("cpu"), "out")


def test_destinations_lie_apart():
    base = torch.zeros(6, 32)
    cases = [  # destination, input, whether they share memory
        (base[:3], base[3:], False), (base[:3], base[2:], True), (base[:, :16], base[:, 16:], False),
        (base[:, :16], base[:, 15:], True), (base[:, 8:], base[:, :8], False), (base[1:, :8], base[:, 8:], False),
        (base[:, 20:], base[:, 24:30], True), (base, base, True), (base[0], base[1:], False),
        (base[0, :4], base[:, 4:], False), (base[0, :4], base[:, 3:], True), (base[:0], base, False),
        (base[:2], torch.zeros(4), False), (base[:, :16], base[:, :1].expand(6, 16), True),
    ]
    for out, t, shared in cases:
        for a, b in ((out, t), (t, out)):
            assert int8._overlap(a, b) or not shared, (a.shape, b.shape)
    # conservative only where the rows' distances differ
    assert not int8._overlap(base[:, :16], base[:, 16:]) and not int8._overlap(base[1:, :8], base[:, 8:])
    with pytest.raises(ValueError, match="out overlaps an input"):
        int8._check_apart((("out", base, ()),), (base,))
    int8._check_apart((("out", base, (base,)),), (base,))
    with pytest.raises(ValueError, match="overlaps an input"):
        int8._check_apart((("out", base[1:], (base,)),), (base,))
    with pytest.raises(ValueError, match="scale overlaps out"):
        int8._check_apart((("out", base, ()), ("scale", base[0], ())), ())


def test_pending_negations_are_refused():
    """A view whose negation is pending shows other values than those in memory."""
    x = torch._neg_view(torch.ones(2, 8))
    for call in (lambda: int8.quantize_int8(x), lambda: int8.silu_mul_int8(x),
                 lambda: int8.rms_norm_int8(torch.ones(2, 8), x[0]),
                 lambda: int8.dequantize_int8(_x(2, 8, dtype=torch.int8), x[:, 0]),
                 lambda: _linear(dtype=torch.float32, bias=x[0, :4]),
                 lambda: _linear(x_scale=x[0, :3]), lambda: _linear(weight_scale=x[0, :4])):
        with pytest.raises(ValueError, match="negation"):
            call()


def test_without_the_extension(monkeypatch):
    """An extension that does not load costs a warning and time, not the operators."""
    def missing():
        raise ImportError("built for another torch")

    monkeypatch.setattr(int8, "_plain", None)
    monkeypatch.setattr(int8._native, "torch_ops", missing)
    with pytest.warns(RuntimeWarning, match="built for another torch"), pytest.raises(ValueError, match="CUDA"):
        int8.quantize_int8(_x(2, 8))
    with pytest.raises(ValueError, match="CUDA"):  # and no second warning
        int8.quantize_int8(_x(2, 8))


def _every_call(x):
    """Each operator on ``x [2, 8]`` in one of its places."""
    q, s = _x(2, 8, dtype=torch.int8), torch.ones(2)
    return (lambda: int8.quantize_int8(x), lambda: int8.silu_mul_int8(x), lambda: int8.rms_norm_int8(x, torch.ones(8)),
            lambda: int8.rms_norm_int8(torch.ones(2, 8), x[0]), lambda: int8.dequantize_int8(q, x[:, 0]),
            lambda: int8.rms_norm_int8(torch.ones(2, 8), torch.ones(8), residual=x),
            lambda: int8.dequantize_int8(q, s, out=x), lambda: _linear(x_scale=x[0, :3]),
            lambda: _linear(dtype=torch.float32, bias=x[0, :4]))


def test_tangents_are_refused():
    """A dual tensor requires no gradient, and its tangent would be lost; also where no gradient is recorded, which does
    not end the forward mode."""
    from torch.autograd import forward_ad

    with forward_ad.dual_level():
        x = forward_ad.make_dual(torch.ones(2, 8), torch.ones(2, 8))
        for call in _every_call(x):
            with pytest.raises(ValueError, match="no derivative"):
                call()
            with torch.no_grad(), pytest.raises(ValueError, match="no derivative"):
                call()
        with pytest.raises(ValueError, match="CUDA"):
            int8.quantize_int8(forward_ad.unpack_dual(x).primal)


@pytest.mark.filterwarnings("ignore::torch.jit.TracerWarning")
def test_traces_are_refused():
    """A trace would hold the results as constants."""
    from torch.fx.experimental.proxy_tensor import make_fx

    seen = []

    def f(x):
        for call in _every_call(x):
            with pytest.raises(ValueError, match="traced"):
                call()
            seen.append(1)
        return x + 1

    torch.jit.trace(f, (torch.ones(2, 8),), check_trace=False)
    make_fx(f)(torch.ones(2, 8))
    make_fx(f, pre_dispatch=True)(torch.ones(2, 8))
    assert len(seen) == 3 * len(_every_call(torch.ones(2, 8)))
    with pytest.raises(ValueError, match="CUDA"):
        int8.quantize_int8(torch.ones(2, 8))
