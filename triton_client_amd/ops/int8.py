"""8-bit integer operators for serving language models (inference).

``quantize_int8``    rows to 8-bit integers with one fp32 scale per row
``dequantize_int8``  the values such rows stand for
``rms_norm_int8``    root-mean-square norm with the residual's addition, straight to 8-bit rows
``silu_mul_int8``    the gated activation of an MLP, straight to 8-bit rows
``linear_int8``      matrix product of 8-bit rows with 8-bit weights, a scale per token and per output channel,
                     bias and residual in the epilogue

The kernels are ``csrc/hip/int8_rows.hip`` and ``csrc/hip/int8_linear.hip``.  A block of a model runs them back to back,
activations crossing memory in 8 bits between the products::

    w1, s1 = quantize_int8(gate_up_weight)                      # once, [2 * F, D]
    w2, s2 = quantize_int8(down_weight)                         # once, [D, F]
    q, s, h = rms_norm_int8(x, norm_weight, residual=h)
    y = linear_int8(q, s, w1, s1, dtype=torch.bfloat16)         # [tokens, 2 * F]
    q, s = silu_mul_int8(y)
    h = linear_int8(q, s, w2, s2, residual=h, dtype=torch.bfloat16)

Rows are everything but the last axis.  Inputs are torch CUDA tensors of fp16, bf16 or fp32 (integers: int8); rows may
lie apart (a 2-D view with a row stride), other layouts are copied first.  Work is enqueued on the current torch stream
of the tensors' device and nothing waits for it; results may be captured into graphs.  The integers have no gradient:
operands that require one are refused while gradients are recorded, those with a forward-mode tangent always, and so
are calls inside ``torch.jit.trace`` or ``make_fx``, which would record the results as constants.

A row with a value that is not finite gets integers of 0 and a scale of NaN, so that whatever is computed from it is NaN
instead of a number.  The reference has no model code (its models run in the server it talks to, e.g.
``src/python/examples/image_client.py:59-150`` only inspects metadata); this is the serving side of that contract.
"""

from __future__ import annotations

import subprocess
import sys
import warnings

import torch
from torch.autograd import forward_ad

from .. import _native
from ._device import check, lib

# 128 * 128 * k has to stay below 2^31
MAX_K = 131071
MAX_WIDTH = 1 << 29

_CODES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}


# the extension that takes the plain case of a call (contiguous operands, new results) without the checks below
_plain = None


class _General:
    """In the place of an extension that this torch does not load and that cannot be built here: no call is plain."""

    def __getattr__(self, name):
        return lambda *args: None


def _load_plain():
    global _plain
    lib()  # without the kernels there is no way to go on
    try:
        _plain = _native.torch_ops()
    except (ImportError, FileNotFoundError, subprocess.CalledProcessError) as e:
        warnings.warn(f"8-bit operators: calls take their slower way in Python, the extension is not there ({e})",
                      RuntimeWarning, stacklevel=3)
        _plain = _General()
    return _plain


def _output_code(dtype):
    code = _CODES.get(dtype)
    if code is None:
        raise TypeError("dtype must be torch.float16, torch.bfloat16 or torch.float32")
    return code


def _check_operands(first, others):
    """Index of the operands' common CUDA device; no operand may require a gradient while gradients are recorded, carry a
    tangent, or stand for other values than those in memory, and no trace may be under way."""
    device = first.get_device()
    duals = getattr(forward_ad, "_current_level", 0) >= 0  # tangents live inside a level
    for t in (first, *others):
        if t is not None:
            if t.requires_grad:
                _refuse_gradient()
            if duals and forward_ad.unpack_dual(t).tangent is not None:
                raise ValueError("8-bit operators have no derivative: take the primal of forward_ad.unpack_dual()")
            if t.is_neg():
                raise ValueError("an operand's negation is pending: call its resolve_neg()")
            if t.get_device() != device:
                raise ValueError("the operands must be on one device")
    # what launches a kernel by itself would enter a trace as a constant
    if torch.jit.is_tracing() or _proxy_mode():
        raise ValueError("8-bit operators cannot be traced: call them outside of the traced function")
    if device < 0:
        raise ValueError("the operands must be CUDA tensors")
    return device


def _proxy_mode():
    """Whether ``make_fx`` records the operations of this thread."""
    proxies = sys.modules.get("torch.fx.experimental.proxy_tensor")  # there if one does
    return proxies is not None and proxies.get_proxy_mode() is not None


def _refuse_gradient():
    if torch.is_grad_enabled():
        raise ValueError("8-bit operators have no gradient: detach the operands or call under torch.no_grad()")


def _rows(t):
    """``(tensor, row stride)`` of an input: as it is where the values of a row lie side by side, else a copy."""
    if t.is_contiguous():
        return t, t.shape[-1]
    if t.dim() == 2 and t.stride(1) == 1:
        return t, t.stride(0)
    return t.contiguous(), t.shape[-1]


def _out_rows(out, shape, dtype, device, name):
    """Row stride of a caller's destination."""
    if tuple(out.shape) != tuple(shape) or out.dtype != dtype or out.device != device:
        raise ValueError(f"{name} must be a {dtype} tensor of shape {list(shape)} on {device}")
    if out.requires_grad:
        raise ValueError(f"{name} must not require a gradient")
    if out.is_contiguous():
        return out.shape[-1] if out.dim() else 1
    if out.dim() == 2 and out.stride(1) == 1 and out.stride(0) >= out.shape[1]:
        return out.stride(0)
    raise ValueError(f"{name} must be contiguous, or 2-D with contiguous rows that do not overlap")


def _extent(t):
    """``(first byte, one past the last, bytes between rows, bytes of a row)`` of a tensor with contiguous rows."""
    first, size = t.data_ptr(), t.element_size()
    if t.is_contiguous():
        return first, first + t.numel() * size, 0, 0
    stride, row = t.stride(0) * size, t.shape[1] * size
    return first, first + (t.shape[0] - 1) * stride + row, stride, row


def _overlap(a, b):
    if not a.numel() or not b.numel():
        return False
    a0, a1, a_stride, a_row = _extent(a)
    b0, b1, b_stride, b_row = _extent(b)
    if a0 >= b1 or b0 >= a1:
        return False
    if a_stride == b_stride and a_stride:  # column ranges of one buffer
        apart = (a0 - b0) % a_stride
        return apart < b_row or apart + a_row > a_stride
    return True


def _check_apart(outputs, inputs):
    """Destinations ``(name, tensor or None, inputs that it may be)`` lie apart from the inputs and each other."""
    given = [o for o in outputs if o[1] is not None]
    for i, (name, out, may_be) in enumerate(given):
        for t in inputs:
            # an input that IS the destination: every value is read by the thread that writes it, before it does
            if t is not None and _overlap(out, t) and not (any(t is m for m in may_be)
                                                           and out.data_ptr() == t.data_ptr()
                                                           and out.stride() == t.stride()):
                raise ValueError(f"{name} overlaps an input")
        for other, t, _ in given[:i]:
            if _overlap(out, t):
                raise ValueError(f"{name} overlaps {other}")


def _raw_stream(index):
    return torch.cuda.current_stream(index).cuda_stream


# the handle alone, where torch gives it: an object around it costs as much as a third of a call's checks
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", _raw_stream)


def _launch(what, device, *args):
    fn = getattr(lib(), what)
    if torch.cuda.current_device() == device:
        rc = fn(*args, _raw_stream(device))
    else:
        with torch.cuda.device(device):
            rc = fn(*args, _raw_stream(device))
    if rc:
        check(rc, what)


def _written(*destinations):
    """A caller's tensors have other values now: a backward pass that has saved one of them has to find out, as it does
    after torch's own operators.  (Inference tensors have no version, and no backward pass saves them.)"""
    for t in destinations:
        if t is not None and not t.is_inference():
            torch.autograd.graph.increment_version(t)


def _row_outputs(x, shape, out, scale):
    """``(q, q stride, scale)``: the destinations given, or new ones."""
    if out is None:
        out, stride = torch.empty(shape, dtype=torch.int8, device=x.device), shape[-1]
    else:
        stride = _out_rows(out, shape, torch.int8, x.device, "out")
    if scale is None:
        scale = torch.empty(shape[:-1], dtype=torch.float32, device=x.device)
    else:
        _check_scale_out(scale, shape[:-1], x.device)
    return out, stride, scale


def _check_scale_out(scale, shape, device):
    if (scale.dtype != torch.float32 or tuple(scale.shape) != tuple(shape) or scale.device != device
            or not scale.is_contiguous() or scale.requires_grad):
        raise ValueError(f"scale must be a contiguous fp32 tensor of shape {list(shape)} on {device}")


def _quantize(x, gated, out, scale):
    code = _CODES.get(x.dtype)
    if code is None:
        raise TypeError("x must be an fp16, bf16 or fp32 tensor")
    shape = x.shape
    if not shape or not 1 <= shape[-1] <= MAX_WIDTH:
        raise ValueError(f"x must have a last axis of 1 to {MAX_WIDTH} values")
    if gated:
        if shape[-1] % 2:
            raise ValueError("the last axis of x must hold two halves of equal size")
        shape = (*shape[:-1], shape[-1] // 2)
    device = _check_operands(x, (out, scale))
    x, x_stride = _rows(x)
    q, q_stride, s = _row_outputs(x, shape, out, scale)
    if out is not None or scale is not None:
        _check_apart((("out", out, ()), ("scale", scale, ())), (x,))
    rows = s.numel()
    if rows:
        _launch("tca_int8_quantize_launch", device, x.data_ptr(), q.data_ptr(), s.data_ptr(), code, gated, rows,
                shape[-1], x_stride, q_stride)
        _written(out, scale)
    return q, s


def quantize_int8(x, out=None, scale=None):
    """``(q int8 [..., K], scale fp32 [...])`` of ``x [..., K]``: with ``m`` the largest magnitude of a row, ``q`` is the
    integer nearest to ``127 x / m`` (ties to even, decided exactly) and ``scale = m / 127`` (one step less where
    ``127 * scale`` would leave fp32's range).  A row of zeros has the scale 0.  ``out`` and ``scale`` may be
    destinations of the results' shapes."""
    if out is None and scale is None:
        made = (_plain or _load_plain()).quantize(x, False)
        if made is not None:
            return made
    return _quantize(x, 0, out, scale)


def silu_mul_int8(x, out=None, scale=None):
    """8-bit rows ``(q [..., K], scale [...])``, as of :func:`quantize_int8`, of ``silu(gate) * up`` for
    ``x [..., 2 K]`` with the gate in the first half of the last axis and the other factor in the second.  The product
    is taken in fp32."""
    if out is None and scale is None:
        made = (_plain or _load_plain()).quantize(x, True)
        if made is not None:
            return made
    return _quantize(x, 1, out, scale)


def rms_norm_int8(x, weight, residual=None, eps=1e-6, out=None, scale=None, sum_out=None):
    """8-bit rows of ``h / sqrt(mean(h^2) + eps) * weight``: ``(q, scale)`` for ``h = x``, or ``(q, scale, h)`` for
    ``h = x + residual``.

    x         ``[..., K]``
    weight    ``[K]``, contiguous, of x's type or fp32
    residual  of x's shape and type, or None.  The sum is rounded to x's type, and the rounded sum is what is
              normalised and returned: what the next block reads is what this one saw
    sum_out   destination of the sum; may be ``x`` or ``residual`` itself

    ``q`` is the integer nearest to ``127 p / max|p|`` (ties to even, decided exactly) for ``p = h weight`` in fp32: the
    norm's factor cancels and only enters the scale.  Sums of squares are held in 64 bits."""
    if out is None and scale is None and sum_out is None:
        made = (_plain or _load_plain()).rms_norm(x, weight, residual, eps)
        if made is not None:
            return made
    dtype = x.dtype
    code = _CODES.get(dtype)
    if code is None:
        raise TypeError("x must be an fp16, bf16 or fp32 tensor")
    shape = x.shape
    if not shape or not 1 <= shape[-1] <= MAX_WIDTH:
        raise ValueError(f"x must have a last axis of 1 to {MAX_WIDTH} values")
    width = shape[-1]
    weight_f32 = weight.dtype == torch.float32
    if not weight_f32 and weight.dtype != dtype:
        raise TypeError("weight must have x's type or be fp32")
    if weight.dim() != 1 or weight.shape[0] != width or not weight.is_contiguous():
        raise ValueError(f"weight must be a contiguous vector of {width} values")
    if not 0.0 < eps < float("inf"):
        raise ValueError("eps must be a positive number")
    if residual is None:
        if sum_out is not None:
            raise ValueError("sum_out needs a residual")
    elif residual.dtype != dtype or residual.shape != shape:
        raise ValueError("residual must have x's type and shape")
    device = _check_operands(x, (weight, residual, out, scale, sum_out))
    x, x_stride = _rows(x)
    q, q_stride, s = _row_outputs(x, shape, out, scale)
    summed, r_ptr, sum_ptr, r_stride, sum_stride = None, None, None, 0, 0
    if residual is not None:
        residual, r_stride = _rows(residual)
        if sum_out is None:
            summed, sum_stride = torch.empty(shape, dtype=dtype, device=x.device), width
        else:
            summed, sum_stride = sum_out, _out_rows(sum_out, shape, dtype, x.device, "sum_out")
        r_ptr, sum_ptr = residual.data_ptr(), summed.data_ptr()
    if out is not None or scale is not None or sum_out is not None:
        _check_apart((("out", out, ()), ("scale", scale, ()), ("sum_out", sum_out, (x, residual))),
                     (x, weight, residual))
    rows = s.numel()
    if rows:
        _launch("tca_int8_rms_norm_launch", device, x.data_ptr(), r_ptr, weight.data_ptr(), q.data_ptr(), s.data_ptr(),
                sum_ptr, code, weight_f32, eps, rows, width, x_stride, r_stride, q_stride, sum_stride)
        _written(out, scale, sum_out)
    return (q, s) if residual is None else (q, s, summed)


def _check_quantized(q, scale, name, scale_name):
    if q.dtype != torch.int8:
        raise TypeError(f"{name} must be an int8 tensor")
    if scale.dtype != torch.float32:
        raise TypeError(f"{scale_name} must be an fp32 tensor")
    shape = q.shape
    if not shape or scale.shape != shape[:-1]:
        raise ValueError(f"{name} [..., K] needs a scale for each row, of shape [...]")
    return shape


def dequantize_int8(q, scale, dtype=None, out=None):
    """``q * scale`` of 8-bit rows ``q [..., K]`` with ``scale [...]``, in ``dtype`` (default fp16, or out's)."""
    if out is None:
        code = _output_code(torch.float16 if dtype is None else dtype)
        made = (_plain or _load_plain()).dequantize(q, scale, code)
        if made is not None:
            return made
    shape = _check_quantized(q, scale, "q", "scale")
    if not 1 <= shape[-1] <= MAX_WIDTH:
        raise ValueError(f"q must have a last axis of 1 to {MAX_WIDTH} values")
    if dtype is None:
        dtype = torch.float16 if out is None else out.dtype
    code = _output_code(dtype)
    device = _check_operands(scale, (q, out))
    q, q_stride = _rows(q)
    scale, given = scale.contiguous(), out
    if out is None:
        out, out_stride = torch.empty(shape, dtype=dtype, device=q.device), shape[-1]
    else:
        out_stride = _out_rows(out, shape, dtype, q.device, "out")
        _check_apart((("out", out, ()),), (q, scale))
    rows = scale.numel()
    if rows:
        _launch("tca_int8_dequantize_launch", device, q.data_ptr(), scale.data_ptr(), out.data_ptr(), code, rows,
                shape[-1], q_stride, out_stride)
        _written(given)
    return out


def linear_int8(x, x_scale, weight, weight_scale, bias=None, residual=None, dtype=None, out=None):
    """``(x weight^T) * x_scale * weight_scale + bias (+ residual)`` in ``dtype`` (default fp16, or out's).

    x, x_scale            8-bit rows ``[..., K]`` with a scale per token ``[...]``
    weight, weight_scale  8-bit rows ``[N, K]`` with a scale per output channel ``[N]``
    bias                  ``[N]`` in ``dtype``, contiguous, or None
    residual              ``[..., N]`` in ``dtype``, or None; ``out`` may be the residual itself

    Sums are int32 and exact for K up to 131071; scales, bias and residual are applied in fp32 and the result is rounded
    once.  The product of the two scales is taken first, in fp32: below 1.2e-38 it has fewer digits, and the result with it;
    beyond 3.4e38 it is infinite.  Operands whose rows start at multiples of 16 bytes (K and the row strides multiples of
    16) are read as they are; others are read more slowly or, in a large product, first copied to such rows in a workspace
    of the call."""
    if out is None:
        code = _output_code(torch.float16 if dtype is None else dtype)
        made = (_plain or _load_plain()).linear(x, x_scale, weight, weight_scale, bias, residual, code)
        if made is not None:
            return made
    shape = _check_quantized(x, x_scale, "x", "x_scale")
    w_shape = _check_quantized(weight, weight_scale, "weight", "weight_scale")
    if len(w_shape) != 2:
        raise ValueError("weight must be an [N, K] matrix")
    n, k = w_shape
    if shape[-1] != k:
        raise ValueError(f"x has rows of {shape[-1]} integers, weight of {k}")
    if not 1 <= k <= MAX_K:
        raise ValueError(f"K must be 1 to {MAX_K}: the int32 sums hold no more")
    if dtype is None:
        dtype = torch.float16 if out is None else out.dtype
    code = _output_code(dtype)
    shape = (*shape[:-1], n)
    if bias is not None and (bias.dtype != dtype or tuple(bias.shape) != (n,) or not bias.is_contiguous()):
        raise ValueError(f"bias must be a contiguous {dtype} vector of {n} values")
    if residual is not None and (residual.dtype != dtype or tuple(residual.shape) != shape):
        raise ValueError(f"residual must be a {dtype} tensor of shape {list(shape)}")
    device = _check_operands(x_scale, (x, weight, weight_scale, bias, residual, out))
    x, x_stride = _rows(x)
    weight, w_stride = _rows(weight)
    x_scale, weight_scale = x_scale.contiguous(), weight_scale.contiguous()
    r_ptr, r_stride, given = None, 0, out
    if residual is not None:
        residual, r_stride = _rows(residual)
        r_ptr = residual.data_ptr()
    if out is None:
        out, out_stride = torch.empty(shape, dtype=dtype, device=x.device), n
    else:
        out_stride = _out_rows(out, shape, dtype, x.device, "out")
        _check_apart((("out", out, (residual,)),), (x, x_scale, weight, weight_scale, bias, residual))
    tokens = x_scale.numel()
    if tokens and n:
        x_ptr, w_ptr = x.data_ptr(), weight.data_ptr()
        workspace = None
        if (x_ptr | w_ptr | x_stride | w_stride | k) & 15:
            size = lib().tca_int8_linear_workspace_bytes(x_ptr, w_ptr, tokens, n, k, x_stride, w_stride)
            if size:  # of this call: the allocator orders its reuse, also inside a graph's own pool
                workspace = torch.empty(size, dtype=torch.int8, device=x.device)
        _launch("tca_int8_linear_launch", device, x_ptr, x_scale.data_ptr(), w_ptr, weight_scale.data_ptr(),
                None if bias is None else bias.data_ptr(), r_ptr, out.data_ptr(), code, tokens, n, k, x_stride,
                w_stride, r_stride, out_stride, None if workspace is None else workspace.data_ptr())
        _written(given)
    return out
