"""Microscaled 4-bit floating point (MXFP4): quantization, its inverse, the fake quantization of
training, and the product on the 4-bit tensor cores.

Blocks of 32 values along the last axis share one power-of-two scale; an element is one of 0, 0.5, 1,
1.5, 2, 3, 4, 6 or its negative (``include/lucid_b200.h`` states the rounding and the layouts).  Unlike the
affine grids there is nothing to calibrate: a scale is the exponent of its block's largest magnitude, so
weights and activations are encoded by the same call, activations on every forward.

``mx_quantize`` returns ``(codes, scales)``: ``codes`` is uint8 ``(..., K / 2)``, two elements a byte, and
``scales`` uint8 ``(ceil(rows / 128), ceil(K / 256), 1024)``, the scale bytes in the tiles the tensor cores
read (``rows`` being the product of the leading axes).  ``mx_quantize`` fills the tiles' padding with 0; tiles
made elsewhere may hold anything there but 255 (NaN) past ``K``, which a product multiplies with zeros."""

from __future__ import annotations

import torch
import torch.autograd.forward_ad as forward_ad

from .. import _lib

_FLOATS = (torch.float32, torch.bfloat16)


def _addr(t):
    return None if t is None else t.data_ptr()


def _float_input(x, what: str) -> torch.Tensor:
    _lib.require_cuda(x, what)
    if x.dtype not in _FLOATS:
        raise _lib.DtypeMismatch(f"{what} must be float32 or bfloat16, got {x.dtype}")
    shape = x.shape
    if not shape or shape[-1] == 0 or shape[-1] % 32:
        raise _lib.ShapeMismatch(f"{what} needs a last axis that is a multiple of 32, got {tuple(shape)}")
    return x.detach() if x.requires_grad else x


def _rows(x: torch.Tensor) -> tuple:
    """``(x2, rows, K, row stride)``: ``x`` as (rows, K) with unit column stride and 16-byte aligned rows,
    copied only if it has to be."""
    k = x.shape[-1]
    if x.is_contiguous() and x.data_ptr() % 16 == 0:
        return x, x.numel() // k, k, k
    x2 = x if x.dim() == 2 else x.reshape(-1, k)
    ld, one = x2.stride()
    if one != 1 or ld * x2.element_size() % 16 or ld < k or x2.data_ptr() % 16:
        x2, ld = x2.clone(memory_format=torch.contiguous_format), k
    return x2, x2.shape[0], k, ld


def _dense(x: torch.Tensor) -> torch.Tensor:
    x = x.contiguous()
    return x.clone() if x.data_ptr() % 16 else x


def _scale_shape(rows: int, k: int) -> tuple:
    return ((rows + 127) // 128, (k + 255) // 256, 1024)


def _check_packed(codes, scales, what: str) -> tuple:
    """``(codes, scales, rows, K)`` of a packed matrix, its two tensors checked against each other."""
    _lib.require_cuda(codes, what)
    _lib.require_cuda(scales, what)
    if codes.dtype != torch.uint8 or scales.dtype != torch.uint8:
        raise _lib.DtypeMismatch(f"{what}: codes and scales must be uint8, got {codes.dtype}, {scales.dtype}")
    if scales.device != codes.device:
        raise _lib.DeviceMismatch(f"{what}: codes on {codes.device}, scales on {scales.device}")
    shape = codes.shape
    if not shape or shape[-1] == 0 or shape[-1] % 16:
        raise _lib.ShapeMismatch(f"{what} codes need a last axis that is a multiple of 16, got {tuple(shape)}")
    k = shape[-1] * 2
    rows = shape[0] if len(shape) == 2 else codes.numel() * 2 // k
    if scales.shape != _scale_shape(rows, k):
        raise _lib.ShapeMismatch(f"{what} scales are {tuple(scales.shape)}, expected {_scale_shape(rows, k)}")
    return _dense(codes), _dense(scales), rows, k


def mx_quantize(x: torch.Tensor):
    """``(codes, scales)`` of ``x`` (float32 or bfloat16, the last axis a multiple of 32).  A block with
    a NaN or an infinity decodes to NaN."""
    x = _float_input(x, "mx_quantize input")
    x2, rows, k, ld = _rows(x)
    dev = x.device
    codes = torch.empty(*x.shape[:-1], k // 2, dtype=torch.uint8, device=dev)
    scales = torch.empty(*_scale_shape(rows, k), dtype=torch.uint8, device=dev)
    _lib.call("lq_mx_quantize", dev, x2.data_ptr(), _lib.code_of(x.dtype), rows, k, ld, codes.data_ptr(), scales.data_ptr())
    return codes, scales


def mx_dequantize(codes: torch.Tensor, scales: torch.Tensor, out_dtype: torch.dtype = torch.float32) -> torch.Tensor:
    """The values ``(codes, scales)`` stand for: exact in float32 and in bfloat16, up to the float32 range (which a
    scale byte of 253 or 254 can pass; ``mx_quantize`` writes none above 252)."""
    if out_dtype not in _FLOATS:
        raise _lib.DtypeMismatch(f"mx_dequantize writes float32 or bfloat16, got {out_dtype}")
    c, s, rows, k = _check_packed(codes, scales, "mx_dequantize")
    dev = codes.device
    out = torch.empty(*codes.shape[:-1], k, dtype=out_dtype, device=dev)
    _lib.call("lq_mx_dequantize", dev, c.data_ptr(), s.data_ptr(), rows, k, out.data_ptr(), _lib.code_of(out_dtype))
    return out


def _pass_gradient(grad: torch.Tensor, mask: torch.Tensor) -> torch.Tensor:
    g = _dense(grad.detach())
    out = torch.empty_like(g)
    _lib.call("lq_mx_fake_quantize_grad", g.device, g.data_ptr(), _lib.code_of(g.dtype), mask.data_ptr(), g.numel(),
              out.data_ptr())
    return out


def _has_tangent(t: torch.Tensor) -> bool:
    return forward_ad.unpack_dual(t).tangent is not None


class _StraightThrough(torch.autograd.Function):
    """The gradient of the fake quantization: linear in the gradient that comes in, so it is its own
    derivative, forwards and backwards."""

    @staticmethod
    def forward(ctx, grad, mask):
        ctx.save_for_backward(mask)
        ctx.save_for_forward(mask)
        return _pass_gradient(grad, mask)

    @staticmethod
    def backward(ctx, grad):
        (mask,) = ctx.saved_tensors
        return _StraightThrough.apply(grad, mask), None

    @staticmethod
    def jvp(ctx, tangent, _):
        return _StraightThrough.apply(tangent, *ctx.saved_tensors)


def _fake_quantize(x: torch.Tensor, want_mask: bool):
    xc = _dense(_float_input(x, "mx_fake_quantize input"))
    out = torch.empty_like(xc)
    mask = torch.empty(xc.numel() // 8, dtype=torch.uint8, device=xc.device) if want_mask else None
    _lib.call("lq_mx_fake_quantize", xc.device, xc.data_ptr(), _lib.code_of(xc.dtype), xc.numel(), out.data_ptr(), _addr(mask))
    return out, mask


class _MXFakeQuantize(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x):
        out, mask = _fake_quantize(x, True)
        ctx.save_for_backward(mask)
        ctx.save_for_forward(mask)
        return out

    @staticmethod
    def backward(ctx, grad):
        (mask,) = ctx.saved_tensors
        if torch.is_grad_enabled() or _has_tangent(grad):  # somebody differentiates the gradient
            return _StraightThrough.apply(grad, mask)
        return _pass_gradient(grad, mask)

    @staticmethod
    def jvp(ctx, tangent):
        return _StraightThrough.apply(tangent, *ctx.saved_tensors)


def mx_fake_quantize(x: torch.Tensor) -> torch.Tensor:
    """``mx_dequantize(*mx_quantize(x))`` in one pass, in ``x``'s dtype, with the straight-through
    gradient: it passes where the element was rounded inside the grid and is zero where it was clamped
    (and in blocks that decode to NaN); a forward-mode tangent passes likewise.  A backward pass is captured in a
    CUDA graph as any of torch's: with no eager graph of the same leaves alive on another stream."""
    if isinstance(x, torch.Tensor) and (x.requires_grad and torch.is_grad_enabled() or _has_tangent(x)):
        return _MXFakeQuantize.apply(x)
    return _fake_quantize(x, False)[0]


def _bias_of(bias, n: int, device) -> torch.Tensor | None:
    if bias is None:
        return None
    _lib.require_cuda(bias, "bias")
    if bias.device != device:
        raise _lib.DeviceMismatch(f"bias on {bias.device}, the product runs on {device}")
    if bias.dim() != 1 or bias.shape[0] != n:
        raise _lib.ShapeMismatch(f"bias is {tuple(bias.shape)}, expected {(n,)}")
    if bias.dtype == torch.float32 and bias.is_contiguous():
        return bias
    return bias.detach().to(torch.float32).contiguous()


def mx_matmul(a_codes: torch.Tensor, a_scales: torch.Tensor, w_codes: torch.Tensor, w_scales: torch.Tensor,
              bias: torch.Tensor | None = None, relu: bool = False, out_dtype: torch.dtype = torch.float32) -> torch.Tensor:
    """``a @ w.T (+ bias)`` of two packed matrices, ``a`` ``(..., K)`` and ``w`` ``(N, K)``, with float32
    accumulation; float32 or bfloat16 out."""
    if out_dtype not in _FLOATS:
        raise _lib.DtypeMismatch(f"mx_matmul writes float32 or bfloat16, got {out_dtype}")
    ac, sa, m, k = _check_packed(a_codes, a_scales, "mx_matmul left operand")
    wc, sw, n, kw = _check_packed(w_codes, w_scales, "mx_matmul weight")
    if w_codes.dim() != 2:
        raise _lib.ShapeMismatch(f"the weight's codes must be (N, K / 2), got {tuple(w_codes.shape)}")
    if k != kw:
        raise _lib.ShapeMismatch(f"the left operand has {k} features, the weight {kw}")
    dev = a_codes.device
    if w_codes.device != dev:
        raise _lib.DeviceMismatch(f"left operand on {dev}, weight on {w_codes.device}")
    b = _bias_of(bias, n, dev)
    out = torch.empty(*a_codes.shape[:-1], n, dtype=out_dtype, device=dev)
    _lib.call("lq_mx_matmul", dev, ac.data_ptr(), sa.data_ptr(), m, wc.data_ptr(), sw.data_ptr(), n, k, _addr(b),
              int(relu), out.data_ptr(), _lib.code_of(out_dtype), n, _lib.status_ptr(dev))
    return out


def mx_linear(x: torch.Tensor, w_codes: torch.Tensor, w_scales: torch.Tensor, bias: torch.Tensor | None = None,
              relu: bool = False) -> torch.Tensor:
    """``mx_matmul(*mx_quantize(x), ...)`` in one call; the result has ``x``'s dtype.  For inference, like the other
    quantized products: no derivative passes (training goes through ``mx_fake_quantize``)."""
    x = _float_input(x, "mx_linear input")
    wc, sw, n, k = _check_packed(w_codes, w_scales, "mx_linear weight")
    if w_codes.dim() != 2:
        raise _lib.ShapeMismatch(f"the weight's codes must be (N, K / 2), got {tuple(w_codes.shape)}")
    if x.shape[-1] != k:
        raise _lib.ShapeMismatch(f"the input has {x.shape[-1]} features, the weight {k}")
    dev = x.device
    if w_codes.device != dev:
        raise _lib.DeviceMismatch(f"input on {dev}, weight on {w_codes.device}")
    b = _bias_of(bias, n, dev)
    x2, m, _, ld = _rows(x)
    out = torch.empty(*x.shape[:-1], n, dtype=x.dtype, device=dev)
    # lq_mx_linear_workspace_bytes
    room = 0 if m <= 16 else (m * (k // 2) + 1023) // 1024 * 1024 + (m + 127) // 128 * ((k + 255) // 256) * 1024
    ws = torch.empty(room, dtype=torch.uint8, device=dev) if room else None
    code = _lib.code_of(x.dtype)
    _lib.call("lq_mx_linear", dev, x2.data_ptr(), code, m, ld, wc.data_ptr(), sw.data_ptr(), n, k, _addr(b),
              int(relu), out.data_ptr(), code, n, _addr(ws), room, _lib.status_ptr(dev))
    return out
