"""Products in 8-bit integers with a scale for each token and each row of the weights, for serving.

``quantize_rows`` lays weights out once; ``int8_linear`` takes tokens as they come, forms their codes and multiplies on the
integer matrix instructions (twice the rate of bf16, half the weights' bytes).  Sums are exact 32-bit integers, so a result
is off by the rounding of the codes (half a step of 1/127 of the largest magnitude of a row) and of the result itself::

    codes, scale = quantize_rows(weight)           # (out, in), once
    y = int8_linear(x, codes, scale, bias)         # (..., in) -> (..., out)

The reference has no counterpart; its projections are ``nn.Linear`` under bf16 autocast.  No gradient; CPU tensors raise.
"""

from __future__ import annotations

import ctypes

import torch

from . import _lib
from ._attn import _unit_inner

MAX_IN = 1 << 17  # a sum of so many products of two codes stays below 2^31
MAX_ROWS = (1 << 31) - 256  # rows of tokens or weights, and the ends of their tiles, are counted in 32 bits


def _dtype_code(what, t):
    if t.dtype not in (torch.bfloat16, torch.float32):
        raise TypeError(f"{what}: {t.dtype} is neither bf16 nor fp32")
    return _lib.DFL_BF16 if t.dtype == torch.bfloat16 else _lib.DFL_F32


def _no_grad(what, *tensors):
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors):
        raise RuntimeError(f"{what} has no gradient: call it under torch.no_grad()")


def _quantize(x):
    M, K = x.shape
    dev, xc = x.device, _unit_inner(x)
    stride = -(-K // 16) * 16
    codes = torch.empty(M, stride, dtype=torch.int8, device=dev)
    scale = torch.empty(M, dtype=torch.float32, device=dev)
    p = _lib.QuantizeRowsParams(_dtype_code("quantize_rows", x), xc.data_ptr(), xc.stride(0), M, K, codes.data_ptr(), stride,
                                scale.data_ptr())
    lib = _lib.load()
    with _lib.on_device(dev):
        rc = _lib.timed_launch("quantize_rows", dev, lambda: lib.dfl_quantize_rows(
            ctypes.byref(p), _lib.stream_handle(dev)))
    _lib.check(rc, "dfl_quantize_rows")
    return codes[:, :K], scale


def _linear(x, codes, scale, bias):
    N, K = codes.shape
    dev = x.device
    xc = _unit_inner(x if x.dim() == 2 else x.reshape(-1, K))
    M = xc.shape[0]
    y = torch.empty(*x.shape[:-1], N, dtype=x.dtype, device=dev)
    b = None if bias is None else bias.to(x.dtype).contiguous()
    scale = scale.contiguous()
    row = codes.stride(0) if N > 1 else -(-K // 16) * 16
    p = _lib.Int8LinearParams(_dtype_code("int8_linear", x), xc.data_ptr(), xc.stride(0), codes.data_ptr(), row, scale.data_ptr(),
                              _lib.ptr(b), y.data_ptr(), M, K, N)
    lib = _lib.load()
    # the tokens' codes, in a workspace of the call's own: calls on other streams and captured graphs cannot share it
    nbytes = lib.dfl_int8_linear_workspace_size(M, K, N)
    ws = torch.empty(nbytes, dtype=torch.uint8, device=dev) if nbytes else None
    with _lib.on_device(dev):
        rc = _lib.timed_launch("int8_linear", dev, lambda: lib.dfl_int8_linear(
            ctypes.byref(p), _lib.ptr(ws), nbytes, _lib.stream_handle(dev)))
    _lib.check(rc, "dfl_int8_linear")
    return y


class _QuantizeRowsFn(torch.autograd.Function):
    """A call as a node of a trace, without a gradient."""

    @staticmethod
    def forward(ctx, x):
        out = _quantize(x)
        ctx.mark_non_differentiable(*out)
        return out


class _Int8LinearFn(torch.autograd.Function):
    """A call as a node of a trace, without a gradient."""

    @staticmethod
    def forward(ctx, *args):
        y = _linear(*args)
        ctx.mark_non_differentiable(y)
        return y


def quantize_rows(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """Codes (M,K) int8 and scale (M,) fp32 of the rows of x (M,K) bf16 or fp32, any strides, K at most 131072.

    scale = max |row| / 127 rounded to fp32, at least 2^-100; code the integer nearest to x / scale, ties to even.  A row
    that holds an infinity or NaN has scale NaN and codes 0.  The codes are a view of rows that are padded to a multiple
    of 16 bytes, the layout that ``int8_linear`` takes."""
    what = "quantize_rows"
    if x.dim() != 2 or 0 in x.shape or x.shape[1] > MAX_IN:
        raise ValueError(f"{what}: x {tuple(x.shape)} must be (M,K), not empty, with K at most {MAX_IN}")
    _dtype_code(what, x)
    _no_grad(what, x)
    _lib.require_gpu(x)
    return _QuantizeRowsFn.apply(x) if _lib.recording() else _quantize(x)


def int8_linear(
    x: torch.Tensor,
    codes: torch.Tensor,
    scale: torch.Tensor,
    bias: torch.Tensor | None = None,
) -> torch.Tensor:
    """x W^T + bias with W the rows that codes (N,K) int8 and scale (N,) fp32 stand for (``quantize_rows``).

    x (..., K) bf16 or fp32, any strides; each of its rows is rounded to codes as ``quantize_rows`` does it, the products
    are summed exactly and multiplied by both scales in fp32.  codes in rows of a multiple of 16 bytes, 16-byte aligned,
    as ``quantize_rows`` lays them out.  bias (N,) is added in x's type.  Returns (..., N) in x's type; rows with an
    infinity or NaN are NaN.  No gradient."""
    what = "int8_linear"
    if codes.dim() != 2 or codes.dtype != torch.int8:
        raise TypeError(f"{what}: codes must be (N,K) int8")
    N, K = codes.shape
    if N < 1 or not 1 <= K <= MAX_IN:
        raise ValueError(f"{what}: codes {tuple(codes.shape)} must not be empty, with K at most {MAX_IN}")
    if x.dim() < 1 or x.shape[-1] != K:
        raise ValueError(f"{what}: x {tuple(x.shape)} does not fit codes {tuple(codes.shape)}")
    if scale.shape != (N,) or scale.dtype != torch.float32:
        raise ValueError(f"{what}: scale must be ({N},) fp32")
    if bias is not None and (bias.shape != (N,) or not bias.is_floating_point()):
        raise ValueError(f"{what}: bias must be ({N},) floating point")
    _dtype_code(what, x)
    _no_grad(what, x, scale, bias)
    _lib.require_gpu(x, codes, scale, bias)
    if x.numel() == 0 or x.numel() // K > MAX_ROWS or N > MAX_ROWS:
        raise ValueError(f"{what}: no tokens, or above {MAX_ROWS} of them or of the weights' rows")
    stride = codes.stride()
    if N == 1:
        stride = (-(-K // 16) * 16, stride[1])
    whole = -(-K // 16) * 16  # bytes of a row that are read
    if ((stride[1] != 1 and K > 1) or stride[0] % 16 or stride[0] < K or codes.data_ptr() % 16 or codes.storage_offset() +
            (N - 1) * stride[0] + whole > codes.untyped_storage().nbytes()):
        raise ValueError(f"{what}: codes' rows must be 16-byte aligned and in memory of a multiple of 16 bytes, as "
                         "quantize_rows lays them out")
    run = _Int8LinearFn.apply if _lib.recording() else _linear
    return run(x, codes, scale, bias)
