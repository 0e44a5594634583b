"""Linear layers in 8-bit integers: weights with a scale for each output channel, activations quantised in the call with a scale
for each token."""
from __future__ import annotations

from typing import Optional, Tuple

import torch

from ._cabi import check, ctx, load
from .ops import BF16, _ptr, _stream, _Workspace
from .position_ops import _device, _refuse

F32, I8 = torch.float32, torch.int8


def _rows(x: torch.Tensor) -> torch.Tensor:
    """[..., K] as rows that are one stride apart, their elements next to each other."""
    if x.dim() != 2:
        x = x.reshape(-1, x.shape[-1])
    (m, k), (ld, e) = x.shape, x.stride()
    return x if (e == 1 or k <= 1) and (ld >= k or m <= 1) else x.contiguous()


def _ld(x2: torch.Tensor) -> int:
    return max(x2.stride(0), x2.shape[1])   # (the stride of a single row may be anything)


def quantize_rows(x: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
    """(q, scale) of x bfloat16 or float32 [..., K]: scale float32 [...] = max |x| / 127 of each row, q int8 [..., K] = x / scale
    rounded to the nearest whole number, ties to even.  q's rows are a multiple of 64 bytes apart: ``linear_int8`` wants its
    weights (a row for each output channel) and ``linear_int8_quantized`` both operands 16 bytes apart, and reads them faster so.  A row of zeros has scale 0, one that
    holds something not finite scale NaN and zeros."""
    if (x.dtype is not BF16 and x.dtype is not F32) or x.dim() < 1 or x.shape[-1] < 1:
        _refuse("quantize rows: bfloat16 or float32 [..., K]")
    dev = _device(x)
    x2 = _rows(x)
    m, k = x2.shape
    kp = (k + 63) // 64 * 64
    q, scale = x.new_empty((m, kp), dtype=I8), x.new_empty(x.shape[:-1], dtype=F32)
    check(load().xfold_quantize_rows_fwd(ctx(dev), _ptr(x2), int(x.dtype == F32), _ld(x2), m, k, _ptr(q), kp, _ptr(scale), _stream(dev)),
          dev, "xfold_quantize_rows_fwd")
    return q.view(*x.shape[:-1], kp)[..., :k], scale


def _operand(t: torch.Tensor, what: str) -> Tuple[int, int, int, int]:
    """(address, row stride, rows, inner width) of int8 rows that the kernel can take."""
    if t.dtype is not I8 or t.dim() != 2:
        _refuse("int8 linear: " + what + " int8 [rows, K]")
    (n, k), (ld, e), at = t.shape, t.stride(), t.data_ptr()
    if n <= 1:
        ld = (k + 15) // 16 * 16
    if at % 16 or ld % 16 or ld < k or (e != 1 and k > 1):
        _refuse("int8 linear: rows of " + what + " start at multiples of 16 bytes (as quantize_rows leaves them)")
    return at, ld, n, k


def _check_channels(n: int, w_scale, bias) -> None:
    if w_scale.dtype is not F32 or w_scale.shape != (n,) or not w_scale.is_contiguous():
        _refuse("int8 linear: a float32 scale for each output channel")
    if bias is not None and (bias.dtype is not F32 or bias.shape != (n,) or not bias.is_contiguous()):
        _refuse("int8 linear: bias is float32 [channels]")


def linear_int8(x: torch.Tensor, w: torch.Tensor, w_scale: torch.Tensor, bias: Optional[torch.Tensor] = None,
                dtype: Optional[torch.dtype] = None) -> torch.Tensor:
    """x bfloat16 or float32 [..., K], w int8 [N, K] (rows a multiple of 16 bytes apart, see ``quantize_rows``), w_scale float32
    [N] -> [..., N] in ``dtype`` (x's): rows of x quantised as by ``quantize_rows``, products and sums in whole numbers, then
    times the row's and the channel's scale, plus ``bias`` (float32 [N])."""
    xt = x.dtype
    dtype = xt if dtype is None else dtype
    if (xt is not BF16 and xt is not F32) or x.dim() < 1 or x.shape[-1] < 1:
        _refuse("int8 linear: activations bfloat16 or float32 [..., K]")
    at, ldw, n, kw = _operand(w, "weights")
    x2 = _rows(x)
    m, k = x2.shape
    if kw != k:
        _refuse("int8 linear: activations and weights have the same inner width")
    _check_channels(n, w_scale, bias)
    if dtype is not BF16 and dtype is not F32:
        _refuse("int8 linear: bfloat16 or float32")
    dev, lib = _device(x, w, w_scale, bias), load()
    out = x.new_empty((m, n) if x2 is x else (*x.shape[:-1], n), dtype=dtype)
    need = lib.xfold_linear_int8_workspace_bytes(m, k)   # (a row or two: none)
    ws = _Workspace.get(dev, need) if need else None
    rc = lib.xfold_linear_int8_fwd(ctx(dev), x2.data_ptr(), xt is F32, _ld(x2), m, k, at, ldw, n, w_scale.data_ptr(), _ptr(bias),
                                   out.data_ptr(), dtype is F32, n, _ptr(ws), need, _stream(dev))
    check(rc, dev, "xfold_linear_int8_fwd")
    return out


def linear_int8_quantized(xq: torch.Tensor, x_scale: torch.Tensor, w: torch.Tensor, w_scale: torch.Tensor,
                          bias: Optional[torch.Tensor] = None, dtype: torch.dtype = BF16) -> torch.Tensor:
    """The product of ``linear_int8`` with rows that are quantised already (``quantize_rows``; one quantisation serves several
    layers): xq int8 [tokens, K], x_scale float32 [tokens]."""
    ax, ldx, m, k = _operand(xq, "activations")
    if x_scale.dtype is not F32 or x_scale.shape != (m,) or not x_scale.is_contiguous():
        _refuse("int8 linear: a float32 scale for each token")
    at, ldw, n, kw = _operand(w, "weights")
    if kw != k:
        _refuse("int8 linear: activations and weights have the same inner width")
    _check_channels(n, w_scale, bias)
    if dtype is not BF16 and dtype is not F32:
        _refuse("int8 linear: bfloat16 or float32")
    dev = _device(xq, x_scale, w, w_scale, bias)
    out = x_scale.new_empty((m, n), dtype=dtype)
    rc = load().xfold_linear_int8_quantized_fwd(ctx(dev), ax, ldx, x_scale.data_ptr(), m, k, at, ldw, n, w_scale.data_ptr(), _ptr(bias),
                                                out.data_ptr(), dtype is F32, n, _stream(dev))
    check(rc, dev, "xfold_linear_int8_quantized_fwd")
    return out
