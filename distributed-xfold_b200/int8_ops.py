"""Linear layers in 8-bit integers: weights with a scale for each output channel, activations quantised in the call with a scale
for each token."""
from __future__ import annotations

from typing import Optional, Tuple

import torch

from ._cabi import XfoldError, check, ctx, load
from .ops import BF16, _dev, _need_cuda, _ptr, _stream, _Workspace

F32, I8 = torch.float32, torch.int8


def _require(ok: bool, what: str) -> None:
    if not ok:
        raise XfoldError(what)


def _gpu(first: torch.Tensor, *others: Optional[torch.Tensor]) -> None:
    _need_cuda(first, *others)
    for t in others:
        _require(t is None or t.device == first.device, "tensors of one call lie on one device")


def _rows(x: torch.Tensor) -> torch.Tensor:
    """[..., K] as rows that are one stride apart, their elements next to each other."""
    x2 = x if x.dim() == 2 else x.reshape(-1, x.shape[-1])
    return x2 if x2.shape[1] <= 1 or (x2.stride(1) == 1 and x2.stride(0) >= x2.shape[1]) else x2.contiguous()


def _ld(x2: torch.Tensor) -> int:
    return x2.stride(0) if x2.shape[0] > 1 else max(x2.stride(0), x2.shape[1])


def quantize_rows(x: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
    """(q, scale) of x bfloat16 or float32 [..., K]: scale float32 [...] = max |x| / 127 of each row, q int8 [..., K] = x / scale
    rounded to the nearest whole number, ties to even.  q's rows are a multiple of 16 bytes apart, as ``linear_int8`` wants its
    weights (a row for each output channel) and ``linear_int8_quantized`` both operands.  A row of zeros has scale 0, one that
    holds something not finite scale NaN and zeros."""
    _require(x.dtype in (BF16, F32) and x.dim() >= 1 and x.shape[-1] >= 1, "quantize rows: bfloat16 or float32 [..., K]")
    _gpu(x)
    x2 = _rows(x)
    m, k = x2.shape
    kp = (k + 15) // 16 * 16
    q = torch.empty(m, kp, dtype=I8, device=x.device)
    scale = torch.empty(x.shape[:-1], dtype=F32, device=x.device)
    dev = _dev(x)
    check(load().xfold_quantize_rows_fwd(ctx(dev), _ptr(x2), int(x.dtype == F32), _ld(x2), m, k, _ptr(q), kp, _ptr(scale), _stream(dev)),
          dev, "xfold_quantize_rows_fwd")
    return q.view(*x.shape[:-1], kp)[..., :k], scale


def _operand(t: torch.Tensor, what: str) -> torch.Tensor:
    """int8 rows for the kernel, 16-byte aligned, whose memory goes on to a multiple of 16 bytes behind the last."""
    _require(t.dtype == I8 and t.dim() == 2, f"int8 linear: {what} int8 [rows, K]")
    ok = (t.stride(1) == 1 or t.shape[1] == 1) and (t.shape[0] <= 1 or (t.stride(0) % 16 == 0 and t.stride(0) >= t.shape[1]))
    _require(ok and t.data_ptr() % 16 == 0, f"int8 linear: rows of {what} start at multiples of 16 bytes (as quantize_rows leaves them)")
    return t


def _ld16(t: torch.Tensor) -> int:
    return t.stride(0) if t.shape[0] > 1 else (t.shape[1] + 15) // 16 * 16


def _check_linear(k: int, w, w_scale, bias, dtype) -> None:
    _operand(w, "weights")
    _require(w.shape[1] == k, "int8 linear: activations and weights have the same inner width")
    n = w.shape[0]
    _require(w_scale.dtype == F32 and tuple(w_scale.shape) == (n,) and w_scale.is_contiguous(), "int8 linear: a float32 scale for each output channel")
    _require(bias is None or (bias.dtype == F32 and tuple(bias.shape) == (n,) and bias.is_contiguous()), "int8 linear: bias is float32 [channels]")
    _require(dtype in (BF16, F32), "int8 linear: bfloat16 or float32")


def linear_int8(x: torch.Tensor, w: torch.Tensor, w_scale: torch.Tensor, bias: Optional[torch.Tensor] = None,
                dtype: Optional[torch.dtype] = None) -> torch.Tensor:
    """x bfloat16 or float32 [..., K], w int8 [N, K] (rows a multiple of 16 bytes apart, see ``quantize_rows``), w_scale float32
    [N] -> [..., N] in ``dtype`` (x's): rows of x quantised as by ``quantize_rows``, products and sums in whole numbers, then
    times the row's and the channel's scale, plus ``bias`` (float32 [N])."""
    dtype = x.dtype if dtype is None else dtype
    _require(x.dtype in (BF16, F32) and x.dim() >= 1 and x.shape[-1] >= 1, "int8 linear: activations bfloat16 or float32 [..., K]")
    _check_linear(x.shape[-1], w, w_scale, bias, dtype)
    _gpu(x, w, w_scale, bias)
    x2 = _rows(x)
    (m, k), n, dev, lib = x2.shape, w.shape[0], _dev(x), load()
    out = torch.empty(*x.shape[:-1], n, dtype=dtype, device=x.device)
    ws = _Workspace.get(dev, lib.xfold_linear_int8_workspace_bytes(m, k))
    check(lib.xfold_linear_int8_fwd(ctx(dev), _ptr(x2), int(x.dtype == F32), _ld(x2), m, k, _ptr(w), _ld16(w), n, _ptr(w_scale), _ptr(bias),
                                    _ptr(out), int(dtype == F32), n, _ptr(ws), ws.numel(), _stream(dev)), dev, "xfold_linear_int8_fwd")
    return out


def linear_int8_quantized(xq: torch.Tensor, x_scale: torch.Tensor, w: torch.Tensor, w_scale: torch.Tensor,
                          bias: Optional[torch.Tensor] = None, dtype: torch.dtype = BF16) -> torch.Tensor:
    """The product of ``linear_int8`` with rows that are quantised already (``quantize_rows``; one quantisation serves several
    layers): xq int8 [tokens, K], x_scale float32 [tokens]."""
    _operand(xq, "activations")
    m, k = xq.shape
    _require(x_scale.dtype == F32 and tuple(x_scale.shape) == (m,) and x_scale.is_contiguous(), "int8 linear: a float32 scale for each token")
    _check_linear(k, w, w_scale, bias, dtype)
    _gpu(xq, x_scale, w, w_scale, bias)
    n, dev = w.shape[0], _dev(xq)
    out = torch.empty(m, n, dtype=dtype, device=xq.device)
    check(load().xfold_linear_int8_quantized_fwd(ctx(dev), _ptr(xq), _ld16(xq), _ptr(x_scale), m, k, _ptr(w), _ld16(w), n, _ptr(w_scale),
                                                 _ptr(bias), _ptr(out), int(dtype == F32), n, _stream(dev)), dev,
          "xfold_linear_int8_quantized_fwd")
    return out
