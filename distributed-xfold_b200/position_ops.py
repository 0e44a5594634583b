"""Positions in attention: a learned bias of the logits by buckets of relative position (with the gradient of its table), and
the norms of queries and keys for each head together with their rotation by position (with their gradients).

Like the rest of the package these calls are not part of an autograd graph: the backward of each is a call of its own.
"""
from __future__ import annotations

import ctypes as C
from typing import NamedTuple, Optional, Tuple

import torch

from ._cabi import QkNorm, XfoldError, check, ctx, load
from .ops import BF16, _dev, _need_cuda, _ptr, _stream, _Workspace

F32, I32 = torch.float32, torch.int32


def _require(ok: bool, what: str) -> None:
    if not ok:
        raise XfoldError(what)


def _gpu(first: torch.Tensor, *others: Optional[torch.Tensor]) -> None:
    _need_cuda(first, *others)
    for t in others:
        _require(t is None or t.device == first.device, "tensors of one call lie on one device")


# ---------------------------------------------------------------------------------------------
# relative position bias
# ---------------------------------------------------------------------------------------------
def clipped_buckets(max_distance: int) -> Tuple[int, ...]:
    """A bucket for each offset (key minus query) from -max_distance to max_distance; offsets beyond share the last ones."""
    return tuple(range(2 * max_distance + 1))


def logarithmic_buckets(num_buckets: int, max_distance: int, both_sides: bool = True) -> Tuple[int, ...]:
    """Buckets that widen with the distance: half of a side's buckets for single distances, the others for ranges that grow by
    the same factor up to ``max_distance``, beyond which all share the last.  ``both_sides``: keys behind the query have the
    second half of the buckets; otherwise they share the bucket of distance 0.  Borders are found in whole numbers."""
    side = num_buckets // 2 if both_sides else num_buckets
    single = side // 2
    steps = side - single
    _require(single >= 1 and max_distance > single and not (both_sides and num_buckets % 2), "logarithmic buckets: too few, or odd")

    def bucket(n: int) -> int:
        if n < single:
            return n
        if n >= max_distance:
            return side - 1
        # the last step s with n / single >= (max_distance / single) ^ (s / steps)
        return single + max(s for s in range(steps) if n ** steps >= max_distance ** s * single ** (steps - s))

    if both_sides:
        return tuple((side if d > 0 else 0) + bucket(abs(d)) for d in range(-max_distance, max_distance + 1))
    return tuple(bucket(max(-d, 0)) for d in range(-max_distance, max_distance + 1))


def _check_relative(buckets, q_pos, k_pos, q_group, k_group) -> None:
    for t, name in ((buckets, "buckets"), (q_pos, "query positions"), (k_pos, "key positions"), (q_group, "query groups"),
                    (k_group, "key groups")):
        _require(t is None or (t.dtype == I32 and t.dim() == 1 and t.is_contiguous()), f"relative bias: {name} are an int32 vector")
    _require(buckets.numel() % 2 == 1, "relative bias: buckets of the offsets -reach .. reach")
    _require((q_group is None) == (k_group is None), "relative bias: groups of queries and keys come together")
    if q_group is not None:
        _require(q_group.shape == q_pos.shape and k_group.shape == k_pos.shape, "relative bias: a group for each position")


def relative_position_bias(table: torch.Tensor, buckets: torch.Tensor, q_pos: torch.Tensor, k_pos: Optional[torch.Tensor] = None,
                           q_group: Optional[torch.Tensor] = None, k_group: Optional[torch.Tensor] = None, *,
                           dtype: torch.dtype = F32, prepared: bool = False) -> torch.Tensor:
    """out[h, i, j] = table[b(i, j), h] with b the bucket of ``k_pos[j] - q_pos[i]``: ``buckets`` (int32 [2 R + 1], see
    ``clipped_buckets`` and ``logarithmic_buckets``) has those of the offsets -R to R, beyond which the last ones hold.  Where
    the groups differ (chains of a complex) b is the table's last row.  table float32 [buckets, H]; positions int32 [queries],
    [keys] (``k_pos`` None: the queries').

    Returns [H, queries, keys] in float32 or bfloat16, or ``prepared``: float16 [H, queries, pad8(keys)] times log2(e), what
    ``ops.attention_pair_bias_core`` takes (as from ``ops.prepare_pair_bias``).  A bucket that names no row of the table makes
    its entries not a number."""
    if k_pos is None:
        k_pos, k_group = q_pos, (q_group if k_group is None else k_group)
    _require(table.dtype == F32 and table.dim() == 2 and table.is_contiguous(), "relative bias: table is float32 [buckets, heads]")
    _check_relative(buckets, q_pos, k_pos, q_group, k_group)
    _require(prepared or dtype in (F32, BF16), "relative bias: float32 or bfloat16")
    _gpu(table, buckets, q_pos, k_pos, q_group, k_group)
    dev = _dev(table)
    (nb, h), sq, sk = table.shape, q_pos.numel(), k_pos.numel()
    shape = (h, sq, (sk + 7) // 8 * 8 if prepared else sk)
    out = torch.empty(shape, dtype=torch.float16 if prepared else dtype, device=table.device)
    check(load().xfold_relative_bias_fwd(ctx(dev), _ptr(table), nb, h, _ptr(buckets), buckets.numel() // 2, _ptr(q_pos), _ptr(k_pos),
                                         _ptr(q_group), _ptr(k_group), sq, sk, 2 if prepared else int(dtype == BF16), _ptr(out),
                                         _stream(dev)), dev, "xfold_relative_bias_fwd")
    return out


def relative_position_bias_backward(grad: torch.Tensor, num_buckets: int, buckets: torch.Tensor, q_pos: torch.Tensor,
                                    k_pos: Optional[torch.Tensor] = None, q_group: Optional[torch.Tensor] = None,
                                    k_group: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Gradient of the table of ``relative_position_bias``, float32 [num_buckets, H], from that of its result: float32 or bfloat16
    [H, queries, keys], the keys next to each other, heads and queries any stride apart (0 too: a gradient that was
    broadcast).  Sums in 32 bits, in a fixed order."""
    if k_pos is None:
        k_pos, k_group = q_pos, (q_group if k_group is None else k_group)
    _check_relative(buckets, q_pos, k_pos, q_group, k_group)
    _require(grad.dtype in (F32, BF16) and grad.dim() == 3, "relative bias gradient: float32 or bfloat16 [heads, queries, keys]")
    h, sq, sk = grad.shape
    _require(sq == q_pos.numel() and sk == k_pos.numel(), "relative bias gradient: a position for each query and key")
    _gpu(grad, buckets, q_pos, k_pos, q_group, k_group)
    if sk > 1 and grad.stride(2) != 1:
        grad = grad.contiguous()
    dev = _dev(grad)
    lib = load()
    dtable = torch.empty(num_buckets, h, dtype=F32, device=grad.device)
    ws = _Workspace.get(dev, max(lib.xfold_relative_bias_bwd_workspace_bytes(ctx(dev), num_buckets, h, sq, sk), 16))
    check(lib.xfold_relative_bias_bwd(ctx(dev), _ptr(grad), int(grad.dtype == F32), grad.stride(0), grad.stride(1), num_buckets, h,
                                      _ptr(buckets), buckets.numel() // 2, _ptr(q_pos), _ptr(k_pos), _ptr(q_group), _ptr(k_group),
                                      sq, sk, _ptr(dtable), _ptr(ws), ws.numel(), _stream(dev)), dev, "xfold_relative_bias_bwd")
    return dtable


# ---------------------------------------------------------------------------------------------
# norms of queries and keys, rotation
# ---------------------------------------------------------------------------------------------
class Rotation(NamedTuple):
    """Angles of the rotation: ``freqs`` float64 [rot / 2] on the GPU, radians for each position, for the pairs of a head's first
    ``rot`` elements: (i, i + rot / 2), or with ``interleaved`` the neighbours (2 i, 2 i + 1)."""
    freqs: torch.Tensor
    interleaved: bool = False

    @classmethod
    def make(cls, rot: int, base: float = 10000.0, interleaved: bool = False, device="cuda") -> "Rotation":
        half = rot // 2
        return cls(float(base) ** (-torch.arange(half, dtype=torch.float64) / max(half, 1)).to(device), interleaved)


_Strides = C.c_longlong * 3


def _strides(t: torch.Tensor) -> "C.Array":
    s = t.stride()
    return _Strides(s[0], s[1], s[2]) if len(s) == 4 else _Strides(0, s[0], s[1])


def _heads(t: torch.Tensor, like: Optional[torch.Tensor], name: str) -> None:
    _require(t.dim() in (3, 4) and t.dtype in (BF16, F32), f"{name}: bfloat16 or float32 [tokens, heads, width] or [batch, tokens, heads, width]")
    _require(t.stride(-1) == 1 or t.shape[-1] == 1, f"{name}: a head's elements lie next to each other")
    if like is not None:
        _require(t.shape == like.shape and t.dtype == like.dtype, f"{name}: of the same shape and type as its input")


def _qk_norm(q, k, q_weight, k_weight, rotation, positions, eps, q_scale) -> QkNorm:
    _heads(q, None, "queries")
    _heads(k, None, "keys")
    _require(q.dim() == k.dim() and q.dtype == k.dtype and q.shape[:-2] == k.shape[:-2] and q.shape[-1] == k.shape[-1],
             "queries and keys: the same tokens, width and type")
    b, s = (1, q.shape[0]) if q.dim() == 3 else q.shape[:2]
    d = q.shape[-1]
    for w in (q_weight, k_weight):
        _require(w is None or (w.dtype == F32 and tuple(w.shape) == (d,) and w.is_contiguous()), "norm weights: float32 [width]")
    rot, pos_b = 0, 0
    if rotation is not None:
        f = rotation.freqs
        _require(f.dtype == torch.float64 and f.dim() == 1 and f.is_contiguous() and 2 * f.numel() <= d,
                 "rotation: float64 frequencies for pairs of a head's elements")
        rot = 2 * f.numel()
    if positions is not None:
        _require(positions.dtype == I32 and tuple(positions.shape) in ((s,), (b, s)), "positions: int32 [tokens] or [batch, tokens]")
        _require(positions.stride(-1) == 1 or s <= 1, "positions: a sequence's lie next to each other")
        pos_b = positions.stride(0) if positions.dim() == 2 else 0
    _gpu(q, k, q_weight, k_weight, positions, None if rotation is None else rotation.freqs)
    return QkNorm(b, s, q.shape[-2], k.shape[-2], d, rot, int(rotation is not None and rotation.interleaved), int(q.dtype == F32),
                  _ptr(q_weight), _ptr(k_weight), None if rotation is None or not rot else _ptr(rotation.freqs), _ptr(positions), pos_b,
                  eps, q_scale)


def norm_rotate_qk(q: torch.Tensor, k: torch.Tensor, q_weight: Optional[torch.Tensor], k_weight: Optional[torch.Tensor],
                   rotation: Optional[Rotation] = None, positions: Optional[torch.Tensor] = None, *, eps: float = 1e-6,
                   q_scale: float = 1.0, out: Optional[Tuple[torch.Tensor, torch.Tensor]] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """Root-mean-square norm of each head of q and k, times its weight (float32 [width], None: ones) and for q ``q_scale``, then
    the rotation by position, in one pass.  q and k: bfloat16 or float32 [batch, tokens, heads, width] or without the batch, widths
    even up to 256, with as many heads each as they like and any strides between them (views of a fused projection).  positions
    int32 [tokens] or [batch, tokens] (None: 0, 1, ...).  Results are new, or written to ``out``, which may be the inputs."""
    n = _qk_norm(q, k, q_weight, k_weight, rotation, positions, eps, q_scale)
    if out is None:
        out = torch.empty(q.shape, dtype=q.dtype, device=q.device), torch.empty(k.shape, dtype=k.dtype, device=k.device)
    qo, ko = out
    _heads(qo, q, "result of the queries")
    _heads(ko, k, "result of the keys")
    _gpu(q, qo, ko)
    dev = _dev(q)
    check(load().xfold_qk_norm_rotate_fwd(ctx(dev), C.byref(n), _ptr(q), _strides(q), _ptr(k), _strides(k), _ptr(qo), _strides(qo),
                                          _ptr(ko), _strides(ko), _stream(dev)), dev, "xfold_qk_norm_rotate_fwd")
    return qo, ko


def norm_rotate_qk_(q, k, q_weight, k_weight, rotation=None, positions=None, *, eps: float = 1e-6, q_scale: float = 1.0):
    """``norm_rotate_qk`` in place."""
    return norm_rotate_qk(q, k, q_weight, k_weight, rotation, positions, eps=eps, q_scale=q_scale, out=(q, k))


def norm_rotate_qk_backward(dq_out: torch.Tensor, dk_out: torch.Tensor, q: torch.Tensor, k: torch.Tensor,
                            q_weight: Optional[torch.Tensor], k_weight: Optional[torch.Tensor], rotation: Optional[Rotation] = None,
                            positions: Optional[torch.Tensor] = None, *, eps: float = 1e-6, q_scale: float = 1.0):
    """(dq, dk, dq_weight, dk_weight) of ``norm_rotate_qk`` from the gradients of its results; q and k are its inputs (kept, where
    the forward ran in place).  The weights' gradients are float32, summed in a fixed order; None for a weight that is None."""
    n = _qk_norm(q, k, q_weight, k_weight, rotation, positions, eps, q_scale)
    _gpu(q, dq_out, dk_out)
    _require(dq_out.shape == q.shape and dq_out.dtype == q.dtype and dk_out.shape == k.shape and dk_out.dtype == k.dtype,
             "gradients of the results: of the same shape and type as queries and keys")
    if dq_out.stride(-1) != 1:   # (a gradient that was broadcast along the head)
        dq_out = dq_out.contiguous()
    if dk_out.stride(-1) != 1:
        dk_out = dk_out.contiguous()
    dq, dk = torch.empty(q.shape, dtype=q.dtype, device=q.device), torch.empty(k.shape, dtype=k.dtype, device=k.device)
    dqw, dkw = (None if w is None else torch.empty_like(w) for w in (q_weight, k_weight))
    dev = _dev(q)
    lib = load()
    ws = _Workspace.get(dev, lib.xfold_qk_norm_rotate_bwd_workspace_bytes(ctx(dev), n.D))
    check(lib.xfold_qk_norm_rotate_bwd(ctx(dev), C.byref(n), _ptr(dq_out), _strides(dq_out), _ptr(dk_out), _strides(dk_out), _ptr(q),
                                       _strides(q), _ptr(k), _strides(k), _ptr(dq), _strides(dq), _ptr(dk), _strides(dk), _ptr(dqw),
                                       _ptr(dkw), _ptr(ws), ws.numel(), _stream(dev)), dev, "xfold_qk_norm_rotate_bwd")
    return dq, dk, dqw, dkw
