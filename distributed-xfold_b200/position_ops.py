"""Positions in attention: a learned bias of the logits by buckets of relative position (with the gradient of its table), and
the norms of queries and keys for each head together with their rotation by position (with their gradients).

Like the rest of the package these calls are not part of an autograd graph, whether their inputs require gradients or not: the
backward of each is a call of its own, which a user's ``torch.autograd.Function`` may make.
"""
from __future__ import annotations

from typing import NamedTuple, Optional, Tuple

import torch

from ._cabi import QK_NORM, XfoldError, check, ctx, load
from .ops import BF16, _need_cuda, _ptr, _stream, _Workspace

F32, I32 = torch.float32, torch.int32


def _refuse(what: str):
    raise XfoldError(what)


def _device(first: torch.Tensor, *others: Optional[torch.Tensor]) -> int:
    dev = first.get_device()
    for t in others:
        if t is not None and t.get_device() != dev:
            _need_cuda(first, *others)
            _refuse("tensors of one call lie on one device")
    if dev < 0:
        _need_cuda(first)
    return dev


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
    if single < 1 or max_distance <= single or (both_sides and num_buckets % 2):
        _refuse("logarithmic buckets: too few, or odd")

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


def _vector(t: torch.Tensor, name: str) -> int:
    if t.dtype is not I32 or (t.stride() != (1,) and (t.dim() != 1 or t.numel() > 1)):
        _refuse("relative bias: " + name + " are an int32 vector")
    return t.numel()


def _check_relative(buckets, q_pos, k_pos, q_group, k_group) -> Tuple[int, int, int]:
    """(reach, queries, keys)"""
    n, sq, sk = _vector(buckets, "buckets"), _vector(q_pos, "query positions"), _vector(k_pos, "key positions")
    if n % 2 == 0:
        _refuse("relative bias: buckets of the offsets -reach .. reach")
    if (q_group is None) is not (k_group is None):
        _refuse("relative bias: groups of queries and keys come together")
    if q_group is not None and (_vector(q_group, "query groups") != sq or _vector(k_group, "key groups") != sk):
        _refuse("relative bias: a group for each position")
    return n // 2, sq, sk


def relative_position_bias(table: torch.Tensor, buckets: torch.Tensor, q_pos: torch.Tensor, k_pos: Optional[torch.Tensor] = None,
                           q_group: Optional[torch.Tensor] = None, k_group: Optional[torch.Tensor] = None, *,
                           dtype: torch.dtype = F32, prepared: bool = False) -> torch.Tensor:
    """out[h, i, j] = table[b(i, j), h] with b the bucket of ``k_pos[j] - q_pos[i]``: ``buckets`` (int32 [2 R + 1], see
    ``clipped_buckets`` and ``logarithmic_buckets``) has those of the offsets -R to R, beyond which the last ones hold.  Where
    the groups differ (chains of a complex) b is the table's last row.  table float32 [buckets, H]; positions int32 [queries],
    [keys] (``k_pos`` None: the queries').

    Returns [H, queries, keys] in float32 or bfloat16, or ``prepared``: float16 [H, queries, pad8(keys)] times log2(e), what
    ``ops.attention_pair_bias_core`` takes (as from ``ops.prepare_pair_bias``).  A bucket that names no row of the table makes
    its entries not a number.  In the prepared form numbers end at +-60000, and what is not a number is -60000, as in
    ``ops.prepare_pair_bias``: such a key is masked, and no error shows."""
    if k_pos is None:
        k_pos, k_group = q_pos, (q_group if k_group is None else k_group)
    if table.dtype is not F32 or table.dim() != 2 or not table.is_contiguous():
        _refuse("relative bias: table is float32 [buckets, heads]")
    reach, sq, sk = _check_relative(buckets, q_pos, k_pos, q_group, k_group)
    nb, h = table.shape
    if prepared:
        out, form = (h, sq, (sk + 7) // 8 * 8), 2
    else:
        out, form = (h, sq, sk), 0 if dtype is F32 else 1 if dtype is BF16 else _refuse("relative bias: float32 or bfloat16")
    dev = _device(table, buckets, q_pos, k_pos, q_group, k_group)
    out = table.new_empty(out) if form == 0 else table.new_empty(out, dtype=torch.float16 if prepared else dtype)
    rc = load().xfold_relative_bias_fwd(ctx(dev), table.data_ptr(), nb, h, buckets.data_ptr(), reach, q_pos.data_ptr(), k_pos.data_ptr(),
                                        _ptr(q_group), _ptr(k_group), sq, sk, form, out.data_ptr(), _stream(dev))
    check(rc, dev, "xfold_relative_bias_fwd")
    return out


def relative_position_bias_backward(grad: torch.Tensor, num_buckets: int, buckets: torch.Tensor, q_pos: torch.Tensor,
                                    k_pos: Optional[torch.Tensor] = None, q_group: Optional[torch.Tensor] = None,
                                    k_group: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Gradient of the table of ``relative_position_bias``, float32 [num_buckets, H], from that of its result: float32 or bfloat16
    [H, queries, keys], the keys next to each other, heads and queries any stride apart (0 too: a gradient that was
    broadcast).  Sums in 32 bits, in a fixed order."""
    if k_pos is None:
        k_pos, k_group = q_pos, (q_group if k_group is None else k_group)
    reach, sq, sk = _check_relative(buckets, q_pos, k_pos, q_group, k_group)
    f32 = grad.dtype is F32
    if not (f32 or grad.dtype is BF16) or grad.dim() != 3:
        _refuse("relative bias gradient: float32 or bfloat16 [heads, queries, keys]")
    h = grad.shape[0]
    if grad.shape[1] != sq or grad.shape[2] != sk:
        _refuse("relative bias gradient: a position for each query and key")
    dev = _device(grad, buckets, q_pos, k_pos, q_group, k_group)
    if sk > 1 and grad.stride(2) != 1:
        grad = grad.contiguous()
    sh, sr, _ = grad.stride()
    lib, c = load(), ctx(dev)
    dtable = q_pos.new_empty((num_buckets, h), dtype=F32)
    ws = _Workspace.get(dev, lib.xfold_relative_bias_bwd_workspace_bytes(c, num_buckets, h, sq, sk) or 16)
    rc = lib.xfold_relative_bias_bwd(c, grad.data_ptr(), f32, sh, sr, num_buckets, h, buckets.data_ptr(), reach, q_pos.data_ptr(),
                                     k_pos.data_ptr(), _ptr(q_group), _ptr(k_group), sq, sk, dtable.data_ptr(), ws.data_ptr(), ws.numel(),
                                     _stream(dev))
    check(rc, dev, "xfold_relative_bias_bwd")
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


def _heads(t: torch.Tensor, name: str) -> Tuple[int, int, int, int]:
    """(address, strides of batch, tokens and heads)"""
    s = t.stride()
    if len(s) == 4:
        b, n, h, e = s
    elif len(s) == 3:
        (n, h, e), b = s, 0
    else:
        _refuse(name + ": bfloat16 or float32 [tokens, heads, width] or [batch, tokens, heads, width]")
    if e != 1 and t.shape[-1] > 1:
        _refuse(name + ": a head's elements lie next to each other")
    return t.data_ptr(), b, n, h


def _qk_norm(q, k, q_weight, k_weight, rotation, positions, eps, q_scale):
    """(device, the call's description up to q and k)"""
    at_q, at_k = _heads(q, "queries"), _heads(k, "keys")
    shape, of_k, dt = q.shape, k.shape, q.dtype
    if dt is not BF16 and dt is not F32:
        _refuse("queries and keys: bfloat16 or float32 [tokens, heads, width] or [batch, tokens, heads, width]")
    if len(shape) == 3:
        shape, of_k = (1, *shape), (1, *of_k)
    b, s, hq, d = shape
    hk = of_k[-2]
    if of_k != (b, s, hk, d) or k.dtype is not dt or q.dim() != k.dim():
        _refuse("queries and keys: the same tokens, width and type")
    dev = q.get_device()
    same = k.get_device() == dev
    qw = kw = rot = inter = freqs = pos = pos_b = 0
    if q_weight is not None:
        qw, same = _weight(q_weight, d), same and q_weight.get_device() == dev
    if k_weight is not None:
        kw, same = _weight(k_weight, d), same and k_weight.get_device() == dev
    if rotation is not None:
        f, inter = rotation
        rot = 2 * f.numel()
        if f.dtype is not torch.float64 or f.dim() != 1 or rot > d or (f.stride(0) != 1 and rot > 2):
            _refuse("rotation: float64 frequencies for pairs of a head's elements")
        freqs, same = f.data_ptr(), same and f.get_device() == dev
    if positions is not None:
        step = positions.stride()
        if positions.dtype is not I32 or positions.shape != ((s,) if len(step) == 1 else (b, s)):
            _refuse("positions: int32 [tokens] or [batch, tokens]")
        if step[-1] != 1 and s > 1:
            _refuse("positions: a sequence's lie next to each other")
        pos, pos_b, same = positions.data_ptr(), step[0] if len(step) == 2 else 0, same and positions.get_device() == dev
    if dev < 0 or not same:
        _device(q, k, q_weight, k_weight, positions, None if rotation is None else f)
    return dev, (b, s, hq, hk, d, rot, bool(inter), dt is F32, qw, kw, freqs, pos, pos_b, eps, q_scale, *at_q, *at_k)


def _new(x: torch.Tensor) -> torch.Tensor:
    return torch.empty_like(x, memory_format=torch.contiguous_format)   # (half the host time of new_empty)


def _reaches(steps, at: int) -> bool:
    """Whether at + sum step * n can be 0, for whole numbers first <= n <= last of each (step, first, last).  Past some thousands
    of tries: yes.  (Axes that lie within each other leave two or three tries for each.)"""
    one = []
    for step, first, last in sorted(steps):
        if one and step % one[-1][0] == 0 and one[-1][2] - one[-1][1] + 1 >= step // one[-1][0]:   # together: every multiple of the shorter
            short, a, b = one.pop()
            step, first, last = short, a + first * (step // short), b + last * (step // short)
        one.append((step, first, last))
    steps = one[::-1]
    ends = [(0, 0)]   # what the steps from each on can add
    for step, first, last in reversed(steps):
        ends.append((ends[-1][0] + step * first, ends[-1][1] + step * last))
    ends.reverse()
    tries = 4096

    def find(i: int, at: int) -> bool:
        nonlocal tries
        tries -= 1
        if tries < 0 or i == len(steps):
            return tries < 0 or at == 0
        step, first, last = steps[i]
        down, up = ends[i + 1]
        return any(find(i + 1, at + step * n) for n in range(max(first, -((at + up) // step)), min(last, (-at - down) // step) + 1))

    return find(0, at)


def _axes(t: torch.Tensor):
    return [(st, n - 1) for st, n in zip(t.stride(), t.shape) if n > 1]


def _meet(a: torch.Tensor, b: torch.Tensor) -> bool:
    """Whether an element of one lies where one of the other does (both of one type)."""
    if not (a.numel() and b.numel()):
        return False
    (ra, rb), size = (_axes(a), _axes(b)), a.element_size()
    at, odd = divmod(b.data_ptr() - a.data_ptr(), size)
    if at > sum(st * n for st, n in ra) or at + 1 < -sum(st * n for st, n in rb):
        return False
    steps = {}
    for st, n in rb:
        steps[st] = (0, n) if st not in steps else (0, steps[st][1] + n)
    for st, n in ra:
        first, last = steps.get(st, (0, 0))
        steps[st] = (first - n, last)
    steps = [(st, *n) for st, n in steps.items() if st]
    return _reaches(steps, at) or (odd > 0 and _reaches(steps, at + 1))


def _one_place_each(t: torch.Tensor) -> bool:
    axes, wide = sorted(_axes(t)), 1
    for st, n in axes:
        if st < wide:
            break
        wide += st * n
    else:
        return True
    # not one axis within the other: two elements share a place where steps that are not all none lead nowhere
    return not t.numel() or not any(_reaches([(st, -n, n) for st, n in axes[:i] if st] + [(axes[i][0], 1, axes[i][1])], 0) if axes[i][0] else True
                                    for i in range(len(axes)))


def _side_by_side(b: int, s: int, hq: int, hk: int, d: int, size: int, pq: int, qb: int, qt: int, qh: int, pk: int, kb: int, kt: int, kh: int) -> bool:
    """Whether queries and keys by their sizes, addresses and strides are seen at once to have a place for each element: tensors one
    behind the other, or heads side by side in the rows of one projection, as nearly all are.  (Not seen so: they may still.)"""
    if hq < 1 or hk < 1 or b < 1 or s < 1:
        return False
    wq, wk = (hq - 1) * qh + d, (hk - 1) * kh + d
    if qh < d or kh < d or (s > 1 and (qt < wq or kt < wk)) or (b > 1 and (qb < (s - 1) * qt + wq or kb < (s - 1) * kt + wk)):
        return False
    at = pk - pq
    if at >= ((b - 1) * qb + (s - 1) * qt + wq) * size or -at >= ((b - 1) * kb + (s - 1) * kt + wk) * size:
        return True
    # (rows as long as their distance, of which both have a part)
    return (qt == kt and (b == 1 or (qb == kb and qb >= s * qt))
            and (wq * size <= at <= (qt - wk) * size or wk * size <= -at <= (qt - wq) * size))


def _same_view(a: torch.Tensor, b: torch.Tensor) -> bool:
    return a.data_ptr() == b.data_ptr() and _axes(a) == _axes(b)


def _result(o: torch.Tensor, x: torch.Tensor, dev: int, name: str) -> Tuple[int, int, int, int]:
    if o.shape != x.shape or o.dtype is not x.dtype or o.get_device() != dev:
        _refuse("results of queries and keys: shape, type and device of their inputs")
    return _heads(o, name)


def _check_results(q, k, qo, ko, sizes, at_q, at_k, at_qo, at_ko) -> None:
    """Refuses results without a place for each element, or that meet what is read."""
    b, s, hq, hk, d, size = sizes
    if _side_by_side(*sizes, *at_qo, *at_ko) and (
            at_ko == at_k or _side_by_side(*sizes, *at_qo, *at_k) and _side_by_side(b, s, hk, hk, d, size, *at_ko, *at_k)) and (
            at_qo == at_q or _side_by_side(*sizes, *at_q, *at_ko) and _side_by_side(b, s, hq, hq, d, size, *at_qo, *at_q)):
        return
    for o in (qo, ko):
        if not _one_place_each(o):
            _refuse("results of queries and keys: one place for each element")
    if _meet(qo, ko) or _meet(qo, k) or _meet(ko, q) or any(not _same_view(o, x) and _meet(o, x) for o, x in ((qo, q), (ko, k))):
        _refuse("results of queries and keys: new, or each over its own input")


def _weight(w: torch.Tensor, d: int) -> int:
    if w.dtype is not F32 or w.shape != (d,) or (w.stride(0) != 1 and d > 1):
        _refuse("norm weights: float32 [width]")
    return w.data_ptr()


def norm_rotate_qk(q: torch.Tensor, k: torch.Tensor, q_weight: Optional[torch.Tensor], k_weight: Optional[torch.Tensor],
                   rotation: Optional[Rotation] = None, positions: Optional[torch.Tensor] = None, *, eps: float = 1e-6,
                   q_scale: float = 1.0, out: Optional[Tuple[torch.Tensor, torch.Tensor]] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """Root-mean-square norm of each head of q and k, times its weight (float32 [width], None: ones) and for q ``q_scale``, then
    the rotation by position, in one pass.  q and k: bfloat16 or float32 [batch, tokens, heads, width] or without the batch, widths
    even up to 256, with as many heads each as they like and any strides between them (views of a fused projection).  positions
    int32 [tokens] or [batch, tokens] (None: 0, 1, ...).  Results are new, or written to ``out``, each of which may be
    its own input (the same view of it) and otherwise lies apart from the inputs and from the other."""
    dev, n = _qk_norm(q, k, q_weight, k_weight, rotation, positions, eps, q_scale)
    at = n[-8:]   # where queries, keys and results lie
    if out is None:
        qo, ko = _new(q), _new(k)
        at += _heads(qo, "") + _heads(ko, "")
    else:
        qo, ko = out
        if qo is not q or ko is not k:
            at += _result(qo, q, dev, "result of the queries") + _result(ko, k, dev, "result of the keys")
        _check_results(q, k, qo, ko, n[:5] + (4 if n[7] else 2,), at[:4], at[4:8], at[-8:-4], at[-4:])
    rc = load().xfold_qk_norm_rotate_fwd(ctx(dev), QK_NORM.pack(*n, *at[-8:], 0, 0, 0, 0, 0, 0, 0, 0), _stream(dev))
    check(rc, dev, "xfold_qk_norm_rotate_fwd")
    return qo, ko


def norm_rotate_qk_(q, k, q_weight, k_weight, rotation=None, positions=None, *, eps: float = 1e-6, q_scale: float = 1.0):
    """``norm_rotate_qk`` in place."""
    return norm_rotate_qk(q, k, q_weight, k_weight, rotation, positions, eps=eps, q_scale=q_scale, out=(q, k))


def norm_rotate_qk_backward(dq_out: torch.Tensor, dk_out: torch.Tensor, q: torch.Tensor, k: torch.Tensor,
                            q_weight: Optional[torch.Tensor], k_weight: Optional[torch.Tensor], rotation: Optional[Rotation] = None,
                            positions: Optional[torch.Tensor] = None, *, eps: float = 1e-6, q_scale: float = 1.0):
    """(dq, dk, dq_weight, dk_weight) of ``norm_rotate_qk`` from the gradients of its results; q and k are its inputs (kept, where
    the forward ran in place).  The weights' gradients are float32, summed in a fixed order; None for a weight that is None."""
    dev, n = _qk_norm(q, k, q_weight, k_weight, rotation, positions, eps, q_scale)
    for g, x in ((dq_out, q), (dk_out, k)):
        if g.shape != x.shape or g.dtype is not x.dtype or g.get_device() != dev:
            _refuse("gradients of the results: shape, type and device of queries and keys")
    if dq_out.stride(-1) != 1:   # (a gradient that was broadcast along the head)
        dq_out = dq_out.contiguous()
    if dk_out.stride(-1) != 1:
        dk_out = dk_out.contiguous()
    dq, dk = _new(q), _new(k)
    dqw = None if q_weight is None else _new(q_weight)
    dkw = None if k_weight is None else _new(k_weight)
    lib, c = load(), ctx(dev)
    ws = _Workspace.get(dev, lib.xfold_qk_norm_rotate_bwd_workspace_bytes(c, n[4]))
    desc = QK_NORM.pack(*n, *_heads(dq, ""), *_heads(dk, ""), *_heads(dq_out, ""), *_heads(dk_out, ""))
    rc = lib.xfold_qk_norm_rotate_bwd(c, desc, _ptr(dqw), _ptr(dkw), ws.data_ptr(), ws.numel(), _stream(dev))
    check(rc, dev, "xfold_qk_norm_rotate_bwd")
    return dq, dk, dqw, dkw
