"""CPU: bucket rules of the relative position bias against their definition, and the calls that are refused."""
import math

import pytest
import torch

BF = torch.bfloat16


@pytest.fixture(scope="module")
def P(pkg):
    from distributed_xfold_b200 import position_ops
    return position_ops


def test_clipped_buckets(P):
    b = P.clipped_buckets(3)
    assert b == (0, 1, 2, 3, 4, 5, 6)
    assert P.clipped_buckets(0) == (0,)


@pytest.mark.parametrize("n,far,both", [(32, 128, True), (32, 128, False), (16, 50, True), (6, 4, False), (64, 1000, True), (4, 2, True)])
def test_logarithmic_buckets(P, n, far, both):
    """Against the definition by logarithms, wherever those leave no doubt about the border."""
    b = P.logarithmic_buckets(n, far, both)
    side = n // 2 if both else n
    single = side // 2
    assert len(b) == 2 * far + 1 and 0 <= min(b) and max(b) == n - 1 if both else max(b) == n - 1
    for d in range(-far, far + 1):
        got = b[d + far]
        if both:
            assert (got >= side) == (d > 0)
            got -= side if d > 0 else 0
        dist = abs(d) if both else max(-d, 0)
        if dist < single:
            assert got == dist
            continue
        t = math.log(dist / single) / math.log(far / single) * (side - single)
        want = {min(single + math.floor(t + e), side - 1) for e in (-1e-9, 1e-9)}
        assert got in want
    mono = b[far::-1]
    assert all(x <= y for x, y in zip(mono, mono[1:]))


def test_refused_rules(P):
    from distributed_xfold_b200._cabi import XfoldError
    for args in ((2, 10, True), (33, 128, True), (32, 8, True), (1, 10, False)):
        with pytest.raises(XfoldError, match="logarithmic buckets"):
            P.logarithmic_buckets(*args)


def _bias_args(**kw):
    a = dict(table=torch.zeros(7, 4), buckets=torch.arange(7, dtype=torch.int32), q_pos=torch.arange(5, dtype=torch.int32),
             k_pos=torch.arange(6, dtype=torch.int32), q_group=None, k_group=None)
    a.update(kw)
    return a


@pytest.mark.parametrize("kw,what", [
    (dict(table=torch.zeros(7, 4, dtype=BF)), "table is float32"),
    (dict(table=torch.zeros(4, 7).t()), "table is float32"),
    (dict(buckets=torch.arange(7)), "buckets are an int32 vector"),
    (dict(buckets=torch.arange(6, dtype=torch.int32)), "buckets of the offsets"),
    (dict(q_pos=torch.arange(5).float()), "query positions are an int32"),
    (dict(k_pos=torch.arange(12, dtype=torch.int32)[::2]), "key positions are an int32"),
    (dict(q_group=torch.zeros(5, dtype=torch.int32)), "groups of queries and keys come together"),
    (dict(q_group=torch.zeros(5, dtype=torch.int32), k_group=torch.zeros(5, dtype=torch.int32)), "a group for each position"),
    (dict(dtype=torch.float64), "float32 or bfloat16"),
    (dict(), "GPU only"),
])
def test_refused_bias(P, kw, what):
    from distributed_xfold_b200._cabi import XfoldError
    with pytest.raises(XfoldError, match=what):
        P.relative_position_bias(**_bias_args(**kw))


@pytest.mark.parametrize("kw,what", [
    (dict(grad=torch.zeros(4, 5, 6, dtype=torch.float16)), "float32 or bfloat16"),
    (dict(grad=torch.zeros(5, 6)), "float32 or bfloat16"),
    (dict(grad=torch.zeros(4, 6, 5)), "a position for each"),
    (dict(), "GPU only"),
])
def test_refused_bias_backward(P, kw, what):
    from distributed_xfold_b200._cabi import XfoldError
    a = _bias_args(grad=torch.zeros(4, 5, 6), num_buckets=7, **kw) if not kw else {**_bias_args(num_buckets=7), **kw}
    a.pop("table")
    with pytest.raises(XfoldError, match=what):
        P.relative_position_bias_backward(**a)


def _qk(**kw):
    a = dict(q=torch.zeros(2, 5, 4, 8, dtype=BF), k=torch.zeros(2, 5, 2, 8, dtype=BF), q_weight=torch.ones(8), k_weight=None,
             rotation=None, positions=None)
    a.update(kw)
    return a


@pytest.mark.parametrize("kw,what", [
    (dict(q=torch.zeros(2, 5, 4, 8, dtype=torch.float16)), "bfloat16 or float32"),
    (dict(q=torch.zeros(5, 8)), "bfloat16 or float32"),
    (dict(q=torch.zeros(2, 5, 8, 4, dtype=BF).transpose(2, 3)), "elements lie next"),
    (dict(k=torch.zeros(2, 5, 2, 8)), "the same tokens, width and type"),
    (dict(k=torch.zeros(2, 6, 2, 8, dtype=BF)), "the same tokens, width and type"),
    (dict(k=torch.zeros(2, 5, 2, 6, dtype=BF)), "the same tokens, width and type"),
    (dict(q_weight=torch.ones(8, dtype=BF)), "norm weights"),
    (dict(k_weight=torch.ones(6)), "norm weights"),
    (dict(freqs=torch.ones(4)), "float64 frequencies"),
    (dict(freqs=torch.ones(5, dtype=torch.float64)), "float64 frequencies"),
    (dict(positions=torch.arange(5)), "positions: int32"),
    (dict(positions=torch.arange(10, dtype=torch.int32)), "positions: int32"),
    (dict(out=(torch.zeros(2, 5, 4, 8), torch.zeros(2, 5, 2, 8, dtype=BF))), "shape and type as its input"),
    (dict(), "GPU only"),
])
def test_refused_qk(P, kw, what):
    from distributed_xfold_b200._cabi import XfoldError
    if "freqs" in kw:
        kw["rotation"] = P.Rotation(kw.pop("freqs"))
    with pytest.raises(XfoldError, match=what if "out" not in kw else "GPU only"):
        P.norm_rotate_qk(**_qk(**kw))


def test_rotation_of_a_base(P):
    r = P.Rotation.make(8, base=100.0, device="cpu")
    assert r.freqs.dtype == torch.float64 and not r.interleaved
    assert torch.allclose(r.freqs, torch.tensor([1.0, 100 ** -0.25, 100 ** -0.5, 100 ** -0.75], dtype=torch.float64))


def _places(t):
    """Bytes of a tensor's elements."""
    at = torch.zeros(t.shape, dtype=torch.int64)
    for axis, (n, st) in enumerate(zip(t.shape, t.stride())):
        at += (torch.arange(n) * st).view(-1, *[1] * (t.dim() - 1 - axis))
    return ((at.flatten() + t.storage_offset()) * t.element_size()).tolist()


@pytest.mark.parametrize("dtype", [BF, torch.float32])
def test_where_tensors_lie(P, dtype):
    """Whether two views of one buffer meet, and whether a view has a place for each element, against all of their places."""
    g = torch.Generator().manual_seed(7)
    pick = lambda *n: n[int(torch.randint(0, len(n), (1,), generator=g))]
    buf, seen, at_once = torch.zeros(200000, dtype=dtype), {}, 0
    for _ in range(3000):
        dims = pick(3, 4)
        shape = [pick(1, 2, 3, 5) for _ in range(dims)]
        views = []
        for _ in range(2):
            strides, inner = [0] * dims, 1
            for axis in ([dims - 1, *torch.randperm(dims - 1, generator=g).tolist()] if pick(0, 1) else range(dims - 1, -1, -1)):
                strides[axis] = pick(inner, inner, inner, inner + 1, 2 * inner, max(inner - 1, 0), 0, pick(2, 3, 7))
                inner = max(inner, strides[axis] * shape[axis])
            if len(views) == 1 and pick(0, 1):
                strides = list(views[0].stride())
                shape[-2] = pick(1, 2, 3)
            views.append(torch.as_strided(buf, shape, strides, pick(0, 0, 1, 2, 6, 12, 30, 31, 64)))
        a, b = views
        pa, pb = _places(a), _places(b)
        assert P._meet(a, b) == bool(set(pa) & set(pb)) == P._meet(b, a)
        assert P._one_place_each(a) == (len(set(pa)) == len(pa))
        if dims == 4 and a.shape[:2] == b.shape[:2] and a.shape[3] == b.shape[3]:   # what is seen at once is so
            d = a.shape[3]
            if P._side_by_side(*a.shape[:2], a.shape[2], b.shape[2], d, a.element_size(), *(x for t in views for x in (t.data_ptr(), *t.stride()[:3]))) \
                    and all(d == 1 or t.stride(3) == 1 for t in views):
                assert not P._meet(a, b) and P._one_place_each(a) and P._one_place_each(b)
                at_once += 1
        seen[P._meet(a, b), P._one_place_each(a)] = seen.get((P._meet(a, b), P._one_place_each(a)), 0) + 1
    assert min(seen.values()) > 100 and len(seen) == 4 and at_once > 20, (seen, at_once)


def test_where_large_tensors_lie(P):
    """Projections of many tokens: queries and keys side by side, one shifted by an element, transposed, in another order."""
    store = torch.empty(4 * 4096 * 8192, dtype=BF)   # (never touched)
    view = lambda shape, strides, offset=0: store.as_strided(shape, strides, offset)
    q, k = view((4, 4096, 32, 128), (4096 * 8192, 8192, 128, 1)), view((4, 4096, 8, 128), (4096 * 8192, 8192, 128, 1), 4096)
    assert not P._meet(q, k) and not P._meet(k, q) and P._one_place_each(q) and P._one_place_each(k)
    for a, b in ((q, k), (k, q)):
        lies = lambda t: (t.data_ptr(), *t.stride()[:3])
        assert P._side_by_side(4, 4096, a.shape[2], b.shape[2], 128, 2, *lies(a), *lies(b))
        assert not P._side_by_side(4, 4096, a.shape[2], b.shape[2], 128, 2, *lies(a), a.data_ptr(), *lies(b)[1:])
    assert P._meet(q, view((4, 4096, 8, 128), (4096 * 8192, 8192, 128, 1), 4095))
    padded = [view((4, 4096, 16, 48), (4096 * 8192, 8192, 128, 1), at) for at in (0, 48, 2048)]
    assert not any(P._meet(x, y) for i, x in enumerate(padded) for y in padded[:i])
    assert P._meet(padded[0], view((4, 4096, 16, 48), (4096 * 8192, 8192, 128, 1), 47))
    long = view((1, 16384, 32, 128), (0, 8192, 128, 1))
    assert P._meet(long, q) and not P._meet(long, k)
    other = view((4, 4096, 8, 128), (8192, 4 * 8192, 128, 1), 4096)   # tokens before the batch
    assert not P._meet(q, other) and P._meet(k, other) and P._one_place_each(other)
    assert not P._one_place_each(view((4, 4096, 32, 128), (4096 * 8192, 8192, 127, 1)))
    square = view((64, 64, 8), (512, 8, 1))
    assert P._same_view(square, view((64, 64, 8), (512, 8, 1))) and not P._same_view(square, square.transpose(0, 1))
    assert P._same_view(view((1, 5, 3, 8), (7, 24, 8, 1)), view((1, 5, 3, 8), (120, 24, 8, 1)))
    raw = torch.empty(40, dtype=torch.uint8)
    a, b = raw[:16].view(BF), raw[16:32].view(BF)
    assert not P._meet(a, b) and P._meet(a, raw[14:30].view(BF))
