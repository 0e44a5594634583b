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
