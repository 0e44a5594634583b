"""CPU: calls of the 8-bit linear layers that are refused before any launch."""
import pytest
import torch

BF, I8 = torch.bfloat16, torch.int8


@pytest.fixture(scope="module")
def Q(pkg):
    from distributed_xfold_b200 import int8_ops
    return int8_ops


def _args(**kw):
    a = dict(x=torch.zeros(3, 32, dtype=BF), w=torch.zeros(5, 32, dtype=I8), w_scale=torch.ones(5), bias=None)
    a.update(kw)
    return a


REFUSED = [
    (dict(x=torch.zeros(3, 32, dtype=torch.float16)), "activations bfloat16 or float32"),
    (dict(x=torch.zeros(3, 0)), "activations bfloat16 or float32"),
    (dict(w=torch.zeros(5, 32)), "weights int8"),
    (dict(w=torch.zeros(5, 30, dtype=I8)), "start at multiples of 16 bytes"),
    (dict(w=torch.zeros(5, 48, dtype=I8)[:, 1:33]), "start at multiples of 16 bytes"),
    (dict(w=torch.zeros(32, 5, dtype=I8).t()), "start at multiples of 16 bytes"),
    (dict(w=torch.zeros(1, 32, dtype=I8).expand(5, -1)), "start at multiples of 16 bytes"),
    (dict(w=torch.zeros(5, 48, dtype=I8)), "the same inner width"),
    (dict(w_scale=torch.ones(4)), "a float32 scale for each output channel"),
    (dict(w_scale=torch.ones(5, dtype=BF)), "a float32 scale for each output channel"),
    (dict(w_scale=torch.ones(10)[::2]), "a float32 scale for each output channel"),
    (dict(bias=torch.ones(4)), "bias is float32"),
    (dict(dtype=torch.float16), "bfloat16 or float32"),
    (dict(), "GPU only"),
]


@pytest.mark.parametrize("kw,what", REFUSED)
def test_refused_linear(Q, kw, what):
    from distributed_xfold_b200._cabi import XfoldError
    with pytest.raises(XfoldError, match=what):
        Q.linear_int8(**_args(**kw))


def test_refused_quantized(Q):
    from distributed_xfold_b200._cabi import XfoldError
    x, w, s = torch.zeros(3, 32, dtype=I8), torch.zeros(5, 32, dtype=I8), torch.ones(5)
    for args, what in (((torch.zeros(3, 32), torch.ones(3), w, s), "activations int8"), ((x, torch.ones(4), w, s), "scale for each token"),
                       ((x[:, :16].contiguous()[:, :10], torch.ones(3), w, s), "the same inner width"), ((x, torch.ones(3), w, s), "GPU only")):
        with pytest.raises(XfoldError, match=what):
            Q.linear_int8_quantized(*args)
    with pytest.raises(XfoldError, match="bfloat16 or float32"):
        Q.quantize_rows(torch.zeros(3, 4, dtype=torch.float64))
    with pytest.raises(XfoldError, match="GPU only"):
        Q.quantize_rows(torch.zeros(3, 4))


@pytest.mark.parametrize("shape,strides", [((5, 1), (0, 1)), ((5, 1), (0, 7)), ((5, 1), (3, 9)), ((1, 1), (0, 0)), ((5, 4), (0, 1)), ((5, 4), (2, 1)), ((1, 4), (0, 1)),
                                           ((5, 4), (8, 2)), ((5, 4), (6, 1)), ((2, 3, 1), (0, 0, 1)), ((2, 3, 4), (0, 4, 1))])
def test_rows_of_activations_lie_in_their_memory(Q, shape, strides):
    """Whatever the strides: the rows that a call hands on, taken one row stride apart, hold x and end where its memory ends."""
    x = torch.as_strided(torch.randn(1 + sum((n - 1) * s for n, s in zip(shape, strides))), shape, strides)
    rows = Q._rows(x)
    m, k = rows.shape
    read = rows.storage_offset() + (m - 1) * Q._ld(rows) + k
    assert read * 4 <= rows.untyped_storage().nbytes()
    assert torch.equal(torch.as_strided(rows, (m, k), (Q._ld(rows), 1)), x.reshape(-1, k))
