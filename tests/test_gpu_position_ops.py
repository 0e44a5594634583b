"""GPU: relative position bias, norms and rotation of queries and keys, and their gradients, against plain forms in 64 bits.

Tolerances.  u = 2^-24 is the step of a float32 rounding, h the half step of the result's type (bf16 2^-8, float32 u).
  bias: the table's numbers as they are, rounded once: equal.
  its gradient: whole numbers whose sums stay below 2^24 are exact in any order: equal.  Otherwise a chain of n additions is off
      by at most n u times the sum of the absolute values.
  norm and rotation: sum of squares (chains of up to 21 additions and products) 22 u, half of that after the root, rsqrt 4 u, three
      products 3 u; the angle's rounding in turns 2 u and sincospi 2 u each, products and sum of the rotation 3 u: below 32 u of
      the rotated pair's length, then h of the result.
  gradients of q and k: the same factors, two sums over the head and one more product each: 96 u of r (|g w| + |x| r^2 mean |g w x|).
"""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
BF, F32, F64 = torch.bfloat16, torch.float32, torch.float64
U = 2.0 ** -24
HALF = {BF: 2.0 ** -8, F32: U}


@pytest.fixture(scope="module")
def P(ops):
    from distributed_xfold_b200 import position_ops
    return position_ops


def gen(seed):
    return torch.Generator().manual_seed(seed)


# ---------------------------------------------------------------------------------------------------------------
# relative position bias
# ---------------------------------------------------------------------------------------------------------------
def bias_case(P, seed, sq, sk, heads, rule, groups=0, shuffled=False):
    g = gen(seed)
    lut = P.clipped_buckets(rule[0]) if len(rule) == 1 else P.logarithmic_buckets(*rule)
    pos = torch.cumsum(torch.randint(0, 3, (max(sq, sk),), generator=g), 0).int()
    if shuffled:
        pos = pos[torch.randperm(len(pos), generator=g)]
    grp = torch.randint(0, groups, (max(sq, sk),), generator=g).int().sort().values if groups else None
    nb = max(lut) + 1 + (1 if groups else 0)
    table = torch.randn(nb, heads, generator=g)
    qp, kp = pos[len(pos) - sq:], pos[:sk]
    qg, kg = (None, None) if grp is None else (grp[len(pos) - sq:], grp[:sk])
    reach = len(lut) // 2
    d = (kp.long()[None] - qp.long()[:, None]).clamp(-reach, reach) + reach
    b = torch.tensor(lut)[d]
    if groups:
        b = torch.where(qg[:, None] == kg[None], b, nb - 1)
    cu = lambda t: None if t is None else t.contiguous().cuda()
    return table, nb, b, (torch.tensor(lut, dtype=torch.int32).cuda(), cu(qp), cu(kp), cu(qg), cu(kg))


BIAS = [  # queries, keys, heads, rule, groups, shuffled
    (1, 1, 1, (0,), 0, False),
    (1, 4097, 32, (32, 128, False), 0, False),
    (3, 5, 2, (4,), 2, False),
    (40, 64, 3, (32,), 3, False),
    (64, 40, 16, (32, 128, True), 0, True),
    (129, 257, 5, (8, 20, True), 4, True),
    (300, 300, 16, (32,), 5, False),
    (77, 1000, 4, (1024, 3000, False), 0, False),
    (520, 1032, 8, (32, 128, True), 2, False),
]


@pytest.mark.parametrize("sq,sk,heads,rule,groups,shuffled", BIAS)
def test_relative_bias(P, ops, sq, sk, heads, rule, groups, shuffled):
    table, nb, b, args = bias_case(P, sq + sk, sq, sk, heads, rule, groups, shuffled)
    want = table[b].permute(2, 0, 1)
    t = table.cuda()
    assert torch.equal(P.relative_position_bias(t, *args).cpu(), want)
    assert torch.equal(P.relative_position_bias(t, *args, dtype=BF).cpu(), want.to(BF))
    got = P.relative_position_bias(t, *args, prepared=True)
    assert tuple(got.shape) == (heads, sq, (sk + 7) // 8 * 8)
    assert torch.equal(got[..., :sk].cpu(), (want * 1.4426950408889634).clamp(-60000, 60000).half())
    assert not got[..., sk:].any()
    if sq == sk:
        assert torch.equal(got, ops.prepare_pair_bias(want.contiguous().cuda()))
    ops.synchronize_and_check()


def test_relative_bias_of_far_and_extreme_positions(P):
    table, lut = torch.randn(5, 2, generator=gen(1)), torch.tensor([0, 1, 2, 3, 4], dtype=torch.int32).cuda()
    q = torch.tensor([-2 ** 31, -7, 0, 2 ** 31 - 1], dtype=torch.int32).cuda()
    k = torch.tensor([2 ** 31 - 1, -2 ** 31, -6, 1, 0, 2 ** 31 - 2], dtype=torch.int32).cuda()
    d = (k.long()[None] - q.long()[:, None]).clamp(-2, 2).cpu() + 2
    assert torch.equal(P.relative_position_bias(table.cuda(), lut, q, k).cpu(), table[d].permute(2, 0, 1))


def test_relative_bias_of_values_that_are_not_finite(P):
    inf = float("inf")
    table = torch.tensor([[inf], [-inf], [1e30], [float("nan")], [-5e4]]).cuda()
    lut, q, k = torch.arange(5, dtype=torch.int32).cuda(), torch.tensor([0], dtype=torch.int32).cuda(), torch.arange(-2, 3, dtype=torch.int32).cuda()
    out = P.relative_position_bias(table, lut, q, k)[0, 0]
    assert out[0] == inf and out[1] == -inf and out[2] == 1e30 and out[3].isnan() and out[4] == -5e4
    assert P.relative_position_bias(table, lut, q, k, prepared=True)[0, 0, :5].tolist() == [60000, -60000, 60000, -60000, -60000]


def test_relative_bias_of_buckets_that_name_no_row(P):
    table, lut = torch.ones(3, 2).cuda(), torch.tensor([0, 3, -1, 2, 1], dtype=torch.int32).cuda()
    q, k = torch.zeros(1, dtype=torch.int32).cuda(), torch.arange(-2, 3, dtype=torch.int32).cuda()
    out = P.relative_position_bias(table, lut, q, k)
    assert out.isnan()[:, 0].tolist() == [[False, True, True, False, False]] * 2
    got = P.relative_position_bias_backward(torch.ones(2, 1, 5).cuda(), 3, lut, q, k)
    assert got.tolist() == [[1, 1], [1, 1], [1, 1]]


@pytest.mark.parametrize("dtype", [F32, BF])
@pytest.mark.parametrize("sq,sk,heads,rule,groups,shuffled", BIAS)
def test_relative_bias_gradient(P, ops, dtype, sq, sk, heads, rule, groups, shuffled):
    _, nb, b, args = bias_case(P, sq + sk, sq, sk, heads, rule, groups, shuffled)
    grad = torch.randint(-8, 9, (heads, sq, sk), generator=gen(sq)).to(dtype)
    hot = torch.nn.functional.one_hot(b.flatten().long(), nb).double()
    want = (grad.flatten(1).double() @ hot).T
    assert float(want.abs().max()) < 2 ** 24
    got = P.relative_position_bias_backward(grad.cuda(), nb, *args)
    assert torch.equal(got.double().cpu(), want)
    real = torch.randn(heads, sq, sk, generator=gen(sq + 1)).to(dtype)
    got = P.relative_position_bias_backward(real.cuda(), nb, *args)
    again = P.relative_position_bias_backward(real.cuda(), nb, *args)
    assert torch.equal(got, again)
    want, mass = ((x.flatten(1).double() @ hot).T for x in (real, real.abs()))
    # a lane adds at most 8 columns of every row, then 8 warps, 32 lanes and 10 rounds of CTAs are added
    assert ((got.double().cpu() - want).abs() <= (8 * sq + 64) * U * mass).all()
    ops.synchronize_and_check()


@pytest.mark.parametrize("dtype", [F32, BF])
def test_relative_bias_gradient_of_strided_input(P, dtype):
    """Heads next to each other in rows, a slice at an odd element, a broadcast gradient, keys not next to each other."""
    sq, sk, heads = 37, 48, 6
    _, nb, b, args = bias_case(P, 5, sq, sk, heads, (8,), 3)
    hot = torch.nn.functional.one_hot(b.flatten().long(), nb).double()
    base = torch.randint(-8, 9, (sq + 1, heads, sk + 9), generator=gen(2)).to(dtype).cuda()
    views = [base[:sq, :, :sk].permute(1, 0, 2), base[1:, :, 1:sk + 1].permute(1, 0, 2), base[:1, :, 8:sk + 8].expand(sq, -1, -1).permute(1, 0, 2),
             base[:sq, :1, :1].expand(sq, heads, sk).permute(1, 0, 2)]
    for v in views:
        got = P.relative_position_bias_backward(v, nb, *args)
        assert torch.equal(got.double().cpu(), (v.cpu().reshape(heads, -1).double() @ hot).T)


def test_relative_bias_gradient_is_that_of_the_bias(P):
    """The bias is linear in its table: differences are exact up to rounding."""
    table, nb, b, args = bias_case(P, 11, 60, 90, 4, (16, 40, True), 3)
    step = torch.randint(-4, 5, (nb, 4), generator=gen(3)).float()
    grad = torch.randint(-4, 5, (4, 60, 90), generator=gen(4)).float()
    zero = torch.zeros_like(table)
    diff = P.relative_position_bias((zero + step).cuda(), *args) - P.relative_position_bias(zero.cuda(), *args)
    got = P.relative_position_bias_backward(grad.cuda(), nb, *args)
    assert float((diff.cpu() * grad).double().sum()) == float((got.cpu() * step).double().sum())


def test_relative_bias_without_queries_or_keys(P):
    lut, none, some = torch.arange(3, dtype=torch.int32).cuda(), torch.zeros(0, dtype=torch.int32).cuda(), torch.zeros(4, dtype=torch.int32).cuda()
    table = torch.ones(3, 2).cuda()
    for q, k in ((none, some), (some, none), (none, none)):
        assert tuple(P.relative_position_bias(table, lut, q, k).shape) == (2, q.numel(), k.numel())
        got = P.relative_position_bias_backward(torch.ones(2, q.numel(), k.numel()).cuda(), 3, lut, q, k)
        assert got.tolist() == [[0, 0]] * 3


def test_relative_bias_refusals_of_the_library(P):
    from distributed_xfold_b200._cabi import XfoldError
    q = torch.zeros(2, dtype=torch.int32).cuda()
    with pytest.raises(XfoldError, match="1024 buckets"):
        P.relative_position_bias(torch.ones(1025, 1).cuda(), torch.zeros(3, dtype=torch.int32).cuda(), q)
    with pytest.raises(XfoldError, match="1024 buckets"):
        P.relative_position_bias(torch.ones(4, 1).cuda(), torch.zeros(2 * 4097 + 1, dtype=torch.int32).cuda(), q)
    with pytest.raises(XfoldError, match="1024 buckets"):
        P.relative_position_bias_backward(torch.ones(1, 2, 2).cuda(), 1025, torch.zeros(3, dtype=torch.int32).cuda(), q)


# ---------------------------------------------------------------------------------------------------------------
# norms and rotation
# ---------------------------------------------------------------------------------------------------------------
def turned(x, rotation, pos, back=False):
    """x [b, s, h, d] in 64 bits; pos [b, s]"""
    if rotation is None:
        return x
    f = rotation.freqs.double().cpu()
    rot = 2 * len(f)
    t = (pos.double()[..., None] * f)[:, :, None]
    c, s = t.cos(), (-t.sin() if back else t.sin())
    y = x.clone()
    a, b = (slice(0, rot, 2), slice(1, rot, 2)) if rotation.interleaved else (slice(0, rot // 2), slice(rot // 2, rot))
    y[..., a] = x[..., a] * c - x[..., b] * s
    y[..., b] = x[..., b] * c + x[..., a] * s
    return y


def pair_length(x, rotation):
    y = x.abs().clone()
    if rotation is not None:
        rot = 2 * rotation.freqs.numel()
        a, b = (slice(0, rot, 2), slice(1, rot, 2)) if rotation.interleaved else (slice(0, rot // 2), slice(rot // 2, rot))
        y[..., a] = y[..., b] = (x[..., a] ** 2 + x[..., b] ** 2).sqrt()
    return y


def plain(x, w, rotation, pos, eps, scale):
    x = x.double().cpu()
    w = torch.ones(x.shape[-1], dtype=F64) if w is None else w.double().cpu()
    return x * (x.square().mean(-1, keepdim=True) + eps).rsqrt() * w * scale


def check_forward(P, q, k, qw, kw, rotation, pos, positions, eps, scale, out):
    for x, w, f, got in ((q, qw, scale, out[0]), (k, kw, 1.0, out[1])):
        y = plain(x, w, rotation, pos, eps, f)
        want, tol = turned(y, rotation, pos), 32 * U * pair_length(y, rotation)
        tol = tol + HALF[x.dtype] * (want.abs() + tol) + 2.0 ** -133   # (the last: half of the smallest number's step)
        err = (got.double().cpu() - want).abs()
        assert got.dtype == x.dtype and (err <= tol).all(), float((err / tol).max())


QK = [  # batch, tokens, q heads, k heads, width, rotated, interleaved, type, first position
    (1, 1, 1, 1, 2, 2, False, F32, 0),
    (1, 1, 1, 1, 2, 0, True, BF, 0),
    (8, 1, 32, 8, 128, 128, False, BF, 100000),
    (2, 5, 4, 4, 24, 24, False, BF, 3),
    (2, 5, 4, 2, 24, 12, True, BF, 3),
    (3, 7, 16, 16, 48, 48, False, BF, 1000),
    (1, 33, 3, 5, 64, 32, True, BF, 0),
    (1, 33, 5, 3, 64, 32, False, F32, 500000),
    (2, 9, 12, 4, 80, 40, False, BF, 0),
    (1, 17, 2, 1, 256, 256, True, F32, 7),
    (1, 17, 2, 1, 256, 128, False, BF, 7),
    (2, 11, 3, 2, 66, 6, False, F32, 0),
    (2, 11, 3, 2, 250, 250, True, BF, 2000000000),
    (1, 700, 7, 7, 32, 32, False, F32, 0),
]


def qk_case(P, b, s, hq, hk, d, rot, inter, dtype, start, seed=0):
    g = gen(seed + s + d)
    q, k = (torch.randn(b, s, h, d, generator=g).mul(2.0).to(dtype).cuda() for h in (hq, hk))
    qw, kw = (1 + 0.2 * torch.randn(d, generator=g) for _ in range(2))
    rotation = P.Rotation.make(rot, interleaved=inter) if rot else None
    pos = (start + torch.randint(0, 50, (b, s), generator=g)).int()
    return q, k, qw.cuda(), kw.cuda(), rotation, pos


@pytest.mark.parametrize("case", QK)
def test_norm_rotate(P, ops, case):
    q, k, qw, kw, rotation, pos = qk_case(P, *case)
    args = dict(eps=1e-6, q_scale=0.25)
    out = P.norm_rotate_qk(q, k, qw, kw, rotation, pos.cuda(), **args)
    check_forward(P, q, k, qw, kw, rotation, pos, pos, 1e-6, 0.25, out)
    # without the weights, with one row of positions, without positions
    b, s = pos.shape
    row = pos[:1].expand(b, -1)
    check_forward(P, q, k, None, kw, rotation, row, None, 1e-2, 1.0, P.norm_rotate_qk(q, k, None, kw, rotation, pos[0].cuda(), eps=1e-2))
    at = torch.arange(s).expand(b, -1)
    check_forward(P, q, k, qw, None, rotation, at, None, 1e-6, 1.0, P.norm_rotate_qk(q, k, qw, None, rotation))
    # in place; one sequence without the batch axis
    q2, k2 = q.clone(), k.clone()
    got = P.norm_rotate_qk_(q2, k2, qw, kw, rotation, pos.cuda(), **args)
    assert got[0] is q2 and torch.equal(q2, out[0]) and torch.equal(k2, out[1])
    one = P.norm_rotate_qk(q[0], k[0], qw, kw, rotation, pos[0].cuda(), **args)
    assert torch.equal(one[0], out[0][0]) and torch.equal(one[1], out[1][0])
    ops.synchronize_and_check()


@pytest.mark.parametrize("dtype", [BF, F32])
def test_norm_rotate_of_views(P, dtype):
    """Heads in a fused projection, padded and not, at odd elements; batch and head axes exchanged; broadcast tokens."""
    b, s, hq, hk, d, pitch = 2, 13, 4, 2, 24, 32
    q, k, qw, kw, rotation, pos = qk_case(P, b, s, hq, hk, d, d, False, dtype, 5)
    ref = P.norm_rotate_qk(q, k, qw, kw, rotation, pos.cuda())
    for off in (0, 1, 2, 4):
        buf = torch.full((b, s, off + (hq + hk) * pitch), 7.0, dtype=dtype, device="cuda")
        vq = buf[..., off:off + hq * pitch].unflatten(-1, (hq, pitch))[..., :d]
        vk = buf[..., off + hq * pitch:].unflatten(-1, (hk, pitch))[..., :d]
        vq.copy_(q), vk.copy_(k)
        before = buf.clone()
        got = P.norm_rotate_qk(vq, vk, qw, kw, rotation, pos.cuda())
        assert torch.equal(buf, before)
        for x, y in zip(got, ref):   # another piece width adds in another order
            assert ((x.double() - y.double()).abs() <= 2 * HALF[dtype] * y.double().abs() + 64 * U * y.double().abs().max()).all()
        P.norm_rotate_qk_(vq, vk, qw, kw, rotation, pos.cuda())
        assert torch.equal(vq, got[0]) and torch.equal(vk, got[1])
        vq.fill_(7.0), vk.fill_(7.0)
        assert (buf == 7).all()   # padding and what lies in front stay
    tq, tk = (x.transpose(1, 2).contiguous().transpose(1, 2) for x in (q, k))
    got = P.norm_rotate_qk(tq, tk, qw, kw, rotation, pos.cuda())
    assert torch.equal(got[0], ref[0]) and torch.equal(got[1], ref[1])
    same = P.norm_rotate_qk(q[:, :1].expand(-1, s, -1, -1), k[:, :1].expand(-1, s, -1, -1), qw, kw, rotation, pos.cuda())
    assert torch.equal(same[0][:, 0], ref[0][:, 0]) and torch.equal(same[1][:, 0], ref[1][:, 0])


def test_norm_rotate_of_rows_of_zeros_and_of_numbers_that_are_not_finite(P):
    q = torch.zeros(1, 4, 2, 16, dtype=F32)
    q[0, 1, 0, 3], q[0, 2, 1, 5] = float("nan"), float("inf")
    k = q.clone()
    r = P.Rotation.make(16)
    a, b = P.norm_rotate_qk(q.cuda(), k.cuda(), None, None, r)
    for x in (a.cpu(), b.cpu()):
        assert not x[0, 0].any() and not x[0, 3].any() and not x[0, 1, 1].any() and not x[0, 2, 0].any()
        assert x[0, 1, 0].isnan().all() and x[0, 2, 1].isnan().any()
    z = P.norm_rotate_qk(torch.zeros(1, 2, 8).cuda(), torch.zeros(1, 2, 8).cuda(), None, None, eps=0.0)
    assert z[0].isnan().all()   # 0 * inf, as the formula has it


@pytest.mark.parametrize("case", QK)
def test_norm_rotate_gradient(P, ops, case):
    q, k, qw, kw, rotation, pos = qk_case(P, *case, seed=100)
    eps, scale = 1e-6, 0.25
    g = gen(case[1])
    dq, dk = (torch.randn(x.shape, generator=g).to(x.dtype).cuda() for x in (q, k))
    got = P.norm_rotate_qk_backward(dq, dk, q, k, qw, kw, rotation, pos.cuda(), eps=eps, q_scale=scale)
    again = P.norm_rotate_qk_backward(dq, dk, q, k, qw, kw, rotation, pos.cuda(), eps=eps, q_scale=scale)
    assert all(torch.equal(x, y) for x, y in zip(got, again))
    for x, d, w, f, dx, dw in ((q, dq, qw, scale, got[0], got[2]), (k, dk, kw, 1.0, got[1], got[3])):
        x64, d64, w64 = x.double().cpu(), d.double().cpu(), w.double().cpu()
        back = turned(d64, rotation, pos, back=True) * f
        size = pair_length(d64, rotation) * f
        r = (x64.square().mean(-1, keepdim=True) + eps).rsqrt()
        want = r * (back * w64 - x64 * r * r * (back * w64 * x64).mean(-1, keepdim=True))
        most = r * (size * w64.abs() + x64.abs() * r * r * (size * (w64 * x64).abs()).mean(-1, keepdim=True))
        tol = 96 * U * most
        tol = tol + HALF[x.dtype] * (want.abs() + tol) + 2.0 ** -133
        err = (dx.double().cpu() - want).abs()
        assert (err <= tol).all(), float((err / tol).max())
        n = x[..., 0].numel()
        want, most = (back * x64 * r).sum((0, 1, 2)), (size * x64.abs() * r).sum((0, 1, 2))
        err = (dw.double().cpu() - want).abs()
        assert (err <= (n + 64) * U * most).all(), float((err / most).max() / U)
    # no weights: the gradients of q and k alone; a gradient that was broadcast, and one whose heads lie apart
    none = P.norm_rotate_qk_backward(dq, dk, q, k, None, None, rotation, pos.cuda(), eps=eps, q_scale=scale)
    ones = torch.ones_like(qw)
    with_ones = P.norm_rotate_qk_backward(dq, dk, q, k, ones, ones, rotation, pos.cuda(), eps=eps, q_scale=scale)
    assert none[2] is None and none[3] is None and torch.equal(none[0], with_ones[0]) and torch.equal(none[1], with_ones[1])
    tq, tk = (x.transpose(1, 2).contiguous().transpose(1, 2) for x in (dq, dk))
    apart = P.norm_rotate_qk_backward(tq, tk, q, k, qw, kw, rotation, pos.cuda(), eps=eps, q_scale=scale)
    assert all(torch.equal(x, y) for x, y in zip(apart, got))
    wide = dq[..., :1].expand_as(dq), dk[:, :1].expand_as(dk)
    a = P.norm_rotate_qk_backward(*wide, q, k, qw, kw, rotation, pos.cuda(), eps=eps, q_scale=scale)
    b = P.norm_rotate_qk_backward(*(x.contiguous() for x in wide), q, k, qw, kw, rotation, pos.cuda(), eps=eps, q_scale=scale)
    assert all(torch.equal(x, y) for x, y in zip(a, b))
    ops.synchronize_and_check()


@pytest.mark.parametrize("inter", [False, True])
def test_norm_rotate_gradient_against_differences(P, inter):
    """Central differences of the definition in 64 bits along a direction, step 1e-4: their error is of the order of the step's
    square; the kernel's gradients are 32-bit numbers (relative 1e-6 of the sum of absolute products)."""
    q, k, qw, kw, rotation, pos = qk_case(P, 2, 6, 3, 2, 32, 16, inter, F32, 40)
    g = gen(9)
    for x, w, f, i in ((q, qw, 0.5, 0), (k, kw, 1.0, 1)):
        d = torch.randn(x.shape, generator=g)
        grads = P.norm_rotate_qk_backward(*((d.cuda(), torch.zeros_like(k)) if i == 0 else (torch.zeros_like(q), d.cuda())), q, k, qw, kw,
                                          rotation, pos.cuda(), q_scale=0.5)
        vx, vw = torch.randn(x.shape, generator=g).double(), torch.randn(w.shape, generator=g).double()
        f64 = lambda t: (turned(plain(x.double().cpu() + t * vx, w.double().cpu() + t * vw, rotation, pos, 1e-6, f), rotation, pos) * d.double()).sum()
        diff = (f64(1e-4) - f64(-1e-4)) / 2e-4
        mine = (grads[i].double().cpu() * vx).sum() + (grads[2 + i].double().cpu() * vw).sum()
        mass = (grads[i].double().cpu() * vx).abs().sum() + (grads[2 + i].double().cpu() * vw).abs().sum()
        assert abs(float(diff - mine)) <= 1e-6 * float(mass)


def test_norm_rotate_without_tokens_or_heads(P):
    w, r = torch.ones(8).cuda(), P.Rotation.make(8)
    for shape_q, shape_k in (((0, 4, 8), (0, 2, 8)), ((2, 0, 4, 8), (2, 0, 4, 8)), ((3, 4, 8), (3, 0, 8)), ((3, 0, 8), (3, 2, 8))):
        q, k = torch.randn(shape_q).cuda(), torch.randn(shape_k).cuda()
        a, b = P.norm_rotate_qk(q, k, w, w, r)
        assert a.shape == q.shape and b.shape == k.shape
        dq, dk, dqw, dkw = P.norm_rotate_qk_backward(torch.ones_like(q), torch.ones_like(k), q, k, w, w, r)
        assert dq.shape == q.shape and (q.numel() > 0 or not dqw.any()) and (k.numel() > 0 or not dkw.any())
    full = torch.randn(3, 2, 8).cuda()
    a = P.norm_rotate_qk(full, full, w, w, r)
    b = P.norm_rotate_qk(full[:, :0], full, w, w, r)
    assert torch.equal(a[1], b[1])


def test_norm_rotate_refusals_of_the_library(P):
    from distributed_xfold_b200._cabi import XfoldError
    for d in (7, 258, 1):
        x = torch.zeros(2, 3, d).cuda()
        with pytest.raises(XfoldError, match="even width"):
            P.norm_rotate_qk(x, x, None, None)
        with pytest.raises(XfoldError, match="even width"):
            P.norm_rotate_qk_backward(x, x, x, x, None, None)
    x = torch.zeros(2, 3, 8).cuda()
    for eps in (-1.0, float("nan")):
        with pytest.raises(XfoldError, match="eps"):
            P.norm_rotate_qk(x, x, None, None, eps=eps)


# ---------------------------------------------------------------------------------------------------------------
# streams, graphs
# ---------------------------------------------------------------------------------------------------------------
def calls(P):
    table, nb, b, args = bias_case(P, 1, 90, 130, 4, (16, 40, True), 3)
    table = table.cuda()
    _, _, qw, kw, rotation, pos = qk_case(P, 2, 40, 6, 2, 64, 64, False, BF, 9)
    pos = pos.cuda()

    def make(seed):
        g = gen(seed)
        return (torch.randn(4, 90, 130, generator=g).cuda(), *(torch.randn(2, 40, h, 64, generator=g).to(BF).cuda() for h in (6, 2, 6, 2)))

    def call(grad, q, k, dq, dk):
        bias = P.relative_position_bias(table + grad[0, 0, 0], *args)
        return (bias, P.relative_position_bias_backward(grad, nb, *args), *P.norm_rotate_qk(q, k, qw, kw, rotation, pos),
                *P.norm_rotate_qk_backward(dq, dk, q, k, qw, kw, rotation, pos))

    return make, call


def test_position_calls_on_several_streams(P, ops):
    make, call = calls(P)
    inputs = [make(s) for s in range(3)]
    want = [[t.clone() for t in call(*x)] for x in inputs]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in range(3)], [[] for _ in range(3)]
    for _ in range(4):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                got[i].append(call(*inputs[i]))
    torch.cuda.synchronize()
    for i in range(3):
        for out in got[i]:
            assert all(torch.equal(a, b) for a, b in zip(out, want[i]))


def test_position_calls_captured(P, ops):
    make, call = calls(P)
    static, want = make(0), [[t.clone() for t in call(*make(s))] for s in range(2)]
    graphs = [torch.cuda.CUDAGraph() for _ in range(2)]
    torch.cuda.synchronize()
    outs = []
    for graph in graphs:   # two graphs: scratch of their own
        with torch.cuda.graph(graph, stream=torch.cuda.Stream()):
            outs.append(call(*static))
    ops._Workspace.release()
    filler = torch.full((1 << 26,), 0x7F, dtype=torch.uint8, device="cuda")
    for seed in (1, 0):
        for dst, src in zip(static, make(seed)):
            dst.copy_(src)
        for graph, out in zip(graphs, outs):
            graph.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(out, want[seed]))
    del filler


def test_norm_rotate_results_that_are_refused(P):
    from distributed_xfold_b200._cabi import XfoldError
    q, k = torch.randn(3, 4, 8).cuda(), torch.randn(3, 4, 8).cuda()
    for out in ((k, q), (k, torch.empty_like(k)), (q, q), (q[:1].expand(3, -1, -1), k), (q[..., :4], k), (q, k.to(BF))):
        with pytest.raises(XfoldError, match="results of queries and keys"):
            P.norm_rotate_qk(q, k, None, None, out=out)


RANGES = [  # batch, tokens, q heads, k heads, width, rotated, interleaved, type: warps whose passes begin and end inside tokens
    (3, 700, 12, 4, 128, 128, False, BF),
    (2, 1300, 16, 16, 64, 32, True, BF),
    (1, 5000, 5, 0, 48, 48, False, F32),
    (5, 401, 0, 9, 80, 40, True, BF),
    (2, 900, 33, 1, 256, 256, True, BF),
]


@pytest.mark.parametrize("case", RANGES)
def test_norm_rotate_of_many_tokens(P, ops, case):
    """Positions on both sides of zero; every token against the definition, forward and backward."""
    b, s, hq, hk, d, rot, inter, dtype = case
    q, k, qw, kw, rotation, pos = qk_case(P, b, s, hq, hk, d, rot, inter, dtype, -20, seed=3)
    pos = pos * torch.tensor([1, -1000003])[torch.arange(s) % 2].int()
    check_forward(P, q, k, qw, kw, rotation, pos, pos, 1e-6, 0.25, P.norm_rotate_qk(q, k, qw, kw, rotation, pos.cuda(), q_scale=0.25)) \
        if hq and hk else None
    g = gen(s)
    dq, dk = (torch.randn(x.shape, generator=g).to(dtype).cuda() for x in (q, k))
    got = P.norm_rotate_qk_backward(dq, dk, q, k, qw, kw, rotation, pos.cuda(), q_scale=0.25)
    for x, dy, w, f, dx, dw in ((q, dq, qw, 0.25, got[0], got[2]), (k, dk, kw, 1.0, got[1], got[3])):
        if not x.numel():
            assert not dw.any()
            continue
        x64, w64, d64 = x.double().cpu(), w.double().cpu(), dy.double().cpu()
        back, size = turned(d64, rotation, pos, back=True) * f, pair_length(d64, rotation) * f
        r = (x64.square().mean(-1, keepdim=True) + 1e-6).rsqrt()
        want = r * (back * w64 - x64 * r * r * (back * w64 * x64).mean(-1, keepdim=True))
        tol = 96 * U * r * (size * w64.abs() + x64.abs() * r * r * (size * (w64 * x64).abs()).mean(-1, keepdim=True))
        tol = tol + HALF[dtype] * (want.abs() + tol) + 2.0 ** -133
        assert ((dx.double().cpu() - want).abs() <= tol).all()
        want, most = (back * x64 * r).sum((0, 1, 2)), (size * x64.abs() * r).sum((0, 1, 2))
        # a lane's chain, the lanes of a warp, four warps, the CTAs in 32 chains: far fewer additions than heads and tokens
        assert ((dw.double().cpu() - want).abs() <= (x[..., 0].numel() / 16 + 512) * U * most).all()
    ops.synchronize_and_check()


@pytest.mark.parametrize("dtype", [F32, BF])
@pytest.mark.parametrize("sq,sk,heads,groups,reach", [(1, 700, 3, 2, 5), (9, 8, 2, 0, 0), (1000, 264, 16, 3, 0), (257, 1000, 40, 7, 64), (2050, 96, 2, 0, 700)])
def test_relative_bias_gradient_of_eights(P, ops, dtype, sq, sk, heads, groups, reach):
    """Rows in eights that end anywhere, groups and positions that change inside an eight; whole numbers: equal."""
    g = gen(sq + reach)
    qp, kp = (torch.randint(-400, 400, (n,), generator=g).int().sort().values for n in (sq, sk))
    qp[::5] = qp[torch.randint(0, sq, (len(qp[::5]),), generator=g)]
    qg, kg = (torch.randint(0, groups, (n,), generator=g).int().sort().values if groups else None for n in (sq, sk))
    nb = 2 * reach + 1 + bool(groups)
    b = (kp.long()[None] - qp.long()[:, None]).clamp(-reach, reach) + reach
    if groups:
        b = torch.where(qg[:, None] == kg[None], b, nb - 1)
    if nb > 1024:
        b = b.clamp(max=1023)
    grad = torch.randint(-4, 5, (heads, sq, sk), generator=g).to(dtype)
    lut = torch.arange(2 * reach + 1, dtype=torch.int32).clamp(max=1023)
    cu = lambda t: None if t is None else t.cuda()
    got = P.relative_position_bias_backward(grad.cuda(), min(nb, 1024), lut.cuda(), cu(qp), cu(kp), cu(qg), cu(kg))
    want = torch.zeros(heads, min(nb, 1024), dtype=F64).index_add_(1, b.flatten(), grad.flatten(1).double()).T
    assert torch.equal(got.double().cpu(), want)
    ops.synchronize_and_check()


def test_norm_rotate_of_odd_frequencies(P):
    """Whole and half turns for each position, many turns, and frequencies that are not finite: those pairs are not numbers."""
    f = torch.tensor([math.pi, 2 * math.pi, 3 * math.pi, 1e5, -0.3, 0.0, float("nan"), float("inf")], dtype=F64)
    q = torch.randn(1, 9, 2, 16, generator=gen(4)).cuda()
    pos = torch.tensor([[0, 1, 2, 3, -1, 7, 1000001, -2 ** 31, 2 ** 31 - 1]]).int()
    finite = P.Rotation(f[:6])
    keep = torch.cat([q[..., :6], q[..., 8:14]], -1).contiguous()
    a, b = P.norm_rotate_qk(keep, keep, None, None, P.Rotation(f[:6].cuda()), pos.cuda())
    y = plain(keep, None, None, pos, 1e-6, 1.0)
    # the definition's own angle is a product in 64 bits: up to 2^31 * 1e5 radians, off by 2^-53 of it, beside the kernel's
    tol = 32 * U * pair_length(y, finite) + (pos.double().abs()[..., None] * f[:6].abs() * 2.0 ** -51).repeat(1, 1, 2)[:, :, None] * pair_length(y, finite)
    want = turned(y, finite, pos)
    for got in (a, b):
        assert ((got.double().cpu() - want).abs() <= tol + U * want.abs()).all()
    a, _ = P.norm_rotate_qk(q, q, None, None, P.Rotation(f.cuda()), pos.cuda())
    assert a[..., [6, 7, 14, 15]].isnan().all() and a[..., [0, 1, 2, 3, 4, 5, 8, 9, 10, 11, 12, 13]].isfinite().all()


@pytest.mark.parametrize("dtype", [BF, F32])
def test_norm_rotate_results_that_meet_the_inputs_are_refused(P, ops, dtype):
    """A transposed view of the input, views an element, a head or a token on, the other's place: refused before any launch.  Side by
    side in one buffer, and each over its own input: as with new results."""
    from distributed_xfold_b200._cabi import XfoldError
    n, d = 6, 8
    q, k = torch.randn(n, n, d, generator=gen(1)).to(dtype).cuda(), torch.randn(n, 3, d, generator=gen(2)).to(dtype).cuda()
    new_k = torch.empty_like(k)
    buf = torch.randn((n + 1) * n * d + 1, generator=gen(3)).to(dtype).cuda()
    at = lambda off: buf[off:off + n * n * d].view(n, n, d)
    keep = q.clone(), buf.clone()
    for q_in, out in ((q, q.transpose(0, 1)), (at(0), at(1)), (at(0), at(d)), (at(0), at(n * d)), (at(n * d), at(0)),
                      (q, q.as_strided((n, n, d), (d, d, 1)))):
        with pytest.raises(XfoldError, match="results of queries and keys"):
            P.norm_rotate_qk(q_in, k, None, None, out=(out, new_k))
    wide = torch.randn(n, 4, d, generator=gen(4)).to(dtype).cuda()
    for args in ((wide[:, :3], k, (wide[:, 1:], new_k)), (k, wide[:, :3], (wide[:, 1:], new_k)), (k, q[:, :3], (wide[:, :3], wide[:, 1:])),
                 (wide[:, :3], wide[:, 1:], (wide[:, :3], wide[:, 1:]))):
        with pytest.raises(XfoldError, match="results of queries and keys"):
            P.norm_rotate_qk(*args[:2], None, None, out=args[2])
    assert torch.equal(q, keep[0]) and torch.equal(buf, keep[1])
    fused = torch.randn(n, 12, d, generator=gen(5)).to(dtype).cuda()
    ref = P.norm_rotate_qk(fused[:, :4], fused[:, 4:7], None, None)
    P.norm_rotate_qk(fused[:, :4], fused[:, 4:7], None, None, out=(fused[:, 8:], fused[:, 4:7]))
    assert torch.equal(fused[:, 8:], ref[0]) and torch.equal(fused[:, 4:7], ref[1])
    P.norm_rotate_qk_(fused[:, :4], new_k, None, None)
    assert torch.equal(fused[:, :4], ref[0])
    ops.synchronize_and_check()


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("d,pitch,first", [(24, 24, 0), (24, 26, 0), (24, 24, 1), (48, 48, 4), (6, 6, 0), (64, 64, 0)])
def test_norm_rotate_in_place_time_after_time(P, ops, d, pitch, first, dtype):
    """Pieces of all widths in one buffer, each call behind the other, also from a graph: what calls with results of their own give."""
    g = gen(d + pitch)
    b, s, hq, hk, rounds = 3, 400, 7, 5, 6
    start = torch.randn(b, s, first + (hq + hk) * pitch, generator=g).to(dtype).cuda()
    w = [(1 + 0.2 * torch.randn(d, generator=g)).cuda() for _ in range(2)]
    r = P.Rotation.make(d)

    def views(buf):
        return [buf[..., first + i * hq * pitch:first + (hq if i == 0 else hq + hk) * pitch].unflatten(-1, (-1, pitch))[..., :d] for i in range(2)]
    apart = torch.empty_like(start), torch.empty_like(start)
    for i in range(rounds):
        src, dst = (start if i == 0 else apart[(i + 1) % 2]), apart[i % 2]
        dst.copy_(src)
        P.norm_rotate_qk(*views(src), *w, r, out=tuple(views(dst)))
    want = apart[(rounds - 1) % 2]
    got = start.clone()
    for _ in range(rounds):
        P.norm_rotate_qk_(*views(got), *w, r)
    assert torch.equal(got, want)
    static, graph = start.clone(), torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=torch.cuda.Stream()):
        for _ in range(rounds):
            P.norm_rotate_qk_(*views(static), *w, r)
    for _ in range(5):
        static.copy_(start)
        graph.replay()
        assert torch.equal(static, want)
    ops.synchronize_and_check()


def test_relative_bias_of_too_many_queries_or_keys(P):
    """Lengths that rows counted in 32 bits would run past."""
    from distributed_xfold_b200._cabi import XfoldError
    table, lut, one = torch.ones(3, 1).cuda(), torch.arange(3, dtype=torch.int32).cuda(), torch.zeros(1, dtype=torch.int32).cuda()
    many = torch.empty(2 ** 31 - 1000, dtype=torch.int32, device="cuda")
    for q, k in ((many, one), (one, many)):
        with pytest.raises(XfoldError, match="too many queries or keys"):
            P.relative_position_bias(table, lut, q, k, dtype=BF)
        with pytest.raises(XfoldError, match="too many queries or keys"):
            P.relative_position_bias_backward(torch.empty(1, 1, 1, device="cuda").expand(1, q.numel(), k.numel()) if k is one
                                              else torch.empty(1, 1, k.numel(), dtype=BF, device="cuda"), 3, lut, q, k)
    del many
    torch.cuda.empty_cache()


@pytest.mark.parametrize("form", ["f32", "bf16", "prepared"])
@pytest.mark.parametrize("nb,heads", [(254, 32), (510, 16), (510, 32), (908, 9), (1022, 8), (1022, 16), (1024, 5)])
@pytest.mark.parametrize("sk", [264, 257])
def test_relative_bias_of_the_largest_reach(P, ops, nb, heads, form, sk):
    g = gen(nb + heads)
    sq, reach = 700, 4096
    lut = torch.randint(0, nb, (2 * reach + 1,), generator=g).int()
    qp, kp = (torch.randint(-4500, 4500, (n,), generator=g).int() for n in (sq, sk))
    table = torch.randn(nb, heads, generator=g)
    want = table[lut[(kp.long()[None] - qp.long()[:, None]).clamp(-reach, reach) + reach].long()].permute(2, 0, 1)
    got = P.relative_position_bias(table.cuda(), lut.cuda(), qp.cuda(), kp.cuda(), dtype=BF if form == "bf16" else F32, prepared=form == "prepared")
    if form == "prepared":
        want = (want * 1.4426950408889634).clamp(-60000, 60000).half()
    assert torch.equal(got[..., :sk].cpu(), want.to(got.dtype))
    ops.synchronize_and_check()


def same(got, want):
    """The same not-a-numbers and infinities."""
    got = got.double().cpu()
    assert torch.equal(got.isnan(), want.isnan()), (got.isnan() ^ want.isnan()).nonzero()[:5]
    assert torch.equal(got.isposinf(), want.isposinf()) and torch.equal(got.isneginf(), want.isneginf())


WHERE = [(24, 0, False), (24, 12, True), (64, 32, False), (64, 16, True), (66, 6, False), (80, 40, False), (128, 64, True), (256, 128, False), (26, 2, True)]


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("d,rot,inter", WHERE)
@pytest.mark.parametrize("at", [0, -1, -3])
def test_norm_rotate_keeps_what_is_not_finite_to_its_pair(P, ops, d, rot, inter, dtype, at):
    g = gen(d + rot)
    q, k = (torch.randn(2, 5, h, d, generator=g).to(dtype) for h in (3, 2))
    dq, dk = (torch.randn(x.shape, generator=g).to(dtype) for x in (q, k))
    qw, kw = (1 + 0.2 * torch.randn(d, generator=g) for _ in range(2))
    qw[at], kw[at] = float("inf"), float("nan")
    rotation = P.Rotation.make(rot, interleaved=inter) if rot else None
    pos = torch.randint(1, 50, (2, 5), generator=g).int()
    cu = lambda *t: [x.cuda() for x in t]
    out = P.norm_rotate_qk(*cu(q, k, qw, kw), rotation, pos.cuda())
    for x, w, o in ((q, qw, out[0]), (k, kw, out[1])):
        same(o, turned(plain(x, w, None, None, 1e-6, 1.0), rotation, pos))
    ones = torch.ones(d)
    x = q.clone()
    x[0, 1, 0, at], x[1, 2, 2, at] = float("inf"), float("nan")
    same(P.norm_rotate_qk(*cu(x, k, ones, ones), rotation, pos.cuda())[0], turned(plain(x, None, None, None, 1e-6, 1.0), rotation, pos))
    y = dq.clone()
    y[0, 1, 0, at] = float("inf")
    got = P.norm_rotate_qk_backward(*cu(y, dk, q, k, ones, ones), rotation, pos.cuda())
    back, x64 = turned(y.double(), rotation, pos, back=True), q.double()
    r = (x64.square().mean(-1, keepdim=True) + 1e-6).rsqrt()
    same(got[2], (back * x64 * r).sum((0, 1, 2)))
    same(got[0], r * (back - x64 * r * r * (back * x64).mean(-1, keepdim=True)))


def test_calls_of_two_contexts_in_two_threads(P, ops):
    """Contexts have locks of their own: what the library keeps for all of them is found by both at once."""
    import ctypes
    import threading
    from distributed_xfold_b200._cabi import QK_NORM, load
    lib, handles = load(), [ctypes.c_void_p() for _ in range(2)]
    for h in handles:
        assert lib.xfold_ctx_create(0, ctypes.byref(h)) == 0
    shapes = [(d, rot, dt) for d in (6, 20, 40, 128) for rot in (d, d // 4 * 2) for dt in (BF, F32)]
    work = []
    for d, rot, dt in shapes:
        q, k = torch.randn(2, 30, 5, d, generator=gen(d)).to(dt).cuda(), torch.randn(2, 30, 3, d, generator=gen(d + 1)).to(dt).cuda()
        r = P.Rotation.make(rot)
        work.append((q, k, r, P.norm_rotate_qk(q, k, None, None, r), [[torch.empty_like(t) for t in (q, k)] for _ in handles]))
    torch.cuda.synchronize()
    gate, wrong = threading.Barrier(2, timeout=60), []

    def go(i):
        stream = torch.cuda.Stream()
        for q, k, r, _, outs in work:
            heads = lambda t: (t.data_ptr(), *t.stride()[:3])
            desc = QK_NORM.pack(2, 30, 5, 3, q.shape[-1], 2 * r.freqs.numel(), 0, q.dtype is F32, 0, 0, r.freqs.data_ptr(), 0, 0, 1e-6, 1.0,
                                *heads(q), *heads(k), *heads(outs[i][0]), *heads(outs[i][1]), *[0] * 8)
            gate.wait()
            if lib.xfold_qk_norm_rotate_fwd(handles[i], desc, stream.cuda_stream):
                wrong.append(i)
        stream.synchronize()
    threads = [threading.Thread(target=go, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong
    for _, _, _, want, outs in work:
        for out in outs:
            assert torch.equal(out[0], want[0]) and torch.equal(out[1], want[1])
    for h in handles:
        lib.xfold_ctx_destroy(h)


@pytest.mark.parametrize("case", [c for c in RANGES if not (c[2] and c[3])])
def test_norm_rotate_of_many_tokens_on_one_side(P, ops, case):
    """Queries without keys, and keys without queries, over many tokens."""
    b, s, hq, hk, d, rot, inter, dtype = case
    q, k, qw, kw, rotation, pos = qk_case(P, b, s, hq, hk, d, rot, inter, dtype, -20, seed=3)
    out = P.norm_rotate_qk(q, k, qw, kw, rotation, pos.cuda(), q_scale=0.25)
    for x, w, f, got in ((q, qw, 0.25, out[0]), (k, kw, 1.0, out[1])):
        assert got.shape == x.shape
        if x.numel():
            check_forward(P, x, x, w, w, rotation, pos, pos, 1e-6, f, (got, P.norm_rotate_qk(x, x, w, w, rotation, pos.cuda(), q_scale=f)[1]))
    ops.synchronize_and_check()


@pytest.mark.parametrize("dtype", [F32, BF])
@pytest.mark.parametrize("reach", [0, 2, 500])
def test_relative_bias_gradient_of_far_and_extreme_positions(P, ops, dtype, reach):
    """Positions at both ends of 32 bits, next to ordinary ones, in eights and in blocks of columns."""
    g = gen(reach)
    ends = torch.tensor([-2 ** 31, -2 ** 31 + 1, -2 ** 31 + 400, -7, 0, 5, 2 ** 31 - 400, 2 ** 31 - 2, 2 ** 31 - 1])
    qp, kp = (ends[torch.randint(0, len(ends), (n,), generator=g)].sort().values.int() for n in (50, 300))
    nb = 2 * reach + 1
    b = (kp.long()[None] - qp.long()[:, None]).clamp(-reach, reach) + reach
    grad = torch.randint(-4, 5, (2, 50, 300), generator=g).to(dtype)
    got = P.relative_position_bias_backward(grad.cuda(), nb, torch.arange(nb, dtype=torch.int32).cuda(), qp.cuda(), kp.cuda())
    want = torch.zeros(2, nb, dtype=F64).index_add_(1, b.flatten(), grad.flatten(1).double()).T
    assert torch.equal(got.double().cpu(), want)
    ops.synchronize_and_check()
