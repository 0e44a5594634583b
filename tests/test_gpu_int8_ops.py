"""GPU: linear layers in 8-bit integers against whole numbers and 64 bits.

The quantised rows are whole numbers by definition: equal to x / scale in 64 bits, rounded to even (two 24-bit numbers' quotient
is never nearer than 2^-32 to a border that it does not lie on).  The sums are exact; a result has the roundings of the sum to
float32, of two products and of the bias' addition (u = 2^-24 each, below 4 u of |sum s w| + |bias|), then half a step of its type."""
import pytest
import torch

pytestmark = pytest.mark.gpu
BF, F32, I8 = torch.bfloat16, torch.float32, torch.int8
U = 2.0 ** -24
HALF = {BF: 2.0 ** -8, F32: U}


@pytest.fixture(scope="module")
def Q(ops):
    from distributed_xfold_b200 import int8_ops
    return int8_ops


def gen(seed):
    return torch.Generator().manual_seed(seed)


def plain_rows(x):
    x = x.cpu()
    scale = x.float().abs().amax(-1) / 127
    return torch.where(scale[..., None] > 0, x.double() / scale.double()[..., None].clamp_min(1e-300), 0.0).round(), scale


def weights(n, k, seed):
    w = torch.zeros(n, (k + 15) // 16 * 16, dtype=I8)
    w[:, :k] = torch.randint(-127, 128, (n, k), generator=gen(seed)).to(I8)
    w = w.cuda()
    if k % 16:
        w[:, k:] = 77   # what lies between the rows is not read as weights
    return w[:, :k], (torch.rand(n, generator=gen(seed + 1)) + 0.5).div(k).cuda()


def check_linear(out, q, s, w, ws, bias, dtype):
    acc = q.reshape(-1, q.shape[-1]) @ w.cpu().double().T
    y = acc * s.reshape(-1, 1).double() * ws.cpu().double()
    b = torch.zeros(w.shape[0], dtype=torch.float64) if bias is None else bias.cpu().double()
    want, tol = y + b, 4 * U * (y.abs() + b.abs())
    tol = tol + HALF[dtype] * (want.abs() + tol)
    got = out.double().cpu().reshape(want.shape)
    assert out.dtype == dtype and ((got - want).abs() <= tol).all(), float(((got - want).abs() / tol.clamp_min(1e-300)).max())


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("m,k", [(1, 1), (1, 768), (3, 7), (5, 33), (130, 384), (17, 1000), (9, 1024), (4, 1032), (2, 5001), (3, 16384), (2, 40000), (1, 131072)])
def test_quantize_rows(Q, ops, m, k, dtype):
    x = (torch.randn(m, k, generator=gen(m + k)) * torch.logspace(-3, 3, m)[:, None]).to(dtype)
    q, s = Q.quantize_rows(x.cuda())
    want, scale = plain_rows(x)
    assert q.dtype == I8 and q.stride(0) % 16 == 0 and torch.equal(s.cpu(), scale) and torch.equal(q.cpu().double(), want)
    whole = torch.as_strided(q, (m, q.stride(0)), (q.stride(0), 1))
    assert not whole[:, k:].any()
    ops.synchronize_and_check()


def test_quantize_rows_at_borders(Q):
    """Ties, and quotients a step of the last bit away from them."""
    half = torch.arange(-126, 126).float() + 0.5
    near = torch.nextafter(half, torch.full_like(half, 1e9)), torch.nextafter(half, torch.full_like(half, -1e9))
    base = torch.cat([torch.tensor([127.0]), half, *near])
    for f in (1.0, 2.0 ** -20, 3.0, 0.1, 1e30, 1e-30):
        x = base * f
        q, s = Q.quantize_rows(x[None].cuda())
        want, scale = plain_rows(x[None])
        assert torch.equal(s.cpu(), scale) and torch.equal(q.cpu().double(), want)
    assert torch.equal(Q.quantize_rows(base[None].cuda())[0].cpu().double()[0, 1:253], torch.round(half.double()))


def test_quantize_rows_that_are_empty_or_not_finite(Q):
    x = torch.zeros(6, 40)
    x[1, 3], x[2, 5], x[3, 7], x[4, 0], x[5, 39] = float("nan"), float("inf"), -float("inf"), 1e-39, 3e38
    for t in (x, x[:, :33].contiguous()):
        q, s = Q.quantize_rows(t.cuda())
        assert s[0] == 0 and s[4] == 0 and not q[:5].any()
        assert s[1:4].isnan().tolist() == [True, True, True]
    q, s = Q.quantize_rows(x.cuda())
    assert q[5, 39] == 127 and s[5] == torch.tensor(3e38) / 127
    w, ws = weights(24, 40, 3)
    out = Q.linear_int8(x.cuda(), w, ws, dtype=F32)
    large = (127.0 * w[:, 39].double() * s[5].double() * ws.double()).float()   # some beyond the largest float32, others not
    assert out[1:4].isnan().all() and not out[0].any() and torch.equal(out[5].isfinite(), large.isfinite())


LINEAR = [  # rows, inner, channels
    (1, 1, 1), (1, 768, 4096), (2, 100, 130), (7, 16, 8), (8, 1000, 1030), (9, 512, 640), (16, 4096, 96), (17, 48, 4097), (31, 2050, 33), (64, 768, 1536),
    (77, 384, 1536), (127, 130, 1000), (128, 128, 256), (129, 4096, 257), (300, 1536, 768), (1000, 200, 2000), (2500, 768, 1152), (700, 5000, 350)]


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("m,k,n", LINEAR)
def test_linear_int8(Q, ops, m, k, n, dtype):
    x = torch.randn(m, k, generator=gen(m + n)).to(dtype)
    w, ws = weights(n, k, k)
    bias = torch.randn(n, generator=gen(7)).cuda()
    q, s = plain_rows(x)
    out = Q.linear_int8(x.cuda(), w, ws, bias)
    check_linear(out, q, s, w, ws, bias, dtype)
    other = F32 if dtype == BF else BF
    check_linear(Q.linear_int8(x.cuda(), w, ws, dtype=other), q, s, w, ws, None, other)
    xq, xs = Q.quantize_rows(x.cuda())
    assert torch.equal(Q.linear_int8_quantized(xq, xs, w, ws, bias, dtype), out)
    assert torch.equal(Q.linear_int8(x.cuda(), w, ws, bias), out)
    ops.synchronize_and_check()


@pytest.mark.parametrize("m", [1, 5, 40, 200])
def test_linear_int8_with_the_largest_sums(Q, m):
    """The longest row of largest numbers: sums of 127 * 127 * 131072, which only whole numbers hold exactly."""
    k, n = 131072, 40
    x = torch.full((m, k), 1.0)
    x[:, ::3] = -1.0
    w = torch.full((n, k), 127, dtype=I8)
    w[1::2] = torch.where(torch.arange(k) % 3 == 0, -127, 127).to(I8)
    ws = torch.ones(n)
    out = Q.linear_int8(x.cuda(), w.cuda(), ws.cuda(), dtype=F32)
    q, s = plain_rows(x)
    check_linear(out, q, s, w, ws, None, F32)


def test_linear_int8_of_views(Q):
    """Rows apart, a leading axis, weights with longer rows, activations at odd elements."""
    m, k, n = 30, 96, 72
    base = torch.randn(2, m, k + 9, generator=gen(1)).to(BF).cuda()
    wide = torch.randint(-127, 128, (n, 160), generator=gen(2)).to(I8).cuda()
    w, ws = wide[:, 32:32 + k], torch.rand(n, generator=gen(3)).cuda()
    for x in (base[0, :, :k], base[1, :, 1:k + 1], base[..., :k], base[:, ::2, 8:k + 8], base[:1, :1, :k].expand(2, 5, k), base[0, :, :k].t()[:, :24].t()):
        out = Q.linear_int8(x, w, ws)
        assert out.shape == (*x.shape[:-1], n)
        q, s = plain_rows(x)
        check_linear(out, q, s, w, ws, None, BF)
    vec = base[0, 3, :k]
    assert torch.equal(Q.linear_int8(vec, w, ws), Q.linear_int8(vec[None], w, ws)[0])


def test_linear_int8_without_rows_or_channels(Q):
    w, ws = weights(5, 32, 1)
    assert tuple(Q.linear_int8(torch.zeros(0, 32).cuda(), w, ws).shape) == (0, 5)
    assert tuple(Q.linear_int8(torch.zeros(2, 0, 32).cuda(), w, ws).shape) == (2, 0, 5)
    assert tuple(Q.linear_int8(torch.zeros(3, 32).cuda(), w[:0], ws[:0]).shape) == (3, 0)
    q, s = Q.quantize_rows(torch.zeros(0, 32).cuda())
    assert tuple(q.shape) == (0, 32) and tuple(s.shape) == (0,)
    assert tuple(Q.linear_int8_quantized(q, s, w, ws).shape) == (0, 5)


def test_linear_int8_refusals_of_the_library(Q):
    from distributed_xfold_b200._cabi import XfoldError
    with pytest.raises(XfoldError, match="K up to 131072"):
        Q.quantize_rows(torch.zeros(1, 131073).cuda())
    w = torch.zeros(2, 131088, dtype=I8).cuda()
    with pytest.raises(XfoldError, match="K up to 131072"):
        Q.linear_int8(torch.zeros(1, 131088).cuda(), w, torch.ones(2).cuda())


def calls(Q):
    w, ws = weights(520, 200, 4)
    w2, ws2 = weights(200, 520, 5)

    def make(seed):
        return (torch.randn(150, 200, generator=gen(seed)).to(BF).cuda(), torch.randn(2, 200, generator=gen(seed + 9)).to(BF).cuda())

    def call(x, y):
        outs = [Q.linear_int8(t, w, ws) for t in (x, y)]
        return (*outs, *(Q.linear_int8(t, w2, ws2, dtype=F32) for t in outs))

    return make, call


def test_int8_calls_on_several_streams(Q):
    make, call = calls(Q)
    inputs = [make(s) for s in range(3)]
    want = [[t.clone() for t in call(*x)] for x in inputs]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in range(3)], [[] for _ in range(3)]
    for _ in range(6):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                got[i].append(call(*inputs[i]))
    torch.cuda.synchronize()
    for i in range(3):
        for out in got[i]:
            assert all(torch.equal(a, b) for a, b in zip(out, want[i]))


def test_int8_calls_captured(Q, ops):
    make, call = calls(Q)
    static, want = make(0), [[t.clone() for t in call(*make(s))] for s in range(2)]
    graphs, outs = [torch.cuda.CUDAGraph() for _ in range(2)], []
    torch.cuda.synchronize()
    for graph in graphs:
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


def test_projections_norms_and_bias_of_an_attention_layer(Q, ops):
    """The operators in a row, as an attention layer has them: 8-bit projection to queries, keys, values and gate, norms and
    rotation where q and k lie in it, and the prepared bias in the attention core against the same core with the bias as numbers."""
    from distributed_xfold_b200 import position_ops as P
    n, c, heads, d = 70, 384, 16, 24
    g = gen(6)
    x = torch.randn(1, n, c, generator=g).to(BF).cuda()
    wq, ws = Q.quantize_rows((torch.randn(4 * c, c, generator=g) * c ** -0.5).cuda())
    proj = Q.linear_int8(x, wq, ws)
    q, s = plain_rows(x)
    check_linear(proj, q, s, wq, ws, None, BF)
    views = [proj[..., i * c:(i + 1) * c].unflatten(-1, (heads, d)) for i in range(2)]
    w = [(1 + 0.1 * torch.randn(d, generator=g)).cuda() for _ in range(2)]
    rotation, keep = P.Rotation.make(d), proj.clone()
    want = P.norm_rotate_qk(*(v.contiguous() for v in views), *w, rotation, q_scale=d ** -0.5)
    P.norm_rotate_qk_(*views, *w, rotation, q_scale=d ** -0.5)
    assert torch.equal(views[0], want[0]) and torch.equal(views[1], want[1]) and torch.equal(proj[..., 2 * c:], keep[..., 2 * c:])
    lut = torch.tensor(P.clipped_buckets(32), dtype=torch.int32).cuda()
    chain = (torch.arange(n) // 40).int().cuda()
    pos = torch.arange(n, dtype=torch.int32).cuda()
    table = torch.randn(66, heads, generator=g).cuda()
    packed = ops.PackedSelfAttention(_attention_state(g, c), "", "cuda", heads)
    out = ops.attention_pair_bias_core(x, packed, P.relative_position_bias(table, lut, pos, None, chain, prepared=True), None)
    ref = ops.attention_pair_bias_core(x, packed, P.relative_position_bias(table, lut, pos, None, chain), None)
    assert torch.equal(out, ref) and out.isfinite().all()
    ops.synchronize_and_check()


def _attention_state(g, c):
    st = {n + ".weight": torch.randn(c, c, generator=g) * c ** -0.5 for n in ("q_projection", "k_projection", "v_projection", "gating_query")}
    st["adaptive_zero_init.transition2.weight"] = torch.randn(c, c, generator=g) * c ** -0.5
    return st


@pytest.mark.parametrize("dtype", [BF, F32])
def test_quantize_rows_that_start_anywhere(Q, dtype):
    """Rows at any element of an array that ends with them, widths on both sides of eight and sixteen; whole and apart."""
    g = gen(31)
    for k in (1, 7, 8, 9, 15, 16, 17, 31, 40, 250):
        for off in range(8):
            flat = torch.randn(off + 5 * k, generator=g).to(dtype).cuda()
            views = [flat[off:].view(5, k)]
            if k > off:
                views.append(torch.randn(5, k, generator=g).to(dtype).cuda()[:, off:])
            for x in views:
                want, scale = plain_rows(x.cpu())
                q, s = Q.quantize_rows(x)
                assert torch.equal(s.cpu(), scale) and torch.equal(q.cpu().double(), want)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("scale", [1.0, 3.7e-5, 1e-30, 1e19, 3e22, 1e36])
def test_quantize_rows_near_to_halves(Q, dtype, scale):
    """Quotients at and next to a half, as 16-bit numbers have many: whole numbers and halves, their largest 127 or anything."""
    g = gen(17)
    x = (torch.randn(300, 1001, generator=g) * 40).clamp(-126, 126)
    for t in (x.round() + 0.5, x.round(), x):
        for first in (127.0, 126.0, None):
            y = t.clone()
            if first is not None:
                y[:, 0] = first
            y = (y * scale).to(dtype)
            want, s64 = plain_rows(y)
            q, s = Q.quantize_rows(y.cuda())
            assert torch.equal(s.cpu(), s64) and torch.equal(q.cpu().double(), want)


@pytest.mark.parametrize("m", [1, 2, 3, 4, 5])
@pytest.mark.parametrize("k,n", [(1, 3), (15, 1), (17, 40), (1000, 37), (2048, 100), (4096, 64), (4100, 33), (9000, 20), (50000, 9)])
def test_linear_int8_of_few_rows(Q, ops, m, k, n):
    """A decoding step: the same bits whether the rows are quantised in the call, before it, or among many rows."""
    g = gen(m * k + n)
    x = torch.randn(m, k, generator=g).to(BF).cuda()
    w, ws = weights(n, k, 5)
    bias = torch.randn(n, generator=g).cuda()
    out = Q.linear_int8(x, w, ws, bias)
    q, s = plain_rows(x.cpu())
    check_linear(out, q, s, w, ws, bias, BF)
    xq, xs = Q.quantize_rows(x)
    assert torch.equal(Q.linear_int8_quantized(xq, xs, w, ws, bias, BF), out)
    many = torch.cat([x, torch.ones(130, k, dtype=BF, device="cuda")])
    assert torch.equal(Q.linear_int8(many, w, ws, bias)[:m], out)
    f = Q.linear_int8(x.float(), w, ws, None, dtype=F32)
    check_linear(f, *plain_rows(x.float().cpu()), w, ws, None, F32)
    ops.synchronize_and_check()


def test_linear_int8_does_not_read_behind_the_last_row(Q):
    """Weights whose last row ends with the array, at widths that are no multiple of 16; rows of x that hold nothing finite."""
    for k in (1, 33, 1000, 1023):
        pitch = (k + 15) // 16 * 16
        flat = torch.full((4 * pitch + k,), 3, dtype=I8, device="cuda")
        w = torch.as_strided(flat, (5, k), (pitch, 1))
        x = torch.ones(3, k, dtype=F32, device="cuda")
        x[1, k // 2] = float("inf")
        out = Q.linear_int8(x, w, torch.ones(5).cuda())
        assert out[1].isnan().all() and torch.equal(out[0], out[2])
        assert float((out[0].double() - 3.0 * k).abs().max()) <= 3.0 * k * 4 * U


@pytest.mark.parametrize("dtype", [BF, F32])
def test_one_number_broadcast_over_the_rows(Q, ops, dtype):
    """Rows of one element that all are the same one, as an expanded tensor has them."""
    x = torch.full((1, 1), -2.5, dtype=dtype).cuda()
    w, ws = weights(20, 1, 3)
    for m in (2, 5, 300):
        wide = x.expand(m, 1)
        q, s = Q.quantize_rows(wide)
        assert (q == -127).all() and torch.equal(s, Q.quantize_rows(x)[1].expand(m))
        assert torch.equal(Q.linear_int8(wide, w, ws), Q.linear_int8(wide.contiguous(), w, ws))
    ops.synchronize_and_check()


@pytest.mark.parametrize("m", [1, 4, 40, 200])
def test_linear_int8_of_the_largest_products(Q, ops, m):
    k, n = 131072, 70
    x = torch.full((m, k), -128, dtype=I8)
    x[1::2, ::5] = 127
    w = torch.full((n, k), -128, dtype=I8)
    w[1::2, 1::3] = 127
    out = Q.linear_int8_quantized(x.cuda(), torch.ones(m).cuda(), w.cuda(), torch.ones(n).cuda(), dtype=F32)
    want = x.double() @ w.double().T
    assert want[0, 0] == 2.0 ** 31 and torch.equal(out.cpu(), want.float())


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("m,k,n", [(1, 100, 70), (3, 40, 9), (40, 100, 70), (300, 333, 257)])
@pytest.mark.parametrize("sx,sw", [(2.0 ** -100, 2.0 ** -40), (2.0 ** -30, 2.0 ** -105), (1e-25, 1e-20), (1e-38, 1.7e-4), (2.0 ** -130, 2.0 ** 3), (1e30, 1e-30), (1e-20, 1e25)])
def test_linear_int8_of_small_scales(Q, ops, m, k, n, sx, sw, dtype):
    g = gen(m + k)
    x = torch.randint(-127, 128, (m, (k + 15) // 16 * 16), generator=g).to(I8)[:, :k]
    w, _ = weights(n, k, 3)
    xs, ws = (torch.rand(m, generator=g) + 0.5) * sx, (torch.rand(n, generator=g) + 0.5) * sw
    out = Q.linear_int8_quantized(x.cuda() if k % 16 == 0 else torch.nn.functional.pad(x, (0, -k % 16)).cuda()[:, :k], xs.cuda(), w, ws.cuda(), dtype=dtype)
    want = (x.double() @ w.cpu().double().T) * xs.double()[:, None] * ws.double()
    tol = 4 * U * want.abs() + 2.0 ** -149
    tol = tol + HALF[dtype] * (want.abs() + tol) + (2.0 ** -134 if dtype == BF else 0)
    err = (out.double().cpu() - want).abs()
    assert (err <= tol).all(), float((err / tol).max())


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("m,k,n", [(1, 64, 70), (3, 64, 9), (40, 64, 70), (300, 320, 257)])
@pytest.mark.parametrize("sx,sw", [(1e30, 1e30), (3e38, 2.0), (2.0 ** 100, 2.0 ** 27), (1e20, -1e20)])
def test_linear_int8_of_large_scales(Q, ops, m, k, n, sx, sw, dtype):
    """Scales whose product is beyond all numbers: a sum of 0 is 0 all the same, others overflow by their sign."""
    g = gen(m + k)
    x, w = (torch.randint(-2, 3, (r, k), generator=g).to(I8) for r in (m, n))
    x[:, 8:], w[1::2, 3:] = 0, 0
    bias = torch.randn(n, generator=g)
    out = Q.linear_int8_quantized(x.cuda(), torch.full((m,), sx).cuda(), w.cuda(), torch.full((n,), sw).cuda(), bias.cuda(), dtype=dtype).float().cpu()
    sums = (x.double() @ w.double().T)
    assert (sums == 0).any() and (sums > 0).any() and (sums < 0).any()
    want = (sums * (float(torch.tensor(sx)) * float(torch.tensor(sw))) + bias.double()).float().to(dtype).float()
    assert torch.equal(out, want)


@pytest.mark.parametrize("m", [1, 2, 3, 4, 5, 200])
@pytest.mark.parametrize("k", [1, 15, 33, 1000, 1023])
def test_products_of_rows_with_numbers_behind_them(Q, m, k):
    """Rows of both operands whose bytes up to the next row are not zero: none of them is in a sum."""
    pitch, g = (k + 15) // 16 * 16 + 16, gen(k)
    wide = [torch.randint(1, 128, (n, pitch), generator=g).to(I8) for n in (m, 70)]
    x, w = (t.cuda()[:, :k] for t in wide)
    out = Q.linear_int8_quantized(x, torch.ones(m).cuda(), w, torch.ones(70).cuda(), dtype=F32)
    want = wide[0][:, :k].double() @ wide[1][:, :k].double().T
    assert float(want.max()) < 2 ** 24 and torch.equal(out.double().cpu(), want)


def test_attention_over_what_the_operators_make(Q, ops):
    """A layer as a user writes it around them: 8-bit projection to queries, keys and values, norms and rotation where they lie, the
    bias of two chains; logits, softmax and sum over the values in 64 bits, against the same of 64-bit norms and rotation.

    A query's or key's element is off by its rounding (half a step of bf16 and below 32 u of its pair's length), a logit by at most the
    sum of those times the other's, d; then a weight of the softmax by a factor within exp(-2 d) and exp(2 d)."""
    import test_gpu_position_ops as T
    from distributed_xfold_b200 import position_ops as P
    n, c, heads, d = 70, 384, 16, 24
    g = gen(8)
    x = torch.randn(2, n, c, generator=g).to(BF).cuda()
    w8, ws = Q.quantize_rows((torch.randn(3 * c, c, generator=g) * c ** -0.5).cuda())
    proj = Q.linear_int8(x, w8, ws)
    check_linear(proj, *plain_rows(x), w8, ws, None, BF)
    q, k, v = (proj[..., i * c:(i + 1) * c].unflatten(-1, (heads, d)) for i in range(3))
    qw, kw = ((1 + 0.1 * torch.randn(d, generator=g)).cuda() for _ in range(2))
    rotation, pos = P.Rotation.make(d), torch.arange(n, dtype=torch.int32).cuda()
    chain, table = (torch.arange(n) // 40).int().cuda(), torch.randn(66, heads, generator=g).cuda()
    lut = torch.tensor(P.clipped_buckets(32), dtype=torch.int32).cuda()
    at = torch.arange(n).expand(2, -1)
    plain = [T.plain(t, w, None, None, 1e-6, f) for t, w, f in ((q, qw, d ** -0.5), (k, kw, 1.0))]
    want = [T.turned(y, rotation, at) for y in plain]
    off = [32 * U * T.pair_length(y, rotation) for y in plain]
    off = [e + HALF[BF] * (y.abs() + e) for e, y in zip(off, want)]
    P.norm_rotate_qk_(q, k, qw, kw, rotation, pos, q_scale=d ** -0.5)
    bias = P.relative_position_bias(table, lut, pos, None, chain, chain).double().cpu()
    b = (torch.arange(n)[None] - torch.arange(n)[:, None]).clamp(-32, 32) + 32
    assert torch.equal(bias, table.cpu().double()[torch.where(chain.cpu()[:, None] == chain.cpu(), b, 65)].permute(2, 0, 1))
    dot = lambda a, e: torch.einsum("bihd,bjhd->bhij", a, e)
    attend = lambda a, e: torch.softmax(dot(a, e) + bias, -1)
    out = torch.einsum("bhij,bjhd->bihd", attend(q.double().cpu(), k.double().cpu()), v.double().cpu())
    p = attend(*want)
    ref, mass = (torch.einsum("bhij,bjhd->bihd", p, t) for t in (v.double().cpu(), v.double().cpu().abs()))
    worst = (dot(off[0], want[1].abs() + off[1]) + dot(want[0].abs(), off[1])).amax(-1).permute(0, 2, 1)[..., None]
    assert ((out - ref).abs() <= torch.expm1(2 * worst) * mass + 1e-12).all() and float(worst.max()) < 0.1
    ops.synchronize_and_check()
