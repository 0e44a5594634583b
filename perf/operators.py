"""What an attention layer's inputs pass through, as cases that can be timed and compared.

  bias       a learned relative position bias by buckets, [heads, queries, keys], as numbers or in the form that the attention
             kernel reads (float16 times log2(e), rows padded to eight keys)
  bias_grad  the gradient of its table
  qk         root-mean-square norms of queries and keys for each head and the rotation by their positions
  qk_grad    the gradients of queries, keys and of the norms' weights
  int8       a linear layer in 8-bit integers: rows of activations are quantised in the call, a scale for each row and for each
             output channel

``run`` is the plain form of each, or, with ``own``, the call that a user makes.
"""
from __future__ import annotations

import functools
import math

import torch

own = False

DEV = "cuda"
LOG2E = 1.4426950408889634
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16}
EPS = 1e-6


def listed():
    return [
        # one new token against a long cache: latency alone
        {"name": "bias 1 x 4097", "op": "bias", "q": 1, "k": 4097, "heads": 32, "rule": "log_past", "groups": 0, "form": "f32"},
        # the trunk's 16 heads over an odd number of tokens of four chains, for the attention kernel
        {"name": "bias 1000 prepared", "op": "bias", "q": 1000, "k": 1000, "heads": 16, "rule": "clip", "groups": 4, "form": "prepared"},
        # the diffusion transformer's largest token count, as numbers
        {"name": "bias 2048", "op": "bias", "q": 2048, "k": 2048, "heads": 16, "rule": "log", "groups": 0, "form": "f32"},
        # fine-tuning: a short ragged sequence with a pair attention's four heads, then the largest
        {"name": "bias_grad 777", "op": "bias_grad", "q": 777, "k": 777, "heads": 4, "rule": "clip", "groups": 3, "form": "f32"},
        {"name": "bias_grad 2048", "op": "bias_grad", "q": 2048, "k": 2048, "heads": 16, "rule": "log", "groups": 0, "form": "bf16"},
        # eight sequences that each add a token far from their start
        {"name": "qk 8 x 1", "op": "qk", "batch": 8, "len": 1, "q_heads": 32, "k_heads": 8, "dim": 128, "rot": 128, "pairs": "halves", "type": "bf16", "start": 100000, "fused": 0},
        # five samples of an ordinary protein: heads of 48 in a fused projection, padded to 64
        {"name": "qk 5 x 384 fused", "op": "qk", "batch": 5, "len": 384, "q_heads": 16, "k_heads": 16, "dim": 48, "rot": 48, "pairs": "halves", "type": "bf16", "start": 0, "fused": 64},
        # long prompts with shared keys
        {"name": "qk 4 x 4096", "op": "qk", "batch": 4, "len": 4096, "q_heads": 32, "k_heads": 8, "dim": 128, "rot": 128, "pairs": "halves", "type": "bf16", "start": 0, "fused": 0},
        # training, half of each head rotated
        {"name": "qk_grad 2 x 2048", "op": "qk_grad", "batch": 2, "len": 2048, "q_heads": 16, "k_heads": 16, "dim": 64, "rot": 32, "pairs": "neighbours", "type": "bf16", "start": 0, "fused": 0},
        # one token through the diffusion transformer's width
        {"name": "int8 1 x 768 x 4096", "op": "int8", "rows": 1, "inner": 768, "cols": 4096, "type": "bf16", "bias": True},
        # five samples of 385 tokens; widths that are multiples of nothing wide
        {"name": "int8 1925 x 1000 x 1030", "op": "int8", "rows": 1925, "inner": 1000, "cols": 1030, "type": "bf16", "bias": True},
        # a long batch through wide layers
        {"name": "int8 8192 x 4096 x 4096", "op": "int8", "rows": 8192, "inner": 4096, "cols": 4096, "type": "bf16", "bias": False},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["bias", "bias_grad", "qk", "qk", "qk_grad", "int8", "int8", "int8"])
    if op in ("bias", "bias_grad"):
        heads = rng.choice([1, 4, 8, 16])
        k = _log(rng, 16, 2048)
        square = op == "bias" and rng.random() < 0.4
        q = k if square or rng.random() < 0.6 else _log(rng, 1, 2048)
        form = "prepared" if square else rng.choice(["f32", "bf16"])
        return {"op": op, "q": q, "k": k, "heads": heads, "rule": rng.choice(["clip", "log", "log_past"]), "groups": rng.choice([0, 2, 5]), "form": form}
    if op in ("qk", "qk_grad"):
        heads, shared = rng.choice([(4, 1), (16, 1), (32, 4), (12, 3)])
        dim = rng.choice([24, 32, 48, 64, 80, 128])
        rot = rng.choice([dim, dim // 2])
        tokens = _log(rng, 1, 8192 if op == "qk" else 4096)
        batch = rng.choice([1, 1, 2, 5])
        return {"op": op, "batch": batch, "len": max(1, tokens // batch), "q_heads": heads, "k_heads": heads // shared, "dim": dim, "rot": rot,
                "pairs": rng.choice(["halves", "neighbours"]), "type": rng.choice(["bf16", "bf16", "f32"]), "start": rng.choice([0, 1000, 500000]),
                "fused": rng.choice([0, dim, -(-dim // 32) * 32])}
    rows = rng.choice([_log(rng, 1, 64), _log(rng, 32, 6000)])
    return {"op": op, "rows": rows, "inner": _log(rng, 100, 5000), "cols": _log(rng, 100, 5000), "type": rng.choice(["bf16", "bf16", "f32"]),
            "bias": rng.random() < 0.5}


# ---------------------------------------------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------------------------------------------
def _log_bucket(distance, exact, last, buckets):
    """Distances below `exact` have a bucket each; those up to `last` share the rest, each as many times longer as the one before."""
    b = distance if distance < exact else buckets - 1
    if exact <= distance < last:
        steps = buckets - exact   # the largest step with distance / exact >= (last / exact) ^ (step / steps), in whole numbers
        b = exact + max(s for s in range(steps) if distance ** steps >= last ** s * exact ** (steps - s))
    return b


def _rule(name):
    """Buckets of the offsets -reach .. reach (key minus query); offsets beyond are taken as the last ones."""
    if name == "clip":       # 65 buckets, one for each offset up to 32
        return 32, list(range(65))
    if name == "log":        # 32 buckets, half of them for keys behind the query
        return 128, [(16 if d > 0 else 0) + _log_bucket(abs(d), 8, 128, 16) for d in range(-128, 129)]
    return 128, [_log_bucket(max(-d, 0), 16, 128, 32) for d in range(-128, 129)]   # 32 buckets, keys before the query


def _positions(g, n, groups):
    """Residue numbers as complexes have them: chains one after the other, a few numbers left out, some tokens with the same one."""
    if not groups:
        return torch.arange(n, device=DEV, dtype=torch.int32), None
    step = torch.randint(0, 20, (n,), generator=g, device=DEV)
    step = torch.where(step == 0, 0, torch.where(step == 1, 3, 1))
    return torch.cumsum(step, 0).to(torch.int32), (torch.arange(n, device=DEV) * groups // n).to(torch.int32)


def _heads(g, case, heads, at):
    b, n, d, t = case["batch"], case["len"], case["dim"], TYPES[case["type"]]
    x = torch.randn(b, n, heads, d, generator=g, device=DEV) * (0.5 + torch.rand(d, generator=g, device=DEV))
    if not case["fused"]:
        return x.to(t)
    # where a projection to queries, keys, values and gate leaves them: heads `fused` apart, rows of all four
    pitch, width = case["fused"], case["fused"] * (case["q_heads"] + case["k_heads"]) * 2
    buf = torch.zeros(b, n, width, dtype=t, device=DEV)
    view = buf[..., at * pitch:(at + heads) * pitch].unflatten(-1, (heads, pitch))[..., :d]
    view.copy_(x)
    return view


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    rand = lambda *s: torch.randn(*s, generator=g, device=DEV)  # noqa: E731
    s = {"case": case}
    if case["op"] in ("bias", "bias_grad"):
        reach, lut = _rule(case["rule"])
        s["reach"], s["buckets"] = reach, torch.tensor(lut, dtype=torch.int32, device=DEV)
        n = max(lut) + 1 + (1 if case["groups"] else 0)
        longest = max(case["q"], case["k"])
        pos, grp = _positions(g, longest, case["groups"])
        s["k_pos"], s["q_pos"] = pos[:case["k"]], pos[longest - case["q"]:] if case["q"] < case["k"] else pos[:case["q"]]
        s["k_grp"], s["q_grp"] = (None, None) if grp is None else (grp[:case["k"]], grp[longest - case["q"]:] if case["q"] < case["k"] else grp[:case["q"]])
        s["rows"] = n
        if case["op"] == "bias":
            s["table"] = rand(n, case["heads"])
        else:
            s["grad"] = rand(case["heads"], case["q"], case["k"]).to(TYPES[case["form"]])
    elif case["op"] in ("qk", "qk_grad"):
        s["q"], s["k"] = _heads(g, case, case["q_heads"], 0), _heads(g, case, case["k_heads"], case["q_heads"])
        s["q_w"], s["k_w"] = (1.0 + 0.1 * rand(case["dim"]) for _ in range(2))
        half = case["rot"] // 2
        s["freqs"] = 10000.0 ** (-torch.arange(half, dtype=torch.float64, device=DEV) / half)
        s["pos"] = (case["start"] + torch.arange(case["len"], device=DEV)).to(torch.int32).expand(case["batch"], -1).contiguous()
        s["scale"] = case["dim"] ** -0.5
        if case["op"] == "qk_grad":
            s["dq"], s["dk"] = (rand(case["batch"], case["len"], case[h], case["dim"]).to(TYPES[case["type"]]) for h in ("q_heads", "k_heads"))
    else:
        m, kk, n, t = case["rows"], case["inner"], case["cols"], TYPES[case["type"]]
        # a few input channels are much larger than the others, as behind a LayerNorm
        x = rand(m, kk) * torch.where(torch.rand(kk, generator=g, device=DEV) < 0.01, 8.0, 1.0)
        s["x"] = x.to(t)
        # weights as they are kept: rows of 8-bit integers, a multiple of 16 bytes apart
        w = torch.zeros(n, -(-kk // 16) * 16, dtype=torch.int8, device=DEV)
        w[:, :kk] = (rand(n, kk) * 32).round().clamp(-127, 127).to(torch.int8)
        s["w"] = w[:, :kk]
        s["w_scale"] = kk ** -0.5 / 32 * (0.5 + torch.rand(n, generator=g, device=DEV))
        s["b"] = 0.1 * rand(n) if case["bias"] else None
    return s


# ---------------------------------------------------------------------------------------------------------------
# plain forms
# ---------------------------------------------------------------------------------------------------------------
def _buckets(s):
    d = (s["k_pos"][None, :] - s["q_pos"][:, None]).clamp(-s["reach"], s["reach"]) + s["reach"]
    b = s["buckets"][d].long()
    return b if s["k_grp"] is None else torch.where(s["q_grp"][:, None] == s["k_grp"][None, :], b, s["rows"] - 1)


def _plain_bias(s):
    out = s["table"].t()[:, _buckets(s)]
    form = s["case"]["form"]
    return (out * LOG2E).clamp(-60000.0, 60000.0).half() if form == "prepared" else out.to(TYPES[form])


def _plain_bias_grad(s):
    hot = _buckets(s).flatten()[:, None] == torch.arange(s["rows"], device=DEV)   # long sums: in 64 bits
    return (s["grad"].flatten(1).double() @ hot.double()).t().float().contiguous()


def _turn(x, c, s, pairs):
    """The pairs of x's last axis turned by angles with cosine c and sine s."""
    if pairs == "halves":
        a, b = x.chunk(2, -1)
        return torch.cat([a * c - b * s, b * c + a * s], -1)
    a, b = x[..., 0::2], x[..., 1::2]
    return torch.stack([a * c - b * s, b * c + a * s], -1).flatten(-2)


def _angles(s):
    t = s["pos"].double()[..., None] * s["freqs"]   # far positions: in 64 bits
    return t.cos().float()[:, :, None], t.sin().float()[:, :, None]


def _plain_qk(s):
    rot, pairs = s["case"]["rot"], s["case"]["pairs"]
    c, sn = _angles(s)

    def one(x, w, scale):
        y = x.float()
        y = y * torch.rsqrt((y * y).mean(-1, keepdim=True) + EPS) * (w * scale)
        return torch.cat([_turn(y[..., :rot], c, sn, pairs), y[..., rot:]], -1).to(x.dtype)
    return one(s["q"], s["q_w"], s["scale"]), one(s["k"], s["k_w"], 1.0)


def _plain_qk_grad(s):
    rot, pairs = s["case"]["rot"], s["case"]["pairs"]
    c, sn = _angles(s)

    def one(d, x, w, scale):
        g, y = d.float(), x.float()
        g = torch.cat([_turn(g[..., :rot], c, -sn, pairs), g[..., rot:]], -1) * scale
        r = torch.rsqrt((y * y).mean(-1, keepdim=True) + EPS)
        dw = (g * y * r).double().sum((0, 1, 2)).float()   # long sums: in 64 bits
        gw = g * w
        return (r * (gw - y * (r * r * (gw * y).mean(-1, keepdim=True)))).to(x.dtype), dw
    (dq, dqw), (dk, dkw) = one(s["dq"], s["q"], s["q_w"], s["scale"]), one(s["dk"], s["k"], s["k_w"], 1.0)
    return dq, dk, dqw, dkw


def _plain_int8(s):
    x = s["x"].float()
    scale = x.abs().amax(1, keepdim=True) / 127
    q = (x.double() / scale.double()).round().float()   # next to a border: in 64 bits
    y = q @ s["w"].float().t() * scale * s["w_scale"]
    return (y if s["b"] is None else y + s["b"]).to(s["x"].dtype)


@functools.cache
def _package():
    import __graft_entry__ as entry
    entry.load_package()
    from distributed_xfold_b200 import int8_ops, position_ops
    return int8_ops, position_ops


def run(state):
    s, case = state, state["case"]
    if own:
        int8_ops, position_ops = _package()
        if case["op"] == "bias":
            out = position_ops.relative_position_bias(s["table"], s["buckets"], s["q_pos"], s["k_pos"], s["q_grp"], s["k_grp"],
                                                      dtype=TYPES.get(case["form"], torch.float16), prepared=case["form"] == "prepared")
            return out[..., :case["k"]]
        if case["op"] == "bias_grad":
            return position_ops.relative_position_bias_backward(s["grad"], s["rows"], s["buckets"], s["q_pos"], s["k_pos"], s["q_grp"], s["k_grp"])
        if case["op"] == "int8":
            return int8_ops.linear_int8(s["x"], s["w"], s["w_scale"], s["b"])
        rotation = position_ops.Rotation(s["freqs"], interleaved=case["pairs"] == "neighbours")
        if case["op"] == "qk":
            return position_ops.norm_rotate_qk(s["q"], s["k"], s["q_w"], s["k_w"], rotation, s["pos"], eps=EPS, q_scale=s["scale"])
        return position_ops.norm_rotate_qk_backward(s["dq"], s["dk"], s["q"], s["k"], s["q_w"], s["k_w"], rotation, s["pos"], eps=EPS, q_scale=s["scale"])
    return {"bias": _plain_bias, "bias_grad": _plain_bias_grad, "qk": _plain_qk, "qk_grad": _plain_qk_grad, "int8": _plain_int8}[case["op"]](s)


# ---------------------------------------------------------------------------------------------------------------
# the work, and the definition in 64 bits
# ---------------------------------------------------------------------------------------------------------------
def work(case):
    if case["op"] in ("bias", "bias_grad"):
        n = case["heads"] * case["q"] * case["k"]
        return {"bytes": n * (4 if case["form"] == "f32" else 2) + 4 * (case["q"] + case["k"]), "flops": n}
    if case["op"] in ("qk", "qk_grad"):
        n = case["batch"] * case["len"] * (case["q_heads"] + case["k_heads"]) * case["dim"]
        e, passes = (4 if case["type"] == "f32" else 2), (2 if case["op"] == "qk" else 3)
        return {"bytes": n * e * passes + 4 * case["batch"] * case["len"], "flops": n * (8 if case["op"] == "qk" else 16)}
    m, k, n, e = case["rows"], case["inner"], case["cols"], (4 if case["type"] == "f32" else 2)
    return {"bytes": m * k * e + n * k + m * n * e + 8 * n, "flops": 2 * m * n * k}


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] in ("bias", "bias_grad"):
        reach, lut = _rule(case["rule"])
        far = s["k_pos"].long()[None, :] - s["q_pos"].long()[:, None]
        b = torch.tensor(lut, device=DEV)[far.clamp(min=-reach).clamp(max=reach) + reach]
        if case["groups"]:
            b = b.masked_fill(s["q_grp"].long()[:, None] != s["k_grp"].long()[None, :], s["rows"] - 1)
        if case["op"] == "bias":
            out = s["table"].double()[b].permute(2, 0, 1)
            return (out * math.log2(math.e)).clamp(-6e4, 6e4) if case["form"] == "prepared" else out
        grad = s["grad"].double()
        return torch.stack([torch.where(b == row, grad, 0.0).sum((1, 2)) for row in range(s["rows"])])
    if case["op"] == "int8":
        x = s["x"].double()
        scale = (x.abs().max(1).values / 127).float().double()   # the scale is a 32-bit number
        y = torch.einsum("mk,nk->mn", torch.round(x / scale[:, None]), s["w"].double()) * torch.outer(scale, s["w_scale"].double())
        return y if s["b"] is None else y + s["b"].double()
    # pairs as complex numbers; the gradient through a graph of the forward in 64 bits
    rot, half = case["rot"], case["rot"] // 2
    turn = torch.polar(torch.ones((), dtype=torch.float64, device=DEV), s["pos"].double()[:, :, None, None] * s["freqs"])

    def forward(x, w, scale):
        y = scale * w * x / (x.square().mean(-1, keepdim=True) + EPS).sqrt()
        z = y[..., :rot]
        z = torch.complex(z[..., :half], z[..., half:]) if case["pairs"] == "halves" else torch.view_as_complex(z.unflatten(-1, (half, 2)).contiguous())
        z = torch.view_as_real(z * turn)
        z = torch.cat([z[..., 0], z[..., 1]], -1) if case["pairs"] == "halves" else z.flatten(-2)
        return torch.cat([z, y[..., rot:]], -1)
    args = [(s[n].double(), s[n + "_w"].double(), f) for n, f in (("q", s["scale"]), ("k", 1.0))]
    if case["op"] == "qk":
        return [forward(*a) for a in args]
    got = []
    for (x, w, f), d in zip(args, (s["dq"], s["dk"])):
        x, w = x.requires_grad_(), w.requires_grad_()
        got.append(torch.autograd.grad(forward(x, w, f), [x, w], d.double()))
    return got[0][0], got[1][0], got[0][1], got[1][1]
