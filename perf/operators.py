"""The operators of a transformer over point patches, as cases that can be timed and checked.

A model that reads or writes clouds patch by patch normalises its tokens (layer norm), lets
the tokens of one cloud attend to each other (attention over packed sequences of different
lengths, or of one new token over a cache), and widens them through a gated projection.  Each
case is one call, or one forward and backward pass, of one of the three.  `own` chooses between
the package's operators and their plain form in elementary operations of torch.
"""
import math
import os
import sys

import torch

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "f16": 2, "bf16": 2}
EPS = 1e-5


def listed():
    return [
        # layer norm of the newest token of 16 clouds that are generated together
        {"name": "norm_bf16_16x512", "op": "norm", "rows": 16, "width": 512, "dtype": "bf16",
         "mode": "forward"},
        # a training step's tokens: 16 clouds of 2048 patches
        {"name": "norm_train_bf16_32768x1024", "op": "norm", "rows": 32768, "width": 1024,
         "dtype": "bf16", "mode": "train"},
        # features of ungrouped points with their coordinates appended, in full precision
        {"name": "norm_train_f32_5000x771", "op": "norm", "rows": 5000, "width": 771,
         "dtype": "f32", "mode": "train"},
        # one cloud's next token over a short cache: the latency of interactive generation
        {"name": "step_f16_1x300", "op": "attention", "B": 1, "queries": 1, "room": 512,
         "longest": 300, "heads": 8, "group": 1, "D": 64, "causal": True, "dtype": "f16",
         "mode": "forward"},
        # the next token of 64 clouds over long caches, four query heads to a cached head
        {"name": "step_bf16_64x16384", "op": "attention", "B": 64, "queries": 1, "room": 16384,
         "longest": 16384, "heads": 4, "group": 4, "D": 128, "causal": True, "dtype": "bf16",
         "mode": "forward"},
        # the prompts of eight clouds, packed, before generation
        {"name": "prompt_bf16_8x4096", "op": "attention", "B": 8, "queries": 0, "room": 0,
         "longest": 4096, "heads": 4, "group": 4, "D": 128, "causal": True, "dtype": "bf16",
         "mode": "forward"},
        # a training step of an autoregressive patch decoder
        {"name": "prompt_train_bf16_8x2048", "op": "attention", "B": 8, "queries": 0, "room": 0,
         "longest": 2048, "heads": 8, "group": 2, "D": 64, "causal": True, "dtype": "bf16",
         "mode": "train"},
        # an encoder's training step in full precision: every patch sees its whole cloud
        {"name": "prompt_train_f32_5x600", "op": "attention", "B": 5, "queries": 0, "room": 0,
         "longest": 600, "heads": 6, "group": 1, "D": 40, "causal": False, "dtype": "f32",
         "mode": "train"},
        # gated projection of the newest tokens of 16 clouds: reading the weights
        {"name": "gated_bf16_16x512x1408", "op": "gated", "rows": 16, "K": 512, "F": 1408,
         "activation": "silu", "dtype": "bf16", "mode": "forward"},
        # a training step's tokens: 8 clouds of 2048 patches
        {"name": "gated_train_bf16_16384x1024x4096", "op": "gated", "rows": 16384, "K": 1024,
         "F": 4096, "activation": "silu", "dtype": "bf16", "mode": "train"},
        # the prompts of a wide model
        {"name": "gated_bf16_8192x2048x8192", "op": "gated", "rows": 8192, "K": 2048, "F": 8192,
         "activation": "gelu", "dtype": "bf16", "mode": "forward"},
        # a small model's step in full precision, features with odd widths
        {"name": "gated_train_f32_1000x385x1023", "op": "gated", "rows": 1000, "K": 385,
         "F": 1023, "activation": "gelu", "dtype": "f32", "mode": "train"},
    ]


def _size(rng, lo, hi):
    """A size of [lo, hi], spread over its logarithm; every other one a multiple of 64."""
    n = int(round(lo * (hi / lo) ** rng.random()))
    if rng.random() < 0.5 and n >= 64:
        n -= n % 64
    n = max(lo, min(hi, n))
    return n - 1 if n == 3072 else n


def draw(rng):
    op = rng.choice(["norm", "step", "prompt", "prompt", "gated", "gated"])
    dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
    mode = rng.choice(["forward", "train"])
    if op == "norm":
        c = {"op": op, "rows": _size(rng, 1, 32768), "width": _size(rng, 64, 8192),
             "dtype": dtype, "mode": mode}
        while c["rows"] * c["width"] * SIZE[dtype] > 32768 * 1024 * 2:
            c["rows"] = c["rows"] * 3 // 4
        return c
    if op == "gated":
        c = {"op": op, "rows": _size(rng, 1, 16384), "K": _size(rng, 64, 2048),
             "F": _size(rng, 128, 8192), "activation": rng.choice(["silu", "silu", "gelu"]),
             "dtype": dtype, "mode": mode}
        while c["rows"] * c["K"] * c["F"] * (3 if mode == "train" else 1) > 3 * 2 ** 36:
            c["rows"] = c["rows"] * 3 // 4
        return c
    D, group = rng.choice([32, 40, 64, 64, 80, 96, 128, 128]), rng.choice([1, 2, 4, 8])
    if op == "step":
        c = {"op": "attention", "B": _size(rng, 1, 64), "queries": rng.choice([1, 1, 1, 2, 5]),
             "room": 0, "longest": _size(rng, 64, 16384), "heads": rng.choice([1, 2, 4, 8]),
             "group": group, "D": D, "causal": True, "dtype": dtype, "mode": "forward"}
        c["room"] = c["longest"] + rng.choice([0, 0, 1, 100])
        while c["B"] > 1 and c["B"] * c["room"] * c["heads"] * D * SIZE[dtype] > 2 ** 30:
            c["B"] -= 1
        if c["room"] == 3072:
            c["room"] += 1
        return c
    c = {"op": "attention", "B": _size(rng, 1, 16), "queries": 0, "room": 0,
         "longest": _size(rng, 16, 4096), "heads": rng.choice([1, 2, 4, 8]), "group": group,
         "D": D, "causal": rng.random() < 0.7, "dtype": dtype, "mode": mode}
    most = 2 ** 28 if mode == "train" else 2 ** 31
    while c["B"] > 1 and c["B"] * c["longest"] ** 2 * c["heads"] * group > most:
        c["B"] -= 1
    while c["longest"] ** 2 * c["heads"] * group > most:
        c["longest"] = c["longest"] * 3 // 4
    return c


def _lengths(case):
    """Tokens of each sequence: the longest, and others down to a quarter of it (in steps of
    the golden section, so that any number of them covers the range evenly)."""
    top = case["longest"]
    low = max(1, top // 4, case["queries"])
    return [top] + [low + int((top - low) * (b * 0.6180339887 % 1)) for b in range(1, case["B"])]


def _randn(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda")


def prepare(case, seed):
    g = torch.Generator("cuda").manual_seed(seed)
    t, train = DTYPES[case["dtype"]], case["mode"] == "train"
    s = {"case": case}
    if case["op"] == "norm":
        R, C = case["rows"], case["width"]
        # a residual stream: every token has a level and a scale of its own
        s["x"] = (_randn(g, R, C) * (0.5 + 1.5 * torch.rand(R, 1, generator=g, device="cuda"))
                  + 0.3 * _randn(g, R, 1)).to(t)
        s["w"] = (1 + 0.1 * _randn(g, C)).to(t)
        s["b"] = (0.1 * _randn(g, C)).to(t)
        s["gy"] = _randn(g, R, C).to(t) if train else None
        leaves = ("x", "w", "b")
    elif case["op"] == "gated":
        R, K, F = case["rows"], case["K"], case["F"]
        s["x"] = _randn(g, R, K).to(t)  # as a norm leaves it
        s["wg"] = (_randn(g, F, K) / K ** 0.5).to(t)
        s["wu"] = (_randn(g, F, K) / K ** 0.5).to(t)
        s["gh"] = _randn(g, R, F).to(t) if train else None
        leaves = ("x", "wg", "wu")
    else:
        B, D, Hk = case["B"], case["D"], case["heads"]
        Hq = Hk * case["group"]
        lengths = _lengths(case)
        order = torch.randperm(B, generator=g, device="cuda")
        lk = torch.tensor(lengths, device="cuda")[order]
        if case["queries"]:  # a cache with room for every sequence, filled in part
            s["ok"] = torch.arange(B + 1, device="cuda") * case["room"]
            s["lk"] = lk
            s["oq"] = torch.arange(B + 1, device="cuda") * case["queries"]
            Tq, Tk = B * case["queries"], B * case["room"]
            s["longest_q"] = case["queries"]
        else:
            s["oq"] = s["ok"] = torch.nn.functional.pad(lk.cumsum(0), (1, 0))
            s["lk"] = None
            Tq = Tk = sum(lengths)
            s["longest_q"] = case["longest"]
        s["longest_k"] = case["longest"]
        s["q"] = _randn(g, Tq, Hq, D).to(t)
        s["k"] = _randn(g, Tk, Hk, D).to(t)
        s["v"] = _randn(g, Tk, Hk, D).to(t)
        s["go"] = _randn(g, Tq, Hq, D).to(t) if train else None
        leaves = ("q", "k", "v")
    if train:
        for n in leaves:
            s[n].requires_grad_(True)
    return s


def _package():
    """The package, from the torch-point-ops_amd folder of the working folder."""
    at = os.path.abspath("torch-point-ops_amd")
    if at not in sys.path:
        sys.path.insert(0, at)
    import torch_point_ops

    return torch_point_ops


def _own(s, case):
    tpo = _package()
    train = case["mode"] == "train"
    if case["op"] == "norm":
        y = tpo.layer_norm(s["x"], s["w"], s["b"], EPS)
        return (y, *torch.autograd.grad(y, (s["x"], s["w"], s["b"]), s["gy"])) if train else y
    if case["op"] == "gated":
        h = tpo.gated_projection(s["x"], s["wg"], s["wu"], activation=case["activation"])
        return (h, *torch.autograd.grad(h, (s["x"], s["wg"], s["wu"]), s["gh"])) if train else h
    o = tpo.packed_attention(s["q"], s["k"], s["v"], s["oq"], s["ok"], lengths_k=s["lk"],
                             causal=case["causal"])
    return (o, *torch.autograd.grad(o, (s["q"], s["k"], s["v"]), s["go"])) if train else o


def _plain_norm(s, train):
    t, x, w = s["x"].dtype, s["x"].float(), s["w"].float()
    mean = x.mean(1, keepdim=True)
    x = x - mean
    r = torch.rsqrt((x * x).mean(1, keepdim=True) + EPS)
    x = x * r
    y = (x * w + s["b"].float()).to(t)
    if not train:
        return y
    gy = s["gy"].float()
    g = gy * w
    gx = r * (g - g.mean(1, keepdim=True) - x * (g * x).mean(1, keepdim=True))
    return y, gx.to(t), (gy * x).sum(0).to(t), gy.sum(0).to(t)


def _act(g, name):
    """The activation and its derivative."""
    if name == "silu":
        e = torch.sigmoid(g)
        return g * e, e * (1 + g * (1 - e))
    c = 0.5 * (1 + torch.erf(g * 0.5 ** 0.5))
    return g * c, c + g * torch.exp(-0.5 * g * g) * (2 * math.pi) ** -0.5


def _plain_gated(s, name, train):
    t, x, wg, wu = s["x"].dtype, s["x"].float(), s["wg"].float(), s["wu"].float()
    g, u = x @ wg.t(), x @ wu.t()
    a, d = _act(g, name)
    h = (a * u).to(t)
    if not train:
        return h
    gh = s["gh"].float()
    dg, du = gh * u * d, gh * a
    return (h, (dg @ wg + du @ wu).to(t), (dg.t() @ x).to(t), (du.t() @ x).to(t))


def _padded(x, offsets, lengths, longest):
    """(B, longest, heads, D) in float of rows packed in x, where each row stands, and which
    of them are a sequence's."""
    at = torch.arange(longest, device="cuda")
    there = at < lengths[:, None]
    at = offsets[:-1, None] + at
    rows = x[torch.where(there, at, 0)].float()
    return rows * there[..., None, None], torch.where(there, at, x.shape[0]), there


def _packed(x, at, like):
    """Rows of a padded batch back in their places, in like's shape and type."""
    out = torch.zeros(like.shape[0] + 1, *like.shape[1:], device="cuda")
    out[at] = x
    return out[:-1].to(like.dtype)


def _plain_attention(s, case, train):
    B, Hk, G, D = case["B"], case["heads"], case["group"], case["D"]
    lq = s["oq"][1:] - s["oq"][:-1]
    lk = s["lk"] if s["lk"] is not None else s["ok"][1:] - s["ok"][:-1]
    Lq, Lk = s["longest_q"], s["longest_k"]

    def by_head(x, L):  # (B, L, Hk g, D) -> (B Hk, g L, D)
        return x.view(B, L, Hk, -1, D).permute(0, 2, 3, 1, 4).reshape(B * Hk, -1, D)

    def by_token(x, L):
        return x.view(B, Hk, -1, L, D).permute(0, 3, 1, 2, 4).reshape(B, L, -1, D)

    q, at_q, in_q = _padded(s["q"], s["oq"], lq, Lq)
    k, at_k, in_k = _padded(s["k"], s["ok"], lk, Lk)
    v = _padded(s["v"], s["ok"], lk, Lk)[0]
    q, k, v = by_head(q, Lq), by_head(k, Lk), by_head(v, Lk)
    seen = in_q[:, :, None] & in_k[:, None]
    if case["causal"]:
        i, j = torch.arange(Lq, device="cuda"), torch.arange(Lk, device="cuda")
        seen &= j <= i[:, None] + (lk - lq)[:, None, None]
    seen = seen[:, None, None]  # (B, 1, 1, Lq, Lk)
    scale = D ** -0.5
    p = torch.bmm(q, k.transpose(1, 2).contiguous()).mul_(scale).view(B, Hk, G, Lq, Lk)
    p = p.masked_fill_(~seen, float("-inf"))
    top = p.amax(-1, keepdim=True)
    p = p.sub_(torch.where(top == float("-inf"), 0, top)).exp_()
    p = p.div_(p.sum(-1, keepdim=True).clamp_(min=1e-30)).view(B * Hk, G * Lq, Lk)
    out = torch.bmm(p, v)
    o = _packed(by_token(out, Lq), at_q, s["q"])
    if not train:
        return o
    go = by_head(_padded(s["go"], s["oq"], lq, Lq)[0], Lq)
    pt = p.transpose(1, 2).contiguous()
    dv = torch.bmm(pt, go)
    ds = torch.bmm(go, v.transpose(1, 2).contiguous())
    ds = ds.sub_((go * out).sum(-1, keepdim=True)).mul_(p).mul_(scale)
    dq = torch.bmm(ds, k)
    dk = torch.bmm(ds.transpose(1, 2).contiguous(), q)
    return (o, _packed(by_token(dq, Lq), at_q, s["q"]), _packed(by_token(dk, Lk), at_k, s["k"]),
            _packed(by_token(dv, Lk), at_k, s["v"]))


def run(s):
    case = s["case"]
    if own:
        return _own(s, case)
    train = case["mode"] == "train"
    with torch.no_grad():
        if case["op"] == "norm":
            return _plain_norm(s, train)
        if case["op"] == "gated":
            return _plain_gated(s, case["activation"], train)
        return _plain_attention(s, case, train)


def work(case):
    z, train = SIZE[case["dtype"]], case["mode"] == "train"
    if case["op"] == "norm":
        n = case["rows"] * case["width"]
        return {"bytes": n * z * (4 if train else 2) + case["width"] * z * (4 if train else 2),
                "flops": n * (20 if train else 8)}
    if case["op"] == "gated":
        R, K, F = case["rows"], case["K"], case["F"]
        once = R * K + 2 * F * K
        return {"bytes": z * ((2 * once + 2 * R * F) if train else (once + R * F)),
                "flops": R * K * F * (12 if train else 4)}
    lk = _lengths(case)
    lq = [case["queries"] or n for n in lk]
    Hk, D = case["heads"], case["D"]
    Hq = Hk * case["group"]
    # keys that the rows of a sequence see: all, or one more for each row up to the last
    pairs = sum(a * b - (a * (a - 1) // 2 if case["causal"] else 0) for a, b in zip(lq, lk))
    q, kv = sum(lq) * Hq * D, 2 * sum(lk) * Hk * D
    return {"bytes": z * ((4 * q + 2 * kv) if train else (2 * q + kv)),
            "flops": pairs * Hq * D * (14 if train else 4)}


def _with_grads(f, leaves, grad):
    """f of the leaves in 64 bits and, where an output gradient is given, theirs."""
    x = [v.detach().double().requires_grad_(grad is not None) for v in leaves]
    y = f(*x)
    if grad is None:
        return y
    return (y.detach(), *torch.autograd.grad(y, x, grad.double()))


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "norm":
        def norm(x, w, b):
            var, mean = torch.var_mean(x, -1, correction=0, keepdim=True)
            return (x - mean) / (var + EPS).sqrt() * w + b
        return _with_grads(norm, (s["x"], s["w"], s["b"]), s["gy"])
    if case["op"] == "gated":
        def gated(x, wg, wu):
            g = torch.matmul(x, wg.T)
            a = g / (1 + torch.exp(-g)) if case["activation"] == "silu" else \
                g * torch.special.ndtr(g)
            return a * torch.matmul(x, wu.T)
        return _with_grads(gated, (s["x"], s["wg"], s["wu"]), s["gh"])
    # one sequence after another, each a dense problem of its own
    group, whole = case["group"], [torch.zeros(s[n].shape, dtype=torch.float64, device="cuda")
                                   for n in ("q", "q", "k", "v")]
    for b in range(case["B"]):
        q0, q1 = int(s["oq"][b]), int(s["oq"][b + 1])
        k0 = int(s["ok"][b])
        k1 = int(s["ok"][b + 1]) if s["lk"] is None else k0 + int(s["lk"][b])

        def attend(q, k, v):
            k, v = k.repeat_interleave(group, 1), v.repeat_interleave(group, 1)
            a = torch.matmul(q.transpose(0, 1), k.permute(1, 2, 0)) / case["D"] ** 0.5
            if case["causal"]:
                keep = torch.ones(a.shape[1:], dtype=torch.bool, device="cuda")
                a = a.masked_fill(~keep.tril(a.shape[2] - a.shape[1]), -math.inf)
            return torch.matmul(torch.softmax(a, -1), v.transpose(0, 1)).transpose(0, 1)

        go = None if s["go"] is None else s["go"][q0:q1]
        r = _with_grads(attend, (s["q"][q0:q1], s["k"][k0:k1], s["v"][k0:k1]), go)
        for out, part, at in zip(whole, r if go is not None else (r,),
                                 (slice(q0, q1), slice(q0, q1), slice(k0, k1), slice(k0, k1))):
            out[at] = part
    return tuple(whole) if s["go"] is not None else whole[0]
