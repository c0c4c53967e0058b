"""Positions and the 8-bit cache of a transformer over point patches, as cases that can be timed
and checked.

A model that generates clouds patch by patch turns its queries and keys by their places or
coordinates (rotary positions), puts the keys and values of new tokens into the pages of a cache
that holds them in 8 bits, and attends over that cache.  Each case is one call, or one forward and
backward pass, of one of the three.  `own` chooses between the package's operators and their plain
form in elementary operations of torch.

The cache, in blocks of 32 tokens (Dr: the head size D rounded up to 16):
  keys (pages, Hk, page / 32, Dr / 16, 32, 16), values (pages, Hk, page / 32, Dr, 32), e4m3 codes
  key_scales, value_scales (pages, Hk): a value is its code times the scale of its page and head
  table (B, M): the pages of each sequence; lengths (B): its tokens, those of this call included
"""
import os
import sys

import torch

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "f16": 2, "bf16": 2}
CODE = torch.float8_e4m3fn
MOST = 448.0  # the largest code


def listed():
    return [
        # queries and keys of the newest token of 16 clouds that are generated together
        {"name": "turn_f16_16x10x64", "op": "turn", "tokens": 16, "heads": 10, "D": 64,
         "part": 64, "axes": 1, "interleaved": False, "dtype": "f16", "mode": "forward"},
        # a training step's queries and keys: 16 clouds of 2048 patches
        {"name": "turn_train_bf16_32768x20x128", "op": "turn", "tokens": 32768, "heads": 20,
         "D": 128, "part": 128, "axes": 1, "interleaved": False, "dtype": "bf16",
         "mode": "train"},
        # an encoder in full precision: a part of each head turned by the patches' coordinates
        {"name": "turn_train_f32_3000x12x40", "op": "turn", "tokens": 3000, "heads": 12, "D": 40,
         "part": 24, "axes": 3, "interleaved": True, "dtype": "f32", "mode": "train"},
        # the newest token of 64 clouds goes into their pages, its queries turned on the way
        {"name": "append_bf16_64x1", "op": "append", "B": 64, "new": 1, "held": 1023, "heads": 8,
         "group": 4, "D": 128, "page": 64, "part": 128, "interleaved": False, "dtype": "bf16"},
        # the prompts of eight clouds into an empty cache
        {"name": "append_bf16_8x4096", "op": "append", "B": 8, "new": 4096, "held": 0, "heads": 4,
         "group": 4, "D": 128, "page": 64, "part": 128, "interleaved": False, "dtype": "bf16"},
        # pieces of prompts behind what is there, half of an odd head turned
        {"name": "append_f16_5x300", "op": "append", "B": 5, "new": 300, "held": 777, "heads": 6,
         "group": 1, "D": 80, "page": 32, "part": 40, "interleaved": True, "dtype": "f16"},
        # one cloud's next token over a short cache: the latency of interactive generation
        {"name": "cached_f16_1x300", "op": "cached", "B": 1, "queries": 1, "longest": 300,
         "heads": 8, "group": 1, "D": 64, "page": 64, "causal": True, "dtype": "f16"},
        # the next token of 64 clouds over long caches, four query heads to a cached head
        {"name": "cached_bf16_64x16384", "op": "cached", "B": 64, "queries": 1, "longest": 16384,
         "heads": 4, "group": 4, "D": 128, "page": 64, "causal": True, "dtype": "bf16"},
        # five guessed tokens at a time in full precision, heads of no power of two
        {"name": "cached_f32_7x2500x5", "op": "cached", "B": 7, "queries": 5, "longest": 2500,
         "heads": 6, "group": 2, "D": 40, "page": 32, "causal": True, "dtype": "f32"},
        # a piece of a long prompt over what its sequences hold already
        {"name": "cached_bf16_8x8192x1024", "op": "cached", "B": 8, "queries": 1024,
         "longest": 8192, "heads": 4, "group": 4, "D": 128, "page": 128, "causal": True,
         "dtype": "bf16"},
        # a short piece
        {"name": "cached_f16_3x1500x200", "op": "cached", "B": 3, "queries": 200,
         "longest": 1500, "heads": 8, "group": 1, "D": 96, "page": 64, "causal": True,
         "dtype": "f16"},
    ]


def _size(rng, lo, hi):
    """A size of [lo, hi], spread over its logarithm; every other one a multiple of 64."""
    n = int(round(lo * (hi / lo) ** rng.random()))
    if rng.random() < 0.5 and n >= 64:
        n -= n % 64
    return max(lo, min(hi, n))


def draw(rng):
    op = rng.choice(["turn", "append", "append", "cached", "cached", "cached"])
    dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
    D = rng.choice([32, 40, 64, 64, 80, 96, 128, 128])
    if op == "turn":
        axes = rng.choice([1, 1, 3])
        part = D if rng.random() < 0.6 else D // 2
        part -= part % (2 * axes)
        c = {"op": op, "tokens": _size(rng, 1, 32768), "heads": _size(rng, 1, 40), "D": D,
             "part": part, "axes": axes, "interleaved": rng.random() < 0.4, "dtype": dtype,
             "mode": rng.choice(["forward", "train"])}
        while c["tokens"] * c["heads"] * D * SIZE[dtype] > 32768 * 20 * 128 * 2:
            c["tokens"] = c["tokens"] * 3 // 4
        return c
    heads, group = rng.choice([1, 2, 4, 6, 8]), rng.choice([1, 2, 4, 8])
    page = rng.choice([32, 64, 64, 128])
    if op == "append":
        c = {"op": op, "B": _size(rng, 1, 64), "new": rng.choice([1, 1, 5, _size(rng, 16, 4096)]),
             "held": rng.choice([0, _size(rng, 1, 2000)]), "heads": heads, "group": group, "D": D,
             "page": page, "part": D if rng.random() < 0.6 else D // 4 * 2,
             "interleaved": rng.random() < 0.4, "dtype": dtype}
        most = 8 * 4096 * 4 * 128
        while c["B"] > 1 and (c["B"] * c["new"] * heads * (2 + group) * D * SIZE[dtype] > 12 * most
                              or c["B"] * (c["new"] + c["held"]) * heads * D > most):
            c["B"] -= 1
        return c
    c = {"op": op, "B": _size(rng, 1, 64),
         "queries": rng.choice([1, 1, 1, 2, 5, _size(rng, 16, 1024)]), "longest": 0,
         "heads": heads, "group": group, "D": D, "page": page, "causal": rng.random() < 0.8,
         "dtype": dtype}
    c["longest"] = _size(rng, max(16, c["queries"]), 16384)
    # keys' values, pairs
    while c["B"] > 1 and c["B"] * c["longest"] * heads * max(D, c["queries"] * group) > 2 ** 29:
        c["B"] -= 1
    return c


def _spread(top, low, B):
    """B counts: the largest, and others down to the lowest (in steps of the golden section, so
    that any number of them covers the range evenly)."""
    return [top] + [low + int((top - low) * (b * 0.6180339887 % 1)) for b in range(1, B)]


def _counts(case):
    """(tokens that are new, tokens with them) of each sequence."""
    if case["op"] == "cached":
        n = case["longest"]
        return [case["queries"]] * case["B"], _spread(n, max(1, n // 4, case["queries"]),
                                                      case["B"])
    new = _spread(case["new"], max(1, case["new"] // 4), case["B"])
    held = _spread(case["held"], case["held"] // 4, case["B"])
    return new, [a + b for a, b in zip(new, held)]


def _randn(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda")


def _frequencies(case):
    """Places: wave lengths of 2 pi to 20000 pi; coordinates of [-1, 1]: of 4 down to 1 / 16."""
    n = case["part"] // 2
    if case.get("axes", 1) == 1:
        return 1e4 ** (-torch.arange(n, device="cuda", dtype=torch.float64) / n)
    each = n // case["axes"]
    return (torch.pi / 2 * 64 ** (torch.arange(each, device="cuda", dtype=torch.float64)
                                  / each)).repeat(case["axes"])


def _pages(g, x):
    """x (pages, Hk, page, Dr) as codes, and the scales: powers of two, so that every code's
    value is exact in all types."""
    top = x.abs().amax((2, 3))
    scale = torch.exp2(torch.ceil(torch.log2(top / MOST)))
    return (x / scale[:, :, None, None]).to(CODE), scale


def prepare(case, seed):
    g = torch.Generator("cuda").manual_seed(seed)
    t = DTYPES[case["dtype"]]
    s = {"case": case}
    D = case["D"]
    if case["op"] == "turn":
        T, H = case["tokens"], case["heads"]
        # a slice of the product that makes queries, keys and values
        s["x"] = _randn(g, T, H + max(1, H // 4), D).to(t)[:, :H]
        if case["axes"] == 1:
            s["at"] = torch.randint(0, 16384, (T,), generator=g, device="cuda")
        else:
            s["at"] = 2 * torch.rand(T, case["axes"], generator=g, device="cuda") - 1
        s["f"] = _frequencies(case)
        s["gy"] = _randn(g, T, H, D).to(t) if case["mode"] == "train" else None
        if s["gy"] is not None:
            s["x"].requires_grad_(True)
        return s
    B, Hk, page = case["B"], case["heads"], case["page"]
    Hq, Dr = Hk * case["group"], (D + 15) // 16 * 16
    new, lengths = _counts(case)
    M = (max(lengths) + page - 1) // page
    P = B * M + 3
    order = torch.randperm(B, generator=g, device="cuda")
    new = torch.tensor(new, device="cuda")[order]
    s["lengths"] = torch.tensor(lengths, device="cuda")[order]
    s["offsets"] = torch.nn.functional.pad(new.cumsum(0), (1, 0))
    s["longest_new"] = max(_counts(case)[0])
    # pages anywhere in the pool, none behind a sequence's last
    table = torch.randperm(P, generator=g, device="cuda")[:B * M].view(B, M)
    used = torch.arange(M, device="cuda") * page < s["lengths"][:, None]
    s["table"] = torch.where(used, table, -1).int()
    # levels of their own for pages, and for the keys' values; the places past a sequence's
    # last token hold what an earlier one left there
    level = torch.exp(0.5 * _randn(g, P, Hk, 1, 1))
    spread = torch.exp(0.5 * _randn(g, 1, Hk, 1, Dr)) * (torch.arange(Dr, device="cuda") < D)
    codes, s["key_scales"] = _pages(g, _randn(g, P, Hk, page, Dr) * level * spread)
    s["keys"] = codes.view(torch.uint8).view(P, Hk, page // 32, 32, Dr // 16, 16).transpose(
        3, 4).contiguous().view(CODE)
    codes, s["value_scales"] = _pages(g, _randn(g, P, Hk, page, Dr) * level)
    s["values"] = codes.view(torch.uint8).view(P, Hk, page // 32, 32, Dr).transpose(
        3, 4).contiguous().view(CODE)
    T = sum(_counts(case)[0])
    if case["op"] == "cached":
        s["q"] = _randn(g, T, Hq, D).to(t)
        return s
    # slices of one projection; each token has a level of its own
    y = (_randn(g, T, Hq + 2 * Hk, D) * torch.exp(0.5 * _randn(g, T, 1, 1))).to(t)
    s["q"], s["k"], s["v"] = y.split([Hq, Hk, Hk], 1)
    s["f"] = _frequencies(case)
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
    if case["op"] == "turn":
        y = tpo.rotary_positions(s["x"], s["at"], s["f"], interleaved=case["interleaved"])
        return y if s["gy"] is None else (y, *torch.autograd.grad(y, (s["x"],), s["gy"]))
    cache = tpo.PagedCache(s["keys"], s["values"], s["key_scales"], s["value_scales"], s["table"],
                           s["lengths"])
    if case["op"] == "cached":
        return tpo.cached_attention(s["q"], cache, s["offsets"], causal=case["causal"])
    q = tpo.cache_append(cache, s["k"], s["v"], s["offsets"], q=s["q"], frequencies=s["f"],
                         interleaved=case["interleaved"])
    return q, s["keys"], s["values"], s["key_scales"], s["value_scales"]


def _turn(x, at, f, interleaved, back=False, wide=torch.float32):
    """x (T, H, D) turned by its places: at (T) or (T, axes)."""
    n = len(f)
    at = at.view(len(x), -1).double()
    angle = at.repeat_interleave(n // at.shape[1], 1) * f
    c, s = angle.cos().to(wide)[:, None], angle.sin().to(wide)[:, None]
    s = -s if back else s
    x = x.to(wide)
    if interleaved:
        a, b = x[..., 0:2 * n:2], x[..., 1:2 * n:2]
        y = torch.stack([a * c - b * s, b * c + a * s], -1).flatten(2)
    else:
        a, b = x[..., :n], x[..., n:2 * n]
        y = torch.cat([a * c - b * s, b * c + a * s], 2)
    return torch.cat([y, x[..., 2 * n:]], 2)


def _exponent(top):
    """The smallest e with top <= 448 2^e, between -40 and 40."""
    m, e = torch.frexp(top)
    e = e - 9 + (m > 0.875)
    return torch.where(top == 0, -40, e).clamp(-40, 40)


def _places(s, case):
    """Of every new token: its sequence, its place there, its page's number and its slot."""
    new = s["offsets"][1:] - s["offsets"][:-1]
    T = s["k"].shape[0]
    b = torch.searchsorted(s["offsets"], torch.arange(T, device="cuda"), right=True) - 1
    at = torch.arange(T, device="cuda") - s["offsets"][b] + (s["lengths"] - new)[b]
    return b, at, s["table"][b, at // case["page"]].long(), at % case["page"]


def _put(x, page, slot, first, kept, codes, scales):
    """x (T, Hk, Dr) into codes (pages, Hk, page, Dr, as bytes): `first` are the pages
    that hold `kept` older tokens already (0: none)."""
    P, Hk = scales.shape
    top = torch.zeros(P, Hk, device="cuda", dtype=x.dtype).scatter_reduce(
        0, page[:, None].expand(-1, Hk), x.abs().amax(2), "amax")
    need = _exponent(top)
    touched = torch.zeros(P, dtype=torch.bool, device="cuda").index_fill(0, page, True)
    held = torch.zeros(P, dtype=torch.bool, device="cuda").scatter(0, first, kept > 0)
    old = torch.where(held[:, None], torch.frexp(scales)[1] - 1, -40)
    e = torch.where(touched[:, None], torch.maximum(need, old), torch.frexp(scales)[1] - 1)
    # older codes at the new scale
    f = torch.exp2((old - e).float())[first][:, :, None, None]
    was = codes[first].view(CODE).float()
    now = (was * f).to(CODE).view(torch.uint8)
    keep = (torch.arange(codes.shape[2], device="cuda") < kept[:, None])[:, None, :, None]
    codes[first] = torch.where(keep, now, codes[first])
    to = torch.exp2(-e.float())[page][:, :, None]
    codes[page, :, slot] = (x * to).to(CODE).view(torch.uint8)
    scales.copy_(torch.exp2(e.float()))


def _plain_append(s, case):
    t, D = s["k"].dtype, case["D"]
    P, Hk, blocks, chunks = s["keys"].shape[:4]
    b, at, page, slot = _places(s, case)
    before = s["lengths"] - (s["offsets"][1:] - s["offsets"][:-1])
    kept = before % case["page"]
    first = s["table"].gather(1, (before // case["page"])[:, None])[:, 0].long()

    # keys in 64 bits: they are rounded to codes, and some are next to a border
    k = _turn(s["k"], at, s["f"], case["interleaved"], wide=torch.float64)
    pad = (0, 16 * chunks - D)
    codes = s["keys"].view(torch.uint8).transpose(3, 4).clone(
        memory_format=torch.contiguous_format).view(P, Hk, 32 * blocks, -1)
    _put(torch.nn.functional.pad(k, pad), page, slot, first, kept, codes, s["key_scales"])
    s["keys"].view(torch.uint8).copy_(codes.view(P, Hk, blocks, 32, chunks, 16).transpose(3, 4))
    codes = s["values"].view(torch.uint8).transpose(3, 4).clone(
        memory_format=torch.contiguous_format).view(P, Hk, 32 * blocks, -1)
    _put(torch.nn.functional.pad(s["v"].float(), pad), page, slot, first, kept, codes,
         s["value_scales"])
    s["values"].view(torch.uint8).copy_(codes.view(P, Hk, blocks, 32, -1).transpose(3, 4))
    q = _turn(s["q"], at, s["f"], case["interleaved"]).to(t)
    return q, s["keys"], s["values"], s["key_scales"], s["value_scales"]


def _rows(s, case):
    """Keys and values (B Hk, longest, D) of the sequences' pages, in float."""
    B, Hk, D, L = case["B"], case["heads"], case["D"], case["longest"]
    table = s["table"].long().clamp(min=0)
    k = s["keys"].view(torch.uint8)[table].view(CODE).float()
    k = k * s["key_scales"][table][..., None, None, None, None]
    k = k.permute(0, 2, 1, 3, 5, 4, 6).reshape(B * Hk, -1, k.shape[4] * 16)
    v = s["values"].view(torch.uint8)[table].view(CODE).float()
    v = v * s["value_scales"][table][..., None, None, None]
    v = v.permute(0, 2, 1, 3, 5, 4).reshape(B * Hk, -1, v.shape[4])
    return k[:, :L, :D].contiguous(), v[:, :L, :D].contiguous()


def _plain_cached(s, case):
    B, Q, Hk, G, D = case["B"], case["queries"], case["heads"], case["group"], case["D"]
    L, lk = case["longest"], s["lengths"]
    k, v = _rows(s, case)
    q = s["q"].float().view(B, Q, Hk, G, D).permute(0, 2, 3, 1, 4).reshape(B * Hk, G * Q, D)
    j = torch.arange(L, device="cuda")
    seen = (j < lk[:, None])[:, None].expand(B, Q, L)
    if case["causal"]:
        seen = seen & (j <= torch.arange(Q, device="cuda")[:, None] + (lk - Q)[:, None, None])
    p = torch.bmm(q, k.transpose(1, 2).contiguous()).mul_(D ** -0.5).view(B, Hk, G, Q, L)
    p = p.masked_fill_(~seen[:, None, None], float("-inf"))
    top = p.amax(-1, keepdim=True)
    p = p.sub_(torch.where(top == float("-inf"), 0, top)).exp_()
    p = p.div_(p.sum(-1, keepdim=True).clamp_(min=1e-30)).view(B * Hk, G * Q, L)
    # places behind a sequence's end hold anything
    v = v * (j < lk[:, None]).repeat_interleave(Hk, 0)[..., None]
    o = torch.bmm(p, v).view(B, Hk, G, Q, D).permute(0, 3, 1, 2, 4)
    return o.reshape(B * Q, Hk * G, D).to(s["q"].dtype)


def run(s):
    case = s["case"]
    if own:
        return _own(s, case)
    with torch.no_grad():
        if case["op"] == "append":
            return _plain_append(s, case)
        if case["op"] == "cached":
            return _plain_cached(s, case)
        y = _turn(s["x"], s["at"], s["f"], case["interleaved"]).to(s["x"].dtype)
        if s["gy"] is None:
            return y
        return y, _turn(s["gy"], s["at"], s["f"], case["interleaved"], True).to(s["x"].dtype)


def work(case):
    z, D = SIZE[case["dtype"]], case["D"]
    if case["op"] == "turn":
        passes = 2 if case["mode"] == "train" else 1
        n = case["tokens"] * case["heads"]
        return {"bytes": passes * 2 * n * D * z + case["tokens"] * 8,
                "flops": passes * n * case["part"] * 3}
    new, lengths = _counts(case)
    Hk, Hq = case["heads"], case["heads"] * case["group"]
    if case["op"] == "append":
        T = sum(new)
        return {"bytes": T * D * (2 * Hk * (z + 1) + 2 * Hq * z),
                "flops": T * ((Hk + Hq) * case["part"] * 3 + 4 * Hk * D)}
    # keys that the rows of a sequence see: all, or one more for each row up to the last
    pairs = sum(a * b - (a * (a - 1) // 2 if case["causal"] else 0)
                for a, b in zip(new, lengths))
    return {"bytes": 2 * sum(new) * Hq * D * z + 2 * sum(lengths) * Hk * D,
            "flops": pairs * Hq * D * 4}


def _polar(x, at, f, interleaved):
    """x (T, H, D) in 64 bits as complex numbers times exp(i angle)."""
    n, at = len(f), at.double()
    at = at.view(len(x), -1)
    angle = (at[:, :, None] * f.view(at.shape[1], -1)).flatten(1)
    w = torch.polar(torch.ones_like(angle), angle)[:, None]
    x = x.detach().double()
    head = x[..., :2 * n].unflatten(2, (n, 2) if interleaved else (2, n))
    head = head if interleaved else head.transpose(2, 3)
    y = torch.view_as_real(torch.view_as_complex(head.contiguous()) * w)
    return torch.cat([(y if interleaved else y.transpose(2, 3)).flatten(2), x[..., 2 * n:]], 2)


def _code(x):
    """x in 64 bits rounded to the values that e4m3 has (ties to even), as 64 bits."""
    step = torch.exp2(torch.floor(torch.log2(x.abs().clamp(min=2.0 ** -6))) - 3)
    return torch.round(x / step) * step


def _exact_append(s, case):
    page, D = case["page"], case["D"]
    P, Hk, blocks, chunks = s["keys"].shape[:4]
    offsets, lengths, table = (s[n].tolist() for n in ("offsets", "lengths", "table"))
    at = torch.cat([torch.arange(n - (o1 - o0), n, device="cuda")
                    for o0, o1, n in zip(offsets, offsets[1:], lengths)])
    k = _polar(s["k"], at, s["f"], case["interleaved"])
    # (pages, Hk, page, D) of what the codes stand for
    K = s["keys"].double().permute(0, 1, 2, 4, 3, 5).reshape(P, Hk, page, -1)
    V = s["values"].double().transpose(3, 4).reshape(P, Hk, page, -1)
    for X, x, scales in ((K, k, s["key_scales"]), (V, s["v"].double(), s["value_scales"])):
        for o0, o1, n, row in zip(offsets, offsets[1:], lengths, table):
            p = n - (o1 - o0)
            while p < n:
                a, m = p % page, min(n - p, page - p % page)
                i = row[p // page]
                part = x[o0 + p - n + o1 - o0:][:m].transpose(0, 1)  # (Hk, m, D)
                top = part.abs().amax((1, 2))
                # 2^e with top <= 448 2^e
                e = torch.ceil(torch.log2(top / MOST)).clamp(-40, 40)
                if a:
                    was = scales[i].double().log2()
                    e = torch.maximum(e, was)
                    X[i, :, :a] = _code(X[i, :, :a] * torch.exp2(was - e)[:, None, None])
                X[i, :, a:a + m] = 0
                X[i, :, a:a + m, :D] = _code(part * torch.exp2(-e)[:, None, None])
                scales[i] = torch.exp2(e).float()
                p += m
    K = K.view(P, Hk, blocks, 32, chunks, 16).transpose(3, 4).contiguous()
    V = V.view(P, Hk, blocks, 32, -1).transpose(3, 4).contiguous()
    return (_polar(s["q"], at, s["f"], case["interleaved"]), K, V, s["key_scales"].double(),
            s["value_scales"].double())


def _exact_cached(s, case):
    Q, Hk, G, D, page = (case[n] for n in ("queries", "heads", "group", "D", "page"))
    out = []
    # one sequence after another, each a dense problem of its own
    for b, n in enumerate(s["lengths"].tolist()):
        i = s["table"][b, :(n + page - 1) // page].long()
        k = s["keys"].view(torch.uint8)[i].view(CODE).double()
        k = (k * s["key_scales"].double()[i][..., None, None, None, None]).permute(
            1, 0, 2, 4, 3, 5).reshape(Hk, -1, k.shape[3] * 16)[:, :n, :D]
        v = s["values"].view(torch.uint8)[i].view(CODE).double()
        v = (v * s["value_scales"].double()[i][..., None, None, None]).permute(
            1, 0, 2, 4, 3).reshape(Hk, -1, v.shape[3])[:, :n, :D]
        q = s["q"][b * Q:(b + 1) * Q].double().view(Q, Hk, G, D).permute(1, 2, 0, 3)
        a = torch.matmul(q.reshape(Hk, G * Q, D), k.transpose(1, 2)).view(Hk, G, Q, n) / D ** 0.5
        if case["causal"]:
            keep = torch.ones(Q, n, dtype=torch.bool, device="cuda").tril(n - Q)
            a = a.masked_fill(~keep, -torch.inf)
        o = torch.matmul(torch.softmax(a, -1).view(Hk, G * Q, n), v)
        out.append(o.view(Hk, G, Q, D).permute(2, 0, 1, 3).reshape(Q, Hk * G, D))
    return torch.cat(out)


def exact(case, seed):
    s = prepare(case, seed)
    with torch.no_grad():
        if case["op"] == "append":
            return _exact_append(s, case)
        if case["op"] == "cached":
            return _exact_cached(s, case)
        y = _polar(s["x"], s["at"], s["f"], case["interleaved"])
        if s["gy"] is None:
            return y
        return y, _polar(s["gy"], s["at"], -s["f"], case["interleaved"])
