"""Rotary positions and the 8-bit cache in float64 on the CPU, from their definitions.

Codes: every value is rounded once, so a cache has to hold exactly what `append` here computes.
"""
import math

import torch


def turn(x, at, f, interleaved=False, amplitude=1.0, back=False):
    """x (T, H, D) turned by its places at (T) or (T, A)."""
    x, n = x.double(), len(f)
    at = at.double().reshape(len(x), 1 if at.dim() == 1 else at.shape[1])
    angle = torch.stack([at[:, j * at.shape[1] // n] * f[j] for j in range(n)], 1) if n else \
        torch.zeros(len(x), 0, dtype=torch.float64)
    c, s = amplitude * angle.cos()[:, None], amplitude * angle.sin()[:, None]
    if back:
        s = -s
    y = x.clone()
    i = torch.arange(n)
    a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + n)
    y[..., a] = x[..., a] * c - x[..., b] * s
    y[..., b] = x[..., b] * c + x[..., a] * s
    return y


def to_code(x):
    """float64 rounded to what e4m3 has, ties to even; beyond 448: 448; not finite: NaN."""
    m, e = torch.frexp(x.abs().clamp(min=2.0 ** -6))
    step = torch.exp2((e - 4).double())  # 2^(floor(log2) - 3)
    y = (torch.round(x / step) * step).clamp(-448, 448)
    return torch.where(torch.isfinite(x), y, math.nan)


def exponent(top):
    """The smallest e with top <= 448 2^e, between -40 and 40."""
    e = -40
    while e < 40 and top > 448 * 2.0 ** e:
        e += 1
    return e


class Cache:
    """A PagedCache's tensors taken apart: codes (pages, Hk, page, Dr) and scales in float64."""

    def __init__(self, cache):
        self.P, self.Hk, blocks = cache.keys.shape[:3]
        self.page = 32 * blocks
        self.k, self.v = (t.cpu().float().double().transpose(3, 4).reshape(
            self.P, self.Hk, self.page, -1) for t in (cache.keys, cache.values))
        self.ks, self.vs = cache.key_scales.cpu().double(), cache.value_scales.cpu().double()
        self.table, self.lengths = cache.table.cpu(), cache.lengths.cpu()
        self.M = self.table.shape[1]

    def length(self, b):
        return max(0, min(int(self.lengths[b]), self.M * self.page))

    def spans(self, offsets, lengths, T):
        """(sequence, first row, rows in use) with bounds kept inside the rows."""
        o = [max(0, min(T, int(v))) for v in offsets]
        for b in range(len(o) - 1):
            room = max(0, o[b + 1] - o[b])
            yield b, o[b], room if lengths is None else max(0, min(room, int(lengths[b])))

    def append(self, k, v, offsets, lengths=None, q=None, f=None, at=None, interleaved=False,
               amplitude=1.0):
        T, D = k.shape[0], k.shape[2]
        place = torch.zeros(T, dtype=torch.int64)
        live = torch.zeros(T, dtype=torch.bool)
        for b, r0, n in self.spans(offsets, lengths, T):
            for i in range(n):
                place[r0 + i] = self.length(b) - n + i
                live[r0 + i] = place[r0 + i] >= 0
        f = torch.zeros(0, dtype=torch.float64) if f is None else f
        at = place if at is None else at
        k = turn(k, at, f, interleaved, amplitude)
        v = v.double()
        pages = {}
        for b, r0, n in self.spans(offsets, lengths, T):
            for t in range(r0, r0 + n):
                if live[t]:
                    p = int(self.table[b, place[t] // self.page])
                    if 0 <= p < self.P:
                        pages.setdefault(p, []).append((int(place[t]) % self.page, t))
        for p, tokens in pages.items():
            first = min(s for s, _ in tokens)
            rows = [t for _, t in tokens]
            for h in range(self.Hk):
                for X, x, scales in ((self.k, k, self.ks), (self.v, v, self.vs)):
                    y = x[rows, h]
                    y_ok = torch.where(torch.isfinite(y), y, 0)
                    e = exponent(float(y_ok.abs().max()))
                    if first > 0:
                        e = max(e, int(math.log2(scales[p, h])))
                        X[p, h, :first] = to_code(X[p, h, :first] * scales[p, h] / 2.0 ** e)
                    scales[p, h] = 2.0 ** e
                    for (slot, _), row in zip(tokens, y):
                        X[p, h, slot] = 0
                        X[p, h, slot, :D] = to_code(row / 2.0 ** e)
        if q is None:
            return None
        return turn(q, at, f, interleaved, amplitude) * live[:, None, None]

    def rows(self, b, D):
        """Keys and values (Hk, length, D) of sequence b, and which of them are there."""
        n, k, v, there = self.length(b), [], [], []
        for j in range(n):
            p = int(self.table[b, j // self.page])
            there.append(0 <= p < self.P)
            p, s = p if there[-1] else 0, j % self.page
            k.append(self.k[p, :, s, :D] * self.ks[p, :, None])
            v.append(self.v[p, :, s, :D] * self.vs[p, :, None])
        empty = torch.zeros(self.Hk, 0, D, dtype=torch.float64)
        return (torch.stack(k, 1) if n else empty, torch.stack(v, 1) if n else empty,
                torch.tensor(there, dtype=torch.bool))

    def attention(self, q, offsets, lengths=None, causal=True, scale=None):
        T, Hq, D = q.shape
        scale = D ** -0.5 if scale is None else scale
        out = torch.zeros(T, Hq, D, dtype=torch.float64)
        G, kept = Hq // self.Hk, {}
        for b, r0, n in self.spans(offsets, lengths, T):
            if n == 0:
                continue
            key = (tuple(self.table[b].tolist()), self.length(b))
            if key not in kept:
                kept[key] = self.rows(b, D)
            k, v, there = kept[key]
            L = k.shape[1]
            for i in range(n):
                m = max(0, min(L, i + L - n + 1)) if causal else L
                at = torch.arange(m)[there[:m]]
                if len(at) == 0:
                    continue
                a = q[r0 + i].double().view(self.Hk, G, D) @ k[:, at].transpose(1, 2) * scale
                out[r0 + i] = (torch.softmax(a, -1) @ v[:, at]).reshape(Hq, D)
        return out


def pool(P, Hk, page, D, seed, spread=0.5):
    """Tensors of a cache whose pages hold normal values at levels of their own: keys, values and
    scales, on the CPU."""
    g = torch.Generator().manual_seed(seed)
    Dr = (D + 15) // 16 * 16
    out = []
    for _ in range(2):
        x = torch.randn(P, Hk, page, Dr, generator=g) * (torch.arange(Dr) < D)
        x = x * torch.exp(spread * torch.randn(P, Hk, 1, 1, generator=g))
        scale = torch.exp2(torch.ceil(torch.log2(x.abs().amax((2, 3)) / 448)))
        out += [(x / scale[..., None, None]).to(torch.float8_e4m3fn), scale]
    kc, ks, vc, vs = out
    k = kc.view(torch.uint8).view(P, Hk, page // 32, 32, Dr // 16, 16).transpose(3, 4)
    v = vc.view(torch.uint8).view(P, Hk, page // 32, 32, Dr).transpose(3, 4)
    return (k.clone(memory_format=torch.contiguous_format).view(torch.float8_e4m3fn),
            v.clone(memory_format=torch.contiguous_format).view(torch.float8_e4m3fn), ks, vs)


def paged(tpo, dev, lengths, Hk, D, page=64, seed=0, spare=2, extra=0, spread=0.5):
    """A PagedCache on the GPU whose sequences' pages lie anywhere in its pool; `extra`: entries
    of the table behind the longest sequence."""
    g = torch.Generator().manual_seed(seed + 1000)
    M = max([1] + [-(-n // page) for n in lengths]) + extra
    used = [-(-n // page) for n in lengths]
    P = sum(used) + spare
    order = torch.randperm(P, generator=g)
    table = torch.full((len(lengths), M), -1, dtype=torch.int32)
    at = 0
    for b, n in enumerate(used):
        table[b, :n] = order[at:at + n].int()
        at += n
    return tpo.PagedCache(*(t.to(dev) for t in pool(P, Hk, page, D, seed, spread)),
                          table.to(dev), torch.tensor(lengths, dtype=torch.int64, device=dev))
