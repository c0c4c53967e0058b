"""The transformer operators' definitions in float64 on the CPU, and how far the kernels may be.

A result that is computed in float and rounded once to its type is off by at most the unit
roundoff u of that type, relative to each value, so by u in the 2-norm; float sums add their
own error, a few 2^-24 for these sizes (2e-6 bounds it, conditioning included).  A product of
rounded operands (probabilities, gradients at the projections) adds another u for each operand
that was rounded; `roundings` counts them all.
"""
import torch

U = {torch.float32: 0.0, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
FLOAT = 2e-6


def near(got, want, roundings=1, floats=FLOAT):
    """got of the GPU against want in float64: relative 2-norm, and every value within eight
    times that of the largest."""
    assert got.shape == want.shape
    got = got.detach()
    tol = roundings * U[got.dtype] + floats
    got = got.cpu().double()
    assert torch.isfinite(got).all()
    if want.numel() == 0:
        return
    err = got - want
    # values under the type's normal range have an absolute error instead
    floor = 1e-7 * want.numel() ** 0.5
    assert err.norm() <= tol * want.norm() + floor, (err.norm() / want.norm()).item()
    assert err.abs().max() <= 8 * tol * want.abs().max() + 1e-6, err.abs().max().item()


def layer_norm(x, w, b, eps):
    x = x.double()
    m = x.mean(-1, keepdim=True)
    y = (x - m) / (((x - m) ** 2).mean(-1, keepdim=True) + eps).sqrt()
    if w is not None:
        y = y * w.double()
    return y if b is None else y + b.double()


def sequences(offsets, lengths, T):
    out = []
    for b in range(len(offsets) - 1):
        n = offsets[b + 1] - offsets[b]
        out.append((offsets[b], n if lengths is None else max(0, min(n, lengths[b]))))
    return out


def attention(q, k, v, oq, ok, lq, lk, causal, scale):
    """The output; a row without keys is 0.  Rows that are not in use take no part."""
    G = q.shape[1] // k.shape[1]
    out = torch.zeros(q.shape, dtype=torch.float64)
    for (q0, nq), (k0, nk) in zip(sequences(oq, lq, q.shape[0]), sequences(ok, lk, k.shape[0])):
        if nq == 0 or nk == 0:
            continue
        a = q[q0:q0 + nq].double().transpose(0, 1)
        c = k[k0:k0 + nk].double().repeat_interleave(G, 1).transpose(0, 1)
        e = v[k0:k0 + nk].double().repeat_interleave(G, 1).transpose(0, 1)
        s = a @ c.transpose(1, 2) * scale
        if causal:
            i, j = torch.arange(nq)[:, None], torch.arange(nk)
            s = s.masked_fill(j > i + nk - nq, float("-inf"))
        seen = s.isfinite().any(-1, keepdim=True)
        p = torch.softmax(s.masked_fill(~seen, 0.0), -1) * seen
        out = out.index_put((torch.arange(q0, q0 + nq),), (p @ e).transpose(0, 1))
    return out


def act(g, name):
    if name == "silu":
        return g * torch.sigmoid(g)
    if name == "gelu":
        return g * 0.5 * (1 + torch.erf(g / 2 ** 0.5))
    return torch.relu(g) if name == "relu" else torch.sigmoid(g)


def gated(x, wg, wu, name):
    x = x.double()
    return act(x @ wg.double().t(), name) * (x @ wu.double().t())


def grads(f, inputs, grad):
    """f of the inputs in float64, and the gradients in them by its own differentiation."""
    leaves = [t.detach().double().requires_grad_(True) for t in inputs]
    y = f(*leaves)
    return y.detach(), torch.autograd.grad(y, leaves, grad.double(), allow_unused=True)


def slope(f, inputs, directions, step):
    """Central difference of the scalar f (float64 in, float64 out) along the directions."""
    up = f(*[t + step * d for t, d in zip(inputs, directions)])
    down = f(*[t - step * d for t, d in zip(inputs, directions)])
    return (up - down) / (2 * step)
