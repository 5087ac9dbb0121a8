"""The selective scan, the short convolution and the add and layer norm in 64 bits, forward and backward written out, and the same of their magnitudes.

Magnitudes (`mag`): every product and sum with absolute values in it, the decays as they are.  Each rounding of a kernel is at most U = 2^-24 of a magnitude on the way to an output, so
that n roundings on that way stay below n U of the output's magnitude: the bounds of the tests."""
import torch

U = 2.0 ** -24
HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8}


def f64(t):
    return t.detach().double().cpu() if t is not None else None


def silu(v):
    return v * torch.sigmoid(v)


def dsilu(v):
    s = torch.sigmoid(v)
    return s * (1 + v * (1 - s))


def scan(x, delta, A, B, C, D=None, z=None, delta_bias=None, delta_softplus=False, initial_state=None, reverse=False, d_o=None, d_final=None, mag=False):
    """{name: value}; with d_o the gradients too."""
    m = torch.abs if mag else (lambda t: t)
    walk = lambda t: None if t is None else (f64(t).flip(1) if reverse else f64(t))  # noqa: E731
    back = lambda t: t.flip(1) if reverse else t  # noqa: E731
    x, raw, Bc, Cc, z = (walk(t) for t in (x, delta, B, C, z))
    A, D, bias, h = f64(A), f64(D), f64(delta_bias), f64(initial_state)
    batch, L, width = x.shape
    shared = Bc
    N, G = Bc.shape[-1], Bc.shape[2] if Bc.dim() == 4 else 1
    spread = lambda t: t.reshape(batch, L, G, 1, N).expand(-1, -1, -1, width // G, -1).reshape(batch, L, width, N)  # noqa: E731
    gather = lambda t: t.reshape(batch, L, G, width // G, N).sum(3).reshape(shared.shape)  # noqa: E731
    raw = raw + bias if bias is not None else raw
    s = torch.nn.functional.softplus(raw, threshold=1e9) if delta_softplus else raw
    ds = torch.sigmoid(raw) if delta_softplus else torch.ones_like(raw)
    a = torch.exp(s.unsqueeze(-1) * A)
    x, Bc, Cc = m(x), m(spread(Bc)), m(spread(Cc))
    h = m(h) if h is not None else torch.zeros(batch, width, N, dtype=torch.float64)
    u = s * x
    H, P = torch.empty(batch, L, width, N, dtype=torch.float64), torch.empty(batch, L, width, N, dtype=torch.float64)
    for t in range(L):
        P[:, t] = a[:, t] * h
        h = P[:, t] + u[:, t].unsqueeze(-1) * Bc[:, t]
        H[:, t] = h
    skip = m(D) if D is not None else torch.zeros(width, dtype=torch.float64)
    y = (H * Cc).sum(-1) + skip * x
    out = {"o": back(y * m(silu(z)) if z is not None else y), "final": h}
    if d_o is None:
        return out
    dy = m(walk(d_o))
    if z is not None:
        out["dz"] = back(dy * y * m(dsilu(z)))
        dy = dy * m(silu(z))
    g = m(f64(d_final)) if d_final is not None else torch.zeros_like(h)
    dh = torch.empty_like(H)
    for t in range(L - 1, -1, -1):
        g = g + dy[:, t].unsqueeze(-1) * Cc[:, t]
        dh[:, t] = g
        g = a[:, t] * g
    out["dinitial"] = g
    out["dC"], out["dB"] = back(gather(H * dy.unsqueeze(-1))), back(gather(dh * u.unsqueeze(-1)))
    du, e = (dh * Bc).sum(-1), dh * P
    out["dx"] = back(s * du + skip * dy)
    out["dA"] = (e * s.unsqueeze(-1)).sum((0, 1))
    step = ((e * m(A)).sum(-1) + x * du) * ds
    out["ddelta"] = back(step)
    out["dD"], out["dbias"] = (dy * x).sum((0, 1)), step.sum((0, 1))
    return out


def conv(x, weight, bias=None, act=False, initial_state=None, reverse=False, dy=None, d_final=None, mag=False):
    m = torch.abs if mag else (lambda t: t)
    walk = lambda t: f64(t).flip(1) if reverse else f64(t)  # noqa: E731
    back = lambda t: t.flip(1) if reverse else t  # noqa: E731
    w = f64(weight)
    W, (batch, L, width) = w.shape[1], x.shape
    first = f64(initial_state) if initial_state is not None else torch.zeros(batch, W - 1, width, dtype=torch.float64)
    rows = torch.cat([first, walk(x)], 1)
    pre = sum(w[:, k] * rows[:, k:k + L] for k in range(W)) + (f64(bias) if bias is not None else 0)
    size = sum(w[:, k].abs() * rows[:, k:k + L].abs() for k in range(W)) + (f64(bias).abs() if bias is not None else 0)
    # (a sum's error passes the activation with a slope of at most 1.1; the derivative's own slope is at most a half)
    y = back((1.1 * size if mag else silu(pre)) if act else (size if mag else pre))
    out = {"y": y, "final": rows[:, L:]}
    if dy is None:
        return out
    d = m(walk(dy))
    if act:
        d = d * (1.1 + 0.5 * size if mag else dsilu(pre))
    grads = torch.zeros_like(rows)
    for k in range(W):
        grads[:, k:k + L] += m(w[:, k]) * d
    if d_final is not None:
        grads[:, L:] += m(f64(d_final))
    return out | {"dx": back(grads[:, W - 1:]), "dinitial": grads[:, :W - 1], "dweight": torch.stack([(d * m(rows[:, k:k + L])).sum((0, 1)) for k in range(W)], 1), "dbias": d.sum((0, 1))}


def norm(x, weight, bias=None, eps=1e-5, residual=None, dy=None, d_sum=None):
    """{name: (value, magnitude)}"""
    total = f64(x)
    if residual is not None:
        total = (x.detach().cpu().float() + residual.detach().cpu().float()).to(residual.dtype).double()  # (the sum as it is stored, which is what is normalised)
    w = f64(weight)
    b = f64(bias) if bias is not None else torch.zeros_like(w)
    mean, var = total.mean(-1, keepdim=True), total.var(-1, correction=0, keepdim=True)
    rstd = 1 / (var + eps).sqrt()
    hat = (total - mean) * rstd
    # a value's own roundings, those of the mean (of all magnitudes of the row), and the reciprocal root's
    size = rstd * (total.abs() + total.abs().mean(-1, keepdim=True)) + hat.abs()
    out = {"y": (hat * w + b, size * w.abs() + b.abs()), "sum": (total, total.abs())}
    if dy is None:
        return out
    dy = f64(dy)
    axes = tuple(range(dy.dim() - 1))
    out["dweight"], out["dbias"] = ((dy * hat).sum(axes), (dy.abs() * size).sum(axes)), (dy.sum(axes), dy.abs().sum(axes))
    g = dy * w
    d = rstd * (g - g.mean(-1, keepdim=True) - hat * (g * hat).mean(-1, keepdim=True))
    dm = rstd * (g.abs() + g.abs().mean(-1, keepdim=True) + 2 * size * (g.abs() * size).mean(-1, keepdim=True))
    if d_sum is not None:
        d, dm = d + f64(d_sum), dm + f64(d_sum).abs()
    return out | {"dx": (d, dm), "dresidual": (d, dm)}


def close(got, want, size, roundings, what):
    """Every element within `roundings` of its magnitude and half a step of its type."""
    got = got.detach()
    assert got.shape == want.shape, f"{what}: {tuple(got.shape)} for {tuple(want.shape)}"
    half = HALF[got.dtype]
    off = (got.double().cpu() - want).abs()
    most = roundings * U * size * (1 + half) + half * want.abs() + 2.0 ** -126
    bad = ~(off <= most)
    assert not bool(bad.any()), f"{what}: {int(bad.sum())} of {bad.numel()} off, by {float(off[bad].max()):.3e} where {float(most[bad][off[bad].argmax()]):.3e} is the most"
