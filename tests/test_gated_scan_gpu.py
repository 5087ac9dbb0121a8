"""The gated scan against its recurrence in 64 bits, token by token, with bounds on every element.

Bounds.  u = 2^-24.  A factor e^g is off by at most 3 u of itself and |g| u more (the product with log2 e, the hardware's exponential to one unit), and every step on an input's
way to an output rounds once: with k = 5 the recurrence E_t = a_t E_{t-1} + k u (1 + |g_t|) H_t on the magnitudes H_t = a_t H_{t-1} + |x_t| holds what the steps add.  Runs of tokens are
folded in a tree: eight tokens, up to two steps in a wave, up to 16 waves, and the same again over the chunks of a long sequence, at most 60 more roundings on
one way: 60 u H_t.  The output's rounding is half a step of its type."""
import math

import pytest
import torch

import vig_amd
from vig_amd import _ext

from .util import announce

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
F32, BF16 = torch.float32, torch.bfloat16
HALF = {F32: 2.0 ** -24, BF16: 2.0 ** -8}


def _walk(a, x, h0, reverse=False, k=None):
    """(h, H, E) of every token in 64 bits: the state, its magnitude and the bound on its error; k None: of exact factors."""
    B, L, D = x.shape
    h, H, E = (torch.empty(B, L, D, dtype=torch.float64) for _ in range(3))
    s = torch.zeros(B, D, dtype=torch.float64) if h0 is None else h0.double().cpu()
    m, e = s.abs(), torch.zeros_like(s)
    for t in range(L - 1, -1, -1) if reverse else range(L):
        s, m = a[:, t] * s + x[:, t], a[:, t] * m + x[:, t].abs()
        e = a[:, t] * e + k[:, t] * m
        h[:, t], H[:, t], E[:, t] = s, m, e
    return h, H, E + 60 * U * H


def _shift(first, t):
    return torch.cat([(torch.zeros_like(t[:, :1]) if first is None else first[:, None]), t[:, :-1]], 1)


def reference(x, g, h0=None, both=False, d_o=None, d_final=None):
    """Outputs and gradients with their bounds, without the outputs' rounding: {name: (value, bound)}."""
    x, g = x.detach().double().cpu(), g.detach().double().cpu()
    h0 = h0.detach().double().cpu() if h0 is not None else None
    B, s = x.shape[0], 0.5 if both else 1.0
    halves = [g[:B], g[B:]] if both else [g]
    a = [t.exp() for t in halves]
    k = [5 * U * (1 + t.abs().nan_to_num(0, 0, 0)) for t in halves]
    walks = [_walk(a[w], x, h0 if w == 0 else None, w == 1, k[w]) for w in range(len(a))]
    out = {"o": (s * sum(w[0] for w in walks), s * sum(w[2] for w in walks) + 2 * U * s * sum(w[1] for w in walks))}
    out["final"] = (walks[0][0][:, -1], walks[0][2][:, -1])
    if d_o is None:
        return out
    do = s * d_o.detach().double().cpu()
    dx, dxb, dg, dgb = 0, 0, [], []
    for w in range(len(a)):
        back = w == 0  # the gradient walks against its direction
        end = do.clone()
        if back and d_final is not None:
            end[:, -1] += d_final.double().cpu()
        zero = torch.zeros_like(a[w][:, :1])
        af = torch.cat([a[w][:, 1:], zero], 1) if back else torch.cat([zero, a[w][:, :-1]], 1)
        kf = torch.cat([k[w][:, 1:], k[w][:, -1:]], 1) if back else torch.cat([k[w][:, :1], k[w][:, :-1]], 1)
        d, D, E = _walk(af, end, None, back, kf)
        h, H, Eh = walks[w]
        if back:
            prev, P, Ep = (_shift(i, t) for i, t in ((h0, h), (h0.abs() if h0 is not None else None, H), (None, Eh)))
        else:
            prev, P, Ep = (_shift(None, t.flip(1)).flip(1) for t in (h, H, Eh))
        dx, dxb = dx + d, dxb + E + 2 * U * D
        dg.append(d * a[w] * prev)
        dgb.append(a[w] * (E * P + D * Ep) + (k[w] + 4 * U) * D * a[w] * P)
        if back:
            out["dh0"] = (d[:, 0] * a[w][:, 0], E[:, 0] * a[w][:, 0] + (k[w][:, 0] + 2 * U) * D[:, 0])
    return out | {"dx": (dx, dxb), "dg": (torch.cat(dg), torch.cat(dgb))}


def close(got, want, what):
    value, bound = want
    got, half = got.detach(), HALF[got.dtype]
    off = (got.double().cpu() - value).abs()
    limit = bound + half * (value.abs() + bound) + 1e-37
    assert bool((off <= limit).all()), f"{what}: {float((off / limit).max()):.3g} of the bound, {float(off.max()):.3g} off"


def draw(B, L, D, x_type, g_type, both, seed, strong=False, state=False):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    r = lambda *s: torch.randn(*s, device="cuda", generator=gen)  # noqa: E731
    g = torch.nn.functional.logsigmoid(r(2 * B if both else B, L, D)) / (1 if strong else 16)
    return r(B, L, D).to(x_type), g.to(g_type), r(B, D) if state else None, r(B, L, D).to(x_type), r(B, D) if state else None


SIZES = [(1, 1, 1), (2, 1, 64), (1, 2, 3), (1, 7, 5), (3, 8, 64), (2, 9, 36), (1, 31, 200), (2, 32, 4), (1, 33, 68), (3, 127, 66), (2, 128, 65), (2, 129, 7), (2, 196, 192),
         (1, 197, 100), (1, 511, 64), (1, 512, 12), (1, 513, 64), (2, 700, 132), (1, 1025, 8), (1, 1300, 3)]
TYPES = [(BF16, BF16), (F32, F32), (BF16, F32), (F32, BF16)]


@pytest.mark.parametrize("both", [False, True])
@pytest.mark.parametrize("types", TYPES)
@pytest.mark.parametrize("B,L,D", SIZES)
def test_against_the_recurrence(B, L, D, types, both):
    announce(f"gated scan B{B} L{L} D{D} {types} both={both}")
    x, g, h0, do, dh = draw(B, L, D, *types, both, B + L + D, strong=L % 2 == 0, state=not both)
    for t in (x, g, h0):
        if t is not None:
            t.requires_grad_()
    if both:
        o, h = vig_amd.bid_gated_scan(x, g)
        assert h is None
        dx, dg = torch.autograd.grad(o, (x, g), do)
    else:
        o, h = vig_amd.gated_scan(x, g, h0, True)
        dx, dg, dh0 = torch.autograd.grad((o, h), (x, g, h0), (do, dh))
    assert o.dtype == x.dtype and dx.dtype == x.dtype and dg.dtype == g.dtype
    want = reference(x, g, h0, both, do, dh)
    close(o, want["o"], "o"), close(dx, want["dx"], "dx"), close(dg, want["dg"], "dg")
    if not both:
        assert h.dtype == F32
        close(h, want["final"], "final"), close(dh0, want["dh0"], "dh0")


@pytest.mark.parametrize("both", [False, True])
@pytest.mark.parametrize("B,L,D", [(300, 1, 64), (260, 8, 64), (300, 15, 64), (257, 16, 64), (300, 17, 64), (130, 40, 120), (256, 196, 64), (64, 197, 256), (258, 255, 64), (256, 256, 64)])
def test_many_short_sequences(B, L, D, both):
    """bf16 rows that move 16 bytes a lane, from 256 workgroups on."""
    announce(f"gated scan, many: B{B} L{L} D{D} both={both}")
    x, g, h0, do, dh = draw(B, L, D, BF16, BF16, both, B + L, strong=L % 2 == 0, state=not both)
    wide = torch.randn(B, L + 2, D + 16, device="cuda").bfloat16()
    rows = wide[:, 1:L + 1, 8:D + 8]  # (the same rows in the columns of wider ones, on 16-byte boundaries)
    rows.copy_(x)
    for rows in (x, rows):
        given = [t.detach().requires_grad_() for t in ((rows, g) if both else (rows, g, h0))]
        o, h = vig_amd.bid_gated_scan(*given) if both else vig_amd.gated_scan(*given, True)
        got = torch.autograd.grad((o,) if both else (o, h), given, (do,) if both else (do, dh))
        want = reference(x, g, h0, both, do, dh)
        close(o, want["o"], "o")
        for name, t in zip(("dx", "dg", "dh0"), got):
            close(t, want[name], name)
        if not both:
            close(h, want["final"], "final")


@pytest.mark.parametrize("both", [False, True])
@pytest.mark.parametrize("types", TYPES)
@pytest.mark.parametrize("B,L,D", [(1, 1024, 36), (2, 1000, 7), (1, 1023, 66)])
def test_one_workgroup_up_to_1024_tokens(B, L, D, types, both):
    test_against_the_recurrence(B, L, D, types, both)


def test_many_chunks_of_many_channels():
    """Gradients of long causal sequences in so many workgroups that a thread takes 16 tokens."""
    B, L, D = 1, 1100, 16384
    announce(f"gated scan B{B} L{L} D{D}")
    x, g, h0, do, dh = draw(B, L, D, BF16, BF16, False, 5, state=True)
    given = [t.requires_grad_() for t in (x, g, h0)]
    o, h = vig_amd.gated_scan(*given, True)
    got = torch.autograd.grad((o, h), given, (do, dh))
    some = slice(8000, 8100)
    want = reference(x[..., some], g[..., some], h0[:, some], False, do[..., some], dh[:, some])
    close(o[..., some], want["o"], "o"), close(h[:, some], want["final"], "final"), close(got[2][:, some], want["dh0"], "dh0")
    close(got[0][..., some], want["dx"], "dx"), close(got[1][..., some], want["dg"], "dg")


@pytest.mark.parametrize("both", [False, True])
@pytest.mark.parametrize("B,L,D", [(1, 4100, 68), (2, 9001, 5), (1, 70000, 4)])
def test_many_chunks(B, L, D, both):
    announce(f"gated scan, long: B{B} L{L} D{D} both={both}")
    x, g, h0, do, dh = draw(B, L, D, F32, F32, both, L, state=not both)
    for t in (x, g, h0):
        if t is not None:
            t.requires_grad_()
    o, h = vig_amd.bid_gated_scan(x, g) if both else vig_amd.gated_scan(x, g, h0, True)
    got = torch.autograd.grad((o,) if both else (o, h), (x, g) if both else (x, g, h0), (do,) if both else (do, dh))
    want = reference(x, g, h0, both, do, dh)
    close(o, want["o"], "o")
    for name, t in zip(("dx", "dg", "dh0"), got):
        close(t, want[name], name)
    if not both:
        close(h, want["final"], "final")


@pytest.mark.parametrize("both", [False, True])
@pytest.mark.parametrize("where", ["columns", "odd columns", "off the boundary", "tokens of more", "swapped axes", "every second channel", "repeated rows"])
def test_rows_as_they_lie(where, both):
    announce(f"gated scan of {where} both={both}")
    B, L, D = 3, 150, 68
    gen = torch.Generator(device="cuda").manual_seed(7)
    r = lambda *s: torch.randn(*s, device="cuda", generator=gen).bfloat16()  # noqa: E731

    def made(b, gates):
        if where == "columns":
            t = r(b, L, 3 * D)[..., D:2 * D]
        elif where == "odd columns":
            t = r(b, L, 2 * D + 1)[..., 1:D + 1]
        elif where == "off the boundary":
            t = r(b * L * D + 3)[3:].view(b, L, D)
        elif where == "tokens of more":
            t = r(b, L + 9, D)[:, 4:4 + L]
        elif where == "swapped axes":
            t = r(L, b, D).transpose(0, 1)
        elif where == "every second channel":
            t = r(b, L, 2 * D)[..., ::2]
        else:
            t = r(1, L, D).expand(b, L, D)
        if not gates:
            return t
        with torch.no_grad():
            base = t if where != "repeated rows" else t[:1]
            base.copy_(torch.nn.functional.logsigmoid(base.float()) / 4)
        return t

    x, g = made(B, False).requires_grad_(), made(2 * B if both else B, True).requires_grad_()
    before = (x.detach().clone(), g.detach().clone())
    o, _ = (vig_amd.bid_gated_scan if both else vig_amd.gated_scan)(x, g)
    do = r(B, L, D)
    dx, dg = torch.autograd.grad(o, (x, g), do)
    want = reference(x, g, None, both, do)
    close(o, want["o"], "o"), close(dx, want["dx"], "dx"), close(dg, want["dg"], "dg")
    assert torch.equal(x, before[0]) and torch.equal(g, before[1])


def test_gradients_of_shared_inputs_and_of_one_output():
    """Rows shared by the batch get the sum of its gradients; an output that nothing hangs on has none."""
    x, g, h0, do, dh = draw(3, 50, 24, F32, F32, False, 3, state=True)
    one, gate = x[:1].clone().requires_grad_(), g[:, :1].clone().requires_grad_()
    o, _ = vig_amd.gated_scan(one.expand(3, 50, 24), gate.expand(3, 50, 24))
    d1, d2 = torch.autograd.grad(o, (one, gate), do)
    want = reference(one.expand(3, 50, 24), gate.expand(3, 50, 24), None, False, do)
    close(d1, tuple(t.sum(0, keepdim=True) for t in want["dx"]), "shared rows")
    value, bound = (t.sum(1, keepdim=True) for t in want["dg"])
    close(d2, (value, bound + 50 * U * want["dg"][0].abs().sum(1, keepdim=True)), "shared gates")
    x.requires_grad_(), h0.requires_grad_()
    for outputs in ("o", "final"):
        o, h = vig_amd.gated_scan(x, g, h0, True)
        got = torch.autograd.grad(o, (x, h0), do) if outputs == "o" else torch.autograd.grad(h, (x, h0), dh)
        want = reference(x, g, h0, False, do if outputs == "o" else torch.zeros_like(do), dh if outputs == "final" else None)
        close(got[0], want["dx"], outputs), close(got[1], want["dh0"], outputs)
    o, _ = vig_amd.gated_scan(x.detach(), g, h0)  # the state alone
    (got,) = torch.autograd.grad(o, h0, do)
    close(got, reference(x, g, h0, False, do)["dh0"], "state alone")


def test_gradients_against_differences():
    x, g, h0, do, dh = draw(2, 40, 6, F32, F32, False, 11, state=True)
    for t in (x, g, h0):
        t.requires_grad_()
    o, h = vig_amd.gated_scan(x, g, h0, True)
    grads = torch.autograd.grad((o, h), (x, g, h0), (do, dh))

    def loss(*t):  # in 64 bits: the recurrence alone is differentiated
        r = reference(*t)
        return float((r["o"][0] * do.double().cpu()).sum() + (r["final"][0] * dh.double().cpu()).sum())

    gen = torch.Generator().manual_seed(1)
    for i, grad in enumerate(grads):
        base = [t.detach().double().cpu() for t in (x, g, h0)]
        way = torch.randn(base[i].shape, generator=gen, dtype=torch.float64)
        step = 1e-5  # (a central difference: error ~ step^2 of third derivatives, and 1e-16 / step of rounding)
        at = [loss(*[t + s * step * way if k == i else t for k, t in enumerate(base)]) for s in (1, -1)]
        slope = float((grad.double().cpu() * way).sum())
        scale = float((grad.double().cpu() * way).abs().sum())
        assert abs((at[0] - at[1]) / (2 * step) - slope) <= 1e-5 * scale


def test_heads_are_sequences():
    x, g, h0, do, _ = draw(6, 40, 32, BF16, BF16, False, 5, state=True)
    heads = lambda t: t.view(2, 3, *t.shape[1:])  # noqa: E731
    o, h = vig_amd.gated_scan(heads(x), heads(g), heads(h0), True)
    o1, h1 = vig_amd.gated_scan(x, g, h0, True)
    assert torch.equal(o.view_as(o1), o1) and torch.equal(h.view_as(h1), h1) and o.shape == (2, 3, 40, 32) and h.shape == (2, 3, 32)
    both = torch.cat([g, g.flip(1)])
    o2, _ = vig_amd.bid_gated_scan(heads(x), both.view(4, 3, 40, 32))
    assert torch.equal(o2.view_as(o1), vig_amd.bid_gated_scan(x, both)[0])


@pytest.mark.parametrize("L", [90, 1500])
def test_packed_and_padded_sequences(L):
    """A gate of -inf starts a sequence anew, and a token of zeros is none."""
    announce(f"packed and padded sequences L{L}")
    x, g, _, do, _ = draw(2, L, 36, F32, F32, True, L)
    cuts = [0, 1, 30, 31, L // 2, L - 1, L]
    gf, gb = g[:2].clone(), g[2:].clone()
    for a, b in zip(cuts, cuts[1:]):
        gf[:, a], gb[:, b - 1] = -math.inf, -math.inf
    packed = torch.cat([gf, gb]).requires_grad_()
    xp = x.clone().requires_grad_()
    o, _ = vig_amd.bid_gated_scan(xp, packed)
    dx, dg = torch.autograd.grad(o, (xp, packed), do)
    assert bool(torch.isfinite(o).all() and torch.isfinite(dx).all() and torch.isfinite(dg).all())
    assert not bool(dg[:2, cuts[:-1]].any()) and not bool(dg[2:, [c - 1 for c in cuts[1:]]].any())
    for a, b in zip(cuts, cuts[1:]):
        want = reference(x[:, a:b], g[:, a:b], None, True, do[:, a:b])
        close(o[:, a:b], want["o"], f"packed {a}:{b}"), close(dx[:, a:b], want["dx"], f"packed dx {a}:{b}")
    n = L - 17
    xq, gq = x.clone(), g.clone()
    xq[:, n:], gq[:, n:] = 0, 0
    o, _ = vig_amd.bid_gated_scan(xq, gq)
    close(o[:, :n], reference(x[:, :n], g[:, :n], None, True)["o"], "padded")
    o, h = vig_amd.gated_scan(xq, gq[:2], None, True)
    close(h, reference(x[:, :n], g[:2, :n])["final"], "state behind the padding")


def test_values_that_are_not_finite_stay_in_their_channel():
    for L in (100, 1200):
        x, g, _, _, _ = draw(2, L, 20, F32, F32, False, L)
        clean, _ = vig_amd.gated_scan(x, g)
        x[0, 40, 3], x[1, 60, 5], g[1, 10, 7] = math.nan, math.inf, math.nan
        o, _ = vig_amd.gated_scan(x, g)
        bad = ~torch.isfinite(o)
        for b, c, t in ((0, 3, 40), (1, 5, 60), (1, 7, 10)):
            assert bool(bad[b, t:, c].all()) and not bool(bad[b, :t, c].any())
            bad[b, :, c], clean[b, t:, c], o[b, t:, c] = False, 0, 0
        assert not bool(bad.any()) and torch.equal(o, clean)


@pytest.mark.parametrize("cut", [1, 100, 512, 600])
def test_a_sequence_in_two_pieces(cut):
    x, g, h0, _, _ = draw(2, 1100, 36, F32, F32, False, cut, state=True)
    a, h = vig_amd.gated_scan(x[:, :cut], g[:, :cut], h0, True)
    b, h = vig_amd.gated_scan(x[:, cut:], g[:, cut:], h, True)
    want = reference(x, g, h0)
    close(torch.cat([a, b], 1), want["o"], "two pieces"), close(h, want["final"], "final")


@pytest.mark.parametrize("types", TYPES)
@pytest.mark.parametrize("B,D", [(1, 1), (1, 384), (3, 5), (7, 68), (300, 192), (2, 1023)])
def test_step(B, D, types):
    announce(f"step B{B} D{D} {types}")
    x, g, h0, _, _ = draw(B, 6, D, *types, False, B + D, state=True)
    h, got = h0.clone(), []
    version = h._version
    for t in range(6):  # rows of the sequences, six tokens apart
        got.append(vig_amd.gated_scan_step(x[:, t], g[:, t], h))
    assert h._version == version + 6
    want = reference(x, g, h0)
    assert got[0].dtype == x.dtype and got[0].shape == (B, D)
    close(torch.stack(got, 1), want["o"], "o"), close(h, want["final"], "state")


def test_nothing_to_do():
    for B, L, D in ((2, 0, 8), (0, 5, 8), (2, 5, 0)):
        x = torch.zeros(B, L, D, device="cuda", requires_grad=True)
        h0 = torch.randn(B, D, device="cuda")
        o, h = vig_amd.gated_scan(x, torch.zeros_like(x), h0, True)
        assert o.shape == x.shape and torch.equal(h, h0)
        o, _ = vig_amd.bid_gated_scan(x, torch.zeros(2 * B, L, D, device="cuda"))
        assert o.shape == x.shape
        o.sum().backward()
        assert x.grad.shape == x.shape


def test_the_same_bits_whichever_way_the_call_goes(monkeypatch):
    for both, B, L, D in ((False, 2, 700, 36), (True, 3, 196, 65)):
        x, g, h0, do, dh = draw(B, L, D, BF16, F32, both, L, state=not both)
        given = [t.requires_grad_() for t in (x, g, h0) if t is not None]

        def run():
            o, h = vig_amd.bid_gated_scan(x, g) if both else vig_amd.gated_scan(x, g, h0, True)
            return [o] + ([] if both else [h]) + list(torch.autograd.grad((o,) if both else (o, h), given, (do,) if both else (do, dh)))

        first, again = run(), run()
        monkeypatch.setattr(_ext, "calls", lambda: None)
        plain = run()
        step = vig_amd.gated_scan_step(x[:, 0].detach(), g[:B, 0].detach(), torch.zeros(B, D, device="cuda"))
        monkeypatch.undo()
        assert all(torch.equal(a, b) and torch.equal(a, c) for a, b, c in zip(first, again, plain))
        assert torch.equal(step, vig_amd.gated_scan_step(x[:, 0].detach(), g[:B, 0].detach(), torch.zeros(B, D, device="cuda")))


def test_on_another_stream_and_in_graphs():
    """Captured once, replayed with other values, two graphs in turn, each replay against the eager call."""
    announce("gated scan in graphs")

    def run(leaves, do, dh):
        o, h = vig_amd.gated_scan(*leaves, True)
        return [t.detach().clone() for t in (o, h) + torch.autograd.grad((o, h), leaves, (do, dh))]

    made, side = [], torch.cuda.Stream()
    for L in (196, 1400):
        x, g, h0, do, dh = draw(2, L, 68, BF16, BF16, False, L, state=True)
        fresh = lambda ts: [t.detach().clone().requires_grad_() for t in ts]  # noqa: E731
        eager = run(fresh((x, g, h0)), do, dh)
        leaves = fresh((x, g, h0))
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            warm = run(leaves, do, dh)
        torch.cuda.current_stream().wait_stream(side)
        assert all(torch.equal(a, b) for a, b in zip(warm, eager))
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = run(leaves, do, dh)
        made.append((graph, out, leaves, do, dh))
    for turn in range(4):
        for graph, out, leaves, do, dh in made:
            with torch.no_grad():
                for t in leaves:
                    t.mul_(0.9)
            graph.replay()
            torch.cuda.synchronize()
            eager = run(fresh(leaves), do, dh)
            assert all(torch.equal(a, b) for a, b in zip(out, eager)), turn


@pytest.mark.parametrize("both", [False, True])
def test_the_widest_rows(both):
    """1024 rows of 262144 channels in fp32, 2^30 bytes of one workgroup's reach; then a few channels of such rows."""
    L, D = 1024, 1 << 18
    announce(f"gated scan of {D} channels both={both}")
    x, g, h0, do, dh = draw(1, L, D, F32, F32, both, 1, state=not both)
    some = slice(D - 70, D)
    for cut in (slice(None), some):
        given = [t[..., cut].detach().requires_grad_() for t in ((x, g) if both else (x, g, h0))]
        o, h = vig_amd.bid_gated_scan(*given) if both else vig_amd.gated_scan(*given, True)
        got = torch.autograd.grad((o,) if both else (o, h), given, (do[..., cut],) if both else (do[..., cut], dh[:, cut]))
        want = reference(x[..., some], g[..., some], None if both else h0[:, some], both, do[..., some], None if both else dh[:, some])
        close(o[..., -70:], want["o"], "o"), close(got[0][..., -70:], want["dx"], "dx"), close(got[1][..., -70:], want["dg"], "dg")
    with pytest.raises(Exception):
        vig_amd.gated_scan(torch.zeros(1, 2, D + 1, device="cuda"), torch.zeros(1, 2, D + 1, device="cuda"))


@pytest.mark.parametrize("native", [True, False])
def test_inference_mode(native, monkeypatch):
    if not native:
        monkeypatch.setattr(_ext, "calls", lambda: None)
    x, g, h0, _, _ = draw(3, 5, 12, F32, F32, False, 7, state=True)
    with torch.inference_mode():
        h = h0.clone()
        o = torch.stack([vig_amd.gated_scan_step(x[:, t], g[:, t], h) for t in range(5)], 1)
        whole, last = vig_amd.gated_scan(x.clone(), g, h0, True)
    want = reference(x, g, h0, False)
    close(o, want["o"], "steps"), close(whole, want["o"], "o"), close(h, want["final"], "state"), close(last, want["final"], "state")


def test_a_capture_with_a_leaf_that_an_eager_graph_holds():
    """Refused while the graph lives; captured and replayed once it is gone."""
    x, g, h0, do, dh = draw(2, 70, 10, F32, F32, False, 3, state=True)
    leaves = [t.detach().requires_grad_() for t in (x, g, h0)]
    alive = vig_amd.gated_scan(*leaves)[0]
    want = torch.autograd.grad(alive, leaves, do, retain_graph=True)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError, match="still holds a leaf"):
        with torch.cuda.graph(graph):
            vig_amd.gated_scan(*leaves)
    del alive
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        o, _ = vig_amd.gated_scan(*leaves)
        got = torch.autograd.grad(o, leaves, do)
    for _ in range(3):
        for t in got:
            t.fill_(float("nan"))
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_no_second_derivative(monkeypatch):
    x, g, h0, _, _ = draw(1, 9, 4, F32, F32, False, 1, state=True)
    for way in range(2):
        if way:
            monkeypatch.setattr(_ext, "calls", lambda: None)
        x = x.detach().requires_grad_()
        o, _ = vig_amd.gated_scan(x, g, h0)
        (dx,) = torch.autograd.grad(o.square().sum(), x, create_graph=True)
        want = reference(x, g, h0, False, 2 * o)["dx"]
        close(dx.detach(), (want[0], want[1] + 4 * U * want[0].abs().max()), "first")
        with pytest.raises(RuntimeError):
            dx.sum().backward()


@pytest.mark.parametrize("both", [False, True])
def test_more_sequences_than_a_launch_takes(both):
    """Seventy million sequences of two tokens: a launch takes 2^32 threads."""
    B = 70_000_000
    announce(f"gated scan of {B} sequences both={both}")
    gen = torch.Generator(device="cuda").manual_seed(2)
    r = lambda *s: torch.randn(*s, device="cuda", generator=gen, dtype=F32).to(BF16)  # noqa: E731
    x, g, do = r(B, 2, 1), -r(2 * B if both else B, 2, 1).abs(), r(B, 2, 1)
    h0, dh = (None, None) if both else (torch.randn(B, 1, device="cuda", generator=gen), torch.randn(B, 1, device="cuda", generator=gen))
    given = [t.requires_grad_() for t in ((x, g) if both else (x, g, h0))]
    o, h = vig_amd.bid_gated_scan(*given) if both else vig_amd.gated_scan(*given, True)
    got = torch.autograd.grad((o,) if both else (o, h), given, (do,) if both else (do, dh))
    with torch.no_grad():
        for some in (slice(0, 1000), slice(67_108_000, 67_110_000), slice(B - 1000, B)):
            gates = torch.cat([g[:B][some], g[B:][some]]) if both else g[some]
            want = reference(x[some], gates, None if both else h0[some], both, do[some], None if both else dh[some])
            close(o[some], want["o"], "o"), close(got[0][some], want["dx"], "dx")
            close(torch.cat([got[1][:B][some], got[1][B:][some]]) if both else got[1][some], want["dg"], "dg")
            if not both:
                close(h[some], want["final"], "final"), close(got[2][some], want["dh0"], "dh0")


def test_offsets_past_32_bits():
    """70000 tokens of 32768 channels: the last rows lie past 2^32 bytes, the last elements past 2^31."""
    L, D = 70000, 32768
    announce("gated scan past 2^31 elements")
    gen = torch.Generator(device="cuda").manual_seed(1)
    x = torch.zeros(1, L, D, device="cuda", dtype=BF16)
    g = torch.full((1, L, D), -1.0, device="cuda", dtype=BF16)
    tail = 100  # what lies further back has decayed below e^-100
    x[:, -tail:] = torch.randn(1, tail, D, device="cuda", generator=gen).bfloat16()
    o, h = vig_amd.gated_scan(x, g, None, True)
    want = reference(x[:, -tail:], g[:, -tail:])
    close(o[:, -tail:], want["o"], "o"), close(h, want["final"], "final")
    assert not bool(o[:, :-tail].any())
    del o
    g2 = torch.cat([g, g])
    del g
    o, _ = vig_amd.bid_gated_scan(x, g2)
    close(o[:, -tail:], reference(x[:, -tail:], g2[:, -tail:], None, True)["o"], "both")
