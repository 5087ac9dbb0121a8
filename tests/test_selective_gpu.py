"""The selective scan and its step against their recurrence in 64 bits, token by token.

Roundings on the way from an input to an output: a step's softplus up to 12 (exponential, series, sum), what is made of it and its products 6; a decay e^{sA} is off by its
exponent's error, (12 + 3) U |sA|, and 3 U of its own; the walk takes a product and a multiply-add a token, and chunks of it are joined by decays of sums of up to L steps, whose exponent is off
by (12 + L) U |sum A| at most where the decay matters (t e^-t < 0.4).  So each of L tokens adds at most 8 + 15 |sA|, the joins 2 (12 + L).  Sums over N states, over a group's channels
and over all tokens are added up in trees or runs of at most N + 64 + L + batch.  Gradients pass two walks.  Gates take 8, |z| U in their exponent another |z|."""
import math

import pytest
import torch

import vig_amd

from . import selective_ref as R
from .util import announce

pytestmark = pytest.mark.gpu

F32, BF16 = torch.float32, torch.bfloat16


def make(seed, batch, L, width, N, G=1, dtype=F32, gated=True, skip=True, softplus=True, biased=True, state=False, wide=False, padded=False, strong=1.0):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    r = lambda *s: torch.randn(*s, device="cuda", generator=gen)  # noqa: E731
    rows = lambda n: r(batch, L, n + 5).to(dtype)[..., 3:n + 3] if wide else r(batch, L, n).to(dtype)  # noqa: E731
    t = {"x": rows(width), "delta": rows(width), "A": -strong * torch.rand(width, N, device="cuda", generator=gen) * torch.arange(1, N + 1, device="cuda"),
         "D": r(width) if skip else None, "z": rows(width) if gated else None, "delta_bias": r(width) - 3 if biased else None}
    if G > 1 or wide:
        both = r(batch, L, 2 * G * (N + 1) + 1).to(dtype)[..., 1:].unflatten(-1, (2, G, N + 1))
        t |= {"B": both[:, :, 0, :, :N], "C": both[:, :, 1, :, 1:]}
    else:
        t |= {"B": rows(N), "C": rows(N)}
    if not softplus:
        t["delta"] = (t["delta"].abs() * 0.05).to(dtype)
        t["delta_bias"] = t["delta_bias"].abs() * 0.01 if biased else None
    if padded:
        t["delta"] = t["delta"].clone()
        t["delta"][::2, L // 2:] = -math.inf if softplus else 0
    t["initial_state"] = r(batch, width, N) if state else None
    return t | {"delta_softplus": softplus}


def roundings(t, L, grads=False):
    s = R.f64(t["delta"]) + (R.f64(t["delta_bias"]) if t["delta_bias"] is not None else 0)
    s = torch.nn.functional.softplus(s) if t["delta_softplus"] else s
    most = float((s.amax((0, 1)).unsqueeze(-1) * R.f64(t["A"]).abs()).max())
    N, zs = t["A"].shape[1], float(t["z"].abs().max()) if t["z"] is not None else 0
    one = 40 + L * (8 + 15 * most) + 2 * (12 + L) + N + 2 * zs
    return one * (2 if grads else 1) + (N + 64 + L * t["x"].shape[0] if grads else 0)


NAMES = ["x", "delta", "A", "B", "C", "D", "z", "delta_bias", "initial_state"]


def check(t, reverse=False, final=False, seed=0, grads=False, native=True):
    given = dict(t)
    if grads:
        given |= {k: t[k].detach().requires_grad_() for k in NAMES if t[k] is not None}
    o, h = vig_amd.selective_scan(**given, output_final_state=final, reverse=reverse)
    assert (h is not None) == final
    gen = torch.Generator(device="cuda").manual_seed(seed + 1000)
    d_o = torch.randn(o.shape, device="cuda", generator=gen).to(o.dtype) if grads else None
    d_final = torch.randn(h.shape, device="cuda", generator=gen) if grads and final else None
    want, size = (R.scan(**t, reverse=reverse, d_o=d_o, d_final=d_final, mag=mag) for mag in (False, True))
    L = t["x"].shape[1]
    R.close(o, want["o"], size["o"], roundings(t, L), "o")
    if final:
        R.close(h, want["final"], size["final"], roundings(t, L), "final")
    if not grads:
        return
    names = [k for k in NAMES if t[k] is not None]
    got = torch.autograd.grad([o] + [h] * final, [given[k] for k in names], [d_o] + [d_final] * final)
    for k, g in zip(names, got):
        key = {"delta_bias": "dbias", "initial_state": "dinitial"}.get(k, "d" + k)
        assert g.dtype == t[k].dtype
        R.close(g, want[key], size[key], roundings(t, L, True), key)


SHAPES = [
    # batch, L, width, N
    (1, 1, 1, 1), (2, 1, 16, 16), (1, 15, 17, 3), (2, 16, 64, 4), (3, 17, 65, 5), (1, 33, 48, 8), (2, 50, 20, 13), (1, 100, 130, 16), (2, 37, 33, 17), (1, 41, 16, 32), (1, 23, 18, 33),
    (2, 19, 31, 64),
]


@pytest.mark.parametrize("grads", [False, True])
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("shape", SHAPES)
def test_sizes(shape, dtype, grads):
    announce(f"selective scan {shape} {dtype} grads {grads}")
    check(make(1, *shape, dtype=dtype, state=True), final=True, grads=grads)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("flags", [
    dict(gated=False), dict(skip=False), dict(softplus=False), dict(biased=False, gated=False, skip=False, softplus=False), dict(wide=True), dict(padded=True), dict(padded=True, softplus=False),
    dict(strong=30.0), dict(G=2), dict(G=3, wide=True), dict(G=6), dict(state=True),
])
def test_forms(flags, dtype):
    announce(f"selective scan {flags} {dtype}")
    for reverse in (False, True):
        check(make(2, 2, 45, 18, 6, dtype=dtype, **flags), reverse=reverse, final=reverse, grads=True)


@pytest.mark.parametrize("N", [2, 7, 16, 20, 64])
def test_sequences_that_are_not_cut(N):
    """As many sequences as fill the chip by themselves: no chunks, several tiles of tokens, the last one short."""
    announce(f"1100 sequences, N {N}")
    t = make(3, 1100, 35, 4, N, dtype=BF16, state=True)
    check(t, final=True, grads=True)
    check(make(4, 1100, 18, 3, N, dtype=F32, padded=True), reverse=True, grads=True)


@pytest.mark.parametrize("batch,L,N", [(199, 200, 16), (200, 200, 16), (127, 120, 5), (128, 120, 5), (299, 259, 16), (300, 259, 16), (320, 257, 40), (351, 256, 7), (352, 256, 7), (255, 255, 33)])
def test_where_sequences_begin_to_go_through_whole(batch, L, N):
    """Forward and backward on either side of their borders: both cut, only the backward (300 to 351 sequences of 16 channels, 16 states), neither."""
    announce(f"selective scan, {batch} sequences of {L} tokens, {N} states")
    check(make(batch + N, batch, L, 16, N, state=True), final=True, grads=True)
    check(make(batch + N + 1, batch, L, 16, N, dtype=BF16), reverse=True, grads=True)


@pytest.mark.parametrize("L", [1000, 4097])
def test_long(L):
    announce(f"selective scan of {L} tokens")
    check(make(5, 1, L, 20, 16, dtype=BF16, state=True, strong=0.1), final=True, grads=True)
    check(make(5, 1, L, 20, 5, dtype=F32, strong=0.1), reverse=True, final=True)


def test_pieces_follow_one_another():
    """Two pieces with the state handed on are the whole, with its gradients."""
    announce("pieces")
    t = make(6, 2, 90, 24, 16, state=True)
    whole = {k: t[k].detach().clone().requires_grad_() for k in NAMES}
    o, h = vig_amd.selective_scan(**whole, delta_softplus=True, output_final_state=True)
    parts = {k: t[k].detach().clone().requires_grad_() for k in NAMES}
    cut = lambda a, b: {k: parts[k][:, a:b] if k in ("x", "delta", "B", "C", "z") else parts[k] for k in NAMES}  # noqa: E731
    o1, h1 = vig_amd.selective_scan(**cut(0, 37), delta_softplus=True, output_final_state=True)
    o2, h2 = vig_amd.selective_scan(**{**cut(37, 90), "initial_state": h1}, delta_softplus=True, output_final_state=True)
    d, dh = torch.randn_like(o), torch.randn_like(h)
    want = torch.autograd.grad([o, h], list(whole.values()), [d, dh])
    got = torch.autograd.grad([torch.cat([o1, o2], 1), h2], list(parts.values()), [d, dh])
    size = R.scan(**t, d_o=d, d_final=dh, mag=True)
    for k, a, b in zip(NAMES, got, want):
        key = {"delta_bias": "dbias", "initial_state": "dinitial"}.get(k, "d" + k)
        R.close(a, R.f64(b), size[key], 2 * roundings(t, 90, True), key)
    R.close(torch.cat([o1, o2], 1), R.f64(o), size["o"], 2 * roundings(t, 90), "o")


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("N,G,wide", [(1, 1, False), (3, 1, True), (4, 2, False), (13, 1, False), (16, 1, False), (16, 3, True), (33, 1, False), (64, 2, False)])
def test_step(N, G, wide, dtype):
    announce(f"selective scan step N {N} G {G} wide {wide} {dtype}")
    batch, width = 5, 66
    t = make(7, batch, 6, width, N, G, dtype, state=True, wide=wide)
    state = t["initial_state"].clone()
    for k in range(6):
        now = {n: t[n][:, k] for n in ("x", "delta", "B", "C", "z")}
        before, version = state.clone(), state._version
        o = vig_amd.selective_scan_step(**now, A=t["A"], state=state, D=t["D"], delta_bias=t["delta_bias"], delta_softplus=True)
        one = {**t, **{n: v.unsqueeze(1) for n, v in now.items()}, "initial_state": before}
        want, size = (R.scan(**one, mag=m) for m in (False, True))
        R.close(o, want["o"][:, 0], size["o"][:, 0], roundings(one, 1), f"o of token {k}")
        R.close(state, want["final"], size["final"], roundings(one, 1), f"state behind token {k}")
        assert state._version > version


def test_step_whose_state_begins_on_any_element():
    announce("step, odd addresses")
    t = make(8, 3, 1, 10, 8, state=True)
    room = torch.zeros(3 * 10 * 8 + 1, device="cuda")
    state = room[1:].view(3, 10, 8)
    state.copy_(t["initial_state"])
    call = lambda s: vig_amd.selective_scan_step(*(t[n][:, 0] for n in ("x", "delta")), t["A"], t["B"][:, 0], t["C"][:, 0], s, delta_softplus=True)  # noqa: E731
    other = t["initial_state"].clone()
    a, b = call(state), call(other)
    R.close(a, R.f64(b), R.f64(b).abs() + 1, 60, "o")
    R.close(state, R.f64(other), R.f64(other).abs() + 1, 60, "state")
    assert float(room[0]) == 0


def test_not_finite_stays_in_its_channel():
    announce("selective scan, NaN and infinities")
    for bad in (math.nan, math.inf):
        t = make(9, 2, 40, 33, 16)
        clean = vig_amd.selective_scan(**t)[0]
        t["x"][1, 20, 7] = bad
        o = vig_amd.selective_scan(**t)[0]
        keep = torch.ones_like(o, dtype=torch.bool)
        keep[1, 20:, 7] = False
        assert torch.equal(o[keep], clean[keep]) and not bool(torch.isfinite(o[1, 20:, 7]).any())


def test_padding_leaves_the_state():
    """Sequences padded behind their end: outputs in front and states as without, also where the padding's B, C and z hold anything finite.  (Not the states' bits: sequences of another
    length are cut elsewhere, and a state that was joined from chunks is rounded in other places than one that was walked to.  Both are within the bound.)"""
    announce("padded sequences")
    t = make(10, 2, 48, 40, 16, dtype=BF16, state=True)
    t["delta"][:, 32:] = -math.inf
    o, h = vig_amd.selective_scan(**t, output_final_state=True)
    short = {k: v[:, :32] if k in ("x", "delta", "B", "C", "z") else v for k, v in t.items()}
    o2, h2 = vig_amd.selective_scan(**short, output_final_state=True)
    want, size = (R.scan(**short, mag=m) for m in (False, True))
    for a, b in ((o[:, :32], h), (o2, h2)):
        R.close(a, want["o"], size["o"], roundings(short, 48), "o")
        R.close(b, want["final"], size["final"], roundings(short, 48), "final")


def test_same_bits_again_on_another_stream():
    announce("selective scan, repeated, on another stream")
    t = make(11, 4, 300, 100, 16, dtype=BF16)
    given = {**t, **{k: t[k].detach().requires_grad_() for k in NAMES if t[k] is not None}}
    names = [k for k in NAMES if t[k] is not None]

    def run():
        o = vig_amd.selective_scan(**given)[0]
        return (o.detach(), *torch.autograd.grad(o, [given[k] for k in names], torch.ones_like(o)))

    first = run()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        second = run()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(first, second))
