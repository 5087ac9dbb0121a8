"""Calls of the gated scan that have to be refused, on the GPU both ways and, with the library replaced by its formula, without one."""
import os

import pytest
import torch
import torch.autograd.forward_ad as forward_ad

import vig_amd
from vig_amd import _ext, _lib

from .test_recorded_calls import device, formula, inputs  # noqa: F401
from .util import announce


@pytest.mark.parametrize("leaf", [False, True])
@pytest.mark.parametrize("call,which", [(c, w) for c in ("gated_scan", "bid_gated_scan", "gated_scan_step") for w in "xgh" if (c, w) != ("bid_gated_scan", "h")])
def test_no_forward_derivative(call, which, leaf, device):  # noqa: F811
    """A tangent is not dropped without a word; a tensor without one passes beside an open level."""
    announce(f"{call}, tangent of {which}, leaf {leaf} on {device}")

    def run(t):
        if call == "gated_scan":
            return vig_amd.gated_scan(t["x"], t["g"], t["h"])[0]
        if call == "bid_gated_scan":
            return vig_amd.bid_gated_scan(t["x"], torch.cat([t["g"], t["g"]]))[0]
        return vig_amd.gated_scan_step(t["x"][:, 0], t["g"][:, 0], t["h"])

    given = dict(zip("xgh", inputs(device, 1)))
    with forward_ad.dual_level():
        want = run({k: t.clone() for k, t in given.items()})
        at = given[which].clone().requires_grad_(leaf)
        with pytest.raises((RuntimeError, ValueError)):
            run(given | {which: forward_ad.make_dual(at, torch.ones_like(at))})
    assert bool(torch.isfinite(want).all())


class OnGpu(torch.Tensor):
    """A tensor in host memory that says it is on the GPU."""
    is_cuda = property(lambda self: True)


def kinds(made):
    """The forms of a call: names of its leaves -> the call."""
    x, g, h = made
    heads = [t.detach()[:, None].requires_grad_() for t in (x, g, h)]
    half = h.detach().bfloat16().requires_grad_()
    return {
        "plain": ([x, g, h], lambda: vig_amd.gated_scan(x, g, h)),
        "heads": (heads, lambda: vig_amd.gated_scan(*heads)),
        "heads, rows alone": (heads[:1], lambda: vig_amd.gated_scan(heads[0], heads[1].detach())),
        "state in bf16": ([half], lambda: vig_amd.gated_scan(x.detach(), g.detach(), half)),
        "both": ([x], lambda: vig_amd.bid_gated_scan(x, torch.cat([g, g]).detach())),
    }


@pytest.mark.parametrize("native", [True, False])
@pytest.mark.parametrize("kind", ["plain", "heads", "heads, rows alone", "state in bf16", "both"])
def test_leaves_are_looked_at_before_a_capture(kind, native, monkeypatch, request):
    """The caller's own leaves, not what is made of them on the way, are asked for; where nothing can be asked, the call is refused."""
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
    seen = []

    class Calls:
        gated_scan = staticmethod(lambda *a: None)

        @staticmethod
        def refuse_held_leaves(*ts):
            seen.extend(ts)
            raise RuntimeError("held")

    request.getfixturevalue("formula")
    monkeypatch.setattr(_ext, "calls", lambda: Calls if native else None)
    leaves, call = kinds([t.as_subclass(OnGpu).detach().requires_grad_() for t in inputs("cpu", 1)])[kind]
    with pytest.raises(RuntimeError, match="held" if native else "capture"):
        call()
    assert [id(t) for t in seen] == ([id(t) for t in leaves] if native else [])
    with torch.no_grad():
        call()
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    call()


@pytest.mark.gpu
@pytest.mark.parametrize("native", [True, False])
@pytest.mark.parametrize("kind", ["heads", "heads, rows alone", "state in bf16", "both"])
def test_captures_of_held_leaves(kind, native, monkeypatch):
    """Refused while an eager graph lives, whichever form the leaf comes in; captured and replayed once it is gone."""
    announce(f"held leaves: {kind}, native {native}")
    if not native:
        monkeypatch.setattr(_ext, "calls", lambda: None)
    leaves, call = kinds([t.requires_grad_() for t in inputs("cuda", 1, L=70)])[kind]
    alive = call()[0]
    d = torch.randn_like(alive)
    want = torch.autograd.grad(alive, leaves, d, retain_graph=True)
    torch.cuda.synchronize()
    with pytest.raises(RuntimeError, match="capture"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            call()
    if not native:
        return
    del alive
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = torch.autograd.grad(call()[0], leaves, d)
    for _ in range(3):
        for t in got:
            t.fill_(float("nan"))
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_sequences_longer_than_the_chunks_are_folded_for():
    """Every chunk folds all in front of it: past 2^24 tokens the square of their number is refused."""
    if not os.path.exists(_lib.LIB_PATH):
        pytest.skip("library not built here")
    lib = _lib.load()
    P, most = 1 << 20, 1 << 24
    fwd = lambda L: lib.vig_gated_scan_fwd(P, 2 * P, None, None, 3 * P, None, None, 0, 1, L, 8, None, None, 1.0, 1, 1, None)  # noqa: E731
    bwd = lambda L: lib.vig_gated_scan_bwd(P, 2 * P, None, None, 3 * P, None, 4 * P, 5 * P, None, None, None, 0, 1, L, 8, None, None, 1.0, 1, 1, None)  # noqa: E731
    assert fwd(most) == bwd(most) == _lib.VIG_ENOSPC and lib.vig_gated_scan_fwd_workspace(1, most, 8, 1) > 0
    assert fwd(most + 1) == bwd(most + 1) == _lib.VIG_ENOTSUP
    assert lib.vig_gated_scan_fwd_workspace(1, most + 1, 8, 0) == lib.vig_gated_scan_bwd_workspace(1, most + 1, 8, 1) == 0


@pytest.mark.gpu
def test_the_longest_sequences():
    """2^24 tokens that change nothing but for a few: sums of whole numbers, which are exact; one token more is refused."""
    L, D = 1 << 24, 2
    announce(f"gated scan of {L} tokens")
    x = torch.zeros(1, L, D, device="cuda")
    at = torch.tensor([0, 1, 511, 512, 70_000, 1 << 20, (1 << 23) + 5, L - 513, L - 1], device="cuda")
    x[0, at, 0], x[0, at, 1] = torch.arange(1.0, 10.0, device="cuda"), 3.0
    g, h0 = torch.zeros_like(x), torch.full((1, D), 5.0, device="cuda")
    o, h = vig_amd.gated_scan(x, g, h0, True)
    want = 5 + x.double().cumsum(1)
    assert torch.equal(o.double(), want) and torch.equal(h.double(), want[:, -1])
    x.requires_grad_()
    o, _ = vig_amd.bid_gated_scan(x, torch.cat([g, g]))
    back = x.detach().double().flip(1).cumsum(1).flip(1)
    assert torch.equal(o.detach().double(), (want - 5 + back) / 2)
    (dx,) = torch.autograd.grad(o, x, x.detach())
    assert torch.equal(dx.double(), (want - 5 + back) / 2)
    with pytest.raises(Exception):
        vig_amd.gated_scan(torch.zeros(1, L + 1, 1, device="cuda"), torch.zeros(1, L + 1, 1, device="cuda"))
