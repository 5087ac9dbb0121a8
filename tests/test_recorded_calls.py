"""The gated scan, its step and the gradients' norm under a trace: what is recorded has to compute on new inputs, on the GPU and, with
the library replaced by the formula in numpy, without one."""
import contextlib
import ctypes

import numpy as np
import pytest
import torch
from torch.fx.experimental.proxy_tensor import make_fx

import vig_amd
from vig_amd import _ext, _lib, ops

from .util import announce

pytestmark = pytest.mark.filterwarnings("ignore::torch.jit.TracerWarning")


class Formula:
    """The library's entry points on dense fp32 arrays in host memory."""

    @staticmethod
    def at(p, *shape):
        return np.ctypeslib.as_array(ctypes.cast(p, ctypes.POINTER(ctypes.c_float)), shape)

    def vig_gated_scan_fwd_workspace(self, *a):
        return 0

    vig_gated_scan_bwd_workspace = vig_gated_scan_fwd_workspace

    def vig_grad_norm_workspace(self, *a):
        return 8

    def vig_gated_scan_fwd(self, x, gf, gb, h0, o, hT, ws, need, B, L, D, xs, gs, scale, *rest):
        x, o = self.at(x, B, L, D), self.at(o, B, L, D)
        o[:] = 0
        for p, order in ((gf, range(L)), (gb, range(L - 1, -1, -1))):
            if p is None:
                continue
            g, h = self.at(p, B, L, D), self.at(h0, B, D).copy() if h0 else np.zeros((B, D), np.float32)
            for t in order:
                h = np.exp(g[:, t]) * h + x[:, t]
                o[:, t] += scale * h
        if hT:
            self.at(hT, B, D)[:] = h
        return 0

    def vig_gated_scan_bwd(self, x, gf, gb, h0, do, dT, dx, dgf, dgb, dh0, ws, need, B, L, D, xs, gs, scale, *rest):
        x, do, dx = (self.at(p, B, L, D) for p in (x, do, dx))
        dx[:] = 0
        for p, dp, order in ((gf, dgf, range(L)), (gb, dgb, range(L - 1, -1, -1))):
            if p is None:
                continue
            g, dg, h, us = self.at(p, B, L, D), self.at(dp, B, L, D), self.at(h0, B, D).copy() if h0 else np.zeros((B, D), np.float32), {}
            for t in order:
                us[t] = np.exp(g[:, t]) * h
                h = us[t] + x[:, t]
            d = self.at(dT, B, D).copy() if dT else np.zeros((B, D), np.float32)
            for t in reversed(order):
                d = d + scale * do[:, t]
                dx[:, t] += d
                dg[:, t] = d * us[t]
                d = np.exp(g[:, t]) * d
        if dh0:
            self.at(dh0, B, D)[:] = d
        return 0

    def vig_gated_scan_step(self, x, g, h, o, B, D, *rest):
        x, g, h, o = (self.at(p, B, D) for p in (x, g, h, o))
        h[:] = np.exp(g) * h + x
        o[:] = h
        return 0

    def vig_grad_norm(self, ptrs, n, types, count, most, norm, scale, *rest):
        r = sum(float((self.at(ptrs[j], n[j]).astype(np.float64) ** 2).sum()) for j in range(count)) ** 0.5
        self.at(norm, 1)[:] = r
        if scale:
            self.at(scale, 1)[:] = min(1.0, most / (r + 1e-6))
        return 0


@pytest.fixture
def formula(monkeypatch):
    """The formula in place of the library, for tensors in host memory."""
    lib = Formula()
    monkeypatch.setattr(_lib, "load", lambda: lib)
    monkeypatch.setattr(ops, "_check_cuda", lambda *ts: None)
    monkeypatch.setattr(ops, "_stream_ptr", lambda t: 0)
    monkeypatch.setattr(torch.cuda, "device", lambda d: contextlib.nullcontext())


@pytest.fixture(params=["cpu", pytest.param("cuda", marks=pytest.mark.gpu), pytest.param("ctypes", marks=pytest.mark.gpu)])
def device(request, monkeypatch):
    if request.param != "cuda":
        monkeypatch.setattr(_ext, "calls", lambda: None)
    if request.param != "cpu":
        return "cuda"
    request.getfixturevalue("formula")
    return "cpu"


def inputs(device, seed, B=2, L=9, D=8, both=False):
    gen = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=gen)  # noqa: E731
    return [t.to(device) for t in (r(B, L, D), -r(2 * B if both else B, L, D).abs(), r(B, D))]


def recorded(f, args, way):
    if way == "trace":
        return torch.jit.trace(f, tuple(args), check_trace=False)
    return make_fx(f)(*args)


def scan(x, g, h):
    return vig_amd.gated_scan(x, g, h, True)


def both(x, g, h):
    return vig_amd.bid_gated_scan(x, torch.cat([g, g]))[0]


def heads(x, g, h):
    return vig_amd.gated_scan(x.unsqueeze(1), g.unsqueeze(1))[0]


def step(x, g, h):
    h = h.clone()
    return vig_amd.gated_scan_step(x[:, 0], g[:, 0], h), h


def norm(x, g, h):
    return vig_amd.grad_norm([x, g, h], 0.5)


@pytest.mark.parametrize("way", ["trace", "fx"])
@pytest.mark.parametrize("f", [scan, both, heads, step, norm])
def test_a_record_computes_on_new_inputs(f, way, device):
    announce(f"{f.__name__} recorded by {way} on {device}")
    r = recorded(f, inputs(device, 1), way)
    assert "empty" not in str(r.inlined_graph if way == "trace" else r.graph)
    for seed in (2, 3):
        args = inputs(device, seed)
        got, want = r(*args), f(*args)
        for a, b in zip(*((t,) if isinstance(t, torch.Tensor) else t for t in (got, want))):
            assert torch.equal(a, b)


@pytest.mark.parametrize("way", ["trace", "fx"])
def test_a_recorded_step_moves_its_state(way, device):
    f = lambda x, g, h: vig_amd.gated_scan_step(x[:, 0], g[:, 0], h)  # noqa: E731
    r = recorded(f, inputs(device, 1), way)
    x, g, h = inputs(device, 2)
    other = h.clone()
    version = h._version
    assert torch.equal(r(x, g, h), f(x, g, other)) and torch.equal(h, other) and h._version > version


@pytest.mark.parametrize("f", [scan, both])
def test_recorded_gradients(f, device):
    def grads(x, g, h):
        x, g, h = (t.detach().requires_grad_() for t in (x, g, h))
        out = f(x, g, h)
        out = (out,) if isinstance(out, torch.Tensor) else out
        return torch.autograd.grad(sum(t.cos().sum() for t in out), (x, g, h) if f is scan else (x, g))

    r = make_fx(grads)(*inputs(device, 1))
    args = inputs(device, 2)
    assert all(torch.equal(a, b) for a, b in zip(r(*args), grads(*args)))


def test_a_trace_of_leaves(device):
    """A traced call whose inputs require gradients computes on new ones too."""
    x, g, h = inputs(device, 1)
    r = torch.jit.trace(lambda x, g, h: vig_amd.gated_scan(x, g, h)[0], (x.requires_grad_(), g, h), check_trace=False)
    x, g, h = inputs(device, 2)
    assert torch.equal(r(x, g, h), vig_amd.gated_scan(x, g, h)[0])


@pytest.mark.parametrize("way", ["trace", "fx"])
def test_an_update_is_not_recorded(way, device):
    """Its lists are changed in place, which no record here would hold."""
    def f(p, g, m):
        vig_amd.adamw_step([p], [g], [m], [m.clone()], step=1)
        return p

    with pytest.raises(RuntimeError, match="record"):
        recorded(f, [torch.ones(5, device=device) for _ in range(3)], way)
