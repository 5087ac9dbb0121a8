"""Calls of the selective scan, the short convolution, their steps and the add and layer norm that have to be refused: by the C ABI before anything is enqueued, by the Python calls with
and without a GPU."""
import os

import pytest
import torch
import torch.autograd.forward_ad as forward_ad

import vig_amd
from vig_amd import _ext, _lib, ops

from .util import announce


@pytest.fixture(params=["cpu", pytest.param("cuda", marks=pytest.mark.gpu), pytest.param("ctypes", marks=pytest.mark.gpu)])
def device(request, monkeypatch):
    """The GPU, through the native calls and through ctypes; host memory that passes for it, where no launch may follow."""
    if request.param != "cuda":
        monkeypatch.setattr(_ext, "calls", lambda: None)
    if request.param != "cpu":
        return "cuda"
    monkeypatch.setattr(ops, "_check_cuda", lambda *ts: None)
    monkeypatch.setattr(_lib, "load", lambda: pytest.fail("a call went through to the library"))
    return "cpu"


def scan_args(device, batch=2, L=5, D=6, N=4, dtype=torch.float32):
    r = lambda *s: torch.randn(*s, device=device).to(dtype)  # noqa: E731
    f = lambda *s: torch.randn(*s, device=device)  # noqa: E731
    return {"x": r(batch, L, D), "delta": r(batch, L, D), "A": -f(D, N).abs(), "B": r(batch, L, N), "C": r(batch, L, N), "D": f(D), "z": r(batch, L, D), "delta_bias": f(D),
            "initial_state": f(batch, D, N)}


def step_args(device, **kw):
    t = scan_args(device, **kw)
    return {k: v[:, 0] if k in ("x", "delta", "B", "C", "z") else v for k, v in t.items() if k != "initial_state"} | {"state": t["initial_state"]}


def conv_args(device, batch=2, L=5, D=6, W=4):
    r = lambda *s: torch.randn(*s, device=device)  # noqa: E731
    return {"x": r(batch, L, D), "weight": r(D, W), "bias": r(D), "initial_state": r(batch, W - 1, D)}


def conv_step_args(device):
    t = conv_args(device)
    return {"x": t["x"][:, 0], "weight": t["weight"], "state": t["initial_state"], "bias": t["bias"]}


def norm_args(device, rows=4, C=6):
    r = lambda *s: torch.randn(*s, device=device)  # noqa: E731
    return {"x": r(rows, C), "weight": r(C), "bias": r(C), "residual": r(rows, C)}


CALLS = {"selective_scan": scan_args, "selective_scan_step": step_args, "causal_conv1d": conv_args, "causal_conv1d_step": conv_step_args, "add_layernorm": norm_args}
H, I = torch.float16, torch.int64
WRONG = [
    ("selective_scan", "x", lambda t: t[0]), ("selective_scan", "x", lambda t: t[:, :, :5]), ("selective_scan", "x", lambda t: t.to(H)), ("selective_scan", "x", lambda t: t.bfloat16()),
    ("selective_scan", "delta", lambda t: t[:, :4]), ("selective_scan", "delta", lambda t: t.bfloat16()), ("selective_scan", "A", lambda t: t[:, :3]), ("selective_scan", "A", lambda t: t.to(I)),
    ("selective_scan", "A", lambda t: t[:5]), ("selective_scan", "B", lambda t: t[:, :, :3]), ("selective_scan", "B", lambda t: t.double()), ("selective_scan", "C", lambda t: t[:, :4]),
    ("selective_scan", "C", lambda t: t.unsqueeze(2)), ("selective_scan", "D", lambda t: t[:5]), ("selective_scan", "z", lambda t: t[:1]), ("selective_scan", "z", lambda t: t.bfloat16()),
    ("selective_scan", "delta_bias", lambda t: t.unsqueeze(0)), ("selective_scan", "initial_state", lambda t: t[:1]), ("selective_scan", "initial_state", lambda t: t.transpose(1, 2)),
    ("selective_scan_step", "x", lambda t: t[0]), ("selective_scan_step", "delta", lambda t: t[:, :5]), ("selective_scan_step", "B", lambda t: t[:, :3]),
    ("selective_scan_step", "state", lambda t: t[:1]), ("selective_scan_step", "state", lambda t: t.bfloat16()), ("selective_scan_step", "state", lambda t: t.transpose(1, 2).contiguous().transpose(1, 2)),
    ("selective_scan_step", "A", lambda t: t.requires_grad_()), ("selective_scan_step", "state", lambda t: t.requires_grad_()), ("selective_scan_step", "z", lambda t: t.to(H)),
    ("causal_conv1d", "x", lambda t: t[0]), ("causal_conv1d", "x", lambda t: t.to(H)), ("causal_conv1d", "weight", lambda t: t[:5]), ("causal_conv1d", "weight", lambda t: t[:, :1]),
    ("causal_conv1d", "weight", lambda t: torch.cat([t, t], 1)), ("causal_conv1d", "weight", lambda t: t.unsqueeze(0)), ("causal_conv1d", "bias", lambda t: t[:5]),
    ("causal_conv1d", "initial_state", lambda t: t[:, :2]), ("causal_conv1d", "initial_state", lambda t: t.bfloat16()),
    ("causal_conv1d_step", "x", lambda t: t.unsqueeze(1)), ("causal_conv1d_step", "state", lambda t: t.bfloat16()), ("causal_conv1d_step", "state", lambda t: t[:, 1:]),
    ("causal_conv1d_step", "state", lambda t: t.transpose(1, 2).contiguous().transpose(1, 2)), ("causal_conv1d_step", "weight", lambda t: t.requires_grad_()),
    ("add_layernorm", "x", lambda t: t[0, 0]), ("add_layernorm", "x", lambda t: t.to(H)), ("add_layernorm", "weight", lambda t: t[:5]), ("add_layernorm", "bias", lambda t: t[:5]),
    ("add_layernorm", "residual", lambda t: t[:3]), ("add_layernorm", "residual", lambda t: t.bfloat16()), ("add_layernorm", "x", lambda t: torch.zeros(1, 16385, device=t.device)),
]


@pytest.mark.parametrize("case", range(len(WRONG)))
def test_wrong_arguments(case, device):
    call, name, change = WRONG[case]
    announce(f"{call}, wrong {name} ({case}) on {device}")
    t = CALLS[call](device)
    before = t["state"].clone() if "state" in t else None
    state = t.get("state")
    with pytest.raises((ValueError, TypeError)):
        getattr(vig_amd, call)(**{**t, name: change(t[name])})
    if before is not None:
        assert torch.equal(state.detach(), before)


@pytest.mark.parametrize("N,G,D", [(65, 1, 6), (4, 4, 6), (0, 1, 6)])
def test_states_and_groups_that_are_not_built(N, G, D, device):
    announce(f"N {N} G {G} D {D} on {device}")
    t = scan_args(device, D=D, N=N)
    for k in "BC":
        t[k] = torch.randn(2, 5, G, N, device=device)
    with pytest.raises(ValueError):
        vig_amd.selective_scan(**t)


@pytest.mark.parametrize("call", list(CALLS))
def test_no_forward_derivative(call, device):
    announce(f"{call}, tangents on {device}")
    for name in CALLS[call](device):
        t = CALLS[call](device)
        with forward_ad.dual_level():
            with pytest.raises((RuntimeError, ValueError)):
                getattr(vig_amd, call)(**{**t, name: forward_ad.make_dual(t[name], torch.ones_like(t[name]))})


@pytest.mark.parametrize("call", list(CALLS))
def test_host_memory_is_refused(call):
    with pytest.raises(_lib.VigGlaError):
        getattr(vig_amd, call)(**CALLS[call]("cpu"))


def test_nothing_to_do(device):
    """No tokens, no sequences, no rows: outputs of those sizes, and a state that stays."""
    t = scan_args(device, L=0)
    o, h = vig_amd.selective_scan(**t, output_final_state=True)
    assert o.shape == (2, 0, 6) and torch.equal(h, t["initial_state"]) and h is not t["initial_state"]
    o, h = vig_amd.selective_scan(**scan_args(device, batch=0), output_final_state=True)
    assert o.shape == (0, 5, 6) and h.shape == (0, 6, 4)
    t = conv_args(device, L=0)
    y, h = vig_amd.causal_conv1d(**t, output_final_state=True)
    assert y.shape == (2, 0, 6) and torch.equal(h, t["initial_state"])
    t = norm_args(device, rows=0)
    t = {k: v.requires_grad_() for k, v in t.items()}
    y, total = vig_amd.add_layernorm(**t, prenorm=True)
    assert y.shape == total.shape == (0, 6)
    assert torch.equal(torch.autograd.grad(y.sum() + total.sum(), t["weight"])[0], torch.zeros(6, device=device))


def _lib_or_skip():
    if not os.path.exists(_lib.LIB_PATH):
        pytest.skip("library not built here")
    return _lib.load()


P = 1 << 20  # addresses that are never used: the calls below have to end before a launch


def scan_call(lib, bwd=False, **kw):
    a = dict(x=P, delta=2 * P, A=3 * P, B=4 * P, C=5 * P, D=6 * P, z=7 * P, bias=8 * P, h0=9 * P, o=10 * P, hT=11 * P, kept=12 * P, ws=None, need=0, batch=1, L=5, width=6, N=4, G=1,
             xs=None, ds=None, bs=None, cs=None, zs=None, soft=1, rev=0, dt=1, d_o=13 * P, dT=14 * P, dx=15 * P, dd=16 * P, dB=17 * P, dC=18 * P, dz=19 * P, dp=20 * P, dh0=21 * P) | kw
    front, sizes, back = [a[k] for k in ("x", "delta", "A", "B", "C", "D", "z", "bias")], [a[k] for k in ("batch", "L", "width", "N", "G")], [a[k] for k in ("xs", "ds", "bs", "cs", "zs", "soft", "rev", "dt")]
    if bwd:
        return lib.vig_selective_scan_bwd(*front, a["kept"], a["d_o"], a["dT"], a["dx"], a["dd"], a["dB"], a["dC"], a["dz"], a["dp"], a["dh0"], a["ws"], a["need"], *sizes, *back, None)
    return lib.vig_selective_scan_fwd(*front, a["h0"], a["o"], a["hT"], a["kept"], a["ws"], a["need"], *sizes, *back, None)


def strides(*v):
    import ctypes

    return (ctypes.c_longlong * len(v))(*v)


def test_scan_abi():
    lib = _lib_or_skip()
    fwd, bwd = (lambda **k: scan_call(lib, **k)), (lambda **k: scan_call(lib, True, **k))
    EINVAL, ENOTSUP, ENOSPC = _lib.VIG_EINVAL, _lib.VIG_ENOTSUP, _lib.VIG_ENOSPC
    assert bwd() == ENOSPC  # (all in order but for the workspace)
    assert fwd(L=4000) == bwd(L=4000) == ENOSPC and lib.vig_selective_scan_fwd_workspace(1, 4000, 6, 4, 1) > 0
    for call in (fwd, bwd):
        for name in ("x", "delta", "A", "B", "C"):
            assert call(**{name: None}) == EINVAL
        for name in ("batch", "L", "width", "N", "G"):
            assert call(**{name: 0}) == EINVAL
        assert call(G=4) == EINVAL and call(N=65) == ENOTSUP and call(dt=2) == ENOTSUP and call(L=(1 << 24) + 1) == ENOTSUP and call(width=(1 << 18) + 1) == ENOTSUP
        assert call(x=P + 1) == call(A=3 * P + 2) == call(D=6 * P + 1) == EINVAL
        assert call(kept=12 * P + 4) == call(ws=22 * P + 8) == EINVAL
        assert call(xs=strides(30, 5)) == call(xs=strides(-1, 6)) == call(bs=strides(20, 3, 4)) == call(zs=strides(0, (1 << 18) + 1)) == EINVAL
        assert call(G=2, bs=strides(40, 8, 3)) == call(G=2, bs=strides(40, 8, 5)) == EINVAL
    assert fwd(o=None) == fwd(o=P) == fwd(o=7 * P) == fwd(hT=9 * P) == fwd(hT=11 * P + 2) == EINVAL
    assert fwd(batch=1 << 28, L=1, width=1 << 10, kept=None) in (ENOTSUP, ENOSPC)
    for name in ("kept", "d_o", "dx", "dd", "dB", "dC", "dz", "dp"):
        assert bwd(**{name: None}) == EINVAL
    assert bwd(z=None) == bwd(dx=2 * P) == bwd(dB=18 * P) == bwd(dh0=14 * P) == bwd(dp=20 * P + 2) == EINVAL and bwd(z=None, dz=None) == ENOSPC


def test_step_conv_and_norm_abi():
    lib = _lib_or_skip()
    EINVAL, ENOTSUP, ENOSPC = _lib.VIG_EINVAL, _lib.VIG_ENOTSUP, _lib.VIG_ENOSPC

    def step(x=P, delta=2 * P, A=3 * P, B=4 * P, C=5 * P, state=6 * P, o=7 * P, batch=2, D=6, N=4, G=1, xs=0, bs=None, dt=1):
        return lib.vig_selective_scan_step(x, delta, A, B, C, None, None, None, state, o, batch, D, N, G, xs, 0, bs, None, 0, 1, dt, None)

    assert step(x=None) == step(state=None) == step(o=None) == step(o=P) == step(state=3 * P) == step(state=6 * P + 2) == step(batch=0) == step(G=4) == step(xs=5) == step(o=6 * P) == EINVAL
    assert step(N=65) == step(dt=3) == ENOTSUP and step(G=2, bs=strides(8, 3)) == EINVAL

    def conv(x=P, w=2 * P, b=3 * P, h0=4 * P, y=5 * P, hT=6 * P, B=1, L=5, D=6, W=4, xs=None, dt=1):
        return lib.vig_causal_conv1d_fwd(x, w, b, h0, y, hT, B, L, D, W, xs, 1, 0, dt, None)

    assert conv(x=None) == conv(w=None) == conv(y=None) == conv(y=P) == conv(y=6 * P) == conv(hT=4 * P) == conv(x=P + 1) == conv(L=0) == conv(W=0) == conv(xs=strides(30, 5)) == EINVAL
    assert conv(W=1) == conv(W=5) == conv(dt=9) == conv(L=(1 << 24) + 1) == ENOTSUP

    def conv_bwd(dy=7 * P, dT=8 * P, dx=9 * P, dh0=10 * P, dw=11 * P, ws=None, need=0):
        return lib.vig_causal_conv1d_bwd(P, 2 * P, 3 * P, 4 * P, dy, dT, dx, dh0, dw, ws, need, 1, 5, 6, 4, None, 1, 0, 1, None)

    assert conv_bwd() == ENOSPC and conv_bwd(dy=None) == conv_bwd(dx=None) == conv_bwd(dx=P) == conv_bwd(dx=7 * P) == conv_bwd(dh0=4 * P) == conv_bwd(dw=2 * P) == conv_bwd(dw=9 * P) == EINVAL
    assert lib.vig_causal_conv1d_step(P, 2 * P, None, None, 5 * P, 1, 6, 4, 0, 1, 1, None) == EINVAL
    assert lib.vig_causal_conv1d_step(P, 2 * P, None, 4 * P, 4 * P, 1, 6, 4, 0, 1, 1, None) == lib.vig_causal_conv1d_step(P, 2 * P, None, 4 * P, 5 * P, 1, 6, 4, 5, 1, 1, None) == EINVAL

    def norm(x=P, r=2 * P, w=3 * P, b=4 * P, s=5 * P, y=6 * P, st=7 * P, rows=4, C=6, eps=1e-5, dt=1, sdt=0):
        return lib.vig_add_layernorm_fwd(x, r, w, b, s, y, st, rows, C, eps, dt, sdt, None)

    assert norm(x=None) == norm(w=None) == norm(y=None) == norm(s=None) == norm(r=None) == norm(r=None, s=None) == norm(y=P) == norm(s=2 * P) == norm(s=6 * P) == norm(eps=-1.0) == EINVAL
    assert norm(rows=0) == norm(C=0) == norm(x=P + 1) == norm(st=7 * P + 1) == EINVAL and norm(C=16385) == norm(dt=0, sdt=1) == norm(rows=(1 << 24) + 1) == ENOTSUP

    def norm_bwd(s=P, st=2 * P, w=3 * P, dy=4 * P, ds=5 * P, dr=6 * P, dx=7 * P, dw=8 * P, ws=None, need=0):
        return lib.vig_add_layernorm_bwd(s, st, w, dy, ds, dr, dx, dw, ws, need, 4, 6, 1, 0, None)

    assert norm_bwd() == ENOSPC and norm_bwd(s=None) == norm_bwd(st=None) == norm_bwd(w=None) == norm_bwd(dy=None) == norm_bwd(dr=None, dx=None, dw=None) == EINVAL
    assert norm_bwd(dx=4 * P) == norm_bwd(dr=5 * P) == norm_bwd(dw=3 * P) == norm_bwd(dx=8 * P) == norm_bwd(dr=7 * P) == EINVAL


@pytest.mark.gpu
@pytest.mark.parametrize("native", [True, False])
@pytest.mark.parametrize("call", ["selective_scan", "causal_conv1d", "add_layernorm"])
def test_captures_of_held_leaves(call, native, monkeypatch):
    """Refused while an eager graph of the leaves lives; captured and replayed once it is gone."""
    announce(f"held leaves: {call}, native {native}")
    if not native:
        monkeypatch.setattr(_ext, "calls", lambda: None)
    leaves = {k: t.requires_grad_() for k, t in CALLS[call]("cuda").items()}
    first = lambda r: r[0] if isinstance(r, tuple) else r  # noqa: E731
    run = lambda: first(getattr(vig_amd, call)(**leaves))  # noqa: E731
    alive = run()
    d = torch.randn_like(alive)
    want = torch.autograd.grad(alive, list(leaves.values()), d, retain_graph=True)
    torch.cuda.synchronize()
    with pytest.raises(RuntimeError, match="capture"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            run()
    if not native:
        return
    del alive
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = torch.autograd.grad(run(), list(leaves.values()), d)
    for _ in range(3):
        for t in got:
            t.fill_(float("nan"))
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.gpu
@pytest.mark.parametrize("native", [True, False])
@pytest.mark.parametrize("call", ["selective_scan", "causal_conv1d", "add_layernorm"])
def test_no_second_derivative(call, native, monkeypatch):
    announce(f"second derivative: {call}, native {native}")
    if not native:
        monkeypatch.setattr(_ext, "calls", lambda: None)
    leaves = {k: t.requires_grad_() for k, t in CALLS[call]("cuda").items()}
    r = getattr(vig_amd, call)(**leaves)
    o = r[0] if isinstance(r, tuple) else r
    g = torch.autograd.grad(o.sum(), list(leaves.values()), create_graph=True)
    with pytest.raises(RuntimeError):
        sum(t.square().sum() for t in g).backward()
