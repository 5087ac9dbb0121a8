"""What the gated scan, the update and the gradients' norm refuse before anything reaches the GPU (none is needed)."""
import ctypes
import os

import pytest
import torch

import vig_amd
from vig_amd import _lib, optim

INVALID, UNBUILT, SPACE = _lib.VIG_EINVAL, _lib.VIG_ENOTSUP, _lib.VIG_ENOSPC
P = 1 << 20  # addresses of nothing: a refused call never reads them


@pytest.fixture()
def lib():
    if not os.path.exists(_lib.LIB_PATH):
        pytest.skip("library not built here")
    return _lib.load()


def _strides(*v):
    return (ctypes.c_longlong * 2)(*v)


def test_scan(lib):
    def fwd(x=P, gf=2 * P, gb=None, h0=None, o=3 * P, hT=None, ws=None, n=0, B=2, L=9, D=8, xs=None, gs=None, io=1, gd=1):
        return lib.vig_gated_scan_fwd(x, gf, gb, h0, o, hT, ws, n, B, L, D, xs, gs, 1.0, io, gd, None)

    for bad in (dict(x=None), dict(gf=None), dict(o=None), dict(o=P), dict(o=2 * P), dict(gb=3 * P), dict(B=0), dict(L=0), dict(D=-1), dict(x=P + 1), dict(o=3 * P + 1), dict(gf=2 * P + 2, gd=0),
                dict(gb=5 * P, h0=4 * P), dict(gb=5 * P, hT=4 * P), dict(h0=4 * P + 2), dict(h0=4 * P, hT=4 * P), dict(xs=_strides(72, 7)), dict(gs=_strides(72, 0)), dict(xs=_strides(-1, 8)),
                dict(L=5000, ws=P + 8, n=1 << 30)):
        assert fwd(**bad) == INVALID, bad
    for unbuilt in (dict(io=2), dict(gd=-1), dict(D=(1 << 18) + 1), dict(L=(1 << 30) + 1), dict(xs=_strides(0, (1 << 18) + 1)), dict(B=1, L=1 << 30, D=1 << 18, ws=4 * P, n=1 << 62)):
        assert fwd(**unbuilt) == UNBUILT, unbuilt
    need = lib.vig_gated_scan_fwd_workspace(2, 5000, 8, 0)
    assert need > 0 and lib.vig_gated_scan_fwd_workspace(2, 5000, 8, 1) == 2 * need and lib.vig_gated_scan_bwd_workspace(2, 5000, 8, 1) == 4 * need
    assert fwd(L=5000) == fwd(L=5000, ws=4 * P, n=need - 1) == SPACE
    assert lib.vig_gated_scan_fwd_workspace(0, 5000, 8, 0) == lib.vig_gated_scan_fwd_workspace(1, -1, 8, 0) == lib.vig_gated_scan_bwd_workspace(1, 1, 1 << 20, 0) == 0

    def bwd(x=P, gf=2 * P, gb=None, h0=None, do=3 * P, dT=None, dx=4 * P, df=5 * P, db=None, d0=None, ws=None, n=0, B=2, L=9, D=8, io=1, gd=1):
        return lib.vig_gated_scan_bwd(x, gf, gb, h0, do, dT, dx, df, db, d0, ws, n, B, L, D, None, None, 1.0, io, gd, None)

    for bad in (dict(do=None), dict(dx=None), dict(df=None), dict(gb=6 * P), dict(db=6 * P), dict(dx=P), dict(dx=3 * P), dict(df=2 * P), dict(df=4 * P), dict(gb=6 * P, db=5 * P),
                dict(gb=6 * P, db=7 * P, d0=8 * P), dict(gb=6 * P, db=7 * P, dT=8 * P), dict(d0=8 * P, h0=8 * P), dict(d0=8 * P, dT=8 * P), dict(do=3 * P + 1), dict(dx=4 * P + 1), dict(d0=8 * P + 2)):
        assert bwd(**bad) == INVALID, bad
    assert bwd(L=5000) == SPACE and bwd(io=7) == UNBUILT

    def step(x=P, g=2 * P, h=3 * P, o=4 * P, B=2, D=8, xs=0, gs=0, io=1, gd=1):
        return lib.vig_gated_scan_step(x, g, h, o, B, D, xs, gs, io, gd, None)

    for bad in (dict(x=None), dict(g=None), dict(h=None), dict(o=None), dict(o=P), dict(o=2 * P), dict(o=3 * P), dict(h=P), dict(h=2 * P), dict(B=0), dict(D=0), dict(xs=7), dict(gs=-8), dict(h=3 * P + 2), dict(x=P + 1)):
        assert step(**bad) == INVALID, bad
    for unbuilt in (dict(io=2), dict(gd=3), dict(B=1 << 16, D=1 << 15)):
        assert step(**unbuilt) == UNBUILT, unbuilt


def _update(lib, p, g, m, v, n, ms=None, vs=None, types=None, bits=32, step=1, b1=0.9, b2=0.999, eps=1e-8, scale=None, step_at=None, lr_at=None, first=None):
    ptr = lambda a: (ctypes.c_void_p * len(a))(*a)  # noqa: E731
    dt = (ctypes.c_int * len(p))(*(types or [0] * len(p)))
    return lib.vig_adamw_many(ptr(p), ptr(g), ptr(m), ptr(v), ptr(ms) if ms else None, ptr(vs) if vs else None, (ctypes.c_longlong * len(p))(*n), (ctypes.c_longlong * len(p))(*first) if first else None, dt, dt, len(p), bits, 1e-3, b1, b2, eps,
                              0.0, step, lr_at, step_at, scale, 0, None)


def test_adamw(lib):
    good = ([P, 2 * P], [3 * P, 4 * P], [5 * P, 6 * P], [7 * P, 8 * P], [100, 300])
    for bad in (dict(step=0), dict(b1=1.0), dict(b1=-0.1), dict(b1=float("nan")), dict(b2=1.0), dict(b2=float("nan")), dict(eps=-1.0), dict(eps=float("nan")), dict(bits=8), dict(scale=P + 2), dict(step_at=P + 4), dict(first=[0, -1]),
                dict(lr_at=P + 1)):
        assert _update(lib, *good, **bad) == INVALID, bad
    assert _update(lib, *good, first=[0, (1 << 40) + 1]) == UNBUILT
    assert _update(lib, *good, bits=16) == _update(lib, *good, types=[0, 2]) == UNBUILT
    change = lambda k, v: [list(x) if i != k else v for i, x in enumerate(good)]  # noqa: E731
    assert _update(lib, *change(4, [100, -1])) == INVALID
    assert _update(lib, *change(4, [100, (1 << 40) + 1])) == UNBUILT and _update(lib, *change(4, [1 << 40, 1])) == UNBUILT
    for k, values in ((0, [P, None]), (1, [None, P]), (2, [5 * P, None]), (3, [7 * P, 8 * P + 2]), (0, [P + 2, 2 * P]),
                      (0, [P, P]), (0, [P, P + 396]), (0, [P, 3 * P]), (2, [P, 6 * P]), (3, [7 * P, 2 * P + 1196]), (1, [8 * P + 1196, 4 * P]), (2, [5 * P, 7 * P + 4])):
        assert _update(lib, *change(k, values)) == INVALID, (k, values)
    scales = dict(ms=[9 * P, 10 * P], vs=[11 * P, 12 * P], bits=8)
    for more in (dict(ms=[9 * P, None]), dict(vs=[11 * P + 1, 12 * P]), dict(ms=[9 * P, 11 * P]), dict(vs=[5 * P + 96, 12 * P])):
        assert _update(lib, *good, **(scales | more)) == INVALID, more
    assert lib.vig_adamw_many(None, None, None, None, None, None, None, None, None, None, 1, 32, 1e-3, 0.9, 0.999, 1e-8, 0.0, 1, None, None, None, 0, None) == INVALID


def test_grad_norm(lib):
    ptr, longs, ints = (lambda *v: (ctypes.c_void_p * 2)(*v)), (lambda *v: (ctypes.c_longlong * 2)(*v)), (lambda *v: (ctypes.c_int * 2)(*v))

    def norm(g=(P, 2 * P), n=(5, 9), types=(0, 1), most=1.0, out=3 * P, scale=4 * P, ws=5 * P, space=1 << 20):
        return lib.vig_grad_norm(ptr(*g), longs(*n), ints(*types), 2, most, out, scale, ws, space, None)

    for bad in (dict(g=(P, None)), dict(g=(P + 2, P)), dict(g=(P, P + 1)), dict(n=(5, -1)), dict(out=None), dict(out=4 * P), dict(scale=4 * P + 1), dict(most=-1.0), dict(most=float("nan")), dict(ws=5 * P + 4)):
        assert norm(**bad) == INVALID, bad
    assert norm(types=(0, 3)) == UNBUILT and norm(n=(1 << 40, 1)) == UNBUILT
    assert lib.vig_grad_norm_workspace(longs(8192, 8193), 2) == 24
    assert norm(ws=None) == norm(space=15) == SPACE


def test_python_side():
    x, g, h = torch.zeros(2, 3, 8), torch.zeros(2, 3, 8), torch.zeros(2, 8)
    for call in (lambda: vig_amd.gated_scan(x, g), lambda: vig_amd.bid_gated_scan(x, torch.cat([g, g])), lambda: vig_amd.gated_scan_step(h, h, h.clone()),
                 lambda: vig_amd.grad_norm([x]), lambda: vig_amd.adamw_step([x], [g], [x.clone()], [x.clone()], step=1)):
        with pytest.raises(_lib.VigGlaError):  # there is no CPU path
            call()
    with pytest.raises(ValueError):
        vig_amd.grad_norm([])
    with pytest.raises(ValueError):
        vig_amd.grad_norm([x], max_norm=-1.0)
    p = [torch.nn.Parameter(torch.zeros(3))]
    for bad in (dict(lr=-1.0), dict(betas=(1.0, 0.9)), dict(eps=-1.0), dict(weight_decay=-0.1), dict(state_bits=16), dict(max_norm=-1.0)):
        with pytest.raises(ValueError):
            optim.AdamW(p, **bad)


def test_words_spread():
    """The word of neighbouring elements and steps: every bit half of the time, and no bit of the input without a say in it."""
    M = 0xFFFFFFFF

    def mix(x):
        x = ((x ^ (x >> 16)) * 0x6A09E667) & M
        x = ((x ^ (x >> 15)) * 0xBB67AE85) & M
        return x ^ (x >> 16)

    import numpy as np

    n = 1 << 16
    x = np.arange(n, dtype=np.uint64)
    w = mix(x)
    bits = (w[:, None] >> np.arange(32, dtype=np.uint64)) & 1
    assert np.abs(bits.mean(0) - 0.5).max() < 5 * 0.5 / n ** 0.5
    for b in range(32):
        flipped = mix(x ^ np.uint64(1 << b)) ^ w
        change = ((flipped[:, None] >> np.arange(32, dtype=np.uint64)) & 1).mean(0)
        assert 0.05 < change.min() and change.max() < 0.95, b
    half = (w & 0xFFFF).astype(float) / 65536
    assert abs(half.mean() - 0.5) < 5 / (12 * n) ** 0.5 and abs(np.corrcoef(half[1:], half[:-1])[0, 1]) < 5 / n ** 0.5
