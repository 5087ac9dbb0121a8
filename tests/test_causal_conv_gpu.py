"""The short causal convolution and its step against the sum in 64 bits.

Roundings: W + 1 of the sum, 8 of the activation and its derivative, |pre| in its exponent; W + 1 more for a row's gradient; a weight's gradient is added up over all tokens of all
sequences, at most that many roundings."""
import pytest
import torch

import vig_amd

from . import selective_ref as R
from .util import announce

pytestmark = pytest.mark.gpu

F32, BF16 = torch.float32, torch.bfloat16


def make(seed, batch, L, width, W, dtype=F32, bias=True, state=False, wide=0):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    r = lambda *s: torch.randn(*s, device="cuda", generator=gen)  # noqa: E731
    x = r(batch, L, width + wide).to(dtype)[..., wide // 2:wide // 2 + width]
    return {"x": x, "weight": r(width, W), "bias": r(width) if bias else None, "initial_state": r(batch, W - 1, width).to(dtype) if state else None}


def check(t, act, reverse=False, final=False, grads=False, params=True):
    names = [k for k in ("x", "weight", "bias", "initial_state") if t[k] is not None and (params or k in ("x", "initial_state"))]
    given = t | ({k: t[k].detach().requires_grad_() for k in names} if grads else {})
    y, h = vig_amd.causal_conv1d(given["x"], given["weight"], given["bias"], act, given["initial_state"], final, reverse)
    gen = torch.Generator(device="cuda").manual_seed(77)
    dy = torch.randn(y.shape, device="cuda", generator=gen).to(y.dtype) if grads else None
    dh = torch.randn(h.shape, device="cuda", generator=gen).to(h.dtype) if grads and final else None
    want, size = (R.conv(**t, act=act, reverse=reverse, dy=dy, d_final=dh, mag=m) for m in (False, True))
    W, (batch, L, _) = t["weight"].shape[1], t["x"].shape
    n = W + 10 + float(size["y"].max())
    R.close(y, want["y"], size["y"], n, "y")
    if final:
        assert torch.equal(R.f64(h), want["final"])
    if not grads:
        return
    got = torch.autograd.grad([y] + [h] * final, [given[k] for k in names], [dy] + [dh] * final)
    for k, g in zip(names, got):
        key = "dinitial" if k == "initial_state" else "d" + k
        R.close(g, want[key], size[key], n + W + 2 + (batch * L if k in ("weight", "bias") else 0), key)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("W", [2, 3, 4])
@pytest.mark.parametrize("shape", [(1, 1, 1), (2, 1, 16), (3, 2, 5), (2, 3, 64), (1, 17, 33), (2, 100, 136), (1, 70, 130), (2, 1030, 24), (40, 65, 200)])
def test_sizes(shape, W, dtype):
    announce(f"causal conv {shape} W {W} {dtype}")
    batch, L, width = shape
    for state in (False, True):
        t = make(1, batch, L, width, W, dtype, state=state)
        check(t, act=state, final=state, grads=True)
        check(t, act=not state, reverse=True, final=state, grads=True)
        check(t, act=True, final=True)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("wide", [8, 3, 64])
def test_columns_of_wider_rows(wide, dtype):
    announce(f"causal conv, columns {wide} {dtype}")
    check(make(2, 3, 50, 48, 4, dtype, wide=wide, state=True), act=True, final=True, grads=True)
    check(make(2, 3, 50, 48, 4, dtype, wide=wide, bias=False), act=True, grads=True, params=False)


def test_weights_as_torch_has_them():
    """[D, 1, W] and bf16 parameters, against torch's convolution of the same numbers."""
    announce("causal conv, torch's weight")
    t = make(3, 2, 30, 24, 4)
    m = torch.nn.Conv1d(24, 24, 4, groups=24, padding=3).cuda().bfloat16()
    y = vig_amd.causal_conv1d(t["x"], m.weight, m.bias)[0]
    (g,) = torch.autograd.grad(y, m.weight, torch.ones_like(y))
    want, size = (R.conv(t["x"], m.weight.squeeze(1), m.bias, dy=torch.ones_like(y), mag=k) for k in (False, True))
    R.close(y, want["y"], size["y"], 20, "y")
    assert g.shape == m.weight.shape and g.dtype == torch.bfloat16
    R.close(g.squeeze(1), want["dweight"], size["dweight"], 80, "dweight")


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("W,width,wide", [(2, 1, 0), (3, 17, 0), (4, 64, 0), (4, 64, 7), (4, 768, 768)])
def test_step(W, width, wide, dtype):
    announce(f"causal conv step W {W} width {width} wide {wide} {dtype}")
    t = make(4, 5, 9, width, W, dtype, state=True, wide=wide)
    whole, last = vig_amd.causal_conv1d(t["x"], t["weight"], t["bias"], True, t["initial_state"], True)
    state = t["initial_state"].clone()
    for k in range(9):
        version = state._version
        y = vig_amd.causal_conv1d_step(t["x"][:, k], t["weight"], state, t["bias"], True)
        assert torch.equal(y, whole[:, k]) and state._version > version
    assert torch.equal(state, last)


def test_same_bits_again():
    announce("causal conv, repeated")
    t = make(5, 8, 300, 200, 4, BF16)
    given = {k: t[k].detach().requires_grad_() for k in ("x", "weight", "bias")}

    def run():
        y = vig_amd.causal_conv1d(**given, silu=True)[0]
        return (y.detach(), *torch.autograd.grad(y, list(given.values()), torch.ones_like(y)))

    assert all(torch.equal(a, b) for a, b in zip(run(), run()))
