"""Residual add and layer norm against the formula in 64 bits.

Roundings: a row's sums over C elements are added up in trees of lanes over runs of a thread, at most 64 + 16 + 8 of them on a way; the mean, the square, the root and the products
16 more; a gradient takes two such sums: 2 (88 + 16).  Weight and bias: over the rows too, at most their number."""
import pytest
import torch

import vig_amd

from . import selective_ref as R
from .util import announce

pytestmark = pytest.mark.gpu

F32, BF16 = torch.float32, torch.bfloat16
N = 104


def make(seed, lead, C, dtype, residual=None, bias=True, far=0.0):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    r = lambda *s: torch.randn(*s, device="cuda", generator=gen)  # noqa: E731
    return {"x": (r(*lead, C) + far).to(dtype), "weight": 1 + 0.2 * r(C), "bias": r(C) if bias else None, "residual": (2 * r(*lead, C)).to(residual) if residual else None}


def check(t, grads, prenorm=True, eps=1e-5, use_sum=True):
    names = [k for k in ("x", "weight", "bias", "residual") if t[k] is not None]
    given = t | ({k: t[k].detach().requires_grad_() for k in names} if grads else {})
    y = vig_amd.add_layernorm(given["x"], given["weight"], given["bias"], eps, given["residual"], prenorm)
    y, total = y if prenorm else (y, None)
    gen = torch.Generator(device="cuda").manual_seed(5)
    dy = torch.randn(y.shape, device="cuda", generator=gen).to(y.dtype)
    both = grads and prenorm and use_sum
    d_sum = torch.randn(total.shape, device="cuda", generator=gen).to(total.dtype) if both else None
    want = R.norm(**t, eps=eps, dy=dy, d_sum=d_sum)
    rows = t["x"].numel() // t["x"].shape[-1]
    R.close(y, *want["y"], N, "y")
    if prenorm:
        assert total.dtype == (t["residual"] if t["residual"] is not None else t["x"]).dtype
        assert torch.equal(R.f64(total), want["sum"][0])
    if not grads:
        return
    got = torch.autograd.grad([y] + [total] * both, [given[k] for k in names], [dy] + [d_sum] * both)
    for k, g in zip(names, got):
        assert g.dtype == t[k].dtype and g.shape == t[k].shape
        # (without a residual the sum is x itself, to which autograd adds its gradient, in x's dtype)
        extra = R.HALF[g.dtype] * want["d" + k][1] / R.U if k == "x" and both and t["residual"] is None else 0
        R.close(g, *want["d" + k], 2 * N + (rows if k in ("weight", "bias") else 0) + extra, "d" + k)


@pytest.mark.parametrize("kinds", [(F32, None), (BF16, None), (F32, F32), (BF16, BF16), (BF16, F32)])
@pytest.mark.parametrize("C", [1, 2, 7, 8, 63, 192, 256, 264, 384, 500, 512, 768, 999, 1024, 1032, 2048, 2056, 4095, 4096, 4104, 8192, 16383, 16384])
def test_widths(C, kinds):
    announce(f"add and layer norm C {C} {kinds}")
    t = make(C, (3, 5), C, *kinds)
    check(t, grads=False)
    check(t, grads=True)
    check(t, grads=True, prenorm=False)
    check(t, grads=True, use_sum=False)


@pytest.mark.parametrize("rows", [1, 2, 9, 1000, 5003])
@pytest.mark.parametrize("C", [40, 384, 129])
def test_rows(rows, C):
    announce(f"add and layer norm {rows} rows of {C}")
    check(make(rows, (rows,), C, BF16, F32), grads=True)
    check(make(rows, (rows,), C, F32, None, bias=False), grads=True, prenorm=False)


def test_far_from_zero():
    """A mean that is many times the deviation: the square's sum is taken of distances."""
    announce("layer norm, a large mean")
    t = make(1, (64,), 768, F32, far=300.0)
    y = vig_amd.add_layernorm(t["x"], t["weight"], t["bias"])
    want = R.norm(**t)
    R.close(y, *want["y"], N, "y")
    assert float((R.f64(y) - want["y"][0]).abs().max()) < 300 * N * R.U * 2


def test_rows_of_one_value_and_of_huge_ones():
    announce("layer norm, rows without deviation")
    x = torch.full((4, 64), 3.0, device="cuda")
    w, b = torch.full((64,), 2.0, device="cuda"), torch.arange(64.0, device="cuda")
    assert torch.equal(vig_amd.add_layernorm(x, w, b), b.expand(4, 64))
    x[1, 3] = float("nan")
    y = vig_amd.add_layernorm(x, w, b)
    assert bool(y[1].isnan().all()) and torch.equal(y[2:], b.expand(2, 64))


def test_any_address_and_order():
    announce("layer norm, views")
    t = make(2, (6, 50), 24, BF16, BF16)
    room = torch.zeros(6 * 50 * 24 + 1, device="cuda", dtype=BF16)
    odd = room[1:].view(6, 50, 24)
    odd.copy_(t["x"])
    y = vig_amd.add_layernorm(t["x"], t["weight"], t["bias"], residual=t["residual"])
    R.close(vig_amd.add_layernorm(odd, t["weight"], t["bias"], residual=t["residual"]), *R.norm(**t)["y"], N, "odd address")
    turned = t["x"].transpose(0, 1).contiguous().transpose(0, 1)
    assert torch.equal(vig_amd.add_layernorm(turned, t["weight"], t["bias"], residual=t["residual"]), y)


def test_same_bits_again():
    announce("layer norm, repeated")
    t = make(3, (3000,), 768, BF16, F32)
    given = {k: t[k].detach().requires_grad_() for k in ("x", "weight", "bias", "residual")}

    def run():
        y, s = vig_amd.add_layernorm(**given, prenorm=True)
        return (y.detach(), s.detach(), *torch.autograd.grad([y, s], list(given.values()), [torch.ones_like(y), torch.ones_like(s)]))

    assert all(torch.equal(a, b) for a, b in zip(run(), run()))


@pytest.mark.parametrize("rows", [511, 512, 513, 1023, 1024, 1025])
@pytest.mark.parametrize("C", [256, 257, 513, 520, 768, 1024, 1025, 2048])
def test_lone_rows(rows, C):
    """Where a row goes from a workgroup of its own to a wave, for rows in whole pieces and others; the backward keeps its form on both sides."""
    announce(f"add and layer norm {rows} rows of {C}")
    check(make(rows + C, (rows,), C, BF16, BF16), grads=True)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_gradients_of_the_summands_lie_apart(dtype):
    """x and the residual get the same gradient where their types are alike, and neither changes with the other's."""
    announce(f"add and layer norm, gradients of both summands, {dtype}")
    t = make(3, (4,), 64, dtype, dtype)
    x, residual = t["x"].requires_grad_(), t["residual"].requires_grad_()
    y, total = vig_amd.add_layernorm(x, t["weight"], t["bias"], residual=residual, prenorm=True)
    torch.autograd.backward([y, total], [torch.randn_like(y), torch.randn_like(total)])
    assert torch.equal(x.grad, residual.grad)
    before = residual.grad.clone()
    x.grad.mul_(2)
    assert torch.equal(residual.grad, before)


@pytest.mark.parametrize("rows,C", [(8192, 264), (8200, 257), (11999, 40), (12001, 40), (12001, 1032), (8193, 1501), (513, 4104)])
def test_many_rows(rows, C):
    """As many partial sums of the parameters' gradients as there are at most, for rows in whole pieces and others."""
    announce(f"add and layer norm {rows} rows of {C}")
    check(make(rows + C, (rows,), C, BF16, BF16), grads=True)
