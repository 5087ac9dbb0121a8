"""add_layernorm adds x to a residual, and both get the same gradient.  Two leaves behind them never share a buffer, however they reach the call: a second backward pass adds to each gradient
once.  (Views hand a gradient's memory on, and what arrives at a leaf is kept as it is where nobody else holds that tensor: two tensors over one memory would both be kept.)"""
import pytest
import torch

import vig_amd
from vig_amd import _ext

from .util import announce

pytestmark = pytest.mark.gpu

ROWS, C = 6, 64
FORMS = {"leaf": lambda p: p, "view": lambda p: p.view(ROWS, C), "sum": lambda p: p + 1, "view and sum": lambda p: p.view(ROWS, C) + 1, "turned": lambda p: p.t().t().view(2, 3, C).flatten(0, 1)}
LIKE = {"leaf": (ROWS, C), "view": (ROWS * C,), "sum": (ROWS, C), "view and sum": (ROWS * C,), "turned": (ROWS, C)}


@pytest.mark.parametrize("native", [True, False])
@pytest.mark.parametrize("dtype,held", [(torch.float32, torch.float32), (torch.bfloat16, torch.bfloat16), (torch.bfloat16, torch.float32)])
@pytest.mark.parametrize("x_form", list(FORMS))
@pytest.mark.parametrize("r_form", list(FORMS))
def test_two_passes_add_twice(x_form, r_form, dtype, held, native, monkeypatch):
    announce(f"add and layer norm, x {x_form} {dtype}, residual {r_form} {held}, native {native}")
    if not native:
        monkeypatch.setattr(_ext, "calls", lambda: None)
    gen = torch.Generator(device="cuda").manual_seed(1)
    p = torch.randn(LIKE[x_form], device="cuda", generator=gen).to(dtype).requires_grad_()
    q = torch.randn(LIKE[r_form], device="cuda", generator=gen).to(held).requires_grad_()
    w, dy = torch.randn(C, device="cuda", generator=gen), torch.randn(ROWS, C, device="cuda", generator=gen).to(dtype)

    def one():
        y, total = vig_amd.add_layernorm(FORMS[x_form](p), w, residual=FORMS[r_form](q), prenorm=True)
        torch.autograd.backward([y, total], [dy, torch.ones_like(total)])

    one()
    first = [t.grad.clone() for t in (p, q)]
    one()
    assert p.grad.untyped_storage().data_ptr() != q.grad.untyped_storage().data_ptr()
    for t, g in zip((p, q), first):  # (twice a number has its digits)
        assert torch.equal(t.grad, 2 * g)


@pytest.mark.parametrize("native", [True, False])
@pytest.mark.parametrize("who", ["x", "residual", "both", "the same"])
def test_whoever_wants_a_gradient_gets_the_sums(who, native, monkeypatch):
    """The gradient of one summand alone, of both, of a tensor added to itself."""
    announce(f"add and layer norm, gradient of {who}, native {native}")
    if not native:
        monkeypatch.setattr(_ext, "calls", lambda: None)
    gen = torch.Generator(device="cuda").manual_seed(2)
    x, r, dy, ds = (torch.randn(ROWS, C, device="cuda", generator=gen) for _ in range(4))
    w = torch.randn(C, device="cuda", generator=gen)
    given = (x, x) if who == "the same" else (x, r)
    both = [t.detach().requires_grad_() for t in given]
    y, total = vig_amd.add_layernorm(both[0], w, residual=both[1], prenorm=True)
    want = torch.autograd.grad([y, total], both, [dy, ds])
    assert torch.equal(*want)
    a = x.detach().requires_grad_(who != "residual")
    b = a if who == "the same" else r.detach().requires_grad_(who != "x")
    y, total = vig_amd.add_layernorm(a, w, residual=b, prenorm=True)
    torch.autograd.backward([y, total], [dy, ds])
    if who == "the same":
        assert torch.equal(a.grad, 2 * want[0])
    else:
        assert all(t.grad is None if not t.requires_grad else torch.equal(t.grad, g) for t, g in zip((a, b), want))
