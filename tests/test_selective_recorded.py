"""The selective mixer's operators under a trace: what is recorded computes on new inputs, with gradients too; shapes without data."""
import pytest
import torch
from torch.fx.experimental.proxy_tensor import make_fx

import vig_amd
from vig_amd import _ext, _lib

from .test_selective_refusals import CALLS
from .util import announce

pytestmark = pytest.mark.filterwarnings("ignore::torch.jit.TracerWarning")


def outputs(call, given):
    r = getattr(vig_amd, call)(**given)
    kept = [given["state"]] if "state" in given else []
    return [t for t in (r if isinstance(r, tuple) else (r,)) if t is not None] + kept


@pytest.fixture(params=["cuda", "ctypes"])
def way(request, monkeypatch):
    if request.param == "ctypes":
        monkeypatch.setattr(_ext, "calls", lambda: None)
    return request.param


@pytest.mark.gpu
@pytest.mark.parametrize("how", ["trace", "fx"])
@pytest.mark.parametrize("call", list(CALLS))
def test_a_record_computes_on_new_inputs(call, how, way):
    announce(f"{call} recorded by {how}, {way}")
    names = list(CALLS[call]("cuda"))

    def f(*ts):
        given = {k: t.clone() if k == "state" else t for k, t in zip(names, ts)}
        return outputs(call, given)

    args = list(CALLS[call]("cuda").values())
    r = torch.jit.trace(f, tuple(args), check_trace=False) if how == "trace" else make_fx(f)(*args)
    for _ in range(2):
        args = list(CALLS[call]("cuda").values())
        for a, b in zip(r(*args), f(*args)):
            assert torch.equal(a, b)


@pytest.mark.gpu
@pytest.mark.parametrize("call", ["selective_scan", "causal_conv1d", "add_layernorm"])
def test_recorded_gradients(call, way):
    announce(f"{call}, recorded gradients, {way}")
    names = list(CALLS[call]("cuda"))

    def grads(*ts):
        leaves = [t.detach().requires_grad_() for t in ts]
        return torch.autograd.grad(sum(t.cos().sum() for t in outputs(call, dict(zip(names, leaves)))), leaves)

    r = make_fx(grads)(*CALLS[call]("cuda").values())
    args = list(CALLS[call]("cuda").values())
    assert all(torch.equal(a, b) for a, b in zip(r(*args), grads(*args)))


@pytest.mark.parametrize("N", [1, 5, 16, 33, 64])
@pytest.mark.parametrize("L", [1, 16, 17, 100])
def test_shapes_of_what_is_kept(L, N):
    """What a trace believes of the kept states is what the library asks for."""
    from vig_amd.selective import _kept_like

    x = torch.empty(3, L, 10, device="meta")
    assert _kept_like(x, N).numel() == _lib.load().vig_selective_scan_kept(3, L, 10, N)
