"""Calls of the gated scan that have to be refused, on the GPU both ways and, with the library replaced by its formula, without one."""
import pytest
import torch
import torch.autograd.forward_ad as forward_ad

import vig_amd

from .test_recorded_calls import device, inputs  # noqa: F401
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
