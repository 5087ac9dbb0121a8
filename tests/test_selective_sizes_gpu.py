"""The selective scan at sizes and addresses at the edge of what is documented."""
import pytest
import torch

import vig_amd
from vig_amd import _ext

from . import selective_ref as R
from .test_selective_gpu import BF16, make, roundings
from .util import announce

pytestmark = pytest.mark.gpu


def test_two_to_the_31_numbers_of_b():
    """8192 sequences of 4096 tokens with 64 states: B and C of 2^31 numbers (one sequence's, for all of them), their gradients and their partial sums of 2^32 beside them.  The sequences are
    alike, and so is what they give; the first is compared with 64 bits."""
    announce("selective scan, 8192 x 4096 x 1, N 64")
    batch, L = 8192, 4096
    one = make(21, 1, L, 1, 64, dtype=BF16, strong=0.1)
    rows = ("x", "delta", "B", "C", "z")
    given = {k: t.expand(batch, -1, -1).detach().requires_grad_() if k in rows else t for k, t in one.items()}
    with torch.no_grad():
        alone = vig_amd.selective_scan(**given)[0]
    o, _ = vig_amd.selective_scan(**given)
    assert torch.equal(o, alone)
    d_o = torch.randn(1, L, 1, device="cuda", generator=torch.Generator(device="cuda").manual_seed(22)).to(BF16)
    grads = torch.autograd.grad(o, [given[k] for k in rows], d_o.expand(batch, -1, -1))
    want, size = (R.scan(**one, d_o=d_o, mag=m) for m in (False, True))
    for name, t, n in [("o", o.detach(), roundings(one, L)), *(("d" + k, g, roundings(one, L, True)) for k, g in zip(rows, grads))]:
        R.close(t[:1], want[name], size[name], n, name)
        for at in range(0, batch, 1024):
            assert bool((t[at:at + 1024] == t[:1]).all()), name


@pytest.mark.parametrize("native", [True, False])
def test_groups_far_apart_in_one_token(native, monkeypatch):
    """One token's B and C, taken out of [B, G, L, N]: groups as far apart as a sequence is long."""
    announce(f"selective scan, groups 2^19 elements apart, native {native}")
    if not native:
        monkeypatch.setattr(_ext, "calls", lambda: None)
    t = make(23, 2, 1, 6, 16, G=2, state=True)
    room = torch.randn(2, 2, 1 << 15, 16, device="cuda")
    want = vig_amd.selective_scan(**t, output_final_state=True)
    for k in "BC":
        far = room.clone()[:, :, 77:78].permute(0, 2, 1, 3)
        far.copy_(t[k])
        assert far.stride(2) == 1 << 19
        t[k] = far
    got = vig_amd.selective_scan(**t, output_final_state=True)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    with torch.no_grad():
        state = t["initial_state"].clone()
        step = {k: t[k][:, 0] for k in ("x", "delta", "B", "C", "z")}
        o = vig_amd.selective_scan_step(**step, A=t["A"], state=state, D=t["D"], delta_bias=t["delta_bias"], delta_softplus=True)
    want, size = (R.scan(**t, mag=m) for m in (False, True))
    R.close(o, want["o"][:, 0], size["o"][:, 0], roundings(t, 1), "o"), R.close(state, want["final"], size["final"], roundings(t, 1), "state")
