"""The selective scan at sizes and addresses at the edge of what is documented."""
import pytest
import torch

import vig_amd

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
