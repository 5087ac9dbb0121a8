"""The add and layer norm of as many rows as it takes."""
import pytest
import torch

import vig_amd

from . import selective_ref as R
from .test_add_norm_gpu import BF16, N
from .util import announce

pytestmark = pytest.mark.gpu


def test_two_to_the_24_rows_of_a_workgroup_each():
    """34 GB in and 34 out: rows of zeros, whose norm is the bias, and a few others on the edges of the launches' pieces."""
    rows, C = 1 << 24, 1025
    announce(f"layer norm, {rows} rows of {C}")
    gen = torch.Generator(device="cuda").manual_seed(41)
    x = torch.zeros(rows, C, device="cuda", dtype=BF16)
    some = [0, 1, (1 << 23) - 1, 1 << 23, rows - 2, rows - 1]
    x[some] = torch.randn(len(some), C, device="cuda", generator=gen).to(BF16)
    w, b = (torch.randn(C, device="cuda", generator=gen) for _ in range(2))
    y = vig_amd.add_layernorm(x, w, b)
    R.close(y[some], *R.norm(x[some], w, b)["y"], N, "y")
    plain = b.to(BF16)
    y[some] = plain
    for at in range(0, rows, 1 << 20):
        assert bool((y[at:at + (1 << 20)] == plain).all()), f"rows from {at} on"
    del x, y
    torch.cuda.empty_cache()
