"""Loops that the sizes of a model go through more than once: the sum of dB and dC over a group's workgroups, runs of tokens of the short convolution, two sequences a thread of the step."""
import math

import pytest
import torch

import vig_amd

from . import selective_ref as R
from .test_causal_conv_gpu import check as check_conv, make as make_conv
from .test_selective_gpu import BF16, F32, check as check_scan, make as make_scan, roundings
from .util import announce

pytestmark = pytest.mark.gpu


@pytest.fixture
def gate_terms(monkeypatch):
    """The magnitude of dz by the terms of silu'(z) = s + z s (1 - s), s = 1 / (1 + e^-z), and not by their sum: near z = -1.278 they cancel.  At z = -1.2784892 (one of 21546 gates of 513
    channels) s = 0.2178075, z s (1 - s) = -0.2178129 and silu' = -5.4e-6, while each term is rounded by up to U = 2^-24 of itself: 2 x 0.2178 U, 8 10^4 U of the sum, where roundings() counts
    5604 of it.  (The kernel was 4.0e-10 off, 0.12 U of dy y (|s| + |z s (1 - s)|).)  As the other magnitudes are taken: every sum with absolute values in it."""
    whole = R.scan

    def scan(*args, mag=False, **given):
        out = whole(*args, mag=mag, **given)
        if mag and "dz" in out:
            z = R.f64(given["z"])
            s = torch.sigmoid(z)
            out["dz"] = out["dz"] / R.dsilu(z).abs() * s * (1 + z.abs() * (1 - s))
        return out

    monkeypatch.setattr(R, "scan", scan)


# 64 channels a workgroup, four workgroups' sums on their way together: 5, 6, 8, 9 and 12 of a group
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("width,N,G", [(257, 16, 1), (384, 16, 1), (512, 13, 1), (513, 5, 1), (768, 16, 1), (768, 40, 2), (1152, 3, 3)])
def test_groups_of_many_channels(width, N, G, dtype, gate_terms):
    announce(f"selective scan, {width} channels in {G} groups, N {N} {dtype}")
    check_scan(make_scan(31, 2, 21, width, N, G, dtype, state=True), final=True, grads=True)


# One group of runs for each 8192 tokens of all sequences, here one workgroup wide.  Tokens of a run, forward and backward: 5 and 5, 7 and 7,
# 13 and 13, 16 and 16, 16 and 63, 16 and 64, 15 and 60
@pytest.mark.parametrize("dtype,width", [(F32, 4), (F32, 3), (BF16, 8), (BF16, 5)])
@pytest.mark.parametrize("batch,L", [(512, 80), (512, 112), (512, 208), (34, 4096), (512, 1008), (64, 8192), (300, 1919)])
def test_long_runs(batch, L, dtype, width):
    announce(f"causal conv, {batch} sequences of {L} tokens, {width} channels {dtype}")
    W = 2 + (batch + L) % 3
    check_conv(make_conv(32, batch, L, width, W, dtype, state=True), act=True, final=True, grads=True)
    check_conv(make_conv(33, batch, L, width, W, dtype, bias=False), act=False, reverse=True, grads=True)


def test_long_runs_of_four_taps_reversed():
    announce("causal conv, 4 taps, long runs, reversed, columns of wider rows")
    check_conv(make_conv(34, 512, 1008, 8, 4, BF16, state=True, wide=8), act=True, reverse=True, final=True, grads=True)
    check_conv(make_conv(35, 65, 2050, 6, 4, F32, state=True, wide=3), act=True, reverse=True, final=True, grads=True)


# batch x channels x lanes of a channel (a quarter of N, as a power of two) of 524288 on: two sequences a thread
STEPS = [(170, 768, 16, 1), (171, 768, 16, 1), (172, 768, 16, 2), (171, 768, 12, 1), (171, 770, 13, 2), (683, 768, 1, 1), (341, 771, 6, 3), (43, 768, 64, 1), (87, 769, 17, 1)]


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("odd", [False, True])
@pytest.mark.parametrize("batch,width,N,G", STEPS)
def test_two_sequences_a_thread(batch, width, N, G, odd, dtype):
    """The state between guards, on 16 bytes or on an odd element."""
    announce(f"selective scan step, {batch} x {width}, N {N}, G {G}, odd address {odd}, {dtype}")
    t = make_scan(36, batch, 1, width, N, G, dtype, state=True, wide=odd)
    n, guard = batch * width * N, 4096
    room = torch.full((n + 2 * guard + 1,), math.pi, device="cuda")
    state = room[guard + odd:guard + odd + n].view(batch, width, N)
    state.copy_(t["initial_state"])
    with torch.no_grad():
        o = vig_amd.selective_scan_step(**{k: t[k][:, 0] for k in ("x", "delta", "B", "C", "z")}, A=t["A"], state=state, D=t["D"], delta_bias=t["delta_bias"], delta_softplus=True)
    want, size = (R.scan(**t, mag=m) for m in (False, True))
    R.close(o, want["o"][:, 0], size["o"][:, 0], roundings(t, 1), "o")
    R.close(state, want["final"], size["final"], roundings(t, 1), "state")
    assert bool((room[:guard + odd] == torch.tensor(math.pi)).all()) and bool((room[guard + odd + n:] == torch.tensor(math.pi)).all())
