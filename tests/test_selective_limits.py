"""Sizes of the selective scan beyond a launch's threads: refused before a workspace is asked for, and only where a launch of that call is meant."""
from .test_selective_refusals import _lib_or_skip, scan_call
from vig_amd import _lib


def test_what_does_not_fit_a_launch_is_refused_first():
    lib = _lib_or_skip()
    many = dict(batch=1 << 26, L=1, width=64)  # as many workgroups of the walk
    assert scan_call(lib, **many, kept=None) == scan_call(lib, **many) == scan_call(lib, True, **many) == _lib.VIG_ENOTSUP
    assert lib.vig_selective_scan_fwd_workspace(1 << 26, 1, 64, 4, 1) == lib.vig_selective_scan_bwd_workspace(1 << 26, 1, 64, 4, 1) == 0


def test_the_sum_of_shared_gradients_bounds_training_alone():
    """2^34 numbers of dB: past the launch that adds them up, also for a forward that keeps states for it; not for any other forward, which goes on to ask for its workspace."""
    lib = _lib_or_skip()
    large = dict(batch=1, L=1 << 24, width=16, N=64, G=16)
    assert scan_call(lib, True, **large) == scan_call(lib, **large) == _lib.VIG_ENOTSUP
    assert scan_call(lib, **large, kept=None) == _lib.VIG_ENOSPC and lib.vig_selective_scan_fwd_workspace(1, 1 << 24, 16, 64, 16) > 0
    half = large | dict(L=(1 << 23) - 8192)
    assert scan_call(lib, True, **half) == scan_call(lib, **half) == _lib.VIG_ENOSPC
