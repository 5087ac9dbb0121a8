"""What is neither true nor false, and who speaks in a refusal."""
import pytest
import torch

import vig_amd
from vig_amd import _ext

from .test_selective_refusals import CALLS
from .util import announce

pytestmark = pytest.mark.gpu

FLAGS = [("selective_scan", "delta_softplus"), ("selective_scan", "reverse"), ("selective_scan", "output_final_state"), ("selective_scan_step", "delta_softplus"), ("causal_conv1d", "silu"),
         ("causal_conv1d", "reverse"), ("causal_conv1d", "output_final_state"), ("causal_conv1d_step", "silu")]


@pytest.mark.parametrize("native", [True, False])
@pytest.mark.parametrize("call,flag", FLAGS)
def test_a_flag_without_a_truth(call, flag, native, monkeypatch):
    announce(f"{call}, {flag} of two numbers, native {native}")
    if not native:
        monkeypatch.setattr(_ext, "calls", lambda: None)
    t = CALLS[call]("cuda")
    before = t["state"].clone() if "state" in t else None
    with pytest.raises(RuntimeError, match="ambiguous"):
        getattr(vig_amd, call)(**t, **{flag: torch.tensor([True, False])})
    assert before is None or torch.equal(t["state"], before)


@pytest.mark.parametrize("call", ["selective_scan", "causal_conv1d", "add_layernorm"])
def test_a_refused_capture_names_its_call(call, monkeypatch):
    announce(f"{call}, leaves in a capture without the native calls")
    monkeypatch.setattr(_ext, "calls", lambda: None)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
    leaves = {k: t.requires_grad_() for k, t in CALLS[call]("cuda").items()}
    with pytest.raises(RuntimeError, match=f"^{call}: .*capture"):
        getattr(vig_amd, call)(**leaves)
