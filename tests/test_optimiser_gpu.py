"""optim.AdamW on the GPU: captures, counts and numbers of elements as they reach the kernels."""
import pytest
import torch

from vig_amd import optim

from .util import announce

pytestmark = pytest.mark.gpu


def made(*shapes, dtype=torch.float32):
    gen = torch.Generator(device="cuda").manual_seed(sum(len(s) for s in shapes))
    return [torch.nn.Parameter(torch.randn(s, device="cuda", generator=gen).to(dtype)) for s in shapes]


def give(*ps, seed=1):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    for p in ps:
        p.grad = torch.randn(p.shape, device="cuda", generator=gen).to(p.dtype)


def test_captures_that_replay_something_else():
    """Refused while nothing is recorded yet; the step that follows outside is as if they had not been tried."""
    announce("captured steps that are refused")
    a, b, c = made((5000,), (3,), (4,))
    opt = optim.AdamW([{"params": [a, b], "capturable": True}, {"params": [c]}], lr=0.1, max_norm=1.0)
    give(a)
    opt.step()
    for more, words in ((c, "capturable"), (b, "outside of the capture")):
        give(a, more)
        before = a.detach().clone()
        torch.cuda.synchronize()
        with pytest.raises(RuntimeError, match=words):
            with torch.cuda.graph(torch.cuda.CUDAGraph()):
                opt.step()
        torch.cuda.synchronize()
        assert torch.equal(a, before) and not opt.state.get(more) and int(opt.param_groups[0]["step_on_device"]["cuda:0"]) == 1
        more.grad = None
    opt.step()
    assert not torch.equal(a, before)
