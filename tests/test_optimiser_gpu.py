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


@pytest.mark.parametrize("bits", [8, 32])
def test_counts_of_a_captured_step(bits):
    """Parameters that joined at different steps, captured and replayed: each goes by its own count, as it does counted on the host."""
    announce(f"captured counts, states in {bits} bits")
    both = [made((5000,), (3,), (70, 64)) for _ in range(2)]
    ref, opt = (optim.AdamW(ps, lr=0.01, state_bits=bits, capturable=c) for ps, c in zip(both, (False, True)))
    plan = [(0, 2), (0, 1, 2), (0, 2)] + [(0, 1, 2)] * 5
    graph = torch.cuda.CUDAGraph()
    for i, some in enumerate(plan):
        for ps in both:
            for p in ps:
                p.grad = p.grad if i > 4 else None
        gen = torch.Generator(device="cuda").manual_seed(i)
        for j in some:
            g = torch.randn(both[0][j].shape, device="cuda", generator=gen)
            for ps in both:
                if i > 4:
                    ps[j].grad.copy_(g)
                else:
                    ps[j].grad = g.clone()
        ref.step()
        if i < 4:
            opt.step()
            continue
        if i == 4:
            torch.cuda.synchronize()
            with torch.cuda.graph(graph):
                opt.step()
        graph.replay()
        torch.cuda.synchronize()
    assert [int(opt.state[p]["step"]) for p in both[1]] == [ref.state[p]["step"] for p in both[0]] == [8, 6, 8]
    assert len(opt.param_groups[0]["step_on_device"]) == 2
    for p, q in zip(*both):
        # (the corrections of either way agree but for a rounding of 24 bits, which may turn codes of 8 bits over: a step of one is up to 1/8 of a moment, and a move is about lr)
        off = float((p - q).detach().abs().max())
        assert off <= (8 * 4 * 2.0 ** -24 * float(q.detach().abs().max()) if bits == 32 or p.numel() == 3 else 8 * 0.01 / 4)
