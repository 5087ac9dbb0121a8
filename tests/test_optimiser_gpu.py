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


@pytest.mark.parametrize("bits", [8, 32])
def test_groups_of_equal_tensors_are_rounded_apart(bits):
    """The same weights and gradients in two groups: the same update before the rounding, another one after it; and as one list whose numbers are given."""
    announce(f"rounding over groups, states in {bits} bits")
    w = made((5000,), dtype=torch.bfloat16)[0].detach()
    ps = [torch.nn.Parameter(w.clone()) for _ in range(3)]
    opt = optim.AdamW([{"params": ps[:1]}, {"params": ps[1:]}], lr=1e-3, state_bits=bits, seed=5)
    for p in ps:
        give(p)
    opt.step()
    step = torch.exp2(torch.floor(torch.log2(w.float().abs() * 1.01 + 2e-3)) - 7)  # of bf16, the larger one at a border
    for p, q in ((ps[0], ps[1]), (ps[1], ps[2]), (ps[0], ps[2])):
        off = (p - q).detach().float().abs()
        # (a move of 1e-3 and a decay of 1e-5 are not bf16's steps of about 4e-3: most elements are rounded, one way or the other)
        assert bool((off <= step).all()) and float((off > 0).float().mean()) > 0.05
    alone = [torch.nn.Parameter(w.clone()) for _ in range(3)]
    other = optim.AdamW(alone, lr=1e-3, state_bits=bits, seed=5)
    for p in alone:
        give(p)
    other.step()
    assert all(torch.equal(p, q) for p, q in zip(ps, alone))
