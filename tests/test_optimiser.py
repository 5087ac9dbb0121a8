"""What optim.AdamW asks of the update and keeps beside it, with the update replaced by a record of its calls (no GPU is needed)."""
import copy

import pytest
import torch

from vig_amd import ops, optim

F32, BF16, E4M3 = torch.float32, torch.bfloat16, torch.float8_e4m3fn


@pytest.fixture
def calls(monkeypatch):
    """The calls of adamw_step as dicts, made to move the moments by one: what lies there is seen to be carried on."""
    seen = []

    def step(params, grads, avgs, sqs, avg_scales=None, sq_scales=None, **kw):
        kw["step"] = int(kw["step"])
        seen.append({"params": list(params), "avgs": list(avgs), "scales": avg_scales, **kw})
        for t in avgs + sqs:
            if t.dtype == F32:
                t += 1

    monkeypatch.setattr(ops, "adamw_step", step)
    return seen


def params(*shapes, dtype=F32):
    return [torch.nn.Parameter(torch.zeros(s, dtype=dtype)) for s in shapes]


def give(*ps):
    for p in ps:
        p.grad = torch.ones_like(p)


def counts(calls):
    """The count each parameter was last updated with."""
    return {id(p): c["step"] for c in calls for p in c["params"]}


@pytest.mark.parametrize("bits", [8, 32])
@pytest.mark.parametrize("lies", [torch.contiguous_format, torch.channels_last])
def test_states_of_torch_in_bf16(bits, lies, calls):
    """torch holds the moments of bf16 parameters in bf16; they are fp32 here, lying as the parameter does."""
    theirs, ours = (params((6, 5, 32, 8), (7,), dtype=BF16) for _ in range(2))
    ours[0].data = ours[0].data.to(memory_format=lies)
    ref, opt = torch.optim.AdamW(theirs), optim.AdamW(ours, state_bits=bits)
    give(*theirs), give(*ours)
    ref.step()
    opt.load_state_dict(ref.state_dict())
    opt.step()
    assert counts(calls) == {id(p): 2 for p in ours}
    for p, q in zip(theirs, ours):
        for name in ("exp_avg", "exp_avg_sq"):
            got = opt.state[q][name]
            assert got.dtype == F32 and got.stride() == q.stride() and torch.equal(got, ref.state[p][name].float() + 1)


def capture(monkeypatch, on=True):
    monkeypatch.setattr(optim, "_capturing", lambda: on)


@pytest.mark.parametrize("max_norm", [None, 1.0])
def test_captures_that_replay_something_else(max_norm, calls, monkeypatch):
    """Refused before anything is counted, made or recorded: a count on the host, and a state that the capture would make (and clear in each replay)."""
    norms = []
    monkeypatch.setattr(ops, "grad_norm", lambda grads, most: norms.append(len(grads)) or (None, None))
    a, b, c = params((5000,), (3,), (4,))
    opt = optim.AdamW([{"params": [a, b], "capturable": True}, {"params": [c]}], max_norm=max_norm)

    def refused(words):
        before = copy.deepcopy(opt.state_dict())
        done = len(calls), len(norms)
        capture(monkeypatch)
        with pytest.raises(RuntimeError, match=words):
            opt.step()
        capture(monkeypatch, False)
        after = opt.state_dict()
        assert (len(calls), len(norms)) == done and str(after) == str(before)

    give(a)
    refused("outside of the capture")  # nothing has been there yet
    opt.step()
    give(c)
    refused("capturable")
    c.grad = None
    give(b)
    refused("outside of the capture")  # b has no state yet
    opt.step()
    capture(monkeypatch)
    opt.step()
    assert counts(calls)[id(a)] == 3
    a.grad = b.grad = None
    opt.step()  # (nothing to do)
    assert counts(calls)[id(a)] == 3


@pytest.mark.parametrize("capturable", [True, False])
@pytest.mark.parametrize("name", ["cpu", "cuda:7"])
def test_counts_of_another_device(name, capturable, calls):
    """A checkpoint of a device that is not here, or that holds the parameters no longer: the count goes on where they are."""
    ps = params((5000,), (3,))
    opt = optim.AdamW(ps, capturable=True, state_bits=8)
    give(*ps)
    for _ in range(3):
        opt.step()
    state = copy.deepcopy(opt.state_dict())
    group = state["param_groups"][0]
    group["step_on_device"] = {name: v for v in group["step_on_device"].values()}
    for s in state["state"].values():  # (as states were saved whose steps the group alone counted)
        s["step"] = 0
    group["capturable"] = capturable
    others = params((5000,), (3,))
    opt = optim.AdamW(others)
    opt.load_state_dict(state)
    assert ("step_on_device" in opt.param_groups[0]) == capturable
    give(*others)
    opt.step()
    assert counts(calls)[id(others[0])] == counts(calls)[id(others[1])] == 4


def test_counts_of_several_devices(calls):
    """Saved by a group on two devices, neither of which holds the parameters: the larger count, wherever the numbers lie."""
    ps = params((5000,), (3,))
    opt = optim.AdamW(ps, capturable=True)
    give(*ps)
    opt.step()
    state = copy.deepcopy(opt.state_dict())

    class There:
        """A number on another device: it compares with nothing that lies elsewhere."""
        def __init__(self, v):
            self.v = v

        def __int__(self):
            return self.v

    state["param_groups"][0]["step_on_device"] = {"cuda:6": There(3), "cuda:7": There(8)}
    for s in state["state"].values():
        s["step"] = 0
    opt.load_state_dict(state)
    opt.step()
    assert set(counts(calls).values()) == {9}


@pytest.mark.parametrize("capturable", [True, False])
def test_each_parameter_counts_its_own_steps(capturable, calls):
    """One that joins late begins at 1, one that misses a step stands still in it, whether counted on the device, on the host, or saved and loaded in between."""
    a, b, c = ps = params((5000,), (3,), (6,))
    opt = optim.AdamW(ps, capturable=capturable)
    want = dict.fromkeys(map(id, ps), 0)

    def step(*some):
        for p in ps:
            p.grad = torch.ones_like(p) if any(p is q for q in some) else None
        del calls[:]
        opt.step()
        for p in some:
            want[id(p)] += 1
        assert counts(calls) == {id(p): want[id(p)] for p in some}

    step(a, c), step(a, c)
    step(a, b, c)  # b joins
    step(b, c)  # a misses one
    step(a, b, c)
    assert len(calls) == 3 and want == {id(a): 4, id(b): 3, id(c): 5}
    assert [int(opt.state[p]["step"]) for p in ps] == [4, 3, 5]
    opt.param_groups[0]["capturable"] = not capturable
    step(a, b, c)
    saved = copy.deepcopy(opt.state_dict())
    assert ("step_on_device" in saved["param_groups"][0]) != capturable
    opt = optim.AdamW(ps)
    opt.load_state_dict(saved)
    step(a, b, c), step(b)
    opt.param_groups[0]["capturable"] = capturable
    step(a, b, c)
    opt, ps = copy.deepcopy((opt, ps))
    a, b, c = ps
    want = dict(zip(map(id, ps), want.values()))
    step(a, b, c), step(a, c), step(a, b, c)
    assert list(want.values()) == [10, 9, 11]


def test_parameters_that_a_graph_counts_together(calls, monkeypatch):
    """A replay moves one number for all of them: to count them apart is refused, before anything is counted or made, until the states are loaded anew."""
    a, b = ps = params((5000,), (3,))
    opt = optim.AdamW(ps, capturable=True)
    give(a, b)
    opt.step()
    capture(monkeypatch)
    opt.step()
    a.grad = None
    with pytest.raises(RuntimeError, match="gradients of the same parameters"):  # (in a capture, the number would be copied in each replay)
        opt.step()
    capture(monkeypatch, False)
    before = str(opt.state_dict()), len(calls)
    with pytest.raises(RuntimeError, match="captured"):
        opt.step()
    assert (str(opt.state_dict()), len(calls)) == before
    give(a)
    opt.step()
    assert counts(calls) == {id(a): 3, id(b): 3}
    opt.load_state_dict(copy.deepcopy(opt.state_dict()))
    a.grad = None
    opt.step()
    assert counts(calls) == {id(a): 3, id(b): 4}
    # both ways have been there before the captures: two graphs, each with what it counts
    give(a)
    opt.step()
    capture(monkeypatch)
    opt.step()
    a.grad = None
    opt.step()
    assert counts(calls) == {id(a): 5, id(b): 7}


def spans(calls):
    """{parameter: its elements' numbers}"""
    return {id(p): range(n, n + p.numel()) for c in calls for p, n in zip(c["params"], c["first"])}


@pytest.mark.parametrize("capturable", [True, False])
@pytest.mark.parametrize("bits", [8, 32])
def test_no_two_elements_are_rounded_by_the_same_word(bits, capturable, calls):
    """Numbers go on over groups and kinds of states, and stay a parameter's whichever others have gradients."""
    a, b, c, d, e = ps = params((300,), (5000,), (4096,), (7,), (20, 300), dtype=BF16)
    opt = optim.AdamW([{"params": [a, b]}, {"params": [c, d], "state_bits": 40 - bits}, {"params": [e], "capturable": not capturable}], state_bits=bits, capturable=capturable, seed=3)
    give(*ps)
    opt.step()
    first = spans(calls)
    assert len(first) == 5 and all(c["seed"] == 3 for c in calls)
    taken = [set(range(r.start // 256, -(-r.stop // 256))) for r in first.values()]
    assert all(r.start % 256 == 0 for r in first.values()) and sum(map(len, taken)) == len(set().union(*taken))
    del calls[:]
    a.grad = c.grad = None
    opt.step()
    opt.add_param_group({"params": params((9,), dtype=BF16)})
    opt.step()
    later = spans(calls)
    assert sorted(later) == sorted(map(id, (b, d, e))) and all(first[k] == r for k, r in later.items())


@pytest.mark.parametrize("capturable", [True, False])
def test_counts_that_move_while_one_stands_still(capturable, calls):
    """Equal counts go to the device or back in a step that only one of their parameters takes."""
    a, b = ps = params((5000,), (3,))
    opt = optim.AdamW(ps, capturable=not capturable)
    give(a, b)
    opt.step(), opt.step()
    opt.param_groups[0]["capturable"] = capturable
    a.grad = None
    opt.step()
    give(a)
    opt.step()
    assert counts(calls) == {id(a): 3, id(b): 4}


def test_a_sparse_gradient_is_refused_before_anything_is_counted(calls, monkeypatch):
    norms = []
    monkeypatch.setattr(ops, "grad_norm", lambda grads, most: norms.append(1) or (None, None))
    for capturable in (False, True):
        a, b = ps = params((50,), (30, 2))
        opt = optim.AdamW(ps, capturable=capturable, max_norm=1.0)
        give(a)
        b.grad = torch.ones_like(b).to_sparse()
        with pytest.raises(RuntimeError, match="sparse"):
            opt.step()
        assert not opt.state[a] and not calls and not norms
