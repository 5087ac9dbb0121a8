"""A run of the selective mixer's operators as a layer uses them: add and layer norm, projection, short convolution, projection of steps, B and C, selective scan with its gate, projection.

Tolerances.  Against 64 bits, in fp32: each product of the layer sums up to 64 terms, each operator rounds as in its own tests, about 10^3 U on magnitudes of a few units: 2e-4 of the largest
value.  A prompt against its tokens one by one goes through the same operators with sums in other orders: the same."""
import pytest
import torch
import torch.nn.functional as F

import vig_amd
from vig_amd import _ext

from .util import announce

pytestmark = pytest.mark.gpu

TOL = 2e-4


class Mixer(torch.nn.Module):
    def __init__(self, width=32, inner=64, states=16, rank=4, taps=4):
        super().__init__()
        self.inner, self.states, self.rank, self.taps = inner, states, rank, taps
        g = torch.Generator().manual_seed(0)
        p = lambda *s, scale=None: torch.nn.Parameter(torch.randn(*s, generator=g) * (scale if scale is not None else s[-1] ** -0.5))  # noqa: E731
        self.norm_w, self.norm_b = torch.nn.Parameter(1 + 0.1 * torch.randn(width, generator=g)), p(width, scale=0.1)
        self.w_in, self.w_out, self.w_x, self.w_dt = p(2 * inner, width), p(width, inner), p(rank + 2 * states, inner), p(inner, rank)
        self.conv_w, self.conv_b, self.dt_bias, self.D = p(inner, taps), p(inner, scale=0.1), torch.nn.Parameter(torch.rand(inner, generator=g) * 3 - 4), p(inner, scale=1.0)
        self.A_log = torch.nn.Parameter(torch.log(torch.arange(1.0, states + 1)).repeat(inner, 1))

    def shared(self, x):
        dt, B, C = F.linear(x, self.w_x.to(x.dtype)).split([self.rank, self.states, self.states], -1)
        return F.linear(dt, self.w_dt.to(x.dtype)), B, C

    def forward(self, x, residual, state=None, reverse=False):
        """(output, residual, states)"""
        y, residual = vig_amd.add_layernorm(x, self.norm_w, self.norm_b, residual=residual, prenorm=True)
        u, z = F.linear(y, self.w_in.to(x.dtype)).chunk(2, -1)
        conv, h = state if state is not None else (None, None)
        u, conv = vig_amd.causal_conv1d(u, self.conv_w, self.conv_b, True, conv, True, reverse)
        delta, B, C = self.shared(u)
        o, h = vig_amd.selective_scan(u, delta, -self.A_log.exp(), B, C, self.D, z, self.dt_bias, True, h, True, reverse)
        return F.linear(o, self.w_out.to(x.dtype)), residual, (conv, h)

    def step(self, x, residual, state):
        y, residual = vig_amd.add_layernorm(x, self.norm_w, self.norm_b, residual=residual, prenorm=True)
        u, z = F.linear(y, self.w_in.to(x.dtype)).chunk(2, -1)
        u = vig_amd.causal_conv1d_step(u, self.conv_w, state[0], self.conv_b, True)
        delta, B, C = self.shared(u)
        o = vig_amd.selective_scan_step(u, delta, -self.A_log.exp(), B, C, state[1], self.D, z, self.dt_bias, True)
        return F.linear(o, self.w_out.to(x.dtype)), residual

    def plain(self, x, residual, reverse=False):
        """The same from elementary operations, in whatever precision the parameters have."""
        residual = x + residual
        y = F.layer_norm(residual, residual.shape[-1:], self.norm_w, self.norm_b)
        u, z = F.linear(y, self.w_in).chunk(2, -1)
        turn = (lambda t: t.flip(1)) if reverse else (lambda t: t)
        u = F.silu(F.conv1d(F.pad(turn(u).transpose(1, 2), (self.taps - 1, 0)), self.conv_w.unsqueeze(1), self.conv_b, groups=self.inner)).transpose(1, 2)
        dt, B, C = F.linear(u, self.w_x).split([self.rank, self.states, self.states], -1)
        s, A = F.softplus(F.linear(dt, self.w_dt) + self.dt_bias), -self.A_log.exp()
        h, out = torch.zeros(x.shape[0], self.inner, self.states, dtype=x.dtype), []
        for t in range(x.shape[1]):
            h = torch.exp(s[:, t].unsqueeze(-1) * A) * h + (s[:, t] * u[:, t]).unsqueeze(-1) * B[:, t].unsqueeze(1)
            out.append((h * C[:, t].unsqueeze(1)).sum(-1) + self.D * u[:, t])
        return F.linear(turn(torch.stack(out, 1)) * F.silu(z), self.w_out), residual


def made(seed, batch=3, L=70, width=32, dtype=torch.float32):
    gen = torch.Generator().manual_seed(seed)
    return [torch.randn(batch, L, width, generator=gen).to(dtype) for _ in range(2)]


def near(a, b, what):
    a, b = a.detach().double().cpu(), b.detach().double().cpu()
    assert float((a - b).abs().max()) <= TOL * float(b.abs().max()), f"{what}: off by {float((a - b).abs().max()):.3e} of {float(b.abs().max()):.3e}"


@pytest.mark.parametrize("reverse", [False, True])
def test_layer_and_gradients(reverse):
    announce(f"mixer, reverse {reverse}")
    x, residual = made(1)
    ref = Mixer().double()
    a, b = (t.double().requires_grad_() for t in (x, residual))
    o, r = ref.plain(a, b, reverse)
    (o.sin().sum() + r.cos().sum()).backward()
    m = Mixer().cuda()
    p, q = (t.cuda().requires_grad_() for t in (x, residual))
    o2, r2, _ = m(p, q, reverse=reverse)
    (o2.sin().sum() + r2.cos().sum()).backward()
    near(o2, o, "output"), near(r2, r, "residual"), near(p.grad, a.grad, "dx"), near(q.grad, b.grad, "dresidual")
    for (name, u), (_, v) in zip(m.named_parameters(), ref.named_parameters()):
        near(u.grad, v.grad, name)


@torch.no_grad()
def test_prompt_and_tokens_one_by_one():
    """A prompt, its continuation by another prompt and by single tokens."""
    announce("mixer, prompt and tokens")
    m = Mixer().cuda()
    x, residual = (t.cuda() for t in made(2))
    whole, _, (conv, h) = m(x, residual)
    first, _, state = m(x[:, :30], residual[:, :30])
    second, _, state = m(x[:, 30:50], residual[:, 30:50], state)
    near(torch.cat([first, second], 1), whole[:, :50], "prompts")
    for t in range(50, 70):
        o, _ = m.step(x[:, t], residual[:, t], state)
        near(o, whole[:, t], f"token {t}")
    near(state[0], conv, "convolution's state"), near(state[1], h, "scan's state")


@torch.no_grad()
def test_captured_tokens():
    """One token's run in a graph: replays move the states on as eager runs do, with eager work between them."""
    announce("mixer, captured token")
    m = Mixer().cuda().bfloat16().float()
    x, residual = (t.cuda() for t in made(3, L=6))
    _, _, state = m(x[:, :2], residual[:, :2])
    mine = tuple(t.clone() for t in state)
    token, skip = x[:, 2].clone(), residual[:, 2].clone()
    m.step(token, skip, tuple(t.clone() for t in state))
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out, _ = m.step(token, skip, mine)
    for t, s in zip(mine, state):
        t.copy_(s)
    for k in range(2, 6):
        token.copy_(x[:, k]), skip.copy_(residual[:, k])
        graph.replay()
        want, _ = m.step(x[:, k], residual[:, k], state)
        torch.cuda.synchronize()
        assert torch.equal(out, want) and all(torch.equal(a, b) for a, b in zip(mine, state))


def test_captured_training_step():
    """Forward and backward of the layer in a graph, replayed on new inputs and checked against eager runs between the replays."""
    announce("mixer, captured training step")
    m = Mixer().cuda()
    names, params = zip(*m.named_parameters())
    x, residual = (t.cuda() for t in made(4, batch=2, L=300))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())

    def run(x, residual):
        o, r, _ = m(x, residual)
        return torch.autograd.grad((o * o).sum() + (r * o).sum(), params)

    with torch.cuda.stream(side):
        run(x, residual)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = run(x, residual)
    for seed in (5, 6, 7):
        new = [t.cuda() for t in made(seed, batch=2, L=300)]
        x.copy_(new[0]), residual.copy_(new[1])
        graph.replay()
        torch.cuda.synchronize()
        for name, a, b in zip(names, got, run(*new)):
            near(a, b, name)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_native_calls_and_ctypes_give_the_same_bits(dtype, monkeypatch):
    announce(f"mixer, both ways, {dtype}")
    x, residual = (t.cuda() for t in made(8, dtype=dtype))
    residual = residual.float()

    def run():
        m = Mixer().cuda()
        p, q = x.clone().requires_grad_(), residual.clone().requires_grad_()
        o, r, state = m(p, q)
        (o.float().sum() + r.sum() + state[0].float().sum() + state[1].sum()).backward()
        with torch.no_grad():
            after = m.step(x[:, 0], residual[:, 0], tuple(t.detach().clone() for t in state))[0]
        return [o, r, *state, p.grad, q.grad, after, *(t.grad for t in m.parameters())]

    native = run()
    monkeypatch.setattr(_ext, "calls", lambda: None)
    assert all(torch.equal(a, b) for a, b in zip(native, run()))
