"""AdamW over many tensors and the norm of their gradients against their formulas in 64 bits, with bounds on every element.

Bounds.  u = 2^-24.  A moment is two products and a sum of constants rounded once: off by at most 4 u of the sum of its terms' magnitudes (g's square and the clip's
product add 3 u of that term).  The parameter's step has eight more roundings: 12 u of itself, its moment's relative error and half of the square's.  A rounding to 8 or
16 bits by given random bits is a function Q that never falls: what lies within d of x ends between Q(x - d) and Q(x + d), which differ for few."""
import copy
import math

import pytest
import torch

import vig_amd
from vig_amd import _ext, layers, optim

from .util import announce

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
F32, BF16, E4M3 = torch.float32, torch.bfloat16, torch.float8_e4m3fn
B1, B2, EPS, LR, DECAY = 0.9, 0.999, 1e-8, 3e-3, 0.05
M32 = 0xFFFFFFFF


def mix(x):
    x = ((x ^ (x >> 16)) * 0x6A09E667) & M32
    x = ((x ^ (x >> 15)) * 0xBB67AE85) & M32
    return x ^ (x >> 16)


def key_of(seed, t):
    return mix((mix((mix(seed & M32) + (seed >> 32)) & M32) + t) & M32)


def words(first, n, key):
    """The random words of n elements, in Python's integers where a product passes 63 bits."""
    x = torch.arange(n, dtype=torch.int64) + first
    x = (x & M32) ^ ((key + (x >> 32) * 0x9E3779B9) & M32)
    for shift, factor in ((16, 0x6A09E667), (15, 0xBB67AE85)):
        x = x ^ (x >> shift)
        x = (x * (factor & 0xFFFF) + (((x & 0xFFFF) * (factor >> 16) & 0xFFFF) << 16)) & M32
    return x ^ (x >> 16)


def round_8(y, bits, least):
    """y >= 0 in units of the scale -> e4m3's values, up where the bits reach past what the step lacks."""
    gap = torch.exp2(torch.floor(torch.log2(y.clamp_min(2.0 ** -6))) - 3)
    q = torch.floor(y / gap + bits.double() / 65536) * gap
    return torch.where((y > 0) & (q == 0), torch.full_like(q, 2.0 ** -9), q) if least else q


def round_16(y, bits):
    gap = torch.exp2(torch.floor(torch.log2(y.clamp_min(2.0 ** -126))) - 7)
    return torch.floor(y / gap + bits.double() / 65536) * gap


def blocks(t, n):
    full = torch.zeros(-(-n // 256) * 256, dtype=torch.float64)
    full[:n] = t
    return full.view(-1, 256)


def between(got, x, off, rounded, what):
    """got is what `rounded` makes of something within `off` of x; signs apart."""
    low, high = rounded((x.abs() - off).clamp_min(0)), rounded(x.abs() + off)
    got = torch.where(x < 0, -got, got)
    fine = (low <= got) & (got <= high) | (x.abs() <= off)
    assert bool(fine.all()), f"{what}: {int((~fine).sum())} of {fine.numel()} outside, first at {int((~fine).nonzero()[0])}"
    assert float((low != high).double().mean()) < 1e-2, what
    return True


class Case:
    """A list of tensors of drawn types and their states, beginning on any element where `tight`."""

    def __init__(self, sizes, p_types, g_types, bits8, seed, tight=False, scale=1e-2):
        gen = torch.Generator(device="cuda").manual_seed(seed)
        r = lambda n: torch.randn(n, device="cuda", generator=gen)  # noqa: E731

        def cut(n, dtype, make):
            if not tight:
                return make(n).to(dtype)
            return torch.cat([torch.zeros(3, device="cuda"), make(n)]).to(dtype)[3:]

        self.sizes, self.bits8 = sizes, bits8
        self.p = [cut(n, p_types[j % len(p_types)], r) for j, n in enumerate(sizes)]
        self.g = [cut(n, g_types[j % len(g_types)], lambda n: r(n) * scale) for j, n in enumerate(sizes)]
        if bits8:
            self.m, self.v = ([torch.zeros(n, dtype=torch.uint8, device="cuda").view(E4M3) for n in sizes] for _ in range(2))
            self.ms, self.vs = ([torch.zeros(-(-n // 256), device="cuda") for n in sizes] for _ in range(2))
        else:
            self.m, self.v = ([cut(n, F32, lambda n: r(n).square() * s) for n in sizes] for s in (3e-3, 1e-5))
            self.ms = self.vs = None
        self.gen = r

    def new_gradients(self, scale=1e-2):
        for g in self.g:
            g.copy_(self.gen(g.numel()) * scale)

    def held(self):
        d = lambda ts: [t.detach().double().cpu() if t.dtype != E4M3 else t.float().double().cpu() for t in ts]  # noqa: E731
        return {k: d(getattr(self, k)) if getattr(self, k) is not None else None for k in ("p", "g", "m", "v", "ms", "vs")}

    def step(self, t, **more):
        kw = {"step": t, "lr": LR, "betas": (B1, B2), "eps": EPS, "weight_decay": DECAY} | more
        vig_amd.adamw_step(self.p, self.g, self.m, self.v, self.ms, self.vs, **kw)

    def check(self, before, t, seed=0, clip=1.0, lr=LR, numbers=None):
        after, first = self.held(), 0
        for j, n in enumerate(self.sizes):
            if n == 0:
                continue
            p, g = before["p"][j], before["g"][j] * clip
            w = words(first if numbers is None else numbers[j], n, key_of(seed, t))
            first += -(-n // 256) * 256
            if self.bits8:
                spread = lambda s: s.repeat_interleave(256)[:n]  # noqa: E731
                m, root = before["m"][j] * spread(before["ms"][j]), before["v"][j] * spread(before["vs"][j])
                v = root * root
            else:
                m, v = before["m"][j], before["v"][j]
            em = 8 * U * (B1 * m.abs() + (1 - B1) * g.abs())
            m = B1 * m + (1 - B1) * g
            ev = 9 * U * (B2 * v + (1 - B2) * g * g)
            v = B2 * v + (1 - B2) * g * g
            root = v.sqrt()
            er = ev / (2 * root).clamp_min(1e-30) + U * root
            den = root / math.sqrt(1 - B2 ** t) + EPS
            move = lr / (1 - B1 ** t) * m / den
            ep = 3 * U * p.abs() + 12 * U * move.abs() + lr / (1 - B1 ** t) * em / den + move.abs() * (er / math.sqrt(1 - B2 ** t)) / den
            p = p * (1 - lr * DECAY) - move
            what = f"tensor {j} of {n}"
            if self.p[j].dtype == BF16:
                up = ((w * 0x79B9 + (((w & 0xFFFF) * 0x9E37 & 0xFFFF) << 16)) & M32) >> 16
                between(after["p"][j], p, ep, lambda y, up=up: round_16(y, up), what + ": p")
            else:
                assert bool(((after["p"][j] - p).abs() <= ep + U * p.abs()).all()), what + ": p"
            if not self.bits8:
                assert bool(((after["m"][j] - m).abs() <= em).all()), what + ": m"
                assert bool(((after["v"][j] - v).abs() <= ev).all()), what + ": v"
                continue
            for name, x, off, bits in (("m", m, em, w & 0xFFFF), ("v", root, er, w >> 16)):
                most = blocks(x, n).abs().amax(1)
                scale, off_scale = most / 448, blocks(off, n).amax(1) / 448 + 3 * U * most / 448
                got = after[name + "s"][j]
                assert bool(((got - scale).abs() <= off_scale + 1e-45).all()), what + ": scale"
                s = got.repeat_interleave(256)[:n]  # (the codes go by the scale that was stored)
                y, off_y = x / s.clamp_min(1e-45), off / s.clamp_min(1e-45) + 4 * U * x.abs() / s.clamp_min(1e-45)
                between(after[name][j], y, off_y, lambda y, bits=bits, name=name: round_8(y, bits, name == "v"), what + ": " + name)


SIZES = [1, 2, 3, 5, 255, 256, 257, 1000, 4095, 4096, 4097, 8193, 20011]


@pytest.mark.parametrize("tight", [False, True])
@pytest.mark.parametrize("bits8", [False, True])
@pytest.mark.parametrize("p_types,g_types", [((F32,), (F32,)), ((BF16,), (BF16,)), ((F32,), (BF16,)), ((BF16,), (F32,)), ((F32, BF16, F32), (F32, F32, BF16, BF16))])
def test_adamw_against_the_formula(p_types, g_types, bits8, tight):
    announce(f"AdamW {p_types} {g_types} 8 bits {bits8} tight {tight}")
    c = Case(SIZES, p_types, g_types, bits8, 5, tight)
    for t in (1, 2, 3, 1000):
        c.new_gradients(1e-2 if t < 3 else 1.0)
        before = c.held()
        c.step(t, seed=(7 << 32) + 9)
        c.check(before, t, seed=(7 << 32) + 9)


@pytest.mark.parametrize("bits8", [False, True])
def test_more_tensors_than_a_launch_takes(bits8):
    announce(f"AdamW over 301 tensors, 8 bits {bits8}")
    sizes = [(37 * j * j) % 5000 + 1 for j in range(300)] + [70000]
    c = Case(sizes, (F32, F32, BF16), (F32, BF16), bits8, 6)
    for t in (1, 2):
        before = c.held()
        c.step(t, grad_scale=torch.tensor(0.25, device="cuda"))
        c.check(before, t, clip=0.25)


@pytest.mark.parametrize("bits8", [False, True])
def test_numbers_of_elements(bits8, monkeypatch):
    """A list rounded as part of a larger one: numbers in any order, past 32 bits, and across that border within a lane's elements."""
    sizes = [1000, 5000, 300, 9000]
    numbers = [5, (1 << 32) - 4001, 1 << 39, 77]
    for way in range(2):
        if way:
            monkeypatch.setattr(_ext, "calls", lambda: None)
        c = Case(sizes, (BF16, F32), (F32,), bits8, 6)
        for t in (1, 2):
            before = c.held()
            c.step(t, seed=3, first=numbers)
            c.check(before, t, seed=3, numbers=numbers)
    monkeypatch.undo()
    whole, parts = Case([700, 300, 5000], (BF16,), (F32,), bits8, 2), Case([700, 300, 5000], (BF16,), (F32,), bits8, 2)
    whole.step(1)
    for some, first in ((slice(0, 1), [0]), (slice(1, 3), [768, 1280])):  # (behind blocks of 256)
        lists = [t[some] if t is not None else None for t in (parts.p, parts.g, parts.m, parts.v, parts.ms, parts.vs)]
        vig_amd.adamw_step(*lists, step=1, lr=LR, betas=(B1, B2), eps=EPS, weight_decay=DECAY, first=first)
    assert all(torch.equal(a, b) for a, b in zip(whole.p, parts.p)) and all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip(whole.m + whole.v, parts.m + parts.v))


def test_empty_tensors_and_lists():
    vig_amd.adamw_step([], [], [], [], step=1)
    c = Case([0, 5, 0, 300], (F32,), (F32,), False, 1)
    before = c.held()
    c.step(1)
    c.check(before, 1)
    d = Case([0, 0], (F32,), (F32,), True, 1)
    d.step(1)
    for j in (1, 3):
        assert not torch.equal(c.p[j].double().cpu(), before["p"][j])
    norm, scale = vig_amd.grad_norm(d.g, 1.0)
    assert float(norm) == 0.0 and float(scale) == 1.0


def test_what_is_not_written_stays():
    """Elements beside a tensor in its storage, and a list's gradients."""
    for bits8 in (False, True):
        sizes = [5, 700, 4097]
        c = Case(sizes, (F32, BF16), (F32,), bits8, 3)
        hold = []
        for name in ("p", "m", "v"):
            ts = getattr(c, name)
            for j, t in enumerate(ts):
                raw = t.view(torch.uint8)
                wide = torch.full((raw.numel() + 64,), 0x5A, dtype=torch.uint8, device="cuda")
                wide[32:32 + raw.numel()] = raw
                ts[j] = wide[32:32 + raw.numel()].view(t.dtype)
                hold.append((wide, raw.numel()))
        kept = [g.clone() for g in c.g]
        c.step(1)
        for wide, n in hold:
            assert bool((wide[:32] == 0x5A).all() and (wide[32 + n:] == 0x5A).all())
        assert all(torch.equal(a, b) for a, b in zip(kept, c.g))


def test_rounding_is_right_on_average():
    """Sixteen bits decide: the mean of 2^20 roundings of one value is off by at most half a bit's worth and five standard deviations."""
    n = 1 << 20
    for value in (0.3, 0.77, 1.0, 0.011):
        p = [torch.full((n,), value, device="cuda", dtype=BF16)]
        g, m, v = ([torch.zeros(n, device="cuda")] for _ in range(3))
        start = float(p[0][0])
        vig_amd.adamw_step(p, g, m, v, step=1, lr=1e-3, weight_decay=0.5, seed=3)
        want = start * (1 - 1e-3 * 0.5)
        step = 2.0 ** (math.floor(math.log2(want)) - 7)
        assert abs(float(p[0].double().mean()) - want) <= step * (2.0 ** -17 + 5 * 0.5 / math.sqrt(n)) + 2 * U * want
        assert set(((p[0].double() - want).abs() < step).unique().tolist()) == {True}
    # states: m = 0.1 g with the block's largest value 448 times its scale
    g = [torch.full((n,), 0.37, device="cuda")]
    g[0][::256] = 1.0
    p, codes = [torch.zeros(n, device="cuda")], [[torch.zeros(n, dtype=torch.uint8, device="cuda").view(E4M3)] for _ in range(2)]
    scales = [[torch.zeros(n // 256, device="cuda")] for _ in range(2)]
    vig_amd.adamw_step(p, g, *codes, *scales, step=1, seed=4)
    for k in range(2):
        y = codes[k][0].float().view(-1, 256)[:, 1:].double()
        step = 16.0  # 0.37 * 448 = 165.8: between 160 and 176
        assert abs(float(y.mean()) - 0.37 * 448) <= step * (2.0 ** -17 + 5 * 0.5 / math.sqrt(y.numel())) + 1e-4
        assert set(y.unique().tolist()) == {160.0, 176.0}


def test_a_root_above_zero_stays_above():
    n = 512
    g = torch.full((n,), 1e-9, device="cuda")
    g[0], g[256], g[300:] = 1.0, 1.0, 0.0
    p, m, r = torch.zeros(n, device="cuda"), *(torch.zeros(n, dtype=torch.uint8, device="cuda").view(E4M3) for _ in range(2))
    ms, rs = torch.zeros(2, device="cuda"), torch.zeros(2, device="cuda")
    vig_amd.adamw_step([p], [g], [m], [r], [ms], [rs], step=1)
    r = r.float()
    assert float(r[0]) == 448.0 and bool((r[1:256] == 2.0 ** -9).all()) and bool((r[300:] == 0).all())


@pytest.mark.parametrize("bits8", [False, True])
def test_values_that_are_not_finite(bits8):
    for bad in (math.nan, math.inf, -math.inf):
        c = Case([1000], (F32,), (F32,), bits8, 2)
        if bits8:
            c.step(1)
        c.g[0][300] = bad
        c.step(2)
        m, p = c.m[0].float(), c.p[0]
        if bits8:  # the block of 256 around it
            m = m * c.ms[0].repeat_interleave(256)[:1000]
            assert bool(m[256:512].isnan().all()) and bool(m[:256].isfinite().all() and m[512:].isfinite().all())
        else:
            assert not bool(m[300].isfinite()) and int((~m.isfinite()).sum()) == 1
        assert int((~p.isfinite()).sum()) == 1 and not bool(p[300].isfinite())


@pytest.mark.parametrize("bits8", [False, True])
def test_a_step_that_is_left_out(bits8):
    c = Case(SIZES, (F32, BF16), (F32,), bits8, 2)
    before = c.held()
    c.g[3][0] = math.inf
    norm, scale = vig_amd.grad_norm(c.g, 1.0)
    assert float(norm) == math.inf and math.isnan(float(scale))
    c.step(1, grad_scale=scale)
    after = c.held()
    for k in ("p", "m", "v") + (("ms", "vs") if bits8 else ()):
        assert all(torch.equal(a, b) for a, b in zip(before[k], after[k]))


@pytest.mark.parametrize("bits8", [False, True])
def test_numbers_on_the_device(bits8):
    """The step's number and the learning rate there: what the host works out in 64 bits, the device does too."""
    for t in (1, 2, 17, 100000):
        a, b = (Case([4097, 300], (F32, BF16), (F32,), bits8, 2) for _ in range(2))
        a.step(t, seed=5, lr=0.125)
        b.step(torch.tensor(t, device="cuda"), seed=5, lr=torch.tensor(0.125, device="cuda"))
        for x, y in zip(a.held().values(), b.held().values()):
            # (logarithm and exponential of 64 bits against a power: the same 24 bits but for a rounding)
            assert x is None or all(torch.allclose(s, r, rtol=2.0 ** -7 if r.numel() == 300 else 4 * U, atol=0 if not bits8 else 1e-3) for s, r in zip(x, y))


def test_betas_of_zero():
    c = Case([777], (F32,), (F32,), False, 2)
    for step in (3, torch.tensor(3, device="cuda")):
        before = c.held()
        c.step(step, betas=(0.0, 0.0), weight_decay=0.0)
        want = before["p"][0] - LR * before["g"][0] / (before["g"][0].abs() + EPS)
        assert float((c.p[0].double().cpu() - want).abs().max()) <= 4 * U * float(want.abs().max())


@pytest.mark.parametrize("axes", [(0, 2, 3, 1), (3, 2, 1, 0)])
def test_tensors_that_lie_otherwise(axes):
    """Channels-last weights: moments lie as they do, a gradient may lie otherwise."""
    gen = torch.Generator(device="cuda").manual_seed(1)
    back = [axes.index(i) for i in range(4)]
    lies = lambda t: t.permute(axes).contiguous().permute(back)  # noqa: E731
    w, g = (torch.randn(6, 5, 3, 4, device="cuda", generator=gen) for _ in range(2))
    a, b = (w.clone(), torch.zeros_like(w), torch.zeros_like(w)), tuple(lies(t) for t in (w, torch.zeros_like(w), torch.zeros_like(w)))
    vig_amd.adamw_step([a[0]], [g], [a[1]], [a[2]], step=1)
    vig_amd.adamw_step([b[0]], [g], [b[1]], [b[2]], step=1)
    assert all(torch.equal(x, y) for x, y in zip(a, b)) and b[0].stride() == lies(w).stride()


def test_versions_move():
    c = Case([300, 20], (F32,), (F32,), True, 2)
    ts = c.p + c.m + c.v + c.ms + c.vs
    before = [t._version for t in ts]
    c.step(1)
    assert [t._version for t in ts] == [v + 1 for v in before]


@pytest.mark.parametrize("tight", [False, True])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_grad_norm(dtype, tight):
    for sizes in ([1], SIZES, [16383, 16384, 16385, 100001], [(91 * j) % 700 + 1 for j in range(500)]):
        c = Case(sizes, (F32,), (dtype,), False, len(sizes), tight)
        norm, scale = vig_amd.grad_norm(c.g, 0.5)
        want = math.sqrt(sum(float(g.double().square().sum()) for g in c.g))
        assert norm.shape == () and abs(float(norm) - want) <= 2 * U * want
        clip = min(1.0, 0.5 / (want + 1e-6))
        assert abs(float(scale) - clip) <= 6 * U * clip
        assert torch.equal(norm, vig_amd.grad_norm(c.g)[0]) and vig_amd.grad_norm(c.g)[1] is None


def test_grad_norm_of_large_and_small_values():
    for value in (1e30, 1e-30):  # squares past fp32 both ways
        g = [torch.full((1000,), value, device="cuda")]
        assert abs(float(vig_amd.grad_norm(g)[0]) / (value * math.sqrt(1000)) - 1) <= 4 * U
    for bad in (math.nan, math.inf):
        g = [torch.zeros(5000, device="cuda"), torch.zeros(7, device="cuda", dtype=BF16)]
        g[1][6] = bad
        norm, scale = vig_amd.grad_norm(g, 1.0)
        assert not math.isfinite(float(norm)) and math.isnan(float(scale))


def test_the_same_bits_whichever_way_the_call_goes(monkeypatch):
    for bits8 in (False, True):
        made = []
        for way in range(3):
            if way == 2:
                monkeypatch.setattr(_ext, "calls", lambda: None)
            c = Case(SIZES, (F32, BF16), (F32, BF16, BF16), bits8, 8)
            for t in (1, 2):
                norm, scale = vig_amd.grad_norm(c.g, 0.5)
                c.step(t, grad_scale=scale, seed=t)
            made.append([norm, scale] + c.p + [x for x in c.m + c.v] + (c.ms + c.vs if bits8 else []))
            monkeypatch.undo()
        for other in made[1:]:
            assert all(torch.equal(a.view(torch.uint8) if a.dtype == E4M3 else a, b.view(torch.uint8) if b.dtype == E4M3 else b) for a, b in zip(made[0], other))


def test_past_2_to_the_31_elements():
    """One tensor of 2^31 + 300 elements in bf16 with its states in 8 bits: pieces, numbers of elements and offsets pass 31 bits."""
    n = (1 << 31) + 300
    announce("AdamW past 2^31 elements")
    p = torch.zeros(n, device="cuda", dtype=BF16)
    g = torch.zeros(n, device="cuda", dtype=BF16)
    m, r = (torch.zeros(n, dtype=torch.uint8, device="cuda").view(E4M3) for _ in range(2))
    ms, rs = (torch.zeros(-(-n // 256), device="cuda") for _ in range(2))
    tail = 1000
    g[-tail:] = torch.randn(tail, device="cuda", generator=torch.Generator(device="cuda").manual_seed(1)).to(BF16)
    p[-tail:] = 1.0
    norm, _ = vig_amd.grad_norm([g])
    want = math.sqrt(float(g[-tail:].double().square().sum()))
    assert abs(float(norm) - want) <= 2 * U * want
    vig_amd.adamw_step([p], [g], [m], [r], [ms], [rs], step=1, lr=LR, seed=2)
    assert not bool(p[:-tail].any()) and not bool(m[:-tail].view(torch.uint8).any()) and not bool(rs[:(n - tail) // 256].any())
    # the last blocks alone, as a list of their own whose numbers are shifted: moments (not their roundings) agree to the codes' step
    first = (n - tail) // 256 * 256
    k = n - first
    q = [torch.zeros(k, dtype=torch.uint8, device="cuda").view(E4M3) for _ in range(2)]
    s = [torch.zeros(-(-k // 256), device="cuda") for _ in range(2)]
    vig_amd.adamw_step([p[first:].clone()], [g[first:].clone()], [q[0]], [q[1]], [s[0]], [s[1]], step=1, lr=LR, seed=2)
    assert torch.equal(s[0], ms[first // 256:]) and torch.equal(s[1], rs[first // 256:])
    d = (q[0].float() - m[first:].float()).abs()
    assert bool((d <= q[0].float().abs() * 2.0 ** -3 + 2.0 ** -9).all()) and bool(((p[-tail:].float() - 1).abs() < 0.02).all())


# ---- the optimiser, and a training step of all of it


def test_optimiser_against_torch():
    """The same parameters, gradients and settings: within the roundings of ten steps of either."""
    gen = torch.Generator(device="cuda").manual_seed(4)
    shapes = [(64, 33), (7,), (5000,), (3, 2, 4, 4)]
    make = lambda: [torch.nn.Parameter(t.clone()) for t in base]  # noqa: E731
    base = [torch.randn(s, device="cuda", generator=gen) for s in shapes]
    ours, theirs = make(), make()
    kw = {"lr": 1e-2, "betas": (0.8, 0.95), "eps": 1e-6, "weight_decay": 0.1}
    a = optim.AdamW([{"params": ours[:2]}, {"params": ours[2:], "lr": 1e-3}], max_norm=3.0, **kw)
    b = torch.optim.AdamW([{"params": theirs[:2]}, {"params": theirs[2:], "lr": 1e-3}], **kw)
    for i in range(10):
        for p, q in zip(ours, theirs):
            g = torch.randn(p.shape, device="cuda", generator=gen)
            p.grad, q.grad = (None, None) if i % 3 == 1 and p.numel() == 7 else (g.clone(), g.clone())
        norm = torch.nn.utils.clip_grad_norm_(theirs, 3.0)
        a.step(), b.step()
        assert abs(float(a.grad_norm) / float(norm) - 1) < 1e-5
    for p, q, start in zip(ours, theirs, base):
        moved = float((q.detach() - start).abs().max())
        assert float((p - q).detach().abs().max()) <= 1e-4 * moved + 4 * U * float(q.detach().abs().max())
    assert sorted(a.state[ours[1]]) == ["exp_avg", "exp_avg_sq", "step"] and a.state[ours[1]]["step"] == 7


@pytest.mark.parametrize("bits", [8, 32])
def test_optimiser_keeps_its_state(bits, tmp_path):
    torch.manual_seed(0)
    make = lambda: [torch.nn.Parameter(torch.linspace(-1, 1, n, device="cuda").to(t)) for n, t in ((5000, F32), (4096, BF16), (100, F32))]  # noqa: E731
    ours, other = make(), make()
    a, b = optim.AdamW(ours, lr=1e-2, state_bits=bits), optim.AdamW(other, lr=1.0, state_bits=bits)
    gen = torch.Generator(device="cuda").manual_seed(4)
    grads = [[torch.randn(p.shape, device="cuda", generator=gen).to(p.dtype) for p in ours] for _ in range(4)]

    def step(opt, params, g):
        for p, t in zip(params, g):
            p.grad = t
        opt.step()

    for g in grads[:2]:
        step(a, ours, g)
    path = str(tmp_path / "o.pt")
    torch.save(a.state_dict(), path)
    with torch.no_grad():
        for p, q in zip(ours, other):
            q.copy_(p)
    b.load_state_dict(torch.load(path, weights_only=True))
    assert b.param_groups[0]["lr"] == 1e-2 and b.state[other[1]]["exp_avg"].dtype == (E4M3 if bits == 8 else F32)
    assert b.state[other[2]]["exp_avg"].dtype == F32
    for g in grads[2:]:
        step(a, ours, g), step(b, other, g)
    assert all(torch.equal(p, q) for p, q in zip(ours, other))


def test_optimiser_becomes_capturable_and_back():
    """The number of steps goes with the state, whichever way it is counted."""
    w = torch.linspace(-1, 1, 5000, device="cuda")
    make = lambda c, p: optim.AdamW([p], lr=1e-2, capturable=c)  # noqa: E731
    want, ours = torch.nn.Parameter(w.clone()), torch.nn.Parameter(w.clone())
    ref, opt = make(False, want), make(False, ours)
    for i in range(6):
        if i in (2, 4):  # to be captured from now on, and back
            state = opt.state_dict()
            state["param_groups"][0]["capturable"] = i == 2
            opt = make(i == 2, ours)
            opt.load_state_dict(state)
        for o, p in ((ref, want), (opt, ours)):
            p.grad = torch.cos(w * (i + 1))
            o.step()
    # (the two ways to the corrections agree but for a rounding a step)
    assert float((want - ours).detach().abs().max()) <= 6 * 4 * U


def test_optimiser_counts_where_it_is_told():
    """Captured, not captured, saved and captured again, by the group's own entry or a loaded state: the count goes on."""
    w = torch.linspace(-1, 1, 5000, device="cuda")
    p = torch.nn.Parameter(w.clone())
    opt = optim.AdamW([p], lr=1e-2)
    for i, capturable in enumerate((True, True, False, False, True, False)):
        opt.param_groups[0]["capturable"] = capturable
        p.grad = w.cos()
        opt.step()
        state = opt.state_dict()
        opt = optim.AdamW([p], lr=1e-2)
        opt.load_state_dict(state)
        counted = opt.param_groups[0].get("step_on_device", {"": opt.state[p]["step"]})
        assert [int(v) for v in counted.values()] == [i + 1]
        assert capturable == ("step_on_device" in opt.param_groups[0])


def test_optimiser_copied_and_taken_over_from_torch():
    w = torch.linspace(-1, 1, 5000, device="cuda")
    want, ours = torch.nn.Parameter(w.clone()), torch.nn.Parameter(w.clone())
    ref, opt = torch.optim.AdamW([want], lr=1e-2), optim.AdamW([ours], lr=1e-2, max_norm=1e9, seed=5)
    for i in range(6):
        for o, q in ((ref, want), (opt, ours)):
            q.grad = torch.cos(w * (i + 1))
            o.step()
        if i == 1:
            opt.load_state_dict(ref.state_dict())
        if i == 3:
            opt, ours = copy.deepcopy((opt, ours))
            assert opt.max_norm == 1e9 and opt.seed == 5
    # (each side's step is off by a few roundings of the parameter, at most 1, and of a move of at most lr (1 + its part of the moments' roundings))
    assert float((want - ours).detach().abs().max()) <= 6 * 8 * U
    with pytest.raises(ValueError):
        opt.load_state_dict(torch.optim.AdamW([want], amsgrad=True).state_dict())


def test_refused_on_the_gpu():
    c = Case([300, 20], (F32,), (F32,), False, 2)
    cpu = torch.zeros(300)
    for bad in (lambda: vig_amd.adamw_step([c.p[0], c.p[0]], c.g[:1] * 2, [c.m[0], c.m[0]], [c.v[0], c.v[0]], step=1), lambda: c.step(0), lambda: c.step(1, grad_scale=0.5),
                lambda: c.step(torch.tensor(1)), lambda: c.step(1, lr=torch.tensor(0.1)), lambda: c.step(1, betas=(1.0, 0.9)), lambda: c.step(1, eps=-1.0), lambda: c.step(1, first=[0]),
                lambda: c.step(1, first=[0, -1]), lambda: vig_amd.adamw_step(c.p, c.g, c.m, c.v[:1], step=1), lambda: vig_amd.adamw_step(c.p[:1], [cpu], c.m[:1], c.v[:1], step=1),
                lambda: vig_amd.adamw_step(c.p, c.g, c.p, c.v, step=1), lambda: vig_amd.adamw_step(c.p, c.p, c.m, c.v, step=1),
                lambda: vig_amd.adamw_step(c.p, c.g, [t.bfloat16() for t in c.m], c.v, step=1), lambda: vig_amd.adamw_step(c.p, c.g, c.m, c.v, c.ms, [torch.zeros(1, device="cuda")], step=1),
                lambda: vig_amd.adamw_step([t.half() for t in c.p], c.g, c.m, c.v, step=1), lambda: vig_amd.adamw_step([c.p[0][::2]], [c.g[0][::2]], [c.m[0][::2]], [c.v[0][::2]], step=1),
                lambda: vig_amd.grad_norm([c.g[0], cpu]), lambda: vig_amd.grad_norm([c.g[0].half()]), lambda: vig_amd.grad_norm(c.g, float("nan"))):
        before = c.held()
        with pytest.raises((ValueError, TypeError, RuntimeError)):
            bad()
        after = c.held()
        assert all(torch.equal(a, b) for k in ("p", "g", "m", "v") for a, b in zip(before[k], after[k]))
    norm, _ = vig_amd.grad_norm([c.g[0][::2], c.g[1].expand(3, 20)])  # (gaps and repeats are copied)
    want = math.sqrt(float(c.g[0][::2].double().square().sum()) + 3 * float(c.g[1].double().square().sum()))
    assert abs(float(norm) - want) <= 2 * U * want


def test_weight_copies_of_the_layers_follow():
    torch.manual_seed(0)
    norm = layers.RMSNorm(384).cuda()
    norm.weight.data = norm.weight.data.to(BF16)
    first = norm._w32().clone()
    opt = optim.AdamW(norm.parameters(), lr=0.5)
    norm.weight.grad = torch.ones_like(norm.weight)
    opt.step()
    assert torch.equal(norm._w32(), norm.weight.detach().float()) and not torch.equal(norm._w32(), first)


class _Mixer(torch.nn.Module):
    def __init__(self, d):
        super().__init__()
        self.rows, self.gates, self.out = (torch.nn.Linear(d, n, bias=False) for n in (d, 2 * d, 5))

    def forward(self, x):
        g = torch.nn.functional.logsigmoid(self.gates(x)) / 16
        d = x.shape[-1]
        o, _ = vig_amd.bid_gated_scan(self.rows(x), torch.cat([g[..., :d], g[..., d:]]))
        return self.out(o.mean(1))


@pytest.mark.parametrize("bits", [8, 32])
def test_a_training_step_eager_and_captured(bits):
    """Scan, its gradients, their norm and the update together: the captured step, replayed on other inputs, gives the eager steps' bits."""
    announce(f"training step in a graph, states in {bits} bits")
    gen = torch.Generator(device="cuda").manual_seed(9)
    inputs = [(torch.randn(4, 50, 64, device="cuda", generator=gen), torch.randint(0, 5, (4,), device="cuda", generator=gen)) for _ in range(6)]

    def made():
        torch.manual_seed(3)
        net = _Mixer(64).cuda()
        return net, optim.AdamW(net.parameters(), lr=1e-2, state_bits=bits, max_norm=0.1, capturable=True)

    def step(net, opt, x, y):
        params = list(net.parameters())
        loss = torch.nn.functional.cross_entropy(net(x), y)
        # (gradients as values: nothing accumulates into the leaves, whatever other graph holds them)
        for p, g in zip(params, torch.autograd.grad(loss, params)):
            p.grad = g
        opt.step()
        return loss.detach()

    eager = made()
    want = []
    for x, y in inputs:
        loss = step(*eager, x, y)
        want.append([loss] + [p.detach().clone() for p in eager[0].parameters()])
    net, opt = made()
    x, y = (t.clone() for t in inputs[0])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        first = step(net, opt, x, y)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(first, want[0][0])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        loss = step(net, opt, x, y)
    for (a, b), expected in zip(inputs[1:], want[1:]):
        x.copy_(a), y.copy_(b)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(loss, expected[0])
        assert all(torch.equal(p, q) for p, q in zip(net.parameters(), expected[1:]))
        torch.randn(1000, device="cuda").sum().item()  # (the program's own work in between)
