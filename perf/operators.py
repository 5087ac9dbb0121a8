"""The operators of a training step around a gated linear recurrence, as a dozen measurable cases and a generator of more.

    scan   vig_amd.gated_scan (causal, with a state in and out) and vig_amd.bid_gated_scan (both directions averaged) on
           [B, L, D] rows; with grad the gradients of the rows, of the gates and of the state too
    step   vig_amd.gated_scan_step, the recurrence for one more token of every sequence, its state updated in place
    adamw  vig_amd.adamw_step over a list of tensors, with states in 32 bits or in 8, and with clip the gradients' norm in
           front of it
    norm   vig_amd.grad_norm over a list of tensors

Widths, lengths and parameter lists are those of the ViG models (192, 384 and 768 channels, 196 tokens of a 224 x 224
image and 4096 of a 1024 x 1024 one, 180 parameters), longer sequences and odd sizes generic ones.
"""
import math
import random

import torch
import torch.nn.functional as F

own = False

DEV = "cuda"
DTYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}
BYTES = {"bf16": 2, "fp32": 4}
WIDTH = {"t": 192, "s": 384, "b": 768}
DEPTH, CLASSES = 12, 1000
LR, BETA1, BETA2, EPS, DECAY, MAX_NORM, SEED = 1e-3, 0.9, 0.999, 1e-8, 0.05, 1.0, 20240229

# the most a case may hold, as the listed cases do: channels of all tokens of a scan (a quarter with gradients, half in
# fp32), of a step's sequences, and parameters of a list
MOST_SCAN = 65536 * 1024
MOST_STEP = 2048 * 1024
MOST_PARAMETERS = 89_100_000


def _scan_case(name, B, L, D, dtype="bf16", both=False, state=False, grad=False, wide=False, packed=1):
    return {"name": name, "kind": "scan", "B": B, "L": L, "D": D, "dtype": dtype, "both": both, "state": state, "grad": grad, "wide": wide, "packed": packed}


def _adamw_case(name, model, bits, p, g, clip=False):
    return {"name": name, "kind": "adamw", "model": model, "bits": bits, "p": p, "g": g, "clip": clip, "tight": False}


def listed():
    return [
        # the mixer of one ViG-T layer on one image: latency and host time only
        _scan_case("scan_one_image", 1, 196, 192, both=True),
        # a ViG-S layer of the benchmark's batch, the rows in the columns of a projection's output
        _scan_case("scan_vig_s", 128, 196, 384, both=True, wide=True),
        # one long sequence, carried on from a state: few rows, a long axis
        _scan_case("scan_65536_tokens", 1, 65536, 1024, state=True),
        # training such a layer
        _scan_case("scan_grad_vig_s", 128, 196, 384, both=True, grad=True),
        # training in fp32 on seven images of different sizes packed behind one another, an odd length and width
        _scan_case("scan_grad_packed_fp32", 4, 2305, 333, dtype="fp32", grad=True, state=True, packed=7),
        # one more token of one sequence
        {"name": "step_one_sequence", "kind": "step", "B": 1, "D": 384, "dtype": "bf16"},
        # one more token of all sequences of a large serving batch
        {"name": "step_2048_sequences", "kind": "step", "B": 2048, "D": 1024, "dtype": "bf16"},
        # the update of a ViG-T, the smallest model: 180 tensors, the gradients clipped to a norm
        _adamw_case("adamw_vig_t_clipped", "t", 32, "fp32", "fp32", clip=True),
        # ... of a ViG-B, the largest
        _adamw_case("adamw_vig_b", "b", 32, "fp32", "fp32"),
        # states in 8 bits beside fp32 parameters
        _adamw_case("adamw_8_bit_vig_s", "s", 8, "fp32", "fp32"),
        # states in 8 bits beside parameters and gradients in bf16: the least memory
        _adamw_case("adamw_8_bit_vig_b_bf16", "b", 8, "bf16", "bf16"),
        # the norm of a ViG-B's gradients
        {"name": "norm_vig_b", "kind": "norm", "model": "b", "g": "bf16", "tight": False},
    ]


def _log_int(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    kind = rng.choice(["scan", "scan", "scan", "scan", "step", "adamw", "adamw", "norm"])
    if kind == "scan":
        grad, both, dtype = rng.random() < 0.5, rng.random() < 0.5, rng.choice(["bf16", "bf16", "fp32"])
        most = MOST_SCAN // (4 if grad else 1) // (2 if dtype == "fp32" else 1) // (2 if both else 1)
        L = _log_int(rng, 1, 65536)
        D = rng.choice([192, 384, 768, 8 * rng.randint(1, 128), rng.randint(1, 1024)])
        B = _log_int(rng, 1, max(1, min(4096, most // (L * D))))
        return {"kind": "scan", "B": B, "L": L, "D": D, "dtype": dtype, "both": both, "state": not both and rng.random() < 0.5, "grad": grad,
                "wide": rng.random() < 0.3, "packed": rng.choice([1, 1, min(L, rng.randint(2, 40))])}
    if kind == "step":
        B, dtype = _log_int(rng, 1, 2048), rng.choice(["bf16", "fp32"])
        return {"kind": "step", "B": B, "D": rng.choice([192, 384, 768, rng.randint(1, 1024)]), "dtype": dtype}
    many, low, high = _log_int(rng, 1, 400), rng.choice([1, 64, 1000]), _log_int(rng, 2000, 1 << 24)
    while many * high > 2 * MOST_PARAMETERS:
        high //= 2
    case = {"kind": kind, "model": "", "tensors": many, "low": low, "high": high, "sizes": rng.randint(0, 1 << 30), "g": rng.choice(["fp32", "fp32", "bf16"])}
    if kind == "norm":
        return {**case, "tight": rng.random() < 0.25}
    bits = rng.choice([8, 32])
    return {**case, "bits": bits, "p": case["g"] if rng.random() < 0.7 else rng.choice(["fp32", "bf16"]), "clip": rng.random() < 0.5,
            "tight": bits == 32 and rng.random() < 0.25}


def _sizes(case):
    """Elements of each tensor of the list: a model's parameters, or drawn ones."""
    if case["model"]:
        C = WIDTH[case["model"]]
        inner = 256 * math.ceil(C * 8 / 3 / 256)
        block = [C, 9 * C, 2 * C * C, 16 * C, 16 * C, C, C * C, 64, 64, C * C, C, C, 2 * inner * C, inner * C]
        return [196 * C, C // 2 * 243, C // 2, C // 2, C // 2, C * C // 2 * 9, C, C, C, CLASSES * C, CLASSES] + DEPTH * block + [C]
    rng, got, left = random.Random(case["sizes"]), [], MOST_PARAMETERS
    for _ in range(case["tensors"]):
        got.append(max(1, min(left, _log_int(rng, case["low"], case["high"]))))
        left = max(0, left - got[-1] - 256)
    return got


def _flat(sizes, tight):
    """(first elements of the tensors in one buffer, its length): behind one another, or each on a multiple of 256."""
    at, n = [], 0
    for s in sizes:
        at.append(n)
        n += s if tight else -(-s // 256) * 256
    return at, n


def _filled(at, sizes, n, values):
    """A buffer whose gaps between the tensors hold zeros."""
    flat = torch.zeros(n, device=DEV)
    if sum(sizes) == n:
        return values(n)
    keep = torch.zeros(n + 1, dtype=torch.int8, device=DEV)
    keep[torch.tensor(at, device=DEV)] += 1
    ends = torch.tensor([a + s for a, s in zip(at, sizes)], device=DEV)
    keep.index_add_(0, ends, torch.full_like(ends, -1, dtype=torch.int8))
    keep = keep.cumsum(0, dtype=torch.int8)[:n].bool()
    return torch.where(keep, values(n), flat)


def prepare(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    r = lambda *s: torch.randn(*s, device=DEV, generator=gen)  # noqa: E731
    state = {"case": case}
    if case["kind"] == "scan":
        # rows ~ N(0, 1), log-gates logsigmoid(N(0, 1)) / 16 as the models' gates are made; a packed sequence starts with a
        # gate that lets nothing through
        B, L, D, dtype = case["B"], case["L"], case["D"], DTYPES[case["dtype"]]
        x = r(B, L, 2 * D if case["wide"] else D).to(dtype)[..., :D]
        g = F.logsigmoid(r(2 * B if case["both"] else B, L, D)) / 16
        if case["packed"] > 1:
            starts = torch.tensor([i * L // case["packed"] for i in range(1, case["packed"])], device=DEV)
            g[:B, starts] = -math.inf
            if case["both"]:
                g[B:, starts - 1] = -math.inf
        state |= {"x": x, "g": g.to(dtype), "h0": r(B, D) if case["state"] else None}
        if case["grad"]:
            for k in ("x", "g", "h0"):
                if state[k] is not None:
                    state[k] = state[k].detach().requires_grad_()
            state["do"] = r(B, L, D).to(dtype)
            state["dh"] = r(B, D) if case["state"] else None
        return state
    if case["kind"] == "step":
        dtype = DTYPES[case["dtype"]]
        return state | {"x": r(case["B"], case["D"]).to(dtype), "g": (F.logsigmoid(r(case["B"], case["D"])) / 16).to(dtype), "h": r(case["B"], case["D"])}
    # tensors are slices of flat buffers, as a trainer that reduces its gradients in one piece keeps them
    sizes = _sizes(case)
    at, n = _flat(sizes, case["tight"])
    cut = lambda flat: [flat[a:a + s] for a, s in zip(at, sizes)]  # noqa: E731
    state["flat"] = flat = {"g": _filled(at, sizes, n, lambda n: r(n) * 1e-3).to(DTYPES[case["g"]])}
    if case["kind"] == "adamw":
        flat["p"] = _filled(at, sizes, n, lambda n: r(n) * 0.02).to(DTYPES[case["p"]])
        # (moments of a run under way: steps of about the size that the gradients have)
        m, v = _filled(at, sizes, n, lambda n: r(n) * 3e-4), _filled(at, sizes, n, lambda n: (0.5 + r(n).square()) * 5e-7)
        if case["bits"] == 32:
            flat |= {"m": m, "v": v}
        else:
            for k, t in (("m", m), ("r", v.sqrt())):
                scale = t.reshape(-1, 256).abs().amax(1) / 448
                flat[k] = (t.reshape(-1, 256) / scale.clamp_min(1e-30)[:, None]).to(torch.float8_e4m3fn).reshape(-1)
                flat[k + "s"] = scale
            blocks = [(a // 256, -(-(a + s) // 256)) for a, s in zip(at, sizes)]
            state |= {k: [flat[k][a:b] for a, b in blocks] for k in ("ms", "rs")}
        state["t"] = 1000
    return state | {k: cut(flat[k]) for k in flat if k not in ("ms", "rs")}


# ---- the plain forms: elementary operations in 32 bits, rounded once


def _scan(a, x):
    """h_t = a_t h_{t-1} + x_t along the second axis, from nothing: every second h by the same recurrence over pairs."""
    n = x.shape[1]
    if n == 1:
        return x
    m = n // 2
    odd = _scan(a[:, 1::2] * a[:, 0:2 * m:2], a[:, 1::2] * x[:, 0:2 * m:2] + x[:, 1::2])
    h = torch.empty_like(x)
    h[:, 0] = x[:, 0]
    h[:, 1::2] = odd
    h[:, 2::2] = a[:, 2::2] * odd[:, :(n - 1) // 2] + x[:, 2::2]
    return h


def _scan_back(a, x):
    return _scan(a.flip(1), x.flip(1)).flip(1)


def _scan_from(a, x, h0):
    return _scan(a, torch.cat([x[:, :1] + (a[:, 0] * h0)[:, None], x[:, 1:]], 1)) if h0 is not None else _scan(a, x)


def _behind(first, h):
    """h one token later, `first` (nothing: zeros) in front."""
    return torch.cat([torch.zeros_like(h[:, :1]) if first is None else first[:, None], h[:, :-1]], 1)


def _ahead(h):
    return torch.cat([h[:, 1:], torch.zeros_like(h[:, :1])], 1)


def _plain_scan(s):
    case, dtype, B = s["case"], s["x"].dtype, s["case"]["B"]
    x, a, h0 = s["x"].detach().float(), s["g"].detach().float().exp(), s["h0"].detach() if s["h0"] is not None else None
    h = _scan_from(a[:B], x, h0)
    both = case["both"]
    if both:
        hb = _scan_back(a[B:], x)
    out = {"o": ((h + hb) / 2 if both else h).to(dtype)}
    if case["state"]:
        out["h"] = h[:, -1].clone()
    if not case["grad"]:
        return out
    do = s["do"].float() / 2 if both else s["do"].float()
    last = do if s["dh"] is None else torch.cat([do[:, :-1], do[:, -1:] + s["dh"][:, None]], 1)
    dh = _scan_back(_ahead(a[:B]), last)
    dg = dh * a[:B] * _behind(h0, h)
    if both:
        dhb = _scan(_behind(None, a[B:]), do)
        out |= {"dx": (dh + dhb).to(dtype), "dg": torch.cat([dg, dhb * a[B:] * _ahead(hb)]).to(dtype)}
    else:
        out |= {"dx": dh.to(dtype), "dg": dg.to(dtype)}
    if h0 is not None:
        out["dh0"] = dh[:, 0] * a[:B][:, 0]
    return out


M32 = 0xFFFFFFFF
GOLDEN, ROOT2, ROOT3 = 0x9E3779B9, 0x6A09E667, 0xBB67AE85  # 2^32 times the fractional parts of the golden ratio and of two roots


def _mix(x):
    """One 32-bit word from another: each bit of x decides about every bit of it."""
    x = ((x ^ (x >> 16)) * ROOT2) & M32
    x = ((x ^ (x >> 15)) * ROOT3) & M32
    return x ^ (x >> 16)


def _key(seed, t):
    return _mix((_mix((_mix(seed & M32) + (seed >> 32)) & M32) + t) & M32)


def _wrapped(v):
    return v - (1 << 32) if v >= 1 << 31 else v


def _words(n, key):
    """The random word of each element: _mix() of its number and the key, in 32-bit integers that wrap."""
    x = torch.arange(n, device=DEV, dtype=torch.int64).to(torch.int32) ^ _wrapped(key)
    x = (x ^ ((x >> 16) & 0xFFFF)) * _wrapped(ROOT2)
    x = (x ^ ((x >> 15) & 0x1FFFF)) * _wrapped(ROOT3)
    return x ^ ((x >> 16) & 0xFFFF)


def _to_8_bits(x, u, least=False):
    """(e4m3 codes, scales) of fp32 values in blocks of 256, rounded up where u in [0, 1) reaches past the distance."""
    x = x.reshape(-1, 256)
    scale = x.abs().amax(1) / 448
    y = torch.where(scale[:, None] > 0, x.abs() / scale[:, None], 0)
    step = torch.ldexp(torch.ones_like(y), (torch.frexp(y)[1] - 1).clamp_min(-6) - 3)
    q = torch.floor(y / step + u.reshape(-1, 256)) * step
    if least:
        q = torch.where(x > 0, q.clamp_min(2.0 ** -9), q)
    return torch.copysign(q, x).to(torch.float8_e4m3fn).reshape(-1), scale


def _from_8_bits(q, scale):
    return (q.float().reshape(-1, 256) * scale[:, None]).reshape(-1)


def _plain_norm(g):
    norm = g.float().square().sum().sqrt()
    return norm, (MAX_NORM / (norm + 1e-6)).clamp_max(1.0)


def _plain_adamw(s):
    case, f = s["case"], s["flat"]
    s["t"] += 1
    p, g = f["p"].float(), f["g"].float()
    norm = None
    if case["clip"]:
        norm, scale = _plain_norm(f["g"])
        g = g * scale
    m, v = (f["m"], f["v"]) if case["bits"] == 32 else (_from_8_bits(f["m"], f["ms"]), _from_8_bits(f["r"], f["rs"]).square())
    m, v = BETA1 * m + (1 - BETA1) * g, BETA2 * v + (1 - BETA2) * g * g
    root = v.sqrt()
    p = p * (1 - LR * DECAY) - LR / (1 - BETA1 ** s["t"]) * m / (root / math.sqrt(1 - BETA2 ** s["t"]) + EPS)
    w = _words(p.numel(), _key(SEED, s["t"])) if case["bits"] == 8 or case["p"] == "bf16" else None
    if case["p"] == "bf16":
        u = ((w * _wrapped(GOLDEN)) >> 16) & 0xFFFF
        p = ((p.view(torch.int32) + u) & -65536).view(torch.float32)
    f["p"].copy_(p)
    if case["bits"] == 32:
        f["m"].copy_(m)
        f["v"].copy_(v)
    else:
        for k, t, u in (("m", m, w & 0xFFFF), ("r", root, (w >> 16) & 0xFFFF)):
            q, scale = _to_8_bits(t, u.float() / 65536, least=k == "r")
            f[k].copy_(q)
            f[k + "s"].copy_(scale)
    return {k: f[k] for k in f if k != "g"} | ({} if norm is None else {"norm": norm})


def run(state):
    case = state["case"]
    if own:
        return _own(state)
    if case["kind"] == "scan":
        return _plain_scan(state)
    if case["kind"] == "step":
        state["h"].mul_(state["g"].float().exp()).add_(state["x"])
        return {"o": state["h"].to(state["x"].dtype), "h": state["h"]}
    if case["kind"] == "norm":
        return _plain_norm(state["flat"]["g"])
    return _plain_adamw(state)


def _own(state):
    import vig_amd

    case = state["case"]
    if case["kind"] == "scan":
        x, g, h0 = state["x"], state["g"], state["h0"]
        if case["both"]:
            o, h = vig_amd.bid_gated_scan(x, g)[0], None
        else:
            o, h = vig_amd.gated_scan(x, g, initial_state=h0, output_final_state=case["state"])
        out = {"o": o.detach()} | ({"h": h.detach()} if case["state"] else {})
        if case["grad"]:
            inputs = [t for t in (x, g, h0) if t is not None]
            outputs, given = ([o, h], [state["do"], state["dh"]]) if case["state"] else ([o], [state["do"]])
            out |= dict(zip(("dx", "dg", "dh0"), torch.autograd.grad(outputs, inputs, given)))
        return out
    if case["kind"] == "step":
        return {"o": vig_amd.gated_scan_step(state["x"], state["g"], state["h"]), "h": state["h"]}
    if case["kind"] == "norm":
        return vig_amd.grad_norm(state["g"], max_norm=MAX_NORM)
    state["t"] += 1
    norm = scale = None
    if case["clip"]:
        norm, scale = vig_amd.grad_norm(state["g"], max_norm=MAX_NORM)
    moments = (state["m"], state["v"]) if case["bits"] == 32 else (state["m"], state["r"], state["ms"], state["rs"])
    # (elements are numbered by their places in the flat buffers; tensors in whole blocks of 256 are so by themselves)
    first = [t.storage_offset() for t in state["p"]] if case["tight"] and case["p"] == "bf16" else None
    vig_amd.adamw_step(state["p"], state["g"], *moments, step=state["t"], lr=LR, betas=(BETA1, BETA2), eps=EPS, weight_decay=DECAY, grad_scale=scale, seed=SEED, first=first)
    return {k: v for k, v in state["flat"].items() if k != "g"} | ({} if norm is None else {"norm": norm})


def work(case):
    if case["kind"] == "scan":
        e, n = BYTES[case["dtype"]], case["B"] * case["L"] * case["D"]
        ways = 2 if case["both"] else 1
        moved, ops = 2 + ways, 4 * ways  # rows, gates, output; the gate's exponential, a product, two sums
        if case["grad"]:
            moved += 2 + ways  # output's gradient, rows' and gates' gradients
            ops += 8 * ways
        states = case["B"] * case["D"] * 4 * (4 if case["grad"] else 2) if case["state"] else 0
        return {"bytes": n * moved * e + states, "flops": n * ops}
    if case["kind"] == "step":
        n = case["B"] * case["D"]
        return {"bytes": n * (3 * BYTES[case["dtype"]] + 8), "flops": 4 * n}
    n, g = sum(_sizes(case)), BYTES[case["g"]]
    if case["kind"] == "norm":
        return {"bytes": n * g, "flops": 2 * n}
    states = 16 if case["bits"] == 32 else 4 + 16 / 256
    return {"bytes": n * (2 * BYTES[case["p"]] + g + states), "flops": 15 * n}


# ---- the definitions in 64 bits, token by token and element by element


def _walk(a, x, h, tokens, before=False):
    """h = a_t h + x_t along `tokens`; every h behind its token, or in front of it (a_t h of that one)."""
    out = torch.empty_like(x)
    for t in tokens:
        if before:
            torch.mul(a[t], h, out=out[t])
            h = out[t] + x[t]
        else:
            h = torch.addcmul(x[t], a[t], h, out=out[t])
    return out


def _exact_scan(case, s):
    B, L = case["B"], case["L"]
    tokens_first = lambda t: t.detach().double().transpose(0, 1).contiguous()  # noqa: E731
    back = lambda t, name: t.transpose(0, 1) if name else t  # noqa: E731
    x, g = tokens_first(s["x"]), tokens_first(s["g"])
    x = x.contiguous()
    zero = torch.zeros_like(x[0])
    h0 = s["h0"].detach().double() if s["h0"] is not None else zero
    ways = [(g[:, :B].exp().contiguous(), range(L), h0)] + ([(g[:, B:].exp().contiguous(), range(L - 1, -1, -1), zero)] if case["both"] else [])
    h = [_walk(a, x, start, order) for a, order, start in ways]
    got = {"o": back(sum(h) / len(h), True)}
    if case["state"]:
        got["h"] = h[0][-1]
    if not case["grad"]:
        return got
    do = tokens_first(s["do"]) / len(ways)
    dx, dg = torch.zeros_like(x), []
    for k, (a, order, start) in enumerate(ways):
        held = _walk(a, x, start, order, before=True)
        d, grad = (s["dh"].double() if s["dh"] is not None else zero), torch.empty_like(x)
        for t in reversed(order):
            d = d + do[t]
            dx[t] += d
            grad[t] = d * held[t]
            d = d * a[t]
        dg.append(back(grad, True))
        if k == 0 and s["h0"] is not None:
            got["dh0"] = d
    return got | {"dx": back(dx, True), "dg": torch.cat(dg)}


def _exact_codes(x, bits, least):
    """The e4m3 values around x in units of its block's scale: the one below, or the next one where the 16 random bits fall short of x's share."""
    x = x.reshape(-1, 256)
    scale = x.abs().max(1, keepdim=True).values / 448
    y = (x.abs() / scale).nan_to_num(0.0)
    gap = torch.exp2(torch.floor(torch.log2(y.clamp_min(2.0 ** -6))) - 3)
    low = torch.floor(y / gap)
    q = (low + (((y / gap - low) + bits.reshape(-1, 256).double() / 65536) >= 1).double()) * gap
    if least:
        q = torch.where((x > 0) & (q == 0), torch.full_like(q, 2.0 ** -9), q)
    return (q * torch.sign(x)).reshape(-1), scale.reshape(-1)


def _exact_words(n, key):
    x = torch.arange(n, device=DEV) ^ key
    for shift, factor in ((16, ROOT2), (15, ROOT3)):
        x = x ^ (x >> shift)
        # (a product of two 32-bit words by halves: it passes 63 bits)
        x = ((x * (factor & 0xFFFF)) + (((x & 0xFFFF) * (factor >> 16)) << 16)) & M32
    return x ^ (x >> 16)


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "scan":
        return _exact_scan(case, s)
    if case["kind"] == "step":
        h = s["g"].double().exp() * s["h"].double() + s["x"].double()
        return {"o": h, "h": h}
    f = s["flat"]
    norm = torch.linalg.vector_norm(f["g"].double())
    clip = min(1.0, MAX_NORM / (float(norm) + 1e-6))
    if case["kind"] == "norm":
        return norm, torch.tensor(clip, dtype=torch.float64)
    t, g = s["t"] + 1, f["g"].double() * (clip if case["clip"] else 1.0)
    wide = lambda k: f[k].double() * f[k + "s"].double().repeat_interleave(256)  # noqa: E731
    m, v = (f["m"].double(), f["v"].double()) if case["bits"] == 32 else (wide("m"), wide("r") ** 2)
    m, v = m + (1 - BETA1) * (g - m), v + (1 - BETA2) * (g * g - v)
    del g
    first, second = 1 - BETA1 ** t, 1 - BETA2 ** t
    p = f["p"].double()
    p = p - LR * (DECAY * p + (m / first) / ((v / second).sqrt() + EPS))
    got = {"p": p, "m": m, "v": v} if case["bits"] == 32 else {}
    if case["bits"] == 8 or case["p"] == "bf16":
        w = _exact_words(p.numel(), _key(SEED, t))
    if case["bits"] == 8:
        q, scale = _exact_codes(m, w & 0xFFFF, False)
        got |= {"p": p, "m": q, "ms": scale}
        del q, m
        q, scale = _exact_codes(v.sqrt(), w >> 16, True)
        got |= {"r": q, "rs": scale}
        del q, v
    if case["p"] == "bf16":
        # the bf16 value towards zero, or the next one behind it where the bits and p's share of the step reach one
        u = ((((w & 0xFFFF) * (GOLDEN & 0xFFFF)) + (((((w >> 16) * (GOLDEN & 0xFFFF)) + ((w & 0xFFFF) * (GOLDEN >> 16))) & 0xFFFF) << 16)) & M32) >> 16
        gap = torch.exp2(torch.floor(torch.log2(p.abs().clamp_min(2.0 ** -126))) - 7)
        got["p"] = torch.sign(p) * torch.floor(p.abs() / gap + u.double() / 65536) * gap
    return got | ({"norm": norm} if case["clip"] else {})
