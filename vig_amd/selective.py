"""The selective state space mixer's operators: the scan with its step for one token, the short causal convolution in front of it with its step, and the
residual add and layer norm in front of both.

Beside the gated scan (ops.gated_scan), whose state is one number a channel with a decay of its own, the selective scan holds N numbers a channel, read and written
through rows B and C that the channels of a group share.  All are differentiable once, in reverse mode; forward-mode derivatives are refused, a trace or dispatch
mode sees torch.ops.vig_amd operators, and leaves that a graph recorded on the default stream still holds are refused in a capture that records gradients.
"""
from __future__ import annotations

import ctypes
from typing import Optional, Tuple

import torch

from . import _ext, _lib, ops
from .ops import _dt, _operator, _refuse_held_leaves, _refuse_tangents, _scan_rows, _scan_strides

MOST_STATES = 64  # of a channel
MOST_WIDTH = 16384  # of a layer norm's rows


def _ptr(t):
    return t.data_ptr() if t is not None else None


def _needs_graph(*ts):
    return torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in ts)


def _number(name, t, shape, like):
    """A parameter or state as the kernels take it: float32, packed."""
    if t is None:
        return None
    if tuple(t.shape) != tuple(shape):
        raise ValueError(f"{name} must be {list(shape)}; got {list(t.shape)}")
    if not t.is_floating_point():
        raise TypeError(f"{name} must be a floating point tensor")
    return t.float()


def _same_type(x, **others):
    _dt(x)
    for name, t in others.items():
        if t is not None and t.dtype != x.dtype:
            raise TypeError(f"{name} must have x's dtype {x.dtype}; got {t.dtype}")


# ---------------------------------------------------------------------------
# selective scan
# ---------------------------------------------------------------------------

def selective_scan(x: torch.Tensor, delta: torch.Tensor, A: torch.Tensor, B: torch.Tensor, C: torch.Tensor, D: Optional[torch.Tensor] = None,
                   z: Optional[torch.Tensor] = None, delta_bias: Optional[torch.Tensor] = None, delta_softplus: bool = False,
                   initial_state: Optional[torch.Tensor] = None, output_final_state: bool = False,
                   reverse: bool = False) -> Tuple[torch.Tensor, Optional[torch.Tensor]]:
    """s_t = softplus(delta_t + delta_bias),  h_t = e^{s_t A} h_{t-1} + s_t x_t B_t,  o_t = (C_t h_t + D x_t) silu(z_t):  (o, final_state or None).

    x, delta, z: [B,L,D] in fp32 or bf16, B and C of that type too: [B,L,N], or [B,L,G,N] for G groups of D/G channels side by side, N up to 64.  A [D,N] (its values <= 0), D and
    delta_bias [D]; without delta_softplus the steps are delta + delta_bias as they are (>= 0).  No D: nothing is skipped; no z: no gate.  initial_state and final_state: fp32 [B,D,N], in
    front of the first token of the walk and behind its last.  reverse: the walk goes from the last token to the first (the other direction of a bidirectional mixer, without
    turning anything round).  A token whose step is 0 (delta of -infinity in front of the softplus) and whose x and B are finite leaves the state as it is: padding.  A value of x
    or delta that is not finite stays in its sequence's channel, where every later output is not finite then, and in gradients of the rows that channels share; one of B or C reaches its group's.
    x, delta, z, B, C may be columns of wider rows (read in place).  Up to 2^24 tokens of 2^18 channels, G N up to 2^18, batch G ceil(D / G / 64) below 2^24; with gradients batch L G N
    (N rounded up to a power of two, 4 at least) below 2^33.  States and sums are held in fp32, in an order fixed by the sizes.
    Differentiable in every tensor; the forward then keeps the state in front of every 16th token (8th above 16, 4th above 32 states): 4 bytes a channel and token at 16 states, 16 at
    32, 64 at 64."""
    calls = _ext.calls()
    if calls is not None:  # one native call for what the kernels take; None: not of that kind
        r = calls.selective_scan(x, delta, A, B, C, D, z, delta_bias, initial_state, delta_softplus, reverse, output_final_state)
        if r is not None:
            return r if output_final_state else (r, None)
    ops._check_cuda(x, delta, A, B, C, D, z, delta_bias, initial_state)
    if x.dim() != 3 or delta.shape != x.shape or (z is not None and z.shape != x.shape):
        raise ValueError("x, delta and z must be [B,L,D] of the same sizes")
    _check_shared(x, B, C, x.shape[:2])
    _same_type(x, delta=delta, B=B, C=C, z=z)
    given = (x, delta, A, B, C, D, z, delta_bias, initial_state)
    _refuse_tangents("selective_scan", *given)
    _refuse_held_leaves(*given, by="selective_scan")
    batch, L, width = x.shape
    N = B.shape[-1]
    A, D, delta_bias = _number("A", A, (width, N), x), _number("D", D, (width,), x), _number("delta_bias", delta_bias, (width,), x)
    h0 = _number("initial_state", initial_state, (batch, width, N), x)
    if x.numel() == 0:  # nothing happens to the state
        h = h0 if h0 is not None else torch.zeros(batch, width, N, dtype=torch.float32, device=x.device)
        return x.clone(), h.clone() if output_final_state else None
    if _needs_graph(x, delta, A, B, C, D, z, delta_bias, h0):
        return _SelectiveScan.apply(x, delta, A, B, C, D, z, delta_bias, h0, bool(delta_softplus), bool(reverse), bool(output_final_state))
    return _scan_forward(x, delta, A, B, C, D, z, delta_bias, h0, bool(delta_softplus), bool(reverse), bool(output_final_state), False)[:2]


def _check_shared(x, B, C, front):
    n = len(front)
    if B.shape != C.shape or B.dim() not in (n + 1, n + 2) or B.shape[:n] != front:
        raise ValueError(f"B and C must be {'[B,L,N] or [B,L,G,N]' if n == 2 else '[B,N] or [B,G,N]'}, of x's leading sizes and alike")
    N, G = B.shape[-1], B.shape[-2] if B.dim() == n + 2 else 1
    if not 1 <= N <= MOST_STATES:
        raise ValueError(f"1 to {MOST_STATES} states a channel are built; got {N}")
    if G < 1 or x.shape[-1] % G:
        raise ValueError(f"{x.shape[-1]} channels do not make {G} groups")


def _shared_rows(t, dims):
    """B or C with its axis of groups, its states side by side in rows that do not overlap, else packed."""
    if t.dim() == dims:
        t = t.unsqueeze(-2)
    G, N = t.shape[-2:]
    if N > 1 and t.stride(-1) != 1:
        return t.contiguous()
    apart = (G - 1) * t.stride(-2) + N if G > 1 else N
    # (a token alone is as far from the next as its groups reach)
    if (G > 1 and t.stride(-2) < N) or (dims == 3 and not apart <= (t.stride(1) if t.shape[1] > 1 else apart) <= 1 << 18):
        return t.contiguous()
    return t


def _shared_strides(t):
    """Of batch element, token (of [B,L,G,N]) and group."""
    G, N = t.shape[-2:]
    group = t.stride(-2) if G > 1 else N
    whole = (G - 1) * group + N
    if t.dim() == 3:
        return (ctypes.c_longlong * 2)(t.stride(0) if t.shape[0] > 1 else 0, group)
    return (ctypes.c_longlong * 3)(t.stride(0) if t.shape[0] > 1 else 0, t.stride(1) if t.shape[1] > 1 else whole, group)


def _scan_call(x, delta, A, B, C, D, z, bias):
    """The tensors as the kernels take them, and what a call says of them."""
    x, delta, z = (_scan_rows(t) if t is not None else None for t in (x, delta, z))
    B, C = _shared_rows(B, 3), _shared_rows(C, 3)
    A, D, bias = (t.contiguous() if t is not None else None for t in (A, D, bias))
    batch, L, width = x.shape
    G, N = B.shape[-2:]
    sizes = (batch, L, width, N, G)
    strides = (_scan_strides(x), _scan_strides(delta), _shared_strides(B), _shared_strides(C), _scan_strides(z) if z is not None else None)
    return (x, delta, A, B, C, D, z, bias), sizes, strides


def _scan_forward(x, delta, A, B, C, D, z, bias, h0, softplus, reverse, want_final, keep):
    if ops.observed():
        o, h, kept = torch.ops.vig_amd.selective_scan_fwd(x, delta, A, B, C, D, z, bias, h0, softplus, reverse, keep)
        return o, h if want_final else None, kept if keep else None
    return _scan_launch(x, delta, A, B, C, D, z, bias, h0, softplus, reverse, want_final, keep)


def _scan_launch(x, delta, A, B, C, D, z, bias, h0, softplus, reverse, want_final, keep):
    lib = _lib.load()
    ops._check_cuda(x, delta, A, B, C, D, z, bias, h0)
    tensors, sizes, strides = _scan_call(x, delta, A, B, C, D, z, bias)
    h0 = h0.contiguous() if h0 is not None else None
    batch, L, width, N, G = sizes
    o = torch.empty(batch, L, width, dtype=x.dtype, device=x.device)
    h = torch.empty(batch, width, N, dtype=torch.float32, device=x.device) if want_final else None
    kept = torch.empty(lib.vig_selective_scan_kept(batch, L, width, N), dtype=torch.uint8, device=x.device) if keep else None
    need = lib.vig_selective_scan_fwd_workspace(*sizes)
    ws = torch.empty(need, dtype=torch.uint8, device=x.device) if need else None
    with torch.cuda.device(x.device):
        rc = lib.vig_selective_scan_fwd(*(_ptr(t) for t in tensors), _ptr(h0), _ptr(o), _ptr(h), _ptr(kept), _ptr(ws), need, *sizes, *strides, int(softplus), int(reverse),
                                        _dt(x), ops._stream_ptr(x))
    _lib.check(rc, "vig_selective_scan_fwd")
    return o, h, kept


class _SelectiveScan(torch.autograd.Function):
    """Autograd node of the selective scan: forward and backward each the library's kernels."""

    @staticmethod
    def forward(ctx, x, delta, A, B, C, D, z, bias, h0, softplus, reverse, want_final):
        o, h, kept = _scan_forward(x, delta, A, B, C, D, z, bias, h0, softplus, reverse, want_final, True)
        ctx.save_for_backward(x, delta, A, B, C, D, z, bias, kept)
        ctx.flags = softplus, reverse
        ctx.has_state = h0 is not None
        ctx.set_materialize_grads(False)
        return o, h

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, d_o, d_final):
        x, delta, A, B, C, D, z, bias, kept = ctx.saved_tensors
        d_o = d_o if d_o is not None else torch.zeros(x.shape, dtype=x.dtype, device=x.device)
        wanted = ctx.has_state and ctx.needs_input_grad[8]
        call = torch.ops.vig_amd.selective_scan_bwd if ops.observed() else _scan_backward
        dx, ddelta, dB, dC, dz, dparams, dh0 = call(x, delta, A, B, C, D, z, bias, kept, d_o, d_final, *ctx.flags, wanted)
        width, N = A.shape
        dA, dD, dbias = dparams[:width * N].view(width, N), dparams[width * N:-width], dparams[-width:]
        return dx, ddelta, dA, dB, dC, dD if D is not None else None, dz if z is not None else None, dbias if bias is not None else None, dh0 if wanted else None, None, None, None


def _scan_backward(x, delta, A, B, C, D, z, bias, kept, d_o, d_final, softplus, reverse, want_state):
    lib = _lib.load()
    ops._check_cuda(x, delta, A, B, C, D, z, bias, kept, d_o, d_final)
    d_o, d_final = d_o.contiguous(), d_final.contiguous() if d_final is not None else None
    tensors, sizes, strides = _scan_call(x, delta, A, B, C, D, z, bias)
    batch, L, width, N, G = sizes
    new = lambda t: torch.empty(t.shape, dtype=t.dtype, device=t.device)  # noqa: E731
    dx, ddelta, dB, dC = new(x), new(delta), new(B), new(C)
    dz = new(z) if z is not None else None
    dparams = torch.empty(width * (N + 2), dtype=torch.float32, device=x.device)
    dh0 = torch.empty(batch, width, N, dtype=torch.float32, device=x.device) if want_state else None
    need = lib.vig_selective_scan_bwd_workspace(*sizes)
    ws = torch.empty(need, dtype=torch.uint8, device=x.device)
    with torch.cuda.device(x.device):
        rc = lib.vig_selective_scan_bwd(*(_ptr(t) for t in tensors), _ptr(kept), _ptr(d_o), _ptr(d_final), _ptr(dx), _ptr(ddelta), _ptr(dB), _ptr(dC), _ptr(dz), _ptr(dparams),
                                        _ptr(dh0), _ptr(ws), need, *sizes, *strides, int(softplus), int(reverse), _dt(x), ops._stream_ptr(x))
    _lib.check(rc, "vig_selective_scan_bwd")
    return dx, ddelta, dB, dC, dz, dparams, dh0


def selective_scan_step(x: torch.Tensor, delta: torch.Tensor, A: torch.Tensor, B: torch.Tensor, C: torch.Tensor, state: torch.Tensor, D: Optional[torch.Tensor] = None,
                        z: Optional[torch.Tensor] = None, delta_bias: Optional[torch.Tensor] = None, delta_softplus: bool = False) -> torch.Tensor:
    """selective_scan for one token of every sequence: x, delta, z [B,D], B and C [B,N] or [B,G,N]; state (fp32 [B,D,N], contiguous, apart from the others' memory) is moved on
    in place, the output returned in x's dtype.  Inference only."""
    calls = _ext.calls()
    if calls is not None:
        o = calls.selective_scan_step(x, delta, A, B, C, D, z, delta_bias, state, delta_softplus)
        if o is not None:
            return o
    ops._check_cuda(x, delta, A, B, C, state, D, z, delta_bias)
    given = (x, delta, A, B, C, state, D, z, delta_bias)
    if _needs_graph(*given):
        raise ValueError("selective_scan_step updates its state in place and records no gradient; use selective_scan")
    _refuse_tangents("selective_scan_step", *given)
    if x.dim() != 2 or delta.shape != x.shape or (z is not None and z.shape != x.shape):
        raise ValueError("x, delta and z must be [B,D] of the same sizes")
    _check_shared(x, B, C, x.shape[:1])
    _same_type(x, delta=delta, B=B, C=C, z=z)
    batch, width = x.shape
    N = B.shape[-1]
    if state.shape != (batch, width, N) or state.dtype != torch.float32 or not state.is_contiguous():
        raise ValueError(f"state must be a contiguous float32 tensor {[batch, width, N]} (it is updated in place)")
    A, D, delta_bias = _number("A", A, (width, N), x), _number("D", D, (width,), x), _number("delta_bias", delta_bias, (width,), x)
    call = torch.ops.vig_amd.selective_scan_step if ops.observed() else _step_launch
    return call(x, delta, A, B, C, state, D, z, delta_bias, bool(delta_softplus))


def _step_launch(x, delta, A, B, C, state, D, z, bias, softplus):
    lib = _lib.load()
    ops._check_cuda(x, delta, A, B, C, state, D, z, bias)
    batch, width = x.shape
    o = torch.empty(batch, width, dtype=x.dtype, device=x.device)
    if x.numel() == 0:
        return o
    x, delta, z = (_scan_rows(t) if t is not None else None for t in (x, delta, z))
    B, C = _shared_rows(B, 2), _shared_rows(C, 2)
    A, D, bias = (t.contiguous() if t is not None else None for t in (A, D, bias))
    pitch = lambda t: t.stride(0) if t is not None and batch > 1 else width  # noqa: E731
    with torch.cuda.device(x.device):
        rc = lib.vig_selective_scan_step(_ptr(x), _ptr(delta), _ptr(A), _ptr(B), _ptr(C), _ptr(D), _ptr(z), _ptr(bias), _ptr(state), _ptr(o), batch, width, B.shape[-1], B.shape[-2],
                                         pitch(x), pitch(delta), _shared_strides(B), _shared_strides(C), pitch(z), int(softplus), _dt(x), ops._stream_ptr(x))
    _lib.check(rc, "vig_selective_scan_step")
    _written(state)
    return o


def _written(t):
    if not t.is_inference():
        torch.autograd.graph.increment_version(t)


# ---------------------------------------------------------------------------
# short causal convolution
# ---------------------------------------------------------------------------

def causal_conv1d(x: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor] = None, silu: bool = False, initial_state: Optional[torch.Tensor] = None,
                  output_final_state: bool = False, reverse: bool = False) -> Tuple[torch.Tensor, Optional[torch.Tensor]]:
    """Depthwise causal convolution along the tokens: y_t = f(bias + sum_k weight[k] x_{t-W+1+k}), f silu or nothing:  (y, final_state or None).

    x: [B,L,D] in fp32 or bf16, or columns of wider rows (read in place); weight [D,W] (or [D,1,W], as torch.nn.Conv1d has it), W 2, 3 or 4; bias [D].  initial_state: the W - 1 rows in
    front of the first token, [B,W-1,D] of x's dtype (zeros without it); final_state: the last W - 1 rows, for what follows.  reverse: the walk goes from the last token to the first, and the
    states' rows with it.  Sums are held in fp32, in an order fixed by the sizes and by how the rows lie.  Differentiable in every tensor."""
    calls = _ext.calls()
    if calls is not None:
        r = calls.causal_conv1d(x, weight, bias, initial_state, silu, reverse, output_final_state)
        if r is not None:
            return r if output_final_state else (r, None)
    ops._check_cuda(x, weight, bias, initial_state)
    if x.dim() != 3:
        raise ValueError("x must be [B,L,D]")
    given = (x, weight, bias, initial_state)
    _refuse_tangents("causal_conv1d", *given)
    _refuse_held_leaves(*given, by="causal_conv1d")
    batch, L, width = x.shape
    w = _taps(weight, width)
    W = w.shape[1]
    b = _number("bias", bias, (width,), x)
    _same_type(x, initial_state=initial_state)
    if initial_state is not None and initial_state.shape != (batch, W - 1, width):
        raise ValueError(f"initial_state must be {[batch, W - 1, width]}; got {list(initial_state.shape)}")
    if x.numel() == 0:
        h = initial_state if initial_state is not None else x.new_zeros(batch, W - 1, width)
        return x.clone(), h.clone() if output_final_state else None
    if _needs_graph(x, w, b, initial_state):
        return _CausalConv.apply(x, w, b, initial_state, bool(silu), bool(reverse), bool(output_final_state))
    return _conv_forward(x, w, b, initial_state, bool(silu), bool(reverse), bool(output_final_state))


def _taps(weight, width):
    if weight.dim() == 3 and weight.shape[1] == 1:
        weight = weight.squeeze(1)
    if weight.dim() != 2 or weight.shape[0] != width or not 2 <= weight.shape[1] <= 4:
        raise ValueError(f"weight must be [{width},W] with W 2, 3 or 4; got {list(weight.shape)}")
    return _number("weight", weight, weight.shape, weight)


def _conv_forward(x, w, b, h0, silu, reverse, want_final):
    if ops.observed():
        y, h = torch.ops.vig_amd.causal_conv1d_fwd(x, w, b, h0, silu, reverse)
        return y, h if want_final else None
    return _conv_launch(x, w, b, h0, silu, reverse, want_final)


def _conv_launch(x, w, b, h0, silu, reverse, want_final):
    lib = _lib.load()
    ops._check_cuda(x, w, b, h0)
    x, w = _scan_rows(x), w.contiguous()
    b, h0 = (t.contiguous() if t is not None else None for t in (b, h0))
    batch, L, width = x.shape
    W = w.shape[1]
    y = torch.empty(batch, L, width, dtype=x.dtype, device=x.device)
    h = torch.empty(batch, W - 1, width, dtype=x.dtype, device=x.device) if want_final else None
    with torch.cuda.device(x.device):
        rc = lib.vig_causal_conv1d_fwd(_ptr(x), _ptr(w), _ptr(b), _ptr(h0), _ptr(y), _ptr(h), batch, L, width, W, _scan_strides(x), int(silu), int(reverse), _dt(x), ops._stream_ptr(x))
    _lib.check(rc, "vig_causal_conv1d_fwd")
    return y, h


class _CausalConv(torch.autograd.Function):
    """Autograd node of the short convolution: forward and backward each the library's kernels."""

    @staticmethod
    def forward(ctx, x, w, b, h0, silu, reverse, want_final):
        ctx.save_for_backward(x, w, b, h0)
        ctx.flags = silu, reverse
        ctx.set_materialize_grads(False)
        return _conv_forward(x, w, b, h0, silu, reverse, want_final)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy, d_final):
        x, w, b, h0 = ctx.saved_tensors
        dy = dy if dy is not None else torch.zeros(x.shape, dtype=x.dtype, device=x.device)
        state, params = h0 is not None and ctx.needs_input_grad[3], ctx.needs_input_grad[1] or ctx.needs_input_grad[2]
        call = torch.ops.vig_amd.causal_conv1d_bwd if ops.observed() else _conv_backward
        dx, dparams, dh0 = call(x, w, b, h0, dy, d_final, *ctx.flags, state, params)
        n = w.numel()
        return dx, dparams[:n].view(w.shape) if params else None, dparams[n:] if params and b is not None else None, dh0 if state else None, None, None, None


def _conv_backward(x, w, b, h0, dy, d_final, silu, reverse, want_state, want_params):
    lib = _lib.load()
    ops._check_cuda(x, w, b, h0, dy, d_final)
    x, w, dy = _scan_rows(x), w.contiguous(), dy.contiguous()
    b, h0, d_final = (t.contiguous() if t is not None else None for t in (b, h0, d_final))
    batch, L, width = x.shape
    W = w.shape[1]
    dx = torch.empty(batch, L, width, dtype=x.dtype, device=x.device)
    dh0 = torch.empty(batch, W - 1, width, dtype=x.dtype, device=x.device) if want_state else None
    dparams = torch.empty(width * (W + 1), dtype=torch.float32, device=x.device) if want_params else None
    need = lib.vig_causal_conv1d_bwd_workspace(batch, L, width, W) if want_params else 0
    ws = torch.empty(need, dtype=torch.uint8, device=x.device) if need else None
    with torch.cuda.device(x.device):
        rc = lib.vig_causal_conv1d_bwd(_ptr(x), _ptr(w), _ptr(b), _ptr(h0), _ptr(dy), _ptr(d_final), _ptr(dx), _ptr(dh0), _ptr(dparams), _ptr(ws), need, batch, L, width, W,
                                       _scan_strides(x), int(silu), int(reverse), _dt(x), ops._stream_ptr(x))
    _lib.check(rc, "vig_causal_conv1d_bwd")
    return dx, dparams, dh0


def causal_conv1d_step(x: torch.Tensor, weight: torch.Tensor, state: torch.Tensor, bias: Optional[torch.Tensor] = None, silu: bool = False) -> torch.Tensor:
    """causal_conv1d for one token of every sequence: x [B,D]; state, the W - 1 rows in front ([B,W-1,D] of x's dtype, contiguous, apart from x's memory), takes x in and lets its
    oldest row go, in place.  Inference only."""
    calls = _ext.calls()
    if calls is not None:
        y = calls.causal_conv1d_step(x, weight, state, bias, silu)
        if y is not None:
            return y
    ops._check_cuda(x, weight, state, bias)
    if _needs_graph(x, weight, state, bias):
        raise ValueError("causal_conv1d_step updates its state in place and records no gradient; use causal_conv1d")
    _refuse_tangents("causal_conv1d_step", x, weight, state, bias)
    if x.dim() != 2:
        raise ValueError("x must be [B,D]")
    w = _taps(weight, x.shape[1])
    b = _number("bias", bias, x.shape[1:], x)
    _same_type(x, state=state)
    if state.shape != (x.shape[0], w.shape[1] - 1, x.shape[1]) or not state.is_contiguous():
        raise ValueError(f"state must be a contiguous tensor {[x.shape[0], w.shape[1] - 1, x.shape[1]]} (it is updated in place)")
    call = torch.ops.vig_amd.causal_conv1d_step if ops.observed() else _conv_step_launch
    return call(x, w, state, b, bool(silu))


def _conv_step_launch(x, w, state, b, silu):
    lib = _lib.load()
    ops._check_cuda(x, w, state, b)
    batch, width = x.shape
    y = torch.empty(batch, width, dtype=x.dtype, device=x.device)
    if x.numel() == 0:
        return y
    x, w, b = _scan_rows(x), w.contiguous(), b.contiguous() if b is not None else None
    with torch.cuda.device(x.device):
        rc = lib.vig_causal_conv1d_step(_ptr(x), _ptr(w), _ptr(b), _ptr(state), _ptr(y), batch, width, w.shape[1], x.stride(0) if batch > 1 else width, int(silu), _dt(x),
                                        ops._stream_ptr(x))
    _lib.check(rc, "vig_causal_conv1d_step")
    _written(state)
    return y


# ---------------------------------------------------------------------------
# residual add and layer norm
# ---------------------------------------------------------------------------

def add_layernorm(x: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor] = None, eps: float = 1e-5, residual: Optional[torch.Tensor] = None, prenorm: bool = False):
    """Residual add and layer norm over the last dimension: y, or (y, x + residual) with prenorm=True (without a residual: (y, x)).

    As rmsnorm(), with a mean and a bias, and a gradient for each.  x [..., C] in fp32 or bf16, C up to 16384; residual of its dtype or in fp32 (a residual stream in fp32 beside bf16
    branches), which is the dtype of the sum.  The sum as it is stored is what is normalised.  weight, bias [C].  Up to 2^24 rows.  Differentiable in every tensor, the weight's and
    the bias's gradient added up in an order fixed by the sizes and by how the rows lie; x's and the residual's are alike, each in memory of its own."""
    calls = _ext.calls()
    if calls is not None:
        r = calls.add_layernorm(x, weight, bias, residual, eps)
        if r is not None:
            y, total = (r, x) if residual is None else r
            return (y, total) if prenorm else y
    ops._check_cuda(x, weight, bias, residual)
    given = (x, weight, bias, residual)
    _refuse_tangents("add_layernorm", *given)
    _refuse_held_leaves(*given, by="add_layernorm")
    if x.dim() < 1 or not 1 <= x.shape[-1] <= MOST_WIDTH:
        raise ValueError(f"x must be [..., C] with C from 1 to {MOST_WIDTH}")
    if not eps >= 0:
        raise ValueError(f"eps must not be negative; got {eps}")
    _dt(x)
    if residual is not None and (residual.shape != x.shape or residual.dtype not in (x.dtype, torch.float32)):
        raise ValueError("residual must match x in shape, and in dtype or be float32")
    C = x.shape[-1]
    w, b = _number("weight", weight, (C,), x), _number("bias", bias, (C,), x)
    if x.numel() == 0:
        total = x + residual if residual is not None else x
        y = (total * w + (b if b is not None else 0)).to(x.dtype)
    elif _needs_graph(x, w, b, residual):
        if residual is None:
            y, total = _AddLayerNorm.apply(x, w, b, None, float(eps)), x
        else:
            y, total = _AddLayerNorm.apply(x, w, b, residual, float(eps))
    else:
        y, total, _ = _norm_forward(x, w, b, residual, float(eps), False)
        total = total if residual is not None else x
    return (y, total) if prenorm else y


def _norm_forward(x, w, b, residual, eps, keep):
    """(y, the sum as held, statistics of the rows or None)"""
    if ops.observed():
        y, total, stats = torch.ops.vig_amd.add_layernorm_fwd(x, w, b, residual, eps)
        return y, total if residual is not None else x, stats
    return _norm_launch(x, w, b, residual, eps, keep)


def _norm_launch(x, w, b, residual, eps, keep):
    lib = _lib.load()
    ops._check_cuda(x, w, b, residual)
    x, w = x.contiguous(), w.contiguous()
    b, residual = (t.contiguous() if t is not None else None for t in (b, residual))
    C = x.shape[-1]
    rows = x.numel() // C
    y = torch.empty_like(x)
    total = torch.empty_like(residual) if residual is not None else None
    stats = torch.empty(rows, 2, dtype=torch.float32, device=x.device) if keep else None
    with torch.cuda.device(x.device):
        rc = lib.vig_add_layernorm_fwd(_ptr(x), _ptr(residual), _ptr(w), _ptr(b), _ptr(total), _ptr(y), _ptr(stats), rows, C, eps, _dt(x), _dt(residual) if residual is not None else _dt(x),
                                       ops._stream_ptr(x))
    _lib.check(rc, "vig_add_layernorm_fwd")
    return y, total if total is not None else x, stats


class _AddLayerNorm(torch.autograd.Function):
    """Autograd node of the residual add and layer norm; with a residual it returns (y, x + residual)."""

    @staticmethod
    def forward(ctx, x, w, b, residual, eps):
        y, total, stats = _norm_forward(x, w, b, residual, eps, True)
        ctx.save_for_backward(total, stats, w)
        ctx.set_materialize_grads(False)
        ctx.kinds = x.dtype, b is not None, residual is not None
        return (y, total) if residual is not None else y

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy, d_total=None):
        total, stats, w = ctx.saved_tensors
        dtype, has_bias, has_residual = ctx.kinds
        dy = dy if dy is not None else torch.zeros(total.shape, dtype=dtype, device=total.device)
        params = ctx.needs_input_grad[1] or ctx.needs_input_grad[2]
        # (two who want the gradient of one sum get a buffer each: behind views of leaves autograd keeps both as they are, and adds the next pass's to one memory twice)
        both = has_residual and ctx.needs_input_grad[0] and ctx.needs_input_grad[3]
        call = torch.ops.vig_amd.add_layernorm_bwd if ops.observed() else _norm_backward
        dx, d_residual, dparams = call(total, stats, w, dy, d_total, params, both)
        C = w.numel()
        if has_residual and dtype == total.dtype and not both:
            dx, d_residual = (dx, None) if ctx.needs_input_grad[0] else (None, dx)
        return dx, dparams[:C] if params else None, dparams[C:] if params and has_bias else None, d_residual if has_residual else None, None


def _norm_backward(total, stats, w, dy, d_total, want_params, both=False):
    """(dx, the residual's gradient where its type is another or both are wanted, weight's and bias's gradient behind one another)"""
    lib = _lib.load()
    ops._check_cuda(total, stats, w, dy, d_total)
    total, dy = total.contiguous(), dy.contiguous()
    w, d_total = w.contiguous(), d_total.contiguous() if d_total is not None else None
    C = total.shape[-1]
    rows = total.numel() // C
    dx = torch.empty(total.shape, dtype=dy.dtype, device=total.device)
    d_residual = torch.empty_like(total) if both or total.dtype != dy.dtype else None
    dparams = torch.empty(2 * C, dtype=torch.float32, device=total.device) if want_params else None
    need = lib.vig_add_layernorm_bwd_workspace(rows, C) if want_params else 0
    ws = torch.empty(need, dtype=torch.uint8, device=total.device) if need else None
    with torch.cuda.device(total.device):
        rc = lib.vig_add_layernorm_bwd(_ptr(total), _ptr(stats), _ptr(w), _ptr(dy), _ptr(d_total), _ptr(d_residual), _ptr(dx), _ptr(dparams), _ptr(ws), need, rows, C, _dt(dy), _dt(total),
                                       ops._stream_ptr(total))
    _lib.check(rc, "vig_add_layernorm_bwd")
    return dx, d_residual, dparams


# ---------------------------------------------------------------------------
# the same as operators, for whoever records them; what a call leaves out is empty here
# ---------------------------------------------------------------------------

def _or_empty(like, *ts):
    return tuple(t if t is not None else like.new_empty(0, dtype=torch.float32) for t in ts)


def _packed(t):
    return t.new_empty(t.shape)


def _numbers(like, *shape):
    return like.new_empty(shape, dtype=torch.float32)


def _kept_like(x, N):
    CN = 1
    while 4 * CN < N:
        CN *= 2
    T = 16 if CN <= 4 else 64 // CN
    return x.new_empty(x.shape[0] * -(-x.shape[1] // T) * x.shape[2] * 16 * CN, dtype=torch.uint8)


def _scan_shapes(x, delta, A, B, C, D, z, bias, h0, softplus, reverse, keep):
    return _packed(x), _numbers(x, x.shape[0], *A.shape), _kept_like(x, A.shape[1]) if keep else _numbers(x, 0)


@_operator("selective_scan_fwd(Tensor x, Tensor delta, Tensor A, Tensor B, Tensor C, Tensor? D, Tensor? z, Tensor? delta_bias, Tensor? initial_state, bool softplus, bool reverse, "
           "bool keep) -> (Tensor, Tensor, Tensor)", _scan_shapes)
def _scan_operator(x, delta, A, B, C, D, z, bias, h0, softplus, reverse, keep):
    o, h, kept = _scan_launch(x, delta, A, B, C, D, z, bias, h0, softplus, reverse, True, keep)
    return o, h, *_or_empty(x, kept)


def _scan_bwd_shapes(x, delta, A, B, C, D, z, bias, kept, d_o, d_final, softplus, reverse, state):
    return (_packed(x), _packed(delta), _packed(B), _packed(C), _packed(z) if z is not None else _numbers(x, 0), _numbers(x, A.numel() + 2 * A.shape[0]),
            _numbers(x, x.shape[0], *A.shape) if state else _numbers(x, 0))


@_operator("selective_scan_bwd(Tensor x, Tensor delta, Tensor A, Tensor B, Tensor C, Tensor? D, Tensor? z, Tensor? delta_bias, Tensor kept, Tensor d_o, Tensor? d_final, bool softplus, "
           "bool reverse, bool state) -> (Tensor, Tensor, Tensor, Tensor, Tensor, Tensor, Tensor)", _scan_bwd_shapes)
def _scan_bwd_operator(x, *rest):
    return _or_empty(x, *_scan_backward(x, *rest))


@_operator("selective_scan_step(Tensor x, Tensor delta, Tensor A, Tensor B, Tensor C, Tensor(a!) state, Tensor? D, Tensor? z, Tensor? delta_bias, bool softplus) -> Tensor",
           lambda x, *rest: _packed(x))
def _step_operator(*given):
    return _step_launch(*given)


@_operator("causal_conv1d_fwd(Tensor x, Tensor weight, Tensor? bias, Tensor? initial_state, bool silu, bool reverse) -> (Tensor, Tensor)",
           lambda x, w, b, h0, silu, reverse: (_packed(x), x.new_empty(x.shape[0], w.shape[1] - 1, x.shape[2])))
def _conv_operator(x, w, b, h0, silu, reverse):
    return _conv_launch(x, w, b, h0, silu, reverse, True)


@_operator("causal_conv1d_bwd(Tensor x, Tensor weight, Tensor? bias, Tensor? initial_state, Tensor dy, Tensor? d_final, bool silu, bool reverse, bool state, bool params) -> "
           "(Tensor, Tensor, Tensor)",
           lambda x, w, b, h0, dy, d_final, silu, reverse, state, params: (_packed(x), _numbers(x, w.numel() + w.shape[0] if params else 0),
                                                                          x.new_empty(x.shape[0], w.shape[1] - 1, x.shape[2]) if state else _numbers(x, 0)))
def _conv_bwd_operator(x, *rest):
    return _or_empty(x, *_conv_backward(x, *rest))


@_operator("causal_conv1d_step(Tensor x, Tensor weight, Tensor(a!) state, Tensor? bias, bool silu) -> Tensor", lambda x, *rest: _packed(x))
def _conv_step_operator(*given):
    return _conv_step_launch(*given)


@_operator("add_layernorm_fwd(Tensor x, Tensor weight, Tensor? bias, Tensor? residual, float eps) -> (Tensor, Tensor, Tensor)",
           lambda x, w, b, residual, eps: (_packed(x), _packed(residual) if residual is not None else _numbers(x, 0), _numbers(x, x.numel() // x.shape[-1], 2)))
def _norm_operator(x, w, b, residual, eps):
    y, total, stats = _norm_launch(x, w, b, residual, eps, True)
    return y, total if residual is not None else _or_empty(x, None)[0], stats


@_operator("add_layernorm_bwd(Tensor sum, Tensor stats, Tensor weight, Tensor dy, Tensor? d_sum, bool params, bool both=False) -> (Tensor, Tensor, Tensor)",
           lambda total, stats, w, dy, d_total, params, both=False: (_packed(dy), _packed(total) if both or total.dtype != dy.dtype else _numbers(total, 0),
                                                                     _numbers(total, 2 * w.numel() if params else 0)))
def _norm_bwd_operator(total, stats, w, dy, d_total, params, both=False):
    return _or_empty(total, *_norm_backward(total, stats, w, dy, d_total, params, both))
