"""Autograd functions of the sequence blocks: linear attention with a decay for each head (parallel over a whole sequence in training, one token at a time
with a carried state at inference) and the norms before and after a block, fused with its gate, residual scale and residual sum.

Token tensors are float32 or bfloat16, parameters and states float32, all on one HIP device.  Arithmetic follows the storage type, not the compute mode of the
convolutions (``set_compute_dtype``): sums, states, statistics and decays are held in float32, outputs are rounded once.  Products of float32 tensors are float32-accurate.
Of bfloat16 tensors the inner operands of linear attention - scores and states where they are multiplied, the values' share of a state that does not leave the call - are
taken with 16 bits (2^-17 of the operand, below the 2^-9 of the output's rounding); states that leave are float32-accurate.  exp and the gate's sigmoid are the hardware's.

Derivatives are backward ones of the first order; forward-mode (dual) tensors are refused.

Everything can be captured into a HIP graph.  A captured backward pass must not meet leaves that an eager graph still holds (their gradient accumulation belongs to
the eager stream, as for any torch function): capture on leaves of its own, or after the eager graph is gone.
"""
from __future__ import annotations

from typing import Optional, Tuple, Union

import torch
from torch import Tensor
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable

from . import _hip
from . import kernels as K
from ._hip import require_device

_TOKEN_TYPES = (torch.float32, torch.bfloat16)


def _fail(what: str) -> None:
    raise RuntimeError(f"satflow_amd: {what}")


def _same_device(first: Tensor, name: str, others, names) -> None:
    index = first.get_device()
    if index < 0:
        require_device(first, name)
    for t, n in zip(others, names):
        if t is not None and t.get_device() != index:
            _fail(f"`{n}` lives on {t.device}, `{name}` on {first.device}")


class _NoGuard:
    def __enter__(self):
        return self

    def __exit__(self, *exc):
        return False


_HERE = _NoGuard()


def _on(t: Tensor):
    """A context in which t's device is the current one (its current stream is what a launch goes to)."""
    return _HERE if t.get_device() == _hip.current_device() else torch.cuda.device(t.device)


def _wants_grad(*tensors: Optional[Tensor]) -> bool:
    if torch.is_grad_enabled():
        for t in tensors:
            if t is not None and t.requires_grad:
                return True
    return False


def _no_tangent(what: str, *tensors: Optional[Tensor]) -> None:
    """Forward-mode differentiation is refused, as the other operators' autograd functions refuse it: a dual tensor does not say ``requires_grad``, and its tangent
    would be lost on a call that goes straight to the kernels."""
    if forward_ad._current_level >= 0:
        for t in tensors:
            if t is not None and forward_ad.unpack_dual(t).tangent is not None:
                raise NotImplementedError(f"satflow_amd: {what} has no forward-mode derivative")


def _channels_contiguous(t: Tensor) -> Tensor:
    """The tensor itself, or a dense copy where its channels are not contiguous (a broadcast gradient, a transposed view)."""
    return t if t.shape[-1] <= 1 or t.stride(-1) == 1 else t.contiguous()


# ----------------------------------------------------------------------------------------------
# linear attention
# ----------------------------------------------------------------------------------------------
class _LinearAttentionFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q: Tensor, k: Tensor, v: Tensor, log_decay: Tensor, state: Optional[Tensor], lengths: Optional[Tensor], scale: float, want_state: bool):
        ctx.set_materialize_grads(False)
        with _on(q):
            o, last, states = K.linear_attention_fwd(q, k, v, log_decay, state, lengths, scale, want_state)
        ctx.save_for_backward(q, k, v, log_decay, state, lengths, states)
        ctx.scale = scale
        return o, last

    @staticmethod
    @once_differentiable
    def backward(ctx, do: Optional[Tensor], dlast: Optional[Tensor]):
        q, k, v, log_decay, state, lengths, states = ctx.saved_tensors
        if do is None and dlast is None:
            return (None,) * 8
        do = torch.zeros_like(v) if do is None else _channels_contiguous(do)
        dlast = dlast.contiguous() if dlast is not None else None
        need = ctx.needs_input_grad
        with _on(q):
            dq, dk, dv, ds = K.linear_attention_bwd(q, k, v, log_decay, state, lengths, states, ctx.scale, do, dlast, need[4])
        return dq if need[0] else None, dk if need[1] else None, dv if need[2] else None, None, ds, None, None, None


def _check_attention(q: Tensor, k: Tensor, v: Tensor, log_decay: Tensor, dims: int) -> None:
    if q.dim() != dims or k.dim() != dims or v.dim() != dims or k.shape != q.shape or v.shape[:-1] != q.shape[:-1]:
        _fail(f"linear attention takes q, k {'[B, T, H, dk]' if dims == 4 else '[B, H, dk]'} and v of the same leading sizes: got {tuple(q.shape)}, {tuple(k.shape)}, "
              f"{tuple(v.shape)}")
    if q.dtype not in _TOKEN_TYPES or k.dtype != q.dtype or v.dtype != q.dtype:
        _fail(f"linear attention takes q, k, v of one type, float32 or bfloat16: got {q.dtype}, {k.dtype}, {v.dtype}")
    H, dk = q.shape[-2:]
    if not (1 <= dk <= 128 and 1 <= v.shape[-1] <= 128) or H < 1:
        _fail(f"linear attention takes head widths of 1 to 128: got {dk} and {v.shape[-1]} ({H} heads)")
    if q.shape[0] * H > 1 << 22:
        _fail(f"linear attention takes at most 2^22 sequences times heads: got {q.shape[0]} * {H}")
    if log_decay.shape != (H,) or log_decay.dtype != torch.float32:
        _fail(f"log_decay is a float32 tensor of {H} values, one for each head: got {tuple(log_decay.shape)} {log_decay.dtype}")
    if log_decay.requires_grad:
        _fail("log_decay is a constant of the layer: it has no gradient")


def _check_state(state: Tensor, q: Tensor, v: Tensor, name: str) -> None:
    want = (q.shape[0], q.shape[-2], q.shape[-1], v.shape[-1])
    if state.shape != want or state.dtype != torch.float32:
        _fail(f"`{name}` is a float32 tensor of shape {want}: got {tuple(state.shape)} {state.dtype}")


def linear_attention(q: Tensor, k: Tensor, v: Tensor, log_decay: Tensor, scale: Optional[float] = None, initial_state: Optional[Tensor] = None,
                     lengths: Optional[Tensor] = None, return_state: bool = False) -> Union[Tensor, Tuple[Tensor, Tensor]]:
    """``S_t = exp(log_decay[h]) S_{t-1} + k_t v_t^T``, ``o_t = scale * S_t^T q_t`` over ``q, k [B, T, H, dk]`` and ``v [B, T, H, dv]``.

    ``log_decay [H]``: float32, at most 0 (``-inf``: a head that keeps nothing); not differentiable.  ``scale``: ``dk ** -0.5`` by default.
    ``initial_state [B, H, dk, dv]``: float32, the state in front of the first token (zeros by default).  ``lengths [B]``: int32 tensor on the device, the
    tokens of each sequence (clipped to 0 .. T): what lies behind is not read, its outputs and gradients are zero.
    Returns ``o [B, T, H, dv]``, with ``return_state`` also the state behind the last token of each sequence (``[B, H, dk, dv]``, float32), from which
    :func:`linear_attention_step` or another call goes on.  Differentiable (once) in q, k, v and initial_state; any strides with contiguous channels are
    read in place.  At most 2^22 sequences times heads.  A value that is not finite reaches the outputs of its own and later tokens (as NaN), never earlier
    ones; a repeated call gives the same bits.  The fast kernels move 16 bytes at a time: widths that are multiples of 8 (both), aligned pointers and strides; other tensors
    take one kernel of all widths, up to nine times slower."""
    _check_attention(q, k, v, log_decay, 4)
    _no_tangent("linear_attention", q, k, v, log_decay, initial_state)
    if initial_state is not None:
        _check_state(initial_state, q, v, "initial_state")
        initial_state = initial_state.contiguous()
    if lengths is not None and (lengths.shape != (q.shape[0],) or lengths.dtype != torch.int32):
        _fail(f"`lengths` is an int32 tensor of {q.shape[0]} values: got {tuple(lengths.shape)} {lengths.dtype}")
    _same_device(q, "q", (k, v, log_decay, initial_state, lengths), ("k", "v", "log_decay", "initial_state", "lengths"))
    args = (_channels_contiguous(q), _channels_contiguous(k), _channels_contiguous(v), log_decay.contiguous(), initial_state,
            lengths.contiguous() if lengths is not None else None, float(q.shape[-1] ** -0.5 if scale is None else scale), return_state)
    if _wants_grad(q, k, v, initial_state):
        o, last = _LinearAttentionFn.apply(*args)
    else:
        with _on(q):
            o, last, _ = K.linear_attention_fwd(*args)
    return (o, last) if return_state else o


def linear_attention_step(q: Tensor, k: Tensor, v: Tensor, log_decay: Tensor, state: Tensor, scale: Optional[float] = None,
                          out_state: Optional[Tensor] = None) -> Tuple[Tensor, Tensor]:
    """One token of every sequence: ``q, k [B, H, dk]``, ``v [B, H, dv]``, ``state [B, H, dk, dv]`` (float32) -> ``(o [B, H, dv], new state)``.

    The new state goes to ``out_state`` (contiguous; ``out_state=state`` updates in place; a new tensor by default).  Inference only: no gradient."""
    _check_attention(q, k, v, log_decay, 3)
    _no_tangent("linear_attention_step", q, k, v, log_decay, state, out_state)
    _check_state(state, q, v, "state")
    if _wants_grad(q, k, v, state):
        _fail("linear_attention_step has no gradient: call it under torch.no_grad(), or linear_attention with one token")
    given = out_state is not None
    if not given:
        out_state = torch.empty_like(state, memory_format=torch.contiguous_format)
    else:
        _check_state(out_state, q, v, "out_state")
        if not out_state.is_contiguous() or (out_state is not state and _overlap(out_state, state)):
            _fail("`out_state` is contiguous, and `state` itself or memory of its own")
        if out_state.requires_grad:
            _fail("`out_state` is written in place: it cannot require a gradient")
    _same_device(q, "q", (k, v, log_decay, state, out_state), ("k", "v", "log_decay", "state", "out_state"))
    if given and not out_state.is_inference():
        torch.autograd.graph.increment_version(out_state)   # (a graph that saved it notices)
    with _on(q):
        o = K.linear_attention_step(_channels_contiguous(q), _channels_contiguous(k), _channels_contiguous(v), log_decay.contiguous(), state.contiguous(), out_state,
                                    float(q.shape[-1] ** -0.5 if scale is None else scale))
    return o, out_state


def _overlap(out: Tensor, state: Tensor) -> bool:
    """Whether a contiguous tensor shares memory with another one of its shape without being the same elements in the same order."""
    lo, at = out.data_ptr(), state.data_ptr()
    if state.is_contiguous():
        return at != lo and abs(at - lo) < 4 * out.numel()
    end = at + 4 * (1 + sum((n - 1) * st for n, st in zip(state.shape, state.stride())))
    return out.numel() > 0 and max(lo, at) < min(lo + 4 * out.numel(), end)


# ----------------------------------------------------------------------------------------------
# norms before and after a block
# ----------------------------------------------------------------------------------------------
class _BlockNormFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, u, w, b, gate, scale, residual, next_w, next_b, groups: int, kind: int, eps: float):
        ctx.set_materialize_grads(False)
        train = any(ctx.needs_input_grad)
        with _on(u):
            r, y, stats = K.block_norm_fwd(u, w, b, gate, scale, residual, next_w, next_b, groups, kind, eps, train)
        if train:
            ctx.save_for_backward(u, w, b, gate, scale, residual, next_w, stats)
        ctx.meta = (groups, kind)
        return r, y

    @staticmethod
    @once_differentiable
    def backward(ctx, dr: Optional[Tensor], dy: Optional[Tensor]):
        u, w, b, gate, scale, residual, next_w, stats = ctx.saved_tensors
        need = ctx.needs_input_grad[:8]
        if dr is None and dy is None:
            return (None,) * 11
        if u.shape[0] == 0:
            return tuple(torch.zeros_like(t) if n else None for t, n in zip((u, w, b, gate, scale, residual, next_w, next_w), need)) + (None,) * 3
        dr, dy = (_row_major(t) if t is not None else None for t in (dr, dy))
        with _on(u):
            return K.block_norm_bwd(u, w, b, gate, scale, residual, next_w, stats, dr, dy, *ctx.meta, need) + (None,) * 3


def _row_major(t: Tensor) -> Tensor:
    """A ``[rows, C]`` matrix whose channels are contiguous and whose rows do not overlap: the tensor itself, or a dense copy."""
    if (t.shape[1] <= 1 or t.stride(1) == 1) and (t.shape[0] <= 1 or t.stride(0) >= t.shape[1]):
        return t
    return t.contiguous()


def _rows_of(t: Optional[Tensor], C: int) -> Optional[Tensor]:
    return None if t is None else _row_major(t if t.dim() == 2 else t.reshape(-1, C))


def _param(p: Optional[Tensor], C: int, name: str) -> Optional[Tensor]:
    if p is None:
        return None
    if p.dtype != torch.float32 or p.dim() != 1 or p.shape[0] != C:
        _fail(f"`{name}` is a float32 tensor of {C} values: got {tuple(p.shape)} {p.dtype}")
    return p if p.is_contiguous() else p.contiguous()


_KINDS = {"rms": _hip.SF_NORM_RMS, "layer": _hip.SF_NORM_LAYER}


def _kind(kind: str) -> int:
    if kind not in _KINDS:
        _fail(f"norm kind {kind!r}: 'rms' or 'layer'")
    return _KINDS[kind]


def pre_norm(x: Tensor, weight: Optional[Tensor], bias: Optional[Tensor] = None, kind: str = "rms", eps: float = 1e-6) -> Tensor:
    """The norm before a block over the last axis of ``x [..., C]``: ``x / sqrt(mean(x^2) + eps) * weight + bias`` (``kind="rms"``) or
    ``(x - mean) / sqrt(var + eps) * weight + bias`` (``"layer"``).  Statistics in float32; the output has x's type.  Differentiable (once)."""
    return post_norm(x, weight, bias, None, None, None, 1, None, None, kind, eps)


def post_norm(u: Tensor, weight: Optional[Tensor], bias: Optional[Tensor] = None, gate: Optional[Tensor] = None, scale: Optional[Tensor] = None,
              residual: Optional[Tensor] = None, groups: int = 1, next_weight: Optional[Tensor] = None, next_bias: Optional[Tensor] = None, kind: str = "rms",
              eps: float = 1e-6) -> Union[Tensor, Tuple[Tensor, Tensor]]:
    """The norm after a block, its gate, residual scale and residual sum, and the norm before the next block, in one pass over the tokens:

        r = residual + scale * silu(gate) * (norm(u) * weight + bias)        and with ``next_weight``:   y = norm(r) * next_weight + next_bias

    ``u, gate, residual [..., C]``; ``weight, bias, scale, next_weight, next_bias [C]`` float32; whatever is None is left out.  ``groups``: the norm of u
    is taken over each of that many groups of channels (heads); the next norm over all (one group only).  ``u`` and ``gate`` are float32 or bfloat16, the
    residual has their type or is float32; r has the residual's type (u's without one), y has u's, and y is the norm of r before r is rounded.
    Returns ``r``, or ``(r, y)``.  Differentiable (once) in every tensor; parameter gradients are summed in a fixed order."""
    if u.dim() < 1 or u.shape[-1] < 1:
        _fail(f"a norm takes tokens of at least one channel: got {tuple(u.shape)}")
    C = u.shape[-1]
    if groups < 1 or C % groups or C // groups > 16384 or groups > 65535:
        _fail(f"{C} channels in {groups} groups: equal groups of at most 16384 channels")
    if u.dtype not in _TOKEN_TYPES or (gate is not None and gate.dtype != u.dtype):
        _fail(f"a norm takes u and gate of one type, float32 or bfloat16: got {u.dtype}" + (f", {gate.dtype}" if gate is not None else ""))
    if residual is not None and residual.dtype not in (u.dtype, torch.float32):
        _fail(f"the residual has the type of u ({u.dtype}) or float32: got {residual.dtype}")
    if next_weight is None and next_bias is not None:
        _fail("next_bias without next_weight")
    if next_weight is not None and groups != 1:
        _fail("the next norm is taken over all channels: it goes with groups=1")
    if not eps >= 0:
        _fail(f"eps {eps}")
    code = _kind(kind)
    _no_tangent("a norm", u, weight, bias, gate, scale, residual, next_weight, next_bias)
    params = (_param(weight, C, "weight"), _param(bias, C, "bias"), _param(scale, C, "scale"), _param(next_weight, C, "next_weight"), _param(next_bias, C, "next_bias"))
    for t, n in ((gate, "gate"), (residual, "residual")):
        if t is not None and t.shape != u.shape:
            _fail(f"`{n}` has the shape of the block's output, {tuple(u.shape)}: got {tuple(t.shape)}")
    _same_device(u, "u", (gate, residual, *params), ("gate", "residual", "weight", "bias", "scale", "next_weight", "next_bias"))
    args = (_rows_of(u, C), params[0], params[1], _rows_of(gate, C), params[2], _rows_of(residual, C), params[3], params[4], groups, code, float(eps))
    if _wants_grad(u, weight, bias, gate, scale, residual, next_weight, next_bias):
        r, y = _BlockNormFn.apply(*args)
    else:
        with _on(u):
            r, y, _ = K.block_norm_fwd(*args, False)
    if u.dim() != 2:
        r, y = r.view(u.shape), y.view(u.shape) if y is not None else None
    return r if next_weight is None else (r, y)
