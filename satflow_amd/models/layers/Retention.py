"""Retention layers: a temporal encoder with a carried state, next to the recurrent cells (``ConvGRU``, ``ConvLSTM``) and the attention layers.

Trained over whole sequences at once like attention, run frame by frame with a state of fixed size like a recurrent cell.  A layer, on tokens ``x [B, T, dim]``:

    h = norm(x)
    q, k, v, g = split(W_in h)
    S_t = exp(log_decay) S_{t-1} + k_t v_t^T ,   o_t = dk^-1/2 S_t^T q_t           for each head
    x = x + scale * norm(W_out (silu(g) * norm_heads(o)))

Execution: the recurrence is ``functional_seq.linear_attention`` (``linear_attention_step`` for a single frame), the norms with their gate, scale, residual and
the next layer's norm are ``functional_seq.post_norm`` - one pass over the tokens at the boundary of two layers -, the projections are ``sf_linear_*``.
"""
from __future__ import annotations

from typing import List, Optional, Tuple, Union

import torch
import torch.nn as nn
from torch import Tensor

from ... import functional as F
from ... import functional_seq as FS
from ..._hip import SF_CPAD


class RetentionLayer(nn.Module):
    """One layer: its parameters, and the two halves between which the recurrence runs.  :class:`Retention` chains them."""

    def __init__(self, dim: int, heads: int = 4, key_dim: Optional[int] = None, value_dim: Optional[int] = None, layer_scale: float = 1.0, eps: float = 1e-6):
        super().__init__()
        if heads < 1:
            raise ValueError(f"a retention layer of {heads} heads")
        key_dim = dim // heads if key_dim is None else key_dim
        value_dim = dim // heads if value_dim is None else value_dim
        if dim < 1 or dim % SF_CPAD or (heads * value_dim) % SF_CPAD:
            raise ValueError(f"a retention layer takes a width and heads * value_dim that are multiples of {SF_CPAD}: got {dim} and {heads} * {value_dim}")
        if not (1 <= key_dim <= 128 and 1 <= value_dim <= 128):
            raise ValueError(f"a retention layer takes head widths of 1 to 128: got {key_dim} and {value_dim}")
        self.dim, self.heads, self.key_dim, self.value_dim, self.eps = dim, heads, key_dim, value_dim, eps
        self.norm_in = nn.Parameter(torch.ones(dim))
        self.to_qkvg = nn.Linear(dim, 2 * heads * (key_dim + value_dim), bias=False)
        self.norm_heads = nn.Parameter(torch.ones(heads * value_dim))
        self.to_out = nn.Linear(heads * value_dim, dim, bias=False)
        self.norm_out = nn.Parameter(torch.ones(dim))
        self.scale = nn.Parameter(torch.full((dim,), float(layer_scale)))
        # horizons from 4 frames to 4096, evenly spread over the heads on a logarithmic scale
        spread = torch.arange(heads, dtype=torch.float64) * (10.0 / max(1, heads - 1))
        self.register_buffer("log_decay", torch.log1p(-torch.exp2(-2.0 - spread)).float())

    def _heads_of(self, h: Tensor) -> Tuple[Tensor, Tensor, Tensor, Tensor]:
        n, d, e = self.heads, self.key_dim, self.value_dim
        p = F.linear(h, self.to_qkvg.weight, None, lowp=True)
        q, k, v, g, _ = p.split((n * d, n * d, n * e, n * e, p.shape[-1] - 2 * n * (d + e)), -1)   # (views: read in place)
        return q.unflatten(-1, (n, d)), k.unflatten(-1, (n, d)), v.unflatten(-1, (n, e)), g

    def _leave(self, o: Tensor, g: Tensor, x: Tensor, following: Optional["RetentionLayer"]) -> Tuple[Tensor, Optional[Tensor]]:
        a = FS.post_norm(o.flatten(-2), self.norm_heads, gate=g, groups=self.heads, eps=self.eps)
        u = F.linear(a, self.to_out.weight, None, lowp=True)
        if following is None:
            return FS.post_norm(u, self.norm_out, scale=self.scale, residual=x, eps=self.eps), None
        return FS.post_norm(u, self.norm_out, scale=self.scale, residual=x, next_weight=following.norm_in, eps=self.eps)

    def run(self, x: Tensor, h: Tensor, state: Optional[Tensor], lengths: Optional[Tensor], following: Optional["RetentionLayer"], want_state: bool):
        """``x [B, T, dim]`` and its norm ``h`` -> the layer's output, its norm for the layer that follows, the state behind the last token."""
        q, k, v, g = self._heads_of(h)
        o = FS.linear_attention(q, k, v, self.log_decay, initial_state=state, lengths=lengths, return_state=want_state)
        o, state = o if want_state else (o, None)
        return (*self._leave(o, g, x, following), state)

    def run_step(self, x: Tensor, h: Tensor, state: Tensor, following: Optional["RetentionLayer"]):
        """The same for one token, ``x [B, dim]``; the state is updated in place."""
        q, k, v, g = self._heads_of(h)
        o, _ = FS.linear_attention_step(q, k, v, self.log_decay, state, out_state=state)
        return self._leave(o, g, x, following)


class Retention(nn.Module):
    """A stack of retention layers over float32 tokens ``[B, T, dim]`` or frames ``[B, T, dim, H, W]`` (each pixel a sequence over time)."""

    def __init__(self, dim: int, num_layers: int = 1, heads: int = 4, key_dim: Optional[int] = None, value_dim: Optional[int] = None, layer_scale: float = 1.0,
                 eps: float = 1e-6):
        super().__init__()
        if num_layers < 1:
            raise ValueError(f"a retention stack of {num_layers} layers")
        self.dim = dim
        self.layers = nn.ModuleList(RetentionLayer(dim, heads, key_dim, value_dim, layer_scale, eps) for _ in range(num_layers))

    def _check(self, x: Tensor, dims: Tuple[int, ...], channels: int) -> None:
        if x.dim() not in dims or x.shape[channels] != self.dim or x.dtype != torch.float32:
            raise RuntimeError(f"satflow_amd: Retention({self.dim}) got {tuple(x.shape)} {x.dtype}")

    def initial_state(self, batch: int, device=None) -> List[Tensor]:
        """Zero states for :meth:`step`, one ``[batch, heads, key_dim, value_dim]`` for each layer (``batch``: sequences, or sequences times pixels)."""
        return [torch.zeros(batch, m.heads, m.key_dim, m.value_dim, device=device or m.norm_in.device) for m in self.layers]

    def forward(self, x: Tensor, state: Optional[List[Tensor]] = None, lengths: Optional[Tensor] = None,
                return_state: bool = False) -> Union[Tensor, Tuple[Tensor, List[Tensor]]]:
        """``state``: what an earlier call returned or :meth:`initial_state`; ``lengths [B]`` int32: the tokens of each sequence, the outputs behind them are
        those of a layer that saw nothing (they are not to be used; what stands behind has to be finite, norms and projections read it).  Frames take one length for
        all pixels of a sequence."""
        if x.dim() == 5:
            self._check(x, (5,), 2)
            B, T, C, H, W = x.shape
            tokens = x.permute(0, 3, 4, 1, 2).reshape(B * H * W, T, C)
            y = self.forward(tokens, state, lengths.repeat_interleave(H * W) if lengths is not None else None, return_state)
            y, last = y if return_state else (y, None)
            y = y.view(B, H, W, T, C).permute(0, 3, 4, 1, 2).contiguous()
            return (y, last) if return_state else y
        self._check(x, (3,), 2)
        if state is not None and len(state) != len(self.layers):
            raise RuntimeError(f"satflow_amd: {len(state)} states for {len(self.layers)} retention layers")
        h = FS.pre_norm(x, self.layers[0].norm_in, eps=self.layers[0].eps)
        last = []
        for i, m in enumerate(self.layers):
            x, h, s = m.run(x, h, state[i] if state is not None else None, lengths, self.layers[i + 1] if i + 1 < len(self.layers) else None, return_state)
            last.append(s)
        return (x, last) if return_state else x

    @torch.no_grad()
    def step(self, x: Tensor, state: List[Tensor]) -> Tensor:
        """One frame: tokens ``[B, dim]`` or a map ``[B, dim, H, W]``; the states are updated in place.  Inference only."""
        if x.dim() == 4:
            self._check(x, (4,), 1)
            B, C, H, W = x.shape
            y = self.step(x.permute(0, 2, 3, 1).reshape(B * H * W, C), state)
            return y.view(B, H, W, C).permute(0, 3, 1, 2).contiguous()
        self._check(x, (2,), 1)
        if len(state) != len(self.layers):
            raise RuntimeError(f"satflow_amd: {len(state)} states for {len(self.layers)} retention layers")
        h = FS.pre_norm(x, self.layers[0].norm_in, eps=self.layers[0].eps)
        for i, m in enumerate(self.layers):
            x, h = m.run_step(x, h, state[i], self.layers[i + 1] if i + 1 < len(self.layers) else None)
        return x
