"""Residual stack of PoM layers with a GELU feed-forward block, run frame by frame with the layers'
running-mean state — the block-causal video pattern of the reference's README (README.md:28-35, 48-61):

    for each frame:  for each layer:  x = x + pom.state_forward(x, x, state[l]);  x = x + W2·gelu(W1·x)

The frame loop is inference plumbing around ``PoM.state_forward``: the two feed-forward products run on the tcgen05
GEMM with the activation and the residual add fused into its epilogue, and a whole multi-frame pass can be captured once
into a CUDA graph and replayed, which removes the per-launch host latency that dominates at a few hundred tokens per
frame.  ``train_forward`` is the same stack over whole sequences with a backward pass, in bfloat16 or float32.
"""
from __future__ import annotations

from typing import List, Optional

import torch
import torch.nn as nn

from . import _abi, ops
from .block_ops import layer_norm, linear
from .functional import BlockCausal, eager_only, on_tensor_device
from .pom import PoM


class PoMStack(nn.Module):
    """``n_layers`` x (PoM + feed-forward), each with a residual connection.

    Args:
        dim, degree, expand, n_sel_heads: of every mixer (see :class:`pom_b200.PoM`).
        n_layers:   mixers, and feed-forward blocks of width ``ffn_mult * dim``.
        norm:       a layer norm in front of every mixer and every feed-forward block (``norm_mix``, ``norm_ffn``).
        bias:       biases in the feed-forward products.
        activation: between them: "gelu" (exact), "gelu_tanh", "silu" or "relu".
    """

    def __init__(self, dim: int, degree: int, expand: int, n_layers: int, ffn_mult: int = 4, n_sel_heads: int = 1, *,
                 norm: bool = False, bias: bool = False, activation: str = "gelu"):
        super().__init__()
        if activation is None or activation not in _abi.ACTIVATIONS:
            raise ValueError(f"activation must be one of {sorted(k for k in _abi.ACTIVATIONS if k)}, got {activation!r}")
        self.dim = dim
        self.activation = activation
        self.mixers = nn.ModuleList([PoM(dim, degree, expand, 1, n_sel_heads) for _ in range(n_layers)])
        self.ffn_in = nn.ModuleList([nn.Linear(dim, ffn_mult * dim, bias=bias) for _ in range(n_layers)])
        self.ffn_out = nn.ModuleList([nn.Linear(ffn_mult * dim, dim, bias=bias) for _ in range(n_layers)])
        self.norm_mix = nn.ModuleList([nn.LayerNorm(dim) for _ in range(n_layers if norm else 0)])
        self.norm_ffn = nn.ModuleList([nn.LayerNorm(dim) for _ in range(n_layers if norm else 0)])

    def __setstate__(self, state):
        """A stack that was pickled whole before it could have norms and other activations."""
        super().__setstate__(state)
        self.__dict__.setdefault("activation", "gelu")
        for name in ("norm_mix", "norm_ffn"):
            if name not in self._modules:
                setattr(self, name, nn.ModuleList())

    @staticmethod
    def _normed(norms: nn.ModuleList, i: int, h: torch.Tensor) -> torch.Tensor:
        return layer_norm(h, norms[i].weight, norms[i].bias, norms[i].eps) if len(norms) else h

    def _feed_forward(self, i: int, h: torch.Tensor) -> torch.Tensor:
        """h + W2·act(W1·norm(h) + b1) + b2."""
        up, down = self.ffn_in[i], self.ffn_out[i]
        u = linear(self._normed(self.norm_ffn, i, h), up.weight, up.bias, activation=self.activation)
        if h.dtype == torch.float32 and PoM._autocast_dtype() is not None:
            return h + linear(u, down.weight, down.bias)  # the fused add would round the tokens with the operands
        return linear(u, down.weight, down.bias, residual=h)

    def _feed_forward_infer(self, i: int, h: torch.Tensor) -> torch.Tensor:
        """The same without a backward pass, on contiguous bf16 tokens."""
        if self.activation != "gelu" or self.ffn_in[i].bias is not None:
            return self._feed_forward(i, h)
        h2 = h.view(-1, self.dim)
        n2 = self._normed(self.norm_ffn, i, h2)
        u = ops.gemm(n2, self.ffn_in[i].weight, act="gelu")
        return ops.gemm(u, self.ffn_out[i].weight, residual=h2).view(h.shape)

    @eager_only
    @on_tensor_device
    @torch.no_grad()
    def frame_forward(self, x: torch.Tensor, states: Optional[List[Optional[dict]]] = None):
        """One frame (B, L, D) bf16 through all layers; ``states`` is the per-layer list returned by the
        previous frame (None for the first).  Returns (output, new states)."""
        if x.dtype != torch.bfloat16 or not x.is_cuda:
            raise TypeError("PoMStack runs on CUDA bfloat16 tensors")
        states = list(states) if states is not None else [None] * len(self.mixers)
        h = x.contiguous()
        for i, mixer in enumerate(self.mixers):
            n = self._normed(self.norm_mix, i, h)
            y, states[i] = mixer.state_forward(n, None, states[i], residual=h)  # x + mixer(x), add fused
            h = self._feed_forward_infer(i, y)
        return h, states

    @eager_only
    @on_tensor_device
    @torch.no_grad()
    def forward_single_pass(self, x: torch.Tensor, frame_len: int) -> torch.Tensor:
        """Same result as :meth:`forward`, all frames at once: each mixer runs with ``BlockCausal(frame_len)``, so
        every GEMM sees the whole (B·N)-row batch instead of one frame's rows."""
        if x.dtype != torch.bfloat16 or not x.is_cuda:
            raise TypeError("PoMStack runs on CUDA bfloat16 tensors")
        mask = BlockCausal(frame_len)
        h = x.contiguous()
        for i, mixer in enumerate(self.mixers):
            y = mixer(self._normed(self.norm_mix, i, h), None, mask, residual=h)
            h = self._feed_forward_infer(i, y)
        return h

    @eager_only
    @on_tensor_device
    def train_forward(self, x: torch.Tensor, mask=None) -> torch.Tensor:
        """The whole stack over (B, N, D) tokens with a backward pass, in bfloat16 or float32 (or under autocast to
        bfloat16 over float32 parameters: products in bfloat16, while float32 tokens and their gradient stay float32 along
        the residual path, as with ``torch.nn``).  ``mask`` as in ``PoM.forward``: None, "causal", a (B, N) or (B, N, N) tensor,
        or ``BlockCausal(frame_len)`` for the pattern of :meth:`forward`."""
        if x.dtype not in (torch.bfloat16, torch.float32) or not x.is_cuda:
            raise TypeError("PoMStack runs on CUDA bfloat16 or float32 tensors")
        h = x
        for i, mixer in enumerate(self.mixers):
            n = self._normed(self.norm_mix, i, h)
            # the add rides in the output projection's epilogue; float32 has none
            y = mixer(n, None, mask, residual=h) if h.dtype == torch.bfloat16 else h + mixer(n, None, mask)
            h = self._feed_forward(i, y)
        return h

    @eager_only
    @on_tensor_device
    @torch.no_grad()
    def forward(self, x: torch.Tensor, frame_len: int) -> torch.Tensor:
        """Full sequence (B, F·frame_len, D), processed frame by frame with state carried across frames."""
        outs, states = [], None
        for f in range(x.shape[1] // frame_len):
            y, states = self.frame_forward(x[:, f * frame_len:(f + 1) * frame_len], states)
            outs.append(y)
        return torch.cat(outs, dim=1)

