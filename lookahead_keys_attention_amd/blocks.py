"""Modules around the attention of a residual stream, on the HIP kernels where they can be: the gated feed-forward block and
what stands between two blocks, the counterparts of the feed-forward block and the residual sums of train_triton.py:102-107,
161-164.

`use_triton` means what it means for `Castle`: None selects the kernels for GPU tensors, False always runs the PyTorch
formulation.  True runs the kernels wherever they can be used and the formulation elsewhere (other types, autocast, modules with
hooks, sizes that the kernels do not take).
"""
from __future__ import annotations

import torch
import torch.nn.functional as F
from torch import nn
from torch.nn.modules.module import _has_any_global_hook

from . import _native, ops
from .castle import _unmodified


def _native_tensors(use_triton, *tensors) -> bool:
    """True if the kernels may take these tensors: on one GPU, of one type that they have, nothing that casts in between and no hooks on all modules."""
    first = tensors[0]
    return (use_triton is not False and first.is_cuda and first.dtype in _native.DTYPE_CODES and _native.is_built() and not torch.is_autocast_enabled("cuda") and not _has_any_global_hook()
            and all(t is None or t.dtype == first.dtype and t.device == first.device for t in tensors))


def _norm_of_rows(norm, width) -> bool:
    return _unmodified(norm, nn.RMSNorm) and norm.weight is not None and norm.weight.shape == (width,)


class GatedFeedForward(nn.Module):
    """to_out(act(g) * v) with (g, v) the halves of to_hidden(x); two thirds of the hidden width of a block without a gate give it the same number of parameters."""

    def __init__(self, dim, hidden=None, activation="silu", use_triton=None):
        super().__init__()
        if activation not in ops.GATE_ACTIVATIONS:
            raise ValueError(f"GatedFeedForward: unknown activation {activation!r}")
        hidden = -(-8 * dim // 192) * 64 if hidden is None else hidden   # 8/3 of dim, in whole 64s
        self.activation, self.use_triton = activation, use_triton
        self.to_hidden = nn.Linear(dim, 2 * hidden, bias=False)
        self.to_out = nn.Linear(hidden, dim, bias=False)

    def forward(self, x):
        up, down = self.to_hidden, self.to_out
        if (_native_tensors(self.use_triton, x, up.weight, down.weight) and _unmodified(up, nn.Linear) and _unmodified(down, nn.Linear) and up.bias is None and down.bias is None
                and ops.gated_sizes_ok(x.numel() // max(x.shape[-1], 1), x.shape[-1], down.weight.shape[1])):
            return ops.gated_feed_forward(x, up.weight, down.weight, self.activation)
        gate, value = up(x).chunk(2, dim=-1)
        return down((F.silu(gate) if self.activation == "silu" else F.gelu(gate)) * value)


class ResidualBranch(nn.Module):
    """Ends a block: residual + scale * norm(x), and the norm of that sum in front of the next block: forward(x, residual, next_norm) -> (sum, its norm).

    post_norm: an RMS norm of what the block gives; scale: None, or where the learned scale of the branch, a number for each column, begins."""

    def __init__(self, dim, post_norm=True, scale=None, use_triton=None):
        super().__init__()
        self.use_triton = use_triton
        self.norm = nn.RMSNorm(dim) if post_norm else None
        self.scale = None if scale is None else nn.Parameter(torch.full((dim,), float(scale)))

    def forward(self, x, residual, next_norm):
        norm = self.norm
        width = x.shape[-1]
        if (_norm_of_rows(next_norm, width) and (norm is None or _norm_of_rows(norm, width) and norm.eps == next_norm.eps) and x.shape == residual.shape and width <= ops.RESIDUAL_NORM_MAX_WIDTH
                and (self.scale is None or self.scale.shape == (width,))
                and _native_tensors(self.use_triton, x, residual, None if norm is None else norm.weight, self.scale, next_norm.weight)):
            return ops.residual_norm(x, residual, weight=None if norm is None else norm.weight, scale=self.scale, next_weight=next_norm.weight, eps=next_norm.eps)
        if norm is not None:
            x = norm(x)
        if self.scale is not None:
            x = x * self.scale
        y = residual + x
        return y, next_norm(y)
