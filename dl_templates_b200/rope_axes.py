"""Rotary positions with several axes (time, height, width) for sequences of text, images and video.

  ``RotaryPEAxes.apply(q, k, positions, *tables) -> (q_rot, k_rot)``     differentiable, q and k stay untouched
  ``RotaryPositionEncodingAxes(components, max_positions)``              module holding the tables
  ``rope_axes_apply_to(x, positions, tables, inverse=False)``            one tensor, no autograd graph

The layout is that of ``RotaryPE2D`` (``fused_rope2d.py``) for any number of axes up to four: axis ``a`` with ``R_a`` pairs takes the next
``2 R_a`` dims of a row and turns dims ``i`` and ``R_a + i`` of them by the angle of the token's position on that axis; dims behind
the last axis pass through.  One axis is the rotary embedding of text, two with equal pairs are ``RotaryPE2D``.
A negative position leaves that axis of the token unrotated (a text token among image patches); a position behind the end of
an axis' table takes the table's last row.
"""
from __future__ import annotations

import torch

from ._lib import native as _native
from .fused_rope2d import make_cs_table
from .sink_swa import SinkSwa


def rope_axes_apply_to(x: torch.Tensor, positions: torch.Tensor, tables, inverse: bool = False) -> torch.Tensor:
    """The rotation (or its inverse) of ``x [B,H,N,C]`` in a new contiguous tensor; no autograd graph (tangents and jit traces are
    refused).  ``positions``: int32 ``[axes, N]`` or ``[B, axes, N]``; ``tables``: one fp32 ``[max_position, pairs, 2]`` (cos, sin)
    table per axis (``make_cs_table``)."""
    return _native.rope_axes_to(x, positions, tables, int(inverse))


class RotaryPEAxes(torch.autograd.Function):
    """``RotaryPEAxes.apply(q, k, positions, *tables) -> (q_rot, k_rot)``: q ``[B,Hq,N,C]`` and k ``[B,Hkv,N,C]`` (any strides)
    rotated in one launch into new contiguous tensors; backward turns the gradients back in one launch.  ``apply`` runs natively;
    ``forward`` and ``backward`` are the general path (functorch, tracing), as in ``TiledSwa``."""

    apply = staticmethod(_native.rope_axes)

    @staticmethod
    def forward(ctx, q, k, positions, *tables):
        ctx.save_for_backward(positions, *tables)
        return _native.rope_axes_to_body(q, positions, tables, 0), _native.rope_axes_to_body(k, positions, tables, 0)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dq, dk):
        positions, *tables = ctx.saved_tensors
        return (_native.rope_axes_to_body(dq, positions, tables, 1), _native.rope_axes_to_body(dk, positions, tables, 1), None,
                *(None,) * len(tables))


class RotaryPositionEncodingAxes(torch.nn.Module):
    """Module form: ``components[a]`` pairs and ``max_positions[a]`` positions of each axis."""

    def __init__(self, components, max_positions, theta: float = 10000.0):
        super().__init__()
        if len(components) != len(max_positions) or not 1 <= len(components) <= 4:
            raise ValueError("one component count and one length for each of 1 to 4 axes expected")
        self.n_axes = len(components)
        for a, (r, n) in enumerate(zip(components, max_positions)):
            self.register_buffer(f"cs_{a}", make_cs_table(r, n, theta), persistent=False)

    @property
    def tables(self):
        return tuple(getattr(self, f"cs_{a}") for a in range(self.n_axes))

    @staticmethod
    def grid_positions(*shape: int) -> torch.Tensor:
        """Positions ``[axes, N]`` of the cells of a grid (frames, height, width, ...) in row-major order."""
        axes = torch.meshgrid(*(torch.arange(n, dtype=torch.int32) for n in shape), indexing="ij")
        return torch.stack([a.reshape(-1) for a in axes]).contiguous()

    def forward(self, q: torch.Tensor, k: torch.Tensor, positions: torch.Tensor):
        return RotaryPEAxes.apply(q, k, positions, *self.tables)


_native.set_general_sequence(super(RotaryPEAxes, RotaryPEAxes).apply, super(SinkSwa, SinkSwa).apply)
