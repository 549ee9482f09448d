"""Rotary positions over several axes (time, height and width of video tokens, or text).

`apply_rotary` turns the pairs of dims of every query and key row by angles that
follow from the token's position on each axis. It reads rows in the layout the
projections leave them in and writes the [B, H, N, 128] that the attention entry
points take, so no transposed copy is made. The rows are read and written once;
angles are computed in 64 bits on the fly. Like the rest of the package it has
no autograd; the turn is orthogonal, so its gradient is the turn back:
``apply_rotary(grad_q, grad_k, positions, axes, inverse=True)``.
"""
from __future__ import annotations

from typing import NamedTuple

import torch


class RotaryAxes(NamedTuple):
    """Which dims of a head turn with which axis of a position, and how fast.

    ``sections`` - even numbers of dims, one per axis (1 to 4 axes), in order; they sum to 128.
    ``theta``    - pair i of an axis with d dims turns by position * theta^(-2i/d).
    ``paired``   - True: dims (2i, 2i + 1) form a pair; False: (i, i + 64).
    ``shared``   - True: frequencies run over the whole head (theta^(-2i/128), i of all 64
                   pairs) and the axes share its pairs out; False: each axis has its own.
    """

    sections: tuple[int, ...] = (44, 42, 42)
    theta: float = 10000.0
    paired: bool = True
    shared: bool = False


VIDEO_AXES = RotaryAxes()


def grid_positions(frames: int, height: int, width: int, *, first_frame: int = 0, device=None) -> torch.Tensor:
    """int32 [frames * height * width, 3]: (frame, row, column) of the tokens in row-major
    order; index it with `cube_layout`'s order for tokens in cubes."""
    t, h, w = (torch.arange(n, dtype=torch.int32, device=device) for n in (frames, height, width))
    return torch.stack(torch.meshgrid(t + first_frame, h, w, indexing="ij"), -1).reshape(-1, 3)


def _on_gpu(x: torch.Tensor) -> None:
    if x.is_cpu:
        raise ValueError("B200 operators require CUDA tensors")


def apply_rotary(q, k, positions, axes=VIDEO_AXES, *, inverse=False):
    """Turns q [B, H, N, 128] and k [B, Hk, N, 128] (or None); bf16, fp16 or f32.

    positions: int32 [N, axes] or [B, N, axes]. Returns contiguous (q, k), which carry no gradient. Rows may be
    strided (a [B, N, H, 128] projection transposed to [B, H, N, 128]) as long as the 128
    dims are contiguous and rows start on 16-byte boundaries; else they are copied first.
    """
    _on_gpu(q)
    sections, theta, paired, shared = axes
    q_out, k_out = torch.ops.ab_attention.rotary(q, k, positions, sections, theta, shared, not paired, inverse)
    return q_out, None if k is None else k_out
