"""Functional forms of the paged int8 key/value cache operators, and the table of the position rotation.

``paged_append`` and ``paged_attention`` are those of ``torch_int._CUDA``; see there for shapes and types.
"""
import torch

from torch_int import _CUDA as _ops

paged_append = _ops.paged_append
paged_attention = _ops.paged_attention


def rotary_table(rotary_dim, positions, base=10000.0, scale=1.0, device=None):
    """fp32 [positions, rotary_dim]: cosines, then sines, of position * scale * base ** (-2 i / rotary_dim).
    The angles are formed in 64 bits: in 32 bits an angle of position 10^5 is off by 4e-3 already."""
    if rotary_dim <= 0 or rotary_dim % 16 != 0:
        raise ValueError(f"rotary_dim must be a positive multiple of 16, got {rotary_dim}")
    if positions <= 0:
        raise ValueError(f"positions must be positive, got {positions}")
    i = torch.arange(0, rotary_dim, 2, dtype=torch.float64, device=device)
    angle = torch.arange(positions, dtype=torch.float64, device=device)[:, None] * (scale * base ** (-i / rotary_dim))
    return torch.cat((angle.cos(), angle.sin()), dim=1).float().contiguous()
