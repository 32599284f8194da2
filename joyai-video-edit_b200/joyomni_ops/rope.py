"""Host-side RoPE table construction for the fused q/k kernels.

The tables are built once per forward and shared by every block, exactly as
the reference does (deploy/xvideo/models/dit/dit.py:896-934 and :1159-1163):

* ``rope_1d``: interleaved (repeat-interleaved) cos/sin of one axis,
  ``freqs = 1 / theta ** (arange(0, dim, 2)[:dim//2] / dim)``
  (deploy/xvideo/models/dit/rope.py:31-52);
* ``rope_3d``: the (t, h, w) tables concatenated along the head dimension;
* ``paired_tables``: the half-width bf16 ``[L, D/2]`` tables the paired kernels
  read, taken as every other column of the full-width tables
  (deploy/xvideo/models/dit/sgl_fused_ops.py:94-119);
* ``rotary_tables``: the half-width fp32 tables of ``rotary_embed``, with the frequencies
  stretched for long contexts (``scaled_freqs``; no reference counterpart).

These are small torch tensor computations, not kernels; the hot path only
consumes their output.
"""
from __future__ import annotations

import math
from typing import Sequence, Tuple

import torch


def rope_1d(dim: int, pos: torch.Tensor, theta: float = 10000.0) -> Tuple[torch.Tensor, torch.Tensor]:
    """Full-width interleaved cos/sin [len(pos), dim] (fp32) for one axis."""
    if dim % 2:
        raise ValueError(f"RoPE dimension must be even, got {dim}")
    pos = pos.to(torch.float32)
    freqs = 1.0 / (theta ** (torch.arange(0, dim, 2, device=pos.device)[: dim // 2].float() / dim))
    ang = torch.outer(pos, freqs)
    return ang.cos().repeat_interleave(2, dim=1), ang.sin().repeat_interleave(2, dim=1)


def grid_positions(frames: int, height: int, width: int, t0: int = 0, device=None):
    """(t, h, w) integer positions of a frames x height x width token grid, frame-major."""
    t = torch.arange(frames, device=device, dtype=torch.float32) + float(t0)
    h = torch.arange(height, device=device, dtype=torch.float32)
    w = torch.arange(width, device=device, dtype=torch.float32)
    tt = t.repeat_interleave(height * width)
    hh = h.repeat_interleave(width).repeat(frames)
    ww = w.repeat(frames * height)
    return tt, hh, ww


def rope_3d(positions: Sequence[torch.Tensor], dims: Sequence[int], theta: float = 10000.0):
    """Concatenate per-axis tables: returns full-width fp32 cos/sin [L, sum(dims)]."""
    cos, sin = [], []
    for d, p in zip(dims, positions):
        c, s = rope_1d(d, p, theta)
        cos.append(c)
        sin.append(s)
    return torch.cat(cos, dim=1), torch.cat(sin, dim=1)


def paired_tables(cos: torch.Tensor, sin: torch.Tensor, device=None):
    """Half-width bf16 [L, D/2] tables (one entry per rotated pair)."""
    return (cos[..., ::2].to(device=device, dtype=torch.bfloat16).contiguous(),
            sin[..., ::2].to(device=device, dtype=torch.bfloat16).contiguous())


def video_chunk_tables(frames: int = 3, height: int = 45, width: int = 80, t0: int = 0,
                       dims: Sequence[int] = (44, 42, 42), theta: float = 10000.0, device=None):
    """bf16 [F*H*W, D/2] cos/sin for one streaming chunk's token grid."""
    pos = grid_positions(frames, height, width, t0)
    cos, sin = rope_3d(pos, dims, theta)
    return paired_tables(cos, sin, device=device)


def scaled_freqs(dim: int, theta: float = 10000.0, scaling: str = "none", factor: float = 1.0,
                 original: int = 8192, beta: Tuple[float, float] = (32.0, 1.0)) -> Tuple[torch.Tensor, float]:
    """Inverse frequencies (fp64 [dim/2]) and the tables' scale for contexts ``factor`` times longer.

    ``"none"``: theta^(-2i/dim).  ``"linear"``: positions divided by factor.  ``"ntk"``: theta times
    factor^(dim / (dim - 2)), so the lowest frequency is divided by factor and the highest stays.
    ``"yarn"`` (Peng et al., "YaRN", 2023): frequencies that turn more than beta[0] times within the
    ``original`` context stay, those below beta[1] turns are divided by factor, a ramp in between that is
    linear in the turns, as in the paper; the tables are scaled by 0.1 ln(factor) + 1.  (Many programs have a
    ramp that is linear in the frequency's index: weights tuned with it expect other frequencies in between.)
    """
    if dim % 2 or dim <= 0:
        raise ValueError(f"RoPE dimension must be even and positive, got {dim}")
    if not factor >= 1.0:
        raise ValueError(f"factor must be at least 1, got {factor}")
    i = torch.arange(0, dim, 2, dtype=torch.float64)
    if scaling == "ntk":
        if dim == 2:
            raise ValueError("ntk scaling needs more than one frequency")
        theta = theta * factor ** (dim / (dim - 2))
    freq = theta ** (-i / dim)
    if scaling in ("none", "ntk"):
        return freq, 1.0
    if scaling == "linear":
        return freq / factor, 1.0
    if scaling == "yarn":
        fast, slow = beta
        turns = original * freq / (2 * math.pi)
        keep = ((turns - slow) / (fast - slow)).clamp(0.0, 1.0)
        return freq / factor * (1 - keep) + freq * keep, 0.1 * math.log(factor) + 1.0
    raise ValueError(f"unknown scaling {scaling!r}")


def rotary_tables(length: int, dim: int, theta: float = 10000.0, scaling: str = "none", factor: float = 1.0,
                  original: int = 8192, beta: Tuple[float, float] = (32.0, 1.0), device=None):
    """fp32 cos/sin [length, dim/2] of positions 0..length-1 for ``joyomni_ops.rotary_embed`` (angles in fp64,
    so that a position of any size keeps its phase); arguments as ``scaled_freqs``."""
    freq, scale = scaled_freqs(dim, theta, scaling, factor, original, beta)
    angle = torch.outer(torch.arange(length, dtype=torch.float64), freq)
    return ((angle.cos() * scale).to(device=device, dtype=torch.float32),
            (angle.sin() * scale).to(device=device, dtype=torch.float32))
