"""Operators of a policy that reads ray fans (PyTorch only hands tensors over).

- :func:`cross_attention`    queries of a policy against the tokens of a fan, with gradients
- :func:`qk_norm_rotary`     per-head RMS norm of queries and keys and the rotation by the
  token's angles in the same pass, with gradients
- :func:`clip_grad_norm`     global norm of a list of gradients, and their clipping
- :func:`fan_rotary_table`   cosines and sines for the tokens of an azimuth x elevation grid

The tensors are float32 or bfloat16 on a B200.  Every call is asynchronous on the caller's
current CUDA stream and never synchronises the host; its outputs and scratch come from torch's
allocator on that stream.  There is no CPU path: a missing native library or a non-CUDA tensor raises
RuntimeError, and so does a tensor of the wrong shape or dtype (what is no tensor: TypeError).  Derivatives are those of reverse mode:
a tensor that carries a forward-mode tangent raises RuntimeError, and so does a call inside ``torch.jit.trace``.
"""

from __future__ import annotations

import math
from typing import Iterable, Sequence

import torch

from . import _native
from .tracer import _NVTX, _nvtx

__all__ = ["cross_attention", "qk_norm_rotary", "clip_grad_norm", "fan_rotary_table"]


def _call(name: str, *args):
    fn = getattr(_native.policy_torch(), name)
    if not _NVTX:
        return fn(*args)
    with _nvtx(f"policy_{name}"):
        return fn(*args)


def cross_attention(
    q: torch.Tensor,
    k: torch.Tensor,
    v: torch.Tensor,
    *,
    key_mask: torch.Tensor | None = None,
    key_lengths: torch.Tensor | None = None,
    scale: float | None = None,
) -> torch.Tensor:
    """Attention of ``q`` [batch, lq, heads, dim] to ``k``, ``v`` [batch, lk, kv_heads, dim].

    ``heads`` is a multiple of ``kv_heads``; query head h reads key head h // (heads // kv_heads).
    ``dim`` is a multiple of 8 up to 128.  ``key_mask`` [batch, lk] (bool) marks the visible keys,
    such as the valid rays of an observation; ``key_lengths`` [batch] (int32) makes the keys
    from that index on invisible.  What invisible keys hold (NaN and infinities included) reaches
    no output, and their gradients are 0.  A query with no visible key gives 0 and receives
    gradient 0.  A visible value that is not finite makes what it reaches not finite.  ``scale`` defaults
    to 1 / sqrt(dim).

    Returns [batch, lq, heads, dim], contiguous; differentiable once in q, k and v.  Scores,
    softmax and sums are held in 32 bits; with bfloat16 the softmax weights enter the product with
    v (and with their gradients that with q and k) in bfloat16, are divided by their own sum, and the outputs
    are rounded once.
    Tensors whose rows are not dense and 16-byte aligned are copied first.
    """
    return _call("cross_attention", q, k, v, key_mask, key_lengths, scale)


def qk_norm_rotary(
    q: torch.Tensor,
    k: torch.Tensor,
    q_weight: torch.Tensor | None = None,
    k_weight: torch.Tensor | None = None,
    *,
    q_table: torch.Tensor | None = None,
    k_table: torch.Tensor | None = None,
    q_positions: torch.Tensor | None = None,
    k_positions: torch.Tensor | None = None,
    eps: float = 1e-6,
) -> tuple[torch.Tensor, torch.Tensor]:
    """RMS norm of every head of ``q`` [batch, lq, heads, dim] and ``k`` [batch, lk, kv_heads, dim],
    then the rotation of the first ``rotary_dim`` values of each head.

    ``u = weight * x / sqrt(mean(x^2) + eps)``; with the cosines c and sines s of the token's row of
    the table [rows, 2, rotary_dim / 2] (:func:`fan_rotary_table`) and n = rotary_dim / 2,
    ``y[i] = u[i] c[i] - u[i + n] s[i]`` and ``y[i + n] = u[i + n] c[i] + u[i] s[i]``.  The row is
    the token's index, or its entry of ``positions`` [batch, tokens] (int32); a position outside
    the table gives a row of NaN.  Both tables or neither are given, with the same rotary_dim.
    ``dim`` is a multiple of 8 up to 256, ``rotary_dim`` of 16.  The two lengths are independent and
    may be 0.

    Returns both results, contiguous, in the type of q; differentiable once in q, k and the weights
    (not in the tables).  Everything up to the one rounding of the result is in 32 bits.
    """
    return _call("qk_norm_rotary", q, k, q_weight, k_weight, q_table, k_table, q_positions, k_positions, eps)


def fan_rotary_table(azimuth_bins: int, elevation_bins: int, rotary_dim: int,
                     device: torch.device | str = "cuda") -> torch.Tensor:
    """Cosines and sines [azimuth_bins * elevation_bins, 2, rotary_dim / 2] for the tokens of a fan.

    Tokens are azimuth-major, as a fan's rays are.  The first rotary_dim / 4 pairs turn by the harmonics
    1, 2, ... of the token's azimuth, so a score depends on the azimuths' difference around the full turn; the
    others by those of its elevation (from +pi/2 down to -pi/2).  Computed in 64 bits on the host.
    """
    if azimuth_bins < 1 or elevation_bins < 1:
        raise RuntimeError("azimuth_bins and elevation_bins must be positive")
    if rotary_dim < 1 or rotary_dim % 16 != 0:
        raise RuntimeError("rotary_dim must be a positive multiple of 16")
    az = torch.arange(azimuth_bins, dtype=torch.float64) * (2.0 * math.pi / azimuth_bins)
    el = torch.linspace(math.pi / 2, -math.pi / 2, elevation_bins, dtype=torch.float64)
    harmonics = torch.arange(1, rotary_dim // 4 + 1, dtype=torch.float64)
    turn_az = (az[:, None] * harmonics)[:, None, :].expand(-1, elevation_bins, -1)
    turn_el = (el[:, None] * harmonics)[None, :, :].expand(azimuth_bins, -1, -1)
    turn = torch.cat([turn_az, turn_el], -1).reshape(azimuth_bins * elevation_bins, rotary_dim // 2)
    return torch.stack([turn.cos(), turn.sin()], 1).float().to(device)


def clip_grad_norm(grads: Iterable[torch.Tensor], max_norm: float, *,
                   out: Sequence[torch.Tensor] | None = None) -> torch.Tensor:
    """The 2-norm over all values of ``grads``, and every gradient times min(1, max_norm / (norm + 1e-6)).

    The gradients are changed in place, or written to ``out`` (tensors of the same shapes, types and
    strides).  They are float32 or bfloat16, in any mixture, dense in memory, all on one device.  What is written shares
    memory with nothing else: no two of the changed gradients, and no ``out`` with a gradient other than its
    own.  Returns the norm before clipping, a float32 tensor without axes on the device: nothing waits for it.
    The sums do not depend on timing.  A norm that is not finite scales as the formula says: an infinite one
    by 0, NaN by NaN.
    """
    return _call("clip_grad_norm", list(grads), max_norm, None if out is None else list(out))
