"""The policy operators restated in 64 bits (torch, any device), and the comparison with them.

Tolerances, as the 2-norm of the difference over that of the result, are derived, not fitted:

- bfloat16 keeps 8 bits: one rounding is off by at most 2^-8 of the value, and, with the value's
  place between two numbers even, by less than 2^-9 in the mean square.  An output of one rounding
  is within 2^-8, however few values it has.  Attention is compared on at least a few dozen values,
  in the mean square: 2^-9 for the output's rounding; another for that of the softmax weights (or,
  for dq and dk, the weights' gradients), whose roundings are independent over the keys and, with
  values of independent signs, add in quadrature as the products themselves do; the gradients read
  the rounded output through D = do . out: a third 2^-9.
- float32 attention splits every operand into two TF32 values; what it leaves out of a product
  is below 2^-21 of it, and the exponent of a softmax weight carries the error of one product sum
  (the scores' size, a few units, times 2^-21).  8 * 2^-21 forward; twice that for gradients, which
  go through two products after the weights.
- norms, rotations and clipping in float32 are a handful of roundings of 2^-24 each: 8 * 2^-24 = 2^-21;
  the weights' gradients sum over all rows, n roundings of partial sums in quadrature: 2^-21 as well at
  the sizes here (a thread sums at most a few hundred rows).

A single value may be off by 16 times that, relative to the larger of itself and the root mean square.
"""

from __future__ import annotations

import math

import torch

FORWARD = {torch.bfloat16: 2 * 2.0 ** -9, torch.float32: 8 * 2.0 ** -21}
GRADIENT = {torch.bfloat16: 3 * 2.0 ** -9, torch.float32: 16 * 2.0 ** -21}
ONE_ROUNDING = {torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -21}


def attention(q, k, v, visible=None, scale=None):
    """[B, Lq, H, D] x [B, Lk, Hk, D] in 64 bits; visible [B, Lk]; rows without a visible key give 0."""
    b, lq, h, d = q.shape
    lk, hk = k.shape[1], k.shape[2]
    scale = 1 / math.sqrt(d) if scale is None else scale
    if visible is None:
        visible = torch.ones(b, lk, dtype=torch.bool, device=q.device)
    keep = visible[:, :, None, None]
    q = q.double()
    k = torch.where(keep, k.double(), 0.0).repeat_interleave(h // hk, 2)
    v = torch.where(keep, v.double(), 0.0).repeat_interleave(h // hk, 2)
    s = torch.einsum("blhd,bkhd->bhlk", q, k) * scale
    s = torch.where(visible[:, None, None, :], s, -math.inf)
    m = s.amax(-1, keepdim=True) if lk else s.new_zeros(b, h, lq, 1)
    e = torch.exp(s - torch.where(m == -math.inf, 0.0, m))
    total = e.sum(-1, keepdim=True)
    p = e / torch.where(total == 0, 1.0, total)
    return torch.einsum("bhlk,bkhd->blhd", p, v)


def attention_gradients(q, k, v, dout, visible=None, scale=None):
    """out, dq, dk, dv by the formulas of the softmax's gradient."""
    b, lq, h, d = q.shape
    lk, hk = k.shape[1], k.shape[2]
    g = h // hk
    scale = 1 / math.sqrt(d) if scale is None else scale
    if visible is None:
        visible = torch.ones(b, lk, dtype=torch.bool, device=q.device)
    out = attention(q, k, v, visible, scale)
    keep = visible[:, :, None, None]
    kd = torch.where(keep, k.double(), 0.0).repeat_interleave(g, 2)
    vd = torch.where(keep, v.double(), 0.0).repeat_interleave(g, 2)
    qd, dd = q.double(), dout.double()
    s = torch.einsum("blhd,bkhd->bhlk", qd, kd) * scale
    s = torch.where(visible[:, None, None, :], s, -math.inf)
    m = s.amax(-1, keepdim=True)
    e = torch.exp(s - torch.where(m == -math.inf, 0.0, m))
    total = e.sum(-1, keepdim=True)
    p = e / torch.where(total == 0, 1.0, total)
    dp = torch.einsum("blhd,bkhd->bhlk", dd, vd)
    ds = p * (dp - (dd * out).sum(-1).permute(0, 2, 1)[..., None]) * scale
    dq = torch.einsum("bhlk,bkhd->blhd", ds, kd)
    dk = torch.einsum("bhlk,blhd->bkhd", ds, qd).reshape(b, lk, hk, g, d).sum(3)
    dv = torch.einsum("bhlk,blhd->bkhd", p, dd).reshape(b, lk, hk, g, d).sum(3)
    return out, dq, dk, dv


def norm_rotary(x, weight=None, table=None, positions=None, eps=1e-6):
    x = x.double()
    u = x / torch.sqrt((x * x).mean(-1, keepdim=True) + eps)
    if weight is not None:
        u = u * weight.double()
    if table is None:
        return u
    t = table.double()
    rows = t[positions.long()] if positions is not None else t[: x.shape[1]].expand(x.shape[0], -1, -1, -1)
    c, s = rows[..., 0, :].unsqueeze(2), rows[..., 1, :].unsqueeze(2)
    n = table.shape[2]
    return torch.cat([u[..., :n] * c - u[..., n:2 * n] * s, u[..., n:2 * n] * c + u[..., :n] * s, u[..., 2 * n:]], -1)


def norm_rotary_gradients(x, weight, table, positions, dy, eps=1e-6):
    """dx and dweight by the formulas: back through the rotation, then through the norm."""
    x, d = x.double(), x.shape[-1]
    w = weight.double() if weight is not None else torch.ones(d, dtype=torch.float64, device=x.device)
    g = dy.double()
    if table is not None:
        t = table.double()
        rows = t[positions.long()] if positions is not None else t[: x.shape[1]].expand(x.shape[0], -1, -1, -1)
        c, s = rows[..., 0, :].unsqueeze(2), rows[..., 1, :].unsqueeze(2)
        n = table.shape[2]
        g = torch.cat([g[..., :n] * c + g[..., n:2 * n] * s, g[..., n:2 * n] * c - g[..., :n] * s, g[..., 2 * n:]], -1)
    r = 1 / torch.sqrt((x * x).mean(-1, keepdim=True) + eps)
    dx = r * w * g - r ** 3 * x * (w * g * x).mean(-1, keepdim=True)
    return dx, (g * x * r).sum((0, 1, 2))


def assert_close(got: torch.Tensor, want: torch.Tensor, tol: float, what: str) -> None:
    got, want = got.detach().double(), want.double()
    assert got.shape == want.shape, f"{what}: shape {tuple(got.shape)}, expected {tuple(want.shape)}"
    if want.numel() == 0:
        return
    assert torch.isfinite(got).all(), f"{what}: {int((~torch.isfinite(got)).sum())} values are not finite"
    diff = got - want
    norm = float(want.norm())
    if norm == 0:
        assert float(diff.norm()) == 0, f"{what}: expected zeros"
        return
    rel = float(diff.norm()) / norm
    rms = norm / math.sqrt(want.numel())
    worst = float((diff.abs() / want.abs().clamp(min=rms)).max())
    assert rel <= tol, f"{what}: relative error {rel:.3g} over {tol:.3g}"
    assert worst <= 16 * tol, f"{what}: a value is off by {worst:.3g}, over {16 * tol:.3g}"
