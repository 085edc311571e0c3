"""Operators of a policy that reads ray fans (PyTorch only hands tensors over).

- :func:`cross_attention`    queries of a policy against the tokens of a fan, with gradients
- :func:`qk_norm_rotary`     per-head RMS norm of queries and keys and the rotation by the
  token's angles in the same pass, with gradients
- :func:`clip_grad_norm`     global norm of a list of gradients, and their clipping
- :func:`fan_rotary_table`   cosines and sines for the tokens of an azimuth x elevation grid

The tensors are float32 or bfloat16 on a B200.  Every call is asynchronous on the caller's
current CUDA stream and never synchronises the host; its scratch comes from torch's allocator
on that stream.  There is no CPU path: a missing native library or a non-CUDA tensor raises
RuntimeError, and so does an argument of the wrong shape or type.
"""

from __future__ import annotations

import ctypes
import math
from typing import Iterable, Sequence

import torch
from torch.autograd.function import once_differentiable

from . import _native
from .tracer import _nvtx, _stream_handle

__all__ = ["cross_attention", "qk_norm_rotary", "clip_grad_norm", "fan_rotary_table"]

_DTYPES = {torch.float32: _native.POLICY_F32, torch.bfloat16: _native.POLICY_BF16}


def _require(ok: bool, text: str) -> None:
    if not ok:
        raise RuntimeError(text)


def _check_heads(name: str, t: torch.Tensor, like: torch.Tensor) -> None:
    _require(isinstance(t, torch.Tensor) and t.is_cuda, f"{name} must be a CUDA tensor. CPU tensors are not supported.")
    _require(t.dim() == 4, f"{name} must have shape [batch, tokens, heads, dim]")
    _require(t.dtype in _DTYPES, f"{name} must be float32 or bfloat16")
    _require(t.dtype == like.dtype, f"{name} must have the type of q")
    _require(t.device == like.device, f"{name} must be on the device of q")


def _rows(t: torch.Tensor) -> torch.Tensor:
    """`t` itself where its rows are dense and 16-byte aligned, else a contiguous copy."""
    e = t.element_size()
    b, n, h, d = t.shape
    sb, sn, sh, sd = t.stride()
    if ((sd == 1 or d <= 1) and t.data_ptr() % 16 == 0
            and ((sb if b > 1 else 0) | (sn if n > 1 else 0) | (sh if h > 1 else 0)) * e % 16 == 0):
        return t
    return t.clone(memory_format=torch.contiguous_format)


def _strides(t: torch.Tensor) -> tuple[int, int, int]:
    # the stride of an axis with one entry is never used and may be anything
    return tuple(s if n > 1 else 0 for s, n in zip(t.stride()[:3], t.shape[:3]))


def _ptr(t: torch.Tensor | None) -> int | None:
    return None if t is None else t.data_ptr()


def _scratch(n: int, device: torch.device) -> torch.Tensor | None:
    return torch.empty(n, dtype=torch.uint8, device=device) if n else None


# --- cross attention -----------------------------------------------------------


def _attention_args(q, k, v, key_mask, key_lengths, scale) -> _native.PolicyAttention:
    a = _native.PolicyAttention()
    a.device = q.device.index
    a.dtype = _DTYPES[q.dtype]
    a.batch, a.lq, a.heads, a.dim = q.shape
    a.lk, a.kv_heads = k.shape[1], k.shape[2]
    a.scale = scale
    a.q, a.k, a.v = q.data_ptr(), k.data_ptr(), v.data_ptr()
    a.q_strides[:] = _strides(q)
    a.k_strides[:] = _strides(k)
    a.v_strides[:] = _strides(v)
    if key_mask is not None:
        a.key_mask = key_mask.data_ptr()
        a.key_mask_stride = key_mask.stride(0) if key_mask.shape[0] > 1 else 0
    a.key_lengths = _ptr(key_lengths)
    return a


def _attend(q, k, v, key_mask, key_lengths, scale, want_lse):
    lib = _native.policy_lib()
    q, k, v = _rows(q), _rows(k), _rows(v)
    out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
    lse = torch.empty(q.shape[:3], dtype=torch.float32, device=q.device) if want_lse else None
    a = _attention_args(q, k, v, key_mask, key_lengths, scale)
    a.out, a.lse = out.data_ptr(), _ptr(lse)
    ws = _scratch(lib.policy_cross_attention_workspace_bytes(a, 0), q.device)
    a.workspace = _ptr(ws)
    with _nvtx("policy_cross_attention"):
        rc = lib.policy_cross_attention(a, _stream_handle(q.device))
    _native.check_policy(rc, "policy_cross_attention")
    return q, k, v, out, lse


class _CrossAttention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, key_mask, key_lengths, scale):
        q, k, v, out, lse = _attend(q, k, v, key_mask, key_lengths, scale, True)
        ctx.save_for_backward(q, k, v, key_mask, key_lengths, out, lse)
        ctx.scale = scale
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx, dout):
        q, k, v, key_mask, key_lengths, out, lse = ctx.saved_tensors
        lib = _native.policy_lib()
        dout = _rows(dout)
        dq = torch.empty(q.shape, dtype=q.dtype, device=q.device)
        dk = torch.empty(k.shape, dtype=k.dtype, device=k.device)
        dv = torch.empty(v.shape, dtype=v.dtype, device=v.device)
        a = _attention_args(q, k, v, key_mask, key_lengths, ctx.scale)
        a.out, a.lse, a.dout = out.data_ptr(), lse.data_ptr(), dout.data_ptr()
        a.dout_strides[:] = _strides(dout)
        a.dq, a.dk, a.dv = dq.data_ptr(), dk.data_ptr(), dv.data_ptr()
        ws = _scratch(lib.policy_cross_attention_workspace_bytes(a, 1), q.device)
        a.workspace = _ptr(ws)
        with _nvtx("policy_cross_attention_backward"):
            rc = lib.policy_cross_attention_backward(a, _stream_handle(q.device))
        _native.check_policy(rc, "policy_cross_attention_backward")
        return dq, dk, dv, None, None, None


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
    gradient 0.  ``scale`` defaults to 1 / sqrt(dim).

    Returns [batch, lq, heads, dim], contiguous; differentiable once in q, k and v.  Scores,
    softmax and sums are held in 32 bits; with bfloat16 the softmax weights enter the product with
    v (and with their gradients that with q and k) in bfloat16, and the outputs are rounded once.
    Tensors whose rows are not dense and 16-byte aligned are copied first.
    """
    _check_heads("q", q, q)
    _check_heads("k", k, q)
    _check_heads("v", v, q)
    b, _, h, d = q.shape
    _require(k.shape == v.shape, "k and v must have the same shape")
    _require(k.shape[0] == b and k.shape[3] == d, "k and v must have the batch and the dim of q")
    _require(k.shape[2] > 0 and h > 0 and h % k.shape[2] == 0, "the heads of q must be a positive multiple of those of k")
    _require(8 <= d <= 128 and d % 8 == 0, "dim must be a multiple of 8 from 8 to 128")
    scale = 1.0 / math.sqrt(d) if scale is None else float(scale)
    _require(0.0 < scale < math.inf, "scale must be positive and finite")
    if key_mask is not None:
        _require(key_mask.device == q.device, "key_mask must be on the device of q")
        _require(key_mask.dtype == torch.bool and tuple(key_mask.shape) == (b, k.shape[1]),
                 "key_mask must be a bool tensor of shape [batch, lk]")
        if key_mask.stride(1) != 1 and key_mask.shape[1] > 1:
            key_mask = key_mask.contiguous()
    if key_lengths is not None:
        _require(key_lengths.device == q.device, "key_lengths must be on the device of q")
        _require(key_lengths.dtype == torch.int32 and tuple(key_lengths.shape) == (b,),
                 "key_lengths must be an int32 tensor of shape [batch]")
        key_lengths = key_lengths.contiguous()
    if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad):
        return _CrossAttention.apply(q, k, v, key_mask, key_lengths, scale)
    return _attend(q, k, v, key_mask, key_lengths, scale, False)[3]


# --- norms of queries and keys with rotation -----------------------------------


def _norm_args(x2, weight2, table2, positions2, eps) -> _native.PolicyQkNorm:
    a = _native.PolicyQkNorm()
    q = x2[0]
    a.device = q.device.index
    a.dtype = _DTYPES[q.dtype]
    a.batch, a.dim = q.shape[0], q.shape[3]
    a.rotary = 2 * table2[0].shape[2] if table2[0] is not None else 0
    a.eps = eps
    for s, x, w, t, p in zip(a.side, x2, weight2, table2, positions2):
        s.x = x.data_ptr()
        s.strides[:] = _strides(x)
        s.tokens, s.heads = x.shape[1], x.shape[2]
        s.weight = _ptr(w)
        if t is not None:
            s.table, s.table_rows = t.data_ptr(), t.shape[0]
        s.positions = _ptr(p)
    return a


def _norm(q, k, q_weight, k_weight, q_table, k_table, q_positions, k_positions, eps):
    lib = _native.policy_lib()
    q, k = _rows(q), _rows(k)
    yq = torch.empty(q.shape, dtype=q.dtype, device=q.device)
    yk = torch.empty(k.shape, dtype=k.dtype, device=k.device)
    a = _norm_args((q, k), (q_weight, k_weight), (q_table, k_table), (q_positions, k_positions), eps)
    a.side[0].y, a.side[1].y = yq.data_ptr(), yk.data_ptr()
    with _nvtx("policy_qk_norm_rotary"):
        rc = lib.policy_qk_norm_rotary(a, _stream_handle(q.device))
    _native.check_policy(rc, "policy_qk_norm_rotary")
    return q, k, yq, yk


class _QkNormRotary(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, q_weight, k_weight, q_table, k_table, q_positions, k_positions, eps):
        q, k, yq, yk = _norm(q, k, q_weight, k_weight, q_table, k_table, q_positions, k_positions, eps)
        ctx.save_for_backward(q, k, q_weight, k_weight, q_table, k_table, q_positions, k_positions)
        ctx.eps = eps
        return yq, yk

    @staticmethod
    @once_differentiable
    def backward(ctx, dyq, dyk):
        q, k, q_weight, k_weight, q_table, k_table, q_positions, k_positions = ctx.saved_tensors
        lib = _native.policy_lib()
        dyq, dyk = _rows(dyq), _rows(dyk)
        a = _norm_args((q, k), (q_weight, k_weight), (q_table, k_table), (q_positions, k_positions), ctx.eps)
        dx, dw = [], []
        for s, x, dy, w, want in zip(a.side, (q, k), (dyq, dyk), (q_weight, k_weight), ctx.needs_input_grad[2:4]):
            dx.append(torch.empty(x.shape, dtype=x.dtype, device=x.device))
            dw.append(torch.empty(x.shape[3], dtype=torch.float32, device=x.device) if want else None)
            s.dy = dy.data_ptr()
            s.dy_strides[:] = _strides(dy)
            s.dx, s.dweight = dx[-1].data_ptr(), _ptr(dw[-1])
        ws = _scratch(lib.policy_qk_norm_workspace_bytes(a) if dw[0] is not None or dw[1] is not None else 0, q.device)
        a.workspace = _ptr(ws)
        with _nvtx("policy_qk_norm_rotary_backward"):
            rc = lib.policy_qk_norm_rotary_backward(a, _stream_handle(q.device))
        _native.check_policy(rc, "policy_qk_norm_rotary_backward")
        return dx[0], dx[1], dw[0], dw[1], None, None, None, None, None


def _check_weight(name: str, w: torch.Tensor | None, x: torch.Tensor) -> torch.Tensor | None:
    if w is None:
        return None
    _require(w.device == x.device and w.dtype in (torch.float32, x.dtype) and tuple(w.shape) == (x.shape[3],),
             f"{name} must be a [dim] tensor in float32 or the type of q, on its device")
    w = w.float().contiguous()
    return w if w.data_ptr() % 16 == 0 else w.clone()


def _check_table(name: str, table: torch.Tensor, x: torch.Tensor, positions: torch.Tensor | None) -> torch.Tensor:
    _require(table.device == x.device and table.dtype == torch.float32 and table.dim() == 3 and table.shape[1] == 2,
             f"{name} must be a float32 tensor of shape [rows, 2, rotary_dim / 2] on the device of q")
    _require(table.shape[2] % 8 == 0 and 0 < 2 * table.shape[2] <= x.shape[3],
             f"{name}: rotary_dim must be a multiple of 16 from 16 to dim")
    _require(positions is not None or table.shape[0] >= x.shape[1], f"{name} must have a row for every token")
    table = table.detach().contiguous()
    return table if table.data_ptr() % 16 == 0 else table.clone()


def _check_positions(name: str, p: torch.Tensor | None, x: torch.Tensor) -> torch.Tensor | None:
    if p is None:
        return None
    _require(p.device == x.device and p.dtype == torch.int32 and tuple(p.shape) == (x.shape[0], x.shape[1]),
             f"{name} must be an int32 tensor of shape [batch, tokens] on the device of q")
    return p.contiguous()


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
    _check_heads("q", q, q)
    _check_heads("k", k, q)
    _require(k.shape[0] == q.shape[0] and k.shape[3] == q.shape[3], "k must have the batch and the dim of q")
    _require(q.shape[2] > 0 and k.shape[2] > 0, "q and k must have at least one head")
    d = q.shape[3]
    _require(8 <= d <= 256 and d % 8 == 0, "dim must be a multiple of 8 from 8 to 256")
    _require((q_table is None) == (k_table is None), "q_table and k_table must be given together")
    _require(q_table is not None or (q_positions is None and k_positions is None), "positions need tables")
    _require(eps >= 0.0, "eps must not be negative")
    q_weight = _check_weight("q_weight", q_weight, q)
    k_weight = _check_weight("k_weight", k_weight, q)
    if q_table is not None:
        q_positions = _check_positions("q_positions", q_positions, q)
        k_positions = _check_positions("k_positions", k_positions, k)
        q_table = _check_table("q_table", q_table, q, q_positions)
        k_table = _check_table("k_table", k_table, k, k_positions)
        _require(q_table.shape[2] == k_table.shape[2], "q_table and k_table must have the same rotary_dim")
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (q, k, q_weight, k_weight)):
        return _QkNormRotary.apply(q, k, q_weight, k_weight, q_table, k_table, q_positions, k_positions, float(eps))
    return _norm(q, k, q_weight, k_weight, q_table, k_table, q_positions, k_positions, float(eps))[2:]


def fan_rotary_table(azimuth_bins: int, elevation_bins: int, rotary_dim: int,
                     device: torch.device | str = "cuda") -> torch.Tensor:
    """Cosines and sines [azimuth_bins * elevation_bins, 2, rotary_dim / 2] for the tokens of a fan.

    Tokens are azimuth-major, as a fan's rays are.  The first rotary_dim / 4 pairs turn by the harmonics
    1, 2, ... of the token's azimuth, so a score depends on the azimuths' difference around the full turn; the
    others by those of its elevation (from +pi/2 down to -pi/2).  Computed in 64 bits on the host.
    """
    _require(azimuth_bins > 0 and elevation_bins > 0, "azimuth_bins and elevation_bins must be positive")
    _require(rotary_dim > 0 and rotary_dim % 16 == 0, "rotary_dim must be a positive multiple of 16")
    az = torch.arange(azimuth_bins, dtype=torch.float64) * (2.0 * math.pi / azimuth_bins)
    el = torch.linspace(math.pi / 2, -math.pi / 2, elevation_bins, dtype=torch.float64)
    harmonics = torch.arange(1, rotary_dim // 4 + 1, dtype=torch.float64)
    turn_az = (az[:, None] * harmonics)[:, None, :].expand(-1, elevation_bins, -1)
    turn_el = (el[:, None] * harmonics)[None, :, :].expand(azimuth_bins, -1, -1)
    turn = torch.cat([turn_az, turn_el], -1).reshape(azimuth_bins * elevation_bins, rotary_dim // 2)
    return torch.stack([turn.cos(), turn.sin()], 1).float().to(device)


# --- global gradient norm and clipping -----------------------------------------


def _dense(t: torch.Tensor) -> bool:
    """Whether the values fill one block of memory, in whatever order."""
    if t.is_contiguous():
        return True
    expect = 1
    for stride, size in sorted((st, n) for st, n in zip(t.stride(), t.shape) if n != 1):
        if stride != expect:
            return False
        expect *= size
    return True


def clip_grad_norm(grads: Iterable[torch.Tensor], max_norm: float, *,
                   out: Sequence[torch.Tensor] | None = None) -> torch.Tensor:
    """The 2-norm over all values of ``grads``, and every gradient times min(1, max_norm / (norm + 1e-6)).

    The gradients are changed in place, or written to ``out`` (tensors of the same shapes, types and
    strides).  They are float32 or bfloat16, in any mixture, dense in memory, all on one device, and no two share
    memory.  Returns the norm before clipping, a float32 tensor without axes on the device: nothing waits for it.
    The sums do not depend on timing.  A norm that is not finite scales as the formula says: an infinite one
    by 0, NaN by NaN.
    """
    grads = list(grads)
    max_norm = float(max_norm)
    _require(max_norm >= 0.0, "max_norm must not be negative")
    _require(len(grads) > 0, "grads must not be empty")
    outs = grads if out is None else list(out)
    _require(len(outs) == len(grads), "out must have one tensor for every gradient")
    device = grads[0].device
    _require(device.type == "cuda", "grads must be CUDA tensors. CPU tensors are not supported.")
    table = (_native.PolicyGrad * len(grads))()
    seen = set()
    for entry, g, o in zip(table, grads, outs):
        dtype = _DTYPES.get(g.dtype)
        _require(dtype is not None, "grads must be float32 or bfloat16")
        _require(g.device == device, "grads must all be on one device")
        _require(_dense(g), "grads must be dense in memory")
        at = entry.out = entry.grad = g.data_ptr()
        n = entry.count = g.numel()
        entry.dtype = dtype
        if o is not g:
            _require(o.device == device and o.dtype == g.dtype and o.shape == g.shape and o.stride() == g.stride(),
                     "out must have the shapes, types, strides and device of grads")
            at = entry.out = o.data_ptr()
        if n:
            _require(at not in seen, "the tensors that are written must not share memory")
            seen.add(at)
    lib = _native.policy_lib()
    norm = torch.empty((), dtype=torch.float32, device=device)
    ws = _scratch(lib.policy_clip_grad_workspace_bytes(table, len(grads)), device)
    with _nvtx("policy_clip_grad_norm"):
        rc = lib.policy_clip_grad_norm(table, len(grads), max_norm, norm.data_ptr(), device.index, _ptr(ws),
                                       _stream_handle(device))
    _native.check_policy(rc, "policy_clip_grad_norm")
    torch.autograd.graph.increment_version(outs)  # as torch's in-place operations do
    return norm
