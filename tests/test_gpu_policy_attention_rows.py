"""Cross attention and its gradients row by row: few visible keys, peaked scores, values with a mean.

A norm over a whole tensor hides rows whose gradients are small because their terms cancel, so every
row of out and dq and every key of dk and dv is held to a bound of its own, of its terms before they
cancel.  u is the largest relative error of one rounding to bfloat16, 2^-8 (0 in float32, where no weight
is rounded), h that of a softmax weight in 32 bits (that of the exponential, and of the score: 2^-21 of the
largest that it could be), e that of a sum of products (float32: two TF32 parts and what they leave out,
2^-20; bfloat16: the tensor core's truncated accumulation over the keys, and what two bfloat16 parts of out
leave off, 2^-16).

- The weights that multiply v are rounded, and divided by their own sum: each is off by 2 (u + h) of
  itself and they still add up to 1.  So out is off by sum_j 2 (u + h) p_j |v_j - out|, not by the mean of
  v, plus e sum_j p_j |v_j| and its own rounding u |out|.
- D = dout . out is off by sum_j 2 (u + h) p_j |dp_j - D| + e |dout| sum_j p_j |v_j|, with dp_j = dout . v_j.
- ds_j = p_j (dp_j - D) is off by (2 u + 2 h) |ds_j| (the division by the rounded sum, the rounding of
  ds_j) + p_j (the error of D + e |dout| |v_j|).
- dq and dk are sums of these times |k_j| and |q_i|, off by e of the sums of |ds_j| |k_j| more; dv of the
  weights, off by 2 (u + h) each; every gradient is rounded once (u).
"""

from __future__ import annotations

import math

import pytest
import torch

from navi_b200 import policy
from tests import policy_ref as ref

pytestmark = pytest.mark.gpu

DEV = torch.device("cuda", 0)
DTYPES = [torch.float32, torch.bfloat16]


def bounds(q, k, v, do, visible):
    """The largest 2-norms of the errors of the rows of out, dq, dk and dv."""
    b, lq, h, d = q.shape
    lk, hk = k.shape[1], k.shape[2]
    scale = 1 / math.sqrt(d)
    narrow = q.dtype == torch.bfloat16
    u, e = (2.0 ** -8, 2.0 ** -16) if narrow else (2.0 ** -23, 2.0 ** -20)
    uw = u if narrow else 0.0
    keep = visible[:, :, None, None]
    wide = lambda t: torch.where(keep, t.double(), 0.0).repeat_interleave(h // hk, 2)  # noqa: E731
    q, k, v, do = q.double(), wide(k), wide(v), do.double()
    nq, nk, nv, nd = (t.norm(dim=-1).transpose(1, 2) for t in (q, k, v, do))  # [b, h, tokens]
    s = torch.einsum("blhd,bkhd->bhlk", q, k) * scale
    s = s.masked_fill(~visible[:, None, None, :], -math.inf)
    p = torch.softmax(s, -1).nan_to_num()  # rows that see nothing
    largest = (nq[..., None] * nk[:, :, None, :] * scale).amax(-1, keepdim=True)
    w = 2 * (uw + 8 * 2.0 ** -21 + 2.0 ** -21 * largest)  # of a weight
    out = torch.einsum("bhlk,bkhd->bhld", p, v)
    dp = torch.einsum("blhd,bkhd->bhlk", do, v)
    delta = (p * dp).sum(-1, keepdim=True)
    ds = p * (dp - delta)
    spread = (v.transpose(1, 2)[:, :, None] - out[..., None, :]).norm(dim=-1) if b * h * lq * lk * d <= 2 ** 26 else None
    if spread is None:
        spread = torch.stack([torch.stack([torch.cdist(out[i, j], v[i, :, j]) for j in range(h)]) for i in range(b)])
    seen = (p * nv[:, :, None, :]).sum(-1, keepdim=True)
    e_out = (w * (p * spread)).sum(-1) + e * seen[..., 0] + u * out.norm(dim=-1)
    e_delta = (w * p * (dp - delta).abs()).sum(-1, keepdim=True) + e * nd[..., None] * seen
    e_ds = w * ds.abs() + p * (e_delta + e * nd[..., None] * nv[:, :, None, :])
    group = lambda t: t.reshape(b, hk, h // hk, lk).sum(2).transpose(1, 2)  # noqa: E731
    dq = torch.einsum("bhlk,bkhd->bhld", ds, k) * scale
    dk = torch.einsum("bhlk,blhd->bhkd", ds, q).reshape(b, hk, h // hk, lk, d).sum(2).transpose(1, 2) * scale
    dv = torch.einsum("bhlk,blhd->bhkd", p, do).reshape(b, hk, h // hk, lk, d).sum(2).transpose(1, 2)
    e_dq = scale * ((e_ds + e * ds.abs()) * nk[:, :, None, :]).sum(-1) + u * dq.norm(dim=-1)
    e_dk = scale * group(((e_ds + e * ds.abs()) * nq[..., None]).sum(2)) + u * dk.norm(dim=-1)
    e_dv = group(((w + e) * p * nd[..., None]).sum(2)) + u * dv.norm(dim=-1)
    return e_out.transpose(1, 2), e_dq.transpose(1, 2), e_dk, e_dv


def hide(kind, b, lk, gen):
    """Visible keys [b, lk] and the arguments that say so: two of a longer list, by mask or by length."""
    visible = torch.ones(b, lk, dtype=torch.bool, device=DEV)
    if kind == "two by mask":
        at = torch.rand(b, lk, generator=gen, device=DEV).argsort(1)[:, :2]
        visible = torch.zeros_like(visible).scatter_(1, at, True)
        return visible, {"key_mask": visible}
    if kind == "two by length":
        visible[:, 2:] = False
        return visible, {"key_lengths": torch.full((b,), 2, dtype=torch.int32, device=DEV)}
    return visible, {}


def check(shape, dtype, kind, peak, mean, seed=0):
    b, lq, lk, h, hk, d = shape
    gen = torch.Generator(device=DEV).manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=gen, device=DEV)  # noqa: E731
    q, k = (r(b, lq, h, d) * peak).to(dtype), r(b, lk, hk, d).to(dtype)
    v, do = (r(b, lk, hk, d) + mean).to(dtype), r(b, lq, h, d).to(dtype)
    visible, kw = hide(kind, b, lk, gen)
    leaves = [t.requires_grad_() for t in (q, k, v)]
    out = policy.cross_attention(*leaves, **kw)
    got = (out.detach(), *torch.autograd.grad(out, leaves, do))
    q, k, v = (t.detach() for t in leaves)
    want = ref.attention_gradients(q, k, v, do, visible)
    for name, x, y, limit in zip(("out", "dq", "dk", "dv"), got, want, bounds(q, k, v, do, visible)):
        over = (x.double() - y).norm(dim=-1) / limit.clamp(min=1e-30)
        assert torch.isfinite(x).all() and float(over.max()) <= 1, f"{name}: a row is off by {float(over.max()):.3g} of its bound"


# 16, 60 and 200 rows to a key head: the three ways of the gradients
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("mean", [0.0, 30.0])
@pytest.mark.parametrize("kind,lk", [("all", 2), ("all", 3), ("two by mask", 200), ("two by length", 200), ("two by mask", 24)])
@pytest.mark.parametrize("lq", [8, 30, 100])
def test_few_visible_keys(lq, kind, lk, mean, dtype):
    check((3, lq, lk, 4, 2, 64), dtype, kind, 1.0, mean)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("mean", [0.0, 30.0])
@pytest.mark.parametrize("peak", [1.0, 6.0])
@pytest.mark.parametrize("lk,dim", [(48, 64), (768, 64), (300, 128), (90, 40)])
@pytest.mark.parametrize("lq", [8, 30, 100])
def test_many_keys(lq, lk, dim, peak, mean, dtype):
    check((2, lq, lk, 4, 2, dim), dtype, "all", peak, mean)


# the error of few keys in float32 is that of dp and D before they cancel; the last shape has 8 values a head
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape,kind", [((6, 1, 2, 2, 2, 64), "all"), ((1, 1, 3, 1, 1, 112), "all"), ((4, 2, 14, 1, 1, 8), "two by mask")], ids=str)
def test_small_calls(shape, kind, dtype):
    for seed in range(50):
        check(shape, dtype, kind, 1.0, 0.0, seed)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("lk", [5, 70, 512, 1300])  # rows of the mask that start on 16 bytes and do not
@pytest.mark.parametrize("lq,dim", [(1, 64), (17, 64), (100, 64), (100, 128)])
def test_one_visible_key(lq, dim, lk, dtype):
    """The softmax of one score is constant: however the key is made the only one, dq and dk are 0 and not a rounding of it."""
    q, k, v, do = (torch.randn(5, n, h, dim, device=DEV).to(dtype) for n, h in ((lq, 4), (lk, 2), (lk, 2), (lq, 4)))
    where = [0, lk - 1, lk // 2, 1]
    mask = torch.zeros(5, lk, dtype=torch.bool, device=DEV)
    mask[range(4), where] = True
    mask[4, [0, lk - 1]] = True
    mask[3, 2:] = True  # beyond its length
    lengths = torch.tensor([lk, lk, lk, 2, lk], dtype=torch.int32, device=DEV)
    leaves = [t.requires_grad_() for t in (q, k, v)]
    out = policy.cross_attention(*leaves, key_mask=mask, key_lengths=lengths)
    dq, dk, dv = torch.autograd.grad(out, leaves, do)
    assert not dq[:4].any() and not dk[:4].any()
    for b, j in enumerate(where):
        ref.assert_close(out[b], v.detach()[b, j].double().repeat_interleave(2, 0).expand_as(out[b]), ref.ONE_ROUNDING[dtype], "out")
        ref.assert_close(dv[b, j], do[b].double().reshape(lq, 2, 2, dim).sum((0, 2)), 2 * ref.ONE_ROUNDING[dtype], "dv")
    assert (dq[4] != 0).double().mean() > 0.9 and (dk[4, [0, lk - 1]] != 0).double().mean() > 0.9  # two visible keys
