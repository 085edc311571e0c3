"""Norms of queries and keys with rotation against the 64-bit restatement (tests/policy_ref.py)."""

from __future__ import annotations

import math

import pytest
import torch

from navi_b200 import policy
from tests import policy_ref as ref

pytestmark = pytest.mark.gpu

DEV = torch.device("cuda", 0)
DTYPES = [torch.float32, torch.bfloat16]

# batch, lq, lk, heads, kv_heads, dim, rotary
SHAPES = [
    (1, 1, 1, 1, 1, 8, 0),
    (1, 1, 1, 1, 1, 16, 16),
    (2, 1, 77, 4, 2, 32, 32),
    (3, 9, 130, 6, 3, 40, 16),
    (2, 33, 5, 5, 1, 64, 48),
    (2, 7, 300, 9, 4, 96, 96),
    (1, 64, 65, 8, 8, 128, 64),
    (2, 3, 19, 3, 2, 256, 256),
    (2, 3, 19, 3, 2, 200, 160),
    (16, 40, 900, 8, 2, 64, 64),
]


def inputs(shape, dtype, positions, seed=0):
    b, lq, lk, h, hk, d, rot = shape
    gen = torch.Generator(device=DEV).manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=gen, device=DEV)  # noqa: E731
    q, k = r(b, lq, h, d).to(dtype), r(b, lk, hk, d).to(dtype)
    dq, dk = r(b, lq, h, d).to(dtype), r(b, lk, hk, d).to(dtype)
    wq, wk = 1 + 0.2 * r(d), 1 + 0.2 * r(d)
    kw = {}
    if rot:
        for name, n in (("q", lq), ("k", lk)):
            rows = n + 3
            angle = 7 * r(rows, rot // 2)
            kw[name + "_table"] = torch.stack([angle.cos(), angle.sin()], 1)
            if positions:
                kw[name + "_positions"] = torch.randint(0, rows, (b, n), generator=gen, device=DEV, dtype=torch.int32)
    return q, k, wq, wk, dq, dk, kw


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("positions", [False, True])
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_output_and_gradients(shape, positions, dtype):
    q, k, wq, wk, dq, dk, kw = inputs(shape, dtype, positions)
    leaves = [t.requires_grad_() for t in (q, k, wq, wk)]
    yq, yk = policy.qk_norm_rotary(*leaves, **kw)
    got = torch.autograd.grad((yq, yk), leaves, (dq, dk))
    with torch.no_grad():
        pq, pk = policy.qk_norm_rotary(*leaves, **kw)
    assert torch.equal(pq, yq.detach()) and torch.equal(pk, yk.detach())
    for i, (x, w, y, dy, n) in enumerate(((q, wq, yq, dq, "q"), (k, wk, yk, dk, "k"))):
        table, pos = kw.get(n + "_table"), kw.get(n + "_positions")
        ref.assert_close(y, ref.norm_rotary(x.detach(), w.detach(), table, pos), ref.ONE_ROUNDING[dtype], n)
        dx, dw = ref.norm_rotary_gradients(x.detach(), w.detach(), table, pos, dy)
        ref.assert_close(got[i], dx, ref.ONE_ROUNDING[dtype], "d" + n)
        ref.assert_close(got[2 + i], dw, 2.0 ** -21, "dweight of " + n)


@pytest.mark.parametrize("dtype", DTYPES)
def test_without_weights_or_tables(dtype):
    q, k, _, _, dq, dk, _ = inputs((2, 5, 40, 4, 2, 48, 0), dtype, False)
    leaves = [t.requires_grad_() for t in (q, k)]
    yq, yk = policy.qk_norm_rotary(q, k)
    gq, gk = torch.autograd.grad((yq, yk), leaves, (dq, dk))
    for x, y, dy, g in ((q, yq, dq, gq), (k, yk, dk, gk)):
        ref.assert_close(y, ref.norm_rotary(x.detach()), ref.ONE_ROUNDING[dtype], "y")
        ref.assert_close(g, ref.norm_rotary_gradients(x.detach(), None, None, None, dy)[0], ref.ONE_ROUNDING[dtype], "dx")


def test_weights_in_the_inputs_type():
    q, k, wq, wk, dq, dk, kw = inputs((2, 5, 40, 4, 2, 48, 32), torch.bfloat16, False)
    wq, wk = wq.bfloat16().requires_grad_(), wk.bfloat16().requires_grad_()
    yq, yk = policy.qk_norm_rotary(q, k, wq, wk, **kw)
    gq, gk = torch.autograd.grad((yq, yk), (wq, wk), (dq, dk))
    for x, w, y, dy, g, n in ((q, wq, yq, dq, gq, "q"), (k, wk, yk, dk, gk, "k")):
        ref.assert_close(y, ref.norm_rotary(x, w.detach(), kw[n + "_table"]), ref.ONE_ROUNDING[torch.bfloat16], n)
        want = ref.norm_rotary_gradients(x, w.detach(), kw[n + "_table"], None, dy)[1]
        assert g.dtype == torch.bfloat16
        ref.assert_close(g, want, ref.ONE_ROUNDING[torch.bfloat16], "dweight of " + n)


def test_one_result_used_and_one_input_wanted():
    q, k, wq, wk, dq, _, kw = inputs((2, 5, 40, 4, 2, 48, 32), torch.float32, False)
    q.requires_grad_()
    yq, yk = policy.qk_norm_rotary(q, k, wq, wk, **kw)
    (g,) = torch.autograd.grad(yq, q, dq)
    ref.assert_close(g, ref.norm_rotary_gradients(q.detach(), wq, kw["q_table"], None, dq)[0], 2.0 ** -21, "dq")


@pytest.mark.parametrize("lq,lk,b", [(0, 7, 2), (7, 0, 2), (3, 3, 0)])
def test_empty(b, lq, lk):
    q, k, wq, wk, dq, dk, kw = inputs((b, lq, lk, 4, 2, 32, 16), torch.float32, False)
    leaves = [t.requires_grad_() for t in (q, k, wq, wk)]
    yq, yk = policy.qk_norm_rotary(*leaves, **kw)
    grads = torch.autograd.grad((yq, yk), leaves, (dq, dk))
    assert yq.shape == q.shape and yk.shape == k.shape
    for g, t in zip(grads, leaves):
        assert g.shape == t.shape and torch.isfinite(g).all()
    assert bool(grads[2].any()) == (b * lq > 0) and bool(grads[3].any()) == (b * lk > 0)


@pytest.mark.parametrize("dtype", DTYPES)
def test_zero_rows_and_padding_lanes_without_eps(dtype):
    """Rows of zeros give zeros with eps; heads that do not fill a group and dims that do not fill the lanes leave
    no NaN in the weights' gradients without it."""
    q, k, wq, wk, dq, dk, kw = inputs((1, 3, 5, 5, 3, 40, 16), dtype, False)
    leaves = [t.requires_grad_() for t in (q, k, wq, wk)]
    grads = torch.autograd.grad(policy.qk_norm_rotary(*leaves, **kw, eps=0.0), leaves, (dq, dk))
    assert all(torch.isfinite(g).all() for g in grads)
    with torch.no_grad():
        y, _ = policy.qk_norm_rotary(torch.zeros_like(q), k, wq, wk, **kw)
    assert not y.any()


def test_positions_outside_the_table_give_nan():
    q, k, wq, wk, dq, dk, kw = inputs((2, 4, 6, 2, 2, 32, 16), torch.float32, True)
    kw["q_positions"][0, 1] = -1
    kw["k_positions"][1, 2] = kw["k_table"].shape[0]
    yq, yk = policy.qk_norm_rotary(q, k, wq, wk, **kw)
    assert torch.isnan(yq[0, 1]).all() and torch.isnan(yk[1, 2]).all()
    assert int(torch.isnan(yq).sum()) == 64 and int(torch.isnan(yk).sum()) == 64


@pytest.mark.parametrize("dtype", DTYPES)
def test_strided_views_give_the_same_bits(dtype):
    b, n, h, d = 3, 50, 4, 64
    gen = torch.Generator(device=DEV).manual_seed(1)
    fused = torch.randn(b, n, 2 * h * d, generator=gen, device=DEV).to(dtype)
    q, k = fused[..., : h * d].view(b, n, h, d), fused[..., h * d:].view(b, n, h, d)
    dy = torch.randn(b, h, n, d, generator=gen, device=DEV).to(dtype).transpose(1, 2)
    table = torch.randn(n, 2, 16, generator=gen, device=DEV)
    w = torch.randn(d, generator=gen, device=DEV)

    def run(q, k, dy):
        q, k, wq, wk = (t.detach().requires_grad_() for t in (q, k, w, w))
        y = policy.qk_norm_rotary(q, k, wq, wk, q_table=table, k_table=table)
        return (*(t.detach() for t in y), *torch.autograd.grad(y, (q, k, wq, wk), (dy, dy)))

    want = run(q.contiguous(), k.contiguous(), dy.contiguous())
    odd = lambda t: torch.nn.functional.pad(t, (1, 2))[..., 1:-2]  # noqa: E731
    for got in (run(q, k, dy), run(odd(q), odd(k), odd(dy))):
        for x, y in zip(got, want):
            assert torch.equal(x, y)


def test_gradient_against_differences():
    q, k, wq, wk, dq, dk, kw = inputs((2, 6, 9, 3, 2, 40, 32), torch.float32, True, 4)
    leaves = [t.requires_grad_() for t in (q, k, wq, wk)]
    grads = torch.autograd.grad(policy.qk_norm_rotary(*leaves, **kw), leaves, (dq, dk))
    h = 1e-4
    for i, g in enumerate(grads):
        direction = torch.randn_like(g, dtype=torch.float64)

        def value(sign, i=i, direction=direction):
            x = [t.detach().double() for t in leaves]
            x[i] = x[i] + sign * h * direction
            yq = ref.norm_rotary(x[0], x[2], kw["q_table"], kw["q_positions"])
            yk = ref.norm_rotary(x[1], x[3], kw["k_table"], kw["k_positions"])
            return float((yq * dq.double()).sum() + (yk * dk.double()).sum())

        want = (value(1) - value(-1)) / (2 * h)
        got = float((g.double() * direction).sum())
        size = float(g.double().norm() * direction.norm()) / math.sqrt(g.numel())
        # the differences' own error is h^2 times the third derivative, about 1e-7
        assert abs(got - want) <= 16 * 2.0 ** -21 * max(abs(want), size) + 1e-6 * size, (i, got, want)


def test_bits_do_not_depend_on_timing():
    q, k, wq, wk, dq, dk, kw = inputs((64, 16, 700, 8, 2, 64, 64), torch.bfloat16, False)
    leaves = [t.requires_grad_() for t in (q, k, wq, wk)]
    runs = [torch.autograd.grad(policy.qk_norm_rotary(*leaves, **kw), leaves, (dq, dk)) for _ in range(4)]
    for r in runs[1:]:
        assert all(torch.equal(x, y) for x, y in zip(r, runs[0]))


@pytest.mark.parametrize("az,el,rot", [(8, 4, 32), (5, 1, 16), (64, 16, 64)])
def test_fan_table(az, el, rot):
    """Scores of rotated tokens depend on the azimuths' difference around the full turn."""
    table = policy.fan_rotary_table(az, el, rot, DEV)
    assert table.shape == (az * el, 2, rot // 2) and table.dtype == torch.float32
    x = torch.randn(1, 1, 1, rot, device=DEV)
    y = torch.randn(1, 1, 1, rot, device=DEV)
    n = az * el
    rx, ry = policy.qk_norm_rotary(x.expand(1, n, 1, rot), y.expand(1, n, 1, rot), q_table=table, k_table=table)
    rx, ry = rx.view(az, el, rot).double(), ry.view(az, el, rot).double()
    base = (rx[0] * ry[1 % az]).sum(-1)
    for a in range(az):
        # float32 cosines and results: a few roundings of 2^-24 in each of rot products
        assert torch.allclose((rx[a] * ry[(a + 1) % az]).sum(-1), base, rtol=0, atol=rot * 2.0 ** -21)


def test_refusals():
    q, k, wq, wk, _, _, kw = inputs((2, 4, 6, 4, 2, 32, 16), torch.float32, True)
    t, p = kw["q_table"], kw["q_positions"]
    bad = [
        ((q.cpu(), k), {}, "q must be a CUDA tensor"),
        ((q, k.cpu()), {}, "k must be a CUDA tensor"),
        ((q, k.bfloat16()), {}, "k must have the type of q"),
        ((q, k[..., :16]), {}, "the batch and the dim of q"),
        ((q[..., :12], k[..., :12]), {}, "multiple of 8"),
        ((q, k, wq[:16]), {}, "q_weight must be"),
        ((q, k, wq.double()), {}, "q_weight must be"),
        ((q, k, wq, wk), {"q_table": t}, "given together"),
        ((q, k), {"q_positions": p}, "positions need tables"),
        ((q, k), {"q_table": t[:3], "k_table": kw["k_table"]}, "a row for every token"),
        ((q, k), {"q_table": t.double(), "k_table": kw["k_table"]}, "q_table must be a float32"),
        ((q, k), {"q_table": t[..., :4], "k_table": kw["k_table"]}, "multiple of 16"),
        ((q, k), {**kw, "q_positions": p.long()}, "q_positions must be an int32"),
        ((q, k), {"eps": -1.0}, "eps must not be negative"),
    ]
    for args, more, text in bad:
        with pytest.raises(RuntimeError, match=text):
            policy.qk_norm_rotary(*args, **more)
    with pytest.raises(RuntimeError, match="same rotary_dim"):
        policy.qk_norm_rotary(q, k, q_table=torch.randn(9, 2, 8, device=DEV), k_table=torch.randn(9, 2, 16, device=DEV))
