"""Cross attention against the 64-bit restatement (tests/policy_ref.py, which derives the tolerances)."""

from __future__ import annotations

import math

import pytest
import torch

from navi_b200 import policy
from tests import policy_ref as ref

pytestmark = pytest.mark.gpu

DEV = torch.device("cuda", 0)
DTYPES = [torch.float32, torch.bfloat16]

# batch, lq, lk, heads, kv_heads, dim: one value of everything, every padded head dimension and row tile, tiles
# that end inside, shared heads, keys split over blocks, rows split over blocks
SHAPES = [
    (1, 1, 1, 1, 1, 8),
    (2, 1, 17, 4, 2, 32),
    (3, 5, 129, 6, 3, 40),
    (2, 16, 192, 8, 8, 64),
    (2, 17, 65, 4, 4, 64),
    (1, 33, 257, 8, 1, 96),
    (2, 70, 130, 4, 2, 128),
    (1, 3, 5001, 2, 1, 64),
    (1, 2, 4099, 16, 1, 128),
    (1, 1500, 3, 2, 2, 16),
    (2, 300, 1031, 2, 1, 80),
    (1, 9, 2000, 4, 2, 24),
]


def inputs(shape, dtype, seed=0, mask="none", poison=False):
    b, lq, lk, h, hk, d = shape
    gen = torch.Generator(device=DEV).manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=gen, device=DEV)  # noqa: E731
    q, k, v, do = r(b, lq, h, d).to(dtype), r(b, lk, hk, d).to(dtype), r(b, lk, hk, d).to(dtype), r(b, lq, h, d).to(dtype)
    kw, visible = {}, torch.ones(b, lk, dtype=torch.bool, device=DEV)
    if mask in ("mask", "both"):
        kw["key_mask"] = torch.rand(b, lk, generator=gen, device=DEV) > 0.3
        kw["key_mask"][0] = False  # rows that see nothing
        visible &= kw["key_mask"]
    if mask in ("lengths", "both"):
        kw["key_lengths"] = torch.randint(0, lk + 1, (b,), generator=gen, device=DEV, dtype=torch.int32)
        visible &= torch.arange(lk, device=DEV)[None] < kw["key_lengths"][:, None]
    if poison:  # what invisible keys hold must not matter
        bad = torch.tensor([math.nan, math.inf, -math.inf, 3e38], device=DEV).to(dtype)
        fill = bad[torch.arange(lk, device=DEV) % 4][None, :, None, None].expand_as(k)
        k = torch.where(visible[:, :, None, None], k, fill)
        v = torch.where(visible[:, :, None, None], v, fill)
    return q, k, v, do, kw, visible


def check(shape, dtype, mask, seed=0, poison=False, **extra):
    q, k, v, do, kw, visible = inputs(shape, dtype, seed, mask, poison)
    q, k, v = (t.requires_grad_() for t in (q, k, v))
    out = policy.cross_attention(q, k, v, **kw, **extra)
    grads = torch.autograd.grad(out, (q, k, v), do)
    want = ref.attention_gradients(q.detach(), k.detach(), v.detach(), do, visible, extra.get("scale"))
    with torch.no_grad():
        plain = policy.cross_attention(q, k, v, **kw, **extra)
    assert torch.equal(plain, out.detach()), "the result without gradients differs"
    ref.assert_close(out, want[0], ref.FORWARD[dtype], "out")
    hidden = ~visible[:, :, None, None].expand_as(k)
    for name, g, w in zip(("dq", "dk", "dv"), grads, want[1:]):
        ref.assert_close(g, w, ref.GRADIENT[dtype], name)
        if name != "dq":
            assert not g[hidden].any(), f"{name} of invisible keys must be 0"
    return out, grads


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("mask", ["none", "mask", "lengths", "both"])
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_output_and_gradients(shape, mask, dtype):
    if shape[2] == 1 and mask == "none":
        # one key: the softmax is constant and dq, dk vanish; what is left of them is rounding
        q, k, v, do, kw, _ = inputs(shape, dtype)
        out = policy.cross_attention(q, k, v)
        ref.assert_close(out, v.double().expand_as(out), ref.ONE_ROUNDING[dtype], "out")
        return
    if shape[2] == 1:
        pytest.skip("one key that may be invisible is in test_no_visible_key")
    check(shape, dtype, mask)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", [(3, 4, 200, 4, 2, 64), (3, 40, 200, 4, 2, 64), (3, 100, 77, 2, 1, 128)], ids=str)
def test_what_invisible_keys_hold_does_not_matter(shape, dtype):
    check(shape, dtype, "both", poison=True)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("mask", ["none", "both"])
@pytest.mark.parametrize("dim", [24, 64, 96])
@pytest.mark.parametrize("lk", [1, 2, 15, 16, 17, 31, 32, 33])
@pytest.mark.parametrize("lq", [1, 13, 30])  # 2, 26 and 60 rows to a key head: the three row tiles
def test_short_key_lists(lq, lk, dim, mask, dtype):
    q, k, v, do, kw, visible = inputs((3, lq, lk, 4, 2, dim), dtype, seed=lk, mask=mask, poison=True)
    out = policy.cross_attention(q, k, v, **kw)
    want = ref.attention_gradients(q, k, v, do, visible)[0]
    ref.assert_close(out, want, ref.FORWARD[dtype], "out")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("lq", [1, 16, 17, 100])
def test_no_visible_key(lq, dtype):
    q, k, v, do, _, _ = inputs((2, lq, 70, 4, 2, 64), dtype)
    k[0], v[0] = math.nan, math.inf
    do[0] = math.nan  # the gradient of a constant is 0 whatever comes in
    q, k, v = (t.requires_grad_() for t in (q, k, v))
    lengths = torch.tensor([0, 70], dtype=torch.int32, device=DEV)
    out = policy.cross_attention(q, k, v, key_lengths=lengths)
    dq, dk, dv = torch.autograd.grad(out, (q, k, v), do)
    for t in (out, dq, dk, dv):
        assert not t[0].any() and torch.isfinite(t[1]).all() and t[1].any()


@pytest.mark.parametrize("dtype", DTYPES)
def test_lengths_outside_the_keys_are_clamped(dtype):
    q, k, v, _, _, _ = inputs((3, 2, 40, 2, 2, 32), dtype)
    got = policy.cross_attention(q, k, v, key_lengths=torch.tensor([-5, 1000, 40], dtype=torch.int32, device=DEV))
    full = policy.cross_attention(q, k, v)
    assert not got[0].any() and torch.equal(got[1:], full[1:])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("b,lq,lk", [(0, 3, 5), (2, 0, 5), (2, 3, 0)])
def test_empty(b, lq, lk, dtype):
    q = torch.randn(b, lq, 4, 32, device=DEV).to(dtype).requires_grad_()
    k = torch.randn(b, lk, 2, 32, device=DEV).to(dtype).requires_grad_()
    v = torch.randn(b, lk, 2, 32, device=DEV).to(dtype).requires_grad_()
    out = policy.cross_attention(q, k, v)
    grads = torch.autograd.grad(out, (q, k, v), torch.ones_like(out))
    assert out.shape == q.shape and not out.any()
    for g, t in zip(grads, (q, k, v)):
        assert g.shape == t.shape and not g.any()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("lq", [2, 50])
def test_strided_views_give_the_same_bits(lq, dtype):
    """Slices of one projection's output, another axis order, rows that are not aligned, a broadcast batch."""
    b, lk, h, hk, d = 3, 90, 4, 2, 64
    gen = torch.Generator(device=DEV).manual_seed(3)
    fused = torch.randn(b, lk, 2 * hk * d, generator=gen, device=DEV).to(dtype)
    k, v = fused[..., : hk * d].view(b, lk, hk, d), fused[..., hk * d:].view(b, lk, hk, d)
    q = torch.randn(b, h, lq, d, generator=gen, device=DEV).to(dtype).transpose(1, 2)
    do = torch.randn(b, h, lq, d, generator=gen, device=DEV).to(dtype).transpose(1, 2)
    mask = (torch.rand(lk, b, generator=gen, device=DEV) > 0.2).t()

    def run(q, k, v, do, mask):
        q, k, v = (t.detach().requires_grad_() for t in (q, k, v))
        out = policy.cross_attention(q, k, v, key_mask=mask)
        return (out.detach(), *torch.autograd.grad(out, (q, k, v), do))

    want = run(*(t.contiguous() for t in (q, k, v, do, mask)))
    for x, y in zip(run(q, k, v, do, mask), want):
        assert torch.equal(x, y)
    odd = lambda t: torch.nn.functional.pad(t, (1, 2))[..., 1:-2]  # noqa: E731
    for x, y in zip(run(odd(q), odd(k), odd(v), odd(do), mask), want):
        assert torch.equal(x, y)
    shared = k[:1].expand(b, -1, -1, -1)
    for x, y in zip(run(q, shared, v, do[:1].expand_as(do), mask), run(q, shared.contiguous(), v, do[:1].expand_as(do).contiguous(), mask)):
        assert torch.equal(x, y)


def test_broadcast_inputs_and_outputs_through_autograd():
    q = torch.randn(1, 3, 2, 32, device=DEV, requires_grad=True)
    k, v = torch.randn(4, 50, 2, 32, device=DEV), torch.randn(4, 50, 2, 32, device=DEV)
    out = policy.cross_attention(q.expand(4, -1, -1, -1), k, v)
    (dq,) = torch.autograd.grad(out.sum(), q)  # the incoming gradient has stride 0 everywhere
    _, each, _, _ = ref.attention_gradients(q.detach().expand(4, -1, -1, -1), k, v, torch.ones_like(out))
    ref.assert_close(dq, each.sum(0, keepdim=True), 2 * ref.GRADIENT[torch.float32], "dq")


def test_gradient_against_differences():
    """d/dh of <out, do> along a direction, by central differences of the 64-bit restatement: their own error is
    h^2 times the third derivative, about 1e-8 here."""
    q, k, v, do, kw, visible = inputs((2, 19, 75, 4, 2, 40), torch.float32, 5, "mask")
    leaves = [t.requires_grad_() for t in (q, k, v)]
    out = policy.cross_attention(*leaves, **kw)
    grads = torch.autograd.grad(out, leaves, do)
    h = 1e-4
    for i, g in enumerate(grads):
        direction = torch.randn_like(g, dtype=torch.float64)

        def value(sign, i=i, direction=direction):
            x = [t.detach().double() for t in leaves]
            x[i] = x[i] + sign * h * direction
            return float((ref.attention(*x, visible) * do.double()).sum())

        want = (value(1) - value(-1)) / (2 * h)
        got = float((g.double() * direction).sum())
        size = float(g.double().norm() * direction.norm()) / math.sqrt(g.numel())
        assert abs(got - want) <= 16 * ref.GRADIENT[torch.float32] * max(abs(want), size), (i, got, want)


@pytest.mark.parametrize("dtype", DTYPES)
def test_large_scores_and_scale(dtype):
    """Scores of hundreds: a softmax without its maximum would overflow.  The scores' own rounding is 2^-24 of
    them in 32 bits, so float32 is compared at that times the largest score."""
    shape = (2, 20, 150, 2, 2, 64)
    q, k, v, do, _, visible = inputs(shape, dtype, 7)
    q = q * 20
    out = policy.cross_attention(q, k, v, scale=0.5)
    want = ref.attention(q, k, v, visible, 0.5)
    top = float((torch.einsum("blhd,bkhd->bhlk", q.double(), k.double()) * 0.5).abs().max())
    assert top > 200
    ref.assert_close(out, want, ref.FORWARD[dtype] + top * 2.0 ** -21, "out")


@pytest.mark.parametrize("dtype", DTYPES)
def test_non_finite_visible_values_propagate(dtype):
    q, k, v, _, _, _ = inputs((2, 4, 60, 2, 2, 32), dtype)
    v[0, 7, 1, 3] = math.nan
    k[1, 9, 0, 0] = math.nan
    out = policy.cross_attention(q, k, v)
    assert torch.isnan(out[0, :, 1, 3]).all() and int(torch.isnan(out[0]).sum()) == 4
    assert torch.isnan(out[1, :, 0]).all() and torch.isfinite(out[1, :, 1]).all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", [(2, 3, 6000, 4, 2, 64), (1, 200, 40, 2, 1, 64)], ids=str)
def test_bits_do_not_depend_on_timing(shape, dtype):
    first = check(shape, dtype, "mask")
    for _ in range(3):
        again = check(shape, dtype, "mask")
        assert torch.equal(first[0], again[0]) and all(torch.equal(x, y) for x, y in zip(first[1], again[1]))


def test_offsets_past_32_bits():
    """Two batches more than 2^31 elements apart, and keys 2^27 elements apart."""
    n = 2 ** 31 + 2 ** 12
    big = torch.zeros(n + 40 * 64 * 2, dtype=torch.bfloat16, device=DEV)
    k = big.as_strided((2, 40, 1, 64), (n, 64, 64, 1))
    v = big.as_strided((2, 40, 1, 64), (n, 64, 64, 1), 40 * 64)
    far = big.as_strided((1, 17, 1, 64), (0, 2 ** 27, 64, 1), 128)
    for t in (k, v, far):
        t.copy_(torch.randn(t.shape, device=DEV))
    q = torch.randn(2, 3, 2, 64, device=DEV).bfloat16()
    for kk, vv, qq in ((k, v, q), (far, far, q[:1])):
        want = ref.attention(qq, kk.contiguous(), vv.contiguous())
        ref.assert_close(policy.cross_attention(qq, kk, vv), want, ref.FORWARD[torch.bfloat16], "out")
    qg = q.clone().requires_grad_()
    kg, vg = k.detach().requires_grad_(), v.detach().requires_grad_()
    out = policy.cross_attention(qg, kg, vg)
    grads = torch.autograd.grad(out, (qg, kg, vg), torch.ones_like(out))
    want = ref.attention_gradients(q, k.contiguous(), v.contiguous(), torch.ones_like(out))
    for name, g, w in zip(("dq", "dk", "dv"), grads, want[1:]):
        ref.assert_close(g, w, ref.GRADIENT[torch.bfloat16], name)


def test_runs_on_the_callers_stream():
    q, k, v, do, _, visible = inputs((4, 20, 500, 4, 2, 64), torch.bfloat16)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        torch.cuda._sleep(20_000_000)  # q is written late on this stream only
        late = (q.float() * 1.0).to(q.dtype)
        leaves = [t.requires_grad_() for t in (late, k, v)]
        out = policy.cross_attention(*leaves)
        grads = torch.autograd.grad(out, leaves, do)
    torch.cuda.current_stream().wait_stream(side)
    want = ref.attention_gradients(q, k.detach(), v.detach(), do, visible)
    ref.assert_close(out, want[0], ref.FORWARD[torch.bfloat16], "out")
    for g, w in zip(grads, want[1:]):
        ref.assert_close(g, w, ref.GRADIENT[torch.bfloat16], "gradient")


def test_captured_in_a_graph():
    q, k, v, _, kw, visible = inputs((2, 1, 3000, 4, 2, 64), torch.bfloat16, mask="mask")
    policy.cross_attention(q, k, v, **kw)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = policy.cross_attention(q, k, v, **kw)
    q.copy_(torch.randn_like(q))
    graph.replay()
    ref.assert_close(out, ref.attention(q, k, v, visible), ref.FORWARD[torch.bfloat16], "out")


def test_gradients_of_gradients_are_an_error():
    q, k, v, do, _, _ = inputs((1, 2, 9, 2, 2, 32), torch.float32)
    q.requires_grad_()
    out = policy.cross_attention(q, k, v)
    (dq,) = torch.autograd.grad(out, q, do, create_graph=True)
    with pytest.raises(RuntimeError, match="once only"):
        dq.sum().backward()


def test_refusals():
    q, k, v, _, _, _ = inputs((2, 3, 10, 4, 2, 32), torch.float32)
    bad = [
        ((q.cpu(), k, v), {}, "q must be a CUDA tensor"),
        ((q, k.cpu(), v), {}, "k must be a CUDA tensor"),
        ((q[0], k, v), {}, "q must have shape"),
        ((q.half(), k.half(), v.half()), {}, "q must be float32 or bfloat16"),
        ((q, k.bfloat16(), v), {}, "k must have the type of q"),
        ((q, k, v[:, :5]), {}, "k and v must have the same shape"),
        ((q[:1], k, v), {}, "the batch and the dim of q"),
        ((q[:, :, :3], k, v), {}, "positive multiple"),
        ((q[..., :12], k[..., :12], v[..., :12]), {}, "multiple of 8"),
        ((torch.randn(1, 1, 1, 136, device=DEV),) * 3, {}, "from 8 to 128"),
        ((q, k, v), {"scale": 0.0}, "scale must be positive"),
        ((q, k, v), {"scale": math.inf}, "scale must be positive"),
        ((q, k, v), {"key_mask": torch.ones(2, 10, device=DEV)}, "key_mask must be a bool"),
        ((q, k, v), {"key_mask": torch.ones(2, 9, dtype=torch.bool, device=DEV)}, "key_mask must be a bool"),
        ((q, k, v), {"key_mask": torch.ones(2, 10, dtype=torch.bool)}, "on the device of q"),
        ((q, k, v), {"key_lengths": torch.ones(2, dtype=torch.int64, device=DEV)}, "key_lengths must be an int32"),
        ((q, k, v), {"key_lengths": torch.ones(3, dtype=torch.int32, device=DEV)}, "key_lengths must be an int32"),
    ]
    for args, kw, text in bad:
        with pytest.raises(RuntimeError, match=text):
            policy.cross_attention(*args, **kw)
