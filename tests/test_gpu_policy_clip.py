"""Global gradient norm and clipping against 64-bit sums.

Tolerances: the norm is a sum of squares, each rounded twice in 32 bits (2^-23), a few of them added in 32
bits per thread and the rest in 64: 2^-22 of the sum, 2^-23 of the norm, plus its own rounding: 2^-21 with
room.  A clipped value is the product of a value and a factor of that error: 2^-20 in float32, one more
rounding of 2^-8 in bfloat16; below the type's normal numbers half of its smallest one.
"""

from __future__ import annotations

import math

import pytest
import torch

from navi_b200 import policy

pytestmark = pytest.mark.gpu

DEV = torch.device("cuda", 0)
VALUE = {torch.float32: 2.0 ** -20, torch.bfloat16: 2.0 ** -8 + 2.0 ** -20}
SMALLEST = {torch.float32: 2.0 ** -149, torch.bfloat16: 2.0 ** -133}

LISTS = {
    "one value": [((), torch.float32)],
    "one bfloat16": [((1,), torch.bfloat16)],
    "a network": [((64, 192), torch.float32), ((64,), torch.float32), ((3, 5, 7), torch.bfloat16), ((0,), torch.float32),
                  ((4096,), torch.float32), ((4097,), torch.bfloat16), ((1000, 333), torch.bfloat16), ((4095,), torch.float32)],
    "large": [((5_000_011,), torch.float32), ((3_000_007,), torch.bfloat16)],
    "many": [((17 + i,), torch.float32 if i % 3 else torch.bfloat16) for i in range(1300)],
}


def make(shapes, seed=0):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    return [torch.randn(s, generator=gen, device=DEV).to(t) for s, t in shapes]


def norm64(grads):
    return math.sqrt(sum(float(g.double().square().sum()) for g in grads))


def check(grads, before, norm, max_norm):
    want = norm64(before)
    assert norm.shape == () and norm.dtype == torch.float32
    assert abs(float(norm) - want) <= 2.0 ** -21 * want
    c = min(1.0, max_norm / (want + 1e-6))
    for g, b in zip(grads, before):
        w = b.double() * c
        assert ((g.double() - w).abs() <= VALUE[g.dtype] * w.abs() + 0.5 * SMALLEST[g.dtype]).all()


@pytest.mark.parametrize("share", [0.01, 0.999, 2.0])
@pytest.mark.parametrize("name", LISTS)
def test_in_place(name, share):
    grads = make(LISTS[name])
    before = [g.clone() for g in grads]
    limit = share * norm64(before)
    versions = [g._version for g in grads]
    check(grads, before, policy.clip_grad_norm(grads, limit), limit)
    assert all(g._version > v for g, v in zip(grads, versions))
    if share > 1:
        assert all(torch.equal(g, b) for g, b in zip(grads, before))


@pytest.mark.parametrize("name", LISTS)
def test_into_other_tensors(name):
    grads = make(LISTS[name])
    before = [g.clone() for g in grads]
    out = [torch.full_like(g, 7.0) for g in grads]
    limit = 0.3 * norm64(before)
    check(out, before, policy.clip_grad_norm(iter(grads), limit, out=out), limit)
    assert all(torch.equal(g, b) for g, b in zip(grads, before))
    limit = 3 * norm64(before)
    policy.clip_grad_norm(grads, limit, out=out)
    assert all(torch.equal(g, b) for g, b in zip(out, before))


def test_unaligned_views_and_other_orders():
    base = make([((20_000,), torch.float32), ((20_001,), torch.bfloat16), ((60, 50, 40), torch.float32)])
    grads = [base[0][1:9000], base[0][9001:], base[1][3:], base[2].permute(2, 0, 1)]
    before = [g.clone(memory_format=torch.preserve_format) for g in grads]
    edge = base[0][0].clone(), base[0][9000].clone(), base[1][:3].clone()
    check(grads, before, policy.clip_grad_norm(grads, 1.0), 1.0)
    assert torch.equal(edge[0], base[0][0]) and torch.equal(edge[1], base[0][9000]) and torch.equal(edge[2], base[1][:3])


def test_values_whose_squares_leave_the_type():
    """bfloat16 values near 1e-25 and 1e18: the squares of the first underflow to 0 in 32 bits and are far below the
    bound, the norm of the second stays finite."""
    grads = [torch.full((5000,), 1e18, device=DEV), torch.full((100,), 1e-25, device=DEV).bfloat16()]
    before = [g.clone() for g in grads]
    check(grads, before, policy.clip_grad_norm(grads, 1.0), 1.0)


def test_norms_that_are_not_finite():
    g = torch.ones(10_000, device=DEV)
    g[77] = math.inf
    norm = policy.clip_grad_norm([g], 1.0)
    assert math.isinf(float(norm)) and torch.isnan(g[77]) and not g[:77].any() and not g[78:].any()
    g = torch.ones(10_000, device=DEV)
    g[5] = math.nan
    assert math.isnan(float(policy.clip_grad_norm([g], 1.0))) and torch.isnan(g).all()


def test_zero_gradients_and_zero_bound():
    g = torch.zeros(1000, device=DEV)
    assert float(policy.clip_grad_norm([g], 1.0)) == 0 and not g.any()
    g = torch.ones(1000, device=DEV)
    policy.clip_grad_norm([g], 0.0)
    assert not g.any()
    assert float(policy.clip_grad_norm([torch.empty(0, device=DEV)], 1.0)) == 0


def test_bits_do_not_depend_on_timing():
    grads = make(LISTS["large"] + LISTS["a network"])
    runs = []
    for _ in range(4):
        out = [torch.empty_like(g) for g in grads]
        runs.append((policy.clip_grad_norm(grads, 1.0, out=out), out))
    for norm, out in runs[1:]:
        assert torch.equal(norm, runs[0][0]) and all(torch.equal(x, y) for x, y in zip(out, runs[0][1]))


def test_runs_on_the_callers_stream():
    g = torch.zeros(300_000, device=DEV)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        torch.cuda._sleep(20_000_000)
        g.fill_(2.0)
        norm = policy.clip_grad_norm([g], 1.0)
    torch.cuda.current_stream().wait_stream(side)
    want = 2 * math.sqrt(300_000)
    assert abs(float(norm) - want) <= 2.0 ** -21 * want
    assert abs(float(g[0]) - 2 / want) <= 2.0 ** -20 * 2 / want


def test_refusals():
    g = torch.ones(10, 10, device=DEV)
    for args, kw, text in [
        (([], 1.0), {}, "must not be empty"),
        (([g], -1.0), {}, "max_norm must not be negative"),
        (([g], math.nan), {}, "max_norm must not be negative"),
        (([g.cpu()], 1.0), {}, "CUDA tensors"),
        (([g, g.cpu()[:0]], 1.0), {}, "one device"),
        (([g.half()], 1.0), {}, "float32 or bfloat16"),
        (([g[:, ::2]], 1.0), {}, "dense"),
        (([g, g], 1.0), {}, "must not share memory"),
        (([g], 1.0), {"out": []}, "one tensor for every gradient"),
        (([g], 1.0), {"out": [g.bfloat16()]}, "out must have the shapes"),
        (([g], 1.0), {"out": [g.t()]}, "out must have the shapes"),
    ]:
        with pytest.raises(RuntimeError, match=text):
            policy.clip_grad_norm(*args, **kw)
