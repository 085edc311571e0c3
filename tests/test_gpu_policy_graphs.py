"""The policy operators in CUDA graphs: replays read what their inputs hold then."""

from __future__ import annotations

import subprocess
import sys
from pathlib import Path

import pytest
import torch

from navi_b200 import policy
from tests import policy_ref as ref

pytestmark = pytest.mark.gpu

DEV = torch.device("cuda", 0)


def capture(call):
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        call()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        result = call()
    return graph, result


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("lq,lk", [(4, 900), (25, 300), (200, 300)])
def test_attention_and_its_gradients(lq, lk, dtype):
    shapes = [(2, lq, 4, 64), (2, lk, 2, 64), (2, lk, 2, 64)]
    leaves = [torch.randn(s, device=DEV).to(dtype).requires_grad_() for s in shapes]
    do = torch.randn(shapes[0], device=DEV).to(dtype)
    mask = torch.rand(2, lk, device=DEV) > 0.3

    def call():
        out = policy.cross_attention(*leaves, key_mask=mask)
        return (out.detach(), *torch.autograd.grad(out, leaves, do))

    graph, got = capture(call)
    with torch.no_grad():
        for t in (*leaves, do):
            t.copy_(torch.randn(t.shape, device=DEV))
        mask.copy_(torch.rand(2, lk, device=DEV) > 0.6)
    for _ in range(2):
        graph.replay()
    want = ref.attention_gradients(*(t.detach() for t in leaves), do, mask)
    ref.assert_close(got[0], want[0], ref.FORWARD[dtype], "out")
    for name, x, y in zip(("dq", "dk", "dv"), got[1:], want[1:]):
        ref.assert_close(x, y, ref.GRADIENT[dtype], name)


def test_norms_and_their_gradients():
    q, k, w = (torch.randn(s, device=DEV).requires_grad_() for s in ((2, 5, 4, 64), (2, 90, 2, 64), (64,)))
    table = policy.fan_rotary_table(18, 5, 32, DEV)

    def call():
        y = policy.qk_norm_rotary(q, k, w, w, q_table=table, k_table=table)
        return (y[1].detach(), *torch.autograd.grad(y, (q, k, w), y))

    graph, got = capture(call)
    with torch.no_grad():
        for t in (q, k, w):
            t.copy_(torch.randn(t.shape, device=DEV))
    graph.replay()
    want = ref.norm_rotary(k.detach(), w.detach(), table)
    ref.assert_close(got[0], want, ref.ONE_ROUNDING[torch.float32], "k")
    for x, y in zip(got[1:], torch.autograd.grad((ref.norm_rotary(q, w, table), ref.norm_rotary(k, w, table)), (q, k, w),
                                                 (ref.norm_rotary(q, w, table).detach(), want))):
        ref.assert_close(x, y, 4 * ref.ONE_ROUNDING[torch.float32], "gradient")  # the incoming gradient is a result as well


@pytest.mark.parametrize("n", [1, 40, 700])
def test_clipping(n):
    grads = [torch.randn(1 + 37 * i % 5000, device=DEV) for i in range(n)]
    out = [torch.empty_like(g) for g in grads]
    graph, norm = capture(lambda: policy.clip_grad_norm(grads, 0.25, out=out))
    for g in grads:
        g.copy_(torch.randn_like(g))
    for _ in range(3):
        graph.replay()
    want = float(torch.cat(grads).double().norm())
    assert abs(float(norm) - want) <= 2.0 ** -21 * want
    c = min(1.0, 0.25 / (want + 1e-6))
    for g, o in zip(grads, out):
        assert ((o.double() - g.double() * c).abs() <= 2.0 ** -20 * (g.double() * c).abs()).all()


def test_the_first_call_of_a_process_may_be_captured():
    code = """
import torch
from navi_b200 import policy
q, k = torch.randn(1, 200, 1, 64, device="cuda").bfloat16(), torch.randn(1, 300, 1, 64, device="cuda").bfloat16()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    out = policy.cross_attention(q, k, k)
graph.replay()
assert torch.equal(out, policy.cross_attention(q, k, k)) and out.any()
"""
    run = subprocess.run([sys.executable, "-c", code], cwd=Path(__file__).resolve().parents[1], capture_output=True, text=True, timeout=300)
    assert run.returncode == 0, run.stderr[-2000:]
