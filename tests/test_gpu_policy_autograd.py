"""What the policy operators cannot differentiate or hand to a trace is an error, not a result that has lost its inputs."""

from __future__ import annotations

import pytest
import torch
import torch.autograd.forward_ad as forward_ad

from navi_b200 import policy

pytestmark = pytest.mark.gpu

DEV = torch.device("cuda", 0)


def values(*shape):
    return torch.randn(*shape, device=DEV)


@pytest.mark.parametrize("requires_grad", [False, True])
@pytest.mark.parametrize("which", [0, 1, 2])
def test_a_tangent_of_attention_is_refused(which, requires_grad):
    args = [values(2, 3, 4, 32), values(2, 9, 2, 32), values(2, 9, 2, 32)]
    args[which].requires_grad_(requires_grad)
    with forward_ad.dual_level():
        args[which] = forward_ad.make_dual(args[which], torch.ones_like(args[which]))
        for call in (args, [t[:1] for t in args]):  # a view carries it too
            with pytest.raises(RuntimeError, match="forward-mode"):
                policy.cross_attention(*call)
        args[which] = forward_ad.unpack_dual(args[which]).primal
        assert policy.cross_attention(*args).shape == (2, 3, 4, 32)


@pytest.mark.parametrize("which", [0, 1, 2, 3])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_a_tangent_of_the_norms_is_refused(which, dtype):
    args = [t.to(dtype) for t in (values(2, 3, 4, 32), values(2, 9, 2, 32), values(32), values(32))]
    with forward_ad.dual_level():
        args[which] = forward_ad.make_dual(args[which], torch.ones_like(args[which]))
        with pytest.raises(RuntimeError, match="forward-mode"):
            policy.qk_norm_rotary(*args)


def test_a_tangent_of_a_clipped_gradient_is_refused():
    g, out = values(50), values(50)
    before = g.clone()
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(g, torch.ones_like(g))
        for grads, outs in (([dual], None), ([before], [dual]), ([dual], [out])):
            with pytest.raises(RuntimeError, match="forward-mode"):
                policy.clip_grad_norm(grads, 0.1, out=outs)
    assert torch.equal(g, before)


def test_tracing_is_refused():
    """A trace would keep the result of the inputs that it was made with."""
    q, k = values(2, 3, 4, 32), values(2, 9, 2, 32)
    for call in (lambda x: policy.cross_attention(x, k, k), lambda x: policy.qk_norm_rotary(x, k)[0], lambda x: policy.clip_grad_norm([x], 1.0)):
        with pytest.raises(RuntimeError, match="cannot be traced"):
            torch.jit.trace(call, q)
        call(q)
