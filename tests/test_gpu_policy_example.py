"""The example policy: casts, attention, norms and clipping together."""

from __future__ import annotations

import math

import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = torch.device("cuda", 0)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_acts_and_learns_on_its_fans(dtype):
    from examples.fan_policy import train

    history = train(actors=16, steps=8, dtype=dtype)
    assert len(history) == 8
    assert all(math.isfinite(loss) and math.isfinite(norm) and norm > 0 for loss, norm in history)


def test_the_network_is_its_formula():
    """The forward pass and all gradients against the same network in 64 bits.  The linear layers around the
    operators run in float32 (a few hundred terms, 2^-24 each in quadrature), the operators within
    16 * 2^-21: 1e-4 leaves room for both through five layers."""
    from examples.fan_policy import FanPolicy
    from tests import policy_ref as ref

    torch.manual_seed(1)
    model = FanPolicy(64, 16, device=DEV)
    observation = torch.rand(5, 3, 64, 16, device=DEV)
    observation[:, 2] = (torch.rand(5, 64, 16, device=DEV) > 0.7).float()
    observation[0, 2, :32] = 0.0
    parameters = dict(model.named_parameters())
    wide = {n: p.detach().double().requires_grad_() for n, p in parameters.items()}
    a, (n_az, n_el), p = 5, model.grid, model.patch
    planes = observation.double().view(a, 3, n_az, p, n_el, p)
    tokens = planes.permute(0, 2, 4, 1, 3, 5).reshape(a, n_az * n_el, -1) @ wide["embed.weight"].t() + wide["embed.bias"]
    seen = (planes[:, 2].amax((2, 4)) > 0).reshape(a, -1)
    latents = wide["latents"].expand(a, -1, -1)
    q = (latents @ wide["to_q.weight"].t()).view(a, -1, model.heads, model.dim)
    k, v = (tokens @ wide["to_kv.weight"].t()).view(a, n_az * n_el, 2, model.kv_heads, model.dim).unbind(2)
    q = ref.norm_rotary(q, wide["q_weight"], model.table, model.latent_positions.expand(a, -1))
    k = ref.norm_rotary(k, wide["k_weight"], model.table)
    read = ref.attention(q, k, v, seen)
    want = (latents + read.flatten(2)).flatten(1) @ wide["head.weight"].t() + wide["head.bias"]
    action = model(observation)
    ref.assert_close(action, want.detach(), 1e-4, "action")
    got = torch.autograd.grad(action.square().sum(), list(parameters.values()))
    expected = torch.autograd.grad(want.square().sum(), list(wide.values()))
    for name, g, w in zip(parameters, got, expected):
        ref.assert_close(g, w, 1e-4, name)


def test_an_observation_without_a_valid_ray():
    """An actor whose rays are all invalid reads nothing: its action is that of the latents alone, and finite."""
    from examples.fan_policy import FanPolicy

    torch.manual_seed(0)
    model = FanPolicy(64, 16, device=DEV)
    observation = torch.rand(3, 3, 64, 16, device=DEV)
    observation[:, 2] = 1.0
    observation[1, 0] = math.nan
    observation[1, 2] = 0.0
    action = model(observation)
    alone = model.head(model.latents.flatten())
    assert torch.isfinite(action).all()
    assert torch.allclose(action[1], alone, rtol=1e-5, atol=1e-6) and not torch.allclose(action[0], alone, atol=1e-3)
    grads = torch.autograd.grad(action.square().sum(), list(model.parameters()))
    assert all(torch.isfinite(g).all() for g in grads)
