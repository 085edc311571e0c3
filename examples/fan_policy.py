"""A policy that reads ray fans, acting and learning: the tracer and the policy operators together.

    python -m examples.fan_policy --actors 64 --steps 10

Each step casts every actor's fan with its observation (``tracer.cast_fan_observe``), cuts the
[3, azimuth, elevation] planes into patches, and lets a few latent queries attend to them:
``policy.qk_norm_rotary`` turns queries and keys by their directions around the fan,
``policy.cross_attention`` reads the patches that hold a valid ray.  Acting is the forward pass
without gradients; learning fits the actions that steer towards the most open direction, with the
gradients clipped by ``policy.clip_grad_norm`` as PPO's are.
"""

from __future__ import annotations

import argparse
import math

import torch
from torch import nn

from navi_b200 import fan as fan_tables
from navi_b200 import policy, scenes, tracer, workloads


class FanPolicy(nn.Module):
    """Latent queries over the patches of an observation [actors, 3, azimuth, elevation]."""

    def __init__(self, azimuth_bins: int, elevation_bins: int, *, patch: int = 4, dim: int = 32, heads: int = 4,
                 kv_heads: int = 2, latents: int = 8, actions: int = 2, dtype: torch.dtype = torch.float32,
                 device: torch.device | str = "cuda") -> None:
        super().__init__()
        if azimuth_bins % patch or elevation_bins % patch:
            raise ValueError("the patch must divide both sides of the fan")
        self.patch, self.dim, self.heads, self.kv_heads, self.dtype = patch, dim, heads, kv_heads, dtype
        self.grid = azimuth_bins // patch, elevation_bins // patch
        width = heads * dim
        kw = {"device": device, "dtype": torch.float32}
        self.embed = nn.Linear(3 * patch * patch, width, **kw)
        self.latents = nn.Parameter(torch.randn(latents, width, **kw) / math.sqrt(width))
        self.to_q = nn.Linear(width, heads * dim, bias=False, **kw)
        self.to_kv = nn.Linear(width, 2 * kv_heads * dim, bias=False, **kw)
        self.q_weight = nn.Parameter(torch.ones(dim, **kw))
        self.k_weight = nn.Parameter(torch.ones(dim, **kw))
        self.head = nn.Linear(latents * width, actions, **kw)
        # the patches' directions, and for the latents directions around the horizon
        table = policy.fan_rotary_table(*self.grid, dim // 16 * 16, device)
        az = torch.arange(latents, device=device) * self.grid[0] // latents
        self.register_buffer("table", table)
        self.register_buffer("latent_positions", (az * self.grid[1] + self.grid[1] // 2).to(torch.int32))

    def forward(self, observation: torch.Tensor) -> torch.Tensor:
        a, (n_az, n_el), p = observation.shape[0], self.grid, self.patch
        planes = torch.nan_to_num(observation, posinf=1.0, neginf=0.0).view(a, 3, n_az, p, n_el, p)
        tokens = self.embed(planes.permute(0, 2, 4, 1, 3, 5).reshape(a, n_az * n_el, -1))
        seen = (planes[:, 2].amax((2, 4)) > 0).reshape(a, n_az * n_el)  # patches with a valid ray
        latents = self.latents.expand(a, -1, -1)
        q = self.to_q(latents).to(self.dtype).view(a, -1, self.heads, self.dim)
        k, v = self.to_kv(tokens).to(self.dtype).view(a, n_az * n_el, 2, self.kv_heads, self.dim).unbind(2)
        q, k = policy.qk_norm_rotary(q, k, self.q_weight, self.k_weight, q_table=self.table, k_table=self.table,
                                     q_positions=self.latent_positions.expand(a, -1).contiguous())
        read = policy.cross_attention(q, k, v, key_mask=seen)
        return self.head((latents + read.flatten(2).float()).flatten(1))


def open_direction(distances: torch.Tensor, fan: torch.Tensor, horizon: float) -> torch.Tensor:
    """The mean horizontal direction of each actor's fan, weighted by how far its rays go: [actors, 2]."""
    far = torch.nan_to_num(distances, posinf=horizon).clamp(0.0, horizon)
    return nn.functional.normalize((far[..., None] * fan[None, :, ::2]).mean(1), dim=-1)


def train(actors: int = 64, steps: int = 10, *, dtype: torch.dtype = torch.float32, max_norm: float = 0.5, rate: float = 0.1,
          seed: int = 0, device: torch.device | str = "cuda") -> list[tuple[float, float]]:
    """(loss, gradient norm) of each step on the 10 m room of the smallest benchmark scene."""
    dev = torch.device(device, torch.cuda.current_device()) if torch.device(device).index is None else torch.device(device)
    torch.manual_seed(seed)
    cfg = scenes.CONFIGS[1]
    cs = workloads.compiled_scene(1)
    az, el = cfg.azimuth_bins, cfg.elevation_bins
    sset = tracer.SceneSet([tracer.NodePool.from_words(cs.words, dev)], [cs.bbox_min], [cs.bbox_max], [cs.hit_epsilon])
    fan = torch.from_numpy(fan_tables.build_spherical_ray_directions(az, el)).to(dev)
    distances = torch.empty(actors * az * el, device=dev)
    semantics = torch.empty(actors * az * el, dtype=torch.int32, device=dev)
    observation = torch.empty((actors, 3, az, el), device=dev)
    stats = torch.empty((actors, 5), device=dev)
    model = FanPolicy(az, el, dtype=dtype, device=dev)
    parameters = list(model.parameters())
    low, high = (torch.tensor(x, device=dev) for x in (cs.bbox_min, cs.bbox_max))
    position = low + (high - low) * (0.2 + 0.6 * torch.rand(actors, 3, device=dev))
    yaw = torch.rand(actors, device=dev) * (2 * math.pi)
    history = []
    for _ in range(steps):
        tracer.cast_fan_observe(sset, tracer.make_poses(position, yaw), fan, az, el, distances, semantics, observation, stats,
                                max_steps=cfg.max_steps, max_distance=cfg.max_distance)
        with torch.no_grad():  # acting: turn towards where the policy points
            action = model(observation)
            yaw = yaw + 0.1 * torch.atan2(action[:, 0], -action[:, 1])
        target = open_direction(distances.view(actors, -1), fan, cfg.max_distance)
        loss = (model(observation) - target).square().mean()
        grads = torch.autograd.grad(loss, parameters)
        norm = policy.clip_grad_norm(grads, max_norm)
        with torch.no_grad():
            for weight, g in zip(parameters, grads):
                weight -= rate * g
        history.append((loss.detach(), norm))
    return [(float(loss), float(norm)) for loss, norm in history]


def main() -> None:
    parser = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    parser.add_argument("--actors", type=int, default=64)
    parser.add_argument("--steps", type=int, default=10)
    parser.add_argument("--dtype", choices=["float32", "bfloat16"], default="float32")
    args = parser.parse_args()
    for i, (loss, norm) in enumerate(train(args.actors, args.steps, dtype=getattr(torch, args.dtype))):
        print(f"step {i}: loss {loss:.4f}, gradient norm {norm:.4f}")


if __name__ == "__main__":
    main()
