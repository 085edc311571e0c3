"""The policy operators that run beside the tracer, and what they are measured on.

- ``attend``: cross attention of an actor's queries to the tokens of its ray fan
  (``policy.cross_attention``), forward alone or with the gradients of q, k and v;
- ``norm``: per-head RMS norm of queries and keys with the rotation by the token's
  angles in the same pass (``policy.qk_norm_rotary``), forward alone or with gradients;
- ``clip``: the global norm of a list of gradients and their clipping
  (``policy.clip_grad_norm``).

``run`` computes a case in its plain form (elementary torch operations in 32 bits) or,
where ``own`` is true, by the calls a user of navi_b200 makes.
"""

from __future__ import annotations

import math
import random

import torch

own = False

DTYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16}


# --- cases ---------------------------------------------------------------------


def _attend(name, batch, lq, lk, heads, kv_heads, dim, dtype, train, mask):
    return {"name": name, "op": "attend", "batch": batch, "lq": lq, "lk": lk, "heads": heads, "kv_heads": kv_heads,
            "dim": dim, "dtype": dtype, "train": train, "mask": mask}


def _norm(name, batch, lq, lk, heads, kv_heads, dim, rotary, dtype, train, positions):
    return {"name": name, "op": "norm", "batch": batch, "lq": lq, "lk": lk, "heads": heads, "kv_heads": kv_heads,
            "dim": dim, "rotary": rotary, "dtype": dtype, "train": train, "positions": positions}


def _clip(name, tensors, elements, dtype, shapes):
    return {"name": name, "op": "clip", "tensors": tensors, "elements": elements, "dtype": dtype, "shapes": shapes}


def listed():
    return [
        # acting with config 1's 4 actors: one query each, a 64 x 16 fan in 4 x 4 patches
        _attend("attend act 4 actors", 4, 1, 64, 4, 4, 32, "float32", False, "lengths"),
        # acting with config 2's 64 actors, one query each over every ray of a 256 x 48 fan, rays without a
        # valid distance masked, four query heads to a key head
        _attend("attend act every ray", 64, 1, 12288, 8, 2, 64, "bfloat16", False, "mask"),
        # an update over 1,024 observations: 16 latent queries, 8 x 8 patches of a 256 x 48 fan
        _attend("attend update patches", 1024, 16, 192, 8, 8, 64, "bfloat16", True, "mask"),
        # an update in 32 bits with odd sizes everywhere and shared key heads
        _attend("attend update odd fp32", 37, 9, 385, 6, 3, 40, "float32", True, "lengths"),
        # a decoder that predicts every ray of a 256 x 48 fan from the 4 x 4 patches of another
        _attend("attend decode rays", 16, 12288, 768, 8, 8, 128, "bfloat16", False, "none"),
        # the same kind of decoder trained on 64 x 64 output cells
        _attend("attend update decoder", 8, 4096, 768, 8, 4, 64, "bfloat16", True, "mask"),
        # the queries and keys of the first case
        _norm("norm act 4 actors", 4, 1, 64, 4, 4, 32, 32, "float32", False, False),
        # the queries and keys of the second
        _norm("norm act every ray", 64, 1, 12288, 8, 2, 64, 64, "bfloat16", False, False),
        # the queries and keys of the update over patches, a quarter of each head without rotation
        _norm("norm update patches", 1024, 16, 192, 8, 8, 64, 48, "bfloat16", True, True),
        # odd sizes in 32 bits
        _norm("norm update odd fp32", 37, 101, 385, 6, 3, 40, 16, "float32", True, False),
        # a small policy: matrices and vectors, 1.2 M values
        _clip("clip small policy", 40, 1_200_000, "float32", 1),
        # a policy with a large encoder: gradients in both types, 150 M values
        _clip("clip large policy", 60, 150_000_000, "mixed", 2),
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.99))))))


def draw(rng):
    op = rng.choice(["attend", "attend", "norm", "clip"])
    if op == "clip":
        tensors = rng.randint(1, 60)
        return {k: v for k, v in _clip("", tensors, _log(rng, max(1000, tensors), 150_000_000),
                                       rng.choice(["float32", "bfloat16", "mixed"]), rng.randrange(1 << 20)).items() if k != "name"}
    while True:
        kv_heads, group = rng.choice([1, 2, 3, 4, 8]), rng.choice([1, 1, 2, 4])
        dim = rng.choice([16, 32, 40, 64, 80, 96, 128])
        dtype, train = rng.choice(["float32", "bfloat16"]), rng.random() < 0.5
        batch = _log(rng, 1, 1024)
        lk = _log(rng, 1, 12288)
        lq = _log(rng, 1, 12288) if rng.random() < 0.5 else _log(rng, 1, 32)
        if op == "norm":
            case = _norm("", batch, lq, lk, kv_heads * group, kv_heads, dim, rng.choice([0, 16, dim // 16 * 16]),
                         dtype, train, rng.random() < 0.5)
        else:
            case = _attend("", batch, lq, lk, kv_heads * group, kv_heads, dim, dtype, train,
                           rng.choice(["none", "mask", "lengths"]))
        w = work(case)
        if w["bytes"] > 1.1e9 or w["flops"] > (6e11 if not train else 1e11):
            continue
        if op == "attend" and batch * kv_heads * group * lq * lk > (1.2e9 if not train else 4e8):
            continue
        return {k: v for k, v in case.items() if k != "name"}


def _shapes(case):
    """The gradients' shapes and types: matrices of a network and their vectors, odd sizes among them."""
    rng = random.Random(case["shapes"])
    n = case["tensors"]
    weight = [rng.choice([1.0, 1.0, 0.01]) * rng.uniform(0.2, 1.0) for _ in range(n)]
    total = sum(weight)
    sizes = [max(1, int(case["elements"] * w / total)) for w in weight]
    kinds = [DTYPES[case["dtype"]] if case["dtype"] != "mixed" else rng.choice([torch.float32, torch.bfloat16]) for _ in range(n)]
    return sizes, kinds


def work(case):
    if case["op"] == "clip":
        sizes, kinds = _shapes(case)
        return {"bytes": sum(2 * n * (4 if t == torch.float32 else 2) for n, t in zip(sizes, kinds)) + 4,
                "flops": 3 * sum(sizes)}
    e = 4 if case["dtype"] == "float32" else 2
    q = case["batch"] * case["lq"] * case["heads"] * case["dim"]
    k = case["batch"] * case["lk"] * case["kv_heads"] * case["dim"]
    if case["op"] == "norm":
        table = case["lq"] + case["lk"]
        small = 4 * table * case["rotary"] + 8 * case["dim"]
        if case["positions"]:
            small += 4 * case["batch"] * table
        # forward: x in, y out; with gradients also dy in and dx out (x is read once)
        return {"bytes": (q + k) * e * (4 if case["train"] else 2) + small + (8 * case["dim"] if case["train"] else 0),
                "flops": (q + k) * (24 if case["train"] else 8)}
    product = 2 * case["batch"] * case["heads"] * case["lq"] * case["lk"] * case["dim"]
    mask = {"none": 0, "mask": case["batch"] * case["lk"], "lengths": 4 * case["batch"]}[case["mask"]]
    if case["train"]:  # q, k, v, do in; o, dq, dk, dv out; two products forward, five backward
        return {"bytes": (4 * q + 4 * k) * e + mask, "flops": 7 * product}
    return {"bytes": (2 * q + 2 * k) * e + mask, "flops": 2 * product}


# --- inputs --------------------------------------------------------------------


def prepare(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev).manual_seed(seed)
    randn = lambda *shape: torch.randn(*shape, generator=gen, device=dev)  # noqa: E731
    state = dict(case)
    if case["op"] == "clip":
        sizes, kinds = _shapes(case)
        state["grads"] = [(randn(n) * 1e-3).to(t) for n, t in zip(sizes, kinds)]
        state["out"] = [torch.empty_like(g) for g in state["grads"]]
        # a bound that the gradients pass: PPO clips at 0.5, and the norm of these is about 1e-3 sqrt(n)
        state["max_norm"] = min(0.5, 2.5e-4 * math.sqrt(sum(sizes)))
        return state
    b, lq, lk, d = case["batch"], case["lq"], case["lk"], case["dim"]
    t, train = DTYPES[case["dtype"]], case["train"]
    state["q"] = randn(b, lq, case["heads"], d).to(t).requires_grad_(train)
    state["k"] = randn(b, lk, case["kv_heads"], d).to(t).requires_grad_(train)
    if case["op"] == "norm":
        state["q_weight"] = (1 + 0.1 * randn(d)).requires_grad_(train)
        state["k_weight"] = (1 + 0.1 * randn(d)).requires_grad_(train)
        for x, n in (("q", lq), ("k", lk)):
            # a token's angle times the harmonics of a full turn, cosines then sines
            turn = torch.arange(n, device=dev, dtype=torch.float64)[:, None] * (2 * math.pi / n)
            angle = turn * torch.arange(1, case["rotary"] // 2 + 1, device=dev, dtype=torch.float64)
            state[x + "_table"] = torch.stack([angle.cos(), angle.sin()], 1).float() if case["rotary"] else None
            state[x + "_positions"] = (torch.randint(0, n, (b, n), generator=gen, device=dev, dtype=torch.int32)
                                       if case["positions"] and case["rotary"] else None)
        if train:
            state["dq"], state["dk"] = randn(b, lq, case["heads"], d).to(t), randn(b, lk, case["kv_heads"], d).to(t)
        return state
    state["v"] = randn(b, lk, case["kv_heads"], d).to(t).requires_grad_(train)
    state["key_mask"] = state["key_lengths"] = None
    if case["mask"] == "mask":  # rays without a valid distance; an actor outside its scene has none at all
        none = torch.rand(b, 1, generator=gen, device=dev) < 1 / 16
        state["key_mask"] = (torch.rand(b, lk, generator=gen, device=dev) > 0.1) & ~none
    elif case["mask"] == "lengths":
        state["key_lengths"] = torch.randint(0, lk + 1, (b,), generator=gen, device=dev, dtype=torch.int32)
    if train:
        state["do"] = randn(b, lq, case["heads"], d).to(t)
    return state


# --- plain forms ---------------------------------------------------------------


def _visible(s):
    """[B, 1, 1, Lk], true where a key may be seen; None where all may."""
    if s["key_mask"] is not None:
        return s["key_mask"][:, None, None, :]
    if s["key_lengths"] is not None:
        at = torch.arange(s["lk"], device=s["k"].device)
        return (at[None, :] < s["key_lengths"][:, None])[:, None, None, :]
    return None


def _plain_attend(s):
    b, lq, lk, h, hk, d = (s[x] for x in ("batch", "lq", "lk", "heads", "kv_heads", "dim"))
    g = h // hk
    q = s["q"].float().view(b, lq, hk, g, d).permute(0, 2, 3, 1, 4).reshape(b, hk, g * lq, d)
    k = s["k"].float().permute(0, 2, 3, 1)
    v = s["v"].float().permute(0, 2, 1, 3)
    score = q @ k * (1 / math.sqrt(d))
    visible = _visible(s)
    if visible is not None:
        score = score.masked_fill(~visible, -math.inf)
    top = score.detach().amax(-1, keepdim=True)
    top = torch.where(top == -math.inf, 0.0, top)
    p = (score - top).exp()
    total = p.sum(-1, keepdim=True)
    p = p / torch.where(total == 0, 1.0, total)
    out = (p @ v).view(b, hk, g, lq, d).permute(0, 3, 1, 2, 4).reshape(b, lq, h, d)
    return out.to(s["q"].dtype)


def _plain_norm(x, weight, table, positions, eps=1e-6):
    f = x.float()
    f = f * (f.square().mean(-1, keepdim=True) + eps).rsqrt() * weight
    if table is not None:
        rows = table[positions.long()] if positions is not None else table[None]
        cos, sin = rows[..., 0, :].unsqueeze(2), rows[..., 1, :].unsqueeze(2)
        n = cos.shape[-1]
        a, c = f[..., :n], f[..., n:2 * n]
        f = torch.cat([a * cos - c * sin, c * cos + a * sin, f[..., 2 * n:]], -1)
    return f.to(x.dtype)


def _plain_clip(s):
    norm = torch.stack([g.float().square().sum() for g in s["grads"]]).sum().sqrt()
    scale = (s["max_norm"] / (norm + 1e-6)).clamp(max=1.0)
    return {"norm": norm, "grads": [(g.float() * scale).to(g.dtype) for g in s["grads"]]}


def run(state):
    s = state
    if s["op"] == "clip":
        if not own:
            return _plain_clip(s)
        from navi_b200 import policy

        norm = policy.clip_grad_norm(s["grads"], s["max_norm"], out=s["out"])
        return {"norm": norm, "grads": s["out"]}
    if s["op"] == "norm":
        if own:
            from navi_b200 import policy

            q, k = policy.qk_norm_rotary(s["q"], s["k"], s["q_weight"], s["k_weight"], q_table=s["q_table"],
                                         k_table=s["k_table"], q_positions=s["q_positions"], k_positions=s["k_positions"])
        else:
            q = _plain_norm(s["q"], s["q_weight"], s["q_table"], s["q_positions"])
            k = _plain_norm(s["k"], s["k_weight"], s["k_table"], s["k_positions"])
        if not s["train"]:
            return {"q": q, "k": k}
        grads = torch.autograd.grad((q, k), (s["q"], s["k"], s["q_weight"], s["k_weight"]), (s["dq"], s["dk"]))
        return {"q": q.detach(), "k": k.detach(), **dict(zip(("dq", "dk", "dq_weight", "dk_weight"), grads))}
    if own:
        from navi_b200 import policy

        out = policy.cross_attention(s["q"], s["k"], s["v"], key_mask=s["key_mask"], key_lengths=s["key_lengths"])
    else:
        out = _plain_attend(s)
    if not s["train"]:
        return out
    dq, dk, dv = torch.autograd.grad(out, (s["q"], s["k"], s["v"]), s["do"])
    return {"out": out.detach(), "dq": dq, "dk": dk, "dv": dv}


# --- 64 bits -------------------------------------------------------------------


def _exact_attend(s):
    """One (actor, key head) after another would be slow: one actor after another, by the formulas of softmax
    and of its gradient."""
    h, hk, d = s["heads"], s["kv_heads"], s["dim"]
    g, scale = h // hk, 1 / math.sqrt(d)
    outs = {"out": [], "dq": [], "dk": [], "dv": []}
    for i in range(s["batch"]):
        q = s["q"][i].detach().double().transpose(0, 1).reshape(hk, g, s["lq"], d)
        k = s["k"][i].detach().double().transpose(0, 1)[:, None]
        v = s["v"][i].detach().double().transpose(0, 1)[:, None]
        e = torch.matmul(q, k.transpose(-1, -2)).mul_(scale)
        seen = torch.ones(s["lk"], dtype=torch.bool, device=q.device)
        if s["key_mask"] is not None:
            seen = s["key_mask"][i]
        elif s["key_lengths"] is not None:
            seen = torch.arange(s["lk"], device=q.device) < s["key_lengths"][i]
        if bool(seen.any()):
            e[..., ~seen] = -math.inf
            p = torch.softmax(e, -1)
        else:
            p = torch.zeros_like(e)
        o = torch.matmul(p, v)
        outs["out"].append(o.reshape(h, s["lq"], d).transpose(0, 1))
        if s["train"]:
            do = s["do"][i].double().transpose(0, 1).reshape(hk, g, s["lq"], d)
            ds = p * (torch.matmul(do, v.transpose(-1, -2)) - (do * o).sum(-1, keepdim=True)) * scale
            outs["dv"].append(torch.matmul(p.transpose(-1, -2), do).sum(1).transpose(0, 1))
            outs["dq"].append(torch.matmul(ds, k).reshape(h, s["lq"], d).transpose(0, 1))
            outs["dk"].append(torch.matmul(ds.transpose(-1, -2), q).sum(1).transpose(0, 1))
    outs = {n: torch.stack(x) for n, x in outs.items() if x}
    return outs if s["train"] else outs["out"]


def _exact_norm(x, weight, table, positions, dy):
    """y = R(w x / rms(x)) and, for dy, dx and dw: R is a rotation, so its gradient is the rotation back."""
    x, w = x.detach().double(), weight.detach().double()
    r = 1 / torch.sqrt((x * x).sum(-1, keepdim=True) / x.shape[-1] + 1e-6)

    def turn(u, sign):
        if table is None:
            return u
        z = torch.complex(table[:, 0].double(), sign * table[:, 1].double())
        z = z[positions.long()] if positions is not None else z.unsqueeze(0)
        n = z.shape[-1]
        t = torch.complex(u[..., :n].contiguous(), u[..., n:2 * n].contiguous()) * z.unsqueeze(2)
        return torch.cat((t.real, t.imag, u[..., 2 * n:]), -1)

    y = turn(x * r * w, 1.0)
    if dy is None:
        return y, None, None
    du = turn(dy.double(), -1.0)
    inner = (du * w * x).sum(-1, keepdim=True) / x.shape[-1]
    return y, r * (du * w) - r ** 3 * x * inner, (du * x * r).sum((0, 1, 2))


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "clip":
        total = sum(float((g.double() ** 2).sum()) for g in s["grads"])
        norm = math.sqrt(total)
        c = min(1.0, s["max_norm"] / (norm + 1e-6))
        return {"norm": torch.tensor(norm, dtype=torch.float64), "grads": [g.double() * c for g in s["grads"]]}
    if case["op"] == "attend":
        return _exact_attend(s)
    q, dq, dqw = _exact_norm(s["q"], s["q_weight"], s["q_table"], s["q_positions"], s.get("dq"))
    k, dk, dkw = _exact_norm(s["k"], s["k_weight"], s["k_table"], s["k_positions"], s.get("dk"))
    if not case["train"]:
        return {"q": q, "k": k}
    return {"q": q, "k": k, "dq": dq, "dk": dk, "dq_weight": dqw, "dk_weight": dkw}
