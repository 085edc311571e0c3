"""libnavi_policy.so exports what include/policy.h declares and refuses bad arguments before any CUDA call."""

from __future__ import annotations

import ctypes
import re
from pathlib import Path

import pytest
import torch

from navi_b200 import _native, policy

ROOT = Path(__file__).resolve().parents[1]


def _declared() -> list[str]:
    text = (ROOT / "include" / "policy.h").read_text()
    return re.findall(r"^POLICY_API\s+[\w\s\*]+?\b(policy_\w+)\s*\(", text, flags=re.M)


def test_library_exports_every_declared_symbol():
    names = _declared()
    assert set(names) == set(_native.POLICY_SIGNATURES)
    lib = _native.policy_lib()
    for name in names:
        assert hasattr(lib, name), name
    assert lib.policy_version() == 1


@pytest.mark.parametrize("struct,name", [(_native.PolicyAttention, "policy_attention"), (_native.PolicyNormSide, "policy_norm_side"),
                                         (_native.PolicyQkNorm, "policy_qk_norm"), (_native.PolicyGrad, "policy_grad")])
def test_structures_have_the_headers_fields(struct, name):
    text = (ROOT / "include" / "policy.h").read_text()
    body = re.search(r"typedef struct %s \{(.*?)\} %s;" % (name, name), text, flags=re.S).group(1)
    body = re.sub(r"/\*.*?\*/", "", body, flags=re.S)
    fields = []
    for line in body.split(";"):
        m = re.match(r"\s*(?:const\s+)?\w+[\s\*]+(.*)", line.strip(), flags=re.S)
        if m:
            fields += [re.sub(r"[\s\*]|\[.*?\]", "", x) for x in m.group(1).split(",")]
    assert fields == [f for f, _ in struct._fields_]


def _attention(**kw) -> _native.PolicyAttention:
    a = _native.PolicyAttention(dtype=0, batch=1, lq=1, lk=1, heads=1, kv_heads=1, dim=32, scale=1.0)
    for n, v in kw.items():
        setattr(a, n, v)
    return a


@pytest.mark.parametrize("change,text", [
    ({"dtype": 5}, "dtype"), ({"batch": -1}, "negative"), ({"lk": -1}, "negative"), ({"heads": 3, "kv_heads": 2}, "multiple of kv_heads"),
    ({"kv_heads": 0}, "multiple of kv_heads"), ({"dim": 12}, "multiple of 8"), ({"dim": 136}, "multiple of 8"), ({"dim": 0}, "multiple of 8"),
    ({"scale": 0.0}, "scale"), ({"scale": float("nan")}, "scale"), ({"lk": 2 ** 31}, "below 2"), ({"lq": 2 ** 31}, "below 2"),
    ({"batch": 2 ** 31}, "below 2"), ({}, "q must not be null"), ({"q": 8}, "q must have 16-byte"), ({"q": 16}, "out must not be null"),
    ({"q": 16, "q_strides": (ctypes.c_int64 * 3)(0, 2, 0), "out": 16}, "q must have 16-byte"), ({"q": 16, "out": 16}, "k must not be null"),
    ({"q": 16, "out": 16, "k": 16}, "v must not be null"),
])
def test_attention_refuses(change, text):
    lib = _native.policy_lib()
    assert lib.policy_cross_attention(ctypes.byref(_attention(**change)), None) == -1
    assert text in lib.policy_last_error().decode()


@pytest.mark.parametrize("change,text", [
    ({}, "dout must not be null"), ({"dout": 16}, "stats must not be null"), ({"dout": 16, "stats": 16}, "dq must not be null"),
    ({"dout": 16, "stats": 16, "dq": 16}, "dk must not be null"), ({"dout": 16, "stats": 16, "dq": 16, "dk": 16}, "dv must not be null"),
])
def test_attention_backward_refuses(change, text):
    lib = _native.policy_lib()
    a = _attention(q=16, k=16, v=16, out=16, **change)
    assert lib.policy_cross_attention_backward(ctypes.byref(a), None) == -1
    assert text in lib.policy_last_error().decode()


def test_null_arguments():
    lib = _native.policy_lib()
    assert lib.policy_cross_attention(None, None) == -1
    assert lib.policy_cross_attention_backward(None, None) == -1
    assert lib.policy_cross_attention_workspace_bytes(None, 0) == 0
    assert lib.policy_qk_norm_rotary(None, None) == -1
    assert lib.policy_qk_norm_rotary_backward(None, None) == -1
    assert lib.policy_qk_norm_workspace_bytes(None) == 0
    assert lib.policy_clip_grad_norm(None, 1, 1.0, None, 0, None, None) == -1
    assert b"grads must not be null" in lib.policy_last_error()


@pytest.mark.parametrize("change,text", [
    ({"dtype": 5}, "dtype"), ({"dim": 12}, "dim"), ({"dim": 264}, "dim"), ({"rotary": 8}, "rotary"), ({"rotary": 48}, "rotary"),
    ({"eps": -1.0}, "eps"), ({"eps": float("nan")}, "eps"), ({"batch": -1}, "batch"), ({}, "x must not be null"),
])
def test_norm_refuses(change, text):
    lib = _native.policy_lib()
    a = _native.PolicyQkNorm(dtype=0, batch=1, dim=32, rotary=0, eps=1e-6)
    for s in a.side:
        s.tokens, s.heads = 1, 1
    for n, v in change.items():
        setattr(a, n, v)
    assert lib.policy_qk_norm_rotary(ctypes.byref(a), None) == -1
    assert text in lib.policy_last_error().decode()


def test_clip_refuses():
    lib = _native.policy_lib()
    for entry, text in [((16, 16, 4, 7), "dtype"), ((0, 0, 4, 0), "must not be null"), ((17, 16, 4, 0), "aligned"),
                        ((16, 16, 2 ** 41, 0), "count")]:
        g = (_native.PolicyGrad * 1)(_native.PolicyGrad(*entry, 0))
        assert lib.policy_clip_grad_norm(g, 1, 1.0, 16, 0, None, None) == -1
        assert text in lib.policy_last_error().decode()
    g = (_native.PolicyGrad * 1)(_native.PolicyGrad(16, 16, 4, 0, 0))
    assert lib.policy_clip_grad_norm(g, 1, -1.0, 16, 0, None, None) == -1
    assert lib.policy_clip_grad_norm(g, 1, 1.0, None, 0, None, None) == -1


def test_cpu_tensors_are_refused():
    t = torch.zeros(1, 1, 1, 32)
    with pytest.raises(RuntimeError, match="CPU tensors are not supported"):
        policy.cross_attention(t, t, t)
    with pytest.raises(RuntimeError, match="CPU tensors are not supported"):
        policy.qk_norm_rotary(t, t)
    with pytest.raises(RuntimeError, match="CPU tensors are not supported"):
        policy.clip_grad_norm([t], 1.0)


def test_fan_table_on_the_host():
    table = policy.fan_rotary_table(4, 3, 16, "cpu")
    assert table.shape == (12, 2, 8)
    # token 3 is azimuth 1 (a quarter turn), elevation +pi/2; pairs 0-3 azimuth harmonics, 4-7 elevation
    quarter = torch.tensor([1.0, 2.0, 3.0, 4.0], dtype=torch.float64) * torch.pi / 2
    assert torch.allclose(table[3, 0].double(), torch.cat([quarter.cos(), quarter.cos()]), atol=1e-7)
    assert torch.allclose(table[3, 1].double(), torch.cat([quarter.sin(), quarter.sin()]), atol=1e-7)
    with pytest.raises(RuntimeError, match="multiple of 16"):
        policy.fan_rotary_table(4, 3, 24, "cpu")
