"""Gradient clipping refuses lists whose result would depend on the order in which blocks run."""

from __future__ import annotations

import pytest
import torch

from navi_b200 import _native, policy

F32, BF16 = _native.POLICY_F32, _native.POLICY_BF16


def status(*entries):
    """(code, message) of a call that no device takes: entries are (grad, out, count, type)."""
    lib = _native.policy_lib()
    grads = (_native.PolicyGrad * len(entries))(*(_native.PolicyGrad(*e, 0) for e in entries))
    return lib.policy_clip_grad_norm(grads, len(entries), 1.0, 16, -1, None, None), lib.policy_last_error().decode()


@pytest.mark.parametrize("entries", [
    [(1024, 4096, 64, F32), (4096, 1024, 64, F32)],                             # swapped
    [(1024, 1024, 64, F32), (1024, 1024, 64, F32)],                             # the same one twice
    [(1024, 1024, 64, F32), (1276, 1276, 64, F32)],                             # one value in common
    [(1024, 1024, 64, F32), (1278, 1278, 64, BF16)],                            # two bytes in common
    [(1024, 4096, 64, F32), (2048, 4348, 64, F32)],                             # outputs that overlap
    [(1024, 1028, 64, F32)],                                                    # an output shifted over its gradient
    [(1024, 1020, 64, F32)],
    [(4096, 8192, 64, F32), (1024, 4128, 4, F32)],                              # an output inside another's gradient
    [(1024, 1024, 64, F32), (1028, 4096, 4, F32)],                              # a gradient inside another's output
    [(1024, 1024, 64, F32), (1024, 4096, 64, F32)],                             # read by one, changed by the other
], ids=str)
def test_shared_memory_is_refused(entries):
    for order in (entries, entries[::-1]):
        code, text = status(*order)
        assert code == -1 and "must not share memory" in text


@pytest.mark.parametrize("entries", [
    [(1024, 1024, 64, F32), (1280, 1280, 64, F32)],                             # neighbours
    [(1024, 1024, 64, F32), (1280, 1280, 64, BF16), (1408, 1408, 1, F32)],
    [(1024, 4096, 64, F32), (1280, 4352, 64, F32)],
    [(1024, 4096, 64, F32), (1024, 8192, 64, F32)],                             # read twice, written apart
    [(1024, 1024, 64, F32), (1024, 1024, 0, F32), (0, 0, 0, F32)],              # nothing to write
], ids=str)
def test_separate_memory_is_taken(entries):
    code, text = status(*entries)
    assert code == -1 and "device must be a CUDA device index" in text


@pytest.mark.gpu
def test_tensors_that_share_memory():
    base = torch.arange(4096.0, device="cuda")
    a, b = base[:2048], base[2048:]
    other = torch.zeros(2048, device="cuda")
    for grads, out in (([a, b], [b, a]), ([base[:3000], base[2000:]], None), ([a], [base[1:2049]]), ([a, b], [other, a]),
                       ([a, b], [base[1024:3072], other])):
        with pytest.raises(RuntimeError, match="must not share memory"):
            policy.clip_grad_norm(grads, 1.0, out=out)
    assert torch.equal(base, torch.arange(4096.0, device="cuda")) and not other.any()
    want = float(base.double().norm())
    assert abs(float(policy.clip_grad_norm([a, b], 1.0, out=[a, other])) - want) <= 2.0 ** -21 * want
    assert torch.equal(b, torch.arange(2048.0, 4096.0, device="cuda")) and abs(float(torch.cat([a, other]).double().norm()) - 1) <= 2.0 ** -19
