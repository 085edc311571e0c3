"""A wait inside an attention kernel that runs out reaches the caller as an error, and the context stays usable."""

from __future__ import annotations

import ctypes

import pytest
import torch

from navi_b200 import _native, policy

pytestmark = pytest.mark.gpu

DEV = torch.device("cuda", 0)


def wait(arrive_ns: int, limit_ns: int, word: int) -> bool:
    """Whether the kernels' bounded wait sees an arrival after arrive_ns (negative: none comes)."""
    lib = ctypes.CDLL(str(_native.LIB_DIR / "libnavi_probe.so"))
    lib.navi_check_wait.argtypes = [ctypes.c_longlong, ctypes.c_ulonglong, ctypes.c_void_p, ctypes.c_void_p, ctypes.c_void_p]
    result = torch.full((1,), -1, dtype=torch.int32, device=DEV)
    assert lib.navi_check_wait(arrive_ns, limit_ns, result.data_ptr(), word, torch.cuda.current_stream().cuda_stream) == 0
    torch.cuda.synchronize()
    return bool(result.item())


def test_a_wait_that_runs_out_is_an_error_of_the_next_call():
    torch.cuda.init()
    address = _native.policy_lib().policy_stall_word()
    word = ctypes.cast(address, ctypes.POINTER(ctypes.c_int32))
    assert address and word[0] == 0
    q, k = torch.randn(1, 100, 1, 64, device=DEV).bfloat16(), torch.randn(1, 50, 1, 64, device=DEV).bfloat16()
    want = policy.cross_attention(q, k, k)
    assert wait(1_000_000, 500_000_000, address) and word[0] == 0
    assert not wait(-1, 100_000_000, address) and word[0] == 1
    with pytest.raises(RuntimeError, match="ran out of time"):
        policy.cross_attention(q, k, k)
    assert word[0] == 0 and torch.equal(policy.cross_attention(q, k, k), want)
    assert not wait(-1, 1_000_000, address)
    q.requires_grad_()
    word[0] = 0
    out = policy.cross_attention(q, k, k)
    assert not wait(-1, 1_000_000, address)
    with pytest.raises(RuntimeError, match="ran out of time"):
        torch.autograd.grad(out, q, out)
    torch.autograd.grad(policy.cross_attention(q, k, k), q, out)


def test_polls_last_as_long_as_the_limit_takes_them_to():
    """The limit counts polls, so that the time for which a context is paused is none of it."""
    torch.cuda.init()
    address = _native.policy_lib().policy_stall_word()
    begin, end = (torch.cuda.Event(enable_timing=True) for _ in range(2))
    assert not wait(-1, 1_000_000, address)
    begin.record()
    assert not wait(-1, 200_000_000, address)
    end.record()
    end.synchronize()
    ctypes.cast(address, ctypes.POINTER(ctypes.c_int32))[0] = 0
    assert 100 < begin.elapsed_time(end) < 400
