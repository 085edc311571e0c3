"""navi_policy_torch.so belongs to one release of torch: it is rebuilt for another, and not loaded beside it."""

from __future__ import annotations

import pytest
import torch

from navi_b200 import _native, build


class Built(Exception):
    pass


@pytest.fixture
def no_compiler(monkeypatch):
    def run(cmd, *args, **kwargs):
        raise Built(cmd)

    monkeypatch.setattr(build, "_run", run)
    # newer than every source
    newest = max(p.stat().st_mtime for p in (build.CSRC / "policy_torch.cpp", build.INCLUDE / "policy.h"))
    assert _native.POLICY_TORCH_PATH.stat().st_mtime >= newest, "build first"


def test_the_module_is_built_for_the_installed_torch(no_compiler):
    assert _native.policy_torch_fits()
    assert build.build_policy_torch() == _native.POLICY_TORCH_PATH


@pytest.mark.parametrize("version", ["0.0.0", torch.__version__ + "1", torch.__version__[:-1]])
def test_another_torch_is_a_reason_to_build(no_compiler, monkeypatch, version):
    monkeypatch.setattr(torch, "__version__", version)
    with pytest.raises(Built) as built:
        build.build_policy_torch()
    assert f'-DNAVI_TORCH_VERSION="{version}"' in built.value.args[0]


def test_a_module_for_another_torch_is_not_loaded(monkeypatch):
    monkeypatch.setattr(_native, "_policy_torch", None)
    monkeypatch.setattr(torch, "__version__", "0.0.0")
    with pytest.raises(RuntimeError, match="not built for torch 0.0.0"):
        _native.policy_torch()
