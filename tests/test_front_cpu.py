"""beacon_front is a shortcut, not a condition: the library builds without torch and a C++ compiler, and the
operators work where beacon_front cannot be loaded."""
import os
import subprocess

import pytest

from beacon_b200 import _lib


def _plan(*targets):
    return subprocess.run(["make", "-n", "-B", "-C", _lib.CSRC, *targets], check=True, capture_output=True, text=True).stdout


def test_plain_make_needs_nvcc_alone():
    plan = _plan()
    assert "libbeacon_cuda.so" in plan and "front.cpp" not in plan and "torch" not in plan
    assert "front.cpp" in _plan("front")


@pytest.mark.parametrize("broken", ["missing", "not a module", "another binding"])
def test_operators_without_the_front(monkeypatch, tmp_path, broken):
    import torch
    from beacon_b200 import errors, ops
    path = tmp_path / "beacon_front.so"
    if broken == "not a module":
        path.write_bytes(b"no ELF file")
    monkeypatch.setattr(_lib, "FRONT_PATH", str(path))
    if broken == "another binding":
        class Old:
            def bind(self, *addresses):
                raise ValueError("bind: four addresses")
        monkeypatch.setattr(_lib, "_load_front", lambda: Old().bind(1, 2))
    monkeypatch.setattr(_lib, "_front", None)
    x, g = torch.zeros(4, 8 * 64, dtype=torch.bfloat16), torch.ones(64, dtype=torch.bfloat16)
    with pytest.warns(RuntimeWarning, match="beacon_front.so is not used"):
        with pytest.raises(errors.InvalidLaunchConfig, match="CUDA"):
            ops.qk_norm_rope_fwd(x, g, g, None, 1, 4, 4, 2)
    with pytest.raises(errors.InvalidLaunchConfig, match="is not 5 rows"):
        ops.qk_norm_rope_fwd(x, g, g, None, 1, 5, 4, 2)


def test_the_front_is_built_here():
    assert os.path.exists(_lib.FRONT_PATH)
    assert not isinstance(_lib.front(), _lib._NoFront)
