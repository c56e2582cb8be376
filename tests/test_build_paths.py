"""Where the build looks for ROCm."""

import importlib.util
import os

import pytest

REPO = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture()
def build():
    path = os.path.join(REPO, "mlx-primitives_amd", "build.py")
    spec = importlib.util.spec_from_file_location("mpx_build_paths", path)
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    return mod


@pytest.mark.parametrize("name", ["ROCM_HOME", "ROCM_PATH"])
def test_rocm_of_the_environment(build, monkeypatch, tmp_path, name):
    for var in ("ROCM_HOME", "ROCM_PATH", "HIPCC"):
        monkeypatch.delenv(var, raising=False)
    assert build.rocm_home() == "/opt/rocm"
    (tmp_path / "bin").mkdir()
    (tmp_path / "bin" / "hipcc").write_text("")
    monkeypatch.setenv(name, str(tmp_path))
    assert build.hipcc() == str(tmp_path / "bin" / "hipcc")
    assert f"-isystem{tmp_path}/include" in build.host_command("x.so")
    monkeypatch.setenv(name, str(tmp_path / "none"))  # (no such folder)
    assert build.rocm_home() == "/opt/rocm"
