"""The build on hosts that cannot build the operators' calls on torch tensors: without torch, with a torch that is not HIP's, without Python's or
HIP's headers, without a host compiler.  The libraries, the plugin and the native tools need none of that and have to come out all the same."""
from pathlib import Path

import pytest

from hugectr_backend_amd import build as hb


def _tree(root):
    for f in ("torch/lib/libc10_hip.so", "torch/include/c10/hip/HIPStream.h", "py/Python.h", "rocm/hip/hip_runtime_api.h"):
        (root / f).parent.mkdir(parents=True, exist_ok=True)
        (root / f).write_text("")
    return root / "torch", root / "py", root / "rocm"


def test_what_the_module_needs(tmp_path):
    home, py, rocm = _tree(tmp_path)
    assert hb.torch_module_lacks(home, py, rocm, "sh") is None
    assert hb.torch_module_lacks(None, py, rocm, "sh") == "torch"
    assert hb.torch_module_lacks(home, py, rocm, "no-such-compiler") == "no-such-compiler"
    for f in (home / "lib/libc10_hip.so", home / "include/c10/hip/HIPStream.h", py / "Python.h", rocm / "hip/hip_runtime_api.h"):
        f.unlink()
        assert hb.torch_module_lacks(home, py, rocm, "sh") == str(f)
        f.write_text("")


@pytest.fixture
def dry(monkeypatch, tmp_path):
    """build() that compiles nothing and writes what it would have built under tmp_path"""
    def made(path):
        Path(path).parent.mkdir(parents=True, exist_ok=True)
        Path(path).write_text("")
        return Path(path)
    monkeypatch.setattr(hb, "LIB", tmp_path / "lib")
    monkeypatch.setattr(hb, "OBJ", tmp_path / "obj")
    (tmp_path / "lib").mkdir()
    (tmp_path / "obj").mkdir()
    monkeypatch.setattr(hb, "_compile", lambda rel, force: made(tmp_path / "obj" / rel.replace("/", "__")))
    monkeypatch.setattr(hb, "_link", lambda out, objs, extra=(): made(out))
    monkeypatch.setattr(hb, "_run", lambda cmd: made(cmd[cmd.index("-o") + 1]))
    return tmp_path


def test_another_torch_does_not_stop_the_build(dry, monkeypatch, capsys):
    home, _, _ = _tree(dry)
    (home / "lib/libc10_hip.so").unlink()
    monkeypatch.setattr(hb, "_torch_home", lambda: home)
    outs = hb.build(force=True)
    assert "torch_calls" not in outs and "libc10_hip" in capsys.readouterr().err
    for k in ("hps_amd", "triton_hps", "mock_core", "triton_abi_bench"):
        assert Path(outs[k]).exists(), k


def test_a_module_that_does_not_compile_comes_last(dry, monkeypatch):
    """Where it should build and does not that is an error, but everything else is there by then."""
    monkeypatch.setattr(hb, "torch_module_lacks", lambda *a: None)

    def no(*a):
        raise RuntimeError("compiler says no")
    monkeypatch.setattr(hb, "_torch_module", no)
    with pytest.raises(RuntimeError, match="compiler says no"):
        hb.build(force=True)
    assert (dry / "lib" / "triton_abi_bench.bin").exists()


def test_the_entry_check_takes_a_build_without_the_module(dry, monkeypatch):
    import __graft_entry__ as entry
    import subprocess
    monkeypatch.setattr(hb, "_torch_home", lambda: None)
    monkeypatch.setattr(subprocess, "run", lambda *a, **k: None)
    entry.build()


def test_the_headers_follow_the_compiler(monkeypatch, tmp_path):
    (tmp_path / "bin").mkdir()
    (tmp_path / "include" / "hip").mkdir(parents=True)
    monkeypatch.setattr(hb, "HIPCC", str(tmp_path / "bin" / "hipcc"))
    assert hb._rocm_include() == tmp_path / "include"
