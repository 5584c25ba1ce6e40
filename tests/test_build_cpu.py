"""build.py with stand-ins for the compilers."""
import os
import subprocess
import sys

import pytest
import torch

import build


@pytest.fixture
def fake(tmp_path, monkeypatch):
    """Compilers that write their output file, or fail where `fail` names them;
    what they were called for is in `calls`."""
    log = tmp_path / "calls"

    class Fake:
        fail = ()

        def calls(self):
            return log.read_text().split() if log.exists() else []

        def tool(self, name):
            path = tmp_path / name
            path.write_text(f"#!{sys.executable}\nimport sys\nopen({str(log)!r}, 'a').write('{name} ')\n"
                            f"if {name in self.fail}: sys.exit(3)\n"
                            "open(sys.argv[sys.argv.index('-o') + 1], 'w').write('x')\n")
            path.chmod(0o755)
            return str(path)

    f = Fake()
    monkeypatch.setattr(build, "LIBDIR", str(tmp_path / "lib"))
    monkeypatch.setattr(build, "LIB", str(tmp_path / "lib" / "libb200edsl.so"))
    monkeypatch.setattr(build, "TORCH_LIB", str(tmp_path / "lib" / "b200torch.so"))
    monkeypatch.setattr(build, "TORCH_ABI", str(tmp_path / "lib" / "b200torch.abi"))
    monkeypatch.setattr(build, "nvcc", lambda: f.tool("nvcc"))
    monkeypatch.setattr(build, "torch_commands", lambda: (
        [f.tool("g++"), "-o", build.TORCH_LIB + ".o"], [f.tool("ld"), "-o", build.TORCH_LIB + ".tmp"]))
    return f


def test_both_are_built(fake):
    assert build.needs_build()
    build.build()
    assert os.path.exists(build.LIB) and os.path.exists(build.TORCH_LIB)
    assert sorted(os.listdir(build.LIBDIR)) == ["b200torch.abi", "b200torch.so", "libb200edsl.so"]
    calls = fake.calls()
    assert sorted(calls) == ["g++", "ld", "nvcc"] and not build.needs_build()
    build.build()
    assert fake.calls() == calls


@pytest.mark.parametrize("tool", ["g++", "ld"])
def test_a_torch_module_that_fails_leaves_the_library(fake, tool):
    fake.fail = (tool,)
    with pytest.raises(subprocess.CalledProcessError):
        build.build()
    assert os.path.exists(build.LIB) and not os.path.exists(build.TORCH_LIB)


def test_without_torch_the_library_is_built(fake, monkeypatch):
    def no_torch():
        raise ImportError("no torch")
    monkeypatch.setattr(build, "torch_commands", no_torch)
    build.build()
    assert os.path.exists(build.LIB) and not os.path.exists(build.TORCH_LIB)


def test_a_library_that_fails_is_raised(fake):
    fake.fail = ("nvcc",)
    with pytest.raises(subprocess.CalledProcessError):
        build.build()
    assert not os.path.exists(build.LIB) and not os.path.exists(build.TORCH_LIB)


def test_the_module_is_built_again_for_another_torch(fake, monkeypatch):
    build.build()
    now = build.torch_abi()
    assert torch.__version__ in now
    monkeypatch.setattr(build, "torch_abi", lambda: now + ".1")
    assert build.needs_build()
    build.build()
    assert sorted(fake.calls()) == ["g++", "g++", "ld", "ld", "nvcc"] and not build.needs_build()
    os.remove(build.TORCH_ABI)  # built by who knows what
    assert build.needs_build()
