"""What ``xtile_b200/build.py`` builds, with its compilers replaced by one that writes empty files."""
import importlib.util
from pathlib import Path

import pytest

pytest.importorskip("pybind11")
ROOT = Path(__file__).resolve().parents[1]


@pytest.fixture
def built(tmp_path, monkeypatch):
    """The module building into an empty directory, and the outputs of its steps so far."""
    spec = importlib.util.spec_from_file_location("build_under_test", ROOT / "xtile_b200" / "build.py")
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    outputs = []

    def run(cmd):
        out = Path(cmd[cmd.index("-o") + 1])
        out.write_bytes(b"")
        outputs.append(out.name)

    monkeypatch.setattr(module, "_run", run)
    monkeypatch.setattr(module, "BUILD", tmp_path / "_build")
    for name in ("LIB", "EXT", "SERVING_EXT"):
        monkeypatch.setattr(module, name, tmp_path / getattr(module, name).name)
    return module, outputs


def hide_torch(monkeypatch):
    find = importlib.util.find_spec
    monkeypatch.setattr(importlib.util, "find_spec", lambda name, *a: None if name == "torch" else find(name, *a))


def test_the_library_and_the_extension_build_without_torch(built, monkeypatch):
    module, outputs = built
    hide_torch(monkeypatch)
    module.build()
    assert module.LIB.exists() and module.EXT.exists()
    assert not module.SERVING_EXT.exists() and "serving_module.o" not in outputs
    outputs.clear()
    module.build()
    assert outputs == []


def test_the_serving_extension_follows_torch(built, monkeypatch, tmp_path):
    module, outputs = built
    torch = tmp_path / "torch"
    torch.mkdir()
    (torch / "version.py").write_text("__version__ = '1'\n")
    monkeypatch.setattr(module, "_torch_dir", lambda: torch)
    module.build()
    assert {"serving_module.o", module.SERVING_EXT.name} <= set(outputs)
    outputs.clear()
    module.build()
    assert outputs == []
    (torch / "version.py").write_text("__version__ = '2'\n")  # another torch in its place
    module.build()
    assert outputs == ["serving_module.o", module.SERVING_EXT.name]
    outputs.clear()
    module.build()
    assert outputs == []
