"""When the HIP extensions are compiled."""
import importlib.util
import os
import sys

import pytest
import setuptools

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def _load(name, monkeypatch):
    monkeypatch.setattr(setuptools, "setup", lambda **kw: None)
    spec = importlib.util.spec_from_file_location(
        "under_test", os.path.join(ROOT, name))
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


@pytest.fixture
def built(monkeypatch, tmp_path):
    """setup.py over a folder of its own, and the commands that it runs."""
    module = _load("setup.py", monkeypatch)
    (tmp_path / "csrc" / "hip").mkdir(parents=True)
    (tmp_path / "pkg").mkdir()
    files = [tmp_path / "setup.py"] + [
        tmp_path / "csrc" / "hip" / f for f in module.HIP_EXTENSIONS.values()]
    for f in files:
        f.write_text("")
        os.utime(f, (1000, 1000))
    monkeypatch.setattr(module, "ROOT", str(tmp_path))
    monkeypatch.setattr(module, "PKG", str(tmp_path / "pkg"))
    monkeypatch.setattr(module.shutil, "which", lambda name: sys.executable)
    commands = []

    def run(cmd, cwd):
        commands.append(cmd)
        with open(cmd[cmd.index("-o") + 1], "w"):
            pass
    monkeypatch.setattr(module.subprocess, "check_call", run)
    return module, files, commands


def test_compiled_when_a_source_or_a_switch_changes(built):
    module, files, commands = built
    for name, source in module.HIP_EXTENSIONS.items():
        before = len(commands)
        out = module.build_hip_extension(name)
        assert len(commands) == before + 1
        assert module.build_hip_extension(name) == out
        assert len(commands) == before + 1
        for f in files:
            if f.name not in (source, "setup.py"):
                continue
            os.utime(out, (2000, 2000))
            os.utime(f, (3000, 3000))
            module.build_hip_extension(name)
            os.utime(f, (1000, 1000))
        assert len(commands) == before + 3
        module.build_hip_extension(name, force=True)
        assert len(commands) == before + 4


def test_the_entry_compiles_whatever_is_built(monkeypatch):
    entry = _load("__graft_entry__.py", monkeypatch)
    seen = []

    def stop(cmd, cwd):
        seen.append(cmd)
        raise InterruptedError
    monkeypatch.setattr(entry.subprocess, "check_call", stop)
    with pytest.raises(InterruptedError):
        entry.build()
    assert "--force" in seen[0]
    module = _load("setup.py", monkeypatch)
    asked = []
    monkeypatch.setattr(module.build_ext, "run", lambda self: None)
    monkeypatch.setattr(module, "build_hip_extension",
                        lambda name, force: asked.append((name, force)))
    command = module.BuildExt(setuptools.Distribution())
    command.force = 1
    command.run()
    assert sorted(asked) == sorted((n, True) for n in module.HIP_EXTENSIONS)
