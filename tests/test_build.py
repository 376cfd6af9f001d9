"""The in-tree build replaces both libraries or neither (CPU only; the
compilers are stood in for)."""

from __future__ import annotations

import importlib.util
from pathlib import Path

import pytest

ROOT = Path(__file__).resolve().parent.parent


@pytest.fixture
def build(tmp_path, monkeypatch):
    """_build.py on a package folder of its own that holds an old pair; its
    commands write their outputs and keep a record."""
    spec = importlib.util.spec_from_file_location("_build_under_test",
                                                  ROOT / "maxsim_amd" / "_build.py")
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    for name, value in (("PKG", tmp_path), ("LIB", tmp_path / mod.LIB.name),
                        ("TORCH_LIB", tmp_path / mod.TORCH_LIB.name),
                        ("BUILD_INFO", tmp_path / mod.BUILD_INFO.name)):
        monkeypatch.setattr(mod, name, value)
    mod.LIB.write_text("old")
    mod.TORCH_LIB.write_text("old")
    mod.seen = []
    mod.fails = None

    def run(cmds):
        for cmd in cmds:
            mod.seen.append(cmd)
            if mod.fails and mod.fails(cmd):
                raise RuntimeError("native build failed")
            Path(cmd[cmd.index("-o") + 1]).write_text("new")

    monkeypatch.setattr(mod, "_run", run)
    return mod


def _pair(mod):
    return mod.LIB.read_text(), mod.TORCH_LIB.read_text()


def test_a_whole_build_replaces_both(build):
    build.build()
    assert _pair(build) == ("new", "new")
    # the binding is linked against the library that was built with it
    link = next(c for c in build.seen if "-lmaxsim_amd" in c)
    folder = Path(link[link.index("-L") + 1])
    made = [Path(c[c.index("-o") + 1]) for c in build.seen if "-o" in c]
    assert folder / build.LIB.name in made
    # nothing half made is left where it could be taken for a library
    assert sorted(p.name for p in build.PKG.glob("*.so*")) == sorted(
        [build.LIB.name, build.TORCH_LIB.name])


@pytest.mark.parametrize("what", ["hip source", "library", "binding source", "binding"])
def test_a_failed_build_replaces_neither(build, what):
    build.fails = {
        "hip source": lambda c: any(str(a).endswith(".hip") for a in c),
        "library": lambda c: "hipcc" in c[0] and "-shared" in c,
        "binding source": lambda c: any(str(a).endswith("torch_training.cpp") for a in c),
        "binding": lambda c: "-lmaxsim_amd" in c,
    }[what]
    with pytest.raises(RuntimeError, match="native build failed"):
        build.build()
    assert _pair(build) == ("old", "old")
