"""The torch binding is rebuilt for another interpreter, torch or compiler command, and not otherwise (no compiler run)."""

import importlib.util
import os
import subprocess
from pathlib import Path

import torch

PKG = Path(__file__).resolve().parents[1] / "qwen2-int4-systems_b200"


def test_objects_belong_to_what_they_were_compiled_against(tmp_path, monkeypatch):
    spec = importlib.util.spec_from_file_location("_build_under_test", PKG / "build.py")
    build = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(build)
    csrc = tmp_path / "csrc"
    csrc.mkdir()
    (tmp_path / "include").mkdir()
    (csrc / "one.cpp").write_text("")
    (csrc / "two.cpp").write_text("")
    (tmp_path / "include" / "qi4_b200.h").write_text("")
    lib = tmp_path / "libqi4_b200.so"
    lib.write_text("")
    for name, value in (("ROOT", tmp_path), ("PKG", tmp_path), ("CSRC", csrc), ("BUILD", tmp_path / "_build"),
                        ("LIB", lib)):
        monkeypatch.setattr(build, name, value)
    ran = []

    def run(cmd, **kw):
        out = Path(cmd[cmd.index("-o") + 1])
        out.write_text(" ".join(cmd))
        ran.append("compile" if "-c" in cmd else "link")
        return subprocess.CompletedProcess(cmd, 0, "", "")

    monkeypatch.setattr(build.subprocess, "run", run)

    def built(version):
        monkeypatch.setattr(torch, "__version__", version)
        ran.clear()
        out = build.build_torch_binding()
        return sorted(ran), out.read_text()

    both = ["compile", "compile", "link"]
    first = built("2.0")
    assert first[0] == both
    assert built("2.0") == ([], first[1])
    other = built("2.1")
    assert other[0] == both
    objects = [w for w in other[1].split() if w.endswith(".o")]
    assert len(objects) == 2 and not set(objects) & set(first[1].split())
    # Back: the objects are there, the module is linked from them again.
    assert built("2.0") == (["link"], first[1])
    (csrc / "one.cpp").write_text("x")
    later = lib.stat().st_mtime + 5
    os.utime(csrc / "one.cpp", (later, later))
    assert built("2.0")[0] == ["compile", "link"]
