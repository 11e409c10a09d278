"""CPU: how the library's sources are compiled, with hipcc replaced by a program that only makes its output file."""
import os
import subprocess
import sys
import types

from conftest import ROOT
from satflow_amd import build


def test_every_source_is_compiled_without_packed_fp32_and_again_when_the_flags_change(monkeypatch, tmp_path):
    commands = []

    def hipcc(cmd, **kw):
        commands.append(cmd)
        open(cmd[cmd.index("-o") + 1], "w").close()
        return types.SimpleNamespace(returncode=0, stdout="", stderr="")

    monkeypatch.setattr(build, "subprocess", types.SimpleNamespace(run=hipcc))
    monkeypatch.setattr(build, "LIBDIR", str(tmp_path))
    monkeypatch.setattr(build, "LIB", str(tmp_path / "lib.so"))
    flags = tmp_path / "build.py"
    flags.write_text("")
    monkeypatch.setattr(build, "SELF", str(flags))
    build.build_library(verbose=False)
    compiled = {os.path.basename(c[c.index("-c") + 1]): c for c in commands if "-c" in c}
    assert sorted(compiled) == sorted(f for f in os.listdir(build.CSRC) if f.endswith(".hip"))
    for c in compiled.values():
        assert c[c.index("-packed-fp32-ops") - 3:c.index("-packed-fp32-ops") + 1] == ["-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops"]
    commands.clear()
    build.build_library(verbose=False)
    assert not commands
    os.utime(flags, (os.path.getmtime(flags) + 3600,) * 2)
    build.build_library(verbose=False)
    assert len([c for c in commands if "-c" in c]) == len(compiled) and len(commands) == len(compiled) + 1


def test_flags_for_scripts():
    r = subprocess.run([sys.executable, "-m", "satflow_amd.build", "--flags"], capture_output=True, text=True, cwd=ROOT)
    assert r.returncode == 0 and r.stdout.split() == build.FLAGS
