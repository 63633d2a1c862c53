"""One list of compiler flags for every build of the library's sources: the arithmetic that the product's build leaves out (packed fp32) must
not come back in an A/B or timing build, and objects compiled with other flags are not kept."""
import glob
import os
import re
import types

import __graft_entry__ as ge
from uncltmo_amd import _hip

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_packed_fp32_is_off_and_every_compile_line_takes_the_shared_flags():
    assert "-packed-fp32-ops" in ge.FLAGS
    lines = 0
    for f in glob.glob(os.path.join(ROOT, "tools", "*")) + [os.path.join(ROOT, "__graft_entry__.py")]:
        text = open(f, errors="replace").read()
        for m in re.finditer(r'hipcc(?:\(\))?["\']?[, ].*', text):
            line = m.group(0)
            if "-c" in line.split() or '"-c"' in line or "-O3" in line or "-D" in line:      # compiles, does not only link
                lines += 1
                assert "__graft_entry__.py" in line or "$BASE" in line or "*FLAGS" in line, (f, line)
    assert lines >= 6
    base = [line for line in open(os.path.join(ROOT, "tools", "ab_variants.sh")) if line.startswith("BASE=")]
    assert len(base) == 1 and "__graft_entry__.py" in base[0]


def test_objects_compiled_with_other_flags_are_not_kept(monkeypatch, tmp_path):
    """build(force=False) in a folder of its own, the compiler replaced by one that writes its flags down"""
    csrc, made = tmp_path / "csrc", []
    csrc.mkdir()
    (tmp_path / "include").mkdir()
    for name in ("csrc/a.hip", "csrc/b.hip", "include/uncltmo_hip.h"):
        (tmp_path / name).write_text("")

    class Done:
        def __init__(self, cmd):
            made.append(cmd)
            open(cmd[cmd.index("-o") + 1], "w").write("x")

        def wait(self):
            return 0
    monkeypatch.setattr(_hip, "lib", lambda: types.SimpleNamespace(uncl_version=lambda: 1))
    monkeypatch.syspath_prepend(str(tmp_path))
    monkeypatch.setattr(ge, "ROOT", str(tmp_path))
    monkeypatch.setattr(ge, "CSRC", str(csrc))
    monkeypatch.setattr(ge, "LIB", str(tmp_path / "lib.so"))
    monkeypatch.setattr(ge.subprocess, "Popen", Done)
    monkeypatch.setattr(ge.subprocess, "check_call", Done)

    def compiled(**kw):
        made.clear()
        ge.build(**kw)
        return sum("-c" in c for c in made)
    assert compiled(force=False) == 2 and compiled(force=False) == 0
    assert compiled() == 2                                              # the check that everything builds compiles everything
    os.utime(tmp_path / "csrc" / "a.hip", (4e9, 4e9))
    assert compiled(force=False) == 1
    os.utime(tmp_path / "csrc" / "a.hip", (1, 1))
    monkeypatch.setattr(ge, "FLAGS", ge.FLAGS + ["-DOTHER"])
    assert compiled(force=False) == 2 and all("-DOTHER" in c for c in made if "-c" in c) and compiled(force=False) == 0
