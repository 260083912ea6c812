"""CPU tests of when hallo_amd.build compiles what: a changed source, header or set of flags, and nothing else."""
import os

import pytest

from hallo_amd import build as b


@pytest.fixture
def tree(tmp_path, monkeypatch):
    """Two sources and a header in a folder of their own, a compiler that only writes its output."""
    ran = []

    def run(cmd, check):
        out = cmd[cmd.index("-o") + 1]
        with open(out, "w") as f:
            f.write("built")
        ran.append(os.path.basename(out))
    src = tmp_path / "csrc"
    src.mkdir()
    for n in ("a.hip", "b.hip", "c.h"):
        (src / n).write_text("")
        os.utime(src / n, (1, 1))
    monkeypatch.setattr(b, "HERE", str(tmp_path))
    monkeypatch.setattr(b, "CSRC", str(src))
    monkeypatch.setattr(b, "LIB", str(tmp_path / "lib.so"))
    monkeypatch.setattr(b, "SOURCES", ["a.hip", "b.hip"])
    monkeypatch.setattr(b, "HEADERS", [str(src / "c.h")])
    monkeypatch.setattr(b.subprocess, "run", run)
    monkeypatch.delenv("HALLO_ABLATIONS", raising=False)

    def built(**kw):
        ran.clear()
        b.build(**kw)
        return sorted(ran)
    return src, built, monkeypatch


ALL = ["a.o", "b.o", "lib.so"]


def test_first_build_then_nothing(tree):
    _, built, _ = tree
    assert built() == ALL and built() == [] and built(force=True) == ALL


def test_newer_source_or_header(tree):
    src, built, _ = tree
    built()
    later = os.path.getmtime(src.parent / "lib.so") + 10
    os.utime(src / "a.hip", (later, later))
    assert built()[0] == "a.o" and "b.o" not in built()
    os.utime(src / "c.h", (later, later))
    assert built()[:2] == ["a.o", "b.o"]


def test_other_flags(tree):
    _, built, m = tree
    built()
    m.setattr(b, "NO_PACKED_FP32", [*b.NO_PACKED_FP32, "-DX"])
    assert built()[:2] == ["a.o", "b.o"] and "a.o" not in built()
    m.setenv("HALLO_ABLATIONS", "1")
    assert built()[:2] == ["a.o", "b.o"]
    m.delenv("HALLO_ABLATIONS")
    assert built()[:2] == ["a.o", "b.o"]


def test_every_compile_line_leaves_packed_fp32_out():
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    flags, lines = " ".join(b.NO_PACKED_FP32), []
    for top in ("hallo_amd", "tools"):
        for folder, _, files in os.walk(os.path.join(root, top)):
            for n in files:
                if n.endswith((".sh", ".hip", ".h")):
                    with open(os.path.join(folder, n), errors="replace") as f:
                        lines += [(n, line) for line in f if "hipcc" in line and "--offload-arch" in line]
    assert len(lines) >= 4 and all(flags in line for _, line in lines), lines
