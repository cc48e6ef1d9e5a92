"""The library's build (detrpose_amd.build): which objects it takes for current. The compiler here is a stand-in
that writes its own command line as the object."""
import os
import stat

import pytest

from detrpose_amd import build as B

COMPILER = """#!/bin/sh
out=; prev=
for a in "$@"; do [ "$prev" = -o ] && out=$a; prev=$a; done
case "$*" in *b.hip*-DHALF*|*-DHALF*b.hip*) exit 1;; esac
echo "$*" > "$out"
"""


@pytest.fixture
def tree(tmp_path, monkeypatch):
    hipcc, src = tmp_path / "hipcc", tmp_path / "csrc"
    hipcc.write_text(COMPILER)
    hipcc.chmod(hipcc.stat().st_mode | stat.S_IXUSR)
    src.mkdir()
    for n in ("a.hip", "b.hip"):
        (src / n).write_text("")
    monkeypatch.setattr(B, "_hipcc", lambda: str(hipcc))
    monkeypatch.setattr(B, "CSRC", str(src))
    monkeypatch.setattr(B, "BUILD", str(tmp_path / "obj"))
    monkeypatch.setattr(B, "LIB", str(tmp_path / "lib" / "lib.so"))
    monkeypatch.delenv("DETRPOSE_EXTRA_FLAGS", raising=False)
    return tmp_path


def test_a_build_that_failed_leaves_no_mixed_objects(tree, monkeypatch):
    """Objects of other flags that a failed build left behind are compiled again when the flags return."""
    flags = lambda n: (tree / "obj" / n).read_text()  # noqa: E731
    assert os.path.exists(B.build())
    monkeypatch.setenv("DETRPOSE_EXTRA_FLAGS", "-DHALF")
    with pytest.raises(RuntimeError, match="b.hip"):
        B.build()
    assert "-DHALF" in flags("a.hip.o") and "-DHALF" not in flags("b.hip.o")
    monkeypatch.delenv("DETRPOSE_EXTRA_FLAGS")
    B.build()
    assert "-DHALF" not in flags("a.hip.o") + flags("b.hip.o")
    old = os.stat(tree / "obj" / "a.hip.o").st_mtime_ns
    B.build()                                             # nothing has changed: nothing is compiled
    assert os.stat(tree / "obj" / "a.hip.o").st_mtime_ns == old
