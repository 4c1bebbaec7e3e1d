"""The library is one of the sources as they are: not a mix of two versions of a
header that changed while the files were compiled."""
import os

import pytest

from orthossm_b200 import build


@pytest.fixture
def tree(tmp_path, monkeypatch):
    """A small source tree and a compiler that writes what it was given."""
    for d in ("csrc", "include", "lib"):
        (tmp_path / d).mkdir()
    for f in ("a.cu", "b.cu", "c.cuh"):
        (tmp_path / "csrc" / f).write_text(f)
    (tmp_path / "include" / "orthossm_b200.h").write_text("h")
    cc = tmp_path / "nvcc"
    cc.write_text(f'''#!/bin/sh
while [ $# -gt 1 ]; do [ "$1" = -o ] && out=$2; shift; done
cat {tmp_path}/csrc/c.cuh > "$out"
mv {tmp_path}/edit {tmp_path}/csrc/c.cuh 2>/dev/null
exit 0
''')
    cc.chmod(0o755)
    monkeypatch.setattr(build, "SOURCES", ["a.cu", "b.cu"])
    for name, d in (("CSRC", "csrc"), ("INCLUDE", "include"), ("LIBDIR", "lib")):
        monkeypatch.setattr(build, name, str(tmp_path / d))
    monkeypatch.setattr(build, "nvcc", lambda: str(cc))
    return tmp_path


def test_a_header_that_changes_while_it_compiles(tree):
    (tree / "edit").write_text("another")
    with pytest.raises(RuntimeError, match="c.cuh"):
        build.build()
    assert os.listdir(tree / "lib") == []
    out = build.build()
    assert open(out).read() == "another" and os.listdir(tree / "lib") == [build.LIBNAME]
    when = os.path.getmtime(out)
    assert build.build() == out and os.path.getmtime(out) == when  # nothing to do


def test_a_file_that_does_not_compile(tree):
    old = build.build()
    (tree / "nvcc").write_text("#!/bin/sh\nexit 3\n")
    with pytest.raises(Exception):
        build.build(force=True)
    assert open(old).read() == "c.cuh" and os.listdir(tree / "lib") == [build.LIBNAME]
