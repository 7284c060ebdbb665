"""The build of the kernel library, with a compiler that only writes files."""
import os
import stat

from cpmcu_b200.ops import build


def _compiler(folder):
    path = os.path.join(folder, "nvcc")
    with open(path, "w") as f:
        f.write('#!/bin/sh\nwhile [ $# -gt 0 ]; do if [ "$1" = -o ]; then echo built > "$2"; fi; shift; done\n')
    os.chmod(path, os.stat(path).st_mode | stat.S_IXUSR)
    return path


def test_a_build_leaves_the_library_and_no_objects(tmp_path, monkeypatch):
    """Objects take as much room as the library they went into, in a tree that is copied with its built files."""
    monkeypatch.setenv("CPMCU_BUILD_DIR", str(tmp_path / "lib"))
    monkeypatch.setattr(build, "find_nvcc", lambda: _compiler(str(tmp_path)))
    for checked in (False, True):
        path = build.build(force=True, verbose=False, check_bounds=checked)
        assert path == build.existing_library(checked) and os.path.isfile(path)
        assert sorted(os.listdir(os.path.dirname(path)))[-2:] == ["fingerprint", build.LIB_NAME]
    left = [f for _, _, files in os.walk(tmp_path / "lib") for f in files if f.endswith(".o")]
    assert not left, left
