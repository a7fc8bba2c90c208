"""When the build sees that a library is out of date."""
import os

import pytest

from silent_speech_amd import build


@pytest.mark.parametrize("lib,stale", [("SO", "stale"), ("TORCH_SO", "torch_side_stale")])
def test_a_library_older_than_the_flags_is_built_again(lib, stale, tmp_path, monkeypatch):
    """The flags stand in build.py: a library that was built before it was last changed may lack some."""
    so = tmp_path / "lib.so"
    monkeypatch.setattr(build, lib, so)
    assert getattr(build, stale)()                              # none is there
    so.touch()
    newest = max(os.stat(p).st_mtime for p in [build.CSRC / s for s in build.SOURCES] + build.HEADERS + [build.TORCH_SOURCE])
    flags = tmp_path / "build.py"
    flags.touch()
    monkeypatch.setattr(build, "__file__", str(flags))
    later = max(newest, so.stat().st_mtime) + 10
    os.utime(flags, (later, later))
    os.utime(so, (later - 1, later - 1))
    assert getattr(build, stale)()
    os.utime(so, (later + 1, later + 1))
    assert not getattr(build, stale)()


def test_the_torch_side_belongs_to_its_torch(tmp_path, monkeypatch):
    so, package = tmp_path / "lib.so", tmp_path / "torch"
    package.mkdir()
    for f in (so, package / "__init__.py", package / "version.py"):
        f.touch()
    spec = type("Spec", (), {"origin": str(package / "__init__.py")})
    monkeypatch.setattr(build, "TORCH_SO", so)
    monkeypatch.setattr(build.importlib.util, "find_spec", lambda name: spec)
    later = max(os.stat(p).st_mtime for p in (build.TORCH_SOURCE, build.API, build.__file__, so)) + 10
    os.utime(so, (later, later))
    assert not build.torch_side_stale()
    os.utime(package / "version.py", (later + 1, later + 1))
    assert build.torch_side_stale()
