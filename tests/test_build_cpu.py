"""The build's notion of an up-to-date object."""
import os

from speaksense_amd import build


def test_objects_of_other_flags_are_stale(tmp_path, monkeypatch):
    """A changed command rebuilds every object, as a touched source or header does; nothing else does."""
    monkeypatch.setattr(build, "HERE", str(tmp_path))
    monkeypatch.setattr(build, "CSRC", str(tmp_path))
    monkeypatch.setattr(build, "HEADERS", ["a.h"])
    os.makedirs(tmp_path / "build")
    src, obj = tmp_path / "a.hip", tmp_path / "build" / "a.hip.o"
    (tmp_path / "a.h").write_text("")
    src.write_text("")
    cmd = ["hipcc", "-O3", "-c", str(src), "-o", str(obj)]
    stale = lambda c=cmd: build._stale(str(obj), str(src), c)  # noqa: E731
    assert stale()                                        # no object
    obj.write_text("")
    assert stale()                                        # an object of an unknown command
    build._built(str(obj), cmd)
    assert not stale()
    assert stale(["hipcc", "-O2"] + cmd[2:])
    for dep in (src, tmp_path / "a.h"):
        os.utime(dep, (os.path.getmtime(obj) + 10,) * 2)
        assert stale()
        os.utime(dep, (os.path.getmtime(obj) - 10,) * 2)
        assert not stale()


def test_all_device_code_is_built_without_packed_float32():
    at = build.FLAGS.index("-packed-fp32-ops")
    assert build.FLAGS[at - 3:at] == ["-Xclang", "-target-feature", "-Xclang"]
