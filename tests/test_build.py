"""CPU tests of what is built for whom (lyradiff_b200/build.py) and of the loader of the extension module."""

import os
import sysconfig

import pytest

from lyradiff_b200 import _lib, build


def test_the_classes_build_where_the_extension_module_cannot(monkeypatch, tmp_path):
    """Without Python's headers the module behind some of ops.py does not compile; the library of torch classes does not need them."""
    build.build()
    started = []

    class Compiler:
        def __init__(self, cmd, **_):
            self.module = build.HOST_SRC in cmd
            started.append(cmd[cmd.index("-o") + 1])

        def wait(self):
            return int(self.module)
    monkeypatch.setattr(build.subprocess, "Popen", Compiler)
    monkeypatch.setattr(build, "CLASSES_LIB", str(tmp_path / "classes.so"))
    monkeypatch.setattr(build, "HOST_LIB", str(tmp_path / "host.so"))
    assert build.build_classes() == build.CLASSES_LIB and build.CLASSES_LIB in started
    with pytest.raises(RuntimeError, match="host.so"):
        build.build_host()
    started.clear()
    with pytest.raises(RuntimeError, match="host.so"):
        build.build_all()
    assert sorted(started) == sorted([build.CLASSES_LIB, build.HOST_LIB])


def test_the_extension_module_is_this_interpreters(monkeypatch, tmp_path):
    """Its name carries the interpreter's tag, so that no other loads it; a file without one is not taken for it."""
    build.build_host()
    suffix = sysconfig.get_config_var("EXT_SUFFIX")
    assert os.path.basename(build.HOST_LIB) == "_host" + suffix != "_host.so"
    assert _lib.host().__file__ == build.HOST_LIB
    (tmp_path / "_host.so").write_bytes(b"")
    monkeypatch.setattr(_lib, "_host", None)
    monkeypatch.setattr(_lib, "_HERE", str(tmp_path))
    with pytest.raises(ImportError, match="not built"):
        _lib.host()
