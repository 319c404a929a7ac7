"""What cactus_amd/build.py compiles again, with a compiler that only notes its command lines."""
import importlib.util
import os
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture
def builder(tmp_path, monkeypatch):
    """The module on a folder of its own with two sources; .ran: what was compiled or linked since it was last asked."""
    spec = importlib.util.spec_from_file_location("_build_under_test", os.path.join(ROOT, "cactus_amd", "build.py"))
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    (tmp_path / "csrc").mkdir()
    for name in ("a.hip", "b.cpp", "x.h"):
        (tmp_path / "csrc" / name).write_text("")
    ran, failing = [], set()

    class Compiler:
        def __init__(self, cmd):
            self.out = cmd[cmd.index("-o") + 1]
            ran.append(os.path.basename(self.out))
            self.bad = os.path.basename(self.out) in failing
            if not self.bad:
                open(self.out, "w").close()

        def wait(self):
            return 1 if self.bad else 0

    monkeypatch.setattr(mod, "HERE", str(tmp_path))
    monkeypatch.setattr(mod, "CSRC", str(tmp_path / "csrc"))
    monkeypatch.setattr(mod, "LIBDIR", str(tmp_path / "lib"))
    monkeypatch.setattr(mod, "SO", str(tmp_path / "lib" / "lib.so"))
    monkeypatch.setattr(mod, "SOURCES", ["a.hip", "b.cpp"])
    monkeypatch.setattr(mod, "HEADERS", ["x.h"])
    monkeypatch.setattr(mod, "EXTRA_FLAGS", {})
    monkeypatch.setattr(mod, "build_examples", lambda *a: [])
    monkeypatch.setattr(subprocess, "Popen", Compiler)
    monkeypatch.setattr(subprocess, "check_call", lambda cmd: Compiler(cmd).wait())

    def built(**kw):
        ran.clear()
        mod.build(**kw)
        return sorted(ran)
    mod.built, mod.failing = built, failing
    return mod


def test_nothing_changed_nothing_is_built(builder):
    assert builder.built() == ["a.hip.o", "b.cpp.o", "lib.so"]
    assert builder.built() == []
    assert builder.built(force=True) == ["a.hip.o", "b.cpp.o", "lib.so"]


def test_other_flags_build_everything_again(builder, monkeypatch):
    builder.built()
    monkeypatch.setattr(builder, "FLAGS", builder.FLAGS + ["-DMORE"])
    assert builder.built() == ["a.hip.o", "b.cpp.o", "lib.so"]
    assert builder.built() == []


def test_other_flags_of_one_file_build_that_file_again(builder, monkeypatch):
    builder.built()
    monkeypatch.setattr(builder, "EXTRA_FLAGS", {"a.hip": ["-fno-slp-vectorize"]})
    assert builder.built() == ["a.hip.o", "lib.so"]
    monkeypatch.setattr(builder, "EXTRA_FLAGS", {})
    assert builder.built() == ["a.hip.o", "lib.so"]


def test_objects_of_unknown_flags_are_built_again(builder):
    """A tree from before the command lines were kept."""
    builder.built()
    objdir = os.path.join(builder.HERE, "build")
    for name in os.listdir(objdir):
        if not name.endswith(".o"):
            os.remove(os.path.join(objdir, name))
    assert builder.built() == ["a.hip.o", "b.cpp.o", "lib.so"]


def test_a_failed_build_is_not_taken_for_a_built_one(builder, monkeypatch):
    builder.built()
    monkeypatch.setattr(builder, "FLAGS", builder.FLAGS + ["-DMORE"])
    builder.failing.add("b.cpp.o")
    with pytest.raises(RuntimeError, match="b.cpp"):
        builder.built()
    builder.failing.clear()
    assert "b.cpp.o" in builder.built()
    assert builder.built() == []


def test_the_entry_compiles_every_source_each_time(tmp_path, monkeypatch):
    import __graft_entry__ as entry
    (tmp_path / "cactus_amd").mkdir()
    note = tmp_path / "called"
    (tmp_path / "cactus_amd" / "build.py").write_text(
        f"def build(force=False, verbose=False):\n    open({str(note)!r}, 'a').write('all ' if force else 'some ')\n")
    monkeypatch.setattr(entry, "ROOT", str(tmp_path))
    entry.build()
    entry.build()
    assert note.read_text() == "all all "
