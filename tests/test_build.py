"""What titan_amd.build needs: hipcc for the C libraries, torch for its binding alone."""

import sys

import pytest

from titan_amd import build as b


@pytest.fixture
def steps(monkeypatch, tmp_path):
    """The build's steps in order, nothing compiled."""
    done = []
    monkeypatch.setattr(b, "BUILD", tmp_path / "build")
    monkeypatch.setattr(b, "LIB_DIR", tmp_path / "lib")
    monkeypatch.setattr(b, "_compile", lambda src, variant="", defines=(): tmp_path / (src.stem + variant + ".o"))
    monkeypatch.setattr(b, "_link", lambda objs, lib: done.append(lib))
    monkeypatch.setattr(b, "_link_binding", lambda obj: done.append(b.BINDING_LIB))
    return done


def test_the_libraries_need_no_torch(steps, monkeypatch, capsys):
    monkeypatch.setitem(sys.modules, "torch", None)  # an import of it raises ImportError
    assert b.build() == b.LIB
    assert steps == [b.LIB, b.PEAKS_LIB, b.STAMPS_LIB]
    assert "torch" in capsys.readouterr().out


def test_a_binding_that_does_not_compile_leaves_the_libraries(steps, monkeypatch):
    def fail():
        raise RuntimeError("hipcc failed on binding.cpp")

    monkeypatch.setattr(b, "_compile_binding", fail)
    with pytest.raises(RuntimeError, match="binding.cpp"):
        b.build()
    assert steps == [b.LIB, b.PEAKS_LIB, b.STAMPS_LIB]


def test_with_torch_the_binding_is_linked_last(steps, monkeypatch, tmp_path):
    monkeypatch.setattr(b, "_compile_binding", lambda: tmp_path / "binding.o")
    b.build()
    assert steps == [b.LIB, b.PEAKS_LIB, b.STAMPS_LIB, b.BINDING_LIB]
