"""The library does not depend on the cleartext operators' Python binding, which needs g++ and PyTorch's headers."""

import pytest

from holmes_amd import build as hb


@pytest.fixture
def made(tmp_path, monkeypatch):
    """A build whose compilers only note what they are asked for; a failing step is put in by the test."""
    monkeypatch.setattr(hb, "OUT_DIR", tmp_path)
    monkeypatch.setattr(hb, "LIB", tmp_path / "libholmes_ckks.so")
    monkeypatch.setattr(hb, "CLEAR", tmp_path / "_clear.so")
    commands = []

    class Done:
        returncode, stderr = 0, ""

    def run(cmd, **kw):
        commands.append(cmd)
        with open(cmd[cmd.index("-o") + 1], "w") as f:
            f.write("made")
        return Done

    monkeypatch.setattr(hb.subprocess, "run", run)
    return commands


def test_both(made, capsys):
    assert hb.build() == hb.LIB
    assert hb.LIB.exists() and hb.CLEAR.exists() and "not available" not in capsys.readouterr().err
    binding = [c for c in made if str(hb.CSRC / "clear_bind.cpp") in c]
    assert len(binding) == 1 and any(a.startswith("-D_GLIBCXX_USE_CXX11_ABI=") for a in binding[0])


@pytest.mark.parametrize("step", ["_compile_binding", "_link_binding"])
@pytest.mark.parametrize("error", [RuntimeError("g++ failed"), FileNotFoundError("g++"), ImportError("torch")])
def test_the_library_without_the_binding(made, monkeypatch, capsys, step, error):
    def fail(*a):
        raise error

    monkeypatch.setattr(hb, step, fail)
    hb.CLEAR.write_text("of an earlier library")
    assert hb.build() == hb.LIB
    assert hb.LIB.read_text() == "made" and not hb.CLEAR.exists()
    assert "holmes_amd.clear is not available" in capsys.readouterr().err


def test_a_library_that_fails_is_an_error(made, monkeypatch):
    def fail(src, build_dir):
        raise RuntimeError(f"hipcc failed for {src}")

    monkeypatch.setattr(hb, "_compile", fail)
    with pytest.raises(RuntimeError, match="hipcc"):
        hb.build()
    assert not hb.LIB.exists()
