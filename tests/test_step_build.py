"""CPU: _step.so belongs to one torch and one Python; another's is rebuilt, and refused before it is loaded."""
import pytest

from on_device_sd_b200 import _lib, build


def stale_copy(tmp_path):
    data = build.STEP.read_bytes()
    tag = build.step_tag().encode()
    assert data.count(tag) == 1
    path = tmp_path / "_step.so"
    path.write_bytes(data.replace(tag, tag.replace(b"torch ", b"torch 0", 1)[: len(tag)]))
    return path


def test_the_built_file_names_what_it_was_built_for():
    build.build()
    assert build.built_for(build.STEP) == build.step_tag()
    import torch
    assert torch.__version__ in build.step_tag()


def test_a_file_for_another_torch_is_rebuilt(tmp_path, monkeypatch):
    build.build()
    path = stale_copy(tmp_path)
    calls = []

    class Done:
        returncode, stdout, stderr = 0, "", ""

    monkeypatch.setattr(build.subprocess, "run", lambda cmd, **kw: calls.append(cmd) or Done)
    build._build_step(False, False)
    assert not calls, "the current file stays"
    monkeypatch.setattr(build, "STEP", path)
    build._build_step(False, False)
    assert len(calls) == 1 and str(path) in calls[0]


def test_a_file_for_another_torch_is_not_loaded(tmp_path, monkeypatch):
    build.build()
    monkeypatch.setattr(_lib, "STEP_PATH", stale_copy(tmp_path))
    monkeypatch.setattr(_lib, "_step", None)
    with pytest.raises(ImportError, match="rebuild"):
        _lib.load_step()
    (tmp_path / "none.so").write_bytes(b"\x7fELF of an earlier build")
    monkeypatch.setattr(_lib, "STEP_PATH", tmp_path / "none.so")
    with pytest.raises(ImportError, match="rebuild"):
        _lib.load_step()


def test_the_library_alone_needs_no_tensor_entry_points(monkeypatch):
    build.build()
    monkeypatch.setattr(build, "_build_step", lambda *a: pytest.fail("not asked for"))
    assert build.build(step=False) == build.LIB
