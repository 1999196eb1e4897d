"""The build without torch (a caller of the C ABI alone): the library is built,
the attention calls' Python side is left out, and said so."""

from __future__ import annotations

import importlib.util

import pytest

from colormlm_amd import build as b


@pytest.mark.parametrize("torch_there", [True, False])
def test_build_without_torch_is_the_library_alone(monkeypatch, tmp_path, capsys, torch_there):
    find = importlib.util.find_spec
    monkeypatch.setattr(importlib.util, "find_spec", lambda name, *a: find(name, *a) if torch_there or name != "torch" else None)
    if not torch_there:
        monkeypatch.setitem(__import__("sys").modules, "torch", None)  # an import of it fails
    for name in ("OUT", "PY_OUT", "OBJ"):
        monkeypatch.setattr(b, name, tmp_path / getattr(b, name).name)
    made = []

    def run(cmd, verbose):
        made.append(cmd[cmd.index("-o") + 1])
        open(made[-1], "w").close()

    monkeypatch.setattr(b, "_run", run)
    assert b.build() == tmp_path / "libs14hip.so"
    assert (tmp_path / "libs14hip.so").exists()
    assert (tmp_path / "_s14attn.so").exists() == torch_there
    assert ("torch" in capsys.readouterr().err) == (not torch_there)
