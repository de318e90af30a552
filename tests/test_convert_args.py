"""The converter's arguments: host logic."""
import runpy
import sys

import pytest


@pytest.mark.parametrize("args", [["--zeros"], ["--group", "64"], ["--group", "128", "--zeros"], ["--group", "16", "--int4"], []])
def test_refused_arguments(monkeypatch, capsys, args):
    """What only 4 bits have is not taken without --int4, where it would change nothing."""
    monkeypatch.setattr(sys, "argv", ["convert", "in", *(["out"] if args else []), *args])
    monkeypatch.delitem(sys.modules, "estudiocanciones_amd.convert", raising=False)
    with pytest.raises(SystemExit) as e:
        runpy.run_module("estudiocanciones_amd.convert", run_name="__main__")
    assert e.value.code != 0
    if args and "--int4" not in args:
        assert "--int4" in capsys.readouterr().err.splitlines()[-1]
