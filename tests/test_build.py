"""build(): what it compiles, and that a library which is already there is no reason not to compile (CPU; no compiler runs)."""
import os

import __graft_entry__ as g
from oracle import oracle


def test_build_compiles_everything_each_time_it_is_called(monkeypatch):
    assert os.path.exists(g.LIB) and os.path.exists(g.UBENCH_BIN)   # both are there, and up to date
    compiled, checker = [], []
    monkeypatch.setattr(g, "_compile", lambda cmd: compiled.append(cmd[cmd.index("-o") + 1]))
    monkeypatch.setattr(oracle, "build", lambda force=False: checker.append(force))
    for _ in range(2):
        g.build()
    assert compiled == [g.LIB, g.UBENCH_BIN] * 2
    assert checker == [True, True]
