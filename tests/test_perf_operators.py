"""perf/operators.py: what its calls pass on."""
from __future__ import annotations

import importlib.util
from pathlib import Path
from types import SimpleNamespace

import pytest
import torch

ROOT = Path(__file__).resolve().parents[1]


@pytest.mark.parametrize("op", ["rope", "score", "attend", "append", "read", "round"])
def test_each_pass_runs_on_the_current_stream(monkeypatch, op):
    spec = importlib.util.spec_from_file_location("perf_operators", ROOT / "perf" / "operators.py")
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    mod.own = True
    streams = []

    class Lib:
        def __getattr__(self, name):
            return lambda *args: streams.append(args[-1]) or 0

    cell = torch.zeros(1)
    s = {"case": {"op": op}, "own": {"lib": Lib(), "rope": None, "cache": None, "seqs": None, "append": None, "read": None, "args": None}}
    s.update({name: cell for name in ("out", "lp", "ent", "ids", "top", "k_out", "v_out", "scales", "q_out")}, codes=torch.zeros(1, dtype=torch.uint8))
    for current in (7, 9):
        monkeypatch.setattr(torch.cuda, "current_stream", lambda: SimpleNamespace(cuda_stream=current))
        mod.run(s)
    calls = 2 if op == "round" else 1
    assert streams == [7] * calls + [9] * calls
