"""perf/operators.py's calls of this package, on the CPU: what is prepared for
them is complete before the package's own stream may read it."""
import importlib.util
import os

import pytest
import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

CASES = [
    {"kind": "attend", "heads": 2, "kv_heads": 1, "head_dim": 64, "batch": 2, "tokens": 3, "first": 5, "ragged": True, "page_size": 4, "holes": 0},
    {"kind": "append", "heads": 2, "kv_heads": 1, "head_dim": 64, "batch": 1, "tokens": 1, "first": 5, "ragged": False, "page_size": 4, "holes": 0},
    {"kind": "copy", "kv_heads": 1, "head_dim": 64, "layers": 1, "page_size": 2, "pages": 8, "pairs": 2, "fan": 1},
    {"kind": "sample", "rows": 2, "count": 100, "rule": "mixed"},
]


@pytest.mark.parametrize("case", CASES, ids=[c["kind"] for c in CASES])
def test_prepared_inputs_are_complete_for_the_package_s_stream(monkeypatch, case):
    spec = importlib.util.spec_from_file_location("operators", os.path.join(ROOT, "perf", "operators.py"))
    operators = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(operators)
    waits = []
    monkeypatch.setattr(torch.cuda, "synchronize", lambda *a: waits.append(a))
    operators.DEVICE = "cpu"
    operators.prepare(case, 1)
    assert not waits  # the plain form runs on torch's stream itself
    operators.own = True
    state = operators.prepare(case, 1)
    assert len(waits) == 1 and state.case is case
