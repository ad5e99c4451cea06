"""examples/serve_step.py runs: prompts, then a captured step replayed, each
checked against float64 by the example itself."""
import runpy
import os
import sys

import pytest

pytestmark = pytest.mark.gpu
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_serve_step_example(gpu, monkeypatch, capsys):
    monkeypatch.setattr(sys, "argv", ["serve_step.py", "--steps", "3"])
    runpy.run_path(os.path.join(ROOT, "examples", "serve_step.py"), run_name="__main__")
    assert "3 steps of 4 sequences" in capsys.readouterr().out
