"""examples/shared_prompt.py runs: a picture's prompt in shared pages, questions
behind it, a captured step replayed, tokens read back, each checked against
float64 by the example itself."""
import os
import runpy
import sys

import pytest

pytestmark = pytest.mark.gpu
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_shared_prompt_example(gpu, monkeypatch, capsys):
    monkeypatch.setattr(sys, "argv", ["shared_prompt.py", "--steps", "3"])
    runpy.run_path(os.path.join(ROOT, "examples", "shared_prompt.py"), run_name="__main__")
    out = capsys.readouterr().out
    assert "3 steps of 6 conversations" in out and "tokens read back" in out
