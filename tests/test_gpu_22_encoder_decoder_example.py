"""The example of the 16-bit cache's operators runs, eager and captured, and its results are those of 64 bits (it checks them)."""
import importlib.util
from pathlib import Path

import pytest

pytestmark = pytest.mark.gpu


def test_encoder_decoder_step(capsys):
    path = Path(__file__).resolve().parent.parent / "examples" / "encoder_decoder_step.py"
    spec = importlib.util.spec_from_file_location("encoder_decoder_step", path)
    example = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(example)
    example.main()
    assert capsys.readouterr().out.count("relative error") == 1 + 2 * example.STEPS
