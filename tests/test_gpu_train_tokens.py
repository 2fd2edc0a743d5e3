"""The example network: lookups, layers, gradients and AdamW with states in 8 bits together, in training and token by
token. Its language is learnt without error, which starts from a loss of about ln(96) = 4.6."""
import importlib.util
from pathlib import Path

import pytest

pytestmark = pytest.mark.gpu


def test_example_learns():
    path = Path(__file__).resolve().parents[1] / "examples" / "train_tokens.py"
    spec = importlib.util.spec_from_file_location("train_tokens", path)
    m = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(m)
    losses, right = m.main()
    assert losses[0] > 4.0 and losses[-1] < 0.1 and right == 1.0
