"""The example that trains a token encoder through maxsim and serves it from an INT8 index."""
import importlib.util
from pathlib import Path

import pytest

pytestmark = pytest.mark.gpu


def test_train_token_encoder():
    at = Path(__file__).resolve().parent.parent / "examples" / "train_token_encoder.py"
    spec = importlib.util.spec_from_file_location("train_token_encoder", at)
    example = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(example)
    for bits in (8, 32):
        losses, top1, top10 = example.main(steps=60, bits=bits, say=lambda *_: None)
        # untrained the loss is that of chance, ln 64 = 4.2
        assert losses[0] > 3.5 and sum(losses[-5:]) / 5 < 1.5
        # by chance 1 in 256 and 10 in 256
        assert top1 > 0.5 and top10 > 0.8
