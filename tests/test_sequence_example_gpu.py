"""The example layer on the sequence operators: it learns, and serving in parts
gives what whole sequences give."""
import importlib.util
from pathlib import Path

import pytest

pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


def load():
    path = Path(__file__).resolve().parent.parent / "examples" / "sequence_mixer.py"
    spec = importlib.util.spec_from_file_location("sequence_mixer", path)
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    return mod


def test_training_lowers_the_loss():
    losses = load().train(width=256, heads=4, kv_heads=2, tokens=600, steps=12)
    assert all(b < a for a, b in zip(losses, losses[1:])), losses
    assert losses[-1] < 0.9 * losses[0], losses


def test_prompts_and_tokens_agree_with_whole_sequences():
    # outputs of bf16 rows: two roundings of 2^-9 on either side, and sums of 256 such values
    # through the last projection; the largest of some 400,000 differences lies at five sigma
    assert load().serve(width=256, heads=4, kv_heads=2, lengths=[300, 1, 129], new=5) <= 5 * 4 * 2.0 ** -9
