"""The projection, the loss, their gradients and the search in one program."""
from __future__ import annotations

import sys
from pathlib import Path

import pytest

sys.path.insert(0, str(Path(__file__).resolve().parent.parent / "examples"))


@pytest.mark.gpu
def test_training_brings_rows_of_a_class_together(cuda_ok):
    from train_search_rows import run

    got = run(rows=6000, classes=100, steps=60, batch=2048, report=lambda line: None)
    # 100 classes: unrelated neighbours agree in 1 of 100; noise of variance 4 in 112 of 128 directions hides them.
    assert got["before"] < 0.2
    assert got["last_loss"] < 0.5 * got["first_loss"]
    assert got["after"] > 0.6 and got["after"] > 3 * got["before"]
