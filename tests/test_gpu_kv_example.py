"""The drafted page of examples/drafted_page.py: the outputs of accepted drafts are those of the same tokens read one at a
time. Both ways attend the same quantised rows, except where the projections of a chunk and of single rows differ in
their last bits, which moves a value to the next of 16 levels now and then: 2e-2 of the largest output (a level is an
eighth of its block's largest value; a position's weight in 500 bounds what one such move does)."""
from __future__ import annotations

import importlib.util
from pathlib import Path

import pytest

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("prompt", [300, 1500])  # before the window slides, and long after
def test_drafted_page(ocr, prompt):
    spec = importlib.util.spec_from_file_location("drafted_page", Path(__file__).resolve().parent.parent / "examples" / "drafted_page.py")
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    assert mod.main(prompt, 12) <= 2e-2
