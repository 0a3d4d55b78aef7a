"""The guide's serving example is the one that the tests run."""
from pathlib import Path

import pytest

from tests.serving_example import FORK, REST, SETUP, STEP

GUIDES = sorted(Path(__file__).resolve().parent.parent.glob("*.md"))


@pytest.mark.skipif(not GUIDES, reason="a tree without its documents")
def test_the_guide_shows_what_the_tests_run():
    blocks = [b.split("```")[0] for g in GUIDES for b in g.read_text().split("```python")[1:]]
    shown = [b for b in blocks if "rt.tree_verify(" in b]
    assert len(shown) == 1
    assert shown[0].strip() == "".join((SETUP, STEP, FORK, REST)).strip()
