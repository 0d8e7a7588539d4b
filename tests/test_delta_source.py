"""The matrix instructions' results must not be read by inline assembly: the compiler keeps the distance that such a reading
needs between its own instructions alone. No GPU needed."""
import os
import re

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "df-ssm_amd", "csrc")


@pytest.mark.parametrize("name", ["delta.hip", "delta_chunk.hip", "draw.hip"])
def test_no_instructions_in_assembly(name):
    """An empty template (a fence for the compiler) is allowed."""
    with open(os.path.join(CSRC, name)) as f:
        text = re.sub(r"//[^\n]*", "", f.read())
    found = re.findall(r'\basm\b\s*(?:volatile)?\s*\(\s*"([^"]*)"', text)
    assert [t for t in found if t.strip()] == []
