"""CPU tests of the token operators at their edges: that the GPU tests' shapes reach what they are for, and refusals."""
import pytest

import token_cases


@pytest.mark.parametrize("shape", token_cases.PARTS_WITHOUT_TILES)
def test_shapes_reach_parts_without_tiles(shape):
    assert token_cases.parts_without_tiles(*shape), shape
