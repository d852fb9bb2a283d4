"""CPU tests of the token operators at their edges: that the GPU tests' shapes reach what they are for, and refusals."""
import pytest

import token_cases
import wst_amd  # noqa: F401
from wst_amd import _lib


@pytest.mark.parametrize("shape", token_cases.PARTS_WITHOUT_TILES)
def test_shapes_reach_parts_without_tiles(shape):
    assert token_cases.parts_without_tiles(*shape), shape


@pytest.mark.parametrize("cap,code", [(9e-31, 1), (2e30, 1), (3e38, 1), (-1e-3, 1)])
def test_caps_beyond_the_range_are_refused(cap, code):
    lib = _lib.load()
    d = _lib.AttentionDesc(batch=1, q_len=2, k_len=2, q=256, k=256, v=256, scale=1.0, cap=cap, q_heads=1, k_heads=1, dim=8)
    assert lib.wst_attention_forward(d, 256, None, 256, 1 << 16, None) == code
    assert b"cap" in lib.wst_tokens_last_error()
