"""CPU tests of the token operators at their edges: that the GPU tests' shapes reach what they are for, and refusals."""
import ctypes

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


@pytest.mark.parametrize("sizes", [dict(q_len=0), dict(k_len=0), dict(batch=0)])
def test_side_arguments_of_no_tokens_may_be_null(sizes):
    """A tensor without elements has no address; the workspace call makes every check that does not need one."""
    lib, need = _lib.load(), ctypes.c_size_t()
    d = dict(batch=1, q_len=2, k_len=2, q=256, k=256, v=256, scale=1.0, slopes=256, q_heads=1, k_heads=1, dim=8, axes=1)
    for side in (dict(q_doc=256), dict(k_doc=256), dict(q_pos=256), dict(k_pos=256)):
        assert lib.wst_attention_workspace(_lib.AttentionDesc(**{**d, **sizes, **side}), 0, ctypes.byref(need)) == 0
        assert lib.wst_attention_workspace(_lib.AttentionDesc(**{**d, **side}), 0, ctypes.byref(need)) == 1
