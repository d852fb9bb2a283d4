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


@pytest.mark.parametrize("kw", [dict(q_len=1 << 28, q_heads=8, k_heads=8), dict(q_len=1 << 27, dim=5), dict(q_len=1 << 27, dtype=1, causal=1)])
def test_more_threads_than_a_launch_holds_are_refused(kw):
    lib = _lib.load()
    d = dict(batch=1, q_len=2, k_len=300, q=256, k=256, v=256, scale=1.0, q_heads=8, k_heads=8, dim=8)
    d = _lib.AttentionDesc(**{**d, **kw})
    need = ctypes.c_size_t()
    assert lib.wst_attention_forward(d, 256, None, 256, 1 << 62, None) == 2
    assert b"too many rows" in lib.wst_tokens_last_error()
    assert lib.wst_attention_workspace(d, 1, ctypes.byref(need)) == 0
    g = _lib.AttentionGrads(o=256, d_o=256, lse=256, dq=256)
    assert lib.wst_attention_backward(d, g, 256, need.value, None) == 2
    assert b"too many rows" in lib.wst_tokens_last_error()


def test_backward_of_more_keys_than_a_launch_holds_is_refused():
    lib, need = _lib.load(), ctypes.c_size_t()
    d = _lib.AttentionDesc(batch=1, q_len=2, k_len=1 << 27, q=256, k=256, v=256, scale=1.0, q_heads=1, k_heads=1, dim=5)
    assert lib.wst_attention_workspace(d, 1, ctypes.byref(need)) == 0
    g = _lib.AttentionGrads(o=256, d_o=256, lse=256, dk=256)
    assert lib.wst_attention_backward(d, g, 256, need.value, None) == 2
    assert b"too many rows" in lib.wst_tokens_last_error()


def test_rotary_of_more_tokens_than_a_launch_holds_is_refused():
    lib = _lib.load()
    d = _lib.RotaryDesc(batch=1, tokens=1 << 30, base=1e4, q_heads=1, dim=64, axes=1, sections=(ctypes.c_int32 * 4)(32, 0, 0, 0))
    assert lib.wst_rotary(d, 256, 256, None, None, 256, None) == 2
    assert b"too many tokens" in lib.wst_tokens_last_error()
