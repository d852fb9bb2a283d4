"""CPU tests of the token operators: the oracle's gradients against differences, and what the library and the Python
entry points refuse before any GPU work."""
import ctypes

import pytest
import torch

import wst_amd  # noqa: F401
from oracle import token_ops as ref
from wst_amd import _lib, tokens

F64 = torch.float64


def _gen(seed):
    return torch.Generator().manual_seed(seed)


def _directional(f, x, d, h=1e-5):
    return (f(x + h * d) - f(x - h * d)) / (2 * h)


def test_oracle_layer_norm_gradients_match_differences():
    g = _gen(0)
    x, w, b, dy = (torch.randn(*s, generator=g, dtype=F64) for s in ((5, 7), (7,), (7,), (5, 7)))
    out = ref.layer_norm(x, w, b, 1e-5, F64, dy)
    loss = lambda x, w, b: (ref.layer_norm(x, w, b, 1e-5, F64)["y"][0] * dy).sum()   # noqa: E731
    for name, at, f in (("dx", x, lambda t: loss(t, w, b)), ("dw", w, lambda t: loss(x, t, b)),
                        ("db", b, lambda t: loss(x, w, t))):
        d = torch.randn(*at.shape, generator=g, dtype=F64)
        assert abs(_directional(f, at, d) - (out[name][0] * d).sum()) < 1e-7, name


def test_oracle_rotary_inverse_is_the_gradient():
    g = _gen(1)
    x, dy = torch.randn(2, 3, 2, 10, generator=g, dtype=F64), torch.randn(2, 3, 2, 10, generator=g, dtype=F64)
    pos = torch.randint(-50, 1000, (2, 3, 2), generator=g)
    y = ref.rotary(x, pos, (2, 2), 100.0, True)[0]
    dx = ref.rotary(dy, pos, (2, 2), 100.0, True, inverse=True)[0]
    assert abs((y * dy).sum() - (x * dx).sum()) < 1e-9          # linear: <A x, dy> = <x, A^T dy>


@pytest.mark.parametrize("cap,bias,causal,prefix,docs", [(0.0, False, False, None, False), (1.5, True, True, None, False),
                                                         (0.8, True, True, [2, 0], True)])
def test_oracle_attention_gradients_match_differences(cap, bias, causal, prefix, docs):
    g = _gen(2)
    B, Tq, Tk, H, Hk, D = 2, 5, 6, 4, 2, 3
    q, do = torch.randn(B, Tq, H, D, generator=g, dtype=F64), torch.randn(B, Tq, H, D, generator=g, dtype=F64)
    k, v = torch.randn(B, Tk, Hk, D, generator=g, dtype=F64), torch.randn(B, Tk, Hk, D, generator=g, dtype=F64)
    slopes = torch.rand(H, generator=g, dtype=F64) if bias else None
    kw = dict(cap=cap, causal=causal, prefix=None if prefix is None else torch.tensor(prefix))
    if docs:
        kw.update(q_documents=torch.tensor([0, 0, 1, -1, 1]), k_documents=torch.tensor([0, 0, 1, 1, -1, 1]))
    out = ref.attention(q, k, v, slopes=slopes, do=do, **kw)
    loss = lambda q, k, v, s: (ref.attention(q, k, v, slopes=s, **kw)["o"][0] * do).sum()   # noqa: E731
    checks = [("dq", q, lambda t: loss(t, k, v, slopes)), ("dk", k, lambda t: loss(q, t, v, slopes)),
              ("dv", v, lambda t: loss(q, k, t, slopes))]
    if bias:
        checks.append(("dslopes", slopes, lambda t: loss(q, k, v, t)))
    for name, at, f in checks:
        d = torch.randn(*at.shape, generator=g, dtype=F64)
        assert abs(_directional(f, at, d) - (out[name][0] * d).sum()) < 1e-7, name


def _norm(**kw):
    d = dict(batch=1, points=2, n=8, x_stride_batch=0, x_stride_point=8, x_stride_n=1, dx_stride_batch=0,
             dx_stride_point=8, dx_stride_n=1, x_dtype=0, y_dtype=0, w_dtype=0, eps=1e-5)
    d.update(kw)
    return _lib.NormDesc(**d)


@pytest.mark.parametrize("kw,code", [
    (dict(n=0), 1), (dict(points=-1), 1), (dict(x_dtype=7), 1), (dict(eps=-1.0), 1), (dict(eps=float("nan")), 1),
    (dict(x_stride_n=3, x_stride_point=5), 1), (dict(batch=1 << 20, points=1 << 20), 2), (dict(n=1 << 40), 2)])
def test_layer_norm_refusals(kw, code):
    lib = _lib.load()
    assert lib.wst_layer_norm_forward(_norm(**kw), 256, None, None, 256, None, None, None) == code
    assert b"layer norm" in lib.wst_tokens_last_error()


def test_layer_norm_pointer_refusals():
    lib = _lib.load()
    d, need = _norm(), ctypes.c_size_t()
    assert lib.wst_layer_norm_forward(None, 256, None, None, 256, None, None, None) == 1
    assert lib.wst_layer_norm_forward(d, None, None, None, 256, None, None, None) == 1
    assert lib.wst_layer_norm_forward(d, 256, None, None, 256, 256, None, None) == 1
    assert lib.wst_layer_norm_workspace(d, None) == 1
    assert lib.wst_layer_norm_workspace(d, ctypes.byref(need)) == 0 and need.value > 0
    assert lib.wst_layer_norm_backward(d, 256, None, 256, 256, 256, 256, None, None, 256, need.value - 1, None) == 1
    assert b"workspace" in lib.wst_tokens_last_error()
    assert lib.wst_layer_norm_backward(d, 256, None, 256, 256, 256, 256, None, None, None, 1 << 20, None) == 1
    assert lib.wst_layer_norm_backward(_norm(dx_stride_n=4), 256, None, 256, 256, 256, 256, None, None, 256, 1 << 20,
                                       None) == 1
    # nothing to do: no launch
    assert lib.wst_layer_norm_forward(_norm(points=0), None, None, None, None, None, None, None) == 0


def _rot(**kw):
    d = dict(batch=1, tokens=1, base=10000.0, q_heads=1, k_heads=0, dim=8, dtype=0, axes=2,
             sections=(ctypes.c_int32 * 4)(1, 1, 0, 0))
    d.update(kw)
    return _lib.RotaryDesc(**d)


@pytest.mark.parametrize("kw,code", [
    (dict(dim=0), 1), (dict(tokens=-1), 1), (dict(dtype=3), 1), (dict(axes=0), 1), (dict(axes=5), 1), (dict(base=0.0), 1),
    (dict(base=float("inf")), 1), (dict(sections=(ctypes.c_int32 * 4)(3, 2, 0, 0)), 1),
    (dict(sections=(ctypes.c_int32 * 4)(-1, 2, 0, 0)), 1), (dict(dim=1024, sections=(ctypes.c_int32 * 4)(100, 100, 0, 0)), 2)])
def test_rotary_refusals(kw, code):
    lib = _lib.load()
    assert lib.wst_rotary(_rot(**kw), 256, 256, None, None, 256, None) == code
    assert b"rotary" in lib.wst_tokens_last_error()


def test_rotary_pointer_refusals():
    lib = _lib.load()
    assert lib.wst_rotary(None, 256, 256, None, None, 256, None) == 1
    assert lib.wst_rotary(_rot(), 256, None, None, None, 256, None) == 1
    assert lib.wst_rotary(_rot(k_heads=1), 256, 256, None, None, 256, None) == 1
    assert lib.wst_rotary(_rot(), 256, 256, None, None, None, None) == 1
    assert lib.wst_rotary(_rot(tokens=0), None, None, None, None, None, None) == 0


def _attn(**kw):
    d = dict(batch=1, q_len=2, k_len=2, q=256, k=256, v=256, scale=1.0, cap=0.0, q_heads=2, k_heads=1, dim=8, dtype=0)
    d.update(kw)
    return _lib.AttentionDesc(**d)


@pytest.mark.parametrize("kw,code", [
    (dict(q_len=-1), 1), (dict(q_heads=3, k_heads=2), 1), (dict(k_heads=0), 1), (dict(dim=0), 1), (dict(dim=257), 2),
    (dict(dtype=9), 1), (dict(scale=float("inf")), 1), (dict(cap=-1.0), 1), (dict(cap=float("nan")), 1),
    (dict(q_pos=256), 1), (dict(k_doc=256), 1), (dict(q_pos=256, k_pos=256, axes=0), 1),
    (dict(q_pos=256, k_pos=256, axes=5), 1), (dict(prefix=256), 1), (dict(batch=70000), 2), (dict(k_len=1 << 31), 2),
    (dict(q=None), 1), (dict(v=None), 1)])
def test_attention_refusals(kw, code):
    lib = _lib.load()
    ws = torch.empty(1 << 16, dtype=torch.uint8)
    assert lib.wst_attention_forward(_attn(**kw), 256, None, ws.data_ptr(), ws.numel(), None) == code
    assert b"attention" in lib.wst_tokens_last_error()


def test_attention_pointer_refusals():
    lib = _lib.load()
    need = ctypes.c_size_t()
    d = _attn(slopes=256)
    assert lib.wst_attention_forward(None, 256, None, None, 0, None) == 1
    assert lib.wst_attention_forward(d, None, None, None, 0, None) == 1
    assert lib.wst_attention_workspace(d, 1, None) == 1
    assert lib.wst_attention_workspace(d, 1, ctypes.byref(need)) == 0 and need.value > 0
    g = _lib.AttentionGrads(o=256, d_o=256, lse=256, dq=256)
    assert lib.wst_attention_backward(d, None, 256, need.value, None) == 1
    assert lib.wst_attention_backward(d, g, 256, need.value - 1, None) == 1
    assert lib.wst_attention_backward(d, g, None, need.value, None) == 1
    assert lib.wst_attention_backward(d, _lib.AttentionGrads(o=256, d_o=256), 256, need.value, None) == 1
    assert lib.wst_attention_backward(_attn(), _lib.AttentionGrads(o=256, d_o=256, lse=256, dslopes=256), 256, 1 << 20,
                                      None) == 1
    assert lib.wst_attention_backward(_attn(k_len=0), g, 256, 1 << 20, None) == 1
    assert lib.wst_attention_forward(_attn(batch=0), None, None, None, 0, None) == 0


def test_python_entry_points_refuse_cpu_tensors():
    x = torch.zeros(2, 3, 2, 8)
    pos = torch.zeros(3, 1, dtype=torch.int32)
    for call in (lambda: tokens.layer_norm(x), lambda: tokens.rotary(x, pos, (2,)), lambda: tokens.attention(x, x, x)):
        with pytest.raises(RuntimeError):
            call()
    with pytest.raises(TypeError):
        tokens.layer_norm([1.0])


def test_grid_positions_order():
    p = tokens.grid_positions(2, 3, 4)
    assert p.shape == (24, 3) and p.dtype == torch.int32
    assert p[0].tolist() == [0, 0, 0] and p[1].tolist() == [0, 0, 1] and p[4].tolist() == [0, 1, 0] and p[12].tolist() == [1, 0, 0]


@pytest.mark.parametrize("shape,permute,view", [
    ((4, 6), None, (1, 4, 6, 0, 6, 1)), ((2, 3, 6), None, (1, 6, 6, 0, 6, 1)),
    ((2, 6, 5), (0, 2, 1), (2, 5, 6, 30, 1, 5)), ((6, 5), (1, 0), (1, 5, 6, 0, 1, 5)), ((6,), None, (1, 1, 6, 0, 6, 1))])
def test_token_view(shape, permute, view):
    x = torch.zeros(shape)
    x = x if permute is None else x.permute(permute)
    t, got = tokens._token_view(x)
    assert tuple(got) == view and t.data_ptr() == x.data_ptr()


def test_token_view_copies_what_it_cannot_read():
    x = torch.zeros(2, 3, 4, 5)[:, ::2, :, ::2]
    t, got = tokens._token_view(x)
    assert t.is_contiguous() and tuple(got) == (1, 16, 3, 0, 3, 1)


@pytest.mark.parametrize("sizes", [dict(batch=0), dict(q_len=0), dict(k_len=0), dict(q_len=0, k_len=0), dict()])
@pytest.mark.parametrize("dim", [8, 5, 128])
def test_attention_workspace_of_empty_sizes(sizes, dim):
    lib, need = _lib.load(), ctypes.c_size_t(1)
    for backward in (0, 1):
        assert lib.wst_attention_workspace(_attn(dim=dim, slopes=256, **sizes), backward, ctypes.byref(need)) == 0


def test_packed_descriptors_match_the_structures():
    for pack, kind in ((_lib.NORM_PACK, _lib.NormDesc), (_lib.ROTARY_PACK, _lib.RotaryDesc),
                       (_lib.ATTENTION_PACK, _lib.AttentionDesc), (_lib.GRADS_PACK, _lib.AttentionGrads)):
        assert pack.size == ctypes.sizeof(kind), kind
    d = _lib.AttentionDesc.from_buffer_copy(_lib.ATTENTION_PACK.pack(*range(1, 31), 0.5, 2.0, *range(32, 38)))
    assert (d.batch, d.k_len, d.v_strides[2], d.k_doc_stride, d.q, d.prefix, d.o_rest, d.scale, d.q_heads, d.causal) == (
        1, 3, 12, 19, 20, 29, 30, 0.5, 32, 37)
    r = _lib.RotaryDesc.from_buffer_copy(_lib.ROTARY_PACK.pack(*range(1, 15), 0.25, *range(16, 28)))
    assert (r.tokens, r.k_out_strides[2], r.base, r.q_heads, r.sections[0], r.positions_shared) == (2, 14, 0.25, 16, 21, 27)


def test_scattering_attention_refusals_and_parameters():
    from wst_amd.torch import ScatteringAttention
    m = ScatteringAttention(2, (32, 32), channels=3, heads=4, dim=32, key_heads=2)
    assert {k: tuple(v.shape) for k, v in m.state_dict().items()} == {
        "norm_weight": (243,), "norm_bias": (243,), "qkv.weight": (256, 243), "slopes": (4,), "pool_kv.weight": (128, 128),
        "pool_query": (4, 32)}
    assert m.sections == (5, 6, 5) and m.slopes.dtype == torch.float32
    for kw, error in ((dict(heads=3, key_heads=2), RuntimeError), (dict(dim=0), RuntimeError), (dict(dim=257), RuntimeError),
                      (dict(dtype=torch.float64), TypeError), (dict(dim=8, sections=(2, 2, 1)), RuntimeError),
                      (dict(sections=(2, 2)), RuntimeError), (dict(J=6), RuntimeError), (dict(channels=0), RuntimeError)):
        with pytest.raises(error):
            ScatteringAttention(**{"J": 2, "shape": (32, 32), **kw})
    x = torch.rand(2, 3, 32, 32)
    with pytest.raises(TypeError):
        m(x.numpy())
    for bad in (x[0], x[:, :2], x[None, None]):
        with pytest.raises(RuntimeError):
            m(bad)
    with pytest.raises(TypeError):
        m(x, torch.zeros(2, 1))
    with pytest.raises(RuntimeError):
        m(x, torch.zeros(2, 3, dtype=torch.int32))
    for count in (0, 2):
        with pytest.raises(RuntimeError):
            m.pooled(x, count=count)
    if not torch.cuda.is_available():
        with pytest.raises(RuntimeError, match="no ROCm GPU"):
            m(x)
        from wst_amd import features
        with pytest.raises(RuntimeError, match="no ROCm GPU"):
            features.extract_wst_tokens_batch(x)
