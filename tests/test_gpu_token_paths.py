"""GPU tests of the paths that use the token operators together: features.extract_wst_tokens_batch and
torch.ScatteringAttention, against a plain float64 network on the maps that the transform made."""
import pytest
import torch

import wst_amd  # noqa: F401
from wst_amd import features
from wst_amd.torch import ScatteringAttention, Scattering2D

pytestmark = pytest.mark.gpu

F32, BF16, F16, F64 = torch.float32, torch.bfloat16, torch.float16, torch.float64


def _gen(seed):
    return torch.Generator().manual_seed(seed)


def _norm(x, w, b):
    mu = x.mean(-1, keepdim=True)
    return (x - mu) / ((x - mu).square().mean(-1, keepdim=True) + 1e-5).sqrt() * w + b


def _turn(x, places, sections, base):
    P, out, p = sum(sections), x.clone(), 0
    for axis, s in enumerate(sections):
        for i in range(s):
            ang = places[:, axis].to(F64) * base ** (-i / s)
            c, n = ang.cos()[:, None], ang.sin()[:, None]
            out[..., p] = x[..., p] * c - x[..., p + P] * n
            out[..., p + P] = x[..., p + P] * c + x[..., p] * n
            p += 1
    return out


def _attend(q, k, v, bias, cap, see):
    """q (B, Tq, H, D), k, v (B, Tk, Hk, D), bias (H, Tq, Tk) or None, see (B, Tq, Tk)."""
    g = q.shape[2] // k.shape[2]
    k, v = k.repeat_interleave(g, 2), v.repeat_interleave(g, 2)
    z = (q.transpose(1, 2) @ k.permute(0, 2, 3, 1)) * q.shape[-1] ** -0.5
    if cap:
        z = cap * torch.tanh(z / cap)
    if bias is not None:
        z = z + bias
    z = z.masked_fill(~see[:, None], float("-inf"))
    some = see.any(-1)[:, None, :, None]
    p = torch.softmax(torch.where(some, z, 0.0), -1).masked_fill(~some, 0.0)
    return (p @ v.transpose(1, 2)).transpose(1, 2)


class _Plain:
    """The module's formulas in float64, on leaves that are copies of its parameters."""

    def __init__(self, m):
        self.m = m
        self.leaves = {n: p.detach().cpu().to(F64).requires_grad_() for n, p in m.named_parameters()}

    def tokens(self, S, documents):
        m, w = self.m, self.leaves
        B, F, C, K, Mo, No = S.shape
        x = S.cpu().to(F64).reshape(B, F, C * K, Mo * No).transpose(2, 3).reshape(B, F * Mo * No, C * K)
        x = _norm(x, w["norm_weight"], w["norm_bias"])
        T = x.shape[1]
        y = (x @ w["qkv.weight"].T).reshape(B, T, -1, m.dim)
        q, k, v = y.split((m.heads, m.key_heads, m.key_heads), 2)
        f, r, c = torch.meshgrid(torch.arange(F), torch.arange(Mo), torch.arange(No), indexing="ij")
        places = torch.stack((f, r, c), -1).reshape(T, 3)
        q, k = (_turn(t, places, m.sections, m.base) for t in (q, k))
        away = (places[:, None] - places[None]).abs().sum(-1)
        doc = torch.zeros(B, T) if documents is None else documents.cpu().repeat_interleave(Mo * No, 1)
        self.doc = doc
        see = (doc[:, :, None] == doc[:, None]) & (doc[:, :, None] >= 0)
        return _attend(q, k, v, -w["slopes"][:, None, None] * away, m.cap, see).reshape(B, T, -1)

    def pooled(self, S, documents, count):
        m, w = self.m, self.leaves
        x = self.tokens(S, documents)
        B, T = x.shape[:2]
        k, v = (x @ w["pool_kv.weight"].T).reshape(B, T, -1, m.dim).split((m.key_heads, m.key_heads), 2)
        self.pool = [float(t.detach().norm(dim=-1).max()) for t in (k, v)]
        see = self.doc[:, None] == torch.arange(count)[None, :, None]
        return _attend(w["pool_query"].expand(B, count, -1, -1), k, v, None, 0.0, see).reshape(B, count, -1)


def _maps(m, images):
    x = images if images.dim() == 5 else images.unsqueeze(1)
    return Scattering2D(m.transform.J, m.transform.shape, m.transform.L, m.transform.max_order)(x.contiguous())


def _module(seed, **kw):
    torch.manual_seed(seed)
    m = ScatteringAttention(**kw).cuda()
    with torch.no_grad():
        m.norm_weight += 0.2 * torch.randn_like(m.norm_weight)
        m.norm_bias += 0.2 * torch.randn_like(m.norm_bias)
    return m


@pytest.mark.parametrize("out_dtype", [None, BF16, F16])
@pytest.mark.parametrize("B,C,size,J,L,order", [(2, 3, 32, 2, 8, 2), (1, 1, 64, 4, 8, 2), (3, 4, 32, 2, 6, 1)])
def test_extract_wst_tokens_batch(B, C, size, J, L, order, out_dtype):
    """Against the plain norm of the transform's own maps. Rounding: the statistics and the value's three operations in
    float32, each within 2^-24 of a magnitude up to the row's largest, and the last rounding to out_dtype."""
    x = torch.rand(B, C, size, size, generator=_gen(B + size)).cuda()
    S = Scattering2D(J, (size, size), L, order)(x)
    n = C * S.shape[2]
    w = (1 + 0.3 * torch.randn(n, generator=_gen(1))).cuda().requires_grad_()
    b = torch.randn(n, generator=_gen(2)).cuda().requires_grad_()
    y = features.extract_wst_tokens_batch(x, J, L, order, w, b, out_dtype=out_dtype)
    want = _norm(S.cpu().to(F64).reshape(B, n, -1).transpose(1, 2), w.detach().cpu().to(F64), b.detach().cpu().to(F64))
    dtype = F32 if out_dtype is None else out_dtype
    assert y.dtype == dtype and y.shape == want.shape and y.is_contiguous()
    got = y.detach().cpu().to(F64)
    # the mean and the variance each lose at most 8 + log2(n) roundings of the row's magnitude, which the norm scales to
    # at most sqrt(n); w is below 3 here
    bound = 3 * n ** 0.5 * (16 + 2 * torch.tensor(float(n)).log2()) * 2.0 ** -24 + want.abs() * torch.finfo(dtype).eps / 2
    assert bool(((got - want).abs() <= bound).all())
    dw, db = torch.autograd.grad(y.float().sum(), (w, b))
    assert dw.shape == (n,) and torch.equal(db.cpu(), torch.full((n,), float(want.shape[0] * want.shape[1])))
    with torch.no_grad():
        assert torch.equal(features.extract_wst_tokens_batch(x.cpu().numpy(), J, L, order, w, b, out_dtype=out_dtype), y)


CASES = {
    "one image": (dict(J=2, shape=(32, 32), channels=3, heads=4, dim=32), (2, 3, 32, 32), None),
    "shared keys, order 1, no cap": (dict(J=2, shape=(32, 32), channels=1, heads=4, dim=24, key_heads=2, max_order=1, cap=0.0,
                                          sections=(0, 3, 5)), (1, 1, 32, 32), None),
    "series": (dict(J=3, shape=(32, 32), channels=2, heads=2, dim=64, key_heads=1, L=6), (2, 3, 2, 32, 32), None),
    "series packed": (dict(J=2, shape=(16, 16), channels=2, heads=2, dim=20, L=4, cap=2.0), (2, 5, 2, 16, 16),
                      [[0, 0, 1, 1, -1], [1, -1, 1, 1, 1]]),
}


@pytest.mark.parametrize("name", CASES)
def test_scattering_attention_and_gradients(name):
    """Values and the gradients of every parameter, in float32. Every product sums at most n = 486 terms (n roundings of
    2^-24, 2.9e-5), scores pass through exp, so their error of at most n 2^-24 max|z| joins relatively with max|z| below
    8 here; the two layers and their backward passes chain four such steps: 1e-3 of the largest value holds it all.

    The gradient of pool_query needs more: it is sum_b sum_j ds_j k_j scale with ds_j = p_j (dp_j - sum_i p_i dp_i), whose
    terms cancel where the keys are alike (sum_j ds_j = 0; tokens of one image are).  v has lost up to n 2^-24 |v|, so each
    of dp_j = do.v_j and their mean up to e = n 2^-24 |do| |v|, and with sum_j p_j = 1 the gradient up to
    B scale 2 e |k|, however small it is itself."""
    kw, shape, doc = CASES[name]
    m = _module(3, **kw)
    images = torch.rand(*shape, generator=_gen(5)).cuda()
    documents = None if doc is None else torch.tensor(doc, dtype=torch.int32).cuda()
    count = 1 if doc is None else 3                       # series 2 has no frames
    plain = _Plain(m)
    S = _maps(m, images)
    for got, want in ((m(images, documents), plain.tokens(S, documents)),
                      (m.pooled(images, documents, count), plain.pooled(S, documents, count))):
        assert got.shape == want.shape and got.dtype == F32
        assert float((got.detach().cpu().to(F64) - want.detach()).abs().max()) <= 1e-3 * float(want.detach().abs().max())
        do = torch.randn(want.shape, generator=_gen(6), dtype=F64)
        m.zero_grad()
        got.backward(do.float().cuda())
        names = [n for n, p in m.named_parameters() if p.grad is not None]
        want_g = torch.autograd.grad(want, [plain.leaves[n] for n in names], do)
        for n, w in zip(names, want_g):
            g = dict(m.named_parameters())[n].grad.cpu().to(F64)
            lost = 0.0
            if n == "pool_query":
                reach = float(do.reshape(*do.shape[:2], m.heads, m.dim).norm(dim=-1).max())
                lost = len(do) * m.dim ** -0.5 * 2 * (486 * 2.0 ** -24 * reach * plain.pool[1]) * plain.pool[0]
            assert float((g - w).abs().max()) <= 1e-3 * float(w.abs().max()) + lost, n
    assert {"pool_query", "pool_kv.weight", "qkv.weight", "slopes", "norm_weight", "norm_bias"} == set(names)
    if doc is not None:
        assert not bool(m.pooled(images, documents, count)[:, 2].any())
        assert not bool(m(images, documents).reshape(2, 5, -1)[documents.cpu() < 0].any())


def test_scattering_attention_padding_frames_and_types():
    """Frames of no series change nothing, whatever they hold; the module in 16 bits; CPU images reach its device."""
    kw = dict(J=2, shape=(16, 16), channels=2, heads=2, dim=32, L=4)
    doc = torch.tensor([[0, 0, -1]], dtype=torch.int32).cuda()
    x = torch.rand(1, 3, 2, 16, 16, generator=_gen(8)).cuda()
    for dtype in (F32, BF16, F16):
        m = _module(9, dtype=dtype, **kw)
        y = m.pooled(x, doc)
        assert y.dtype == dtype
        bad = x.clone()
        bad[:, 2] = float("nan")
        assert torch.equal(m.pooled(bad, doc), y)
        # the same without the padding, up to the order of sums over other tiles: a few steps of the type
        close = m.pooled(x[:, :2])
        assert float((close - y).detach().abs().max()) <= 16 * torch.finfo(dtype).eps * float(y.detach().abs().max())
        assert torch.equal(m.pooled(x.cpu(), doc), y)
        m.pooled(x, doc).float().square().sum().backward()
        assert all(p.grad is not None and bool(torch.isfinite(p.grad).all()) for p in m.parameters())


def test_scattering_attention_without_images():
    m = _module(1, J=2, shape=(16, 16), channels=1, heads=1, dim=8, L=4)
    assert m(torch.empty(0, 1, 16, 16).cuda()).shape == (0, 16, 8)
    assert m.pooled(torch.empty(0, 1, 16, 16).cuda()).shape == (0, 1, 8)


def test_scattering_attention_captured():
    """A training step captured: forward and backward replay with new images, and eager work between."""
    m = _module(2, J=2, shape=(32, 32), channels=3, heads=4, dim=32, dtype=BF16)
    x = torch.rand(4, 3, 32, 32, generator=_gen(1)).cuda()
    params = list(m.parameters())

    def step():
        return torch.autograd.grad(m.pooled(x).float().square().mean(), params)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = step()
    for seed in (11, 12, 13):
        x.copy_(torch.rand(4, 3, 32, 32, generator=_gen(seed)))
        want = [t.clone() for t in step()]
        g.replay()
        torch.cuda.synchronize()
        for a, b, p in zip(out, want, params):
            assert torch.equal(a, b), tuple(p.shape)
