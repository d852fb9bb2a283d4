"""GPU tests of the token operators at their edges, against the float64 restatement (oracle/token_ops.py)."""
import pytest
import torch
from torch.autograd import forward_ad

import token_cases
import wst_amd  # noqa: F401
from oracle import token_ops as ref
from test_gpu_tokens import BF16, F16, F32, _attention_inputs, _check_attention, _documents, _gen, _hold, _norm_inputs
from wst_amd import tokens
from wst_amd.torch import ScatteringAttention

pytestmark = pytest.mark.gpu


def _out_of_the_caches():
    """Writes more than the caches hold, so that what comes next is fetched from memory."""
    torch.empty(1 << 29, dtype=torch.uint8, device="cuda").fill_(1)


def _key_gradients(q, k, v, do, want, **kw):
    """dk and dv alone, keys and values first read by the kernel that sums them, several times."""
    leaves, dev = [t.cuda().requires_grad_() for t in (k, v)], {n: t.cuda() if torch.is_tensor(t) else t for n, t in kw.items()}
    q, do, first = q.cuda(), do.cuda(), None
    for _ in range(4):
        o = tokens.attention(q, *leaves, **dev)
        _out_of_the_caches()
        got = torch.autograd.grad(o, leaves, do)
        if first is None:
            first = got
            _hold(got[0], want["dk"], "dk")
            _hold(got[1], want["dv"], "dv")
        assert all(torch.equal(a, b) for a, b in zip(got, first))


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("B,T,H,Hk,D", token_cases.PARTS_WITHOUT_TILES)
def test_attention_parts_without_tiles(B, T, H, Hk, D, dtype):
    """The last keys in order have fewer tiles of queries than there are parts: a part without one adds nothing."""
    q, k, v, do, _ = _attention_inputs(B, T, T, H, Hk, D, dtype, T + D)
    _key_gradients(q, k, v, do, ref.attention(q, k, v, do=do, causal=True), causal=True)


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("D", [96, 128])
def test_attention_documents_that_no_query_has(D, dtype):
    q, k, v, do, _ = _attention_inputs(2, 300, 700, 4, 2, D, dtype, D)
    docs = torch.zeros(2, 700, dtype=torch.int32)
    docs[:, 128:384] = 5                                    # two blocks of keys whose document no query has
    docs[1, 400:] = 9
    kw = dict(q_documents=torch.zeros(2, 300, dtype=torch.int32), k_documents=docs)
    want = ref.attention(q, k, v, do=do, **kw)
    assert not bool(want["dv"][0][:, 128:384].any())
    _key_gradients(q, k, v, do, want, **kw)


CAPS = [1e-30, 1e-2, 50.0, 64.0, 65.0, 1e3, 1e6, 1e30]


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("D", [64, 128, 12])
@pytest.mark.parametrize("cap", CAPS)
def test_attention_caps_of_any_size(cap, D, dtype):
    """The cap's error is one of the score, not of the cap: a large cap is no cap, a small one takes the scores away."""
    q, k, v, do, g = _attention_inputs(1, 200, 200, 4, 2, D, dtype, 41, gain=4.0)
    slopes = torch.rand(4, generator=g) * 0.1
    pos = torch.randint(-20, 20, (1, 200, 2), generator=g, dtype=torch.int32)
    docs = _documents(g, 1, 200, 3)
    for kw in (dict(), dict(slopes=slopes, causal=True), dict(scale=-0.2, slopes=slopes, q_positions=pos, k_positions=pos),
               dict(q_documents=docs, k_documents=docs)):
        o, _ = _check_attention(q, k, v, do, cap=cap, **kw)
    if cap == 1e30:
        want = ref.attention(q, k, v, **kw)
        _hold(o, want["o"], "no cap")


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("cap", CAPS)
def test_attention_caps_of_any_size_few_queries(cap, dtype):
    q, k, v, do, g = _attention_inputs(2, 2, 1500, 4, 2, 64, dtype, 42, gain=4.0)
    lengths = torch.tensor([1500, 700], dtype=torch.int32)
    for kw in (dict(), dict(k_lengths=lengths, slopes=torch.rand(4, generator=g) * 0.01)):
        _check_attention(q, k, v, do, train=False, cap=cap, **kw)


def _calls():
    """Each operator on its differentiable arguments: (call, arguments)."""
    x, w = torch.randn(2, 5, 2, 8, device="cuda"), torch.ones(8, device="cuda")
    pos, slopes = torch.arange(5, dtype=torch.int32, device="cuda")[:, None], torch.ones(2, device="cuda")
    return [(lambda x, w, b: tokens.layer_norm(x, w, b), (x, w, w.clone())),
            (lambda q, k: torch.cat(tokens.rotary(q, pos, (4,), k=k)), (x, x.clone())),
            (lambda q, k, v, s: tokens.attention(q, k, v, slopes=s), (x, x.clone(), x.clone(), slopes))]


def test_forward_mode_is_refused():
    """A tangent on any argument: without gradients too, and in either spelling."""
    for call, args in _calls():
        for n, t in enumerate(args):
            for leaf in (t, t.clone().requires_grad_()):
                with forward_ad.dual_level(), pytest.raises(RuntimeError, match="forward-mode"):
                    call(*args[:n], forward_ad.make_dual(leaf, torch.ones_like(t)), *args[n + 1:])
            with pytest.raises(RuntimeError):
                torch.func.jvp(lambda u: call(*args[:n], u, *args[n + 1:]), (t,), (torch.ones_like(t),))
        with forward_ad.dual_level():
            assert torch.equal(call(*args), call(*args))        # a level without tangents takes nothing away


def test_tracing_is_refused():
    for call, args in _calls():
        with pytest.raises(RuntimeError, match="traced"):
            torch.jit.trace(call, args)
        for transform in (torch.func.vmap(call, (0,) + (None,) * (len(args) - 1)), torch.func.grad(lambda *a: call(*a).sum())):
            with pytest.raises(RuntimeError):
                transform(*args)


@pytest.mark.parametrize("B,Tq,Tk", [(2, 3, 0), (2, 70, 0), (2, 0, 5), (2, 0, 0), (0, 3, 5), (0, 3, 0)])
@pytest.mark.parametrize("D", [8, 5])
def test_attention_of_no_tokens_with_documents_and_positions(B, Tq, Tk, D):
    """An empty store of keys, or an empty batch, takes the arguments that a full one takes."""
    ints = lambda *s: torch.zeros(*s, dtype=torch.int32, device="cuda")   # noqa: E731
    leaves = [torch.randn(B, t, h, D, device="cuda", requires_grad=True) for t, h in ((Tq, 2), (Tk, 1), (Tk, 1))]
    slopes = torch.ones(2, device="cuda", requires_grad=True)
    for batched in (True, False):
        side = {f"{n}_{what}": ints(*((B, t) if batched or n == "q" else (t,)), *a)
                for n, t in (("q", Tq), ("k", Tk)) for what, a in (("documents", ()), ("positions", (2,)))}
        o, lse = tokens.attention(*leaves, slopes=slopes, k_lengths=ints(B), return_lse=True, causal=True, **side)
        assert o.shape == (B, Tq, 2, D) and not bool(o.any()) and bool((lse == -torch.inf).all())
        for t in torch.autograd.grad(o, [*leaves, slopes], torch.ones_like(o)):
            assert not bool(t.any())


@pytest.mark.parametrize("rows,n,layout", [((1 << 26) + 7, 2, "rows"), ((1 << 23) + 5, 3, "maps"), ((1 << 22) + 3, 650, "maps")])
def test_layer_norm_of_more_rows_than_a_launch_holds(rows, n, layout):
    """A launch has fewer than 2^32 threads; these calls need more. Rows of the first and the last launch are checked, and
    between them rows of zeros, whose result is the bias; the weight's gradient comes from the checked rows alone."""
    points = 1 if layout == "rows" else 2                       # maps of two points
    ends = 4 // points
    x, w, b, dy = _norm_inputs(2 * ends * points, n, BF16, F32, n)
    dy = dy.to(BF16)
    want = ref.layer_norm(x, w, b, 1e-5, BF16, dy)
    at = lambda t: torch.cat((t[:ends], t[-ends:])).reshape(-1, n)   # noqa: E731
    if layout == "rows":
        xs = torch.zeros(rows, n, dtype=BF16, device="cuda")
    else:
        xs = torch.zeros(rows, n, points, dtype=BF16, device="cuda").transpose(1, 2)
    xs[:ends], xs[-ends:] = x.cuda().reshape(2 * ends, *xs.shape[1:]).split(ends)
    xs.requires_grad_()
    ws, bs = w.cuda().requires_grad_(), b.cuda().requires_grad_()
    y = tokens.layer_norm(xs, ws, bs)
    _hold(at(y), want["y"], "y")
    plain = b.cuda().to(BF16)
    for part in y.detach()[ends:-ends].split(1 << 20):
        assert bool((part == plain).all())
    dys = torch.zeros(y.shape, dtype=BF16, device="cuda")
    dys[:ends], dys[-ends:] = dy.cuda().reshape(2 * ends, *xs.shape[1:]).split(ends)
    dx, dw, db = torch.autograd.grad(y, (xs, ws, bs), dys)
    _hold(at(dx), want["dx"], "dx")
    _hold(dw, want["dw"], "dw")
    _hold(db, want["db"], "db")
    for part in dx[ends:-ends].split(1 << 20):
        assert not bool(part.any())


def test_views_that_negate_when_read():
    """The imaginary part of a conjugate holds the number's own, and a flag; gradients may come as such views too."""
    x = torch.randn(2, 6, 2, 8, device="cuda")
    pos, slopes = torch.arange(6, dtype=torch.int32, device="cuda")[:, None], torch.ones(2, device="cuda")
    calls = [lambda x: tokens.layer_norm(x), lambda x: tokens.layer_norm(x[0, 0, 0]),
             lambda x: tokens.layer_norm(x, x[0, 0, 0], x[0, 0, 1]), lambda x: torch.cat(tokens.rotary(x, pos, (4,), k=x)),
             lambda x: tokens.attention(x, x, x, slopes=x[0, 0, :, 0])]
    imag = torch.complex(torch.zeros_like(x), x).conj().imag
    for view, value in ((imag, -x), (torch._neg_view(x), -x)):
        assert view.is_neg() and torch.equal(view, value)
        for n, call in enumerate(calls):
            assert torch.equal(call(view), call(value)), n
            leaf = value.clone().requires_grad_()
            y = call(leaf)
            dy = torch.randn_like(y)
            got, want = (torch.autograd.grad(y, leaf, d, retain_graph=True)[0] for d in (torch._neg_view(dy), -dy))
            assert torch.equal(got, want), n


def test_rotary_of_more_pairs_than_it_has_is_refused():
    q, pos = torch.zeros(1, 3, 1, 300, device="cuda"), torch.zeros(3, 2, dtype=torch.int32, device="cuda")
    with pytest.raises(RuntimeError, match="sections must turn at most 128 pairs, not 129"):
        tokens.rotary(q, pos, (64, 65))
    assert torch.equal(tokens.rotary(q, pos, (64, 64)), q)


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("gain", [2.0 ** 6, 2.0 ** 10, 2.0 ** 13])
def test_attention_float16_large_output_gradients(gain, D):
    """Output gradients under a loss scale: score gradients beyond 2^10 overflow on their way through float16 and are done
    over in float32 (gain 2^13 takes most keys there); the bound is that of any call, with the gradients' own size."""
    q, k, v, do, g = _attention_inputs(1, 150, 150, 4, 2, D, F16, 61, gain=3.0)
    do = (do.float() * gain).clamp(-6e4, 6e4).to(F16)
    k, q = (k.float() / 4).to(F16), (q.float() / 4).to(F16)    # and the results within it
    slopes = torch.rand(4, generator=g) * 0.1
    for kw in (dict(causal=True), dict(cap=5.0, slopes=slopes)):
        _check_attention(q, k, v, do, **kw)


@pytest.mark.parametrize("D", [32, 64, 12])
@pytest.mark.parametrize("height", [0.0, 1000.0, 100000.0])
def test_attention_float32_gradients_of_high_scores(height, D):
    """Every score is a height plus small steps, all exact in float32. Weights rebuilt from a float32 log-sum-exp of that height
    alone would be off by half an ulp of it, 2^-24 * 2^16 = 4e-3 of themselves at 1e5, and every gradient with them.
    Normalised, what is left of a weight's error is its own exponent's (two roundings of numbers below 16, log2 e's times the
    steps, 4 for exp2) and that of the sum over T weights; a result adds a sum over D, T or both: below (2 T + 64 + D) 2^-24 of
    the magnitudes' sums, and twice for a score gradient of two parts."""
    T, H = 96, 2
    g = _gen(int(height) + D)
    # q.k = height exactly: one column of q and k; the others hold eighths, whose products are exact
    q, k = (torch.randint(-4, 5, (1, T, h, D), generator=g).float() / 8 for h in (H, H))
    q[..., 4:], k[..., 4:] = 0, 0
    q[..., 0], k[..., 0] = height, 1.0
    v, do = torch.randn(1, T, H, D, generator=g), torch.randn(1, T, H, D, generator=g)
    slopes = torch.full((H,), 2.0 ** -6)                        # distances below 96 times 2^-6: exact
    leaves = [t.cuda().requires_grad_() for t in (q, k, v, slopes)]
    o = tokens.attention(*leaves[:3], scale=1.0, slopes=leaves[3])
    grads = torch.autograd.grad(o, leaves, do.cuda())
    Q, K, V, G = (t.double().transpose(1, 2) for t in (q, k, v, do))
    far = (torch.arange(T)[:, None] - torch.arange(T)).abs().double()
    p = (Q @ K.transpose(2, 3) - 2.0 ** -6 * far).softmax(-1)
    dp = G @ V.transpose(2, 3)
    delta = (p * dp).sum(-1, keepdim=True)
    ds, size = p * (dp - delta), p * (G.abs() @ V.abs().transpose(2, 3) + (p * (G.abs() @ V.abs().transpose(2, 3))).sum(-1, keepdim=True))
    tol = 2 * (2 * T + 64 + D) * 2.0 ** -24
    for got, want, most in zip(grads, ((ds @ K), (ds.transpose(2, 3) @ Q), (p.transpose(2, 3) @ G), -(ds * far).sum((0, 2, 3))),
                               ((size @ K.abs()), (size.transpose(2, 3) @ Q.abs()), (p.transpose(2, 3) @ G.abs()), (size * far).sum((0, 2, 3)))):
        got = got.double().cpu()
        got = got if got.dim() == 1 else got.transpose(1, 2)
        assert bool(((got - want).abs() <= tol * most).all()), float(((got - want).abs() / most).max() / tol)


def test_scattering_attention_under_autocast():
    """The projections come in the autocast's type, the other parameters are float32: the read-out takes both. Against the same
    module without autocast: weights, projections, rotary, attention and read-out round to bfloat16 eight times in a row or
    fewer, each by at most 2^-8 of a value, and a score's relative error comes out of the softmax at most cap = 4 times as
    large."""
    torch.manual_seed(5)
    net = ScatteringAttention(2, (32, 32), channels=1, heads=2, dim=24, L=2, cap=4.0).cuda()
    images, owner = torch.rand(2, 3, 1, 32, 32, device="cuda"), torch.tensor([[0, 0, 1], [1, -1, 0]], dtype=torch.int32)
    want = [net(images, owner), net.pooled(images, owner, 2)]
    with torch.autocast("cuda", dtype=BF16):
        got = [net(images, owner), net.pooled(images, owner, 2)]
    for a, b in zip(got, want):
        assert a.dtype == BF16 and float(((a.float() - b).norm() / b.norm()).detach()) < 8 * 2 ** -8 * 4
    got[1].float().square().sum().backward()
    for name, t in net.named_parameters():
        assert t.grad is not None and t.grad.dtype == F32 and bool(torch.isfinite(t.grad).all()) and bool(t.grad.any()), name


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("D", [32, 128, 12])
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("height", [0.0, 2.0 ** 10, 2.0 ** 17])
def test_attention_16_bit_slope_gradients_of_high_scores(height, causal, D, dtype):
    """The slopes' gradient is a float32 sum in 16-bit calls too, and meets the log-sum-exp's rounding as float32 gradients do.
    delta, taken from an output in two 16-bit parts, leaves the gradient where the weights add up to 1: sum ds (far - sum p far)
    is the same for every delta. A pair's own error is at most (64 + D) 2^-24 of its magnitude (the exponent's and the sums'
    roundings as above, a row's sum of weights being a tree of T / 16 steps and 4); pairs round independently, and a sum of
    independent errors lies within 8 times the root of the sum of their squares."""
    T, H = 160, 2
    g = _gen(int(height) + D)
    q, k = (torch.randint(-4, 5, (1, T, H, D), generator=g).float() / 8 for _ in range(2))
    q[..., 4:], k[..., 4:] = 0, 0
    q[..., 0], k[..., 0] = height / 4, 4.0
    v, do = torch.randn(1, T, H, D, generator=g), torch.randn(1, T, H, D, generator=g)
    q, k, v, do = (t.to(dtype) for t in (q, k, v, do))
    slopes = torch.full((H,), 2.0 ** -6, device="cuda", requires_grad=True)
    leaves = [t.cuda().requires_grad_() for t in (q, k, v)]
    o = tokens.attention(*leaves, scale=1.0, slopes=slopes, causal=causal)
    got = torch.autograd.grad(o, slopes, do.cuda())[0].double().cpu()
    Q, K, V, G = (t.double().transpose(1, 2) for t in (q, k, v, do))
    far = (torch.arange(T)[:, None] - torch.arange(T)).abs().double()
    z = Q @ K.transpose(2, 3) - 2.0 ** -6 * far
    p = (z.masked_fill(~torch.ones(T, T).tril().bool(), -torch.inf) if causal else z).softmax(-1)
    dp, most = G @ V.transpose(2, 3), G.abs() @ V.abs().transpose(2, 3)
    ds, size = p * (dp - (p * dp).sum(-1, keepdim=True)), p * (most + (p * most).sum(-1, keepdim=True))
    want, bound = -(ds * far).sum((0, 2, 3)), 8 * (64 + D) * 2.0 ** -24 * (size * far).square().sum((0, 2, 3)).sqrt()
    assert bool(((got - want).abs() <= bound).all()), ((got - want).abs() / bound).tolist()
