"""GPU tests of the token operators (wst_amd.tokens) against their float64 restatement (oracle/token_ops.py), whose
bounds on rounding are the tolerances: every value must lie within its own."""
import ctypes
import math

import pytest
import torch

import wst_amd  # noqa: F401
from oracle import token_ops as ref
from wst_amd import _lib, tokens

pytestmark = pytest.mark.gpu

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


def _gen(seed):
    return torch.Generator().manual_seed(seed)


def _hold(got, want, what):
    value, bound = want
    got = got.detach().cpu().to(torch.float64).reshape(value.shape)
    same = torch.isfinite(got) == torch.isfinite(value)
    assert bool(same.all()), f"{what}: {int((~same).sum())} values differ in being finite"
    fine = torch.isfinite(value)
    off = (got - value).abs()[fine]
    over = off > bound[fine]
    assert not bool(over.any()), (f"{what}: {int(over.sum())} of {over.numel()} outside, worst "
                                  f"{float((off / bound[fine].clamp(min=1e-300)).max()):.3g} times its bound")


# ------------------------------------------------------------------------------------------ layer norm
def _norm_inputs(rows, n, x_dtype, w_dtype, seed, offset=0.0):
    g = _gen(seed)
    scale = torch.exp(torch.randn(n, generator=g) * 1.5 - 3)
    x = ((torch.randn(rows, n, generator=g) * 0.4 + 1) * scale + offset).to(x_dtype)
    w = None if w_dtype is None else (1 + 0.3 * torch.randn(n, generator=g)).to(w_dtype)
    b = None if w_dtype is None else torch.randn(n, generator=g).to(w_dtype)
    return x, w, b, torch.randn(rows, n, generator=g)


@pytest.mark.parametrize("x_dtype,out_dtype,w_dtype", [(F32, F32, F32), (BF16, BF16, F32), (F16, F16, F16), (F32, BF16, F32),
                                                       (BF16, F32, BF16), (F32, F32, None)])
@pytest.mark.parametrize("rows,n", [(1, 1), (3, 1), (2, 7), (5, 64), (9, 243), (2100, 257), (3, 486), (7, 1251), (4, 2048),
                                    (2, 2049), (3, 8192), (2, 8193), (2, 8932), (2, 33000)])
def test_layer_norm_rows(rows, n, x_dtype, out_dtype, w_dtype):
    x, w, b, dy = _norm_inputs(rows, n, x_dtype, w_dtype, rows + n)
    dy = dy.to(out_dtype)
    want = ref.layer_norm(x, w, b, 1e-5, out_dtype, dy)
    xs = x.cuda().requires_grad_()
    leaves = [xs] + ([] if w is None else [w.cuda().requires_grad_(), b.cuda().requires_grad_()])
    y = tokens.layer_norm(xs, *leaves[1:], out_dtype=out_dtype)
    assert y.dtype == out_dtype and y.shape == xs.shape
    _hold(y, want["y"], "y")
    for t, name in zip(torch.autograd.grad(y, leaves, dy.cuda()), ("dx", "dw", "db")):
        _hold(t, want[name], name)
    with torch.no_grad():
        assert torch.equal(tokens.layer_norm(xs, *leaves[1:], out_dtype=out_dtype), y)


@pytest.mark.parametrize("x_dtype,out_dtype", [(F32, F32), (F32, BF16), (BF16, BF16), (F16, F32)])
@pytest.mark.parametrize("batch,points,n", [(1, 2, 3), (2, 16, 417), (3, 16, 1251), (2, 256, 81), (1, 1024, 243), (2, 5, 30),
                                            (2, 17, 700), (1, 63, 100), (2, 4, 4466), (1, 3, 9001), (40, 16, 64)])
def test_layer_norm_maps(batch, points, n, x_dtype, out_dtype):
    """Maps read where the transform writes them: the points adjacent."""
    x, w, b, dy = _norm_inputs(batch * points, n, x_dtype, F32, points + n)
    dy = dy.to(out_dtype)
    want = ref.layer_norm(x, w, b, 1e-5, out_dtype, dy)
    maps = x.reshape(batch, points, n).transpose(1, 2).contiguous().cuda()
    xs = maps.transpose(1, 2).requires_grad_()
    ws, bs = w.cuda().requires_grad_(), b.cuda().requires_grad_()
    y = tokens.layer_norm(xs, ws, bs, out_dtype=out_dtype)
    assert y.is_contiguous()
    _hold(y, want["y"], "y")
    dyc = dy.cuda().reshape(batch, points, n)
    dx, dw, db = torch.autograd.grad(y, (xs, ws, bs), dyc)
    _hold(dx, want["dx"], "dx")
    _hold(dw, want["dw"], "dw")
    _hold(db, want["db"], "db")
    # without the gradient of x (the transform has none) the others are the same
    dw2, db2 = torch.autograd.grad(tokens.layer_norm(xs.detach(), ws, bs, out_dtype=out_dtype), (ws, bs), dyc)
    assert torch.equal(dw2, dw) and torch.equal(db2, db)


def test_layer_norm_strides_and_views():
    x, w, b, dy = _norm_inputs(24, 40, F32, F32, 5)
    want = ref.layer_norm(x, w, b, 1e-5, F32, dy)
    w, b, dy = w.cuda(), b.cuda(), dy.cuda()
    wide = torch.full((24, 51), math.nan, device="cuda")
    wide[:, 3:43] = x.cuda()
    four = x.cuda().reshape(2, 3, 4, 40).permute(2, 0, 1, 3).contiguous().permute(1, 2, 0, 3)   # three strides: copied
    for view in (wide[:, 3:43], four, x.cuda().reshape(2, 12, 40)):
        leaf = view.detach().requires_grad_()
        y = tokens.layer_norm(leaf, w, b)
        assert y.shape == view.shape
        _hold(y, want["y"], "y")
        dx, = torch.autograd.grad(y, leaf, dy.reshape(view.shape))
        _hold(dx, want["dx"], "dx")
    row = x[:1].cuda().expand(5, 40).requires_grad_()
    y = tokens.layer_norm(row, w, b)
    assert torch.equal(y, y[:1].expand_as(y))
    dx, = torch.autograd.grad(y, row, dy[:5])
    _hold(dx, ref.layer_norm(x[:1].expand(5, 40), w.cpu(), b.cpu(), 1e-5, F32, dy[:5].cpu())["dx"], "dx")


def test_layer_norm_far_from_zero_and_constant_rows():
    x, w, b, dy = _norm_inputs(6, 500, F32, F32, 6, offset=1000.0)
    x[2] = 3.0                                                 # constant: y = b
    want = ref.layer_norm(x, w, b, 1e-5, F32, dy)
    leaf = x.cuda().requires_grad_()
    y = tokens.layer_norm(leaf, w.cuda(), b.cuda())
    _hold(y, want["y"], "y")
    assert bool((y[2].detach().cpu() == b).all())
    _hold(torch.autograd.grad(y, leaf, dy.cuda())[0], want["dx"], "dx")


def test_layer_norm_not_finite_values_stay_in_their_row():
    x, w, b, _ = _norm_inputs(8, 300, F32, F32, 7)
    y0 = tokens.layer_norm(x.cuda(), w.cuda(), b.cuda())
    x[3, 5], x[6, 299] = math.nan, math.inf
    y = tokens.layer_norm(x.cuda(), w.cuda(), b.cuda())
    keep = [0, 1, 2, 4, 5, 7]
    assert torch.equal(y[keep], y0[keep]) and bool(y[[3, 6]].isnan().all())


def test_layer_norm_empty():
    w = torch.ones(4, device="cuda", requires_grad=True)
    x = torch.zeros(0, 3, 4, device="cuda", requires_grad=True)
    y = tokens.layer_norm(x, w)
    dx, dw = torch.autograd.grad(y, (x, w), y.detach())
    assert y.shape == (0, 3, 4) and dx.shape == x.shape and torch.equal(dw, torch.zeros_like(dw))


# ------------------------------------------------------------------------------------------ rotary
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("B,T,H,Hk,D,sections,interleaved", [
    (1, 1, 1, 1, 2, (1,), False), (2, 1, 8, 2, 64, (8, 12, 12), False), (2, 33, 3, 1, 40, (0, 7, 9), True),
    (1, 50, 2, 2, 128, (16, 24, 24), False), (2, 9, 4, 4, 37, (3, 2, 1, 4), False), (2, 9, 4, 4, 37, (3, 2, 1, 4), True),
    (1, 300, 2, 1, 256, (128,), True), (3, 5, 2, 1, 16, (0, 0), False)])
def test_rotary(B, T, H, Hk, D, sections, interleaved, dtype):
    g = _gen(D + T)
    qk = torch.randn(B, T, H + Hk, D, generator=g).to(dtype)
    pos = torch.randint(-300, 2 ** 31 - 1, (B, T, len(sections)), generator=g, dtype=torch.int64)
    pos = torch.where(torch.rand(pos.shape, generator=g) < 0.5, pos % 1000, pos).to(torch.int32)   # near and far
    dq, dk = torch.randn(B, T, H, D, generator=g).to(dtype), torch.randn(B, T, Hk, D, generator=g).to(dtype)
    both = qk.cuda()
    q, k = both[:, :, :H].requires_grad_(), both[:, :, H:].requires_grad_()
    qo, ko = tokens.rotary(q, pos.cuda(), sections, base=500.0, interleaved=interleaved, k=k)
    how = (pos, sections, 500.0, interleaved)
    _hold(qo, ref.rotary(qk[:, :, :H], *how), "q")
    _hold(ko, ref.rotary(qk[:, :, H:], *how), "k")
    gq, gk = torch.autograd.grad((qo, ko), (q, k), (dq.cuda(), dk.cuda()))
    _hold(gq, ref.rotary(dq, *how, inverse=True), "dq")
    _hold(gk, ref.rotary(dk, *how, inverse=True), "dk")
    # one tensor alone, positions shared by the batch
    one = tokens.rotary(q.detach(), pos[0].cuda(), sections, base=500.0, interleaved=interleaved)
    _hold(one, ref.rotary(qk[:, :, :H], pos[:1].expand(B, -1, -1), *how[1:]), "shared positions")


def test_rotary_strides_gradients_and_empty():
    g = _gen(3)
    x = torch.randn(2, 4, 6, 16, generator=g)
    pos = torch.randint(0, 99, (2, 6, 2), generator=g, dtype=torch.int32)
    heads_first = x.cuda().transpose(1, 2)                     # (2, 6, 4, 16) over (2, 4, 6, 16)
    want = ref.rotary(x.transpose(1, 2), pos, (4, 3), 10.0, False)
    _hold(tokens.rotary(heads_first, pos.cuda(), (4, 3), base=10.0), want, "heads first")
    spread = torch.zeros(2, 6, 4, 32, device="cuda")
    spread[..., ::2] = heads_first
    _hold(tokens.rotary(spread[..., ::2], pos.cuda(), (4, 3), base=10.0), want, "every second value")
    leaf = heads_first.detach().requires_grad_()
    out = tokens.rotary(leaf, pos.cuda(), (4, 3), base=10.0)
    dx, = torch.autograd.grad(out.sum(), leaf)                  # an expanded gradient, all strides 0
    _hold(dx, ref.rotary(torch.ones(2, 6, 4, 16), pos, (4, 3), 10.0, False, inverse=True), "dx")
    empty = tokens.rotary(torch.zeros(2, 0, 4, 16, device="cuda"), torch.zeros(0, 2, dtype=torch.int32, device="cuda"), (4, 3))
    assert empty.shape == (2, 0, 4, 16)


# ------------------------------------------------------------------------------------------ attention
def _attention_inputs(B, Tq, Tk, H, Hk, D, dtype, seed, gain=1.0):
    g = _gen(seed)
    q = (torch.randn(B, Tq, H, D, generator=g) * gain).to(dtype)
    k, v = (torch.randn(B, Tk, Hk, D, generator=g).to(dtype) for _ in range(2))
    return q, k, v, torch.randn(B, Tq, H, D, generator=g).to(dtype), g


def _documents(g, B, T, count, empty=0.1):
    d = torch.sort(torch.randint(0, count, (B, T), generator=g, dtype=torch.int32), 1)[0]
    return torch.where(torch.rand(B, T, generator=g) < empty, torch.full_like(d, -1), d)


def _check_attention(q, k, v, do, train=True, **kw):
    dev = {n: t.cuda() if torch.is_tensor(t) else t for n, t in kw.items()}
    want = ref.attention(q, k, v, do=do if train else None, **kw)
    leaves = [t.cuda().requires_grad_(train) for t in (q, k, v)]
    if kw.get("slopes") is not None:
        dev["slopes"] = dev["slopes"].requires_grad_(train)
        leaves.append(dev["slopes"])
    o, lse = tokens.attention(*leaves[:3], return_lse=True, **dev)
    assert o.dtype == q.dtype and lse.dtype == F32
    _hold(o, want["o"], "o")
    _hold(lse, want["lse"], "lse")
    if train:
        grads = torch.autograd.grad(o, leaves, do.cuda())
        for t, name in zip(grads, ("dq", "dk", "dv", "dslopes")):
            _hold(t, want[name], name)
        return o, grads
    return o, None


SIZES = [(1, 1, 1, 1, 1, 8), (2, 1, 65, 4, 1, 32), (1, 5, 300, 6, 2, 64), (2, 63, 63, 2, 2, 16), (1, 129, 129, 2, 1, 128),
         (1, 200, 333, 3, 3, 80), (2, 333, 200, 2, 1, 40), (1, 257, 257, 4, 2, 96), (1, 31, 70, 2, 1, 5), (1, 40, 40, 1, 1, 200),
         (1, 64, 128, 8, 2, 24)]


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("B,Tq,Tk,H,Hk,D", SIZES)
@pytest.mark.parametrize("mask", ["none", "causal", "prefix"])
def test_attention_masks(B, Tq, Tk, H, Hk, D, mask, dtype):
    q, k, v, do, g = _attention_inputs(B, Tq, Tk, H, Hk, D, dtype, Tq + Tk + D)
    kw = dict(causal=mask != "none")
    if mask == "prefix":
        kw["prefix"] = torch.randint(0, Tk + 5, (B,), generator=g, dtype=torch.int32)
    _check_attention(q, k, v, do, **kw)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("B,Tq,Tk,H,Hk,D", SIZES)
def test_attention_cap_bias_documents_lengths(B, Tq, Tk, H, Hk, D, dtype):
    q, k, v, do, g = _attention_inputs(B, Tq, Tk, H, Hk, D, dtype, Tq * Tk + D, gain=2.0)
    slopes = 2.0 ** -(1 + 7 * torch.rand(H, generator=g))
    lengths = torch.randint(0, Tk + 1, (B,), generator=g, dtype=torch.int32)
    positions = {n: torch.randint(-20, 20, (B, t, 3), generator=g, dtype=torch.int32) for n, t in (("q", Tq), ("k", Tk))}
    docs = {n: _documents(g, B, t, 3) for n, t in (("q", Tq), ("k", Tk))}
    _check_attention(q, k, v, do, cap=3.0)
    _check_attention(q, k, v, do, slopes=slopes, causal=True)
    _check_attention(q, k, v, do, slopes=slopes, q_positions=positions["q"], k_positions=positions["k"])
    _check_attention(q, k, v, do, q_documents=docs["q"], k_documents=docs["k"])
    _check_attention(q, k, v, do, k_lengths=lengths, slopes=slopes)
    _check_attention(q, k, v, do, cap=2.0, slopes=slopes, q_positions=positions["q"][0], k_positions=positions["k"][0],
                     q_documents=docs["q"][0], k_documents=docs["k"][0], causal=True, scale=0.3,
                     prefix=torch.randint(0, Tk, (B,), generator=g, dtype=torch.int32), k_lengths=lengths)


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("Tq,G,Hk,D,Tk", [(1, 1, 1, 64, 4000), (1, 8, 2, 128, 5000), (3, 4, 1, 64, 1025), (16, 2, 2, 32, 2100),
                                          (2, 5, 2, 96, 70), (1, 40, 1, 64, 900)])
def test_attention_few_queries(Tq, G, Hk, D, Tk, dtype):
    """The serving form: a few new queries over many stored keys."""
    q, k, v, do, g = _attention_inputs(3, Tq, Tk, G * Hk, Hk, D, dtype, Tk)
    lengths = torch.tensor([Tk, max(1, Tk // 3), 0], dtype=torch.int32)
    slopes = 2.0 ** -(1 + 7 * torch.rand(G * Hk, generator=g))
    for kw in (dict(), dict(causal=True, k_lengths=lengths), dict(k_lengths=lengths, cap=5.0, slopes=slopes)):
        _check_attention(q, k, v, do, train=False, **kw)
    docs = _documents(g, 3, Tk, 4)
    _check_attention(q, k, v, do, train=False, q_documents=torch.full((3, Tq), 2, dtype=torch.int32), k_documents=docs)


def test_attention_one_document_a_token_and_no_visible_key():
    q, k, v, do, g = _attention_inputs(2, 150, 150, 2, 2, 32, BF16, 8)
    own = torch.arange(150, dtype=torch.int32).expand(2, 150).contiguous()
    o, _ = _check_attention(q, k, v, do, q_documents=own, k_documents=own)
    assert torch.equal(o.cpu(), v)                             # each sees itself alone
    o, grads = _check_attention(q, k, v, do, q_documents=own, k_documents=own + 1000)
    assert not bool(o.any()) and not any(bool(t.any()) for t in grads)
    o, grads = _check_attention(q, k, v, do, k_lengths=torch.zeros(2, dtype=torch.int32))
    assert not bool(o.any()) and not any(bool(t.any()) for t in grads)
    # lengths outside 0..Tk are held to it
    o, _ = _check_attention(q, k, v, do, k_lengths=torch.tensor([-3, 4000], dtype=torch.int32))


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("D,bad", [(64, math.nan), (64, math.inf), (5, math.nan), (128, -math.inf)])
def test_attention_not_finite_values_that_are_not_seen(D, bad, dtype):
    """Keys, values, queries and gradients that no visible pair touches may hold anything; a query that does not see a
    bad key is right though others of its tile do."""
    B, T, H, Hk = 2, 200, 4, 2
    q, k, v, do, g = _attention_inputs(B, T, T, H, Hk, D, dtype, 9)
    docs = _documents(g, B, T, 3, empty=0.2)
    gone = docs < 0
    for t in (q, k, v, do):
        t[gone] = bad
    _check_attention(q, k, v, do, q_documents=docs, k_documents=docs)
    _check_attention(q, k, v, do, q_documents=docs, k_documents=docs, causal=True, cap=4.0)
    lengths = torch.tensor([150, 37], dtype=torch.int32)
    q, k, v, do, g = _attention_inputs(B, T, T, H, Hk, D, dtype, 10)
    for b in range(B):
        k[b, lengths[b]:] = bad
        v[b, lengths[b]:] = bad
    _check_attention(q, k, v, do, k_lengths=lengths)
    _check_attention(q[:, :2], k, v, do[:, :2], train=False, k_lengths=lengths)
    # causal: key 100 is bad; queries below 100 do not see it, the others do
    q, k, v, do, g = _attention_inputs(1, T, T, H, Hk, D, dtype, 11)
    clean = ref.attention(q, k, v, do=do, causal=True)["o"]
    v[:, 100] = bad
    o = tokens.attention(q.cuda(), k.cuda(), v.cuda(), causal=True).cpu()
    _hold(o[:, :100], (clean[0][:, :100], clean[1][:, :100]), "o before the bad key")
    assert not bool(torch.isfinite(o[:, 100:].float()).any())
    # and its gradients: queries below 100 take part alone
    do[:, 100:] = 0
    leaves = [t.cuda().requires_grad_() for t in (q, k, v)]
    dq, dk, dv = torch.autograd.grad(tokens.attention(*leaves, causal=True), leaves, do.cuda())
    want = ref.attention(q[:, :100], k[:, :100], v[:, :100], do=do[:, :100], causal=True)
    _hold(dq[:, :100], want["dq"], "dq before the bad key")


def test_attention_gradients_match_differences():
    """Directional differences of the operator's own float32 outputs."""
    q, k, v, do, g = _attention_inputs(1, 70, 90, 4, 2, 16, F32, 12)
    slopes = torch.rand(4, generator=g)
    leaves = [t.cuda().requires_grad_() for t in (q, k, v, slopes)]
    kw = dict(cap=2.0, causal=True)
    call = lambda q, k, v, s: tokens.attention(q, k, v, slopes=s, **kw)   # noqa: E731
    grads = torch.autograd.grad(call(*leaves), leaves, do.cuda())
    h = 2.0 ** -8
    for n, name in enumerate(("q", "k", "v", "slopes")):
        d = torch.randn(leaves[n].shape, generator=g).cuda()
        at = lambda e: (call(*[t.detach() + (e * d if m == n else 0) for m, t in enumerate(leaves)]).double()   # noqa: E731
                        * do.cuda().double()).sum()
        # Richardson: the h^2 term cancels, what is left is of order h^4 times fifth derivatives (of order one here,
        # 280 rows) and 2^-24 / h of rounding, each of the 4480 outputs' errors at random
        diff = (8 * (at(h) - at(-h)) - (at(2 * h) - at(-2 * h))) / (12 * h)
        want = (grads[n].double() * d.double()).sum()
        noise = 2.0 ** -24 / h * 4 * float(do.norm()) * 8
        assert abs(float(diff - want)) < noise + h ** 4 * 280 * 10 + 1e-6, name


def test_attention_strides_views_and_shared_tensors():
    g = _gen(13)
    B, T, H, D = 2, 90, 4, 64
    qkv = torch.randn(B, T, 3, H, D, generator=g).to(BF16)
    do = torch.randn(B, T, H, D, generator=g).to(BF16)
    want = ref.attention(qkv[:, :, 0], qkv[:, :, 1], qkv[:, :, 2], do=do, causal=True)
    leaf = qkv.cuda().requires_grad_()
    o = tokens.attention(leaf[:, :, 0], leaf[:, :, 1], leaf[:, :, 2], causal=True)   # one projection's output
    _hold(o, want["o"], "o")
    grad, = torch.autograd.grad(o, leaf, do.cuda())
    for i, name in enumerate(("dq", "dk", "dv")):
        _hold(grad[:, :, i], want[name], name)
    # heads before tokens, gradients of such strides too
    q, k, v = (leaf.detach()[:, :, i].transpose(1, 2).contiguous().transpose(1, 2).requires_grad_() for i in range(3))
    o2 = tokens.attention(q, k, v, causal=True)
    assert torch.equal(o2, o)
    dh = do.cuda().transpose(1, 2).contiguous().transpose(1, 2)
    for t, name in zip(torch.autograd.grad(o2, (q, k, v), dh), ("dq", "dk", "dv")):
        _hold(t, want[name], name)
    # unaligned rows, and every second value
    flat = torch.zeros(B * T * H * 65 + 3, dtype=BF16, device="cuda")
    odd = flat[3:].view(B, T, H, 65)[..., :64]
    odd.copy_(leaf.detach()[:, :, 0])
    spread = torch.zeros(B, T, H, 2 * D, dtype=BF16, device="cuda")
    spread[..., ::2] = leaf.detach()[:, :, 1]
    assert torch.equal(tokens.attention(odd, spread[..., ::2], leaf.detach()[:, :, 2], causal=True), o)
    # one key and value for all tokens and batch entries
    kb = leaf.detach()[:1, :1, 1].expand(B, T, H, D)
    assert torch.equal(tokens.attention(odd, kb, kb), kb)


def test_attention_far_offsets():
    """A stored series whose rows lie more than 2^31 elements and 2^32 bytes apart."""
    q, k, v, _, _ = _attention_inputs(2, 1, 130, 2, 1, 64, BF16, 14)
    store = torch.empty((1 << 31) + (1 << 25), dtype=BF16, device="cuda")
    far = [store.as_strided((2, 130, 1, 64), (1 << 31, 256, 64, 1), 64 * i) for i in range(2)]
    far[0].copy_(k)
    far[1].copy_(v)
    o = tokens.attention(q.cuda(), far[0], far[1])
    _hold(o, ref.attention(q, k, v)["o"], "o")
    apart = [store.as_strided((1, 130, 1, 64), (0, 1 << 24, 64, 1), 64 * i) for i in range(2)]   # token 128 is at 2^31
    apart[0].copy_(k[:1])
    apart[1].copy_(v[:1])
    _hold(tokens.attention(q[:1].cuda(), apart[0], apart[1]), ref.attention(q[:1], k[:1], v[:1])["o"], "o")
    o = tokens.attention(q[:1].expand(1, 1, 2, 64).cuda().expand(1, 70, 2, 64), apart[0], apart[1])
    _hold(o, ref.attention(q[:1].expand(1, 70, 2, 64), k[:1], v[:1])["o"], "many queries")


def test_attention_rows_behind_the_length_stay():
    """Nothing is written but the results: a gradient of keys behind the length is zero, and inputs keep their bits."""
    q, k, v, do, _ = _attention_inputs(2, 40, 100, 2, 2, 32, BF16, 15)
    lengths = torch.tensor([60, 0], dtype=torch.int32)
    kc, vc = k.cuda(), v.cuda()
    k0, v0 = kc.clone(), vc.clone()
    _, grads = _check_attention(q, k, v, do, k_lengths=lengths)
    tokens.attention(q.cuda(), kc, vc, k_lengths=lengths.cuda())
    assert torch.equal(kc, k0) and torch.equal(vc, v0)
    assert not bool(grads[1][0, 60:].any()) and not bool(grads[2][1].any())


def test_attention_empty_sizes():
    q = torch.zeros(2, 3, 2, 8, device="cuda", requires_grad=True)
    k = torch.zeros(2, 0, 1, 8, device="cuda", requires_grad=True)
    slopes = torch.ones(2, device="cuda", requires_grad=True)
    o, lse = tokens.attention(q, k, k, slopes=slopes, return_lse=True)
    assert not bool(o.any()) and bool((lse == -math.inf).all())
    for t in torch.autograd.grad(o, (q, k, slopes), torch.ones_like(o)):
        assert not bool(t.any())
    o = tokens.attention(q[:, :0], q[:, :, :1], q[:, :, :1])
    assert o.shape == (2, 0, 2, 8)


# ------------------------------------------------------------------------------------------ together
def test_repeats_bit_for_bit():
    q, k, v, do, g = _attention_inputs(2, 300, 300, 4, 2, 64, BF16, 16)
    slopes = torch.rand(4, generator=g).cuda().requires_grad_()
    leaves = [t.cuda().requires_grad_() for t in (q, k, v)] + [slopes]
    run = lambda: torch.autograd.grad(tokens.attention(*leaves[:3], slopes=slopes, causal=True), leaves, do.cuda())   # noqa: E731
    first = run()
    for _ in range(3):
        assert all(torch.equal(a, b) for a, b in zip(run(), first))
    x = torch.randn(5000, 300, generator=g).cuda()
    w = torch.ones(300, device="cuda", requires_grad=True)
    run = lambda: torch.autograd.grad(tokens.layer_norm(x, w).sum(), w)[0]   # noqa: E731
    first = run()
    assert torch.equal(run(), first)


def test_streams_run_apart():
    q, k, v, _, _ = _attention_inputs(1, 1, 3000, 4, 1, 64, BF16, 17)
    q, k, v = q.cuda(), k.cuda(), v.cuda()
    want = tokens.attention(q, k, v)
    x = torch.randn(700, 1251, device="cuda")
    norm = tokens.layer_norm(x)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(3)]
    got = []
    for _ in range(5):
        for s in streams:
            with torch.cuda.stream(s):
                got.append((tokens.attention(q, k, v), tokens.layer_norm(x)))
    torch.cuda.synchronize()
    assert all(torch.equal(o, want) and torch.equal(y, norm) for o, y in got)


def test_captured_graphs():
    """Forward and backward captured; two graphs replayed in turn, with eager work between the replays."""
    B, T, H, Hk, D = 1, 140, 4, 2, 32
    pos = tokens.grid_positions(1, 10, 14, device="cuda")
    w = torch.ones(H * D, device="cuda")

    def step(x, leafs):
        y = tokens.layer_norm(x, leafs[0]).view(B, T, H, D)
        q, k = tokens.rotary(y, pos, (4, 6, 6), k=y[:, :, :Hk])
        return tokens.attention(q, k, y[:, :, Hk:], cap=5.0, slopes=leafs[1], q_positions=pos, k_positions=pos, causal=True)

    def both(x):
        leafs = [w.detach().requires_grad_(), torch.full((H,), 0.1, device="cuda").requires_grad_(), x.detach().requires_grad_()]
        o = step(leafs[2], leafs)
        return (o.detach(), *torch.autograd.grad(o, leafs, torch.ones_like(o)))

    xs = [torch.randn(B, T, H * D, device="cuda", generator=torch.Generator("cuda").manual_seed(i)) for i in range(4)]
    want = [both(x) for x in xs]
    static = [xs[0].clone() for _ in range(2)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for s in static:
            both(s)
    torch.cuda.current_stream().wait_stream(side)
    graphs, outs = [], []
    for s in static:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(both(s))
        graphs.append(g)
    for i in range(8):
        n = i % 2
        static[n].copy_(xs[i % 4])
        graphs[n].replay()
        eager = both(xs[(i + 1) % 4])
        assert all(torch.equal(a, b) for a, b in zip(outs[n], want[i % 4])), i
        assert all(torch.equal(a, b) for a, b in zip(eager, want[(i + 1) % 4])), i


def test_refusals_name_the_argument():
    x = torch.zeros(2, 6, 4, 8, device="cuda")
    ints = torch.zeros(6, 3, dtype=torch.int32, device="cuda")
    bad = [
        (TypeError, lambda: tokens.layer_norm(x.double())), (TypeError, lambda: tokens.layer_norm(x, out_dtype=torch.int32)),
        (RuntimeError, lambda: tokens.layer_norm(x, x[0, 0, 0, :4])), (RuntimeError, lambda: tokens.layer_norm(x, eps=-1)),
        (TypeError, lambda: tokens.layer_norm(x, x[0, 0, 0], x[0, 0, 0].half())),
        (RuntimeError, lambda: tokens.layer_norm(x, torch.ones(8))),
        (RuntimeError, lambda: tokens.layer_norm(x[..., :0])),
        (RuntimeError, lambda: tokens.rotary(x[0], ints, (1, 1, 1))), (RuntimeError, lambda: tokens.rotary(x, ints, (1, 1))),
        (RuntimeError, lambda: tokens.rotary(x, ints, (2, 2, 1))), (TypeError, lambda: tokens.rotary(x, ints.long(), (1, 1, 1))),
        (RuntimeError, lambda: tokens.rotary(x, ints, (1, 1, 1), base=0.0)), (RuntimeError, lambda: tokens.rotary(x, ints, ())),
        (RuntimeError, lambda: tokens.rotary(x, ints[:5], (1, 1, 1))),
        (TypeError, lambda: tokens.rotary(x, ints, (1, 1, 1), k=x.half())),
        (RuntimeError, lambda: tokens.rotary(x, ints, (1, 1, 1), k=x[:, :3])),
        (TypeError, lambda: tokens.attention(x, x.half(), x)), (RuntimeError, lambda: tokens.attention(x, x, x[:, :3])),
        (RuntimeError, lambda: tokens.attention(x, x[:, :, :3], x[:, :, :3])),
        (RuntimeError, lambda: tokens.attention(x, x, x, slopes=torch.ones(3, device="cuda"))),
        (TypeError, lambda: tokens.attention(x, x, x, slopes=torch.ones(4, device="cuda").half())),
        (RuntimeError, lambda: tokens.attention(x, x, x, q_positions=ints)),
        (RuntimeError, lambda: tokens.attention(x, x, x, q_positions=ints, k_positions=ints)),
        (RuntimeError, lambda: tokens.attention(x, x, x, k_documents=ints[:, 0])),
        (RuntimeError, lambda: tokens.attention(x, x, x, k_lengths=ints[:, 0])),
        (TypeError, lambda: tokens.attention(x, x, x, k_lengths=torch.zeros(2, device="cuda"))),
        (RuntimeError, lambda: tokens.attention(x, x, x, cap=-1.0)), (RuntimeError, lambda: tokens.attention(x, x, x, scale=math.inf)),
        (RuntimeError, lambda: tokens.attention(*[torch.zeros(1, 2, 1, 300, device="cuda")] * 3)),
    ]
    for n, (kind, call) in enumerate(bad):
        with pytest.raises(kind):
            call()
            pytest.fail(f"case {n} was taken")
    y = tokens.layer_norm(x.requires_grad_())
    g, = torch.autograd.grad(y.sum(), x)
    assert g.shape == x.shape                                   # a refusal leaves nothing behind


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("D,Tq,causal", [(64, 200, False), (128, 200, True), (32, 20, False), (12, 40, False)])
def test_attention_gradient_of_rows_with_one_large_weight(D, Tq, causal, dtype):
    """Where one weight is nearly 1, every do.v_j - delta that counts is a small difference: delta taken from the rounded
    output would miss it by |do| |o| half an eps, a multiple of the difference itself. With p_1 = 1 - t the exact
    ds_1 = p_1 (do.v_1 - delta) is t do.(v_1 - mean of the rest), and |do| |o| eps / 2 against t |do| |v| sqrt(2) is a
    relative error of eps / (2 sqrt 2 t) without, and eps^2 / (2 sqrt 2 t) with what the rounding took. Here t < eps / 2:
    the first is over 0.7, the second under eps, beside the roundings of score gradients and dq (eps together). A tenth of
    the first holds all of the second's (8 eps of bfloat16)."""
    g = _gen(D + Tq)
    eps = torch.finfo(dtype).eps
    q, k, v, do = (torch.randn(1, Tq, 1, D, generator=g) for _ in range(4))
    k = k / k.norm(dim=-1, keepdim=True)
    k[:, 0] = k[:, 0] * 0 + D ** -0.5                    # key 0 stands out by -log(eps / 2 / Tq), from every query
    far = -math.log(eps / 4 / Tq)
    q = 0.01 * q + far
    q, k, v, do = (t.to(dtype) for t in (q, k, v, do))
    scale = D ** -0.5
    want = ref.attention(q, k, v, causal=causal, scale=scale, do=do)["dq"][0]
    leaves = [t.cuda().requires_grad_() for t in (q, k, v)]
    o = tokens.attention(*leaves, causal=causal, scale=scale)
    dq = torch.autograd.grad(o, leaves[0], do.cuda())[0].cpu().to(torch.float64)
    rows = slice(1, None)                                # query 0 in order sees key 0 alone: no gradient
    off = (dq - want)[:, rows].norm() / want[:, rows].norm()
    assert float(off) < 0.07, float(off)


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("D", [32, 64, 128])
@pytest.mark.parametrize("order", ["rising", "falling", "mixed"])
def test_attention_scores_that_outgrow_the_first_maximum(D, order, dtype):
    """Scores that grow by 58 powers of two from one tile of keys to the next: the running maximum has to move, for some
    queries of a wave and not for others, in both directions of a walk and in order."""
    T = 330
    g = _gen(D)
    step = torch.arange(T) // 64
    step = {"rising": step, "falling": step.flip(0), "mixed": step[torch.randperm(T, generator=g)]}[order].float()
    gain = torch.where(torch.arange(T) % 3 == 0, 40.0, torch.where(torch.arange(T) % 3 == 1, -7.0, 0.0))
    q = (gain[:, None].expand(T, D) * D ** -0.5).reshape(1, T, 1, D).repeat(1, 1, 2, 1)
    k = step[:, None].expand(T, D).reshape(1, T, 1, D).clone()
    q, k = q + 0.01 * torch.randn(1, T, 2, D, generator=g), k + 0.01 * torch.randn(1, T, 1, D, generator=g)
    v, do = torch.randn(1, T, 1, D, generator=g), torch.randn(1, T, 2, D, generator=g)
    q, k, v, do = (t.to(dtype) for t in (q, k, v, do))
    for kw in (dict(), dict(causal=True), dict(q_documents=_documents(g, 1, T, 2, 0.05), k_documents=_documents(g, 1, T, 2, 0.05))):
        _check_attention(q, k, v, do, **kw)
    _check_attention(q[:, 4:7], k, v, do[:, 4:7], train=False)


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("scale", [-0.3, 0.0, -0.0])
@pytest.mark.parametrize("Tq,D", [(150, 64), (150, 12), (2, 64), (140, 128)])
def test_attention_scales_of_any_sign(Tq, D, scale, dtype):
    q, k, v, do, g = _attention_inputs(1, Tq, 1100 if Tq == 2 else 150, 4, 2, D, dtype, 31)
    slopes = torch.rand(4, generator=g)
    for kw in (dict(), dict(cap=2.0), dict(slopes=slopes, causal=True), dict(cap=2.0, slopes=-slopes)):
        _check_attention(q, k, v, do, scale=scale, **kw)


@pytest.mark.parametrize("B,T,H,Hk,D", [(1, 700, 6, 1, 64), (1, 300, 5, 1, 128), (1, 64, 7, 1, 96), (60, 130, 10, 1, 32),
                                        (1, 400, 12, 4, 128), (2, 129, 3, 1, 80), (1, 193, 1, 1, 64)])
@pytest.mark.parametrize("how", ["plain", "causal", "documents"])
def test_attention_heads_in_parts(B, T, H, Hk, D, how):
    """Sums of dk and dv in parts: whole heads a part, whole parts a head, and neither."""
    q, k, v, do, g = _attention_inputs(B, T, T, H, Hk, D, BF16, T + H)
    docs = _documents(g, B, T, 3)
    kw = {"plain": {}, "causal": dict(causal=True, slopes=torch.rand(H, generator=g) * 0.1),
          "documents": dict(q_documents=docs, k_documents=docs, causal=True)}[how]
    _check_attention(q, k, v, do, **kw)


def _bare_call(q, k, v, do, lse, o, causal=True):
    """The C entries on the tensors as they lie: forward, then backward; returns dq, dk, dv."""
    lib = _lib.load()
    B, T, H, D = q.shape
    d = _lib.AttentionDesc(batch=B, q_len=T, k_len=k.shape[1], q_strides=q.stride()[:3], k_strides=k.stride()[:3],
                           v_strides=v.stride()[:3], o_strides=o.stride()[:3], q=q.data_ptr(), k=k.data_ptr(), v=v.data_ptr(),
                           scale=D ** -0.5, q_heads=H, k_heads=k.shape[2], dim=D, dtype=tokens.DTYPES[q.dtype], causal=causal)
    need, st = ctypes.c_size_t(), torch.cuda.current_stream().cuda_stream
    for backward in (0, 1):
        assert lib.wst_attention_workspace(d, backward, ctypes.byref(need)) == 0
        ws = torch.empty(need.value + 1, dtype=torch.uint8, device="cuda")
        if not backward:
            assert lib.wst_attention_forward(d, o.data_ptr(), lse.data_ptr(), ws.data_ptr(), need.value, st) == 0
    out = [torch.empty_like(t) for t in (q, k, v)]
    g = _lib.AttentionGrads(o=o.data_ptr(), d_o=do.data_ptr(), lse=lse.data_ptr(), dq=out[0].data_ptr(), dk=out[1].data_ptr(),
                            dv=out[2].data_ptr(), do_strides=do.stride()[:3], dq_strides=out[0].stride()[:3],
                            dk_strides=out[1].stride()[:3], dv_strides=out[2].stride()[:3])
    assert lib.wst_attention_backward(d, g, ws.data_ptr(), need.value, st) == 0
    torch.cuda.synchronize()
    return out


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("odd", ["q", "k", "do", "none"])
def test_attention_c_entries_without_alignment(odd, dtype):
    """Rows that do not begin on 16 bytes are taken value by value, each call by its own tensors. Without o_rest delta is
    that of the rounded output, which the tolerance counts: |do| |o| half an eps for each ds."""
    B, T, H, Hk, D = 1, 140, 2, 1, 64
    q, k, v, do, _ = _attention_inputs(B, T, T, H, Hk, D, dtype, 77)
    want = ref.attention(q, k, v, causal=True, do=do)

    def place(t, name):
        flat = torch.empty(t.numel() + 8, dtype=dtype, device="cuda")
        out = flat[1 if name == odd else 0:][:t.numel()].view(t.shape)
        return out.copy_(t)

    qd, kd, vd, dod = place(q, "q"), place(k, "k"), place(v, "v"), place(do, "do")
    o, lse = torch.empty_like(qd), torch.empty(B, H, T, device="cuda")
    grads = _bare_call(qd, kd, vd, dod, lse, o)
    _hold(o, want["o"], "o")
    _hold(lse, want["lse"], "lse")
    p, lost = torch.exp(-want["lse"][0]), torch.finfo(dtype).eps / 2 * (do.double().abs() * want["o"][0].abs()).sum(-1)
    z = q.double().permute(0, 2, 1, 3) @ k.double().repeat_interleave(H // Hk, 2).permute(0, 2, 3, 1) * D ** -0.5
    p = torch.where(torch.ones(T, T).tril().bool(), torch.exp(z) * p[..., None], 0.0) * lost.transpose(1, 2)[..., None] * D ** -0.5
    kk, qq = k.double().abs().repeat_interleave(H // Hk, 2).transpose(1, 2), q.double().abs().transpose(1, 2)
    extra = {"dq": (p @ kk).transpose(1, 2), "dk": (p.transpose(2, 3) @ qq).sum(1, keepdim=True).transpose(1, 2), "dv": 0.0}
    for t, name in zip(grads, ("dq", "dk", "dv")):
        _hold(t, (want[name][0], want[name][1] + extra[name]), name)


def test_first_order_gradients_only():
    x = torch.randn(3, 8, device="cuda", requires_grad=True)
    q = torch.randn(1, 3, 1, 8, device="cuda", requires_grad=True)
    pos = torch.arange(3, dtype=torch.int32, device="cuda")[:, None]
    for y, leaf in ((tokens.layer_norm(x), x), (tokens.rotary(q, pos, (4,)), q), (tokens.attention(q, q, q), q)):
        with pytest.raises(RuntimeError, match="first-order"):
            torch.autograd.grad(y.sum(), leaf, create_graph=True)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("Tq,Tk,H,Hk,D", [(100, 1500, 2, 1, 64), (1100, 1100, 1, 1, 32), (1030, 2000, 2, 2, 128), (33, 1024, 3, 1, 96)])
def test_attention_few_blocks_over_many_keys(Tq, Tk, H, Hk, D, dtype):
    """Too few queries to fill the chip: keys are split for these too, with documents, order and a length."""
    q, k, v, do, g = _attention_inputs(1, Tq, Tk, H, Hk, D, dtype, Tq + D)
    docs = {n: _documents(g, 1, t, 3) for n, t in (("q", Tq), ("k", Tk))}
    slopes = torch.rand(H, generator=g) * 0.1
    _check_attention(q, k, v, do, causal=True, slopes=slopes)
    _check_attention(q, k, v, do, q_documents=docs["q"], k_documents=docs["k"], cap=4.0, causal=True,
                     k_lengths=torch.tensor([Tk - 70], dtype=torch.int32))


@pytest.mark.parametrize("layout,points,n", [("rows", 70000, 31000), ("maps", 9000000, 243), ("maps", 66000, 33000)])
def test_layer_norm_offsets_past_32_bits(layout, points, n):
    """More than 2^31 values: the last rows, whose gradient alone is not zero, are checked."""
    last = 5
    g = _gen(n)
    x, w, b, dy = _norm_inputs(last, n, BF16, F32, n)
    dy = dy.to(BF16)
    want = ref.layer_norm(x, w, b, 1e-5, BF16, dy)
    if layout == "rows":
        xs = torch.zeros(points, n, dtype=BF16, device="cuda")
    else:
        xs = torch.zeros(n, points, dtype=BF16, device="cuda").t()
    xs[-last:] = x.cuda()
    xs.requires_grad_()
    ws, bs = w.cuda().requires_grad_(), b.cuda().requires_grad_()
    y = tokens.layer_norm(xs, ws, bs)
    _hold(y[-last:], want["y"], "y")
    assert torch.equal(y[0], b.cuda().to(BF16)) and torch.equal(y[points - last - 1], y[0])
    dys = torch.zeros(points, n, dtype=BF16, device="cuda")
    dys[-last:] = dy.cuda()
    dx, dw, db = torch.autograd.grad(y, (xs, ws, bs), dys)
    _hold(dx[-last:], want["dx"], "dx")
    assert not bool(dx[0].any()) and not bool(dx[points - last - 1].any())
    _hold(dw, want["dw"], "dw")
    _hold(db, want["db"], "db")


def test_rotary_offsets_past_32_bits():
    T, H, D = 9000000, 4, 64
    g = _gen(3)
    x = torch.randn(1, 5, H, D, generator=g).to(BF16)
    pos = torch.randint(-(1 << 20), 1 << 20, (5, 2), generator=g, dtype=torch.int32)
    xs = torch.zeros(1, T, H, D, dtype=BF16, device="cuda")
    ps = torch.zeros(T, 2, dtype=torch.int32, device="cuda")
    xs[:, -5:], ps[-5:] = x.cuda(), pos.cuda()
    y = tokens.rotary(xs, ps, (20, 12), base=100.0)
    _hold(y[:, -5:], ref.rotary(x, pos, (20, 12), 100.0, False), "y")
    assert not bool(y[:, :1000].any()) and not bool(y[:, T - 1000:T - 5].any())


@pytest.mark.parametrize("Tq,Tk,D,how", [(300, 300, 128, "causal"), (300, 300, 64, "documents"), (1, 3000, 64, "few"), (70, 70, 12, "rows")])
def test_captured_attention_variants(Tq, Tk, D, how):
    """Each way through the kernels captured and replayed with new inputs, eager calls between."""
    q, k, v, do, g = _attention_inputs(2, Tq, Tk, 4, 2, D, BF16, 5)
    docs = _documents(g, 2, Tk, 3).cuda()
    kw = {"causal": dict(causal=True, cap=3.0), "documents": dict(q_documents=docs, k_documents=docs), "rows": dict(causal=True),
          "few": dict(k_lengths=torch.tensor([3000, 1234], dtype=torch.int32).cuda())}[how]
    still = [t.cuda() for t in (q, k, v)]
    do = do.cuda()

    def step():
        leaves = [t.detach().requires_grad_(how != "few") for t in still]
        o = tokens.attention(*leaves, **kw)
        return (o,) if how == "few" else (o.detach(), *torch.autograd.grad(o, leaves, do))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for n in range(4):
        for t in still:
            t.copy_(torch.randn(t.shape, generator=g).to(BF16))
        want = [t.clone() for t in step()]
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, want)), n


def test_calls_from_several_threads():
    """Two threads, each on a stream of its own, training steps and refusals mixed: results and messages stay apart."""
    import threading
    q, k, v, do, _ = _attention_inputs(1, 200, 200, 2, 1, 64, BF16, 6)
    leaves = [[t.cuda().requires_grad_() for t in (q, k, v)] for _ in range(2)]
    do = do.cuda()
    x = torch.randn(300, 700, device="cuda")
    want = torch.autograd.grad(tokens.attention(*leaves[0], causal=True), leaves[0], do)
    norm = tokens.layer_norm(x)
    torch.cuda.synchronize()
    wrong = []

    def work(n):
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(20):
                got = torch.autograd.grad(tokens.attention(*leaves[n], causal=True), leaves[n], do)
                y = tokens.layer_norm(x)
                try:
                    _lib.check_tokens(_lib.load().wst_layer_norm_workspace(None, None))
                    wrong.append("no refusal")
                except Exception as e:
                    if "bytes is NULL" not in str(e):
                        wrong.append(str(e))
                torch.cuda.current_stream().synchronize()
                if not all(torch.equal(a, b) for a, b in zip(got, want)) or not torch.equal(y, norm):
                    wrong.append(n)

    threads = [threading.Thread(target=work, args=(n,)) for n in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong, wrong[:3]
