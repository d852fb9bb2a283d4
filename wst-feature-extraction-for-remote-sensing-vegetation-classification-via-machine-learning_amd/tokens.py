"""Operators on coefficient tokens: what a network behind the transform does with its maps.

A scattering map of (C, K, Mo, No) is a sequence of Mo * No tokens of C * K values each.  The reference reads such maps
out by the mean and standard deviation of each coefficient (train_and_save_model.py:371-375); these operators are the
learned counterpart, for training and inference:

* ``layer_norm``  -- over a token's values; reads tokens, or maps where the transform wrote them;
* ``rotary``      -- positions with several axes (time, row, column) turned into queries and keys;
* ``attention``   -- scores capped by tanh, a bias that depends on distance, documents, order and a prefix.

All run in the HIP library on the tensors' device and current stream, have gradients (torch autograd, first order), and
can be captured into a graph (a backward pass: while no eager autograd graph of the same leaves is alive, since torch's
engine would wait for that graph's stream inside the capture).  Forward-mode derivatives and tracing
(``torch.jit.trace``) are refused.  float32, bfloat16 and float16; sums and statistics are held in float32.  There is
no CPU execution: tensors must live on a ROCm GPU.
"""
from __future__ import annotations

import ctypes

import torch
from torch.autograd import forward_ad

from . import _lib
from .frontend import require_gpu

DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
MAX_HEAD_DIM = _lib.MAX_HEAD_DIM


def _dtype_id(t, name):
    try:
        return DTYPES[t.dtype]
    except KeyError:
        raise TypeError(f"{name} must be float32, bfloat16 or float16, not {t.dtype}") from None


def _check_tensor(t, name, like=None):
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a PyTorch Tensor.")
    if not t.is_cuda:
        require_gpu()
        raise RuntimeError(f"{name} must be on a ROCm GPU, not on {t.device}")
    if like is not None and t.get_device() != like.get_device():
        raise RuntimeError(f"{name} is on {t.device}, expected {like.device}")


def _check_ints(t, name, like):
    _check_tensor(t, name, like)
    if t.dtype != torch.int32:
        raise TypeError(f"{name} must be int32, not {t.dtype}")


def _call(index, fn, *args):
    """Run a library call on the tensors' device and its current stream, and check the status."""
    stream = torch._C._cuda_getCurrentRawStream(index)
    if index == torch._C._cuda_getDevice():
        code = fn(*args, stream)
    else:
        with torch.cuda.device(index):
            code = fn(*args, stream)
    if code:
        _lib.check_tokens(code)


def _first_order():
    """Called by the backward passes: they have no backward pass of their own."""
    if torch.is_grad_enabled():
        raise RuntimeError("the token operators have first-order gradients only")


def _wants_grad(*tensors):
    # The library reads memory that neither of these follows: a tangent would be dropped, a trace would hold the result's
    # allocation without the call.
    if torch._C._is_tracing():
        raise RuntimeError("the token operators cannot be traced")
    if forward_ad._current_level >= 0 and any(t is not None and forward_ad.unpack_dual(t).tangent is not None for t in tensors):
        raise RuntimeError("the token operators have no forward-mode derivatives")
    return torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors)


# ------------------------------------------------------------------------------------------ layer norm
def _token_view(x):
    """x (..., n) as (batch, points, n) strides the library reads, copied only when it has none."""
    n = x.shape[-1]
    if x.is_contiguous():
        return x, (1, x.numel() // n, n, 0, n, 1)
    lead = []                                   # (size, stride) of the leading dimensions, merged where adjacent
    for size, stride in zip(x.shape[:-1], x.stride()[:-1]):
        if size == 1:
            continue
        if lead and lead[-1][1] == size * stride:
            lead[-1] = (lead[-1][0] * size, stride)
        else:
            lead.append((size, stride))
    sn = x.stride(-1)
    batch, sb = lead[0] if len(lead) == 2 else (1, 0)
    points, sp = lead[-1] if lead else (1, n)
    if len(lead) > 2 or not (sn == 1 or n == 1 or sp == 1 or points == 1):
        x, rows = x.contiguous(), x.numel() // n
        return x, (1, rows, n, 0, n, 1)
    return x, (batch, points, n, sb, sp, sn)


def _norm_desc(view, dview, x, out_dtype, weight, bias, eps):
    w = weight if weight is not None else bias
    return _lib.NORM_PACK.pack(*view, *dview, DTYPES[x.dtype], DTYPES[out_dtype], 0 if w is None else DTYPES[w.dtype], eps)


def _ptr(t):
    return None if t is None else t.data_ptr()


def _like(t):
    """A new contiguous tensor of t's size and type; empty_like takes half the time of empty with its arguments."""
    return torch.empty_like(t) if t.is_contiguous() else torch.empty(t.shape, dtype=t.dtype, device=t.device)


def _norm_forward(x, weight, bias, eps, out_dtype, stats):
    xs, view = _token_view(x)
    y = _like(x) if out_dtype == x.dtype else torch.empty(x.shape, dtype=out_dtype, device=x.device)
    rows = view[0] * view[1]
    kept = mean = rstd = None
    if stats:                                   # means, then 1 / deviations
        kept = torch.empty(2 * rows, dtype=torch.float32, device=x.device)
        mean = kept.data_ptr()
        rstd = mean + 4 * rows
    if x.numel():
        d = _norm_desc(view, (0, 0, 0), x, out_dtype, weight, bias, eps)
        _call(x.get_device(), _lib.token_calls().layer_norm_forward, d, xs.data_ptr(), _ptr(weight), _ptr(bias), y.data_ptr(),
              mean, rstd)
    return y, xs, kept


class _LayerNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, eps, out_dtype):
        y, xs, kept = _norm_forward(x, weight, bias, eps, out_dtype, True)
        ctx.save_for_backward(xs, weight, kept)
        ctx.bias_like = None if bias is None else (bias.shape, bias.dtype)
        ctx.eps, ctx.x_shape = eps, x.shape
        return y

    @staticmethod
    def backward(ctx, dy):
        _first_order()
        xs, weight, kept = ctx.saved_tensors
        want_x, want_w, want_b = ctx.needs_input_grad[:3]
        dx = dw = db = None
        dev = xs.device
        if want_w:
            dw = torch.empty_like(weight)
        if want_b:
            db = torch.empty(ctx.bias_like[0], dtype=ctx.bias_like[1], device=dev) if weight is None else torch.empty_like(weight)
        if not xs.numel():
            return (torch.empty(ctx.x_shape, dtype=xs.dtype, device=dev) if want_x else None,
                    dw.zero_() if want_w else None, db.zero_() if want_b else None, None, None)
        _, view = _token_view(xs)
        batch, points, n = view[:3]
        dview = (points * n, n, 1)
        if want_x:
            if view[5] != 1 and n > 1:          # maps: the gradient lies as they do
                dx = torch.empty((batch, n, points), dtype=xs.dtype, device=dev).transpose(1, 2)
                dview = (points * n, 1, points)
                dx = dx.view(ctx.x_shape)
            else:
                dx = _like(xs)
        dy = dy.resolve_neg().contiguous()
        d = _lib.NORM_PACK.pack(*view, *dview, DTYPES[xs.dtype], DTYPES[dy.dtype],
                                DTYPES[weight.dtype] if weight is not None else DTYPES[db.dtype] if want_b else 0, ctx.eps)
        lib, need = _lib.token_calls(), ctypes.c_size_t()
        _lib.check_tokens(lib.layer_norm_workspace(d, ctypes.byref(need)))
        ws = torch.empty(need.value, dtype=torch.uint8, device=dev)
        _call(xs.get_device(), lib.layer_norm_backward, d, xs.data_ptr(), _ptr(weight), dy.data_ptr(), kept.data_ptr(),
              kept.data_ptr() + 4 * batch * points, _ptr(dx), _ptr(dw), _ptr(db), ws.data_ptr(), need.value)
        return dx, dw, db, None, None


def layer_norm(x, weight=None, bias=None, eps=1e-5, out_dtype=None):
    """Layer norm over the last axis: ``(x - mean) / sqrt(var + eps) * weight + bias`` (population variance).

    x (..., n) may lie with its values adjacent, or with its tokens adjacent: ``maps.flatten(-2).transpose(-1, -2)`` of
    the transform's maps is read in place.  The result is contiguous, of ``out_dtype`` (default x's).  weight and bias
    (n,) may have a type of their own, the same for both; either may be None."""
    _check_tensor(x, "x")
    _dtype_id(x, "x")
    if x.dim() < 1 or x.shape[-1] < 1:
        raise RuntimeError("x must have a last axis of at least one value")
    out_dtype = x.dtype if out_dtype is None else out_dtype
    if out_dtype not in DTYPES:
        raise TypeError(f"out_dtype must be float32, bfloat16 or float16, not {out_dtype}")
    for t, name in ((weight, "weight"), (bias, "bias")):
        if t is not None:
            _check_tensor(t, name, x)
            _dtype_id(t, name)
            if t.shape != x.shape[-1:]:
                raise RuntimeError(f"{name} must be of shape ({x.shape[-1]},), not {tuple(t.shape)}")
    if weight is not None and bias is not None and weight.dtype != bias.dtype:
        raise TypeError("weight and bias must have the same type")
    eps = float(eps)
    if not eps >= 0.0:
        raise RuntimeError("eps must not be negative")
    x = x.resolve_neg()                         # a view that negates when it is read, which the library would not
    weight = None if weight is None else weight.resolve_neg().contiguous()
    bias = None if bias is None else bias.resolve_neg().contiguous()
    if _wants_grad(x, weight, bias):
        return _LayerNorm.apply(x, weight, bias, eps, out_dtype)
    return _norm_forward(x, weight, bias, eps, out_dtype, False)[0]


# ------------------------------------------------------------------------------------------ rotary
def grid_positions(frames, rows, cols, device=None):
    """(frames * rows * cols, 3) int32 positions (time, row, column) of a series of maps, in the maps' order."""
    axes = [torch.arange(n, dtype=torch.int32, device=device) for n in (frames, rows, cols)]
    return torch.stack(torch.meshgrid(*axes, indexing="ij"), -1).reshape(-1, 3)


def _rows_of(t):
    return t if t.stride(-1) == 1 or t.shape[-1] == 1 else t.contiguous()


def _strides(t):
    return t.stride()[:3]


def _lined_up(t):
    """t with rows the library can fetch 16 bytes at a time (heads of other widths go value by value anyway)."""
    if t.is_contiguous() and t.data_ptr() % 16 == 0:
        return t
    t = _rows_of(t)
    if t.shape[-1] % 8 == 0:
        size = t.element_size()
        if t.data_ptr() % 16 or any(s * size % 16 for s, n in zip(t.stride()[:3], t.shape) if n > 1):
            return t.clone(memory_format=torch.contiguous_format)
    return t


def _call_strides(t):
    """The strides of t for a call; of an axis of one entry, which is never stepped along, 0."""
    if t.is_contiguous():
        return t.stride()[:3]
    return tuple(s if n > 1 else 0 for s, n in zip(t.stride()[:3], t.shape))


def _rotate(q, k, positions, sections, base, interleaved, inverse):
    q = _rows_of(q)
    B, T, H, D = q.shape
    qo = _like(q)
    ko, ks, kos, Hk = None, (0, 0, 0), (0, 0, 0), 0
    if k is not None:
        k = _rows_of(k)
        ko, Hk = _like(k), k.shape[2]
        ks, kos = _strides(k), _strides(ko)
    d = _lib.ROTARY_PACK.pack(B, T, *_strides(q), *ks, *_strides(qo), *kos, base, H, Hk, D, DTYPES[q.dtype], len(sections),
                              *sections, *(0,) * (_lib.MAX_AXES - len(sections)), interleaved, inverse, positions.dim() == 2)
    _call(q.get_device(), _lib.token_calls().rotary, d, q.data_ptr(), qo.data_ptr(), _ptr(k), _ptr(ko), positions.data_ptr())
    return qo, ko


class _Rotary(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, positions, sections, base, interleaved):
        ctx.save_for_backward(positions)
        ctx.how = (sections, base, interleaved)
        qo, ko = _rotate(q, k, positions, sections, base, interleaved, 0)
        return qo if k is None else (qo, ko)

    @staticmethod
    def backward(ctx, dq, dk=None):
        _first_order()
        positions, = ctx.saved_tensors
        gq, gk = _rotate(dq.resolve_neg(), None if dk is None else dk.resolve_neg(), positions, *ctx.how, 1)
        return gq, gk, None, None, None, None


def rotary(q, positions, sections, base=10000.0, interleaved=False, k=None):
    """Rotary positions with several axes.

    q (B, T, H, D) and, in the same call, k (B, T, Hk, D); positions int32 (T, A) or (B, T, A), 1 <= A <= 4, such as
    ``grid_positions``; sections: the pairs that each of the A axes turns, 128 in all at most.  The first
    2 * sum(sections) values of a head are turned, the rest copied.  Pair i of an axis with s pairs turns by ``position * base**(-i / s)``.  With P pairs in
    all, pair p is the values (p, p + P), or (2p, 2p + 1) when ``interleaved``.  Returns q turned, or (q, k)."""
    _check_tensor(q, "q")
    _dtype_id(q, "q")
    if q.dim() != 4:
        raise RuntimeError("q must be (batch, tokens, heads, dim)")
    B, T, _, D = q.shape
    if k is not None:
        _check_tensor(k, "k", q)
        if k.dtype != q.dtype:
            raise TypeError("q and k must have the same type")
        if k.dim() != 4 or k.shape[:2] != q.shape[:2] or k.shape[3] != D:
            raise RuntimeError(f"k must be ({B}, {T}, heads, {D}), not {tuple(k.shape)}")
    sections = tuple(int(s) for s in sections)
    if not 1 <= len(sections) <= _lib.MAX_AXES or min(sections) < 0:
        raise RuntimeError(f"sections must be 1 to {_lib.MAX_AXES} numbers of pairs")
    if 2 * sum(sections) > D:
        raise RuntimeError(f"{sum(sections)} pairs do not fit heads of {D} values")
    if sum(sections) > _lib.MAX_PAIRS:
        raise RuntimeError(f"sections must turn at most {_lib.MAX_PAIRS} pairs, not {sum(sections)}")
    _check_ints(positions, "positions", q)
    A = len(sections)
    if tuple(positions.shape) not in ((T, A), (B, T, A)):
        raise RuntimeError(f"positions must be ({T}, {A}) or ({B}, {T}, {A}), not {tuple(positions.shape)}")
    base = float(base)
    if not 0.0 < base < float("inf"):
        raise RuntimeError("base must be positive")
    positions = positions.contiguous()
    q, k = q.resolve_neg(), None if k is None else k.resolve_neg()
    if _wants_grad(q, k):
        return _Rotary.apply(q, k, positions, sections, base, bool(interleaved))
    qo, ko = _rotate(q, k, positions, sections, base, bool(interleaved), 0)
    return qo if k is None else (qo, ko)


# ------------------------------------------------------------------------------------------ attention
class _Side:
    """The arguments of a call that have no gradient, and their part of the descriptor."""
    __slots__ = ("scale", "cap", "q_pos", "k_pos", "q_doc", "k_doc", "k_lengths", "prefix", "causal", "axes", "strides", "ptrs")

    def tensors(self):
        return (self.q_pos, self.k_pos, self.q_doc, self.k_doc, self.k_lengths, self.prefix)

    def settle(self):
        q_pos, k_pos, q_doc, k_doc, k_lengths, prefix = self.tensors()
        self.axes = 0 if q_pos is None else q_pos.shape[-1]
        self.strides = (_per_batch(q_pos, 3), _per_batch(k_pos, 3), _per_batch(q_doc, 2), _per_batch(k_doc, 2))
        self.ptrs = (_ptr0(q_pos), _ptr0(k_pos), _ptr0(q_doc), _ptr0(k_doc), _ptr0(k_lengths), _ptr0(prefix))


def _per_batch(t, dims):
    return 0 if t is None or t.dim() < dims else t.stride(0)


def _ptr0(t):
    return 0 if t is None else t.data_ptr()


def _attention_desc(q, k, v, slopes, side, o, rest):
    B, Tq, H, D = q.shape
    return _lib.ATTENTION_PACK.pack(
        B, Tq, k.shape[1], *_call_strides(q), *_call_strides(k), *_call_strides(v), *_strides(o), *side.strides, q.data_ptr(),
        k.data_ptr(), v.data_ptr(), _ptr0(slopes), *side.ptrs, _ptr0(rest), side.scale, side.cap, H, k.shape[2], D,
        DTYPES[q.dtype], side.axes, side.causal)


def _grad_strides(t):
    return (0, 0, 0) if t is None else t.stride()[:3]


def _workspace(d, backward, device):
    need = ctypes.c_size_t()
    _lib.check_tokens(_lib.token_calls().attention_workspace(d, backward, ctypes.byref(need)))
    return torch.empty(need.value, dtype=torch.uint8, device=device) if need.value else None, need.value


def _attend(q, k, v, slopes, side, want_lse, want_rest):
    """o, the scores' log-sum-exp, and for a backward pass what rounding o took from it (nothing in float32)."""
    B, Tq, H, _ = q.shape
    o = _like(q)
    rest = torch.empty_like(o) if want_rest and q.dtype != torch.float32 else None
    lse = torch.empty((B, H, Tq), dtype=torch.float32, device=q.device) if want_lse else None
    d = _attention_desc(q, k, v, slopes, side, o, rest)
    ws, size = _workspace(d, 0, q.device)
    _call(q.get_device(), _lib.token_calls().attention_forward, d, o.data_ptr(), _ptr(lse), _ptr(ws), size)
    return o, lse, rest


class _Attention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, slopes, side):
        o, lse, rest = _attend(q, k, v, slopes, side, True, True)
        ctx.save_for_backward(q, k, v, slopes, o, lse, rest, *side.tensors())
        ctx.side = side
        ctx.mark_non_differentiable(lse)
        return o, lse

    @staticmethod
    def backward(ctx, do, _):
        _first_order()
        q, k, v, slopes, o, lse, rest = ctx.saved_tensors[:7]
        want = ctx.needs_input_grad
        dq, dk, dv = _like(q) if want[0] else None, _like(k) if want[1] else None, _like(v) if want[2] else None
        dslopes = torch.empty_like(slopes) if want[3] else None
        if not q.numel() or not k.numel():
            return tuple(None if t is None else t.zero_() for t in (dq, dk, dv, dslopes)) + (None,)
        do = _lined_up(do.resolve_neg())
        d = _attention_desc(q, k, v, slopes, ctx.side, o, rest)
        g = _lib.GRADS_PACK.pack(o.data_ptr(), do.data_ptr(), lse.data_ptr(), _ptr0(dq), _ptr0(dk), _ptr0(dv), _ptr0(dslopes),
                                 *_call_strides(do), *_grad_strides(dq), *_grad_strides(dk), *_grad_strides(dv))
        ws, size = _workspace(d, 1, q.device)
        _call(q.get_device(), _lib.token_calls().attention_backward, d, g, _ptr(ws), size)
        return dq, dk, dv, dslopes, None


def _check_side(t, name, like, shapes):
    if t is None:
        return None
    _check_ints(t, name, like)
    if tuple(t.shape) not in shapes:
        raise RuntimeError(f"{name} must be of shape {' or '.join(str(s) for s in shapes)}, not {tuple(t.shape)}")
    return t.contiguous()


def attention(q, k, v, *, scale=None, cap=0.0, slopes=None, q_positions=None, k_positions=None, q_documents=None,
              k_documents=None, causal=False, prefix=None, k_lengths=None, return_lse=False):
    """Softmax attention of q (B, Tq, H, D) over k, v (B, Tk, Hk, D); H a multiple of Hk, D <= 256, B and H <= 65535.

    With ``L = k_lengths[b]`` (default Tk) and ``place(i) = i + L - Tq``, query i scores key j as
    ``z = scale * q_i.k_j`` (scale defaults to ``D ** -0.5``), ``z = cap * tanh(z / cap)`` where ``cap > 0`` (1e-30 to 1e30), and
    ``z - slopes[h] * distance``: slopes float32 (H,); the distance is the sum over axes of
    ``|q_positions[i] - k_positions[j]|`` (int32 (T, A) or (B, T, A), A <= 3, within +-2**29), or ``|place(i) - j|``
    without positions.  Key j is seen iff

    * ``j < L`` (k_lengths int32 (B,): keys behind are not read into any result), and
    * ``j <= place(i)`` where ``causal`` or a prefix is given, or ``j < prefix[b]`` (int32 (B,)), and
    * ``q_documents[i] == k_documents[j] >= 0`` where given (int32 (T,) or (B, T); negative belongs to none).

    What is not seen has no influence, not even infinities or NaN.  A query that sees nothing gets 0, and no gradient.
    16-bit types round the weights that multiply v, and the score gradients that multiply q and k, to their own type.
    Gradients reach q, k, v and slopes.  In float16 the backward pass does rows and keys whose score gradients exceed
    2**10 over, one by one: right, but slow where a loss scale makes that most of them (1024 tokens, 8 heads of 64: 100 us,
    with output gradients of 2**10 450 us and of 2**13 5.3 ms); bfloat16 has no such bound.  So it is in every type for
    rows and keys that see a value that is not finite.  Returns o (B, Tq, H, D), and with ``return_lse`` the float32 (B, H, Tq)
    log-sum-exp of the scores (-inf where nothing is seen; it has no gradient)."""
    for t, name in ((q, "q"), (k, "k"), (v, "v")):
        _check_tensor(t, name, q if t is not q else None)
        _dtype_id(t, name)
        if t.dim() != 4:
            raise RuntimeError(f"{name} must be (batch, tokens, heads, dim)")
        if t.dtype != q.dtype:
            raise TypeError("q, k and v must have the same type")
    B, Tq, H, D = q.shape
    Tk, Hk = k.shape[1:3]
    if k.shape != v.shape or k.shape[0] != B or k.shape[3] != D:
        raise RuntimeError(f"k and v must be ({B}, tokens, heads, {D}), not {tuple(k.shape)} and {tuple(v.shape)}")
    if Hk < 1 or H < 1 or H % Hk:
        raise RuntimeError(f"{H} query heads do not share {Hk} key heads evenly")
    if not 1 <= D <= _lib.MAX_HEAD_DIM:
        raise RuntimeError(f"heads must have 1 to {_lib.MAX_HEAD_DIM} values, not {D}")
    if slopes is not None:
        _check_tensor(slopes, "slopes", q)
        if slopes.dtype != torch.float32:
            raise TypeError(f"slopes must be float32, not {slopes.dtype}")
        if slopes.shape != (H,):
            raise RuntimeError(f"slopes must be of shape ({H},), not {tuple(slopes.shape)}")
        slopes = slopes.resolve_neg().contiguous()
    if (q_positions is None) != (k_positions is None) or (q_documents is None) != (k_documents is None):
        raise RuntimeError("positions and documents are given for queries and keys alike")
    if q_positions is not None and slopes is None:
        raise RuntimeError("positions are of use with slopes only")
    s = _Side()
    A = 0
    if q_positions is not None and torch.is_tensor(q_positions):
        A = q_positions.shape[-1] if q_positions.dim() else 0
        if not 1 <= A <= _lib.MAX_DISTANCE_AXES:
            raise RuntimeError(f"positions must have 1 to {_lib.MAX_DISTANCE_AXES} axes")
    s.q_pos = _check_side(q_positions, "q_positions", q, ((Tq, A), (B, Tq, A)))
    s.k_pos = _check_side(k_positions, "k_positions", q, ((Tk, A), (B, Tk, A)))
    s.q_doc = _check_side(q_documents, "q_documents", q, ((Tq,), (B, Tq)))
    s.k_doc = _check_side(k_documents, "k_documents", q, ((Tk,), (B, Tk)))
    s.k_lengths = _check_side(k_lengths, "k_lengths", q, ((B,),))
    s.prefix = _check_side(prefix, "prefix", q, ((B,),))
    s.causal = bool(causal) or prefix is not None
    s.scale = D ** -0.5 if scale is None else float(scale)
    s.cap = float(cap)
    if s.cap != 0.0 and not 1e-30 <= s.cap <= 1e30:
        raise RuntimeError("cap must be 0 (none) or from 1e-30 to 1e30")
    if not abs(s.scale) < float("inf"):
        raise RuntimeError("scale must be finite")
    s.settle()
    q, k, v = _lined_up(q.resolve_neg()), _lined_up(k.resolve_neg()), _lined_up(v.resolve_neg())
    if _wants_grad(q, k, v, slopes):
        o, lse = _Attention.apply(q, k, v, slopes, s)
    else:
        o, lse, _ = _attend(q, k, v, slopes, s, return_lse, False)
    return (o, lse) if return_lse else o
