"""Torch frontend: drop-in for ``from kymatio.torch import Scattering2D``.

Reference call site: src/inference/inference.py:39,242,250-254 (``S(channel_tensor)`` on a
contiguous float32 ``(1,1,H,W)`` tensor under ``torch.no_grad()``).  CUDA (ROCm) tensors are
transformed in place on their device with zero copies; CPU tensors are staged to the current
GPU and the result is returned on the CPU, so the reference's CPU-tensor call keeps working.
Gradients of the transform are not implemented (the reference only runs it under no_grad).

``ScatteringAttention`` is a trainable read-out of the transform's maps: layer norm, rotary positions and attention of
``tokens`` over the places of one image or of a series of images.
"""
from __future__ import annotations

import torch

from . import tokens
from .frontend import ScatteringBase2D, require_gpu, scatter_device


class Scattering2D(ScatteringBase2D, torch.nn.Module):
    """Scattering2D(J, shape, L=8, max_order=2, pre_pad=False, backend=None, out_type='array')."""

    def __init__(self, J, shape, L=8, max_order=2, pre_pad=False, backend=None,
                 out_type="array"):
        torch.nn.Module.__init__(self)
        ScatteringBase2D.__init__(self, J, shape, L, max_order, pre_pad, backend, out_type)

    def _prepare(self, input):
        if not torch.is_tensor(input):
            raise TypeError("The input should be a PyTorch Tensor.")
        if input.is_complex():
            raise TypeError("The input should be real.")
        self._check_spatial(tuple(input.shape), "tensor")
        if not input.is_contiguous():
            raise RuntimeError("Tensor must be contiguous.")
        require_gpu()
        batch_shape = tuple(input.shape[:-2])
        x = input.detach().reshape((-1,) + tuple(input.shape[-2:]))
        if x.dtype != torch.float32:
            x = x.to(torch.float32)
        on_cpu = not x.is_cuda
        if on_cpu:
            x = x.to("cuda")
        return x.contiguous(), batch_shape, on_cpu

    def scattering(self, input):
        x, batch_shape, on_cpu = self._prepare(input)
        with torch.no_grad():
            S = scatter_device(x, self.M, self.N, self.J, self.L, self.max_order, self.pre_pad)
        if on_cpu:
            S = S.cpu()
        S = S.reshape(batch_shape + tuple(S.shape[-3:]))
        if self.out_type == "list":
            return self._to_list(S, batch_shape)
        return S

    def pooled(self, input):
        """Per-coefficient spatial [mean | std] (population std): (..., 2K) float32."""
        x, batch_shape, on_cpu = self._prepare(input)
        with torch.no_grad():
            F = scatter_device(x, self.M, self.N, self.J, self.L, self.max_order, self.pre_pad,
                               pooled=True)
        if on_cpu:
            F = F.cpu()
        return F.reshape(batch_shape + (2 * self.K,))

    def forward(self, input):
        return self.scattering(input)

    def __call__(self, input):
        return self.scattering(input)


class ScatteringAttention(torch.nn.Module):
    """ScatteringAttention(J, shape, channels=3, heads=4, dim=32, key_heads=None, L=8, max_order=2, sections=None,
    base=10000.0, cap=30.0, dtype=torch.float32).

    Images (B, C, M, N), or series of F frames (B, F, C, M, N) -> tokens (B, F*Mo*No, heads*dim) of ``dtype``: the
    transform's maps, layer norm over a place's C*K coefficients, queries and keys turned by the place's (time, row,
    column), and attention whose scores are capped at ``cap`` (0: not) and lowered by a learned slope per head times the
    distance in time, rows and columns.  ``documents`` (B, F) int32 lays several series into one batch entry: a place
    sees the frames of its own series only, and frames of a negative number (padding) give and receive nothing (for
    gradients they have to be finite).

    ``pooled`` answers per series instead, with a learned query per head: (B, count, heads*dim).

    sections: pairs of a head that time, row and column turn (default: dim // 2 shared out evenly, the rest to rows,
    then columns).  Parameters are float32 for the norm and slopes and ``dtype`` for the projections; gradients reach
    all of them, and stop before the transform."""

    def __init__(self, J, shape, channels=3, heads=4, dim=32, key_heads=None, L=8, max_order=2, sections=None,
                 base=10000.0, cap=30.0, dtype=torch.float32):
        super().__init__()
        self.transform = Scattering2D(J, shape, L, max_order)
        self.channels, self.heads, self.dim = int(channels), int(heads), int(dim)
        self.key_heads = self.heads if key_heads is None else int(key_heads)
        self.base, self.cap = float(base), float(cap)
        if self.channels < 1 or self.heads < 1 or self.key_heads < 1 or self.heads % self.key_heads:
            raise RuntimeError(f"{self.heads} heads do not share {self.key_heads} key heads evenly")
        if not 1 <= self.dim <= tokens.MAX_HEAD_DIM:
            raise RuntimeError(f"heads must have 1 to {tokens.MAX_HEAD_DIM} values, not {self.dim}")
        if dtype not in tokens.DTYPES:
            raise TypeError(f"dtype must be float32, bfloat16 or float16, not {dtype}")
        if sections is None:
            pairs = self.dim // 2
            sections = (pairs // 3, (pairs - pairs // 3 + 1) // 2, (pairs - pairs // 3) // 2)
        self.sections = tuple(int(s) for s in sections)
        if len(self.sections) != 3 or min(self.sections) < 0 or 2 * sum(self.sections) > self.dim:
            raise RuntimeError(f"sections must be three numbers of pairs that fit heads of {self.dim} values")
        n, width, keys = self.channels * self.transform.K, self.heads * self.dim, self.key_heads * self.dim
        self.norm_weight = torch.nn.Parameter(torch.ones(n))
        self.norm_bias = torch.nn.Parameter(torch.zeros(n))
        self.qkv = torch.nn.Linear(n, width + 2 * keys, bias=False, dtype=dtype)
        # head h forgets by a factor of two within 2, 4, 8, ... places
        self.slopes = torch.nn.Parameter(0.6931472 * 2.0 ** -(1.0 + torch.arange(self.heads, dtype=torch.float32)))
        self.pool_kv = torch.nn.Linear(width, 2 * keys, bias=False, dtype=dtype)
        self.pool_query = torch.nn.Parameter(torch.randn(self.heads, self.dim, dtype=dtype))

    def _places(self, documents, x):
        """(B, F) numbers of the frames as (B, T) of their places."""
        return documents.to(x.device).repeat_interleave(self.transform.Mo * self.transform.No, 1)

    def _tokens(self, images, documents):
        if not torch.is_tensor(images):
            raise TypeError("The input should be a PyTorch Tensor.")
        if images.dim() not in (4, 5) or images.shape[-3] != self.channels:
            raise RuntimeError(f"images must be (B, {self.channels}, M, N) or (B, F, {self.channels}, M, N)")
        if images.dim() == 4:
            images = images.unsqueeze(1)
        B, F = images.shape[:2]
        if documents is not None:
            if documents.dtype != torch.int32:
                raise TypeError(f"documents must be int32, not {documents.dtype}")
            if tuple(documents.shape) != (B, F):
                raise RuntimeError(f"documents must be of shape ({B}, {F}), not {tuple(documents.shape)}")
        S = self.transform(images.to(self.slopes.device).contiguous())
        rows, cols = S.shape[-2:]
        maps = S.reshape(B, F, self.norm_weight.numel(), rows * cols)
        x = tokens.layer_norm(maps.transpose(-1, -2), self.norm_weight, self.norm_bias, out_dtype=self.qkv.weight.dtype)
        T = F * rows * cols
        if documents is not None:
            documents = self._places(documents, x)
        return x.reshape(B, T, maps.shape[2]), tokens.grid_positions(F, rows, cols, x.device), documents

    def forward(self, images, documents=None):
        x, places, documents = self._tokens(images, documents)
        B, T = x.shape[:2]
        q, k, v = self.qkv(x).view(B, T, self.heads + 2 * self.key_heads, self.dim).split((self.heads, self.key_heads, self.key_heads), 2)
        q, k = tokens.rotary(q, places, self.sections, self.base, k=k)
        o = tokens.attention(q, k, v, cap=self.cap, slopes=self.slopes.float(), q_positions=places, k_positions=places,
                             q_documents=documents, k_documents=documents)
        return o.reshape(B, T, self.heads * self.dim)

    def pooled(self, images, documents=None, count=1):
        """(B, count, heads*dim): series 0 to count - 1 of each batch entry (without documents, count is 1), each read
        out by one query; a series without frames gives 0."""
        count = int(count)
        if count < 1 or (documents is None and count != 1):
            raise RuntimeError("count is the number of series that documents tell apart")
        x = self.forward(images, documents)
        B, T = x.shape[:2]
        k, v = self.pool_kv(x).view(B, T, 2 * self.key_heads, self.dim).split((self.key_heads, self.key_heads), 2)
        q = self.pool_query.to(k.dtype).expand(B, count, -1, -1)        # autocast gives k another type
        if documents is not None:
            documents = self._places(documents, x)
            series = torch.arange(count, dtype=torch.int32, device=x.device)
            o = tokens.attention(q, k, v, q_documents=series, k_documents=documents)
        else:
            o = tokens.attention(q, k, v)
        return o.reshape(B, count, self.heads * self.dim)
