"""Drop-in for src/model/embeddings.py: TokenEmbedding (parameter ``embedding.weight``), whose
weight the Transformer ties to its output projection (src/model/embeddings.py:7-34), and the scaled
lookup ``embedding`` behind its ``scale``: HIP kernels, forward (pe_embed_fwd) and the weight's
gradient (pe_embed_bwd), which sorts the tokens by id and adds each id's rows in order.
"""

from typing import Optional

import torch
import torch.nn as nn
import torch.nn.functional as F

from . import _lib
from .functional import _call, _ptr, _stream, plain_autograd

_FLOATS = {torch.bfloat16: _lib.PE_DTYPE_BF16, torch.float32: _lib.PE_DTYPE_FP32, torch.float16: _lib.PE_DTYPE_FP16}
_INTS = (torch.int64, torch.int32)
_MAX_TOKENS = 1 << 24


def _check(ids: torch.Tensor, weight: torch.Tensor, padding_idx: Optional[int]) -> int:
    """The checks of an embedding call; padding_idx as the C ABI takes it (-1 for none)."""
    if not weight.is_cuda:
        raise RuntimeError("embedding runs on the GPU only (got a CPU weight)")
    if weight.dim() != 2:
        raise ValueError(f"embedding: weight must be (vocab, dim), got shape {tuple(weight.shape)}")
    return _check_parts(ids, weight.shape[0], weight.shape[1], weight.dtype, weight.device, padding_idx)


def _check_parts(ids, V: int, H: int, dtype: torch.dtype, dev: torch.device, padding_idx: Optional[int]) -> int:
    if V <= 0 or H <= 0:
        raise ValueError(f"embedding: the weight must have rows and columns, got ({V}, {H})")
    if dtype not in _FLOATS:
        raise TypeError(f"embedding supports bf16 / fp16 / fp32 weights, got {dtype}")
    if ids.dtype not in _INTS:
        raise TypeError(f"embedding: ids must be int64 or int32, got {ids.dtype}")
    if ids.device != dev:
        raise ValueError(f"embedding: ids are on {ids.device}, the weight on {dev}")
    if padding_idx is None:
        return -1
    if not -V <= padding_idx < V:
        raise ValueError(f"embedding: padding_idx {padding_idx} is outside a vocabulary of {V}")
    return padding_idx % V


def _rows(t: torch.Tensor, H: int) -> torch.Tensor:
    """A (rows, H) tensor that the library can read: unit stride, rows not overlapping (one row may have any)."""
    return t if t.stride(1) == 1 and t.stride(0) >= H else t.contiguous()


def _lookup(ids: torch.Tensor, weight: torch.Tensor, scale: float) -> torch.Tensor:
    V, H = weight.shape
    weight, ids = _rows(weight, H), ids.contiguous()
    dev = weight.device
    out = torch.empty(ids.shape + (H,), dtype=weight.dtype, device=dev)
    n = ids.numel()
    if n:
        _call(dev, _lib.lib().pe_embed_fwd, ids.data_ptr(), ids.element_size(), n, weight.data_ptr(),
              _FLOATS[weight.dtype], V, H, max(weight.stride(0), H), scale, out.data_ptr(), H, _stream(dev))
    return out


def _gradient(ids: torch.Tensor, dy: torch.Tensor, V: int, scale: float, pad: int) -> torch.Tensor:
    """embedding_backward on checked arguments (pad: -1 for none)."""
    H, n, dev = dy.shape[-1], ids.numel(), dy.device
    if dy.dim() != 2:
        dy = dy.reshape(-1, H)
    dy, ids = _rows(dy, H), ids.contiguous()
    dw = torch.empty((V, H), dtype=dy.dtype, device=dev)
    L = _lib.lib()
    nb = L.pe_embed_bwd_workspace_bytes(n, V, H)
    ws = torch.empty(nb, dtype=torch.uint8, device=dev) if nb else None  # held until the launch is enqueued
    _call(dev, L.pe_embed_bwd, ids.data_ptr(), ids.element_size(), n, dy.data_ptr(), _FLOATS[dy.dtype],
          max(dy.stride(0), H), V, H, scale, pad, dw.data_ptr(), H, _ptr(ws), nb, _stream(dev))
    return dw


def embedding_backward(ids: torch.Tensor, dy: torch.Tensor, vocab_size: int, *, scale: float = 1.0,
                       padding_idx: Optional[int] = None) -> torch.Tensor:
    """The weight gradient (vocab_size, dim) of ``embedding(ids, weight, scale=scale)`` for the upstream
    gradient dy (*ids.shape, dim), in dy's dtype: scale times the sum of each id's rows, in the order of the
    tokens, in fp32 (bitwise reproducible).  padding_idx's row is 0; ids outside the vocabulary add nothing."""
    if not dy.is_cuda:
        raise RuntimeError("embedding_backward runs on the GPU only (got a CPU tensor)")
    if dy.dim() != ids.dim() + 1 or dy.shape[:-1] != ids.shape:
        raise ValueError(f"embedding_backward: dy {tuple(dy.shape)} must be ids {tuple(ids.shape)} plus a last dim")
    if ids.numel() > _MAX_TOKENS:
        raise ValueError(f"embedding_backward: {ids.numel()} tokens in one call, at most {_MAX_TOKENS} are supported")
    pad = _check_parts(ids, vocab_size, dy.shape[-1], dy.dtype, dy.device, padding_idx)
    return _gradient(ids, dy, vocab_size, float(scale), pad)


def _gradient_expression(ids: torch.Tensor, dy: torch.Tensor, V: int, scale: float, pad: int) -> torch.Tensor:
    """_gradient in torch operations, which higher derivatives differentiate (it is linear in dy)."""
    ids = ids.reshape(-1).long()
    keep = (ids >= 0) & (ids < V) & (ids != pad)
    rows = torch.where(keep[:, None], dy.reshape(ids.numel(), dy.shape[-1]).float(), 0.0)
    dw = torch.zeros((V, dy.shape[-1]), device=dy.device).index_add(0, torch.where(keep, ids, 0), rows)
    return (dw * scale).to(dy.dtype)


class EmbeddingFn(torch.autograd.Function):
    """The lookup with pe_embed_bwd as its backward.  It keeps the ids alone, as F.embedding does: the weight may be
    changed in place before the backward.  Under create_graph and with batched gradients the backward is the
    gradient in torch operations."""

    @staticmethod
    def forward(ctx, weight, ids, scale, pad):
        ctx.save_for_backward(ids)
        ctx.rows, ctx.scale, ctx.pad = weight.shape[0], scale, pad
        return _lookup(ids, weight, scale)

    @staticmethod
    def backward(ctx, dy):
        (ids,) = ctx.saved_tensors
        fn = _gradient if plain_autograd(dy) and not torch.is_grad_enabled() else _gradient_expression
        return fn(ids, dy, ctx.rows, ctx.scale, ctx.pad), None, None, None


def embedding(ids: torch.Tensor, weight: torch.Tensor, *, scale: float = 1.0,
              padding_idx: Optional[int] = None) -> torch.Tensor:
    """weight[ids] * scale, (*ids.shape, dim) in the weight's dtype, the product in fp32 and rounded once.
    weight (vocab, dim) bf16 / fp16 / fp32 on the GPU, ids int64 / int32 on the same device.  Differentiable in
    the weight (embedding_backward); the rows of padding_idx get no gradient.  An id outside the vocabulary
    cannot be refused without waiting for the GPU: its row is NaN.  Where something other than plain autograd looks
    at the weight (functorch, forward mode, tracing, compiling) it is F.embedding(ids, weight) * scale."""
    pad = _check(ids, weight, padding_idx)
    if not plain_autograd(weight):
        return F.embedding(ids, weight, None if pad < 0 else pad) * scale
    if weight.requires_grad and torch.is_grad_enabled():
        if ids.numel() > _MAX_TOKENS:
            raise ValueError(f"embedding: {ids.numel()} tokens in one call with gradients, at most {_MAX_TOKENS}")
        return EmbeddingFn.apply(weight, ids, float(scale), pad)
    return _lookup(ids, weight, float(scale))


class TokenEmbedding(nn.Module):
    """``scale`` (an addition; default None = the reference's plain lookup through torch): the rows times this
    factor, sqrt(embed_dim) in models that tie the weight to an output projection, through ``embedding``."""

    scale: Optional[float] = None  # also of a module pickled without one

    def __init__(self, vocab_size: int, embed_dim: int, scale: Optional[float] = None):
        super().__init__()
        self.vocab_size = vocab_size
        self.embed_dim = embed_dim
        self.scale = scale
        self.embedding = nn.Embedding(vocab_size, embed_dim)

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        if self.scale is None:
            return self.embedding(x)
        return embedding(x, self.embedding.weight, scale=self.scale)

    @property
    def weight(self) -> torch.Tensor:
        return self.embedding.weight
