"""Losses over the vocabulary, forward and backward in HIP kernels (include/pe_vocab.h).

``cross_entropy`` is the next-token loss of src/model/transformer.py:357-364, ``distillation_loss`` adds the
divergence from a teacher's top logits, and ``loss_and_grad`` gives either with the gradient of the logits from
one call, which reads the logits once where a forward and a backward read them twice.

For a row with logits z (V,), label y and teacher pairs (id_k, t_k):

    hard = -log softmax(z)[y]
    soft = T^2 * sum_k p_k (log p_k - log softmax(z / T)[id_k]),   p = softmax(t / T) over the row's pairs
    row  = (1 - soft_weight) * hard + soft_weight * soft

A row whose label is ignore_index does not count: its loss and gradient are 0, and its logits are not read.
``reduction`` "mean" divides by the rows that count (none: NaN, as F.cross_entropy), "sum" adds them up, "none"
gives every row's loss (its negative is the token's log probability).  ``shift=True`` takes logits (..., S, V) and
labels (..., S) of the same positions and holds row s to label s + 1, without the shifted copy of the logits that
slicing would make; the last row of each sequence does not count.

At high temperatures the soft part is T^2 times a small difference of numbers near log V and keeps that many digits
fewer (about 1e-4 absolute at T = 10); its gradient does not suffer.

Everything is computed in fp32 from bf16, fp16 or fp32 logits, losses are fp32, gradients are rounded once to the
logits' dtype; sums run in a fixed order.  The differentiable forms keep the logits for their backward, so these must
not be changed in place in between (autograd notices).  Where something other than plain autograd looks at the logits
(functorch, forward mode, tracing, compiling) the losses are the same expressions in torch operations.  A label that is neither in the vocabulary nor ignore_index, which
cannot be refused without waiting for the GPU, makes its row's loss and gradient NaN.
"""

from __future__ import annotations

import ctypes
from typing import Optional, Union

import torch

from . import _lib
from .functional import _call, _expression_grads, _ptr, _stream, plain_autograd

_FLOATS = {torch.bfloat16: _lib.PE_DTYPE_BF16, torch.float32: _lib.PE_DTYPE_FP32, torch.float16: _lib.PE_DTYPE_FP16}
_INTS = (torch.int64, torch.int32)
_REDUCTION = {"none": _lib.PE_LOSS_NONE, "sum": _lib.PE_LOSS_SUM, "mean": _lib.PE_LOSS_MEAN}


def _prepare(what, logits, labels, teacher_ids, teacher_logits, temperature, soft_weight, ignore_index, reduction, shift):
    """Checks a call; (parameter block, logits as rows, labels, teacher ids, teacher logits)."""
    if not logits.is_cuda:
        raise RuntimeError(f"{what} runs on the GPU only (got CPU logits)")
    if logits.dtype not in _FLOATS:
        raise TypeError(f"{what} supports bf16 / fp16 / fp32 logits, got {logits.dtype}")
    if logits.dim() < (2 if shift else 1) or logits.shape[-1] == 0:
        raise ValueError(f"{what}: logits must be ({'..., S, V' if shift else '..., V'}), got shape {tuple(logits.shape)}")
    lead, V, dev = logits.shape[:-1], logits.shape[-1], logits.device
    if reduction not in _REDUCTION:
        raise ValueError(f"{what}: reduction must be 'none', 'sum' or 'mean', got {reduction!r}")
    if labels is None:
        if soft_weight != 1.0:
            raise ValueError(f"{what}: without labels there is no hard part, soft_weight must be 1, got {soft_weight}")
        if shift:
            raise ValueError(f"{what}: shift moves the labels, there are none")
    else:
        if labels.dtype not in _INTS:
            raise TypeError(f"{what}: labels must be int64 or int32, got {labels.dtype}")
        if labels.shape != lead:
            raise ValueError(f"{what}: labels {tuple(labels.shape)} must have the shape of the logits' rows {tuple(lead)}")
        if labels.device != dev:
            raise ValueError(f"{what}: labels are on {labels.device}, the logits on {dev}")
        labels = labels.contiguous()
    x = logits.reshape(-1, V)
    if x.stride(1) != 1 or x.stride(0) < V:
        x = x.contiguous()
    p = _lib.PeLossParams()
    p.rows, p.vocab, p.dtype = x.shape[0], V, _FLOATS[x.dtype]
    p.row_stride, p.grad_row_stride = max(x.stride(0), V), V
    p.shift = lead[-1] if shift else 0
    p.ignore_index = ignore_index
    p.label_bytes = 8 if labels is None else labels.element_size()
    p.reduction = _REDUCTION[reduction]
    p.hard_weight, p.soft_weight, p.temperature, p.grad_factor = 1.0 - soft_weight, soft_weight, 1.0, 1.0
    if teacher_ids is not None:
        tid, tlog = teacher_ids, teacher_logits
        if tid.dtype not in _INTS or tlog.dtype not in _FLOATS:
            raise TypeError(f"{what}: teacher_ids must be int64 / int32 and teacher_logits bf16 / fp16 / fp32, got "
                            f"{tid.dtype} and {tlog.dtype}")
        if tid.dim() != len(lead) + 1 or tid.shape[:-1] != lead or tlog.shape != tid.shape:
            raise ValueError(f"{what}: teacher_ids {tuple(tid.shape)} and teacher_logits {tuple(tlog.shape)} must both be "
                             f"the logits' rows {tuple(lead)} plus a last dim")
        K = tid.shape[-1]
        if not 1 <= K <= _lib.PE_LOSS_MAX_TOP_K:
            raise ValueError(f"{what}: 1 to {_lib.PE_LOSS_MAX_TOP_K} teacher logits a row are supported, got {K}")
        if tid.device != dev or tlog.device != dev:
            raise ValueError(f"{what}: the teacher's tensors must be on {dev}")
        if not 0.0 <= soft_weight <= 1.0:
            raise ValueError(f"{what}: soft_weight must be in [0, 1], got {soft_weight}")
        if not 1e-3 <= temperature <= 1e3:
            raise ValueError(f"{what}: temperature must be in [0.001, 1000], got {temperature}")
        teacher_ids, teacher_logits = tid.reshape(-1, K).contiguous(), tlog.detach().reshape(-1, K).contiguous()
        p.top_k, p.teacher_dtype, p.teacher_id_bytes = K, _FLOATS[tlog.dtype], tid.element_size()
        p.teacher_id_stride = p.teacher_row_stride = K
        p.temperature = temperature
    return p, x, labels, teacher_ids, teacher_logits


def _forward(p, x, labels, tid, tlog, keep):
    """The loss (rows floats, or one) and, with `keep`, the rows' statistics for the backward."""
    L, dev = _lib.lib(), x.device
    whole = p.reduction != _lib.PE_LOSS_NONE
    loss = torch.empty((1,) if whole else (p.rows,), dtype=torch.float32, device=dev)
    ref = ctypes.byref(p)
    # one buffer: the statistics, then the workspace
    n = L.pe_loss_stats_floats(ref) if keep else 0
    nb = L.pe_loss_workspace_bytes(ref)
    buf = torch.empty(n + nb // 4, dtype=torch.float32, device=dev)
    at = buf.data_ptr()
    _call(dev, L.pe_loss_fwd, ref, x.data_ptr(), _ptr(labels), _ptr(tid), _ptr(tlog), loss.data_ptr(),
          at if keep else None, at + 4 * n, nb, _stream(dev))
    return loss, buf


def _expression(logits, labels, teacher_ids, teacher_logits, temperature, soft_weight, ignore_index, reduction, shift):
    """The loss in torch operations, which higher derivatives differentiate."""
    V = logits.shape[-1]
    z = logits.reshape(-1, V).float()
    counts = torch.ones(z.shape[0], dtype=torch.bool, device=z.device)
    if labels is not None:
        y = labels.long()
        if shift:
            y = torch.cat([y[..., 1:], torch.full_like(y[..., :1], ignore_index)], -1)
        y = y.reshape(-1)
        counts = y != ignore_index
    z = torch.where(counts[:, None], z, 0.0)  # rows that do not count: no NaN of theirs in the gradient
    row = torch.zeros(z.shape[0], device=z.device)
    if soft_weight < 1.0:
        known = counts & (y >= 0) & (y < V)
        lq = torch.log_softmax(z, -1).gather(-1, torch.where(known, y, 0)[:, None])[:, 0]
        row = row - (1.0 - soft_weight) * torch.where(known, lq, torch.nan)
    if teacher_ids is not None and soft_weight > 0.0:
        K, T = teacher_ids.shape[-1], temperature
        tid, t = teacher_ids.reshape(-1, K).long(), teacher_logits.detach().reshape(-1, K).float() / T
        have = (tid >= 0) & (tid < V) & (t > -torch.inf)
        some = have.any(-1, keepdim=True)
        lp = torch.log_softmax(torch.where(have, t, torch.where(some, -torch.inf, 0.0)), -1)
        p = torch.where(have, lp.exp(), 0.0)
        lq = torch.log_softmax(z / T, -1).gather(-1, torch.where(have, tid, 0))
        use = p > 0
        row = row + soft_weight * T * T * torch.where(use, p * (torch.where(use, lp, 0.0) - torch.where(use, lq, 0.0)),
                                                      0.0).sum(-1)
    row = torch.where(counts, row, 0.0)
    if reduction == "none":
        return row.reshape(logits.shape[:-1])
    return row.sum() / counts.sum() if reduction == "mean" else row.sum()


class LossFn(torch.autograd.Function):
    """A loss of this module with pe_loss_bwd as its backward; under create_graph and with batched gradients the
    backward differentiates the torch expression (as functional.RMSNormFn)."""

    @staticmethod
    def forward(ctx, logits, labels, teacher_ids, teacher_logits, args, prepared):
        p, x, lab, tid, tlog = prepared
        loss, buf = _forward(p, x, lab, tid, tlog, True)
        ctx.save_for_backward(logits, x, lab, tid, tlog, buf)
        ctx.p, ctx.args, ctx.lead = p, args, logits.shape[:-1]
        return loss.view(logits.shape[:-1] if args[3] == "none" else ())

    @staticmethod
    def backward(ctx, dloss):
        logits, x, lab, tid, tlog, buf = ctx.saved_tensors
        if torch.is_grad_enabled() or not plain_autograd(dloss):
            def rows(t):
                return None if t is None else t.view(*ctx.lead, -1)
            return _expression_grads(lambda: _expression(logits, lab, rows(tid), rows(tlog), *ctx.args), (logits,), ctx,
                                     dloss) + (None,) * 5
        p = ctx.p
        dev = x.device
        dz = torch.empty(logits.shape, dtype=x.dtype, device=dev)
        g = dloss.contiguous()
        _call(dev, _lib.lib().pe_loss_bwd, ctypes.byref(p), x.data_ptr(), _ptr(lab), _ptr(tid), _ptr(tlog),
              buf.data_ptr(), g.data_ptr(), dz.data_ptr(), _stream(dev))
        return (dz,) + (None,) * 5


def _loss(what, logits, labels, teacher_ids, teacher_logits, temperature, soft_weight, ignore_index, reduction, shift):
    args = (float(temperature), float(soft_weight), int(ignore_index), reduction, bool(shift))
    if logits.is_cuda and not plain_autograd(logits):
        return _expression(logits, labels, teacher_ids, teacher_logits, *args)
    prepared = _prepare(what, logits, labels, teacher_ids, teacher_logits, *args)
    if torch.is_grad_enabled() and logits.requires_grad:
        return LossFn.apply(logits, labels, teacher_ids, teacher_logits, args, prepared)
    loss, _ = _forward(*prepared, False)
    return loss.view(logits.shape[:-1] if reduction == "none" else ())


def cross_entropy(logits: torch.Tensor, labels: torch.Tensor, *, ignore_index: int = -100, reduction: str = "mean",
                  shift: bool = False) -> torch.Tensor:
    """-log softmax(logits)[labels] over the last dim: logits (..., V), labels (...), see the module's docstring.
    F.cross_entropy(logits, labels) computed in fp32 whatever the logits' dtype.  Differentiable in the logits."""
    if labels is None:
        raise ValueError("cross_entropy needs labels")
    return _loss("cross_entropy", logits, labels, None, None, 1.0, 0.0, ignore_index, reduction, shift)


def distillation_loss(logits: torch.Tensor, labels: Optional[torch.Tensor], teacher_ids: torch.Tensor,
                      teacher_logits: torch.Tensor, *, temperature: float = 1.0, soft_weight: float = 0.5,
                      ignore_index: int = -100, reduction: str = "mean", shift: bool = False) -> torch.Tensor:
    """(1 - soft_weight) * cross entropy + soft_weight * T^2 * KL(teacher || student at T), see the module's
    docstring.  teacher_ids / teacher_logits (..., K), K <= 1024: the teacher's top logits at the same position as the
    student's logits.  Pairs whose id is outside the vocabulary (-1 to pad short rows) or whose logit is -inf are
    absent; a row without any has no soft part.  labels None (every row counts) needs soft_weight 1.  Differentiable in
    the logits; the teacher gets no gradient."""
    if teacher_ids is None or teacher_logits is None:
        raise ValueError("distillation_loss needs the teacher's ids and logits")
    return _loss("distillation_loss", logits, labels, teacher_ids, teacher_logits, temperature, soft_weight, ignore_index,
                 reduction, shift)


@torch.no_grad()
def loss_and_grad(logits: torch.Tensor, labels: Optional[torch.Tensor], *, teacher_ids: Optional[torch.Tensor] = None,
                  teacher_logits: Optional[torch.Tensor] = None, temperature: float = 1.0, soft_weight: float = 0.5,
                  ignore_index: int = -100, reduction: str = "mean", shift: bool = False,
                  grad_scale: Union[float, torch.Tensor] = 1.0) -> tuple[torch.Tensor, torch.Tensor]:
    """(loss, d(grad_scale * loss) / d logits) of ``cross_entropy``, or with a teacher of ``distillation_loss``, from
    one pass over the logits and outside autograd: ``logits.backward(grad)`` takes it on.  grad_scale, a number or
    a one-element fp32 tensor on the logits' device (a gradient scaler's scale), multiplies the gradient before it is
    rounded to the logits' dtype.  reduction "mean" or "sum"."""
    if (teacher_ids is None) != (teacher_logits is None):
        raise ValueError("loss_and_grad: the teacher needs both ids and logits")
    if reduction == "none":
        raise ValueError("loss_and_grad: reduction must be 'mean' or 'sum'")
    soft = float(soft_weight) if teacher_ids is not None else 0.0
    if labels is None and teacher_ids is None:
        raise ValueError("loss_and_grad needs labels or a teacher")
    p, x, lab, tid, tlog = _prepare("loss_and_grad", logits, labels, teacher_ids, teacher_logits, float(temperature), soft,
                                    int(ignore_index), reduction, bool(shift))
    dev, scale = x.device, None
    if isinstance(grad_scale, torch.Tensor):
        scale = grad_scale.detach()
        if scale.numel() != 1 or scale.dtype != torch.float32 or scale.device != dev:
            raise ValueError(f"loss_and_grad: grad_scale must be a number or one fp32 element on {dev}")
    else:
        p.grad_factor = float(grad_scale)
    L, ref = _lib.lib(), ctypes.byref(p)
    nb = L.pe_loss_workspace_bytes(ref)
    loss = torch.empty((), dtype=torch.float32, device=dev)
    ws = torch.empty(nb, dtype=torch.uint8, device=dev)
    dz = torch.empty(logits.shape, dtype=x.dtype, device=dev)
    _call(dev, L.pe_loss_step, ref, x.data_ptr(), _ptr(lab), _ptr(tid), _ptr(tlog), _ptr(scale), loss.data_ptr(),
          dz.data_ptr(), ws.data_ptr(), nb, _stream(dev))
    return loss, dz
