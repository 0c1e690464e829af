"""The operators over the vocabulary without a GPU: the C ABI's symbols, its parameter block and its host-side
refusals, the Python layer's refusals that need no launch, the torch expressions behind higher derivatives
against 64-bit loops, and the configuration fields."""

import ctypes
import math
import os
import re

import pytest
import torch

from pe_ablations_amd import _lib, losses
from pe_ablations_amd.embeddings import TokenEmbedding, embedding, embedding_backward
from pe_ablations_amd.evaluation import config_from_checkpoint
from pe_ablations_amd.losses import cross_entropy, distillation_loss, loss_and_grad
from pe_ablations_amd.transformer import Transformer, TransformerConfig

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
E = _lib.ERRORS


@pytest.fixture(scope="module")
def lib():
    if not _lib.available():
        pytest.fail("libpe_attn.so is not built (python -m pe_ablations_amd.build)")
    return _lib.lib()


def test_every_declared_symbol_is_exported(lib):
    text = re.sub(r"/\*.*?\*/", "", open(os.path.join(ROOT, "include", "pe_vocab.h")).read(), flags=re.S)
    names = sorted(set(re.findall(r"\b(pe_(?:embed|loss)_\w+)\s*\(", text)))
    assert names == sorted(_lib.EXPORTED_VOCAB)
    for n in names:
        assert hasattr(lib, n), n
    for name in ("PE_LOSS_NONE", "PE_LOSS_SUM", "PE_LOSS_MEAN"):
        assert int(re.search(rf"\b{name}\s*=\s*(\d+)", text).group(1)) == getattr(_lib, name)
    assert int(re.search(r"PE_LOSS_MAX_TOP_K\s+(\d+)", text).group(1)) == _lib.PE_LOSS_MAX_TOP_K


def test_loss_params_layout():
    # int64 x 7, int32 x 7, float x 4, int32
    assert ctypes.sizeof(_lib.PeLossParams) == 104
    assert _lib.PeLossParams.vocab.offset == 56 and _lib.PeLossParams.hard_weight.offset == 84


def params(**kw):
    p = _lib.PeLossParams()
    base = dict(rows=6, row_stride=11, grad_row_stride=11, shift=0, ignore_index=-100, teacher_id_stride=4,
                teacher_row_stride=4, vocab=11, dtype=_lib.PE_DTYPE_BF16, label_bytes=8, reduction=_lib.PE_LOSS_MEAN,
                top_k=4, teacher_dtype=_lib.PE_DTYPE_BF16, teacher_id_bytes=4, hard_weight=0.5, soft_weight=0.5,
                temperature=2.0, grad_factor=1.0)
    base.update(kw)
    for k, v in base.items():
        setattr(p, k, v)
    return p


@pytest.mark.parametrize("over,code", [
    ({}, "PE_OK"), (dict(rows=0), "PE_OK"), (dict(shift=3), "PE_OK"), (dict(top_k=0, soft_weight=0.0), "PE_OK"),
    (dict(rows=-1), "PE_ERR_SHAPE"), (dict(rows=1 << 31), "PE_ERR_SHAPE"), (dict(vocab=0), "PE_ERR_SHAPE"),
    (dict(shift=4), "PE_ERR_SHAPE"), (dict(shift=-1), "PE_ERR_SHAPE"), (dict(top_k=1025), "PE_ERR_SHAPE"),
    (dict(dtype=3), "PE_ERR_MODE"), (dict(label_bytes=2), "PE_ERR_MODE"), (dict(reduction=3), "PE_ERR_MODE"),
    (dict(teacher_dtype=7), "PE_ERR_MODE"), (dict(teacher_id_bytes=1), "PE_ERR_MODE"),
    (dict(temperature=0.0), "PE_ERR_MODE"), (dict(temperature=math.nan), "PE_ERR_MODE"),
    (dict(hard_weight=-0.1), "PE_ERR_MODE"), (dict(hard_weight=0.0, soft_weight=0.0), "PE_ERR_MODE"),
    (dict(soft_weight=math.nan), "PE_ERR_MODE"), (dict(top_k=0), "PE_ERR_MODE"),
    (dict(row_stride=10), "PE_ERR_STRIDE"), (dict(grad_row_stride=0), "PE_ERR_STRIDE"),
    (dict(teacher_row_stride=3), "PE_ERR_STRIDE"),
])
def test_loss_check(lib, over, code):
    p = params(**over)
    assert lib.pe_loss_check(ctypes.byref(p)) == E[code]
    good = code == "PE_OK"
    teacher = p.rows * (2 * p.top_k + 4) if p.soft_weight > 0 else 0
    assert lib.pe_loss_stats_floats(ctypes.byref(p)) == (3 * p.rows + 1 + teacher if good else 0)
    nb = lib.pe_loss_workspace_bytes(ctypes.byref(p))
    assert nb >= 4 * (p.rows + 1) if good else nb == 0


def test_loss_entry_points_refuse(lib):
    assert lib.pe_loss_check(None) == E["PE_ERR_NULL"]
    p, big = params(), 1 << 20
    ref = ctypes.byref(p)
    # fake, never dereferenced addresses: every case ends before a launch
    z, y, i, t, out, ws = 64, 128, 256, 512, 1024, 2048
    assert lib.pe_loss_fwd(ref, None, y, i, t, out, None, ws, big, None) == E["PE_ERR_NULL"]
    assert lib.pe_loss_fwd(ref, z, None, i, t, out, None, ws, big, None) == E["PE_ERR_NULL"]
    assert lib.pe_loss_fwd(ref, z, y, None, t, out, None, ws, big, None) == E["PE_ERR_NULL"]
    assert lib.pe_loss_fwd(ref, z, y, i, t, None, None, ws, big, None) == E["PE_ERR_NULL"]
    assert lib.pe_loss_fwd(ref, z + 1, y, i, t, out, None, ws, big, None) == E["PE_ERR_STRIDE"]
    assert lib.pe_loss_fwd(ref, z, y + 4, i, t, out, None, ws, big, None) == E["PE_ERR_STRIDE"]
    assert lib.pe_loss_fwd(ref, z, y, i, t, out, None, ws, 4, None) == E["PE_ERR_WORKSPACE"]
    assert lib.pe_loss_fwd(ref, z, y, i, t, out, None, None, big, None) == E["PE_ERR_WORKSPACE"]
    assert lib.pe_loss_bwd(ref, z, y, i, t, None, out, out, None) == E["PE_ERR_NULL"]
    assert lib.pe_loss_bwd(ref, z, y, i, t, ws, None, out, None) == E["PE_ERR_NULL"]
    assert lib.pe_loss_bwd(ref, z, y, i, t, ws, out, out + 1, None) == E["PE_ERR_STRIDE"]
    assert lib.pe_loss_step(ref, z, y, i, t, None, out, None, ws, big, None) == E["PE_ERR_NULL"]
    none = params(reduction=_lib.PE_LOSS_NONE)
    assert lib.pe_loss_step(ctypes.byref(none), z, y, i, t, None, out, out, ws, big, None) == E["PE_ERR_MODE"]


def test_embed_entry_points_refuse(lib):
    def fwd(ids=64, ib=8, n=5, w=128, dt=0, V=7, H=8, ws=8, out=256, os_=8):
        return lib.pe_embed_fwd(ids, ib, n, w, dt, V, H, ws, 1.0, out, os_, None)
    assert fwd(ids=None) == fwd(w=None) == fwd(out=None) == E["PE_ERR_NULL"]
    assert fwd(n=-1) == fwd(V=0) == fwd(H=0) == fwd(n=1 << 31) == E["PE_ERR_SHAPE"]
    assert fwd(dt=3) == fwd(ib=2) == E["PE_ERR_MODE"]
    assert fwd(ws=7) == fwd(os_=7) == fwd(ids=60) == fwd(w=129) == E["PE_ERR_STRIDE"]
    assert fwd(n=0) == E["PE_OK"]

    nb = lib.pe_embed_bwd_workspace_bytes(5000, 7, 8)
    assert nb > 0 and lib.pe_embed_bwd_workspace_bytes((1 << 24) + 1, 7, 8) == 0
    assert lib.pe_embed_bwd_workspace_bytes(4096, 7, 8) == 0  # a few tokens need none

    def bwd(ids=64, n=5000, dy=128, V=7, pad=-1, dw=256, ws=512, wb=nb, stride=8):
        return lib.pe_embed_bwd(ids, 8, n, dy, 0, stride, V, 8, 1.0, pad, dw, 8, ws, wb, None)
    assert bwd(ids=None) == bwd(dy=None) == bwd(dw=None) == E["PE_ERR_NULL"]
    assert bwd(pad=7) == bwd(pad=-2) == bwd(n=(1 << 24) + 1) == E["PE_ERR_SHAPE"]
    assert bwd(ws=None) == bwd(wb=nb - 1) == bwd(ws=520) == E["PE_ERR_WORKSPACE"]
    assert bwd(stride=0) == E["PE_ERR_STRIDE"]


def test_cpu_tensors_are_refused():
    w, ids = torch.zeros(7, 8), torch.zeros(3, dtype=torch.long)
    with pytest.raises(RuntimeError, match="GPU"):
        embedding(ids, w)
    with pytest.raises(RuntimeError, match="GPU"):
        embedding_backward(ids, torch.zeros(3, 8), 7)
    z, y = torch.zeros(3, 7), torch.zeros(3, dtype=torch.long)
    k, t = torch.zeros(3, 2, dtype=torch.long), torch.zeros(3, 2)
    for call in (lambda: cross_entropy(z, y), lambda: distillation_loss(z, y, k, t), lambda: loss_and_grad(z, y)):
        with pytest.raises(RuntimeError, match="GPU"):
            call()
    with pytest.raises(ValueError):
        cross_entropy(z, None)
    with pytest.raises(ValueError):
        distillation_loss(z, y, None, None)
    with pytest.raises(ValueError):
        loss_and_grad(z, y, teacher_ids=k)
    with pytest.raises(ValueError):
        loss_and_grad(z, y, reduction="none")
    with pytest.raises(ValueError):
        loss_and_grad(z, None)


def loop_loss(z, y, tid, tlog, T, soft, ignore, shift):
    """The definition, a row and a pair at a time."""
    rows = []
    B, S, V = z.shape
    for b in range(B):
        for s in range(S):
            lab = (y[b, s + 1] if s + 1 < S else ignore) if shift else y[b, s]
            if int(lab) == ignore:
                rows.append(z.new_zeros(()))
                continue
            row = -(1 - soft) * torch.log_softmax(z[b, s], -1)[int(lab)]
            if tid is not None:
                have = [k for k in range(tid.shape[-1]) if 0 <= int(tid[b, s, k]) < V and tlog[b, s, k] > -math.inf]
                if have:
                    p = torch.softmax(tlog[b, s, have] / T, -1)
                    lq = torch.log_softmax(z[b, s] / T, -1)
                    row = row + soft * T * T * sum(p[i] * (p[i].log() - lq[int(tid[b, s, k])]) for i, k in enumerate(have))
            rows.append(row)
    return torch.stack(rows).view(B, S)


@pytest.mark.parametrize("teacher", [False, True])
@pytest.mark.parametrize("shift", [False, True])
def test_expression_is_the_definition(teacher, shift):
    g = torch.Generator().manual_seed(1)
    z = torch.randn(2, 4, 9, generator=g) * 3
    y = torch.randint(0, 9, (2, 4), generator=g)
    y[0, 2] = -100
    tid = torch.randint(-1, 10, (2, 4, 5), generator=g) if teacher else None  # ids out of range, some twice
    tlog = torch.randn(2, 4, 5, generator=g) if teacher else None
    if teacher:
        tid[1, 0] = -1
        tlog[1, 1, 2] = -math.inf
    soft = 0.3 if teacher else 0.0
    a = z.clone().requires_grad_(True)
    rows = losses._expression(a, y, tid, tlog, 1.7, soft, -100, "none", shift)
    b = z.double().requires_grad_(True)
    want = loop_loss(b, y, tid, None if tlog is None else tlog.double(), 1.7, soft, -100, shift)
    assert (rows - want).abs().max() < 2e-6  # about 20 roundings of values below 16
    w = torch.rand(2, 4, generator=g)
    (ga,) = torch.autograd.grad((rows * w).sum(), a)
    (gb,) = torch.autograd.grad((want * w.double()).sum(), b)
    assert (ga - gb).abs().max() < 2e-6
    n = (want != 0).sum()
    assert abs(losses._expression(z, y, tid, tlog, 1.7, soft, -100, "mean", shift) - want.sum() / n) < 2e-6


def test_expression_marks_labels_outside_the_vocabulary():
    z, y = torch.zeros(3, 4), torch.tensor([1, 4, -100])
    rows = losses._expression(z, y, None, None, 1.0, 0.0, -100, "none", False)
    assert abs(rows[0] - math.log(4)) < 1e-6 and rows[1].isnan() and rows[2] == 0


def test_configuration_fields():
    c = TransformerConfig(vocab_size=32, hidden_dim=16, num_layers=1, num_heads=2, num_kv_heads=1, head_dim=8, ffn_dim=32)
    assert c.embedding_scale is None and c.fused_loss is False
    m = Transformer(c)
    ids = torch.tensor([[3, 1]])
    assert m.token_embedding.scale is None
    assert torch.equal(m.token_embedding(ids), m.token_embedding.weight[ids])  # the plain lookup, on any device
    with pytest.raises(ValueError, match="labels"):
        m(ids, teacher=(ids[..., None], torch.zeros(1, 2, 1)))
    assert TokenEmbedding(8, 4).scale is None and TokenEmbedding(8, 4, scale=2.0).scale == 2.0
    assert list(TokenEmbedding(8, 4, scale=2.0).state_dict()) == ["embedding.weight"]
    # a checkpoint keeps them
    got = config_from_checkpoint({"model_config": dict(c.__dict__, embedding_scale=4.0, fused_loss=True)})
    assert got.embedding_scale == 4.0 and got.fused_loss is True
    old = {k: v for k, v in c.__dict__.items() if k not in ("embedding_scale", "fused_loss")}
    got = config_from_checkpoint({"model_config": old})
    assert got.embedding_scale is None and got.fused_loss is False
