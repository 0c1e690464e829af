"""The embedding and the losses together, as a model uses them: Transformer with embedding_scale, fused_loss and a
teacher, its training step captured in a HIP graph, and the unchanged default path."""

import pytest
import torch
import torch.nn.functional as F

from pe_ablations_amd.losses import cross_entropy, distillation_loss, loss_and_grad
from pe_ablations_amd.embeddings import embedding
from pe_ablations_amd.transformer import Transformer, TransformerConfig

pytestmark = pytest.mark.gpu


def model(cuda, **kw):
    torch.manual_seed(0)
    c = TransformerConfig(vocab_size=301, hidden_dim=64, num_layers=2, num_heads=4, num_kv_heads=2, head_dim=64,
                          ffn_dim=128, pe_mode="pope", max_seq_len=64, **kw)
    return Transformer(c).to(cuda)


def batch(cuda, B=3, S=33):
    g = torch.Generator(device=cuda).manual_seed(5)
    ids = torch.randint(0, 301, (B, S), generator=g, device=cuda)
    labels = ids.clone()
    labels[0, :10] = -100
    return ids, labels


def plain_loss(logits, labels):
    return F.cross_entropy(logits[:, :-1].reshape(-1, logits.shape[-1]).float(), labels[:, 1:].reshape(-1),
                           ignore_index=-100)


@pytest.mark.parametrize("tie", [True, False])
def test_training_step(cuda, tie):
    """Scaled embedding and fused loss against the same model in torch operations: the embedding's weight gets the
    gradients of both ends when it is tied."""
    ids, labels = batch(cuda)
    m = model(cuda, embedding_scale=8.0, fused_loss=True, tie_embeddings=tie)
    out = m(ids, labels=labels)
    out["loss"].backward()
    got = {n: p.grad.clone() for n, p in m.named_parameters()}
    m.zero_grad()
    # the same graph with the plain lookup: a hook-free replacement of the module's call
    m.token_embedding.forward = lambda x: F.embedding(x, m.token_embedding.weight) * 8.0
    ref = m(ids)["logits"]
    assert torch.equal(ref, out["logits"])
    loss = plain_loss(ref, labels)
    loss.backward()
    assert abs(float(loss.detach()) - float(out["loss"].detach())) < 1e-5
    for n, p in m.named_parameters():
        # fp32 gradients through the same kernels: the two paths differ by roundings of their sums
        assert (p.grad - got[n]).norm() <= 1e-4 * p.grad.norm() + 1e-9, n


def test_default_path_is_unchanged(cuda):
    ids, labels = batch(cuda)
    m = model(cuda)
    out = m(ids, labels=labels)
    shift = out["logits"][..., :-1, :].contiguous().view(-1, 301)
    assert torch.equal(out["loss"], F.cross_entropy(shift, labels[..., 1:].contiguous().view(-1), ignore_index=-100))


def test_distillation_of_a_rope_teacher(cuda):
    ids, labels = batch(cuda)
    torch.manual_seed(1)
    teacher = Transformer(TransformerConfig(vocab_size=301, hidden_dim=64, num_layers=1, num_heads=4, num_kv_heads=2,
                                            head_dim=64, ffn_dim=128, pe_mode="rope", max_seq_len=64)).to(cuda).eval()
    with torch.no_grad():
        top = torch.topk(teacher(ids)["logits"] * 20, 16, dim=-1)
    m = model(cuda, embedding_scale=8.0)
    out = m(ids, labels=labels, teacher=(top.indices, top.values), temperature=2.0, soft_weight=0.7)
    out["loss"].backward()
    grads = [p.grad for p in m.parameters()]
    assert all(g is not None and bool(torch.isfinite(g).all()) for g in grads) and torch.isfinite(out["loss"])
    z = out["logits"].detach()
    assert torch.equal(out["loss"].detach(), distillation_loss(z, labels, top.indices, top.values, temperature=2.0,
                                                               soft_weight=0.7, shift=True))
    # the definition on the shifted rows
    zz, y = z[:, :-1].reshape(-1, 301).double(), labels[:, 1:].reshape(-1)
    tid, t = (x[:, :-1].reshape(-1, 16) for x in (top.indices, top.values))
    p = torch.softmax(t.double() / 2, -1)
    soft = 4 * (p * (p.log() - torch.log_softmax(zz / 2, -1).gather(-1, tid))).sum(-1)
    hard = F.cross_entropy(zz, y, ignore_index=-100, reduction="none")
    keep = y != -100
    want = ((0.3 * hard + 0.7 * soft)[keep]).mean()
    assert abs(float(want) - float(out["loss"].detach())) < 1e-4 * float(want)


def test_autocast_training_step(cuda):
    ids, labels = batch(cuda)
    m = model(cuda, embedding_scale=8.0, fused_loss=True)
    with torch.autocast("cuda", dtype=torch.bfloat16):
        out = m(ids, labels=labels)
    assert out["logits"].dtype == torch.bfloat16 and out["loss"].dtype == torch.float32
    assert abs(float(out["loss"].detach()) - float(plain_loss(out["logits"], labels).detach())) < 1e-5
    out["loss"].backward()
    assert bool(torch.isfinite(m.token_embedding.weight.grad).all())


def test_step_through_loss_and_grad(cuda):
    """The one-call form hands autograd the same gradients."""
    ids, labels = batch(cuda)
    m = model(cuda, embedding_scale=8.0, fused_loss=True)
    m(ids, labels=labels)["loss"].backward()
    want = {n: p.grad.clone() for n, p in m.named_parameters()}
    m.zero_grad()
    logits = m(ids)["logits"]
    loss, grad = loss_and_grad(logits.detach(), labels, shift=True)
    logits.backward(grad)
    for n, p in m.named_parameters():
        assert (p.grad - want[n]).norm() <= 1e-5 * want[n].norm() + 1e-9, n


def test_graph_replay(cuda):
    """Embedding, both loss forms and their gradients in one captured graph, replayed with new contents."""
    g = torch.Generator(device=cuda).manual_seed(9)
    V, H, N, K = 3001, 64, 96, 8
    w = torch.randn(V, H, generator=g, device=cuda).requires_grad_(True)
    head = torch.randn(V, H, generator=g, device=cuda).bfloat16() * 0.1
    ids = torch.randint(0, V, (2, N // 2), generator=g, device=cuda)
    tid = torch.randint(0, V, (2, N // 2, K), generator=g, device=cuda)
    tlog = torch.randn(2, N // 2, K, generator=g, device=cuda)

    def step():
        x = embedding(ids, w, scale=2.0)
        logits = F.linear(x.bfloat16(), head)
        loss = distillation_loss(logits, ids, tid, tlog, temperature=2.0, shift=True) + cross_entropy(logits, ids, shift=True)
        (dw,) = torch.autograd.grad(loss, w)
        one, dz = loss_and_grad(logits.detach(), ids, shift=True)
        return loss.detach(), dw, one, dz

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step()
    for rep in range(5):
        if rep >= 2:
            with torch.no_grad():
                ids.copy_(torch.randint(0, V if rep % 2 else 3, ids.shape, generator=g, device=cuda))
                tlog.copy_(torch.randn(tlog.shape, generator=g, device=cuda))
                if rep == 4:
                    ids[0, 5:] = 7
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in outs]
        want = step()
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert torch.equal(a, b), rep


@pytest.mark.parametrize("n", [700, 5000])
def test_two_graphs(cuda, n):
    """Two captured graphs, replayed in turn with eager work between them: neither touches the other's workspace; both
    forms of the embedding's gradient."""
    g = torch.Generator(device=cuda).manual_seed(n)

    def make(V, H, dtype):
        w = torch.randn(V, H, generator=g, device=cuda).to(dtype).requires_grad_(True)
        ids = torch.randint(0, V, (n,), generator=g, device=cuda)
        dy = torch.randn(n, H, generator=g, device=cuda).to(dtype)
        z = torch.randn(60, V, generator=g, device=cuda).to(dtype)
        y = torch.randint(0, V, (60,), generator=g, device=cuda)
        tid, tlog = torch.randint(0, V, (60, 6), generator=g, device=cuda), torch.randn(60, 6, generator=g, device=cuda)

        def step():
            (dw,) = torch.autograd.grad(embedding(ids, w, scale=2.0), w, dy)
            loss, dz = loss_and_grad(z, y, teacher_ids=tid, teacher_logits=tlog, temperature=2.0)
            return dw, loss, dz, cross_entropy(z, y, reduction="none")

        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            for _ in range(2):
                step()
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs = step()
        return step, graph, outs

    both = [make(2000, 40, torch.float32), make(901, 72, torch.bfloat16)]
    want = [[t.clone() for t in step()] for step, _, _ in both]
    for rep in range(4):
        for step, graph, outs in both[::-1] if rep % 2 else both:
            for t in outs:
                t.fill_(float("nan"))
            graph.replay()
            step()
        torch.cuda.synchronize()
        for (_, _, outs), w in zip(both, want):
            for a, b in zip(outs, w):
                assert torch.equal(a, b), rep
