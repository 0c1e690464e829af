"""The scaled token embedding (pe_embed_fwd) and its gradient (pe_embed_bwd) against the definition in 64 bits.

Forward: one product in fp32, rounded once, so every value is torch's own for (weight.float() * scale).to(dtype),
bit for bit.  Gradient: n terms of one id added in fp32 in any fixed order are at most (n - 1) 2^-24 sum|dy| off,
the scale adds one rounding of 2^-24, and the rounding to the gradient's type half a step (eps / 2 relative, or half
of the smallest subnormal)."""

import math

import pytest
import torch

from pe_ablations_amd.embeddings import TokenEmbedding, embedding, embedding_backward

pytestmark = pytest.mark.gpu

DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
TINY = {"bf16": 2.0 ** -133, "fp16": 2.0 ** -24, "fp32": 2.0 ** -149}


def make(cuda, n, V, H, dtype, seed=0, kind="zipf"):
    g = torch.Generator().manual_seed(seed * 1000 + n + V + H)
    if kind == "zipf":
        ids = (torch.rand(n, generator=g, dtype=torch.float64) * math.log(V + 1)).exp().sub(1).long().clamp(0, V - 1)
    elif kind == "one":
        ids = torch.full((n,), V // 2)
    elif kind == "two":  # long runs beside each other, their ends inside a tile
        ids = torch.where(torch.arange(n) % 3 == 0, 0, V - 1)
    else:
        ids = torch.randint(0, V, (n,), generator=g)
    w = torch.randn(V, H, generator=g).to(DT[dtype])
    dy = torch.randn(n, H, generator=g).to(DT[dtype])
    return ids.to(cuda), w.to(cuda), dy.to(cuda)


def check_grad(dw, ids, dy, V, scale, dtype, pad=None):
    ids, dy = ids.reshape(-1).cpu(), dy.reshape(ids.numel(), -1).cpu().double()
    keep = (ids >= 0) & (ids < V)
    if pad is not None:
        keep &= ids != pad
    k, d = ids[keep].long(), dy[keep]
    want = torch.zeros(V, dy.shape[1], dtype=torch.float64).index_add_(0, k, d) * scale
    mass = torch.zeros(V, dy.shape[1], dtype=torch.float64).index_add_(0, k, d.abs()) * abs(scale)
    n = torch.zeros(V, dtype=torch.float64).index_add_(0, k, torch.ones(len(k), dtype=torch.float64))[:, None]
    tol = (n + 1) * 2.0 ** -24 * mass
    tol = tol + (want.abs() + tol) * (0 if dtype == "fp32" else torch.finfo(DT[dtype]).eps / 2) + TINY[dtype] / 2
    off = (dw.cpu().double() - want).abs()
    assert bool((off <= tol).all()), float((off - tol).max())
    assert bool((dw.cpu()[(n == 0)[:, 0]] == 0).all())


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("n,V,H", [(1, 1, 1), (1, 50257, 512), (3, 7, 5), (16, 1000, 512), (65, 300, 100),
                                   (1000, 10007, 77), (257, 129, 2048), (2, 3, 4099)])
def test_lookup(cuda, n, V, H, dtype):
    ids, w, _ = make(cuda, n, V, H, dtype)
    for scale in (1.0, 22.627417, -0.3):
        out = embedding(ids, w, scale=scale)
        assert out.dtype == w.dtype and torch.equal(out, (w.float()[ids] * scale).to(w.dtype))
    assert torch.equal(embedding(ids.int(), w, scale=2.0), embedding(ids, w, scale=2.0))


def test_lookup_views(cuda):
    g = torch.Generator(device=cuda).manual_seed(3)
    w = torch.randn(50, 72, generator=g, device=cuda)
    ids = torch.randint(0, 50, (6, 8), generator=g, device=cuda)
    for v in (w[:, :64], w[:, 3:40], w[::2], w.t()[:50].t(), w[7:], w.half()[:, 1:60]):
        i = ids % v.shape[0]
        for x in (i, i.t(), i[:, ::3], i[:0], i[2, 5]):
            assert torch.equal(embedding(x, v, scale=0.7), (v.float()[x] * 0.7).to(v.dtype))


def test_lookup_ids_outside(cuda):
    w = torch.ones(5, 33, device=cuda)
    out = embedding(torch.tensor([4, -1, 5, 1 << 40, 0], device=cuda), w)
    assert out.isnan().all(-1).tolist() == [False, True, True, True, False]


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("kind", ["zipf", "one", "two", "uniform"])
@pytest.mark.parametrize("n,V,H", [(1, 1, 1), (1, 5000, 512), (5, 7, 3), (64, 64, 64), (300, 11, 100), (4096, 3000, 64),
                                   (1023, 40000, 8), (2500, 50, 520), (20000, 1500, 40)])
def test_gradient(cuda, n, V, H, kind, dtype):
    ids, w, dy = make(cuda, n, V, H, dtype, kind=kind)
    w.requires_grad_(True)
    out = embedding(ids, w, scale=1.5)
    (dw,) = torch.autograd.grad(out, w, dy)
    assert dw.dtype == w.dtype and dw.shape == w.shape
    check_grad(dw, ids, dy, V, 1.5, dtype)
    assert torch.equal(dw, embedding_backward(ids.int(), dy, V, scale=1.5))  # reproducible, either id type


@pytest.mark.parametrize("n", [70000, 140001])
def test_gradient_many_tokens(cuda, n):
    """Many tokens, and ids above 2^16."""
    ids, _, dy = make(cuda, n, 70001, 16, "fp32", kind="uniform")
    ids[: n // 3] = 69999
    ids[n // 3: n // 2] = 2
    check_grad(embedding_backward(ids, dy, 70001), ids, dy, 70001, 1.0, "fp32")


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("n,V,H,kind", [
    (4096, 16384, 1030, "zipf"), (4096, 16383, 1030, "zipf"),  # where the lanes on a row change, several slices
    (4096, 700, 264, "one"), (4097, 700, 264, "one"),          # one launch and a sort, a long run
    (4096, 64, 8, "two"), (4097, 1, 40, "one"), (5000, 2, 8, "two"),
    (4200, 1 << 20, 4, "uniform"), (4200, (1 << 20) + 3, 2, "uniform"), (700, 3_000_001, 1, "zipf"),  # digits of the sort
    (65536, 900, 16, "zipf"), (65537, 900, 16, "zipf"), (66000, 5, 8, "one"),  # tiles and chunks of the sort
])
def test_gradient_borders(cuda, n, V, H, kind, dtype):
    """Sizes on either side of the kernels' borders."""
    ids, _, dy = make(cuda, n, V, H, dtype, kind=kind)
    if kind == "uniform":
        ids[::7], ids[3] = V - 1, 0
    check_grad(embedding_backward(ids, dy, V, scale=-0.5), ids, dy, V, -0.5, dtype)


def test_gradient_padding_and_outside(cuda):
    ids, _, dy = make(cuda, 3000, 100, 24, "fp32")
    ids[::2] = 7
    ids[5] = -3
    ids[6] = 100
    ids[9] = 1 << 33
    check_grad(embedding_backward(ids, dy, 100, padding_idx=7), ids, dy, 100, 1.0, "fp32", pad=7)
    check_grad(embedding_backward(ids, dy, 100), ids, dy, 100, 1.0, "fp32")
    assert torch.equal(embedding_backward(ids, dy, 100, padding_idx=-93), embedding_backward(ids, dy, 100, padding_idx=7))
    w = torch.randn(100, 24, device=cuda, requires_grad=True)
    ok = ids.clamp(0, 99)
    out = embedding(ok, w, padding_idx=7)
    assert torch.equal(out, w.detach()[ok])
    (dw,) = torch.autograd.grad(out, w, dy)
    check_grad(dw, ok, dy, 100, 1.0, "fp32", pad=7)
    all_pad = torch.full((9,), 7, device=cuda)
    assert bool((embedding_backward(all_pad, dy[:9], 100, padding_idx=7) == 0).all())


def test_gradient_strides_and_empty(cuda):
    ids = torch.randint(0, 20, (6, 10), device=cuda)
    base = torch.randn(6, 10, 80, device=cuda)
    for dy in (base[..., :64], base[..., 5:70], base.transpose(0, 1).contiguous().transpose(0, 1),
               base[..., :1].expand(6, 10, 33)):
        check_grad(embedding_backward(ids, dy, 20, scale=0.5), ids, dy, 20, 0.5, "fp32")
    assert bool((embedding_backward(ids[:0], base[:0], 20) == 0).all())
    w = torch.randn(20, 8, device=cuda, requires_grad=True)
    embedding(ids[:0], w).sum().backward()
    assert bool((w.grad == 0).all())


def test_gradient_of_infinities(cuda):
    """An infinity or NaN stays in its own id's column."""
    ids = torch.tensor([3, 1, 3, 0, 1], device=cuda)
    dy = torch.ones(5, 16, device=cuda)
    dy[0, 2], dy[1, 5], dy[2, 2] = math.inf, math.nan, -math.inf
    dw = embedding_backward(ids, dy, 6)
    bad = ~torch.isfinite(dw)
    assert bad.nonzero().tolist() == [[1, 5], [3, 2]] and dw[1, 5].isnan() and dw[3, 2].isnan()


def test_gradient_by_differences(cuda):
    """The loss is linear in the weight: a difference of losses is the gradient, to the rounding of the sums."""
    g = torch.Generator(device=cuda).manual_seed(0)
    w = torch.randn(9, 8, generator=g, device=cuda, requires_grad=True)
    ids = torch.randint(0, 9, (40,), generator=g, device=cuda)
    dy = torch.randn(40, 8, generator=g, device=cuda)
    (dw,) = torch.autograd.grad((embedding(ids, w, scale=1.25) * dy).sum(), w)
    for v, j in ((0, 0), (4, 3), (8, 7)):
        e = torch.zeros_like(w)
        e[v, j] = 1.0
        up, down = (float((embedding(ids, w.detach() + s * e, scale=1.25).double() * dy.double()).sum()) for s in (1, -1))
        assert abs((up - down) / 2 - float(dw[v, j])) < 1e-4  # 40 products, each off by 2^-24 of values below 8


def test_higher_derivatives_and_batched_gradients(cuda):
    w = torch.randn(6, 8, device=cuda, requires_grad=True)
    ids = torch.tensor([1, 1, 5], device=cuda)
    out = embedding(ids, w, scale=2.0)
    (g1,) = torch.autograd.grad(out.pow(3).sum(), w, create_graph=True)
    (g2,) = torch.autograd.grad(g1.sum(), w)
    want = torch.zeros_like(g2).index_add_(0, ids, 2 * 2 * 6 * (2 * w.detach()[ids]))
    assert torch.allclose(g2, want, rtol=1e-5, atol=1e-5)
    out = embedding(ids, w, scale=2.0)
    (gb,) = torch.autograd.grad(out, w, torch.eye(24, device=cuda).view(24, 3, 8), is_grads_batched=True)
    assert gb.shape == (24, 6, 8) and float(gb.sum()) == 48.0


def test_transforms_of_torch(cuda):
    """functorch and forward mode see F.embedding's expression."""
    w = torch.randn(9, 8, device=cuda)
    ids = torch.tensor([1, 8, 1], device=cuda)
    f = lambda x: (embedding(ids, x, scale=2.0, padding_idx=8) ** 2).sum()  # noqa: E731
    want = torch.zeros_like(w)
    want[1] = 2 * 8 * w[1]
    assert torch.allclose(torch.func.grad(f)(w), want, rtol=1e-5, atol=1e-5)
    ws = torch.stack([w, w * 2])
    assert torch.allclose(torch.func.vmap(lambda x: embedding(ids, x, scale=2.0))(ws), 2.0 * ws[:, ids])
    out, tangent = torch.func.jvp(lambda x: embedding(ids, x, scale=2.0), (w,), (torch.ones_like(w),))
    assert torch.equal(out, 2 * w[ids]) and bool((tangent == 2).all())


def test_weight_changed_before_the_backward(cuda):
    """As with F.embedding, whose backward needs the ids alone."""
    w = torch.randn(9, 8, device=cuda, requires_grad=True)
    ids = torch.tensor([1, 8, 1], device=cuda)
    out = embedding(ids, w)
    with torch.no_grad():
        w.mul_(2)
    out.sum().backward()
    assert w.grad[1, 0] == 2 and w.grad[8, 3] == 1 and w.grad[0, 0] == 0


def test_past_32_bit_offsets(cuda):
    """A table and gradients of over 2^32 bytes and 2^31 elements."""
    V, H, n = 70001, 32768, 66000
    w = torch.zeros(V, H, dtype=torch.bfloat16, device=cuda)
    w[V - 1], w[V - 2], w[3] = 3.0, 2.0, 1.0
    out = embedding(torch.tensor([V - 1, 3, V - 2, 0], device=cuda), w, scale=2.0)
    assert out.float().mean(-1).tolist() == [6.0, 2.0, 4.0, 0.0]
    ids = torch.arange(n, device=cuda) % 5000 + (V - 5000)
    dy = w[:n]
    dy[n - 1] = 1.0
    dw = embedding_backward(ids, dy, V)
    rows = dw.float().sum(-1)
    want = torch.zeros(V, device=cuda).index_add_(0, ids, dy.float().mean(-1) * H)
    assert torch.equal(rows, want) and int((rows != 0).sum()) == 2


def test_module(cuda):
    m = TokenEmbedding(64, 32, scale=4.0).to(cuda)
    ids = torch.randint(0, 64, (2, 9), device=cuda)
    m(ids).sum().backward()
    want = torch.zeros(64, 32, device=cuda).index_add_(0, ids.reshape(-1), torch.full((18, 32), 4.0, device=cuda))
    assert torch.equal(m.weight.grad, want)
    assert torch.equal(m(ids), m.weight.detach()[ids] * 4.0)


def test_another_stream(cuda):
    ids, w, dy = make(cuda, 2000, 500, 64, "fp32")
    want, dwant = embedding(ids, w, scale=3.0), embedding_backward(ids, dy, 500)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        got, dgot = embedding(ids, w, scale=3.0), embedding_backward(ids, dy, 500)
    side.synchronize()
    assert torch.equal(got, want) and torch.equal(dgot, dwant)


def test_refusals(cuda):
    w, ids = torch.zeros(7, 8, device=cuda), torch.zeros(3, dtype=torch.long, device=cuda)
    for call, err in ((lambda: embedding(ids.cpu(), w), ValueError), (lambda: embedding(ids.float(), w), TypeError),
                      (lambda: embedding(ids, w.double()), TypeError), (lambda: embedding(ids, w[0]), ValueError),
                      (lambda: embedding(ids, w[:0]), ValueError), (lambda: embedding(ids, w, padding_idx=7), ValueError),
                      (lambda: embedding(ids, w, padding_idx=-8), ValueError),
                      (lambda: embedding_backward(ids, torch.zeros(4, 8, device=cuda), 7), ValueError),
                      (lambda: embedding_backward(ids, torch.zeros(3, 8, device=cuda), 0), ValueError),
                      (lambda: embedding_backward(ids.short(), torch.zeros(3, 8, device=cuda), 7), TypeError)):
        with pytest.raises(err):
            call()
