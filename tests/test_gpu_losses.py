"""Cross entropy and distillation (pe_loss_fwd / _bwd / _step) against the definition in 64 bits.

Tolerances, in units of u = 2^-24.  An exponential of (z - m) is off by the rounding of the difference and of its
product with log2 e, 2 |z - m| u, and by exp2 itself, 4 u; a thread adds at most V / 64 of them and the threads'
sums are joined in at most 32 steps, so a sum s is off by E = (V / 64 + 40 + 3 D) u relative, D the row's range (over T
for the sum at the temperature), taking terms beyond exp(-20) of the maximum as 0.  ln s then is off by E plus a
rounding of its own; the row's loss by that and a few roundings of its terms.  The gradient's q = e / s is off by twice
E relative, the difference with the named entry by a rounding, and the store by half a step of the type.  The GPU's
exp2 instruction gives 0 for results below 2^-126, so a q below it may be 0."""

import math

import pytest
import torch

from pe_ablations_amd.losses import cross_entropy, distillation_loss, loss_and_grad

pytestmark = pytest.mark.gpu

DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
TINY = {torch.bfloat16: 2.0 ** -126, torch.float16: 2.0 ** -24, torch.float32: 2.0 ** -126}
U = 2.0 ** -24


def definition(z, y, tid, tlog, T, soft, ignore=-100):
    """(row losses, d row / dz, which rows count, error of the losses, error of the gradient) in 64 bits; rows
    (N, V), labels (N,) or None.  The errors are the fp32 ones above."""
    z = z.double()
    N, V = z.shape
    dev = z.device
    counts = torch.ones(N, dtype=torch.bool, device=dev) if y is None else y != ignore
    z = torch.where(counts[:, None], z, 0.0)
    D = torch.where(z == -math.inf, 0.0, z.amax(-1, keepdim=True) - z).amax(-1).clamp(max=20.0)
    E = (V / 64 + 40 + 3 * D) * U
    rows, grad = torch.zeros(N, dtype=torch.float64, device=dev), torch.zeros_like(z)
    el, eg = torch.zeros_like(rows), torch.zeros_like(z)
    ar = torch.arange(N, device=dev)
    if soft < 1:
        lq = torch.log_softmax(z, -1)
        yc = torch.where(counts, y.long(), 0)
        rows -= (1 - soft) * lq[ar, yc]
        q = lq.exp()
        hot = torch.zeros_like(z)
        hot[ar, yc] = 1
        grad += (1 - soft) * (q - hot)
        el += (1 - soft) * (E + 8 * U * (z.abs().amax(-1).clamp(max=1e30) + 16))
        eg += (1 - soft) * (2 * E[:, None] * q + 4 * U * hot)
    if tid is not None and soft > 0:
        have = (tid >= 0) & (tid < V) & (tlog > -math.inf)
        some = have.any(-1, keepdim=True)
        t = tlog.double() / T
        lp = torch.log_softmax(torch.where(have, t, torch.where(some, -math.inf, 0.0)), -1)
        p = torch.where(have, lp.exp(), 0.0)
        lt = torch.log_softmax(z / T, -1)
        use = p > 0
        at = torch.where(have, tid.long(), 0)
        rows += soft * T * T * torch.where(use, p * (torch.where(use, lp, 0.0) - torch.where(use, lt.gather(-1, at), 0.0)),
                                           0.0).sum(-1)
        full = torch.zeros_like(z).scatter_add_(-1, at, p)
        qt = lt.exp() * some
        grad += soft * T * (qt - full)
        K = tid.shape[-1]
        ET = E * max(1.0, 1 / T)
        tr = torch.where(have, t, 0.0)
        EP = (K + 40 + 3 * (tr.amax(-1) - tr.amin(-1)).clamp(max=20)) * U
        big = (z.abs().amax(-1).clamp(max=1e30) + torch.where(have, tlog.double(), 0.0).abs().amax(-1)) / T + 16
        el += soft * T * T * (ET + 2 * EP * big + 16 * U * big)
        eg += soft * T * (2 * ET[:, None] * qt + (2 * EP[:, None] + 8 * U) * full)
    return torch.where(counts, rows, 0.0), grad * counts[:, None], counts, el, eg * counts[:, None]


def off_by(got, want, tol):
    got, want = got.double(), want.double()
    same = (got == want) | (got.isnan() & want.isnan())
    d = torch.where(same, 0.0, (got - want).abs())
    return float((d - tol).nan_to_num(nan=math.inf).max()) if d.numel() else 0.0


def check_all(z, y, tid=None, tlog=None, T=1.0, soft=0.0, ignore=-100, upstream=1.0):
    """Every path over rows (N, V) against the definition."""
    rows, grad, counts, el, eg = definition(z, y, tid, tlog, T, soft, ignore)
    n = int(counts.sum())
    kw = dict(ignore_index=ignore)
    if tid is not None:
        kw.update(temperature=T, soft_weight=soft)
        call = lambda x, **k: distillation_loss(x, y, tid, tlog, **kw, **k)  # noqa: E731
        step = lambda x, **k: loss_and_grad(x, y, teacher_ids=tid, teacher_logits=tlog, **kw, **k)  # noqa: E731
    else:
        call = lambda x, **k: cross_entropy(x, y, **kw, **k)  # noqa: E731
        step = lambda x, **k: loss_and_grad(x, y, **kw, **k)  # noqa: E731
    got = call(z, reduction="none")
    assert got.dtype == torch.float32 and got.shape == z.shape[:-1]
    assert off_by(got, rows, el) <= 0, off_by(got, rows, el)

    def grad_ok(g, c):  # c: (N,) factor of each row
        assert g.dtype == z.dtype and g.shape == z.shape
        want, tol = grad * c[:, None], (eg + 4 * U * grad.abs()) * c[:, None].abs()
        half = 0 if z.dtype == torch.float32 else torch.finfo(z.dtype).eps / 2
        tol = tol + (want.abs() + tol) * half + TINY[z.dtype]
        assert off_by(g, want, tol) <= 0, off_by(g, want, tol)

    w = torch.rand(z.shape[0], device=z.device) + 0.5
    x = z.detach().requires_grad_(True)
    (g,) = torch.autograd.grad(call(x, reduction="none"), x, w * upstream)
    grad_ok(g, w.double() * upstream)
    for red, c in (("sum", 1.0), ("mean", 1.0 / max(n, 1))):
        if red == "mean" and n == 0:
            continue
        tol = float((el * counts).sum()) * c + 4 * U * float(rows.abs().sum()) * c
        want = float(rows.sum()) * c
        loss = call(x, reduction=red)
        assert loss.shape == () and abs(float(loss.detach()) - want) <= tol
        assert torch.equal(loss.detach(), call(z, reduction=red))
        up = torch.tensor(upstream, device=z.device)
        (g,) = torch.autograd.grad(loss, x, up)
        grad_ok(g, torch.full_like(rows, c * upstream))
        for s in (upstream, up):
            loss1, g1 = step(z, reduction=red, grad_scale=s)
            assert abs(float(loss1) - want) <= tol
            grad_ok(g1, torch.full_like(rows, c * upstream))
            assert bool((g1[~counts] == 0).all())


def make(cuda, N, V, dtype, K=0, seed=0, ignored=0.2, spread=3.0):
    g = torch.Generator(device=cuda).manual_seed(seed + N * 7 + V)
    z = (torch.randn(N, V, generator=g, device=cuda) * spread).to(DT[dtype])
    y = torch.randint(0, V, (N,), generator=g, device=cuda)
    y[torch.rand(N, generator=g, device=cuda) < ignored] = -100
    if not K:
        return z, y, None, None
    tid = torch.randint(0, V, (N, K), generator=g, device=cuda)  # some ids twice
    tlog = (torch.randn(N, K, generator=g, device=cuda) * 2 + 5).to(DT[dtype])
    return z, y, tid, tlog


SIZES = [(1, 1), (1, 2), (2, 7), (5, 64), (33, 100), (7, 257), (4, 1000), (3, 2049), (2, 4097), (3, 8193), (2, 16385),
         (3, 32001), (2, 50257), (2, 65537), (1, 131073), (1, 200003)]


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("N,V", SIZES)
def test_cross_entropy(cuda, N, V, dtype):
    check_all(*make(cuda, N, V, dtype)[:2], upstream=512.0 if dtype == "fp16" else 1.0)


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("N,V,K,T,soft", [(1, 2, 1, 1.0, 1.0), (5, 64, 64, 2.0, 0.5), (9, 257, 20, 0.7, 0.25),
                                          (4, 4097, 128, 2.0, 0.5), (3, 1000, 1024, 4.0, 0.9), (2, 50257, 64, 2.0, 0.5),
                                          (2, 32000, 300, 1.0, 1.0), (2, 70001, 33, 1.5, 0.5), (1, 140001, 7, 1.0, 0.5),
                                          (6, 100, 5, 1.0, 0.0)])
def test_distillation(cuda, N, V, K, T, soft, dtype):
    z, y, tid, tlog = make(cuda, N, V, dtype, K)
    check_all(z, y, tid, tlog, T, soft, upstream=64.0 if dtype == "fp16" else 1.0)
    check_all(z, y.int(), tid.int(), tlog.float(), T, soft, upstream=64.0 if dtype == "fp16" else 1.0)


@pytest.mark.parametrize("soft", [0.4, 1.0])
def test_teacher_pairs_absent_or_twice(cuda, soft):
    z, y, tid, tlog = make(cuda, 8, 500, "fp32", 12)
    tid[0, 5:] = -1
    tid[1] = -1                       # none at all
    tlog[2, 3:9] = -math.inf
    tlog[3] = -math.inf               # none at all
    tid[4] = 17                       # one id K times
    tid[5, :6], y[5] = 499, 499       # the label among them, twice and more
    tid[6, 0], tid[6, 1] = 500, 1 << 20
    y[6], y[1], y[3] = 3, 4, 5
    check_all(z, y, tid, tlog, 1.3, soft)


def test_without_labels(cuda):
    z, _, tid, tlog = make(cuda, 5, 300, "bf16", 9)
    check_all(z, None, tid, tlog, 2.0, 1.0)


@pytest.mark.parametrize("N,V", [(4, 300), (3, 20001), (2, 140001)])
def test_special_values(cuda, N, V):
    """Masked logits (-inf, and the type's lowest value), a row of one value, large values; ignored rows of NaN."""
    z, y, tid, tlog = make(cuda, N + 4, V, "fp32", 6, ignored=0.0)
    keep = y.clone()
    z[0, : V // 2] = -math.inf
    z[1, : V // 2] = torch.finfo(torch.float32).min
    z[2] = 1.75
    z[3] = z[3] * 1000
    y[0], y[1] = V - 1, V - 2
    tid[0], tid[1] = V // 2 + torch.arange(6, device=cuda), V // 2 + torch.arange(6, device=cuda)
    z[4:5] = math.nan
    y[4] = -100
    check_all(z, y)
    check_all(z[:3], y[:3], tid[:3], tlog[:3], 2.0, 0.5)
    # a whole row of -inf, an infinity, a NaN: NaN losses and gradients as log_softmax's, of those rows alone
    z, y = z[: N + 3].clone(), keep[: N + 3].clone()
    z[:] = torch.randn(z.shape, device=cuda)
    z[0], z[1, 0], z[2, 1] = -math.inf, math.inf, math.nan
    y[:3] = V - 1
    rows = cross_entropy(z, y, reduction="none")
    want = torch.nn.functional.cross_entropy(z.double(), y, reduction="none")
    assert torch.equal(rows.isnan(), want.isnan())
    x = z.requires_grad_(True)
    (g,) = torch.autograd.grad(cross_entropy(x, y, reduction="sum"), x)
    assert bool(g[:3].isnan().any(-1).all()) and bool(torch.isfinite(g[3:]).all())
    # the label masked: an infinite loss, as F.cross_entropy's
    z = torch.zeros(2, V, device=cuda)
    z[0, 0] = -math.inf
    y = torch.zeros(2, dtype=torch.long, device=cuda)
    assert cross_entropy(z, y, reduction="none")[0] == math.inf
    _, g = loss_and_grad(z, y, reduction="sum")
    assert g[0, 0] == -1 and abs(float(g[0, 1:].sum()) - 1) < 1e-4


def test_labels_outside_the_vocabulary(cuda):
    z = torch.randn(5, 40, device=cuda)
    y = torch.tensor([3, 40, -1, 1 << 40, -100], device=cuda)
    rows = cross_entropy(z, y, reduction="none")
    assert rows.isnan().tolist() == [False, True, True, True, False] and rows[4] == 0
    x = z.clone().requires_grad_(True)
    (g,) = torch.autograd.grad(cross_entropy(x, y, reduction="sum"), x)
    assert g.isnan().all(-1).tolist() == [False, True, True, True, False] and bool((g[4] == 0).all())
    assert not cross_entropy(z, y, ignore_index=40, reduction="none")[1].isnan()


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("B,S,V", [(2, 5, 33), (3, 1, 50), (1, 9, 5001)])
def test_shift(cuda, B, S, V, dtype):
    """Row s against label s + 1: the same as slicing and copying, without it."""
    z, y, tid, tlog = make(cuda, B * S, V, dtype, 8)
    z, y, tid, tlog = z.view(B, S, V), y.view(B, S), tid.view(B, S, 8), tlog.view(B, S, 8)
    moved = torch.cat([y[:, 1:], torch.full_like(y[:, :1], -100)], 1)
    for kw in ({}, dict(teacher_ids=tid, teacher_logits=tlog, temperature=2.0)):
        a, ga = loss_and_grad(z, y, shift=True, **kw)
        b, gb = loss_and_grad(z, moved, **kw)
        assert torch.equal(a, b) or (a.isnan() and b.isnan())
        assert ga.shape == z.shape and torch.equal(ga, gb)
    rows = cross_entropy(z, y, shift=True, reduction="none")
    assert rows.shape == (B, S) and bool((rows[:, -1] == 0).all())
    assert torch.equal(rows, cross_entropy(z, moved, reduction="none"))


def test_nothing_counts(cuda):
    z = torch.randn(3, 50, device=cuda, requires_grad=True)
    y = torch.full((3,), -100, device=cuda)
    loss = cross_entropy(z, y)
    assert loss.isnan()
    (g,) = torch.autograd.grad(loss, z)
    assert bool((g == 0).all())
    loss, g = loss_and_grad(z.detach(), y)
    assert loss.isnan() and bool((g == 0).all())
    assert cross_entropy(z.detach(), y, reduction="sum") == 0
    e = torch.zeros(0, 7, device=cuda)
    n = torch.zeros(0, dtype=torch.long, device=cuda)
    assert cross_entropy(e, n).isnan() and cross_entropy(e, n, reduction="sum") == 0
    assert cross_entropy(e, n, reduction="none").shape == (0,) and loss_and_grad(e, n)[1].shape == (0, 7)


def test_views(cuda):
    """Row strides and addresses other than those of a contiguous tensor; one row without any other."""
    base = torch.randn(6, 1037, device=cuda).bfloat16()
    y = torch.randint(0, 900, (6,), device=cuda)
    tid, tlog = torch.randint(0, 900, (6, 40), device=cuda), torch.randn(6, 40, device=cuda)
    for v in (base[:, :1000], base[:, 1:1001], base[:, 3:], base[::2], base.t().contiguous().t(), base[2:3, 5:],
              base.float()[:, 2:], base.float()[:, :1036]):
        n = v.shape[0]
        check_all(v, y[:n], tid[:n, ::2], tlog[:n, 4:24], 2.0, 0.5)
        check_all(v, y[:n])
    one = cross_entropy(base[0], y[0])  # (V,) and a single label
    assert one.shape == () and torch.equal(one, cross_entropy(base[:1], y[:1]))


def test_reproducible(cuda):
    z, y, tid, tlog = make(cuda, 64, 5000, "bf16", 50)
    a = loss_and_grad(z, y, teacher_ids=tid, teacher_logits=tlog, temperature=2.0)
    for _ in range(3):
        b = loss_and_grad(z, y, teacher_ids=tid, teacher_logits=tlog, temperature=2.0)
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


def test_gradient_by_differences(cuda):
    g = torch.Generator(device=cuda).manual_seed(0)
    z = torch.randn(3, 40, generator=g, device=cuda)
    y = torch.randint(0, 40, (3,), generator=g, device=cuda)
    tid = torch.randint(0, 40, (3, 6), generator=g, device=cuda)
    tlog = torch.randn(3, 6, generator=g, device=cuda)
    fn = lambda x: distillation_loss(x, y, tid, tlog, temperature=1.5, soft_weight=0.4, reduction="sum")  # noqa: E731
    x = z.clone().requires_grad_(True)
    (d,) = torch.autograd.grad(fn(x), x)
    for r, j in ((0, 0), (1, int(y[1])), (2, int(tid[2, 3])), (0, 39)):
        e = torch.zeros_like(z)
        e[r, j] = 2.0 ** -5
        # the difference's own error: the third derivative (below 1) times h^2 / 6, and 2e-6 of the losses over 2 h
        assert abs((float(fn(z + e)) - float(fn(z - e))) * 2.0 ** 4 - float(d[r, j])) < 2e-4 + 4e-5 * 16


def test_higher_derivatives_and_batched_gradients(cuda):
    z = torch.randn(3, 20, device=cuda, requires_grad=True)
    y = torch.tensor([1, -100, 4], device=cuda)
    tid, tlog = torch.randint(0, 20, (3, 4), device=cuda), torch.randn(3, 4, device=cuda)
    loss = distillation_loss(z, y, tid, tlog, temperature=2.0)
    (g1,) = torch.autograd.grad(loss, z, create_graph=True)
    (g2,) = torch.autograd.grad((g1 * g1).sum(), z)
    _, first = loss_and_grad(z.detach(), y, teacher_ids=tid, teacher_logits=tlog, temperature=2.0)
    assert torch.allclose(g1, first, atol=1e-6) and bool((g2[1] == 0).all()) and bool((g2[0] != 0).any())
    rows = cross_entropy(z, y, reduction="none")
    (gb,) = torch.autograd.grad(rows, z, torch.eye(3, device=cuda), is_grads_batched=True)
    assert gb.shape == (3, 3, 20) and bool((gb[1] == 0).all())


def test_transforms_of_torch(cuda):
    z, y, tid, tlog = make(cuda, 4, 30, "fp32", 5)
    kw = dict(temperature=2.0, reduction="sum")
    _, want = loss_and_grad(z, y, teacher_ids=tid, teacher_logits=tlog, **kw)
    got = torch.func.grad(lambda x: distillation_loss(x, y, tid, tlog, **kw))(z)
    assert torch.allclose(got, want, atol=1e-6)
    loss, tangent = torch.func.jvp(lambda x: cross_entropy(x, y, reduction="none"), (z,), (torch.ones_like(z),))
    assert torch.allclose(loss, cross_entropy(z, y, reduction="none"), atol=1e-5) and bool((tangent.abs() < 1e-5).all())


def test_past_32_bit_offsets(cuda):
    """Logits and a gradient of over 2^32 bytes and 2^31 elements: the last rows are those of the rows alone."""
    N, V = 44000, 50257
    z = torch.zeros(N, V, dtype=torch.bfloat16, device=cuda)
    g = torch.Generator(device=cuda).manual_seed(1)
    z[-3:] = torch.randn(3, V, generator=g, device=cuda).bfloat16() * 3
    y = torch.full((N,), -100, device=cuda)
    y[-3:], y[0] = torch.tensor([5, 50256, 777], device=cuda), 1
    rows = cross_entropy(z, y, reduction="none")
    assert torch.equal(rows[-3:], cross_entropy(z[-3:], y[-3:], reduction="none")) and bool((rows[1:-3] == 0).all())
    _, dz = loss_and_grad(z, y, reduction="sum")
    _, alone = loss_and_grad(z[-3:], y[-3:], reduction="sum")
    assert torch.equal(dz[-3:], alone) and not bool(dz[1:-3].any())
    del dz
    x = z.requires_grad_(True)
    (dz,) = torch.autograd.grad(cross_entropy(x, y, reduction="sum"), x)
    assert off_by(dz[-3:], alone, 2.0 ** -8 * alone.double().abs() + 1e-30) <= 0 and not bool(dz[1:-3].any())


def test_leaf_changed_before_the_backward_is_noticed(cuda):
    z = torch.randn(3, 20, device=cuda, requires_grad=True)
    x = z * 1
    loss = cross_entropy(x, torch.zeros(3, dtype=torch.long, device=cuda))
    x.add_(1)
    with pytest.raises(RuntimeError, match="modified"):
        loss.backward()


def test_another_stream(cuda):
    z, y, tid, tlog = make(cuda, 40, 3001, "bf16", 16)
    want = loss_and_grad(z, y, teacher_ids=tid, teacher_logits=tlog)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        got = loss_and_grad(z, y, teacher_ids=tid, teacher_logits=tlog)
    side.synchronize()
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_refusals(cuda):
    z, y = torch.zeros(4, 9, device=cuda), torch.zeros(4, dtype=torch.long, device=cuda)
    k, t = torch.zeros(4, 3, dtype=torch.long, device=cuda), torch.zeros(4, 3, device=cuda)
    for call, err in (
            (lambda: cross_entropy(z.double(), y), TypeError), (lambda: cross_entropy(z, y.float()), TypeError),
            (lambda: cross_entropy(z, y[:3]), ValueError), (lambda: cross_entropy(z, y.cpu()), ValueError),
            (lambda: cross_entropy(z[:, :0], y), ValueError), (lambda: cross_entropy(z, y, reduction="avg"), ValueError),
            (lambda: cross_entropy(z[0], y[0], shift=True), ValueError),
            (lambda: distillation_loss(z, y, k, t, temperature=0.0), ValueError),
            (lambda: distillation_loss(z, y, k, t, temperature=math.nan), ValueError),
            (lambda: distillation_loss(z, y, k, t, soft_weight=1.5), ValueError),
            (lambda: distillation_loss(z, None, k, t), ValueError),
            (lambda: distillation_loss(z[None], None, k[None], t[None], soft_weight=1.0, shift=True), ValueError),
            (lambda: distillation_loss(z, y, k[:3], t[:3]), ValueError),
            (lambda: distillation_loss(z, y, k, t[:, :2]), ValueError),
            (lambda: distillation_loss(z, y, k.float(), t), TypeError),
            (lambda: distillation_loss(z, y, k, t.double()), TypeError),
            (lambda: distillation_loss(z, y, k.cpu(), t), ValueError),
            (lambda: distillation_loss(z, y, k[:, :0], t[:, :0]), ValueError),
            (lambda: distillation_loss(z, y, k.repeat(1, 400), t.repeat(1, 400)), ValueError),
            (lambda: loss_and_grad(z, y, grad_scale=torch.ones(2, device=cuda)), ValueError),
            (lambda: loss_and_grad(z, y, grad_scale=torch.ones(())), ValueError)):
        with pytest.raises(err):
            call()
