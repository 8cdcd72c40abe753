"""layer_norm, label_loss and sample_labels on the GPU against plain implementations in 64 bits on the CPU.

Tolerances count roundings.  A result held in type t is off by at most half a step, `eps(t) / 2` relative to its value; what is computed
in float32 before that adds E = 2^-24 per operation on the magnitudes that meet in it."""
import math

import pytest
import torch

import bournemouth_forced_aligner_amd as bfa

pytestmark = pytest.mark.gpu
E = 2.0 ** -24
TYPES = [torch.float32, torch.float16, torch.bfloat16]
ids = lambda t: str(t).replace("torch.", "")  # noqa: E731


def half_step(t):
    return torch.finfo(t).eps / 2


def rows_of(B, T, C, dtype, seed, pitch=0, scale=1.0, shift=0.0):
    """[B, T, C] on the GPU (a view into rows of `pitch` elements) and in 64 bits on the CPU"""
    g = torch.Generator().manual_seed(seed)
    x = (torch.randn((B, T, C), generator=g) * scale + shift).to(dtype)
    store = torch.full((B, T, max(pitch, C)), float("nan"), dtype=dtype)
    store[..., :C] = x
    return store.cuda()[..., :C], x.double()


def held_of(B, T, lengths):
    if lengths is None:
        return torch.ones(B, T, dtype=torch.bool)
    return torch.arange(T)[None] < torch.tensor(lengths)[:, None]


# ---- layer_norm --------------------------------------------------------------------------------------------------------------

def norm_ref(x, w, b, gy, held, eps):
    """y, dx, dw, db, mean, rstd by the formulas, and a bound on |y| and |dx| before cancellation"""
    x = torch.where(held[..., None], x, torch.zeros(()).double())
    gy = torch.where(held[..., None], gy, torch.zeros(()).double())
    mean = x.mean(-1, keepdim=True)
    var = ((x - mean) ** 2).mean(-1, keepdim=True)
    r = 1 / torch.sqrt(var + eps)
    xh = (x - mean) * r
    h = held[..., None].double()
    y = (xh * w + b) * h
    g = gy * w
    dx = r * (g - g.mean(-1, keepdim=True) - xh * (g * xh).mean(-1, keepdim=True)) * h
    return y, dx, (gy * xh).sum((0, 1)), gy.sum((0, 1)), mean[..., 0] * h[..., 0], r[..., 0] * h[..., 0], xh


CASES = [  # B, T, C, pitch, lengths: one row and many, every layout of threads (16, 64, 256, 1024, swept), odd ends
    (1, 1, 1, 0, None), (3, 5, 2, 0, None), (2, 3, 7, 11, [3, 1]), (1, 1, 8, 0, None), (2, 9, 17, 0, [0, 9]), (4, 33, 67, 68, [33, 1, 0, 20]),
    (1, 300, 256, 0, None), (2, 5, 257, 0, None), (3, 50, 768, 0, [50, 2, 49]), (1, 7, 1001, 1007, None), (2, 4, 1024, 0, None),
    (2, 3, 1025, 0, [1, 3]), (1, 5, 4096, 0, None), (1, 3, 4099, 4100, None), (2, 2, 16384, 0, None), (1, 2, 16385, 0, None),
    (2, 3, 20003, 20010, [2, 3]),
]


@pytest.mark.parametrize("dtype", TYPES, ids=ids)
@pytest.mark.parametrize("case", CASES, ids=lambda c: "x".join(map(str, c[:3])))
def test_layer_norm_and_its_gradients(case, dtype, gpu_device):
    B, T, C, pitch, lengths = case
    wt = torch.float32 if C % 2 else dtype
    x, xd = rows_of(B, T, C, dtype, 1, pitch, 1.5, 0.5)
    gy, gyd = rows_of(B, T, C, dtype, 2)
    w = (1 + 0.2 * torch.randn(C, generator=torch.Generator().manual_seed(3))).to(wt)
    b = (0.2 * torch.randn(C, generator=torch.Generator().manual_seed(4))).to(wt)
    held = held_of(B, T, lengths)
    want = norm_ref(xd, w.double(), b.double(), gyd, held, 1e-5)
    xs, ws, bs = x.requires_grad_(), w.cuda().requires_grad_(), b.cuda().requires_grad_()
    y = bfa.layer_norm(xs, ws, bs, lengths=lengths)
    dx, dw, db = torch.autograd.grad(y, (xs, ws, bs), gy)
    assert y.dtype == dx.dtype == dtype and dw.dtype == db.dtype == wt
    y, dx, dw, db = (t.detach().cpu().double() for t in (y, dx, dw, db))
    wy, wdx, wdw, wdb, _, rstd, xh = want
    h = half_step(dtype)
    # a row's statistics: a sum of C terms in float32, log2(C) + 16 additions deep, of magnitudes up to max |x|
    deep = math.log2(C) + 24
    amp = xd.abs().amax(-1, keepdim=True) * rstd[..., None] + xh.abs().amax(-1, keepdim=True)
    tol = h * wy.abs() + E * deep * (amp * w.double().abs() + b.double().abs()) * (1 + xh.abs()) + 1e-30
    assert bool(((y - wy).abs() <= tol).all()), float(((y - wy).abs() / tol).max())
    assert bool((y[~held] == 0).all()) and bool((dx[~held] == 0).all())
    g = (gyd * w.double()).abs().amax(-1, keepdim=True)
    tol = h * wdx.abs() + E * deep * rstd[..., None] * g * (1 + amp) ** 2 * 4 + (6e-8 if dtype == torch.float16 else 1e-30)  # (fp16: half its smallest step)
    assert bool(((dx - wdx).abs() <= tol).all()), float(((dx - wdx).abs() / tol).max())
    n = int(held.sum())
    depth = n / 1.0 + 32  # at most every row in one chain
    hw = half_step(wt)
    terms = (gyd.abs() * held[..., None] * (xh.abs() + amp * deep)).sum((0, 1))
    assert bool(((dw - wdw).abs() <= hw * wdw.abs() + E * depth * terms + 1e-7).all())
    assert bool(((db - wdb).abs() <= hw * wdb.abs() + E * depth * (gyd.abs() * held[..., None]).sum((0, 1)) + 1e-7).all())


def test_layer_norm_statistics_parts_and_flat_rows(gpu_device):
    x, xd = rows_of(6, 5, 40, torch.float32, 5)
    y, mean, rstd = bfa.layer_norm_forward(x, eps=1e-3, lengths=[5, 0, 1, 2, 5, 4])
    held = held_of(6, 5, [5, 0, 1, 2, 5, 4])
    one, zero = torch.ones(40).double(), torch.zeros(40).double()
    wy, _, _, _, wm, wr, _ = norm_ref(xd, one, zero, xd, held, 1e-3)
    assert torch.allclose(mean.cpu().double(), wm, atol=1e-6) and torch.allclose(rstd.cpu().double(), wr, rtol=1e-6)
    assert torch.allclose(y.cpu().double(), wy, atol=1e-5)
    flat = bfa.layer_norm(x.reshape(30, 40))
    assert torch.equal(flat.reshape(6, 5, 40), bfa.layer_norm(x)) and torch.equal(bfa.layer_norm(x[0, 0]), flat[0])
    assert torch.equal(bfa.layer_norm(x.reshape(2, 3, 5, 40)).reshape(6, 5, 40), bfa.layer_norm(x))
    g, _ = rows_of(6, 5, 40, torch.float32, 6)
    y, mean, rstd = bfa.layer_norm_forward(x)
    full = bfa.layer_norm_backward(g, x, mean, rstd)
    for need in ((True, False, False), (False, True, False), (False, False, True), (False, False, False)):
        part = bfa.layer_norm_backward(g, x, mean, rstd, need=need)
        for got, all_, n in zip(part, full, need):
            assert (got is None) == (not n) and (got is None or torch.equal(got, all_))


@pytest.mark.parametrize("dtype", TYPES, ids=ids)
def test_layer_norm_of_constant_rows_and_far_means(dtype, gpu_device):
    """a constant row is its bias; a mean far from 0 costs no more than the inputs' own rounding"""
    x = torch.full((3, 130), 7.0, dtype=dtype, device="cuda")
    b = torch.arange(130, dtype=torch.float32, device="cuda")
    assert torch.equal(bfa.layer_norm(x, None, b), b.to(dtype).expand(3, 130))
    x, xd = rows_of(2, 4, 512, torch.float32, 9, scale=1.0, shift=1000.0)
    m = xd.mean(-1, keepdim=True)
    want = (xd - m) / torch.sqrt(((xd - m) ** 2).mean(-1, keepdim=True) + 1e-5)
    # the mean is off by at most 1000 * E * (log2(512) + 8)
    assert float((bfa.layer_norm(x).cpu().double() - want).abs().max()) <= 1004 * E * 17 * 1.2 + 1e-5


def test_layer_norm_not_finite_rows_stay_in_their_row(gpu_device):
    x, _ = rows_of(4, 1, 300, torch.float32, 11)
    x = x.clone()
    x[1, 0, 5], x[2, 0, 299] = float("nan"), float("inf")
    y = bfa.layer_norm(x)
    ok = bfa.layer_norm(x[[0, 3]])
    assert torch.equal(y[[0, 3]], ok) and bool(torch.isnan(y[1]).all()) and bool(torch.isnan(y[2]).any())


def test_layer_norm_gradient_against_differences(gpu_device):
    x, xd = rows_of(2, 3, 33, torch.float32, 12)
    w, b = torch.rand(33, device="cuda") + 0.5, torch.rand(33, device="cuda")
    g, gd = rows_of(2, 3, 33, torch.float32, 13)
    f = lambda v: torch.nn.functional.layer_norm(v, (33,), w.cpu().double(), b.cpu().double(), 1e-5)  # noqa: E731
    xs = x.clone().requires_grad_()
    dx, = torch.autograd.grad(bfa.layer_norm(xs, w, b), (xs,), g)
    d = torch.randn(2, 3, 33, generator=torch.Generator().manual_seed(14)).double()
    step = 1e-5
    want = float(((f(xd + step * d) - f(xd - step * d)) / (2 * step) * gd).sum())
    assert abs(float((dx.cpu().double() * d).sum()) - want) <= 1e-4


# ---- label_loss --------------------------------------------------------------------------------------------------------------

def loss_ref(z, labels, weights, held, reduction):
    C = z.shape[-1]
    w = torch.ones(labels.shape).double() if weights is None else weights.double()
    counts = held & (labels >= 0) & (w != 0)
    m = z.amax(-1, keepdim=True)
    e = torch.exp(z - m)
    s = e.sum(-1, keepdim=True)
    lab = labels.clamp(0, C - 1).long()[..., None]
    nll = (m + torch.log(s) - z.gather(-1, lab))[..., 0]
    zero = torch.zeros(()).double()
    nll = torch.where(counts, w * nll, zero)
    p = e / s - torch.zeros_like(z).scatter_(-1, lab, 1.0)
    total = torch.where(counts, w, zero).sum()
    scale = 1.0 if reduction != "mean" else (0.0 if total == 0 else 1.0 / float(total))
    grad = torch.where(counts[..., None], p * w[..., None] * scale, zero)
    loss = nll if reduction == "none" else nll.sum() * scale
    return loss, grad, (e / s), counts, scale


LOSS_CASES = [  # B, T, C, pitch, lengths, weighted
    (1, 1, 1, 0, None, False), (1, 1, 2, 0, None, True), (3, 40, 3, 5, [40, 0, 7], True), (2, 65, 17, 0, [65, 30], False), (2, 20, 32, 0, None, True),
    (4, 100, 67, 68, [100, 1, 0, 55], True), (5, 31, 67, 0, None, False), (1, 9, 128, 0, None, True), (2, 7, 129, 130, [7, 2], False),
    (1, 5, 512, 0, None, True), (3, 6, 513, 0, [6, 0, 3], True), (1, 4, 2049, 2051, None, False), (2, 3, 5003, 0, [3, 2], True), (1, 3, 8193, 0, None, True),
    (1, 2, 32769, 0, None, False), (1, 2, 70001, 70010, None, True), (1, 2, 140003, 0, None, True),
]


@pytest.mark.parametrize("reduction", ["mean", "sum", "none"])
@pytest.mark.parametrize("dtype", TYPES, ids=ids)
@pytest.mark.parametrize("case", LOSS_CASES, ids=lambda c: "x".join(map(str, c[:3])))
def test_label_loss_and_its_gradient(case, dtype, reduction, gpu_device):
    B, T, C, pitch, lengths, weighted = case
    z, zd = rows_of(B, T, C, dtype, 21, pitch, 3.0)
    g = torch.Generator().manual_seed(22)
    labels = torch.randint(-1, C, (B, T), generator=g, dtype=torch.int32)
    weights = torch.rand((B, T), generator=g).masked_fill_(torch.rand((B, T), generator=g) < 0.2, 0.0) if weighted else None
    held = held_of(B, T, lengths)
    loss, grad, p, counts, scale = loss_ref(zd, labels, weights, held, reduction)
    up = 1.5 if reduction != "none" else 1.0
    args = dict(weights=None if weights is None else weights.cuda(), lengths=lengths, reduction=reduction)
    got, ggrad = bfa.label_loss_and_grad(z, labels.cuda(), grad_scale=up, **args)
    assert ggrad.dtype == dtype and got.dtype == torch.float32
    # exp and the sum: each factor off by a few E (|z - m| <= 40: its difference, product and exponential), sums log2(C) + 16 deep
    deep = math.log2(C) + 32
    mag = (zd.abs().amax(-1) + math.log(C) + 1)
    wt = torch.ones(B, T).double() if weights is None else weights.double()
    each = E * deep * mag * wt * counts
    tol = each if reduction == "none" else each.sum() * scale + E * float(loss.abs()) * 4
    assert bool(((got.cpu().double() - loss).abs() <= tol + 1e-12).all()), (got, loss)
    tol = half_step(dtype) * (grad * up).abs() + E * up * scale * (wt * counts)[..., None] * (p * (deep + 4 * mag[..., None]) + 4)
    tol = tol + {torch.float16: 2.0 ** -25, torch.bfloat16: 1e-38, torch.float32: 1e-38}[dtype]
    err = (ggrad.cpu().double() - grad * up).abs()
    assert bool((err <= tol).all()), float((err / tol).max())
    assert bool((ggrad.cpu()[~counts] == 0).all())
    # the same through autograd, and the loss alone
    zs = z.detach().requires_grad_()
    l2 = bfa.label_loss(zs, labels.cuda(), **args)
    g2, = torch.autograd.grad(l2, (zs,), torch.full_like(l2, up))
    assert torch.equal(l2, got) and torch.equal(g2, ggrad)
    assert torch.equal(bfa.label_loss(z.detach(), labels.cuda(), **args), got)


def test_label_loss_upstream_per_row(gpu_device):
    z, zd = rows_of(3, 11, 67, torch.float32, 23)
    labels = torch.randint(0, 67, (3, 11), generator=torch.Generator().manual_seed(1))
    up = torch.randn(3, 11, generator=torch.Generator().manual_seed(2))
    zs = z.requires_grad_()
    g, = torch.autograd.grad(bfa.label_loss(zs, labels.cuda(), reduction="none"), (zs,), up.cuda())
    _, want, p, _, _ = loss_ref(zd, labels, None, held_of(3, 11, None), "none")
    assert bool(((g.cpu().double() - want * up.double()[..., None]).abs() <= E * up.double().abs()[..., None] * (64 * p + 8)).all())


def test_label_loss_gradient_against_differences(gpu_device):
    z, zd = rows_of(2, 5, 67, torch.float32, 24, scale=2.0)
    labels = torch.randint(0, 67, (2, 5), generator=torch.Generator().manual_seed(3))
    w = torch.rand(2, 5, generator=torch.Generator().manual_seed(4))
    d = torch.randn(2, 5, 67, generator=torch.Generator().manual_seed(5)).double()
    f = lambda v: float(loss_ref(v, labels, w, held_of(2, 5, [5, 3]), "mean")[0])  # noqa: E731
    _, g = bfa.label_loss_and_grad(z, labels.cuda(), weights=w.cuda(), lengths=[5, 3])
    want = (f(zd + 1e-5 * d) - f(zd - 1e-5 * d)) / 2e-5
    assert abs(float((g.cpu().double() * d).sum()) - want) <= 1e-6


@pytest.mark.parametrize("C", [67, 300, 3000])
def test_label_loss_masks_and_bad_rows(C, gpu_device):
    z, zd = rows_of(1, 9, C, torch.float32, 25)
    z = z.clone()
    z[0, 0, 1:] = float("-inf")          # one class left, and it is the label: loss 0
    z[0, 1, :] = torch.finfo(torch.float32).min  # the type's lowest everywhere: even
    z[0, 2, 3] = float("nan")
    z[0, 3, :] = float("-inf")           # nothing left
    z[0, 4, 2] = float("-inf")           # the label itself masked
    labels = torch.tensor([[0, 5, 1, 1, 2, C, -1, -100, 4]], dtype=torch.int64)
    loss, grad = bfa.label_loss_and_grad(z, labels.cuda(), reduction="none")
    loss, grad = loss.cpu()[0], grad.cpu()[0]
    assert float(loss[0]) == 0.0 and bool((grad[0] == 0).all())
    assert abs(float(loss[1]) - math.log(C)) <= 1e-5 and abs(float(grad[1, 5]) - (1 / C - 1)) <= 1e-6
    assert bool(torch.isnan(loss[2])) and bool(torch.isnan(grad[2]).all())
    assert bool(torch.isnan(loss[3])) and float(loss[4]) == math.inf and float(grad[4, 2]) == -1.0
    assert bool(torch.isnan(loss[5])) and bool(torch.isnan(grad[5]).all())   # a label the row does not have
    assert float(loss[6]) == float(loss[7]) == 0.0 and bool((grad[6:8] == 0).all())
    want = loss_ref(zd[:, 8:], torch.tensor([[4]]), None, held_of(1, 1, None), "none")[0]
    assert abs(float(loss[8]) - float(want)) <= 1e-5


def test_label_loss_with_nothing_that_counts(gpu_device):
    z, _ = rows_of(2, 3, 67, torch.float32, 26)
    for kw in (dict(labels=torch.full((2, 3), -1)), dict(labels=torch.zeros(2, 3, dtype=torch.int32), lengths=[0, 0]),
               dict(labels=torch.zeros(2, 3, dtype=torch.int32), weights=torch.zeros(2, 3))):
        kw = {k: v.cuda() if isinstance(v, torch.Tensor) else v for k, v in kw.items()}
        for red in ("mean", "sum"):
            loss, g = bfa.label_loss_and_grad(z, reduction=red, **kw)
            assert float(loss) == 0.0 and bool((g == 0).all())
    for shape in ((0, 3, 67), (2, 0, 67)):
        e = torch.empty(shape, device="cuda")
        lab = torch.empty(shape[:2], dtype=torch.int32, device="cuda")
        loss, g = bfa.label_loss_and_grad(e, lab)
        assert float(loss) == 0.0 and g.shape == shape
        assert bfa.label_loss(e, lab, reduction="none").shape == shape[:2]
        assert bfa.layer_norm(e).shape == shape
        assert bfa.sample_labels(e, torch.empty(shape[:2], device="cuda"))[0].shape == shape[:2]
        y, mean, rstd = bfa.layer_norm_forward(e)
        assert all(bool((t == 0).all()) for t in bfa.layer_norm_backward(e, e, mean, rstd)[1:])


# ---- sample_labels -----------------------------------------------------------------------------------------------------------

def sample_ref(z, u, temperature, top_k, top_p, min_p, held):
    """row by row, as the definition says it; parameters [B] as the call rounds them"""
    B, T, C = z.shape
    labels, logp = torch.full((B, T), -1, dtype=torch.int32), torch.zeros(B, T).double()
    for b in range(B):
        t, k, p, q = float(temperature[b]), int(top_k[b]), float(top_p[b]), float(min_p[b])
        for i in range(T):
            row = torch.where(torch.isnan(z[b, i]), -math.inf, z[b, i])
            best = float(row.max())
            if not held[b, i] or best == -math.inf:
                continue
            order = sorted(range(C), key=lambda c: (-float(row[c]), c))
            if not t > 0:
                labels[b, i] = order[0]
                continue
            w = [1.0 if float(row[c]) == best else (0.0 if float(row[c]) == -math.inf else math.exp((float(row[c]) - best) / t)) for c in order]
            n = C if k <= 0 else min(k, C)
            if p < 1:
                target, M, m = p * math.fsum(w[:n]), 0.0, 0
                while m < n and M < target:
                    M += w[m]
                    m += 1
                n = m
            n = max(1, min(n, sum(1 for v in w if v >= q)))
            kept = sorted((c, v) for c, v in zip(order[:n], w[:n]))
            W = math.fsum(v for _, v in kept)
            M, pick = 0.0, None
            for c, v in kept:
                M += v
                if v > 0:
                    pick = (c, v)
                    if M > float(u[b, i]) * W:
                        break
            labels[b, i] = pick[0]
            logp[b, i] = math.log(pick[1]) - math.log(W)
    return labels, logp


def run_sample(B, T, C, dtype, seed, lengths=None, pitch=0, scale=2.0, prep=None, each=True, **prm):
    z, zd = rows_of(B, T, C, dtype, seed, pitch, scale)
    if prep is not None:
        z = prep(z.clone())
        zd = z.cpu().double()
    u = torch.rand(B, T, generator=torch.Generator().manual_seed(seed + 1))
    full = dict(temperature=torch.ones(B), top_k=torch.zeros(B, dtype=torch.int32), top_p=torch.ones(B), min_p=torch.zeros(B))
    for k, v in prm.items():
        full[k] = torch.as_tensor(v, dtype=full[k].dtype).expand(B).contiguous() if not torch.is_tensor(v) or v.dim() == 0 else v.to(full[k].dtype)
    want, wlp = sample_ref(zd, u, **full, held=held_of(B, T, lengths))
    call = {k: v.cuda() for k, v in full.items()} if each else prm
    got, lp = bfa.sample_labels(z, u.cuda(), lengths=lengths, **call)
    assert got.dtype == torch.int32 and lp.dtype == torch.float32
    assert torch.equal(got.cpu(), want), (got.cpu()[got.cpu() != want], want[got.cpu() != want])
    # log1p of W - 1 and the difference, in float32
    tol = E * (16 + 4 * wlp.abs()) + E * 8 * math.log(C + 1)
    assert bool(((lp.cpu().double() - wlp).abs() <= tol).all())


PARAMS = [dict(), dict(temperature=0.7), dict(temperature=0.0), dict(top_k=1), dict(top_k=5), dict(top_p=0.3), dict(top_p=0.9), dict(top_p=0.99),
          dict(min_p=0.1), dict(min_p=1.0), dict(temperature=1.4, top_k=7, top_p=0.8, min_p=0.05), dict(top_k=3, top_p=0.999), dict(temperature=20.0, top_p=0.5)]


@pytest.mark.parametrize("prm", PARAMS, ids=lambda p: "-".join(f"{k}{v}" for k, v in p.items()) or "plain")
@pytest.mark.parametrize("shape", [(3, 20, 17), (2, 25, 67), (2, 6, 300), (1, 3, 2500)], ids=lambda s: str(s[2]))
def test_sample_labels(shape, prm, gpu_device):
    run_sample(*shape, torch.float32, 31, **prm)
    run_sample(*shape, torch.bfloat16, 32, each=False, **prm)  # (bfloat16: many equal logits)


@pytest.mark.parametrize("dtype", TYPES, ids=ids)
@pytest.mark.parametrize("C", [1, 2, 3, 4, 5, 16, 31, 32, 33, 64, 65, 127, 128, 129, 511, 512, 513, 1023, 4097])
def test_sample_labels_widths(C, dtype, gpu_device):
    run_sample(2, 4, C, dtype, 40 + C, lengths=[4, 3], pitch=C + 3, temperature=0.9, top_k=max(1, C // 2), top_p=0.95, min_p=0.001)
    run_sample(2, 3, C, dtype, 41 + C, top_p=0.6)


@pytest.mark.parametrize("C", [17, 67, 400, 3001])
def test_sample_labels_ties_and_masks(C, gpu_device):
    even = lambda z: z.zero_()  # noqa: E731
    for prm in (dict(), dict(top_k=4), dict(top_p=0.5), dict(top_k=10, top_p=0.7), dict(min_p=1.0)):
        run_sample(2, 5, C, torch.float32, 51, prep=even, **prm)
        run_sample(2, 5, C, torch.float16, 52, prep=lambda z: z.mul_(0.5).round_(), **prm)

    def mask(z):
        z[:, 0] = -math.inf                       # nothing left
        z[:, 1, : C - 1] = -math.inf              # the last class alone
        z[:, 2, ::2] = -math.inf
        z[:, 3, 1::2] = float("nan")
        z[:, 4, 3] = math.inf                     # takes all
        z[:, 5, 2], z[:, 5, 5] = math.inf, math.inf
        z[:, 6] = torch.finfo(z.dtype).min        # even
        z[:, 7, : C // 2] = torch.finfo(z.dtype).min
        z[:, 8] = -0.0
        z[:, 8, ::3] = 0.0
        return z
    for prm in (dict(), dict(top_k=3), dict(top_p=0.8), dict(temperature=0.0), dict(temperature=1e-30), dict(min_p=0.2)):
        run_sample(2, 10, C, torch.float32, 53, prep=mask, **prm)


def test_sample_labels_long_ranges_of_logits(gpu_device):
    """values over many binades: the boundary of a prefix is found whatever their spread"""
    def spread(z):
        g = torch.Generator().manual_seed(7)
        e = torch.randint(-120, 120, z.shape, generator=g).double()
        return (torch.sign(z.cpu().double()) * torch.pow(2.0, e)).float().cuda()
    for C in (67, 300, 2500):
        for prm in (dict(top_k=40), dict(top_k=C - 1), dict(top_p=0.5), dict(temperature=1e20, top_p=0.9), dict(temperature=1e30, top_k=100, top_p=0.99)):
            run_sample(1, 4, C, torch.float32, 61, prep=spread, **prm)


@pytest.mark.parametrize("C", [67, 700])
def test_sample_labels_numbers_outside_the_range(C, gpu_device):
    z, zd = rows_of(1, 5, C, torch.float32, 71)
    u = torch.tensor([[0.0, -1.0, 1.0, 2.0, float("nan")]]).cuda()
    got = bfa.sample_labels(z, u, top_k=6)[0].cpu()[0].tolist()
    kept = [sorted(torch.topk(zd[0, i], 6).indices.tolist()) for i in range(5)]
    assert got == [kept[0][0], kept[1][0], kept[2][-1], kept[3][-1], kept[4][0]]


@pytest.mark.parametrize("C", [17, 67, 1500])
def test_sample_labels_follow_the_distribution(C, gpu_device):
    """every share of the kept probability gets its share of evenly spread numbers: exactly, up to one number a class"""
    z, zd = rows_of(1, 1, C, torch.float32, 81, scale=1.5)
    n = 4096
    u = (torch.arange(n).float() / n).reshape(1, n).cuda()
    got = bfa.sample_labels(z.expand(1, n, C), u, temperature=0.8, top_p=0.9)[0].cpu()[0]
    assert bool((got[1:] >= got[:-1]).all())  # in the order of the classes
    w = torch.exp((zd[0, 0] - zd.max()) / float(torch.tensor(0.8)))
    order = torch.argsort(-w, stable=True)
    before = torch.cumsum(w[order], 0) - w[order]
    kept = order[before < float(torch.tensor(0.9)) * w.sum()]
    share = torch.zeros(C).double()
    share[kept] = w[kept] / w[kept].sum()
    assert bool(((torch.bincount(got, minlength=C) - n * share).abs() <= 1.0).all())


# ---- together ----------------------------------------------------------------------------------------------------------------

def test_long_strides_pass_32_bits(gpu_device):
    """rows more than 2^31 elements apart (8 GiB of bytes in between are never touched)"""
    far = (1 << 31) + 12
    store = torch.empty(far + 1000, dtype=torch.float16, device="cuda")
    x = store.as_strided((2, 2, 300), (far, 400, 1))
    g = torch.Generator().manual_seed(91)
    xc = torch.randn((2, 2, 300), generator=g).half()
    x.copy_(xc)
    near = xc.cuda()
    labels = torch.tensor([[1, 2], [3, 299]], device="cuda")
    assert torch.equal(bfa.layer_norm(x), bfa.layer_norm(near))
    a, b = bfa.label_loss_and_grad(x, labels), bfa.label_loss_and_grad(near, labels)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    u = torch.rand(2, 2, generator=g).cuda()
    assert torch.equal(bfa.sample_labels(x, u, top_p=0.9)[0], bfa.sample_labels(near, u, top_p=0.9)[0])


def test_strides_and_orders(gpu_device):
    x, _ = rows_of(6, 10, 67, torch.float32, 92)
    labels = torch.randint(0, 67, (6, 10), device="cuda")
    u = torch.rand(6, 10, device="cuda")
    views = {"transposed": x.transpose(0, 1).contiguous().transpose(0, 1), "columns": x.transpose(1, 2).contiguous().transpose(1, 2),
             "shifted": torch.cat([x.new_zeros(3), x.reshape(-1)])[3:].reshape(6, 10, 67)}
    for name, v in views.items():
        assert torch.equal(bfa.layer_norm(v), bfa.layer_norm(x)), name
        assert torch.equal(bfa.label_loss_and_grad(v, labels)[1], bfa.label_loss_and_grad(x, labels)[1]), name
        assert torch.equal(bfa.sample_labels(v, u)[0], bfa.sample_labels(x, u)[0]), name
    one = x[:1, :1].expand(6, 10, 67)
    assert torch.equal(bfa.layer_norm(one), bfa.layer_norm(one.contiguous()))
    # a gradient that is broadcast, as that of a sum is
    xs = x.clone().requires_grad_()
    bfa.layer_norm(xs, torch.ones(67, device="cuda")).sum().backward()
    y, mean, rstd = bfa.layer_norm_forward(x, torch.ones(67, device="cuda"))
    assert torch.equal(xs.grad, bfa.layer_norm_backward(torch.ones_like(x), x, mean, rstd, torch.ones(67, device="cuda"))[0])


def test_same_bits_every_time_and_on_another_stream(gpu_device):
    x, _ = rows_of(40, 50, 768, torch.bfloat16, 93)
    w = torch.rand(768, device="cuda")
    g, _ = rows_of(40, 50, 768, torch.bfloat16, 94)
    labels = torch.randint(0, 768, (40, 50), device="cuda")
    u = torch.rand(40, 50, device="cuda")

    def all_of_it():
        y, mean, rstd = bfa.layer_norm_forward(x, w)
        return [y, *bfa.layer_norm_backward(g, x, mean, rstd, w), *bfa.label_loss_and_grad(x, labels), *bfa.sample_labels(x, u, top_p=0.9)]
    first = all_of_it()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = all_of_it()
    again = all_of_it()
    torch.cuda.synchronize()
    for a, b, c in zip(first, other, again):
        assert torch.equal(a, b) and torch.equal(a, c)


def test_a_captured_step_replays(gpu_device):
    """loss, gradient, normalisation and draw captured once and replayed on new inputs, with eager work in between"""
    B, T, D, C = 4, 30, 96, 67
    x, _ = rows_of(B, T, D, torch.float32, 95)
    x = x.clone()
    w, b = torch.rand(D, device="cuda"), torch.rand(D, device="cuda")
    proj = torch.randn(D, C, device="cuda")
    labels = torch.randint(0, C, (B, T), device="cuda", dtype=torch.int32)
    u = torch.rand(B, T, device="cuda")
    lengths = torch.tensor([30, 1, 0, 17], dtype=torch.int32, device="cuda")

    def step():
        y, mean, rstd = bfa.layer_norm_forward(x, w, b, lengths=lengths)
        z = (y.reshape(-1, D) @ proj).reshape(B, T, C)
        loss, dz = bfa.label_loss_and_grad(z, labels, lengths=lengths)
        dy = (dz.reshape(-1, C) @ proj.t().contiguous()).reshape(B, T, D)
        return [loss, *bfa.layer_norm_backward(dy, x, mean, rstd, w, lengths=lengths), *bfa.sample_labels(z, u, top_k=9, lengths=lengths)]
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step()
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for seed in range(4):
        x.copy_(rows_of(B, T, D, torch.float32, 100 + seed)[0])
        labels.copy_(torch.randint(-1, C, (B, T), device="cuda", dtype=torch.int32))
        lengths.copy_(torch.tensor([30 - seed, seed, 5 * seed, 17], dtype=torch.int32))
        u.uniform_()
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in out]
        for a, e in zip(got, step()):
            assert torch.equal(a, e)


def test_a_captured_backward_beside_an_eager_graph(gpu_device):
    """the functions without a graph of their own may be captured while an eager graph of the same leaf is alive"""
    x = torch.randn(8, 67, device="cuda", requires_grad=True)
    labels = torch.randint(0, 67, (8,), device="cuda")
    eager = bfa.label_loss(bfa.layer_norm(x), labels)  # stays alive
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y, mean, rstd = bfa.layer_norm_forward(x)
        loss, dz = bfa.label_loss_and_grad(y, labels)
        dx = bfa.layer_norm_backward(dz, x, mean, rstd, need=(True, False, False))[0]
    for _ in range(3):
        graph.replay()
    torch.cuda.synchronize()
    want, = torch.autograd.grad(eager, (x,))
    assert torch.equal(loss, eager.detach()) and torch.allclose(dx, want, atol=1e-6)


def test_training_a_head_on_its_alignments(gpu_device):
    """embeddings -> layer_norm -> projection -> logits; the alignment's frame labels -> loss -> gradients; labels drawn from the
    same logits.  The gradients of the whole are those of the same head in 64 bits."""
    import cases
    import numpy as np
    B, T, D, C = 3, 120, 80, 67
    lengths = [120, 77, 100]
    rng = np.random.default_rng(5)
    proj = torch.randn(D, C, generator=torch.Generator().manual_seed(6), dtype=torch.float32) / 4
    emb = torch.randn(B, T, D, generator=torch.Generator().manual_seed(7))
    toks = [rng.integers(1, 66, 8).astype(np.int32) for _ in range(B)]
    w, b = torch.rand(D) + 0.5, torch.rand(D)
    xs, ws, bs, ps = (t.cuda().requires_grad_() for t in (emb, w, b, proj))
    y = bfa.layer_norm(xs, ws, bs, lengths=lengths)
    z = (y.reshape(-1, D) @ ps).reshape(B, T, C)
    au = bfa.AlignmentUtils(blank_id=66, silence_id=0)
    res = au.decode_alignments_device(bfa.log_softmax(z.detach()), torch.from_numpy(np.stack(toks)), lengths, [8] * B)
    res.raise_for_status()
    labels = res.frame_phonemes.clone()
    assert labels.shape == (B, T)
    labels[torch.arange(T, device="cuda")[None] >= torch.tensor(lengths, device="cuda")[:, None]] = -1
    loss = bfa.label_loss(z, labels, lengths=lengths)
    got = torch.autograd.grad(loss, (xs, ws, bs, ps))
    held = held_of(B, T, lengths)
    dl = [t.double().requires_grad_() for t in (emb, w, b, proj)]
    zz = torch.nn.functional.layer_norm(dl[0], (D,), dl[1], dl[2], 1e-5) @ dl[3]
    ref = torch.nn.functional.cross_entropy(zz[held], labels.cpu()[held].long())
    want = torch.autograd.grad(ref, dl)
    assert abs(float(loss) - float(ref)) <= 1e-4
    for g, e in zip(got, want):
        assert float((g.cpu().double() - e).abs().max()) <= 1e-4 * float(e.abs().max()) + 1e-7
    drawn, logp = bfa.sample_labels(z.detach(), torch.rand(B, T, device="cuda"), top_p=0.9, lengths=lengths)
    assert bool((drawn.cpu()[~held] == -1).all()) and bool((drawn.cpu()[held] >= 0).all())
    # the drawn labels with their probabilities as weights are labels like any others
    again = bfa.label_loss(z.detach(), drawn, weights=logp.exp(), lengths=lengths)
    lp = torch.log_softmax(z.detach().cpu().double(), -1).gather(-1, drawn.cpu().clamp(min=0).long()[..., None])[..., 0]
    wt = torch.where(held, logp.cpu().double().exp(), 0.0)
    assert abs(float(again) + float((lp * wt).sum() / wt.sum())) <= 1e-4
    assert cases is not None


def test_refusals_on_the_device(gpu_device):
    x = torch.zeros(2, 3, 8, device="cuda")
    with pytest.raises(ValueError, match="labels is on|labels must"):
        bfa.label_loss(x, torch.zeros(3, 2, dtype=torch.int32, device="cuda"))
    with pytest.raises(RuntimeError, match="at most 524288"):
        bfa.sample_labels(torch.zeros(1, (1 << 19) + 1, device="cuda"), torch.zeros(1, device="cuda"))
    with pytest.raises(ValueError, match="2\\^31"):
        bfa.layer_norm(torch.zeros(1, 1, 1, device="cuda").expand(1 << 16, 1 << 15, 1))


@pytest.mark.parametrize("dtype", TYPES, ids=ids)
@pytest.mark.parametrize("prm", [dict(top_k=1), dict(top_k=50, top_p=0.9, temperature=0.8), dict(top_k=224), dict(top_k=225), dict(top_k=3000, top_p=0.7),
                                 dict(top_p=0.95, temperature=1.2), dict(top_p=0.05), dict(min_p=0.01), dict(temperature=40.0, top_p=0.5),
                                 dict(temperature=1e-3, top_p=0.9999), dict()],
                         ids=lambda p: "-".join(f"{k}{v}" for k, v in p.items()) or "plain")
def test_sample_labels_of_long_rows(prm, dtype, gpu_device):
    run_sample(1, 2, 40009, dtype, 101, pitch=40013, **prm)

    def lumps(z):  # thousands of equal values; most of the row masked
        z[:, 0] = torch.round(z[:, 0])
        z[:, 1, 50:] = -math.inf
        return z
    run_sample(1, 2, 9001, dtype, 102, prep=lumps, **prm)


@pytest.mark.parametrize("rows,C,dtype", [(9001, 600, torch.float32), (2100, 5000, torch.float16), (1100, 5000, torch.float32), (700, 33000, torch.bfloat16),
                                          (530, 70001, torch.bfloat16), (3, 140001, torch.bfloat16), (3, 70003, torch.float32)], ids=str)
def test_label_loss_workgroups_take_several_rows(rows, C, dtype, gpu_device):
    """more rows than workgroups, some of which do not count, so that rows are fetched ahead of their turn or not at all"""
    g = torch.Generator(device="cuda").manual_seed(C)
    z = torch.randn(1, rows, C, generator=g, device="cuda").to(dtype)
    labels = torch.randint(0, C, (1, rows), generator=g, device="cuda")
    labels[torch.rand(1, rows, generator=g, device="cuda") < 0.3] = -1
    weights = torch.rand(1, rows, generator=g, device="cuda")
    weights[0, ::7] = 0.0
    z[0, 5 if rows > 5 else 1] = float("nan")  # in a row that does not count
    labels[0, 5 if rows > 5 else 1] = -1
    n = rows - rows // 9
    loss, grad = bfa.label_loss_and_grad(z, labels, weights=weights, lengths=[n], reduction="sum")
    counts = (labels[0] >= 0) & (weights[0] > 0) & (torch.arange(rows, device="cuda") < n)
    total = 0.0
    for i in range(0, rows, 128):
        s = slice(i, min(rows, i + 128))
        zd = torch.where(counts[s, None], z[0, s].double(), 0.0)
        lp, w = torch.log_softmax(zd, -1), torch.where(counts[s], weights[0, s].double(), 0.0)
        at = labels[0, s].clamp(min=0)
        total -= float((lp.gather(-1, at[:, None])[:, 0] * w).sum())
        want = lp.exp()
        want[torch.arange(want.shape[0], device="cuda"), at] -= 1.0
        want *= w[:, None]
        # a step of the type, and the exponent's roundings (|z| <= 6: at most 12 + 4 of them)
        tol = half_step(dtype) * want.abs() + 32 * E * w[:, None] * (lp.exp() + (want < 0)) + 1e-30
        if dtype == torch.float16:
            tol = tol + 2.0 ** -25
        assert bool(((grad[0, s].double() - want).abs() <= tol).all()), i
    assert abs(float(loss) - total) <= 32 * E * abs(total) + E * rows


def test_sample_labels_of_more_rows_than_workgroups(gpu_device):
    g = torch.Generator(device="cuda").manual_seed(7)
    for rows, C, cut in ((1500, 520, 1000), (600001, 5, 300000), (40000, 400, 30000)):
        z, u = torch.randn(rows, C, generator=g, device="cuda"), torch.rand(rows, generator=g, device="cuda")
        for prm in (dict(top_p=0.8), dict(top_k=3, temperature=0.7)):
            got = bfa.sample_labels(z, u, **prm)
            parts = [bfa.sample_labels(z[s], u[s], **prm) for s in (slice(0, cut), slice(cut, rows))]
            assert torch.equal(got[0], torch.cat([p[0] for p in parts])) and torch.equal(got[1], torch.cat([p[1] for p in parts]))


@pytest.mark.parametrize("C", [17, 67, 200, 500])
def test_sample_labels_near_the_borders(C, gpu_device):
    """numbers within a few steps of float32 of the borders between classes, and prefixes that end within them: the label is the
    one float64 gives"""
    z, zd = rows_of(1, 1, C, torch.float32, 111)
    for top_p in (1.0, 0.9):
        w = torch.exp(zd[0, 0] - zd.max())
        order = torch.argsort(-w, stable=True)
        front = torch.cumsum(w[order], 0) - w[order]
        kept = torch.zeros(C, dtype=torch.bool)
        kept[order[(front < float(torch.tensor(top_p)) * w.sum()) | (top_p == 1.0)]] = True
        wk = torch.where(kept, w, 0.0)
        borders = (torch.cumsum(wk, 0) / wk.sum()).float()
        u = torch.cat([(borders.double() * (1 + k * 2.0 ** -24)).float() for k in (-40, -3, -1, 0, 1, 3, 40)]).clamp(0, 1 - 2.0 ** -24)
        got = bfa.sample_labels(z.expand(1, len(u), C), u[None].cuda(), top_p=top_p)[0].cpu()[0]
        run = torch.cumsum(wk, 0)
        goal = u.double() * wk.sum()
        want = (run[None] <= goal[:, None]).sum(1)
        clear = ((run[None] - goal[:, None]).abs() > 1e-12 * C).all(1)  # (closer than the order of a float64 sum tells apart)
        assert bool(clear.any()) and torch.equal(got[clear], want.int()[clear])


def test_rows_of_more_elements_than_indexes_reach_are_refused(gpu_device):
    x = torch.zeros(1, 1, 1, device="cuda").expand(1, 1, (1 << 30) + 1)
    for call in (lambda: bfa.layer_norm(x), lambda: bfa.label_loss(x, torch.zeros(1, 1, dtype=torch.int32, device="cuda")),
                 lambda: bfa.sample_labels(x, torch.zeros(1, 1, device="cuda"))):
        with pytest.raises(ValueError, match="2\\^30"):
            call()


@pytest.mark.parametrize("prm", [dict(), dict(top_k=50), dict(top_p=0.9), dict(top_k=100000, top_p=0.5)], ids=str)
def test_sample_labels_of_the_longest_rows(prm, gpu_device):
    C = 1 << 19
    run_sample(1, 1, C, torch.float32, 121, **prm)
    run_sample(1, 1, C, torch.bfloat16, 122, prep=lambda z: z.zero_(), **prm)
