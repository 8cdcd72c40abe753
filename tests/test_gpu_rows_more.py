"""layer_norm, label_loss and sample_labels on the GPU at the sizes and values that the loops over rows, far means and near borders need,
against plain implementations in 64 bits.

Tolerances count roundings: E = 2^-24 is half a step of float32 relative to a value."""
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


# ---- layer_norm: means that are large against the spread ---------------------------------------------------------------------

@pytest.mark.parametrize("dtype", TYPES, ids=ids)
@pytest.mark.parametrize("value", [1.0, 7.0, 1000.0])
@pytest.mark.parametrize("C", [3, 41, 55, 130, 1001, 5000, 16400])
def test_constant_rows_come_out_as_the_bias(C, value, dtype):
    """the sum C * value is a whole number below 2^24: mean and deviations are exact, y is the bias"""
    x = torch.full((5, C), value, dtype=dtype, device="cuda")
    w = torch.full((C,), 3.0, dtype=dtype, device="cuda")
    b = torch.linspace(-2, 2, C).to(dtype).cuda()
    y, mean, rstd = bfa.layer_norm_forward(x, w, b, eps=1e-5)
    assert torch.equal(y, b.expand(5, C))
    assert torch.equal(mean, torch.full((5,), value, device="cuda"))
    assert float((rstd.double() * math.sqrt(float(torch.tensor(1e-5))) - 1).abs().max()) <= 4 * E  # (sum, root, quotient)


@pytest.mark.parametrize("C", [48, 768, 1001, 4097, 16400])
@pytest.mark.parametrize("mean", [1000.0, -30000.0])
def test_far_means(C, mean):
    """Deviations x - m are exact where x and m are within a factor of two.  Their sum and the sum of their squares take at most 16 additions
    in a thread, 6 in a wave, 15 between waves and (rows beyond 16384) 17 more in a thread: 54 E of the magnitudes; shift: 56 E of
    the spread, rstd: half of 58 E, root and quotient, y: three more.  So |dy| <= (64 E + 40 E |xh|) |w| + E |y|."""
    g = torch.Generator().manual_seed(C)
    x = (torch.randn(37, C, generator=g) + mean).cuda()
    w, b = (1 + 0.1 * torch.randn(C, generator=g)), torch.randn(C, generator=g)
    y = bfa.layer_norm(x, w.cuda(), b.cuda(), eps=1e-5).cpu().double()
    d = x.cpu().double()
    d = d - d.mean(1, keepdim=True)
    xh = d / torch.sqrt((d * d).mean(1, keepdim=True) + float(torch.tensor(1e-5)))
    ref = xh * w.double() + b.double()
    assert ((y - ref).abs() <= (64 * E + 40 * E * xh.abs()) * w.double().abs() + E * ref.abs()).all()


def test_rows_with_infinities_and_nan_have_no_statistics():
    x = torch.randn(6, 300, device="cuda")
    x[1, 7], x[2, 8], x[3, 9] = math.inf, -math.inf, math.nan
    y, mean, rstd = bfa.layer_norm_forward(x)
    bad = torch.tensor([False, True, True, True, False, False], device="cuda")
    assert torch.isnan(y[bad]).all() and torch.isnan(rstd[bad]).all() and not torch.isfinite(mean[bad]).any()
    assert torch.isfinite(y[~bad]).all() and torch.isfinite(rstd[~bad]).all()


# ---- sample_labels: many borders close together ------------------------------------------------------------------------------

def drawn_in_order(z, u, p):
    """labels of rows [R, C] by the definition in 64 bits (temperature 1), and the nearest that any comparison came to a tie, relative
    to the mass"""
    R, C = z.shape
    v, order = torch.sort(z, dim=1, descending=True, stable=True)
    w = torch.exp(v - v[:, :1])
    run = w.cumsum(1)
    front, target = run - w, p * run[:, -1:]
    keep = front < target
    keep[:, 0] = True
    near = ((front - target).abs() / run[:, -1:]).min(1).values
    kept = torch.zeros_like(w).scatter_(1, order, w * keep)
    mass = kept.cumsum(1)
    goal = u[:, None] * mass[:, -1:]
    label = (mass > goal).int().argmax(1)
    near = torch.minimum(near, ((mass - goal).abs() / mass[:, -1:]).min(1).values)
    return label.int(), near


@pytest.mark.parametrize("C", [5, 20, 67, 80, 81, 250, 320, 321, 512])
@pytest.mark.parametrize("step", [1e-6, 1e-4, 1e-2, 1.0])
def test_classes_a_hair_apart(C, step):
    """Logits `step` apart in shuffled order: the halvings of the range of values leave up to all classes to walk past one by one, and
    neighbouring borders are 1 / C of the mass apart.  Labels are whole numbers: equal wherever 64 bits decide (2^-40 of the mass)."""
    g = torch.Generator().manual_seed(C)
    R = 3000
    z = torch.stack([torch.randperm(C, generator=g) for _ in range(R)]).float() * step
    u, p = torch.rand(R, generator=g), torch.rand(R, generator=g) * 0.998 + 0.001
    want, near = drawn_in_order(z.double(), u.double(), p.double()[:, None])
    got, logp = bfa.sample_labels(z.reshape(R, 1, C).cuda(), u.reshape(R, 1).cuda(), top_p=p.cuda())
    sure = near > 2.0 ** -40
    assert sure.float().mean() > 0.99
    assert torch.equal(got[:, 0].cpu()[sure], want[sure])


def test_numbers_at_the_borders():
    """numbers a few steps of float32 on either side of every border between the classes of a row, even and uneven"""
    for C in (17, 67, 80, 300, 512):
        g = torch.Generator().manual_seed(C + 1)
        row = torch.randn(C, generator=g) * 2
        for z in (row, torch.zeros(C)):
            w = torch.exp(z.double() - z.double().max())
            edge = (w.cumsum(0) / w.sum())[:-1].float()
            u = torch.cat([edge] + [torch.nextafter(edge, torch.full_like(edge, s)) for s in (0.0, 1.0)]).clamp(0, 1 - 2.0 ** -24)
            rows_in = z.expand(u.numel(), C).contiguous()
            want, near = drawn_in_order(rows_in.double(), u.double(), torch.full((u.numel(), 1), 2.0, dtype=torch.float64))
            got = bfa.sample_labels(rows_in.reshape(-1, 1, C).cuda(), u.reshape(-1, 1).cuda())[0][:, 0].cpu()
            sure = near > 2.0 ** -40
            assert torch.equal(got[sure], want[sure])


# ---- more rows than the workgroups of a launch take at a time ----------------------------------------------------------------

def ragged(B, T, seed):
    """lengths, and which rows they hold"""
    lengths = torch.randint(T // 2, T + 1, (B,), generator=torch.Generator().manual_seed(seed), dtype=torch.int32)
    lengths[0] = T
    return lengths.cuda(), (torch.arange(T)[None] < lengths[:, None]).cuda()


def rows_64(B, T, C, dtype, seed, scale=1.0, shift=0.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = (torch.randn(B, T, C, generator=g, device="cuda") * scale + shift).to(dtype)
    return x, x.double()


# rows of 16, 64, 256 and 1024 threads, 16 / 4 / 1 / 1 rows to a workgroup of up to 2048 (backward 1024; 512 of 1024 threads), and swept
# rows of up to 512 workgroups, 64 of column sums
NORM_MANY = [(8, 5000, 33), (4, 2500, 300), (3, 900, 1100), (2, 320, 4200), (2, 300, 16400)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=ids)
@pytest.mark.parametrize("shape", NORM_MANY, ids=lambda s: "x".join(map(str, s)))
def test_layer_norm_of_many_rows(shape, dtype):
    """Statistics as in test_far_means; the backward pass takes mean and rstd as float32.  Sums over rows: rows / 512 in a thread at
    most, 16 in a workgroup, then 64 + 16 of partial sums."""
    B, T, C = shape
    lengths, held = ragged(B, T, 5)
    x, xd = rows_64(B, T, C, dtype, 1, 1.5, 0.5)
    gy, gd = rows_64(B, T, C, dtype, 2)
    w = (1 + 0.2 * torch.randn(C, generator=torch.Generator().manual_seed(3))).to(dtype).cuda().requires_grad_()
    b = (0.2 * torch.randn(C, generator=torch.Generator().manual_seed(4))).to(dtype).cuda().requires_grad_()
    x.requires_grad_()
    y = bfa.layer_norm(x, w, b, lengths=lengths)
    dx, dw, db = torch.autograd.grad(y, (x, w, b), gy)
    h, wd, bd, rows_held = half_step(dtype), w.detach().double(), b.detach().double(), held[..., None]
    mean = xd.mean(-1, keepdim=True)
    r = 1 / torch.sqrt(((xd - mean) ** 2).mean(-1, keepdim=True) + float(torch.tensor(1e-5)))
    xh = (xd - mean) * r
    want = (xh * wd + bd) * rows_held
    tol = (64 * E + 40 * E * xh.abs()) * wd.abs() + (h + E) * want.abs()
    assert ((y.detach().double() - want).abs() <= tol).all() and (y.detach()[~held] == 0).all()
    off = E * (mean * r).abs() + 30 * E * xh.abs() + E * (1 + xh.abs())  # of xh: the mean's rounding, rstd, two operations
    g = gd * wd
    g1, g2 = g.abs().mean(-1, keepdim=True), (g * xh).abs().mean(-1, keepdim=True)
    want = r * (g - g.mean(-1, keepdim=True) - xh * (g * xh).mean(-1, keepdim=True)) * rows_held
    far = off.amax(-1, keepdim=True)
    tol = (h + 32 * E) * want.abs() + r * (4 * E * g.abs() + 60 * E * g1 + (60 * E * g2 + g1 * far) * xh.abs() + off * g2 + 4 * E * xh.abs() * g2)
    assert ((dx.double() - want).abs() <= tol * rows_held + 1e-30).all() and (dx[~held] == 0).all()
    depth = E * (B * T / 512 + 128)
    gh = gd.abs() * rows_held
    want = (gd * xh * rows_held).sum((0, 1))
    assert ((dw.double() - want).abs() <= h * want.abs() + (gh * (depth * xh.abs() + off)).sum((0, 1))).all()
    want = (gd * rows_held).sum((0, 1))
    assert ((db.double() - want).abs() <= h * want.abs() + depth * gh.sum((0, 1))).all()


# rows of 4, 16 and 64 lanes (64 / 16 / 4 to each of 2048 workgroups), then of 64, 256 and 1024 threads (4 / 1 / 1 to 2048 / 2048 / 512);
# the last: more rows than 256 workgroups add weights of at a time
LOSS_MANY = [(8, 17000, 17), (5, 7000, 67), (3, 3000, 300), (3, 3000, 600), (3, 800, 1100), (2, 300, 4200), (16, 66000, 2)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16], ids=ids)
@pytest.mark.parametrize("shape", LOSS_MANY, ids=lambda s: "x".join(map(str, s)))
def test_label_loss_of_many_rows(shape, dtype):
    """A row's exponentials are off by a few E, their sum by log2(C) + 16 additions more, its logarithm and the differences by E of their
    magnitudes; the sums over rows are float64."""
    B, T, C = shape
    lengths, held = ragged(B, T, 6)
    z, zd = rows_64(B, T, C, dtype, 7, 2.0)
    g = torch.Generator(device="cuda").manual_seed(8)
    labels = torch.randint(-1, C, (B, T), generator=g, device="cuda", dtype=torch.int32)
    weights = torch.rand(B, T, generator=g, device="cuda")
    counts = held & (labels >= 0)
    wt = weights.double() * counts
    p = torch.softmax(zd, -1)
    at = labels.clamp(min=0).long()[..., None]
    nll = (torch.logsumexp(zd, -1) - zd.gather(-1, at)[..., 0]) * wt
    loss, grad = bfa.label_loss_and_grad(z, labels, weights=weights, lengths=lengths)
    deep = math.log2(C) + 32
    mag = zd.abs().amax(-1) + math.log(C) + 1
    total = wt.sum()
    want = nll.sum() / total
    assert abs(float(loss) - float(want)) <= float(E * (deep * mag * wt).sum() / total) + 4 * E * float(want)
    one = torch.zeros_like(p).scatter_(-1, at, 1.0)
    want = (p - one) * (wt / total)[..., None]
    tol = half_step(dtype) * want.abs() + E * (wt / total)[..., None] * (p * (deep + 4 * mag[..., None]) + 4)
    tol = tol + (2.0 ** -25 if dtype == torch.float16 else 1e-38)  # (half of float16's smallest step)
    assert ((grad.double() - want).abs() <= tol).all() and (grad[~counts] == 0).all()
    each = bfa.label_loss(z, labels, weights=weights, lengths=lengths, reduction="none")
    assert ((each.double() - nll).abs() <= E * deep * mag * wt).all()


# rows of 4, 16 and 64 lanes (64 / 16 / 4 to each of 8192 workgroups), and a workgroup of 1024 to each of them
@pytest.mark.parametrize("shape", [(8, 70000, 17), (4, 34000, 100), (3, 11500, 400), (2, 600, 600)], ids=lambda s: "x".join(map(str, s)))
def test_sample_labels_of_many_rows(shape):
    B, T, C = shape
    lengths, held = ragged(B, T, 9)
    z, zd = rows_64(B, T, C, torch.float32, 10, 2.0)
    g = torch.Generator(device="cuda").manual_seed(11)
    u = torch.rand(B, T, generator=g, device="cuda")
    p = torch.rand(B, generator=g, device="cuda") * 0.9 + 0.05
    got, logp = bfa.sample_labels(z, u, top_p=p, lengths=lengths)
    want, near = drawn_in_order(zd.reshape(-1, C), u.reshape(-1).double(), p.double()[:, None].expand(B, T).reshape(-1, 1))
    sure = held & (near.reshape(B, T) > 2.0 ** -40)
    assert float(sure.sum() / held.sum()) > 0.999
    assert torch.equal(got[sure], want.reshape(B, T)[sure])
    assert (got[~held] == -1).all() and (logp[~held] == 0).all()
