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
