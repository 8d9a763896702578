"""The distillation loss where the entries a teacher lists lie far above all others, and at the ends of the range of
logits and temperatures: losses and gradients element by element against the definition in 64 bits."""
import math

import pytest
import torch

from test_gpu_distill import DEV, DTYPES, _ps, make

pytestmark = pytest.mark.gpu


def definition(z, idx, teacher, tau, tail):
    """Row losses (before weight) and their gradients, in 64 bits.  Logarithms of sums are taken of differences from the
    largest logit: next to logits of 3e38, where numbers of 64 bits are 2^75 apart, they would be lost."""
    z, teacher, idx = z.double().cpu(), teacher.double().cpu(), idx.cpu().long()
    losses, grads = [], []
    for zr, ir, tr in zip(z / tau, idx, teacher):
        outside = torch.ones_like(zr, dtype=torch.bool)
        outside[ir] = False
        log_sum = (zr - zr.max()).exp().sum().log()
        logq = zr - zr.max() - log_sum
        logp = tr if tail == "bucket" else torch.log_softmax(tr / tau, 0)
        p = logp.exp()
        rest = max(0.0, 1.0 - float(p.sum())) if tail == "bucket" and outside.any() else 0.0
        loss = torch.where(p > 0, p * (logp - logq[ir]), 0.0).sum()
        grad = (float(p.sum()) + rest) * logq.exp()
        grad.index_add_(0, ir, -p)
        if rest > 0:
            others = zr[outside]
            e = (others - others.max()).exp()
            log_rest = others.max() - zr.max() + (e.sum().log() - log_sum)
            loss = loss + rest * (math.log(rest) - log_rest)
            grad[outside] -= rest * e / e.sum()
        losses.append(loss * tau * tau)
        grads.append(grad * tau)
    return torch.stack(losses), torch.stack(grads)


def bounds(z, tau, want, wgrad, factor, dt):
    """How far the row losses and the gradient of `factor` times their sum may be off.

    Sums of powers of two in 32 bits are off by d, relative: the power itself 2^-22, its argument four roundings of at
    most 126 (log2(e) / T, which is rounded, and the operation's own, twice where a sum is brought to another origin),
    smaller terms vanish; then the additions.  A log-probability is off by d of each of the two sums it is made of and,
    through log2(e) / T, by 2^-24 of the gap between the largest logit and its own; the loss weighs these with
    probabilities that sum up to 1, and is rounded once.  The gradient's two terms are off by 2 d (the element's power
    and its sum's; the unlisted mass counts twice more in the first), and what is below 2^-126 of the largest vanishes."""
    z = z.double().cpu()
    fine = torch.where(torch.isfinite(z), z, z[torch.isfinite(z)].max())
    gap = (fine.amax(1) - fine.amin(1)) / tau
    a = (gap * 1.4427).clamp(max=126).max()
    d = 2.0 ** -22 + 4 * 2.0 ** -24 * float(a) * 0.6931 + (z.shape[1] / 512 + 64) * 2.0 ** -24
    loss = tau * tau * (4 * d + 2.0 ** -23 * gap) + 2.0 ** -23 * want.abs()
    size = torch.log_softmax(z / tau, 1).exp() * factor * tau
    grad = 4 * d * (size + (wgrad - size).abs()) + torch.finfo(dt).eps / 2 * wgrad.abs() + \
        2.0 ** -125 * factor * tau + torch.finfo(dt).smallest_normal * torch.finfo(dt).eps
    return loss, grad


def check(z, idx, teacher, tau, tail, got, grad, factor):
    want, wgrad = definition(z, idx, teacher, tau, tail)
    wgrad = wgrad * factor
    dt = grad.dtype
    loss_bound, grad_bound = bounds(z, tau, want, wgrad, factor, dt)
    assert torch.isfinite(got).all() and ((got.double().cpu() - want).abs() <= loss_bound).all()
    grad = grad.double().cpu()
    # beyond the type's largest value a gradient is infinite; next to it either way
    top = torch.finfo(dt).max
    over, under = wgrad.abs() - grad_bound > top, wgrad.abs() + grad_bound < top
    assert torch.equal(grad[over], torch.sign(wgrad[over]) * float("inf"))
    assert torch.isfinite(grad[under]).all()
    assert ((grad - wgrad).abs() <= grad_bound)[under].all()


def both(z, idx, teacher, tau, tail, scale):
    """The gradient of the backward call and the one of the forward call, at `scale`."""
    ps = _ps()
    z = z.detach().clone().requires_grad_(True)
    rows = ps.distillation_loss(z, idx, teacher, temperature=tau, tail=tail, reduction="none")
    check(z.detach(), idx, teacher, tau, tail, rows.detach(),
          torch.autograd.grad(rows, z, torch.full_like(rows, scale))[0], scale)
    scaler = ps.LossScaler(scale)
    total = ps.distillation_loss(z, idx, teacher, temperature=tau, tail=tail, reduction="sum", scaler=scaler)
    check(z.detach(), idx, teacher, tau, tail, rows.detach(),
          torch.autograd.grad(scaler.scale_loss(total), z)[0], scale)


@pytest.mark.parametrize("scale", [1.0, 2.0 ** 32])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("gap", [50.0, 80.0, 90.0, 1000.0])
@pytest.mark.parametrize("vocab,tau", [(300, 1.0), (5003, 2.0), (50257, 0.5)])
def test_listed_entries_far_above_the_others(vocab, tau, gap, dtype, scale):
    """The student is sure of listed entries; the rest that the teacher leaves is compared with what is hardly there."""
    z, idx, teacher = make(5, vocab, 6, torch.float32, int(gap) + vocab, "bucket")
    teacher = teacher - 0.5     # leaves a rest in every row
    top = z.amax(1)
    for r in range(4):
        z[r, idx[r, r]] = top[r] + gap * tau
    z[3, idx[3, 5]] = z[3, idx[3, 3]]    # two of them
    z[4, :] = z[4, :] - top[4]           # and a row whose unlisted elements are far above the listed ones
    z[4, idx[4]] = -gap * tau
    both(z.to(dtype), idx, teacher, tau, "bucket", scale)


@pytest.mark.parametrize("dtype", DTYPES)
def test_the_elements_outside_of_the_entries_are_masked(dtype):
    """With the type's lowest value, they are still where the rest goes; an odd number of leading elements."""
    z, idx, teacher = make(4, 1001, 5, dtype, 3, "bucket")
    low = torch.finfo(dtype).min
    listed = torch.zeros_like(z, dtype=torch.bool).scatter_(1, idx, True)
    z = torch.where(listed, z, low)
    both(z, idx, teacher - 0.25, 1.0, "bucket", 16.0)
    big = torch.full((4, 1004), 7.0, dtype=dtype, device=DEV)
    big[:, 3:] = z
    both(big[:, 3:], idx, teacher - 0.25, 1.0, "bucket", 16.0)


@pytest.mark.parametrize("tail", ["drop", "bucket"])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("tau", [2.0 ** -15, 2.0 ** -4, 2.0 ** 12])
def test_extreme_logits_and_temperatures_element_by_element(dtype, tail, tau):
    """Whole numbers as logits, small ones and such near the end of the type: differences are exact, and at the small
    temperature nothing but the largest (or two of them, when equal) is left of a row."""
    gen = torch.Generator().manual_seed(31)
    z = torch.stack([torch.randint(-100, 101, (700,), generator=gen) for _ in range(6)]).float()
    _, idx, teacher = make(6, 700, 5, torch.float32, 32, "bucket")
    if dtype == torch.float16:
        z[2:4] *= 512.0
    else:
        z[2:4] *= 2.0 ** 100
    idx = idx.cpu()
    for r in (0, 2, 4):                  # the largest is listed, and in one row its equal is not
        z[r, idx[r, 1]] = z[r].abs().max() * 1.25
    z[4, 699 if 699 not in idx[4] else 698] = z[4, idx[4, 1]]
    both(z.to(dtype).to(DEV), idx.to(DEV), teacher - 0.5, tau, tail, 1.0)
