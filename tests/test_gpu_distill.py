"""The distillation loss and its gradient against the definition in 64 bits."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
DTYPES = [torch.float16, torch.bfloat16, torch.float32]


def _ps():
    import patrickstar_b200
    return patrickstar_b200


def definition(z, idx, teacher, tau, tail):
    """Row losses (before weight) and their gradients with respect to z, in 64 bits, row by row."""
    z, teacher = z.double().cpu(), teacher.double().cpu()
    idx = idx.cpu().long()
    losses, grads = [], []
    for zr, ir, tr in zip(z, idx, teacher):
        listed = ir >= 0
        ir, tr = ir[listed], tr[listed]
        logq = torch.log_softmax(zr / tau, 0)
        q = logq.exp()
        outside = torch.ones_like(zr, dtype=torch.bool)
        outside[ir] = False
        if tail == "bucket":
            logp, p = tr, tr.exp()
            rest = max(0.0, 1.0 - float(p.sum())) if outside.any() else 0.0
        else:
            logp = torch.log_softmax(tr / tau, 0)
            p, rest = logp.exp(), 0.0
        loss = torch.where(p > 0, p * (logp - logq[ir]), p * 0).sum() if len(ir) else torch.zeros((), dtype=torch.float64)
        grad = (float(p.sum()) + rest) * q
        grad.index_add_(0, ir, -p)
        if rest > 0:
            log_rest = torch.logsumexp(logq[outside], 0)
            loss = loss + rest * (math.log(rest) - log_rest)
            grad = grad - torch.where(outside, rest * (logq - log_rest).exp(), 0.0)
        losses.append(loss * tau * tau)
        grads.append(grad * tau)
    return torch.stack(losses), torch.stack(grads)


def exponential_error(z, tau):
    """Relative error of a sum of 2^((z - M) c) in 32 bits: the power 2^-22, its argument three roundings
    of at most 126 (smaller terms vanish), the sum a chain of vocab / 512 terms and a tree."""
    z = z.double().cpu()
    fine = torch.where(torch.isfinite(z), z, z[torch.isfinite(z)].max())
    a = ((fine.amax(1) - fine.amin(1)) / tau * 1.4427).clamp(max=126).max()
    return 2.0 ** -22 + 3 * 2.0 ** -24 * float(a) * 0.6931 + (z.shape[1] / 512 + 64) * 2.0 ** -24


def check(z, idx, teacher, tau, tail, got, grad, factor):
    """`got`: row losses; `grad`: gradient of factor * sum of them."""
    want, wgrad = definition(z, idx, teacher, tau, tail)
    d = exponential_error(z, tau)
    # log Z and log of the outside sum are each off by d; the loss weighs them with at most sum p + p_r, 1 or so
    assert ((got.double().cpu() - want).abs() <= 4 * d * tau * tau + 2.0 ** -22 * want.abs()).all()
    dt = grad.dtype
    wgrad = wgrad * factor
    logq = torch.log_softmax(z.double().cpu() / tau, 1)
    # every term carries its exponential's error and the sum's: 4 d of q_v and of p_r q_v / q_r (of which their
    # difference is made; the second is at most q_v / q_r); listed probabilities are rounded to 32 bits
    size = logq.exp() * factor * tau
    tail_size = (wgrad - size).abs()
    bound = 4 * d * (size.abs() + tail_size) + torch.finfo(dt).eps / 2 * wgrad.abs() + \
        (torch.finfo(dt).smallest_normal * torch.finfo(dt).eps)
    assert grad.shape == z.shape
    assert ((grad.double().cpu() - wgrad).abs() <= bound).all()


def make(rows, vocab, k, dtype, seed, tail, idx_dtype=torch.int64):
    gen = torch.Generator().manual_seed(seed)
    z = torch.randn(rows, vocab, generator=gen) * 3
    idx = torch.stack([torch.randperm(vocab, generator=gen)[:k] for _ in range(rows)]).to(idx_dtype) if rows else \
        torch.zeros(0, k, dtype=idx_dtype)
    teacher = torch.randn(rows, k, generator=gen) * 2
    if tail == "bucket":
        teacher = torch.log_softmax(torch.cat([teacher, torch.randn(rows, 1, generator=gen)], 1), 1)[:, :k]
    return z.to(dtype).to(DEV), idx.to(DEV), teacher.to(DEV)


@pytest.mark.parametrize("tail", ["drop", "bucket"])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,vocab,k,tau", [(1, 1, 1, 1.0), (3, 5, 5, 2.0), (2, 7, 3, 0.5), (5, 511, 8, 1.0),
                                              (4, 4097, 33, 1.5), (3, 50257, 64, 2.0), (2, 131073, 100, 1.0),
                                              (700, 130, 4, 1.0), (1, 2000, 1024, 1.0)])
def test_rows_and_gradients(rows, vocab, k, tau, dtype, tail):
    ps = _ps()
    z, idx, teacher = make(rows, vocab, k, dtype, rows + vocab, tail, torch.int32 if rows % 2 else torch.int64)
    z.requires_grad_(True)
    loss = ps.distillation_loss(z, idx, teacher, temperature=tau, tail=tail, reduction="none")
    g = torch.autograd.grad(loss, z, torch.full_like(loss, 64.0))[0]
    check(z.detach(), idx, teacher, tau, tail, loss.detach(), g, 64.0)


@pytest.mark.parametrize("tail", ["drop", "bucket"])
def test_reductions_mask_weight_and_leading_dimensions(tail):
    ps = _ps()
    z, idx, teacher = make(24, 1003, 6, torch.float32, 1, tail)
    rows = ps.distillation_loss(z, idx, teacher, tail=tail, reduction="none").double()
    z4, i4, t4 = z.view(2, 3, 4, -1), idx.view(2, 3, 4, -1), teacher.view(2, 3, 4, -1)
    assert torch.equal(ps.distillation_loss(z4, i4, t4, tail=tail, reduction="none").double(), rows.view(2, 3, 4))
    mask = torch.arange(24, device=DEV).view(2, 3, 4) % 3 != 1
    kept = rows[mask.view(-1)]
    for m in (mask, mask.to(torch.uint8)):
        # sums of 24 in 64 bits, then a factor and one rounding to 32: two steps at most
        for reduction, want in (("sum", kept.sum()), ("mean", kept.mean())):
            got = ps.distillation_loss(z4, i4, t4, tail=tail, mask=m, reduction=reduction, weight=0.25)
            assert abs(float(got) - 0.25 * float(want)) <= 2.0 ** -22 * abs(float(want))
    none = torch.zeros(2, 3, 4, dtype=torch.bool, device=DEV)
    z4 = z4.clone().requires_grad_(True)
    for reduction in ("sum", "mean"):
        loss = ps.distillation_loss(z4, i4, t4, tail=tail, mask=none, reduction=reduction)
        assert float(loss.detach()) == 0.0 and not torch.autograd.grad(loss, z4)[0].any()


@pytest.mark.parametrize("tail", ["drop", "bucket"])
@pytest.mark.parametrize("dtype", DTYPES)
def test_masked_rows_are_not_read(dtype, tail):
    ps = _ps()
    z, idx, teacher = make(9, 777, 5, dtype, 2, tail)
    mask = torch.arange(9, device=DEV) % 2 == 0
    clean = z.clone().requires_grad_(True)
    want = ps.distillation_loss(clean, idx, teacher, tail=tail, mask=mask)
    wg = torch.autograd.grad(want, clean)[0]
    z[1], z[3, 5], z[5] = float("nan"), float("inf"), -float("inf")
    teacher[3], teacher[7], idx[7] = float("nan"), float("inf"), 10 ** 6
    z.requires_grad_(True)
    got = ps.distillation_loss(z, idx, teacher, tail=tail, mask=mask)
    assert torch.equal(got, want) and torch.equal(torch.autograd.grad(got, z)[0], wg)
    assert not wg[1::2].any()


@pytest.mark.parametrize("dtype", DTYPES)
def test_masked_logits(dtype):
    """Minus infinity and the type's lowest value among the logits; a row of nothing but the lowest is uniform."""
    ps = _ps()
    low = torch.finfo(dtype).min
    for tail in ("drop", "bucket"):
        z, idx, teacher = make(4, 900, 4, dtype, 3, tail)
        idx[:, :] = torch.tensor([1, 899, 450, 7], device=DEV)
        z[0, 100:200], z[1, 100:200], z[2] = -float("inf"), low, low
        z[3, :], z[3, 7:12] = -float("inf"), 1.0
        teacher[3, :3] = -float("inf")     # only entry 7 counts in this row
        z.requires_grad_(True)
        loss = ps.distillation_loss(z, idx, teacher, tail=tail, reduction="none")
        g = torch.autograd.grad(loss.sum(), z)[0]
        check(z.detach(), idx, teacher, 1.0, tail, loss.detach(), g, 1.0)


def test_entries_that_list_nothing_or_twice():
    ps = _ps()
    for tail in ("drop", "bucket"):
        z, idx, teacher = make(6, 333, 6, torch.float32, 4, tail)
        teacher = teacher - 1.0
        idx[0, 2:] = -1                 # two entries
        idx[1] = -1                     # none
        idx[2] = idx[2, 0]              # the same six times
        idx[3, 1::2] = idx[3, ::2]      # pairs
        idx[4, 5] = 332                 # the last index
        idx[4, 4] = 0
        if tail == "bucket":
            teacher[5] = math.log(0.25)  # six quarters: more than 1, no rest
        z.requires_grad_(True)
        loss = ps.distillation_loss(z, idx, teacher, tail=tail, reduction="none")
        g = torch.autograd.grad(loss.sum(), z)[0]
        check(z.detach(), idx, teacher, 1.0, tail, loss.detach(), g, 1.0)
        assert float(loss[1].detach()) == 0.0


@pytest.mark.parametrize("bad", [333, -2, 2 ** 40, -2 ** 40])
def test_an_index_outside_of_the_vocabulary_makes_its_row_nan(bad):
    ps = _ps()
    z, idx, teacher = make(4, 333, 6, torch.float16, 5, "drop")
    idx[2, 3] = bad
    for scaler in (None, ps.LossScaler(8.0)):
        z = z.detach().requires_grad_(True)
        loss = ps.distillation_loss(z, idx, teacher, reduction="sum", scaler=scaler)
        g = torch.autograd.grad(loss * 8.0, z)[0]
        assert math.isnan(float(loss.detach())) and torch.isnan(g[2]).all() and torch.isfinite(g[[0, 1, 3]]).all()


def test_values_that_are_not_finite_are_seen():
    ps = _ps()
    for v in (float("nan"), float("inf")):
        z, idx, teacher = make(3, 700, 4, torch.float16, 6, "drop")
        z[1, 650] = v
        z.requires_grad_(True)
        loss = ps.distillation_loss(z, idx, teacher, reduction="none")
        g = torch.autograd.grad(loss.sum(), z)[0]
        assert torch.isnan(loss).tolist() == [False, True, False]
        assert torch.isnan(g[1]).any() and torch.isfinite(g[[0, 2]]).all()
    z, idx, teacher = make(3, 700, 4, torch.float16, 6, "drop")
    z[1] = -float("inf")               # a row that leaves nothing: no distribution
    assert torch.isnan(ps.distillation_loss(z, idx, teacher, reduction="none")).tolist() == [False, True, False]


def test_strides_offsets_and_types_of_the_teacher():
    ps = _ps()
    z, idx, teacher = make(8, 1000, 6, torch.float16, 7, "drop")
    want = ps.distillation_loss(z, idx, teacher.half(), reduction="none")
    # Where a row starts decides which terms a thread adds up: the same terms in another order.  Each result is
    # off by at most d from the exact sum, so two of them by 2 d in log Z, and the rounding of the loss on top;
    # the gradient by 2 d of its size and one step of its type.
    d = exponential_error(z, 1.0)
    near = lambda p, q: bool(((p - q).abs() <= 2 * d + 2.0 ** -22 * q.abs()).all())  # noqa: E731
    zs = z.clone().requires_grad_(True)
    wg = torch.autograd.grad(ps.distillation_loss(zs, idx, teacher.half()), zs)[0]
    step = 2 * d * wg.abs().float() + 2.0 ** -10 * wg.abs().float() + 2.0 ** -24
    big = torch.zeros(8, 1003, dtype=torch.float16, device=DEV)
    for off in (0, 1, 3):
        big[:, off:off + 1000] = z
        leaf = big.clone().requires_grad_(True)
        view = leaf[:, off:off + 1000]
        wide = torch.zeros(8, 12, dtype=torch.int64, device=DEV)
        wide[:, ::2] = idx
        tt = torch.zeros(6, 8, dtype=torch.float16, device=DEV)
        tt.copy_(teacher.half().t())
        got = ps.distillation_loss(view, wide[:, ::2], tt.t(), reduction="none")
        assert near(got.detach(), want)
        for scaler in (None, ps.LossScaler(1.0)):
            g = torch.autograd.grad(ps.distillation_loss(view, idx, teacher.half(), scaler=scaler), leaf)[0]
            assert ((g[:, off:off + 1000].float() - wg.float()).abs() <= step).all()
    col = z.t().contiguous().t()        # vocabulary not contiguous
    assert near(ps.distillation_loss(col, idx, teacher.half(), reduction="none"), want)
    one = z[:1].expand(8, 1000)         # a broadcast row
    leaf = z[:1].clone().requires_grad_(True)
    ps.distillation_loss(leaf.expand(8, 1000), idx, teacher, reduction="sum").backward()
    ref = one.contiguous().requires_grad_(True)
    ps.distillation_loss(ref, idx, teacher, reduction="sum").backward()
    assert torch.equal(leaf.grad, ref.grad.sum(0, keepdim=True))


@pytest.mark.parametrize("tail", ["drop", "bucket"])
@pytest.mark.parametrize("dtype", DTYPES)
def test_gradient_of_the_forward_call_is_the_backward_call_s(dtype, tail):
    """Scaled by the scaler the gradient comes out of the forward call, with any other factor out of the
    backward call: the same bits where the factor is the same, powers of two exactly apart where not."""
    ps = _ps()
    z, idx, teacher = make(37, 5003, 12, dtype, 8, tail)
    mask = torch.arange(37, device=DEV) % 5 != 2
    kw = dict(temperature=2.0, tail=tail, mask=mask, weight=0.5)
    scaler = ps.DynamicLossScaler(init_scale=2.0 ** 10)

    def leaf():
        return z.detach().clone().requires_grad_(True)

    a, b, c, d = leaf(), leaf(), leaf(), leaf()
    la = ps.distillation_loss(a, idx, teacher, scaler=scaler, **kw)
    scaler.backward(la)
    lb = ps.distillation_loss(b, idx, teacher, **kw)
    scaler.backward(lb)
    assert torch.equal(la, lb) and torch.equal(a.grad, b.grad)
    lc = ps.distillation_loss(c, idx, teacher, scaler=scaler, **kw)
    (lc * 2.0 ** 9).backward()          # not the scale that was prepared for
    (ps.distillation_loss(d, idx, teacher, **kw) * 2.0 ** 9).backward()
    assert torch.equal(c.grad, d.grad)
    # the scale changes between the forward call and backward
    e = leaf()
    le = ps.distillation_loss(e, idx, teacher, scaler=scaler, **kw)
    scaler.update_scale(True)
    scaler.backward(le)
    assert scaler.loss_scale == 2 ** 9 and torch.equal(e.grad, d.grad)
    # a graph that is walked twice: the first gradient may have been added to in place
    f = leaf()
    lf = ps.distillation_loss(f, idx, teacher, scaler=scaler, **kw)
    scaler.backward(lf, retain_graph=True)
    f.grad.mul_(0)
    scaler.backward(lf)
    assert torch.equal(f.grad, d.grad)


def test_gradient_against_differences():
    ps = _ps()
    z, idx, teacher = make(2, 40, 5, torch.float32, 9, "bucket")
    for tail in ("drop", "bucket"):
        leaf = z.clone().requires_grad_(True)
        g = torch.autograd.grad(ps.distillation_loss(leaf, idx, teacher, temperature=1.5, tail=tail,
                                                     reduction="sum"), leaf)[0]
        for r in range(2):
            for v in (int(idx[r, 0]), int(idx[r, 4]), 0, 17, 39):
                h, vals = 2.0 ** -5, []
                for s in (h, -h):
                    zz = z.clone()
                    zz[r, v] += s
                    vals.append(float(ps.distillation_loss(zz, idx, teacher, temperature=1.5, tail=tail,
                                                           reduction="none").double().sum()))
                # central differences: h^2 / 6 of a third derivative that is below 1.5 here, and the losses'
                # own error (four roundings of values below 16) over 2 h
                assert abs((vals[0] - vals[1]) / (2 * h) - float(g[r, v])) <= h * h / 4 + 4 * 16 * 2.0 ** -23 / h


def test_no_rows():
    ps = _ps()
    z, idx, teacher = make(0, 50, 3, torch.float16, 10, "drop")
    z.requires_grad_(True)
    for kw in (dict(), dict(scaler=ps.LossScaler(4.0)), dict(mask=torch.zeros(0, dtype=torch.bool, device=DEV)),
               dict(reduction="sum"), dict(reduction="none")):
        loss = ps.distillation_loss(z, idx, teacher, **kw)
        assert loss.shape == ((0,) if kw.get("reduction") == "none" else ()) and float(loss.detach().sum()) == 0.0
        assert torch.autograd.grad(loss.sum(), z)[0].shape == (0, 50)


def test_refusals():
    ps = _ps()
    z, idx, teacher = make(4, 50, 3, torch.float16, 11, "drop")
    cpu_scaler = ps.LossScaler(2.0)
    cpu_scaler.device = torch.device("cuda", 1)
    for error, args, kw in ((TypeError, (z.double(), idx, teacher), {}), (TypeError, (z, idx.float(), teacher), {}),
                            (TypeError, (z, idx, teacher.double()), {}), (ValueError, (z, idx[:3], teacher), {}),
                            (ValueError, (z, idx[:, :2], teacher), {}), (ValueError, (z, idx[0], teacher[0]), {}),
                            (ValueError, (z, idx, teacher), dict(temperature=0.0)),
                            (ValueError, (z, idx, teacher), dict(temperature=float("inf"))),
                            (ValueError, (z, idx, teacher), dict(weight=float("nan"))),
                            (ValueError, (z, idx, teacher), dict(tail="keep")),
                            (ValueError, (z, idx, teacher), dict(reduction="batch")),
                            (ValueError, (z, idx.cpu(), teacher), {}),
                            (ValueError, (z, idx[:, :0], teacher[:, :0]), {}),
                            (ValueError, (z, idx, teacher.clone().requires_grad_(True)), {}),
                            (ValueError, (z, idx, teacher), dict(mask=torch.ones(3, dtype=torch.bool, device=DEV))),
                            (TypeError, (z, idx, teacher), dict(mask=torch.ones(4, device=DEV))),
                            (ValueError, (z, idx, teacher), dict(scaler=cpu_scaler)),
                            (ValueError, (z, idx, teacher), dict(scaler=ps.LossScaler(2.0), reduction="none"))):
        with pytest.raises(error):
            ps.distillation_loss(*args, **kw)


def test_same_bits_every_time_other_stream_and_replay():
    ps = _ps()
    z, idx, teacher = make(300, 3001, 16, torch.bfloat16, 12, "bucket")
    idx[:, 3] = idx[:, 4]
    mask = torch.arange(300, device=DEV) % 7 != 0
    scaler = ps.LossScaler(256.0)
    leaf = z.clone().requires_grad_(True)

    def step():
        loss = ps.distillation_loss(leaf, idx, teacher, tail="bucket", mask=mask, scaler=scaler)
        return loss.detach(), torch.autograd.grad(scaler.scale_loss(loss), leaf)[0]

    first = step()
    assert all(torch.equal(p, q) for _ in range(3) for p, q in zip(step(), first))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = step()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(p, q) for p, q in zip(other, first))
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        captured = step()
    for seed in (12, 13):
        z2, i2, t2 = make(300, 3001, 16, torch.bfloat16, seed, "bucket")
        with torch.no_grad():
            leaf.copy_(z2)
            idx.copy_(i2)
            teacher.copy_(t2)
        g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(captured, step()))


@pytest.mark.parametrize("tail", ["drop", "bucket"])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("tau", [1e-4, 1e4])
def test_extreme_logits_and_temperatures(dtype, tail, tau):
    """Exponents beyond 2^30 (a small temperature, logits near the end of the type) and nearly none."""
    ps = _ps()
    z, idx, teacher = make(3, 300, 5, torch.float32, 20, "bucket")
    z[1] = z[1] * (torch.finfo(dtype).max / 16)
    z = z.to(dtype)
    z.requires_grad_(True)
    loss = ps.distillation_loss(z, idx, teacher, temperature=tau, tail=tail, reduction="none")
    g = torch.autograd.grad(loss.sum(), z)[0]
    want, wgrad = definition(z.detach(), idx, teacher, tau, tail)
    # an exponent |z - M| / tau has a relative error of three roundings (and of 2^-24 in 1 / tau): of the exponents
    # themselves where entries are far below the maximum, and those are summed with probabilities of at most 1 in all
    size = (z.detach().double().cpu().amax(1) - z.detach().double().cpu().amin(1)) / tau
    bound = (4 * 2.0 ** -24 * size + 4 * exponential_error(z.detach(), tau)) * tau * tau * 2 + 2.0 ** -22 * want.abs()
    fine = torch.isfinite(want.float())
    assert ((loss.detach().double().cpu() - want).abs() <= bound)[fine].all() and torch.isfinite(loss[fine.to(DEV)]).all()
    # the gradient of a softmax whose exponents are off by e is off by at most 2 e of q (1 - q), and by q itself
    # where e is large: then only its sign and size are held
    q = (wgrad / tau).abs().max()
    assert torch.isfinite(g).all() and float((g.double().cpu() / tau).abs().max()) <= 1.01 * float(q) + 1e-3


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("vocab,k,tail", [(2 ** 19, 1024, "bucket"), (2 ** 19, 1, "bucket"), (2 ** 20, 1024, "drop"),
                                          (300001, 700, "bucket")])
def test_the_largest_sizes(vocab, k, tail, dtype):
    """Bitmaps and listed entries that leave little shared memory for anything else."""
    ps = _ps()
    for rows in (1, 150):
        z, idx, teacher = make(1, vocab, k, dtype, k, tail)
        z, idx, teacher = z.repeat(rows, 1).requires_grad_(True), idx.repeat(rows, 1), teacher.repeat(rows, 1)
        loss = ps.distillation_loss(z, idx, teacher, tail=tail, reduction="none")
        g = torch.autograd.grad(loss, z, torch.full_like(loss, 256.0))[0]
        check(z[-1:].detach(), idx[-1:], teacher[-1:], 1.0, tail, loss[-1:].detach(), g[-1:], 256.0)
        scaler = ps.LossScaler(256.0 * rows)
        total = ps.distillation_loss(z, idx, teacher, tail=tail, scaler=scaler)
        fused = torch.autograd.grad(scaler.scale_loss(total), z)[0]
        # every eighth row starts at the same offset from a 16-byte boundary (8 vocab elements are a multiple of it),
        # so its terms are added in the same order; the others' in another one, as above
        for t in (fused, g):
            assert torch.equal(t[:1].expand(len(t[::8]), -1), t[::8])
        check(z[:1].detach(), idx[:1], teacher[:1], 1.0, tail, total.detach().view(1), fused[:1], 256.0)


def test_offsets_beyond_32_bits():
    """More than 2^32 bytes and 2^31 elements of logits; the last rows are right."""
    ps = _ps()
    rows, vocab = 2049, 2 ** 20
    z = torch.zeros(rows, vocab, dtype=torch.float16, device=DEV)
    idx = torch.zeros(rows, 2, dtype=torch.int32, device=DEV)
    idx[:, 1] = vocab - 1
    teacher = torch.zeros(rows, 2, device=DEV)
    z[-1, -1], z[-1, 0] = 4.0, -2.0
    z[-2, 12345] = 9.0
    z.requires_grad_(True)
    loss = ps.distillation_loss(z, idx, teacher, reduction="none")
    g = torch.autograd.grad(loss, z, torch.full_like(loss, 2.0 ** 14))[0]
    for r in (0, rows - 2, rows - 1):
        check(z[r:r + 1].detach(), idx[r:r + 1], teacher[r:r + 1], 1.0, "drop", loss[r:r + 1].detach(), g[r:r + 1],
              2.0 ** 14)


def test_saved_tensors_that_come_back_elsewhere():
    """Under save_on_cpu the saved tensors return as other tensors."""
    ps = _ps()
    z, idx, teacher = make(20, 501, 4, torch.float16, 14, "drop")
    w = (torch.randn(501, 33, device=DEV) * 0.1).half()
    x = torch.randn(20, 33, device=DEV).half()

    def run():
        leaves = [t.clone().requires_grad_(True) for t in (x, w)]
        loss = ps.distillation_loss(ps.fp8_linear(*leaves), idx, teacher)
        return torch.autograd.grad(loss * 64.0, leaves)

    want = run()
    with torch.autograd.graph.save_on_cpu():
        got = run()
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_no_wait_ran_out():
    import ctypes as C
    from patrickstar_b200 import _lib as L
    n = C.c_uint32(7)
    L.check(L.lib.ps_distill_gave_up(C.byref(n)), "ps_distill_gave_up")
    assert n.value == 0
