"""Calls of the distillation loss from several threads, by its module, under forward-mode differentiation and with
a scaler that was given a device without its number."""
import threading

import pytest
import torch
import torch.autograd.forward_ad as fwd

from test_gpu_distill import DEV, _ps, make

pytestmark = pytest.mark.gpu


def test_threads_with_different_sizes():
    """Vocabularies that take very different amounts of shared memory in the same kernel, from eight threads with as
    little as possible between the calls: none of them may find the kernel set up for another's size."""
    import ctypes as C
    from patrickstar_b200 import _lib as L
    vocabs = [2 ** 19, 20000, 100000, 2 ** 19, 40000, 30000, 2 ** 19, 20000]
    wrong, ready = [], threading.Barrier(len(vocabs), timeout=120)

    def work(i):
        z, idx, teacher = make(1, vocabs[i], 1, torch.float16, i, "bucket")
        problem = L.DistillProblem(z.data_ptr(), idx.data_ptr(), teacher.data_ptr(), None, vocabs[i], 1, 1, 1, vocabs[i], 1,
                                   L.PS_DTYPE_F16, 8, L.PS_DTYPE_F32, L.PS_TAIL_BUCKET, L.PS_REDUCE_NONE, 1.0, 1.0)
        out = torch.zeros(8, device=DEV)
        stream = torch.cuda.Stream()
        stream.wait_stream(torch.cuda.current_stream())
        args = (C.byref(problem), None, out.data_ptr(), out.data_ptr() + 16, None, None, None, 0, None, stream.cuda_stream)
        ready.wait()
        codes = [L.lib.ps_distill_forward(*args) for _ in range(2000)]
        stream.synchronize()
        want = _ps().distillation_loss(z, idx, teacher, tail="bucket", reduction="none")
        if any(codes) or not torch.equal(out[:1], want):
            wrong.append((vocabs[i], sum(c != 0 for c in codes)))

    threads = [threading.Thread(target=work, args=(i,)) for i in range(len(vocabs))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    assert not wrong


@pytest.mark.parametrize("which", [0, 2])
def test_a_forward_mode_derivative_is_refused(which):
    ps = _ps()
    args = list(make(4, 333, 5, torch.float32, 1, "drop"))
    ps_loss = ps.distillation_loss(*args)
    with fwd.dual_level():
        assert torch.equal(ps.distillation_loss(*args), ps_loss)     # no tangent: as ever
        args[which] = fwd.make_dual(args[which], torch.ones_like(args[which]))
        with pytest.raises(RuntimeError):
            ps.distillation_loss(*args)
        with torch.no_grad(), pytest.raises(RuntimeError):
            ps.distillation_loss(*args)


def test_jvp_is_refused():
    ps = _ps()
    z, idx, teacher = make(4, 333, 5, torch.float32, 1, "drop")
    with pytest.raises(RuntimeError):
        torch.func.jvp(lambda t: ps.distillation_loss(t, idx, teacher), (z,), (torch.ones_like(z),))


@pytest.mark.parametrize("kind", ["LossScaler", "DynamicLossScaler"])
def test_a_scaler_on_the_current_device_by_its_type(kind):
    """`device="cuda"` is the current device."""
    ps = _ps()
    z, idx, teacher = make(4, 333, 5, torch.float16, 2, "drop")
    scaler = getattr(ps, kind)(8.0, device="cuda")
    assert scaler.device == z.device
    z.requires_grad_(True)
    loss = ps.distillation_loss(z, idx, teacher, scaler=scaler)
    scaler.backward(loss)
    other = z.detach().clone().requires_grad_(True)
    (ps.distillation_loss(other, idx, teacher) * 8.0).backward()
    assert torch.equal(z.grad, other.grad)


def test_temperatures_at_the_ends():
    """1 / T has to be a number of 32 bits."""
    ps = _ps()
    z, idx, teacher = make(4, 333, 5, torch.float32, 3, "drop")
    for t in (1e-39, 1e-46, 1e39):
        with pytest.raises(ValueError):
            ps.distillation_loss(z, idx, teacher, temperature=t)
    with pytest.raises(ValueError):
        ps.distillation_loss(z, idx, teacher, weight=1e39)
    assert torch.isfinite(ps.distillation_loss(z, idx, teacher, temperature=1e-30))


def test_the_module_is_the_function():
    ps = _ps()
    z, idx, teacher = make(12, 700, 6, torch.bfloat16, 4, "bucket")
    mask = torch.arange(12, device=DEV) % 3 != 0
    scaler = ps.LossScaler(32.0)
    kw = dict(temperature=2.0, tail="bucket", reduction="sum", weight=0.5, scaler=scaler)
    module = ps.DistillationLoss(**kw)
    for m in (None, mask):
        a, b = z.clone().requires_grad_(True), z.clone().requires_grad_(True)
        la, lb = module(a, idx, teacher, m), ps.distillation_loss(b, idx, teacher, mask=m, **kw)
        assert torch.equal(la, lb)
        scaler.backward(la)
        scaler.backward(lb)
        assert torch.equal(a.grad, b.grad)
