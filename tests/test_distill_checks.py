"""What the distillation loss refuses, without a GPU."""
import ctypes as C

import pytest
import torch


@pytest.fixture(scope="module")
def ps():
    from patrickstar_b200 import build
    build.build()
    import patrickstar_b200
    return patrickstar_b200


def test_the_python_entry_refuses_what_is_not_on_a_gpu(ps):
    z, i, t = torch.zeros(2, 10), torch.zeros(2, 3, dtype=torch.int64), torch.zeros(2, 3)
    for args in ((z, i, t), (z.double(), i, t), (None, i, t)):
        with pytest.raises(TypeError):
            ps.distillation_loss(*args)
    with pytest.raises(ValueError):
        ps.DistillationLoss(tail="rest")
    with pytest.raises(ValueError):
        ps.DistillationLoss(reduction="batchmean")


def test_the_c_entries_refuse(ps):
    from patrickstar_b200 import _lib as L
    lib, p = L.lib, 4096

    def problem(**kw):
        d = dict(logits=p, indices=p, teacher=p, mask=None, ld_logits=10, ld_indices=3, ld_teacher=3, rows=2, vocab=10,
                 k=3, dtype=0, index_bytes=8, teacher_dtype=2, tail=0, reduction=2, temperature=1.0, weight=1.0)
        d.update(kw)
        return L.DistillProblem(**d)

    def forward(q=None, loss=p, row=p, stats=p, inv_n=None, scaler=None, grad=None, ld=10, used=None, **kw):
        return lib.ps_distill_forward(C.byref(q or problem(**kw)), loss, row, stats, inv_n, scaler, grad, ld, used, None)

    def backward(stats=p, inv_n=None, g=p, stride=0, used=None, grad=p, ld=10, **kw):
        return lib.ps_distill_backward(C.byref(problem(**kw)), stats, inv_n, g, stride, used, grad, ld, None)

    nan, inf = float("nan"), float("inf")
    for call in (forward, backward):
        for bad in (dict(dtype=3), dict(teacher_dtype=-1), dict(index_bytes=2), dict(tail=2), dict(reduction=3),
                    dict(temperature=0.0), dict(temperature=-1.0), dict(temperature=nan), dict(temperature=inf),
                    dict(weight=nan), dict(weight=-inf), dict(vocab=0), dict(k=0), dict(logits=None),
                    dict(indices=None), dict(teacher=None), dict(mask=p, inv_n=None), dict(stats=None)):
            assert call(**bad) == L.PS_ERR_INVALID, bad
        assert call(vocab=L.PS_DISTILL_MAX_VOCAB + 1) == L.PS_ERR_LIMIT
        assert call(k=L.PS_DISTILL_MAX_K + 1) == L.PS_ERR_LIMIT
        assert call(vocab=L.PS_DISTILL_MAX_VOCAB // 2 + 1, tail=1) == L.PS_ERR_LIMIT
        assert call(rows=2 ** 31) == L.PS_ERR_LIMIT
        for bad in (dict(logits=p + 1), dict(teacher=p + 2), dict(indices=p + 4), dict(stats=p + 8)):
            assert call(**bad) == L.PS_ERR_ALIGN, bad
    assert lib.ps_distill_forward(None, p, p, p, None, None, None, 0, None, None) == L.PS_ERR_INVALID
    for bad in (dict(loss=None), dict(row=None), dict(grad=p), dict(grad=p, scaler=p),
                dict(grad=p, scaler=p, used=p, ld=9), dict(grad=p, scaler=p, used=p, reduction=0)):
        assert forward(**bad) == L.PS_ERR_INVALID, bad
    assert forward(grad=p + 1, scaler=p, used=p) == L.PS_ERR_ALIGN
    for bad in (dict(g=None), dict(grad=None), dict(ld=9), dict(used=p, reduction=0)):
        assert backward(**bad) == L.PS_ERR_INVALID, bad
    assert backward(grad=p + 1) == L.PS_ERR_ALIGN
    assert lib.ps_distill_gave_up(None) == L.PS_ERR_INVALID
    assert backward(rows=0, logits=None) == 0 and forward(rows=0, logits=None, reduction=0, row=None, stats=None) == 0
