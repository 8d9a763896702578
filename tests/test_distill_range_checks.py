"""Temperatures of the distillation loss that 32 bits cannot hold, without a GPU."""
import ctypes as C

import pytest


@pytest.mark.parametrize("temperature,ok", [(2.0 ** -126, True), (2.0 ** -127, False), (2.0 ** -149, False), (3e38, True)])
def test_temperatures_below_the_normal_numbers_are_refused(temperature, ok):
    """log2(e) / temperature would be infinite."""
    from patrickstar_b200 import build
    build.build()
    from patrickstar_b200 import _lib as L
    p = 4096
    q = L.DistillProblem(logits=p, indices=p, teacher=p, mask=None, ld_logits=10, ld_indices=3, ld_teacher=3, rows=0, vocab=10,
                         k=3, dtype=0, index_bytes=8, teacher_dtype=2, tail=0, reduction=0, temperature=temperature, weight=1.0)
    want = 0 if ok else L.PS_ERR_INVALID    # no rows: nothing to launch
    assert L.lib.ps_distill_forward(C.byref(q), None, None, None, None, None, None, 0, None, None) == want
    assert L.lib.ps_distill_backward(C.byref(q), None, None, None, 0, None, None, 10, None) == want
