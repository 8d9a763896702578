"""The 8-bit layer where a model has it in the place of `torch.nn.Linear`: forward-mode differentiation."""
import pytest
import torch
import torch.autograd.forward_ad as fwd

from test_gpu_block_fp8 import DEV, _ps, linear_case

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("which", [0, 1, 2])
def test_a_forward_mode_derivative_is_refused(which):
    ps = _ps()
    args = [t.to(DEV) for t in linear_case(20, 64, 48, torch.float32, 1)[:3]]
    want = ps.fp8_linear(*args)
    with fwd.dual_level():
        assert torch.equal(ps.fp8_linear(*args), want)     # no tangent: as ever
        args[which] = fwd.make_dual(args[which], torch.ones_like(args[which]))
        with pytest.raises(RuntimeError):
            ps.fp8_linear(*args)
        with torch.no_grad(), pytest.raises(RuntimeError):
            ps.fp8_linear(*args)
        if which == 0:
            with pytest.raises(RuntimeError):
                ps.fp8_linear(args[0], ps.block_quantize(args[1], "tile"), args[2])


def test_jvp_is_refused():
    ps = _ps()
    x, w, b, _ = (t.to(DEV) for t in linear_case(20, 64, 48, torch.float32, 1))
    with pytest.raises(RuntimeError):
        torch.func.jvp(lambda t: ps.fp8_linear(t, w, b), (x,), (torch.ones_like(x),))
