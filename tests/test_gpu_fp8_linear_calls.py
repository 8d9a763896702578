"""The 8-bit layer where a model has it in the place of `torch.nn.Linear`: results changed in place or
viewed in another shape, forward-mode differentiation."""
import pytest
import torch
import torch.autograd.forward_ad as fwd

from test_gpu_block_fp8 import DEV, _ps, linear_case

pytestmark = pytest.mark.gpu
WIDTHS = [1, 2, 13, 130, 2305]


def layer(n, k=96, dtype=torch.float16, bias=True):
    torch.manual_seed(n)
    m = torch.nn.Linear(k, n, bias=bias).to(DEV, dtype)
    assert _ps().use_fp8_linears(m) == 1
    return m


@pytest.mark.parametrize("n", WIDTHS)
@pytest.mark.parametrize("op,args", [("relu", ()), ("add", (1.5,)), ("div", (2.0,))])
@pytest.mark.parametrize("how", ["layer", "function", "matrix"])
def test_results_are_changed_in_place(how, op, args, n):
    """... by what reads them next, at any width, with the gradients of the same operation out of place."""
    ps = _ps()
    m = layer(n)
    x = torch.randn(4, 33, 96, device=DEV).half()
    got = []
    for name in (op + "_", op):
        leaves = [t.detach().clone().requires_grad_(True) for t in (x, m.weight, m.bias)]
        if how == "layer":
            y = torch.func.functional_call(m, {"weight": leaves[1], "bias": leaves[2]}, (leaves[0],))
        else:
            y = ps.fp8_linear(leaves[0] if how == "function" else leaves[0].view(-1, 96), leaves[1], leaves[2])
        z = getattr(y, name)(*args)
        assert (z is y) == name.endswith("_")
        got.append([z.detach()] + list(torch.autograd.grad(z.float().sum(), leaves)))
    assert all(torch.equal(p, q) for p, q in zip(*got))


@pytest.mark.parametrize("n", WIDTHS)
@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
def test_the_layer_s_results_can_be_viewed_in_any_shape(n, dtype):
    """As those of the layer it replaces: across the last dimension too."""
    m = layer(n, dtype=dtype)
    x = torch.randn(4, 34, 96, device=DEV).to(dtype).requires_grad_(True)
    y = m(x)
    assert y.is_contiguous() and y.shape == (4, 34, n)
    flat = y.view(-1)
    a = torch.autograd.grad(flat.float().square().sum(), [x, m.weight])
    y = m(x)
    b = torch.autograd.grad(y.float().square().sum(), [x, m.weight])
    assert all(torch.equal(p, q) for p, q in zip(a, b))
    assert torch.equal(m(x).view(2, -1), _ps().fp8_linear(x, m.weight, m.bias).reshape(2, -1))
    with torch.no_grad():
        assert m(x[0]).view(-1).shape == (34 * n,)
    m.contiguous = False    # rows on 16-byte boundaries
    assert torch.equal(m(x), y) and m(x).stride(1) * m(x).element_size() % 16 == 0


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
