"""The 8-bit layer where a model has it in the place of `torch.nn.Linear`: results changed in place or
viewed in another shape, forward-mode differentiation, operands of different types,
kept weights."""
import pytest
import torch
import torch.autograd.forward_ad as fwd

from test_gpu_block_fp8 import DEV, _ps, linear_case, product_bound, rounded

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


@pytest.mark.parametrize("kinds", [("float16", "float32", "bfloat16"), ("bfloat16", "float16", "float32"),
                                   ("float32", "bfloat16", "float16")])
def test_input_weight_and_bias_of_different_types(kinds):
    ps = _ps()
    tx, tw, tb = (getattr(torch, k) for k in kinds)
    x, w, b, dy = linear_case(130, 257, 129, torch.float32, 5)
    x, w, b, dy = x.to(tx), w.to(tw), b.to(tb), dy.to(tx)
    leaves = [t.to(DEV).requires_grad_(True) for t in (x, w, b)]
    y = ps.fp8_linear(*leaves)
    grads = torch.autograd.grad(y, leaves, dy.to(DEV))
    assert (y.dtype,) + tuple(g.dtype for g in grads) == (tx, tx, tw, tb)
    xr, xc, wt = rounded(x, "row", "e4m3"), rounded(x, "col", "e4m3"), rounded(w, "tile", "e4m3")
    dr, dc = rounded(dy, "row", "e4m3"), rounded(dy, "col", "e4m3")
    for got, p, q, length, extra in ((y, xr, wt, 257, b.double()), (grads[0], dr, wt.t(), 129, None),
                                     (grads[1], dc.t(), xc.t(), 130, None)):
        want = p @ q.t()
        bound = product_bound(p, q, length, got.dtype, want)
        if extra is not None:    # one more addition, of the bias, in 32 bits
            want = want + extra
            bound = bound + 2.0 ** -24 * want.abs() + torch.finfo(got.dtype).eps / 2 * want.abs()
        assert ((got.detach().cpu().double() - want).abs() <= bound).all()
    want = dy.double().sum(0)    # runs of 128 rows in 32 bits, the runs in 64, two roundings
    bound = 130 * 2.0 ** -24 * dy.double().abs().sum(0) + torch.finfo(tb).eps / 2 * want.abs()
    assert ((grads[2].cpu().double() - want).abs() <= bound).all()


@pytest.mark.parametrize("fmt", ["e4m3", "e5m2"])
@pytest.mark.parametrize("tokens,k,n", [(1, 64, 48), (130, 257, 129), (300, 130, 1)])
def test_a_kept_weight_in_either_format_and_under_hooks(tokens, k, n, fmt):
    """Forward and input gradient from it; under hooks its saved parts come back packed, elsewhere."""
    ps = _ps()
    x, w, b, dy = linear_case(tokens, k, n, torch.float16, 6)
    kept = ps.block_quantize(w.to(DEV), "tile", fmt)
    wt = rounded(w, "tile", fmt)

    def run():
        leaf = x.to(DEV).requires_grad_(True)
        y = ps.fp8_linear(leaf, kept, b.to(DEV))
        return y.detach(), torch.autograd.grad(y, leaf, dy.to(DEV))[0]

    y, dx = run()
    xr, dr = rounded(x, "row", "e4m3"), rounded(dy, "row", "e4m3")
    want = xr @ wt.t()
    bound = product_bound(xr, wt, k, torch.float16, want) + 2.0 ** -24 * (want + b.double()).abs() + \
        2.0 ** -11 * (want + b.double()).abs()
    assert ((y.cpu().double() - want - b.double()).abs() <= bound).all()
    want = dr @ wt
    assert ((dx.cpu().double() - want).abs() <= product_bound(dr, wt.t(), n, torch.float16, want)).all()
    with torch.autograd.graph.save_on_cpu():
        again = run()
    assert torch.equal(again[0], y) and torch.equal(again[1], dx)


def test_gradients_against_differences_with_the_scales_pinned():
    """Every block of the input, the weight and the incoming gradient holds an element of full scale (448 2^j), the others
    are whole numbers up to 7 times 2^j: with the scale 2^j that this element asks for, all of them are values of the format.
    The layer is then exactly linear in the small elements, and differences of its outputs are its gradients."""
    ps = _ps()
    gen = torch.Generator().manual_seed(10)

    def whole(r, c):
        return torch.randint(-7, 8, (r, c), generator=gen).float()

    x, w, dy = whole(128, 256), whole(128, 256), whole(128, 128)
    # one element of full scale in each row and column of a tile: its diagonal
    d = torch.arange(128)
    for t in (x, w, dy):
        for j in range(0, t.shape[1], 128):
            t[d, j + d] = 448.0
    X, W = x.half().to(DEV).requires_grad_(True), w.half().to(DEV).requires_grad_(True)
    gx, gw = torch.autograd.grad(ps.fp8_linear(X.float(), W.float()), [X, W], dy.to(DEV))

    def value(xx, ww):
        # sums of at most 256 products of up to 448 448 are whole numbers below 2^26; in 32 bits those here are exact
        # when they stay below 2^24, which the assertion on them holds
        y = ps.fp8_linear(xx.to(DEV), ww.to(DEV)).double().cpu()
        assert torch.equal(y, xx.double() @ ww.double().t()) and float(y.abs().max()) < 2 ** 24
        return float((y * dy.double()).sum())

    base = value(x, w)
    for i, j in ((0, 1), (127, 200), (64, 130)):
        moved = x.clone()
        moved[i, j] += 1
        assert value(moved, w) - base == float((dy.double() @ w.double())[i, j])
        # the gradient itself is rounded to 16 bits
        want = float((dy.double() @ w.double())[i, j])
        assert abs(float(gx[i, j]) - want) <= 2.0 ** -11 * abs(want)
        moved = w.clone()
        moved[i, j] += 1
        want = float((dy.double().t() @ x.double())[i, j])
        assert value(x, moved) - base == want
        assert abs(float(gw[i, j]) - want) <= 2.0 ** -11 * abs(want)
