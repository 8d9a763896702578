"""8-bit quantization and products against their definitions in 64 bits."""
import numpy as np
import pytest
import torch

import fp8_plain

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
TORCH_FMT = {"e4m3": torch.float8_e4m3fn, "e5m2": torch.float8_e5m2}
FORMS = {"forward": ("row", 1, "tile", 1), "input_grad": ("row", 1, "tile", 0), "weight_grad": ("col", 0, "col", 0),
         "rows": ("row", 1, "row", 1), "mixed": ("col", 0, "row", 1), "tiles": ("tile", 0, "tile", 0)}


def _ps():
    import patrickstar_b200
    return patrickstar_b200


def integer_operand(rows, cols, blocks, fmt, gen):
    """Small whole numbers with scales 2^0 .. 2^2, as BlockQuantized and as the numbers they stand for."""
    ps = _ps()
    v = torch.randint(-4, 5, (rows, cols), generator=gen).double()
    rb, cb = -(-rows // 128), -(-cols // 128)
    grid = {"row": (rows, cb), "col": (rb, cols), "tile": (rb, cb)}[blocks]
    e = torch.randint(0, 3, grid, generator=gen)
    by = e if blocks == "row" else e.repeat_interleave(128, 0)[:rows]
    by = by if blocks == "col" else by.repeat_interleave(128, 1)[:, :cols]
    b = (by + 127).numpy()
    ld = -(-cols // 16) * 16
    # what lies behind the last column is not part of the matrix
    data = torch.full((rows, ld), 7.0).to(TORCH_FMT[fmt])
    data[:, :cols] = v.to(TORCH_FMT[fmt])
    q = ps.BlockQuantized(data.to(DEV)[:, :cols], blocks,
                          torch.from_numpy(fp8_plain.packed(b, 1)).to(DEV) if blocks != "col" else None,
                          torch.from_numpy(fp8_plain.packed(b, 0)).to(DEV) if blocks != "row" else None)
    return q, v * torch.exp2(by.double())


SHAPES = [(1, 16, 16), (1, 1, 1), (128, 128, 128), (128, 128, 512), (7, 250, 129), (130, 129, 640), (257, 384, 1000),
          (300, 17, 1537), (64, 1600, 800), (513, 1025, 300), (640, 640, 2100), (1, 4096, 1024), (2300, 2090, 1100), (2560, 2304, 128), (1281, 4099, 257)]


@pytest.mark.parametrize("form", sorted(FORMS))
@pytest.mark.parametrize("m,n,k", SHAPES)
def test_products_of_whole_numbers_are_exact(form, m, n, k):
    """Every partial sum is a whole number below 2^24 (|a b| <= 4 4 * 4 4 = 256, k <= 2100), so the result
    does not depend on the order of the additions and has to be equal."""
    ps = _ps()
    gen = torch.Generator().manual_seed(m * 7 + n * 3 + k)
    ba, da, bb, db = FORMS[form]
    fa, fb = ("e4m3", "e4m3") if (m + n + k) % 3 else ("e5m2", "e4m3") if (m + n) % 2 else ("e4m3", "e5m2")
    a, av = integer_operand(*((m, k) if da else (k, m)), ba, fa, gen)
    b, bv = integer_operand(*((n, k) if db else (k, n)), bb, fb, gen)
    bias = torch.randint(-100, 100, (n,), generator=gen).float()
    want = (av if da else av.t()) @ (bv.t() if db else bv)
    got = ps.block_matmul(a, b, a_dim=da, b_dim=db, out_dtype=torch.float32)
    assert torch.equal(got.cpu().double(), want)
    got = ps.block_matmul(a, b, a_dim=da, b_dim=db, bias=bias.to(DEV), out_dtype=torch.float32)
    assert torch.equal(got.cpu().double(), want + bias.double())


def test_accumulator_holds_24_bits():
    """2^23 from the first block, then 1408 ones of either sign: every partial sum is a whole number of at
    most 2^24, exact in 32 bits and not in fewer."""
    ps = _ps()
    gen = torch.Generator().manual_seed(5)
    m, n, k = 130, 140, 128 * 12
    a = torch.zeros(m, k)
    b = torch.zeros(n, k)
    a[:, 0], b[:, 0] = 1.0, 1.0
    a[:, 128:] = torch.randint(0, 2, (m, k - 128), generator=gen) * 2.0 - 1
    b[:, 128:] = torch.randint(0, 2, (n, k - 128), generator=gen) * 2.0 - 1
    by = torch.full((m, k), 127)
    by[:, :128] = 127 + 23
    ones = torch.full((n, k), 127)
    qa = ps.BlockQuantized(a.to(torch.float8_e4m3fn).to(DEV), "row",
                           torch.from_numpy(fp8_plain.packed(by.numpy(), 1)).to(DEV))
    qb = ps.BlockQuantized(b.to(torch.float8_e4m3fn).to(DEV), "row",
                           torch.from_numpy(fp8_plain.packed(ones.numpy(), 1)).to(DEV))
    want = 2.0 ** 23 + a[:, 128:].double() @ b[:, 128:].double().t()
    assert torch.equal(ps.block_matmul(qa, qb, out_dtype=torch.float32).cpu().double(), want)


def special(rows, cols, gen, dtype):
    """Values of many magnitudes, with blocks of zeros, subnormals, borders of the scale and single outliers."""
    x = torch.randn(rows, cols, generator=gen) * torch.exp2(torch.randint(-6, 7, (rows, cols), generator=gen).float())
    if rows > 2:
        x[1] = 0.0
        x[2] *= 2.0 ** -20
    if cols > 3:
        x[:, 3] = 1.75 * torch.exp2(torch.randint(-3, 14, (rows,), generator=gen).float())
    x = x.to(dtype)
    if rows > 5 and cols > 5:
        x[4, 0] = torch.finfo(dtype).max
        x[5, 5] = -torch.finfo(dtype).smallest_normal
        x[5, 4] = torch.finfo(dtype).max / 2
    return x


def as_numpy(q):
    return q.data.float().cpu().numpy().astype(np.float64)


def same(got, want):
    assert got.shape == want.shape
    ok = (got == want) | (np.isnan(got) & np.isnan(want))
    assert ok.all(), "%d of %d differ" % ((~ok).sum(), ok.size)


@pytest.mark.parametrize("fmt", ["e4m3", "e5m2"])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("shape", [(1, 1), (1, 700), (700, 1), (129, 130), (128, 512), (260, 641), (37, 1031)])
@pytest.mark.parametrize("blocks", ["row", "col", "tile", "row+col"])
def test_quantize_is_its_definition_bit_for_bit(shape, blocks, dtype, fmt):
    ps = _ps()
    gen = torch.Generator().manual_seed(shape[0] + 31 * shape[1])
    x = special(*shape, gen, dtype)
    out = ps.block_quantize(x.to(DEV), blocks, fmt)
    for q in out if isinstance(out, tuple) else (out,):
        want, by = fp8_plain.quantize(x.double().numpy(), q.blocks, fmt)
        same(as_numpy(q), want)
        for dim, s in ((1, q.scales1), (0, q.scales0)):
            if s is not None:
                assert np.array_equal(s.cpu().numpy(), fp8_plain.packed(by, dim))
        same(q.dequantize(torch.float64).cpu().numpy(),
             (torch.from_numpy(want).float() * torch.exp2(torch.from_numpy(by).float() - 127)).double().numpy())


@pytest.mark.parametrize("fmt", ["e4m3", "e5m2"])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
def test_elements_that_are_not_finite_stay_visible_and_leave_the_scale_alone(dtype, fmt):
    ps = _ps()
    gen = torch.Generator().manual_seed(3)
    x = torch.randn(140, 300, generator=gen).to(dtype)
    x[0, 0], x[0, 130], x[77, 299], x[139, 5] = float("inf"), float("-inf"), float("nan"), float("inf")
    x[20] = float("inf")     # a whole row without a finite element
    for blocks in ("row", "col", "tile"):
        q = ps.block_quantize(x.to(DEV), blocks, fmt)
        want, by = fp8_plain.quantize(x.double().numpy(), blocks, fmt)
        same(as_numpy(q), want)
        s, dim = (q.scales0, 0) if blocks == "col" else (q.scales1, 1)
        assert np.array_equal(s.cpu().numpy(), fp8_plain.packed(by, dim))


def test_quantize_takes_any_stride_and_alignment():
    ps = _ps()
    gen = torch.Generator().manual_seed(4)
    big = torch.randn(300, 515, generator=gen).half().to(DEV)
    for x in (big[:, 1:514], big[3:, :256], big[::2, 5:], big.t(), big[:, ::2], big[7:8, 3:]):
        q, p = ps.block_quantize(x, "row"), ps.block_quantize(x.contiguous().clone(), "row")
        assert torch.equal(q.data.view(torch.uint8), p.data.view(torch.uint8)) and torch.equal(q.scales1, p.scales1)


def test_quantize_writes_nothing_behind_its_rows():
    """Through the C entry: values behind the last column beyond the next multiple of 8, and behind the last
    row, stay as they were."""
    import ctypes as C
    from patrickstar_b200 import _lib as L
    x = torch.ones(3, 17, dtype=torch.float16, device=DEV)
    q = torch.full((5, 48), 0x55, dtype=torch.uint8, device=DEV)
    s = torch.zeros(1, 1, 32, 4, 4, dtype=torch.uint8, device=DEV)
    st = C.c_void_p(torch.cuda.current_stream().cuda_stream)
    L.check(L.lib.ps_block_quantize(x.data_ptr(), L.PS_DTYPE_F16, 17, 3, 17, L.PS_BLOCKS_ROW, L.PS_FP8_E4M3,
                                    q.data_ptr(), s.data_ptr(), None, None, 48, None, st), "ps_block_quantize")
    got = q.cpu()
    assert (got[:3, 24:] == 0x55).all() and (got[3:] == 0x55).all() and (got[:3, 17:24] == 0).all()


def product_bound(a, b, k, out_dtype, want):
    """Every product of two 8-bit values is exact in 32 bits (4 + 4 significant bits).  A sum of k of them in
    32 bits makes k additions, each off by at most 2^-23 (truncation) of a partial sum, which is at most
    S = sum |a b|; the result is rounded once, by at most half a step."""
    s = a.abs() @ b.abs().t()
    return k * 2.0 ** -23 * s + torch.finfo(out_dtype).eps / 2 * want.abs() + torch.finfo(out_dtype).tiny


@pytest.mark.parametrize("out_dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("form", ["forward", "input_grad", "weight_grad"])
@pytest.mark.parametrize("m,n,k", [(1, 257, 300), (200, 513, 1601), (1030, 700, 128), (2311, 2049, 640)])
def test_products_of_ordinary_matrices(form, m, n, k, out_dtype):
    ps = _ps()
    gen = torch.Generator().manual_seed(m + n + k)
    ba, da, bb, db = FORMS[form]
    a = torch.randn(*((m, k) if da else (k, m)), generator=gen) * torch.exp2(torch.randn(1, generator=gen))
    b = torch.randn(*((n, k) if db else (k, n)), generator=gen) * 0.02
    qa, qb = ps.block_quantize(a.to(DEV), ba, "e5m2"), ps.block_quantize(b.to(DEV), bb)
    av, bv = qa.dequantize(torch.float64).cpu(), qb.dequantize(torch.float64).cpu()
    av, bv = av if da else av.t(), bv if db else bv.t()
    want = av @ bv.t()
    got = ps.block_matmul(qa, qb, a_dim=da, b_dim=db, out_dtype=out_dtype).cpu().double()
    assert ((got - want).abs() <= product_bound(av, bv, k, out_dtype, want)).all()


def test_empty_and_one():
    ps = _ps()
    w = torch.randn(24, 40, device=DEV).half().requires_grad_(True)
    b = torch.randn(24, device=DEV).half().requires_grad_(True)
    x = torch.randn(0, 40, device=DEV).half().requires_grad_(True)
    y = ps.fp8_linear(x, w, b)
    assert y.shape == (0, 24) and y.dtype == torch.float16
    gx, gw, gb = torch.autograd.grad(y, [x, w, b], torch.zeros_like(y))
    assert gx.shape == x.shape and not gw.any() and not gb.any() and gw.shape == w.shape and gb.shape == b.shape
    x = torch.randn(3, 0, device=DEV).half()
    w0 = torch.zeros(24, 0, device=DEV).half()
    assert torch.equal(ps.fp8_linear(x, w0, b.detach()), b.detach().expand(3, 24))
    one = ps.fp8_linear(torch.full((1,), 3.0, device=DEV).half(), torch.full((1, 1), 5.0, device=DEV).half())
    assert one.shape == (1,) and float(one) == 15.0
    assert ps.fp8_linear(torch.zeros(2, 3, 40, device=DEV).half(), w.detach()).shape == (2, 3, 24)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("m,n,ldo", [(5, 19, 32), (130, 131, 140), (1000, 900, 913), (1000, 900, 912), (300, 257, 264),
                                     (2100, 2303, 2304), (2100, 2305, 2320), (600, 2001, 2001), (129, 512, 520)])
def test_output_behind_the_last_column_and_row_stays(m, n, ldo, dtype):
    """Through the C entry with a row stride larger than the columns.  Sums of 100 products of at most 4 4 in
    size and scales of at most 2^2 each are whole numbers below 25600; those above 2048 (fp16) or 256 (bf16) are
    rounded once."""
    import ctypes as C
    from patrickstar_b200 import _lib as L
    code = {torch.float16: L.PS_DTYPE_F16, torch.bfloat16: L.PS_DTYPE_BF16, torch.float32: L.PS_DTYPE_F32}[dtype]
    gen = torch.Generator().manual_seed(n)
    a, av = integer_operand(m, 100, "row", "e4m3", gen)
    b, bv = integer_operand(n, 100, "row", "e4m3", gen)
    bias = torch.randint(-100, 100, (n,), generator=gen).to(dtype)
    for shift in (0, 1):    # the second time from an address that is not on a 16-byte boundary
        flat = torch.full(((m + 2) * ldo + shift,), 123.0, dtype=dtype, device=DEV)
        out = flat[shift:].view(m + 2, ldo)
        L.check(L.lib.ps_block_matmul(C.byref(a._operand(1)), C.byref(b._operand(1)), m, n, 100, bias.to(DEV).data_ptr(),
                                      code, out.data_ptr(), code, ldo,
                                      C.c_void_p(torch.cuda.current_stream().cuda_stream)), "ps_block_matmul")
        got = out.cpu()
        assert torch.equal(got[:m, :n], (av @ bv.t() + bias.double()).to(dtype))
        assert (got[m:] == 123.0).all() and (got[:, n:] == 123.0).all()


def test_infinities_and_nan_reach_their_rows_and_columns_only():
    ps = _ps()
    x = torch.randn(200, 300, device=DEV).half()
    w = (torch.randn(150, 300, device=DEV) * 0.1).half()
    x[3, 7], x[190, 299] = float("inf"), float("nan")
    w[140, 0] = float("-inf")
    y = ps.fp8_linear(x, w)
    bad = torch.zeros(200, 150, dtype=torch.bool, device=DEV)
    bad[3], bad[190], bad[:, 140] = True, True, True
    assert torch.equal(~torch.isfinite(y), bad)


def linear_case(tokens, k, n, dtype, seed):
    gen = torch.Generator().manual_seed(seed)
    x = (torch.randn(tokens, k, generator=gen) * torch.exp2(torch.randn(k, generator=gen))).to(dtype)
    w = (torch.randn(n, k, generator=gen) * 0.02).to(dtype)
    b = (torch.randn(n, generator=gen) * 0.1).to(dtype)
    dy = (torch.randn(tokens, n, generator=gen) * 0.01).to(dtype)
    return x, w, b, dy


def rounded(t, blocks, fmt):
    v, by = fp8_plain.quantize(t.double().numpy(), blocks, fmt)
    return torch.from_numpy(v * np.exp2(by - 127.0))


@pytest.mark.parametrize("grad_fmt", ["e4m3", "e5m2"])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("tokens,k,n", [(1, 64, 48), (130, 257, 129), (515, 384, 200)])
def test_linear_and_its_gradients_are_the_formula(tokens, k, n, dtype, grad_fmt):
    ps = _ps()
    x, w, b, dy = linear_case(tokens, k, n, dtype, tokens + k)
    leaves = [t.to(DEV).requires_grad_(True) for t in (x, w, b)]
    y = ps.fp8_linear(*leaves, grad_fmt=grad_fmt)
    grads = torch.autograd.grad(y, leaves, dy.to(DEV))
    xr, xc, wt = rounded(x, "row", "e4m3"), rounded(x, "col", "e4m3"), rounded(w, "tile", "e4m3")
    dr, dc = rounded(dy, "row", grad_fmt), rounded(dy, "col", grad_fmt)
    for got, (p, q, length, extra) in zip((y,) + grads[:2], ((xr, wt, k, b.double()), (dr, wt.t(), n, None),
                                                            (dc.t(), xc.t(), tokens, None))):
        want = p @ q.t()
        bound = product_bound(p, q, length, dtype, want)
        if extra is not None:    # one more addition, of the bias, in 32 bits
            want = want + extra
            bound = bound + 2.0 ** -24 * want.abs() + torch.finfo(dtype).eps / 2 * want.abs()
        assert got.dtype == dtype
        assert ((got.detach().cpu().double() - want).abs() <= bound).all()
    want = dy.double().sum(0)
    # runs of 128 rows in 32 bits (at most 128 additions), the runs in 64, two roundings to 32 bits or fewer
    bound = 130 * 2.0 ** -24 * dy.double().abs().sum(0) + torch.finfo(dtype).eps / 2 * want.abs()
    assert ((grads[2].cpu().double() - want).abs() <= bound).all()


def test_linear_gradients_against_differences():
    """Inputs, weights and incoming gradients are whole numbers below 16 with a full-scale element in each
    block, so that quantization changes nothing and the layer is exactly linear: differences of its outputs
    are its gradients exactly."""
    ps = _ps()
    gen = torch.Generator().manual_seed(9)
    x = torch.randint(-7, 8, (33, 130), generator=gen).half()
    w = torch.randint(-7, 8, (20, 130), generator=gen).half()
    dy = torch.randint(-7, 8, (33, 20), generator=gen).half()
    X, W = x.to(DEV).requires_grad_(True), w.to(DEV).requires_grad_(True)
    y = ps.fp8_linear(X, W)
    gx, gw = torch.autograd.grad(y, [X, W], dy.to(DEV))

    def value(xx, ww):
        return float((ps.fp8_linear(xx.float().to(DEV), ww.float().to(DEV)).double().cpu() * dy.double()).sum())

    base = value(x, w)
    for i, j in ((0, 0), (32, 129), (7, 128)):
        moved = x.clone()
        moved[i, j] += 1
        assert value(moved, w) - base == float(gx[i, j])
    for i, j in ((0, 0), (19, 129), (3, 127)):
        moved = w.clone()
        moved[i, j] += 1
        assert value(x, moved) - base == float(gw[i, j])


def test_linear_needs_only_what_is_asked():
    ps = _ps()
    x, w, b, dy = (t.to(DEV) for t in linear_case(130, 200, 96, torch.float16, 1))
    full = [t.clone().requires_grad_(True) for t in (x, w, b)]
    want = torch.autograd.grad(ps.fp8_linear(*full), full, dy)
    for pick in ((0,), (1,), (2,), (0, 1), (1, 2), (0, 2)):
        args = [t.clone().requires_grad_(i in pick) for i, t in enumerate((x, w, b))]
        got = torch.autograd.grad(ps.fp8_linear(*args), [args[i] for i in pick], dy)
        assert all(torch.equal(g, want[i]) for g, i in zip(got, pick))
    kept = ps.block_quantize(w, "tile")
    X = x.clone().requires_grad_(True)
    y = ps.fp8_linear(X, kept, b)
    assert torch.equal(y, ps.fp8_linear(x, w, b)) and torch.equal(torch.autograd.grad(y, X, dy)[0], want[0])


def test_gradients_of_broadcast_and_strided_inputs():
    ps = _ps()
    x, w, b, dy = (t.to(DEV) for t in linear_case(64, 96, 80, torch.float16, 2))
    row = x[:1].clone().requires_grad_(True)
    ps.fp8_linear(row.expand(64, 96), w, b).backward(torch.ones(1, device=DEV).half().expand(64, 80))
    one = x[:1].clone().requires_grad_(True)
    ps.fp8_linear(one.expand(64, 96).contiguous(), w, b).backward(torch.ones(64, 80, device=DEV).half())
    assert torch.equal(row.grad, one.grad)
    wt = w.t().contiguous().requires_grad_(True)   # a weight that is a transposed view
    W = w.clone().requires_grad_(True)
    a = torch.autograd.grad(ps.fp8_linear(x, wt.t(), b), wt, dy)[0]
    c = torch.autograd.grad(ps.fp8_linear(x, W, b), W, dy)[0]
    assert torch.equal(a.t(), c)


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
@pytest.mark.parametrize("shape", [(130, 129, 41), (700, 260, 2305)])
def test_rows_of_results_start_on_16_byte_boundaries(shape, dtype):
    """Widths that are no multiple of 16 bytes: results are views of longer rows, and what reads them (a next layer,
    its backward pass) takes them as they are."""
    ps = _ps()
    tokens, k, n = shape
    x, w, _, _ = (t.to(DEV) for t in linear_case(tokens, k, n, dtype, 7))
    x = x.view(2, tokens // 2, k).requires_grad_(True)
    y = ps.fp8_linear(x, w)
    assert y.shape == (2, tokens // 2, n) and (y.stride(1) * y.element_size()) % 16 == 0 and y.stride(2) == 1
    assert torch.equal(y.view(-1, n), y.reshape(-1, n))
    w2 = (torch.randn(24, n, device=DEV) * 0.1).to(dtype)
    out = ps.fp8_linear(y, w2)
    assert torch.equal(out, ps.fp8_linear(y.contiguous(), w2))
    g = torch.randn_like(out)
    got = torch.autograd.grad(out, x, g)[0]
    leaf = y.detach().contiguous().requires_grad_(True)
    dy = torch.autograd.grad(ps.fp8_linear(leaf, w2), leaf, g)[0]
    assert torch.equal(got, torch.autograd.grad(ps.fp8_linear(x, w), x, dy.contiguous())[0])


def test_a_second_derivative_is_refused():
    ps = _ps()
    x = torch.randn(8, 32, device=DEV).half().requires_grad_(True)
    w = torch.randn(16, 32, device=DEV).half()
    g = torch.autograd.grad(ps.fp8_linear(x, w).float().square().sum(), x, create_graph=True)[0]
    with pytest.raises(RuntimeError):
        torch.autograd.grad(g.sum(), x)


def test_two_threads_at_once():
    import threading
    ps = _ps()
    cases = [[t.to(DEV) for t in linear_case(300 + 100 * i, 640, 200, torch.float16, i)] for i in range(4)]
    want = [ps.fp8_linear(x, w, b) for x, w, b, _ in cases]
    torch.cuda.synchronize()
    wrong = []

    def work(i):
        stream = torch.cuda.Stream()
        with torch.cuda.stream(stream):
            for _ in range(20):
                x, w, b, _ = cases[i]
                if not torch.equal(ps.fp8_linear(x, w, b), want[i]):
                    wrong.append(i)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong


def test_same_bits_every_time_and_on_another_stream():
    ps = _ps()
    x, w, b, dy = (t.to(DEV) for t in linear_case(700, 1600, 300, torch.bfloat16, 3))

    def step():
        leaves = [t.clone().requires_grad_(True) for t in (x, w, b)]
        y = ps.fp8_linear(*leaves)
        return (y.detach(),) + torch.autograd.grad(y, leaves, dy)

    first = step()
    assert all(torch.equal(p, q) for _ in range(3) for p, q in zip(step(), first))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    assert all(torch.equal(p, q) for p, q in zip(other, first))


def test_captured_step_replays_on_new_inputs():
    ps = _ps()
    x, w, b, dy = (t.to(DEV) for t in linear_case(300, 640, 200, torch.float16, 4))
    leaves = [t.clone().requires_grad_(True) for t in (x, w, b)]
    grad = dy.clone()

    def step():
        y = ps.fp8_linear(*leaves)
        return (y.detach(),) + torch.autograd.grad(y, leaves, grad)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        captured = step()
    for seed in (4, 5):
        with torch.no_grad():
            for t, v in zip(leaves + [grad], linear_case(300, 640, 200, torch.float16, seed)):
                t.copy_(v.to(DEV))
        g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(captured, step()))


def test_no_wait_ran_out():
    import ctypes as C
    from patrickstar_b200 import _lib as L
    n = C.c_uint32(7)
    L.check(L.lib.ps_block_matmul_gave_up(C.byref(n)), "ps_block_matmul_gave_up")
    assert n.value == 0
