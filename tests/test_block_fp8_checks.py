"""What the 8-bit operators refuse, without a GPU."""
import ctypes as C

import pytest
import torch


@pytest.fixture(scope="module")
def ps():
    from patrickstar_b200 import build
    build.build()
    import patrickstar_b200
    return patrickstar_b200


@pytest.fixture(scope="module")
def L(ps):
    from patrickstar_b200 import _lib
    return _lib


def scales(outer, length):
    return torch.zeros(-(-length // 512), -(-outer // 128), 32, 4, 4, dtype=torch.uint8)


def operand(ps, rows=20, cols=32, blocks="row"):
    return ps.BlockQuantized(torch.zeros(rows, cols).to(torch.float8_e4m3fn), blocks,
                             None if blocks == "col" else scales(rows, cols),
                             None if blocks == "row" else scales(cols, rows))


def test_tensors_that_are_not_on_a_gpu_or_not_floating_are_refused(ps):
    x = torch.zeros(4, 32)
    for call in (lambda: ps.block_quantize(x), lambda: ps.fp8_linear(x, x), lambda: ps.block_quantize([1.0]),
                 lambda: ps.block_quantize(torch.zeros(4, 32, dtype=torch.float64)),
                 lambda: ps.block_matmul(operand(ps), operand(ps)), lambda: ps.block_matmul(x, x)):
        with pytest.raises(TypeError):
            call()


def test_parts_that_do_not_fit_are_refused(ps):
    data = torch.zeros(20, 32).to(torch.float8_e4m3fn)
    good = scales(20, 32)
    for error, args in (
            (TypeError, (torch.zeros(20, 32), "row", good)),
            (ValueError, (data, "column", good)),
            (ValueError, (data[0], "row", good)),
            (ValueError, (data, "row", None)),
            (ValueError, (data, "row", good, scales(32, 20))),
            (ValueError, (data, "col", good)),
            (ValueError, (data, "tile", good)),
            (ValueError, (data, "row", good[0])),
            (ValueError, (data, "row", good.float())),
            (ValueError, (data, "row", scales(200, 32))),
            (ValueError, (data.t(), "row", scales(32, 20))),
            (ValueError, (data[:, 1:17], "row", scales(20, 16))),
            (ValueError, (torch.zeros(20, 33).to(torch.float8_e4m3fn), "row", scales(20, 33)))):
        with pytest.raises(error):
            ps.BlockQuantized(*args)
    for blocks in ("row", "col", "tile"):
        assert operand(ps, blocks=blocks).shape == (20, 32)


def test_exponents_and_dequantize_follow_the_layout(ps):
    import fp8_plain
    gen = torch.Generator().manual_seed(0)
    for blocks in ("row", "col", "tile"):
        x = torch.randn(300, 700, generator=gen) * torch.exp2(torch.randn(300, 700, generator=gen) * 3)
        v, by = fp8_plain.quantize(x.double().numpy(), blocks, "e4m3")
        data = torch.zeros(300, 704, dtype=torch.float8_e4m3fn)
        data[:, :700] = torch.from_numpy(v).float().to(torch.float8_e4m3fn)
        q = ps.BlockQuantized(data[:, :700], blocks,
                              None if blocks == "col" else torch.from_numpy(fp8_plain.packed(by, 1)),
                              None if blocks == "row" else torch.from_numpy(fp8_plain.packed(by, 0)))
        want = torch.from_numpy(v).float() * torch.exp2(torch.from_numpy(by).float() - 127)
        assert torch.equal(q.dequantize(), want)
        # 8 bits hold 4 significant ones: half a step is 2^-4 of the value, or of the block's smallest normal
        assert ((want - x).abs() <= 2.0 ** -4 * x.abs() + 2.0 ** -10 * torch.exp2(torch.from_numpy(by) - 127)).all()


def test_the_c_entries_refuse(L):
    lib, p = L.lib, C.c_void_p(4096)
    F16, ROW, COL, BOTH, TILE, E4 = (L.PS_DTYPE_F16, L.PS_BLOCKS_ROW, L.PS_BLOCKS_COL, L.PS_BLOCKS_ROW_COL,
                                     L.PS_BLOCKS_TILE, L.PS_FP8_E4M3)

    def quantize(x=p, dtype=F16, ld=64, rows=4, cols=64, blocks=ROW, fmt=E4, q1=p, s1=p, q0=p, s0=p, ldq=64, sums=None):
        return lib.ps_block_quantize(x, dtype, ld, rows, cols, blocks, fmt, q1, s1, q0, s0, ldq, sums, None)

    assert quantize(rows=0) == 0 and quantize(cols=0) == 0
    for bad in (dict(x=None), dict(dtype=3), dict(dtype=-1), dict(blocks=4), dict(fmt=2), dict(ldq=48),
                dict(q1=None), dict(s1=None), dict(blocks=COL, q0=None), dict(blocks=COL, s0=None),
                dict(blocks=BOTH, q0=None), dict(blocks=TILE, s0=None), dict(sums=p), dict(blocks=TILE, sums=p)):
        assert quantize(**bad) == L.PS_ERR_INVALID, bad
    for bad in (dict(x=C.c_void_p(4097)), dict(ldq=72), dict(q1=C.c_void_p(4104)), dict(blocks=COL, q0=C.c_void_p(4104))):
        assert quantize(**bad) == L.PS_ERR_ALIGN, bad

    def op(data=4096, scales=4096, ld=64, fmt=0, k_dim=1):
        return C.byref(L.BlockOperand(data=data, scales=scales, ld=ld, fmt=fmt, k_dim=k_dim))

    def matmul(a=None, b=None, m=4, n=4, k=64, bias=None, bias_dtype=0, out=p, out_dtype=F16, ldo=4):
        return lib.ps_block_matmul(a or op(), b or op(), m, n, k, bias, bias_dtype, out, out_dtype, ldo, None)

    assert matmul(m=0) == 0 and matmul(n=0) == 0
    for bad in (dict(out=None), dict(ldo=3), dict(out_dtype=3), dict(bias=p, bias_dtype=5), dict(a=op(data=0)),
                dict(b=op(scales=0)), dict(a=op(fmt=2)), dict(a=op(k_dim=2)), dict(k=65), dict(m=65, a=op(k_dim=0))):
        assert matmul(**bad) == L.PS_ERR_INVALID, bad
    for bad in (dict(a=op(data=4104)), dict(b=op(scales=4100)), dict(a=op(ld=72)), dict(out=C.c_void_p(4097))):
        assert matmul(**bad) == L.PS_ERR_ALIGN, bad
    assert matmul(m=2 ** 31) == L.PS_ERR_LIMIT and matmul(k=2 ** 32 - 1) == L.PS_ERR_LIMIT
    assert lib.ps_block_matmul(None, None, 1, 1, 16, None, 0, p, F16, 1, None) == L.PS_ERR_INVALID
    assert lib.ps_column_sum(None, 1, 4, p, F16, None) == L.PS_ERR_INVALID
    assert lib.ps_column_sum(p, 1, 4, p, 9, None) == L.PS_ERR_INVALID and lib.ps_column_sum(p, 1, 0, p, F16, None) == 0
    assert lib.ps_block_matmul_gave_up(None) == L.PS_ERR_INVALID


def test_the_layer_entries_refuse(L):
    lib, p = L.lib, 4096

    def layer(**kw):
        d = dict(x=p, weight=p, ld_x=64, ld_weight=64, tokens=4, k=64, n=32)
        d.update(kw)
        return C.byref(L.Fp8LinearLayer(**d))

    def forward(keep=0, y=p, ld=32, saved=p, scratch=p, **kw):
        return lib.ps_fp8_linear_forward(layer(**kw), keep, y, ld, saved, scratch, None)

    def backward(keep=3, saved=p, dy=p, ld=32, fmt=0, dx=p, dw=p, db=p, scratch=p, **kw):
        return lib.ps_fp8_linear_backward(layer(**kw), keep, saved, dy, ld, fmt, dx, 64, dw, db, scratch, None)

    for call in (forward, backward):
        for bad in (dict(x_dtype=3), dict(x_dtype=-1), dict(kept_data=p, kept_fmt=2), dict(scratch=None)):
            assert call(**bad) == L.PS_ERR_INVALID, bad
        assert call(tokens=2 ** 31) == L.PS_ERR_LIMIT and call(k=2 ** 32 - 1) == L.PS_ERR_LIMIT
        for bad in (dict(saved=p + 16), dict(scratch=p + 128)):
            assert call(**bad) == L.PS_ERR_ALIGN, bad
    assert forward(tokens=0, scratch=None) == 0 and forward(n=0) == 0
    for bad in (dict(x=None), dict(weight=None), dict(weight_dtype=7), dict(keep=3, saved=None)):
        assert forward(**bad) == L.PS_ERR_INVALID, bad
    for bad in (dict(fmt=2), dict(keep=0), dict(keep=1), dict(keep=2), dict(saved=None), dict(dy=None)):
        assert backward(**bad) == L.PS_ERR_INVALID, bad
    assert backward(dx=None, dw=None, db=None) == 0
    sizes = (C.c_uint64 * 3)()
    assert lib.ps_fp8_linear_sizes(layer(), 3, None) == L.PS_ERR_INVALID
    assert lib.ps_fp8_linear_sizes(None, 3, sizes) == L.PS_ERR_INVALID
    assert lib.ps_fp8_linear_sizes(layer(tokens=130, k=70, n=40), 0, sizes) == 0 and sizes[0] == 0
    # x and weight in rows of 80 bytes, scales of 128 for each of 512 contracted, pieces rounded up to 256
    assert sizes[1] == (130 * 80 + 96) + 1024 + 512 + 3328 + 512
    assert lib.ps_fp8_linear_sizes(layer(tokens=130, k=70, n=40), 3, sizes) == 0
    assert sizes[0] == 3328 + 512 + (130 * 80 + 96) + 512


def test_layers_are_changed_in_place(ps):
    net = torch.nn.Sequential(torch.nn.Linear(4, 5), torch.nn.Tanh(), torch.nn.Bilinear(2, 2, 2),
                              torch.nn.Sequential(torch.nn.Linear(5, 6, bias=False)))
    names, ids = [n for n, _ in net.named_parameters()], [id(p) for p in net.parameters()]
    assert ps.use_fp8_linears(net, "e5m2") == 2
    assert isinstance(net[0], ps.Fp8Linear) and net[3][0].grad_fmt == "e5m2" and type(net[2]) is torch.nn.Bilinear
    assert [n for n, _ in net.named_parameters()] == names and [id(p) for p in net.parameters()] == ids
    assert ps.use_fp8_linears(net) == 0     # they are changed already
    with pytest.raises(ValueError):
        ps.use_fp8_linears(net, "e3m4")
