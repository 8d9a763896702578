"""8-bit matrix products of a training step, with one scale for each block of 128.

The matrix products of a model's forward and backward pass on the tensor cores'
8-bit path, next to the fp16 parameters and gradients the chunk step works on:

  * ``block_quantize``  a matrix into e4m3 or e5m2 with a power-of-two scale for
    each block of 1 x 128, 128 x 1 or 128 x 128 elements,
  * ``block_matmul``    the product of two such matrices, accumulated in 32 bits,
  * ``fp8_linear``, ``Fp8Linear``  the linear layer made of them, with its three
    gradients, on ordinary fp16 / bf16 / fp32 tensors and parameters.

The scales are powers of two like the loss scale: scaling is exact, and the
tensor core applies them.  An element that is not finite stays visible (NaN in
e4m3, itself in e5m2), so a gradient that overflowed still reaches the overflow
test of the step.  No counterpart in the reference.
"""
import ctypes as C
import functools
import math

import torch
from torch.autograd import forward_ad

from ._lib import (PS_BLOCKS_COL, PS_BLOCKS_ROW, PS_BLOCKS_ROW_COL, PS_BLOCKS_TILE, PS_DTYPE_BF16, PS_DTYPE_F16,
                   PS_DTYPE_F32, PS_FP8_E4M3, PS_FP8_E5M2, PS_KEEP_INPUT, PS_KEEP_WEIGHT, BlockOperand, Fp8LinearLayer,
                   check, lib)
from .streams import current_device, raw_stream

BLOCK = 128

_DTYPES = {torch.float16: PS_DTYPE_F16, torch.bfloat16: PS_DTYPE_BF16, torch.float32: PS_DTYPE_F32}
_FORMATS = {"e4m3": (torch.float8_e4m3fn, PS_FP8_E4M3), "e5m2": (torch.float8_e5m2, PS_FP8_E5M2)}
_FORMAT_OF = {dtype: code for dtype, code in _FORMATS.values()}
_BLOCKS = {"row": PS_BLOCKS_ROW, "col": PS_BLOCKS_COL, "row+col": PS_BLOCKS_ROW_COL, "tile": PS_BLOCKS_TILE}


def _scales_shape(outer, contracted):
    return (-(-contracted // (4 * BLOCK)), -(-outer // BLOCK), 32, 4, 4)


def _check_scales(name, scales, blocks, used, outer, contracted, data):
    if (scales is not None) != used:
        raise ValueError("%s blocks %s scales in %s" % (blocks, "need" if used else "have no", name))
    if scales is None:
        return
    shape = _scales_shape(outer, contracted)
    if scales.dtype != torch.uint8 or scales.shape != shape or not scales.is_contiguous():
        raise ValueError("%s must be contiguous uint8 of shape %s; got %s of shape %s"
                         % (name, shape, scales.dtype, tuple(scales.shape)))
    if scales.device != data.device:
        raise ValueError("values on %s, %s on %s" % (data.device, name, scales.device))


class BlockQuantized:
    """A matrix [rows, cols] in 8-bit floating point with a scale for each block.

    ``data``     float8_e4m3fn or float8_e5m2, rows a multiple of 16 bytes apart
    ``blocks``   "row" (1 x 128), "col" (128 x 1) or "tile" (128 x 128)
    ``scales1``  scale bytes for a contraction over dimension 1 ("row", "tile"), else None
    ``scales0``  scale bytes for a contraction over dimension 0 ("col", "tile"), else None

    A byte s stands for the scale 2^(s - 127).  For L contracted and O outer
    elements the array is ``uint8[ceil(L / 512), ceil(O / 128), 32, 4, 4]`` and the
    byte of outer element ``o`` and contracted block ``kb`` is at ``[kb // 4, o // 128,
    o % 32, o % 128 // 32, kb % 4]``: the order in which the tensor core reads them.
    """

    __slots__ = ("data", "blocks", "scales1", "scales0")

    def __init__(self, data, blocks, scales1=None, scales0=None):
        if not isinstance(data, torch.Tensor) or data.dtype not in _FORMAT_OF:
            raise TypeError("BlockQuantized needs float8_e4m3fn or float8_e5m2 values, got %s"
                            % getattr(data, "dtype", type(data)))
        if blocks not in ("row", "col", "tile"):
            raise ValueError("blocks must be row, col or tile; got %r" % (blocks,))
        if data.dim() != 2:
            raise ValueError("BlockQuantized needs a matrix, got %d dimensions" % data.dim())
        rows, cols = data.shape
        if rows and cols:
            if cols > 1 and data.stride(1) != 1:
                raise ValueError("the values of a row must be adjacent")
            if data.data_ptr() % 16 or (rows > 1 and (data.stride(0) % 16 or data.stride(0) < cols)):
                raise ValueError("rows of values must start on 16-byte boundaries")
        _check_scales("scales1", scales1, blocks, blocks != "col", rows, cols, data)
        _check_scales("scales0", scales0, blocks, blocks != "row", cols, rows, data)
        self.data, self.blocks, self.scales1, self.scales0 = data, blocks, scales1, scales0

    @classmethod
    def _of(cls, data, blocks, scales1, scales0):
        q = cls.__new__(cls)    # parts that this module allocated: nothing to check
        q.data, q.blocks, q.scales1, q.scales0 = data, blocks, scales1, scales0
        return q

    @property
    def shape(self):
        return self.data.shape

    @property
    def device(self):
        return self.data.device

    @property
    def dtype(self):
        return self.data.dtype

    def exponents(self):
        """int32 exponents of the scales, one for each block: [rows, ceil(cols / 128)] for "row",
        [ceil(rows / 128), cols] for "col", [ceil(rows / 128), ceil(cols / 128)] for "tile"."""
        rows, cols = self.data.shape
        s, outer, contracted = ((self.scales0, cols, rows) if self.blocks == "col" else (self.scales1, rows, cols))
        groups, blocks = s.shape[:2]
        flat = s.permute(1, 3, 2, 0, 4).reshape(blocks * BLOCK, groups * 4)[:outer, :-(-contracted // BLOCK)]
        e = flat.to(torch.int32) - 127
        return e.t() if self.blocks == "col" else e[::BLOCK] if self.blocks == "tile" else e

    def dequantize(self, dtype=torch.float32):
        """The values times their scales."""
        rows, cols = self.data.shape
        e = self.exponents()
        if self.blocks != "row":
            e = e.repeat_interleave(BLOCK, 0)[:rows]
        if self.blocks != "col":
            e = e.repeat_interleave(BLOCK, 1)[:, :cols]
        return torch.ldexp(self.data.float(), e).to(dtype)

    def _operand(self, dim):
        scales = self.scales1 if dim else self.scales0
        rows, cols = self.data.shape
        ld = self.data.stride(0) if rows > 1 else -(-cols // 16) * 16
        return BlockOperand(data=self.data.data_ptr(), scales=scales.data_ptr(), ld=ld,
                            fmt=_FORMAT_OF[self.data.dtype], k_dim=dim)


def _check_float(t, what):
    if not isinstance(t, torch.Tensor) or not t.is_cuda or t.dtype not in _DTYPES:
        raise TypeError("%s must be a CUDA tensor of float16, bfloat16 or float32, got %s" % (
            what, "%s on %s" % (t.dtype, t.device) if isinstance(t, torch.Tensor) else type(t).__name__))


def _format(fmt):
    if fmt not in _FORMATS:
        raise ValueError("the format must be e4m3 or e5m2; got %r" % (fmt,))
    return _FORMATS[fmt]


def _quantize(x, blocks, fmt):
    """block_quantize for a checked matrix."""
    dtype, code = _FORMATS[fmt]
    x = _adjacent(x)
    rows, cols = x.shape
    ldq = -(-cols // 16) * 16
    dev = x.device
    q1 = s1 = q0 = s0 = None
    if blocks != "col":
        q1 = x.new_empty((rows, ldq), dtype=dtype)
        s1 = x.new_empty(_scales_shape(rows, cols), dtype=torch.uint8)
    if blocks in ("col", "row+col"):
        q0 = x.new_empty((rows, ldq), dtype=dtype)
    if blocks != "row":
        s0 = x.new_empty(_scales_shape(cols, rows), dtype=torch.uint8)
    with current_device(dev):
        check(lib.ps_block_quantize(
            x.data_ptr(), _DTYPES[x.dtype], x.stride(0) if rows > 1 else cols, rows, cols, _BLOCKS[blocks], code,
            q1.data_ptr() if q1 is not None else None, s1.data_ptr() if s1 is not None else None,
            q0.data_ptr() if q0 is not None else None, s0.data_ptr() if s0 is not None else None, ldq,
            None, raw_stream(dev)), "ps_block_quantize")
    if cols != ldq:
        q1 = q1 if q1 is None else q1[:, :cols]
        q0 = q0 if q0 is None else q0[:, :cols]
    if blocks == "tile":
        return BlockQuantized._of(q1, "tile", s1, s0)
    row = None if q1 is None else BlockQuantized._of(q1, "row", s1, None)
    col = None if q0 is None else BlockQuantized._of(q0, "col", None, s0)
    return row if blocks == "row" else col if blocks == "col" else (row, col)


def block_quantize(x, blocks="row", fmt="e4m3"):
    """Quantizes the matrix ``x`` (CUDA, float16 / bfloat16 / float32) with a power-of-two scale for each block.

    ``blocks``: "row" for 1 x 128 (to be contracted over dimension 1), "col" for 128 x 1 (over
    dimension 0), "tile" for 128 x 128 (over either), "row+col" for a tuple of the first two
    from one read.  The scale of a block is the smallest power of two that brings its largest
    finite magnitude within the format's range (448 for ``fmt`` "e4m3", 57344 for "e5m2"), not
    below 2^-126; values are rounded to nearest even.  Infinite and NaN elements become NaN in
    e4m3 and stay themselves in e5m2.  No gradient flows through.
    """
    _check_float(x, "block_quantize: x")
    if x.dim() != 2:
        raise ValueError("block_quantize needs a matrix, got %d dimensions" % x.dim())
    if blocks not in _BLOCKS:
        raise ValueError("blocks must be row, col, row+col or tile; got %r" % (blocks,))
    _format(fmt)
    return _quantize(x.detach(), blocks, fmt)


def _rows(like, m, n, dtype):
    """An uninitialised [m, n] tensor on the device of ``like`` whose rows start on 16-byte boundaries: the product then
    leaves the SM in whole boxes.  It is no view: autograd refuses in-place operations on views that a function made."""
    per = 16 // dtype.itemsize
    return like.new_empty_strided((m, n), (-(-n // per) * per, 1), dtype=dtype)


def _matmul(a, a_dim, b, b_dim, bias, out_dtype):
    m, n, k = a.shape[1 - a_dim], b.shape[1 - b_dim], a.shape[a_dim]
    out = _rows(a.data, m, n, out_dtype)
    with current_device(a.device):
        check(lib.ps_block_matmul(
            C.byref(a._operand(a_dim)), C.byref(b._operand(b_dim)), m, n, k,
            bias.data_ptr() if bias is not None else None, _DTYPES[bias.dtype] if bias is not None else 0,
            out.data_ptr(), _DTYPES[out_dtype], max(n, out.stride(0)), raw_stream(a.device)), "ps_block_matmul")
    return out


def _dim(q, dim, what):
    if not isinstance(q, BlockQuantized):
        raise TypeError("block_matmul: %s must be BlockQuantized, got %s" % (what, type(q).__name__))
    if not q.data.is_cuda:
        raise TypeError("block_matmul: %s must be on a CUDA device, got %s" % (what, q.device))
    if dim is None:
        dim = 0 if q.blocks == "col" else 1
    if dim not in (0, 1) or (q.scales1 if dim else q.scales0) is None:
        raise ValueError("block_matmul: %s has %s blocks: they cannot be contracted over dimension %r"
                         % (what, q.blocks, dim))
    return dim


def block_matmul(a, b, a_dim=None, b_dim=None, bias=None, out_dtype=torch.float16):
    """The product of two ``BlockQuantized`` matrices, contracted over dimension ``a_dim`` of ``a`` and
    ``b_dim`` of ``b`` (each by default the one its blocks lie along; 1 for "tile" blocks).

    Returns ``[outer size of a, outer size of b]`` in ``out_dtype`` (float16, bfloat16 or float32),
    accumulated in 32 bits and rounded once, after ``bias`` (one value for each column) was added.  No
    gradient flows through, to ``bias`` either.
    Rows of the result start on 16-byte boundaries: where a row is not a multiple of 16 bytes the result
    is not contiguous.
    """
    a_dim, b_dim = _dim(a, a_dim, "a"), _dim(b, b_dim, "b")
    if a.device != b.device:
        raise ValueError("block_matmul: a on %s, b on %s" % (a.device, b.device))
    if a.shape[a_dim] != b.shape[b_dim]:
        raise ValueError("block_matmul: contracted sizes differ: %d and %d" % (a.shape[a_dim], b.shape[b_dim]))
    if out_dtype not in _DTYPES:
        raise TypeError("block_matmul: out_dtype must be float16, bfloat16 or float32, got %s" % (out_dtype,))
    if bias is not None:
        _check_bias(bias, b.shape[1 - b_dim], a.device, "block_matmul")
        bias = bias.detach().contiguous()
    return _matmul(a, a_dim, b, b_dim, bias, out_dtype)


def _check_bias(bias, n, device, where):
    _check_float(bias, where + ": bias")
    if tuple(bias.shape) != (n,):
        raise ValueError("%s: bias must have shape (%d,), got %s" % (where, n, tuple(bias.shape)))
    if bias.device != device:
        raise ValueError("%s: bias on %s, the product on %s" % (where, bias.device, device))


@functools.lru_cache(maxsize=4096)
def _layer_bytes(tokens, k, n, kept, keep):
    """Bytes of the buffers of ps_fp8_linear_forward and _backward: (saved, forward scratch, backward scratch)."""
    sizes = (C.c_uint64 * 3)()
    check(lib.ps_fp8_linear_sizes(C.byref(Fp8LinearLayer(kept_data=1 if kept else None, tokens=tokens, k=k, n=n)), keep,
                                  sizes), "ps_fp8_linear_sizes")
    return tuple(sizes)


def _layer(x, weight, bias, kept, tokens, k, n):
    """The C struct of a layer.  ``x``, ``weight`` and ``bias`` have adjacent elements."""
    if kept is None:
        return Fp8LinearLayer(x.data_ptr(), weight.data_ptr(), None if bias is None else bias.data_ptr(), None, None,
                              None, x.stride(0) if tokens > 1 else k, weight.stride(0) if n > 1 else k, 0, tokens, k, n,
                              _DTYPES[x.dtype], _DTYPES[weight.dtype], 0 if bias is None else _DTYPES[bias.dtype], 0, 0)
    op = kept._operand(1)
    return Fp8LinearLayer(x.data_ptr(), None, None if bias is None else bias.data_ptr(), op.data, op.scales,
                          kept.scales0.data_ptr(), x.stride(0) if tokens > 1 else k, 0, op.ld, tokens, k, n,
                          _DTYPES[x.dtype], 0, 0 if bias is None else _DTYPES[bias.dtype], op.fmt, 0)


def _adjacent(t):
    return t if t.shape[1] == 1 or t.stride(1) == 1 else t.contiguous()


def _linear_forward(x, weight, bias, kept, keep, contiguous):
    """(y, saved buffer or None, layer struct) of matrices that are checked."""
    tokens, k = x.shape
    n = (weight if kept is None else kept).shape[0]
    x = _adjacent(x)
    if kept is None:
        weight = _adjacent(weight)
    if bias is not None:
        bias = bias.contiguous()
    dev = x.device
    saved_bytes, scratch_bytes, _ = _layer_bytes(tokens, k, n, kept is not None, keep)
    y = x.new_empty((tokens, n)) if contiguous else _rows(x, tokens, n, x.dtype)
    saved = x.new_empty(saved_bytes, dtype=torch.uint8) if saved_bytes else None
    scratch = x.new_empty(scratch_bytes, dtype=torch.uint8)
    layer = _layer(x, weight, bias, kept, tokens, k, n)
    with current_device(dev):
        check(lib.ps_fp8_linear_forward(C.byref(layer), keep, y.data_ptr(), max(n, y.stride(0)),
                                        None if saved is None else saved.data_ptr(), scratch.data_ptr(),
                                        raw_stream(dev)), "ps_fp8_linear_forward")
    return y, saved, layer


def _aligned(data):
    """8-bit values whose rows start on 16-byte boundaries: ``data``, or a copy where a saved tensor came back packed."""
    if data.data_ptr() % 16 == 0 and (data.shape[0] < 2 or data.stride(0) % 16 == 0):
        return data
    out = torch.empty((data.shape[0], -(-data.shape[1] // 16) * 16), dtype=data.dtype, device=data.device)
    out = out[:, :data.shape[1]]
    out.view(torch.uint8).copy_(data.view(torch.uint8))
    return out


def _autograd_sees(*tensors):
    """Whether a call has to go through its autograd function: for a gradient, or inside of a forward-mode level, where
    the function refuses tensors that carry a tangent (``requires_grad`` does not tell) instead of losing it."""
    if forward_ad._current_level >= 0:
        return True
    return torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors)


class _Fp8Linear(torch.autograd.Function):
    """y = Q_row(x) Q_tile(w)^T + b;  dx = Q_row(dy) Q_tile(w);  dw = Q_col(dy)^T Q_col(x);  db = sum of dy."""

    @staticmethod
    def forward(ctx, x, weight, bias, kept, grad_fmt, contiguous):
        need_x, need_w = ctx.needs_input_grad[:2]
        keep = (PS_KEEP_WEIGHT if need_x else 0) | (PS_KEEP_INPUT if need_w else 0)
        y, saved, ctx.layer = _linear_forward(x, weight, bias, kept, keep, contiguous)
        ctx.keep, ctx.grad_fmt, ctx.x_dtype = keep, grad_fmt, x.dtype
        ctx.w_dtype = None if weight is None else weight.dtype
        ctx.b_dtype = None if bias is None else bias.dtype
        ctx.save_for_backward(saved, *((kept.data, kept.scales1, kept.scales0) if kept is not None and need_x else ()))
        return y

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        saved, *kept = ctx.saved_tensors
        layer, dev = ctx.layer, dy.device
        if kept:    # saved tensors may come back elsewhere
            kept[0] = _aligned(kept[0])
            op = BlockQuantized._of(kept[0], "tile", kept[1], kept[2])._operand(0)
            layer.kept_data, layer.kept_scales0, layer.ld_kept = op.data, op.scales, op.ld
        need_x, need_w, need_b = ctx.needs_input_grad[:3]
        dy = _adjacent(dy)
        tokens, k, n = layer.tokens, layer.k, layer.n
        dx = _rows(dy, tokens, k, ctx.x_dtype) if need_x else None
        dw = dy.new_empty((n, k), dtype=ctx.w_dtype) if need_w else None
        db = dy.new_empty(n, dtype=ctx.b_dtype) if need_b else None
        scratch = dy.new_empty(_layer_bytes(tokens, k, n, bool(layer.kept_data), ctx.keep)[2], dtype=torch.uint8)
        with current_device(dev):
            check(lib.ps_fp8_linear_backward(
                C.byref(layer), ctx.keep, None if saved is None else saved.data_ptr(), dy.data_ptr(),
                dy.stride(0) if tokens > 1 else n, _FORMATS[ctx.grad_fmt][1], dx.data_ptr() if need_x else None,
                max(k, dx.stride(0)) if need_x else k, dw.data_ptr() if need_w else None,
                db.data_ptr() if need_b else None, scratch.data_ptr(), raw_stream(dev)), "ps_fp8_linear_backward")
        return dx, dw, db, None, None, None


def fp8_linear(x, weight, bias=None, grad_fmt="e4m3", contiguous=False):
    """``x @ weight.T + bias`` on the 8-bit path; ``x`` [..., K], ``weight`` [N, K], ``bias`` [N].

    ``x`` and ``weight`` are quantized to e4m3 within the call (1 x 128 and 128 x 128 blocks),
    the incoming gradient in the backward pass to ``grad_fmt`` (1 x 128 and 128 x 1 blocks).
    The result and the gradient of ``x`` have the type of ``x``, the gradients of ``weight`` and
    ``bias`` theirs; the gradient of ``bias`` is summed from the unquantized gradient.  Rows of the
    result and of the gradient of ``x`` start on 16-byte boundaries: where N (or K) is not a multiple of
    16 bytes they are not contiguous, but for the result if ``contiguous`` asks for it.  ``weight`` may
    also be a ``BlockQuantized`` with "tile" blocks, quantized once and kept; it has no gradient then.
    Between forward and backward the quantized ``x`` and ``weight`` are kept (one byte an element; that of
    ``weight`` comes on top of the parameter itself), not the originals.  A second derivative and forward-mode derivatives are refused.
    """
    _check_float(x, "fp8_linear: x")
    if x.dim() < 1:
        raise ValueError("fp8_linear: x needs at least one dimension")
    _format(grad_fmt)
    kept = None
    if isinstance(weight, BlockQuantized):
        kept, weight = weight, None
        if kept.blocks != "tile":
            raise ValueError("fp8_linear: a quantized weight needs tile blocks, got %s" % kept.blocks)
        (n, k), dev = kept.shape, kept.device
    else:
        _check_float(weight, "fp8_linear: weight")
        if weight.dim() != 2:
            raise ValueError("fp8_linear: weight must be a matrix, got %d dimensions" % weight.dim())
        (n, k), dev = weight.shape, weight.device
    shape = x.shape
    if shape[-1] != k:
        raise ValueError("fp8_linear: x has %d features, weight takes %d" % (shape[-1], k))
    if dev != x.device:
        raise ValueError("fp8_linear: x on %s, weight on %s" % (x.device, dev))
    if bias is not None:
        _check_bias(bias, n, dev, "fp8_linear")
    x2 = x if len(shape) == 2 else x.reshape(math.prod(shape[:-1]), k)
    if _autograd_sees(x, weight, bias):
        y = _Fp8Linear.apply(x2, weight, bias, kept, grad_fmt, contiguous)
    else:
        y = _linear_forward(x2, weight, bias, kept, 0, contiguous)[0]
    return y if len(shape) == 2 else y.view(shape[:-1] + (n,))


class Fp8Linear(torch.nn.Linear):
    """``torch.nn.Linear`` whose products run through ``fp8_linear``; same parameters and state.

    Its results are contiguous, as those of the layer it stands for: a model may view them in any
    shape.  Rows that are no multiple of 16 bytes then leave the product in small pieces, and the
    gradient that comes back is read in such (4096 x 1600 -> 50257 fp16: product 475 us, 274 us with
    rows on 16-byte boundaries; the gradient's quantization 257 us, not 164 us).  Where the layer's
    reader takes such rows, ``layer.contiguous = False`` saves that."""

    grad_fmt = "e4m3"
    contiguous = True

    def forward(self, x):
        return fp8_linear(x, self.weight, self.bias, self.grad_fmt, self.contiguous)

    def extra_repr(self):
        return super().extra_repr() + ", grad_fmt=%s" % self.grad_fmt


def use_fp8_linears(module, grad_fmt="e4m3"):
    """Makes every ``torch.nn.Linear`` of ``module`` (itself included; not subclasses) an ``Fp8Linear`` in
    place: parameters, buffers, hooks and names stay.  Returns the number of layers changed."""
    _format(grad_fmt)
    n = 0
    for m in module.modules():
        if type(m) is torch.nn.Linear:
            m.__class__ = Fp8Linear
            m.grad_fmt = grad_fmt
            n += 1
    return n
