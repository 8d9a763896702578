"""The measured cases of the training step's 8-bit matrix products and of its distillation loss.

Four operators, as a step around ``FP16Adam`` uses them:

``quantize``  a matrix into 8-bit floating point with one power-of-two scale for each block of 128
``matmul``    the product of two such matrices, accumulated in 32 bits
``linear``    the linear layer made of the two: forward alone, or with its three gradients
``distill``   the divergence from a teacher's top entries: forward alone, or with its gradient

``run`` computes them with the package's kernels when ``own`` is true and with elementary torch
operations in 32 bits otherwise; ``exact`` evaluates the definitions in 64 bits.
"""
import math

import torch

own = False

BLOCK = 128
TYPES = {"float16": torch.float16, "bfloat16": torch.bfloat16, "float32": torch.float32}
SIZE = {"float16": 2, "bfloat16": 2, "float32": 4}
FORMATS = {"e4m3": (torch.float8_e4m3fn, 8), "e5m2": (torch.float8_e5m2, 15)}
LOSS_SCALE = 1024.0


def listed():
    return [
        # one token through the up projection of the 1600-wide layout: what latency costs
        dict(name="linear_1x1600x6400", op="linear", step=False, tokens=1, k=1600, n=6400, dtype="float16",
             bias=True, grad="e4m3"),
        # a micro-batch through the vocabulary head: odd width, ragged contraction
        dict(name="linear_777x1600x50257", op="linear", step=False, tokens=777, k=1600, n=50257, dtype="bfloat16",
             bias=False, grad="e4m3"),
        # four sequences of 1024 through the attention projection of the 1600-wide layout, with gradients
        dict(name="linear_step_4096x1600x4800", op="linear", step=True, tokens=4096, k=1600, n=4800,
             dtype="float16", bias=True, grad="e5m2"),
        # eight sequences through the up projection of the 5120-wide layout, with gradients
        dict(name="linear_step_8192x5120x20480", op="linear", step=True, tokens=8192, k=5120, n=20480,
             dtype="float16", bias=True, grad="e4m3"),
        # a product alone: both operands are in 8 bits already
        dict(name="matmul_8192x8192x8192", op="matmul", m=8192, n=8192, k=8192, form="forward", fmt_a="e4m3",
             dtype="bfloat16"),
        # a weight gradient alone: few outputs, a long contraction of odd length
        dict(name="matmul_grad_1600x1600x16385", op="matmul", m=1600, n=1600, k=16385, form="weight_grad",
             fmt_a="e5m2", dtype="float16"),
        # activations in both directions, as a training step keeps them
        dict(name="quantize_pair_8192x5120", op="quantize", rows=8192, cols=5120, blocks="row+col",
             dtype="float16", fmt="e4m3"),
        # a weight of odd width
        dict(name="quantize_tile_4801x1599", op="quantize", rows=4801, cols=1599, blocks="tile", dtype="bfloat16",
             fmt="e4m3"),
        # one row of logits
        dict(name="distill_1x50257", op="distill", step=False, rows=1, vocab=50257, k=8, dtype="float16",
             tail="drop", temperature=1.0, masked=False),
        # a long batch with its gradient
        dict(name="distill_step_8192x50257", op="distill", step=True, rows=8192, vocab=50257, k=64,
             dtype="float16", tail="drop", temperature=2.0, masked=True),
        # a large vocabulary in bf16, the mass outside of the top entries kept
        dict(name="distill_step_1021x131073", op="distill", step=True, rows=1021, vocab=131073, k=100,
             dtype="bfloat16", tail="bucket", temperature=1.0, masked=False),
        # logits in 32 bits, the loss alone (evaluation)
        dict(name="distill_2048x32000_f32", op="distill", step=False, rows=2048, vocab=32000, k=20,
             dtype="float32", tail="bucket", temperature=1.0, masked=True),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["linear", "linear", "matmul", "quantize", "distill", "distill"])
    half = rng.choice(["float16", "bfloat16"])
    if op == "linear":
        k, n = _log(rng, 32, 8192), _log(rng, 32, 20480)
        most = 8192 * 5120 * 20480 // (k * n)
        return dict(op=op, step=rng.random() < 0.6, tokens=_log(rng, 1, min(16384, most)), k=k, n=n, dtype=half,
                    bias=rng.random() < 0.5, grad=rng.choice(["e4m3", "e5m2"]))
    if op == "matmul":
        m, n, k = _log(rng, 1, 8192), _log(rng, 16, 8192), _log(rng, 16, 16384)
        return dict(op=op, m=m, n=n, k=k, form=rng.choice(["forward", "input_grad", "weight_grad"]),
                    fmt_a=rng.choice(["e4m3", "e5m2"]), dtype=half)
    if op == "quantize":
        return dict(op=op, rows=_log(rng, 1, 16384), cols=_log(rng, 16, 20480),
                    blocks=rng.choice(["row", "col", "tile", "row+col"]),
                    dtype=rng.choice(["float16", "bfloat16", "float32"]), fmt=rng.choice(["e4m3", "e5m2"]))
    vocab = _log(rng, 500, 131073)
    return dict(op=op, step=rng.random() < 0.6, rows=_log(rng, 1, min(16384, 8192 * 50257 // vocab)), vocab=vocab,
                k=_log(rng, 1, 128), dtype=rng.choice(["float16", "bfloat16", "float32"]),
                tail=rng.choice(["drop", "bucket"]), temperature=rng.choice([1.0, 2.0, 1.5]),
                masked=rng.random() < 0.5)


# ------------------------------------------------------------------------------------------------- inputs
def _pack(byte, outer_blocks, group_blocks):
    """[outer, contracted blocks] scale bytes in the layout the product reads: [groups of four contracted
    blocks, blocks of 128 outer elements, 32, 4, 4], zeros where nothing is."""
    full = torch.zeros(outer_blocks * 128, group_blocks * 4, dtype=torch.uint8, device=byte.device)
    full[:byte.shape[0], :byte.shape[1]] = byte
    return full.view(outer_blocks, 4, 32, group_blocks, 4).permute(3, 0, 2, 1, 4).contiguous()


def _quantized(shape, blocks, fmt, g, spread):
    """A matrix in 8 bits as one comes out of a checkpoint or another step: values and scale bytes."""
    dtype, top = FORMATS[fmt]
    r, c = shape
    ld = -(-c // 16) * 16
    data = torch.zeros(r, ld, dtype=dtype, device="cuda")
    data[:, :c] = (torch.randn(r, c, device="cuda", generator=g) * 2.0 ** (top - 3)).to(dtype)
    rb, cb = -(-r // BLOCK), -(-c // BLOCK)
    grid = {"row": (r, cb), "col": (rb, c), "tile": (rb, cb)}[blocks]
    byte = (127 - top + spread + torch.randint(-2, 3, grid, device="cuda", generator=g)).to(torch.uint8)
    by_row = byte if blocks == "row" else byte.repeat_interleave(BLOCK, 0)[:r] if blocks == "tile" else None
    by_col = byte if blocks == "col" else byte.repeat_interleave(BLOCK, 1)[:, :c] if blocks == "tile" else None
    scales1 = None if by_row is None else _pack(by_row, rb, -(-cb // 4))
    scales0 = None if by_col is None else _pack(by_col.t(), cb, -(-rb // 4))
    return dict(data=data[:, :c], byte=byte, scales1=scales1, scales0=scales0, blocks=blocks)


_FORMS = {  # blocks and contracted dimension of a and of b
    "forward": ("row", 1, "tile", 1), "input_grad": ("row", 1, "tile", 0), "weight_grad": ("col", 0, "col", 0)}


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed))

    def randn(*shape):
        return torch.randn(*shape, device="cuda", generator=g)

    s = dict(case=case)
    if case["op"] == "linear":
        t, k, n, dt = case["tokens"], case["k"], case["n"], TYPES[case["dtype"]]
        channels = torch.exp2(randn(k))    # some channels of activations are much larger than others
        s["x"] = (randn(t, k) * channels).to(dt)
        s["w"] = (randn(n, k) * 0.02).to(dt)
        s["b"] = (randn(n) * 0.1).to(dt) if case["bias"] else None
        if case["step"]:
            s["dy"] = (randn(t, n) * 0.01 * torch.exp2(randn(t, 1))).to(dt)
            for name in ("x", "w", "b"):
                if s[name] is not None:
                    s[name].requires_grad_(True)
    elif case["op"] == "matmul":
        ba, da, bb, db = _FORMS[case["form"]]
        m, n, k = case["m"], case["n"], case["k"]
        s["a"] = _quantized((m, k) if da else (k, m), ba, case["fmt_a"], g, 0)
        s["b"] = _quantized((n, k) if db else (k, n), bb, "e4m3", g, -5)
    elif case["op"] == "quantize":
        s["x"] = (randn(case["rows"], case["cols"]) * torch.exp2(2 * randn(case["cols"]))).to(TYPES[case["dtype"]])
    else:
        r, v, k, dt = case["rows"], case["vocab"], case["k"], TYPES[case["dtype"]]
        k = min(k, v)
        z = randn(r, v) * 2.0
        slot = (torch.arange(k, device="cuda") + torch.rand(r, k, device="cuda", generator=g) * 0.999) * (v / k)
        idx = slot.to(torch.int64).clamp_(max=v - 1)
        idx = idx.gather(1, torch.rand(r, k, device="cuda", generator=g).argsort(1))
        teacher = (randn(r, k) * 2.0 + 3.0).sort(1, descending=True).values
        z.scatter_add_(1, idx, teacher + randn(r, k))    # the student agrees with the teacher in part
        rest = randn(r, 1) + math.log(v)
        s["teacher"] = teacher - torch.logaddexp(teacher.logsumexp(1, keepdim=True), rest)
        s["z"] = z.to(dt).requires_grad_(case["step"])
        s["idx"] = idx
        s["mask"] = torch.rand(r, device="cuda", generator=g) < 0.8 if case["masked"] else None
    return s


# --------------------------------------------------------------------------------------------- plain forms
def _by_block(v, blocks):
    """v [R, C] cut into its blocks: a tensor whose dimensions 1 and 3 run inside of a block."""
    r, c = v.shape
    br = 1 if blocks == "row" else BLOCK
    bc = 1 if blocks == "col" else BLOCK
    rb, cb = -(-r // br), -(-c // bc)
    if (rb * br, cb * bc) != (r, c):
        v = torch.nn.functional.pad(v, (0, cb * bc - c, 0, rb * br - r))
    return v.view(rb, br, cb, bc)


def _quantize(x, blocks, fmt):
    """(8-bit values [R, C], scale bytes [row blocks, column blocks])."""
    dtype, top = FORMATS[fmt]
    r, c = x.shape
    v = _by_block(x.float(), blocks)
    mag = v.abs()
    amax = torch.where(mag < math.inf, mag, 0.0).amax((1, 3), keepdim=True)
    frac, e = torch.frexp(amax)
    byte = torch.where(amax > 0, e - 1 - top + (frac > 0.875) + 127, 1).clamp(1, 254)
    q = torch.ldexp(v, 127 - byte).to(dtype)
    return q.reshape(q.shape[0] * q.shape[1], -1)[:r, :c], byte[:, 0, :, 0].to(torch.uint8)


def _dequantize(data, byte, blocks):
    r, c = data.shape
    v = _by_block(data.float(), blocks)
    return torch.ldexp(v, byte.int()[:, None, :, None] - 127).reshape(v.shape[0] * v.shape[1], -1)[:r, :c]


def _rounded(x, blocks, fmt):
    return _dequantize(*_quantize(x, blocks, fmt), blocks)


def _packed(byte, blocks, rows, cols):
    rb, cb = -(-rows // BLOCK), -(-cols // BLOCK)
    out = []
    if blocks in ("row", "tile"):
        out.append(_pack(byte.repeat_interleave(BLOCK, 0)[:rows] if blocks == "tile" else byte, rb, -(-cb // 4)))
    if blocks in ("col", "tile"):
        out.append(_pack((byte.repeat_interleave(BLOCK, 1)[:, :cols] if blocks == "tile" else byte).t(), cb,
                         -(-rb // 4)))
    return out


def _plain_linear(s):
    case = s["case"]
    x, w = s["x"].detach(), s["w"].detach()
    dt = x.dtype
    wq = _rounded(w, "tile", "e4m3")
    y = _rounded(x, "row", "e4m3") @ wq.t()
    if s["b"] is not None:
        y = y + s["b"].detach().float()
    if not case["step"]:
        return (y.to(dt),)
    dy = s["dy"]
    dx = _rounded(dy, "row", case["grad"]) @ wq
    dw = _rounded(dy, "col", case["grad"]).t() @ _rounded(x, "col", "e4m3")
    out = (y.to(dt), dx.to(dt), dw.to(dt))
    return out if s["b"] is None else out + (dy.sum(0, dtype=torch.float64).to(dt),)


def _plain_distill(s):
    case = s["case"]
    z, idx, tau = s["z"].detach(), s["idx"], case["temperature"]
    bucket = case["tail"] == "bucket"
    keep = torch.ones(z.shape[0], dtype=torch.bool, device=z.device) if s["mask"] is None else s["mask"]
    z = z.float() / tau
    top = z.amax(1, keepdim=True)
    e = torch.exp(z - top)
    total = e.sum(1, dtype=torch.float64, keepdim=True)
    logq = z.gather(1, idx).double() - top.double() - total.log()
    if bucket:
        logp = s["teacher"].double()
        p = logp.exp()
        p_rest = (1 - p.sum(1, keepdim=True)).clamp_min(0)
        rest = e.scatter(1, idx, 0.0).sum(1, dtype=torch.float64, keepdim=True)
        off = p_rest * (p_rest.log() - (rest / total).log())
        off = torch.where(p_rest > 0, off, 0.0)[:, 0]
    else:
        t = s["teacher"].double() / tau
        t = t - t.amax(1, keepdim=True)
        logp = t - t.exp().sum(1, keepdim=True).log()
        p = logp.exp()
        off = 0.0
    row = torch.where(p > 0, p * (logp - logq), 0.0).sum(1) + off
    n = keep.sum().clamp_min(1)
    loss = (torch.where(keep, row, 0.0).sum() * tau * tau / n).float()
    if not case["step"]:
        return (loss,)
    if bucket:
        outside = torch.ones_like(z).scatter_(1, idx, 0.0)
        grad = e / total.float() - outside * e * (p_rest / rest).float()
    else:
        grad = e / total.float()
    grad = grad.scatter_add_(1, idx, -p.float()) * (tau * LOSS_SCALE / n.float())
    return loss, torch.where(keep[:, None], grad, 0.0).to(s["z"].dtype)


def _plain(s):
    case = s["case"]
    if case["op"] == "linear":
        return _plain_linear(s)
    if case["op"] == "matmul":
        ba, da, bb, db = _FORMS[case["form"]]
        a = _dequantize(s["a"]["data"], s["a"]["byte"], ba)
        b = _dequantize(s["b"]["data"], s["b"]["byte"], bb)
        return ((a if da else a.t()) @ (b.t() if db else b)).to(TYPES[case["dtype"]])
    if case["op"] == "quantize":
        out = []
        for blocks in case["blocks"].split("+"):
            data, byte = _quantize(s["x"], blocks, case["fmt"])
            out += [data.contiguous()] + _packed(byte, blocks, *s["x"].shape)
        return out
    return _plain_distill(s)


# ----------------------------------------------------------------------------------------- package's calls
def _own(s):
    import patrickstar_b200 as ps
    case = s["case"]
    if case["op"] == "linear":
        y = ps.fp8_linear(s["x"], s["w"], s["b"], grad_fmt=case["grad"])
        if not case["step"]:
            return (y,)
        leaves = [t for t in (s["x"], s["w"], s["b"]) if t is not None]
        return (y.detach(),) + torch.autograd.grad(y, leaves, s["dy"])
    if case["op"] == "matmul":
        _, da, _, db = _FORMS[case["form"]]
        a, b = (ps.BlockQuantized(q["data"], q["blocks"], q["scales1"], q["scales0"]) for q in (s["a"], s["b"]))
        return ps.block_matmul(a, b, a_dim=da, b_dim=db, out_dtype=TYPES[case["dtype"]])
    if case["op"] == "quantize":
        q = ps.block_quantize(s["x"], case["blocks"], case["fmt"])
        out = []
        for one in q if isinstance(q, tuple) else (q,):
            out += [t for t in (one.data, one.scales1, one.scales0) if t is not None]
        return out
    if "scaler" not in s:
        s["scaler"] = ps.LossScaler(LOSS_SCALE)
    loss = ps.distillation_loss(s["z"], s["idx"], s["teacher"], temperature=case["temperature"], tail=case["tail"],
                                mask=s["mask"], scaler=s["scaler"] if case["step"] else None)
    if not case["step"]:
        return (loss,)
    return (loss.detach(),) + torch.autograd.grad(s["scaler"].scale_loss(loss), s["z"])


def run(state):
    return _own(state) if own else _plain(state)


# ------------------------------------------------------------------------------------------------- 64 bits
def _exact_bytes(amax, fmt):
    largest = {"e4m3": 448.0, "e5m2": 57344.0}[fmt]
    # inputs have 24 bits: the slack is far below their spacing and far above the logarithm's error
    return torch.where(amax > 0, torch.ceil(torch.log2(amax / largest) - 1e-9) + 127, 1).clamp(1, 254)


def _exact_values(v, fmt):
    """v rounded to the nearest value of the format, ties to the even one."""
    bits, low = {"e4m3": (3, -6), "e5m2": (2, -14)}[fmt]
    e = torch.floor(torch.log2(v.abs().clamp_min(1e-300))).clamp_min(low) - bits
    return torch.round(v * torch.exp2(-e)) * torch.exp2(e)


def _exact_quantize(x, blocks, fmt):
    """(values before the scale, scale of every element) in 64 bits."""
    x = x.double()
    r, c = x.shape
    amax = x.abs()
    for dim, size in ((0, r), (1, c)):
        if blocks == "tile" or (blocks == "col") == (dim == 0):
            parts = [p.amax(dim, keepdim=True) for p in amax.split(BLOCK, dim)]
            amax = torch.cat(parts, dim).repeat_interleave(BLOCK, dim).narrow(dim, 0, size)
    scale = torch.exp2(_exact_bytes(amax, fmt) - 127).expand(r, c)
    return _exact_values(x / scale, fmt), scale


def _exact_rounded(x, blocks, fmt):
    v, scale = _exact_quantize(x, blocks, fmt)
    return v * scale


def _exact_scaled(q):
    data, byte, blocks = q["data"].double(), q["byte"].double(), q["blocks"]
    scale = torch.exp2(byte - 127)
    if blocks != "row":
        scale = scale.repeat_interleave(BLOCK, 0)[:data.shape[0]]
    if blocks != "col":
        scale = scale.repeat_interleave(BLOCK, 1)[:, :data.shape[1]]
    return data * scale


def _exact_distill(s):
    case = s["case"]
    tau, tail = case["temperature"], case["tail"]
    rows = s["z"].shape[0]
    keep = torch.ones(rows, dtype=torch.bool, device="cuda") if s["mask"] is None else s["mask"]
    n = max(1, int(keep.sum()))
    loss, grads = 0.0, []
    for at in range(0, rows, 512):
        z = s["z"][at:at + 512].detach().double().requires_grad_(True)
        idx, teacher = s["idx"][at:at + 512], s["teacher"][at:at + 512].double()
        log_q = torch.log_softmax(z / tau, 1)
        if tail == "bucket":
            listed_ = torch.zeros_like(z, dtype=torch.bool).scatter_(1, idx, True)
            p = teacher.exp()
            p_rest = (1 - p.sum(1)).clamp_min(0)
            kl = torch.special.xlogy(p_rest, p_rest) - p_rest * log_q.masked_fill(listed_, -math.inf).logsumexp(1)
        else:
            p = torch.softmax(teacher / tau, 1)
            kl = 0.0
        kl = kl + (torch.special.xlogy(p, p) - p * log_q.gather(1, idx)).sum(1)
        part = (kl * keep[at:at + 512]).sum() * (tau * tau / n)
        loss = loss + part.detach()
        if case["step"]:
            grads.append(torch.autograd.grad(part * LOSS_SCALE, z)[0])
    return (loss, torch.cat(grads)) if case["step"] else (loss,)


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "linear":
        x, w = s["x"].detach(), s["w"].detach()
        wq = _exact_rounded(w, "tile", "e4m3")
        y = _exact_rounded(x, "row", "e4m3") @ wq.t()
        if s["b"] is not None:
            y += s["b"].detach().double()
        if not case["step"]:
            return (y,)
        dx = _exact_rounded(s["dy"], "row", case["grad"]) @ wq
        dw = _exact_rounded(s["dy"], "col", case["grad"]).t() @ _exact_rounded(x, "col", "e4m3")
        return (y, dx, dw) if s["b"] is None else (y, dx, dw, s["dy"].double().sum(0))
    if case["op"] == "matmul":
        _, da, _, db = _FORMS[case["form"]]
        a, b = _exact_scaled(s["a"]), _exact_scaled(s["b"])
        return (a if da else a.t()) @ (b.t() if db else b)
    if case["op"] == "quantize":
        out = []
        for blocks in case["blocks"].split("+"):
            out += [_exact_quantize(s["x"], blocks, case["fmt"])[0]] + [None] * (2 if blocks == "tile" else 1)
        return out
    return _exact_distill(s)


# ---------------------------------------------------------------------------------------------------- work
def work(case):
    if case["op"] == "linear":
        t, k, n, b = case["tokens"], case["k"], case["n"], SIZE[case["dtype"]]
        io = t * k + n * k + t * n + (n if case["bias"] else 0)
        return {"bytes": (2 if case["step"] else 1) * io * b, "flops": (6 if case["step"] else 2) * t * k * n}
    if case["op"] == "matmul":
        m, n, k = case["m"], case["n"], case["k"]
        return {"bytes": (m * k + n * k) * (1 + 1 / BLOCK) + m * n * SIZE[case["dtype"]], "flops": 2 * m * n * k}
    if case["op"] == "quantize":
        r, c = case["rows"], case["cols"]
        per = {"row": 1 / BLOCK, "col": 1 / BLOCK, "tile": 2 / BLOCK, "row+col": 1 + 2 / BLOCK}[case["blocks"]]
        return {"bytes": r * c * (SIZE[case["dtype"]] + 1 + per), "flops": 2 * r * c}
    r, v, k = case["rows"], case["vocab"], case["k"]
    return {"bytes": (2 if case["step"] else 1) * r * v * SIZE[case["dtype"]] + r * k * 12,
            "flops": (8 if case["step"] else 4) * r * v}
