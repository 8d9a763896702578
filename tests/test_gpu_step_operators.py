"""The 8-bit layers and the distillation loss together, through the engine's forward, backward and step."""
import copy

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
CONFIG = {
    "optimizer": {"type": "AdamW", "params": {"lr": 1e-3, "betas": (0.9, 0.999), "eps": 1e-6, "weight_decay": 0.01,
                                              "use_hybrid_adam": True}},
    "fp16": {"enabled": True, "loss_scale": 0, "initial_scale_power": 10, "loss_scale_window": 1000, "hysteresis": 2,
             "min_loss_scale": 1},
    "default_chunk_size": 1 << 18,
    "fp8": {"enabled": True, "grad_format": "e5m2"},
    "distillation": {"temperature": 2.0, "tail": "bucket", "weight": 0.5},
}
VOCAB, WIDTH, ROWS, K = 515, 96, 70, 9


def model_func():
    torch.manual_seed(0)
    return torch.nn.Sequential(torch.nn.Embedding(VOCAB, WIDTH), torch.nn.Linear(WIDTH, 130), torch.nn.GELU(),
                               torch.nn.Linear(130, WIDTH), torch.nn.LayerNorm(WIDTH),
                               torch.nn.Linear(WIDTH, VOCAB, bias=False))


def batch(seed):
    gen = torch.Generator().manual_seed(seed)
    tokens = torch.randint(0, VOCAB, (2, ROWS // 2), generator=gen)
    logp = torch.log_softmax(torch.randn(2, ROWS // 2, VOCAB, generator=gen) * 3, -1)
    teacher, idx = logp.topk(K, -1)
    mask = torch.rand(2, ROWS // 2, generator=gen) < 0.8
    return tokens.to(DEV), idx.to(DEV), teacher.to(DEV), mask.to(DEV)


def test_a_step_through_the_engine_is_the_operators_own():
    from patrickstar_b200 import Fp8Linear, distillation_loss, initialize_engine
    engine, opt = initialize_engine(model_func, 0, CONFIG)
    assert sum(isinstance(m, Fp8Linear) for m in engine.module.modules()) == 3
    assert all(m.grad_fmt == "e5m2" for m in engine.module.modules() if isinstance(m, Fp8Linear))
    lay = engine.client.layout
    for it in range(6):
        tokens, idx, teacher, mask = batch(it)
        # the same parameters outside of the engine, at the same places of a buffer: torch's own kernels (the
        # normalisation's backward) choose by alignment, and round differently
        mirror, chunks = copy.deepcopy(engine.module), engine.client.fp16.clone()
        for name, p in mirror.named_parameters():
            at = lay.tensor(name).flat_start(lay.chunk_size)
            p.data = chunks[at:at + p.numel()].view(p.shape)
        scale = engine.loss_scaler.loss_scale
        want = distillation_loss(mirror(tokens), idx, teacher, temperature=2.0, tail="bucket", weight=0.5, mask=mask)
        (want * float(scale)).backward()
        loss = engine.distillation_loss(engine(tokens), idx, teacher, mask=mask)
        assert torch.equal(loss.detach(), want.detach())
        engine.backward(loss)
        for (name, _), q in zip(engine.module.named_parameters(), mirror.parameters()):
            # an embedding's gradient adds up the rows of a token in an order of its own
            got, ref = engine.client.fp16_view(lay.tensor(name)).view(q.shape), q.grad
            if name.startswith("0."):
                assert torch.allclose(got.float(), ref.float(), rtol=2 ** -8, atol=float(ref.abs().max()) * 2 ** -8)
            else:
                assert torch.equal(got, ref), name
        before = [p.detach().clone() for p in engine.module.parameters()]
        engine.step()
        assert opt.step_count == it + 1 and opt.skipped_steps == 0
    assert any(not torch.equal(p, b) for p, b in zip(engine.module.parameters(), before))


def test_an_overflow_in_8_bits_skips_the_step_and_lowers_the_scale():
    from patrickstar_b200 import initialize_engine
    cfg = copy.deepcopy(CONFIG)
    cfg["fp16"]["initial_scale_power"] = 30         # gradients of 16 bits cannot hold this
    for fmt in ("e4m3", "e5m2"):
        cfg["fp8"]["grad_format"] = fmt
        engine, opt = initialize_engine(model_func, 0, cfg)
        start = [p.detach().clone() for p in engine.module.parameters()]
        tokens, idx, teacher, mask = batch(1)
        engine.backward(engine.distillation_loss(engine(tokens), idx, teacher, mask=mask))
        engine.step()
        assert opt.skipped_steps == 1 and engine.loss_scaler.loss_scale == 2 ** 29
        assert all(torch.equal(p, q) for p, q in zip(engine.module.parameters(), start))


def test_without_the_keys_the_layers_stay():
    from patrickstar_b200 import Fp8Linear, initialize_engine
    cfg = {k: v for k, v in CONFIG.items() if k not in ("fp8", "distillation")}
    engine, _ = initialize_engine(model_func, 0, cfg)
    assert not any(isinstance(m, Fp8Linear) for m in engine.module.modules())
    tokens, idx, teacher, mask = batch(2)
    rows = engine.distillation_loss(engine(tokens), idx, teacher, mask=mask, reduction="none")
    assert rows.shape == mask.shape and not rows[~mask].any()
