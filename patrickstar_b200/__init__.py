"""patrickstar_b200 — PatrickStar's per-chunk mixed-precision optimizer step on B200.

Public names mirror the reference's for this path:

    from patrickstar_b200 import FP16Adam, DynamicLossScaler, LossScaler, initialize_engine
    from patrickstar_b200 import cpu_adam_op      # create_adam / adam_update / destroy_adam

Operators of the training step around it, which the reference leaves to torch:

    from patrickstar_b200 import fp8_linear, Fp8Linear, block_quantize, block_matmul
    from patrickstar_b200 import distillation_loss, DistillationLoss

Everything that computes goes through ``libps_b200.so`` (hand-written sm_100a
CUDA behind a C ABI, ``include/ps_b200.h``).  There is no CPU or PyTorch
fallback: importing a compute name without the built library raises.
"""
__version__ = "0.1.0"

_LAZY = {
    "FP16Adam": ("fp16_adam", "FP16Adam"),
    "LossScaler": ("loss_scaler", "LossScaler"),
    "DynamicLossScaler": ("loss_scaler", "DynamicLossScaler"),
    "ChunkClient": ("client", "ChunkClient"),
    "ChunkLayout": ("chunk_list", "ChunkLayout"),
    "initialize_engine": ("engine", "initialize_engine"),
    "ChunkStepEngine": ("engine", "ChunkStepEngine"),
    "cpu_adam_op": ("cpu_adam_op", None),
    "BlockQuantized": ("block_fp8", "BlockQuantized"),
    "block_quantize": ("block_fp8", "block_quantize"),
    "block_matmul": ("block_fp8", "block_matmul"),
    "fp8_linear": ("block_fp8", "fp8_linear"),
    "Fp8Linear": ("block_fp8", "Fp8Linear"),
    "use_fp8_linears": ("block_fp8", "use_fp8_linears"),
    "distillation_loss": ("distill_loss", "distillation_loss"),
    "DistillationLoss": ("distill_loss", "DistillationLoss"),
}


def __getattr__(name):
    if name in _LAZY:
        import importlib
        mod, attr = _LAZY[name]
        m = importlib.import_module("." + mod, __name__)
        globals()[name] = m if attr is None else getattr(m, attr)   # looked up once
        return globals()[name]
    raise AttributeError("module %r has no attribute %r" % (__name__, name))
