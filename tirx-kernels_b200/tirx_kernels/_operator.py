"""What the operator modules share: type names, and the prepared benchmark of an operator whose launch is one closure."""

from __future__ import annotations

ACTIVATIONS = ("none", "relu", "gelu", "gelu_tanh", "silu")
DTYPES = ("bfloat16", "float16")


def torch_dtype(name: str):
    import torch

    return {"float16": torch.float16, "bfloat16": torch.bfloat16}[name]


def dtype_name(dtype) -> str:
    import torch

    try:
        return {torch.float16: "float16", torch.bfloat16: "bfloat16"}[dtype]
    except KeyError:
        raise ValueError(f"Unsupported dtype: {dtype}") from None


def prepared_benchmark(make_launch, roofline, config: dict):
    """`make_launch(**config)` -> closure that launches once, called on the GPU; `roofline(us, **config)` -> dict."""
    from tirx_kernels.runner import bench, prepared_gpu_benchmark

    def run_gpu(state, *, warmup=None, repeat=None, timer=None, rounds=1, cooldown_s=1.0, **kwargs):
        result = bench({"tirx": make_launch(**state)}, warmup=warmup, repeat=repeat, timer=timer, rounds=rounds,
                       cooldown_s=cooldown_s)
        result["roofline"] = roofline(result["impls"]["tirx"], **state)
        return result

    return prepared_gpu_benchmark(run_gpu, dict(config))


def run_prepared(prepared, kwargs: dict):
    """The one-shot form: the timing protocol's arguments to run_gpu."""
    names = ("warmup", "repeat", "timer", "rounds", "cooldown_s")
    return prepared.run_gpu(**{k: v for k, v in kwargs.items() if k in names})


def config_only(kwargs: dict) -> dict:
    return {k: v for k, v in kwargs.items() if k not in ("warmup", "repeat", "timer", "rounds", "cooldown_s")}
