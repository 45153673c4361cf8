"""``nvfp4_gemm_epilogue``: NVFP4 product with bias, activation and residual in its epilogue.

``D[M,N] = residual + act(alpha * A[M,K] . B[N,K]^T + bias)`` on the operands of ``nvfp4_gemm`` (packed E2M1,
128x4-swizzled E4M3 block scales, ``alpha`` the reciprocal of the product of the two encode scales).  Sums, bias,
activation and residual are fp32 with one rounding to the 16-bit output; ``bias [N]`` and ``residual [M,N]`` have the
output's type and may be None; ``residual`` may be ``D`` itself.  Shapes: any ``M >= 0``, ``N % 8 == 0``, ``K % 64 == 0``
(``nvfp4_gemm`` needs 128 and 256).  The kernel is ``b2_nvfp4_gemm_epilogue`` in the C-ABI library.

Not in the reference's registry: found by name through ``registry.load_kernel`` and the CLIs' ``--kernel``.
"""

from __future__ import annotations

from tirx_kernels import _checks, _native, _operator
from tirx_kernels._protocol import KernelHandle

OPERATOR_META = {"name": "nvfp4_gemm_epilogue", "category": "basic", "compute_capability": 10}


def _validate(M: int, N: int, K: int, activation: str, out_dtype: str) -> None:
    if M < 0 or N < 1 or K < 1:
        raise ValueError(f"M must be >= 0, N and K positive, got {M}, {N}, {K}")
    if N % 8 != 0 or K % 64 != 0:
        raise ValueError(f"N, K must be divisible by 8, 64 respectively, got {N}, {K}")
    if activation not in _operator.ACTIVATIONS:
        raise ValueError(f"Unsupported activation: {activation}")
    if out_dtype not in _operator.DTYPES:
        raise ValueError(f"Unsupported dtype: {out_dtype}")


class _Runner:
    """Executable for one (M, N, K, activation, out_dtype)."""

    def __init__(self, M: int, N: int, K: int, activation: str, out_dtype: str):
        _validate(M, N, K, activation, out_dtype)
        spec = _checks.tensor_spec
        self.specs = (
            spec("A", "uint8", (M, K // 2)), spec("B", "uint8", (N, K // 2)),
            spec("SFA", "uint8", _checks.sf_numel(M, K // 16, "128x4")), spec("SFB", "uint8", _checks.sf_numel(N, K // 16, "128x4")),
            spec("alpha", "float32", 1), spec("bias", out_dtype, (N,), True), spec("residual", out_dtype, (M, N), True),
            spec("D", out_dtype, (M, N)),
        )
        self.launch = _native.Launch("b2_nvfp4_gemm_epilogue", self.specs, (M, N, K, _native.DTYPE_CODES[out_dtype],
                                                                       _native.ACTIVATION_CODES[activation]))

    def __call__(self, A, B, SFA, SFB, alpha, bias, residual, D) -> None:
        self.launch(A, B, SFA, SFB, alpha, bias, residual, D)


def get_kernel(M: int, N: int, K: int, activation: str = "none", out_dtype: str = "bfloat16", **kwargs) -> KernelHandle:
    return KernelHandle("b2_nvfp4_gemm_epilogue", {"launcher": _Runner(M, N, K, activation, out_dtype), "M": M, "N": N,
                                                   "K": K, "activation": activation, "out_dtype": out_dtype})


def prepare_data(M: int, N: int, K: int, out_dtype: str = "bfloat16", bias: bool = True, residual: bool = True, **kwargs):
    """Seeded operands (A ~ N(0,1), B ~ N(0, 0.02)), quantized on the GPU: (A, B, SFA, SFB, alpha, bias, residual)."""
    import torch

    from tirx_kernels.basic.nvfp4_gemm import quantize_operand

    generator = torch.Generator().manual_seed(0)
    draw = lambda *shape: torch.randn(*shape, generator=generator)
    a, b = draw(M, K).to(torch.bfloat16).cuda(), (0.02 * draw(N, K)).to(torch.bfloat16).cuda()
    gs_a, gs_b = 2688.0 / a.float().abs().max(), 2688.0 / b.float().abs().max()
    A, SFA = quantize_operand(a, gs_a)
    B, SFB = quantize_operand(b, gs_b)
    dtype = _operator.torch_dtype(out_dtype)
    return (A, B, SFA, SFB, (1.0 / (gs_a * gs_b)).reshape(1), draw(N).to(dtype).cuda() if bias else None,
            draw(M, N).to(dtype).cuda() if residual else None)


def expected(A, B, SFA, SFB, alpha, bias, residual, activation: str):
    """(the formula in float64, the magnitude of its terms sum |a b| alpha + |bias|), on the operands' device."""
    import torch

    rows = lambda packed: torch.arange(packed.shape[0], device=packed.device)
    a, b = _checks.dequantize_rows(A, SFA, rows(A)), _checks.dequantize_rows(B, SFB, rows(B))
    d, size = a @ b.T * alpha.double(), a.abs() @ b.abs().T * alpha.double().abs()
    if bias is not None:
        d, size = d + bias.double(), size + bias.double().abs()
    d = _checks.activation(d, activation)
    return (d if residual is None else d + residual.double()), size


def tolerance(want, size, K: int, out_dtype: str):
    """How far the kernel may be off, elementwise: half a step of the output type, and what fp32 loses in front of it.

    The tensor cores add 64 products at a time, exactly or with a truncation of 2^-23, and K / 64 such sums one by one,
    each off by at most 2^-23 of the terms; alpha, bias and residual add three roundings; no activation's slope exceeds
    1.13; their approximations are within 2^-20 of max(|v|, 1) (the error function's tail: 1.5e-7)."""
    import torch

    fp32 = 1.13 * (K / 64 + 4) * 2.0**-23 * size + 2.0**-20 * (1 + size.clamp(max=8.0)) + 2.0**-23 * want.abs()
    return torch.finfo(_operator.torch_dtype(out_dtype)).eps / 2 * (want.abs() + fp32) + fp32


def run_test(M: int, N: int, K: int, activation: str = "none", out_dtype: str = "bfloat16", bias: bool = True,
             residual: bool = True, **kwargs) -> None:
    import torch

    from tirx_kernels.runner import compile_kernel

    data = prepare_data(M, N, K, out_dtype=out_dtype, bias=bias, residual=residual)
    D = torch.full((M, N), float("nan"), dtype=_operator.torch_dtype(out_dtype), device="cuda")
    compile_kernel(get_kernel(M=M, N=N, K=K, activation=activation, out_dtype=out_dtype))(*data, D)
    torch.cuda.synchronize()
    _native.nvfp4_grouped_gemm_status()
    want, size = expected(*data, activation)
    excess = ((D.double() - want).abs() - tolerance(want, size, K, out_dtype)).max().item()
    assert excess <= 0, f"nvfp4_gemm_epilogue is off by {excess:.3e} more than fp32 sums and one rounding allow"


def flops(M: int, N: int, K: int) -> int:
    return 2 * M * N * K


def algorithmic_bytes(M: int, N: int, K: int, bias: bool = True, residual: bool = True) -> int:
    return (M + N) * K * 9 // 16 + M * N * 2 * (2 if residual else 1) + (2 * N if bias else 0)


def _make_launch(M, N, K, activation="none", out_dtype="bfloat16", bias=True, residual=True):
    import torch

    ex = _Runner(M, N, K, activation, out_dtype)
    data = prepare_data(M, N, K, out_dtype=out_dtype, bias=bias, residual=residual)
    D = torch.empty(M, N, dtype=_operator.torch_dtype(out_dtype), device="cuda")
    return lambda: ex(*data, D)


def _roofline(us, M, N, K, bias=True, residual=True, **kwargs):
    if M >= 1024:
        return _checks.roofline_nvfp4(flops(M, N, K), us)
    return _checks.roofline_hbm(algorithmic_bytes(M, N, K, bias, residual), us)


def prepare_bench(**kwargs):
    config = _operator.config_only(kwargs)
    get_kernel(**config)
    return _operator.prepared_benchmark(_make_launch, _roofline, config)


def run_bench(**kwargs):
    return _operator.run_prepared(prepare_bench(**kwargs), kwargs)


def _cfg(M, N, K, activation="none", bias=True, residual=True, out_dtype="bfloat16"):
    label = f"{M}x{N}x{K}_{activation}" + ("_bias" if bias else "") + ("_residual" if residual else "")
    return {"label": label + {"bfloat16": "", "float16": "_fp16"}[out_dtype], "M": M, "N": N, "K": K,
            "activation": activation, "bias": bias, "residual": residual, "out_dtype": out_dtype}


CONFIGS = [
    _cfg(1, 8, 64),
    _cfg(16, 8192, 8192),
    _cfg(100, 1352, 1088, "gelu"),
    _cfg(384, 640, 768, "relu", residual=False),
    _cfg(1000, 3592, 7104, "gelu_tanh", residual=False, out_dtype="float16"),
    _cfg(4096, 8192, 4096),
    _cfg(2048, 4096, 4096, "silu", bias=False, residual=False),
]
BENCH_CONFIGS = [
    _cfg(16, 8192, 8192),
    _cfg(1000, 3592, 7104, "gelu", residual=False, out_dtype="float16"),
    _cfg(4096, 8192, 4096),
    _cfg(8192, 28672, 8192, "silu", bias=False, residual=False),
]
