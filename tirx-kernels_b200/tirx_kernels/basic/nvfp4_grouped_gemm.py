"""``nvfp4_grouped_gemm``: NVFP4 products grouped by expert, with ragged groups, bias and activation.

Rows ``offsets[g] .. offsets[g+1]`` of ``D[rows, N] = act(alpha[g] * A[rows, K] . B[g]^T + bias[g])``, ``B [groups, N, K]``.
``A`` and its scales come from ``nvfp4_quantize_grouped`` (128x4 scale tiles that start anew with every group), ``B``'s from
``nvfp4_quantize`` per group.  ``offsets`` (int32) is read on the device: the host never waits for the routing.  Groups may
be empty; rows that no group has are left as they were.  ``N % 8 == 0``, ``K % 64 == 0``, up to 384 groups.
"""

from __future__ import annotations

from tirx_kernels import _checks, _native, _operator
from tirx_kernels._protocol import KernelHandle

OPERATOR_META = {"name": "nvfp4_grouped_gemm", "category": "basic", "compute_capability": 10}


def _validate(rows: int, groups: int, N: int, K: int, activation: str, out_dtype: str) -> None:
    if rows < 0 or N < 1 or K < 1:
        raise ValueError(f"rows must be >= 0, N and K positive, got {rows}, {N}, {K}")
    if N % 8 != 0 or K % 64 != 0:
        raise ValueError(f"N, K must be divisible by 8, 64 respectively, got {N}, {K}")
    if not 1 <= groups <= _native.MAX_GROUPS:
        raise ValueError(f"groups={groups} outside 1..{_native.MAX_GROUPS}")
    if activation not in _operator.ACTIVATIONS:
        raise ValueError(f"Unsupported activation: {activation}")
    if out_dtype not in _operator.DTYPES:
        raise ValueError(f"Unsupported dtype: {out_dtype}")


class _Runner:
    def __init__(self, rows: int, groups: int, N: int, K: int, activation: str, out_dtype: str):
        _validate(rows, groups, N, K, activation, out_dtype)
        spec = _checks.tensor_spec
        self.specs = (
            spec("A", "uint8", (rows, K // 2)), spec("B", "uint8", (groups, N, K // 2)),
            spec("SFA", "uint8", _checks.grouped_sf_numel(rows, groups, K)),
            spec("SFB", "uint8", groups * _checks.sf_numel(N, K // 16, "128x4")), spec("alpha", "float32", (groups,)),
            spec("offsets", "int32", (groups + 1,)), spec("bias", out_dtype, (groups, N), True), spec("D", out_dtype, (rows, N)),
        )
        self.launch = _native.Launch("b2_nvfp4_grouped_gemm", self.specs, (rows, groups, N, K, _native.DTYPE_CODES[out_dtype],
                                                                      _native.ACTIVATION_CODES[activation]))

    def __call__(self, A, B, SFA, SFB, alpha, offsets, bias, D) -> None:
        self.launch(A, B, SFA, SFB, alpha, offsets, bias, D)


def get_kernel(rows: int, groups: int, N: int, K: int, activation: str = "none", out_dtype: str = "bfloat16", **kwargs) -> KernelHandle:
    return KernelHandle("b2_nvfp4_grouped_gemm", {"launcher": _Runner(rows, groups, N, K, activation, out_dtype),
                                                  "rows": rows, "groups": groups, "N": N, "K": K,
                                                  "activation": activation, "out_dtype": out_dtype})


def quantize_weights(w):
    """bf16/fp16 [groups, N, K] -> (packed [groups, N, K/2], scale tiles of all groups, fp32 encode scale per group)."""
    import torch

    from tirx_kernels.basic.nvfp4_gemm import quantize_operand

    gs = 2688.0 / w.float().abs().amax((1, 2))
    parts = [quantize_operand(w[g], gs[g]) for g in range(w.shape[0])]
    return torch.stack([p for p, _ in parts]), torch.cat([s for _, s in parts]), gs


def _uneven(rows: int, groups: int, generator):
    """Offsets of `groups` groups cut at random places."""
    import torch

    cuts = torch.randint(0, rows + 1, (groups - 1,), generator=generator).sort().values
    return torch.cat([torch.zeros(1, dtype=torch.long), cuts, torch.tensor([rows])])


def prepare_data(rows: int, groups: int, N: int, K: int, out_dtype: str = "bfloat16", bias: bool = True, sizes=None, **kwargs):
    """Seeded (A, B, SFA, SFB, alpha, offsets, bias); `sizes` rows per group, else uneven groups, some of them empty."""
    import torch

    from tirx_kernels.basic import nvfp4_quantize_grouped

    generator = torch.Generator().manual_seed(1)
    draw = lambda *shape: torch.randn(*shape, generator=generator)
    if sizes is None:
        offsets = _uneven(rows, groups, generator)
    else:
        offsets = torch.cat([torch.zeros(1, dtype=torch.long), torch.tensor(list(sizes)).cumsum(0)])
    offsets = offsets.to(torch.int32).cuda()
    x = draw(rows, K).to(torch.bfloat16).cuda()
    gs = (2688.0 / (5.0 + torch.rand(groups, generator=generator))).cuda()
    A = torch.zeros(rows, K // 2, dtype=torch.uint8, device="cuda")
    SFA = torch.full((_checks.grouped_sf_numel(rows, groups, K),), 0xFF, dtype=torch.uint8, device="cuda")  # NaN where no row is
    nvfp4_quantize_grouped.get_kernel("bfloat16", rows, rows, groups, K).config["launcher"](x, None, offsets, A, SFA, gs)
    B, SFB, gs_b = quantize_weights((0.02 * draw(groups, N, K)).to(torch.bfloat16).cuda())
    return A, B, SFA, SFB, 1.0 / (gs * gs_b), offsets, draw(groups, N).to(_operator.torch_dtype(out_dtype)).cuda() if bias else None


def expected(A, B, SFA, SFB, alpha, offsets, bias, activation: str):
    """(the formula in float64 group by group, NaN in rows that no group has; the magnitude of its terms)."""
    import torch

    groups, N, half = B.shape
    want = torch.full((A.shape[0], N), float("nan"), dtype=torch.float64, device=A.device)
    size = torch.zeros_like(want)
    per = SFB.numel() // groups
    ends = offsets.tolist()
    for g, (first, last) in enumerate(zip(ends, ends[1:])):
        rows = torch.arange(last - first, device=A.device)
        a = _checks.dequantize_rows(A[first:last], SFA, (first // 128 + g) * 128 + rows)
        b = _checks.dequantize_rows(B[g], SFB[g * per:(g + 1) * per], torch.arange(N, device=A.device))
        d, terms = a @ b.T * alpha[g].double(), a.abs() @ b.abs().T * alpha[g].double().abs()
        if bias is not None:
            d, terms = d + bias[g].double(), terms + bias[g].double().abs()
        want[first:last], size[first:last] = _checks.activation(d, activation), terms
    return want, size


def run_test(rows: int, groups: int, N: int, K: int, activation: str = "none", out_dtype: str = "bfloat16", bias: bool = True,
             sizes=None, **kwargs) -> None:
    import torch

    from tirx_kernels.basic.nvfp4_gemm_epilogue import tolerance
    from tirx_kernels.runner import compile_kernel

    data = prepare_data(rows, groups, N, K, out_dtype=out_dtype, bias=bias, sizes=sizes)
    D = torch.full((rows, N), float("nan"), dtype=_operator.torch_dtype(out_dtype), device="cuda")
    compile_kernel(get_kernel(rows=rows, groups=groups, N=N, K=K, activation=activation, out_dtype=out_dtype))(*data, D)
    torch.cuda.synchronize()
    _native.nvfp4_grouped_gemm_status()
    want, size = expected(*data, activation)
    nowhere = want.isnan()
    assert torch.equal(D.isnan(), nowhere), "nvfp4_grouped_gemm wrote rows that no group has, or left out some that one has"
    if nowhere.all():
        return
    want, size, got = want[~nowhere], size[~nowhere], D[~nowhere].double()
    excess = ((got - want).abs() - tolerance(want, size, K, out_dtype)).max().item()
    assert excess <= 0, f"nvfp4_grouped_gemm is off by {excess:.3e} more than fp32 sums and one rounding allow"


def flops(rows: int, N: int, K: int) -> int:
    return 2 * rows * N * K


def algorithmic_bytes(rows: int, groups: int, N: int, K: int) -> int:
    """Operands, the weights of the groups that have rows (of `prepare_data`'s uneven ones) and the output."""
    import torch

    touched = int((_uneven(rows, groups, torch.Generator().manual_seed(1)).diff() > 0).sum())
    return rows * K * 9 // 16 + touched * N * K * 9 // 16 + rows * N * 2


def _make_launch(rows, groups, N, K, activation="none", out_dtype="bfloat16", bias=True, sizes=None):
    import torch

    ex = _Runner(rows, groups, N, K, activation, out_dtype)
    data = prepare_data(rows, groups, N, K, out_dtype=out_dtype, bias=bias, sizes=sizes)
    D = torch.empty(rows, N, dtype=_operator.torch_dtype(out_dtype), device="cuda")
    return lambda: ex(*data, D)


def _roofline(us, rows, groups, N, K, **kwargs):
    if rows >= 256 * groups:
        return _checks.roofline_nvfp4(flops(rows, N, K), us)
    return _checks.roofline_hbm(algorithmic_bytes(rows, groups, N, K), us)


def prepare_bench(**kwargs):
    config = _operator.config_only(kwargs)
    get_kernel(**config)
    return _operator.prepared_benchmark(_make_launch, _roofline, config)


def run_bench(**kwargs):
    return _operator.run_prepared(prepare_bench(**kwargs), kwargs)


def _cfg(rows, groups, N, K, activation="none", bias=False, out_dtype="bfloat16"):
    label = f"r{rows}_g{groups}_n{N}_k{K}_{activation}" + ("_bias" if bias else "")
    return {"label": label + {"bfloat16": "", "float16": "_fp16"}[out_dtype], "rows": rows, "groups": groups, "N": N, "K": K,
            "activation": activation, "bias": bias, "out_dtype": out_dtype}


CONFIGS = [
    _cfg(1, 1, 8, 64),
    _cfg(96, 64, 1024, 512),
    _cfg(777, 7, 1352, 1088, "gelu_tanh", True, "float16"),
    _cfg(500, 384, 256, 320, "silu", True),
    _cfg(4096, 8, 2048, 1024),
]
BENCH_CONFIGS = [
    _cfg(96, 64, 4096, 2048),
    _cfg(777, 7, 1352, 1088, "gelu_tanh", True, "float16"),
    _cfg(16384, 16, 4096, 4096),
]
