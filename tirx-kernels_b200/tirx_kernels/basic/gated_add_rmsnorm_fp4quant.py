"""``gated_add_rmsnorm_fp4quant``: the norms after a block and before the next one, with the block's gate and residual scale.

    u = x * rsqrt(mean(x^2) + eps) * w_post        (u = x when w_post is None)
    h = residual_scale * residual + gate * u       (one gate row per `rows_per_gate` rows; 1 when gate is None)
    y = h * rsqrt(mean(h^2) + eps) * w_pre         (h as rounded to the input type)

``h`` goes to ``residual_out`` (may be ``residual``), ``y`` to a tensor of the input type or, with ``quantize``, to packed
E2M1 and E4M3 block scales as ``flashinfer_add_rmsnorm_fp4quant`` gives them (row-major, or 128x4-swizzled with padding
left untouched).  Norms and sums are fp32.  ``H % 16 == 0``, ``16 <= H <= 32768``, any ``M >= 0``.
"""

from __future__ import annotations

from tirx_kernels import _checks, _native, _operator
from tirx_kernels._protocol import KernelHandle

OPERATOR_META = {"name": "gated_add_rmsnorm_fp4quant", "category": "basic", "compute_capability": 10}


def _validate(input_dtype: str, M: int, H: int, rows_per_gate: int) -> None:
    if input_dtype not in _operator.DTYPES:
        raise ValueError(f"Unsupported dtype: {input_dtype}")
    if M < 0 or not 16 <= H <= 32768 or H % 16 != 0:
        raise ValueError(f"M={M} must be >= 0, H={H} a multiple of 16 in [16, 32768]")
    if rows_per_gate < 1:
        raise ValueError(f"rows_per_gate={rows_per_gate} must be >= 1")


class _Executable:
    def __init__(self, input_dtype: str, M: int, H: int, quantize: bool, swizzled: bool, rows_per_gate: int):
        _validate(input_dtype, M, H, rows_per_gate)
        self.quantize = bool(quantize)
        spec = _checks.tensor_spec
        rows = input_dtype, (M, H)
        self.specs = (
            spec("x", *rows), spec("residual", *rows), spec("w_post", input_dtype, (H,), True),
            spec("gate", input_dtype, (_checks.ceil_div(M, rows_per_gate), H), True), spec("w_pre", input_dtype, (H,)),
            spec("residual_out", *rows), spec("y", "uint8", (M, H // 2)) if quantize else spec("y", *rows),
        )
        sf = _checks.sf_numel(M, H // 16, "128x4" if swizzled else "linear") if quantize else -1
        self.specs += (spec("sf", "uint8", sf, not quantize), spec("global_scale", "float32", 1, not quantize))
        self.launch = _native.Launch("b2_gated_add_rmsnorm_fp4quant", self.specs, (
            M, H, rows_per_gate, None, None, _native.DTYPE_CODES[input_dtype], int(self.quantize), int(bool(swizzled))))

    def __call__(self, x, residual, w_post, gate, w_pre, residual_out, y, sf, global_scale, residual_scale: float, eps: float) -> None:
        if not self.quantize and (sf is not None or global_scale is not None):
            raise ValueError("sf and global_scale belong to the quantized form")
        self.launch(x, residual, w_post, gate, w_pre, residual_out, y, sf, global_scale, residual_scale, eps)


def get_kernel(input_dtype: str, M: int, H: int, quantize: bool = True, swizzled: bool = True, rows_per_gate: int = 1, **kwargs) -> KernelHandle:
    config = dict(input_dtype=input_dtype, M=M, H=H, quantize=quantize, swizzled=swizzled, rows_per_gate=rows_per_gate)
    return KernelHandle("b2_gated_add_rmsnorm_fp4quant", {"launcher": _Executable(**config), **config})


def prepare_data(input_dtype: str, M: int, H: int, rows_per_gate: int = 1, post: bool = True, gate: bool = True, **kwargs):
    """Seeded (x, residual, w_post, gate, w_pre, global_scale)."""
    import torch

    generator = torch.Generator().manual_seed(7)
    dtype = _operator.torch_dtype(input_dtype)
    draw = lambda *shape: torch.randn(*shape, generator=generator)
    to = lambda t: t.to(dtype).cuda()
    return (to(draw(M, H)), to(2.0 * draw(M, H)), to(1.0 + 0.1 * draw(H)) if post else None,
            to(0.5 * draw(_checks.ceil_div(M, rows_per_gate), H)) if gate else None, to(1.0 + 0.1 * draw(H)),
            (300.0 + 100.0 * torch.rand(1, generator=generator)).cuda())


def expected(x, residual, w_post, gate, w_pre, rows_per_gate: int, residual_scale: float, eps: float, h=None):
    """(h, y) in float64; with `h`, the stored residual, y is the norm of that one."""
    u = x.double()
    if w_post is not None:
        u = u / (u.square().mean(-1, keepdim=True) + eps).sqrt() * w_post.double()
    if gate is not None:
        u = u * gate.double().repeat_interleave(rows_per_gate, 0)[: x.shape[0]]
    want = residual_scale * residual.double() + u
    v = want if h is None else h.double()
    return want, v / (v.square().mean(-1, keepdim=True) + eps).sqrt() * w_pre.double()


def run_test(input_dtype: str, M: int, H: int, quantize: bool = True, swizzled: bool = True, rows_per_gate: int = 1, post: bool = True,
             gate: bool = True, residual_scale: float = 0.9, eps: float = 1e-6, **kwargs) -> None:
    import torch

    from tirx_kernels.runner import compile_kernel

    x, residual, w_post, g, w_pre, gs = prepare_data(input_dtype, M, H, rows_per_gate, post, gate)
    ex = compile_kernel(get_kernel(input_dtype=input_dtype, M=M, H=H, quantize=quantize, swizzled=swizzled, rows_per_gate=rows_per_gate))
    out = torch.full_like(x, float("nan"))
    layout = "128x4" if swizzled else "linear"
    if quantize:
        y = torch.empty(M, H // 2, dtype=torch.uint8, device="cuda")
        sf = torch.full((_checks.sf_numel(M, H // 16, layout),), _checks.GUARD_BYTE, dtype=torch.uint8, device="cuda")
        ex(x, residual, w_post, g, w_pre, out, y, sf, gs, residual_scale, eps)
    else:
        y = torch.full_like(x, float("nan"))
        ex(x, residual, w_post, g, w_pre, out, y, None, None, residual_scale, eps)
    want_h, want_y = expected(x, residual, w_post, g, w_pre, rows_per_gate, residual_scale, eps, h=out)
    torch.cuda.synchronize()
    _native.gated_add_rmsnorm_fp4quant_status()
    # h: one rounding, and fp32 arithmetic on terms up to |residual| + |u|
    step = torch.finfo(x.dtype).eps
    terms = want_h.abs() + 2 * residual.double().abs()
    assert ((out.double() - want_h).abs() <= step / 2 * want_h.abs() + 2e-6 * terms + 1e-7).all(), "residual differs"
    if not quantize:
        assert ((y.double() - want_y).abs() <= (step / 2 + 4e-6) * want_y.abs() + 1e-7).all(), "normalized rows differ"
        return
    deq = _checks.dequantize(y, sf, layout, global_scale=float(gs.item())).double()
    block = want_y.view(M, -1, 16)
    amax = block.abs().amax(-1, keepdim=True)
    got = _checks.logical_scale_bytes(sf, M, H // 16, layout).view(torch.float8_e4m3fn).double()
    # a scale is within half an E4M3 step of gs * amax / 6 (subnormal steps below 2^-6), a value within half an E2M1 step
    want_scale = (float(gs.item()) * amax[..., 0] / 6).clamp(max=448)
    assert ((got - want_scale).abs() <= want_scale * (2.0**-4 + 1e-5) + 2.0**-10).all(), "scales differ"
    err = (deq.view(M, -1, 16) - block).abs()
    # E2M1 steps are 0.5, 1 and 2 below 2, 4 and 6 of the scale; beyond 6 it saturates (a scale rounded down)
    unit = got[..., None] / float(gs.item())
    half = torch.where(block.abs() <= 2 * unit, 0.25, torch.where(block.abs() <= 4 * unit, 0.5, 1.0)) * unit
    beyond = (block.abs() - 6 * unit).clamp(min=0)
    assert (err <= half * (1 + 1e-4) + beyond + 1e-7).all(), "quantized values differ"
    if swizzled:
        mask = _checks.padding_mask(M, H // 16, layout, sf.device)
        assert (sf[mask] == _checks.GUARD_BYTE).all(), "padding scale positions were written"


def algorithmic_bytes(M: int, H: int, quantize: bool) -> int:
    return M * H * 6 + (M * H * 9 // 16 if quantize else M * H * 2)


def _make_launch(input_dtype, M, H, quantize=True, swizzled=True, rows_per_gate=1, post=True, gate=True):
    import torch

    x, residual, w_post, g, w_pre, gs = prepare_data(input_dtype, M, H, rows_per_gate, post, gate)
    ex = _Executable(input_dtype, M, H, quantize, swizzled, rows_per_gate)
    out = torch.empty_like(x)
    if not quantize:
        y = torch.empty_like(x)
        return lambda: ex(x, residual, w_post, g, w_pre, out, y, None, None, 0.9, 1e-6)
    y = torch.empty(M, H // 2, dtype=torch.uint8, device="cuda")
    sf = torch.empty(_checks.sf_numel(M, H // 16, "128x4" if swizzled else "linear"), dtype=torch.uint8, device="cuda")
    return lambda: ex(x, residual, w_post, g, w_pre, out, y, sf, gs, 0.9, 1e-6)


def _roofline(us, M, H, quantize=True, **kwargs):
    return _checks.roofline_hbm(algorithmic_bytes(M, H, quantize), us)


def prepare_bench(**kwargs):
    config = _operator.config_only(kwargs)
    get_kernel(**config)
    return _operator.prepared_benchmark(_make_launch, _roofline, config)


def run_bench(**kwargs):
    return _operator.run_prepared(prepare_bench(**kwargs), kwargs)


def _cfg(input_dtype, M, H, quantize=True, swizzled=True, rows_per_gate=1, post=True, gate=True):
    short = {"float16": "fp16", "bfloat16": "bf16"}[input_dtype]
    label = f"{short}_m{M}_h{H}" + (("_fp4" + ("_swizzled" if swizzled else "")) if quantize else "") + ("_post" if post else "")
    return {"label": label + (f"_gate{rows_per_gate}" if gate else ""), "input_dtype": input_dtype, "M": M, "H": H, "quantize": quantize,
            "swizzled": swizzled, "rows_per_gate": rows_per_gate, "post": post, "gate": gate}


CONFIGS = [
    _cfg("bfloat16", 3000, 528, rows_per_gate=7),
    _cfg("float16", 3001, 7168, quantize=False, rows_per_gate=1000),
    _cfg("bfloat16", 1200, 16384, swizzled=False, gate=False),
    _cfg("float16", 5000, 1040, post=False, gate=False),
    _cfg("bfloat16", 1, 8192),
    _cfg("bfloat16", 3, 16, gate=False),
    _cfg("float16", 500, 5136, swizzled=False, gate=False),
    _cfg("float16", 77, 1040, rows_per_gate=10, post=False),
    _cfg("bfloat16", 130, 32768, rows_per_gate=64),
    _cfg("bfloat16", 1001, 512, quantize=False, rows_per_gate=1001),
    _cfg("float16", 257, 7168, quantize=False, gate=False, post=False),
]
BENCH_CONFIGS = [
    _cfg("bfloat16", 1, 8192),
    _cfg("bfloat16", 8192, 7168, rows_per_gate=2048),
    _cfg("bfloat16", 8192, 7168, quantize=False, rows_per_gate=2048),
]
