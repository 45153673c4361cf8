"""``moe_expert_ffn``: the routed NVFP4 feed-forward, from a router's choice to the weighted sum.

``out[t] = residual[t] + sum_k gate[t, k] * W2[e] . q(SiLU(g) * u)``, ``[g | u] = W1[e] . q(x[t])``, ``e = ids[t, k]``: q is the
NVFP4 block quantizer with a fixed encode scale per expert, the products are ``nvfp4_grouped_gemm``, intermediates are in
the 16-bit type of ``x``.  Experts outside ``[0, experts)`` are dropped; a token may name an expert twice.

``expert_ffn`` is the whole of it (one C call of four to six launches, no host synchronisation: it can be captured into a
CUDA graph after a first call); ``plan``, ``dispatch``, ``gated_product`` and ``combine`` are its steps on their own, next to
``nvfp4_quantize_grouped`` and ``nvfp4_grouped_gemm``.
"""

from __future__ import annotations

import functools
from dataclasses import dataclass

from tirx_kernels import _checks, _native, _operator
from tirx_kernels._protocol import KernelHandle

OPERATOR_META = {"name": "moe_expert_ffn", "category": "basic", "compute_capability": 10}


@functools.lru_cache(maxsize=64)
def _weight_specs(experts: int, inner: int, hidden: int) -> tuple:
    if not 1 <= experts <= _native.MAX_GROUPS or hidden % 64 or inner % 64 or not hidden or not inner:
        raise ValueError(f"{experts} experts, hidden={hidden}, inner={inner}: need 1..{_native.MAX_GROUPS} experts, "
                         "hidden and inner multiples of 64")
    spec = _checks.tensor_spec
    scalars = lambda name: spec(name, "float32", (experts,))
    return (spec("w1", "uint8", (experts, 2 * inner, hidden // 2)),
            spec("sf1", "uint8", experts * _checks.sf_numel(2 * inner, hidden // 16, "128x4")), scalars("alpha1"), scalars("gs1"),
            spec("w2", "uint8", (experts, hidden, inner // 2)),
            spec("sf2", "uint8", experts * _checks.sf_numel(hidden, inner // 16, "128x4")), scalars("alpha2"), scalars("gs2"))


@functools.lru_cache(maxsize=64)
def _weight_check(experts: int, inner: int, hidden: int):
    return _native.Launch(None, _weight_specs(experts, inner, hidden))


@functools.lru_cache(maxsize=256)
def _ffn_launch(tokens: int, topk: int, experts: int, hidden: int, inner: int, dtype: str) -> tuple:
    """(launch, workspace bytes) of a shape."""
    spec = _checks.tensor_spec
    rows = dtype, (tokens, hidden)
    specs = (spec("x", *rows), spec("ids", "int32", (tokens, topk)), spec("gates", "float32", (tokens, topk)),
             *_weight_specs(experts, inner, hidden), spec("residual", *rows, True), spec("out", *rows), spec("workspace", "uint8", -1))
    size = workspace_bytes(tokens, topk, experts, hidden, inner)
    return _native.Launch("b2_moe_expert_ffn", specs, (None, tokens, topk, experts, hidden, inner, _native.DTYPE_CODES[dtype])), size


@dataclass(frozen=True)
class ExpertWeights:
    """Quantized weights of all experts and the scales around their products.

    ``w1`` uint8 [experts, 2 * inner, hidden/2] (gate rows in front of up rows), ``w2`` uint8 [experts, hidden, inner/2],
    ``sf1``/``sf2`` their 128x4 scale tiles, expert after expert; ``gs1``/``gs2`` fp32 [experts], the encode scales of the
    two activations; ``alpha1``/``alpha2`` fp32 [experts], 1 / (activation's * weight's encode scale).
    """

    w1: object
    sf1: object
    alpha1: object
    gs1: object
    w2: object
    sf2: object
    alpha2: object
    gs2: object

    def __post_init__(self):
        if getattr(self.w1, "ndim", 0) != 3 or getattr(self.w2, "ndim", 0) != 3 or self.w1.shape[1] % 2:
            raise ValueError("w1 and w2 must be [experts, 2 * inner, hidden / 2] and [experts, hidden, inner / 2]")
        (experts, gate_up, half) = self.w1.shape
        _weight_check(experts, gate_up // 2, half * 2)(self.w1, self.sf1, self.alpha1, self.gs1, self.w2, self.sf2, self.alpha2,
                                                       self.gs2)

    @property
    def experts(self) -> int:
        return self.w1.shape[0]

    @property
    def hidden(self) -> int:
        return self.w1.shape[2] * 2

    @property
    def inner(self) -> int:
        return self.w1.shape[1] // 2


def plan(ids, experts: int):
    """int32 [tokens, topk] -> (offsets [experts + 1], row_token [tokens * topk], position [tokens, topk]), all int32.

    Rows are sorted by expert, in order of (token, k) within an expert; ``row_token`` is -1 behind the last row,
    ``position`` -1 for a dropped assignment."""
    import torch

    if ids.ndim != 2 or ids.shape[1] < 1:
        raise ValueError(f"ids must be [tokens, topk] with topk >= 1, got {tuple(ids.shape)}")
    if not 1 <= experts <= _native.MAX_GROUPS:
        raise ValueError(f"experts={experts} outside 1..{_native.MAX_GROUPS}")
    device = _checks.require_tensors((_checks.tensor_spec("ids", "int32", tuple(ids.shape)),), (ids,))
    tokens, topk = ids.shape
    offsets = torch.empty(experts + 1, dtype=torch.int32, device=ids.device)
    row_token = torch.empty(tokens * topk, dtype=torch.int32, device=ids.device)
    position = torch.empty_like(ids)
    _native.call("b2_moe_plan", device, (ids, offsets, row_token, position), tokens, topk, experts)
    return offsets, row_token, position


def dispatch(x, ids, gs):
    """``plan`` and the quantizer in one: every row of x [tokens, hidden] in NVFP4 for each of its experts.

    ``gs`` fp32 [experts], the encode scales.  Returns (packed [tokens * topk, hidden/2], scale tiles, offsets, position)."""
    import torch

    if x.ndim != 2 or ids.ndim != 2 or not 1 <= ids.shape[1] <= _native.MAX_TOPK:
        raise ValueError(f"x must be [tokens, hidden], ids [tokens, topk] with 1 <= topk <= {_native.MAX_TOPK}")
    (tokens, hidden), topk, experts = x.shape, ids.shape[1], gs.numel()
    dtype = _operator.dtype_name(x.dtype)
    if hidden < 64 or hidden % 64 or not 1 <= experts <= _native.MAX_GROUPS:
        raise ValueError(f"hidden={hidden} must be a multiple of 64, experts={experts} in 1..{_native.MAX_GROUPS}")
    spec = _checks.tensor_spec
    device = _checks.require_tensors((spec("x", dtype, (tokens, hidden)), spec("ids", "int32", (tokens, topk)),
                                      spec("gs", "float32", (experts,))), (x, ids, gs))
    rows = tokens * topk
    out = torch.empty(rows, hidden // 2, dtype=torch.uint8, device=x.device)
    sf = torch.empty(_checks.grouped_sf_numel(rows, experts, hidden), dtype=torch.uint8, device=x.device)
    offsets = torch.zeros(experts + 1, dtype=torch.int32, device=x.device)
    position, row_token = torch.empty_like(ids), torch.empty(rows, dtype=torch.int32, device=x.device)
    _native.call("b2_moe_dispatch", device, (x, ids, gs, offsets, row_token, position, out, sf), tokens, topk, experts, hidden,
                 _native.DTYPE_CODES[dtype])
    return out, sf, offsets, position


def gated_product(A, SFA, offsets, w1, sf1, alpha, gs, dtype: str = "bfloat16"):
    """SiLU(gate) * up of ``[gate | up] = alpha[g] * A . w1[g]^T``, quantized with ``gs[g]``: (packed [rows, inner/2], scale tiles).

    The bytes are those of ``nvfp4_grouped_gemm`` to `dtype` followed by ``nvfp4_quantize_grouped`` with ``fuse_silu``;
    ``w1`` [groups, 2 * inner, hidden/2], inner a multiple of 128.  Rows that no group has are left undefined."""
    import torch

    if A.ndim != 2 or w1.ndim != 3 or w1.shape[1] % 256 or not w1.shape[1]:
        raise ValueError("A must be [rows, hidden / 2], w1 [groups, 2 * inner, hidden / 2] with inner a multiple of 128")
    (rows, half), (groups, gate_up, _) = A.shape, w1.shape
    inner, hidden = gate_up // 2, half * 2
    if hidden < 64 or hidden % 64 or not 1 <= groups <= _native.MAX_GROUPS or dtype not in _operator.DTYPES:
        raise ValueError(f"hidden={hidden}, groups={groups}, dtype={dtype} outside the domain")
    spec = _checks.tensor_spec
    device = _checks.require_tensors(
        (spec("A", "uint8", (rows, half)), spec("SFA", "uint8", _checks.grouped_sf_numel(rows, groups, hidden)),
         spec("offsets", "int32", (groups + 1,)), spec("w1", "uint8", (groups, gate_up, half)),
         spec("sf1", "uint8", groups * _checks.sf_numel(gate_up, hidden // 16, "128x4")), spec("alpha", "float32", (groups,)),
         spec("gs", "float32", (groups,))), (A, SFA, offsets, w1, sf1, alpha, gs))
    out = torch.empty(rows, inner // 2, dtype=torch.uint8, device=A.device)
    sf = torch.empty(_checks.grouped_sf_numel(rows, groups, inner), dtype=torch.uint8, device=A.device)
    _native.call("b2_nvfp4_grouped_gemm_gated", device, (A, w1, SFA, sf1, alpha, offsets, gs, out, sf), rows, groups, inner,
                 hidden, _native.DTYPE_CODES[dtype])
    return out, sf


def combine(y, position, gates, residual=None, out=None):
    """``out[t] = residual[t] + sum_k gates[t, k] * y[position[t, k]]``; positions outside ``y`` add nothing."""
    import torch

    if y.ndim != 2 or position.ndim != 2 or position.shape[1] < 1:
        raise ValueError("y must be [rows, n], position [tokens, topk]")
    (rows, n), (tokens, topk) = y.shape, position.shape
    dtype = _operator.dtype_name(y.dtype)
    if n < 8 or n % 8:
        raise ValueError(f"n={n} must be a positive multiple of 8")
    if out is None:
        out = torch.empty(tokens, n, dtype=y.dtype, device=y.device)
    spec = _checks.tensor_spec
    device = _checks.require_tensors(
        (spec("y", dtype, (rows, n)), spec("position", "int32", (tokens, topk)), spec("gates", "float32", (tokens, topk)),
         spec("residual", dtype, (tokens, n), True), spec("out", dtype, (tokens, n))), (y, position, gates, residual, out))
    _native.call("b2_moe_combine", device, (y, position, gates, residual, out), rows, tokens, topk, n, _native.DTYPE_CODES[dtype])
    return out


def workspace_bytes(tokens: int, topk: int, experts: int, hidden: int, inner: int) -> int:
    size = _native.lib().b2_moe_expert_ffn_workspace_bytes(tokens, topk, experts, hidden, inner)
    if size < 0:
        raise ValueError(f"tokens={tokens} topk={topk} experts={experts} hidden={hidden} inner={inner} outside the domain")
    return size


def expert_ffn(x, ids, gates, weights: ExpertWeights, *, residual=None, out=None, workspace=None):
    """The routed feed-forward of ``x`` [tokens, hidden]; ``ids`` int32 and ``gates`` fp32 [tokens, topk].

    ``out`` (may be ``residual``) and ``workspace`` (uint8, at least ``workspace_bytes(...)``) are allocated on the current
    stream when not given; a workspace serves one call at a time."""
    import torch

    if getattr(ids, "ndim", 0) != 2 or ids.shape[1] < 1:
        raise ValueError("ids must be [tokens, topk] with topk >= 1")
    tokens, topk = ids.shape
    sizes = tokens, topk, *weights.w2.shape[:2], weights.w2.shape[2] * 2
    dtype = _operator.dtype_name(x.dtype)
    launch, size = _ffn_launch(*sizes, dtype)
    if out is None:
        out = torch.empty_like(x)
    if workspace is None:
        workspace = torch.empty(size, dtype=torch.uint8, device=x.device)
    elif workspace.numel() < size:
        raise ValueError(f"workspace must have at least {size} elements, got {workspace.numel()}")
    w = weights
    launch(x, ids, gates, w.w1, w.sf1, w.alpha1, w.gs1, w.w2, w.sf2, w.alpha2, w.gs2, residual, out, workspace, workspace.numel())
    return out


class _Executable:
    def __init__(self, tokens: int, topk: int, experts: int, hidden: int, inner: int, dtype: str):
        if tokens < 0 or not 1 <= topk <= _native.MAX_TOPK:
            raise ValueError(f"tokens must be >= 0 and topk in 1..{_native.MAX_TOPK}, got {tokens}, {topk}")
        if not 1 <= experts <= _native.MAX_GROUPS or hidden < 64 or hidden % 64 or inner < 64 or inner % 64:
            raise ValueError(f"experts={experts} hidden={hidden} inner={inner}: need 1..{_native.MAX_GROUPS} experts, multiples of 64")
        if dtype not in _operator.DTYPES:
            raise ValueError(f"Unsupported dtype: {dtype}")

    def __call__(self, x, ids, gates, weights, out) -> None:
        expert_ffn(x, ids, gates, weights, out=out)


def get_kernel(tokens: int, topk: int, experts: int, hidden: int, inner: int, dtype: str = "bfloat16", **kwargs) -> KernelHandle:
    config = dict(tokens=tokens, topk=topk, experts=experts, hidden=hidden, inner=inner, dtype=dtype)
    return KernelHandle("b2_moe_expert_ffn", {"launcher": _Executable(**config), **config})


def prepare_data(tokens: int, topk: int, experts: int, hidden: int, inner: int, dtype: str = "bfloat16", **kwargs):
    """Seeded (x, ids, gates, weights); distinct experts per token, weights N(0, 0.02) quantized on the GPU."""
    import torch

    from tirx_kernels.basic.nvfp4_grouped_gemm import quantize_weights

    generator = torch.Generator().manual_seed(5)
    draw = lambda *shape: torch.randn(*shape, generator=generator)
    score, ids = (draw(tokens, experts) + 0.5 * draw(experts)).topk(min(topk, experts), dim=-1)
    if topk > experts:
        ids, score = ids.repeat(1, topk)[:, :topk], score.repeat(1, topk)[:, :topk]
    w1, sf1, gsw1 = quantize_weights((0.02 * draw(experts, 2 * inner, hidden)).to(torch.bfloat16).cuda())
    w2, sf2, gsw2 = quantize_weights((0.02 * draw(experts, hidden, inner)).to(torch.bfloat16).cuda())
    gs1 = torch.full((experts,), 2688.0 / 5.0).cuda()
    gs2 = (2688.0 / ((8.0 + torch.rand(experts, generator=generator)) * 0.02**2 * hidden)).cuda()
    weights = ExpertWeights(w1, sf1, 1.0 / (gs1 * gsw1), gs1, w2, sf2, 1.0 / (gs2 * gsw2), gs2)
    return (draw(tokens, hidden).to(_operator.torch_dtype(dtype)).cuda(), ids.to(torch.int32).cuda().contiguous(),
            torch.softmax(score, -1).cuda().contiguous(), weights)


def run_test(tokens: int, topk: int, experts: int, hidden: int, inner: int, dtype: str = "bfloat16", **kwargs) -> None:
    """Against the steps one by one: quantizer and products that are tested on their own, the rest in float64."""
    import torch

    x, ids, gates, weights = prepare_data(tokens, topk, experts, hidden, inner, dtype)
    out = expert_ffn(x, ids, gates, weights)
    torch.cuda.synchronize()
    _native.nvfp4_grouped_gemm_status()
    want = torch.zeros(tokens, hidden, dtype=torch.float64, device="cuda")
    scale = torch.zeros(tokens, hidden, dtype=torch.float64, device="cuda")
    for e in range(experts):
        token, slot = torch.nonzero(ids == e, as_tuple=True)
        if token.numel():
            z = _expert(x[token], weights, e, dtype)
            want.index_add_(0, token, z * gates[token, slot].double()[:, None])
            scale.index_add_(0, token, z.abs() * gates[token, slot].double()[:, None])
    eps = torch.finfo(x.dtype).eps
    # One rounding of the sum and one of each product, as in the steps (which may fall on the other side of a border
    # where fp32 adds in another order), fp32 sums.
    excess = ((out.double() - want).abs() - eps * (want.abs() + scale) - 1e-5 * scale.max()).max().item()
    assert excess <= 0, f"moe_expert_ffn is off by {excess:.3e} more than its roundings allow"


def _expert(x, weights: ExpertWeights, e: int, dtype: str):
    """Rows through one expert by the package's dense kernels, float64 result."""
    import torch

    from tirx_kernels.basic import nvfp4_gemm_epilogue

    rows, hidden, inner = x.shape[0], weights.hidden, weights.inner
    per1, per2 = weights.sf1.numel() // weights.experts, weights.sf2.numel() // weights.experts
    a = torch.empty(rows, hidden // 2, dtype=torch.uint8, device="cuda")
    sfa = torch.empty(_checks.sf_numel(rows, hidden // 16, "128x4"), dtype=torch.uint8, device="cuda")
    y = torch.empty(rows, 2 * inner, dtype=x.dtype, device="cuda")
    _native.nvfp4_quantize(x.contiguous(), a, sfa, weights.gs1[e:e + 1], rows, hidden, dtype, "128x4")
    product = lambda N, K: nvfp4_gemm_epilogue.get_kernel(rows, N, K, out_dtype=dtype).config["launcher"]
    product(2 * inner, hidden)(a, weights.w1[e], sfa, weights.sf1[e * per1:(e + 1) * per1], weights.alpha1[e:e + 1], None, None, y)
    a = torch.empty(rows, inner // 2, dtype=torch.uint8, device="cuda")
    sfa = torch.empty(_checks.sf_numel(rows, inner // 16, "128x4"), dtype=torch.uint8, device="cuda")
    z = torch.empty(rows, hidden, dtype=x.dtype, device="cuda")
    _native.nvfp4_quantize(y, a, sfa, weights.gs2[e:e + 1], rows, inner, dtype, "128x4", fuse_silu=True)
    product(hidden, inner)(a, weights.w2[e], sfa, weights.sf2[e * per2:(e + 1) * per2], weights.alpha2[e:e + 1], None, None, z)
    return z.double()


def flops(tokens: int, topk: int, hidden: int, inner: int) -> int:
    return 6 * tokens * topk * hidden * inner


def algorithmic_bytes(tokens: int, topk: int, experts: int, hidden: int, inner: int) -> int:
    """x, out and the weights of the experts that uniform routing touches."""
    touched = experts * (1.0 - (1.0 - min(1.0, topk / experts)) ** tokens)
    return int(4 * tokens * hidden + touched * 3 * hidden * inner * 9 / 16)


def _make_launch(**config):
    data = prepare_data(**config)
    return lambda: expert_ffn(*data)


def _roofline(us, tokens, topk, experts, hidden, inner, **kwargs):
    if tokens * topk >= 256 * experts:
        return _checks.roofline_nvfp4(flops(tokens, topk, hidden, inner), us)
    return _checks.roofline_hbm(algorithmic_bytes(tokens, topk, experts, hidden, inner), us)


def prepare_bench(**kwargs):
    config = _operator.config_only(kwargs)
    get_kernel(**config)
    return _operator.prepared_benchmark(_make_launch, _roofline, config)


def run_bench(**kwargs):
    return _operator.run_prepared(prepare_bench(**kwargs), kwargs)


def _cfg(tokens, topk, experts, hidden, inner, dtype="bfloat16"):
    label = f"t{tokens}_top{topk}_e{experts}_h{hidden}_i{inner}" + {"bfloat16": "", "float16": "_fp16"}[dtype]
    return {"label": label, "tokens": tokens, "topk": topk, "experts": experts, "hidden": hidden, "inner": inner, "dtype": dtype}


CONFIGS = [_cfg(1, 8, 16, 1024, 256), _cfg(37, 2, 5, 320, 192, "float16"), _cfg(300, 4, 8, 512, 704)]
BENCH_CONFIGS = [_cfg(1, 8, 64, 4096, 1024), _cfg(64, 8, 64, 4096, 1024), _cfg(4096, 4, 32, 2048, 1408)]
