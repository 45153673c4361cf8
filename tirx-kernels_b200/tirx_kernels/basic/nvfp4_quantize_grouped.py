"""``nvfp4_quantize_grouped``: NVFP4 quantizer that gathers rows and lays their scales out by group.

Row ``r`` of the output is row ``index[r]`` of the input (row ``r`` without an index), quantized as ``nvfp4_quantize``
does with the encode scale of its group; ``fuse_silu`` quantizes SiLU(gate) * up of a ``[in_rows, 2k]`` input.  Scale
factors lie in 128x4 tiles that start anew with every group: group ``g``, rows ``offsets[g] .. offsets[g+1]``, begins at
tile ``offsets[g] // 128 + g``, which is what ``nvfp4_grouped_gemm`` reads.  ``offsets`` is read on the device.  An index
outside the input gives a row of zeros; rows from ``offsets[groups]`` on are left as they were.
"""

from __future__ import annotations

from tirx_kernels import _checks, _native, _operator
from tirx_kernels._protocol import KernelHandle

OPERATOR_META = {"name": "nvfp4_quantize_grouped", "category": "basic", "compute_capability": 10}


def _validate(dtype: str, in_rows: int, rows: int, groups: int, k: int) -> None:
    if dtype not in _operator.DTYPES:
        raise ValueError(f"Unsupported dtype: {dtype}")
    if in_rows < 0 or rows < 0:
        raise ValueError(f"in_rows and rows must be >= 0, got {in_rows}, {rows}")
    if not 1 <= groups <= _native.MAX_GROUPS:
        raise ValueError(f"groups={groups} outside 1..{_native.MAX_GROUPS}")
    if k < 64 or k % 64 != 0:
        raise ValueError(f"k={k} must be a positive multiple of 64")


class _Executable:
    def __init__(self, dtype: str, in_rows: int, rows: int, groups: int, k: int, fuse_silu: bool):
        _validate(dtype, in_rows, rows, groups, k)
        spec = _checks.tensor_spec
        self.specs = (
            spec("x", dtype, (in_rows, k * (2 if fuse_silu else 1))), spec("index", "int32", (rows,), True),
            spec("offsets", "int32", (groups + 1,)), spec("out", "uint8", (rows, k // 2)),
            spec("sf", "uint8", _checks.grouped_sf_numel(rows, groups, k)), spec("global_scale", "float32", (groups,)),
        )
        self.launch = _native.Launch("b2_nvfp4_quantize_grouped", self.specs, (in_rows, rows, groups, k, _native.DTYPE_CODES[dtype],
                                                                          int(fuse_silu)))

    def __call__(self, x, index, offsets, out, sf, global_scale) -> None:
        self.launch(x, index, offsets, out, sf, global_scale)


def get_kernel(dtype: str, in_rows: int, rows: int, groups: int, k: int, fuse_silu: bool = False, **kwargs) -> KernelHandle:
    launcher = _Executable(dtype, in_rows, rows, groups, k, fuse_silu)
    return KernelHandle("b2_nvfp4_quantize_grouped", {"launcher": launcher, "dtype": dtype, "in_rows": in_rows,
                                                      "rows": rows, "groups": groups, "k": k, "fuse_silu": fuse_silu})


def prepare_data(dtype: str, in_rows: int, rows: int, groups: int, k: int, fuse_silu: bool = False, **kwargs):
    """Seeded (x, index, offsets, global_scale); uneven groups, some of them empty."""
    import torch

    generator = torch.Generator().manual_seed(3)
    x = torch.randn(in_rows, k * (2 if fuse_silu else 1), generator=generator).to(_operator.torch_dtype(dtype))
    index = torch.randint(0, in_rows, (rows,), generator=generator, dtype=torch.int32)
    cuts = torch.randint(0, rows + 1, (groups - 1,), generator=generator).sort().values
    offsets = torch.cat([torch.zeros(1, dtype=torch.long), cuts, torch.tensor([rows])]).to(torch.int32)
    gs = 300.0 + 400.0 * torch.rand(groups, generator=generator)
    return x.cuda(), index.cuda(), offsets.cuda(), gs.cuda()


def run_test(dtype: str, in_rows: int, rows: int, groups: int, k: int, fuse_silu: bool = False, **kwargs) -> None:
    """The bytes of every group are those that ``nvfp4_quantize`` gives for its rows with its scale."""
    import torch

    from tirx_kernels.runner import compile_kernel

    x, index, offsets, gs = prepare_data(dtype, in_rows, rows, groups, k, fuse_silu)
    out = torch.full((rows, k // 2), _checks.GUARD_BYTE, dtype=torch.uint8, device="cuda")
    sf = torch.full((_checks.grouped_sf_numel(rows, groups, k),), _checks.GUARD_BYTE, dtype=torch.uint8, device="cuda")
    config = dict(dtype=dtype, in_rows=in_rows, rows=rows, groups=groups, k=k, fuse_silu=fuse_silu)
    compile_kernel(get_kernel(**config))(x, index, offsets, out, sf, gs)
    ends = offsets.tolist()
    untouched = torch.ones_like(sf, dtype=torch.bool)
    tiles = _checks.logical_scale_bytes(sf, sf.numel() // (k // 16), k // 16, "128x4")
    at = _checks.sf_offsets("128x4", sf.numel() // (k // 16), k // 16, sf.device)
    for g, (first, last) in enumerate(zip(ends, ends[1:])):
        m = last - first
        if m == 0:
            continue
        want = torch.empty(m, k // 2, dtype=torch.uint8, device="cuda")
        want_sf = torch.empty(m * (k // 16), dtype=torch.uint8, device="cuda")
        _native.nvfp4_quantize(x[index[first:last].long()].contiguous(), want, want_sf, gs[g:g + 1], m, k, dtype, "linear", fuse_silu)
        start = (first // 128 + g) * 128
        assert torch.equal(out[first:last], want), f"group {g}: packed bytes differ from nvfp4_quantize"
        assert torch.equal(tiles[start:start + m], want_sf.view(m, -1)), f"group {g}: scale bytes differ from nvfp4_quantize"
        untouched[at[start:start + m].reshape(-1)] = False
    assert (sf[untouched] == _checks.GUARD_BYTE).all(), "scale bytes that no row has were written"


def algorithmic_bytes(rows: int, k: int, fuse_silu: bool = False) -> int:
    return rows * k * (4 if fuse_silu else 2) + rows * k * 9 // 16


def _make_launch(dtype, in_rows, rows, groups, k, fuse_silu=False):
    import torch

    ex = _Executable(dtype, in_rows, rows, groups, k, fuse_silu)
    x, index, offsets, gs = prepare_data(dtype, in_rows, rows, groups, k, fuse_silu)
    out = torch.empty(rows, k // 2, dtype=torch.uint8, device="cuda")
    sf = torch.empty(_checks.grouped_sf_numel(rows, groups, k), dtype=torch.uint8, device="cuda")
    return lambda: ex(x, index, offsets, out, sf, gs)


def _roofline(us, rows, k, fuse_silu=False, **kwargs):
    return _checks.roofline_hbm(algorithmic_bytes(rows, k, fuse_silu), us)


def prepare_bench(**kwargs):
    config = _operator.config_only(kwargs)
    get_kernel(**config)
    return _operator.prepared_benchmark(_make_launch, _roofline, config)


def run_bench(**kwargs):
    return _operator.run_prepared(prepare_bench(**kwargs), kwargs)


def _cfg(dtype, in_rows, rows, groups, k, fuse_silu=False):
    short = {"float16": "fp16", "bfloat16": "bf16"}[dtype]
    return {"label": f"{short}_r{rows}_g{groups}_k{k}" + ("_silu" if fuse_silu else ""), "dtype": dtype, "in_rows": in_rows,
            "rows": rows, "groups": groups, "k": k, "fuse_silu": fuse_silu}


CONFIGS = [
    _cfg("bfloat16", 1, 1, 1, 64),
    _cfg("bfloat16", 3, 8, 64, 4096),
    _cfg("float16", 777, 777, 7, 1088),
    _cfg("bfloat16", 500, 2001, 384, 2048),
    _cfg("float16", 300, 300, 5, 1408, True),
    _cfg("bfloat16", 4096, 16384, 32, 2048),
]
BENCH_CONFIGS = [
    _cfg("bfloat16", 1, 8, 64, 4096),
    _cfg("bfloat16", 4096, 16384, 32, 2048),
    _cfg("bfloat16", 16384, 16384, 32, 1408, True),
]
